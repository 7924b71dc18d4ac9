"""Arrays exchanged with another library on the same device without a copy (DLPack): shapes and bytes both ways, the
order between the two libraries' streams, lifetimes on either side, and what is refused."""
import gc

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def scale_module(n, et="f32"):
    t = f"tensor<{n}x{et}>"
    return f"""module {{
  func.func @main(%arg0: {t}) -> {t} {{
    %c = stablehlo.constant dense<2.000000e+00> : {t}
    %0 = stablehlo.multiply %arg0, %c : {t}
    return %0 : {t}
  }}
}}
"""


@pytest.mark.parametrize("dt", ["float32", "bfloat16", "int32", "int64", "float64", "bool"])
@pytest.mark.parametrize("shape", [(), (5,), (3, 4), (2, 3, 4), (0, 4), (1, 7)])
def test_round_trip_shares_memory(rx, client, dt, shape):
    n = int(np.prod(shape))
    x = torch.arange(n, device="cuda").reshape(shape).to(getattr(torch, dt))
    turned = x.permute(tuple(reversed(range(len(shape)))))  # first dimension contiguous: the Julia view
    a = rx.from_dlpack(turned, client)
    assert a.shape == tuple(turned.shape)
    back = torch.from_dlpack(a)
    assert back.dtype == x.dtype and back.shape == turned.shape and torch.equal(back, turned)
    if n:
        assert back.data_ptr() == x.data_ptr()
        x.fill_(1)
        torch.cuda.synchronize()
        assert back.bool().all()


def test_results_and_inputs_follow_the_streams(rx, client):
    """A long chain on a stream of torch's feeds the engine, whose result feeds the chain again, with no wait on the host."""
    n = 1 << 22
    f = rx.compile(scale_module(n), client)
    side = torch.cuda.Stream()
    for where in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(where):
            x = torch.ones(n, device="cuda")
            for _ in range(10):
                big = torch.randn(2048, 2048, device="cuda")
                for _ in range(5):
                    big = big @ big * 1e-3  # keeps the stream busy
                x = x + 1
                x = torch.from_dlpack(f(rx.from_dlpack(x, client)))
                gc.collect()
        torch.cuda.synchronize()
        want = 1.0
        for _ in range(10):
            want = (want + 1) * 2
        assert (x == want).all()


def test_memory_goes_back_when_both_sides_are_done(rx, client):
    n = 1 << 24
    f = rx.compile(scale_module(n), client)
    base = client.addressable_devices[0].allocator_stats()["bytes_in_use"]
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    x = torch.ones(n, device="cuda")
    a = rx.from_dlpack(x, client)
    y = f(a)
    out = torch.from_dlpack(y)
    del x, a, y  # the engine's view keeps the input, torch's view the result
    assert (out == 2).all()
    del out
    client.addressable_devices[0].synchronize()
    rx.from_dlpack(torch.ones(4, device="cuda"), client)  # any later call hands back what is free by now
    f(rx.to_rarray(np.ones(n, np.float32), client))
    gc.collect()
    client.addressable_devices[0].synchronize()
    f(rx.to_rarray(np.ones(n, np.float32), client))
    assert client.addressable_devices[0].allocator_stats()["bytes_in_use"] <= base
    assert torch.cuda.memory_allocated() <= held + 4096


def test_unused_capsules_and_many_views(rx, client):
    a = rx.to_rarray(np.arange(8, dtype=np.float32), client)
    for _ in range(100):
        a.__dlpack__()            # nobody takes it
        a.__dlpack__(stream=-1)
    views = [torch.from_dlpack(a) for _ in range(10)]
    del a
    gc.collect()
    assert all(v.tolist() == list(range(8)) for v in views)


def test_refusals(rx, client):
    with pytest.raises(rx.ReactantError, match="first dimension contiguous"):
        rx.from_dlpack(torch.ones(3, 4, device="cuda"), client)  # row-major: its transposed view would do
    with pytest.raises(rx.ReactantError, match="first dimension contiguous"):
        rx.from_dlpack(torch.ones(8, device="cuda")[::2], client)
    with pytest.raises(rx.ReactantError, match="16-byte"):
        rx.from_dlpack(torch.ones(8, device="cuda")[1:], client)
    with pytest.raises(rx.ReactantError, match="not one of this client's"):
        rx.from_dlpack(torch.ones(8), client)
    with pytest.raises(rx.ReactantError, match="element type"):
        rx.from_dlpack(torch.ones(8, device="cuda", dtype=torch.complex64), client)
    a = rx.to_rarray(np.ones(4, np.float32), client)
    with pytest.raises(BufferError):
        a.__dlpack__(copy=True)
    with pytest.raises(rx.ReactantError, match="ambiguous"):
        a.__dlpack__(stream=0)


def test_donated_arrays_are_not_handed_out(rx, client):
    text = scale_module(16).replace("%arg0: tensor<16xf32>", "%arg0: tensor<16xf32> {tf.aliasing_output = 0 : i32}")
    f = rx.compile(text, client)
    a = rx.to_rarray(np.ones(16, np.float32), client)
    old = rx.ConcreteRArray(list(a.data), a.shape, a.dtype)
    f(a)
    with pytest.raises(rx.ReactantError, match="donated"):
        old.__dlpack__()
    assert torch.from_dlpack(a).tolist() == [2.0] * 16


def test_results_are_waited_for_while_another_thread_exports(rx, client):
    """One thread takes its results to another stream while a second one keeps exporting an array of its own: what the
    second thread waits for, recorded while the first one is still queueing work, must not pass for the first one's."""
    import threading

    n, steps = 1 << 24, 60
    f = rx.compile(scale_module(n), client)
    mine = rx.from_dlpack(torch.zeros(16, device="cuda"), client)
    stop = threading.Event()

    def export():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            while not stop.is_set():
                torch.from_dlpack(mine)

    other = threading.Thread(target=export)
    other.start()
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            wrong = torch.zeros((), device="cuda", dtype=torch.int64)
            for k in range(steps):
                x = torch.full((n,), float(k + 1), device="cuda")
                y = torch.from_dlpack(f(f(rx.from_dlpack(x, client))))
                wrong += (y != 4.0 * (k + 1)).sum()
            torch.cuda.current_stream().synchronize()
    finally:
        stop.set()
        other.join()
    assert wrong.item() == 0


CAPTURE = """
import gc, torch
import __graft_entry__ as entry
rx = entry.load_package()
client = rx.default_client()
n = 1 << 16
f = rx.compile('''{module}''', client)
x = torch.ones(n, device="cuda")
a = rx.from_dlpack(x, client)
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    y = torch.from_dlpack(f(a))
side.synchronize()


def refused(act):
    try:
        act()
    except rx.ReactantError as e:
        assert "captured" in str(e), e
        return
    raise AssertionError("not refused")


# in order: a consumer that is being captured; a result let go of on a stream that is being captured; a producer that is
stream = torch.cuda.Stream()
z = f(a)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
w = torch.zeros(n, device="cuda")
with torch.cuda.stream(stream):
    g.capture_begin()
    refused(lambda: torch.from_dlpack(z))
    w += 1
    g.capture_end()
g.replay()
torch.cuda.synchronize()
assert (w == 1).all()

where = y.data_ptr()
with torch.cuda.stream(side):
    g2 = torch.cuda.CUDAGraph()
    g2.capture_begin()
    w += 1
    del y
    gc.collect()
    w += 1
    g2.capture_end()
g2.replay()
torch.cuda.synchronize()
assert (w == 3).all()
for _ in range(4):
    got = torch.from_dlpack(f(a))
    torch.cuda.synchronize()
    assert (got == 2).all()

with torch.cuda.stream(stream):
    g3 = torch.cuda.CUDAGraph()
    g3.capture_begin()
    refused(lambda: rx.from_dlpack(x, client))
    refused(lambda: f(a))
    try:
        g3.capture_end()
    except RuntimeError:
        pass  # a stream that was drawn into the graph never came back to it
torch.cuda.synchronize()
for _ in range(4):
    got = torch.from_dlpack(f(a))
    torch.cuda.synchronize()
    assert (got == 2).all()
print("fine")
"""


def test_streams_under_capture_are_refused(tmp_path):
    """Exchanging with, or executing on, a stream that is being captured into a graph is an error, and the device goes on
    working afterwards.  In a process of its own: the last capture ends in an error of torch's."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "capture.py"
    script.write_text(CAPTURE.replace("{module}", scale_module(1 << 16)))
    env = dict(os.environ, PYTHONPATH=root)
    r = subprocess.run([sys.executable, str(script)], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr


def carried_lookup(rows, features, trips, gradient=False):
    """A loop that carries an array through lookups of its own rows (or through the gradient of one)."""
    t = f"tensor<{rows}x{features}xf32>"
    call = "rx.embedding_grad" if gradient else "rx.embedding"
    return f"""module {{
  func.func @main(%x: {t} {{tf.aliasing_output = 0 : i32}}, %ids: tensor<{rows}xi32>) -> {t} {{
    %c0 = stablehlo.constant dense<0> : tensor<i64>
    %c1 = stablehlo.constant dense<1> : tensor<i64>
    %cn = stablehlo.constant dense<{trips}> : tensor<i64>
    %r:2 = stablehlo.while(%i = %c0, %a = %x) : tensor<i64>, {t}
     cond {{
      %p = stablehlo.compare LT, %i, %cn : (tensor<i64>, tensor<i64>) -> tensor<i1>
      stablehlo.return %p : tensor<i1>
    }} do {{
      %n = stablehlo.add %i, %c1 : tensor<i64>
      %b = stablehlo.custom_call @{call}(%a, %ids) {{api_version = 4 : i32, backend_config = {{scale = 1.0 : f64}}}} : ({t}, tensor<{rows}xi32>) -> {t}
      stablehlo.return %n, %b : tensor<i64>, {t}
    }}
    return %r#1 : {t}
  }}
}}
"""


@pytest.mark.parametrize("gradient", [False, True])
@pytest.mark.parametrize("rows,features", [(6, 8), (40, 64), (700, 1024), (3000, 264)])
@pytest.mark.parametrize("start", [4, 8])
def test_loop_carries_an_array_off_its_vectors(rx, client, ref, rows, features, start, gradient):
    """Memory of another library starts on 16 bytes, not on the eight elements that the lookup stores at once; a donated
    argument that a loop carries may be what the body writes to from the second trip on."""
    rng = np.random.default_rng(rows)
    values = rng.integers(-4, 5, (rows, features)).astype(np.float32)
    ids = rng.permutation(rows).astype(np.int32)  # a gradient of a permutation sums nothing: exact
    ids[rows // 2] = -1
    for trips in (1, 2, 3):
        text = carried_lookup(rows, features, trips, gradient)
        block = torch.full((rows * features + 16,), 7.0, device="cuda")
        x = block[start:start + rows * features].view(rows, features)
        x.copy_(torch.from_numpy(values))
        a = rx.from_dlpack(x.mT, client)
        got = torch.from_dlpack(rx.compile(text, client)(a, rx.to_rarray(ids, client))).mT
        assert np.array_equal(got.cpu().numpy(), ref.run_module(text, [values, ids])[0])
        assert (block[:start] == 7).all() and (block[start + rows * features:] == 7).all()


def updated(n):
    """An array whose first elements are replaced: in place, where the argument may be written."""
    t = f"tensor<{n}xf32>"
    return f"""module {{
  func.func @main(%x: {t} {{tf.aliasing_output = 0 : i32}}, %v: tensor<4xf32>) -> {t} {{
    %c0 = stablehlo.constant dense<0> : tensor<i32>
    %0 = stablehlo.dynamic_update_slice %x, %v, %c0 : ({t}, tensor<4xf32>, tensor<i32>) -> {t}
    return %0 : {t}
  }}
}}
"""


def test_donated_memory_that_another_library_sees_is_left_alone(rx, client):
    """Donation ends an array's life here, not that of the tensor it came from or of the views that were handed out."""
    n = 1 << 20
    f = rx.compile(updated(n), client)
    v = rx.to_rarray(np.full(4, 5, np.float32), client)
    x = torch.ones(n, device="cuda")
    a = rx.from_dlpack(x, client)
    for k in range(2):  # the second time the argument is the first call's result
        f(a, v)
        got = torch.from_dlpack(a)
        torch.cuda.synchronize()
        assert (got[:4] == 5).all() and (got[4:] == 1).all() and (x == 1).all()
        del got
    b = rx.to_rarray(np.ones(n, np.float32), client)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            view = torch.from_dlpack(b)
            before = view.clone()
            f(b, v)
            torch.cuda.synchronize()
            assert torch.equal(view, before)
            del view
            f(b, rx.to_rarray(np.full(4, 1, np.float32), client))
    unordered = torch.from_dlpack(b.__dlpack__(stream=-1))
    f(b, v)
    torch.cuda.synchronize()
    assert (unordered == 1).all()


def test_donated_memory_that_nobody_sees_is_reused(rx, client):
    """Handed out and let go of, or never: the result takes the argument's place."""
    n = 1 << 20
    f = rx.compile(updated(n), client)
    v = rx.to_rarray(np.full(4, 5, np.float32), client)
    b = rx.to_rarray(np.ones(n, np.float32), client)
    view = torch.from_dlpack(b)
    where = view.data_ptr()
    b.__dlpack__()  # nobody takes it
    del view
    f(b, v)
    again = torch.from_dlpack(b)
    assert again.data_ptr() == where and again[:5].tolist() == [5, 5, 5, 5, 1]


def busy_writes(x, value):
    """Work that keeps the current stream busy for a while and then writes the value."""
    big = torch.ones(4096, 4096, device="cuda")
    for _ in range(12):
        big = big @ big * 2.0 ** -12
    return x.copy_(big.flatten()[:1].expand(x.numel()) * 0 + value)


def test_an_imported_array_is_waited_for_where_it_is_handed_on(rx, client):
    """Imported under the stream that writes it, handed on to another stream that has waited for this device before, with
    no execution in between: that stream waits for the producer."""
    n = 1 << 20
    first, second, third = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    f = rx.compile(scale_module(n), client)
    warm = rx.to_rarray(np.ones(n, np.float32), client)
    for k in range(1, 6):
        x = torch.zeros(n, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(first):
            torch.from_dlpack(f(warm)).sum()
        with torch.cuda.stream(second):
            busy_writes(x, k)
            a = rx.from_dlpack(x, client)
        for stream in (first, third):
            with torch.cuda.stream(stream):
                got = torch.from_dlpack(a).sum()
            stream.synchronize()
            assert got.item() == k * n
        second.synchronize()


def test_work_of_a_caller_on_the_device_stream_is_waited_for(rx, client):
    """The device's stream is public: what a caller queues there itself is part of what a consumer waits for."""
    n = 1 << 20
    own = torch.cuda.ExternalStream(rx._lib.lib().RxDeviceStream(client.addressable_devices[0].handle))
    f = rx.compile(scale_module(n), client)
    a = f(rx.to_rarray(np.ones(n, np.float32), client))
    side = torch.cuda.Stream()
    for k in range(1, 4):
        with torch.cuda.stream(side):
            torch.from_dlpack(a).sum()
        torch.cuda.synchronize()
        view = torch.from_dlpack(a)
        with torch.cuda.stream(own):
            busy_writes(view, k)
        with torch.cuda.stream(side):
            got = torch.from_dlpack(a).sum()
        side.synchronize()
        assert got.item() == k * n
        torch.cuda.synchronize()


def test_per_thread_streams_of_different_threads(rx, client):
    """Handed to one thread's own default stream and let go of on another thread, whose own is another stream: the memory is
    used again behind everything."""
    import threading

    n = 1 << 12
    f = rx.compile(scale_module(n), client)
    x = rx.to_rarray(np.ones(n, np.float32), client)
    base = client.addressable_devices[0].allocator_stats()["bytes_in_use"]
    for _ in range(20):
        held = [f(x).__dlpack__(stream=2)]
        t = threading.Thread(target=held.clear)
        t.start()
        t.join()
    assert client.addressable_devices[0].allocator_stats()["bytes_in_use"] == base
    assert np.array_equal(np.asarray(f(x)), np.full(n, 2, np.float32))


def test_stream_of_a_consumer_that_outlives_the_array(rx, client):
    import ctypes

    rt = ctypes.CDLL("libcudart.so.12")
    stream = ctypes.c_void_p()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    n = 1 << 12
    f = rx.compile(scale_module(n), client)
    x = rx.to_rarray(np.ones(n, np.float32), client)
    base = client.addressable_devices[0].allocator_stats()["bytes_in_use"]
    for _ in range(20):
        capsule = f(x).__dlpack__(stream=stream.value)
        del capsule
    assert rt.cudaStreamDestroy(stream) == 0
    assert client.addressable_devices[0].allocator_stats()["bytes_in_use"] == base
    assert np.array_equal(np.asarray(f(x)), np.full(n, 2, np.float32))


BESIDE = """
import gc, threading, torch
import __graft_entry__ as entry
rx = entry.load_package()
client = rx.default_client()
n = 1 << 16
f = rx.compile('''{module}''', client)
held = [rx.from_dlpack(torch.ones(n, device="cuda"), client) for _ in range(4)]
results = [f(a) for a in held]
views = [torch.from_dlpack(f(a)) for a in held]
torch.cuda.synchronize()
w = torch.zeros(n, device="cuda")
done = 0


def captured(act):
    global done
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.add_(1)
        act()
        gc.collect()
        w.add_(1)
    g.replay()
    torch.cuda.synchronize()
    done += 2
    assert (w == done).all()


def elsewhere():
    global got
    with torch.cuda.stream(torch.cuda.Stream()):
        b = f(held[0])
        got = torch.from_dlpack(f(b))
        held.pop()  # (torch's own synchronisation is not allowed meanwhile)


def thread():
    t = threading.Thread(target=elsewhere)
    t.start()
    t.join()


captured(held.pop)                       # an array that was taken over
captured(results.pop)                    # one of the engine's own
captured(views.pop)                      # a view, let go of on the stream that is captured
captured(lambda: results.append(f(held[0])))
captured(thread)
assert (got == 4).all()
for _ in range(4):
    assert (torch.from_dlpack(f(held[0])) == 2).all()
print("fine")
"""


def test_work_beside_a_capture(tmp_path):
    """While a stream of another library is captured into a graph, arrays are let go of and programs run on the device's own
    stream: the capture goes on and holds nothing of it."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "beside.py"
    script.write_text(BESIDE.replace("{module}", scale_module(1 << 16)))
    env = dict(os.environ, PYTHONPATH=root)
    r = subprocess.run([sys.executable, str(script)], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr


@pytest.mark.parametrize("first", ["view", "client"])
def test_memory_outlives_its_client_until_its_consumer_is_done(rx, first):
    """A consumer still reads a view when the client is closed and the array dropped: the owner gets its memory back behind
    that read, whichever goes first."""
    n = 1 << 20
    side = torch.cuda.Stream()
    for k in range(1, 4):
        other = rx.Client(allowed_devices=[0])
        x = torch.full((n,), float(k), device="cuda")
        where = x.data_ptr()
        a = rx.from_dlpack(x, other)
        with torch.cuda.stream(side):
            view = torch.from_dlpack(a)
            busy_writes(torch.empty(4, device="cuda"), 0)
            got = view.clone()
        del x
        if first == "view":
            del view
            other.close()
        else:
            other.close()
            del view
        del a
        gc.collect()
        again = torch.full((n,), -1.0, device="cuda")  # on the current stream, as the tensor was
        torch.cuda.synchronize()
        assert again.data_ptr() == where, "the owner did not get its memory back"
        assert (got == k).all()
        del again


@pytest.mark.parametrize("n", [1 << 12, 1 << 20, 1 << 23])
def test_a_slow_consumer_does_not_hold_up_the_others(rx, client, n):
    """Results of one size go to two streams, one of them busy for a long time: the device's stream never waits for that one
    as long as the other's blocks are free."""
    f = rx.compile(scale_module(n), client)
    a = rx.to_rarray(np.ones(n, np.float32), client)
    slow, fast = torch.cuda.Stream(), torch.cuda.Stream()
    warm = [torch.from_dlpack(f(a)) for _ in range(20)]
    torch.cuda.synchronize()
    del warm
    with torch.cuda.stream(slow):
        for _ in range(3):
            torch.from_dlpack(f(a)).sum()
        torch.cuda._sleep(int(1e9))  # about half a second
        torch.from_dlpack(f(a))
        done = torch.cuda.Event()
        done.record()
    with torch.cuda.stream(fast):
        for _ in range(60):
            got = torch.from_dlpack(f(a))
            fast.synchronize()
    assert not done.query(), "the calls waited for the slow consumer"
    assert (got == 2).all()
    slow.synchronize()


def test_reduction_of_an_array_that_is_still_being_written(rx, client):
    """A full reduction may begin while the kernel in front of it ends; not while a producer still writes what it reads."""
    n = 1 << 20
    total = rx.compile(f"""module {{
  func.func @main(%arg0: tensor<{n}xf32>) -> tensor<f32> {{
    %c = stablehlo.constant dense<0.000000e+00> : tensor<f32>
    %0 = stablehlo.reduce(%arg0 init: %c) applies stablehlo.add across dimensions = [0] : (tensor<{n}xf32>, tensor<f32>) -> tensor<f32>
    return %0 : tensor<f32>
  }}
}}
""", client)
    own = rx.to_rarray(np.ones(n, np.float32), client)
    side = torch.cuda.Stream()
    for k in range(1, 5):
        x = torch.zeros(n, device="cuda")
        torch.cuda.synchronize()
        total(own)
        with torch.cuda.stream(side):
            busy_writes(x, k)
            a = rx.from_dlpack(x, client)
        assert float(total(a)) == k * n


def test_one_array_as_two_arguments_of_which_one_is_donated(rx, client):
    """The other argument keeps its values while the donated one is updated."""
    n = 1 << 16
    t = f"tensor<{n}xf32>"
    f = rx.compile(f"""module {{
  func.func @main(%x: {t} {{tf.aliasing_output = 0 : i32}}, %v: tensor<4xf32>, %y: {t}) -> ({t}, {t}) {{
    %c0 = stablehlo.constant dense<0> : tensor<i32>
    %0 = stablehlo.dynamic_update_slice %x, %v, %c0 : ({t}, tensor<4xf32>, tensor<i32>) -> {t}
    %1 = stablehlo.add %0, %y : {t}
    return %0, %1 : {t}, {t}
  }}
}}
""", client)
    v = rx.to_rarray(np.full(4, 5, np.float32), client)
    x = np.arange(n, dtype=np.float32)
    want = x.copy()
    want[:4] = 5
    for again in range(2):
        a = rx.to_rarray(x, client)
        got = f(a, v, a)
        assert np.array_equal(np.asarray(got[0]), want) and np.array_equal(np.asarray(got[1]), want + x)
        b = rx.to_rarray(x, client)  # and as two
        got = f(b, v, rx.to_rarray(x, client))
        assert np.array_equal(np.asarray(got[0]), want) and np.array_equal(np.asarray(got[1]), want + x)
        same = rx.ConcreteRArray(list(b.data), b.shape, b.dtype)  # two array objects of one buffer
        got = f(b, v, same)
        assert np.array_equal(np.asarray(got[1]), want + want)


def test_an_argument_returned_as_it_came_survives_its_donation(rx, client):
    """A result that is one of the arguments shares its memory; donating either leaves the other's values."""
    n = 1 << 16
    t = f"tensor<{n}xf32>"
    same = rx.compile(f"module {{\n  func.func @main(%x: {t}) -> {t} {{\n    return %x : {t}\n  }}\n}}\n", client)
    f = rx.compile(updated(n), client)
    v = rx.to_rarray(np.full(4, 5, np.float32), client)
    x = np.arange(n, dtype=np.float32)
    a = rx.to_rarray(x, client)
    b = same(a)
    f(b, v)
    assert np.array_equal(np.asarray(a), x) and np.asarray(b)[:4].tolist() == [5, 5, 5, 5]
    c = same(a)
    f(a, v)
    assert np.array_equal(np.asarray(c), x) and np.asarray(a)[:4].tolist() == [5, 5, 5, 5]
