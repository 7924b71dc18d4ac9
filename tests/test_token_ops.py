"""The operators at the two ends of a token model (custom calls): embedding lookup and its gradient, counter-based
dropout, log probabilities of given tokens and their gradient.  CPU: the oracle against direct formulas, against
differences and against torch's autograd; plans, sharding rules and refusals.  GPU: the engine against the oracle.

Tolerances are bounds on the arithmetic, with u = 2^-24 the rounding of a 32-bit operation (2^-8 for a bf16 result):
  lookup      scale and product are rounded once each, the result once
  gradient    n terms summed in any order are off by at most n u times the sum of their magnitudes
  dropout     scale, product and sum; the mask is exact
  logprobs    see `logprob_bounds`
"""
import math

import numpy as np
import pytest

U = 2.0 ** -24
HALF = {"f32": U, "bf16": 2.0 ** -8}  # half a step, relative to the value: finfo.eps / 2


def np_et(rx, et):
    return {"f32": np.float32, "bf16": rx.bfloat16, "i32": np.int32, "i64": np.int64}[et]


def run(rx, client, text, inputs):
    """Row-major in, row-major out (the module's own dims)."""
    out = rx.compile(text, client)(*[rx.to_rarray(np.asarray(x).T, client) for x in inputs])
    return [np.asarray(o).T for o in (out if isinstance(out, tuple) else (out,))]


def close(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(bound, got.shape)[bad][:4])


def some_ids(rng, tokens, vocab, et, odd=True):
    """Few distinct tokens take most of the places; some are outside the table."""
    n = int(np.prod(tokens))
    ids = np.minimum((vocab * rng.random(n) ** 3).astype(np.int64), vocab - 1)
    if odd and n > 3:
        ids[rng.integers(n)] = -1
        ids[rng.integers(n)] = vocab
        if et == "i64":
            ids[rng.integers(n)] = 2 ** 32 + 1  # its low word is a token
    return ids.astype(np.int32 if et == "i32" else np.int64).reshape(tokens)


def values(rx, rng, shape, et, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(np.float32).astype(np_et(rx, et))


def f64(a):
    return np.asarray(a).astype(np.float64)


# ---- CPU: the oracle itself ---------------------------------------------------------------------------------------------
def test_oracle_generator_known_answers(ref):
    # the published known-answer vectors of Philox4x32-10 for the zero and the all-ones counter are checked in torch-free
    # integer arithmetic; the counters reachable here have a zero fourth word
    def philox(c, k):
        c, k = list(c), list(k)
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    words = philox([5, 1, 7, 0], [0xFFFFFFFE, 3])
    bits = [w >> s & 0xFFFF for w in words for s in (0, 16)]
    first = (5 + (1 << 32)) * 8
    for rate in (0.1, 0.5, 0.9):
        got = ref.dropout_mask(8, np.array([-2, 3], np.int32), rate, site=7, first=first)
        assert got.tolist() == [b >= math.floor(rate * 65536 + 0.5) for b in bits]


def test_oracle_gradients_against_differences(ref, rx):
    rng = np.random.default_rng(0)
    T, V, temp = 5, 13, 0.7
    x = rng.standard_normal((T, V))
    ids = np.array([0, 12, -1, 4, 7], np.int32)
    g, gh, gl = rng.standard_normal((3, T))

    def forward(x):
        z = x / temp
        lse = np.log(np.exp(z).sum(1))
        lp = np.where(ids < 0, 0, z[np.arange(T), np.maximum(ids, 0)] - lse)
        p = np.exp(z - lse[:, None])
        return lp, -(p * np.log(p)).sum(1), lse

    lp, h, lse = forward(x)
    text = rx.programs.token_logprobs(T, V, et="f64", temperature=temp)  # the oracle takes any type
    got = ref.run_module(text, [x, ids])
    for a, b in zip(got, (lp, h, lse)):
        np.testing.assert_allclose(a, b, rtol=3e-7, atol=1e-7)
    text = rx.programs.token_logprobs_grad(T, V, et="f64", temperature=temp)
    dx = ref.run_module(text, [x, ids, lse, h, g, gh, gl])[0]
    loss = lambda x: sum((a * b).sum() for a, b in zip(forward(x), (g, gh, gl)))  # noqa: E731
    num = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-5
        num[i] = (loss(x + e) - loss(x - e)) / 2e-5
    # lse, entropy and the incoming gradients reach the oracle rounded to f32 values
    np.testing.assert_allclose(dx, num, rtol=2e-5, atol=2e-6)


def test_oracle_lookup_gradient_is_the_transpose(ref, rx):
    rng = np.random.default_rng(1)
    V, D, T = 11, 3, 9
    table, dy = rng.standard_normal((V, D)), rng.standard_normal((T, D))
    ids = np.array([3, 3, -1, 10, 0, 11, 3, 10, 5], np.int32)
    y = ref.run_module(rx.programs.embedding(V, D, T, et="f64", scale=2.5), [table, ids])[0]
    dt = ref.run_module(rx.programs.embedding_grad(V, D, T, et="f64", out_et="f64", scale=2.5), [dy, ids])[0]
    np.testing.assert_allclose((y * dy).sum(), (table * dt).sum(), rtol=1e-12)
    assert not dt[[1, 2, 4, 6, 7, 8, 9]].any() and not y[[2, 5]].any()


# ---- CPU: plans and refusals ------------------------------------------------------------------------------------------------
def steps(rx, text):
    return [s["kind"] for s in rx.plan_describe(text)["steps"]]


def test_calls_are_single_steps(rx):
    p = rx.programs
    assert steps(rx, p.embedding(100, 64, (3, 5), ids_et="i64")) == ["embedding"]
    assert steps(rx, p.embedding_grad(100, 64, 7)) == ["embedding_grad"]
    assert steps(rx, p.dropout((3, 5), 0.1, residual=True)) == ["dropout"]
    assert steps(rx, p.token_logprobs((2, 3), 50, top_k=5)) == ["token_logprobs"]
    assert steps(rx, p.token_logprobs_grad(6, 50)) == ["token_logprobs_grad"]


def test_mesh_rules(rx):
    p = rx.programs
    assert steps(rx, p.embedding(100, 64, 8, num_partitions=2)) == ["embedding"]
    assert steps(rx, p.embedding_grad(100, 64, 8, num_partitions=2)) == ["embedding_grad", "all_reduce"]
    assert steps(rx, p.token_logprobs_grad(6, 50, num_partitions=2)) == ["token_logprobs_grad"]
    assert "20 elements" in rx.plan_describe(p.dropout((8, 5), 0.1, num_partitions=2))["steps"][0]["note"]
    kinds = steps(rx, p.token_model_grad(512, 256, 512, 512, num_partitions=2))
    assert kinds.count("all_reduce") == 6  # four gradients, two means
    with pytest.raises(rx.ReactantError, match="bf16"):
        rx.plan_describe(p.embedding_grad(100, 64, 8, out_et="bf16", num_partitions=2))
    text = p.token_logprobs(6, 50, num_partitions=2)
    with pytest.raises(rx.ReactantError, match="sharded along the rows' own dimension"):
        rx.plan_describe(text.replace('[{"x"}, {}]', '[{}, {"x"}]', 1))
    text = p.dropout((8, 6), 0.1, num_partitions=2)
    with pytest.raises(rx.ReactantError, match="other than the first"):
        rx.plan_describe(text.replace('[{"x"}, {}]', '[{}, {"x"}]'))
    text = p.embedding(100, 64, 8, num_partitions=2)
    with pytest.raises(rx.ReactantError, match="sharded table"):
        rx.plan_describe(text.replace("tensor<100x64xbf16>,", 'tensor<100x64xbf16> {sdy.sharding = #sdy.sharding<@mesh, [{"x"}, {}]>},', 1))


REFUSALS = [
    ("unknown target", lambda p: p.embedding(8, 4, 3).replace("@rx.embedding", "@rx.other"), 2, "@rx.other"),
    ("unknown setting", lambda p: p.embedding(8, 4, 3).replace("scale =", "scales ="), 12, "scales"),
    ("infinite scale", lambda p: p.embedding(8, 4, 3, scale=math.inf).replace("inf", "0x7FF0000000000000"), 12, "scale"),
    ("half-precision table", lambda p: p.embedding(8, 4, 3, et="f16"), 3, "f16"),
    ("double table", lambda p: p.embedding(8, 4, 3, et="f64"), 3, "f64"),
    ("float ids", lambda p: p.embedding(8, 4, 3, ids_et="f32"), 3, "ids"),
    ("result of another shape", lambda p: p.embedding(8, 4, 3).replace("tensor<3x4xbf16>", "tensor<3x5xbf16>"), 6, "the result"),
    ("one operand", lambda p: p.embedding(8, 4, 3).replace("(%arg0, %arg1)", "(%arg0)").replace("(tensor<8x4xbf16>, tensor<3xi32>) ->", "(tensor<8x4xbf16>) ->"), 12, "operands"),
    ("gradient of another length", lambda p: p.embedding_grad(8, 4, 3).replace("tensor<3xi32>", "tensor<2xi32>"), 6, "the gradient"),
    ("signature that is not the operands'", lambda p: p.embedding_grad(8, 4, 3).replace(": (tensor<3x4xbf16>, tensor<3xi32>)", ": (tensor<3x4xbf16>, tensor<2xi32>)"), 1, "signature"),
    ("rate of one", lambda p: p.dropout(8, 1.0), 12, "rate"),
    ("rate that rounds to one", lambda p: p.dropout(8, 0.999999), 12, "rate"),
    ("negative rate", lambda p: p.dropout(8, -0.1), 12, "rate"),
    ("rate that is no number", lambda p: p.dropout(8, 0.5).replace("0.5 : f64", "0x7FF8000000000000 : f64"), 12, "rate"),
    ("no rate", lambda p: p.dropout(8, 0.5).replace("rate = 0.5 : f64, ", ""), 12, "rate"),
    ("negative site", lambda p: p.dropout(8, 0.5, site=-1), 12, "site"),
    ("site of 33 bits", lambda p: p.dropout(8, 0.5, site=2 ** 32), 12, "site"),
    ("key of one word", lambda p: p.dropout(8, 0.5).replace("tensor<2xi32>", "tensor<1xi32>"), 6, "key"),
    ("residual of another type", lambda p: p.dropout(8, 0.5, residual=True).replace("%arg2: tensor<8xbf16>", "%arg2: tensor<8xf32>").replace("tensor<2xi32>, tensor<8xbf16>) ->", "tensor<2xi32>, tensor<8xf32>) ->"), 3, "residual"),
    ("temperature of zero", lambda p: p.token_logprobs(3, 8, temperature=0.0), 12, "temperature"),
    ("negative temperature", lambda p: p.token_logprobs_grad(3, 8, temperature=-1.0), 12, "temperature"),
    ("temperature below the range of floats", lambda p: p.token_logprobs(3, 8, temperature=1e-300), 12, "temperature"),
    ("more alternatives than tokens", lambda p: p.token_logprobs(3, 8, top_k=9), 12, "top_k"),
    ("more alternatives than are kept", lambda p: p.token_logprobs(3, 800, top_k=65), 12, "top_k"),
    ("five results without alternatives", lambda p: p.token_logprobs(3, 8, top_k=2).replace("top_k = 2", "top_k = 0"), 12, "results"),
    ("double logits", lambda p: p.token_logprobs(3, 8, et="f64"), 3, "logits"),
    ("ids of another shape", lambda p: p.token_logprobs(3, 8).replace("tensor<3xi32>", "tensor<4xi32>"), 6, "ids"),
    ("narrow row values", lambda p: p.token_logprobs_grad(3, 8).replace("tensor<3xf32>", "tensor<3xbf16>"), 3, "lse"),
    ("config that is no dictionary", lambda p: p.embedding(8, 4, 3).replace("{scale = 1.0 : f64}", '"scale=1"'), 1, "dictionary"),
    ("aliased results", lambda p: p.embedding(8, 4, 3).replace("api_version = 4 : i32", "output_operand_aliases = [#stablehlo.alias<0>]"), 2, "output_operand_aliases"),
]


@pytest.mark.parametrize("what,text,code,match", REFUSALS, ids=[r[0] for r in REFUSALS])
def test_refusals(rx, what, text, code, match):
    with pytest.raises(rx.ReactantError, match=match) as e:
        rx.plan_describe(text(rx.programs))
    assert e.value.code == code


def test_operands_are_windows_or_copies(rx):
    """Logits cut out of a padded array are read in place; a transposed array is copied first; a constant zero gradient is not made."""
    p = rx.programs
    cut = p.token_logprobs(4, 50, et="f32").replace("%arg0: tensor<4x50xf32>", "%arg0: tensor<4x64xf32>").replace(
        "    %0:3 =", "    %w = stablehlo.slice %arg0 [0:4, 0:50] : (tensor<4x64xf32>) -> tensor<4x50xf32>\n    %0:3 =").replace("custom_call @rx.token_logprobs(%arg0", "custom_call @rx.token_logprobs(%w")
    assert steps(rx, cut) == ["token_logprobs"]
    turned = p.token_logprobs(4, 50, et="f32").replace("%arg0: tensor<4x50xf32>", "%arg0: tensor<50x4xf32>").replace(
        "    %0:3 =", "    %w = stablehlo.transpose %arg0, dims = [1, 0] : (tensor<50x4xf32>) -> tensor<4x50xf32>\n    %0:3 =").replace("custom_call @rx.token_logprobs(%arg0", "custom_call @rx.token_logprobs(%w")
    assert steps(rx, turned) == ["map", "token_logprobs"]
    kinds = steps(rx, p.token_model_grad(512, 256, 512, 256))
    assert kinds.count("map") == 3  # the loss's share of each row, and the two means


# ---- GPU: the engine against the oracle ---------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 8, 5), (7, 33, 100), ((2, 3), 128, 50), (300, 1000, 999), (129, 2048, 40), (0, 8, 5), (5, 0, 7), (33, 1029, 60), (1, 8191, 3), (40, 3, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("et,out_et,ids_et", [("f32", "f32", "i32"), ("bf16", "bf16", "i64"), ("bf16", "f32", "i32"), ("f32", "bf16", "i64")])
@pytest.mark.parametrize("tokens,features,vocab", SIZES)
def test_embedding(rx, ref, client, tokens, features, vocab, et, out_et, ids_et):
    rng = np.random.default_rng(3)
    table = values(rx, rng, (vocab, features), et)
    ids = some_ids(rng, tokens, vocab, ids_et)
    text = rx.programs.embedding(vocab, features, tokens, et=et, out_et=out_et, ids_et=ids_et, scale=math.sqrt(7.0))
    got, = run(rx, client, text, [table, ids])
    want = ref.run_module(text, [table.astype(np.float32), ids])[0]
    close(f64(got), f64(want), (2 * HALF[out_et] + 2 * U) * np.abs(f64(want)))
    assert not f64(got)[(ids < 0) | (ids >= vocab)].any()


@pytest.mark.gpu
@pytest.mark.parametrize("et,out_et,ids_et", [("f32", "f32", "i64"), ("bf16", "f32", "i32"), ("bf16", "bf16", "i32")])
@pytest.mark.parametrize("tokens,features,vocab", SIZES + [(5000, 24, 3), (4097, 65, 70000), (20000, 8, 300), (8192, 300, 2000), (8193, 301, 20), (70000, 9, 5000)])
def test_embedding_grad(rx, ref, client, tokens, features, vocab, et, out_et, ids_et):
    rng = np.random.default_rng(4)
    n = int(np.prod(tokens))
    dy = values(rx, rng, (tuple(tokens) if isinstance(tokens, tuple) else (tokens,)) + (features,), et)
    ids = some_ids(rng, tokens, vocab, ids_et)
    text = rx.programs.embedding_grad(vocab, features, tokens, et=et, out_et=out_et, ids_et=ids_et, scale=3.0)
    got, = run(rx, client, text, [dy, ids])
    want = ref.run_module(text, [dy.astype(np.float32), ids])[0]
    size = ref.run_module(rx.programs.embedding_grad(vocab, features, tokens, et="f64", out_et="f64", ids_et=ids_et, scale=3.0), [np.abs(f64(dy)), ids])[0]
    live = ids.reshape(-1)[(ids.reshape(-1) >= 0) & (ids.reshape(-1) < vocab)]
    counts = np.bincount(live.astype(np.int64), minlength=vocab)[:, None] if n else np.zeros((vocab, 1))
    close(f64(got), f64(want), (counts + 2) * U * size + 2 * HALF[out_et] * np.abs(f64(want)))
    again, = run(rx, client, text, [dy, ids])
    assert np.array_equal(f64(got), f64(again))  # a fixed order of additions


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("shape,rate,site,residual", [(1, 0.5, 0, False), (7, 0.3, 1, True), ((3, 5), 0.1, 2 ** 32 - 1, False), (1000, 0.0, 3, True), ((129, 255), 0.25, 0, True), ((512, 1024), 0.9, 5, False), (0, 0.5, 0, False),
                                                     (70001, 1e-6, 0, False), (4099, 65535 / 65536, 0, True)])
def test_dropout(rx, ref, client, shape, rate, site, residual, et):
    rng = np.random.default_rng(5)
    x, r = values(rx, rng, shape, et), values(rx, rng, shape, et)
    key = rng.integers(-2 ** 31, 2 ** 31, 2).astype(np.int32)
    text = rx.programs.dropout(shape, rate, et=et, site=site, residual=residual)
    ins = [x, key] + ([r] if residual else [])
    got, = run(rx, client, text, ins)
    want = ref.run_module(text, [a.astype(np.float32) if a.dtype != np.int32 else a for a in ins])[0]
    scale = 65536 / (65536 - math.floor(rate * 65536 + 0.5))
    close(f64(got), f64(want), 2 * U * np.abs(f64(x)) * scale + 2 * HALF[et] * np.abs(f64(want)))
    if not residual and rate:
        mask = ref.dropout_mask(x.size, key, rate, site).reshape(x.shape)
        assert np.array_equal(f64(got) != 0, mask & (f64(x) != 0))


@pytest.mark.gpu
def test_dropout_drops_what_is_not_finite(rx, client, ref):
    key = np.array([1, 2], np.int32)
    mask = ref.dropout_mask(64, key, 0.5)
    for bad in (np.inf, -np.inf, np.nan):
        got, = run(rx, client, rx.programs.dropout(64, 0.5, et="f32"), [np.full(64, bad, np.float32), key])
        assert not got[~mask].any() and not np.isfinite(got[mask]).any()


def logprob_bounds(z, top, h):
    """How far lse, entropy and log probabilities may be off, from u = 2^-24, per row.  z' = z (1 + 2u) of two roundings;
    an exponential of an argument of size R is off by 3 R u of its argument's roundings and 4 u of its own; a thread adds
    at most V / 32 terms and a few levels of merges, each of which rounds (and rescales) once."""
    counts = np.isfinite(z) & (top[..., None] - np.where(np.isfinite(z), z, 0.0) < 105)  # exp(-105) is no 32-bit number any more
    finite = np.where(counts, z, 0.0)
    zmax = np.abs(finite).max(-1)
    spread = (np.where(counts, top[..., None] - z, 0.0)).max(-1)
    s = (3 * spread + z.shape[-1] / 32 + 64) * U
    dz = 2 * 2 * U * zmax
    lse = s + dz + 2 * U * (zmax + np.log(max(2, z.shape[-1])))
    ent = s * (1 + 2 * spread) + 2 * dz + 4 * U * (np.abs(h) + 2 * np.log(max(2, z.shape[-1])) + spread)
    far = np.where(np.isfinite(z), np.abs(z), 0.0).max(-1)  # a token's own logit may lie anywhere
    return lse, ent, lse + dz + 6 * U * (far + zmax + np.log(max(2, z.shape[-1])))


def masked_logits(rx, rng, shape, et, scale=3.0):
    x = (scale * rng.standard_normal(shape)).astype(np.float32)
    if shape[-1] > 4:
        x[rng.random(shape) < 0.1] = -np.inf
    return x.astype(np_et(rx, et))


LOGPROB_SIZES = [(1, 1, 1), (1, 8, 3), ((2, 3), 33, 5), (5, 1000, 64), (3, 1025, 20), (2, 50021, 7), (64, 259, 0), (0, 16, 2), (1, 131072, 32), (300, 64, 1),
                 (37, 64, 64), (35, 128, 33), (33, 256, 20), (9, 257, 32), (5, 4096, 32), (2, 4097, 33), (2400, 1030, 20), (2400, 513, 33), (4800, 8200, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("et,ids_et,temperature", [("f32", "i32", 1.0), ("bf16", "i64", 0.7), ("bf16", "i32", 1.0)])
@pytest.mark.parametrize("tokens,vocab,top_k", LOGPROB_SIZES)
def test_token_logprobs(rx, ref, client, tokens, vocab, top_k, et, ids_et, temperature):
    rng = np.random.default_rng(6)
    shape = (tuple(tokens) if isinstance(tokens, tuple) else (tokens,)) + (vocab,)
    x = masked_logits(rx, rng, shape, et)
    ids = some_ids(rng, tokens, vocab, ids_et)
    text = rx.programs.token_logprobs(tokens, vocab, et=et, ids_et=ids_et, top_k=top_k, temperature=temperature)
    check_logprobs(run(rx, client, text, [x, ids]), ref.run_module(text, [x.astype(np.float32), ids]), x, temperature, top_k)


def check_logprobs(got, want, x, temperature, top_k):
    z = f64(x) / temperature
    b_lse, b_ent, b_lp = logprob_bounds(z, z.max(-1), f64(want[1]))
    close(got[2], want[2], b_lse, "lse")
    close(got[1], want[1], b_ent, "entropy")
    close(got[0], want[0], b_lp, "logprob")
    if top_k:
        assert np.array_equal(got[4], want[4])
        close(got[3], want[3], b_lp[..., None], "top")


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("pattern", ["equal", "rising", "falling", "two values", "zeros of both signs", "one finite", "nothing", "huge", "far apart", "lowest"])
@pytest.mark.parametrize("t,vocab", [(3, 37), (3, 250), (3, 600), (3, 3001), (3, 9001), (2400, 1500)])
def test_token_logprobs_patterns(rx, ref, client, pattern, t, vocab, et):
    """Ties, orders that defeat a running threshold, rows that a mask empties, values at the ends of the range."""
    lowest = -3.3895313892515355e38  # the largest finite bf16
    rows = {"equal": np.full(vocab, 1.25), "rising": np.arange(vocab) * 0.125, "falling": np.arange(vocab) * -0.125, "two values": np.arange(vocab) % 2.0,
            "zeros of both signs": np.where(np.arange(vocab) % 3 == 0, 0.0, -0.0), "one finite": np.where(np.arange(vocab) == vocab - 2, -7.0, -np.inf), "nothing": np.full(vocab, -np.inf),
            "huge": np.where(np.arange(vocab) % 5 == 0, 1e30, -1e30), "far apart": np.arange(vocab) % 7 * 40.0, "lowest": np.where(np.arange(vocab) % 4 == 0, 1.0, lowest)}[pattern]
    x = np.broadcast_to(rows, (t, vocab)).astype(np.float32).astype(np_et(rx, et))
    ids = np.resize(np.array([0, vocab - 2, -1], np.int32), t)
    text = rx.programs.token_logprobs(t, vocab, et=et, top_k=20)
    small = rx.programs.token_logprobs(3, vocab, et=et, top_k=20)  # all rows are alike
    got, want = run(rx, client, text, [x, ids]), [np.resize(w, (t,) + w.shape[1:]) for w in ref.run_module(small, [x[:3].astype(np.float32), ids[:3]])]
    if pattern == "nothing":
        assert (got[2] == -np.inf).all() and not got[1].any() and np.array_equal(got[0], np.resize([-np.inf, -np.inf, 0.0], t))
        assert (got[3] == -np.inf).all() and (got[4] == np.arange(20)).all()
    else:
        check_logprobs(got, want, x, 1.0, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("t,vocab", [(3, 40), (3, 300), (3, 5000), (2400, 1100)])
def test_token_logprobs_not_finite(rx, ref, client, bad, t, vocab):
    """A row with a NaN or +inf has no probabilities; the rows around it are untouched; NaN ranks above everything."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((t, vocab)).astype(np.float32)
    x[1, vocab - 3] = bad
    ids = np.ones(t, np.int32)
    text = rx.programs.token_logprobs(t, vocab, et="f32", top_k=4)
    got, want = run(rx, client, text, [x, ids]), ref.run_module(text, [x, ids])
    assert np.isnan(got[0][1]) and np.isnan(got[1][1]) and np.isnan(got[2][1]) and np.isnan(got[3][1]).all()
    assert np.array_equal(got[4], want[4]) and got[4][1, 0] == vocab - 3
    keep = [0, 2]
    check_logprobs([g[keep] for g in got], [w[keep] for w in want], x[keep], 1.0, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("et,ids_et,temperature", [("f32", "i32", 1.0), ("bf16", "i64", 0.7)])
@pytest.mark.parametrize("tokens,vocab,top_k", [s for s in LOGPROB_SIZES if s[0] != 0] + [(0, 5, 1), (2049, 130, 0)])
def test_token_logprobs_grad(rx, ref, client, tokens, vocab, top_k, et, ids_et, temperature):
    rng = np.random.default_rng(8)
    shape = tuple(tokens) if isinstance(tokens, tuple) else (tokens,)
    x = masked_logits(rx, rng, shape + (vocab,), et)
    if shape[0] > 1:
        x[-1] = -np.inf  # a row that a mask empties
    ids = some_ids(rng, tokens, vocab, ids_et)
    lp, h, lse = ref.run_module(rx.programs.token_logprobs(tokens, vocab, et=et, ids_et=ids_et, temperature=temperature), [x.astype(np.float32), ids])
    g, gh, gl = (rng.standard_normal((3,) + shape) * np.array([1, 0.1, 0.01]).reshape((3,) + (1,) * len(shape))).astype(np.float32)
    text = rx.programs.token_logprobs_grad(tokens, vocab, et=et, ids_et=ids_et, temperature=temperature)
    got, = run(rx, client, text, [x, ids, lse, h, g, gh, gl])
    want = ref.run_module(text, [x.astype(np.float32), ids, lse, h, g, gh, gl])[0]
    z = f64(x) / temperature
    far = np.where(np.isfinite(z) & np.isfinite(lse)[..., None], np.abs(z - np.where(np.isfinite(lse), f64(lse), 0)[..., None]), 0.0)
    p = np.exp(-np.minimum(far, 700.0)) * np.isfinite(z)
    dlogp = 4 * U * (np.abs(np.where(np.isfinite(z), z, 0)) + np.abs(np.where(np.isfinite(lse), f64(lse), 0))[..., None] + far)
    col = lambda v: np.abs(f64(v))[..., None]  # noqa: E731
    size = col(gl) + col(g) + col(gh) * (far + col(h))
    bound = (p * size * (dlogp + 12 * U) + p * col(gh) * dlogp + 4 * U * col(g)) / temperature + 2 * HALF[et] * np.abs(f64(want)) + 2.0 ** -126
    close(f64(got), f64(want), bound)
    if shape[0] > 1:
        assert not f64(got)[-1].any()


@pytest.mark.gpu
def test_windows_of_wider_arrays(rx, ref, client):
    """Operands that are windows (padded vocabulary, odd starts and pitches) or transposed give what their copies give."""
    rng = np.random.default_rng(9)
    for et in ("f32", "bf16"):
        wide = masked_logits(rx, rng, (6, 1111), et)
        ids = np.array([0, 3, -1, 700], np.int32)
        base = rx.programs.token_logprobs(4, 1001, et=et, top_k=6)
        cut = base.replace(f"%arg0: tensor<4x1001x{et}>", f"%arg0: tensor<6x1111x{et}>").replace(
            "    %0:5 =", f"    %w = stablehlo.slice %arg0 [1:5, 7:1008] : (tensor<6x1111x{et}>) -> tensor<4x1001x{et}>\n    %0:5 =").replace("custom_call @rx.token_logprobs(%arg0", "custom_call @rx.token_logprobs(%w")
        for a, b in zip(run(rx, client, cut, [wide, ids]), run(rx, client, base, [np.ascontiguousarray(wide[1:5, 7:1008]), ids])):
            close(a, b, 64 * U * np.maximum(1, np.abs(b)))  # the two may split their sums differently
        table = values(rx, rng, (50, 77), et)
        base = rx.programs.embedding(40, 33, 4, et=et)
        cut = base.replace(f"%arg0: tensor<40x33x{et}>", f"%arg0: tensor<50x77x{et}>").replace(
            "    %0 =", f"    %w = stablehlo.slice %arg0 [3:43, 5:38] : (tensor<50x77x{et}>) -> tensor<40x33x{et}>\n    %0 =").replace("custom_call @rx.embedding(%arg0", "custom_call @rx.embedding(%w")
        ids = np.array([0, 39, 40, 7], np.int32)
        a, = run(rx, client, cut, [table, ids])
        b, = run(rx, client, base, [np.ascontiguousarray(table[3:43, 5:38]), ids])
        assert np.array_equal(f64(a), f64(b)) and f64(a)[0].any()
        dy = values(rx, rng, (9, 77), et)
        ids = np.array([1, 1, 5, 1, 0], np.int32)
        base = rx.programs.embedding_grad(6, 33, 5, et=et)
        cut = base.replace(f"%arg0: tensor<5x33x{et}>", f"%arg0: tensor<9x77x{et}>").replace(
            "    %0 =", f"    %w = stablehlo.slice %arg0 [3:8, 5:38] : (tensor<9x77x{et}>) -> tensor<5x33x{et}>\n    %0 =").replace("custom_call @rx.embedding_grad(%arg0", "custom_call @rx.embedding_grad(%w")
        a, = run(rx, client, cut, [dy, ids])
        b, = run(rx, client, base, [np.ascontiguousarray(dy[3:8, 5:38]), ids])
        assert np.array_equal(f64(a), f64(b))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,features,hidden,tokens", [(512, 256, 512, 256), (300, 96, 160, 77)])
def test_token_model_step(rx, ref, client, vocab, features, hidden, tokens):
    """All of them in one program with the matrix products between, against the float64 oracle.  Every value between
    two steps is rounded to bf16 in both, so what differs is a rounding that falls the other way here and there."""
    rng = np.random.default_rng(10)
    E, U_ = values(rx, rng, (vocab, features), "bf16", features ** -0.5), values(rx, rng, (features, vocab), "bf16", features ** -0.5)
    W1, W2 = values(rx, rng, (features, hidden), "bf16", features ** -0.5), values(rx, rng, (hidden, features), "bf16", hidden ** -0.5)
    ids, targets = some_ids(rng, tokens, vocab, "i32", odd=False), some_ids(rng, tokens, vocab, "i32", odd=False)
    targets[-3:] = -1
    key = np.array([11, -12], np.int32)
    text = rx.programs.token_model_grad(vocab, features, hidden, tokens, rate=0.2)
    ins = [E, W1, W2, U_, ids, targets, key]
    got = run(rx, client, text, ins)
    want = ref.run_module(text, [a.astype(np.float32) if a.dtype not in (np.int32,) else a for a in ins])
    for name, a, b in zip(("dE", "dW1", "dW2", "dU", "loss", "entropy"), got, want):
        a, b = f64(a), f64(b)
        # a bf16 value's half step is 2^-8; a gradient passes through at most six of them in a row
        assert np.linalg.norm(a - b) <= 6 * 2.0 ** -8 * np.linalg.norm(b), name


@pytest.mark.gpu
def test_step_repeats_itself_and_follows_its_key(rx, client):
    rng = np.random.default_rng(11)
    V, F, H, T = 256, 256, 256, 256
    text = rx.programs.token_model_grad(V, F, H, T, rate=0.1)
    p = [values(rx, rng, s, "bf16", F ** -0.5) for s in ((V, F), (F, H), (H, F), (F, V))]
    ids = rng.integers(0, V, T).astype(np.int32)
    ins = p + [ids, np.roll(ids, -1), np.array([1, 2], np.int32)]
    a, b = run(rx, client, text, ins), run(rx, client, text, ins)
    assert all(np.array_equal(f64(x), f64(y)) for x, y in zip(a, b))
    c = run(rx, client, text, p + [ids, np.roll(ids, -1), np.array([1, 3], np.int32)])
    assert not np.array_equal(f64(a[0]), f64(c[0]))  # another key, another mask


@pytest.mark.gpu
@pytest.mark.parametrize("pattern", ["one", "two", "all different", "padding only", "runs of 33", "falling", "first and last"])
@pytest.mark.parametrize("tokens,features", [(31, 8), (1024, 40), (1025, 41), (8193, 8), (9000, 7), (4000, 2056), (4000, 2049)])
def test_embedding_grad_patterns(rx, ref, client, pattern, tokens, features):
    """Runs that fill, cross and end at the borders of the pieces the work is cut into."""
    vocab = 9000
    i = np.arange(tokens)
    ids = {"one": np.full(tokens, 77), "two": np.where(i % 2, 8999, 0), "all different": i % vocab, "padding only": np.where(i % 2, -1, vocab), "runs of 33": i // 33, "falling": (vocab - 1 - i // 8) % vocab,
           "first and last": np.where(i < tokens // 2, 0, vocab - 1)}[pattern].astype(np.int32)
    rng = np.random.default_rng(12)
    dy = rng.integers(-8, 9, (tokens, features)).astype(np.float32)  # whole numbers: every sum is exact
    text = rx.programs.embedding_grad(vocab, features, tokens, et="f32")
    got, = run(rx, client, text, [dy, ids])
    assert np.array_equal(got, ref.run_module(text, [dy, ids])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("pattern", ["random", "equal", "rising", "falling", "one finite", "lowest"])
@pytest.mark.parametrize("t,vocab", [(2, 131079), (30, 65543), (70, 33001), (148, 16411), (149, 33001), (290, 17000)])
def test_token_logprobs_of_few_rows(rx, ref, client, pattern, t, vocab, et):
    """Rows that one, two, four or eight blocks share, with the top tokens anywhere among them."""
    rng = np.random.default_rng(21)
    i = np.arange(vocab)
    rows = {"random": rng.standard_normal(vocab) * 3, "equal": np.full(vocab, 1.25), "rising": i * 2.0 ** -6, "falling": i * -2.0 ** -6,
            "one finite": np.where(i == vocab - 2, -7.0, -np.inf), "lowest": np.where(i > vocab - 30, 1.0, -3.3895313892515355e38)}[pattern]
    x = np.broadcast_to(rows, (t, vocab)).astype(np.float32).astype(np_et(rx, et))
    ids = np.resize(np.array([0, vocab - 2, -1], np.int32), t)
    n = min(t, 3)  # all rows are alike, and three of them have all the ids
    for top_k in (0, 1, 24, 25, 64):
        got = run(rx, client, rx.programs.token_logprobs(t, vocab, et=et, top_k=top_k), [x, ids])
        small = rx.programs.token_logprobs(n, vocab, et=et, top_k=top_k)
        want = ref.run_module(small, [x[:n].astype(np.float32), ids[:n]])
        z = f64(x[:n])
        bounds = logprob_bounds(z, z.max(-1), f64(want[1]))
        want, (b_lse, b_ent, b_lp) = [np.resize(w, (t,) + w.shape[1:]) for w in want], [np.resize(b, t) for b in bounds]
        close(got[2], want[2], b_lse, "lse")
        close(got[1], want[1], b_ent, "entropy")
        close(got[0], want[0], b_lp, "logprob")
        if top_k:
            assert np.array_equal(got[4], want[4])
            close(got[3], want[3], b_lp[..., None], "top")


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [1, 7, 8, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025, 9000])
def test_the_most_likely_token(rx, client, vocab, et):
    """One top token: the lowest index of the largest value, of NaN where there is any, and of -inf where there is nothing else."""
    i = np.arange(vocab)
    rows = [np.full(vocab, 2.0), i % 2.0, -(i % 3.0), np.where(i % 2, 0.0, -0.0), np.where(i == vocab - 1, -7.0, -np.inf), np.full(vocab, -np.inf), i * 0.5, i * -0.5,
            np.where(i >= vocab // 2, np.nan, 5.0), np.where(i == vocab - 1, np.nan, -np.inf), np.where(i >= vocab // 3, np.inf, 1.0), np.full(vocab, -3.3895313892515355e38)]
    x = np.stack(rows).astype(np.float32).astype(np_et(rx, et))
    got = run(rx, client, rx.programs.token_logprobs(len(rows), vocab, et=et, top_k=1), [x, np.zeros(len(rows), np.int32)])
    z = f64(x)
    want = [int(np.argmax(np.isnan(r))) if np.isnan(r).any() else int(np.argmax(r)) for r in z]
    assert got[4][:, 0].tolist() == want
    # The same number as the log probability of that token, which another kernel may give: each is within its bound of the
    # true one, so the two are within twice the bound of each other.
    again = run(rx, client, rx.programs.token_logprobs(len(rows), vocab, et=et, top_k=0), [x, np.array(want, np.int32)])
    finite = np.isfinite(z.max(-1))
    bound = np.zeros(len(rows))
    bound[finite] = 2 * logprob_bounds(z[finite], z[finite].max(-1), f64(again[1])[finite])[2]
    close(got[3][:, 0], again[0], bound, "top")


@pytest.mark.gpu
@pytest.mark.parametrize("features,et,out_et", [(257, "f32", "f32"), (512, "f32", "f32"), (1024, "bf16", "bf16"), (1001, "bf16", "f32")])
@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 64, 65, 700, 1023, 1024, 1025])
def test_embedding_grad_of_few_tokens(rx, ref, client, tokens, features, et, out_et):
    """Rows are found among the sorted tokens: first, last, repeated and absent ones, at every length of the list's pieces."""
    vocab = 2003
    rng = np.random.default_rng(22)
    for ids in (rng.integers(-1, vocab + 1, tokens), np.full(tokens, vocab - 1), np.zeros(tokens), np.arange(tokens) * 2, np.where(np.arange(tokens) % 2, 5, vocab), np.full(tokens, -1)):
        ids = ids.astype(np.int32)
        dy = rng.integers(-2, 3, (tokens, features)).astype(np.float32).astype(np_et(rx, et))
        if out_et == "bf16":
            dy[1:] = 0  # sums stay exact in the result's type
        text = rx.programs.embedding_grad(vocab, features, tokens, et=et, out_et=out_et)
        got, = run(rx, client, text, [dy, ids])
        assert np.array_equal(f64(got), f64(ref.run_module(text, [dy.astype(np.float32), ids])[0]))


@pytest.mark.gpu
def test_empty_vocabulary(rx, client):
    """Nothing to look up, nothing to choose from: rows of zeros, and rows without any probability."""
    ids = np.array([0, -1, 3], np.int32)
    got, = run(rx, client, rx.programs.embedding(0, 5, 3, et="f32"), [np.zeros((0, 5), np.float32), ids])
    assert got.shape == (3, 5) and not got.any()
    got, = run(rx, client, rx.programs.embedding_grad(0, 5, 3, et="f32"), [np.ones((3, 5), np.float32), ids])
    assert got.shape == (0, 5)
    lp, h, lse = run(rx, client, rx.programs.token_logprobs(3, 0, et="f32"), [np.zeros((3, 0), np.float32), ids])
    assert not lp.any() and not h.any() and (lse == -np.inf).all()
    z = np.zeros(3, np.float32)
    got, = run(rx, client, rx.programs.token_logprobs_grad(3, 0, et="f32"), [np.zeros((3, 0), np.float32), ids, lse, h, z, z, z])
    assert got.shape == (3, 0)


def loop_module(n, trips, rate):
    t = f"tensor<{n}xf32>"
    return f"""module {{
  func.func @main(%x: {t}, %key: tensor<2xi32>) -> {t} {{
    %c0 = stablehlo.constant dense<0> : tensor<i64>
    %c1 = stablehlo.constant dense<1> : tensor<i64>
    %cn = stablehlo.constant dense<{trips}> : tensor<i64>
    %one = stablehlo.constant dense<1.000000e+00> : {t}
    %r:2 = stablehlo.while(%i = %c0, %a = %x) : tensor<i64>, {t}
     cond {{
      %p = stablehlo.compare LT, %i, %cn : (tensor<i64>, tensor<i64>) -> tensor<i1>
      stablehlo.return %p : tensor<i1>
    }} do {{
      %n = stablehlo.add %i, %c1 : tensor<i64>
      %b = stablehlo.add %a, %one : {t}
      %d = stablehlo.custom_call @rx.dropout(%b, %key, %a) {{api_version = 4 : i32, backend_config = {{rate = {rate!r} : f64, site = 2 : i64}}}} : ({t}, tensor<2xi32>, {t}) -> {t}
      stablehlo.return %n, %d : tensor<i64>, {t}
    }}
    return %r#1 : {t}
  }}
}}
"""


def test_calls_inside_a_loop_are_planned(rx):
    d = rx.plan_describe(loop_module(100, 3, 0.25))
    loop = next(s for s in d["steps"] if s["kind"] == "loop")
    assert "dropout" in [s["kind"] for s in loop["body"]]


@pytest.mark.gpu
def test_calls_inside_a_loop(rx, ref, client):
    x, key = np.arange(1000, dtype=np.float32), np.array([5, 6], np.int32)
    for trips in (1, 2, 5):
        text = loop_module(1000, trips, 0.25)
        got, = run(rx, client, text, [x, key])
        want = ref.run_module(text, [x, key])[0]
        close(got, want, 8 * trips * U * np.abs(f64(want)))


@pytest.mark.gpu
def test_threads_share_a_device(rx, ref, client):
    """Calls of several host threads at once, each with its own arrays, give what they give one after another."""
    from concurrent.futures import ThreadPoolExecutor
    rng = np.random.default_rng(13)
    V, D, T = 5000, 72, 12000
    text = rx.programs.embedding_grad(V, D, T, et="f32")
    thunk = rx.compile(text, client)
    sets = []
    for _ in range(4):
        dy, ids = rng.integers(-4, 5, (T, D)).astype(np.float32), some_ids(rng, T, V, "i32")
        sets.append((rx.to_rarray(dy.T, client), rx.to_rarray(ids, client), ref.run_module(text, [dy, ids])[0]))

    def work(k):
        a, b, want = sets[k % 4]
        return all(np.array_equal(np.asarray(thunk(a, b)).T, want) for _ in range(5))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(8)))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(rx, client):
    """More than 2^31 elements in the large operand or result: the last rows are what they are alone.  (Arrays are made on
    the device and handed over; rows that are left out of the comparison are there for their addresses.)"""
    torch = pytest.importorskip("torch")
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    cases = torch.device("cuda")
    call = lambda text, *a: [torch.from_dlpack(o) for o in (lambda r: r if isinstance(r, tuple) else (r,))(rx.compile(text, client)(*[rx.from_dlpack(t.mT if t.dim() == 2 else t, client) for t in a]))]  # noqa: E731
    same = lambda a, b: torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b)  # noqa: E731
    T, V, tail = 16500, 131071, 700  # rows that do not start on 16 bytes
    x = torch.randn(T, V, device=cases, dtype=torch.bfloat16, generator=gen)
    ids = torch.randint(0, V, (T,), device=cases, generator=gen, dtype=torch.int32)
    whole = call(rx.programs.token_logprobs(T, V, top_k=3), x, ids)
    part = call(rx.programs.token_logprobs(tail, V, top_k=3), x[-tail:].clone(), ids[-tail:].clone())
    for a, b in zip(whole, part):
        a = a.mT if a.dim() == 2 else a
        b = b.mT if b.dim() == 2 else b
        if a.dtype == torch.int32:
            assert torch.equal(a[-tail:], b)
        else:
            assert (a[-tail:] - b).abs().max() <= 64 * U * 16  # the two may be cut differently: 64 roundings of values up to 16
    g = torch.randn(T, device=cases, generator=gen)
    zero = torch.zeros_like(g)
    grad = call(rx.programs.token_logprobs_grad(T, V), x, ids, whole[2], whole[1], g, zero, zero)[0].mT
    want = call(rx.programs.token_logprobs_grad(tail, V), x[-tail:].clone(), ids[-tail:].clone(), whole[2][-tail:].clone(), whole[1][-tail:].clone(), g[-tail:].clone(), zero[-tail:].clone(), zero[-tail:].clone())[0].mT
    assert same(grad[-tail:].contiguous(), want.contiguous())
    # the same memory as activations to drop, and as a table
    key = torch.tensor([7, 8], device=cases, dtype=torch.int32)
    dropped = call(rx.programs.dropout((T, V), 0.5), x, key)[0].mT
    n = 8 * 1000
    flat = dropped.reshape(-1)[-n:].float()
    kept = flat != 0
    assert ((flat == 2 * x.reshape(-1)[-n:].float()) | ~kept).all() and 0.45 < kept.float().mean() < 0.55
    del dropped, grad
    looked = call(rx.programs.embedding(T, V, 40, scale=1.0), x, torch.arange(T - 40, T, device=cases, dtype=torch.int32))[0].mT
    assert same(looked.contiguous(), x[-40:])
    out = call(rx.programs.embedding(40, V, T), x[:40].clone(), (torch.arange(T, device=cases, dtype=torch.int32) % 40))[0].mT
    assert same(out[-tail:].contiguous(), x[:40][(torch.arange(T, device=cases) % 40)[-tail:]])
    del out
    d = call(rx.programs.embedding_grad(T, V, 5, et="bf16", out_et="bf16"), x[:5].clone(), torch.tensor([T - 1, 0, T - 1, 77, -1], device=cases, dtype=torch.int32))[0].mT
    assert same(d[T - 1].contiguous(), (x[0].float() + x[2].float()).to(torch.bfloat16)) and same(d[77].contiguous(), x[3]) and not d[-700:-1].any()


def test_sizes_beyond_what_rows_are_counted_in(rx):
    """Places inside a row, tokens and rows are 32-bit numbers: the largest are planned, longer ones refused."""
    p, most = rx.programs, 2 ** 31 - 1
    for build in (p.embedding, p.embedding_grad):
        assert steps(rx, build(1, most, 1)) and steps(rx, build(most, 8, 1)) and steps(rx, build(8, 8, most))
        for vocab, features, tokens in ((1, most + 1, 1), (2, most + 2, 3), (most + 1, 8, 1), (8, 8, most + 1)):
            with pytest.raises(rx.ReactantError, match="2\\^31") as e:
                rx.plan_describe(build(vocab, features, tokens))
            assert e.value.code == 13
    for build in (p.token_logprobs, p.token_logprobs_grad):
        with pytest.raises(rx.ReactantError, match="2\\^31"):
            rx.plan_describe(build(1, most + 1))
    assert steps(rx, p.dropout((most + 1,), 0.5)) == ["dropout"]  # elements are counted in 64 bits


@pytest.mark.gpu
@pytest.mark.parametrize("features", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 33])
def test_longest_rows(rx, client, features):
    """Rows whose last places are near 2^31: looked up, and their gradient with its zeros, whole and nothing behind them."""
    torch = pytest.importorskip("torch")
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    x = torch.randint(-2 ** 15, 2 ** 15, (2, features), device="cuda", dtype=torch.int16)
    x &= 0x3FFF  # any finite positive number
    table = x.view(torch.bfloat16)
    call = lambda text, *a: torch.from_dlpack(rx.compile(text, client)(*[rx.from_dlpack(t.mT if t.dim() == 2 else t, client) for t in a])).mT  # noqa: E731
    ids = torch.tensor([1, 0, 2], device="cuda", dtype=torch.int32)
    got = call(rx.programs.embedding(2, features, 3), table, ids).view(torch.int16)
    assert torch.equal(got[0], x[1]) and torch.equal(got[1], x[0]) and not got[2].any()
    del got
    got = call(rx.programs.embedding_grad(3, features, 2, out_et="bf16"), table, ids[:2].clone()).view(torch.int16)
    assert torch.equal(got[0], x[1]) and torch.equal(got[1], x[0]) and not got[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("et,t,vocab,temperature,peak", [("f32", 512, 50016, 0.7, 6.0), ("f32", 512, 50016, 1.0, 20.0), ("bf16", 256, 131072, 1.0, 6.0), ("f32", 2400, 4100, 1.0, 6.0), ("bf16", 5000, 16500, 0.7, 14.0),
                                                        ("f32", 64, 65536, 1.0, 12.0), ("f32", 2000, 900, 1.0, 12.0)])
def test_entropy_of_peaked_rows(rx, client, et, t, vocab, temperature, peak):
    """One token stands out, by little or by much: the entropy is a small difference of larger numbers.  The definition
    evaluated in 32 bits refers to the row's largest logit; a kernel in one pass cannot, and may lose as much again, and
    the half step U of a sum that lies next to one."""
    rng = np.random.default_rng(31)
    x = (2.5 * rng.standard_normal((t, vocab))).astype(np.float32)
    ids = rng.integers(0, vocab, t).astype(np.int32)
    x[np.arange(t), ids] += np.float32(peak)
    x = x.astype(np_et(rx, et))
    got = run(rx, client, rx.programs.token_logprobs(t, vocab, et=et, temperature=temperature), [x, ids])[1]

    def entropy(z):
        d = z - z.max(-1, keepdims=True)
        e = np.exp(d)
        s = e.sum(-1)
        return np.log(s) - (e * d).sum(-1) / s

    want = entropy(f64(x) / temperature)
    plain = entropy(x.astype(np.float32) / np.float32(temperature))
    rms = lambda v: math.sqrt((v ** 2).mean())  # noqa: E731
    assert rms(f64(got) - want) <= 2 * rms(f64(plain) - want) + U


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("t,vocab,pitch,start", [(4, 1001, 1111, 7), (3, 64, 67, 0), (5, 130, 261, 3), (40, 999, 1001, 1), (2, 40003, 40010, 5), (1, 5000, 5003, 1), (300, 260, 263, 0), (6, 2048, 2056, 3), (7, 2048, 2052, 0)])
def test_gradient_of_windows_of_wider_logits(rx, client, t, vocab, pitch, start, et):
    """Logits that lie otherwise than their gradient does (another pitch, another start) give, bit for bit, what their copy gives."""
    rng = np.random.default_rng(32)
    wide = masked_logits(rx, rng, (t + 2, pitch), et)
    x = np.ascontiguousarray(wide[1:t + 1, start:start + vocab])
    ids = some_ids(rng, t, vocab, "i32")
    lse, h, g, gh, gl = rng.standard_normal((5, t)).astype(np.float32)
    lse += 12
    base = rx.programs.token_logprobs_grad(t, vocab, et=et, temperature=0.8)
    cut = base.replace(f"%arg0: tensor<{t}x{vocab}x{et}>", f"%arg0: tensor<{t + 2}x{pitch}x{et}>").replace(
        "    %0 =", f"    %w = stablehlo.slice %arg0 [1:{t + 1}, {start}:{start + vocab}] : (tensor<{t + 2}x{pitch}x{et}>) -> tensor<{t}x{vocab}x{et}>\n    %0 =").replace(
        "custom_call @rx.token_logprobs_grad(%arg0", "custom_call @rx.token_logprobs_grad(%w")
    assert steps(rx, cut) == ["token_logprobs_grad"]  # read in place
    a, = run(rx, client, cut, [wide, ids, lse, h, g, gh, gl])
    b, = run(rx, client, base, [x, ids, lse, h, g, gh, gl])
    assert np.array_equal(f64(a), f64(b)) and f64(a).any()


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,residual", [(1, 7, False), (3, 5, True), (64, 129, True), (700, 1024, False), (33, 1001, False)])
def test_dropout_of_windows(rx, ref, client, rows, cols, residual, et):
    """Operands that start anywhere inside their arrays."""
    rng = np.random.default_rng(33)
    wide, r = values(rx, rng, (rows + 3, cols), et), values(rx, rng, (rows, cols), et)
    key = np.array([3, -4], np.int32)
    base = rx.programs.dropout((rows, cols), 0.4, et=et, site=2, residual=residual)
    cut = base.replace(f"%arg0: tensor<{rows}x{cols}x{et}>", f"%arg0: tensor<{rows + 3}x{cols}x{et}>").replace(
        "    %0 =", f"    %w = stablehlo.slice %arg0 [3:{rows + 3}, 0:{cols}] : (tensor<{rows + 3}x{cols}x{et}>) -> tensor<{rows}x{cols}x{et}>\n    %0 =").replace(
        "custom_call @rx.dropout(%arg0", "custom_call @rx.dropout(%w")
    assert steps(rx, cut) == ["dropout"]
    more = [key] + ([r] if residual else [])
    a, = run(rx, client, cut, [wide] + more)
    b, = run(rx, client, base, [np.ascontiguousarray(wide[3:])] + more)
    assert np.array_equal(f64(a), f64(b)) and f64(a).any()


@pytest.mark.gpu
@pytest.mark.parametrize("et", ["f32", "bf16"])
@pytest.mark.parametrize("nodes,node", [(2, 0), (2, 1), (4, 3), (8, 5)])
@pytest.mark.parametrize("rows,cols,residual", [(8, 5, False), (16, 8, True), (64, 257, True), (8, 3001, False)])
def test_dropout_of_a_share(rx, ref, rows, cols, residual, nodes, node, et):
    """A process that holds one share of an array split over a mesh drops what the whole array's mask says.  (Nothing is
    exchanged between the shares, so one device can be any of them.)"""
    rng = np.random.default_rng(34)
    client = rx.Client(node_id=node, num_nodes=nodes, allowed_devices=[0])
    try:
        x, r = values(rx, rng, (rows, cols), et), values(rx, rng, (rows, cols), et)
        key = rng.integers(-2 ** 31, 2 ** 31, 2).astype(np.int32)
        text = rx.programs.dropout((rows, cols), 0.3, et=et, site=9, residual=residual, num_partitions=nodes)
        mesh = rx.Mesh(client.devices)
        share = rows // nodes
        mine = slice(node * share, (node + 1) * share)
        split = rx.NamedSharding(mesh, (None, "x"))  # Julia's order of dims
        arrays = [rx.from_local_shards([np.ascontiguousarray(v[mine].T)], (cols, rows), split, client) for v in ([x, r] if residual else [x])]
        arrays.insert(1, rx.to_rarray(key, client, sharding=rx.NamedSharding(mesh, (None,))))
        got = np.asarray(rx.compile(text, client)(*arrays).data[0].to_host()).reshape(share, cols)
        keep = ref.dropout_mask(share * cols, key, 0.3, 9, first=node * share * cols).reshape(share, cols)
        cut = math.floor(0.3 * 65536 + 0.5)
        want = np.where(keep, f64(x[mine]) * (65536 / (65536 - cut)), 0) + (f64(r[mine]) if residual else 0)
        close(f64(got), want, 2 * U * np.abs(f64(x[mine])) * 65536 / (65536 - cut) + 2 * HALF[et] * np.abs(want))
        assert residual or np.array_equal(f64(got) != 0, keep & (f64(x[mine]) != 0))
    finally:
        client.close()


def grad_on_the_device(rx, client, torch, ids, features, vocab, et="f32"):
    """The gradient of whole numbers, whose sums are exact in any order, and torch's."""
    n = ids.numel()
    dy = torch.randint(-8, 9, (n, features), device="cuda", dtype=torch.int8).to(torch.float32 if et == "f32" else torch.bfloat16)
    text = rx.programs.embedding_grad(vocab, features, n, et=et, ids_et="i32" if ids.dtype == torch.int32 else "i64")
    got = torch.from_dlpack(rx.compile(text, client)(rx.from_dlpack(dy.mT, client), rx.from_dlpack(ids, client))).mT
    want = torch.zeros(vocab, features, device="cuda")
    live = (ids >= 0) & (ids < vocab)
    want.index_add_(0, ids.clamp(0, vocab - 1).long(), dy.float() * live[:, None])
    return torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("features,et", [(2048, "bf16"), (2049, "f32"), (264, "f32"), (1500, "bf16")])
@pytest.mark.parametrize("tokens", [17000, 33000, 66000, 140000])
def test_embedding_grad_of_long_pieces(rx, client, tokens, features, et):
    """Many tokens, whose sorted places are cut into long pieces: runs about as long as a piece, and as several, that begin
    anywhere in one."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(35)
    for piece in (32, 64, 128):
        lengths = rng.choice([1, 2, piece - 1, piece, piece + 1, 2 * piece - 1, 2 * piece, 2 * piece + 1, 3 * piece + 5, 9 * piece], size=2 * tokens)
        ids = np.repeat(np.arange(len(lengths)), lengths)[:tokens]
        vocab = int(ids[-1]) + 3
        ids = np.where(rng.random(tokens) < 0.001, vocab, rng.permutation(ids)).astype(np.int32)
        assert grad_on_the_device(rx, client, torch, torch.from_numpy(ids).cuda(), features, vocab, et)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,features,ids_et", [(9000, 2 ** 18 - 1, 8, "i32"), (9000, 2 ** 18, 8, "i64"), (70000, 2 ** 18 + 1, 5, "i32"), (20000, 2 ** 27, 1, "i32"), (10000, 2 ** 27 + 7, 2, "i64"), (8193, 1, 3, "i32"),
                                                          (262144, 5000, 8, "i32"), (262177, 5000, 8, "i64"), (300000, 70000, 8, "i32"), (300000, 300000, 3, "i32"), (1000003, 9, 16, "i32")])
def test_embedding_grad_of_long_sorts(rx, client, tokens, vocab, features, ids_et):
    """Every number of passes of the sort, and more tokens than its warps hold in registers."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(36)
    for spread in (1, 3):
        ids = np.minimum((vocab * rng.random(tokens) ** spread).astype(np.int64), vocab - 1)
        ids[rng.integers(0, tokens, 20)] = -1
        ids[rng.integers(0, tokens, 20)] = vocab
        ids[[0, -1]] = 0, vocab - 1
        ids = torch.from_numpy(ids).cuda().to(torch.int32 if ids_et == "i32" else torch.int64)
        assert grad_on_the_device(rx, client, torch, ids, features, vocab)
