"""StableHLO module text for the benchmark configurations, in the form Reactant
hands to its runtime: `func.func @main` over reversed-dim tensors, printed by
MLIR's default printer.

Reactant's tracer and pass pipeline cannot run where this engine is built (no
Julia), so these are written out by hand from the op emitters:
  sum / maximum  -> stablehlo.reduce       src/TracedRArray.jl:187-230, src/Ops.jl:3491-3622
  broadcasting   -> elementwise ops        src/TracedUtils.jl:1202-1352
  A[r, c]        -> stablehlo.slice        src/Indexing.jl:552-627, src/Ops.jl:761-793
  B[r, c] = v    -> dynamic_update_slice   src/Indexing.jl:350-446, src/Ops.jl:3662-3678
  @trace for     -> stablehlo.while        src/Ops.jl:2349-2447
  W * X          -> stablehlo.dot_general  src/stdlibs/LinearAlgebra.jl:274-330
  sharding attrs -> sdy.mesh / sdy.sharding src/Sharding.jl:512-575
Each generator offers the optimised form (`raw=False`: layout transposes already
propagated away) and, where it differs, the raw trace form (`raw=True`: every
argument and result wrapped in the reversed-dims transposes of
src/TracedUtils.jl:608-626).
"""
from __future__ import annotations

import math


def _t(shape, et="f32"):
    return "tensor<" + "".join(f"{d}x" for d in shape) + et + ">"


def sinsum_add(n: int, raw: bool = False, num_partitions: int = 1) -> str:
    """f(x, y) = sum(sin.(x) .+ y) on Float32 vectors of length n.
    With num_partitions > 1 both vectors are sharded along a 1-D mesh "x"."""
    t = _t([n])
    shard = ' {sdy.sharding = #sdy.sharding<@mesh, [{"x"}]>}' if num_partitions > 1 else ""
    mesh = f'  sdy.mesh @mesh = <["x"={num_partitions}]>\n' if num_partitions > 1 else ""
    body = []
    x, y = "%arg0", "%arg1"
    if raw:
        body.append(f"    %t0 = stablehlo.transpose %arg0, dims = [0] : ({t}) -> {t}")
        body.append(f"    %t1 = stablehlo.transpose %arg1, dims = [0] : ({t}) -> {t}")
        x, y = "%t0", "%t1"
    body += [
        "    %cst = stablehlo.constant dense<0.000000e+00> : tensor<f32>",
        f"    %0 = stablehlo.sine {x} : {t}",
        f"    %1 = stablehlo.add %0, {y} : {t}",
        f"    %2 = stablehlo.reduce(%1 init: %cst) applies stablehlo.add across dimensions = [0] : ({t}, tensor<f32>) -> tensor<f32>",
        "    return %2 : tensor<f32>",
    ]
    return (f"module @reactant_sinsum_add attributes {{mhlo.num_partitions = {num_partitions} : i64, mhlo.num_replicas = 1 : i64}} {{\n"
            f"{mesh}  func.func @main(%arg0: {t}{shard}, %arg1: {t}{shard}) -> tensor<f32> {{\n" + "\n".join(body) + "\n  }\n}\n")


def logsumexp_dims1(rows: int, cols: int, raw: bool = False) -> str:
    """m = maximum(x; dims=1); m .+ log.(sum(exp.(x .- m); dims=1)) for a Julia
    rows x cols Float32 matrix (argument tensor is cols x rows)."""
    ta, tc, tr = _t([cols, rows]), _t([cols]), _t([cols, 1])
    if not raw:
        body = f"""    %cst = stablehlo.constant dense<0.000000e+00> : tensor<f32>
    %cst_0 = stablehlo.constant dense<0xFF800000> : tensor<f32>
    %0 = stablehlo.reduce(%arg0 init: %cst_0) applies stablehlo.maximum across dimensions = [1] : ({ta}, tensor<f32>) -> {tc}
    %1 = stablehlo.broadcast_in_dim %0, dims = [0] : ({tc}) -> {ta}
    %2 = stablehlo.subtract %arg0, %1 : {ta}
    %3 = stablehlo.exponential %2 : {ta}
    %4 = stablehlo.reduce(%3 init: %cst) applies stablehlo.add across dimensions = [1] : ({ta}, tensor<f32>) -> {tc}
    %5 = stablehlo.log %4 : {tc}
    %6 = stablehlo.add %0, %5 : {tc}
    %7 = stablehlo.reshape %6 : ({tc}) -> {tr}
    return %7 : {tr}"""
    else:
        tl, t1 = _t([rows, cols]), _t([1, cols])
        body = f"""    %cst = stablehlo.constant dense<0.000000e+00> : tensor<f32>
    %cst_0 = stablehlo.constant dense<0xFF800000> : tensor<f32>
    %0 = stablehlo.transpose %arg0, dims = [1, 0] : ({ta}) -> {tl}
    %1 = stablehlo.reduce(%0 init: %cst_0) applies stablehlo.maximum across dimensions = [0] : ({tl}, tensor<f32>) -> {tc}
    %2 = stablehlo.reshape %1 : ({tc}) -> {t1}
    %3 = stablehlo.broadcast_in_dim %2, dims = [0, 1] : ({t1}) -> {tl}
    %4 = stablehlo.subtract %0, %3 : {tl}
    %5 = stablehlo.exponential %4 : {tl}
    %6 = stablehlo.reduce(%5 init: %cst) applies stablehlo.add across dimensions = [0] : ({tl}, tensor<f32>) -> {tc}
    %7 = stablehlo.reshape %6 : ({tc}) -> {t1}
    %8 = stablehlo.log %7 : {t1}
    %9 = stablehlo.add %2, %8 : {t1}
    %10 = stablehlo.transpose %9, dims = [1, 0] : ({t1}) -> {tr}
    return %10 : {tr}"""
    return ("module @reactant_logsumexp attributes {mhlo.num_partitions = 1 : i64, mhlo.num_replicas = 1 : i64} {\n"
            f"  func.func @main(%arg0: {ta}) -> {tr} {{\n{body}\n  }}\n}}\n")


def jacobi2d(n: int, steps: int, form: str = "dus", num_partitions: int = 1) -> str:
    """Jacobi-2D on n x n Float32 arrays; both arrays are mutated, hence donated and aliased to the two results.

    form="dus" / "pad": `steps` sweeps of
        B[2:end-1,2:end-1] = 0.2f0 .* (A[c] .+ A[i-1] .+ A[i+1] .+ A[j-1] .+ A[j+1]); A, B = B, A
    with the interior written by dynamic_update_slice ("dus") or by the pad + select rewrite that Enzyme-JAX's
    communication patterns can produce ("pad", src/compiler/OptimizationPasses.jl:356-372).
    form="concat": the same update with the interior placed by two nested concatenates -- the borders of B's rows
    around the new interior, then B's first and last row around that -- which is what the rewrite of a
    dynamic_update_slice into concatenates leaves (src/CompileOptions.jl:22-41).
    form="halfsteps": the spelling of benchmark/polybench/stencil.jl:263-289 -- every one of the `steps`
    iterations updates B from A and then A from B (two sweeps, no swap), the five terms added in that file's
    order: centre, j-1, j+1, i+1, i-1.
    With num_partitions > 1 both arrays are split over a 1-D mesh along Julia's second dimension (the first, i.e.
    row, dimension of the tensors): NamedSharding(mesh, (nothing, :x))."""
    t, ti = _t([n, n]), _t([n - 2, n - 2])
    shard = ', sdy.sharding = #sdy.sharding<@mesh, [{"x"}, {}]>' if num_partitions > 1 else ""
    mesh = f'  sdy.mesh @mesh = <["x"={num_partitions}]>\n' if num_partitions > 1 else ""
    m = n - 1
    # physical dims are reversed Julia dims: Julia A[i-1, j] is the minor-dim neighbour
    centre, i_lo, i_hi, j_lo, j_hi = f"[1:{m}, 1:{m}]", f"[1:{m}, 0:{n - 2}]", f"[1:{m}, 2:{n}]", f"[0:{n - 2}, 1:{m}]", f"[2:{n}, 1:{m}]"

    def sweep(src, tag, order):
        out = [f"      %s{tag}{k} = stablehlo.slice {src} {sl} : ({t}) -> {ti}" for k, sl in enumerate(order)]
        out += [
            f"      %a{tag}0 = stablehlo.add %s{tag}0, %s{tag}1 : {ti}",
            f"      %a{tag}1 = stablehlo.add %a{tag}0, %s{tag}2 : {ti}",
            f"      %a{tag}2 = stablehlo.add %a{tag}1, %s{tag}3 : {ti}",
            f"      %a{tag}3 = stablehlo.add %a{tag}2, %s{tag}4 : {ti}",
            f"      %u{tag} = stablehlo.multiply %cst, %a{tag}3 : {ti}",
        ]
        return out

    dus = lambda dst, upd, res: f"      {res} = stablehlo.dynamic_update_slice {dst}, {upd}, %c_1, %c_1 : ({t}, {ti}, tensor<i32>, tensor<i32>) -> {t}"
    extra = ""
    if form == "halfsteps":
        order = [centre, j_lo, j_hi, i_hi, i_lo]
        lines = sweep("%iterArg_0", "p", order) + [dus("%iterArg_1", "%up", "%nb")] + sweep("%nb", "q", order) + [dus("%iterArg_0", "%uq", "%na")]
        yields = "%1, %na, %nb"
    else:
        lines = sweep("%iterArg_0", "", [centre, i_lo, i_hi, j_lo, j_hi])
        if form == "dus":
            lines.append(dus("%iterArg_1", "%u", "%nb"))
        elif form == "concat":
            tc, tr, tm = _t([n - 2, 1]), _t([1, n]), _t([n - 2, n])
            lines += [
                f"      %left = stablehlo.slice %iterArg_1 [1:{m}, 0:1] : ({t}) -> {tc}",
                f"      %right = stablehlo.slice %iterArg_1 [1:{m}, {m}:{n}] : ({t}) -> {tc}",
                f"      %mid = stablehlo.concatenate %left, %u, %right, dim = 1 : ({tc}, {ti}, {tc}) -> {tm}",
                f"      %top = stablehlo.slice %iterArg_1 [0:1, 0:{n}] : ({t}) -> {tr}",
                f"      %bot = stablehlo.slice %iterArg_1 [{m}:{n}, 0:{n}] : ({t}) -> {tr}",
                f"      %nb = stablehlo.concatenate %top, %mid, %bot, dim = 0 : ({tr}, {tm}, {tr}) -> {t}",
            ]
        else:
            lines += [
                f"      %pu = stablehlo.pad %u, %cst_z, low = [1, 1], high = [1, 1], interior = [0, 0] : ({ti}, tensor<f32>) -> {t}",
                f"      %nb = stablehlo.select %pm, %pu, %iterArg_1 : {_t([n, n], 'i1')}, {t}",
            ]
            extra = (f"    %cst_z = stablehlo.constant dense<0.000000e+00> : tensor<f32>\n"
                     f"    %false = stablehlo.constant dense<false> : tensor<i1>\n"
                     f"    %ones = stablehlo.constant dense<true> : {_t([n - 2, n - 2], 'i1')}\n"
                     f"    %pm = stablehlo.pad %ones, %false, low = [1, 1], high = [1, 1], interior = [0, 0] : ({_t([n - 2, n - 2], 'i1')}, tensor<i1>) -> {_t([n, n], 'i1')}\n")
        yields = "%1, %nb, %iterArg_0"
    body = "\n".join(lines)
    return f"""module @reactant_jacobi2d attributes {{mhlo.num_partitions = {num_partitions} : i64, mhlo.num_replicas = 1 : i64}} {{
{mesh}  func.func @main(%arg0: {t} {{tf.aliasing_output = 0 : i32{shard}}}, %arg1: {t} {{tf.aliasing_output = 1 : i32{shard}}}) -> ({t}, {t}) {{
    %c = stablehlo.constant dense<0> : tensor<i64>
    %c_0 = stablehlo.constant dense<{steps}> : tensor<i64>
    %c_2 = stablehlo.constant dense<1> : tensor<i64>
    %c_1 = stablehlo.constant dense<1> : tensor<i32>
    %cst = stablehlo.constant dense<2.000000e-01> : {ti}
{extra}    %0:3 = stablehlo.while(%iterArg = %c, %iterArg_0 = %arg0, %iterArg_1 = %arg1) : tensor<i64>, {t}, {t} attributes {{enzyme.disable_mincut}}
     cond {{
      %1 = stablehlo.compare  LT, %iterArg, %c_0 : (tensor<i64>, tensor<i64>) -> tensor<i1>
      stablehlo.return %1 : tensor<i1>
    }} do {{
      %1 = stablehlo.add %iterArg, %c_2 : tensor<i64>
{body}
      stablehlo.return {yields} : tensor<i64>, {t}, {t}
    }}
    return %0#1, %0#2 : {t}, {t}
  }}
}}
"""


def mlp_grad(features: int = 1024, hidden: int = 4096, out: int = 1024, batch: int = 4096, num_partitions: int = 1) -> str:
    """Two-layer MLP forward + reverse-mode gradient, as it reaches the runtime
    after Enzyme's pass has synthesised the reverse program: five dot_generals
    (two forward, three transposed-operand backward), gelu(tanh) and its
    derivative as elementwise chains, bias gradients as column reductions.

    Julia shapes: W1 hidden x features (bf16), b1 hidden (f32), W2 out x hidden
    (bf16), b2 out (f32), X features x batch (bf16), Y out x batch (f32).
    Results: dW1, db1, dW2, db2, loss.

    With num_partitions > 1 the batch is split over a 1-D mesh (data parallelism): X and Y carry
    `sdy.sharding` on their batch dimension, the weights are replicated, and every gradient is a
    sum over devices, so the runtime has to all-reduce them.
    """
    F, H, O, B = features, hidden, out, batch
    tW1, tW2, tX, tY = _t([F, H], "bf16"), _t([H, O], "bf16"), _t([B, F], "bf16"), _t([B, O])
    tb1, tb2 = _t([H]), _t([O])
    tZ1b, tZ1 = _t([B, H], "bf16"), _t([B, H])
    tZ2b, tZ2 = _t([B, O], "bf16"), _t([B, O])
    c = math.sqrt(2.0 / math.pi)
    inv = 1.0 / (B * O)

    def k(v, t):
        return f"stablehlo.constant dense<{v:.9e}> : {t}"

    sh = ' {sdy.sharding = #sdy.sharding<@mesh, [{"x"}, {}]>}' if num_partitions > 1 else ""
    mesh = f'  sdy.mesh @mesh = <["x"={num_partitions}]>\n' if num_partitions > 1 else ""
    return f"""module @reactant_mlp_grad attributes {{mhlo.num_partitions = {num_partitions} : i64, mhlo.num_replicas = 1 : i64}} {{
{mesh}  func.func @main(%arg0: {tW1}, %arg1: {tb1}, %arg2: {tW2}, %arg3: {tb2}, %arg4: {tX}{sh}, %arg5: {tY}{sh}) -> ({tW1}, {tb1}, {tW2}, {tb2}, tensor<f32>) {{
    %zero = stablehlo.constant dense<0.000000e+00> : tensor<f32>
    %half = {k(0.5, tZ1)}
    %one = {k(1.0, tZ1)}
    %ca = {k(0.044715, tZ1)}
    %c3a = {k(3 * 0.044715, tZ1)}
    %cc = {k(c, tZ1)}
    %cinv = {k(inv, "tensor<f32>")}
    %c2inv = {k(2 * inv, tZ2)}
    %0 = stablehlo.dot_general %arg4, %arg0, contracting_dims = [1] x [0], precision = [DEFAULT, DEFAULT] : ({tX}, {tW1}) -> {tZ1b}
    %1 = stablehlo.convert %0 : ({tZ1b}) -> {tZ1}
    %2 = stablehlo.broadcast_in_dim %arg1, dims = [1] : ({tb1}) -> {tZ1}
    %z1 = stablehlo.add %1, %2 : {tZ1}
    %z1sq = stablehlo.multiply %z1, %z1 : {tZ1}
    %z1cu = stablehlo.multiply %z1sq, %z1 : {tZ1}
    %3 = stablehlo.multiply %ca, %z1cu : {tZ1}
    %4 = stablehlo.add %z1, %3 : {tZ1}
    %5 = stablehlo.multiply %cc, %4 : {tZ1}
    %th = stablehlo.tanh %5 : {tZ1}
    %6 = stablehlo.add %one, %th : {tZ1}
    %7 = stablehlo.multiply %half, %z1 : {tZ1}
    %h = stablehlo.multiply %7, %6 : {tZ1}
    %hb = stablehlo.convert %h : ({tZ1}) -> {tZ1b}
    %8 = stablehlo.dot_general %hb, %arg2, contracting_dims = [1] x [0], precision = [DEFAULT, DEFAULT] : ({tZ1b}, {tW2}) -> {tZ2b}
    %9 = stablehlo.convert %8 : ({tZ2b}) -> {tZ2}
    %10 = stablehlo.broadcast_in_dim %arg3, dims = [1] : ({tb2}) -> {tZ2}
    %z2 = stablehlo.add %9, %10 : {tZ2}
    %d = stablehlo.subtract %z2, %arg5 : {tZ2}
    %dd = stablehlo.multiply %d, %d : {tZ2}
    %11 = stablehlo.reduce(%dd init: %zero) applies stablehlo.add across dimensions = [0, 1] : ({tZ2}, tensor<f32>) -> tensor<f32>
    %loss = stablehlo.multiply %11, %cinv : tensor<f32>
    %dz2 = stablehlo.multiply %c2inv, %d : {tZ2}
    %db2 = stablehlo.reduce(%dz2 init: %zero) applies stablehlo.add across dimensions = [0] : ({tZ2}, tensor<f32>) -> {tb2}
    %dz2b = stablehlo.convert %dz2 : ({tZ2}) -> {tZ2b}
    %dw2 = stablehlo.dot_general %hb, %dz2b, contracting_dims = [0] x [0], precision = [DEFAULT, DEFAULT] : ({tZ1b}, {tZ2b}) -> {tW2}
    %dhb = stablehlo.dot_general %dz2b, %arg2, contracting_dims = [1] x [1], precision = [DEFAULT, DEFAULT] : ({tZ2b}, {tW2}) -> {tZ1b}
    %dh = stablehlo.convert %dhb : ({tZ1b}) -> {tZ1}
    %12 = stablehlo.multiply %th, %th : {tZ1}
    %13 = stablehlo.subtract %one, %12 : {tZ1}
    %14 = stablehlo.multiply %c3a, %z1sq : {tZ1}
    %15 = stablehlo.add %one, %14 : {tZ1}
    %16 = stablehlo.multiply %cc, %15 : {tZ1}
    %17 = stablehlo.multiply %13, %16 : {tZ1}
    %18 = stablehlo.multiply %7, %17 : {tZ1}
    %19 = stablehlo.multiply %half, %6 : {tZ1}
    %gp = stablehlo.add %19, %18 : {tZ1}
    %dz1 = stablehlo.multiply %dh, %gp : {tZ1}
    %db1 = stablehlo.reduce(%dz1 init: %zero) applies stablehlo.add across dimensions = [0] : ({tZ1}, tensor<f32>) -> {tb1}
    %dz1b = stablehlo.convert %dz1 : ({tZ1}) -> {tZ1b}
    %dw1 = stablehlo.dot_general %arg4, %dz1b, contracting_dims = [0] x [0], precision = [DEFAULT, DEFAULT] : ({tX}, {tZ1b}) -> {tW1}
    return %dw1, %db1, %dw2, %db2, %loss : {tW1}, {tb1}, {tW2}, {tb2}, tensor<f32>
  }}
}}
"""


# ---- the operators at the two ends of a token model ------------------------------------------------------------------
# StableHLO has no op for these; they are custom_calls with a typed backend_config, which pass through Reactant's
# pipeline untouched.  Shapes below are the module's (row-major) ones; in Julia the dims come in reverse: a table is
# features x vocabulary, logits are vocabulary x tokens.  Token ids count from 0.
def _call(target: str, operands, results, **config) -> str:
    """One `stablehlo.custom_call`: operands are (name, type) pairs; settings are written as f64 or i64."""
    cfg = ", ".join(f"{k} = {v!r} : f64" if isinstance(v, float) else f"{k} = {int(v)} : i64" for k, v in config.items())
    res = results[0] if len(results) == 1 else "(" + ", ".join(results) + ")"
    return (f"stablehlo.custom_call @{target}({', '.join(n for n, _ in operands)}) {{api_version = 4 : i32, backend_config = {{{cfg}}}}} : "
            f"({', '.join(t for _, t in operands)}) -> {res}")


def _dims(tokens) -> list:
    return list(tokens) if isinstance(tokens, (tuple, list)) else [tokens]


def _one_call(name: str, target: str, types, results, num_partitions: int = 1, split=(), **config) -> str:
    """A module whose @main is one custom call; arguments whose index is in `split` are split along their first dim."""
    args = [(f"%arg{k}", t) for k, t in enumerate(types)]
    mesh = f'  sdy.mesh @mesh = <["x"={num_partitions}]>\n' if num_partitions > 1 else ""

    def attr(k, t):
        if num_partitions == 1 or k not in split:
            return ""
        rank = t.count("x")
        return " {sdy.sharding = #sdy.sharding<@mesh, [" + ", ".join(['{"x"}'] + ["{}"] * (rank - 1)) + "]>}"

    sig = ", ".join(f"{n}: {t}{attr(k, t)}" for k, (n, t) in enumerate(args))
    res = results[0] if len(results) == 1 else "(" + ", ".join(results) + ")"
    lhs = "%0" if len(results) == 1 else f"%0:{len(results)}"
    outs = "%0" if len(results) == 1 else ", ".join(f"%0#{k}" for k in range(len(results)))
    return (f"module @reactant_{name} attributes {{mhlo.num_partitions = {num_partitions} : i64, mhlo.num_replicas = 1 : i64}} {{\n{mesh}"
            f"  func.func @main({sig}) -> {res} {{\n    {lhs} = {_call(target, args, results, **config)}\n    return {outs} : {', '.join(results)}\n  }}\n}}\n")


def embedding(vocab: int, features: int, tokens, et: str = "bf16", out_et: str | None = None, ids_et: str = "i32", scale: float = 1.0, num_partitions: int = 1) -> str:
    """out[t, :] = scale * table[ids[t], :] for a table of `vocab` rows; `tokens` is a count or a tuple of dims.
    A token outside the table (padding) is a row of zeros.  Products are formed in 32 bits and rounded once.
    Arguments: table, ids.  With num_partitions > 1 the tokens are split along their first dim."""
    n = _dims(tokens)
    return _one_call("embedding", "rx.embedding", [_t([vocab, features], et), _t(n, ids_et)], [_t(n + [features], out_et or et)], num_partitions, (1,), scale=float(scale))


def embedding_grad(vocab: int, features: int, tokens, et: str = "bf16", out_et: str = "f32", ids_et: str = "i32", scale: float = 1.0, num_partitions: int = 1) -> str:
    """The gradient of `embedding` with respect to the table: row v is scale times the sum, in 32 bits and in a fixed
    order, of the gradients of the tokens with id v; zeros where there are none.  Arguments: dy, ids."""
    n = _dims(tokens)
    return _one_call("embedding_grad", "rx.embedding_grad", [_t(n + [features], et), _t(n, ids_et)], [_t([vocab, features], out_et)], num_partitions, (0, 1), scale=float(scale))


def dropout(shape, rate: float, et: str = "bf16", site: int = 0, residual: bool = False, num_partitions: int = 1) -> str:
    """x with a share `rate` of its elements set to zero and the others scaled to keep the mean, plus a residual if
    there is one.  Arguments: x, key (two 32-bit words), [residual].  The mask is a function of the key, the number
    `site` (one for each place in a model) and the element's index only -- the same call on a gradient is the gradient:
    element i has 16 of the 128 bits Philox4x32-10 gives at the counter (i // 8, site), and stays if they reach
    round(65536 * rate), so rates are kept in steps of 1 / 65536."""
    t = _t(_dims(shape), et)
    return _one_call("dropout", "rx.dropout", [t, _t([2], "i32")] + ([t] if residual else []), [t], num_partitions, (0, 2), rate=float(rate), site=site)


def token_logprobs(tokens, vocab: int, et: str = "bf16", ids_et: str = "i32", top_k: int = 0, temperature: float = 1.0, num_partitions: int = 1) -> str:
    """Of every row of logits / temperature: the log probability of its token, the entropy, and the log-sum-exp; with
    top_k the largest log probabilities and their tokens too (equal ones by the lower token).  Arguments: logits, ids.
    All results are f32 (tokens i32).  A token outside the vocabulary (padding) has log probability 0.  A row of
    nothing but -inf has the entropy 0, and -inf for everything else."""
    n = _dims(tokens)
    f = _t(n)
    return _one_call("token_logprobs", "rx.token_logprobs", [_t(n + [vocab], et), _t(n, ids_et)], [f, f, f] + ([_t(n + [top_k]), _t(n + [top_k], "i32")] if top_k else []),
                     num_partitions, (0, 1), temperature=float(temperature), top_k=top_k)


def token_logprobs_grad(tokens, vocab: int, et: str = "bf16", ids_et: str = "i32", temperature: float = 1.0, num_partitions: int = 1) -> str:
    """The gradient of the first three results of `token_logprobs` with respect to the logits.  Arguments: logits, ids,
    the entropy's and the log-sum-exp's values in the order (lse, entropy), then the gradients that arrive at the log
    probability, the entropy and the log-sum-exp.  Padding rows take no gradient through their log probability."""
    n = _dims(tokens)
    return _one_call("token_logprobs_grad", "rx.token_logprobs_grad", [_t(n + [vocab], et), _t(n, ids_et)] + [_t(n)] * 5, [_t(n + [vocab], et)], num_partitions, tuple(range(7)),
                     temperature=float(temperature))


def token_model_grad(vocab: int = 32768, features: int = 1024, hidden: int = 4096, tokens: int = 4096, rate: float = 0.1, num_partitions: int = 1) -> str:
    """One training step of a small token model, as it reaches the runtime with its reverse program: embedding lookup,
    a tanh layer with dropout on the residual stream, a vocabulary projection, and the mean negative log probability
    of the next tokens.

    Arguments: E vocab x features, W1 features x hidden, W2 hidden x features, U features x vocab (all bf16, module
    dims), ids and targets (i32, `tokens` of each; a target of -1 is padding), key (two i32).
    Results: dE (f32), dW1, dW2, dU (bf16), loss, mean entropy (f32).

        x = sqrt(features) E[ids];  h = tanh(x W1);  y = x + dropout(h W2);  loss = -sum(log softmax(y U)[targets]) / tokens
    """
    V, F, H, T = vocab, features, hidden, tokens
    b = lambda *d: _t(d, "bf16")  # noqa: E731
    tE, tW1, tW2, tU, tI, tK = b(V, F), b(F, H), b(H, F), b(F, V), _t([T], "i32"), _t([2], "i32")
    tX, tH, tL, tR, tS = b(T, F), b(T, H), b(T, V), _t([T]), "tensor<f32>"
    scale = math.sqrt(F)
    sh = ' {sdy.sharding = #sdy.sharding<@mesh, [{"x"}]>}' if num_partitions > 1 else ""
    mesh = f'  sdy.mesh @mesh = <["x"={num_partitions}]>\n' if num_partitions > 1 else ""

    def dot(a, ta, c, tc, ac, cc, out):
        return f"stablehlo.dot_general {a}, {c}, contracting_dims = [{ac}] x [{cc}], precision = [DEFAULT, DEFAULT] : ({ta}, {tc}) -> {out}"

    tHf, tLp = _t([T, H]), [tR, tR, tR]
    return f"""module @reactant_token_model_grad attributes {{mhlo.num_partitions = {num_partitions} : i64, mhlo.num_replicas = 1 : i64}} {{
{mesh}  func.func @main(%E: {tE}, %W1: {tW1}, %W2: {tW2}, %U: {tU}, %ids: {tI}{sh}, %targets: {tI}{sh}, %key: {tK}) -> ({_t([V, F])}, {tW1}, {tW2}, {tU}, {tS}, {tS}) {{
    %zero = stablehlo.constant dense<0.000000e+00> : {tS}
    %none = stablehlo.constant dense<0.000000e+00> : {tR}
    %one = stablehlo.constant dense<1.000000e+00> : {tHf}
    %inv = stablehlo.constant dense<{1.0 / T:.9e}> : {tS}
    %minus = stablehlo.constant dense<{-1.0 / T:.9e}> : {tS}
    %g = stablehlo.constant dense<{-1.0 / T:.9e}> : {tR}
    %x = {_call("rx.embedding", [("%E", tE), ("%ids", tI)], [tX], scale=scale)}
    %0 = {dot("%x", tX, "%W1", tW1, 1, 0, tH)}
    %1 = stablehlo.convert %0 : ({tH}) -> {tHf}
    %2 = stablehlo.tanh %1 : {tHf}
    %h = stablehlo.convert %2 : ({tHf}) -> {tH}
    %3 = {dot("%h", tH, "%W2", tW2, 1, 0, tX)}
    %y = {_call("rx.dropout", [("%3", tX), ("%key", tK), ("%x", tX)], [tX], rate=rate, site=1)}
    %logits = {dot("%y", tX, "%U", tU, 1, 0, tL)}
    %lp:3 = {_call("rx.token_logprobs", [("%logits", tL), ("%targets", tI)], tLp)}
    %4 = stablehlo.reduce(%lp#0 init: %zero) applies stablehlo.add across dimensions = [0] : ({tR}, {tS}) -> {tS}
    %loss = stablehlo.multiply %4, %minus : {tS}
    %5 = stablehlo.reduce(%lp#1 init: %zero) applies stablehlo.add across dimensions = [0] : ({tR}, {tS}) -> {tS}
    %entropy = stablehlo.multiply %5, %inv : {tS}
    %dl = {_call("rx.token_logprobs_grad", [("%logits", tL), ("%targets", tI), ("%lp#2", tR), ("%lp#1", tR), ("%g", tR), ("%none", tR), ("%none", tR)], [tL])}
    %dU = {dot("%y", tX, "%dl", tL, 0, 0, tU)}
    %dy = {dot("%dl", tL, "%U", tU, 1, 1, tX)}
    %d3 = {_call("rx.dropout", [("%dy", tX), ("%key", tK)], [tX], rate=rate, site=1)}
    %dW2 = {dot("%h", tH, "%d3", tX, 0, 0, tW2)}
    %6 = {dot("%d3", tX, "%W2", tW2, 1, 1, tH)}
    %7 = stablehlo.convert %6 : ({tH}) -> {tHf}
    %8 = stablehlo.multiply %2, %2 : {tHf}
    %9 = stablehlo.subtract %one, %8 : {tHf}
    %10 = stablehlo.multiply %7, %9 : {tHf}
    %dz = stablehlo.convert %10 : ({tHf}) -> {tH}
    %dW1 = {dot("%x", tX, "%dz", tH, 0, 0, tW1)}
    %11 = {dot("%dz", tH, "%W1", tW1, 1, 1, tX)}
    %dx = stablehlo.add %dy, %11 : {tX}
    %dE = {_call("rx.embedding_grad", [("%dx", tX), ("%ids", tI)], [_t([V, F])], scale=scale)}
    return %dE, %dW1, %dW2, %dU, %loss, %entropy : {_t([V, F])}, {tW1}, {tW2}, {tU}, {tS}, {tS}
  }}
}}
"""


def matmul(m: int, k: int, n: int, et: str = "f32") -> str:
    """C = A * B for Julia A (m x k), B (k x n): the arguments arrive as k x m and
    n x k tensors and the product as n x m (test/core/compile.jl:350-355)."""
    ta, tb, tc = _t([k, m], et), _t([n, k], et), _t([n, m], et)
    return f"""module @reactant_matmul attributes {{mhlo.num_partitions = 1 : i64, mhlo.num_replicas = 1 : i64}} {{
  func.func @main(%arg0: {ta}, %arg1: {tb}) -> {tc} {{
    %0 = stablehlo.dot_general %arg1, %arg0, contracting_dims = [1] x [0], precision = [DEFAULT, DEFAULT] : ({tb}, {ta}) -> {tc}
    return %0 : {tc}
  }}
}}
"""


def scan(xla_dims, xla_axis: int, kind: str = "add", et: str = "f32") -> str:
    """cumsum / cumprod / accumulate(max|min) along one dimension, as Reactant's scan_impl! lowers it
    (src/TracedRArray.jl:1049-1107): stablehlo.reduce_window whose window is the whole dimension, padded low by
    its extent minus one, with the combiner's identity as init value.  `xla_dims` are the boundary (reversed)
    dims; Julia `dims = d` of an N-d array is boundary dim N - d."""
    rank = len(xla_dims)
    win = [1] * rank
    win[xla_axis] = xla_dims[xla_axis]
    pads = "[" + ", ".join(f"[{xla_dims[d] - 1 if d == xla_axis else 0}, 0]" for d in range(rank)) + "]"
    ones = ", ".join(["1"] * rank)
    flt = et in ("f32", "bf16")
    init = {"add": "0.000000e+00" if flt else "0", "multiply": "1.000000e+00" if flt else "1",
            "maximum": "0xFF800000" if flt else "-2147483648", "minimum": "0x7F800000" if flt else "2147483647"}[kind]
    ty, sc = _t(list(xla_dims), et), _t([], et)
    return f"""module @reactant_scan attributes {{mhlo.num_partitions = 1 : i64, mhlo.num_replicas = 1 : i64}} {{
  func.func @main(%arg0: {ty}) -> {ty} {{
    %cst = stablehlo.constant dense<{init}> : {sc}
    %0 = "stablehlo.reduce_window"(%arg0, %cst) <{{base_dilations = array<i64: {ones}>, padding = dense<{pads}> : tensor<{rank}x2xi64>, window_dilations = array<i64: {ones}>, window_dimensions = array<i64: {', '.join(map(str, win))}>, window_strides = array<i64: {ones}>}}> ({{
    ^bb0(%arg1: {sc}, %arg2: {sc}):
      %1 = stablehlo.{kind} %arg1, %arg2 : {sc}
      stablehlo.return %1 : {sc}
    }}) : ({ty}, {sc}) -> {ty}
    return %0 : {ty}
  }}
}}
"""


class _Body:
    """Emits the ops of a loop body line by line, naming results %v0, %v1, ..."""

    def __init__(self):
        self.lines, self.n = [], 0

    def op(self, text, ty):
        name = f"%v{self.n}"
        self.n += 1
        self.lines.append(f"      {name} = {text} : {ty}")
        return name

    def slice(self, src, ranges, t_in, t_out):
        name = f"%v{self.n}"
        self.n += 1
        spec = ", ".join(f"{a}:{b}" for a, b in ranges)
        self.lines.append(f"      {name} = stablehlo.slice {src} [{spec}] : ({t_in}) -> {t_out}")
        return name

    def dus(self, dst, upd, starts, t, tu):
        name = f"%v{self.n}"
        self.n += 1
        idx = ", ".join(starts)
        types = ", ".join([t, tu] + ["tensor<i32>"] * len(starts))
        self.lines.append(f"      {name} = stablehlo.dynamic_update_slice {dst}, {upd}, {idx} : ({types}) -> {t}")
        return name


def _two_array_loop(name, shape, steps, consts, body_lines, yield_a, yield_b):
    t = _t(shape)
    cs = "\n".join(f"    {n} = stablehlo.constant dense<{v}> : {ty}" for n, v, ty in consts)
    body = "\n".join(body_lines)
    return f"""module @reactant_{name} attributes {{mhlo.num_partitions = 1 : i64, mhlo.num_replicas = 1 : i64}} {{
  func.func @main(%arg0: {t} {{tf.aliasing_output = 0 : i32}}, %arg1: {t} {{tf.aliasing_output = 1 : i32}}) -> ({t}, {t}) {{
    %c = stablehlo.constant dense<0> : tensor<i64>
    %c_0 = stablehlo.constant dense<{steps}> : tensor<i64>
    %c_2 = stablehlo.constant dense<1> : tensor<i64>
    %c_1 = stablehlo.constant dense<1> : tensor<i32>
{cs}
    %0:3 = stablehlo.while(%iterArg = %c, %iterArg_0 = %arg0, %iterArg_1 = %arg1) : tensor<i64>, {t}, {t} attributes {{enzyme.disable_mincut}}
     cond {{
      %1 = stablehlo.compare  LT, %iterArg, %c_0 : (tensor<i64>, tensor<i64>) -> tensor<i1>
      stablehlo.return %1 : tensor<i1>
    }} do {{
      %1 = stablehlo.add %iterArg, %c_2 : tensor<i64>
{body}
      stablehlo.return %1, {yield_a}, {yield_b} : tensor<i64>, {t}, {t}
    }}
    return %0#1, %0#2 : {t}, {t}
  }}
}}
"""


def fdtd2d(nx: int, ny: int, tmax: int) -> str:
    """benchmark/polybench/stencil.jl:42-72 (fdtd_2d_vectorized): per time step t
        EY[1, :] .= fict[t]
        EY[2:NX, :]       .-= 0.5 .* (HZ[2:NX, :] .- HZ[1:NX-1, :])
        EX[:, 2:NY]       .-= 0.5 .* (HZ[:, 2:NY] .- HZ[:, 1:NY-1])
        HZ[1:NX-1,1:NY-1] .-= 0.7 .* (EX[1:NX-1,2:NY] .- EX[1:NX-1,1:NY-1] .+ EY[2:NX,1:NY-1] .- EY[1:NX-1,1:NY-1])
    on NX x NY Float32 arrays (tensors [NY][NX]).  `fict[t]` is a scalar read at the traced loop variable: the
    induction value start + i * step of the counter (src/ControlFlow / ReactantCore `@trace for`), converted to Int32 and
    made 0-based (src/Ops.jl:3624-3646), a dynamic_slice of one element (src/Indexing.jl:25-31) reshaped to a scalar and
    broadcast into the first row.  All three arrays are mutated, hence donated and returned."""
    t, tf = _t([ny, nx]), _t([tmax])
    b = _Body()
    ti = b.op("stablehlo.multiply %iterArg, %c_2", "tensor<i64>")
    ti = b.op(f"stablehlo.add {ti}, %c_2", "tensor<i64>")
    t32 = f"%v{b.n}"
    b.n += 1
    b.lines.append(f"      {t32} = stablehlo.convert {ti} : (tensor<i64>) -> tensor<i32>")
    idx = b.op(f"stablehlo.subtract {t32}, %c_1", "tensor<i32>")
    fs = f"%v{b.n}"
    b.n += 1
    b.lines.append(f"      {fs} = stablehlo.dynamic_slice %arg3, {idx}, sizes = [1] : ({tf}, tensor<i32>) -> tensor<1xf32>")
    f0 = f"%v{b.n}"
    b.n += 1
    b.lines.append(f"      {f0} = stablehlo.reshape {fs} : (tensor<1xf32>) -> tensor<f32>")
    tcol = _t([ny, 1])
    row = f"%v{b.n}"
    b.n += 1
    b.lines.append(f"      {row} = stablehlo.broadcast_in_dim {f0}, dims = [] : (tensor<f32>) -> {tcol}")
    ey1 = b.dus("%iterArg_1", row, ["%c_z", "%c_z"], t, tcol)
    # EY[2:NX, :]: tensor columns 1..NX-1
    te = _t([ny, nx - 1])
    a = b.slice(ey1, [(0, ny), (1, nx)], t, te)
    h1 = b.slice("%iterArg_2", [(0, ny), (1, nx)], t, te)
    h0 = b.slice("%iterArg_2", [(0, ny), (0, nx - 1)], t, te)
    d = b.op(f"stablehlo.subtract {h1}, {h0}", te)
    mm = b.op(f"stablehlo.multiply %half_e, {d}", te)
    u = b.op(f"stablehlo.subtract {a}, {mm}", te)
    ey2 = b.dus(ey1, u, ["%c_z", "%c_1"], t, te)
    # EX[:, 2:NY]: tensor rows 1..NY-1
    tx = _t([ny - 1, nx])
    a = b.slice("%iterArg_0", [(1, ny), (0, nx)], t, tx)
    h1 = b.slice("%iterArg_2", [(1, ny), (0, nx)], t, tx)
    h0 = b.slice("%iterArg_2", [(0, ny - 1), (0, nx)], t, tx)
    d = b.op(f"stablehlo.subtract {h1}, {h0}", tx)
    mm = b.op(f"stablehlo.multiply %half_x, {d}", tx)
    u = b.op(f"stablehlo.subtract {a}, {mm}", tx)
    ex2 = b.dus("%iterArg_0", u, ["%c_1", "%c_z"], t, tx)
    # HZ[1:NX-1, 1:NY-1]
    th = _t([ny - 1, nx - 1])
    hz = b.slice("%iterArg_2", [(0, ny - 1), (0, nx - 1)], t, th)
    x1 = b.slice(ex2, [(1, ny), (0, nx - 1)], t, th)
    x0 = b.slice(ex2, [(0, ny - 1), (0, nx - 1)], t, th)
    y1 = b.slice(ey2, [(0, ny - 1), (1, nx)], t, th)
    y0 = b.slice(ey2, [(0, ny - 1), (0, nx - 1)], t, th)
    s1 = b.op(f"stablehlo.subtract {x1}, {x0}", th)
    s2 = b.op(f"stablehlo.add {s1}, {y1}", th)
    s3 = b.op(f"stablehlo.subtract {s2}, {y0}", th)
    mm = b.op(f"stablehlo.multiply %seven, {s3}", th)
    u = b.op(f"stablehlo.subtract {hz}, {mm}", th)
    hz2 = b.dus("%iterArg_2", u, ["%c_z", "%c_z"], t, th)
    body = "\n".join(b.lines)
    return f"""module @reactant_fdtd2d attributes {{mhlo.num_partitions = 1 : i64, mhlo.num_replicas = 1 : i64}} {{
  func.func @main(%arg0: {t} {{tf.aliasing_output = 0 : i32}}, %arg1: {t} {{tf.aliasing_output = 1 : i32}}, %arg2: {t} {{tf.aliasing_output = 2 : i32}}, %arg3: {tf}) -> ({t}, {t}, {t}) {{
    %c = stablehlo.constant dense<0> : tensor<i64>
    %c_0 = stablehlo.constant dense<{tmax}> : tensor<i64>
    %c_2 = stablehlo.constant dense<1> : tensor<i64>
    %c_1 = stablehlo.constant dense<1> : tensor<i32>
    %c_z = stablehlo.constant dense<0> : tensor<i32>
    %half_e = stablehlo.constant dense<5.000000e-01> : {te}
    %half_x = stablehlo.constant dense<5.000000e-01> : {tx}
    %seven = stablehlo.constant dense<0.699999988> : {th}
    %0:4 = stablehlo.while(%iterArg = %c, %iterArg_0 = %arg0, %iterArg_1 = %arg1, %iterArg_2 = %arg2) : tensor<i64>, {t}, {t}, {t} attributes {{enzyme.disable_mincut}}
     cond {{
      %1 = stablehlo.compare  LT, %iterArg, %c_0 : (tensor<i64>, tensor<i64>) -> tensor<i1>
      stablehlo.return %1 : tensor<i1>
    }} do {{
      %1 = stablehlo.add %iterArg, %c_2 : tensor<i64>
{body}
      stablehlo.return %1, {ex2}, {ey2}, {hz2} : tensor<i64>, {t}, {t}, {t}
    }}
    return %0#1, %0#2, %0#3 : {t}, {t}, {t}
  }}
}}
"""


def jacobi1d(n: int, steps: int) -> str:
    """benchmark/polybench/stencil.jl:201-221 (jacobi_1d_vectorized): per iteration
    B[2:N-1] = (1/3) .* (A[1:N-2] .+ A[2:N-1] .+ A[3:N]), then the same from B into A."""
    t, ti = _t([n]), _t([n - 2])
    b = _Body()

    def half(src, dst):
        l, c, r = (b.slice(src, [(k, n - 2 + k)], t, ti) for k in range(3))
        s = b.op(f"stablehlo.add {l}, {c}", ti)
        s = b.op(f"stablehlo.add {s}, {r}", ti)
        u = b.op(f"stablehlo.multiply %third, {s}", ti)
        return b.dus(dst, u, ["%c_1"], t, ti)

    nb = half("%iterArg_0", "%iterArg_1")
    na = half(nb, "%iterArg_0")
    third = repr(float(__import__("numpy").float32(1.0 / 3.0)))
    return _two_array_loop("jacobi1d", [n], steps, [("%third", f"{float(third):.9e}", ti)], b.lines, na, nb)


def heat3d(n: int, steps: int) -> str:
    """benchmark/polybench/stencil.jl:125-169 (heat_3d_vectorized): per iteration the 7-point update
    0.125*(x[i+1] - 2x + x[i-1]) + 0.125*(x[j+1] - 2x + x[j-1]) + 0.125*(x[k+1] - 2x + x[k-1]) + x of the interior,
    from A into B and then from B into A.  Julia dim 1 (i) is the contiguous, i.e. last, tensor dim."""
    t, ti = _t([n, n, n]), _t([n - 2, n - 2, n - 2])
    b = _Body()
    m = n - 1

    def sl(src, dk, dj, di):  # offsets along Julia k, j, i = tensor dims 0, 1, 2
        return b.slice(src, [(1 + dk, m + dk), (1 + dj, m + dj), (1 + di, m + di)], t, ti)

    def half(src, dst):
        c = sl(src, 0, 0, 0)
        terms = []
        for axis in ("i", "j", "k"):
            d = {"i": (0, 0, 1), "j": (0, 1, 0), "k": (1, 0, 0)}[axis]
            hi = sl(src, *d)
            lo = sl(src, *(-x for x in d))
            two_c = b.op(f"stablehlo.multiply %two, {c}", ti)
            s = b.op(f"stablehlo.subtract {hi}, {two_c}", ti)
            s = b.op(f"stablehlo.add {s}, {lo}", ti)
            terms.append(b.op(f"stablehlo.multiply %eighth, {s}", ti))
        s = b.op(f"stablehlo.add {terms[0]}, {terms[1]}", ti)
        s = b.op(f"stablehlo.add {s}, {terms[2]}", ti)
        s = b.op(f"stablehlo.add {s}, {c}", ti)
        return b.dus(dst, s, ["%c_1", "%c_1", "%c_1"], t, ti)

    nb = half("%iterArg_0", "%iterArg_1")
    na = half(nb, "%iterArg_0")
    return _two_array_loop("heat3d", [n, n, n], steps, [("%two", "2.000000e+00", ti), ("%eighth", "1.250000e-01", ti)], b.lines, na, nb)
