"""The operators at the two ends of a token model, as cases that can be timed and compared.

A token model starts with a row of the embedding table for each token, drops activations while it trains, and
ends with the log probability of the token that really came next.  The four operators here are those ends and
their gradients:

  embedding            out[t] = scale * table[id_t]; a token outside the table (padding) gives a row of zeros
  embedding_grad       dtable[v] = scale * sum of dy[t] over the tokens t with id_t = v
  dropout              keeps an element where 16 bits of a counter-based generator reach a threshold, and scales it;
                       optionally added to a residual stream; its gradient is the same call on the gradient
  token_logprobs       log softmax of each row at its token, the row's entropy and log-sum-exp, its top k tokens
  token_logprobs_grad  the gradient of the first three with respect to the logits

`own` false: plain torch operations in 32 bits.  `own` true: the framework's calls on its own arrays.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
BYTES = {"f32": 4, "bf16": 2, "i32": 4, "i64": 8}

# the most elements of logits (or of a table, or of activations) that a drawn case may have
MOST_LOGITS = 4096 * 131072
MOST_TABLE = 131072 * 2048
MOST_LOOKED_UP = 65536 * 2048


def listed():
    return [
        # one decoding step of a small batch: eight tokens looked up, bf16 table and activations
        {"name": "lookup_decode", "op": "embedding", "tokens": 8, "vocab": 32768, "features": 4096, "et": "bf16", "out_et": "bf16", "ids": "i32", "scale": 1.0, "pad": False},
        # the tokens of a whole training batch, rows scaled by the root of their length
        {"name": "lookup_batch", "op": "embedding", "tokens": 65536, "vocab": 131072, "features": 2048, "et": "bf16", "out_et": "bf16", "ids": "i32", "scale": math.sqrt(2048.0), "pad": False},
        # a short fine-tuning batch with padding, 32-bit table of odd width, 64-bit ids (the host language's integers)
        {"name": "lookup_grad_short", "op": "embedding_grad", "tokens": 700, "vocab": 10007, "features": 1001, "et": "f32", "out_et": "f32", "ids": "i64", "scale": 1.0, "pad": True},
        # the gradient of the training batch's lookup: few distinct tokens take most of the places
        {"name": "lookup_grad_batch", "op": "embedding_grad", "tokens": 65536, "vocab": 131072, "features": 2048, "et": "bf16", "out_et": "f32", "ids": "i32", "scale": math.sqrt(2048.0), "pad": False},
        # activations of a handful of tokens
        {"name": "dropout_few", "op": "dropout", "rows": 16, "cols": 1024, "et": "bf16", "rate": 0.1, "residual": False},
        # activations of a training batch dropped and added to the residual stream in one pass
        {"name": "dropout_residual", "op": "dropout", "rows": 16384, "cols": 4096, "et": "bf16", "rate": 0.1, "residual": True},
        # the last token of a few requests being served: log probabilities with twenty alternatives
        {"name": "logprobs_decode", "op": "token_logprobs", "tokens": 4, "vocab": 131072, "et": "bf16", "ids": "i32", "top_k": 20, "temperature": 1.0, "masked": False, "pad": False},
        # scoring a training batch: half a billion logits, no alternatives
        {"name": "logprobs_batch", "op": "token_logprobs", "tokens": 4096, "vocab": 131072, "et": "bf16", "ids": "i32", "top_k": 0, "temperature": 1.0, "masked": False, "pad": False},
        # scoring sampled answers: 32-bit logits of an odd vocabulary, forbidden tokens at minus infinity, padding, five alternatives
        {"name": "logprobs_sampled", "op": "token_logprobs", "tokens": 2049, "vocab": 50021, "et": "f32", "ids": "i64", "top_k": 5, "temperature": 0.7, "masked": True, "pad": True},
        # the gradient of the training batch's scores
        {"name": "logprobs_grad_batch", "op": "token_logprobs_grad", "tokens": 4096, "vocab": 131072, "et": "bf16", "ids": "i32", "temperature": 1.0, "masked": False, "pad": False},
        # the gradient of the sampled answers' scores, with the entropy's share
        {"name": "logprobs_grad_sampled", "op": "token_logprobs_grad", "tokens": 513, "vocab": 32003, "et": "f32", "ids": "i64", "temperature": 0.7, "masked": True, "pad": True},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "dropout", "token_logprobs", "token_logprobs_grad"])
    et, ids = rng.choice(["bf16", "f32"]), rng.choice(["i32", "i64"])
    wide = 2 if et == "f32" else 1  # 32-bit cases get half the elements
    if op in ("embedding", "embedding_grad"):
        features = _spread(rng, 16, 8192)
        vocab = _spread(rng, 64, min(262144, MOST_TABLE // (features * wide)))
        tokens = _spread(rng, 1, min(65536, MOST_LOOKED_UP // (features * wide)))
        return {"op": op, "tokens": tokens, "vocab": vocab, "features": features, "et": et, "out_et": rng.choice(["bf16", "f32"]), "ids": ids, "scale": rng.choice([1.0, math.sqrt(features)]),
                "pad": rng.random() < 0.5}
    if op == "dropout":
        cols = _spread(rng, 1, 16384)
        return {"op": op, "rows": _spread(rng, 1, 16384 * 4096 // (cols * wide)), "cols": cols, "et": et, "rate": rng.choice([0.05, 0.1, 0.25, 0.5, rng.uniform(0.01, 0.9)]), "residual": rng.random() < 0.5}
    vocab = _spread(rng, 64, 262144)
    case = {"op": op, "tokens": _spread(rng, 1, MOST_LOGITS // (vocab * wide)), "vocab": vocab, "et": et, "ids": ids, "temperature": rng.choice([1.0, 0.7, rng.uniform(0.3, 2.0)]),
            "masked": rng.random() < 0.5, "pad": rng.random() < 0.5}
    if op == "token_logprobs":
        case["top_k"] = rng.choice([0, 1, 5, 20, rng.randint(2, 32)])
    return case


def _padding(case):
    return case["tokens"] // 16 if case["pad"] else 0


def _frequency(vocab):
    """How often each token comes, most frequent first: one over its place, as in running text."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return p / p.sum()


def _ids(case, gen, dev):
    """Token ids with the frequencies of running text, frequent ones anywhere in the table; the end of the batch is padding (-1)."""
    order = torch.randperm(case["vocab"], generator=gen, device=dev)
    p = torch.from_numpy(_frequency(case["vocab"])).to(dev)
    reach = torch.cumsum(p, 0)
    place = torch.searchsorted(reach, torch.rand(case["tokens"], generator=gen, device=dev, dtype=torch.float64)).clamp(max=case["vocab"] - 1)
    ids = order[place]
    if _padding(case):
        ids[case["tokens"] - _padding(case):] = -1
    return ids.to(DTYPES[case["ids"]])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, dt = case["op"], DTYPES[case["et"]]
    state = {"case": case}
    if op == "embedding":
        table = torch.randn(case["vocab"], case["features"], generator=gen, device=dev, dtype=dt)
        state["in"] = [table, _ids(case, gen, dev)]
    elif op == "embedding_grad":
        dy = torch.randn(case["tokens"], case["features"], generator=gen, device=dev, dtype=dt)
        state["in"] = [dy, _ids(case, gen, dev)]
    elif op == "dropout":
        x = torch.randn(case["rows"], case["cols"], generator=gen, device=dev, dtype=dt)
        key = torch.randint(-2**31, 2**31, (2,), generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
        state["in"] = [x, key]
        if case["residual"]:
            state["in"].append(torch.randn(case["rows"], case["cols"], generator=gen, device=dev, dtype=dt))
    else:
        tokens, vocab = case["tokens"], case["vocab"]
        logits = torch.randn(tokens, vocab, generator=gen, device=dev, dtype=dt).mul_(2.5)
        ids = _ids(case, gen, dev)
        if case["masked"]:
            # the same tenth of the vocabulary is forbidden everywhere, though never the wanted token
            forbidden = torch.rand(vocab, generator=gen, device=dev) < 0.1
            wanted = logits.gather(1, ids.clamp(min=0).long()[:, None])
            logits[:, forbidden] = -math.inf
            logits.scatter_(1, ids.clamp(min=0).long()[:, None], wanted)
        # a model that has learnt something: the wanted token stands out
        logits.scatter_add_(1, ids.clamp(min=0).long()[:, None], torch.full((tokens, 1), 6.0, device=dev, dtype=dt))
        state["in"] = [logits, ids]
        if op == "token_logprobs_grad":
            # what the forward pass kept of each row, and the gradients that arrive
            parts = _row_sums(logits, case["temperature"])
            state["in"] += [parts["lse"], parts["entropy"]]
            state["in"].append(torch.randn(tokens, generator=gen, device=dev) / tokens)
            state["in"].append(torch.randn(tokens, generator=gen, device=dev) * (0.01 / tokens))
            state["in"].append(torch.rand(tokens, generator=gen, device=dev) * (1e-3 / tokens))
    if own:
        # a program's own handles: the compiled module, and its arrays over the same device memory
        import __graft_entry__ as entry
        rx = entry.load_package()
        state["thunk"] = rx.compile(_module(rx, case))
        state["arrays"] = [rx.from_dlpack(x.mT if x.dim() == 2 else x) for x in state["in"]]
    return state


def _module(rx, case):
    op, p = case["op"], rx.programs
    if op == "embedding":
        return p.embedding(case["vocab"], case["features"], case["tokens"], et=case["et"], out_et=case["out_et"], ids_et=case["ids"], scale=case["scale"])
    if op == "embedding_grad":
        return p.embedding_grad(case["vocab"], case["features"], case["tokens"], et=case["et"], out_et=case["out_et"], ids_et=case["ids"], scale=case["scale"])
    if op == "dropout":
        return p.dropout((case["rows"], case["cols"]), rate=case["rate"], et=case["et"], residual=case["residual"])
    if op == "token_logprobs":
        return p.token_logprobs(case["tokens"], case["vocab"], et=case["et"], ids_et=case["ids"], top_k=case["top_k"], temperature=case["temperature"])
    return p.token_logprobs_grad(case["tokens"], case["vocab"], et=case["et"], ids_et=case["ids"], temperature=case["temperature"])


def run(state):
    if own:
        got = state["thunk"](*state["arrays"])
        got = got if isinstance(got, tuple) else (got,)
        stream = torch.cuda.current_stream().cuda_stream or 1
        return tuple(t.mT if t.dim() == 2 else t for t in (torch.from_dlpack(x.__dlpack__(stream=stream)) for x in got))
    case = state["case"]
    return {"embedding": _embedding, "embedding_grad": _embedding_grad, "dropout": _dropout, "token_logprobs": _token_logprobs,
            "token_logprobs_grad": _token_logprobs_grad}[case["op"]](case, *state["in"])


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _embedding(case, table, ids):
    live = (ids >= 0) & (ids < case["vocab"])
    rows = table[ids.clamp(0, case["vocab"] - 1).long()].float() * case["scale"]
    return (torch.where(live[:, None], rows, 0.0).to(DTYPES[case["out_et"]]),)


def _embedding_grad(case, dy, ids):
    live = (ids >= 0) & (ids < case["vocab"])
    total = torch.zeros(case["vocab"], case["features"], device=dy.device)
    total.index_add_(0, ids.clamp(0, case["vocab"] - 1).long(), torch.where(live[:, None], dy.float(), 0.0))
    return ((total * case["scale"]).to(DTYPES[case["out_et"]]),)


def _threshold(rate):
    return math.floor(rate * 65536.0 + 0.5)


def _generator(key, groups, dev):
    """Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011) at the counters (group, 0, 0, 0): four words of 32 bits each."""
    low = 0xFFFFFFFF
    k0, k1 = key[0].long() & low, key[1].long() & low
    c0 = torch.arange(groups, device=dev)
    c1, c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0), torch.zeros_like(c0)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


def _kept(case, key, n, dev):
    """Which of n elements stay: eight elements share a counter, 16 bits each, low halves first."""
    words = _generator(key, -(-n // 8), dev)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return bits >= _threshold(case["rate"])


def _dropout(case, x, key, residual=None):
    keep = _kept(case, key, x.numel(), x.device).reshape(x.shape)
    y = torch.where(keep, x.float() * (65536.0 / (65536.0 - _threshold(case["rate"]))), 0.0)
    if residual is not None:
        y = y + residual.float()
    return (y.to(x.dtype),)


def _row_sums(logits, temperature):
    z = logits.float() / temperature
    top = z.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(z - top)
    total = e.sum(1)
    lse = top[:, 0] + torch.log(total)
    weighted = torch.where(e > 0, e * (z - top), 0.0).sum(1)
    return {"z": z, "lse": lse, "entropy": torch.log(total) - weighted / total}


def _token_logprobs(case, logits, ids):
    parts = _row_sums(logits, case["temperature"])
    live = (ids >= 0) & (ids < case["vocab"])
    wanted = parts["z"].gather(1, ids.clamp(0, case["vocab"] - 1).long()[:, None])[:, 0]
    out = (torch.where(live, wanted - parts["lse"], 0.0), parts["entropy"], parts["lse"])
    if not case["top_k"]:
        return out
    # order by value, then by place: one whole number per logit, larger for larger values and for earlier places
    bits = (logits.float() + 0.0).view(torch.int32).long()
    value = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    keys = value * 2**32 + (2**32 - 1 - torch.arange(case["vocab"], device=logits.device))
    best = 2**32 - 1 - (torch.topk(keys, case["top_k"], dim=1).values & 0xFFFFFFFF)
    return out + (parts["z"].gather(1, best) - parts["lse"][:, None], best.to(torch.int32))


def _token_logprobs_grad(case, logits, ids, lse, entropy, dlogprob, dentropy, dlse):
    logp = logits.float() / case["temperature"] - lse[:, None]
    p = torch.exp(logp)
    live = (ids >= 0) & (ids < case["vocab"])
    arrived = torch.where(live, dlogprob, 0.0)
    dz = torch.where(p > 0, p * ((dlse - arrived)[:, None] - dentropy[:, None] * (logp + entropy[:, None])), 0.0)
    dz.scatter_add_(1, ids.clamp(0, case["vocab"] - 1).long()[:, None], arrived[:, None])
    return ((dz / case["temperature"]).to(logits.dtype),)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * BYTES[case["et"]] * (3 if case["residual"] else 2) + 8, "flops": n * 2}
    tokens, vocab = case["tokens"], case["vocab"]
    if op in ("embedding", "embedding_grad"):
        cells, out = tokens * case["features"], BYTES[case["out_et"]]
        if op == "embedding":  # each distinct row of the table once, as many as such a draw of tokens is expected to hold
            rows = float((1.0 - (1.0 - _frequency(vocab)) ** (tokens - _padding(case))).sum())
            return {"bytes": rows * case["features"] * BYTES[case["et"]] + cells * out + tokens * BYTES[case["ids"]], "flops": cells}
        live = cells - _padding(case) * case["features"]
        return {"bytes": live * BYTES[case["et"]] + vocab * case["features"] * out + tokens * BYTES[case["ids"]], "flops": 2 * live}
    n, ids = tokens * vocab, tokens * BYTES[case["ids"]]
    if op == "token_logprobs":
        return {"bytes": n * BYTES[case["et"]] + ids + tokens * (12 + 8 * case["top_k"]), "flops": 6 * n}
    return {"bytes": 2 * n * BYTES[case["et"]] + ids + 20 * tokens, "flops": 7 * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    inputs = prepare(case, seed)["in"]
    op = case["op"]
    if op == "embedding":
        table, ids = inputs
        known = torch.cat([table, torch.zeros_like(table[:1])])  # one more row, of zeros, for what is not in the table
        return (known[torch.where(ids < 0, case["vocab"], ids).long()].double() * case["scale"],)
    if op == "embedding_grad":
        dy, ids = inputs
        total = torch.zeros(case["vocab"], case["features"], device=dy.device, dtype=torch.float64)
        for at in range(0, case["tokens"], 8192):
            some = ids[at:at + 8192]
            total.index_add_(0, some[some >= 0].long(), dy[at:at + 8192][some >= 0].double())
        return (total.mul_(case["scale"]),)
    if op == "dropout":
        return _exact_dropout(case, *inputs)
    if op == "token_logprobs":
        parts = [_exact_logprobs(case, *(x[at:at + 512] for x in inputs)) for at in range(0, case["tokens"], 512)]
        columns = [torch.cat(column) for column in zip(*parts)]
        return tuple(columns) + (None,) if case["top_k"] else tuple(columns)
    return (torch.cat([_exact_logprobs_grad(case, *(x[at:at + 512] for x in inputs)) for at in range(0, case["tokens"], 512)]),)


def _exact_dropout(case, x, key, residual=None):
    # the generator again, in the host's unsigned integers
    n = x.numel()
    k = [np.uint64(int(v) & 0xFFFFFFFF) for v in key.tolist()]
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.arange(-(-n // 8), dtype=np.uint64)] + [np.zeros(-(-n // 8), np.uint64)] * 3
    for r in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> shift) ^ c[1] ^ k[0], b & low, (a >> shift) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    sixteen = np.ascontiguousarray(np.stack(c, 1).astype("<u4")).view("<u2").reshape(-1)[:n]
    cut = round(case["rate"] * 65536)
    kept = torch.from_numpy(sixteen >= cut).to(x.device).reshape(x.shape)
    y = x.double() * (65536 / (65536 - cut)) * kept
    return (y if residual is None else y + residual.double(),)


def _exact_logprobs(case, logits, ids):
    z = logits.double() / case["temperature"]
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    entropy = -torch.special.xlogy(torch.exp(logp), torch.exp(logp)).sum(1)
    at = torch.where(ids < 0, 0, ids).long()
    chosen = torch.where(ids < 0, 0.0, logp[torch.arange(len(at), device=at.device), at])
    if not case["top_k"]:
        return chosen, entropy, lse
    return chosen, entropy, lse, torch.sort(logp, 1, descending=True).values[:, :case["top_k"]]


def _exact_logprobs_grad(case, logits, ids, lse, entropy, dlogprob, dentropy, dlse):
    logp = logits.double() / case["temperature"] - lse.double()[:, None]
    p = torch.exp(logp)
    given = torch.where(ids < 0, 0.0, dlogprob.double())
    hot = torch.arange(case["vocab"], device=ids.device)[None, :] == ids[:, None]
    slope = p * (dlse.double() - given)[:, None] - dentropy.double()[:, None] * (torch.special.xlogy(p, p) + p * entropy.double()[:, None])
    return (slope + hot * given[:, None]) / case["temperature"]
