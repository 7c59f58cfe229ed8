"""Measured cases of the catalogue-softmax operators and the 8-bit product that feeds them.

Three families, each a call of ``models_amd.ops``:

* ``fp8_linear`` / ``fp8_linear_backward``: a Dense layer whose operands are e4m3 with one power-of-two scale for each row and each 128
  entries of the summed axis;
* ``token_logprobs`` / ``token_logprobs_backward``: log probabilities of given ids, entropy, log-sum-exp and the top alternatives of
  ``[N, V]`` logits, and the gradient;
* ``distill_topk`` / ``distill_topk_train``: Kullback-Leibler distillation from a teacher's top entries, and the gradient.

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BLOCK = 128


# ---- cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one query through a projection: the smallest call, bound by latency
        {"name": "fp8 one row", "op": "fp8_linear", "M": 1, "K": 1024, "N": 4096, "dtype": "bf16", "out": "bf16", "bias": False},
        # a serving batch of a few queries: the weights are read once, little else is
        {"name": "fp8 few rows", "op": "fp8_linear", "M": 48, "K": 4096, "N": 14341, "dtype": "bf16", "out": "bf16", "bias": True},
        # the wide Dense layer of the DCN-v2 configuration (3341 -> 512 at batch 64 K), fp32 activations as the framework holds them
        {"name": "fp8 dcn 3341-512", "op": "fp8_linear", "M": 65536, "K": 3341, "N": 512, "dtype": "f32", "out": "f32", "bias": True},
        # a square product: the matrix pipe is the bound
        {"name": "fp8 square 8192", "op": "fp8_linear", "M": 8192, "K": 8192, "N": 8192, "dtype": "bf16", "out": "bf16", "bias": False},
        # both gradients of a Dense layer in training
        {"name": "fp8 gradients", "op": "fp8_grad", "M": 16384, "K": 1024, "N": 2048, "dtype": "f32"},
        # one decoding step: one row, the next id's alternatives
        {"name": "logprobs one row", "op": "logprobs", "N": 1, "V": 131072, "k": 20, "dtype": "bf16", "T": 0.8, "pad": 0},
        # the repository's catalogue of a million items, its top 100 beside the given item's log probability
        {"name": "logprobs catalogue 1M", "op": "logprobs", "N": 64, "V": 1000000, "k": 100, "dtype": "f32", "T": 1.0, "pad": 0},
        # a training step on in-batch logits [B, 1 + B] with an entropy bonus: odd rows, so no row but the first is aligned
        {"name": "logprobs train 8K x 32769", "op": "logprobs_grad", "N": 8192, "V": 32769, "k": 0, "dtype": "f32", "T": 0.05, "pad": 0},
        # the same over a large vocabulary in 16 bits, rows padded to a multiple of 64
        {"name": "logprobs train 4K x 131003", "op": "logprobs_grad", "N": 4096, "V": 131003, "k": 8, "dtype": "bf16", "T": 1.0, "pad": 69},
        # distilling a small ranker: latency
        {"name": "distill small", "op": "distill_grad", "N": 16, "V": 1009, "K": 5, "dtype": "f32", "T": 2.0, "tail": False, "pad": 0},
        # evaluating a student: the loss alone
        {"name": "distill loss 2K x 50021", "op": "distill", "N": 2048, "V": 50021, "K": 64, "dtype": "f16", "T": 1.0, "tail": False, "pad": 27},
        # a training step of a student over a large vocabulary, the teacher's remaining mass kept
        {"name": "distill train 4K x 131072", "op": "distill_grad", "N": 4096, "V": 131072, "K": 128, "dtype": "bf16", "T": 1.0, "tail": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["fp8_linear", "fp8_linear", "fp8_grad", "logprobs", "logprobs", "logprobs_grad", "distill", "distill_grad"])
    if op == "fp8_linear":
        while True:
            M, K, N = _log(rng, 1, 65536), _log(rng, 64, 8192), _log(rng, 64, 16384)
            if M * K * N <= 8192 ** 3 and M * N <= 1 << 28:
                break
        return {"op": op, "M": M, "K": K, "N": N, "dtype": rng.choice(["f32", "bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5}
    if op == "fp8_grad":
        while True:
            M, K, N = _log(rng, 64, 65536), _log(rng, 64, 4096), _log(rng, 64, 4096)
            if M * K * N <= 8192 ** 3 // 4:
                break
        return {"op": op, "M": M, "K": K, "N": N, "dtype": rng.choice(["f32", "bf16"])}
    most = 1 << 28  # entries: the largest listed case has twice that
    V = _log(rng, 500, 1000000 if op == "logprobs" else 200000)
    N = min(_log(rng, 1, 16384), max(1, most // V))
    c = {"op": op, "N": N, "V": V, "dtype": rng.choice(["f32", "bf16", "f16"]), "T": round(rng.uniform(0.25, 2.0), 3),
         "pad": rng.choice([0, 0, 1, 8, 61])}
    if op.startswith("logprobs"):
        c["k"] = rng.choice([0, 1, 5, 20, _log(rng, 1, 128)])
    else:
        c["K"], c["tail"] = _log(rng, 1, 256), rng.random() < 0.5
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _two(e):
    """2^e as a 32-bit value, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantized(x):
    """The stored form of a matrix: e4m3 ``[R, ceil(K / 128) 128]`` and the biased exponents of its scales ``[R, blocks rounded up to 4]``."""
    R, K = x.shape
    kb = -(-K // _BLOCK)
    p = torch.zeros(R, kb * _BLOCK, device=x.device)
    p[:, :K] = x
    p = p.view(R, kb, _BLOCK)
    f, e = torch.frexp(p.abs().amax(2))
    e = torch.where(f == 0, 0, e - 9 + (f > 0.875).int()).clamp(-126, 120)  # the least e with amax <= 448 * 2^e
    q = (p * _two(-e)[:, :, None]).to(torch.float8_e4m3fn).view(R, kb * _BLOCK)
    s = torch.full((R, -(-kb // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    s[:, :kb] = (e + 127).to(torch.uint8)
    return q, s


def _logits(case, g):
    """Logits as a trained head gives them: a popularity slope over the catalogue, a few strong candidates a row, and some masked items."""
    N, V, ld = case["N"], case["V"], case["V"] + case["pad"]
    x = torch.empty(N, ld, dtype=_DT[case["dtype"]], device="cuda")
    slope = -torch.log1p(torch.randperm(V, generator=g, device="cuda").float() / 64.0)
    masked = torch.rand(V, generator=g, device="cuda") < 0.02
    step = max(1, (1 << 26) // ld)
    for a in range(0, N, step):  # in parts, to keep the temporaries small
        n = min(step, N - a)
        part = torch.randn(n, V, generator=g, device="cuda") * 1.7 + slope
        hot = torch.randint(0, V, (n, 4), generator=g, device="cuda")
        part.scatter_add_(1, hot, torch.rand(n, 4, generator=g, device="cuda") * 6)
        part[:, masked] = -math.inf
        x[a:a + n, :V] = part * case["T"]
        if ld > V:
            x[a:a + n, V:] = 1e4  # behind the row: never to be read as part of it
    return x[:, :V]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op = case["op"]
    if op.startswith("fp8"):
        M, K, N = case["M"], case["K"], case["N"]
        st = dict(case)
        st["x"] = (rand(M, K) * torch.exp(rand(1, K))).to(_DT[case["dtype"]])  # columns of unlike size, as features are
        if op == "fp8_linear":
            st["w"], st["ws"] = _quantized(rand(N, K) / math.sqrt(K))
            st["b"] = rand(N) if case["bias"] else None
        else:
            st["w"], st["ws"] = _quantized(rand(K, N) / math.sqrt(K))  # W[K, N] with its blocks along N
            st["dy"] = (rand(M, N) * 1e-3).to(_DT[case["dtype"]])
        return st
    N, V = case["N"], case["V"]
    st = dict(case)
    st["logits"] = _logits(case, g)
    if op.startswith("logprobs"):
        ids = torch.randint(0, V, (N,), generator=g, device="cuda")
        # where the given id is a masked one the row's value is -inf; training data holds no such id
        best = st["logits"].argmax(1)
        ids = torch.where(torch.isinf(st["logits"].gather(1, ids[:, None])[:, 0]), best, ids)
        if N > 8:
            ids[torch.rand(N, generator=g, device="cuda") < 0.03] = -1  # padding
        st["ids"] = ids
        st["dlogp"] = -torch.rand(N, generator=g, device="cuda") / N
        st["dent"] = torch.full((N,), -0.01 / N, device="cuda")
    else:
        K = case["K"]
        t = st["logits"][:, :V].float() if N * V <= 1 << 24 else None
        # the teacher's best are near the student's: half from the student's strong items, half drawn
        ids = torch.randint(0, V, (N, K), generator=g, device="cuda", dtype=torch.int64)
        if t is not None:
            top = t.topk(min(K, V), 1).indices[:, : K // 2]
            ids[:, : top.shape[1]] = top
        ids = torch.where(torch.isinf(st["logits"].gather(1, ids)), st["logits"].argmax(1, keepdim=True), ids)
        lp = torch.log_softmax(rand(N, K + 1) * 2, 1)[:, :K]  # log probabilities that leave some mass over
        ids[torch.rand(N, K, generator=g, device="cuda") < 0.02] = -1
        if N > 8:
            ids[torch.rand(N, generator=g, device="cuda") < 0.03] = -1  # padded rows
        st["tid"], st["tlp"] = ids.to(torch.int32), lp
        st["dloss"] = torch.rand(N, generator=g, device="cuda") / N
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _round8(x):
    """x rounded to e4m3 with the power-of-two scale of each 128 of its last axis, as 32-bit values."""
    R, K = x.shape
    kb = -(-K // _BLOCK)
    p = torch.nn.functional.pad(x.float(), (0, kb * _BLOCK - K)).view(R, kb, _BLOCK)
    f, e = torch.frexp(p.abs().amax(2, keepdim=True))
    e = torch.where(f == 0, 0, e - 9 + (f > 0.875).int()).clamp(-126, 120)
    return ((p * _two(-e)).to(torch.float8_e4m3fn).float() * _two(e)).view(R, kb * _BLOCK)[:, :K]


def _values(q, s, K):
    kb = q.shape[1] // _BLOCK
    v = q.float().view(q.shape[0], kb, _BLOCK) * _two(s[:, :kb, None].int() - 127)
    return v.view(q.shape[0], kb * _BLOCK)[:, :K]


def _softmax(x, T):
    """Row statistics of x / T: (shifted x / T, exp of it, sum, row maximum), masked rows left with a sum of zero."""
    z = x.float() / T
    m = z.amax(1, keepdim=True)
    z = z - torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(z)
    return z, e, e.sum(1, keepdim=True), m


def _logprobs(st, grad):
    x, ids, k, T = st["logits"], st["ids"].long(), st["k"], st["T"]
    N, V = x.shape
    z, e, s, m = _softmax(x, T)
    has = ids >= 0
    at = ids.clamp(min=0)[:, None]
    logs = s.log()
    logp = torch.where(has, (z.gather(1, at) - logs)[:, 0], 0.0)
    fin = torch.where(e > 0, z, 0.0)
    ent = (logs - (e * fin).sum(1, keepdim=True) / s)[:, 0]
    out = [logp, ent, (logs + m)[:, 0]]
    if k:
        # ties go to the lowest index: the place is part of the key
        bits = x.float().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2 ** 31 + (2 ** 31 - 1 - torch.arange(V, device=x.device))
        top = key.topk(k, 1).indices
        out += [z.gather(1, top) - logs, top.int()]
    if grad:
        g, h = torch.where(has, st["dlogp"], 0.0)[:, None], st["dent"][:, None]
        p = e / s
        d = -p * (g + h * (fin - logs + ent[:, None]))
        d.scatter_add_(1, at, g)
        out.append((d / T).to(x.dtype))
    return out


def _distill(st, grad):
    x, ids, T = st["logits"], st["tid"].long(), st["T"]
    z, e, s, _ = _softmax(x, T)
    ok = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(ok, st["tlp"].double(), -math.inf)
    row = ok.any(1, keepdim=True)
    logs = s.log()
    lp = z.gather(1, at) - logs
    if st["tail"]:
        q = torch.exp(t)
        r = torch.where(row, (1 - q.sum(1, keepdim=True)).clamp(min=0), 0.0)
        hit = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, at, ok.int()) > 0
        rest = torch.where(hit, 0.0, e).sum(1, keepdim=True)
        r = torch.where(rest > 0, r, 0.0)
    else:
        q = torch.exp(t - torch.where(row, t.amax(1, keepdim=True), 0.0))
        q = torch.where(row, q / q.sum(1, keepdim=True), 0.0)
        r = torch.zeros_like(row, dtype=torch.float64)
    lq = torch.where(q > 0, torch.log(q), 0.0)
    loss = torch.where(q > 0, q * (lq - lp), 0.0).sum(1, keepdim=True)
    if st["tail"]:
        lr = torch.log(rest) - logs
        loss = loss + torch.where(r > 0, r * (torch.where(r > 0, torch.log(r), 0.0) - lr), 0.0)
    out = [loss[:, 0].float()]
    if grad:
        p = e / s
        c = (q.sum(1, keepdim=True) + r)
        if st["tail"]:
            d = p * torch.where(hit, c.float(), torch.where(rest > 0, (c - r * s / rest), 0.0).float())
        else:
            d = p * c.float()
        d.scatter_add_(1, at, torch.where(ok, -q, 0.0).float())
        out.append((d * (st["dloss"][:, None] / T)).to(x.dtype))
    return out


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        return _own(st)
    op = st["op"]
    if op == "fp8_linear":
        y = _round8(st["x"]) @ _values(st["w"], st["ws"], st["K"]).t()
        if st["b"] is not None:
            y = y + st["b"]
        return y.to(_DT[st["out"]])
    if op == "fp8_grad":
        x, dy = st["x"], st["dy"]
        dx = _round8(dy) @ _values(st["w"], st["ws"], st["N"]).t()
        dw = _round8(x.t()) @ _round8(dy.t()).t()
        return dx, dw
    if op.startswith("logprobs"):
        return _logprobs(st, op.endswith("grad"))
    return _distill(st, op.endswith("grad"))


def _own(st):
    from models_amd import ops

    op = st["op"]
    if op == "fp8_linear":
        return ops.fp8_linear(st["x"], ops.Fp8Matrix(st["w"], st["ws"], st["K"]), st["b"], out_dtype=_DT[st["out"]])
    if op == "fp8_grad":
        return ops.fp8_linear_backward(st["x"], ops.Fp8Matrix(st["w"], st["ws"], st["N"]), st["dy"])
    if op.startswith("logprobs"):
        r = ops.token_logprobs(st["logits"], st["ids"], k=st["k"], temperature=st["T"])
        out = [r.logp, r.entropy, r.lse]
        if st["k"]:
            out += [r.top_logp, r.top_ids]
        if op.endswith("grad"):
            out.append(ops.token_logprobs_backward(st["logits"], st["ids"], r, dlogp=st["dlogp"], dentropy=st["dent"], temperature=st["T"]))
        return out
    if op == "distill":
        return [ops.distill_topk(st["logits"], st["tid"], st["tlp"], temperature=st["T"], tail=st["tail"]).loss]
    r, d = ops.distill_topk_train(st["logits"], st["tid"], st["tlp"], st["dloss"], temperature=st["T"], tail=st["tail"])
    return [r.loss, d]


def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "f32" else 2
    if op.startswith("fp8"):
        M, K, N = case["M"], case["K"], case["N"]
        if op == "fp8_linear":
            return {"bytes": M * K * es + N * K + N * K // 128 + M * N * (4 if case["out"] == "f32" else 2) + (4 * N if case["bias"] else 0),
                    "flops": 2 * M * K * N}
        return {"bytes": M * K * es + M * N * es + K * N + 4 * M * K + 4 * K * N, "flops": 4 * M * K * N}
    N, V = case["N"], case["V"]
    grad = op.endswith("grad")
    per_row = 8 + 12 + 8 * case["k"] + (8 if grad else 0) if "k" in case else 8 * case["K"] + 4 + (4 if grad else 0)
    return {"bytes": N * V * es * (2 if grad else 1) + N * per_row, "flops": N * V * (12 if grad else 6)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _e4m3(v):
    """v (double, within +-448) to the nearest e4m3 value, ties to even: steps of 2^(exponent - 3), the least 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact8(x):
    """e4m3 values of x by blocks of 128 along its rows, in double; the scale is found by trying: the least power of two that fits."""
    R, K = x.shape
    out = torch.empty(R, K, dtype=torch.float64, device=x.device)
    for a in range(0, K, _BLOCK):
        v = x[:, a:a + _BLOCK].double()
        big = v.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(torch.where(big > 0, big, 448.0) / 448.0)) - 1
        for _ in range(3):
            e = e + (big > 448.0 * torch.exp2(e)).double()
        e = e.clamp(-126, 120)
        out[:, a:a + _BLOCK] = _e4m3(v / torch.exp2(e)) * torch.exp2(e)
    return out


def _stored8(q, s, K):
    scale = torch.exp2(s.double() - 127).repeat_interleave(_BLOCK, 1)[:, :K]
    return q.double()[:, :K] * scale


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "fp8_linear":
        y = torch.matmul(_exact8(st["x"]), _stored8(st["w"], st["ws"], case["K"]).t())
        return y if st["b"] is None else y + st["b"].double()
    if op == "fp8_grad":
        dx = torch.matmul(_exact8(st["dy"]), _stored8(st["w"], st["ws"], case["N"]).t())
        return dx, torch.matmul(_exact8(st["x"].t()), _exact8(st["dy"].t()).t())
    N, V = st["logits"].shape
    parts, step = [], max(1, (1 << 27) // V)
    for a in range(0, N, step):
        rows = slice(a, min(N, a + step))
        lp = torch.log_softmax(st["logits"][rows].double() / case["T"], 1)
        parts.append(_exact_logprobs(st, rows, lp) if op.startswith("logprobs") else _exact_distill(st, rows, lp))
    return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]


def _exact_logprobs(st, rows, lp):
    x, ids = st["logits"][rows], st["ids"][rows]
    real = ids >= 0
    one = torch.zeros_like(lp)
    one[torch.arange(len(ids), device=ids.device)[real], ids[real]] = 1.0
    p = lp.exp()
    plogp = torch.nan_to_num(p * lp, nan=0.0)
    ent = -plogp.sum(1)
    out = [torch.nan_to_num(one * lp, nan=0.0).sum(1), ent, torch.logsumexp(x.double() / st["T"], 1)]
    if st["k"]:
        order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, : st["k"]]
        out += [lp.gather(1, order), order.int()]
    if st["op"].endswith("grad"):
        g, h = st["dlogp"][rows].double() * real, st["dent"][rows].double()
        out.append((g[:, None] * (one - p) - h[:, None] * (plogp + p * ent[:, None])) / st["T"])
    return out


def _exact_distill(st, rows, lp):
    ids, t = st["tid"][rows].long(), st["tlp"][rows].double()
    real = ids >= 0
    n, V = lp.shape
    at = torch.arange(n, device=lp.device)[:, None].expand_as(ids)
    mass = torch.where(real, torch.exp(t), 0.0)
    if not st["tail"]:
        mass = mass / mass.sum(1, keepdim=True).clamp(min=1e-300)
    q = torch.zeros_like(lp).index_put_((at[real], ids[real]), mass[real], accumulate=True)
    own_lp = lp.gather(1, ids.clamp(min=0))
    loss = torch.where(real & (mass > 0), mass * (torch.log(mass.clamp(min=1e-300)) - own_lp), 0.0).sum(1)
    p = lp.exp()
    grad = mass.sum(1, keepdim=True) * p - q
    if st["tail"]:
        top = torch.zeros_like(lp, dtype=torch.bool).index_put_((at[real], ids[real]), torch.tensor(True, device=lp.device))
        rest = torch.where(top, -math.inf, lp)
        lrest = torch.logsumexp(rest, 1, keepdim=True)
        left = (1 - mass.sum(1, keepdim=True)).clamp(min=0) * real.any(1, keepdim=True) * torch.isfinite(lrest)
        loss = loss + torch.where(left > 0, left * (torch.log(left.clamp(min=1e-300)) - lrest), 0.0)[:, 0]
        grad = grad + left * (p - torch.exp(rest - lrest))
    out = [loss]
    if st["op"].endswith("grad"):
        out.append(grad * st["dloss"][rows].double()[:, None] / st["T"])
    return out
