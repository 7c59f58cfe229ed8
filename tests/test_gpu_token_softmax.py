"""Log probabilities, entropy, alternatives and distillation (mh_token_softmax.hip) against the definitions in float64.

Tolerances.  z = l / T.  A row's sum is V positive terms added in at most V / 256 + 40 steps (a thread's share and the tree), each step and each
term off by 2^-24 of itself, an exponential by 2^-22: EPS(V) = (V / 256 + 64) 2^-24 of the sum, and as much of ln s absolutely.  (l - m) / T is off by
4 roundings, 2^-22 |z - max z| (for the terms of the sum that error is weighted by e^-|z - max|, which is inside the 64).  So log p is off by at most
EPS + 2^-22 (|z - max z| + |ln s|); the entropy, ln s - u / s of two such sums, by (2 + 2 ln V) EPS; lse as log p with |max z| for the distance.  A
gradient is p times a factor of g, h and ln p: relative 2 EPS + 2^-21 |z - max z| of the magnitudes that are added, and half a step of its type; a p below 2^-126 (with p |ln p| <= 2^-126 88) is 0,
the exponential instruction's least, so 2^-126 times the factor is added."""
import math

import numpy as np
import pytest
import torch

from models_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}  # results below are flushed or half a least step off
INF = math.inf


def eps(V):
    return (V / 256 + 64) * 2.0 ** -24


def make(rng, N, V, dtype, device, pad=0, off=0, scale=2.0, masked=0.02):
    x = rng.normal(size=(N, V)) * scale
    if masked:
        x[rng.random((N, V)) < masked] = -INF
    t = torch.tensor(x, dtype=torch.float32).to(TYPES[dtype]).to(device)
    if pad or off:
        wide = torch.full((N, V + pad + off), 900.0, dtype=TYPES[dtype], device=device)
        wide[:, off:off + V] = t
        t = wide[:, off:off + V]
    return t


def reference(x, T):
    """(z, log p with masked rows at -inf, entropy, lse) in float64 on the host."""
    z = x.double().cpu().numpy() / T
    m = z.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        d = np.where(np.isneginf(m), -INF, z - m)
        e = np.exp(d)
        s = e.sum(1, keepdims=True)
        lp = np.where(s > 0, d - np.log(s), -INF)
        lp = np.where(np.isnan(s), np.nan, lp)
        p = np.exp(lp)
        ent = -(np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp))).sum(1)
        lse = np.where(np.isnan(s[:, 0]), np.nan, np.where(s[:, 0] > 0, m[:, 0] + np.log(s[:, 0]), -INF))
    return z, lp, ent, lse


def close(got, want, tol):
    got, want, tol = np.broadcast_arrays(np.asarray(got, np.float64), want, tol)
    with np.errstate(all="ignore"):  # a value beyond fp32 is an infinity there
        same = (got == want) | (got == want.astype(np.float32)) | (np.isnan(got) & np.isnan(want))
    with np.errstate(all="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])


def spread(z):
    m = z.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        return np.where(np.isfinite(z) & np.isfinite(m), m - z, 0.0)


def check_logprobs(x, ids, k, T):
    N, V = x.shape
    r = ops.token_logprobs(x, ids, k=k, temperature=T)
    z, lp, ent, lse = reference(x, T)
    far, e = spread(z), eps(V)
    big = np.where(np.isfinite(z.max(1)), np.abs(z.max(1)), 0.0)
    if ids is not None:
        i = ids.cpu().numpy().astype(np.int64)
        ok = (i >= 0) & (i < V)
        at = np.where(ok, i, 0)[:, None]
        want = np.where(ok, np.take_along_axis(lp, at, 1)[:, 0], 0.0)
        close(r.logp.cpu().numpy(), want, e + 2.0 ** -22 * (np.take_along_axis(far, at, 1)[:, 0] + math.log(V)))
    else:
        assert r.logp is None
    close(r.entropy.cpu().numpy(), ent, (2 + 2 * math.log(V)) * e)
    close(r.lse.cpu().numpy(), lse, e + 2.0 ** -22 * (big + math.log(V)))
    if k:
        v = x.double().cpu().numpy()
        order = np.argsort(-np.where(np.isnan(v), -INF, v), 1, kind="stable")[:, :k]
        some = np.take_along_axis(np.where(np.isnan(v), -INF, v), order, 1) > -INF
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), np.where(some, order, -1))
        close(r.top_logp.cpu().numpy(), np.where(some, np.take_along_axis(lp, order, 1), -INF),
              e + 2.0 ** -22 * (np.take_along_axis(far, order, 1) + math.log(V)))
    return r, z, lp, ent


def check_grad(x, ids, r, z, lp, ent, T, g, h, c, inplace=False):
    N, V = x.shape
    f = lambda t: None if t is None else t.cpu().numpy().astype(np.float64)[:, None]  # noqa: E731
    one = np.zeros((N, V))
    if ids is not None:
        i = ids.cpu().numpy().astype(np.int64)
        ok = (i >= 0) & (i < V)
        one[np.arange(N)[ok], i[ok]] = 1.0
        live = ok[:, None]
    gg = np.zeros((N, 1)) if g is None else f(g) * live
    hh = np.zeros((N, 1)) if h is None else f(h)
    cc = np.zeros((N, 1)) if c is None else f(c)
    p = np.exp(lp)
    q = np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp))
    want = (gg * (one - p) - hh * (q + p * ent[:, None]) + cc * p) / T
    want[np.isneginf(z.max(1))] = 0.0  # nothing left: no gradient
    mag = (np.abs(gg) * (one + p) + np.abs(hh) * (np.abs(q) + p * ent[:, None]) + np.abs(cc) * p) / T
    # entropy and log p in the factor are themselves off by (2 + 2 ln V) EPS: relative to p, not to the factor
    tol = (2 * eps(V) + 2.0 ** -21 * (spread(z) + 4)) * mag + np.abs(hh) * p * (4 + 2 * math.log(V)) * eps(V) / T
    src = x.clone() if inplace else x
    d = ops.token_logprobs_backward(src, ids, r, g, h, c, temperature=T, out=src if inplace else None)
    assert d.dtype == x.dtype and d.shape == x.shape
    tol = tol + 2.0 ** -126 * (np.abs(gg) + np.abs(hh) * (88 + ent[:, None]) + np.abs(cc)) / T
    tol = tol * (1 + HALF[x.dtype]) + HALF[x.dtype] * np.abs(want) + LEAST[x.dtype]
    close(d.double().cpu().numpy(), want, tol)
    return d


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,k,T,pad,off", [(1, 1, 1, 1.0, 0, 0), (3, 2, 2, 0.5, 1, 0), (5, 63, 5, 2.0, 0, 1), (4, 500, 256, 1.0, 13, 3), (7, 4096, 1, 0.05, 0, 0),
                                             (2, 4097, 20, 1.0, 0, 0), (1030, 777, 7, 1.0, 0, 0), (6, 8200, 100, 1.3, 5, 7), (1, 70001, 256, 1.0, 0, 0),
                                             (3, 262147, 33, 0.7, 2, 1), (1100, 9001, 0, 1.0, 0, 0),
                                             (1025, 33001, 9, 1.0, 6, 2)])
def test_logprobs_and_gradient(device, dtype, N, V, k, T, pad, off):
    rng = np.random.default_rng(N + V + k)
    x = make(rng, N, V, dtype, device, pad, off, masked=0.02 if V > 4 else 0.0)
    ids = rng.integers(-1, V, size=N)
    ids[0] = V + 3 if N > 1 else V - 1
    ids = torch.tensor(ids, dtype=torch.int32 if N % 2 else torch.int64, device=device)
    r, z, lp, ent = check_logprobs(x, ids, k, T)
    f = lambda: torch.tensor(rng.normal(size=N), dtype=torch.float32, device=device)  # noqa: E731
    g, h, c = f(), f(), f()
    for a in ((g, None, None), (g, h, None), (None, None, c), (g, h, c)):
        check_grad(x, ids, r, z, lp, ent, T, *a)
    d = check_grad(x, ids, r, z, lp, ent, T, g, h, c, inplace=True)
    assert torch.equal(d, ops.token_logprobs_backward(x, ids, r, g, h, c, temperature=T))  # the same in place
    wide = torch.full((N, V + 9), 5.0, dtype=TYPES[dtype], device=device)
    ops.token_logprobs_backward(x, ids, r, g, h, c, temperature=T, out=wide[:, 2:2 + V])
    assert torch.equal(wide[:, 2:2 + V], d) and (wide[:, :2] == 5).all() and (wide[:, 2 + V:] == 5).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,k", [(1030, 300011, 40), (1030, 66001, 256), (1, 3000017, 256), (2, 5000, 200)])
def test_alternatives_of_long_rows(device, dtype, N, V, k):
    """Rows longer than the stretches whose largest entries are kept, large entries placed at the ends of rows and of stretches; against a sort of
    (value, place) pairs on the device."""
    g = torch.Generator(device=device).manual_seed(V)
    x = torch.empty(N, V, dtype=TYPES[dtype], device=device)
    for n in range(0, N, 64):
        x[n:n + 64] = torch.randn(min(64, N - n), V, generator=g, device=device).to(x.dtype)
    for at in (0, 1, 31, 32, 4095 * 8, 32767, V // 2, V - 1, V - 2, V - 9, V - 33):
        if 0 <= at < V:
            x[::3, at] = 9.0 + at % 3
    r = ops.token_logprobs(x, None, k=k)
    lse = torch.empty(N, device=device, dtype=torch.float64)
    for n in range(0, N, 64):
        part = x[n:n + 64]
        bits = part.float().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2 ** 31 + (2 ** 31 - 1 - torch.arange(V, device=device))
        top = key.topk(k, 1).indices
        assert torch.equal(r.top_ids[n:n + 64].long(), top)
        lse[n:n + 64] = torch.logsumexp(part.double(), 1)
        want = part.gather(1, top).double() - lse[n:n + 64, None]
        assert ((r.top_logp[n:n + 64].double() - want).abs() <= eps(V) + 2.0 ** -22 * (want.abs() + math.log(V))).all()
    assert ((r.lse.double() - lse).abs() <= eps(V) + 2.0 ** -22 * (12 + math.log(V))).all()


def awkward(dtype, V, rng):
    low = float(torch.finfo(TYPES[dtype]).min)
    base = rng.normal(size=V)
    rows = [np.full(V, -INF), np.full(V, low), np.full(V, -1e9 if dtype != "f16" else -6e4), np.zeros(V), np.full(V, 3e4)]
    a = base.copy(); a[:] = -INF; a[V // 2] = -3.0; rows.append(a)                        # one left
    a = np.full(V, low); a[[3 % V, V - 1]] = [1.0, 1.0]; rows.append(a)                       # two left, ties of the lowest value behind them
    a = np.where(rng.random(V) < 0.5, -1e9 if dtype != "f16" else -6e4, base); rows.append(a)  # masks of a large negative value
    a = np.full(V, -INF); a[: V // 3] = low; rows.append(a)                               # both kinds, nothing else
    a = np.round(base); rows.append(a)                                                    # ties
    a = base.copy(); a[::4096] = 50 + np.arange(len(a[::4096])) % 3; rows.append(a)        # the largest at one stride
    a = np.where(np.arange(V) < V // 2, -1e8 if dtype != "f16" else -5e4, base); rows.append(a)  # a long masked prefix
    if dtype == "f32":  # around the place where a thread's maximum starts
        step = 16.0 * np.round(rng.normal(size=V))
        rows += [-2.0 ** 28 / 1.4426950408889634 - 100 + step, -2.0 ** 28 / 1.4426950408889634 + step]
    if dtype != "f16":
        rows += [np.full(V, 1e10), np.full(V, -1e20), base * 1e12, base * 1e30, np.full(V, 3e38)]
    a = base.copy(); a[V // 3] = np.nan; rows.append(a)
    a = base.copy(); a[V // 3] = INF; rows.append(a)
    rows.append(np.full(V, np.nan))
    return np.stack(rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,k,T", [(37, 37, 1.0), (5000, 20, 1.0), (40000, 256, 0.5), (40000, 3, 100.0)])
def test_awkward_rows(device, dtype, V, k, T):
    rng = np.random.default_rng(V)
    rows = awkward(dtype, V, rng)
    x = torch.tensor(rows, dtype=torch.float32).to(TYPES[dtype]).to(device)
    for y in (x, x.repeat(60, 1)):  # in parts, and a workgroup a row
        n = y.shape[0]
        ids = torch.full((n,), V // 2, dtype=torch.int64, device=device)
        # far from the maximum of a row of huge values a difference of 2^-22 of it is all that is asked: check_logprobs scales with it
        r, z, lp, ent = check_logprobs(y, ids, k, T)
        w = torch.ones(n, device=device)
        d = ops.token_logprobs_backward(y, ids, r, w, w, w, temperature=T).float().cpu().numpy()
        sick = np.isnan(lp).all(1)
        assert np.isnan(d[sick]).all() and np.isfinite(d[~sick]).all()
        assert (d[np.isneginf(z.max(1))] == 0).all()


def test_padded_rows_take_no_gradient(device):
    x = torch.randn(4, 1000, device=device)
    x[2] = float("nan")
    ids = torch.tensor([5, -1, -1, 1000], device=device)
    r = ops.token_logprobs(x, ids)
    assert r.logp[1] == 0 and r.logp[2] == 0 and r.logp[3] == 0
    d = ops.token_logprobs_backward(x, ids, r, dlogp=torch.ones(4, device=device))
    assert (d[1:] == 0).all() and d[0, 5] > 0


def test_gradient_against_differences(device):
    """Directional differences of the definition in float64 (step 1e-4: off by 1e-8 of the third derivatives) against the kernel's gradient."""
    rng = np.random.default_rng(0)
    N, V, T = 6, 300, 0.7
    x = make(rng, N, V, "f32", device, masked=0.0)
    ids = torch.tensor(rng.integers(0, V, N), device=device)
    w = [torch.tensor(rng.normal(size=N), dtype=torch.float32, device=device) for _ in range(3)]
    r = ops.token_logprobs(x, ids, temperature=T)
    d = ops.token_logprobs_backward(x, ids, r, *w, temperature=T).double().cpu().numpy()

    def value(y):
        _, lp, ent, lse = reference(torch.tensor(y), T)
        i = ids.cpu().numpy()
        return sum((a.double().cpu().numpy() * b).sum() for a, b in zip(w, (lp[np.arange(N), i], ent, lse)))

    y = x.double().cpu().numpy()
    for _ in range(4):
        u = rng.normal(size=y.shape)
        num = (value(y + 1e-4 * u) - value(y - 1e-4 * u)) / 2e-4
        assert abs(num - (d * u).sum()) <= 1e-5 * np.abs(d * u).sum() + 1e-6


# ---- distillation --------------------------------------------------------------------------------------------------------------------------
def teacher(rng, N, V, K, device, dups=True, full=0.9):
    ids = np.stack([rng.choice(V, K, replace=dups or K > V) for _ in range(N)])
    lp = rng.normal(size=(N, K)) * 2
    lp = lp - np.log(np.exp(lp).sum(1, keepdims=True)) + np.log(full)
    ids[rng.random((N, K)) < 0.1] = -1
    if N > 2:
        ids[1] = -1
        lp[2, 0] = -INF
    return torch.tensor(ids, dtype=torch.int64, device=device), torch.tensor(lp, dtype=torch.float32, device=device)


def distill_reference(x, ids, tlp, T, tail):
    """loss, d loss / d logits and the magnitudes that the gradient adds up, row by row in float64."""
    N, V = x.shape
    z, lp, _, _ = reference(x, T)
    ids, t = ids.cpu().numpy(), tlp.double().cpu().numpy()
    loss, grad, mag = np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    with np.errstate(all="ignore"):
        for n in range(N):
            ok = (ids[n] >= 0) & (ids[n] < V)
            i, a = ids[n][ok], t[n][ok]
            if not len(i) or (not tail and np.isneginf(a).all()):
                continue
            lq = a if tail else a - (a.max() + np.log(np.exp(a - a.max()).sum()))
            q = np.exp(lq)
            loss[n] = np.where(q == 0, 0.0, q * (np.where(q == 0, 0.0, lq) - lp[n, i])).sum()
            dist = np.zeros(V)
            np.add.at(dist, i, q)
            p = np.exp(lp[n])
            c, r = q.sum(), 0.0
            top = np.zeros(V, bool)
            top[i] = True
            pi = np.zeros(V)
            if tail and (z[n][~top] > -INF).any():
                rest = lp[n][~top]
                lr = rest.max() + np.log(np.exp(rest - rest.max()).sum())
                r = max(0.0, 1.0 - c)
                if r > 0:
                    loss[n] += r * (np.log(r) - lr)
                pi[~top] = np.exp(rest - lr)
            if np.isneginf(z[n].max()):
                continue
            grad[n] = ((c + r) * p - dist - r * pi) / T
            mag[n] = ((c + r) * p + dist + r * pi) / T
    return z, lp, loss, grad, mag


def check_distill(x, ids, tlp, T, tail, rng):
    N, V = x.shape
    z, lp, loss, grad, mag = distill_reference(x, ids, tlp, T, tail)
    far = spread(z)
    i = np.where((ids.cpu().numpy() >= 0) & (ids.cpu().numpy() < V), ids.cpu().numpy(), 0)
    tol = eps(V) + 2.0 ** -22 * (np.take_along_axis(far, i, 1).max(1) + math.log(V)) + 2.0 ** -23 * np.abs(np.where(np.isfinite(loss), loss, 0))
    for need in (True, False):
        res = ops.distill_topk(x, ids, tlp, T, tail, need_grad=need)
        close(res.loss.cpu().numpy(), loss, tol)
    w = torch.tensor(rng.normal(size=N), dtype=torch.float32, device=x.device)
    ww = w.double().cpu().numpy()[:, None]
    res, d = ops.distill_topk_train(x, ids, tlp, w, T, tail)
    close(res.loss.cpu().numpy(), loss, tol)
    rel = 3 * eps(V) + 2.0 ** -21 * (far + 4)
    gt = (rel * mag + 2.0 ** -126 * 3 / T) * np.abs(ww) * (1 + HALF[x.dtype]) + HALF[x.dtype] * np.abs(grad * ww) + LEAST[x.dtype]
    close(d.double().cpu().numpy(), grad * ww, gt)
    parts = ops.distill_topk(x, ids, tlp, T, tail)
    again = ops.distill_topk_backward(x, ids, parts, w, T)
    close(again.double().cpu().numpy(), grad * ww, gt)
    ones = ops.distill_topk_backward(x, ids, parts, temperature=T)
    gt1 = (rel * mag + 2.0 ** -126 * 3 / T) * (1 + HALF[x.dtype]) + HALF[x.dtype] * np.abs(grad) + LEAST[x.dtype]
    close(ones.double().cpu().numpy(), grad, gt1)
    i2, t2 = (torch.cat([a, a.flip(1)], 1)[:, : a.shape[1]] for a in (ids, tlp))  # parts of wider rows
    r2, d2 = ops.distill_topk_train(x, i2, t2, w, T, tail)
    assert torch.equal(d2, d) and torch.equal(r2.loss, res.loss)
    y = x.clone()
    _, inplace = ops.distill_topk_train(y, ids, tlp, w, T, tail, out=y)
    assert inplace.data_ptr() == y.data_ptr() and torch.equal(inplace, d)
    return d


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,K,T,pad,off", [(1, 1, 1, 1.0, 0, 0), (3, 4, 4, 2.0, 0, 1), (5, 63, 7, 1.0, 3, 0), (9, 1009, 256, 0.5, 0, 0), (4, 4100, 33, 1.0, 7, 5),
                                             (1030, 600, 5, 1.0, 0, 0), (2, 70001, 128, 1.0, 0, 0), (3, 300007, 64, 3.0, 1, 0), (1040, 8300, 16, 1.0, 0, 0),
                                             (2, 4096, 9, 1.0, 0, 0), (2, 16385, 64, 1.0, 0, 3), (66, 65543, 40, 1.0, 3, 0), (65, 131072, 128, 2.0, 0, 0)])
def test_distill(device, dtype, tail, N, V, K, T, pad, off):
    rng = np.random.default_rng(N + V + K)
    x = make(rng, N, V, dtype, device, pad, off, masked=0.0)
    ids, tlp = teacher(rng, N, V, K, device)
    check_distill(x, ids if N % 2 else ids.to(torch.int32), tlp, T, tail, rng)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,T", [(37, 1.0), (9000, 0.5)])
def test_distill_awkward_rows(device, dtype, tail, V, T):
    rng = np.random.default_rng(V)
    rows = awkward(dtype, V, rng)
    x = torch.tensor(rows, dtype=torch.float32).to(TYPES[dtype]).to(device)
    N = len(rows)
    _, tlp = teacher(rng, N, V, 8, device)
    ids = torch.tensor(rng.integers(0, V, size=(N, 8)), device=device)
    ids[:, 0] = V // 2
    for rep in (1, 60):
        y, i, t = x.repeat(rep, 1), ids.repeat(rep, 1), tlp.repeat(rep, 1)
        z, lp, loss, grad, mag = distill_reference(y, i, t, T, tail)
        r, d = ops.distill_topk_train(y, i, t, None, T, tail)
        far = np.take_along_axis(spread(z), i.cpu().numpy(), 1).max(1)
        close(r.loss.cpu().numpy(), loss, eps(V) + 2.0 ** -22 * (far + math.log(V)) + 2.0 ** -22 * np.abs(np.where(np.isfinite(loss), loss, 0)))
        sick = np.isnan(lp).all(1)
        d = d.double().cpu().numpy()
        assert np.isnan(d[sick]).any(1).all() and np.isfinite(d[~sick]).all()
        # a gradient of huge logits: where probabilities are 0 or 1 to the last bit it is exact, and nothing else is asked of it here
        flat = ~sick & (np.abs(z).max(1, where=np.isfinite(z), initial=0) < 1e5)
        gt = ((3 * eps(V) + 2.0 ** -21 * (spread(z) + 4)) * mag + 2.0 ** -126 * 3 / T) * (1 + HALF[x.dtype]) + HALF[x.dtype] * np.abs(grad) + LEAST[x.dtype]
        close(d[flat], grad[flat], gt[flat])


def test_distill_teacher_covers_the_catalogue_or_its_mass(device):
    """No column besides the teacher's entries, masses that leave nothing over, and entries without mass."""
    rng = np.random.default_rng(4)
    x = make(rng, 6, 12, "f32", device, masked=0.0)
    ids = torch.arange(12, device=device).repeat(6, 1)
    _, tlp = teacher(rng, 6, 12, 12, device)
    check_distill(x, ids, tlp, 1.0, True, rng)
    check_distill(x, ids[:, :3].contiguous(), torch.log_softmax(tlp[:, 3:6], 1).contiguous(), 1.0, True, rng)
    check_distill(x, ids[:, :3].contiguous(), torch.full((6, 3), -INF, device=device), 1.0, False, rng)
    check_distill(x, ids[:, :3].contiguous(), torch.full((6, 3), -INF, device=device), 1.0, True, rng)
    x[:, 5:] = -INF  # the student has nothing outside five columns
    check_distill(x, ids[:, :5].contiguous(), torch.log_softmax(tlp[:, 3:8], 1).contiguous() - 0.5, 1.0, True, rng)


def test_distill_gradient_against_differences(device):
    rng = np.random.default_rng(1)
    N, V, K, T = 5, 200, 9, 1.5
    x = make(rng, N, V, "f32", device, masked=0.0)
    ids, tlp = teacher(rng, N, V, K, device)
    for tail in (False, True):
        _, d = ops.distill_topk_train(x, ids, tlp, None, T, tail)
        d, y = d.double().cpu().numpy(), x.double().cpu().numpy()
        value = lambda v: distill_reference(torch.tensor(v), ids, tlp, T, tail)[2].sum()  # noqa: E731
        for _ in range(3):
            u = rng.normal(size=y.shape)
            num = (value(y + 1e-4 * u) - value(y - 1e-4 * u)) / 2e-4
            assert abs(num - (d * u).sum()) <= 1e-5 * np.abs(d * u).sum() + 1e-6


# ---- used together ------------------------------------------------------------------------------------------------------------------------
def test_teacher_to_student(device):
    """8-bit catalogue logits of a teacher, its top alternatives, the student's distillation loss and the gradients of its own 8-bit head."""
    g = torch.Generator(device=device).manual_seed(3)
    B, E, V, K, T = 70, 128, 5003, 32, 2.0
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    q, table, sq, st = rand(B, E) * 0.3, rand(V, E) * 0.3, rand(B, E) * 0.3, rand(V, E) * 0.3
    t8, s8 = ops.fp8_quantize(table), ops.fp8_quantize(st)
    t = ops.token_logprobs(ops.fp8_linear(q, t8), k=K, temperature=T)
    logits = ops.fp8_linear(sq, s8)
    w = torch.full((B,), 1.0 / B, device=device)
    res, d = ops.distill_topk_train(logits, t.top_ids, t.top_logp, w, T, True)
    z, lp, loss, grad, mag = distill_reference(logits, t.top_ids.long(), t.top_logp, T, True)
    close(res.loss.cpu().numpy(), loss, 4 * eps(V) + 2.0 ** -20)
    dq, dtable = ops.fp8_linear_backward(sq, ops.fp8_quantize(st.T.contiguous()), d)
    assert dq.shape == (B, E) and dtable.shape == (E, V)
    full = torch.matmul(d.double(), st.double())
    assert ((dq.double() - full).abs() <= 0.13 * torch.matmul(d.double().abs(), st.double().abs()) + 1e-9).all()
    # a step against that gradient lowers the loss of the layer it belongs to: the directional derivative is negative
    assert (torch.matmul(d.double().T.contiguous(), sq.double()) * dtable.T.double()).sum() > 0


def test_streams_and_graphs(device):
    """Two streams at once, and a captured step replayed on new logits with eager work between, give the eager results bit for bit."""
    rng = np.random.default_rng(9)
    N, V, K = 3, 50000, 20
    xs = [make(rng, N, V, "bf16", device) for _ in range(2)]
    ids = torch.tensor(rng.integers(0, V, N), device=device)
    tid, tlp = teacher(rng, N, V, K, device)
    w = torch.ones(N, device=device)

    def step(x):
        r = ops.token_logprobs(x, ids, k=K)
        d = ops.token_logprobs_backward(x, ids, r, w, w)
        s, e = ops.distill_topk_train(x, tid, tlp, w, 1.0, True)
        return [r.logp, r.entropy, r.lse, r.top_logp, r.top_ids, d, s.loss, e]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step(xs[i % 2]))
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(u.nan_to_num(7), v.nan_to_num(7)) for u, v in zip(a, b))  # noqa: E731
    for i, o in enumerate(got):
        assert same(o, want[i % 2])
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in (1, 0, 1):
        static.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want[i])
        assert same(step(xs[i]), want[i])


def test_recorded_and_replayed(device):
    """The library's own launch recording replays the calls on new inputs in the same buffers."""
    import ctypes as C

    from models_amd import _lib

    lib = _lib.load()
    rng = np.random.default_rng(2)
    xs = [make(rng, 5, 3000, "f32", device) for _ in range(2)]
    ids, (tid, tlp) = torch.tensor(rng.integers(0, 3000, 5), device=device), teacher(rng, 5, 3000, 7, device)
    w8 = ops.fp8_quantize(torch.randn(40, 3000, device=device))
    keep = []

    def step(x):
        r = ops.token_logprobs(x, ids, k=4)
        s, d = ops.distill_topk_train(x, tid, tlp, None, 1.0, True)
        keep.append((r, s, d))
        return [r.logp, r.entropy, r.top_logp, r.top_ids, s.loss, d, ops.fp8_linear(x, w8)]

    static = xs[0].clone()
    h = C.c_void_p()
    assert lib.mh_record_begin() == 0
    out = step(static)
    assert lib.mh_record_end(C.byref(h)) == 0
    for i in (1, 0, 1):
        static.copy_(xs[i])
        torch.cuda.synchronize()
        assert lib.mh_record_replay(h) == 0
        torch.cuda.synchronize()
        want = ops.token_logprobs(xs[i], ids, k=4)
        s, d = ops.distill_topk_train(xs[i], tid, tlp, None, 1.0, True)
        y = ops.fp8_linear(xs[i], w8)
        for a, b in zip(out, [want.logp, want.entropy, want.top_logp, want.top_ids, s.loss, d, y]):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    lib.mh_record_free(h)


def test_refusals(device):
    x = torch.zeros(4, 10, device=device)
    ids = torch.zeros(4, dtype=torch.int64, device=device)
    tid, tlp = torch.zeros(4, 3, dtype=torch.int64, device=device), torch.zeros(4, 3, device=device)
    r, s = ops.token_logprobs(x, ids), ops.distill_topk(x, tid, tlp)
    one = torch.ones(4, device=device)
    for bad in (lambda: ops.token_logprobs(x.T), lambda: ops.token_logprobs(x[0]), lambda: ops.token_logprobs(x[:1].expand(4, 10)),
                lambda: ops.token_logprobs(x, ids[:3]), lambda: ops.token_logprobs(x, k=11), lambda: ops.token_logprobs(x, k=-1),
                lambda: ops.token_logprobs(x, temperature=0.0), lambda: ops.token_logprobs(x, temperature=float("nan")),
                lambda: ops.token_logprobs(x[:, :0]), lambda: ops.token_logprobs(torch.zeros(2, 400, device=device), k=257),
                lambda: ops.token_logprobs_backward(x, None, r, dlogp=one), lambda: ops.token_logprobs_backward(x, ids, r, dlogp=one[:3]),
                lambda: ops.token_logprobs_backward(x, ids, r, dlogp=one, out=x[:, :9]),
                lambda: ops.token_logprobs_backward(x[:3], ids[:3], r, dlogp=one[:3]),
                lambda: ops.distill_topk(x, tid[:3], tlp), lambda: ops.distill_topk(x, tid, tlp[:, :2]), lambda: ops.distill_topk(x, tid, None),
                lambda: ops.distill_topk(x, tid[:, :0], tlp[:, :0]), lambda: ops.distill_topk(x, tid[:, 0], tlp), lambda: ops.distill_topk(x, tid[:, ::2], tlp[:, :2]),
                lambda: ops.distill_topk(x, tid, tlp[:1].expand(4, 3)),
                lambda: ops.distill_topk(x, torch.zeros(4, 257, dtype=torch.int64, device=device), torch.zeros(4, 257, device=device)),
                lambda: ops.distill_topk_backward(x, tid, ops.distill_topk(x, tid, tlp, need_grad=False)),
                lambda: ops.distill_topk_backward(x, tid, s, dloss=one[:3]), lambda: ops.distill_topk_train(x, tid, tlp, one[:3])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.token_logprobs(x.double()), lambda: ops.token_logprobs(x, ids.float()), lambda: ops.distill_topk(x, tid, tlp.half()),
                lambda: ops.token_logprobs_backward(x, ids, r, dlogp=one.half())):
        with pytest.raises(TypeError):
            bad()
    assert ops.token_logprobs(x, ids, temperature=np.float32(0.5)).logp.shape == (4,)
    wide = torch.zeros(4, 12, device=device)
    with pytest.raises(ValueError):
        ops.token_logprobs_backward(wide[:2, :10], ids[:2], ops.token_logprobs(wide[:2, :10], ids[:2]), one[:2], out=wide.view(-1)[:20].view(2, 10))
    assert ops.token_logprobs(x[:0], ids[:0], k=2).top_ids.shape == (0, 2)
    assert ops.token_logprobs_backward(x[:0], ids[:0], ops.token_logprobs(x[:0], ids[:0]), dlogp=one[:0]).shape == (0, 10)
    assert ops.distill_topk_train(x[:0], tid[:0], tlp[:0])[1].shape == (0, 10)
