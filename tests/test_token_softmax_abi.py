"""What the entry points of the catalogue softmax refuse, on the host: every check comes before the first use of the device."""
import ctypes as C

import pytest
import torch

from models_amd import _lib, ops

P = C.c_void_p
A = 0x1000  # an address that is never used: the calls below end before a launch


def call(name, order, defaults, **kw):
    a = dict(defaults, **kw)
    return getattr(_lib.load(), name)(*[P(a[n]) if n in POINTERS else a[n] for n in order])


POINTERS = {"x", "ids", "logp", "ent", "lse", "tlogp", "tids", "stats", "ws", "stream", "g", "h", "c", "d", "tlp", "loss", "top", "w"}
LP = dict(x=A, dt=0, ld=1000, N=2, V=1000, ids=A, idt=1, k=5, T=1.0, logp=A, ent=A, lse=A, tlogp=A, tids=A, stats=A, ws=A, nws=1 << 20, stream=0)
LPB = dict(x=A, dt=0, ld=1000, N=2, V=1000, ids=A, idt=1, T=1.0, stats=A, ent=A, g=A, h=A, c=A, d=A, ldd=1000, stream=0)
DS = dict(x=A, dt=0, ld=1000, N=2, V=1000, ids=A, idt=1, ldi=5, tlp=A, ldt=5, K=5, T=1.0, tail=1, loss=A, stats=A, top=A, ws=A, nws=1 << 20, stream=0)
DSB = dict(x=A, dt=0, ld=1000, N=2, V=1000, ids=A, idt=1, ldi=5, K=5, T=1.0, stats=A, top=A, w=A, d=A, ldd=1000, stream=0)
COMMON = [dict(x=None), dict(dt=3), dict(ld=999), dict(N=-1), dict(V=0), dict(V=(1 << 31) - 1, ld=1 << 31), dict(idt=2), dict(T=0.0), dict(T=float("nan")),
          dict(T=-1.0), dict(T=1e5), dict(stats=None)]


@pytest.mark.parametrize("kw", COMMON + [dict(k=-1), dict(k=257), dict(k=1001), dict(ent=None), dict(lse=None), dict(logp=None), dict(tids=None), dict(tlogp=None),
                                         dict(N=1 << 23), dict(N=(1 << 31) - 1, V=20000, ld=20000)])
def test_logprobs_refuses(kw):
    assert call("mh_token_logprobs", LP, LP, **kw) == -1


@pytest.mark.parametrize("kw", COMMON + [dict(d=None), dict(ldd=999), dict(ent=None), dict(ids=None), dict(N=1 << 23), dict(d=A, ldd=1001)])
def test_logprobs_bwd_refuses(kw):
    assert call("mh_token_logprobs_bwd", LPB, LPB, **kw) == -1


@pytest.mark.parametrize("kw", COMMON + [dict(K=0), dict(K=257), dict(ids=None), dict(tlp=None), dict(loss=None), dict(top=None), dict(ldi=4), dict(ldt=4), dict(N=1 << 23)])
def test_distill_refuses(kw):
    assert call("mh_distill_topk", DS, DS, **kw) == -1


@pytest.mark.parametrize("kw", COMMON + [dict(K=0), dict(K=257), dict(ids=None), dict(top=None), dict(d=None), dict(ldd=10), dict(ldi=4), dict(N=1 << 23), dict(ldd=1001)])
def test_distill_bwd_refuses(kw):
    assert call("mh_distill_topk_bwd", DSB, DSB, **kw) == -1


def test_workspaces():
    lib = _lib.load()
    need = lib.mh_token_logprobs_workspace_bytes(2, 100000, 5)
    assert need > 0 and lib.mh_token_logprobs_workspace_bytes(5000, 100000, 5) == 0
    for kw in (dict(nws=need - 1), dict(ws=None), dict(ws=A + 8)):
        assert call("mh_token_logprobs", LP, LP, **dict(dict(V=100000, ld=100000, nws=need), **kw)) == -4
    need = lib.mh_distill_topk_workspace_bytes(2, 100000, 1)
    assert need > 0 and lib.mh_distill_topk_workspace_bytes(5000, 100000, 1) == 0 < lib.mh_distill_topk_workspace_bytes(5000, 1000000, 1)
    for kw in (dict(nws=need - 1), dict(ws=None), dict(ws=A + 8)):
        assert call("mh_distill_topk", DS, DS, **dict(dict(V=100000, ld=100000, nws=need), **kw)) == -4


def test_no_rows_are_no_error():
    assert call("mh_token_logprobs", LP, LP, N=0, x=None) == 0 and call("mh_token_logprobs_bwd", LPB, LPB, N=0, x=None) == 0
    assert call("mh_distill_topk", DS, DS, N=0, x=None) == 0 and call("mh_distill_topk_bwd", DSB, DSB, N=0, x=None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 5)
    with pytest.raises(_lib.MerlinHipError):
        ops.token_logprobs(x)
    with pytest.raises(_lib.MerlinHipError):
        ops.distill_topk(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))


DST = dict(x=A, dt=0, ld=1000, N=2, V=1000, ids=A, idt=1, ldi=5, tlp=A, ldt=5, K=5, T=1.0, tail=1, w=A, loss=A, d=A, ldd=1000, ws=A, nws=1 << 20, stream=0)


@pytest.mark.parametrize("kw", COMMON[:-1] + [dict(K=0), dict(K=257), dict(ids=None), dict(tlp=None), dict(loss=None), dict(d=None), dict(ldi=4), dict(ldt=4), dict(ldd=999), dict(N=1 << 23), dict(ldd=1001)])
def test_distill_train_refuses(kw):
    assert call("mh_distill_topk_train", DST, DST, **kw) == -1


def test_distill_train_workspace():
    lib = _lib.load()
    assert lib.mh_distill_topk_train_workspace_bytes(4096, 32768, 64, 1, 1) == 0 == lib.mh_distill_topk_train_workspace_bytes(16, 1009, 5, 0, 0)
    need = lib.mh_distill_topk_train_workspace_bytes(2, 200000, 5, 0, 1)
    assert need > 0
    for kw in (dict(nws=need - 1), dict(ws=None), dict(ws=A + 8)):
        assert call("mh_distill_topk_train", DST, DST, **dict(dict(V=200000, ld=200000, ldd=200000, nws=need), **kw)) == -4
    assert call("mh_distill_topk_train", DST, DST, N=0, x=None) == 0
