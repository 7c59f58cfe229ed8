"""What the entry points of the 8-bit products refuse, on the host: every check comes before the first use of the device."""
import ctypes as C

import pytest
import torch

from models_amd import _lib, ops

P = C.c_void_p
A = 0x1000  # an address that is never used: the calls below end before a launch


def quantize(x=A, dtype=0, ldx=256, R=4, K=256, transpose=0, q=A, ldq=256, s=A, lds=4, colsum=None, ws=None, nws=0):
    return _lib.load().mh_fp8_quantize(P(x), dtype, ldx, R, K, transpose, P(q), ldq, P(s), lds, P(colsum), P(ws), nws, P(0))


def matmul(a=A, lda=256, sa=A, ldsa=4, b=A, ldb=256, sb=A, ldsb=4, M=4, N=8, K=256, bias=None, dt=0, out=A, ldo=8, ws=None, nws=0):
    return _lib.load().mh_fp8_matmul(P(a), lda, P(sa), ldsa, P(b), ldb, P(sb), ldsb, M, N, K, P(bias), dt, P(out), ldo, P(ws), nws, P(0))


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(ldx=255), dict(R=-1), dict(K=1 << 31), dict(x=None), dict(q=None), dict(s=None),
                                dict(ldq=128), dict(ldq=264), dict(q=A + 8), dict(lds=2), dict(lds=6), dict(s=A + 2), dict(colsum=A),
                                dict(transpose=1, R=300, ldq=256),
                                dict(R=1 << 27), dict(R=1 << 27, K=1024, ldx=1024, transpose=1, ldq=1 << 27, lds=1 << 20)])
def test_quantize_refuses(kw):
    assert quantize(**kw) == -1
    assert _lib.load().mh_last_error()


def both(x=A, dtype=0, ldx=256, R=4, K=256, q=A, ldq=256, s=A, lds=4, qt=A, ldqt=128, st=A, ldst=4, colsum=None, ws=None, nws=0):
    return _lib.load().mh_fp8_quantize_both(P(x), dtype, ldx, R, K, P(q), ldq, P(s), lds, P(qt), ldqt, P(st), ldst, P(colsum), P(ws), nws, P(0))


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(ldx=255), dict(R=-1), dict(x=None), dict(q=None), dict(s=None), dict(ldq=128), dict(q=A + 8), dict(lds=2),
                                dict(qt=None), dict(st=None), dict(ldqt=112), dict(qt=A + 8), dict(ldst=2), dict(st=A + 2)])
def test_quantize_both_refuses(kw):
    assert both(**kw) == -1
    assert _lib.load().mh_last_error()


def test_quantize_needs_its_workspace_for_column_sums():
    assert quantize(transpose=1, R=128, ldq=128, colsum=A) == -4
    assert quantize(transpose=1, R=128, ldq=128, colsum=A, ws=A, nws=256 * 4 - 1) == -4
    assert both(colsum=A) == -4 and both(colsum=A, ws=A, nws=256 * 4 - 1) == -4 and both(R=0) == 0 and both(K=0, ldx=0) == 0


@pytest.mark.parametrize("kw", [dict(a=None), dict(sb=None), dict(lda=240), dict(ldb=128), dict(ldsa=3), dict(dt=7), dict(ldo=7), dict(out=None), dict(K=0),
                                dict(M=-1), dict(b=A + 4), dict(ldsb=0), dict(M=1 << 27), dict(N=1 << 27, ldo=1 << 27), dict(M=1 << 26, N=1 << 20, ldo=1 << 20),
                                dict(K=1 << 24, lda=1 << 24, ldb=1 << 24, ldsa=1 << 17, ldsb=1 << 17), dict(lda=(1 << 24) + 16), dict(ldsa=(1 << 24) + 4),
                                dict(ldsb=1 << 30)])
def test_matmul_refuses(kw):
    assert matmul(**kw) == -1


def test_matmul_needs_its_workspace_where_the_sum_is_cut():
    need = _lib.load().mh_fp8_matmul_workspace_bytes(128, 128, 8192)
    assert need > 0
    assert matmul(M=128, N=128, K=8192, lda=8192, ldb=8192, ldsa=64, ldsb=64, ldo=128, ws=A, nws=need - 1) == -4
    assert matmul(M=128, N=128, K=8192, lda=8192, ldb=8192, ldsa=64, ldsb=64, ldo=128, ws=A + 8, nws=need + 8) == -4


def test_nothing_to_do_is_no_error():
    assert quantize(R=0) == 0 and quantize(K=0, ldx=0) == 0 and matmul(M=0) == 0 and matmul(N=0) == 0


def test_host_tensors_are_refused():
    with pytest.raises(_lib.MerlinHipError):
        ops.fp8_quantize(torch.zeros(4, 128))
    m = ops.Fp8Matrix(torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 4, dtype=torch.uint8), 128)
    with pytest.raises(_lib.MerlinHipError):
        ops.fp8_matmul(m, m)
