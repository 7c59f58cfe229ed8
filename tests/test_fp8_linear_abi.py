"""What mh_fp8_linear refuses, on the host: every check comes before the first use of the device."""
import pytest

from models_amd import _lib
from tests.test_fp8_abi import A, P


def linear(x=A, xdt=0, ldx=256, w=2 * A, ldw=256, sw=3 * A, ldsw=4, M=4, N=256, K=256, bias=None, dt=0, out=16 * A, ldo=256, ws=None, nws=0):
    return _lib.load().mh_fp8_linear(P(x), xdt, ldx, P(w), ldw, P(sw), ldsw, M, N, K, P(bias), dt, P(out), ldo, P(ws), nws, P(0))


@pytest.mark.parametrize("kw", [dict(x=None), dict(xdt=3), dict(ldx=255), dict(w=None), dict(sw=None), dict(ldw=128), dict(ldw=264), dict(w=A + 8), dict(ldsw=2),
                                dict(sw=A + 2), dict(M=-1), dict(K=0), dict(dt=5), dict(out=None), dict(ldo=255), dict(ldw=(1 << 24) + 16)])
def test_linear_refuses(kw):
    assert linear(**kw) == -1


@pytest.mark.parametrize("kw", [dict(out=A), dict(out=A, M=1), dict(out=A + 1020, M=1), dict(out=A + 1024), dict(out=A - 4), dict(out=A, M=16), dict(out=A, dt=1),
                                dict(out=A + 512, ldx=400, ldo=400)])
def test_few_rows_are_not_written_over_what_they_are_made_of(kw):
    assert linear(**kw) == -1 and b"overlaps" in _lib.load().mh_last_error()


def test_more_rows_need_their_workspace():
    need = _lib.load().mh_fp8_linear_workspace_bytes(17, 256, 256)
    assert need > 0 == _lib.load().mh_fp8_linear_workspace_bytes(16, 256, 256)
    for kw in (dict(ws=None, nws=need), dict(ws=A, nws=need - 1), dict(ws=A + 8, nws=need)):
        assert linear(M=17, out=A, **kw) == -4
