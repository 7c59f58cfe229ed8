"""Which gradients of the catalogue softmax lie where they may, on the host: every check comes before the first use of the device."""
import pytest

from models_amd import _lib
from tests.test_token_softmax_abi import A, DSB, DST, LPB, call


SHIFTS = [dict(d=A + 4), dict(d=A - 4), dict(d=A + 3996), dict(d=A + 4000), dict(d=A - 4000), dict(d=A + 2, dt=1), dict(N=1, d=A + 3996), dict(N=1, d=A - 3996),
          dict(d=A + 4, ld=2000, ldd=1500), dict(ld=2000, ldd=2000, d=A + 3996), dict(ld=2000, ldd=2000, d=A + 4004), dict(ld=2000, ldd=2000, d=A - 8000 + 8)]


@pytest.mark.parametrize("kw", SHIFTS)
def test_a_gradient_that_overlaps_the_logits_elsewhere_is_refused(kw):
    assert call("mh_token_logprobs_bwd", LPB, LPB, **kw) == -1
    assert call("mh_distill_topk_bwd", DSB, DSB, **kw) == -1
    assert call("mh_distill_topk_train", DST, DST, **kw) == -1
    assert b"overlaps" in _lib.load().mh_last_error()


@pytest.mark.parametrize("kw", [dict(d=A), dict(d=A + 800000, ld=400000, ldd=400000), dict(d=A - 800000, ld=400000, ldd=400000), dict(d=A + 1600000),
                                dict(d=A - 1600000), dict(d=A + 1600000, ldd=200001), dict(d=A + 800000, N=1)])
def test_a_gradient_in_place_or_apart_is_not(kw):
    """Other columns of one buffer, the memory before and behind: the next check, of the workspace, is what ends these calls."""
    big = dict(V=200000, ld=200000, ldd=200000, ws=None, nws=0)
    assert call("mh_distill_topk_train", DST, DST, **dict(big, **kw)) == -4
