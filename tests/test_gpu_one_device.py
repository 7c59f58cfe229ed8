"""Every tensor of a call has to lie where the first one does: each argument in turn claims to lie on another device."""
import pytest
import torch

from models_amd import ops

pytestmark = pytest.mark.gpu


class Elsewhere(torch.Tensor):
    def get_device(self):
        return 7


def away(t):
    return t.as_subclass(Elsewhere)


def test_arguments_on_another_device_are_refused(device):
    f = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    x, ids, w = f(4, 200), torch.zeros(4, dtype=torch.int64, device=device), torch.ones(4, device=device)
    tid, tlp = torch.zeros(4, 3, dtype=torch.int64, device=device), f(4, 3) - 2
    r, s = ops.token_logprobs(x, ids), ops.distill_topk(x, tid, tlp)
    a, b, kernel, dy = ops.fp8_quantize(f(20, 200)), ops.fp8_quantize(f(8, 200)), ops.fp8_quantize(f(200, 8)), f(20, 8)
    y, bias, out, big = f(20, 200), f(8), f(20, 8), f(4, 200)
    calls = {
        "token_logprobs ids": lambda: ops.token_logprobs(x, away(ids)),
        "token_logprobs_backward ids": lambda: ops.token_logprobs_backward(x, away(ids), r, w),
        "token_logprobs_backward dlogp": lambda: ops.token_logprobs_backward(x, ids, r, away(w)),
        "token_logprobs_backward dentropy": lambda: ops.token_logprobs_backward(x, ids, r, None, away(w)),
        "token_logprobs_backward dlse": lambda: ops.token_logprobs_backward(x, ids, r, None, None, away(w)),
        "token_logprobs_backward stats": lambda: ops.token_logprobs_backward(x, ids, r._replace(stats=away(r.stats)), w),
        "token_logprobs_backward entropy": lambda: ops.token_logprobs_backward(x, ids, r._replace(entropy=away(r.entropy)), w, w),
        "token_logprobs_backward out": lambda: ops.token_logprobs_backward(x, ids, r, w, out=away(big)),
        "distill_topk ids": lambda: ops.distill_topk(x, away(tid), tlp),
        "distill_topk logp": lambda: ops.distill_topk(x, tid, away(tlp)),
        "distill_topk_backward ids": lambda: ops.distill_topk_backward(x, away(tid), s),
        "distill_topk_backward stats": lambda: ops.distill_topk_backward(x, tid, s._replace(stats=away(s.stats))),
        "distill_topk_backward top_grad": lambda: ops.distill_topk_backward(x, tid, s._replace(top_grad=away(s.top_grad))),
        "distill_topk_backward dloss": lambda: ops.distill_topk_backward(x, tid, s, away(w)),
        "distill_topk_backward out": lambda: ops.distill_topk_backward(x, tid, s, out=away(big)),
        "distill_topk_train ids": lambda: ops.distill_topk_train(x, away(tid), tlp),
        "distill_topk_train logp": lambda: ops.distill_topk_train(x, tid, away(tlp)),
        "distill_topk_train dloss": lambda: ops.distill_topk_train(x, tid, tlp, away(w)),
        "distill_topk_train out": lambda: ops.distill_topk_train(x, tid, tlp, out=away(big)),
        "fp8_matmul a scales": lambda: ops.fp8_matmul(a._replace(scales=away(a.scales)), b),
        "fp8_matmul b": lambda: ops.fp8_matmul(a, b._replace(values=away(b.values), scales=away(b.scales))),
        "fp8_matmul b scales": lambda: ops.fp8_matmul(a, b._replace(scales=away(b.scales))),
        "fp8_matmul bias": lambda: ops.fp8_matmul(a, b, away(bias)),
        "fp8_matmul out": lambda: ops.fp8_matmul(a, b, out=away(out)),
        "fp8_linear w": lambda: ops.fp8_linear(y, b._replace(values=away(b.values), scales=away(b.scales))),
        "fp8_linear bias": lambda: ops.fp8_linear(y, b, away(bias)),
        "fp8_linear out": lambda: ops.fp8_linear(y, b, out=away(out)),
        "fp8_linear_backward w": lambda: ops.fp8_linear_backward(y, kernel._replace(values=away(kernel.values), scales=away(kernel.scales)), dy),
        "fp8_linear_backward dy": lambda: ops.fp8_linear_backward(y, kernel, away(dy)),
    }
    allowed = []
    for name, call in calls.items():
        try:
            call()
            allowed.append(name)
        except ValueError:
            pass
    assert not allowed
