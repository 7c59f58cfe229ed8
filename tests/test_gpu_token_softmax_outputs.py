"""Where a gradient may be written: in place of the logits or apart from them, other columns of the same buffer included."""
import pytest
import torch

from models_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,V", [(3, 1009), (70, 6000), (1, 50000), (1030, 16500)])
def test_gradients_beside_their_logits(device, N, V):
    g = torch.Generator(device=device).manual_seed(V)
    both = torch.randn(N, 2 * V + 3, generator=g, device=device)
    x, out = both[:, 1:V + 1], both[:, V + 2:2 * V + 2]
    edge = both[:, [0, V + 1, 2 * V + 2]].clone()
    ids = torch.randint(0, V, (N,), generator=g, device=device)
    tid = torch.randint(0, V, (N, 5), generator=g, device=device)
    tlp = torch.log_softmax(torch.randn(N, 6, generator=g, device=device), 1)[:, :5]
    w = torch.ones(N, device=device)
    same = x.contiguous()
    r, s = ops.token_logprobs(x, ids), ops.distill_topk(x, tid, tlp)
    calls = [lambda y, o: ops.token_logprobs_backward(y, ids, r, w, w, w, out=o), lambda y, o: ops.distill_topk_backward(y, tid, s, w, out=o),
             lambda y, o: ops.distill_topk_train(y, tid, tlp, w, out=o)[1]]
    for call in calls:
        want = call(same, None)
        assert torch.equal(call(x, out), want) and torch.equal(x, same) and torch.equal(both[:, [0, V + 1, 2 * V + 2]], edge)
        place = both.clone()
        assert torch.equal(call(place[:, 1:V + 1], place[:, 1:V + 1]), want)


def test_overlapping_gradients_are_refused(device):
    x = torch.zeros(40, 100, device=device)
    ids, w = torch.zeros(40, dtype=torch.int64, device=device), torch.ones(40, device=device)
    tid, tlp = ids[:, None].contiguous(), torch.zeros(40, 1, device=device)
    y = x[:20, :60]
    r, s = ops.token_logprobs(y, ids[:20]), ops.distill_topk(y, tid[:20], tlp[:20])
    flat = x.view(-1)
    for out in (x[:20, 1:61], x[:20, 40:], x[1:21, :60], x[19:39, 30:90], flat[1:1201].view(20, 60), flat[600:600 + 1200].view(20, 60)):
        for call in (lambda: ops.token_logprobs_backward(y, ids[:20], r, w[:20], out=out), lambda: ops.distill_topk_backward(y, tid[:20], s, out=out),
                     lambda: ops.distill_topk_train(y, tid[:20], tlp[:20], out=out)):
            with pytest.raises(ValueError):
                call()
    for out in (x[20:, :60], x[20:, 40:], flat[2000:3200].view(20, 60)):
        assert ops.token_logprobs_backward(y, ids[:20], r, w[:20], out=out).data_ptr() == out.data_ptr()
