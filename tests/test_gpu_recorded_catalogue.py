"""Calls of the catalogue softmax and the 8-bit products that need workspaces, in a recorded step: what the step allocated stays its own, whatever the
program allocates and frees between the replays."""
import numpy as np
import pytest
import torch

from models_amd import ops
from models_amd.graph import RecordedStep
from tests.test_gpu_token_softmax import teacher

pytestmark = pytest.mark.gpu


def test_steps_with_workspaces(device):
    rng = np.random.default_rng(5)
    N, V, K, M, E, F = 3, 70001, 9, 40, 4096, 300  # rows cut into parts, a sum cut into slices, more than 16 rows
    ids, (tid, tlp) = torch.tensor(rng.integers(0, V, N), device=device), teacher(rng, N, V, K, device)
    g = torch.Generator(device=device).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    kernel = rand(E, F)
    w8, kernel8 = ops.fp8_quantize(kernel, transpose=True), ops.fp8_quantize(kernel)
    ones = torch.ones(N, device=device)

    def step(b):
        x, q, dy = b["x"], b["q"], b["dy"]
        r = ops.token_logprobs(x, ids, k=7)
        d = ops.token_logprobs_backward(x, ids, r, ones, ones)
        s, e = ops.distill_topk_train(x, tid, tlp, ones, 1.0, True)
        y = ops.fp8_linear(q, w8)
        z = ops.fp8_linear(b["many"], w8, out_dtype=torch.bfloat16)
        dx, dw, db = ops.fp8_linear_backward(q, kernel8, dy, need_db=True)
        return [r.logp, r.entropy, r.lse, r.top_logp, r.top_ids, d, s.loss, e, y, z, dx, dw, db]

    batches = [{"x": rand(N, V), "q": rand(M, E), "dy": rand(M, F), "many": rand(200, E)} for _ in range(3)]
    assert ops._lib.load().mh_fp8_linear_workspace_bytes(200, F, E) > 0
    rec = RecordedStep(step, batches[0])
    for i in (1, 2, 0, 1):
        waste = [torch.full((n,), float("nan"), device=device) for n in (N * V, 1 << 14, 1 << 18, 1 << 20, 200 * E)]
        del waste  # blocks that the recorded calls' workspaces would have been, had they been given back
        got = [t.clone() for t in rec.replay(batches[i])]
        torch.cuda.synchronize()
        want = step(batches[i])
        for a, b in zip(got, want):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
