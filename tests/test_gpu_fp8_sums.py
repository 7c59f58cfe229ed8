"""What the sums of the 8-bit products are worth where their terms cancel: 32-bit sums are off by K 2^-24 of sum |a b| and a rounding of the result;
bf16 outputs of more than 16 rows come from the 8-bit instruction and are off by up to 7 2^-13 of sum |a b| besides (test_gpu_fp8 derives both)."""
import numpy as np
import pytest
import torch

from models_amd import ops
from tests.test_gpu_fp8 import HALF, TYPES, f64, quantized

pytestmark = pytest.mark.gpu


def cancelling(rng, M, N, K, device):
    """Of every sixteen products the first, 1, is taken back by the ninth; what is left are seven between 2^-14 and 2^-13 beside the first."""
    k = np.arange(K) % 16
    a, b = (np.where((k == 0) | (k == 8), 1.0, np.where(k < 8, 2.0 ** rng.uniform(-7, -6.5, size=(R, K)), 0.0)) for R in (M, N))
    b = np.where(k == 8, -b, b)
    t = lambda v: torch.tensor(v, dtype=torch.float32, device=device)  # noqa: E731
    return t(a * 2.0 ** rng.integers(-9, 9, size=(M, 1))), t(b * 2.0 ** rng.integers(-9, 9, size=(N, 1)))


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 300, 256), (7, 130, 1024), (16, 4097, 1000), (16, 70, 128), (17, 300, 1024), (48, 1000, 4096), (64, 130, 640),
                                   (129, 257, 520), (300, 515, 8192)])
def test_sums_that_cancel(device, M, N, K, out):
    x, w = cancelling(np.random.default_rng(M + N), M, N, K, device)
    x8, w8 = ops.fp8_quantize(x), ops.fp8_quantize(w)
    a, b = quantized(f64(x))[0], quantized(f64(w))[0]
    ref, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    tight = lambda t: (K + 1) * 2.0 ** -24 * mag + HALF[t] * np.abs(ref) + (2.0 ** -25 if t == "f16" else 0.0)  # noqa: E731
    for y in (ops.fp8_matmul(x8, w8, out_dtype=TYPES[out]), ops.fp8_linear(x, w8, out_dtype=TYPES[out])):
        y = f64(y)
        if out == "f16":  # a last first product that no ninth takes back is up to 2^16, and fp16 ends at 65504
            beyond = np.abs(ref) >= 65520.0
            assert (y[beyond] == np.sign(ref[beyond]) * np.inf).all()
            y = np.where(beyond, ref, y)
        err = np.abs(y - ref)
        assert (err <= tight(out) + (7 * 2.0 ** -13 * mag if out == "bf16" and M > 16 else 0.0)).all(), (err - tight(out)).max()
    if out == "bf16":  # a 32-bit output rounded afterwards has no more than the rounding
        y = ops.fp8_linear(x, w8).to(torch.bfloat16)
        assert (np.abs(f64(y) - ref) <= tight("bf16") + 2.0 ** -8 * (K + 1) * 2.0 ** -24 * mag).all()
