"""Where the 8-bit layer may write: over its input, beside it, and not over its weights."""
import pytest
import torch

from models_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 5, 16, 17, 100, 700])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_over_its_input(device, M, dt):
    g = torch.Generator(device=device).manual_seed(M)
    K = 2048
    w8 = ops.fp8_quantize(torch.randn(K, K, generator=g, device=device))
    buf = torch.randn(M, 2 * K, generator=g, device=device).to(dt)
    want = ops.fp8_linear(buf[:, :K], w8, out_dtype=dt)
    for cols in (slice(0, K), slice(8, K + 8), slice(K, 2 * K)):  # in place, over a part, beside
        y = buf.clone()
        assert torch.equal(ops.fp8_linear(y[:, :K], w8, out_dtype=dt, out=y[:, cols]), want)
        assert torch.equal(y[:, cols.stop:], buf[:, cols.stop:]) and torch.equal(y[:, : cols.start], buf[:, : cols.start])


def test_over_its_weights_is_refused(device):
    w = torch.zeros(128 * 128, device=device)
    values = w.view(torch.uint8)[: 128 * 128].view(torch.float8_e4m3fn).view(128, 128)
    w8 = ops.Fp8Matrix(values, torch.full((128, 4), 127, dtype=torch.uint8, device=device), 128)
    x = torch.ones(20, 128, device=device)
    x8 = ops.fp8_quantize(x)
    bias = torch.zeros(128, device=device)
    over, room = w.view(128, 128)[:20], w.view(128, 128)[40:60]
    for bad in (lambda: ops.fp8_linear(x, w8, out=over), lambda: ops.fp8_matmul(x8, w8, out=over), lambda: ops.fp8_matmul(w8, x8, out=w[:2560].view(128, 20)),
                lambda: ops.fp8_linear(x[:1], w8, bias, out=bias.view(1, 128))):
        with pytest.raises(ValueError):
            bad()
    assert (ops.fp8_linear(x, w8, out=room) == 0).all()
