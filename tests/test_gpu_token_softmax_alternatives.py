"""The alternatives of rows where finding them is least regular.  Tolerances are those of test_gpu_token_softmax; the ids are equal."""
import numpy as np
import pytest
import torch

from models_amd import ops
from tests.test_gpu_token_softmax import TYPES, check_logprobs

pytestmark = pytest.mark.gpu


NAN = {"f32": (torch.int32, 0x7FC00000), "bf16": (torch.int16, 0x7FC0), "f16": (torch.int16, 0x7E00)}


def check(rows, dtype, k, device, T=1.0):
    """The rows themselves (few: a long row is cut into parts), and enough copies of them for a workgroup a row: the same alternatives."""
    x = torch.tensor(rows, dtype=torch.float32).to(TYPES[dtype])
    word, bits = NAN[dtype]  # a conversion need not keep the sign of a NaN
    x = torch.where(torch.tensor(np.isnan(rows) & ~np.signbit(rows)), torch.tensor(bits, dtype=word), x.view(word)).view(TYPES[dtype]).to(device)
    r, *_ = check_logprobs(x, None, k, T)
    rep = -(-1030 // len(rows))
    many = ops.token_logprobs(x.repeat(rep, 1), None, k=k, temperature=T)
    assert torch.equal(many.top_ids, r.top_ids.repeat(rep, 1))


def nan_rows(V, rng):
    """Rows that hold NaN over whole 16-byte vectors (4 entries of 32 bits, 8 of 16) and over whole 128 bytes, of both signs."""
    base = rng.normal(size=V)
    rows = []
    for sign in (1.0, -1.0):
        nan = np.copysign(np.nan, sign)
        for at, n in ((0, 4), (0, 8), (8, 8), (0, 32), (32, 64), (V - V % 64 - 64, 64), (V // 2, V), (0, V // 2), (3, 9)):
            a = base.copy()
            a[max(at, 0):at + n] = nan
            rows.append(a)
        a = base.copy()
        a[(np.arange(V) // 64) % 2 == 0] = nan  # every other 128 bytes and more
        rows.append(a)
        a = np.full(V, nan)
        a[[V // 7, V // 3, V - 1]] = [0.5, -2.0, 0.25]
        rows.append(a)
        a = np.where(np.arange(V) < V // 2, nan, -np.inf)
        a[V - 2] = 1.0
        rows.append(a)
    return np.stack(rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,k", [(96, 1), (3000, 3), (5000, 20), (20011, 256), (40000, 1), (70001, 33)])
def test_alternatives_beside_runs_of_nan(device, dtype, V, k):
    check(nan_rows(V, np.random.default_rng(V)), dtype, k, device)
