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


def crowded_rows(V, k, dtype, rng):
    """Rows of which far more than the k largest entries come close to the k-th, or are equal to it."""
    low = float(torch.finfo(TYPES[dtype]).min)
    mask = -1e9 if dtype != "f16" else -6e4
    base = rng.normal(size=V)
    rows = [np.full(V, 0.5), np.full(V, low), 300.0 + base, -3000.0 + base, np.round(base), np.round(300 + base), np.sort(base), np.sort(base)[::-1]]
    for few in (1, k - 1, k, k + 3):  # a constant mask, and fewer, as many or a few more entries than asked for beside it
        a = np.full(V, mask)
        a[rng.choice(V, few, replace=False)] = rng.normal(size=few)
        rows.append(a)
    a = np.where(np.arange(V) < V // 2, mask, base)  # a part of the row masked throughout
    rows.append(a)
    a = np.full(V, mask)
    a[V - 5000 if V > 5000 else V // 2:] = mask / 2  # two constants, the larger one behind
    a[V - 1] = 1.0
    rows.append(a)
    a = np.full(V, -np.inf)
    a[V // 3:] = 2.0
    rows.append(a)
    for ve in (4, 8):  # what one in two threads reads is large, for 256 and 512 threads
        for nt in (256, 512):
            a = base.copy()
            some = (np.arange(V) // ve) % nt < min(k, nt) - 1
            a[some] = 100 + rng.normal(size=some.sum())
            rows.append(a)
    return np.stack(rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,k", [(3001, 20), (4096, 256), (9000, 7), (16384, 256), (40003, 100), (131072, 20)])
def test_alternatives_of_crowded_rows(device, dtype, V, k):
    rows = crowded_rows(V, k, dtype, np.random.default_rng(V + k))
    if V > 100000:  # the copies' logits in 32 bits stay under a gigabyte
        rows = rows[:: 2]
    check(rows, dtype, k, device)
