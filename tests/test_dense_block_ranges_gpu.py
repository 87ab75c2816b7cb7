"""adapter_add, kv_rope_append and paged_decode at the ends of their types' ranges and where a coarser intermediate would show,
against the formulas in 64 bits (bounds: tests/dense_block.py)."""
import math

import pytest
import torch

from tests.dense_block import F32, adapters64, half_step
from tests.test_dense_block_gpu import randn, status_is_clean  # noqa: F401  (the fixture)
from wsvd_b200 import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------------ adapters: the sums x A

def _adapters(y, x, a, b, adapter, scale=None, cu=None):
    """ops.adapter_add of CPU tensors, back on the CPU."""
    got = ops.adapter_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), torch.tensor(adapter, dtype=torch.int32).cuda(),
                          scale=None if scale is None else scale.cuda(), cu_new=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda())
    return got.cpu()


def _rows(cu, rows):
    return dict(cu=cu, adapter=[0] * (len(cu) - 1)) if cu else dict(adapter=[0] * rows)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("n_in", [4096, 4093])  # the second one off 16 bytes, on the kernels for any shape
def test_a_sum_beyond_f16_is_not_infinite(packed, n_in):
    """x A = 131072 (f16 ends at 65504), the adapter's share 0.001 131072 0.25 16 = 524."""
    rows, r, n_out = 70, 16, 72
    x, a = torch.full((rows, n_in), 64.0, dtype=F16), torch.full((1, n_in, r), 0.5, dtype=F16)
    b, y = torch.full((1, r, n_out), 0.25, dtype=F16), randn(torch.Generator().manual_seed(1), rows, n_out)
    b[0, :, 1] = 0  # an infinite sum would make this column NaN
    scale = torch.tensor([0.001])
    how = _rows([0, 3, rows], rows) if packed else _rows(None, rows)
    want, bound, _ = adapters64(y, x, a, b, torch.tensor(how["adapter"]), scale, how.get("cu"))
    got = _adapters(y, x, a, b, scale=scale, **how)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max().item()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("r", [8, 48, 64, 128, 200])
@pytest.mark.parametrize("x_size,a_size,b_size,scale", [(300.0, 300.0, 1e-4, 0.05), (2e-4, 2e-4, 400.0, 3000.0), (1.0, 1e-3, 1.0, 1.0)])
def test_sums_of_any_size(packed, dtype, r, x_size, a_size, b_size, scale):
    """Sums of some 6e6, 3e-7 and 0.03 where the adapter's share is of the order of one to a hundred; a row among them whose sums are
    2^12 times smaller than the others', and one of zeros."""
    g = torch.Generator().manual_seed(r)
    rows, n_in, n_out = 75, 4096, 64
    x, a = randn(g, rows, n_in, scale=x_size, dtype=dtype), randn(g, 2, n_in, r, scale=a_size, dtype=dtype)
    b, y = randn(g, 2, r, n_out, scale=b_size, dtype=dtype), randn(g, rows, n_out, scale=0.01, dtype=dtype)
    x[5] *= 2.0 ** -12
    x[6] = 0
    how = dict(cu=[0, 71, rows], adapter=[1, 0]) if packed else dict(adapter=[1] * 71 + [0] * (rows - 71))
    s = torch.full((2,), scale)
    want, bound, _ = adapters64(y, x, a, b, torch.tensor(how["adapter"]), s, how.get("cu"))
    assert torch.isfinite(want).all() and (want.abs() < 60000).all()
    got = _adapters(y, x, a, b, scale=s, **how)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max().item()
    assert torch.equal(got[6], y[6])


@pytest.mark.parametrize("packed", [False, True])
def test_a_rank_with_an_infinite_sum_leaves_the_others_their_range(packed):
    """Sums inf in one rank and 131072 in the others, whose products have the other sign: the results are infinite, not NaN."""
    rows, n_in, n_out, r = 66, 512, 64, 16
    x, a = torch.full((rows, n_in), 64.0, dtype=F16), torch.full((1, n_in, r), 4.0, dtype=F16)
    a[0, 7, 0] = float("inf")
    b = torch.full((1, r, n_out), -1e-4, dtype=F16)
    b[0, 0] = 1e-4
    how = _rows([0, 60, rows], rows) if packed else _rows(None, rows)
    got = _adapters(randn(torch.Generator().manual_seed(3), rows, n_out), x, a, b, **how)
    assert (got == float("inf")).all()


@pytest.mark.parametrize("n_in,n_out", [(64, 64), (61, 60)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_sums_of_single_rows_are_f32(dtype, n_in, n_out):
    """y cancels the adapter's share but for its own rounding: the bound has no rounding of x A to 16 bits (planted
    here in the oracle, it is beyond the bound)."""
    g = torch.Generator().manual_seed(8)
    rows, r = 9, 16
    x, a = randn(g, rows, n_in, dtype=dtype), randn(g, 2, n_in, r, scale=1 / math.sqrt(n_in), dtype=dtype)
    b = randn(g, 2, r, n_out, dtype=dtype)
    ad = [0, 1, 1, 0, 1, 1, 1, 0, 1]
    h = torch.stack([x[i].double() @ a[ad[i]].double() for i in range(rows)])
    share = torch.stack([h[i] @ b[ad[i]].double() for i in range(rows)])
    y = (-share).to(dtype)
    want = y.double() + share
    habs = torch.stack([x[i].double().abs() @ a[ad[i]].double().abs() for i in range(rows)])
    weight = torch.stack([habs[i] @ b[ad[i]].double().abs() for i in range(rows)])
    bound = half_step(dtype) * want.abs() + (n_in + r + 8) * F32 * weight + 2 * F32 * y.double().abs() + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    rounded = torch.stack([h[i].to(dtype).double() @ b[ad[i]].double() for i in range(rows)])
    assert ((y.double() + rounded - want).abs() > bound).double().mean() > 0.2  # the bound tells a 16-bit x A apart
    got = _adapters(y, x, a, b, ad)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max().item()
