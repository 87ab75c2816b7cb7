"""adapter_add, kv_rope_append and paged_decode at the ends of their types' ranges and where a coarser intermediate would show,
against the formulas in 64 bits (bounds: tests/dense_block.py)."""
import math

import pytest
import torch

from tests.dense_block import F32, adapters64, attend64, half_step, pages, quantize, state
from tests.test_dense_block_gpu import gpu, randn, status_is_clean  # noqa: F401  (the fixture)
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


# ------------------------------------------------------------------ attention: bf16 queries on bytes

def _coarse(q):
    """Rows of q (f64) as 16-bit whole numbers of steps below the power of two of their largest."""
    step = 2.0 ** (torch.floor(torch.log2(q.abs().amax(-1, keepdim=True))) - 14)
    return (q / step).round() * step


def _long_bytes(g, lens, H, K, D, outlier, dtype=BF16):
    """Queries [B, H, D] (outlier: the size of one value of each row, whose keys are 0), keys of which one is along the mean of its
    queries, so that it has nearly all the weight; (q, state, k, v, ks, vs)."""
    table, T = pages(len(lens), max(lens), 16, g)
    st = state(lens, table)
    q = torch.randn(len(lens), H, D, generator=g)
    k, v = torch.randn(T, K, D, generator=g), torch.randn(T, K, D, generator=g)
    for b, n in enumerate(lens):
        heads = q[b].view(K, H // K, D)
        k[int(table[b, n // 3])] = 3.0 * heads.mean(1) * (H // K) ** 0.5
    if outlier:
        q[..., 5] = outlier
        k[..., 5] = 0
    (k, ks), (v, vs) = quantize(k.double()), quantize(v.double())
    return q.to(dtype), st, k, v, ks, vs


def _check_long_bytes(q, st, k, v, ks, vs):
    want, lse, bound, lse_bound = attend64(q, st, k, v, ks, vs, 0, 0.0)
    # a weight in f16 (two terms, lifted by 2^7): the last step of f16 is 2^-24, so it is off by up to 2^-25 2^-7 of the largest weight,
    # where its own bits end.  Next to a weight of one that meets a value of zero, the others of 2^-36 each are below that.
    values = (v.double() * vs.double()[..., None]).abs().max()
    bound = bound + st.b_seq_len.double()[:, None, None] * 2.0 ** -32 * values
    got, got_lse = ops.paged_decode(q.cuda(), gpu(st), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), return_lse=True)
    off, off_lse = (got.cpu().double() - want).abs() - bound, (got_lse.cpu().double() - lse).abs() - lse_bound
    assert (off_lse <= 0).all(), off_lse.max().item()
    assert (off <= 0).all(), off.max().item()
    return lse, lse_bound


@pytest.mark.parametrize("H,K,D", [(8, 2, 128), (8, 1, 128), (16, 1, 128), (4, 4, 64), (8, 2, 256), (6, 2, 96)])
@pytest.mark.parametrize("outlier", [24.0, 192.0])
def test_bf16_queries_with_an_outlier_keep_the_scores_of_bytes(H, K, D, outlier):
    """One value that is large against the others': at 16 bits below it the others' scores would be lost."""
    g = torch.Generator().manual_seed(H + D)
    case = _long_bytes(g, [511, 512, 513, 3001], H, K, D, outlier)
    q, st = case[:2]
    lse, lse_bound = _check_long_bytes(*case)
    if outlier > 100:  # planted in the oracle, a query of 16 bits is beyond the bound
        planted = attend64(_coarse(q.double()), st, *case[2:], 0, 0.0)[1]
        assert ((planted - lse).abs() > lse_bound).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D", [(8, 2, 128), (8, 1, 64), (16, 1, 128), (4, 1, 256)])
def test_queries_on_bytes_of_long_sequences(dtype, H, K, D):
    g = torch.Generator().manual_seed(H * D)
    _check_long_bytes(*_long_bytes(g, [513, 5000, 700], H, K, D, 0.0, dtype))


def test_an_outlier_in_one_head_of_a_group():
    g = torch.Generator().manual_seed(12)
    q, st, k, v, ks, vs = _long_bytes(g, [1500], 4, 1, 128, 0.0)
    q[0, 2, 5] = 200.0
    k[..., 5] = 0
    _check_long_bytes(q, st, k, v, ks, vs)


# ------------------------------------------------------------------ append: bytes of values between two steps

def _between_steps(dtype, D):
    """Rows [n, D] of values whose quotient by the row's scale and whose product with 1 / scale round to different steps."""
    found = []
    ones = torch.arange(128 if dtype is BF16 else 1024, dtype=torch.float32) / (128 if dtype is BF16 else 1024) + 1
    for amax in ones.tolist():
        scale = (torch.tensor(amax) / 127).half().float()
        x = torch.cat([ones * 2.0 ** -e for e in range(1, 8)])
        x = x[(x.to(dtype).float() == x) & (x <= amax)]
        apart = x[(x / scale).round() != (x * (1 / scale)).round()]
        if len(apart):
            row = torch.full((D,), amax)
            row[1:] = apart[torch.arange(D - 1) % len(apart)] * torch.where(torch.arange(D - 1) % 3 == 0, -1.0, 1.0)
            found.append(row)
    return torch.stack(found).to(dtype) if found else torch.zeros(0, D, dtype=dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [128, 40])  # the second one on the kernel for any shape
@pytest.mark.parametrize("many", [False, True])
def test_bytes_are_those_of_the_quotient(dtype, D, many):
    """int8 rows are round(x / scale), as latent_quant_append stores them: equal, also between two steps."""
    rows = _between_steps(dtype, D)
    assert (len(rows) > 3) == (dtype is F16)  # (8 bits of bf16 meet no such scale)
    n = 30000 if many and D == 128 else 300
    rows = torch.cat([rows, randn(torch.Generator().manual_seed(D), 61, D, dtype=dtype)])
    rows = rows.repeat(n // len(rows) + 1, 1)[:n]
    kv = torch.stack([rows, rows.flip(0)], 1).cuda()  # [n, 2, D]
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int()[None].contiguous()
    st = gpu(state([0], table))
    caches = [torch.zeros(n, 2, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(n, 2, dtype=torch.float16, device="cuda") for _ in range(2)]
    ops.kv_rope_append(kv, kv, st, *caches, torch.zeros(0, device="cuda"), cache_k_scale=scales[0], cache_v_scale=scales[1],
                       cu_new=torch.tensor([0, n], dtype=torch.int32).cuda())
    x = kv.cpu().float()
    scale = (x.abs().amax(-1) / 127).half()
    want = (x / scale.float()[..., None]).round().clamp(-128, 127).to(torch.int8)
    at = table[0].long()
    for cache, held in zip(caches, scales):
        assert torch.equal(held.cpu()[at], scale)
        assert torch.equal(cache.cpu()[at], want)


# ------------------------------------------------------------------ attention: values as large as their type's

@pytest.mark.parametrize("D", [128, 40])
@pytest.mark.parametrize("largest", [3e38, 1.0])
def test_bf16_values_at_the_end_of_their_range(D, largest):
    """Scores that grow by e^5.4 inside a share (four tiles of 64 tokens), less than what makes the kernel take a new reference for the
    weights; one token has a value, so that the result is its weight times it, below f32's end."""
    n = 128 * 256
    q, k, v = torch.zeros(1, 1, D, dtype=BF16), torch.zeros(n, 1, D, dtype=BF16), torch.zeros(n, 1, D, dtype=BF16)
    q[..., 0] = 1
    k[torch.arange(n) % 256 >= 64, 0, 0] = 5.4
    v[200] = largest
    st = state([n], torch.arange(n, dtype=torch.int32)[None].contiguous())
    want, lse, bound, lse_bound = attend64(q, st, k, v, None, None, 0, 1.0)
    got, got_lse = ops.paged_decode(q.cuda(), gpu(st), k.cuda(), v.cuda(), sm_scale=1.0, return_lse=True)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert ((got_lse.cpu().double() - lse).abs() <= lse_bound).all()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("n_in", [512, 509])
@pytest.mark.parametrize("x_size,scale", [(1e33, 1e-33), (1e-33, 1e33)])
def test_bf16_sums_whose_products_pass_f32(packed, n_in, x_size, scale):
    """Sums of some 1e33, whose products with 1e6 are beyond f32 before the adapter's scale brings them back; and small ones."""
    g = torch.Generator().manual_seed(9)
    rows, r, n_out = 70, 16, 64
    x, a = randn(g, rows, n_in, scale=x_size, dtype=BF16), randn(g, 1, n_in, r, scale=n_in ** -0.5, dtype=BF16)
    b = randn(g, 1, r, n_out, scale=1e6 if scale < 1 else 1e-6, dtype=BF16)
    y, s = randn(g, rows, n_out, dtype=BF16), torch.tensor([scale])
    how = _rows([0, 66, rows], rows) if packed else _rows(None, rows)
    want, bound, _ = adapters64(y, x, a, b, torch.tensor(how["adapter"]), s, how.get("cu"))
    got = _adapters(y, x, a, b, scale=s, **how)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max().item()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [128, 40])
def test_bytes_at_the_ends_of_the_scale(dtype, D):
    """Rows whose scale is among f16's subnormals, below them, at f16's end and beyond it, 0, infinite and NaN: the same formula, the scale
    kept inside f16, NaN as the lowest byte, as latent_quant_append has it."""
    g = torch.Generator().manual_seed(D)
    sizes = [127 * 6.2e-5, 127 * 3e-5, 127 * 1e-6, 6e-6, 1e-7, 0.0, 60000.0] + ([1e4 * 127, 6.6e4 * 127, 1e30, 3e38] if dtype is BF16 else [])
    rows = torch.stack([(torch.rand(D, generator=g) * 2 - 1) * s for s in sizes for _ in range(5)]).to(dtype)
    special = randn(g, 6, D, dtype=dtype)
    special[0, 3], special[1, 3], special[2, 7], special[3] = float("inf"), float("-inf"), float("nan"), float("nan")
    special[4, 1], special[4, 2] = float("nan"), float("inf")
    x = torch.cat([rows, special])[:, None]
    n = len(x)
    caches = [torch.zeros(n, 1, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(n, 1, dtype=torch.float16, device="cuda") for _ in range(2)]
    st = gpu(state([0], torch.arange(n, dtype=torch.int32)[None].contiguous()))
    ops.kv_rope_append(x.cuda(), x.cuda(), st, *caches, torch.zeros(0, device="cuda"), cache_k_scale=scales[0], cache_v_scale=scales[1],
                       cu_new=torch.tensor([0, n], dtype=torch.int32).cuda())
    f = x.float()
    amax = torch.nan_to_num(f.abs(), nan=0.0, posinf=float("inf")).amax(-1)
    scale = torch.where(amax == 0, torch.ones(()), (amax / 127).clamp(2.0 ** -24, 65504.0)).half()
    want = torch.nan_to_num((f / scale.float()[..., None]).round().clamp(-128, 127), nan=-128.0).to(torch.int8)
    for cache, held in zip(caches, scales):
        assert torch.equal(held.cpu(), scale)
        assert torch.equal(cache.cpu(), want)
