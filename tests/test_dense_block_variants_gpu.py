"""kv_rope_append, paged_decode and adapter_add at sizes that take the kernels' variants for much work: many units a block, shares over
several tiles, clusters of every size, several rounds of loads.  Against the formulas in 64 bits, all rows at once (bounds as in
tests/dense_block.py)."""
import math

import pytest
import torch

from tests.dense_block import F32, assert_held, half_step, pages, state
from tests.test_dense_block_gpu import randn, status_is_clean  # noqa: F401  (the fixture)
from wsvd_b200 import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rotated(x, place, inv_freq, layout):
    """x [n, heads, D] in f64 at the positions `place` [n]."""
    half = inv_freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64), place.double()[:, None] * inv_freq.double())[:, None, :]
    y = x.double().clone()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(x[..., a].double(), x[..., b].double()) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _close(got, want, x, dtype, what):
    """tests.dense_block.assert_rotated over many rows."""
    tol = half_step(dtype) * want.abs() + 10 * F32 * 2 * x.double().abs().amax(-1, keepdim=True) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    assert ((got.double() - want).abs() <= tol).all(), (what, ((got.double() - want).abs() - tol).max().item())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("H,K,D,rot,layout", [(32, 8, 128, 128, "half"), (32, 8, 128, 64, "interleaved"), (28, 4, 96, 96, "half"),
                                              (8, 8, 256, 256, "half")])
def test_append_of_long_prompts(dtype, i8, H, K, D, rot, layout):
    """From 606208 units (two 16-byte vectors each, a head's rounded up to a power of two) a thread has four of them."""
    lanes = 1 << math.ceil(math.log2(D / 16))
    rows = 606208 // ((H + 2 * K) * lanes) + 1
    new = [rows - 1 - 700 - 3, 1, 700, 0, 3]
    g = torch.Generator().manual_seed(D + H)
    lens, pad, offset = [0, 40, 7, 3, 11], 5, [0, 3, 100000, 0, 7]
    table, T = pages(5, max(a + b for a, b in zip(lens, new)), 16, g)
    n = rows + pad
    assert n * (H + 2 * K) * lanes >= 606208 and sum(new) == rows
    qkv = randn(g, n, (H + 2 * K) * D, dtype=dtype)
    inv = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    caches = [torch.randint(-128, 128, (T, K, D), generator=g, dtype=torch.int8) if i8 else randn(g, T, K, D, dtype=dtype) for _ in range(2)]
    scales = [torch.rand(T, K, generator=g).half() if i8 else None for _ in range(2)]
    got, held = [c.cuda() for c in caches], [None if s is None else s.cuda() for s in scales]

    def cut(t):
        return (t[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))

    q, k, v = cut(qkv)
    gq, gk, gv = cut(qkv.cuda())
    q_out = ops.kv_rope_append(gk, gv, state(lens, table, device="cuda"), *got, inv.cuda(), cache_k_scale=held[0], cache_v_scale=held[1], q=gq,
                               cu_new=cu.cuda(), pos_offset=torch.tensor(offset, dtype=torch.int32).cuda(), rope_layout=layout).cpu()
    assert ops.kernel_status() == 0
    of = torch.repeat_interleave(torch.arange(5), torch.tensor(new))
    at = torch.tensor(lens)[of] + torch.arange(rows) - cu.long()[of]
    place, slot = at + torch.tensor(offset)[of], table[of, at].long()
    _close(q_out[:rows], _rotated(q[:rows], place, inv, layout), q[:rows], dtype, "q")
    assert (q_out[rows:] == 0).all()
    other = torch.ones(T, dtype=torch.bool)
    other[slot] = False
    for name, x, turned, before, scale, cache, s in (("k", k, True, caches[0], scales[0], got[0], held[0]), ("v", v, False, caches[1], scales[1], got[1], held[1])):
        want = _rotated(x[:rows], place, inv, layout) if turned else x[:rows].double()
        cache = cache.cpu()
        assert torch.equal(cache[other], before[other]), name
        if i8:
            assert torch.equal(s.cpu()[other], scale[other]), name
            assert_held(cache[slot], s.cpu()[slot], want, name)
        elif turned:
            _close(cache[slot], want, x[:rows], dtype, name)
        else:
            assert torch.equal(cache[slot], x[:rows])


def _adapters(g, rows, n_in, n_out, r, count, dtype, packed, pad=0, in_place=False):
    n = sum(rows) + pad
    x, y = randn(g, n, n_in, dtype=dtype), randn(g, n, n_out, dtype=dtype)
    a, b = randn(g, count, n_in, r, scale=1 / math.sqrt(n_in), dtype=dtype), randn(g, count, r, n_out, scale=0.5 / math.sqrt(r), dtype=dtype)
    scale = torch.rand(count, generator=g) * 2 - 0.5
    ad = torch.randint(0, count, (len(rows),), generator=g, dtype=torch.int32)
    if len(rows) > 2:
        ad[1] = -1
    gy = y.cuda()
    cu = torch.tensor([0, *torch.tensor(rows).cumsum(0).tolist()], dtype=torch.int32)
    got = ops.adapter_add(gy, x.cuda(), a.cuda(), b.cuda(), ad.cuda(), scale=scale.cuda(), cu_new=cu.cuda() if packed else None,
                          out=gy if in_place else None).cpu()
    assert ops.kernel_status() == 0
    of = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    assert torch.equal(got[sum(rows):], y[sum(rows):])
    for i in range(-1, count):
        mine = (ad[of] == i).nonzero()[:, 0]
        if i < 0:
            assert torch.equal(got[mine], y[mine])
            continue
        xx, aa, bb, s = x[mine].double(), a[i].double(), b[i].double(), float(scale[i])
        h, habs = xx @ aa, xx.abs() @ aa.abs()
        want = y[mine].double() + s * (h @ bb)
        # as tests.dense_block.adapters64, the rounding of x A to 16 bits where rows are packed alone
        err = (n_in + 4) * F32 * habs + (half_step(dtype) * h.abs() if packed else 0)
        bound = half_step(dtype) * want.abs() + abs(s) * (err @ bb.abs() + (r + 4) * F32 * (habs @ bb.abs())) + \
            torch.finfo(dtype).smallest_normal * half_step(dtype) * 2 + 2 * F32 * y[mine].double().abs()
        off = (got[mine].double() - want).abs() - bound
        assert (off <= 0).all(), (i, off.max().item())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("r", [8, 16, 40, 64, 100, 128, 256])
@pytest.mark.parametrize("n_out", [4096, 2056])
def test_adapters_of_prompts_with_shares_over_several_units_and_tiles(dtype, r, n_out):
    """25 tiles of 128 rows and up to 64 blocks of columns, three to four a CTA; the last block of columns of 8."""
    _adapters(torch.Generator().manual_seed(r), [1, 300, 1500, 700, 129, 64, 0, 128], 64, n_out, r, 3, dtype, packed=True, pad=7, in_place=r == 40)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_in", [1024, 1032, 2048, 4096, 11008, 264])
@pytest.mark.parametrize("r", [16, 32, 64, 128, 200])
def test_adapters_of_prompts_with_long_inputs(dtype, n_in, r):
    """Clusters of four (from 1024 inputs) and eight (from 2048), slices that end inside a stage."""
    _adapters(torch.Generator().manual_seed(n_in + r), [70, 3, 64, 1], n_in, 200, r, 2, dtype, packed=True)


def test_adapters_of_prompts_with_enough_tiles_for_small_clusters():
    """240 tiles: a cluster of two is enough for every SM."""
    _adapters(torch.Generator().manual_seed(3), [7000, 1, 8300], 1024, 64, 16, 2, BF16, packed=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_in,r", [(4096, 128), (11008, 64), (4104, 64), (2056, 128), (2048, 256), (11008, 4), (5120, 100), (131072, 16), (131080, 8)])
def test_adapters_of_single_rows_with_long_inputs(dtype, n_in, r):
    """Slices that a thread asks for in several rounds; 131072 inputs are the most that slices are made for."""
    _adapters(torch.Generator().manual_seed(n_in + r), [1] * 7, n_in, 520, r, 2, dtype, packed=False)


def test_adapters_of_many_requests_of_a_few_rows():
    """Single tokens and chunks of a few in one call."""
    rows = torch.randint(0, 9, (150,), generator=torch.Generator().manual_seed(4)).tolist()
    _adapters(torch.Generator().manual_seed(5), rows, 1024, 1032, 16, 12, F16, packed=True, pad=3)
