"""kv_rope_append, paged_decode and adapter_add against the formulas in 64 bits (bounds: tests/dense_block.py)."""
import math

import pytest
import torch

from tests.dense_block import (F32, adapters64, append64, assert_held, assert_rotated, attend64, half_step, pages, rotate64, rows_of,
                               state)
from wsvd_b200 import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def status_is_clean():
    from wsvd_b200 import _lib

    _lib.check(_lib.lib().wsvd_kernel_status_reset(), "reset")
    yield
    _lib.check(_lib.lib().wsvd_kernel_status_reset(), "reset")


def gpu(st):
    table = st.req_manager.req_to_token_indexs
    return state(st.b_seq_len.tolist(), table, st.b_req_idx.tolist(), device="cuda")


def randn(g, *shape, dtype=F16, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------ append

def _cache(g, T, H, D, dtype, i8, head_major=False):
    """A cache with values in every slot, token-major or as a strided view of a head-major store, and its scales."""
    shape = (H, T, D) if head_major else (T, H, D)
    store = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8) if i8 else randn(g, *shape, dtype=dtype)
    scale = (torch.rand(shape[:2], generator=g) + 0.5).half() if i8 else None
    if head_major:
        store, scale = store.transpose(0, 1), None if scale is None else scale.transpose(0, 1)
    return store, scale


def _to_gpu(t):
    """The same strides on the GPU."""
    if t is None:
        return None
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda").copy_(t)


def _run_append(g, new, lens, H, K, D, rot, dtype, i8, layout="half", offset=None, packed=True, pad=0, page=4, width=None, n_req=None,
                idx=None, shift=0, head_major=False, table=None, T=None, with_q=True):
    B = len(lens)
    width = width or max(a + b for a, b in zip(lens, new)) + 1
    if table is None:
        table, T = pages(n_req or B, width, page, g)
    st = state(lens, table, idx)
    n = sum(new) + pad
    cu = None if not packed else [sum(new[:i]) for i in range(B + 1)]
    # column slices of a joined projection; shift: two bytes off 16
    wide = (H + 2 * K) * D + 8
    flat = randn(g, n * wide + 8, dtype=dtype)[shift:]
    qkv = flat[:n * wide].view(n, wide)
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + K) * D].unflatten(1, (K, D))
    v = qkv[:, (H + K) * D:(H + 2 * K) * D].unflatten(1, (K, D))
    inv = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float()
    off = None if offset is None else torch.tensor(offset, dtype=torch.int32)
    caches = [_cache(g, T, K, D, dtype, i8, head_major) for _ in range(2)]
    (ck, ks), (cv, vs) = caches
    gk, gks, gv, gvs = (_to_gpu(t) for t in (ck, ks, cv, vs))
    base = torch.empty(flat.numel() + shift, dtype=dtype, device="cuda")[shift:].copy_(flat)
    gqkv = base[:n * wide].view(n, wide)
    gq = gqkv[:, :H * D].unflatten(1, (H, D))
    got = ops.kv_rope_append(gqkv[:, H * D:(H + K) * D].unflatten(1, (K, D)), gqkv[:, (H + K) * D:(H + 2 * K) * D].unflatten(1, (K, D)),
                             gpu(st), gk, gv, inv.cuda(), cache_k_scale=gks, cache_v_scale=gvs, q=gq if with_q else None,
                             cu_new=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda(),
                             pos_offset=None if off is None else off.cuda(), rope_layout=layout)
    torch.cuda.synchronize()
    stored, turned = append64(k, v, q, st, cu, inv, off, layout, T)
    gk, gks, gv, gvs = (None if t is None else t.cpu() for t in (gk, gks, gv, gvs))
    if with_q:
        got = got.cpu()
        for i, want in enumerate(turned):
            if want is None:
                assert (got[i] == 0).all()
            else:
                assert_rotated(got[i], want, q[i].double(), dtype, f"q row {i}")
    else:
        assert got is None
    of_slot = {}
    for i, at in enumerate(rows_of(cu, n)):
        if at is not None and 0 <= int(st.b_req_idx[at[0]]) < table.shape[0]:
            pos = int(st.b_seq_len[at[0]]) + at[1]
            if 0 <= pos < table.shape[1]:
                of_slot[int(table[int(st.b_req_idx[at[0]]), pos])] = i
    for t in range(T):
        if t not in stored:
            for a, b in ((gk, ck), (gv, cv), (gks, ks), (gvs, vs)):
                assert a is None or torch.equal(a[t], b[t]), t
            continue
        wk, wv = stored[t]
        if i8:
            assert_held(gk[t], gks[t], wk, f"k slot {t}")
            assert_held(gv[t], gvs[t], wv, f"v slot {t}")
        else:
            assert_rotated(gk[t], wk, k[of_slot[t]].double(), dtype, f"k slot {t}")
            assert torch.equal(gv[t].double(), wv), t
    return stored


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("H,K,D,rot", [(4, 4, 128, 128), (8, 2, 64, 64), (7, 1, 96, 96), (4, 2, 256, 128), (2, 2, 80, 80),
                                       (3, 1, 34, 10), (6, 2, 128, 0), (2, 1, 2, 2), (4, 2, 192, 64)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_append_prompts(dtype, i8, H, K, D, rot, layout):
    g = torch.Generator().manual_seed(D + H)
    _run_append(g, [3, 0, 1, 17, 5], [0, 4, 9, 2, 1], H, K, D, rot, dtype, i8, layout, offset=[0, 5, 70000, 131072, 3], pad=2,
                idx=[4, 0, 3, 1, 2])
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, True)])
@pytest.mark.parametrize("B", [1, 3, 70])
@pytest.mark.parametrize("shift,head_major", [(0, False), (0, True), (1, False), (4, False)])
def test_append_single_tokens(dtype, i8, B, shift, head_major):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    _run_append(g, [1] * B, lens, 8, 2, 128, 128, dtype, i8, packed=False, shift=shift, head_major=head_major)
    assert ops.kernel_status() == 0


def test_append_without_queries_and_of_nothing():
    g = torch.Generator().manual_seed(5)
    _run_append(g, [2, 3], [1, 0], 4, 2, 64, 64, F16, False, with_q=False)
    _run_append(g, [0, 0], [1, 0], 4, 2, 64, 64, F16, False, pad=3)
    _run_append(g, [0, 0], [1, 0], 4, 2, 64, 64, F16, False)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D", [128, 34])
def test_append_far_positions(i8, D):
    """An f32 angle would be off by 2^31 2^-24 = 128 radians here."""
    g = torch.Generator().manual_seed(6)
    _run_append(g, [4, 3], [0, 1], 2, 2, D, D, F16, i8, offset=[2_000_000_000, 16_777_217])


def test_append_skips_rows_without_a_place():
    g = torch.Generator().manual_seed(7)
    for D in (128, 30):
        table, T = pages(3, 6, 2, g)
        table[0, 2], table[1, 1] = -1, T
        st = _run_append(g, [4, 2, 3, 1], [0, 1, 4, 0], 4, 2, D, 2 * (D // 4), BF16, False, table=table.clone(), T=T, idx=[0, 1, 2, 9])
        # 3 of row 0's, 1 of row 1's, 2 of row 2's (its third is beyond the table), none of a request that does not exist
        assert len(st) == 6
        assert ops.kernel_status() == 7


def test_append_keeps_the_callers_padding_rows_and_works_in_place():
    g = torch.Generator().manual_seed(8)
    for D in (128, 30):
        table, T = pages(2, 8, 4, g)
        st = state([0, 2], table)
        q = randn(g, 6, 4, D)
        k, v = randn(g, 6, 2, D), randn(g, 6, 2, D)
        ck, cv = torch.zeros(T, 2, D, dtype=F16).cuda(), torch.zeros(T, 2, D, dtype=F16).cuda()
        inv = torch.rand(D // 2, generator=g)
        cu = torch.tensor([0, 3, 4], dtype=torch.int32).cuda()
        mine = torch.full((6, 4, D), 7.0, dtype=F16).cuda()
        got = ops.kv_rope_append(k.cuda(), v.cuda(), gpu(st), ck, cv, inv.cuda(), q=q.cuda(), q_out=mine, cu_new=cu)
        assert got is mine and (mine[4:] == 7).all()
        here = q.cuda()
        got2 = ops.kv_rope_append(k.cuda(), v.cuda(), gpu(st), ck, cv, inv.cuda(), q=here, q_out=here, cu_new=cu)
        assert got2 is here and torch.equal(here[:4], mine[:4]) and torch.equal(here[4:].cpu(), q[4:])


def test_append_slots_beyond_32_bits_of_bytes():
    """Offsets of more than 2^31 elements."""
    g = torch.Generator().manual_seed(9)
    T, K, D = 2_200_000, 8, 128
    ck = torch.zeros(T, K, D, dtype=torch.int8, device="cuda")
    cv, ks = torch.zeros_like(ck), torch.ones(T, K, dtype=F16, device="cuda")
    vs = ks.clone()
    table = torch.tensor([[T - 1, 5]], dtype=torch.int32)
    k, v = randn(g, 1, K, D), randn(g, 1, K, D)
    st = state([0], table)
    ops.kv_rope_append(k.cuda(), v.cuda(), gpu(st), ck, cv, torch.ones(D // 2).cuda(), cache_k_scale=ks, cache_v_scale=vs)
    assert_held(ck[T - 1].cpu(), ks[T - 1].cpu(), rotate64(k[0].double(), 0, torch.ones(D // 2), "half"), "last slot")
    q = randn(g, 1, 8, D)
    st = state([2], table)
    got = ops.paged_decode(q.cuda(), gpu(st), ck, cv, ks, vs)
    small = torch.tensor([[1, 0]], dtype=torch.int32)
    pick = torch.tensor([5, T - 1])
    want, _, bound, _ = attend64(q, state([2], small), *(t[pick.cuda()].cpu() for t in (ck, cv, ks, vs)), 0, 0.0)
    assert ((got.cpu().double() - want).abs() <= bound).all()


# ------------------------------------------------------------------ attention

def _run_paged(g, lens, H, K, D, dtype, i8, window=0, page=16, width=None, sm_scale=0.0, idx=None, n_req=None, shift=0,
               head_major=False, break_table=None, scale=1.0, spread=1.0):
    B = len(lens)
    n_req = n_req or B
    width = width or max([1, *lens])
    table, T = pages(n_req, width, page, g)
    if break_table:
        break_table(table, T)
    st = state(lens, table, idx)
    q = randn(g, B, H, D, dtype=dtype, scale=scale)
    if i8:
        k, v = (torch.randint(-127, 128, (T, K, D), generator=g, dtype=torch.int8) for _ in range(2))
        ks, vs = ((torch.rand(T, K, generator=g) * 0.02 * spread + 0.001).half() for _ in range(2))
    else:
        k, v = randn(g, T, K, D, dtype=dtype), randn(g, T, K, D, dtype=dtype)
        ks = vs = None
    want, lse, bound, lse_bound = attend64(q, st, k, v, ks, vs, window, sm_scale)
    # what no position names is never read: poison
    named = torch.zeros(T, dtype=torch.bool)
    for b in range(B):
        n = min(max(lens[b], 0), width)
        r = int(st.b_req_idx[b])
        if 0 <= r < n_req:
            s = table[r, max(0, n - window) if window else 0:n]
            named[s[(s >= 0) & (s < T)].long()] = True
    if i8:
        k[~named], v[~named] = -128, -128
        ks[~named], vs[~named] = float("nan"), float("inf")
    else:
        k[~named], v[~named] = float("nan"), float("inf")

    def on_gpu(t):
        if t is None:
            return None
        if head_major:
            return t.transpose(0, 1).contiguous().cuda().transpose(0, 1)
        if shift and t.dim() == 3:
            buf = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:].view(t.shape)
            return buf.copy_(t)
        return t.cuda()

    got, got_lse = ops.paged_decode(on_gpu(q) if shift else q.cuda(), gpu(st), *(on_gpu(t) for t in (k, v, ks, vs)), window=window,
                                    sm_scale=sm_scale, return_lse=True)
    torch.cuda.synchronize()
    assert got.dtype == dtype and got.shape == q.shape and got_lse.dtype == torch.float32
    off = (got.cpu().double() - want).abs() - bound
    assert (off <= 0).all(), off.max().item()  # (a NaN fails)
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse.cpu()), empty) and (got_lse.cpu()[empty] < 0).all()
    off = ((got_lse.cpu().double() - lse).abs() - lse_bound)[~empty]
    assert (off <= 0).all(), off.max().item()
    return got


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 300, 129]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("H,K,D", [(2, 2, 128), (8, 2, 128), (8, 1, 64), (7, 1, 96), (16, 1, 128), (20, 1, 64), (4, 2, 256), (9, 1, 256),
                                   (4, 2, 80), (2, 1, 16), (3, 1, 33)])
def test_paged_lengths_and_heads(dtype, i8, H, K, D):
    g = torch.Generator().manual_seed(H * D)
    _run_paged(g, LENS, H, K, D, dtype, i8, idx=[9, 1, 2, 8, 4, 5, 6, 7, 3, 0])
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, False), (BF16, True)])
@pytest.mark.parametrize("window", [1, 16, 40, 64, 299, 100000])
@pytest.mark.parametrize("D", [128, 40])
def test_paged_window(dtype, i8, window, D):
    g = torch.Generator().manual_seed(window)
    _run_paged(g, LENS, 8, 2, D, dtype, i8, window=window, page=1)


@pytest.mark.parametrize("lens,H,K,D,dtype,i8", [
    ([20000], 8, 1, 128, BF16, False),        # one sequence over all SMs
    ([30001], 1, 1, 64, F16, False),
    ([9000, 3], 16, 2, 128, F16, True),
    ([5000, 1, 0, 777], 6, 2, 256, BF16, False),
])
def test_paged_long(lens, H, K, D, dtype, i8):
    g = torch.Generator().manual_seed(lens[0])
    _run_paged(g, lens, H, K, D, dtype, i8, page=64)


@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, True)])
def test_paged_many_sequences(dtype, i8):
    """More sequences and items than blocks."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (400,), generator=g).tolist()
    _run_paged(g, lens, 4, 2, 64, dtype, i8, page=8)


@pytest.mark.parametrize("D", [128, 24])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("shift,head_major", [(1, False), (16, False), (0, True)])
def test_paged_strides_and_addresses(D, i8, shift, head_major):
    g = torch.Generator().manual_seed(D)
    _run_paged(g, [70, 3, 130], 4, 2, D, F16, i8, shift=shift, head_major=head_major)


@pytest.mark.parametrize("D", [128, 24])
def test_paged_bad_pages(D):
    g = torch.Generator().manual_seed(11)

    def bad(table, T):
        table[0, 3], table[0, 70], table[1, :], table[2, 0] = -1, T, 2 ** 31 - 1, -5

    _run_paged(g, [100, 50, 2, 20], 4, 2, D, F16, False, break_table=bad)
    assert ops.kernel_status() == 7


@pytest.mark.parametrize("D", [128, 24])
def test_paged_bad_requests_and_lengths(D):
    g = torch.Generator().manual_seed(12)
    _run_paged(g, [100, 50, 200, -4], 4, 2, D, BF16, True, width=120, idx=[0, 7, 1, 2], n_req=3)
    assert ops.kernel_status() == 7


@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("scale,sm_scale", [(30.0, 0.0), (1e-3, 0.0), (1.0, 0.5), (1e-6, 2000.0)])
def test_paged_ranges(dtype, i8, scale, sm_scale):
    """Peaked and flat weights, queries from the smallest to large values, scales of a wide range."""
    g = torch.Generator().manual_seed(13)
    _run_paged(g, [200, 33, 1], 4, 2, 128, dtype, i8, scale=scale, sm_scale=sm_scale, spread=50.0)


def test_paged_large_bf16_queries_on_bytes():
    """Queries beyond the range of f16."""
    g = torch.Generator().manual_seed(14)
    _run_paged(g, [100, 3], 4, 2, 128, BF16, True, scale=1e9, sm_scale=1e-9)


@pytest.mark.parametrize("D", [128, 40])
def test_paged_scores_of_lowest_value_and_nan(D):
    """A key row of -inf gets weight zero; a NaN key makes its row NaN and no other."""
    g = torch.Generator().manual_seed(15)
    table, T = pages(3, 20, 4, g)
    st = state([20, 20, 20], table)
    q = randn(g, 3, 2, D).abs()
    k, v = randn(g, T, 1, D), randn(g, T, 1, D)
    k[table[0, 7].long()] = -65504.0
    k[table[1, 7].long(), 0, 3] = float("-inf")
    k[table[2, 7].long(), 0, 3] = float("nan")
    got = ops.paged_decode(q.cuda(), gpu(st), k.cuda(), v.cuda()).cpu()
    keep = [s for s in range(20) if s != 7]
    for b in (0, 1):
        s = table[b, keep].long()
        for h in range(2):
            w = torch.softmax(k[s, 0].double() @ q[b, h].double() / math.sqrt(D), 0)
            assert ((got[b, h].double() - w @ v[s, 0].double()).abs() <= 2e-3 * (w @ v[s, 0].double().abs()) + 1e-3).all()
    assert torch.isnan(got[2]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_short_sequences_of_bytes_keep_the_scores(dtype):
    """Sequences of one to three tokens, whose weights average nothing out: lse of one token is its score.  With the query as 24
    bits the products are exact, so that a score is off by the query's half step, 2^-23 of its row's largest power of two, and
    four roundings of f32.  lse is then r + log2(sum) of a reference r that may lie up to 16 (a factor 2^16) below the score: a
    logarithm of 8 to 16 has steps of 2^-20, and so has the difference that went into the exponential (a half step, 2^-21); the
    exponential and the sum are off by 2^-22 more.  In all 2^-20 + 2^-21 + 2^-22 < 2^-19 in base 2, which the first run of this test
    (0.0447, off by 2^-21) showed to be missing from the bound."""
    g = torch.Generator().manual_seed(31)
    table, T = pages(64, 4, 2, g)
    st = state([1] * 64, table)
    q = randn(g, 64, 4, 128, dtype=dtype)
    k, v = (torch.randint(-127, 128, (T, 2, 128), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = ((torch.rand(T, 2, generator=g) * 0.02 + 0.001).half() for _ in range(2))
    _, lse = ops.paged_decode(q.cuda(), gpu(st), *(t.cuda() for t in (k, v, ks, vs)), return_lse=True)
    lse = lse.cpu().double()
    for b in range(64):
        s = int(table[b, 0])
        for h in range(4):
            kk = k[s, h // 2].double() * ks[s, h // 2].double()
            qq = q[b, h].double()
            z = float(kk @ qq) / math.sqrt(128)
            tol = (2.0 ** -23 * float(qq.abs().max()) * float(kk.abs().sum())) / math.sqrt(128) + 8 * 2.0 ** -24 * abs(z) + 2.0 ** -19 * math.log(2)
            assert abs(float(lse[b, h]) - z) <= tol, (b, h, float(lse[b, h]) - z, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_paged_sums_of_bytes_at_their_largest(D):
    """Every key -128 and queries whose lower two bytes are all but full: the integer sums are at the ends of their range.  Each
    product is exact, the sum is off by f32's roundings; all tokens weigh the same, so that out is their mean value."""
    g = torch.Generator().manual_seed(36)
    n = 45
    table, T = pages(1, n, 8, g)
    st = state([n], table)
    q = torch.full((1, 2, D), 65504 * 2.0 ** -22, dtype=F16)
    q[0, :, 5] = 1.0
    q[0, 1] *= -1
    k = torch.full((T, 1, D), -128, dtype=torch.int8)
    v = torch.randint(-128, 128, (T, 1, D), generator=g, dtype=torch.int8)
    ks, vs = torch.full((T, 1), 0.5).half(), torch.full((T, 1), 0.25).half()
    out, lse = ops.paged_decode(q.cuda(), gpu(st), *(t.cuda() for t in (k, v, ks, vs)), return_lse=True)
    z = (q[0].double().sum(1) * -64 / math.sqrt(D) + math.log(n)).unsqueeze(0)
    assert ((lse.cpu().double() - z).abs() <= 2.0 ** -19 * math.log(2) + 8 * F32 * z.abs()).all()
    mean = v[table[0].long(), 0].double().mean(0) * 0.25
    assert ((out.cpu().double() - mean).abs() <= 2.0 ** -11 * mean.abs() + 2.0 ** -16 * 32).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D", [128, 40])
def test_paged_queries_that_are_not_numbers_stay_in_their_heads(D, i8, bad):
    g = torch.Generator().manual_seed(32)
    lens = [20, 700]
    table, T = pages(2, 700, 4, g)
    st = state(lens, table)
    q = randn(g, 2, 8, D)
    k, v = (torch.randint(-127, 128, (T, 2, D), generator=g, dtype=torch.int8) for _ in range(2)) if i8 else (randn(g, T, 2, D) for _ in range(2))
    scales = [(torch.rand(T, 2, generator=g) * 0.02 + 0.001).half().cuda() for _ in range(2)] if i8 else []
    args = (gpu(st), k.cuda(), v.cuda(), *scales)
    want = ops.paged_decode(q.cuda(), *args).cpu()
    q[0, 1, 3] = q[1, 6, D - 1] = bad
    got, lse = ops.paged_decode(q.cuda(), *args, return_lse=True)
    got, lse = got.cpu(), lse.cpu()
    hit = torch.zeros(2, 8, dtype=torch.bool)
    hit[0, 1] = hit[1, 6] = True
    assert torch.equal(got[~hit], want[~hit]) and torch.isfinite(lse[~hit]).all()
    assert torch.isnan(got[hit]).all()


def test_paged_runs_are_bitwise_equal_and_take_a_workspace():
    g = torch.Generator().manual_seed(16)
    table, T = pages(3, 3000, 16, g)
    st = gpu(state([3000, 1500, 2999], table))
    q, k, v = randn(g, 3, 8, 128).cuda(), randn(g, T, 2, 128).cuda(), randn(g, T, 2, 128).cuda()
    want = ops.paged_decode(q, st, k, v)
    ws = torch.full((1 << 22,), float("nan"), device="cuda")  # nothing in it has to be set
    out = torch.empty(3, 16, 128, dtype=F16, device="cuda")[:, ::2]
    for _ in range(3):
        assert ops.paged_decode(q, st, k, v, workspace=ws, out=out) is out
        assert torch.equal(out, want)
        ws.fill_(float("inf"))


# ------------------------------------------------------------------ adapters

def _run_adapters(g, rows, adapter, n_in, n_out, r, count, dtype, packed=True, pad=0, with_scale=True, shift=0, in_place=False,
                  a_scale=None):
    n = sum(rows) + pad
    cu = [sum(rows[:i]) for i in range(len(rows) + 1)] if packed else None

    def strided(rows_, cols):  # column slices of wider matrices; shift: off 16 bytes
        buf = randn(g, rows_ * (cols + 8) + 8, dtype=dtype)
        dev = torch.empty(buf.numel(), dtype=dtype, device="cuda").copy_(buf)
        return tuple(t[shift:shift + rows_ * (cols + 8)].view(rows_, cols + 8)[:, :cols] for t in (buf, dev))

    x, gx = strided(n, n_in)
    y, gy = strided(n, n_out)
    a = randn(g, count, n_in, r, dtype=dtype, scale=a_scale or 1 / math.sqrt(n_in))
    b = randn(g, count, r, n_out, dtype=dtype, scale=0.5 / math.sqrt(r))
    scale = (torch.rand(count, generator=g) * 2 - 0.5) if with_scale else None
    ad = torch.tensor(adapter, dtype=torch.int32)
    want, bound, padding = adapters64(y, x, a, b, ad, scale, cu)
    got = ops.adapter_add(gy, gx, a.cuda(), b.cuda(), ad.cuda(), scale=None if scale is None else scale.cuda(),
                          cu_new=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda(), out=gy if in_place else None)
    torch.cuda.synchronize()
    if in_place:
        assert got is gy
    assert got.dtype == dtype
    off = (got.cpu().double() - want).abs() - bound
    assert (off <= 0).all(), off.max().item()
    untouched = [i for i in range(n) if padding[i]] + [
        i for i, p in enumerate(rows_of(cu, n)) if p is not None and not 0 <= adapter[p[0]] < count]
    assert torch.equal(got.cpu()[untouched], y[untouched])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_in,n_out,r", [(256, 512, 16), (1000, 2040, 8), (512, 264, 64), (96, 64, 128), (320, 136, 100), (64, 72, 4),
                                          (33, 17, 3), (128, 1024, 256), (4096, 64, 1), (8, 8, 8)])
@pytest.mark.parametrize("packed", [False, True])
def test_adapters(dtype, n_in, n_out, r, packed):
    g = torch.Generator().manual_seed(n_in + r)
    adapter = [2, -1, 0, 2, 2, 1, 0, 2, 2, 2, 2, 2]
    rows = [1] * 12 if not packed else [1, 3, 0, 65, 64, 2, 1, 130, 16, 0, 7, 1]
    _run_adapters(g, rows, adapter, n_in, n_out, r, 3, dtype, packed=packed, pad=5 if packed else 0)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("B,count", [(1, 1), (5, 64), (150, 1), (300, 7), (64, 48)])
@pytest.mark.parametrize("r", [16, 40])
def test_adapters_single_rows(B, count, r):
    g = torch.Generator().manual_seed(B)
    ad = torch.randint(-1, count, (B,), generator=g).tolist()
    _run_adapters(g, [1] * B, ad, 1024, 1536, r, count, BF16, packed=False, with_scale=B != 5)


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("packed", [False, True])
def test_adapters_strides_and_in_place(shift, packed):
    g = torch.Generator().manual_seed(shift)
    rows = [70, 3, 64] if packed else [1, 1, 1]
    _run_adapters(g, rows, [1, -1, 0], 256, 320, 16, 2, F16, packed=packed, shift=shift, in_place=True, pad=2 if packed else 0)


def test_adapters_that_do_not_exist():
    g = torch.Generator().manual_seed(4)
    for n_in in (256, 33):
        for packed in (False, True):
            _run_adapters(g, [1, 1, 1, 1], [3, 0, -2, 2 ** 30], n_in, 64, 8, 3, BF16, packed=packed)
            assert ops.kernel_status() == 7


@pytest.mark.parametrize("n_in", [64, 61])
def test_adapters_rows_in_front_of_the_first_request(n_in):
    """cu_new that begins behind row 0: those rows are padding like the ones behind."""
    g = torch.Generator().manual_seed(33)
    x, y = randn(g, 200, n_in), randn(g, 200, 48)
    a, b = randn(g, 2, n_in, 8, scale=0.1).cuda(), randn(g, 2, 8, 48).cuda()
    args = dict(cu_new=torch.tensor([70, 150, 151], dtype=torch.int32).cuda())
    ad = torch.tensor([1, 0], dtype=torch.int32).cuda()
    got = ops.adapter_add(y.cuda(), x.cuda(), a, b, ad, **args).cpu()
    assert torch.equal(got[:70], y[:70]) and torch.equal(got[151:], y[151:])
    mine = torch.full((200, 48), 7.0, dtype=F16, device="cuda")
    kept = ops.adapter_add(y.cuda(), x.cuda(), a, b, ad, out=mine, **args).cpu()
    assert (kept[:70] == 7).all() and (kept[151:] == 7).all() and torch.equal(kept[70:151], got[70:151])


@pytest.mark.parametrize("n_in", [256, 33])
def test_adapters_with_infinities_stay_in_their_rows(n_in):
    g = torch.Generator().manual_seed(5)
    x, y = randn(g, 70, n_in), randn(g, 70, 64)
    a, b = randn(g, 2, n_in, 8, scale=0.05), randn(g, 2, 8, 64)
    for cu, ad in ((None, [0] * 35 + [1] * 35), ([0, 35, 70], [0, 1])):
        args = dict(cu_new=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda())
        ad = torch.tensor(ad, dtype=torch.int32).cuda()
        want = ops.adapter_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), ad, **args)
        bad = x.clone()
        bad[3], bad[50] = float("nan"), float("inf")
        got = ops.adapter_add(y.cuda(), bad.cuda(), a.cuda(), b.cuda(), ad, **args)
        keep = [i for i in range(70) if i not in (3, 50)]
        assert torch.equal(got[keep], want[keep])
        assert not torch.isfinite(got[[3, 50]]).any()


# ------------------------------------------------------------------ together, on streams, in graphs

def _block(g, dtype, i8, H=8, K=2, D=128, M=256, B=3, width=80):
    r = 8
    W = randn(g, M, (H + 2 * K) * D, dtype=dtype, scale=1 / math.sqrt(M))
    a, b = randn(g, 2, M, r, dtype=dtype, scale=1 / math.sqrt(M)), randn(g, 2, r, W.shape[1], dtype=dtype, scale=0.3)
    table, T = pages(B, width, 16, g)
    if i8:
        caches = [torch.zeros(T, K, D, dtype=torch.int8), torch.zeros(T, K, D, dtype=torch.int8)]
        scales = [torch.zeros(T, K, dtype=F16), torch.zeros(T, K, dtype=F16)]
    else:
        caches, scales = [torch.zeros(T, K, D, dtype=dtype), torch.zeros(T, K, D, dtype=dtype)], [None, None]
    inv = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float()
    return W, a, b, table, T, caches, scales, inv


@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, False), (BF16, True)])
def test_prompt_then_steps(dtype, i8):
    """Prompts of three requests (one without an adapter), then four steps of one token each: projection, adapters, append,
    attention, against the whole in 64 bits."""
    g = torch.Generator().manual_seed(21)
    H, K, D, M = 8, 2, 128, 256
    W, a, b, table, T, caches, scales, inv = _block(g, dtype, i8)
    gW, ga, gb, ginv = (t.cuda() for t in (W, a, b, inv))
    gc, gs = [t.cuda() for t in caches], [None if t is None else t.cuda() for t in scales]
    adapter = torch.tensor([1, -1, 0], dtype=torch.int32)
    prompts = [20, 1, 37]
    history = [[], [], []]  # each sequence's inputs in f64
    st = gpu(state([0, 0, 0], table))

    def qkv64(x, i):
        y = x.double() @ W.double()
        return y if i < 0 else y + (x.double() @ a[i].double()) @ b[i].double()

    def step(xs, cu):
        x = torch.cat(xs)
        y = ops.adapter_add(x.cuda() @ gW, x.cuda(), ga, gb, adapter.cuda(), cu_new=cu)
        q = ops.kv_rope_append(y[:, H * D:(H + K) * D].unflatten(1, (K, D)), y[:, (H + K) * D:].unflatten(1, (K, D)), st, *gc, ginv,
                               cache_k_scale=gs[0], cache_v_scale=gs[1], q=y[:, :H * D].unflatten(1, (H, D)), cu_new=cu)
        for i, t in enumerate(xs):
            history[i] += list(t)
        st.b_seq_len += torch.tensor([len(t) for t in xs], dtype=torch.int32, device="cuda")
        return q

    step([randn(g, n, M, dtype=dtype) for n in prompts], torch.tensor([0, 20, 21, 58], dtype=torch.int32).cuda())
    for _ in range(4):
        q = step([randn(g, 1, M, dtype=dtype) for _ in range(3)], None)
        got = ops.paged_decode(q, st, *gc, *gs).cpu().double()
        for i in range(3):
            y = torch.stack([qkv64(x, int(adapter[i])) for x in history[i]])
            n = len(history[i])
            kk = torch.stack([rotate64(y[s, H * D:(H + K) * D].view(K, D), s, inv, "half") for s in range(n)])
            qq = rotate64(y[-1, :H * D].view(H, D), n - 1, inv, "half")
            vv = y[:, (H + K) * D:].view(n, K, D)
            for h in range(H):
                w = torch.softmax(kk[:, h // 4] @ qq[h] / math.sqrt(D), 0)
                want = w @ vv[:, h // 4]
                # q, k, v, the projection and the result are rounded to the type (bytes: half a step of 1/127 of the largest):
                # a score of |z| <= 5 moves by a few roundings of its terms, the values by two
                u = half_step(dtype) * 4 + (0.5 / 127 * 3 if i8 else 0)
                zmag = (kk[:, h // 4].abs() @ qq[h].abs() / math.sqrt(D)).max()
                tol = (u + u * zmag) * 2 * (w @ vv[:, h // 4].abs()) + u * vv.abs().max()
                assert ((got[i, h] - want).abs() <= tol).all(), (i, h)
    assert ops.kernel_status() == 0


def test_two_graphs_and_an_eager_call_share_nothing():
    """The whole block captured twice (two batches), replayed on two streams at once, beside an eager call: each gives what it
    gives alone."""
    g = torch.Generator().manual_seed(22)
    H, K, D = 8, 2, 128
    runs = []
    for seed in (1, 2):
        W, a, b, table, T, caches, scales, inv = _block(g, F16, False, width=700)
        gc = [randn(g, T, K, D).cuda() for _ in range(2)]
        st = gpu(state([600, 333, 1], table))
        x = randn(g, 3, 256).cuda()
        args = (x, W.cuda(), a.cuda(), b.cuda(), torch.tensor([0, 1, -1], dtype=torch.int32).cuda(), st, gc, inv.cuda())

        def block(x, W, a, b, ad, st, gc, inv):
            y = ops.adapter_add(x @ W, x, a, b, ad)
            q = ops.kv_rope_append(y[:, H * D:(H + K) * D].unflatten(1, (K, D)), y[:, (H + K) * D:].unflatten(1, (K, D)), st, *gc, inv,
                                   q=y[:, :H * D].unflatten(1, (H, D)))
            return ops.paged_decode(q, st, *gc)

        want = block(*args).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(*args)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(*args)
        runs.append((graph, out, want, block, args, side))
    for _ in range(5):
        torch.cuda.synchronize()
        for graph, out, *_, side in runs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, *_, side in runs:
            with torch.cuda.stream(side):
                graph.replay()
        eager = runs[0][3](*runs[0][4])
        torch.cuda.synchronize()
        assert torch.equal(eager, runs[0][2])
        for _, out, want, *_ in runs:
            assert torch.equal(out, want)


def test_calls_of_nothing_and_next_to_nothing():
    """No rows, no sequences, no positions, no adapters, a table without columns."""
    none = lambda *shape, dtype=F16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    empty = gpu(state([], torch.zeros(0, 0, dtype=torch.int32)))
    cache = none(0, 2, 64)
    assert ops.paged_decode(none(0, 4, 64), empty, cache, cache).shape == (0, 4, 64)
    assert ops.kv_rope_append(none(0, 2, 64), none(0, 2, 64), empty, none(8, 2, 64), none(8, 2, 64), none(32, dtype=torch.float32),
                              q=none(0, 4, 64)).shape == (0, 4, 64)
    for D in (64, 40):
        for width, slots in ((0, 8), (4, 0)):
            st = gpu(state([3, 0], torch.zeros(2, width, dtype=torch.int32)))
            ck, cv = none(slots, 2, D), none(slots, 2, D)
            out, lse = ops.paged_decode(randn(torch.Generator().manual_seed(1), 2, 4, D).cuda(), st, ck, cv, return_lse=True)
            assert (out == 0).all() and (lse == -math.inf).all()
            assert ops.kernel_status() in (5, 7)
            ops.kv_rope_append(none(2, 2, D), none(2, 2, D), st, ck, cv, none(D // 2, dtype=torch.float32))
            assert (ck == 0).all() and ops.kernel_status() in (5, 7)
    y = randn(torch.Generator().manual_seed(2), 5, 48).cuda()
    for n_in in (64, 61):
        for cu in (None, torch.tensor([0, 2, 2, 4, 4, 4], dtype=torch.int32).cuda()):
            got = ops.adapter_add(y, none(5, n_in), none(0, n_in, 8), none(0, 8, 48), torch.full((5,), -1, dtype=torch.int32, device="cuda"), cu_new=cu)
            assert torch.equal(got, y)
            assert ops.adapter_add(none(0, 48), none(0, n_in), none(2, n_in, 8), none(2, 8, 48), none(0, dtype=torch.int32),
                                   cu_new=None if cu is None else none(1, dtype=torch.int32)).shape == (0, 48)


@pytest.mark.parametrize("D", [64, 40])
def test_paged_batches_of_tens_of_thousands(D):
    """One token each: out is its value row (weight one, a rounding of a sum of one term)."""
    g = torch.Generator().manual_seed(34)
    B = 40000
    q, k, v = randn(g, B, 2, D), randn(g, B, 1, D), randn(g, B, 1, D)
    table = torch.randperm(B, generator=g).to(torch.int32)[:, None].contiguous()
    got = ops.paged_decode(q.cuda(), gpu(state([1] * B, table)), k.cuda(), v.cuda()).cpu()
    want = v[table[:, 0].long()].expand(B, 2, D)
    assert ((got.double() - want.double()).abs() <= (2.0 ** -11 + 2.0 ** -17) * want.double().abs() + 2.0 ** -24).all()


def test_two_streams_at_once():
    """Calls that run side by side have workspaces of their own."""
    g = torch.Generator().manual_seed(35)
    lens = [9000, 20, 4000]
    table, T = pages(3, 9000, 16, g)
    st = gpu(state(lens, table))
    k, v = randn(g, T, 2, 128).cuda(), randn(g, T, 2, 128).cuda()
    qs = [randn(g, 3, 8, 128).cuda() for _ in range(2)]
    x, y = randn(g, 3, 512).cuda(), randn(g, 3, 256).cuda()
    a, b = randn(g, 2, 512, 16, scale=0.05).cuda(), randn(g, 2, 16, 256).cuda()
    ads = [torch.tensor(t, dtype=torch.int32).cuda() for t in ([0, 1, 0], [1, -1, 1])]
    want = [(ops.paged_decode(q, st, k, v), ops.adapter_add(y, x, a, b, ad)) for q, ad in zip(qs, ads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.paged_decode(qs[i], st, k, v), ops.adapter_add(y, x, a, b, ads[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for o, z in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(z, want[i][1])


def test_ops_on_another_stream():
    g = torch.Generator().manual_seed(23)
    table, T = pages(2, 500, 16, g)
    st = gpu(state([500, 77], table))
    q, k, v = randn(g, 2, 8, 128).cuda(), randn(g, T, 2, 128).cuda(), randn(g, T, 2, 128).cuda()
    want = ops.paged_decode(q, st, k, v)
    x, y, a, b = randn(g, 9, 64).cuda(), randn(g, 9, 64).cuda(), randn(g, 1, 64, 8).cuda(), randn(g, 1, 8, 64).cuda()
    ad = torch.zeros(9, dtype=torch.int32).cuda()
    want_y = ops.adapter_add(y, x, a, b, ad)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(10):
        got = ops.paged_decode(q, st, k, v, stream=other)
        got_y = ops.adapter_add(y, x, a, b, ad, stream=other)
        noise = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(4)]  # takes freed memory at once
        other.synchronize()
        assert torch.equal(got, want) and torch.equal(got_y, want_y)
        del noise


def test_the_long_way_round_gives_the_same():
    """An allocator of the caller's, a stream of the caller's: not csrc/bind.cpp's ordinary call."""
    g = torch.Generator().manual_seed(24)
    table, T = pages(3, 90, 16, g)
    st = gpu(state([90, 7, 0], table))
    q, k, v = randn(g, 3, 8, 128).cuda(), randn(g, T, 2, 128).cuda(), randn(g, T, 2, 128).cuda()
    mine = lambda shape, dtype, device: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
    out, lse = ops.paged_decode(q, st, k, v, return_lse=True, window=50)
    out2, lse2 = ops.paged_decode(q, st, k, v, return_lse=True, window=50, alloc_tensor_func=mine)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    x, y, a, b = randn(g, 9, 64).cuda(), randn(g, 9, 64).cuda(), randn(g, 2, 64, 8).cuda(), randn(g, 2, 8, 64).cuda()
    ad = torch.tensor([0, 1, -1, 1, 0, 0, 1, 1, 0], dtype=torch.int32).cuda()
    assert torch.equal(ops.adapter_add(y, x, a, b, ad), ops.adapter_add(y, x, a, b, ad, alloc_tensor_func=mine))
    new = state([3, 0, 50], table)
    inv = torch.rand(64, generator=g).cuda()
    kk, vv = randn(g, 3, 2, 128).cuda(), randn(g, 3, 2, 128).cuda()
    caches = [(k.clone(), v.clone()) for _ in range(2)]
    here = torch.cuda.current_stream()
    got = [ops.kv_rope_append(kk, vv, gpu(new), *c, inv, q=q, **kw) for c, kw in zip(caches, ({}, dict(stream=here)))]
    assert torch.equal(got[0], got[1]) and all(torch.equal(a, b) for a, b in zip(*caches))


@pytest.mark.parametrize("call", ["append", "paged", "adapter"])
def test_refusals_on_the_gpu_launch_nothing(call):
    g = torch.Generator().manual_seed(25)
    table, T = pages(2, 8, 4, g)
    st = gpu(state([1, 2], table))
    z = lambda *s: torch.zeros(*s, dtype=F16, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="must be a CUDA tensor|expected cuda"):
        if call == "append":
            ops.kv_rope_append(z(2, 2, 16), z(2, 2, 16), st, z(T, 2, 16), z(T, 2, 16), torch.ones(8))
        elif call == "paged":
            ops.paged_decode(z(2, 4, 16), st, z(T, 2, 16).cpu(), z(T, 2, 16))
        else:
            ops.adapter_add(z(2, 8), z(2, 8), z(1, 8, 4), z(1, 4, 8), torch.zeros(2, dtype=torch.int32))
    if call == "paged":
        with pytest.raises(Exception, match="workspace"):
            ops.paged_decode(z(2, 4, 128), st, z(T, 2, 128), z(T, 2, 128), workspace=torch.zeros(4, device="cuda"))
