"""The dense attention block's operators in 64 bits, a row at a time, with the bound of what each kernel may be off by.

A rounding to a type is off by at most half a step (`half_step`, relative); sums of n products in f32 by n 2^-24 of the sum
of their magnitudes."""
import math
from types import SimpleNamespace

import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def state(lens, table, idx=None, device="cpu"):
    idx = torch.arange(len(lens), dtype=torch.int32) if idx is None else torch.as_tensor(idx, dtype=torch.int32)
    return SimpleNamespace(batch_size=len(lens), max_len_in_batch=max([0, *lens]),
                           b_seq_len=torch.tensor(lens, dtype=torch.int32).to(device), b_req_idx=idx.to(device),
                           req_manager=SimpleNamespace(req_to_token_indexs=table.to(device)))


def pages(n_req, width, page, gen, spare=3):
    """[n_req, width] token slots handed out page by page in a shuffled order, and the number of slots."""
    per = max(1, (width + page - 1) // page)
    perm = torch.randperm(n_req * per + spare, generator=gen)[:n_req * per]
    table = (perm[:, None] * page + torch.arange(page)[None, :]).reshape(n_req, per * page)[:, :width]
    return table.to(torch.int32).contiguous(), (n_req * per + spare) * page


def quantize(x):
    """int8 rows and f16 scales of x (f64), and the values that they stand for."""
    amax = x.abs().amax(dim=-1)
    s = torch.where(amax > 0, amax / 127, torch.ones_like(amax)).half()
    q = (x / s.double()[..., None]).round().clamp(-128, 127)
    return q.to(torch.int8), s


def rotate64(x, place, inv_freq, layout):
    """x [heads, D] in f64 at one position."""
    half = inv_freq.numel()
    ang = float(place) * inv_freq.double()
    c, s = ang.cos(), ang.sin()
    y = x.clone()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[:, a] = x[:, a] * c - x[:, b] * s
    y[:, b] = x[:, b] * c + x[:, a] * s
    return y


def rows_of(cu, n):
    """(sequence, place in it) of each packed row, None for padding."""
    if cu is None:
        return [(i, 0) for i in range(n)]
    got = [None] * n
    for b in range(len(cu) - 1):
        for i in range(cu[b], cu[b + 1]):
            got[i] = (b, i - cu[b])
    return got


def slot_of(st, b, pos, slots):
    table = st.req_manager.req_to_token_indexs
    req = int(st.b_req_idx[b])
    if not 0 <= pos < table.shape[1] or not 0 <= req < table.shape[0]:
        return None
    slot = int(table[req, pos])
    return slot if 0 <= slot < slots else None


def append64(k, v, q, st, cu, inv_freq, offset, layout, slots):
    """{slot: (rotated k, v)} in f64, and the rotated queries (None where padding)."""
    stored, turned = {}, []
    for n, at in enumerate(rows_of(cu, k.shape[0])):
        if at is None:
            turned.append(None)
            continue
        b, i = at
        pos = int(st.b_seq_len[b]) + i
        place = pos + (0 if offset is None else int(offset[b]))
        turned.append(rotate64(q[n].double(), place, inv_freq, layout))
        slot = slot_of(st, b, pos, slots)
        if slot is not None:
            stored[slot] = (rotate64(k[n].double(), place, inv_freq, layout), v[n].double())
    return stored, turned


def assert_rotated(got, want, x, dtype, what):
    """A rotated row in `dtype`: one rounding of the result; in f32 three roundings of terms no larger than the pair's
    magnitude sum, and an angle that is off by at most pi 2^-24 (its f32 rounding) and two steps of sine and cosine."""
    pair = x.abs().max() * 2
    tol = half_step(dtype) * want.abs() + 10 * F32 * pair + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    assert ((got.double() - want).abs() <= tol).all(), (what, ((got.double() - want).abs() - tol).max().item())


def assert_held(q, s, want, what):
    """Bytes and scale of rows: the scale is one rounding to f16 of max|x| / 127 (and the f32 row's own error, 10 2^-24 of
    two magnitudes), the value that the bytes stand for at most half a scale off."""
    amax = want.abs().amax(dim=-1)
    ideal = torch.where(amax > 0, amax / 127, torch.ones_like(amax)).clamp(2.0 ** -24, 65504.0)
    tol = ideal * (2.0 ** -11 + 30 * F32) + 2.0 ** -25
    assert ((s.double() - ideal).abs() <= tol).all(), what
    off = (q.double() * s.double()[..., None] - want).abs()
    assert (off <= s.double()[..., None] * 0.5 + 30 * F32 * amax[..., None]).all(), (what, off.max().item())


def attend64(q, st, k, v, ks, vs, window, sm_scale):
    """out, lse and the bound of the kernels' error [B, Hq, D], [B, Hq] in f64."""
    B, Hq, D = q.shape
    T, Hkv = k.shape[:2]
    width = st.req_manager.req_to_token_indexs.shape[1]
    c = sm_scale or 1 / math.sqrt(D)
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    bound, lse_bound = torch.zeros_like(out), torch.zeros(B, Hq, dtype=torch.float64)
    for b in range(B):
        n = min(int(st.b_seq_len[b]), width)
        slots = [slot_of(st, b, s, T) for s in range(max(0, n - window) if window else 0, max(n, 0))]
        slots = torch.tensor([s for s in slots if s is not None], dtype=torch.long)
        if not len(slots):
            continue
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            kk, vv = k[slots, hk].double(), v[slots, hk].double()
            if ks is not None:
                kk, vv = kk * ks[slots, hk].double()[:, None], vv * vs[slots, hk].double()[:, None]
            qq = q[b, h].double()
            z = kk @ qq * c
            w = torch.softmax(z, dim=0)
            out[b, h], lse[b, h] = w @ vv, torch.logsumexp(z, dim=0)
            # a score: D products summed in f32 (and two more factors); a weight: e^z of that, an exponential within two steps
            # of f32 and, on the tensor cores, two 16-bit terms (2^-17 together); sums of len(slots) terms in f32
            dz = float((D + 4) * F32 * (kk.abs() @ qq.abs()).max() * c + 4 * F32 * z.abs().max())
            dw = 2 * dz + 4 * F32 + 2.0 ** -17
            n_sum = min(len(slots), 4096) * F32  # (partial sums of a few hundred terms, then a few tens of partials)
            bound[b, h] = half_step(q.dtype) * out[b, h].abs() + (dw * 2 + n_sum) * (w @ vv.abs()) + \
                torch.finfo(q.dtype).smallest_normal * half_step(q.dtype) * 2
            lse_bound[b, h] = dz + dw + n_sum + 4 * F32 * lse[b, h].abs()
    return out, lse, bound, lse_bound


def adapters64(y, x, a, b, adapter, scale, cu):
    """out (None rows: padding) and the bound of the kernels' error, f64."""
    out, bound = y.double().clone(), half_step(y.dtype) * y.double().abs()
    at = rows_of(cu, x.shape[0])
    for n, place in enumerate(at):
        if place is None:
            continue
        i = int(adapter[place[0]])
        if not 0 <= i < a.shape[0]:
            continue
        s = 1.0 if scale is None else float(scale[i])
        h = x[n].double() @ a[i].double()
        out[n] += s * (h @ b[i].double())
        habs = x[n].double().abs() @ a[i].double().abs()
        # the product x A: n_in terms in f32, then at most one rounding to the 16-bit type; h B: rank terms in f32
        err = (x.shape[1] + 4) * F32 * habs + half_step(y.dtype) * h.abs()
        r = a.shape[2]
        bound[n] = half_step(y.dtype) * out[n].abs() + abs(s) * (err @ b[i].double().abs() + (r + 4) * F32 * (habs @ b[i].double().abs())) + \
            torch.finfo(y.dtype).smallest_normal * half_step(y.dtype) * 2 + 2 * F32 * y[n].double().abs()
    return out, bound, [p is None for p in at]
