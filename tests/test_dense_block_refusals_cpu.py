"""What the dense attention block's operators refuse beyond tests/test_dense_block_cpu.py: both ways of a call, without a GPU."""
import ctypes
import random

import pytest
import torch

from tests.dense_block import pages, state
from tests.test_dense_block_cpu import FAKE, H16, _adapter_params, _adapters, _append, _bind_args, _paged, _paged_params
from wsvd_b200 import _lib, ops

CALLS = {"append": _append, "paged": _paged, "adapter": _adapters}


def refused(op, match, exc=ValueError, **kw):
    assert not getattr(_lib.bind(), op + "_fits")(*_bind_args(op, kw))
    with pytest.raises(exc, match=match):
        CALLS[op](**kw)()


def accepted(op, **kw):
    """Nothing but the device is wrong with the call."""
    assert getattr(_lib.bind(), op + "_fits")(*_bind_args(op, kw))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        CALLS[op](**kw)()


# ------------------------------------------------------------------ outputs over inputs

def test_a_shifted_output_is_refused():
    """y = buf[:-1], out = buf[1:]: blocks would write rows of y that others have yet to read."""
    rows = torch.zeros(4, 24, dtype=H16)
    refused("adapter", "out may be y itself", y=rows[:-1], out=rows[1:])
    refused("adapter", "out may be y itself", y=rows[1:], out=rows[:-1])
    flat = torch.zeros(3 * 24 + 8, dtype=H16)
    refused("adapter", "out may be y itself", y=flat[:72].view(3, 24), out=flat[8:].view(3, 24))
    tokens = torch.zeros(3, 4, 16, dtype=H16)
    refused("append", "q_out may be q itself", q=tokens[:-1], q_out=tokens[1:])
    refused("append", "q_out may be q itself", q=tokens[:2], q_out=tokens[:2].flatten().view(4, 2, 16).transpose(0, 1))
    refused("paged", "out may be q itself", q=tokens[1:], out=tokens[:-1])


def test_an_output_over_another_input_is_refused():
    qkv = torch.zeros(2, 8 * 16, dtype=H16)
    q, k, v = (qkv[:, a:b].unflatten(1, (-1, 16)) for a, b in ((0, 64), (64, 96), (96, 128)))
    refused("append", "must not overlap k", q=q, k=k, v=v, q_out=qkv[:, 64:].unflatten(1, (-1, 16)))
    refused("append", "must not overlap v", q=torch.zeros_like(q), v=v, q_out=qkv[:, 64:].unflatten(1, (-1, 16)))
    x = torch.zeros(3, 16 + 24, dtype=H16)
    refused("adapter", "must not overlap x", x=x[:, :16], out=x[:, 15:39])
    a = torch.zeros(2, 16, 4, dtype=H16)
    refused("adapter", "must not overlap a", a=a, out=a.flatten()[:72].view(3, 24))
    b = torch.zeros(2, 4, 24, dtype=H16)
    refused("adapter", "must not overlap b", b=b, out=b[1, 1:])
    table, T = pages(2, 8, 4, torch.Generator().manual_seed(1))
    cache = torch.zeros(T, 2, 16, dtype=H16)
    for name in ("cache_k", "cache_v"):
        refused("paged", "must not overlap " + name, out=cache[2:6].view(2, 4, 16), **{name: cache})


def test_outputs_beside_inputs_in_one_buffer_are_served():
    """Disjoint columns, heads or halves of one buffer, and an input itself."""
    qkv = torch.zeros(2, 12 * 16, dtype=H16)
    cut = [qkv[:, a * 16:b * 16].unflatten(1, (-1, 16)) for a, b in ((0, 4), (4, 6), (6, 8), (8, 12))]
    accepted("append", q=cut[0], k=cut[1], v=cut[2], q_out=cut[3])
    accepted("append", q=cut[0], k=cut[1], v=cut[2], q_out=cut[0])
    by_head = torch.zeros(2, 2, 3, 16, dtype=H16)  # q, k and v of a head side by side
    q, k, v = by_head.unbind(2)
    accepted("append", q=q, k=k, v=v, q_out=q)
    outside = torch.zeros(8, 2, 16, dtype=H16).transpose(0, 1)  # heads outside
    accepted("append", q=outside[:, :4], k=outside[:, 4:6], v=outside[:, 6:], q_out=outside[:, :4])
    both = torch.zeros(3, 48, dtype=H16)
    accepted("adapter", y=both[:, :24], out=both[:, 24:])
    accepted("adapter", y=both[:, :24], out=both[:, :24])
    every = torch.zeros(6, 24, dtype=H16)
    accepted("adapter", y=every[::2], out=every[1::2])
    accepted("adapter", y=every[:3], out=every[3:])
    one = torch.zeros(1, 64, dtype=H16)  # one row: its stride is nobody's
    accepted("adapter", x=torch.zeros(1, 16, dtype=H16), adapter=torch.zeros(1, dtype=torch.int32), y=one[:, :24], out=one.as_strided((1, 24), (24, 1)))
    q = torch.zeros(2, 4, 16, dtype=H16)
    accepted("paged", q=q, out=q)


def test_views_of_one_buffer_meet_where_their_elements_do():
    rng = random.Random(7)
    buf = torch.zeros(4000, dtype=H16)
    where = torch.arange(4000)
    met = 0
    for _ in range(1500):
        views = []
        pitch = [rng.choice([1, 2, 3, 8]), rng.choice([8, 24, 40, 41]), rng.choice([80, 200, 206])]
        for _ in range(2):
            if rng.random() < 0.15:
                pitch = [rng.randint(0, 6), rng.randint(0, 50), rng.randint(0, 220)]
            shape = [rng.randint(0 if rng.random() < 0.02 else 1, 5) for _ in range(3)]
            views.append((shape, [pitch[2], pitch[1], pitch[0]], rng.randint(0, 300)))
        a, b = (buf.as_strided(*v) for v in views)
        want = bool(set(where.as_strided(*views[0]).flatten().tolist()) & set(where.as_strided(*views[1]).flatten().tolist()))
        got = ops._meet(a, b)
        assert got == want or (got and not want and views[0][1] != views[1][1]), views  # (long searches count as met)
        assert ops._meet(b, a) == got
        met += want
    assert 200 < met < 1300


def test_both_ways_of_a_call_refuse_the_same_views():
    rng = random.Random(11)
    buf = torch.zeros(600, dtype=H16)
    seen = {True: 0, False: 0}
    for _ in range(400):
        pitch = rng.choice([24, 25, 32, 48, 56])
        y = buf.as_strided((3, 24), (pitch, 1), rng.randint(0, 100))
        out = buf.as_strided((3, 24), (pitch if rng.random() < 0.8 else 40, 1), rng.randint(0, 250))
        fits = _lib.bind().adapter_fits(*_bind_args("adapter", dict(y=y, out=out)))
        with pytest.raises(ValueError) as error:
            _adapters(y=y, out=out)()
        assert fits == ("CUDA tensor" in str(error.value)), (y.stride(), out.stride(), y.storage_offset(), out.storage_offset(), error.value)
        seen[fits] += 1
    assert min(seen.values()) > 50


# ------------------------------------------------------------------ derivatives

def test_forward_mode_tangents_are_refused_under_no_grad_too():
    def dual(*shape, dtype=H16):
        t = torch.zeros(*shape, dtype=dtype)
        return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

    table, T = pages(2, 8, 4, torch.Generator().manual_seed(1))
    store, scale = torch.zeros(T, 2, 16, dtype=torch.int8), torch.ones(T, 2, dtype=H16)
    with torch.autograd.forward_ad.dual_level():
        calls = [("append", dict(k=dual(2, 2, 16))), ("append", dict(v=dual(2, 2, 16))), ("append", dict(q=dual(2, 4, 16))),
                 ("append", dict(inv_freq=dual(8, dtype=torch.float32))),
                 ("paged", dict(q=dual(2, 4, 16))), ("paged", dict(cache_v=dual(T, 2, 16))),
                 ("paged", dict(cache_k=store, cache_v=store, k_scale=scale, v_scale=dual(T, 2))),
                 ("adapter", dict(x=dual(3, 16))), ("adapter", dict(y=dual(3, 24))), ("adapter", dict(a=dual(2, 16, 4))),
                 ("adapter", dict(b=dual(2, 4, 24))), ("adapter", dict(scale=dual(2, dtype=torch.float32)))]
        for op, kw in calls:
            refused(op, "no forward-mode derivative", **kw)
            with torch.no_grad():
                refused(op, "no forward-mode derivative", **kw)
        accepted("adapter", x=torch.autograd.forward_ad.unpack_dual(dual(3, 16)).primal)


# ------------------------------------------------------------------ sizes

def test_sizes_beyond_32_bits_are_refused_not_cut():
    """2^32 + 3 rows would be 3 (tensors of one element's memory)."""
    many = 2 ** 32 + 3
    cu = torch.zeros(3, dtype=torch.int32)
    rows = torch.zeros(1, 2, 16, dtype=H16).expand(many, 2, 16)
    refused("append", "rows of k", k=rows, v=rows, cu_new=cu)
    none = torch.zeros(2, 0, 16, dtype=H16)
    heads = torch.zeros(2, 1, 16, dtype=H16).expand(2, many, 16)
    refused("append", "heads of q", q=heads)
    refused("append", "heads of k", k=heads, v=heads, cache_k=heads, cache_v=heads)
    refused("paged", "heads of q", q=torch.zeros(2, 1, 16, dtype=H16).expand(2, 2 ** 32 + 4, 16))
    table = torch.zeros(1, 8, dtype=torch.int32).expand(many, 8)
    refused("append", "rows of req_to_token_indexs", infer_state=state([1, 2], table))
    refused("paged", "rows of req_to_token_indexs", infer_state=state([1, 2], table))
    two = torch.zeros(2, dtype=torch.int32)
    refused("adapter", "rows of x", x=torch.zeros(1, 16, dtype=H16).expand(many, 16), y=torch.zeros(1, 24, dtype=H16).expand(many, 24),
            adapter=two, cu_new=cu)
    refused("adapter", "adapters", a=torch.zeros(1, 16, 4, dtype=H16).expand(many, 16, 4), b=torch.zeros(1, 4, 24, dtype=H16).expand(many, 4, 24))
    accepted("append", q=none)


def test_lengths_that_a_last_step_would_carry_past_32_bits_are_refused():
    """A page table of 2^31 - 1 columns: the step behind the last position would count on from below zero."""
    lib = _lib.lib()
    for most, status in ((2 ** 31 - 1, 8), (2 ** 31 - 1024, 8)):
        assert lib.wsvd_paged_decode(ctypes.byref(_paged_params(max_len=most)), FAKE, 1 << 60, None) == status
        for kw in (dict(rows=most), dict(batch=most), dict(n_in=most), dict(rows=most, batch=most, cu_new=None)):
            assert lib.wsvd_adapter_add(ctypes.byref(_adapter_params(**kw)), FAKE, 1 << 60, None) == status
    assert lib.wsvd_adapter_add(ctypes.byref(_adapter_params(n_out=2 ** 31 - 1)), FAKE, 1 << 60, None) == 8


def test_outputs_over_one_another_are_refused():
    """Keys and values of a token would go to one place."""
    table, T = pages(2, 8, 4, torch.Generator().manual_seed(1))
    cache = torch.zeros(T + 1, 2, 16, dtype=H16)
    refused("append", "cache_k and cache_v overlap", cache_k=cache[1:], cache_v=cache[1:])
    refused("append", "cache_k and cache_v overlap", cache_k=cache[1:], cache_v=cache[:-1])
    q = torch.zeros(2, 4, 16, dtype=H16)
    refused("append", "q_out and cache_k overlap", cache_k=cache[1:], q=q, q_out=cache[3:7].view(2, 4, 16))
    refused("append", "q_out and cache_v overlap", cache_v=cache[1:], q=q, q_out=cache[3:7].view(2, 4, 16))
    both = torch.zeros(T, 2, 2, 16, dtype=H16)
    accepted("append", cache_k=both[:, 0], cache_v=both[:, 1])
    accepted("append", cache_k=both[:, :, 0], cache_v=both[:, :, 1])
    halves = torch.zeros(2 * T, 2, 16, dtype=H16)
    accepted("append", cache_k=halves[:T], cache_v=halves[T:])
    accepted("append", cache_k=halves[::2], cache_v=halves[1::2])
