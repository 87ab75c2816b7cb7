"""kv_rope_append, paged_decode and adapter_add without a GPU: what they refuse, and the C entries' status codes."""
import ctypes

import pytest
import torch

from tests.dense_block import append64, attend64, pages, state
from wsvd_b200 import _lib, ops

H16 = torch.float16


def _append(**kw):
    g = torch.Generator().manual_seed(1)
    table, T = pages(2, 8, 4, g)
    a = dict(k=torch.zeros(2, 2, 16, dtype=H16), v=torch.zeros(2, 2, 16, dtype=H16), infer_state=state([1, 2], table),
             cache_k=torch.zeros(T, 2, 16, dtype=H16), cache_v=torch.zeros(T, 2, 16, dtype=H16), inv_freq=torch.ones(8))
    a.update(kw)
    return lambda: ops.kv_rope_append(a.pop("k"), a.pop("v"), a.pop("infer_state"), a.pop("cache_k"), a.pop("cache_v"),
                                      a.pop("inv_freq"), **a)


def _paged(**kw):
    g = torch.Generator().manual_seed(1)
    table, T = pages(2, 8, 4, g)
    a = dict(q=torch.zeros(2, 4, 16, dtype=H16), infer_state=state([1, 2], table), cache_k=torch.zeros(T, 2, 16, dtype=H16),
             cache_v=torch.zeros(T, 2, 16, dtype=H16))
    a.update(kw)
    return lambda: ops.paged_decode(a.pop("q"), a.pop("infer_state"), a.pop("cache_k"), a.pop("cache_v"), **a)


def _adapters(**kw):
    a = dict(y=torch.zeros(3, 24, dtype=H16), x=torch.zeros(3, 16, dtype=H16), a=torch.zeros(2, 16, 4, dtype=H16),
             b=torch.zeros(2, 4, 24, dtype=H16), adapter=torch.zeros(3, dtype=torch.int32))
    a.update(kw)
    return lambda: ops.adapter_add(a.pop("y"), a.pop("x"), a.pop("a"), a.pop("b"), a.pop("adapter"), **a)


def _bind_args(op, kw):
    """The arguments of csrc/bind.cpp's function for a call of `op`, in its order."""
    g = torch.Generator().manual_seed(1)
    table, T = pages(2, 8, 4, g)
    st = kw.get("infer_state") or state([1, 2], table)
    meta = [st.b_seq_len, st.b_req_idx, st.req_manager.req_to_token_indexs]
    if op == "append":
        d = dict(k=torch.zeros(2, 2, 16, dtype=H16), v=torch.zeros(2, 2, 16, dtype=H16), cache_k=torch.zeros(T, 2, 16, dtype=H16),
                 cache_v=torch.zeros(T, 2, 16, dtype=H16), inv_freq=torch.ones(8))
        d.update(kw)
        return [d["k"], d["v"], *meta, *(d.get(n) for n in ("cache_k", "cache_v", "inv_freq", "cache_k_scale", "cache_v_scale", "q", "q_out",
                                                           "cu_new", "pos_offset")), 0]
    if op == "paged":
        d = dict(q=torch.zeros(2, 4, 16, dtype=H16), cache_k=torch.zeros(T, 2, 16, dtype=H16), cache_v=torch.zeros(T, 2, 16, dtype=H16))
        d.update(kw)
        return [d["q"], *meta, *(d.get(n) for n in ("cache_k", "cache_v", "k_scale", "v_scale", "out", "workspace")), False,
                d.get("window", 0), 0.0]
    d = dict(y=torch.zeros(3, 24, dtype=H16), x=torch.zeros(3, 16, dtype=H16), a=torch.zeros(2, 16, 4, dtype=H16),
             b=torch.zeros(2, 4, 24, dtype=H16), adapter=torch.zeros(3, dtype=torch.int32))
    d.update(kw)
    return [d.get(n) for n in ("y", "x", "a", "b", "adapter", "scale", "cu_new", "out", "workspace")]


def _fits(op, **kw):
    return getattr(_lib.bind(), op + "_fits")(*_bind_args(op, kw))


def test_ordinary_calls_fit_and_no_cpu_tensor_is_launched_on():
    g = torch.Generator().manual_seed(1)
    i8 = dict(cache_k=_i8(20, 2, 16), cache_v=_i8(20, 2, 16))
    sc = torch.zeros(20, 2, dtype=H16)
    q = torch.zeros(2, 4, 16, dtype=H16)
    for kw in ({}, dict(q=q), dict(q=q, q_out=q), dict(cu_new=torch.zeros(3, dtype=torch.int32)), dict(pos_offset=torch.zeros(2, dtype=torch.int32)),
               dict(cache_k_scale=sc, cache_v_scale=sc, **i8), dict(inv_freq=torch.ones(0))):
        assert _fits("append", **kw), kw
        assert _lib.bind().append(*_bind_args("append", kw)) is None
    for kw in ({}, dict(out=q), dict(window=5), dict(k_scale=sc, v_scale=sc, **i8), dict(workspace=torch.zeros(4))):
        assert _fits("paged", **kw), kw
        assert _lib.bind().paged(*_bind_args("paged", kw)) is None
    for kw in ({}, dict(scale=torch.ones(2)), dict(adapter=torch.zeros(2, dtype=torch.int32), cu_new=torch.zeros(3, dtype=torch.int32))):
        assert _fits("adapter", **kw), kw
        assert _lib.bind().adapter(*_bind_args("adapter", kw)) is None
    y = torch.zeros(3, 24, dtype=H16)
    assert _fits("adapter", y=y, out=y)


def _i8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


@pytest.mark.parametrize("call", [_append(), _paged(), _adapters()])
def test_a_valid_call_without_a_gpu_is_refused_for_the_device_alone(call):
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        call()


@pytest.mark.parametrize("kw,exc,match", [
    (dict(k=torch.zeros(2, 2, 16)), TypeError, "k has dtype"),
    (dict(v=torch.zeros(2, 2, 16, dtype=torch.bfloat16)), TypeError, "v has dtype"),
    (dict(v=torch.zeros(2, 1, 16, dtype=H16)), ValueError, "one shape"),
    (dict(k=torch.zeros(2, 16, 2, dtype=H16).transpose(1, 2)), ValueError, "innermost"),
    (dict(k=torch.zeros(2, 16, dtype=H16)), ValueError, "3 dims"),
    (dict(k=[1]), TypeError, "torch.Tensor"),
    (dict(inv_freq=torch.ones(9)), ValueError, "frequencies"),
    (dict(inv_freq=torch.ones(8, dtype=torch.float64)), TypeError, "inv_freq"),
    (dict(cache_k=_i8(32, 2, 16)), TypeError, "cache_v has dtype"),
    (dict(cache_k=_i8(32, 2, 16), cache_v=_i8(32, 2, 16)), TypeError, "scales"),
    (dict(cache_k=_i8(32, 2, 16), cache_v=_i8(32, 2, 16), cache_k_scale=torch.zeros(32, 2), cache_v_scale=torch.zeros(32, 2)),
     TypeError, "scale has dtype"),
    (dict(cache_k=_i8(32, 2, 16), cache_v=_i8(32, 2, 16), cache_k_scale=torch.zeros(31, 2, dtype=H16),
          cache_v_scale=torch.zeros(32, 2, dtype=H16)), ValueError, "scale must be"),
    (dict(cache_k_scale=torch.zeros(32, 2, dtype=H16)), TypeError, "only int8"),
    (dict(cache_v=torch.zeros(3, 2, 16, dtype=H16)), ValueError, r"\[T, 2, 16\]"),
    (dict(cu_new=torch.zeros(2, dtype=torch.int32)), ValueError, "one entry per sequence"),
    (dict(cu_new=torch.zeros(0, dtype=torch.int32)), ValueError, "cu_new"),
    (dict(cu_new=torch.zeros(3)), TypeError, "cu_new"),
    (dict(pos_offset=torch.zeros(3, dtype=torch.int32)), ValueError, "pos_offset"),
    (dict(rope_layout="other"), ValueError, "rope_layout"),
    (dict(q=torch.zeros(2, 4, 8, dtype=H16)), ValueError, "q must be"),
    (dict(q_out=torch.zeros(2, 4, 16, dtype=H16)), ValueError, "without q"),
    (dict(q=torch.zeros(2, 4, 16, dtype=H16), q_out=torch.zeros(2, 4, 8, dtype=H16)), ValueError, "q_out must be"),
    (dict(k=torch.zeros(2, 2, 16, dtype=H16, requires_grad=True)), ValueError, "no backward"),
])
def test_append_refusals(kw, exc, match):
    assert "rope_layout" in kw or not _fits("append", **kw)
    with pytest.raises(exc, match=match):
        _append(**kw)()


def test_append_refuses_a_shifted_view_as_q_out():
    buf = torch.zeros(2, 4, 32, dtype=H16)
    kw = dict(q=buf[..., :16], q_out=buf.view(-1)[:128].view(2, 4, 16))
    assert not _fits("append", **kw)
    with pytest.raises(ValueError, match="another view"):
        _append(**kw)()


@pytest.mark.parametrize("kw,exc,match", [
    (dict(q=torch.zeros(2, 4, 16)), TypeError, "q has dtype"),
    (dict(q=torch.zeros(2, 3, 16, dtype=H16)), ValueError, "multiple"),
    (dict(q=torch.zeros(2, 4, 512, dtype=H16)), ValueError, "head_dim"),
    (dict(q=torch.zeros(2, 4, 32, dtype=H16)), ValueError, r"\[T, 2, 32\]"),
    (dict(q=torch.zeros(3, 4, 16, dtype=H16)), ValueError, "one entry per sequence"),
    (dict(cache_k=torch.zeros(32, 2, 16, dtype=torch.bfloat16)), TypeError, "cache_k has dtype"),
    (dict(cache_k=_i8(32, 2, 16), cache_v=_i8(32, 2, 16)), TypeError, "scales"),
    (dict(out=torch.zeros(2, 4, 8, dtype=H16)), ValueError, "out must be"),
    (dict(window=-1), ValueError, "window"),
    (dict(workspace=torch.zeros(4, 4).t()[:2]), ValueError, "contiguous"),
    (dict(q=torch.zeros(2, 4, 16, dtype=H16, requires_grad=True)), ValueError, "no backward"),
])
def test_paged_decode_refusals(kw, exc, match):
    assert not _fits("paged", **kw)
    with pytest.raises(exc, match=match):
        _paged(**kw)()


@pytest.mark.parametrize("kw,exc,match", [
    (dict(x=torch.zeros(3, 16)), TypeError, "x has dtype"),
    (dict(y=torch.zeros(3, 24, dtype=torch.bfloat16)), TypeError, "y has dtype"),
    (dict(y=torch.zeros(2, 24, dtype=H16)), ValueError, "same rows"),
    (dict(a=torch.zeros(2, 15, 4, dtype=H16)), ValueError, "a must be"),
    (dict(b=torch.zeros(1, 4, 24, dtype=H16)), ValueError, "a must be"),
    (dict(a=torch.zeros(2, 16, 257, dtype=H16), b=torch.zeros(2, 257, 24, dtype=H16)), ValueError, "rank 257"),
    (dict(a=torch.zeros(2, 16, 0, dtype=H16), b=torch.zeros(2, 0, 24, dtype=H16)), ValueError, "rank 0"),
    (dict(adapter=torch.zeros(3)), TypeError, "adapter has dtype"),
    (dict(adapter=torch.zeros(2, dtype=torch.int32)), ValueError, "one entry per row"),
    (dict(cu_new=torch.zeros(3, dtype=torch.int32)), ValueError, "cu_new"),
    (dict(scale=torch.zeros(3)), ValueError, "scale"),
    (dict(scale=torch.zeros(2, dtype=H16)), TypeError, "scale"),
    (dict(out=torch.zeros(3, 23, dtype=H16)), ValueError, "out must be"),
    (dict(b=torch.zeros(2, 4, 24, dtype=H16, requires_grad=True)), ValueError, "no backward"),
])
def test_adapter_refusals(kw, exc, match):
    assert not _fits("adapter", **kw)
    with pytest.raises(exc, match=match):
        _adapters(**kw)()


def test_adapter_refuses_a_shifted_view_as_out():
    y = torch.zeros(3, 24, dtype=H16)
    assert not _fits("adapter", y=y, out=y.as_strided((3, 24), (1, 1)))
    with pytest.raises(ValueError, match="another view"):
        _adapters(y=y, out=y.as_strided((3, 24), (1, 1)))()


# ---- the C entries: a status before any CUDA call

FAKE = 0x10000  # never dereferenced on the host


def _filled(cls, **kw):
    p = cls()
    for name, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(p, name, FAKE)
    p.dtype = 1
    for n, v in kw.items():
        setattr(p, n, v)
    return p


def _append_params(**kw):
    return _filled(_lib.KvRopeAppendParams, **{**dict(rows=2, batch=2, n_q_heads=4, n_kv_heads=2, head_dim=16, rot_dim=16, max_len=8,
                                                      n_req=2, cache_dtype=1, n_token_slots=32), **kw})


def _paged_params(**kw):
    return _filled(_lib.PagedDecodeParams, **{**dict(batch=2, n_q_heads=4, n_kv_heads=2, head_dim=128, max_len=8, n_req=2,
                                                     cache_dtype=1, n_token_slots=32), **kw})


def _adapter_params(**kw):
    return _filled(_lib.AdapterAddParams, **{**dict(rows=2, batch=2, n_in=64, n_out=64, rank=8, n_adapters=2), **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), 2), (dict(n_kv_heads=0), 2), (dict(head_dim=15), 2), (dict(head_dim=258), 2), (dict(rot_dim=18), 2),
    (dict(rot_dim=3), 2), (dict(dtype=2), 3), (dict(cache_dtype=3), 3), (dict(rope_layout=2), 3),
    (dict(cu_new=None, rows=3), 2), (dict(k=None), 1), (dict(inv_freq=None), 1), (dict(q_out=None), 1),
    (dict(cache_dtype=0, v_scale=None), 3), (dict(rows=1 << 30), 8), (dict(rows=0), 0)])
def test_append_status(kw, status):
    assert _lib.lib().wsvd_kv_rope_append(ctypes.byref(_append_params(**kw)), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 2), (dict(n_kv_heads=3), 2), (dict(head_dim=0), 2), (dict(head_dim=257), 2), (dict(window=-1), 2),
    (dict(dtype=0), 3), (dict(cache_dtype=3), 3), (dict(batch=70000), 8), (dict(q=None), 1), (dict(b_req_idx=None), 1),
    (dict(cache_dtype=0, k_scale=None), 3), (dict(batch=0), 0)])
def test_paged_decode_status(kw, status):
    assert _lib.lib().wsvd_paged_decode(ctypes.byref(_paged_params(**kw)), FAKE, 1 << 40, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), 2), (dict(n_in=0), 2), (dict(rank=0), 2), (dict(rank=257), 2), (dict(dtype=2), 3),
    (dict(cu_new=None, rows=3), 2), (dict(x=None), 1), (dict(adapter=None), 1), (dict(rows=0), 0)])
def test_adapter_status(kw, status):
    assert _lib.lib().wsvd_adapter_add(ctypes.byref(_adapter_params(**kw)), FAKE, 1 << 40, None) == status


def test_workspace_checks():
    lib = _lib.lib()
    for name, p in (("wsvd_adapter_add", _adapter_params()), ("wsvd_paged_decode", _paged_params(max_len=8192, n_q_heads=8))):
        need = getattr(lib, name + "_workspace_bytes")(ctypes.byref(p))
        if need == 0:
            continue
        call = getattr(lib, name)
        assert call(ctypes.byref(p), None, need, None) == 1
        assert call(ctypes.byref(p), FAKE, need - 1, None) == 5
        assert call(ctypes.byref(p), FAKE + 4, need, None) == 4
        assert call(None, FAKE, need, None) == 1


@pytest.mark.parametrize("cls", [_lib.KvRopeAppendParams, _lib.PagedDecodeParams, _lib.AdapterAddParams])
def test_packed_bytes_are_the_structure(cls):
    values = [float(i) if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
    p = cls.from_buffer_copy(_lib.packer(cls)(*values))
    assert [getattr(p, n) for n, _ in cls._fields_] == values


# ---- the oracle on bad pages and empty sequences, before a kernel sees them

def test_the_oracle_leaves_out_what_does_not_exist():
    g = torch.Generator().manual_seed(2)
    table, T = pages(2, 6, 2, g)
    table[0, 1], table[1, 0] = T, -1
    st = state([3, 9, 0], table, idx=[0, 1, 5])
    k, v = torch.randn(T, 1, 8, generator=g).half(), torch.randn(T, 1, 8, generator=g).half()
    q = torch.randn(3, 2, 8, generator=g).half()
    out, lse, _, _ = attend64(q, st, k, v, None, None, 0, 0.0)
    slots = table[0, [0, 2]].long()
    z = k[slots, 0].double() @ q[0, 0].double() / 8 ** 0.5
    assert torch.allclose(out[0, 0], torch.softmax(z, 0) @ v[slots, 0].double())
    assert (out[2] == 0).all() and (lse[2] == -float("inf")).all()
    stored, turned = append64(k[:3], v[:3], q, state([1, 6, 0], table, idx=[0, 1, 5]), None, torch.ones(4), None, "half", T)
    assert not stored and len(turned) == 3


def _bytes(T=None):
    table, T = pages(2, 8, 4, torch.Generator().manual_seed(1))
    store, scale = torch.zeros(T, 2, 16, dtype=torch.int8), torch.ones(T, 2, dtype=H16)
    return dict(cache_k=store, cache_v=store.clone()), scale


def test_gradients_of_the_small_arguments_are_refused_too():
    caches, scale = _bytes()
    wanted = scale.clone().requires_grad_()
    calls = [("append", _append, dict(inv_freq=torch.ones(8, requires_grad=True))),
             ("append", _append, dict(**caches, cache_k_scale=wanted, cache_v_scale=scale)),
             ("paged", _paged, dict(**caches, k_scale=scale, v_scale=wanted)),
             ("adapter", _adapters, dict(scale=torch.ones(2, requires_grad=True)))]
    for op, call, kw in calls:
        assert not getattr(_lib.bind(), op + "_fits")(*_bind_args(op, kw))
        with pytest.raises(ValueError, match="no backward"):
            call(**kw)()


def test_outputs_whose_elements_share_memory_are_refused():
    caches, scale = _bytes()
    T = scale.shape[0]
    calls = [("append", _append, dict(q=torch.zeros(2, 4, 16, dtype=H16), q_out=torch.zeros(1, 4, 16, dtype=H16).expand(2, 4, 16))),
             ("append", _append, dict(cache_k=torch.zeros(T, 1, 16, dtype=H16).expand(T, 2, 16))),
             ("append", _append, dict(**caches, cache_k_scale=scale, cache_v_scale=scale[:1].expand(T, 2))),
             ("paged", _paged, dict(out=torch.zeros(2, 1, 16, dtype=H16).expand(2, 4, 16))),
             ("adapter", _adapters, dict(out=torch.zeros(1, 24, dtype=H16).expand(3, 24))),
             ("adapter", _adapters, dict(out=torch.zeros(72, dtype=H16).as_strided((3, 24), (16, 1))))]
    for op, call, kw in calls:
        assert not getattr(_lib.bind(), op + "_fits")(*_bind_args(op, kw))
        with pytest.raises(ValueError, match="share memory"):
            call(**kw)()
    # heads outside, tokens inside, and K beside V in one buffer are as good as any order
    both = torch.zeros(T, 2, 2, 16, dtype=H16)
    for kw in (dict(cache_k=both[:, 0], cache_v=both[:, 1]), dict(cache_k=torch.zeros(2, T, 16, dtype=H16).transpose(0, 1))):
        assert getattr(_lib.bind(), "append_fits")(*_bind_args("append", kw))
