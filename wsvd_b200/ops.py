"""Tensor -> C-ABI marshalling for the latent decode-attention op.

The functions here take torch CUDA tensors, check the preconditions the reference
wrappers assert (efficiency/kernel/flash_int8_latent_per_head_decoding_rope_stage1.py:
231-243) and call libwsvd_b200.so on the current CUDA stream.  No CPU path exists.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import warnings
from typing import Callable, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import LatentDecodeParams, check

I8, F16 = 0, 1
ROPE = {"half": 0, "interleaved": 1}
KERNEL = {"auto": 0, "generic": 1, "tc": 2, "mma": 3}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _need(cond: bool, msg: str, exc=ValueError):
    if not cond:
        raise exc(msg)


def _cuda_tensor(name, t, dtypes, ndim, inner_contiguous=True):
    # (the messages are formatted only when they are needed: formatting them was most of a small call's host time)
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (no CPU path exists)")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got {tuple(t.shape)}")
    if inner_contiguous and t.stride(-1) != 1 and t.numel() != 0:
        raise ValueError(f"{name}: innermost dimension must be contiguous")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _on_device(device):
    """Context in which `device` is the current one; entered only where it is not already."""
    index = device.index
    return _HERE if index is None or index == torch.cuda.current_device() else torch.cuda.device(device)


_HERE = contextlib.nullcontext()
_TABLES = {}
_RETIRED_TABLES = []  # superseded tables stay allocated: cached argument blocks and captured graphs may point at them
_CALLS = {}


def _sig(t):
    return None if t is None else (t.data_ptr(), t.shape, t.stride(), t.dtype)


def rope_table(device, positions: int, head_dim: int = 128, theta: float = 10000.0, stream=None):
    """cos/sin position table for the tensor-core kernel, built once per
    (device, theta, head_dim) and grown geometrically with the longest context seen.

    Returns (buffer, rows, event).  The table is built on `stream` (default: the current
    stream); `event` is recorded right after the build so that a launch on another stream
    can order itself behind it.  A table that is replaced by a larger one is never freed:
    argument blocks handed out earlier, and CUDA graphs captured with them, keep pointing
    at memory that still holds a valid (shorter) table."""
    dev = device if isinstance(device, torch.device) else torch.device(device)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), float(theta), int(head_dim))
    have = _TABLES.get(key)
    if have is not None and have[1] >= positions:
        return have
    rows = 4096
    while rows < positions:
        rows *= 2
    nbytes = int(_lib.lib().wsvd_rope_table_bytes(rows, head_dim))
    buf = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        s = torch.cuda.current_stream() if stream is None else stream
        check(_lib.lib().wsvd_rope_table_init(_ptr(buf), nbytes, rows, head_dim, float(theta),
                                              ctypes.c_void_p(s.cuda_stream)), "wsvd_rope_table_init")
        ev = torch.cuda.Event()
        ev.record(s)
    if have is not None:
        _RETIRED_TABLES.append(have)
    _TABLES[key] = [buf, rows, ev, s.cuda_stream, False]
    return _TABLES[key]


def _order_after_table(entry, stream) -> None:
    """Make `stream` wait for the table's build when it was enqueued on another stream and
    has not finished yet.  Once the build is known to have finished nothing is done (and no
    event is queried, which a stream capture would not allow)."""
    if entry[4]:
        return
    _buf, _rows, ev, built_on, _done = entry
    s = torch.cuda.current_stream() if stream is None else stream
    if torch.cuda.is_current_stream_capturing():
        if s.cuda_stream != built_on:
            s.wait_event(ev)  # becomes a dependency of the captured graph on the build
        return
    if ev.query():
        entry[4] = True
    elif s.cuda_stream != built_on:
        s.wait_event(ev)


def kernel_status() -> int:
    """Status word of the tensor-core kernel (0 = no bounded wait timed out).  Synchronises."""
    v = ctypes.c_uint32()
    check(_lib.lib().wsvd_kernel_status(ctypes.byref(v)), "wsvd_kernel_status")
    return v.value


def build_params(
    q, b_seq_len, b_req_idx, req_to_token, max_len, latent_k, k_scale, latent_v, v_scale, wk, wk_scale=None,
    wv=None, out=None, pos_offset=None, theta=10000.0, sm_scale=0.0, rope_layout="half", split_len=0,
    kernel="auto", stream=None, max_position=None,
) -> Tuple[LatentDecodeParams, list]:
    """Validate tensors and fill a WsvdLatentDecodeParams.  Returns the struct and the
    list of tensors it points into (keep them alive until the launch is enqueued).

    `max_position`: with `pos_offset`, an upper bound of pos_offset[b] + len_b (the position
    table must reach it); when absent it is read from `pos_offset` with a device
    synchronisation."""
    _cuda_tensor("q", q, (torch.float16,), 3)
    B, Hq, D = q.shape
    _cuda_tensor("cache_latent_k", latent_k, (torch.int8, torch.float16), 3)
    _cuda_tensor("cache_latent_v", latent_v, (torch.int8, torch.float16), 3)
    _need(latent_k.dtype == latent_v.dtype, "latent K and V must share a dtype", TypeError)
    is_i8 = latent_k.dtype == torch.int8
    Hkv, Rk = latent_k.shape[1], latent_k.shape[2]
    Rv = latent_v.shape[2]
    _need(latent_v.shape[1] == Hkv, "latent K and V disagree on the number of KV heads")
    _need(Hq % Hkv == 0, f"q heads ({Hq}) must be a multiple of KV heads ({Hkv})")
    _need(D in (16, 32, 64, 128), f"head_dim {D} not in {{16, 32, 64, 128}}")
    _need(1 <= Rk <= 128 and 1 <= Rv <= 128, "per-head rank must be in [1, 128]")
    _cuda_tensor("wk", wk, (torch.int8, torch.float16), 2)
    _need(wk.shape[1] == D * Hkv, f"wk.shape[1] ({wk.shape[1]}) != head_dim * kv_heads ({D * Hkv})")
    _need(wk.shape[0] == Rk, f"wk.shape[0] ({wk.shape[0]}) != rank_k ({Rk})")
    if is_i8:
        _need(k_scale is not None and v_scale is not None, "int8 latents need k_scale and v_scale", TypeError)
        _cuda_tensor("cache_latent_k_scale", k_scale, (torch.float16,), 2, inner_contiguous=False)
        _cuda_tensor("cache_latent_v_scale", v_scale, (torch.float16,), 2, inner_contiguous=False)
        _need(k_scale.shape[0] == latent_k.shape[0] and k_scale.shape[1] == Hkv, "k_scale must be [T, Hkv]")
        _need(v_scale.shape[0] == latent_v.shape[0] and v_scale.shape[1] == Hkv, "v_scale must be [T, Hkv]")
    else:
        _need(k_scale is None and v_scale is None, "f16 latents take no scales", TypeError)
    if wk.dtype == torch.int8:
        _need(wk_scale is not None, "int8 wk needs wk_scale", TypeError)
        _need(wk_scale.is_cuda and wk_scale.dtype == torch.float16, "wk_scale must be a CUDA f16 tensor", TypeError)
        _need(wk_scale.numel() == D * Hkv and wk_scale.is_contiguous(),
              f"wk_scale must hold head_dim * kv_heads = {D * Hkv} contiguous values")
    else:
        _need(wk_scale is None, "f16 wk takes no wk_scale", TypeError)
    if wv is not None:
        _cuda_tensor("wv", wv, (torch.float16,), 2)
        _need(tuple(wv.shape) == (Rv, D * Hkv), f"wv must be [rank_v, head_dim*kv_heads] = {(Rv, D * Hkv)}")
    for name, t in (("b_seq_len", b_seq_len), ("b_req_idx", b_req_idx)):
        _cuda_tensor(name, t, (torch.int32,), 1)
        _need(t.shape[0] == B, f"{name} must have batch ({B}) entries")
    _cuda_tensor("req_to_token_indexs", req_to_token, (torch.int32,), 2)
    _need(0 <= max_len <= req_to_token.shape[1], "max_len_in_batch exceeds the page-table width")
    if pos_offset is not None:
        _cuda_tensor("pos_offset", pos_offset, (torch.int32,), 1)
        _need(pos_offset.shape[0] == B, "pos_offset must have batch entries")
    out_w = D if wv is not None else Rv
    if out is not None:
        _cuda_tensor("out", out, (torch.float16,), 3)
        _need(tuple(out.shape) == (B, Hq, out_w), f"out must be {(B, Hq, out_w)}, got {tuple(out.shape)}")
    _need(rope_layout in ROPE, f"rope_layout must be one of {list(ROPE)}")
    _need(kernel in KERNEL, f"kernel must be one of {list(KERNEL)}")

    p = LatentDecodeParams()
    p.q, p.q_stride_b, p.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    p.latent_k, p.k_stride_t, p.k_stride_h = latent_k.data_ptr(), latent_k.stride(0), latent_k.stride(1)
    p.latent_v, p.v_stride_t, p.v_stride_h = latent_v.data_ptr(), latent_v.stride(0), latent_v.stride(1)
    if is_i8:
        p.k_scale, p.ks_stride_t, p.ks_stride_h = k_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1)
        p.v_scale, p.vs_stride_t, p.vs_stride_h = v_scale.data_ptr(), v_scale.stride(0), v_scale.stride(1)
    p.wk, p.wk_stride_r = wk.data_ptr(), wk.stride(0)
    p.wk_scale = None if wk_scale is None else wk_scale.data_ptr()
    if wv is not None:
        p.wv, p.wv_stride_r = wv.data_ptr(), wv.stride(0)
    p.req_to_token, p.rtt_stride = req_to_token.data_ptr(), req_to_token.stride(0)
    p.b_req_idx, p.b_seq_len = b_req_idx.data_ptr(), b_seq_len.data_ptr()
    p.pos_offset = None if pos_offset is None else pos_offset.data_ptr()
    if out is not None:
        p.out, p.out_stride_b, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    p.batch, p.n_q_heads, p.n_kv_heads, p.head_dim, p.rank_k, p.rank_v = B, Hq, Hkv, D, Rk, Rv
    p.max_len = int(max_len)
    p.latent_dtype = I8 if is_i8 else F16
    p.wk_dtype = I8 if wk.dtype == torch.int8 else F16
    p.rope_layout = ROPE[rope_layout]
    p.split_len = int(split_len)
    p.kernel = KERNEL[kernel]
    p.theta, p.sm_scale = float(theta), float(sm_scale)
    p.n_token_slots = min(latent_k.shape[0], latent_v.shape[0])
    if D == 128 and kernel != "generic":
        reach = int(max_len)
        if pos_offset is not None:
            reach = int(max_position) if max_position is not None else reach + max(0, int(pos_offset.max().item()))
        table, rows = rope_table(q.device, reach, D, theta, stream=stream)[:2]
        p.rope_table, p.rope_table_rows = table.data_ptr(), rows
    keep = [q, latent_k, latent_v, k_scale, v_scale, wk, wk_scale, wv, req_to_token, b_req_idx, b_seq_len,
            pos_offset, out]
    return p, keep


def plan(p: LatentDecodeParams) -> Tuple[int, int]:
    sl, ns = ctypes.c_int32(), ctypes.c_int32()
    check(_lib.lib().wsvd_latent_decode_plan(ctypes.byref(p), ctypes.byref(sl), ctypes.byref(ns)), "plan")
    return sl.value, ns.value


def workspace_bytes(p: LatentDecodeParams) -> int:
    return int(_lib.lib().wsvd_latent_decode_workspace_bytes(ctypes.byref(p)))


def _stream(stream) -> ctypes.c_void_p:
    if stream is not None:
        return ctypes.c_void_p(stream.cuda_stream)
    if _raw_stream is not None:  # the handle without building a Stream object around it
        return ctypes.c_void_p(_raw_stream(torch.cuda.current_device()))
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _cached_params(tag, q3, infer_state, latent_k, k_scale, latent_v, v_scale, wk, wk_scale, wv, pos_offset, theta,
                   rope_layout, split_len, kernel, stream):
    """A private copy of the validated argument block for this set of buffers and options.

    A decode loop calls with the same buffers every step, so the validated block is kept
    per (address, shape, stride) signature.  What can change underneath a cached block is
    refreshed on every hit: the position table (it is replaced by a larger one when a
    longer context arrives).  The caller gets a copy, so that filling in `out` does not
    touch the cached block and calls from several threads do not share mutable state."""
    rtt = infer_state.req_manager.req_to_token_indexs
    max_len = int(infer_state.max_len_in_batch)
    key = (tag, _sig(q3), _sig(infer_state.b_seq_len), _sig(infer_state.b_req_idx), _sig(rtt), max_len,
           _sig(latent_k), _sig(k_scale), _sig(latent_v), _sig(v_scale), _sig(wk), _sig(wk_scale), _sig(wv),
           _sig(pos_offset), float(theta), rope_layout, int(split_len), kernel)
    # position offsets may change inside the same buffer and decide how far the position table must
    # reach, so such calls are validated (and the reach read back from the device) every time
    hit = _CALLS.get(key) if pos_offset is None else None
    if hit is None:
        p, _keep = build_params(
            q3, infer_state.b_seq_len, infer_state.b_req_idx, rtt, max_len, latent_k, k_scale, latent_v, v_scale,
            wk, wk_scale, wv=wv, out=None, pos_offset=pos_offset, theta=theta, rope_layout=rope_layout,
            split_len=split_len, kernel=kernel, stream=stream)
        hit = (p, workspace_bytes(p))
        if pos_offset is None:
            if len(_CALLS) >= 64:
                _CALLS.clear()
            _CALLS[key] = hit
    cached, need = hit
    p = LatentDecodeParams.from_buffer_copy(cached)
    if cached.rope_table:
        entry = rope_table(q3.device, max(max_len, cached.rope_table_rows if pos_offset is not None else 0),
                           p.head_dim, theta, stream=stream)
        p.rope_table, p.rope_table_rows = entry[0].data_ptr(), entry[1]
        _order_after_table(entry, stream)
    return p, need


def latent_decode(
    q, infer_state, latent_k, k_scale, latent_v, v_scale, wk, wk_scale=None, *, wv=None, out=None,
    workspace: Optional[torch.Tensor] = None, alloc_tensor_func: Callable = torch.empty, pos_offset=None,
    theta=10000.0, rope_layout="half", split_len=0, kernel="auto", stream=None,
) -> torch.Tensor:
    """Fused latent decode attention.  Returns O_lat [B,Hq,Rv] (f16), or O [B,Hq,D] when
    `wv` ([Rv, Hkv*D] f16) is given.  `workspace` is an optional CUDA byte/float buffer of
    at least workspace_bytes(); when absent it is taken from `alloc_tensor_func`."""
    B = int(infer_state.batch_size)
    q3 = q.view(B, q.shape[-2], q.shape[-1]) if q.dim() != 3 else q
    p, need = _cached_params("decode", q3, infer_state, latent_k, k_scale, latent_v, v_scale, wk, wk_scale, wv,
                             pos_offset, theta, rope_layout, split_len, kernel, stream)
    out_w = p.head_dim if wv is not None else p.rank_v
    if out is None:
        out = alloc_tensor_func((B, p.n_q_heads, out_w), dtype=q.dtype, device=q.device)
    else:
        _cuda_tensor("out", out, (torch.float16,), 3)
        if tuple(out.shape) != (B, p.n_q_heads, out_w):
            raise ValueError(f"out must be {(B, p.n_q_heads, out_w)}")
    p.out, p.out_stride_b, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    if workspace is None:
        workspace = alloc_tensor_func(((need + 3) // 4,), dtype=torch.float32, device=q.device)
    else:
        _need(workspace.is_cuda and workspace.is_contiguous(), "workspace must be a contiguous CUDA tensor")
    have = workspace.numel() * workspace.element_size()
    with _on_device(q.device):
        check(_lib.lib().wsvd_latent_decode(ctypes.byref(p), _ptr(workspace), have, _stream(stream)),
              "wsvd_latent_decode")
    return out


@torch.no_grad()
def latent_decode_gather(q, infer_state, latent_k, k_scale, latent_v, v_scale, wk, wk_scale, peers, *, wv=None,
                         workspace: Optional[torch.Tensor] = None, theta=10000.0, rope_layout="half", split_len=0,
                         kernel="auto", stream=None) -> None:
    """This rank's head shard of the op with the head all-gather fused into the merge
    kernel: rows go straight into every rank's gathered buffer (`peers`, a filled
    `_lib.PeerSet`, see `wsvd_b200.dist.PeerGather`).  Arguments as `latent_decode`, with the
    LOCAL heads."""
    B = int(infer_state.batch_size)
    q3 = q.view(B, q.shape[-2], q.shape[-1]) if q.dim() != 3 else q
    p, need = _cached_params("gather", q3, infer_state, latent_k, k_scale, latent_v, v_scale, wk, wk_scale, wv,
                             None, theta, rope_layout, split_len, kernel, stream)
    if workspace is None:
        workspace = torch.empty(((need + 3) // 4,), dtype=torch.float32, device=q.device)
    have = workspace.numel() * workspace.element_size()
    with _on_device(q.device):
        check(_lib.lib().wsvd_latent_decode_gather(ctypes.byref(p), ctypes.byref(peers), _ptr(workspace), have,
                                                   _stream(stream)), "wsvd_latent_decode_gather")


@torch.no_grad()
def latent_decode_stage1(q, latent_k, k_scale, latent_v, v_scale, wk, wk_scale, req_to_token, b_req_idx, b_seq_len,
                         max_len, mid_out, mid_out_lse, block_seq, *, theta=10000.0, rope_layout="half",
                         kernel="auto", stream=None):
    """Split-KV stage 1 into caller-owned partial buffers mid_out [B,Hq,n_splits,Rv] f32
    and mid_out_lse [B,Hq,n_splits] f32."""
    p, keep = build_params(q, b_seq_len, b_req_idx, req_to_token, int(max_len), latent_k, k_scale, latent_v, v_scale,
                           wk, wk_scale, theta=theta, rope_layout=rope_layout, split_len=int(block_seq),
                           kernel=kernel)
    _need(mid_out.is_cuda and mid_out.dtype == torch.float32 and mid_out.is_contiguous(), "mid_out: contiguous CUDA f32")
    _need(mid_out_lse.is_cuda and mid_out_lse.dtype == torch.float32 and mid_out_lse.is_contiguous(),
          "mid_out_logsumexp: contiguous CUDA f32")
    B, Hq, ns, Rv = mid_out.shape
    _need((B, Hq, Rv) == (p.batch, p.n_q_heads, p.rank_v), "mid_out must be [B, Hq, n_splits, rank_v]")
    _need(tuple(mid_out_lse.shape) == (B, Hq, ns), "mid_out_logsumexp must be [B, Hq, n_splits]")
    with torch.cuda.device(q.device):
        check(_lib.lib().wsvd_latent_decode_stage1(ctypes.byref(p), _ptr(mid_out), _ptr(mid_out_lse), ns,
                                                   _stream(stream)), "wsvd_latent_decode_stage1")


@torch.no_grad()
def decode_stage2(mid_out, mid_out_lse, b_seq_len, out, block_seq, *, wv=None, n_kv_heads=None, stream=None):
    """Split-KV stage 2: merge partials by log-sum-exp weights into `out` (f16)."""
    for name, t in (("mid_out", mid_out), ("mid_out_logexpsum", mid_out_lse)):
        _need(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous(), f"{name}: contiguous CUDA f32")
    B, Hq, ns, W = mid_out.shape
    _need(tuple(mid_out_lse.shape) == (B, Hq, ns), "mid_out_logexpsum must be [B, Hq, n_splits]")
    _cuda_tensor("B_Seqlen", b_seq_len, (torch.int32,), 1)
    _cuda_tensor("O", out, (torch.float16,), 3)
    head_dim, hkv, wv_stride = 0, 1, 0
    if wv is not None:
        _cuda_tensor("wv", wv, (torch.float16,), 2)
        hkv = int(n_kv_heads or Hq)
        head_dim = wv.shape[1] // hkv
        wv_stride = wv.stride(0)
        _need(tuple(out.shape) == (B, Hq, head_dim), "out must be [B, Hq, head_dim] when wv is given")
    else:
        _need(tuple(out.shape) == (B, Hq, W), "out must be [B, Hq, width]")
    with torch.cuda.device(out.device):
        check(_lib.lib().wsvd_decode_stage2(
            _ptr(mid_out), _ptr(mid_out_lse), _ptr(b_seq_len), _ptr(out), out.stride(0), out.stride(1),
            B, Hq, ns, W, int(block_seq), _ptr(wv), wv_stride, hkv, head_dim, _stream(stream)), "wsvd_decode_stage2")


def dense_decode(q, infer_state, cache_k, cache_v, out=None, alloc_tensor_func: Callable = torch.empty,
                 workspace=None, split_len=0, stream=None):
    """Dense f16 flash-decoding baseline: q [B,Hq,D], caches [T,Hkv,D] f16 -> [B,Hq,D] f16."""
    from ._lib import DenseDecodeParams

    _cuda_tensor("q", q, (torch.float16,), 3)
    B, Hq, D = q.shape
    _cuda_tensor("cache_k", cache_k, (torch.float16,), 3)
    _cuda_tensor("cache_v", cache_v, (torch.float16,), 3)
    Hkv = cache_k.shape[1]
    _need(cache_k.shape[2] == D and cache_v.shape[2] == D, "q and K/V disagree on head_dim")
    _need(cache_v.shape[1] == Hkv and Hq % Hkv == 0, "bad head counts")
    if D not in (16, 32, 64, 128):
        raise ValueError(f"head_dim {D} not in {{16, 32, 64, 128}}")
    rtt = infer_state.req_manager.req_to_token_indexs
    _cuda_tensor("b_seq_len", infer_state.b_seq_len, (torch.int32,), 1)
    _cuda_tensor("b_req_idx", infer_state.b_req_idx, (torch.int32,), 1)
    _cuda_tensor("req_to_token_indexs", rtt, (torch.int32,), 2)
    if out is None:
        out = alloc_tensor_func((B, Hq, D), dtype=q.dtype, device=q.device)
    _cuda_tensor("out", out, (torch.float16,), 3)
    p = DenseDecodeParams()
    p.q, p.q_stride_b, p.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    p.k, p.k_stride_t, p.k_stride_h = cache_k.data_ptr(), cache_k.stride(0), cache_k.stride(1)
    p.v, p.v_stride_t, p.v_stride_h = cache_v.data_ptr(), cache_v.stride(0), cache_v.stride(1)
    p.req_to_token, p.rtt_stride = rtt.data_ptr(), rtt.stride(0)
    p.b_req_idx, p.b_seq_len = infer_state.b_req_idx.data_ptr(), infer_state.b_seq_len.data_ptr()
    p.out, p.out_stride_b, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    p.batch, p.n_q_heads, p.n_kv_heads, p.head_dim = B, Hq, Hkv, D
    p.max_len, p.split_len = int(infer_state.max_len_in_batch), int(split_len)
    need = int(_lib.lib().wsvd_dense_decode_workspace_bytes(ctypes.byref(p)))
    if workspace is None:
        workspace = alloc_tensor_func(((need + 3) // 4,), dtype=torch.float32, device=q.device)
    have = workspace.numel() * workspace.element_size()
    with _on_device(q.device):
        check(_lib.lib().wsvd_dense_decode_f16(ctypes.byref(p), _ptr(workspace), have, _stream(stream)),
              "wsvd_dense_decode_f16")
    return out


def latent_quant_append(x_k, x_v, infer_state, cache_latent_k, cache_latent_k_scale, cache_latent_v,
                        cache_latent_v_scale, stream=None):
    """Quantise the new token's latents and store them in the cache (in place).

    x_k [B, Hkv, Rk], x_v [B, Hkv, Rv] (f16 or f32) are written, as int8 with one f16 scale
    per (sequence, head), to token slot ``req_to_token_indexs[b_req_idx[b], b_seq_len[b]]``:
    ``infer_state.b_seq_len`` holds the lengths before the append, the caller increments it
    afterwards.  Quantiser: fake_quant/quant_utils.py:30-33,175-184 against the stored f16
    scale.  The reference has no counterpart (efficiency/layer_utils.py:319-321 drops the
    new latents)."""
    from ._lib import QuantAppendParams

    _cuda_tensor("x_k", x_k, (torch.float16, torch.float32), 3)
    _cuda_tensor("x_v", x_v, (torch.float16, torch.float32), 3)
    _need(x_k.dtype == x_v.dtype, "x_k and x_v must share a dtype", TypeError)
    B, Hkv, Rk = x_k.shape
    Rv = x_v.shape[2]
    _need(x_v.shape[:2] == (B, Hkv), "x_k and x_v disagree on batch or heads")
    _cuda_tensor("cache_latent_k", cache_latent_k, (torch.int8,), 3)
    _cuda_tensor("cache_latent_v", cache_latent_v, (torch.int8,), 3)
    _cuda_tensor("cache_latent_k_scale", cache_latent_k_scale, (torch.float16,), 2, inner_contiguous=False)
    _cuda_tensor("cache_latent_v_scale", cache_latent_v_scale, (torch.float16,), 2, inner_contiguous=False)
    _need(cache_latent_k.shape[1:] == (Hkv, Rk) and cache_latent_v.shape[1:] == (Hkv, Rv),
          "cache shapes must be [T, Hkv, Rk] and [T, Hkv, Rv]")
    _need(0 < Rk <= 128 and 0 < Rv <= 128, "ranks must be in 1..128")
    rtt = infer_state.req_manager.req_to_token_indexs
    _cuda_tensor("b_seq_len", infer_state.b_seq_len, (torch.int32,), 1)
    _cuda_tensor("b_req_idx", infer_state.b_req_idx, (torch.int32,), 1)
    _cuda_tensor("req_to_token_indexs", rtt, (torch.int32,), 2)
    _need(infer_state.b_seq_len.numel() == B and infer_state.b_req_idx.numel() == B, "batch metadata must have B entries")
    p = QuantAppendParams()
    p.x_k, p.xk_stride_b, p.xk_stride_h = x_k.data_ptr(), x_k.stride(0), x_k.stride(1)
    p.x_v, p.xv_stride_b, p.xv_stride_h = x_v.data_ptr(), x_v.stride(0), x_v.stride(1)
    p.latent_k, p.k_stride_t, p.k_stride_h = cache_latent_k.data_ptr(), cache_latent_k.stride(0), cache_latent_k.stride(1)
    p.latent_v, p.v_stride_t, p.v_stride_h = cache_latent_v.data_ptr(), cache_latent_v.stride(0), cache_latent_v.stride(1)
    p.k_scale, p.ks_stride_t, p.ks_stride_h = (cache_latent_k_scale.data_ptr(), cache_latent_k_scale.stride(0),
                                               cache_latent_k_scale.stride(1))
    p.v_scale, p.vs_stride_t, p.vs_stride_h = (cache_latent_v_scale.data_ptr(), cache_latent_v_scale.stride(0),
                                               cache_latent_v_scale.stride(1))
    p.req_to_token, p.rtt_stride = rtt.data_ptr(), rtt.stride(0)
    p.b_req_idx, p.b_seq_len = infer_state.b_req_idx.data_ptr(), infer_state.b_seq_len.data_ptr()
    p.batch, p.n_kv_heads, p.rank_k, p.rank_v = B, Hkv, Rk, Rv
    p.max_len = rtt.shape[1]
    p.x_dtype = 1 if x_k.dtype == torch.float16 else 2
    with _on_device(x_k.device):
        check(_lib.lib().wsvd_latent_quant_append_i8(ctypes.byref(p), _stream(stream)), "wsvd_latent_quant_append_i8")


# ---- the dense attention block of a step: adapters beside a projection, rotate-and-append, attention over the paged cache

BF16 = 3
_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.int8: I8}
_HALVES = (torch.float16, torch.bfloat16)
_pack_append = _lib.packer(_lib.KvRopeAppendParams)
_pack_paged = _lib.packer(_lib.PagedDecodeParams)
_pack_adapter = _lib.packer(_lib.AdapterAddParams)


# An ordinary call (the current stream, torch's allocator, arguments as they should be) goes through csrc/bind.cpp, which
# answers None to any other: the checks below say what is wrong with it, or it is made the long way.  (A single token's append
# takes the GPU 3 us; with its arguments looked at in Python the call took 14, so it takes 6.)  Where that module cannot be built or
# loaded all calls are made the long way, to the same entries of the library.

_fast = None


class _LongWay:
    @staticmethod
    def append(*args):
        return None

    paged = adapter = append


def _ordinary():
    global _fast
    if _fast is None:
        try:
            _fast = _lib.bind()
        except _lib.NO_BIND as e:
            warnings.warn(f"csrc/bind.cpp is not there, calls go through ctypes and take some 10 us more: {e}", RuntimeWarning, stacklevel=3)
            _fast = _LongWay
    return _fast


def _done(answer, name):
    """bind.cpp's answer, where it is one."""
    if answer.__class__ is int:
        check(answer, name)
    return answer

def _tensor(name, t, dtypes, ndim, inner_contiguous=True):
    """As `_cuda_tensor`, the device left to `_on_one_gpu`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got {tuple(t.shape)}")
    if inner_contiguous and t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel() != 0:
        raise ValueError(f"{name}: innermost dimension must be contiguous")


def _countable(**sizes):
    """Sizes that the C entries take as 32-bit numbers."""
    for name, n in sizes.items():
        if n > 2 ** 31 - 1:
            raise ValueError(f"{name}: {n} is beyond 2^31 - 1")


def _apart(name, t):
    """An output's elements have a place in memory each."""
    reach = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1 and t.numel() > 0:
            if stride < reach:
                raise ValueError(f"{name}: elements share memory (shape {tuple(t.shape)}, strides {t.stride()})")
            reach += stride * (size - 1)


def _meet(a, b):
    """Whether two tensors have a byte of memory in common.  (Exact for views of one layout, column slices of a joined
    matrix or heads of a joined projection among them; strides of two layouts that would take long to look through count as yes.)"""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size, apart = max(a.element_size(), b.element_size()), b.data_ptr() - a.data_ptr()
    # apart = sum of i stride over a's dims - the same over b's, but for the last element's bytes
    terms = {}
    for t, sign in ((a, 1), (b, -1)):
        for n, s in zip(t.shape, t.stride()):
            if n > 1 and s > 0:
                r = terms.setdefault(s * t.element_size(), [0, 0])
                r[sign > 0] += sign * (n - 1)
    terms = sorted(terms.items(), reverse=True)
    budget = 256

    def reach(at, left):
        nonlocal budget
        low = sum(s * r[0] for s, r in terms[at:])
        high = sum(s * r[1] for s, r in terms[at:])
        if not low - size < left < high + size:
            return False
        if at == len(terms):
            return True
        s, (first, last) = terms[at]
        low, high = low - s * first, high - s * last
        for i in range(max(first, -((high + size - 1 - left) // s)), min(last, (left - low + size - 1) // s) + 1):
            budget -= 1
            if budget < 0 or reach(at + 1, left - i * s):
                return True
        return False

    return reach(0, apart)


def _same_places(a, b):
    """Two tensors of one shape whose elements are at the same addresses."""
    return a.data_ptr() == b.data_ptr() and all(n < 2 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _no_overlap(name, out, in_place, t, **others):
    """An output may be the input `in_place` itself, and has no memory of any input otherwise."""
    if not _same_places(out, t) and _meet(out, t):
        raise ValueError(f"{name} may be {in_place} itself, not another view of its storage")
    for other, o in others.items():
        if o is not None and _meet(out, o):
            raise ValueError(f"{name} must not overlap {other}")


def _on_one_gpu(**tensors):
    index = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (no CPU path exists)")
        if index is None:
            index = t.get_device()
        elif t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _no_gradient(op, *tensors):
    tensors = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{op} has no backward: call it under torch.no_grad() or on detached tensors")
    # (torch.no_grad() does not switch forward mode off)
    if any(t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{op} has no forward-mode derivative: call it on the primal tensors")


def _metadata(lens, idx, table, B):
    _tensor("b_seq_len", lens, (torch.int32,), 1)
    _tensor("b_req_idx", idx, (torch.int32,), 1)
    _tensor("req_to_token_indexs", table, (torch.int32,), 2)
    if lens.shape[0] != B or idx.shape[0] != B:
        raise ValueError("batch metadata must have one entry per sequence")
    _countable(batch=B, **{"rows of req_to_token_indexs": table.shape[0], "columns of req_to_token_indexs": table.shape[1]})


def _dense_cache(cache_k, cache_v, k_scale, v_scale, dtype, Hkv, D):
    """Checks of a dense cache [T, Hkv, D] (and scales [T, Hkv] of an int8 one)."""
    _tensor("cache_k", cache_k, (dtype, torch.int8), 3)
    _tensor("cache_v", cache_v, (cache_k.dtype,), 3)
    if cache_k.shape[1:] != (Hkv, D) or cache_v.shape != cache_k.shape:
        raise ValueError(f"cache_k and cache_v must be [T, {Hkv}, {D}], got {tuple(cache_k.shape)} and {tuple(cache_v.shape)}")
    if cache_k.dtype == torch.int8:
        if k_scale is None or v_scale is None:
            raise TypeError("int8 caches need their scales")
        for name, t in (("cache_k's scale", k_scale), ("cache_v's scale", v_scale)):
            _tensor(name, t, (torch.float16,), 2, inner_contiguous=False)
            if t.shape != cache_k.shape[:2]:
                raise ValueError(f"{name} must be [T, Hkv] = {tuple(cache_k.shape[:2])}, got {tuple(t.shape)}")
    elif k_scale is not None or v_scale is not None:
        raise TypeError("only int8 caches have scales")


def _new(alloc_tensor_func, like, shape, dtype, stream):
    """A buffer of the op's own.  For a stream of the caller's it comes from that stream's pool (what the current stream's pool hands
    out may still be in use there, by work that the other stream has not waited for), and goes back once the current stream, where the
    caller may read it, has done with it too."""
    if stream is None:
        return alloc_tensor_func(shape, dtype=dtype, device=like.device)
    current = torch.cuda.current_stream(like.device)
    with torch.cuda.stream(stream):
        t = alloc_tensor_func(shape, dtype=dtype, device=like.device)
    t.record_stream(current)
    return t


def _run(name, index, stream, *args):
    """Call a C entry on GPU `index`, on `stream` or that GPU's current stream."""
    entry = getattr(_lib.lib(), name)
    if stream is None and _raw_stream is not None and torch.cuda.current_device() == index:
        check(entry(*args, _raw_stream(index)), name)
        return
    with torch.cuda.device(index):
        check(entry(*args, _stream(stream)), name)


def _check_append(k, v, lens, idx, table, cache_k, cache_v, inv_freq, cache_k_scale, cache_v_scale, q, q_out, cu_new, pos_offset,
                  rope_layout):
    _tensor("k", k, _HALVES, 3)
    dtype = k.dtype
    _tensor("v", v, (dtype,), 3)
    N, Hkv, D = k.shape
    if v.shape != k.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    _tensor("inv_freq", inv_freq, (torch.float32,), 1)
    if Hkv < 1:
        raise ValueError("k and v must have heads")
    _countable(**{"rows of k": N, "heads of k": Hkv})
    if D < 2 or D % 2 or D > 256 or 2 * inv_freq.shape[0] > D:
        raise ValueError(f"head_dim must be even and at most 256, with at most head_dim / 2 frequencies: {D}, {inv_freq.shape[0]}")
    _dense_cache(cache_k, cache_v, cache_k_scale, cache_v_scale, dtype, Hkv, D)
    B = N
    if cu_new is not None:
        _tensor("cu_new", cu_new, (torch.int32,), 1)
        B = cu_new.shape[0] - 1
        if B < 0:
            raise ValueError("cu_new must have batch + 1 entries")
    _metadata(lens, idx, table, B)
    if pos_offset is not None:
        _tensor("pos_offset", pos_offset, (torch.int32,), 1)
        if pos_offset.shape[0] != B:
            raise ValueError("pos_offset must have batch entries")
    if rope_layout not in ROPE:
        raise ValueError(f"rope_layout must be one of {list(ROPE)}")
    if q is not None:
        _tensor("q", q, (dtype,), 3)
        if q.shape[0] != N or q.shape[2] != D:
            raise ValueError(f"q must be [{N}, Hq, {D}], got {tuple(q.shape)}")
        _countable(**{"heads of q": q.shape[1]})
        if q_out is not None:
            _tensor("q_out", q_out, (dtype,), 3)
            if q_out.shape != q.shape:
                raise ValueError(f"q_out must be {tuple(q.shape)}, got {tuple(q_out.shape)}")
            _no_overlap("q_out", q_out, "q", q, k=k, v=v)
            _apart("q_out", q_out)
    elif q_out is not None:
        raise ValueError("q_out without q")
    for name, t in (("cache_k", cache_k), ("cache_v", cache_v), ("cache_k_scale", cache_k_scale), ("cache_v_scale", cache_v_scale)):
        if t is not None:
            _apart(name, t)
    for a, b, names in ((cache_k, cache_v, "cache_k and cache_v"), (q_out, cache_k, "q_out and cache_k"), (q_out, cache_v, "q_out and cache_v")):
        if a is not None and _meet(a, b):
            raise ValueError(f"{names} overlap")
    _no_gradient("kv_rope_append", k, v, q, q_out, cache_k, cache_v, cache_k_scale, cache_v_scale, inv_freq)
    _on_one_gpu(k=k, v=v, q=q, q_out=q_out, cache_k=cache_k, cache_v=cache_v, cache_k_scale=cache_k_scale,
                cache_v_scale=cache_v_scale, inv_freq=inv_freq, b_seq_len=lens, b_req_idx=idx, req_to_token_indexs=table,
                cu_new=cu_new, pos_offset=pos_offset)


def kv_rope_append(k, v, infer_state, cache_k, cache_v, inv_freq, *, cache_k_scale=None, cache_v_scale=None, q=None,
                   q_out=None, cu_new=None, pos_offset=None, rope_layout="half", stream=None):
    """Store new keys and values in the paged cache (in place), the keys rotated to their positions on the way; with `q`,
    return the queries rotated beside them.  For prompts, chunks of them and single tokens.

    k, v [N, Hkv, D], q [N, Hq, D] (f16 or bf16, any stride between rows and heads: column slices of one joined
    projection will do) are rows packed by sequence; `cu_new` [B + 1] int32 has each sequence's first row, None means
    one row per sequence.  Row i of sequence b goes to position ``b_seq_len[b] + i`` in token slot
    ``req_to_token_indexs[b_req_idx[b], position]``: ``infer_state.b_seq_len`` holds the lengths before the append, the caller
    adds the new rows afterwards.  The first ``2 * len(inv_freq)`` dims are rotated by ``(position + pos_offset[b]) *
    inv_freq`` (`rope_layout` as in `latent_decode`), the others and v go through.
    cache_k, cache_v [T, Hkv, D] in the rows' dtype, or int8 with f16 scales [T, Hkv] (the quantiser of
    `latent_quant_append`, on the rotated f32 row).  `q_out` may be q, and shares no memory with q, k or v otherwise, nor do
    the outputs with one another.

    Rows behind cu_new[B] are padding: nothing of them is stored, a `q_out` of the caller's keeps its rows, the op's own has
    zeros there.  A row without a place in the table or the cache is skipped and reported by `kernel_status`.  No two rows may
    name the same slot, and none may be read from memory that the call writes.
    The reference's dense caches are made by its test script (efficiency/test_timing_layer.py)."""
    lens, idx, table = infer_state.b_seq_len, infer_state.b_req_idx, infer_state.req_manager.req_to_token_indexs
    if stream is None and rope_layout in ROPE:
        done = _ordinary().append(k, v, lens, idx, table, cache_k, cache_v, inv_freq, cache_k_scale, cache_v_scale, q, q_out, cu_new,
                                  pos_offset, ROPE[rope_layout])
        if done is not None:
            return None if _done(done, "wsvd_kv_rope_append") is True else done
    _check_append(k, v, lens, idx, table, cache_k, cache_v, inv_freq, cache_k_scale, cache_v_scale, q, q_out, cu_new, pos_offset,
                  rope_layout)
    N, Hkv, D = k.shape
    dtype, held, index = k.dtype, cache_k.dtype, k.get_device()
    B = N if cu_new is None else cu_new.shape[0] - 1
    own = q is not None and q_out is None
    if own:
        q_out = _new(torch.empty, q, q.shape, dtype, stream)
    code, i8 = _CODE[dtype], held is torch.int8
    args = _pack_append(
        k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
        *((0, 0, 0, 0, 0, 0) if q is None else (q.data_ptr(), *q.stride()[:2], q_out.data_ptr(), *q_out.stride()[:2])),
        cache_k.data_ptr(), *cache_k.stride()[:2], cache_v.data_ptr(), *cache_v.stride()[:2],
        *((cache_k_scale.data_ptr(), *cache_k_scale.stride(), cache_v_scale.data_ptr(), *cache_v_scale.stride()) if i8 else
          (0, 0, 0, 0, 0, 0)),
        inv_freq.data_ptr(), table.data_ptr(), table.stride(0), idx.data_ptr(), lens.data_ptr(),
        0 if cu_new is None else cu_new.data_ptr(), 0 if pos_offset is None else pos_offset.data_ptr(), cache_k.shape[0],
        N, B, 0 if q is None else q.shape[1], Hkv, D, 2 * inv_freq.shape[0], table.shape[1], table.shape[0], code,
        I8 if i8 else code, ROPE[rope_layout], own)
    _run("wsvd_kv_rope_append", index, stream, args)
    return q_out


@functools.lru_cache(maxsize=256)
def paged_decode_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim) -> int:
    """Bytes of scratch that `paged_decode` needs for these sizes, whatever the lengths (nothing in it has to be set)."""
    p = _lib.PagedDecodeParams()
    p.batch, p.n_q_heads, p.n_kv_heads, p.head_dim = batch, n_q_heads, n_kv_heads, head_dim
    return int(_lib.lib().wsvd_paged_decode_workspace_bytes(ctypes.byref(p)))


def _check_paged(q, lens, idx, table, cache_k, cache_v, k_scale, v_scale, out, window, workspace):
    _tensor("q", q, _HALVES, 3)
    B, Hq, D = q.shape
    _tensor("cache_k", cache_k, (q.dtype, torch.int8), 3)
    Hkv = cache_k.shape[1]
    if D < 1 or D > 256:
        raise ValueError(f"head_dim {D} not in [1, 256]")
    _dense_cache(cache_k, cache_v, k_scale, v_scale, q.dtype, Hkv, D)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"q heads ({Hq}) must be a multiple of KV heads ({Hkv})")
    _countable(**{"heads of q": Hq})
    _metadata(lens, idx, table, B)
    if out is not None:
        _tensor("out", out, (q.dtype,), 3)
        if out.shape != q.shape:
            raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
        _no_overlap("out", out, "q", q, cache_k=cache_k, cache_v=cache_v)
        _apart("out", out)
    if window < 0:
        raise ValueError("window must not be negative")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _no_gradient("paged_decode", q, cache_k, cache_v, k_scale, v_scale, out)
    _on_one_gpu(q=q, cache_k=cache_k, cache_v=cache_v, k_scale=k_scale, v_scale=v_scale, b_seq_len=lens, b_req_idx=idx,
                req_to_token_indexs=table, out=out, workspace=workspace)


def paged_decode(q, infer_state, cache_k, cache_v, k_scale=None, v_scale=None, *, out=None, return_lse=False, window=0,
                 sm_scale=0.0, workspace: Optional[torch.Tensor] = None, alloc_tensor_func: Callable = torch.empty,
                 stream=None):
    """Attention of one new token per sequence over a paged cache: q [B, Hq, D] (f16 or bf16), caches [T, Hkv, D] in q's
    dtype or int8 with f16 scales [T, Hkv], as `kv_rope_append` fills them -> [B, Hq, D]; with `return_lse` also the log of
    the sum of exponentials [B, Hq] f32.

    Sequence b attends to the positions ``max(0, b_seq_len[b] - window) <= s < b_seq_len[b]`` (window 0: all), position s in
    token slot ``req_to_token_indexs[b_req_idx[b], s]``.  Query heads that share a KV head share its loads.  A
    sequence without positions gives zeros and -inf.  A page-table entry outside the cache is left out and
    reported by `kernel_status`, a length is clamped to the table's width.  `sm_scale` 0 means 1/sqrt(D).  `out` may be q, and shares
    no memory with q or the caches otherwise.
    `workspace`: an optional CUDA byte/float buffer of `paged_decode_workspace_bytes` bytes; calls that may
    run at the same time need one each.  (`dense_decode` is the reference's f16 baseline.)"""
    lens, idx, table = infer_state.b_seq_len, infer_state.b_req_idx, infer_state.req_manager.req_to_token_indexs
    window = int(window)
    if stream is None and alloc_tensor_func is torch.empty:
        done = _ordinary().paged(q, lens, idx, table, cache_k, cache_v, k_scale, v_scale, out, workspace, return_lse, window,
                                 float(sm_scale))
        if done is not None:
            return _done(done, "wsvd_paged_decode")
    _check_paged(q, lens, idx, table, cache_k, cache_v, k_scale, v_scale, out, window, workspace)
    B, Hq, D = shape = q.shape
    Hkv, dtype, held, index = cache_k.shape[1], q.dtype, cache_k.dtype, q.get_device()
    if out is None:
        out = _new(alloc_tensor_func, q, shape, dtype, stream)
    lse = _new(alloc_tensor_func, q, (B, Hq), torch.float32, stream) if return_lse else None
    if workspace is None:
        workspace = _new(alloc_tensor_func, q, (paged_decode_workspace_bytes(B, Hq, Hkv, D) // 2,), dtype, stream)
        have = workspace.numel() * 2
    else:
        have = workspace.numel() * workspace.element_size()
    code, i8 = _CODE[dtype], held is torch.int8
    args = _pack_paged(
        q.data_ptr(), *q.stride()[:2], cache_k.data_ptr(), *cache_k.stride()[:2], cache_v.data_ptr(), *cache_v.stride()[:2],
        *((k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride()) if i8 else (0, 0, 0, 0, 0, 0)),
        table.data_ptr(), table.stride(0), idx.data_ptr(), lens.data_ptr(), out.data_ptr(), *out.stride()[:2],
        0 if lse is None else lse.data_ptr(), cache_k.shape[0], B, Hq, Hkv, D, table.shape[1], table.shape[0], code,
        I8 if i8 else code, min(window, 2 ** 31 - 1), float(sm_scale))
    _run("wsvd_paged_decode", index, stream, args, workspace.data_ptr(), have)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def adapter_add_workspace_bytes(rows, batch, n_in, rank, packed) -> int:
    """Bytes of scratch that `adapter_add` needs for these sizes (packed: with a cu_new; nothing in it has to be set)."""
    p = _lib.AdapterAddParams()
    p.rows, p.batch, p.n_in, p.rank, p.cu_new = rows, batch, n_in, rank, 1 if packed else None
    return int(_lib.lib().wsvd_adapter_add_workspace_bytes(ctypes.byref(p)))


def _check_adapters(y, x, a, b, adapter, scale, cu_new, out, workspace):
    _tensor("x", x, _HALVES, 2)
    one = (x.dtype,)
    _tensor("y", y, one, 2)
    _tensor("a", a, one, 3)
    _tensor("b", b, one, 3)
    _tensor("adapter", adapter, (torch.int32,), 1)
    N, n_in = x.shape
    n_out = y.shape[1]
    count, _, rank = a.shape
    if y.shape[0] != N:
        raise ValueError(f"x and y must have the same rows, got {N} and {y.shape[0]}")
    if a.shape[1] != n_in or b.shape != (count, rank, n_out):
        raise ValueError(f"a must be [n_adapters, {n_in}, rank] and b [n_adapters, rank, {n_out}], got {tuple(a.shape)} and "
                         f"{tuple(b.shape)}")
    if not 1 <= rank <= 256:
        raise ValueError(f"rank {rank} not in [1, 256]")
    if n_in < 1 or n_out < 1:
        raise ValueError("x and y must have columns")
    B = adapter.shape[0]
    _countable(**{"rows of x": N, "columns of x": n_in, "columns of y": n_out, "adapters": count, "entries of adapter": B})
    if scale is not None:
        _tensor("scale", scale, (torch.float32,), 1)
        if scale.shape[0] != count:
            raise ValueError(f"scale must have n_adapters = {count} entries")
    if cu_new is None:
        if B != N:
            raise ValueError("adapter must have one entry per row where there is no cu_new")
    else:
        _tensor("cu_new", cu_new, (torch.int32,), 1)
        if cu_new.shape[0] != B + 1:
            raise ValueError("cu_new must have batch + 1 entries")
    if out is not None:
        _tensor("out", out, one, 2)
        if out.shape != y.shape:
            raise ValueError(f"out must be {tuple(y.shape)}, got {tuple(out.shape)}")
        _no_overlap("out", out, "y", y, x=x, a=a, b=b)
        _apart("out", out)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _no_gradient("adapter_add", y, x, a, b, scale, out)
    _on_one_gpu(x=x, y=y, a=a, b=b, adapter=adapter, scale=scale, cu_new=cu_new, out=out, workspace=workspace)


def adapter_add(y, x, a, b, adapter, *, scale=None, cu_new=None, out=None, workspace: Optional[torch.Tensor] = None,
                alloc_tensor_func: Callable = torch.empty, stream=None):
    """Low-rank adapters of many requests beside a shared projection: ``out[n] = y[n] + scale[i] * (x[n] @ a[i]) @ b[i]``
    with ``i = adapter[request of row n]`` (-1: ``out[n] = y[n]``).

    x [N, n_in], y [N, n_out] (the projection's result), a [n_adapters, n_in, rank], b [n_adapters, rank, n_out], all f16 or all
    bf16 (rows at any stride: y and out may be column slices); adapter [B] int32; scale [n_adapters] f32, None means
    1.  Rows are packed by request, `cu_new` [B + 1] int32 as in `kv_rope_append` (None: one row per request).  Returns
    out; `out=y` adds in place (an `out` that has memory of y, x, a or b otherwise is refused).  x a is summed in f32 (and, of packed
    rows, rounded to their type's number of bits, with the range of f32).  Rows behind cu_new[B] are padding: a caller's `out` keeps its
    rows, the op's own has y's there.  An adapter that does not exist adds nothing and is reported by `kernel_status`.
    `workspace`: an optional CUDA buffer of `adapter_add_workspace_bytes` bytes; calls that may run at the same time need one
    each."""
    if stream is None and alloc_tensor_func is torch.empty:
        done = _ordinary().adapter(y, x, a, b, adapter, scale, cu_new, out, workspace)
        if done is not None:
            return _done(done, "wsvd_adapter_add")
    _check_adapters(y, x, a, b, adapter, scale, cu_new, out, workspace)
    N, n_in = x.shape
    count, _, rank = a.shape
    n_out, B, dtype, index = y.shape[1], adapter.shape[0], x.dtype, x.get_device()
    own = out is None
    if own:
        out = _new(alloc_tensor_func, y, (N, n_out), dtype, stream)
    if workspace is None:
        workspace = _new(alloc_tensor_func, y, (adapter_add_workspace_bytes(N, B, n_in, rank, cu_new is not None) // 2,), dtype, stream)
        have = workspace.numel() * 2
    else:
        have = workspace.numel() * workspace.element_size()
    args = _pack_adapter(
        y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), a.data_ptr(), *a.stride()[:2], b.data_ptr(), *b.stride()[:2],
        out.data_ptr(), out.stride(0), adapter.data_ptr(), 0 if scale is None else scale.data_ptr(),
        0 if cu_new is None else cu_new.data_ptr(), N, B, n_in, n_out, rank, count, _CODE[dtype], own)
    _run("wsvd_adapter_add", index, stream, args, workspace.data_ptr(), have)
    return out


# ---- element-wise pieces of the decode step (one kernel each), launched on the device of their tensors

def _one_device(x, **others):
    for name, t in others.items():
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, expected {x.device}")


def rms_norm(x: torch.Tensor, eps: float = 1e-5, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [rows, cols] f16 -> x * rsqrt(mean(x^2) + eps), f16 (no weight vector)."""
    _cuda_tensor("x", x, (torch.float16,), 2)
    _need(x.is_contiguous(), "x must be contiguous")
    if out is None:
        out = torch.empty_like(x)
    _one_device(x, out=out)
    with _on_device(x.device):
        check(_lib.lib().wsvd_rms_norm_f16(_ptr(x), _ptr(out), x.shape[0], x.shape[1], float(eps), _stream(stream)),
              "wsvd_rms_norm_f16")
    return out


def add_rms_norm(x: torch.Tensor, delta: torch.Tensor, eps: float = 1e-5, stream=None):
    """(x + delta, RMSNorm(x + delta)) for x, delta [rows, cols] f16: the residual update and the
    next block's normalisation as one kernel."""
    _cuda_tensor("x", x, (torch.float16,), 2)
    _cuda_tensor("delta", delta, (torch.float16,), 2)
    _need(x.is_contiguous() and delta.is_contiguous() and x.shape == delta.shape, "x and delta: same contiguous shape")
    _one_device(x, delta=delta)
    x_out, y = torch.empty_like(x), torch.empty_like(x)
    with _on_device(x.device):
        check(_lib.lib().wsvd_add_rms_norm_f16(_ptr(x), _ptr(delta), _ptr(x_out), _ptr(y), x.shape[0], x.shape[1],
                                               float(eps), _stream(stream)), "wsvd_add_rms_norm_f16")
    return x_out, y


def rope_half_(q: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, stream=None) -> torch.Tensor:
    """Half-split rotary embedding of q [B, H, D] f16 in place at positions pos [B] int32;
    inv_freq [D/2] f32 on the device.  q may be a column slice of a wider matrix (any stride between
    sequences; the heads of a sequence are contiguous)."""
    _cuda_tensor("q", q, (torch.float16,), 3)
    _cuda_tensor("pos", pos, (torch.int32,), 1)
    _cuda_tensor("inv_freq", inv_freq, (torch.float32,), 1)
    _need(q.stride(1) == q.shape[2] and pos.numel() == q.shape[0] and inv_freq.numel() * 2 == q.shape[2],
          "q must be [B, H, D] with contiguous heads, B positions and D/2 frequencies")
    _one_device(q, pos=pos, inv_freq=inv_freq)
    with _on_device(q.device):
        check(_lib.lib().wsvd_rope_half_f16(_ptr(q), q.stride(0), _ptr(pos), _ptr(inv_freq), q.shape[0], q.shape[1],
                                            q.shape[2], _stream(stream)), "wsvd_rope_half_f16")
    return q


def silu_mul(up: torch.Tensor, gate: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """up * silu(gate), f16 [rows, cols]; up and gate may be column slices of one wider matrix."""
    _cuda_tensor("up", up, (torch.float16,), 2)
    _cuda_tensor("gate", gate, (torch.float16,), 2)
    _need(up.shape == gate.shape, "up and gate must have the same shape")
    if out is None:
        out = torch.empty(up.shape, dtype=up.dtype, device=up.device)
    _need(out.is_contiguous() and out.shape == up.shape, "out must be contiguous and shaped like up")
    _one_device(up, gate=gate, out=out)
    with _on_device(up.device):
        check(_lib.lib().wsvd_silu_mul_f16(_ptr(up), up.stride(0), _ptr(gate), gate.stride(0), _ptr(out), up.shape[0],
                                           up.shape[1], _stream(stream)), "wsvd_silu_mul_f16")
    return out
