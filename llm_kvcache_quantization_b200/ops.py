"""Thin tensor-level wrappers over the C ABI (pointers, strides, stream, workspace).

torch is used for device memory, streams and dtype bookkeeping only; all
arithmetic happens in libkvq.so.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import (FMT_FP16, FMT_INT4, FMT_INT8, F_ADAPTIVE, F_MIXED_RESCUE, F_RESCUE_THR,
                   SCALE_ASYM_MINMAX, SCALE_DYNAMIC_PCT, SCALE_STATIC)

_WORKSPACES = {}


def _stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_cuda(*tensors) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("libkvq requires CUDA tensors (there is no CPU path).")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"device mismatch: {t.device} vs {dev}")
    return dev


_RETIRED = []      # outgrown workspaces: a CUDA graph captured earlier may still hold their addresses


def get_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Per-(device, stream) scratch buffer for split-K partials; grows, never shrinks.  A buffer that has been handed
    out is never returned to the allocator while the process lives (unless `release_workspaces` is called): a CUDA
    graph captured around an earlier call replays with the old address, which must stay ours."""
    key = (device.index, _stream_ptr(device))
    buf = _WORKSPACES.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _RETIRED.append(buf)
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WORKSPACES[key] = buf
    return buf


def release_workspaces() -> None:
    """Drop every scratch buffer.  Only when no captured graph that used them will be replayed again."""
    _WORKSPACES.clear()
    _RETIRED.clear()


_LAST_SPLITS = 0


def last_splits() -> int:
    """KV split count used by the most recent decode_attn call (diagnostics)."""
    return _LAST_SPLITS


# --------------------------------------------------------------------------- append
def _append_side(src, payload, scale, zp, scale_f32, side, static_scale, rescue_thr) -> _lib.KvqAppendSide:
    s = _lib.KvqAppendSide()
    if src.stride(-1) != 1:
        raise ValueError("new K/V tokens must be contiguous in head_dim")
    s.src = src.data_ptr()
    s.src_stride_b, s.src_stride_h, s.src_stride_t = src.stride(0), src.stride(1), src.stride(2)
    es = payload.element_size()
    if payload.stride(-1) != 1:
        raise ValueError("cache payload must be contiguous in its last dimension")
    s.payload = payload.data_ptr()
    s.pay_stride_b, s.pay_stride_h, s.pay_stride_s = (payload.stride(0) * es, payload.stride(1) * es,
                                                      payload.stride(2) * es)
    if scale is not None:
        if scale.dtype != torch.float16 or scale.stride(-1) != 1:
            raise ValueError("cache scale buffer must be fp16, contiguous in groups")
        s.scale = scale.data_ptr()
        s.sc_stride_b, s.sc_stride_h, s.sc_stride_s = scale.stride(0), scale.stride(1), scale.stride(2)
    if zp is not None:
        if zp.dtype != torch.float16 or zp.stride() != scale.stride():
            raise ValueError("zero-point buffer must be fp16 with the strides of the scale buffer")
        s.zp = zp.data_ptr()
    if scale_f32 is not None:
        if scale_f32.dtype != torch.float32 or scale_f32.stride() != scale.stride():
            raise ValueError("fp32 scale copy must share the strides of the fp16 scale buffer")
        s.scale_f32 = scale_f32.data_ptr()
    if side is not None:
        if side.dtype != torch.float16 or side.stride(-1) != 1:
            raise ValueError("outlier side buffer must be fp16, contiguous in its last dimension")
        s.side = side.data_ptr()
        s.side_stride_b, s.side_stride_h, s.side_stride_s = side.stride(0), side.stride(1), side.stride(2)
    if static_scale is not None:
        if static_scale.dtype not in (torch.float16, torch.float32) or not static_scale.is_contiguous():
            raise ValueError("static scale table must be a contiguous fp16/fp32 [Hkv, G] tensor")
        s.static_scale = static_scale.data_ptr()
        s.static_scale_is_f32 = 1 if static_scale.dtype == torch.float32 else 0
    if rescue_thr is not None:
        s.rescue_threshold = rescue_thr.data_ptr()
    return s


def quantize_append(fmt: int, policy: int, k_new: torch.Tensor, v_new: torch.Tensor,
                    k_payload: torch.Tensor, v_payload: torch.Tensor,
                    k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                    write_pos, group_size: int, *,
                    k_zp=None, v_zp=None, k_scale_f32=None, v_scale_f32=None,
                    k_static=None, v_static=None, flags: int = 0, adaptive_margin: float = 1.0,
                    quantile: float = 1.0, k_rescue_thr=None, v_rescue_thr=None,
                    outlier_idx=None, k_side=None, v_side=None,
                    rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                    q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None):
    """Quantize `k_new`, `v_new` ([B,Hkv,T,D] fp16) into cache slots
    [write_pos, write_pos+T) of the given payload / scale buffers in one launch (`v_new=None`: K side only).
    `write_pos` is an int or an int32 device tensor (read on the device).

    With `rope_cos` / `rope_sin` (fp16 [B or 1, T, rotary_dim]) the same launch applies rotate-half
    RoPE to K before quantizing it and, when `q` ([B,Hq,T,D] fp16, before rotation) is given, to the
    query; the rotated query is returned (`q_out` or a new tensor)."""
    dev = _require_cuda(k_new, v_new, k_payload, v_payload, k_scale, v_scale)
    if k_new.dtype != torch.float16 or (v_new is not None and v_new.dtype != torch.float16):
        raise ValueError("quantize_append expects fp16 K/V")
    if k_new.ndim != 4 or (v_new is not None and k_new.shape != v_new.shape):
        raise ValueError(f"k/v shape mismatch or not 4D: {tuple(k_new.shape)}")
    B, H, T, D = k_new.shape
    a = _lib.KvqAppendArgs()
    a.format, a.policy, a.flags = fmt, policy, flags
    a.B, a.Hkv, a.T, a.D = B, H, T, D
    a.group_size = group_size
    a.adaptive_margin = float(adaptive_margin)
    a.quantile = float(quantile)
    if outlier_idx is not None:
        if outlier_idx.dtype != torch.int16 or not outlier_idx.is_contiguous() or outlier_idx.shape[0] != H:
            raise ValueError("outlier_idx must be a contiguous int16 [Hkv, n_out] tensor")
        a.n_out = outlier_idx.shape[1]
        a.outlier_idx = outlier_idx.data_ptr()
    # the kernel itself refuses slots at or beyond the smallest destination buffer (a device-side position that ran
    # past the capacity stores nothing and raises bit 1 of kvq_debug_error_flag)
    cap = k_payload.shape[2] if v_payload is None or v_new is None else min(k_payload.shape[2], v_payload.shape[2])
    a.max_slots = cap
    if isinstance(write_pos, torch.Tensor):
        if write_pos.dtype != torch.int32 or not write_pos.is_cuda:
            raise ValueError("device write_pos must be an int32 CUDA tensor")
        a.write_pos_dev = write_pos.data_ptr()
    else:
        a.write_pos = int(write_pos)
        if a.write_pos < 0 or a.write_pos + T > cap:
            raise ValueError(f"append of {T} tokens at {a.write_pos} exceeds capacity {cap}")
    a.k = _append_side(k_new, k_payload, k_scale, k_zp, k_scale_f32, k_side, k_static, k_rescue_thr)
    if v_new is not None:
        a.v = _append_side(v_new, v_payload, v_scale, v_zp, v_scale_f32, v_side, v_static, v_rescue_thr)
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    if q is not None and rope_cos is None:
        raise ValueError("a query is only taken together with rope_cos / rope_sin")
    if rope_cos is not None:
        for name, t in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
            if t.dtype != torch.float16 or t.ndim != 3 or t.stride(-1) != 1 or t.shape[1] != T or \
                    t.shape[0] not in (1, B) or not t.is_cuda:
                raise ValueError(f"{name} must be an fp16 CUDA tensor [B or 1, T, rotary_dim]")
        if rope_cos.shape != rope_sin.shape or rope_cos.stride() != rope_sin.stride():
            raise ValueError("rope_cos / rope_sin must share shape and strides")
        rd = rope_cos.shape[-1]
        if rd % 2 or rd > D:
            raise ValueError(f"RoPE dim {rd} must be even and <= head_dim {D}")
        a.rope_cos, a.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
        a.rope_stride_b = 0 if rope_cos.shape[0] == 1 else rope_cos.stride(0)
        a.rope_stride_t = rope_cos.stride(1)
        a.rotary_dim = rd
        if q is not None:
            if q.dtype != torch.float16 or q.ndim != 4 or q.shape[0] != B or q.shape[2] != T or q.shape[3] != D or \
                    q.stride(-1) != 1:
                raise ValueError("q must be fp16 [B, Hq, T, D], contiguous in head_dim")
            if q_out is None:
                q_out = torch.empty((B, q.shape[1], T, D), dtype=torch.float16, device=dev)
            elif q_out.shape != q.shape or q_out.dtype != torch.float16 or q_out.stride(-1) != 1:
                raise ValueError("q_out must match q")
            a.Hq = q.shape[1]
            a.q_src = q.data_ptr()
            a.q_stride_b, a.q_stride_h, a.q_stride_t = q.stride(0), q.stride(1), q.stride(2)
            a.q_out = q_out.data_ptr()
            a.qo_stride_b, a.qo_stride_h, a.qo_stride_t = q_out.stride(0), q_out.stride(1), q_out.stride(2)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_quantize_append(C.byref(a), _stream_ptr(dev))
    _lib.check("kvq_quantize_append", rc)
    return q_out


# --------------------------------------------------------------------------- attention
def _cache_side(payload, scale, zp, side) -> _lib.KvqCacheSide:
    s = _lib.KvqCacheSide()
    es = payload.element_size()
    s.payload = payload.data_ptr()
    s.pay_stride_b, s.pay_stride_h, s.pay_stride_s = (payload.stride(0) * es, payload.stride(1) * es,
                                                      payload.stride(2) * es)
    if scale is not None:
        s.scale = scale.data_ptr()
        s.sc_stride_b, s.sc_stride_h, s.sc_stride_s = scale.stride(0), scale.stride(1), scale.stride(2)
    if zp is not None:
        if zp.stride() != scale.stride():
            raise ValueError("zero-points must share the strides of the scales")
        s.zp = zp.data_ptr()
    if side is not None:
        s.side = side.data_ptr()
        s.side_stride_b, s.side_stride_h, s.side_stride_s = side.stride(0), side.stride(1), side.stride(2)
    return s


def decode_attn(fmt: int, q: torch.Tensor, k_payload: torch.Tensor, v_payload: torch.Tensor,
                k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                context_lens: Optional[torch.Tensor], sm_scale: float, *, head_dim: int,
                k_zp=None, v_zp=None, inv_tau: Optional[torch.Tensor] = None,
                outlier_idx=None, k_side=None, v_side=None,
                splits: int = 0, out: Optional[torch.Tensor] = None,
                return_partial: bool = False, max_ctx: Optional[int] = None, stages: int = 0,
                packed_partial: Optional[torch.Tensor] = None, fast_dequant: Optional[bool] = None,
                tail_tokens: int = 0, exchange: Optional[dict] = None,
                q_chan_scale: Optional[torch.Tensor] = None):
    """Fused q_len==1 attention over a (quantized) cache.  q fp16 [B,Hq,D].

    Returns `out` fp16 [B,Hq,D]; with `return_partial` also the normalised
    partial `(o fp32 [B,Hq,D], m fp32 [B,Hq], l fp32 [B,Hq])` used by the
    sequence-sharded merge.  `packed_partial` (fp32 [B,Hq,D+2], contiguous) receives the
    same partial as one buffer `[o (D) | m | l]` per (b, h) - the send buffer of the
    sequence-sharded all-gather.  No host synchronisation happens here.

    `exchange` (sequence sharding, see `parallel.PeerExchange`): the combine stage becomes the fused
    combine / peer-store exchange / merge kernel, and `out` receives the attention over ALL ranks' tokens.
    """
    dev = _require_cuda(q, k_payload, v_payload, k_scale, v_scale, context_lens)
    if q.dtype != torch.float16:
        raise ValueError("decode_attn expects an fp16 query")
    B, Hq, D = q.shape
    if D != head_dim:
        raise ValueError(f"Head dim mismatch: q={D}, expected {head_dim}")
    Hkv = k_payload.shape[1]
    S = k_payload.shape[2]
    a = _lib.KvqAttnArgs()
    a.format = fmt
    a.B, a.Hq, a.Hkv, a.D = B, Hq, Hkv, D
    G = 1 if k_scale is None else k_scale.shape[-1]
    a.group_size = D // G
    a.max_ctx = S if max_ctx is None else min(int(max_ctx), S)
    if q.stride(-1) != 1:
        q = q.contiguous()
    a.q = q.data_ptr()
    a.q_stride_b, a.q_stride_h = q.stride(0), q.stride(1)
    if inv_tau is not None:
        if inv_tau.dtype != torch.float32 or not inv_tau.is_contiguous() or inv_tau.numel() != Hq:
            raise ValueError("inv_tau must be a contiguous fp32 [Hq] tensor")
        a.inv_tau = inv_tau.data_ptr()
    a.sm_scale = float(sm_scale)
    a.stages = int(stages)
    # packed INT4, groups of >= 32 channels: 0 = library default (factored scales), 1 = factored scales, 2 = bit-faithful
    # fp16 dequantisation; KVQ_INT4_FAST=1 / 0 picks one for calls that do not say
    if fast_dequant is None:
        env = os.environ.get("KVQ_INT4_FAST")
        a.fast_dequant = 0 if env is None else (1 if env == "1" else 2)
    else:
        a.fast_dequant = 1 if fast_dequant else 2
    if q_chan_scale is not None:       # fp32 [B, Hkv, D]: per-channel factor applied to the query inside the kernel
        if q_chan_scale.dtype != torch.float32 or tuple(q_chan_scale.shape) != (B, Hkv, D) or q_chan_scale.stride(-1) != 1:
            raise ValueError("q_chan_scale must be an fp32 [B, Hkv, D] tensor, contiguous in head_dim")
        a.q_chan_scale = q_chan_scale.data_ptr()
        a.qcs_stride_b, a.qcs_stride_h = q_chan_scale.stride(0), q_chan_scale.stride(1)
    a.tail_tokens = int(tail_tokens)   # 1: the last token of each row is attended by the combine stage (see kvq.h)
    a.k = _cache_side(k_payload, k_scale, k_zp, k_side)
    a.v = _cache_side(v_payload, v_scale, v_zp, v_side)
    if outlier_idx is not None:
        a.n_out = outlier_idx.shape[1]
        a.outlier_idx = outlier_idx.data_ptr()
    if context_lens is not None:        # None: every row attends over all max_ctx tokens of the view
        if context_lens.dtype != torch.int32 or not context_lens.is_contiguous():
            context_lens = context_lens.to(torch.int32).contiguous()
        a.context_lens = context_lens.data_ptr()
    lib = _lib.load()
    with torch.cuda.device(dev):
        a.splits = int(splits) if splits else int(lib.kvq_decode_pick_splits(C.byref(a)))
        global _LAST_SPLITS
        _LAST_SPLITS = a.splits
        need = int(lib.kvq_decode_workspace_bytes(B, Hq, D, a.splits))
        ws = get_workspace(dev, need)
        a.workspace = ws.data_ptr()
        a.workspace_bytes = ws.numel()
        if out is None:
            out = torch.empty((B, Hq, D), dtype=torch.float16, device=dev)
        a.out = out.data_ptr()
        a.out_stride_b, a.out_stride_h = out.stride(0), out.stride(1)
        part = None
        if return_partial:
            po = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
            pm = torch.empty((B, Hq), dtype=torch.float32, device=dev)
            pl = torch.empty((B, Hq), dtype=torch.float32, device=dev)
            a.part_o, a.part_m, a.part_l = po.data_ptr(), pm.data_ptr(), pl.data_ptr()
            part = (po, pm, pl)
        elif packed_partial is not None:
            pp = packed_partial
            if pp.dtype != torch.float32 or not pp.is_contiguous() or tuple(pp.shape) != (B, Hq, D + 2):
                raise ValueError("packed_partial must be a contiguous fp32 [B, Hq, D+2] tensor")
            a.part_o, a.part_m, a.part_l = pp.data_ptr(), pp.data_ptr() + 4 * D, pp.data_ptr() + 4 * (D + 1)
            a.part_o_stride = a.part_ml_stride = D + 2
            part = (pp[..., :D], pp[..., D], pp[..., D + 1])
        if exchange is not None:
            if return_partial or packed_partial is not None or not (B > 0 and a.max_ctx > 0):
                raise ValueError("exchange needs a non-empty local chunk and no partial outputs")
            rc = 0
            if a.stages != 2:
                a.stages = 1
                rc = lib.kvq_decode_attn(C.byref(a), _stream_ptr(dev))
            if rc == 0 and int(stages) != 1:
                combine_exchange(exchange["peer_ptrs"], exchange["rank"], exchange["slot"], exchange["slots"],
                                 exchange["epoch"], out, splits=a.splits, status=exchange.get("status"),
                                 wait_ns=exchange.get("wait_ns", 0), tail_attn=a if a.tail_tokens else None)
        elif B > 0 and a.max_ctx > 0:
            rc = lib.kvq_decode_attn(C.byref(a), _stream_ptr(dev))
        else:
            # nothing cached (an empty sequence shard): zeros, and the neutral partial (l = 0, m = -inf)
            rc = 0
            out.zero_()
            if part is not None:
                part[0].zero_(); part[1].fill_(float("-inf")); part[2].zero_()
    _lib.check("kvq_decode_attn", rc)
    if return_partial:
        return out, part
    return out


def group_absmax(x: torch.Tensor, group_size: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp32 [H, G] table of max |x| per (head, channel group) over batch rows and tokens of `x`
    ([B,H,S,D] or [H,S,D] fp16); max-accumulates into `out` when given (zero-filled by the caller)."""
    dev = _require_cuda(x)
    if x.dtype != torch.float16:
        raise ValueError("group_absmax expects an fp16 tensor")
    if x.ndim == 3:
        x = x[None]
    if x.ndim != 4 or x.stride(-1) != 1:
        raise ValueError("expected [B,H,S,D] (or [H,S,D]) with a contiguous last dimension")
    B, H, S, D = x.shape
    gs = D if group_size == -1 else int(group_size)
    if gs <= 0 or D % gs != 0:
        raise ValueError(f"head_dim ({D}) must be divisible by group_size ({group_size})")
    if out is None:
        out = torch.zeros((H, D // gs), dtype=torch.float32, device=dev)
    elif out.dtype != torch.float32 or tuple(out.shape) != (H, D // gs) or not out.is_contiguous():
        raise ValueError("out must be a contiguous fp32 [H, G] tensor")
    a = _lib.KvqAbsmaxArgs()
    a.B, a.H, a.S, a.D, a.group_size = B, H, S, D, gs
    a.x = x.data_ptr()
    a.stride_b, a.stride_h, a.stride_s = x.stride(0), x.stride(1), x.stride(2)
    a.out = out.data_ptr()
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_group_absmax(C.byref(a), _stream_ptr(dev))
    _lib.check("kvq_group_absmax", rc)
    return out


def neutral_partial(B: int, Hq: int, D: int, dev) -> None:
    """Fill the split-K workspace with ONE empty split per (batch, head) row (o = 0, m = -inf, l = 0):
    what a rank without cached tokens hands to `combine_exchange`."""
    need = int(_lib.load().kvq_decode_workspace_bytes(B, Hq, D, 1))
    ws = get_workspace(torch.device(dev), need)
    o_bytes = (B * Hq * D * 4 + 255) & ~255
    ws[:o_bytes].zero_()
    ml = ws[o_bytes:o_bytes + B * Hq * 8].view(torch.float32).view(B * Hq, 2)
    ml[:, 0] = float("-inf")
    ml[:, 1] = 0.0


def exchange_bytes(B: int, Hq: int, D: int, slots: int, world: int) -> int:
    """Bytes of one rank's receive buffer of the fused exchange."""
    return int(_lib.load().kvq_exchange_bytes(B, Hq, D, slots, world))


def combine_exchange(peer_ptrs, rank: int, slot: int, slots: int, epoch: torch.Tensor, out: torch.Tensor, *,
                     splits: int, status: Optional[torch.Tensor] = None, wait_ns: int = 0,
                     tail_attn=None) -> torch.Tensor:
    """Second half of a sequence-sharded decode_attn(..., stages=1) call on this rank: merge the KV
    splits left in the workspace, exchange the normalised partial with every peer by direct stores
    into their receive buffers (`peer_ptrs[q]` = rank q's buffer mapped into this process), wait for
    theirs and write the merged fp16 `out` [B,Hq,D].  One launch; `epoch` is a device int32 >= 1."""
    dev = _require_cuda(out, epoch)
    B, Hq, D = out.shape
    world = len(peer_ptrs)
    if out.dtype != torch.float16 or out.stride(-1) != 1:
        raise ValueError("out must be an fp16 [B,Hq,D] tensor, contiguous in head_dim")
    if epoch.dtype != torch.int32 or (status is not None and status.dtype != torch.int32):
        raise ValueError("epoch / status must be int32 device tensors")
    x = _lib.KvqExchangeArgs()
    x.B, x.Hq, x.D, x.splits = B, Hq, D, int(splits)
    need = int(_lib.load().kvq_decode_workspace_bytes(B, Hq, D, x.splits))
    ws = get_workspace(dev, need)
    x.workspace, x.workspace_bytes = ws.data_ptr(), ws.numel()
    x.rank, x.world = int(rank), world
    arr = (C.c_void_p * world)(*[int(p) for p in peer_ptrs])
    x.peer_base = C.cast(arr, C.POINTER(C.c_void_p))
    x.slot, x.slots = int(slot), int(slots)
    x.epoch = epoch.data_ptr()
    x.wait_ns = int(wait_ns)
    x.status = status.data_ptr() if status is not None else None
    x.out = out.data_ptr()
    x.out_stride_b, x.out_stride_h = out.stride(0), out.stride(1)
    if tail_attn is not None:          # the KvqAttnArgs of the stage-1 call (tail_tokens = 1)
        x.tail_attn = C.pointer(tail_attn)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_combine_exchange(C.byref(x), _stream_ptr(dev))
    _lib.check("kvq_combine_exchange", rc)
    return out


def dequantize(fmt: int, k_payload: torch.Tensor, v_payload: Optional[torch.Tensor], k_scale: torch.Tensor,
               v_scale: Optional[torch.Tensor], *, k_zp=None, v_zp=None, outlier_idx=None, k_side=None, v_side=None):
    """Quantized cache views -> fp16 [B,Hkv,S,D] (K and V in one launch; V optional).
    Values are RN16(code * scale) (+ zero-point, rounded again); outlier channels take the side value."""
    dev = _require_cuda(k_payload, v_payload, k_scale, v_scale)
    if k_payload.dtype != torch.int8 or k_scale.dtype != torch.float16:
        raise ValueError("dequantize expects an int8 payload and fp16 scales")
    B, H, S, Dp = k_payload.shape
    D = Dp * 2 if fmt == _lib.FMT_INT4 else Dp
    a = _lib.KvqDequantArgs()
    a.format, a.B, a.Hkv, a.S, a.D = fmt, B, H, S, D
    a.group_size = D // k_scale.shape[-1]
    if k_payload.stride(-1) != 1 or (v_payload is not None and v_payload.stride(-1) != 1):
        raise ValueError("payload last dimension must be contiguous")
    a.k = _cache_side(k_payload, k_scale, k_zp, k_side)
    k_out = torch.empty((B, H, S, D), dtype=torch.float16, device=dev)
    a.k_out = k_out.data_ptr()
    v_out = None
    if v_payload is not None:
        if v_payload.shape != k_payload.shape:
            raise ValueError("k / v payload shapes differ")
        a.v = _cache_side(v_payload, v_scale, v_zp, v_side)
        v_out = torch.empty_like(k_out)
        a.v_out = v_out.data_ptr()
    a.out_stride_b, a.out_stride_h, a.out_stride_s = k_out.stride(0), k_out.stride(1), k_out.stride(2)
    if outlier_idx is not None:
        if outlier_idx.dtype != torch.int16 or not outlier_idx.is_contiguous() or outlier_idx.shape[0] != H:
            raise ValueError("outlier_idx must be a contiguous int16 [Hkv, n_out] tensor")
        a.n_out = outlier_idx.shape[1]
        a.outlier_idx = outlier_idx.data_ptr()
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_dequantize(C.byref(a), _stream_ptr(dev))
    _lib.check("kvq_dequantize", rc)
    return k_out, v_out


def decode_kernel_kind(fmt: int, q, k_payload, v_payload, k_scale, v_scale, *, k_zp=None, v_zp=None,
                       n_out: int = 0) -> int:
    """Which kernel kvq_decode_attn would launch for these tensors: 1 = tensor-core TMA kernel,
    0 = generic kernel.  Pure host-side query (no launch)."""
    a = _lib.KvqAttnArgs()
    B, Hq, D = q.shape
    a.format, a.B, a.Hq, a.Hkv, a.D = fmt, B, Hq, k_payload.shape[1], D
    a.group_size = D // (1 if k_scale is None else k_scale.shape[-1])
    a.max_ctx = k_payload.shape[2]
    a.q, a.q_stride_b, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.k = _cache_side(k_payload, k_scale, k_zp, None)
    a.v = _cache_side(v_payload, v_scale, v_zp, None)
    a.n_out = n_out
    return int(_lib.load().kvq_decode_kernel_kind(C.byref(a)))


def lse_combine(part_o: torch.Tensor, part_m: torch.Tensor, part_l: torch.Tensor,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Merge P normalised partials ([P,B,Hq,D], [P,B,Hq], [P,B,Hq] fp32) -> fp16 [B,Hq,D]."""
    dev = _require_cuda(part_o, part_m, part_l)
    P, B, Hq, D = part_o.shape
    for t in (part_o, part_m, part_l):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("partials must be contiguous fp32 tensors")
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float16, device=dev)
    c = _lib.KvqCombineArgs()
    c.P, c.B, c.Hq, c.D = P, B, Hq, D
    c.part_o, c.part_m, c.part_l = part_o.data_ptr(), part_m.data_ptr(), part_l.data_ptr()
    c.out = out.data_ptr()
    c.out_stride_b, c.out_stride_h = out.stride(0), out.stride(1)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_lse_combine(C.byref(c), _stream_ptr(dev))
    _lib.check("kvq_lse_combine", rc)
    return out


def lse_combine_packed(packed: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Merge P packed partials (fp32 [P,B,Hq,D+2], rows `[o (D) | m | l]`, e.g. the receive buffer
    of an all-gather) -> fp16 [B,Hq,D]."""
    dev = _require_cuda(packed)
    if packed.dtype != torch.float32 or not packed.is_contiguous() or packed.ndim != 4:
        raise ValueError("packed partials must be a contiguous fp32 [P, B, Hq, D+2] tensor")
    P, B, Hq, W = packed.shape
    D = W - 2
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float16, device=dev)
    c = _lib.KvqCombineArgs()
    c.P, c.B, c.Hq, c.D = P, B, Hq, D
    base = packed.data_ptr()
    c.part_o, c.part_m, c.part_l = base, base + 4 * D, base + 4 * (D + 1)
    c.part_o_stride = c.part_ml_stride = W
    c.part_o_stride_p = c.part_ml_stride_p = B * Hq * W
    c.out = out.data_ptr()
    c.out_stride_b, c.out_stride_h = out.stride(0), out.stride(1)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_lse_combine(C.byref(c), _stream_ptr(dev))
    _lib.check("kvq_lse_combine", rc)
    return out


def decode_attn_static(fmt: int, q: torch.Tensor, k_payload: torch.Tensor, v_payload: torch.Tensor,
                       k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                       context_lens: Optional[torch.Tensor], sm_scale: float, out: torch.Tensor, *,
                       k_zp=None, v_zp=None, inv_tau: Optional[torch.Tensor] = None,
                       outlier_idx=None, k_side=None, v_side=None, splits: int = 0) -> torch.Tensor:
    """Fused decode attention through `kvq_decode_attn_static`, the entry point for hosts that are
    not allowed to allocate GPU memory at call time (for instance a serving process whose memory
    pool already owns all of HBM).  The split-K partials go to an 8 MiB array inside the library
    instead of a torch-allocated workspace, and this wrapper allocates nothing either: the caller
    passes `out` (fp16 [B,Hq,D]).

    Raises `KvqError` with code `KVQ_ELIMIT` when B*Hq*splits*(D+2)*4 bytes exceed the array.
    Calls on one device share that array: keep them on one stream (overlapping calls race).
    The first call per device resolves the array's address; do it before capturing a CUDA graph.
    """
    dev = _require_cuda(q, k_payload, v_payload, k_scale, v_scale, context_lens, out)
    if q.dtype != torch.float16 or out.dtype != torch.float16:
        raise ValueError("decode_attn_static expects fp16 q and out")
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("q and out must be contiguous in head_dim")
    B, Hq, D = q.shape
    a = _lib.KvqAttnArgs()
    a.format = fmt
    a.B, a.Hq, a.Hkv, a.D = B, Hq, k_payload.shape[1], D
    a.group_size = D // (1 if k_scale is None else k_scale.shape[-1])
    a.max_ctx = k_payload.shape[2]
    a.q, a.q_stride_b, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    if inv_tau is not None:
        a.inv_tau = inv_tau.data_ptr()
    a.sm_scale = float(sm_scale)
    a.k = _cache_side(k_payload, k_scale, k_zp, k_side)
    a.v = _cache_side(v_payload, v_scale, v_zp, v_side)
    if outlier_idx is not None:
        a.n_out = outlier_idx.shape[1]
        a.outlier_idx = outlier_idx.data_ptr()
    if context_lens is not None:
        if context_lens.dtype != torch.int32 or not context_lens.is_contiguous():
            raise ValueError("context_lens must be a contiguous int32 tensor (no conversion is done here)")
        a.context_lens = context_lens.data_ptr()
    a.splits = int(splits)
    a.out, a.out_stride_b, a.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_decode_attn_static(C.byref(a), _stream_ptr(dev))
    _lib.check("kvq_decode_attn_static", rc)
    return out


# --------------------------------------------------------------------------- bounded and paged caches
def _scratch(nbytes: int, device) -> torch.Tensor:
    """Scratch memory of ONE call.  From torch's allocator and not from a buffer kept per stream: a call inside a graph
    capture gets memory of that graph's pool, so graphs captured on one stream do not share it when they are replayed
    side by side."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def cache_format(payload: torch.Tensor, head_dim: int) -> int:
    """Payload format by dtype and width: fp16 [.., D], int8 [.., D], or nibble-packed [.., D/2]."""
    if payload.dtype == torch.float16:
        if payload.shape[-1] != head_dim:
            raise ValueError(f"Head dim mismatch: q={head_dim}, cache={payload.shape[-1]}")
        return FMT_FP16
    if payload.dtype != torch.int8:
        raise ValueError(f"cache payload must be torch.float16 or torch.int8, got {payload.dtype}")
    if payload.shape[-1] == head_dim:
        return FMT_INT8
    if payload.shape[-1] * 2 == head_dim:
        return FMT_INT4
    raise ValueError(f"Head dim mismatch: q={head_dim}, int8 payload width {payload.shape[-1]} "
                     "(expected head_dim, or head_dim / 2 for packed INT4)")


def _check_pool(fmt: int, head_dim: int, k, v, k_scale, v_scale, k_zp, v_zp) -> int:
    """Shapes, types and layout of one cache (contiguous or pool); returns the group size."""
    if k.ndim != 4 or v.ndim != 4:
        raise ValueError(f"cache payload must be 4D, got {tuple(k.shape)} / {tuple(v.shape)}")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k/v cache mismatch: {tuple(k.shape)} {k.dtype} vs {tuple(v.shape)} {v.dtype}")
    for name, t in (("k", k), ("v", v)):
        es = t.element_size()
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} cache inner dim must be contiguous (stride=1), got stride={t.stride(-1)}")
        if t.data_ptr() % 16 or any(t.stride(d) * es % 16 for d in range(3) if t.shape[d] > 1):
            raise ValueError(f"{name} cache rows must start on 16-byte boundaries, got strides {t.stride()}")
    if fmt == FMT_FP16:
        if any(t is not None for t in (k_scale, v_scale, k_zp, v_zp)):
            raise ValueError("an fp16 cache has no scales and no zero-points")
        return head_dim
    if k_scale is None or v_scale is None:
        raise ValueError("a quantized cache needs k_scale and v_scale")
    if (k_zp is None) != (v_zp is None):
        raise ValueError("k_zp and v_zp go together")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale), ("k_zp", k_zp), ("v_zp", v_zp)):
        if t is None:
            continue
        if t.dtype != torch.float16 or t.ndim != 4 or t.shape[:3] != k.shape[:3]:
            raise ValueError(f"{name} must be fp16 with the leading shape of the cache {tuple(k.shape[:3])}, "
                             f"got {t.dtype} {tuple(t.shape)}")
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in its groups")
    groups = k_scale.shape[3]
    if v_scale.shape[3] != groups:
        raise ValueError(f"k_scale/v_scale num_groups mismatch: k={groups} vs v={v_scale.shape[3]}.")
    if groups <= 0 or head_dim % groups or (head_dim // groups) % 8:
        raise ValueError(f"head_dim {head_dim} must be a multiple of num_groups {groups} with groups of a multiple of 8 channels")
    for z, s in ((k_zp, k_scale), (v_zp, v_scale)):
        if z is not None and (z.shape != s.shape or z.stride() != s.stride()):
            raise ValueError("zero-points must share the shape and strides of the scales")
    return head_dim // groups


def _int32(t: torch.Tensor, what: str, n: int) -> torch.Tensor:
    if t.ndim != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must be 1D with one entry per batch row ({n}), got {tuple(t.shape)}")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _page_table(table: torch.Tensor, batch: int, pool: torch.Tensor) -> _lib.KvqPageTable:
    if table.dtype != torch.int32 or table.ndim != 2 or table.shape[0] != batch or table.shape[1] < 1:
        raise ValueError(f"block_table must be int32 [B={batch}, pages >= 1], got {table.dtype} {tuple(table.shape)}")
    if table.shape[1] > 1 and table.stride(1) != 1:
        raise ValueError("block_table rows must be contiguous")
    if pool.shape[0] < 1 or pool.shape[2] < 1:
        raise ValueError(f"the page pool {tuple(pool.shape)} holds no token")
    return _lib.KvqPageTable(table.data_ptr(), table.stride(0), table.shape[1], pool.shape[2], pool.shape[0])


_MARSHAL = None


def _marshal():
    """_marshal.so takes the ordinary calls of the functions below; it returns None, with nothing done, for any other, and
    the function then goes on in Python, where every check, conversion and message is."""
    global _MARSHAL
    _MARSHAL = _lib.marshal()
    return _MARSHAL


def span_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor],
              v_scale: Optional[torch.Tensor], context_lens: Optional[torch.Tensor], sm_scale: Optional[float] = None, *,
              k_zp=None, v_zp=None, block_table: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0,
              weights: Optional[torch.Tensor] = None, max_ctx: Optional[int] = None,
              inv_tau: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q_len == 1 attention over the visible span of a contiguous cache [B, Hkv, S, .] or, with `block_table`, of page
    pools [num_pages, Hkv, page_size, .] (`kvq_span_attn`).  No host synchronisation: lengths are clamped on the device."""
    done = (_MARSHAL or _marshal()).span_attn(q, k, v, k_scale, v_scale, context_lens, sm_scale, k_zp, v_zp, block_table,
                                              window, sinks, weights, max_ctx, inv_tau, out)
    if done is not None:
        return done
    dev = _require_cuda(q, k, v, k_scale, v_scale, k_zp, v_zp, context_lens, block_table, weights, inv_tau, out)
    if q.ndim != 3:
        raise ValueError(f"q must have shape [B, Hq, D], got {tuple(q.shape)}")
    if q.dtype != torch.float16:
        raise ValueError("span_attn expects an fp16 query")
    B, Hq, D = q.shape
    if D not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {D}")
    fmt = cache_format(k, D)
    gs = _check_pool(fmt, D, k, v, k_scale, v_scale, k_zp, v_zp)
    Hkv = k.shape[1]
    if Hkv < 1 or Hq % Hkv != 0:
        raise ValueError(f"GQA head mismatch: q_heads={Hq} must be a multiple of kv_heads={Hkv}")
    if window is None:
        if sinks:
            raise ValueError("sinks go with a window")
        window = 0
    elif window < 1 or sinks < 0:
        raise ValueError(f"window must be >= 1 and sinks >= 0, got {window}, {sinks}")
    window, sinks = min(int(window), 2 ** 31 - 1), min(int(sinks), 2 ** 31 - 1)     # no row is longer
    s = _lib.KvqSpanAttnArgs()
    a = s.attn
    if block_table is None:
        if k.shape[0] != B:
            raise ValueError(f"Batch mismatch: q={B}, k={k.shape[0]}")
        span = k.shape[2]
        if span >= 2 ** 31:
            raise ValueError(f"a cache holds less than 2^31 slots, got {span}")
    else:
        s.pages = _page_table(block_table, B, k)
        span = min(block_table.shape[1] * k.shape[2], 2 ** 31 - 1)
    if max_ctx is not None:
        if max_ctx < 0:
            raise ValueError(f"max_ctx must be >= 0, got {max_ctx}")
        span = min(span, int(max_ctx))
    if q.stride(2) != 1 or q.stride(0) % 2 or q.stride(1) % 2 or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float16, device=dev)
    elif out.dtype != torch.float16 or tuple(out.shape) != (B, Hq, D) or out.stride(2) != 1:
        raise ValueError("out must be an fp16 [B, Hq, D] tensor, contiguous in head_dim")
    a.format, a.B, a.Hq, a.Hkv, a.D, a.group_size, a.max_ctx = fmt, B, Hq, Hkv, D, gs, span
    a.q, a.q_stride_b, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.out, a.out_stride_b, a.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    a.sm_scale = 1.0 / D ** 0.5 if sm_scale is None else float(sm_scale)
    if inv_tau is not None:
        if inv_tau.numel() != Hq:
            raise ValueError(f"inv_tau must have one entry per query head ({Hq}), got {tuple(inv_tau.shape)}")
        inv_tau = inv_tau.to(torch.float32).contiguous()
        a.inv_tau = inv_tau.data_ptr()
    if context_lens is not None:
        context_lens = _int32(context_lens, "context_lens", B)
        a.context_lens = context_lens.data_ptr()
    elif block_table is not None:
        raise ValueError("a paged cache needs context_lens")
    a.k = _cache_side(k, k_scale, k_zp, None)
    a.v = _cache_side(v, v_scale, v_zp, None)
    s.window, s.sinks = window, sinks
    if weights is not None:
        if weights.dtype != torch.float32 or weights.ndim != 3 or weights.shape[:2] != (B, Hkv) or weights.shape[2] < span:
            raise ValueError(f"weights must be fp32 [B={B}, Hkv={Hkv}, >= {span}], got {weights.dtype} {tuple(weights.shape)}")
        if weights.shape[2] > 1 and weights.stride(2) != 1 or \
                any(weights.shape[d] > 1 and weights.stride(d) < weights.shape[2] for d in (0, 1)):
            raise ValueError("weights must be contiguous in its slots, with rows that do not overlap")
        s.weights, s.w_stride_b, s.w_stride_h = weights.data_ptr(), weights.stride(0), weights.stride(1)
    if B == 0:
        return out
    lib = _lib.load()
    with torch.cuda.device(dev):
        need = int(lib.kvq_span_attn_workspace_bytes(C.byref(s)))
        ws = _scratch(max(need, 256), dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = lib.kvq_span_attn(C.byref(s), _stream_ptr(dev))
    _lib.check("kvq_span_attn", rc)
    return out


def paged_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor], block_table: torch.Tensor,
                 start_pos: torch.Tensor, new_lens: Optional[torch.Tensor] = None, *, k_zp=None, v_zp=None,
                 k_static=None, v_static=None, clip_percentile: float = 100.0) -> None:
    """Quantize new tokens [B, Hkv, T, D] into pages, one launch (`kvq_paged_append`): token t of row b goes to position
    start_pos[b] + t of the row, t < new_lens[b] (default: all).  Scales: min / max with zero-points when zero-point pools
    are given, the static tables [Hkv, G] when those are given, else the `clip_percentile` of each group's magnitudes."""
    if (_MARSHAL or _marshal()).paged_append(k_new, v_new, k_pages, v_pages, k_scale, v_scale, block_table, start_pos, new_lens,
                                             k_zp, v_zp, k_static, v_static, clip_percentile):
        return
    dev = _require_cuda(k_new, v_new, k_pages, v_pages, k_scale, v_scale, k_zp, v_zp, block_table, start_pos, new_lens,
                        k_static, v_static)
    if k_new.ndim != 4 or k_new.shape != v_new.shape:
        raise ValueError(f"k/v shape mismatch or not 4D: {tuple(k_new.shape)} vs {tuple(v_new.shape)}")
    B, H, T, D = k_new.shape
    fmt = cache_format(k_pages, D)
    gs = _check_pool(fmt, D, k_pages, v_pages, k_scale, v_scale, k_zp, v_zp)
    if k_pages.shape[1] != H:
        raise ValueError(f"heads mismatch: new tokens {H}, pages {k_pages.shape[1]}")
    if (k_static is None) != (v_static is None):
        raise ValueError("k_static and v_static go together")
    if k_static is not None and (k_zp is not None or fmt == FMT_FP16):
        raise ValueError("static scales are for symmetric quantized pages")
    if not 0.0 < clip_percentile <= 100.0:
        raise ValueError(f"clip_percentile must be in (0, 100], got {clip_percentile}")
    for name, t in (("k_static", k_static), ("v_static", v_static)):
        if t is not None and (tuple(t.shape) != (H, D // gs) or t.dtype not in (torch.float16, torch.float32)
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp16/fp32 [Hkv={H}, G={D // gs}] tensor, got {t.dtype} {tuple(t.shape)}")
    k_new, v_new = k_new.to(torch.float16), v_new.to(torch.float16)
    if k_new.stride(3) != 1:
        k_new = k_new.contiguous()
    if v_new.stride(3) != 1:
        v_new = v_new.contiguous()
    p = _lib.KvqPagedAppendArgs()
    p.pages = _page_table(block_table, B, k_pages)
    start_pos = _int32(start_pos, "start_pos", B)
    p.start_pos = start_pos.data_ptr()
    if new_lens is not None:
        new_lens = _int32(new_lens, "new_lens", B)
        p.new_lens = new_lens.data_ptr()
    a = p.append
    a.format, a.B, a.Hkv, a.T, a.D, a.group_size = fmt, B, H, T, D, gs
    a.adaptive_margin = 1.0
    a.quantile = clip_percentile / 100.0 if clip_percentile < 100.0 else 1.0
    a.policy = SCALE_STATIC if fmt == FMT_FP16 or k_static is not None else \
        SCALE_ASYM_MINMAX if k_zp is not None else SCALE_DYNAMIC_PCT
    a.k = _append_side(k_new, k_pages, k_scale, k_zp, None, None, k_static, None)
    a.v = _append_side(v_new, v_pages, v_scale, v_zp, None, None, v_static, None)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_paged_append(C.byref(p), _stream_ptr(dev))
    _lib.check("kvq_paged_append", rc)


def paged_read(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: Optional[torch.Tensor],
               v_scale: Optional[torch.Tensor], block_table: torch.Tensor, start_pos: Optional[torch.Tensor], tokens: int,
               lens: Optional[torch.Tensor] = None, *, head_dim: int, k_zp=None, v_zp=None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens start_pos[b] + t (default start 0), t < lens[b] (default `tokens`), of every row as fp16 (k, v)
    [B, Hkv, tokens, head_dim]; zeros behind lens[b] (`kvq_paged_read`).  Values are code * scale (+ zero-point), rounded
    once.  `head_dim` tells nibble-packed pages (width head_dim / 2) from INT8 ones."""
    done = (_MARSHAL or _marshal()).paged_read(k_pages, v_pages, k_scale, v_scale, block_table, start_pos, tokens, lens,
                                               head_dim, k_zp, v_zp)
    if done is not None:
        return done
    dev = _require_cuda(k_pages, v_pages, k_scale, v_scale, k_zp, v_zp, block_table, start_pos, lens)
    D, T = int(head_dim), int(tokens)
    if D not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {D}")
    if T < 0:
        raise ValueError(f"tokens must be >= 0, got {T}")
    fmt = cache_format(k_pages, D)
    gs = _check_pool(fmt, D, k_pages, v_pages, k_scale, v_scale, k_zp, v_zp)
    B, H = block_table.shape[0], k_pages.shape[1]
    p = _lib.KvqPagedReadArgs()
    p.pages = _page_table(block_table, B, k_pages)
    p.format, p.B, p.Hkv, p.T, p.D, p.group_size = fmt, B, H, T, D, gs
    if start_pos is not None:
        start_pos = _int32(start_pos, "start_pos", B)
        p.start_pos = start_pos.data_ptr()
    if lens is not None:
        lens = _int32(lens, "lens", B)
        p.lens = lens.data_ptr()
    p.k = _cache_side(k_pages, k_scale, k_zp, None)
    p.v = _cache_side(v_pages, v_scale, v_zp, None)
    k = torch.empty((B, H, T, D), dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    p.k_out, p.v_out = k.data_ptr(), v.data_ptr()
    p.out_stride_b, p.out_stride_h, p.out_stride_t = k.stride(0), k.stride(1), k.stride(2)
    with torch.cuda.device(dev):
        rc = _lib.load().kvq_paged_read(C.byref(p), _stream_ptr(dev))
    _lib.check("kvq_paged_read", rc)
    return k, v


def evict(weights: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor, seen: torch.Tensor, budget: int, buffers,
          *, sinks: int = 0, recent: int = 0) -> torch.Tensor:
    """Shrink every (batch row, kv head) of a contiguous cache to `budget` tokens, in place (`kvq_evict`); returns the new
    lengths, int32 [B]."""
    buffers = tuple(buffers)
    done = (_MARSHAL or _marshal()).evict(weights, positions, lengths, seen, budget, buffers, sinks, recent)
    if done is not None:
        return done
    dev = _require_cuda(weights, positions, lengths, seen, *buffers)
    if weights.dtype != torch.float32 or weights.ndim != 3:
        raise ValueError(f"weights must be fp32 [B, Hkv, slots], got {weights.dtype} {tuple(weights.shape)}")
    if positions.dtype != torch.int32 or positions.shape != weights.shape:
        raise ValueError(f"positions must be int32 {tuple(weights.shape)}, got {positions.dtype} {tuple(positions.shape)}")
    B, H, cap = weights.shape
    for name, t in (("weights", weights), ("positions", positions)):
        if (cap > 1 and t.stride(2) != 1) or any(t.shape[d] > 1 and t.stride(d) < cap for d in (0, 1)):
            raise ValueError(f"{name} must be contiguous in its slots, with rows that do not overlap")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"need budget >= 1 and 0 <= sinks + recent <= budget, got {budget}, {sinks}, {recent}")
    if budget >= 2 ** 31:
        raise ValueError(f"budget must be less than 2^31, got {budget}")
    if len(buffers) > _lib.EVICT_MAX_BUFS:
        raise ValueError(f"at most {_lib.EVICT_MAX_BUFS} buffers, got {len(buffers)}")
    e = _lib.KvqEvictArgs()
    e.B, e.Hkv, e.cap, e.budget, e.sinks, e.recent = B, H, cap, budget, sinks, recent
    for i, t in enumerate(buffers):
        if t.ndim < 3 or t.shape[:2] != (B, H) or t.shape[2] < cap:
            raise ValueError(f"buffer {i} must be [B={B}, Hkv={H}, >= {cap} slots, ...], got {tuple(t.shape)}")
        row = 1
        for d in range(t.ndim - 1, 2, -1):
            if t.shape[d] > 1 and t.stride(d) != row:
                raise ValueError(f"buffer {i}: the row of a slot must be contiguous")
            row *= t.shape[d]
        if any(t.shape[d] > 1 and t.stride(d) < row for d in range(3)):
            raise ValueError(f"buffer {i}: rows must not overlap, got strides {t.stride()}")
        if row == 0:
            raise ValueError(f"buffer {i} has empty rows: {tuple(t.shape)}")
        es = t.element_size()
        e.bufs[i] = _lib.KvqEvictBuf(t.data_ptr(), t.stride(0) * es, t.stride(1) * es, t.stride(2) * es, row * es)
    e.n_bufs = len(buffers)
    lengths, seen = _int32(lengths, "lengths", B), _int32(seen, "seen", B)
    new = torch.empty(B, dtype=torch.int32, device=dev)
    if B == 0 or H == 0:
        return new
    e.lengths, e.seen, e.new_lengths = lengths.data_ptr(), seen.data_ptr(), new.data_ptr()
    e.weights, e.w_stride_b, e.w_stride_h = weights.data_ptr(), weights.stride(0), weights.stride(1)
    e.positions, e.p_stride_b, e.p_stride_h = positions.data_ptr(), positions.stride(0), positions.stride(1)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws = _scratch(int(lib.kvq_evict_workspace_bytes(B, H, cap, budget)), dev)
        e.workspace, e.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = lib.kvq_evict(C.byref(e), _stream_ptr(dev))
    _lib.check("kvq_evict", rc)
    return new
