"""Operators of a serving step over a paged KV cache, on torch CUDA tensors.

    got = plan(past_len, new_len, table, free_pages, page, max_tokens)
    append(k, v, kpool, vpool, got.slot)                      # per layer
    out, lse = paged_attention(q, kpool, vpool, table, got.cu_new, got.kv_len,
                               max_new, max_kv)               # per layer
    out, lse = prompt_attention(q, k, v, cu_new, max_new)     # whole prompts, no cache

The kernels are those of include/qwen3tts_b200.h (qtb_paged_plan,
qtb_paged_append, qtb_paged_attention, qtb_prompt_attention); this module
checks tensors, allocates results and passes pointers.  Every call is
asynchronous on the current stream of the tensors' device, so tensors that
another stream made or still uses need the usual torch ordering
(wait_stream / record_stream).  Pools are [page][head][position][dim] with any
strides over a contiguous last dimension, so a pool laid out [page][position]
[head][dim] is passed as pool.transpose(1, 2).

What the device finds wrong with lengths, pages or slots (QTB_PS_* below) is
ORed into `status`, an int32 tensor of one element that the caller zeroes and
reads when it likes; check_status raises for it.

These are operators of serving and have no backward: attention of tensors that
require a gradient returns results whose backward raises, and what append writes
into a cache is data.
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

import qtts_b200 as Q

NO_PAGES, ROW_FULL, ROOM, LENGTH, PAGE, TIMEOUT = 1, 2, 4, 8, 16, 32
_STATUS = {NO_PAGES: "the free list ran out", ROW_FULL: "a request outgrew its table row",
           ROOM: "more new tokens than max_tokens", LENGTH: "a negative length, or offsets that fall or leave the tokens",
           PAGE: "a page or slot outside the pool", TIMEOUT: "a wait inside a kernel ran out"}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# the descriptors of include/qwen3tts_b200.h, field by field (all 64 bits wide)
_PLAN = struct.Struct("12Q6q").pack       # qtb_paged_plan_t
_APPEND = struct.Struct("6Q17q").pack     # qtb_paged_append_t
_ATTN = struct.Struct("10Q25qd").pack     # qtb_attn_t

# A call's host side is a few microseconds of Python beside kernels of as many, so
# each function checks all of its tensors in one condition, and names what is wrong
# (_refuse) only when that fails.
_i32, _i64, _f32 = torch.int32, torch.int64, torch.float32
_this_device = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream   # what torch.cuda.current_stream(i).cuda_stream is, without the object

_NEEDS = -6                 # QTB_E_WORKSPACE
_sizes = {}                 # bytes of workspace of paged calls by (device, head_dim, few rows?)
_calls = None


def _lib():
    global _calls
    if _calls is None:
        L = Q.lib()
        for n in ("qtb_paged_plan", "qtb_paged_append", "qtb_paged_attention", "qtb_prompt_attention"):
            getattr(L, n).argtypes = [Q.C.c_char_p, Q._vp]
        L.qtb_attn_workspace.argtypes = [Q.C.c_char_p, Q.C.c_int]
        L.qtb_attn_workspace.restype = Q.C.c_int64
        _calls = L
    return _calls


def _on_device(dev: int, fn, *args):
    if dev == _this_device():
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _refuse(dev, *wanted):
    """Raise for the first tensor that is not as wanted: (name, tensor, dtype, shape with None for any extent)."""
    for name, t, dtype, shape in wanted:
        if t is None:
            continue
        if not (t.is_cuda and t.get_device() == dev and t.dtype is dtype and t.dim() == len(shape)
                and all(w is None or w == s for w, s in zip(shape, t.shape)) and (t.dim() == 0 or t.stride(-1) == 1 or t.shape[-1] < 2)
                and (t.dim() != 1 or t.is_contiguous())):
            dims = "".join("[*]" if w is None else f"[{w}]" for w in shape)
            raise ValueError(f"{name}: {dtype} {dims}, contiguous in its last dimension, on cuda:{dev} wanted, got {t.dtype} "
                             f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")
    raise ValueError("tensors that do not go together")


class Plan(NamedTuple):
    cu_new: torch.Tensor     # int32 [requests + 1] packed offsets of the new tokens
    kv_len: torch.Tensor     # int32 [requests] past + new
    slot: torch.Tensor       # int64 [max_tokens] place of each new token in the cache, -1 behind the last
    pos: torch.Tensor        # int32 [max_tokens] its position
    req: torch.Tensor        # int32 [max_tokens] its request
    free_head: torch.Tensor  # int32 [1] first page of the list that is still free


def plan(past_len, new_len, table, free_pages, page: int, max_tokens: int, free_head=None, status=None) -> Plan:
    """Block tables and slot maps from request lengths (qtb_paged_plan).

    past_len, new_len: int32 [requests], cached and new tokens; table: int32
    [requests][columns], its rows hold the pages of the cached tokens and
    receive those of the new ones, taken in request order from free_pages
    (int32) at free_head (int32 [1], default 0; pass the last plan's)."""
    dev = past_len.get_device()
    n = past_len.numel()
    cols = table.shape[-1]
    if not (dev >= 0 and past_len.dtype is new_len.dtype is table.dtype is free_pages.dtype is _i32
            and past_len.shape == new_len.shape == (n,) and table.shape == (n, cols) and free_pages.dim() == 1
            and new_len.get_device() == table.get_device() == free_pages.get_device() == dev
            and past_len.is_contiguous() and new_len.is_contiguous() and free_pages.is_contiguous()
            and (cols < 2 or table.stride(1) == 1)
            and (free_head is None or free_head.dtype is _i32 and free_head.shape == (1,) and free_head.get_device() == dev)
            and (status is None or status.dtype is _i32 and status.shape == (1,) and status.get_device() == dev)):
        _refuse(dev, ("past_len", past_len, _i32, (n,)), ("new_len", new_len, _i32, (n,)), ("table", table, _i32, (n, None)),
                ("free_pages", free_pages, _i32, (None,)), ("free_head", free_head, _i32, (1,)), ("status", status, _i32, (1,)))
    ints = past_len.new_empty(2 * n + 2 + 2 * max_tokens)
    slot = past_len.new_empty(max_tokens, dtype=_i64)
    at = ints.data_ptr()
    rc = _on_device(dev, _lib().qtb_paged_plan, _PLAN(
        past_len.data_ptr(), new_len.data_ptr(), table.data_ptr(), free_pages.data_ptr(),
        0 if free_head is None else free_head.data_ptr(), at, at + 4 * n + 4, slot.data_ptr(), at + 8 * n + 8,
        at + 8 * n + 8 + 4 * max_tokens, at + 8 * n + 4, 0 if status is None else status.data_ptr(),
        n, max_tokens, cols, table.stride(0), free_pages.shape[0], page), _stream_of(dev))
    if rc:
        Q.check(rc)
    cu, kv, head, pos, req = torch.split_with_sizes(ints, (n + 1, n, 1, max_tokens, max_tokens))
    return Plan(cu, kv, slot, pos, req, head)


def append(k, v, kpool, vpool, slot, status=None) -> None:
    """New keys and values into the cache (qtb_paged_append).

    k, v: [tokens][heads][dim] of the pools' type or f32 (rounded to nearest
    even); slot: int64 [tokens], negative = skip.  Pools: bf16 or f16
    [pages][heads][position][dim], updated in place."""
    dev = k.get_device()
    t, h, d = shape = k.shape
    pages, _, page, _ = pools = kpool.shape
    src, dst = k.dtype, kpool.dtype
    ks, vs, kp, vp = k.stride(), v.stride(), kpool.stride(), vpool.stride()
    if not (dev >= 0 and src in _TYPES and dst in _TYPES and v.dtype is src and vpool.dtype is dst and slot.dtype is _i64
            and v.shape == shape and pools[1] == h and pools[3] == d and vpool.shape == pools and slot.shape == (t,)
            and v.get_device() == kpool.get_device() == vpool.get_device() == slot.get_device() == dev
            and ks[2] == vs[2] == kp[3] == vp[3] == 1 and slot.is_contiguous()
            and (status is None or status.dtype is _i32 and status.shape == (1,) and status.get_device() == dev)):
        _refuse(dev, ("k", k, src if src in _TYPES else _f32, (t, h, d)), ("v", v, src, (t, h, d)),
                ("kpool", kpool, dst if dst in _TYPES else torch.bfloat16, (None, h, None, d)), ("vpool", vpool, dst, tuple(pools)),
                ("slot", slot, _i64, (t,)), ("status", status, _i32, (1,)))
    rc = _on_device(dev, _lib().qtb_paged_append, _APPEND(
        k.data_ptr(), v.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), slot.data_ptr(), 0 if status is None else status.data_ptr(),
        ks[0], ks[1], vs[0], vs[1], kp[0], kp[1], kp[2], vp[0], vp[1], vp[2], t, h, d, page, pages, _TYPES[src], _TYPES[dst]),
        _stream_of(dev))
    if rc:
        Q.check(rc)


def _results(q, out, lse, status, dev):
    """out and lse of a call: those given, checked, or new ones."""
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    elif not (out.dtype is q.dtype and out.shape == q.shape and out.stride(2) == 1 and out.get_device() == dev):
        _refuse(dev, ("out", out, q.dtype, tuple(q.shape)))
    if lse is None:
        lse = q.new_empty(q.shape[:2], dtype=_f32)
    elif not (lse.dtype is _f32 and lse.shape == q.shape[:2] and lse.is_contiguous() and lse.get_device() == dev):
        raise ValueError(f"lse: contiguous {_f32} {tuple(q.shape[:2])} on cuda:{dev} wanted, got {lse.dtype} {tuple(lse.shape)} with "
                         f"strides {lse.stride()} on {lse.device}")
    if status is not None and not (status.dtype is _i32 and status.shape == (1,) and status.get_device() == dev):
        _refuse(dev, ("status", status, _i32, (1,)))
    return out, lse


class _NoBackward(torch.autograd.Function):
    """Results that were computed from tensors which require a gradient: asking for it raises."""

    @staticmethod
    def forward(ctx, out, lse, *inputs):
        ctx.mark_dirty(out, lse)
        return out, lse

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("paged operators: attention has no backward")


def _wants_gradient(out, lse) -> bool:
    """Whether a call on tensors that require a gradient is recorded."""
    if not torch.is_grad_enabled():
        return False
    if out is not None or lse is not None:
        raise RuntimeError("paged operators: out and lse cannot be given where an input requires a gradient (use no_grad)")
    return True


def _attend(fn, pool, dev, q, head, tail, few=False):
    """One attention call with the workspace that calls of its kind have needed so far, and again with what
    qtb_attn_workspace asks for where that is not enough."""
    key = (dev, q.shape[2], few) if pool else None
    size = _sizes.get(key, 0)
    ws = q.new_empty(size // 2) if size else None          # of two-byte values
    rc = _on_device(dev, fn, _ATTN(*head, 0 if ws is None else ws.data_ptr(), size, *tail), _stream_of(dev))
    if rc == _NEEDS:
        size = _on_device(dev, _lib().qtb_attn_workspace, _ATTN(*head, 0, 0, *tail), pool)
        if size < 0:
            Q.check(size)
        if pool:
            _sizes[key] = size
        ws = q.new_empty(size // 2)
        rc = _on_device(dev, fn, _ATTN(*head, ws.data_ptr(), size, *tail), _stream_of(dev))
    if rc:
        Q.check(rc)


def paged_attention(q, kpool, vpool, table, cu_new, kv_len, max_new: int = 0, max_kv: int = 0, scale=None,
                    causal: bool = True, window: int = 0, out=None, lse=None, status=None):
    """Attention of each request's new tokens over its pages (qtb_paged_attention).

    q: [tokens][heads][dim], packed by cu_new (int32 [requests + 1]); kv_len:
    int32 [requests], cached tokens with the new ones, which are the last.
    window: how many keys a token looks back on, itself included (0: all).
    max_new, max_kv: bounds of new tokens and keys per request, to choose the
    split of the work (0: not known).  Returns (out, lse), whose rows past
    cu_new[-1] are not written."""
    dev = q.get_device()
    t, h, d = q.shape
    pages, kv, page, _ = pools = kpool.shape
    n, cols, kind = kv_len.numel(), table.shape[-1], q.dtype
    qs, ks, vs = q.stride(), kpool.stride(), vpool.stride()
    if not (dev >= 0 and kind in _TYPES and kpool.dtype is vpool.dtype is kind and table.dtype is cu_new.dtype is kv_len.dtype is _i32
            and pools[3] == d and vpool.shape == pools and table.shape == (n, cols) and cu_new.shape == (n + 1,) and kv_len.dim() == 1
            and kpool.get_device() == vpool.get_device() == table.get_device() == cu_new.get_device() == kv_len.get_device() == dev
            and qs[2] == ks[3] == vs[3] == 1 and (cols < 2 or table.stride(1) == 1) and cu_new.is_contiguous() and kv_len.is_contiguous()):
        _refuse(dev, ("q", q, kind if kind in _TYPES else torch.bfloat16, (t, h, d)), ("kpool", kpool, kind, (None, None, None, d)),
                ("vpool", vpool, kind, tuple(pools)), ("table", table, _i32, (n, None)), ("cu_new", cu_new, _i32, (n + 1,)),
                ("kv_len", kv_len, _i32, (n,)))
    grad = (q.requires_grad or kpool.requires_grad or vpool.requires_grad) and _wants_gradient(out, lse)
    out, lse = _results(q, out, lse, status, dev)
    os = out.stride()
    _attend(_lib().qtb_paged_attention, 1, dev, q,
            (q.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), out.data_ptr(), lse.data_ptr(), cu_new.data_ptr(), kv_len.data_ptr(),
             table.data_ptr(), 0 if status is None else status.data_ptr()),
            (qs[0], qs[1], os[0], os[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table.stride(0), cols, page, pages, n, t, h, kv, d,
             max_new, max_kv, _TYPES[kind], causal, window or 0, 1 / math.sqrt(d) if scale is None else scale),
            0 < max_new * h <= 16 * kv)
    return _NoBackward.apply(out, lse, q, kpool, vpool) if grad else (out, lse)


def prompt_attention(q, k, v, cu_new, max_new: int = 0, scale=None, causal: bool = True, window: int = 0, out=None,
                     lse=None, status=None):
    """Attention within packed prompts (qtb_prompt_attention): q [tokens][heads]
    [dim], k and v [tokens][key heads][dim].  Returns (out, lse)."""
    dev = q.get_device()
    t, h, d = q.shape
    kv, n, kind = k.shape[1], cu_new.numel() - 1, q.dtype
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if not (dev >= 0 and n >= 0 and kind in _TYPES and k.dtype is v.dtype is kind and cu_new.dtype is _i32
            and k.shape == v.shape == (t, kv, d) and cu_new.dim() == 1
            and k.get_device() == v.get_device() == cu_new.get_device() == dev
            and qs[2] == ks[2] == vs[2] == 1 and cu_new.is_contiguous()):
        _refuse(dev, ("q", q, kind if kind in _TYPES else torch.bfloat16, (t, h, d)), ("k", k, kind, (t, None, d)), ("v", v, kind, (t, kv, d)),
                ("cu_new", cu_new, _i32, (None,)))
    grad = (q.requires_grad or k.requires_grad or v.requires_grad) and _wants_gradient(out, lse)
    out, lse = _results(q, out, lse, status, dev)
    os = out.stride()
    _attend(_lib().qtb_prompt_attention, 0, dev, q,
            (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), cu_new.data_ptr(), 0, 0,
             0 if status is None else status.data_ptr()),
            (qs[0], qs[1], os[0], os[1], ks[0], ks[1], 0, vs[0], vs[1], 0, 0, 0, 0, 0, n, t, h, kv, d,
             max_new, max_new, _TYPES[kind], causal, window or 0, 1 / math.sqrt(d) if scale is None else scale))
    return _NoBackward.apply(out, lse, q, k, v) if grad else (out, lse)


def check_status(status) -> None:
    """Raise for what the kernels reported in `status` (synchronises)."""
    bits = int(status)
    if bits:
        raise RuntimeError("paged operators: " + ", ".join(t for b, t in _STATUS.items() if bits & b))
