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
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

import qtts_b200 as Q

NO_PAGES, ROW_FULL, ROOM, LENGTH, PAGE, TIMEOUT = 1, 2, 4, 8, 16, 32
_STATUS = {NO_PAGES: "the free list ran out", ROW_FULL: "a request outgrew its table row",
           ROOM: "more new tokens than max_tokens", LENGTH: "a negative length",
           PAGE: "a page or slot outside the pool", TIMEOUT: "a wait inside a kernel ran out"}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# the descriptors of include/qwen3tts_b200.h, field by field (all 64 bits wide)
_PLAN = struct.Struct("12Q6q").pack       # qtb_paged_plan_t
_APPEND = struct.Struct("6Q17q").pack     # qtb_paged_append_t
_ATTN = struct.Struct("10Q25qd").pack     # qtb_attn_t

# A call's host side is a few microseconds of Python next to kernels of as many:
# the checks below are flat on purpose.
_i32, _i64, _f32 = torch.int32, torch.int64, torch.float32
_this_device = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream   # what torch.cuda.current_stream(i).cuda_stream is, without the object

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


def _call(dev: int, fn, desc: bytes):
    """fn(desc, stream) on the current stream of device `dev`."""
    if dev == _this_device():
        rc = fn(desc, _stream_of(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(desc, _stream_of(dev))
    if rc:
        Q.check(rc)


def _refuse(name, want, t):
    raise ValueError(f"{name}: {want} wanted, got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _index(name, t, dev, n=None, dtype=_i32):
    """Pointer of a contiguous one-dimensional index tensor of `n` elements."""
    if t.dtype is not dtype or t.get_device() != dev or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        _refuse(name, f"contiguous {dtype} [{'*' if n is None else n}] on cuda:{dev}", t)
    return t.data_ptr()


def _table(table, dev, n):
    if table.dtype is not _i32 or table.get_device() != dev or table.dim() != 2 or table.shape[0] != n or (
            table.shape[1] > 1 and table.stride(1) != 1):
        _refuse("table", f"int32 [{n}][columns] with contiguous rows on cuda:{dev}", table)
    return table.data_ptr()


def _cuda(t):
    if not t.is_cuda:
        raise ValueError(f"CUDA tensors wanted, got one on {t.device}")
    return t.get_device()


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
    dev = _cuda(past_len)
    n = past_len.shape[0]
    ints = past_len.new_empty(2 * n + 2 + 2 * max_tokens)
    slot = past_len.new_empty(max_tokens, dtype=_i64)
    if ints.dtype is not _i32:
        _refuse("past_len", "int32", past_len)
    at = ints.data_ptr()
    _call(dev, _lib().qtb_paged_plan, _PLAN(
        _index("past_len", past_len, dev), _index("new_len", new_len, dev, n), _table(table, dev, n),
        _index("free_pages", free_pages, dev), 0 if free_head is None else _index("free_head", free_head, dev, 1),
        at, at + 4 * n + 4, slot.data_ptr(), at + 8 * n + 8, at + 8 * n + 8 + 4 * max_tokens, at + 8 * n + 4,
        0 if status is None else _index("status", status, dev, 1),
        n, max_tokens, table.shape[1], table.stride(0), free_pages.shape[0], page))
    cu, kv, head, pos, req = torch.split_with_sizes(ints, (n + 1, n, 1, max_tokens, max_tokens))
    return Plan(cu, kv, slot, pos, req, head)


def append(k, v, kpool, vpool, slot, status=None) -> None:
    """New keys and values into the cache (qtb_paged_append).

    k, v: [tokens][heads][dim] of the pools' type or f32 (rounded to nearest
    even); slot: int64 [tokens], negative = skip.  Pools: bf16 or f16
    [pages][heads][position][dim], updated in place."""
    dev = _cuda(k)
    t, h, d = k.shape
    src, dst, pools = k.dtype, kpool.dtype, kpool.shape
    if src not in _TYPES or dst not in _TYPES:
        raise ValueError(f"append: {src} into {dst} is not supported")
    if v.dtype is not src or v.get_device() != dev or v.shape != k.shape:
        _refuse("v", f"{src} {tuple(k.shape)} on cuda:{dev}", v)
    if kpool.get_device() != dev or len(pools) != 4 or pools[1] != h or pools[3] != d:
        _refuse("kpool", f"[pages][{h}][position][{d}] on cuda:{dev}", kpool)
    if vpool.dtype is not dst or vpool.get_device() != dev or vpool.shape != pools:
        _refuse("vpool", f"{dst} {tuple(pools)} on cuda:{dev}", vpool)
    ks, vs, kp, vp = k.stride(), v.stride(), kpool.stride(), vpool.stride()
    if not ks[2] == vs[2] == kp[3] == vp[3] == 1:
        raise ValueError("append: the last dimension has to be contiguous")
    _call(dev, _lib().qtb_paged_append, _APPEND(
        k.data_ptr(), v.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), _index("slot", slot, dev, t, _i64),
        0 if status is None else _index("status", status, dev, 1), ks[0], ks[1], vs[0], vs[1],
        kp[0], kp[1], kp[2], vp[0], vp[1], vp[2], t, h, d, pools[2], pools[0], _TYPES[src], _TYPES[dst]))


def _attend(q, k, v, cu, kv_len, table, pool, max_new, max_kv, scale, causal, window, out, lse, status):
    dev = _cuda(q)
    t, h, d = q.shape
    kind, n = q.dtype, cu.shape[0] - 1
    if kind not in _TYPES:
        raise ValueError(f"attention of {kind} is not supported")
    if k.dtype is not kind or k.get_device() != dev or k.dim() != 3 + pool or k.shape[-1] != d or (not pool and k.shape[0] != t):
        _refuse("kpool" if pool else "k", f"{kind} " + (f"[pages][head][position][{d}]" if pool else f"[{t}][head][{d}]") + f" on cuda:{dev}", k)
    if v.dtype is not kind or v.get_device() != dev or v.shape != k.shape:
        _refuse("vpool" if pool else "v", f"{kind} {tuple(k.shape)} on cuda:{dev}", v)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if pool:
        pages, kv, page, _ = k.shape
        lens, rows, cols, width = _index("kv_len", kv_len, dev, n), _table(table, dev, n), table.shape[1], table.stride(0)
    else:
        kv = k.shape[1]
        pages = page = lens = rows = cols = width = 0
    if out is None:
        out = q.new_empty((t, h, d))
    elif out.dtype is not kind or out.get_device() != dev or out.shape != q.shape:
        _refuse("out", f"{kind} {tuple(q.shape)} on cuda:{dev}", out)
    os = out.stride()
    if not qs[2] == ks[-1] == vs[-1] == os[2] == 1:
        raise ValueError("attention: the last dimension has to be contiguous")
    if lse is None:
        lse = q.new_empty((t, h), dtype=_f32)
    elif lse.dtype is not _f32 or lse.get_device() != dev or lse.shape != (t, h) or not lse.is_contiguous():
        _refuse("lse", f"contiguous float32 [{t}][{h}] on cuda:{dev}", lse)
    if scale is None:
        scale = 1 / math.sqrt(d)
    L = _lib()
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _index("cu_new", cu, dev), lens, rows,
            0 if status is None else _index("status", status, dev, 1))
    tail = (qs[0], qs[1], os[0], os[1], ks[0], ks[1], ks[2] if pool else 0, vs[0], vs[1], vs[2] if pool else 0,
            width, cols, page, pages, n, t, h, kv, d, max_new, max_kv, _TYPES[kind], causal, window or 0, scale)
    if dev == _this_device():
        size = L.qtb_attn_workspace(_ATTN(*head, 0, 0, *tail), pool)
    else:
        with torch.cuda.device(dev):
            size = L.qtb_attn_workspace(_ATTN(*head, 0, 0, *tail), pool)
    if size < 0:
        Q.check(size)
    at, ws = 0, None
    if size:
        ws = q.new_empty(size // 2)          # of two-byte values
        at = ws.data_ptr()
    _call(dev, L.qtb_paged_attention if pool else L.qtb_prompt_attention, _ATTN(*head, at, size, *tail))
    return out, lse


def paged_attention(q, kpool, vpool, table, cu_new, kv_len, max_new: int = 0, max_kv: int = 0, scale=None,
                    causal: bool = True, window: int = 0, out=None, lse=None, status=None):
    """Attention of each request's new tokens over its pages (qtb_paged_attention).

    q: [tokens][heads][dim], packed by cu_new (int32 [requests + 1]); kv_len:
    int32 [requests], cached tokens with the new ones, which are the last.
    window: how many keys a token looks back on, itself included (0: all).
    max_new, max_kv: bounds of new tokens and keys per request, to choose the
    split of the work (0: not known).  Returns (out, lse)."""
    return _attend(q, kpool, vpool, cu_new, kv_len, table, True, max_new, max_kv, scale, causal, window, out, lse, status)


def prompt_attention(q, k, v, cu_new, max_new: int = 0, scale=None, causal: bool = True, window: int = 0, out=None,
                     lse=None, status=None):
    """Attention within packed prompts (qtb_prompt_attention): q [tokens][heads]
    [dim], k and v [tokens][key heads][dim].  Returns (out, lse)."""
    return _attend(q, k, v, cu_new, None, None, False, max_new, max_new, scale, causal, window, out, lse, status)


def check_status(status) -> None:
    """Raise for what the kernels reported in `status` (synchronises)."""
    bits = int(status)
    if bits:
        raise RuntimeError("paged operators: " + ", ".join(t for b, t in _STATUS.items() if bits & b))
