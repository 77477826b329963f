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

_calls = None


def _lib():
    global _calls
    if _calls is None:
        L = Q.lib()
        for n in ("qtb_paged_plan", "qtb_paged_append", "qtb_paged_attention", "qtb_prompt_attention"):
            getattr(L, n).argtypes = [Q.C.c_char_p, Q._vp]
        L.qtb_attn_workspace.argtypes = [Q.C.c_char_p]
        L.qtb_attn_workspace.restype = Q.C.c_int64
        _calls = L
    return _calls


def _on(dev: torch.device, fn, desc: bytes):
    """fn(desc, stream) on the current stream of `dev`."""
    if dev.index == torch.cuda.current_device():
        rc = fn(desc, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(desc, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        Q.check(rc)


def _index(name, t, dev, dtype=torch.int32, n=None):
    """Pointer of a contiguous one-dimensional index tensor."""
    if t.dtype is not dtype or t.device != dev or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: contiguous {dtype} [{'*' if n is None else n}] on {dev} wanted, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")
    return t.data_ptr()


def _status(status, dev):
    return 0 if status is None else _index("status", status, dev, n=1)


def _table(table, dev, n_req):
    if (table.dtype is not torch.int32 or table.device != dev or table.dim() != 2 or table.shape[0] != n_req
            or (table.shape[1] > 1 and table.stride(1) != 1)):
        raise ValueError(f"table: int32 [{n_req}][columns] with contiguous rows on {dev} wanted, got {table.dtype} "
                         f"{tuple(table.shape)} with strides {table.stride()} on {table.device}")
    return table.data_ptr()


def _tensor(name, t, dev, dtype, shape):
    """Shape None = any; the last dimension is contiguous."""
    if (t.dtype is not dtype or t.device != dev or t.dim() != len(shape) or t.stride(-1) != 1
            or any(w is not None and w != s for w, s in zip(shape, t.shape))):
        want = "".join("[*]" if w is None else f"[{w}]" for w in shape)
        raise ValueError(f"{name}: {dtype} {want} with a contiguous last dimension on {dev} wanted, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _cuda(t):
    if not t.is_cuda:
        raise ValueError(f"CUDA tensors wanted, got one on {t.device}")
    return t.device


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
    ints = torch.empty(2 * n + 2 + 2 * max_tokens, dtype=torch.int32, device=dev)
    slot = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    cu, kv, head, pos, req = ints.split([n + 1, n, 1, max_tokens, max_tokens])
    at = ints.data_ptr()
    _on(dev, _lib().qtb_paged_plan, _PLAN(
        _index("past_len", past_len, dev), _index("new_len", new_len, dev, n=n), _table(table, dev, n),
        _index("free_pages", free_pages, dev), 0 if free_head is None else _index("free_head", free_head, dev, n=1),
        at, at + 4 * (n + 1), slot.data_ptr(), at + 4 * (2 * n + 2), at + 4 * (2 * n + 2 + max_tokens),
        at + 4 * (2 * n + 1), _status(status, dev),
        n, max_tokens, table.shape[1], table.stride(0), free_pages.shape[0], page))
    return Plan(cu, kv, slot, pos, req, head)


def append(k, v, kpool, vpool, slot, status=None) -> None:
    """New keys and values into the cache (qtb_paged_append).

    k, v: [tokens][heads][dim] of the pools' type or f32 (rounded to nearest
    even); slot: int64 [tokens], negative = skip.  Pools: bf16 or f16
    [pages][heads][position][dim], updated in place."""
    dev = _cuda(k)
    t, h, d = k.shape
    _tensor("k", k, dev, k.dtype, (t, h, d))
    _tensor("v", v, dev, k.dtype, (t, h, d))
    _tensor("kpool", kpool, dev, kpool.dtype, (None, h, None, d))
    _tensor("vpool", vpool, dev, kpool.dtype, kpool.shape)
    if kpool.dtype not in _TYPES or k.dtype not in _TYPES:
        raise ValueError(f"append: {k.dtype} into {kpool.dtype} is not supported")
    _on(dev, _lib().qtb_paged_append, _APPEND(
        k.data_ptr(), v.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), _index("slot", slot, dev, torch.int64, t),
        _status(status, dev), *k.stride()[:2], *v.stride()[:2], *kpool.stride()[:3], *vpool.stride()[:3],
        t, h, d, kpool.shape[2], kpool.shape[0], _TYPES[k.dtype], _TYPES[kpool.dtype]))


def _attend(fn, q, k, v, cu, kv_len, table, pool, max_new, max_kv, scale, causal, window, out, lse, status):
    dev = _cuda(q)
    t, h, d = q.shape
    if q.dtype not in _TYPES:
        raise ValueError(f"attention of {q.dtype} is not supported")
    n = cu.shape[0] - 1
    if pool:
        pages, kv, page, _ = k.shape
        _tensor("kpool", k, dev, q.dtype, (None, None, None, d))
        _tensor("vpool", v, dev, q.dtype, k.shape)
        lens, rows, cols, width = _index("kv_len", kv_len, dev, n=n), _table(table, dev, n), table.shape[1], table.stride(0)
        ks, vs = k.stride()[:3], v.stride()[:3]
    else:
        kv = k.shape[1]
        _tensor("k", k, dev, q.dtype, (t, None, d))
        _tensor("v", v, dev, q.dtype, k.shape)
        pages = page = lens = rows = cols = width = 0
        ks, vs = (*k.stride()[:2], 0), (*v.stride()[:2], 0)
    _tensor("q", q, dev, q.dtype, (t, h, d))
    if out is None:
        out = torch.empty((t, h, d), dtype=q.dtype, device=dev)
    else:
        _tensor("out", out, dev, q.dtype, (t, h, d))
    if lse is None:
        lse = torch.empty((t, h), dtype=torch.float32, device=dev)
    elif lse.dtype is not torch.float32 or lse.device != dev or lse.shape != (t, h) or not lse.is_contiguous():
        raise ValueError(f"lse: contiguous float32 [{t}][{h}] on {dev} wanted")
    L = _lib()
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _index("cu_new", cu, dev), lens, rows,
            _status(status, dev))
    tail = (*q.stride()[:2], *out.stride()[:2], *ks, *vs, width, cols, page, pages, n, t, h, kv, d, max_new, max_kv,
            _TYPES[q.dtype], bool(causal), window or 0, 1 / math.sqrt(d) if scale is None else scale)
    size = L.qtb_attn_workspace(_ATTN(*head, 0, 0, *tail))
    if size < 0:
        Q.check(size)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _on(dev, getattr(L, fn), _ATTN(*head, ws.data_ptr(), size, *tail))
    return out, lse


def paged_attention(q, kpool, vpool, table, cu_new, kv_len, max_new: int = 0, max_kv: int = 0, scale=None,
                    causal: bool = True, window: int = 0, out=None, lse=None, status=None):
    """Attention of each request's new tokens over its pages (qtb_paged_attention).

    q: [tokens][heads][dim], packed by cu_new (int32 [requests + 1]); kv_len:
    int32 [requests], cached tokens with the new ones, which are the last.
    window: how many keys a token looks back on, itself included (0: all).
    max_new, max_kv: bounds of new tokens and keys per request, to choose the
    split of the work (0: not known).  Returns (out, lse)."""
    return _attend("qtb_paged_attention", q, kpool, vpool, cu_new, kv_len, table, True, max_new, max_kv, scale, causal,
                   window, out, lse, status)


def prompt_attention(q, k, v, cu_new, max_new: int = 0, scale=None, causal: bool = True, window: int = 0, out=None,
                     lse=None, status=None):
    """Attention within packed prompts (qtb_prompt_attention): q [tokens][heads]
    [dim], k and v [tokens][key heads][dim].  Returns (out, lse)."""
    return _attend("qtb_prompt_attention", q, k, v, cu_new, None, None, False, max_new, max_new, scale, causal, window,
                   out, lse, status)


def check_status(status) -> None:
    """Raise for what the kernels reported in `status` (synchronises)."""
    bits = int(status)
    if bits:
        raise RuntimeError("paged operators: " + ", ".join(t for b, t in _STATUS.items() if bits & b))
