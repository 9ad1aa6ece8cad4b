"""Attention operators (include/mrl_kv.h): a paged key/value cache held in 8 bits, attention over it, and
sliding-window attention over ragged 16-bit inputs. Tensors are torch CUDA tensors.

    cache = KvCache.create(layers, pages, kv_heads, head_dim, max_seqs, max_pages)
    cache.reserve(seqs, new_tokens)                    # int32 CUDA tensors
    cache.append(layer, k, v, seqs, cu)                # quantise the new rows
    out = cache.attend(layer, q, seqs, cu, max_q=...)  # or one token per sequence: cache.attend(layer, q, seqs)
    cache.fork(parents, children); cache.release(seqs); cache.trim(seqs, window, sinks); cache.compact()

    out = window_attention(q, k, v, cu, max_len, causal=False, window=512)

Every call is asynchronous and ordered after the work on torch's current stream, and later work on that
stream after it: a Device whose launches are on that stream (Device.use_torch_stream) needs nothing for
this, another one gets events. What only the contents of index tensors can show (a sequence out of
range, a full pool) does not raise: it sets bits of `cache.status`, and a page operation does nothing, while
append, read and attend leave out the rows that are meant (not stored, 0, 0 with lse -inf).

Nothing here has a backward pass: a tensor that requires gradients is refused while gradients are recorded.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional

from ._capi import AttnC, KvCacheC, check
from .api import Device, default_device

PAGE_TOKENS = 64  # MRL_KV_PAGE
KV_NO_PAGES, KV_ROW_FULL, KV_BAD_INDEX, KV_NONFINITE, KV_TIMEOUT = 1, 2, 4, 8, 16
HEAD_DIMS = (64, 128, 256)

_ATTN = struct.Struct("@8P8q10IfI")
assert _ATTN.size == C.sizeof(AttnC)


_torch_module = None
_dtype_codes = {}
_raw_stream = None


def _torch():
    global _torch_module, _raw_stream
    if _torch_module is None:
        import torch

        _torch_module = torch
        _dtype_codes.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _torch_module


def _call(dev: Device, fn, *args) -> None:
    """One entry point of the library, its work after torch's current stream and that stream after it."""
    stream = _raw_stream(dev.index) or 1
    if stream == dev.torch_stream:
        rc = fn(dev.ptr, *args)
    else:
        check(dev.ptr, dev.lib.mrl_ctx_join(dev.ptr, stream, 1))
        rc = fn(dev.ptr, *args)
        check(dev.ptr, dev.lib.mrl_ctx_join(dev.ptr, stream, 0))
    if rc:
        check(dev.ptr, rc)


def _index(x, name: str, dev: Device, n: Optional[int] = None):
    """An int32 CUDA vector of the context's device."""
    torch = _torch_module
    if x.dtype is not torch.int32 or x.dim() != 1 or x.get_device() != dev.index:
        raise ValueError(f"{name} must be a 1-d int32 tensor on cuda:{dev.index}")
    if x.stride(0) != 1 and x.shape[0] > 1:
        raise ValueError(f"{name} must be contiguous")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, not {x.shape[0]}")
    return x


def _rows(x, name: str, dev: Device, heads=None, dims=None, dtype=None, tokens=None):
    """A [tokens, heads, dims] 16-bit tensor whose dims are contiguous; (row stride, head stride)."""
    shape = x.shape
    if len(shape) != 3 or x.get_device() != dev.index or _dtype_codes.get(x.dtype, 2) == 2:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] float16 or bfloat16 tensor on cuda:{dev.index}")
    t, h, d = shape
    if (heads is not None and h != heads) or (dims is not None and d != dims) or (tokens is not None and t != tokens):
        raise ValueError(f"{name} has shape {tuple(x.shape)}; expected [{tokens if tokens is not None else 'tokens'}, "
                         f"{heads if heads is not None else 'heads'}, {dims if dims is not None else 'head_dim'}]")
    if dtype is not None and x.dtype is not dtype:
        raise ValueError(f"{name} is {x.dtype}, not {dtype}")
    if x.requires_grad and _torch_module.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and there is none here: call under torch.no_grad() or detach it")
    row, head, one = x.stride()
    if one != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return (row if t > 1 else h * d), (head if h > 1 else d)


class KvCache:
    """A paged key/value cache held in 8 bits, over tensors that the caller owns (struct mrl_kv_cache):

    codes int8 [layers, pages, 2, kv_heads, 64 * head_dim], scales float32 [layers, pages, 2, kv_heads],
    tables int32 [max_seqs, max_pages] (-1: no page), lens int32 [max_seqs], refs int32 [pages], status
    int32 [1] (KV_* bits, made here when not given). A page holds 64 tokens of a sequence; the K and the V
    of each head have one scale per page, value = code * scale."""

    def __init__(self, codes, scales, tables, lens, refs, status=None, dev: Optional[Device] = None):
        torch = _torch()
        self.dev = dev = dev or default_device()
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=codes.device)
        for x, name, dtype, dim in ((codes, "codes", torch.int8, 5), (scales, "scales", torch.float32, 4),
                                    (tables, "tables", torch.int32, 2), (lens, "lens", torch.int32, 1),
                                    (refs, "refs", torch.int32, 1), (status, "status", torch.int32, 1)):
            if x.dtype is not dtype or x.dim() != dim or x.get_device() != dev.index or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dim}-d {dtype} tensor on cuda:{dev.index}")
        layers, pages, two, heads, block = codes.shape
        if two != 2 or block not in tuple(PAGE_TOKENS * d for d in HEAD_DIMS):
            raise ValueError("codes must be [layers, pages, 2, kv_heads, 64 * head_dim], head_dim 64, 128 or 256")
        if tuple(scales.shape) != (layers, pages, 2, heads):
            raise ValueError("scales must be [layers, pages, 2, kv_heads]")
        if refs.shape[0] != pages or lens.shape[0] != tables.shape[0] or status.shape[0] != 1:
            raise ValueError("refs must be [pages], lens [max_seqs] with tables [max_seqs, max_pages], status [1]")
        self.codes, self.scales, self.tables, self.lens, self.refs, self.status = codes, scales, tables, lens, refs, status
        self.layers, self.pages, self.kv_heads, self.head_dim = layers, pages, heads, block // PAGE_TOKENS
        self._c = KvCacheC(codes.data_ptr(), scales.data_ptr(), tables.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                           status.data_ptr(), layers, pages, heads, self.head_dim, tables.shape[0], tables.shape[1])
        self._p = C.addressof(self._c)
        self._args = bytearray(_ATTN.size)
        self._args_p = C.addressof((C.c_char * _ATTN.size).from_buffer(self._args))
        self._scale = 1.0 / math.sqrt(self.head_dim)

    @staticmethod
    def create(layers: int, pages: int, kv_heads: int, head_dim: int, max_seqs: int, max_pages: int,
               dev: Optional[Device] = None) -> "KvCache":
        """An empty cache in new tensors."""
        torch = _torch()
        dev = dev or default_device()
        if head_dim not in HEAD_DIMS:
            raise ValueError("head_dim must be 64, 128 or 256")
        if min(layers, pages, kv_heads, max_seqs, max_pages) < 1:
            raise ValueError("layers, pages, kv_heads, max_seqs and max_pages must be at least 1")
        cuda = torch.device("cuda", dev.index)
        return KvCache(torch.zeros(layers, pages, 2, kv_heads, PAGE_TOKENS * head_dim, dtype=torch.int8, device=cuda),
                       torch.zeros(layers, pages, 2, kv_heads, device=cuda),
                       torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=cuda),
                       torch.zeros(max_seqs, dtype=torch.int32, device=cuda),
                       torch.zeros(pages, dtype=torch.int32, device=cuda), dev=dev)

    # -- pages --

    def reserve(self, seqs, tokens) -> None:
        """Make room for tokens[i] more tokens of sequence seqs[i]; their lengths grow (mrl_kv_reserve)."""
        dev = self.dev
        _index(seqs, "seqs", dev)
        _index(tokens, "tokens", dev, seqs.shape[0])
        _call(dev, dev.lib.mrl_kv_reserve, self._p, seqs.data_ptr(), tokens.data_ptr(), seqs.shape[0])

    def fork(self, parents, children) -> None:
        """children[i] (empty) becomes a copy of parents[i] that shares its full pages (mrl_kv_fork)."""
        dev = self.dev
        _index(parents, "parents", dev)
        _index(children, "children", dev, parents.shape[0])
        _call(dev, dev.lib.mrl_kv_fork, self._p, parents.data_ptr(), children.data_ptr(), parents.shape[0])

    def release(self, seqs) -> None:
        """Drop the sequences and give their pages back (mrl_kv_release)."""
        dev = self.dev
        _index(seqs, "seqs", dev)
        _call(dev, dev.lib.mrl_kv_release, self._p, seqs.data_ptr(), seqs.shape[0])

    def trim(self, seqs, window: int, sinks: int = 0) -> None:
        """Give back the pages that no later query sees through the window and the sinks (mrl_kv_trim)."""
        dev = self.dev
        _index(seqs, "seqs", dev)
        _call(dev, dev.lib.mrl_kv_trim, self._p, seqs.data_ptr(), seqs.shape[0], _count(window, "window"), _count(sinks, "sinks"))

    def compact(self) -> None:
        """Move the held pages to the front of the pool (mrl_kv_compact)."""
        dev = self.dev
        _call(dev, dev.lib.mrl_kv_compact, self._p)

    def copy_pages(self, src, dst) -> None:
        """Copy the contents of page src[i] to page dst[i], all layers (mrl_kv_copy_pages)."""
        dev = self.dev
        _index(src, "src", dev)
        _index(dst, "dst", dev, src.shape[0])
        _call(dev, dev.lib.mrl_kv_copy_pages, self._p, src.data_ptr(), dst.data_ptr(), src.shape[0])

    # -- tokens --

    def _cu(self, cu, n_seqs: int, tokens: int):
        if cu is None:
            if tokens != n_seqs:
                raise ValueError(f"without cu there is one row per sequence: {tokens} rows for {n_seqs} sequences")
            return None
        return _index(cu, "cu", self.dev, n_seqs + 1).data_ptr()

    def append(self, layer: int, k, v, seqs, cu=None) -> None:
        """Quantise k and v, [tokens, kv_heads, head_dim] float16 or bfloat16, as the last rows of the
        sequences: cu[b] .. cu[b+1] - 1 are those of seqs[b]; without cu, one row each (mrl_kv_append)."""
        dev = self.dev
        k_row, k_head = _rows(k, "k", dev, self.kv_heads, self.head_dim)
        v_row, v_head = _rows(v, "v", dev, self.kv_heads, self.head_dim, k.dtype, k.shape[0])
        _index(seqs, "seqs", dev)
        n, t = seqs.shape[0], k.shape[0]
        cu_ptr = self._cu(cu, n, t)
        _call(dev, dev.lib.mrl_kv_append, self._p, layer, _dtype_codes[k.dtype], k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, seqs.data_ptr(), cu_ptr, n, t)

    def read(self, layer: int, seqs, cu=None, tokens: Optional[int] = None, dtype=None):
        """(k, v), [tokens, kv_heads, head_dim]: the values held for the same rows as append's
        (mrl_kv_read), tokens in all where cu is given. dtype float32 (default), float16 or bfloat16."""
        torch, dev = _torch_module, self.dev
        _index(seqs, "seqs", dev)
        n = seqs.shape[0]
        if cu is not None and tokens is None:
            raise ValueError("with cu, tokens says how many rows there are: cu[-1], which is on the device")
        t = n if tokens is None else _count(tokens, "tokens")
        cu_ptr = self._cu(cu, n, t)  # cu itself stays referenced: what is allocated below must not take its memory
        dtype = dtype or torch.float32
        if dtype not in _dtype_codes:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        kv = seqs.new_empty((2, t, self.kv_heads, self.head_dim), dtype=dtype)
        k, v = kv[0], kv[1]
        _call(dev, dev.lib.mrl_kv_read, self._p, layer, _dtype_codes[dtype], k.data_ptr(), v.data_ptr(), seqs.data_ptr(), cu_ptr, n, t)
        return k, v

    def attend(self, layer: int, q, seqs, cu=None, max_q: int = 1, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None, out=None, return_lse: bool = False):
        """Causal attention of q, [tokens, q_heads, head_dim], the last rows of the sequences, over the
        cache (mrl_kv_attend): without cu one row per sequence, else rows cu[b] .. cu[b+1] - 1 of seqs[b],
        at most max_q each. window 0: every earlier key is visible. Returns out, or (out, lse [tokens,
        q_heads] float32)."""
        dev = self.dev
        q_row, q_head = _rows(q, "q", dev, None, self.head_dim)
        _index(seqs, "seqs", dev)
        n, (t, heads, _) = seqs.shape[0], q.shape
        cu_ptr = self._cu(cu, n, t)  # cu itself stays referenced: what is allocated below must not take its memory
        out, o_row, o_head = _out(out, q, dev)
        lse = q.new_empty((t, heads), dtype=_torch_module.float32) if return_lse else None
        _ATTN.pack_into(self._args, 0, q.data_ptr(), 0, 0, out.data_ptr(), lse.data_ptr() if return_lse else 0,
                        seqs.data_ptr(), cu_ptr or 0, 0, q_row, q_head, 0, 0, 0, 0, o_row, o_head, n, t, _count(max_q, "max_q"), heads,
                        self.kv_heads, self.head_dim, _dtype_codes[q.dtype], 1, _count(window, "window"),
                        _count(sinks, "sinks"), self._scale if scale is None else scale, _count(layer, "layer"))
        _call(dev, dev.lib.mrl_kv_attend, self._p, self._args_p)
        return (out, lse) if return_lse else out


def _call_buffer(dev: Device, like):
    """What a device's calls without a cache keep: the argument struct, its address, and the status
    word (Device.attention_status: KV_TIMEOUT and KV_BAD_INDEX bits)."""
    dev.attention_status = _torch_module.zeros(1, dtype=_torch_module.int32, device=like.device)
    buf = bytearray(_ATTN.size)
    dev.attention_call = (buf, C.addressof((C.c_char * _ATTN.size).from_buffer(buf)), dev.attention_status)
    return dev.attention_call


def _count(x, name: str) -> int:
    if type(x) is not int:
        x = int(x)
    if not 0 <= x < 2147483648:
        raise ValueError(f"{name} must be in [0, 2^31)")
    return x


def _out(out, q, dev: Device):
    if out is None:
        out = q.new_empty(q.shape)
        return out, q.shape[1] * q.shape[2], q.shape[2]
    return (out, *_rows(out, "out", dev, q.shape[1], q.shape[2], q.dtype, q.shape[0]))


def window_attention(q, k, v, cu, max_len: int, causal: bool = True, window: int = 0, sinks: int = 0,
                     scale: Optional[float] = None, out=None, return_lse: bool = False, dev: Optional[Device] = None):
    """Self-attention over ragged packed sequences (mrl_window_attention): q [tokens, q_heads, head_dim],
    k and v [tokens, kv_heads, head_dim], float16 or bfloat16; sequence b is rows cu[b] .. cu[b+1] - 1 (cu
    int32), at most max_len of them. A query at position p sees key j where j <= p (causal) and, with
    window > 0, |p - j| < window or j < sinks. Returns out, or (out, lse [tokens, q_heads] float32).
    dev.attention_status, an int32 CUDA tensor from the first call on, gets
    KV_BAD_INDEX if cu decreases (nothing is computed then) and KV_TIMEOUT if a kernel gave up."""
    torch = _torch()
    dev = dev or default_device()
    q_row, q_head = _rows(q, "q", dev)
    t, heads, d = q.shape
    k_row, k_head = _rows(k, "k", dev, None, d, q.dtype, t)
    v_row, v_head = _rows(v, "v", dev, k.shape[1], d, q.dtype, t)
    _index(cu, "cu", dev)
    if cu.shape[0] < 1:
        raise ValueError("cu must have one entry more than there are sequences")
    out, o_row, o_head = _out(out, q, dev)
    lse = q.new_empty((t, heads), dtype=torch.float32) if return_lse else None
    buf, ptr, status = dev.attention_call or _call_buffer(dev, q)
    _ATTN.pack_into(buf, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, 0,
                    cu.data_ptr(), status.data_ptr(), q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head,
                    cu.shape[0] - 1, t, _count(max_len, "max_len"), heads, k.shape[1], d, _dtype_codes[q.dtype], 1 if causal else 0,
                    _count(window, "window"), _count(sinks, "sinks"), 1.0 / math.sqrt(d) if scale is None else scale, 0)
    _call(dev, dev.lib.mrl_window_attention, ptr)
    return (out, lse) if return_lse else out
