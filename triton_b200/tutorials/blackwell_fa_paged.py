"""Attention for serving: grouped heads, packed sequences of different lengths, and a paged key / value cache.

``append_paged_kv(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_seqlens=None, ...)`` rotates new queries and
keys by their positions and appends keys and values to the cache; ``attention_decode(q, k_cache, v_cache, page_table,
seq_lens, sm_scale)`` is the attention of one new token per sequence over it; ``attention_varlen(q, k, v, cu_seqlens_q,
cu_seqlens_k, sm_scale, causal)`` that of whole packed prompts, ``attention_varlen_paged(q, k_cache, v_cache,
cu_seqlens_q, page_table, seq_lens, sm_scale, causal)`` that of prompts whose beginning is cached. The ``_with_lse``
forms also return the base-2 log-sum-exp of the scaled scores, as ``attention_with_lse`` does.

The reference has no counterpart; the calls continue its ``attention(q, k, v, sm_scale, causal)``
(``third_party/tlx/tutorials/blackwell_fa_ws_pipelined_persistent.py:3491``) where it stops: equal head counts and one
sequence length per batch. They are forward passes: an input that requires grad is refused.

Conventions:

* q, k, v, o are ``[tokens, heads, head_dim]`` (decode: ``[batch, heads, head_dim]``), fp16 or bf16, head_dim 64, 128 or
  256, any strides (rows that the kernels cannot address are copied first). ``heads`` is a multiple of the kv heads; query
  head h reads kv head ``h // (heads // kv_heads)``.
* A cache is two tensors ``[pages, page_size, kv_heads, head_dim]`` of q's dtype, or of ``torch.float8_e4m3fn`` with
  ``k_scale`` / ``v_scale`` (float32, one element or one per kv head; a cached value stands for value * scale). Any strides
  of the first three dimensions that are multiples of 16 bytes: a ``[pages, kv_heads, page_size, head_dim]`` pool is
  passed as its ``transpose(1, 2)``.
* ``page_table`` int32 ``[batch, max_pages]``: position p of sequence b lies in page ``page_table[b, p // page_size]``.
  ``seq_lens`` int32 ``[batch]``: tokens of each sequence in the cache, those of this call included. ``cu_seqlens`` int32
  ``[batch + 1]``: where each sequence's rows begin in the packed tensors. All of them stay on the device: no call
  synchronises, so every call can be captured into a CUDA graph and replayed with other lengths. A length beyond the page
  table is cut to it; a page outside the pool is never accessed, it reads as zeros and is not written.
* ``out`` (``q_out``, ``k_out``): where results go; rows outside every sequence are left as they were (in a tensor that the
  call allocates: uninitialised). Outputs of the attention calls must not overlap their inputs.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib

_DT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_HEAD_DIMS = (64, 128, 256)


def _check_q(q, what):
    if not q.is_cuda:
        raise RuntimeError(f"triton_b200 {what} needs CUDA tensors (there is no CPU path)")
    assert q.dim() == 3, f"{what}: rows are [tokens, heads, head_dim]"
    if q.dtype not in _DT:
        raise NotImplementedError(f"{what}: dtype {q.dtype} (bfloat16 and float16 are implemented)")
    if q.shape[2] not in _HEAD_DIMS:
        raise NotImplementedError(f"{what}: head_dim {q.shape[2]} (64, 128 and 256 are implemented)")


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad(), or train with attention()")


def _strides(t):
    """Token and head stride of ``[tokens, heads, d]`` rows; a dimension of size one has the stride it would have packed."""
    n, h, d = t.shape
    sh = t.stride(1) if h > 1 else d
    return (t.stride(0) if n > 1 else max(sh * h, d)), sh


def _rows_ok(t):
    st, sh = _strides(t)
    return t.stride(2) == 1 and st % 8 == 0 and sh % 8 == 0 and min(st, sh) >= t.shape[2] and t.data_ptr() % 16 == 0


def _in_rows(t):
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _out_rows(out, like, name):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    assert out.shape == like.shape and out.dtype == like.dtype and out.device == like.device, \
        f"{name} has the shape, dtype and device of its input"
    assert _rows_ok(out), f"{name}: contiguous head_dim, strides that are multiples of 8 elements, 16-byte aligned"
    return out


def _index(t, dev, name, n=None):
    """A vector of int32 on the device of the data (n: its length)."""
    assert t.dtype == torch.int32 and t.dim() == 1 and (n is None or t.shape[0] == n), f"{name}: int32, one dimension, {n} entries"
    assert t.device == dev, f"{name} is on {t.device}, the data on {dev}"
    return t.contiguous()


def _pool(t, dtype, dev, name):
    """Page, token and head stride of a ``[pages, page_size, kv_heads, d]`` pool."""
    assert t.dim() == 4 and t.dtype == dtype and t.device == dev, f"{name}: [pages, page_size, kv_heads, head_dim] on {dev}"
    n, s, h, d = t.shape
    st = [t.stride(i) if t.shape[i] > 1 else s * h * d for i in range(3)]
    step = 16 // t.element_size()
    assert t.stride(3) == 1 and all(x % step == 0 and x >= d for x in st) and t.data_ptr() % 16 == 0, \
        f"{name}: contiguous head_dim, strides that are multiples of 16 bytes, 16-byte aligned"
    return st


def _check_cache(q, k_cache, v_cache, page_table, seq_lens, k_scale, v_scale, what):
    dev = q.device
    assert k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype
    n_pages, page_size, kv_heads, d = k_cache.shape
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    if not fp8 and k_cache.dtype != q.dtype:
        raise NotImplementedError(f"{what}: a {k_cache.dtype} cache with {q.dtype} queries")
    assert d == q.shape[2] and page_size > 0 and kv_heads > 0 and q.shape[1] % kv_heads == 0
    kst, vst = _pool(k_cache, k_cache.dtype, dev, "k_cache"), _pool(v_cache, k_cache.dtype, dev, "v_cache")
    assert page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == dev, "page_table: int32 [batch, max_pages]"
    if page_table.stride(1) != 1 and page_table.shape[1] > 1:
        page_table = page_table.contiguous()
    seq_lens = _index(seq_lens, dev, "seq_lens", page_table.shape[0])
    if fp8:
        assert k_scale is not None and v_scale is not None, "a float8_e4m3fn cache needs k_scale and v_scale"
        for s in (k_scale, v_scale):
            assert s.dtype == torch.float32 and s.numel() in (1, kv_heads) and s.device == dev, "scales: float32, one or one per kv head"
        k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
    else:
        assert k_scale is None and v_scale is None, "scales belong to a float8_e4m3fn cache"
    return kst, vst, page_table, seq_lens, k_scale, v_scale


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, args, dev):
    with _lib.device_guard(dev):
        rc = getattr(_lib.lib(), name)(ctypes.byref(args), ctypes.c_void_p(_lib.current_stream_ptr(dev)))
    _lib.check(rc, name)


def append_paged_kv(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_seqlens=None, *, cos=None, sin=None,
                    interleaved=False, k_scale=None, v_scale=None, q_out=None, k_out=None):
    """Rotates new queries and keys by their positions, appends keys and values to the cache, returns the rotated queries.

    k, v: ``[tokens, kv_heads, d]``; q: ``[tokens, heads, d]`` or None (then None is returned). Row t of sequence b (rows
    ``cu_seqlens[b] .. cu_seqlens[b + 1]``; without ``cu_seqlens`` one row per sequence) has position
    ``seq_lens[b] - (cu_seqlens[b + 1] - t)``: ``seq_lens`` counts the new tokens already. ``cos``, ``sin``: float32
    ``[positions, rotary_dim // 2]``, row p for position p; the first rotary_dim columns (a multiple of 16) turn, pairs are
    ``(i, i + rotary_dim // 2)`` or, with ``interleaved``, ``(2 i, 2 i + 1)``; the others are copied. Without them nothing
    turns. The arithmetic is in float32 with one rounding; an e4m3 cache takes value / scale, saturating.

    ``q_out`` may be q itself; ``k_out`` (``[tokens, kv_heads, d]``, may be k itself) also receives the rotated keys, for
    ``attention_varlen``. A row whose position lies outside the page table or the rotation table (a padded batch entry with
    ``seq_lens[b] == 0``) appends nothing and comes back as zeros. Rows past ``cu_seqlens[-1]`` are left alone. Two rows
    that share a slot of the cache race for it.
    """
    what = "append_paged_kv"
    rows = k if q is None else q
    _check_q(rows, what)
    _no_grad(what, q, k, v)
    dev, d = k.device, k.shape[2]
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == rows.dtype and rows.device == v.device == dev
    assert rows.shape[0] == k.shape[0] and rows.shape[2] == d and k_cache.shape[2] == k.shape[1]
    kst, vst, page_table, seq_lens, k_scale, v_scale = _check_cache(rows, k_cache, v_cache, page_table, seq_lens, k_scale,
                                                                    v_scale, what)
    tokens, batch = k.shape[0], page_table.shape[0]
    if cu_seqlens is None:
        assert tokens == batch, "without cu_seqlens there is one row per sequence"
    else:
        cu_seqlens = _index(cu_seqlens, dev, "cu_seqlens", batch + 1)
    assert (cos is None) == (sin is None)
    positions = rotary = rot_stride = 0
    if cos is not None:
        assert cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32
        assert cos.device == sin.device == dev
        cos, sin = cos.contiguous(), sin.contiguous()
        positions, rotary, rot_stride = cos.shape[0], 2 * cos.shape[1], cos.shape[1]
        assert 0 < rotary <= d and rotary % 16 == 0, "rotary_dim: a multiple of 16, at most head_dim"
    ko = None if k_out is None else _out_rows(k_out, k, "k_out")
    qo = None if q is None else _out_rows(q_out, q, "q_out")
    q = None if q is None else _in_rows(q)
    k, v = _in_rows(k), _in_rows(v)
    args = _lib.KvAppendArgs(
        _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(qo), _ptr(ko), k_cache.data_ptr(), v_cache.data_ptr(),
        page_table.data_ptr(), seq_lens.data_ptr(), _ptr(cu_seqlens), _ptr(cos), _ptr(sin), _ptr(k_scale), _ptr(v_scale),
        tokens, batch, 0 if q is None else q.shape[1], k.shape[1],
        *(_strides(q) if q is not None else (0, 0)), *_strides(k), *_strides(v),
        *(_strides(qo) if q is not None else (0, 0)), *(_strides(ko) if ko is not None else (0, 0)), *kst, *vst,
        page_table.stride(0), rot_stride, k_cache.shape[0], page_table.shape[1], positions,
        k_cache.shape[1], d, rotary, 1 if interleaved else 0, _DT[k.dtype],
        _lib.E4M3 if k_scale is not None else _DT[k.dtype],
        0 if k_scale is None else k_scale.numel(), 0 if v_scale is None else v_scale.numel())
    _call("tb200_kv_append", args, dev)
    return qo


def _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, with_lse):
    what = "attention_decode"
    _check_q(q, what)
    _no_grad(what, q)
    dev = q.device
    kst, vst, page_table, seq_lens, k_scale, v_scale = _check_cache(q, k_cache, v_cache, page_table, seq_lens, k_scale,
                                                                    v_scale, what)
    batch, heads, d = q.shape
    assert page_table.shape[0] == batch, "one query row per sequence"
    o = _out_rows(out, q, "out")
    q = _in_rows(q)
    lse = torch.empty((batch, heads), dtype=torch.float32, device=dev) if with_lse else None
    args = _lib.AttentionDecodeArgs(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), _ptr(lse), page_table.data_ptr(),
        seq_lens.data_ptr(), _ptr(k_scale), _ptr(v_scale), None, 0, batch, heads, k_cache.shape[2],
        *_strides(q), *_strides(o), *kst, *vst, page_table.stride(0), k_cache.shape[0], page_table.shape[1],
        k_cache.shape[1], d, _DT[q.dtype], _lib.E4M3 if k_scale is not None else _DT[q.dtype],
        0 if k_scale is None else k_scale.numel(), 0 if v_scale is None else v_scale.numel(), float(sm_scale))
    need = _lib.lib().tb200_attention_decode_workspace_bytes(ctypes.byref(args))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _call("tb200_attention_decode", args, dev)
    return o, lse


def attention_decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale=None, v_scale=None, out=None):
    """``o[b] = softmax(sm_scale q[b] K_b^T) V_b`` over the ``seq_lens[b]`` cached positions of sequence b, one query token
    ``q[b]`` (``[heads, d]``) each. A sequence of length 0 gives zeros."""
    return _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, False)[0]


def attention_decode_with_lse(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale=None, v_scale=None, out=None):
    """``attention_decode`` and its base-2 log-sum-exp, float32 ``[batch, heads]`` (-inf where the length is 0)."""
    return _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, True)


def _varlen(what, q, k, v, kst, vst, cu_q, cu_k, page_table, seq_lens, n_pages, page_size, kv_heads, sm_scale, causal, out,
            with_lse):
    dev = q.device
    tokens, heads, d = q.shape
    o = _out_rows(out, q, "out")
    q = _in_rows(q)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if with_lse else None
    args = _lib.AttentionVarlenArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), cu_q.data_ptr(), _ptr(cu_k), _ptr(page_table),
        _ptr(seq_lens), None, 0, tokens, 0 if page_size else k.shape[0], cu_q.shape[0] - 1, heads, kv_heads,
        *_strides(q), *_strides(o), *kst, *vst, page_table.stride(0) if page_size else 0, n_pages,
        page_table.shape[1] if page_size else 0, page_size, d, _DT[q.dtype], 1 if causal else 0, float(sm_scale))
    need = _lib.lib().tb200_attention_varlen_workspace_bytes(ctypes.byref(args))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _call("tb200_attention_varlen_fwd", args, dev)
    return o, lse


def _varlen_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out, with_lse):
    what = "attention_varlen"
    _check_q(q, what)
    _no_grad(what, q, k, v)
    dev = q.device
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == q.dtype and k.device == v.device == dev
    assert k.shape[2] == q.shape[2] and k.shape[1] > 0 and q.shape[1] % k.shape[1] == 0
    cu_q = _index(cu_seqlens_q, dev, "cu_seqlens_q")
    assert cu_q.shape[0] >= 1
    cu_k = cu_q if cu_seqlens_k is cu_seqlens_q else _index(cu_seqlens_k, dev, "cu_seqlens_k", cu_q.shape[0])
    k, v = _in_rows(k), _in_rows(v)
    return _varlen(what, q, k, v, (0, *_strides(k)), (0, *_strides(v)), cu_q, cu_k, None, None, 0, 0, k.shape[1], sm_scale,
                   causal, out, with_lse)


def attention_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out=None):
    """Attention of packed sequences: queries ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]`` over keys
    ``cu_seqlens_k[b] .. cu_seqlens_k[b + 1]``. Causal: the last query of a sequence sees all of its keys, each earlier one
    a key less; a query that sees none gives zeros. No sequence's rows depend on another's, whatever those hold."""
    return _varlen_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out, False)[0]


def attention_varlen_with_lse(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out=None):
    """``attention_varlen`` and its base-2 log-sum-exp, float32 ``[tokens, heads]`` (-inf for a row that sees no key)."""
    return _varlen_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out, True)


def _varlen_over_pages(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out, with_lse):
    what = "attention_varlen_paged"
    _check_q(q, what)
    _no_grad(what, q)
    if k_cache.dtype == torch.float8_e4m3fn:
        raise NotImplementedError(f"{what}: 8-bit caches are read by attention_decode only")
    if k_cache.shape[1] % 8:
        raise NotImplementedError(f"{what}: page_size {k_cache.shape[1]} (multiples of 8 are implemented)")
    kst, vst, page_table, seq_lens, _, _ = _check_cache(q, k_cache, v_cache, page_table, seq_lens, None, None, what)
    cu_q = _index(cu_seqlens_q, q.device, "cu_seqlens_q", page_table.shape[0] + 1)
    return _varlen(what, q, k_cache, v_cache, kst, vst, cu_q, None, page_table, seq_lens, k_cache.shape[0], k_cache.shape[1],
                   k_cache.shape[2], sm_scale, causal, out, with_lse)


def attention_varlen_paged(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out=None):
    """``attention_varlen`` with the keys and values of sequence b in the first ``seq_lens[b]`` positions of its pages (a
    16-bit cache, page_size a multiple of 8): a prompt that continues what is cached, its own keys appended already."""
    return _varlen_over_pages(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out, False)[0]


def attention_varlen_paged_with_lse(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out=None):
    """``attention_varlen_paged`` and its base-2 log-sum-exp, as in ``attention_varlen_with_lse``."""
    return _varlen_over_pages(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out, True)
