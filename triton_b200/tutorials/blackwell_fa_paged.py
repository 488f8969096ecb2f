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
  synchronises, so every call can be captured into a CUDA graph and replayed with other lengths. Page tables of up to 2^30
  tokens a sequence (prompts: 2^25 keys) are read. A length beyond the page table is cut to it;
  a page outside the pool is never accessed, it reads as zeros and is not written.
* ``out`` (``q_out``, ``k_out``): where results go; rows outside every sequence are left as they were (in a tensor that the
  call allocates: uninitialised). Outputs of the attention calls must not overlap their inputs.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib

_DT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_HEAD_DIMS = (64, 128, 256)
_append_args, _decode_args, _varlen_args = map(_lib.packed, (_lib.KvAppendArgs, _lib.AttentionDecodeArgs, _lib.AttentionVarlenArgs))


# The checks below run on every call of a decode step, whose kernels take a few microseconds: each tensor's shape and strides
# are read once, and what is rare (copies, dimensions of size one) has a function of its own.
def _check_q(q, what):
    """Device index, tokens, heads and head_dim of the query rows."""
    if not q.is_cuda:
        raise RuntimeError(f"triton_b200 {what} needs CUDA tensors (there is no CPU path)")
    assert q.dim() == 3, f"{what}: rows are [tokens, heads, head_dim]"
    if q.dtype not in _DT:
        raise NotImplementedError(f"{what}: dtype {q.dtype} (bfloat16 and float16 are implemented)")
    n, h, d = q.shape
    if d not in _HEAD_DIMS:
        raise NotImplementedError(f"{what}: head_dim {d} (64, 128 and 256 are implemented)")
    return q.get_device(), n, h, d


def _refuse_grad(what):
    if torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad(), or train with attention()")


def _packed_strides(t):
    """Strides of rows or of a pool whose dimensions of size one have the stride they would have if packed."""
    shape, strides = t.shape, list(t.stride())
    size = 1
    for i in range(t.dim() - 1, -1, -1):
        if shape[i] == 1:
            strides[i] = size
        size = max(size, strides[i] * shape[i])
    return strides


def _in_rows(t):
    """(rows, token stride, head stride): t itself where the kernels can address it, else a packed copy."""
    n, h, d = t.shape
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) & 7 or st < d or sh < d or t.data_ptr() & 15:
        st, sh, sd = _packed_strides(t)
        if sd != 1 or (st | sh) & 7 or st < d or sh < d or t.data_ptr() & 15:
            return t.clone(memory_format=torch.contiguous_format), h * d, d
    return t, st, sh


def _out_rows(out, like, name):
    """(rows, token stride, head stride) of a result shaped like `like`."""
    if out is None:
        _, h, d = like.shape
        return torch.empty_like(like, memory_format=torch.contiguous_format), h * d, d
    assert out.shape == like.shape and out.dtype == like.dtype and out.device == like.device, \
        f"{name} has the shape, dtype and device of its input"
    rows, st, sh = _in_rows(out)
    assert rows is out, f"{name}: contiguous head_dim, strides that are multiples of 8 elements, 16-byte aligned"
    return out, st, sh


def _index(t, idx, name, n=None):
    """A vector of int32 on the device of the data (n: its length)."""
    assert t.dtype == torch.int32 and t.dim() == 1 and (n is None or t.shape[0] == n), f"{name}: int32, one dimension, {n} entries"
    assert t.get_device() == idx, f"{name} is on {t.device}, the data on cuda:{idx}"
    return t if t.is_contiguous() else t.contiguous()


def _pool_strides(t, d, step, name):
    """Page, token and head stride of a ``[pages, page_size, kv_heads, d]`` pool (`step`: elements in 16 bytes)."""
    a, b, c, e = t.stride()
    if e != 1 or (a | b | c) & (step - 1) or a < d or b < d or c < d or t.data_ptr() & 15:
        a, b, c, e = _packed_strides(t)
        assert e == 1 and not (a | b | c) & (step - 1) and min(a, b, c) >= d and not t.data_ptr() & 15, \
            f"{name}: contiguous head_dim, strides that are multiples of 16 bytes, 16-byte aligned"
    return a, b, c


def _check_cache(k_cache, v_cache, page_table, seq_lens, k_scale, v_scale, idx, heads, d, dtype, what):
    """The cache as the kernels take it: sizes, strides, index tensors, scales and their counts."""
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype, "caches: two equal pools"
    assert k_cache.get_device() == idx and v_cache.get_device() == idx, f"{what}: the caches are not on the device of the rows"
    n_pages, page_size, kv_heads, dim = k_cache.shape
    cache_dtype = k_cache.dtype
    fp8 = cache_dtype == torch.float8_e4m3fn
    if not fp8 and cache_dtype != dtype:
        raise NotImplementedError(f"{what}: a {cache_dtype} cache with {dtype} rows")
    assert dim == d and page_size > 0 and kv_heads > 0 and heads % kv_heads == 0
    kst = _pool_strides(k_cache, d, 16 if fp8 else 8, "k_cache")
    vst = _pool_strides(v_cache, d, 16 if fp8 else 8, "v_cache")
    assert page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.get_device() == idx, \
        "page_table: int32 [batch, max_pages] on the device of the rows"
    batch, max_pages = page_table.shape
    table_stride, one = page_table.stride()
    if one != 1 and max_pages > 1:
        page_table = page_table.contiguous()
        table_stride = max_pages
    seq_lens = _index(seq_lens, idx, "seq_lens", batch)
    kn = vn = 0
    if fp8:
        assert k_scale is not None and v_scale is not None, "a float8_e4m3fn cache needs k_scale and v_scale"
        kn, vn = k_scale.numel(), v_scale.numel()
        for t, n in ((k_scale, kn), (v_scale, vn)):
            assert t.dtype == torch.float32 and (n == 1 or n == kv_heads) and t.get_device() == idx, \
                "scales: float32, one element or one per kv head"
        k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
    else:
        assert k_scale is None and v_scale is None, "scales belong to a float8_e4m3fn cache"
    return (n_pages, page_size, kv_heads, kst, vst, page_table, batch, max_pages, table_stride, seq_lens, k_scale, v_scale, kn, vn,
            _lib.E4M3 if fp8 else _DT[dtype])


def _aligned(t):
    """A table as the kernels read it, 16 bytes at a time."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _call(name, args, idx, rows=None):
    """Launches on the current stream of the data's device; `rows`: any tensor there, to allocate the call's workspace from."""
    if torch._C._cuda_getDevice() != idx:
        with torch.cuda.device(idx):
            return _call(name, args, idx, rows)
    lib, ref = _lib.lib(), ctypes.byref(args)
    if rows is not None:
        need = getattr(lib, name[0])(ref)
        ws = rows.new_empty(need // 2 + 1)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    rc = getattr(lib, name[-1])(ref, torch._C._cuda_getCurrentRawStream(idx))
    if rc:
        _lib.check(rc, name[-1])


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
    idx, tokens, heads, d = _check_q(rows, what)
    if k.requires_grad or v.requires_grad or rows.requires_grad:
        _refuse_grad(what)
    dtype = rows.dtype
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == dtype and k.get_device() == v.get_device() == idx
    n, kv, dk = k.shape
    assert n == tokens and dk == d
    (n_pages, page_size, kv_heads, kst, vst, page_table, batch, max_pages, table_stride, seq_lens, k_scale, v_scale, kn, vn,
     cache_dt) = _check_cache(k_cache, v_cache, page_table, seq_lens, k_scale, v_scale, idx, heads, d, dtype, what)
    assert kv == kv_heads, "k and v have the heads of the cache"
    if cu_seqlens is None:
        assert tokens == batch, "without cu_seqlens there is one row per sequence"
    else:
        cu_seqlens = _index(cu_seqlens, idx, "cu_seqlens", batch + 1)
    assert (cos is None) == (sin is None)
    positions = half = 0
    if cos is not None:
        assert cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32
        assert cos.get_device() == sin.get_device() == idx
        cos, sin = _aligned(cos), _aligned(sin)
        positions, half = cos.shape
        assert 0 < 2 * half <= d and half % 8 == 0, "rotary_dim: a multiple of 16, at most head_dim"
    assert q is not None or q_out is None, "q_out without q"
    qo, qos, qoh = (None, 0, 0) if q is None else _out_rows(q_out, q, "q_out")
    ko, kos, koh = (None, 0, 0) if k_out is None else _out_rows(k_out, k, "k_out")
    q, qs, qh = (None, 0, 0) if q is None else _in_rows(q)
    k, ks, kh = _in_rows(k)
    v, vs, vh = _in_rows(v)
    args = _append_args(
        _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(qo), _ptr(ko), k_cache.data_ptr(), v_cache.data_ptr(),
        page_table.data_ptr(), seq_lens.data_ptr(), _ptr(cu_seqlens), _ptr(cos), _ptr(sin), _ptr(k_scale), _ptr(v_scale),
        tokens, batch, 0 if q is None else heads, kv_heads, qs, qh, ks, kh, vs, vh, qos, qoh, kos, koh, *kst, *vst,
        table_stride, half, n_pages, max_pages, positions, page_size, d, 2 * half, 1 if interleaved else 0, _DT[dtype], cache_dt,
        kn, vn)
    _call(("tb200_kv_append", ), args, idx)
    return qo


def _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, with_lse):
    what = "attention_decode"
    idx, n, heads, d = _check_q(q, what)
    if q.requires_grad:
        _refuse_grad(what)
    dtype = q.dtype
    (n_pages, page_size, kv_heads, kst, vst, page_table, batch, max_pages, table_stride, seq_lens, k_scale, v_scale, kn, vn,
     cache_dt) = _check_cache(k_cache, v_cache, page_table, seq_lens, k_scale, v_scale, idx, heads, d, dtype, what)
    assert n == batch, "one query row per sequence"
    o, os, oh = _out_rows(out, q, "out")
    q, qs, qh = _in_rows(q)
    lse = torch.empty((batch, heads), dtype=torch.float32, device=q.device) if with_lse else None
    args = _decode_args(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), _ptr(lse), page_table.data_ptr(),
        seq_lens.data_ptr(), _ptr(k_scale), _ptr(v_scale), 0, 0, batch, heads, kv_heads, qs, qh, os, oh, *kst, *vst,
        table_stride, n_pages, max_pages, page_size, d, _DT[dtype], cache_dt, kn, vn, float(sm_scale), 0)
    _call(("tb200_attention_decode_workspace_bytes", "tb200_attention_decode"), args, idx, q)
    return o, lse


def attention_decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale=None, v_scale=None, out=None):
    """``o[b] = softmax(sm_scale q[b] K_b^T) V_b`` over the ``seq_lens[b]`` cached positions of sequence b, one query token
    ``q[b]`` (``[heads, d]``) each. A sequence of length 0 gives zeros."""
    return _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, False)[0]


def attention_decode_with_lse(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale=None, v_scale=None, out=None):
    """``attention_decode`` and its base-2 log-sum-exp, float32 ``[batch, heads]`` (-inf where the length is 0)."""
    return _decode(q, k_cache, v_cache, page_table, seq_lens, sm_scale, k_scale, v_scale, out, True)


def _varlen(what, q, k, v, kst, vst, cu_q, cu_k, page_table, seq_lens, tokens_k, table_stride, n_pages, max_pages, page_size,
            kv_heads, sm_scale, causal, out, with_lse):
    idx, tokens, heads, d = q.get_device(), *q.shape
    o, os, oh = _out_rows(out, q, "out")
    q, qs, qh = _in_rows(q)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if with_lse else None
    args = _varlen_args(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), cu_q.data_ptr(), _ptr(cu_k), _ptr(page_table),
        _ptr(seq_lens), 0, 0, tokens, tokens_k, cu_q.shape[0] - 1, heads, kv_heads, qs, qh, os, oh, *kst, *vst,
        table_stride, n_pages, max_pages, page_size, d, _DT[q.dtype], 1 if causal else 0, float(sm_scale), 0)
    _call(("tb200_attention_varlen_workspace_bytes", "tb200_attention_varlen_fwd"), args, idx, q)
    return o, lse


def _varlen_packed(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal, out, with_lse):
    what = "attention_varlen"
    idx, _, heads, d = _check_q(q, what)
    if q.requires_grad or k.requires_grad or v.requires_grad:
        _refuse_grad(what)
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == q.dtype and k.get_device() == v.get_device() == idx
    tokens_k, kv_heads, dk = k.shape
    assert dk == d and kv_heads > 0 and heads % kv_heads == 0
    cu_q = _index(cu_seqlens_q, idx, "cu_seqlens_q")
    assert cu_q.shape[0] >= 1
    cu_k = cu_q if cu_seqlens_k is cu_seqlens_q else _index(cu_seqlens_k, idx, "cu_seqlens_k", cu_q.shape[0])
    k, *kst = _in_rows(k)
    v, *vst = _in_rows(v)
    return _varlen(what, q, k, v, (0, *kst), (0, *vst), cu_q, cu_k, None, None, tokens_k, 0, 0, 0, 0, kv_heads, sm_scale, causal,
                   out, with_lse)


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
    idx, _, heads, d = _check_q(q, what)
    if q.requires_grad:
        _refuse_grad(what)
    if k_cache.dtype == torch.float8_e4m3fn:
        raise NotImplementedError(f"{what}: 8-bit caches are read by attention_decode only")
    n_pages, page_size, kv_heads, kst, vst, page_table, batch, max_pages, table_stride, seq_lens, *_ = _check_cache(
        k_cache, v_cache, page_table, seq_lens, None, None, idx, heads, d, q.dtype, what)
    if page_size % 8:
        raise NotImplementedError(f"{what}: page_size {page_size} (multiples of 8 are implemented)")
    cu_q = _index(cu_seqlens_q, idx, "cu_seqlens_q", batch + 1)
    return _varlen(what, q, k_cache, v_cache, kst, vst, cu_q, None, page_table, seq_lens, 0, table_stride, n_pages, max_pages,
                   page_size, kv_heads, sm_scale, causal, out, with_lse)


def attention_varlen_paged(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out=None):
    """``attention_varlen`` with the keys and values of sequence b in the first ``seq_lens[b]`` positions of its pages (a
    16-bit cache, page_size a multiple of 8): a prompt that continues what is cached, its own keys appended already."""
    return _varlen_over_pages(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out, False)[0]


def attention_varlen_paged_with_lse(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out=None):
    """``attention_varlen_paged`` and its base-2 log-sum-exp, as in ``attention_varlen_with_lse``."""
    return _varlen_over_pages(q, k_cache, v_cache, cu_seqlens_q, page_table, seq_lens, sm_scale, causal, out, True)
