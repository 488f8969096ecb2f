"""The paged-cache operators against their definition in 64 bits (oracle/paged.py).

Tolerances are bounds on rounding errors, u = eps / 2 of a type. Attention: the probabilities are rounded once to the type
of the product P V (that of the cache; float16 over an 8-bit cache) and the result once to the output type, so an element
is off by at most u_p sum_j p_j |v_j| + u_o |o| plus what 32-bit scores and exponentials add, which stays below
2^-13 sum_j p_j |v_j| at these sizes (scores below 2^4, products of 256 terms: 2^4 * 2^-24 * 256 = 2^-12 at the very worst
order of summation, 2^-16 typically). float16 probabilities below 2^-14 are subnormal: each is off by up to 2^-25 of the
largest, together keys * 2^-25 * max |v|. Rotation: 2^-22 (|x| + |y|) for two products and a sum in 32 bits, and one rounding.
"""
import ctypes
import math

import pytest
import torch

from oracle import paged as ref

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
gpu = pytest.mark.gpu


def fa():
    from triton_b200.tutorials import blackwell_fa_paged
    return blackwell_fa_paged


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_attention(got, want, size, p_dtype, keys, v_max):
    tol = (half_step(p_dtype) + 2**-13) * size + half_step(got.dtype) * (want.abs() + size * 2**-7) + 1e-30
    if p_dtype == F16:
        tol = tol + keys * 2**-25 * v_max
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert (off <= tol).all(), f"off by {float((off / tol.clamp(min=1e-30)).max()):.3f} of the bound"


def check_lse(got, want):
    assert torch.equal(got == -math.inf, want == -math.inf)
    seen = want != -math.inf
    torch.testing.assert_close(got[seen].double(), want[seen], rtol=1e-6, atol=5e-4)


def offsets(counts, dev):
    return torch.tensor([0] + list(counts), device=dev).cumsum(0).to(torch.int32)


class Cache:
    """Two pools whose every slot holds NaN, and a page table of pages in random order (-1 where a sequence has none)."""

    def __init__(self, dev, lens, kv_heads, d, dtype, page, layout="token", spare=2, width=None, seed=3):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.page, self.lens, self.dev = page, list(lens), dev
        n_pages = sum(need) + spare
        shape = (n_pages, page, kv_heads, d) if layout == "token" else (n_pages, kv_heads, page, d)
        self.k, self.v = (torch.full(shape, math.nan, device=dev).to(dtype) for _ in "kv")
        if layout == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(n_pages, generator=g)
        self.table = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n].int()
            at += n
        self.table = self.table.to(dev)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=dev)

    def fill(self, seed=4, std=1.0):
        """Random rows in every position that a sequence has; the others keep their NaN."""
        g = torch.Generator(device=self.dev).manual_seed(seed)
        for i, n in enumerate(self.lens):
            for j in range(-(-n // self.page)):
                rows = min(self.page, n - j * self.page)
                for pool in (self.k, self.v):
                    x = torch.randn(rows, *pool.shape[2:], generator=g, device=self.dev) * std
                    if pool.dtype == E4M3:
                        pool.view(torch.uint8)[int(self.table[i, j]), :rows] = x.clamp(-448, 448).to(E4M3).view(torch.uint8)
                    else:
                        pool[int(self.table[i, j]), :rows] = x.to(pool.dtype)
        return self

    def rows(self, i, k_scale=None, v_scale=None):
        n = self.lens[i]
        return (ref.cached_rows(self.k, self.table[i], self.page, n, k_scale),
                ref.cached_rows(self.v, self.table[i], self.page, n, v_scale))


def tables(positions, rotary, dev):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0**(-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


# ------------------------------------------------------------------------------------------------ append
def check_append(cache, q, k, v, q_out, k_out, positions, seq_of, cos, sin, interleaved, before, k_scale=None, v_scale=None):
    """Every appended row within its bound; every other slot of the cache bit for bit as it was."""
    d = k.shape[2]

    def near(got, x, dtype, scale=None):
        want = ref.rotated(x, positions, cos, sin, interleaved) if scale is not False else x.double()
        size = x.double().abs()
        if cos is not None and scale is not False:
            half = cos.shape[1]
            size = size.clone()
            if interleaved:
                pair = size[..., 0:2 * half:2] + size[..., 1:2 * half:2]
                size[..., 0:2 * half:2] = size[..., 1:2 * half:2] = pair
            else:
                size[..., :2 * half] = (size[..., :half] + size[..., half:2 * half]).repeat(1, 1, 2)
        return want, 2**-22 * size

    if q is not None:
        want, tol = near(q_out, q, q.dtype)
        assert ((q_out.double() - want).abs() <= half_step(q.dtype) * want.abs() + tol + 2**-25).all()
    for pool, x, out, scale, old in ((cache.k, k, k_out, k_scale, before[0]), (cache.v, v, None, v_scale, before[1])):
        want, tol = near(None, x, x.dtype, None if pool is cache.k else False)
        if out is not None:
            assert ((out.double() - want).abs() <= half_step(k.dtype) * want.abs() + tol + 2**-25).all()
        page = cache.table[seq_of, positions // cache.page].long()
        raw = pool.view(torch.uint8) if pool.dtype == E4M3 else pool
        got = raw[page, positions % cache.page].contiguous().view(pool.dtype).float().double()
        if scale is not None:
            s = scale.double().reshape(-1, 1)
            want, tol = (want / s).clamp(-448, 448), tol / s
            assert ((got - want).abs() <= 2**-4 * want.abs() + 2**-10 + tol * 1.07).all()
        else:
            assert ((got - want).abs() <= half_step(pool.dtype) * want.abs() + tol + 2**-25).all()
        touched = torch.zeros(pool.shape[:2], dtype=torch.bool, device=pool.device)
        touched[page, positions % cache.page] = True
        same = pool.contiguous().view(torch.uint8) == old.contiguous().view(torch.uint8)
        assert same[~touched].all(), "a slot that belongs to no new token was written"


def append_inputs(dev, tokens, heads, kv_heads, d, dtype, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    return tuple(torch.randn(tokens, h, d, generator=g, device=dev).to(dtype) for h in (heads, kv_heads, kv_heads))


@gpu
@pytest.mark.parametrize("d,rotary,interleaved", [(64, 64, False), (128, 128, False), (128, 64, True), (128, 128, True),
                                                  (256, 256, False), (256, 16, False), (64, 48, False), (128, 0, False)])
@pytest.mark.parametrize("dtype,cache_dtype,page,layout", [(BF16, BF16, 16, "token"), (F16, F16, 5, "head"), (BF16, E4M3, 64, "head"),
                                                           (F16, E4M3, 1, "token")])
def test_append_prompts(cuda, d, rotary, interleaved, dtype, cache_dtype, page, layout):
    past, new = [3, 0, 40, 7, 0], [17, 1, 0, 30, 64]
    lens = [p + n for p, n in zip(past, new)]
    cache = Cache(cuda, lens, 3, d, cache_dtype, page, layout).fill()
    q, k, v = append_inputs(cuda, sum(new), 9, 3, d, dtype)
    cos, sin = tables(80, rotary, cuda) if rotary else (None, None)
    scales = (torch.tensor([0.01, 0.02, 0.004], device=cuda), torch.tensor([0.008], device=cuda)) if cache_dtype == E4M3 else (None, None)
    before = cache.k.clone(), cache.v.clone()
    k_out = torch.empty_like(k)
    q_out = fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cache.seq_lens, offsets(new, cuda), cos=cos, sin=sin,
                                 interleaved=interleaved, k_scale=scales[0], v_scale=scales[1], k_out=k_out)
    seq_of = torch.cat([torch.full((n, ), i) for i, n in enumerate(new)]).to(cuda)
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(cuda)
    check_append(cache, q, k, v, q_out, k_out, positions, seq_of, cos, sin, interleaved, before, *scales)


@gpu
@pytest.mark.parametrize("batch,heads,kv_heads", [(1, 32, 8), (1, 1, 1), (37, 6, 2), (3, 5, 5)])
def test_append_one_token_each(cuda, batch, heads, kv_heads):
    lens = [1 + (i * 13) % 50 for i in range(batch)]
    cache = Cache(cuda, lens, kv_heads, 128, BF16, 16).fill()
    q, k, v = append_inputs(cuda, batch, heads, kv_heads, 128, BF16)
    cos, sin = tables(64, 128, cuda)
    before = cache.k.clone(), cache.v.clone()
    q_out = fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cache.seq_lens, cos=cos, sin=sin)
    check_append(cache, q, k, v, q_out, None, cache.seq_lens.long() - 1, torch.arange(batch, device=cuda), cos, sin, False, before)


@gpu
def test_append_strided_in_place_and_without_queries(cuda):
    """Queries, keys and values as slices of one projection; rotated in place; the same rows without queries."""
    cache = Cache(cuda, [20, 33], 2, 64, BF16, 8).fill()
    g = torch.Generator(device=cuda).manual_seed(9)
    qkv = torch.randn(12, 8 + 2 + 2, 64, generator=g, device=cuda).to(BF16)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    cos, sin = tables(40, 64, cuda)
    cu = offsets([5, 7], cuda)
    seq_of = torch.tensor([0] * 5 + [1] * 7, device=cuda)
    positions = torch.cat([torch.arange(15, 20), torch.arange(26, 33)]).to(cuda)
    before = cache.k.clone(), cache.v.clone()
    got = fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cache.seq_lens, cu, cos=cos, sin=sin, q_out=q, k_out=k)
    assert got is q
    check_append(cache, q0, k0, v0, q, k, positions, seq_of, cos, sin, False, before)
    first = cache.k.clone(), cache.v.clone()
    odd = torch.empty(12 * 2 * 64 + 1, dtype=BF16, device=cuda)[1:].view(12, 2, 64)  # rows off the 16-byte grid are copied
    odd.copy_(k0)
    cache.k.copy_(before[0]), cache.v.copy_(before[1])
    off = torch.empty(40 * 32 + 1, device=cuda)[1:].view(40, 32)
    off.copy_(cos)  # a table off the grid too
    assert fa().append_paged_kv(None, odd, v0, cache.k, cache.v, cache.table, cache.seq_lens, cu, cos=off, sin=sin) is None
    assert torch.equal(cache.k.view(torch.int16), first[0].view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), first[1].view(torch.int16))


@gpu
def test_append_leaves_what_has_no_place(cuda):
    """A padded entry (length 0), a position past the page table or the rotation table, a page outside the pool, rows
    behind the last sequence: nothing is written to the cache; the first three come back as zeros, the last untouched."""
    cache = Cache(cuda, [8, 8, 8, 8], 1, 64, BF16, 4, width=3).fill()
    cache.table[3, 1] = cache.k.shape[0]                                   # position 7 of sequence 3 has no page
    cache.seq_lens = torch.tensor([0, 13, 12, 8], dtype=torch.int32, device=cuda)
    cache.table[2, 2] = 0
    q, k, v = append_inputs(cuda, 6, 2, 1, 64, BF16)
    cos, sin = tables(11, 64, cuda)                                        # position 11 of sequence 2 is not in it
    before = cache.k.clone(), cache.v.clone()
    q_out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cache.seq_lens, offsets([1] * 4, cuda), cos=cos, sin=sin,
                         q_out=q_out, k_out=k_out)
    assert torch.equal(cache.k.view(torch.int16), before[0].view(torch.int16))
    assert torch.equal(cache.v.view(torch.int16), before[1].view(torch.int16))
    assert (q_out[:3] == 0).all() and (k_out[:3] == 0).all()
    assert (q_out[4:] == 7).all() and (k_out[4:] == 7).all()
    want = ref.rotated(q[3:4], torch.tensor([7], device=cuda), cos, sin, False)  # its query turns all the same
    assert ((q_out[3:4].double() - want).abs() <= 2**-8 * want.abs() + 2**-20).all()


@gpu
def test_append_saturates_and_keeps_nan(cuda):
    cache = Cache(cuda, [1], 1, 64, E4M3, 16)
    one = torch.ones(1, device=cuda)
    k = torch.zeros(1, 1, 64, dtype=BF16, device=cuda)
    k[0, 0, :5] = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan])
    fa().append_paged_kv(None, k, k, cache.k, cache.v, cache.table, cache.seq_lens, k_scale=one, v_scale=one)
    for pool in (cache.k, cache.v):
        got = pool[int(cache.table[0, 0]), 0, 0].float().tolist()
        assert got[:4] == [448.0, -448.0, 448.0, -448.0] and math.isnan(got[4]) and got[5:] == [0.0] * 59


# ------------------------------------------------------------------------------------------------ decode
def check_decode(cache, q, sm_scale, k_scale=None, v_scale=None, q_in=None):
    o, lse = fa().attention_decode_with_lse(q if q_in is None else q_in, cache.k, cache.v, cache.table, cache.seq_lens, sm_scale,
                                            k_scale=k_scale, v_scale=v_scale)
    p_dtype = F16 if cache.k.dtype == E4M3 else cache.k.dtype
    for i, n in enumerate(cache.lens):
        k, v = cache.rows(i, k_scale, v_scale)
        want, row, size = ref.sequence_attention(q[i:i + 1].double(), k, v, sm_scale, False)
        check_attention(o[i:i + 1], want, size, p_dtype, n, float(v.abs().max()) if n else 0.0)
        check_lse(lse[i:i + 1], row)
    return o


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 300, 1000]


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,cache_dtype,page,layout", [(BF16, BF16, 16, "token"), (F16, F16, 5, "head"), (BF16, E4M3, 64, "head"),
                                                           (F16, E4M3, 16, "token"), (BF16, BF16, 1, "token"),
                                                           (BF16, E4M3, 7, "token")])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (24, 2)])
def test_decode(cuda, d, dtype, cache_dtype, page, layout, heads, kv_heads):
    cache = Cache(cuda, LENS, kv_heads, d, cache_dtype, page, layout).fill()
    g = torch.Generator(device=cuda).manual_seed(5)
    q = torch.randn(len(LENS), heads, d, generator=g, device=cuda).to(dtype)
    scales = (torch.rand(kv_heads, device=cuda) + 0.5, torch.rand(1, device=cuda) + 0.5) if cache_dtype == E4M3 else (None, None)
    check_decode(cache, q, 1 / math.sqrt(d), *scales)


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (8, 1), (9, 1), (16, 1), (17, 1), (64, 1), (40, 8), (128, 2)])
@pytest.mark.parametrize("d", [128, 256])
def test_decode_group_sizes(cuda, heads, kv_heads, d):
    cache = Cache(cuda, [200, 3, 0, 77], kv_heads, d, BF16, 32).fill()
    g = torch.Generator(device=cuda).manual_seed(6)
    check_decode(cache, torch.randn(4, heads, d, generator=g, device=cuda).to(BF16), 1 / math.sqrt(d))


@gpu
@pytest.mark.parametrize("cache_dtype", [BF16, E4M3])
@pytest.mark.parametrize("batch,length", [(1, 20001), (3, 9000), (70, 700)])
def test_decode_long_and_many(cuda, batch, length, cache_dtype):
    lens = [max(1, length - 37 * i * i % length) for i in range(batch)]
    cache = Cache(cuda, lens, 2, 128, cache_dtype, 64).fill()
    g = torch.Generator(device=cuda).manual_seed(7)
    q = torch.randn(batch, 8, 128, generator=g, device=cuda).to(BF16)
    s = torch.tensor([0.7, 1.3], device=cuda) if cache_dtype == E4M3 else None
    check_decode(cache, q, 1 / math.sqrt(128), s, s)


@gpu
@pytest.mark.parametrize("batch", [127, 128, 129, 300, 1500])
def test_many_sequences(cuda, batch):
    """More sequences than threads of a block, than 32 and than 1024 probes of a search; some of them empty."""
    g = torch.Generator(device=cuda).manual_seed(22)
    past = [(i * 7) % 40 if i % 5 else 0 for i in range(batch)]
    new = [(i * 3) % 4 for i in range(batch)]
    lens = [p + n for p, n in zip(past, new)]
    cache = Cache(cuda, lens, 1, 64, BF16, 8).fill()
    q, k, v = append_inputs(cuda, sum(new), 2, 1, 64, BF16)
    before = cache.k.clone(), cache.v.clone()
    q_out = fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cache.seq_lens, offsets(new, cuda))
    seq_of = torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).to(cuda)
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(cuda)
    check_append(cache, q, k, v, q_out, None, positions, seq_of, None, None, False, before)
    check_decode(cache, torch.randn(batch, 2, 64, generator=g, device=cuda).to(BF16), 0.125)
    o, lse = fa().attention_varlen_paged_with_lse(q, cache.k, cache.v, offsets(new, cuda), cache.table, cache.seq_lens, 0.125, True)
    at = 0
    for i, n in enumerate(new):
        kk, vv = cache.rows(i)
        want, row, size = ref.sequence_attention(q[at:at + n].double(), kk, vv, 0.125, True)
        check_attention(o[at:at + n], want, size, BF16, lens[i], 1.0)
        check_lse(lse[at:at + n], row)
        at += n


@gpu
def test_decode_scores_that_grow_and_large_scores(cuda):
    """The running maximum moves by far more than the accumulator's headroom, up along one sequence and down along another;
    the largest scores are near 2^9, where a 32-bit score is off by up to 2^9 * 2^-24 * 128 = 2^-8 in the exponent."""
    cache = Cache(cuda, [640, 640], 1, 128, BF16, 16).fill()
    ramp = torch.linspace(0.05, 4.0, 640, device=cuda)[:, None, None]
    g = torch.Generator(device=cuda).manual_seed(8)
    for i, r in enumerate((ramp, ramp.flip(0))):
        x = (torch.randn(640, 1, 128, generator=g, device=cuda).abs() * r).to(BF16)
        cache.k[cache.table[i].long()] = x.view(40, 16, 1, 128)
    q = torch.randn(2, 4, 128, generator=g, device=cuda).abs().to(BF16)
    o, lse = fa().attention_decode_with_lse(q, cache.k, cache.v, cache.table, cache.seq_lens, 1.0)
    for i in range(2):
        k, v = cache.rows(i)
        want, row, size = ref.sequence_attention(q[i:i + 1].double(), k, v, 1.0, False)
        assert ((o[i:i + 1].double() - want).abs() <= (2**-8 + 2**-8) * size + 2**-8 * want.abs() + 1e-6).all()
        torch.testing.assert_close(lse[i:i + 1].double(), row, rtol=1e-5, atol=0)


@gpu
def test_decode_strides_out_and_missing_pages(cuda):
    """Queries as a slice of a projection, an output with rows apart, a page table that is a slice, pages that do not exist
    (read as zeros), a length beyond the page table (cut to it)."""
    cache = Cache(cuda, [40, 64, 9], 2, 128, BF16, 16).fill()
    g = torch.Generator(device=cuda).manual_seed(10)
    qkv = torch.randn(3, 12, 128, generator=g, device=cuda).to(BF16)
    q = qkv[:, 2:10]
    out = torch.full((3, 16, 128), 5.0, dtype=BF16, device=cuda)
    wide = torch.full((3, 9), 12345, dtype=torch.int32, device=cuda)
    wide[:, :4] = cache.table
    cache.table = wide[:, :4]
    cache.table[0, 1], cache.table[1, 3] = -1, cache.k.shape[0]
    got = fa().attention_decode(q, cache.k, cache.v, cache.table, torch.tensor([40, 1000, 9], dtype=torch.int32, device=cuda), 0.1,
                                out=out[:, ::2])
    assert (out[:, 1::2] == 5).all()
    for i in range(3):
        k, v = cache.rows(i)
        want, _, size = ref.sequence_attention(q[i:i + 1].double(), k, v, 0.1, False)
        check_attention(got[i:i + 1], want, size, BF16, 64, 1.0)


@gpu
def test_offsets_past_31_bits(cuda):
    """A pool of more than 2^31 elements whose last pages are the used ones, for every call that reads or writes it."""
    page, kv, d = 64, 8, 128
    n_pages = (1 << 31) // (page * kv * d) + 40
    pool_k, pool_v = (torch.zeros(n_pages, page, kv, d, dtype=BF16, device=cuda) for _ in "kv")
    cache = Cache(cuda, [150, 90], kv, d, BF16, page)
    cache.k, cache.v = pool_k, pool_v
    cache.table = torch.tensor([[n_pages - 1, n_pages - 5, n_pages - 2], [n_pages - 9, n_pages - 30, -1]], dtype=torch.int32, device=cuda)
    cache.fill()
    g = torch.Generator(device=cuda).manual_seed(11)
    q, k, v = (torch.randn(2, h, d, generator=g, device=cuda).to(BF16) for h in (16, kv, kv))
    fa().append_paged_kv(q, k, v, pool_k, pool_v, cache.table, cache.seq_lens)
    for i, n in enumerate(cache.lens):
        assert torch.equal(pool_k[int(cache.table[i, (n - 1) // page]), (n - 1) % page], k[i])
        assert torch.equal(pool_v[int(cache.table[i, (n - 1) // page]), (n - 1) % page], v[i])
    o = check_decode(cache, q, 0.1)
    o2 = fa().attention_varlen_paged(q, pool_k, pool_v, offsets([1, 1], cuda), cache.table, cache.seq_lens, 0.1, True)
    for i in range(2):
        kk, vv = cache.rows(i)
        want, _, size = ref.sequence_attention(q[i:i + 1].double(), kk, vv, 0.1, True)
        check_attention(o2[i:i + 1], want, size, BF16, 150, 1.0)
    assert o.shape == o2.shape


# ------------------------------------------------------------------------------------------------ packed prompts
def check_varlen(q, k, v, q_lens, k_lens, sm_scale, causal, got, lse):
    at_q = at_k = 0
    for n_q, n_k in zip(q_lens, k_lens):
        qq, kk, vv = q[at_q:at_q + n_q].double(), k[at_k:at_k + n_k].double(), v[at_k:at_k + n_k].double()
        want, row, size = ref.sequence_attention(qq, kk, vv, sm_scale, causal)
        check_attention(got[at_q:at_q + n_q], want, size, q.dtype, n_k, float(vv.abs().max()) if n_k else 0.0)
        check_lse(lse[at_q:at_q + n_q], row)
        at_q, at_k = at_q + n_q, at_k + n_k


def varlen_inputs(dev, n_q, n_k, heads, kv_heads, d, dtype, seed=12):
    g = torch.Generator(device=dev).manual_seed(seed)
    return tuple(torch.randn(n, h, d, generator=g, device=dev).to(dtype) for n, h in ((n_q, heads), (n_k, kv_heads), (n_k, kv_heads)))


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, BF16), (128, F16), (256, BF16), (256, F16), (64, F16)])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (6, 1), (5, 1), (16, 1)])
def test_varlen_prompts(cuda, causal, d, dtype, heads, kv_heads):
    lens = [1, 0, 37, 128, 129, 5, 300, 64, 0]
    q, k, v = varlen_inputs(cuda, sum(lens), sum(lens), heads, kv_heads, d, dtype)
    cu = offsets(lens, cuda)
    o, lse = fa().attention_varlen_with_lse(q, k, v, cu, cu, 1 / math.sqrt(d), causal)
    check_varlen(q, k, v, lens, lens, 1 / math.sqrt(d), causal, o, lse)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (3, 1, 64), (4, 2, 256), (64, 1, 128), (128, 1, 64), (256, 1, 64)])
def test_varlen_other_key_counts(cuda, causal, heads, kv_heads, d):
    """More keys than queries, fewer (rows that see nothing), none at all, one of each."""
    q_lens, k_lens = [5, 200, 70, 1, 9, 130], [260, 50, 70, 500, 0, 131]
    q, k, v = varlen_inputs(cuda, sum(q_lens), sum(k_lens), heads, kv_heads, d, BF16)
    o, lse = fa().attention_varlen_with_lse(q, k, v, offsets(q_lens, cuda), offsets(k_lens, cuda), 1 / math.sqrt(d), causal)
    check_varlen(q, k, v, q_lens, k_lens, 1 / math.sqrt(d), causal, o, lse)


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_varlen_neighbours_do_not_matter(cuda, d):
    """NaN and infinities in the sequences before and behind, and in rows outside every sequence, change nothing."""
    lens = [50, 100, 77]
    q, k, v = varlen_inputs(cuda, 260, 260, 4, 1, d, BF16)
    cu = offsets(lens, cuda) + 10
    cu[0] = 10
    clean = fa().attention_varlen(q, k, v, cu, cu, 0.1, True)
    inside = slice(60, 160)
    for bad in (math.nan, math.inf, -math.inf):
        dirty = [torch.full_like(t, bad) for t in (q, k, v)]
        for t, s in zip(dirty, (q, k, v)):
            t[inside] = s[inside]
        out = torch.full_like(q, 3.0)
        fa().attention_varlen(*dirty, cu, cu, 0.1, True, out=out)
        assert torch.equal(out[inside].view(torch.int16), clean[inside].view(torch.int16))
        assert (out[:10] == 3).all() and (out[237:] == 3).all()


@gpu
def test_varlen_longer_prompts_and_strides(cuda):
    """Several tiles per CTA, walks of many blocks; q, k, v as slices of one projection, rows of the output apart."""
    lens = [1500, 3, 700, 2200, 129, 64, 1024]
    total = sum(lens)
    g = torch.Generator(device=cuda).manual_seed(13)
    qkv = torch.randn(total, 16 + 2 + 2, 128, generator=g, device=cuda).to(BF16)
    q, k, v = qkv[:, :16], qkv[:, 16:18], qkv[:, 18:]
    cu = offsets(lens, cuda)
    out = torch.full((total, 32, 128), 2.0, dtype=BF16, device=cuda)
    o, lse = fa().attention_varlen_with_lse(q, k, v, cu, cu, 1 / math.sqrt(128), True, out=out[:, :16])
    assert (out[:, 16:] == 2).all()
    check_varlen(q, k, v, lens, lens, 1 / math.sqrt(128), True, o, lse)


@gpu
def test_varlen_rescales(cuda):
    """Keys that grow along the sequence move the running maximum by more than the accumulator's headroom."""
    lens = [1024, 300]
    q, k, v = varlen_inputs(cuda, sum(lens), sum(lens), 4, 1, 128, BF16)
    k = (k.abs() * torch.cat([torch.linspace(0.05, 3.0, n) for n in lens]).to(cuda)[:, None, None]).to(BF16)
    q = q.abs()
    cu = offsets(lens, cuda)
    o, lse = fa().attention_varlen_with_lse(q, k, v, cu, cu, 1 / math.sqrt(128), True)
    check_varlen(q, k, v, lens, lens, 1 / math.sqrt(128), True, o, lse)


@gpu
def test_varlen_agrees_with_attention(cuda):
    """Equal lengths and heads: the packed call gives what the batched call gives."""
    from triton_b200.tutorials.blackwell_fa_ws_pipelined_persistent import attention_with_lse
    g = torch.Generator(device=cuda).manual_seed(14)
    q, k, v = (torch.randn(3, 4, 500, 128, generator=g, device=cuda).to(BF16) for _ in range(3))
    o1, m1 = attention_with_lse(q, k, v, 0.09, True)
    cu = offsets([500] * 3, cuda)
    o2, m2 = fa().attention_varlen_with_lse(*(t.transpose(1, 2).reshape(1500, 4, 128) for t in (q, k, v)), cu, cu, 0.09, True)
    assert torch.equal(o1.transpose(1, 2).reshape(1500, 4, 128).view(torch.int16), o2.view(torch.int16))
    torch.testing.assert_close(m1.transpose(1, 2).reshape(1500, 4), m2, rtol=0, atol=0)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,layout", [(8, "token"), (16, "token"), (24, "head"), (48, "token"), (64, "head"), (128, "token"), (256, "head")])
@pytest.mark.parametrize("d,dtype,heads,kv_heads", [(128, BF16, 8, 2), (64, F16, 3, 3), (256, BF16, 6, 2)])
def test_varlen_paged(cuda, causal, page, layout, d, dtype, heads, kv_heads):
    new, lens = [1, 0, 150, 33, 260, 7, 4], [1, 100, 150, 400, 300, 1000, 0]
    cache = Cache(cuda, lens, kv_heads, d, dtype, page, layout).fill()
    g = torch.Generator(device=cuda).manual_seed(15)
    q = torch.randn(sum(new), heads, d, generator=g, device=cuda).to(dtype)
    o, lse = fa().attention_varlen_paged_with_lse(q, cache.k, cache.v, offsets(new, cuda), cache.table, cache.seq_lens,
                                                  1 / math.sqrt(d), causal)
    at = 0
    for i, n in enumerate(new):
        k, v = cache.rows(i)
        want, row, size = ref.sequence_attention(q[at:at + n].double(), k, v, 1 / math.sqrt(d), causal)
        check_attention(o[at:at + n], want, size, dtype, lens[i], float(v.abs().max()) if lens[i] else 0.0)
        check_lse(lse[at:at + n], row)
        at += n


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dtype,heads,kv_heads", [(128, BF16, 8, 2), (64, F16, 3, 1), (256, BF16, 4, 2), (128, F16, 12, 1)])
@pytest.mark.parametrize("q_lens,k_lens", [([5], [9000]), ([1, 300, 2], [7000, 300, 1]), ([40, 0, 260], [3000, 4000, 2900]),
                                           ([130] * 3, [2177] * 3), ([700], [700])])
def test_varlen_split_walks(cuda, causal, d, dtype, heads, kv_heads, q_lens, k_lens):
    """Few queries over many keys: walks are cut and joined, packed and over pages; the same bits every time. float16 keys of
    a long sequence: the sum over subnormal probabilities is part of the bound."""
    q, k, v = varlen_inputs(cuda, sum(q_lens), sum(k_lens), heads, kv_heads, d, dtype)
    cu_q, cu_k = offsets(q_lens, cuda), offsets(k_lens, cuda)
    o, lse = fa().attention_varlen_with_lse(q, k, v, cu_q, cu_k, 1 / math.sqrt(d), causal)
    check_varlen(q, k, v, q_lens, k_lens, 1 / math.sqrt(d), causal, o, lse)
    for _ in range(5):
        again = fa().attention_varlen(q, k, v, cu_q, cu_k, 1 / math.sqrt(d), causal)
        assert torch.equal(again.view(torch.int16), o.view(torch.int16))
    cache = Cache(cuda, k_lens, kv_heads, d, dtype, 16)
    fa().append_paged_kv(None, k, v, cache.k, cache.v, cache.table, cache.seq_lens, cu_k)
    paged = fa().attention_varlen_paged(q, cache.k, cache.v, cu_q, cache.table, cache.seq_lens, 1 / math.sqrt(d), causal)
    assert torch.equal(paged.view(torch.int16), o.view(torch.int16))


@gpu
@pytest.mark.parametrize("units", [147, 148, 149, 297])
def test_varlen_as_many_parts_as_there_can_be(cuda, units):
    """Equal walks just longer than an even share: every tile is cut, the parts fill the workspace."""
    q_lens, k_lens = [1] * units, [640 + 128 * (i % 2) for i in range(units)]
    q, k, v = varlen_inputs(cuda, units, sum(k_lens), 1, 1, 64, BF16)
    o, lse = fa().attention_varlen_with_lse(q, k, v, offsets(q_lens, cuda), offsets(k_lens, cuda), 0.125, True)
    check_varlen(q, k, v, q_lens, k_lens, 0.125, True, o, lse)


@gpu
def test_offsets_that_are_no_offsets(cuda):
    """Offsets that run backwards, overlap or leave the tensors are wrong calls that nothing on the host can see: whatever
    comes out, nothing outside the tensors is touched and the next call is right."""
    q, k, v = varlen_inputs(cuda, 300, 300, 4, 2, 64, BF16)
    cache = Cache(cuda, [300] * 3, 2, 64, BF16, 16).fill()
    good = offsets([100, 50, 150], cuda)
    want = fa().attention_varlen(q, k, v, good, good, 0.1, True)
    guard = torch.full((400, 4, 64), 6.0, dtype=BF16, device=cuda)
    for bad in ([0, 200, 100, 300], [0, 300, 0, 300], [-50, 100, 200, 4000], [2**31 - 1, -2**31, 5, 7], [300, 200, 100, 0]):
        cu = torch.tensor(bad, dtype=torch.int32, device=cuda)
        fa().attention_varlen(q, k, v, cu, cu, 0.1, True, out=guard[50:350])
        fa().attention_varlen(q, k, v, good, cu, 0.1, False, out=guard[50:350])
        fa().attention_varlen_paged(q, cache.k, cache.v, cu, cache.table, cu[:3].contiguous(), 0.1, True, out=guard[50:350])
        fa().attention_decode(q[:3], cache.k, cache.v, cache.table, cu[:3].contiguous(), 0.1)
        before = cache.k.clone()
        fa().append_paged_kv(q, k, v, cache.k, cache.v, cache.table, cu[:3].contiguous(), cu, q_out=guard[50:350])
        cache.k.copy_(before)
        assert (guard[:50] == 6).all() and (guard[350:] == 6).all()
    assert torch.equal(fa().attention_varlen(q, k, v, good, good, 0.1, True).view(torch.int16), want.view(torch.int16))


@gpu
def test_pools_of_different_order(cuda):
    """Keys stored token by token, values head by head, and both in one tensor: the strides of the two pools are their own."""
    cache = Cache(cuda, [130, 17, 64], 2, 128, BF16, 16).fill()
    both = torch.full((cache.k.shape[0], 2, 16, 3, 128), math.nan, dtype=BF16, device=cuda)
    both[:, 0, :, :2], both[:, 1, :, 1:] = cache.k, cache.v
    head = cache.v.transpose(1, 2).contiguous().transpose(1, 2)
    g = torch.Generator(device=cuda).manual_seed(20)
    q = torch.randn(3, 8, 128, generator=g, device=cuda).to(BF16)
    cu = offsets([1, 1, 1], cuda)
    want = fa().attention_decode(q, cache.k, cache.v, cache.table, cache.seq_lens, 0.1)
    want2 = fa().attention_varlen_paged(q, cache.k, cache.v, cu, cache.table, cache.seq_lens, 0.1, True)
    for kk, vv in ((cache.k, head), (both[:, 0, :, :2], both[:, 1, :, 1:])):
        got = fa().attention_decode(q, kk, vv, cache.table, cache.seq_lens, 0.1)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
        got = fa().attention_varlen_paged(q, kk, vv, cu, cache.table, cache.seq_lens, 0.1, True)
        assert torch.equal(got.view(torch.int16), want2.view(torch.int16))
        new = torch.randn(3, 2, 128, generator=g, device=cuda).to(BF16)
        fa().append_paged_kv(None, new, -new, kk, vv, cache.table, cache.seq_lens)
        for i, n in enumerate(cache.lens):
            page, at = int(cache.table[i, (n - 1) // 16]), (n - 1) % 16
            assert torch.equal(kk[page, at], new[i]) and torch.equal(vv[page, at], -new[i])
        kk.copy_(cache.k) if kk is not cache.k else kk.copy_(both[:, 0, :, :2])
    assert both[:, 0, :, 2].isnan().all() and both[:, 1, :, 0].isnan().all()


@gpu
def test_decode_same_bits_every_time(cuda):
    for lens, heads, kv in (([9000], 8, 1), ([700] * 70, 8, 2), ([0, 5, 3000, 1], 24, 2)):
        cache = Cache(cuda, lens, kv, 128, BF16, 16).fill()
        g = torch.Generator(device=cuda).manual_seed(21)
        q = torch.randn(len(lens), heads, 128, generator=g, device=cuda).to(BF16)
        want, lse = fa().attention_decode_with_lse(q, cache.k, cache.v, cache.table, cache.seq_lens, 0.1)
        for _ in range(10):
            got, lse2 = fa().attention_decode_with_lse(q, cache.k, cache.v, cache.table, cache.seq_lens, 0.1)
            assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and torch.equal(lse, lse2)


@gpu
def test_varlen_paged_missing_pages(cuda):
    cache = Cache(cuda, [300, 200], 2, 128, BF16, 16).fill()
    cache.table[0, 3], cache.table[0, 18], cache.table[1, 0] = -1, 1 << 30, cache.k.shape[0]
    g = torch.Generator(device=cuda).manual_seed(16)
    q = torch.randn(60, 4, 128, generator=g, device=cuda).to(BF16)
    o = fa().attention_varlen_paged(q, cache.k, cache.v, offsets([50, 10], cuda), cache.table, cache.seq_lens, 0.1, True)
    for i, rows in enumerate((slice(0, 50), slice(50, 60))):
        k, v = cache.rows(i)
        want, _, size = ref.sequence_attention(q[rows].double(), k, v, 0.1, True)
        check_attention(o[rows], want, size, BF16, 300, 1.0)


# ------------------------------------------------------------------------------------------------ together
def serve(cuda, dtype, cache_dtype, graph):
    """Prompts, then further turns, then single tokens with a padded batch, layer by layer as a server runs them; every
    output is held against attention over the whole history in 64 bits (rotated and, in an 8-bit cache, rounded as cached)."""
    f = fa()
    heads, kv, d, page, batch = 8, 2, 128, 16, 4
    cos, sin = tables(600, d, cuda)
    g = torch.Generator(device=cuda).manual_seed(17)
    scales = dict(k_scale=torch.tensor([0.02, 0.03], device=cuda), v_scale=torch.tensor([0.02], device=cuda)) if cache_dtype == E4M3 else {}
    cache = Cache(cuda, [400] * batch, kv, d, cache_dtype, page)
    lens = torch.zeros(batch, dtype=torch.int32, device=cuda)

    def rows(n):
        return tuple(torch.randn(n, h, d, generator=g, device=cuda).to(dtype) for h in (heads, kv, kv))

    def check(o, q, counts, host_lens):
        at = 0
        for i, n in enumerate(counts):
            cache.lens[i] = host_lens[i]
            k, v = cache.rows(i, scales.get("k_scale"), scales.get("v_scale"))
            want, _, size = ref.sequence_attention(q[at:at + n].double(), k, v, 0.1, True)
            check_attention(o[at:at + n], want, size, F16 if cache_dtype == E4M3 else dtype, 400, float(v.abs().max()) if host_lens[i] else 0.0)
            at += n

    # prompts: packed attention over the rotated keys themselves
    new = [70, 1, 0, 200]
    q, k, v = rows(sum(new))
    cu = offsets(new, cuda)
    lens += torch.tensor(new, dtype=torch.int32, device=cuda)
    k_rot = torch.empty_like(k)
    q_rot = f.append_paged_kv(q, k, v, cache.k, cache.v, cache.table, lens, cu, cos=cos, sin=sin, k_out=k_rot, **scales)
    o, lse = f.attention_varlen_with_lse(q_rot, k_rot, v, cu, cu, 0.1, True)
    check_varlen(q_rot, k_rot, v, new, new, 0.1, True, o, lse)
    host = list(new)
    if cache_dtype != E4M3:
        check(f.attention_varlen_paged(q_rot, cache.k, cache.v, cu, cache.table, lens, 0.1, True), q_rot, new, host)
        new = [9, 130, 40, 0]
        q, k, v = rows(sum(new))
        cu = offsets(new, cuda)
        lens += torch.tensor(new, dtype=torch.int32, device=cuda)
        host = [a + b for a, b in zip(host, new)]
        q_rot = f.append_paged_kv(q, k, v, cache.k, cache.v, cache.table, lens, cu, cos=cos, sin=sin, **scales)
        check(f.attention_varlen_paged(q_rot, cache.k, cache.v, cu, cache.table, lens, 0.1, True), q_rot, new, host)
    # single tokens; sequence 1 stops (a padded entry) after two of them
    q, k, v = (t.clone() for t in rows(batch))
    q_rot, o = torch.empty_like(q), torch.empty_like(q)

    def step():
        f.append_paged_kv(q, k, v, cache.k, cache.v, cache.table, lens, cos=cos, sin=sin, q_out=q_rot, **scales)
        f.attention_decode(q_rot, cache.k, cache.v, cache.table, lens, 0.1, out=o, **scales)

    replay = step
    if graph:
        kept = lens.clone()
        lens.zero_()  # nothing is appended while the graph is made
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
        lens.copy_(kept)
        replay = captured.replay
    for i in range(5):
        active = [1, 1 if i < 2 else 0, 1, 1]
        for t, new_t in zip((q, k, v), rows(batch)):
            t.copy_(new_t)
        host = [(a + b if b else 0) for a, b in zip(host, active)]
        lens.copy_(torch.tensor(host, dtype=torch.int32))
        replay()
        check(o, q_rot, [1] * batch, host)


@gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, E4M3)])
def test_serving_steps(cuda, dtype, cache_dtype, graph):
    from triton_b200 import _lib
    serve(cuda, dtype, cache_dtype, graph)
    _lib.sync_check()


@gpu
def test_captured_prompt_with_other_lengths(cuda):
    """One captured packed call serves any lengths that fit its tensors; two graphs and an eager call run at the same time."""
    f = fa()
    q, k, v = varlen_inputs(cuda, 700, 700, 4, 2, 128, BF16)
    cu = offsets([300, 200, 100], cuda)
    graphs, outs = [], []
    f.attention_varlen(q, k, v, cu, cu, 0.1, True)
    for _ in range(2):
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            f.attention_varlen(q, k, v, cu, cu, 0.1, True, out=out)
        graphs.append(graph)
        outs.append(out)
    for lens in ([300, 200, 100], [0, 700, 0], [1, 2, 3], [350, 0, 350]):
        cu.copy_(offsets(lens, cuda))
        want = f.attention_varlen(q, k, v, cu, cu, 0.1, True)
        for out in outs:
            out.fill_(9)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        again = f.attention_varlen(q, k, v, cu, cu, 0.1, True)
        torch.cuda.synchronize()
        n = sum(lens)
        for out in [again] + outs:
            assert torch.equal(out[:n].view(torch.int16), want[:n].view(torch.int16))
        assert all((out[n:] == 9).all() for out in outs)


@gpu
def test_calls_on_two_streams(cuda):
    """Two decode calls on two streams do not share scratch."""
    cache = Cache(cuda, [5000, 3000, 1], 2, 128, BF16, 16).fill()
    g = torch.Generator(device=cuda).manual_seed(18)
    qs = [torch.randn(3, 8, 128, generator=g, device=cuda).to(BF16) for _ in range(2)]
    want = [fa().attention_decode(q, cache.k, cache.v, cache.table, cache.seq_lens, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(fa().attention_decode(q, cache.k, cache.v, cache.table, cache.seq_lens, 0.1))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@gpu
def test_other_device(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    other = torch.device("cuda:1")
    with torch.cuda.device(0):
        cache = Cache(other, [100, 17], 2, 128, BF16, 16).fill()
        g = torch.Generator(device=other).manual_seed(19)
        check_decode(cache, torch.randn(2, 8, 128, generator=g, device=other).to(BF16), 0.1)


@gpu
def test_empty_calls(cuda):
    f = fa()
    cache = Cache(cuda, [], 2, 128, BF16, 16)
    none = torch.empty(0, 8, 128, dtype=BF16, device=cuda)
    kv = torch.empty(0, 2, 128, dtype=BF16, device=cuda)
    table, lens = torch.empty(0, 1, dtype=torch.int32, device=cuda), torch.empty(0, dtype=torch.int32, device=cuda)
    zero = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert f.attention_decode(none, cache.k, cache.v, table, lens, 0.1).shape == none.shape
    assert f.append_paged_kv(none, kv, kv, cache.k, cache.v, table, lens).shape == none.shape
    assert f.attention_varlen(none, kv, kv, zero, zero, 0.1, True).shape == none.shape
    assert f.attention_varlen_paged(none, cache.k, cache.v, zero, table, lens, 0.1, True).shape == none.shape
    # queries without a single key anywhere
    q = torch.ones(3, 8, 128, dtype=BF16, device=cuda)
    o = f.attention_varlen(q, kv, kv, offsets([3], cuda), offsets([0], cuda), 0.1, True)
    assert (o == 0).all()
    no_pages = torch.empty(0, 16, 2, 128, dtype=BF16, device=cuda)
    o = f.attention_decode(q, no_pages, no_pages, torch.empty(3, 0, dtype=torch.int32, device=cuda),
                           torch.tensor([0, 4, 9], dtype=torch.int32, device=cuda), 0.1)
    assert (o == 0).all()


# ------------------------------------------------------------------------------------------------ refusals
def test_cpu_tensors_are_refused():
    f = fa()
    q, kv = torch.zeros(2, 4, 128, dtype=BF16), torch.zeros(2, 2, 128, dtype=BF16)
    pool = torch.zeros(3, 16, 2, 128, dtype=BF16)
    table, lens, cu = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    for call in (lambda: f.append_paged_kv(q, kv, kv, pool, pool, table, lens),
                 lambda: f.attention_decode(q, pool, pool, table, lens, 1.0),
                 lambda: f.attention_varlen(q, kv, kv, cu, cu, 1.0, True),
                 lambda: f.attention_varlen_paged(q, pool, pool, cu, table, lens, 1.0, True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def filled(cls, **kw):
    """Arguments that pass every check but for what `kw` changes (addresses are never read: each call is refused or empty)."""
    a = cls()
    for name, typ in cls._fields_:
        if typ is ctypes.c_void_p:
            setattr(a, name, 4096)
        elif "stride" in name:
            setattr(a, name, 1024)
    for name, value in dict(batch=2, heads=8, kv_heads=2, n_pages=4, max_pages=4, page_size=16, head_dim=128, k_scale_n=1, v_scale_n=1,
                            sm_scale=0.1, tokens=2, tokens_q=2, tokens_k=2, rotary_dim=128, n_positions=64, workspace_bytes=1 << 20).items():
        if any(name == n for n, _ in cls._fields_):
            setattr(a, name, value)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(k=None), -1), (dict(q_out=None), -1), (dict(sin=None), -1), (dict(tokens=-1), -1), (dict(kv_heads=0), -1),
    (dict(page_size=0), -1), (dict(cu_seqlens=None, tokens=3), -1), (dict(head_dim=96), -2), (dict(dtype=2), -2),
    (dict(cache_dtype=1), -2), (dict(cache_dtype=4), -2), (dict(cache_dtype=3, k_scale=None), -1), (dict(cache_dtype=3, k_scale_n=3), -1),
    (dict(rotary_dim=24), -1), (dict(rotary_dim=144), -1), (dict(q=4104), -1), (dict(k_cache=4100), -1), (dict(kc_stride_tok=100), -1),
    (dict(cos=4100), -1), (dict(rot_stride=6), -1), (dict(tokens=1 << 32), -2), (dict(tokens=0), 0)])
def test_append_refusals(lib, change, code):
    from triton_b200 import _lib
    assert lib.tb200_kv_append(ctypes.byref(filled(_lib.KvAppendArgs, **change)), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(seq_lens=None), -1), (dict(heads=7), -1), (dict(kv_heads=0), -1), (dict(page_size=0), -1),
    (dict(head_dim=32), -2), (dict(dtype=3), -2), (dict(cache_dtype=1), -2), (dict(cache_dtype=3, v_scale=None), -1),
    (dict(cache_dtype=3, kc_stride_tok=1032), -1), (dict(sm_scale=0.0), -1), (dict(sm_scale=float("nan")), -1), (dict(o=4098), -1),
    (dict(q_stride_b=1001), -1), (dict(batch=0), 0), (dict(max_pages=1 << 40), -2), (dict(batch=1 << 40), -2),
    (dict(batch=(1 << 30) - (1 << 21), max_pages=1, heads=2), -2), (dict(batch=1 << 7, max_pages=1 << 23, heads=2), -2)])
def test_decode_refusals(lib, change, code):
    from triton_b200 import _lib
    assert lib.tb200_attention_decode(ctypes.byref(filled(_lib.AttentionDecodeArgs, **change)), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(cu_seqlens_q=None), -1), (dict(seq_lens=None), -1), (dict(page_size=0, cu_seqlens_k=None), -1),
    (dict(heads=9), -1), (dict(page_size=12), -2), (dict(page_size=-1), -1), (dict(head_dim=32), -2), (dict(dtype=3), -2),
    (dict(sm_scale=-1.0), -1), (dict(v=4104), -1), (dict(k_stride_head=64), -1), (dict(q_stride_tok=1004), -1),
    (dict(tokens_q=1 << 40), -2), (dict(max_pages=(1 << 21) + 1), -2), (dict(max_pages=1 << 62), -2),
    (dict(page_size=0, tokens_k=(1 << 25) + 1), -2), (dict(workspace=None), -1), (dict(workspace_bytes=8), -1), (dict(workspace=4112), -1),
    (dict(tokens_q=0), 0), (dict(batch=0), 0)])
def test_varlen_refusals(lib, change, code):
    from triton_b200 import _lib
    assert lib.tb200_attention_varlen_fwd(ctypes.byref(filled(_lib.AttentionVarlenArgs, **change)), None) == code


def test_varlen_workspace_holds_every_tile(lib):
    """Lengths are not known to the host: the bound on the tiles covers any split of the tokens."""
    from triton_b200 import _lib
    for heads, kv, d, tokens, batch in ((8, 2, 128, 1000, 7), (5, 1, 64, 1, 1), (6, 1, 256, 513, 40), (512, 1, 128, 9, 9)):
        a = filled(_lib.AttentionVarlenArgs, heads=heads, kv_heads=kv, head_dim=d, tokens_q=tokens, batch=batch)
        pack = 1
        while pack < 128 and heads // kv % (2 * pack) == 0:
            pack *= 2
        tile = 128 // pack * (1 if d == 256 else 2)
        worst = max(sum(-(-n // tile) for n in [1] * i + [tokens - i]) for i in range(min(batch, tokens)))
        assert lib.tb200_attention_varlen_workspace_bytes(ctypes.byref(a)) >= 32 + 32 * worst


@gpu
def test_argument_checks(cuda):
    f = fa()
    cache = Cache(cuda, [10, 20], 2, 128, BF16, 16).fill()
    q = torch.zeros(2, 8, 128, dtype=BF16, device=cuda)
    kv = torch.zeros(2, 2, 128, dtype=BF16, device=cuda)
    cu = offsets([1, 1], cuda)
    decode = lambda **kw: f.attention_decode(**{**dict(q=q, k_cache=cache.k, v_cache=cache.v, page_table=cache.table,
                                                       seq_lens=cache.seq_lens, sm_scale=0.1), **kw})
    varlen = lambda **kw: f.attention_varlen(**{**dict(q=q, k=kv, v=kv, cu_seqlens_q=cu, cu_seqlens_k=cu, sm_scale=0.1, causal=True), **kw})
    append = lambda **kw: f.append_paged_kv(**{**dict(q=q, k=kv, v=kv, k_cache=cache.k, v_cache=cache.v, page_table=cache.table,
                                                      seq_lens=cache.seq_lens), **kw})
    scale = torch.ones(1, device=cuda)
    pool8 = cache.k.to(E4M3)
    for bad in (dict(q=q[:1]), dict(q=q[:, :7]), dict(q=q[0]), dict(seq_lens=cache.seq_lens.long()), dict(seq_lens=cache.seq_lens.cpu()),
                dict(page_table=cache.table.cpu()), dict(k_cache=cache.k[:, :8]), dict(k_scale=scale, v_scale=scale),
                dict(k_cache=pool8, v_cache=pool8), dict(out=q[:1]), dict(out=q.float()), dict(out=q.transpose(0, 1)),
                dict(v_cache=cache.v.cpu()), dict(k_cache=cache.k[..., :64].contiguous())):
        with pytest.raises((AssertionError, RuntimeError)):
            decode(**bad)
    for bad in (dict(q=q[..., :96]), dict(q=q.float()), dict(q=q.half()), dict(q=q.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            decode(**bad)
    for bad in (dict(k=kv[:1]), dict(v=kv[..., :64]), dict(cu_seqlens_q=cu.long()), dict(cu_seqlens_k=cu[:2]), dict(k=kv.half()), dict(k=kv.cpu())):
        with pytest.raises(AssertionError):
            varlen(**bad)
    with pytest.raises(NotImplementedError):
        varlen(k=kv.clone().requires_grad_())
    cos, sin = tables(64, 128, cuda)
    for bad in (dict(k=kv[:1], v=kv[:1]), dict(cos=cos), dict(cos=cos.double(), sin=sin.double()), dict(cos=cos[:, :4], sin=sin[:, :4]),
                dict(cu_seqlens=cu[:2]), dict(q=None, q_out=q), dict(q=torch.zeros(3, 8, 128, dtype=BF16, device=cuda)), dict(q_out=q[:1]), dict(k_out=q),
                dict(k_cache=cache.k[:, :, :1], v_cache=cache.v[:, :, :1])):
        with pytest.raises(AssertionError):
            append(**bad)
    with pytest.raises(NotImplementedError):
        f.attention_varlen_paged(q, pool8, pool8, cu, cache.table, cache.seq_lens, 0.1, True)
    odd = torch.zeros(4, 12, 2, 128, dtype=BF16, device=cuda)
    with pytest.raises(NotImplementedError):
        f.attention_varlen_paged(q, odd, odd, cu, cache.table, cache.seq_lens, 0.1, True)
    from triton_b200 import _lib
    with pytest.raises(_lib.Tb200Error):
        decode(sm_scale=0.0)
