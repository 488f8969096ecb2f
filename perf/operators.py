"""The operators of a serving step around a paged key / value cache, as cases that can be run and timed.

``append``    rotates new queries and keys by their positions and appends keys and values to the cache;
``decode``    attention of one new token per sequence over the cache;
``prompt``    causal attention of whole prompts, packed one behind the other, keys and values packed too;
``continue``  the same for prompts whose beginning is in the cache already: keys and values come from its pages.

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the framework's calls.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
_E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def _case(name, op, batch, past, new, heads, kv_heads, head_dim, dtype="bf16", cache="same", page=16, layout="token",
          rotary_dim=0, interleaved=False, mix=1):
    """`past`, `new`: (least, most) tokens per sequence that were there before, and that come with this call."""
    c = {"op": op, "batch": batch, "past_min": past[0], "past_max": past[1], "new_min": new[0], "new_max": new[1],
         "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "cache": cache, "page": page,
         "layout": layout, "rotary_dim": rotary_dim, "interleaved": interleaved, "mix": mix}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user's next token: the call is as long as its launch
        _case("append_1", "append", 1, (700, 700), (1, 1), 32, 8, 128, rotary_dim=128),
        # a full decode batch into an 8-bit cache, pages stored head by head
        _case("append_batch_fp8", "append", 200, (1, 900), (1, 1), 64, 8, 128, cache="e4m3", page=64, layout="head",
              rotary_dim=128, mix=2),
        # prompts of many lengths that came in together
        _case("append_prompt", "append", 9, (0, 600), (50, 8000), 32, 8, 128, rotary_dim=128, mix=3),
        # one user's next token over a short conversation
        _case("decode_1", "decode", 1, (900, 900), (1, 1), 32, 8, 128),
        # an ordinary batch: lengths from a first token to some thousands
        _case("decode_batch", "decode", 48, (0, 6000), (1, 1), 32, 8, 128, mix=4),
        # many users of a small model whose heads share nothing
        _case("decode_mha", "decode", 130, (17, 2000), (1, 1), 16, 16, 64, dtype="fp16", page=32, layout="head", mix=5),
        # two documents of some hundred thousand tokens: few rows, a very long axis
        _case("decode_long", "decode", 2, (200000, 400000), (1, 1), 64, 8, 128, page=64, mix=6),
        # long contexts in an 8-bit cache
        _case("decode_fp8", "decode", 64, (2000, 30000), (1, 1), 64, 8, 128, cache="e4m3", page=64, layout="head", mix=7),
        # one short question
        _case("prompt_short", "prompt", 1, (0, 0), (37, 37), 32, 8, 128),
        # questions of many lengths packed into one call
        _case("prompt_packed", "prompt", 24, (0, 0), (5, 3000), 32, 8, 128, mix=8),
        # one long document
        _case("prompt_long", "prompt", 1, (0, 0), (16001, 16001), 32, 8, 128),
        # further turns of conversations whose beginning is cached
        _case("continue_pages", "continue", 5, (1000, 12000), (100, 2000), 16, 2, 128, page=64, mix=9),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt", "continue"])
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    group = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    while kv_heads * group > 64:
        group = rng.choice([1, 2, 3, 4])
    heads = kv_heads * group
    dtype, layout, mix = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["token", "head"]), rng.randrange(1 << 20)
    page = rng.choice([16, 16, 32, 64, 128, 48])
    if op == "append":
        rotary = rng.choice([head_dim, head_dim, head_dim // 2])
        one = rng.random() < 0.5
        batch = _log_int(rng, 1, 300) if one else _log_int(rng, 1, 12)
        new = (1, 1) if one else (_log_int(rng, 1, 60), _log_int(rng, 61, 16000 // batch))
        return _case("", op, batch, (0, _log_int(rng, 1, 1000)), new, heads, kv_heads, head_dim, dtype,
                     rng.choice(["same", "e4m3"]), rng.choice([page, page, 5]), layout, rotary, rng.random() < 0.3, mix)
    if op == "decode":
        # at most 8 GB of keys and values once the plain form has padded every sequence to the longest
        batch = _log_int(rng, 1, 256)
        most = min(400000, int(1e9 / (batch * kv_heads * head_dim)))
        length = _log_int(rng, 20, most)
        return _case("", op, batch, (rng.choice([0, length // 4]), length), (1, 1), heads, kv_heads, head_dim, dtype,
                     rng.choice(["same", "same", "e4m3"]), rng.choice([page, page, 5]), layout, mix=mix)
    batch = _log_int(rng, 1, 24)
    most = int(math.sqrt(32.0 * 16001 ** 2 / (batch * heads)) * math.sqrt(128.0 / max(head_dim, 128)))
    new_max = _log_int(rng, 30, min(most, 12000, 40000 // batch))
    new = (max(1, new_max // rng.choice([1, 4, 40])), new_max)
    if op == "prompt":
        return _case("", op, batch, (0, 0), new, heads, kv_heads, head_dim, dtype, mix=mix)
    new = (min(new[0], 2000), min(new[1], 2000))
    past_max = max(1, min(most * most // (2 * new[1]) - new[1], 20000))
    return _case("", op, batch, (0, past_max), new, heads, kv_heads, head_dim, dtype, "same", page, layout, mix=mix)


def _lengths(case):
    """(tokens before the call, new tokens) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])

    def some(low, high):
        if low == high:
            return low
        return min(high, max(low, int(math.exp(rng.uniform(math.log(low + 1), math.log(high + 2)))) - 1))

    past = [some(case["past_min"], case["past_max"]) for _ in range(case["batch"])]
    new = [some(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    past[-1], new[-1] = case["past_max"], case["new_max"]  # the longest is always there
    return past, new


# ------------------------------------------------------------------------------------------------ inputs
def _randn(shape, dtype, g, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _pages(case, n_pages, g, dtype):
    """One of the two caches, seen as [pages, tokens of a page, heads, head_dim] whatever its order in memory."""
    shape = [n_pages, case["page"], case["kv_heads"], case["head_dim"]]
    if case["layout"] == "head":
        shape[1], shape[2] = shape[2], shape[1]
    cache = torch.empty(shape, dtype=dtype, device="cuda")
    flat = cache.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i:i + (1 << 28)]
        if dtype == torch.float8_e4m3fn:
            part.copy_(_randn(part.shape, torch.float32, g, 40.0).clamp_(-_E4M3_MAX, _E4M3_MAX).to(dtype))
        else:
            part.copy_(_randn(part.shape, dtype, g))
    return cache.transpose(1, 2) if case["layout"] == "head" else cache


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    past, new = _lengths(case)
    total = sum(new)
    dtype, d = _DTYPES[case["dtype"]], case["head_dim"]
    s = {"op": case["op"], "sm_scale": 1.0 / math.sqrt(d), "max_new": max(new), "max_len": max(p + n for p, n in zip(past, new))}
    s["q"] = _randn((total, case["heads"], d), dtype, g)
    s["cu_new"] = _offsets(new)
    if case["op"] in ("append", "prompt"):
        s["k"] = _randn((total, case["kv_heads"], d), dtype, g)
        s["v"] = _randn((total, case["kv_heads"], d), dtype, g)
    if case["op"] == "prompt":
        return s
    # the cache: every sequence's pages lie anywhere in the pool, and the pool has some pages to spare
    s["seq_lens"] = torch.tensor([p + n for p, n in zip(past, new)], dtype=torch.int32, device="cuda")
    need = [-(-(p + n) // case["page"]) for p, n in zip(past, new)]
    n_pages, width = sum(need) + 3, max(need)
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    has = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[has] = order[:sum(need)]
    s["page_table"] = table
    cache_dtype = dtype if case["cache"] == "same" else _DTYPES[case["cache"]]
    s["k_cache"] = _pages(case, n_pages, g, cache_dtype)
    s["v_cache"] = _pages(case, n_pages, g, cache_dtype)
    s["k_scale"] = s["v_scale"] = None
    if cache_dtype == torch.float8_e4m3fn:
        s["k_scale"], s["v_scale"] = (0.02 + 0.01 * torch.rand(case["kv_heads"], generator=g, device="cuda") for _ in "kv")
    s["one_each"] = case["new_max"] == 1
    s["interleaved"] = case["interleaved"]
    if case["op"] == "append":
        s["cos"], s["sin"] = _rotation(case, s["max_len"])
    return s


def _rotation(case, positions):
    """The tables that a model keeps: cosines and sines of every position, angles in 64 bits, rounded once."""
    half = case["rotary_dim"] // 2
    speed = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * speed
    return angle.cos().float(), angle.sin().float()


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"append": _append, "decode": _decode, "prompt": _prompt, "continue": _continue}[s["op"]](s)


def _own(s):
    from triton_b200.tutorials import blackwell_fa_paged as fa
    op = s["op"]
    if op == "decode":
        return fa.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["seq_lens"], s["sm_scale"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "append":
        q = fa.append_paged_kv(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["seq_lens"],
                               None if s["one_each"] else s["cu_new"], cos=s["cos"], sin=s["sin"],
                               interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "prompt":
        return fa.attention_varlen(s["q"], s["k"], s["v"], s["cu_new"], s["cu_new"], s["sm_scale"], True)
    return fa.attention_varlen_paged(s["q"], s["k_cache"], s["v_cache"], s["cu_new"], s["page_table"], s["seq_lens"],
                                     s["sm_scale"], True)


def _rotate(x, cos, sin, interleaved):
    """x [tokens, heads, d]; cos, sin [tokens, rotary_dim / 2]: the first rotary_dim columns turn, the others stay."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _append(s):
    t = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    cu = s["cu_new"]
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = (s["seq_lens"][b] - (cu[b + 1] - cu[b]) + t - cu[b]).long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["q"].float(), cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, s["interleaved"])
    v = s["v"].float()
    size = s["k_cache"].shape[1]
    page, at = s["page_table"][b, pos // size].long(), pos % size
    if s["k_scale"] is not None:
        k = (k / s["k_scale"][:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        v = (v / s["v_scale"][:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        s["k_cache"].view(torch.uint8)[page, at] = k.to(torch.float8_e4m3fn).view(torch.uint8)
        s["v_cache"].view(torch.uint8)[page, at] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["k_cache"][page, at] = k.to(s["k_cache"].dtype)
        s["v_cache"][page, at] = v.to(s["v_cache"].dtype)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _from_pages(s, cache, scale):
    """Every sequence's keys or values, padded to the longest: [batch, kv_heads, max_len, d] in 32 bits."""
    pos = torch.arange(s["max_len"], device="cuda")
    size = cache.shape[1]
    page = s["page_table"][:, pos // size].long().clamp(min=0)
    x = cache.view(torch.uint8)[page, pos % size].view(cache.dtype) if scale is not None else cache[page, pos % size]
    x = x.float().transpose(1, 2)
    return x if scale is None else x * scale[:, None, None]


def _attend(q, k, v, visible, sm_scale):
    """q [batch, kv_heads, rows, d], k and v [batch, kv_heads, keys, d], visible broadcast to [batch, kv_heads, rows, keys]."""
    p = torch.matmul(q * sm_scale, k.transpose(2, 3))
    p.masked_fill_(~visible, float("-inf"))
    p.sub_(p.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _decode(s):
    k, v = _from_pages(s, s["k_cache"], s["k_scale"]), _from_pages(s, s["v_cache"], s["v_scale"])
    batch, heads, d = s["q"].shape
    q = s["q"].float().view(batch, k.shape[1], -1, d)
    visible = torch.arange(s["max_len"], device="cuda") < s["seq_lens"][:, None, None, None]
    return _attend(q, k, v, visible, s["sm_scale"]).reshape(batch, heads, d).to(s["q"].dtype)


def _padded(x, cu, longest):
    """Packed rows [tokens, heads, d] as [batch, longest, heads, d] in 32 bits; rows past a sequence's end are another's."""
    at = cu[:-1, None] + torch.arange(longest, device="cuda")
    return x[at.clamp(max=x.shape[0] - 1).long()].float()


def _prompt_over(s, k, v, k_lens):
    """Causal attention of the packed queries over padded keys: the last query of a sequence sees all of its keys."""
    tokens, heads, d = s["q"].shape
    cu, longest, kv_heads = s["cu_new"], s["max_new"], k.shape[1]
    batch, group = cu.numel() - 1, heads // kv_heads
    q = _padded(s["q"], cu, longest).view(batch, longest, kv_heads, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, kv_heads, group * longest, d)
    row = torch.arange(longest, device="cuda")
    last = row + (k_lens - (cu[1:] - cu[:-1]))[:, None]
    visible = torch.arange(k.shape[2], device="cuda") <= last[:, :, None]
    visible = visible.repeat(1, group, 1)[:, None]
    o = _attend(q, k, v, visible, s["sm_scale"]).view(batch, kv_heads, group, longest, d)
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o.permute(0, 3, 1, 2, 4)[b, (t - cu[b]).long()].reshape(tokens, heads, d).to(s["q"].dtype)


def _prompt(s):
    k, v = (_padded(x, s["cu_new"], s["max_new"]).transpose(1, 2) for x in (s["k"], s["v"]))
    return _prompt_over(s, k, v, s["cu_new"][1:] - s["cu_new"][:-1])


def _continue(s):
    return _prompt_over(s, _from_pages(s, s["k_cache"], None), _from_pages(s, s["v_cache"], None), s["seq_lens"])


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    past, new = _lengths(case)
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    size, cache = 2, 1 if case["cache"] == "e4m3" else 2
    tokens = sum(new)
    length = [p + n for p, n in zip(past, new)]
    rows = 2 * tokens * heads * d * size  # queries in; queries or outputs out
    if case["op"] == "append":
        table = 4 * case["rotary_dim"] * sum(min(n, m) for n, m in zip(new, length))
        return {"bytes": rows + 2 * tokens * kv_heads * d * (size + cache) + table,
                "flops": 3 * tokens * (heads + kv_heads) * case["rotary_dim"]}
    if case["op"] == "decode":
        return {"bytes": rows + 2 * sum(length) * kv_heads * d * cache, "flops": 4 * sum(length) * heads * d}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": rows + 2 * sum(length) * kv_heads * d * size, "flops": 4 * pairs * heads * d}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    size = case["page"]
    group = case["heads"] // case["kv_heads"]
    if case["op"] == "append":
        return _exact_append(case, s, past, new)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (p, n) in enumerate(zip(past, new)):
        q = s["q"][first:first + n].double()
        if case["op"] == "prompt":
            k, v = s["k"][first:first + n], s["v"][first:first + n]
        else:
            k, v = (_exact_rows(x, s["page_table"][i, :-(-(p + n) // size)], p + n) for x in (s["k_cache"], s["v_cache"]))
        later = torch.arange(p + n, device="cuda")[None] > p + torch.arange(n, device="cuda")[:, None]
        for h in range(case["heads"]):
            kh, vh = k[:, h // group].double(), v[:, h // group].double()
            if s.get("k_scale") is not None:
                kh, vh = kh * s["k_scale"][h // group].double(), vh * s["v_scale"][h // group].double()
            score = (q[:, h] @ kh.T) * s["sm_scale"]
            score[later] = float("-inf")
            out[first:first + n, h] = torch.softmax(score, dim=1) @ vh
        first += n
    return out


def _exact_rows(cache, pages, length):
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    return raw[pages.long()].flatten(0, 1)[:length].contiguous().view(cache.dtype)


def _exact_append(case, s, past, new):
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(past, new)])
    seq = torch.cat([torch.full((n, ), i, device="cuda") for i, n in enumerate(new)])
    half = case["rotary_dim"] // 2
    # a pair (a, b) is the complex number a + ib: the rotation multiplies it by cos + i sin
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]

    def rotated(x):
        x = x.double().clone()
        if case["interleaved"]:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        else:
            a, b = x[..., :half], x[..., half:2 * half]
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        a.copy_(z.real)
        b.copy_(z.imag)
        return x

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k, v = rotated(s["k"]), s["v"].double()
    if s["k_scale"] is not None:
        k = (k / s["k_scale"].double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        v = (v / s["v_scale"].double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
    page = s["page_table"][seq, pos // case["page"]].long()
    k_cache[page, pos % case["page"]] = k
    v_cache[page, pos % case["page"]] = v
    return {"q": rotated(s["q"]), "k_cache": k_cache, "v_cache": v_cache}
