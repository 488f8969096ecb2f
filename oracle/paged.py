"""Oracle for the paged-cache operators (test infrastructure only): rotation and append, attention of packed sequences and
of single tokens over a cache, restated in 64 bits, one sequence and head at a time. Works on any device."""
import math

import torch


def cached_rows(cache, pages, page_size, length, scale=None):
    """The first `length` rows of one sequence, [length, kv_heads, d] in 64 bits; a page outside the pool is zeros."""
    n, d = cache.shape[0], cache.shape[3]
    out = torch.zeros(length, cache.shape[2], d, dtype=torch.float64, device=cache.device)
    for i in range(-(-length // page_size)):
        page = int(pages[i])
        rows = min(page_size, length - i * page_size)
        if 0 <= page < n:
            out[i * page_size:i * page_size + rows] = cache[page, :rows].to(torch.float32).double()
    return out if scale is None else out * scale.double().reshape(-1, 1)


def sequence_attention(q, k, v, sm_scale, causal):
    """q [n_q, heads, d], k and v [n_k, kv_heads, d] (64 bits). Returns o, base-2 log-sum-exp [n_q, heads], and
    sum_j p_j |v_j|, the scale of the rounding errors of the probabilities."""
    n_q, heads, d = q.shape
    n_k, group = k.shape[0], heads // k.shape[1]
    o = torch.zeros(n_q, heads, d, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(o)
    lse = torch.full((n_q, heads), -math.inf, dtype=torch.float64, device=q.device)
    if n_q == 0 or n_k == 0:
        return o, lse, size
    hidden = torch.arange(n_k, device=q.device)[None] > torch.arange(n_q, device=q.device)[:, None] + (n_k - n_q)
    for h in range(heads):
        s = q[:, h] @ k[:, h // group].T * sm_scale
        if causal:
            s = s.masked_fill(hidden, -math.inf)
        row = torch.logsumexp(s, dim=1)
        p = torch.exp(s - row.masked_fill(row == -math.inf, 0.0)[:, None])
        o[:, h], size[:, h] = p @ v[:, h // group], p @ v[:, h // group].abs()
        lse[:, h] = row / math.log(2.0)
    return o, lse, size


def rotated(x, positions, cos, sin, interleaved):
    """x [tokens, heads, d]; the first 2 * cos.shape[1] columns turn by the angles of row `positions`. 64 bits."""
    x = x.double().clone()
    if cos is None:
        return x
    half = cos.shape[1]
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c, s = cos[positions, j].double()[:, None], sin[positions, j].double()[:, None]
        xa, xb = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x
