"""The serving operators in plain 64-bit form, and the bounds their tests use.

u(t) = torch.finfo(t).eps / 2 is the largest relative error of one rounding
to t. Attention, for a row with weights w_j = p_j / sum p and A = sum w_j |v_j|:
  * rounding p to the operand type: u(operand) A;
  * a score that is off by d moves a weight by at most 2 d: the sum of D exact
    products in fp32 is off by at most D 2^-22 sum |q k| scale (each partial
    sum rounded or cut at 2^-23 of the largest), exp2 and the scaling add
    2^-20 relative: 2 d A;
  * fp8 caches: q is scaled by a power of two into fp16, elements below 2^-14
    of the row's largest lose at most 2^-25 of it: d += 2^-25 max|q| sum |k| scale;
  * sums over n keys in fp32: (n + 64) 2^-23 A;
  * the result's own rounding: u(out) |o|, and half the smallest step.
"""
from __future__ import annotations

import math

import torch

FP8_MAX = 448.0


def u(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def attention_row_block(q, k, v, scale, out_dtype, operand_dtype, visible=None, fp8=False):
    """q [M, D], k, v [N, D] float64; visible [M, N] bool. Returns (o, bound) [M, D]."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = q @ k.t() * scale
    if visible is not None:
        s = s.masked_fill(~visible, -math.inf)
    w = torch.softmax(s, -1)
    w = torch.nan_to_num(w, nan=0.0)  # rows that see nothing
    o = w @ v
    a = w @ v.abs()
    d = (q.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale * q.shape[1] * 2.0 ** -22 + 2.0 ** -20
    if fp8:
        d = d + 2.0 ** -25 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1).max() * scale
    n = k.shape[0]
    bound = (a * (u(operand_dtype) + 2 * d + (n + 64) * 2.0 ** -23) * (1 + u(out_dtype))
             + u(out_dtype) * o.abs() + torch.finfo(out_dtype).smallest_normal * u(out_dtype) * 2)
    return o, bound


def prompt(q, k, v, starts, scale=None):
    """(out, bound) float64 [T, Hq, D]; rows outside every sequence are NaN."""
    t, hq, d = q.shape
    group = hq // k.shape[1]
    scale = scale if scale is not None else 1 / math.sqrt(d)
    out = torch.full((t, hq, d), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for a, b in zip(starts[:-1], starts[1:]):
        if b <= a:
            continue
        seen = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()
        for h in range(hq):
            out[a:b, h], bound[a:b, h] = attention_row_block(
                q[a:b, h].double(), k[a:b, h // group].double(), v[a:b, h // group].double(),
                scale, q.dtype, q.dtype, seen)
    return out, bound


def cache_tokens(cache, ids, layout, scale=None):
    """Tokens of blocks `ids` as [n, Hk, D] float64 and which of them exist."""
    ids = torch.as_tensor(ids, dtype=torch.long, device=cache.device)
    there = (ids >= 0) & (ids < cache.shape[0])
    x = cache[ids.clamp(0, max(cache.shape[0] - 1, 0))]
    if x.dtype == torch.uint8:
        x = x.view(torch.float8_e4m3fn)
    x = x.double()
    if layout == "HND":
        x = x.transpose(1, 2)
    if scale is not None:
        x = x * scale.double()
    bs = x.shape[1]
    return x.reshape(-1, *x.shape[2:]), there.repeat_interleave(bs)


def decode(q, kc, vc, table, lens, prefix, layout="NHD", k_scale=None, v_scale=None, scale=None):
    """(out, bound) float64 [B, Hq, D]."""
    b, hq, d = q.shape
    hk, bs = (kc.shape[2], kc.shape[1]) if layout == "NHD" else (kc.shape[1], kc.shape[2])
    group = hq // hk
    scale = scale if scale is not None else 1 / math.sqrt(d)
    fp8 = k_scale is not None
    prefix = prefix.tolist() if prefix is not None else []
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for r in range(b):
        n = min(max(int(lens[r]), 0), table.shape[1] * bs)
        row = table[r].tolist()
        ids = prefix + row[len(prefix):] if n >= len(prefix) * bs else row
        ids = ids[:-(-n // bs)]
        if not ids:
            continue
        k, there = cache_tokens(kc, ids, layout, k_scale)
        v, _ = cache_tokens(vc, ids, layout, v_scale)
        keep = there & (torch.arange(k.shape[0], device=q.device) < n)
        k, v = k[keep], v[keep]
        for h in range(hk):
            rows = slice(h * group, (h + 1) * group)
            out[r, rows], bound[r, rows] = attention_row_block(
                q[r, rows].double(), k[:, h], v[:, h], scale, q.dtype,
                torch.float16 if fp8 else q.dtype, fp8=fp8)
    return out, bound


def axis_of(sections, in_turns):
    axes = len(sections)
    if in_turns:
        return [i % axes if i % axes and i < axes * sections[i % axes] else 0
                for i in range(sum(sections))]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def mrope(x, w, positions, table, sections, in_turns, neox, eps=1e-6):
    """(y, bound before rounding, valid) float64 [T, H, D]. fp32 against 64 bits:
    the mean of D squares and its root are off by (D / 2 + 8) 2^-24 relative at
    most, the products and the sum of a rotation by 4 2^-24 of their parts."""
    rows, rotary = table.shape
    half = rotary // 2
    d = x.shape[-1]
    valid = ((positions >= 0) & (positions < rows)).all(0)
    place = positions.clamp(0, rows - 1)
    axis = torch.tensor(axis_of(sections, in_turns), device=x.device)
    pair = torch.arange(half, device=x.device)
    at = place[axis].t()  # [T, half]
    cos, sin = table.double()[at, pair][:, None], table.double()[at, half + pair][:, None]
    n = x.double()
    n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + eps) * w.double()
    first = slice(0, half) if neox else slice(0, rotary, 2)
    second = slice(half, rotary) if neox else slice(1, rotary, 2)
    a, b = n[..., first].clone(), n[..., second].clone()
    y, parts = n.clone(), n.abs()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    parts[..., first] = (a * cos).abs() + (b * sin).abs()
    parts[..., second] = (b * cos).abs() + (a * sin).abs()
    return y, parts * (d / 2 + 16) * 2.0 ** -24, valid


def plan(context, query, table, free, count, block_size, tokens):
    """The step plan by a plain walk over the requests (lists of ints, table a
    list of rows, changed in place)."""
    pool = len(free)
    width = len(table[0]) if table else 0
    starts, lens = [0], []
    positions, slots = [-1] * tokens, [-1] * tokens
    left = min(max(count, 0), pool)
    total, needed = 0, 0
    for r, (c, q) in enumerate(zip(context, query)):
        c, q = max(c, 0), max(q, 0)
        held, want = -(-c // block_size), -(-(c + q) // block_size)
        narrow = want > width or c + q >= 2 ** 31
        need = 0 if narrow else want - held
        total += q
        needed += need
        served = not narrow and total <= tokens and (need == 0 or needed <= min(max(count, 0), pool))
        if served:
            for b in range(held, want):
                left -= 1
                table[r][b] = free[left]
        for i in range(q):
            t = total - q + i
            if t >= tokens:
                break
            positions[t] = c + i
            block = table[r][(c + i) // block_size] if served else -1
            slots[t] = block * block_size + (c + i) % block_size if 0 <= block < pool else -1
        starts.append(min(total, tokens))
        lens.append(c + q if served else c)
    return starts, lens, positions, slots, left


def release(lens, finished, table, free, count, block_size, shared):
    pool = len(free)
    count = min(max(count, 0), pool)
    for n, done, row in zip(lens, finished, table):
        if not done:
            continue
        for block in row[shared:-(-max(n, 0) // block_size)]:
            if 0 <= block < pool and count < pool:
                free[count] = block
                count += 1
    return count
