"""Operators of a serving step around the paged KV cache, with the calls that are timed.

Four operators that a serving step runs one after the other:

* ``plan`` / ``release``: block tables, positions and slot maps from request
  lengths, with the free blocks of the pool as a stack; finished requests
  give their blocks back;
* ``mrope``: per-head Q/K RMSNorm + rotation by positions with several axes
  (time, height, width) + the paged KV store;
* ``prompt``: causal attention of packed prompts of different lengths with
  grouped heads;
* ``decode``: attention of one new token per request over the paged cache,
  for a batch whose requests begin with the same blocks.

``run`` computes them with elementary torch operations where ``own`` is false,
and with this repository's operators where it is true.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "sm120-norm-fusion-kernels_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
_DEVICE = "cuda"
_EPS = 1e-6
_FP8_MAX = 448.0


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from sm120_rmsnorm import extensions, serving
    return extensions, serving


# ---- the cases --------------------------------------------------------------------------
def listed():
    return [
        # one request decoding alone: nothing but latency
        dict(name="plan_decode_1", op="plan", requests=1, query="one", context=4096, block_size=16,
             padding=0, short=False, shape_seed=1),
        # a full decode batch in a graph-sized buffer, 23 rows of it padding
        dict(name="plan_decode_1001", op="plan", requests=1001, query="one", context=32768,
             block_size=16, padding=23, short=False, shape_seed=2),
        # a chunked-prefill step: ragged prompts, some of them continued
        dict(name="plan_prefill_ragged", op="plan", requests=67, query=1900, context=8192,
             block_size=16, padding=100, short=False, shape_seed=3),
        # about a third of a batch finishes in the same step
        dict(name="release_1001", op="release", requests=1001, context=8192, block_size=16,
             shared=8, shape_seed=4),
        # decode of a small batch, fp8 cache, heads before slots
        dict(name="mrope_decode_33_fp8", op="mrope", tokens=33, hq=32, hk=8, d=128, rotary=128,
             dtype="bf16", sections="24,20,20", mixed=True, neox=True, cache="fp8", layout="HND",
             block_size=16, padding=0),
        # a prompt with pictures in it
        dict(name="mrope_prefill_8191", op="mrope", tokens=8191, hq=64, hk=8, d=128, rotary=128,
             dtype="bf16", sections="16,24,24", mixed=False, neox=True, cache="same",
             layout="NHD", block_size=16, padding=57),
        # a few chat turns at once
        dict(name="prompt_short", op="prompt", requests=7, length=190, uneven=True, hq=32, hk=8,
             d=128, dtype="bf16", padding=3, shape_seed=5),
        # a prefill step of mixed lengths, small heads
        dict(name="prompt_mixed_fp16_d64", op="prompt", requests=19, length=1500, uneven=True,
             hq=16, hk=8, d=64, dtype="fp16", padding=0, shape_seed=6),
        # one long document
        dict(name="prompt_long", op="prompt", requests=1, length=16384, uneven=False, hq=32, hk=8,
             d=128, dtype="bf16", padding=0, shape_seed=7),
        # a handful of chats behind one system prompt
        dict(name="decode_5", op="decode", batch=5, prefix=64, suffix=100, hq=32, hk=8, d=128,
             dtype="bf16", cache="same", layout="NHD", block_size=16, empty=False, shape_seed=8),
        # a middling batch over an fp8 cache, one row of it padding
        dict(name="decode_61_fp8", op="decode", batch=61, prefix=512, suffix=600, hq=32, hk=8,
             d=128, dtype="bf16", cache="fp8", layout="HND", block_size=16, empty=True,
             shape_seed=9),
        # a large batch of questions about one long document
        dict(name="decode_256", op="decode", batch=256, prefix=2048, suffix=1024, hq=32, hk=8,
             d=128, dtype="bf16", cache="same", layout="NHD", block_size=16, empty=False,
             shape_seed=10),
    ]


def _log(rng, low, high):
    """A whole number spread evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["plan", "release", "mrope", "mrope", "prompt", "prompt", "prompt", "decode",
                     "decode", "decode"])
    seed = rng.randrange(1 << 30)
    if op == "plan":
        requests = _log(rng, 1, 2048)
        query = "one" if rng.random() < 0.4 else _log(rng, 1, max(1, min(8192, 65536 // requests)))
        return dict(op=op, requests=requests, query=query, context=_log(rng, 1, 32768),
                    block_size=rng.choice([16, 32, 64]), padding=rng.choice([0, rng.randrange(64)]),
                    short=rng.random() < 0.2, shape_seed=seed)
    if op == "release":
        return dict(op=op, requests=_log(rng, 1, 2048), context=_log(rng, 1, 16384),
                    block_size=rng.choice([16, 32, 64]), shared=rng.choice([0, rng.randrange(16)]),
                    shape_seed=seed)
    if op == "mrope":
        d = rng.choice([64, 128, 128, 256])
        rotary = rng.choice([d, d, d // 2])
        half = rotary // 2
        first = rng.randrange(1, half // 2)
        mixed = rng.random() < 0.5
        if mixed:  # the axes take turns: height and width as often as there is room
            second = rng.randrange(1, half // 3 + 1)
            third = rng.randrange(1, half // 3 + 1)
            sections = [half - second - third, second, third]
        elif rng.random() < 0.5:  # whole multiples of eight
            sections = [half // 4, 3 * half // 8, 3 * half // 8]
        else:
            second = rng.randrange(1, half - first)
            sections = [first, second, half - first - second]
        hq, hk = rng.choice([(32, 8), (64, 8), (16, 8), (4, 2), (28, 4)])
        return dict(op=op, tokens=_log(rng, 1, 16384), hq=hq, hk=hk, d=d, rotary=rotary,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    sections=",".join(map(str, sections)), mixed=mixed, neox=rng.random() < 0.8,
                    cache=rng.choice(["same", "fp8", "none"]), layout=rng.choice(["NHD", "HND"]),
                    block_size=rng.choice([16, 32]), padding=rng.choice([0, rng.randrange(20)]))
    if op == "prompt":
        d = rng.choice([64, 128, 128, 128, 256])
        hq, hk = rng.choice([(32, 8), (32, 8), (16, 8), (8, 8), (4, 2), (28, 4), (40, 8)])
        requests = _log(rng, 1, 64)
        # at most 8192 tokens a sequence for the wide forms: no dearer than the longest listed
        longest = 16384 if hq * d <= 4096 else 8192
        return dict(op=op, requests=requests, length=_log(rng, 1, max(1, longest // requests)),
                    uneven=rng.random() < 0.8, hq=hq, hk=hk, d=d,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    padding=rng.choice([0, rng.randrange(20)]), shape_seed=seed)
    batch = _log(rng, 1, 256)
    hq, hk = rng.choice([(32, 8), (32, 8), (64, 8), (16, 8), (8, 8), (28, 4)])
    return dict(op="decode", batch=batch, prefix=rng.choice([0, _log(rng, 1, 1024)]),
                suffix=_log(rng, 1, max(1, min(16384, 262144 // batch))), hq=hq, hk=hk,
                d=rng.choice([64, 128, 128, 256]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                cache=rng.choice(["same", "same", "fp8"]), layout=rng.choice(["NHD", "HND"]),
                block_size=rng.choice([16, 16, 32, 64]), empty=rng.random() < 0.3, shape_seed=seed)


def _lengths(case):
    """The lengths that a case stands for: part of its shape, the same for every seed."""
    r = random.Random(case["shape_seed"])
    if case["op"] == "plan":
        n = case["requests"]
        context = [_log(r, 1, case["context"]) for _ in range(n)]
        if case["query"] == "one":
            return context, [1] * n
        # about half of the prompts are new, the others go on
        context = [0 if r.random() < 0.5 else c for c in context]
        top = case["query"]
        return context, [r.randint(0 if r.random() < 0.1 else 1, top) for _ in range(n)]
    if case["op"] == "release":
        return [r.randint(0, case["context"]) for _ in range(case["requests"])], None
    if case["op"] == "prompt":
        n, top = case["requests"], case["length"]
        return ([r.randint(1, top) for _ in range(n)] if case["uneven"] else [top] * n), None
    own_tokens = [r.randint(1, case["suffix"]) for _ in range(case["batch"])]
    total = [case["prefix"] * case["block_size"] + n for n in own_tokens]
    if case["empty"]:  # a padding row, and one that does not reach the end of the prefix
        total[-1] = 0
        if case["batch"] > 2:
            total[1] = min(total[1], 7)
    return total, None


def _blocks(tokens, block_size):
    return -(-tokens // block_size)


# ---- inputs -----------------------------------------------------------------------------
def _rng(seed):
    return torch.Generator(device=_DEVICE).manual_seed(int(seed))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=_DEVICE)


def _cos_sin(positions, rotary, base=1e6):
    inv = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=_DEVICE) / rotary)
    f = torch.outer(torch.arange(positions, dtype=torch.float64, device=_DEVICE), inv)
    return torch.cat((f.cos(), f.sin()), dim=-1).float()


def _prepare_plan(case, g):
    context, query = _lengths(case)
    bs = case["block_size"]
    width = _blocks(case["context"] + (1 if case["query"] == "one" else case["query"]), bs)
    n = case["requests"]
    held = [_blocks(c, bs) for c in context]
    need = [_blocks(c + q, bs) - h for c, q, h in zip(context, query, held)]
    spare = max(1, sum(need) // 2) if case["short"] else sum(need) + 64
    pool = sum(held) + spare
    ids = torch.randperm(pool, device=_DEVICE, generator=g).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=_DEVICE)
    column = torch.arange(width, device=_DEVICE)
    filled = column[None, :] < _ints(held)[:, None]
    table[filled] = ids[:sum(held)]
    free = torch.full((pool,), -1, dtype=torch.int32, device=_DEVICE)
    free[:spare] = ids[sum(held):]
    tokens = sum(query) + case["padding"]
    return dict(op="plan", block_size=bs, context=_ints(context), query=_ints(query), table=table,
                free=free, count=_ints([spare]), count_out=_ints([0]),
                query_start=_ints([0] * (n + 1)), seq_lens=_ints([0] * n),
                positions=torch.zeros(tokens, dtype=torch.int64, device=_DEVICE),
                slots=torch.zeros(tokens, dtype=torch.int32, device=_DEVICE))


def _prepare_release(case, g):
    lengths, _ = _lengths(case)
    bs = case["block_size"]
    width = _blocks(case["context"], bs)
    n = case["requests"]
    held = [_blocks(c, bs) for c in lengths]
    pool = sum(held) + 64
    ids = torch.randperm(pool, device=_DEVICE, generator=g).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=_DEVICE)
    filled = torch.arange(width, device=_DEVICE)[None, :] < _ints(held)[:, None]
    table[filled] = ids[:sum(held)]
    free = torch.full((pool,), -1, dtype=torch.int32, device=_DEVICE)
    free[:64] = ids[sum(held):]
    finished = torch.rand(n, device=_DEVICE, generator=g) < 0.35
    return dict(op="release", block_size=bs, shared=case["shared"], seq_lens=_ints(lengths),
                finished=finished, table=table, free=free, count=_ints([64]),
                count_out=_ints([0]))


def _cache_pages(blocks, hk, d, block_size, layout, dtype):
    """A paged cache and the larger buffer that it is the front of (one block more)."""
    shape = (blocks + 1, block_size, hk, d) if layout == "NHD" else (blocks + 1, hk, block_size, d)
    whole = torch.zeros(shape, dtype=dtype, device=_DEVICE)
    return whole[:-1], whole


def _prepare_mrope(case, g):
    t, hq, hk, d = case["tokens"] + case["padding"], case["hq"], case["hk"], case["d"]
    dtype = _DTYPES[case["dtype"]]
    table_rows = 32768
    # the output of one Q/K/V projection, split into views
    qkv = torch.randn(t, (hq + 2 * hk) * d, device=_DEVICE, generator=g).to(dtype)
    q = qkv[:, :hq * d].view(t, hq, d)
    k = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
    v = qkv[:, (hq + hk) * d:].view(t, hk, d)
    # runs of text (all axes alike) and pictures (a place in a grid behind a start)
    base = torch.randint(0, table_rows - 2048, (1,), device=_DEVICE, generator=g)
    step = torch.arange(t, device=_DEVICE)
    picture = (step // 600) % 2 == 1
    inside = step % 600
    time = base + torch.where(picture, step // 600 * 2, step // 16)
    height = torch.where(picture, time + inside // 30, time)
    width = torch.where(picture, time + inside % 30, time)
    positions = torch.stack((time, height, width)).clamp_(max=table_rows - 1)
    if case["padding"]:
        positions[:, -case["padding"]:] = -1
    state = dict(op="mrope", q=q, k=k, v=v, positions=positions,
                 qw=(1 + 0.1 * torch.randn(d, device=_DEVICE, generator=g)).to(dtype),
                 kw=(1 + 0.1 * torch.randn(d, device=_DEVICE, generator=g)).to(dtype),
                 table=_cos_sin(table_rows, case["rotary"]), neox=case["neox"],
                 sections=[int(s) for s in case["sections"].split(",")], mixed=case["mixed"],
                 layout=case["layout"], block_size=case["block_size"],
                 q_out=torch.zeros(t, hq, d, dtype=dtype, device=_DEVICE),
                 k_out=torch.zeros(t, hk, d, dtype=dtype, device=_DEVICE),
                 kc=None, vc=None, slots=None, k_scale=None, v_scale=None)
    if case["cache"] != "none":
        blocks = _blocks(t, case["block_size"]) + 2
        stored = torch.float8_e4m3fn if case["cache"] == "fp8" else dtype
        for name in ("kc", "vc"):
            state[name], state[name + "_whole"] = _cache_pages(blocks, hk, d, case["block_size"],
                                                               case["layout"], stored)
        slots = torch.randperm(blocks * case["block_size"], device=_DEVICE, generator=g)[:t]
        slots[torch.rand(t, device=_DEVICE, generator=g) < 0.02] = -1
        state["slots"] = slots.to(torch.int32)
        if case["cache"] == "fp8":
            state["k_scale"] = torch.tensor([0.02], device=_DEVICE)
            state["v_scale"] = torch.tensor([0.015], device=_DEVICE)
    return state


def _prepare_prompt(case, g):
    lengths, _ = _lengths(case)
    t, hq, hk, d = sum(lengths) + case["padding"], case["hq"], case["hk"], case["d"]
    dtype = _DTYPES[case["dtype"]]
    start = [0]
    for n in lengths:
        start.append(start[-1] + n)
    # normalised queries and keys, and values, as views of one projection's output
    qkv = torch.randn(t, (hq + 2 * hk) * d, device=_DEVICE, generator=g).to(dtype)
    q = qkv[:, :hq * d].view(t, hq, d)
    k = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
    v = qkv[:, (hq + hk) * d:].view(t, hk, d)
    q.mul_(1.5)
    return dict(op="prompt", q=q, k=k, v=v, start=_ints(start), lengths=lengths,
                out=torch.zeros(t, hq, d, dtype=dtype, device=_DEVICE))


def _prepare_decode(case, g):
    total, _ = _lengths(case)
    b, hq, hk, d, bs = case["batch"], case["hq"], case["hk"], case["d"], case["block_size"]
    dtype = _DTYPES[case["dtype"]]
    p = case["prefix"]
    held = [max(0, _blocks(n, bs) - p) if n >= p * bs else _blocks(n, bs) for n in total]
    blocks = p + sum(held) + 3
    shape = (blocks, bs, hk, d) if case["layout"] == "NHD" else (blocks, hk, bs, d)
    ids = torch.randperm(blocks, device=_DEVICE, generator=g).to(torch.int32)
    width = max(1, max(_blocks(n, bs) for n in total))
    table = torch.full((b, width), -1, dtype=torch.int32, device=_DEVICE)
    column = torch.arange(width, device=_DEVICE)[None, :]
    first = _ints([p if n >= p * bs else 0 for n in total])[:, None]
    filled = (column >= first) & (column < first + _ints(held)[:, None])
    table[filled] = ids[p:p + sum(held)]
    table = torch.where((column < p) & (first == p), ids[column.clamp(max=max(p, 1) - 1)], table)
    state = dict(op="decode", layout=case["layout"], block_size=bs, table=table,
                 seq_lens=_ints(total), prefix=ids[:p].clone(), k_scale=None, v_scale=None,
                 longest_own=max([n - p * bs if n >= p * bs else n for n in total]),
                 q=1.5 * torch.randn(b, hq, d, device=_DEVICE, generator=g),
                 out=torch.zeros(b, hq, d, dtype=dtype, device=_DEVICE))
    state["q"] = state["q"].to(dtype)
    for name in ("kc", "vc"):
        x = torch.empty(shape, dtype=dtype, device=_DEVICE).normal_(generator=g)
        if case["cache"] == "fp8":
            x = (x.float() / 0.02).clamp_(-_FP8_MAX, _FP8_MAX).to(torch.float8_e4m3fn)
            state[name[0] + "_scale"] = torch.tensor([0.02], device=_DEVICE)
        state[name] = x
    return state


def prepare(case, seed):
    g = _rng(seed)
    return {"plan": _prepare_plan, "release": _prepare_release, "mrope": _prepare_mrope,
            "prompt": _prepare_prompt, "decode": _prepare_decode}[case["op"]](case, g)


# ---- the plain forms --------------------------------------------------------------------
def _plain_plan(s):
    bs = s["block_size"]
    context, query = s["context"].long().clamp(min=0), s["query"].long().clamp(min=0)
    table, free = s["table"], s["free"]
    width, tokens = table.shape[1], s["positions"].numel()
    count = s["count"].long()
    end = torch.cumsum(query, 0)
    total = context + query
    held, want = (context + bs - 1) // bs, (total + bs - 1) // bs
    fits = (want <= width) & (end <= tokens)
    need = torch.where(fits, want - held, torch.zeros_like(want))
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= count))
    column = torch.arange(width, device=table.device)[None, :]
    fresh = served[:, None] & (column >= held[:, None]) & (column < want[:, None])
    index = count - 1 - ((upto - need - held)[:, None] + column)
    table.copy_(torch.where(fresh, free[index.clamp(0, free.numel() - 1)], table))
    s["query_start"][1:] = end.clamp(max=tokens).to(torch.int32)
    s["seq_lens"].copy_(torch.where(served, total, context))
    s["count_out"].copy_(count - torch.where(served, need, torch.zeros_like(need)).sum())
    t = torch.arange(tokens, device=table.device)
    row = torch.searchsorted(end, t, right=True)
    live = row < context.numel()
    row = row.clamp(max=context.numel() - 1)
    position = context[row] + t - (end - query)[row]
    block = table[row, (position // bs).clamp(0, width - 1)].long()
    stored = live & served[row] & (block >= 0)
    s["positions"].copy_(torch.where(live, position, torch.full_like(position, -1)))
    s["slots"].copy_(torch.where(stored, block * bs + position % bs, torch.full_like(position, -1)))
    return _plan_outputs(s)


def _plan_outputs(s):
    return [s["table"], s["query_start"], s["seq_lens"], s["positions"], s["slots"], s["count_out"]]


def _plain_release(s):
    bs, table, free = s["block_size"], s["table"], s["free"]
    pool = free.numel()
    held = (s["seq_lens"].long().clamp(min=0) + bs - 1) // bs
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    back = (s["finished"][:, None] & (column >= s["shared"]) & (column < held[:, None])
            & (table >= 0) & (table < pool)).reshape(-1)
    place = s["count"].long() + torch.cumsum(back, 0) - 1
    place = torch.where(back & (place < pool), place, torch.full_like(place, pool))
    larger = torch.cat((free, free.new_zeros(1)))
    larger[place] = table.reshape(-1)
    free.copy_(larger[:pool])
    s["count_out"].copy_((s["count"].long() + back.sum()).clamp(max=pool))
    return [s["free"], s["count_out"]]


def _axis_of(sections, mixed):
    """The axis whose position turns each pair of a head."""
    half = sum(sections)
    if mixed:
        axes = len(sections)
        return [i % axes if i % axes and i < axes * sections[i % axes] else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _turned(x, weight, cos, sin, neox, wide):
    """RMSNorm and rotation of [T, H, D] heads in the type `wide`."""
    x = x.to(wide)
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.to(wide)
    half = cos.shape[-1]
    if neox:
        a, b = n[..., :half], n[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, n[..., 2 * half:]), dim=-1)
    a, b = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    return torch.cat((y, n[..., 2 * half:]), dim=-1)


def _store(whole, x, slots, layout, block_size):
    """x[t] at slots[t]; what has no slot goes to the block behind the cache."""
    last = (whole.shape[0] - 1) * block_size
    slots = torch.where((slots >= 0) & (slots < last), slots, torch.full_like(slots, last)).long()
    if layout == "NHD":
        whole[slots // block_size, slots % block_size] = x
    else:
        whole[slots // block_size, :, slots % block_size] = x


def _stored_as(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x / scale).clamp(-_FP8_MAX, _FP8_MAX).to(dtype)


def _mrope_rows(s, wide):
    """Rotated queries and keys, and which tokens have a position."""
    axis = torch.tensor(_axis_of(s["sections"], s["mixed"]), device=_DEVICE)
    rows, rotary = s["table"].shape
    half = rotary // 2
    valid = ((s["positions"] >= 0) & (s["positions"] < rows)).all(0)
    place = s["positions"].clamp(0, rows - 1)[axis].t()  # [T, half]
    pair = torch.arange(half, device=_DEVICE)[None, :]
    cos = s["table"][place, pair][:, None].to(wide)
    sin = s["table"][place, half + pair][:, None].to(wide)
    return (_turned(s["q"], s["qw"], cos, sin, s["neox"], wide),
            _turned(s["k"], s["kw"], cos, sin, s["neox"], wide), valid)


def _plain_mrope(s):
    q, k, valid = _mrope_rows(s, torch.float32)
    keep = valid[:, None, None]
    s["q_out"].copy_(torch.where(keep, q.to(s["q"].dtype), s["q_out"]))
    s["k_out"].copy_(torch.where(keep, k.to(s["k"].dtype), s["k_out"]))
    if s["kc"] is None:
        return [s["q_out"], s["k_out"]]
    slots = torch.where(valid, s["slots"], torch.full_like(s["slots"], -1))
    _store(s["kc_whole"], _stored_as(k, s["k_scale"], s["kc"].dtype), slots, s["layout"],
           s["block_size"])
    v = s["v"].float() if s["v_scale"] is not None else s["v"]
    _store(s["vc_whole"], _stored_as(v, s["v_scale"], s["vc"].dtype), slots, s["layout"],
           s["block_size"])
    return [s["q_out"], s["k_out"], s["kc"], s["vc"]]


def _causal(q, k, v, out, wide, budget):
    """Causal attention of one sequence, rows in slices whose scores take about `budget` bytes."""
    n, hq, d = q.shape
    hk = k.shape[1]
    group = hq // hk
    kt = k.to(wide).permute(1, 2, 0)  # [Hk, D, N]
    vt = v.to(wide).permute(1, 0, 2)  # [Hk, N, D]
    slice_rows = max(1, min(n, budget // (4 * hq * n)))
    for first in range(0, n, slice_rows):
        last = min(n, first + slice_rows)
        rows = last - first
        qs = q[first:last].to(wide) * (1.0 / math.sqrt(d))
        qs = qs.view(rows, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * rows, d)
        scores = torch.matmul(qs, kt[..., :last]).view(hk, group, rows, last)
        later = torch.arange(last, device=q.device)[None, :] > torch.arange(first, last, device=q.device)[:, None]
        scores.masked_fill_(later, -math.inf)
        scores -= scores.amax(-1, keepdim=True)
        scores.exp_()
        norm = scores.sum(-1, keepdim=True)
        y = torch.matmul(scores.view(hk, group * rows, last), vt[:, :last]).view(hk, group, rows, d)
        y = (y / norm).permute(2, 0, 1, 3).reshape(rows, hq, d)
        out[first:last] = y.to(out.dtype)


def _plain_prompt(s):
    first = 0
    for n in s["lengths"]:
        _causal(s["q"][first:first + n], s["k"][first:first + n], s["v"][first:first + n],
                s["out"][first:first + n], torch.float32, 1 << 30)
        first += n
    return s["out"]


def _pages(cache, ids, layout, scale, wide):
    """Blocks `ids` [..., n] of a cache as [..., n * block_size, Hk, D]."""
    x = cache[ids.clamp(min=0)].to(wide)
    if layout == "HND":
        x = x.transpose(-3, -2)
    if scale is not None:
        x = x * scale.to(wide)
    return x.flatten(-4, -3)


def _weighted(scores, values):
    """Row maximum, sum of exp and the weighted values of one part of the keys."""
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(scores - top)
    return top, e.sum(-1, keepdim=True), torch.matmul(e, values)


def _plain_decode(s):
    b, hq, d = s["q"].shape
    kc, vc, bs, p = s["kc"], s["vc"], s["block_size"], s["prefix"].numel()
    hk = kc.shape[2] if s["layout"] == "NHD" else kc.shape[1]
    q = s["q"].float().view(b, hk, hq // hk, d) * (1.0 / math.sqrt(d))
    lens = s["seq_lens"].long()
    shares = lens >= p * bs
    # each request's own blocks, side by side
    first = torch.where(shares, p, 0)
    n_own = torch.where(shares, lens - p * bs, lens)
    most = _blocks(max(1, s["longest_own"]), bs)
    column = (first[:, None] + torch.arange(most, device=q.device)[None, :])
    ids = torch.gather(s["table"].long(), 1, column.clamp(max=s["table"].shape[1] - 1))
    k = _pages(kc, ids, s["layout"], s["k_scale"], torch.float32)  # [B, N, Hk, D]
    v = _pages(vc, ids, s["layout"], s["v_scale"], torch.float32)
    outside = torch.arange(k.shape[1], device=q.device)[None, :] >= n_own[:, None]
    scores = torch.matmul(q, k.permute(0, 2, 3, 1))
    scores.masked_fill_(outside[:, None, None, :], -math.inf)
    top, norm, y = _weighted(scores, v.permute(0, 2, 1, 3).masked_fill(outside[:, None, :, None], 0))
    del k, v, scores
    if p:
        k = _pages(kc, s["prefix"].long(), s["layout"], s["k_scale"], torch.float32)
        v = _pages(vc, s["prefix"].long(), s["layout"], s["v_scale"], torch.float32)
        rows = q.permute(1, 0, 2, 3).reshape(hk, -1, d)
        top2, norm2, y2 = _weighted(torch.matmul(rows, k.permute(1, 2, 0)), v.permute(1, 0, 2))

        def back(x):
            return x.view(hk, b, hq // hk, -1).permute(1, 0, 2, 3)
        part = shares[:, None, None, None]
        top2 = torch.where(part, back(top2), torch.full_like(top, -1e30))
        both = torch.maximum(top, top2)
        own_weight = torch.exp(top - both)
        weight = torch.where(part, torch.exp(top2 - both), torch.zeros_like(top))
        norm = norm * own_weight + back(norm2) * weight
        y = y * own_weight + back(y2) * weight
    y = torch.where(norm > 0, y / norm.clamp(min=1e-30), torch.zeros_like(y))
    s["out"].copy_(y.reshape(b, hq, d))
    return s["out"]


# ---- this repository's operators --------------------------------------------------------
def _own_plan(s):
    _, serving = _package()
    serving.plan_step_(s["context"], s["query"], s["table"], s["free"], s["count"],
                       s["block_size"], s["query_start"], s["seq_lens"], s["positions"],
                       s["slots"], s["count_out"])
    return _plan_outputs(s)


def _own_release(s):
    _, serving = _package()
    serving.release_blocks_(s["seq_lens"], s["finished"], s["table"], s["free"], s["count"],
                            s["block_size"], s["shared"], s["count_out"])
    return [s["free"], s["count_out"]]


def _own_mrope(s):
    extensions, _ = _package()
    extensions.qk_norm_mrope_cache_(
        s["q"], s["k"], s["v"], s["qw"], s["kw"], s["positions"], s["table"], s["sections"],
        s["kc"], s["vc"], s["slots"], s["k_scale"], s["v_scale"], is_neox=s["neox"],
        interleaved_sections=s["mixed"], kv_cache_layout=s["layout"], query_out=s["q_out"],
        key_out=s["k_out"])
    return [s["q_out"], s["k_out"]] if s["kc"] is None else [s["q_out"], s["k_out"], s["kc"], s["vc"]]


def _own_prompt(s):
    _, serving = _package()
    serving.prompt_attention(s["out"], s["q"], s["k"], s["v"], s["start"])
    return s["out"]


def _own_decode(s):
    _, serving = _package()
    serving.paged_decode_attention(s["out"], s["q"], s["kc"], s["vc"], s["table"], s["seq_lens"],
                                   s["prefix"], s["k_scale"], s["v_scale"],
                                   kv_cache_layout=s["layout"])
    return s["out"]


def run(state):
    if own:
        return {"plan": _own_plan, "release": _own_release, "mrope": _own_mrope,
                "prompt": _own_prompt, "decode": _own_decode}[state["op"]](state)
    return {"plan": _plain_plan, "release": _plain_release, "mrope": _plain_mrope,
            "prompt": _plain_prompt, "decode": _plain_decode}[state["op"]](state)


# ---- the work that a pass cannot do without ---------------------------------------------
def work(case):
    if case["op"] == "plan":
        context, query = _lengths(case)
        bs = case["block_size"]
        fresh = sum(_blocks(c + q, bs) - _blocks(c, bs) for c, q in zip(context, query))
        old = sum(1 for c, q in zip(context, query) if q and c % bs)  # half-full last blocks
        tokens = sum(query) + case["padding"]
        n = case["requests"]
        # two lengths in, a start and a length out, ids from the stack into the table, and per
        # token a position and a slot
        return {"bytes": 8 * n + 8 * n + 4 + 8 * fresh + 4 * old + 12 * tokens + 8,
                "flops": 4 * tokens + 8 * n}
    if case["op"] == "release":
        lengths, _ = _lengths(case)
        held = sum(max(0, _blocks(c, case["block_size"]) - case["shared"]) for c in lengths)
        return {"bytes": int(5 * case["requests"] + 8 * 0.35 * held + 8),
                "flops": int(case["requests"] * 4 + 0.35 * held)}
    if case["op"] == "mrope":
        t, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        e = _BYTES[case["dtype"]]
        moved = 2 * t * (hq + hk) * d * e + 24 * t + t * case["rotary"] * 4
        if case["cache"] != "none":
            c = 1 if case["cache"] == "fp8" else e
            moved += t * hk * d * e + 2 * t * hk * d * c + 4 * t
        return {"bytes": moved, "flops": 8 * t * (hq + hk) * d}
    if case["op"] == "prompt":
        lengths, _ = _lengths(case)
        hq, hk, d, e = case["hq"], case["hk"], case["d"], _BYTES[case["dtype"]]
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        return {"bytes": sum(lengths) * d * e * (2 * hq + 2 * hk) + 4 * (len(lengths) + 1),
                "flops": 4 * pairs * hq * d}
    total, _ = _lengths(case)
    hq, hk, d, p = case["hq"], case["hk"], case["d"], case["prefix"] * case["block_size"]
    e = _BYTES["fp8"] if case["cache"] == "fp8" else _BYTES[case["dtype"]]
    own_tokens = sum(n - p if n >= p else n for n in total)
    blocks = sum(_blocks(n - p if n >= p else n, case["block_size"]) for n in total) + case["prefix"]
    return {"bytes": (own_tokens + p) * hk * d * 2 * e
            + 2 * case["batch"] * hq * d * _BYTES[case["dtype"]] + 4 * blocks + 4 * case["batch"],
            "flops": 4 * sum(total) * hq * d}


# ---- the definitions in 64 bits ---------------------------------------------------------
def _exact_plan(case, seed):
    s = prepare(case, seed)
    context, query = s["context"].tolist(), s["query"].tolist()
    table, free, left = s["table"].tolist(), s["free"].tolist(), int(s["count"])
    bs, width, tokens = s["block_size"], s["table"].shape[1], s["positions"].numel()
    start, lens, positions, slots = [0], [], [-1] * tokens, [-1] * tokens
    full = False
    for r, (c, q) in enumerate(zip(context, query)):
        held, want = -(-c // bs), -(-(c + q) // bs)
        ok = want <= width and start[-1] + q <= tokens
        if ok and want > held:
            full = full or want - held > left
            ok = not full
            if ok:
                for b in range(held, want):
                    left -= 1
                    table[r][b] = free[left]
        for i in range(q):
            t = start[-1] + i
            if t < tokens:
                positions[t] = c + i
                block = table[r][(c + i) // bs] if ok else -1
                slots[t] = block * bs + (c + i) % bs if block >= 0 else -1
        start.append(start[-1] + q)
        lens.append(c + q if ok else c)
    return [_ints(table), _ints(start), _ints(lens), _ints(positions, torch.int64), _ints(slots),
            _ints([left])]


def _exact_release(case, seed):
    s = prepare(case, seed)
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["count"])
    for row, n, done in zip(table, s["seq_lens"].tolist(), s["finished"].tolist()):
        if done:
            for block in row[s["shared"]:-(-n // s["block_size"])]:
                if 0 <= block < len(free) and count < len(free):
                    free[count] = block
                    count += 1
    return [_ints(free), _ints([count])]


def _exact_mrope(case, seed):
    s = prepare(case, seed)
    rows, rotary = s["table"].shape
    half, sections = rotary // 2, s["sections"]
    table = s["table"].double()
    valid = ((s["positions"] >= 0) & (s["positions"] < rows)).all(0)
    place = s["positions"].clamp(0, rows - 1)
    angle = torch.empty(place.shape[1], rotary, dtype=torch.float64, device=_DEVICE)
    for i in range(half):
        if s["mixed"]:
            axis = i % 3 if i % 3 > 0 and i < 3 * sections[i % 3] else 0
        else:
            axis = 0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2
        angle[:, i] = table[place[axis], i]
        angle[:, half + i] = table[place[axis], half + i]
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = torch.zeros(x.shape, dtype=torch.float64, device=_DEVICE)
        for h in range(x.shape[1]):
            n = x[:, h].double()
            n = n / (n.pow(2).sum(-1, keepdim=True) / n.shape[-1] + _EPS).sqrt() * w.double()
            z = torch.complex(n[:, :half], n[:, half:rotary]) if s["neox"] else \
                torch.complex(n[:, 0:rotary:2], n[:, 1:rotary:2])
            z = z * torch.complex(angle[:, :half], angle[:, half:])
            if s["neox"]:
                n = torch.cat((z.real, z.imag, n[:, rotary:]), dim=-1)
            else:
                n = torch.cat((torch.view_as_real(z).flatten(-2), n[:, rotary:]), dim=-1)
            y[:, h] = torch.where(valid[:, None], n, torch.zeros_like(n))
        out.append(y)
    if s["kc"] is None:
        return out
    capacity = s["kc"].shape[0] * s["block_size"]
    hk, d = s["k"].shape[1:]
    place = torch.arange(capacity, device=_DEVICE)
    source = torch.full((capacity + 1,), -1, dtype=torch.long, device=_DEVICE)
    live = valid & (s["slots"] >= 0) & (s["slots"] < capacity)
    source[s["slots"][live].long()] = torch.arange(valid.numel(), device=_DEVICE)[live]
    source = source[place]
    for x, scale in ((out[1], s["k_scale"]), (s["v"].double(), s["v_scale"])):
        flat = torch.where((source >= 0)[:, None, None], x[source.clamp(min=0)],
                           torch.zeros(1, 1, 1, dtype=torch.float64, device=_DEVICE))
        if scale is not None:
            flat = (flat / scale.double()).clamp(-_FP8_MAX, _FP8_MAX)
        flat = flat.view(-1, s["block_size"], hk, d)
        out.append(flat if s["layout"] == "NHD" else flat.transpose(1, 2).contiguous())
    return out


def _exact_prompt(case, seed):
    s = prepare(case, seed)
    t, hq, d = s["q"].shape
    hk = s["k"].shape[1]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=_DEVICE)
    start = s["start"].tolist()
    for a, b in zip(start[:-1], start[1:]):
        n = b - a
        rows = max(1, min(n, (1 << 28) // max(n, 1)))
        for h in range(hq):
            q = s["q"][a:b, h].double() / d ** 0.5
            k, v = s["k"][a:b, h * hk // hq].double(), s["v"][a:b, h * hk // hq].double()
            for i in range(0, n, rows):
                j = min(n, i + rows)
                w = q[i:j] @ k[:j].t()
                w = w.masked_fill(torch.ones_like(w, dtype=torch.bool).triu(i + 1), -math.inf)
                out[a + i:a + j, h] = torch.softmax(w, -1) @ v[:j]
    return out


def _exact_decode(case, seed):
    s = prepare(case, seed)
    b, hq, d = s["q"].shape
    kc, vc, bs = s["kc"], s["vc"], s["block_size"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=_DEVICE)
    prefix = s["prefix"].long()
    shared = prefix.numel() * bs

    def tokens(cache, ids, scale):
        x = cache[ids].double() if scale is None else cache[ids].double() * scale.double()
        x = x if s["layout"] == "NHD" else x.transpose(1, 2)
        return x.reshape(-1, x.shape[2], d).transpose(0, 1)  # [Hk, N, D]

    pk, pv = tokens(kc, prefix, s["k_scale"]), tokens(vc, prefix, s["v_scale"])
    hk = pk.shape[0]
    for r, n in enumerate(s["seq_lens"].tolist()):
        if n == 0:
            continue
        skip = prefix.numel() if n >= shared else 0
        ids = s["table"][r, skip:-(-n // bs)].long()
        k, v = tokens(kc, ids, s["k_scale"]), tokens(vc, ids, s["v_scale"])
        own_n = n - skip * bs
        k, v = k[:, :own_n], v[:, :own_n]
        if skip:
            k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
        q = s["q"][r].double().view(hk, hq // hk, d) / d ** 0.5
        out[r] = (torch.softmax(q @ k.transpose(1, 2), -1) @ v).reshape(hq, d)
    return out


def exact(case, seed):
    return {"plan": _exact_plan, "release": _exact_release, "mrope": _exact_mrope,
            "prompt": _exact_prompt, "decode": _exact_decode}[case["op"]](case, seed)
