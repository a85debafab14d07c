"""The serving operators as a serving loop uses them (sm120_rmsnorm.engine):
plan, prologue with the KV store, attention of prompts, then decode steps. What
the cache holds must be the layer's own keys and values, and every attention
output the 64-bit attention over them, within the bounds of
tests/serving_reference.py."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm.engine import (PagedSteps, Qwen3Attention, Qwen3AttentionPrologue,
                                  Qwen3AttentionShape, rope_cos_sin_cache)

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = Qwen3AttentionShape(hidden=512, query_heads=8, key_heads=2, max_positions=4096)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def layer(layout="NHD", fp8=False, blocks=300, block_size=16, seed=0, shape=SHAPE):
    g = torch.Generator(device=DEV).manual_seed(seed)
    prologue = Qwen3AttentionPrologue(shape, DEV, generator=g)
    size = (blocks, block_size, shape.key_heads, shape.head_dim) if layout == "NHD" else \
        (blocks, shape.key_heads, block_size, shape.head_dim)
    caches = [torch.zeros(size, device=DEV).to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
              for _ in "kv"]
    scales = [torch.tensor([s], device=DEV) if fp8 else None for s in (0.02, 0.03)]
    return Qwen3Attention(prologue, *caches, rope_cos_sin_cache(shape, DEV), *scales, layout), g


def hidden_states(tokens, g, shape=SHAPE):
    return [torch.randn(tokens, shape.hidden, device=DEV, generator=g).to(torch.bfloat16) for _ in "hr"]


def check_decode(attention, steps, q, out, lens):
    want, bound = ref.decode(q, attention.key_cache, attention.value_cache, steps.block_table, lens,
                             steps.prefix, attention.kv_cache_layout, attention.k_scale,
                             attention.v_scale)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("layout, fp8, axes", [("NHD", False, 1), ("HND", True, 1), ("NHD", True, 3)])
def test_prompts_then_decode_steps(layout, fp8, axes):
    attention, g = layer(layout, fp8)
    lens = [5, 130, 33, 1, 64]
    total = sum(lens)
    steps = PagedSteps(5, 300, 40, total + 6, DEV)
    steps.plan(ints(lens))
    assert steps.query_start.tolist() == [0, 5, 135, 168, 169, 233]
    hidden, residual = hidden_states(total + 6, g)
    qkv = torch.empty(total + 6, SHAPE.qkv_width, device=DEV, dtype=torch.bfloat16)
    positions = steps.positions.clone()
    if axes == 3:  # a picture in the second prompt
        positions = torch.stack([positions] * 3)
        positions[1, 20:80] += torch.arange(60, device=DEV) // 10
        positions[2, 20:80] += torch.arange(60, device=DEV) % 10
    out = attention.prompts(hidden, residual, steps, None if axes == 1 else positions, qkv)
    q, k, v = attention.prologue.split(qkv)
    want, bound = ref.prompt(q, k, v, steps.query_start.tolist())
    live = ~want.isnan()
    assert ((out.double() - want).abs() <= bound)[live].all()
    assert (out[total:] == 0).all()
    # the cache holds the prompts' keys, in the order of the tables
    for r, n in enumerate(lens):
        ids = steps.block_table[r].tolist()[:-(-n // 16)]
        stored, _ = ref.cache_tokens(attention.key_cache, ids, layout, attention.k_scale)
        mine = k[steps.query_start[r]:steps.query_start[r] + n].double()
        tol = mine.abs() * (0.07 if fp8 else 0) + (0.02 * 2.0 ** -9 if fp8 else 0)
        assert ((stored[:n] - mine).abs() <= tol).all()
    for step in range(20):
        steps.plan(ints([1] * 5))
        lens = [n + 1 for n in lens]
        assert steps.context_lens.tolist() == lens
        hidden, residual = hidden_states(5, g)
        qkv = torch.empty(5, SHAPE.qkv_width, device=DEV, dtype=torch.bfloat16)
        place = None if axes == 1 else steps.positions[:5].expand(3, -1)
        out = attention.decode(hidden, residual, steps, place, qkv)
        check_decode(attention, steps, attention.prologue.split(qkv)[0], out, lens)
    free = int(steps.free_count)
    steps.release(torch.tensor([True, False, True, False, False], device=DEV))
    assert int(steps.free_count) == free + -(-lens[0] // 16) + -(-lens[2] // 16)
    assert steps.context_lens.tolist() == [0, lens[1], 0, lens[3], lens[4]]


def test_decode_of_a_prompt_is_prompt_attention():
    """The same tokens as one prompt and one after the other: the two attentions
    read the same keys, so they agree within both bounds."""
    attention, g = layer(blocks=40)
    n = 70
    hidden, residual = hidden_states(n, g)
    whole = PagedSteps(1, 40, 10, n, DEV)
    whole.plan(ints([n]))
    qkv = torch.empty(n, SHAPE.qkv_width, device=DEV, dtype=torch.bfloat16)
    out = attention.prompts(hidden.clone(), residual.clone(), whole, qkv=qkv)
    q, k, v = attention.prologue.split(qkv)
    _, bound = ref.prompt(q, k, v, [0, n])
    for t in (0, 1, 15, 16, 40, 69):
        one = torch.zeros(1, *q.shape[1:], dtype=q.dtype, device=DEV)
        from sm120_rmsnorm import serving
        serving.paged_decode_attention(one, q[t:t + 1].contiguous(), attention.key_cache,
                                       attention.value_cache, whole.block_table, ints([t + 1]))
        assert ((one[0].double() - out[t].double()).abs() <= 2 * bound[t]).all()


@pytest.mark.parametrize("prefix", [0, 9])
def test_a_captured_decode_step(prefix):
    """Plan, prologue and attention in one graph, replayed with lengths that grow
    on the GPU; a second graph of another batch runs in between."""
    runs = []
    for seed, batch in ((1, 6), (2, 3)):
        attention, g = layer(seed=seed)
        steps = PagedSteps(batch, 300, 40, batch, DEV, prefix_blocks=prefix)
        if prefix:  # filled as one prompt would have
            for cache in (attention.key_cache, attention.value_cache):
                cache[steps.prefix.long()] = torch.randn(
                    prefix, 16, 2, 128, device=DEV, generator=g).to(torch.bfloat16)
            steps.context_lens.fill_(prefix * 16)
        hidden, residual = hidden_states(batch, g)
        out = torch.empty(batch, 8, 128, device=DEV, dtype=torch.bfloat16)
        qkv = torch.empty(batch, SHAPE.qkv_width, device=DEV, dtype=torch.bfloat16)
        one = ints([1] * batch)

        def step(steps=steps, attention=attention, hidden=hidden, residual=residual, out=out,
                 qkv=qkv, one=one):
            steps.plan(one)
            attention.decode(hidden, residual, steps, qkv=qkv, out=out)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, attention, steps, hidden, residual, out, qkv, batch, g, one))  # all kept alive
    for k in range(40):
        for graph, attention, steps, hidden, residual, out, qkv, batch, g, _ in runs:
            for buffer in (hidden, residual):
                buffer.copy_(torch.randn(batch, SHAPE.hidden, device=DEV, generator=g))
            graph.replay()
        if k % 13 == 0:
            for graph, attention, steps, hidden, residual, out, qkv, batch, g, _ in runs:
                lens = steps.context_lens.tolist()
                assert lens == [prefix * 16 + 2 + k] * batch
                check_decode(attention, steps, attention.prologue.split(qkv)[0], out, lens)
