"""Shapes between and beyond those of the other serving tests: every kind of block
size, rows far apart, several calls at once."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import extensions, serving
from test_gpu_attention import RAGGED, Decode, Prompt, assert_within, ints

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("block_size", [2, 4, 8, 24, 40, 64, 96, 128, 192, 320])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache, layout", [("same", "NHD"), ("fp8", "HND"), ("same", "HND"), ("u8", "NHD")])
def test_block_sizes(block_size, d, cache, layout):
    for prefix in (0, max(1, 400 // block_size)):
        p = prefix * block_size
        Decode([p + n for n in RAGGED] + [p, max(p - 1, 0)], prefix, d=d, cache=cache, layout=layout,
               block_size=block_size, seed=block_size).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_request_of_every_small_length(d):
    Decode(list(range(70)), d=d, seed=1).check()
    Decode([32 + n for n in range(70)], 2, d=d, cache="fp8", seed=2).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompts_of_every_small_length(d):
    Prompt(list(range(40)) + [39 - n for n in range(40)], d=d, padding=1, seed=3).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_rows_past_32_bits(d):
    """Rows 2^20 elements apart: the last tokens lie past 2^32."""
    t, hq, hk = 4500, 2, 1
    whole = torch.empty(t, 1 << 20, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    views, at = [], 0
    for h in (hq, hk, hk, hq):
        view = whole[:, at:at + h * d].view(t, h, d)
        view.copy_(torch.randn(t, h, d, device=DEV, generator=g))
        views.append(view)
        at += 4096
    q, k, v, out = views
    starts = [0, 100, 4400, t]
    want, bound = ref.prompt(q, k, v, starts)
    serving.prompt_attention(out, q, k, v, ints(starts))
    assert_within(out, want, bound)


def test_rotated_rows_and_slots_past_32_bits():
    t, d = 4500, 128
    whole = torch.empty(t, 1 << 20, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (whole[:, at:at + 256].view(t, 2, d) for at in (0, 4096, 8192))
    for x in (q, k, v):
        x.copy_(torch.randn(t, 2, d, device=DEV, generator=g))
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    places = torch.randint(0, 500, (3, t), device=DEV, generator=g)
    table = torch.randn(500, d, device=DEV, generator=g)
    kc, vc = (torch.zeros(300, 1 << 24, dtype=torch.bfloat16, device=DEV)[:, :16 * 2 * d].unflatten(
        1, (16, 2, d)) for _ in "kv")
    slots = torch.randperm(300 * 16, device=DEV, generator=g)[:t].to(torch.int32)
    near = [x.clone() for x in (q, k)]
    small = [torch.zeros(300, 16, 2, d, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
    extensions.qk_norm_mrope_cache_(*near, v.clone(), w, w, places, table, [16, 24, 24], *small, slots)
    extensions.qk_norm_mrope_cache_(q, k, v, w, w, places, table, [16, 24, 24], kc, vc, slots)
    for far, close in zip((q, k, kc, vc), (*near, *small)):
        assert torch.equal(far, close)


@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_calls_on_several_streams_at_once(cache):
    cases = [Decode([16 * 20 + n for n in RAGGED], 20, cache=cache, seed=s) for s in range(4)]
    prompts = [Prompt([300, 70], d=d, seed=d) for d in (64, 128)]
    want = [c.run().clone() for c in cases + prompts]
    lens = [ints(c.lens) for c in cases]
    starts = [ints(c.starts) for c in prompts]
    streams = [torch.cuda.Stream() for _ in want]
    for c in cases + prompts:
        c.out.fill_(3.0)
    torch.cuda.synchronize()
    for _ in range(30):
        for c, n, stream in zip(cases, lens, streams):
            with torch.cuda.stream(stream):
                serving.paged_decode_attention(c.out, c.q, c.kc, c.vc, c.table, n, c.prefix, *c.scales)
        for c, n, stream in zip(prompts, starts, streams[4:]):
            with torch.cuda.stream(stream):
                serving.prompt_attention(c.out, c.q, c.k, c.v, n)
    torch.cuda.synchronize()
    for c, w in zip(cases + prompts, want):
        assert torch.equal(c.out, w)


def test_one_block_many_times():
    """A table and a prefix may name a block as often as they like."""
    c = Decode([16 * 6 + 40, 16 * 6 + 3], 6, seed=6)
    c.prefix[:] = c.prefix[0]
    c.table[0, 6:9] = c.prefix[0]
    c.check()
