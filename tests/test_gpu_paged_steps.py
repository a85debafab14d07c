"""Batches that live through several requests (engine.PagedSteps and
engine.Qwen3Attention): what a decode step returns must be the 64-bit attention
over the keys and values that the request's own tokens had, kept beside the cache
as they were computed, within the bounds of tests/serving_reference.py."""
import random

import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm.engine import (PagedSteps, Qwen3Attention, Qwen3AttentionPrologue,
                                  Qwen3AttentionShape, rope_cos_sin_cache)

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = Qwen3AttentionShape(hidden=512, query_heads=8, key_heads=2, max_positions=4096)
BLOCKS = 60


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def bools(values):
    return torch.tensor(values, dtype=torch.bool, device=DEV)


class Layer:
    """A layer with a cache, and each request's keys and values in its own order."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        caches = [torch.zeros(BLOCKS, 16, SHAPE.key_heads, SHAPE.head_dim, device=DEV,
                              dtype=torch.bfloat16) for _ in "kv"]
        self.attention = Qwen3Attention(Qwen3AttentionPrologue(SHAPE, DEV, generator=self.g),
                                        *caches, rope_cos_sin_cache(SHAPE, DEV))
        self.seen = {}  # of a request: keys, values

    def rows(self, n):
        return [torch.randn(n, SHAPE.hidden, device=DEV, generator=self.g).to(torch.bfloat16)
                for _ in "hr"]

    def qkv(self, n):
        return torch.empty(n, SHAPE.qkv_width, device=DEV, dtype=torch.bfloat16)

    def remember(self, name, k, v):
        old = self.seen.get(name)
        self.seen[name] = (k.clone(), v.clone()) if old is None else \
            (torch.cat((old[0], k)), torch.cat((old[1], v)))

    def prompt(self, steps, lens, names):
        """A step of whole prompts, named row by row."""
        steps.plan(ints(lens))
        n = sum(lens)
        qkv = self.qkv(n)
        out = self.attention.prompts(*self.rows(n), steps, qkv=qkv)
        q, k, v = self.attention.prologue.split(qkv)
        starts = steps.query_start.tolist()
        want, bound = ref.prompt(q, k, v, starts)
        assert ((out.double() - want).abs() <= bound).all()
        for name, a, b in zip(names, starts[:-1], starts[1:]):
            self.remember(name, k[a:b], v[a:b])

    def decode(self, steps, names):
        """A step of one token for every row whose name is not None."""
        steps.plan(ints([int(name is not None) for name in names]))
        qkv = self.qkv(len(names))
        out = self.attention.decode(*self.rows(len(names)), steps, qkv=qkv)
        q, k, v = self.attention.prologue.split(qkv)
        for r, name in enumerate(names):
            if name is None:
                assert (out[r] == 0).all()
                continue
            self.remember(name, k[r:r + 1], v[r:r + 1])
            keys, values = (x.double() for x in self.seen[name])
            for h in range(SHAPE.key_heads):
                heads = slice(4 * h, 4 * h + 4)
                want, bound = ref.attention_row_block(
                    q[r, heads].double(), keys[:, h], values[:, h], SHAPE.head_dim ** -0.5,
                    torch.bfloat16, torch.bfloat16)
                assert ((out[r, heads].double() - want).abs() <= bound).all(), (r, name)


def begin_behind(layer, prefix_name, *names):
    for name in names:
        layer.seen[name] = layer.seen[prefix_name]


def test_requests_behind_a_prefix_end_and_make_room():
    layer = Layer(1)
    steps = PagedSteps(3, BLOCKS, 20, 3, DEV, prefix_blocks=2)
    layer.prompt(steps.prefix_writer(), [32], ["prefix"])
    pool = int(steps.free_count)
    assert pool == BLOCKS - 2
    begin_behind(layer, "prefix", "a", "b", "c", "d", "e", "f", "g")
    for _ in range(35):  # past two blocks of their own
        layer.decode(steps, ["a", "b", "c"])
    assert int(steps.free_count) == pool - 9
    steps.release(bools([False, True, False]))
    assert int(steps.free_count) == pool - 6
    assert steps.context_lens.tolist() == [67, 32, 67]
    for _ in range(40):  # a second request in the row that was given back
        layer.decode(steps, ["a", "d", "c"])
    steps.release(bools([True, True, True]))
    assert int(steps.free_count) == pool
    assert steps.context_lens.tolist() == [32] * 3
    for _ in range(3):
        layer.decode(steps, ["e", "f", "g"])


def test_a_batch_without_the_prefix_over_the_same_pool():
    layer = Layer(2)
    sharing = PagedSteps(2, BLOCKS, 20, 2, DEV, prefix_blocks=3)
    alone = PagedSteps(2, BLOCKS, 20, 90, DEV, pool=sharing)
    layer.prompt(sharing.prefix_writer(), [48], ["prefix"])
    begin_behind(layer, "prefix", "a", "b", "c")
    for names in (("p", "q"), ("r", "s")):
        layer.prompt(alone, [70, 20], names)
        for _ in range(20):
            layer.decode(sharing, ["a", "b"])
            layer.decode(alone, list(names))
        alone.release(bools([True, True]))
    sharing.release(bools([True, False]))
    for _ in range(5):
        layer.decode(sharing, ["c", "b"])
    sharing.release(bools([True, True]))
    assert int(sharing.free_count) == BLOCKS - 3


@pytest.mark.parametrize("prefix", [0, 2])
def test_idle_rows_keep_every_request_with_its_own_tokens(prefix):
    layer = Layer(3)
    steps = PagedSteps(4, BLOCKS, 20, 90, DEV, prefix_blocks=prefix)
    if prefix:
        layer.prompt(steps.prefix_writer(), [32], ["prefix"])
        begin_behind(layer, "prefix", "a", "b", "c", "d", "e")
    else:
        layer.prompt(steps, [40, 3, 17, 30], ["a", "b", "c", "d"])
    pool = int(steps.free_count)
    layer.decode(steps, ["a", "b", "c", "d"])
    steps.release(bools([False, True, False, False]))
    for _ in range(20):  # a middle row without a request takes no block
        layer.decode(steps, ["a", None, "c", "d"])
    assert steps.context_lens[1] == prefix * 16
    layer.decode(steps, [None, "e", None, None])
    layer.decode(steps, [None, None, None, None])
    for _ in range(17):
        layer.decode(steps, ["a", "e", None, "d"])
    steps.release(bools([True, True, True, True]))
    assert int(steps.free_count) == (pool if prefix else BLOCKS)


def test_a_request_without_room_comes_out_as_zeros():
    layer = Layer(4)
    steps = PagedSteps(3, BLOCKS, 20, 3, DEV)
    steps.free_count.fill_(2)
    layer.decode(steps, ["a", "b", None])
    steps.plan(ints([1, 0, 1]))
    out = layer.attention.decode(*layer.rows(3), steps)
    assert steps.unserved.tolist() == [False, False, True]
    assert (out[1:] == 0).all() and out[0].abs().max() > 0


def test_a_captured_step_with_rows_that_come_and_go():
    layer = Layer(5)
    steps = PagedSteps(3, BLOCKS, 20, 3, DEV)
    query = ints([1, 1, 1])
    hidden, residual = layer.rows(3)
    qkv = layer.qkv(3)
    out = torch.empty(3, 8, 128, device=DEV, dtype=torch.bfloat16)

    def step():
        steps.plan(query)
        layer.attention.decode(hidden, residual, steps, qkv=qkv, out=out)

    step()
    torch.cuda.synchronize()
    q, k, v = layer.attention.prologue.split(qkv)
    for r in range(3):
        layer.remember(r, k[r:r + 1], v[r:r + 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(30):
        there = [int((i + r) % 3 > 0) for r in range(3)]
        query.copy_(ints(there))
        for buffer, values in zip((hidden, residual), layer.rows(3)):
            buffer.copy_(values)
        graph.replay()
        for r in range(3):
            if not there[r]:
                assert (out[r] == 0).all()
                continue
            layer.remember(r, k[r:r + 1], v[r:r + 1])
            keys, values = (x.double() for x in layer.seen[r])
            for h in range(2):
                want, bound = ref.attention_row_block(
                    q[r, 4 * h:4 * h + 4].double(), keys[:, h], values[:, h], 128 ** -0.5,
                    torch.bfloat16, torch.bfloat16)
                assert ((out[r, 4 * h:4 * h + 4].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("prefix", [0, 3])
@pytest.mark.parametrize("seed", range(4))
def test_requests_that_come_wait_and_go_at_random(seed, prefix):
    """Rows take part in a step or not, run out of blocks, end and begin again; the
    pool is too small for all. Every output against the request's own tokens."""
    rng = random.Random(seed)
    layer = Layer(10 + seed)
    rows = 6
    steps = PagedSteps(rows, BLOCKS, 20, rows, DEV, prefix_blocks=prefix)
    if prefix:
        layer.prompt(steps.prefix_writer(), [16 * prefix], ["prefix"])
    kept = steps.free_blocks[:rng.randint(5, 7)].clone()
    steps.free_count.fill_(len(kept))  # the others are somebody else's
    born = 0
    names = [None] * rows
    waited = 0
    for _ in range(120):
        for r in range(rows):
            if names[r] is None and rng.random() < 0.3:
                names[r] = born
                born += 1
                if prefix:
                    begin_behind(layer, "prefix", names[r])
        takes = [name is not None and rng.random() < 0.8 for name in names]
        before = steps.context_lens.tolist()
        steps.plan(ints([int(t) for t in takes]))
        qkv = layer.qkv(rows)
        out = layer.attention.decode(*layer.rows(rows), steps, qkv=qkv)
        q, k, v = layer.attention.prologue.split(qkv)
        unserved, after = steps.unserved.tolist(), steps.context_lens.tolist()
        waited += sum(unserved)
        for r in range(rows):
            served = takes[r] and not unserved[r]
            assert after[r] == before[r] + served and not (unserved[r] and not takes[r])
            if not served:
                assert (out[r] == 0).all()
                continue
            layer.remember(names[r], k[r:r + 1], v[r:r + 1])
            keys, values = (x.double() for x in layer.seen[names[r]])
            assert len(keys) == after[r]
            for h in range(SHAPE.key_heads):
                heads = slice(4 * h, 4 * h + 4)
                want, bound = ref.attention_row_block(
                    q[r, heads].double(), keys[:, h], values[:, h], SHAPE.head_dim ** -0.5,
                    torch.bfloat16, torch.bfloat16)
                assert ((out[r, heads].double() - want).abs() <= bound).all()
        done = [name is not None and rng.random() < 0.03 for name in names]
        if any(done):
            steps.release(bools(done))
            names = [None if d else name for d, name in zip(done, names)]
    assert waited > 0 and born > rows
    steps.release(bools([True] * rows))
    assert int(steps.free_count) == len(kept)
    assert sorted(steps.free_blocks[:len(kept)].tolist()) == sorted(kept.tolist())
