"""plan_step_ and release_blocks_ against a plain walk over the requests
(tests/serving_reference.py); whole numbers, so everything must be equal."""
import copy
import random

import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


class Step:
    """A step's inputs, with blocks handed out at random."""

    def __init__(self, context, query, block_size=16, width=None, spare=None, padding=0, seed=0,
                 tokens=None):
        r = random.Random(seed)
        self.context, self.query, self.bs = context, query, block_size
        held = [-(-max(c, 0) // block_size) for c in context]
        need = [-(-(max(c, 0) + max(q, 0)) // block_size) - h
                for c, q, h in zip(context, query, held)]
        self.width = width if width is not None else max(h + n for h, n in zip(held, need)) + 2
        spare = sum(need) + 3 if spare is None else spare
        pool = sum(held) + spare
        ids = r.sample(range(pool), pool)
        self.table = [[-1] * self.width for _ in context]
        for row, h in zip(self.table, held):
            for b in range(h):
                id_ = ids.pop()
                if b < self.width:
                    row[b] = id_
        self.count = len(ids)
        self.free = ids + [-7] * (pool - len(ids))
        self.tokens = sum(max(q, 0) for q in query) + padding if tokens is None else tokens

    def device(self, stride=None):
        stride = stride or self.width
        store = torch.full((len(self.context), stride), -5, dtype=torch.int32, device=DEV)
        table = store[:, :self.width]
        if self.context:
            table.copy_(ints(self.table))
        n = len(self.context)
        return dict(context_lens=ints(self.context), query_lens=ints(self.query), block_table=table,
                    free_blocks=ints(self.free), free_count=ints([self.count]),
                    block_size=self.bs, query_start=ints([-9] * (n + 1)), seq_lens=ints([-9] * n),
                    positions=ints([-9] * self.tokens, torch.int64),
                    slot_mapping=ints([-9] * self.tokens)), store

    def check(self, in_place=False, stride=None):
        args, store = self.device(stride)
        table = copy.deepcopy(self.table)
        starts, lens, positions, slots, left = ref.plan(
            self.context, self.query, table, self.free, self.count, self.bs, self.tokens)
        if in_place:
            args["seq_lens"] = args["context_lens"]
            after = args["free_count"]
        else:
            args["free_count_out"] = after = ints([-9])
        serving.plan_step_(**args)
        assert args["query_start"].tolist() == starts
        assert args["seq_lens"].tolist() == lens
        assert args["positions"].tolist() == positions
        assert args["slot_mapping"].tolist() == slots
        assert args["block_table"].tolist() == table
        assert after.tolist() == [left]
        if not in_place:
            assert args["free_count"].tolist() == [self.count]
            assert args["context_lens"].tolist() == self.context
        assert (store[:, self.width:] == -5).all()
        assert args["free_blocks"].tolist() == self.free


def lengths(n, top, seed, low=0):
    r = random.Random(seed)
    return [r.randint(low, top) for _ in range(n)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests", [1, 2, 31, 33, 255, 1023, 1024, 1025, 2500])
def test_decode_steps(requests, in_place):
    Step(lengths(requests, 200, requests), [1] * requests, seed=1).check(in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests, top", [(1, 1), (1, 4097), (1, 9000), (3, 5000), (70, 700),
                                           (1100, 30), (5, 3)])
@pytest.mark.parametrize("block_size", [1, 16, 48])
def test_prefill_steps(requests, top, block_size, in_place):
    Step(lengths(requests, 300, 3), lengths(requests, top, 4), block_size, padding=7, seed=2).check(
        in_place)


@pytest.mark.parametrize("requests, top", [(40, 60), (1300, 9), (20, 900)])
@pytest.mark.parametrize("spare", [0, 1, 37, 200])
def test_too_few_free_blocks(requests, top, spare):
    Step(lengths(requests, 100, 5), lengths(requests, top, 6), spare=spare, seed=3).check()


def test_tables_too_narrow_and_tokens_past_the_buffer():
    Step([0, 100, 20, 0], [64, 30, 5, 200], width=8, seed=4).check()
    step = Step([0, 10, 20, 30], [40, 50, 60, 70], seed=5, tokens=120)
    step.check()
    Step([0, 10], [3, 5], seed=6, tokens=0).check()


def test_zero_and_negative_lengths_and_no_requests():
    Step([0, -5, 7, 0, 16], [0, 3, -2, 1, 0], seed=7, padding=5).check()
    Step([], [], seed=8, width=4, tokens=9, spare=3).check()
    Step([], [], seed=8, width=4, tokens=5000, spare=0).check(in_place=True)


def test_rows_of_a_wider_table_and_empty_table():
    Step(lengths(17, 90, 8), lengths(17, 40, 9), seed=9).check(stride=33)
    Step([0, 0], [3, 0], width=0, seed=10, spare=4).check()


def test_entries_outside_the_pool_give_no_slots():
    step = Step([20, 20, 20], [1, 1, 1], seed=11)
    step.table[0][1], step.table[1][1] = -1, 10 ** 6
    step.check()


def test_captured_decode_steps_replay_with_updates_in_place():
    step = Step(lengths(9, 50, 12), [1] * 9, spare=200, seed=12, padding=3)
    step.width += 20
    step.table = [row + [-1] * 20 for row in step.table]
    args, _ = step.device()
    args["seq_lens"] = args["context_lens"]
    serving.plan_step_(**args)  # loads the kernel
    start = {k: v.clone() for k, v in step.device()[0].items() if torch.is_tensor(v)}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.plan_step_(**args)
    for k, v in start.items():
        if k != "seq_lens":
            args[k].copy_(v)
    context, table, count = list(step.context), copy.deepcopy(step.table), step.count
    for _ in range(70):
        graph.replay()
        _, context, positions, slots, count = ref.plan(context, step.query, table, step.free, count,
                                                       step.bs, step.tokens)
        assert args["context_lens"].tolist() == context
        assert args["slot_mapping"].tolist() == slots
        assert args["positions"].tolist() == positions
        assert args["free_count"].tolist() == [count]
    assert args["block_table"].tolist() == table


# ---- blocks given back --------------------------------------------------------------------
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests, width, shared", [(1, 5, 0), (7, 40, 2), (32, 33, 0), (33, 9, 1),
                                                     (1000, 70, 3), (1025, 6, 0), (2100, 40, 0)])
def test_release(requests, width, shared, in_place):
    r = random.Random(requests)
    bs = 16
    lens = [r.randint(0, width * bs) for _ in range(requests)]
    finished = [r.random() < 0.4 for _ in range(requests)]
    pool = requests * width + 5
    ids = r.sample(range(pool), requests * width)
    table = [[ids.pop() for _ in range(width)] for _ in range(requests)]
    for _ in range(requests // 3):  # entries that are no blocks
        table[r.randrange(requests)][r.randrange(width)] = r.choice([-1, pool, 2 ** 31 - 1, -2 ** 31])
    free = [-3] * pool
    want = list(free)
    count = ref.release(lens, finished, table, want, 4, bs, shared)
    got, before = ints(free), ints([4])
    after = None if in_place else ints([-9])
    serving.release_blocks_(ints(lens), ints(finished, torch.bool), ints(table), got, before, bs,
                            shared, after)
    assert got.tolist() == want
    assert (before if in_place else after).tolist() == [count]


def test_release_past_the_pool_and_of_nothing():
    table = [[0, 1, 2], [3, 2, 1]]
    free = ints([9, 9, 9, 9])
    count = ints([2])
    serving.release_blocks_(ints([48, 48]), ints([True, True], torch.bool), ints(table), free, count, 16)
    assert free.tolist() == [9, 9, 0, 1] and count.tolist() == [4]
    serving.release_blocks_(ints([]), ints([], torch.bool), torch.empty(0, 3, dtype=torch.int32, device=DEV),
                            free, count, 16)
    assert count.tolist() == [4]
    serving.release_blocks_(ints([48, 48]), ints([False, True], torch.bool), ints(table), free, count,
                            16, shared_blocks=50)
    assert count.tolist() == [4]


def test_plan_and_release_return_the_pool_to_where_it_was():
    step = Step([0] * 50, lengths(50, 400, 13, low=1), spare=2000, seed=13)
    args, _ = step.device()
    serving.plan_step_(**args)
    used = step.count - int(args["free_count"])
    assert used == sum(-(-q // 16) for q in step.query)
    serving.release_blocks_(args["seq_lens"], torch.ones(50, dtype=torch.bool, device=DEV),
                            args["block_table"], args["free_blocks"], args["free_count"], 16)
    assert int(args["free_count"]) == step.count
    assert sorted(args["free_blocks"].tolist()) == sorted(step.free)


def test_on_another_stream():
    step = Step(lengths(200, 300, 14), lengths(200, 40, 15), seed=14)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step.check()
