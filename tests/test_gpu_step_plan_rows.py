"""plan_step_'s step with one row per request, against the packed step of the same
plan by a plain walk over the requests; whole numbers, so all must be equal."""
import copy

import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import serving
from test_gpu_step_plan import Step, ints, lengths

pytestmark = pytest.mark.gpu


def check(step, in_place=False, stride=None):
    args, _ = step.device(stride)
    n = len(step.context)
    rows = dict(row_positions=ints([-9] * n, torch.int64), row_slots=ints([-9] * n),
                row_lens=ints([-9] * n))
    table = copy.deepcopy(step.table)
    starts, lens, positions, slots, left = ref.plan(step.context, step.query, table, step.free,
                                                    step.count, step.bs, step.tokens)
    want, total = [], 0
    for r, (c, q) in enumerate(zip(step.context, step.query)):
        c, q = max(c, 0), max(q, 0)
        total += q
        if q == 0:
            want.append((-1, -1, 0))
        elif total > step.tokens or slots[starts[r]] < 0:
            want.append((-1, -2, 0))
        else:
            want.append((c, slots[starts[r]], c + q))
    if in_place:
        args["seq_lens"] = args["context_lens"]
    serving.plan_step_(**args, **rows)
    got = list(zip(*(rows[k].tolist() for k in ("row_positions", "row_slots", "row_lens"))))
    assert got == want
    # and the rest of the plan is what it is without them
    assert args["query_start"].tolist() == starts and args["seq_lens"].tolist() == lens
    assert args["positions"].tolist() == positions and args["slot_mapping"].tolist() == slots
    assert args["free_count"].tolist() == [left]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests", [1, 5, 64, 1001, 1024, 1025, 2500])
@pytest.mark.parametrize("block_size", [1, 16, 48])
def test_decode_steps_with_idle_rows(requests, block_size, in_place):
    query = [int(n > 0) for n in lengths(requests, 3, 2)]
    check(Step(lengths(requests, 200, 1), query, block_size, padding=5, seed=1), in_place)


@pytest.mark.parametrize("requests, top", [(1, 9000), (70, 700), (1100, 30), (3, 5000)])
def test_prompt_steps(requests, top):
    check(Step(lengths(requests, 300, 3), lengths(requests, top, 4), 16, padding=7, seed=2))


@pytest.mark.parametrize("spare", [0, 1, 37, 200])
def test_requests_without_room(spare):
    check(Step(lengths(1300, 100, 5), lengths(1300, 9, 6), spare=spare, seed=3))
    check(Step(lengths(40, 100, 5), [1] * 40, spare=spare, seed=3))


def test_edges():
    check(Step([0, 100, 20, 0], [64, 30, 5, 200], width=8, seed=4))
    check(Step([0, 10, 20, 30], [40, 50, 60, 70], seed=5, tokens=120))
    check(Step([0, 10], [3, 5], seed=6, tokens=0))
    check(Step([0, -5, 7, 0, 16], [0, 3, -2, 1, 0], seed=7, padding=5))
    check(Step([], [], seed=8, width=4, tokens=9, spare=3))
    check(Step(lengths(17, 90, 8), [1] * 17, seed=9), stride=33)
    check(Step([0, 0], [3, 0], width=0, seed=10, spare=4))
    step = Step([20, 20, 20], [1, 1, 1], seed=11)
    step.table[0][1], step.table[1][1] = -1, 10 ** 6
    check(step)


def test_refusals():
    step = Step([5, 6], [1, 1], seed=1)
    for rows, message in ((dict(row_slots=ints([0, 0])), "go together"),
                          (dict(row_slots=ints([0])), "row_slots"),
                          (dict(row_positions=ints([0, 0])), "row_positions"),
                          (dict(row_lens=torch.zeros(2, dtype=torch.int32)), "row_lens")):
        with pytest.raises(RuntimeError, match=message):
            serving.plan_step_(**step.device()[0], **rows)
