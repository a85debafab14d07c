"""engine.PagedSteps without a GPU: the two operators that it calls are replaced
by the plain walks of tests/serving_reference.py, on CPU tensors. What is tested
is which lengths, tables and pools it hands them over several requests."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import engine

BLOCK = 16


def ints(values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.fixture(autouse=True)
def plain_operators(monkeypatch):
    def plan(context, query, table, free, count, block_size, start, lens, positions, slots,
             count_out, row_positions, row_slots, row_lens):
        rows, before, asked = table.tolist(), context.tolist(), query.tolist()
        got = ref.plan(context.tolist(), query.tolist(), rows, free.tolist(), int(count),
                       block_size, positions.numel())
        table.copy_(ints(rows).view_as(table))
        for to, values in zip((start, lens, positions, slots), got):
            to.copy_(torch.tensor(values))
        (count if count_out is None else count_out).fill_(got[4])
        for r, (c, q, first) in enumerate(zip(before, asked, got[0])):
            fits = q > 0 and sum(asked[:r + 1]) <= positions.numel() and got[3][first] >= 0
            row_slots[r] = got[3][first] if fits else -2 if q > 0 else -1
            row_lens[r] = c + q if fits else 0
            row_positions[r] = c if fits else -1

    def release(lens, finished, table, free, count, block_size, shared=0, count_out=None):
        stack = free.tolist()
        left = ref.release(lens.tolist(), finished.tolist(), table.tolist(), stack, int(count),
                           block_size, shared)
        free.copy_(ints(stack))
        (count if count_out is None else count_out).fill_(left)

    monkeypatch.setattr(engine.serving, "plan_step_", plan)
    monkeypatch.setattr(engine.serving, "release_blocks_", release)


def steps_of(requests=2, blocks=20, width=10, tokens=64, **kw):
    return engine.PagedSteps(requests, blocks, width, tokens, "cpu", BLOCK, **kw)


def row_blocks(steps, row):
    """The blocks of a request as decode attention finds them."""
    n = int(steps.context_lens[row])
    prefix = steps.prefix.tolist()
    own = steps.block_table[row].tolist()
    ids = prefix + own[len(prefix):] if n >= len(prefix) * BLOCK else own
    return ids[:-(-n // BLOCK)]


def slots_of(ids, first, count):
    return [ids[p // BLOCK] * BLOCK + p % BLOCK for p in range(first, first + count)]


@pytest.mark.parametrize("prefix", [0, 2])
def test_what_is_stored_is_what_attention_reads(prefix):
    """Requests come, grow, end and make room for others: every token's slot is
    where attention looks for it, and no block is lost."""
    steps = steps_of(tokens=66, prefix_blocks=prefix)
    pool = int(steps.free_count)
    assert pool == 20 - prefix
    begin = prefix * BLOCK
    for lengths in ((50, 3), (7, 40), (33, 33)):
        context = [begin, begin]
        assert steps.context_lens.tolist() == context
        for query in (list(lengths), [1, 1], [0, 1], [14, 17]):
            steps.plan(ints(query))
            for r, n in enumerate(query):
                ids = row_blocks(steps, r)
                start = int(steps.query_start[r])
                assert steps.context_lens[r] == context[r] + n
                assert ids[:prefix] == steps.prefix.tolist()
                assert len(set(ids)) == len(ids)
                assert steps.slot_mapping[start:start + n].tolist() == slots_of(ids, context[r], n)
                context[r] += n
            held = [row_blocks(steps, r)[prefix:] for r in range(2)]
            assert not set(held[0]) & set(held[1])
        steps.release(torch.tensor([True, False]))
        steps.release(torch.tensor([True, True]))  # the first has nothing left to give
        assert int(steps.free_count) == pool
        assert sorted(steps.free_blocks[:pool].tolist()) == sorted(set(range(20)) - set(steps.prefix.tolist()))


def test_the_prefix_is_written_as_a_prompt_of_its_own():
    steps = steps_of(prefix_blocks=3)
    writer = steps.prefix_writer()
    writer.plan(ints([3 * BLOCK]))
    assert writer.slot_mapping.tolist() == slots_of(steps.prefix.tolist(), 0, 3 * BLOCK)
    assert writer.positions.tolist() == list(range(3 * BLOCK))
    assert int(steps.free_count) == 17  # the batch's pool is not touched


def test_rows_that_do_not_share_the_prefix_stand_in_a_batch_over_the_same_pool():
    sharing = steps_of(prefix_blocks=2)
    alone = steps_of(pool=sharing)
    alone.plan(ints([50, 1]))
    sharing.plan(ints([20, 1]))
    assert int(sharing.free_count) == int(alone.free_count) == 18 - 4 - 1 - 2 - 1
    held = [b for s in (alone, sharing) for r in range(2) for b in row_blocks(s, r)[len(s.prefix):]]
    assert len(set(held)) == len(held) and not set(held) & set(sharing.prefix.tolist())
    assert alone.slot_mapping[:50].tolist() == slots_of(row_blocks(alone, 0), 0, 50)
    alone.release(torch.tensor([True, True]))
    sharing.release(torch.tensor([True, True]))
    assert int(sharing.free_count) == 18


def rows_of(steps, query):
    steps.plan(ints(query))
    lens = steps.row_lens.tolist()
    assert steps.row_positions.tolist() == [n - 1 for n in lens]
    return [max(s, -1) for s in steps.row_slots.tolist()], lens, steps.unserved.nonzero().flatten().tolist()


def test_decode_rows_are_requests_whoever_has_a_token():
    steps = steps_of(requests=4, blocks=4, tokens=4)
    assert rows_of(steps, [1, 1, 0, 1]) == ([0, 16, -1, 32], [1, 1, 0, 1], [])
    assert rows_of(steps, [0, 1, 0, 1]) == ([-1, 17, -1, 33], [0, 2, 0, 2], [])
    steps.release(torch.tensor([False, True, False, False]))
    assert rows_of(steps, [1, 0, 1, 1]) == ([1, -1, 16, 34], [2, 0, 1, 3], [])
    # block 3 alone is left, for the second row; the first request waits
    steps.release(torch.tensor([True, False, False, False]))
    steps.free_count.fill_(1)
    assert rows_of(steps, [0, 1, 1, 0]) == ([-1, 48, 17, -1], [0, 1, 2, 0], [])
    assert rows_of(steps, [1, 1, 0, 1]) == ([-1, 49, -1, 35], [0, 2, 0, 4], [0])
    assert steps.context_lens.tolist() == [0, 2, 2, 4]


def test_tokens_past_the_buffer_are_unserved():
    steps = steps_of(requests=3, blocks=9, tokens=2)
    assert rows_of(steps, [1, 1, 1]) == ([0, 16, -1], [1, 1, 0], [2])


def test_decode_wants_a_row_per_request():
    with pytest.raises(ValueError, match="one row per request"):
        engine.Qwen3Attention(None, None, None, None).decode(torch.zeros(1, 8), None, steps_of())


def test_prompts_behind_a_prefix_are_refused():
    """Prompt attention sees the packed tokens alone, not the prefix."""
    with pytest.raises(ValueError, match="prefix"):
        engine.Qwen3Attention(None, None, None, None).prompts(None, None, steps_of(prefix_blocks=1))


@pytest.mark.parametrize("bad", [dict(prefix_blocks=-1), dict(prefix_blocks=21, width=30),
                                 dict(prefix_blocks=11)])
def test_prefixes_that_do_not_fit_are_refused(bad):
    with pytest.raises(ValueError, match="prefix_blocks"):
        steps_of(**bad)


def test_pools_that_do_not_fit_are_refused():
    with pytest.raises(ValueError, match="pool"):
        steps_of(blocks=21, pool=steps_of())
    with pytest.raises(ValueError, match="pool"):
        steps_of(prefix_blocks=1, pool=steps_of())
