"""Bounded waits of the attention kernels give up safely and can be told from
the outputs and the fault counter.

With the poll limit lowered to one non-blocking poll (sm120n_set_wait_limit) a
wait gives up before any load can have landed. Nothing faults or hangs: loads
and matrix instructions that were begun complete before their block ends. What
was not computed is left as it was (prompts) or NaN (decode)."""
import pytest
import torch

from sm120_rmsnorm import capi, serving_capi
from test_gpu_attention import RAGGED, Decode, Prompt

pytestmark = pytest.mark.gpu


@pytest.fixture
def one_poll():
    serving_capi.reset_device_faults()
    capi.set_wait_limit(1)
    yield
    torch.cuda.synchronize()
    capi.set_wait_limit(0)
    serving_capi.reset_device_faults()


def recovers(case):
    """With the default limit the same call is right and counts nothing."""
    capi.set_wait_limit(0)
    serving_capi.reset_device_faults()
    case.out.fill_(3.0)
    case.check()
    torch.cuda.synchronize()
    assert serving_capi.device_faults() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[300, 5, 77], [900]])
def test_prompt_rows_stay_as_they_were(one_poll, d, lens):
    c = Prompt(lens, d=d, padding=3, seed=1)
    out = c.run()
    torch.cuda.synchronize()
    assert serving_capi.device_faults() > 0
    assert (out == 3.0).all(-1).any()
    recovers(c)


@pytest.mark.parametrize("d", [64, 128])
def test_prompts_of_two_tile_blocks(one_poll, d):
    """Blocks of two row tiles come with large batches (12 blocks to an SM)."""
    c = Prompt([700] * 12, hq=64, hk=8, d=d, seed=2)
    out = c.run()
    torch.cuda.synchronize()
    assert serving_capi.device_faults() > 0
    assert (out == 3.0).all(-1).any()
    capi.set_wait_limit(0)
    first = c.run().clone()
    assert torch.equal(c.run(), first) and not (first == 3.0).all(-1).any()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("prefix, block_size", [(0, 16), (0, 5), (12, 16), (40, 32)])
def test_decode_rows_are_nan(one_poll, d, cache, prefix, block_size):
    c = Decode([prefix * block_size + n for n in RAGGED], prefix, d=d, cache=cache,
               block_size=block_size, seed=3)
    out = c.run()
    torch.cuda.synchronize()
    assert serving_capi.device_faults() > 0
    bad = out.isnan().all(-1)
    assert bad.any()
    # a row is either NaN as a whole or right
    capi.set_wait_limit(0)
    wrong = out.clone()
    c.out.fill_(3.0)
    right = c.run()
    assert torch.equal(wrong[~bad], right[~bad]) and not right.isnan().any()
    recovers(c)


def test_a_limit_between_loses_no_row(one_poll):
    """At limits that some waits meet and others do not, rows are right or NaN."""
    c = Decode([16 * 40 + n for n in RAGGED], 40, seed=4)
    capi.set_wait_limit(0)
    right = c.run().clone()
    for polls in (2, 5, 10, 20, 40, 80, 160, 320, 640):
        capi.set_wait_limit(polls)
        for _ in range(5):
            c.out.fill_(3.0)
            out = c.run()
            torch.cuda.synchronize()
            bad = out.isnan().all(-1)
            assert torch.equal(out[~bad], right[~bad])
    recovers(c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens, hq, hk", [([300, 5, 900], 4, 2), ([700] * 12, 64, 8)])
def test_a_limit_between_leaves_whole_prompt_rows(one_poll, d, lens, hq, hk):
    c = Prompt(lens, hq=hq, hk=hk, d=d, seed=5)
    capi.set_wait_limit(0)
    right = c.run().clone()
    for polls in (2, 5, 10, 20, 40, 80, 160, 320, 640):
        capi.set_wait_limit(polls)
        for _ in range(3):
            c.out.fill_(3.0)
            out = c.run()
            torch.cuda.synchronize()
            left = (out == 3.0).all(-1)
            assert torch.equal(out[~left], right[~left])
