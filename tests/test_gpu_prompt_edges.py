"""prompt_attention where sequences fall back over earlier ones, and at values at
the ends of the types' ranges."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import serving
from test_gpu_attention import Prompt, assert_within, ints

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("starts", [[0, 50, 20, 90], [10, 300, 100, 400], [0, 130, 0, 131]])
def test_sequences_that_overlap_leave_each_others_rows_alone(d, starts):
    """Sequences 0 and 2 overlap: rows of one alone have its answer."""
    c = Prompt([400], d=d, seed=4)
    c.starts = starts
    out = c.run()
    first, second = ((starts[0], starts[1]), (starts[2], starts[3]))
    answers = []
    for a, b in (first, second):
        want, bound = ref.prompt(c.q[a:b], c.k[a:b], c.v[a:b], [0, b - a])
        inside = torch.zeros(400, dtype=torch.bool, device="cuda")
        inside[a:b] = True
        near = torch.zeros(400, c.q.shape[1], dtype=torch.bool, device="cuda")
        near[a:b] = ((out[a:b].double() - want).abs() <= bound).all(-1)
        answers.append((inside, near))
    (in_first, near_first), (in_second, near_second) = answers
    assert near_first[in_first & ~in_second].all()
    assert near_second[in_second & ~in_first].all()
    assert (out[~in_first & ~in_second] == 3.0).all()


def equal_weights(v, starts, group):
    """(out, bound) where all scores of a row are equal, to every bit: p is 1 without
    a rounding, the sums are fp32 ones over n keys, the result is rounded once."""
    hq = v.shape[1] * group
    out = torch.full((v.shape[0], hq, v.shape[2]), torch.nan, dtype=torch.float64, device=v.device)
    bound = torch.zeros_like(out)
    for a, b in zip(starts[:-1], starts[1:]):
        n = torch.arange(1, b - a + 1, device=v.device).view(-1, 1, 1)
        x = v[a:b].double().repeat_interleave(group, 1)
        out[a:b] = x.cumsum(0) / n
        bound[a:b] = (x.abs().cumsum(0) / n * (n + 64) * 2.0 ** -23 * (1 + ref.u(v.dtype))
                      + ref.u(v.dtype) * out[a:b].abs())
    return out, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_lowest_values_with_equal_scores(dtype, d):
    c = Prompt([150, 90], d=d, dtype=dtype, seed=7)
    want, bound = equal_weights(c.v, c.starts, 2)
    # every product is -2^2 or so and exact, all scores the same
    c.k.fill_(torch.finfo(dtype).min)
    c.q.fill_(2.0 ** (-126 if dtype == torch.bfloat16 else -14))
    assert_within(c.run(), want, bound, "lowest values")
    # products of d terms that cancel, none of their sums past the range of fp32
    huge = 2.0 ** 119 if dtype == torch.bfloat16 else 2.0 ** 15
    c.k.fill_(huge)
    c.k[:, :, 1::2] *= -1
    c.q.fill_(1.0 if dtype == torch.bfloat16 else 2.0 ** 15)
    assert_within(c.run(), want, bound, "cancelling scores")
