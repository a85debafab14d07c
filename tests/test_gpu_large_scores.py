"""Scores so large that a row's largest keys take all of its weight: every product
q . k is q0 k_j D for a power of two q0, exact in fp32, and the keys' values are
so far apart for the type that two scores are equal or 2^20 apart and more.

With m equal largest scores the result is the mean of their m values: each weight
p / (m p) with p = 2^x, x in [0, 8] (a running maximum may lag), rounded to the operand
type (u A), sums of at most n + 64 fp32 steps, one rounding of the result."""
import pytest
import torch

import serving_reference as ref
from test_gpu_attention import Decode, Prompt

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def check_row(out, scores, values, operand, what):
    """out [H, D] of rows with the same scores [n] over values [n, D]."""
    top = scores == scores.max()
    v = values.double()[top]
    want, a = v.mean(0), v.abs().mean(0)
    bound = (a * (ref.u(operand) + (len(scores) + 64) * 2.0 ** -23) * (1 + ref.u(out.dtype))
             + ref.u(out.dtype) * want.abs())
    assert ((out.double() - want).abs() <= bound).all(), what


def query(dtype, q):
    """Every score above 2^22 in units of exp2, and as far as the type reaches."""
    q.fill_({"large": 2.0 ** 13, "largest": 2.0 ** (100 if dtype == torch.bfloat16 else 15)}[query.size])


@pytest.fixture(params=["large", "largest"], autouse=True)
def size(request):
    query.size = request.param


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("sign", [1, -1])
def test_prompts(dtype, d, order, sign):
    n = 300
    c = Prompt([n], hq=2, hk=1, d=d, dtype=dtype, seed=8)
    steps = torch.arange(n, device="cuda") // 3
    steps = steps if order > 0 else steps.flip(0)
    c.k.copy_((4096 * (1 + steps / 128.0) * sign).view(-1, 1, 1))  # 1 + i / 128: 7 bits
    query(dtype, c.q)
    out = c.run()
    scores = c.k[:, 0, 0].double()
    for i in range(n):
        check_row(out[i], scores[:i + 1], c.v[:i + 1, 0], dtype, i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("prefix, block_size", [(0, 16), (12, 16), (3, 48)])
def test_decode(dtype, d, cache, prefix, block_size):
    p = prefix * block_size
    lens = [p + n for n in (1, 40, 130, 700)]
    c = Decode(lens, prefix, hq=4, hk=2, d=d, dtype=dtype, cache=cache, block_size=block_size, seed=9)
    g = torch.Generator(device="cuda").manual_seed(3)
    # 8 values that every type holds, the largest in prefix and own tokens alike
    values = torch.tensor([16., 18, 20, 22, 24, 26, 28, 30], device="cuda") * (1 if cache == "fp8" else 256)
    pick = torch.randint(0, 8, c.kc.shape[:2] + (1, 1), device="cuda", generator=g)
    c.kc.copy_(values[pick].expand(c.kc.shape).to(c.kc.dtype))
    query(dtype, c.q)
    if cache == "fp8":
        c.scales[0].fill_(256.0)
    out = c.run()
    for r, n in enumerate(lens):
        row = c.table[r].tolist()
        ids = ([] if c.prefix is None else c.prefix.tolist()) + row[prefix:]
        k, _ = ref.cache_tokens(c.kc, ids[:-(-n // block_size)], "NHD", c.scales[0])
        v, _ = ref.cache_tokens(c.vc, ids[:-(-n // block_size)], "NHD", c.scales[1])
        for h in range(2):
            check_row(out[r, 2 * h:2 * h + 2], k[:n, h, 0], v[:n, h],
                      torch.float16 if cache == "fp8" else dtype, (r, h))
