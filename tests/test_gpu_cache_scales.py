"""fp8 caches with scales of any sign and size: keys stand for code * k_scale,
also where that is zero, negative or so small that the scores all but vanish."""
import pytest
import torch

from test_gpu_attention import RAGGED, Decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("prefix, block_size", [(0, 16), (9, 16), (40, 32), (3, 48)])
@pytest.mark.parametrize("k_scale", [0.0, -0.0, -0.011, 1e-30, -1e-42, 2.0])
def test_key_scales(d, prefix, block_size, k_scale):
    p = prefix * block_size
    c = Decode([p + n for n in RAGGED], prefix, d=d, cache="fp8", block_size=block_size, seed=d)
    c.scales[0].fill_(k_scale)
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("k_scale", [0.011, 1e-8])
def test_queries_of_zeros(d, k_scale):
    """A row of zeros has no exponent to scale by; all its weights are equal."""
    c = Decode([144 + n for n in RAGGED], 9, d=d, cache="fp8", seed=d)
    c.scales[0].fill_(k_scale)
    c.q[::2] = 0
    c.q[1] = torch.finfo(c.q.dtype).smallest_normal
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("v_scale", [0.0, -0.5])
def test_value_scales(d, v_scale):
    c = Decode([144 + n for n in RAGGED], 9, d=d, cache="fp8", seed=d)
    c.scales[1].fill_(v_scale)
    c.check()
