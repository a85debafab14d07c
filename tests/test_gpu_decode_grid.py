"""The decode pass over own tokens has as many blocks as the SMs hold at once: the
workspace, which has a row of partial results for each, tells how many. And its
outputs with groups on both sides of where that number changes."""
import pytest
import torch

from sm120_rmsnorm import serving_capi as sc
from test_gpu_attention import RAGGED, Decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype, d, group, blocks", [
    (0, 64, 8, 2), (0, 64, 16, 2), (0, 128, 8, 2), (0, 128, 9, 1), (0, 128, 16, 1), (0, 128, 40, 1),
    (0, 256, 8, 1), (0, 256, 16, 1), (1, 64, 16, 2), (1, 128, 8, 2), (1, 128, 16, 2), (1, 256, 16, 1)])
def test_blocks_of_the_grid(cache_dtype, d, group, blocks):
    batch, key_heads = 100, 4
    got = sc.paged_decode_workspace(sc.DecodeArgs(
        dtype=sc.BF16, cache_dtype=cache_dtype, batch=batch, query_heads=group * key_heads,
        key_heads=key_heads, head_dim=d, num_blocks=100, block_size=16, table_width=64, scale=0.1))
    grid = blocks * torch.cuda.get_device_properties(0).multi_processor_count
    rows = (batch * key_heads * -(-group // 16) + grid) * 16
    assert got == -(-(batch + 1) * 8 // 16) * 16 + rows * (8 + 4 * d)


@pytest.mark.parametrize("group", [8, 9, 16, 17])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("prefix", [0, 30])
def test_groups_around_the_change(group, cache, prefix):
    Decode([prefix * 16 + n for n in RAGGED] * 4, prefix, hq=2 * group, hk=2, cache=cache,
           seed=group).check()
