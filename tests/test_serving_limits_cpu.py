"""Sizes at the ends of what the serving operators' 32-bit indices can hold are
refused before anything is launched."""
import pytest

from sm120_rmsnorm import capi
from test_serving_cpu import plan, prompt, release


@pytest.mark.parametrize("call", [plan, release])
@pytest.mark.parametrize("sizes", [dict(requests=2 ** 31 - 1), dict(requests=2 ** 31 - 1000),
                                   dict(requests=2 ** 30 + 1),
                                   dict(table_width=2 ** 31 - 1, table_stride=2 ** 31),
                                   dict(table_width=2 ** 30 + 1, table_stride=2 ** 31)])
def test_rows_and_entries_whose_rounds_would_overflow(call, sizes):
    with pytest.raises(capi.CApiError, match="2\\^30") as error:
        call(**sizes)
    assert error.value.status == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("sequences", [2 ** 31 - 200, 2 ** 31 - 2])
def test_sequences_whose_search_would_overflow(sequences):
    with pytest.raises(capi.CApiError, match="sequences must be") as error:
        prompt(sequences=sequences, query_heads=1, key_heads=1)
    assert error.value.status == capi.ERR_INVALID_ARGUMENT
