"""Outputs that share memory with what a call reads are refused, views of one
buffer whose columns do not meet are not: the decision itself against a byte map,
and the refusals of the C ABI (no call here launches anything)."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

from sm120_rmsnorm import capi, serving_capi as sc

CSRC = Path(__file__).resolve().parents[1] / "sm120-norm-fusion-kernels_b200" / "csrc"
P = 1 << 20  # a non-null, aligned address that no refused call touches


@pytest.fixture(scope="module")
def rows_overlap(tmp_path_factory):
    folder = tmp_path_factory.mktemp("overlap")
    (folder / "o.cpp").write_text(
        '#include "row_overlap.h"\nusing namespace sm120n;\n'
        'extern "C" int overlap(long a, long na, long sa, long wa, long b, long nb, long sb, long wb) {\n'
        '  return rows_overlap({(void*)a, na, sa, wa}, {(void*)b, nb, sb, wb});\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(folder / "o.cpp"),
                    "-o", str(folder / "o.so")], check=True)
    fn = ctypes.CDLL(str(folder / "o.so")).overlap
    fn.argtypes = [ctypes.c_long] * 8
    return fn


def test_the_decision_against_a_map_of_bytes(rows_overlap):
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(20000):
        sets = []
        stride = rng.randint(1, 30)
        for _ in "ab":
            s = stride if rng.random() < 0.6 else rng.randint(1, 30)
            sets.append((1000 + rng.randint(0, 60), rng.randint(0, 6), s, rng.randint(0, s)))
        want = bool(set.intersection(*({p + i * s + k for i in range(n) for k in range(w)}
                                       for p, n, s, w in sets)))
        assert bool(rows_overlap(*sets[0], *sets[1])) == want, sets
        assert bool(rows_overlap(*sets[1], *sets[0])) == want, sets
        seen[want] += 1
    assert min(seen) > 2000


def test_far_addresses_and_strides(rows_overlap):
    far = 2 ** 62
    assert not rows_overlap(P, 1 << 31, far // 2 ** 20, 64, far, 5, far // 2 ** 20, 64)
    assert rows_overlap(P, 1 << 31, 4096, 64, P + 4096 * (2 ** 31 - 1), 1, 0, 64)
    assert not rows_overlap(P, 1 << 31, 4096, 64, P + 4096 * (2 ** 31 - 1) + 64, 9, 4096, 4032)


D = 128


def prompt(out, stride=8 * D, tokens=10, heads=2):
    """q, k, v as the columns of one buffer of `stride` elements a row; bytes of `out`."""
    sc.prompt_attention(sc.PromptArgs(
        dtype=sc.BF16, tokens=tokens, sequences=2, query_heads=heads, key_heads=2, head_dim=D,
        query=P, query_token_stride=stride, key=P + 2 * 2 * D, key_token_stride=stride,
        value=P + 2 * 4 * D, value_token_stride=stride, out=out, out_token_stride=stride,
        query_start=P, scale=0.1))


def decode(**kw):
    a = dict(dtype=sc.BF16, batch=3, query_heads=4, key_heads=2, head_dim=D, query=P,
             query_token_stride=1024, out=P + 2 * 512, out_token_stride=1024, key_cache=8 * P,
             value_cache=16 * P, num_blocks=9, block_size=16, cache_block_stride=4096,
             cache_slot_stride=256, cache_head_stride=128, block_table=P, table_width=8,
             table_stride=8, seq_lens=P, scale=0.1)
    sc.paged_decode_attention(sc.DecodeArgs(**(a | kw)))


def mrope(value=None, cache=None, key=P + 2 * 512, **kw):
    store = dict(value=value or 64 * P, value_token_stride=1024, key_cache=cache or 8 * P,
                 value_cache=16 * P, slot_mapping=P, num_blocks=9, block_size=16,
                 cache_block_stride=4096, cache_slot_stride=256, cache_head_stride=128)
    qk = dict(dtype=sc.BF16, tokens=4, query_heads=4, key_heads=2, head_dim=D, rotary_dim=D,
              query=P, query_token_stride=1024, key=key, key_token_stride=1024,
              query_weight=P, key_weight=P, positions=P, cos_sin_cache=P, rope_positions=10)
    args = sc.QkCacheArgs(**qk, **(store if value or cache else {}))
    sc.qk_norm_mrope_cache(args, sc.MropeArgs(axes=1, sections=(sc._i32 * 4)(64),
                                              position_axis_stride=4, **kw))


@pytest.mark.parametrize("call, message", [
    (lambda: prompt(P), "out may not overlap query"),
    (lambda: prompt(P + 2 * 2 * D), "out may not overlap key"),
    (lambda: prompt(P + 2 * 4 * D), "out may not overlap value"),
    (lambda: prompt(P + 2 * 5 * D), "out may not overlap value"),
    (lambda: prompt(P + 2 * 7 * D), "out may not overlap query"),  # reaches into the next row
    (lambda: prompt(P + 2 * 8 * D * 9), "out may not overlap query"),  # begins at the last row
    (lambda: prompt(P - 2 * 8 * D * 9), "out may not overlap query"),
    (lambda: decode(out=P), "out may not overlap query"),
    (lambda: decode(out=P + 2 * 600), "out may not overlap query"),
    (lambda: decode(out=8 * P + 2 * 4096 * 8), "out may not overlap key_cache"),
    (lambda: decode(out=16 * P - 16), "out may not overlap value_cache"),
    (lambda: mrope(query_out=P + 256, query_out_token_stride=1024), "query_out may not overlap its input"),
    (lambda: mrope(query_out=P, query_out_token_stride=1032), "query_out may not overlap its input"),
    (lambda: mrope(query_out=P + 2 * 512, query_out_token_stride=1024), "query_out may not overlap key"),
    (lambda: mrope(key_out=P + 2 * 256, key_out_token_stride=1024), "key_out may not overlap query"),
    (lambda: mrope(query_out=32 * P, query_out_token_stride=1024, key_out=32 * P + 2 * 500,
                   key_out_token_stride=1024), "query_out may not overlap key_out"),
    (lambda: mrope(value=64 * P, query_out=64 * P, query_out_token_stride=1024),
     "query_out may not overlap value"),
    (lambda: mrope(value=64 * P, key_out=64 * P + 2 * 200, key_out_token_stride=1024),
     "key_out may not overlap value"),
    (lambda: mrope(cache=8 * P, key_out=16 * P + 2 * 4096, key_out_token_stride=1024),
     "key_out may not overlap the caches"),
    (lambda: mrope(cache=P + 2 * 800), "query may not overlap the caches"),
    (lambda: mrope(key=P + 2 * 500), "query may not overlap key"),
])
def test_refusals(call, message):
    with pytest.raises(capi.CApiError) as error:
        call()
    assert error.value.status == capi.ERR_INVALID_ARGUMENT and message in str(error.value)
