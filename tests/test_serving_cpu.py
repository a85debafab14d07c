"""Serving operators without a GPU: the library's exports, refusals of the C ABI
(nothing is launched), the binding's refusals, and the 64-bit references."""
import re
import subprocess
from pathlib import Path

import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import capi, extensions, serving, serving_capi as sc

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "sm120norm_b200_serving.h"
P = 1 << 20  # a non-null, aligned address that no refused call touches


def test_library_exports_what_the_header_declares_and_nothing_else():
    declared = set(re.findall(r"SM120N_API\s+[\w\s\*]+?\b(sm120s_\w+)\s*\(", HEADER.read_text()))
    assert declared == set(sc.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", str(sc.LIBRARY_PATH)],
                         capture_output=True, text=True, check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if " T " in line} == declared
    assert sc.abi_version() == 1


def plan(**kw):
    a = dict(context_lens_ptr=P, query_lens_ptr=P, block_table_ptr=P, table_stride=8,
             free_blocks_ptr=P, free_count_ptr=P, free_count_out_ptr=P, query_start_ptr=P,
             seq_lens_ptr=P, positions_ptr=P, slot_mapping_ptr=P, requests=3, table_width=8,
             pool=50, block_size=16, tokens=10)
    sc.plan_step(**(a | kw))


def release(**kw):
    a = dict(seq_lens_ptr=P, finished_ptr=P, block_table_ptr=P, table_stride=8, free_blocks_ptr=P,
             free_count_ptr=P, free_count_out_ptr=P, requests=3, table_width=8, pool=50,
             block_size=16)
    sc.release_blocks(**(a | kw))


def mrope(sections=(16, 24, 24), axes=None, qk=None, **kw):
    n = len(sections) if axes is None else axes
    args = dict(dtype=sc.BF16, tokens=4, query_heads=4, key_heads=2, head_dim=128, rotary_dim=128,
                query=P, query_token_stride=512, key=P, key_token_stride=256, query_weight=P,
                key_weight=P, positions=P, cos_sin_cache=P, rope_positions=10)
    m = dict(axes=n, sections=(sc._i32 * 4)(*sections), position_axis_stride=4)
    sc.qk_norm_mrope_cache(sc.QkCacheArgs(**(args | (qk or {}))), sc.MropeArgs(**(m | kw)))


def prompt(**kw):
    a = dict(dtype=sc.BF16, tokens=10, sequences=2, query_heads=4, key_heads=2, head_dim=128,
             query=P, query_token_stride=512, key=P, key_token_stride=256, value=P,
             value_token_stride=256, out=P, out_token_stride=512, query_start=P, scale=0.1)
    sc.prompt_attention(sc.PromptArgs(**(a | kw)))


def decode(**kw):
    a = dict(dtype=sc.BF16, batch=3, query_heads=4, key_heads=2, head_dim=128, query=P,
             query_token_stride=512, out=P, out_token_stride=512, key_cache=P, value_cache=P,
             num_blocks=9, block_size=16, cache_block_stride=4096, cache_slot_stride=256,
             cache_head_stride=128, block_table=P, table_width=8, table_stride=8, seq_lens=P,
             scale=0.1)
    sc.paged_decode_attention(sc.DecodeArgs(**(a | kw)))


INVALID, UNSUPPORTED = capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED


@pytest.mark.parametrize("call, status, message", [
    (lambda: plan(requests=-1), INVALID, "requests"),
    (lambda: plan(tokens=-1), INVALID, "tokens"),
    (lambda: plan(tokens=2 ** 31), INVALID, "tokens"),
    (lambda: plan(block_size=0), INVALID, "block_size"),
    (lambda: plan(pool=2 ** 28, block_size=16), INVALID, "at most 2^31"),
    (lambda: plan(table_stride=7), INVALID, "overlap"),
    (lambda: plan(free_count_ptr=0), INVALID, "non-null"),
    (lambda: plan(positions_ptr=0), INVALID, "non-null"),
    (lambda: plan(query_start_ptr=0), INVALID, "non-null"),
    (lambda: release(shared_blocks=-1), INVALID, "shared_blocks"),
    (lambda: release(finished_ptr=0), INVALID, "non-null"),
    (lambda: release(table_width=2 ** 31), INVALID, "2^31"),
    (lambda: mrope(axes=0), UNSUPPORTED, "1 to 4 axes"),
    (lambda: mrope(axes=5), UNSUPPORTED, "1 to 4 axes"),
    (lambda: mrope((16, 24, 25)), INVALID, "half the rotary width"),
    (lambda: mrope((80, -8, -8)), INVALID, "non-negative"),
    (lambda: mrope((20, 22, 22), interleaved_sections=1), INVALID, "more pairs than its turns"),
    (lambda: mrope(position_axis_stride=-1), INVALID, "position_axis_stride"),
    (lambda: mrope(query_out=P, query_out_token_stride=511), INVALID, "may not overlap"),
    (lambda: mrope(qk=dict(head_dim=96)), UNSUPPORTED, "head_dim"),
    (lambda: mrope(qk=dict(positions=None)), INVALID, "non-null"),
    (lambda: prompt(dtype=sc.F32), UNSUPPORTED, "float16 and bfloat16"),
    (lambda: prompt(head_dim=80), UNSUPPORTED, "head_dim"),
    (lambda: prompt(query_heads=5), INVALID, "multiple of key_heads"),
    (lambda: prompt(key_heads=0), INVALID, "multiple of key_heads"),
    (lambda: prompt(scale=0.0), INVALID, "scale"),
    (lambda: prompt(scale=-1.0), INVALID, "scale"),
    (lambda: prompt(scale=float("nan")), INVALID, "scale"),
    (lambda: prompt(scale=float("inf")), INVALID, "scale"),
    (lambda: prompt(tokens=-1), INVALID, "tokens"),
    (lambda: prompt(tokens=2 ** 31 - 300, query_heads=128, key_heads=128), INVALID, "too many tokens"),
    (lambda: prompt(key=None), INVALID, "non-null"),
    (lambda: prompt(query_start=None), INVALID, "non-null"),
    (lambda: prompt(value=P + 8), INVALID, "value rows must be 16-byte aligned"),
    (lambda: prompt(key_token_stride=260), INVALID, "key rows must be 16-byte aligned"),
    (lambda: prompt(out_token_stride=504), INVALID, "may not overlap"),
    (lambda: decode(dtype=sc.F32), UNSUPPORTED, "float16 and bfloat16"),
    (lambda: decode(head_dim=32), UNSUPPORTED, "head_dim"),
    (lambda: decode(cache_dtype=7), INVALID, "cache_dtype"),
    (lambda: decode(block_size=0), INVALID, "block_size"),
    (lambda: decode(num_blocks=2 ** 28), INVALID, "at most 2^31"),
    (lambda: decode(table_width=2 ** 28), INVALID, "table_width"),
    (lambda: decode(prefix_blocks=P, prefix_blocks_count=9), INVALID, "past the prefix"),
    (lambda: decode(prefix_blocks_count=2), INVALID, "non-null"),
    (lambda: decode(table_stride=7), INVALID, "overlap"),
    (lambda: decode(cache_slot_stride=250), INVALID, "cache rows must be 16-byte aligned"),
    (lambda: decode(cache_dtype=1, k_scale=P, v_scale=P, cache_slot_stride=264), INVALID, "16-byte"),
    (lambda: decode(cache_block_stride=-8), INVALID, "non-negative"),
    (lambda: decode(cache_dtype=1), INVALID, "k_scale"),
    (lambda: decode(query_token_stride=100), INVALID, "may not overlap"),
    (lambda: decode(seq_lens=None), INVALID, "non-null"),
    (lambda: decode(scale=0.0), INVALID, "scale"),
])
def test_refusals(call, status, message):
    with pytest.raises(capi.CApiError) as error:
        call()
    assert error.value.status == status and message in str(error.value)


def test_structs_of_another_size_are_refused():
    for args, call in ((sc.PromptArgs(), sc.prompt_attention), (sc.DecodeArgs(), sc.paged_decode_attention)):
        args.struct_size += 8
        with pytest.raises(capi.CApiError, match="struct_size"):
            call(args)


def test_calls_without_work_need_no_device():
    prompt(tokens=0)
    prompt(sequences=0, query_start=None)
    decode(batch=0)
    mrope(qk=dict(tokens=0))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (
        lambda: serving.prompt_attention(x, x, x, x, i),
        lambda: serving.paged_decode_attention(x, x, x[None], x[None], i[None], i),
        lambda: serving.release_blocks_(i, i.bool(), i[None], i, i[:1], 16),
        lambda: serving.plan_step_(i, i, i[None], i, i[:1], 16, i, i, i.long(), i),
        lambda: extensions.qk_norm_mrope_cache_(x, x, None, x[0, 0], x[0, 0], i.long()[None],
                                                x[0].float(), [64]),
    ):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_operators_can_be_traced_without_data():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 4, 128, dtype=torch.bfloat16, device="cuda")
        cache = torch.empty(8, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        i = torch.empty(2, dtype=torch.int32, device="cuda")
        serving.prompt_attention(x, x, x, x, i)
        serving.paged_decode_attention(x, x, cache, cache, i[None], i)
        extensions.qk_norm_mrope_cache_(x, x, None, x[0, 0], x[0, 0], i.long()[None],
                                        x[0].float(), [64])


# ---- the references themselves --------------------------------------------------------------
def test_prompt_reference_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(9, h, 64, generator=g).to(torch.bfloat16) for h in (4, 2, 2))
    out, bound = ref.prompt(q, k, v, [0, 4, 9])
    for i, (first, h) in enumerate([(0, 0), (0, 3), (4, 1)]):
        row = [3, 2, 8][i]
        s = (k[first:row + 1, h // 2].double() @ q[row, h].double()) / 8
        w = (s - s.max()).exp()
        want = (w[:, None] * v[first:row + 1, h // 2].double()).sum(0) / w.sum()
        assert torch.allclose(out[row, h], want, rtol=1e-12, atol=1e-14)
    assert (bound > 0).all() and (bound < 0.1).all()


def test_plan_reference_hands_out_whole_requests_in_order():
    table = [[5, -1, -1], [-1, -1, -1], [7, -1, -1]]
    starts, lens, positions, slots, left = ref.plan(
        [3, 0, 16], [2, 17, 1], table, [1, 2, 3, 4, 0, 0, 0, 0, 0], 3, 16, 22)
    assert starts == [0, 2, 19, 20] and lens == [5, 17, 17] and left == 0
    assert table == [[5, -1, -1], [3, 2, -1], [7, 1, -1]]
    assert slots[:2] == [83, 84] and slots[2:4] == [48, 49] and slots[18] == 32 and slots[19] == 16
    assert slots[20:] == [-1, -1] and positions[20:] == [-1, -1]
    table = [[-1], [-1], [0]]
    _, lens, _, slots, left = ref.plan([0, 0, 1], [1, 1, 1], table, [4, 9, 9, 9, 9], 1, 16, 3)
    assert lens == [1, 0, 2] and slots == [64, -1, 1] and left == 0


def test_sections_of_the_rotation():
    assert ref.axis_of([1, 2, 3], False) == [0, 1, 1, 2, 2, 2]
    assert ref.axis_of([4, 1, 1], True) == [0, 1, 2, 0, 0, 0]


@pytest.mark.parametrize("stride", ["cache_block_stride", "cache_slot_stride", "cache_head_stride"])
@pytest.mark.parametrize("value", [0, 8, -256])
def test_caches_whose_rows_overlap_are_refused(stride, value):
    with pytest.raises(capi.CApiError, match="may not overlap|non-negative"):
        decode(**{stride: value})
