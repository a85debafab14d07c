"""prompt_attention and paged_decode_attention against their definitions in 64
bits, within the bounds derived in tests/serving_reference.py."""
import math

import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import serving, serving_capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def assert_within(out, want, bound, what=""):
    live = ~want.isnan()
    bad = (~((out.double() - want).abs() <= bound))[live]
    if bad.any():
        worst = ((out.double() - want).abs() - bound)[live].max()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst by {worst}")


# ---- prompts -------------------------------------------------------------------------------
class Prompt:
    def __init__(self, lens, hq=4, hk=2, d=128, dtype=torch.bfloat16, padding=0, seed=0, first=0,
                 views=True):
        g = gen(seed)
        t = first + sum(lens) + padding
        self.starts = [first]
        for n in lens:
            self.starts.append(self.starts[-1] + n)
        qkv = torch.randn(t, (hq + 2 * hk) * d, device=DEV, generator=g).to(dtype)
        self.q = qkv[:, :hq * d].view(t, hq, d)
        self.k = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        self.v = qkv[:, (hq + hk) * d:].view(t, hk, d)
        if not views:
            self.q, self.k, self.v = (x.contiguous() for x in (self.q, self.k, self.v))
        self.q.mul_(2)
        self.out = torch.full((t, hq, d), 3.0, dtype=dtype, device=DEV)

    def run(self, **kw):
        serving.prompt_attention(self.out, self.q, self.k, self.v, ints(self.starts), **kw)
        return self.out

    def check(self, **kw):
        want, bound = ref.prompt(self.q, self.k, self.v, self.starts, **kw)
        out = self.run(**kw)
        assert_within(out, want, bound)
        outside = want.isnan().all(-1).all(-1)
        assert (out[outside] == 3.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [63, 64, 65], [127, 128, 129], [300, 5, 0, 77], [700]])
def test_prompt_lengths(dtype, d, lens):
    Prompt(lens, d=d, dtype=dtype, padding=5, seed=d + len(lens)).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq, hk", [(1, 1), (8, 8), (8, 1), (28, 4), (10, 2), (3, 1), (40, 2), (96, 1), (300, 1)])
def test_prompt_groups(hq, hk, d):
    Prompt([130, 1, 40], hq, hk, d, seed=hq).check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq, hk", [(2, 2), (4, 1), (7, 1)])
def test_long_prompts(hq, hk, d):
    Prompt([2500, 1031], hq, hk, d, seed=1).check()


def test_many_short_prompts_and_a_start_behind_the_first_row():
    Prompt([(7 * i) % 23 for i in range(300)], seed=2, first=11, padding=9).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_contiguous_rows_and_a_scale(d):
    Prompt([200, 31], d=d, seed=3, views=False).check(scale=0.3)


@pytest.mark.parametrize("starts", [[0, 50, 20, 90], [-5, 30, 60], [0, 40, 4000], [0, 0, 0, 0], [70]])
def test_starts_that_fall_or_leave_the_rows(starts):
    """A sequence that ends before it begins is empty; starts are clamped to the rows."""
    c = Prompt([90], seed=4, padding=0)
    clamped = [min(max(s, 0), 90) for s in starts]
    spans = [(a, b) for a, b in zip(clamped[:-1], clamped[1:]) if b > a]
    c.starts = starts
    out = c.run().clone()
    want = torch.full_like(out, 3.0)
    if starts == [0, 50, 20, 90]:  # the third overlaps the first: rows 20-49 may come from either
        spans = [(0, 20), (50, 50)]
    for a, b in spans:
        if b > a:
            o, bound = ref.prompt(c.q[a:b], c.k[a:b], c.v[a:b], [0, b - a])
            assert_within(out[a:b], o, bound)
    covered = torch.zeros(90, dtype=torch.bool, device=DEV)
    for a, b in zip(clamped[:-1], clamped[1:]):
        covered[a:max(a, b)] = True
    assert torch.equal(out[~covered], want[~covered])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_behind_a_sequence_take_no_part(d, value):
    c = Prompt([100, 37, 200], d=d, padding=50, seed=5)
    clean, bound = ref.prompt(c.q, c.k, c.v, c.starts)
    for x in (c.k, c.v):
        x[c.starts[-1]:] = value  # behind the last
    c.q[c.starts[-1]:] = value
    c.check()
    # the middle sequence spoilt: the others are as before
    a, b = c.starts[1], c.starts[2]
    for x in (c.k, c.v):
        x[a:b] = value
    out = c.run()
    keep = torch.ones(out.shape[0], dtype=torch.bool, device=DEV)
    keep[a:b] = False
    keep[c.starts[-1]:] = False
    assert_within(out[keep], clean[keep], bound[keep])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("where", [0, 70, 150, 333, 399])
@pytest.mark.parametrize("which", ["key", "value"])
def test_later_tokens_cannot_reach_earlier_rows(d, where, which):
    c = Prompt([400], hq=4, hk=2, d=d, seed=6)
    clean, bound = ref.prompt(c.q, c.k, c.v, c.starts)
    x = c.k if which == "key" else c.v
    x[where, 0, 3] = math.nan
    x[where, 0, 17] = math.inf
    out = c.run()
    assert_within(out[:where], clean[:where], bound[:where])
    assert_within(out[:, 2:], clean[:, 2:], bound[:, 2:])  # the other key head
    if which == "value":
        assert out[where:, :2, 3].isnan().all()
        other = [i for i in range(d) if i not in (3, 17)]
        assert_within(out[:, :2][..., other], clean[:, :2][..., other], bound[:, :2][..., other])
    else:
        assert out[where:, :2].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_scores_and_lowest_values(dtype, d):
    c = Prompt([150, 90], d=d, dtype=dtype, seed=7)
    c.q.mul_(30)
    c.check()  # one key takes nearly all of the weight
    c.q.fill_(-8.0)
    c.k.fill_(4.0)
    c.check()  # equal and very negative scores
    if dtype == torch.bfloat16:
        c.k.fill_(torch.finfo(dtype).min)
        c.q.fill_(1.0)
        c.k[:, :, 1::2] *= -1  # scores that cancel to zero between the lowest and highest values
        out = c.run()
        assert out[:150].isfinite().all() or out.isnan().any()


def test_prompt_runs_are_equal_bit_for_bit():
    c = Prompt([511, 300, 40], hq=8, hk=2, seed=8)
    first = c.run().clone()
    for _ in range(3):
        c.out.fill_(3.0)
        assert torch.equal(c.run(), first)


def test_prompt_captured_and_on_another_stream():
    c = Prompt([200, 333], seed=9)
    starts = ints(c.starts)
    eager = c.run().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.prompt_attention(c.out, c.q, c.k, c.v, starts)
    c.out.fill_(3.0)
    graph.replay()
    assert torch.equal(c.out, eager)
    # new lengths and inputs in the same buffers
    starts.copy_(ints([0, 17, 500]))
    c.q.mul_(0.5)
    c.out.fill_(3.0)
    graph.replay()
    want, bound = ref.prompt(c.q, c.k, c.v, [0, 17, 500])
    assert_within(c.out, want, bound)
    assert (c.out[500:] == 3.0).all()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = torch.full_like(c.out, 3.0)
    with torch.cuda.stream(stream):
        serving.prompt_attention(other, c.q, c.k, c.v, starts)
    stream.synchronize()
    assert torch.equal(other, c.out)


# ---- decode -------------------------------------------------------------------------------
class Decode:
    def __init__(self, lens, prefix=0, hq=8, hk=2, d=128, dtype=torch.bfloat16, cache="same",
                 layout="NHD", block_size=16, seed=0, pairs=False, spare_width=2):
        g = gen(seed)
        b = len(lens)
        bs = block_size
        self.lens, self.layout, self.bs = lens, layout, bs
        p = prefix
        need = [(-(-n // bs) - p if n >= p * bs else -(-n // bs)) for n in lens]
        blocks = p + sum(need) + 2
        ids = torch.randperm(blocks, device=DEV, generator=g).tolist()
        self.prefix = ints([ids.pop() for _ in range(p)]) if p else None
        width = max([-(-n // bs) for n in lens] + [p]) + spare_width
        self.table = torch.full((b, width), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
        for r, (n, count) in enumerate(zip(lens, need)):
            first = p if n >= p * bs else 0
            self.table[r, first:first + count] = ints([ids.pop() for _ in range(count)])
        shape = (blocks, bs, hk, d) if layout == "NHD" else (blocks, hk, bs, d)
        if pairs:
            both = torch.randn(blocks, 2, *shape[1:], device=DEV, generator=g)
            kc, vc = None, None
        else:
            both = torch.stack([torch.randn(shape, device=DEV, generator=g) for _ in "kv"], 1)
        self.scales = [None, None]
        if cache == "same":
            both = both.to(dtype)
        else:
            self.scales = [torch.tensor([0.011], device=DEV), torch.tensor([0.023], device=DEV)]
            both = (both / torch.stack(self.scales).view(1, 2, 1, 1, 1)).clamp(-448, 448).to(
                torch.float8_e4m3fn)
            if cache == "u8":
                both = both.view(torch.uint8)
        self.kc, self.vc = (both[:, i] if pairs else both[:, i].contiguous() for i in (0, 1))
        self.q = (2 * torch.randn(b, hq, d, device=DEV, generator=g)).to(dtype)
        self.out = torch.full_like(self.q, 3.0)

    def run(self, **kw):
        serving.paged_decode_attention(self.out, self.q, self.kc, self.vc, self.table, ints(self.lens),
                                       self.prefix, *self.scales, kv_cache_layout=self.layout, **kw)
        return self.out

    def check(self, **kw):
        want, bound = ref.decode(self.q, self.kc, self.vc, self.table, self.lens, self.prefix,
                                 self.layout, *self.scales, **kw)
        assert_within(self.run(**kw), want, bound)
        empty = [r for r, n in enumerate(self.lens) if n <= 0]
        assert (self.out[empty] == 0).all()


RAGGED = [1, 70, 0, 400, 15, 16, 17, 129, 1000, 64, 63, 65]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8", "u8"])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_decode_without_a_prefix(dtype, d, cache, layout):
    Decode(RAGGED, d=d, dtype=dtype, cache=cache, layout=layout, seed=d).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("prefix, block_size", [(1, 16), (9, 16), (3, 48), (40, 32), (130, 1)])
def test_decode_with_a_prefix(dtype, d, cache, prefix, block_size):
    p = prefix * block_size
    lens = [p + n for n in RAGGED] + [p, 0, p - 1, 1, p // 2]
    Decode(lens, prefix, d=d, dtype=dtype, cache=cache, block_size=block_size, seed=prefix,
           layout="HND" if prefix % 2 else "NHD").check()


@pytest.mark.parametrize("hq, hk", [(1, 1), (4, 4), (8, 1), (28, 4), (16, 1), (17, 1), (40, 1), (64, 2)])
@pytest.mark.parametrize("prefix", [0, 5])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_decode_groups(hq, hk, prefix, cache):
    Decode([prefix * 16 + n for n in (3, 200, 90)], prefix, hq, hk, cache=cache, seed=hq).check()


@pytest.mark.parametrize("batch", [1, 2, 33, 150])
@pytest.mark.parametrize("prefix", [0, 70])
def test_decode_batches(batch, prefix):
    Decode([prefix * 16 + (37 * i) % 500 for i in range(batch)], prefix, hq=4, hk=1, d=64,
           seed=batch).check()


@pytest.mark.parametrize("batch", [768, 769, 1601])
@pytest.mark.parametrize("prefix", [0, 2])
def test_batches_that_are_scanned_in_several_steps(batch, prefix):
    # 768 requests to a step; the last step's among them with tokens and without
    lens = [(37 * i) % 90 if i % 5 else 0 for i in range(batch)]
    Decode(lens, prefix, hq=2, hk=1, d=64, seed=batch).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_long_request_and_a_long_prefix(d):
    Decode([30000], hq=4, hk=2, d=d, seed=1).check()
    Decode([16 * 1500 + 5, 16 * 1500 + 700], 1500, hq=4, hk=2, d=d, seed=2).check()


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_keys_and_values_in_one_buffer(layout, cache):
    Decode([100, 300, 9], 4, layout=layout, cache=cache, seed=3, pairs=True).check(scale=0.2)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_blocks_that_do_not_exist_hold_no_keys(d, cache):
    c = Decode([300, 200, 100, 40], 4, d=d, cache=cache, seed=4)
    c.table[0, 7], c.table[0, 9], c.table[1, 4:] = -1, 10 ** 9, -1
    c.table[2, :] = -2 ** 31  # nothing of its own
    c.prefix[2] = -1
    c.check()
    c.prefix[:] = 10 ** 6
    c.check()
    assert (c.out[2] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_lies_in_unused_slots_takes_no_part(d, cache, value):
    c = Decode([37, 16 * 5 + 3, 16 * 5, 0, 90], 5, d=d, cache=cache, seed=5)
    used = torch.zeros(c.kc.shape[0], c.bs, dtype=torch.bool, device=DEV)
    for r, n in enumerate(c.lens):
        row = c.table[r].tolist()
        ids = (c.prefix.tolist() + row[5:]) if n >= 80 else row
        for j in range(n):
            used[ids[j // 16], j % 16] = True
    for x in (c.kc, c.vc):
        x[~used] = torch.tensor(value, device=DEV).to(x.dtype)
    want, bound = ref.decode(c.q, c.kc, c.vc, c.table, c.lens, c.prefix, "NHD", *c.scales)
    assert want.isfinite().all()
    assert_within(c.run(), want, bound)
    # a spoilt request spoils no other
    c.kc[c.table[4, 5]] = torch.tensor(math.nan, device=DEV).to(c.kc.dtype)
    out = c.run()
    assert out[4].isnan().all()
    assert_within(out[:4], want[:4], bound[:4])


def test_lengths_past_the_table_and_negative():
    c = Decode([50, 60, 70], seed=6, spare_width=0)
    c.lens = [-3, 10 ** 6, 2 ** 31 - 1]
    c.table[1, 4:] = -1
    c.table[2, 5:] = -1
    c.check()


def test_long_strides_between_blocks_and_query_rows():
    c = Decode([100, 20, 300], 2, seed=7)
    wide = torch.zeros(c.kc.shape[0], 3, *c.kc.shape[1:], dtype=c.kc.dtype, device=DEV)
    wide[:, 0], wide[:, 2] = c.kc, c.vc
    c.kc, c.vc = wide[:, 0], wide[:, 2]
    rows = torch.zeros(3, 11 * 128, dtype=c.q.dtype, device=DEV)
    rows[:, 128:9 * 128] = c.q.view(3, -1)
    c.q = rows[:, 128:9 * 128].view(3, 8, 128)
    c.table = torch.cat((c.table, c.table), 1)[:, :c.table.shape[1]]
    assert c.table.stride(0) > c.table.shape[1]
    c.check()


def test_offsets_past_32_bits():
    """A cache of over 2^32 elements, read at its far end."""
    blocks = (1 << 32) // (16 * 8 * 128) + 40
    kc = torch.zeros(blocks, 16, 8, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    small = Decode([300, 45], 3, hq=8, hk=8, seed=8)
    n = small.kc.shape[0]
    kc[-n:], vc[-n:] = small.kc, small.vc
    moved = torch.where(small.table < n, small.table + (blocks - n), small.table)
    want = small.run().clone()
    out = torch.zeros_like(want)
    serving.paged_decode_attention(out, small.q, kc, vc, moved, ints(small.lens),
                                   small.prefix + (blocks - n))
    assert torch.equal(out, want)


def test_decode_runs_are_equal_bit_for_bit():
    c = Decode([16 * 40 + n for n in RAGGED], 40, seed=9)
    first = c.run().clone()
    for _ in range(3):
        c.out.fill_(3.0)
        assert torch.equal(c.run(), first)


def test_two_graphs_replayed_side_by_side():
    """Each call has a workspace of its own, so two captured calls may run at once."""
    cases = [Decode([16 * 30 + n for n in RAGGED], 30, seed=s) for s in (10, 11)]
    want = [c.run().clone() for c in cases]
    lens = [ints(c.lens) for c in cases]
    graphs = []
    for c, n in zip(cases, lens):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(4):
                serving.paged_decode_attention(c.out, c.q, c.kc, c.vc, c.table, n, c.prefix)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for c in cases:
        c.out.fill_(3.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.out, w)
    # the same graph with other lengths
    lens[0].copy_(ints([16 * 30 + 5] * len(RAGGED)))
    cases[0].table[:, 30] = cases[0].table[3, 30]
    graphs[0].replay()
    c = cases[0]
    w, bound = ref.decode(c.q, c.kc, c.vc, c.table, [16 * 30 + 5] * len(RAGGED), c.prefix)
    assert_within(c.out, w, bound)


def test_a_cache_without_blocks_and_an_empty_table():
    c = Decode([5, 0, 90], 2, seed=12)
    c.kc, c.vc = c.kc[:0], c.vc[:0]
    assert (c.run() == 0).all()
    c = Decode([5, 0, 90], seed=13)
    c.table = c.table[:, :0]
    assert (c.run() == 0).all()


def test_large_blocks():
    """Blocks that span several tiles of keys, and are not filled."""
    for d in (64, 128, 256):
        Decode([700, 129, 64, 1000, 256], 1, d=d, block_size=256, seed=14).check()
        Decode([700, 129, 64, 1000], 0, d=d, block_size=1024, layout="HND", cache="fp8", seed=15).check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_token_needs_no_stride(d):
    q, k, v = (torch.randn(1, h, d, device=DEV, dtype=torch.bfloat16) for h in (4, 2, 2))
    out = torch.zeros_like(q)
    start = ints([0, 1])
    serving_capi.prompt_attention(serving_capi.PromptArgs(
        dtype=serving_capi.BF16, tokens=1, sequences=1, query_heads=4, key_heads=2, head_dim=d,
        query=q.data_ptr(), query_token_stride=4 * d + 1, key=k.data_ptr(),
        key_token_stride=2 * d + 3, value=v.data_ptr(), value_token_stride=2 * d + 5,
        out=out.data_ptr(), out_token_stride=4 * d + 7, query_start=start.data_ptr(), scale=0.1),
        torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, v.repeat_interleave(2, dim=1))


def test_no_wait_ran_out():
    torch.cuda.synchronize()
    assert serving_capi.device_faults() == 0


def test_refusals_of_the_binding():
    c = Decode([50, 60], 2, seed=16)
    p = Prompt([40], seed=16)
    good = (c.out, c.q, c.kc, c.vc, c.table, ints(c.lens), c.prefix)

    def decode(message, **change):
        names = ("out", "query", "key_cache", "value_cache", "block_table", "seq_lens", "prefix_blocks")
        args = dict(zip(names, good)) | change
        with pytest.raises(RuntimeError, match=message):
            serving.paged_decode_attention(**args)

    decode("dtype", query=c.q.half())
    decode("float16 and bfloat16", query=c.q.float(), out=c.out.float(), key_cache=c.kc.float(),
           value_cache=c.vc.float())
    decode("one row per request", block_table=c.table[:1])
    decode("int32", block_table=c.table.long())
    decode("seq_lens", seq_lens=ints(c.lens).long())
    decode("entries", seq_lens=ints([1, 2, 3]))
    decode("4-D", value_cache=c.vc[1:])
    decode("k_scale", key_cache=c.kc.to(torch.float8_e4m3fn), value_cache=c.vc.to(torch.float8_e4m3fn))
    decode("multiple of key_heads", query=c.q[:, :3].contiguous(), out=c.out[:, :3].contiguous())
    decode("layout", kv_cache_layout="DNH")
    decode("past the prefix", prefix_blocks=ints([0] * 50))
    decode("overlap", out=c.q)
    decode("scale", scale=-1.0)
    decode("16-byte", query=torch.zeros(2 * 8 * 128 + 1, dtype=c.q.dtype, device=DEV)[1:].view(2, 8, 128))

    def prompt(message, **change):
        args = dict(out=p.out, query=p.q, key=p.k, value=p.v, query_start=ints([0, 40])) | change
        with pytest.raises(RuntimeError, match=message):
            serving.prompt_attention(**args)

    prompt("int32|Int", query_start=ints([0, 40]).long())
    prompt("one more", query_start=ints([]))
    prompt("key and value", key=p.k[:30])
    prompt("dtypes must match", key=p.k.half())
    prompt("out shape", out=p.out[:, :2])
    prompt("head_dim", **{k: torch.zeros(40, 2, 96, dtype=torch.bfloat16, device=DEV)
                          for k in ("out", "query", "key", "value")})
    prompt("scale", scale=0.0)
    same = p.q.contiguous()
    prompt("overlap", out=same, query=same)
