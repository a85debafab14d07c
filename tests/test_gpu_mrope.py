"""qk_norm_mrope_cache_ against its definition in 64 bits (tests/serving_reference.py:
the fp32 error of the definition, one rounding to the output, one to the cache)."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import extensions

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cos_sin(rows, rotary, base=1e6):
    inv = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    f = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEV), inv)
    return torch.cat((f.cos(), f.sin()), dim=-1).float()


class Case:
    def __init__(self, dtype=torch.bfloat16, d=128, rotary=None, tokens=37, hq=4, hk=2,
                 sections=None, in_turns=False, neox=True, cache="same", layout="NHD",
                 block_size=16, seed=0, rows=500, axes=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rotary = rotary or d
        half = rotary // 2
        self.sections = sections or [half - 2 * (half // 3), half // 3, half // 3]
        self.in_turns, self.neox, self.layout, self.dtype = in_turns, neox, layout, dtype
        self.qkv = torch.randn(tokens, (hq + 2 * hk) * d, device=DEV, generator=g).to(dtype)
        self.q = self.qkv[:, :hq * d].view(tokens, hq, d)
        self.k = self.qkv[:, hq * d:(hq + hk) * d].view(tokens, hk, d)
        self.v = self.qkv[:, (hq + hk) * d:].view(tokens, hk, d)
        self.qw, self.kw = ((1 + 0.2 * torch.randn(d, device=DEV, generator=g)).to(dtype) for _ in "qk")
        self.pos = torch.randint(0, rows, (len(self.sections), tokens), device=DEV, generator=g)
        self.pos[:, ::3] = self.pos[:1, ::3]  # text: all axes alike
        self.table = cos_sin(rows, rotary)
        self.bs = block_size
        blocks = -(-tokens // block_size) + 2
        self.slots = torch.randperm(blocks * block_size, device=DEV, generator=g)[:tokens].to(torch.int32)
        self.scales = [None, None]
        self.kc = self.vc = None
        if cache != "none":
            shape = (blocks, block_size, hk, d) if layout == "NHD" else (blocks, hk, block_size, d)
            store = {"same": dtype, "fp8": torch.float8_e4m3fn, "u8": torch.uint8}[cache]
            self.kc, self.vc = (torch.zeros(shape, device=DEV).to(store) for _ in "kv")
            if cache != "same":
                self.scales = [torch.tensor([0.02], device=DEV), torch.tensor([0.5], device=DEV)]

    def expected(self, x, w):
        return ref.mrope(x, w, self.pos, self.table, self.sections, self.in_turns, self.neox)

    def run(self, **kw):
        extensions.qk_norm_mrope_cache_(
            self.q, self.k, self.v, self.qw, self.kw, self.pos, self.table, self.sections, self.kc,
            self.vc, self.slots if self.kc is not None else None, *self.scales, is_neox=self.neox,
            interleaved_sections=self.in_turns, kv_cache_layout=self.layout, **kw)

    def check(self, in_place=True):
        want = [(*self.expected(x, w), x.clone()) for x, w in ((self.q, self.qw), (self.k, self.kw))]
        v = self.v.clone()
        if in_place:
            outs = [self.q, self.k]
            self.run()
            before = [want[0][3], want[1][3]]
        else:
            outs = [torch.full_like(x.contiguous(), 7) for x in (self.q, self.k)]
            before = [o.clone() for o in outs]
            self.run(query_out=outs[0], key_out=outs[1])
            assert torch.equal(self.q, want[0][3]) and torch.equal(self.k, want[1][3])
        assert torch.equal(self.v, v)
        for out, old, (y, bound, valid, _) in zip(outs, before, want):
            tol = bound + ref.u(self.dtype) * (y.abs() + bound) + 1e-30
            if self.dtype == torch.float16:
                tol = tol + 2.0 ** -25  # half a step among the subnormal values
            bad = ((out.double() - y).abs() > tol)[valid]
            assert not bad.any(), (int(bad.sum()), bad.numel())
            assert torch.equal(out[~valid], old[~valid])
        if self.kc is None:
            return
        valid = want[1][2]
        flat = [c.view(torch.float8_e4m3fn) if c.dtype == torch.uint8 else c for c in (self.kc, self.vc)]
        flat = [(c if self.layout == "NHD" else c.transpose(1, 2)).reshape(-1, *self.k.shape[1:])
                for c in flat]
        there = valid & (self.slots >= 0) & (self.slots < flat[0].shape[0])
        at = self.slots[there].long()
        if self.scales[0] is None:
            assert torch.equal(flat[0][at], outs[1][there])
            assert torch.equal(flat[1][at], v[there])
        else:
            for c, x, bound, scale in ((flat[0], want[1][0], want[1][1], self.scales[0]),
                                       (flat[1], v.double(), torch.zeros(1, device=DEV), self.scales[1])):
                x = (x / scale.double()).expand(valid.numel(), -1, -1)[there]
                bound = (bound / scale.double()).expand(valid.numel(), *x.shape[1:])[there]
                # the quotient is rounded to fp32, then once to e4m3 (half a step: 2^-4, or
                # 2^-10 among the subnormal codes); a shifted value may round the other way
                tol = (bound + 2.0 ** -23 * x.abs()) * 1.0625 + torch.clamp(x.abs() * 2.0 ** -4, min=2.0 ** -10)
                assert ((c[at].double() - x.clamp(-448, 448)).abs() <= tol).all()
        untouched = torch.ones(flat[0].shape[0], dtype=torch.bool, device=DEV)
        untouched[at] = False
        for c in flat:
            assert (c[untouched].float() == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d, rotary", [(64, 64), (128, 128), (128, 64), (256, 256), (256, 16)])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("in_turns", [True, False])
def test_types_head_sizes_and_sections(dtype, d, rotary, neox, in_turns):
    Case(dtype, d, rotary, neox=neox, in_turns=in_turns, seed=d + rotary).check()


@pytest.mark.parametrize("sections", [[16, 24, 24], [24, 20, 20], [64], [1, 63], [0, 0, 64],
                                      [10, 20, 30, 4], [62, 1, 1]])
@pytest.mark.parametrize("in_turns", [True, False])
def test_sections(sections, in_turns):
    if in_turns and any(k + (n - 1) * len(sections) >= 64 for k, n in enumerate(sections) if k and n):
        pytest.skip("no such turns: a test of the refusals covers it")
    Case(sections=sections, in_turns=in_turns, seed=1).check()


@pytest.mark.parametrize("cache", ["none", "same", "fp8", "u8"])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_caches_and_out_of_place(cache, layout, in_place, dtype):
    Case(dtype, cache=cache, layout=layout, seed=2, block_size=5).check(in_place)


@pytest.mark.parametrize("tokens", [1, 2, 700, 3001])
@pytest.mark.parametrize("hq, hk", [(1, 1), (28, 4), (3, 0)])
def test_token_and_head_counts(tokens, hq, hk):
    Case(tokens=tokens, hq=hq, hk=hk, seed=3, cache="none" if hk == 0 else "same").check()


def test_positions_and_slots_out_of_range_leave_everything_untouched():
    c = Case(cache="fp8", seed=4, in_turns=True)
    c.pos[0, 1], c.pos[1, 2], c.pos[2, 4], c.pos[2, 5] = -1, 500, -2 ** 62, 2 ** 62
    c.slots[7], c.slots[8], c.slots[9] = -1, 10 ** 6, -2 ** 31
    c.check(in_place=False)


def test_one_row_of_positions_for_all_axes():
    c = Case(seed=5, sections=[16, 24, 24])
    c.pos = c.pos[:1].expand(3, -1)
    assert c.pos.stride(0) == 0
    c.check()


def test_rows_without_16_byte_alignment():
    c = Case(seed=6, tokens=9)
    t, width = c.qkv.shape
    odd = torch.zeros(t * (width + 3) + 1, dtype=c.dtype, device=DEV)[1:].view(t, width + 3)
    odd[:, :width] = c.qkv
    hq, hk, d = 4, 2, 128
    c.q = odd.as_strided((t, hq, d), (width + 3, d, 1), 1)
    c.k = odd.as_strided((t, hk, d), (width + 3, d, 1), 1 + hq * d)
    c.v = odd.as_strided((t, hk, d), (width + 3, d, 1), 1 + (hq + hk) * d)
    c.check()


def test_close_to_the_single_axis_operator_and_repeatable():
    """All axes alike: the operator with one axis rounds after each stage, so
    the two agree within its roundings (three of bf16 at most, on the parts of
    the rotation), and two runs of this one agree in every bit."""
    c = Case(seed=7, sections=[16, 24, 24], cache="none", tokens=200)
    c.pos = c.pos[:1].expand(3, -1)
    y, bound, _ = c.expected(c.q, c.qw)
    parts = bound / ((128 / 2 + 16) * 2.0 ** -24)
    outs = [torch.empty_like(c.q.contiguous()) for _ in range(2)]
    k_out = torch.empty_like(c.k.contiguous())
    for o in outs:
        c.run(query_out=o, key_out=k_out)
    assert torch.equal(*outs)
    extensions.qk_norm_rope_cache_(c.q, c.k, None, c.qw, c.kw, c.pos[0].contiguous(), c.table)
    u = ref.u(torch.bfloat16)
    assert ((c.q.double() - outs[0].double()).abs() <= 2 * u * y.abs() + 2.1 * u * parts + 2 * bound).all()


def test_captured_on_another_stream():
    c = Case(seed=8, cache="same")
    q0 = c.qkv.clone()
    want_q = c.expected(c.q, c.qw)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        c.run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    eager = c.q.clone()
    c.qkv.copy_(q0)
    graph.replay()
    assert torch.equal(c.q, eager)
    assert (c.q.double() - want_q).norm() < 1e-2 * want_q.norm()
