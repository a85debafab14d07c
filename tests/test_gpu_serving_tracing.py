"""Traced serving operators are in the graph, and the graph computes them."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from sm120_rmsnorm import serving

pytestmark = pytest.mark.gpu


def attention():
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(40, h, 128, device="cuda", generator=g).to(torch.bfloat16) for h in (4, 2, 2))
    starts = torch.tensor([0, 30, 40], dtype=torch.int32, device="cuda")

    def f(q, k, v, starts):
        out = torch.zeros_like(q)
        serving.prompt_attention(out, q, k, v, starts)
        return out

    return f, (q, k, v, starts)


@pytest.mark.parametrize("mode", ["real", "fake"])
def test_make_fx_records_the_operator(mode):
    f, args = attention()
    want = f(*args)
    traced = make_fx(f, tracing_mode=mode)(*args)
    assert any("prompt_attention" in str(n.target) for n in traced.graph.nodes)
    assert torch.equal(traced(*args), want)


def test_compiled_without_a_break():
    f, args = attention()
    want = f(*args)
    assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(*args), want)
