"""Outputs beside their inputs in one buffer: columns that do not meet are
written as if they were tensors of their own, columns that do are refused."""
import pytest
import torch

import serving_reference as ref
from sm120_rmsnorm import extensions, serving

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def columns(rows, heads, d=128, seed=0):
    """Views of consecutive columns of one random buffer, and the buffer."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    whole = torch.randn(rows, sum(heads) * d, device=DEV, generator=g).to(torch.bfloat16)
    views, at = [], 0
    for h in heads:
        views.append(whole[:, at * d:(at + h) * d].view(rows, h, d))
        at += h
    return views, whole


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_output_between_its_inputs(d):
    (q, out, k, v), whole = columns(150, (4, 4, 2, 2), d)
    want, bound = ref.prompt(q, k, v, [0, 100, 140])
    before = whole.clone()
    serving.prompt_attention(out, q, k, v, ints([0, 100, 140]))
    live = ~want.isnan()
    assert ((out.double() - want).abs() <= bound)[live].all()
    out.copy_(before[:, 4 * d:8 * d].view_as(out))
    assert torch.equal(whole, before)  # nothing else was written


def test_prompt_output_over_its_inputs():
    (q, k, v), whole = columns(150, (2, 2, 2))
    before = whole.clone()
    for out, name in ((q, "query"), (k, "key"), (v, "value"), (whole[:, 64:320].view(150, 2, 128), "query")):
        with pytest.raises(RuntimeError, match=f"out may not overlap {name}"):
            serving.prompt_attention(out, q, k, v, ints([0, 150]))
    assert torch.equal(whole, before)


def test_decode_output_beside_and_over_the_query():
    (q, out, k, v), whole = columns(3, (4, 4, 2, 2))
    kc, vc = (torch.randn(9, 16, 2, 128, device=DEV).to(torch.bfloat16) for _ in "kv")
    table = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    want, bound = ref.decode(q, kc, vc, table, [40, 3, 17], None)
    serving.paged_decode_attention(out, q, kc, vc, table, ints([40, 3, 17]))
    assert ((out.double() - want).abs() <= bound).all()
    with pytest.raises(RuntimeError, match="out may not overlap query"):
        serving.paged_decode_attention(whole[:, 256:768].view(3, 4, 128), q, kc, vc, table,
                                       ints([40, 3, 17]))
    with pytest.raises(RuntimeError, match="out may not overlap value_cache"):
        serving.paged_decode_attention(vc.view(-1)[:3 * 512].view(3, 4, 128), q, kc, vc, table,
                                       ints([40, 3, 17]))


def test_rotation_beside_and_over_its_inputs():
    (q, k, v, q_out, k_out), whole = columns(20, (4, 2, 2, 4, 2))
    w = torch.ones(128, device=DEV, dtype=torch.bfloat16)
    places = torch.arange(20, device=DEV).expand(3, -1)
    table = torch.randn(64, 128, device=DEV)

    def run(query, key, **kw):
        extensions.qk_norm_mrope_cache_(query, key, v, w, w, places, table, [16, 24, 24], **kw)

    want = q.clone(), k.clone()
    run(*want)
    before = whole.clone()
    run(q, k, query_out=q_out, key_out=k_out)
    assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1])
    assert torch.equal(whole[:, :8 * 128], before[:, :8 * 128])
    for kw, name in ((dict(query_out=whole[:, 64:576].view(20, 4, 128)), "its input"),
                     (dict(key_out=q[:, :2]), "query"), (dict(query_out=q_out, key_out=q_out[:, 1:3]), "key_out"),
                     (dict(query_out=whole[:, 256:768].view(20, 4, 128)), "its input")):
        with pytest.raises(RuntimeError, match=f"may not overlap {name}"):
            run(q, k, **kw)
    run(q, k, query_out=q, key_out=k)  # in place, said twice
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rotation_of_keys_that_are_the_values_too(d):
    """In place, with value the same rows as key: the cache gets the values as they were."""
    (q, k, v), whole = columns(20, (4, 2, 2), d)
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    places = torch.arange(20, device=DEV).expand(3, -1)
    table = torch.randn(64, d, device=DEV)
    slots = torch.randperm(48, device=DEV)[:20].to(torch.int32)
    results = []
    for shared in (False, True):
        key = k.clone()
        caches = [torch.zeros(3, 16, 2, d, device=DEV, dtype=torch.bfloat16) for _ in "kv"]
        extensions.qk_norm_mrope_cache_(q.clone(), key, key if shared else k, w, w, places, table,
                                        [d // 4, d // 8, d // 8], *caches, slots)
        results.append((key, *caches))
    for apart, together in zip(*results):
        assert torch.equal(apart, together)
    assert torch.equal(results[1][2].view(48, 2, d)[slots.long()], k)
