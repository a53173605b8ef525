"""Calls of the sequence ops that their documentation allows, against the
calls of contiguous tensors of one type."""
import math

import pytest
import torch

import sequence_oracle as so
import zerograd_b200 as zg
from zerograd_b200 import _lib as L

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _rand(shape, dtype, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, generator=g, device=device).to(dtype)


@pytest.mark.parametrize("types", [(BF, F32), (F32, BF)])
def test_rotary_of_two_types(cuda, types):
    """Each result has its own type, with the bits of a call of that type."""
    q, k = _rand((2, 7, 4, 64), types[0], 1, cuda), _rand((2, 7, 2, 64), types[1], 2, cuda)
    pos = torch.arange(7, device=cuda)[:, None] + 5000
    a, b = zg.rotary(q, k, pos, (64,))
    assert a.dtype is types[0] and b.dtype is types[1]
    assert torch.equal(a, zg.rotary(q, k.to(types[0]), pos, (64,))[0])
    assert torch.equal(b, zg.rotary(q.to(types[1]), k, pos, (64,))[1])
    va, vb = torch.func.vmap(lambda x, y: zg.rotary(x, y, pos, (64,)))(q, k)
    assert torch.equal(va, a) and torch.equal(vb, b)


def test_negated_views(cuda):
    """Views with the negative bit, called one by one and under vmap, count with their sign."""
    g = [_rand((2, 9, 2, 64), F32, s, cuda) for s in range(3)]
    pos = torch.arange(9, device=cuda)[:, None]
    table, n = torch.tensor([[2, 0], [1, 3]], device=cuda), torch.tensor([9, 4], device=cuda)
    pool = [_rand((4, 8, 2, 64), F32, s, cuda) for s in (4, 5)]

    def fresh():
        return [t.clone() for t in pool]

    def run(q, k, v, kp, vp, wk, wv):
        return (*zg.rotary(q, k, pos, (64,)), zg.window_attention(q, k, v), zg.paged_attention(q[:, 0], kp, vp, table, n),
                zg.append_pages(wk, wv, k, v, table, torch.zeros_like(n)))

    neg = torch._neg_view
    w1, w2 = fresh(), fresh()
    want = run(*(-t for t in g), *(-t for t in pool), *w1)
    for a, b in zip(run(*map(neg, g), *map(neg, pool), *w2), want):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(w1, w2))
    both = torch.func.vmap(lambda q, k, v: (*zg.rotary(q, k, pos, (64,)), zg.window_attention(q, k, v)))
    for a, b in zip(both(*map(neg, g)), want):
        assert torch.equal(a, b)
    one = torch.func.vmap(lambda q, t, m: zg.paged_attention(q, neg(pool[0]), neg(pool[1]), t, m))
    assert torch.equal(one(neg(g[0][:, 0]), table, n), want[3])
    w3 = fresh()
    put = torch.func.vmap(lambda k, v, t, m: zg.append_pages(*w3, k, v, t, m))
    put(neg(g[1]), neg(g[2]), table, torch.zeros_like(n))
    assert all(torch.equal(a, b) for a, b in zip(w1, w3))
    with pytest.raises(ValueError):
        torch.func.vmap(lambda k, t, m: zg.append_pages(neg(pool[0]), neg(pool[1]), k, k, t, m))(g[1], table, n)
