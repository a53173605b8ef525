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
