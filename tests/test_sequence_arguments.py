"""What the sequence ops hand to the entry points, looked at on the host: the
calls are recorded instead of made, on tensors without memory."""
import pytest
import torch

from zerograd_b200 import _lib as L
from zerograd_b200 import _sequence

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(_sequence, "_device", lambda *ts: ts[0].device)
    monkeypatch.setattr(_sequence, "_call", lambda dev, name, *args: made.append((name, args)))
    return made


def _meta(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_rotary_of_two_types_keeps_both(calls):
    """Queries and keys of different types come back each in its own, neither cast to the other's."""
    pos = torch.zeros(5, 1, dtype=torch.int32)
    for a, b in ((BF, F32), (F32, BF)):
        calls.clear()
        q, k = _sequence.rotary(torch.zeros(2, 5, 4, 64, dtype=a), torch.zeros(2, 5, 2, 64, dtype=b), pos, (64,))
        assert q.dtype is a and k.dtype is b and q.shape == (2, 5, 4, 64) and k.shape == (2, 5, 2, 64)
        # one launch for each: query and key heads, type
        assert [(c[8], c[9], c[-3]) for _, c in calls] == [(4, 0, L.dtype_code(a)), (0, 2, L.dtype_code(b))]
    with pytest.raises(TypeError):
        _sequence.rotary(torch.zeros(2, 5, 4, 64, dtype=a), torch.zeros(2, 5, 2, 64, dtype=torch.half), pos, (64,))
