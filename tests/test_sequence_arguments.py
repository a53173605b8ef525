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


def test_sizes_beyond_32_bits_are_refused(calls):
    """An axis, a page size, a table or heads of 2^32 and a few are not taken for the few."""
    wide = 2 ** 32
    q, k, pos = _meta(2, 5, 4, 64), _meta(2, 5, 2, 64), torch.zeros(5, 1, dtype=torch.int32)
    table, n = _meta(2, 3, dtype=torch.int32), _meta(2, dtype=torch.int32)
    pool = _meta(4, 8, 2, 64)
    for call in (lambda: _sequence.rotary(q, k, pos, (wide + 64,)),
                 lambda: _sequence.rotary(q, k, pos, (64 - wide,)),
                 lambda: _sequence.rotary(_meta(1, 1, wide + 4, 64), k[:1, :1], pos[:1], (64,)),
                 lambda: _sequence.window_attention(_meta(1, 1, wide + 4, 64), k[:1, :1], k[:1, :1]),
                 lambda: _sequence.window_attention(*[_meta(1, 1, 1, wide + 64)] * 3),
                 lambda: _sequence.append_pages(*[_meta(1, wide + 8, 2, 64)] * 2, k, k, table, n),
                 lambda: _sequence.append_pages(pool, pool, k, k, _meta(2, wide + 1, dtype=torch.int32), n),
                 lambda: _sequence.paged_attention(q[:, 0], *[_meta(1, wide + 8, 2, 64)] * 2, table, n),
                 lambda: _sequence.paged_attention(_meta(2, wide + 4, 64), pool, pool, table, n)):
        with pytest.raises(ValueError):
            call()
    assert not calls


def test_negated_views_take_the_dispatcher():
    """A tensor whose memory does not hold its values is not read as it lies
    there, nor in a vmap rule one without memory."""
    x = torch.ones(2, 3)
    assert _sequence._plain_call(x) and not _sequence._plain_call(x, torch._neg_view(x))
    m = _sequence._mapped(torch._neg_view(x), 1)
    assert not m.is_neg() and m.tolist() == [[-1.0, -1.0]] * 3
    m = _sequence._mapped(torch._efficientzerotensor((2,)), None, 4)
    assert m.shape == (4, 2) and not m._is_zerotensor() and m.sum() == 0
    assert _sequence._mapped(None, None, 4) is None


def test_paged_attention_copies_queries_for_the_tensor_cores_alone(calls, monkeypatch):
    """A float32 q of odd pitch, or bf16 with D not a multiple of 8, reaches the entry point as it is."""
    monkeypatch.setattr(_sequence, "_paged_workspace", lambda *sizes: 0)
    table, n = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for dtype, D, copied in ((F32, 7, False), (F32, 8, False), (BF, 7, False), (BF, 8, True)):
        pool = torch.zeros(1, 4, 1, D, dtype=dtype)
        q = torch.zeros(2, D + 1, dtype=dtype)[:, :D].unflatten(-1, (1, D)) if D % 2 == 0 else torch.zeros(2, 1, D, dtype=dtype)
        calls.clear()
        _sequence.paged_attention(q, pool, pool, table, n)
        (_, args), = calls
        assert (args[0] != q.data_ptr()) == copied and args[1] == (D if copied else q.stride(0)), (dtype, D)


def test_window_attention_of_more_heads_than_a_grid_counts():
    """Sequences times heads beyond 31 bits are refused before their product with the tiles wraps."""
    for Z, S, H, K, D in ((2 ** 31 - 1, 2 ** 30, 2 ** 30, 1, 4), (2 ** 30, 256, 8, 8, 64)):
        assert L.load().zg_window_attention(None, H * D, None, K * D, None, K * D, None, Z, S, H, K, D, 0, 0, L.ZG_BF16, None,
                                            None) == L.ZG_ERR_INVALID
        assert b"bad sizes" in L.load().zg_last_error()
