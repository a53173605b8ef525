"""Argument checks of the sequence ops' entry points, made on the host before any launch."""
import ctypes

import pytest
import torch

from zerograd_b200 import _lib as L
from zerograd_b200 import _sequence


def _axes(*widths):
    return (ctypes.c_int32 * len(widths))(*widths)


def _rotary(T=0, H=2, K=1, D=64, axes=(64,), ldq=None, ldk=None, base=1e4, pos_type=1, pos_rows=1, dtype=L.ZG_BF16,
            q=None):
    return L.load().zg_rotary(q, ldq if ldq is not None else H * D, q, ldk if ldk is not None else K * D, q, pos_type, T,
                              pos_rows, H, K, D, len(axes), _axes(*axes), base, 0, 0, 0, dtype, q, q, None)


def test_rotary_arguments():
    assert _rotary() == L.ZG_OK  # no tokens
    for bad in (dict(T=-1), dict(D=1), dict(axes=(63,)), dict(axes=(0, 64)), dict(axes=(40, 40)), dict(ldq=100),
                dict(ldk=63), dict(base=0.0), dict(base=float("inf")), dict(pos_type=3), dict(dtype=7), dict(H=0, K=0),
                dict(H=-1)):
        assert _rotary(**bad) == L.ZG_ERR_INVALID, bad
    assert _rotary(D=258) == L.ZG_ERR_UNSUPPORTED
    assert _rotary(T=6, pos_rows=4) == L.ZG_ERR_INVALID and b"divide" in L.load().zg_last_error()
    assert _rotary(T=6, pos_rows=3) == L.ZG_ERR_INVALID and b"null" in L.load().zg_last_error()


def _window(Z=0, S=8, H=4, K=2, D=64, window=0, sinks=0, dtype=L.ZG_BF16, ldq=None, ldk=None):
    return L.load().zg_window_attention(None, ldq or H * D, None, ldk or K * D, None, K * D, None, Z, S, H, K, D, window,
                                        sinks, dtype, None, None)


def test_window_attention_arguments():
    assert _window() == L.ZG_OK and _window(Z=1, S=0) == L.ZG_OK
    for bad in (dict(Z=-1), dict(S=-1), dict(H=3), dict(K=0), dict(D=0), dict(window=-1), dict(sinks=-1), dict(dtype=9),
                dict(ldq=255), dict(ldk=127), dict(Z=1)):
        assert _window(**bad) == L.ZG_ERR_INVALID, bad
    assert _window(D=257) == L.ZG_ERR_UNSUPPORTED


def _append(B=0, S=1, N=4, page=16, K=2, D=64, M=3, dtype=L.ZG_BF16, ldk=None):
    return L.load().zg_append_pages(None, None, N, page, K, D, None, ldk or K * D, None, K * D, B, S, None, M, None, None,
                                    dtype, None, None)


def test_append_pages_arguments():
    assert _append() == L.ZG_OK
    for bad in (dict(B=-1), dict(S=-1), dict(N=-1), dict(page=0), dict(K=0), dict(D=0), dict(M=-1), dict(dtype=2),
                dict(ldk=127), dict(M=1 << 20, page=1 << 20), dict(B=1)):
        assert _append(**bad) == L.ZG_ERR_INVALID, bad


def _paged(B=0, N=4, page=16, M=3, H=4, K=2, D=64, window=0, sinks=0, dtype=L.ZG_BF16, ldq=None):
    return L.load().zg_paged_attention(None, ldq or H * D, None, None, N, page, None, M, None, B, H, K, D, window, sinks,
                                       dtype, None, None, 0, None)


def test_paged_attention_arguments():
    assert _paged() == L.ZG_OK
    for bad in (dict(B=-1), dict(N=-1), dict(page=0), dict(H=3), dict(H=0), dict(K=0), dict(D=0), dict(window=-1),
                dict(sinks=-1), dict(dtype=5), dict(ldq=255), dict(B=1), dict(N=1 << 20, page=1 << 12),
                dict(M=1 << 20, page=1 << 12)):
        assert _paged(**bad) == L.ZG_ERR_INVALID, bad
    assert _paged(D=264) == L.ZG_ERR_UNSUPPORTED


def test_paged_attention_workspace():
    size = L.load().zg_paged_attention_workspace_size
    bf, f32 = L.ZG_BF16, L.ZG_F32
    # a cluster joins up to eight splits: no workspace
    assert size(64, 12, 12, 64, 250, 16, 0, 0, bf) == 0 and size(8, 16, 4, 128, 500, 32, 1000, 4, bf) == 0
    # one sequence of 131072 positions over 4 key heads: 74 splits of 16 rows of 128, their maxima and sums
    assert size(1, 16, 4, 128, 2048, 64, 0, 0, bf) >= 4 * 74 * 16 * 130 * 4
    assert size(1, 16, 4, 128, 2048, 64, 0, 0, f32) > 0
    assert size(1, 16, 3, 128, 2048, 64, 0, 0, bf) == 0 and size(1, 16, 4, 512, 2048, 64, 0, 0, bf) == 0
    assert size(0, 16, 4, 128, 2048, 64, 0, 0, bf) == 0 and size(1, 16, 4, 128, 0, 64, 0, 0, bf) == 0


def test_rows_with_a_pitch():
    """What the kernels take as it is, and what is copied first (the same on any device)."""
    x = torch.arange(2 * 6 * 5 * 8).reshape(2, 6, 5, 8)
    assert _sequence._pitched(x)[1] == 40 and _sequence._pitched(x[:, :, 1:3])[1] == 40
    assert _sequence._pitched(x[:, :1, :2])[1] == 240
    y, ld = _sequence._pitched(x[:, :, ::2])
    assert y.is_contiguous() and ld == 24
    assert _sequence._pitched(x[:0])[1] >= 40
    assert _sequence._pitched(x[:, :, :, :3])[1] == 15  # heads apart: copied


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(L.ZgLibraryError):
        _sequence.window_attention(x, x, x)
    with pytest.raises(L.ZgLibraryError):
        _sequence.rotary(x, x, torch.zeros(2, 1, dtype=torch.int32), (8,))
    with pytest.raises(ValueError):
        _sequence.window_attention(x, x, x, window=0)


def test_plain_calls_skip_the_dispatcher():
    x = torch.zeros(2)
    assert _sequence._plain_call(x, None)
    assert not _sequence._plain_call(x, torch.zeros(2, requires_grad=True))
    with torch.no_grad():
        assert _sequence._plain_call(torch.zeros(2, requires_grad=True))
    seen = []
    torch.func.vmap(lambda t: seen.append(_sequence._plain_call(x)) or t)(torch.zeros(3))
    assert seen == [False]


def test_a_call_is_made_with_its_tensors_device_current(monkeypatch):
    current, made = [0], []

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            current.append(self.dev.index)

        def __exit__(self, *exc):
            current.pop()

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(L, "stream_ptr", lambda dev: ("stream of", dev.index))
    monkeypatch.setattr(L, "call", lambda name, *args: made.append((name, current[-1], args)))
    _sequence._call(torch.device("cuda", 0), "f", 1)
    _sequence._call(torch.device("cuda", 3), "g", 2, 3)
    assert made == [("f", 0, (1, ("stream of", 0))), ("g", 3, (2, 3, ("stream of", 3)))] and current == [0]
