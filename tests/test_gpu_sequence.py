"""Rotary positions, windowed attention and the paged cache against plain
float64 forms, at the sizes and masks where they can go wrong.  The bounds
are derived in ``sequence_oracle``."""
import math

import pytest
import torch

import sequence_oracle as so
import zerograd_b200 as zg
from zerograd_b200 import _lib as L

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _rand(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _ok():
    torch.cuda.synchronize()
    assert L.load().zg_device_error(1) == 0


# ------------------------------------------------------------------- rotary


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("joint,inverse", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("lead,S,H,K,D,axes", [
    ((2,), 5, 3, 1, 64, (64,)),
    ((), 1, 12, 4, 64, (64,)),
    ((3, 2), 7, 4, 2, 128, (32, 48, 48)),
    ((1,), 63, 6, 6, 72, (36, 36)),
    ((2,), 9, 2, 2, 80, (16, 8)),      # columns behind the pairs stay
    ((2,), 3, 2, 1, 10, (2, 6)),       # no 16-byte words
    ((300,), 4, 1, 1, 256, (256,)),
])
def test_rotary(cuda, dtype, interleaved, joint, inverse, lead, S, H, K, D, axes):
    g = torch.Generator().manual_seed(S * D + H)
    x = _rand((*lead, S, H + 2 * K, D), dtype, g)
    pos = torch.randint(0, 200000, (S, len(axes)), generator=g)
    xc = x.to(cuda)
    q, k = zg.rotary(xc[..., :H, :], xc[..., H:H + K, :], pos.to(cuda), axes, interleaved=interleaved, joint=joint,
                     inverse=inverse)
    want = so.rotary(x[..., :H, :], x[..., H:H + K, :], pos, axes, 10000.0, interleaved, joint, inverse)
    for got, (w, size), name in ((q, want[0], "q"), (k, want[1], "k")):
        assert got.dtype == dtype and got.is_contiguous()
        so.assert_within(got, w, so.rotary_tolerance(w, size, dtype), name)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_rotary_positions_per_sequence(cuda, kind):
    g = torch.Generator().manual_seed(1)
    q, k = _rand((3, 4, 5, 2, 32), F32, g), _rand((3, 4, 5, 1, 32), F32, g)
    for shape in ((5, 2), (4, 5, 2), (3, 4, 5, 2)):
        pos = torch.randint(-1000, 1 << 20, shape, generator=g).to(kind)
        if kind == torch.float32:
            pos = pos / 8
        got = zg.rotary(q.to(cuda), k.to(cuda), pos.to(cuda), (20, 12), base=500.0)
        for y, (w, size) in zip(got, so.rotary(q, k, pos, (20, 12), 500.0)):
            so.assert_within(y, w, so.rotary_tolerance(w, size, F32), str(shape))


def test_rotary_inverse_is_the_transpose(cuda):
    """<R q, y> = <q, R' y>, and R' R = 1, within float32's roundings."""
    g = torch.Generator().manual_seed(2)
    q, k, y = (_rand((2, 6, 3, 48), F32, g).to(cuda) for _ in range(3))
    pos = torch.randint(0, 5000, (6, 3), generator=g).to(cuda)
    r, _ = zg.rotary(q, k, pos, (16, 16, 16), joint=True)
    back, ry = zg.rotary(r, y, pos, (16, 16, 16), joint=True, inverse=True)
    assert (back - q).abs().max() < 4 * 2.0 ** -21 * q.abs().max()
    lhs, rhs = (r.double() * y.double()).sum(), (q.double() * ry.double()).sum()
    assert abs(lhs - rhs) < 4 * 2.0 ** -21 * (q.double().norm() * y.double().norm())


def test_rotary_of_nothing(cuda):
    q = torch.empty(0, 5, 2, 32, device=cuda)
    a, b = zg.rotary(q, q, torch.zeros(5, 1, dtype=torch.int64, device=cuda), (32,))
    assert a.shape == b.shape == q.shape


# --------------------------------------------------------- window attention

WINDOW_CASES = [
    # Z, S, H, K, D, window, sinks, ragged
    (1, 1, 1, 1, 64, None, 0, False),
    (2, 17, 4, 2, 64, None, 0, False),
    (2, 128, 2, 2, 64, None, 0, False),
    (1, 129, 2, 1, 128, 1, 0, False),      # each token sees itself alone
    (1, 300, 3, 1, 128, 1, 4, False),
    (2, 256, 4, 4, 64, 64, 4, False),
    (2, 511, 2, 2, 64, 127, 0, True),
    (1, 640, 6, 2, 128, 200, 130, True),   # sinks over more than one tile
    (3, 333, 2, 1, 128, 100, 3, True),
    (1, 777, 2, 2, 80, 200, 3, True),
    (2, 400, 2, 1, 40, None, 0, True),
    (1, 1100, 2, 1, 96, 257, 1, False),
    (1, 900, 1, 1, 64, 899, 1, False),
    (1, 900, 1, 1, 64, 5000, 9000, False),  # wider than the sequence
    (70, 40, 5, 1, 32, 16, 2, True),
    (2, 150, 2, 2, 20, 33, 2, True),        # no 16-byte rows: the FMA path in bf16 too
    (2, 150, 4, 2, 256, 33, 2, True),
    (1, 70, 1, 1, 3, None, 0, False),
]


def _lengths(Z, S):
    return torch.tensor([(S, 0, 1, S // 2 + 1, max(S - 1, 0))[z % 5] for z in range(Z)], dtype=torch.int32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Z,S,H,K,D,window,sinks,ragged", WINDOW_CASES)
def test_window_attention(cuda, dtype, Z, S, H, K, D, window, sinks, ragged):
    g = torch.Generator().manual_seed(S * D + H)
    x = _rand((Z, S, H + 2 * K, D), dtype, g)
    q, k, v = x[:, :, :H], x[:, :, H:H + K], x[:, :, H + K:]
    lengths = _lengths(Z, S) if ragged else None
    xc = x.to(cuda)
    o = zg.window_attention(xc[:, :, :H], xc[:, :, H:H + K], xc[:, :, H + K:], window, sinks,
                            None if lengths is None else lengths.to(cuda))
    _ok()
    assert o.dtype == dtype and o.is_contiguous()
    want, mag = so.window_attention(q, k, v, window, sinks, lengths)
    so.assert_within(o, want, so.attention_tolerance(q, k, want, mag, dtype, S))


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (BF, 20)])
def test_window_attention_masked_places_hold_anything(cuda, dtype, D):
    """Infinities, NaN and the type's lowest value behind a sequence and in
    positions that a row does not see leave it as it is."""
    Z, S, H, K, window, sinks = 2, 300, 2, 1, 50, 2
    g = torch.Generator().manual_seed(5)
    q, k, v = _rand((Z, S, H, D), dtype, g), _rand((Z, S, K, D), dtype, g), _rand((Z, S, K, D), dtype, g)
    lengths = torch.tensor([190, 300], dtype=torch.int32)
    want, mag = so.window_attention(q, k, v, window, sinks, lengths)
    low = torch.finfo(dtype).min
    for at, t in ((200, q), (230, k), (260, k)):
        t[0, at:at + 20] = math.nan if at != 260 else low
    k[0, 191], v[0, 191], v[0, 192], v[0, 255] = math.inf, math.nan, -math.inf, low
    # position 100 of sequence 1: seen by rows 100 .. 149 alone
    v[1, 100, 0, 3], k[1, 101] = math.nan, 0
    want1, mag1 = so.window_attention(q[1:], k[1:], v[1:], window, sinks)
    want[1:], mag[1:] = want1, mag1
    o = zg.window_attention(*(t.to(cuda) for t in (q, k, v)), window, sinks, lengths.to(cuda))
    _ok()
    assert torch.isnan(o[1, 100:150, :, 3]).all() and int(torch.isnan(o).sum()) == 50 * H
    tol = so.attention_tolerance(q, torch.where(k.double().abs() < 1e3, k, 0), want, mag, dtype, S)
    so.assert_within(o, want, tol)


def test_window_attention_bad_lengths(cuda):
    q = torch.ones(3, 5, 2, 64, device=cuda, dtype=BF)
    o = zg.window_attention(q, q, q, lengths=torch.tensor([-1, 6, 3], device=cuda))
    assert torch.isnan(o[:2]).all() and (o[2, :3] == 1).all() and (o[2, 3:] == 0).all()


def test_window_attention_large_scores(cuda):
    """Scores to several hundred, the largest coming late: the running maximum moves."""
    g = torch.Generator().manual_seed(6)
    S, D = 600, 64
    q, k, v = (_rand((1, S, 2, D), BF, g, 3) for _ in range(3))
    k *= torch.linspace(0.1, 6, S)[None, :, None, None].to(BF)
    o = zg.window_attention(*(t.to(cuda) for t in (q, k, v)), 400, 2)
    want, mag = so.window_attention(q, k, v, 400, 2)
    so.assert_within(o, want, so.attention_tolerance(q, k, want, mag, BF, S))


# -------------------------------------------------------------- paged cache


def _pool(lengths, page, K, D, dtype, g, spare=3):
    need = [-(-n // page) for n in lengths]
    n = sum(need) + spare
    kp, vp = _rand((n, page, K, D), dtype, g), _rand((n, page, K, D), dtype, g)
    order = torch.randperm(n, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1])), -7, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return kp, vp, table


PAGED_CASES = [
    # lengths, H, K, D, page, window, sinks
    ([1], 1, 1, 64, 16, None, 0),
    ([0, 1, 15, 16, 17], 4, 2, 64, 16, None, 0),
    ([700], 12, 4, 128, 16, None, 0),
    ([3000, 10, 2047], 4, 1, 128, 64, None, 0),
    ([3000, 10, 2047], 4, 4, 64, 24, 100, 4),
    ([5000, 1], 2, 1, 128, 1, 1, 0),
    ([1500, 64, 200], 40, 2, 64, 8, None, 0),     # 20 heads of a key head: two row tiles
    ([900, 333], 16, 1, 80, 16, 512, 1),
    ([900, 333], 3, 3, 256, 128, None, 0),
    ([400, 333, 77], 5, 1, 20, 16, 300, 2),       # no 16-byte rows in bf16
    ([60, 3], 2, 2, 7, 5, None, 0),
    ([40000], 8, 8, 32, 256, None, 0),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,H,K,D,page,window,sinks", PAGED_CASES)
def test_paged_attention(cuda, dtype, lengths, H, K, D, page, window, sinks):
    g = torch.Generator().manual_seed(sum(lengths) + D)
    kp, vp, table = _pool(lengths, page, K, D, dtype, g)
    n = torch.tensor(lengths, dtype=torch.int32)
    q = _rand((len(lengths), H, D), dtype, g)
    want, mag = so.paged_attention(q, kp, vp, table, n, window, sinks)
    tol = so.attention_tolerance(q, kp, want, mag, dtype, max(lengths))
    # what lies behind a sequence, in its last page and in pages of nobody, is not read
    seen = torch.zeros(kp.shape[:2], dtype=torch.bool)
    for b, m in enumerate(lengths):
        j = torch.arange(m)
        if window is not None:
            j = j[(j >= m - window) | (j < sinks)]
        seen[table[b].long()[j // page], j % page] = True
    kp[~seen], vp[~seen] = math.nan, math.inf
    o = zg.paged_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), n.to(cuda), window, sinks)
    torch.cuda.synchronize()
    assert o.dtype == dtype
    so.assert_within(o, want, tol)
    again = zg.paged_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda).long(), n.to(cuda).long(), window,
                               sinks)
    assert torch.equal(o, again)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_paged_attention_bad_pages_and_lengths(cuda, dtype):
    """A page outside the pool or a length outside the table gives that sequence NaN."""
    g = torch.Generator().manual_seed(3)
    lengths = [900, 900, 900, 40, 900, 900]
    kp, vp, table = _pool(lengths, 16, 2, 64, dtype, g)
    q = _rand((6, 4, 64), dtype, g)
    table[0, 30], table[1, 2] = -1, kp.shape[0]
    n = torch.tensor(lengths, dtype=torch.int32)
    n[4], n[5] = -1, table.shape[1] * 16 + 1
    o = zg.paged_attention(q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), n.to(cuda))
    assert torch.isnan(o[[0, 1, 4, 5]]).all()
    want, mag = so.paged_attention(q[2:4], kp, vp, table[2:4], n[2:4])
    so.assert_within(o[2:4], want, so.attention_tolerance(q, kp, want, mag, dtype, 900))
    # the bad entries do not matter where the token does not see them
    o = zg.paged_attention(q[:2].to(cuda), kp.to(cuda), vp.to(cuda), table[:2].to(cuda), n[:2].to(cuda), 100, 3)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("S,K,D,page", [(1, 4, 128, 16), (37, 2, 64, 16), (5, 1, 3, 4), (130, 2, 20, 1), (9, 12, 64, 64)])
def test_append_pages(cuda, dtype, S, K, D, page):
    g = torch.Generator().manual_seed(S + D)
    had = [0, 3, page, 2 * page - 1, 50]
    counts = [S, S // 2, 0, S, 1]
    kp, vp, table = _pool([h + S for h in had], page, K, D, dtype, g)
    x = _rand((5, S, 2 * K, D), dtype, g)
    k, v = x[:, :, :K], x[:, :, K:]
    wk, wv = kp.clone(), vp.clone()
    for b in range(5):
        for s in range(counts[b]):
            at = had[b] + s
            wk[table[b, at // page], at % page], wv[table[b, at // page], at % page] = k[b, s], v[b, s]
    ck, cv, xc = kp.to(cuda), vp.to(cuda), x.to(cuda)
    n = torch.tensor(had, device=cuda)
    new = zg.append_pages(ck, cv, xc[:, :, :K], xc[:, :, K:], table.to(cuda), n, torch.tensor(counts, device=cuda))
    assert new.tolist() == [h + c for h, c in zip(had, counts)] and n.tolist() == had
    assert torch.equal(ck.cpu(), wk) and torch.equal(cv.cpu(), wv)


def test_append_pages_that_do_not_fit(cuda):
    """Nothing is written past a table's row, for bad lengths and counts, or to a page outside the pool."""
    page, K, D, S = 4, 1, 64, 6
    kp = torch.zeros(8, page, K, D, device=cuda, dtype=BF)
    vp = torch.zeros_like(kp)
    table = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 7], [-1, 7], [6, 8]], dtype=torch.int32, device=cuda)
    x = torch.ones(6, S, K, D, device=cuda, dtype=BF)
    had = torch.tensor([0, 3, -1, 0, 2, 2], device=cuda)
    counts = torch.tensor([6, 6, 1, 7, 3, 3], device=cuda)
    new = zg.append_pages(kp, vp, x, x, table, had, counts)
    assert new.tolist() == [6, -1, -1, -1, -1, -1]
    filled = kp.float().sum((2, 3)) / D
    want = torch.zeros(8, page, device=cuda)
    want[0], want[1, :2] = 1, 1
    want[7, 0] = 1      # the token of sequence 4 whose page is one of the pool's
    want[6, 2:] = 1     # those of sequence 5
    assert torch.equal(filled, want) and torch.equal(kp, vp)
    o = zg.paged_attention(torch.ones(6, 2, D, device=cuda, dtype=BF), kp, vp, table, new)
    assert (o[0] == 1).all() and torch.isnan(o[1:]).all()


# ------------------------------------------------------- a run of them together


@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 48)])
def test_prompt_and_tokens(cuda, dtype, D):
    """A padded batch's prompt (rotary, windowed attention, append) and then
    token after token (rotary, append, paged attention) agree with the windowed
    attention of the whole sequences."""
    B, S, T, H, K, page, window, sinks = 3, 50, 30, 4, 2, 16, 24, 3
    g = torch.Generator().manual_seed(8)
    prompt = torch.tensor([50, 17, 1], dtype=torch.int32)
    x = _rand((B, S + T, H + 2 * K, D), dtype, g).to(cuda)  # a fused projection of the whole sequences
    kp, vp, table = (t.to(cuda) for t in _pool([S + T] * B, page, K, D, dtype, g))
    lengths = prompt.to(cuda)
    pos = torch.arange(S + T, device=cuda)[:, None]
    qr, kr = zg.rotary(x[:, :, :H], x[:, :, H:H + K], pos, (D,))
    v = x[:, :, H + K:]
    whole = zg.window_attention(qr, kr, v, window, sinks)
    o = zg.window_attention(qr[:, :S].contiguous(), kr[:, :S].contiguous(), v[:, :S], window, sinks, lengths)
    n = zg.append_pages(kp, vp, kr[:, :S], v[:, :S], table, torch.zeros_like(lengths), lengths)
    assert torch.equal(n, lengths)
    tol = 2.0 ** -6 if dtype == BF else 2.0 ** -18  # two results of values below 4, each off by its own bound
    for b in range(B):
        assert (o[b, :prompt[b]] - whole[b, :prompt[b]]).abs().max() <= 4 * tol
    rows = torch.arange(B, device=cuda)
    for _ in range(T):
        tok = x[rows, n.long()]
        q1, k1 = zg.rotary(tok[:, None, :H], tok[:, None, H:H + K], n[:, None, None], (D,))
        n = zg.append_pages(kp, vp, k1, tok[:, None, H + K:], table, n)
        o1 = zg.paged_attention(q1[:, 0], kp, vp, table, n, window, sinks)
        want = whole[rows, n.long() - 1]
        assert (o1 - want).abs().max() <= 4 * tol
    assert n.tolist() == [80, 47, 31]


def test_under_vmap(cuda):
    """Each op of a candidate's forward is one launch for the population, with
    the bits of the calls candidate by candidate."""
    P, B, S, H, K, D, page = 3, 2, 20, 4, 2, 64, 8
    g = torch.Generator().manual_seed(9)
    x = _rand((P, B, S, H + 2 * K, D), BF, g).to(cuda)
    kp, vp, table = (t.to(cuda) for t in _pool([S] * (P * B), page, K, D, BF, g))
    table = table.reshape(P, B, -1)
    pos = torch.arange(S, device=cuda)[:, None]
    lengths = torch.tensor([S, 7], dtype=torch.int32, device=cuda)

    def candidate(xx, tt):
        q, k = zg.rotary(xx[:, :, :H], xx[:, :, H:H + K], pos, (32,))
        v = xx[:, :, H + K:]
        o = zg.window_attention(q, k, v, 9, 1, lengths)
        n = zg.append_pages(kp, vp, k, v, tt, torch.zeros_like(lengths), lengths)
        return o, zg.paged_attention(q[:, 0], kp, vp, tt, n, 9, 1), n

    kp0, vp0 = kp.clone(), vp.clone()
    L.profile_begin()
    got = torch.func.vmap(candidate)(x, table)
    prof = L.profile_end()
    assert len(prof) == 4 and all(c == 1 for c, _ in prof.values()), prof
    k1, v1 = kp.clone(), vp.clone()
    kp.copy_(kp0)
    vp.copy_(vp0)
    want = [candidate(x[p], table[p]) for p in range(P)]
    for i in range(3):
        assert torch.equal(got[i], torch.stack([w[i] for w in want]))
    assert torch.equal(kp, k1) and torch.equal(vp, v1)
    # per-candidate positions, the same for each of a candidate's sequences
    shift = torch.arange(P, device=cuda)[:, None, None] * 100 + pos
    a, _ = torch.func.vmap(lambda xx, pp: zg.rotary(xx[:, :, :H], xx[:, :, H:H + K], pp, (32,)))(x, shift)
    b = torch.stack([zg.rotary(x[p, :, :, :H], x[p, :, :, H:H + K], shift[p], (32,))[0] for p in range(P)])
    assert torch.equal(a, b)
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda c: zg.paged_attention(x[0, :, 0, :H], c, c, table[0], lengths))(
            torch.stack([kp, kp]))


def test_views_of_a_fused_projection_are_not_copied(cuda):
    """Rows with a pitch, also of single tokens and through a transposed batch
    of length one, reach the kernels as they are; other strides are copied."""
    from zerograd_b200 import _sequence

    x = torch.arange(4 * 6 * 5 * 8, device=cuda, dtype=F32).reshape(4, 6, 5, 8)
    for t, pitch in ((x[:, :, :2], 40), (x[:, :1, :2], 240), (x[:1, :, 1:3], 40), (x[0, 0, 1:3], 16), (x[:, 2:3, 4:], 240),
                     (x.reshape(24, 5, 8)[:, :3], 40), (x[::2, :, :2], None), (x[:, ::2, :2], 80),
                     (x[:, :, ::2], None), (x[..., :4], None), (x[:1].expand(3, 6, 5, 8)[:, :, :2], None),
                     (x.transpose(0, 1), None), (x[:, :, 1:2, :3], 40)):
        y, ld = _sequence._pitched(t)
        assert (y.data_ptr() == t.data_ptr()) == (pitch is not None), tuple(t.shape)
        assert ld == (pitch if pitch is not None else t.shape[-2] * t.shape[-1])
        assert torch.equal(y, t)


# ------------------------------------------- larger calls, streams, graphs, refusals


@pytest.mark.parametrize("Z,S,H,K,D,window,sinks,ragged,dtype", [
    (2, 1500, 40, 8, 64, None, 0, False, BF),    # several units a CTA, of all lengths
    (3, 1300, 40, 5, 128, 300, 70, True, BF),
    (1, 5000, 3, 1, 64, 1000, 4, False, BF),
    (1, 5000, 3, 1, 128, 4999, 1, False, BF),
    (150, 130, 4, 2, 64, 60, 1, True, BF),
    (2, 1500, 6, 6, 96, 500, 2, True, F32),
])
def test_window_attention_many_units(cuda, Z, S, H, K, D, window, sinks, ragged, dtype):
    g = torch.Generator(device=cuda).manual_seed(S + D)
    x = torch.randn(Z, S, H + 2 * K, D, generator=g, device=cuda).to(dtype)
    q, k, v = x[:, :, :H], x[:, :, H:H + K], x[:, :, H + K:]
    lengths = _lengths(Z, S).to(cuda) if ragged else None
    o = zg.window_attention(q, k, v, window, sinks, lengths)
    _ok()
    want, mag = so.window_attention(q, k, v, window, sinks, lengths)
    so.assert_within(o, want.cpu(), so.attention_tolerance(q, k, want, mag, dtype, S).cpu())
    for _ in range(20):  # the same bits whatever the order the blocks run in
        assert torch.equal(zg.window_attention(q, k, v, window, sinks, lengths), o)
    _ok()


@pytest.mark.parametrize("B,L,H,K,D,page,window,dtype", [
    (1, 70000, 8, 2, 128, 64, None, BF),    # more splits than a cluster holds: a kernel of its own joins them
    (3, 20000, 4, 1, 64, 16, None, BF),
    (40, 900, 12, 6, 192, 32, 500, BF),
    (2, 9000, 10, 1, 96, 16, None, F32),
    (5, 3000, 3, 3, 200, 8, 2000, F32),
])
def test_paged_attention_long(cuda, B, L, H, K, D, page, window, dtype):
    g = torch.Generator().manual_seed(L + D)
    lengths = [L - (3 * L * b) // (4 * B) for b in range(B)]
    kp, vp, table = _pool(lengths, page, K, D, dtype, g)
    q = _rand((B, H, D), dtype, g)
    n = torch.tensor(lengths, dtype=torch.int32)
    want, mag = so.paged_attention(q, kp, vp, table, n, window, 3)
    args = tuple(t.to(cuda) for t in (q, kp, vp, table, n))
    o = zg.paged_attention(*args, window, 3)
    so.assert_within(o, want, so.attention_tolerance(q, kp, want, mag, dtype, L))
    for _ in range(5):
        assert torch.equal(zg.paged_attention(*args, window, 3), o)


def _step(cuda, dtype=BF, S=200, D=64):
    """A step's inputs and the call of it."""
    g = torch.Generator(device=cuda).manual_seed(4)
    B, H, K, page = 3, 4, 2, 16
    x = torch.randn(B, S, H + 2 * K, D, generator=g, device=cuda).to(dtype)
    kp = torch.zeros(3 * 32, page, K, D, device=cuda, dtype=dtype)
    vp = torch.zeros_like(kp)
    table = torch.randperm(96, generator=torch.Generator().manual_seed(1)).reshape(3, 32).to(cuda, torch.int32)
    lengths = torch.tensor([S, 17, 0], dtype=torch.int32, device=cuda)
    pos = torch.arange(S, device=cuda)[:, None]

    def run():
        q, k = zg.rotary(x[:, :, :H], x[:, :, H:H + K], pos, (D,))
        o = zg.window_attention(q, k, x[:, :, H + K:], 50, 2, lengths)
        n = zg.append_pages(kp, vp, k, x[:, :, H + K:], table, torch.zeros_like(lengths), lengths)
        return o, n, zg.paged_attention(q[:, 0], kp, vp, table, n)

    return x, kp, run


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 40)])
def test_captured_and_replayed(cuda, dtype, D):
    """The run of them in a CUDA graph, replayed on new values, twice captured
    at once, gives the bits of the eager calls."""
    x, kp, run = _step(cuda, dtype, D=D)
    run()
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        run()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = run()
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda))
        want = [t.clone() for t in run()]
        for graph, out in graphs:
            kp.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    _ok()


def test_on_two_streams_at_once(cuda):
    x, _, run = _step(cuda, S=300)
    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    steps = [_step(cuda, S=300) for _ in streams]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, (_, _, r) in zip(streams, steps):
            with torch.cuda.stream(s):
                outs.append(r())
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


def test_in_inference_mode_and_with_gradients_asked(cuda):
    """Serving under inference_mode; and an op of tensors that require grad gives
    its values, but has no backward pass (evolution strategies take no gradients)."""
    _, _, run = _step(cuda)
    want = run()
    with torch.inference_mode():
        _, _, again = _step(cuda)
        for a, b in zip(again(), want):
            assert torch.equal(a, b)
    q = torch.randn(1, 5, 2, 64, device=cuda, requires_grad=True)
    o = zg.window_attention(q, q, q)
    assert torch.equal(o.detach(), zg.window_attention(*[q.detach()] * 3))
    with pytest.raises(RuntimeError):
        o.sum().backward()


def test_append_is_seen_as_an_in_place_change(cuda):
    kp = torch.zeros(2, 4, 1, 8, device=cuda)
    v0 = kp._version
    t = torch.ones(1, 1, 1, 8, device=cuda)
    zg.append_pages(kp, torch.zeros_like(kp), t, t, torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                    torch.zeros(1, dtype=torch.int32, device=cuda))
    assert kp._version > v0


def test_refusals(cuda):
    q = torch.zeros(2, 5, 4, 64, device=cuda, dtype=BF)
    k = torch.zeros(2, 5, 2, 64, device=cuda, dtype=BF)
    pos = torch.zeros(5, 1, dtype=torch.int64, device=cuda)
    kp = torch.zeros(4, 8, 2, 64, device=cuda, dtype=BF)
    table = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    n = torch.zeros(2, dtype=torch.int32, device=cuda)
    bad = [
        (ValueError, lambda: zg.rotary(q, k[:, :3], pos, (64,))),
        (ValueError, lambda: zg.rotary(q, k, pos, (63,))),
        (ValueError, lambda: zg.rotary(q, k, pos, ())),
        (ValueError, lambda: zg.rotary(q, k, pos, (66,))),
        (ValueError, lambda: zg.rotary(q, k, pos, (32, 32))),
        (ValueError, lambda: zg.rotary(q, k, pos[:3], (64,))),
        (ValueError, lambda: zg.rotary(q, k, pos, (64,), base=-1.0)),
        (ValueError, lambda: zg.rotary(q, k, pos, (64,), base=math.nan)),
        (TypeError, lambda: zg.rotary(q, k, pos.to(torch.int16), (64,))),
        (TypeError, lambda: zg.rotary(q.half(), k.half(), pos, (64,))),
        (ValueError, lambda: zg.window_attention(q, k, k[:, :4])),
        (ValueError, lambda: zg.window_attention(q[:, :, :3], k, k)),
        (ValueError, lambda: zg.window_attention(q, k, k, window=0)),
        (ValueError, lambda: zg.window_attention(q, k, k, window=4, sinks=-1)),
        (ValueError, lambda: zg.window_attention(q, k, k, lengths=n[:1])),
        (TypeError, lambda: zg.window_attention(q, k, k, lengths=n.float())),
        (TypeError, lambda: zg.window_attention(q.double(), k.double(), k.double())),
        (L.ZgLibraryError, lambda: zg.window_attention(*[torch.zeros(1, 2, 1, 300, device=cuda)] * 3)),
        (L.ZgLibraryError, lambda: zg.window_attention(q.cpu(), k.cpu(), k.cpu())),
        (ValueError, lambda: zg.append_pages(kp, kp[:3], k, k, table, n)),
        (ValueError, lambda: zg.append_pages(kp[:, ::2], kp[:, ::2], k, k, table, n)),
        (ValueError, lambda: zg.append_pages(kp, kp, q, q, table, n)),
        (TypeError, lambda: zg.append_pages(kp, kp, k.float(), k.float(), table, n)),
        (ValueError, lambda: zg.append_pages(kp, kp, k, k, table[:1], n)),
        (ValueError, lambda: zg.append_pages(kp, kp, k, k, table, n, counts=n[:1])),
        (TypeError, lambda: zg.append_pages(kp, kp, k, k, table.float(), n)),
        (ValueError, lambda: zg.paged_attention(q[:, 0, :3], kp, kp, table, n)),
        (TypeError, lambda: zg.paged_attention(q[:, 0].float(), kp, kp, table, n)),
        (ValueError, lambda: zg.paged_attention(q[:, 0], kp, kp, table, n[:1])),
        (ValueError, lambda: zg.paged_attention(q[:, 0], kp, kp, table, n, window=-3)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_wide_integers_do_not_wrap(cuda):
    """A length or page number beyond 32 bits is refused as itself, not as what is left of it."""
    kp = torch.ones(4, 8, 1, 64, device=cuda, dtype=BF)
    q = torch.ones(2, 1, 64, device=cuda, dtype=BF)
    table = torch.zeros(2, 2, dtype=torch.int64, device=cuda)
    table[1, 0] = 2 ** 32
    o = zg.paged_attention(q, kp, kp, table, torch.tensor([2 ** 32 + 3, 3], device=cuda))
    assert torch.isnan(o).all()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 72), (F32, 64)])
def test_window_attention_not_finite_inputs(cuda, dtype, D):
    """NaN and infinite keys and values reach exactly the rows that see them,
    NaN queries their own row; all-NaN activations cost no more than others."""
    Z, S, H, K = 2, 700, 4, 2
    g = torch.Generator(device=cuda).manual_seed(D)
    q, k, v = (torch.randn(Z, S, h, D, generator=g, device=cuda).to(dtype) for h in (H, K, K))
    q[0, 5, 1] = math.nan
    k[0, 300, 0, 3] = math.nan
    v[0, 301, 1, 7] = math.inf
    v[1, 650, 0, 2] = -math.inf
    v[1, 651, 0, 2] = math.inf
    k[1, 100, 1] = 0.0
    k[1, 100, 1, 0] = math.inf
    for window, sinks in ((None, 0), (60, 2), (100, 310)):
        o = zg.window_attention(q, k, v, window, sinks)
        want, mag = so.window_attention(q, k, v, window, sinks)
        assert torch.isnan(want).any() and torch.isinf(want).any()
        so.assert_within(o, want.cpu(), so.attention_tolerance(q, k, want, mag, dtype, S).cpu())
    nan = torch.full_like(q, math.nan)
    assert torch.isnan(zg.window_attention(nan, nan[:, :, :K], nan[:, :, :K], 100, 2)).all()
    _ok()


@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_padding_of_any_bits(cuda, D):
    """Long padded sequences whose padding holds NaN: as fast and the same bits as with zeros there."""
    Z, S, H = 3, 6000, 4
    g = torch.Generator(device=cuda).manual_seed(D)
    q, k, v = (torch.randn(Z, S, H, D, generator=g, device=cuda).to(BF) for _ in range(3))
    lengths = torch.tensor([5873, 129, 4001], device=cuda)
    for t in (q, k, v):
        for z, n in enumerate(lengths.tolist()):
            t[z, n:] = 0
    want = zg.window_attention(q, k, v, lengths=lengths)
    for t in (q, k, v):
        for z, n in enumerate(lengths.tolist()):
            t[z, n:] = math.nan
    assert torch.equal(zg.window_attention(q, k, v, lengths=lengths), want)
    _ok()


def test_window_attention_rows_formed_again_in_a_long_sequence(cuda):
    """An infinite value late in a long sequence: the rows of its block that do
    not see it are formed again, for longer than the kernel's waits last."""
    S, D = 60000, 64
    g = torch.Generator(device=cuda).manual_seed(2)
    q, k, v = (torch.randn(1, S, 1, D, generator=g, device=cuda).to(BF) for _ in range(3))
    want = zg.window_attention(q, k, v)
    at = 59990
    v[0, at] = math.inf
    o = zg.window_attention(q, k, v)
    _ok()
    assert torch.isinf(o[0, at:]).all() and torch.isfinite(o[0, :at]).all()
    # each is off by 2^-8 sum w |v| + 2^-8 |o| at most (float32's part is far below)
    err = (o[0, :at].double() - want[0, :at].double()).abs()
    assert float(err.max()) <= 2 * 2.0 ** -7 * float(v[0, :at].abs().max())


# ------------------------------------------------ offsets beyond 32 bits of elements


def test_offsets_beyond_32_bits(cuda):
    """Rows more than 2^31 elements into q, o, the pages and the cache's pool."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator(device=cuda).manual_seed(8)
    S, H, D, tail = 140010, 120, 128, 300
    assert S * H * D > 2 ** 31
    q = torch.zeros(1, S, H, D, device=cuda, dtype=BF)
    k, v = (torch.zeros(1, S, 2, D, device=cuda, dtype=BF) for _ in range(2))
    for t in (q, k, v):
        t[:, -tail:] = torch.randn(1, tail, t.shape[2], D, generator=g, device=cuda).to(BF)
    o = zg.window_attention(q, k, v, 64)[:, -tail:]
    part = [t[:, -tail:] for t in (q, k, v)]
    want, mag = so.window_attention(*part, 64)
    tol = so.attention_tolerance(part[0], part[1], want, mag, BF, tail)
    so.assert_within(o[:, 64:], want[:, 64:].cpu(), tol[:, 64:].cpu())
    pos = torch.arange(S, device=cuda)[:, None]
    rq, _ = zg.rotary(q, k, pos, (D,))
    few, _ = zg.rotary(part[0], part[1], pos[-tail:], (D,))
    assert torch.equal(rq[:, -tail:], few)
    del q, k, v, o, rq
    N, page, K = 33000, 64, 8
    assert N * page * K * D > 2 ** 31
    kp, vp = (torch.empty(N, page, K, D, device=cuda, dtype=BF) for _ in range(2))
    k, v = (torch.randn(2, 150, K, D, generator=g, device=cuda).to(BF) for _ in range(2))
    table = torch.tensor([[N - 1, 0, N - 2], [5, N - 3, 6]], device=cuda)
    n = zg.append_pages(kp, vp, k, v, table, torch.zeros(2, dtype=torch.int64, device=cuda))
    assert n.tolist() == [150, 150] and torch.equal(kp[N - 2, 21], k[0, 149]) and torch.equal(vp[N - 3, 0], v[1, 64])
    q = torch.randn(2, 16, D, generator=g, device=cuda).to(BF)
    o = zg.paged_attention(q, kp, vp, table, n)
    small = torch.tensor([[0, 1, 2], [3, 4, 5]], device=cuda)
    at = table.flatten()
    assert torch.equal(o, zg.paged_attention(q, kp[at].contiguous(), vp[at].contiguous(), small, n))
    _ok()


@pytest.mark.parametrize("dtype,D", [(BF, 256), (F32, 128)])
def test_window_attention_fma_offsets_beyond_32_bits(cuda, dtype, D):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator(device=cuda).manual_seed(D)
    H, tail = 120, 200
    S = 2 ** 31 // (H * D) + 10
    q = torch.zeros(1, S, H, D, device=cuda, dtype=dtype)
    k, v = (torch.zeros(1, S, 1, D, device=cuda, dtype=dtype) for _ in range(2))
    for t in (q, k, v):
        t[:, -tail:] = torch.randn(1, tail, t.shape[2], D, generator=g, device=cuda).to(dtype)
    o = zg.window_attention(q, k, v, 20)[:, -tail:]
    part = [t[:, -tail:] for t in (q, k, v)]
    want, mag = so.window_attention(*part, 20)
    tol = so.attention_tolerance(part[0], part[1], want, mag, dtype, tail)
    so.assert_within(o[:, 20:], want[:, 20:].cpu(), tol[:, 20:].cpu())


@pytest.mark.parametrize("dtype,lengths", [
    (BF, [5000, 0, -1, 130]), (F32, [1, 3000, 60001, 60000]), (BF, [7000]), (BF, [0, 0]), (F32, [-3]),
    (BF, [12000, 11, 4097, 1, 128, 129, 8191]),
])
def test_paged_attention_in_wide_tables(cuda, dtype, lengths):
    """Tables wider than the sequences: the work is shared out by the lengths."""
    H, K, D, page, M = 4, 2, 64, 16, 3750
    g = torch.Generator().manual_seed(len(lengths))
    fits = [n if 0 <= n <= M * page else 0 for n in lengths]
    kp, vp, table = _pool(fits, page, K, D, dtype, g)
    wide = torch.full((len(lengths), M), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = _rand((len(lengths), H, D), dtype, g)
    n = torch.tensor(lengths, dtype=torch.int32)
    want, mag = so.paged_attention(q, kp, vp, table, torch.tensor(fits, dtype=torch.int32))
    o = zg.paged_attention(*(t.to(cuda) for t in (q, kp, vp, wide, n)))
    good = torch.tensor([a == b for a, b in zip(lengths, fits)])
    assert torch.isnan(o[~good.to(cuda)]).all()
    tol = so.attention_tolerance(q, kp, want, mag, dtype, max(max(fits), 1))
    so.assert_within(o[good.to(cuda)], want[good], tol[good])
