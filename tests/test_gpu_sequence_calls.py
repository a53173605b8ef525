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


# ------------------------------------------ values that are infinite or NaN, or nearly


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 72), (BF, 20), (F32, 64), (F32, 136)])
@pytest.mark.parametrize("window,sinks,ragged", [(None, 0, False), (40, 3, True), (130, 70, False), (1, 1, True)])
def test_window_attention_values_not_finite_in_many_places(cuda, dtype, D, window, sinks, ragged):
    """NaN and infinities in single places, in a whole position and in a whole
    column reach the rows that see them, and what is masked no row at all."""
    Z, S, H, K = 3, 420, 4, 2
    q, k, v = (_rand((Z, S, h, D), dtype, D + h + i, cuda) for i, h in enumerate((H, K, K)))
    g = torch.Generator().manual_seed(D)
    for z in range(Z):  # up to 12 places a sequence, more blocks than are listed in the last
        for _ in range((1, 4, 12)[z]):
            j, h, d = (int(torch.randint(0, n, (1,), generator=g)) for n in (S, K, D))
            v[z, j, h, d] = (math.nan, math.inf, -math.inf)[int(torch.randint(0, 3, (1,), generator=g))]
    v[0, 100, 0] = math.nan
    v[1, :, 1, 5] = math.inf
    v[2, 200:, 0, 7] = -math.inf
    v[2, 20, 1, 9], v[2, 300, 1, 9] = math.inf, -math.inf
    lengths = torch.tensor([S, 150, 333], device=cuda) if ragged else None
    o = zg.window_attention(q, k, v, window, sinks, lengths)
    want, mag = so.window_attention(q, k, v, window, sinks, lengths)
    assert L.load().zg_device_error(1) == 0
    assert torch.isnan(want).any() and torch.isinf(want).any()
    so.assert_within(o, want.cpu(), so.attention_tolerance(q, k, want, mag, dtype, S).cpu())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (F32, 64)])
def test_window_attention_weights_of_zero_on_infinite_values(cuda, dtype, D):
    """A visible score of -inf is a weight of zero, and 0 * inf is NaN."""
    S = 200
    q, k, v = (_rand((1, S, 1, D), dtype, s, cuda) for s in range(3))
    q[..., 0] = q[..., 0].abs() + 0.5
    k[0, 30, 0], v[0, 30, 0, :4] = 0, math.inf
    k[0, 30, 0, 0] = -math.inf
    v[0, 90, 0, 2:6] = math.inf
    o = zg.window_attention(q, k, v, 100)
    want, mag = so.window_attention(q, k, v, 100)
    assert int(torch.isnan(want).sum()) == 4 * 100 and int(torch.isinf(want).sum()) == 4 * 100 - 2 * 40
    so.assert_within(o, want.cpu(), so.attention_tolerance(q, torch.nan_to_num(k, 0, 0, 0), want, mag, dtype, S).cpu())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 20), (F32, 64), (F32, 256)])
def test_window_attention_of_values_near_the_largest(cuda, dtype, D):
    """Sums of finite values do not overflow on the way to an average of them."""
    S = 700
    q, k = (_rand((1, S, 2, D), dtype, s, cuda) for s in range(2))
    v = 2.5e38 * (1 + 0.1 * torch.rand(1, S, 2, D, generator=torch.Generator(device=cuda).manual_seed(3), device=cuda))
    v = v.to(dtype)
    v[:, :, 1] *= -1
    for window, sinks in ((None, 0), (90, 5)):
        o = zg.window_attention(q, k, v, window, sinks)
        want, mag = so.window_attention(q, k, v, window, sinks)
        so.assert_within(o, want.cpu(), so.attention_tolerance(q, k, want, mag, dtype, S).cpu())


def _time(run, n=10):
    """Device time of a call in ms: the least of n, after one untimed."""
    run()
    times = []
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        run()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("dtype,H,K,D,window,sinks", [
    (BF, 12, 4, 64, None, 0), (BF, 8, 4, 128, 1024, 4), (F32, 4, 2, 64, None, 0), (F32, 4, 2, 128, 700, 4)])
def test_window_attention_time_with_values_not_finite(cuda, dtype, H, K, D, window, sinks):
    """One infinite value that most rows see, one beside the sinks, a NaN late,
    a column of one sign, all-NaN values, all-NaN activations, padding of NaN:
    without a cost where no row that does not see it is touched, and bounded
    where many are."""
    S = 4096
    q, k, v = (_rand((2, S, h, D), dtype, h, cuda) for h in (H, K, K))
    lengths = torch.tensor([S, S // 2 + 1], device=cuda)
    plain = _time(lambda: zg.window_attention(q, k, v, window, sinks))
    padded = _time(lambda: zg.window_attention(q, k, v, window, sinks, lengths))
    slow = {}
    for name, at, value in (("first", (0, 0, slice(None), 3), math.inf), ("beside the sinks", (0, 50), math.inf),
                            ("late", (1, S - 60), math.nan), ("column", (slice(None), slice(None), slice(None), 1), math.inf),
                            ("all", (), math.nan)):
        bad = v.clone()
        bad[at] = value
        slow[name] = _time(lambda: zg.window_attention(q, k, bad, window, sinks)) / plain
    nan = [torch.full_like(t, math.nan) for t in (q, k, v)]
    slow["activations"] = _time(lambda: zg.window_attention(*nan, window, sinks)) / plain
    for t in (q, k, v):
        t[1, S // 2 + 1:] = math.nan
    slow["padding"] = _time(lambda: zg.window_attention(q, k, v, window, sinks, lengths)) / padded
    print({n: round(x, 2) for n, x in slow.items()}, round(plain * 1e3, 1), "us")
    assert L.load().zg_device_error(1) == 0
    assert slow["first"] < 3 and slow["activations"] < 3 and slow["padding"] < 3, slow
    assert slow["late"] < 12 and slow["beside the sinks"] < 12 and slow["column"] < 50 and slow["all"] < 50, slow


# ------------------------------------------------ a sequence's result is its own


def _cache(lengths, page, K, D, dtype, device, seed=1, spare=2):
    """A pool that holds the sequences, and their table (-1 behind each one's pages)."""
    need = [-(-n // page) for n in lengths]
    g = torch.Generator(device=device).manual_seed(seed)
    kp, vp = (torch.randn((sum(need) + spare, page, K, D), generator=g, device=device).to(dtype) for _ in range(2))
    order = torch.randperm(sum(need) + spare, generator=g, device=device).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32, device=device)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return kp, vp, table


@pytest.mark.parametrize("dtype,H,K,D,window,sinks", [
    (BF, 4, 2, 64, None, 0), (BF, 8, 1, 128, None, 0), (BF, 12, 12, 64, 3000, 4), (BF, 4, 4, 192, None, 0),
    (BF, 20, 1, 128, None, 0), (BF, 12, 1, 256, None, 0), (BF, 3, 1, 20, None, 0), (F32, 4, 2, 64, None, 0), (F32, 16, 2, 136, 2500, 0),
    (F32, 2, 2, 128, None, 0)])
def test_paged_attention_of_a_sequence_whatever_else_is_in_the_launch(cuda, dtype, H, K, D, window, sinks):
    """The bits of a sequence's output do not depend on the other sequences,
    their number, or the table's width: a candidate's loss is its own."""
    lengths = [9000, 0, 4096, 130, 1, 2000, 700, 1024, 5555, 300]
    kp, vp, table = _cache(lengths, 16, K, D, dtype, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = _rand((len(lengths), H, D), dtype, 3, cuda)
    want = zg.paged_attention(q, kp, vp, table, n, window, sinks)
    full, mag = so.paged_attention(q.cpu(), kp.cpu(), vp.cpu(), table.cpu(), n.cpu(), window, sinks)
    so.assert_within(want, full, so.attention_tolerance(q.cpu(), kp.cpu(), full, mag, dtype, max(lengths)))
    wide = torch.nn.functional.pad(table, (0, 4000), value=-1)
    assert torch.equal(zg.paged_attention(q, kp, vp, wide, n, window, sinks), want)
    for b, m in enumerate(lengths):
        own = table[b:b + 1, :max(1, -(-m // 16))].contiguous()
        for t in (own, wide[b:b + 1]):
            assert torch.equal(zg.paged_attention(q[b:b + 1], kp, vp, t, n[b:b + 1], window, sinks)[0], want[b]), m
    for some in ([0, 3], [2, 5, 7, 8], [9, 6, 3] * 20, list(range(10)) * 7, [5, 7, 0, 4] * 110):
        at = torch.tensor(some, device=cuda)
        for t in (table, wide):
            got = zg.paged_attention(q[at], kp, vp, t[at], n[at], window, sinks)
            assert torch.equal(got, want[at]), len(some)


@pytest.mark.parametrize("dtype,D,longest", [(BF, 64, 5000), (BF, 128, 900), (F32, 64, 5000)])
def test_paged_attention_under_vmap_over_long_caches(cuda, dtype, D, longest):
    """Three candidates of two sequences: the bits of the calls candidate by candidate."""
    P, H, K = 3, 4, 2
    lengths = [longest, longest // 3, 17, longest - 1, longest // 2, 640]
    kp, vp, table = _cache(lengths, 16, K, D, dtype, cuda)
    table, n = table.reshape(P, 2, -1), torch.tensor(lengths, device=cuda).reshape(P, 2)
    q = _rand((P, 2, H, D), dtype, 5, cuda)
    got = torch.func.vmap(lambda qq, tt, nn: zg.paged_attention(qq, kp, vp, tt, nn))(q, table, n)
    for p in range(P):
        assert torch.equal(zg.paged_attention(q[p], kp, vp, table[p], n[p]), got[p])


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 256), (BF, 20), (F32, 64), (F32, 200)])
def test_paged_attention_of_values_near_the_largest(cuda, dtype, D):
    """Sums of finite values do not overflow on the way to an average of them."""
    lengths = [700, 3, 4000]
    kp, vp, table = _cache(lengths, 16, 2, D, dtype, cuda)
    vp = (2.5e38 * (1 + 0.1 * vp.float().sigmoid())).to(dtype) * torch.tensor([1, -1], device=cuda, dtype=dtype)[:, None]
    q, n = _rand((3, 4, D), dtype, 6, cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda)
    for window in (None, 90):
        o = zg.paged_attention(q, kp, vp, table, n, window, 2)
        want, mag = so.paged_attention(q.cpu(), kp.cpu(), vp.cpu(), table.cpu(), n.cpu(), window, 2)
        so.assert_within(o, want, so.attention_tolerance(q.cpu(), kp.cpu(), want, mag, dtype, 4000))


# ------------------------------------------------ the form that shares work out, with its workspace and second kernel


SHARED = [
    # dtype, H, K, D, lengths: few units, tables above 1024 positions
    (BF, 4, 2, 64, [3000, 40, 5000]), (BF, 8, 1, 128, [20000]), (F32, 4, 2, 64, [9000, 1, 2500]), (BF, 6, 2, 192, [0, 6000]),
    (BF, 16, 2, 64, [1100] * 30),  # equal parts of a unit
]


def _sharing_step(cuda, dtype, H, K, D, lengths, seed=1):
    """The newest tokens written and attended, in new tensors: the inputs and the call."""
    kp, vp, table = _cache([n + 1 for n in lengths], 16, K, D, dtype, cuda, seed)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    x = _rand((len(lengths), 1, H + 2 * K, D), dtype, seed + 9, cuda)

    def run():
        m = zg.append_pages(kp, vp, x[:, :, H:H + K], x[:, :, H + K:], table, n)
        return zg.paged_attention(x[:, 0, :H], kp, vp, table, m)

    return x, run, (kp, vp, table, n + 1)


def _workspace_of(x, K, table, D, dtype, H):
    B, M = table.shape
    return L.load().zg_paged_attention_workspace_size(B, H, K, D, M, 16, 0, 0, L.dtype_code(dtype))


@pytest.mark.parametrize("dtype,H,K,D,lengths", SHARED)
def test_sharing_form_captured_and_replayed(cuda, dtype, H, K, D, lengths):
    """Two calls' graphs, replayed in turn and on two streams at once on new
    values, give the bits of the eager calls, which hold against the oracle."""
    steps = [_sharing_step(cuda, dtype, H, K, D, lengths, seed) for seed in (1, 5)]
    graphs = []
    for x, run, (_, _, table, _) in steps:
        assert _workspace_of(x, K, table, D, dtype, H) > 0
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in (2, 3):
        want = []
        for i, (x, run, (kp, vp, table, n)) in enumerate(steps):
            x.copy_(_rand(x.shape, F32, 10 * i + seed, cuda))
            want.append(run().clone())
            full, mag = so.paged_attention(x[:, 0, :H].cpu(), kp.cpu(), vp.cpu(), table.cpu(), n.cpu())
            so.assert_within(want[i], full, so.attention_tolerance(x.cpu(), kp.cpu(), full, mag, dtype, max(lengths)))
        for at_once in (False, True):
            for _, out in graphs:
                out.zero_()
            torch.cuda.synchronize()
            for (graph, _), stream in zip(graphs, streams):
                with torch.cuda.stream(stream if at_once else torch.cuda.current_stream()):
                    graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out, w) for (_, out), w in zip(graphs, want))


@pytest.mark.parametrize("dtype,H,K,D,lengths", SHARED)
def test_sharing_form_on_two_streams_at_once(cuda, dtype, H, K, D, lengths):
    steps = [_sharing_step(cuda, dtype, H, K, D, lengths, seed) for seed in (1, 5)]
    want = [run() for _, run, _ in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for i, (stream, (_, run, _)) in enumerate(zip(streams, steps)):
            with torch.cuda.stream(stream):
                outs.append((i, run()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)


@pytest.mark.parametrize("dtype,H,K,D,lengths", SHARED)
def test_sharing_form_with_a_page_outside_the_pool(cuda, dtype, H, K, D, lengths):
    """A bad page in the middle of a sequence makes that one NaN and no other."""
    kp, vp, table = _cache(lengths, 16, K, D, dtype, cuda)
    q, n = _rand((len(lengths), H, D), dtype, 8, cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda)
    assert _workspace_of(q, K, table, D, dtype, H) > 0
    want = zg.paged_attention(q, kp, vp, table, n)
    at = max(range(len(lengths)), key=lambda b: lengths[b])
    for page, bad in ((0, -1), (lengths[at] // 32, kp.shape[0]), ((lengths[at] - 1) // 16, 2 ** 31 - 1)):
        broken = table.clone()
        broken[at, page] = bad
        o = zg.paged_attention(q, kp, vp, broken, n)
        assert torch.isnan(o[at]).all()
        rest = torch.arange(len(lengths), device=cuda) != at
        assert torch.equal(o[rest], want[rest])
    for length in (-1, table.shape[1] * 16 + 1):
        m = n.clone()
        m[at] = length
        o = zg.paged_attention(q, kp, vp, table, m)
        assert torch.isnan(o[at]).all() and torch.equal(o[rest], want[rest])
