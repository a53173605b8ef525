"""Cases of the long-context attention operators: rotary positions, sliding-window
attention with sinks, writing tokens into a paged key-value cache, and the attention
of one new token over it.  ``run`` computes a case in plain torch operations, or,
with ``own`` set, by the framework's calls; ``exact`` gives its outputs in 64 bits.

Shapes: head dimension 64 with 12 heads and 256 positions is the decoder LM of
``bench.py``, 6 heads over 64 patches its ViT; the others are generic (grouped key
heads, head dimension 128, odd ones such as 72 and 80).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------- cases

def listed():
    return [
        # one new token of 64 sequences, each at its own far position: a decoding step, where the call's latency counts
        {"name": "rotary step", "op": "rotary", "dtype": "bf16", "Z": 64, "S": 1, "H": 12, "K": 4, "D": 64,
         "axes": "64", "base": 10000.0, "interleaved": False, "joint": False, "inverse": False, "shared": False},
        # a batch of images on an odd 9 x 7 grid of patches, the inverse rotation (the gradient's) in float32
        {"name": "rotary patches", "op": "rotary", "dtype": "f32", "Z": 96, "S": 63, "H": 6, "K": 6, "D": 72,
         "axes": "36,36", "base": 100.0, "interleaved": True, "joint": False, "inverse": True, "shared": True},
        # two videos of 16 frames of 32 x 32 patches, one spectrum dealt out to time, height and width
        {"name": "rotary video", "op": "rotary", "dtype": "bf16", "Z": 2, "S": 16384, "H": 16, "K": 4, "D": 128,
         "axes": "32,48,48", "base": 1000000.0, "interleaved": False, "joint": True, "inverse": False,
         "shared": False},
        # the decoder LM's batch of 16 sequences with a window of 64
        {"name": "window short", "op": "window", "dtype": "bf16", "Z": 16, "S": 256, "H": 12, "K": 12, "D": 64,
         "window": 64, "sinks": 4, "ragged": False},
        # plain causal attention of long sequences (no window), grouped key heads
        {"name": "causal long", "op": "window", "dtype": "bf16", "Z": 2, "S": 4096, "H": 12, "K": 4, "D": 64,
         "window": 0, "sinks": 0, "ragged": False},
        # a long document under a window of 1024 with four sinks
        {"name": "window long", "op": "window", "dtype": "bf16", "Z": 1, "S": 8192, "H": 16, "K": 4, "D": 128,
         "window": 1024, "sinks": 4, "ragged": False},
        # a padded batch of odd sizes in float32
        {"name": "window padded", "op": "window", "dtype": "f32", "Z": 3, "S": 777, "H": 8, "K": 2, "D": 80,
         "window": 200, "sinks": 3, "ragged": True},
        # the new token of 64 sequences into their pages
        {"name": "append step", "op": "append", "dtype": "bf16", "B": 64, "S": 1, "K": 4, "D": 128, "page": 16,
         "L": 2048, "ragged": False},
        # a padded batch of 16 prompts into empty and part-filled caches
        {"name": "append prompts", "op": "append", "dtype": "bf16", "B": 16, "S": 2000, "K": 4, "D": 128, "page": 64,
         "L": 500, "ragged": True},
        # one sequence with a long cache: the work has to be split over its length
        {"name": "paged one long", "op": "paged", "dtype": "bf16", "B": 1, "L": 131000, "H": 16, "K": 4, "D": 128,
         "page": 64, "window": 0, "sinks": 0},
        # 64 sequences of the decoder LM's heads, lengths from a quarter of the longest to it, small pages
        {"name": "paged batch", "op": "paged", "dtype": "bf16", "B": 64, "L": 4000, "H": 12, "K": 12, "D": 64,
         "page": 16, "window": 0, "sinks": 0},
        # a step of 8 sequences that see the last 1000 tokens and four sinks of a long cache
        {"name": "paged window", "op": "paged", "dtype": "bf16", "B": 8, "L": 16000, "H": 16, "K": 4, "D": 128,
         "page": 32, "window": 1000, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    K = rng.choice([1, 2, 3, 4, 6, 8, 12])
    return K * rng.choice([1, 1, 2, 3, 4, 5, 8]), K


def draw(rng):
    op = rng.choice(["rotary", "window", "window", "append", "paged", "paged"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    H, K = _heads(rng)
    D = rng.choice([64, 64, 128, 128, 32, 40, 72, 80, 96, 192, 256])
    esize = 2 if dtype == "bf16" else 4
    if op == "rotary":
        # prompts and single tokens, images, videos; up to a few hundred megabytes
        n = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, D // 2), n - 1)) + [D // 2 - rng.choice([0, 0, 0, 1])]
        axes = ",".join(str(2 * (b - a)) for a, b in zip([0] + cuts, cuts) if b > a)
        tokens = _log(rng, 1, max(2, 80_000_000 // ((H + K) * D * esize)))
        S = _log(rng, 1, tokens)
        return {"op": op, "dtype": dtype, "Z": max(1, tokens // S), "S": S, "H": H, "K": K, "D": D, "axes": axes,
                "base": rng.choice([100.0, 10000.0, 500000.0]), "interleaved": rng.random() < 0.5,
                "joint": rng.random() < 0.5, "inverse": rng.random() < 0.3, "shared": rng.random() < 0.5}
    if op == "window":
        # sequences of one token to thousands; the plain form's scores stay below the largest listed case's
        S, D = _log(rng, 1, 6000), min(D, 128)
        most = 2.4e8 if dtype == "bf16" else 1e8  # Z H S^2
        H, K = (H, K) if H * S * S <= most else (4, rng.choice([1, 2, 4]))
        Z = min(_log(rng, 1, 64), max(1, int(min(most // (H * S * S), 1e8 // (S * H * D)))))
        return {"op": op, "dtype": dtype, "Z": Z, "S": S, "H": H, "K": K, "D": D,
                "window": rng.choice([0, _log(rng, 1, S), _log(rng, 1, S)]), "sinks": rng.choice([0, 1, 4, 37]),
                "ragged": rng.random() < 0.5}
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256])
    if op == "append":
        # decoding steps and prompts, into short and long caches
        tokens = _log(rng, 1, max(2, 30_000_000 // (K * D * esize)))
        S = rng.choice([1, _log(rng, 1, min(tokens, 8000))])
        B = max(1, min(512, tokens // S))
        return {"op": op, "dtype": dtype, "B": B, "S": S, "K": K, "D": D, "page": page,
                "L": _log(rng, 1, max(2, min(8000, 100_000_000 // (B * K * D * esize)))), "ragged": rng.random() < 0.5}
    # one sequence to many, caches of one token to 100000
    B = _log(rng, 1, 256)
    L = _log(rng, 1, max(2, min(100_000, 120_000_000 // (B * K * D * esize))))
    return {"op": op, "dtype": dtype, "B": B, "L": L, "H": H, "K": K, "D": D, "page": page,
            "window": rng.choice([0, 0, _log(rng, 1, L)]), "sinks": rng.choice([0, 4, 9])}


# --------------------------------------------------------------------- inputs

def _lengths(n, longest, ragged):
    """Lengths from the longest down to a quarter of it (at least one), in even steps."""
    if not ragged:
        return [longest] * n
    return [max(1, longest - (3 * longest * i) // (4 * n)) for i in range(n)]


def _pages_for(lengths, page):
    return [-(-n // page) for n in lengths]


def _axes(case):
    return tuple(int(a) for a in case["axes"].split(","))


def _pool(case, totals, g):
    """Key and value pages, and a table of page numbers in no order: pages that no sequence holds are -1."""
    dt, page = DTYPES[case["dtype"]], case["page"]
    need = _pages_for(totals, page)
    n = sum(need) + 3
    k = torch.randn((n, page, case["K"], case["D"]), generator=g, device="cuda").to(dt)
    v = torch.randn((n, page, case["K"], case["D"]), generator=g, device="cuda").to(dt)
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    per = torch.tensor(need, device="cuda")
    first = per.cumsum(0) - per
    col = torch.arange(max(need), device="cuda")
    held = col[None, :] < per[:, None]
    table = torch.where(held, order[(first[:, None] + col[None, :]).clamp(max=n - 1)], -1)
    return k, v, table.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["op"] == "rotary":
        Z, S, H, K, D = (case[n] for n in "ZSHKD")
        n_axes = len(_axes(case))
        # one fused projection's output; queries and keys are views of it
        x = torch.randn((Z, S, H + 2 * K, D), generator=g, device="cuda").to(dt)
        lead = () if case["shared"] else (Z,)
        if n_axes == 1:  # text: a run of positions from each sequence's own start
            start = torch.randint(0, 100000, lead + (1,), generator=g, device="cuda")
            pos = (start + torch.arange(S, device="cuda"))[..., None]
        else:  # a grid of patches, the last axis fastest, moved by a start per sequence
            side = max(1, int(round(S ** (1.0 / n_axes))))
            t = torch.arange(S, device="cuda")
            grid = [t // side ** (n_axes - 1 - a) % (side if a else S) for a in range(n_axes)]
            start = torch.randint(0, 5000, lead + (1, n_axes), generator=g, device="cuda")
            pos = torch.stack(grid, dim=-1) + start
        state.update(q=x[:, :, :H], k=x[:, :, H:H + K], positions=pos.contiguous())
    elif case["op"] == "window":
        Z, S, H, K, D = (case[n] for n in "ZSHKD")
        x = torch.randn((Z, S, H + 2 * K, D), generator=g, device="cuda").to(dt)
        state.update(q=x[:, :, :H], k=x[:, :, H:H + K], v=x[:, :, H + K:], lengths=None)
        if case["ragged"]:
            order = torch.randperm(Z, generator=g, device="cuda")
            state["lengths"] = torch.tensor(_lengths(Z, S, True), dtype=torch.int32, device="cuda")[order]
    elif case["op"] == "append":
        B, S = case["B"], case["S"]
        had = _lengths(B, case["L"], True)
        kp, vp, table = _pool(case, [n + S for n in had], g)
        state.update(k_pages=kp, v_pages=vp, table=table, counts=None,
                     lengths=torch.tensor(had, dtype=torch.int32, device="cuda"))
        x = torch.randn((B, S, 2 * case["K"], case["D"]), generator=g, device="cuda").to(dt)
        state.update(k=x[:, :, :case["K"]], v=x[:, :, case["K"]:])
        if case["ragged"]:
            order = torch.randperm(B, generator=g, device="cuda")
            state["counts"] = torch.tensor(_lengths(B, S, True), dtype=torch.int32, device="cuda")[order]
    else:
        B = case["B"]
        had = _lengths(B, case["L"], True)
        kp, vp, table = _pool(case, had, g)
        q = torch.randn((B, case["H"], case["D"]), generator=g, device="cuda").to(dt)
        state.update(q=q, k_pages=kp, v_pages=vp, table=table,
                     lengths=torch.tensor(had, dtype=torch.int32, device="cuda"))
    return state


# ----------------------------------------------------------------- plain forms

def _rotary_plain(x, cos, sin, interleaved):
    """x [Z, S, H, D], cos and sin [.., S, n]: the pairs of the first 2 n columns turned."""
    n = cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    f = x.float()
    a, b = (f[..., 0:2 * n:2], f[..., 1:2 * n:2]) if interleaved else (f[..., :n], f[..., n:2 * n])
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack((u, w), dim=-1).flatten(-2) if interleaved else torch.cat((u, w), dim=-1)
    return torch.cat((turned, f[..., 2 * n:]), dim=-1).to(x.dtype)


def _spectrum(case, device, dtype):
    """The frequency and the axis of each rotated pair."""
    halves = torch.tensor([a // 2 for a in _axes(case)], device=device)
    n = sum(_axes(case)) // 2
    axis = torch.repeat_interleave(torch.arange(len(halves), device=device), halves, output_size=n)
    i = torch.arange(n, device=device)
    if case["joint"]:
        e = i.to(dtype) / n
    else:
        e = (i - (halves.cumsum(0) - halves)[axis]).to(dtype) / halves[axis].to(dtype)
    return torch.exp(-e * math.log(case["base"])), axis


def _run_rotary(st):
    case = st["case"]
    freq, axis = _spectrum(case, st["q"].device, torch.float64)
    angle = st["positions"].double()[..., axis] * freq
    sign = -1.0 if case["inverse"] else 1.0
    cos, sin = angle.cos().float(), (angle.sin() * sign).float()
    return {"q": _rotary_plain(st["q"], cos, sin, case["interleaved"]),
            "k": _rotary_plain(st["k"], cos, sin, case["interleaved"])}


def _run_window(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    Z, S, H, D = q.shape
    K = k.shape[2]
    qf = q.float().permute(0, 2, 1, 3).reshape(Z, K, H // K, S, D)
    kf, vf = (t.float().permute(0, 2, 1, 3).unsqueeze(2) for t in (k, v))
    s = (qf / math.sqrt(D)) @ kf.transpose(-1, -2)
    i = torch.arange(S, device=q.device)
    seen = i[None, :] <= i[:, None]
    if case["window"]:
        seen = seen & ((i[:, None] - i[None, :] < case["window"]) | (i[None, :] < case["sinks"]))
    if st["lengths"] is not None:
        live = i[None, :] < st["lengths"][:, None]
        seen = (seen & live[:, None, :])[:, None, None]
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = (p @ vf) / p.sum(dim=-1, keepdim=True)
    o = o.reshape(Z, H, S, D).permute(0, 2, 1, 3)
    if st["lengths"] is not None:
        o = torch.where(live[:, :, None, None], o, 0.0)
    return o.to(q.dtype).contiguous()


def _run_append(st):
    kp, vp, k, v = st["k_pages"], st["v_pages"], st["k"], st["v"]
    B, S, K, D = k.shape
    page = kp.shape[1]
    counts = st["counts"] if st["counts"] is not None else torch.full_like(st["lengths"], S)
    # rows of padding repeat the sequence's last row, at that row's place
    row = torch.minimum(torch.arange(S, device=k.device)[None, :], counts[:, None].long() - 1)
    at = st["lengths"][:, None].long() + row
    slot = torch.gather(st["table"].long(), 1, at // page) * page + at % page
    b = torch.arange(B, device=k.device)[:, None]
    kp.view(-1, K, D)[slot] = k[b, row]
    vp.view(-1, K, D)[slot] = v[b, row]
    return {"k_pages": kp, "v_pages": vp, "lengths": st["lengths"] + counts}


def _run_paged(st):
    case, q = st["case"], st["q"]
    B, H, D = q.shape
    N, page, K, _ = st["k_pages"].shape
    pages = st["table"].clamp(min=0).long()
    T = pages.shape[1] * page
    kf, vf = (t[pages].reshape(B, T, K, D).float().permute(0, 2, 1, 3) for t in (st["k_pages"], st["v_pages"]))
    s = (q.float().reshape(B, K, H // K, D) / math.sqrt(D)) @ kf.transpose(-1, -2)
    j, n = torch.arange(T, device=q.device)[None, :], st["lengths"][:, None]
    seen = j < n
    if case["window"]:
        seen = seen & ((j >= n - case["window"]) | (j < case["sinks"]))
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = (p @ vf) / p.sum(dim=-1, keepdim=True)
    return o.reshape(B, H, D).to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        import zerograd_b200 as zg

        if case["op"] == "rotary":
            q, k = zg.rotary(state["q"], state["k"], state["positions"], _axes(case), base=case["base"],
                             interleaved=case["interleaved"], joint=case["joint"], inverse=case["inverse"])
            return {"q": q, "k": k}
        if case["op"] == "window":
            return zg.window_attention(state["q"], state["k"], state["v"], window=case["window"] or None,
                                       sinks=case["sinks"], lengths=state["lengths"])
        if case["op"] == "append":
            lengths = zg.append_pages(state["k_pages"], state["v_pages"], state["k"], state["v"], state["table"],
                                      state["lengths"], counts=state["counts"])
            return {"k_pages": state["k_pages"], "v_pages": state["v_pages"], "lengths": lengths}
        return zg.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["lengths"],
                                  window=case["window"] or None, sinks=case["sinks"])
    plain = {"rotary": _run_rotary, "window": _run_window, "append": _run_append, "paged": _run_paged}
    return plain[case["op"]](state)


# ----------------------------------------------------------------------- work

def _pairs(n, window, sinks):
    """Keys seen by the n queries of a sequence, in all."""
    if not window or window >= n:
        return n * (n + 1) // 2
    late = n - window  # queries window .. n - 1 see the window and the sinks before it
    m = min(sinks, late)
    return window * (window + 1) // 2 + late * window + m * (m + 1) // 2 + (late - m) * m


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rotary":
        n_axes, tokens = len(_axes(case)), case["Z"] * case["S"]
        x = tokens * (case["H"] + case["K"]) * case["D"]
        pos = (case["S"] if case["shared"] else tokens) * n_axes * 8
        return {"bytes": 2 * x * e + pos, "flops": 3 * x}
    if case["op"] == "window":
        n = _lengths(case["Z"], case["S"], case["ragged"])
        live = sum(n) * (case["H"] + 2 * case["K"]) + case["Z"] * case["S"] * case["H"]
        pairs = sum(_pairs(m, case["window"], case["sinks"]) for m in n)
        return {"bytes": live * case["D"] * e, "flops": 4 * pairs * case["H"] * case["D"]}
    if case["op"] == "append":
        tokens = sum(_lengths(case["B"], case["S"], case["ragged"]))
        return {"bytes": 4 * tokens * case["K"] * case["D"] * e + 8 * case["B"], "flops": 0}
    had = _lengths(case["B"], case["L"], True)
    seen = had
    if case["window"]:
        seen = [min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in had]
    q = case["B"] * case["H"] * case["D"]
    return {"bytes": (2 * sum(seen) * case["K"] * case["D"] + 2 * q) * e, "flops": 4 * sum(seen) * case["H"] * case["D"]}


# ---------------------------------------------------------------------- exact

def _softmax_rows(q, k, v, see):
    """softmax(q k' / sqrt(D)) v in 64 bits: q [H, M, D], k and v [K, T, D], see [M, T] -> [H, M, D]."""
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    G = q.shape[0] // k.shape[0]
    for h in range(q.shape[0]):
        z = torch.einsum("md,td->mt", q[h].double(), k[h // G].double()) * q.shape[-1] ** -0.5
        z = torch.where(see, z, torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
        out[h] = torch.softmax(z, dim=-1) @ v[h // G].double()
    return out


def _exact_rotary(st):
    case = st["case"]
    axes, base = _axes(case), case["base"]
    cols, total = [], sum(axes) // 2
    for a, width in enumerate(axes):
        for i in range(width // 2):
            e = len(cols) / total if case["joint"] else i / (width // 2)
            cols.append(st["positions"][..., a].double() * base ** -e)
    turn = torch.polar(torch.ones_like(torch.stack(cols, -1)), torch.stack(cols, -1))
    turn = (turn.conj() if case["inverse"] else turn).unsqueeze(-2)
    out = {}
    for name in ("q", "k"):
        x = st[name].double()
        first = torch.arange(total, device=x.device) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else total)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out[name] = x
    return out


def _exact_window(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    Z, S, H, D = q.shape
    out = torch.zeros((Z, S, H, D), dtype=torch.float64, device=q.device)
    window = case["window"] or S
    for z in range(Z):
        n = int(st["lengths"][z]) if st["lengths"] is not None else S
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            i, j = torch.arange(a, b, device=q.device)[:, None], torch.arange(b, device=q.device)[None, :]
            see = (j <= i) & ((j > i - window) | (j < case["sinks"]))
            rows = _softmax_rows(q[z, a:b].transpose(0, 1), k[z, :b].transpose(0, 1), v[z, :b].transpose(0, 1), see)
            out[z, a:b] = rows.transpose(0, 1)
    return out


def _exact_paged(st):
    case, q = st["case"], st["q"]
    page = st["k_pages"].shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(st["lengths"].tolist()):
        j = torch.arange(n, device=q.device)
        if case["window"]:
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        held = st["table"][b].long()[j // page]
        k, v = (t[held, j % page].transpose(0, 1) for t in (st["k_pages"], st["v_pages"]))
        see = torch.ones((1, len(j)), dtype=torch.bool, device=q.device)
        out[b] = _softmax_rows(q[b].unsqueeze(1), k, v, see)[:, 0]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(st)
    if case["op"] == "window":
        return _exact_window(st)
    if case["op"] == "paged":
        return _exact_paged(st)
    # a cache is written, not computed: the tokens of each sequence, one page at a time
    kp, vp, page = st["k_pages"].double(), st["v_pages"].double(), st["k_pages"].shape[1]
    lengths = st["lengths"].tolist()
    counts = st["counts"].tolist() if st["counts"] is not None else [case["S"]] * case["B"]
    table = st["table"].tolist()
    for b, (start, m) in enumerate(zip(lengths, counts)):
        t = 0
        while t < m:
            at = start + t
            take = min(m - t, page - at % page)
            spot = slice(at % page, at % page + take)
            kp[table[b][at // page], spot] = st["k"][b, t:t + take].double()
            vp[table[b][at // page], spot] = st["v"][b, t:t + take].double()
            t += take
    return {"k_pages": kp, "v_pages": vp, "lengths": st["lengths"] + torch.tensor(counts, dtype=torch.int32,
                                                                                device=st["lengths"].device)}
