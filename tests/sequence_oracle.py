"""Plain float64 forms of the sequence ops, and the error their kernels may have.

A rounding is off by at most half a step: 2^-8 of the value in bf16
(``torch.finfo(torch.bfloat16).eps / 2``), 2^-24 in float32.
"""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rotary(q, k, positions, axes, base=10000.0, interleaved=False, joint=False, inverse=False):
    total = sum(axes) // 2
    freq, axis = [], []
    for a, width in enumerate(axes):
        for i in range(width // 2):
            e = len(freq) / total if joint else i / (width // 2)
            freq.append(base ** -e)
            axis.append(a)
    t = positions.double()[..., axis] * torch.tensor(freq, dtype=torch.float64)
    c, s = t.cos().unsqueeze(-2), t.sin().unsqueeze(-2) * (-1 if inverse else 1)
    first = torch.arange(total) * (2 if interleaved else 1)
    second = first + (1 if interleaved else total)
    out = []
    for x in (q, k):
        y = x.double().clone()
        u, w = x.double()[..., first], x.double()[..., second]
        y[..., first], y[..., second] = u * c - w * s, u * s + w * c
        size = torch.zeros_like(y)  # |x_a| + |x_b| of each column's pair
        size[..., first] = size[..., second] = u.abs() + w.abs()
        out.append((y, size))
    return out


def rotary_tolerance(want, size, dtype):
    """The output's rounding, and (|x_a| + |x_b|) times what cos and sin are
    off by: the angle, at most pi, rounded to float32 (2^-24 of it, 2^-22.3),
    sincospi's own 2 ulp (2^-23), two products and a sum (2^-23): below 2^-21."""
    return HALF_STEP[dtype] * want.abs() + size * 2.0 ** -21


def window_mask(S, window, sinks, device="cpu"):
    i, j = torch.arange(S, device=device)[:, None], torch.arange(S, device=device)[None, :]
    seen = j <= i
    if window is not None:
        seen = seen & ((i - j < window) | (j < sinks))
    return seen


def _attend(q, k, v, seen):
    """q [H, M, D], k, v [K, T, D], seen [M, T] -> output, and sum_j w_j |v_j|."""
    G = q.shape[0] // k.shape[0]
    k, v = (t.double().repeat_interleave(G, 0) for t in (k, v))
    s = (q.double() @ k.transpose(1, 2) / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf)
    w = torch.softmax(s, -1)
    # weights of zero multiply nothing: what is masked does not reach the row
    v = torch.where(seen.any(0)[None, :, None], v, 0.0)
    if not torch.isfinite(v).all():
        o, a = torch.empty_like(q.double()), torch.empty_like(q.double())
        for m in range(q.shape[1]):
            on = seen[m]
            o[:, m] = (w[:, m:m + 1, on] @ v[:, on])[:, 0]
            a[:, m] = (w[:, m:m + 1, on] @ v[:, on].abs())[:, 0]
        return o, a
    return w @ v, w @ v.abs()


def window_attention(q, k, v, window=None, sinks=0, lengths=None):
    """q [Z, S, H, D], k, v [Z, S, K, D] -> output and sum w |v|, [Z, S, H, D]."""
    Z, S, H, D = q.shape
    out = torch.zeros(Z, S, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for z in range(Z):
        n = S if lengths is None else int(lengths[z])
        if n == 0:
            continue
        o, a = _attend(*(t[z, :n].transpose(0, 1) for t in (q, k, v)), window_mask(n, window, sinks, q.device))
        out[z, :n], mag[z, :n] = o.transpose(0, 1), a.transpose(0, 1)
    return out, mag


def paged_attention(q, k_pages, v_pages, table, lengths, window=None, sinks=0):
    """q [B, H, D] (CPU) -> output and sum w |v|."""
    page = k_pages.shape[1]
    out, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        j = torch.arange(n)
        if window is not None:
            j = j[(j >= n - window) | (j < sinks)]
        if n == 0:
            continue
        at = table[b].long()[j // page]
        k, v = (t[at, j % page].transpose(0, 1) for t in (k_pages, v_pages))
        o, a = _attend(q[b].unsqueeze(1), k, v, torch.ones(1, len(j), dtype=torch.bool))
        out[b], mag[b] = o[:, 0], a[:, 0]
    return out, mag


def attention_tolerance(q, k, want, mag, dtype, n):
    """With A = sum_j w_j |v_j|: in bf16 each weight is rounded (2^-8 A) and
    the output is (2^-8 |o|).  In float32 everywhere: a score, D products of
    size at most S = max |q| |k| / sqrt(D) in all, is off by (D + 8) 2^-24 S
    and moves a weight by as much, and the weights' sum by as much again; the
    sums over n keys and their rescaling are off by 2 n 2^-24, the
    exponentials by 2^-22 each."""
    D = q.shape[-1]
    fin = [torch.nan_to_num(t.double(), 0.0, 0.0, 0.0) for t in (q, k)]
    size = float((fin[0].norm(dim=-1).max() * fin[1].norm(dim=-1).max()) / math.sqrt(D)) if k.numel() else 0.0
    f32 = 2.0 ** -24 * (2 * (D + 8) * size + 2 * n + 16)
    weights = HALF_STEP[dtype] if dtype == torch.bfloat16 else 0.0
    return (weights + f32) * mag + HALF_STEP[dtype] * want.abs()


def assert_within(got, want, tol, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    same = torch.isnan(got) & torch.isnan(want) | (got == want)
    bad = ~(((got - want).abs() <= tol) | same)
    if bad.any():
        i = tuple(int(x) for x in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, first at {i}: got "
                             f"{float(got[i])!r}, want {float(want[i])!r}, bound {float(tol[i]):.3g}")
