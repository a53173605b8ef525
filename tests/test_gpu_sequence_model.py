"""The sequence ops inside a candidate: a small language model with rotary
positions and windowed attention evaluated, stepped, chunked and captured by
``ZeroGrad``, and a fitness taken from generated answers over a paged cache.

Tolerance of a loss against the same model with attention in float32 torch
operations: rel 5e-3, as for the other whole models (bf16 activations, float32
cross-entropy).  Everything else is compared bit for bit."""
import math

import pytest
import torch

import sequence_oracle as so
import zerograd_b200 as zg
from zerograd_b200 import _lib as L
from zerograd_b200 import _ops

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
B, S, E, H, K, D, V, P, RANK, SIGMA = 2, 150, 128, 4, 2, 64, 512, 6, 8, 0.01
WINDOW, SINKS = 40, 3
SHAPES = {"emb": (V, E), "qkv": (E, (H + 2 * K) * D), "o": (H * D, E)}


def _model(device):
    g = torch.Generator(device=device).manual_seed(0)
    params = {n: (torch.randn(s, generator=g, device=device) * (0.3 if n == "emb" else 0.08)).to(BF) for n, s in SHAPES.items()}
    layout = {"emb": zg.ParameterLayout.TABLE}
    manifest = zg.Manifest(1, tuple(zg.ManifestEntry((n,), layout.get(n, zg.ParameterLayout.MATRIX), n) for n in SHAPES))
    tokens = torch.randint(0, V, (B, S), generator=g, device=device, dtype=torch.int32)
    labels = torch.randint(0, V, (B, S), generator=g, device=device, dtype=torch.int32)
    return params, manifest, (tokens, labels, torch.tensor([S, S - 37], dtype=torch.int32, device=device))


def _plain_attention(q, k, v, pos, lengths):
    """Rotary positions and windowed attention in float32 torch operations."""
    f = 10000.0 ** (-torch.arange(D // 2, device=q.device) / (D // 2))
    t = pos.double() * f
    c, s = t.cos().float()[:, None], t.sin().float()[:, None]

    def turn(x):
        a, b = x.float()[..., :D // 2], x.float()[..., D // 2:]
        return torch.cat((a * c - b * s, a * s + b * c), -1).to(BF).float()

    q, k = turn(q).transpose(1, 2), turn(k).transpose(1, 2).repeat_interleave(H // K, 1)
    v = v.float().transpose(1, 2).repeat_interleave(H // K, 1)
    seen = so.window_mask(S, WINDOW, SINKS, q.device)[None, None] & (torch.arange(S, device=q.device) < lengths[:, None, None, None])
    w = torch.softmax((q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill(~seen, -torch.inf), -1)
    o = (w @ v).transpose(1, 2)
    return torch.where((torch.arange(S, device=q.device) < lengths[:, None])[:, :, None, None], o, 0.0).to(BF)


def _loss(plain=False):
    def loss_fn(p, ctx, batch, rng):
        tokens, labels, lengths = batch
        pos = torch.arange(S, device=tokens.device)[:, None]
        x = ctx.table_lookup(p, ("emb",), tokens)
        qkv = ctx.linear(p, ("qkv",), x).view(B, S, H + 2 * K, D)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + K], qkv[:, :, H + K:]
        if plain:
            a = _plain_attention(q, k, v, pos, lengths)
        else:
            q, k = zg.rotary(q, k, pos, (D,))
            a = zg.window_attention(q, k, v, WINDOW, SINKS, lengths)
        x = ctx.linear(p, ("o",), a.reshape(B, S, H * D), residual=x)
        return ctx.tied_logits_cross_entropy(p, ("emb",), x, labels, reduction="mean"), None

    return loss_fn


def test_a_generation_with_rotary_and_windowed_attention(cuda):
    """Losses against plain attention; the same in chunks, stepped and captured."""
    params, manifest, batch = _model(cuda)
    opt = zg.ZeroGrad(manifest, zg.sgd(0.01), P, RANK, SIGMA, 0, "sequence-lm")
    losses = opt.evaluate_shard(params, 0, _loss(), batch, range(P))
    plain = opt.evaluate_shard(params, 0, _loss(plain=True), batch, range(P))
    assert torch.isfinite(losses).all() and losses.unique().numel() == P
    torch.testing.assert_close(losses, plain, rtol=5e-3, atol=0)
    chunked = zg.ZeroGrad(manifest, zg.sgd(0.01), P, RANK, SIGMA, 0, "sequence-lm", chunk_size=2)
    assert torch.equal(chunked.evaluate_shard(params, 0, _loss(), batch, range(P)), losses)
    assert torch.equal(opt.evaluate_shard(params, 0, _loss(), batch, range(2, 5)), losses[2:5])
    state = opt.init(params)
    stepped, state1, metrics = opt.step(state, params, batch, _loss())
    assert metrics.mean_loss == pytest.approx(float(losses.mean()), rel=1e-6)
    captured = opt.capture(params, _loss(), batch)
    got, _, m = captured.step(state, batch)
    for n in SHAPES:
        assert torch.equal(stepped[n], got[n]) and not torch.equal(stepped[n], params[n])
    assert m.mean_loss == metrics.mean_loss and L.load().zg_device_error(1) == 0


@pytest.mark.parametrize("window", [None, 64])
def test_a_fitness_of_generated_answers(cuda, window):
    """Prompts into a paged cache that already holds a long context, then token
    after token: a candidate's loss does not depend on who is evaluated with
    it, and the population takes its step from the losses."""
    params, manifest, (tokens, labels, lengths) = _model(cuda)
    page, T, context = 16, 5, 1500
    pages = -(-(context + S + T) // page)
    g = torch.Generator(device=cuda).manual_seed(2)
    k0, v0 = (torch.randn(P * B * pages, page, K, D, generator=g, device=cuda).to(BF) for _ in range(2))
    tables = torch.randperm(P * B * pages, generator=g, device=cuda).reshape(P, B, pages).to(torch.int32)
    had = torch.full((B,), context, dtype=torch.int32, device=cuda)
    base = zg.step_key(0, "answers", 0, 1)
    keys = _ops.launch_fold_in(base, torch.arange(P, dtype=torch.int32, device=cuda))
    rows = torch.arange(B, device=cuda)

    def losses_of(who):
        kp, vp = k0.clone(), v0.clone()

        def project(ctx, x):
            qkv = ctx.linear(params, ("qkv",), x).view(*x.shape[:-1], H + 2 * K, D)
            return qkv[..., :H, :], qkv[..., H:H + K, :], qkv[..., H + K:, :]

        def answer(key, table):
            ctx = zg.CandidateContext(manifest, key, RANK, SIGMA)
            q, k, v = project(ctx, ctx.table_lookup(params, ("emb",), tokens))
            q, k = zg.rotary(q, k, context + torch.arange(S, device=cuda)[:, None], (D,))
            n = zg.append_pages(kp, vp, k, v, table, had, counts=lengths)
            loss = 0.0
            for t in range(T):
                x = ctx.table_lookup(params, ("emb",), tokens[:, t])
                q, k, v = project(ctx, x[:, None])
                q, k = zg.rotary(q, k, n[:, None, None], (D,))
                n = zg.append_pages(kp, vp, k, v, table, n)
                a = zg.paged_attention(q[:, 0], kp, vp, table, n, window, SINKS)
                x = ctx.linear(params, ("o",), a.reshape(B, H * D), residual=x)
                loss = loss + ctx.tied_logits_cross_entropy(params, ("emb",), x, labels[rows, t], reduction="mean")
            return loss / T

        return torch.func.vmap(answer)(keys.view(torch.int32)[who].view(torch.uint32), tables[who])

    everyone = torch.arange(P, device=cuda)
    L.profile_begin()
    losses = losses_of(everyone)
    launches = L.profile_end()
    assert sum(c for name, (c, _) in launches.items() if name == "paged_attention") == T  # one for all candidates
    assert torch.isfinite(losses).all() and losses.unique().numel() == P
    for who in (everyone[:2], everyone[3:], everyone[[5, 0, 2]]):
        assert torch.equal(losses_of(who), losses[who])
    opt = zg.ZeroGrad(manifest, zg.sgd(0.01), P, RANK, SIGMA, 0, "answers")
    new, state, metrics = opt.step_from_losses(opt.init(params), params, losses)
    assert state.generation == 1 and metrics.min_loss == float(losses.min())
    assert all(torch.isfinite(new[n]).all() and not torch.equal(new[n], params[n]) for n in SHAPES)
    assert L.load().zg_device_error(1) == 0
