"""training.windowed_attention: autograd through norms, rotation and windowed attention of packed heads, against the
operators one by one (the same bits) and against 64-bit gradients.

A gradient of the attention is off by e, elementwise at most u (|d| + c M) + 3 SLACK M as for the operator alone.  The norm's
gradient is linear in it: dx = r (w o e' - xh mean(w o e' o xh)) with e' a rotation of e, so an element of a head is off by
at most r max|w| |e| (1 + |xh| / sqrt(D)) with |e| the head's 2-norm, and a weight's gradient by sums of |xh| |e|; its own
rounding adds u |dx|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from slsmi import _lib, ops, training
from test_window_gpu import DEV, DTYPES, SLACK, attention64, close, freqs_of, norm_rope64, rnd, unit

CASES = [  # B, T, heads, kv_heads, D, left, right, sinks, lengths, R, interleaved
    (2, 70, 4, 2, 64, 16, 4, 3, [70, 33], 64, False), (1, 201, 2, 2, 128, None, 0, 0, None, 96, False),
    (3, 40, 3, 1, 64, 7, 0, 40, [1, 0, 40], 32, True), (1, 1, 1, 1, 128, 0, 0, 0, None, 0, False)]


def inputs(B, T, H, Hk, D, R, dtype):
    qkv = rnd(B, T, (H + 2 * Hk) * D, seed=T + D, dtype=dtype)
    return qkv, 1 + 0.3 * rnd(D, seed=1), 1 + 0.3 * rnd(D, seed=2), freqs_of(R), rnd(B, T, H, D, seed=3, dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_gradients(case, dtype):
    B, T, H, Hk, D, left, right, sinks, lens, R, inter = case
    qkv, wq, wk, fr, do = inputs(B, T, H, Hk, D, R, dtype)
    nf = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = training.windowed_attention(leaves[0], H, Hk, left, right, sinks, nf, None, leaves[1], leaves[2], fr, eps=1e-5,
                                      interleaved=inter)
    gx, gq, gk = torch.autograd.grad(out, leaves, do)
    # the operators one by one
    n = H + Hk
    qk = ops.qk_norm_rope(qkv, H, Hk, wq, wk, fr, eps=1e-5, interleaved=inter).view(B, T, n, D)
    v = qkv.view(B, T, n + Hk, D)[:, :, n:]
    want_out, lse = ops.window_attention(qk[:, :, :H], qk[:, :, H:], v, left, right, sinks, nf, return_lse=True)
    dq, dk, dv = ops.window_attention_backward(do, qk[:, :, :H], qk[:, :, H:], v, want_out, lse, left, right, sinks, nf)
    d, dwq, dwk = ops.qk_norm_rope_backward(torch.cat((dq, dk), 2).view(B, T, n * D), qkv, H, Hk, wq, wk, fr, eps=1e-5,
                                            interleaved=inter)
    assert torch.equal(out, want_out) and torch.equal(gx, torch.cat((d, dv.reshape(B, T, -1)), 2))
    assert torch.equal(gq, dwq) and torch.equal(gk, dwk)
    # 64 bits
    r = attention64(qk[:, :, :H], qk[:, :, H:], v, lens, left, right, sinks, D ** -0.5, do)
    u = unit(dtype)
    x64 = qkv.double().view(B, T, n + Hk, D)[:, :, :n].requires_grad_()
    w64 = [wq.double().requires_grad_(), wk.double().requires_grad_()]
    per_row = torch.arange(T, device=DEV).expand(B, T)
    y = norm_rope64(x64, torch.cat((w64[0].expand(H, D), w64[1].expand(Hk, D))), per_row, fr, 1e-5, inter)
    ref = torch.autograd.grad(y, [x64] + w64, torch.cat((r["dq"], r["dk"]), 2))
    e = torch.cat([u * (r[g].abs() + 3 * r[m]) + 3 * SLACK * r[m] + 2 ** -24 for g, m in (("dq", "Mq"), ("dk", "Mk"))], 2)
    en = e.norm(dim=-1, keepdim=True)
    rs = torch.rsqrt(x64.detach().square().mean(-1, keepdim=True) + 1e-5)
    xh = (x64.detach() * rs).abs()
    wmax = max(wq.abs().max(), wk.abs().max()).double()
    close(gx.view(B, T, n + Hk, D)[:, :, :n], ref[0], u * ref[0].abs() + 1.01 * rs * wmax * en * (1 + xh / math.sqrt(D)) + 2 ** -24)
    close(gx.view(B, T, n + Hk, D)[:, :, n:], r["dv"], u * (r["dv"].abs() + r["Mv"]) + 3 * SLACK * r["Mv"] + 2 ** -24)
    for g, want, at in ((gq, ref[1], slice(0, H)), (gk, ref[2], slice(H, n))):
        close(g, want, 1.01 * (xh * en)[:, :, at].sum((0, 1, 2)) + 1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_norms_and_with_an_expanded_gradient(dtype):
    qkv, _, _, _, _ = inputs(2, 50, 4, 2, 64, 0, dtype)
    leaf = qkv.clone().requires_grad_()
    out = training.windowed_attention(leaf, 4, 2, 9, 0, 2)
    out.sum().backward()
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in qkv.split((256, 128, 128), -1))
    want, lse = ops.window_attention(q, k, v, 9, 0, 2, return_lse=True)
    grads = ops.window_attention_backward(torch.ones_like(want), q, k, v, want, lse, 9, 0, 2)
    assert torch.equal(out, want) and torch.equal(leaf.grad, torch.cat([g.reshape(2, 50, -1) for g in grads], 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_padded_frames_may_hold_anything(dtype, bad):
    """Gradients to a padded batch are those with zeros in the padding, weights' included; the padding's own are zeros."""
    qkv, wq, wk, fr, do = inputs(3, 90, 4, 2, 64, 64, dtype)
    lens = [90, 41, 0]
    nf = torch.tensor(lens, dtype=torch.int32, device=DEV)
    results = []
    for fill in (0.0, bad):
        x = qkv.clone()
        for b, n in enumerate(lens):
            x[b, n:] = fill
        leaves = [x.requires_grad_(), wq.clone().requires_grad_(), wk.clone().requires_grad_()]
        out = training.windowed_attention(leaves[0], 4, 2, 12, 3, 2, nf, None, leaves[1], leaves[2], fr)
        results.append((out,) + torch.autograd.grad(out, leaves, do))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    for b, n in enumerate(lens):
        assert bool((results[1][1][b, n:] == 0).all())


def test_half_of_the_gradients_and_a_layer_in_a_loss():
    """Only the weights ask for gradients; a loss through a projection before and after runs and gives finite ones."""
    qkv, wq, wk, fr, _ = inputs(1, 33, 2, 1, 64, 64, torch.float16)
    w = wq.clone().requires_grad_()
    training.windowed_attention(qkv, 2, 1, 5, q_weight=w, k_weight=wk, freqs=fr).float().square().mean().backward()
    assert w.grad.shape == (64,) and bool(torch.isfinite(w.grad).all()) and bool((w.grad != 0).any())
    x, proj = rnd(1, 33, 96, seed=4), rnd(96, 256, seed=5, scale=0.1).requires_grad_()
    y = training.windowed_attention((x @ proj).half(), 2, 1, 5, q_weight=wq, k_weight=wk, freqs=fr)
    (y.flatten(2) @ rnd(128, 8, seed=6, dtype=torch.float16)).float().square().mean().backward()
    assert bool(torch.isfinite(proj.grad).all()) and bool((proj.grad != 0).any())


def test_refusals():
    qkv, wq, wk, fr, _ = inputs(1, 8, 2, 1, 64, 64, torch.float16)
    for bad in (dict(q_weight=wq), dict(freqs=fr), dict(q_weight=wq[:32], k_weight=wk[:32])):
        with pytest.raises(_lib.SlsmiError):
            training.windowed_attention(qkv, 2, 1, 5, **bad)
    for x, h, kv in ((qkv[:, ::2], 2, 1), (qkv[0], 2, 1), (qkv, 2, 2), (qkv.float(), 2, 1)):
        with pytest.raises(_lib.SlsmiError):
            training.windowed_attention(x, h, kv, 5)
    x = qkv.clone().requires_grad_()
    g, = torch.autograd.grad(training.windowed_attention(x, 2, 1, 5).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):     # one differentiation only
        g.float().sum().backward()
