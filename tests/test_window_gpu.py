"""Query / key norms with rotation, windowed attention with sinks, its gradient, its single-frame form and the cache's
prefill, against plain computations in 64 bits.

Tolerances count roundings.  u = eps / 2 of the 16-bit type is the largest relative error of one rounding; a result that
is a sum of products p x with p rounded once is off by at most u sum |p| |x|, plus u times itself for its own rounding.
`slack` covers 32-bit arithmetic (scores, exponentials, sums of a few hundred terms): 2^-24 times the terms of a sum and
the magnitude of a score's exponent, well under 4e-5 of sum |p| |x| for what is drawn here."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import slsmi
from slsmi import _lib, ops

DEV = "cuda:0"
SLACK = 4e-5
DTYPES = [torch.bfloat16, torch.float16]


def rnd(*shape, seed, dtype=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g) * scale).to(DEV)
    return x if dtype is None else x.to(dtype)


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, bound, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), (what, (got - want).abs().max().item(), over.max().item(), int((over > 0).sum()))


# ---- 64-bit references -------------------------------------------------------------------------------------------------

def freqs_of(R):
    return (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).to(DEV) if R else None


def norm_rope64(x, w, positions, freqs, eps, interleaved):
    """x [..., H, D] float64 with positions [...]."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    if freqs is None:
        return y
    R = 2 * freqs.numel()
    ang = positions.double()[..., None, None] * freqs
    c, s = torch.cos(ang), torch.sin(ang)
    out = y.clone()
    i, j = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    out[..., i] = y[..., i] * c - y[..., j] * s
    out[..., j] = y[..., j] * c + y[..., i] * s
    return out


def visible(T, n, left, right, sinks):
    i, j = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)[None, :]
    left, right = (T if left is None else left), (T if right is None else right)
    return (j <= i + right) & ((j >= i - left) | (j < sinks)) & (j < n) & (i < n)


def attention64(q, k, v, lens, left, right, sinks, scale, dout=None):
    """Everything in 64 bits with the sums of magnitudes the bounds need: o, lse, A = P |V| and, with dout, the gradients
    and their magnitudes."""
    B, T, H, D = q.shape
    g = H // k.shape[2]
    r = {n: torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV) for n in ("o", "A", "dq", "Mq")}
    r.update({n: torch.zeros(B, T, k.shape[2], D, dtype=torch.float64, device=DEV) for n in ("dk", "dv", "Mk", "Mv")})
    r["lse"] = torch.full((B, H, T), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = T if lens is None else max(0, min(T, int(lens[b])))
        m = visible(T, n, left, right, sinks)
        for h in range(H):
            Q, K, V = q[b, :n, h].double(), k[b, :n, h // g].double(), v[b, :n, h // g].double()
            if n == 0:
                continue
            mm = m[:n, :n]
            S = torch.where(mm, Q @ K.t() * scale, torch.tensor(-math.inf, dtype=torch.float64, device=DEV))
            lse = torch.logsumexp(S, -1)
            P = torch.exp(S - lse[:, None])
            O = P @ V
            r["o"][b, :n, h], r["A"][b, :n, h], r["lse"][b, h, :n] = O, P @ V.abs(), lse
            if dout is not None:
                dO = dout[b, :n, h].double()
                dP = dO @ V.t()
                delta = (dO * O).sum(-1, keepdim=True)
                dS = P * (dP - delta)
                # what a rounded O adds to delta, and with it to every dS of its row
                bump = P * (dO.abs() * O.abs()).sum(-1, keepdim=True)
                r["dq"][b, :n, h] = scale * dS @ K
                r["Mq"][b, :n, h] = scale * (dS.abs() + bump) @ K.abs()
                r["dk"][b, :n, h // g] += scale * dS.t() @ Q
                r["Mk"][b, :n, h // g] += scale * (dS.abs() + bump).t() @ Q.abs()
                r["dv"][b, :n, h // g] += P.t() @ dO
                r["Mv"][b, :n, h // g] += P.t() @ dO.abs()
    return r


# ---- norms and rotation ------------------------------------------------------------------------------------------------

NORM_CASES = [  # rows, T (None: 2-D), heads, kv_heads, D, R, interleaved, positions, width beyond the heads
    (1, None, 1, 1, 64, 64, False, None, 0), (7, None, 16, 16, 64, 64, True, "far", 1024), (402, 201, 16, 16, 64, 32, False, None, 1024),
    (35, 7, 5, 1, 128, 128, False, "frames", 128), (3000, 1000, 3, 2, 128, 96, False, "far", 64), (66, 33, 6, 2, 64, 16, True, "frames", 0),
    (9, 3, 8, 8, 128, 0, False, None, 8), (5, None, 0, 3, 64, 48, False, "far", 0), (2100, None, 2, 0, 64, 64, False, None, 0)]


def norm_case(rows, T, H, Hk, D, R, inter, pos, extra, dtype):
    lead = (rows,) if T is None else (rows // T, T)
    x = rnd(*lead, (H + Hk) * D + extra, seed=rows + D, dtype=dtype, scale=1.3)
    wq, wk = 1 + 0.3 * rnd(D, seed=1), 1 + 0.3 * rnd(D, seed=2)
    g = torch.Generator().manual_seed(rows)
    per_row = torch.arange(lead[-1], device=DEV).expand(lead)
    positions = None
    if pos == "far":
        positions = torch.randint(0, 1 << 33, lead, generator=g).to(DEV)
        per_row = positions
    elif pos == "frames":
        positions = torch.randint(0, 5000, (lead[-1],), generator=g).to(DEV)
        per_row = positions.expand(lead)
    return x, wq, wk, freqs_of(R), positions, per_row


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", NORM_CASES)
def test_qk_norm_rope(case, dtype):
    rows, T, H, Hk, D, R, inter, pos, extra = case
    x, wq, wk, fr, positions, per_row = norm_case(*case, dtype)
    got = ops.qk_norm_rope(x, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter)
    W = (H + Hk) * D
    heads = x[..., :W].double().unflatten(-1, (H + Hk, D))
    w = torch.cat((wq.expand(H, D), wk.expand(Hk, D)))
    want = norm_rope64(heads, w, per_row, fr, 1e-5, inter)
    # one rounding at the end; 32-bit arithmetic on |pair| before it (a rotated value can cancel against its pair)
    size = norm_rope64(heads, w, per_row, None, 1e-5, inter).abs().amax(-1, keepdim=True)
    close(got.unflatten(-1, (H + Hk, D)), want, unit(dtype) * want.abs() + 4e-6 * size + 2 ** -25)
    # in place: the heads' columns change, the others do not
    y = x.clone()
    assert ops.qk_norm_rope(y, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter, out=y) is y
    assert torch.equal(y[..., :W], got) and torch.equal(y[..., W:], x[..., W:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", NORM_CASES)
def test_qk_norm_rope_backward(case, dtype):
    rows, T, H, Hk, D, R, inter, pos, extra = case
    x, wq, wk, fr, positions, per_row = norm_case(*case, dtype)
    W = (H + Hk) * D
    dy = rnd(*x.shape[:-1], W, seed=5, dtype=dtype)
    got, dwq, dwk = ops.qk_norm_rope_backward(dy, x, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter)
    x64 = x[..., :W].double().requires_grad_()
    w64 = [wq.double().requires_grad_(), wk.double().requires_grad_()]
    w = torch.cat((w64[0].expand(H, D), w64[1].expand(Hk, D)))
    y = norm_rope64(x64.unflatten(-1, (H + Hk, D)), w, per_row, fr, 1e-5, inter).flatten(-2)
    gx, gq, gk = torch.autograd.grad(y, [x64] + w64, dy.double(), allow_unused=True)
    gxh = gx.unflatten(-1, (H + Hk, D))
    # the terms of dx are at most r |w| |dy| each
    xh = x64.detach().unflatten(-1, (H + Hk, D))
    r = torch.rsqrt(xh.square().mean(-1, keepdim=True) + 1e-5)
    size = (r * dy.double().unflatten(-1, (H + Hk, D)).abs().amax(-1, keepdim=True) * w.detach().abs().max() * 4)
    close(got.unflatten(-1, (H + Hk, D)), gxh, unit(dtype) * gxh.abs() + 1e-5 * size + 2 ** -25)
    # weights: 32-bit sums of `rows * heads` products of magnitude |dy| |r x|: 2^-24 of the sum of magnitudes per addition
    # level; a thousandth of a percent of that sum is over a hundred times what blocked sums lose
    for d, g, h in ((dwq, gq, H), (dwk, gk, Hk)):
        want = g if g is not None else torch.zeros(D, dtype=torch.float64, device=DEV)
        mag = 4.0 * rows * max(h, 1) * (r * xh.abs()).mean() * dy.double().abs().mean()
        close(d, want, 1e-5 * mag + 1e-6)
    # the same bits again, and in place of dy
    again, q2, k2 = ops.qk_norm_rope_backward(dy.clone(), x, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter)
    assert torch.equal(again, got) and torch.equal(q2, dwq) and torch.equal(k2, dwk)
    d2 = dy.clone()
    ops.qk_norm_rope_backward(d2, x, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter, out=d2)
    assert torch.equal(d2, got)


def test_qk_norm_rope_backward_against_differences():
    """Directional derivative of sum(y o dy) in the inputs and both weights, by central differences of the 64-bit formula."""
    x, wq, wk, fr, positions, per_row = norm_case(35, 7, 5, 1, 128, 128, False, "frames", 128, torch.float16)
    dy = rnd(5, 7, 6 * 128, seed=5, dtype=torch.float16)
    got, dwq, dwk = ops.qk_norm_rope_backward(dy, x, 5, 1, wq, wk, fr, positions, eps=1e-5)
    vx, vq, vk = rnd(5, 7, 768, seed=6).double(), rnd(128, seed=7).double(), rnd(128, seed=8).double()

    def f(t):
        w = torch.cat(((wq.double() + t * vq).expand(5, 128), (wk.double() + t * vk).expand(1, 128)))
        y = norm_rope64((x[..., :768].double() + t * vx).unflatten(-1, (6, 128)), w, per_row, fr, 1e-5, False)
        return float((y.flatten(-2) * dy.double()).sum())

    num = (f(1e-5) - f(-1e-5)) / 2e-5
    parts = (got.double() * vx).sum() + (dwq.double() * vq).sum() + (dwk.double() * vk).sum()
    # roundings of `got` average out over 26880 products: u sqrt(sum (got v)^2) is one standard deviation at most
    bound = 8 * unit(torch.float16) * float((got.double() * vx).square().sum().sqrt()) + 1e-4 * abs(num)
    assert abs(num - float(parts)) < bound


def test_norm_of_zero_and_of_no_rows():
    w = torch.ones(64, device=DEV)
    z = torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV)
    assert bool((ops.qk_norm_rope(z, 1, 1, w, w, freqs_of(64)) == 0).all())
    e = torch.zeros(2, 0, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.qk_norm_rope(e, 1, 1, w, w).shape == (2, 0, 128)
    dx, dq, dk = ops.qk_norm_rope_backward(e, e, 1, 1, w, w)
    assert dx.shape == (2, 0, 128) and bool((dq == 0).all()) and bool((dk == 0).all())


# ---- windowed attention ------------------------------------------------------------------------------------------------

WIN_CASES = [  # B, T, heads, kv_heads, D, left, right, sinks, lengths
    (1, 1, 1, 1, 64, 0, 0, 0, None), (2, 5, 2, 1, 128, 1, 1, 0, [5, 0]), (1, 64, 2, 2, 64, None, None, 0, None),
    (1, 65, 3, 1, 64, None, 0, 0, None), (2, 130, 4, 2, 128, 16, 0, 4, [130, 77]), (1, 201, 2, 2, 64, 32, 32, 1, None),
    (3, 300, 2, 1, 64, 40, 7, 3, [300, 1, 129]), (1, 517, 2, 2, 64, 100, 0, 33, None), (1, 1500, 2, 1, 64, 63, 0, 4, None),
    (1, 1400, 2, 2, 128, 127, 127, 128, None), (2, 700, 1, 1, 64, 31, 5, 70, [700, 333]), (1, 1025, 1, 1, 128, None, 0, 4, None),
    (1, 257, 8, 1, 64, 0, 0, 0, None), (1, 400, 1, 1, 64, 0, 0, 40, None), (2, 33, 2, 2, 64, 4, 60, 8, [33, 31]),
    (1, 2600, 1, 1, 64, 20, 3, 100, None)]


def win_case(B, T, H, Hk, D, left, right, sinks, lens, dtype, packed=True):
    x = rnd(B, T, (H + 2 * Hk) * D, seed=T + D, dtype=dtype)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split((H * D, Hk * D, Hk * D), -1))
    nf = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    return q, k, v, nf


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", WIN_CASES)
def test_window_attention(case, dtype):
    B, T, H, Hk, D, left, right, sinks, lens = case
    q, k, v, nf = win_case(*case, dtype)
    got, lse = ops.window_attention(q, k, v, left, right, sinks, nframes=nf, return_lse=True)
    r = attention64(q, k, v, lens, left, right, sinks, D ** -0.5)
    u = unit(dtype)
    close(got, r["o"], u * (r["o"].abs() + r["A"]) + SLACK * r["A"] + 2 ** -24)
    fin = torch.isfinite(r["lse"])
    assert torch.equal(torch.isfinite(lse), fin) and bool((lse[~fin] == -math.inf).all())
    close(lse[fin], r["lse"][fin], 1e-5 + 1e-6 * r["lse"][fin].abs())
    assert torch.equal(ops.window_attention(q, k, v, left, right, sinks, nframes=nf), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", WIN_CASES)
def test_window_attention_backward(case, dtype):
    B, T, H, Hk, D, left, right, sinks, lens = case
    q, k, v, nf = win_case(*case, dtype)
    do = rnd(B, T, H, D, seed=9, dtype=dtype)
    out, lse = ops.window_attention(q, k, v, left, right, sinks, nframes=nf, return_lse=True)
    got = ops.window_attention_backward(do, q, k, v, out, lse, left, right, sinks, nframes=nf)
    r = attention64(q, k, v, lens, left, right, sinks, D ** -0.5, do)
    u = unit(dtype)
    # P or dS rounded once per product, the result once; for dq, dk the output that delta is formed from was off by up to
    # u (|o| + A), of which Mq, Mk count |o|; A enters through `bump` being formed with it (A >= |o|: twice that is enough)
    for g, n, m, c in ((got[0], "dq", "Mq", 3), (got[1], "dk", "Mk", 3), (got[2], "dv", "Mv", 1)):
        close(g, r[n], u * (r[n].abs() + c * r[m]) + 3 * SLACK * r[m] + 2 ** -24, n)
    again = ops.window_attention_backward(do, q, k, v, out, lse, left, right, sinks, nframes=nf)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_padding_and_neighbours_may_hold_anything():
    """NaN and infinities in padded rows change nothing; rows of packed buffers around the written columns stay."""
    B, T, H, Hk, D = 2, 150, 2, 1, 64
    for dtype in DTYPES:
        q, k, v, nf = win_case(B, T, H, Hk, D, 20, 4, 2, [150, 70], dtype)
        do = rnd(B, T, H, D, seed=9, dtype=dtype)
        args = dict(left=20, right=4, sinks=2, nframes=nf)
        out, lse = ops.window_attention(q, k, v, return_lse=True, **args)
        want = ops.window_attention_backward(do, q, k, v, out, lse, **args)
        dirty = [t.clone() for t in (q, k, v, do, out)]
        for t, bad in zip(dirty, (math.nan, math.inf, math.nan, -math.inf, math.nan)):
            t[1, 70:] = bad
        out2, lse2 = ops.window_attention(*dirty[:3], return_lse=True, **args)
        assert torch.equal(out2, out) and torch.equal(lse2, lse)
        assert bool((out[1, 70:] == 0).all()) and bool((lse[1, :, 70:] == -math.inf).all())
        lse2[1, :, 70:] = math.nan
        pack = torch.full((B, T, (H + 2 * Hk + 1) * D), 7.0, dtype=dtype, device=DEV)
        dq, dk, dv, rest = (t.unflatten(-1, (-1, D)) for t in pack.split((H * D, Hk * D, Hk * D, D), -1))
        got = ops.window_attention_backward(dirty[3], *dirty[:3], dirty[4], lse2, dq=dq, dk=dk, dv=dv, **args)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((rest == 7.0).all())
        assert all(bool((g[1, 70:] == 0).all()) for g in got)


@pytest.mark.parametrize("lens", [[0, 0], [-3, 500]])
def test_lengths_outside_the_batch_are_clamped(lens):
    q, k, v, nf = win_case(2, 40, 2, 2, 64, 8, 0, 1, lens, torch.float16)
    ok = [max(0, min(40, n)) for n in lens]
    out, lse = ops.window_attention(q, k, v, 8, 0, 1, nframes=nf, return_lse=True)
    ref, lref = ops.window_attention(q, k, v, 8, 0, 1, nframes=torch.tensor(ok, dtype=torch.int32, device=DEV), return_lse=True)
    assert torch.equal(out, ref) and torch.equal(lse, lref) and bool((out[0] == 0).all())
    g = ops.window_attention_backward(out, q, k, v, out, lse, 8, 0, 1, nframes=nf)
    assert all(bool(torch.isfinite(t).all()) and bool((t[0] == 0).all()) for t in g)


@pytest.mark.parametrize("D", [64, 128])
def test_strides_layouts_and_given_results(D):
    """Heads-first memory, rows of another pitch, views at an offset: the same bits as contiguous tensors."""
    B, T, H, Hk, dtype = 2, 190, 4, 2, torch.bfloat16
    q, k, v = (t.contiguous() for t in win_case(B, T, H, Hk, D, 30, 0, 4, None, dtype)[:3])
    do = rnd(B, T, H, D, seed=9, dtype=dtype)
    want, lse = ops.window_attention(q, k, v, 30, 0, 4, return_lse=True)
    grads = ops.window_attention_backward(do, q, k, v, want, lse, 30, 0, 4)
    hf = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    wide = torch.empty(B, T + 3, H + 5, D, dtype=dtype, device=DEV)[:, 2:T + 2, 1:H + 1]
    got, l2 = ops.window_attention(*hf[:3], 30, 0, 4, return_lse=True, out=wide)
    assert got is wide and torch.equal(wide, want) and torch.equal(l2, lse)
    g2 = ops.window_attention_backward(hf[3], *hf[:3], wide, l2, 30, 0, 4, dq=torch.empty_like(hf[0]), dk=torch.empty_like(hf[1]))
    assert all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_window_attention_agrees_with_the_whole_clip_kernel():
    """No limits, no sinks: the encoder's own attention (ops.attention, q scaled by 1 / 8 beforehand)."""
    B, T = 2, 201
    qkv = rnd(B * T, 3 * 1024, seed=4, dtype=torch.float16)
    ref = ops.attention(qkv, B, T).view(B, T, 16, 64)
    q, k, v = (t.unflatten(-1, (16, 64)) for t in qkv.view(B, T, 3 * 1024).split(1024, -1))
    got = ops.window_attention(q, k, v, None, None, scale=1.0)
    r = attention64(q, k, v, None, None, None, 0, 1.0)
    bound = unit(torch.float16) * (r["o"].abs() + r["A"]) + SLACK * r["A"] * 4
    close(got, r["o"], bound)
    close(got, ref.double(), 2 * bound)


def test_gradients_against_differences():
    B, T, H, Hk, D, dtype = 1, 90, 4, 2, 64, torch.float16
    q, k, v, _ = win_case(B, T, H, Hk, D, 17, 3, 2, None, dtype)
    do = rnd(B, T, H, D, seed=9, dtype=dtype)
    out, lse = ops.window_attention(q, k, v, 17, 3, 2, return_lse=True)
    grads = ops.window_attention_backward(do, q, k, v, out, lse, 17, 3, 2)
    dirs = [rnd(*t.shape, seed=20 + i).double() for i, t in enumerate((q, k, v))]

    def f(t):
        x = [a.double() + t * d for a, d in zip((q, k, v), dirs)]
        return float((attention64(*x, None, 17, 3, 2, D ** -0.5)["o"] * do.double()).sum())

    num = (f(1e-5) - f(-1e-5)) / 2e-5
    got = sum(float((g.double() * d).sum()) for g, d in zip(grads, dirs))
    noise = math.sqrt(sum(float((g.double() * d).square().sum()) for g, d in zip(grads, dirs)))
    assert abs(num - got) < 16 * unit(dtype) * noise + 1e-4 * abs(num)   # a few independent roundings per product


# ---- rolling cache -----------------------------------------------------------------------------------------------------

STEP_CASES = [  # heads, kv_heads, D, R, interleaved, norm, sinks, window, positions
    (1, 1, 64, 64, False, True, 0, 1, [0]), (16, 16, 64, 64, False, True, 4, 256, [5000]), (4, 1, 128, 64, True, True, 2, 100, [0, 1, 2, 50, 101, 102, 7777]),
    (12, 2, 64, 0, False, True, 1, 33, [-1, 3, 33, 34]), (8, 1, 128, 128, False, True, 16, 3000, [1 << 40, 12, -5]), (3, 3, 64, 0, False, False, 0, 700, [699, 700, 1500]),
    (10, 1, 64, 16, False, True, 128, 5, [130, 60]), (16, 1, 64, 64, False, True, 0, 1024, [3]), (2, 1, 128, 0, False, False, 4, 20000, [19000, 30000])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", STEP_CASES)
def test_window_attention_step(case, dtype):
    H, Hk, D, R, inter, norm, sinks, window, pos = case
    B, slots = len(pos), sinks + window
    qkv = rnd(B, (H + 2 * Hk) * D, seed=H + window, dtype=dtype, scale=1.3)
    kc, vc = (rnd(B, Hk, slots, D, seed=i, dtype=dtype) for i in (3, 4))
    for b, p in enumerate(pos):   # slots no frame has reached yet
        kc[b, :, max(p, 0):slots] = math.nan if p < slots else kc[b, :, max(p, 0):slots]
        vc[b, :, max(p, 0):slots] = math.inf if p < slots else vc[b, :, max(p, 0):slots]
    old = kc.clone(), vc.clone()
    wq, wk, fr = 1 + 0.3 * rnd(D, seed=1), 1 + 0.3 * rnd(D, seed=2), freqs_of(R)
    positions = torch.tensor(pos, dtype=torch.int64, device=DEV)
    kw = dict(q_weight=wq, k_weight=wk, freqs=fr, interleaved=inter, eps=1e-5) if norm else {}
    got = ops.window_attention_step(qkv, kc, vc, positions, H, sinks, **kw)
    x = qkv.double().unflatten(-1, (H + 2 * Hk, D))
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    if norm:
        q, k = (norm_rope64(t, w, positions, fr, 1e-5, inter) for t, w in ((q, wq), (k, wk)))
        packed = ops.qk_norm_rope(qkv, H, Hk, wq, wk, fr, positions, eps=1e-5, interleaved=inter)
    u = unit(dtype)
    for b, p in enumerate(pos):
        if p < 0:
            assert bool((got[b] == 0).all())
            assert torch.equal(kc[b].view(torch.int16), old[0][b].view(torch.int16)) and torch.equal(vc[b].view(torch.int16), old[1][b].view(torch.int16))
            continue
        at = p if p < sinks else sinks + (p - sinks) % window
        assert torch.equal(vc[b, :, at], qkv[b].unflatten(-1, (-1, D))[H + Hk:])
        if norm:
            assert torch.equal(kc[b, :, at], packed[b].unflatten(-1, (-1, D))[H:])
        else:
            assert torch.equal(kc[b, :, at], qkv[b].unflatten(-1, (-1, D))[H:H + Hk])
        rest = [i for i in range(slots) if i != at]
        for c, o in zip((kc, vc), old):
            assert torch.equal(c[b][:, rest].view(torch.int16), o[b][:, rest].view(torch.int16))
        n = min(p + 1, slots)
        K, V = (c[b, :, :n].double().repeat_interleave(H // Hk, 0) for c in (kc, vc))
        P = torch.softmax((K @ q[b][..., None])[..., 0] * D ** -0.5, -1)[:, None]
        o, A = (P @ V)[:, 0], (P @ V.abs())[:, 0]
        # q and P are held in 32 bits: one rounding, and 32-bit scores of magnitude up to |q| |k|
        close(got[b], o, u * o.abs() + 2 * SLACK * A + 2 ** -24, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hk,D,sinks,window,lens", [(1, 1, 64, 0, 1, None), (50, 2, 128, 4, 16, [50, 17, 3]), (40, 3, 64, 8, 100, [40, 0, 9]),
                                                     (300, 1, 64, 0, 7, [300, 6, 7]), (129, 2, 64, 128, 1, [129, 128])])
def test_cache_fill(T, Hk, D, sinks, window, lens, dtype):
    B, slots = len(lens) if lens else 1, sinks + window
    kv = rnd(B, T, 2 * Hk * D, seed=T, dtype=dtype)
    k, v = (t.unflatten(-1, (Hk, D)) for t in kv.split(Hk * D, -1))
    kc, vc = (torch.full((B, Hk, slots, D), 9.0, dtype=dtype, device=DEV) for _ in range(2))
    want = kc.clone(), vc.clone()
    for b in range(B):
        for p in range(lens[b] if lens else T):
            at = p if p < sinks else sinks + (p - sinks) % window
            want[0][b, :, at], want[1][b, :, at] = k[b, p], v[b, p]
    nf = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
    ops.window_cache_fill(k, v, kc, vc, sinks, nframes=nf)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def stream_of(qkv, H, Hk, D, wq, wk, fr, left, sinks):
    """A whole recording in one go: norms and rotation, windowed attention."""
    qk = ops.qk_norm_rope(qkv, H, Hk, wq, wk, fr)
    q, k = (t.unflatten(-1, (-1, D)) for t in qk.split((H * D, Hk * D), -1))
    v = qkv[..., (H + Hk) * D:].unflatten(-1, (Hk, D))
    return q, k, v, ops.window_attention(q, k, v, left, 0, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_then_steps_follow_the_whole_recording(dtype):
    """norm + rotation -> windowed attention -> prefill of two recordings of different lengths, then one frame at a time
    past the ring's end, against the whole recording's attention."""
    B, T, H, Hk, D, sinks, window = 2, 70, 4, 2, 64, 3, 20
    qkv = rnd(B, T, (H + 2 * Hk) * D, seed=8, dtype=dtype)
    wq, wk, fr = 1 + 0.3 * rnd(D, seed=1), 1 + 0.3 * rnd(D, seed=2), freqs_of(D)
    q, k, v, whole = stream_of(qkv, H, Hk, D, wq, wk, fr, window - 1, sinks)
    start = torch.tensor([31, 9], dtype=torch.int32, device=DEV)
    kc, vc = (torch.full((B, Hk, sinks + window, D), math.nan, dtype=dtype, device=DEV) for _ in range(2))
    ops.window_cache_fill(k, v, kc, vc, sinks, nframes=start)
    pos = start.long()
    A = attention64(q, k, v, None, window - 1, 0, sinks, D ** -0.5)["A"]
    for _ in range(38):
        at = torch.arange(B, device=DEV)
        got = ops.window_attention_step(qkv[at, pos], kc, vc, pos, H, sinks, q_weight=wq, k_weight=wk, freqs=fr)
        # both round the result once; the whole form also rounds q (a score moves by at most u sum |q k| / 8 <= 8 u) and P
        ref, mag = whole[at, pos].double(), A[at, pos]
        close(got, ref, unit(dtype) * (2 * ref.abs() + 17 * mag) + 4 * SLACK * mag)
        pos = pos + 1


def test_operators_in_a_captured_graph_on_a_side_stream():
    """All operators of a frame and of a training pass captured once and replayed on new contents, eager work and
    synchronizations between; two graphs captured one after the other share no workspace."""
    B, T, H, Hk, D, sinks, window, dtype = 2, 400, 4, 2, 64, 4, 200, torch.bfloat16
    wq, wk, fr = 1 + 0.3 * rnd(D, seed=1), 1 + 0.3 * rnd(D, seed=2), freqs_of(D)
    qkv = torch.empty(B, T, (H + 2 * Hk) * D, dtype=dtype, device=DEV)
    do = torch.empty(B, T, H, D, dtype=dtype, device=DEV)
    frame = torch.empty(B, (H + 2 * Hk) * D, dtype=dtype, device=DEV)
    pos = torch.empty(B, dtype=torch.int64, device=DEV)
    kc, vc = (torch.empty(B, Hk, sinks + window, D, dtype=dtype, device=DEV) for _ in range(2))

    def train():
        q, k, v, _ = stream_of(qkv, H, Hk, D, wq, wk, fr, window - 1, sinks)
        o, lse = ops.window_attention(q, k, v, window - 1, 0, sinks, return_lse=True)
        dqk = torch.empty(B, T, (H + Hk) * D, dtype=dtype, device=DEV)
        dq, dk = (t.unflatten(-1, (-1, D)) for t in dqk.split((H * D, Hk * D), -1))
        _, _, dv = ops.window_attention_backward(do, q, k, v, o, lse, window - 1, 0, sinks, dq=dq, dk=dk)
        ops.window_cache_fill(k, v, kc, vc, sinks)
        return (o, dv) + ops.qk_norm_rope_backward(dqk, qkv, H, Hk, wq, wk, fr)

    def step():
        out = ops.window_attention_step(frame, kc, vc, pos, H, sinks, q_weight=wq, k_weight=wk, freqs=fr)
        pos.add_(1)
        return (out,)

    def load(seed):
        qkv.copy_(rnd(*qkv.shape, seed=seed))
        do.copy_(rnd(*do.shape, seed=seed + 1))
        frame.copy_(rnd(*frame.shape, seed=seed + 2))
        pos.fill_(T)

    load(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for fn in (train, step):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = fn()
        graphs.append((g, res))
    for seed in (10, 20, 30):
        load(seed)
        want = [t.clone() for t in train()]
        want += [t.clone() for _ in range(3) for t in step()]
        torch.cuda.synchronize()
        load(seed)
        kc.zero_()
        graphs[0][0].replay()
        got = [t.clone() for t in graphs[0][1]]
        for _ in range(3):
            graphs[1][0].replay()
            got += [t.clone() for t in graphs[1][1]]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(pos[0]) == T + 3


def test_two_streams_at_once():
    """Two calls in flight on two streams: each has its own workspace."""
    case = (1, 2600, 2, 1, 64, 20, 3, 100, None)
    sets = []
    for seed in (1, 2):
        q, k, v = (t.unflatten(-1, (-1, 64)) for t in rnd(1, 2600, 256, seed=seed, dtype=torch.float16).split((128, 64, 64), -1))
        do = rnd(1, 2600, 2, 64, seed=seed + 5, dtype=torch.float16)
        o, lse = ops.window_attention(q, k, v, 20, 3, 100, return_lse=True)
        sets.append((do, q, k, v, o, lse))
    want = [ops.window_attention_backward(*s, 20, 3, 100) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(ops.window_attention_backward(*s, 20, 3, 100))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


# ---- refusals ----------------------------------------------------------------------------------------------------------

def test_refusals():
    x = rnd(2, 10, 4 * 64, seed=1, dtype=torch.float16)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in x.split((128, 64, 64), -1))
    w = torch.ones(64, device=DEV)
    nf = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    lse = torch.zeros(2, 2, 10, device=DEV)
    kc = torch.zeros(2, 1, 8, 64, dtype=torch.float16, device=DEV)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    f64 = freqs_of(64)
    row = rnd(2, 256, seed=1, dtype=torch.float16)
    bad = [
        lambda: ops.window_attention(q.float(), k.float(), v.float(), 4), lambda: ops.window_attention(q, k.bfloat16(), v, 4),
        lambda: ops.window_attention(q.cpu(), k.cpu(), v.cpu(), 4), lambda: ops.window_attention(q, k[:, :9], v, 4),
        lambda: ops.window_attention(q, k, v, -1), lambda: ops.window_attention(q, k, v, 4, -2), lambda: ops.window_attention(q, k, v, 4, 0, 129),
        lambda: ops.window_attention(q, k, v, 4, nframes=nf.long()), lambda: ops.window_attention(q, k, v, 4, nframes=nf[:1]),
        lambda: ops.window_attention(q, k, v, 4, scale=0.0), lambda: ops.window_attention(q, k, v, 4, scale=-1.0),
        lambda: ops.window_attention(q[..., :32], k[..., :32], v[..., :32], 4), lambda: ops.window_attention(k, q, q, 4),
        lambda: ops.window_attention(x[:, :, 4:132].unflatten(-1, (2, 64)), k, v, 4),          # 8-byte alignment
        lambda: ops.window_attention(q, k[:, :1].expand(2, 10, 1, 64), v, 4),                  # rows that share memory
        lambda: ops.window_attention(q, k, v, 4, out=torch.empty(2, 1, 2, 64, dtype=torch.float16, device=DEV).expand(2, 10, 2, 64)),
        lambda: ops.window_attention(q, k, v, 4, out=torch.empty(1, 10, 2, 64, dtype=torch.float16, device=DEV).expand(2, 10, 2, 64)),
        lambda: ops.window_attention_backward(q, q, k, v, q, lse[:, :1], 4), lambda: ops.window_attention_backward(q, q, k, v, q, lse.double(), 4),
        lambda: ops.qk_norm_rope(x, 2, 1, w[:32], w[:32]), lambda: ops.qk_norm_rope(x, 4, 1, w, w), lambda: ops.qk_norm_rope(x, 2, 1, w.half(), w),
        lambda: ops.qk_norm_rope(x, 2, 1, w, w, f64.float()), lambda: ops.qk_norm_rope(x, 2, 1, w, w, f64[:5]),
        lambda: ops.qk_norm_rope(x, 2, 1, w, w, f64, pos), lambda: ops.qk_norm_rope(x[:, ::2][:, :3], 2, 1, w, w),
        lambda: ops.qk_norm_rope(x.float(), 2, 1, w, w), lambda: ops.qk_norm_rope(x, 0, 0, w, w), lambda: ops.qk_norm_rope(x, 2, 1, w, w.cpu()),
        lambda: ops.window_attention_step(row, kc, kc, pos, 2, 8), lambda: ops.window_attention_step(row, kc, kc[:, :, :4], pos, 2, 1),
        lambda: ops.window_attention_step(row, kc, kc.clone(), pos.int(), 2, 1), lambda: ops.window_attention_step(row, kc, kc.clone(), pos, 3, 1),
        lambda: ops.window_attention_step(row, kc, kc.clone(), pos, 2, 1, freqs=f64), lambda: ops.window_attention_step(row, kc, kc.clone(), pos, 2, 1, q_weight=w),
        lambda: ops.window_attention_step(row.bfloat16(), kc, kc.clone(), pos, 2, 1), lambda: ops.window_cache_fill(k, v, kc[:1], kc[:1], 1),
        lambda: ops.window_cache_fill(k, v, kc, kc.clone(), -1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.SlsmiError):
            f()
            print("not refused:", i)


@pytest.mark.parametrize("power", [-14, -7, 6])
def test_half_precision_gradients_follow_small_and_large_dout(power):
    """Gradients are linear in dout: scaled by a power of two they keep their bits, but for what falls below half
    precision's normal range (spacing 2^-24, so 2^-25 per rounding of the result, and of a 16-bit dout itself)."""
    case = (1, 700, 2, 1, 64, None, 0, 0, None)
    q, k, v, _ = win_case(*case, torch.float16)
    do = rnd(1, 700, 2, 64, seed=9, dtype=torch.float16)
    small = (do.float() * 2.0 ** power).to(torch.float16)
    out, lse = ops.window_attention(q, k, v, None, 0, return_lse=True)
    r = attention64(q, k, v, None, None, 0, 0, 64 ** -0.5, small)
    got = ops.window_attention_backward(small, q, k, v, out, lse, None, 0)
    u = unit(torch.float16)
    for g, n, m, c in ((got[0], "dq", "Mq", 3), (got[1], "dk", "Mk", 3), (got[2], "dv", "Mv", 1)):
        close(g, r[n], u * (r[n].abs() + c * r[m]) + 3 * SLACK * r[m] + 2.0 ** -25, n)


@pytest.mark.parametrize("window", [(None, 0, 0), (12, 4, 0), (40, 0, 70)])
def test_half_precision_gradients_under_a_loss_scale(window):
    """dout of thousands against values of tens to a hundred: dS itself passes half precision's largest value, the gradients do not."""
    left, right, sinks = window
    q, k, v, _ = win_case(1, 300, 2, 1, 64, left, right, sinks, None, torch.float16)
    v = v * 32
    do = rnd(1, 300, 2, 64, seed=9, dtype=torch.float16) * 2048
    args, scale = (left, right, sinks), 2.0 ** -10
    out, lse = ops.window_attention(q, k, v, *args, scale=scale, return_lse=True)
    r = attention64(q, k, v, None, *args, scale, do)
    assert bool((r["dq"].abs().max() < 60000) & (r["dk"].abs().max() < 60000) & (r["dv"].abs().max() < 60000))
    got = ops.window_attention_backward(do, q, k, v, out, lse, *args, scale=scale)
    u = unit(torch.float16)
    for g, n, m, c in ((got[0], "dq", "Mq", 3), (got[1], "dk", "Mk", 3), (got[2], "dv", "Mv", 1)):
        close(g, r[n], u * (r[n].abs() + c * r[m]) + 3 * SLACK * r[m] + 2 ** -24, n)


def test_half_precision_gradient_of_quiet_rows_beside_loud_ones():
    """A row's dq keeps its own precision however large its neighbours' dout is (2^3 against 2^-20 in turn)."""
    q, k, v, _ = win_case(1, 200, 1, 1, 128, 1, 1, 0, None, torch.float16)
    q, k = q / 1024, k * 1024
    do = rnd(1, 200, 1, 128, seed=9) * torch.where(torch.arange(200, device=DEV) % 2 == 0, 8.0, 2.0 ** -20)[None, :, None, None]
    do = do.half()
    out, lse = ops.window_attention(q, k, v, 1, 1, return_lse=True)
    r = attention64(q, k, v, None, 1, 1, 0, 128 ** -0.5, do)
    assert bool(r["dq"].abs().max() < 60000)
    dq, _, _ = ops.window_attention_backward(do, q, k, v, out, lse, 1, 1)
    u = unit(torch.float16)
    close(dq, r["dq"], u * (r["dq"].abs() + 3 * r["Mq"]) + 3 * SLACK * r["Mq"] + 2 ** -25, "dq")


@pytest.mark.parametrize("size", [1000.0, 2.0 ** -9])
def test_half_precision_key_gradients_with_large_and_small_values(size):
    """dK under a loss scale, values of a thousand; and with values of thousandths beside ordinary ones in turn."""
    q, k, v, _ = win_case(1, 300, 2, 1, 64, 20, 20, 0, None, torch.float16)
    v = v * torch.where(torch.arange(300, device=DEV) % 2 == 0, size, 1.0).half()[None, :, None, None]
    do = rnd(1, 300, 2, 64, seed=9, dtype=torch.float16) * (256 if size > 1 else 2.0 ** -6)
    scale = 2.0 ** (-10 if size > 1 else -3)
    out, lse = ops.window_attention(q, k, v, 20, 20, scale=scale, return_lse=True)
    r = attention64(q, k, v, None, 20, 20, 0, scale, do)
    assert bool((r["dk"].abs().max() < 60000) & (r["dv"].abs().max() < 60000))
    _, dk, dv = ops.window_attention_backward(do, q, k, v, out, lse, 20, 20, scale=scale)
    u = unit(torch.float16)
    for g, n, m, c in ((dk, "dk", "Mk", 3), (dv, "dv", "Mv", 1)):
        close(g, r[n], u * (r[n].abs() + c * r[m]) + 3 * SLACK * r[m] + 2 ** -25, n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_reach_what_sees_them(dtype):
    """A NaN among the values makes the rows that see it NaN, one in dout its row's dq and the dv of the keys it sees; the
    norms keep one, and an infinity in dout stays out of range rather than becoming a large number."""
    case = (1, 300, 2, 2, 64, 20, 4, 0, None)
    q, k, v, _ = win_case(*case, dtype)
    do = rnd(1, 300, 2, 64, seed=9, dtype=dtype)
    out, lse = ops.window_attention(q, k, v, 20, 4, return_lse=True)
    bad = v.clone()
    bad[0, 100, 1, 7] = math.nan
    got = ops.window_attention(q, k, bad, 20, 4)
    assert bool(got[0, 96:121, 1, 7].isnan().all())
    far = torch.ones(300, dtype=torch.bool, device=DEV)
    far[0:256] = False     # (tiles of up to 64 keys, workgroups of 128 rows: beyond these nothing is near)
    assert torch.equal(got[:, far], out[:, far]) and torch.equal(got[:, :, 0], out[:, :, 0])
    for value in (math.nan, math.inf):
        bad = do.clone()
        bad[0, 100, 1, 7] = value
        dq, dk, dv = ops.window_attention_backward(bad, q, k, v, out, lse, 20, 4)
        assert not bool(dq[0, 100, 1].isfinite().any()) and not bool(dv[0, 80:105, 1, 7].isfinite().any())
        assert not bool(dk[0, 80:105, 1].isfinite().any())
        assert all(bool(t[:, :, 0].isfinite().all()) and bool(t[:, 256:].isfinite().all()) for t in (dq, dk, dv))
    x = rnd(5, 3 * 64, seed=4, dtype=dtype)
    x[2, 70] = math.nan
    w = torch.ones(64, device=DEV)
    y = ops.qk_norm_rope(x, 2, 1, w, w, freqs_of(64))
    assert bool(y[2, 64:128].isnan().all()) and int(y.isnan().sum()) == 64
    dx, dwq, dwk = ops.qk_norm_rope_backward(rnd(5, 192, seed=5, dtype=dtype), x, 2, 1, w, w, freqs_of(64))
    assert bool(dx[2, 64:128].isnan().all()) and int(dx.isnan().sum()) == 64 and bool(dwk.isfinite().all())
    assert bool(dwq.isnan().all())
    cache = [rnd(1, 2, 40, 64, seed=i, dtype=dtype) for i in (6, 7)]
    cache[1][0, 1, 3, 5] = math.nan
    o = ops.window_attention_step(rnd(1, 6 * 64, seed=8, dtype=dtype), *cache, torch.tensor([100], device=DEV), 2, 0)
    assert bool(o[0, 1, 5].isnan()) and int(o.isnan().sum()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_and_frequencies_at_odd_addresses(dtype):
    """fp32 weights one value past an aligned address and float64 frequencies one value past one: the same results."""
    x, wq, wk, fr, _, _ = norm_case(35, 7, 5, 1, 128, 96, False, None, 128, dtype)
    odd = [torch.cat((w[:1], w))[1:] for w in (wq, wk, fr)]
    assert all(w.data_ptr() % 16 for w in odd)
    dy = rnd(5, 7, 768, seed=5, dtype=dtype)
    assert torch.equal(ops.qk_norm_rope(x, 5, 1, *odd), ops.qk_norm_rope(x, 5, 1, wq, wk, fr))
    for a, b in zip(ops.qk_norm_rope_backward(dy, x, 5, 1, *odd), ops.qk_norm_rope_backward(dy, x, 5, 1, wq, wk, fr)):
        assert torch.equal(a, b)
    results = []
    for w in ((wq, wk, fr), odd):
        cache = [rnd(35, 1, 40, 128, seed=i, dtype=dtype) for i in (6, 7)]
        p = torch.arange(35, device=DEV) * 3
        results.append([ops.window_attention_step(x.view(35, 896)[:, :896], *cache, p, 5, 4, *w)] + cache)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 1300, 2, 1, 64, None, 0, 0, None), (2, 1100, 2, 2, 64, 300, 300, 4, [1100, 700]),
                                  (1, 1700, 2, 1, 64, 200, 0, 128, None), (3, 500, 2, 1, 128, 90, 90, 0, [500, 0, 411]),
                                  (1, 1600, 1, 1, 128, 180, 3, 40, [1500])])
def test_window_attention_of_many_keys(case, dtype):
    """Rows that see hundreds of keys, some through far sinks: forward and gradients."""
    test_window_attention(case, dtype)
    test_window_attention_backward(case, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(16, 4, 128, 0, False, False, 16, 20000, [25000]), (1, 1, 64, 64, False, True, 4, 20000, [19990, -1]),
                                  (24, 3, 64, 32, False, True, 0, 12000, [11999]), (7, 1, 128, 128, True, True, 3, 9000, [40, -3, 9003]),
                                  (5, 1, 64, 64, False, True, 1, 31, [0, 31, 32, 63])])
def test_window_attention_step_of_long_and_of_grouped_caches(case, dtype):
    """Shares joined by both forms of the join, groups of three to eight heads and not a multiple of them, shares without a
    slot and streams without a frame."""
    test_window_attention_step(case, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(2, 330, 8, 1, 64, 28, 28, 1, [330, 100]), (1, 500, 6, 2, 128, None, 0, 0, None), (1, 700, 12, 2, 64, 60, 0, 70, [650]),
                                  (2, 260, 10, 1, 64, None, None, 0, [260, 0]), (1, 33, 4, 1, 128, 5, 5, 33, None), (1, 1200, 16, 2, 64, 250, 250, 40, None)])
def test_window_attention_with_shared_heads(case, dtype):
    """Several query heads to a key head and few key tiles: the heads' sums for a key come from several workgroups."""
    test_window_attention(case, dtype)
    test_window_attention_backward(case, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(2, 200, 4, 4, 64, 1, 0, 0, [200, 77]), (2, 150, 4, 2, 128, 2, 2, 0, None), (1, 300, 2, 1, 64, 4, 0, 1, None),
                                  (3, 29, 4, 1, 64, None, 0, 0, [29, 1, 0]), (1, 400, 2, 2, 64, 5, 0, 10, [390]), (2, 48, 6, 2, 128, None, None, 0, None)])
def test_gradients_of_rows_that_see_a_handful_of_keys(case, dtype):
    """Neither the rounding of the saved output nor that of dS shows: dq and dk are off by their own rounding and what two
    16-bit operands leave of dS (2^-17 or 2^-22 of each term; u 2^-7 is more) and 32-bit arithmetic."""
    B, T, H, Hk, D, left, right, sinks, lens = case
    q, k, v, nf = win_case(*case, dtype)
    do = rnd(B, T, H, D, seed=9, dtype=dtype)
    out, lse = ops.window_attention(q, k, v, left, right, sinks, nframes=nf, return_lse=True)
    dq, dk, _ = ops.window_attention_backward(do, q, k, v, out, lse, left, right, sinks, nframes=nf)
    r = attention64(q, k, v, lens, left, right, sinks, D ** -0.5, do)
    u = unit(dtype)
    for g, n, m in ((dq, "dq", "Mq"), (dk, "dk", "Mk")):
        close(g, r[n], u * (r[n].abs() + r[m] * 2 ** -7) + 3 * SLACK * r[m] + 2 ** -24, n)


def test_grouped_heads_in_a_captured_graph():
    """Shared key heads: forward, gradient (heads shared among workgroups, sums joined) and a step on the matrix units,
    captured once and replayed on new inputs with eager work in between."""
    q, k, v, nf = win_case(2, 330, 8, 1, 64, 28, 28, 1, [330, 100], torch.float16)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    do = rnd(2, 330, 8, 64, seed=9, dtype=torch.float16)
    row = rnd(2, 10 * 64, seed=11, dtype=torch.float16)
    cache = [rnd(2, 1, 600, 64, seed=i, dtype=torch.float16) for i in (6, 7)]
    pos = torch.tensor([700, 20], device=DEV)

    def run():
        out, lse = ops.window_attention(q, k, v, 28, 28, 1, nframes=nf, return_lse=True)
        grads = ops.window_attention_backward(do, q, k, v, out, lse, 28, 28, 1, nframes=nf)
        return (out, lse) + grads + (ops.window_attention_step(row, *cache, pos, 8, 4),)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        for t, s in ((q, 20), (k, 30), (v, 40), (do, 50)):
            t.copy_(rnd(*t.shape, seed=s + i, dtype=torch.float16))
        pos += 1
        before = [c.clone() for c in cache]
        graph.replay()
        torch.cuda.synchronize()
        after = [c.clone() for c in cache]
        for c, b in zip(cache, before):
            c.copy_(b)
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and all(torch.equal(a, b) for a, b in zip(after, cache))


@pytest.mark.parametrize("dtype", DTYPES)
def test_result_in_the_place_of_the_queries_and_refused_places(dtype):
    q, k, v, nf = win_case(2, 300, 4, 4, 64, 40, 7, 3, [300, 129], dtype)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    want, lse = ops.window_attention(q, k, v, 40, 7, 3, nframes=nf, return_lse=True)
    own = q.clone()
    assert torch.equal(ops.window_attention(own, k, v, 40, 7, 3, nframes=nf, out=own), want) and torch.equal(own, want)
    do = rnd(2, 300, 4, 64, seed=9, dtype=dtype)
    for bad in (lambda: ops.window_attention(q, k, v, 40, 7, 3, out=k), lambda: ops.window_attention(q, k, v, 40, 7, 3, out=v),
                lambda: ops.window_attention_backward(do, q, k, v, want, lse, 40, 7, 3, dq=do),
                lambda: ops.window_attention_backward(do, q, k, v, want, lse, 40, 7, 3, dk=k),
                lambda: ops.window_attention_backward(do, q, k, v, want, lse, 40, 7, 3, dq=own, dk=own)):
        with pytest.raises(_lib.SlsmiError):
            bad()
