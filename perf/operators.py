"""Measured cases of the windowed-attention operators: slsmi.ops.qk_norm_rope (and its backward), window_attention (and
its backward), window_attention_step and window_cache_fill.

`run` with `own` false is the plain form: elementary torch operations in 32 bits (rotation angles in 64), rounded once at
the end.  With `own` true it makes the calls a user makes.  `exact` computes the same results in 64 bits.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one clip of 4.04 s (201 frames) through one layer's query / key norms: launch latency
        dict(name="norm one clip", op="norm", B=1, T=201, Hq=16, Hk=16, D=64, R=64, interleaved=False, far=0, dtype="f16"),
        # minutes of audio in one batch, grouped heads, half of every head rotated, positions deep in a stream
        dict(name="norm long batch", op="norm", B=8, T=2999, Hq=32, Hk=8, D=128, R=64, interleaved=False, far=1 << 20,
             dtype="bf16"),
        # a training batch of 40 s recordings: gradients of the rows and of both weights
        dict(name="norm backward", op="norm_bwd", B=5, T=2003, Hq=16, Hk=16, D=64, R=64, interleaved=True, far=0,
             dtype="bf16"),
        # one second of audio (49 frames), two-sided window: the smallest scoring call
        dict(name="attend one second", op="attn", B=1, T=49, Hq=16, Hk=16, D=64, left=32, right=32, sinks=1, ragged=False,
             dtype="f16"),
        # a recording of 164 s, one-sided window of 1024 frames, four first frames kept, grouped wide heads
        dict(name="attend long causal", op="attn", B=1, T=8192, Hq=16, Hk=4, D=128, left=1023, right=0, sinks=4,
             ragged=False, dtype="bf16"),
        # a padded batch of recordings of different lengths, two-sided window, forward and backward
        dict(name="train ragged batch", op="attn_train", B=4, T=1001, Hq=16, Hk=16, D=64, left=100, right=100, sinks=1,
             ragged=True, dtype="f16"),
        # a long recording, forward and backward
        dict(name="train long causal", op="attn_train", B=1, T=8192, Hq=16, Hk=16, D=64, left=511, right=0, sinks=4,
             ragged=False, dtype="bf16"),
        # one live stream, one new frame: launch latency
        dict(name="step one stream", op="step", B=1, Hq=16, Hk=16, D=64, R=64, window=256, sinks=4, norm=True, far=5000,
             dtype="f16"),
        # 64 live streams with 20 s of context each
        dict(name="step many streams", op="step", B=64, Hq=16, Hk=16, D=64, R=64, window=1023, sinks=4, norm=True, far=9000,
             dtype="f16"),
        # one stream with eleven minutes of context, grouped wide heads: few rows, a long axis
        dict(name="step long context", op="step", B=1, Hq=16, Hk=4, D=128, R=128, window=32768, sinks=16, norm=False,
             far=1 << 21, dtype="bf16"),
        # prefill of one stream's cache after a clip shorter than the window
        dict(name="fill short", op="fill", B=1, T=201, Hk=16, D=64, window=256, sinks=4, ragged=False, dtype="f16"),
        # prefill of eight streams after long recordings of different lengths
        dict(name="fill long", op="fill", B=8, T=4003, Hk=16, D=64, window=2048, sinks=4, ragged=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "attn", "attn", "attn_train", "attn_train", "step", "step", "fill"])
    dtype = rng.choice(["bf16", "f16"])
    D = rng.choice([64, 128])
    Hq, Hk = rng.choice([(16, 16), (16, 4), (8, 8), (8, 1), (12, 12), (6, 2)])
    if op in ("norm", "norm_bwd"):
        rows = _log(rng, 1, 20000)
        B = rng.choice([1, 2, 5, 8])
        return dict(op=op, B=B, T=max(1, rows // B), Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D // 2]),
                    interleaved=rng.random() < 0.5, far=rng.choice([0, 1 << 20]), dtype=dtype)
    if op in ("attn", "attn_train"):
        T = _log(rng, 1, 7000)
        B = _log(rng, 1, max(1, min(16, (1 << 30) // (2 * Hq * T * T))))
        left = rng.choice([_log(rng, 1, max(2, T)), _log(rng, 16, 600), -1])
        case = dict(op=op, B=B, T=T, Hq=Hq, Hk=Hk, D=D, left=left, right=rng.choice([0, left]),
                    sinks=rng.choice([0, 1, 4, 64]), ragged=B > 1 and rng.random() < 0.5, dtype=dtype)
        while work(case)["flops"] > 5e10:   # no dearer than the listed ones
            case["T"] = case["T"] * 3 // 4
        return case
    if op == "step":
        window = _log(rng, 1, 30000)
        B = _log(rng, 1, max(1, min(64, (1 << 16) // window)))
        return dict(op=op, B=B, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D // 2]), window=window, sinks=rng.choice([0, 1, 4, 64]),
                    norm=rng.random() < 0.5, far=_log(rng, 1, 1 << 20), dtype=dtype)
    T = _log(rng, 1, 5000)
    B = rng.choice([1, 3, 8])
    return dict(op=op, B=B, T=T, Hk=Hk, D=D, window=_log(rng, 1, 4000), sinks=rng.choice([0, 1, 4, 64]), ragged=B > 1,
                dtype=dtype)


def _lengths(case):
    """Frames of every recording: the full length, then shorter ones."""
    return [case["T"] - (b * case["T"]) // (2 * case["B"]) if case["ragged"] else case["T"] for b in range(case["B"])]


def _positions_now(case):
    """Index of every stream's new frame: streams that began at different times."""
    return [case["far"] + 37 * b for b in range(case["B"])]


def _visible_pairs(case):
    total = 0
    left = case["left"] if case["left"] >= 0 else case["T"]
    right = case["right"] if case["right"] >= 0 else case["T"]
    for n in _lengths(case):
        i = np.arange(n, dtype=np.int64)
        last = np.minimum(i + right, n - 1)
        first = np.maximum(i - left, 0)
        total += int((last - first + 1).sum() + np.minimum(np.minimum(case["sinks"], first), last + 1).sum())
    return total


def work(case):
    op, D = case["op"], case["D"]
    if op in ("norm", "norm_bwd"):
        n = case["B"] * case["T"] * (case["Hq"] + case["Hk"]) * D
        return {"bytes": n * (4 if op == "norm" else 6), "flops": n * (8 if op == "norm" else 16)}
    if op in ("attn", "attn_train"):
        rows = case["B"] * case["T"]
        q, kv = rows * case["Hq"] * D * 2, rows * case["Hk"] * D * 2
        pairs = _visible_pairs(case) * case["Hq"]
        if op == "attn":
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + 4 * kv + rows * case["Hq"] * 4, "flops": 14 * D * pairs}
    slots = case["window"] + case["sinks"]
    if op == "step":
        n = sum(min(p + 1, slots) for p in _positions_now(case))
        return {"bytes": 4 * n * case["Hk"] * D + 4 * case["B"] * (case["Hq"] + case["Hk"]) * D,
                "flops": 4 * n * case["Hq"] * D}
    n = sum(min(t, slots) for t in _lengths(case))
    return {"bytes": 8 * n * case["Hk"] * D, "flops": 0}


# ---- what a program has in hand -------------------------------------------------------------------------------------

def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _norm_params(g, case):
    R = case["R"]
    return dict(wq=1.0 + 0.2 * torch.randn(case["D"], generator=g, device=DEV),
                wk=1.0 + 0.2 * torch.randn(case["D"], generator=g, device=DEV),
                freqs=10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, op, D = DTYPES[case["dtype"]], case["op"], case["D"]
    s = {"case": dict(case)}
    if op in ("norm", "norm_bwd"):
        B, T, H = case["B"], case["T"], case["Hq"] + case["Hk"]
        s.update(_norm_params(g, case))
        s["qkv"] = _randn(g, (B, T, (H + case["Hk"]) * D), dt, 1.3)   # what the projection of a layer writes: q | k | v
        s["positions"] = case["far"] + torch.arange(T, device=DEV)
        if op == "norm_bwd":
            s["dout"] = _randn(g, (B, T, H * D), dt)
    elif op in ("attn", "attn_train"):
        B, T, Hq, Hk = case["B"], case["T"], case["Hq"], case["Hk"]
        qkv = _randn(g, (B, T, (Hq + 2 * Hk) * D), dt)
        qkv[..., :Hq * D] *= 1.5
        s["q"], s["k"], s["v"] = _heads(qkv, Hq, Hk, D)
        s["nframes"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
        if op == "attn_train":
            s["dout"] = _randn(g, (B, T, Hq, D), dt)
    elif op == "step":
        B, Hq, Hk = case["B"], case["Hq"], case["Hk"]
        slots = case["window"] + case["sinks"]
        s.update(_norm_params(g, case))
        s["qkv"] = _randn(g, (B, (Hq + 2 * Hk) * D), dt, 1.3)
        s["k_cache"] = _randn(g, (B, Hk, slots, D), dt)
        s["v_cache"] = _randn(g, (B, Hk, slots, D), dt)
        s["positions"] = torch.tensor(_positions_now(case), dtype=torch.int64, device=DEV)
    else:
        B, T, Hk = case["B"], case["T"], case["Hk"]
        slots = case["window"] + case["sinks"]
        kv = _randn(g, (B, T, 2 * Hk * D), dt)
        _, s["k"], s["v"] = _heads(kv, 0, Hk, D)
        s["k_cache"] = torch.zeros(B, Hk, slots, D, dtype=dt, device=DEV)
        s["v_cache"] = torch.zeros(B, Hk, slots, D, dtype=dt, device=DEV)
        s["nframes"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    return s


def _heads(qkv, Hq, Hk, D):
    """Views of packed rows q | k | v as [..., heads, D]."""
    lead = qkv.shape[:-1]
    cut = (Hq * D, (Hq + Hk) * D)
    return (qkv[..., :cut[0]].view(*lead, Hq, D), qkv[..., cut[0]:cut[1]].view(*lead, Hk, D),
            qkv[..., cut[1]:].view(*lead, Hk, D))


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _cos_sin(positions, freqs):
    a = positions.to(torch.float64)[:, None] * freqs
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, interleaved, back=False):
    """x [..., H, D] float; cos, sin broadcastable to [..., 1, R / 2]."""
    R = 2 * cos.shape[-1]
    sin = -sin if back else sin
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _plain_norm(x, w, cos, sin, interleaved):
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return _rotate(n, cos, sin, interleaved)


def _plain_norm_rows(s):
    c = s["case"]
    q, k, _ = _heads(s["qkv"], c["Hq"], c["Hk"], c["D"])
    cos, sin = (t[:, None, :] for t in _cos_sin(s["positions"], s["freqs"]))
    out = torch.cat((_plain_norm(q.float(), s["wq"], cos, sin, c["interleaved"]),
                     _plain_norm(k.float(), s["wk"], cos, sin, c["interleaved"])), -2)
    return out.flatten(-2).to(s["qkv"].dtype)


def _plain_norm_backward_one(x, d, w, cos, sin, interleaved):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    dn = _rotate(d, cos, sin, interleaved, back=True)
    dw = (dn * x * r).flatten(0, -2).sum(0, dtype=torch.float64).float()
    g = dn * w
    return r * (g - x * r * r * (g * x).mean(-1, keepdim=True)), dw


def _plain_norm_backward(s):
    c = s["case"]
    q, k, _ = _heads(s["qkv"], c["Hq"], c["Hk"], c["D"])
    dq, dk = s["dout"].float().view(*q.shape[:-2], c["Hq"] + c["Hk"], c["D"]).split((c["Hq"], c["Hk"]), -2)
    cos, sin = (t[:, None, :] for t in _cos_sin(s["positions"], s["freqs"]))
    dq, dwq = _plain_norm_backward_one(q.float(), dq, s["wq"], cos, sin, c["interleaved"])
    dk, dwk = _plain_norm_backward_one(k.float(), dk, s["wk"], cos, sin, c["interleaved"])
    return torch.cat((dq, dk), -2).flatten(-2).to(s["qkv"].dtype), dwq, dwk


def _hidden(case, nframes):
    """[B or 1, 1, T, T] truth values: the pairs a query does not see."""
    T = case["T"]
    i = torch.arange(T, device=DEV)[:, None]
    j = torch.arange(T, device=DEV)[None, :]
    left = case["left"] if case["left"] >= 0 else T
    right = case["right"] if case["right"] >= 0 else T
    hide = ((j > i + right) | ((j < i - left) & (j >= case["sinks"])))[None]
    if nframes is not None:
        n = nframes[:, None, None]
        hide = hide | (j[None] >= n) | (i[None] >= n)
    return hide[:, None]


def _repeat(x, g):
    return x.repeat_interleave(g, 1) if g > 1 else x


def _plain_attention(s):
    """P, the output and the log-sum-exp in float, heads second."""
    c = s["case"]
    g = c["Hq"] // c["Hk"]
    q, k, v = s["q"].float().transpose(1, 2), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    p = torch.matmul(q, _repeat(k, g).transpose(2, 3)).mul_(c["D"] ** -0.5)
    p.masked_fill_(_hidden(c, s["nframes"]), -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = top + total.log()
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return p, torch.matmul(p, _repeat(v, g)), lse[..., 0]


def _plain_attention_forward(s):
    _, o, _ = _plain_attention(s)
    return o.transpose(1, 2).contiguous().to(s["q"].dtype)


def _plain_attention_train(s):
    c, dt = s["case"], s["q"].dtype
    g = c["Hq"] // c["Hk"]
    B, T, Hq, Hk, D = c["B"], c["T"], c["Hq"], c["Hk"], c["D"]
    p, o, lse = _plain_attention(s)
    d = s["dout"].float().transpose(1, 2)
    q, k, v = s["q"].float().transpose(1, 2), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(2, 3), d)
    ds = torch.matmul(d, _repeat(v, g).transpose(2, 3)).sub_((d * o).sum(-1, keepdim=True)).mul_(p).mul_(D ** -0.5)
    dq = torch.matmul(ds, _repeat(k, g))
    dk = torch.matmul(ds.transpose(2, 3), q)
    dk, dv = dk.view(B, Hk, g, T, D).sum(2), dv.view(B, Hk, g, T, D).sum(2)
    return [t.transpose(1, 2).contiguous().to(dt) for t in (o, dq, dk, dv)] + [lse]


def _plain_step(s):
    c = s["case"]
    B, Hq, Hk, D, W, S = c["B"], c["Hq"], c["Hk"], c["D"], c["window"], c["sinks"]
    q, k, v = _heads(s["qkv"], Hq, Hk, D)
    dt, pos = s["qkv"].dtype, s["positions"]
    q, k = q.float(), k.float()
    if c["norm"]:
        cos, sin = (t[:, None, :] for t in _cos_sin(pos, s["freqs"]))
        q, k = _plain_norm(q, s["wq"], cos, sin, False), _plain_norm(k, s["wk"], cos, sin, False)
    slot = torch.where(pos < S, pos, S + (pos - S) % W)
    b = torch.arange(B, device=DEV)
    s["k_cache"][b, :, slot] = k.to(dt)
    s["v_cache"][b, :, slot] = v
    live = (torch.arange(W + S, device=DEV)[None, :] <= pos[:, None])[:, None, None, :]
    a = torch.matmul(q.view(B, Hk, Hq // Hk, D), s["k_cache"].float().transpose(2, 3)) * D ** -0.5
    a = a.masked_fill(~live, -math.inf)
    a = (a - a.amax(-1, keepdim=True)).exp()
    a = a / a.sum(-1, keepdim=True)
    vals = s["v_cache"].float().masked_fill(~live.transpose(2, 3), 0.0)
    return torch.matmul(a, vals).view(B, Hq, D).to(dt), s["k_cache"], s["v_cache"]


def _plain_fill(s):
    c = s["case"]
    B, T, W, S = c["B"], c["T"], c["window"], c["sinks"]
    n = s["nframes"].long() if s["nframes"] is not None else torch.full((B,), T, dtype=torch.int64, device=DEV)
    at = torch.arange(W + S, device=DEV)[None, :]
    last = n[:, None] - 1
    pos = torch.where(at < S, at.expand(B, -1), last - (last - at) % W)   # the newest position of every slot
    ok = (pos < n[:, None]) & ((at < S) | (pos >= S))
    b = torch.arange(B, device=DEV)[:, None]
    for name in ("k", "v"):
        rows = s[name][b, pos.clamp(0, T - 1)].transpose(1, 2)
        s[name + "_cache"].copy_(torch.where(ok[:, None, :, None], rows, s[name + "_cache"]))
    return s["k_cache"], s["v_cache"]


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"norm": _plain_norm_rows, "norm_bwd": _plain_norm_backward, "attn": _plain_attention_forward,
                "attn_train": _plain_attention_train, "step": _plain_step, "fill": _plain_fill}[op](s)
    import slsmi
    ops = slsmi.ops
    if op == "norm":
        return ops.qk_norm_rope(s["qkv"], c["Hq"], c["Hk"], s["wq"], s["wk"], s["freqs"], s["positions"], eps=EPS,
                                interleaved=c["interleaved"])
    if op == "norm_bwd":
        return ops.qk_norm_rope_backward(s["dout"], s["qkv"], c["Hq"], c["Hk"], s["wq"], s["wk"], s["freqs"],
                                         s["positions"], eps=EPS, interleaved=c["interleaved"])
    if op == "step":
        norm = dict(q_weight=s["wq"], k_weight=s["wk"], freqs=s["freqs"], eps=EPS) if c["norm"] else {}
        out = ops.window_attention_step(s["qkv"], s["k_cache"], s["v_cache"], s["positions"], c["Hq"], c["sinks"], **norm)
        return out, s["k_cache"], s["v_cache"]
    if op == "fill":
        ops.window_cache_fill(s["k"], s["v"], s["k_cache"], s["v_cache"], c["sinks"], nframes=s["nframes"])
        return s["k_cache"], s["v_cache"]
    window = dict(left=c["left"] if c["left"] >= 0 else None, right=c["right"] if c["right"] >= 0 else None,
                  sinks=c["sinks"], nframes=s["nframes"])
    if op == "attn":
        return ops.window_attention(s["q"], s["k"], s["v"], **window)
    o, lse = ops.window_attention(s["q"], s["k"], s["v"], return_lse=True, **window)
    dq, dk, dv = ops.window_attention_backward(s["dout"], s["q"], s["k"], s["v"], o, lse, **window)
    return [o, dq, dk, dv, lse]


# ---- 64 bits --------------------------------------------------------------------------------------------------------

def _exact_norm(x, w, positions, freqs, interleaved):
    """x [..., T, H, D] in 64 bits: pairs as complex numbers, turned by a unit number."""
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    R = 2 * freqs.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV).expand(positions.numel(), R // 2),
                       torch.outer(positions.double(), freqs))[:, None, :]
    head = y[..., :R]
    pairs = head.unflatten(-1, (R // 2, 2)) if interleaved else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z if interleaved else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), y[..., R:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, D = case["op"], case["D"]
    if op in ("norm", "norm_bwd"):
        q, k, _ = _heads(s["qkv"], case["Hq"], case["Hk"], D)
        xs, ws = [t.double().requires_grad_() for t in (q, k)], [s[n].double().requires_grad_() for n in ("wq", "wk")]
        y = torch.cat([_exact_norm(x, w, s["positions"], s["freqs"], case["interleaved"]) for x, w in zip(xs, ws)],
                      -2).flatten(-2)
        if op == "norm":
            return y.detach()
        gx = torch.autograd.grad(y, xs + ws, s["dout"].double())
        return torch.cat(gx[:2], -2).flatten(-2), gx[2], gx[3]
    if op == "fill":
        return _exact_fill(case, s)
    if op == "step":
        return _exact_step(case, s)
    return _exact_attention(case, s)


def _exact_attention(case, s):
    B, T, Hq, Hk, D = (case[n] for n in ("B", "T", "Hq", "Hk", "D"))
    train, g = case["op"] == "attn_train", case["Hq"] // case["Hk"]
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(B, T, Hk, D, dtype=torch.float64, device=DEV) for _ in range(2))
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(case)):
        i, j = torch.meshgrid(torch.arange(n, device=DEV), torch.arange(n, device=DEV), indexing="ij")
        near = (j - i).abs() <= 2 * T
        if case["left"] >= 0:
            near &= (i - j <= case["left"]) | (j < case["sinks"])
        if case["right"] >= 0:
            near &= j - i <= case["right"]
        bias = torch.zeros(n, n, dtype=torch.float64, device=DEV).masked_fill_(~near, -math.inf)
        del i, j, near
        for h in range(Hq):
            q, k, v = (x[b, :n, y].double().requires_grad_(train) for x, y in ((s["q"], h), (s["k"], h // g), (s["v"], h // g)))
            a = torch.addmm(bias, q, k.t(), alpha=1.0 / math.sqrt(D))
            y = torch.softmax(a, -1) @ v
            o[b, :n, h] = y.detach()
            if train:
                lse[b, h, :n] = torch.logsumexp(a.detach(), -1)
                gq, gk, gv = torch.autograd.grad(y, (q, k, v), s["dout"][b, :n, h].double())
                dq[b, :n, h] = gq
                dk[b, :n, h // g] += gk
                dv[b, :n, h // g] += gv
    return [o, dq, dk, dv, lse] if train else o


def _exact_step(case, s):
    B, Hq, Hk, D, W, S = (case[n] for n in ("B", "Hq", "Hk", "D", "window", "sinks"))
    q, k, v = (t.double() for t in _heads(s["qkv"], Hq, Hk, D))
    if case["norm"]:
        q, k = (_exact_norm(t, w, s["positions"], s["freqs"], False) for t, w in ((q, s["wq"]), (k, s["wk"])))
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    out = torch.empty(B, Hq, D, dtype=torch.float64, device=DEV)
    for b, p in enumerate(_positions_now(case)):
        at = p if p < S else S + (p - S) % W
        kc[b, :, at], vc[b, :, at] = k[b], v[b]
        n = min(p + 1, W + S)
        for h in range(Hq):
            a = torch.softmax(kc[b, h // (Hq // Hk), :n] @ q[b, h] / math.sqrt(D), 0)
            out[b, h] = a @ vc[b, h // (Hq // Hk), :n]
    return out, kc, vc


def _exact_fill(case, s):
    W, S = case["window"], case["sinks"]
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    for b, n in enumerate(_lengths(case)):
        kept = list(range(min(S, n))) + list(range(max(S, n - W), n))
        slots = [p if p < S else S + (p - S) % W for p in kept]
        for c, x in zip(caches, (s["k"], s["v"])):
            c[b][:, slots] = x[b, kept].double().transpose(0, 1)
    return tuple(caches)
