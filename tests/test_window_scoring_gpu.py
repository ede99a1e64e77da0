"""The scoring forward with a sliding attention window (Model(attention_window=, attention_sinks=)) against the CPU
oracle whose attention carries the same mask.  Tolerances are those of the whole-clip forward: the window adds no rounding
(16-bit operands, fp32 softmax statistics and sums, as the whole-clip kernel)."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

import slsmi
from slsmi.config import BackboneConfig
from slsmi.model import Model
from slsmi.weights import synth_state_dict
from oracle import reference_cpu as orc
from tolerances import LAYER_RMS, TOL

DEV = torch.device("cuda:0")
CFG = BackboneConfig(layers=2)


def noise(B, frames, seed=77):
    g = torch.Generator().manual_seed(seed)
    return (0.1 * torch.randn(B, 320 * frames + 80, generator=g)).clamp(-1, 1)


def masked_attention(left, right, sinks):
    def attend(sd, p, x, heads, key_padding_mask=None, attn_drop=None):
        T, B, C = x.shape
        i, j = torch.arange(T)[:, None], torch.arange(T)[None, :]
        see = (j <= i + right) if right >= 0 else torch.ones(T, T, dtype=torch.bool)
        if left >= 0:
            see = see & ((j >= i - left) | (j < sinks))
        q, k, v = (F.linear(x, sd[p + n + "_proj.weight"], sd[p + n + "_proj.bias"]).view(T, B, heads, C // heads)
                   .permute(1, 2, 0, 3) for n in "qkv")
        s = (q * (C // heads) ** -0.5) @ k.transpose(-1, -2)
        a = torch.softmax(s.masked_fill(~see, float("-inf")), -1) @ v
        return F.linear(a.permute(2, 0, 1, 3).reshape(T, B, C), sd[p + "out_proj.weight"], sd[p + "out_proj.bias"])
    return attend


def make(head, window, sinks=0, **kw):
    sd = synth_state_dict(CFG, head, 201, 1234)
    extra = dict(use_sae=False) if head == "ssl" else dict(head=head)
    m = Model(None, DEV, cp_path=None, cfg=CFG, precision="f16", attention_window=window, attention_sinks=sinks,
              **extra, **kw).eval()
    m.load_state_dict(sd)
    return m, sd


def score(logp):
    return torch.exp(logp.detach().float().cpu())[:, 1]


@pytest.mark.parametrize("frames,window,sinks", [
    (201, (None, None), 0), (201, (20, 8), 4), (201, (16, 0), 0), (130, (0, 0), 0),
    (513, (None, None), 0), (700, (64, 64), 16), (1031, (100, 0), 2), (700, (None, 3), 0)])
def test_features_and_score_against_the_masked_oracle(monkeypatch, frames, window, sinks):
    m, sd = make("ssl", window, sinks)
    wav = noise(2, frames)
    with torch.no_grad():
        logp = m(wav.to(DEV), return_sae_loss=False).cpu()
        x = m.ssl_model.extract_feat(wav.to(DEV)).cpu()
    left, right = (-1 if n is None else n for n in window)
    monkeypatch.setattr(orc, "self_attention", masked_attention(left, right, sinks))
    oc = orc.OracleConfig(layers=2)
    bb = orc.backbone_forward(sd, wav, oc, pfx="ssl_model.model.")
    ref = orc.model_forward(sd, wav, oc, "ssl")
    rel = ((x - bb["x"]).pow(2).mean().sqrt() / bb["x"].pow(2).mean().sqrt()).item()
    err = (score(logp) - score(ref)).abs().max().item()
    print(f"[{frames} frames, window {window}, {sinks} sinks] x rms err {rel:.2e}, score err {err:.2e}")
    assert x.shape[1] == frames
    assert rel < LAYER_RMS["f16"] and err < TOL[("sae", "f16")]


def test_padded_batch_scores_each_long_clip_as_alone():
    m, _ = make("ssl", (50, 10), 8)
    frames = [900, 513, 640, 40]
    wav = noise(4, 900, seed=5)
    lengths = torch.tensor([320 * f + 80 for f in frames])
    with torch.no_grad():
        together = score(m(wav.to(DEV), return_sae_loss=False, lengths=lengths))
        alone = torch.cat([score(m(wav[b:b + 1, :int(n)].to(DEV), return_sae_loss=False)) for b, n in enumerate(lengths)])
    print(together.tolist(), alone.tolist())
    assert (together - alone).abs().max() < 2e-5    # the batch-size invariance of the default schedule


def test_sls_head_and_whole_clip_agree_without_a_limit():
    """With nothing outside the window the two attention kernels compute one function: scores within twice the head's
    tolerance of the oracle's."""
    whole, _ = make("sls", None)
    wide, _ = make("sls", (None, None))
    wav = noise(3, 201).to(DEV)
    with torch.no_grad():
        a, b = score(whole(wav, return_sae_loss=False)), score(wide(wav, return_sae_loss=False))
    assert (a - b).abs().max() < 2 * TOL[("sls", "f16")]


def test_refusals():
    with pytest.raises(slsmi._lib.SlsmiError, match="sinks"):
        make("ssl", (10, 10), 129)[0](noise(1, 60).to(DEV))
    with pytest.raises(ValueError, match="attention_window"):
        make("ssl", (10,))
    m, _ = make("ssl", (10, 10))
    with pytest.raises(slsmi._lib.SlsmiError, match="unsupported batch/length"):   # one frame too many
        with torch.no_grad():
            m(noise(1, 16385).to(DEV), return_sae_loss=False)
    with pytest.raises(slsmi._lib.SlsmiError, match="unsupported batch/length"):   # and a batch too large
        with torch.no_grad():
            m(noise(55, 600).to(DEV), return_sae_loss=False)
    m.train()
    with pytest.raises(slsmi._lib.SlsmiError, match="scoring option"):
        m(noise(1, 201).to(DEV))
    whole, _ = make("ssl", None)
    with pytest.raises(slsmi._lib.SlsmiError, match="unsupported batch/length"):
        with torch.no_grad():
            whole(noise(1, 600).to(DEV), return_sae_loss=False)


def test_the_window_reaches_the_features():
    """A window of one frame and no window give features that differ by far more than the tolerances above."""
    wav = noise(2, 201).to(DEV)
    with torch.no_grad():
        a, b = (make("ssl", w)[0].ssl_model.extract_feat(wav) for w in ((0, 0), (None, None)))
    assert ((a - b).pow(2).mean().sqrt() / b.pow(2).mean().sqrt()).item() > 4 * LAYER_RMS["f16"]


def test_the_longest_recording():
    """16384 frames, 5.5 minutes: features of the first and the last frames equal those of the clip's own ends, which a
    window of 40 frames and two layers separate from the rest (the positional convolution reaches 64 frames)."""
    m, _ = make("ssl", (40, 40))
    wav = noise(1, 16384, seed=9).to(DEV)
    with torch.no_grad():
        x = m.ssl_model.extract_feat(wav)
        head = m.ssl_model.extract_feat(wav[:, :320 * 600 + 80])
        tail = m.ssl_model.extract_feat(wav[:, 320 * (16384 - 600):])
    assert x.shape == (1, 16384, 1024) and torch.isfinite(x).all()
    scale = x.pow(2).mean().sqrt()
    for whole, own in ((x[:, :400], head[:, :400]), (x[:, -400:], tail[:, -400:])):
        assert ((whole - own).pow(2).mean().sqrt() / scale).item() < 2 * LAYER_RMS["f16"]


def test_eval_driver_scores_long_recordings(tmp_path):
    """eval_sharded.py --variable_length --attention_window: thirteen recordings of 62 to 68 seconds and a short one at the default batch size;
    together the long ones exceed what one batch may hold, and every trial gets its score."""
    import os
    import subprocess
    import sys
    import wave
    import numpy as np
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    rng = np.random.default_rng(3)
    ids = [f"{i}.wav" for i in range(14)]
    for i, u in enumerate(ids):
        n = 48000 if i == 13 else 16000 * 62 + 8000 * i
        with wave.open(str(tmp_path / u), "wb") as w:
            w.setnchannels(1), w.setsampwidth(2), w.setframerate(16000)
            w.writeframes((rng.standard_normal(n) * 3000).clip(-32768, 32767).astype("<i2").tobytes())
    (tmp_path / "trials.txt").write_text("".join(u + "\n" for u in ids))
    out = tmp_path / "scores.txt"
    r = subprocess.run([sys.executable, os.path.join(root, "eval_sharded.py"), "--track", "In-the-Wild", "--synthetic_weights",
                        "--database_path", str(tmp_path) + "/", "--protocols_path", str(tmp_path / "trials.txt"),
                        "--variable_length", "--max_seconds", "327", "--attention_window", "100", "100",
                        "--attention_sinks", "4", "--eval_output", str(out)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout[-1000:] + r.stderr[-3000:]
    lines = [line.split() for line in out.read_text().splitlines()]
    assert [u for u, _ in lines] == ids and all(0.0 <= float(s) <= 1.0 for _, s in lines)
