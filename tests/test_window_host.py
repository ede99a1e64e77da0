"""What the windowed-attention entry points refuse through the C ABI (no GPU: a refused call enqueues nothing), and the
sizes of their workspaces."""
import ctypes as C

import pytest

import slsmi
from slsmi import _lib

INVALID, WORKSPACE = -1, -4
PTR = 1 << 20   # an aligned address that nothing reads


def shape(**kw):
    d = dict(batch=2, frames=300, heads=4, kv_heads=2, head_dim=64, left=16, right=0, sinks=4, fmt=1, scale=0.125)
    d.update(kw)
    return _lib.WindowShape(**d)


def heads(p=PTR, batch=300 * 512, row=512, head=64):
    return _lib.Heads(p, batch, row, head)


def forward(s, q=None, k=None, out=None):
    lib = _lib.load()
    args = [q or heads(), k or heads(), heads(), out or heads()]
    return lib.slsmi_window_attention(C.byref(s), *(C.byref(a) for a in args), None, None, None)


@pytest.mark.parametrize("kw", [dict(head_dim=32), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(left=-2), dict(right=-2),
                                dict(sinks=-1), dict(sinks=129), dict(fmt=2), dict(scale=0.0), dict(scale=float("nan")),
                                dict(frames=-1), dict(batch=-1), dict(frames=(1 << 29) + 1), dict(batch=1 << 30)])
def test_window_attention_refuses_shapes(kw):
    lib = _lib.load()
    assert forward(shape(**kw)) == INVALID
    assert lib.slsmi_window_attention_backward_workspace_bytes(C.byref(shape(**kw))) == 0


@pytest.mark.parametrize("h", [heads(0), heads(PTR + 8), heads(row=508), heads(row=32), heads(head=32), heads(batch=4), heads(row=-512)])
def test_window_attention_refuses_layouts(h):
    assert forward(shape(), q=h) == INVALID
    assert forward(shape(), k=h) == INVALID
    assert forward(shape(), out=h) == INVALID


def test_nothing_to_do_is_not_an_error():
    assert forward(shape(batch=0)) == 0 and forward(shape(frames=0)) == 0


def backward(s, ws, nbytes):
    lib = _lib.load()
    h = C.byref(heads())
    return lib.slsmi_window_attention_backward(C.byref(s), h, h, h, h, h, PTR, None, h, h, h, ws, nbytes, None)


def test_backward_workspace():
    lib = _lib.load()
    s = shape()
    need = lib.slsmi_window_attention_backward_workspace_bytes(C.byref(s))
    assert need >= 2 * 4 * 300 * 4
    assert backward(s, PTR, need - 1) == WORKSPACE and backward(s, None, need) == WORKSPACE and backward(s, PTR + 4, need) == WORKSPACE
    no_far = lib.slsmi_window_attention_backward_workspace_bytes(C.byref(shape(left=-1)))
    assert no_far < need   # without a limit the sinks need no sums of their own


def norm(rows=4, ldx=256, ldy=256, heads_=2, kv=1, D=64, R=64, npos=4, x=PTR, w=PTR, fr=PTR, fmt=0):
    return _lib.load().slsmi_qk_norm_rope(x, ldx, PTR, ldy, rows, heads_, kv, D, w, PTR, 1e-6, fr, R, 0, None, npos, fmt, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(ldx=252), dict(ldx=128), dict(ldy=128), dict(heads_=-1), dict(heads_=0, kv=0), dict(D=96),
                                dict(R=24), dict(R=128), dict(R=-16), dict(npos=0), dict(npos=1 << 40), dict(x=PTR + 2), dict(x=None), dict(w=None),
                                dict(fr=None), dict(fmt=3), dict(rows=1 << 31)])
def test_qk_norm_rope_refuses(kw):
    assert norm(**kw) == INVALID


def test_qk_norm_rope_backward_workspace():
    lib = _lib.load()
    need = lib.slsmi_qk_norm_rope_backward_workspace_bytes(100, 64)
    assert need > 0 and lib.slsmi_qk_norm_rope_backward_workspace_bytes(-1, 64) == 0

    def call(ws, n, dy=PTR, dwq=PTR):
        return lib.slsmi_qk_norm_rope_backward(dy, 256, PTR, 256, PTR, 256, 100, 2, 1, 64, PTR, PTR, 1e-6, PTR, 64, 0, None, 100, dwq, PTR, ws, n,
                                               0, None)

    assert call(PTR, need - 1) == WORKSPACE and call(None, need) == WORKSPACE and call(PTR + 4, need) == WORKSPACE
    assert call(PTR, need, dy=None) == INVALID and call(PTR, need, dwq=None) == INVALID


def step(s, slots=100, ld=512, kc=PTR, pos=PTR, wq=PTR, wk=PTR, fr=PTR, R=64, ws=PTR, n=1 << 40):
    return _lib.load().slsmi_window_step(C.byref(s), slots, PTR, ld, kc, PTR, pos, wq, wk, 1e-6, fr, R, 0, PTR, ws, n, None)


@pytest.mark.parametrize("kw", [dict(slots=4), dict(slots=(1 << 24) + 1), dict(ld=504), dict(kc=None), dict(kc=PTR + 8), dict(pos=None), dict(wk=None),
                                dict(wq=None, wk=None), dict(fr=None), dict(R=8), dict(R=80)])
def test_step_refuses(kw):
    assert step(shape(), **kw) == INVALID


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(heads=3), dict(sinks=-1), dict(scale=0.0), dict(fmt=5), dict(batch=65536), dict(batch=-1)])
def test_step_refuses_shapes(kw):
    assert step(shape(**kw)) == INVALID


def test_step_workspace():
    lib = _lib.load()
    s = shape(batch=1)
    need = lib.slsmi_window_step_workspace_bytes(C.byref(s), 20000)
    assert need > 0 and step(s, slots=20000, ws=PTR, n=need - 1) == WORKSPACE and step(s, slots=20000, ws=None, n=need) == WORKSPACE
    assert lib.slsmi_window_step_workspace_bytes(C.byref(shape(batch=0)), 100) == 0


def test_cache_fill_refuses():
    lib = _lib.load()
    ok = heads()

    def call(s, slots=100, k=ok, kc=PTR):
        return lib.slsmi_window_cache_fill(C.byref(s), slots, C.byref(k), C.byref(ok), kc, PTR, None, None)

    assert call(shape(), slots=4) == INVALID and call(shape(), k=heads(PTR + 2)) == INVALID and call(shape(), kc=None) == INVALID
    assert call(shape(head_dim=80)) == INVALID and call(shape(), k=heads(row=100)) == INVALID and call(shape(batch=0)) == 0


@pytest.mark.parametrize("kw", [dict(scale=2.0 ** -65), dict(scale=2.0 ** 65), dict(scale=float("inf")), dict(batch=1 << 13, heads=4096, frames=1),
                                dict(batch=1, heads=64, kv_heads=64, frames=1 << 26)])
def test_launches_that_could_not_be_counted_and_scales_without_an_inverse(kw):
    s = shape(**kw)
    lib = _lib.load()
    h = [C.byref(heads(PTR * (i + 1), row=512, batch=0)) for i in range(8)]
    assert lib.slsmi_window_attention(C.byref(s), h[0], h[1], h[2], h[3], None, None, None) == INVALID
    assert lib.slsmi_window_attention_backward(C.byref(s), *h[:5], PTR, None, *h[5:], PTR, 1 << 60, None) == INVALID


def test_backward_refuses_too_many_workgroups_of_both_sides_and_of_the_sinks():
    """Forwards that can be launched whose backward cannot."""
    lib = _lib.load()
    for s in (shape(batch=1, heads=64, kv_heads=64, frames=1 << 24, left=-1, sinks=0),
              shape(batch=4096, heads=64, kv_heads=64, frames=300, left=0, sinks=128)):
        h = [C.byref(heads(PTR * (i + 1), row=64 * 64, batch=0)) for i in range(8)]
        need = lib.slsmi_window_attention_backward_workspace_bytes(C.byref(s))
        assert need > 0
        assert lib.slsmi_window_attention_backward(C.byref(s), *h[:5], PTR, None, *h[5:], PTR, need, None) == INVALID


def test_results_in_the_place_of_what_is_read():
    lib = _lib.load()
    s = shape()
    need = lib.slsmi_window_attention_backward_workspace_bytes(C.byref(s))
    at = [heads(PTR * (i + 1)) for i in range(8)]   # dout q k v out dq dk dv
    for target, other in [(3, 1), (3, 2)]:
        args = [C.byref(at[other] if i == target else at[i]) for i in range(4)]
        assert lib.slsmi_window_attention(C.byref(s), *args, None, None, None) == INVALID
    for target in (5, 6, 7):
        for other in range(8):
            if other != target:
                h = [C.byref(at[other] if i == target else at[i]) for i in range(8)]
                assert lib.slsmi_window_attention_backward(C.byref(s), *h[:5], PTR, None, *h[5:], PTR, need, None) == INVALID


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_norms_refuse_an_eps_without_a_root_and_more_rows_than_a_launch_counts(eps):
    lib = _lib.load()

    def norm(rows=8, eps=1e-6):
        return lib.slsmi_qk_norm_rope(PTR, 256, 2 * PTR, 256, rows, 2, 1, 64, PTR, PTR, eps, None, 0, 0, None, rows, 1, None)
    assert norm(eps=eps) == INVALID and norm(rows=(1 << 25) + 1) == INVALID
    s = shape(frames=1, left=0)
    assert lib.slsmi_window_step(C.byref(s), 40, PTR, 512, 2 * PTR, 3 * PTR, PTR, PTR, PTR, eps, None, 0, 0, 4 * PTR, None, 0,
                                 None) == INVALID
