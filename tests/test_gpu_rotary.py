"""Rotary encoding and the per-head norm with rotation against their plain 64-bit forms, forward and backward.

Tolerances. A cosine or sine of the kernel is off by at most 2^-25 (its reduced argument rounded to fp32) + 2^-23 (the
polynomial), the amplitude, the two products and their sum round at 2^-24 each: below 2^-22 of the magnitudes that enter
a value; then one rounding to the type (fp16 below 2^-14: half its smallest subnormal, 2^-25). The norm's sum of squares has at most 32 additions in a row (relative 2^-19,
halved by the root), and three more roundings: below 2^-18 with the rotation. Gradients take the norm's path twice:
2^-17; a weight's gradient also sums N H terms: N H 2^-24."""
import pytest
import torch

import attn_plain as plain
from starrygl_amd.nn.model import QKNormRotary, RotaryEncoder, qk_norm_rotary, rotary_encode, rotary_frequencies

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, tol, tag=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (tag, got.shape, want.shape)
    off = (got - want).abs() - tol
    assert not (off > 0).any() and not got.isnan().any(), f"{tag}: {int((off > 0).sum())} beyond, by {off.max():.3g}"


def _x(n, heads, dim, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=g) * scale).to(dtype).cuda()


def _pos(n, seed, top=2_600_000):
    g = torch.Generator().manual_seed(seed + 1000)
    p = torch.randint(-top, top, (n,), generator=g)
    p[: min(n, 4)] = torch.tensor([0, 1, -1, top])[: min(n, 4)]
    return p.cuda()


SHAPES = [  # rows, heads, dim, rot
    (1, 1, 2, 2), (1, 8, 64, 64), (3, 2, 50, 50), (65, 3, 100, 100), (257, 16, 128, 64), (40, 1, 86, 20), (33, 5, 7, 4),
    (1000, 2, 32, 32), (5, 70, 64, 64), (2, 1, 1024, 1024), (3, 1, 1023, 6), (7, 2, 600, 300), (9, 4, 16, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,dim,rot", SHAPES)
def test_rotary(hot, n, heads, dim, rot, interleaved, dtype):
    x, pos = _x(n, heads, dim, dtype, n + dim), _pos(n, n)
    freq, amp = rotary_frequencies(rot)
    want, mag = plain.rotate(x.cpu(), pos.cpu(), freq, interleaved, 1.5)
    y = rotary_encode(x, pos, freq.cuda(), interleaved=interleaved, amplitude=1.5)
    _close(y, want, plain.rounding(dtype, want) + 2.0 ** -22 * mag, "y")
    x.requires_grad_()
    g = _x(n, heads, dim, dtype, n + dim + 1)
    dx, = torch.autograd.grad(rotary_encode(x, pos, freq.cuda(), interleaved=interleaved, amplitude=1.5), x, g)
    want, mag = plain.rotate(g.cpu(), pos.cpu(), freq, interleaved, 1.5, inverse=True)
    _close(dx, want, plain.rounding(dtype, want) + 2.0 ** -22 * mag, "dx")


def test_rotary_far_positions_and_in_place(hot):
    """angles keep their precision at positions up to 2^53 and turn the library's way beyond 1e15"""
    pos = torch.tensor([2**40, -2**40 + 1, 2**49, 2**53 - 1, 2**60, 12345678901], device="cuda")
    freq = torch.tensor([1.0, 0.37, 1e-3, 1e-9], dtype=torch.float64)
    x = _x(6, 3, 8, torch.float32, 5)
    want, mag = plain.rotate(x.cpu(), pos.cpu(), freq)
    _close(rotary_encode(x, pos, freq.cuda()), want, 2.0 ** -22 * mag)
    out = hot.rotary(x, pos, freq.cuda(), out=x)
    assert out is x
    _close(x, want, 2.0 ** -22 * mag)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides_and_live_rows(hot, interleaved):
    """a view of a fused projection, an output with strides of its own, a live count; rows behind it stay as they were"""
    base = _x(50, 9, 72, torch.bfloat16, 1)
    x = base[:, 2:7, 4:68]
    pos, (freq, _) = _pos(50, 2), rotary_frequencies(64)
    want, mag = plain.rotate(x.cpu(), pos.cpu(), freq, interleaved)
    tol = plain.rounding(torch.bfloat16, want) + 2.0 ** -22 * mag
    _close(rotary_encode(x, pos, freq.cuda(), interleaved=interleaved), want, tol)
    out = torch.full((5, 50, 80), 7.0, dtype=torch.bfloat16, device="cuda")
    hot.rotary(x, pos, freq.cuda(), out=out.transpose(0, 1)[:, :, 8:72], interleaved=interleaved,
               N_dev=torch.tensor([31], device="cuda"))
    _close(out.transpose(0, 1)[:31, :, 8:72], want[:31], tol[:31])
    assert (out[:, 31:] == 7).all() and (out[:, :, :8] == 7).all() and (out[:, :, 72:] == 7).all()
    z = _x(50, 64, 5, torch.bfloat16, 3).transpose(1, 2)          # last axis not contiguous: taken as a copy
    want, mag = plain.rotate(z.cpu(), pos.cpu(), freq, interleaved)
    _close(rotary_encode(z, pos, freq.cuda(), interleaved=interleaved), want, plain.rounding(torch.bfloat16, want) + 2.0 ** -22 * mag)


@pytest.mark.parametrize("scaling", [dict(type="linear", factor=4), dict(type="base", factor=8), dict(type="by_parts", factor=8, length=4096)])
def test_rotary_module_with_scaled_frequencies(hot, scaling):
    enc = RotaryEncoder(64, 32, scaling=scaling).cuda().half()
    assert enc.freq.dtype == torch.float64 and enc.freq.is_cuda
    freq, amp = rotary_frequencies(32, scaling=scaling)
    x, pos = _x(20, 2, 64, torch.float16, 3), _pos(20, 3)
    want, mag = plain.rotate(x.cpu(), pos.cpu(), freq, False, amp)
    _close(enc(x, pos), want, plain.rounding(torch.float16, want) + 2.0 ** -22 * mag)


NORM = [  # rows q, rows k, heads q, heads k, dim, rot, weights
    (1, 1, 1, 1, 16, 16, "shared"), (32, 32, 16, 4, 64, 64, "shared"), (5, 60, 4, 4, 32, 32, "per head"), (70, 7, 2, 1, 25, 24, "shared"),
    (33, 33, 6, 3, 100, 50, "per head"), (300, 300, 8, 2, 128, 128, "shared"), (9, 0, 2, 2, 50, 50, "shared"), (4, 9, 1, 1, 1024, 512, "shared"),
    (3, 2, 2, 2, 513, 6, "per head"), (17, 17, 2, 2, 64, 0, "shared"), (12, 40, 2, 2, 32, 32, "none"), (2000, 100, 3, 2, 8, 8, "shared"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("nq,nk,hq,hk,dim,rot,weights", NORM)
def test_qk_norm_rotary(hot, nq, nk, hq, hk, dim, rot, weights, interleaved, dtype):
    eps = 1e-5
    q, k = _x(nq, hq, dim, dtype, 1, 2.0), _x(nk, hk, dim, dtype, 2, 0.5)
    pq, pk = _pos(nq, 3), _pos(nk, 4)
    g = torch.Generator().manual_seed(5)
    shape = lambda h: (h, dim) if weights == "per head" else (dim,)  # noqa: E731
    wq, wk = ((1 + 0.3 * torch.randn(shape(h), generator=g)).cuda() if weights != "none" else None for h in (hq, hk))
    freq, _ = rotary_frequencies(rot)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    yq, yk = qk_norm_rotary(q, k, pq, pk, wq, wk, freq.cuda(), eps=eps, interleaved=interleaved, amplitude=1.25)
    gq, gk = _x(nq, hq, dim, dtype, 6), _x(nk, hk, dim, dtype, 7)
    grads = torch.autograd.grad([yq, yk], leaves, [gq, gk])
    for i, (x, y, w, pos, gr, tag) in enumerate(((q, yq, wq, pq, gq, "q"), (k, yk, wk, pk, gk, "k"))):
        cpu = [t.detach().cpu() for t in (x, pos)] + [None if w is None else w.detach().cpu()]
        want, mag = plain.norm_rotate(cpu[0], cpu[1], cpu[2], freq, eps, interleaved, 1.25)
        _close(y, want, plain.rounding(dtype, want) + 2.0 ** -18 * mag, tag)
        dx, dxm, dw, dwm = plain.norm_rotate_grads(cpu[0], cpu[1], cpu[2], freq, eps, gr.cpu(), interleaved, 1.25)
        _close(grads[i], dx, plain.rounding(dtype, dx) + 2.0 ** -17 * dxm, "d" + tag)
        if w is not None:
            _close(grads[2 + i], dw, (2.0 ** -17 + x.shape[0] * x.shape[1] * plain.U) * dwm, "dw" + tag)


def test_qk_norm_partial_gradients_types_and_zero_rows(hot):
    """only the keys or only a weight want a gradient; weights of 16 bits; a row of zeros"""
    q, k = _x(6, 2, 64, torch.bfloat16, 1), _x(8, 2, 64, torch.bfloat16, 2).requires_grad_()
    with torch.no_grad():
        k[3] = 0
    freq, _ = rotary_frequencies(64)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16).requires_grad_()
    yq, yk = qk_norm_rotary(q, k, _pos(6, 1), _pos(8, 2), None, w, freq.cuda())
    gk = _x(8, 2, 64, torch.bfloat16, 9)
    dk, dw = torch.autograd.grad(yk, [k, w], gk)
    assert dw.dtype == torch.bfloat16 and (yk[3] == 0).all()
    dx, dxm, dwr, dwm = plain.norm_rotate_grads(k.detach().cpu(), _pos(8, 2).cpu(), w.detach().cpu(), freq, 1e-6, gk.cpu())
    _close(dk, dx, plain.rounding(torch.bfloat16, dx) + 2.0 ** -17 * dxm)
    _close(dw, dwr, plain.rounding(torch.bfloat16, dwr) + 2.0 ** -16 * dwm)
    mod = QKNormRotary(64, q_heads=2).cuda()
    a, b = mod(q, k.detach(), _pos(6, 1), _pos(8, 2))
    want, mag = plain.norm_rotate(q.cpu(), _pos(6, 1).cpu(), None, freq, 1e-6)
    _close(a, want, plain.rounding(torch.bfloat16, want) + 2.0 ** -18 * mag)
    assert a.requires_grad and set(dict(mod.named_parameters())) == {"q_weight", "k_weight"}


def test_qk_norm_gradient_against_differences(hot):
    """directional derivative of a scalar of the outputs, fp32, step 2^-7: the central difference's own error is the third
    derivative's (below 2^-14 of the magnitudes here) plus rounding 2^-18 / 2^-7"""
    x, w = _x(10, 2, 16, torch.float32, 1), (1 + 0.1 * torch.randn(16, generator=torch.Generator().manual_seed(3))).cuda()
    pos, (freq, _) = _pos(10, 1), rotary_frequencies(16)
    g, d = _x(10, 2, 16, torch.float32, 2), _x(10, 2, 16, torch.float32, 4)
    f = lambda t: float((qk_norm_rotary(t, t, pos, pos, w, w, freq.cuda())[0] * g).double().sum())  # noqa: E731
    t = 2.0 ** -7
    diff = (f(x + t * d) - f(x - t * d)) / (2 * t)
    x.requires_grad_()
    dx, = torch.autograd.grad(qk_norm_rotary(x, x.detach(), pos, pos, w, w, freq.cuda())[0], x, g)
    exact = float((dx * d).double().sum())
    scale = float((dx * d).abs().double().sum())
    assert abs(diff - exact) <= scale * 2.0 ** -9


def test_norm_and_rotary_in_a_graph(hot):
    """captured once, replayed with other inputs, positions and live counts, eager work between the replays"""
    from starrygl_amd.lib.driver import graph_capture
    freq = rotary_frequencies(32)[0].cuda()
    x, pos, n = _x(64, 4, 32, torch.bfloat16, 1), _pos(64, 1), torch.tensor([64], device="cuda")
    w = torch.ones(32, device="cuda")
    y, r = torch.zeros_like(x), torch.zeros_like(x)

    def step():
        hot.qk_norm_rotary([dict(x=x, y=y, pos=pos, weight=w, N_dev=n)], freq)
        hot.rotary(y, pos, freq, out=r, inverse=True, N_dev=n)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        step()
    for k in range(4):
        x.copy_(_x(64, 4, 32, torch.bfloat16, 10 + k)); pos.copy_(_pos(64, 20 + k)); n.fill_(64 - 7 * k)
        y.zero_(); r.zero_()
        graph.replay()
        torch.cuda.synchronize()
        live = 64 - 7 * k
        ye = qk_norm_rotary(x, x, pos, pos, w, w, freq)[0]
        assert torch.equal(y[:live], ye[:live]) and not y[live:].any() and not r[live:].any()
        assert torch.equal(r[:live], hot.rotary(ye, pos, freq, inverse=True)[:live])
