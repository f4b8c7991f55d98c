"""Differential attention against its plain 64-bit form, forward and backward; bounds as derived in attn_plain."""
import math

import numpy as np
import pytest
import torch

import attn_plain as plain
from starrygl_amd.nn.model import diff_attention

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _lens(rng, n, top, ragged, zeros=True):
    return [int(rng.integers(0 if zeros else 1, top + 1)) if ragged else top for _ in range(n)]


def _ptr(lens, first=0):
    return torch.from_numpy(np.cumsum([first] + list(lens))).long().cuda()


def _inputs(Tq, Tk, Hq, Hk, D, Dv, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, go = r(Tq, Hq, 2, D) * scale, r(Tk, Hk, 2, D), r(Tk, Hk, Dv), r(Tq, Hq, Dv)
    lam = 0.2 + 0.6 * torch.rand(Hq, generator=g)
    return [t.to(dtype).cuda() for t in (q, k, v)] + [lam.cuda(), go.to(dtype).cuda()]


def _within(got, ref, name):
    got, want, tol = got.detach().cpu().double(), ref[name], ref[name + "_tol"]
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    bad = (off > 0) | got.isnan()
    if bad.any():
        at = np.unravel_index(int(torch.where(got.isnan(), torch.full_like(off, math.inf), off).argmax()), got.shape)
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond their bound, worst at {at}: {got[at]:.6g} for {want[at]:.6g} +- {tol[at]:.3g}")


def _check(q, k, v, lam, go, k_ptr, q_ptr=None, train=True, **kw):
    ref = plain.diff_attention(q, k, v, lam, k_ptr, q_ptr, grad=go if train else None, **kw)
    y0 = diff_attention(q, k, v, lam, k_ptr, q_ptr, **kw)
    _within(y0, ref, "out")
    if not train:
        return y0, ref
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, k_ptr, q_ptr, **kw)
    assert torch.equal(y, y0)
    grads = torch.autograd.grad(y, leaves, go)
    for n, t in zip(("dq", "dk", "dv", "dlam"), grads):
        _within(t, ref, n)
    return y, ref


HEADS = [  # Hq, Hk, D, Dv
    (2, 2, 32, 64), (4, 1, 64, 128), (6, 2, 25, 50), (1, 1, 128, 256), (3, 3, 7, 9), (8, 2, 50, 100), (2, 1, 100, 200), (2, 2, 16, 16), (1, 1, 1, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,Hk,D,Dv", HEADS)
def test_one_query_per_sequence(hot, Hq, Hk, D, Dv, dtype):
    """roots over their sampled neighbours: some roots without neighbours, keys before the first and behind the last"""
    rng = np.random.default_rng(D)
    lens = _lens(rng, 70, 20, True)
    k_ptr = _ptr(lens, 3)
    ins = _inputs(70, sum(lens) + 8, Hq, Hk, D, Dv, dtype, D)
    _check(*ins, k_ptr)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,Hk,D,Dv", HEADS)
@pytest.mark.parametrize("causal", [False, True])
def test_ragged_histories(hot, Hq, Hk, D, Dv, causal, dtype):
    rng = np.random.default_rng(Dv)
    nk = _lens(rng, 5, 90, True) + [0, 1, 64, 33]
    nq = list(nk) if causal else _lens(rng, len(nk), 40, True)
    ins = _inputs(sum(nq) + 5, sum(nk) + 7, Hq, Hk, D, Dv, dtype, D + 1)
    _check(*ins, _ptr(nk, 4), _ptr(nq, 2), causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_lengths_around_tiles(hot, n, dtype):
    ins = _inputs(n, n, 2, 1, 64, 128, dtype, n)
    _check(*ins, _ptr([n]), _ptr([n]), causal=True)
    ins = _inputs(n, 2 * n + 1, 2, 1, 64, 128, dtype, n)
    _check(*ins, _ptr([2 * n + 1]), _ptr([n]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 5, 40, 1000])
def test_window(hot, window, dtype):
    nk = [100, 3, 0, 150]
    ins = _inputs(sum(nk), sum(nk), 4, 2, 32, 64, dtype, window)
    _check(*ins, _ptr(nk), _ptr(nk), causal=True, window=window)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_causal_with_more_queries_than_keys_and_fewer(hot, dtype):
    """queries and keys end together: the first queries of a sequence with fewer keys see none"""
    nq, nk = [40, 10, 7, 0, 5], [12, 70, 0, 9, 5]
    ins = _inputs(sum(nq), sum(nk), 2, 2, 32, 64, dtype, 3)
    y, _ = _check(*ins, _ptr(nk), _ptr(nq), causal=True)
    assert not y[:28].any() and not y[50:57].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("form", ["roots", "histories"])
def test_key_mask(hot, form, dtype):
    """hidden keys hold NaN and infinities; whole sequences are hidden; their rows give zeros and no gradient"""
    rng = np.random.default_rng(8)
    nk = [20, 75, 1, 0, 33, 64]
    nq = [1] * 6 if form == "roots" else nk
    q, k, v, lam, go = _inputs(sum(nq), sum(nk), 4, 2, 32, 64, dtype, 5)
    mask = torch.from_numpy(rng.random(sum(nk)) < 0.6).cuda()
    mask[20:95] = False
    k[~mask], v[~mask] = float("nan"), float("inf")
    kp, qp = _ptr(nk), None if form == "roots" else _ptr(nq)
    clean = [torch.where(mask.view(-1, *[1] * (t.dim() - 1)), t, 0.0) for t in (k, v)]
    ref = plain.diff_attention(q, *clean, lam, kp, qp, key_mask=mask, grad=go)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, kp, qp, key_mask=mask)
    grads = torch.autograd.grad(y, leaves, go)
    _within(y, ref, "out")
    for n, t in zip(("dq", "dk", "dv", "dlam"), grads):
        _within(t, ref, n)
    assert not grads[1][~mask].any() and not grads[2][~mask].any()
    rows = slice(1, 2) if form == "roots" else slice(20, 95)
    assert not y[rows].any() and not grads[0][rows].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_is_not_finite_stays_with_those_who_see_it(hot, dtype):
    """NaN and infinities in one sequence, in a later event and in a row of no sequence change no other result"""
    nk = [40, 25, 70, 10]
    q, k, v, lam, go = _inputs(150, 150, 2, 1, 32, 64, dtype, 6)
    kp = _ptr(nk)
    base = [t.clone() for t in (q, k, v, go)]
    q[50], k[52], v[41], v[45], go[60] = float("nan"), float("inf"), float("nan"), float("inf"), float("nan")   # sequence 1
    q[100], k[101], v[102] = float("nan"), float("nan"), -float("inf")                                            # events 35-37 of sequence 2
    k[146], v[147], q[148], go[149] = [float("nan")] * 4                                                         # no sequence
    ref = plain.diff_attention(base[0], base[1], base[2], lam, kp, kp, causal=True, grad=base[3])
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, kp, kp, causal=True)
    grads = torch.autograd.grad(y, leaves, go)
    clean = torch.ones(150, dtype=torch.bool)
    clean[40:65] = clean[100:135] = False                # rows that see something of it
    keys = torch.ones(150, dtype=torch.bool)
    keys[40:65] = keys[65:135] = False                   # keys that such a row sees
    for got, name, ok in ((y, "out", clean), (grads[0], "dq", clean), (grads[1], "dk", keys), (grads[2], "dv", keys)):
        part = {name: ref[name][ok], name + "_tol": ref[name + "_tol"][ok]}
        _within(got.detach().cpu()[ok], part, name)
    assert y[100:135].isnan().any() and y[50].isnan().all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_large_scores(hot, dtype):
    """scores of several hundred: the running maximum moves far between keys, most probabilities vanish"""
    rng = np.random.default_rng(1)
    nk = [200, 60, 130]
    ins = _inputs(sum(nk), sum(nk), 2, 2, 32, 64, dtype, 9, scale=60.0)
    _check(*ins, _ptr(nk), _ptr(nk), train=dtype != F16)
    ins = _inputs(3, sum(nk), 2, 2, 32, 64, dtype, 9, scale=60.0)
    _check(*ins, _ptr(nk), None, train=dtype != F16)


def test_rising_scores(hot):
    """every key's score beats all before it by a little: the maximum is never final"""
    n = 500
    q, k, v, lam, go = _inputs(64, n, 1, 1, 32, 64, BF16, 2)
    q[:], k[:] = 0, 0
    q[..., 0], k[:, 0, 0, 0], k[:, 0, 1, 0] = 8.0, torch.arange(n, device="cuda").to(BF16) / 32, -torch.arange(n, device="cuda").to(BF16) / 32
    _check(q, k, v, lam, go, _ptr([n]), _ptr([64]))
    _check(q[:1], k, v, lam, go[:1], _ptr([n]), None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_broadcasts_and_shared_leaves(hot, dtype):
    """views of one fused projection, an expanded v, the same tensor as query and key"""
    g = torch.Generator().manual_seed(4)
    T, H, D = 90, 2, 32
    fused = torch.randn(T, 6 * H * D + 5, generator=g).to(dtype).cuda().requires_grad_()
    kp = _ptr([50, 40])
    part = lambda t, i: t[:, i * 2 * H * D + 3: (i + 1) * 2 * H * D + 3]  # noqa: E731
    lam = torch.tensor([0.3, 0.7]).cuda()
    go = torch.randn(T, H, 2 * D, generator=g).to(dtype).cuda()

    def of(t, f):
        q, k = part(t, 0).view(T, H, 2, D), part(t, 1).view(T, H, 2, D)
        return f(q, k, part(t, 2).view(T, H, 2 * D))
    y = of(fused, lambda q, k, v: diff_attention(q, k, v, lam, kp, kp, causal=True))
    got, = torch.autograd.grad(y, fused, go)
    q, k, v = of(fused.detach(), lambda q, k, v: (q, k, v))
    ref = plain.diff_attention(q, k, v, lam, kp, kp, causal=True, grad=go)
    _within(y, ref, "out")
    for i, (n, s) in enumerate((("dq", (T, H, 2, D)), ("dk", (T, H, 2, D)), ("dv", (T, H, 2 * D)))):
        _within(part(got, i).reshape(s), ref, n)
    # one value row for all keys of a head: the gradient of the broadcast leaf is the sum
    one = torch.randn(1, H, 2 * D, generator=g).to(dtype).cuda().requires_grad_()
    y = diff_attention(q, k, one.expand(T, H, 2 * D), lam, kp, kp)
    ref = plain.diff_attention(q, k, one.expand(T, H, 2 * D), lam, kp, kp, grad=go)
    _within(y, ref, "out")
    dv, = torch.autograd.grad(y, one, go)
    want, tol = ref["dv"].sum(0, keepdim=True), ref["dv_tol"].sum(0, keepdim=True) + plain.h(dtype) * T * ref["dv"].sum(0, keepdim=True).abs() + \
        plain.h(dtype) * ref["dv"].abs().cumsum(0).amax(0, keepdim=True) * 8
    assert ((dv.cpu().double() - want).abs() <= tol).all()
    # queries and keys from one leaf: both gradients arrive
    leaf = q.clone().requires_grad_()
    dx, = torch.autograd.grad(diff_attention(leaf, leaf, v, lam, kp, kp), leaf, go)
    ref = plain.diff_attention(q, q, v, lam, kp, kp, grad=go)
    tol = ref["dq_tol"] + ref["dk_tol"] + plain.h(dtype) * (ref["dq"] + ref["dk"]).abs()
    assert ((dx.cpu().double() - ref["dq"] - ref["dk"]).abs() <= tol).all()


def test_gradients_against_differences(hot):
    """directional derivatives in fp32, step 2^-6; the results are smooth on that scale (third derivatives of order one),
    so the central difference is off by about 2^-12 / 6 of the magnitudes, and rounding adds 2^-20 / 2^-6"""
    q, k, v, lam, go = _inputs(30, 45, 2, 1, 16, 32, F32, 12)
    kp, qp = _ptr([25, 20]), _ptr([10, 20])
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    grads = torch.autograd.grad(diff_attention(*leaves, kp, qp, causal=True), leaves, go)
    f = lambda *t: float((diff_attention(*t, kp, qp, causal=True).double() * go).sum())  # noqa: E731
    with torch.no_grad():
        for i in range(4):
            g = torch.Generator().manual_seed(i)
            d = torch.randn(leaves[i].shape, generator=g).cuda()
            d = d / d.norm()
            at = lambda s: f(*[t + s * d if j == i else t for j, t in enumerate(leaves)])  # noqa: E731
            diff = (at(2.0 ** -6) - at(-(2.0 ** -6))) * 2.0 ** 5
            scale = float((go.abs().double()).sum()) * 2.0 ** -14 + float((grads[i] * d).double().abs().sum()) * 2.0 ** -8
            assert abs(diff - float((grads[i] * d).double().sum())) <= scale


def test_same_bits_every_time_and_on_other_streams(hot):
    nk = [500, 3, 700, 41]
    q, k, v, lam, go = _inputs(sum(nk), sum(nk), 4, 2, 64, 128, BF16, 7)
    kp = _ptr(nk)

    def once():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        y = diff_attention(*leaves, kp, kp, causal=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, go)]
    first = once()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(once())
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.parametrize("dtype,Hq,Hk", [(F32, 2, 2), (BF16, 8, 2), (F16, 4, 4), (BF16, 12, 1)])
@pytest.mark.parametrize("seqs,top", [(3, 5000), (1, 1), (1, 20_000), (200, 300)])
def test_single_queries_over_long_histories(hot, seqs, top, dtype, Hq, Hk):
    rng = np.random.default_rng(top)
    nk = _lens(rng, seqs, top, True, zeros=seqs > 1)
    ins = _inputs(seqs, sum(nk), Hq, Hk, 64, 128, dtype, 3)
    _check(*ins, _ptr(nk), train=top <= 5000)
    mask = torch.rand(sum(nk), generator=torch.Generator().manual_seed(1)).cuda() < 0.5
    _check(*ins, _ptr(nk), train=False, key_mask=mask)


def test_few_queries_over_long_histories(hot):
    nq, nk = [4, 1, 7, 2], [6000, 9000, 300, 4500]
    ins = _inputs(sum(nq), sum(nk), 4, 1, 64, 128, BF16, 3)
    _check(*ins, _ptr(nk), _ptr(nq), causal=True)


def test_many_heads_in_a_group(hot):
    """40 query heads read one key head"""
    nk = [70, 2, 33]
    ins = _inputs(3, sum(nk), 40, 1, 16, 32, BF16, 3)
    _check(*ins, _ptr(nk))
    ins = _inputs(sum(nk), sum(nk), 40, 1, 16, 32, BF16, 4)
    _check(*ins, _ptr(nk), _ptr(nk), causal=True)


def test_live_sequences_and_rows_behind_them(hot):
    """worst-case buffers: the live number of sequences is on the device, rows behind them keep what they held; with
    zero_rest they are cleared"""
    nk = [10, 20, 5, 9]
    kp, qp = _ptr(nk), _ptr([3, 2, 4, 6])
    B = torch.tensor([2], device="cuda")
    for q_ptr, Tq, live in ((None, 4, 2), (qp, 15, 5)):
        q, k, v, lam, go = _inputs(Tq, 44, 2, 1, 32, 64, BF16, 3)
        flat = (q.view(Tq, 4, 32), k.view(44, 2, 32), v)
        cut = lambda p: None if p is None else p[:3].contiguous()  # noqa: E731
        ref = plain.diff_attention(q[:live], k[:30], v[:30], lam, kp[:3], cut(q_ptr), grad=go[:live])
        for rest in (False, True):
            out, o2 = (torch.full((Tq, 2, 64), 7.0, dtype=BF16, device="cuda") for _ in range(2))
            lse = torch.full((Tq, 2, 2), 7.0, device="cuda")
            hot.diff_attn(*flat, lam, kp, q_ptr, B_dev=B, zero_rest=rest, out=out, lse=lse, o2=o2)
            _within(out[:live], ref, "out")
            assert (out[live:] == (0 if rest else 7)).all()
            d = [torch.full(t.shape, 7.0, dtype=BF16, device="cuda") for t in flat]
            got = hot.diff_attn_backward(go, *flat, lam, out, lse, o2, kp, q_ptr, B_dev=B, zero_rest=rest, d_q=d[0], d_k=d[1], d_v=d[2])
            ref4 = {n: t.view(t.shape[0], -1, t.shape[-1]) if t.dim() == 4 else t for n, t in ref.items()}
            _within(got[0][:live], ref4, "dq")
            _within(got[1][:30], ref4, "dk")
            _within(got[2][:30], ref4, "dv")
            _within(got[3], ref4, "dlam")
            for t, n in zip(d, (live, 30, 30)):
                assert (t[n:] == (0 if rest else 7)).all()


@pytest.mark.parametrize("form", ["roots", "histories"])
def test_captured_training_step(hot, form):
    """forward and backward in one graph while an eager graph of other leaves lives, replayed on new inputs"""
    from starrygl_amd.lib.driver import graph_capture
    nk = [30, 64, 7, 100]
    qp = None if form == "roots" else _ptr(nk)
    kp = _ptr(nk)
    Tq = 4 if qp is None else sum(nk)
    ins = _inputs(Tq, sum(nk), 4, 2, 32, 64, BF16, 1)
    leaves = [t.clone().requires_grad_() for t in ins[:4]]
    go = ins[4].clone()
    alive = diff_attention(*[t.detach().clone().requires_grad_() for t in leaves], kp, qp)   # keeps its own graph
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(diff_attention(*leaves, kp, qp), leaves, go)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        y = diff_attention(*leaves, kp, qp)
        grads = torch.autograd.grad(y, leaves, go)
    for k in range(4):
        new = _inputs(Tq, sum(nk), 4, 2, 32, 64, BF16, 30 + k)
        with torch.no_grad():
            for t, n in zip(leaves, new):
                t.copy_(n)
        go.copy_(new[4])
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.clone().requires_grad_() for t in new[:4]]
        ye = diff_attention(*eager, kp, qp)
        ge = torch.autograd.grad(ye, eager, new[4])
        assert torch.equal(y, ye) and all(torch.equal(a, b) for a, b in zip(grads, ge))
    assert alive.grad_fn is not None


def test_empty_calls(hot):
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    lam, p = z(2), torch.zeros(1, dtype=torch.long, device="cuda")
    assert diff_attention(z(0, 2, 2, 8), z(0, 1, 2, 8), z(0, 1, 16), lam, p).shape == (0, 2, 16)
    kp = torch.zeros(4, dtype=torch.long, device="cuda")
    leaves = [t.requires_grad_() for t in (z(3, 2, 2, 8), z(0, 1, 2, 8), z(0, 1, 16), lam)]
    y = diff_attention(*leaves, kp)
    assert not y.any()
    for g in torch.autograd.grad(y.sum(), leaves):
        assert not g.any()
    leaves = [t.requires_grad_() for t in (z(0, 2, 2, 8), z(5, 1, 2, 8), z(5, 1, 16), z(2))]
    kp = torch.tensor([0, 5], device="cuda")
    y = diff_attention(*leaves, kp, torch.zeros(2, dtype=torch.long, device="cuda"))
    grads = torch.autograd.grad(y.sum(), leaves)
    assert all(not g.any() for g in grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences_most_of_them_empty(hot, dtype):
    """runs of more empty sequences than a wave looks at side by side, thousands of pointers, rows and keys before and behind"""
    rng = np.random.default_rng(5)
    B = 5000
    nq, nk = np.zeros(B, np.int64), np.zeros(B, np.int64)
    some = rng.choice(B, 120, replace=False)
    some = some[(some < 1000) | (some > 1300)]
    nq[some], nk[some] = rng.integers(0, 5, some.size), rng.integers(0, 40, some.size)
    nq[700:900] = 0
    q_ptr, k_ptr = _ptr(nq, 3), _ptr(nk, 2)
    q, k, v, lam, go = _inputs(int(q_ptr[-1]) + 4, int(k_ptr[-1]) + 6, 2, 1, 32, 64, dtype, 7)
    _check(q, k, v, lam, go, k_ptr, q_ptr)
    _check(q, k, v, lam, go, k_ptr, q_ptr, causal=True, window=4)


def test_a_window_wider_than_any_sequence(hot):
    q, k, v, lam, _ = _inputs(90, 90, 2, 2, 32, 64, BF16, 3)
    p = _ptr([40, 50])
    free = diff_attention(q, k, v, lam, p, p, causal=True)
    for window in (50, 2 ** 31 - 1, 2 ** 31, 2 ** 62):
        assert torch.equal(diff_attention(q, k, v, lam, p, p, causal=True, window=window), free)


@pytest.mark.parametrize("one_query", [False, True])
def test_offsets_past_32_bits(hot, one_query):
    """sequences at the end of tensors of more than 2^31 elements: what stands before them belongs to none"""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    T = (1 << 31) // 512 + 1000
    nk, nq = [200, 100], [1, 1] if one_query else [200, 100]
    q, k, v, lam, go = _inputs(sum(nq), 300, 8, 4, 64, 128, BF16, 11)
    big = [torch.zeros(T, *t.shape[1:], dtype=BF16, device="cuda") for t in (k, v)]
    for b, t in zip(big, (k, v)):
        b[-300:] = t
        b.requires_grad_()
    leaves = [q.requires_grad_(), *big, lam.requires_grad_()]
    q_ptr = None if one_query else _ptr(nq)
    y = diff_attention(*leaves, _ptr(nk, T - 300), q_ptr)
    got = torch.autograd.grad(y, leaves, go)
    ref = plain.diff_attention(q, k, v, lam, _ptr(nk), q_ptr, grad=go)
    _within(y, ref, "out")
    for name, t in zip(("dq", "dk", "dv", "dlam"), got):
        _within(t[-300:] if name in ("dk", "dv") else t, ref, name)
    assert not got[1][:-300].any() and not got[2][:-300].any()
