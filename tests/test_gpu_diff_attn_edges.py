"""Calls of differential attention at the edges of what it takes: rows without keys in split tiles, sizes past 32 bits, values
that are not finite in every kernel, pointers behind the rows; bounds as derived in attn_plain."""
import math

import pytest
import torch

import attn_plain as plain
from starrygl_amd.nn.model import diff_attention, qk_norm_rotary, rotary_encode, rotary_frequencies
from test_gpu_diff_attn import BF16, F16, F32, _check, _inputs, _ptr, _within

pytestmark = pytest.mark.gpu

# D, Dv, dtype: both maps in a wave, and one (rows of 512 and of 1024 bytes)
WIDTHS = [(32, 64, BF16), (32, 64, F32), (64, 128, BF16), (64, 128, F32), (128, 256, F16), (128, 256, F32), (100, 200, BF16), (7, 9, F16)]


@pytest.mark.parametrize("D,Dv,dtype", WIDTHS)
@pytest.mark.parametrize("causal", [False, True])
def test_rows_without_keys_beside_a_split_sequence(hot, causal, D, Dv, dtype):
    """a sequence with queries and no keys, queries that come before the first key (causal), and rows before and behind all
    sequences share a row tile with a sequence long enough to be split over blocks: they give zeros, lse = inf"""
    # (a wave that has a column of few keys looks at every mask: only causal calls have one here, beside the six rows that it hides)
    more = 1 if causal else 0
    q_ptr, k_ptr = _ptr([10, 12, 4] + [6] * more, 5), _ptr([0, 2048, 0] + [3] * more, 3)
    Tq, Tk = 42, 2060
    q, k, v, lam, go = _inputs(Tq, Tk, 2, 1, D, Dv, dtype, D)
    _, ref = _check(q, k, v, lam, go, k_ptr, q_ptr, causal=causal)
    dead = torch.ones(Tq, dtype=torch.bool)
    dead[15:27] = False
    if causal:
        dead[34:37] = False                     # six queries over three keys
    out, o2 = (torch.full((Tq, 2, Dv), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    lse = torch.full((Tq, 2, 2), 7.0, device="cuda")
    flat = q.flatten(1, 2), k.flatten(1, 2), v
    hot.diff_attn(*flat, lam, k_ptr, q_ptr, causal=causal, zero_rest=True, out=out, lse=lse, o2=o2)
    _within(out, ref, "out")
    dead = dead.cuda()
    assert not o2[dead].any() and (lse[dead] == math.inf).all() and lse[~dead].isfinite().all()
    # left as they were without zero_rest: rows of no sequence only
    for t in (out, o2, lse):
        t.fill_(7.0)
    hot.diff_attn(*flat, lam, k_ptr, q_ptr, causal=causal, out=out, lse=lse, o2=o2)
    for t in (out, o2):
        assert (t[:5] == 7).all() and (t[37:] == 7).all() and not t[5:15].any() and not t[27:31].any()
    assert (lse[:5] == 7).all() and (lse[37:] == 7).all()


@pytest.mark.parametrize("Tq", [1 << 26, (1 << 27) - 16])
def test_rows_times_heads_past_30_bits(hot, Tq):
    """2^26 rows of 16 heads and more: the numbers kept for (row, head, map) are 2^31 and more, the row tiles of the second call are
    2^24 (one launch takes fewer than 2^24 blocks of 256); only the last rows belong to sequences"""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    nq, nk = [200, 100], [70, 130]
    q, k, v, lam, go = _inputs(300, 200, 16, 4, 1, 1, BF16, 13)
    big = [torch.zeros(Tq, *t.shape[1:], dtype=BF16, device="cuda") for t in (q, go)]
    for b, t in zip(big, (q, go)):
        b[-300:] = t
        b[:64] = 1.0                            # (rows of no sequence)
    k_ptr, q_ptr = _ptr(nk), _ptr(nq, Tq - 300)
    ref = plain.diff_attention(q, k, v, lam, k_ptr, _ptr(nq), grad=go)
    out, lse = torch.empty(Tq, 16, 1, dtype=BF16, device="cuda"), torch.empty(Tq, 16, 2, device="cuda")
    o2 = torch.empty_like(out)
    flat = big[0].view(Tq, 32, 1), k.view(200, 8, 1), v
    hot.diff_attn(*flat, lam, k_ptr, q_ptr, zero_rest=True, out=out, lse=lse, o2=o2)
    _within(out[-300:], ref, "out")
    assert not out[:-300].any() and not o2[:-300].any() and lse[-300:].isfinite().all() and (lse[:-300] == math.inf).all()
    got = hot.diff_attn_backward(big[1], *flat, lam, out, lse, o2, k_ptr, q_ptr, zero_rest=True)
    assert not got[0][:-300].any()
    for name, t in zip(("dq", "dk", "dv", "dlam"), (got[0][-300:].view(q.shape), got[1].view(k.shape), *got[2:])):
        _within(t, ref, name)


def test_more_single_queries_over_few_keys_than_a_launch_has_waves(hot):
    """2^26 roots with one neighbour each: P = 1, out = (1 - lam) v"""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    B = (1 << 26) + 5
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v, go = (torch.randn(B, 1, n, generator=g, device="cuda").to(BF16) for n in (2, 2, 1, 1))
    lam, k_ptr = torch.tensor([0.375], device="cuda"), torch.arange(B + 1, device="cuda")
    v.requires_grad_()
    y = diff_attention(q.view(B, 1, 2, 1), k.view(B, 1, 2, 1), v, lam, k_ptr)
    dv, = torch.autograd.grad(y, v, go)
    for got, x in ((y.detach(), v.detach()), (dv, go)):
        want = x.double() * 0.625
        assert ((got.double() - want).abs() <= (plain.h(BF16) + 16 * plain.U) * want.abs()).all()


def test_more_single_queries_over_long_histories_than_a_launch_has_blocks(hot):
    """2^24 sequences of 64 keys, three query heads over one: some of them, the last among them, against the plain form"""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    B, n = (1 << 24) + 3, 64
    g = torch.Generator("cuda").manual_seed(2)
    q = torch.randn(B, 3, 2, 1, generator=g, device="cuda").to(BF16)
    k, v = torch.empty(B * n, 1, 2, 1, dtype=BF16, device="cuda").normal_(generator=g), torch.empty(B * n, 1, 1, dtype=BF16, device="cuda").normal_(generator=g)
    lam = torch.tensor([0.2, 0.5, 0.7], device="cuda")
    y = diff_attention(q, k, v, lam, torch.arange(B + 1, device="cuda") * n)
    some = torch.cat([torch.arange(0, B, B // 40), torch.arange((1 << 22) - 3, (1 << 22) + 3), torch.arange((1 << 24) - 2, B)]).cuda()
    keys = (some[:, None] * n + torch.arange(n, device="cuda")).flatten()
    ref = plain.diff_attention(q[some], k[keys], v[keys], lam, torch.arange(some.numel() + 1) * n)
    _within(y[some], ref, "out")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", ["few keys", "single queries", "split rows", "rows"])
def test_a_seen_value_that_is_not_finite_counts_whatever_its_weight(hot, form, dtype):
    """one key's score beats all others by hundreds of powers of two; a NaN value of another key that the query sees, wherever it
    lies among the parts that a sequence is split into, makes its element NaN, and no other"""
    n, nq = {"few keys": (12, 1), "single queries": (3000, 1), "split rows": (3000, 5), "rows": (400, 50)}[form]
    q, k, v, lam, go = _inputs(nq, n, 4, 2, 32, 64, dtype, 17)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[n // 2, ..., 0] = 300.0
    q_ptr = None if nq == 1 else _ptr([nq])
    want = plain.diff_attention(q, k, v, lam, _ptr([n]), q_ptr)
    for at in (0, 1, 2, 3, n // 2 - 1, n // 2 + 1, n - 1):
        bad = v.clone()
        bad[at, :, 3] = float("nan")
        bad[at, :, 60] = float("inf")
        y = diff_attention(q, k, bad, lam, _ptr([n]), q_ptr)
        assert y[..., 3].isnan().all() and y[..., 60].isnan().all(), at
        keep = [d for d in range(64) if d not in (3, 60)]
        _within(y[..., keep], {"out": want["out"][..., keep], "out_tol": want["out_tol"][..., keep]}, "out")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", ["few keys", "single queries", "split rows", "rows"])
def test_scores_of_minus_infinity(hot, form, dtype):
    """keys whose score overflows to -inf weigh nothing; a query with no others gets zeros, lse = inf and no gradient"""
    n, nq = {"few keys": (12, 1), "single queries": (3000, 1), "split rows": (3000, 5), "rows": (400, 50)}[form]
    q, k, v, lam, go = _inputs(2 * nq, 2 * n, 4, 2, 32, 64, dtype, 18)
    q[..., 0], k[..., 0] = 2.0 ** 100, -(2.0 ** 100)
    k[n // 2: n // 2 + 2, ..., 0] = k[:n // 3, ..., 0] = 0.0             # the first sequence has some others
    k_ptr, q_ptr = _ptr([n, n]), None if nq == 1 else _ptr([nq, nq])
    mask = torch.ones(2 * n, dtype=torch.bool, device="cuda")
    mask[:n] = k[:n, 0, 0, 0] == 0
    ref = plain.diff_attention(q[:nq], k[:n].clamp(min=-1e4), v[:n], lam, _ptr([n]), None if nq == 1 else _ptr([nq]), key_mask=mask[:n], grad=go[:nq])
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, k_ptr, q_ptr)
    grads = torch.autograd.grad(y, leaves, go)
    _within(y[:nq], ref, "out")
    assert not y[nq:].any() and not grads[0][nq:].any() and not grads[1][n:].any() and not grads[2][n:].any()
    for got, name, m in ((grads[1], "dk", n), (grads[2], "dv", n), (grads[3], "dlam", None)):
        _within(got if m is None else got[:m], ref, name)


def test_forward_mode_derivatives_are_refused(hot):
    """a tangent of any input is not dropped without a word"""
    import torch.autograd.forward_ad as fwAD
    q, k, v, lam, _ = _inputs(3, 9, 2, 1, 16, 32, F32, 1)
    kp, pos, freq = _ptr([2, 4, 3]), torch.arange(3, device="cuda"), rotary_frequencies(16)[0].cuda()
    w = torch.ones(16, device="cuda")
    calls = [(lambda *t: diff_attention(*t, kp), (q, k, v, lam)),
             (lambda x: rotary_encode(x, pos, freq), (q.flatten(1, 2),)),
             (lambda a, b, c, d: qk_norm_rotary(a, b, pos, pos, c, d, freq), (q.flatten(1, 2), q[:, 0], w, w.clone()))]
    for call, args in calls:
        call(*args)
        for i in range(len(args)):
            for strided in (False, True):                  # brought into the plain form first, or not
                with fwAD.dual_level():
                    ins = list(args)
                    t = ins[i]
                    if strided and t.dim() > 1:
                        t = t.repeat_interleave(2, -1)[..., ::2]
                    ins[i] = fwAD.make_dual(t, torch.ones_like(t))
                    with pytest.raises(NotImplementedError, match="forward"):
                        call(*ins)
        # nor that of a gradient on its way back
        leaves = [t.detach().clone().requires_grad_() for t in args]
        y = call(*leaves)
        y = y[0] if isinstance(y, tuple) else y
        with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward"):
            torch.autograd.grad(y, leaves[0], fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [None, 9])
def test_pointers_behind_the_rows_count_as_the_last_row(hot, window, dtype):
    """worst-case pointers may say more rows than there are: forward and gradients as with the pointers clamped"""
    q, k, v, lam, go = _inputs(90, 100, 2, 1, 32, 64, dtype, 3)
    q_ptr, k_ptr = torch.tensor([0, 40, 130], device="cuda"), torch.tensor([0, 40, 117], device="cuda")
    got = _check(q, k, v, lam, go, k_ptr.clamp(max=100), q_ptr.clamp(max=90), causal=True, window=window)[0]
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, k_ptr, q_ptr, causal=True, window=window)
    assert torch.equal(y, got)
    grads = torch.autograd.grad(y, leaves, go)
    ref = plain.diff_attention(q, k, v, lam, k_ptr.clamp(max=100), q_ptr.clamp(max=90), causal=True, window=window, grad=go)
    for n, t in zip(("dq", "dk", "dv", "dlam"), grads):
        _within(t, ref, n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-36, -1e-36])
@pytest.mark.parametrize("form", ["few keys", "single queries", "rows"])
def test_tiny_scales_of_huge_scores(hot, form, scale, dtype):
    """products of 10^37 times a scale of 10^-36 are scores like any other; times zero they all are zero"""
    n, nq = {"few keys": (12, 1), "single queries": (300, 1), "rows": (70, 50)}[form]
    q, k, v, lam, go = _inputs(nq, n, 4, 2, 32, 64, dtype, 19)
    mask = torch.arange(n, device="cuda") % 5 != 3
    _check(q * 2.0 ** 60, k * 2.0 ** 60, v, lam, go, _ptr([n]), None if nq == 1 else _ptr([nq]), scale=scale, key_mask=mask)


def test_scales_past_32_bits_are_refused(hot):
    q, k, v, lam, _ = _inputs(1, 4, 2, 1, 16, 32, F32, 1)
    for scale in (1e39, -1e39, 3e38, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale is not finite"):
            diff_attention(q, k, v, lam, _ptr([4]), scale=scale)


def _one_key_bounds(q, k, v, lam, go, key):
    """|dQ|, |dK| of rows i that see the one key key[i]: both are zero, a kernel with fp32 sums and states may be off by
      e = 2 ((D + 4) U c sum |q k| + 4 U (|s| + 1))        the probability, from a score formed twice and an lse,
      |dS| <= 1.01 (2 e + 2 (Dv + 8) U) sum |go v|,        two sums over the values (dP, t) and a result off by e + 4 U,
    dS rounded to the type: in fp16 by up to 2^-25 absolutely"""
    q, k, v, lam, go = (t.detach().cpu().double() for t in (q, k, v, lam, go))
    Tq, Hq, _, D = q.shape
    G, Dv, c = Hq // k.shape[1], v.shape[2], D ** -0.5
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    for i, j in enumerate(key):
        if j < 0:
            continue
        K, V = k[j].repeat_interleave(G, 0), v[j].repeat_interleave(G, 0)
        for m in range(2):
            mag, s = c * (q[i, :, m] * K[:, m]).abs().sum(-1), c * (q[i, :, m] * K[:, m]).sum(-1).abs()
            e = 2 * ((D + 4) * plain.U * mag + 4 * plain.U * (s + 1))
            dS = 1.01 * (2 * e + 2 * (Dv + 8) * plain.U) * (go[i] * V).abs().sum(-1) * (1 if m == 0 else lam.abs()) + 2.0 ** -24
            dq[i, :, m] += c * dS[:, None] * K[:, m].abs() + 2.0 ** -24
            dk[j, :, m] += (c * dS[:, None] * q[i, :, m].abs() + 2.0 ** -24).view(-1, G, D).sum(1)
    return dq, dk


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,Hk,D,Dv", [(2, 2, 32, 64), (4, 1, 64, 128), (2, 1, 128, 256), (2, 2, 25, 50)])
@pytest.mark.parametrize("form", ["roots", "rows", "split rows"])
def test_a_single_visible_key_passes_no_gradient_to_queries_and_keys(hot, form, Hq, Hk, D, Dv, dtype):
    """its probability is one whatever the score: the gradient's two terms cancel to what fp32 sums leave"""
    n = 40
    if form == "roots":
        Tq, Tk, k_ptr, q_ptr, mask, key = n, n, _ptr([1] * n), None, None, list(range(n))
    elif form == "rows":
        Tq, Tk, k_ptr, q_ptr, mask = 3 * n, n, _ptr([1] * n), _ptr([3] * n), None
        key = [i // 3 for i in range(Tq)]
    else:
        Tq, Tk, k_ptr, q_ptr = 6, 3000, _ptr([3000]), _ptr([6])
        mask, key = torch.zeros(Tk, dtype=torch.bool, device="cuda"), [1500] * 6
        mask[1500] = True
    q, k, v, lam, go = _inputs(Tq, Tk, Hq, Hk, D, Dv, dtype, D)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    dq, dk, _, _ = torch.autograd.grad(diff_attention(*leaves, k_ptr, q_ptr, key_mask=mask), leaves, go)
    tq, tk = _one_key_bounds(q, k, v, lam, go, key)
    assert (dq.cpu().double().abs() <= tq).all() and (dk.cpu().double().abs() <= tk).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D,Dv", [(32, 64), (64, 128), (128, 256), (25, 50), (7, 9)])
@pytest.mark.parametrize("form", ["roots", "long", "rows", "split rows"])
def test_unrounded_results_kept_for_the_backward_call(hot, form, D, Dv, dtype):
    """maps, with and without o2 beside it: rows behind the live sequences stay as they were, gradients need no out and o2"""
    nk = {"roots": [5, 0, 9, 4], "long": [700, 0, 900, 40], "rows": [40, 0, 70, 9], "split rows": [900, 0, 1100, 40]}[form]
    nq = {"roots": [1] * 4, "long": [1] * 4, "rows": [20, 3, 50, 8], "split rows": [3, 2, 4, 1]}[form]
    kp, q_ptr = _ptr(nk), None if nq[0] == 1 else _ptr(nq)
    Tq, Tk, live = sum(nq), sum(nk), sum(nq[:3])
    q, k, v, lam, go = _inputs(Tq, Tk, 4, 2, D, Dv, dtype, 23)
    flat, B = (q.flatten(1, 2), k.flatten(1, 2), v), torch.tensor([3], device="cuda")
    cut = None if q_ptr is None else q_ptr[:4]
    ref = plain.diff_attention(q[:live], k, v, lam, kp[:4], cut, grad=go[:live])
    got = []
    for o2 in (None, torch.full((Tq, 4, Dv), 7.0, dtype=dtype, device="cuda")):
        lse, maps = torch.full((Tq, 4, 2), 7.0, device="cuda"), torch.full((Tq, 4, 2, Dv), 7.0, device="cuda")
        out = hot.diff_attn(*flat, lam, kp, q_ptr, B_dev=B, lse=lse, o2=o2, maps=maps)
        _within(out[:live], ref, "out")
        assert (maps[live:] == 7).all()
        joined = maps[:live, :, 0] - lam[:, None] * maps[:live, :, 1]
        _within(joined, ref, "out")
        assert torch.equal(joined.to(dtype), out[:live]) or (joined - out[:live].float()).abs().max() <= 2 * plain.h(dtype) * joined.abs().max()
        if o2 is not None:
            assert torch.equal(o2[:live], maps[:live, :, 1].to(dtype)) and (o2[live:] == 7).all()
        d = hot.diff_attn_backward(go, *flat, lam, None, lse, None, kp, q_ptr, B_dev=B, zero_rest=True, maps=maps)
        for n, t, like in zip(("dq", "dk", "dv", "dlam"), d, (q, k, v, lam)):
            r = t.view(like.shape)
            if n == "dq":
                assert not r[live:].any()
                r = r[:live]
            _within(r, ref, n)
        got.append(d)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    with pytest.raises(ValueError, match="maps, or out and o2"):
        hot.diff_attn_backward(go, *flat, lam, out, lse, None, kp, q_ptr)
    with pytest.raises(ValueError, match="lse comes with"):
        hot.diff_attn(*flat, lam, kp, q_ptr, lse=lse)
    with pytest.raises(ValueError, match="maps"):
        hot.diff_attn(*flat, lam, kp, q_ptr, lse=lse, maps=maps[:, :, 0])


# every kernel and way of staging: 16-byte chunks whole, padded, and through registers
KERNELS = [(64, 128, BF16), (128, 256, BF16), (64, 128, F32), (128, 256, F32), (48, 96, BF16), (80, 160, F16), (100, 200, F32), (50, 100, BF16), (100, 200, F16), (25, 50, F32)]


def _layout(form):
    """-> lengths of the keys, of the queries (None: one each), causal"""
    if form == "single queries":
        return [300, 75, 0, 220, 1], None, False
    if form == "split rows":
        return [700, 1, 900, 600], [5, 1, 9, 3], True
    return [40, 25, 70, 10], [40, 25, 70, 10], True


def _visibility(nk, nq, causal):
    nq = nq or [1] * len(nk)
    see = torch.zeros(sum(nq), sum(nk), dtype=torch.bool)
    q0 = k0 = 0
    for a, b in zip(nq, nk):
        see[q0:q0 + a, k0:k0 + b] = plain.visible(a, b, causal, None)
        q0, k0 = q0 + a, k0 + b
    return see


def _held(got, ref, name, clean):
    """within bounds where `clean` says that nothing of it got in"""
    got, clean = got.detach().cpu().double(), clean.expand(got.shape)
    off = (got - ref[name]).abs() - ref[name + "_tol"]
    assert not ((off > 0) | got.isnan())[clean].any(), name


@pytest.mark.parametrize("D,Dv,dtype", KERNELS)
@pytest.mark.parametrize("form", ["rows", "split rows", "single queries"])
@pytest.mark.parametrize("what", ["q", "k", "v", "go"])
def test_a_nan_reaches_what_sees_it_and_nothing_else(hot, what, form, D, Dv, dtype):
    nk, nq, causal = _layout(form)
    see = _visibility(nk, nq, causal)
    Tq, Tk = see.shape
    q, k, v, lam, go = _inputs(Tq, Tk, 4, 1, D, Dv, dtype, 29)
    k_ptr, q_ptr = _ptr(nk), None if nq is None else _ptr(nq)
    ref = plain.diff_attention(q, k, v, lam, k_ptr, q_ptr, causal=causal, grad=go)
    # in the middle of a long sequence: a row, a key, and an element of either's value
    i, j = {"rows": (50, 100), "split rows": (8, 900), "single queries": (1, 310)}[form]
    rows, keys = torch.zeros(Tq, dtype=torch.bool), torch.zeros(Tk, dtype=torch.bool)
    bad = [t.clone() for t in (q, k, v, go)]
    if what in "kv":
        bad["qkv".index(what)][j, :, 5 if what == "v" else 1] = float("nan")           # (k: the second map)
        rows = see[:, j]
        keys = see[rows].any(0)
    else:
        bad[0 if what == "q" else 3][(i, slice(None), 0) if what == "q" else (i, slice(None), 5)] = float("nan")
        rows[i] = True
        keys = see[i]
    leaves = [t.requires_grad_() for t in (*bad[:3], lam)]
    y = diff_attention(*leaves, k_ptr, q_ptr, causal=causal)
    dq, dk, dv, dlam = torch.autograd.grad(y, leaves, bad[3])
    five = torch.arange(Dv) == 5
    r3, k3, r4, k4 = rows[:, None, None], keys[:, None, None], rows[:, None, None, None], keys[:, None, None, None]
    assert rows.any() and keys.any() and not rows.all() and not keys.all()
    # what it enters
    hit = {"q": (r3, r4, k4, k3), "k": (r3, r4, k4, k3), "v": (r3 & five, r4, k4, k3 & False), "go": (r3 & False, r4, k4, k3 & five)}[what]
    for t, name, m in zip((y, dq, dk, dv), ("out", "dq", "dk", "dv"), hit):
        _held(t, ref, name, ~m)
        m = m.expand(t.shape).to(t.device)
        if name in ("dq", "dk") and what in "qk":                   # (of one map for sure)
            of = 0 if what == "q" else 1
            assert t[:, :, of][m[:, :, of]].isnan().all(), name
        else:
            assert t[m].isnan().all(), name
    assert dlam.isnan().any() or what == "q"


@pytest.mark.parametrize("D,Dv,dtype", KERNELS)
@pytest.mark.parametrize("form", ["rows", "split rows", "single queries"])
def test_hidden_keys_may_hold_anything(hot, form, D, Dv, dtype):
    """NaN and infinities in the keys and values that the mask hides, and in rows of no sequence"""
    nk, nq, causal = _layout(form)
    lead = 3
    Tq, Tk = sum(nq) + 2 * lead if nq else len(nk), sum(nk) + 2 * lead
    q, k, v, lam, go = _inputs(Tq, Tk, 4, 1, D, Dv, dtype, 31)
    k_ptr, q_ptr = _ptr(nk, lead), None if nq is None else _ptr(nq, lead)
    mask = torch.rand(Tk, generator=torch.Generator().manual_seed(5)).cuda() < 0.6
    mask[lead:lead + 3] = False
    clean = [torch.where(mask.view(-1, *[1] * (t.dim() - 1)), t, 0.0) for t in (k, v)]
    ref = plain.diff_attention(q, *clean, lam, k_ptr, q_ptr, causal=causal, key_mask=mask, grad=go)
    k[~mask], v[~mask] = float("nan"), float("-inf")
    none = torch.ones(Tk, dtype=torch.bool, device="cuda")
    none[lead:-lead] = False
    k[none], v[none] = float("inf"), float("nan")
    if nq is not None:
        q[:lead], go[-lead:] = float("nan"), float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    y = diff_attention(*leaves, k_ptr, q_ptr, causal=causal, key_mask=mask)
    grads = torch.autograd.grad(y, leaves, go)
    for t, name in zip((y, *grads), ("out", "dq", "dk", "dv", "dlam")):
        _within(t, ref, name)
    assert not grads[1][~mask].any() and not grads[2][none].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hk", [(2, 2), (4, 2)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("window", [1, 3, 40])
def test_window_of_single_queries(hot, window, rest, Hq, Hk, dtype):
    """keys of a sequence in front of the window get gradients of zero, whatever the buffers held"""
    nk, lead = [5, 0, 30, 1, 100], 3
    k_ptr, Tk = _ptr(nk, lead), sum(nk) + 2 * lead
    q, k, v, lam, go = _inputs(5, Tk, Hq, Hk, 32, 64, dtype, 37)
    _, ref = _check(q, k, v, lam, go, k_ptr, causal=True, window=window)
    flat, how = (q.flatten(1, 2), k.flatten(1, 2), v), dict(causal=True, window=window, zero_rest=rest)
    lse, maps = torch.empty(5, Hq, 2, device="cuda"), torch.empty(5, Hq, 2, 64, device="cuda")
    hot.diff_attn(*flat, lam, k_ptr, lse=lse, maps=maps, **how)
    d_k, d_v = torch.full_like(flat[1], 7.0), torch.full_like(v, 7.0)
    got = hot.diff_attn_backward(go, *flat, lam, None, lse, None, k_ptr, maps=maps, d_k=d_k, d_v=d_v, **how)
    live = slice(lead, Tk - lead)
    for n, t, like in zip(("dq", "dk", "dv", "dlam"), got, (q, k, v, lam)):
        cut = live if n in ("dk", "dv") else slice(None)
        _within(t.view(like.shape)[cut], {n: ref[n][cut], n + "_tol": ref[n + "_tol"][cut]}, n)
    for t in (d_k, d_v):
        assert (t[:lead] == (0 if rest else 7)).all() and (t[Tk - lead:] == (0 if rest else 7)).all()
