"""Plain 64-bit forms (on the CPU) of the attention-layer operators, with error bounds of a 32-bit evaluation.

Units: a rounding to type t is off by at most h(t) = finfo(t).eps / 2 relative to the value; U = 2^-24 is fp32's."""
import math

import torch

U = 2.0 ** -24


def h(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, value):
    """the most that one rounding of `value` to the type is off: half a step, which below the smallest normal number is
    half the smallest subnormal (fp16: 2^-25) whatever the value"""
    return torch.maximum(h(dtype) * value.abs(), torch.tensor(torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2, dtype=torch.float64))


def rotate(x, pos, freq, interleaved=False, amplitude=1.0, inverse=False):
    """-> (rotated x, sum of the magnitudes that enter each value), float64"""
    x = x.double()
    r = freq.numel()
    t = pos.double()[:, None] * freq[None, :]
    c, s = (amplitude * t.cos())[:, None], (amplitude * t.sin())[:, None] * (-1 if inverse else 1)
    a, b = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    y, mag = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    both = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    mag[..., a], mag[..., b] = both, both
    return y, mag


def norm_rotate(x, pos, w, freq, eps, interleaved=False, amplitude=1.0):
    x = x.double()
    n = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    if w is not None:
        n = n * w.double()
    return rotate(n, pos, freq, interleaved, amplitude)


def norm_rotate_grads(x, pos, w, freq, eps, g, interleaved=False, amplitude=1.0):
    """-> (dx, magnitudes in dx, dw, magnitudes in dw); dw has the shape of w (or [D])"""
    x = x.double()
    inv = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * inv
    d, mag = rotate(g, pos, freq, interleaved, amplitude, inverse=True)
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    over = (0,) if wd.dim() == 2 else (0, 1)
    dw, dw_mag = (d * xh).sum(over), (mag * xh.abs()).sum(over)
    e, em = d * wd, mag * wd.abs()
    dx = inv * (e - xh * (e * xh).mean(-1, keepdim=True))
    return dx, inv * (em + xh.abs() * (em * xh.abs()).mean(-1, keepdim=True)), dw, dw_mag


def visible(nq, nk, causal, window):
    i, j = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)[None, :]
    see = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        see &= j <= i
        if window:
            see &= j > i - window
    return see


def diff_attention(q, k, v, lam, k_ptr, q_ptr=None, scale=None, causal=False, window=None, key_mask=None, grad=None):
    """q [Tq, Hq, 2, D] ... as nn.model.diff_attention, float64 -> dict of results and, under the same names with "_tol",
    bounds of what a kernel may be off that sums in fp32, rounds P and dS to the inputs' type before their products and
    keeps out and o2 in it.

    A score: D products and sums of fp32, the scaling, the exponent's argument: e_s = scale (D + 4) U sum |q k| + U |s|;
    a probability is off by 2 e_s (its exponential and the sum below it) + (n + 8) U, then by h when it is rounded.
    In fp16 a probability below 2^-14 is off by up to 2^-25 absolutely, or by itself where such values are flushed; in the
    other types that happens below 2^-126, where fp32's exponential ends."""
    dt = q.dtype
    r = h(dt) if dt != torch.float32 else U
    floor = 2.0 ** -14 if dt == torch.float16 else 2.0 ** -126
    q, k, v, lam = (t.detach().cpu().double() for t in (q, k, v, lam))
    Tq, Hq, _, D = q.shape
    Tk, Hk, Dv = v.shape
    G = Hq // Hk
    c = D ** -0.5 if scale is None else scale
    k_ptr = k_ptr.cpu().tolist()
    q_ptr = list(range(len(k_ptr))) if q_ptr is None else q_ptr.cpu().tolist()
    key_mask = None if key_mask is None else key_mask.cpu().bool()
    names = dict(out=(Tq, Hq, Dv), dq=q.shape, dk=k.shape, dv=v.shape, dlam=(Hq,))
    got = {n + s: torch.zeros(*shape, dtype=torch.float64) for n, shape in names.items() for s in ("", "_tol")}
    for b in range(len(k_ptr) - 1):
        q0, q1, k0, k1 = q_ptr[b], q_ptr[b + 1], k_ptr[b], k_ptr[b + 1]
        nq, nk = q1 - q0, k1 - k0
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, causal, window)
        if key_mask is not None:
            see = see & key_mask[k0:k1][None, :]
        for hd in range(Hq):
            hk = hd // G
            Q, K, V = q[q0:q1, hd], k[k0:k1, hk], v[k0:k1, hk]
            used = see.any(0)                                   # what no query sees must not enter, not even as 0 * NaN
            V, K = torch.where(used[:, None], V, 0.0), torch.where(used[:, None, None], K, 0.0)
            P, E = [], []
            for m in range(2):
                s = (Q[:, m] @ K[:, m].T) * c
                mag = (Q[:, m].abs() @ K[:, m].abs().T) * abs(c)
                s = s.masked_fill(~see, -math.inf)
                top = s.amax(-1, keepdim=True)
                e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
                z = e.sum(-1, keepdim=True)
                p = torch.where(z > 0, e / z, torch.zeros_like(e))
                err = torch.where(see, (D + 4) * U * mag + U * s.abs().nan_to_num(0, 0, 0), torch.zeros_like(mag))
                P.append(p)
                E.append(2 * err.amax(-1, keepdim=True) + (nk + 8) * U)
            lm = lam[hd]
            W = P[0] - lm * P[1]
            Wmag = P[0] + lm.abs() * P[1]
            Werr = P[0] * (E[0] + r) + lm.abs() * P[1] * (E[1] + r) + floor * see * (1 + lm.abs())
            y = W @ V
            ytol = Werr @ V.abs() + (nk + 2) * U * (Wmag @ V.abs())
            got["out"][q0:q1, hd], got["out_tol"][q0:q1, hd] = y, ytol + rounding(dt, y)
            if grad is None:
                continue
            dO = grad[q0:q1, hd].cpu().double()
            dP = dO @ V.T
            dPmag = dO.abs() @ V.abs().T
            dPerr = (Dv + 2) * U * dPmag
            got["dv"][k0:k1, hk] += W.T @ dO
            got["dv_tol"][k0:k1, hk] += (Werr.T + (nq * G + 2) * U * Wmag.T) @ dO.abs()
            o2 = P[1] @ V
            for m in range(2):
                t = (P[m] * dP).sum(-1, keepdim=True)
                f = 1.0 if m == 0 else -lm
                # t from the stored out and o2 (each rounded to the type), or summed from P dP: the larger of the two
                stored = (dO.abs() * (rounding(dt, y) + (1 + lm.abs()) * rounding(dt, o2) + ytol * (2 + lm.abs()))).sum(-1, keepdim=True)
                terr = stored + (P[m] * dPmag).sum(-1, keepdim=True) * ((nk + Dv + 8) * U + E[m])
                dS = P[m] * (dP - t) * f
                dSerr = dS.abs() * (E[m] + r) + P[m] * abs(f) * (dPerr + terr) + floor * see * abs(f) * (dPmag + t.abs())
                if dt == torch.float16:
                    dSerr = dSerr + 2.0 ** -24 * see
                dSmag = P[m] * abs(f) * (dP.abs() + t.abs())
                got["dq"][q0:q1, hd, m] = c * (dS @ K[:, m])
                got["dq_tol"][q0:q1, hd, m] = abs(c) * ((dSerr + (nk + 2) * U * dSmag) @ K[:, m].abs())
                got["dk"][k0:k1, hk, m] += c * (dS.T @ Q[:, m])
                got["dk_tol"][k0:k1, hk, m] += abs(c) * ((dSerr + (nq * G + 2) * U * dSmag).T @ Q[:, m].abs())
                if m == 1:
                    got["dlam"][hd] -= t.sum()
                    # t_2 of a row: summed from P dP in fp32 (no rounding to the type enters)
                    got["dlam_tol"][hd] += ((P[m] * dPmag) * ((nk + Dv + 8 + Tq) * U + E[m])).sum()
    if grad is not None:
        for n in ("dq", "dk", "dv"):
            got[n + "_tol"] += rounding(dt, got[n])
    return got
