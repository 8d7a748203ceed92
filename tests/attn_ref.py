"""The attention operators in 64 bits on the CPU, from their formulas, with bounds
of what 32-bit sums and 16-bit operands can be off by.

u is half a step of the 16-bit type.  A score's error is that of a D-term 32-bit
sum of exact products, (D + 4) 2^-24 sum|q||k| scale, and of the score map, 2^-21
(|s| + cap + 1) (a dozen roundings and the hardware's exp2 and reciprocal); P's
relative error twice the row's largest one and 2^-21 of exp2 itself.  The kernels
round P and dS to 16 bits as matrix operands (u each) and their outputs (u).
f16 has an absolute floor besides: half its smallest number, 2^-25."""
import math

import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor16(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def scores(q, k, scale, cap, dist, R, past, lim):
    """(s, dx/ds factor, error bound) of one head's clip; lim: keys that each query sees."""
    x = scale * (q @ k.t())
    err = scale * (q.shape[1] + 4) * F32 * (q.abs() @ k.abs().t())
    slope = torch.ones_like(x)
    s = x
    if cap:
        t = torch.tanh(x / cap)
        s, slope = cap * t, 1 - t * t
    r = torch.arange(k.shape[0])[None, :] - (torch.arange(q.shape[0])[:, None] + past)
    at = r.clamp(-R, R) + R if dist is not None else None
    if dist is not None:
        s = s + dist[at]
    fin = torch.where(torch.isfinite(s), s, torch.zeros_like(s))
    err = err + 2.0 ** -21 * (fin.abs() + cap + 1)
    seen = torch.arange(k.shape[0])[None, :] < lim[:, None]
    return torch.where(seen, s, torch.full_like(s, -math.inf)), slope, torch.where(seen, err, torch.zeros_like(err)), at


def softmax(s):
    if s.shape[1] == 0:
        return s, torch.full((s.shape[0],), -math.inf, dtype=torch.float64)
    m = s.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    tot = p.sum(1, keepdim=True)
    return p / torch.where(tot > 0, tot, torch.ones_like(tot)), (m + torch.log(tot)).squeeze(1)


def attend(q, k, v, q_at, kv_at, scale, cap=0.0, dist=None, causal=False, prefix=None, do=None):
    """Outputs and bounds as dicts of [total][heads][D] (lse [heads][total]) in 64 bits; with do the gradients too."""
    dt = q.dtype
    u, fl = half_step(dt), floor16(dt)
    H, kv = q.shape[1], k.shape[1]
    G = H // kv
    q, k, v = (x.double() for x in (q, k, v))
    R = (dist.shape[1] - 1) // 2 if dist is not None else 0
    out, tol = {}, {}
    names = ["o", "lse"] + (["dq", "dk", "dv"] if do is not None else [])
    for d in (out, tol):
        for n in names:
            d[n] = torch.zeros(H, q.shape[0], dtype=torch.float64) if n == "lse" else torch.zeros_like(
                q if n in ("o", "dq") else k)
        if do is not None and dist is not None:
            d["ddist"] = torch.zeros_like(dist, dtype=torch.float64)
    if do is not None:
        do = do.double()
    for c in range(len(q_at) - 1):
        a, b, e, f = q_at[c], q_at[c + 1], kv_at[c], kv_at[c + 1]
        nq, nk = b - a, f - e
        past, pre = nk - nq, prefix[c] if prefix else 0
        i = torch.arange(nq)
        lim = (past + i + 1).clamp_min(pre).clamp(0, nk) if causal else torch.full((nq,), nk)
        for h in range(H):
            g = h // G
            Q, K, V = q[a:b, h], k[e:f, g], v[e:f, g]
            dh = dist[h].double() if dist is not None else None
            s, slope, es, at = scores(Q, K, scale, cap, dh, R, past, lim)
            P, lse = softmax(s)
            O = P @ V
            rel = 2 * (es.amax(1, keepdim=True) if nk else torch.zeros(nq, 1, dtype=torch.float64)) + 2.0 ** -21
            A = P @ V.abs()
            few = nk * fl * (V.abs().amax(0, keepdim=True) if nk else 0)
            out["o"][a:b, h], out["lse"][h, a:b] = O, lse
            tol["o"][a:b, h] = (rel + u) * A + u * O.abs() + few + fl
            tol["lse"][h, a:b] = rel.squeeze(1) + 2.0 ** -21 * torch.where(torch.isinf(lse), torch.zeros_like(lse), lse).abs()
            if do is None:
                continue
            DO = do[a:b, h]
            dP = DO @ V.t()
            delta = (O * DO).sum(1, keepdim=True)
            dS = P * (dP - delta)
            us = u * u * 2 + 2.0 ** -21   # o_f32 comes from P in two parts
            edp = (Q.shape[1] + 4) * F32 * (DO.abs() @ V.abs().t())
            edl = (DO.abs() * ((rel + us) * A + few * u + (Q.shape[1] + 4) * F32 * O.abs())).sum(1, keepdim=True)
            eds = P * (rel * (dP - delta).abs() + edp + edl) + 2.0 ** -21 * dS.abs()
            if dist is not None:
                flat = at + 0 * at
                for o_, x in ((out, dS), (tol, eds + 2.0 ** -20 * dS.abs())):
                    o_["ddist"][h].index_add_(0, flat.reshape(-1), x.reshape(-1))
            dX = dS * slope
            # (the slope's own error: that of tanh, 2^-22 or so, on dS)
            row = DO.abs().amax(1, keepdim=True)
            top = DO.abs().amax() if nq else torch.zeros(())
            ex = eds * slope + 2.0 ** -20 * dS.abs() + u * dX.abs()
            fq, fk = (2.0 ** -21 * row, 2.0 ** -21 * top) if fl else (0.0 * row, 0.0 * top)
            out["dq"][a:b, h] = scale * (dX @ K)
            tol["dq"][a:b, h] = scale * ((ex + fq) @ K.abs()) + u * out["dq"][a:b, h].abs() + fl
            dk, dv = scale * (dX.t() @ Q), P.t() @ DO
            out["dk"][e:f, g] += dk
            out["dv"][e:f, g] += dv
            tol["dk"][e:f, g] += scale * ((ex + fk).t() @ Q.abs())
            tol["dv"][e:f, g] += (P * (rel + u + 2.0 ** -20)).t() @ DO.abs() + fl / 256 * DO.abs().sum(0, keepdim=True)
    if do is not None:
        for n in ("dk", "dv"):
            tol[n] += u * out[n].abs() + fl
    return out, tol


def bucket(r, n_buckets, bidirectional, far):
    half = n_buckets // 2 if bidirectional else n_buckets
    near, d = half // 2, abs(r) if bidirectional else max(-r, 0)
    b = d if d < near else min(half - 1, near + int(math.floor(math.log(d / near) / math.log(far / near) * (half - near) + 1e-9)))
    return b + (half if bidirectional and r > 0 else 0)


def check(got, want, tol, what):
    """Elementwise |got - want| <= tol; infinities and zeros of empty rows exactly."""
    got = got.double().cpu()
    same = (got == want) | ((got - want).abs() <= tol)
    assert same.all(), (f"{what}: {int((~same).sum())} of {same.numel()} off, worst "
                        f"{float(((got - want).abs() / tol.clamp_min(1e-300))[~same].max()):.2f} x the bound, first at "
                        f"{[int(x) for x in (~same).nonzero()[0]]}: {float(got[~same][0])} for {float(want[~same][0])}")
