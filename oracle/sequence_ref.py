"""Plain 64-bit forms of the sequence operators (rotary positions, differential attention, group norm) with the error bounds their tests use.

Every function takes tensors of the operator's type, works in float64 on the CPU and returns a dict name -> (value, bound): ``bound`` is how far a
correct kernel may be off at each place.  The bounds count roundings: ``u`` = half a step of the type, ``e`` = half a step of fp32.
"""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny_step(dtype):
    """absolute rounding error below the type's smallest normal number"""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def _d(t):
    return t.detach().cpu().double()


def rotary(x, freq, positions, layout, amplitude, inverse=False):
    """one fp32 sine and cosine of a reduced angle (an error of 2 e from the angle's own rounding, pi e at most, and 2 e from the function: 6 e),
    two products and a sum (3 e), one rounding to the type.  The angle itself is a 64-bit product: in the kernel the frequency is divided by 2 pi
    and multiplied by the position (2 roundings, and the constant's own), here multiplied once: 4 * 2^-53 of the angle, which shows from
    positions of 1e9 on (2^33: 8.6e9 * 4 * 2^-53 = 3.8e-6)"""
    y = _d(x).clone()
    half = freq.numel()
    b, n = y.shape[:2]
    pos = torch.arange(n).expand(b, n) if positions is None else _d(positions).expand(b, n)
    t = pos.double()[:, :, None, None] * freq
    c, s = t.cos() * amplitude, t.sin() * amplitude * (-1 if inverse else 1)
    i = torch.arange(half)
    i0, i1 = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    u, v = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = u * c - v * s, u * s + v * c
    bound = half_step(x.dtype) * y.abs() + tiny_step(x.dtype)
    both = (u.abs() + v.abs()) * abs(amplitude) * (10 * E32 + 4 * 2.0 ** -53 * t.abs())
    bound[..., i0] += both
    bound[..., i1] += both
    bound[..., 2 * half:] = 0.0
    return y, bound


def _activation(z, kind):
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def group_norm(x, groups, weight, bias, eps, activation, lengths, dy=None):
    """A sum of E terms is a chain of at most E / 64 additions (64 lanes or more) and a tree: K = E / 64 + 32 roundings of 32 bits, which also
    cover the dozen of the formula itself and of exp / erf; slopes of the activations are below 1.2, their slopes below 1."""
    u, tiny = half_step(x.dtype), tiny_step(x.dtype)
    X = _d(x)
    b, n, c = X.shape
    w = _d(weight) if weight is not None else torch.ones(c).double()
    o = _d(bias) if bias is not None else torch.zeros(c).double()
    wu = half_step(weight.dtype) if weight is not None else 0.0
    DY = _d(dy) if dy is not None else torch.zeros_like(X)
    out = {k: (torch.zeros_like(X), torch.zeros_like(X)) for k in ("y", "dx")}
    grads = {k: (torch.zeros(c).double(), torch.zeros(c).double()) for k in ("dweight", "dbias")}
    cg = c // groups
    for i in range(b):
        length = n if lengths is None else int(lengths[i])
        if length == 0:
            continue
        for g in range(groups):
            s = slice(g * cg, (g + 1) * cg)
            part = X[i, :length, s]
            k = (part.numel() / 64 + 32) * E32
            mean, var = part.mean(), part.var(correction=0)
            r = 1 / torch.sqrt(var + eps)
            hat = (part - mean) * r
            big = part.abs().max() * r      # what the mean's own rounding is relative to
            dhat = k * (big + hat.abs() * (1 + big * big * k))
            z = hat * w[s] + o[s]
            y, slope = _activation(z, activation)
            out["y"][0][i, :length, s] = y
            dz_bound = dhat * w[s].abs() + 4 * E32 * (z.abs() + o[s].abs())
            out["y"][1][i, :length, s] = 1.2 * dz_bound + 32 * E32 * (y.abs() + z.abs()) + u * y.abs() + tiny
            if dy is None:
                continue
            d = DY[i, :length, s] * slope
            if activation == "relu":      # a kink: places closer to it than the error of z may fall on either side
                dslope = (z.abs() <= 2 * dz_bound).double()
            else:
                dslope = dz_bound + 32 * E32
            dd = DY[i, :length, s].abs() * dslope + 4 * E32 * d.abs()
            t, dt = d * w[s], dd * w[s].abs() + 2 * E32 * (d * w[s]).abs()
            m1, m2 = t.mean(), (t * hat).mean()
            dm1, dm2 = dt.mean() + k * t.abs().mean(), (dt * hat.abs() + t.abs() * dhat).mean() + k * (t * hat).abs().mean()
            dx = r * (t - m1 - hat * m2)
            out["dx"][0][i, :length, s] = dx
            out["dx"][1][i, :length, s] = (r * (dt + dm1 + hat.abs() * dm2 + dhat * m2.abs()) + (k + 8 * E32) * r * (t.abs() + m1.abs() + (hat * m2).abs())
                                           + u * dx.abs() + tiny)
            grads["dweight"][0][s] += (d * hat).sum(0)
            grads["dweight"][1][s] += (dd * hat.abs() + d.abs() * dhat + k * (d * hat).abs()).sum(0)
            grads["dbias"][0][s] += d.sum(0)
            grads["dbias"][1][s] += (dd + k * d.abs()).sum(0)
    if dy is None:
        return {"y": out["y"]}
    more = (b / 4 + 8) * E32      # the records of the samples, added in a few chains
    for k, (v, e) in grads.items():
        # (the rounding to the weight's type has a relative part and, below the smallest normal number, a fixed one: an fp16 gradient of 2.4e-5 lies
        # under 2^-14, where the steps are 2^-24 apart: off by up to 2^-25 = 3.0e-8, where 2^-11 of it is 1.2e-8)
        grads[k] = (v, e * (1 + more) + more * v.abs() * 4 + wu * v.abs() + E32 * e + (tiny_step(weight.dtype) if weight is not None else 0.0))
    return {**out, **grads}


def differential_attention(q, k, v, lam, lengths, causal, scale, do=None, full=False):
    """Scores: d products summed in 32 bits (d e of the sum of magnitudes), an exponential (8 e); weights P rounded once (u) for the product
    with V, summed in 32 bits (64 e: chains per 32 keys and the rescalings); D from the rounded outputs (u each); dS rounded once (u).

    ``full``: nothing but the results is rounded to the type.  P and dS enter as two terms of the type, the second one the first one's remainder
    (at most u of it, rounded by u: u^2 is left out of 1), and D is a sum in 32 bits over 32-bit factors (no u)."""
    u = half_step(q.dtype) if q.dtype != torch.float32 else 0.0      # 32-bit operands enter the matrix instructions as they are
    ot, tiny = half_step(q.dtype), tiny_step(q.dtype)
    saved, saved_tiny = (0.0, 0.0) if full else (ot, tiny)      # of the outputs that D is formed from
    u = u * u if full else u
    Q, K, V, L = _d(q), _d(k), _d(v), _d(lam)
    b, nq, h2, d = Q.shape
    nk, hk, dv = V.shape[1:]
    h = h2 // 2
    out = {"o": (torch.zeros(b, nq, h, dv).double(), torch.zeros(b, nq, h, dv).double())}
    if do is not None:
        DO = _d(do)
        out.update({name: (torch.zeros_like(t), torch.zeros_like(t)) for name, t in (("dq", Q), ("dk", K), ("dv", V), ("dlam", L))})
    for i in range(b):
        n = nk if lengths is None else max(0, min(nk, int(lengths[i])))
        if n == 0:
            continue
        seen = torch.ones(nq, n, dtype=torch.bool)
        if causal is not None:
            at = torch.arange(nq)[:, None] + (n - nq if causal == "end" else 0)
            seen = torch.arange(n)[None, :] <= at
        for head in range(h):
            kv = head // (h // hk)
            val, lm = V[i, :n, kv], L[head]
            p, f = [], []
            for m in range(2):
                qm, km = Q[i, :, 2 * head + m], K[i, :n, 2 * kv + m]
                s = (qm @ km.t() * scale).masked_fill(~seen, -math.inf)
                top = s.amax(1, keepdim=True)
                e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
                t = e.sum(1, keepdim=True)
                p.append(e / t.masked_fill(t == 0, 1.0))
                ds = (qm.abs() @ km.abs().t() * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True) * (d + 4) * E32
                f.append(2 * ds + 72 * E32)      # relative error of a 32-bit weight
            o = [x @ val for x in p]
            sub = tiny if q.dtype == torch.float16 else 0.0      # weights below the normal range
            do_ = [((fi + u) * x + sub) @ val.abs() for x, fi in zip(p, f)]
            res = o[0] - lm * o[1]
            out["o"][0][i, :, head] = res
            err_o = do_[0] + lm.abs() * do_[1] + 4 * E32 * (o[0].abs() + (lm * o[1]).abs())
            out["o"][1][i, :, head] = err_o + ot * res.abs() + tiny
            if do is None:
                continue
            g = DO[i, :, head]
            ga = g.abs()
            w = p[0] - lm * p[1]
            # (each map's weights are rounded on their own and multiplied with dO on their own: |d(P1 - lam P2)| <= u P1 + u |lam| P2)
            wa = p[0] + lm.abs() * p[1]
            dw = f[0] * p[0] + lm.abs() * f[1] * p[1]
            out["dv"][0][i, :n, kv] += w.t() @ g
            out["dv"][1][i, :n, kv] += (dw + u * wa + 2 * sub + 64 * E32 * wa).t() @ ga
            dp, dpa = g @ val.t(), (dv + 4) * E32 * (ga @ val.abs().t())
            d2 = (g * o[1]).sum(1, keepdim=True)
            e2 = (ga * (do_[1] + saved * o[1].abs() + saved_tiny + dv * E32 * o[1].abs())).sum(1, keepdim=True)
            d1 = (g * o[0]).sum(1, keepdim=True)
            e1 = (ga * (err_o + saved * res.abs() + saved_tiny + dv * E32 * res.abs())).sum(1, keepdim=True) + lm.abs() * (e2 + dv * E32 * (ga * o[1].abs()).sum(1, keepdim=True))
            out["dlam"][0][head] -= d2.sum()
            out["dlam"][1][head] += e2.sum() + (b * nq / 1024 + 32) * E32 * d2.abs().sum()
            for m, (sign, dm, em) in enumerate(((1.0, d1, e1), (-lm, d2, e2))):
                ds = sign * p[m] * (dp - dm)
                eds = abs(sign) * p[m] * (dpa + em + 4 * E32 * (dp.abs() + dm.abs())) + (f[m] + u + 4 * E32) * ds.abs() + sub + 64 * E32 * ds.abs()
                eds = torch.where(seen, eds, torch.zeros_like(eds))
                km, qm = K[i, :n, 2 * kv + m], Q[i, :, 2 * head + m]
                out["dq"][0][i, :, 2 * head + m] = scale * ds @ km
                out["dq"][1][i, :, 2 * head + m] = scale * eds @ km.abs()
                out["dk"][0][i, :n, 2 * kv + m] += scale * ds.t() @ qm
                out["dk"][1][i, :n, 2 * kv + m] += scale * eds.t() @ qm.abs()
    if do is not None:
        for name, t in (("dq", ot), ("dk", ot), ("dv", ot), ("dlam", half_step(lam.dtype))):
            val, e = out[name]
            out[name] = (val, e * (1 + 1e-3) + t * (val.abs() + e) + tiny)
    return out
