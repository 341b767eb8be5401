"""Plain 64-bit CPU forms of the token operators with their gradients by formula, and for every output a bound on what
rounding may do to it: the same sums taken over absolute values. Test infrastructure only."""
import math

import torch

U32, UBF = 2.0 ** -24, 2.0 ** -8      # half a step of f32 and bf16, relative


def rotary(x, w, pos, axes, base, eps, gy=None):
    """x, gy [B, T, H, D] double, w [D] or None, pos [B, T, A]. Returns y, or (y, gx, gw) with gy."""
    b, t, h, d = x.shape
    cos, sin = torch.ones(b, t, 1, d // 2, dtype=torch.double), torch.zeros(b, t, 1, d // 2, dtype=torch.double)
    at = 0
    for a, width in enumerate(axes):
        for i in range(width // 2):
            theta = pos[:, :, a].double() * base ** (-2.0 * i / width)
            cos[:, :, 0, at + i], sin[:, :, 0, at + i] = theta.cos(), theta.sin()
        at += width // 2

    def turn(v, s):
        out = torch.empty_like(v)
        out[..., 0::2] = v[..., 0::2] * cos - v[..., 1::2] * s
        out[..., 1::2] = v[..., 0::2] * s + v[..., 1::2] * cos
        return out

    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if w is not None else torch.ones(b, t, h, 1, dtype=torch.double)
    n = x * r * w if w is not None else x
    y = turn(n, sin)
    if gy is None:
        return y
    gn = turn(gy, -sin)
    if w is None:
        return y, gn, None
    xhat = x * r
    return y, r * (w * gn - xhat * (w * gn * xhat).mean(-1, keepdim=True)), (gn * xhat).sum((0, 1, 2))


def attention(q, k, v, ql=None, kl=None, scale=None, go=None):
    """Double [B, T, H, D] tensors. Returns a dict of outputs and, under "abs", their sums over absolute values; scores_abs
    is the largest sum |scale| |q| |k| of a score."""
    b, tq, hq, d = q.shape
    tk, hk = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out = {"o": torch.zeros_like(q), "gq": torch.zeros_like(q), "gk": torch.zeros_like(k), "gv": torch.zeros_like(v)}
    mag = {n: torch.zeros_like(x) for n, x in out.items()}
    top = 0.0
    for i in range(b):
        m = tq if ql is None else min(max(int(ql[i]), 0), tq)
        n = tk if kl is None else min(max(int(kl[i]), 0), tk)
        if not m or not n:
            continue
        for h in range(hq):
            kh = h // (hq // hk)
            Q, K, V = q[i, :m, h], k[i, :n, kh], v[i, :n, kh]
            s = scale * (Q @ K.T)
            top = max(top, (abs(scale) * (Q.abs() @ K.abs().T)).max().item())
            p = torch.softmax(s, 1)
            O = p @ V
            out["o"][i, :m, h], mag["o"][i, :m, h] = O, p @ V.abs()
            if go is None:
                continue
            G = go[i, :m, h]
            dp, dpa = G @ V.T, G.abs() @ V.abs().T
            delta, deltaa = (G * O).sum(1, keepdim=True), (G.abs() * (p @ V.abs())).sum(1, keepdim=True)
            ds, dsa = p * (dp - delta), p * (dpa + deltaa)
            out["gv"][i, :n, kh] += p.T @ G
            mag["gv"][i, :n, kh] += p.T @ G.abs()
            out["gq"][i, :m, h], mag["gq"][i, :m, h] = scale * ds @ K, abs(scale) * dsa @ K.abs()
            out["gk"][i, :n, kh] += scale * ds.T @ Q
            mag["gk"][i, :n, kh] += abs(scale) * dsa.T @ Q.abs()
    out["abs"], out["scores_abs"] = mag, top
    return out


def gate(g, act):
    """act(g), act'(g)"""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s + g * s * (1 - s))


def gated(x, w, b, act, gh=None):
    """Double x [M, C], w [2F, C], b [2F] or None. Returns a dict with the outputs, their sums over absolute values ("abs")
    and the rounding-free magnitude of the pre-activations ("z_abs")."""
    f = w.shape[0] // 2
    z = x @ w.T + (0 if b is None else b)
    za = x.abs() @ w.abs().T + (0 if b is None else b.abs())
    g, u = z[:, :f], z[:, f:]
    a, d = gate(g, act)
    out = {"h": a * u, "z_abs": za}
    # an error of e |z|_abs in the pre-activations reaches h through act' (at most 1.13 in size) and u, and through act(g)
    out["abs"] = {"h": a.abs() * za[:, f:] + 1.13 * za[:, :f] * u.abs() + (a * u).abs()}
    if gh is not None:
        gz = torch.cat((gh * u * d, gh * a), 1)
        # |act''| <= 1 for every gate here (relu: no second derivative away from zero)
        ga = torch.cat((gh.abs() * (za[:, f:] * d.abs() + u.abs() * za[:, :f] + (u * d).abs()), gh.abs() * (1.13 * za[:, :f] + a.abs())), 1)
        out.update(gz=gz, gx=gz @ w, gw=gz.T @ x, gb=gz.sum(0))
        out["abs"].update(gx=ga @ w.abs(), gw=ga.T @ x.abs(), gb=ga.sum(0))
        # the same, for a rounding of gz itself
        out["gz_abs"] = {"gx": gz.abs() @ w.abs(), "gw": gz.abs().T @ x.abs()}
    return out
