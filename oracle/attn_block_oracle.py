"""64-bit numpy restatements of the attention block's operators: the norms around a block
with its gate and residual scale (forward and backward), rotary positions with several
axes, and softmax attention over a paged cache.  Written from the formulas, row by row
where that is plainest; test infrastructure only."""
import numpy as np


def _rows(gate, R):
    if gate is None:
        return 1.0
    g = np.asarray(gate, np.float64)
    g = g[None] if g.ndim == 1 else g
    return np.repeat(g, R // g.shape[0], axis=0)


def rms(x, eps):
    return 1.0 / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)


def block_norm(y, h, gamma_post=None, gate=None, gamma_pre=None, alpha=1.0, eps=1e-6):
    """(h', x): h' = alpha h + gate (RMSNorm(y) gamma_post), x = RMSNorm(h') gamma_pre."""
    y, h = np.asarray(y, np.float64), np.asarray(h, np.float64)
    u = y if gamma_post is None else y * rms(y, eps) * np.asarray(gamma_post, np.float64)
    hn = alpha * h + _rows(gate, y.shape[0]) * u
    return hn, None if gamma_pre is None else hn * rms(hn, eps) * np.asarray(gamma_pre, np.float64)


def block_norm_backward(y, h_out, dh_out=None, dx=None, gamma_post=None, gate=None, gamma_pre=None, alpha=1.0, eps=1e-6):
    """Gradients of block_norm from y and h'; also the sum of the terms' magnitudes of
    every result (key "mag"), which bounds what 32-bit arithmetic may lose."""
    y, hn = np.asarray(y, np.float64), np.asarray(h_out, np.float64)
    R, D = y.shape
    dt = np.zeros_like(hn) if dh_out is None else np.asarray(dh_out, np.float64).copy()
    mag = np.abs(dt)
    out, m = {}, {}
    if gamma_pre is not None:
        r2, gq = rms(hn, eps), np.asarray(gamma_pre, np.float64)
        n2, dx = hn * r2, np.asarray(dx, np.float64)
        g2 = dx * gq
        dt = dt + r2 * (g2 - n2 * np.mean(g2 * n2, axis=1, keepdims=True))
        mag = mag + r2 * (np.abs(g2) + np.abs(n2) * np.mean(np.abs(g2 * n2), axis=1, keepdims=True))
        out["dgamma_pre"], m["dgamma_pre"] = (dx * n2).sum(0), np.abs(dx * n2).sum(0)
    out["dh"], m["dh"] = alpha * dt, abs(alpha) * mag
    gt = _rows(gate, R)
    r1 = rms(y, eps) if gamma_post is not None else 1.0
    gp = 1.0 if gamma_post is None else np.asarray(gamma_post, np.float64)
    n1 = y * r1
    if gate is not None:
        G = 1 if np.ndim(gate) == 1 else gate.shape[0]
        shape = np.shape(gate)
        out["dgate"] = (dt * n1 * gp).reshape(G, R // G, D).sum(1).reshape(shape)
        m["dgate"] = (mag * np.abs(n1 * gp)).reshape(G, R // G, D).sum(1).reshape(shape)
    du, mdu = dt * gt, mag * np.abs(gt)
    if gamma_post is None:
        out["dy"], m["dy"] = du, mdu
    else:
        out["dgamma_post"], m["dgamma_post"] = (du * n1).sum(0), (mdu * np.abs(n1)).sum(0)
        g1, mg1 = du * gp, mdu * np.abs(gp)
        out["dy"] = r1 * (g1 - n1 * np.mean(g1 * n1, axis=1, keepdims=True))
        m["dy"] = r1 * (mg1 + np.abs(n1) * np.mean(mg1 * np.abs(n1), axis=1, keepdims=True))
    out["mag"] = m
    return out


def axis_of_pairs(sections):
    return np.repeat(np.arange(len(sections)), sections)


def rope(x, positions, inv_freq, sections, style="half", inverse=False):
    """x [T, H, D] turned pair by pair; positions [axes, T], inv_freq as stored (fp32 values)."""
    x = np.asarray(x, np.float64)
    ang = np.asarray(positions, np.float64)[axis_of_pairs(sections)] * np.asarray(inv_freq, np.float64)[:, None]
    c, s = np.cos(ang).T[:, None], np.sin(ang).T[:, None] * (-1.0 if inverse else 1.0)
    n = len(inv_freq)
    first, second = (slice(0, n), slice(n, 2 * n)) if style == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    out = x.copy()
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def attention(q, k, v, scale, causal=True, window=0):
    """One sequence: q [n, Hq, D] (its last n positions), k, v [L, Hkv, D].  Returns
    (out [n, Hq, D], lse [n, Hq], A): A = softmax @ |v|, which bounds what rounding the
    softmax's weights may lose.  Keys that a token does not see are left out altogether."""
    n, Hq, D = q.shape
    L, Hk, _ = k.shape
    G = Hq // Hk
    out, A = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    lse = np.full((n, Hq), -np.inf)
    for i in range(n):
        pos = L - n + i
        hi = min(pos + 1, L) if causal else L
        lo = max(0, pos + 1 - window) if window else 0
        if hi <= lo:
            continue
        for h in range(Hq):
            K, V = k[lo:hi, h // G].astype(np.float64), v[lo:hi, h // G].astype(np.float64)
            s = scale * (K @ q[i, h].astype(np.float64))
            m = s.max()
            p = np.exp(s - m)
            l = p.sum()
            out[i, h], A[i, h] = p @ V / l, p @ np.abs(V) / l
            lse[i, h] = m + np.log(l)
    return out, lse, A
