"""The sequence operators in float64, token by token: what the tests compare the kernels with."""
import numpy as np


def sigmoid(v):
    return 1 / (1 + np.exp(-v))


def layer_norm(x, gamma, beta, eps):
    x = x.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    hat = (x - mean) * rstd
    return hat * (1 if gamma is None else gamma.astype(np.float64)) + (0 if beta is None else beta.astype(np.float64)), mean[..., 0], rstd[..., 0]


def layer_norm_grad(dy, x, gamma, eps):
    dy, x = dy.astype(np.float64), x.astype(np.float64)
    _, mean, rstd = layer_norm(x, None, None, eps)
    hat = (x - mean[..., None]) * rstd[..., None]
    g = dy * (1 if gamma is None else gamma.astype(np.float64))
    dx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - hat * (g * hat).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    return dx, (dy * hat).sum(rows), dy.sum(rows)


def _conv_one(x, w, bias, silu, initial):
    """One sequence [T][C] -> (y, pre, extended x)."""
    taps = w.shape[1]
    ext = np.concatenate([initial, x])
    pre = np.zeros(x.shape) + (0 if bias is None else bias)
    for k in range(taps):
        pre += ext[taps - 1 - k:taps - 1 - k + len(x)] * w[:, k]
    return (pre * sigmoid(pre) if silu else pre), pre, ext


def causal_conv(xs, w, bias, silu, flip, initials=None):
    """Sequences (a list of [T][C]) -> (ys, final states)."""
    w = w.astype(np.float64)
    w = w if flip else w[:, ::-1]
    bias = None if bias is None else bias.astype(np.float64)
    ys, finals = [], []
    for i, x in enumerate(xs):
        x = x.astype(np.float64)
        init = np.zeros((w.shape[1] - 1, x.shape[1])) if initials is None else initials[i].astype(np.float64)
        y, _, ext = _conv_one(x, w, bias, silu, init)
        ys.append(y)
        finals.append(ext[len(x):])
    return ys, np.stack(finals)


def causal_conv_grad(dys, xs, w, bias, silu, flip, initials=None):
    """-> (dxs, dw, dbias, dinitials)"""
    w = w.astype(np.float64)
    w = w if flip else w[:, ::-1]
    taps = w.shape[1]
    bias = None if bias is None else bias.astype(np.float64)
    dw, db, dxs, dinits = np.zeros(w.shape), np.zeros(w.shape[0]), [], []
    for i, x in enumerate(xs):
        x, g = x.astype(np.float64), dys[i].astype(np.float64)
        init = np.zeros((taps - 1, x.shape[1])) if initials is None else initials[i].astype(np.float64)
        _, pre, ext = _conv_one(x, w, bias, silu, init)
        if silu:
            s = sigmoid(pre)
            g = g * s * (1 + pre * (1 - s))
        dext = np.zeros(ext.shape)
        for k in range(taps):
            at = slice(taps - 1 - k, taps - 1 - k + len(x))
            dext[at] += g * w[:, k]
            dw[:, k] += (g * ext[at]).sum(0)
        db += g.sum(0)
        dxs.append(dext[taps - 1:])
        dinits.append(dext[:taps - 1])
    return dxs, dw if flip else dw[:, ::-1], db, np.stack(dinits)


def selective_scan(xs, dts, A, Bs, Cs, D=None, zs=None, dt_bias=None, softplus=False, initials=None, dys=None, dfinals=None, magnitudes=False):
    """Sequences: x, dt, z [T][C], B, C [T][G][N].  -> dict(y=[...], final) and, with dys, the gradients.  `magnitudes`: every sum with
    the magnitudes of its terms (the decays as they are), which bounds what relative errors of the factors can do."""
    mag = np.abs if magnitudes else lambda v: v
    A = A.astype(np.float64)
    channels, N = A.shape
    out = dict(y=[], final=[])
    grads = {k: [] for k in ("x", "dt", "z", "B", "C", "initial")}
    grads.update(A=np.zeros(A.shape), D=np.zeros(channels), dt_bias=np.zeros(channels))
    D64 = np.zeros(channels) if D is None else mag(D.astype(np.float64))
    for i in range(len(xs)):
        x, dt, B, C = (np.asarray(v[i], np.float64) for v in (xs, dts, Bs, Cs))
        T, G = len(x), B.shape[1]
        share = np.arange(channels) // (channels // G)
        raw = dt + (0 if dt_bias is None else dt_bias.astype(np.float64))
        delta = np.logaddexp(0, raw) if softplus else raw
        decay = np.exp(delta[..., None] * A)
        x, B, C, delta = mag(x), mag(B), mag(C), mag(delta)
        h = np.zeros((channels, N)) if initials is None else mag(initials[i].astype(np.float64))
        hs, first = [], h
        y0 = np.zeros(x.shape)
        for t in range(T):
            h = decay[t] * h + (delta[t] * x[t])[:, None] * B[t, share]
            hs.append(h)
            y0[t] = (h * C[t, share]).sum(-1) + D64 * x[t]
        z = None if zs is None else np.asarray(zs[i], np.float64)
        out["y"].append(y0 if z is None else y0 * mag(z * sigmoid(z)))
        out["final"].append(h)
        if dys is None:
            continue
        dy = mag(np.asarray(dys[i], np.float64))
        if z is not None:
            s = sigmoid(z)
            grads["z"].append(dy * y0 * (s + np.abs(z) * s * (1 - s) if magnitudes else s * (1 + z * (1 - s))))
            dy = dy * mag(z * s)
        lam = np.zeros((channels, N)) if dfinals is None else mag(dfinals[i].astype(np.float64))
        dx, ddelta, dB, dC = D64 * dy, np.zeros(x.shape), np.zeros(B.shape), np.zeros(C.shape)
        for t in range(T - 1, -1, -1):
            lam = lam + dy[t][:, None] * C[t, share]
            dC[t] = (dy[t][:, None] * hs[t]).reshape(G, -1, N).sum(1)
            dB[t] = (lam * (delta[t] * x[t])[:, None]).reshape(G, -1, N).sum(1)
            lb = (lam * B[t, share]).sum(-1)
            lam = lam * decay[t]
            through = lam * (hs[t - 1] if t else first)
            grads["A"] += through * delta[t, :, None]
            ddelta[t] = (through * mag(A)).sum(-1) + x[t] * lb
            dx[t] += delta[t] * lb
        draw = ddelta * sigmoid(raw) if softplus else ddelta
        for k, v in (("x", dx), ("dt", draw), ("B", dB), ("C", dC), ("initial", lam)):
            grads[k].append(v)
        grads["D"] += (dy * x).sum(0)
        grads["dt_bias"] += draw.sum(0)
    out["final"] = np.stack(out["final"])
    if dys is not None:
        grads["initial"] = np.stack(grads["initial"])
        out.update({"d" + k: v for k, v in grads.items()})
    return out
