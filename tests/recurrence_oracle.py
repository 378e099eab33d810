"""The gated recurrence and its gradient in float64 on the host, token by token.

    a = sigmoid(f + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y = h silu(gate)
"""
import numpy as np


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _sigmoid(u):
    return 1.0 / (1.0 + np.exp(-u))


def recurrence(x, f, bias=None, gate=None, h0=None, reset=None, dy=None, dh=None):
    """Results (and, with dy, gradients) as a dict of float64 arrays; arguments are torch tensors."""
    x, f, bias, gate, h0, dy, dh = (_f64(t) for t in (x, f, bias, gate, h0, dy, dh))
    cut = np.zeros(x.shape[:2], bool) if reset is None else reset.cpu().numpy().astype(bool)
    B, L, C = x.shape
    u = f if bias is None else f + bias
    a, z = _sigmoid(u), _sigmoid(-u)
    h, prev = np.zeros_like(x), np.zeros_like(x)
    s = np.zeros((B, C)) if h0 is None else h0.copy()
    for t in range(L):
        s = np.where(cut[:, t, None], 0.0, s)
        prev[:, t] = s
        s = a[:, t] * s + z[:, t] * x[:, t]
        h[:, t] = s
    sg = None if gate is None else _sigmoid(gate)
    out = {"y": h if gate is None else h * gate * sg, "h": s}
    if dy is None:
        return out
    g, c = np.zeros_like(x), np.zeros((B, C)) if dh is None else dh.copy()
    into = dy if gate is None else dy * gate * sg
    for t in range(L - 1, -1, -1):
        g[:, t] = into[:, t] + c
        c = np.where(cut[:, t, None], 0.0, a[:, t] * g[:, t])
    df = g * (prev - x) * a * z
    out.update(dx=g * z, df=df, dbias=df.sum((0, 1)), dbias_abs=np.abs(df).sum((0, 1)), dh0=c)
    if gate is not None:
        out["dgate"] = dy * h * sg * (1.0 + gate * (1.0 - sg))
    return out
