"""Float64 restatement of the recurrent layers' operators, token by token and channel by channel from their definitions
(include/kvhip.h).  Test infrastructure only; pinned to nothing but the formulas."""
import numpy as np


def span(b, n, left_pad, lengths):
    """The tokens of sequence b that are there: [from, end)."""
    first = 0 if left_pad is None else int(min(max(left_pad[b], 0), n))
    end = n if lengths is None else int(min(max(lengths[b], first), n))
    return first, end


def short_convolution(x, weight, bias=None, window=None, silu=True, left_pad=None, lengths=None):
    """x [B,L,C], weight [C,W] -> (y [B,L,C], new window [B,W-1,C])."""
    B, n, c = x.shape
    W = weight.shape[1]
    window = np.zeros((B, W - 1, c)) if window is None else window
    y, new = np.zeros((B, n, c)), np.empty((B, W - 1, c))
    for b in range(B):
        first, end = span(b, n, left_pad, lengths)
        e = np.concatenate([window[b], x[b, first:end]]).astype(np.float64)
        for t in range(end - first):
            s = np.zeros(c) if bias is None else bias.astype(np.float64).copy()
            for w in range(W):
                s += weight[:, w] * e[t + w]
            y[b, first + t] = s / (1 + np.exp(-s)) if silu else s
        new[b] = e[end - first:]
    return y, new


def gated_delta(q, k, v, a, b, a_log=None, dt_bias=None, state=None, scale=None, norm_eps=1e-6, left_pad=None, lengths=None):
    """q, k [B,L,Hk,Dk], v [B,L,Hv,Dv], a, b [B,L,Hv] -> (out [B,L,Hv,Dv], state [B,Hv,Dv,Dk], the largest row of a state or
    element of v that was met)."""
    q, k, v, a, b = (np.asarray(t, np.float64) for t in (q, k, v, a, b))
    B, n, Hk, Dk = k.shape
    Hv, Dv = v.shape[2:]
    scale = Dk ** -0.5 if scale is None else scale
    out, new = np.zeros((B, n, Hv, Dv)), np.zeros((B, Hv, Dv, Dk))
    largest = 0.0
    for i in range(B):
        first, end = span(i, n, left_pad, lengths)
        s = np.zeros((Hv, Dv, Dk)) if state is None else np.asarray(state[i], np.float64).copy()
        largest = max(largest, float(np.sqrt((s * s).sum(-1)).max()))
        for t in range(first, end):
            for h in range(Hv):
                kk, qq = k[i, t, h // (Hv // Hk)], q[i, t, h // (Hv // Hk)] * 1.0
                if norm_eps > 0:
                    kk = kk / np.sqrt((kk * kk).sum() + norm_eps)
                    qq = qq / np.sqrt((qq * qq).sum() + norm_eps)
                if a_log is None:
                    g, beta = np.exp(a[i, t, h]), b[i, t, h]
                else:
                    g = np.exp(-np.exp(a_log[h]) * np.logaddexp(0.0, a[i, t, h] + (0.0 if dt_bias is None else dt_bias[h])))
                    beta = 1 / (1 + np.exp(-b[i, t, h]))
                s[h] = g * s[h]
                u = beta * (v[i, t, h] - s[h] @ kk)
                s[h] = s[h] + np.outer(u, kk)
                out[i, t, h] = s[h] @ (scale * qq)
                largest = max(largest, float(np.sqrt((s[h] * s[h]).sum(-1)).max()), float(np.abs(v[i, t, h]).max()))
        new[i] = s
    return out, new, largest
