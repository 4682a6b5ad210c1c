"""Plain CPU restatement of the delta-rule mixer and of the feed-forward of experts, from the equations, token by token.

TEST INFRASTRUCTURE ONLY; shares no code with the product.  See `layered` for the notation.
"""
import numpy as np

F = np.float64


def _linear(W, x):
    return x @ np.asarray(W, F).T


def _sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1 / (1 + e), e / (1 + e))


def new_state(m):
    ch = m["heads"] * m["vdim"] + 2 * m["key_heads"] * m["dim"]
    return {"S": np.zeros((m["heads"], m["vdim"], m["dim"]), F), "before": np.zeros((m["conv"] - 1, ch), F)}


def delta_rule(q, k, v, la, beta, S, q_scale, eps):
    """q, k [T, G, d], v [T, H, dv], la and beta [T, H]; S [H, dv, d] is advanced in place."""
    T, H = v.shape[:2]
    o = np.zeros(v.shape, F)
    for t in range(T):
        for h in range(H):
            g = h // (H // q.shape[1])
            kh, qh = k[t, g] / np.sqrt(k[t, g] @ k[t, g] + eps), q_scale * q[t, g] / np.sqrt(q[t, g] @ q[t, g] + eps)
            S[h] *= np.exp(la[t, h])
            S[h] += np.outer(beta[t, h] * (v[t, h] - S[h] @ kh), kh)
            o[t, h] = S[h] @ qh
    return o


def gated_delta(h, m, w, eps, st):
    T, H, G, d, dv, taps = h.shape[0], m["heads"], m["key_heads"], m["dim"], m["vdim"], m["conv"]
    nv, nk = H * dv, G * d
    z, u, dt, b = np.split(_linear(w("in"), h), [nv, 2 * nv + 2 * nk, 2 * nv + 2 * nk + H], axis=1)
    u = np.concatenate([st["before"], u])
    conv = np.asarray(w("conv"), F)
    x = np.stack([(conv.T * u[t:t + taps]).sum(axis=0) for t in range(T)]) + np.asarray(w("conv.b"), F)
    st["before"] = u[T:]
    x = x * _sigmoid(x)
    la = -np.exp(np.asarray(w("A_log"), F)) * np.logaddexp(0, dt + np.asarray(w("dt_bias"), F))
    o = delta_rule(x[:, nv + nk:].reshape(T, G, d), x[:, nv:nv + nk].reshape(T, G, d), x[:, :nv].reshape(T, H, dv), la, _sigmoid(b), st["S"],
                   d ** -0.5, 1e-6)
    o = o / np.sqrt((o ** 2).mean(axis=-1, keepdims=True) + eps) * np.asarray(w("norm"), F)
    return _linear(w("o"), o.reshape(T, nv) * z * _sigmoid(z))


def route(l, m, bias):
    """Experts and weights of one row of scores."""
    n = len(l)
    if m.get("score", "softmax") == "softmax":
        s = np.exp(l - l.max())
        s /= s.sum()
    else:
        s = _sigmoid(l)
    c = s + (0 if bias is None else bias)
    groups = m.get("groups", 1)
    size = n // groups
    best = [np.sort(c[g * size:(g + 1) * size])[::-1][:2].sum() for g in range(groups)]
    kept = sorted(range(groups), key=lambda g: (-best[g], g))[:m.get("top_groups", 1)]
    ids = sorted((e for g in kept for e in range(g * size, (g + 1) * size)), key=lambda e: (-c[e], e))[:m["top"]]
    w = s[ids]
    return ids, (w / w.sum() if m.get("renorm", True) else w) * m.get("scale", 1.0)


def experts(h, m, w, glu):
    """glu(gate, up) of rows."""
    scores = _linear(w("router"), h)
    bias = np.asarray(w("router.bias"), F) if m.get("bias") else None
    y = np.zeros((h.shape[0], h.shape[1]), F)
    for t in range(h.shape[0]):
        for e, a in zip(*route(scores[t], m, bias)):
            y[t] += a * _linear(w("down")[e], glu(_linear(w("gate")[e], h[t]), _linear(w("up")[e], h[t])))
    if m.get("shared_ff"):
        y += _linear(w("shared.down"), glu(_linear(w("shared.gate"), h), _linear(w("shared.up"), h)))
    return y
