"""64-bit restatements of rotary positions, linear attention with a decay for each head,
and group norm with an activation, from their definitions (they have no counterpart in
the reference)."""

import numpy as np


def rotary(x, heads, frequencies, gain=1.0, positions=None, offset=0, layout="half", back=False):
    """x (B, T, D) with every head's first pairs turned by position * frequency."""
    x = np.asarray(x, np.float64)
    B, T, D = x.shape
    r = 2 * len(frequencies)
    p = np.arange(T) if positions is None else np.asarray(positions).astype(np.int64)
    angle = np.broadcast_to((p + offset)[..., None] * np.asarray(frequencies), (B, T, r // 2))
    c, s = gain * np.cos(angle)[:, :, None], gain * np.sin(angle)[:, :, None]
    s = -s if back else s
    y = x.reshape(B, T, heads, D // heads).copy()
    i = np.arange(r // 2)
    a, b = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    u, v = y[..., a], y[..., b]
    y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    return y.reshape(B, T, D)


def _heads(t, H):
    t = np.asarray(t, np.float64)
    return t.reshape(*t.shape[:-1], H, t.shape[-1] // H)


def linear_attention(q, k, v, log_decay, h0=None, reset=None, scale=1.0):
    """(o, last) of S_t = exp(log_decay) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t."""
    lam = np.exp(np.asarray(log_decay, np.float64))[None, :, None, None]
    H = lam.shape[1]
    q, k, v = (_heads(t, H) for t in (q, k, v))
    B, T, _, dk = q.shape
    S = np.zeros((B, H, dk, v.shape[-1])) if h0 is None else np.array(h0, np.float64)
    o = np.empty((B, T, H, v.shape[-1]))
    for t in range(T):
        if reset is not None:
            S = np.where(np.asarray(reset)[:, t, None, None, None] != 0, 0.0, lam * S)
        else:
            S = lam * S
        S = S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * np.einsum("bhp,bhpr->bhr", q[:, t], S)
    return o.reshape(B, T, -1), S


def linear_attention_backward(do, q, k, v, log_decay, h0=None, reset=None, dlast=None, scale=1.0):
    """(dq, dk, dv, dh0): the states forwards, their gradients R backwards."""
    lam = np.exp(np.asarray(log_decay, np.float64))[None, :, None, None]
    H = lam.shape[1]
    q, k, v, do = (_heads(t, H) for t in (q, k, v, do))
    B, T, _, dk = q.shape
    S = np.zeros((B, H, dk, v.shape[-1])) if h0 is None else np.array(h0, np.float64)
    cut = np.zeros((B, T), bool) if reset is None else np.asarray(reset) != 0
    dq, dkey, dval = np.empty_like(q), np.empty_like(k), np.empty_like(v)
    for t in range(T):
        S = np.where(cut[:, t, None, None, None], 0.0, lam * S)
        S = S + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * np.einsum("bhpr,bhr->bhp", S, do[:, t])
    R = np.zeros_like(S) if dlast is None else np.array(dlast, np.float64)
    for t in range(T - 1, -1, -1):
        R = R + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dkey[:, t] = np.einsum("bhpr,bhr->bhp", R, v[:, t])
        dval[:, t] = np.einsum("bhpr,bhp->bhr", R, k[:, t])
        R = np.where(cut[:, t, None, None, None], 0.0, lam * R)
    return dq.reshape(B, T, -1), dkey.reshape(B, T, -1), dval.reshape(B, T, -1), R


def _swept(x, y, z, log_decay, start, chunk=128):
    """``(out, last)`` of X_t = l X_{t-1} + y_t z_t^T, out_t = X_t^T x_t a chunk of positions at a
    time; x, y (B, T, H, p), z (B, T, H, r), start (B, H, p, r)."""
    ld = np.asarray(log_decay, np.float64)
    X, out = start, np.empty(z.shape)
    for a in range(0, z.shape[1], chunk):
        xs, ys, zs = (t[:, a:a + chunk].transpose(0, 2, 1, 3) for t in (x, y, z))
        i = np.arange(xs.shape[2])
        n = len(i)
        apart = i[:, None] - i
        w = np.where(apart >= 0, np.exp(np.maximum(apart, 0) * ld[:, None, None]), 0.0)
        before = np.exp((i + 1) * ld[:, None])[..., None]
        left = np.exp((n - 1 - i) * ld[:, None])[..., None]
        out[:, a:a + chunk] = (((xs @ ys.swapaxes(2, 3)) * w) @ zs
                               + before * (xs @ X)).transpose(0, 2, 1, 3)
        X = np.exp(n * ld)[:, None, None] * X + (left * ys).swapaxes(2, 3) @ zs
    return out, X


def linear_attention_long(do, q, k, v, log_decay, h0, dlast):
    """(o, last, dq, dk, dv, dh0) of ``linear_attention`` and its backward without resets, for rows
    too long to go through position by position."""
    H = len(log_decay)
    q, k, v, do = (_heads(t, H) for t in (q, k, v, do))
    h0, R = np.asarray(h0, np.float64), np.asarray(dlast, np.float64)
    o, last = _swept(q, k, v, log_decay, h0)
    dq = _swept(do, v, k, log_decay, h0.swapaxes(2, 3))[0]
    # backwards the decay comes after a position: before the first one it is taken off again
    lam = np.exp(np.asarray(log_decay, np.float64))[:, None, None]
    turned = [t[:, ::-1] for t in (q, k, v, do)]
    dv, last_R = _swept(turned[1], turned[0], turned[3], log_decay, R / lam)
    dk = _swept(turned[2], turned[3], turned[0], log_decay, R.swapaxes(2, 3) / lam)[0]
    flat = (t.reshape(*t.shape[:2], -1) for t in (o, dq, dk[:, ::-1], dv[:, ::-1]))
    o, dq, dk, dv = flat
    return o, last, dq, dk, dv, lam * last_R


def _logistic(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1 / (1 + e), e / (1 + e))


_C = 0.7978845608


def act(v, name):
    if name is None:
        return v
    if name == "relu":
        return np.maximum(v, 0)
    if name == "silu":
        return v * _logistic(v)
    return 0.5 * v * (1 + np.tanh(_C * (v + 0.044715 * v ** 3)))


def slope(v, name):
    if name is None:
        return np.ones_like(v)
    if name == "relu":
        return (v > 0).astype(np.float64)
    if name == "silu":
        p = _logistic(v)
        return p + v * p * _logistic(-v)
    t = np.tanh(_C * (v + 0.044715 * v ** 3))
    return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * _C * (1 + 3 * 0.044715 * v * v)


def _normalised(x, groups, gamma, beta, eps):
    x = np.asarray(x, np.float64)
    N, C = x.shape[0], x.shape[-1]
    w = x.reshape(N, -1, groups, C // groups)
    mean = w.mean((1, 3), keepdims=True)
    inv = 1 / np.sqrt(((w - mean) ** 2).mean((1, 3), keepdims=True) + eps)
    z = (w - mean) * inv
    gamma = np.ones(C) if gamma is None else np.asarray(gamma, np.float64)
    beta = np.zeros(C) if beta is None else np.asarray(beta, np.float64)
    gamma, beta = gamma.reshape(groups, -1), beta.reshape(groups, -1)
    return z, z * gamma + beta, gamma, mean, inv


def group_norm(x, groups, gamma=None, beta=None, activation=None, gate=None, eps=1e-5):
    """(y, mean, inv) over x (N, ..., C)."""
    _, n, _, mean, inv = _normalised(x, groups, gamma, beta, eps)
    n = n.reshape(x.shape)
    y = act(n, activation) if gate is None else n * act(np.asarray(gate, np.float64), activation)
    return y, mean[:, 0, :, 0], inv[:, 0, :, 0]


def group_norm_backward(dy, x, groups, gamma=None, beta=None, activation=None, gate=None, eps=1e-5):
    """(dx, dgamma, dbeta, dgate)."""
    z, n, g, _, inv = _normalised(x, groups, gamma, beta, eps)
    dy = np.asarray(dy, np.float64).reshape(z.shape)
    dgate = None
    if gate is None:
        dn = dy * slope(n, activation)
    else:
        w = np.asarray(gate, np.float64).reshape(z.shape)
        dn = dy * act(w, activation)
        dgate = (dy * n * slope(w, activation)).reshape(x.shape)
    u = dn * g
    dx = inv * (u - u.mean((1, 3), keepdims=True) - z * (u * z).mean((1, 3), keepdims=True))
    return (dx.reshape(x.shape), (dn * z).sum((0, 1)).reshape(-1), dn.sum((0, 1)).reshape(-1),
            dgate)


def retention_forward(sd, pre, x, heads, log_decay, reset=None, off=None):
    """The retention layer ``pre`` of a state_dict on x (B, T, D), in 64 bits.  ``off(value,
    terms)``: what stands in for a value whose terms' sizes sum up to ``terms``."""
    D = x.shape[-1]
    hd = D // heads
    off = off or (lambda value, terms: value)
    f = 10000.0 ** (-2 * np.arange(hd // 2) / hd)

    def lin(name, x):
        w = np.asarray(sd[pre + name + ".weight"], np.float64)
        return off(x @ w, np.abs(x) @ np.abs(w))

    q, k = (rotary(lin(n, x), heads, f) for n in ("q", "k"))
    v = lin("v", x)
    scale = hd ** -0.5
    o = off(linear_attention(q, k, v, log_decay, None, reset, scale)[0],
            linear_attention(np.abs(q), np.abs(k), np.abs(v), log_decay, None, reset, scale)[0])
    rows = (-1, D)
    y = group_norm(o.reshape(rows), heads, sd[pre + "norm.weight"], sd[pre + "norm.bias"], "silu",
                   lin("gate", x).reshape(rows))[0]
    return lin("out", y.reshape(x.shape))


def lm_forward(sd, ids, n_layers, heads, log_decay, reset=None, off=None):
    """Logits of a RecurrentLM whose mixers are retentions, in 64 bits."""
    from .recurrent import _gelu, _layernorm

    w = {k: np.asarray(v, np.float64) for k, v in sd.items()}
    h = w["tok_emb.weight"][np.asarray(ids, np.int64)]
    for i in range(n_layers):
        p = f"blocks.{i}."
        n = _layernorm(h, w[p + "ln1.weightg"], w[p + "ln1.weightb"])
        h = h + retention_forward(w, p + "mixer.", n, heads, log_decay, reset, off)
        n = _layernorm(h, w[p + "ln2.weightg"], w[p + "ln2.weightb"])
        h = h + _gelu(n @ w[p + "mlp.0.weight"] + w[p + "mlp.0.bias"]) @ w[p + "mlp.2.weight"] \
            + w[p + "mlp.2.bias"]
    h = _layernorm(h, w["ln_f.weightg"], w["ln_f.weightb"])
    return h @ w["tok_emb.weight"].T


def lm_error(sd, ids, n_layers, heads, log_decay, reset=None, part=2.0 ** -20, draws=4):
    """(B, T): by how much a position's logits move when every value of the mixers is off by up to ``part`` of
    its terms' sizes: the norm of a head divides by the head's own size, so outputs that
    cancel pass their errors on enlarged."""
    ref = lm_forward(sd, ids, n_layers, heads, log_decay, reset)
    rng = np.random.default_rng(0)

    def off(value, terms):
        return value + rng.uniform(-part, part, value.shape) * terms

    return np.max([np.abs(lm_forward(sd, ids, n_layers, heads, log_decay, reset, off) - ref).max(-1)
                   for _ in range(draws)], 0)
