"""64-bit restatements of the recurrence, distillation, top-k and beam-search
operators, position by position from their definitions (they have no
counterpart in the reference)."""

import numpy as np


def _sigmoid(v):
    with np.errstate(over="ignore"):
        return np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))),
                        np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))


def _wide(gate, D):
    return np.repeat(gate, D // gate.shape[-1], axis=-1)


def recurrence(x, gate, h0=None, reset=None):
    """(h, h_last) of h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(gate)."""
    x, gate = np.asarray(x, np.float64), np.asarray(gate, np.float64)
    B, T, D = x.shape
    g = _wide(gate, D)
    a, z = _sigmoid(g), _sigmoid(-g)
    s = np.zeros((B, D)) if h0 is None else np.array(h0, np.float64)
    h = np.empty_like(x)
    for t in range(T):
        if reset is not None:
            s = np.where(np.asarray(reset)[:, t, None] != 0, 0.0, s)
        s = a[:, t] * s + z[:, t] * x[:, t]
        h[:, t] = s
    return h, s


def recurrence_backward(dh, x, gate, h0=None, reset=None, dlast=None):
    """(dx, dgate, dh0) by walking the positions backwards."""
    x, gate, dh = (np.asarray(v, np.float64) for v in (x, gate, dh))
    B, T, D = x.shape
    H = gate.shape[2]
    g = _wide(gate, D)
    a, z = _sigmoid(g), _sigmoid(-g)
    h, _ = recurrence(x, gate, h0, reset)
    carry = np.zeros((B, D)) if dlast is None else np.array(dlast, np.float64)
    dx, dg = np.empty_like(x), np.empty_like(x)
    for t in range(T - 1, -1, -1):
        before = h[:, t - 1] if t else (np.zeros((B, D)) if h0 is None
                                        else np.asarray(h0, np.float64))
        cut = np.zeros((B, 1), bool) if reset is None else np.asarray(reset)[:, t, None] != 0
        before = np.where(cut, 0.0, before)
        G = dh[:, t] + carry
        dx[:, t] = z[:, t] * G
        dg[:, t] = G * (before - x[:, t]) * a[:, t] * z[:, t]
        carry = np.where(cut, 0.0, a[:, t] * G)
    return dx, dg.reshape(B, T, H, D // H).sum(-1), carry


def distill(logits, top, ids, tau):
    """(loss (N, 1), p (N, K), q (N, V)): stored entries of -inf are absent."""
    z = np.asarray(logits, np.float64) / tau
    t = np.asarray(top, np.float64) / tau
    ids = np.asarray(ids, np.int64)
    N, V = z.shape
    loss, p, q = np.zeros((N, 1)), np.zeros(t.shape), np.zeros((N, V))
    for n in range(N):
        here = np.flatnonzero(t[n] != -np.inf)
        if here.size == 0:
            continue
        logp = t[n, here] - t[n, here].max()
        logp -= np.log(np.exp(logp).sum())
        logq = z[n] - z[n].max()
        logq -= np.log(np.exp(logq).sum())
        p[n, here] = np.exp(logp)
        q[n] = np.exp(logq)
        used = p[n, here] > 0
        loss[n, 0] = tau * tau * (p[n, here] * (logp - logq[ids[n, here]]))[used].sum()
    return loss, p, q


def distill_backward(grad, logits, top, ids, tau):
    _, p, q = distill(logits, top, ids, tau)
    d = q.copy()
    for n in range(d.shape[0]):
        np.add.at(d[n], np.asarray(ids, np.int64)[n][p[n] > 0], -p[n][p[n] > 0])
    return d * (np.asarray(grad, np.float64).reshape(-1, 1) * tau)


def topk(x, k):
    """(values, ids): descending, equal values by the lower id, NaN first."""
    x = np.asarray(x)
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    first = np.isnan(x)
    ids = np.stack([np.lexsort((np.arange(r.size), -r, ~f))[:k] for r, f in zip(key, first)])
    return np.take_along_axis(x, ids, 1), ids


def beam_select(logits, scores, finished=None, stop=None):
    """(scores, parents, tokens, finished), each item's proposals written out
    and sorted by score, beam and rank."""
    z = np.asarray(logits, np.float64)
    scores = np.asarray(scores, np.float64)
    B, W = scores.shape
    V = z.shape[1]
    out = [np.zeros((B, W)), np.zeros((B, W), np.int64), np.zeros((B, W), np.int64),
           np.zeros((B, W), np.int64)]
    for b in range(B):
        found = []
        for w in range(W):
            row, s = z[b * W + w], scores[b, w]
            if finished is not None and finished[b, w]:
                found += [(s if r == 0 else -np.inf, w, r, stop) for r in range(W)]
                continue
            order = np.lexsort((np.arange(V), -np.where(np.isnan(row), -np.inf, row)))[:W]
            with np.errstate(all="ignore"):
                shift = row - row[order[0]]
                logp = shift - np.log(np.exp(shift).sum())
            for r in range(W):
                t = int(order[r]) if r < V else 0
                found.append((s + logp[t] if r < V else -np.inf, w, r, t))
        found = [(-np.inf if np.isnan(c[0]) else c[0],) + c[1:] for c in found]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        for i, (s, w, _, t) in enumerate(found[:W]):
            out[0][b, i], out[1][b, i], out[2][b, i] = s, w, t
            if finished is not None:
                out[3][b, i] = int(bool(finished[b, w]) or t == stop)
    return out[0], out[1], out[2], (None if finished is None else out[3])


def beam_reorder(state, parents, used=None):
    """Rows of ``state`` (B W, ...) moved by ``parents`` (B, W), the first
    ``used`` entries of axis 1 only when given."""
    B, W = parents.shape
    rows = (np.asarray(parents, np.int64) + W * np.arange(B)[:, None]).reshape(-1)
    out = state.copy()
    if used is None:
        out[:] = state[rows]
    else:
        out[:, :used] = state[rows, :used]
    return out


# ------------------------------------------------------------------ the model


def _layernorm(x, g, b):
    mu = x.mean(-1, keepdims=True)
    return (x - mu) / np.sqrt(((x - mu) ** 2).mean(-1, keepdims=True) + 1e-5) * g + b


def _gelu(x):
    return 0.5 * x * (1 + np.tanh(0.7978845608 * (x + 0.044715 * x ** 3)))


def lm_forward(sd, ids, n_layers, reset=None):
    """Logits (batch, time, vocab) of the recurrent language model."""
    sd = {k: np.asarray(v, np.float64) for k, v in sd.items()}
    x = sd["tok_emb.weight"][np.asarray(ids, np.int64)]
    for i in range(n_layers):
        p = f"blocks.{i}."
        u = _layernorm(x, sd[p + "ln1.weightg"], sd[p + "ln1.weightb"])
        gate = u @ sd[p + "mixer.gate.weight"] + sd[p + "mixer.gate.bias"]
        h, _ = recurrence(u @ sd[p + "mixer.value.weight"], gate, None, reset)
        x = x + (h * _gelu(u @ sd[p + "mixer.mix.weight"])) @ sd[p + "mixer.out.weight"]
        u = _layernorm(x, sd[p + "ln2.weightg"], sd[p + "ln2.weightb"])
        u = _gelu(u @ sd[p + "mlp.0.weight"] + sd[p + "mlp.0.bias"])
        x = x + u @ sd[p + "mlp.2.weight"] + sd[p + "mlp.2.bias"]
    return _layernorm(x, sd["ln_f.weightg"], sd["ln_f.weightb"]) @ sd["tok_emb.weight"].T


def beam_search(logits_of, prompt, beams, n_new, stop=None):
    """(ids (batch, beams, seq + n), scores): every step re-runs ``logits_of`` on
    whole prefixes; finished beams are filled up with ``stop``.  ``gap`` is the
    smallest distance between neighbouring proposals around any cut or order."""
    out_ids, out_scores, gap = [], [], np.inf
    for row in np.asarray(prompt):
        live = [(0.0, list(row), False)]
        for _ in range(n_new):
            if all(f for _, _, f in live):
                live = [(s, ids + [stop], f) for s, ids, f in live]
                continue
            found = []
            for w, (s, ids, f) in enumerate(live):
                if f:
                    found.append((s, w, 0, stop))
                    continue
                z = np.asarray(logits_of(np.array([ids])), np.float64)[0, -1]
                logp = z - z.max() - np.log(np.exp(z - z.max()).sum())
                best = np.argsort(-logp, kind="stable")[:beams + 1]
                found += [(s + logp[t], w, r, int(t)) for r, t in enumerate(best)]
            found.sort(key=lambda c: (-c[0], c[1], c[2]))
            top = np.array([c[0] for c in found[:beams + 1]])
            gap = min(gap, np.abs(np.diff(top)).min())
            live = [(s, live[w][1] + [t], live[w][2] or (stop is not None and t == stop))
                    for s, w, _, t in found[:beams]]
        out_ids.append([ids for _, ids, _ in live])
        out_scores.append([s for s, _, _ in live])
    return np.array(out_ids), np.array(out_scores), gap
