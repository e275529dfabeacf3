"""Operators for recurrent students of a language model, as measured cases.

Four operators, each in a plain form (elementary torch operations in 32 bits)
and, with ``own`` set, through the framework's public entry points:

* ``recurrence``: the gated linear recurrence
  ``h_t = a_t h_{t-1} + (1 - a_t) x_t``, ``a_t = sigmoid(gate_t)`` (``a_t``
  taken as 0 where a new document starts), forward, forward and backward, and
  one token at a time;
* ``distill``: the divergence of a student's logits from a teacher's top
  logits, ``tau^2 KL(softmax(top / tau) || softmax(logits / tau))`` per row,
  forward, and forward and backward;
* ``topk``: the k largest logits of each row with their ids, in descending
  order, ties to the lower id;
* ``beam``: one step of beam search, the selection over beams and vocabulary
  and the reordering of the beams' states in place.

The framework's tensors are lent the memory of the torch inputs, and its
outputs are viewed as torch tensors, without copies.  The per-token calls
(``recurrence`` one token at a time, ``beam``) are recorded as a CUDA graph
and replayed, which is how the framework's generation runs its steps; the
others are direct calls.
"""

import math

import numpy as np
import torch

own = False

BIG = 50304          # vocabulary of the GPT2-scaled configuration
STOP = 0             # stop token of the beam cases


def listed():
    return [
        # training on long documents packed into rows of 8192 tokens, a gate
        # per channel (the Hyena benchmark's batch, length and width)
        {"name": "recurrence train long", "op": "recurrence", "mode": "train", "B": 16, "T": 8192,
         "D": 256, "H": 256, "h0": False, "reset": True},
        # a training step at the GPT2-scaled width, one gate a head of 64
        {"name": "recurrence train heads", "op": "recurrence", "mode": "train", "B": 8, "T": 1024,
         "D": 1024, "H": 16, "h0": True, "reset": False},
        # prefill of a ragged batch, rows that no vector width divides
        {"name": "recurrence prefill odd", "op": "recurrence", "mode": "forward", "B": 3,
         "T": 4097, "D": 250, "H": 250, "h0": True, "reset": False},
        # prefill of one long document: few channels, many steps
        {"name": "recurrence prefill one", "op": "recurrence", "mode": "forward", "B": 1,
         "T": 65536, "D": 256, "H": 256, "h0": False, "reset": False},
        # one decode step of 32 sequences
        {"name": "recurrence step", "op": "recurrence", "mode": "step", "B": 32, "T": 1, "D": 1024,
         "H": 1024, "h0": True, "reset": False},
        # a training step of 4 x 1024 tokens against a stored teacher
        {"name": "distill train", "op": "distill", "mode": "train", "N": 4096, "V": BIG, "K": 64,
         "tau": 2.0, "ragged": False},
        # small odd vocabulary, rows with fewer stored teacher logits
        {"name": "distill train odd", "op": "distill", "mode": "train", "N": 1023, "V": 1021,
         "K": 17, "tau": 1.5, "ragged": True},
        # scoring a few held-out rows
        {"name": "distill eval", "op": "distill", "mode": "forward", "N": 48, "V": BIG, "K": 128,
         "tau": 1.0, "ragged": True},
        # storing the teacher's top logits of 4 x 1024 tokens
        {"name": "topk teacher", "op": "topk", "N": 4096, "V": BIG, "K": 64},
        # the same at the small GPT2 configuration (batch 4, 256 tokens)
        {"name": "topk small", "op": "topk", "N": 1024, "V": 1024, "K": 32},
        # beam search over a recurrent model: six states of one vector a beam
        {"name": "beam recurrent", "op": "beam", "B": 1, "W": 4, "V": 1024, "states": 6,
         "width": 256, "positions": 0, "length": 0, "finished": False},
        # beam search over K/V caches, filled to 700 of 1024 positions
        {"name": "beam caches", "op": "beam", "B": 8, "W": 8, "V": BIG, "states": 4, "width": 1024,
         "positions": 1024, "length": 700, "finished": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "distill", "topk", "beam"])
    if op == "recurrence":
        mode = rng.choice(["train", "train", "forward", "step"])
        per = rng.choice([1, 1, 8, 25, 32, 64])          # channels that share a gate
        heads = _log_uniform(rng, 1, max(1, 1024 // per)) if per > 1 else _log_uniform(rng, 16, 1024)
        D = per * heads
        if mode == "step":
            return {"op": op, "mode": mode, "B": _log_uniform(rng, 1, 256), "T": 1, "D": D,
                    "H": heads, "h0": True, "reset": False}
        T = _log_uniform(rng, 16, 16384)
        B = max(1, min(32, _log_uniform(rng, 1, 32), (1 << 24) // (T * D)))
        return {"op": op, "mode": mode, "B": B, "T": T, "D": D, "H": heads,
                "h0": rng.random() < 0.5, "reset": rng.random() < 0.5}
    if op == "distill":
        V = _log_uniform(rng, 200, BIG)
        return {"op": op, "mode": rng.choice(["train", "train", "forward"]), "V": V,
                "N": _log_uniform(rng, 1, max(1, min(4096, (1 << 26) // V))),
                "K": _log_uniform(rng, 1, 128), "tau": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "ragged": rng.random() < 0.5}
    if op == "topk":
        V = _log_uniform(rng, 200, BIG)
        return {"op": op, "V": V, "N": _log_uniform(rng, 1, max(1, min(4096, (1 << 26) // V))),
                "K": _log_uniform(rng, 1, 128)}
    caches = rng.random() < 0.5
    positions = _log_uniform(rng, 16, 512) if caches else 0
    return {"op": op, "B": _log_uniform(rng, 1, 8), "W": rng.randint(2, 12),
            "V": _log_uniform(rng, 200, BIG), "states": rng.randint(1, 6),
            "width": _log_uniform(rng, 16, 512), "positions": positions,
            "length": rng.randint(1, positions) if caches else 0,
            "finished": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs


def _inputs(case, seed):
    """The torch inputs of a case, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op = case["op"]
    if op == "recurrence":
        B, T, D, H = case["B"], case["T"], case["D"], case["H"]
        if case["mode"] == "step":
            return {"x": normal(B, D), "gate": normal(B, H) * 1.5 + 2.0, "state": normal(B, D)}
        d = {"x": normal(B, T, D),
             # forget gates biased towards keeping, as they are initialised
             "gate": normal(B, T, H) * 1.5 + 2.0,
             "h0": normal(B, D) if case["h0"] else None,
             # documents of about 400 tokens packed into a row
             "reset": (uniform(B, T) < 1 / 400).to(torch.int32) if case["reset"] else None}
        if case["mode"] == "train":
            d["dh"] = normal(B, T, D)
            d["dlast"] = normal(B, D) if case["h0"] else None
        return d
    if op == "distill":
        N, V, K = case["N"], case["V"], min(case["K"], case["V"])
        logits = normal(N, V) * 2.5
        # a teacher that the student partly agrees with
        top, ids = (logits + normal(N, V)).topk(K, dim=-1)
        if case["ragged"]:      # fewer stored logits in some rows, none in a few
            keep = (uniform(N, 1) * (K + 1) * 1.1).floor()
            top = torch.where(torch.arange(K, device="cuda") < keep, top, -math.inf)
        d = {"logits": logits, "top": top.contiguous(), "ids": ids.to(torch.int32).contiguous()}
        if case["mode"] == "train":      # the mean over the rows that are not padding
            d["grad"] = (uniform(N, 1) < 0.95).float() / N
        return d
    if op == "topk":
        return {"x": normal(case["N"], case["V"]) * 2.5}
    B, W = case["B"], case["W"]
    rows, P = B * W, case["positions"]
    shape = (rows, P, case["width"]) if P else (rows, case["width"])
    d = {"logits": normal(rows, case["V"]) * 3.0,
         "scores": -10.0 - 2.0 * uniform(B, W),
         "finished": (uniform(B, W) < 0.2).to(torch.int32) if case["finished"] else None,
         "length": torch.tensor([case["length"]], dtype=torch.int32, device="cuda") if P else None,
         "states": [normal(*shape) for _ in range(case["states"])]}
    return d


# ------------------------------------------------------------------ plain forms


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from a zero state, by doubling:
    after step k every position holds its last 2^k terms."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _spread(gate, D):
    """A gate per head as a gate per channel."""
    return gate if gate.shape[-1] == D else gate.repeat_interleave(D // gate.shape[-1], -1)


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _recurrence(s):
    x, h0, reset = s["x"], s["h0"], s["reset"]
    B, T, D = x.shape
    gate = _spread(s["gate"], D)
    a, z = _sigmoid(gate), _sigmoid(-gate)
    keep = a if reset is None else a * (reset == 0).unsqueeze(-1)
    b = z * x
    if h0 is not None:
        b = torch.cat([b[:, :1] + keep[:, :1] * h0.unsqueeze(1), b[:, 1:]], 1)
    h = _scan(keep, b)
    out = {"h": h, "h_last": h[:, -1]}
    if "dh" not in s:
        return out
    dh = s["dh"]
    if s["dlast"] is not None:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dlast"].unsqueeze(1)], 1)
    # the total gradient of h_t, from the last position back
    after = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    g = _scan(after.flip(1), dh.flip(1)).flip(1)
    first = torch.zeros_like(x[:, :1]) if h0 is None else h0.unsqueeze(1)
    before = torch.cat([first, h[:, :-1]], 1)
    if reset is not None:
        before = before * (reset == 0).unsqueeze(-1)
    dgate = g * (before - x) * (a * z)
    H = s["gate"].shape[-1]
    if H != D:
        dgate = dgate.reshape(B, T, H, D // H).sum(-1)
    out |= {"dx": g * z, "dgate": dgate}
    if h0 is not None:
        out["dh0"] = keep[:, 0] * g[:, 0]
    return out


def _step(s):
    gate = _spread(s["gate"], s["x"].shape[-1])
    s["state"].copy_(_sigmoid(gate) * s["state"] + _sigmoid(-gate) * s["x"])
    return {"state": s["state"]}


def _distill(s):
    tau, ids = s["tau"], s["ids"].long()
    z, t = s["logits"] / tau, s["top"] / tau
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    norm = e.sum(-1, keepdim=True)
    some = (t > -math.inf).any(-1, keepdim=True)
    t = t - torch.where(some, t.amax(-1, keepdim=True), 0.0)
    p = torch.exp(t)
    total = torch.where(some, p.sum(-1, keepdim=True), 1.0)
    p = p / total
    apart = (t - torch.log(total)) - (z.gather(1, ids) - torch.log(norm))
    loss = tau * tau * torch.where(p > 0, p * apart, 0.0).sum(-1, keepdim=True)
    if "grad" not in s:
        return {"loss": loss}
    q = torch.where(some, e / norm, 0.0).scatter_add(1, ids, -p)
    return {"loss": loss, "dlogits": q * (s["grad"] * tau)}


def _topk(s):
    values, ids = torch.sort(s["x"], dim=-1, descending=True, stable=True)
    return {"values": values[:, :s["K"]].contiguous(), "ids": ids[:, :s["K"]].to(torch.int32)}


def _beam(s):
    z, scores, done = s["logits"], s["scores"], s["finished"]
    B, W = scores.shape
    top = z.amax(-1, keepdim=True)
    norm = torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    best, token = torch.sort(z, dim=-1, descending=True, stable=True)
    best, token = best[:, :W], token[:, :W].reshape(B, W, W)
    new = scores.unsqueeze(-1) + ((best - top) - norm).reshape(B, W, W)
    if done is not None:
        # a finished beam is carried on by the stop token alone, at no cost
        ended = (done != 0).unsqueeze(-1)
        stay = torch.full_like(new, -math.inf)
        stay[:, :, 0] = scores
        new = torch.where(ended, stay, new)
        token = torch.where(ended, STOP, token)
    best, at = torch.sort(new.reshape(B, W * W), dim=-1, descending=True, stable=True)
    best, at = best[:, :W].contiguous(), at[:, :W]
    parents = at // W
    tokens = token.reshape(B, W * W).gather(1, at)
    out = {"scores": best, "parents": parents.to(torch.int32), "tokens": tokens.to(torch.int32)}
    if done is not None:
        out["finished"] = ((done.gather(1, parents) != 0) | (tokens == STOP)).to(torch.int32)
    rows = (parents + W * torch.arange(B, device=z.device).unsqueeze(1)).reshape(-1)
    for v in s["states"]:
        used = v if s["length"] is None else v[:, :s["used"]]
        used.copy_(used[rows])
    out["states"] = s["states"]
    return out


# ------------------------------------------------------------------ the framework's


class _Memory:
    """A torch tensor's memory as the storage of a framework tensor."""

    def __init__(self, t, uid):
        self.owner, self.ptr, self.size = t, t.data_ptr(), t.numel() * t.element_size()
        self.label, self.uid, self.version = "torch", uid, 0


def _lend(t):
    """A torch tensor as a framework tensor (whole numbers as u32)."""
    import wxx_b200 as wxx

    if t is None:
        return None
    return wxx.Tensor(tuple(t.shape), buffer=_Memory(t, -id(t)),
                      dtype="f32" if t.dtype == torch.float32 else "u32")


class _Outside:
    """A framework tensor's memory, described for torch."""

    def __init__(self, t):
        self.owner = t
        self.__cuda_array_interface__ = {
            "shape": tuple(t.shape), "typestr": "<f4" if t.type == "f32" else "<i4",
            "data": (t.ptr, False), "strides": None, "version": 3}


def _view(t):
    """A dense framework tensor as a torch tensor."""
    return torch.as_tensor(_Outside(t), device="cuda")


def _own_recurrence(s):
    from wxx_b200 import functional as F

    h, last = F.gated_recurrence(s["x"], s["gate"], s["h0"], s["reset"])
    out = {"h": _view(h), "h_last": _view(last)}
    if "dh" in s:
        dx, dgate, dh0 = F.gated_recurrence_backward(s["dh"], s["x"], s["gate"], h, s["h0"],
                                                     s["reset"], s["dlast"])
        out |= {"dx": _view(dx), "dgate": _view(dgate)}
        if dh0 is not None:
            out["dh0"] = _view(dh0)
    return out


def _own_distill(s):
    from wxx_b200 import functional as F

    loss, stats = F.distill_loss(s["logits"], s["top"], s["ids"], s["tau"])
    if "grad" not in s:
        return {"loss": _view(loss)}
    d = F.distill_loss_backward(s["grad"], s["logits"], s["top"], s["ids"], stats, s["tau"])
    return {"loss": _view(loss), "dlogits": _view(d)}


def _own_topk(s):
    from wxx_b200 import functional as F

    values, ids = F.topk(s["x"], s["K"])
    return {"values": _view(values), "ids": _view(ids)}


def _record(s, written, call):
    """Records ``call`` as a graph and puts what it writes in place back to what
    it was before the recording's own run."""
    import wxx_b200 as wxx

    before = [v.clone() for v in written]
    torch.cuda.synchronize()
    s["graph"] = wxx.graph.capture(call)
    wxx.backend.synchronize()
    torch._foreach_copy_(written, before)
    return s["graph"].output


def _own_step(s, torch_state):
    from wxx_b200 import functional as F

    _record(s, [torch_state],
            lambda: F.gated_recurrence_step(s["x"], s["gate"], s["state"]))
    s["out"] = {"state": torch_state}


def _own_beam(s, torch_states):
    from wxx_b200 import functional as F

    def call():
        picked = F.beam_select(s["logits"], s["scores"], s["finished"],
                               None if s["finished"] is None else STOP)
        F.beam_reorder(s["states"], picked[1], s["length"])
        return picked

    scores, parents, tokens, finished = _record(s, torch_states, call)
    s["out"] = {"scores": _view(scores), "parents": _view(parents), "tokens": _view(tokens),
                "states": torch_states}
    if finished is not None:
        s["out"]["finished"] = _view(finished)


def _replay(s):
    s["graph"].replay()
    return s["out"]


_PLAIN = {"recurrence": _recurrence, "step": _step, "distill": _distill, "topk": _topk,
          "beam": _beam}
_OWN = {"recurrence": _own_recurrence, "step": _replay, "distill": _own_distill,
        "topk": _own_topk, "beam": _replay}


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = "step" if case.get("mode") == "step" else case["op"]
    s["kind"] = kind
    s["tau"], s["K"] = case.get("tau"), min(case.get("K", 1), case.get("V", 1))
    s["used"] = case.get("length")
    if not own:
        return s
    held = {k: v for k, v in s.items() if isinstance(v, (torch.Tensor, list))}
    torch.cuda.synchronize()      # the framework's stream is another than torch's
    for k, v in held.items():
        s[k] = [_lend(t) for t in v] if isinstance(v, list) else _lend(v)
    if kind == "step":
        _own_step(s, held["state"])
    elif kind == "beam":
        _own_beam(s, held["states"])
    return s


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def work(case):
    op = case["op"]
    if op == "recurrence":
        E, G = case["B"] * case["T"] * case["D"], case["B"] * case["T"] * case["H"]
        BD = case["B"] * case["D"]
        if case["mode"] == "step":
            return {"bytes": 4 * (3 * E + G), "flops": 3 * E + 6 * G}
        n = 2 * E + G + BD * (2 if case["h0"] else 1)            # x, h, gate, h_last, h0
        n += case["B"] * case["T"] if case["reset"] else 0
        if case["mode"] == "forward":
            return {"bytes": 4 * n, "flops": 3 * E + 6 * G}
        n += 2 * E + G + (2 * BD if case["h0"] else 0)           # dh, dx, dgate, dlast, dh0
        return {"bytes": 4 * n, "flops": 10 * E + 10 * G}
    if op == "distill":
        E, K = case["N"] * case["V"], case["N"] * min(case["K"], case["V"])
        if case["mode"] == "forward":
            return {"bytes": 4 * (E + 2 * K + case["N"]), "flops": 4 * E + 10 * K}
        return {"bytes": 4 * (2 * E + 2 * K + 2 * case["N"]), "flops": 8 * E + 12 * K}
    if op == "topk":
        return {"bytes": 4 * (case["N"] * case["V"] + 2 * case["N"] * min(case["K"], case["V"])),
                "flops": case["N"] * case["V"]}
    B, W = case["B"], case["W"]
    row = case["width"] * (case["length"] if case["positions"] else 1) * case["states"]
    # a beam that is its own parent stays where it is, a parent is read once:
    # the expected numbers of both for parents drawn evenly
    moved = (1 - 1 / W) * W + W * (1 - (1 - 1 / W) ** W)
    return {"bytes": 4 * (B * W * case["V"] + 6 * B * W + B * moved * row),
            "flops": 4 * B * W * case["V"]}


# ------------------------------------------------------------------ 64 bits


def _exact_recurrence(d, D):
    """One position after the other, from the definition."""
    x, gate = d["x"].double(), d["gate"].double()
    B, T, H = gate.shape
    wide = gate.unsqueeze(-1).expand(B, T, H, D // H).reshape(B, T, D)
    a, one_minus_a = torch.sigmoid(wide), torch.sigmoid(-wide)
    zero = torch.zeros(B, D, dtype=torch.float64, device=x.device)
    start = zero if d["h0"] is None else d["h0"].double()
    carried = None if d["reset"] is None else (d["reset"] == 0).double().unsqueeze(-1)
    h, prev = torch.empty_like(x), torch.empty_like(x)
    now = start
    for t in range(T):
        if carried is not None:
            now = now * carried[:, t]
        prev[:, t] = now
        now = torch.addcmul(one_minus_a[:, t] * x[:, t], a[:, t], now)
        h[:, t] = now
    out = {"h": h, "h_last": now}
    if "dh" not in d:
        return out
    dh, dx, da = d["dh"].double(), torch.empty_like(x), torch.empty_like(x)
    back = zero if d["dlast"] is None else d["dlast"].double()
    for t in range(T - 1, -1, -1):
        total = dh[:, t] + back
        dx[:, t] = total * one_minus_a[:, t]
        da[:, t] = total * (prev[:, t] - x[:, t])
        back = total * a[:, t]
        if carried is not None:
            back = back * carried[:, t]
    out["dx"] = dx
    out["dgate"] = (da * a * one_minus_a).reshape(B, T, H, D // H).sum(-1)
    if d["h0"] is not None:
        out["dh0"] = back
    return out


def _exact_distill(d, tau):
    """Row by row blocks, with the library's 64-bit log-softmax."""
    losses, grads = [], []
    for i in range(0, d["logits"].shape[0], 512):
        top = d["top"][i:i + 512].double() / tau
        ids = d["ids"][i:i + 512].long()
        logq = torch.log_softmax(d["logits"][i:i + 512].double() / tau, -1)
        empty = torch.isinf(top).all(-1, keepdim=True)
        logp = torch.log_softmax(torch.where(empty, 0.0, top), -1)
        p = torch.where(empty, 0.0, logp.exp())
        terms = torch.where(p > 0, p * (logp - logq.gather(1, ids)), 0.0)
        losses.append(tau ** 2 * terms.sum(-1, keepdim=True))
        if "grad" in d:
            target = torch.zeros_like(logq).scatter_add_(1, ids, p)
            q = torch.where(empty, 0.0, logq.exp())
            grads.append(tau * d["grad"][i:i + 512].double() * (q - target))
    out = {"loss": torch.cat(losses)}
    if grads:
        out["dlogits"] = torch.cat(grads)
    return out


def _exact_beam(case, d):
    """The search written out on the host."""
    B, W = d["scores"].shape
    logp = torch.log_softmax(d["logits"].double(), -1)
    best, token = (v.cpu().numpy() for v in torch.topk(logp, min(2 * W, logp.shape[1]), -1))
    scores = d["scores"].double().cpu().numpy()
    done = None if d["finished"] is None else d["finished"].cpu().numpy()
    new, rows = np.zeros((B, W)), []
    for b in range(B):
        found = []
        for w in range(W):
            if done is not None and done[b, w]:
                found.append((scores[b, w], w))
            else:
                found += [(scores[b, w] + v, w) for v in best[b * W + w][:W]]
        found.sort(key=lambda c: (-c[0], c[1]))
        new[b] = [c[0] for c in found[:W]]
        rows += [b * W + c[1] for c in found[:W]]
    at = torch.tensor(rows, device=logp.device)
    used = case["length"] if case["positions"] else None
    states = []
    for v in d["states"]:
        moved = v.clone()
        if used is None:
            moved[:] = v[at]
        else:
            moved[:, :used] = v[at, :used]
        states.append(moved)
    return {"scores": torch.from_numpy(new), "parents": None, "tokens": None, "states": states}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "recurrence":
        if case["mode"] == "step":
            gate = d["gate"].double()
            gate = gate.unsqueeze(-1).expand(*gate.shape, case["D"] // case["H"])
            gate = gate.reshape(case["B"], case["D"])
            return {"state": torch.lerp(d["state"].double(), d["x"].double(),
                                        torch.sigmoid(-gate))}
        return _exact_recurrence(d, case["D"])
    if case["op"] == "distill":
        return _exact_distill(d, float(case["tau"]))
    if case["op"] == "topk":
        values, ids = torch.topk(d["x"].double(), min(case["K"], case["V"]), -1)
        return {"values": values, "ids": None}
    return _exact_beam(case, d)
