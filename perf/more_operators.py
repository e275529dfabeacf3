"""Operators of a retention mixer, as measured cases.

A retention layer turns its queries and keys by their positions, mixes the
sequence by linear attention with a decay for each head, and normalises every
head's output under a gate.  The three operators, each in a plain form
(elementary torch operations in 32 bits, angles in 64) and, with ``own`` set,
through the framework's public entry points:

* ``rotary``: rotary positions, ``y_i = m (x_i cos - x_j sin)``, ``y_j = m (x_i
  sin + x_j cos)`` for the pairs (i, j) of a head's first channels, the pair's
  halves apart or next to each other, with frequencies scaled for long contexts;
  forward, and forward and backward;
* ``linear``: linear attention with a decay for each head, ``S_t = lambda S_{t-1}
  + k_t v_t^T`` (the state taken as 0 where a new document starts), ``o_t = scale
  S_t^T q_t``, forward, forward and backward, and one token at a time;
* ``norm``: group norm over the trailing channels with an activation, of the
  result or of a gate that multiplies it; forward, and forward and backward.

The framework's tensors are lent the memory of the torch inputs, and its
outputs are viewed as torch tensors, without copies.  The per-token calls are
recorded as a CUDA graph and replayed, which is how the framework's generation
runs its steps; the others are direct calls.
"""

import math

import numpy as np
import torch

own = False

EPS = 1e-5
ORIGINAL = 2048      # length that scaled frequencies were made for


def listed():
    return [
        # training: queries and keys (32 heads in one tensor) of 8 x 1024 tokens at the
        # GPT2-scaled width
        {"name": "rotary train", "op": "rotary", "mode": "train", "B": 8, "T": 1024, "H": 32,
         "d": 64, "r": 64, "layout": "half", "scaling": "none", "factor": 1.0, "far": 0},
        # prefill of a ragged batch far into a long context, part of each odd-sized head
        {"name": "rotary prefill far", "op": "rotary", "mode": "forward", "B": 3, "T": 4097,
         "H": 10, "d": 50, "r": 24, "layout": "interleaved", "scaling": "yarn", "factor": 16.0,
         "far": 1000000},
        # one decode step of 32 sequences, each at its own position
        {"name": "rotary step", "op": "rotary", "mode": "step", "B": 32, "T": 1, "H": 32, "d": 64,
         "r": 64, "layout": "half", "scaling": "linear", "factor": 4.0, "far": 30000},
        # training at the GPT2-scaled width
        {"name": "linear train", "op": "linear", "mode": "train", "B": 8, "T": 1024, "H": 16,
         "dk": 64, "dv": 64, "h0": False, "reset": False},
        # training on long documents packed into rows of 8192 tokens (the Hyena
        # benchmark's batch, length and width)
        {"name": "linear train long", "op": "linear", "mode": "train", "B": 16, "T": 8192, "H": 4,
         "dk": 64, "dv": 64, "h0": False, "reset": True},
        # prefill of one long document at the small GPT2's heads
        {"name": "linear prefill one", "op": "linear", "mode": "forward", "B": 1, "T": 65536,
         "H": 8, "dk": 32, "dv": 32, "h0": False, "reset": False},
        # prefill of a ragged batch that carries a state on, odd heads
        {"name": "linear prefill odd", "op": "linear", "mode": "forward", "B": 3, "T": 4097,
         "H": 5, "dk": 40, "dv": 72, "h0": True, "reset": False},
        # one decode step of 32 sequences
        {"name": "linear step", "op": "linear", "mode": "step", "B": 32, "T": 1, "H": 16,
         "dk": 64, "dv": 64, "h0": True, "reset": False},
        # training: every head of 8 x 1024 tokens by itself, under a gate
        {"name": "norm train gated", "op": "norm", "mode": "train", "N": 8192, "S": 1, "C": 1024,
         "G": 16, "activation": "silu", "gated": True},
        # training on feature maps of the ResNet's first stage
        {"name": "norm train images", "op": "norm", "mode": "train", "N": 128, "S": 1024, "C": 64,
         "G": 32, "activation": "silu", "gated": False},
        # an odd map, channels that no vector width divides
        {"name": "norm odd", "op": "norm", "mode": "forward", "N": 37, "S": 63, "C": 330, "G": 10,
         "activation": "gelu", "gated": False},
        # one decode step of 32 sequences
        {"name": "norm step", "op": "norm", "mode": "step", "N": 32, "S": 1, "C": 1024, "G": 16,
         "activation": "silu", "gated": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "linear", "linear", "norm"])
    mode = rng.choice(["train", "train", "forward", "step"])
    if op == "rotary":
        d = rng.choice([24, 32, 50, 64, 80, 128])
        r = rng.choice([d, d, 2 * rng.randint(1, d // 2)])
        H = _log_uniform(rng, 1, 32)
        T = 1 if mode == "step" else _log_uniform(rng, 1, 16384)
        B = max(1, min(_log_uniform(rng, 1, 64), (1 << 24) // (T * H * d)))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": op, "mode": mode, "B": B, "T": T, "H": H, "d": d, "r": r,
                "layout": rng.choice(["half", "interleaved"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]),
                "far": rng.choice([0, 0, 5000, 1000000])}
    if op == "linear":
        dk, dv = rng.choice([(64, 64), (32, 32), (rng.randint(8, 128), rng.randint(8, 128))])
        H = _log_uniform(rng, 1, 16)
        T = 1 if mode == "step" else _log_uniform(rng, 1, 16384)
        wide = H * max(dk, dv)
        B = max(1, min(_log_uniform(rng, 1, 64), (1 << 23) // (T * wide)))
        return {"op": op, "mode": mode, "B": B, "T": T, "H": H, "dk": dk, "dv": dv,
                "h0": mode == "step" or rng.random() < 0.5,
                "reset": mode != "step" and rng.random() < 0.5}
    # groups of 16 numbers or more: over one or two a gradient is rounding alone
    S = 1 if mode == "step" or rng.random() < 0.5 else _log_uniform(rng, 16, 4096)
    per = _log_uniform(rng, 16 if S == 1 else 1, 128)
    G = _log_uniform(rng, 1, max(1, 1024 // per))
    most = 256 if mode == "step" else max(1, (1 << 23) // (S * G * per))
    gated = rng.random() < 0.5
    # a result of about 0 has no gradient that two roundings agree on where relu bends
    bends = ["relu"] if gated or mode != "train" else []
    return {"op": op, "mode": mode, "N": _log_uniform(rng, 1, min(most, 16384)), "S": S,
            "C": G * per, "G": G, "activation": rng.choice(["silu", "gelu"] + bends),
            "gated": gated}


# ------------------------------------------------------------------ inputs


def _inputs(case, seed):
    """The torch inputs of a case, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op, mode = case["op"], case["mode"]
    if op == "rotary":
        B, T, D = case["B"], case["T"], case["H"] * case["d"]
        # each row starts somewhere: a sequence's next position, or the documents of a
        # packed row
        start = (uniform(B, 1) * (case["far"] + 1)).to(torch.int32)
        d = {"x": normal(B, T, D), "positions": None}
        if case["far"]:
            d["positions"] = (start + torch.arange(T, device="cuda", dtype=torch.int32)).contiguous()
        if mode == "train":
            d["dy"] = normal(B, T, D)
        return d
    if op == "linear":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        # memories of 2^3 to 2^10 tokens, from the first head to the last
        memory = 2.0 ** torch.linspace(3, 10, H, device="cuda", dtype=torch.float64)
        d = {"q": normal(B, T, H * dk), "k": normal(B, T, H * dk), "v": normal(B, T, H * dv),
             "decay": torch.log1p(-1 / memory).float(),
             "h0": normal(B, H, dk, dv) if case["h0"] else None,
             # documents of about 400 tokens packed into a row
             "reset": (uniform(B, T) < 1 / 400).to(torch.int32) if case["reset"] else None}
        if mode == "train":
            d["do"] = normal(B, T, H * dv)
            d["dlast"] = normal(B, H, dk, dv) if case["h0"] else None
        if mode == "step":
            d["q"], d["k"], d["v"] = d["q"][:, 0], d["k"][:, 0], d["v"][:, 0]
        return d
    shape = (case["N"], case["C"]) if case["S"] == 1 else (case["N"], case["S"], case["C"])
    d = {"x": normal(*shape) * 2 + 0.5, "gamma": 1 + 0.2 * normal(case["C"]),
         "beta": 0.2 * normal(case["C"]), "gate": normal(*shape) if case["gated"] else None}
    if mode == "train":
        d["dy"] = normal(*shape)
    return d


# ------------------------------------------------------------------ plain forms


def _frequencies(case):
    """Angles per position of the pairs, and the factor on the turned channels."""
    r, s, base = case["r"], case["factor"], 10000.0
    if case["scaling"] == "ntk":
        base = base * s ** (r / (r - 2)) if r > 2 else base
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":
        turns = ORIGINAL * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * (keep + (1 - keep) / s), 0.1 * math.log(s) + 1
    return f, 1.0


def _turn(x, cos, sin, heads, r, layout):
    """The first r channels of every head turned; cos, sin (B or 1, T, r / 2)."""
    B, T, D = x.shape
    x = x.reshape(B, T, heads, D // heads)
    cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
    turned, rest = x[..., :r], x[..., r:]
    if layout == "half":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(turned.shape)
    return torch.cat([y, rest], -1).reshape(B, T, D)


def _rotary(s):
    x, r = s["x"], s["case"]["r"]
    positions = s["positions"]
    if positions is None:
        positions = torch.arange(x.shape[1], device=x.device).unsqueeze(0)
    f, m = s["frequencies"]
    angle = positions.double().unsqueeze(-1) * f
    cos, sin = (m * torch.cos(angle)).float(), (m * torch.sin(angle)).float()
    out = {"y": _turn(x, cos, sin, s["case"]["H"], r, s["case"]["layout"])}
    if "dy" in s:
        out["dx"] = _turn(s["dy"], cos, -sin, s["case"]["H"], r, s["case"]["layout"])
    return out


_CHUNK = 64


def _attend(q, k, v, decay, h0, cut, lag):
    """o_t = q_t^T S_t and the last state of S_t = lambda S_{t-1} + k_t v_t^T, over (B, H, T,
    d) and in chunks: what comes from a position of the same chunk by a masked
    product, what comes from earlier ones through the chunks' states.  `cut` (B, T)
    counts the document starts up to each position; h0 reaches position 0 through
    lambda^lag."""
    B, H, T, dk = q.shape
    dv, n = v.shape[-1], -(-T // _CHUNK)
    pad = n * _CHUNK - T
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).reshape(B, H, n, _CHUNK, t.shape[-1])
               for t in (q, k, v))
    cut = torch.cat([cut, cut[:, -1:].expand(B, pad)], 1).reshape(B, 1, n, _CHUNK)
    i = torch.arange(_CHUNK, device=q.device)
    g = decay.reshape(1, H, 1, 1)
    apart = (i.unsqueeze(1) - i).clamp(min=0)
    weight = torch.exp(g * apart).unsqueeze(2) * (i.unsqueeze(1) >= i)
    weight = weight * (cut.unsqueeze(-1) == cut.unsqueeze(-2))
    o = ((q @ k.transpose(-1, -2)) * weight) @ v
    # what every chunk adds to the state after its last position
    c = torch.arange(n, device=q.device)
    length = (T - c * _CHUNK).clamp(max=_CHUNK)
    end = cut[..., -1]                                          # (B, 1, n)
    left = (length.unsqueeze(1) - 1 - i).clamp(min=0)           # (n, chunk)
    keep = torch.exp(g * left) * (cut == end.unsqueeze(-1))
    added = ((k * keep.unsqueeze(-1)).transpose(-1, -2) @ v).reshape(B, H, n, dk * dv)
    # the state before every chunk, c = n for the one after the last
    at = torch.arange(n + 1, device=q.device)
    before = torch.cat([torch.zeros_like(end[..., :1]), end], -1)
    total = torch.cat([torch.zeros_like(length[:1]), length.cumsum(0)])
    passed = (total.unsqueeze(1) - total[1:]).clamp(min=0)      # positions after chunk j's end
    carry = torch.exp(g * passed) * (at.unsqueeze(1) > c)
    carry = carry * (before.unsqueeze(-1) == end.unsqueeze(-2))
    state = (carry @ added).reshape(B, H, n + 1, dk, dv)
    if h0 is not None:
        whole = torch.exp(g.squeeze(-1) * (total + (lag - 1))) * (before == 0)
        state = state + whole.reshape(B, H, n + 1, 1, 1) * h0.unsqueeze(2)
    reach = torch.exp(g * (i + 1)).expand(1, H, n, _CHUNK) * (cut == before[..., :n].unsqueeze(-1))
    o = o + reach.unsqueeze(-1) * (q @ state[:, :, :n])
    return o.reshape(B, H, n * _CHUNK, dv)[:, :, :T], state[:, :, n]


def _linear(s):
    case, scale = s["case"], s["scale"]
    B, T, H = case["B"], case["T"], case["H"]
    q, k, v = (s[n].reshape(B, T, H, -1).transpose(1, 2) for n in ("q", "k", "v"))
    marks = (torch.zeros(B, T, device=q.device, dtype=torch.int32) if s["reset"] is None
             else (s["reset"] != 0).int())
    cut = marks.cumsum(1)
    o, last = _attend(q * scale, k, v, s["decay"], s["h0"], cut, 1)
    out = {"o": o.transpose(1, 2).reshape(B, T, -1), "last": last}
    if "do" not in s:
        return out
    do = s["do"].reshape(B, T, H, -1).transpose(1, 2)
    h0 = None if s["h0"] is None else s["h0"].transpose(-1, -2)
    dq, _ = _attend(do * scale, v, k, s["decay"], h0, cut, 1)
    # backwards in time: a cut before a position is one after it, and the last state's
    # gradient reaches the last position undiminished
    back = torch.cat([torch.zeros_like(marks[:, :1]), marks[:, 1:].flip(1)], 1).cumsum(1)
    dlast = s["dlast"]
    turned = [t.flip(2) for t in (q * scale, k, v, do)]
    dv, first = _attend(turned[1], turned[0], turned[3], s["decay"], dlast, back, 0)
    dk, _ = _attend(turned[2], turned[3], turned[0], s["decay"],
                    None if dlast is None else dlast.transpose(-1, -2), back, 0)
    for name, t in (("dq", dq), ("dk", dk.flip(2)), ("dv", dv.flip(2))):
        out[name] = t.transpose(1, 2).reshape(B, T, -1)
    if s["h0"] is not None:
        kept = torch.exp(s["decay"]) * (marks[:, :1] == 0)
        out["dh0"] = first * kept.reshape(B, H, 1, 1)
    return out


def _linear_step(s):
    case = s["case"]
    B, H = case["B"], case["H"]
    q, k, v = (s[n].reshape(B, H, -1) for n in ("q", "k", "v"))
    state = s["h0"]
    state.mul_(torch.exp(s["decay"]).reshape(1, H, 1, 1))
    state.add_(k.unsqueeze(-1) * v.unsqueeze(-2))
    o = s["scale"] * (q.unsqueeze(-2) @ state).reshape(B, -1)
    return {"o": o, "state": state}


_GELU = 0.7978845608


def _act(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return 0.5 * x * (1 + torch.tanh(_GELU * (x + 0.044715 * x * x * x)))


def _slope(x, name):
    if name == "relu":
        return (x > 0).float()
    if name == "silu":
        p = 1 / (1 + torch.exp(-x))
        return p * (1 + x * (1 - p))
    t = torch.tanh(_GELU * (x + 0.044715 * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * _GELU * (1 + 3 * 0.044715 * x * x)


def _norm(s):
    case, act = s["case"], s["case"]["activation"]
    x, gate = s["x"], s["gate"]
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    wide = (N, S, G, C // G)
    z = x.reshape(wide)
    z = z - z.mean((1, 3), keepdim=True)
    inv = 1 / torch.sqrt((z * z).mean((1, 3), keepdim=True) + EPS)
    z = z * inv
    gamma = s["gamma"].reshape(G, -1)
    n = z * gamma + s["beta"].reshape(G, -1)
    y = _act(n, act) if gate is None else n * _act(gate.reshape(wide), act)
    out = {"y": y.reshape(x.shape)}
    if "dy" not in s:
        return out
    dy = s["dy"].reshape(wide)
    if gate is None:
        dn = dy * _slope(n, act)
    else:
        dn = dy * _act(gate.reshape(wide), act)
        out["dgate"] = (dy * n * _slope(gate.reshape(wide), act)).reshape(x.shape)
    dz = dn * gamma
    dx = inv * (dz - dz.mean((1, 3), keepdim=True) - z * (dz * z).mean((1, 3), keepdim=True))
    out |= {"dx": dx.reshape(x.shape), "dgamma": (dn * z).sum((0, 1)).reshape(-1),
            "dbeta": dn.sum((0, 1)).reshape(-1)}
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

    return wxx.Tensor(tuple(t.shape), buffer=_Memory(t, -id(t)), stride=t.stride(),
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


def _own_frequencies(case):
    from wxx_b200 import functional as F

    scaling = None if case["scaling"] == "none" else case["scaling"]
    return F.rotary_frequencies(case["r"], scaling=scaling, factor=case["factor"],
                                original_length=ORIGINAL)


def _own_rotary(s):
    from wxx_b200 import functional as F

    case = s["case"]
    y = F.rotary(s["x"], case["H"], s["frequencies"], s["positions"], layout=case["layout"])
    if "dy" not in s:
        return {"y": y}
    return {"y": y, "dx": F.rotary_backward(s["dy"], case["H"], s["frequencies"], s["positions"],
                                            layout=case["layout"])}


def _own_linear(s):
    from wxx_b200 import functional as F

    o, last = F.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["h0"], s["reset"],
                                 scale=s["scale"])
    out = {"o": o, "last": last}
    if "do" in s:
        grads = F.linear_attention_backward(s["do"], s["q"], s["k"], s["v"], s["decay"], s["h0"],
                                            s["reset"], s["dlast"], scale=s["scale"])
        out |= {n: t for n, t in zip(("dq", "dk", "dv", "dh0"), grads) if t is not None}
    return out


def _own_linear_step(s):
    from wxx_b200 import functional as F

    o = F.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["h0"], scale=s["scale"])
    return {"o": o, "state": s["h0"]}


def _own_norm(s):
    from wxx_b200 import functional as F

    case = s["case"]
    options = {"activation": case["activation"], "gate": s["gate"], "eps": EPS}
    y, mean, inv = F.group_norm(s["x"], case["G"], s["gamma"], s["beta"], **options)
    if "dy" not in s:
        return {"y": y}
    dx, dgamma, dbeta, dgate = F.group_norm_backward(s["dy"], s["x"], mean, inv, case["G"],
                                                     s["gamma"], s["beta"],
                                                     activation=case["activation"], gate=s["gate"])
    out = {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    return out if dgate is None else out | {"dgate": dgate}


_PLAIN = {"rotary": _rotary, "linear": _linear, "linear step": _linear_step, "norm": _norm}
_OWN = {"rotary": _own_rotary, "linear": _own_linear, "linear step": _own_linear_step,
        "norm": _own_norm}


def _kind(case):
    return "linear step" if case["op"] == "linear" and case["mode"] == "step" else case["op"]


def _record(s):
    """Records a decode step as a graph, and puts the state that it advances back to
    what it was before the recording's own run."""
    import wxx_b200 as wxx

    written = s["torch_state"]
    before = None if written is None else written.clone()
    torch.cuda.synchronize()
    s["graph"] = wxx.graph.capture(_OWN[s["kind"]], s)
    wxx.backend.synchronize()
    if before is not None:
        written.copy_(before)
    s["views"] = {k: written if v is s["h0"] else _view(v)
                  for k, v in s["graph"].output.items()}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["kind"], s["graph"] = case, _kind(case), None
    if case["op"] == "linear":
        s["scale"] = case["dk"] ** -0.5
    if not own:
        if case["op"] == "rotary":
            s["frequencies"] = _frequencies(case)
        return s
    s.setdefault("h0", None)
    s["torch_state"] = s["h0"] if case["mode"] == "step" else None
    held = {k: v for k, v in s.items() if isinstance(v, torch.Tensor) and k != "torch_state"}
    torch.cuda.synchronize()      # the framework's stream is another than torch's
    for k, v in held.items():
        s[k] = _lend(v)
    if case["op"] == "rotary":
        s["frequencies"] = _own_frequencies(case)
    if case["mode"] == "step":
        _record(s)
    return s


def run(state):
    if not own:
        return _PLAIN[state["kind"]](state)
    if state["graph"] is not None:
        state["graph"].replay()
        return state["views"]
    return {k: _view(v) for k, v in _OWN[state["kind"]](state).items()}


def work(case):
    op, train = case["op"], case["mode"] == "train"
    if op == "rotary":
        E = case["B"] * case["T"] * case["H"] * case["d"]
        turned = case["B"] * case["T"] * case["H"] * case["r"]
        P = case["B"] * case["T"] if case["far"] else 0
        return {"bytes": 4 * ((4 if train else 2) * E + P), "flops": (6 if train else 3) * turned}
    if op == "linear":
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        tokens, state = B * T * H, B * H * dk * dv
        if case["mode"] == "step":
            return {"bytes": 4 * (tokens * 2 * (dk + dv) + 2 * state), "flops": 5 * state}
        n = tokens * 2 * (dk + dv) + state * (2 if case["h0"] else 1)
        n += B * T if case["reset"] else 0
        # a position's least: its step of the state and its product with it
        flops = 4 * tokens * dk * dv
        if train:
            # do read, dq, dk, dv written, the states' gradients
            n += tokens * (2 * dk + 2 * dv) + (2 * state if case["h0"] else 0)
            flops *= 3
        return {"bytes": 4 * n, "flops": flops}
    E = case["N"] * case["S"] * case["C"]
    n = E * (3 if case["gated"] else 2)
    if train:
        n += E * (3 if case["gated"] else 2)      # dy read, dx and dgate written
    return {"bytes": 4 * (n + (4 if train else 2) * case["C"]), "flops": (30 if train else 12) * E}


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    d = _inputs(case, seed)
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
            for k, v in d.items()}

    def rotary():
        """Every pair as a complex number, turned by its angle on the host's table."""
        B, T, H, dim, r = (case[k] for k in ("B", "T", "H", "d", "r"))
        i = np.arange(r // 2, dtype=np.float64)
        s, base = case["factor"], 1e4
        if case["scaling"] == "ntk" and r > 2:
            base *= s ** (r / (r - 2))
        rate, gain = np.exp(-2 * i / r * np.log(base)), 1.0
        if case["scaling"] == "linear":
            rate = rate / s
        elif case["scaling"] == "yarn":
            mix = np.clip((ORIGINAL * rate / (2 * np.pi) - 1) / 31, 0, 1)
            rate, gain = (1 - mix) * rate / s + mix * rate, 1 + 0.1 * np.log(s)
        p = d["positions"]
        p = np.arange(T)[None] if p is None else p.cpu().numpy()
        turn = torch.from_numpy(gain * np.exp(1j * (p[..., None] * rate))).to("cuda").unsqueeze(2)
        apart = case["layout"] == "half"

        def turned(x, by):
            x = x.reshape(B, T, H, dim).clone()
            pairs = x[..., :r].reshape(B, T, H, 2, r // 2).transpose(-1, -2) if apart else \
                x[..., :r].reshape(B, T, H, r // 2, 2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
            x[..., :r] = (z.transpose(-1, -2) if apart else z).reshape(B, T, H, r)
            return x.reshape(B, T, H * dim)

        out = {"y": turned(wide["x"], turn)}
        if "dy" in wide:
            out["dx"] = turned(wide["dy"], turn.conj())
        return out

    def linear():
        """One position after the other, from the definition."""
        B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
        scale = dk ** -0.5
        lam = wide["decay"].exp().reshape(1, H, 1, 1)
        first = wide["h0"]
        if first is None:
            first = torch.zeros(B, H, dk, dv, dtype=torch.float64, device="cuda")
        q, k, v = (wide[n].reshape(B, T, H, -1) for n in ("q", "k", "v"))
        step = lam.expand(B, H, 1, 1)
        steps = None
        if d["reset"] is not None:
            steps = (d["reset"] == 0).double().reshape(B, T, 1, 1, 1) * lam.unsqueeze(1)
        do = wide["do"].reshape(B, T, H, dv) if "do" in wide else None
        S, o = first, torch.empty(B, T, H, dv, dtype=torch.float64, device="cuda")
        dq, dkey, dval = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        for t in range(T):
            S = (step if steps is None else steps[:, t]) * S
            S = torch.baddbmm(S.reshape(B * H, dk, dv), k[:, t].reshape(B * H, dk, 1),
                              v[:, t].reshape(B * H, 1, dv)).reshape(B, H, dk, dv)
            o[:, t] = scale * (q[:, t].unsqueeze(-2) @ S).squeeze(-2)
            if do is not None:
                dq[:, t] = scale * (S @ do[:, t].unsqueeze(-1)).squeeze(-1)
        if case["mode"] == "step":
            return {"o": o.reshape(B, H * dv), "state": S}
        out = {"o": o.reshape(B, T, H * dv), "last": S}
        if do is None:
            return out
        R = torch.zeros_like(S) if wide["dlast"] is None else wide["dlast"]
        for t in range(T - 1, -1, -1):
            R = torch.baddbmm(R.reshape(B * H, dk, dv), scale * q[:, t].reshape(B * H, dk, 1),
                              do[:, t].reshape(B * H, 1, dv)).reshape(B, H, dk, dv)
            dkey[:, t] = (R @ v[:, t].unsqueeze(-1)).squeeze(-1)
            dval[:, t] = (k[:, t].unsqueeze(-2) @ R).squeeze(-2)
            R = (step if steps is None else steps[:, t]) * R
        out |= {"dq": dq.reshape(B, T, H * dk), "dk": dkey.reshape(B, T, H * dk),
                "dv": dval.reshape(B, T, H * dv)}
        return out if wide["h0"] is None else out | {"dh0": R}

    def norm():
        """The library's 64-bit normalisation and activations, differentiated."""
        N, S, C = case["N"], case["S"], case["C"]
        acts = {"relu": torch.relu, "silu": torch.nn.functional.silu,
                "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}
        names = ["x", "gamma", "beta"] + (["gate"] if case["gated"] else [])
        leaves = {n: wide[n].requires_grad_("dy" in wide) for n in names}
        x = leaves["x"].reshape(N, S, C).transpose(1, 2)
        n = torch.nn.functional.group_norm(x, case["G"], leaves["gamma"], leaves["beta"], EPS)
        n = n.transpose(1, 2).reshape(d["x"].shape)
        act = acts[case["activation"]]
        y = n * act(leaves["gate"]) if case["gated"] else act(n)
        out = {"y": y.detach()}
        if "dy" in wide:
            grads = torch.autograd.grad(y, list(leaves.values()), wide["dy"])
            out |= {"d" + n: g for n, g in zip(names, grads)}
        return out

    return {"rotary": rotary, "linear": linear, "norm": norm}[case["op"]]()
