"""A language model whose sequence mixer is the gated linear recurrence or a
retention (no reference counterpart): training runs the mixer over whole
sequences, decoding keeps one vector (a retention: one matrix a head) per layer
and sequence, so a token costs the same at any length.  Blocks, initialisation
and parameter names follow ``nn/gpt.py``.
"""

import numpy as np

from .. import autograd, functional
from ..Tensor import Tensor
from ..backend import context
from .module import (
    GELU,
    Embedding,
    GroupNorm,
    LayerNorm,
    Linear,
    Module,
    ModuleList,
    Sequential,
    TiedLinear,
    kmajor_weight,
)


class GatedRecurrence(Module):
    """``out(h * gelu(mix(x)))`` with ``h`` the gated recurrence of ``value(x)``
    under the gates ``gate(x)``: a gate per head of d_model / n_heads channels
    (n_heads = d_model: per channel).  The gates' biases start between 0 and 5,
    memories of about 2 to 150 tokens."""

    def __init__(self, d_model, n_heads=None):
        super().__init__()
        n_heads = d_model if n_heads is None else int(n_heads)
        if n_heads < 1 or d_model % n_heads:
            raise ValueError(f"{d_model} channels cannot be split over {n_heads} gates")
        self.d_model = d_model
        self.n_heads = n_heads
        self.value = Linear(d_model, d_model, bias=False)
        self.mix = Linear(d_model, d_model, bias=False)
        self.gate = Linear(d_model, n_heads)
        self.out = Linear(d_model, d_model, bias=False)
        functional.assign(self.gate.bias, functional.from_numpy(
            np.linspace(0.0, 5.0, n_heads, dtype=np.float32)))

    def forward(self, x, reset=None, state=None):
        """``x`` (batch, time, d_model); ``reset`` (batch, time) u32 marks document
        starts.  ``state`` (batch, d_model; inference): the state before
        position 0, replaced by the one after the last."""
        v, g, m = self.value(x), self.gate(x), self.mix(x)
        if context.MODE != 0:
            h, last = functional.gated_recurrence(v, g, state, reset)
            if state is not None:
                functional.assign(state, last)
        else:
            if state is not None:
                raise RuntimeError("a state is carried under inference mode only")
            h = autograd.gated_recurrence(v, g).forward(v, g, None, reset)
        return self.out(h * m.gelu())

    def decode(self, x, state, residual, ln):
        """One position per sequence (inference): ``residual + out(...)`` of
        ``ln(x)``, x (batch, d_model), with ``state`` advanced in place."""
        D = self.d_model
        rnd = functional.get_matmul_mode() == "tf32"
        w = kmajor_weight(self, "_value_mix_t", [self.value, self.mix], rnd)
        vm = functional.ln_linear(x, ln.weightg, ln.weightb, w)
        g = functional.ln_linear(x, ln.weightg, ln.weightb,
                                 kmajor_weight(self, "_gate_t", [self.gate], rnd), self.gate.bias)
        h = functional.gated_recurrence_step(vm.narrow(1, 0, D), g, state)
        y = functional.pointwise(h, functional.gelu(functional.contiguous(vm.narrow(1, D, D))), 2)
        return functional.linear(y, kmajor_weight(self, "_out_t", [self.out], rnd),
                                 residual=residual, transpose_weight=True)


class Retention(Module):
    """``out(group_norm(o) * silu(gate(x)))`` with ``o`` the linear attention of the rotated
    queries and keys over the values, a decay for each head: memories of 2^3 tokens in the
    first head to 2^9 in the last.  A group of the norm is a head.  The decays and the
    rotary frequencies are constants of the module."""

    def __init__(self, d_model, n_heads, base=10000.0):
        super().__init__()
        n_heads = int(n_heads)
        if n_heads < 1 or d_model % n_heads or d_model // n_heads % 2 or d_model > 256 * n_heads:
            raise ValueError(f"{d_model} channels cannot be split over {n_heads} heads of an even "
                             "number of them, 256 at most")
        self.d_model = d_model
        self.n_heads = n_heads
        self.head_dim = d_model // n_heads
        self.q = Linear(d_model, d_model, bias=False)
        self.k = Linear(d_model, d_model, bias=False)
        self.v = Linear(d_model, d_model, bias=False)
        self.gate = Linear(d_model, d_model, bias=False)
        self.norm = GroupNorm(n_heads, d_model, activation="silu")
        self.out = Linear(d_model, d_model, bias=False)
        self.scale = self.head_dim ** -0.5
        self.frequencies = functional.rotary_frequencies(self.head_dim, base=base)
        self.log_decay = functional.from_numpy(
            np.log1p(-1 / 2.0 ** np.linspace(3, 9, n_heads)).astype(np.float32))

    def new_state(self, batch):
        return Tensor((batch, self.n_heads, self.head_dim, self.head_dim), value=0.0)

    def forward(self, x, reset=None, state=None, offset=0):
        """``x`` (batch, time, d_model); ``reset`` (batch, time) u32 marks document
        starts.  ``state`` (batch, heads, head_dim, head_dim; inference): the state before
        position 0, replaced by the one after the last; ``offset`` the positions before
        it."""
        def turned(t):
            return autograd.rotary(t).forward(t, self.n_heads, self.frequencies, None, offset)

        q, k, v = turned(self.q(x)), turned(self.k(x)), self.v(x)
        if context.MODE != 0:
            o, last = functional.linear_attention(q, k, v, self.log_decay, state, reset, self.scale)
            if state is not None:
                functional.assign(state, last)
        else:
            if state is not None:
                raise RuntimeError("a state is carried under inference mode only")
            o = autograd.linear_attention(q, k, v).forward(q, k, v, self.log_decay, None, reset,
                                                           self.scale)
        rows = (x.shape[0] * x.shape[1], self.d_model)
        y = self.norm.forward(o.reshape(rows), self.gate(x).reshape(rows))
        return self.out(y.reshape(tuple(x.shape)))

    def decode(self, x, state, residual, ln, positions):
        """One position per sequence (inference): ``residual + out(...)`` of
        ``ln(x)``, x (batch, d_model), with ``state`` advanced in place; ``positions`` (1) or
        (batch, 1) u32: the positions before it."""
        D, B = self.d_model, x.shape[0]
        rnd = functional.get_matmul_mode() == "tf32"
        w = kmajor_weight(self, "_qkvg_t", [self.q, self.k, self.v, self.gate], rnd)
        qkvg = functional.ln_linear(x, ln.weightg, ln.weightb, w)
        qk = functional.rotary(qkvg.narrow(1, 0, 2 * D).unsqueeze(1), 2 * self.n_heads,
                               self.frequencies, positions).reshape((B, 2 * D))
        o = functional.linear_attention_step(qk.narrow(1, 0, D), qk.narrow(1, D, D),
                                             qkvg.narrow(1, 2 * D, D), self.log_decay, state,
                                             self.scale)
        y = functional.group_norm(o, self.n_heads, self.norm.weight, self.norm.bias, "silu",
                                  qkvg.narrow(1, 3 * D, D), self.norm.eps)[0]
        return functional.linear(y, kmajor_weight(self, "_out_t", [self.out], rnd),
                                 residual=residual, transpose_weight=True)


class RecurrentBlock(Module):
    """Pre-LN block: gated recurrence or retention + GELU MLP."""

    def __init__(self, d_model, n_heads=None, mixer="gated"):
        super().__init__()
        if mixer not in ("gated", "retention"):
            raise ValueError(f"mixer must be 'gated' or 'retention', got {mixer!r}")
        if mixer == "retention" and n_heads is None:
            raise ValueError("a retention needs its number of heads")
        self.ln1 = LayerNorm(d_model)
        self.mixer = (Retention if mixer == "retention" else GatedRecurrence)(d_model, n_heads)
        self.ln2 = LayerNorm(d_model)
        self.mlp = Sequential(Linear(d_model, 4 * d_model), GELU(), Linear(4 * d_model, d_model))

    def forward(self, x, reset=None, state=None, offset=0):
        where = (offset,) if isinstance(self.mixer, Retention) else ()
        x = x + self.mixer.forward(self.ln1(x), reset, state, *where)
        return x + self.mlp(self.ln2(x))

    def decode(self, x, state, positions=None):
        """The block for one new position per sequence (inference); a retention needs
        the ``positions`` before it, (1) or (batch, 1) u32."""
        where = ()
        if isinstance(self.mixer, Retention):
            if positions is None:
                raise ValueError("a retention decodes with the positions before the new one")
            where = (positions,)
        h = self.mixer.decode(x, state, x, self.ln1, *where)
        fc1, _, fc2 = self.mlp._modules.values()
        rnd = functional.get_matmul_mode() == "tf32"
        u = functional.ln_linear(h, self.ln2.weightg, self.ln2.weightb,
                                 kmajor_weight(self, "_fc1_t", [fc1], rnd), fc1.bias,
                                 activation="gelu", feeds_tf32=True)
        return functional.linear(u, kmajor_weight(self, "_fc2_t", [fc2], rnd), fc2.bias,
                                 residual=h, transpose_weight=True)


class RecurrentLM(Module):
    """Embedding, ``n_layers`` recurrent blocks, final LayerNorm, (tied) head.
    ``mixer``: ``"gated"`` (the gated recurrence) or ``"retention"``."""

    def __init__(self, vocab_size, d_model=256, n_heads=None, n_layers=6, tie_weights=True,
                 mixer="gated"):
        super().__init__()
        self.vocab_size = vocab_size
        self.d_model = d_model
        self.tok_emb = Embedding(vocab_size, d_model, init_std=0.02)
        self.blocks = ModuleList([RecurrentBlock(d_model, n_heads, mixer)
                                  for _ in range(n_layers)])
        self.ln_f = LayerNorm(d_model)
        self.head = TiedLinear(self.tok_emb) if tie_weights else Linear(d_model, vocab_size,
                                                                          bias=False)
        for name, p in self.named_parameters():
            if len(p.shape) >= 2 and not name.endswith("tok_emb.weight"):
                functional.assign(p, functional.normal(0, 0.02, p.shape))

    def new_states(self, batch):
        """Zero states for ``batch`` sequences, one tensor a layer: (batch, d_model), of
        a retention (batch, heads, head_dim, head_dim)."""
        return [b.mixer.new_state(batch) if isinstance(b.mixer, Retention)
                else Tensor((batch, self.d_model), value=0.0) for b in self.blocks]

    def hidden(self, ids, reset=None, states=None, offset=0):
        """The final LayerNorm's output (batch, time, d_model)."""
        h = self.tok_emb(ids)
        for i, block in enumerate(self.blocks):
            h = block.forward(h, reset, None if states is None else states[i], offset)
        return self.ln_f(h)

    def forward(self, ids, reset=None, states=None, offset=0):
        """Logits (batch, time, vocab) of u32 ids; ``reset`` (batch, time) u32
        marks the first token of each document of a packed row; ``states``
        (inference) carries the sequences on from an earlier call, ``offset``
        tokens in all before (which a retention's positions need)."""
        return self.head(self.hidden(ids, reset, states, offset))

    def decode(self, tokens, states, positions=None):
        """Logits (batch, vocab) after one more token (batch, 1) per sequence
        (inference); the states advance in place.  ``positions`` (1) or (batch, 1)
        u32, read on the device: the tokens before it, which a retention needs."""
        h = self.tok_emb(tokens).reshape((tokens.shape[0], self.d_model))
        for block, state in zip(self.blocks, states):
            h = block.decode(h, state, positions)
        if hasattr(self.head, "forward_ln"):
            return self.head.forward_ln(h, self.ln_f)
        return self.head(self.ln_f(h))

    def beam_search(self, prompt, beams=4, max_new_tokens=64, stop_token=None, length_penalty=0.0):
        """Beam search from a u32 prompt (see ``nn.generation.beam_search``)."""
        from .generation import beam_search

        return beam_search(self, prompt, beams=beams, max_new_tokens=max_new_tokens,
                           stop_token=stop_token, length_penalty=length_penalty)


__all__ = ["GatedRecurrence", "RecurrentBlock", "RecurrentLM", "Retention"]
