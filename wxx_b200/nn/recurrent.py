"""A language model whose sequence mixer is the gated linear recurrence (no
reference counterpart): training runs the scan over whole sequences, decoding
keeps one vector per layer and sequence, so a token costs the same at any
length.  Blocks, initialisation and parameter names follow ``nn/gpt.py``.
"""

import numpy as np

from .. import autograd, functional
from ..Tensor import Tensor
from ..backend import context
from .module import (
    GELU,
    Embedding,
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


class RecurrentBlock(Module):
    """Pre-LN block: gated recurrence + GELU MLP."""

    def __init__(self, d_model, n_heads=None):
        super().__init__()
        self.ln1 = LayerNorm(d_model)
        self.mixer = GatedRecurrence(d_model, n_heads)
        self.ln2 = LayerNorm(d_model)
        self.mlp = Sequential(Linear(d_model, 4 * d_model), GELU(), Linear(4 * d_model, d_model))

    def forward(self, x, reset=None, state=None):
        x = x + self.mixer.forward(self.ln1(x), reset, state)
        return x + self.mlp(self.ln2(x))

    def decode(self, x, state):
        """The block for one new position per sequence (inference)."""
        h = self.mixer.decode(x, state, x, self.ln1)
        fc1, _, fc2 = self.mlp._modules.values()
        rnd = functional.get_matmul_mode() == "tf32"
        u = functional.ln_linear(h, self.ln2.weightg, self.ln2.weightb,
                                 kmajor_weight(self, "_fc1_t", [fc1], rnd), fc1.bias,
                                 activation="gelu", feeds_tf32=True)
        return functional.linear(u, kmajor_weight(self, "_fc2_t", [fc2], rnd), fc2.bias,
                                 residual=h, transpose_weight=True)


class RecurrentLM(Module):
    """Embedding, ``n_layers`` recurrent blocks, final LayerNorm, (tied) head."""

    def __init__(self, vocab_size, d_model=256, n_heads=None, n_layers=6, tie_weights=True):
        super().__init__()
        self.vocab_size = vocab_size
        self.d_model = d_model
        self.tok_emb = Embedding(vocab_size, d_model, init_std=0.02)
        self.blocks = ModuleList([RecurrentBlock(d_model, n_heads) for _ in range(n_layers)])
        self.ln_f = LayerNorm(d_model)
        self.head = TiedLinear(self.tok_emb) if tie_weights else Linear(d_model, vocab_size,
                                                                          bias=False)
        for name, p in self.named_parameters():
            if len(p.shape) >= 2 and not name.endswith("tok_emb.weight"):
                functional.assign(p, functional.normal(0, 0.02, p.shape))

    def new_states(self, batch):
        """Zero states for ``batch`` sequences: one (batch, d_model) tensor a layer."""
        return [Tensor((batch, self.d_model), value=0.0) for _ in self.blocks]

    def hidden(self, ids, reset=None, states=None):
        """The final LayerNorm's output (batch, time, d_model)."""
        h = self.tok_emb(ids)
        for i, block in enumerate(self.blocks):
            h = block.forward(h, reset, None if states is None else states[i])
        return self.ln_f(h)

    def forward(self, ids, reset=None, states=None):
        """Logits (batch, time, vocab) of u32 ids; ``reset`` (batch, time) u32
        marks the first token of each document of a packed row; ``states``
        (inference) carries the sequences on from an earlier call."""
        return self.head(self.hidden(ids, reset, states))

    def decode(self, tokens, states):
        """Logits (batch, vocab) after one more token (batch, 1) per sequence
        (inference); the states advance in place."""
        h = self.tok_emb(tokens).reshape((tokens.shape[0], self.d_model))
        for block, state in zip(self.blocks, states):
            h = block.decode(h, state)
        if hasattr(self.head, "forward_ln"):
            return self.head.forward_ln(h, self.ln_f)
        return self.head(self.ln_f(h))

    def beam_search(self, prompt, beams=4, max_new_tokens=64, stop_token=None, length_penalty=0.0):
        """Beam search from a u32 prompt (see ``nn.generation.beam_search``)."""
        from .generation import beam_search

        return beam_search(self, prompt, beams=beams, max_new_tokens=max_new_tokens,
                           stop_token=stop_token, length_penalty=length_penalty)


__all__ = ["GatedRecurrence", "RecurrentBlock", "RecurrentLM"]
