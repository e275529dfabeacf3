"""On-device autoregressive generation for GPT2 (interface: src/wxx/nn/gpt.py
``GPT2.generate``, lines 108-170 of the reference).

The reference samples one token per step by re-running the forward over the
whole prefix and copying the (batch, seq, vocab) logits to the host.  Here:

1. prefill: one forward over the prompt under inference mode fills per-layer
   K / V caches of shape (batch, max_len, d_model) and runs the LM head on the
   last position only;
2. every later token is a decode step over the newest position only
   (``GPT2Block.decode``): embedding, per-layer LayerNorm / QKV GEMM / cached
   attention / out projection / MLP, final LayerNorm, LM head, sampler;
3. the token count lives in device memory, so the decode step is the same
   launch sequence every time: it is recorded once as a CUDA graph and
   replayed; the sampler writes the id into the device token buffer and
   advances the count.

The sampler (``wxx_sample_tokens``) follows the reference's rule: temperature 0
takes the first index of the maximum; otherwise logits / temperature in
float64, top-k masking (values below the k-th largest dropped), softmax, and the
first index whose cumulative probability exceeds the row's uniform draw.  The
draws come from the caller's numpy generator, one ``rng.random((batch, 1))``
per step as in the reference, so equal seeds give equal samples.

The host reads the ids back once at the end, or one column per step when a
``stop_token`` is given (to stop when every row has emitted it).
"""

import numpy as np

from ..Tensor import Tensor
from ..backend import context
from ..backend import device as _dev
from ..backend.lib import F, check


class _DecodeState:
    """Device buffers of one generation call: token ids (batch, max_len),
    the token count, the sampler's counter, the draws and the K / V caches."""

    def __init__(self, model, batch):
        D = model.tok_emb.embedding_dim
        L = model.max_len
        self.batch = batch
        self.ids = Tensor._empty([batch, L], "u32")
        self.cur_len = Tensor._empty([1], "u32")      # read as an int on the device
        self.done = Tensor._empty([1], "u32")
        zero = np.zeros(1, np.uint32)
        check(F.wxx_memcpy_h2d(self.done.ptr, zero.ctypes.data, 4), "clear counter")
        self.draws = _dev.DeviceBuffer(8 * max(1, batch), "generate draws")
        self.caches = [(Tensor._empty([batch, L, D], "f32"), Tensor._empty([batch, L, D], "f32"))
                       for _ in model.blocks]

    def set_count(self, n):
        arr = np.array([n], np.uint32)
        check(F.wxx_memcpy_h2d(self.cur_len.ptr, arr.ctypes.data, 4), "upload count")

    def set_draws(self, draws):
        arr = np.ascontiguousarray(draws, np.float64).reshape(-1)
        check(F.wxx_memcpy_h2d(self.draws.ptr, arr.ctypes.data, arr.nbytes), "upload draws")


def _sample(model, state, logits, temperature, top_k):
    """Next id of every row from (batch, vocab) logits (row stride vocab)."""
    V = model.vocab_size
    check(F.wxx_sample_tokens(state.ids.ptr, model.max_len, state.cur_len.ptr, state.done.ptr,
                              logits.ptr, V, state.batch, V, float(temperature),
                              int(top_k), state.draws.ptr, model.max_len), "sample_tokens")


def _prefill(model, state, seq, temperature, top_k):
    ids = state.ids.narrow(1, 0, seq)
    mask = model.causal_mask(seq)
    h = model.tok_emb(ids) + model.pos_emb(model._positions(seq))
    for block, cache in zip(model.blocks, state.caches):
        h = block.forward(h, mask, kv_cache=cache)
    last = h.narrow(1, seq - 1, 1).reshape((state.batch, h.shape[-1]))
    logits = model.head(model.ln_f.forward_into_gemm(last))
    _sample(model, state, logits, temperature, top_k)


def _decode_step(model, state, temperature, top_k):
    B = state.batch
    D = model.tok_emb.embedding_dim
    h = Tensor._empty([B, D], "f32")
    check(F.wxx_decode_embed(h.buffer.ptr, state.ids.ptr, model.max_len, state.cur_len.ptr,
                             model.tok_emb.weight.ptr, model.pos_emb.weight.ptr, B, D,
                             model.vocab_size, model.max_len), "decode_embed")
    for block, cache in zip(model.blocks, state.caches):
        h = block.decode(h, cache, state.cur_len, model.max_len)
    if hasattr(model.head, "forward_ln"):
        logits = model.head.forward_ln(h, model.ln_f)       # ln_f and the head in one launch
    else:
        logits = model.head(model.ln_f.forward_into_gemm(h))
    _sample(model, state, logits, temperature, top_k)
    return logits


def generate(model, prompt, max_new_tokens=64, temperature=1.0, top_k=None, stop_token=None,
             rng=None, use_graph=True):
    """``GPT2.generate``: the prompt plus up to ``max_new_tokens`` sampled ids
    as a (batch, seq + n) uint32 array (see the module docstring)."""
    if isinstance(prompt, Tensor):
        prompt = prompt.numpy()
    ids = np.asarray(prompt)
    if ids.ndim == 1:
        ids = ids.reshape(1, -1)
    if ids.ndim != 2:
        raise ValueError(f"prompt must be 1D or 2D, got shape {ids.shape}")
    ids = np.ascontiguousarray(ids, np.uint32)
    batch, seq = ids.shape
    if seq == 0:
        raise ValueError("prompt must contain at least one token")
    if seq > model.max_len:
        raise ValueError(f"prompt length {seq} > max_len {model.max_len}")
    if temperature < 0:
        raise ValueError("temperature must be non-negative")
    k = 0
    if top_k is not None:
        if int(top_k) < 0:
            raise ValueError("top_k must be non-negative")
        k = min(int(top_k), model.vocab_size)
        k = 0 if k >= model.vocab_size else k
    if rng is None:
        rng = np.random.default_rng()
    n_new = min(int(max_new_tokens), model.max_len - seq)
    if n_new <= 0 or batch == 0:
        return ids

    prev_mode = context.MODE
    context.MODE = 1
    graph = None
    try:
        state = _DecodeState(model, batch)
        check(F.wxx_memcpy_h2d(state.ids.ptr, np.ascontiguousarray(
            np.pad(ids, ((0, 0), (0, model.max_len - seq)))).ctypes.data,
            batch * model.max_len * 4), "upload prompt")
        state.set_count(seq)
        sampling = temperature != 0.0

        def before_step():
            if sampling:
                state.set_draws(rng.random((batch, 1)))

        def stopped(n_done):
            if stop_token is None:
                return False
            col = state.ids.narrow(1, seq + n_done - 1, 1).numpy()
            return bool(np.all(col == np.uint32(stop_token)))

        before_step()
        _prefill(model, state, seq, temperature, k)
        made = 1
        if made < n_new and not stopped(made):
            while made < n_new:
                before_step()
                if graph is None and use_graph and n_new - made >= 3:
                    # capture() runs the step once (this step) and records it
                    from ..graph import capture

                    graph = capture(_decode_step, model, state, temperature, k)
                elif graph is not None:
                    graph.replay()
                else:
                    _decode_step(model, state, temperature, k)
                made += 1
                if stopped(made):
                    break
        out = state.ids.narrow(1, 0, seq + made).numpy()
    finally:
        context.MODE = prev_mode
        if graph is not None:
            graph.close()
    return out


# ------------------------------------------------------------------ beam search


class _CacheDecoder:
    """GPT2's decode steps for beam search: K / V caches of ``rows`` sequences,
    axis 1 counting positions."""

    def __init__(self, model, rows, total):
        self.model, self.rows, self.total = model, rows, model.max_len
        D = model.tok_emb.embedding_dim
        self.positions = [t for _ in model.blocks
                          for t in (Tensor._empty([rows, self.total, D]),
                                    Tensor._empty([rows, self.total, D]))]
        self.vectors = []
        self._pairs = list(zip(self.positions[::2], self.positions[1::2]))

    def prefill(self, ids, beams):
        """Logits (batch, vocab) after the prompts (batch, seq), whose keys and
        values go to the first beam of each."""
        model, seq = self.model, ids.shape[1]
        mask = model.causal_mask(seq)
        h = model.tok_emb(ids) + model.pos_emb(model._positions(seq))
        for block, (k, v) in zip(model.blocks, self._pairs):
            h = block.forward(h, mask, kv_cache=(k[::beams], v[::beams]))
        last = h.narrow(1, seq - 1, 1).reshape((ids.shape[0], h.shape[-1]))
        return model.head(model.ln_f.forward_into_gemm(last))

    def step(self, state):
        model, D = self.model, self.model.tok_emb.embedding_dim
        h = Tensor._empty([self.rows, D])
        check(F.wxx_decode_embed(h.buffer.ptr, state.ids.ptr, state.total, state.cur_len.ptr,
                                 model.tok_emb.weight.ptr, model.pos_emb.weight.ptr, self.rows, D,
                                 model.vocab_size, model.max_len), "decode_embed")
        for block, cache in zip(model.blocks, self._pairs):
            h = block.decode(h, cache, state.cur_len, model.max_len)
        if hasattr(model.head, "forward_ln"):
            return model.head.forward_ln(h, model.ln_f)
        return model.head(model.ln_f.forward_into_gemm(h))


class _StateDecoder:
    """The recurrent model's decode steps: one state per layer and sequence.  The tokens
    so far are one more than those before the newest, so the prompt's positions start at
    1 (a retention's products depend on distances alone)."""

    def __init__(self, model, rows, total):
        self.model, self.rows, self.total = model, rows, total
        self.positions = []
        self.vectors = model.new_states(rows)

    def prefill(self, ids, beams):
        from .. import functional

        model = self.model
        states = model.new_states(ids.shape[0])
        h = model.hidden(ids, None, states, 1)
        for full, s in zip(self.vectors, states):
            functional.assign(full[::beams], s)
        last = h.narrow(1, ids.shape[1] - 1, 1).reshape((ids.shape[0], h.shape[-1]))
        return model.head(last)

    def step(self, state):
        return self.model.decode(state.last, self.vectors, state.cur_len)


class _BeamState:
    """Device buffers of one search: ids (rows, total) filled to ``cur_len``, the
    rows' last tokens, scores and finished marks."""

    def __init__(self, decoder, batch, beams, stop_token):
        rows = batch * beams
        self.decoder, self.stop = decoder, stop_token
        self.batch, self.beams, self.total = batch, beams, decoder.total
        self.ids = Tensor((rows, self.total), value=0, dtype="u32")
        self.cur_len = Tensor((1,), value=0, dtype="u32")
        self.last = Tensor((rows, 1), value=0, dtype="u32")
        self.scores = Tensor((batch, beams), value=0.0)
        self.finished = (None if stop_token is None
                         else Tensor((batch, beams), value=0, dtype="u32"))

    def take(self, logits):
        """One selection from logits (rows, vocab): the beams' states, ids and
        scores follow their parents, and the chosen tokens are appended."""
        from .. import functional

        scores, parents, tokens, finished = functional.beam_select(
            logits, self.scores, self.finished, self.stop)
        functional.beam_reorder([self.ids] + self.decoder.positions, parents, self.cur_len)
        if self.decoder.vectors:
            functional.beam_reorder(self.decoder.vectors, parents)
        functional.beam_append(self.ids, tokens, self.cur_len)
        functional.assign(self.last, tokens.reshape(tuple(self.last.shape)))
        functional.assign(self.scores, scores)
        if finished is not None:
            functional.assign(self.finished, finished)

    def step(self):
        self.take(self.decoder.step(self))


def beam_search(model, prompt, beams=4, max_new_tokens=64, stop_token=None, length_penalty=0.0,
                use_graph=True):
    """Beam search after ``prompt`` ((batch, seq) or (seq,) ids) with a GPT2 or a
    ``RecurrentLM``: returns ``(ids, scores)``, a (batch, beams, seq + n) uint32
    array and the (batch, beams) float32 scores, the best beam first.

    A beam's score is the sum of its new tokens' log-probabilities, divided by
    (number of new tokens) ** ``length_penalty``.  With ``stop_token`` a beam
    that has produced it is finished: it keeps its score and is filled up with
    the stop token; the search ends when every beam is finished.

    The prompt runs once per item; each later token is one decode step of
    batch * beams rows, a selection (``functional.beam_select``) and the
    reordering of the beams' states in place (``functional.beam_reorder``),
    recorded once as a CUDA graph and replayed."""
    from .. import functional

    if isinstance(prompt, Tensor):
        prompt = prompt.numpy()
    ids = np.asarray(prompt)
    if ids.ndim == 1:
        ids = ids.reshape(1, -1)
    if ids.ndim != 2 or ids.shape[1] == 0:
        raise ValueError(f"prompt must hold at least one token per row, got shape {ids.shape}")
    ids = np.ascontiguousarray(ids, np.uint32)
    batch, seq = ids.shape
    beams = int(beams)
    if not 1 <= beams <= 16:
        raise ValueError(f"beams must be between 1 and 16, got {beams}")
    if stop_token is not None and not 0 <= int(stop_token) < model.vocab_size:
        raise ValueError(f"stop_token {stop_token} outside [0, {model.vocab_size})")
    limit = getattr(model, "max_len", None)
    if limit is not None and seq > limit:
        raise ValueError(f"prompt length {seq} > max_len {limit}")
    n_new = int(max_new_tokens) if limit is None else min(int(max_new_tokens), limit - seq)
    if n_new <= 0 or batch == 0:
        return (np.repeat(ids[:, None], beams, 1), np.zeros((batch, beams), np.float32))

    prev_mode, context.MODE = context.MODE, 1
    graph = None
    try:
        rows = batch * beams
        kind = _CacheDecoder if hasattr(model, "pos_emb") else _StateDecoder
        state = _BeamState(kind(model, rows, seq + n_new), batch, beams, stop_token)
        start = functional.from_numpy(ids, dtype=np.uint32)
        # the first selection: every item's only live beam is its first
        logits = state.decoder.prefill(start, beams)
        wide = Tensor((batch, beams, logits.shape[-1]), buffer=logits.buffer,
                      offset=logits.offset, stride=(logits.shape[-1], 0, 1))
        alive = np.full((batch, beams), -np.inf, np.float32)
        alive[:, 0] = 0.0
        functional.assign(state.scores, functional.from_numpy(alive))
        functional.assign(state.ids.narrow(1, 0, seq),
                          functional.from_numpy(np.repeat(ids, beams, 0), dtype=np.uint32))
        functional.assign(state.cur_len, seq)
        state.take(functional.contiguous(wide).reshape((rows, logits.shape[-1])))
        made = 1

        def stopped():
            return state.finished is not None and bool(state.finished.numpy().all())

        while made < n_new and not stopped():
            if graph is None and use_graph and n_new - made >= 3:
                from ..graph import capture

                graph = capture(state.step)      # runs the step once and records it
            elif graph is not None:
                graph.replay()
            else:
                state.step()
            made += 1
        out = state.ids.narrow(1, 0, seq + made).numpy().reshape(batch, beams, seq + made)
        scores = state.scores.numpy()
    finally:
        context.MODE = prev_mode
        if graph is not None:
            graph.close()
    new = out[:, :, seq:]
    length = np.full((batch, beams), made)
    if stop_token is not None:
        hit = new == np.uint32(stop_token)
        length = np.where(hit.any(-1), hit.argmax(-1) + 1, made)
    scores = (scores / length.astype(np.float64) ** float(length_penalty)).astype(np.float32)
    order = np.argsort(-scores, -1, kind="stable")
    return (np.take_along_axis(out, order[:, :, None], 1), np.take_along_axis(scores, order, 1))
