"""Distils a GPT2 into a recurrent language model and decodes both by beam search.

    python examples/distill_recurrent.py [--steps 300]

1. A small GPT2 is trained on synthetic text (a sparse random bigram process).
2. It is run over packed rows of documents and the 16 largest logits of every
   position are kept (``functional.topk``).
3. A ``RecurrentLM`` is trained on them (``nn.DistillLoss``), its recurrence cut
   at document starts; the training step is recorded once as a CUDA graph.
4. Both models continue a prompt by beam search: the GPT2 over its K/V caches,
   the student over one vector per layer (``beam_search``).
"""

import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import wxx_b200 as wxx  # noqa: E402

F = wxx.functional
VOCAB, ROWS, LENGTH, KEPT = 256, 16, 128, 16


def bigram_text(rng, rows, length):
    """Rows of documents of 16 to 48 tokens: every token has four likely
    successors.  Returns ids and the marks of document starts."""
    follow = np.random.default_rng(7).integers(1, VOCAB, size=(VOCAB, 4))
    ids = np.zeros((rows, length), np.uint32)
    starts = np.zeros((rows, length), np.uint32)
    for r in range(rows):
        left = 0
        for t in range(length):
            if left == 0:
                starts[r, t], left = 1, int(rng.integers(16, 49))
                ids[r, t] = rng.integers(1, VOCAB)
            else:
                ids[r, t] = follow[ids[r, t - 1], rng.choice(4, p=[0.6, 0.2, 0.15, 0.05])]
            left -= 1
    return ids, starts


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    args = ap.parse_args()
    rng = np.random.default_rng(0)
    wxx.manual_seed(0)

    def u32(a):
        return F.from_numpy(a, dtype=np.uint32)

    teacher = wxx.nn.GPT2(VOCAB, 128, 4, 2, max_len=LENGTH, dropout=0.0)
    opt = wxx.nn.AdamW(teacher.parameters(), lr=2e-3)
    for step in range(args.steps):
        ids, _ = bigram_text(rng, ROWS, LENGTH + 1)
        opt.zero_grad()
        logits = teacher(u32(ids[:, :-1])).reshape((ROWS * LENGTH, VOCAB))
        loss = wxx.nn.CCELoss()(logits, u32(ids[:, 1:].reshape(-1)))
        loss.backward()
        opt.step()
        if step % 100 == 0 or step == args.steps - 1:
            print(f"teacher step {step}: loss {loss.item():.3f}")

    student = wxx.nn.RecurrentLM(VOCAB, 128, n_heads=32, n_layers=2)
    opt = wxx.nn.AdamW(student.parameters(), lr=2e-3)
    distill = wxx.nn.DistillLoss(temperature=1.5)
    ids, starts = (u32(a) for a in bigram_text(rng, ROWS, LENGTH))
    top, top_ids = F.topk(F.from_numpy(np.zeros((ROWS * LENGTH, VOCAB), np.float32)), KEPT)

    def train_step():
        opt.zero_grad()
        loss = distill(student(ids, starts).reshape((ROWS * LENGTH, VOCAB)), top, top_ids)
        loss.backward()
        opt.step()
        return loss

    def next_batch():
        new, marks = bigram_text(rng, ROWS, LENGTH)
        F.assign(ids, u32(new))
        F.assign(starts, u32(marks))
        with wxx.backend.inferenceMode():
            t, i = F.topk(teacher(ids).reshape((ROWS * LENGTH, VOCAB)), KEPT)
        F.assign(top, t)
        F.assign(top_ids, i)

    # Module.__call__ passes positional arguments on, so student(ids, starts) is
    # forward(ids, reset=starts)
    next_batch()
    graph = wxx.graph.capture(train_step)
    for step in range(args.steps):
        next_batch()
        loss = graph.replay()
        if step % 100 == 0 or step == args.steps - 1:
            print(f"student step {step}: loss {loss.item():.3f}")
    graph.close()

    prompt = bigram_text(rng, 1, 8)[0]
    for name, model in (("teacher", teacher), ("student", student)):
        t0 = time.perf_counter()
        out, scores = model.beam_search(prompt, beams=4, max_new_tokens=24)
        ms = (time.perf_counter() - t0) * 1e3
        print(f"{name}: {out[0, 0, 8:].tolist()} score {scores[0, 0]:.2f} ({ms:.0f} ms)")
    assert wxx.backend.device_status() == 0


if __name__ == "__main__":
    main()
