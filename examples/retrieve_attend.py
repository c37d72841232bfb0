"""Retrieve, then attend: the index finds passages, the key/value cache holds what a
model made of them, and a question's tokens attend to them.

    python examples/retrieve_attend.py [--bits 4]

Every passage has an embedding (a row of the index) and the keys and values of
its tokens (here random: they stand for what a model computes once per passage).
Each question searches the index, the passages found enter the paged cache one after
the other, the question's tokens follow and attend to all that came before them
in one chunk, and then tokens are generated one at a time: write, attend.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import jhq_gpu_amd as jg  # noqa: E402


def run(device="cuda:0", bits=8, passages=2000, d=64, questions=4, k=5, heads=16, kv_heads=4,
        head_dim=128, generate=8, seed=0):
    """Returns the passages found, what each sequence holds and every output."""
    rng = np.random.default_rng(seed)
    emb = rng.standard_normal((passages, d)).astype(np.float32)
    index = jg.JHQGpuIndex(d, jg.Params(M=8, nlist=32, nprobe=8, alpha=10.0, batch_size=64))
    index.train(emb)
    index.add(emb)
    ask = emb[rng.choice(passages, questions, replace=False)]
    ask = ask + 0.1 * rng.standard_normal(ask.shape).astype(np.float32)
    _, ids = index.search(ask, k)

    gen = torch.Generator().manual_seed(seed)

    def rows(n, h):
        return torch.randn(n, h, head_dim, generator=gen).bfloat16()

    # the keys and values of the passages that were found
    store = {int(i): (rows(n, kv_heads), rows(n, kv_heads))
             for i, n in zip(np.unique(ids), rng.integers(20, 90, ids.size))}
    cache = jg.KVCache(num_pages=questions * 16, page_size=64, kv_heads=kv_heads,
                       head_dim=head_dim, bits=bits, device=device)
    pages = jg.KVPages(cache, questions, 16 * 64)
    held = [([], []) for _ in range(questions)]

    def enter(kk, vv):
        """kk, vv: one tensor a sequence, its new tokens."""
        batch = pages.extend([len(x) for x in kk])
        for s in range(questions):
            held[s][0].append(kk[s])
            held[s][1].append(vv[s])
        cache.write(torch.cat(kk).to(device), torch.cat(vv).to(device), batch)
        return batch

    enter([torch.cat([store[int(i)][0] for i in row]) for row in ids],
          [torch.cat([store[int(i)][1] for i in row]) for row in ids])
    steps = []
    # the questions, of different lengths, in one chunk; then a token each
    for new in [list(rng.integers(5, 40, questions))] + [[1] * questions] * generate:
        batch = enter([rows(n, kv_heads) for n in new], [rows(n, kv_heads) for n in new])
        q = rows(sum(new), heads)
        steps.append(dict(new=[int(n) for n in new], length=[pages.length(s) for s in range(questions)], q=q,
                          out=cache.attend(q.to(device), batch).cpu()))
    return dict(ids=ids, steps=steps, bits=bits,
                k=[torch.cat(x[0]) for x in held], v=[torch.cat(x[1]) for x in held])


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--bits", type=int, default=8, choices=(8, 4))
    r = run(bits=ap.parse_args().bits)
    for s, row in enumerate(r["ids"]):
        print(f"question {s}: passages {row.tolist()}, {len(r['k'][s])} tokens in the cache, "
              f"last output |o| = {r['steps'][-1]['out'][s].float().norm():.4f}")


if __name__ == "__main__":
    main()
