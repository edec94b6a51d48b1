"""Beam decoding over the scaled 8-bit paged cache, on one attention layer with
random weights: ragged prompts are appended and attended in one call each, every
prompt's pages are forked to its beams, beams that lose give up their pages and
the winners' are forked in their place, the best beam's last tokens are attended
again as draft rows, and the pool is compacted at the end.

    python examples/cache8_beams.py [--steps 16] [--code int8]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "unlimited-ocr_b200"))

from srswa.cache8 import Cache8, PageTable  # noqa: E402

VOCAB, H, HKV, D, BLOCK = 512, 16, 4, 128, 64


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Layer:
    """Embedding -> grouped-query attention -> logits."""

    def __init__(self, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        w = lambda a, b: (torch.randn(a, b, device="cuda", generator=g) / a ** 0.5).to(torch.bfloat16)  # noqa: E731
        self.emb, self.out = w(VOCAB, H * D) * VOCAB ** 0.5, w(H * D, VOCAB)
        self.wq, self.wk, self.wv = w(H * D, H * D), w(H * D, HKV * D), w(H * D, HKV * D)

    def qkv(self, tokens):
        x = self.emb[tokens]
        return (x @ self.wq).view(-1, H, D), (x @ self.wk).view(-1, HKV, D), (x @ self.wv).view(-1, HKV, D)

    def logp(self, o):
        return torch.log_softmax((o.flatten(1) @ self.out).float(), -1)


def run(prompt_lens=(700, 90, 1, 333), beams=4, steps=16, window=256, sinks=4, code=torch.float8_e4m3fn, seed=0):
    """Returns the best beams' tokens, the cache, its pages, and the last draft
    rows' queries and outputs (before and after the pool was compacted)."""
    layer, R = Layer(seed), len(prompt_lens)
    rows, blocks = R * beams, -(-(max(prompt_lens) + steps) // BLOCK)
    cache = Cache8(rows * blocks, BLOCK, HKV, D, dtype=code)
    pages = PageTable(rows, blocks, rows * blocks, BLOCK, cache.tensors())
    g = torch.Generator("cuda").manual_seed(seed + 1)
    history = [torch.randint(VOCAB, (n,), device="cuda", generator=g).tolist() for n in prompt_lens for _ in range(1)]

    # the prompts, in the first row of each request
    first = i32([r * beams for r in range(R)])
    short = [pages.extend(first, i32(prompt_lens))]
    q, k, v = layer.qkv(torch.tensor(sum(history, []), device="cuda"))
    cu = torch.nn.functional.pad(i32(prompt_lens).cumsum(0, dtype=torch.int32), (1, 0))
    at = dict(cu_seqlens=cu, prefix_lens=torch.zeros_like(cu[1:]))
    table = pages.block_table[first.long()]
    cache.append(k, v, table, **at)
    o = cache.attend(q, table, window=window, sinks=sinks, **at)
    score, token = layer.logp(o[cu[1:].long() - 1]).topk(beams)  # [R, beams]
    others = [r * beams + b for r in range(R) for b in range(1, beams)]
    short.append(pages.fork(i32([c // beams * beams for c in others]), i32(others)))
    tokens = [history[r] + [int(t)] for r in range(R) for t in token[r]]

    for step in range(1, steps):
        # one new token a row
        all_rows = torch.arange(rows, dtype=torch.int32, device="cuda")
        short.append(pages.extend(all_rows, pages.seq_lens + 1))
        q, k, v = layer.qkv(torch.tensor([t[-1] for t in tokens], device="cuda"))
        cache.append(k, v, pages.block_table, pages.seq_lens)
        o = cache.attend(q, pages.block_table, pages.seq_lens, window=window, sinks=sinks)
        total = (score.view(rows, 1) + layer.logp(o)).view(R, -1)
        score, pick = total.topk(beams)
        # each winner's first continuation stays in its row; the others take the losers' rows
        parents, children, new = [], [], [None] * rows
        for r, p in enumerate(pick.tolist()):
            free = [r * beams + b for b in range(beams) if b not in {x // VOCAB for x in p}]
            order, place = [None] * beams, {}
            for n, x in enumerate(p):
                parent = r * beams + x // VOCAB
                if parent in place:
                    parents.append(parent)
                    children.append(free.pop())
                row = children[-1] if parent in place else parent
                place[parent] = True
                new[row] = tokens[parent] + [x % VOCAB]
                order[row - r * beams] = n
            score[r] = score[r, torch.tensor(order, device="cuda")].clone()
        if children:
            pages.free(i32(children))
            short.append(pages.fork(i32(parents), i32(children)))
        tokens = new

    # only the best beam of each request stays; its last tokens once more, as draft rows
    best = (score.argmax(1) + torch.arange(R, device="cuda") * beams).tolist()
    pages.free(i32([r for r in range(rows) if r not in best]))
    draft = 1 + min(3, steps - 1)
    last = torch.tensor([tokens[b][-1 - draft:-1] for b in best], device="cuda").flatten() if steps > 1 else None
    result = {"tokens": [tokens[b] for b in best], "cache": cache, "pages": pages, "rows": best, "window": window,
              "sinks": sinks}
    look = torch.tensor(best, device="cuda")
    if last is not None:
        q = layer.qkv(last)[0]
        attend = lambda: cache.attend(q, pages.block_table[look], pages.seq_lens[look], window=window, sinks=sinks)  # noqa: E731
        before = attend()
        result["live"] = pages.compact()
        result.update(q=q, before=before, after=attend(), draft=draft)
    assert all(int(s) == 0 for s in short), "the pool ran out of pages"
    return result


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--code", choices=["e4m3", "int8"], default="e4m3")
    a = ap.parse_args()
    out = run(beams=a.beams, steps=a.steps, code=torch.int8 if a.code == "int8" else torch.float8_e4m3fn)
    for n, t in enumerate(out["tokens"]):
        print(f"request {n}: {len(t)} tokens, the last {t[-min(8, a.steps):]}")
    if "live" in out:
        print(f"pages in use after compaction: {int(out['live'])}; draft rows unchanged by it:",
              bool(torch.equal(out["before"], out["after"])))


if __name__ == "__main__":
    main()
