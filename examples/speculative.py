"""Speculative decoding over a paged key/value cache of bounded size, with the operators of
technograd_b200.kvcache: a toy decoder (random weights) drafts trees of tokens from the bigrams it has
seen, checks each tree in one pass (rope to the drafted positions, tree_attention), keeps the longest path that its own greedy
choices confirm (commit), sums up the attention each cached position receives (attention_weights),
and drops the least attended ones when the cache is full (evict).

    python examples/speculative.py [--tokens 200] [--limit 160 --budget 96] [--check]

--check decodes the same prompts one token at a time, without drafts, and compares the tokens: they are
the same as long as nothing has been evicted. Needs a B200 and the built library."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from technograd_b200 import kvcache  # noqa: E402

PAGE = 16


class Toy:
    """A decoder of a few small layers: rmsnorm, grouped-query attention with rotary positions, SwiGLU."""

    def __init__(self, layers=2, hidden=64, nq=4, nkv=2, dim=32, vocab=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.layers, self.nq, self.nkv, self.dim, self.vocab = layers, nq, nkv, dim, vocab
        self.rotary = kvcache.Rotary(dim, theta=1e4)

        def w(*s):
            return torch.randn(s, generator=g, device="cuda") * s[0] ** -0.5

        self.embed = w(vocab, hidden) * vocab ** 0.5
        self.head = w(hidden, vocab)
        self.blocks = [dict(qkv=w(hidden, (nq + 2 * nkv) * dim), out=w(nq * dim, hidden), gate=w(hidden, 2 * hidden), up=w(hidden, 2 * hidden),
                            down=w(2 * hidden, hidden)) for _ in range(layers)]

    def forward(self, tokens, positions, attend):
        """Logits of tokens [seqs, tokens] at their positions; attend(layer, q, k, v) is the attention."""
        def norm(x):
            return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

        at = positions.to(torch.int32).contiguous()
        x = self.embed[tokens]
        for i, p in enumerate(self.blocks):
            qkv = (norm(x) @ p["qkv"]).unflatten(-1, (-1, self.dim))
            q, k, v = qkv.split([self.nq, self.nkv, self.nkv], 2)
            x = x + attend(i, kvcache.rope(q, self.rotary, at), kvcache.rope(k, self.rotary, at), v.contiguous()).flatten(2) @ p["out"]
            h = norm(x)
            x = x + (torch.nn.functional.silu(h @ p["gate"]) * (h @ p["up"])) @ p["down"]
        return norm(x) @ self.head


class Decoder:
    """Greedy decoding of several sequences over paged caches, one per layer.

    limit: positions a sequence may hold; budget: what eviction leaves."""

    def __init__(self, model, seqs, limit, budget):
        self.model, self.seqs, self.limit, self.budget = model, seqs, limit, budget
        cols = -(-(limit + 64) // PAGE)
        shape = (2 * seqs * cols, model.nkv, PAGE, model.dim)
        # two sets of pages per layer: eviction moves what stays from one to the other
        tables = torch.randperm(2 * seqs * cols, device="cuda").to(torch.int32).view(2, seqs, cols)
        self.tables, self.side = [tables[0].contiguous(), tables[1].contiguous()], 0
        self.pools = [(torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda")) for _ in range(model.layers)]
        self.acc = [torch.zeros(seqs, model.nkv, cols * PAGE, device="cuda") for _ in range(model.layers)]
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.positions = torch.zeros(seqs, dtype=torch.long, device="cuda")  # tokens so far, evicted ones among them
        self.longest = 0
        self.evictions = 0

    def caches(self, side=None):
        table = self.tables[self.side if side is None else side]
        return [kvcache.PagedKV(k, v, table, self.lens, max_len=self.longest) for k, v in self.pools]

    def check(self, tokens, depth, mask, accept):
        """One pass over drafted tokens [seqs, tokens]; accept(logits) -> (path, count): the drafted tokens, in order,
        that go into the cache, and how many. Returns the logits."""
        caches, kept = self.caches(), []

        def attend(i, q, k, v):
            k = k.contiguous()
            out, lse = kvcache.tree_attention(caches[i], q, k, v, mask=mask)
            kept.append((q, k, v, lse))
            return out

        logits = self.model.forward(tokens, self.positions[:, None] + depth, attend)
        path, count = accept(logits)
        taken = torch.arange(path.shape[1], device="cuda") < count[:, None]
        select = torch.where(taken, 1 << path.clamp(min=0).long(), 0).sum(1)  # as bits
        for i, (q, k, v, lse) in enumerate(kept):
            acc, fresh = kvcache.attention_weights(caches[i], q, k, lse, mask=mask, select=select, acc=self.acc[i])
            self.acc[i][:, :, :acc.shape[2]] = acc
            lens = kvcache.commit(caches[i], k, v, count, path=path, new=fresh, acc=self.acc[i])
        self.lens, self.positions = lens, self.positions + count
        self.longest += int(count.max())  # an upper bound, without waiting for lens
        if self.longest > self.limit:
            self.evict()
        return logits

    def evict(self):
        """Every layer's and head's most attended positions, and the last quarter, to the other pages."""
        self.longest = int(self.lens.max())
        if self.longest <= self.limit:
            return
        for i, (src, dst) in enumerate(zip(self.caches(), self.caches(1 - self.side))):
            _, acc, lens = kvcache.evict(src, dst, self.acc[i], self.budget, recent=self.budget // 4, sink=1)
            self.acc[i].zero_()
            self.acc[i][:, :, :self.budget] = acc
        self.lens, self.side, self.longest = lens, 1 - self.side, self.budget
        self.evictions += 1

    def prompt(self, tokens):
        """The prompt's tokens [seqs, tokens] into the cache, 64 at a time; the next token of each sequence."""
        for part in tokens.split(64, 1):
            T = part.shape[1]
            path = torch.arange(T, dtype=torch.int32, device="cuda").expand(self.seqs, T).contiguous()
            count = torch.full((self.seqs,), T, dtype=torch.int32, device="cuda")
            logits = self.check(part, torch.arange(T, device="cuda").expand(self.seqs, T), None, lambda _: (path, count))
        return logits[:, -1].argmax(-1).tolist()


def tree(root, followers, width=2, depth=3):
    """Drafted tokens from root on: (tokens, parents, depths), each token's likeliest followers below it."""
    tokens, parents, depths, level = [root], [-1], [0], [0]
    for d in range(1, depth + 1):
        level, above = [], level
        for a in above:
            for t in followers.get(tokens[a], [])[:width]:
                level.append(len(tokens))
                tokens.append(t), parents.append(a), depths.append(d)
    return tokens, parents, depths


def generate(model, prompts, new, limit, budget, speculate):
    """`new` greedy tokens after each prompt; (tokens, passes over the model, evictions)."""
    B = len(prompts)
    dec = Decoder(model, B, limit, budget)
    last = dec.prompt(torch.tensor(prompts, device="cuda"))
    out = [[t] for t in last]
    seen = [{} for _ in range(B)]  # token -> its followers, the latest first

    def learn(b, text):
        for x, y in zip(text, text[1:]):
            f = seen[b].setdefault(x, [])
            if y in f:
                f.remove(y)
            f.insert(0, y)

    for b in range(B):
        learn(b, list(prompts[b]) + out[b])
    passes = 0
    while min(len(o) for o in out) < new:
        drafts = [tree(out[b][-1], seen[b] if speculate else {}) for b in range(B)]
        T = max(len(d[0]) for d in drafts)
        tokens, depth, masks = [], [], []
        for t, parents, d in drafts:
            m = []
            for i, p in enumerate(parents):
                m.append((m[p] if p >= 0 else 0) | 1 << i)
            pad = T - len(t)
            tokens.append(t + [0] * pad), depth.append(d + [0] * pad), masks.append(m + [0] * pad)
        picked = []

        def accept(logits):
            best = logits.argmax(-1).tolist()
            paths = []
            for b, (t, parents, _) in enumerate(drafts):
                at, path = 0, [0]
                while True:
                    child = [i for i, p in enumerate(parents) if p == at and t[i] == best[b][at]]
                    if not child:
                        break
                    at = child[0]
                    path.append(at)
                paths.append(path)
                picked.append([t[i] for i in path[1:]] + [best[b][at]])
            path = torch.tensor([p + [-1] * (T - len(p)) for p in paths], dtype=torch.int32, device="cuda")
            return path, torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")

        dec.check(torch.tensor(tokens, device="cuda"), torch.tensor(depth, device="cuda"), torch.tensor(masks, dtype=torch.int64, device="cuda"), accept)
        passes += 1
        for b, p in enumerate(picked):
            learn(b, [out[b][-1]] + p)
            out[b] += p
    return [o[:new] for o in out], passes, dec.evictions


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--seqs", type=int, default=3)
    ap.add_argument("--prompt", type=int, default=100)
    ap.add_argument("--limit", type=int, default=160)
    ap.add_argument("--budget", type=int, default=96)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    model = Toy()
    g = torch.Generator().manual_seed(1)
    prompts = torch.randint(0, model.vocab, (a.seqs, a.prompt), generator=g).tolist()
    out, passes, evictions = generate(model, prompts, a.tokens, a.limit, a.budget, True)
    print(f"{a.seqs} sequences, {a.tokens} tokens each: {passes} passes over the model, {evictions} evictions")
    if a.check:
        one, steps, _ = generate(model, prompts, a.tokens, a.prompt + a.tokens + 64, a.budget, False)
        room, p, _ = generate(model, prompts, a.tokens, a.prompt + a.tokens + 64, a.budget, True)
        same = sum(x == y for x, y in zip(sum(one, []), sum(room, [])))
        print(f"without drafts: {steps} passes; with drafts and room for all: {p}; {same} of {a.seqs * a.tokens} tokens the same")
        return one == room
    return True


if __name__ == "__main__":
    sys.exit(0 if main() else 1)
