"""Workloads of the paged cache's next operators: rotary positions, the append of new tokens to the cache with the
rotation on the way, and attention for a batch whose sequences share long prefixes.

`own` selects between the plain forms below (elementary torch operations in f32, angles in 64 bits) and the calls of
technograd_b200.kvcache. A case names an operator (`op`) and its sizes:

  seqs, tokens            sequences, new tokens of each
  nkv, group, dim         key/value heads, query heads per key/value head, head dimension (rope: `heads` of them)
  type                    f32, f16 or bf16 of everything but norms, lse and frequencies
  part, layout            rotated elements of a head; "half" (i with i + part / 2) or "pairs" (2 i with 2 i + 1)
  stretch                 context extension: 1, or the factor by which slow frequencies are divided
  train                   rope: forward and gradient
  page, order             positions per page; "head": pools [pages][nkv][page][dim], "pos": [pages][page][nkv][dim]
  len                     append: the longest cache before it; ragged: the others are shorter, down to empty
  short                   true where sequences have fewer new tokens than `tokens`
  query, norm, keys       append: queries rotated too; RMS norm of q and k before; the rotated keys returned as well
  moved                   append: positions are given (after an eviction they are not the cache's)
  groups, alone           shared: groups of sequences with one prefix each, and sequences without one
  prefix, tail            shared: the longest prefix, and the most positions that a sequence has of its own
  tree                    shared: "chain" or "tree" of the new tokens
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
QWEN = dict(nkv=8, group=2, dim=128)  # the Qwen3-0.6B attention layer: 16 query heads over 8
THETA, EPS = 1e6, 1e-6  # its rotary base and norm


def listed():
    return [
        # one user's drafted token: the latency of rotating its queries
        dict(name="rope-one", op="rope", seqs=1, tokens=1, heads=16, dim=128, type="bf16", part=128, layout="half", stretch=1, train=False),
        # drafted trees of a small wave, part of the head, neighbours paired
        dict(name="rope-tree", op="rope", seqs=8, tokens=21, heads=24, dim=80, type="f16", part=32, layout="pairs", stretch=4, train=False),
        # the queries of a training batch, forward and gradient
        dict(name="rope-train", op="rope", seqs=8, tokens=6001, heads=16, dim=128, type="bf16", part=128, layout="half", stretch=1, train=True),
        # the 8-sequence decode wave's step, in the framework's own f32
        dict(name="append-wave-f32", op="append", seqs=8, tokens=1, type="f32", part=128, layout="half", stretch=1, page=64, order="head", len=257,
             ragged=True, short=False, query=True, norm=True, keys=True, moved=False, **QWEN),
        # a large decode wave's step
        dict(name="append-wave", op="append", seqs=256, tokens=1, type="bf16", part=128, layout="half", stretch=1, page=16, order="pos", len=257,
             ragged=True, short=False, query=True, norm=True, keys=True, moved=False, **QWEN),
        # a head of odd size, a part of it rotated, odd pages, after an eviction
        dict(name="append-part", op="append", seqs=3, tokens=33, nkv=2, group=3, dim=80, type="f16", part=40, layout="half", stretch=8, page=5,
             order="pos", len=101, ragged=True, short=True, query=True, norm=False, keys=False, moved=True),
        # whole prompts, ragged, in a stretched context
        dict(name="append-prompt", op="append", seqs=16, tokens=2047, type="bf16", part=128, layout="half", stretch=4, page=64, order="head", len=0,
             ragged=False, short=True, query=True, norm=True, keys=False, moved=False, **QWEN),
        # four samples of one short prompt: latency
        dict(name="shared-samples", op="shared", seqs=4, tokens=1, type="f32", page=16, order="head", groups=1, alone=0, prefix=513, tail=65,
             tree="chain", short=False, **QWEN),
        # a decode wave below one system prompt
        dict(name="shared-wave", op="shared", seqs=64, tokens=1, type="bf16", page=16, order="pos", groups=1, alone=0, prefix=2048, tail=513,
             tree="chain", short=False, **QWEN),
        # a full server: several long system prompts, and requests without one
        dict(name="shared-server", op="shared", seqs=256, tokens=1, type="bf16", page=64, order="head", groups=6, alone=9, prefix=8001, tail=1024,
             tree="chain", short=False, **QWEN),
        # drafted trees over one long document
        dict(name="shared-tree", op="shared", seqs=40, tokens=21, type="bf16", page=64, order="head", groups=1, alone=0, prefix=32768, tail=500,
             tree="tree", short=True, **QWEN),
        # a few readers of one very long document, eight query heads per key head
        dict(name="shared-long", op="shared", seqs=8, tokens=1, nkv=4, group=8, dim=128, type="f16", page=16, order="head", groups=1, alone=0,
             prefix=131009, tail=200, tree="chain", short=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rope", "append", "append", "shared", "shared", "shared"])
    c = dict(op=op, seqs=spread(1, 256), tokens=rng.choice([1, spread(1, 64)]), dim=rng.choice([8, 64, 80, 96, 128, 128, 128, 256]),
             type=rng.choice(["f32", "f16", "bf16"]))
    if op == "rope":
        c["tokens"] = spread(1, 8192)
        c["heads"] = spread(1, 40)
    else:
        c.update(nkv=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 3, 4, 8]), page=rng.choice([1, 5, 16, 16, 24, 64, 128]), order=rng.choice(["head", "pos"]))
    if op in ("rope", "append"):
        c.update(part=rng.choice([c["dim"], c["dim"], 2 * rng.randint(1, c["dim"] // 2)]), layout=rng.choice(["half", "half", "pairs"]),
                 stretch=rng.choice([1, 4, 8]))
    if op == "rope":
        c["train"] = rng.random() < 0.3
    elif op == "append":
        c["tokens"] = rng.choice([c["tokens"], spread(64, 2048)])
        c.update(len=rng.choice([0, spread(1, 300)]), ragged=rng.random() < 0.6, short=rng.random() < 0.5, query=rng.random() < 0.7,
                 norm=rng.random() < 0.5, keys=rng.random() < 0.5, moved=rng.random() < 0.3)
    else:
        c.update(groups=rng.choice([0, 1, 1, spread(1, 12)]), prefix=spread(16, 131072), tail=spread(1, 2000), short=rng.random() < 0.5)
        c["alone"] = rng.choice([0, 0, rng.randint(0, c["seqs"])])
        c["tree"] = rng.choice(["chain", "tree"]) if c["tokens"] > 1 else "chain"

    def cost(x):  # bytes, operations, and what a plain form holds of scores
        if op == "shared":
            x["groups"] = min(x["groups"], x["seqs"])
            x["alone"] = min(x["alone"], x["seqs"] - x["groups"]) if x["groups"] else x["seqs"]
        w = work(x)
        held = 4 * x["seqs"] * x["tokens"] * x["nkv"] * x["group"] * (x["prefix"] + x["tail"] + x["tokens"]) if op == "shared" else 0
        pool = 2 * SIZE[x["type"]] * x["nkv"] * x["dim"] * x["seqs"] * (x["len"] + x["tokens"] if op == "append" else x["tail"]) if op != "rope" else 0
        return w["bytes"], w["flops"], held, pool

    alike = [cost(x) for x in listed() if x["op"] == op]
    most = [max(x[i] for x in alike) for i in range(4)]
    while True:  # no dearer than the dearest listed case of its operator
        if all(x <= y for x, y in zip(cost(c), most)):
            return c
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        elif op == "shared":
            c["prefix"], c["tail"] = (c["prefix"] + 1) // 2, (c["tail"] + 1) // 2
        else:
            c["tokens"] = (c["tokens"] + 1) // 2


def lengths(c):
    """Append: positions that each sequence has in the cache before."""
    r = random.Random(c["seqs"] * 1000003 + c["len"])
    n = [c["len"]] * c["seqs"]
    if c["ragged"]:
        n[1:] = [r.randint(c["len"] // 2, c["len"]) for _ in n[1:]]
        if len(n) >= 4:
            n[2], n[3] = min(1, c["len"]), 0
    return n


def counts(c):
    """New tokens of each sequence."""
    r = random.Random(c["seqs"] * 7919 + c["tokens"])
    return [r.randint(c["tokens"] // 2, c["tokens"]) for _ in range(c["seqs"])] if c["short"] else [c["tokens"]] * c["seqs"]


def grouping(c):
    """Shared: (first sequence, sequences, shared positions) of each group, whole pages; and every sequence's length. Sequences
    without a prefix lie between the groups."""
    r = random.Random(c["seqs"] * 104729 + c["groups"] * 31 + c["prefix"])
    if not c["groups"]:
        return [], [r.randint(c["tail"] // 2, c["tail"]) for _ in range(c["seqs"])]
    rest = c["seqs"] - c["alone"]
    cuts = sorted(r.sample(range(1, rest), c["groups"] - 1)) if c["groups"] > 1 else []
    sizes = [y - x for x, y in zip([0] + cuts, cuts + [rest])]
    gaps = [0] * (c["groups"] + 1)
    for _ in range(c["alone"]):
        gaps[r.randrange(len(gaps))] += 1
    groups, at, lens = [], gaps[0], [None] * c["seqs"]
    for g, size in enumerate(sizes):
        shared = (c["prefix"] if g == 0 else r.randint(c["prefix"] // 4, c["prefix"])) // c["page"] * c["page"]
        for b in range(at, at + size):
            lens[b] = shared + (r.randint(1, c["tail"]) if b > at else c["tail"])
        if shared:
            groups.append((at, size, shared))
        at += size + gaps[g + 1]
    return groups, [r.randint(0, c["tail"]) if n is None else n for n in lens]


def work(c):
    e, d = SIZE[c["type"]], c["dim"]
    if c["op"] == "rope":
        n = c["seqs"] * c["tokens"] * c["heads"]
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * e * n * d + 4 * c["seqs"] * c["tokens"]) + 4 * c["part"], "flops": passes * 3 * n * c["part"]}
    t = counts(c)
    nq = c["nkv"] * c["group"]
    if c["op"] == "append":
        q = nq if c["query"] else 0
        n, padded = sum(t), c["seqs"] * c["tokens"]
        reads, written = n * (q + 2 * c["nkv"]), 2 * n * c["nkv"] + padded * (q + (c["nkv"] if c["keys"] else 0))
        pages = sum(-(-(x + y) // c["page"]) - x // c["page"] for x, y in zip(lengths(c), t))
        return {"bytes": e * d * (reads + written) + 4 * pages + 12 * c["seqs"] + 4 * c["part"] + (4 * n if c["moved"] else 0) + (8 * d if c["norm"] else 0),
                "flops": n * (q + c["nkv"]) * (3 * c["part"] + (4 * d if c["norm"] else 0))}
    groups, lens = grouping(c)
    once = sum(lens) - sum((size - 1) * shared for _, size, shared in groups)
    drafted = c["seqs"] * c["tokens"]
    pairs = sum(k * (x + 1) for k, x in zip(t, lens))
    return {"bytes": 2 * e * c["nkv"] * d * (once + drafted) + 2 * e * drafted * nq * d + 4 * once // c["page"] + 8 * drafted + 4 * drafted * nq,
            "flops": 4 * d * nq * pairs}


def frequencies(c):
    """Radians per position of each pair. A stretched context divides the slow ones by the factor, keeps the fast ones, and goes from one to the other in between
    (between 32 turns and 1 turn within 32768 positions); the gain on the rotated part is what goes with it."""
    i = torch.arange(c["part"] // 2, dtype=torch.float64)
    f = THETA ** (-2 * i / c["part"])
    if c["stretch"] == 1:
        return f, 1.0
    turns = 32768 * f / (2 * math.pi)
    keep = ((torch.log(turns) - math.log(1)) / math.log(32)).clamp(0, 1)
    return f * (keep + (1 - keep) / c["stretch"]), 1 + 0.1 * math.log(c["stretch"])


def tree_masks(c, gen):
    """Bit u of [b][t]: token t sees new token u. A tree's token sees its ancestors and itself."""
    out = []
    for row in torch.randint(0, 1 << 30, (c["seqs"], c["tokens"]), generator=gen).tolist():
        m = []
        for t, x in enumerate(row):
            parent = t - 1 if c["tree"] == "chain" else x % (t + 1) - 1
            m.append((m[parent] if parent >= 0 else 0) | 1 << t)
        out.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(out, dtype=torch.int64)


def pools(c, gen, total):
    """Pools of `total` pages."""
    shape = (total, c["nkv"], c["page"], c["dim"]) if c["order"] == "head" else (total, c["page"], c["nkv"], c["dim"])
    made = [torch.randn(shape, generator=gen, device="cuda", dtype=TYPES[c["type"]]) for _ in range(2)]
    return [x if c["order"] == "head" else x.transpose(1, 2) for x in made]


def table_of(need, gen, host):
    """Pages in random order: a table [seqs][cols] (-1 where no page is) of so many pages each, and the pages' number."""
    cols, total = max(1, max(need)), max(1, sum(need))
    where = torch.randperm(total, generator=host).to(torch.int32)
    table, at = torch.full((len(need), cols), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = where[at:at + n]
        at += n
    return table, total


def prepare(c, seed):
    gen, host = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dt = TYPES[c["type"]]
    s = {"c": c}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if c["op"] != "shared":
        freq, s["gain"] = frequencies(c)
        s["freq"] = freq.cuda()
    if own:
        from technograd_b200 import kvcache
        if c["op"] != "shared":
            s["rotary"] = kvcache.Rotary(c["dim"], freq=s["freq"], gain=s["gain"], interleaved=c["layout"] == "pairs")
    B, T, D = c["seqs"], c["tokens"], c["dim"]
    if c["op"] == "rope":
        s["x"] = randn(B, T, c["heads"], D).to(dt)
        start = torch.randint(0, 131072, (B, 1), generator=gen, device="cuda")
        s["pos"] = (start + torch.arange(T, device="cuda")).to(torch.int32)
        if c["train"]:
            s["grad"] = randn(B, T, c["heads"], D).to(dt)
        return s
    H, G = c["nkv"], c["group"]
    qkv = randn(B, T, H * G + 2 * H, D)
    if c["op"] == "shared":
        qkv[:, :, :H * G] *= 2  # scores of a few units, as trained heads have them
    # the rows of one projection, queries, keys and values of a token next to each other
    s["q"], s["kn"], s["vn"] = qkv.to(dt).split([H * G, H, H], 2)
    s["count"] = torch.tensor(counts(c), dtype=torch.int32, device="cuda")
    if c["op"] == "append":
        n = lengths(c)
        table, total = table_of([-(-(x + T) // c["page"]) for x in n], gen, host)
        s["max_len"] = c["len"]
        if c["norm"]:
            s["q_norm"], s["k_norm"] = (1 + 0.2 * randn(D) for _ in range(2))
        if c["moved"]:
            start = torch.randint(0, 131072, (B, 1), generator=gen, device="cuda")
            s["pos"] = (start + torch.arange(T, device="cuda")).to(torch.int32)
    else:
        groups, n = grouping(c)
        page = c["page"]
        own_pages, led = [-(-x // page) for x in n], {}
        for first, size, shared in groups:
            for b in range(first + 1, first + size):
                own_pages[b] -= shared // page
                led[b] = first, shared // page
        table, total = table_of(own_pages, gen, host)
        cols = max(1, max(-(-x // page) for x in n))
        wide = torch.full((B, cols), -1, dtype=torch.int32)
        for b in range(B):  # the group's first sequence has the prefix's pages, the others name them too
            lead, k = led.get(b, (b, 0))
            wide[b, k:k + own_pages[b]] = table[b, :own_pages[b]]
            wide[b, :k] = wide[lead, :k]
        table = wide
        s["groups"], s["max_len"] = groups, max(n)
        s["mask"] = tree_masks(c, host).cuda()
    s["k"], s["v"] = pools(c, gen, total)
    s["table"], s["len"] = table.cuda(), torch.tensor(n, dtype=torch.int32, device="cuda")
    if own:
        s["cache"] = kvcache.PagedKV(s["k"], s["v"], s["table"], s["len"], max_len=s["max_len"])
        if c["op"] == "shared":
            s["prefix"] = kvcache.SharedPrefix(s["cache"], s["groups"], max_own=c["tail"])
    return s


def run(s):
    c = s["c"]
    if not own:
        return {"rope": plain_rope, "append": plain_append, "shared": plain_shared}[c["op"]](s)
    from technograd_b200 import kvcache
    if c["op"] == "rope":
        if not c["train"]:
            return kvcache.rope(s["x"], s["rotary"], s["pos"])
        x = s["x"].detach().requires_grad_()
        y = kvcache.rope(x, s["rotary"], s["pos"])
        return y.detach(), torch.autograd.grad(y, x, s["grad"])[0]
    if c["op"] == "append":
        lens, q, k = kvcache.append(s["cache"], s["kn"], s["vn"], q=s["q"] if c["query"] else None, rotary=s["rotary"], pos=s.get("pos"), count=s["count"],
                                    q_norm=s.get("q_norm") if c["query"] else None, k_norm=s.get("k_norm"), eps=EPS, keys=c["keys"])
        return result(s, lens, q, k)
    return kvcache.shared_attention(s["cache"], s["prefix"], s["q"], s["kn"], s["vn"], mask=s["mask"], count=s["count"])


def result(s, lens, q, k):
    """Append: the pools and the lengths, and what else the case asks for."""
    out = {"k": s["k"], "v": s["v"], "len": lens}
    if q is not None:
        out["q_rotated"] = q
    if k is not None:
        out["k_rotated"] = k
    return out


# ---- plain forms: elementary torch operations, 32 bits (angles in 64), rounded once at the end --------

def turn(s, x, pos, inverse=False):
    """x f32 [b][t][heads][dim], rotated."""
    c, half = s["c"], s["c"]["part"] // 2
    angle = pos.double()[..., None] * s["freq"]
    cos, sin = (s["gain"] * angle.cos()).float()[:, :, None], (s["gain"] * angle.sin()).float()[:, :, None]
    if inverse:
        sin = -sin
    out = x.clone()
    one, two = (slice(0, half), slice(half, 2 * half)) if c["layout"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    a, b = x[..., one], x[..., two]
    out[..., one] = a * cos - b * sin
    out[..., two] = a * sin + b * cos
    return out


def plain_rope(s):
    dt = s["x"].dtype
    y = turn(s, s["x"].float(), s["pos"]).to(dt)
    return (y, turn(s, s["grad"].float(), s["pos"], True).to(dt)) if s["c"]["train"] else y


def normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def put(s, pool, rows):
    """rows [b][t][h][dim] into the pool at positions len + t, t < count."""
    c, t = s["c"], torch.arange(s["c"]["tokens"], device="cuda")
    b, i = torch.nonzero(t[None] < s["count"][:, None], as_tuple=True)
    p = s["len"][b].long() + i
    pool[s["table"][b, p // c["page"]].long(), :, p % c["page"]] = rows[b, i]


def plain_append(s):
    c, dt = s["c"], s["kn"].dtype
    pos = s["pos"] if c["moved"] else s["len"][:, None] + torch.arange(c["tokens"], device="cuda")
    k = turn(s, normed(s["kn"].float(), s.get("k_norm")), pos).to(dt)
    q = turn(s, normed(s["q"].float(), s.get("q_norm")), pos).to(dt) if c["query"] else None
    put(s, s["k"], k)
    put(s, s["v"], s["vn"])
    if c["short"]:  # nothing past a sequence's count
        gone = (torch.arange(c["tokens"], device="cuda")[None] >= s["count"][:, None])[..., None, None]
        k, q = k.masked_fill(gone, 0), q.masked_fill(gone, 0) if c["query"] else None
    return result(s, s["len"] + s["count"], q, k if c["keys"] else None)


def rows(pool, table, positions):
    """The cache's rows at positions [b][x] as f32 [b][h][x][dim]."""
    page = pool.shape[2]
    at = table.gather(1, (positions // page).clamp(max=table.shape[1] - 1)).clamp(min=0).long()
    return pool[at, :, positions % page].transpose(1, 2).float()


def plain_shared(s):
    """Group by group: the prefix's scores of all rows at once, then each sequence's own positions and the new tokens."""
    c = s["c"]
    T, H, G, D = c["tokens"], c["nkv"], c["group"], c["dim"]
    out, lse = torch.zeros_like(s["q"].contiguous()), torch.full((c["seqs"], T, H * G), -math.inf, device="cuda")
    covered, spans = 0, []
    for first, size, shared in s["groups"] + [(c["seqs"], 0, 0)]:
        if first > covered:
            spans.append((covered, first - covered, 0))
        if size:
            spans.append((first, size, shared))
        covered = first + size
    t = torch.arange(T, device="cuda")
    for first, size, shared in spans:
        pick = slice(first, first + size)
        table, n, count = s["table"][pick].long(), s["len"][pick], s["count"][pick]
        q = s["q"][pick].float().view(size, T, H, G, D).permute(2, 0, 1, 3, 4).reshape(H, size * T * G, D)
        own_x = shared + torch.arange(c["tail"], device="cuda")[None].expand(size, -1)
        there = own_x < n[:, None]
        k = torch.cat([rows(s["k"], table, own_x), s["kn"][pick].float().transpose(1, 2)], 2)
        v = torch.cat([rows(s["v"], table, own_x) * there[:, None, :, None], s["vn"][pick].float().transpose(1, 2)], 2)
        qb = q.view(H, size, T * G, D).transpose(0, 1)
        z = torch.matmul(qb, k.transpose(2, 3)) * (1 / math.sqrt(D))  # [b][h][t g][own | new]
        bits = (s["mask"][pick][:, :, None] >> t) & 1
        see = torch.cat([there[:, None].expand(size, T, -1), (bits == 1) & (t[None] < count[:, None])[:, None]], 2)
        z = z.masked_fill(~see.repeat_interleave(G, 1)[:, None], -math.inf)
        top = z.max(3, keepdim=True).values
        if shared:
            px = torch.arange(shared, device="cuda")[None]
            pk, pv = rows(s["k"], table[:1], px)[0], rows(s["v"], table[:1], px)[0]
            zp = (torch.matmul(q, pk.transpose(1, 2)) * (1 / math.sqrt(D))).view(H, size, T * G, shared).transpose(0, 1)
            top = torch.maximum(top, zp.max(3, keepdim=True).values)
        ref = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(z - ref)
        total, o = p.sum(3, keepdim=True), torch.matmul(p, v)
        if shared:
            p = torch.exp(zp - ref)
            total = total + p.sum(3, keepdim=True)
            o = o + torch.matmul(p.transpose(0, 1).reshape(H, size * T * G, shared), pv).view(H, size, T * G, D).transpose(0, 1)
        o = o / torch.where(total == 0, torch.ones_like(total), total)
        live = (t[None] < count[:, None])[..., None]
        o = o.view(size, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(size, T, H * G, D)
        z = (top + torch.log(total))[..., 0].view(size, H, T, G).permute(0, 2, 1, 3).reshape(size, T, H * G)
        out[pick] = torch.where(live[..., None], o, torch.zeros_like(o)).to(out.dtype)
        lse[pick] = torch.where(live, z, torch.full_like(z, -math.inf))
    return out, lse


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    half, B, T, D = c.get("part", 0) // 2, c["seqs"], c["tokens"], c["dim"]

    def spun(x, pos, sign=1):
        """Each pair as a complex number, times gain e^(i angle)."""
        w = torch.polar(torch.full((B, T, half), s["gain"], dtype=torch.float64, device="cuda"), sign * pos.double()[:, :, None] * s["freq"][None, None])[:, :, None]
        y = x.double().clone()
        if c["layout"] == "half":
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * w
            y[..., :half], y[..., half:2 * half] = z.real, z.imag
        else:
            z = torch.complex(y[..., 0:2 * half:2].contiguous(), y[..., 1:2 * half:2].contiguous()) * w
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
        return y

    if c["op"] == "rope":
        y = spun(s["x"], s["pos"])
        return (y, spun(s["grad"], s["pos"], -1)) if c["train"] else y
    n, count = s["len"].tolist(), s["count"].tolist()
    if c["op"] == "append":
        pos = s["pos"] if c["moved"] else torch.tensor([[x + t for t in range(T)] for x in n], device="cuda")

        def scaled(x, w):
            x = x.double()
            return x if w is None else x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()

        k = spun(scaled(s["kn"], s.get("k_norm")), pos)
        q = spun(scaled(s["q"], s.get("q_norm")), pos)
        pk, pv = s["k"].double(), s["v"].double()
        for b in range(B):
            p = torch.arange(n[b], n[b] + count[b], device="cuda")
            g = s["table"][b][p // c["page"]].long()
            pk[g, :, p % c["page"]], pv[g, :, p % c["page"]] = k[b, :count[b]], s["vn"][b, :count[b]].double()
        out = {"k": pk, "v": pv, "len": s["len"] + s["count"]}
        gone = torch.arange(T, device="cuda")[None] >= s["count"][:, None]
        if c["query"]:
            out["q_rotated"] = q.masked_fill(gone[..., None, None], 0)
        if c["keys"]:
            out["k_rotated"] = k.masked_fill(gone[..., None, None], 0)
        return out
    G, mask, outs, lses = c["group"], s["mask"].tolist(), [], []

    def cached(pool, b):
        p = torch.arange(n[b], device="cuda")
        return pool[s["table"][b][p // c["page"]].long(), :, p % c["page"]].double()  # [len][h][dim]

    for b in range(B):
        m = count[b]
        k, v = (torch.cat([cached(s[x], b), s[y][b, :m].double()]) for x, y in (("k", "kn"), ("v", "vn")))
        q = s["q"][b, :m].double().view(m, c["nkv"], G, D)
        z = torch.einsum("thgd,xhd->hgtx", q, k) / D ** 0.5
        see = torch.ones(m, n[b] + m, dtype=torch.bool)
        for t in range(m):
            see[t, n[b]:] = torch.tensor([mask[b][t] >> u & 1 == 1 for u in range(m)], dtype=torch.bool)
        z = z.masked_fill(~see.cuda(), -math.inf)
        lse = torch.logsumexp(z, 3)
        o = torch.zeros(T, c["nkv"] * G, D, dtype=torch.float64, device="cuda")
        o[:m] = torch.einsum("hgtx,xhd->thgd", torch.exp(z - lse[..., None]), v).reshape(m, c["nkv"] * G, D)
        full = torch.full((T, c["nkv"] * G), -math.inf, dtype=torch.float64, device="cuda")
        full[:m] = lse.permute(2, 0, 1).reshape(m, c["nkv"] * G)
        outs.append(o)
        lses.append(full)
    return torch.stack(outs), torch.stack(lses)
