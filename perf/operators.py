"""Workloads of the paged key/value cache operators: attention of drafted tokens, accumulation of
attention weight, commit of accepted tokens, eviction.

`own` selects between the plain forms below (elementary torch operations in f32) and the calls of
technograd_b200.kvcache. A case names an operator (`op`) and its sizes:

  seqs, nkv, group, dim   sequences, key/value heads, query heads per key/value head, head dimension
  len, ragged             the longest sequence's positions in the cache; ragged: the others are shorter, down to empty
  page, order             positions per page; "head": pools [pages][nkv][page][dim], "pos": [pages][page][nkv][dim]
  type                    f32, f16 or bf16, of the cache and of everything attended with it
  tokens, tree            drafted tokens per sequence; "chain", "tree", or "holes" (some tokens see nothing drafted)
  short                   true where sequences have drafted fewer tokens than `tokens`
  budget, recent, sink    eviction: positions kept per head, of them the last and the first ones always
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
QWEN = dict(nkv=8, group=2, dim=128)  # the Qwen3-0.6B attention layer: 16 query heads over 8


def listed():
    return [
        # one user, one token, a short prompt: the latency of a decode step's attention
        dict(name="attend-one", op="attend", seqs=1, len=97, ragged=False, page=16, order="head", type="bf16", tokens=1,
             tree="chain", short=False, **QWEN),
        # the 8-sequence decode wave (1024-token prompts, 256 new tokens), in the framework's own f32
        dict(name="attend-wave-f32", op="attend", seqs=8, len=1280, ragged=True, page=64, order="head", type="f32", tokens=1,
             tree="chain", short=False, **QWEN),
        # the same wave verifying trees of drafted tokens
        dict(name="attend-tree", op="attend", seqs=8, len=1280, ragged=True, page=24, order="pos", type="bf16", tokens=21,
             tree="tree", short=True, **QWEN),
        # a full server: many ragged sequences, the largest trees
        dict(name="attend-server", op="attend", seqs=48, len=6001, ragged=True, page=64, order="head", type="bf16", tokens=64,
             tree="tree", short=True, **QWEN),
        # one long document, eight query heads per key head
        dict(name="attend-long", op="attend", seqs=1, nkv=4, group=8, dim=128, len=131009, ragged=False, page=16,
             order="head", type="f16", tokens=5, tree="holes", short=False),
        # a large decode wave, one token each
        dict(name="attend-decode", op="attend", seqs=256, len=1280, ragged=True, page=16, order="pos", type="bf16", tokens=1,
             tree="chain", short=False, **QWEN),
        # the weight a decode step of that small wave puts on each cached position
        dict(name="weigh-wave", op="weigh", seqs=8, len=1280, ragged=True, page=64, order="head", type="bf16", tokens=1,
             tree="chain", short=False, **QWEN),
        # the weight of an observation window of the last tokens of long prompts
        dict(name="weigh-window", op="weigh", seqs=16, len=16001, ragged=True, page=24, order="pos", type="f16", tokens=32,
             tree="chain", short=False, **QWEN),
        # eviction in a toy model: small heads, odd pages
        dict(name="evict-small", op="evict", seqs=2, nkv=2, group=2, dim=8, len=301, ragged=False, page=5, order="head",
             type="f32", budget=200, recent=31, sink=4),
        # eviction from long caches to an eighth
        dict(name="evict-long", op="evict", seqs=24, len=32001, ragged=True, page=64, order="head", type="bf16", budget=4000,
             recent=256, sink=4, **QWEN),
        # accepted tokens of the drafted trees into the cache
        dict(name="commit-tree", op="commit", seqs=8, len=1280, ragged=True, page=24, order="pos", type="bf16", tokens=21,
             tree="tree", short=True, **QWEN),
        # the keys and values of whole prompts into the cache
        dict(name="commit-prompt", op="commit", seqs=32, len=0, ragged=False, page=64, order="head", type="f32", tokens=1024,
             tree="chain", short=False, **QWEN),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "weigh", "evict", "commit"])
    c = dict(op=op, seqs=spread(1, 64), nkv=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 3, 4, 8]),
             dim=rng.choice([8, 64, 80, 96, 128, 128, 128, 256]), len=spread(1, 131072), ragged=rng.random() < 0.6,
             page=rng.choice([1, 5, 16, 16, 24, 64, 128]), order=rng.choice(["head", "pos"]),
             type=rng.choice(["f32", "f16", "bf16"]))
    if op == "evict":
        c["budget"] = max(1, int(c["len"] * rng.uniform(0.05, 1.1)))
        c["recent"] = int(c["budget"] * rng.uniform(0, 0.6))
        c["sink"] = min(rng.choice([0, 4]), c["budget"] - c["recent"])
    else:
        c["tokens"] = rng.choice([1, spread(1, 64), spread(1, 64)])
        c["tree"] = rng.choice(["chain", "tree", "holes"]) if c["tokens"] > 1 else "chain"
        c["short"] = rng.random() < 0.5
        if op == "commit":
            c["tokens"] = rng.choice([c["tokens"], spread(64, 2048)])
    def cost(x):  # bytes, operations, scores that a plain form holds, and the pools' size
        w, total = work(x), sum(lengths(x))
        held = total * x["nkv"] * x["group"] * x["tokens"] if w["flops"] and "tokens" in x else 0
        return w["bytes"], w["flops"], held, 2 * SIZE[x["type"]] * total * x["nkv"] * x["dim"]

    alike = [cost(x) for x in listed() if x["op"] == op]
    most = [max(x[i] for x in alike) for i in range(3)] + [max(cost(x)[3] for x in listed())]
    while True:  # no dearer than the dearest listed case of its operator
        if all(x <= y for x, y in zip(cost(c), most)):
            return c
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        else:
            c["len"] = (c["len"] + 1) // 2
            if op == "evict":
                c["budget"], c["recent"] = (c["budget"] + 1) // 2, c["recent"] // 2
                c["sink"] = min(c["sink"], c["budget"] - c["recent"])


def lengths(c):
    """Positions that each sequence has in the cache: the same for every seed."""
    r = random.Random(c["seqs"] * 1000003 + c["len"])
    n = [c["len"]] * c["seqs"]
    if c["ragged"]:
        n[1:] = [r.randint(c["len"] // 2, c["len"]) for _ in n[1:]]
        if len(n) >= 4:
            n[2], n[3] = min(1, c["len"]), 0
    return n


def counts(c):
    """Drafted (commit: accepted) tokens of each sequence."""
    r = random.Random(c["seqs"] * 7919 + c["tokens"])
    return [r.randint(c["tokens"] // 2, c["tokens"]) for _ in range(c["seqs"])] if c["short"] else [c["tokens"]] * c["seqs"]


def work(c):
    e, n, d = SIZE[c["type"]], lengths(c), c["dim"]
    total, rows = sum(n), c["nkv"] * d
    pages = 4 * sum(-(-x // c["page"]) for x in n)
    if c["op"] == "evict":
        kept = sum(min(x, c["budget"]) for x in n)
        return {"bytes": 4 * c["nkv"] * total + 4 * e * rows * kept + 8 * c["nkv"] * c["seqs"] * c["budget"] + pages, "flops": c["nkv"] * total}
    t = counts(c)
    if c["op"] == "commit":
        return {"bytes": 4 * e * rows * sum(t) + 8 * c["nkv"] * sum(t) + 4 * sum(t), "flops": 0}
    drafted, nq = c["seqs"] * c["tokens"], c["nkv"] * c["group"]
    pairs = sum(k * (x + 1) for k, x in zip(t, n))
    small = pages + 8 * drafted + 4 * drafted * nq
    if c["op"] == "weigh":
        return {"bytes": e * rows * (total + drafted) + e * drafted * nq * d + 4 * c["nkv"] * (total + c["seqs"] * c["len"] + drafted) + small,
                "flops": 2 * d * nq * pairs}
    return {"bytes": 2 * e * rows * (total + drafted) + 2 * e * drafted * nq * d + small, "flops": 4 * d * nq * pairs}


def tree_masks(c, gen):
    """Bit u of [b][t]: token t sees drafted token u. A tree's token sees its ancestors and itself."""
    T, out = c["tokens"], []
    pick = torch.randint(0, 1 << 30, (c["seqs"], T), generator=gen).tolist()
    for row in pick:
        m = []
        for t, x in enumerate(row):
            if c["tree"] == "chain":
                m.append((1 << (t + 1)) - 1)
            elif c["tree"] == "tree":
                parent = x % (t + 1) - 1
                m.append((m[parent] if parent >= 0 else 0) | 1 << t)
            else:
                m.append(0 if x % 3 == 0 else (x * 0x9E3779B97F4A7C15 >> 7) & ((1 << T) - 1))
        out.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(out, dtype=torch.int64)


def pools(c, gen, positions, fill):
    """A pool of randomly placed pages that hold `positions` of each sequence, and its table (-1 where no page is)."""
    need = [-(-x // c["page"]) for x in positions]
    cols, total = max(1, max(need)), max(1, sum(need))
    where = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")[:, None]
    col = torch.arange(cols, device="cuda")[None]
    have = col < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(have, where[(first + col).clamp(max=total - 1)], torch.tensor(-1, dtype=torch.int32, device="cuda"))
    shape = (total, c["nkv"], c["page"], c["dim"]) if c["order"] == "head" else (total, c["page"], c["nkv"], c["dim"])
    made = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=TYPES[c["type"]]) if fill else torch.zeros(shape, device="cuda", dtype=TYPES[c["type"]])
        made.append(x if c["order"] == "head" else x.transpose(1, 2))
    return made[0], made[1], table.contiguous()


def prepare(c, seed):
    gen, host = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    n, dt = lengths(c), TYPES[c["type"]]
    s = {"c": c, "len": torch.tensor(n, dtype=torch.int32, device="cuda"), "max_len": c["len"]}
    room = [x + (c["tokens"] if c["op"] == "commit" else 0) for x in n]
    s["k"], s["v"], s["table"] = pools(c, gen, room, True)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if c["op"] != "evict":
        B, T, H, G, D = c["seqs"], c["tokens"], c["nkv"], c["group"], c["dim"]
        s["count"] = torch.tensor(counts(c), dtype=torch.int32, device="cuda")
        s["kn"], s["vn"] = randn(B, T, H, D).to(dt), randn(B, T, H, D).to(dt)
    if c["op"] in ("attend", "weigh"):
        s["q"] = (2 * randn(B, T, H * G, D)).to(dt)  # scores of a few units, as trained heads have them
        s["mask"] = tree_masks(c, host).cuda()
    if c["op"] == "weigh":
        s["lse"] = plain_attend(s)[1]
        s["select"] = torch.full((B,), -1, dtype=torch.int64, device="cuda")
        s["acc"] = randn(B, H, c["len"]).abs()
    if c["op"] == "commit":
        # the accepted path: so many of the drafted tokens, ascending; a prompt is taken whole
        taken = torch.arange(T)[None] < torch.tensor(counts(c))[:, None]
        path = torch.where(taken, torch.rand(B, T, generator=host).argsort(1), torch.tensor(T)).sort(1).values
        s["path"] = torch.where(taken, path, torch.tensor(-1)).to(torch.int32).cuda()
        s["new"], s["acc"] = randn(B, H, T).abs(), randn(B, H, c["len"] + T).abs()
    if c["op"] == "evict":
        # attention weight falls off as a power law, and some positions have exactly the same
        w = torch.exp(2 * randn(c["seqs"], c["nkv"], max(1, c["len"])))
        s["acc"] = torch.where(w < 0.5, (w * 8).floor() / 8, w)
        s["k2"], s["v2"], s["table2"] = pools(c, gen, [min(x, c["budget"]) for x in n], False)
    if own:
        from technograd_b200 import kvcache
        s["cache"] = kvcache.PagedKV(s["k"], s["v"], s["table"], s["len"], max_len=c["len"])
        if c["op"] == "evict":
            s["dst"] = kvcache.PagedKV(s["k2"], s["v2"], s["table2"], torch.zeros_like(s["len"]), max_len=0)
    return s


def run(s):
    op = s["c"]["op"]
    if own:
        from technograd_b200 import kvcache
        if op == "attend":
            return kvcache.tree_attention(s["cache"], s["q"], s["kn"], s["vn"], mask=s["mask"], count=s["count"])
        if op == "weigh":
            return kvcache.attention_weights(s["cache"], s["q"], s["kn"], s["lse"], mask=s["mask"], count=s["count"],
                                             select=s["select"], acc=s["acc"])
        if op == "commit":
            n = kvcache.commit(s["cache"], s["kn"], s["vn"], s["count"], path=s["path"], new=s["new"], acc=s["acc"])
            return s["k"], s["v"], s["acc"], n
        keep, acc, n = kvcache.evict(s["cache"], s["dst"], s["acc"], s["c"]["budget"], recent=s["c"]["recent"], sink=s["c"]["sink"])
        return s["k2"], s["v2"], keep, acc, n
    return {"attend": plain_attend, "weigh": plain_weigh, "commit": plain_commit, "evict": plain_evict}[op](s)


# ---- plain forms: elementary torch operations, 32 bits, rounded once at the end ----------------------

def rows(pool, table, positions):
    """The cache's rows at positions [b][h][x] (or [b][1][x]) as f32 [b][h][x][dim]."""
    page = pool.shape[2]
    b = torch.arange(table.shape[0], device=table.device)[:, None, None]
    at = table[b, (positions // page).clamp(max=table.shape[1] - 1)].clamp(min=0).long()
    h = torch.arange(pool.shape[1], device=table.device)[None, :, None]
    return pool[at, h, positions % page].float()


def scores(s):
    """Scores [b][h][token * group][cached | drafted] in f32, -inf where a token does not look; and the cached
    positions' presence."""
    c = s["c"]
    B, T, H, G, D = c["seqs"], c["tokens"], c["nkv"], c["group"], c["dim"]
    x = torch.arange(s["max_len"], device="cuda")
    k = rows(s["k"], s["table"], x[None, None].expand(B, 1, -1))
    there = x[None] < s["len"][:, None]
    q = s["q"].float().view(B, T, H, G, D).transpose(1, 2).reshape(B, H, T * G, D)
    k = torch.cat([k, s["kn"].float().transpose(1, 2)], 2)
    z = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(D))
    bits = (s["mask"][:, :, None] >> torch.arange(T, device="cuda")) & 1
    token = torch.arange(T, device="cuda")
    live = token[None] < s["count"][:, None]
    see = torch.cat([there[:, None].expand(B, T, -1), (bits == 1) & live[:, None, :]], 2) & live[:, :, None]
    return z.masked_fill_(~see.repeat_interleave(G, 1)[:, None], -math.inf), there


def plain_attend(s):
    c = s["c"]
    B, T, H, G, D = c["seqs"], c["tokens"], c["nkv"], c["group"], c["dim"]
    z, there = scores(s)
    top = z.max(3, keepdim=True).values
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del z
    total = p.sum(3, keepdim=True)
    x = torch.arange(s["max_len"], device="cuda")
    v = torch.cat([rows(s["v"], s["table"], x[None, None].expand(B, 1, -1)) * there[:, None, :, None], s["vn"].float().transpose(1, 2)], 2)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total))[..., 0].view(B, H, T, G).transpose(1, 2).reshape(B, T, H * G)
    return o.view(B, H, T, G, D).transpose(1, 2).reshape(B, T, H * G, D).to(s["q"].dtype), lse


def plain_weigh(s):
    c = s["c"]
    B, T, H, G = c["seqs"], c["tokens"], c["nkv"], c["group"]
    z, there = scores(s)
    lse = s["lse"].view(B, T, H, G).transpose(1, 2).reshape(B, H, T * G, 1)
    counted = ((s["select"][:, None] >> torch.arange(T, device="cuda")) & 1 == 1).repeat_interleave(G, 1)[:, None, :, None]
    w = torch.exp(z - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)).masked_fill_(~counted | (lse == -math.inf), 0).sum(2)
    n = s["max_len"]
    return torch.where(there[:, None], s["acc"] + w[:, :, :n], torch.zeros_like(s["acc"])), w[:, :, n:].contiguous()


def put(pool, table, positions, wanted, values):
    """values [b][h][x][dim] into the cache's rows at positions [b][h][x] where wanted."""
    page = pool.shape[2]
    b, h, x = torch.nonzero(wanted, as_tuple=True)
    p = positions[b, h, x]
    pool[table[b, p // page].long(), h, p % page] = values[b, h, x]


def plain_commit(s):
    c = s["c"]
    B, T, H, D = c["seqs"], c["tokens"], c["nkv"], c["dim"]
    i = torch.arange(T, device="cuda")[None, None].expand(B, H, T)
    wanted = i < s["count"][:, None, None]
    at = s["len"][:, None, None].long() + i
    path = s["path"].long().clamp(min=0)[:, None].expand(B, H, T)
    for pool, new in ((s["k"], s["kn"]), (s["v"], s["vn"])):
        put(pool, s["table"], at, wanted, new.transpose(1, 2).gather(2, path[..., None].expand(B, H, T, D)))
    b, h, x = torch.nonzero(wanted, as_tuple=True)
    s["acc"][b, h, at[b, h, x]] = s["new"].gather(2, path)[b, h, x]
    return s["k"], s["v"], s["acc"], s["len"] + s["count"]


def plain_evict(s):
    c = s["c"]
    B, H, n, budget = c["seqs"], c["nkv"], s["max_len"], c["budget"]
    x = torch.arange(n, device="cuda")[None, None].expand(B, H, n)
    length = s["len"].long()[:, None, None]
    always = (x < c["sink"]) | (x >= length - c["recent"]) | (length <= budget)
    key = s["acc"].masked_fill(always, math.inf).masked_fill(x >= length, -math.inf)
    best = torch.sort(key, dim=2, descending=True, stable=True).indices[:, :, :budget]
    kept = torch.minimum(length, torch.tensor(budget, device="cuda"))
    wide = best.shape[2]
    i = torch.arange(wide, device="cuda")[None, None]
    keep = torch.sort(torch.where(i < kept, best, torch.tensor(n, device="cuda")), 2).values
    wanted = (i < kept).expand(B, H, wide)
    from_ = keep.clamp(max=n - 1)
    page, table = s["k"].shape[2], s["table"]
    b, h = torch.arange(B, device="cuda")[:, None, None], torch.arange(H, device="cuda")[None, :, None]
    at = table[b, from_ // page].clamp(min=0).long()
    for src, dst in ((s["k"], s["k2"]), (s["v"], s["v2"])):
        put(dst, s["table2"], i.expand(B, H, wide), wanted, src[at, h, from_ % page])
    acc = torch.zeros(B, H, budget, device="cuda")
    acc[:, :, :wide] = torch.where(wanted, s["acc"].gather(2, from_), torch.zeros_like(acc[:, :, :wide]))
    out = torch.full((B, H, budget), -1, dtype=torch.int32, device="cuda")
    out[:, :, :wide] = torch.where(wanted, keep, torch.tensor(-1, device="cuda")).int()
    return s["k2"], s["v2"], out, acc, torch.clamp(s["len"], max=budget)


# ---- the definitions in 64 bits, sequence by sequence ------------------------------------------------

def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    n = s["len"].tolist()

    def cached(pool, b, upto):
        p = torch.arange(upto, device="cuda")
        at = s["table"][b][p // c["page"]].long()
        return pool[at, :, p % c["page"]].double()  # [upto][h][dim]

    if c["op"] in ("commit", "evict"):
        return None  # copies and selections: no arithmetic
    G, t_all, D = c["group"], c["tokens"], c["dim"]
    count, mask = s["count"].tolist(), s["mask"].tolist()
    outs, lses, accs, news = [], [], [], []
    for b in range(c["seqs"]):
        T = count[b]
        k = torch.cat([cached(s["k"], b, n[b]), s["kn"][b, :T].double()]).repeat_interleave(G, 1)  # [x][nq][D]
        q = s["q"][b, :T].double()
        z = torch.einsum("tjd,xjd->jtx", q, k) / D ** 0.5
        see = torch.ones(T, n[b] + T, dtype=torch.bool)
        for t in range(T):
            see[t, n[b]:] = torch.tensor([mask[b][t] >> u & 1 == 1 for u in range(T)], dtype=torch.bool)
        z = torch.where(see.cuda()[None], z, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
        if c["op"] == "attend":
            v = torch.cat([cached(s["v"], b, n[b]), s["vn"][b, :T].double()]).repeat_interleave(G, 1)
            lse = torch.logsumexp(z, 2)
            w = torch.nan_to_num(torch.exp(z - lse[:, :, None]), nan=0.0)
            o = torch.zeros(t_all, q.shape[1], D, dtype=torch.float64, device="cuda")
            o[:T] = torch.einsum("jtx,xjd->tjd", w, v)
            full = torch.full((t_all, q.shape[1]), -math.inf, dtype=torch.float64, device="cuda")
            full[:T] = lse.T
            outs.append(o)
            lses.append(full)
        else:
            lse = s["lse"][b, :T].double().T[:, :, None]
            w = torch.nan_to_num(torch.exp(z - lse), nan=0.0, posinf=0.0).sum(1).view(c["nkv"], G, -1).sum(1)
            acc = torch.zeros(c["nkv"], c["len"], dtype=torch.float64, device="cuda")
            acc[:, :n[b]] = s["acc"][b, :, :n[b]].double() + w[:, :n[b]]
            new = torch.zeros(c["nkv"], t_all, dtype=torch.float64, device="cuda")
            new[:, :T] = w[:, n[b]:]
            accs.append(acc)
            news.append(new)
    return (torch.stack(outs), torch.stack(lses)) if outs else (torch.stack(accs), torch.stack(news))
