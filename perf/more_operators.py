"""Operators of a serving program that drafts tokens, samples and keeps its
cache in 8 bits, as cases to time.

Keys and values live in pages: k [layer][page][head][row][value] and v
[layer][page][head][value][row], a table of page ids per sequence; pools of
8 bits (whole numbers or e4m3) have a scale per row and head.  A step with drafted tokens
writes every node's key and value rows behind its sequence, lets each node
attend to the sequence and to its ancestors, samples a token at every node,
follows the drafted tokens that the samples agree with and keeps their rows.

Kinds of case (the "kind" field):
  write8  new key and value rows into 8-bit pages, and those rows read back
  attn8   attention of one new token per row over 8-bit pages
  tree    attention of several new tokens per sequence: trees (a mask) or
          chunks of prompts (each row sees those before it)
  sample  a token per row of logits: temperature, top-k, min-p, top-p
  keep    the accepted path of every tree, and its rows moved together

The plain forms compute in 32 bits with elementary torch operations (samples,
whose cumulative sums decide between tokens, in 64); `exact` computes from the
definitions in 64.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
TOP = {"i8": 127.0, "e4m3": 448.0}  # what a scale's row and head reach at most
VOCAB = 51866


# ----------------------------------------------------------------- cases

def listed():
    return [
        # a step's new rows of a batch, from a fused projection's output
        dict(name="write8_step", kind="write8", type="i8", seqs=64, new=1, past=447, heads=20, head=64, page=32),
        # prompts of a batch: 24 windows of 1500 rows that start inside a page
        dict(name="write8_prompts", kind="write8", type="e4m3", seqs=24, new=1500, past=9, heads=20, head=64, page=32),
        # one short utterance, a tiny model's decoder: a call's own latency
        dict(name="attn8_one_short", kind="attn8", type="i8", trees=1, nodes=1, heads=6, group=1, head=64, page=16, past=27,
             lens="full", form="token"),
        # a served batch with grouped heads, lengths of a few thousand, some slots empty
        dict(name="attn8_batch", kind="attn8", type="e4m3", trees=61, nodes=1, heads=8, group=4, head=128, page=64, past=8190,
             lens="ragged", form="token"),
        # one small tree of a tiny model: latency
        dict(name="tree_one_small", kind="tree", type="f32", trees=1, nodes=13, heads=6, group=1, head=64, page=16, past=101,
             lens="full", form="tree"),
        # a served batch whose sequences have trees of all sizes, grouped heads, an 8-bit cache
        dict(name="tree_batch", kind="tree", type="i8", trees=24, nodes=48, heads=8, group=4, head=128, page=64, past=6000,
             lens="ragged", form="tree"),
        # chunks of prompts whose first parts are in the cache
        dict(name="tree_chunks", kind="tree", type="bf16", trees=4, nodes=512, heads=8, group=4, head=128, page=128,
             past=4100, lens="full", form="chain"),
        # one token of one sequence
        dict(name="sample_one", kind="sample", type="f32", rows=1, vocab=VOCAB, temperature=0.8, top_k=40, top_p=0.95,
             min_p=0.0, mixed=False),
        # a served batch, each row with settings of its own, some greedy
        dict(name="sample_batch", kind="sample", type="bf16", rows=61, vocab=VOCAB, temperature=1.0, top_k=50, top_p=0.9,
             min_p=0.05, mixed=True),
        # every node of a batch's trees, by top-p alone
        dict(name="sample_nodes", kind="sample", type="f32", rows=768, vocab=VOCAB, temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.0, mixed=False),
        # one tree of a small model
        dict(name="keep_one", kind="keep", type="f32", trees=1, nodes=13, layers=4, heads=6, head=64, page=16, past=101),
        # the trees of a served batch, every layer
        dict(name="keep_batch", kind="keep", type="f16", trees=48, nodes=48, layers=24, heads=8, head=128, page=64, past=120),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write8", "attn8", "attn8", "tree", "tree", "tree", "sample", "sample", "keep"))
    heads, head = rng.choice((1, 2, 3, 5, 6, 8, 12, 16, 20)), rng.choice((32, 64, 96, 128))
    page = rng.choice((16, 32, 64, 128, 256))
    group = rng.choice((1, 1, 2, 4, 5, 7, 8, 16, 20))
    n = heads * head
    if kind == "write8":
        seqs = _log_int(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(2, min(2000, (36000 * 1280) // (seqs * n))))
        return dict(kind=kind, type=rng.choice(("i8", "e4m3")), seqs=seqs, new=new, past=_log_int(rng, 1, 1000) - 1, heads=heads,
                    head=head, page=page)
    if kind == "attn8":
        rows = _log_int(rng, 1, 96)
        top = max(64, min(131071, 500_000_000 // (rows * 2 * n)))
        return dict(kind=kind, type=rng.choice(("i8", "e4m3")), trees=rows, nodes=1, heads=heads, group=group, head=head, page=page,
                    past=_log_int(rng, 1, top), lens=rng.choice(("ragged", "ragged", "full")), form="token")
    if kind == "tree":
        trees = _log_int(rng, 1, 48)
        form = rng.choice(("tree", "tree", "chain"))
        nodes = _log_int(rng, 1, 96 if form == "tree" else max(2, min(900, 2000 // trees)))
        group = min(group, 8)
        # no more products than the largest listed case, and room for the plain form's scores
        top = min(16000, 30_000_000_000 // (trees * nodes * n * group), 300_000_000 // (trees * nodes * heads * group),
                  120_000_000 // (trees * n))
        return dict(kind=kind, type=rng.choice(tuple(TYPES)), trees=trees, nodes=nodes, heads=heads, group=group, head=head,
                    page=page, past=_log_int(rng, 1, max(2, top)) - 1, lens=rng.choice(("ragged", "ragged", "full")), form=form)
    if kind == "sample":
        vocab = rng.choice((VOCAB, 51865, _log_int(rng, 100, 260000)))
        return dict(kind=kind, type=rng.choice(("f32", "f16", "bf16")), rows=_log_int(rng, 1, max(2, min(768, 39_000_000 // vocab))),
                    vocab=vocab, temperature=rng.choice((0.0, 0.3, 0.7, 1.0, 1.0, 1.3)), top_k=rng.choice((0, 0, 1, 20, 50, 400)),
                    top_p=rng.choice((1.0, 0.5, 0.9, 0.95)), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)), mixed=rng.random() < 0.5)
    trees, layers = _log_int(rng, 1, 48), rng.choice((4, 6, 12, 24))
    nodes = _log_int(rng, 1, 96)
    kind_type = rng.choice(("f32", "f16", "bf16"))
    top = max(1, 2_400_000_000 // (trees * layers * n * SIZE[kind_type] * 2) - nodes - 256)
    return dict(kind=kind, type=kind_type, trees=trees, nodes=nodes, layers=layers, heads=heads, head=head, page=page,
                past=_log_int(rng, 1, max(2, min(500, top))) - 1)


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(shape, dtype, g):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _floats(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(DEV)


def _pool(kind, layers, pages, heads, page, dim, g):
    """k, v and, for 8 bits, their scales."""
    shapes = (layers, pages, heads, page, dim), (layers, pages, heads, dim, page)
    if kind not in TOP:
        k, v = (_normal(s, TYPES[kind], g) for s in shapes)
        return dict(k=k, v=v)
    top = TOP[kind]
    k, v = ((_normal(s, torch.bfloat16, g) * (0.28 * top)).round().clamp(-top, top).to(TYPES[kind]) for s in shapes)
    ks, vs = (torch.empty(shapes[0][:4], device=DEV).uniform_(2.0 / top, 5.0 / top, generator=g) for _ in range(2))
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def _tables(lens, page, rng, spare=3, width=None):
    """Page ids per sequence, in random order, and how many pages the pool has."""
    used = -(-np.asarray(lens) // page)
    n_pages = int(used.sum()) + spare
    free, at = rng.permutation(n_pages), 0
    table = np.zeros((len(lens), max(1, width or int(used.max()))), np.int32)
    for i, u in enumerate(used):
        table[i, :u] = free[at : at + u]
        at += u
    return table, n_pages


def _ragged(top, n, rng):
    lens = np.round(np.exp(rng.uniform(0, math.log(top + 1), n))).astype(np.int64) - 1  # 0 .. top, most of them short
    long = rng.random(n) < 0.5
    lens[long] = rng.integers(top // 4, top + 1, int(long.sum()))
    lens[int(rng.integers(n))] = top
    return lens


def _sizes(count, least, most):
    """Rows of each of a call's trees, unlike each other and the same for every seed: a case has one number of rows."""
    fixed = np.random.default_rng(1000 * count + most)
    sizes = fixed.integers(least, most + 1, count)
    sizes[int(fixed.integers(count))] = most
    return sizes


def _parents(sizes, rng):
    """Per tree and node its parent (root: -1): nodes come level by level, up to 8 to a level."""
    parents = []
    for n in sizes:
        p, level = [-1], [0]
        while len(p) < n:
            new = range(len(p), min(int(n), len(p) + int(rng.integers(2, 9))))
            p.extend(int(rng.choice(level)) for _ in new)
            level = list(new)
        parents.append(p)
    return parents


def _mask(sizes, parents):
    """int32 words per row: bit j of row r is set where r's tree lets it see node j, an ancestor or itself."""
    words = -(-int(sizes.max()) // 32)
    mask = np.zeros((int(sizes.sum()), words), np.uint32)
    r0 = 0
    for p in parents:
        for j, up in enumerate(p):
            if up >= 0:
                mask[r0 + j] = mask[r0 + up]
            mask[r0 + j, j >> 5] |= np.uint32(1 << (j & 31))
        r0 += len(p)
    return mask.view(np.int32)


def prepare(case, seed):
    c, rng, g = case, np.random.default_rng(int(seed)), _gen(seed)
    if c["kind"] == "sample":
        rows, vocab = c["rows"], c["vocab"]
        logits = _normal((rows, vocab), torch.float32, g) * 2.5
        logits[:, ::37] = -math.inf  # suppressed tokens
        s = dict(case=c, logits=logits.to(TYPES[c["type"]]), u=_floats(rng.random(rows, dtype=np.float32)))
        temperature, top_k = np.full(rows, c["temperature"]), np.full(rows, c["top_k"])
        top_p, min_p = np.full(rows, c["top_p"]), np.full(rows, c["min_p"])
        if c["mixed"]:
            temperature = temperature * rng.choice((0.0, 0.5, 1.0, 1.2), rows)
            top_k = np.where(rng.random(rows) < 0.5, top_k, 0)
            top_p = np.where(rng.random(rows) < 0.5, top_p, 1.0)
            min_p = np.where(rng.random(rows) < 0.5, min_p, 0.0)
        s.update(temperature=_floats(temperature), top_k=_ints(top_k), top_p=_floats(top_p), min_p=_floats(min_p))
        return s
    P, H, D = c["page"], c["heads"], c["head"]
    if c["kind"] == "write8":
        total = c["past"] + c["new"]
        table, n_pages = _tables(np.full(c["seqs"], total), P, rng)
        seq = np.repeat(np.arange(c["seqs"]), c["new"])
        pos = np.tile(c["past"] + np.arange(c["new"]), c["seqs"])
        s = dict(case=c, qkv=_normal((c["seqs"] * c["new"], 3 * H * D), torch.float32, g), table=_ints(table), seq=_ints(seq),
                 pos=_ints(pos), **_pool(c["type"], 2, n_pages, H, P, D, g))
        s["qkv"] *= torch.rand(len(pos), 1, device=DEV, generator=g) * 3 + 0.1  # rows of unlike size
        return s
    if c["kind"] in ("attn8", "tree"):
        n = c["trees"]
        past = np.full(n, c["past"]) if c["lens"] == "full" else _ragged(c["past"], n, rng)
        if c["form"] == "token":
            sizes, lens = np.ones(n, np.int64), past  # the token's own row is among them
        else:
            least = c["nodes"] if c["lens"] == "full" else max(1, c["nodes"] // 4) if c["form"] == "tree" else 0
            sizes = _sizes(n, least, c["nodes"])
            lens = past + sizes
        table, n_pages = _tables(lens, P, rng)
        seq = rng.permutation(n)  # trees in another order than the table's
        s = dict(case=c, q=_normal((int(sizes.sum()), H * c["group"] * D), torch.float32, g) * 2.0, table=_ints(table),
                 seq=_ints(seq), **_pool(c["type"], 1, n_pages, H, P, D, g))
        starts = np.concatenate([[0], np.cumsum(sizes)])
        inverse = lens[seq]
        if c["form"] == "token":
            s.update(lens=_ints(inverse), max_len=int(c["past"]))
            return s
        # `seq` names each tree's table row: that row has to hold the tree's own past and nodes
        table = np.zeros_like(table)
        table[seq] = s["table"].cpu().numpy()
        s.update(table=_ints(table), starts=_ints(starts), past=_ints(past), max_len=int(lens.max()),
                 mask=_ints(_mask(sizes, _parents(sizes, rng))) if c["form"] == "tree" else None)
        return s
    n = c["trees"]
    sizes = _sizes(n, max(1, c["nodes"] // 4), c["nodes"])
    parents = _parents(sizes, rng)
    table, n_pages = _tables(c["past"] + sizes, P, rng)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    tokens = rng.permutation(int(starts[-1])) + 11  # no two alike
    sampled = np.full(int(starts[-1]), 5)  # a token that nobody drafted
    for i, p in enumerate(parents):
        # the path that the samples take: nodes whose rows lie where they will be kept, or behind all that are kept
        # (so a pass may be repeated on the same pages)
        at, depth, goal = 0, 1, int(rng.integers(1, 10))
        while depth < goal:
            down = [j for j, up in enumerate(p) if up == at and (j == depth or j >= goal)]
            if not down:
                break
            nxt = int(rng.choice(down))
            sampled[starts[i] + at] = tokens[starts[i] + nxt]
            at, depth = nxt, depth + 1
    return dict(case=c, tokens=_ints(tokens), sampled=_ints(sampled), parent=_ints(np.concatenate(parents)), starts=_ints(starts),
                past=_ints(np.full(n, c["past"])), mask=_ints(_mask(sizes, parents)), table=_ints(table),
                **_pool(c["type"], c["layers"], n_pages, H, P, D, g))


# ----------------------------------------------------------- plain forms

def _quantized(x, kind):
    """x [rows, heads, dim] in 8 bits, and the scales [rows, heads]: each value is the nearest to the quotient, which
    is formed in 64 bits because it may lie next to a border between two."""
    amax = x.abs().amax(-1)
    scale = torch.clamp(amax / torch.full_like(amax, TOP[kind]), min=2.0 ** -126)
    y = x.double() / scale.double()[..., None]
    if kind == "i8":
        return y.round().to(TYPES[kind]), scale
    # e4m3: steps of 1/8 of the power of two below, of 2^-9 at least
    step = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y).exponent - 1, min=-6) - 3)
    return ((y / step).round() * step).float().to(TYPES[kind]), scale


def _write8(s):
    c = s["case"]
    H, D, P = c["heads"], c["head"], c["page"]
    n = H * D
    pos = s["pos"].long()
    page, slot = s["table"].long()[s["seq"].long(), pos // P], pos % P
    kq, ks = _quantized(s["qkv"][:, n : 2 * n].reshape(-1, H, D), c["type"])
    vq, vs = _quantized(s["qkv"][:, 2 * n :].reshape(-1, H, D), c["type"])
    # (bytes: not every type can be indexed)
    s["k"][1].view(torch.uint8)[page, :, slot] = kq.view(torch.uint8)
    s["v"][1].view(torch.uint8)[page, :, :, slot] = vq.view(torch.uint8)
    s["k_scale"][1][page, :, slot] = ks
    s["v_scale"][1][page, :, slot] = vs
    kr = s["k"][1].view(torch.uint8)[page, :, slot].view(TYPES[c["type"]]).float() * s["k_scale"][1][page, :, slot][..., None]
    vr = s["v"][1].view(torch.uint8)[page, :, :, slot].view(TYPES[c["type"]]).float() * s["v_scale"][1][page, :, slot][..., None]
    return kr.reshape(-1, n), vr.reshape(-1, n)


def _rows_of(s, pages):
    """K, V [trees, heads, rows, dim] in f32 of the pages [trees, n]."""
    c = s["case"]
    n, H, D = pages.shape[0], c["heads"], c["head"]
    if c["type"] in TOP:
        k = s["k"][0].view(torch.uint8)[pages].view(TYPES[c["type"]]).float() * s["k_scale"][0][pages][..., None]
        v = s["v"][0].view(torch.uint8)[pages].view(TYPES[c["type"]]).float() * s["v_scale"][0][pages][..., None, :]
    else:
        k, v = s["k"][0][pages].float(), s["v"][0][pages].float()
    return k.permute(0, 2, 1, 3, 4).reshape(n, H, -1, D), v.permute(0, 2, 1, 4, 3).reshape(n, H, -1, D)


def _attend(q, k, v, seen):
    """q [trees, heads, queries, dim], seen [trees, 1, queries, rows]."""
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(q.shape[-1]))
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - m), 0.0)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _attn(s):
    c = s["case"]
    n, H, G, D = c["trees"], c["heads"], c["group"], c["head"]
    k, v = _rows_of(s, s["table"].long()[s["seq"].long()])
    t = torch.arange(k.shape[2], device=DEV)
    if c["form"] == "token":
        seen = (t < s["lens"][:, None])[:, None, None]
        return _attend(s["q"].reshape(n, H, G, D), k, v, seen).reshape(n, -1)
    # the trees' rows side by side, as many for each as the largest has
    T, starts = c["nodes"], s["starts"].long()
    rows = s["q"].shape[0]
    node = torch.arange(T, device=DEV)
    at = torch.clamp(starts[:-1, None] + node, max=rows - 1)  # [trees, T]
    q = s["q"].reshape(rows, H, G, D)[at].permute(0, 2, 1, 3, 4).reshape(n, H, T * G, D)
    past = s["past"].long()[:, None, None]
    j = t - past  # [trees, 1, rows of the cache]: the node that a row is
    if s["mask"] is None:
        seen = j <= node[:, None]
    else:
        j = j.expand(n, T, -1)
        word = torch.gather(s["mask"][at], 2, torch.clamp(j >> 5, min=0, max=s["mask"].shape[1] - 1))
        seen = (j < 0) | (((word >> (j & 31).int()) & 1 == 1) & (j < (starts[1:] - starts[:-1])[:, None, None]))
    o = _attend(q, k, v, seen[:, None, :, None, :].expand(n, 1, T, G, -1).reshape(n, 1, T * G, -1))
    o = o.reshape(n, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(n * T, -1)
    r = torch.arange(rows, device=DEV)
    tree = torch.searchsorted(starts[1:], r, right=True)
    return o[tree * T + r - starts[tree]]


def _sample(s):
    x, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    x = x.double()
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    y = (x - x[:, :1]) / torch.where(greedy, 1.0, t)
    w = torch.exp(y)
    rank = torch.arange(x.shape[1], device=DEV)
    k = s["top_k"][:, None]
    kept = ((k <= 0) | (rank < k)) & (w >= s["min_p"].double()[:, None]) & (~greedy | (rank == 0))
    w = torch.where(kept, w, 0.0)
    cum = torch.cumsum(w, 1)
    kept = (cum - w < s["top_p"].double()[:, None] * cum[:, -1:]) | (rank == 0)
    w = torch.where(kept, w, 0.0)
    total = w.sum(1, keepdim=True)
    at = (torch.cumsum(w, 1) <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    lp = torch.where(greedy, 0.0, torch.gather(y, 1, at) - torch.log(total))
    return dict(tokens=torch.gather(order, 1, at)[:, 0].int(), logprobs=lp[:, 0].float())


def _keep(s):
    c = s["case"]
    n, T, P, starts = c["trees"], c["nodes"], c["page"], s["starts"].long()
    rows = s["tokens"].shape[0]
    node = torch.arange(T, device=DEV)
    there = node < (starts[1:] - starts[:-1])[:, None]  # [trees, T]
    at = torch.clamp(starts[:-1, None] + node, max=rows - 1)
    up = torch.clamp(s["parent"].long()[at], min=0)
    agrees = (torch.gather(s["sampled"][at], 1, up) == s["tokens"][at]) | (node == 0)
    # a node is accepted where it and all its ancestors agree (drafted tokens are distinct)
    word = s["mask"][at][:, :, node >> 5]  # [trees, T, T]
    above = (word >> (node & 31).int()) & 1 == 1
    path = (agrees[:, None, :] | ~above).all(2) & there
    count = path.sum(1)
    kept = torch.sort(torch.where(path, node, T), dim=1).values
    kept = torch.where(node < count[:, None], kept, -1)
    last = torch.gather(kept, 1, count[:, None] - 1)
    following = torch.gather(s["sampled"][at], 1, last)[:, 0]
    # the rows of the path move together
    tree, j = torch.nonzero(kept >= 0, as_tuple=True)
    past, table = s["past"].long()[tree], s["table"].long()
    src, dst = past + kept[tree, j], past + j
    sp, dp = table[tree, src // P], table[tree, dst // P]
    k, v = s["k"][:, sp, :, src % P].clone(), s["v"][:, sp, :, :, src % P].clone()
    s["k"][:, dp, :, dst % P] = k
    s["v"][:, dp, :, :, dst % P] = v
    return dict(kept=kept.int(), count=count.int(), following=following, k=s["k"], v=s["v"])


# ------------------------------------------------------ the framework's

def _write8_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    n, rows = c["heads"] * c["head"], c["seqs"] * c["new"]
    pages = A.KvPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    A.kv_write_dev(pages, 1, s["qkv"][:, n : 2 * n], s["qkv"][:, 2 * n :], rows, s["table"], s["pos"], seq=s["seq"])
    k, v = torch.empty(rows, n, device=DEV), torch.empty(rows, n, device=DEV)
    A.kv_read_dev(pages, 1, k, v, rows, s["table"], s["pos"], seq=s["seq"])
    return k, v


def _attn_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    pages = A.KvPages(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    out, rows, n_head = torch.empty_like(s["q"]), s["q"].shape[0], c["heads"] * c["group"]
    if c["form"] == "token":
        A.paged_attention_dev(pages, 0, s["q"], rows, n_head, s["table"], s["lens"], s["max_len"], out, seq=s["seq"])
    else:
        A.tree_attention_dev(pages, 0, s["q"], rows, n_head, s["table"], s["starts"], c["nodes"], s["past"], s["max_len"], out,
                             mask=s["mask"], seq=s["seq"])
    return out


def _sample_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    tokens, lp = torch.empty(c["rows"], dtype=torch.int32, device=DEV), torch.empty(c["rows"], device=DEV)
    A.sample_tokens_dev(s["logits"], c["rows"], c["vocab"], s["u"], tokens, logprobs=lp, temperature=s["temperature"],
                        top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return dict(tokens=tokens, logprobs=lp)


def _keep_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    n, T = c["trees"], c["nodes"]
    kept = torch.empty(n, T, dtype=torch.int32, device=DEV)
    count, following = (torch.empty(n, dtype=torch.int32, device=DEV) for _ in range(2))
    A.tree_accept_dev(s["tokens"], s["parent"], s["sampled"], s["tokens"].shape[0], s["starts"], T, kept, count, following)
    A.kv_keep_rows_dev(A.KvPages(s["k"], s["v"]), s["table"], s["past"], kept, count)
    return dict(kept=kept, count=count, following=following, k=s["k"], v=s["v"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"write8": _write8_own, "attn8": _attn_own, "tree": _attn_own, "sample": _sample_own, "keep": _keep_own}[kind](state)
    return {"write8": _write8, "attn8": _attn, "tree": _attn, "sample": _sample, "keep": _keep}[kind](state)


# ------------------------------------------------------------------ work

def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * SIZE[c["type"]] + c["rows"] * 28, flops=4 * n)
    n, es = c["heads"] * c["head"], SIZE[c["type"]]
    row = 2 * (n * es + (4 * c["heads"] if c["type"] in TOP else 0))  # of the cache
    if c["kind"] == "write8":
        # written from f32 rows, and read back as f32 rows
        return dict(bytes=2 * c["seqs"] * c["new"] * (2 * n * 4 + row), flops=0)
    if c["kind"] in ("attn8", "tree"):
        # expected sums: half of the ragged lengths are uniform in the upper three quarters, half log-uniform
        top = c["past"]
        past = top if c["lens"] == "full" else 0.5 * (0.625 * top) + 0.5 * top / math.log(top + 1.001)
        nodes = c["nodes"] * (1.0 if c["lens"] == "full" else 0.625 if c["form"] == "tree" else 1.0 if c["form"] == "token" else 0.5)
        new = 0 if c["form"] == "token" else nodes
        seen = past + (new / 2 if c["form"] == "chain" else min(new, 6))  # a node's ancestors are few
        return dict(bytes=max(1.0, c["trees"] * (past + new) * row) + 8 * c["trees"] * nodes * n * c["group"],
                    flops=4 * c["trees"] * nodes * max(1.0, seen) * n * c["group"])
    # about three rows of each tree move
    return dict(bytes=c["trees"] * (2 * min(3.0, c["nodes"] / 2) * c["layers"] * row + 0.625 * c["nodes"] * 16), flops=0)


# ----------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "sample":
        rows = c["rows"]
        tokens, lps = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.float64, device=DEV)
        temperature, top_k, top_p, min_p = (s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p"))
        u = s["u"].tolist()
        for r in range(rows):
            x = s["logits"][r].double()
            top = torch.argmax((x == x.max()).int())  # the lowest id of the largest
            if temperature[r] == 0:
                tokens[r] = top
                continue
            y = (x - x[top]) / temperature[r]
            ids = torch.nonzero(y > -60.0)[:, 0]  # what lies below 1e-26 of the largest is never drawn
            ids = ids[torch.argsort(-y[ids], stable=True)]
            if top_k[r] > 0:
                ids = ids[: top_k[r]]
            ids = ids[torch.exp(y[ids]) >= min_p[r]]
            p = torch.softmax(y[ids], 0)
            before = torch.cumsum(p, 0).roll(1)
            before[0] = 0
            ids = ids[(before < top_p[r]) | (torch.arange(len(ids), device=DEV) == 0)]
            lp = torch.log_softmax(y[ids], 0)
            at = min(int(torch.searchsorted(torch.cumsum(torch.exp(lp), 0), u[r], right=True)), len(ids) - 1)
            tokens[r], lps[r] = ids[at], lp[at]
        return dict(tokens=tokens, logprobs=lps)
    H, D, P = c["heads"], c["head"], c["page"]
    if c["kind"] == "write8":
        out = []
        for x in s["qkv"].double().reshape(-1, 3, H, D).unbind(1)[1:]:
            scale = (x.abs().amax(-1, keepdim=True) / TOP[c["type"]]).float().double()  # a scale is held in 32 bits
            y = x / scale
            if c["type"] == "i8":
                y = torch.floor(y + 0.5)
            else:  # the nearest of the type's values
                codes = torch.arange(127, dtype=torch.uint8, device=DEV).view(TYPES["e4m3"]).double()
                at = torch.bucketize(y.abs(), (codes[1:] + codes[:-1]) / 2)
                y = torch.copysign(codes[at], y)
            out.append((y * scale).reshape(-1, H * D))
        return tuple(out)
    if c["kind"] in ("attn8", "tree"):
        G = c["group"]
        out = torch.zeros(s["q"].shape[0], H, G, D, dtype=torch.float64, device=DEV)
        seq, table = s["seq"].tolist(), s["table"].long()
        if c["form"] == "token":
            starts, past = range(c["trees"] + 1), s["lens"].tolist()
        else:
            starts, past = s["starts"].tolist(), s["past"].tolist()
        for i in range(c["trees"]):
            a, b = starts[i], starts[i + 1]
            new = 0 if c["form"] == "token" else b - a
            n = past[i] + new
            if n == 0 or a == b:
                continue
            seen = torch.ones(b - a, n, dtype=torch.bool, device=DEV)
            if c["form"] == "chain":
                seen[:, past[i] :] = torch.tril(seen[:, past[i] :])
            elif c["form"] == "tree":
                bits = s["mask"][a:b].cpu().numpy().view(np.uint8)
                bits = np.unpackbits(bits, axis=1, bitorder="little")[:, :new]
                seen[:, past[i] :] = torch.from_numpy(bits.astype(bool)).to(DEV)
            ids = table[seq[i], : -(-n // P)]
            for h in range(H):
                k = s["k"][0, ids, h].double()
                v = s["v"][0, ids, h].double()
                if c["type"] in TOP:
                    k, v = k * s["k_scale"][0, ids, h].double()[..., None], v * s["v_scale"][0, ids, h].double()[:, None]
                k, v = k.reshape(-1, D)[:n], v.transpose(1, 2).reshape(-1, D)[:n]
                for g in range(G):
                    q = s["q"][a:b].reshape(b - a, H, G, D)[:, h, g].double()
                    x = (q @ k.T) / math.sqrt(D)
                    out[a:b, h, g] = torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1) @ v
        return out.reshape(out.shape[0], -1)
    starts, tokens, sampled = s["starts"].tolist(), s["tokens"].tolist(), s["sampled"].tolist()
    parent, past, table = s["parent"].tolist(), s["past"].tolist(), s["table"].tolist()
    kept = np.full((c["trees"], c["nodes"]), -1, np.int32)
    count, following = [], []
    k, v = s["k"], s["v"]
    for i in range(c["trees"]):
        path, a, b = [0], starts[i], starts[i + 1]
        while True:
            down = [j for j in range(b - a) if parent[a + j] == path[-1] and tokens[a + j] == sampled[a + path[-1]]]
            if not down:
                break
            path.append(down[0])
        kept[i, : len(path)] = path
        count.append(len(path))
        following.append(sampled[a + path[-1]])
        for j, r in enumerate(path):
            x, y = past[i] + r, past[i] + j
            k[:, table[i][y // P], :, y % P] = k[:, table[i][x // P], :, x % P].clone()
            v[:, table[i][y // P], :, :, y % P] = v[:, table[i][x // P], :, :, x % P].clone()
    return dict(kept=_ints(kept), count=_ints(count), following=_ints(following), k=k.double(), v=v.double())
