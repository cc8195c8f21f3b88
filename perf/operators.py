"""The operators of a serving or beam-searching program, as cases to time.

Keys and values live in pages: k [layer][page][head][row][value] and v
[layer][page][head][value][row], a table of page ids per sequence.  Each step
such a program writes the new token's key and value rows, lets the token
attend to its sequence's pages, and scores the logits; forks and compaction
copy pages.

Kinds of case (the "kind" field):
  attn    attention of one new token per row over paged keys and values
  write   new key and value rows into their pages
  copy    pages copied over every layer (copy on write, compaction)
  score   log-probs of given tokens, entropy and top alternatives of logits

The plain forms compute in 32 bits with elementary torch operations; `exact`
computes from the definitions in 64.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 51866


# ----------------------------------------------------------------- cases

def listed():
    return [
        # one short utterance, a tiny model's decoder: a call's own latency
        dict(name="attn_one_short", kind="attn", type="f32", rows=1, heads=6, group=1, head=64, page=16, max_len=27,
             lens="full", shared=0),
        # five beams of a large model at the full text context; they share their prompt's pages
        dict(name="attn_beams", kind="attn", type="f16", rows=5, heads=20, group=1, head=64, page=32, max_len=448,
             lens="full", shared=4),
        # a batch of windows at all stages, f32 caches as the decoder keeps them
        dict(name="attn_batch_f32", kind="attn", type="f32", rows=48, heads=20, group=1, head=64, page=32,
             max_len=1500, lens="ragged", shared=0),
        # a served batch with grouped heads, lengths of a few thousand, some slots empty
        dict(name="attn_batch_grouped", kind="attn", type="bf16", rows=61, heads=8, group=4, head=128, page=64,
             max_len=8190, lens="ragged", shared=0),
        # one long context, many query heads per key head: the length is all there is to split
        dict(name="attn_one_long", kind="attn", type="f16", rows=1, heads=8, group=8, head=128, page=128,
             max_len=131071, lens="full", shared=0),
        # a step's new rows of a batch, from a fused projection's output
        dict(name="write_step", kind="write", type="f16", seqs=64, new=1, past=447, heads=20, head=64, page=32),
        # prompts of a batch: 24 windows of 1500 rows that start inside a page
        dict(name="write_prompts", kind="write", type="bf16", seqs=24, new=1500, past=9, heads=20, head=64, page=32),
        # the five beams' last pages after a fork, every layer
        dict(name="copy_fork", kind="copy", type="f16", pairs=5, layers=32, heads=20, head=64, page=16),
        # a pool compacted after many sequences ended
        dict(name="copy_compact", kind="copy", type="bf16", pairs=700, layers=24, heads=8, head=128, page=16),
        # one greedy step: the chosen token, entropy and five alternatives
        dict(name="score_greedy", kind="score", type="f32", rows=1, vocab=VOCAB, tokens=1, top=5),
        # the language tokens of a batch's first logits
        dict(name="score_language", kind="score", type="f16", rows=33, vocab=VOCAB, tokens=100, top=1),
        # transcripts scored in one call: every position of several windows
        dict(name="score_transcripts", kind="score", type="f32", rows=1792, vocab=VOCAB, tokens=1, top=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "write", "copy", "score", "score"))
    kind_type = rng.choice(("f32", "f16", "bf16"))
    heads, head = rng.choice((1, 2, 3, 5, 6, 8, 12, 16, 20)), rng.choice((32, 64, 96, 128))
    page = rng.choice((16, 32, 64, 128, 256))
    row = 2 * heads * head * SIZE[kind_type]
    if kind == "attn":
        rows = _log_int(rng, 1, 96)
        top = max(64, min(131071, (1 << 29) // (rows * row)))
        return dict(kind=kind, type=kind_type, rows=rows, heads=heads, group=rng.choice((1, 1, 2, 4, 5, 7, 8, 16, 20)),
                    head=head, page=page, max_len=_log_int(rng, 1, top), lens=rng.choice(("ragged", "ragged", "full")),
                    shared=rng.choice((0, 0, 1, 3)))
    if kind == "write":
        seqs = _log_int(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(2, min(2000, (36000 * 5120) // (seqs * row))))
        return dict(kind=kind, type=kind_type, seqs=seqs, new=new, past=_log_int(rng, 1, 1000) - 1, heads=heads, head=head,
                    page=page)
    if kind == "copy":
        layers = rng.choice((4, 6, 12, 24, 32))
        top = max(1, min(1500, (1 << 30) // (layers * page * row)))
        return dict(kind=kind, type=kind_type, pairs=_log_int(rng, 1, top), layers=layers, heads=heads, head=head, page=page)
    vocab = rng.choice((VOCAB, 51865, _log_int(rng, 100, 260000)))
    top = rng.choice((0, 1, 5, 10, 16, 20, 32))
    rows = _log_int(rng, 1, max(2, min(1792, 90_000_000 // vocab)))
    return dict(kind=kind, type=kind_type, rows=rows, vocab=vocab, tokens=rng.choice((1, 1, 4, 100)), top=top)


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _filled(shape, dtype, g):
    t = torch.empty(shape, dtype=dtype, device=DEV)
    return t.normal_(generator=g)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _lengths(c, rng):
    n, top = c["rows"], c["max_len"]
    if c["lens"] == "full":
        return np.full(n, top, np.int32)
    lens = np.round(np.exp(rng.uniform(0, math.log(top + 1), n))).astype(np.int32) - 1  # 0 .. top, most of them short
    long = rng.random(n) < 0.5
    lens[long] = rng.integers(top // 4, top + 1, int(long.sum()))
    lens[int(rng.integers(n))] = top
    return lens


def prepare(case, seed):
    c, rng, g = case, np.random.default_rng(int(seed)), _gen(seed)
    if c["kind"] == "score":
        logits = _filled((c["rows"], c["vocab"]), torch.float32, g) * 3.0
        logits[:, :: 37] = -math.inf  # suppressed tokens
        logits = logits.to(TYPES[c["type"]])
        tokens = rng.integers(0, c["vocab"], (c["rows"], c["tokens"]))
        return dict(case=c, logits=logits, tokens=_ints(tokens))
    P, H, D, dt = c["page"], c["heads"], c["head"], TYPES[c["type"]]
    if c["kind"] == "attn":
        lens = _lengths(c, rng)
        n_table = -(-c["max_len"] // P)
        used = -(-lens // P)
        n_pages = int(used.sum()) + 3
        free = rng.permutation(n_pages)
        table = np.zeros((c["rows"], n_table), np.int32)
        at = 0
        for i in range(c["rows"]):
            table[i, : used[i]] = free[at : at + used[i]]
            at += used[i]
        for i in range(1, c["rows"]):  # forked from row 0: the first pages are its own
            n = min(c["shared"], int(used[i]), int(used[0]))
            table[i, :n] = table[0, :n]
        seq = rng.permutation(c["rows"])  # query rows in another order than the table's
        return dict(case=c, k=_filled((1, n_pages, H, P, D), dt, g), v=_filled((1, n_pages, H, D, P), dt, g),
                    q=_filled((c["rows"], H * c["group"] * D), torch.float32, g) * 2.0, table=_ints(table), seq=_ints(seq),
                    lens=_ints(lens[seq]))
    if c["kind"] == "write":
        total = c["past"] + c["new"]
        n_table = -(-total // P)
        n_pages = c["seqs"] * n_table + 2
        table = rng.permutation(n_pages)[: c["seqs"] * n_table].reshape(c["seqs"], n_table)
        seq = np.repeat(np.arange(c["seqs"]), c["new"])
        pos = np.tile(c["past"] + np.arange(c["new"]), c["seqs"])
        qkv = _filled((c["seqs"] * c["new"], 3 * H * D), torch.float32, g)
        return dict(case=c, k=_filled((2, n_pages, H, P, D), dt, g), v=_filled((2, n_pages, H, D, P), dt, g), qkv=qkv,
                    table=_ints(table), seq=_ints(seq), pos=_ints(pos))
    n_pages = 2 * c["pairs"] + 1
    ids = rng.permutation(n_pages)
    return dict(case=c, k=_filled((c["layers"], n_pages, H, P, D), dt, g), v=_filled((c["layers"], n_pages, H, D, P), dt, g),
                src=ids[: c["pairs"]].astype(np.int32), dst=ids[c["pairs"] : 2 * c["pairs"]].astype(np.int32))


# ----------------------------------------------------------- plain forms

def _attn(s):
    c = s["case"]
    rows, H, G, D, P = c["rows"], c["heads"], c["group"], c["head"], c["page"]
    pages = s["table"].long()[s["seq"].long()]  # [rows, n_table]
    k = s["k"][0][pages].float().permute(0, 2, 1, 3, 4).reshape(rows, H, -1, D)  # [rows, H, T, D]
    q = s["q"].reshape(rows, H, G, D)
    t = torch.arange(k.shape[2], device=DEV)
    seen = (t < s["lens"][:, None])[:, None, None]  # [rows, 1, 1, T]
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - m), 0.0)
    v = s["v"][0][pages].float().permute(0, 2, 1, 4, 3).reshape(rows, H, -1, D)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o.reshape(rows, H * G * D)


def _write(s):
    c = s["case"]
    H, D, P = c["heads"], c["head"], c["page"]
    n = H * D
    pos = s["pos"].long()
    page, slot = s["table"].long()[s["seq"].long(), pos // P], pos % P
    s["k"][1][page, :, slot] = s["qkv"][:, n : 2 * n].reshape(-1, H, D).to(s["k"].dtype)
    s["v"][1][page, :, :, slot] = s["qkv"][:, 2 * n :].reshape(-1, H, D).to(s["v"].dtype)
    return s["k"], s["v"]


def _copy(s):
    src, dst = (torch.from_numpy(s[n]).to(DEV).long() for n in ("src", "dst"))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def _score(s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lp = (x - m) - torch.log(z)
    entropy = -torch.where(e > 0, e * lp, 0.0).sum(-1) / z[:, 0]
    out = dict(logprobs=torch.gather(lp, 1, s["tokens"].long()), entropy=entropy)
    k = s["case"]["top"]
    if k:
        # larger logits first, equal ones by lowest id: one integer that orders both
        b = (x + 0.0).view(torch.int32).long()
        key = torch.where(b < 0, b ^ 0x7FFFFFFF, b) * (1 << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=DEV))
        ids = 0xFFFFFFFF - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
        out.update(ids=ids.int(), top=torch.gather(lp, 1, ids))
    return out


# ------------------------------------------------------ the framework's

def _attn_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    out = torch.empty_like(s["q"])
    A.paged_attention_dev(A.KvPages(s["k"], s["v"]), 0, s["q"], c["rows"], c["heads"] * c["group"], s["table"], s["lens"],
                          c["max_len"], out, seq=s["seq"])
    return out


def _write_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    n = c["heads"] * c["head"]
    A.kv_write_dev(A.KvPages(s["k"], s["v"]), 1, s["qkv"][:, n : 2 * n], s["qkv"][:, 2 * n :], c["seqs"] * c["new"],
                   s["table"], s["pos"], seq=s["seq"], ldk=3 * n, ldv=3 * n)
    return s["k"], s["v"]


def _copy_own(s):
    from rusty_whisper_amd import _abi as A

    A.kv_copy_pages_dev(A.KvPages(s["k"], s["v"]), s["src"], s["dst"])
    return s["k"], s["v"]


def _score_own(s):
    from rusty_whisper_amd import _abi as A

    c = s["case"]
    rows, k = c["rows"], c["top"]
    out = dict(logprobs=torch.empty(rows, c["tokens"], device=DEV), entropy=torch.empty(rows, device=DEV))
    if k:
        out.update(ids=torch.empty(rows, k, dtype=torch.int32, device=DEV), top=torch.empty(rows, k, device=DEV))
    A.token_logprobs_dev(s["logits"], rows, c["vocab"], s["tokens"], c["tokens"], out["logprobs"], entropy=out["entropy"],
                         k=k, top_ids=out.get("ids"), top_logprobs=out.get("top"))
    return out


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attn": _attn_own, "write": _write_own, "copy": _copy_own, "score": _score_own}[kind](state)
    return {"attn": _attn, "write": _write, "copy": _copy, "score": _score}[kind](state)


# ------------------------------------------------------------------ work

def work(case):
    c = case
    if c["kind"] == "score":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * SIZE[c["type"]] + c["rows"] * (8 * c["tokens"] + 4 + 8 * c["top"]), flops=6 * n)
    n, es = c["heads"] * c["head"], SIZE[c["type"]]
    if c["kind"] == "attn":
        # the lengths' expected sum: half of the ragged ones are uniform in the upper three quarters, half log-uniform
        top = c["max_len"]
        mean = top if c["lens"] == "full" else 0.5 * (0.625 * top) + 0.5 * top / math.log(top + 1.001)
        shared = c["shared"] * c["page"] * (c["rows"] - 1) if c["lens"] == "full" else 0
        total = max(1.0, c["rows"] * mean - min(shared, (c["rows"] - 1) * mean))
        return dict(bytes=total * 2 * n * es + 8 * c["rows"] * n * c["group"], flops=4 * c["rows"] * mean * n * c["group"])
    if c["kind"] == "write":
        return dict(bytes=c["seqs"] * c["new"] * 2 * n * (4 + es), flops=0)
    return dict(bytes=2 * c["pairs"] * c["layers"] * c["page"] * 2 * n * es, flops=0)


# ----------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "attn":
        H, G, D = c["heads"], c["group"], c["head"]
        out = torch.zeros(c["rows"], H, G, D, dtype=torch.float64, device=DEV)
        lens, seq, table = s["lens"].tolist(), s["seq"].tolist(), s["table"].long()
        for r in range(c["rows"]):
            n = lens[r]
            if n == 0:
                continue
            ids = table[seq[r], : -(-n // c["page"])]
            q = s["q"][r].double().reshape(H, G, D)
            for h in range(H):
                k = s["k"][0, ids, h].double().reshape(-1, D)[:n]
                v = s["v"][0, ids, h].double().transpose(1, 2).reshape(-1, D)[:n]
                w = torch.softmax((q[h] @ k.T) / math.sqrt(D), dim=-1)
                out[r, h] = w @ v
        return out.reshape(c["rows"], -1)
    if c["kind"] == "score":
        x = s["logits"].double()
        lse = torch.logsumexp(x, dim=1, keepdim=True)
        lp = x - lse
        p = torch.exp(lp)
        out = dict(logprobs=torch.gather(lp, 1, s["tokens"].long()), entropy=-torch.special.xlogy(p, p).sum(1))
        if c["top"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : c["top"]]
            out.update(ids=order.int(), top=torch.gather(lp, 1, order))
        return out
    if c["kind"] == "write":
        k, v = s["k"].double(), s["v"].double()
        H, D, P = c["heads"], c["head"], c["page"]
        rows = s["qkv"].double().reshape(-1, 3, H, D)
        table, total = s["table"].long(), c["past"] + c["new"]
        for i in range(c["past"] // P, -(-total // P)):  # one page of every sequence at a time
            lo, hi = max(c["past"], i * P), min(total, (i + 1) * P)
            part = rows.reshape(c["seqs"], c["new"], 3, H, D)[:, lo - c["past"] : hi - c["past"]]
            k[1, table[:, i], :, lo - i * P : hi - i * P] = part[:, :, 1].permute(0, 2, 1, 3)
            v[1, table[:, i], :, :, lo - i * P : hi - i * P] = part[:, :, 2].permute(0, 2, 3, 1)
        return k, v
    k, v = s["k"].double(), s["v"].double()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        k[:, b].copy_(k[:, a])
        v[:, b].copy_(v[:, a])
    return k, v
