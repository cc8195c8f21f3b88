"""Drafted tokens, 8-bit pages and sampling for the tests: inputs, and the
definitions in 64 bits."""
import numpy as np
import torch


POOLS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
CODES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()  # 0, 2^-9, .. 448


def bytes_of(t):
    """An 8-bit tensor as bytes: not every type can be indexed."""
    return t.view(torch.uint8) if t.element_size() == 1 else t


def pool8(kind, layers, n_pages, heads, page, dim, seed):
    """k, v and their scales: values over the whole range of codes."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    out = []
    for shape in ((layers, n_pages, heads, page, dim), (layers, n_pages, heads, dim, page)):
        x = torch.randn(shape, device="cuda", generator=g) * (0.3 * TOP[kind])
        x = x.clamp(-TOP[kind], TOP[kind])
        out.append((x.round() if kind == "i8" else x).to(POOLS[kind]))
    for _ in range(2):
        s = torch.rand((layers, n_pages, heads, page), device="cuda", generator=g) * 3 + 2
        out.append(s / TOP[kind])
    return out


def any_pool(kind, layers, n_pages, heads, page, dim, seed):
    """[k, v] or [k, v, k_scale, v_scale]."""
    if kind in TOP:
        return pool8(kind, layers, n_pages, heads, page, dim, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn((layers, n_pages, heads) + s, device="cuda", generator=g).to(POOLS[kind])
            for s in ((page, dim), (dim, page))]


def gather_any(pool, layer, pages, n):
    """float64 K, V [heads, n, dim] of a page list, as the pool's values read."""
    idx = torch.as_tensor(np.asarray(pages, dtype=np.int64), device=pool[0].device)
    K, V = (bytes_of(x)[layer][idx].view(x.dtype).double() for x in pool[:2])
    if len(pool) == 4:
        K, V = K * pool[2][layer][idx].double()[..., None], V * pool[3][layer][idx].double()[..., None, :]
    h, d = K.shape[1], K.shape[3]
    return (K.permute(1, 0, 2, 3).reshape(h, -1, d)[:, :n].cpu().numpy(),
            V.permute(1, 0, 3, 2).reshape(h, -1, d)[:, :n].cpu().numpy())


def quantized(x, kind):
    """(codes' values, scales) of x [rows, heads, dim] (float32): the nearest
    value to x / s, ties to even, s in float32."""
    amax = np.abs(x).max(-1)
    s = np.maximum(amax / np.float32(TOP[kind]), np.float32(2.0 ** -126)).astype(np.float32)
    odd = ~np.isfinite(x).all(-1)
    s[odd] = np.nan
    y = x.astype(np.float64) / s.astype(np.float64)[..., None]
    if kind == "i8":
        q = np.rint(y)
    else:
        mid = (CODES[1:] + CODES[:-1]) / 2
        a = np.abs(y)
        lo, hi = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
        at = np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))  # in the middle: the even code
        q = np.copysign(CODES[np.minimum(at, 126)], y)
    q[odd] = 0
    return q, s


def trees(rng, sizes):
    """Parents of each tree's nodes (root: -1), a parent before its children."""
    return [[-1] + [int(rng.integers(max(0, j - 6), j)) for j in range(1, n)] if n else [] for n in sizes]


def ancestors(parents):
    """bool [nodes, nodes] of one tree: itself and its ancestors."""
    n = len(parents)
    m = np.eye(n, dtype=bool)
    for j, p in enumerate(parents):
        if p >= 0:
            m[j] |= m[p]
    return m


def words(masks, n_words=None):
    """int32 words of the trees' bool masks, one row per node."""
    n = n_words or max([1] + [-(-m.shape[1] // 32) for m in masks])
    out = np.zeros((sum(m.shape[0] for m in masks), n), np.uint32)
    r = 0
    for m in masks:
        for row in m:
            for j in np.flatnonzero(row):
                if j < 32 * n:
                    out[r, j >> 5] |= np.uint32(1 << (j & 31))
            r += 1
    return out.view(np.int32)


def sample(x, u, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share) of one row of float64 logits."""
    x = np.asarray(x, np.float64)
    order = np.lexsort((np.arange(x.size), -x))
    if t <= 0:
        return int(order[0]), 0.0
    y = (x[order] - x[order[0]]) / t
    w = np.exp(y).astype(np.longdouble)
    n = int((w > 0).sum())
    if top_k > 0:
        n = min(n, top_k)
    if min_p > 0:
        n = max(1, min(n, int((w >= min_p).sum())))
    if top_p < 1:
        c = np.cumsum(w[:n])
        n = int(np.searchsorted(c, np.longdouble(top_p) * c[-1], side="left")) + 1
    c = np.cumsum(w[:n])
    at = min(int(np.searchsorted(c, np.longdouble(u) * c[-1], side="right")), n - 1)
    return int(order[at]), float(y[at] - np.log(c[-1]))


def accept(tokens, parent, sampled):
    """(path, next token) of one tree."""
    if not len(tokens):
        return [], 0xFFFFFFFF
    path = [0]
    while True:
        at = path[-1]
        down = [j for j in range(at + 1, len(tokens)) if parent[j] == at and tokens[j] == sampled[at]]
        if not down:
            return path, int(sampled[at])
        path.append(down[0])
