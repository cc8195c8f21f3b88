"""Pools of keys and values in pages for the tests, and attention over them in
64 bits."""
import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of f32


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def pool(dtype, layers, n_pages, heads, page, dim, seed, fill=None):
    """k, v tensors: N(0, 1), or `fill` everywhere."""
    shape = (layers, n_pages, heads)
    if fill is not None:
        return [torch.full(shape + s, fill, dtype=DTYPES[dtype], device="cuda") for s in ((page, dim), (dim, page))]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(shape + s, device="cuda", generator=g).to(DTYPES[dtype]) for s in ((page, dim), (dim, page))]


def tables(lens, page, n_pages, seed, width=None):
    """int32 [len(lens), width] of distinct random pages (ids that no row
    reaches: one past the pool)."""
    rng = np.random.default_rng(seed)
    used = [-(-max(0, int(n)) // page) for n in lens]
    ids = rng.permutation(n_pages)
    assert sum(used) <= n_pages
    out = np.full((len(lens), width or max(1, max(used))), n_pages, np.int32)
    at = 0
    for i, n in enumerate(used):
        out[i, :n] = ids[at : at + n]
        at += n
    return out


def gather(k, v, layer, pages, n):
    """float64 K [heads, n, dim] and V [heads, n, dim] of a page list."""
    idx = torch.as_tensor(np.asarray(pages, dtype=np.int64), device=k.device)
    K = k[layer][idx].double().permute(1, 0, 2, 3).reshape(k.shape[2], -1, k.shape[4])[:, :n]
    V = v[layer][idx].double().permute(1, 0, 3, 2).reshape(k.shape[2], -1, k.shape[4])[:, :n]
    return K.cpu().numpy(), V.cpu().numpy()


def attend(q, K, V):
    """out [heads_q, dim] of one token, and a bound of the error of an
    implementation whose inputs keep 22 bits, whose products and sums are f32.

    A score is a sum of dim products: off by at most (dim + 16) half steps of
    sum |q k| / sqrt(dim) (16 half steps: 4 for the input's 22 bits, the rest
    for the scaling and for the exponential's argument).  With every score off
    by at most e, each p / sum p is off by 2 e relative to itself (and e^2
    terms, far below); the exponential and p's own 22 bits add 8 half steps; a
    sum of n products adds n.  The result is off by that much of sum p |v|."""
    hq, dim = q.shape
    G = hq // K.shape[0]
    out, tol = np.zeros((hq, dim)), np.zeros((hq, dim))
    for h in range(hq):
        k, v = K[h // G], V[h // G]
        n = k.shape[0]
        if n == 0:
            continue
        s = (k @ q[h]) / np.sqrt(dim)
        e = (dim + 16) * U * float(np.max(np.abs(k) @ np.abs(q[h]))) / np.sqrt(dim)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v
        tol[h] = (2.2 * e + (n + 8) * U) * (p @ np.abs(v))
    return out, tol


def norm_tol(sigma, dim, n):
    """The same as a share of the result's 2-norm, rounding errors taken as
    independent: a score's grow to 0.4 half steps times sigma sqrt(dim) (sigma:
    q's times k's standard deviation), a sum of n products' to 0.4 sqrt(n),
    a few for the exponential and the inputs' 22 bits; three times that."""
    return 3 * U * (0.4 * sigma * np.sqrt(dim) + 0.4 * np.sqrt(n) + 6)
