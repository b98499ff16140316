"""Plain restatement in 64 bits of the paged caches' formulas, on the CPU: rows quantised and read back, and attention over pages, row by row."""
import math

import torch

F64 = torch.float64
LARGEST = {"fp8": 448.0, "int8": 127.0}


def quantise(x, store):
    """(codes as the values they stand for without their scale, scales) of rows [..., size], each step rounded as f32 is."""
    x = x.float().cpu()
    c = LARGEST[store]
    s = torch.maximum(x.abs().amax(-1) * torch.tensor(1.0 / c), torch.tensor(2.0 ** -126))      # 1 / c in f32
    bad = ~torch.isfinite(x).all(-1)
    s = torch.where(bad, torch.tensor(float("nan")), s)
    y = torch.where(bad[..., None], torch.zeros_like(x), x / s[..., None]).clamp(-c, c)
    return (y.to(torch.float8_e4m3fn).float() if store == "fp8" else y.round()), s


def values(cache, which):
    """A pool [pages, kv_heads, page, size] in 64 bits."""
    pool, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    x = pool.cpu().float().to(F64)
    return x if scale is None else x * scale.cpu().to(F64)[..., None]


def places(sequences, page):
    """(sequence, position, page or -1, place in it) of every row of [(new, length, pages)]."""
    out = []
    for b, (new, length, pages) in enumerate(sequences):
        for p in range(length - new, length):
            out.append((b, p, pages[p // page] if 0 <= p // page < len(pages) else -1, p % page))
    return out


def attend(q, cache, sequences, scale, window=0, first=0):
    """(outputs [rows, heads, vdim], sum_j w_j |v_j| / sum_j w_j, largest |scale q . k| of absolute values) in 64 bits."""
    q = q.cpu().to(F64)
    rows, heads, _ = q.shape
    K, V, page = values(cache, "k"), values(cache, "v"), cache.page
    G = heads // cache.kv_heads
    out, mag, dots = torch.zeros(rows, heads, cache.vdim, dtype=F64), torch.zeros(rows, heads, cache.vdim, dtype=F64), torch.zeros(rows, heads, dtype=F64)
    at = 0
    for new, length, pages in sequences:
        there = [j for j in range(length) if 0 <= pages[j // page] < cache.n_pages]
        idx = torch.tensor(there, dtype=torch.long)
        pg, pl = torch.tensor([pages[j // page] for j in there], dtype=torch.long), idx % page
        k, v = (x[pg, :, pl] for x in (K, V))                               # [keys, kv_heads, size]
        for i in range(new):
            p = length - new + i
            seen = idx <= p
            if window:
                seen &= (idx > p - window) | (idx < first)
            if not bool(seen.any()):
                at += 1
                continue
            ks, vs = k[seen], v[seen]
            for h in range(heads):
                s = (ks[:, h // G] @ q[at, h]) * scale
                w = torch.softmax(s, 0)
                out[at, h] = w @ vs[:, h // G]
                mag[at, h] = w @ vs[:, h // G].abs()
                dots[at, h] = (ks[:, h // G].abs() @ q[at, h].abs()).max() * scale
            at += 1
    return out, mag, dots


def tolerance(out, mag, dots, size, keys, f32, store):
    """How far an output may be off, entry by entry.  A score is a sum of `size` products in f32, each addition off by at most 2^-23 of the sum of absolute
    values so far (the tensor core truncates): (size + 8) 2^-23 dots, with the scaling's, and as much again in the reference maximum; exp2 is off by 2^-22.  Weights of bf16 activations: one
    bf16, eps / 2 = 2^-8 (single tokens: two parts, 2^-15); with codes one f16, 2^-11, and either the scale's logarithm (2^-22 of at most 8), 2^-19, or
    a key and a value times their scales in f16, 2^-11 each: a score is then off by 2^-11 of the sum of its products' absolute values, 2^-11 dots, and the
    reference maximum by as much.  Sums of weights and products by keys 2^-23 for every key, and the rounding of a bf16 output by 2^-8 of itself.
    Second-order terms: a quarter more."""
    keys_f16 = 0 if f32 or store == "act" else 2.0 ** -11
    weights = 2 * ((size + 8) * 2.0 ** -23 + keys_f16) * dots[..., None] + 2.0 ** -22 + (0 if f32 else 2.0 ** -8 if store == "act" else 2.0 ** -10) + 2 * min(keys, 4096) * 2.0 ** -23
    return 1.25 * weights * mag + (2.0 ** -22 if f32 else 2.0 ** -8) * out.abs() + 1e-30


def rel(got, want):
    got, want = got.cpu().to(F64), want.cpu().to(F64)
    return float((got - want).norm() / (want.norm() + 1e-300))


def random_pages(sequences, page, n_pages, generator):
    """[(new, length)] -> [(new, length, pages)] with shuffled pages of their own."""
    order = torch.randperm(n_pages, generator=generator).tolist()
    out = []
    for new, length in sequences:
        n = -(-length // page)
        out.append((new, length, [order.pop() for _ in range(n)]))
    return out


__all__ = ["quantise", "values", "places", "attend", "tolerance", "rel", "random_pages", "LARGEST", "F64", "math"]
