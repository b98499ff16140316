"""Plain restatement, on the CPU, of what trees of drafted tokens see and accept, of rows and pages that move, and of beam search's selection."""
import math

import torch

import paged_oracle as O

F64 = torch.float64


def ancestors(parents, window=0, first=0, base=0):
    """(set of the new tokens that each sees, depth) of a sequence's new tokens; a parent that does not come before its child is none."""
    path, out = [], []
    for i, p in enumerate(parents):
        path.append((path[p] if 0 <= p < i else []) + [i])
        d = len(path[i]) - 1
        out.append(({a for k, a in enumerate(path[i]) if not window or d - k < window or base + k < first}, d))
    return out


def bits(sets, words):
    """Masks as int32 rows."""
    out = torch.zeros(len(sets), words, dtype=torch.int64)
    for r, s in enumerate(sets):
        for i in s:
            if i < 32 * words:
                out[r, i // 32] |= 1 << (i % 32)
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)


def attend(q, cache, sequences, sets, depths, scale, window=0, first=0):
    """paged_oracle.attend with, of the new tokens, the sets that each row sees, and positions by depth."""
    q = q.cpu().to(F64)
    rows, heads, _ = q.shape
    K, V, page = O.values(cache, "k"), O.values(cache, "v"), cache.page
    G = heads // cache.kv_heads
    out, mag, dots = torch.zeros(rows, heads, cache.vdim, dtype=F64), torch.zeros(rows, heads, cache.vdim, dtype=F64), torch.zeros(rows, heads, dtype=F64)
    at = 0
    for new, length, pages in sequences:
        base = length - new
        for i in range(new):
            p = base + min(max(depths[at], 0), new - 1)
            seen = [j for j in range(base) if not window or j > p - window or j < first] + [base + a for a in sorted(sets[at]) if a < new]
            seen = [j for j in seen if 0 <= pages[j // page] < cache.n_pages]
            if seen:
                idx = torch.tensor(seen)
                pg = torch.tensor([pages[j // page] for j in seen])
                k, v = K[pg, :, idx % page], V[pg, :, idx % page]
                for h in range(heads):
                    s = (k[:, h // G] @ q[at, h]) * scale
                    w = torch.softmax(s, 0)
                    out[at, h], mag[at, h] = w @ v[:, h // G], w @ v[:, h // G].abs()
                    dots[at, h] = (k[:, h // G].abs() @ q[at, h].abs()).max() * scale
            at += 1
    return out, mag, dots


def targets(logits, temperature=0.0, noise=None):
    x = logits.cpu().to(F64)
    if temperature:
        x = x / float(torch.tensor(temperature, dtype=torch.float32)) - noise.cpu().to(F64).log()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return [int((row == row.max()).nonzero()[0]) if row.max() > -math.inf else 0 for row in x]


def accept(targets, tokens, parents):
    """(kept, following) of one sequence's new tokens."""
    if not tokens:
        return [], -1
    kept = [0]
    while True:
        at = kept[-1]
        child = [j for j in range(at + 1, len(tokens)) if parents[j] == at and tokens[j] == targets[at]]
        if not child:
            return kept, targets[at]
        kept.append(child[0])


def select(logits, scores, count):
    """(values in 64 bits, beams, tokens) of one group."""
    x = logits.cpu().to(F64)
    y = scores.cpu().to(F64)[:, None] + torch.log_softmax(x, -1)
    for w in range(x.shape[0]):
        if not bool(torch.isfinite(scores[w])) or bool(torch.isnan(x[w]).any()) or not math.isfinite(float(x[w].max())):
            y[w] = -math.inf
    value, at = torch.sort(y.flatten(), descending=True, stable=True)
    return value[:count], at[:count] // x.shape[1], at[:count] % x.shape[1]


def random_parents(n, rng, reach=8):
    return [-1] + [rng.randint(max(0, j - reach), j - 1) for j in range(1, n)] if n else []
