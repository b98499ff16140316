"""Several continuations of a sequence over paged key/value caches: trees of drafted tokens and beams.

`op` names the operator:

    tree     softmax attention of drafted tokens over the cache: each sees the context (with a window its last `window` positions and the first `first`) and,
             of the step's new tokens, its ancestors in the draft's tree and itself
    accept   target tokens from the logits of a tree's rows (the largest, or with a temperature and given noise a drawn one), and the path from the root on
             which every drafted token is its parent's target
    keep     the rows of that path moved together, in the pools of all layers
    copy     pages copied in the pools of all layers, as where a sequence is forked
    beam     the `count` largest of score + log-probability over a group's beams and the vocabulary

`prepare` gives what a program holds before the call, `run` is one call, `exact` the same result in 64-bit torch."""
import math
import random

import torch

own = False

BF, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
LARGEST = {"fp8": 448.0, "int8": 127.0}
TINY = 2.0 ** -126
MOST_PAIRS = 2 * 64 * 65536 * 32         # query heads x visible keys of the largest case here, and of any drawn one
MOST_LOGITS = 48 * 8 * 100003            # rows x vocabulary
MOST_POOL = 1 << 29                      # bytes of keys and values that are attended to
MOST_PAGES = 1 << 28                     # bytes of pages copied
MOST_ROWS = 64 * 8 * 32 * 8 * 256 * 4    # bytes of rows moved


def _case(**k):
    return dict(dict(seqs=1, new=1, context=64, heads=32, kv_heads=8, dim=128, vdim=128, page=64, window=0, first=0, store="act", f32=False, ragged=True), **k)


def listed():
    return [
        # eight drafted tokens in the middle of the 7B model's context: latency
        _case(name="tree_one", op="tree", seqs=1, new=8, context=1031, heads=32, kv_heads=32),
        # drafts of a serving batch over an e4m3 pool, trees of up to 32 tokens
        _case(name="tree_batch_fp8", op="tree", seqs=32, new=32, context=8192, store="fp8"),
        # wide trees over two very long sequences
        _case(name="tree_long", op="tree", seqs=2, new=64, context=65536, ragged=False, page=16),
        # drafts in the 32-bit mode of trace replay, window and first tokens
        _case(name="tree_window_f32", op="tree", seqs=5, new=21, context=2000, heads=8, kv_heads=2, window=512, first=16, f32=True, page=16),
        # one sequence's drafts against the 7B model's vocabulary, the largest logit
        dict(name="accept_one", op="accept", seqs=1, new=8, vocab=32000, f32=False, temperature=0.0, ragged=False),
        # a serving batch's drafts, targets drawn
        dict(name="accept_batch", op="accept", seqs=32, new=32, vocab=32000, f32=True, temperature=0.8, ragged=True),
        # the accepted tokens of one sequence's tree, 32 layers of 32 heads (the 7B model's)
        dict(name="keep_one", op="keep", seqs=1, new=26, context=500, layers=32, kv_heads=32, dim=128, page=64, store="act", f32=False),
        # those of a serving batch, int8 pools
        dict(name="keep_batch_int8", op="keep", seqs=64, new=64, context=300, layers=32, kv_heads=8, dim=128, page=64, store="int8", f32=False),
        # a sequence forked: its last page, 32 layers of e4m3
        dict(name="copy_one_fp8", op="copy", pairs=1, layers=32, kv_heads=8, dim=128, page=16, store="fp8", f32=False),
        # the last pages of the beams of a batch
        dict(name="copy_batch", op="copy", pairs=48, layers=32, kv_heads=8, dim=128, page=64, store="act", f32=False),
        # four beams of one request, the 7B model's vocabulary
        dict(name="beam_one", op="beam", groups=1, beams=4, count=8, vocab=32000, f32=True),
        # a batch of requests with eight beams each over a large odd vocabulary
        dict(name="beam_batch", op="beam", groups=48, beams=8, count=16, vocab=100003, f32=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "accept", "keep", "copy", "beam"])
    f32 = rng.random() < 0.2
    if op == "tree":
        heads, kv = rng.choice([(32, 32), (32, 8), (16, 4), (8, 2), (40, 40), (16, 1)])
        c = _case(op=op, heads=heads, kv_heads=kv, dim=rng.choice([128, 128, 128, 64, 192]), vdim=rng.choice([128, 128, 64]), page=rng.choice([16, 32, 64, 128]),
                  store=rng.choice(["act", "fp8", "int8"]), f32=f32, ragged=rng.random() < 0.8)
        if rng.random() < 0.3:
            c["window"], c["first"] = _log(rng, 64, 4096), rng.choice([0, 1, 4, 16, 130])
        c["seqs"], c["new"] = _log(rng, 1, 48), _log(rng, 1, 96)
        most = (MOST_PAIRS // 8 if f32 else MOST_PAIRS) // (c["seqs"] * c["new"] * heads)
        keys = MOST_POOL // (c["seqs"] * kv * (c["dim"] + c["vdim"]) * _size(_types(c)[1]))
        c["context"] = c["new"] + _log(rng, 16, max(17, min(32768, most, keys)))
        return c
    if op == "accept":
        c = dict(op=op, seqs=_log(rng, 1, 48), new=_log(rng, 1, 64), f32=f32, temperature=rng.choice([0.0, 0.0, 0.7, 1.0]), ragged=rng.random() < 0.8)
        c["vocab"] = _log(rng, 1000, max(1001, min(128000, MOST_LOGITS // (2 * c["seqs"] * c["new"]))))
        return c
    if op == "beam":
        c = dict(op=op, groups=_log(rng, 1, 64), beams=_log(rng, 1, 16), f32=f32)
        c["count"] = max(1, rng.choice([c["beams"], 2 * c["beams"]]))
        c["vocab"] = _log(rng, 1000, max(1001, min(200000, MOST_LOGITS // (2 * c["groups"] * c["beams"]))))
        return c
    c = dict(op=op, layers=rng.choice([1, 12, 32, 40, 61]), kv_heads=rng.choice([1, 2, 8, 32]), dim=rng.choice([64, 128, 128, 192]), page=rng.choice([16, 32, 64, 128]),
             store=rng.choice(["act", "fp8", "int8"]), f32=f32)
    token = c["layers"] * c["kv_heads"] * c["dim"] * 2 * _size(_types(c)[1])
    if op == "copy":
        c["pairs"] = _log(rng, 1, max(1, min(96, MOST_PAGES // (token * c["page"]))))
    else:
        c["seqs"], c["new"] = _log(rng, 1, max(1, min(64, MOST_ROWS // (token * 8)))), _log(rng, 3, 64)
        c["context"] = c["new"] + _log(rng, 1, 300)
    return c


def _types(c):
    act = F32 if c["f32"] else BF
    return act, {"act": act, "fp8": FP8, "int8": torch.int8}[c.get("store", "act")]


def _size(t):
    return torch.empty(0, dtype=t).element_size()


def _sequences(c):
    """(new tokens, length with them) of every sequence: the case's largest, or (ragged) spread below it by the case's own numbers; one of four or more
    has a single new token, one has none."""
    context = c.get("context", c["new"])
    if not c.get("ragged", True):
        return [(c["new"], context)] * c["seqs"]
    r = random.Random(c["seqs"] * 1000003 + c["new"] * 1009 + context)
    out = []
    for b in range(c["seqs"]):
        new = c["new"] if b == 0 else r.randint((c["new"] + 1) // 2, c["new"])
        if c["seqs"] >= 4 and c["new"] > 1 and b in (1, 2):
            new = 2 - b
        out.append((new, context if b == 0 else max(new, r.randint(context // 8 + 1, context))))
    return out


def _parents(n, r):
    """A tree's parents, each before its children: a token of the draft continues one of the last eight, the first continues the sequence."""
    return [-1] + [r.randint(max(0, j - 8), j - 1) for j in range(1, n)]


def _trees(c):
    r = random.Random(c["seqs"] * 7919 + c["new"])
    return [_parents(n, r) if n else [] for n, _ in _sequences(c)]


def _ancestors(parents):
    """Lists of the tokens that each sees (itself among them)."""
    out = []
    for j, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [j])
    return out


def _path(n, r):
    """The places of the tokens that a sequence keeps: the first, and some of those behind them."""
    if n < 3:
        return list(range(n))
    count = min(r.randint(2, 8), (n + 1) // 2)
    return [0] + sorted(r.sample(range(count, n), count - 1))


def _paths(c):
    r = random.Random(c["seqs"] * 104729 + c["new"])
    return [_path(n, r) for n, _ in _sequences(c)]


def work(c):
    op = c["op"]
    act, kept = _types(c)
    if op == "beam":
        rows = c["groups"] * c["beams"]
        return {"bytes": rows * c["vocab"] * _size(act) + 4 * rows + 12 * c["groups"] * c["count"], "flops": 3 * rows * c["vocab"]}
    if op in ("copy", "keep"):
        token = c["layers"] * c["kv_heads"] * (c["dim"] * 2 * _size(kept) + (8 if c["store"] != "act" else 0))
        tokens = c["pairs"] * c["page"] if op == "copy" else sum(max(len(p) - 1, 0) for p in _paths(c))
        return {"bytes": 2 * tokens * token, "flops": 0}
    seqs = _sequences(c)
    rows = sum(n for n, _ in seqs)
    if op == "accept":
        return {"bytes": rows * c["vocab"] * (_size(act) + (4 if c["temperature"] else 0)) + 12 * rows, "flops": (4 if c["temperature"] else 1) * rows * c["vocab"]}
    K, V, G = c["dim"], c["vdim"], c["kv_heads"]
    per = (K + V) * _size(kept) + (8 if c["store"] != "act" else 0)
    pairs = keys = 0
    for (n, length), parents in zip(seqs, _trees(c)):
        base, w, first = length - n, c["window"] or length + 1, c["first"]
        for seen in _ancestors(parents):
            p = base + len(seen) - 1
            begin = max(0, min(base, p - w + 1))              # of the context the window's first
            pairs += base - begin + min(first, begin) + len(seen)
        if n:
            begin = max(0, base + 1 - w)
            keys += length - begin + min(first, begin)
    return {"bytes": keys * G * per + rows * c["heads"] * (K + V) * _size(act) + 12 * rows, "flops": 2 * pairs * c["heads"] * (K + V)}


# ---------------------------------------------------------------------------------------------------- inputs
def _quantised(x, store):
    """Codes and scales of rows [..., size]."""
    if store == "act":
        return x, None
    c = LARGEST[store]
    s = (x.float().abs().amax(-1, keepdim=True) / c).clamp_min(TINY)
    y = (x.float() / s).clamp(-c, c)
    return (y.to(FP8) if store == "fp8" else y.round().to(torch.int8)), s[..., 0]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(s, g):
    """A table of shuffled pages of the sequences' own, a few more in the pool than they have."""
    c, seqs = s["case"], s["seqs"]
    need = [max(1, -(-length // c["page"])) for _, length in seqs]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(seqs), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table
    return pages


def _step(s):
    starts = [0]
    for n, _ in s["seqs"]:
        starts.append(starts[-1] + n)
    s["rows"], s["starts"], s["lengths"] = starts[-1], _ints(starts), _ints([m for _, m in s["seqs"]])


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    act, _ = _types(c)
    s = {"case": c}

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    if c["op"] == "beam":
        # logits of a trained model: most far below a few; scores of beams that have come some tokens far
        x = normal(c["groups"], c["beams"], c["vocab"], std=2.0)
        x += 6.0 * (normal(c["groups"], c["beams"], c["vocab"]) > 3.2)
        s["logits"] = x.to(act)
        s["scores"] = -normal(c["groups"], c["beams"], std=3.0).abs()
        return s
    if c["op"] in ("copy", "keep"):
        if c["op"] == "copy":
            pages = 2 * c["pairs"] + 3
            order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
            s["pairs"] = order[:2 * c["pairs"]].view(-1, 2).contiguous()
        else:
            s["seqs"] = _sequences(c)
            pages = _pages(s, g)
            _step(s)
            kept, counts = [], []
            for (n, _), path in zip(s["seqs"], _paths(c)):
                counts.append(len(path))
                kept += path + [-1] * (n - len(path))
            s["kept"], s["counts"] = _ints(kept), _ints(counts)
        # keys, values and their scales of all layers, [layers, pages, ..]
        shape = (c["layers"], pages, c["kv_heads"], c["page"])
        s["pools"] = [torch.empty(shape + (c["dim"],), dtype=_types(c)[1], device="cuda") for _ in range(2)]
        s["pools"] += [torch.empty(shape, device="cuda") for _ in range(2 if c["store"] != "act" else 0)]
        for i in range(c["layers"]):
            for x in range(2):
                code, scale = _quantised(normal(*shape[1:], c["dim"]).to(act), c["store"])
                s["pools"][x][i].copy_(code)
                if scale is not None:
                    s["pools"][2 + x][i].copy_(scale)
        return s
    s["seqs"] = _sequences(c)
    _step(s)
    rows, trees = s["rows"], _trees(c)
    s["parents"] = _ints([p for t in trees for p in t])
    if c["op"] == "accept":
        V = c["vocab"]
        r = random.Random(int(seed) * 31 + c["seqs"])
        x = normal(rows, V, std=2.0)
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        # the target model agrees with one child in most places
        at, agree = 0, []
        for t in trees:
            child = {}
            for j, p in enumerate(t):
                if p >= 0:
                    child.setdefault(p, []).append(j)
            agree += [(at + p, at + r.choice(js)) for p, js in child.items() if r.random() < 0.7]
            at += len(t)
        if agree:
            p, j = (torch.tensor(x_, device="cuda") for x_ in zip(*agree))
            x[p, tokens[j]] = 24.0
        s["logits"], s["tokens"] = x.to(act), tokens
        s["noise"] = torch.empty(rows, V, device="cuda").exponential_(generator=g) if c["temperature"] else None
        return s
    P, G, K, W = c["page"], c["kv_heads"], c["dim"], c["vdim"]
    pages = _pages(s, g)

    def keys(*shape):                                         # a few channels of a trained model's keys are much larger than the others
        return normal(*shape) * (1.0 + 3.0 * (torch.arange(shape[-1], device="cuda") % 37 == 5))

    # the new tokens' projections as one product leaves them
    qkv = normal(rows, c["heads"] * K + G * (K + W)).to(act)
    s["q"] = qkv[:, :c["heads"] * K].view(rows, c["heads"], K)
    s["k"], s["k_scale"] = _quantised(keys(pages, G, P, K).to(act), c["store"])
    s["v"], s["v_scale"] = _quantised((normal(pages, G, P, W) + 0.25).to(act), c["store"])
    return s


# ---------------------------------------------------------------------------------------------------- the plain form
def _rows_of(pool, scale, page, place):
    """Rows [..., G, size] in 32 bits."""
    x = pool.view(torch.uint8)[page, :, place].view(FP8).float() if pool.dtype == FP8 else pool[page, :, place].float()
    return x if scale is None else x * scale[page, :, place].unsqueeze(-1)


def _places(s):
    """Sequence of every row and its place among the sequence's new tokens."""
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    return b, row - s["starts"].long()[b]


def _padded(s, x, fill):
    """x [rows] as [sequences, most new tokens]."""
    b, i = _places(s)
    y = torch.full((len(s["seqs"]), s["case"]["new"]), fill, dtype=x.dtype, device="cuda")
    y[b, i] = x
    return y


def _tree(s):
    c = s["case"]
    act, _ = _types(c)
    P, H, G, K, V = c["page"], c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    B, new, length = len(s["seqs"]), c["new"], max(m for _, m in s["seqs"])
    b, i = _places(s)
    j = torch.arange(length, device="cuda")
    n = s["starts"].long().diff()
    base = (s["lengths"].long() - n)[:, None, None]
    # what of the new tokens a row sees: itself, its parent, its parent's parent ..
    parents = _padded(s, s["parents"].long(), -1)
    node = torch.arange(new, device="cuda").expand(B, new)
    own_bits, at = torch.zeros(B, new, new, dtype=torch.bool, device="cuda"), node
    for _ in range(new):
        own_bits |= (at[:, :, None] == node[:, None, :]) & (at >= 0)[:, :, None]
        at = torch.where(at >= 0, parents.gather(1, at.clamp_min(0)), at)
    p = base + own_bits.sum(-1, keepdim=True) - 1
    seen = (j < base).expand(B, new, length).clone()
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["first"])
    k_of = j - base
    inside = (k_of >= 0) & (k_of < n[:, None, None])
    seen |= inside & own_bits.gather(2, k_of.clamp(0, new - 1).expand(B, new, length))
    q = torch.zeros(B, new, H, K, device="cuda")
    q[b, i] = s["q"].float()
    page, place = s["table"].long()[:, j // P].clamp_min(0), (j % P).expand(B, length)
    k = _rows_of(s["k"], s["k_scale"], page, place).permute(0, 2, 3, 1)                     # [B, G, K, keys]
    scores = torch.matmul(q.view(B, new, G, H // G, K).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * new, K), k).view(B, G, H // G, new, length)
    scores *= K ** -0.5
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp_min(torch.finfo(F32).min)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    v = _rows_of(s["v"], s["v_scale"], page, place).permute(0, 2, 1, 3)                     # [B, G, keys, V]
    o = torch.matmul(scores.view(B, G, H // G * new, length), v).view(B, G, H // G, new, V) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, new, H, V)[b, i].to(act)


def _accept(s):
    c = s["case"]
    B, new = len(s["seqs"]), c["new"]
    x = s["logits"].double()                                  # the largest of values that may be neighbours
    if c["temperature"]:
        x = x / c["temperature"] - s["noise"].double().log()
    target = _padded(s, x.argmax(-1), -1)
    parents, tokens = _padded(s, s["parents"].long(), -2), _padded(s, s["tokens"], -1)
    n = s["starts"].long().diff()
    at = torch.zeros(B, dtype=torch.long, device="cuda")
    live = n > 0
    kept, counts, following = torch.full((B, new), -1, dtype=torch.long, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda"), torch.full((B,), -1, dtype=torch.long, device="cuda")
    for step in range(new):
        kept[:, step] = torch.where(live, at, -1)
        counts += live
        t = target.gather(1, at[:, None])
        following = torch.where(live, t[:, 0], following)
        fits = (parents == at[:, None]) & (tokens == t) & live[:, None]
        live = fits.any(-1)
        at = torch.where(live, fits.int().argmax(-1), at)
    b, i = _places(s)
    return [kept[b, i].int(), counts.int(), following.int()]


def _as_bytes(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t


def _copy(s):
    src, dst = s["pairs"].long().unbind(1)
    for t in s["pools"]:
        t = _as_bytes(t)
        t[:, dst] = t[:, src]
    return s["pools"]


def _keep(s):
    P = s["case"]["page"]
    b, i = _places(s)
    moves = i < s["counts"].long()[b]
    n = s["starts"].long().diff()
    base = (s["lengths"].long() - n)[b]
    frm, to = base + s["kept"].long().clamp_min(0), base + i
    frm = torch.where(moves, frm, to)                         # a row that is not kept stays
    table = s["table"].long()
    for pools in s["pools"]:
        for t in _as_bytes(pools):
            t[table[b, to // P], :, to % P] = t[table[b, frm // P], :, frm % P]
    return s["pools"]


def _beam(s):
    c = s["case"]
    x = s["logits"].double()                                  # the order of values that may be neighbours
    x = s["scores"].double()[..., None] + (x - x.amax(-1, keepdim=True)) - (x - x.amax(-1, keepdim=True)).exp().sum(-1, keepdim=True).log()
    value, at = torch.sort(x.view(c["groups"], -1), dim=-1, descending=True, stable=True)
    value, at = value[:, :c["count"]], at[:, :c["count"]]
    return [value.float(), (at // c["vocab"]).int(), (at % c["vocab"]).int()]


def _handles(s):
    """What a program keeps: pools for good, the step and the tree for all layers of a model."""
    if "made" not in s:
        from lit_llama_b200 import PagedCache, PagedLayers, PagedStep, PagedTree

        c = s["case"]
        act, _ = _types(c)
        made = {}
        if "seqs" in s:
            table = s.get("table")
            if table is None:                                 # of acceptance: no cache is looked at
                table = torch.full((len(s["seqs"]), 1), -1, dtype=torch.int32, device="cuda")
            made["step"] = PagedStep(s["starts"], s["lengths"], table, rows=s["rows"], max_new=max(n for n, _ in s["seqs"]), max_length=max(m for _, m in s["seqs"]))
        if "parents" in s:
            made["tree"] = PagedTree(made["step"], s["parents"])
        if "k" in s:
            made["cache"] = PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"], dtype=act)
        if "pools" in s:
            made["layers"] = PagedLayers([PagedCache(*layer, dtype=act) for layer in zip(*s["pools"])])
        s["made"] = made
    return s["made"]


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"tree": _tree, "accept": _accept, "keep": _keep, "copy": _copy, "beam": _beam}[op](s)
    if op == "beam":
        from lit_llama_b200 import beam_select

        return list(beam_select(s["logits"], s["scores"], c["count"]))
    made = _handles(s)
    if op == "tree":
        return made["cache"].attend(s["q"], made["step"], scale=c["dim"] ** -0.5, window=c["window"], first=c["first"], tree=made["tree"])
    if op == "accept":
        return list(made["tree"].accept(s["logits"], s["tokens"], temperature=c["temperature"], noise=s["noise"]))
    if op == "keep":
        made["layers"].keep(made["step"], s["kept"], s["counts"])
    else:
        made["layers"].copy(s["pairs"])
    return s["pools"]


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("copy", "keep", "accept"):                      # nothing but whole numbers, and values that move
        return None
    s = prepare(case, seed)
    c = s["case"]
    if op == "beam":
        value = []
        for x, score in zip(s["logits"], s["scores"]):
            y = torch.log_softmax(x.double(), -1) + score.double()[:, None]
            value.append(torch.topk(y.flatten(), c["count"]).values)
        return [torch.stack(value), None, None]
    P, H, G = c["page"], c["heads"], c["kv_heads"]
    table = s["table"].tolist()

    def sequence(pool, scale, b, length):                     # [length, G, size], page after page
        pages = table[b][:-(-length // P)]
        x = (pool[pages] if pool.dtype != FP8 else pool.float()[pages]).double()
        if scale is not None:
            x = x * scale[pages].double()[..., None]
        return x.transpose(1, 2).reshape(-1, G, pool.shape[-1])[:length]

    out, at = torch.empty(s["rows"], H, c["vdim"], dtype=F64, device="cuda"), 0
    for b, ((n, length), parents) in enumerate(zip(s["seqs"], _trees(c))):
        if not n:
            continue
        k, v = sequence(s["k"], s["k_scale"], b, length), sequence(s["v"], s["v_scale"], b, length)
        base, j = length - n, torch.arange(length, device="cuda")
        hidden = torch.ones(n, length, dtype=torch.bool, device="cuda")
        for r, seen in enumerate(_ancestors(parents)):
            p = base + len(seen) - 1
            hidden[r, :base] = (j[:base] <= p - c["window"]) & (j[:base] >= c["first"]) if c["window"] else False
            hidden[r, [base + i for i in seen]] = False
        for h in range(H):
            x = s["q"][at:at + n, h].double() @ k[:, h // (H // G)].T * (c["dim"] ** -0.5)
            out[at:at + n, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v[:, h // (H // G)]
        at += n
    return out
