"""Paged key/value caches: rows written (and quantised) as they come, read back, and attention of new tokens over them.

A pool holds pages of `page` tokens, each [kv_heads, page, size], in the activation type, in e4m3 or in int8; the two 8-bit forms have one f32
scale per token and head.  A step gives every sequence some new tokens: sequence b has rows starts[b] .. starts[b + 1] - 1, is lengths[b] tokens
long with them, and lies in the pages table[b].  `op` names the operator:

    write    new keys and values into the pool: scale = max(max |x| / c, 2^-126), code = round(x / scale), c = 448 (e4m3) or 127 (int8)
    read     the step's rows out of the pool, code * scale
    attend   causal softmax attention of the new tokens over everything the pool holds of their sequence; with a window the last `window`
             positions and the first `first` ones

`prepare` gives what a program holds before the call, `run` is one call, `exact` the same result in 64-bit torch."""
import math
import random

import torch

own = False

BF, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
LARGEST = {"fp8": 448.0, "int8": 127.0}
TINY = 2.0 ** -126
MOST_PAIRS = 2048 * 16384 * 32           # query heads x visible keys of the largest case here, and of any drawn one
MOST_ROWS = 16384 * 32                   # tokens x heads written or read


def _case(**k):
    return dict(dict(heads=32, kv_heads=8, dim=128, vdim=128, page=64, window=0, first=0, store="act", f32=False, ragged=True), **k)


def listed():
    return [
        # one decoded token of one sequence written: launch latency
        _case(name="write_one_token", op="write", seqs=1, new=1, context=1031, store="act"),
        # one decoded token of each of a serving batch into an e4m3 pool
        _case(name="write_batch_fp8", op="write", seqs=96, new=1, context=4000, store="fp8", page=16),
        # prompts of eight requests, 32 key/value heads (the 7B model's), into an int8 pool
        _case(name="write_prompts_int8", op="write", seqs=8, new=2048, context=2048, heads=32, kv_heads=32, store="int8"),
        # a sequence fetched out of an e4m3 pool, as for a prefix that moves
        _case(name="read_one_fp8", op="read", seqs=1, new=777, context=777, store="fp8", page=16),
        # a batch of whole sequences out of an int8 pool
        _case(name="read_batch_int8", op="read", seqs=16, new=4096, context=4096, store="int8"),
        # one decoded token in the middle of the 7B model's context
        _case(name="token_one", op="attend", seqs=1, new=1, context=1031, heads=32, kv_heads=32, store="act"),
        # one decoded token of each of 48 sequences of mixed lengths over an e4m3 pool
        _case(name="token_batch_fp8", op="attend", seqs=48, new=1, context=8192, store="fp8"),
        # one decoded token of a very long sequence with few key/value heads: the keys are all there is to share among the SMs
        _case(name="token_long", op="attend", seqs=1, new=1, context=131072, heads=16, kv_heads=4, ragged=False, store="act", page=16),
        # decoded tokens that see a window and the first tokens, int8 pool
        _case(name="token_window_int8", op="attend", seqs=24, new=1, context=30000, heads=16, kv_heads=4, window=4096, first=4, store="int8", page=16),
        # chunks of mixed lengths of a few requests over an e4m3 pool, with a decoding request among them
        _case(name="chunk_batch_fp8", op="attend", seqs=6, new=512, context=6000, store="fp8"),
        # a long prompt's last chunk
        _case(name="chunk_long", op="attend", seqs=1, new=2048, context=16384, ragged=False, store="act"),
        # a chunk in the 32-bit mode of trace replay, window and first tokens
        _case(name="chunk_window_f32", op="attend", seqs=2, new=300, context=2000, heads=8, kv_heads=2, window=512, first=16, store="act", f32=True, page=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    heads, kv = rng.choice([(32, 32), (32, 8), (16, 4), (8, 2), (40, 40), (16, 1)])
    c = _case(op=op, heads=heads, kv_heads=kv, dim=rng.choice([128, 128, 128, 64, 192]), vdim=rng.choice([128, 128, 64]), page=rng.choice([16, 32, 64, 128]),
              store=rng.choice(["act", "fp8", "int8"]), f32=rng.random() < 0.15, ragged=rng.random() < 0.8)
    c["seqs"] = _log(rng, 1, 64)
    if op != "attend":
        c["new"] = _log(rng, 1, max(1, min(4096, MOST_ROWS // (c["seqs"] * kv))))
        c["context"] = c["new"] + _log(rng, 1, 512)
        return c
    if rng.random() < 0.5:
        c["window"], c["first"] = _log(rng, 64, 4096), rng.choice([0, 1, 4, 16, 130])
    chunk = rng.random() < 0.5
    if chunk:
        c["seqs"] = _log(rng, 1, 8)
    c["new"] = _log(rng, 2, 2048) if chunk else 1
    if c["f32"]:
        c["new"] = min(c["new"], 512)
    most = (MOST_PAIRS // 8 if c["f32"] else MOST_PAIRS) // (c["seqs"] * c["new"] * heads)
    c["context"] = c["new"] + _log(rng, 16, max(17, min(32768, most, (1 << 21) // (c["seqs"] * kv))))
    return c


def _sequences(c):
    """(new tokens, length with them) of every sequence: the case's largest, or (ragged) spread below it by the case's own numbers; one of four or more
    that take chunks has a single new token, one has none."""
    if not c["ragged"]:
        return [(c["new"], c["context"])] * c["seqs"]
    r = random.Random(c["seqs"] * 1000003 + c["new"] * 1009 + c["context"])
    out = []
    for b in range(c["seqs"]):
        new = c["new"] if b == 0 else r.randint((c["new"] + 1) // 2, c["new"])
        if c["seqs"] >= 4 and c["new"] > 1 and b in (1, 2):
            new = 2 - b
        whole = c["op"] == "read" or c["context"] - c["new"] < 2
        out.append((new, new if whole and new else c["context"] if b == 0 else max(new, r.randint(c["context"] // 8 + 1, c["context"]))))
    return out


def _types(c):
    act = F32 if c["f32"] else BF
    return act, {"act": act, "fp8": FP8, "int8": torch.int8}[c["store"]]


def _size(t):
    return torch.empty(0, dtype=t).element_size()


def work(c):
    act, kept = _types(c)
    seqs, K, V, G = _sequences(c), c["dim"], c["vdim"], c["kv_heads"]
    rows, per = sum(n for n, _ in seqs), (K + V) * _size(kept) + (8 if c["store"] != "act" else 0)
    if c["op"] != "attend":
        return {"bytes": rows * G * ((K + V) * _size(act) + per), "flops": 2 * rows * G * (K + V)}
    pairs = keys = 0
    for n, length in seqs:
        w, first = c["window"] or length, c["first"]
        for p in range(length - n, length):
            pairs += min(p + 1, w) + max(0, min(first, p + 1 - w))
        if n:
            begin = max(0, length - n + 1 - w)                # the first position that a window reaches
            keys += length - begin + min(first, begin)
    return {"bytes": keys * G * per + rows * c["heads"] * (K + V) * _size(act), "flops": 2 * pairs * c["heads"] * (K + V)}


# ---------------------------------------------------------------------------------------------------- inputs
def _quantised(x, store):
    """Codes and scales of rows [..., size]."""
    if store == "act":
        return x, None
    c = LARGEST[store]
    s = (x.float().abs().amax(-1, keepdim=True) / c).clamp_min(TINY)
    y = (x.float() / s).clamp(-c, c)
    return (y.to(FP8) if store == "fp8" else y.round().to(torch.int8)), s[..., 0]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    act, _ = _types(c)
    seqs, P, G, K, V = _sequences(c), c["page"], c["kv_heads"], c["dim"], c["vdim"]
    rows = sum(n for n, _ in seqs)
    need = [-(-length // P) for _, length in seqs]
    pages = sum(need) + 3                                     # a few that no sequence has
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(need)
    table = torch.full((len(seqs), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    def keys(*shape):                                         # a few channels of a trained model's keys are much larger than the others
        return normal(*shape) * (1.0 + 3.0 * (torch.arange(shape[-1], device="cuda") % 37 == 5))

    # the new tokens' projections as one product leaves them
    qkv = torch.cat([normal(rows, c["heads"] * K), keys(rows, G, K).view(rows, G * K), normal(rows, G * V) + 0.25], dim=1).to(act)
    cut = c["heads"] * K
    k, ks = _quantised(keys(pages, G, P, K).to(act), c["store"])
    v, vs = _quantised((normal(pages, G, P, V) + 0.25).to(act), c["store"])
    return {"case": c, "seqs": seqs, "rows": rows, "q": qkv[:, :cut].view(rows, c["heads"], K), "k_new": qkv[:, cut:cut + G * K].view(rows, G, K),
            "v_new": qkv[:, cut + G * K:].view(rows, G, V), "k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table,
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "lengths": torch.tensor([m for _, m in seqs], dtype=torch.int32, device="cuda")}


# ---------------------------------------------------------------------------------------------------- the plain form
def _places(s):
    """Sequence and position of every row, and the page and the place in it where its key lies."""
    P = s["case"]["page"]
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    p = s["lengths"].long()[b] - s["starts"].long()[b + 1] + row
    return b, p, s["table"].long()[b, p // P], p % P


def _pool(s):
    return [t for t in (s["k"], s["v"], s["k_scale"], s["v_scale"]) if t is not None]


def _write(s):
    _, _, page, place = _places(s)
    for x, pool, scale in ((s["k_new"], s["k"], s["k_scale"]), (s["v_new"], s["v"], s["v_scale"])):
        code, sc = _quantised(x, s["case"]["store"])
        whole = pool.view(torch.uint8) if pool.dtype == FP8 else pool      # rows are moved as bytes
        whole[page, :, place] = code.view(torch.uint8) if pool.dtype == FP8 else code
        if scale is not None:
            scale[page, :, place] = sc
    return _pool(s)


def _rows_of(pool, scale, page, place):
    """Rows [..., G, size] in 32 bits."""
    x = pool.view(torch.uint8)[page, :, place].view(FP8).float() if pool.dtype == FP8 else pool[page, :, place].float()
    return x if scale is None else x * scale[page, :, place].unsqueeze(-1)


def _read(s):
    act, _ = _types(s["case"])
    _, _, page, place = _places(s)
    return [_rows_of(s["k"], s["k_scale"], page, place).to(act), _rows_of(s["v"], s["v_scale"], page, place).to(act)]


def _attend(s):
    c = s["case"]
    act, _ = _types(c)
    P, H, G, K, V = c["page"], c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    B, new, length = len(s["seqs"]), max(n for n, _ in s["seqs"]), max(m for _, m in s["seqs"])
    j = torch.arange(length, device="cuda")
    page, place = s["table"].long()[:, j // P].clamp_min(0), (j % P).expand(B, length)
    b, p, _, _ = _places(s)
    i = torch.arange(s["rows"], device="cuda") - s["starts"].long()[b]
    q = torch.zeros(B, new, H, K, device="cuda")
    q[b, i] = s["q"].float()
    at = torch.full((B, new), -1, dtype=torch.long, device="cuda")
    at[b, i] = p
    k = _rows_of(s["k"], s["k_scale"], page, place).permute(0, 2, 3, 1)                     # [B, G, K, keys]
    scores = torch.matmul(q.view(B, new, G, H // G, K).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * new, K), k).view(B, G, H // G, new, length)
    scores *= K ** -0.5
    seen = j <= at[:, :, None]
    if c["window"]:
        seen &= (j > at[:, :, None] - c["window"]) | (j < c["first"])
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True).clamp_min(torch.finfo(F32).min)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    v = _rows_of(s["v"], s["v_scale"], page, place).permute(0, 2, 1, 3)                     # [B, G, keys, V]
    o = torch.matmul(scores.view(B, G, H // G * new, length), v).view(B, G, H // G, new, V) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, new, H, V)[b, i].to(act)


def _handles(s):
    """The pool and the step as a program keeps them: the pool for good, the step for all layers of a model."""
    if "cache" not in s:
        from lit_llama_b200 import PagedCache, PagedStep

        act, _ = _types(s["case"])
        s["cache"] = PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"], dtype=act)
        s["step"] = PagedStep(s["starts"], s["lengths"], s["table"], rows=s["rows"], max_new=max(n for n, _ in s["seqs"]),
                              max_length=max(m for _, m in s["seqs"]))
    return s["cache"], s["step"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"write": _write, "read": _read, "attend": _attend}[op](s)
    cache, step = _handles(s)
    if op == "write":
        cache.write(s["k_new"], s["v_new"], step)
        return _pool(s)
    if op == "read":
        return list(cache.read(step))
    return cache.attend(s["q"], step, scale=s["case"]["dim"] ** -0.5, window=s["case"]["window"], first=s["case"]["first"])


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c, op, P, H, G = s["case"], case["op"], case["page"], case["heads"], case["kv_heads"]
    table = s["table"].tolist()

    def sequence(pool, scale, b, length):                     # [length, G, size], page after page
        x = pool[table[b][:-(-length // P)]] if pool.dtype != FP8 else pool.float()[table[b][:-(-length // P)]]
        x = x.double()
        if scale is not None:
            x = x * scale[table[b][:-(-length // P)]].double()[..., None]
        return x.transpose(1, 2).reshape(-1, G, pool.shape[-1])[:length]

    if op == "write":
        if c["store"] == "act":
            out = [s["k"].double(), s["v"].double()]
            pairs = list(zip(out, (s["k_new"].double(), s["v_new"].double())))
        else:                                                 # the codes are whole numbers or 8-bit values: no value in 64 bits
            out = [None, None, s["k_scale"].double(), s["v_scale"].double()]
            pairs = list(zip(out[2:], [(x.double().abs().amax(-1) / LARGEST[c["store"]]).clamp_min(TINY) for x in (s["k_new"], s["v_new"])]))
        at = 0
        for b, (n, length) in enumerate(s["seqs"]):
            for pool, new in pairs:
                p = torch.arange(length - n, length, device="cuda")
                pool[s["table"][b].long()[p // P], :, p % P] = new[at:at + n]
            at += n
        return out
    if op == "read":
        return [torch.cat([sequence(pool, scale, b, length)[length - n:] for b, (n, length) in enumerate(s["seqs"])])
                for pool, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))]
    out, at = torch.empty(s["rows"], H, c["vdim"], dtype=F64, device="cuda"), 0
    for b, (n, length) in enumerate(s["seqs"]):
        k, v = sequence(s["k"], s["k_scale"], b, length), sequence(s["v"], s["v_scale"], b, length)
        p, j = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
        hidden = j > p
        if c["window"]:
            hidden |= (p - j >= c["window"]) & (j >= c["first"])
        for h in range(H if n else 0):
            x = s["q"][at:at + n, h].double() @ k[:, h // (H // G)].T * (c["dim"] ** -0.5)
            out[at:at + n, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v[:, h // (H // G)]
        at += n
    return out
