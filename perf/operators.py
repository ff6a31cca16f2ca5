"""The paged key/value cache and the attention that reads it, as they are measured.

A batch is ragged: sequence s has new tokens in rows q_start[s] .. q_start[s + 1] - 1 of the
row tensors, kv_len[s] keys in the cache once they are written, and its keys lie in the pages
pages[s, :]. New token i of n has position kv_len[s] - n + i. The cache is
[n_pages, kv heads, page size, head_dim] for keys and for values, in bfloat16, or in
float8_e4m3fn or int8 with one F32 scale per token and head.

Three kinds of case:
  write   append the new tokens' keys and values to the cache; a quantised cache is then
          read back, so that what is returned are the values that it stands for
  read    the keys and values of whole sequences as dense rows
  attend  causal attention of the new tokens over the cache (optionally a sliding window)
"""
import math
import random

import torch

own = False

HBM = {"bf16": 2, "e4m3": 1, "i8": 1}
TORCH = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8, "f32": torch.float32}
TOP = {"e4m3": 448.0, "i8": 127.0}


def listed():
    return [
        # one stream of a talker writes its token at every layer of every step: latency
        dict(name="write-one-token", kind="write", dtype="f32", cache="i8", seqs=1, heads=16, kv_heads=8, hd=128, page=16, new=1, keys=1000, window=0),
        # a batch of prompts fills an 8-bit cache after its q|k|v projection
        dict(name="write-prompts", kind="write", dtype="bf16", cache="e4m3", seqs=16, heads=16, kv_heads=8, hd=128, page=64, new=1531, keys=1531, window=0),
        # the same for an unquantised cache, next chunks of many sequences
        dict(name="write-chunks", kind="write", dtype="bf16", cache="bf16", seqs=40, heads=16, kv_heads=16, hd=64, page=32, new=257, keys=2000, window=0),
        # one sequence leaves the cache (moved to another pool, or looked at)
        dict(name="read-one", kind="read", dtype="f32", cache="i8", seqs=1, heads=16, kv_heads=8, hd=128, page=16, new=777, keys=777, window=0),
        # a whole pool of sequences is read back
        dict(name="read-pool", kind="read", dtype="bf16", cache="e4m3", seqs=24, heads=16, kv_heads=8, hd=128, page=64, new=4096, keys=4096, window=0),
        # one stream decodes early in its sequence: latency
        dict(name="decode-one", kind="attend", dtype="f32", cache="bf16", seqs=1, heads=16, kv_heads=8, hd=128, page=16, new=1, keys=777, window=0),
        # a server's decode step over the talker's full context
        dict(name="decode-batch", kind="attend", dtype="f32", cache="i8", seqs=64, heads=16, kv_heads=8, hd=128, page=64, new=1, keys=4096, window=0),
        # two long contexts, eight query heads to a key head
        dict(name="decode-long", kind="attend", dtype="bf16", cache="e4m3", seqs=2, heads=32, kv_heads=4, hd=128, page=128, new=1, keys=65000, window=0),
        # drafted tokens are checked: a few rows per sequence
        dict(name="verify-few", kind="attend", dtype="bf16", cache="bf16", seqs=16, heads=16, kv_heads=8, hd=128, page=16, new=5, keys=1500, window=0),
        # a whole prompt over its own keys
        dict(name="prompt", kind="attend", dtype="bf16", cache="bf16", seqs=1, heads=16, kv_heads=8, hd=128, page=64, new=4096, keys=4096, window=0),
        # chunks of prompts over what is cached already
        dict(name="chunks-ragged", kind="attend", dtype="bf16", cache="i8", seqs=8, heads=16, kv_heads=8, hd=128, page=32, new=517, keys=8000, window=0),
        # frames of a small transformer with a sliding window, all in F32
        dict(name="frames-window", kind="attend", dtype="f32", cache="bf16", seqs=4, heads=16, kv_heads=16, hd=64, page=16, new=500, keys=1100, window=250),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    c = dict(kind=kind, dtype=rng.choice(["f32", "bf16"]), cache=rng.choice(["bf16", "e4m3", "i8"]), kv_heads=kv_heads,
             heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), hd=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128, 256]), window=0)
    c["seqs"] = _log(rng, 1, 64)
    c["keys"] = _log(rng, 1, 65536)
    few = kind == "attend" and rng.random() < 0.5
    c["new"] = min(c["keys"], _log(rng, 1, 8 if few else 4096)) if kind != "read" else c["keys"]
    if kind == "attend" and rng.random() < 0.3:
        c["window"] = _log(rng, 1, 4096)
    most = {"write": 24_000, "read": 90_000, "attend": 260_000}[kind]  # rows (or keys) of a batch that the listed cases reach
    while c["seqs"] > 1 and c["seqs"] * (c["new"] if kind == "write" else c["keys"]) * c["kv_heads"] * c["hd"] > most * 8 * 128:
        c["seqs"] = (c["seqs"] + 1) // 2
    while c["seqs"] * (c["new"] if kind == "write" else c["keys"]) * c["kv_heads"] * c["hd"] > most * 8 * 128 or (
            kind == "attend" and c["seqs"] * c["new"] * c["keys"] * c["heads"] > 300_000_000):
        c["keys"] = max(1, c["keys"] // 2)
        c["new"] = c["keys"] if kind == "read" else max(1, min(c["keys"], c["new"] // 2 if c["new"] > 8 else c["new"]))
        c["seqs"] = (c["seqs"] + 1) // 2
    return c


def lengths(case):
    """(new tokens, keys) of every sequence: the first has the largest, the others spread below."""
    r = random.Random("%(seqs)d %(new)d %(keys)d" % case)
    got = []
    for s in range(case["seqs"]):
        part = 1.0 if s == 0 else r.uniform(0.4, 1.0)
        keys = max(1, round(case["keys"] * part))
        new = keys if case["new"] == case["keys"] else min(keys, max(1, round(case["new"] * part)))
        got.append((new, keys))
    return got


def prepare(case, seed):
    d, g = "cuda", torch.Generator(device="cuda").manual_seed(seed)
    hd, hkv, page, fmt = case["hd"], case["kv_heads"], case["page"], case["cache"]
    new, keys = zip(*lengths(case))
    starts = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)
    used = [-(-k // page) for k in keys]
    per, pool = max(used), sum(used) + 3
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pages = torch.zeros(case["seqs"], per, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        pages[s, :n] = order[at:at + n]
        at += n

    def cache():
        x = torch.randn((pool, hkv, page, hd), generator=g, device=d, dtype=torch.bfloat16)
        if fmt == "bf16":
            return x, None
        s = torch.rand((pool, hkv, page), generator=g, device=d) * 0.02 + 0.01
        if fmt == "i8":
            return (x * 42).clamp_(-127, 127).to(torch.int8), s
        return (x * 140).clamp_(-448, 448).to(torch.float8_e4m3fn), s * 0.3

    (kc, ks), (vc, vs) = cache(), cache()
    rows = int(starts[-1])
    # q | k | v as one projection leaves them: column blocks of one row
    qd, kd = case["heads"] * hd, hkv * hd
    qkv = torch.randn((rows, qd + 2 * kd), generator=g, device=d, dtype=torch.float32)
    qkv *= torch.exp(0.5 * torch.randn((rows, 1), generator=g, device=d))
    qkv = qkv.to(TORCH[case["dtype"]])
    return dict(case=case, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, q=qkv[:, :qd], k=qkv[:, qd:qd + kd], v=qkv[:, qd + kd:],
                q_start=starts.to(d), kv_len=torch.tensor(keys, dtype=torch.int32, device=d), pages=pages.to(d), rows=rows,
                max_new=max(new), max_keys=max(keys))


# ---- the plain form -------------------------------------------------------------------------

def _where(st):
    """(page, offset in it) of every new row."""
    row = torch.arange(st["rows"], device="cuda")
    seq = torch.searchsorted(st["q_start"][1:].long(), row, right=True)
    pos = st["kv_len"].long()[seq] - st["q_start"].long()[seq + 1] + row
    page = st["k_cache"].shape[2]
    return st["pages"].long()[seq, pos // page], pos % page


def _plain_write(x, cache, scale, page, off):
    x = x.reshape(x.shape[0], cache.shape[1], cache.shape[3]).float()
    if scale is None:
        cache[page, :, off] = x.to(cache.dtype)
        return
    top = TOP["i8" if cache.dtype == torch.int8 else "e4m3"]
    s = x.abs().amax(-1)
    s = s / torch.full_like(s, top)  # a division: by a number torch multiplies with its reciprocal
    s = torch.where(s > 0, s, torch.ones_like(s))
    q = x / s[..., None]
    q = torch.round(q) if cache.dtype == torch.int8 else q
    raw = cache.view(torch.int8) if cache.dtype != torch.int8 else cache
    raw[page, :, off] = q.clamp(-top, top).to(cache.dtype).view(torch.int8)
    scale[page, :, off] = s


def _values(cache, scale, page, off):
    if cache.dtype == torch.float8_e4m3fn:
        x = cache.view(torch.int8)[page, :, off].view(torch.float8_e4m3fn).float()
    else:
        x = cache[page, :, off].float()
    return x if scale is None else x * scale[page, :, off][..., None]


def _plain_attend(st):
    c = st["case"]
    S, hd, hkv, G, page = c["seqs"], c["hd"], c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    j = torch.arange(st["max_keys"], device="cuda")
    i = torch.arange(st["max_new"], device="cuda")
    at = st["pages"].long()[:, j // page], (j % page).expand(S, -1)
    k = _values(st["k_cache"], st["k_scale"], *at).permute(0, 2, 3, 1)  # [S, hkv, hd, keys]
    v = _values(st["v_cache"], st["v_scale"], *at).permute(0, 2, 1, 3)  # [S, hkv, keys, hd]
    start = st["q_start"].long()
    new = (start[1:] - start[:-1])[:, None]
    pos = st["kv_len"].long()[:, None] - new + i
    real = i < new
    row = torch.where(real, start[:-1, None] + i, 0)
    q = st["q"].float()[row].reshape(S, len(i), hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(S, hkv, G * len(i), hd)
    seen = (j <= pos[..., None]) & (j > pos[..., None] - (c["window"] or 1 << 40))  # [S, new, keys]
    s = (q @ k).reshape(S, hkv, G, len(i), len(j)).mul_(hd ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    s /= s.sum(-1, keepdim=True)
    o = s.reshape(S, hkv, G * len(i), len(j)) @ v.masked_fill_((j >= st["kv_len"][:, None])[:, None, :, None], 0.0)
    o = o.reshape(S, hkv, G, len(i), hd).permute(0, 3, 1, 2, 4).reshape(S, len(i), -1)
    return o[real].to(st["q"].dtype)


def _plain(st):
    if st["case"]["kind"] == "attend":
        return _plain_attend(st)
    page, off = _where(st)
    if st["case"]["kind"] == "write":
        _plain_write(st["k"], st["k_cache"], st["k_scale"], page, off)
        _plain_write(st["v"], st["v_cache"], st["v_scale"], page, off)
        if st["k_scale"] is None:
            return {"k": st["k_cache"], "v": st["v_cache"]}
    t = st["q"].dtype
    return {"k": _values(st["k_cache"], st["k_scale"], page, off).flatten(1).to(t), "v": _values(st["v_cache"], st["v_scale"], page, off).flatten(1).to(t)}


# ---- the framework's -------------------------------------------------------------------------

def _lai():
    import importlib
    import os
    import sys
    p = os.path.join(os.getcwd(), "local-ai-server_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    return importlib.import_module("lai")


def _own(st):
    lai, c = _lai(), st["case"]
    if "kv" not in st:  # what a server makes when it allocates the pool
        st["kv"] = lai.PagedKV(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        st["scratch"] = lai.paged_attention_scratch(c["hd"]) if c["kind"] == "attend" else None
    batch = lai.PagedBatch(st["q_start"], st["kv_len"], st["pages"])  # new at every step
    if c["kind"] == "attend":
        return lai.paged_attention(st["q"], st["kv"], batch, window=c["window"], scratch=st["scratch"])
    if c["kind"] == "write":
        lai.paged_kv_append(st["kv"], batch, st["k"], st["v"])
        if st["k_scale"] is None:
            return {"k": st["k_cache"], "v": st["v_cache"]}
    k, v = lai.paged_kv_read(st["kv"], batch, st["rows"], st["q"].dtype)
    return {"k": k, "v": v}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------

def _pairs(new, keys, window):
    """(query, key) pairs that see each other, and the keys that any query sees."""
    first = keys - new
    if not window:
        return new * first + new * (new + 1) // 2, keys
    n = sum(min(window, p + 1) for p in range(first, keys))
    return n, min(keys, new + window - 1)


def work(case):
    e, ce, kd = 4 if case["dtype"] == "f32" else 2, HBM[case["cache"]], case["kv_heads"] * case["hd"]
    per_row = 2 * (kd * ce + (4 * case["kv_heads"] if ce == 1 else 0))  # one position of the cache, k and v
    size = lengths(case)
    rows = sum(n for n, _ in size)
    if case["kind"] == "attend":
        got = [_pairs(n, k, case["window"]) for n, k in size]
        return {"bytes": 2 * rows * case["heads"] * case["hd"] * e + per_row * sum(k for _, k in got) + 4 * sum(-(-k // case["page"]) for _, k in size),
                "flops": 4 * case["hd"] * case["heads"] * sum(p for p, _ in got)}
    once = rows * (2 * kd * e + per_row)
    twice = case["kind"] == "write" and ce == 1
    return {"bytes": once * (2 if twice else 1), "flops": rows * kd * 2 * (3 if twice else 1)}


# ---- from the definition, in 64 bits ----------------------------------------------------------

def _e4m3_64(x):
    """The nearest value of 4 exponent and 3 mantissa bits (bias 7, largest 448), ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _stored_64(x, fmt):
    """What a cache of format fmt stands for after x [rows, heads, hd] is written: the scale and
    the quotient are F32 by definition."""
    x = x.double()
    if fmt == "bf16":
        return x.bfloat16().double()
    a = x.abs().amax(-1, keepdim=True)
    s = torch.where(a > 0, (a / TOP[fmt]).float().double(), torch.ones_like(a))
    q = (x / s).float().double()
    return (torch.round(q).clamp(-127, 127) if fmt == "i8" else _e4m3_64(q)) * s


def exact(case, seed):
    st = prepare(case, seed)
    hd, hkv, fmt, page = case["hd"], case["kv_heads"], case["cache"], case["page"]
    pages = st["pages"].long()
    kinds = {}
    for name in ("k", "v"):
        c, s = st[name + "_cache"], st[name + "_scale"]

        def seq_values(n, keys, c=c, s=s):
            p = pages[n, : -(-keys // page)]
            x = (c.view(torch.int8)[p].view(c.dtype) if fmt == "e4m3" else c[p]).double()  # [pages, heads, page, hd]
            x = x if s is None else x * s[p].double()[..., None]
            return x.permute(0, 2, 1, 3).reshape(-1, hkv, hd)[:keys]

        kinds[name] = seq_values
    size, at, out = lengths(case), 0, {"k": [], "v": [], "o": []}
    if case["kind"] == "write":
        for name in ("k", "v"):
            x = _stored_64(st[name].reshape(-1, hkv, hd), fmt)
            if fmt != "bf16":
                out[name] = x.flatten(1)
                continue
            out[name], row = st[name + "_cache"].double(), 0
            for n, (new, keys) in enumerate(size):
                p = torch.arange(keys - new, keys, device="cuda")
                out[name][pages[n, p // page], :, p % page] = x[row:row + new]
                row += new
        return {"k": out["k"], "v": out["v"]}
    if case["kind"] == "attend" and work(case)["flops"] > 4e11:
        return None
    for n, (new, keys) in enumerate(size):
        k, v = kinds["k"](n, keys), kinds["v"](n, keys)
        if case["kind"] == "read":
            out["k"].append(k.flatten(1))
            out["v"].append(v.flatten(1))
            continue
        q = st["q"][at:at + new].double().reshape(new, hkv, -1, hd)
        at += new
        j, p = torch.arange(keys, device="cuda"), torch.arange(keys - new, keys, device="cuda")
        for lo in range(0, new, 512):
            pq = p[lo:lo + 512, None]
            seen = (j <= pq) & (j > pq - (case["window"] or 1 << 40))
            t = torch.einsum("nhgd,khd->hgnk", q[lo:lo + 512], k) / math.sqrt(hd)
            t = torch.softmax(t.masked_fill_(~seen, -math.inf), -1)
            out["o"].append(torch.einsum("hgnk,khd->nhgd", t, v).flatten(1))
    if case["kind"] == "read":
        return {"k": torch.cat(out["k"]), "v": torch.cat(out["v"])}
    return torch.cat(out["o"])
