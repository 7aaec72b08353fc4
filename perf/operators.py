"""The operators of a 4-bit key/value cache: appending to it, reading it back, attention over it.

Each case is measured in one of two forms: the framework's own calls (`own` true), or the same
mathematics in elementary torch operations in 32 bits (`own` false).

The cache is one uint8 tensor [pages, kv_heads, page_bytes].  A (page, head) block holds, one
after the other: the codes of the keys [page_size, D/2], of the values [page_size, D/2], and the
fp16 (scale, minimum) pairs of the keys [page_size, D/G, 2] and of the values.  Byte i of a
token's codes holds value 2i in its low and value 2i + 1 in its high four bits; a value is
code * scale + minimum.  Token slot s is page s // page_size, row s % page_size.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_LIMIT = 57344.0     # what is cached is clamped to this, so that every value read back is finite
_THETA = 500000.0


def _framework():
    path = os.path.join(_ROOT, "w4a16-gemm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import w4a16_opt
    return w4a16_opt


# ------------------------------------------------------------------------------ cases

def _append(name, tokens, q_heads, kv_heads, dim, group, page, dtype, axes, rotary=None, interleaved=False,
            fused=True):
    return {"name": name, "op": "append", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "group": group, "page": page, "dtype": dtype, "axes": axes, "rotary": rotary or dim,
            "interleaved": interleaved, "fused": fused}


def _read(name, tokens, kv_heads, dim, group, page, dtype):
    return {"name": name, "op": "read", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "group": group,
            "page": page, "dtype": dtype}


def _attention(name, batch, q_len, kv_len, ragged, q_heads, kv_heads, dim, group, page, dtype, causal=True,
               window=0):
    return {"name": name, "op": "attention", "batch": batch, "q_len": q_len, "kv_len": kv_len, "ragged": ragged,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "group": group, "page": page, "dtype": dtype,
            "causal": causal, "window": window}


def listed():
    return [
        # one decode step of eight sequences, Llama-3-8B heads: the call's latency is all there is
        _append("append step 8", 8, 32, 8, 128, 128, 64, "fp16", 1),
        # the tokens of a long prompt, Llama-3-70B heads: bound by the memory's bandwidth
        _append("append prompt 8192", 8192, 64, 8, 128, 128, 64, "bf16", 1),
        # a prompt of text and images, positions of three axes (time, height, width), small pages, fine groups
        _append("append image 1157", 1157, 28, 4, 128, 64, 16, "fp16", 3),
        # a short context handed to a consumer of 16-bit keys and values, 64-wide heads
        _read("read 777", 777, 4, 64, 64, 16, "fp16"),
        # the contexts of a whole batch
        _read("read 65536", 65536, 8, 128, 128, 64, "bf16"),
        # the next token of one short conversation: latency
        _attention("decode 1x1025", 1, 1, 1025, False, 32, 8, 128, 128, 64, "fp16"),
        # a serving batch of conversations of very different lengths
        _attention("decode 64x8192", 64, 1, 8192, True, 32, 8, 128, 128, 64, "fp16"),
        # the next token of one very long document: a single row of heads over a long cache
        _attention("decode 1x131072", 1, 1, 131072, False, 64, 8, 128, 64, 128, "bf16"),
        # the check of five drafted tokens for each of sixteen sequences
        _attention("verify 16x5x4096", 16, 5, 4096, True, 32, 8, 128, 128, 32, "fp16"),
        # a whole prompt of Llama-3-8B
        _attention("prompt 4096", 1, 4096, 4096, False, 32, 8, 128, 128, 64, "fp16"),
        # a chunk of a long prompt against what is cached of it, Llama-3-70B heads
        _attention("chunk 512 of 32768", 1, 512, 32768, False, 64, 8, 128, 64, 64, "bf16"),
        # prompts of odd lengths in one call, every head with keys of its own, a sliding window
        _attention("prompts 5x1531 window", 5, 1531, 2111, True, 12, 12, 64, 64, 16, "bf16", window=700),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attention", "attention", "attention"])
    dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (64, 128) if g <= dim])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["fp16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    if op == "append":
        shared = rng.choice([1, 2, 3, 4, 7, 8])
        c = _append("", _log(rng, 1, 8192), kv_heads * shared, kv_heads, dim, group, page, dtype,
                    rng.choice([0, 1, 1, 3]), rng.choice([dim, dim, dim // 2]), rng.random() < 0.3,
                    rng.random() < 0.5)
    elif op == "read":
        c = _read("", _log(rng, 1, 65536), kv_heads, dim, group, page, dtype)
    else:
        shared = rng.choice([1, 2, 3, 4, 5, 7, 8])
        kind = rng.choice(["decode", "decode", "few", "prompt"])
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        if kind == "decode":
            batch, q_len = _log(rng, 1, 64), 1
            kv_len = _log(rng, 1, min(131072, 64 * 8192 // batch))
        elif kind == "few":
            batch, q_len = _log(rng, 1, 32), rng.randint(2, 16)
            kv_len = _log(rng, q_len, min(32768, 64 * 8192 // batch))
        else:
            batch = _log(rng, 1, 8)
            q_len = _log(rng, 17, max(18, 4096 // batch))
            kv_len = q_len + rng.choice([0, _log(rng, 1, max(2, 4 * (4096 // batch)))])
        c = _attention("", batch, q_len, kv_len, rng.random() < 0.6, kv_heads * shared, kv_heads, dim, group, page,
                       dtype, rng.random() < 0.85, window)
        # no more than the largest listed cases: pairs of a query row and a key, and cached tokens
        while c["q_heads"] * batch * c["q_len"] * c["kv_len"] > 32 * 4096 * 4096:
            c["kv_len"] = max(c["q_len"], c["kv_len"] // 2)
            if c["kv_len"] == c["q_len"]:
                c["q_len"] = c["kv_len"] = max(17, c["q_len"] // 2)
        while work(c)["bytes"] > work(listed()[6])["bytes"]:
            c["kv_len"] //= 2
    del c["name"]
    return c


def _lengths(case):
    """Query and cached lengths of every sequence: part of the case, the same for every seed."""
    import random
    r = random.Random("%s %s %s" % (case["batch"], case["q_len"], case["kv_len"]))
    ql, kl = [], []
    for b in range(case["batch"]):
        n, q = case["kv_len"], case["q_len"]
        if case["ragged"] and b:     # the first sequence has the full lengths
            q = q if q <= 16 else r.randint(max(1, q // 8), q)
            n = r.randint(min(q, n), n)
        ql.append(q)
        kl.append(n)
    return ql, kl


def _visible(case):
    """Pairs of a query and a key that the mask leaves, summed over the sequences."""
    pairs = 0
    for q, n in zip(*_lengths(case)):
        for i in range(q):
            p = n - q + i
            hi = min(p, n - 1) if case["causal"] else n - 1
            lo = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs += max(0, hi - lo + 1)
    return pairs


def _needed(case):
    """Cached tokens that some query sees, summed over the sequences."""
    tokens = 0
    for q, n in zip(*_lengths(case)):
        lo = max(0, n - q - case["window"] + 1) if case["window"] else 0
        tokens += max(0, n - lo)
    return tokens


def work(case):
    row = case["kv_heads"] * (case["dim"] + 8 * (case["dim"] // case["group"]))    # K and V of one cached token
    row16 = case["kv_heads"] * case["dim"] * 4
    if case["op"] == "append":
        t, q = case["tokens"], case["tokens"] * case["q_heads"] * case["dim"] * 2
        # k and v in, codes out and in again, the values out; with positions also q in and out
        extra = 2 * q + 8 * t * case["axes"] + 4 * case["rotary"] * t if case["axes"] else 0
        turned = (case["q_heads"] + case["kv_heads"]) * case["rotary"] * 3 * t if case["axes"] else 0
        return {"bytes": 2 * t * (row16 + row) + extra, "flops": 10 * t * case["kv_heads"] * case["dim"] + turned}
    if case["op"] == "read":
        t = case["tokens"]
        return {"bytes": t * (row + row16 + 8), "flops": 4 * t * case["kv_heads"] * case["dim"]}
    q = sum(_lengths(case)[0]) * case["q_heads"] * case["dim"] * 2
    return {"bytes": _needed(case) * row + 2 * q, "flops": 4 * case["dim"] * case["q_heads"] * _visible(case)}


# ------------------------------------------------------------------------------ the cache's format, plainly

def _blocks(case, data):
    """Views of a cache (or of pages of it): key codes, value codes, key pairs, value pairs."""
    ps, d, ng = case["page"], case["dim"], case["dim"] // case["group"]
    n = ps * d // 2
    lead = data.shape[:-1]
    pairs = data[..., 2 * n:].view(torch.float16).view(*lead, 2, ps, ng, 2)
    return (data[..., :n].view(*lead, ps, d // 2), data[..., n:2 * n].view(*lead, ps, d // 2),
            pairs[..., 0, :, :, :], pairs[..., 1, :, :, :])


def _page_bytes(case):
    return case["page"] * (case["dim"] + 8 * (case["dim"] // case["group"]))


def _values(case, codes, pairs):
    """fp32 values [..., D] of codes [..., D/2] and fp16 pairs [..., D/G, 2]."""
    low, high = (codes & 15).float(), (codes >> 4).float()
    x = torch.stack((low, high), -1).flatten(-2)
    x = x.unflatten(-1, (case["dim"] // case["group"], case["group"]))
    p = pairs.float()
    return (x * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _quantise(case, x):
    """Codes [..., D/2] and fp16 pairs [..., D/G, 2] of fp32 values [..., D]."""
    x = torch.nan_to_num(x, nan=0.0, posinf=_LIMIT, neginf=-_LIMIT).clamp(-_LIMIT, _LIMIT)
    x = x.unflatten(-1, (case["dim"] // case["group"], case["group"]))
    low = x.amin(-1, keepdim=True).half().float()
    scale = ((x.amax(-1, keepdim=True) - low).clamp_min(0) / x.new_full((), 15.0)).half().float()
    code = torch.where(scale > 0, torch.round((x - low) / torch.where(scale > 0, scale, 1.0)), 0.0).clamp(0, 15)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat((scale, low), -1).half()


def _put(case, data, slots, k, v):
    """Writes fp32 k, v [T, kv_heads, D] to the slots (slots below zero are left out)."""
    kc, vc, kp, vp = _blocks(case, data)
    page, row = slots // case["page"], slots % case["page"]
    for codes, pairs, x in ((kc, kp, k), (vc, vp, v)):
        c, p = _quantise(case, x)
        codes[page, :, row] = c
        pairs[page, :, row] = p


# ------------------------------------------------------------------------------ inputs

def _hidden(gen, shape, dtype, channels=True):
    """What a projection gives: near normal, with a few channels far larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if channels:
        gain = torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.04, 6.0, 1.0)
        x = x * gain
    return x.to(dtype)


def _handle(case, data):
    return _framework().Int4KVCache.wrap(data, head_dim=case["dim"], page_size=case["page"], group_size=case["group"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d, hk = _DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    st = {"case": case}
    if case["op"] in ("append", "read"):
        t = case["tokens"]
        pages = -(-t // case["page"]) + 3
        data = torch.randint(0, 256, (pages, hk, _page_bytes(case)), generator=gen, device="cuda", dtype=torch.uint8)
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(t, device="cuda")
        st["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        k, v = _hidden(gen, (t, hk, d), dtype), _hidden(gen, (t, hk, d), dtype, False)
        if case["op"] == "read":
            _put(case, data, st["slots"], k.float(), v.float())
        else:
            q = _hidden(gen, (t, case["q_heads"], d), dtype)
            if case["fused"]:     # views of the one output of a fused projection
                x = torch.cat((q, k, v), 1)
                q, k, v = x[:, :case["q_heads"]], x[:, case["q_heads"]:case["q_heads"] + hk], x[:, case["q_heads"] + hk:]
            st.update(q=q, k=k, v=v)
            if case["axes"]:
                half = case["rotary"] // 2
                top = 2 * t + 64
                angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * \
                    _THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
                st["cos_sin"] = torch.cat((angle.cos(), angle.sin()), -1).float()
                start = torch.randint(0, t + 64, (), generator=gen, device="cuda")
                line = at + start
                if case["axes"] == 1:
                    st["positions"], st["sections"] = line[None], None
                else:     # time, height and width of patches 32 wide
                    st["positions"] = torch.stack((line // 64 + start, at // 32 % 64 + start, at % 32 + start))
                    st["sections"] = (half // 4, half // 8 * 3, half - half // 4 - half // 8 * 3)
    else:
        ql, kl = _lengths(case)
        b, ps = case["batch"], case["page"]
        width = -(-max(kl) // ps) + 1
        used = [-(-n // ps) for n in kl]
        pages = sum(used) + 2
        # every page starts as whatever was there before: rows past a sequence's end are never written
        data = torch.randint(0, 256, (pages, hk, _page_bytes(case)), generator=gen, device="cuda", dtype=torch.uint8)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, u in enumerate(used):
            table[i, :u] = order[at:at + u]
            at += u
        for i, n in enumerate(kl):
            for lo in range(0, n, 32768):
                pos = torch.arange(lo, min(n, lo + 32768), device="cuda")
                k, v = _hidden(gen, (len(pos), hk, d), dtype), _hidden(gen, (len(pos), hk, d), dtype, False)
                _put(case, data, table[i].long()[pos // ps] * ps + pos % ps, k.float(), v.float())
        st["q"] = _hidden(gen, (sum(ql), case["q_heads"], d), dtype)
        st["table"] = table
        st["lengths"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
        st["starts"] = torch.tensor([0] + ql, device="cuda").cumsum(0).to(torch.int32) if max(ql) > 1 else None
        st["max_q"] = max(ql)
    st["data"] = data
    if own:
        st["cache"] = _handle(case, data)
    return st


# ------------------------------------------------------------------------------ the operators

def run(st):
    if own:
        return _run_own(st)
    return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention}[st["case"]["op"]](st)


def _run_own(st):
    case, w = st["case"], _framework()
    if case["op"] == "append":
        if case["axes"]:
            q = w.cache_append(st["cache"], st["k"], st["v"], st["slots"], q=st["q"], positions=st["positions"],
                               cos_sin=st["cos_sin"], sections=st["sections"], interleaved=case["interleaved"])
        else:
            q = w.cache_append(st["cache"], st["k"], st["v"], st["slots"])
        k, v = w.cache_read(st["cache"], st["slots"], _DTYPES[case["dtype"]])
        return {"q": q, "k": k, "v": v} if case["axes"] else {"k": k, "v": v}
    if case["op"] == "read":
        k, v = w.cache_read(st["cache"], st["slots"], _DTYPES[case["dtype"]])
        return {"k": k, "v": v}
    return w.cache_attention(st["q"], st["cache"], st["table"], st["lengths"], cu_q=st["starts"], max_q=st["max_q"],
                             causal=case["causal"], window=case["window"])


def _plain_rotate(st, x):
    """x [T, heads, D] in fp32, turned by the positions."""
    case, cs = st["case"], st["cos_sin"]
    r, half = case["rotary"], case["rotary"] // 2
    if st["sections"] is None:
        axis = torch.zeros(half, dtype=torch.long, device=x.device)
    else:
        axis = torch.repeat_interleave(torch.arange(case["axes"], device=x.device),
                                       torch.tensor(st["sections"], device=x.device))
    pos = st["positions"][axis].T                       # [T, half]
    c, s = cs[:, :half].gather(0, pos)[:, None], cs[:, half:].gather(0, pos)[:, None]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:r]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, x[..., r:]), -1)


def _plain_read(st):
    case, dtype = st["case"], _DTYPES[st["case"]["dtype"]]
    kc, vc, kp, vp = _blocks(case, st["data"])
    page, row = st["slots"] // case["page"], st["slots"] % case["page"]
    return {"k": _values(case, kc[page, :, row], kp[page, :, row]).to(dtype),
            "v": _values(case, vc[page, :, row], vp[page, :, row]).to(dtype)}


def _plain_append(st):
    case, dtype = st["case"], _DTYPES[st["case"]["dtype"]]
    k, out = st["k"].float(), {}
    if case["axes"]:
        k, out["q"] = _plain_rotate(st, k), _plain_rotate(st, st["q"].float()).to(dtype)
    _put(case, st["data"], st["slots"], k, st["v"].float())
    return {**out, **_plain_read(st)}


def _plain_attention(st):
    case, dtype = st["case"], _DTYPES[st["case"]["dtype"]]
    b, hk, d, ps = case["batch"], case["kv_heads"], case["dim"], case["page"]
    shared = case["q_heads"] // hk
    table, n = st["table"].long().clamp_min(0), st["lengths"].long()
    kc, vc, kp, vp = _blocks(case, st["data"][table].transpose(1, 2))     # [B, heads, pages, ...]
    at = torch.arange(table.shape[1] * ps, device=table.device)
    here = (at < n[:, None])[:, None, :, None]
    k = torch.where(here, _values(case, kc, kp).flatten(2, 3), 0.0)        # [B, heads, L, D]
    v = torch.where(here, _values(case, vc, vp).flatten(2, 3), 0.0)
    t = st["max_q"]
    first = torch.arange(b + 1, device=n.device) if st["starts"] is None else st["starts"].long()
    count = first[1:] - first[:-1]
    i = torch.arange(t, device=n.device)
    inside = i < count[:, None]                                            # [B, T]
    rows = (first[:-1, None] + i).clamp_max(st["q"].shape[0] - 1)
    q = st["q"].float()[rows].unflatten(2, (hk, shared)).permute(0, 2, 3, 1, 4).flatten(2, 3)   # [B, heads, shared*T, D]
    s = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    p = (n - count)[:, None] + i                                           # a query's position
    seen = (at < n[:, None])[:, None, :].expand(b, t, len(at))
    if case["causal"]:
        seen = seen & (at <= p[..., None])
    if case["window"]:
        seen = seen & (at > p[..., None] - case["window"])
    seen = seen.repeat(1, shared, 1)[:, None]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(total > 0, total, 1.0)
    o = o.unflatten(2, (shared, t)).permute(0, 3, 1, 2, 4).flatten(2, 3)   # [B, T, q_heads, D]
    return o[inside].to(dtype)


# ------------------------------------------------------------------------------ 64 bits

def _exact_values(case, data, slots):
    """Keys and values of the slots as fp64 [T, kv_heads, D], byte by byte."""
    ps, d, g = case["page"], case["dim"], case["group"]
    r = (slots % ps)[:, None]
    i = torch.arange(d, device=data.device)
    page, heads = (slots // ps)[:, None, None], torch.arange(data.shape[1], device=data.device)[:, None]
    pick = lambda off: data[page, heads, off[:, None, :]]                  # [T, heads, D] bytes    # noqa: E731
    out = []
    for which in (0, 1):
        byte = pick(which * ps * d // 2 + r * (d // 2) + i // 2).long()
        code = torch.where(i % 2 == 1, byte // 16, byte % 16).double()
        where = ps * d + which * ps * (d // g) * 4 + r * (d // g) * 4 + (i // g) * 4
        scale, low = (torch.stack((pick(where + o), pick(where + o + 1)), -1).view(torch.float16)[..., 0].double()
                      for o in (0, 2))
        out.append(code * scale + low)
    return out


def _exact_cached(case, x):
    """fp64 values as the cache holds them."""
    x = x.nan_to_num(nan=0.0, posinf=_LIMIT, neginf=-_LIMIT).clamp(-_LIMIT, _LIMIT)
    out = torch.empty_like(x)
    for g in range(0, case["dim"], case["group"]):
        y = x[..., g:g + case["group"]]
        low = y.min(-1, keepdim=True).values.to(torch.float16).double()
        step = ((y.max(-1, keepdim=True).values - low).clamp(min=0) / 15).to(torch.float16).double()
        code = ((y - low) / step).round().clamp(0, 15)
        out[..., g:g + case["group"]] = torch.where(step > 0, code, 0.0) * step + low
    return out


def _exact_rotate(st, x):
    case = st["case"]
    half, y = case["rotary"] // 2, x.clone()
    ends = [half] if st["sections"] is None else [sum(st["sections"][:j + 1]) for j in range(case["axes"])]
    cs = st["cos_sin"].double()
    for i in range(half):
        axis = next(j for j, e in enumerate(ends) if i < e)
        c, s = cs[st["positions"][axis], i][:, None], cs[st["positions"][axis], half + i][:, None]
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        k, out = st["k"].double(), {}
        if case["axes"]:
            out["q"], k = _exact_rotate(st, st["q"].double()), _exact_rotate(st, k)
        return {**out, "k": _exact_cached(case, k), "v": _exact_cached(case, st["v"].double())}
    if case["op"] == "read":
        return dict(zip("kv", _exact_values(case, st["data"], st["slots"])))
    ql, kl = _lengths(case)
    shared, out, at = case["q_heads"] // case["kv_heads"], [], 0
    for b, (t, n) in enumerate(zip(ql, kl)):
        pos = torch.arange(n, device="cuda")
        k, v = _exact_values(case, st["data"], st["table"][b].long()[pos // case["page"]] * case["page"] + pos % case["page"])
        q = st["q"][at:at + t].double() / math.sqrt(case["dim"])
        at += t
        o = torch.zeros_like(q)
        for i in range(0, t, 256):
            p = n - t + torch.arange(i, min(t, i + 256), device="cuda")
            seen = torch.ones(len(p), n, dtype=torch.bool, device="cuda")
            if case["causal"]:
                seen &= pos <= p[:, None]
            if case["window"]:
                seen &= pos > p[:, None] - case["window"]
            some = seen.any(1)[:, None]
            for h in range(case["q_heads"]):
                s = (q[i:i + 256, h] @ k[:, h // shared].T).masked_fill(~seen, -math.inf)
                w = torch.softmax(torch.where(some, s, 0.0), -1)
                o[i:i + 256, h] = torch.where(some, w @ v[:, h // shared], 0.0)
        out.append(o)
    return torch.cat(out)
