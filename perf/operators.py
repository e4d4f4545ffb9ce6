"""The paged 8-bit key/value cache: what is measured of its operators.

Four operators make up the cache: ``kv_plan`` (block tables and slot maps from
request lengths), ``kv_append`` (new keys and values quantised into the pages),
``kv_read`` (the values that the codes of given slots stand for) and
``kv_attention`` (attention of new tokens over the cache). This file lists
cases of them, makes their inputs, runs them (the framework's kernels where
``own`` is true, a plain form in elementary torch operations otherwise) and
says what each needs to move and compute.

Layout: codes int8 or e4m3 ``[pages, Hkv, P, dhp]``, one fp32 scale per page and
head ``[pages, Hkv]``, dhp = head_dim rounded up to 32/64/128/256; request r's
pages in order are row r of ``block_table``; slot = page * P + place in page.
"""

import math
import random

import numpy as np
import torch

own = False

_KIND = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _pkg():
    from __graft_entry__ import load_package
    return load_package()


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One decode step of a small server: 32 requests grow by a token. All latency.
        dict(name="plan-decode-32", op="plan", requests=32, page=64, ctx_lo=1, ctx_hi=4096, new_lo=1, new_hi=1,
             finish=0.0, idle=0.0, mix=1),
        # A large server's step: finished requests give pages back, idle rows, whole prompts beside single tokens.
        dict(name="plan-mixed-4096", op="plan", requests=4096, page=16, ctx_lo=1, ctx_hi=8192, new_lo=1, new_hi=512,
             finish=0.1, idle=0.2, mix=2),
        # Decode step of the d=128, H=4 layer: one token per request goes into pages that are partly full.
        dict(name="append-decode-64", op="append", requests=64, page=16, hkv=4, dh=32, kind="int8", dtype="fp16",
             ctx_lo=1, ctx_hi=1024, new_lo=1, new_hi=1, mix=3),
        # Ragged prompts of grouped-query heads in bf16, some starting inside a page.
        dict(name="append-ragged-bf16", op="append", requests=24, page=64, hkv=8, dh=128, kind="int8", dtype="bf16",
             ctx_lo=1, ctx_hi=300, new_lo=1, new_hi=2047, mix=4),
        # Whole prompts of the d=1024, H=16 layer, 64 thousand tokens.
        dict(name="append-prompt-fp8", op="append", requests=8, page=64, hkv=16, dh=64, kind="fp8", dtype="fp16",
             ctx_lo=1, ctx_hi=1, new_lo=8192, new_hi=8192, mix=5),
        # Decode of the smallest configuration (B=4, S=128, d=128, H=4): a handful of microseconds.
        dict(name="decode-small", op="attn", requests=4, page=16, hq=4, hkv=4, dh=32, kind="int8", dtype="fp16",
             ctx_lo=100, ctx_hi=127, new_lo=1, new_hi=1, causal=True, mix=6),
        # An ordinary decode batch with grouped heads and ragged contexts, some rows idle.
        dict(name="decode-gqa-64", op="attn", requests=64, page=64, hq=32, hkv=8, dh=128, kind="int8", dtype="bf16",
             ctx_lo=64, ctx_hi=8191, new_lo=0, new_hi=1, causal=True, mix=7),
        # The long context S=100000 (d=1024, H=16), two sequences: few rows, a long axis.
        dict(name="decode-long-100000", op="attn", requests=2, page=64, hq=16, hkv=16, dh=64, kind="fp8", dtype="fp16",
             ctx_lo=99999, ctx_hi=99999, new_lo=1, new_hi=1, causal=True, mix=8),
        # A full server: 256 requests of about eight thousand tokens, 4 GB of cache read per step.
        dict(name="decode-wide-256", op="attn", requests=256, page=64, hq=32, hkv=8, dh=128, kind="int8", dtype="fp16",
             ctx_lo=6000, ctx_hi=8191, new_lo=1, new_hi=1, causal=True, mix=9),
        # Checking guessed tokens: five new tokens per request, wide heads (d=1024, H=4), large pages.
        dict(name="verify-dh256", op="attn", requests=32, page=128, hq=4, hkv=4, dh=256, kind="fp8", dtype="fp16",
             ctx_lo=1, ctx_hi=4000, new_lo=1, new_hi=5, causal=True, mix=10),
        # A chunk of each of a few prompts over what is already cached, beside decoding requests.
        dict(name="chunk-gqa-mixed", op="attn", requests=6, page=32, hq=32, hkv=8, dh=128, kind="int8", dtype="fp16",
             ctx_lo=1000, ctx_hi=9000, new_lo=1, new_hi=2048, causal=True, mix=26),
        # Whole sequences without a causal mask (d=1024, H=16, S near 1000).
        dict(name="prompt-full-h16", op="attn", requests=8, page=64, hq=16, hkv=16, dh=64, kind="int8", dtype="fp16",
             ctx_lo=0, ctx_hi=0, new_lo=900, new_hi=1024, causal=False, mix=12),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    """One more case: operator, types, heads, lengths over the ranges of the listed ones."""
    op = rng.choice(["plan", "append", "append", "attn", "attn", "attn", "attn"])
    mix = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        hi = _log_int(rng, 100, 8192)
        return dict(op=op, requests=_log_int(rng, 1, 4096), page=page, ctx_lo=rng.choice([0, 1, 50]), ctx_hi=hi,
                    new_lo=rng.choice([0, 1]), new_hi=_log_int(rng, 1, 512), finish=rng.choice([0.0, 0.05, 0.2]),
                    idle=rng.choice([0.0, 0.3]), mix=mix)
    kind, dtype = rng.choice(["int8", "fp8"]), rng.choice(["fp16", "bf16"])
    dh = rng.choice([32, 64, 96, 128, 256, 40, 80])
    hkv = rng.choice([1, 2, 4, 5, 8, 16])
    if op == "append":
        requests = _log_int(rng, 1, 256)
        most = max(1, min(8192, (1 << 26) // (requests * hkv * dh)))
        new_hi = _log_int(rng, 1, most)
        return dict(op=op, requests=requests, page=page, hkv=hkv, dh=dh, kind=kind, dtype=dtype, ctx_lo=0,
                    ctx_hi=_log_int(rng, 1, 2000), new_lo=rng.choice([0, 1]), new_hi=new_hi, mix=mix)
    hq = hkv * rng.choice([1, 1, 2, 3, 4, 8])
    shape = rng.choice(["decode", "decode", "verify", "chunk"])
    requests = _log_int(rng, 1, 256 if shape == "decode" else 64 if shape == "verify" else 8)
    # No more cached values than the largest listed case, and the plain form's padded scores in a few GB.
    most = min(2048, math.isqrt((1 << 30) // (requests * hq)))
    new_hi = 1 if shape == "decode" else min(most, rng.randint(2, 8) if shape == "verify" else _log_int(rng, 17, 2048))
    ctx = min((1 << 31) // (requests * hkv * dh), (1 << 30) // (requests * hq * new_hi), 100000)
    ctx_hi = _log_int(rng, 1, max(1, ctx - new_hi))
    return dict(op=op, requests=requests, page=page, hq=hq, hkv=hkv, dh=dh, kind=kind, dtype=dtype,
                ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi, new_lo=rng.choice([0, 1, new_hi]),
                new_hi=new_hi, causal=rng.random() < 0.8, mix=mix)


def _lengths(case):
    """(old, new) lengths of every request: the case's own, whatever the seed of the values."""
    r = random.Random(case["mix"])
    old, new = [], []
    for i in range(case["requests"]):
        o = r.randint(case["ctx_lo"], case["ctx_hi"])
        n = _log_int(r, case["new_lo"], case["new_hi"]) if r.random() < 0.9 else r.choice([case["new_lo"], case["new_hi"]])
        if case["op"] == "plan":
            x = r.random()
            if x < case["finish"]:
                n = -o if r.random() < 0.7 else -r.randint(0, o)       # done, or some guessed tokens taken back
            elif x < case["finish"] + case["idle"]:
                n = 0
        elif i == 0 and n == 0:
            n = 1
        old.append(o)
        new.append(o + n)
    return old, new


def _dhp(dh):
    return 32 if dh <= 32 else 64 if dh <= 64 else 128 if dh <= 128 else 256


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs
def _codes(shape, kind, dh, gen, dev):
    """Codes as a quantiser leaves them: a bell curve, a few channels wider, padding columns zero."""
    gain = 30.0 + 30.0 * (torch.rand(shape[-1], generator=gen, device=dev) < 0.05).float()
    gain[dh:] = 0.0
    c = torch.empty(shape, dtype=_KIND[kind], device=dev)
    step = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):
        part = c[i:i + step]
        x = torch.randn(part.shape, generator=gen, device=dev).mul_(gain)
        if kind == "int8":
            part.copy_(x.round_().clamp_(-127, 127))
        else:
            part.copy_(x.mul_(3.0).clamp_(-448, 448))
    return c


def _scales(shape, kind, gen, dev):
    """Scales that put the values near one; a power of two for e4m3, as the quantiser makes them."""
    s = torch.rand(shape, generator=gen, device=dev).mul_(1.2).sub_(0.6).exp_().div_(30.0)
    return s if kind == "int8" else torch.exp2(torch.floor(torch.log2(s / 3.0)))


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 7919 + 13)
    P, R = case["page"], case["requests"]
    old, new = _lengths(case)
    rnd = np.random.RandomState((seed * 31 + 7) % (1 << 31))
    po = np.array([_ceil(o, P) for o in old], dtype=np.int64)
    pn = np.array([_ceil(n, P) for n in new], dtype=np.int64)
    n = np.array([max(b - a, 0) for a, b in zip(old, new)], dtype=np.int64)
    T = int(n.sum())
    width = int(max(1, np.maximum(po, pn).max())) + 1
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)  # noqa: E731
    st = {"case": dict(case), "op": case["op"], "page": P}
    if case["op"] == "plan":
        held, grown = int(po.sum()), int(np.maximum(pn - po, 0).sum())
        num = held + grown + 64
        ids = rnd.permutation(num).astype(np.int32)
        table = np.full((R, width), -1, dtype=np.int32)
        table[np.arange(width)[None, :] < po[:, None]] = ids[:held]
        free = np.zeros(num, dtype=np.int32)
        free[:num - held] = ids[held:]
        st |= {"old": i32(old), "new": i32(new), "table": i32(table), "free": i32(free),
               "free_count": i32([num - held]), "max_tokens": max(1, T + 5)}
        return st
    kind, dh, hkv, dhp = case["kind"], case["dh"], case["hkv"], _dhp(case["dh"])
    num = int(np.maximum(po, pn).sum()) + 3
    ids = rnd.permutation(num).astype(np.int32)
    table = np.full((R, width), -1, dtype=np.int32)
    table[np.arange(width)[None, :] < pn[:, None]] = ids[:int(pn.sum())]
    req = np.repeat(np.arange(R), n)
    start = np.concatenate([[0], np.cumsum(n)])
    pos = np.arange(T) - start[req] + np.array(old)[req]
    slots = table[req, pos // P].astype(np.int64) * P + pos % P
    st |= {"k_cache": _codes((num, hkv, P, dhp), kind, dh, gen, dev), "v_cache": _codes((num, hkv, P, dhp), kind, dh, gen, dev),
           "k_scale": _scales((num, hkv), kind, gen, dev), "v_scale": _scales((num, hkv), kind, gen, dev), "dh": dh,
           "table": i32(table), "new": i32(new), "cu_new": i32(start),
           "cu_pages": i32(np.concatenate([[0], np.cumsum(np.where(n > 0, pn, 0))])),
           "slots": torch.tensor(slots, device=dev), "positions": i32(pos), "info": i32([3, 0])}
    dtype = _DTYPE[case["dtype"]]
    if case["op"] == "append":
        # Every live token of the pages that the step touches: those before it in a partly filled page, and its own.
        first = [(r, p) for r in range(R) if n[r] for p in range(old[r] - old[r] % P, new[r])]
        fr = np.array(first, dtype=np.int64)
        live = table[fr[:, 0], fr[:, 1] // P].astype(np.int64) * P + fr[:, 1] % P
        st["live"] = torch.tensor(live, device=dev)
        st["k"] = torch.randn(T, hkv, dh, generator=gen, device=dev).mul_(1.3).to(dtype)
        st["v"] = torch.randn(T, hkv, dh, generator=gen, device=dev).to(dtype)
        return st
    st |= {"q": torch.randn(T, case["hq"], dh, generator=gen, device=dev).mul_(2.0).to(dtype), "causal": bool(case["causal"]),
           "max_new": int(n.max()), "max_len": int(max(new))}
    return st


# ---------------------------------------------------------------- one pass
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    b = _pkg()
    if s["op"] == "plan":
        p = b.kv_plan(s["old"], s["new"], s["table"], s["free"], s["free_count"], page_size=s["page"], max_tokens=s["max_tokens"])
        return {"cu_new": p.cu_new, "cu_pages": p.cu_pages, "positions": p.positions, "slots": p.slots, "info": p.info,
                "table": s["table"], "free": s["free"]}
    cache = b.KVCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        b.kv_append(s["k"], s["v"], s["slots"], cache)
        k, v = b.kv_read(s["live"], cache, s["dh"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    plan = b.KVPlan(s["cu_new"], s["cu_pages"], s["positions"], s["slots"], s["info"])
    return {"out": b.kv_attention(s["q"], cache, s["table"], s["new"], plan, max_new=s["max_new"], causal=s["causal"])}


def _plain(s):
    if s["op"] == "plan":
        return _plain_plan(s)
    if s["op"] == "append":
        return _plain_append(s)
    return _plain_attention(s)


def _expand(counts):
    """For each of sum(counts) items: its owner and its place among the owner's."""
    ends = torch.cumsum(counts, 0)
    owner = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    place = torch.arange(owner.numel(), device=counts.device) - (ends - counts)[owner]
    return owner, place


def _plain_plan(s):
    old, new, table, free, P = s["old"].long(), s["new"].long(), s["table"], s["free"], s["page"]
    po, pn = (old + P - 1) // P, (new + P - 1) // P
    n = (new - old).clamp(min=0)
    zero = torch.zeros(1, dtype=torch.int64, device=old.device)
    cu_new = torch.cat([zero, torch.cumsum(n, 0)])
    cu_pages = torch.cat([zero, torch.cumsum(torch.where(n > 0, pn, 0), 0)])
    count = s["free_count"].long()[0]
    rel, grow = (po - pn).clamp(min=0), (pn - po).clamp(min=0)
    r, j = _expand(rel)                                   # pages given back go on top of the free ones
    free[count + torch.arange(r.numel(), device=r.device)] = table[r, pn[r] + j]
    top = count + r.numel()
    r, j = _expand(grow)                                  # new pages come from the top
    k = top - 1 - torch.arange(r.numel(), device=r.device)
    table[r, po[r] + j] = torch.where(k >= 0, free[k.clamp(min=0)], -1)
    r, j = _expand(n)
    positions = torch.full((s["max_tokens"],), -1, dtype=torch.int32, device=old.device)
    slots = torch.full((s["max_tokens"],), -1, dtype=torch.int64, device=old.device)
    pos = old[r] + j
    page = table[r, pos // P].long()
    positions[:pos.numel()] = pos.int()
    slots[:pos.numel()] = torch.where(page >= 0, page * P + pos % P, -1)
    need = grow.sum()
    info = torch.stack([(top - need).clamp(min=0), (need - top).clamp(min=0)]).int()
    return {"cu_new": cu_new.int(), "cu_pages": cu_pages.int(), "positions": positions, "slots": slots, "info": info,
            "table": table, "free": free}


def _plain_quantise(x, slots, codes, scale, P):
    kind, dh = codes.dtype, x.shape[-1]
    raw = codes.view(torch.uint8)                         # (e4m3 tensors are indexed as the bytes that hold them)
    page, place = slots // P, slots % P
    pages, at = torch.unique(page, return_inverse=True)
    shape = (pages.numel(), x.shape[1])
    x = x.float()
    amax = torch.zeros(shape, device=x.device).scatter_reduce(0, at[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    begin = torch.full((pages.numel(),), P, device=x.device).scatter_reduce(0, at, place, "amin")
    if kind == torch.int8:
        cand = amax / torch.full_like(amax, 127.0)
    else:
        m, e = torch.frexp(amax)                          # the least power of two that takes amax to 448 = 0.875 * 2^9
        cand = torch.where(amax > 0, torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 9, e - 8)), 0.0)
    before = torch.where(begin[:, None] == 0, 0.0, scale[pages])
    after = torch.maximum(before, cand)
    was = raw[pages]
    held = was.view(kind).float() * torch.where(after > 0, before / after, 0.0)[:, :, None, None]
    held = held.round() if kind == torch.int8 else held
    older = (torch.arange(P, device=x.device)[None, :] < begin[:, None])[:, None, :, None] & (after > before)[:, :, None, None]
    raw[pages] = torch.where(older, held.to(kind).view(torch.uint8), was)
    scale[pages] = after
    s = after[at][:, :, None]
    c = torch.where(s > 0, x / s, 0.0)
    c = c.round().clamp(-127, 127) if kind == torch.int8 else c
    raw[page, :, place, :dh] = c.to(kind).view(torch.uint8)


def _plain_append(s):
    P, dh, live = s["page"], s["dh"], s["live"]
    _plain_quantise(s["k"], s["slots"], s["k_cache"], s["k_scale"], P)
    _plain_quantise(s["v"], s["slots"], s["v_cache"], s["v_scale"], P)
    page, place = live // P, live % P
    value = lambda c, scale: (c.view(torch.uint8)[page, :, place, :dh].contiguous().view(c.dtype).float() * scale[page][:, :, None]).to(s["k"].dtype)  # noqa: E731
    return {"k": value(s["k_cache"], s["k_scale"]), "v": value(s["v_cache"], s["v_scale"])}


def _plain_attention(s):
    q, P, dh = s["q"], s["page"], s["dh"]
    cu, lens = s["cu_new"].long(), s["new"].long()
    R, hq, hkv = lens.numel(), q.shape[1], s["k_cache"].shape[1]
    G, N, L = hq // hkv, s["max_new"], s["max_len"]
    n = cu[1:] - cu[:-1]
    r, i = _expand(n)
    qp = torch.zeros(R, N, hq, dh, device=q.device)
    qp[r, i] = q.float()
    qp = qp.view(R, N, hkv, G, dh).permute(0, 2, 1, 3, 4).reshape(R, hkv, N * G, dh)
    pages = s["table"][:, :_ceil(L, P)].long().clamp(min=0)

    def values(c, scale):                                 # [R, Hkv, L, dh] in 32 bits
        x = c.view(torch.uint8)[pages][..., :dh].contiguous().view(c.dtype).float() * scale[pages][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(R, hkv, -1, dh)[:, :, :L]

    j = torch.arange(L, device=q.device)
    last = (lens - n)[:, None] + torch.arange(N, device=q.device)[None, :] if s["causal"] else (lens - 1)[:, None].expand(R, N)
    seen = ((j[None, None, :] <= last[:, :, None]) & (j[None, None, :] < lens[:, None, None])).repeat_interleave(G, 1)[:, None]
    a = torch.matmul(qp, values(s["k_cache"], s["k_scale"]).transpose(-1, -2)).mul_(dh ** -0.5)
    a.masked_fill_(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    a.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = a.sum(-1, keepdim=True)
    o = torch.matmul(a, values(s["v_cache"], s["v_scale"]))
    o = torch.where(total > 0, o / total, 0.0)
    o = o.view(R, hkv, N, G, dh).permute(0, 2, 1, 3, 4).reshape(R, N, hq, dh)
    return {"out": o[r, i].to(q.dtype)}


# ---------------------------------------------------------------- work
def work(case):
    old, new = _lengths(case)
    P, R = case["page"], case["requests"]
    n = [max(b - a, 0) for a, b in zip(old, new)]
    T = sum(n)
    if case["op"] == "plan":
        moved = sum(abs(_ceil(b, P) - _ceil(a, P)) for a, b in zip(old, new))
        read = sum(_ceil(b, P) - a // P for a, b, m in zip(old, new, n) if m)      # table entries behind the slots
        return {"bytes": 8 * R + 8 * (R + 1) + 12 * (T + 5) + 8 * moved + 4 * read, "flops": 0}
    hkv, dh = case["hkv"], case["dh"]
    if case["op"] == "append":
        live = sum(b - (a - a % P) for a, b, m in zip(old, new, n) if m)
        touched = sum(_ceil(b, P) - a // P for a, b, m in zip(old, new, n) if m)
        row = 2 * hkv * dh
        # 16-bit inputs, codes written, codes read back, 16-bit values; scales written and read; slots.
        return {"bytes": T * row * 3 + live * row * 3 + 16 * touched * hkv + 8 * (T + live), "flops": 0}
    hq = case["hq"]
    byte = flop = 0
    for a, b, m in zip(old, new, n):
        if m == 0:
            continue
        byte += 2 * hkv * (b * dh + 4 * _ceil(b, P)) + 4 * _ceil(b, P)
        pairs = m * b - (m * (m - 1) // 2 if case["causal"] else 0)
        flop += 4 * dh * hq * pairs
    return {"bytes": byte + 4 * T * hq * dh + 12 * R, "flops": flop}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definition in 64 bits, request by request and head by head. The plan's outputs are whole numbers."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    old, new = _lengths(case)
    P, dh, table = case["page"], case["dh"], s["table"].long()

    def value(codes, scale, rows, h):
        c = codes.view(torch.uint8)[rows, h].view(codes.dtype).double()
        return (c * scale[rows, h].double()[:, None, None]).reshape(-1, codes.shape[-1])[:, :dh]

    if case["op"] == "append":
        return {"k": _exact_append(s, "k", old, new), "v": _exact_append(s, "v", old, new)}
    hq, hkv = case["hq"], case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r in range(case["requests"]):
        L, m = new[r], new[r] - old[r]
        if m == 0:
            continue
        rows = table[r, :_ceil(L, P)]
        row = torch.arange(L - m, L, device="cuda") if case["causal"] else torch.full((m,), L - 1, device="cuda")
        hidden = torch.arange(L, device="cuda")[None, :] > row[:, None]
        for h in range(hkv):
            k = value(s["k_cache"], s["k_scale"], rows, h)[:L]
            v = value(s["v_cache"], s["v_scale"], rows, h)[:L]
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                a = s["q"][at:at + m, g].double() @ k.T / math.sqrt(dh)
                a[hidden] = -math.inf
                out[at:at + m, g] = torch.softmax(a, -1) @ v
        at += m
    return {"out": out}


def _exact_append(s, which, old, new):
    """Values of the live slots after each page's block is scaled anew, page by page on the host."""
    P, dh, x = s["page"], s["dh"], s[which].double().cpu().numpy()
    table = s["table"].cpu().numpy()
    is_int = s["k_cache"].dtype == torch.int8
    codes, scale = s[which + "_cache"], s[which + "_scale"].double().cpu().numpy()

    def rounded(c):
        if is_int:
            return np.clip(np.rint(c), -127, 127)
        step = np.ldexp(1.0, np.maximum(np.frexp(c)[1] - 1, -6) - 3)            # three bits after the leading one
        return np.rint(c / step) * step

    got, at = [], 0
    for o, b, rows in zip(old, new, table):
        p = o
        while p < b:
            page, place = int(rows[p // P]), p % P
            m = min(P - place, b - p)
            new_x = x[at:at + m]
            a = np.abs(new_x).max(axis=(0, 2))
            want = a / 127.0 if is_int else np.exp2(np.ceil(np.log2(a / 448.0)))
            was = scale[page] if place else np.zeros_like(want)
            now = np.maximum(was, want)
            if place:
                held = codes[page, :, :place, :dh].contiguous().double().cpu().numpy()
                held = np.where((now > was)[:, None, None], rounded(held * (was / now)[:, None, None]), held)
                got.append((held * now[:, None, None]).transpose(1, 0, 2))
            got.append(rounded(new_x / now[None, :, None]) * now[None, :, None])
            at += m
            p += m
    return torch.from_numpy(np.concatenate(got))
