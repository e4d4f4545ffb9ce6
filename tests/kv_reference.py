"""The paged 8-bit cache's operators from their definitions, on the host: whole
numbers in Python, sums in 64 bits, fp32 only where the format itself is fp32
(a quotient rounded from 64 bits to fp32 is the correctly rounded fp32 one)."""

import math

import numpy as np
import torch


def ceil_div(a, b):
    return -(-a // b)


def dhp(dh):
    return 32 if dh <= 32 else 64 if dh <= 64 else 128 if dh <= 128 else 256


# ---------------------------------------------------------------- plan
def plan(old, new, table, free, count, P, max_tokens):
    """(cu_new, cu_pages, positions, slots, info, table, free) as lists."""
    table = [list(r) for r in table]
    free = list(free)
    width = len(table[0])
    cap = width * P
    over = sum(max(0, ceil_div(n, P) - width) for n in new if n > cap)
    old = [min(max(v, 0), cap) for v in old]
    new = [min(max(v, 0), cap) for v in new]
    stack = free[:count]
    for r, (o, n) in enumerate(zip(old, new)):
        stack += table[r][ceil_div(n, P):ceil_div(o, P)]
    for i in range(count, min(len(stack), len(free))):
        free[i] = stack[i]
    lack = 0
    for r, (o, n) in enumerate(zip(old, new)):
        for p in range(ceil_div(o, P), ceil_div(n, P)):
            if stack:
                table[r][p] = stack.pop()
            else:
                table[r][p] = -1
                lack += 1
    cu_new, cu_pages, positions, slots = [0], [0], [], []
    for r, (o, n) in enumerate(zip(old, new)):
        cu_new.append(cu_new[-1] + max(n - o, 0))
        cu_pages.append(cu_pages[-1] + (ceil_div(n, P) if n > o else 0))
        for pos in range(o, n):
            positions.append(pos)
            page = table[r][pos // P]
            slots.append(page * P + pos % P if page >= 0 else -1)
    pad = max_tokens - len(slots)
    return (cu_new, cu_pages, (positions + [-1] * pad)[:max_tokens], (slots + [-1] * pad)[:max_tokens],
            [len(stack), lack + over], table, free)


# ---------------------------------------------------------------- codes
_E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
_E4M3_UP = np.array(sorted((v, c) for c, v in enumerate(_E4M3[:127])), dtype=np.float64)


def e4m3_code(x):
    """Nearest e4m3 float of 64-bit values, ties to the even code, up to 448."""
    mag = np.minimum(np.abs(x), 448.0)
    vals = _E4M3_UP[:, 0]
    i = np.searchsorted(vals, mag, side="right") - 1
    j = np.minimum(i + 1, 126)
    lo, hi = mag - vals[i], vals[j] - mag
    up = (hi < lo) | ((hi == lo) & (i % 2 == 1))
    code = np.where(up, j, i)
    return np.where(np.signbit(x) & (code > 0), code + 128, code).astype(np.uint8)


def decode(codes, kind):
    """64-bit numbers of uint8 codes."""
    return codes.view(np.int8).astype(np.float64) if kind == "int8" else _E4M3[codes]


def encode(x, kind):
    """uint8 codes of 64-bit numbers; -0 is 0, as a code that moves to a larger scale may become."""
    if kind == "int8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    return e4m3_code(x)


def scale_for(amax, kind):
    if not np.isfinite(amax):
        return np.float32(np.nan)
    if kind == "int8":
        return np.float32(np.float64(amax) / 127.0)
    if amax == 0:
        return np.float32(0)
    m, e = math.frexp(float(amax))
    return np.float32(2.0 ** max(e - (9 if m <= 0.875 else 8), -126))


def append(x, slots, codes, scales, kind, P):
    """x [T, H, dh] fp32 numbers (as 64 bits) into codes [pages, H, P, dhp] (uint8) and scales (fp32), in place."""
    T, H, dh = x.shape
    i = 0
    while i < T:
        if slots[i] < 0:
            i += 1
            continue
        j = i + 1
        while j < T and slots[j] == slots[j - 1] + 1 and slots[j] % P:
            j += 1
        page, place = divmod(int(slots[i]), P)
        for h in range(H):
            part = x[i:j, h]
            want = scale_for(np.abs(part).max() if not np.isnan(part).any() else np.nan, kind)
            was = scales[page, h] if place else np.float32(0)
            now = was if (np.isnan(was) or want <= was) else want
            scales[page, h] = now
            if place and now > was:
                f = np.float64(np.float32(np.float64(was) / np.float64(now)))
                held = decode(codes[page, h, :place], kind)
                codes[page, h, :place] = encode(np.float32(held * f).astype(np.float64), kind)
            c = np.zeros((j - i, codes.shape[-1]), dtype=np.uint8)
            if now > 0:
                c[:, :dh] = encode(np.float32(part / np.float64(now)).astype(np.float64), kind)
            codes[page, h, place:place + j - i] = c
        i = j


# ---------------------------------------------------------------- attention
def attention(q, k, v, k_scale, v_scale, kind, table, lens, cu_new, causal, scale):
    """64-bit softmax attention; q [T, Hq, dh] 64-bit, k / v uint8 codes. Also the
    largest |value| that each row may have summed."""
    T, hq, dh = q.shape
    pages, H, P, _ = k.shape
    G = hq // H
    out, vmax = np.zeros((T, hq, dh)), np.zeros((T, hq, 1))
    for r, L in enumerate(lens):
        n, t0 = cu_new[r + 1] - cu_new[r], cu_new[r]
        L = min(L, len(table[r]) * P)
        if n == 0 or L == 0:
            continue
        ids = [table[r][p] for p in range(ceil_div(L, P))]
        there = np.repeat([0 <= i < pages for i in ids], P)[:L]
        ids = [i if 0 <= i < pages else 0 for i in ids]
        for h in range(H):
            with np.errstate(invalid="ignore"):
                kk = (decode(k[ids, h], kind) * k_scale[ids, h].astype(np.float64)[:, None, None]).reshape(-1, k.shape[-1])[:L, :dh]
                vv = (decode(v[ids, h], kind) * v_scale[ids, h].astype(np.float64)[:, None, None]).reshape(-1, k.shape[-1])[:L, :dh]
            for i in range(n):
                see = there & (np.arange(L) <= (L - n + i if causal else L))
                if not see.any():
                    continue
                for g in range(G):
                    s = kk[see] @ q[t0 + i, h * G + g] * scale
                    e = np.exp(s - s.max())
                    out[t0 + i, h * G + g] = (e / e.sum()) @ vv[see]
                    vmax[t0 + i, h * G + g] = np.abs(vv[see]).max()
    return out, vmax
