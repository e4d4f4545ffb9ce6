"""The paged 8-bit key/value cache on a B200 against its definitions in 64 bits."""

import random

import numpy as np
import pytest
import torch

from tests import kv_reference as ref

pytestmark = pytest.mark.gpu

KIND = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# What rounds, relative to the largest value a row sums: the output to its type
# (2^-11 of fp16's, 2^-8 of bf16's last-but-one bit, half of it each), the fp16
# weights (2^-11), and fp32 scores up to 2^7 in the exponent (2^-17 each for the
# product and the scale) with the accumulation, together below 2^-14.
TOL = {"fp16": 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -14, "bf16": 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan
def random_step(rng, R, P, width, spare):
    old = [rng.randint(0, width * P) if rng.random() < 0.9 else 0 for _ in range(R)]
    new = []
    for o in old:
        x = rng.random()
        new.append(0 if x < 0.15 else o if x < 0.3 else rng.randint(0, o) if x < 0.4 else
                   min(o + 1, width * P) if x < 0.7 else rng.randint(o, width * P))
    held = [ref.ceil_div(o, P) for o in old]
    need = sum(max(0, ref.ceil_div(n, P) - h) for n, h in zip(new, held))
    num = sum(held) + max(0, int(need * spare))
    ids = list(range(num))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    free = ids[at:] + [-9] * sum(held)
    return old, new, table, free, num - at


@pytest.mark.parametrize("R,P,width,spare,slack", [
    (1, 16, 1, 1.0, 0), (1, 64, 7, 1.0, 3), (3, 16, 5, 1.0, 1), (32, 64, 9, 1.0, 0), (257, 32, 6, 1.2, 7),
    (1000, 16, 4, 0.3, 2), (33, 128, 3, 0.0, 5), (4097, 16, 3, 1.0, 11)])
def test_plan_matches_definition(pkg, cuda_ok, R, P, width, spare, slack):
    rng = random.Random(R * 131 + P)
    old, new, table, free, count = random_step(rng, R, P, width, spare)
    total = sum(max(0, n - o) for o, n in zip(old, new))
    want = ref.plan(old, new, table, free, count, P, total + slack)
    tab = torch.full((R, width + 3), -5, dtype=torch.int32, device="cuda")[:, 1:width + 1]   # rows apart
    tab.copy_(i32(table))
    fr = i32(free)
    for _ in range(2):                  # a repeated call gives the same answer
        p = pkg.kv_plan(i32(old), i32(new), tab, fr, i32([count]), page_size=P, max_tokens=total + slack)
        got = [p.cu_new, p.cu_pages, p.positions, p.slots, p.info, tab, fr]
        for g, w in zip(got, want):
            assert g.tolist() == w


def test_plan_out_of_range_lengths_are_clamped(pkg, cuda_ok):
    P, width = 16, 2
    old, new = [-3, 0, 5], [4, 100, 32]
    table, free = [[-1, -1], [-1, -1], [9, -1]], list(range(20, 30))
    want = ref.plan(old, new, table, free, 10, P, 80)
    tab, fr = i32(table), i32(free)
    p = pkg.kv_plan(i32(old), i32(new), tab, fr, i32([10]), page_size=P, max_tokens=80)
    for g, w in zip([p.cu_new, p.cu_pages, p.positions, p.slots, p.info, tab, fr], want):
        assert g.tolist() == w
    assert p.info.tolist()[1] == 5      # pages past the table's width


def test_plan_short_of_slots_and_many_steps(pkg, cuda_ok):
    """A few hundred steps of a server, adopted one after another, never hand out a page twice."""
    rng = random.Random(3)
    R, P, width, num = 24, 16, 8, 100
    lens, table, free, count = [0] * R, [[-1] * width for _ in range(R)], list(range(num)), num
    tab, fr = i32(table), i32(free)
    cur, cnt = i32(lens), i32([count])
    for step in range(200):
        new = [0 if l and rng.random() < 0.05 else min(width * P, l + rng.choice([0, 1, 1, 1, 40])) for l in lens]
        want = ref.plan(lens, new, table, free, count, P, 128)
        p = pkg.kv_plan(cur, i32(new), tab, fr, cnt, page_size=P, max_tokens=128)
        assert p.info.tolist() == want[4] and p.slots.tolist() == want[3], step
        assert tab.tolist() == want[5] and fr.tolist() == want[6]
        if want[4][1]:                  # pages missing: somebody has to go before it is planned again
            new = [0 if i == max(range(R), key=lambda r: lens[r]) else l for i, l in enumerate(lens)]
            tab, fr = i32(table), i32(free)
            want = ref.plan(lens, new, table, free, count, P, 128)
            p = pkg.kv_plan(cur, i32(new), tab, fr, cnt, page_size=P, max_tokens=128)
            assert p.info.tolist() == want[4]
        lens, table, free, count = new, want[5], want[6], want[4][0]
        cur, cnt = i32(new), p.info[:1]
        live = [t for l, row in zip(lens, table) for t in row[:ref.ceil_div(l, P)]]
        assert len(set(live) | set(free[:count])) == num == len(live) + count


# ---------------------------------------------------------------- append and read
def raw(t):
    return t.view(torch.uint8).cpu().numpy()


def filled_cache(pkg, rng, pages, H, dh, P, kind):
    """Random codes (what a page held before), and scales."""
    c = pkg.new_kv_cache(pages, H, dh, page_size=P, dtype=KIND[kind])
    shape = tuple(c.k.shape)
    out = []
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        code = rng.randint(-127, 128, size=shape).astype(np.int8).view(np.uint8)
        if kind == "fp8":
            code = rng.randint(0, 127, size=shape).astype(np.uint8) | (rng.randint(0, 2, size=shape) << 7).astype(np.uint8)
        code[..., dh:] = 0
        sc = np.exp(rng.uniform(-6, -3, size=shape[:2])).astype(np.float32)
        if kind == "fp8":
            sc = (2.0 ** np.floor(np.log2(sc))).astype(np.float32)
        t.view(torch.uint8).copy_(torch.from_numpy(code))
        s.copy_(torch.from_numpy(sc))
        out += [code, sc]
    return c, out


def random_slots(rng, P, pages, runs):
    """Runs of tokens, each in a page of its own, some skipped tokens between."""
    ids = rng.permutation(pages)[:len(runs)]
    slots = []
    for page, (place, n) in zip(ids, runs):
        slots += [int(page) * P + place + i for i in range(n)]
        if rng.rand() < 0.3:
            slots += [-1] * rng.randint(1, 3)
    return np.array(slots, dtype=np.int64)


def append_and_compare(pkg, c, held, k, v, kk, vv, slots, kind, P):
    pkg.kv_append(k, v, torch.from_numpy(slots).cuda(), c)
    for x, codes, scales, t, s in ((kk, held[0], held[1], c.k, c.k_scale), (vv, held[2], held[3], c.v, c.v_scale)):
        ref.append(x, slots, codes, scales, kind, P)
        assert np.array_equal(s.cpu().numpy(), scales, equal_nan=True)
        got = raw(t)
        assert np.array_equal(ref.decode(got, kind), ref.decode(codes, kind), equal_nan=True)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,dh,P,runs", [
    ("fp16", 4, 32, 16, [(3, 1), (0, 1), (15, 1), (9, 4), (0, 16)]),
    ("bf16", 1, 128, 64, [(0, 64), (60, 4), (1, 63), (0, 1)]),
    ("fp32", 3, 40, 32, [(5, 1), (0, 32), (31, 1)]),
    ("fp16", 2, 256, 128, [(0, 128), (100, 28), (127, 1)]),
    ("fp32", 2, 7, 16, [(0, 3), (2, 9)]),
    ("bf16", 5, 100, 16, [(i % 16, 1) for i in range(70)]),
    ("fp16", 1, 1, 16, [(0, 1)]),
    ("fp16", 8, 64, 64, [(0, 64)] * 40 + [(7, 9), (8, 40)])])
def test_append_matches_definition(pkg, cuda_ok, kind, dtype, H, dh, P, runs):
    rng = np.random.RandomState(len(runs) * 7 + dh)
    c, held = filled_cache(pkg, rng, len(runs) + 5, H, dh, P, kind)
    slots = random_slots(rng, P, len(runs) + 5, runs)
    T = len(slots)
    x = [torch.from_numpy(rng.randn(T, H, dh) * np.exp(rng.uniform(-2, 2, size=(T, 1, 1)))).to(DTYPE[dtype]) for _ in range(2)]
    append_and_compare(pkg, c, held, x[0].cuda(), x[1].cuda(), *(t.double().numpy() for t in x), slots, kind, P)
    # The values that the codes now stand for, and nothing where there is no slot.
    n = c.k.shape[0] * P
    ask = np.concatenate([rng.permutation(n)[:200], [-1, n, 2 ** 40, 0]]).astype(np.int64)
    for out in ("fp16", "bf16", "fp32"):
        got = pkg.kv_read(torch.from_numpy(ask).cuda(), c, dh, dtype=DTYPE[out])
        for g, codes, scales in ((got[0], held[0], held[1]), (got[1], held[2], held[3])):
            val = (ref.decode(codes, kind).astype(np.float32) * scales[:, :, None, None]).transpose(0, 2, 1, 3)
            val = val.reshape(n, H, -1)[..., :dh]
            ok = (ask >= 0) & (ask < n)
            want = np.where(ok[:, None, None], val[np.where(ok, ask, 0)], 0)
            assert torch.equal(g.cpu(), torch.from_numpy(want).to(DTYPE[out]))


def test_append_strides(pkg, cuda_ok):
    """Dims apart (values as the layer keeps them, transposed), rows out of alignment, heads before tokens."""
    rng = np.random.RandomState(5)
    T, H, dh, P = 90, 2, 64, 16
    for make in (lambda x: x.permute(1, 2, 0).contiguous().permute(2, 0, 1),
                 lambda x: torch.cat([x.new_zeros(T, H, 3), x], -1)[..., 3:],
                 lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)):
        c, held = filled_cache(pkg, rng, 12, H, dh, P, "int8")
        slots = np.concatenate([np.arange(5, 48), -np.ones(2), np.arange(100, 145)]).astype(np.int64)
        x = [torch.from_numpy(rng.randn(T, H, dh)).half() for _ in range(2)]
        append_and_compare(pkg, c, held, make(x[0].cuda()), x[1].cuda(), *(t.double().numpy() for t in x), slots, "int8", P)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_append_token_by_token_and_edges(pkg, cuda_ok, kind):
    """A page filled one token a call, its scale growing; zeros, tiny and huge values."""
    rng = np.random.RandomState(6)
    P, H, dh = 16, 2, 32
    c, held = filled_cache(pkg, rng, 3, H, dh, P, kind)
    for i in range(32):
        size = [0.0, 1e-30, 1e-3, 1.0, 1e4, 3e38, 1e-44][i % 7] if i >= 16 else 1.2 ** i
        x = [torch.from_numpy(np.float32(rng.uniform(-1, 1, size=(1, H, dh)) * size)) for _ in range(2)]
        append_and_compare(pkg, c, held, x[0].cuda(), x[1].cuda(), *(t.double().numpy() for t in x),
                           np.array([16 + i], dtype=np.int64), kind, P)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_not_finite(pkg, cuda_ok, kind, bad):
    rng = np.random.RandomState(7)
    P, H, dh = 16, 2, 64
    c, held = filled_cache(pkg, rng, 4, H, dh, P, kind)
    x = [torch.from_numpy(np.float32(rng.randn(6, H, dh))) for _ in range(2)]
    x[0][4, 1, 33] = bad
    slots = np.array([16, 17, 35, 36, 37, 38], dtype=np.int64)
    append_and_compare(pkg, c, held, x[0].cuda(), x[1].cuda(), *(t.double().numpy() for t in x), slots, kind, P)
    assert torch.isnan(c.k_scale).nonzero().tolist() == [[2, 1]] and not torch.isnan(c.v_scale).any()
    # A fresh run in the page clears it.
    y = torch.ones(1, H, dh, device="cuda")
    pkg.kv_append(y, y, torch.tensor([32], device="cuda"), c)
    assert torch.isfinite(c.k_scale).all()


def test_append_does_not_depend_on_how_it_is_cut(pkg, cuda_ok):
    """Whole prompts in one call and each page by itself leave the same codes."""
    rng = np.random.RandomState(8)
    P, H, dh, T = 64, 4, 128, 64 * 40
    k, v = (torch.from_numpy(np.float32(rng.randn(T, H, dh))).half().cuda() for _ in range(2))
    a, b = (pkg.new_kv_cache(40, H, dh, page_size=P) for _ in range(2))
    slots = (torch.randperm(40)[:, None] * P + torch.arange(P)).reshape(-1).cuda()
    pkg.kv_append(k, v, slots, a)
    for i in range(0, T, P):
        pkg.kv_append(k[i:i + P], v[i:i + P], slots[i:i + P].contiguous(), b)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------- attention
def attention_case(pkg, seed, kind, dtype, hq, hkv, dh, P, lens, new, causal=True, spread=1.0, width_extra=1):
    rng = np.random.RandomState(seed)
    need = [ref.ceil_div(l, P) for l in lens]
    pages = sum(need) + 2
    c, (kc, ks, vc, vs) = filled_cache(pkg, rng, pages, hkv, dh, P, kind)
    ids = rng.permutation(pages)
    width = max(need + [1]) + width_extra
    table, at = [], 0
    for m in need:
        table.append([int(i) for i in ids[at:at + m]] + [-1] * (width - m))
        at += m
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1]
    q = torch.from_numpy(rng.randn(T, hq, dh) * spread).to(DTYPE[dtype])
    cup = [0]
    for m, n in zip(need, new):
        cup.append(cup[-1] + (m if n else 0))
    return dict(c=c, kc=kc, ks=ks, vc=vc, vs=vs, table=table, lens=lens, cu=cu, cup=cup, q=q, new=new, kind=kind,
                dtype=dtype, causal=causal, dh=dh)


def run_attention(pkg, s, q=None, **kw):
    plan = pkg.KVPlan(i32(s["cu"]), i32(s["cup"]), None, None, None)
    return pkg.kv_attention(s["q"].cuda() if q is None else q, s["c"], i32(s["table"]), i32(s["lens"]), plan,
                            max_new=max(s["new"]), causal=s["causal"], **kw)


def check_attention(pkg, s, scale=None, got=None):
    got = run_attention(pkg, s, scale=scale) if got is None else got
    pkg.kv_check_status()
    want, vmax = ref.attention(s["q"].double().numpy(), s["kc"], s["vc"], s["ks"], s["vs"], s["kind"], s["table"],
                               s["lens"], s["cu"], s["causal"], s["dh"] ** -0.5 if scale is None else scale)
    err = np.abs(got.double().cpu().numpy() - want)
    bound = TOL[s["dtype"]] * vmax
    assert (err <= bound).all(), f"worst {(err - bound).max():.3g} over a bound of {bound.max():.3g}"
    return got


LENGTHS = [
    ([1], [1]), ([17], [1]), ([64], [1]), ([500], [1]), ([3, 200, 0, 77, 129], [1, 1, 0, 1, 1]),
    ([2000, 1, 333], [1, 1, 1]), ([40, 300, 5], [2, 5, 5]), ([130, 600], [130, 9]), ([260], [260])]


@pytest.mark.parametrize("lens,new", LENGTHS)
@pytest.mark.parametrize("kind,dtype,hq,hkv,dh,P", [
    ("int8", "fp16", 4, 4, 32, 16), ("fp8", "bf16", 8, 2, 64, 64), ("int8", "bf16", 16, 2, 128, 64),
    ("fp8", "fp16", 2, 1, 256, 128), ("int8", "fp16", 6, 2, 96, 32), ("fp8", "fp16", 3, 3, 40, 16),
    ("int8", "fp16", 4, 2, 256, 16), ("fp8", "bf16", 5, 1, 100, 128)])
def test_attention_matches_definition(pkg, cuda_ok, lens, new, kind, dtype, hq, hkv, dh, P):
    for causal in (True, False):
        check_attention(pkg, attention_case(pkg, sum(lens) + dh, kind, dtype, hq, hkv, dh, P, lens, new, causal, spread=2.0))


@pytest.mark.parametrize("dh", [1, 2, 7, 31, 33, 65, 127, 129, 255])
def test_attention_odd_head_dims(pkg, cuda_ok, dh):
    check_attention(pkg, attention_case(pkg, dh, "int8", "fp16", 2, 1, dh, 16, [50, 33], [1, 3]))


@pytest.mark.parametrize("group", [1, 3, 16, 17, 40])
@pytest.mark.parametrize("n", [1, 2, 7])
def test_attention_rows_of_a_tile(pkg, cuda_ok, group, n):
    """Rows that fill a tile, overflow it, and leave most of it empty."""
    check_attention(pkg, attention_case(pkg, group * 10 + n, "int8", "fp16", 2 * group, 2, 64, 32, [n, 100, 65], [n, n, 1]))


def test_attention_many_requests(pkg, cuda_ok):
    """More requests than a probe round finds, a third of them idle, pages cut at odd places."""
    rng = random.Random(9)
    lens = [rng.choice([0, 1, 15, 16, 17, 90, 400]) for _ in range(700)]
    new = [0 if l == 0 or rng.random() < 0.33 else 1 for l in lens]
    for P in (16, 128):
        check_attention(pkg, attention_case(pkg, P, "int8", "fp16", 2, 1, 32, P, lens, new))


@pytest.mark.parametrize("kind,dh,P", [("int8", 128, 64), ("fp8", 64, 16), ("int8", 256, 128), ("fp8", 32, 32)])
def test_attention_long_and_short_together(pkg, cuda_ok, kind, dh, P):
    """One long request cut over the whole GPU beside short ones; same bits every time."""
    s = attention_case(pkg, 11, kind, "fp16", 4, 1, dh, P, [30000, 3, 0, 5000], [1, 1, 0, 1], spread=3.0)
    a = check_attention(pkg, s)
    for _ in range(3):
        assert torch.equal(a, run_attention(pkg, s))


@pytest.mark.parametrize("kind,dh,hq,hkv", [("int8", 32, 8, 4), ("fp8", 64, 4, 4), ("int8", 128, 12, 3), ("fp8", 256, 4, 4)])
def test_attention_many_row_tiles(pkg, cuda_ok, kind, dh, hq, hkv):
    """More row tiles than SMs, ragged, some requests idle, some with a single new token."""
    rng = random.Random(dh)
    new = [rng.choice([0, 0, 1, 60, 129, 200]) for _ in range(90)] + [300]
    lens = [n + rng.choice([0, 0, 1, 37]) for n in new]
    for causal in (True, False):
        check_attention(pkg, attention_case(pkg, dh, kind, "fp16", hq, hkv, dh, 32, lens, new, causal))


def test_attention_empty_rows(pkg, cuda_ok):
    """No keys at all; fewer keys than new tokens (the first rows see none); tokens past the plan's."""
    s = attention_case(pkg, 12, "int8", "fp16", 4, 2, 64, 16, [0, 3, 20], [2, 5, 4])
    s["q"] = torch.cat([s["q"], torch.full((3, 4, 64), float("nan"), dtype=torch.float16)])
    got = run_attention(pkg, s, out=torch.full_like(s["q"], 7.0).cuda())
    check_attention(pkg, {**s, "q": s["q"][:11]}, got=got[:11])
    assert not got[:4].any() and not got[11:].any()
    for n in (1, 40):
        z = attention_case(pkg, 13, "fp8", "bf16", 2, 2, 32, 16, [0, 0], [n, n])
        assert not run_attention(pkg, z, out=torch.full_like(z["q"], 3.0).cuda()).any()


@pytest.mark.parametrize("dh,P", [(32, 16), (64, 64), (128, 32), (256, 128)])
@pytest.mark.parametrize("n", [1, 6, 150])
def test_attention_what_is_hidden_does_not_count(pkg, cuda_ok, dh, P, n):
    """Not-a-number codes and infinite scales behind the last key, in pages of nobody, and in holes of the table."""
    lens = [P + 5 if n < P else n + 3, 3 * P]
    s = attention_case(pkg, 14 + n, "fp8", "fp16", 2, 1, dh, P, lens, [min(n, lens[0]), min(n, 9)])
    last = s["table"][0][ref.ceil_div(lens[0], P) - 1]
    s["kc"][last, :, lens[0] % P:] = 0x7f
    s["vc"][last, :, lens[0] % P:] = 0xff
    used = {i for row in s["table"] for i in row}
    for i in range(s["kc"].shape[0]):
        if i not in used:
            s["kc"][i], s["vc"][i], s["ks"][i], s["vs"][i] = 0x7f, 0x7f, np.nan, np.inf
    s["table"][1][1] = -1               # a hole, and an id past the cache
    s["table"][1][2] = 1 << 30
    for t, x in ((s["c"].k, s["kc"]), (s["c"].v, s["vc"])):
        t.view(torch.uint8).copy_(torch.from_numpy(x))
    s["c"].k_scale.copy_(torch.from_numpy(s["ks"]))
    s["c"].v_scale.copy_(torch.from_numpy(s["vs"]))
    check_attention(pkg, s)
    s["causal"] = False
    check_attention(pkg, s)


def test_attention_not_a_number_where_it_is_seen(pkg, cuda_ok):
    """A poisoned page reaches the rows that see its keys, and no other."""
    for n in (4, 40):
        for which in ("k_scale", "v_scale"):
            s = attention_case(pkg, 15, "int8", "fp16", 2, 2, 64, 16, [64, 80], [n, n])
            page = s["table"][0][3]             # keys 48..63 of request 0
            getattr(s["c"], which)[page, 1] = float("nan")
            got = torch.isnan(run_attention(pkg, s)).all(-1).cpu()
            some = torch.isnan(run_attention(pkg, s)).any(-1).cpu()
            want = torch.zeros(2 * n, 2, dtype=torch.bool)
            for i in range(n):
                want[i, 1] = 64 - n + i >= 48
            assert torch.equal(got, want) and torch.equal(some, want)


def test_attention_scales_far_apart(pkg, cuda_ok):
    """Zero scales, and value scales over thirty octaves: each page's weight is its own."""
    for n in (1, 40):
        s = attention_case(pkg, 16, "int8", "fp16", 2, 1, 64, 16, [200, 64], [n, n])
        rng = np.random.RandomState(1)
        s["vs"][:] = (2.0 ** rng.uniform(-20, 8, size=s["vs"].shape)).astype(np.float32)
        for i in s["table"][1][:4]:             # a request of zeros
            s["vs"][i] = 0
        s["ks"][s["table"][0][2]] = 0
        s["vs"][s["table"][0][5]] = 0
        s["c"].k_scale.copy_(torch.from_numpy(s["ks"]))
        s["c"].v_scale.copy_(torch.from_numpy(s["vs"]))
        check_attention(pkg, s)


def test_attention_large_scores_and_scale(pkg, cuda_ok):
    """Scores in the hundreds (fp32 in the exponent: 2^9 ulp 2^-15 of a weight), and another softmax scale."""
    s = attention_case(pkg, 17, "fp8", "bf16", 4, 2, 64, 32, [300, 100], [1, 1], spread=1.0)
    check_attention(pkg, s, scale=0.4)
    check_attention(pkg, s, scale=0.001)
    tiny = attention_case(pkg, 18, "int8", "bf16", 4, 2, 64, 32, [300, 100], [1, 1], spread=1e-30)
    check_attention(pkg, tiny)
    check_attention(pkg, tiny, scale=1e29)


def test_attention_strides_streams_and_out(pkg, cuda_ok):
    s = attention_case(pkg, 19, "int8", "fp16", 4, 2, 64, 16, [90, 300, 7], [1, 1, 1])
    want = check_attention(pkg, s)
    T = s["q"].shape[0]
    packed = torch.zeros(T, 12, 67, dtype=torch.float16, device="cuda")
    packed[:, 4:8, 1:65] = s["q"].cuda()
    assert torch.equal(want, run_attention(pkg, s, q=packed[:, 4:8, 1:65]))       # rows out of alignment
    by_head = s["q"].cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, run_attention(pkg, s, q=by_head))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_attention(pkg, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    out = torch.empty_like(want)
    assert run_attention(pkg, s, out=out) is out and torch.equal(out, want)


def test_attention_offsets_past_32_bits(pkg, cuda_ok):
    """A cache of 5 GB of keys: pages near its end."""
    P, H, dh = 64, 8, 128
    pages = 5 * (1 << 30) // (P * H * dh)
    c = pkg.KVCache(*(torch.empty((pages, H, P, dh), dtype=torch.int8, device="cuda") for _ in range(2)),
                    *(torch.empty((pages, H), dtype=torch.float32, device="cuda") for _ in range(2)))
    T = 150
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(T, H, dh, device="cuda", generator=g).half() for _ in range(2))
    ids = [pages - 1, pages - 7, 3]
    slots = torch.tensor([ids[i // P] * P + i % P for i in range(T)], device="cuda")
    pkg.kv_append(k, v, slots, c)
    small = pkg.new_kv_cache(3, H, dh, page_size=P)
    near = torch.arange(T, device="cuda")
    pkg.kv_append(k, v, near, small)
    for a, b in zip(pkg.kv_read(slots, c, dh), pkg.kv_read(near, small, dh)):
        assert torch.equal(a, b)
    for n in (1, 100):
        q = torch.randn(n, 16, dh, device="cuda", generator=g).half()
        plan = pkg.KVPlan(i32([0, n]), i32([0, 3]), None, None, None)
        a = pkg.kv_attention(q, c, i32([ids]), i32([T]), plan, max_new=n)
        b = pkg.kv_attention(q, small, i32([[0, 1, 2]]), i32([T]), plan, max_new=n)
        assert torch.equal(a, b) and a.abs().sum() > 0


def test_step_in_a_graph(pkg, cuda_ok):
    """Plan, append and attention captured once and replayed with other lengths."""
    R, P, H, dh, width = 6, 16, 2, 64, 12
    g = torch.Generator(device="cuda").manual_seed(4)
    free, count = torch.arange(R * width, dtype=torch.int32, device="cuda"), i32([R * width])
    table, old, new = i32([[-1] * width] * R), i32([0] * R), i32([1] * R)
    cache = pkg.new_kv_cache(R * width, H, dh, page_size=P)
    k, v = (torch.randn(R, H, dh, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(R, 4, dh, device="cuda", generator=g).half()

    def step():
        p = pkg.kv_plan(old, new, table, free, count, page_size=P, max_tokens=R)
        pkg.kv_append(k, v, p.slots, cache)
        return p, pkg.kv_attention(q, cache, table, new, p, max_new=1)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step()
    keys, vals = [[] for _ in range(R)], [[] for _ in range(R)]
    for t in range(20):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        new.copy_(old + 1)
        graph.replay()
        torch.cuda.synchronize()
        want, vmax = ref.attention(q.double().cpu().numpy(), raw(cache.k), raw(cache.v), cache.k_scale.cpu().numpy(),
                                   cache.v_scale.cpu().numpy(), "int8", table.tolist(), new.tolist(), list(range(R + 1)),
                                   True, dh ** -0.5)
        assert (np.abs(out.double().cpu().numpy() - want) <= TOL["fp16"] * vmax).all()
        old.copy_(new)
        count.copy_(plan.info[:1])


def test_second_graph_before_the_first(pkg, cuda_ok):
    """Two graphs share the workspace that the first capture made; the second one's replay comes first."""
    s = attention_case(pkg, 20, "int8", "fp16", 4, 2, 64, 16, [90, 3000, 7], [1, 1, 1])
    want = check_attention(pkg, s)
    plan = pkg.KVPlan(i32(s["cu"]), i32(s["cup"]), None, None, None)
    q, table, lens = s["q"].cuda(), i32(s["table"]), i32(s["lens"])
    side, outs, graphs = torch.cuda.Stream(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(pkg.kv_attention(q, s["c"], table, lens, plan, max_new=1))
    for i in (1, 0):
        outs[i].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want)
    pkg.kv_check_status()


def test_refusals(pkg, cuda_ok):
    """What Python refuses before the library is asked, with the reason."""
    c = pkg.new_kv_cache(4, 2, 64, page_size=16)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    for err, msg, call in [
            (ValueError, "k and v", lambda: pkg.kv_append(x, x[:2], s, c)),
            (TypeError, "fp32, fp16 or bf16", lambda: pkg.kv_append(x, x.float(), s, c)),
            (TypeError, "slots", lambda: pkg.kv_append(x, x, s.int(), c)),
            (ValueError, "slots", lambda: pkg.kv_append(x, x, s[:2], c)),
            (ValueError, "slots is on", lambda: pkg.kv_append(x, x, s.cpu(), c)),
            (ValueError, "heads", lambda: pkg.kv_append(x[:, :1], x[:, :1], s, c)),
            (ValueError, "columns", lambda: pkg.kv_append(x[..., :9], x[..., :9], s, c)),
            (ValueError, "cache shapes", lambda: pkg.kv_append(x, x, s, c._replace(k_scale=c.k_scale[:3]))),
            (TypeError, "cache codes", lambda: pkg.kv_append(x, x, s, c._replace(k=c.k.view(torch.uint8)))),
            (ValueError, "cache tensors must be on", lambda: pkg.kv_append(x, x, s, c._replace(k=c.k.cpu()))),
            (ValueError, "contiguous", lambda: pkg.kv_append(x, x, s, c._replace(k_scale=torch.zeros(2, 4, device="cuda").T))),
            (TypeError, "dtype", lambda: pkg.kv_read(s, c, 64, dtype=torch.int8)),
            (ValueError, "slots", lambda: pkg.kv_read(s[None], c, 64))]:
        with pytest.raises(err, match=msg):
            call()
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    plan = pkg.KVPlan(i32([0, 2, 3]), i32([0, 1, 2]), None, None, None)
    ok = dict(q=q, cache=c, block_table=i32([[0, 1], [2, 3]]), seq_lens=i32([4, 5]), plan=plan, max_new=2)
    for err, msg, change in [
            (TypeError, "q must be", dict(q=q.float())), (ValueError, "q must be", dict(q=q[0])),
            (ValueError, "contiguous", dict(q=q.transpose(1, 2))), (ValueError, "do not fit", dict(seq_lens=i32([4]))),
            (TypeError, "seq_lens", dict(seq_lens=i32([4, 5]).long())),
            (TypeError, "block_table", dict(block_table=i32([[0, 1], [2, 3]]).long())),
            (ValueError, "block_table", dict(block_table=i32([[0, 1]]))),
            (ValueError, "rows must be", dict(block_table=i32([[0, 1]]).expand(2, 2))),
            (ValueError, "rows must be", dict(block_table=i32([[0, 1], [2, 3]]).T)),
            (ValueError, "max_new", dict(max_new=-1)), (ValueError, "out must", dict(out=q[:2])),
            (ValueError, "is on", dict(block_table=torch.zeros(2, 2, dtype=torch.int32))),
            (pkg._lib.B200LError, "multiple", dict(q=q[:, :3])), (pkg._lib.B200LError, "scale", dict(scale=-1.0))]:
        with pytest.raises(err, match=msg):
            pkg.kv_attention(**{**ok, **change})
    assert pkg.kv_attention(**ok).shape == q.shape
    assert pkg.kv_attention(**{**ok, "q": q[:0]}).shape == (0, 4, 64)
    ok = dict(old_lens=i32([0]), new_lens=i32([3]), block_table=i32([[-1, -1]]), free_pages=i32([0, 1]), free_count=i32([2]),
              page_size=16, max_tokens=3)
    for err, msg, change in [
            (ValueError, "requests", dict(new_lens=i32([1, 2]))), (TypeError, "old_lens", dict(old_lens=i32([0]).long())),
            (ValueError, "page_size", dict(page_size=24)), (ValueError, "max_tokens", dict(max_tokens=-1)),
            (ValueError, "free_count", dict(free_count=i32([1, 2]))), (ValueError, "is on", dict(free_pages=torch.zeros(2).int())),
            (ValueError, "block_table", dict(block_table=i32([[0], [1]])))]:
        with pytest.raises(err, match=msg):
            pkg.kv_plan(**{**ok, **change})
    assert pkg.kv_plan(**ok).slots.tolist() == [16, 17, 18]
