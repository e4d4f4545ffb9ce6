"""The paged 8-bit cache on a B200 where a step's numbers lie apart or its calls are at odds."""

from importlib import import_module

import numpy as np
import pytest
import torch

from tests import kv_reference as ref
from tests.test_kvcache_gpu import DTYPE, KIND, TOL, append_and_compare, attention_case, filled_cache, i32, run_attention

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- value scales far apart
def unlike_pages(s, small, order):
    """Values of one size throughout a page: full pages, and pages `small` times
    theirs (0: nothing but zeros, as kv_append leaves them). Keys and queries stay."""
    full = 100 if s["kind"] == "int8" else int(np.flatnonzero(ref._E4M3[:127] == 256.0)[0])
    dh, at = s["dh"], 0
    for row in s["table"]:
        ids = [i for i in row if i >= 0]
        for k, page in enumerate(ids):
            is_full = {"full first": k == 0, "full last": k == len(ids) - 1, "in turn": k % 2 == at % 2}[order]
            s["vc"][page] = 0
            if is_full or small:
                s["vc"][page, :, :, :dh] = full
            s["vs"][page] = np.float32(2.0 ** -6 * (1.0 if is_full else small))
        at += 1
    s["c"].v.view(torch.uint8).copy_(torch.from_numpy(s["vc"]))
    s["c"].v_scale.copy_(torch.from_numpy(s["vs"]))


@pytest.mark.parametrize("order", ["full first", "full last", "in turn"])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -16, 2.0 ** -20, 2.0 ** -24])
@pytest.mark.parametrize("kind,dtype,hq,hkv,dh,P", [
    ("int8", "fp16", 4, 4, 32, 16), ("fp8", "bf16", 8, 2, 64, 16), ("int8", "fp16", 8, 2, 128, 32), ("fp8", "fp16", 2, 1, 256, 16)])
def test_attention_counts_keys_of_small_values(pkg, cuda_ok, kind, dtype, hq, hkv, dh, P, small, order):
    """A key's weight in the denominator is its own, however small its values: two
    pages in one key tile, pages in several, and a context cut over the whole GPU, by
    the kernel for few rows and by the one for many.

    All values are of one sign, so the error is bounded by the output itself: what
    rounds as in TOL, and besides the fp16 weights of the small pages' keys, off by up
    to 2^-25 of the largest, 3100 of them at most: below 2^-13."""
    for lens, new in (([2 * P], [1]), ([2 * P], [5]), ([2 * P + 40], [40]), ([7 * P - 3, 2 * P, 3 * P], [1, 1, 1]),
                      ([3100], [1]), ([700, P + 1], [40, 1])):
        for spread in (0.0, 1.0):
            s = attention_case(pkg, 21 + dh, kind, dtype, hq, hkv, dh, P, lens, new, spread=spread)
            unlike_pages(s, small, order)
            got = run_attention(pkg, s)
            pkg.kv_check_status()
            want, _ = ref.attention(s["q"].double().numpy(), s["kc"], s["vc"], s["ks"], s["vs"], s["kind"], s["table"],
                                    s["lens"], s["cu"], s["causal"], dh ** -0.5)
            err = np.abs(got.double().cpu().numpy() - want)
            bound = (TOL[dtype] + 2.0 ** -13) * np.abs(want) + (2.0 ** -25 if dtype == "fp16" else 0.0)   # fp16's least step
            assert (err <= bound).all(), f"{lens} {new} {spread}: {(err / np.abs(want).clip(1e-30)).max():.3g} of the output"


# ---------------------------------------------------------------- calls at odds with their lengths
@pytest.mark.parametrize("R", [3, 700])
def test_plan_says_how_many_tokens_have_no_slot(pkg, cuda_ok, R):
    P, width = 16, 4
    rng = np.random.RandomState(R)
    new = [int(n) for n in rng.randint(0, width * P + 1, size=R)]
    total = sum(new)
    free = torch.arange(R * width, dtype=torch.int32, device="cuda")
    for most in (0, 1, total - 1, total, total + 3):
        plan = pkg.kv_plan(i32([0] * R), i32(new), i32([[-1] * width] * R), free, i32([R * width]), page_size=P, max_tokens=most)
        assert plan.unplaced.tolist() == [max(total - most, 0)]
        assert plan.cu_new[-1].item() == total and int((plan.slots >= 0).sum()) == min(most, total)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,dh", [(2, 2, 64), (6, 2, 32), (8, 1, 128), (6, 2, 256), (80, 2, 64), (3, 3, 33)])
def test_attention_with_more_new_tokens_than_said(pkg, cuda_ok, hq, hkv, dh, dtype):
    """A max_new below the truth: every row is either right or not-a-number, those within it
    are right, and the other requests' too."""
    group = hq // hkv
    s = attention_case(pkg, 23 + dh, "int8", dtype, hq, hkv, dh, 16, [5, 90, 0, 400, 7, 0], [1, 61, 0, 9, 1, 3])
    want, vmax = ref.attention(s["q"].double().numpy(), s["kc"], s["vc"], s["ks"], s["vs"], s["kind"], s["table"],
                               s["lens"], s["cu"], True, dh ** -0.5)
    plan = pkg.KVPlan(i32(s["cu"]), i32(s["cup"]), None, None, None)
    first = np.concatenate([np.arange(n) for n in s["new"]])      # each row's place in its request
    for said in (0, 1, 2, 5, 40):
        out = torch.full_like(s["q"], 7.0).cuda()
        pkg.kv_attention(s["q"].cuda(), s["c"], i32(s["table"]), i32(s["lens"]), plan, max_new=said, out=out)
        pkg.kv_check_status()
        got = out.double().cpu().numpy()
        lost = np.isnan(got).all(-1)
        assert not lost[first < said].any() and not lost[-3:].any()
        assert lost.any() == (61 * group > 32 and said * group <= 32)
        assert (lost | (np.abs(got - want) <= TOL[dtype] * vmax).all(-1)).all()


# ---------------------------------------------------------------- workspaces of cached steps
def one_prompt(pkg, S, d, H, P=16):
    """Pool, cache, lengths and plan of one request's first S tokens."""
    pool = pkg.KVPool(1, ref.ceil_div(S, P) + 1, ref.ceil_div(S, P) + 1, page_size=P)
    lens = i32([S])
    return pool, pkg.new_kv_cache(ref.ceil_div(S, P) + 1, H, d // H, page_size=P), lens, pool.plan(lens, S)


@pytest.mark.parametrize("d,H,B,S", [(128, 4, 2, 16), (256, 4, 2, 40), (1024, 16, 1, 64)])
def test_forward_before_and_after_a_larger_cached_step(pkg, cuda_ok, d, H, B, S):
    """The layer's captured graph does not outlive the workspace that it was captured on."""
    torch.manual_seed(d)
    lay = pkg.B200TransformerLayer(d, H, True).cuda().eval()
    x, long = torch.randn(B, S, d, device="cuda"), torch.randn(900, d, device="cuda")
    with torch.inference_mode():
        want = lay(x).clone()
        lay(x)
        pool, cache, lens, plan = one_prompt(pkg, 900, d, H)
        lay.forward_cached(long, cache, pool.block_table, lens, plan, max_new=900)
        others = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda") for k in range(8, 23)]
        for _ in range(2):
            assert torch.equal(lay(x), want)
        assert all(bool((t == 7).all()) for t in others)
        lay.check_status()


@pytest.mark.parametrize("stack", [False, True])
def test_captured_cached_step_after_a_larger_one(pkg, cuda_ok, stack):
    """A caller's graph of a cached step, replayed after an eager step that needed a larger
    workspace: the same values, and no other tensor touched."""
    d, H, S, P = 256, 4, 20, 16
    torch.manual_seed(5)
    if stack:
        model = pkg.B200Transformer(pkg.TransformerConfig(1, 8, d, H, ffn_dim=512, num_layers=2, causal=True)).cuda().eval()
        caches = model.new_caches(S // P + 2, page_size=P)
    else:
        model = pkg.B200TransformerLayer(d, H, True).cuda().eval()
    pool, cache, lens, plan = one_prompt(pkg, S, d, H, P)
    first = caches if stack else cache
    x, long = torch.randn(S, d, device="cuda"), torch.randn(700, d, device="cuda")
    step = lambda: model.forward_cached(x, first, pool.block_table, lens, plan, max_new=S)  # noqa: E731
    with torch.inference_mode():
        want = step().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        pool2, cache2, lens2, plan2 = one_prompt(pkg, 700, d, H, P)
        caches2 = model.new_caches(700 // P + 2, page_size=P) if stack else cache2
        model.forward_cached(long, caches2, pool2.block_table, lens2, plan2, max_new=700)
        others = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda") for k in range(8, 23)]
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        assert all(bool((t == 7).all()) for t in others)
        model.check_status()
        pkg.kv_check_status()


# ---------------------------------------------------------------- append
def test_a_step_of_no_tokens(pkg, cuda_ok):
    """Every request idle: plan, append, read and attention take no tokens, and the cache stays."""
    c, held = filled_cache(pkg, np.random.RandomState(24), 6, 2, 64, 16, "int8")
    table, lens = i32([[0, 1], [2, -1]]), i32([20, 7])
    plan = pkg.kv_plan(lens, lens, table, i32([3, 4, 5]), i32([3]), page_size=16, max_tokens=0)
    assert plan.cu_new.tolist() == [0, 0, 0] and plan.slots.shape == (0,) and plan.info.tolist() == [3, 0]
    for dtype in DTYPE.values():
        x = torch.empty(0, 2, 64, dtype=dtype, device="cuda")
        pkg.kv_append(x, x, plan.slots, c)
    assert all(t.shape == (0, 2, 64) for t in pkg.kv_read(plan.slots, c, 64))
    assert pkg.kv_attention(x.half(), c, table, lens, plan, max_new=0).shape == (0, 2, 64)
    for t, h in zip((c.k, c.k_scale, c.v, c.v_scale), held):
        assert np.array_equal(t.view(torch.uint8).cpu().numpy() if t.dtype == torch.int8 else t.cpu().numpy(), h)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_append_values_near_the_least_fp32(pkg, cuda_ok, kind, dtype):
    """A page's largest value a few times 2^-149 (the least bf16 number is 2^-133): an int8
    scale then has few bits, and a quotient may be past 127."""
    rng = np.random.RandomState(22)
    P, H, dh = 16, 2, 32
    unit = 2.0 ** -149 if dtype == "fp32" else 2.0 ** -133
    sizes = [1, 2, 63, 64, 100, 127, 128, 150, 190, 191, 250, 317, 1000, 12345]
    c, held = filled_cache(pkg, rng, len(sizes), H, dh, P, kind)
    for place in (0, 5):                        # a fresh page, then more of the same in it
        x = [np.stack([unit * np.rint(rng.uniform(-n, n, size=(H, dh))) for n in sizes for _ in range(3)]) for _ in range(2)]
        for v in x:
            v[::3, :, 0] = [[unit * n] * H for n in sizes]
            v[1::3, :, 1] = [[-unit * n] * H for n in sizes]
        t = [torch.from_numpy(v).to(DTYPE[dtype]) for v in x]
        slots = np.array([i * P + place + k for i in range(len(sizes)) for k in range(3)], dtype=np.int64)
        append_and_compare(pkg, c, held, t[0].cuda(), t[1].cuda(), *(v.double().numpy() for v in t), slots, kind, P)


def test_a_recorded_failure_stays_until_it_is_read(pkg, cuda_ok):
    """In a workspace that a capture made: neither a later call on its stream nor a replay erases
    what an earlier call recorded, and it is no memory that the graph uses otherwise."""
    s = attention_case(pkg, 25, "int8", "fp16", 4, 2, 64, 16, [90, 3000, 7], [1, 1, 1])
    plan = pkg.KVPlan(i32(s["cu"]), i32(s["cup"]), None, None, None)
    q, table, lens = s["q"].cuda(), i32(s["table"]), i32(s["lens"])
    call = lambda: pkg.kv_attention(q, s["c"], table, lens, plan, max_new=1)  # noqa: E731
    want = call()
    pkg.kv_check_status()
    held = import_module(pkg.__name__ + ".kvcache")._workspace._held
    side = next(st for st in (torch.cuda.Stream() for _ in range(64)) if (0, st.cuda_stream) not in held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        temp = torch.empty(1 << 26, dtype=torch.uint8, device="cuda").fill_(0xff)
        span = (temp.data_ptr(), temp.data_ptr() + temp.numel())
        del temp
        call()                                  # as one layer's step and the next one's
        out = call()
    ptr, buf = held[0, side.cuda_stream][-1][0], held[0, side.cuda_stream][-1][-1]
    assert not span[0] <= ptr < span[1]
    code = buf[ptr - buf.data_ptr():][:4].view(torch.int32)

    def eager():
        with torch.cuda.stream(side):
            return call()

    for _ in range(2):
        for go in (lambda: (graph.replay(), out)[1], eager):
            got = go()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            pkg.kv_check_status()
            code.fill_(-7)
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            with pytest.raises(pkg._lib.B200LError, match="TIMEOUT"):
                pkg.kv_check_status()


@pytest.mark.parametrize("stack", [False, True])
def test_workspace_made_by_a_capture(pkg, cuda_ok, stack):
    """A captured cached step that needs a larger workspace than there was: right at each replay,
    in a second graph replayed before it, and its status block clear from the start."""
    d, H, S, P = 128, 4, 50, 16
    torch.manual_seed(6)
    if stack:
        model = pkg.B200Transformer(pkg.TransformerConfig(1, 8, d, H, ffn_dim=256, num_layers=2, causal=True)).cuda().eval()
        small, caches = model.new_caches(2, page_size=P), model.new_caches(S // P + 2, page_size=P)
    else:
        model = pkg.B200TransformerLayer(d, H, True).cuda().eval()
        small, caches = (pkg.new_kv_cache(n, H, d // H, page_size=P) for n in (2, S // P + 2))
    x = torch.randn(S, d, device="cuda")
    with torch.inference_mode():
        pool, _, lens, plan = one_prompt(pkg, 3, d, H, P)
        model.forward_cached(x[:3], small, pool.block_table, lens, plan, max_new=3)       # packs the weights
        before = model.workspace_ptr
        pool, _, lens, plan = one_prompt(pkg, S, d, H, P)
        graphs, outs = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(model.forward_cached(x, caches, pool.block_table, lens, plan, max_new=S))
        assert model.workspace_ptr != before
        model.check_status()
        for i in (1, 0, 1):
            outs[i].zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        model.check_status()
        pkg.kv_check_status()
        want = model.forward_cached(x, caches, pool.block_table, lens, plan, max_new=S)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and want.any()
