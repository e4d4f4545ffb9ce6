"""Cached steps of the layer and the stack on a B200: plan, append and attention
between the layer's own kernels, against the same layer in 64 bits on the values
that the cache holds (what the codes round is the cache's, not the step's)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def gate(y, want):
    """The reference's gate: abs <= 2e-3 or rel <= 2e-2, every element."""
    err = (y.double() - want).abs()
    return bool(((err <= 2e-3) | (err <= 2e-2 * want.abs())).all())


def attend(att, h, k, v, cu, lens, causal):
    """softmax(q K^T / sqrt(dh)) V in 64 bits; k, v: each request's [len, H, dh]."""
    T, d = h.shape
    H, dh = att.num_heads, att.head_dim
    q = (h @ att.q_proj.weight.double().T + att.q_proj.bias.double()).view(T, H, dh)
    ctx = torch.zeros(T, H, dh, dtype=torch.float64, device=h.device)
    for r, L in enumerate(lens):
        n = cu[r + 1] - cu[r]
        s = torch.einsum("thd,lhd->htl", q[cu[r]:cu[r + 1]], k[r]) * dh ** -0.5
        if causal:
            s.masked_fill_(torch.arange(L, device=s.device)[None, :] > torch.arange(L - n, L, device=s.device)[:, None], -torch.inf)
        ctx[cu[r]:cu[r + 1]] = torch.einsum("htl,lhd->thd", torch.softmax(s, -1), v[r])
    return ctx.view(T, d) @ att.out_proj.weight.double().T + att.out_proj.bias.double()


def norm(m, x):
    return torch.nn.functional.layer_norm(x, x.shape[-1:], m.weight.double(), m.bias.double(), m.eps)


def held(pkg, cache, table, lens, P, dh):
    """Each request's cached keys and values as 64-bit numbers."""
    ks, vs = [], []
    for r, L in enumerate(lens):
        pos = torch.arange(L, device="cuda")
        k, v = pkg.kv_read(table[r].long()[pos // P] * P + pos % P, cache, dh, dtype=torch.float32)
        ks.append(k.double())
        vs.append(v.double())
    return ks, vs


# Prompts (one of them in two chunks, one request waiting), then tokens; a
# request that ends, and another in its place.
STEPS = [[40, 100, 0, 1], [40, 130, 17, 2], [41, 131, 18, 3], [42, 132, 0, 4], [43, 133, 60, 5]]


def steps(pkg, d, P=16):
    """(x, plan, lens before, lens after, cu) of each step on a pool."""
    pool = pkg.KVPool(4, 12, 40, page_size=P)
    g = torch.Generator(device="cuda").manual_seed(d)
    old = [0] * 4
    for new in STEPS:
        n = [max(b - a, 0) for a, b in zip(old, new)]
        cu = [sum(n[:i]) for i in range(5)]
        lens = torch.tensor(new, dtype=torch.int32, device="cuda")
        plan = pool.plan(lens, cu[-1])
        assert plan.info.tolist()[1] == 0
        yield torch.randn(cu[-1], d, device="cuda", generator=g), plan, pool, lens, cu, max(n)
        pool.adopt(lens, plan)
        old = new


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("d,H,causal", [(128, 4, True), (1024, 16, True), (256, 2, False), (96, 3, True), (512, 2, True)])
def test_layer_step_matches_64_bits_on_the_cached_values(pkg, cuda_ok, d, H, causal, dtype):
    torch.manual_seed(1)
    lay = pkg.B200TransformerLayer(d, H, causal).cuda().eval()
    cache = pkg.new_kv_cache(40, H, d // H, page_size=16, dtype=dtype)
    with torch.inference_mode():
        for x, plan, pool, lens, cu, most in steps(pkg, d):
            y = lay.forward_cached(x, cache, pool.block_table, lens, plan, max_new=most)
            lay.check_status()
            pkg.kv_check_status()
            k, v = held(pkg, cache, pool.block_table, lens.tolist(), 16, d // H)
            xd = x.double()
            want = norm(lay.norm2, xd + attend(lay.attention, norm(lay.norm1, xd), k, v, cu, lens.tolist(), causal))
            assert gate(y, want)


def test_cached_values_are_the_layers_own(pkg, cuda_ok):
    """What a step leaves in the cache is K and V of LN1(x), to half a code and the projections' own rounding."""
    d, H, P = 256, 4, 16
    torch.manual_seed(2)
    lay = pkg.B200TransformerLayer(d, H, True).cuda().eval()
    cache = pkg.new_kv_cache(40, H, d // H, page_size=P)
    with torch.inference_mode():
        x, plan, pool, lens, cu, most = next(steps(pkg, d, P))
        lay.forward_cached(x, cache, pool.block_table, lens, plan, max_new=most)
        h, att = norm(lay.norm1, x.double()), lay.attention
        got = held(pkg, cache, pool.block_table, lens.tolist(), P, d // H)
        for proj, values in ((att.k_proj, got[0]), (att.v_proj, got[1])):
            want = (h @ proj.weight.double().T + proj.bias.double()).view(-1, H, d // H)
            for r, L in enumerate(lens.tolist()):
                for p in range(0, L, P):
                    w, g = want[cu[r] + p:cu[r] + min(p + P, L)], values[r][p:p + P]
                    half = w.abs().amax(dim=(0, 2), keepdim=True) / 254
                    assert ((g - w).abs() <= half * 1.01 + 2e-3 + 4e-3 * w.abs()).all()


def test_stack_step_matches_64_bits_on_the_cached_values(pkg, cuda_ok):
    d, H, layers = 128, 4, 3
    torch.manual_seed(3)
    cfg = pkg.TransformerConfig(1, 8, d, H, ffn_dim=256, num_layers=layers, causal=True)
    model = pkg.B200Transformer(cfg).cuda().eval()
    caches = model.new_caches(40, page_size=16)
    with torch.inference_mode():
        for x, plan, pool, lens, cu, most in steps(pkg, d):
            y = model.forward_cached(x, caches, pool.block_table, lens, plan, max_new=most)
            model.check_status()
            pkg.kv_check_status()
            z = x.double()
            for blk, cache in zip(model.layers, caches):
                k, v = held(pkg, cache, pool.block_table, lens.tolist(), 16, d // H)
                z = z + attend(blk.attention, norm(blk.norm1, z), k, v, cu, lens.tolist(), True)
                f = torch.nn.functional.gelu(norm(blk.norm2, z) @ blk.ffn_in.weight.double().T + blk.ffn_in.bias.double())
                z = z + f @ blk.ffn_out.weight.double().T + blk.ffn_out.bias.double()
            assert gate(y, norm(model.final_norm, z))


def test_whole_prompt_in_a_cached_step_is_near_the_plain_forward(pkg, cuda_ok):
    """One causal prompt through the cache against the layer without one: the same
    but for what int8 codes round, half a code of a page's largest value each."""
    d, H, S = 128, 4, 200
    torch.manual_seed(4)
    lay = pkg.B200TransformerLayer(d, H, True).cuda().eval()
    x = torch.randn(S, d, device="cuda")
    pool = pkg.KVPool(1, 16, 16, page_size=16)
    cache = pkg.new_kv_cache(16, H, d // H, page_size=16)
    with torch.inference_mode():
        lens = torch.tensor([S], dtype=torch.int32, device="cuda")
        y = lay.forward_cached(x, cache, pool.block_table, lens, pool.plan(lens, S), max_new=S)
        want = lay(x[None])[0]
        # y = LN2 of about unit variance: an error of ctx reaches it through Wo, of norm about 1.
        assert (y - want).abs().max() < 0.05 and (y - want).pow(2).mean().sqrt() < 0.005


def test_step_refusals(pkg, cuda_ok):
    lay = pkg.B200TransformerLayer(128, 4, True).cuda().eval()
    cache = pkg.new_kv_cache(8, 4, 32, page_size=16)
    pool = pkg.KVPool(2, 4, 8, page_size=16)
    lens = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    plan = pool.plan(lens, 5)
    x = torch.randn(5, 128, device="cuda")
    for err, msg, xx in [(ValueError, "expected x", x[None]), (ValueError, "expected x", x[:, :64]), (TypeError, "fp32", x.half()),
                         (RuntimeError, "no CPU path", x.cpu()), (ValueError, "tokens", torch.cat([x, x]))]:
        with pytest.raises(err, match=msg):
            lay.forward_cached(xx, cache, pool.block_table, lens, plan, max_new=3)
    model = pkg.B200Transformer(pkg.TransformerConfig(1, 8, 128, 4, ffn_dim=256, num_layers=2, causal=True)).cuda().eval()
    with pytest.raises(ValueError, match="caches"):
        model.forward_cached(x, [cache], pool.block_table, lens, plan, max_new=3)
    for bad in (dict(requests=0), dict(page_size=20), dict(num_pages=0)):
        with pytest.raises(ValueError):
            pkg.KVPool(**{**dict(requests=2, pages_per_request=4, num_pages=8), **bad})
