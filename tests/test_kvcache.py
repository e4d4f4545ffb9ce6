"""CPU tests of the paged key/value cache: refusals on the host, descriptor layouts, the oracle itself."""

import ctypes

import numpy as np
import pytest
import torch

from tests import kv_reference as ref
from tests.conftest import ROOT


@pytest.mark.parametrize("struct,cls", [("b200l_kv_cache", "KVCacheDesc"), ("b200l_kv_plan_desc", "KVPlanDesc"),
                                        ("b200l_kv_rows", "KVRows"), ("b200l_kv_attn_desc", "KVAttnDesc")])
def test_descriptor_layout_matches_header(pkg, tmp_path, struct, cls):
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    D = getattr(pkg._lib, cls)
    names = [f[0] for f in D._fields_]
    src = tmp_path / "layout.c"
    src.write_text(
        '#include <stdio.h>\n#include <stddef.h>\n#include "cobra_b200.h"\nint main(void) {\n'
        f'  printf("%zu\\n", sizeof({struct}));\n'
        + "".join(f'  printf("%zu\\n", offsetof({struct}, {n}));\n' for n in names) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, "-I", str(ROOT / "include"), "-o", str(exe), str(src)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [ctypes.sizeof(D)] + [getattr(D, n).offset for n in names]


def test_packed_descriptors_have_the_structs_layout(pkg):
    """What kvcache.py packs in one step reads back field by field through the ctypes mirrors."""
    from importlib import import_module
    m, L = import_module(pkg.__name__ + ".kvcache"), pkg._lib
    for pack, cls in ((m._pack_cache, L.KVCacheDesc), (m._pack_plan, L.KVPlanDesc), (m._pack_rows, L.KVRows),
                      (m._pack_attn, L.KVAttnDesc)):
        n = sum(3 if t is ctypes.c_int64 * 3 else 1 for _, t in cls._fields_)
        d = cls.from_buffer_copy(pack(*range(1, n + 1)))
        got = []
        for f, t in cls._fields_:
            got += list(getattr(d, f)) if t is ctypes.c_int64 * 3 else [getattr(d, f)]
        assert got == list(range(1, n + 1))


def cache_desc(pkg, **kw):
    d = dict(k=1024, v=1024, k_scale=1024, v_scale=1024, num_pages=4, num_heads=2, page_size=16, head_dim=64, kind=0)
    return pkg._lib.KVCacheDesc(**{**d, **kw})


@pytest.mark.parametrize("change,code,msg", [
    (dict(num_pages=0), -1, "positive"), (dict(num_heads=-1), -1, "positive"), (dict(page_size=48), -1, "page_size"),
    (dict(head_dim=0), -2, "head_dim"), (dict(head_dim=257), -2, "head_dim"), (dict(kind=2), -1, "kind"),
    (dict(num_pages=1 << 40), -1, "2^31"), (dict(k=None), -3, "NULL"), (dict(v_scale=None), -3, "NULL"),
    (dict(k=1032), -8, "aligned"), (dict(k_scale=1026), -8, "aligned")])
def test_bad_caches_are_rejected_on_the_host(pkg, change, code, msg):
    lib = pkg._lib.lib()
    c = cache_desc(pkg, **change)
    rows = pkg._lib.KVRows(k=1024, v=1024, dtype=1)
    assert lib.b200l_kv_append(ctypes.byref(c), ctypes.byref(rows), None, 0, None) == code
    assert msg in pkg._lib.last_error()
    assert lib.b200l_kv_read(ctypes.byref(c), None, 0, None, None, 1, None) == code


def test_bad_calls_are_rejected_on_the_host(pkg):
    lib, L = pkg._lib.lib(), pkg._lib
    c = cache_desc(pkg)
    assert lib.b200l_kv_append(None, None, None, 0, None) == -3
    assert lib.b200l_kv_append(ctypes.byref(c), None, None, 0, None) == -3
    rows = L.KVRows(k=1024, v=1024, dtype=3)
    assert lib.b200l_kv_append(ctypes.byref(c), ctypes.byref(rows), 1024, 1, None) == -1 and "dtype" in L.last_error()
    rows.dtype = 1
    assert lib.b200l_kv_append(ctypes.byref(c), ctypes.byref(rows), 1024, -1, None) == -1
    assert lib.b200l_kv_append(ctypes.byref(c), ctypes.byref(rows), None, 1, None) == -3
    assert lib.b200l_kv_read(ctypes.byref(c), 1024, -1, 1024, 1024, 1, None) == -1
    assert lib.b200l_kv_read(ctypes.byref(c), 1024, 1, 1024, 1024, 7, None) == -1
    assert lib.b200l_kv_plan(None, None) == -3
    plan = dict(old_lens=1024, new_lens=1024, block_table=1024, table_stride=8, free_pages=1024, free_count=1024,
                cu_new=1024, cu_pages=1024, positions=1024, slots=1024, info=1024, requests=4, table_width=8,
                page_size=16, capacity=9, max_tokens=5)
    for change, code, msg in [(dict(requests=0), -1, "requests"), (dict(requests=16385), -1, "requests"),
                              (dict(page_size=8), -1, "page_size"), (dict(table_width=0), -1, "table_width"),
                              (dict(table_width=1 << 29), -1, "table_width"), (dict(table_stride=7), -1, "table_stride"),
                              (dict(max_tokens=-1), -1, "max_tokens"), (dict(capacity=-1), -1, "capacity"),
                              (dict(old_lens=None), -3, "NULL"), (dict(info=None), -3, "NULL"),
                              (dict(slots=None), -3, "NULL"), (dict(free_pages=None), -3, "NULL")]:
        assert lib.b200l_kv_plan(ctypes.byref(L.KVPlanDesc(**{**plan, **change})), None) == code, change
        assert msg in L.last_error()


def test_bad_attention_is_rejected_on_the_host(pkg):
    lib, L = pkg._lib.lib(), pkg._lib
    c = cache_desc(pkg)
    ok = dict(q=1024, out=1024, q_stride_token=256, q_stride_head=64, block_table=1024, table_stride=8, seq_lens=1024,
              cu_new=1024, cu_pages=1024, requests=2, table_width=8, tokens=3, num_heads=4, max_new=2, causal=1, dtype=1,
              scale=0.125)
    assert lib.b200l_kv_attention(None, None, None, 0, None) == -3
    assert lib.b200l_kv_attention(ctypes.byref(c), None, None, 0, None) == -3
    for change, msg in [(dict(requests=0), "requests"), (dict(requests=16385), "requests"), (dict(num_heads=3), "multiple"),
                        (dict(num_heads=0), "multiple"), (dict(tokens=-1), "tokens"), (dict(max_new=-1), "max_new"),
                        (dict(table_width=0), "table_width"), (dict(table_stride=7), "table_stride"),
                        (dict(dtype=0), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")]:
        d = L.KVAttnDesc(**{**ok, **change})
        assert lib.b200l_kv_attention(ctypes.byref(c), ctypes.byref(d), 1024, 1 << 30, None) == -1, change
        assert msg in L.last_error()
        assert lib.b200l_kv_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(d)) == 0


def _functions(pkg):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    c = pkg.new_kv_cache(2, 1, 8, page_size=16, device="cpu")
    x = torch.zeros(1, 1, 8, dtype=torch.float16)
    plan = pkg.KVPlan(i32(2), i32(2), None, None, None)
    return [lambda: pkg.kv_plan(i32(1), i32(1), i32(1, 2), i32(3), i32(1), page_size=16, max_tokens=1),
            lambda: pkg.kv_append(x, x, torch.zeros(1, dtype=torch.int64), c),
            lambda: pkg.kv_read(torch.zeros(1, dtype=torch.int64), c, 8),
            lambda: pkg.kv_attention(x, c, i32(1, 2), i32(1), plan, max_new=1)]


@pytest.mark.parametrize("i", range(4))
def test_no_cpu_path(pkg, i):
    with pytest.raises(RuntimeError, match="no CPU path"):
        _functions(pkg)[i]()


def test_new_cache(pkg):
    c = pkg.new_kv_cache(3, 2, 40, page_size=32, dtype=torch.float8_e4m3fn, device="cpu")
    assert c.k.shape == c.v.shape == (3, 2, 32, 64) and c.k_scale.shape == (3, 2) and c.k.dtype == torch.float8_e4m3fn
    for bad in (dict(num_pages=0), dict(num_heads=0), dict(page_size=8), dict(head_dim=0), dict(head_dim=300)):
        with pytest.raises(ValueError):
            pkg.new_kv_cache(**{**dict(num_pages=3, num_heads=2, head_dim=40, device="cpu"), **bad})
    with pytest.raises(TypeError):
        pkg.new_kv_cache(3, 2, 40, dtype=torch.float16, device="cpu")


def test_oracle_codes():
    """The oracle's e4m3 rounding is torch's, and its int8 scale takes the largest value to the last code."""
    rng = np.random.RandomState(0)
    x = np.clip(rng.randn(20000) * np.exp(rng.uniform(-9, 6, size=20000)), -448, 448)
    assert np.array_equal(ref.decode(ref.encode(x, "fp8"), "fp8"),
                          torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())
    for a in (1e-38, 0.37, 1.0, 65504.0, 3e38):
        assert ref.encode(np.array([a / np.float64(ref.scale_for(a, "int8"))]), "int8").view(np.int8)[0] == 127
        s = np.float64(ref.scale_for(a, "fp8"))
        assert a <= 448 * s and (a > 224 * s or s == 2.0 ** -126)


def test_oracle_plan_by_hand():
    got = ref.plan([20, 0, 33], [21, 16, 0], [[5, 6, -1], [-1, -1, -1], [1, 2, 3]], [8, 9, 0, 0, 0, 0], 2, 16, 20)
    assert got[0] == [0, 1, 17, 17] and got[1] == [0, 2, 3, 3]
    assert got[5][1][0] == 3 and got[4] == [4, 0]          # the last page given back is the first handed out
    assert got[2][:2] == [20, 0] and got[3][:2] == [6 * 16 + 4, 48] and got[3][17:] == [-1] * 3
    assert got[6][:5] == [8, 9, 1, 2, 3]
