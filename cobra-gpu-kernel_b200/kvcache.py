"""A paged key/value cache in 8 bits, and attention over it.

A causal model that has attended to a sequence can go on from it one token (or
one chunk) at a time if it keeps the sequence's keys and values. Here they are
kept as int8 or e4m3 codes with one fp32 scale per page of tokens and head, in
pages that a block table hands to requests. A step is

    plan = kv_plan(old_lens, new_lens, block_table, free_pages, free_count, page_size=..., max_tokens=...)
    kv_append(k, v, plan.slots, cache)                                            # per layer
    ctx = kv_attention(q, cache, block_table, new_lens, plan, max_new=...)        # per layer

with lengths, tables and slots on the GPU throughout: nothing here waits for
the GPU, and every call can be captured in a CUDA graph. ``KVPool`` keeps the
lengths, the table and the free pages between steps. All calls run on the
current stream of their tensors' device through the sm_100a library
(``include/cobra_b200.h``); there is no CPU path.
"""

from __future__ import annotations

import struct
import threading
from typing import Dict, NamedTuple, Optional, Tuple

import torch

from . import _lib
from .workspace import new_workspace

PAGE_SIZES = (16, 32, 64, 128)
_KINDS = {torch.int8: _lib.KV_INT8, torch.float8_e4m3fn: _lib.KV_E4M3}
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


class KVCache(NamedTuple):
    """One layer's cache: codes ``[num_pages, heads, page_size, dhp]`` and fp32
    scales ``[num_pages, heads]`` (dhp: ``padded_head_dim``)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class KVPlan(NamedTuple):
    """What a step's lengths come to (``kv_plan``), on the GPU."""

    cu_new: torch.Tensor      # int32 [requests + 1]: new tokens before each request
    cu_pages: torch.Tensor    # int32 [requests + 1]: pages of requests with new tokens before each request
    positions: torch.Tensor   # int32 [max_tokens]: each new token's position, -1 past the last
    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + place, -1 for none
    info: torch.Tensor        # int32 [2]: free pages left, pages that were missing
    unplaced: Optional[torch.Tensor] = None   # int32 [1]: new tokens past max_tokens


def padded_head_dim(head_dim: int) -> int:
    """Columns of a cached row: head_dim rounded up to 32, 64, 128 or 256."""
    if not 1 <= head_dim <= 256:
        raise ValueError(f"head_dim must be in [1, 256], got {head_dim}")
    return 32 if head_dim <= 32 else 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256


def new_kv_cache(num_pages: int, num_heads: int, head_dim: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.int8, device="cuda") -> KVCache:
    """An empty cache of one layer (codes and scales zero)."""
    if num_pages <= 0 or num_heads <= 0:
        raise ValueError(f"num_pages and num_heads must be positive, got {num_pages}, {num_heads}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if dtype not in _KINDS:
        raise TypeError(f"a cache holds torch.int8 or torch.float8_e4m3fn, got {dtype}")
    shape = (num_pages, num_heads, page_size, padded_head_dim(head_dim))
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return KVCache(k, v, ks, vs)


# ---------------------------------------------------------------- checks
# Each operator asks once whether everything fits (a decode step's calls are
# short); where something does not, the functions here say what.
def _on(index: int, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _ints(dtype: torch.dtype, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")


def _cuda(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        raise RuntimeError(f"{name} is on {t.device}: the cache runs only on CUDA (sm_100a) devices; there is no CPU path")
    return index


def _table_stride(table: torch.Tensor, requests: int) -> int:
    if table.dtype != torch.int32:
        raise TypeError(f"block_table must be torch.int32, got {table.dtype}")
    if table.dim() != 2 or table.shape[0] != requests or table.shape[1] == 0:
        raise ValueError(f"block_table must be [{requests}, width], got {tuple(table.shape)}")
    width = table.shape[1]
    stride, inner = table.stride()
    if (width > 1 and inner != 1) or (requests > 1 and stride < width):
        raise ValueError("block_table's rows must be contiguous and apart")
    return stride if requests > 1 else width


def _refuse_cache(cache: KVCache, head_dim: int, index: int) -> None:
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError(f"cache shapes do not fit: codes {tuple(shape)}, {tuple(v.shape)}, "
                         f"scales {tuple(ks.shape)}, {tuple(vs.shape)}")
    if k.dtype not in _KINDS or v.dtype != k.dtype or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"cache codes must be int8 or float8_e4m3fn and scales float32, got {k.dtype}, {v.dtype}, "
                        f"{ks.dtype}, {vs.dtype}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if any(t.get_device() != index for t in cache):
        raise ValueError(f"cache tensors must be on cuda:{index}")
    raise ValueError(f"cache rows have {shape[3]} columns, head_dim {head_dim} needs {padded_head_dim(head_dim)}")


# Descriptors as the library reads them (the layouts of ``_lib.KVCacheDesc``,
# ``KVPlanDesc``, ``KVRows`` and ``KVAttnDesc``), packed in one step.
_pack_cache = struct.Struct("@PPPPqiiii").pack
_pack_plan = struct.Struct("@PPPqPPPPPPPPiiiii4x").pack
_pack_rows = struct.Struct("@PPqqqqqqi4x").pack
_pack_attn = struct.Struct("@PPqqPqPPPiiiiiiif").pack


def _cache_desc(cache: KVCache, head_dim: int, index: int) -> bytes:
    k, v, ks, vs = cache
    shape = k.shape
    kind = _KINDS.get(k.dtype)
    scales = shape[:2]
    f32 = torch.float32
    if (kind is None or len(shape) != 4 or v.shape != shape or ks.shape != scales or vs.shape != scales or v.dtype != k.dtype
            or ks.dtype != f32 or vs.dtype != f32 or not k.is_contiguous() or not v.is_contiguous()
            or not ks.is_contiguous() or not vs.is_contiguous() or k.get_device() != index or v.get_device() != index
            or ks.get_device() != index or vs.get_device() != index or shape[3] != padded_head_dim(head_dim)):
        _refuse_cache(cache, head_dim, index)
    pages, heads, page, _ = shape
    return _pack_cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, page, head_dim, kind)


# ---------------------------------------------------------------- workspaces
class _Workspace:
    """A workspace of each (device, stream): calls on one stream run one after
    another, so they can share it. (Graphs captured on one stream share it too and
    are not to be replayed at the same time.) A buffer that was outgrown is kept (a
    captured graph may still use it); each is at least twice the one before. A call is
    several launches that hand one another numbers in it, so threads take turns."""

    def __init__(self) -> None:
        self._held: Dict[Tuple[int, int], list] = {}
        self._turns: Dict[Tuple[int, int], threading.Lock] = {}

    def turn(self, index: int, stream: int) -> threading.Lock:
        """To be held from the choice of the buffer to the call's last launch."""
        key = (index, stream)
        return self._turns.get(key) or self._turns.setdefault(key, threading.Lock())

    def get(self, index: int, stream: int) -> Tuple[int, int]:
        """(address, bytes), 0 bytes if there is none yet."""
        held = self._held.get((index, stream))
        return held[-1][:2] if held else (0, 0)

    def grow(self, index: int, stream: int, need: int) -> Tuple[int, int]:
        held = self._held.setdefault((index, stream), [])
        size = max(need, 2 * held[-1][1] if held else 0)
        buf, off = new_workspace(size, torch.device("cuda", index))
        held.append((buf.data_ptr() + off, size, buf))
        return held[-1][:2]

    def check(self) -> None:
        for (index, stream), held in list(self._held.items()):
            with torch.cuda.device(index):
                for ptr, _, _ in list(held):
                    rc = _lib.lib().b200l_read_status(ptr, stream)
                    if rc:
                        message = _lib.last_error()
                        _lib.lib().b200l_clear_status(ptr, stream)
                        raise _lib.B200LError(rc, message)


_workspace = _Workspace()


def kv_check_status() -> None:
    """Synchronise and raise if an attention kernel recorded a device-side
    failure (a bounded wait that ran out) in a workspace of this module."""
    _workspace.check()


def _on_device(call, index: int, *args):
    """call(stream, *args) with device ``index`` current and its current stream."""
    if torch._C._cuda_getDevice() == index:
        return call(torch._C._cuda_getCurrentRawStream(index), *args)
    with torch.cuda.device(index):
        return call(torch._C._cuda_getCurrentRawStream(index), *args)


# ---------------------------------------------------------------- operators
def kv_plan(old_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
            free_count: torch.Tensor, *, page_size: int, max_tokens: int) -> KVPlan:
    """Block table and slots for a step that takes each request from
    ``old_lens`` to ``new_lens`` cached tokens (int32 ``[requests]``; less than
    before: pages are given back, 0: finished).

    ``block_table`` (int32 ``[requests, width]``, rows may be strided) and the
    stack ``free_pages`` (int32 ``[num_pages]``, ``free_count`` int32 ``[1]`` of
    them free) are updated in place; entries that the call reads it does not
    write, so a repeated call gives the same answer. The step is adopted by going
    on from ``new_lens`` and ``info[0]``. Where ``info[1]`` pages were missing,
    their table entries and slots are -1: plan again with other ``new_lens``.
    ``max_tokens`` bounds the new tokens; entries past them are -1. ``unplaced``
    tokens that it left out have no slot although the lengths count them: not to be
    adopted either, for attention would read what their places held before.
    """
    index = _cuda(old_lens, "old_lens")
    R = old_lens.numel()
    i32 = torch.int32
    if (old_lens.dtype != i32 or new_lens.dtype != i32 or free_pages.dtype != i32 or free_count.dtype != i32
            or old_lens.dim() != 1 or new_lens.shape != old_lens.shape or R == 0 or free_pages.dim() != 1
            or free_count.numel() != 1 or not old_lens.is_contiguous() or not new_lens.is_contiguous()
            or not free_pages.is_contiguous() or page_size not in PAGE_SIZES or max_tokens < 0
            or new_lens.get_device() != index or block_table.get_device() != index or free_pages.get_device() != index
            or free_count.get_device() != index):
        _on(index, new_lens=new_lens, block_table=block_table, free_pages=free_pages, free_count=free_count)
        _ints(i32, old_lens=old_lens, new_lens=new_lens, free_pages=free_pages, free_count=free_count)
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if max_tokens < 0:
            raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
        if free_pages.dim() != 1 or free_count.numel() != 1:
            raise ValueError("free_pages must be one-dimensional and free_count a single number")
        raise ValueError(f"old_lens and new_lens must be [requests], got {tuple(old_lens.shape)}, {tuple(new_lens.shape)}")
    stride = _table_stride(block_table, R)
    return _on_device(_plan, index, old_lens, new_lens, block_table, stride, free_pages, free_count, page_size, max_tokens)


def _plan(stream, old_lens, new_lens, table, stride, free_pages, free_count, page_size, max_tokens) -> KVPlan:
    R, width = table.shape
    # One allocation: slots (8 bytes each), then the int32 outputs.
    buf = old_lens.new_empty(3 * max_tokens + 2 * R + 5)
    at = buf.data_ptr()
    slots, positions, cu_new, cu_pages, info, unplaced = torch.unsafe_split_with_sizes(
        buf, (2 * max_tokens, max_tokens, R + 1, R + 1, 2, 1))
    p_pos = at + 8 * max_tokens
    p_new = p_pos + 4 * max_tokens
    p_pages = p_new + 4 * (R + 1)
    p_info = p_pages + 4 * (R + 1)
    rc = _lib.lib().b200l_kv_plan(
        _pack_plan(old_lens.data_ptr(), new_lens.data_ptr(), table.data_ptr(), stride, free_pages.data_ptr(),
                   free_count.data_ptr(), p_new, p_pages, p_pos, at, p_info, p_info + 8, R, width, page_size,
                   free_pages.numel(), max_tokens), stream)
    if rc:
        _lib.check(rc)
    return KVPlan(cu_new, cu_pages, positions, slots.view(torch.int64), info, unplaced)


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: KVCache) -> None:
    """Quantises new keys and values ``[tokens, heads, head_dim]`` (fp32, fp16 or
    bf16, any strides) into ``slots`` (int64 ``[tokens]``, < 0: not stored).

    The tokens of a page share one scale per head: a page written from its first
    place on gets the scale that its tokens need; later tokens grow it where they
    need more, and the codes before them are moved to the new scale. The slots of
    one page have to follow one another in ``slots``, as ``kv_plan`` makes them.
    Values that are not finite make their page's scale not-a-number.
    """
    index = _cuda(k, "k")
    dtype = _DTYPES.get(k.dtype)
    if (dtype is None or v.dtype != k.dtype or k.dim() != 3 or v.shape != k.shape or v.get_device() != index
            or slots.get_device() != index or slots.dtype != torch.int64 or not slots.is_contiguous() or slots.dim() != 1
            or slots.shape[0] < k.shape[0] or cache[0].dim() != 4 or cache[0].shape[1] != k.shape[1]):
        if k.dim() != 3 or v.shape != k.shape:
            raise ValueError(f"k and v must be [tokens, heads, head_dim], got {tuple(k.shape)}, {tuple(v.shape)}")
        if dtype is None or v.dtype != k.dtype:
            raise TypeError(f"k and v must both be fp32, fp16 or bf16, got {k.dtype}, {v.dtype}")
        _on(index, v=v, slots=slots)
        _ints(torch.int64, slots=slots)
        if slots.dim() != 1 or slots.numel() < k.shape[0]:
            raise ValueError(f"slots must be [at least {k.shape[0]}], got {tuple(slots.shape)}")
        if cache.k.dim() != 4:
            _refuse_cache(cache, k.shape[2], index)
        raise ValueError(f"k has {k.shape[1]} heads, the cache {cache.k.shape[1]}")
    T, _, dh = k.shape
    c = _cache_desc(cache, dh, index)
    rows = _pack_rows(k.data_ptr(), v.data_ptr(), *k.stride(), *v.stride(), dtype)
    _on_device(_append, index, c, rows, slots.data_ptr(), T)


def _append(stream, c, rows, slots, T) -> None:
    rc = _lib.lib().b200l_kv_append(c, rows, slots, T, stream)
    if rc:
        _lib.check(rc)


def kv_read(slots: torch.Tensor, cache: KVCache, head_dim: int, *,
            dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the codes of ``slots`` (int64 ``[n]``) stand for,
    ``[n, heads, head_dim]`` each, code times scale in fp32, rounded to ``dtype``;
    slots outside the cache read as 0."""
    index = _cuda(slots, "slots")
    code = _DTYPES.get(dtype)
    if code is None or slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        _ints(torch.int64, slots=slots)
        if slots.dim() != 1:
            raise ValueError(f"slots must be [n], got {tuple(slots.shape)}")
        raise TypeError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
    c = _cache_desc(cache, head_dim, index)
    return _on_device(_read, index, c, slots, cache.k.shape[1], head_dim, dtype, code)


def _read(stream, c, slots, heads, dh, dtype, code) -> Tuple[torch.Tensor, torch.Tensor]:
    n = slots.shape[0]
    k, v = slots.new_empty((2, n, heads, dh), dtype=dtype).unbind()
    if n:
        rc = _lib.lib().b200l_kv_read(c, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code, stream)
        if rc:
            _lib.check(rc)
    return k, v


def kv_attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, plan: KVPlan, *,
                 max_new: int, causal: bool = True, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q K^T) V of new tokens over their requests' cached tokens.

    ``q`` is fp16 or bf16 ``[tokens, query heads, head_dim]`` (contiguous dims),
    request by request as in ``plan.cu_new``; query head h reads key/value head
    h // (query heads // cache heads). Of a request with n new tokens of
    ``seq_lens[r]`` cached ones (int32, the new ones among them), token i sees
    the keys up to its own position, or all with ``causal=False``. ``max_new``:
    no request has more new tokens (it chooses the kernel; 1 for a decode step;
    of a request that has more, rows may come out as not-a-number).
    ``scale`` is head_dim ** -0.5 if not given. A row that sees no key is 0, and
    so are rows past the plan's tokens. Returns ``out``, contiguous, q's dtype.

    Calls on one stream share a workspace, and so do graphs captured on one stream
    (``torch.cuda.graph`` captures all on the same one unless it is given another):
    such graphs must not be replayed at the same time.
    """
    index = _cuda(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    T, hq, dh = q.shape
    st, sh, sd = q.stride()
    cu_new, cu_pages = plan.cu_new, plan.cu_pages
    i32 = torch.int32
    dtype = q.dtype
    R = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    if ((dtype != torch.float16 and dtype != torch.bfloat16) or (sd != 1 and dh > 1) or seq_lens.dtype != i32
            or cu_new.dtype != i32 or cu_pages.dtype != i32 or not seq_lens.is_contiguous() or not cu_new.is_contiguous()
            or not cu_pages.is_contiguous() or cu_new.numel() != R + 1 or cu_pages.numel() != R + 1 or max_new < 0
            or block_table.get_device() != index or seq_lens.get_device() != index or cu_new.get_device() != index
            or cu_pages.get_device() != index):
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"q must be fp16 or bf16, got {dtype}")
        if sd != 1 and dh > 1:
            raise ValueError("q's dims must be contiguous")
        _on(index, block_table=block_table, seq_lens=seq_lens, cu_new=cu_new, cu_pages=cu_pages)
        _ints(i32, seq_lens=seq_lens, cu_new=cu_new, cu_pages=cu_pages)
        if max_new < 0:
            raise ValueError(f"max_new must not be negative, got {max_new}")
        raise ValueError(f"seq_lens [requests] and the plan's sums [requests + 1] do not fit: {tuple(seq_lens.shape)}, "
                         f"{cu_new.numel()}, {cu_pages.numel()}")
    stride = _table_stride(block_table, R)
    if out is None:
        out = q.new_empty((T, hq, dh))
    elif out.shape != q.shape or out.dtype != dtype or out.get_device() != index or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, dtype and device")
    if T == 0:
        return out
    c = _cache_desc(cache, dh, index)
    desc = _pack_attn(q.data_ptr(), out.data_ptr(), st, sh, block_table.data_ptr(), stride, seq_lens.data_ptr(),
                      cu_new.data_ptr(), cu_pages.data_ptr(), R, block_table.shape[1], T, hq, max_new, 1 if causal else 0,
                      _DTYPES[dtype], dh ** -0.5 if scale is None else scale)
    _on_device(_attention, index, index, c, desc)
    return out


def _attention(stream, index, c, desc) -> None:
    L = _lib.lib()
    with _workspace.turn(index, stream):
        ws, size = _workspace.get(index, stream)
        rc = L.b200l_kv_attention(c, desc, ws, size, stream)
        if rc == _lib.ERR_WORKSPACE:
            need = L.b200l_kv_attention_workspace_bytes(c, desc)
            ws, size = _workspace.grow(index, stream, need)
            rc = L.b200l_kv_attention(c, desc, ws, size, stream)
    if rc:
        _lib.check(rc)


# ---------------------------------------------------------------- between steps
class KVPool:
    """What a server keeps of its requests between steps: cached lengths, block
    table and free pages, on the GPU. Row r of each is one place for a request;
    a place is given up by a new length of 0.

        plan = pool.plan(new_lens, max_tokens)
        ...                                      # kv_append and kv_attention, layer by layer
        pool.adopt(new_lens, plan)
    """

    def __init__(self, requests: int, pages_per_request: int, num_pages: int, *, page_size: int = 64, device="cuda") -> None:
        if requests <= 0 or pages_per_request <= 0 or num_pages <= 0:
            raise ValueError("requests, pages_per_request and num_pages must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        i32 = dict(dtype=torch.int32, device=device)
        self.page_size = page_size
        self.lens = torch.zeros(requests, **i32)
        self.block_table = torch.full((requests, pages_per_request), -1, **i32)
        self.free_pages = torch.arange(num_pages, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)

    def plan(self, new_lens: torch.Tensor, max_tokens: int) -> KVPlan:
        """``kv_plan`` from the pool's lengths to ``new_lens`` (int32 ``[requests]``)."""
        return kv_plan(self.lens, new_lens, self.block_table, self.free_pages, self.free_count, page_size=self.page_size,
                       max_tokens=max_tokens)

    def adopt(self, new_lens: torch.Tensor, plan: KVPlan) -> None:
        """Goes on from the lengths and free pages of a plan that missed no pages and placed every token."""
        self.lens.copy_(new_lens)
        self.free_count.copy_(plan.info[:1])


def attend_cached(lib_qkv, views, cache: KVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, plan: KVPlan,
                  max_new: int, causal: bool) -> None:
    """The attention of a cached layer step: ``lib_qkv()`` fills the q / k / v^T
    regions of a workspace with the new tokens, ``views`` are (q, k, v, ctx) on it
    (``workspace_views``); the new keys and values go to the cache, and ctx is
    attention over it."""
    q, k, v, ctx = views
    lib_qkv()
    kv_append(k, v, plan.slots, cache)
    kv_attention(q, cache, block_table, seq_lens, plan, max_new=max_new, causal=causal, out=ctx)


def workspace_views(ws: torch.Tensor, lay: dict, T: int, heads: int):
    """q, k, v and ctx of one sequence of T tokens in a layer workspace (bytes from
    its start; ``_lib.workspace_layout``), as ``[T, heads, head_dim]`` fp16."""
    dh, dhp, sp = lay["dh"], lay["dhp"], lay["sp"]

    def region(name: str, shape) -> torch.Tensor:
        n = 2 * shape[0] * shape[1] * shape[2]
        return ws[lay[name]:lay[name] + n].view(torch.float16).view(shape)

    q, k = (region(n, (heads, T, dhp))[..., :dh].transpose(0, 1) for n in ("q", "k"))
    v = region("vt", (heads, dhp, sp))[:, :dh, :T].permute(2, 0, 1)
    return q, k, v, region("ctx", (T, heads, dh))


def check_step(x: torch.Tensor, d: int, plan: KVPlan) -> None:
    """x of a cached step: fp32 [tokens, d] on the GPU, at most the plan's tokens."""
    if x.dim() != 2 or x.shape[-1] != d or x.shape[0] == 0:
        raise ValueError(f"expected x of shape [tokens, {d}], got {tuple(x.shape)}")
    if x.dtype != torch.float32:
        raise TypeError(f"a cached step takes fp32 x, got {x.dtype}")
    _cuda(x, "x")
    if plan.slots.shape[0] < x.shape[0]:
        raise ValueError(f"x has {x.shape[0]} tokens, the plan slots for {plan.slots.shape[0]}")
