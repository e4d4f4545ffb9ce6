// kv_capi.cuh -- the entry points of the paged 8-bit key/value cache: checks,
// choice of kernel, launches. Part of capi.cu's translation unit (its helpers
// fail(), device_info(), ensure_smem(), make_map(), launch_pdl() are used).
#pragma once

#include "kv_append.cuh"
#include "kv_common.cuh"
#include "kv_decode.cuh"
#include "kv_plan.cuh"
#include "kv_prompt.cuh"

namespace {

int kv_padded(int dh) { return dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 128 ? 128 : 256; }

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

int kv_check_cache(const b200l_kv_cache* c, KvCache* out) {
  if (!c) return fail(B200L_ERR_NULL_POINTER, "cache descriptor is NULL");
  if (c->num_pages <= 0 || c->num_heads <= 0)
    return fail(B200L_ERR_BAD_SHAPE, "num_pages and num_heads must be positive (got %lld, %d)", (long long)c->num_pages,
                c->num_heads);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(B200L_ERR_BAD_SHAPE, "page_size %d: need 16, 32, 64 or 128", c->page_size);
  if (c->head_dim <= 0 || c->head_dim > 256)
    return fail(B200L_ERR_UNSUPPORTED_HEAD_DIM, "head_dim %d: need 1 to 256", c->head_dim);
  if (c->kind != B200L_KV_INT8 && c->kind != B200L_KV_E4M3)
    return fail(B200L_ERR_BAD_SHAPE, "cache kind %d: need B200L_KV_INT8 or B200L_KV_E4M3", c->kind);
  if (c->num_pages > 0x7fffffffLL / ((long long)c->num_heads * c->page_size))
    return fail(B200L_ERR_BAD_SHAPE, "num_pages * num_heads * page_size must stay below 2^31");
  if (c->num_heads > 65535) return fail(B200L_ERR_BAD_SHAPE, "num_heads %d > 65535", c->num_heads);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(B200L_ERR_NULL_POINTER, "a cache tensor is NULL");
  if (misaligned(c->k, 16) || misaligned(c->v, 16)) return fail(B200L_ERR_ALIGNMENT, "cache codes must be 16-byte aligned");
  if (misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4))
    return fail(B200L_ERR_ALIGNMENT, "cache scales must be 4-byte aligned");
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->num_pages = c->num_pages;
  out->heads = c->num_heads;
  out->page = c->page_size;
  out->log2_page = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  return B200L_OK;
}

// ---------------------------------------------------------------- plan
int kv_plan_run(const b200l_kv_plan_desc* d, cudaStream_t st) {
  if (!d) return fail(B200L_ERR_NULL_POINTER, "plan descriptor is NULL");
  if (d->requests <= 0 || d->requests > B200L_KV_MAX_REQUESTS)
    return fail(B200L_ERR_BAD_SHAPE, "requests %d: need 1 to %d", d->requests, B200L_KV_MAX_REQUESTS);
  if (d->page_size != 16 && d->page_size != 32 && d->page_size != 64 && d->page_size != 128)
    return fail(B200L_ERR_BAD_SHAPE, "page_size %d: need 16, 32, 64 or 128", d->page_size);
  const long long most = 1ll << 30;
  if (d->table_width <= 0 || d->max_tokens < 0 || d->capacity < 0 || d->capacity > most || d->max_tokens > most ||
      (long long)d->table_width * d->page_size > most || (long long)d->requests * d->table_width > most)
    return fail(B200L_ERR_BAD_SHAPE, "table_width %d, capacity %d, max_tokens %d: out of range", d->table_width,
                d->capacity, d->max_tokens);
  if (d->table_stride < d->table_width)
    return fail(B200L_ERR_BAD_SHAPE, "table_stride %lld is below table_width %d", (long long)d->table_stride, d->table_width);
  if (!d->old_lens || !d->new_lens || !d->block_table || !d->free_count || !d->cu_new || !d->cu_pages || !d->info ||
      (d->capacity && !d->free_pages) || (d->max_tokens && (!d->positions || !d->slots)))
    return fail(B200L_ERR_NULL_POINTER, "kv_plan: NULL pointer");
  DevInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  KvPlanArgs a;
  a.old_lens = d->old_lens;
  a.new_lens = d->new_lens;
  a.table = d->block_table;
  a.table_stride = d->table_stride;
  a.free_pages = d->free_pages;
  a.free_count = d->free_count;
  a.cu_new = d->cu_new;
  a.cu_pages = d->cu_pages;
  a.positions = d->positions;
  a.slots = reinterpret_cast<long long*>(d->slots);
  a.info = d->info;
  a.unplaced = d->unplaced;
  a.requests = d->requests;
  a.width = d->table_width;
  a.page = d->page_size;
  a.log2_page = d->page_size == 16 ? 4 : d->page_size == 32 ? 5 : d->page_size == 64 ? 6 : 7;
  a.capacity = d->capacity;
  a.max_tokens = d->max_tokens;
  const int threads = d->requests <= 256 ? 256 : 1024;
  const int smem = 3 * (d->requests + 1) * 4;
  if ((rc = ensure_smem((const void*)kv_plan_kernel, 3 * (B200L_KV_MAX_REQUESTS + 1) * 4))) return rc;
  // A block for every few items a thread; one block where that is all there is.
  const long long items = d->max_tokens / 4 + (long long)d->requests * d->table_width / 16;
  const long long want = (items + threads - 1) / threads;
  const int grid = (int)(want < 1 ? 1 : want < dev.sms ? want : dev.sms);
  cudaError_t e = launch_pdl(kv_plan_kernel, dim3(grid), dim3(threads), smem, st, a);
  if (e != cudaSuccess) return cuda_fail(e, "kv_plan_kernel");
  return check_launch("kv_plan_kernel");
}

// ---------------------------------------------------------------- append, read
template <int DHP, int KIND>
int kv_append_t(const KvAppendArgs& a, cudaStream_t st) {
  const int per = 8 / kv_append_group(DHP);      // groups of a block
  const long long blocks = ((long long)a.windows * ((a.c.heads * 2 + a.pairs - 1) / a.pairs) + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(B200L_ERR_BAD_SHAPE, "kv_append: too many tokens and heads");
  cudaError_t e = a.type == B200L_DTYPE_F32
                      ? launch_pdl(kv_append_kernel<DHP, KIND, 4>, dim3((unsigned)blocks), dim3(256), 0, st, a)
                      : launch_pdl(kv_append_kernel<DHP, KIND, 2>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  if (e != cudaSuccess) return cuda_fail(e, "kv_append_kernel");
  return check_launch("kv_append_kernel");
}

template <int DHP, int KIND>
int kv_read_t(const KvReadArgs& a, int sms, cudaStream_t st) {
  const long long blocks = (a.n * a.c.heads * (DHP / 8) + 511) / 512;   // two pieces a lane
  const long long most = 32ll * sms;
  cudaError_t e = launch_pdl(kv_read_kernel<DHP, KIND>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, a);
  if (e != cudaSuccess) return cuda_fail(e, "kv_read_kernel");
  return check_launch("kv_read_kernel");
}

#define KV_DISPATCH(dh, kind, CALL)                                     \
  switch (kv_padded(dh) * 2 + (kind)) {                                 \
    case 64: return CALL(32, kKvInt8);                                  \
    case 65: return CALL(32, kKvE4M3);                                  \
    case 128: return CALL(64, kKvInt8);                                 \
    case 129: return CALL(64, kKvE4M3);                                 \
    case 256: return CALL(128, kKvInt8);                                \
    case 257: return CALL(128, kKvE4M3);                                \
    case 512: return CALL(256, kKvInt8);                                \
    default: return CALL(256, kKvE4M3);                                 \
  }

int kv_append_run(const b200l_kv_cache* cache, const b200l_kv_rows* rows, const int64_t* slots, int64_t tokens,
                  cudaStream_t st) {
  KvAppendArgs a;
  int rc = kv_check_cache(cache, &a.c);
  if (rc) return rc;
  if (!rows) return fail(B200L_ERR_NULL_POINTER, "kv_append: rows descriptor is NULL");
  if (tokens < 0 || tokens > (1ll << 30)) return fail(B200L_ERR_BAD_SHAPE, "kv_append: %lld tokens", (long long)tokens);
  if (rows->dtype < 0 || rows->dtype > 2)
    return fail(B200L_ERR_BAD_SHAPE, "kv_append: dtype must be B200L_DTYPE_F32 / _F16 / _BF16");
  if (tokens && (!rows->k || !rows->v || !slots)) return fail(B200L_ERR_NULL_POINTER, "kv_append: k, v or slots is NULL");
  DevInfo dev;
  if ((rc = device_info(&dev))) return rc;
  if (tokens == 0) return B200L_OK;
  const int esz = rows->dtype == B200L_DTYPE_F32 ? 4 : 2, piece = 16 / esz;
  a.x[0] = rows->k;
  a.x[1] = rows->v;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? rows->v_strides : rows->k_strides;
    a.st[i] = s[0];
    a.sh[i] = s[1];
    a.sd[i] = s[2];
    if (misaligned(a.x[i], esz)) return fail(B200L_ERR_ALIGNMENT, "kv_append: k or v is not aligned to its elements");
    a.vec[i] = s[2] == 1 && s[0] % piece == 0 && s[1] % piece == 0 && !misaligned(a.x[i], 16);
  }
  a.slots = reinterpret_cast<const long long*>(slots);
  a.tokens = tokens;
  a.num_slots = cache->num_pages * cache->page_size;
  a.type = rows->dtype;
  a.dh = cache->head_dim;
  // Windows from a token per warp to 64 tokens a group, while there are 128
  // warps for every SM.
  const int gw = kv_append_group(kv_padded(a.dh));
  a.window = gw;
  while (a.window < 64 && tokens * cache->num_heads * 2 / (a.window * 2) * gw >= 128ll * dev.sms) a.window *= 2;
  a.windows = (int)((tokens + a.window - 1) / a.window);
  a.pairs = 1;                                    // beyond that, several heads a group
  while (a.pairs < 8 && a.window == 64 && (long long)a.windows * cache->num_heads * 2 / (a.pairs * 2) * gw >= 128ll * dev.sms)
    a.pairs *= 2;
#define KV_CALL(D, K) kv_append_t<D, K>(a, st)
  KV_DISPATCH(cache->head_dim, cache->kind, KV_CALL)
#undef KV_CALL
}

int kv_read_run(const b200l_kv_cache* cache, const int64_t* slots, int64_t n, void* k_out, void* v_out, int dtype,
                cudaStream_t st) {
  KvReadArgs a;
  int rc = kv_check_cache(cache, &a.c);
  if (rc) return rc;
  if (n < 0 || n > (1ll << 30)) return fail(B200L_ERR_BAD_SHAPE, "kv_read: %lld slots", (long long)n);
  if (dtype < 0 || dtype > 2) return fail(B200L_ERR_BAD_SHAPE, "kv_read: dtype must be B200L_DTYPE_F32 / _F16 / _BF16");
  DevInfo dev;
  if ((rc = device_info(&dev))) return rc;
  if (n == 0) return B200L_OK;
  if (!slots || !k_out || !v_out) return fail(B200L_ERR_NULL_POINTER, "kv_read: NULL pointer");
  const size_t align = cache->head_dim % 8 == 0 ? 16 : dtype == B200L_DTYPE_F32 ? 4 : 2;   // rows in 16-byte pieces, or element by element
  if (misaligned(k_out, align) || misaligned(v_out, align))
    return fail(B200L_ERR_ALIGNMENT, "kv_read: outputs must be %zu-byte aligned", align);
  a.slots = reinterpret_cast<const long long*>(slots);
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.n = n;
  a.num_slots = cache->num_pages * cache->page_size;
  a.type = dtype;
  a.dh = cache->head_dim;
#define KV_CALL(D, K) kv_read_t<D, K>(a, dev.sms, st)
  KV_DISPATCH(cache->head_dim, cache->kind, KV_CALL)
#undef KV_CALL
}

// ---------------------------------------------------------------- attention
struct KvAttnPlan {
  KvAttnArgs a;
  int dhp;
  bool prompt;                   // kv_prompt_kernel; else kv_decode_kernel
  int M, workers;                // decode: rows of a tile, warps
  int tiles, blocks;             // prompt: row tiles, stretches
  long long pieces;              // row tiles that the workspace holds
  size_t off_plan, off_o, total;
};

int kv_attn_plan(const b200l_kv_cache* cache, const b200l_kv_attn_desc* d, KvAttnPlan* p) {
  KvAttnArgs& a = p->a;
  int rc = kv_check_cache(cache, &a.c);
  if (rc) return rc;
  if (!d) return fail(B200L_ERR_NULL_POINTER, "attention descriptor is NULL");
  if (d->requests <= 0 || d->requests > B200L_KV_MAX_REQUESTS)
    return fail(B200L_ERR_BAD_SHAPE, "requests %d: need 1 to %d", d->requests, B200L_KV_MAX_REQUESTS);
  if (d->num_heads <= 0 || d->num_heads % cache->num_heads != 0)
    return fail(B200L_ERR_BAD_SHAPE, "%d query heads must be a positive multiple of the cache's %d", d->num_heads,
                cache->num_heads);
  if (d->tokens < 0 || d->max_new < 0 || d->tokens > (1 << 30))
    return fail(B200L_ERR_BAD_SHAPE, "tokens %d and max_new %d must not be negative", d->tokens, d->max_new);
  if (d->table_width <= 0 || (long long)d->table_width * cache->page_size > (1ll << 30) ||
      (long long)d->requests * d->table_width > (1ll << 30) || d->table_stride < d->table_width)
    return fail(B200L_ERR_BAD_SHAPE, "table_width %d, table_stride %lld: out of range", d->table_width,
                (long long)d->table_stride);
  if (d->dtype != B200L_DTYPE_F16 && d->dtype != B200L_DTYPE_BF16)
    return fail(B200L_ERR_BAD_SHAPE, "kv_attention: dtype must be B200L_DTYPE_F16 or _BF16");
  if (!(d->scale > 0.f) || !(d->scale < 1e30f)) return fail(B200L_ERR_BAD_SHAPE, "softmax scale %g must be positive", d->scale);
  a.q = d->q;
  a.out = d->out;
  a.q_st = d->q_stride_token;
  a.q_sh = d->q_stride_head;
  a.table = d->block_table;
  a.table_stride = d->table_stride;
  a.lens = d->seq_lens;
  a.cu_new = d->cu_new;
  a.cu_pages = d->cu_pages;
  a.requests = d->requests;
  a.width = d->table_width;
  a.tokens = d->tokens;
  a.hq = d->num_heads;
  a.group = d->num_heads / cache->num_heads;
  a.dh = cache->head_dim;
  a.type = d->dtype;
  a.causal = d->causal ? 1 : 0;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  a.q_vec = a.q_st % 4 == 0 && a.q_sh % 4 == 0 && !misaligned(d->q, 8);
  a.q_vec8 = a.q_st % 8 == 0 && a.q_sh % 8 == 0 && !misaligned(d->q, 16);
  a.o_vec8 = a.dh % 8 == 0 && !misaligned(d->out, 16);
  p->dhp = kv_padded(a.dh);
  if ((long long)d->tokens * a.group > (1ll << 30))
    return fail(B200L_ERR_BAD_SHAPE, "%d tokens of %d query heads per key head: too many rows", d->tokens, a.group);
  const int rows = (d->max_new < d->tokens ? d->max_new : d->tokens) * a.group;
  DevInfo dev;
  if ((rc = device_info(&dev))) return rc;
  // A request's rows fit one or two tiles of mma.sync, whose kernel is bound by
  // HBM; beyond, tcgen05's 128-row tiles. Both at 33 to 64 rows (8 key heads, int8, us,
  // the few-row kernel in several row tiles first): one request of 30000 tokens
  // 61-68 against 43-44 at head_dim 64, 138-143 against 56-57 at 128, 144-160 against
  // 94-95 at 256; 64 requests of 4000 219-230 against 247-255, 357-372 against
  // 348-352, 654-863 against 564-571. (At 32 rows the few-row kernel takes 80, 178 and
  // 145 on the one long request, 133, 213 and 451 on the 64.)
  p->prompt = rows > 32;
  if (p->prompt) {
    const int mq = p->dhp == 256 ? 128 : 256;
    p->M = mq;
    p->workers = 0;
    a.row_tiles = a.min_units = a.whole = a.log2_unit = 0;
    p->tiles = (int)((long long)d->tokens * a.group / mq) + (d->requests < d->tokens ? d->requests : d->tokens);
    p->blocks = dev.sms;
    p->pieces = 2ll * p->blocks;
  } else {
    p->tiles = p->blocks = 0;
    p->M = rows <= 8 ? 8 : rows <= 16 || p->dhp == 256 ? 16 : 32;
    a.row_tiles = rows > p->M ? (rows + p->M - 1) / p->M : 1;
    const int tk = p->dhp == 256 ? 16 : p->dhp == 128 ? 32 : 64;
    const int unit = cache->page_size < tk ? cache->page_size : tk;
    a.log2_unit = unit == 16 ? 4 : unit == 32 ? 5 : 6;
    a.min_units = 2 * tk / unit;
    // Up to four key tiles a pair: a warp is done with them sooner than two
    // launches are (4 requests of 126 tokens, 4 heads of 32: 8.6 against 11.9 us).
    a.whole = d->table_width * cache->page_size <= 4 * tk;
    // Every SM full, but no more blocks than full tables would have work for.
    const int full = dev.sms * (p->dhp * p->M >= 4096 || p->M == 32 ? 2 : 3);
    const long long units = (long long)cache->num_heads * a.row_tiles * d->requests * d->table_width * (cache->page_size / unit);
    const long long blocks = (units + 4ll * a.min_units - 1) / (4ll * a.min_units);
    p->workers = 4 * (int)(blocks < full ? blocks : full);
    p->pieces = 2ll * p->workers;
  }
  p->off_plan = 1024;
  p->off_o = p->prompt ? align_up(p->off_plan + ((size_t)p->tiles + p->blocks + 1) * 16 + ((size_t)p->tiles + 1) * 4, 1024) : 1024;
  p->total = align_up(p->off_o + (size_t)p->pieces * p->M * (p->dhp + 2) * 4, 1024);
  a.part_o = nullptr;
  a.part_ml = nullptr;
  return B200L_OK;
}

template <int DHP, int KIND, int NR>
int kv_decode_t(KvAttnPlan& p, uint8_t* ws, cudaStream_t st) {
  using C = KvDecCfg<DHP, NR>;
  KvAttnArgs& a = p.a;
  CUtensorMap mk, mv;
  const unsigned long long dims[2] = {(unsigned long long)DHP, (unsigned long long)(a.c.num_pages * a.c.heads * a.c.page)};
  const unsigned long long strides[1] = {(unsigned long long)DHP};
  const unsigned box[2] = {(unsigned)C::ROWB, (unsigned)(a.c.page < C::TK ? a.c.page : C::TK)};
  const CUtensorMapSwizzle swz = DHP == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : DHP == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  int rc = make_map(&mk, a.c.k, 2, dims, strides, box, swz, "k codes", CU_TENSOR_MAP_DATA_TYPE_UINT8);
  if (rc) return rc;
  if ((rc = make_map(&mv, a.c.v, 2, dims, strides, box, swz, "v codes", CU_TENSOR_MAP_DATA_TYPE_UINT8))) return rc;
  auto kern = kv_decode_kernel<DHP, KIND, NR>;
  if ((rc = ensure_smem((const void*)kern, C::SMEM))) return rc;
  const int grid = p.workers / C::WARPS;
  cudaError_t e = launch_pdl(kern, dim3(grid), dim3(128), C::SMEM, st, mk, mv, a, reinterpret_cast<DevStatus*>(ws));
  if (e != cudaSuccess) return cuda_fail(e, "kv_decode_kernel");
  if ((rc = check_launch("kv_decode_kernel")) || a.whole) return rc;
  e = launch_pdl(kv_join_kernel<DHP>, dim3(p.workers), dim3(256), 0, st, a, p.workers, p.M);
  if (e != cudaSuccess) return cuda_fail(e, "kv_join_kernel");
  return check_launch("kv_join_kernel");
}

template <int DHP, int KIND>
int kv_prompt_t(const KvAttnPlan& p, uint8_t* ws, cudaStream_t st) {
  using C = KvPromptCfg<DHP>;
  auto kern = kv_prompt_kernel<DHP, KIND>;
  int rc = ensure_smem((const void*)kern, C::SMEM);
  if (rc) return rc;
  KvPromptArgs pa;
  pa.a = p.a;
  pa.tiles = p.tiles;
  pa.blocks = p.blocks;
  pa.info = reinterpret_cast<int4*>(ws + p.off_plan);
  pa.starts = pa.info + p.tiles;
  pa.cum = reinterpret_cast<int*>(pa.starts + p.blocks + 1);
  cudaError_t e = launch_pdl(kv_prompt_plan_kernel<DHP>, dim3(1), dim3(1024), 0, st, pa);
  if (e != cudaSuccess) return cuda_fail(e, "kv_prompt_plan_kernel");
  e = launch_pdl(kern, dim3(p.blocks), dim3(C::THREADS), C::SMEM, st, pa, reinterpret_cast<DevStatus*>(ws));
  if (e != cudaSuccess) return cuda_fail(e, "kv_prompt_kernel");
  if ((rc = check_launch("kv_prompt_kernel"))) return rc;
  e = launch_pdl(kv_prompt_join_kernel<DHP>, dim3(p.blocks, C::MQ / 8), dim3(256), 0, st, pa);
  if (e != cudaSuccess) return cuda_fail(e, "kv_prompt_join_kernel");
  return check_launch("kv_prompt_join_kernel");
}

int kv_attention_run(const b200l_kv_cache* cache, const b200l_kv_attn_desc* d, void* ws, size_t ws_bytes, cudaStream_t st) {
  KvAttnPlan p;
  int rc = kv_attn_plan(cache, d, &p);
  if (rc) return rc;
  if (d->tokens == 0) return B200L_OK;
  if (!d->q || !d->out || !d->block_table || !d->seq_lens || !d->cu_new || !d->cu_pages)
    return fail(B200L_ERR_NULL_POINTER, "kv_attention: NULL pointer");
  if (misaligned(d->q, 2) || misaligned(d->out, 4)) return fail(B200L_ERR_ALIGNMENT, "kv_attention: q or out is misaligned");
  if (misaligned(ws, 1024)) return fail(B200L_ERR_ALIGNMENT, "workspace must be 1024-byte aligned");
  if (!ws || ws_bytes < p.total)
    return fail(B200L_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", ws ? ws_bytes : 0, p.total);
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.a.part_o = reinterpret_cast<float*>(w + p.off_o);
  p.a.part_ml = p.a.part_o + (size_t)p.pieces * p.M * p.dhp;
  if (p.prompt) {
#define KV_CALL(D, K) kv_prompt_t<D, K>(p, w, st)
    KV_DISPATCH(cache->head_dim, cache->kind, KV_CALL)
#undef KV_CALL
  }
#define KV_CALL(D, K) (p.M == 8 ? kv_decode_t<D, K, 1>(p, w, st) : p.M == 16 ? kv_decode_t<D, K, 2>(p, w, st) : kv_decode_t<D, K, D == 256 ? 2 : 4>(p, w, st))
  KV_DISPATCH(cache->head_dim, cache->kind, KV_CALL)
#undef KV_CALL
}

// No exception crosses the C boundary.
template <typename F>
int kv_guard(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    return B200L_ERR_LAUNCH;
  }
}

}  // namespace

extern "C" {

int b200l_kv_plan(const b200l_kv_plan_desc* desc, void* stream) {
  return kv_guard([&] { return kv_plan_run(desc, static_cast<cudaStream_t>(stream)); });
}

int b200l_kv_append(const b200l_kv_cache* cache, const b200l_kv_rows* rows, const int64_t* slots, int64_t tokens,
                    void* stream) {
  return kv_guard([&] { return kv_append_run(cache, rows, slots, tokens, static_cast<cudaStream_t>(stream)); });
}

int b200l_kv_read(const b200l_kv_cache* cache, const int64_t* slots, int64_t n, void* k_out, void* v_out, int32_t dtype,
                  void* stream) {
  return kv_guard([&] { return kv_read_run(cache, slots, n, k_out, v_out, dtype, static_cast<cudaStream_t>(stream)); });
}

size_t b200l_kv_attention_workspace_bytes(const b200l_kv_cache* cache, const b200l_kv_attn_desc* desc) {
  size_t total = 0;
  kv_guard([&] {
    KvAttnPlan p;
    const int rc = kv_attn_plan(cache, desc, &p);
    if (!rc) total = p.total;
    return rc;
  });
  return total;
}

int b200l_kv_attention(const b200l_kv_cache* cache, const b200l_kv_attn_desc* desc, void* workspace, size_t ws_bytes,
                       void* stream) {
  return kv_guard([&] { return kv_attention_run(cache, desc, workspace, ws_bytes, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
