// kv_decode.cuh -- attention of few rows per request over a paged 8-bit cache.
//
// A row is one query head of one new token; the rows of a request that share a
// key/value head (new tokens x query heads per key head) are one tile of M = 16
// or 32 rows, so the cache is read once for all of them. With codes c, scales
// s_k, s_v per page and head, and key j visible to the row:
//   t_j = log2(e) scale s_k(j) <q, c_k(j)>         u_j = t_j + log2 s_v(j)
//   o   = sum_j 2^(u_j - M) c_v(j) / sum_j 2^(u_j - M) / s_v(j),   M = max u
// so the products run on the codes themselves (exact in fp16), a key's scale
// meets its score in fp32, and a value's scale joins the exponent: the weights
// that multiply codes are at most 2^8 and go into fp16 relative to the largest
// contribution, and no accumulator is rescaled per page. Sums and maxima are
// fp32; fp16 rounds q (scaled by a power of two to [1, 2) at the row's largest
// if it comes as bf16: exact but for what is 2^-14 of it) and the weights.
//
// Bound: HBM, 2 dhp bytes per cached token and head. Work is split evenly over
// warps, not requests: the pages of all (request, head) pairs in a row are cut
// into one stretch per warp, so 2 requests of 100000 tokens and 256 of a
// thousand fill the GPU alike, and warps never wait for one another. A warp
// streams its stretch through two slots of its own shared memory (TMA, one box
// per page, swizzled so that the fragment reads below have no bank conflicts;
// 12 warps x 8-16 KB in flight cover HBM's latency several times over). A pair
// that lies inside one stretch is finished there; of one that is cut, each
// piece leaves (max, sum, accumulator) in the workspace and kv_join_kernel adds
// them in order.
//
// Products are mma.sync m16n8k16: one tile of M rows has too little work for
// tcgen05 (2 FLOP per byte read and row; HBM bounds it below M ~ 250). Which
// dims or keys a fragment's place stands for is free as long as both operands
// agree, so fragments are read straight from the page's rows: as B of Q K^T a
// lane takes 16 consecutive code bytes of its key; as B of P V the same bytes of
// four keys, transposed by byte permutes on the way to fp16.
#pragma once

#include "kv_common.cuh"

namespace b200l {

struct KvAttnArgs {
  KvCache c;
  const void* q;
  void* out;
  long long q_st, q_sh;          // element strides of q per token and head (dims contiguous)
  const int* table;
  long long table_stride;
  const int* lens;
  const int* cu_new;
  const int* cu_pages;
  float* part_o;                 // [2 * workers][M][dhp]
  float* part_ml;                // [2 * workers][M][2]
  int requests, width, tokens, hq, group, dh, type, causal, row_tiles, min_pages, q_vec, q_vec8, o_vec8;
  float scale_log2;              // softmax scale * log2(e)
};

template <int DHP, int MT>
struct KvDecCfg {
  static constexpr int TK = DHP == 256 ? 16 : DHP == 128 ? 32 : 64;   // keys of a tile
  static constexpr int ROWB = DHP < 128 ? DHP : 128;                  // bytes of a swizzled row
  static constexpr int NH = DHP / ROWB;                               // boxes side by side
  static constexpr int CODE = TK * DHP;                               // bytes of K (and of V) in a slot
  static constexpr int SLOTS = 2;
  static constexpr int WARPS = 4;
  static constexpr bool QSM = DHP * MT > 128;                         // Q fragments in shared memory
  static constexpr int QB = QSM ? MT * 16 * DHP * 2 : 0;
  static constexpr int SMEM = WARPS * (SLOTS * 2 * CODE + QB) + WARPS * SLOTS * 8 + WARPS * SLOTS * 4 * 8 + 64 + 1024;
  static constexpr int CTAS = DHP == 256 || MT == 2 ? 2 : 3;            // resident per SM (registers)
  static constexpr int M = 16 * MT;
};

// A warp's stretch of the pages of all (request, head, row tile) triples.
struct KvSpan {
  long long u, u1;
  int r, h, np, len, p0, p1;     // pages [p0, p1) of np; h counts (head, row tile)
  bool done;

  __device__ __forceinline__ void cut(const KvAttnArgs& a, int heads) {
    const long long left = u1 - u;
    p1 = (long long)(np - p0) < left ? np : p0 + (int)left;
    len = min(max(a.lens[r], 0), min(np, a.width) << a.c.log2_page);
  }
  __device__ __forceinline__ void begin(const KvAttnArgs& a, int heads, long long from, long long to, int lane) {
    u = from;
    u1 = to;
    done = u >= u1;
    if (done) return;
    r = warp_find_owner(a.cu_pages, a.requests, u / heads, lane);
    const long long base = (long long)a.cu_pages[r];
    np = (int)(a.cu_pages[r + 1] - base);
    if (np <= 0) {                                // (cu_pages is no prefix sum)
      done = true;
      return;
    }
    const long long off = u - base * heads;
    h = (int)(off / np);
    p0 = (int)(off - (long long)h * np);
    cut(a, heads);
  }
  __device__ __forceinline__ void next(const KvAttnArgs& a, int heads, int lane) {
    u += p1 - p0;
    if (u >= u1) {
      done = true;
      return;
    }
    p0 = 0;
    if (++h == heads) {
      h = 0;
      const int base = a.cu_pages[r + 1];
      np = ++r + 1 <= a.requests ? a.cu_pages[r + 1] - base : 0;
      if (np <= 0) {
        r = warp_find_owner(a.cu_pages, a.requests, base, lane);
        np = a.cu_pages[r + 1] - a.cu_pages[r];
        if (np <= 0) {
          done = true;
          return;
        }
      }
    }
    cut(a, heads);
  }
};

// How the pages are cut: the stretch of worker w of `workers`.
__device__ __forceinline__ long long kv_chunk(const KvAttnArgs& a, int heads, int workers) {
  const long long units = (long long)heads * a.cu_pages[a.requests];
  const long long c = (units + workers - 1) / workers;
  return c < a.min_pages ? a.min_pages : c;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

__device__ __forceinline__ void store_out(const KvAttnArgs& a, long long at, int d, float x, float y) {
  // dims d, d + 1 of a row that begins at element `at`; d is even
  if (d + 1 < a.dh && (a.dh & 1) == 0) {
    *reinterpret_cast<uint32_t*>(static_cast<__half*>(a.out) + at + d) = pack_elem2(x, y, a.type);
    return;
  }
  const uint32_t w = pack_elem2(x, y, a.type);
  unsigned short* o = static_cast<unsigned short*>(a.out) + at;
  if (d < a.dh) o[d] = (unsigned short)(w & 0xffffu);
  if (d + 1 < a.dh) o[d + 1] = (unsigned short)(w >> 16);
}

template <int DHP, int KIND, int MT>
__global__ void __launch_bounds__(128, KvDecCfg<DHP, MT>::CTAS)
    kv_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, KvAttnArgs a,
                     DevStatus* status) {
  using C = KvDecCfg<DHP, MT>;
  constexpr int TK = C::TK, NT = TK / 8, KS = DHP / 16, M = C::M;
  constexpr int KB = DHP >= 64 ? 16 : 8;          // code bytes of a lane's key at a time
  constexpr int KC = DHP / (4 * KB);              // ... and how many times
  constexpr int VB = DHP / 8 < 16 ? DHP / 8 : 16; // the same for values
  constexpr int ND = DHP / 8;                     // 8-dim tiles of the output
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (C::SLOTS * 2 * C::CODE);
  uint8_t* qsm = smem + C::WARPS * (C::SLOTS * 2 * C::CODE) + warp * C::QB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::WARPS * (C::SLOTS * 2 * C::CODE + C::QB)) + warp * C::SLOTS;
  float2* scl = reinterpret_cast<float2*>(smem + C::WARPS * (C::SLOTS * 2 * C::CODE + C::QB) + C::WARPS * C::SLOTS * 8) +
                warp * C::SLOTS * 4;
  WaitCtl* wc = reinterpret_cast<WaitCtl*>(smem + C::SMEM - 1024 - 64);
  pdl_wait_then_release();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::WARPS * C::SLOTS; ++i)
      mbar_init(reinterpret_cast<uint64_t*>(smem + C::WARPS * (C::SLOTS * 2 * C::CODE + C::QB)) + i, 1);
    waitctl_init(wc, status);
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();

  const int P = a.c.page, lp = a.c.log2_page, PB = P < TK ? P : TK;   // keys of a box
  const int heads = a.c.heads * a.row_tiles;
  const int workers = gridDim.x * C::WARPS, w = blockIdx.x * C::WARPS + warp;
  const long long units = (long long)heads * a.cu_pages[a.requests];
  const long long chunk = kv_chunk(a, heads, workers);
  const long long u0 = w * chunk, u1 = units < u0 + chunk ? units : u0 + chunk;

  // ---- the loads, two tiles ahead
  KvSpan ld;
  ld.begin(a, heads, u0, u1, lane);
  int lkey = 0, lend = 0, entry = -1;
  auto fetch_entry = [&]() {                      // page of this lane's box in the tile at lkey
    const int k = lkey + lane * PB;
    entry = (lane * PB < TK && k < lend && (k >> lp) < a.width) ? a.table[ld.r * a.table_stride + (k >> lp)] : -1;
  };
  auto open_span = [&]() {                        // on to the next stretch that has keys
    while (!ld.done) {
      lkey = ld.p0 << lp;
      lend = min(ld.p1 << lp, ld.len);
      if (lkey < lend) break;
      ld.next(a, heads, lane);
    }
    if (!ld.done) fetch_entry();
  };
  open_span();
  int issued = 0;
  auto issue = [&]() {
    if (!ld.done) {
      const int s = issued & 1;
      const bool ok = entry >= 0 && entry < a.c.num_pages;
      const int head = ld.h / a.row_tiles;
      const unsigned boxes = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) mbar_arrive_expect_tx(&bars[s], (uint32_t)__popc(boxes) * 2u * (uint32_t)(PB * DHP));
      __syncwarp();
      if (lane * PB < TK) {
        if (ok) {
          const long long ph = (long long)entry * a.c.heads + head;
          const int row = (int)((ph << lp) + ((lkey + lane * PB) & (P - 1)));
          uint8_t* kd = ring + s * 2 * C::CODE + lane * PB * C::ROWB;
#pragma unroll
          for (int b = 0; b < C::NH; ++b) {
            tma_load_2d(kd + b * TK * C::ROWB, &map_k, &bars[s], b * 128, row);
            tma_load_2d(kd + C::CODE + b * TK * C::ROWB, &map_v, &bars[s], b * 128, row);
          }
          const uint32_t dst = smem_u32(&scl[s * 4 + lane]);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(a.c.k_scale + ph) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4), "l"(a.c.v_scale + ph) : "memory");
        } else {
          scl[s * 4 + lane] = make_float2(0.f, -1.f);           // no such page: its keys are not there
        }
      }
      ++issued;
      lkey += TK;
      if (lkey >= lend) {
        ld.next(a, heads, lane);
        open_span();
      } else {
        fetch_entry();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  issue();
  issue();

  int used = 0;
  bool ok = true;
  KvSpan sp;
  for (sp.begin(a, heads, u0, u1, lane); !sp.done && ok; sp.next(a, heads, lane)) {
    const int head = sp.h / a.row_tiles, rt = sp.h - head * a.row_tiles;
    const int tok0 = a.cu_new[sp.r], n = a.cu_new[sp.r + 1] - tok0, rows = n * a.group;
    const int row0 = rt * M;
    const bool live = row0 < rows;                // (else: no such row tile for this request)
    const int kend = min(sp.p1 << lp, sp.len);
    // ---- Q fragments, and how far each row sees
    uint32_t qf[C::QSM ? 1 : MT][C::QSM ? 1 : KS][4];
    int lim[MT][2], lim_min = kend;
    float qs[MT][2];
    long long oat[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + m * 16 + g + 8 * e;
        const int i = row / a.group, hq = head * a.group + row - i * a.group;
        const bool in = row < rows && tok0 + i < a.tokens;
        oat[m][e] = in ? ((long long)(tok0 + i) * a.hq + hq) * a.dh : -1;
        lim[m][e] = in ? min(kend, a.causal ? sp.len - n + i + 1 : kend) : 0;
        if (in) lim_min = min(lim_min, lim[m][e]);
        const void* q = a.q;
        const long long at = (long long)(tok0 + i) * a.q_st + (long long)hq * a.q_sh;
        float v[KS][4], big = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          // dims of k-step s: chunk s / (KB/4), then 4 of the lane's KB
          constexpr int PER = KB / 4;
          const int c = s / PER, d = (DHP == 32 ? KB * t : DHP == 64 ? KB * t : 128 * (c / 2) + 32 * t + 16 * (c & 1)) + 4 * (s % PER);
          if (in && a.q_vec && d + 4 <= a.dh) {
            const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(q) + at + d);
            if (a.type == kElemF16) {
              const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
              v[s][0] = x.x; v[s][1] = x.y; v[s][2] = y.x; v[s][3] = y.y;
            } else {
              const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
              v[s][0] = x.x; v[s][1] = x.y; v[s][2] = y.x; v[s][3] = y.y;
            }
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[s][k] = in && d + k < a.dh ? load_elem(q, at + d + k, a.type) : 0.f;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) big = fmaxf(big, fabsf(v[s][k]));
        }
        float mul = 1.f;
        qs[m][e] = a.scale_log2;
        big = quad_max(big);
        if (a.type == kElemBF16 && big > 0.f && big < INFINITY) {
          const int ex = min(max(((__float_as_int(big) >> 23) & 255) - 127, -120), 120);
          mul = __int_as_float((127 - ex) << 23);
          qs[m][e] *= __int_as_float((127 + ex) << 23);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint32_t x = pack_half2(v[s][0] * mul, v[s][1] * mul), y = pack_half2(v[s][2] * mul, v[s][3] * mul);
          if constexpr (C::QSM) {
            uint32_t* f = reinterpret_cast<uint32_t*>(qsm) + ((m * KS + s) * 32 + lane) * 4;
            f[e] = x;
            f[2 + e] = y;
          } else {
            qf[m][s][e] = x;
            qf[m][s][2 + e] = y;
          }
        }
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);

    float o[MT][ND][4], mx[MT][2], l[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      mx[m][0] = mx[m][1] = -INFINITY;
      l[m][0] = l[m][1] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[m][d][0] = o[m][d][1] = o[m][d][2] = o[m][d][3] = 0.f;
    }

    for (int key = sp.p0 << lp; key < kend; key += TK) {
      const int s = used & 1;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (!mbar_wait_warp(&bars[s], (used >> 1) & 1, wc)) {
        ok = false;
        break;
      }
      __syncwarp();
      const uint8_t* ks = ring + s * 2 * C::CODE;
      const uint8_t* vs = ks + C::CODE;
      // ---- scores of 8 keys a tile
      float acc[MT][NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
        const int row = 8 * j + g;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          uint32_t wd[KB / 4];
          if constexpr (DHP == 32) {
            // 32-byte rows, 32B swizzle: 16-byte chunk ^= address bit 7
            const uint2 u = *reinterpret_cast<const uint2*>(ks + row * 32 + ((((t >> 1) ^ (row >> 2)) & 1) << 4) + ((t & 1) << 3));
            wd[0] = u.x;
            wd[1] = u.y;
          } else {
            const uint8_t* p;
            if constexpr (DHP == 64) p = ks + swz_offset(row, t, 64);
            else p = ks + (c / 2) * TK * 128 + swz_offset(row, 2 * t + (c & 1), 128);
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            wd[0] = u.x;
            wd[1] = u.y;
            wd[2] = u.z;
            wd[3] = u.w;
          }
#pragma unroll
          for (int i = 0; i < KB / 4; ++i) {
            uint32_t b0, b1;
            codes4_to_half<KIND>(wd[i], b0, b1);
            const int st = c * (KB / 4) + i;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              if constexpr (C::QSM) {
                const uint4 u = *reinterpret_cast<const uint4*>(qsm + ((m * KS + st) * 32 + lane) * 16);
                const uint32_t f[4] = {u.x, u.y, u.z, u.w};
                mma_f16(acc[m][j], f, b0, b1);
              } else {
                mma_f16(acc[m][j], qf[m][st], b0, b1);
              }
            }
          }
        }
      }
      // ---- u = t + log2 s_v, row maxima
      const int nbox = (min(kend - key, TK) + PB - 1) / PB;
      bool hole = key + TK > lim_min;
      float inv[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int box = min(8 * j / PB, nbox - 1);
        const float2 sc = scl[s * 4 + box];
        // A scale of 0 (a page of zeros) has no logarithm: 2^-100 stands for it.
        const float sv = fmaxf(sc.y, 7.8886090522101181e-31f);
        const float lv = sc.y == sc.y ? __log2f(sv) : sc.y;
        inv[j] = sv < INFINITY ? __fdividef(1.0f, sv) : 0.f;
        const bool none = sc.y < 0.f;
        hole |= none;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float c0 = qs[m][0] * sc.x, c1 = qs[m][1] * sc.x;
          acc[m][j][0] = fmaf(acc[m][j][0], c0, lv);
          acc[m][j][1] = fmaf(acc[m][j][1], c0, lv);
          acc[m][j][2] = fmaf(acc[m][j][2], c1, lv);
          acc[m][j][3] = fmaf(acc[m][j][3], c1, lv);
        }
      }
      if (hole) {                                 // (warp-uniform)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bool none = scl[s * 4 + min(8 * j / PB, nbox - 1)].y < 0.f;
          const int k = key + 8 * j + 2 * t;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (none || k >= lim[m][0]) acc[m][j][0] = -INFINITY;
            if (none || k + 1 >= lim[m][0]) acc[m][j][1] = -INFINITY;
            if (none || k >= lim[m][1]) acc[m][j][2] = -INFINITY;
            if (none || k + 1 >= lim[m][1]) acc[m][j][3] = -INFINITY;
          }
        }
      }
      // ---- weights; the accumulators move to a new maximum when it is 2^8 over the old
      uint32_t p[MT][NT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          top0 = fmax3f(top0, acc[m][j][0], acc[m][j][1]);
          top1 = fmax3f(top1, acc[m][j][2], acc[m][j][3]);
        }
        top0 = quad_max(top0);
        top1 = quad_max(top1);
        const bool up0 = top0 > mx[m][0] + 8.f, up1 = top1 > mx[m][1] + 8.f;
        if (__any_sync(0xffffffffu, up0 || up1)) {
          const float a0 = up0 ? ex2_approx(mx[m][0] - top0) : 1.f, a1 = up1 ? ex2_approx(mx[m][1] - top1) : 1.f;
          if (up0) mx[m][0] = top0;
          if (up1) mx[m][1] = top1;
          l[m][0] *= a0;
          l[m][1] *= a1;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            o[m][d][0] *= a0;
            o[m][d][1] *= a0;
            o[m][d][2] *= a1;
            o[m][d][3] *= a1;
          }
        }
        const float m0 = mx[m][0] == -INFINITY ? 0.f : mx[m][0], m1 = mx[m][1] == -INFINITY ? 0.f : mx[m][1];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float x0 = ex2_approx(acc[m][j][0] - m0), x1 = ex2_approx(acc[m][j][1] - m0);
          const float x2 = ex2_approx(acc[m][j][2] - m1), x3 = ex2_approx(acc[m][j][3] - m1);
          l[m][0] = fmaf(x0 + x1, inv[j], l[m][0]);
          l[m][1] = fmaf(x2 + x3, inv[j], l[m][1]);
          p[m][j][0] = pack_half2(x0, x1);
          p[m][j][1] = pack_half2(x2, x3);
        }
      }
      // ---- O += P V, 16 keys a step
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) {
#pragma unroll
        for (int hb = 0; hb < C::NH; ++hb) {
          uint32_t kw[4][VB / 4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 16 * i + 2 * t + (k & 1) + 8 * (k >> 1);
            if constexpr (DHP == 32) {
              kw[k][0] = *reinterpret_cast<const uint32_t*>(vs + row * 32 + ((((g >> 2) ^ (row >> 2)) & 1) << 4) + ((g & 3) << 2));
            } else if constexpr (DHP == 64) {
              const uint2 u = *reinterpret_cast<const uint2*>(vs + swz_offset(row, g >> 1, 64) + ((g & 1) << 3));
              kw[k][0] = u.x;
              kw[k][1] = u.y;
            } else {
              const uint4 u = *reinterpret_cast<const uint4*>(vs + hb * TK * 128 + swz_offset(row, g, 128));
              kw[k][0] = u.x;
              kw[k][1] = u.y;
              kw[k][2] = u.z;
              kw[k][3] = u.w;
            }
            if (hole) {                           // what lies past the keys is not read as a number
              const bool none = row + key >= kend || scl[s * 4 + min(row / PB, nbox - 1)].y < 0.f;
#pragma unroll
              for (int b = 0; b < VB / 4; ++b) kw[k][b] = none ? 0u : kw[k][b];
            }
          }
#pragma unroll
          for (int b = 0; b < VB / 4; ++b) {
            // bytes of four keys for four dims -> per dim the pairs (keys 0, 1) and (2, 3)
            const uint32_t x01 = __byte_perm(kw[0][b], kw[1][b], 0x5140), y01 = __byte_perm(kw[0][b], kw[1][b], 0x7362);
            const uint32_t x23 = __byte_perm(kw[2][b], kw[3][b], 0x5140), y23 = __byte_perm(kw[2][b], kw[3][b], 0x7362);
            uint32_t f01[4], f23[4];
            codes4_to_half<KIND>(x01, f01[0], f01[1]);
            codes4_to_half<KIND>(y01, f01[2], f01[3]);
            codes4_to_half<KIND>(x23, f23[0], f23[1]);
            codes4_to_half<KIND>(y23, f23[2], f23[3]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint32_t pa[4] = {p[m][2 * i][0], p[m][2 * i][1], p[m][2 * i + 1][0], p[m][2 * i + 1][1]};
#pragma unroll
              for (int d = 0; d < 4; ++d) mma_f16(o[m][hb * 16 + 4 * b + d], pa, f01[d], f23[d]);
            }
          }
        }
      }
      __syncwarp();
      ++used;
      issue();
    }
    if (!ok) break;

    // ---- the pair's result, or this piece of it
    const bool whole = sp.p0 == 0 && sp.p1 == sp.np;
    // Pieces: slot 2w holds the one that the stretch begins with, 2w + 1 the one that it ends with.
    const long long slot = 2ll * w + (sp.u == u0 ? 0 : 1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float lt = quad_sum(l[m][e]);
        if (!live || oat[m][e] < 0) continue;
        const int row = m * 16 + g + 8 * e;
        if (whole) {
          const float r = lt == 0.f ? 0.f : 1.0f / lt;
#pragma unroll
          for (int hb = 0; hb < C::NH; ++hb)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int d = 0; d < VB; d += 2)
                store_out(a, oat[m][e], hb * 128 + VB * (2 * t + c) + d, o[m][hb * 16 + d][2 * e + c] * r,
                          o[m][hb * 16 + d + 1][2 * e + c] * r);
        } else {
          float* po = a.part_o + (slot * M + row) * DHP;
          if (t == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * M + row) * 2) = make_float2(mx[m][e], lt);
#pragma unroll
          for (int hb = 0; hb < C::NH; ++hb)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int d = 0; d < VB; d += 4)
                *reinterpret_cast<float4*>(po + hb * 128 + VB * (2 * t + c) + d) =
                    make_float4(o[m][hb * 16 + d][2 * e + c], o[m][hb * 16 + d + 1][2 * e + c],
                                o[m][hb * 16 + d + 2][2 * e + c], o[m][hb * 16 + d + 3][2 * e + c]);
        }
      }
    }
  }
  if (!ok) {                                      // copies in flight land before the block goes
    for (int i = used; i < issued; ++i) mbar_drain(&bars[i & 1], (i >> 1) & 1);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && waitctl_aborted(wc)) record_error(status, -7, kKernelKvDecode, 1);
}

// Joins the pieces of every pair that was cut, in order: with M = max m_i,
// o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i. A block per worker looks
// whether a pair begins in that worker's stretch and goes on past it; warps
// take its rows. Also zeroes the rows that attend to nothing: those of requests
// without keys, and those past the plan's tokens.
template <int DHP>
__global__ void __launch_bounds__(128) kv_join_kernel(KvAttnArgs a, int workers, int M) {
  pdl_wait_then_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gw = blockIdx.x * 4 + warp, nw = gridDim.x * 4;
  auto zero_rows = [&](int t0, int t1) {
    const long long e1 = (long long)min(t1, a.tokens) * a.hq * a.dh;
    for (long long i = (long long)t0 * a.hq * a.dh + lane; i < e1; i += 32) static_cast<unsigned short*>(a.out)[i] = 0;
  };
  for (int r = gw; r < a.requests; r += nw)
    if (a.cu_pages[r + 1] == a.cu_pages[r] && a.cu_new[r + 1] > a.cu_new[r]) zero_rows(a.cu_new[r], a.cu_new[r + 1]);
  for (int i = a.cu_new[a.requests] + gw; i < a.tokens; i += nw) zero_rows(i, i + 1);

  const int heads = a.c.heads * a.row_tiles;
  const long long units = (long long)heads * a.cu_pages[a.requests];
  const long long chunk = kv_chunk(a, heads, workers);
  const int w = blockIdx.x;
  const long long u0 = w * chunk, u1 = u0 + chunk;
  if (u1 >= units) return;                        // nothing lies past this stretch
  // The pair that holds the stretch's last page.
  const int r = warp_find_owner(a.cu_pages, a.requests, (u1 - 1) / heads, lane);
  const long long base = (long long)heads * a.cu_pages[r];
  const int np = a.cu_pages[r + 1] - a.cu_pages[r];
  if (np <= 0) return;
  const int h = (int)((u1 - 1 - base) / np);
  const long long b = base + (long long)h * np, e = b + np;
  if (b < u0 || e <= u1) return;                  // begins earlier, or ends here
  const int pieces = (int)((e - 1) / chunk) - w + 1;
  const int head = h / a.row_tiles, rt = h - head * a.row_tiles;
  const int tok0 = a.cu_new[r], rows = (a.cu_new[r + 1] - tok0) * a.group;
  auto slot = [&](int i) { return i == 0 && b != u0 ? 2ll * w + 1 : 2ll * (w + i); };
  for (int row = warp; row < M; row += 4) {
    const int gr = rt * M + row, i = gr / a.group;
    if (gr >= rows || tok0 + i >= a.tokens) break;
    float top = -INFINITY;
    for (int k = lane; k < pieces; k += 32) top = fmaxf(top, a.part_ml[(slot(k) * M + row) * 2]);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (top == -INFINITY) top = 0.f;
    constexpr int PER = DHP / 32;
    float acc[PER], l = 0.f;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll 4
    for (int k = 0; k < pieces; ++k) {
      const long long at = slot(k) * M + row;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
      const float f = ex2_approx(ml.x - top);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[d] = fmaf(a.part_o[at * DHP + d * 32 + lane], f, acc[d]);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const long long at = ((long long)(tok0 + i) * a.hq + head * a.group + gr - i * a.group) * a.dh;
#pragma unroll
    for (int d = 0; d < PER; ++d) {
      const int dim = d * 32 + lane;
      if (dim < a.dh) {
        if (a.type == kElemF16) static_cast<__half*>(a.out)[at + dim] = __float2half_rn(acc[d] * inv);
        else static_cast<__nv_bfloat16*>(a.out)[at + dim] = __float2bfloat16_rn(acc[d] * inv);
      }
    }
  }
}

}  // namespace b200l
