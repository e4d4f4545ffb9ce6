// kv_decode.cuh -- attention of few rows per request over a paged 8-bit cache.
//
// A row is one query head of one new token; the rows of a request that share a
// key/value head (new tokens x query heads per key head) are one tile of M = 8,
// 16 or 32 rows, so the cache is read once for all of them. With codes c, scales
// s_k, s_v per page and head, and key j visible to the row:
//   t_j = log2(e) scale s_k(j) <q, c_k(j)>         u_j = t_j + log2 s_v(j)
//   o   = sum_j 2^(u_j - M) c_v(j) / sum_j 2^(u_j - M) / s_v(j),   M = max u
// so the products run on the codes themselves (exact in fp16), a key's scale
// meets its score in fp32, and a value's scale joins the exponent: the weights
// that multiply codes are at most 2^8 and go into fp16 relative to the largest
// contribution, and no accumulator is rescaled per page. Sums and maxima are
// fp32; fp16 rounds q (scaled by a power of two to [1, 2) at the row's largest
// if it comes as bf16: exact but for what is 2^-14 of it) and the weights of the
// numerator: to 2^-11 of themselves, below 2^-14 to 2^-25 of the largest
// contribution. The denominator must not lose those, for there a key counts with
// 2^t whatever its values' size: it sums the weights in fp32.
//
// Bound: HBM, 2 dhp bytes per cached token and head. Work is split evenly over
// warps, not requests: the keys of all (request, head) pairs in a row are cut
// into one stretch per warp, so 2 requests of 100000 tokens and 256 of a
// thousand fill the GPU alike, and warps never wait for one another. A warp
// streams its stretch through two slots of its own shared memory (TMA, one box
// per page, swizzled so that the fragment reads below have no bank conflicts;
// 12 warps x 8-16 KB in flight cover HBM's latency several times over). A pair
// that lies inside one stretch is finished there; of one that is cut, each
// piece leaves (max, sum, accumulator) in the workspace and kv_join_kernel adds
// them in order (64 requests, 32 / 8 heads of 128: 5 us more; the last warp to
// leave a piece adding them itself, 8 us). Where tables are too narrow for it to
// be worth it, stretches are whole pairs and there is nothing to join.
//
// Measured: 256 requests of about 7000 tokens, 32 / 8 heads of 128, int8 594-666 us
// (3.7 GB, 86-97 % of HBM's rate); 2 requests of 100000, 16 heads of 64, e4m3 82-83 us
// (77 %); 64 ragged requests, 32 / 8 heads of 128 104-108 us (75-77 %): the rest is the
// first loads' latency, the join, and warps that end apart.
//
// Products are mma.sync m16n8k16: one tile of M rows has too little work for
// tcgen05 (2 FLOP per byte read and row; HBM bounds it below M ~ 130). The
// transposed products are taken, S^T = K Q^T and O^T = V^T P^T, so that the 16
// of the shape are keys or dims, always full, and the 8 are rows: a token's few
// query heads pad to 8, and accumulators, Q and exponentials are half of what
// 16-row tiles of Q K^T hold. Which dims or keys a fragment's place stands for is
// free as long as both operands agree, so fragments are read straight from the
// page's rows: as A of K Q^T a lane takes 16 consecutive code bytes of a key; as A
// of V^T P^T the same bytes of four keys, transposed by byte permutes on the way
// to fp16. P^T goes from accumulator to operand by movmatrix. The row sums take
// the weights rounded to fp16's 11 bits, so that what rounds a weight rounds it
// above and below alike, but with fp32's exponent; a lane sums its own keys, and
// lanes are added once a pair.
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
  int requests, width, tokens, hq, group, dh, type, causal, row_tiles, min_units, whole, log2_unit, q_vec, q_vec8, o_vec8;
  float scale_log2;              // softmax scale * log2(e)
};

template <int DHP, int NR>       // rows of a tile: 8 NR
struct KvDecCfg {
  static constexpr int TK = DHP == 256 ? 16 : DHP == 128 ? 32 : 64;   // keys of a tile
  static constexpr int ROWB = DHP < 128 ? DHP : 128;                  // bytes of a swizzled row
  static constexpr int NH = DHP / ROWB;                               // boxes side by side
  static constexpr int CODE = TK * DHP;                               // bytes of K (and of V) in a slot
  static constexpr int SLOTS = 2;
  static constexpr int WARPS = 4;
  static constexpr bool QSM = DHP * NR >= 512;                        // Q fragments in shared memory
  static constexpr int M = 8 * NR;
  static constexpr int QB = QSM ? M * DHP * 2 : 0;
  static constexpr int SMEM = WARPS * (SLOTS * 2 * CODE + QB) + WARPS * SLOTS * 8 + WARPS * SLOTS * 4 * 8 + 64 + 1024;
  // Blocks of an SM: three of 168 registers, two of 255 where accumulators and Q need
  // them. At DHP NR = 256 three spill 360 bytes (head_dim 256, 8 rows) or 600 (128, 16
  // rows); there two, which do not spill, measured less: 32 requests of 2000 tokens, 8
  // heads, int8, 63 against 77 us and 48 against 66; guesses of 1-5 tokens, 4 heads of
  // 256, 46 against 60. Up to DHP NR = 128 the spills are 0 to 48 bytes; 32 rows spill
  // up to 460 with 255.
  static constexpr int CTAS = DHP * NR >= 512 || NR == 4 ? 2 : 3;
};

// A warp's stretch of the keys of all (request, head, row tile) triples, in
// units of 2^log2_unit keys: a page, or a key tile of one where that is less.
struct KvSpan {
  long long u, u1, stretch;      // units of a stretch, but for the last
  int r, head, rt, nu, len, p0, p1;   // units [p0, p1) of nu, of request r's key head and row tile
  int tok0, n;                   // the request's new tokens
  int base;                      // cu_pages[r]
  bool done;

  __device__ __forceinline__ void cut(const KvAttnArgs& a) {
    const long long left = u1 - u;
    p1 = (long long)(nu - p0) < left || a.whole ? nu : p0 + (int)left;
  }
  __device__ __forceinline__ void set(const KvAttnArgs& a, int c0, int c1, int t0, int t1, int l) {
    const int np = c1 - c0;
    base = c0;
    nu = np << (a.c.log2_page - a.log2_unit);
    tok0 = t0;
    n = t1 - t0;
    len = min(max(l, 0), min(np, a.width) << a.c.log2_page);
  }
  // Request r, from its five numbers at once.
  __device__ __forceinline__ void open(const KvAttnArgs& a) {
    const int c0 = a.cu_pages[r], c1 = a.cu_pages[r + 1], t0 = a.cu_new[r], t1 = a.cu_new[r + 1], l = a.lens[r];
    set(a, c0, c1, t0, t1, l);
  }
  // The stretch of worker w, at the triple that it begins in, or with `last` at
  // the one that holds the last unit of a full stretch (done if there is none).
  __device__ __forceinline__ void begin(const KvAttnArgs& a, int workers, int w, int lane, bool last = false) {
    int cp = 0, cn = 0, l = 0;
    const bool few = a.requests < 32;             // a lane holds what there is of a request: one round trip
    if (few) {
      cp = a.cu_pages[min(lane, a.requests)];
      cn = a.cu_new[min(lane, a.requests)];
      l = a.lens[min(lane, a.requests - 1)];
    }
    const int total = few ? __shfl_sync(0xffffffffu, cp, a.requests) : a.cu_pages[a.requests];
    const long long per = (long long)a.c.heads * a.row_tiles << (a.c.log2_page - a.log2_unit);   // units of a page
    const long long units = per * total;
    const long long c = (units + workers - 1) / workers;
    stretch = c < a.min_units ? a.min_units : c;
    u = w * stretch;
    u1 = units < u + stretch ? units : u + stretch;
    done = u >= u1 || (last && u + stretch >= units);
    if (done) return;
    if (last) u = u1 - 1;
    const long long x = u / per;
    if (few) {
      r = __popc(__ballot_sync(0xffffffffu, lane < a.requests && (long long)cp <= x)) - 1;
      const int c0 = __shfl_sync(0xffffffffu, cp, r), c1 = __shfl_sync(0xffffffffu, cp, r + 1);
      const int t0 = __shfl_sync(0xffffffffu, cn, r), t1 = __shfl_sync(0xffffffffu, cn, r + 1);
      set(a, c0, c1, t0, t1, __shfl_sync(0xffffffffu, l, r));
    } else {
      r = warp_find_owner(a.cu_pages, a.requests, x, lane);
      open(a);
    }
    if (nu <= 0) {                                // (cu_pages is no prefix sum)
      done = true;
      return;
    }
    const long long off = u - base * per;
    const int h = (int)(off / nu);
    p0 = (int)(off - (long long)h * nu);
    head = h / a.row_tiles;
    rt = h - head * a.row_tiles;
    if (a.whole && p0 > 0) {                      // the pair is whose stretch holds its first unit
      u += nu - p0;
      p0 = 0;
      done = u >= u1;
      if (!done) step(a, lane);
    }
    cut(a);
  }
  // On to the triple after this one.
  __device__ __forceinline__ void step(const KvAttnArgs& a, int lane) {
    if (++rt < a.row_tiles) return;
    rt = 0;
    if (++head < a.c.heads) return;
    head = 0;
    const int after = base + (nu >> (a.c.log2_page - a.log2_unit));
    ++r;
    if (r < a.requests) open(a);
    if (r >= a.requests || nu <= 0) {             // requests without new tokens
      r = warp_find_owner(a.cu_pages, a.requests, after, lane);
      open(a);
      if (nu <= 0) done = true;
    }
  }
  __device__ __forceinline__ void next(const KvAttnArgs& a, int lane) {
    u += p1 - p0;
    p0 = 0;
    done = u >= u1;
    if (done) return;
    step(a, lane);
    cut(a);
  }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A weight as fp16 has it where it is 2^-14 or more, and to as many bits where it
// is less. (A not-a-number may come out as 0: the product with V has it.)
__device__ __forceinline__ float round11(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}

// Transposes an 8 x 8 tile of 16-bit values, two of a row a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

template <int DHP, int KIND, int NR>
__global__ void __launch_bounds__(128, KvDecCfg<DHP, NR>::CTAS)
    kv_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ KvAttnArgs a,
                     DevStatus* status) {
  using C = KvDecCfg<DHP, NR>;
  constexpr int TK = C::TK, KT = TK / 16, KS = DHP / 16, M = C::M;
  constexpr int KB = DHP >= 64 ? 16 : 8;          // code bytes of a lane's key at a time
  constexpr int KC = DHP / (4 * KB);              // ... and how many times
  constexpr int VB = DHP / 8 < 16 ? DHP / 8 : 16; // the same for values
  constexpr int ND = DHP / 16;                    // 16-dim tiles of the output
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

  // Keys of a box: a page, or a tile of it (the unit of the cuts, if not a smaller page).
  const int P = a.c.page, lp = a.c.log2_page, lb = a.log2_unit, PB = 1 << lb;
  const int workers = gridDim.x * C::WARPS, w = blockIdx.x * C::WARPS + warp;
  KvSpan sp;
  sp.begin(a, workers, w, lane);
  const long long u0 = sp.u;

  // ---- the loads, two tiles ahead
  KvSpan ld = sp;
  int lkey = 0, lend = 0, entry = -1;
  auto fetch_entry = [&]() {                      // page of this lane's box in the tile at lkey
    const int k = lkey + lane * PB;
    entry = (lane * PB < TK && k < lend && (k >> lp) < a.width) ? a.table[ld.r * a.table_stride + (k >> lp)] : -1;
  };
  auto open_span = [&]() {                        // on to the next stretch that has keys
    while (!ld.done) {
      lkey = ld.p0 << lb;
      lend = min(ld.p1 << lb, ld.len);
      if (lkey < lend) break;
      ld.next(a, lane);
    }
    if (!ld.done) fetch_entry();
  };
  open_span();
  int issued = 0;
  auto issue = [&]() {
    if (!ld.done) {
      const int s = issued & 1;
      const bool ok = entry >= 0 && entry < a.c.num_pages;
      const unsigned boxes = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) mbar_arrive_expect_tx(&bars[s], (uint32_t)__popc(boxes) * 2u * (uint32_t)(PB * DHP));
      __syncwarp();
      if (lane * PB < TK) {
        if (ok) {
          const int ph = entry * a.c.heads + ld.head;     // (rows of the cache stay below 2^31)
          const int row = (ph << lp) + ((lkey + lane * PB) & (P - 1));
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
        ld.next(a, lane);
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
  for (; !sp.done && ok; sp.next(a, lane)) {
    const int head = sp.head, rt = sp.rt;
    const int tok0 = sp.tok0, n = sp.n, rows = n * a.group;
    const int row0 = rt * M;
    const bool live = row0 < rows;                // (else: no such row tile for this request)
    const int kend = min(sp.p1 << lb, sp.len);
    // ---- Q fragments (row g of 8), and of the rows 2t, 2t + 1 that this lane's
    // scores and outputs belong to: how far they see, their factor, their place.
    uint32_t qf[C::QSM ? 1 : NR][C::QSM ? 1 : KS][2];
    int lim[NR][2], lim_min = kend;
    float qs[NR][2];
    long long oat[NR][2];
#pragma unroll
    for (int m = 0; m < NR; ++m) {
      const int row = row0 + m * 8 + g, i = row / a.group, hq = head * a.group + row - i * a.group;
      const bool in = row < rows && tok0 + i < a.tokens;
      const void* q = a.q;
      const long long at = (long long)(tok0 + i) * a.q_st + (long long)hq * a.q_sh;
      uint32_t v[KS][2];
      float big = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        // dims of k-step s: piece s / (KB / 4) of the row, then 4 of the lane's KB
        constexpr int PER = KB / 4;
        const int c = s / PER, d = (DHP <= 64 ? KB * t : 128 * (c / 2) + 32 * t + 16 * (c & 1)) + 4 * (s % PER);
        if (in && a.q_vec && d + 4 <= a.dh) {
          const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(q) + at + d);
          v[s][0] = u.x;
          v[s][1] = u.y;
        } else {
          const unsigned short* p = static_cast<const unsigned short*>(q) + at;
          uint32_t e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) e[k] = in && d + k < a.dh ? p[d + k] : 0u;
          v[s][0] = e[0] | e[1] << 16;
          v[s][1] = e[2] | e[3] << 16;
        }
      }
      float f = a.scale_log2;
      if (a.type == kElemBF16) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[s][k]));
            big = fmax3f(big, fabsf(x.x), fabsf(x.y));
          }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        float mul = 1.f;
        if (big > 0.f && big < INFINITY) {
          const int ex = min(max(((__float_as_int(big) >> 23) & 255) - 127, -120), 120);
          mul = __int_as_float((127 - ex) << 23);
          f *= __int_as_float((127 + ex) << 23);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[s][k]));
            v[s][k] = pack_half2(x.x * mul, x.y * mul);
          }
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (C::QSM) {
          *reinterpret_cast<uint2*>(qsm + ((m * KS + s) * 32 + lane) * 8) = make_uint2(v[s][0], v[s][1]);
        } else {
          qf[m][s][0] = v[s][0];
          qf[m][s][1] = v[s][1];
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[m][e] = __shfl_sync(0xffffffffu, f, 8 * t + 4 * e);
        const int r2 = row0 + m * 8 + 2 * t + e, i2 = r2 / a.group;
        const bool in2 = r2 < rows && tok0 + i2 < a.tokens;
        oat[m][e] = in2 ? ((long long)(tok0 + i2) * a.hq + head * a.group + r2 - i2 * a.group) * a.dh : -1;
        lim[m][e] = in2 ? min(kend, a.causal ? sp.len - n + i2 + 1 : kend) : 0;
        if (in2) lim_min = min(lim_min, lim[m][e]);
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);

    float o[ND][NR][4], mx[NR][2], l[NR][2];
#pragma unroll
    for (int m = 0; m < NR; ++m) {
      mx[m][0] = mx[m][1] = -INFINITY;
      l[m][0] = l[m][1] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d][m][0] = o[d][m][1] = o[d][m][2] = o[d][m][3] = 0.f;
    }

    for (int key = sp.p0 << lb; key < kend; key += TK) {
      const int s = used & 1;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (!mbar_wait_warp(&bars[s], (used >> 1) & 1, wc)) {
        ok = false;
        break;
      }
      __syncwarp();
      const uint8_t* ks = ring + s * 2 * C::CODE;
      const uint8_t* vs = ks + C::CODE;
      // ---- scores, 16 keys x 8 rows a tile: keys g, g + 8, rows 2t, 2t + 1
      float acc[KT][NR][4];
#pragma unroll
      for (int j = 0; j < KT; ++j) {
#pragma unroll
        for (int m = 0; m < NR; ++m) acc[j][m][0] = acc[j][m][1] = acc[j][m][2] = acc[j][m][3] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          uint32_t wd[2][KB / 4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 16 * j + g + 8 * e;
            if constexpr (DHP == 32) {
              // 32-byte rows, 32B swizzle: 16-byte chunk ^= address bit 7
              const uint2 u = *reinterpret_cast<const uint2*>(ks + row * 32 + ((((t >> 1) ^ (row >> 2)) & 1) << 4) + ((t & 1) << 3));
              wd[e][0] = u.x;
              wd[e][1] = u.y;
            } else {
              const uint8_t* p;
              if constexpr (DHP == 64) p = ks + swz_offset(row, t, 64);
              else p = ks + (c / 2) * TK * 128 + swz_offset(row, 2 * t + (c & 1), 128);
              const uint4 u = *reinterpret_cast<const uint4*>(p);
              wd[e][0] = u.x;
              wd[e][1] = u.y;
              wd[e][2] = u.z;
              wd[e][3] = u.w;
            }
          }
#pragma unroll
          for (int i = 0; i < KB / 4; ++i) {
            uint32_t ka[4];
            codes4_to_half<KIND>(wd[0][i], ka[0], ka[2]);
            codes4_to_half<KIND>(wd[1][i], ka[1], ka[3]);
            const int st = c * (KB / 4) + i;
#pragma unroll
            for (int m = 0; m < NR; ++m) {
              if constexpr (C::QSM) {
                const uint2 u = *reinterpret_cast<const uint2*>(qsm + ((m * KS + st) * 32 + lane) * 8);
                mma_f16(acc[j][m], ka, u.x, u.y);
              } else {
                mma_f16(acc[j][m], ka, qf[m][st][0], qf[m][st][1]);
              }
            }
          }
        }
      }
      // ---- u = t + log2 s_v, row maxima
      const int nbox = (min(kend - key, TK) + PB - 1) >> lb;
      bool hole = key + TK > lim_min;
      float inv[KT];
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const float2 sc = scl[s * 4 + min((16 * j) >> lb, nbox - 1)];
        // A scale of 0 (a page of zeros) has no logarithm: 2^-100 stands for it, and
        // for any that is less.
        const float sv = fmaxf(sc.y, 7.8886090522101181e-31f);
        const float lv = sc.y == sc.y ? lg2_approx(sv) : sc.y;
        inv[j] = sv < INFINITY ? rcp_approx(sv) : 0.f;
        hole |= sc.y < 0.f;
#pragma unroll
        for (int m = 0; m < NR; ++m) {
          const float c0 = qs[m][0] * sc.x, c1 = qs[m][1] * sc.x;
          acc[j][m][0] = fmaf(acc[j][m][0], c0, lv);
          acc[j][m][1] = fmaf(acc[j][m][1], c1, lv);
          acc[j][m][2] = fmaf(acc[j][m][2], c0, lv);
          acc[j][m][3] = fmaf(acc[j][m][3], c1, lv);
        }
      }
      if (hole) {                                 // (warp-uniform)
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const bool none = scl[s * 4 + min((16 * j) >> lb, nbox - 1)].y < 0.f;
          const int k = key + 16 * j + g;
#pragma unroll
          for (int m = 0; m < NR; ++m) {
            if (none || k >= lim[m][0]) acc[j][m][0] = -INFINITY;
            if (none || k >= lim[m][1]) acc[j][m][1] = -INFINITY;
            if (none || k + 8 >= lim[m][0]) acc[j][m][2] = -INFINITY;
            if (none || k + 8 >= lim[m][1]) acc[j][m][3] = -INFINITY;
          }
        }
      }
      // ---- weights; the accumulators move to a new maximum when it is 2^8 over the old
      uint32_t p[KT][NR][2];
#pragma unroll
      for (int m = 0; m < NR; ++m) {
        float top0 = fmaxf(acc[0][m][0], acc[0][m][2]), top1 = fmaxf(acc[0][m][1], acc[0][m][3]);
#pragma unroll
        for (int j = 1; j < KT; ++j) {
          top0 = fmax3f(top0, acc[j][m][0], acc[j][m][2]);
          top1 = fmax3f(top1, acc[j][m][1], acc[j][m][3]);
        }
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        const bool up0 = top0 > mx[m][0] + 8.f, up1 = top1 > mx[m][1] + 8.f;
        if (__any_sync(0xffffffffu, up0 || up1)) {
          const float a0 = up0 ? ex2_approx(mx[m][0] - top0) : 1.f, a1 = up1 ? ex2_approx(mx[m][1] - top1) : 1.f;
          if (up0) mx[m][0] = top0;
          if (up1) mx[m][1] = top1;
          l[m][0] *= a0;
          l[m][1] *= a1;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            o[d][m][0] *= a0;
            o[d][m][1] *= a1;
            o[d][m][2] *= a0;
            o[d][m][3] *= a1;
          }
        }
        const float m0 = mx[m][0] == -INFINITY ? 0.f : mx[m][0], m1 = mx[m][1] == -INFINITY ? 0.f : mx[m][1];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const float e0 = ex2_approx(acc[j][m][0] - m0), e1 = ex2_approx(acc[j][m][1] - m1);
          const float e2 = ex2_approx(acc[j][m][2] - m0), e3 = ex2_approx(acc[j][m][3] - m1);
          p[j][m][0] = transpose8x8(pack_half2(e0, e1));
          p[j][m][1] = transpose8x8(pack_half2(e2, e3));
          l[m][0] = fmaf(round11(e0) + round11(e2), inv[j], l[m][0]);
          l[m][1] = fmaf(round11(e1) + round11(e3), inv[j], l[m][1]);
        }
      }
      // ---- O^T += V^T P^T, 16 keys a step
#pragma unroll
      for (int j = 0; j < KT; ++j) {
#pragma unroll
        for (int hb = 0; hb < C::NH; ++hb) {
          uint32_t kw[4][VB / 4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 16 * j + 2 * t + (k & 1) + 8 * (k >> 1);
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
          }
          if (hole) {                             // what lies past the keys is not read as a number
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = 16 * j + 2 * t + (k & 1) + 8 * (k >> 1);
              const bool none = row + key >= kend || scl[s * 4 + min(row >> lb, nbox - 1)].y < 0.f;
#pragma unroll
              for (int b = 0; b < VB / 4; ++b) kw[k][b] = none ? 0u : kw[k][b];
            }
          }
#pragma unroll
          for (int b = 0; b < VB / 4; ++b) {
            // bytes of four keys for four dims -> per dim the pairs (keys 0, 1) and (2, 3)
            const uint32_t x01 = __byte_perm(kw[0][b], kw[1][b], 0x5140), y01 = __byte_perm(kw[0][b], kw[1][b], 0x7362);
            const uint32_t x23 = __byte_perm(kw[2][b], kw[3][b], 0x5140), y23 = __byte_perm(kw[2][b], kw[3][b], 0x7362);
            uint32_t va[2][4];
            codes4_to_half<KIND>(x01, va[0][0], va[0][1]);
            codes4_to_half<KIND>(x23, va[0][2], va[0][3]);
            codes4_to_half<KIND>(y01, va[1][0], va[1][1]);
            codes4_to_half<KIND>(y23, va[1][2], va[1][3]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int m = 0; m < NR; ++m) mma_f16(o[hb * 8 + 2 * b + e][m], va[e], p[j][m][0], p[j][m][1]);
          }
        }
      }
      __syncwarp();
      ++used;
      issue();
    }
    if (!ok) break;
#pragma unroll
    for (int m = 0; m < NR; ++m)
#pragma unroll
      for (int x = 4; x < 32; x *= 2) {           // the sums of this lane's keys -> of all
        l[m][0] += __shfl_xor_sync(0xffffffffu, l[m][0], x);
        l[m][1] += __shfl_xor_sync(0xffffffffu, l[m][1], x);
      }

    // ---- the pair's result, or this piece of it: dims [VB g, VB g + VB) of each box
    const bool whole = sp.p0 == 0 && sp.p1 == sp.nu;
    // Pieces: slot 2w holds the one that the stretch begins with, 2w + 1 the one that it ends with.
    const long long slot = 2ll * w + (sp.u == u0 ? 0 : 1);
#pragma unroll
    for (int m = 0; m < NR; ++m) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (!live || oat[m][e] < 0) continue;
        const int row = m * 8 + 2 * t + e;
        const float lt = l[m][e], r = lt == 0.f ? 0.f : 1.0f / lt;
        if (!whole && g == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * M + row) * 2) = make_float2(mx[m][e], lt);
#pragma unroll
        for (int hb = 0; hb < C::NH; ++hb) {
          const int d0 = hb * 128 + VB * g;
          if (whole) {
#pragma unroll
            for (int d = 0; d < VB; d += 2)
              store_out(a, oat[m][e], d0 + d, o[hb * 8 + d / 2][m][e] * r, o[hb * 8 + d / 2][m][2 + e] * r);
          } else {
#pragma unroll
            for (int d = 0; d < VB; d += 4)
              *reinterpret_cast<float4*>(a.part_o + (slot * M + row) * DHP + d0 + d) =
                  make_float4(o[hb * 8 + d / 2][m][e], o[hb * 8 + d / 2][m][2 + e], o[hb * 8 + d / 2 + 1][m][e],
                              o[hb * 8 + d / 2 + 1][m][2 + e]);
          }
        }
      }
    }
  }
  // Rows that attend to nothing: of requests without keys, and past the plan's
  // tokens. And those that no row tile takes, of a request with more new tokens
  // than the caller said: not-a-number, as there is nobody to tell.
  {
    const long long tok = (long long)a.hq * a.dh;
    auto fill = [&](long long i, long long end, unsigned short x) {
      for (i += lane; i < end; i += 32) static_cast<unsigned short*>(a.out)[i] = x;
    };
    const int have = a.row_tiles * M;
    for (int r = w; r < a.requests; r += workers) {
      const int c0 = a.cu_pages[r], c1 = a.cu_pages[r + 1], t0 = a.cu_new[r], t1 = min(a.cu_new[r + 1], a.tokens);
      if (c0 == c1) fill(t0 * tok, t1 * tok, 0);
      else if ((long long)(t1 - t0) * a.group > have)
        for (int i = have / a.group; i < t1 - t0; ++i)
          for (int h = 0; h < a.c.heads; ++h)
            fill((t0 + i) * tok + (long long)(h * a.group + max(0, have - i * a.group)) * a.dh,
                 (t0 + i) * tok + (long long)(h + 1) * a.group * a.dh, 0x7fff);
    }
    for (int i = a.cu_new[a.requests] + w; i < a.tokens; i += workers) fill(i * tok, (i + 1) * tok, 0);
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
// whether a pair begins in that worker's stretch and goes on past it; its
// threads take 4 dims of a row each and, where rows are few, every so many'th
// piece.
template <int DHP>
__global__ void __launch_bounds__(256) kv_join_kernel(const __grid_constant__ KvAttnArgs a, int workers, int M) {
  pdl_wait_then_release();
  __shared__ float2 s_row[32];                    // maximum, 1 / sum
  __shared__ float4 s_acc[256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = blockIdx.x;
  KvSpan sp;
  sp.begin(a, workers, w, lane, true);
  if (sp.done) return;                            // nothing lies past this stretch
  const long long u0 = w * sp.stretch, u1 = u0 + sp.stretch;
  const long long b = sp.u - sp.p0, e = b + sp.nu;
  if (b < u0 || e <= u1) return;                  // begins earlier, or ends here
  const int pieces = (int)((e - 1) / sp.stretch) - w + 1;
  const int head = sp.head, row0 = sp.rt * M;
  const int tok0 = sp.tok0;
  const int rows = min(M, min(sp.n, a.tokens - tok0) * a.group - row0);
  if (rows <= 0) return;
  auto slot = [&](int i) { return i == 0 && b != u0 ? 2ll * w + 1 : 2ll * (w + i); };
  for (int row = warp; row < rows; row += 8) {
    float top = -INFINITY, l = 0.f;
    for (int k = lane; k < pieces; k += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slot(k) * M + row) * 2);
      const float m = fmaxf(top, ml.x), m0 = m == -INFINITY ? 0.f : m;
      l = l * ex2_approx(top - m0) + ml.y * ex2_approx(ml.x - m0);
      top = m;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      const float t2 = __shfl_xor_sync(0xffffffffu, top, s), l2 = __shfl_xor_sync(0xffffffffu, l, s);
      const float m = fmaxf(top, t2), m0 = m == -INFINITY ? 0.f : m;
      l = l * ex2_approx(top - m0) + l2 * ex2_approx(t2 - m0);
      top = m;
    }
    if (lane == 0) s_row[row] = make_float2(top == -INFINITY ? 0.f : top, l == 0.f ? 0.f : 1.0f / l);
  }
  __syncthreads();
  constexpr int LN = DHP / 4, GROUPS = 256 / LN;
  int rp = 1;
  while (rp < rows && rp < GROUPS) rp *= 2;
  const int split = GROUPS / rp;
  const int q = threadIdx.x / LN, d = (threadIdx.x % LN) * 4, mine = q % rp, part = q / rp;
  for (int r0 = 0; r0 < rows; r0 += rp) {
    const int row = r0 + mine;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) {
      const float top = s_row[row].x;
#pragma unroll 8
      for (int k = part; k < pieces; k += split) {
        const long long at = slot(k) * M + row;
        const float f = ex2_approx(a.part_ml[at * 2] - top);
        const float4 o = *reinterpret_cast<const float4*>(a.part_o + at * DHP + d);
        acc.x = fmaf(o.x, f, acc.x);
        acc.y = fmaf(o.y, f, acc.y);
        acc.z = fmaf(o.z, f, acc.z);
        acc.w = fmaf(o.w, f, acc.w);
      }
    }
    if (split > 1) {
      __syncthreads();
      s_acc[threadIdx.x] = acc;
      __syncthreads();
      if (part == 0)
        for (int p = 1; p < split; ++p) {
          const float4 o = s_acc[threadIdx.x + p * rp * LN];
          acc.x += o.x;
          acc.y += o.y;
          acc.z += o.z;
          acc.w += o.w;
        }
    }
    if (part == 0 && row < rows) {
      const float inv = s_row[row].y;
      const int gr = row0 + row, i = gr / a.group;
      const long long at = ((long long)(tok0 + i) * a.hq + head * a.group + gr - i * a.group) * a.dh;
      store_out(a, at, d, acc.x * inv, acc.y * inv);
      store_out(a, at, d + 2, acc.z * inv, acc.w * inv);
    }
  }
}

}  // namespace b200l
