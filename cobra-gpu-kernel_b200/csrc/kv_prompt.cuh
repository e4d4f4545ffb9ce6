// kv_prompt.cuh -- attention of many rows per request over a paged 8-bit cache:
// prompt chunks, whole prompts, long guesses.
//
// Same definition as kv_decode.cuh. A work item is (request, key head, 256 rows
// = two tiles of 128 that share every K / V tile; 128 rows at dhp 256), a row
// being one query head of one new token. The key tiles of all items in a row are
// cut evenly over the SMs, as kv_decode.cuh cuts them over warps: a small kernel
// sums them up first, a block works off its stretch, and of an item that is cut
// each piece leaves (max, sum, accumulator), which kv_prompt_join_kernel adds in
// order. An item counts for kItemCost key tiles more than it has, for that is what
// its queries, its results and the pipeline between two items take.
//
// tcgen05 multiplies fp16, so codes become fp16 (exactly) on their way: bulk
// copies bring a tile's pages as they lie into shared memory, four warps turn
// them into swizzled fp16 rows (K as the K-major operand of S = Q K^T, V as the
// MN-major one of O += P V, the same layout), and the scales stay out of the
// products: per 16 keys, one page's worth at least, the softmax has c = scale
// log2(e) s_k, log2 s_v and 1 / s_v, so that u = c s + log2 s_v is the one fused
// multiply-add that the exponent needs anyway, the row maximum is taken per 16
// raw scores (c >= 0) and the row sum is corrected once per 16 weights. The sum is
// of the fp32 weights; P has them as fp16, off by 2^-11 of themselves or, below
// 2^-14, by 2^-25 of the largest contribution.
//
// Warps: 0 loads pages and scales, 1 issues S of both tiles, 2 / 3 issue P V of
// tile 0 / 1, 4-7 convert, 8.. are the softmax: eight per tile, 16 rows a warp,
// two threads per row with half the keys each, so that each scheduler has four of
// them in turn at loads, maxima and exponentials. 80 registers a thread hold 32
// scores: the first 32 are read for their maximum, the second kept, and the first
// read again.
// P goes back to TMEM as fp16: in
// its own columns where they suffice (dhp <= 64, and dhp 256 with one tile), so
// that the next S is computed meanwhile; over S at dhp 128, where two O and two
// S fill TMEM and the tiles alternate instead. O is rescaled only when a row's
// maximum grew by 2^8.
//
// Bound: exponentials and products alike at dhp 128 (16 per clock and SM, 2048
// clocks a 256 x 128 tile, and 4 x 512 clocks of tcgen05), exponentials below.
// Measured (int8, 32768 keys, 1024 rows a head, 512 at dhp 256): 275 TFLOP/s at dhp
// 32, 542 at 64 (4350 clocks a tile), 764 at 128, 504 at 256. Blocks that took
// every so many'th item, with the softmax in unrolled passes, reached 293, 545, 797
// and 586, and 103 against 112 us on 8 prompts of 960, 16 heads of 64; the even cut
// with the rolled pass takes 673 against 743 us on 6 chunks of unlike length, 32 / 8
// heads of 128. Issue slots are 59 % full on those.
#pragma once

#include "kv_decode.cuh"

namespace b200l {

constexpr int kItemCost = 4;

struct KvPromptArgs {
  KvAttnArgs a;                  // part_o / part_ml: [2 * blocks][rows]([dhp])
  int* cum;                      // [tiles + 1] cost of the row tiles before each, of one head
  int4* info;                    // [tiles] a row tile's request, its first new token, their number, its keys
  int4* starts;                  // [blocks + 1] where each stretch begins: row tile, head, key tile
  int tiles;                     // row tiles of all requests, at most
  int blocks;                    // stretches
};

template <int DHP>
struct KvPromptCfg {
  static constexpr int NQ = DHP == 256 ? 1 : 2;             // query tiles of an item
  static constexpr int MQ = NQ * 128;
  static constexpr int BN = DHP == 256 ? 64 : 128;          // keys of a tile
  static constexpr int ROWB = DHP == 32 ? 64 : 128;         // bytes of a swizzled fp16 row
  static constexpr int NH = DHP * 2 / ROWB;                 // such rows side by side
  static constexpr int Q_BYTES = 128 * DHP * 2;
  static constexpr int KV_BYTES = BN * DHP * 2;             // an fp16 tile of K or V
  static constexpr int C_BYTES = BN * DHP;                  // its codes
  static constexpr int ST8 = DHP <= 64 ? 2 : 1;             // stages of codes
  static constexpr bool OVER = DHP == 128;                  // P overwrites S
  static constexpr int GR = BN / 16;                        // 16-key groups of a tile
  static constexpr int CSLOTS = 8;                          // stages of their constants
  static constexpr int SM_CONST = CSLOTS * (GR + 1) * 16;
  static constexpr int SMEM = NQ * Q_BYTES + 4 * KV_BYTES + ST8 * 2 * C_BYTES + SM_CONST + 48 * 8 + 4 * 48 + 1024;
  static constexpr int SOFT = NQ * 8;                       // softmax warps
  static constexpr int THREADS = 256 + 32 * SOFT;
  static constexpr int S_COL = 0;                           // + 128 t
  static constexpr int P_COL = OVER ? 0 : DHP == 256 ? 64 : 256;
  static constexpr int P_STEP = OVER ? 128 : 64;
  static constexpr int O_COL = DHP <= 64 ? 384 : 256;
  static constexpr int O_STEP = DHP <= 64 ? 64 : 128;
  // Columns of P's 16-key groups: one after another, or over S at the place of
  // the first of every 32 scores, so that none is overwritten that is still read.
  __host__ __device__ static constexpr int p_col(int k) { return OVER ? 64 * (k >> 2) + 32 * ((k >> 1) & 1) + 8 * (k & 1) : 8 * k; }
};

// Where request r's row tiles begin: at floor(cu_new[r] group / MQ) + min(r,
// cu_new[r]) there is room for every request with new tokens; what is left over
// stays empty.
template <int DHP>
__device__ __forceinline__ int kv_first_tile(const KvAttnArgs& a, int r, int cu) {
  return (int)((long long)cu * a.group / KvPromptCfg<DHP>::MQ) + min(r, cu);
}

// The cost of every row tile (of one key tile at least, so that a row without
// keys is written too) and their exclusive sums. One block; a warp takes 32 requests at a
// time, a lane each, and all lanes the tiles of one that has many.
template <int DHP>
__global__ void __launch_bounds__(1024) kv_prompt_plan_kernel(const __grid_constant__ KvPromptArgs p) {
  pdl_wait_then_release();
  using C = KvPromptCfg<DHP>;
  const KvAttnArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < p.tiles; i += 1024) p.cum[i] = 0;
  __syncthreads();
  for (int r0 = warp * 32; r0 < a.requests; r0 += 1024) {
    const int r = min(r0 + lane, a.requests - 1);
    const int cu = a.cu_new[r], n = r0 + lane < a.requests ? a.cu_new[r + 1] - cu : 0;
    const int len = min(max(a.lens[r], 0), min(a.cu_pages[r + 1] - a.cu_pages[r], a.width) << a.c.log2_page);
    const long long rows = (long long)n * a.group;
    const int nt = rows > 0 ? (int)((rows + C::MQ - 1) / C::MQ) : 0, first = kv_first_tile<DHP>(a, r, cu);
    auto put = [&](int i, int req, int f, int tt, int nn, int ll) {  // row tile i of a request
      const long long last = min((long long)(i + 1) * C::MQ, (long long)nn * a.group) - 1;
      const int end = a.causal ? min(ll, max(0, ll - nn + (int)(last / a.group) + 1)) : ll;
      if (f + i >= p.tiles) return;               // (cu_new is no prefix sum)
      p.cum[f + i] = max(1, (end + C::BN - 1) / C::BN) + kItemCost;
      p.info[f + i] = make_int4(req, tt, nn, ll);
    };
    if (nt > 0 && nt <= 2)
      for (int i = 0; i < nt; ++i) put(i, r, first, cu, n, len);
    unsigned many = __ballot_sync(0xffffffffu, nt > 2);
    while (many) {
      const int src = __ffs(many) - 1;
      many &= many - 1;
      const int f = __shfl_sync(0xffffffffu, first, src), nn = __shfl_sync(0xffffffffu, n, src);
      const int ll = __shfl_sync(0xffffffffu, len, src), cc = __shfl_sync(0xffffffffu, cu, src);
      const int count = __shfl_sync(0xffffffffu, nt, src);
      for (int i = lane; i < count; i += 32) put(i, r0 + src, f, cc, nn, ll);
    }
  }
  __syncthreads();
  __shared__ int part[32];
  const int per = (p.tiles + 1023) / 1024, i0 = min(p.tiles, tid * per), i1 = min(p.tiles, i0 + per);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum += p.cum[i];
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int v = part[lane], s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    part[lane] = s - v;
    if (lane == 31) p.cum[p.tiles] = s;
  }
  __syncthreads();
  int at = part[warp] + inc - sum;
  for (int i = i0; i < i1; ++i) {
    const int v = p.cum[i];
    p.cum[i] = at;
    at += v;
  }
  __syncthreads();
  // Where the stretches begin. Cost u of all lies in the item that it falls into, at
  // the key tile past what the item itself costs; at its first one within that.
  const long long all = (long long)a.c.heads * p.cum[p.tiles], mean = (all + p.blocks - 1) / p.blocks;
  const long long c = mean < kItemCost + 2 ? kItemCost + 2 : mean;
  for (int b = tid; b <= p.blocks; b += 1024) {
    const long long u = b * c;
    int4 s = make_int4(p.tiles, 0, 0, 0);
    if (u < all) {
      s.x = find_owner(p.cum, p.tiles, (int)(u / a.c.heads));
      const int c0 = p.cum[s.x], w = p.cum[s.x + 1] - c0;
      const long long off = u - (long long)c0 * a.c.heads;
      s.y = (int)(off / w);
      s.z = max(0, (int)(off - (long long)s.y * w) - kItemCost);
    }
    p.starts[b] = s;
  }
}

// A piece of work: rows [row0, row0 + MQ) of a request for key head h, key tiles
// [j0, j1). The loading warp finds them and leaves them in a ring for the others.
struct KvItem {
  int done;                      // nothing more to do
  int j0, j1, len;
  int nqt, row0, rows, n;
  int tok0, h, slot;             // slot < 0: the whole item; else where the piece's results go
  int pad;
};
static_assert(sizeof(KvItem) == 48, "four of them in 192 bytes");

// The items of a stretch, one after another.
template <int DHP>
struct KvWalk {
  int x, h, xe, he, je, nt, r;
  KvItem it;
  __device__ __forceinline__ void open(const KvPromptArgs& p) {
    const int c0 = p.cum[x], c1 = p.cum[x + 1];
    const int4 i = p.info[x];
    nt = c1 - c0 - kItemCost;
    r = i.x;
    it.tok0 = i.y;
    it.n = i.z;
    it.len = i.w;
    it.rows = i.z * p.a.group;
    it.row0 = (x - kv_first_tile<DHP>(p.a, i.x, i.y)) * KvPromptCfg<DHP>::MQ;
    it.nqt = it.rows - it.row0 > 128 && KvPromptCfg<DHP>::NQ == 2 ? 2 : 1;
  }
  // Slot 2b holds a piece that an earlier block began, 2b + 1 one that a later block goes on with.
  __device__ __forceinline__ void cut(int b) {
    const bool at_end = x == xe && h == he;
    it.j1 = at_end ? je : nt;
    it.h = h;
    it.done = it.j0 >= it.j1;                     // (at the end, or both ends in what one item itself costs)
    it.slot = it.j0 == 0 && it.j1 == nt ? -1 : 2 * b + (it.j0 == 0 ? 1 : 0);
  }
  __device__ __forceinline__ void begin(const KvPromptArgs& p, int b) {
    const int4 s = p.starts[b], e = p.starts[b + 1];
    x = s.x;
    h = s.y;
    it.j0 = s.z;
    xe = e.x;
    he = e.y;
    je = e.z;
    it.done = x >= p.tiles;
    if (it.done) return;
    open(p);
    cut(b);
  }
  __device__ __forceinline__ void next(const KvPromptArgs& p, int b, int lane) {
    it.done = x == xe && h == he;
    if (it.done) return;
    it.j0 = 0;
    if (++h == p.a.c.heads) {
      h = 0;
      const int after = p.cum[x + 1];
      it.done = after >= p.cum[p.tiles];          // that was the last one
      if (it.done) return;
      if (p.cum[++x + 1] == after) x = warp_find_owner(p.cum, p.tiles, after, lane);   // (empty ones)
      open(p);
    }
    cut(b);
  }
};

// Shared-memory descriptor of an MN-major B operand: K rows of ROWB bytes, 8 of
// them a swizzle atom, atoms SBO = 8 ROWB apart along K and LBO along N.
__device__ __forceinline__ uint64_t sdesc_mnmajor(uint32_t saddr, int row_bytes, uint32_t lbo) {
  uint64_t d = sdesc_kmajor(saddr, row_bytes);
  d &= ~(uint64_t(0x3fff) << 16);
  return d | (uint64_t)((lbo >> 4) & 0x3fff) << 16;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The barrier that every warp ends on. Each kind of warp has its own, and never
// meets the others' code again, so that its register count is its own too.
__device__ __forceinline__ void block_end() {
  __syncwarp();
  asm volatile("bar.sync 0;" ::: "memory");
}

template <int DHP, int KIND>
__global__ void __launch_bounds__(KvPromptCfg<DHP>::THREADS, 1) kv_prompt_kernel(const __grid_constant__ KvPromptArgs p, DevStatus* status) {
  using C = KvPromptCfg<DHP>;
  constexpr int BN = C::BN, GR = C::GR, NP = BN / 64;   // pieces of 32 keys a thread
  const KvAttnArgs& a = p.a;
  pdl_wait_then_release();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::NQ * C::Q_BYTES;
  uint8_t* sV = sK + 2 * C::KV_BYTES;
  uint8_t* c8K = sV + 2 * C::KV_BYTES;
  uint8_t* c8V = c8K + C::ST8 * C::C_BYTES;
  float4* consts = reinterpret_cast<float4*>(c8V + C::ST8 * C::C_BYTES);   // [CSLOTS][GR + 1]; the last: .x = plain
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(consts) + C::SM_CONST);
  uint64_t* q_full = bars;          // [2]
  uint64_t* q_empty = bars + 2;     // [2]
  uint64_t* k8_full = bars + 4;     // [2]
  uint64_t* k8_free = bars + 6;     // [2]
  uint64_t* v8_full = bars + 8;     // [2]
  uint64_t* v8_free = bars + 10;    // [2]
  uint64_t* k_full = bars + 12;     // [2]
  uint64_t* k_empty = bars + 14;    // [2]
  uint64_t* v_full = bars + 16;     // [2]
  uint64_t* v_empty = bars + 18;    // [2]
  uint64_t* s_full = bars + 20;     // [2]
  uint64_t* s_free = bars + 22;     // [2]
  uint64_t* p_full = bars + 24;     // [2]
  uint64_t* pv_done = bars + 26;    // [2]
  uint64_t* c_full = bars + 28;     // [CSLOTS]
  uint64_t* mma_done = bars + 36;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 37);
  WaitCtl* wc = reinterpret_cast<WaitCtl*>(bars + 38);   // 38, 39
  uint64_t* i_full = bars + 40;     // [4]
  uint64_t* i_free = bars + 44;     // [4]
  KvItem* ring = reinterpret_cast<KvItem*>(bars + 48);   // [4]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 8);
      mbar_init(&q_empty[i], 1);
      mbar_init(&k8_full[i], 1);
      mbar_init(&k8_free[i], 4);
      mbar_init(&v8_full[i], 1);
      mbar_init(&v8_free[i], 4);
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], C::NQ);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 8);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < C::CSLOTS; ++i) mbar_init(&c_full[i], 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&i_full[i], 1);
      mbar_init(&i_free[i], 1 + C::NQ + 4 + C::SOFT);
    }
    mbar_init(mma_done, 1 + C::NQ);
    waitctl_init(wc, status);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int P = a.c.page, lp = a.c.log2_page, PB = P < BN ? P : BN;

  if (warp < 4) {
    if (warp == 0) {  // ================= pages and scales
      int g = 0, gk = 0, gv = 0;                  // tiles; K and V copies begun
      bool ok = true;
      KvWalk<DHP> walk;
      walk.begin(p, blockIdx.x);
      for (int k = 0; ok; ++k, walk.next(p, blockIdx.x, lane)) {
        if (!mbar_wait_warp(&i_free[k & 3], ((k >> 2) & 1) ^ 1, wc)) break;
        if (lane == 0) {
          ring[k & 3] = walk.it;
          mbar_arrive(&i_full[k & 3]);
        }
        if (walk.it.done) break;
        const int* row = a.table + walk.r * a.table_stride;
        const int j0 = walk.it.j0, j1 = walk.it.j1, len = walk.it.len, head = walk.it.h;
        auto entry_at = [&](int j) {              // page of this lane's part of key tile j
          const int k = j * BN + lane * PB;
          return (lane * PB < BN && k < len && (k >> lp) < a.width) ? row[k >> lp] : -1;
        };
        int next = j0 < j1 ? entry_at(j0) : -1;
        for (int j = j0; j < j1; ++j, ++g) {
          const int s8 = g % C::ST8, cs = g % C::CSLOTS, id = next;
          if (j + 1 < j1) next = entry_at(j + 1);
          const bool there = id >= 0 && id < a.c.num_pages;
          const long long ph = there ? (long long)id * a.c.heads + head : 0;
          const float sk = there ? a.c.k_scale[ph] : 0.f, sv = there ? a.c.v_scale[ph] : 0.f;
          const long long src = ((ph << lp) + ((j * BN + lane * PB) & (P - 1))) * DHP;
          const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, there));
          const uint32_t parity = ((g / C::ST8) & 1) ^ 1;
          if (!mbar_wait_warp(&k8_free[s8], parity, wc)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(&k8_full[s8], boxes * (uint32_t)(PB * DHP));
          __syncwarp();
          if (there) bulk_load(c8K + s8 * C::C_BYTES + lane * PB * DHP, a.c.k + src, PB * DHP, &k8_full[s8]);
          ++gk;
          bool poison = false;
          // The constants of this lane's keys, 16 at a time.
          if (lane * PB < BN) {
            // w: 0 no such page, 1 a page, 2 one whose scales are no numbers: its keys
            // become not-a-number, and their visible scores with them; its constants are
            // finite.
            const bool fine = sk - sk == 0.f && sv - sv == 0.f;
            const float svc = fmaxf(sv, 7.8886090522101181e-31f);      // 2^-100 for a page of zeros, or less
            float4 c;
            c.x = fine ? sk : 0.f;
            c.y = !there ? -INFINITY : fine ? lg2_approx(svc) : 0.f;
            c.z = !there ? 0.f : fine ? rcp_approx(svc) : 1.f;
            c.w = !there ? 0.f : fine ? 1.f : 2.f;
            poison = there && !fine;
            for (int i = 0; i < PB / 16; ++i) consts[cs * (GR + 1) + lane * (PB / 16) + i] = c;
          }
          const int want = min(BN / PB, (len - j * BN + PB - 1) / PB);
          poison = __any_sync(0xffffffffu, poison);
          if (lane == 0)
            consts[cs * (GR + 1) + GR].x = (int)boxes >= want && (j + 1) * BN <= len && !poison ? 1.f : 0.f;
          __syncwarp();
          if (lane == 0) mbar_arrive(&c_full[cs]);
          if (!mbar_wait_warp(&v8_free[s8], parity, wc)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(&v8_full[s8], boxes * (uint32_t)(PB * DHP));
          __syncwarp();
          if (there) bulk_load(c8V + s8 * C::C_BYTES + lane * PB * DHP, a.c.v + src, PB * DHP, &v8_full[s8]);
          ++gv;
        }
      }
      // Copies in flight land before the block goes (each stage's last one).
      for (int i = max(0, gk - C::ST8); i < gk; ++i) mbar_drain(&k8_full[i % C::ST8], (i / C::ST8) & 1);
      for (int i = max(0, gv - C::ST8); i < gv; ++i) mbar_drain(&v8_full[i % C::ST8], (i / C::ST8) & 1);
      block_end();
      if (lane == 0 && waitctl_aborted(wc)) record_error(status, -7, kKernelKvPrompt, 1);
    } else if (warp == 1) {  // ================= S_t(j) = Q_t K_j^T
      const uint32_t idesc_s = idesc_f16_f32(128, BN);
      const uint64_t dq0 = sdesc_kmajor(smem_u32(sQ), C::ROWB);
      const uint64_t dk0 = sdesc_kmajor(smem_u32(sK), C::ROWB);
      int g = 0, ns[2] = {0, 0}, qi[2] = {0, 0};
      bool ok = true;
      for (int k = 0; ok; ++k) {
        if (!mbar_wait_warp(&i_full[k & 3], (k >> 2) & 1, wc)) break;
        // (shuffled, the values are known to be the same for all lanes: what is
        // computed of them stays in uniform registers, as the products want it)
        const int more = __shfl_sync(0xffffffffu, ring[k & 3].done ? 0 : 1, 0);
        if (!more) break;
        const int j0 = __shfl_sync(0xffffffffu, ring[k & 3].j0, 0), j1 = __shfl_sync(0xffffffffu, ring[k & 3].j1, 0);
        const int nqt = __shfl_sync(0xffffffffu, ring[k & 3].nqt, 0);
        if (lane == 0) {
          mbar_arrive(&i_free[k & 3]);
          for (int t = 0; t < nqt && ok; ++t) ok = mbar_wait(&q_full[t], qi[t]++ & 1, wc);
          for (int j = j0; j < j1 && ok; ++j, ++g) {
            const int st = g & 1;
            if (!mbar_wait(&k_full[st], (g >> 1) & 1, wc)) { ok = false; break; }
            const uint64_t dk = dk0 + (uint64_t)((st * C::KV_BYTES) >> 4);
            for (int t = 0; t < nqt; ++t) {
              // S_t's columns are free once the softmax has read them; where P
              // takes their place, once P V has read that.
              if (ns[t] > 0 && !mbar_wait(C::OVER ? &pv_done[t] : &s_free[t], (ns[t] - 1) & 1, wc)) { ok = false; break; }
              const uint64_t dq = dq0 + (uint64_t)((t * C::Q_BYTES) >> 4);
              const uint32_t d_s = tmem_base + C::S_COL + t * 128;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < DHP / 16; ++k) {
                constexpr int R = C::ROWB;
                const uint32_t off_q = (uint32_t)((k * 32) / R) * (128 * R) + (k * 32) % R;
                const uint32_t off_k = (uint32_t)((k * 32) / R) * (BN * R) + (k * 32) % R;
                umma_f16_ss(d_s, dq + (off_q >> 4), dk + (off_k >> 4), idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit(&s_full[t]);
              ++ns[t];
            }
            if (ok) umma_commit(&k_empty[st]);
          }
          if (ok)
            for (int t = 0; t < nqt; ++t) umma_commit(&q_empty[t]);
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      if (lane == 0) {
        umma_commit(mma_done);
        mbar_drain(mma_done, 0);
      }
      block_end();
      tc_fence_after();
      tmem_dealloc(tmem_base, 512);
    } else if (warp - 2 < C::NQ) {  // ================= O_t += P_t(j) V_j
      const int t = warp - 2;
      const uint32_t idesc_o = idesc_f16_f32(128, DHP) | (1u << 16);       // B is MN-major
      const uint64_t dv0 = sdesc_mnmajor(smem_u32(sV), C::ROWB, BN * C::ROWB);
      const uint32_t a_p = tmem_base + C::P_COL + t * C::P_STEP;
      const uint32_t d_o = tmem_base + C::O_COL + t * C::O_STEP;
      int g = 0, np = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        if (!mbar_wait_warp(&i_full[k & 3], (k >> 2) & 1, wc)) break;
        // (shuffled, the values are known to be the same for all lanes: what is
        // computed of them stays in uniform registers, as the products want it)
        const int more = __shfl_sync(0xffffffffu, ring[k & 3].done ? 0 : 1, 0);
        if (!more) break;
        const int j0 = __shfl_sync(0xffffffffu, ring[k & 3].j0, 0), j1 = __shfl_sync(0xffffffffu, ring[k & 3].j1, 0);
        const int nqt = __shfl_sync(0xffffffffu, ring[k & 3].nqt, 0);
        if (lane == 0) {
          mbar_arrive(&i_free[k & 3]);
          for (int j = j0; j < j1 && ok; ++j, ++g) {
            const int st = g & 1;
            if (!mbar_wait(&v_full[st], (g >> 1) & 1, wc)) { ok = false; break; }
            if (t >= nqt) {                    // no second tile: the stage is released as it comes
              umma_commit(&v_empty[st]);
              continue;
            }
            if (!mbar_wait(&p_full[t], np & 1, wc)) { ok = false; break; }
            const uint64_t dv = dv0 + (uint64_t)((st * C::KV_BYTES) >> 4);
            const uint32_t acc0 = j > j0 ? 1u : 0u;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              umma_f16_ts(d_o, a_p + C::p_col(k), dv + ((uint32_t)(k * 16 * C::ROWB) >> 4), idesc_o, k > 0 ? 1u : acc0);
            umma_commit(&pv_done[t]);
            umma_commit(&v_empty[st]);
            ++np;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      if (lane == 0) {
        umma_commit(mma_done);
        mbar_drain(mma_done, 0);
      }
      block_end();
    } else {
      block_end();
    }
    return;
  } else if (warp < 8) {  // ================= codes -> fp16
    const int tid = threadIdx.x - 128;
    constexpr int UPR = DHP / 16;                 // 16-code pieces of a row
    constexpr int UNITS = BN * UPR / 128;         // ... of a thread
    constexpr int UPH = C::ROWB / 32;             // ... of a swizzled fp16 row
    int g = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!mbar_wait_warp(&i_full[k & 3], (k >> 2) & 1, wc)) break;
      if (ring[k & 3].done) break;
      const int j0 = ring[k & 3].j0, j1 = ring[k & 3].j1, len = ring[k & 3].len;
      __syncwarp();
      if (lane == 0) mbar_arrive(&i_free[k & 3]);
      for (int j = j0; j < j1 && ok; ++j, ++g) {
        const int s8 = g % C::ST8, cs = g % C::CSLOTS, st = g & 1;
        if (!mbar_wait_warp(&c_full[cs], (g / C::CSLOTS) & 1, wc)) { ok = false; break; }
        const float4* cc = consts + cs * (GR + 1);
        const bool plain = cc[GR].x != 0.f;       // every key there, and a number
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          uint64_t* full8 = which ? &v8_full[s8] : &k8_full[s8];
          uint64_t* free8 = which ? &v8_free[s8] : &k8_free[s8];
          uint64_t* full = which ? &v_full[st] : &k_full[st];
          uint64_t* empty = which ? &v_empty[st] : &k_empty[st];
          const uint8_t* src = (which ? c8V : c8K) + s8 * C::C_BYTES;
          const uint32_t dst = smem_u32((which ? sV : sK) + st * C::KV_BYTES);
          if (!mbar_wait_warp(full8, (g / C::ST8) & 1, wc) || !mbar_wait_warp(empty, ((g >> 1) & 1) ^ 1, wc)) {
            ok = false;
            break;
          }
          constexpr int BATCH = UNITS < 4 ? UNITS : 4;
#pragma unroll 1
          for (int u0 = 0; u0 < UNITS; u0 += BATCH) {
            uint4 w[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) w[i] = *reinterpret_cast<const uint4*>(src + ((u0 + i) * 128 + tid) * 16);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int unit = (u0 + i) * 128 + tid, row = unit / UPR, c16 = unit % UPR;
              // What lies past the keys, or in a page that is not there, is no code.
              const float page = plain ? 1.f : cc[row >> 4].w;
              if (!plain && (j * BN + row >= len || page == 0.f)) w[i] = make_uint4(0, 0, 0, 0);
              uint32_t h[8];
              codes4_to_half<KIND>(w[i].x, h[0], h[1]);
              codes4_to_half<KIND>(w[i].y, h[2], h[3]);
              codes4_to_half<KIND>(w[i].z, h[4], h[5]);
              codes4_to_half<KIND>(w[i].w, h[6], h[7]);
              if (page == 2.f && which == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = 0x7e007e00u;
              }
              const int hb = c16 / UPH, ch = 2 * (c16 % UPH), odd = hb & 1;
              const uint32_t base = dst + hb * BN * C::ROWB;
              // (neighbouring halves write their odd pieces first: no bank conflicts)
              st_shared_v4(base + swz_offset(row, ch + odd, C::ROWB), odd ? h[4] : h[0], odd ? h[5] : h[1], odd ? h[6] : h[2],
                           odd ? h[7] : h[3]);
              st_shared_v4(base + swz_offset(row, ch + 1 - odd, C::ROWB), odd ? h[0] : h[4], odd ? h[1] : h[5],
                           odd ? h[2] : h[6], odd ? h[3] : h[7]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(full);
            mbar_arrive(free8);
          }
        }
      }
    }
    block_end();
    return;
  } else {  // ================= softmax
    const int sw = warp - 8, t = sw >> 3, hh = (sw >> 2) & 1, c = lane >> 4;   // c: which half of the keys, and dims
    const int row = (warp & 3) * 32 + hh * 16 + (lane & 15);
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32 + hh * 16) << 16;
    const uint32_t t_s = tmem_base + lane_off + C::S_COL + t * 128;
    const uint32_t t_p = tmem_base + lane_off + C::P_COL + t * C::P_STEP;
    const uint32_t t_o = tmem_base + lane_off + C::O_COL + t * C::O_STEP;
    constexpr int OH = DHP / 2;                   // dims of this thread
    int g = 0, ns = 0, np = 0, qi = 0;
    bool ok = true;
    // Rows past the plan's tokens.
    for (long long i = (long long)a.cu_new[a.requests] * a.hq * a.dh + (blockIdx.x * C::SOFT + sw) * 32 + lane,
                   e = (long long)a.tokens * a.hq * a.dh;
         i < e; i += (long long)gridDim.x * C::SOFT * 32)
      static_cast<unsigned short*>(a.out)[i] = 0;
    for (int k = 0; ok; ++k) {
      if (!mbar_wait_warp(&i_full[k & 3], (k >> 2) & 1, wc)) break;
      const volatile KvItem& it = ring[k & 3];    // (read again after the tiles: registers are what is short)
      if (it.done) break;
      if (t >= it.nqt) {
        g += it.j1 - it.j0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&i_free[k & 3]);
        continue;
      }
      const int gr = it.row0 + t * 128 + row, i = gr / a.group, hq = it.h * a.group + gr - i * a.group;
      const bool in = gr < it.rows && it.tok0 + i < a.tokens;
      const int lim = !in ? 0 : a.causal ? min(it.len, it.len - it.n + i + 1) : it.len;
      const int first = (it.row0 + t * 128) / a.group;              // the tile's first token sees least
      const int lim_min = a.causal ? min(it.len, it.len - it.n + first + 1) : it.len;
      const int jbeg = it.j0, jend = it.j1;
      float qs = a.scale_log2, m_use = 0.f, l = 0.f;
      bool none = true;                           // no visible key so far
      {  // ---- the row of Q as fp16, scaled by a power of two if it comes as bf16
        const long long at = (long long)(it.tok0 + i) * a.q_st + (long long)hq * a.q_sh;
        const uint4* q8 = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + at);
        const unsigned short* q1 = static_cast<const unsigned short*>(a.q) + at;
        const bool vec = a.q_vec8 && DHP == a.dh;  // (uniform)
        auto slow8 = [&](int d) {                 // dims [d, d + 8), one by one
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = in && d + 2 * k < a.dh ? q1[d + 2 * k] : 0u;
            const uint32_t y = in && d + 2 * k + 1 < a.dh ? q1[d + 2 * k + 1] : 0u;
            w[k] = x | y << 16;
          }
          return make_uint4(w[0], w[1], w[2], w[3]);
        };
        const uint32_t dst = smem_u32(sQ + t * C::Q_BYTES);
        auto put8 = [&](int d, uint4 u) {
          const int chunk = d / 8;
          st_shared_v4(dst + (chunk / (C::ROWB / 16)) * 128 * C::ROWB + swz_offset(row, chunk % (C::ROWB / 16), C::ROWB), u.x,
                       u.y, u.z, u.w);
        };
        constexpr int QC = OH / 8 < 4 ? OH / 8 : 4;   // pieces of 8 dims under way at once
        float mul = 1.f;
        if (a.type == kElemBF16) {
          // The largest of the row: as whole numbers, values without their sign are in order.
          uint32_t big = 0;
#pragma unroll 1
          for (int d = 0; d < OH; d += 8 * QC) {
            uint4 u[QC];
#pragma unroll
            for (int k = 0; k < QC; ++k)
              u[k] = vec ? (in ? q8[(c * OH + d) / 8 + k] : make_uint4(0, 0, 0, 0)) : slow8(c * OH + d + 8 * k);
#pragma unroll
            for (int k = 0; k < QC; ++k)
              big = __vmaxu2(big, __vmaxu2(__vmaxu2(u[k].x & 0x7fff7fffu, u[k].y & 0x7fff7fffu),
                                           __vmaxu2(u[k].z & 0x7fff7fffu, u[k].w & 0x7fff7fffu)));
          }
          big = max(big & 0xffffu, big >> 16);
          big = max(big, __shfl_xor_sync(0xffffffffu, big, 16));
          if (big != 0 && big < 0x7f80u) {
            const int ex = min(max((int)(big >> 7) - 127, -120), 120);
            mul = __int_as_float((127 - ex) << 23);
            qs *= __int_as_float((127 + ex) << 23);
          }
        }
        if (!mbar_wait_warp(&q_empty[t], (qi & 1) ^ 1, wc)) { ok = false; break; }
        ++qi;
#pragma unroll 1
        for (int d = 0; d < OH; d += 8 * QC) {
          uint4 u[QC];
#pragma unroll
          for (int k = 0; k < QC; ++k)
            u[k] = vec ? (in ? q8[(c * OH + d) / 8 + k] : make_uint4(0, 0, 0, 0)) : slow8(c * OH + d + 8 * k);
          if (a.type == kElemBF16) {
#pragma unroll
            for (int k = 0; k < QC; ++k) {
              uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_half2(__uint_as_float(w[e] << 16) * mul, __uint_as_float(w[e] & 0xffff0000u) * mul);
              u[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
#pragma unroll
          for (int k = 0; k < QC; ++k) put8(c * OH + d + 8 * k, u[k]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
      }
      for (int j = jbeg; j < jend; ++j, ++g) {
        const int cs = g % C::CSLOTS;
        if (!mbar_wait_warp(&c_full[cs], (g / C::CSLOTS) & 1, wc) || !mbar_wait_warp(&s_full[t], ns & 1, wc)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // This thread's keys: 32 NP from BN/2 c on, in pieces of 32.
        const float4* cc = consts + cs * (GR + 1) + c * (GR / 2);
        const bool edge = (j + 1) * BN > lim_min; // (warp-uniform)
        float s[32];
        auto load = [&](int h) {
          tmem_ld_pair32<BN / 2>(t_s + 32 * h, *reinterpret_cast<uint32_t(*)[32]>(s));
          if (edge) {
            const int left = lim - (j * BN + (BN / 2) * c + 32 * h);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k >= left) s[k] = -INFINITY;
          }
        };
        // (A factor is above 0, so that hidden keys stay hidden: -inf * 0 is no number.)
        auto top = [&](int h) {
          float m[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float2 k2 = *reinterpret_cast<const float2*>(cc + 2 * h + q);
            float m0 = fmaxf(s[16 * q], s[16 * q + 1]), m1 = fmaxf(s[16 * q + 2], s[16 * q + 3]);
#pragma unroll
            for (int k = 4; k < 16; k += 4) {
              m0 = fmax3f(m0, s[16 * q + k], s[16 * q + k + 1]);
              m1 = fmax3f(m1, s[16 * q + k + 2], s[16 * q + k + 3]);
            }
            m[q] = fmaf(fmaxf(m0, m1), fmaxf(k2.x * qs, 1e-37f), k2.y);
          }
          return fmaxf(m[0], m[1]);
        };
        uint32_t pk[16];
        auto weigh = [&](int h) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 k4 = cc[2 * h + q];      // (read again: registers are what is short)
            const float cq = fmaxf(k4.x * qs, 1e-37f), lm = k4.y - m_use;
            const float2 c2 = make_float2(cq, cq), l2 = make_float2(lm, lm);
            float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 x = __ffma2_rn(make_float2(s[16 * q + 2 * k], s[16 * q + 2 * k + 1]), c2, l2);
              const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              if (k & 1) a1 = __fadd2_rn(a1, e);
              else a0 = __fadd2_rn(a0, e);
              pk[8 * q + k] = pack_half2(e.x, e.y);
            }
            const float2 as = __fadd2_rn(a0, a1);
            l = fmaf(as.x + as.y, k4.z, l);
          }
        };
        // P of piece h: its columns, and those of the other half of the keys.
        auto store = [&](int h) {
          if constexpr (C::OVER) tmem_st_pair16<64>(t_p + 32 * h, pk);
          else tmem_st_pair16<BN / 4>(t_p + 16 * h, pk);
        };
        float hm = -INFINITY, alpha = 1.f;
        bool rescale = false;
        // The pieces' maxima, the last one's weights, the first one's: one loop, for the
        // sake of the instruction caches, which four kinds of warps share.
#pragma unroll 1
        for (int pass = 0; pass < 2 * NP - 1; ++pass) {
          const int h = NP == 2 ? pass & 1 : 0;
          load(h);
          if (pass < NP) hm = fmaxf(hm, top(h));
          if (pass < NP - 1) continue;
          if (pass == NP - 1) {
            const float m_cand = fmaxf(hm, __shfl_xor_sync(0xffffffffu, hm, 16));
            if (none) {
              if (m_cand > -INFINITY) {
                none = false;
                m_use = m_cand;
              }
            } else if (m_cand > m_use + 8.f) {
              alpha = ex2_approx(m_use - m_cand);
              m_use = m_cand;
              rescale = true;
            }
            l *= alpha;
          }
          if (pass == 2 * NP - 2) {
            if constexpr (!C::OVER) {             // the next S may come
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_free[t]);
            }
          }
          weigh(h);
          if (pass == NP - 1 && np > 0) {         // P and O are free once the last P V is done
            ok = mbar_wait_warp(&pv_done[t], (np - 1) & 1, wc);
            if (!ok) break;
            tc_fence_after();
          }
          store(h);
        }
        if (!ok) break;
        ++ns;
        if (j > jbeg && __any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int d = 0; d < OH; d += 16) {
            uint32_t r[16];
            tmem_ld_pair16<OH>(t_o + d, r);
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st_pair16<OH>(t_o + d, r);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        ++np;
      }
      if (!ok) break;
      // ---- the rows' results, or this piece of them
      if (!mbar_wait_warp(&pv_done[t], (np - 1) & 1, wc)) { ok = false; break; }
      tc_fence_after();
      const float lt = l + __shfl_xor_sync(0xffffffffu, l, 16);
      const float r1 = lt == 0.f ? 0.f : 1.0f / lt;
      const int slot = it.slot, gr2 = it.row0 + t * 128 + row, i2 = gr2 / a.group, tok = it.tok0 + i2;
      const bool whole = slot < 0, mine = gr2 < it.rows && tok < a.tokens;
      const long long oat = ((long long)tok * a.hq + it.h * a.group + gr2 - i2 * a.group) * a.dh;
      const long long pr = (long long)slot * C::MQ + t * 128 + row;
      if (!whole && mine && c == 0) *reinterpret_cast<float2*>(a.part_ml + pr * 2) = make_float2(none ? -INFINITY : m_use, lt);
#pragma unroll 1
      for (int d = 0; d < OH; d += 16) {
        uint32_t r[16];
        tmem_ld_pair16<OH>(t_o + d, r);
        const int d0 = c * OH + d;
        if (mine) {
          if (!whole) {
            float4* o = reinterpret_cast<float4*>(a.part_o + pr * DHP + d0);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]), __uint_as_float(r[4 * k + 2]),
                                 __uint_as_float(r[4 * k + 3]));
          } else if (a.o_vec8 && d0 + 16 <= a.dh) {
            uint4* o = reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + oat + d0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_elem2(__uint_as_float(r[8 * k + 2 * e]) * r1, __uint_as_float(r[8 * k + 2 * e + 1]) * r1, a.type);
              o[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 2)
              if (d0 + k < a.dh) store_out(a, oat, d0 + k, __uint_as_float(r[k]) * r1, __uint_as_float(r[k + 1]) * r1);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (lane == 0) mbar_arrive(&i_free[k & 3]);
    }
    block_end();
  }
}

// Adds the pieces of every item that was cut, in order. blockIdx.x: the stretch
// that the item begins in and goes on past; blockIdx.y: eight of its rows, a warp
// each.
template <int DHP>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(const __grid_constant__ KvPromptArgs p) {
  pdl_wait_then_release();
  using C = KvPromptCfg<DHP>;
  const KvAttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = blockIdx.x;
  const int4 from = p.starts[w], to = p.starts[w + 1];
  // The stretch's end cuts an item, and its beginning does not cut the same one.
  if (to.x >= p.tiles || to.z == 0 || (from.x == to.x && from.y == to.y && from.z > 0)) return;
  KvWalk<DHP> walk;
  walk.x = to.x;
  walk.open(p);
  KvItem& it = walk.it;
  it.h = to.y;
  int pieces = 2;
  for (int b = w + 2; b <= p.blocks; ++b, ++pieces) {
    const int4 s = p.starts[b];
    if (s.x != to.x || s.y != to.y) break;
  }
  auto slot = [&](int i) { return i == 0 ? 2 * w + 1 : 2 * (w + i); };
  for (int row = blockIdx.y * 8 + warp; row < C::MQ; row += gridDim.y * 8) {
    const int gr = it.row0 + row, i = gr / a.group;
    if (gr >= it.rows || it.tok0 + i >= a.tokens) break;
    float top = -INFINITY;
    for (int k = lane; k < pieces; k += 32) top = fmaxf(top, a.part_ml[((long long)slot(k) * C::MQ + row) * 2]);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (top == -INFINITY) top = 0.f;
    constexpr int PER = DHP / 32;
    float acc[PER], l = 0.f;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll 4
    for (int k = 0; k < pieces; ++k) {
      const long long pr = (long long)slot(k) * C::MQ + row;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + pr * 2);
      const float f = ex2_approx(ml.x - top);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[d] = fmaf(a.part_o[pr * DHP + d * 32 + lane], f, acc[d]);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const long long o = ((long long)(it.tok0 + i) * a.hq + it.h * a.group + gr - i * a.group) * a.dh;
#pragma unroll
    for (int d = 0; d < PER; ++d) {
      const int dim = d * 32 + lane;
      if (dim < a.dh) {
        if (a.type == kElemF16) static_cast<__half*>(a.out)[o + dim] = __float2half_rn(acc[d] * inv);
        else static_cast<__nv_bfloat16*>(a.out)[o + dim] = __float2bfloat16_rn(acc[d] * inv);
      }
    }
  }
}

}  // namespace b200l
