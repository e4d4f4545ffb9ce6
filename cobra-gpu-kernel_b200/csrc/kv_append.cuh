// kv_append.cuh -- new keys and values quantised into the pages of an 8-bit
// cache, and the values that codes stand for read back by slot.
//
// The tokens of a page share one scale per head. With a = max |x| over the
// page's new tokens and the head's dims, their scale has to be at least
//   int8: a / 127        e4m3: the least power of two s with a <= 448 s
// and the page's becomes s = max(scale so far, that), where a page written from
// its first place on has no scale so far. Codes already there move from s' to s
// when it grew: c <- rn(c s' / s); new ones are rn(x / s). (A power of two
// costs an e4m3 code no precision, and moving codes between two of them is
// exact but for the subnormal ones. int8 codes want the whole range: there each
// growth may cost an older code half a step, and a page's running maximum
// grows about ln(P) times when it is written token by token.) All of it is
// fp32 with correctly rounded division, so the codes do not depend on how the
// tokens are spread over warps. Values that are not finite make the scale
// not-a-number: whoever attends to that page gets not-a-number, as without a
// cache; the codes themselves are then 0.
//
// A run is a stretch of tokens whose slots follow one another inside a page;
// each page's new tokens have to be one run. A group of GW warps takes the runs
// that begin in its window of W tokens, for one head of K or V. A few runs (a
// prompt's pages) are shared by the whole group, one run after another; many (a
// decode batch's tokens) go to a warp each. Lanes share a token (8 dims each)
// and hold 4 tokens, all in flight together and loaded once where GW suffices
// for 64 tokens (dhp <= 128). Then the page's scale, the older codes if it grew,
// and the new codes. What does not fit is looked at twice, the second time from
// L1 / L2.
//
// Bound: HBM, 2 (or 4) bytes read and 1 written per value. A run is a chain of
// some 3000 clocks (slots, values and scale, maximum, codes), so about 45 KB of
// values have to be on their way in an SM: 32 warps of 2 KB. A decode step is
// that chain once. Measured: 65536 prompt tokens, 16 heads of 64, fp16 to e4m3 122
// us (403 MB, 51 % of HBM's rate: instructions a value); 6077 tokens of 24 ragged
// prompts, 8 heads of 128, bf16 to int8 29 us (the chain, on too few runs); 64
// single tokens, 4 heads of 32, 4.4 us.
#pragma once

#include "kv_common.cuh"

namespace b200l {

struct KvAppendArgs {
  KvCache c;
  const void* x[2];              // k, v: element strides below
  long long st[2], sh[2], sd[2]; // per token, head, dim
  int vec[2];                    // rows are read in 16-byte pieces
  const long long* slots;
  long long tokens, num_slots;
  int type, dh, window, windows, pairs;   // pairs: (head, K or V) that a group does one after another
};

template <int KIND>
__device__ __forceinline__ float kv_scale_for(float amax) {
  if (!(amax < INFINITY)) return __int_as_float(0x7fc00000);
  if constexpr (KIND == kKvInt8) {
    return __fdiv_rn(amax, 127.0f);
  } else {
    if (amax == 0.f) return 0.f;
    int e;
    const float m = frexpf(amax, &e);             // amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    return ldexpf(1.0f, max(e - (m <= 0.875f ? 9 : 8), -126));
  }
}

// Codes of four values at scale s: the quotient as fp32 rounds it, rounded to the
// code. A scale of 0 (all of them 0) or not-a-number gives 0; a power of two
// divides exactly by its reciprocal.
template <int KIND>
__device__ __forceinline__ uint32_t kv_code4(float a, float b, float c, float d, float s, float inv) {
  if constexpr (KIND == kKvInt8) {
    // The quotient by way of the reciprocal is off by less than 2^-22 of at most
    // 127: where that could matter, within 2^-13 of a tie, it is divided. Adding
    // 1.5 2^23 rounds to a whole number, ties to even, and leaves it in the low
    // bits; it stays in [-127, 127] since s >= max|x| / 127 but for its rounding
    // (of a subnormal s, to a few bits: there it is cut off).
    const float big = 12582912.0f;
    float q[4] = {a * inv, b * inv, c * inv, d * inv}, r[4];
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = q[i] + big;
      off = fmaxf(off, fabsf(q[i] - (r[i] - big)));
    }
    // (nor is the reciprocal of a scale near the ends of the range any use)
    if (off > 0.49987f || !(s > 1e-30f && s < 1e30f)) {
      if (!(s > 0.f)) return 0;
      const float x[4] = {a, b, c, d};
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = fminf(fmaxf(__fdiv_rn(x[i], s), -127.f), 127.f) + big;
    }
    const uint32_t lo = __byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  } else {
    if (!(s > 0.f)) return 0;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}

// Maximum, not-a-number if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

template <int KIND>
__device__ __forceinline__ float kv_value(uint32_t c) {
  if constexpr (KIND == kKvInt8) return (float)(signed char)c;
  __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

// Eight dims of one token and head as they come: 16 bytes of a 16-bit type, 32
// of fp32; zero past dh.
template <int ESZ>
struct KvPiece {
  uint32_t w[ESZ * 2];
  __device__ __forceinline__ void load(const void* x, long long base, long long sd, int d0, int dh, int vec) {
    if (vec && d0 + 8 <= dh) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + (base + d0) * ESZ);
#pragma unroll
      for (int i = 0; i < ESZ / 2; ++i) {
        const uint4 u = p[i];
        w[4 * i] = u.x;
        w[4 * i + 1] = u.y;
        w[4 * i + 2] = u.z;
        w[4 * i + 3] = u.w;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = d0 + i < dh;
      const long long at = base + (d0 + i) * sd;
      if constexpr (ESZ == 4) {
        w[i] = in ? static_cast<const uint32_t*>(x)[at] : 0u;
      } else {
        const uint32_t h = in ? static_cast<const unsigned short*>(x)[at] : 0u;
        if (i & 1) w[i / 2] |= h << 16;
        else w[i / 2] = h;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < ESZ * 2; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float2 two(int i, int type) const {   // dims 2i, 2i + 1
    if constexpr (ESZ == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if (type == kElemF16) return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
  }
  // max(m, |x|), not-a-number if any is
  __device__ __forceinline__ float amax(float m, int type) const {
    if constexpr (ESZ == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(__uint_as_float(w[i])));
      return m;
    } else if (type == kElemF16) {
      const __half2* h = reinterpret_cast<const __half2*>(w);
      const __half2 x = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
      const float2 f = __half22float2(x);
      return max_nan(m, max_nan(f.x, f.y));
    } else {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
      const __nv_bfloat162 x = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
      const float2 f = __bfloat1622float2(x);
      return max_nan(m, max_nan(f.x, f.y));
    }
  }
  template <int KIND>
  __device__ __forceinline__ uint2 codes(float s, float inv, int type) const {
    const float2 a = two(0, type), b = two(1, type), c = two(2, type), d = two(3, type);
    return make_uint2(kv_code4<KIND>(a.x, a.y, b.x, b.y, s, inv), kv_code4<KIND>(c.x, c.y, d.x, d.y, s, inv));
  }
};

// Warps of a group: as many as hold 64 tokens in registers, at most a block.
__host__ __device__ constexpr int kv_append_group(int dhp) { return dhp <= 32 ? 2 : dhp <= 64 ? 4 : 8; }

template <int DHP, int KIND, int ESZ>
__global__ void __launch_bounds__(256, ESZ == 2 ? 4 : 3) kv_append_kernel(KvAppendArgs a) {
  pdl_wait_then_release();
  constexpr int LPT = DHP / 8;                    // lanes that share a token
  constexpr int TPW = 32 / LPT;                   // tokens of a warp at a time
  constexpr int U = 4;                            // ... and how many times at once
  constexpr int GW = kv_append_group(DHP);
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5, gw = warp % GW;
  __shared__ float s_max[2][8];
  const unsigned id = blockIdx.x * (8 / GW) + warp / GW;
  const unsigned chunks = (2u * a.c.heads + a.pairs - 1) / a.pairs;
  const int win = (int)(id / chunks), hk0 = (int)(id - win * chunks) * a.pairs;   // neighbours share tokens: their rows lie side by side
  if (win >= a.windows) return;
  const int hk1 = min(hk0 + a.pairs, 2 * a.c.heads), P = a.c.page;
  const long long t0 = (long long)win * a.window;
  const int W = (int)min((long long)a.window, a.tokens - t0);
  const int sub = lane / LPT, d0 = (lane % LPT) * 8;

  // Whether token t leads a run (1), goes on the one before it (0), or has no slot (2).
  auto kind_of = [&](long long t) {
    const long long s = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
    if (s < 0 || s >= a.num_slots) return 2;
    return before < 0 || s != before + 1 || (s & (P - 1)) == 0 ? 1 : 0;
  };
  unsigned long long lead = 0, stop = 0;          // tokens of the window that lead; that do not go on
  for (int i = 0; i < W; i += 32) {
    const int k = i + lane < W ? kind_of(t0 + i + lane) : 2;
    lead |= (unsigned long long)__ballot_sync(0xffffffffu, k == 1) << i;
    stop |= (unsigned long long)__ballot_sync(0xffffffffu, k != 0 && i + lane < W) << i;
  }
  const bool share = __popcll(lead) <= (GW + 1) / 2;   // (group-uniform)
  const int wv = share ? gw : 0, nw = share ? GW : 1;
  for (int nth = 0, turn = 0; lead; ++nth) {
    const int i = __ffsll((long long)lead) - 1;
    lead &= lead - 1;
    if (!share && nth % GW != gw) continue;
    const unsigned long long after = i < 63 ? stop & (~0ull << (i + 1)) : 0;
    int len;
    if (after) {
      len = __ffsll((long long)after) - 1 - i;
    } else {                                      // on past the window
      len = W - i;
      for (long long t = t0 + W; t < a.tokens; t += 32) {
        const unsigned m = __ballot_sync(0xffffffffu, t + lane >= a.tokens || kind_of(t + lane) != 0);
        const int n = m ? __ffs(m) - 1 : 32;
        len += n;
        if (n < 32) break;
      }
    }
    const long long slot = a.slots[t0 + i];
    const long long page = slot >> a.c.log2_page;
    const int place = (int)(slot & (P - 1));
    for (int hk = hk0; hk < hk1; ++hk, ++turn) {
    const int head = hk >> 1, which = hk & 1, vec = a.vec[which];
    uint8_t* codes = which ? a.c.v : a.c.k;
    const void* x = a.x[which];
    const long long st = a.st[which], sd = a.sd[which], xh = head * a.sh[which];
    float* sp = (which ? a.c.v_scale : a.c.k_scale) + page * a.c.heads + head;
    const float was = place ? *sp : 0.f;
    const long long row0 = (page * a.c.heads + head) << a.c.log2_page;

    KvPiece<ESZ> f[U];
    // Piece u of this warp, counted from token `from`: TPW tokens, nw warps apart.
    const long long at0 = (t0 + i + wv * TPW + sub) * st + xh, at1 = (long long)nw * TPW * st;
    const int first = wv * TPW, span = nw * TPW;
    auto load = [&](int from) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = from + first + u * span;
        if (j >= len) break;                      // (warp-uniform)
        if (j + sub < len) f[u].load(x, at0 + (from / span + u) * at1, sd, d0, a.dh, vec);
        else f[u].zero();
      }
    };
    float m = 0.f;
    for (int from = 0; from < len; from += U * span) {
      load(from);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (from + first + u * span >= len) break;
        m = f[u].amax(m, a.type);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (share) {                                  // (two buffers: the next turn's maxima cannot overtake this one's readers)
      if (lane == 0) s_max[turn & 1][warp] = m;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / GW), "n"(GW * 32) : "memory");
#pragma unroll
      for (int w = 0; w < GW; ++w) m = max_nan(m, s_max[turn & 1][warp / GW * GW + w]);
    }
    const float want = kv_scale_for<KIND>(m);
    const float now = (want <= was || was != was) ? was : want;   // not-a-number stays
    __syncwarp();
    if (lane == 0 && wv == 0) *sp = now;          // (everybody has read it)
    if (place && now > was) {                     // the older codes move to the new scale
      const float r = __fdiv_rn(was, now);
      uint32_t* row = reinterpret_cast<uint32_t*>(codes + row0 * DHP);
      for (int j = wv * 32 + lane; j < place * DHP / 4; j += nw * 32) {
        const uint32_t w = row[j];
        row[j] = kv_code4<KIND>(kv_value<KIND>(w & 0xffu) * r, kv_value<KIND>((w >> 8) & 0xffu) * r,
                                kv_value<KIND>((w >> 16) & 0xffu) * r, kv_value<KIND>(w >> 24) * r, 1.f, 1.f);
      }
    }
    const float inv = __fdiv_rn(1.0f, now);
    for (int from = 0; from < len; from += U * span) {
      if (len > U * span) load(from);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = from + first + u * span;
        if (j >= len) break;
        if (j + sub < len)
          *reinterpret_cast<uint2*>(codes + (row0 + place + j + sub) * DHP + d0) = f[u].template codes<KIND>(now, inv, a.type);
      }
    }
    }
  }
}

struct KvReadArgs {
  KvCache c;
  const long long* slots;
  void* out[2];                  // [n, heads, dh], contiguous
  long long n, num_slots;
  int type, dh;
};

// Value = code * scale in fp32, then rounded to the type; slots outside the cache read as 0.
// A lane takes 8 codes of a token and head, K and V alike, two pieces at a time.
// Bound: HBM; 65536 tokens, 16 heads of 64, e4m3 to fp16 88 us (403 MB, 71 %). The rest
// is the chain slot, codes and scale, values: warps wait for loads most of the time
// (8.8 stalled on them an issue), with 37 of them an SM and issue slots 58 % full.
template <int DHP, int KIND>
__global__ void __launch_bounds__(256) kv_read_kernel(KvReadArgs a) {
  pdl_wait_then_release();
  constexpr int LPT = DHP / 8;
  const bool vec = a.dh % 8 == 0;
  // Lanes of a token and head; (token, head) pairs by 32-bit division.
  const long long pairs = a.n * a.c.heads, step = (long long)gridDim.x * 256 / LPT;
  const int d0 = (threadIdx.x % LPT) * 8;
  if (d0 >= a.dh) return;
  for (long long th0 = ((long long)blockIdx.x * 256 + threadIdx.x) / LPT; th0 < pairs; th0 += 2 * step) {
    uint2 w[2][2];
    float s[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long th = th0 + u * step;
      w[u][0] = w[u][1] = make_uint2(0, 0);
      s[u][0] = s[u][1] = 0.f;
      if (th >= pairs) continue;
      const long long tok = pairs <= 0xffffffffLL ? (long long)((unsigned)th / (unsigned)a.c.heads) : th / a.c.heads;
      const int head = (int)(th - tok * a.c.heads);
      const long long slot = a.slots[tok];
      if (slot < 0 || slot >= a.num_slots) continue;
      const long long ph = (slot >> a.c.log2_page) * a.c.heads + head;
      const long long at = ((ph << a.c.log2_page) + (slot & (a.c.page - 1))) * DHP + d0;
      w[u][0] = *reinterpret_cast<const uint2*>(a.c.k + at);
      w[u][1] = *reinterpret_cast<const uint2*>(a.c.v + at);
      s[u][0] = a.c.k_scale[ph];
      s[u][1] = a.c.v_scale[ph];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long th = th0 + u * step;
      if (th >= pairs) break;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          f[k] = kv_value<KIND>(((k < 4 ? w[u][which].x : w[u][which].y) >> (8 * (k & 3))) & 0xffu) * s[u][which];
        const long long o = th * a.dh + d0;
        if (vec) {
          if (a.type == kElemF32) {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out[which]) + o);
            p[0] = make_float4(f[0], f[1], f[2], f[3]);
            p[1] = make_float4(f[4], f[5], f[6], f[7]);
          } else {
            *reinterpret_cast<uint4*>(static_cast<__half*>(a.out[which]) + o) =
                make_uint4(pack_elem2(f[0], f[1], a.type), pack_elem2(f[2], f[3], a.type),
                           pack_elem2(f[4], f[5], a.type), pack_elem2(f[6], f[7], a.type));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (d0 + k >= a.dh) break;
            if (a.type == kElemF32) static_cast<float*>(a.out[which])[o + k] = f[k];
            else if (a.type == kElemF16) static_cast<__half*>(a.out[which])[o + k] = __float2half_rn(f[k]);
            else static_cast<__nv_bfloat16*>(a.out[which])[o + k] = __float2bfloat16_rn(f[k]);
          }
        }
      }
    }
  }
}

}  // namespace b200l
