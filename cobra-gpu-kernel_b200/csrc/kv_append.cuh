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
// each page's new tokens have to be one run. A block takes the runs that begin
// in its window of W tokens, for one head of K or V:
//   1. max |x| of every token of those runs (lanes share a token, 8 dims each),
//   2. a warp per run: the page's scale, and the older codes if it grew,
//   3. codes of every token.
// The second look at x comes from L1/L2: a window is W tokens of one head.
//
// Bound: HBM, 2 (or 4) bytes read and 1 written per value; a decode step is a
// few microseconds of latency, so W shrinks to a token per warp there.
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
  int type, dh, window;
};

constexpr int kKvAppendThreads = 256;
constexpr int kKvAppendMaxTokens = 64 + 128;   // window + the longest run

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

// Code of x at scale s; s == 0 only where every x is 0.
template <int KIND>
__device__ __forceinline__ uint32_t kv_code(float x, float s, float inv) {
  if constexpr (KIND == kKvInt8) {
    if (!(s > 0.f)) return 0;
    const int c = __float2int_rn(__fdiv_rn(x, s));
    return (uint32_t)max(-127, min(127, c)) & 0xffu;
  } else {
    if (!(s > 0.f)) return 0;
    return __nv_cvt_float_to_fp8(x * inv, __NV_SATFINITE, __NV_E4M3);   // s is a power of two: exact
  }
}

template <int KIND>
__device__ __forceinline__ float kv_value(uint32_t c) {
  if constexpr (KIND == kKvInt8) return (float)(signed char)c;
  __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

// Eight dims [d0, d0 + 8) of one token and head as fp32, zero past dh.
__device__ __forceinline__ void kv_load8(const void* x, long long base, long long sd, int d0, int dh, int type, int vec,
                                         float (&f)[8]) {
  if (vec && d0 + 8 <= dh) {
    if (type == kElemF32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + base + d0);
      const float4 a = p[0], b = p[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __half*>(x) + base + d0);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 p;
        if (type == kElemF16) p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = d0 + i < dh ? load_elem(x, base + (d0 + i) * sd, type) : 0.f;
}

template <int DHP, int KIND>
__global__ void __launch_bounds__(kKvAppendThreads) kv_append_kernel(KvAppendArgs a) {
  pdl_wait_then_release();
  constexpr int LPT = DHP / 8;                    // lanes that share a token
  constexpr int TPW = 32 / LPT;                   // tokens of a warp at a time
  constexpr int NW = kKvAppendThreads / 32;
  __shared__ long long s_slot[kKvAppendMaxTokens];
  __shared__ float s_val[kKvAppendMaxTokens];     // max |x|, then the scale of the token's run
  __shared__ unsigned char s_lead[kKvAppendMaxTokens];
  __shared__ int s_end;                           // tokens from the window's start to its last run's end
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = a.c.page, head = blockIdx.y, which = blockIdx.z;
  const long long t0 = (long long)blockIdx.x * a.window;
  const int W = (int)min((long long)a.window, a.tokens - t0);
  const int reach = (int)min((long long)W + P - 1, a.tokens - t0);
  uint8_t* codes = which ? a.c.v : a.c.k;
  float* scales = which ? a.c.v_scale : a.c.k_scale;
  const void* x = a.x[which];
  const long long st = a.st[which], sd = a.sd[which], xh = head * a.sh[which];

  // Slots of the window and of the tokens that its last run may reach; whether
  // a token leads a run, or goes on the one before it (2: in no run).
  if (tid == 0) s_end = reach;
  for (int i = tid; i < reach; i += kKvAppendThreads) {
    const long long s = a.slots[t0 + i];
    const long long before = t0 + i > 0 ? a.slots[t0 + i - 1] : -1;
    const bool in = s >= 0 && s < a.num_slots;
    s_slot[i] = s;
    s_lead[i] = !in ? 2 : (before < 0 || s != before + 1 || (s & (P - 1)) == 0) ? 1 : 0;
  }
  __syncthreads();
  // Tokens [begin, end): the runs led from inside the window.
  int begin = 0;
  while (begin < W && s_lead[begin] != 1) ++begin;
  if (begin == W) return;
  // The last of them may go on past the window, to the first token that does not.
  for (int i = W + tid; i < reach; i += kKvAppendThreads)
    if (s_lead[i] != 0) atomicMin(&s_end, i);
  __syncthreads();
  const int end = s_end;

  const int sub = lane / LPT, d0 = (lane % LPT) * 8;
  for (int i0 = begin + warp * TPW; i0 < end; i0 += NW * TPW) {
    const int i = i0 + sub;
    float m = 0.f;
    if (i < end && s_lead[i] != 2) {
      float f[8];
      kv_load8(x, (t0 + i) * st + xh, sd, d0, a.dh, a.type, a.vec[which], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = (fabsf(f[k]) <= m || m != m) ? m : fabsf(f[k]);   // not-a-number stays
    }
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, m, o);
      m = (y <= m || m != m) ? m : y;
    }
    if (i < end && d0 == 0) s_val[i] = m;
  }
  __syncthreads();

  for (int i = begin + warp; i < end; i += NW) {
    if (s_lead[i] != 1) continue;                 // (warp-uniform)
    int len = 1;
    while (i + len < end && s_lead[i + len] == 0) ++len;
    float m = 0.f;
    for (int j = lane; j < len; j += 32) {
      const float y = s_val[i + j];
      m = (y <= m || m != m) ? m : y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, m, o);
      m = (y <= m || m != m) ? m : y;
    }
    const long long page = s_slot[i] >> a.c.log2_page;
    const int place = (int)(s_slot[i] & (P - 1));
    float* sp = scales + page * a.c.heads + head;
    const float was = place ? *sp : 0.f;
    const float want = kv_scale_for<KIND>(m);
    const float now = (want <= was || was != was) ? was : want;   // not-a-number stays
    __syncwarp();
    if (lane == 0) *sp = now;
    for (int j = lane; j < len; j += 32) s_val[i + j] = now;
    if (place && now > was) {                     // the older codes move to the new scale
      const float f = __fdiv_rn(was, now);
      uint32_t* row = reinterpret_cast<uint32_t*>(codes + ((page * a.c.heads + head) << a.c.log2_page) * DHP);
      for (int j = lane; j < place * DHP / 4; j += 32) {
        const uint32_t w = row[j];
        uint32_t o = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) o |= kv_code<KIND>(kv_value<KIND>((w >> (8 * k)) & 0xffu) * f, 1.f, 1.f) << (8 * k);
        row[j] = o;
      }
    }
  }
  __syncthreads();

  for (int i = begin + warp * TPW + sub; i < end; i += NW * TPW) {
    if (s_lead[i] == 2) continue;
    float f[8];
    kv_load8(x, (t0 + i) * st + xh, sd, d0, a.dh, a.type, a.vec[which], f);
    const float s = s_val[i], inv = KIND == kKvE4M3 ? __fdiv_rn(1.0f, s) : 0.f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k >> 2] |= kv_code<KIND>(f[k], s, inv) << (8 * (k & 3));
    const long long slot = s_slot[i];
    const long long row = (((slot >> a.c.log2_page) * a.c.heads + head) << a.c.log2_page) + (slot & (P - 1));
    *reinterpret_cast<uint2*>(codes + row * DHP + d0) = make_uint2(w[0], w[1]);
  }
}

struct KvReadArgs {
  KvCache c;
  const long long* slots;
  void* out[2];                  // [n, heads, dh], contiguous
  long long n, num_slots;
  int type, dh;
};

// Value = code * scale, rounded once; slots outside the cache read as 0.
// A lane takes 8 codes of a token and head, K and V alike. Bound: HBM.
template <int DHP, int KIND>
__global__ void __launch_bounds__(256) kv_read_kernel(KvReadArgs a) {
  pdl_wait_then_release();
  constexpr int LPT = DHP / 8;
  const long long items = a.n * a.c.heads * LPT;
  const bool vec = a.dh % 8 == 0;
  for (long long it = (long long)blockIdx.x * 256 + threadIdx.x; it < items; it += (long long)gridDim.x * 256) {
    const int d0 = (int)(it % LPT) * 8;
    const long long th = it / LPT;
    const int head = (int)(th % a.c.heads);
    if (d0 >= a.dh) continue;
    const long long slot = a.slots[th / a.c.heads];
    const bool in = slot >= 0 && slot < a.num_slots;
    const long long ph = in ? (slot >> a.c.log2_page) * a.c.heads + head : 0;
    const long long row = (ph << a.c.log2_page) + (in ? slot & (a.c.page - 1) : 0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint2 w = in ? *reinterpret_cast<const uint2*>((which ? a.c.v : a.c.k) + row * DHP + d0) : make_uint2(0, 0);
      const float s = in ? (which ? a.c.v_scale : a.c.k_scale)[ph] : 0.f;
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = kv_value<KIND>(((k < 4 ? w.x : w.y) >> (8 * (k & 3))) & 0xffu) * s;
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

}  // namespace b200l
