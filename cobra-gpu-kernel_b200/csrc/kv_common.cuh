// kv_common.cuh -- what the paged 8-bit key/value cache's kernels share.
//
// The cache of one layer is two arrays of codes [num_pages, Hkv, P, dhp]
// (int8, or e4m3 floats; dhp = head_dim rounded up to 32/64/128/256, the
// padding columns zero) and two arrays of fp32 scales [num_pages, Hkv]: the
// P tokens of a page share one scale per head, value = code * scale. A slot is
// page * P + place in page. Request r's pages in order are row r of the block
// table.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200l {

enum KvKind : int { kKvInt8 = 0, kKvE4M3 = 1 };
enum KvElem : int { kElemF32 = 0, kElemF16 = 1, kElemBF16 = 2 };   // = B200L_DTYPE_*

constexpr int kKernelKvDecode = 7, kKernelKvPrompt = 8;   // DevStatus::kernel

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  long long num_pages;
  int heads;       // Hkv
  int page;        // P: 16, 32, 64 or 128
  int log2_page;
};

// Four codes as two fp16 pairs, exactly. int8: code + 128 under the fp16
// exponent of 1024 is 1024 + 128 + code to the unit, and the difference to
// 1152 is exact. e4m3 is a subset of fp16.
template <int KIND>
__device__ __forceinline__ void codes4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == kKvInt8) {
    w ^= 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_elem2(float a, float b, int type) {
  if (type == kElemF16) return pack_half2(a, b);
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// The last r in [0, n) with cu[r] <= x (cu ascending, cu[0] = 0): where the
// owner of item x is looked up in a prefix sum. Owners without items are
// passed over, for their cu equals their successor's. One probe per lane and
// round, so a prefix sum of up to 1024 owners takes two round trips.
__device__ __forceinline__ int warp_find_owner(const int* cu, int n, long long x, int lane) {
  int lo = 0, hi = n;                 // cu[lo] <= x, and cu[hi] > x or hi == n
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;
    const bool le = at < hi && (long long)cu[at] <= x;
    const int k = __popc(__ballot_sync(0xffffffffu, le));   // probes pass in order
    const int nhi = lo + (k + 1) * step;
    lo += k * step;
    hi = nhi < hi ? nhi : hi;
  }
  return lo;
}

// The same by one thread, in shared memory.
__device__ __forceinline__ int find_owner(const int* cu, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace b200l
