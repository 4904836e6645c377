// Kernels of the 4-bit paged cache that move rows: quantise rows into their
// slots, and read rows back.
//
// A page holds one block of one tensor (K or V), kv heads outermost:
//   [kv_heads][ block_size * D/2 bytes of codes | block_size * (fp16 scale, fp16 zero) ]
// A value is scale * code + zero, one (scale, zero) for each token and head.
// The codes of a token are D/2 consecutive bytes, even dimension in the low
// nibble.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kvx {
namespace q4 {

constexpr int kBf16 = 0, kFp16 = 1, kFp32 = 2;  // the `dtype` arguments (kvx.h)
constexpr int kRowThreads = 256;
constexpr float kLimit = 65504.f;  // largest finite fp16

// Set by kernels that met a slot, block or length outside its buffer (they
// skip it); read and cleared through kvx_device_status.
static __device__ int g_q4_status;

// Geometry of one cache (a K and a V tensor of one shape).
struct Cache {
  uint8_t* pages[2];   // K, V
  int64_t stride;      // bytes from one page to the next, the same for both
  int64_t num_blocks;
  int kv_heads;
  int block_size;      // tokens of a page, a multiple of 16
  int head_bytes;      // block_size * (D/2 + 4)
};

// Rows [token][head] of one tensor; strides in elements.
struct Rows {
  void* base;
  int64_t token_stride;
  int64_t head_stride;
};

struct RowArgs {
  Cache cache;
  Rows rows[2];
  const int64_t* slots;
  int64_t num_rows;    // tokens * kv_heads
};

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <>
struct Pair<__half> {
  using type = __half2;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ float from_float<float>(float x) {
  return x;
}

// 16 consecutive elements of a row.  kVec: base and strides are multiples of
// 16 bytes, so 16-byte accesses serve; otherwise one element at a time.
template <typename T, bool kVec>
__device__ __forceinline__ void load16(const T* p, T (&x)[16]) {
  if constexpr (kVec) {
    constexpr int n = sizeof(T);  // 16 elements are n 16-byte words
    uint4 w[n];
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    __builtin_memcpy(x, w, sizeof(x));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = p[i];
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store16(T* p, const T (&x)[16]) {
  if constexpr (kVec) {
    constexpr int n = sizeof(T);
    uint4 w[n];
    __builtin_memcpy(w, x, sizeof(x));
#pragma unroll
    for (int i = 0; i < n; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = x[i];
  }
}

// One head's part of a page.
__device__ __forceinline__ int64_t head_offset(const Cache& c, int64_t block, int head) {
  return block * c.stride + int64_t(head) * c.head_bytes;
}

// Code of x in [0, 15]: rint((x - zero) / scale), ties to even, in real
// arithmetic.  The product with the reciprocal is off by at most 3 * 2^-24 of
// a quotient below 16 (three roundings), under 3e-6; only where the quotient
// lies within 1e-5 of a border between two codes does the 64-bit division
// decide, which the 16-bit types' differences enter exactly.
__device__ __forceinline__ uint32_t code_of(float x, float zero, float scale, float inv) {
  const float t = fminf(fmaxf((x - zero) * inv, 0.f), 15.f);
  const float r = t + 12582912.f;  // 1.5 * 2^23: the sum's low bits are rint(t)
  uint32_t c = __float_as_uint(r) & 15u;
  if (fabsf(t - (r - 12582912.f)) > 0.49999f)
    c = uint32_t(fmin(fmax(rint((double(x) - double(zero)) / double(scale)), 0.0), 15.0));
  return c;
}

// Quantise.  D/16 lanes share a row, 16 elements each; every thread takes the
// K row and the V row of one (token, head).
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kRowThreads) q4_write(const RowArgs a) {
  constexpr int kLanes = D / 16;
  const int64_t row = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool inside = row < a.num_rows;
  const int64_t token = inside ? row / a.cache.kv_heads : 0;
  const int head = inside ? int(row % a.cache.kv_heads) : 0;
  const int64_t slot = inside ? a.slots[token] : -1;
  const int64_t block = slot / a.cache.block_size;
  bool live = inside && slot >= 0;
  if (live && block >= a.cache.num_blocks) {
    live = false;
    if (lane == 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
  }
  const int within = int(slot % a.cache.block_size);
  T x[2][16];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (live) {
      load16<T, kVec>(static_cast<const T*>(a.rows[s].base) + token * a.rows[s].token_stride +
                          head * a.rows[s].head_stride + lane * 16,
                      x[s]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[s][i] = from_float<T>(0.f);
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float lo, hi;
    if constexpr (sizeof(T) == 2) {
      // Minimum and maximum in the input's own type (exact), NaN kept.
      using P = typename Pair<T>::type;
      P p[8];
      __builtin_memcpy(p, x[s], sizeof(p));
      P mn = p[0], mx = p[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        mn = __hmin2_nan(mn, p[i]);
        mx = __hmax2_nan(mx, p[i]);
      }
      lo = min_nan(to_float(mn.x), to_float(mn.y));
      hi = max_nan(to_float(mx.x), to_float(mx.y));
    } else {
      lo = hi = to_float(x[s][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) {
        lo = min_nan(lo, to_float(x[s][i]));
        hi = max_nan(hi, to_float(x[s][i]));
      }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
      lo = min_nan(lo, __shfl_xor_sync(~0u, lo, d));
      hi = max_nan(hi, __shfl_xor_sync(~0u, hi, d));
    }
    // A row with a NaN or an infinity reads back as NaN: it is marked, not hidden.
    const bool finite = fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f;
    lo = fminf(fmaxf(lo, -kLimit), kLimit);
    hi = fminf(fmaxf(hi, -kLimit), kLimit);
    const __half scale_h = __float2half_rn((hi - lo) / 15.f);
    const __half zero_h = __float2half_rn(lo);
    const float scale = __half2float(scale_h), zero = __half2float(zero_h);
    uint32_t w[2] = {0u, 0u};
    if (finite && scale > 0.f) {
      const float inv = 1.f / scale;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        w[i / 8] |= code_of(to_float(x[s][i]), zero, scale, inv) << (4 * (i % 8));
    }
    if (live) {
      uint8_t* page = a.cache.pages[s] + head_offset(a.cache, block, head);
      *reinterpret_cast<uint2*>(page + within * (D / 2) + lane * 8) = make_uint2(w[0], w[1]);
      if (lane == 0)
        *reinterpret_cast<__half2*>(page + a.cache.block_size * (D / 2) + within * 4) =
            finite ? __halves2half2(scale_h, zero_h)
                   : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
    }
  }
}

// Read back: scale * code + zero, the product exact in 32 bits, one rounding
// of the sum and one to the output's type.  A negative slot gives zeros.
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kRowThreads) q4_read(const RowArgs a) {
  constexpr int kLanes = D / 16;
  const int64_t row = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (row >= a.num_rows) return;
  const int64_t token = row / a.cache.kv_heads;
  const int head = int(row % a.cache.kv_heads);
  const int64_t slot = a.slots[token];
  const int64_t block = slot / a.cache.block_size;
  bool live = slot >= 0;
  if (live && block >= a.cache.num_blocks) {
    live = false;
    if (lane == 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
  }
  const int within = int(slot % a.cache.block_size);
  uint2 w[2] = {};
  __half2 p[2] = {};
  if (live) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* page = a.cache.pages[s] + head_offset(a.cache, block, head);
      w[s] = *reinterpret_cast<const uint2*>(page + within * (D / 2) + lane * 8);
      p[s] = *reinterpret_cast<const __half2*>(page + a.cache.block_size * (D / 2) + within * 4);
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float scale = __half2float(p[s].x), zero = __half2float(p[s].y);
    T x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t c = ((i < 8 ? w[s].x : w[s].y) >> (4 * (i % 8))) & 15u;
      x[i] = from_float<T>(fmaf(float(c), scale, zero));
    }
    store16<T, kVec>(static_cast<T*>(a.rows[s].base) + token * a.rows[s].token_stride +
                         head * a.rows[s].head_stride + lane * 16,
                     x);
  }
}

}  // namespace q4
}  // namespace kvx
