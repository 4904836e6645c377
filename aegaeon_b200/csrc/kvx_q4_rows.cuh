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

// Division of 32-bit numbers by a divisor known at launch (Granlund and
// Montgomery, "Division by invariant integers using multiplication").
struct Divisor {
  uint32_t d, m, s1, s2;
  __host__ static Divisor of(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && (uint64_t(1) << l) < d) ++l;
    const uint64_t m = ((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1;
    return Divisor{d, uint32_t(m), l < 1 ? l : 1u, l > 1 ? l - 1 : 0u};
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    const uint32_t t = __umulhi(m, n);
    return (t + ((n - t) >> s1)) >> s2;
  }
};

struct RowArgs {
  Cache cache;
  Rows rows[2];
  const int64_t* slots;
  uint32_t num_rows;   // tokens * kv_heads
  Divisor by_heads, by_block;
};

// Block of a slot and token in the block.
__device__ __forceinline__ int64_t block_of(const RowArgs& a, int64_t slot, int* within) {
  if (uint64_t(slot) < (uint64_t(1) << 32)) {
    const uint32_t block = a.by_block.quotient(uint32_t(slot));
    *within = int(uint32_t(slot) - block * a.by_block.d);
    return block;
  }
  *within = int(slot % a.cache.block_size);
  return slot / a.cache.block_size;
}

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
// Two neighbours at once, from the word that holds them.
__device__ __forceinline__ float2 to_float2(const __half* x) {
  __half2 h;
  __builtin_memcpy(&h, x, 4);
  return __half22float2(h);
}
__device__ __forceinline__ float2 to_float2(const __nv_bfloat16* x) {
  uint32_t w;
  __builtin_memcpy(&w, x, 4);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 to_float2(const float* x) { return make_float2(x[0], x[1]); }
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

// Two additions, or two fused multiply-adds, in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float max_abs(float m, float a, float b) {  // max(m, |a|, |b|)
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// The code next to a border, decided exactly: `c` is the nearest code or the one
// beside it.  d + e = x - zero without an error (two-sum), c * scale has at most
// 15 bits, and the difference of d to it, about scale / 2, is representable, as
// is its difference to scale / 2: only the last sum rounds, which keeps its sign.
__device__ __forceinline__ uint32_t settle(float x, float zero, float scale, uint32_t c) {
  const float d = x - zero, near = x - d;
  const float e = (x - (d + near)) + (near - zero);
  const float r = fmaf(-float(c), scale, d), half = 0.5f * scale;
  const float above = (r - half) + e, below = (r + half) + e;
  if (above > 0.f || (above == 0.f && (c & 1u))) return min(c + 1u, 15u);
  if (below < 0.f || (below == 0.f && (c & 1u))) return c ? c - 1u : 0u;
  return c;
}

// Codes of 16 values, two words of eight: rint((x - zero) / scale) in [0, 15],
// ties to even, in real arithmetic.
//
// q = (x - zero) * (1 / scale) carries the roundings of the difference and the
// product and the reciprocal's 2 ulp, below 16 * 4 * 2^-23 < 8e-6 in all.
// q + 1.5 * 2^23 is rounded once, to the nearest integer, which then stands in
// the sum's low bits.  The result can differ from the definition's only where
// what is left over is within 1e-5 of half a step; a thread that has such a value
// settles its 16 again (16-bit values meet exact ties often: about one in three
// thousand of them).  So does a row with clamped values, or whose zero is so far
// from 0 that its rounding to fp16 may move values beyond the codes' ends.
template <typename T>
__device__ __forceinline__ uint2 codes_of(const T (&x)[16], float zero, float scale,
                                          bool clamped) {
  constexpr float kMagic = 12582912.f;
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
  uint32_t w[2] = {0u, 0u};
  float far = 0.f;  // largest distance from a code's value
#pragma unroll
  for (int i = 14; i >= 0; i -= 2) {
    const float2 d = add2(to_float2(x + i), both(-zero));
    const float2 r = add2(mul2(d, both(inverse)), both(kMagic));
    const float2 left = fma2(add2(r, both(-kMagic)), both(-scale), d);
    far = max_abs(far, left.x, left.y);
    w[i / 8] = (w[i / 8] * 16u + __float_as_uint(r.y)) * 16u + __float_as_uint(r.x);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) w[h] -= 0x3F400000u;  // 0x4B400000 * 0x11111111
  // zero is off its value by at most 2^-11 |zero|, scale by 2^-11 of itself: below
  // this bound every quotient stays in (-1/2, 15 1/2).
  const bool beyond = clamped || fabsf(zero) > 900.f * scale || scale < 6.2e-5f;
  const float border = 0.49999f * scale;
  if (beyond || far > border) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = to_float(x[i]);
      if (clamped) y = fminf(fmaxf(y, -kLimit), kLimit);
      const uint32_t was = (w[i / 8] >> (4 * (i % 8))) & 15u;
      if (!beyond && fabsf(fmaf(-float(was), scale, y - zero)) <= border) continue;
      uint32_t c = was;
      if (beyond) c = uint32_t(fminf(fmaxf((y - zero) / scale, 0.f), 15.f) + 0.5f);
      w[i / 8] ^= (was ^ settle(y, zero, scale, c)) << (4 * (i % 8));
    }
  }
  return make_uint2(w[0], w[1]);
}

// Quantise.  D/16 lanes share a row, 16 elements each; every thread takes the
// K row and the V row of one (token, head), so that both loads are in flight.
// 8192 tokens of 32 heads in fp16 take 48 us, 3.5 TB/s (55% of the copy rate): 18
// instructions a value, which fill 71% of the issue slots, bound it, not the memory.
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kRowThreads) q4_write(const RowArgs a) {
  constexpr int kLanes = D / 16;
  const uint32_t row = blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool inside = row < a.num_rows;
  const uint32_t token = inside ? a.by_heads.quotient(row) : 0u;
  const int head = inside ? int(row - token * a.by_heads.d) : 0;
  const int64_t slot = inside ? a.slots[token] : -1;
  T x[2][16];
#pragma unroll
  for (int s = 0; s < 2; ++s) {  // whatever the slot, so that no load waits for it
    if (inside) {
      load16<T, kVec>(static_cast<const T*>(a.rows[s].base) + token * a.rows[s].token_stride +
                          head * a.rows[s].head_stride + lane * 16,
                      x[s]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[s][i] = from_float<T>(0.f);
    }
  }
  int within;
  const int64_t block = block_of(a, slot, &within);
  bool live = slot >= 0;
  if (live && block >= a.cache.num_blocks) {
    live = false;
    if (lane == 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
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
    const bool clamped = fmaxf(fabsf(lo), fabsf(hi)) > kLimit;
    lo = fminf(fmaxf(lo, -kLimit), kLimit);
    hi = fminf(fmaxf(hi, -kLimit), kLimit);
    const __half scale_h = __float2half_rn((hi - lo) / 15.f);
    const __half zero_h = __float2half_rn(lo);
    const float scale = __half2float(scale_h), zero = __half2float(zero_h);
    uint2 w = make_uint2(0u, 0u);
    if (finite && scale > 0.f) w = codes_of(x[s], zero, scale, clamped);
    if (live) {
      uint8_t* page = a.cache.pages[s] + head_offset(a.cache, block, head);
      *reinterpret_cast<uint2*>(page + within * (D / 2) + lane * 8) = w;
      if (lane == 0)
        *reinterpret_cast<__half2*>(page + a.cache.block_size * (D / 2) + within * 4) =
            finite ? __halves2half2(scale_h, zero_h)
                   : __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
    }
  }
}

// Read back: scale * code + zero, the product exact in 32 bits, one rounding
// of the sum and one to the output's type.  A negative slot gives zeros.
// Bound by memory: 65536 tokens of 8 heads to bf16 take 62 us, 5.5 TB/s (85% of the
// copy rate).
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kRowThreads) q4_read(const RowArgs a) {
  constexpr int kLanes = D / 16;
  const uint32_t row = blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (row >= a.num_rows) return;
  const uint32_t token = a.by_heads.quotient(row);
  const int head = int(row - token * a.by_heads.d);
  const int64_t slot = a.slots[token];
  int within;
  const int64_t block = block_of(a, slot, &within);
  bool live = slot >= 0;
  if (live && block >= a.cache.num_blocks) {
    live = false;
    if (lane == 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
  }
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
      // The code in the low bits of 2^23 is that number more.
      const uint32_t c = (((i < 8 ? w[s].x : w[s].y) >> (4 * (i % 8))) & 15u) | 0x4B000000u;
      x[i] = from_float<T>(fmaf(__uint_as_float(c) - 8388608.f, scale, zero));
    }
    store16<T, kVec>(static_cast<T*>(a.rows[s].base) + token * a.rows[s].token_stride +
                         head * a.rows[s].head_stride + lane * 16,
                     x);
  }
}

}  // namespace q4
}  // namespace kvx
