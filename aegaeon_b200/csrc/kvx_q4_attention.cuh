// Attention over the 4-bit paged cache.
//
// Mathematics.  With k_j = s_j c_j + z_j (codes c_j, one scale and zero for each
// token and kv head),
//   q . k_j         = s_j (q . c_j) + z_j sum(q)
//   sum_j p_j v_j   = sum_j (p_j s'_j) c'_j + sum_j p_j z'_j
// so the matrix instructions take the codes themselves and the scales join in
// 32 bits: on the scores for K, on the probabilities for V.  The codes need no
// conversion: four bits in the low end of an fp16 are the subnormal number
// code * 2^-24 (and 2^-20 one nibble further up), exact in the matrix
// instruction's products; the powers of two leave with the epilogue.
//
// The running maximum is kept in powers of two and follows only when a score
// passes it by 2^8, so that most tiles neither reduce it nor rescale.
#pragma once

#include "kvx_q4_rows.cuh"

namespace kvx {
namespace q4 {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;       // steps in flight or in use, per warp
constexpr int kNoWindow = 1 << 30;
// Fewest 16-token units a CTA takes: four for each warp, a whole step.
constexpr int kMinUnits = 4 * kWarps;
// What an item (a tile of query rows with one kv head) costs besides its units,
// in units: its queries, its first block ids and the join of the warps.
constexpr int kItemUnits = 16;

struct AttnArgs {
  Cache cache;
  const void* query;
  int64_t q_token, q_head;  // strides in elements
  void* out;
  int64_t o_token, o_head;
  float* lse;               // [tokens][heads] or null
  const int32_t* tables;
  int64_t table_stride;
  int table_width;
  const int32_t* lens;
  const int32_t* starts;    // null: every sequence has `queries` query tokens
  int batch;
  int queries;
  int num_tokens;
  int group;                // query heads of a kv head
  float scale_log2;         // |softmax scale| * log2(e)
  float sign;               // of the softmax scale
  int window;               // kNoWindow: none
  int sinks;                // 0 without a window
  int upp;                  // 16-token units of a page
  int upp_shift;            // log2(upp), -1 when it is no power of two
  int q_vec, o_vec;         // 16-byte accesses serve for query / out
  float* part_o;            // [2 * grid][rows][D]
  float2* part_ml;          // [2 * grid][rows] (running maximum, sum)
};

struct Seq {
  int start;  // first query token
  int count;  // query tokens
  int len;    // tokens in the cache
};

__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int b) {
  Seq s;
  if (a.starts) {
    s.start = min(max(a.starts[b], 0), a.num_tokens);
    s.count = min(max(a.starts[b + 1], s.start), a.num_tokens) - s.start;
  } else {
    s.start = b * a.queries;
    s.count = a.queries;
  }
  const int64_t room = int64_t(a.table_width) * a.cache.block_size;
  const int len = a.lens[b];
  s.len = int(min(int64_t(max(len, 0)), room));
  if (int64_t(len) > room) atomicExch(&g_q4_status, 4 /* KVX_ERR_EXTENT */);
  return s;
}

// The part of a sequence's cache that a tile of query rows sees: units
// [0, units), of which those from `sink_units` on are `gap` units further up.
struct Span {
  int p_lo, p_hi;  // positions of the tile's first and last row
  int units, sink_units, gap;
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, const Seq& s, int row0, int rows) {
  Span v;
  v.p_lo = s.len - s.count + row0 / a.group;
  v.p_hi = s.len - s.count + (row0 + rows - 1) / a.group;
  v.units = v.sink_units = v.gap = 0;
  if (rows <= 0 || v.p_hi < 0) return v;
  const int all = v.p_hi / 16 + 1;
  const int from = max(v.p_lo - a.window + 1, 0) / 16;
  v.sink_units = min((a.sinks + 15) / 16, all);
  v.gap = max(from - v.sink_units, 0);
  v.units = all - v.gap;
  return v;
}

// Work of all sequences, and the place of a position in its running sum.  Every
// thread takes a run of sequences; `at` maps the total to the position.
struct Place {
  int index;       // the sequence whose part holds the position, n when none does
  int64_t before;  // work of the sequences before it
};

template <class F, class G>
__device__ __forceinline__ int64_t block_locate(F f, int n, G at, int64_t* sm, Place* found,
                                                Place* place) {
  const int run = (n + kThreads - 1) / kThreads, first = threadIdx.x * run;
  const int last = min(first + run, n);
  int64_t own = 0;
  for (int i = first; i < last; ++i) own += f(i);
  int64_t v = own;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t u = __shfl_up_sync(~0u, v, d);
    if (threadIdx.x % 32 >= d) v += u;
  }
  if (threadIdx.x % 32 == 31) sm[threadIdx.x / 32] = v;
  if (threadIdx.x == 0) *found = Place{n, 0};
  __syncthreads();
  int64_t before = v - own, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < int(threadIdx.x / 32)) before += sm[w];
    total += sm[w];
  }
  const int64_t pos = at(total);
  if (pos >= before && pos < before + own) {
    int i = first;
    for (int64_t c = run > 1 ? f(i) : own; pos >= before + c; c = f(i)) {
      before += c;
      ++i;
    }
    *found = Place{i, before};
  }
  __syncthreads();
  *place = *found;
  return total;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// 16 bytes to shared memory; n = 0: nothing is read, zeros are written.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}

constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kEven = 0x000f000fu;  // nibbles 0 and 4: code * 2^-24 in each half
constexpr uint32_t kOdd = 0x00f000f0u;   // nibbles 1 and 5: code * 2^-20

template <int D>
struct Shape {
  static constexpr int kUnit = 8 * D;           // bytes of codes of 16 tokens
  // Units of a step, which a warp takes at a time.  With four, what a step costs
  // besides its units (addresses, the vote on the reference point) is a tenth.
  static constexpr int kUnits = D == 256 ? 2 : 4;
  static constexpr int kParams = kUnits * 64;   // (scale, zero) of the units' tokens, one tensor
  static constexpr int kStage = kUnits * 2 * kUnit + 2 * kParams;
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kRing = kWarps * kWarpBytes;
  static constexpr int kJoin = kWarps * 8 * (D + 4) * 4;
  static constexpr int kShared = kRing > kJoin ? kRing : kJoin;
  static constexpr int kKeyWords = D / 32;      // code words of a thread for one token of K
};

// First dimension of code word w of quad lane j in a K row.  At D = 256 the
// two halves of a row are two 16-byte reads.
template <int D>
__device__ __forceinline__ int key_dim(int j, int w) {
  return D == 256 ? (w / 4) * 128 + 32 * j + 8 * (w % 4) : (D / 4) * j + 8 * w;
}

// Rows of one tile of queries as the CTA keeps them.
template <int D, int NT>
struct TileShared {
  uint2 q[NT][D / 16][32];  // B fragments of the queries, as mma reads them
  float factor[NT * 8];     // |scale| * log2(e) and the powers of two taken out
  float sum[NT * 8];        // sum(q) in the unit of the products with the codes
  int pos[NT * 8];          // position in the sequence, -1 for rows that are none
  float m[kWarps][NT * 8];
  float l[kWarps][NT * 8];
  int64_t scan[kWarps];
  Place place;
};

// Query rows of a tile into B fragments.  A row is scaled by a power of two so
// that its largest element lies in [2^14, 2^15): every 16-bit float within
// 2^-28 of it stays exact in fp16, whatever the row's range.
template <typename T, int D, int NT>
__device__ __forceinline__ void load_queries(const AttnArgs& a, const Seq& s, int row0, int rows,
                                             int head, TileShared<D, NT>& sh) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  static_assert(NT <= kWarps, "a warp for each eight rows");
  if (warp >= NT) return;
  const int r = warp * 8 + g;
  const bool real = r < rows;
  constexpr int kW = Shape<D>::kKeyWords;
  float x[kW][8];
  const T* base = static_cast<const T*>(a.query);
  int pos = -1;
  if (real) {
    const int token = (row0 + r) / a.group, h = (row0 + r) % a.group;
    pos = s.len - s.count + token;
    base += int64_t(s.start + token) * a.q_token + int64_t(head * a.group + h) * a.q_head;
  }
  float top = 0.f, sum = 0.f;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    const T* p = base + key_dim<D>(j, w);
    T v[8];
    if (!real) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from_float<T>(0.f);
    } else if (a.q_vec) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      __builtin_memcpy(v, &u, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[w][i] = to_float(v[i]);
      top = fmaxf(top, fabsf(x[w][i]));
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  // 2^(14 - exponent of top); bounded so that both it and its inverse are normal.
  const int e = min(max(int(__float_as_uint(top) >> 23), 20), 250);
  float up = top > 0.f ? __uint_as_float(uint32_t(min(127 + 14 + 127 - e, 240)) << 23) : 1.f;
  const float factor = a.scale_log2 * 16777216.f / up;
  up *= a.sign;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = (i % 2) ? up * 0.0625f : up;  // odd nibbles are 16 times as large
      const __half2 h = __floats2half2_rn(x[w][i] * u, x[w][i + 4] * u);
      sum += x[w][i] * up + x[w][i + 4] * up;
      __builtin_memcpy(&f[i], &h, 4);
    }
    sh.q[warp][2 * w][lane] = make_uint2(f[0], f[1]);
    sh.q[warp][2 * w + 1][lane] = make_uint2(f[2], f[3]);
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) sum += __shfl_xor_sync(~0u, sum, d);
  if (j == 0) {
    sh.factor[r] = fmaxf(factor, 1e-37f);  // never 0: hidden scores are -inf
    sh.sum[r] = sum * 5.9604644775390625e-8f;
    sh.pos[r] = pos;
  }
}

// One warp's state over the units that it takes.
template <int D, int NT>
struct WarpState {
  float o[NT][D / 16][4];  // sum of p * s * C * code, dimensions as in value_dim()
  float ps[NT][4];         // sum of the same weights as the matrix instruction saw them
  float2 m[NT], l[NT];     // minus the reference point, sum of the weights, by column
  float2 limit[NT];        // raw score that moves the reference point
  float z[NT][2];          // sum of p * (zero + 7.5 scale)
  float c;                 // C: power of two on the V scales, so that weights suit fp16
};

template <int kOffset>
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a), "n"(kOffset));
  return v;
}
template <int kOffset>
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(a), "n"(kOffset));
  return v;
}
template <int kOffset>
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(a), "n"(kOffset));
  return v;
}
__device__ __forceinline__ float2 half2_at(uint32_t x) {
  __half2 h;
  __builtin_memcpy(&h, &x, 4);
  return __half22float2(h);
}
// Shared-memory addresses of a lane's parts of a stage (the stage's base in).
struct LaneAddress {
  uint32_t k;       // its 16 bytes (D = 64: 8) of K row g
  uint32_t k_far;   // D = 256: those of the row's other half
  uint32_t v0, v1;  // its bytes of V rows 2j and 2j + 1
  uint32_t p;       // (scale, zero) of token g
  __device__ __forceinline__ LaneAddress operator+(uint32_t x) const {
    return LaneAddress{k + x, k_far + x, v0 + x, v1 + x, p + x};
  }
};

template <int D>
__device__ __forceinline__ LaneAddress lane_address(uint32_t base, int g, int j) {
  LaneAddress a;
  const uint32_t values = base + Shape<D>::kUnits * Shape<D>::kUnit;
  const uint32_t swizzle = 32u * (D == 64 ? (j >> 1) & 1 : j);
  const uint32_t v = uint32_t(D * j + (D / 16) * g) ^ swizzle;  // row 2j has D/2 bytes
  a.v0 = values + v;
  a.v1 = values + (v ^ (D / 2));
  a.k = base + (D / 2) * g + (D == 256 ? 16 * (j ^ (4 * (g & 1))) : (D / 8) * j);
  a.k_far = D == 256 ? base + 128 * g + (16 * (j ^ (4 * (g & 1))) ^ 64) : 0u;
  a.p = base + 2 * Shape<D>::kUnits * Shape<D>::kUnit + 4 * g;
  return a;
}

// K words of row g + 8 * kHigh of unit kUnitAt.
template <int D, int kUnitAt, int kHigh>
__device__ __forceinline__ void key_words(const LaneAddress& a, uint32_t (&w)[D / 32]) {
  constexpr int at = kUnitAt * Shape<D>::kUnit + kHigh * 4 * D;
  if constexpr (D == 64) {
    const uint2 v = lds64<at>(a.k);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = lds128<at>(a.k);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    if constexpr (D == 256) {
      const uint4 u = lds128<at>(a.k_far);
      w[4] = u.x, w[5] = u.y, w[6] = u.z, w[7] = u.w;
    }
  }
}

// V words of rows 2j + kOdd + 8 * kHigh.
template <int D, int kUnitAt, int kHigh>
__device__ __forceinline__ void value_words(uint32_t a, uint32_t (&w)[D / 64]) {
  constexpr int at = kUnitAt * Shape<D>::kUnit + kHigh * 4 * D;
  if constexpr (D == 64) {
    w[0] = lds32<at>(a);
  } else if constexpr (D == 128) {
    const uint2 v = lds64<at>(a);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = lds128<at>(a);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}

// q . c of one unit's 16 tokens with the tile's rows.
template <int D, int NT, int U>
__device__ __forceinline__ void unit_scores(const LaneAddress& at, const TileShared<D, NT>& sh,
                                            const uint2* qreg, float (&x)[NT][4]) {
  constexpr int kW = D / 32;
  uint32_t lo[kW], hi[kW];
  key_words<D, U, 0>(at, lo);
  key_words<D, U, 1>(at, hi);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[n][i] = 0.f;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t r0 = h ? lo[w] >> 8 : lo[w], r1 = h ? hi[w] >> 8 : hi[w];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint2 q = NT == 1 ? qreg[2 * w + h] : sh.q[n][2 * w + h][threadIdx.x % 32];
        mma(x[n], r0 & kEven, r1 & kEven, r0 & kOdd, r1 & kOdd, q.x, q.y);
      }
    }
  }
}

// Adds one unit's weights times its codes.
template <int D, int NT, int U>
__device__ __forceinline__ void unit_values(const LaneAddress& at, const uint32_t (&b)[NT][2],
                                            WarpState<D, NT>& st) {
  constexpr int kW = D / 64;
  uint32_t w0[kW], w1[kW], w2[kW], w3[kW];
  value_words<D, U, 0>(at.v0, w0);
  value_words<D, U, 0>(at.v1, w1);
  value_words<D, U, 1>(at.v0, w2);
  value_words<D, U, 1>(at.v1, w3);
#pragma unroll
  for (int w = 0; w < kW; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // Byte e of tokens 2j and 2j + 1, each in the low end of a half.
      const uint32_t select = 0x0400u + 0x0101u * e;
      const uint32_t p = __byte_perm(w0[w], w1[w], select), q = __byte_perm(w2[w], w3[w], select);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        mma(st.o[n][4 * w + e], p & kEven, p & kOdd, q & kEven, q & kOdd, b[n][0], b[n][1]);
    }
#pragma unroll
  for (int n = 0; n < NT; ++n)
    mma(st.ps[n], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, b[n][0], b[n][1]);
}

// What a thread keeps of the tile's rows (its columns 2j, 2j + 1 of each eight).
template <int NT>
struct Columns {
  float2 factor[NT];  // on the raw score: scale * log2(e) and the powers of two
  float2 sum[NT];     // sum(q), in the raw score's unit
  int pos[NT][2];
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// f(Index<0>), ..., f(Index<N - 1>): an index known at compile time.
template <int I>
struct Index {
  static constexpr int value = I;
};
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(Index<N - 1>{});
  }
}

// kAb units from unit U of the stage on: scores, softmax, products.  `number`
// gives the units' numbers in the sequence, -1 for one that is not there.
template <int D, int NT, int U, int kAb, bool kMasked>
__device__ __forceinline__ void attend_units(const AttnArgs& a, const TileShared<D, NT>& sh,
                                             const uint2* qreg, const LaneAddress& at,
                                             const int* number, const Columns<NT>& col,
                                             const Span& v, WarpState<D, NT>& st) {
  const int lane = threadIdx.x % 32, g = lane / 4;
  float x[kAb][NT][4];
  // (scale, zero) of tokens g and g + 8 of each unit: K, then V.
  uint32_t kp[kAb][2], vp[kAb][2];
  each<kAb>([&](auto index) {
    constexpr int u = decltype(index)::value, at_u = 64 * (U + u);
    kp[u][0] = lds32<at_u>(at.p), kp[u][1] = lds32<at_u + 32>(at.p);
    vp[u][0] = lds32<Shape<D>::kParams + at_u>(at.p);
    vp[u][1] = lds32<Shape<D>::kParams + at_u + 32>(at.p);
    unit_scores<D, NT, U + u>(at, sh, qreg, x[u]);
  });
  float vs[kAb][2], vz[kAb][2], most = 0.f;
#pragma unroll
  for (int u = 0; u < kAb; ++u) {
    float part[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 k = half2_at(kp[u][r]), w = half2_at(vp[u][r]);
      vs[u][r] = part[r] = w.x;
      vz[u][r] = fmaf(7.5f, w.x, w.y);
      const int unit = kMasked ? number[u] : 0, t = unit * 16 + g + 8 * r;
      // Only of tokens that some row sees: what lies behind a sequence may be anything.
      if (kMasked && !(unit >= 0 && t <= v.p_hi && (t > v.p_lo - a.window || t < a.sinks)))
        part[r] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float& y = x[u][n][2 * r + c];
          y = fmaf(k.x, y, k.y * (c ? col.sum[n].y : col.sum[n].x));
          if constexpr (kMasked) {
            const int p = col.pos[n][c];
            const bool seen = unit >= 0 && t <= p && (t > p - a.window || t < a.sinks);
            y = seen ? y : kNegInf;
          }
        }
    }
    most = max_abs(most, part[0], part[1]);
  }
  // Move the reference point where a score passes it by 2^8, or the weights
  // would leave fp16.  The factors are positive, so raw scores have the order.
  float top[NT][2];
  bool move = !(most * st.c <= 64.f);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      top[n][c] = fmaxf(x[0][n][c], x[0][n][2 + c]);
#pragma unroll
      for (int u = 1; u < kAb; ++u) top[n][c] = max3(top[n][c], x[u][n][c], x[u][n][2 + c]);
    }
    move |= top[n][0] > st.limit[n].x || top[n][1] > st.limit[n].y;
  }
  if (__any_sync(~0u, move)) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    float ratio = 1.f;
    if (st.c == 0.f || !(most * st.c <= 64.f)) {
      // most * C in [32, 64)
      const uint32_t e = __float_as_uint(most) >> 23;
      const float c = most > 0.f ? __uint_as_float((259u - e) << 23) : 16777216.f;
      ratio = st.c == 0.f ? 1.f : c / st.c;
      st.c = c;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float factor = c ? col.factor[n].y : col.factor[n].x;
        float& m = c ? st.m[n].y : st.m[n].x;
        float t = fmaxf(top[n][c] * factor, -m);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
        f[c] = t == kNegInf ? 1.f : ex2(-m - t);
        m = -t;
        (c ? st.limit[n].y : st.limit[n].x) = (t + 8.f) / factor;
      }
      st.l[n].x *= f[0], st.l[n].y *= f[1];
      st.z[n][0] *= f[0], st.z[n][1] *= f[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st.ps[n][i] *= f[i % 2] * ratio;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[n][d][i] *= f[i % 2] * ratio;
      }
    }
  }
  uint32_t b[kAb][NT][2];
#pragma unroll
  for (int u = 0; u < kAb; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float weight = vs[u][r] * st.c;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 m = st.m[n];
        if (kMasked) {
          m.x = m.x == -kNegInf ? 0.f : m.x;
          m.y = m.y == -kNegInf ? 0.f : m.y;
        }
        float2 p = fma2(make_float2(x[u][n][2 * r], x[u][n][2 * r + 1]), col.factor[n], m);
        p.x = ex2(p.x), p.y = ex2(p.y);
        st.l[n] = add2(st.l[n], p);
        float y[2] = {p.x * weight, p.y * weight};
        float z[2] = {fmaf(p.x, vz[u][r], st.z[n][0]), fmaf(p.y, vz[u][r], st.z[n][1])};
        if (kMasked) {  // a hidden token's scale and zero may be anything
          if (p.x == 0.f) y[0] = 0.f, z[0] = st.z[n][0];
          if (p.y == 0.f) y[1] = 0.f, z[1] = st.z[n][1];
        }
        st.z[n][0] = z[0], st.z[n][1] = z[1];
        const __half2 h = __floats2half2_rn(y[0], y[1]);
        uint32_t bits;
        __builtin_memcpy(&bits, &h, 4);
        b[u][n][r] = transpose8x8(bits);
      }
    }
  each<kAb>([&](auto index) {
    constexpr int u = decltype(index)::value;
    unit_values<D, NT, U + u>(at, b[u], st);
  });
}

// The units of a step, as many at a time as the registers hold.
template <int D, int NT, bool kMasked>
__device__ __forceinline__ void attend_step(const AttnArgs& a, const TileShared<D, NT>& sh,
                                            const uint2* qreg, const LaneAddress& at,
                                            const int* number, const Columns<NT>& col,
                                            const Span& v, WarpState<D, NT>& st) {
  constexpr int kAll = Shape<D>::kUnits;
  constexpr int kAb = NT == 4 ? 1 : NT == 2 || D == 256 || kMasked ? 2 : 4;
  each<kAll / kAb>([&](auto index) {
    constexpr int kFirst = decltype(index)::value * kAb;
    if constexpr (kMasked) {  // units behind the last are not there
      bool any = false;
#pragma unroll
      for (int u = 0; u < kAb; ++u) any |= number[kFirst + u] >= 0;
      if (!any) return;
    }
    attend_units<D, NT, kFirst, kAb, kMasked>(a, sh, qreg, at, number + kFirst, col, v, st);
  });
}

// Four dimensions of one row's result: sum / l and log-sum-exp; zeros and -inf
// for a row that sees nothing.
template <typename T>
__device__ __forceinline__ void store_row(const AttnArgs& a, const Seq& s, int row, int head, int d,
                                          float4 o, float m, float l) {
  const int64_t token = s.start + row / a.group;
  const int h = head * a.group + row % a.group;
  const float f = l == 0.f ? 0.f : 1.f / l;
  T x[4] = {from_float<T>(o.x * f), from_float<T>(o.y * f), from_float<T>(o.z * f),
            from_float<T>(o.w * f)};
  T* to = static_cast<T*>(a.out) + token * a.o_token + int64_t(h) * a.o_head + d;
  if (a.o_vec) {
    uint2 w;
    __builtin_memcpy(&w, x, 8);
    *reinterpret_cast<uint2*>(to) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = x[i];
  }
  if (a.lse && d == 0)
    a.lse[token * (int64_t(a.cache.kv_heads) * a.group) + h] =
        l == 0.f ? kNegInf : (m + log2f(l)) * 0.6931471805599453f;
}

// The units [u0, u1) of one (tile of query rows, kv head): every warp takes
// pairs of units in turn through its own ring of cp.async stages, then the
// warps' results are joined.  `slot` < 0: the result is the tile's output,
// otherwise it goes to that place of the workspace.
template <typename T, int D, int NT>
__device__ __forceinline__ void attend_segment(const AttnArgs& a, TileShared<D, NT>& sh, uint8_t* ring, int b,
                               const Seq& s, const Span& v, int row0, int rows, int head, int u0,
                               int u1, int slot) {
  using S = Shape<D>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  uint8_t* mine = ring + warp * S::kWarpBytes;
  const uint32_t mine_s = uint32_t(__cvta_generic_to_shared(mine));
  constexpr int kU = S::kUnits, kGroup = 32 / kU;  // steps whose units the lanes hold
  const int blocks = (u1 - u0 + kU - 1) / kU;
  const int steps = blocks > warp ? (blocks - warp + kWarps - 1) / kWarps : 0;
  const int32_t* table = a.tables + int64_t(b) * a.table_stride;

  // Where the units of the next kGroup steps are, one in every lane: byte
  // offset in the pages and token in the page.  `have` has a bit for each.
  struct Units {
    int64_t offset;
    int within;
    uint32_t have;
  };
  auto fetch = [&](int step) {
    Units f{0, 0, 0u};
    const int i = u0 + kU * (warp + kWarps * (step + lane / kU)) + lane % kU;
    bool real = i < u1;
    if (real) {
      const int n = i < v.sink_units ? i : i + v.gap;
      const int page = a.upp_shift >= 0 ? n >> a.upp_shift : n / a.upp;
      const int id = table[page];
      f.within = n - page * a.upp;
      real = id >= 0 && id < a.cache.num_blocks;
      if (real) f.offset = id * a.cache.stride + f.within * S::kUnit;
      else atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
    }
    f.have = __ballot_sync(~0u, real);
    return f;
  };
  Units now = fetch(0), later{0, 0, 0u};
  if (steps > kGroup) later = fetch(kGroup);
  uint32_t there = 0;  // which units of the steps in flight are there, kU bits a step

  // This lane's part of the copies: 16-byte pieces lane, lane + 32, ... of each
  // unit's codes, and one piece of the runs of scales and zeros.
  const int64_t head_at = int64_t(head) * a.cache.head_bytes;
  const uint8_t* key_from = a.cache.pages[0] + head_at + 16 * lane;
  const uint8_t* value_from = a.cache.pages[1] + head_at + 16 * lane;
  const int param_unit = (lane / 4) % kU;
  const uint8_t* param_from = a.cache.pages[lane / (4 * kU) % 2] + head_at +
                              a.cache.block_size * (D / 2) + 16 * (lane % 4);
  auto load_step = [&](int step, uint32_t dst) {
    const int at = kU * (step % kGroup);
    const uint32_t bits = (now.have >> at) & ((1u << kU) - 1u);
    there = (there << kU) | bits;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t offset = __shfl_sync(~0u, now.offset, at + u);
      const int size = (bits >> u) & 1u ? 16 : 0;
#pragma unroll
      for (int i = 0; i < S::kUnit / 512; ++i) {
        // The pieces' places are permuted so that the fragments' reads meet no bank twice.
        const int c = lane + 32 * i;
        const int kc = D == 256 ? c ^ (4 * ((c >> 3) & 1)) : c;
        const int vc = c ^ (D == 64    ? 2 * ((c >> 3) & 1)
                            : D == 128 ? 2 * ((c >> 3) & 3)
                                       : 2 * ((c >> 4) & 3));
        copy16(dst + u * S::kUnit + 16 * kc, key_from + offset + 512 * i, size);
        copy16(dst + (kU + u) * S::kUnit + 16 * vc, value_from + offset + 512 * i, size);
      }
    }
    const int64_t offset = __shfl_sync(~0u, now.offset, at + param_unit);
    const int within = __shfl_sync(~0u, now.within, at + param_unit);
    if (lane < 8 * kU)
      copy16(dst + 2 * kU * S::kUnit + 16 * lane, param_from + offset - within * (S::kUnit - 64),
             (bits >> param_unit) & 1u ? 16 : 0);
  };

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < steps) load_step(i, mine_s + i * S::kStage);
    else there <<= kU;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  load_queries<T, D, NT>(a, s, row0, rows, head, sh);
  __syncthreads();

  Columns<NT> col;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = 8 * n + 2 * j;
    col.factor[n] = make_float2(sh.factor[c], sh.factor[c + 1]);
    col.sum[n] = make_float2(sh.sum[c], sh.sum[c + 1]);
    col.pos[n][0] = sh.pos[c], col.pos[n][1] = sh.pos[c + 1];
  }
  uint2 qreg[NT == 1 ? D / 16 : 1];
  if constexpr (NT == 1) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qreg[i] = sh.q[0][i][lane];
  }
  WarpState<D, NT> st;
  st.c = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    st.m[n] = make_float2(-kNegInf, -kNegInf), st.l[n] = make_float2(0.f, 0.f);
    st.limit[n] = make_float2(kNegInf, kNegInf);
    st.z[n][0] = st.z[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      st.ps[n][i] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) st.o[n][d][i] = 0.f;
    }
  }

  // Steps that begin in [plain_from, plain_from + plain_units) need no mask:
  // behind no row, and inside every row's window.
  const int plain_from = max(v.sink_units, (max(v.p_hi - a.window + 1, 0) + 15) / 16 - v.gap);
  const unsigned plain_units = unsigned(max((v.p_lo + 1) / 16 - v.gap - plain_from - (kU - 1), 0));
  const LaneAddress lane_at = lane_address<D>(mine_s, g, j);
  uint32_t buffer = 0, ahead = (kStages - 1) * S::kStage;  // bytes into the ring
  int i = u0 + kU * warp;
  for (int step = 0; step < steps; ++step, i += kU * kWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    const int next = step + kStages - 1;
    if (next % kGroup == 0) {
      now = later;
      if (next + kGroup < steps) later = fetch(next + kGroup);
    }
    if (next < steps) load_step(next, mine_s + ahead);
    else there <<= kU;
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t bits = (there >> (kU * (kStages - 1))) & ((1u << kU) - 1u);
    const LaneAddress at = lane_at + buffer;
    if (bits == (1u << kU) - 1u && unsigned(i - plain_from) < plain_units) {
      attend_step<D, NT, false>(a, sh, qreg, at, nullptr, col, v, st);
    } else {
      int number[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        number[u] = (bits >> u) & 1u ? (i + u < v.sink_units ? i + u : i + u + v.gap) : -1;
      attend_step<D, NT, true>(a, sh, qreg, at, number, col, v, st);
    }
    __syncwarp();
    buffer = buffer + S::kStage == S::kWarpBytes ? 0u : buffer + S::kStage;
    ahead = ahead + S::kStage == S::kWarpBytes ? 0u : ahead + S::kStage;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // Join the warps.  Sums over the tokens of a thread's rows first.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = c ? st.l[n].y : st.l[n].x;
#pragma unroll
      for (int d = 4; d < 32; d *= 2) {
        l += __shfl_xor_sync(~0u, l, d);
        st.z[n][c] += __shfl_xor_sync(~0u, st.z[n][c], d);
      }
      if (g == 0) {
        sh.m[warp][8 * n + 2 * j + c] = c ? -st.m[n].y : -st.m[n].x;
        sh.l[warp][8 * n + 2 * j + c] = l;
      }
    }
  const float back = st.c > 0.f ? 1.f / st.c : 0.f;
  float* join = reinterpret_cast<float*>(ring);
  constexpr int kPitch = D + 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (8 * n >= rows) break;  // the same for the whole block
    __syncthreads();           // the ring, or the previous rows, are read
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float* to = join + (warp * 8 + 2 * j + c) * kPitch + g * (D / 8);
      const float mid = 7.5f * st.ps[n][c];
#pragma unroll
      for (int d = 0; d < D / 16; d += 2) {
        float4 f;
        f.x = fmaf(fmaf(st.o[n][d][c], 16777216.f, -mid), back, st.z[n][c]);
        f.y = fmaf(fmaf(st.o[n][d][2 + c], 1048576.f, -mid), back, st.z[n][c]);
        f.z = fmaf(fmaf(st.o[n][d + 1][c], 16777216.f, -mid), back, st.z[n][c]);
        f.w = fmaf(fmaf(st.o[n][d + 1][2 + c], 1048576.f, -mid), back, st.z[n][c]);
        *reinterpret_cast<float4*>(to + 2 * d) = f;
      }
    }
    __syncthreads();
    for (int e = threadIdx.x * 4; e < 8 * D; e += kThreads * 4) {
      const int r = 8 * n + e / D, d = e % D;
      if (r >= rows) continue;
      float m = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh.m[w][r]);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = sh.m[w][r], lw = sh.l[w][r];
        // A warp without a finite score counts for nothing, unless a NaN is among them.
        const float f = mw == kNegInf ? (lw == lw ? 0.f : lw) : ex2(mw - m);
        if (f != 0.f) {
          const float4 x = *reinterpret_cast<const float4*>(join + (w * 8 + r % 8) * kPitch + d);
          l = fmaf(f, lw, l);
          o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y);
          o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
        }
      }
      if (slot >= 0) {
        *reinterpret_cast<float4*>(a.part_o + (int64_t(slot) * (8 * NT) + r) * D + d) = o;
        if (d == 0) a.part_ml[int64_t(slot) * (8 * NT) + r] = make_float2(m, l);
      } else {
        store_row<T>(a, s, row0 + r, head, d, o, m, l);
      }
    }
  }
  __syncthreads();  // before the ring and the rows are used again
}

// Rows of a tile that see nothing.
template <typename T, int D>
__device__ __forceinline__ void store_nothing(const AttnArgs& a, const Seq& s, int row0, int rows,
                                              int head) {
  for (int e = threadIdx.x; e < rows * (D / 4); e += kThreads)
    store_row<T>(a, s, row0 + e / (D / 4), head, e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f),
                 kNegInf, 0.f);
}

// What a sequence adds to the work: items of one tile of query rows with one kv
// head, each counted as long as the longest of the sequence's tiles, behind
// kItemUnits for what an item costs besides.
struct Work {
  Seq s;
  int rows, tiles, units;
  int64_t total;
};

template <int ROWS>
__device__ __forceinline__ Work work_of(const AttnArgs& a, int b) {
  Work w;
  w.s = seq_of(a, b);
  w.rows = w.s.count * a.group;
  w.tiles = (w.rows + ROWS - 1) / ROWS;
  w.units = span_of(a, w.s, 0, w.rows).units;
  w.total = int64_t(w.units + kItemUnits) * w.tiles * a.cache.kv_heads;
  return w;
}

__device__ __forceinline__ int64_t share_of(int64_t total, int shares) {
  return max(int64_t(kMinUnits + kItemUnits), (total + shares - 1) / shares);
}

// Item and offset in it of a position of a sequence's work.
__device__ __forceinline__ void item_of(const Work& w, int64_t in, int* item, int* off) {
  const int length = w.units + kItemUnits;
  if (in < (int64_t(1) << 31)) {  // the common case: no 64-bit division
    *item = int(unsigned(in) / unsigned(length));
    *off = int(unsigned(in) - unsigned(*item) * unsigned(length));
  } else {
    *item = int(in / length);
    *off = int(in - int64_t(*item) * length);
  }
}

// All work of the call, [kv head][tile][units] of one sequence after the other,
// in equal shares: one for each CTA of a grid that is resident at once.  A
// share that begins or ends among an item's units leaves a partial result in
// the workspace (at most two for a CTA), which q4_join brings together.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2)
    q4_attend(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ TileShared<D, NT> sh;
  constexpr int kRows = 8 * NT;
  asm volatile("griddepcontrol.launch_dependents;");
  Place place;
  int64_t share = 0;
  const int64_t total = block_locate(
      [&](int b) { return work_of<kRows>(a, b).total; }, a.batch,
      [&](int64_t all) {
        share = share_of(all, gridDim.x);
        return share * blockIdx.x;
      },
      sh.scan, &sh.place, &place);
  const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
  if (begin >= end) return;
  int b = place.index;
  int64_t before = place.before, pos = begin;
  while (pos < end && b < a.batch) {
    const Work w = work_of<kRows>(a, b);
    if (w.total == 0) {
      ++b;
      continue;
    }
    int item, off;
    item_of(w, pos - before, &item, &off);
    const int n = int(min(int64_t(w.units + kItemUnits - off), end - pos));
    const int head = item / w.tiles, row0 = (item % w.tiles) * kRows;
    const int rows = min(kRows, w.rows - row0);
    // Units of this share; the item's first kItemUnits positions stand for none.
    const int u0 = max(off - kItemUnits, 0), u1 = max(off + n - kItemUnits, 0);
    if (w.units == 0) {
      if (off == 0) store_nothing<T, D>(a, w.s, row0, rows, head);
    } else if (u1 > u0) {
      const Span v = span_of(a, w.s, row0, rows);
      const bool whole = u0 == 0 && u1 == w.units;
      attend_segment<T, D, NT>(a, sh, ring, b, w.s, v, row0, rows, head, min(u0, v.units),
                               min(u1, v.units),
                               whole ? -1 : 2 * int(blockIdx.x) + (pos == begin ? 0 : 1));
    }
    pos += n;
    if (pos - before == w.total) {
      before = pos;
      ++b;
    }
  }
}

// The pieces of an item that starts at `start`: shares first .. last hold units
// of it.  A share's piece is its first (even slot) where the share begins inside
// the item or at its start.
struct Pieces {
  int64_t start, share, first, last;
  __device__ __forceinline__ int64_t slot(int64_t k) const {
    return 2 * k + (start > k * share ? 1 : 0);
  }
};

__device__ __forceinline__ Pieces pieces_of(const Work& w, int64_t start, int64_t share) {
  return Pieces{start, share, (start + kItemUnits) / share,
                (start + kItemUnits + w.units - 1) / share};
}

// Joins one row's pieces, those of warp `part` of `parts`, in their order.
template <int D>
__device__ __forceinline__ void join_row(const AttnArgs& a, const Pieces& p, int kRows, int r,
                                         int part, int parts, float& m, float& l,
                                         float4 (&o)[(D + 127) / 128]) {
  const int lane = threadIdx.x % 32;
  m = kNegInf;
  for (int64_t k = p.first + lane; k <= p.last; k += 32)
    m = fmaxf(m, a.part_ml[p.slot(k) * kRows + r].x);
#pragma unroll
  for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  l = 0.f;
#pragma unroll
  for (int i = 0; i < (D + 127) / 128; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int64_t k = p.first + part; k <= p.last; k += parts) {
    const int64_t at = p.slot(k) * kRows + r;
    const float2 ml = a.part_ml[at];
    float4 x[(D + 127) / 128];
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i) {
      const int d = 128 * i + 4 * lane;
      x[i] = d < D ? *reinterpret_cast<const float4*>(a.part_o + at * D + d)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // A piece without a finite score counts for nothing, unless a NaN is in it.
    const float f = ml.x == kNegInf ? (ml.y == ml.y ? 0.f : ml.y) : ex2(ml.x - m);
    if (f != 0.f) {
      l = fmaf(f, ml.y, l);
#pragma unroll
      for (int i = 0; i < (D + 127) / 128; ++i) {
        o[i].x = fmaf(f, x[i].x, o[i].x), o[i].y = fmaf(f, x[i].y, o[i].y);
        o[i].z = fmaf(f, x[i].z, o[i].z), o[i].w = fmaf(f, x[i].w, o[i].w);
      }
    }
  }
}

// Joins the partial results of items that several CTAs shared; the pieces are
// summed in an order that does not vary.  Two forms:
//   kByRow false: block k looks at the border behind share k and works when it
//     is the first border among an item's units; a warp takes a row.
//   kByRow true: a block for each row of each item, its warps share the pieces:
//     for few items with many pieces, where a warp alone would take long.
template <typename T, int D, int NT, bool kByRow>
__global__ void __launch_bounds__(kThreads) q4_join(const __grid_constant__ AttnArgs a,
                                                    int shares) {
  __shared__ int64_t scan[kWarps];
  __shared__ Place found;
  __shared__ float4 part[kByRow ? kWarps : 1][(D + 127) / 128][32];
  __shared__ float part_l[kWarps];
  constexpr int kRows = 8 * NT;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Place place;           // the item's sequence and the work before it
  int64_t share = 0, start = 0;  // work before the item
  bool none = false;
  if constexpr (kByRow) {
    // Few sequences: one thread walks them.
    __shared__ int64_t walked[2];
    if (threadIdx.x == 0) {
      int64_t left = blockIdx.x / kRows, total = 0;
      found = Place{a.batch, 0};
      for (int b = 0; b < a.batch; ++b) {
        const Work w = work_of<kRows>(a, b);
        const int64_t items = int64_t(w.tiles) * a.cache.kv_heads;
        if (left >= 0 && left < items) {
          found = Place{b, total};
          walked[1] = total + left * (w.units + kItemUnits);
        }
        left -= items;
        total += w.total;
      }
      walked[0] = total;
    }
    __syncthreads();
    place = found;
    share = share_of(walked[0], shares);
    start = walked[1];
    none = place.index >= a.batch;
  } else {
    const int64_t total = block_locate(
        [&](int b) { return work_of<kRows>(a, b).total; }, a.batch,
        [&](int64_t all) {
          share = share_of(all, shares);
          return share * (int64_t(blockIdx.x) + 1);
        },
        scan, &found, &place);
    start = share * (int64_t(blockIdx.x) + 1);  // the border, for now
    none = start >= total;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (none) return;
  const Work w = work_of<kRows>(a, place.index);
  if (w.units == 0) return;
  int item, off;
  item_of(w, start - place.before, &item, &off);
  start -= off;
  const Pieces p = pieces_of(w, start, share);
  if (p.first == p.last || (!kByRow && p.first != blockIdx.x)) return;
  const int row0 = (item % w.tiles) * kRows, rows = min(kRows, w.rows - row0);
  const int head = item / w.tiles;
  float m, l;
  float4 o[(D + 127) / 128];
  if (!kByRow) {
    for (int r = warp; r < rows; r += kWarps) {
      join_row<D>(a, p, kRows, r, 0, 1, m, l, o);
#pragma unroll
      for (int i = 0; i < (D + 127) / 128; ++i)
        if (128 * i + 4 * lane < D)
          store_row<T>(a, w.s, row0 + r, head, 128 * i + 4 * lane, o[i], m, l);
    }
    return;
  }
  const int r = blockIdx.x % kRows;
  if (r >= rows) return;
  join_row<D>(a, p, kRows, r, warp, kWarps, m, l, o);
#pragma unroll
  for (int i = 0; i < (D + 127) / 128; ++i) part[kByRow ? warp : 0][i][lane] = o[i];
  if (lane == 0) part_l[warp] = l;
  __syncthreads();
  if (warp > 0) return;
#pragma unroll
  for (int k = 1; k < kWarps; ++k) {
    l += part_l[k];
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i) {
      const float4 x = part[kByRow ? k : 0][i][lane];
      o[i].x += x.x, o[i].y += x.y, o[i].z += x.z, o[i].w += x.w;
    }
  }
#pragma unroll
  for (int i = 0; i < (D + 127) / 128; ++i)
    if (128 * i + 4 * lane < D)
      store_row<T>(a, w.s, row0 + r, head, 128 * i + 4 * lane, o[i], m, l);
}

}  // namespace q4
}  // namespace kvx
