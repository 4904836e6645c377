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

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;       // pairs of units in flight or in use, per warp
constexpr int kNoWindow = 1 << 30;
// Fewest 16-token units a CTA takes: two for each warp.  Fewer make the join
// the larger part of the work.
constexpr int kMinUnits = 2 * kWarps;

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
  float scale_log2;         // softmax scale * log2(e)
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

// Sum of f(0..n-1) over the block, and the place of `pos` in its running sum.
template <class F>
__device__ int64_t block_total(F f, int n, int64_t* sm) {
  int64_t v = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) v += f(i);
#pragma unroll
  for (int d = 16; d; d /= 2) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) v += sm[i];
  __syncthreads();
  return v;
}

struct Place {
  int index;       // the i whose part holds the position, n when none does
  int64_t before;  // sum of f(0..index-1)
};

template <class F>
__device__ Place block_locate(F f, int n, int64_t pos, int64_t* sm, Place* found) {
  if (threadIdx.x == 0) *found = Place{n, 0};
  int64_t base = 0;
  for (int at = 0; at < n; at += kThreads) {
    const int i = at + threadIdx.x;
    const int64_t own = i < n ? f(i) : 0;
    int64_t v = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t u = __shfl_up_sync(~0u, v, d);
      if (threadIdx.x % 32 >= d) v += u;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 31) sm[threadIdx.x / 32] = v;
    __syncthreads();
    int64_t before = base, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < int(threadIdx.x / 32)) before += sm[w];
      all += sm[w];
    }
    before += v - own;
    if (pos >= before && pos < before + own) *found = Place{i, before};
    base += all;
  }
  __syncthreads();
  const Place p = *found;
  __syncthreads();
  return p;
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

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;  // 0: nothing is read, 16 zero bytes are written
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}

constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kEven = 0x000f000fu;  // nibbles 0 and 4: code * 2^-24 in each half
constexpr uint32_t kOdd = 0x00f000f0u;   // nibbles 1 and 5: code * 2^-20

template <int D>
struct Shape {
  static constexpr int kUnit = 8 * D;           // bytes of codes of 16 tokens
  static constexpr int kStage = 4 * kUnit + 256;  // K and V of two units, (scale, zero) of each
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kRing = kWarps * kWarpBytes;
  static constexpr int kJoin = kWarps * 8 * (D + 4) * 4;
  static constexpr int kShared = kRing > kJoin ? kRing : kJoin;
  static constexpr int kKeyWords = D / 32;      // code words of a thread for one token of K
  static constexpr int kValueWords = D / 64;    // ... for one token of V
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
  float factor[NT * 8];     // scale * log2(e) and the powers of two taken out
  float sum[NT * 8];        // sum(q) * scale * log2(e)
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
      sum += x[w][i];
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    sum += __shfl_xor_sync(~0u, sum, d);
  }
  // 2^(14 - exponent of top); bounded so that both it and its inverse are normal.
  const int e = min(max(int(__float_as_uint(top) >> 23), 20), 250);
  const float up = top > 0.f ? __uint_as_float(uint32_t(min(127 + 14 + 127 - e, 240)) << 23) : 1.f;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = (i % 2) ? up * 0.0625f : up;  // odd nibbles are 16 times as large
      const __half2 h = __floats2half2_rn(x[w][i] * u, x[w][i + 4] * u);
      __builtin_memcpy(&f[i], &h, 4);
    }
    sh.q[warp][2 * w][lane] = make_uint2(f[0], f[1]);
    sh.q[warp][2 * w + 1][lane] = make_uint2(f[2], f[3]);
  }
  if (j == 0) {
    sh.factor[r] = a.scale_log2 * 16777216.f / up;
    sh.sum[r] = a.scale_log2 * sum;
    sh.pos[r] = pos;
  }
}

// One warp's state over the units that it takes.
template <int D, int NT>
struct WarpState {
  float o[NT][D / 16][4];  // sum of p * s * C * code, dimensions as in value_dim()
  float ps[NT][4];         // sum of the same weights as the matrix instruction saw them
  float m[NT][2], l[NT][2], z[NT][2];
  float c;                 // C: power of two on the V scales, so that weights suit fp16
};

// AB units at a time: scores, softmax, products.  `first` is the first unit's
// number in the sequence, -1 for a unit that is not there.
template <int D, int NT, int AB, bool kMasked>
__device__ __forceinline__ void attend_units(const AttnArgs& a, const TileShared<D, NT>& sh,
                                             const uint2* qreg, const uint8_t* stage,
                                             int unit0, const int (&number)[AB],
                                             const float (&factor)[NT][2],
                                             const float (&qsum)[NT][2], const int (&pos)[NT][2],
                                             const Span& v, WarpState<D, NT>& st) {
  const int lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  constexpr int kKW = Shape<D>::kKeyWords, kVW = Shape<D>::kValueWords, kUnit = Shape<D>::kUnit;
  const uint8_t* keys = stage;
  const uint8_t* values = stage + 2 * kUnit;
  const uint8_t* params = stage + 4 * kUnit;
  float x[AB][NT][4];
#pragma unroll
  for (int u = 0; u < AB; ++u) {
    uint32_t kw[2][kKW];
    const uint8_t* unit = keys + (unit0 + u) * kUnit;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* row = unit + (g + 8 * r) * (D / 2);
      if constexpr (D == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 8 * j);
        kw[r][0] = v.x, kw[r][1] = v.y;
      } else if constexpr (D == 128) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * j);
        kw[r][0] = v.x, kw[r][1] = v.y, kw[r][2] = v.z, kw[r][3] = v.w;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * ((4 * h + j) ^ (4 * (g & 1))));
          kw[r][4 * h] = v.x, kw[r][4 * h + 1] = v.y, kw[r][4 * h + 2] = v.z, kw[r][4 * h + 3] = v.w;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][n][i] = 0.f;
#pragma unroll
    for (int w = 0; w < kKW; ++w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r0 = h ? kw[0][w] >> 8 : kw[0][w], r1 = h ? kw[1][w] >> 8 : kw[1][w];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint2 q = NT == 1 ? qreg[2 * w + h] : sh.q[n][2 * w + h][lane];
          mma(x[u][n], r0 & kEven, r1 & kEven, r0 & kOdd, r1 & kOdd, q.x, q.y);
        }
      }
    }
  }
  // Scores in powers of two; this thread's tokens are g and g + 8 of each unit.
  float top[NT][2];
  float vs[AB][2], vz[AB][2], most = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = kNegInf;
#pragma unroll
  for (int u = 0; u < AB; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int at = (unit0 + u) * 64 + (g + 8 * r) * 4;
      const float2 k = __half22float2(*reinterpret_cast<const __half2*>(params + at));
      const float2 w = __half22float2(*reinterpret_cast<const __half2*>(params + 128 + at));
      vs[u][r] = w.x;
      vz[u][r] = fmaf(7.5f, w.x, w.y);
      const int t = number[u] * 16 + g + 8 * r;
      // Only of tokens that some row sees: what lies behind a sequence may be anything.
      if (!kMasked || (number[u] >= 0 && t <= v.p_hi && (t > v.p_lo - a.window || t < a.sinks)))
        most = fmaxf(most, fabsf(w.x));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float& y = x[u][n][2 * r + c];
          y = fmaf(k.x, y * factor[n][c], k.y * qsum[n][c]);
          if constexpr (kMasked) {
            const int p = pos[n][c];
            const bool seen = number[u] >= 0 && t <= p && (t > p - a.window || t < a.sinks);
            y = seen ? y : kNegInf;
          }
          top[n][c] = fmaxf(top[n][c], y);
        }
    }
  // Move the reference point where a score passes it by 2^8, or the weights
  // would leave fp16.
  bool move = !(most * st.c <= 64.f) || st.c == 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) move |= top[n][0] > st.m[n][0] + 8.f || top[n][1] > st.m[n][1] + 8.f;
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
        float t = fmaxf(top[n][c], st.m[n][c]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
        f[c] = t == kNegInf ? 1.f : ex2(st.m[n][c] - t);
        st.m[n][c] = t;
        st.l[n][c] *= f[c];
        st.z[n][c] *= f[c];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st.ps[n][i] *= f[i % 2] * ratio;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[n][d][i] *= f[i % 2] * ratio;
      }
    }
  }
  uint32_t b[AB][NT][2];
#pragma unroll
  for (int u = 0; u < AB; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float weight = vs[u][r] * st.c;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float y[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float m = kMasked && st.m[n][c] == kNegInf ? 0.f : st.m[n][c];
          const float p = ex2(x[u][n][2 * r + c] - m);
          st.l[n][c] += p;
          if (kMasked && p == 0.f) {  // a hidden token's scale and zero may be anything
            y[c] = 0.f;
          } else {
            y[c] = p * weight;
            st.z[n][c] = fmaf(p, vz[u][r], st.z[n][c]);
          }
        }
        const __half2 h = __floats2half2_rn(y[0], y[1]);
        __builtin_memcpy(&b[u][n][r], &h, 4);
        b[u][n][r] = transpose8x8(b[u][n][r]);
      }
    }
#pragma unroll
  for (int u = 0; u < AB; ++u) {
    const uint8_t* unit = values + (unit0 + u) * kUnit;
    uint32_t vw[4][kVW];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 2 * j + (r & 1) + 8 * (r >> 1);
      if constexpr (D == 64) {
        vw[r][0] = *reinterpret_cast<const uint32_t*>(
            unit + ((t * 32 + 4 * g) ^ (32 * ((t >> 2) & 1))));
      } else if constexpr (D == 128) {
        const uint2 v = *reinterpret_cast<const uint2*>(
            unit + ((t * 64 + 8 * g) ^ (32 * ((t >> 1) & 3))));
        vw[r][0] = v.x, vw[r][1] = v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(
            unit + ((t * 128 + 16 * g) ^ (32 * ((t >> 1) & 3))));
        vw[r][0] = v.x, vw[r][1] = v.y, vw[r][2] = v.z, vw[r][3] = v.w;
      }
    }
#pragma unroll
    for (int w = 0; w < kVW; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // Tokens 2j, 2j+1 side by side: the low or high halves of their words.
        const uint32_t sel = e < 2 ? 0x5410u : 0x7632u;
        uint32_t p = __byte_perm(vw[0][w], vw[1][w], sel), q = __byte_perm(vw[2][w], vw[3][w], sel);
        if (e % 2) p >>= 8, q >>= 8;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma(st.o[n][4 * w + e], p & kEven, p & kOdd, q & kEven, q & kOdd, b[u][n][0], b[u][n][1]);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
      mma(st.ps[n], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, b[u][n][0], b[u][n][1]);
  }
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
__device__ void attend_segment(const AttnArgs& a, TileShared<D, NT>& sh, uint8_t* ring, int b,
                               const Seq& s, const Span& v, int row0, int rows, int head, int u0,
                               int u1, int slot) {
  using S = Shape<D>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  uint8_t* mine = ring + warp * S::kWarpBytes;
  const uint32_t mine_s = uint32_t(__cvta_generic_to_shared(mine));
  const int pairs = (u1 - u0 + 1) / 2;
  const int steps = pairs > warp ? (pairs - warp + kWarps - 1) / kWarps : 0;
  const int32_t* table = a.tables + int64_t(b) * a.table_stride;

  // Block ids of the next 16 steps, two units each, one in every lane.
  auto fetch_ids = [&](int step, int& id, int& within) {
    const int i = u0 + 2 * (warp + kWarps * (step + lane / 2)) + lane % 2;
    id = -1;
    within = 0;
    if (i < u1) {
      const int n = i < v.sink_units ? i : i + v.gap;
      const int page = a.upp_shift >= 0 ? n >> a.upp_shift : n / a.upp;
      within = n - page * a.upp;
      id = table[page];
      if (id < 0 || id >= a.cache.num_blocks) {
        id = -1;
        atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
      }
    }
  };
  int id, within, next_id = -1, next_within = 0;
  fetch_ids(0, id, within);
  if (steps > 16) fetch_ids(16, next_id, next_within);
  uint32_t there = 0;  // which units of the steps in flight are there, two bits a step

  auto load_step = [&](int step, int buffer) {
    const int at = 2 * (step % 16);
    const uint32_t dst = mine_s + buffer * S::kStage;
    const int ids[2] = {__shfl_sync(~0u, id, at), __shfl_sync(~0u, id, at + 1)};
    const int in[2] = {__shfl_sync(~0u, within, at), __shfl_sync(~0u, within, at + 1)};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* pages = a.cache.pages[t] + int64_t(head) * a.cache.head_bytes;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool real = ids[u] >= 0;
        const uint8_t* src =
            pages + int64_t(real ? ids[u] : 0) * a.cache.stride[t] + in[u] * S::kUnit;
#pragma unroll
        for (int i = 0; i < S::kUnit / 512; ++i) {
          const int c = lane + 32 * i;
          int swizzle = 0;  // so that the fragments' reads meet no bank twice
          if (t == 1)
            swizzle = D == 64 ? 2 * ((c >> 3) & 1) : D == 128 ? 2 * ((c >> 3) & 3) : 2 * ((c >> 4) & 3);
          else if (D == 256)
            swizzle = 4 * ((c >> 3) & 1);
          copy16(dst + (2 * t + u) * S::kUnit + 16 * (c ^ swizzle), src + 16 * c, real);
        }
      }
    }
    if (lane < 16) {  // scales and zeros: 64 bytes for each unit and tensor
      const int t = lane / 8, u = (lane / 4) % 2;
      const bool real = ids[u] >= 0;
      const uint8_t* src = a.cache.pages[t] + int64_t(real ? ids[u] : 0) * a.cache.stride[t] +
                           int64_t(head) * a.cache.head_bytes + a.cache.block_size * (D / 2) +
                           in[u] * 64 + 16 * (lane % 4);
      copy16(dst + 4 * S::kUnit + 16 * lane, src, real);
    }
    there = (there << 2) | (ids[0] >= 0 ? 1u : 0u) | (ids[1] >= 0 ? 2u : 0u);
  };
  auto advance_ids = [&](int step) {  // before the first load of a new group of 16
    if (step % 16 == 0 && step > 0) {
      id = next_id;
      within = next_within;
      next_id = -1;
      if (step + 16 < steps) fetch_ids(step + 16, next_id, next_within);
    }
  };

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < steps) load_step(i, i);
    else there <<= 2;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  load_queries<T, D, NT>(a, s, row0, rows, head, sh);
  __syncthreads();

  float factor[NT][2], qsum[NT][2];
  int pos[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      factor[n][c] = sh.factor[8 * n + 2 * j + c];
      qsum[n][c] = sh.sum[8 * n + 2 * j + c];
      pos[n][c] = sh.pos[8 * n + 2 * j + c];
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
#pragma unroll
    for (int c = 0; c < 2; ++c) st.m[n][c] = kNegInf, st.l[n][c] = 0.f, st.z[n][c] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      st.ps[n][i] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) st.o[n][d][i] = 0.f;
    }
  }

  int buffer = 0;
  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    {
      const int next = step + kStages - 1;
      int to = buffer + kStages - 1;
      if (to >= kStages) to -= kStages;
      advance_ids(next);
      if (next < steps) load_step(next, to);
      else there <<= 2;
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const uint32_t bits = (there >> (2 * (kStages - 1))) & 3u;
    const int i = u0 + 2 * (warp + kWarps * step);
    int number[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      number[u] = (bits >> u) & 1u ? (i + u < v.sink_units ? i + u : i + u + v.gap) : -1;
    const int last = number[1] * 16 + 15, first = number[0] * 16;
    // Whole pairs need no mask: behind no row, and inside every row's window
    // or among the sinks.
    const bool plain = bits == 3u && last <= v.p_lo &&
                       (first > v.p_hi - a.window || last < a.sinks);
    const uint8_t* stage = mine + buffer * S::kStage;
    if constexpr (NT <= 2) {
      if (plain)
        attend_units<D, NT, 2, false>(a, sh, qreg, stage, 0, number, factor, qsum, pos, v, st);
      else
        attend_units<D, NT, 2, true>(a, sh, qreg, stage, 0, number, factor, qsum, pos, v, st);
    } else {
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        const int one[1] = {u ? number[1] : number[0]};
        if (plain)
          attend_units<D, NT, 1, false>(a, sh, qreg, stage, u, one, factor, qsum, pos, v, st);
        else
          attend_units<D, NT, 1, true>(a, sh, qreg, stage, u, one, factor, qsum, pos, v, st);
      }
    }
    __syncwarp();
    if (++buffer == kStages) buffer = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // Join the warps.  Sums over the tokens of a thread's rows first.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) {
        st.l[n][c] += __shfl_xor_sync(~0u, st.l[n][c], d);
        st.z[n][c] += __shfl_xor_sync(~0u, st.z[n][c], d);
      }
      if (g == 0) {
        sh.m[warp][8 * n + 2 * j + c] = st.m[n][c];
        sh.l[warp][8 * n + 2 * j + c] = st.l[n][c];
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

// What a sequence adds to the work: tiles of query rows x kv heads, each taken
// as long as the longest of the sequence's tiles (at least one unit, so that
// rows that see nothing are written too).
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
  w.units = max(span_of(a, w.s, 0, w.rows).units, 1);
  w.total = int64_t(w.units) * w.tiles * a.cache.kv_heads;
  return w;
}

// All units of the call, [tile x head][unit] of one sequence after the other,
// in equal shares: one for each CTA of a grid that is resident at once.  A
// share that begins or ends inside an item leaves a partial result in the
// workspace (at most two for a CTA), which q4_join brings together.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 && D <= 128 ? 2 : 1)
    q4_attend(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ TileShared<D, NT> sh;
  constexpr int kRows = 8 * NT;
  asm volatile("griddepcontrol.launch_dependents;");
  auto cost = [&](int b) { return work_of<kRows>(a, b).total; };
  const int64_t total = block_total(cost, a.batch, sh.scan);
  const int64_t share = max(int64_t(kMinUnits), (total + gridDim.x - 1) / gridDim.x);
  const int64_t begin = share * blockIdx.x, end = min(begin + share, total);
  if (begin >= end) return;
  const Place place = block_locate(cost, a.batch, begin, sh.scan, &sh.place);
  int b = place.index;
  int64_t before = place.before, pos = begin;
  while (pos < end && b < a.batch) {
    const Work w = work_of<kRows>(a, b);
    if (w.total == 0) {
      ++b;
      continue;
    }
    const int item = int((pos - before) / w.units), off = int((pos - before) % w.units);
    const int n = int(min(int64_t(w.units - off), end - pos));
    const int head = item / w.tiles, row0 = (item % w.tiles) * kRows;
    const int rows = min(kRows, w.rows - row0);
    const Span v = span_of(a, w.s, row0, rows);
    const bool whole = off == 0 && n == w.units;
    attend_segment<T, D, NT>(a, sh, ring, b, w.s, v, row0, rows, head, min(off, v.units),
                             min(off + n, v.units),
                             whole ? -1 : 2 * int(blockIdx.x) + (pos == begin ? 0 : 1));
    pos += n;
    if (pos - before == w.total) {
      before = pos;
      ++b;
    }
  }
}

// Joins the partial results of items that several CTAs shared.  Block k looks
// at the border behind share k and works when it is the first one inside an
// item; the pieces are summed in their order, so results do not vary.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) q4_join(const __grid_constant__ AttnArgs a,
                                                    int shares) {
  __shared__ int64_t scan[kWarps];
  __shared__ Place found;
  constexpr int kRows = 8 * NT;
  auto cost = [&](int b) { return work_of<kRows>(a, b).total; };
  const int64_t total = block_total(cost, a.batch, scan);
  const int64_t share = max(int64_t(kMinUnits), (total + shares - 1) / shares);
  const int64_t border = share * (int64_t(blockIdx.x) + 1);
  const Place place = block_locate(cost, a.batch, border, scan, &found);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (border >= total || place.index >= a.batch) return;
  const Work w = work_of<kRows>(a, place.index);
  const int item = int((border - place.before) / w.units);
  const int64_t start = place.before + int64_t(item) * w.units;
  const int64_t k0 = start / share, k1 = (start + w.units - 1) / share;
  if (start == border || k0 != blockIdx.x) return;
  const int row0 = (item % w.tiles) * kRows, rows = min(kRows, w.rows - row0);
  const int lane = threadIdx.x % 32;
  auto slot_of = [&](int64_t k) { return 2 * k + (k == k0 && start != k0 * share ? 1 : 0); };
  for (int r = threadIdx.x / 32; r < rows; r += kWarps) {
    float m = kNegInf;
    for (int64_t k = k0 + lane; k <= k1; k += 32) m = fmaxf(m, a.part_ml[slot_of(k) * kRows + r].x);
#pragma unroll
    for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    float l = 0.f;
    float4 o[(D + 127) / 128] = {};
    for (int64_t k = k0; k <= k1; ++k) {
      const int64_t at = slot_of(k) * kRows + r;
      const float2 p = a.part_ml[at];
      const float f = p.x == kNegInf ? (p.y == p.y ? 0.f : p.y) : ex2(p.x - m);
      if (f != 0.f) {
        l = fmaf(f, p.y, l);
#pragma unroll
        for (int i = 0; i < (D + 127) / 128; ++i) {
          const int d = 128 * i + 4 * lane;
          if (d < D) {
            const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * D + d);
            o[i].x = fmaf(f, x.x, o[i].x), o[i].y = fmaf(f, x.y, o[i].y);
            o[i].z = fmaf(f, x.z, o[i].z), o[i].w = fmaf(f, x.w, o[i].w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i) {
      const int d = 128 * i + 4 * lane;
      if (d < D) store_row<T>(a, w.s, row0 + r, item / w.tiles, d, o[i], m, l);
    }
  }
}

}  // namespace q4
}  // namespace kvx
