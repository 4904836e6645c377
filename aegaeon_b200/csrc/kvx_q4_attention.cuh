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
// p_j s'_j goes to the matrix instruction in fp16.  So a row's reference point follows
// its largest p_j s'_j, not its largest p_j: a token of large scale that has no
// weight then takes no bits from the others.  p_j itself stays in 32 bits, where
// it may be as large as the scales are apart.  The reference point is kept in powers
// of two and moves only when a product passes it by 2^8, so that most tiles
// neither reduce it nor rescale.
#pragma once

#include "kvx_q4_rows.cuh"

namespace kvx {
namespace q4 {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;       // a step in use and one in flight, per warp
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kNoWindow = 1 << 30;
// What an item (a tile of query rows with one kv head) costs a warp besides its
// 16-token units, in units: its queries, its first block ids, its result.  Measured
// with 3 / 12 / 16 / 24: 16 requests of 1024 to 2048 tokens with 32 kv heads 38.4 /
// 36.2 / 36.4 / 36.0 us, 128 of 4096 to 8192 with 8 170 / 166 / 164 / 168 us.
constexpr int kItemUnits = 16;
// Fewest units of a share when items are cut wherever shares end.
constexpr int kMinShare = 24;
// Units of the pieces that items may be cut into instead, kPiece << 0 ... kPieces - 1.
// Below four a warp's step is not full, and there are more pieces to join (one
// request of 1025 tokens: 10.7 us with single units, 10.3 with four).
constexpr int kPiece = 4, kPieces = 4;
// CTAs that an SM holds.
__host__ __device__ constexpr int ctas_per_sm(int head_dim, int rows) {
  return head_dim == 256 && rows > 8 ? 1 : 2;
}

struct Joint;

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
  float scale_part;         // that, as a number in [1/2, 1) (or 0)
  int scale_exp;            // and a power of two
  float sign;               // of the softmax scale
  int window;               // kNoWindow: none
  int sinks;                // 0 without a window
  int upp;                  // 16-token units of a page
  int upp_shift;            // log2(upp), -1 when it is no power of two
  int q_vec, o_vec;         // 16-byte accesses serve for query, 8-byte ones for out
  int o_vec16;              // 16-byte ones for out
  float* part_o;            // [2 * shares][rows][D]
  float2* part_ml;          // [2 * shares][rows] (reference point, sum of p)
  Joint* joints;            // [shares], or [items]
  int joint_by_item;
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
// Scores stay in the even codes' unit, 2^-24, until the exponent takes them: as part of a
// row's factor, 2^24 would overflow for queries of 2^118 and more.
constexpr float kCodeUnit = 16777216.f;

template <int D>
struct Shape {
  static constexpr int kUnit = 8 * D;           // bytes of codes of 16 tokens
  // Units of a step, which a warp takes at a time.  With four, what a step costs
  // besides its units (addresses, the vote on the reference point) is a tenth.
  static constexpr int kUnits = D == 256 ? 2 : 4;
  static constexpr int kParams = kUnits * 64;   // (scale, zero) of the units' tokens, one tensor
  static constexpr int kStage = kUnits * 2 * kUnit + 2 * kParams;
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kShared = kWarps * kWarpBytes;
};

// First dimension of code word w of quad lane j in a K row.  At D = 256 the
// two halves of a row are two 16-byte reads.
template <int D>
__device__ __forceinline__ int key_dim(int j, int w) {
  return D == 256 ? (w / 4) * 128 + 32 * j + 8 * (w % 4) : (D / 4) * j + 8 * w;
}

// What a thread keeps of the tile's rows (its columns 2j, 2j + 1 of each eight).
template <int NT>
struct Columns {
  float2 factor[NT];  // on the raw score: |scale| * log2(e) and the row's power of two taken out
  float2 sum[NT];     // sum(q) times that, as the raw score counts: in 1 / kCodeUnit
  int pos[NT][2];     // position in the sequence, -1 for rows that are none
};

// B fragments of the queries, as mma reads them: in registers for a tile of
// eight rows, otherwise in the warp's shared memory.
template <int D, int NT>
struct Fragments {
  uint2 reg[NT == 1 ? D / 16 : 1];
  uint2* shared;  // [NT][D / 16][32], this lane's
  __device__ __forceinline__ uint2 at(int n, int k) const {
    return NT == 1 ? reg[k] : shared[(n * (D / 16) + k) * 32];
  }
  __device__ __forceinline__ void set(int n, int k, uint2 x) {
    if constexpr (NT == 1) reg[k] = x;
    else shared[(n * (D / 16) + k) * 32] = x;
  }
};

// A power of two, 2^-113 to 2^127, that brings the largest element of a query row, `top`,
// into [2^14, 2^15), and rows below 2^-113 as near to it as fp32 has a number: every 16-bit
// float within 2^-28 of the largest stays exact in fp16.
__device__ __forceinline__ float row_scale(float top) {
  const int e = min(max(int(__float_as_uint(top) >> 23), 14), 254);
  return top > 0.f ? __uint_as_float(uint32_t(127 + 14 + 127 - e) << 23) : 1.f;
}
// What brings that row's scores back, with the softmax scale: above 0 and finite.
__device__ __forceinline__ float row_factor(float scale_log2, float up) {
  return fminf(fmaxf(scale_log2 / up, 1e-37f), 3.402823466e38f);
}

// A tile's query rows, scaled.
template <typename T, int D, int NT>
__device__ __forceinline__ void load_queries(const AttnArgs& a, const Seq& s, int row0, int rows,
                                             int head, Fragments<D, NT>& f, Columns<NT>& col) {
  const int lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  constexpr int kW = D / 32;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    const bool real = r < rows;
    float x[kW][8];
    const T* base = static_cast<const T*>(a.query);
    int pos = -1;
    if (real) {
      const int token = (row0 + r) / a.group, h = (row0 + r) - token * a.group;
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
    float up = row_scale(top);
    const float factor = row_factor(a.scale_log2, up);
    up *= a.sign;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = (i % 2) ? up * 0.0625f : up;  // odd nibbles are 16 times as large
        const __half2 h = __floats2half2_rn(x[w][i] * u, x[w][i + 4] * u);
        sum += x[w][i] * up + x[w][i + 4] * up;
        __builtin_memcpy(&b[i], &h, 4);
      }
      f.set(n, 2 * w, make_uint2(b[0], b[1]));
      f.set(n, 2 * w + 1, make_uint2(b[2], b[3]));
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) sum += __shfl_xor_sync(~0u, sum, d);
    sum *= factor * (1.f / kCodeUnit);
    // Row 2j is with the lanes 8j ..., row 2j + 1 four lanes on.
    col.factor[n] = make_float2(__shfl_sync(~0u, factor, 8 * j), __shfl_sync(~0u, factor, 8 * j + 4));
    col.sum[n] = make_float2(__shfl_sync(~0u, sum, 8 * j), __shfl_sync(~0u, sum, 8 * j + 4));
    col.pos[n][0] = __shfl_sync(~0u, pos, 8 * j);
    col.pos[n][1] = __shfl_sync(~0u, pos, 8 * j + 4);
  }
}

// log2 of a V scale, from its bits: at most 0.09 below it, which is enough to place
// the reference point.  A row of one value has scale 0 and counts 2^-32, so that its
// p is 2^46 at most.
__device__ __forceinline__ float size_of(float scale) {
  const float bits = __int2float_rn(int(__float_as_uint(scale) & 0x7fffffffu));
  return fmaxf(fmaf(bits, 1.1920928955078125e-7f, -127.f), -32.f);
}
// Where the reference point is put above or below the largest product, in powers of
// two, and how far above it a product may come: below 2^14.1 in all, inside fp16.
constexpr float kLift = 6.f, kSlack = 8.f;
// From this size on the roundings of a score (0.25 and more, in powers of two) eat that
// slack up.  Such a row's reference point is its largest score itself, of which every p is
// exactly what fp32 says, 1 at most; kFar, as a limit, says so: it is looked at in each step.
constexpr float kFarScore = 4194304.f, kFar = -3.402823466e38f;

// One warp's state over the units that it takes.
template <int D, int NT>
struct WarpState {
  float o[NT][D / 16][4];  // sum of p * s * code, dimensions as in value_dim()
  float ps[NT][4];         // sum of the same products as the matrix instruction saw them
  float2 m[NT], l[NT];     // minus the reference point, sum of p, by column
  float2 limit[NT];        // log2(p s) that moves the reference point; -inf: there is none yet
  float z[NT][2];          // sum of p * (zero + 7.5 scale)
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
__device__ __forceinline__ void unit_scores(const LaneAddress& at, const Fragments<D, NT>& f,
                                            float (&x)[NT][4]) {
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
        const uint2 q = f.at(n, 2 * w + h);
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
__device__ __forceinline__ void attend_units(const AttnArgs& a, const Fragments<D, NT>& f,
                                             const LaneAddress& at,
                                             const int* number, const Columns<NT>& col,
                                             WarpState<D, NT>& st) {
  const int lane = threadIdx.x % 32, g = lane / 4;
  float x[kAb][NT][4];
  // (scale, zero) of tokens g and g + 8 of each unit: K, then V.
  uint32_t kp[kAb][2], vp[kAb][2];
  each<kAb>([&](auto index) {
    constexpr int u = decltype(index)::value, at_u = 64 * (U + u);
    kp[u][0] = lds32<at_u>(at.p), kp[u][1] = lds32<at_u + 32>(at.p);
    vp[u][0] = lds32<Shape<D>::kParams + at_u>(at.p);
    vp[u][1] = lds32<Shape<D>::kParams + at_u + 32>(at.p);
    unit_scores<D, NT, U + u>(at, f, x[u]);
  });
  float vs[kAb][2], vz[kAb][2], top[NT][2];  // top: largest log2(p s)
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = kNegInf;
#pragma unroll
  for (int u = 0; u < kAb; ++u) {
    float2 size[NT][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 k = half2_at(kp[u][r]), w = half2_at(vp[u][r]);
      vs[u][r] = w.x;
      vz[u][r] = fmaf(7.5f, w.x, w.y);
      const float scale = size_of(w.x);
      const int unit = kMasked ? number[u] : 0, t = unit * 16 + g + 8 * r;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 y = fma2(make_float2(x[u][n][2 * r], x[u][n][2 * r + 1]),
                        mul2(both(k.x), col.factor[n]), mul2(both(k.y), col.sum[n]));
        if constexpr (kMasked) {
          auto seen = [&](int p) {
            return unit >= 0 && t <= p && (t > p - a.window || t < a.sinks);
          };
          y.x = seen(col.pos[n][0]) ? y.x : kNegInf;
          y.y = seen(col.pos[n][1]) ? y.y : kNegInf;
        }
        x[u][n][2 * r] = y.x, x[u][n][2 * r + 1] = y.y;
        size[n][r] = fma2(y, both(kCodeUnit), both(scale));
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n][0] = max3(top[n][0], size[n][0].x, size[n][1].x);
      top[n][1] = max3(top[n][1], size[n][0].y, size[n][1].y);
    }
  }
  bool move = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    move |= top[n][0] > st.limit[n].x || top[n][1] > st.limit[n].y;
  if (__any_sync(~0u, move)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float by[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float& m = c ? st.m[n].y : st.m[n].x;
        float& limit = c ? st.limit[n].y : st.limit[n].x;
        float t = fmaxf(top[n][c], limit - kSlack);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) t = fmaxf(t, __shfl_xor_sync(~0u, t, d));
        by[c] = 1.f;
        const bool far = limit == kFar || (t != kNegInf && fabsf(t) >= kFarScore);
        if (__any_sync(~0u, far)) {
          float y = kNegInf;
#pragma unroll
          for (int u = 0; u < kAb; ++u) y = max3(y, x[u][n][c], x[u][n][2 + c]);
          y *= kCodeUnit;
#pragma unroll
          for (int d = 4; d < 32; d *= 2) y = fmaxf(y, __shfl_xor_sync(~0u, y, d));
          if (far) {
            if (limit != kNegInf) {
              y = fmaxf(y, -m);
              by[c] = ex2(-y - m);
            }
            m = -y;
            limit = kFar;
          }
        }
        if (!far && t != kNegInf) {
          t = ceilf(t);
          if (limit != kNegInf) by[c] = ex2(kLift - t - m);
          m = kLift - t;
          limit = t + kSlack;
        }
      }
      st.l[n].x *= by[0], st.l[n].y *= by[1];
      st.z[n][0] *= by[0], st.z[n][1] *= by[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st.ps[n][i] *= by[i % 2];
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[n][d][i] *= by[i % 2];
      }
    }
  }
  uint32_t b[kAb][NT][2];
#pragma unroll
  for (int u = 0; u < kAb; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 p =
            fma2(make_float2(x[u][n][2 * r], x[u][n][2 * r + 1]), both(kCodeUnit), st.m[n]);
        p.x = ex2(p.x), p.y = ex2(p.y);
        st.l[n] = add2(st.l[n], p);
        float y[2] = {p.x * vs[u][r], p.y * vs[u][r]};
        float z[2] = {fmaf(p.x, vz[u][r], st.z[n][0]), fmaf(p.y, vz[u][r], st.z[n][1])};
        if (kMasked) {  // a hidden token's scale and zero may be anything
          if (x[u][n][2 * r] == kNegInf) y[0] = 0.f, z[0] = st.z[n][0];
          if (x[u][n][2 * r + 1] == kNegInf) y[1] = 0.f, z[1] = st.z[n][1];
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

// The units of a step.  `plain`: bits of those that need no mask; `there`: of those that
// are there at all; the first is number i of the tile's units.
template <int D, int NT>
__device__ __forceinline__ void attend_step(const AttnArgs& a, const Fragments<D, NT>& f,
                                            const LaneAddress& at, uint32_t there, uint32_t plain,
                                            int i, const Columns<NT>& col, const Span& v,
                                            WarpState<D, NT>& st) {
  constexpr int kU = Shape<D>::kUnits;
  constexpr uint32_t kAll = (1u << kU) - 1u;
  if constexpr (NT == 1 && kU == 4) {
    if (plain == kAll) {
      attend_units<D, NT, 0, 4, false>(a, f, at, nullptr, col, st);
      return;
    }
  }
  constexpr int kAb = NT == 4 ? 1 : 2;  // as many at a time as the registers hold
  constexpr uint32_t kPart = (1u << kAb) - 1u;
  each<kU / kAb>([&](auto index) {
    constexpr int kFirst = decltype(index)::value * kAb;
    if (((plain >> kFirst) & kPart) == kPart) {
      attend_units<D, NT, kFirst, kAb, false>(a, f, at, nullptr, col, st);
    } else if ((there >> kFirst) & kPart) {
      int number[kAb];
#pragma unroll
      for (int u = 0; u < kAb; ++u) {
        const int k = i + kFirst + u;
        number[u] = (there >> (kFirst + u)) & 1u ? (k < v.sink_units ? k : k + v.gap) : -1;
      }
      attend_units<D, NT, kFirst, kAb, true>(a, f, at, number, col, st);
    }
  });
}

// Natural logarithm of 2^m l; m is whole.  l's own power of two joins m first: both may
// be large where the result is not.
__device__ __forceinline__ float log_sum(float m, float l) {
  if (l == 0.f) return kNegInf;
  int e;
  const float part = frexpf(l, &e);
  return ((m + float(e)) + log2f(part)) * 0.6931471805599453f;
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
    a.lse[token * (int64_t(a.cache.kv_heads) * a.group) + h] = log_sum(m, l);
}

// Rows of a tile that see nothing.
template <typename T, int D>
__device__ __forceinline__ void store_nothing(const AttnArgs& a, const Seq& s, int row0, int rows,
                                              int head) {
  for (int e = threadIdx.x % 32; e < rows * (D / 4); e += 32)
    store_row<T>(a, s, row0 + e / (D / 4), head, e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f),
                 kNegInf, 0.f);
}

// ---- how the work is shared --------------------------------------------------
// An item is one tile of query rows with one kv head; it is counted as long as
// the longest of its sequence's tiles.  The warps of a grid that is resident at
// once take equal shares of all items, in one of two ways:
//   pieces: every item is cut into pieces of `piece` units and a share is a
//     piece: where that leaves no more pieces than warps, which have little each;
//   running: an item counts units + kItemUnits, and shares end wherever they do.
// A warp works alone: no barrier, and short items cost it little.  (With a CTA's
// four warps on one item and their results joined in shared memory, 16 requests
// of 1024 to 2048 tokens with 32 kv heads took 42 us, 36 like this.)  What a call's sequences are
// is known on the device only, so every CTA works the plan out from the lengths.
struct Plan {
  int piece;      // 0: running
  int64_t share;  // length of a share (pieces: 1)
  __device__ __forceinline__ int length(int units) const {  // of an item
    return piece ? max((units + piece - 1) / piece, 1) : units + kItemUnits;
  }
  // Unit at which a position of an item begins.
  __device__ __forceinline__ int unit(int units, int off) const {
    return piece ? min(off * piece, units) : max(off - kItemUnits, 0);
  }
};

struct Work {  // of one sequence
  Seq s;
  int rows, tiles, units;
  int64_t items;
};

template <int ROWS>
__device__ __forceinline__ Work work_of(const AttnArgs& a, int b) {
  Work w;
  w.s = seq_of(a, b);
  w.rows = w.s.count * a.group;
  w.tiles = (w.rows + ROWS - 1) / ROWS;
  w.units = span_of(a, w.s, 0, w.rows).units;
  w.items = int64_t(w.tiles) * a.cache.kv_heads;
  return w;
}

// The plan, and the place of the block's first share: the sequence that holds it
// and the work before that sequence.  `shared` has a row for each warp.
struct Place {
  int index;       // the batch's size when no sequence holds it
  int64_t before;
};

struct PlanShared {
  int64_t total[kWarps];
  float count[kWarps][kPieces];
  Place found;
};

template <int ROWS>
__device__ __forceinline__ Plan make_plan(const AttnArgs& a, PlanShared& sh, Place* place) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int shares = int(gridDim.x) * kWarps;
  // Every thread takes a run of sequences; most calls have one at most for each.
  const int run = (a.batch + kThreads - 1) / kThreads;
  const int first = min(int(threadIdx.x) * run, a.batch), last = min(first + run, a.batch);
  int64_t total = 0, items0 = 0;
  int units0 = 0;
  float count[kPieces] = {};  // exact up to 2^24, far above a grid
  for (int b = last - 1; b >= first; --b) {
    const Work w = work_of<ROWS>(a, b);
    items0 = w.items, units0 = w.units;
    total += w.items * (w.units + kItemUnits);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      count[i] +=
          float(w.items) * float(max((w.units + (kPiece << i) - 1) / (kPiece << i), 1));
  }
  auto sum = [&](int64_t v) {
#pragma unroll
    for (int d = 16; d; d /= 2) v += __shfl_xor_sync(~0u, v, d);
    return v;
  };
  const int64_t warp_total = sum(total);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
#pragma unroll
    for (int d = 16; d; d /= 2) count[i] += __shfl_xor_sync(~0u, count[i], d);
  }
  if (lane == 0) {
    sh.total[warp] = warp_total;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) sh.count[warp][i] = count[i];
  }
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += sh.total[w];
  Plan p;
  p.piece = 0;
  p.share = max(int64_t(kMinShare), all < (int64_t(1) << 31)
                                        ? int64_t((unsigned(all) + shares - 1) / unsigned(shares))
                                        : (all + shares - 1) / shares);
#pragma unroll
  for (int i = kPieces - 1; i >= 0; --i) {
    float pieces = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) pieces += sh.count[w][i];
    if (pieces <= float(shares) && int64_t(kPiece << i) <= p.share + kItemUnits)
      p.piece = kPiece << i;
  }
  if (p.piece) p.share = 1;
  // Running sum of the work as the plan counts it.
  const int64_t pos = p.share * kWarps * blockIdx.x;
  int64_t own = 0;
  if (run <= 1) {
    own = items0 * p.length(units0);
  } else {
    for (int b = first; b < last; ++b) {
      const Work w = work_of<ROWS>(a, b);
      own += w.items * p.length(w.units);
    }
  }
  int64_t v = own;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t u = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += u;
  }
  __syncthreads();
  if (lane == 31) sh.total[warp] = v;
  if (threadIdx.x == 0) sh.found = Place{a.batch, 0};
  __syncthreads();
  int64_t before = v - own;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) before += w < warp ? sh.total[w] : 0;
  if (pos >= before && pos < before + own) {
    int b = first;
    for (; b < last - 1; ++b) {
      const Work w = work_of<ROWS>(a, b);
      if (pos < before + w.items * p.length(w.units)) break;
      before += w.items * p.length(w.units);
    }
    sh.found = Place{b, before};
  }
  __syncthreads();
  *place = sh.found;
  return p;
}

// What a warp does at a time: units [u0, u1) of an item's part of the cache.
struct Segment {
  Seq s;
  Span v;
  int b, head, row0, rows;
  int u0, u1;
  int slot;  // place of its partial result in the workspace, -1: the result is whole
};

// An item that several shares have a piece of, for q4_join; rows = 0: none.  The
// pieces are in the slots first, then 2 k for the shares k = first / 2 + 1 .. last.
struct alignas(16) Joint {
  int token, row0;    // the sequence's first query token, the tile's first row
  int rows, head;
  int first, last;
};

// A warp's way through its share.
template <typename T, int D, int NT>
struct Walk {
  Plan plan;
  int64_t share;                    // its number
  int64_t begin, pos, end, before;  // positions; before: the sequence's first
  int b;
  bool told;                        // that an item of several pieces begins in the share

  __device__ __forceinline__ void put(const AttnArgs& a, int at, const Joint& joint) const {
    if (threadIdx.x % 32 == 0) a.joints[at] = joint;
  }

  // The next segment with units; rows that see nothing are written on the way.
  __device__ bool next(const AttnArgs& a, Segment& g) {
    constexpr int kRows = 8 * NT;
    while (pos < end && b < a.batch) {
      const Work w = work_of<kRows>(a, b);
      const int length = plan.length(w.units);
      const int64_t in = pos - before, total = w.items * length;
      if (in >= total) {
        before += total;
        ++b;
        continue;
      }
      int item, off;
      if (in < (int64_t(1) << 31)) {  // the common case: no 64-bit division
        item = int(unsigned(in) / unsigned(length));
        off = int(unsigned(in) - unsigned(item) * unsigned(length));
      } else {
        item = int(in / length);
        off = int(in - int64_t(item) * length);
      }
      const int n = int(min(int64_t(length - off), end - pos));
      const bool first = pos == begin;
      pos += n;
      g.head = item / w.tiles;
      g.row0 = (item % w.tiles) * kRows;
      g.rows = min(kRows, w.rows - g.row0);
      if (w.units == 0) {
        if (off == 0) {
          store_nothing<T, D>(a, w.s, g.row0, g.rows, g.head);
          if (a.joint_by_item) put(a, b * int(w.items) + item, Joint{});
        }
        continue;
      }
      const int u0 = plan.unit(w.units, off), u1 = plan.unit(w.units, off + n);
      if (u1 <= u0) continue;
      g.s = w.s;
      g.b = b;
      g.v = span_of(a, w.s, g.row0, g.rows);
      g.slot = u0 == 0 && u1 == w.units ? -1 : int(2 * share) + (first ? 0 : 1);
      g.u0 = min(u0, g.v.units);
      g.u1 = min(u1, g.v.units);
      if (u0 == 0) {  // the item's first piece: say who else has one
        Joint joint{};
        if (g.slot >= 0) {
          const int64_t end_of = before + int64_t(item + 1) * length - 1;
          joint = Joint{w.s.start, g.row0, g.rows, g.head, g.slot, int(end_of / plan.share)};
        }
        if (a.joint_by_item) put(a, b * int(w.items) + item, joint);
        else if (g.slot >= 0) put(a, int(share), joint), told = true;
      }
      return true;
    }
    if (!a.joint_by_item && !told) {
      put(a, int(share), Joint{});
      told = true;
    }
    return false;
  }
};

// ---- the kernel --------------------------------------------------------------

// Where the units of a warp's next steps are, one in every lane: block id and
// token run in the page.
struct Units {
  int id;
  int within;  // -1: there is no such unit
};

// The 32 units from number i of the tile's on.
__device__ __forceinline__ Units fetch_units(const AttnArgs& a, const Segment& g, int i) {
  Units f{0, -1};
  i += threadIdx.x % 32;
  if (i < g.u1) {
    const int n = i < g.v.sink_units ? i : i + g.v.gap;
    const int page = a.upp_shift >= 0 ? n >> a.upp_shift : n / a.upp;
    f.id = a.tables[int64_t(g.b) * a.table_stride + page];
    f.within = n - page * a.upp;
  }
  return f;
}

// Queues the copies of a step's units, those of lanes `at` ..., into a stage:
// 16-byte pieces lane, lane + 32, ... of each unit's codes, and one piece of the
// runs of scales and zeros.  Returns which units are there.
template <int D>
__device__ __forceinline__ uint32_t load_step(const AttnArgs& a, int head, const Units& f, int at,
                                              uint32_t dst) {
  using S = Shape<D>;
  constexpr int kU = S::kUnits;
  const int lane = threadIdx.x % 32;
  // The four lanes with lane % kU = u look at unit u.
  const int id = __shfl_sync(~0u, f.id, at + lane % kU);
  const int within = __shfl_sync(~0u, f.within, at + lane % kU);
  const bool real = within >= 0 && id >= 0 && id < a.cache.num_blocks;
  if (!real && within >= 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
  // A unit that is not there: its copies read nothing, from the first page.
  const int64_t page = (real ? id : 0) * a.cache.stride + int64_t(head) * a.cache.head_bytes;
  const int run = real ? within : 0;
  const int64_t code = page + run * S::kUnit;
  const uint32_t bits = __ballot_sync(~0u, real) & ((1u << kU) - 1u);
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int64_t offset = __shfl_sync(~0u, code, u) + 16 * lane;
    const int size = (bits >> u) & 1u ? 16 : 0;
#pragma unroll
    for (int i = 0; i < S::kUnit / 512; ++i) {
      // The pieces' places are permuted so that the fragments' reads meet no bank twice.
      const int c = lane + 32 * i;
      const int kc = D == 256 ? c ^ (4 * ((c >> 3) & 1)) : c;
      const int vc = c ^ (D == 64    ? 2 * ((c >> 3) & 1)
                          : D == 128 ? 2 * ((c >> 3) & 3)
                                     : 2 * ((c >> 4) & 3));
      copy16(dst + u * S::kUnit + 16 * kc, a.cache.pages[0] + offset + 512 * i, size);
      copy16(dst + (kU + u) * S::kUnit + 16 * vc, a.cache.pages[1] + offset + 512 * i, size);
    }
  }
  // Lane t * 4 kU + p * kU + u copies piece p of unit u's run of tensor t.
  if (lane < 8 * kU)
    copy16(dst + 2 * kU * S::kUnit + lane / (4 * kU) * S::kParams + 64 * (lane % kU) +
               16 * (lane / kU % 4),
           a.cache.pages[lane / (4 * kU) % 2] + page + a.cache.block_size * (D / 2) +
               run * 64 + 16 * (lane / kU % 4),
           real ? 16 : 0);
  return bits;
}

__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Writes a segment's result: a thread has D/8 dimensions of its columns' rows.
template <typename T, int D, int NT>
__device__ __forceinline__ void store_segment(const AttnArgs& a, const Segment& seg,
                                              WarpState<D, NT>& st) {
  const int lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      // Sums over the tokens of the eight threads with this column.
      float l = c ? st.l[n].y : st.l[n].x, z = st.z[n][c];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) {
        l += __shfl_xor_sync(~0u, l, d);
        z += __shfl_xor_sync(~0u, z, d);
      }
      const int r = 8 * n + 2 * j + c;
      if (r >= seg.rows) continue;
      const bool none = (c ? st.limit[n].y : st.limit[n].x) == kNegInf;
      const float m = none ? kNegInf : c ? -st.m[n].y : -st.m[n].x, mid = 7.5f * st.ps[n][c];
      if (seg.slot >= 0 && g == 0)
        a.part_ml[int64_t(seg.slot) * (8 * NT) + r] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < D / 16; d += 2) {
        float4 o;
        o.x = fmaf(st.o[n][d][c], 16777216.f, -mid) + z;
        o.y = fmaf(st.o[n][d][2 + c], 1048576.f, -mid) + z;
        o.z = fmaf(st.o[n][d + 1][c], 16777216.f, -mid) + z;
        o.w = fmaf(st.o[n][d + 1][2 + c], 1048576.f, -mid) + z;
        const int at = g * (D / 8) + 2 * d;
        if (seg.slot >= 0)
          *reinterpret_cast<float4*>(a.part_o + (int64_t(seg.slot) * (8 * NT) + r) * D + at) = o;
        else
          store_row<T>(a, seg.s, seg.row0 + r, seg.head, at, o, m, l);
      }
    }
}

// What bounds it: the bytes of the cache where sequences are long (128 requests of
// 4096 to 8192 tokens, 8 kv heads: 166 us, 5.2 TB/s, 80% of the card's copy rate)
// beside the latency of its two warps a scheduler (216 instructions for 16 tokens of a
// head, 88 of them unpacking, fill half of the issue slots), and what a launch, an
// item and the join cost where they are short.  Each warp takes its
// share's segments one after the other, their units in steps through its own ring of two cp.async stages; during a segment's last
// step the next one's first is on its way already.  Segments that end or begin
// inside an item leave a partial result in the workspace (at most two for a
// warp), which q4_join brings together.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, 8 * NT))
    q4_attend(const __grid_constant__ AttnArgs a) {
  using S = Shape<D>;
  constexpr int kRows = 8 * NT, kU = S::kUnits;
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ PlanShared plan_shared;
  __shared__ uint2 fragments[NT == 1 ? 1 : kWarps][NT == 1 ? 1 : NT * (D / 16) * 32];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Walk<T, D, NT> walk;
  {
    Place place;
    walk.plan = make_plan<kRows>(a, plan_shared, &place);
    walk.b = place.index;
    walk.before = place.before;
    walk.share = int64_t(blockIdx.x) * kWarps + warp;
    walk.begin = walk.pos = walk.plan.share * walk.share;
    walk.end = walk.begin + walk.plan.share;
    walk.told = false;
  }
  Segment seg, next;
  if (!walk.next(a, seg)) return;
  const uint32_t ring = uint32_t(__cvta_generic_to_shared(shared)) + warp * S::kWarpBytes;
  const LaneAddress lane_at = lane_address<D>(ring, lane / 4, lane % 4);
  uint32_t stage = 0, bits = 0;  // the step to take next: its stage, which of its units are there
  bool loaded = false;           // its copies are on their way
  Units now = fetch_units(a, seg, seg.u0), next_units{0, -1};
  Fragments<D, NT> f;
  f.shared = &fragments[NT == 1 ? 0 : warp][NT == 1 ? 0 : lane];
  while (true) {
    if (!loaded && seg.u0 < seg.u1) {
      bits = load_step<D>(a, seg.head, now, 0, ring + stage);
      commit();
    }
    loaded = false;
    const bool more = walk.next(a, next);
    if (more) next_units = fetch_units(a, next, next.u0);
    Units later = fetch_units(a, seg, seg.u0 + 32);
    Columns<NT> col;
    load_queries<T, D, NT>(a, seg.s, seg.row0, seg.rows, seg.head, f, col);
    WarpState<D, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      st.m[n] = st.l[n] = make_float2(0.f, 0.f);
      st.limit[n] = make_float2(kNegInf, kNegInf);
      st.z[n][0] = st.z[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st.ps[n][i] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[n][d][i] = 0.f;
      }
    }
    // Units [plain_from, plain_to) need no mask: behind no row, and inside every
    // row's window.
    const Span& v = seg.v;
    const int plain_from = max(v.sink_units, (max(v.p_hi - a.window + 1, 0) + 15) / 16 - v.gap);
    const int plain_to = (v.p_lo + 1) / 16 - v.gap;
    int at = 0;  // lane that has the step's first unit
    for (int i = seg.u0; i < seg.u1; i += kU) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      uint32_t next_bits = 0;
      const uint32_t to = ring + (stage ^ uint32_t(S::kStage));
      at = (at + kU) % 32;
      if (i + kU < seg.u1) {
        if (at == 0) {
          now = later;
          later = fetch_units(a, seg, i + kU + 32);
        }
        next_bits = load_step<D>(a, seg.head, now, at, to);
      } else if (more && next.u0 < next.u1) {
        next_bits = load_step<D>(a, next.head, next_units, 0, to);
        loaded = true;
      }
      commit();
      // Bits of the step's units that are there and need no mask.
      const int low = min(max(plain_from - i, 0), kU), high = min(max(plain_to - i, 0), kU);
      const uint32_t plain = bits & ((1u << high) - 1u) & ~((1u << low) - 1u);
      attend_step<D, NT>(a, f, lane_at + stage, bits, plain, i, col, v, st);
      __syncwarp();
      stage ^= uint32_t(S::kStage);
      bits = next_bits;
    }
    store_segment<T, D, NT>(a, seg, st);
    if (!more) break;
    seg = next;
    now = next_units;
  }
}

// ---- the join of partial results ---------------------------------------------

// Weight of a piece with (reference point, sum) ml against the largest of all, m: a
// piece without a finite score counts for nothing, unless a NaN is in it.
__device__ __forceinline__ float piece_weight(float2 ml, float m) {
  return ml.x == kNegInf ? (ml.y == ml.y ? 0.f : ml.y) : ex2(ml.x - m);
}

// Sums the pieces of 1 << kLg rows of a joint that fall to warp `part` of `parts`.  What
// bounds it is the latency of its loads, so a warp has 16 (D = 256: 8) of them in
// flight: slot q is row q & kMask of the piece q >> kLg further on.  Lane q has the
// row's reference point and sum.
template <int D, int kLg>
__device__ __forceinline__ void join_pieces(const AttnArgs& a, const Joint& x, int kRows, int r0,
                                            int rows, int part, int parts, float& m, float& l,
                                            float4 (&o)[1 << kLg][(D + 127) / 128]) {
  constexpr int kParts = (D + 127) / 128, kMask = (1 << kLg) - 1;
  constexpr int kSlots = D == 256 ? 8 : 16, kPer = kSlots >> kLg;  // pieces of a round
  const int lane = threadIdx.x % 32, count = x.last - x.first / 2 + 1;
  auto slot = [&](int k) { return int64_t(k ? 2 * (x.first / 2 + k) : x.first) * kRows; };
  const int r = r0 + min(lane & kMask, rows - 1);
  m = kNegInf;
  for (int k = lane >> kLg; k < count; k += 32 >> kLg) m = fmaxf(m, a.part_ml[slot(k) + r].x);
#pragma unroll
  for (int d = 1 << kLg; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  l = 0.f;
#pragma unroll
  for (int q = 0; q <= kMask; ++q)
#pragma unroll
    for (int i = 0; i < kParts; ++i) o[q][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = part * kPer; k0 < count; k0 += parts * kPer) {
    const int mine = k0 + ((lane % kSlots) >> kLg);
    const float2 ml = mine < count ? a.part_ml[slot(mine) + r] : make_float2(kNegInf, 0.f);
    float4 v[kSlots][kParts];
#pragma unroll
    for (int q = 0; q < kSlots; ++q) {
      const int row = r0 + min(q & kMask, rows - 1);
      const float* from = a.part_o + (slot(min(k0 + (q >> kLg), count - 1)) + row) * D;
#pragma unroll
      for (int i = 0; i < kParts; ++i)
        v[q][i] = 128 * i + 4 * lane < D
                      ? *reinterpret_cast<const float4*>(from + 128 * i + 4 * lane)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float f = piece_weight(ml, m);
    float add = f * ml.y;
#pragma unroll
    for (int d = 1 << kLg; d < kSlots; d *= 2) add += __shfl_xor_sync(~0u, add, d);
    l += add;
#pragma unroll
    for (int q = 0; q < kSlots; ++q) {
      const float fq = __shfl_sync(~0u, f, q);
      // Whatever the weight, which may have underflowed: a piece's NaN is the row's.
      if (k0 + (q >> kLg) < count) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          float4& s = o[q & kMask][i];
          s.x = fmaf(fq, v[q][i].x, s.x), s.y = fmaf(fq, v[q][i].y, s.y);
          s.z = fmaf(fq, v[q][i].z, s.z), s.w = fmaf(fq, v[q][i].w, s.w);
        }
      }
    }
  }
}

template <typename T, int D, int kLg>
__device__ __forceinline__ void join_rows(const AttnArgs& a, const Joint& x, int kRows, int r0,
                                          int rows) {
  const int lane = threadIdx.x % 32;
  float m, l;
  float4 o[1 << kLg][(D + 127) / 128];
  join_pieces<D, kLg>(a, x, kRows, r0, rows, 0, 1, m, l, o);
#pragma unroll
  for (int q = 0; q < 1 << kLg; ++q) {
    const float mq = __shfl_sync(~0u, m, q), lq = __shfl_sync(~0u, l, q);
#pragma unroll
    for (int i = 0; i < (D + 127) / 128; ++i)
      if (q < rows && 128 * i + 4 * lane < D)
        store_row<T>(a, Seq{x.token, 0, 0}, x.row0 + r0 + q, x.head, 128 * i + 4 * lane, o[q][i],
                     mq, lq);
  }
}

// Joins the partial results of items that several warps shared; the pieces are
// summed in an order that does not vary.  kByItem: a block for each row of each
// item, its warps share the pieces; otherwise the block's warps take the rows of
// the items that begin in its shares.
template <typename T, int D, int NT, bool kByItem>
__global__ void __launch_bounds__(kJoinThreads) q4_join(const __grid_constant__ AttnArgs a,
                                                        int shares) {
  constexpr int kRows = 8 * NT, kParts = (D + 127) / 128;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if constexpr (!kByItem) {
    // Two rows at a time for a warp, so that eight of their pieces are in flight.
    const int groups = min((a.group * (a.starts ? kRows : a.queries) + 1) / 2, kRows / 2);
    for (int task = warp; task < kJoinWarps * groups; task += kJoinWarps) {
      const int at = blockIdx.x * kJoinWarps + task / groups, r0 = 2 * (task % groups);
      if (at >= shares) return;
      const Joint x = a.joints[at];
      if (x.rows - r0 >= 2) join_rows<T, D, 1>(a, x, kRows, r0, 2);
      else if (x.rows > r0) join_rows<T, D, 0>(a, x, kRows, r0, 1);
    }
  } else {
    __shared__ float4 part[kJoinWarps][kParts][32];
    __shared__ float part_l[kJoinWarps];
    const Joint x = a.joints[blockIdx.x / kRows];
    const int r = blockIdx.x % kRows;
    if (r >= x.rows) return;
    float m, l;
    float4 o[1][kParts];
    join_pieces<D, 0>(a, x, kRows, r, 1, warp, kJoinWarps, m, l, o);
#pragma unroll
    for (int i = 0; i < kParts; ++i) part[warp][i][lane] = o[0][i];
    if (lane == 0) part_l[warp] = l;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int k = 1; k < kJoinWarps; ++k) {
      l += part_l[k];
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const float4 v = part[k][i][lane];
        o[0][i].x += v.x, o[0][i].y += v.y, o[0][i].z += v.z, o[0][i].w += v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i)
      if (128 * i + 4 * lane < D)
        store_row<T>(a, Seq{x.token, 0, 0}, x.row0 + r, x.head, 128 * i + 4 * lane, o[0][i],
                     m, __shfl_sync(~0u, l, 0));
  }
}

}  // namespace q4
}  // namespace kvx
