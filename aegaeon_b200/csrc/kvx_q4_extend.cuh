// Attention of many query rows over the 4-bit paged cache (pieces of prompts).
//
// With enough rows the products bound it, so they run on the fifth-generation
// tensor cores: a CTA takes 128 rows (query tokens x the heads of a kv head) and
// walks the cache in blocks of 128 tokens.  The codes go to shared memory as fp16
// integers c - 8, exact; S = Q C^T and O += P' C accumulate in tensor memory.  As in
// kvx_q4_attention.cuh the scales join in 32 bits: on the scores for K, on the
// probabilities for V,
//   q . k_j       = s_j (q . (c_j - 8)) + (z_j + 8 s_j) sum(q)
//   sum_j p_j v_j = sum_j (p_j s'_j) (c'_j - 8) + sum_j p_j (z'_j + 8 s'_j).
// P' = p s' is rounded to fp16 once (2^-11 of it) and written over the scores it came
// from; the row's reference point is kept so that it stays below 2^14.
//
// The threads unpack the codes, so they and the softmax share the issue slots: two
// CTAs of 256 threads on an SM overlap one's softmax with the other's products.
#pragma once

#include "kvx_q4_attention.cuh"

namespace kvx {
namespace q4 {

constexpr int kExtendThreads = 256;
constexpr int kExtendRows = 128;   // rows of a tile: M of the products
constexpr int kExtendTokens = 128; // tokens of a block
constexpr int kPanel = 128 * 128;  // bytes of 64 dimensions of 128 rows or tokens

template <int D>
struct ExtendShape {
  static constexpr int kPanels = D / 64;
  static constexpr int kMatrix = kPanels * kPanel;
  static constexpr int kShared = 3 * kMatrix + 1024;  // Q, K, V; aligned to 1024 bytes
  static constexpr int kColumns = 256;                // of tensor memory: S (128), O (D)
};

struct ExtendShared {
  float ks[kExtendTokens], kz[kExtendTokens];  // K: scale, zero + 8 scale
  float vs[kExtendTokens], vz[kExtendTokens];  // V
  float pair[2][kExtendRows];                  // what two threads of a row tell each other
  float pair2[2][kExtendRows];
  float top[4];                                // largest V scale, by warp
  int number[kExtendTokens / 16];              // the block's units, -1: not there
  alignas(8) uint64_t done_s, done_o;          // the products' barriers
  uint32_t tmem;
  int failed;
  int64_t scan[kExtendThreads / 32];
  Place found;
};

__device__ __forceinline__ uint32_t smem_of(const void* p) {
  return uint32_t(__cvta_generic_to_shared(p));
}

// Waits for a phase of a barrier, two seconds at most.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t phase) {
  uint64_t end = 0;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{.reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;}"
        : "=r"(done)
        : "r"(smem_of(bar)), "r"(phase)
        : "memory");
    if (done) return true;
    uint64_t now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (end == 0) end = now + 2000000000ull;
    else if (now > end) return false;
  }
}

// Shared-memory matrix descriptor, 128-byte swizzle: start address, strides (in
// bytes) of the leading and the other dimension.
__device__ __forceinline__ uint64_t matrix_desc(uint32_t address, uint32_t leading,
                                                uint32_t stride) {
  return uint64_t((address & 0x3ffffu) >> 4) | uint64_t((leading >> 4) & 0x3fffu) << 16 |
         uint64_t((stride >> 4) & 0x3fffu) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}

// fp16 x fp16 with sums in fp32; `mn` : B has its N dimension contiguous.
__host__ __device__ constexpr uint32_t product_desc(int m, int n, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | uint32_t(n / 8) << 17 | uint32_t(m / 16) << 24;
}

__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                           bool add) {
  asm volatile(
      "{.reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d),
      "l"(a), "l"(b), "r"(desc), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc,
                                           bool add) {
  asm volatile(
      "{.reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d),
      "r"(a), "l"(b), "r"(desc), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void products_done(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_of(bar))
      : "memory");
}

#define KVX_OUT4(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3])
#define KVX_IN4(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3])

// 32 columns of a thread's row from or to tensor memory.
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : KVX_OUT4(x, 0), KVX_OUT4(x, 4), KVX_OUT4(x, 8), KVX_OUT4(x, 12), KVX_OUT4(x, 16),
        KVX_OUT4(x, 20), KVX_OUT4(x, 24), KVX_OUT4(x, 28)
      : "r"(at));
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::KVX_IN4(
          x, 0),
      KVX_IN4(x, 4), KVX_IN4(x, 8), KVX_IN4(x, 12), KVX_IN4(x, 16), KVX_IN4(x, 20), KVX_IN4(x, 24),
      KVX_IN4(x, 28), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_loaded() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_stored() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void shared_written() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Eight codes as fp16 integers c - 8, in the order 0 4 1 5 2 6 3 7 of the word's
// nibbles: 1024 + c stands in the low bits of an fp16 of 1024, 64 + c in the
// next four of one of 64.
__device__ __forceinline__ uint4 unpack(uint32_t w) {
  const __half2 low = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));   // 1032
  const __half2 high = __halves2half2(__ushort_as_half(0x5480), __ushort_as_half(0x5480));  // 72
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = i < 2 ? w : w >> 8;
    const uint32_t bits = i % 2 ? (s & kOdd) | 0x54005400u : (s & kEven) | 0x64006400u;
    __half2 h;
    __builtin_memcpy(&h, &bits, 4);
    h = __hsub2(h, i % 2 ? high : low);
    __builtin_memcpy(&r[i], &h, 4);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// One thread's codes of a token (D/4 bytes) into a swizzled matrix: token t, the
// D/2 dimensions of half `h`.
template <int D>
__device__ __forceinline__ void store_codes(uint32_t matrix, int t, int h,
                                            const uint4 (&raw)[D / 64]) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint32_t w = i % 4 == 0 ? raw[i / 4].x : i % 4 == 1 ? raw[i / 4].y
                       : i % 4 == 2 ? raw[i / 4].z : raw[i / 4].w;
    const int chunk = h * (D / 16) + i;  // of eight dimensions
    const uint32_t at = matrix + (chunk / 8) * kPanel + t * 128 + (((chunk % 8) ^ (t & 7)) << 4);
    const uint4 v = unpack(w);
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
  }
}

// A thread's part of a block on its way: the codes of token t of K and V, half h,
// and (scale, zero) of token t of tensor h.
template <int D>
struct Block {
  uint4 key[D / 64], value[D / 64];
  uint32_t param;
};

template <typename T, int D>
__global__ void __launch_bounds__(kExtendThreads, 2) q4_extend(const __grid_constant__ AttnArgs a,
                                                               int tiles_most) {
  using S = ExtendShape<D>;
  extern __shared__ uint8_t dynamic[];
  __shared__ ExtendShared sh;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int t = tid % 128, h = tid / 128;  // row or token, half
  // The tile: the longest first, the kv heads of a tile side by side.
  const int heads = a.cache.kv_heads;
  const int tile_at = tiles_most - 1 - int(blockIdx.x) / heads, head = int(blockIdx.x) % heads;
  {  // its sequence
    const int run = (a.batch + kExtendThreads - 1) / kExtendThreads;
    const int first = min(tid * run, a.batch), last = min(first + run, a.batch);
    int64_t own = 0;
    for (int b = first; b < last; ++b)
      own += (seq_of(a, b).count * a.group + kExtendRows - 1) / kExtendRows;
    int64_t v = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t u = __shfl_up_sync(~0u, v, d);
      if (lane >= d) v += u;
    }
    if (lane == 31) sh.scan[warp] = v;
    if (tid == 0) sh.found = Place{a.batch, 0}, sh.failed = 0;
    __syncthreads();
    int64_t before = v - own;
    for (int w = 0; w < warp; ++w) before += sh.scan[w];
    if (tile_at >= before && tile_at < before + own) {
      int b = first;
      for (; b < last - 1; ++b) {
        const int n = (seq_of(a, b).count * a.group + kExtendRows - 1) / kExtendRows;
        if (tile_at < before + n) break;
        before += n;
      }
      sh.found = Place{b, before};
    }
    __syncthreads();
  }
  const int b = sh.found.index;
  if (b >= a.batch) return;  // the whole block
  const Seq s = seq_of(a, b);
  const int row0 = (tile_at - int(sh.found.before)) * kExtendRows;
  const int rows = min(kExtendRows, s.count * a.group - row0);
  const Span v = span_of(a, s, row0, rows);
  const int blocks = (v.units * 16 + kExtendTokens - 1) / kExtendTokens;

  const uint32_t base = (smem_of(dynamic) + 1023u) & ~1023u;
  const uint32_t q_at = base, k_at = base + S::kMatrix, v_at = base + 2 * S::kMatrix;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_of(&sh.tmem)),
                 "n"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_of(&sh.done_s)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_of(&sh.done_o)) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }

  // Where the thread's token of a block is; the id is looked up a block ahead.
  auto fetch_id = [&](int block, int& id, int& within) {
    const int i = block * (kExtendTokens / 16) + t / 16;
    id = 0;
    within = -1;
    if (i < v.units) {
      const int n = i < v.sink_units ? i : i + v.gap;
      const int page = a.upp_shift >= 0 ? n >> a.upp_shift : n / a.upp;
      id = a.tables[int64_t(b) * a.table_stride + page];
      within = (n - page * a.upp) * 16 + t % 16;
    }
  };
  auto fetch = [&](int id, int within, Block<D>& r) {
    const bool real = within >= 0 && id >= 0 && id < a.cache.num_blocks;
    if (!real && within >= 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
    r.param = 0;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) r.key[i] = r.value[i] = make_uint4(0u, 0u, 0u, 0u);
    if (real) {
      const int64_t page = id * a.cache.stride + int64_t(head) * a.cache.head_bytes;
      const int64_t at = page + within * (D / 2) + h * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        r.key[i] = *reinterpret_cast<const uint4*>(a.cache.pages[0] + at + 16 * i);
        r.value[i] = *reinterpret_cast<const uint4*>(a.cache.pages[1] + at + 16 * i);
      }
      r.param = *reinterpret_cast<const uint32_t*>(a.cache.pages[h] + page +
                                                   a.cache.block_size * (D / 2) + within * 4);
    }
    return real;
  };
  int id, within;
  fetch_id(0, id, within);
  Block<D> raw;
  bool there = blocks > 0 && fetch(id, within, raw);
  fetch_id(1, id, within);

  // The query rows: thread (row t, half h) has D/2 of its dimensions.  Scaled by a
  // power of two as in load_queries(), in the order that unpack() gives the codes.
  float factor, qsum;
  int pos = -1;
  {
    const bool real = t < rows;
    const T* from = static_cast<const T*>(a.query);
    if (real) {
      const int token = (row0 + t) / a.group, g = (row0 + t) - token * a.group;
      pos = s.len - s.count + token;
      from += int64_t(s.start + token) * a.q_token + int64_t(head * a.group + g) * a.q_head +
              h * (D / 2);
    }
    T x[D / 16][8];
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      if (!real) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = from_float<T>(0.f);
      } else if (a.q_vec) {
        const uint4 u = *reinterpret_cast<const uint4*>(from + 8 * i);
        __builtin_memcpy(x[i], &u, 16);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = from[8 * i + k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(to_float(x[i][k])));
    }
    sh.pair[h][t] = top;
    __syncthreads();
    top = fmaxf(sh.pair[0][t], sh.pair[1][t]);
    const int e = min(max(int(__float_as_uint(top) >> 23), 20), 250);
    float up = top > 0.f ? __uint_as_float(uint32_t(min(127 + 14 + 127 - e, 240)) << 23) : 1.f;
    factor = fmaxf(a.scale_log2 / up, 1e-37f);  // never 0: hidden scores are -inf
    up *= a.sign;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float y0 = to_float(x[i][k]) * up, y1 = to_float(x[i][k + 4]) * up;
        sum += y0 + y1;
        const __half2 p = __floats2half2_rn(y0, y1);
        __builtin_memcpy(&r[k], &p, 4);
      }
      const int chunk = h * (D / 16) + i;
      const uint32_t at = q_at + (chunk / 8) * kPanel + t * 128 + (((chunk % 8) ^ (t & 7)) << 4);
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]),
                   "r"(r[2]), "r"(r[3])
                   : "memory");
    }
    sh.pair2[h][t] = sum;
    __syncthreads();  // the barriers and the tensor memory's address are there, too
    qsum = sh.pair2[0][t] + sh.pair2[1][t];
  }
  const uint32_t tmem = sh.tmem;
  const uint32_t own_lanes = uint32_t(32 * (warp % 4)) << 16;
  const uint32_t s_cols = tmem, o_cols = tmem + 128;
  const uint32_t s_mine = s_cols + own_lanes + 64 * h, o_mine = o_cols + own_lanes + (D / 2) * h;

  float minus_r = 0.f, limit = kNegInf, l = 0.f, z = 0.f;  // reference point, sums of the row's half
  bool waited = true;  // no wait has run out
  for (int block = 0; block < blocks; ++block) {
    const uint32_t phase = block & 1;
    // K codes, and every token's scales and zeros.  A token that no row sees counts 0.
    store_codes<D>(k_at, t, h, raw.key);
    {
      const int i = block * (kExtendTokens / 16) + t / 16;
      const int n = i < v.sink_units ? i : i + v.gap, token = n * 16 + t % 16;
      const bool seen = there && token <= v.p_hi && (token > v.p_lo - a.window || token < a.sinks);
      const float2 p = seen ? half2_at(raw.param) : make_float2(0.f, 0.f);
      float* scale = h ? sh.vs : sh.ks;
      float* zero = h ? sh.vz : sh.kz;
      scale[t] = p.x;
      zero[t] = fmaf(8.f, p.x, p.y);
      if (t % 16 == 0 && h == 0) sh.number[t / 16] = there ? n : -1;
      if (h) {
        float top = fabsf(p.x);
#pragma unroll
        for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        if (lane == 0) sh.top[warp - 4] = top;
      }
    }
    shared_written();
    if (block > 0 && waited) waited = wait_phase(&sh.done_o, phase ^ 1);  // P and V are read
    tmem_before();
    __syncthreads();
    if (tid == 0) {
      tmem_after();
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t step = (k / 4) * kPanel + (k % 4) * 32;
        product_ss(s_cols, matrix_desc(q_at + step, 16, 1024), matrix_desc(k_at + step, 16, 1024),
                   product_desc(kExtendRows, kExtendTokens, false), k > 0);
      }
      products_done(&sh.done_s);
    }
    // While they run: the V codes, and the next block's loads.
    store_codes<D>(v_at, t, h, raw.value);
    shared_written();
    if (block + 1 < blocks) {
      there = fetch(id, within, raw);
      fetch_id(block + 2, id, within);
    }
    const float vtop = fmaxf(fmaxf(sh.top[0], sh.top[1]), fmaxf(sh.top[2], sh.top[3]));
    const float e_top = vtop > 0.f ? float(int(__float_as_uint(vtop) >> 23) - 126) : -24.f;
    const int first = block * (kExtendTokens / 16);
    bool plain = sh.number[0] >= 0 && first >= v.sink_units &&
                 (first + v.gap) * 16 > v.p_hi - a.window &&
                 (first + v.gap) * 16 + kExtendTokens - 1 <= v.p_lo;
#pragma unroll
    for (int u = 1; u < kExtendTokens / 16; ++u) plain = plain && sh.number[u] >= 0;

    if (waited) waited = wait_phase(&sh.done_s, phase);
    tmem_after();
    // Scores of the thread's row with 64 tokens, in the raw products' unit.
    float y[64];
    float top = kNegInf;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      uint32_t x[32];
      tmem_load(s_mine + 32 * part, x);
      tmem_loaded();
      const float* ks = sh.ks + 64 * h + 32 * part;
      const float* kz = sh.kz + 64 * h + 32 * part;
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 sc = *reinterpret_cast<const float4*>(ks + c);
        const float4 zc = *reinterpret_cast<const float4*>(kz + c);
        const float2 y0 = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])),
                               make_float2(sc.x, sc.y), mul2(make_float2(zc.x, zc.y), both(qsum)));
        const float2 y1 = fma2(make_float2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])),
                               make_float2(sc.z, sc.w), mul2(make_float2(zc.z, zc.w), both(qsum)));
        y[32 * part + c] = y0.x, y[32 * part + c + 1] = y0.y;
        y[32 * part + c + 2] = y1.x, y[32 * part + c + 3] = y1.y;
      }
    }
    if (!plain) {
#pragma unroll
      for (int c = 0; c < 64; ++c) {
        const int n = sh.number[4 * h + c / 16], token = n * 16 + c % 16;
        const bool seen = n >= 0 && token <= pos && (token > pos - a.window || token < a.sinks);
        y[c] = seen ? y[c] : kNegInf;
      }
    }
#pragma unroll
    for (int c = 0; c < 64; c += 2) top = max3(top, y[c], y[c + 1]);
    sh.pair[h][t] = top;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + warp % 4) : "memory");  // the row's two warps
    top = fmaxf(top, sh.pair[h ^ 1][t]) * factor;
    // Move the reference point where P' would pass 2^14.
    if (__any_sync(~0u, top + e_top + minus_r > limit)) {
      float f = 1.f;
      if (top + e_top + minus_r > limit) {
        const float to = -(top + e_top - 6.f);
        if (limit != kNegInf) f = ex2(to - minus_r);
        minus_r = to;
        limit = 14.f;
      }
      l *= f;
      z *= f;
      if (block > 0) {
#pragma unroll
        for (int part = 0; part < D / 64; ++part) {
          uint32_t x[32];
          tmem_load(o_mine + 32 * part, x);
          tmem_loaded();
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * f);
          tmem_store(o_mine + 32 * part, x);
        }
      }
    }
    {
      uint32_t p16[32];
      float2 l2 = make_float2(0.f, 0.f), z2 = make_float2(0.f, 0.f);
      const float* vs = sh.vs + 64 * h;
      const float* vz = sh.vz + 64 * h;
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 sc = *reinterpret_cast<const float4*>(vs + c);
        const float4 zc = *reinterpret_cast<const float4*>(vz + c);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          float2 p = fma2(make_float2(y[c + k], y[c + k + 1]), both(factor), both(minus_r));
          p.x = ex2(p.x), p.y = ex2(p.y);
          l2 = add2(l2, p);
          const float2 zz = k ? make_float2(zc.z, zc.w) : make_float2(zc.x, zc.y);
          float2 w = mul2(p, k ? make_float2(sc.z, sc.w) : make_float2(sc.x, sc.y));
          float2 zn = fma2(p, zz, z2);
          if (!plain) {  // a hidden token's scale and zero may be anything
            if (p.x == 0.f) w.x = 0.f, zn.x = z2.x;
            if (p.y == 0.f) w.y = 0.f, zn.y = z2.y;
          }
          z2 = zn;
          const __half2 half = __floats2half2_rn(w.x, w.y);
          __builtin_memcpy(&p16[(c + k) / 2], &half, 4);
        }
      }
      l += l2.x + l2.y;
      z += z2.x + z2.y;
      tmem_store(s_mine, p16);
    }
    tmem_stored();
    tmem_before();
    __syncthreads();
    if (tid == 0) {
      tmem_after();
#pragma unroll
      for (int k = 0; k < kExtendTokens / 16; ++k)
        product_ts(o_cols, s_cols + (k / 4) * 64 + (k % 4) * 8,
                   matrix_desc(v_at + k * 2048, kPanel, 1024), product_desc(kExtendRows, D, true),
                   block > 0 || k > 0);
      products_done(&sh.done_o);
    }
  }
  if (blocks > 0 && waited) waited = wait_phase(&sh.done_o, (blocks - 1) & 1);
  if (!waited) atomicExch(&g_q4_status, 8 /* KVX_ERR_DEVICE_TIMEOUT */);
  tmem_after();
  sh.pair[h][t] = l;
  sh.pair2[h][t] = z;
  __syncthreads();
  l = sh.pair[0][t] + sh.pair[1][t];
  z = sh.pair2[0][t] + sh.pair2[1][t];
  const float by = l == 0.f ? 0.f : 1.f / l;
  const int64_t token = s.start + (row0 + t) / a.group;
  const int head_out = head * a.group + (row0 + t) % a.group;
  T* to = static_cast<T*>(a.out) + token * a.o_token + int64_t(head_out) * a.o_head + h * (D / 2);
#pragma unroll
  for (int part = 0; part < D / 64; ++part) {
    uint32_t x[32];
    if (blocks > 0) {
      tmem_load(o_mine + 32 * part, x);
      tmem_loaded();
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c) x[c] = 0u;
    }
    if (t < rows) {
#pragma unroll
      for (int c = 0; c < 32; c += 8) {
        T r[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)  // dimension k is column 0 2 4 6 1 3 5 7 of the eight
          r[k] = from_float<T>((__uint_as_float(x[c + (k < 4 ? 2 * k : 2 * k - 7)]) + z) * by);
        if (a.o_vec16) {
          uint4 w;
          __builtin_memcpy(&w, r, 16);
          *reinterpret_cast<uint4*>(to + 32 * part + c) = w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) to[32 * part + c + k] = r[k];
        }
      }
    }
  }
  if (a.lse && h == 0 && t < rows)
    a.lse[token * (int64_t(heads) * a.group) + head_out] =
        l == 0.f ? kNegInf : (log2f(l) - minus_r) * 0.6931471805599453f;
  tmem_before();
  __syncthreads();
  if (warp == 0) {
    tmem_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(S::kColumns));
  }
}

}  // namespace q4
}  // namespace kvx
