// Attention of many query rows over the 4-bit paged cache (pieces of prompts).
//
// With enough rows the products bound it, so they run on the fifth-generation
// tensor cores.  A CTA takes two tiles of 128 rows (query tokens x the heads of a kv
// head) and walks the cache in blocks of 128 tokens.  The codes go to shared memory
// as fp16 integers c - 8, exact; S = Q C^T and O += P' C accumulate in tensor memory.
// As in kvx_q4_attention.cuh the scales join in 32 bits: on the scores for K, on the
// probabilities for V,
//   q . k_j       = s_j (q . (c_j - 8)) + (z_j + 8 s_j) sum(q)
//   sum_j p_j v_j = sum_j (p_j s'_j) (c'_j - 8) + sum_j p_j (z'_j + 8 s'_j).
// P' = p s' is rounded to fp16 once (2^-11 of it) and written over the scores it came
// from; the row's reference point follows its largest P', so that this stays between
// 2^5 and 2^14.1.
//
// Warps have one task each: four for a tile's softmax (a thread a row), four unpack
// the codes, one issues the products.  While one tile's softmax runs, the tensor
// cores work on the other, and both share the unpacked codes.  (128-row CTAs whose
// threads did everything in turn, two to an SM, reached 338 TFLOP/s on 1024-token
// pieces behind 7168 tokens, waiting for loads and for one another; this form 443,
// a quarter of the products' rate.  What bounds it is the softmax: a row's 128
// scores of a block go through one thread, and the two tiles' products, a fifth of
// the time, wait for them in turn.)
#pragma once

#include "kvx_q4_attention.cuh"

namespace kvx {
namespace q4 {

// Sixteen warps, the last three of them idle: 128 registers a thread.  With a
// seventeenth the softmax had 96, and what it spilled did not fit the few
// kilobytes of L1 that the matrices leave.
constexpr int kExtendThreads = 512;
constexpr int kTileRows = 128;     // rows of a tile: M of the products
constexpr int kExtendRows = 256;   // of a CTA
constexpr int kExtendTokens = 128; // tokens of a block
constexpr int kPanel = 128 * 128;  // bytes of 64 dimensions of 128 rows or tokens

template <int D>
struct ExtendShape {
  static constexpr int kMatrix = D / 64 * kPanel;
  static constexpr int kShared = 6 * kMatrix + 1024;  // 2 Q, 2 K, 2 V; aligned to 1024 bytes
  static constexpr int kColumns = 512;                // of tensor memory: 2 S (128), 2 O (D)
};

struct ExtendShared {
  float ks[2][kExtendTokens], kz[2][kExtendTokens];  // K: scale, zero + 8 scale, by scale_part
  float vs[2][kExtendTokens], vz[2][kExtendTokens];  // V
  float top[2][4];                           // largest V scale, by warp
  int number[2][kExtendTokens / 16];         // the block's units, -1: not there
  // Barriers.  By stage: unpacked, read; by tile: scores there, weights there,
  // output added; queries there; all products through.
  alignas(8) uint64_t k_full[2], k_free[2], v_full[2], v_free[2];
  uint64_t s_full[2], p_full[2], o_full[2], q_full, drained;
  uint32_t tmem;
  int cut;  // a wait has run out
  int64_t scan[kExtendThreads / 32];
  Place found;
};

__device__ __forceinline__ uint32_t smem_of(const void* p) {
  return uint32_t(__cvta_generic_to_shared(p));
}

// Waits for a phase of a barrier, about two seconds at most (by the SM's clock:
// reading the global timer takes longer than most waits here).
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t phase) {
  int64_t begin = 0;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{.reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;}"
        : "=r"(done)
        : "r"(smem_of(bar)), "r"(phase)
        : "memory");
    if (done) return true;
    const int64_t now = clock64();
    if (begin == 0) begin = now;
    else if (now - begin > 4000000000ll) return false;
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

// Waits for all products, with the same limit.  Out of line: inside the kernel its few
// instructions took 1 us of each CTA's time (pieces of 411 with a window, 64.5 instead of 63.2).
__device__ __noinline__ void drain(uint64_t* bar) {
  products_done(bar);
  wait_phase(bar, 0);
}

#define KVX_OUT4(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3])
#define KVX_IN4(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3])

// 32 or 16 columns of a thread's row from or to tensor memory.
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
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : KVX_OUT4(x, 0), KVX_OUT4(x, 4), KVX_OUT4(x, 8), KVX_OUT4(x, 12)
      : "r"(at));
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15};" ::KVX_IN4(x, 0),
      KVX_IN4(x, 4), KVX_IN4(x, 8), KVX_IN4(x, 12), "r"(at)
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

// A warp's 32 tokens of a block lie in two runs of 16 in a row; its lanes load them
// as they lie, 16 bytes (32 dimensions) each: load k brings token kTokens * k +
// lane / kParts, part lane % kParts.
template <int D>
struct Lanes {
  static constexpr int kParts = D / 32, kTokens = 32 / kParts, kLoads = D / 32;
};

// Their codes into a swizzled matrix.  Lanes of the second panel take their words in
// another order, so that eight lanes' 16-byte stores meet no bank twice.
template <int D>
__device__ __forceinline__ void store_codes(uint32_t matrix, int t0, const uint4 (&raw)[D / 32]) {
  using L = Lanes<D>;
  const int lane = threadIdx.x % 32, part = lane % L::kParts, other = part & 2;
#pragma unroll
  for (int k = 0; k < L::kLoads; ++k) {
    const int t = t0 + L::kTokens * k + lane / L::kParts;
    const uint4 r = raw[k];
    const uint32_t w[4] = {other ? r.z : r.x, other ? r.w : r.y, other ? r.x : r.z,
                           other ? r.y : r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int chunk = 4 * (part & 1) + (i ^ other);  // of eight dimensions, in its panel
      const uint32_t at = matrix + (part / 2) * kPanel + t * 128 + ((chunk ^ (t & 7)) << 4);
      const uint4 v = unpack(w[i]);
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
                   "r"(v.w)
                   : "memory");
    }
  }
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_of(bar)) : "memory");
}

// A wait that has run out ends all later ones of the thread: the kernel then
// finishes with the status word set instead of hanging.
struct Waiter {
  bool fine = true;
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t phase) {
    if (fine) fine = wait_phase(bar, phase);
  }
  // For a warp: one lane looks at the barrier.
  __device__ __forceinline__ void wait_warp(uint64_t* bar, uint32_t phase) {
    if (threadIdx.x % 32 == 0) wait(bar, phase);
    __syncwarp();
  }
};

// Where a thread's token of a block is.
struct TokenPlace {
  int id;
  int within;  // token in the page, -1: there is none
};

__device__ __forceinline__ TokenPlace token_place(const AttnArgs& a, const Span& v, int b,
                                                  int block, int t) {
  TokenPlace p{0, -1};
  const int i = block * (kExtendTokens / 16) + t / 16;
  if (i < v.units) {
    const int n = i < v.sink_units ? i : i + v.gap;
    const int page = a.upp_shift >= 0 ? n >> a.upp_shift : n / a.upp;
    p.id = a.tables[int64_t(b) * a.table_stride + page];
    p.within = (n - page * a.upp) * 16 + t % 16;
  }
  return p;
}

// A thread's part of a block on its way: codes of the warp's tokens, and for the V
// warps (scale, zero) of its own token in both tensors.
template <int D>
struct RawToken {
  uint4 codes[D / 32];
  uint32_t param[2];
  bool there;
};

template <int D>
__device__ __forceinline__ void fetch_token(const AttnArgs& a, int head, bool values,
                                            const TokenPlace& p, RawToken<D>& r) {
  r.there = p.within >= 0 && p.id >= 0 && p.id < a.cache.num_blocks;
  if (!r.there && p.within >= 0) atomicExch(&g_q4_status, 5 /* KVX_ERR_BLOCK_ID */);
  using L = Lanes<D>;
  const int lane = threadIdx.x % 32;
  const int64_t page = r.there ? p.id * a.cache.stride + int64_t(head) * a.cache.head_bytes : 0;
  const int64_t run = r.there ? page + (p.within & ~15) * (D / 2) : -1;  // of the 16 tokens
  const int64_t runs[2] = {__shfl_sync(~0u, run, 0), __shfl_sync(~0u, run, 16)};
  const uint8_t* from = a.cache.pages[values ? 1 : 0];
#pragma unroll
  for (int k = 0; k < L::kLoads; ++k) {
    const int token = L::kTokens * k + lane / L::kParts;
    const int64_t at = runs[L::kTokens * k / 16];
    r.codes[k] = at >= 0 ? *reinterpret_cast<const uint4*>(from + at + (token % 16) * (D / 2) +
                                                           16 * (lane % L::kParts))
                         : make_uint4(0u, 0u, 0u, 0u);
  }
  r.param[0] = r.param[1] = 0u;
  if (values && r.there) {
    const int64_t at = page + a.cache.block_size * (D / 2) + p.within * 4;
    r.param[0] = *reinterpret_cast<const uint32_t*>(a.cache.pages[0] + at);
    r.param[1] = *reinterpret_cast<const uint32_t*>(a.cache.pages[1] + at);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kExtendThreads, 1) q4_extend(const __grid_constant__ AttnArgs a,
                                                               int tiles_most) {
  using S = ExtendShape<D>;
  extern __shared__ uint8_t dynamic[];
  __shared__ ExtendShared sh;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  // The rows: the longest first, the kv heads of a sequence's rows side by side.
  const int heads = a.cache.kv_heads;
  const int tile_at = tiles_most - 1 - int(blockIdx.x) / heads, head = int(blockIdx.x) % heads;
  {  // their sequence
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
    if (tid == 0) sh.found = Place{a.batch, 0};
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
  const int tiles = rows > kTileRows ? 2 : 1;
  const Span v = span_of(a, s, row0, rows);
  const int blocks = (v.units * 16 + kExtendTokens - 1) / kExtendTokens;

  const uint32_t base = (smem_of(dynamic) + 1023u) & ~1023u;
  const uint32_t q_at = base, k_at = base + 2 * S::kMatrix, v_at = base + 4 * S::kMatrix;
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_of(&sh.tmem)),
                 "n"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      auto init = [](uint64_t* bar, uint32_t arrivals) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_of(bar)), "r"(arrivals)
                     : "memory");
      };
      for (int i = 0; i < 2; ++i) {
        init(&sh.k_full[i], 4), init(&sh.v_full[i], 4), init(&sh.p_full[i], 4);
        init(&sh.k_free[i], 1), init(&sh.v_free[i], 1);
        init(&sh.s_full[i], 1), init(&sh.o_full[i], 1);
      }
      init(&sh.q_full, uint32_t(4 * tiles));
      init(&sh.drained, 1);
      sh.cut = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = sh.tmem;
  Waiter waiter;

  if (warp >= 12) {
    // ---- the products: one thread issues them --------------------------------
    if (warp == 12 && lane == 0 && blocks > 0) {
      auto scores = [&](int tile, int block) {
        const uint32_t q = q_at + tile * S::kMatrix, k = k_at + (block & 1) * S::kMatrix;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t step = (i / 4) * kPanel + (i % 4) * 32;
          product_ss(tmem + 128 * tile, matrix_desc(q + step, 16, 1024),
                     matrix_desc(k + step, 16, 1024),
                     product_desc(kTileRows, kExtendTokens, false), i > 0);
        }
        products_done(&sh.s_full[tile]);
      };
      auto outputs = [&](int tile, int block) {
        const uint32_t val = v_at + (block & 1) * S::kMatrix;
#pragma unroll
        for (int i = 0; i < kExtendTokens / 16; ++i)
          product_ts(tmem + 256 + 128 * tile, tmem + 128 * tile + 8 * i,
                     matrix_desc(val + i * 2048, kPanel, 1024), product_desc(kTileRows, D, true),
                     block > 0 || i > 0);
        products_done(&sh.o_full[tile]);
      };
      // A tile's scores overwrite the weights that its last outputs read, so they
      // wait for them; the other tile's products fill the time.
      waiter.wait(&sh.q_full, 0);
      waiter.wait(&sh.k_full[0], 0);
      tmem_after();
      scores(0, 0);
      for (int i = 0; i < blocks; ++i) {
        const uint32_t st = i & 1, round = (i >> 1) & 1;
        if (tiles == 2) {
          if (i > 0) waiter.wait(&sh.o_full[1], (i - 1) & 1);
          tmem_after();
          scores(1, i);
        }
        if (i + 2 < blocks) products_done(&sh.k_free[st]);  // somebody waits for it
        waiter.wait(&sh.v_full[st], round);
        waiter.wait(&sh.p_full[0], i & 1);
        tmem_after();
        outputs(0, i);
        if (i + 1 < blocks) {
          waiter.wait(&sh.k_full[(i + 1) & 1], ((i + 1) >> 1) & 1);
          waiter.wait(&sh.o_full[0], i & 1);
          tmem_after();
          scores(0, i + 1);
        }
        if (tiles == 2) {
          waiter.wait(&sh.p_full[1], i & 1);
          tmem_after();
          outputs(1, i);
        }
        if (i + 2 < blocks) products_done(&sh.v_free[st]);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ---- unpacking: warps 8 to 11, 32 tokens of a block each ------------------
    const int t = tid % 128;
    RawToken<D> key, value;
    TokenPlace place = token_place(a, v, b, 0, t);
    fetch_token<D>(a, head, false, place, key);
    fetch_token<D>(a, head, true, place, value);
    place = token_place(a, v, b, 1, t);
    for (int i = 0; i < blocks; ++i) {
      const int st = i & 1;
      const uint32_t before = ((i >> 1) - 1) & 1;
      if (i >= 2) waiter.wait_warp(&sh.k_free[st], before);
      store_codes<D>(k_at + st * S::kMatrix, t & ~31, key.codes);
      shared_written();
      __syncwarp();
      if (lane == 0) arrive(&sh.k_full[st]);
      if (i + 1 < blocks) fetch_token<D>(a, head, false, place, key);
      if (i >= 2) waiter.wait_warp(&sh.v_free[st], before);
      store_codes<D>(v_at + st * S::kMatrix, t & ~31, value.codes);
      {
        // Scales and zeros; a token that no row sees counts 0.
        const int u = i * (kExtendTokens / 16) + t / 16;
        const int n = u < v.sink_units ? u : u + v.gap, token = n * 16 + t % 16;
        const bool seen =
            value.there && token <= v.p_hi && (token > v.p_lo - a.window || token < a.sinks);
        const float2 kp = seen ? half2_at(value.param[0]) : make_float2(0.f, 0.f);
        const float2 vp = seen ? half2_at(value.param[1]) : make_float2(0.f, 0.f);
        sh.ks[st][t] = kp.x * a.scale_part, sh.kz[st][t] = fmaf(8.f, kp.x, kp.y) * a.scale_part;
        sh.vs[st][t] = vp.x, sh.vz[st][t] = fmaf(8.f, vp.x, vp.y);
        if (t % 16 == 0) sh.number[st][t / 16] = value.there ? n : -1;
        float top = fabsf(vp.x);
#pragma unroll
        for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        if (lane == 0) sh.top[st][warp - 8] = top;
      }
      shared_written();
      __syncwarp();
      if (lane == 0) arrive(&sh.v_full[st]);
      if (i + 1 < blocks) {
        fetch_token<D>(a, head, true, place, value);
        place = token_place(a, v, b, i + 2, t);
      }
    }
  } else {
    // ---- softmax: warps 0 to 3 the first tile, 4 to 7 the second ---------------
    if (warp / 4 < tiles) {
    const int tile = warp / 4, t = tid % 128;
    const int r = tile * kTileRows + t;  // the thread's row
    const bool real = r < rows;
    const int query = (row0 + r) / a.group, g = (row0 + r) - query * a.group;
    const int pos = real ? s.len - s.count + query : -1;
    const int tile_rows = min(kTileRows, rows - tile * kTileRows);
    const int p_lo = s.len - s.count + (row0 + tile * kTileRows) / a.group;
    const int p_hi = s.len - s.count + (row0 + tile * kTileRows + tile_rows - 1) / a.group;
    float factor, qsum = 0.f;
    {
      // The query row, scaled as in load_queries(), in the order
      // that unpack() gives the codes.
      const T* from = static_cast<const T*>(a.query) +
                      (real ? int64_t(s.start + query) * a.q_token +
                                  int64_t(head * a.group + g) * a.q_head
                            : 0);
      auto eight = [&](int i, T (&x)[8]) {
        if (!real) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = from_float<T>(0.f);
        } else if (a.q_vec) {
          const uint4 u = *reinterpret_cast<const uint4*>(from + 8 * i);
          __builtin_memcpy(x, &u, 16);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = from[8 * i + k];
        }
      };
      float top = 0.f;
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        T x[8];
        eight(i, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(to_float(x[k])));
      }
      float up = row_scale(top);
      // The power of two of the softmax scale; the rest of it is in ks and kz.
      const int k = a.scale_exp + 127 - int(__float_as_uint(up) >> 23);
      factor = __uint_as_float(uint32_t(min(max(k, -126), 127) + 127) << 23);
      up *= a.sign;
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        T x[8];
        eight(i, x);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y0 = to_float(x[k]) * up, y1 = to_float(x[k + 4]) * up;
          qsum += y0 + y1;
          const __half2 p = __floats2half2_rn(y0, y1);
          __builtin_memcpy(&w[k], &p, 4);
        }
        const uint32_t at = q_at + tile * S::kMatrix + (i / 8) * kPanel + t * 128 +
                            (((i % 8) ^ (t & 7)) << 4);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]),
                     "r"(w[2]), "r"(w[3])
                     : "memory");
      }
      shared_written();
      __syncwarp();
      if (lane == 0) arrive(&sh.q_full);
    }
    const uint32_t lanes = uint32_t(32 * (warp % 4)) << 16;
    const uint32_t s_at = tmem + 128 * tile + lanes, o_at = tmem + 256 + 128 * tile + lanes;
    float minus_r = 0.f, limit = kNegInf;  // minus the reference point
    float2 l = make_float2(0.f, 0.f), z = make_float2(0.f, 0.f);
    for (int i = 0; i < blocks; ++i) {
      const int st = i & 1;
      waiter.wait_warp(&sh.v_full[st], (i >> 1) & 1);  // the scales
      const float most = size_of(fmaxf(fmaxf(sh.top[st][0], sh.top[st][1]),
                                       fmaxf(sh.top[st][2], sh.top[st][3])));
      const int first = i * (kExtendTokens / 16);
      bool plain = first >= v.sink_units && (first + v.gap) * 16 > p_hi - a.window &&
                   (first + v.gap) * 16 + kExtendTokens - 1 <= p_lo;
#pragma unroll
      for (int u = 0; u < kExtendTokens / 16; ++u) plain = plain && sh.number[st][u] >= 0;
      waiter.wait_warp(&sh.s_full[tile], i & 1);
      tmem_after();
#pragma unroll 1
      for (int part = 0; part < 4; ++part) {  // 32 tokens at a time
        uint32_t x[32];
        tmem_load(s_at + 32 * part, x);
        const float* ks = sh.ks[st] + 32 * part;
        const float* kz = sh.kz[st] + 32 * part;
        tmem_loaded();
        float y[32], top = kNegInf;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 sc = *reinterpret_cast<const float4*>(ks + c);
          const float4 zc = *reinterpret_cast<const float4*>(kz + c);
          const float2 y0 = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])),
                                 make_float2(sc.x, sc.y), mul2(make_float2(zc.x, zc.y), both(qsum)));
          const float2 y1 = fma2(make_float2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])),
                                 make_float2(sc.z, sc.w), mul2(make_float2(zc.z, zc.w), both(qsum)));
          y[c] = y0.x, y[c + 1] = y0.y, y[c + 2] = y1.x, y[c + 3] = y1.y;
        }
        if (!plain) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int n = sh.number[st][2 * part + c / 16], token = n * 16 + c % 16;
            const bool seen = n >= 0 && token <= pos && (token > pos - a.window || token < a.sinks);
            y[c] = seen ? y[c] : kNegInf;
          }
        }
#pragma unroll
        for (int c = 0; c < 32; c += 2) top = max3(top, y[c], y[c + 1]);
        // The largest score with the block's largest V scale says whether P' may pass 2^14.
        // Only then do the tokens' own products decide: with a look at each of them
        // always, 1024-token pieces behind 7168 tokens took 1227 us, 1176 like this.
        if (__any_sync(~0u, fmaf(top, factor, most) + minus_r > limit)) {
          top = kNegInf;
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 sc = *reinterpret_cast<const float4*>(sh.vs[st] + 32 * part + c);
            top = max3(top, fmaf(y[c], factor, size_of(sc.x)),
                       fmaf(y[c + 1], factor, size_of(sc.y)));
            top = max3(top, fmaf(y[c + 2], factor, size_of(sc.z)),
                       fmaf(y[c + 3], factor, size_of(sc.w)));
          }
          // The reference point moves by whole powers of two: the weights of this block
          // that are written already scale exactly.
          if (__any_sync(~0u, top + minus_r > limit)) {
            float f = 1.f;
            if (top + minus_r > limit) {
              float to = kLift - ceilf(top);
              if (limit == kFar || fabsf(top) >= kFarScore) {
                top = kNegInf;
#pragma unroll
                for (int c = 0; c < 32; c += 2) top = max3(top, y[c], y[c + 1]);
                to = -ceilf(top * factor);
                if (limit != kNegInf) to = fminf(to, minus_r), f = ex2(to - minus_r);
                limit = kFar;
              } else {
                if (limit != kNegInf) f = ex2(to - minus_r);
                limit = kLift + kSlack;
              }
              minus_r = to;
            }
            l.x *= f, l.y *= f, z.x *= f, z.y *= f;
            if (i > 0) {  // the scores waited for the last block's outputs
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                tmem_load(o_at + 32 * c, x);
                tmem_loaded();
#pragma unroll
                for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * f);
                tmem_store(o_at + 32 * c, x);
              }
            }
            tmem_stored();
            const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
            for (int c = 0; c < part; ++c) {
              uint32_t w[16];
              tmem_load(s_at + 16 * c, w);
              tmem_loaded();
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                __half2 h;
                __builtin_memcpy(&h, &w[k], 4);
                h = __hmul2(h, f2);
                __builtin_memcpy(&w[k], &h, 4);
              }
              tmem_store(s_at + 16 * c, w);
            }
          }
        }
        uint32_t w16[16];
        const float* vs = sh.vs[st] + 32 * part;
        const float* vz = sh.vz[st] + 32 * part;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 sc = *reinterpret_cast<const float4*>(vs + c);
          const float4 zc = *reinterpret_cast<const float4*>(vz + c);
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            float2 p = fma2(make_float2(y[c + k], y[c + k + 1]), both(factor), both(minus_r));
            p.x = ex2(p.x), p.y = ex2(p.y);
            l = add2(l, p);
            float2 w = mul2(p, k ? make_float2(sc.z, sc.w) : make_float2(sc.x, sc.y));
            float2 zn = fma2(p, k ? make_float2(zc.z, zc.w) : make_float2(zc.x, zc.y), z);
            if (!plain) {  // a hidden token's scale and zero may be anything
              if (y[c + k] == kNegInf) w.x = 0.f, zn.x = z.x;
              if (y[c + k + 1] == kNegInf) w.y = 0.f, zn.y = z.y;
            }
            z = zn;
            const __half2 half = __floats2half2_rn(w.x, w.y);
            __builtin_memcpy(&w16[(c + k) / 2], &half, 4);
          }
        }
        tmem_store(s_at + 16 * part, w16);  // over scores that are read
      }
      tmem_stored();
      tmem_before();
      __syncwarp();
      if (lane == 0) arrive(&sh.p_full[tile]);
    }
    if (blocks > 0) waiter.wait_warp(&sh.o_full[tile], (blocks - 1) & 1);
    tmem_after();
    const float total = l.x + l.y, zero = z.x + z.y, by = total == 0.f ? 0.f : 1.f / total;
    const int64_t token = s.start + query;
    const int head_out = head * a.group + g;
    T* to = static_cast<T*>(a.out) + token * a.o_token + int64_t(head_out) * a.o_head;
#pragma unroll 1
    for (int part = 0; part < D / 32; ++part) {
      uint32_t x[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) x[c] = 0u;
      if (blocks > 0) {
        tmem_load(o_at + 32 * part, x);
        tmem_loaded();
      }
      if (real) {
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          T y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)  // dimension k is column 0 2 4 6 1 3 5 7 of the eight
            y[k] = from_float<T>((__uint_as_float(x[c + (k < 4 ? 2 * k : 2 * k - 7)]) + zero) * by);
          if (a.o_vec16) {
            uint4 w;
            __builtin_memcpy(&w, y, 16);
            *reinterpret_cast<uint4*>(to + 32 * part + c) = w;
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) to[32 * part + c + k] = y[k];
          }
        }
      }
    }
    if (a.lse && real)
      a.lse[token * (int64_t(heads) * a.group) + head_out] = log_sum(-minus_r, total);
    }
  }
  if (!waiter.fine) {
    sh.cut = 1;
    atomicExch(&g_q4_status, 8 /* KVX_ERR_DEVICE_TIMEOUT */);
  }
  tmem_before();
  __syncthreads();
  if (warp == 12) {
    tmem_after();
    // The last outputs were waited for, and with them every product.  Not so where a wait
    // ran out: none of them may outlive the block's memory.
    if (sh.cut && lane == 0) {
      drain(&sh.drained);
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(S::kColumns));
  }
}

}  // namespace q4
}  // namespace kvx
