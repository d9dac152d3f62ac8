// Attention of chunks of new tokens over a paged cache on the 5th-generation tensor cores.
//
// Same mathematics and the same division into equal runs of 64-key tiles as the few-rows form (paged.cu, paged.cuh), for
// calls with many query rows for each key, which are bound by the products and the softmax's exponentials instead of
// memory. The rows of a 128-row query tile are 128 / group tokens with all the query heads of the group, so that a key tile
// is loaded once for the whole group, and a short chunk still fills the rows of the products. A unit is two query tiles of
// one (sequence, kv head), with one CTA a SM; or one, with two CTAs a SM, for calls whose chunks fit a query tile: the
// two then take different units, and one computes while the other starts or ends its own.
//
// A persistent CTA takes its run of the line of tiles. K and V tiles of 64 keys are streamed by TMA through
// rings, one box per page (or 64 keys of a larger page), the page ids looked up one tile ahead. Boxes past the
// sequence's end load nothing and come as zeros; in the box that holds the end, the rows of V past it are zeroed in
// shared memory before the products see them, so that nothing a page holds past the length (NaN, infinities) reaches
// 0 x v. Rows are 128 B pieces of 64 dims, 128B-swizzled, for Q, K and V alike (dims 96-127 of 96 read as zeros and
// are not multiplied).
//
// Tensor memory: two S buffers of each query tile (fp32, tile t in buffer t % 2 at [128 i + 64 (t % 2), +64)) and O_i
// (fp32, 128 columns each after the S buffers). The softmax writes P(t) (16-bit pairs) over the first 32 columns of the S
// buffer that it has read, so S(t + 2) follows P(t) V(t) there, while S(t + 1) is ready before the softmax of tile t is
// done: the softmax waits for no product but its own tile's. (With one S buffer and P apart the softmax waited 300-450 of
// the 1,800 cycles of a tile for S: clock stamps.)
//
// Warp roles: warp 0 loads Q and the K ring, warp 2 the V ring; a warp for each query tile issues its scores and another
// its products with V (an issuing warp takes a few hundred cycles for a batch of products and its waits, which one warp a
// tile could not hide); each of these loops is warp-converged, one elected lane issuing. Four warps a query tile run its
// softmax, one row a thread. The exponent base is raised lazily (only when a row's maximum grows by more than 8 in log2
// units), a part of the exponentials is evaluated on the FMA pipe; weights are rounded to the cache's type for P V and
// summed unrounded. A query tile without tokens (the second of a unit's) is skipped by its chain, and a warp without live
// rows skips the arithmetic. Every wait is bounded; a timeout sets SVX_STATUS_WAIT_TIMEOUT and skips the rest.
//
// Bound: the tile loop, 1,540 (dim 128) to 1,740 (96) cycles for 256 rows x 64 keys, where products and softmax wait on one
// another: the tensor pipe needs 1,280 or 960 of them (64-wide products of scores take 48 cycles for 32 of arithmetic), the
// exponential unit 768. Without exponentials it ran 10% faster, without the maximum 2%. Measured on B200 (bf16): 4
// chunks of 1500 to 2048 tokens x 32 heads of 128 over 9,000 to 32,768 keys, 8 kv heads, 1,170 to 1,290 us, 990 to 1,095
// TFLOP/s under the power cap; 8 of 1024 rows x 8 heads of 96 over 2368 to 9536 keys without a mask 182 to 190 us, 700 to
// 730 TFLOP/s. The one-tile form spills 36 to 68 bytes a thread at the 128 registers that two CTAs a SM leave.
//
// Built, measured and not kept: two threads a row (16 softmax warps; 2,100 cycles a tile against 1,740: the warps of a
// scheduler reach their exponentials together), and both chains on one query tile, every second key tile each (handing the
// sums over took 4 to 7 us a unit).
#include <math.h>

#include "common.cuh"
#include "gemm.cuh"
#include "paged.cuh"
#include "tc.cuh"

namespace svx {

__device__ uint32_t g_svx_paged_timeouts = 0;

uint32_t paged_timeouts() {
  uint32_t v = 0;
  if (cudaMemcpyFromSymbol(&v, g_svx_paged_timeouts, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
  return v;
}

namespace paged {
namespace {

constexpr int TQ = 128, TK = kTile;

template <int D, int kChains> struct Tiles {
  static constexpr int threads = kChains == 2 ? 448 : 256;
  static constexpr uint32_t tmem_cols = 256 * kChains, s_col = 0, o_col = 128 * kChains;   // + 128 i
  static constexpr int atoms = (D + 63) / 64;             // 128-byte pieces of a row
  static constexpr uint32_t q_atom = TQ * 128, q_bytes = atoms * q_atom;
  static constexpr uint32_t k_atom = TK * 128, k_bytes = atoms * k_atom;
  static constexpr int stages = kChains == 2 ? (atoms == 2 ? 4 : 8) : (atoms == 2 ? 2 : 4);
  static constexpr int out_cols = 32 * kChains;           // columns of each softmax warp's 32 rows on their way out
  static constexpr uint32_t out_row = out_cols * 2, out_bytes = kChains * 4 * 32 * out_row;
  static constexpr int bars = 2 + 4 * stages + 1 + 6 * kChains + 1;
  static constexpr size_t smem = 1024 + kChains * q_bytes + 2 * stages * k_bytes + out_bytes + bars * 8 + 16;
};

// Bounded waits (two to three seconds) that give up as soon as another role of the CTA raised `abort`; the clock is read
// between batches of polls only.
constexpr long long kWaitCycles = 4000000000ll;

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (clock64() - start > kWaitCycles) {
      *abort = 1;
      return false;
    }
  }
}
// Warp-collective: the lanes agree on the outcome, so that none leaves a loop of warp-wide instructions alone where `abort`
// is raised while the phase completes. Every wait of the kernel's loops goes through it.
__device__ __forceinline__ bool wait_w(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort));
}

struct Maps {
  CUtensorMap q, k, v;
};

template <typename T> struct Kind;
template <> struct Kind<__nv_bfloat16> {
  static constexpr uint32_t format = 1;   // of the instruction descriptor's A and B
  static constexpr float shift = 0.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return tc::pack_bf16x2(lo, hi); }
};
template <> struct Kind<__half> {
  static constexpr uint32_t format = 0;
  static constexpr float shift = 7.f;     // weights are held 2^7 larger (at most 2^15 with the lazy base): see paged.cu
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
    return d;
  }
};

// kind::f16, fp32 accumulator, A K-major, B K-major or MN-major.
__host__ __device__ constexpr uint32_t descriptor(uint32_t format, int m, int n, bool b_mn) {
  return (1u << 4) | (format << 7) | (format << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// One product over 16 of K (operand descriptors %1 and %2 moved on by A and B), and the arrival of a barrier once the
// products before it are done, both by the elected lane.
#define SVX_SS_STEP(A, B, ACC)                     \
  "add.s64 x, %1, " #A ";\n\tadd.s64 y, %2, " #B ";\n\t" \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, " ACC ";\n\t"
#define SVX_COMMIT(BAR) "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [" BAR "];\n\t"

// Warp-collective: S = Q K^T over D dims, both operands K-major in 128B-swizzled atoms of 64 dims (a step is 32 bytes,
// +2 in descriptor units; an atom 16 KB of Q and 8 KB of K), then the arrivals on `done` and `release`. One election for
// the whole batch: an elected block of one instruction costs as much as one of ten.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t d, uint64_t q, uint64_t k, uint32_t idesc, uint64_t* done,
                                             uint64_t* release) {
#define SVX_SS_BEGIN                                                                     \
  "{\n\t.reg .pred e, p0, pt;\n\t.reg .b64 x, y;\n\telect.sync _|e, 0xffffffff;\n\t" \
  "setp.ne.b32 p0, %3, %3;\n\tsetp.eq.b32 pt, %3, %3;\n\t"                              \
  SVX_SS_STEP(0, 0, "p0") SVX_SS_STEP(2, 2, "pt") SVX_SS_STEP(4, 4, "pt") SVX_SS_STEP(6, 6, "pt")
#define SVX_SS_END SVX_COMMIT("%4") SVX_COMMIT("%5") "}"
  const uint32_t b0 = smem_addr(done), b1 = smem_addr(release);
  if constexpr (D == 64)
    asm volatile(SVX_SS_BEGIN SVX_SS_END ::"r"(d), "l"(q), "l"(k), "r"(idesc), "r"(b0), "r"(b1) : "memory");
  else if constexpr (D == 96)
    asm volatile(SVX_SS_BEGIN SVX_SS_STEP(1024, 512, "pt") SVX_SS_STEP(1026, 514, "pt") SVX_SS_END
                 ::"r"(d), "l"(q), "l"(k), "r"(idesc), "r"(b0), "r"(b1) : "memory");
  else
    asm volatile(SVX_SS_BEGIN SVX_SS_STEP(1024, 512, "pt") SVX_SS_STEP(1026, 514, "pt") SVX_SS_STEP(1028, 516, "pt")
                 SVX_SS_STEP(1030, 518, "pt") SVX_SS_END
                 ::"r"(d), "l"(q), "l"(k), "r"(idesc), "r"(b0), "r"(b1) : "memory");
#undef SVX_SS_BEGIN
#undef SVX_SS_END
}

// Warp-collective: O (+)= P V over 64 keys: A = P in tensor memory (8 columns a step), B = V MN-major (16 keys x 128 B a
// step, +128 in descriptor units), then the arrivals on `done` and `release`.
__device__ __forceinline__ void issue_values(uint32_t d, uint32_t p, uint64_t v, uint32_t idesc, uint32_t acc,
                                             uint64_t* done, uint64_t* release) {
  asm volatile(
      "{\n\t.reg .pred e, p0, pt;\n\t.reg .b64 y;\n\t.reg .b32 x;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p0, %4, 0;\n\tsetp.eq.b32 pt, %3, %3;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p0;\n\t"
      "add.s32 x, %1, 8;\n\tadd.s64 y, %2, 128;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, pt;\n\t"
      "add.s32 x, %1, 16;\n\tadd.s64 y, %2, 256;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, pt;\n\t"
      "add.s32 x, %1, 24;\n\tadd.s64 y, %2, 384;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, pt;\n\t"
      SVX_COMMIT("%5") SVX_COMMIT("%6") "}"
      ::"r"(d), "r"(p), "l"(v), "r"(idesc), "r"(acc), "r"(smem_addr(done)), "r"(smem_addr(release)) : "memory");
}
#undef SVX_SS_STEP
#undef SVX_COMMIT

__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// max(a, b, c), NaN where any of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 2^x on the FMA pipe for a pair: x = j + f with j = rint(x) from the 1.5 * 2^23 magic sum, a degree-4 polynomial fitted
// to 2^f on [-0.5, 0.5] (relative error 2.7e-6), times 2^j. x is clamped at -127, which gives exactly 0, so that hidden keys
// (-inf) and weights under 2^-127 add nothing, however large the value behind them. kProduct: a product with 2^j, made in
// the exponent field and 0 there; else j added to the exponent field, the sums that fall below it cut to 0 (between 2^-127
// and 2^-126 the fraction is lost). The first is faster with two query tiles a unit (attn-chunk 1,210 us against 1,248,
// attn-windows 184 against 186), the second with one, where registers are short (attn-verify 60.5 against 62.3).
template <bool kProduct>
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = fmaxf(x.x, -127.f);
  x.y = fmaxf(x.y, -127.f);
  const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));
  const float2 j = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = __ffma2_rn(j, make_float2(-1.f, -1.f), x);
  float2 q = __ffma2_rn(make_float2(0.009570068679749966f, 0.009570068679749966f), f,
                        make_float2(0.055917806923389435f, 0.055917806923389435f));
  q = __ffma2_rn(q, f, make_float2(0.240247443318367f, 0.240247443318367f));
  q = __ffma2_rn(q, f, make_float2(0.6931218504905701f, 0.6931218504905701f));
  q = __ffma2_rn(q, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  if (kProduct)
    return __fmul2_rn(q, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                                     __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
  return make_float2(__int_as_float(max(0, __float_as_int(q.x) + (__float_as_int(t.x) << 23))),
                     __int_as_float(max(0, __float_as_int(q.y) + (__float_as_int(t.y) << 23))));
}

// Of every 8 pairs of exponentials, this many go to the FMA pipe.
constexpr int kPolyPairs = 2;

// Live query tiles of a unit (tile_tokens tokens each).
__device__ __forceinline__ int live_tiles(const Params& p, const Cursor& at, int tile_tokens) {
  return at.q.n - at.j * p.unit_tokens > tile_tokens ? 2 : 1;
}

template <typename T, int D, int kChains>
__global__ void __launch_bounds__(Tiles<D, kChains>::threads, 3 - kChains)
    chunk_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Tiles<D, kChains>;
  using K = Kind<T>;
  constexpr int kThreads = C::threads;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PlanShared plan_shared;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sk = sq + kChains * C::q_bytes;
  uint8_t* sv = sk + C::stages * C::k_bytes;
  uint8_t* so = sv + C::stages * C::k_bytes;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(so + C::out_bytes);
  uint64_t* q_empty = q_full + 1;             // both chains are past their last S of a unit
  uint64_t* k_full = q_full + 2;
  uint64_t* k_empty = k_full + C::stages;
  uint64_t* v_full = k_empty + C::stages;
  uint64_t* v_empty = v_full + C::stages;
  uint64_t* v_end = v_empty + C::stages;      // the load of a V tile that holds the sequence's end
  uint64_t* s_full = v_end + 1;               // per query tile and buffer: S computed
  uint64_t* p_full = s_full + 2 * kChains;    // per query tile and buffer, 4 arrivals: P written (and O_i rescaled)
  uint64_t* pv_done = p_full + 2 * kChains;   // per query tile and buffer: P V completed
  uint64_t* drained = pv_done + 2 * kChains;  // 2 arrivals a chain: all products issued are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + C::bars);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  // Tile n of a chain (counted over the CTA's whole run) uses buffer n % 2, whose barriers are in phase n / 2. With one
  // barrier for both buffers a wait could find the phase two tiles back and take it for its own.
  auto buffer_wait = [&](uint64_t* bars, int i, int n) {
    return wait_w(bars + 2 * i + (n & 1), (n >> 1) & 1, abort_flag);
  };
  const int warp = warp_id(), lane = lane_id(), cta = blockIdx.x;
  const int tile_tokens = p.tile_tokens;
  grid_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, kChains);
    for (int i = 0; i < C::stages; ++i) {
      mbar_init(k_full + i, 1); mbar_init(k_empty + i, kChains);
      mbar_init(v_full + i, 1); mbar_init(v_empty + i, kChains);
    }
    mbar_init(v_end, 1);
    for (int i = 0; i < 2 * kChains; ++i) {
      mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); mbar_init(pv_done + i, 1);
    }
    mbar_init(drained, 2 * kChains);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::prefetch_map(&maps.q);
    tc::prefetch_map(&maps.k);
    tc::prefetch_map(&maps.v);
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, C::tmem_cols);
  grid_dependency_wait();
  plan<kThreads, kChains == 2>(p, cta, gridDim.x, plan_shared, reinterpret_cast<int64_t*>(smem));   // before the tiles are loaded
  if (threadIdx.x == 0) p.join[cta].parts = 0;
  tc::fence_async_smem();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const Place& place = plan_shared.place;
  const int page_mask = (1 << p.page_shift) - 1, box = min(TK, 1 << p.page_shift), boxes = TK / box;
  const int nowhere = p.pages * p.kv_heads;   // a coordinate past the pool: loads zeros

  // A chain without live rows in a unit hands its tiles back.
  auto idle = [&](const Walk& w, int i) { return i >= live_tiles(p, w.at, tile_tokens); };
  auto issue_all_scores = [&](int i) {
    constexpr uint32_t idesc = descriptor(K::format, TQ, TK, false);
    const uint32_t d = tmem + C::s_col + 128 * i;
    const uint64_t q = tc::sw128_desc(smem_addr(sq + i * C::q_bytes));
    int g = 0, n = 0;   // tiles of the ring and of this chain
    bool ok = true;
    for (Walk w(p, place, cta); ok && w.more(); w.next(p, place, gridDim.x)) {
      const bool none = idle(w, i);
      if (!wait_w(q_full, w.units & 1, abort_flag)) break;
      for (int t = w.t0; t < w.t1; ++t, ++g) {
        const int s = g % C::stages;
        ok = wait_w(k_full + s, (g / C::stages) & 1, abort_flag);
        if (!ok) break;
        if (none) {
          if (lane == 0) tc::mbar_arrive(k_empty + s);
          continue;
        }
        // S(n) goes where P(n - 2) was
        ok = n < 2 || buffer_wait(pv_done, i, n - 2);
        if (!ok) break;
        tc::fence_after();
        issue_scores<D>(d + 64 * (n & 1), q, tc::sw128_desc(smem_addr(sk + s * C::k_bytes)), idesc,
                        s_full + 2 * i + (n & 1), k_empty + s);
        ++n;
      }
      if (!ok) break;
      if (!none) tc::commit_w(q_empty);
      else if (lane == 0) tc::mbar_arrive(q_empty);
    }
    tc::commit_w(drained);
  };
  auto issue_all_values = [&](int i) {
    constexpr uint32_t idesc = descriptor(K::format, TQ, D, true);
    const uint32_t d = tmem + C::o_col + 128 * i, a = tmem + C::s_col + 128 * i;
    int g = 0, n = 0;
    bool ok = true;
    for (Walk w(p, place, cta); ok && w.more(); w.next(p, place, gridDim.x)) {
      const bool none = idle(w, i);
      for (int t = w.t0; t < w.t1; ++t, ++g) {
        const int s = g % C::stages;
        ok = wait_w(v_full + s, (g / C::stages) & 1, abort_flag);
        if (!ok) break;
        if (none) {
          if (lane == 0) tc::mbar_arrive(v_empty + s);
          continue;
        }
        ok = buffer_wait(p_full, i, n);
        if (!ok) break;
        tc::fence_after();
        issue_values(d, a + 64 * (n & 1), tc::sw128_desc(smem_addr(sv + s * C::k_bytes), C::k_atom, 1024), idesc, t != w.t0,
                     pv_done + 2 * i + (n & 1), v_empty + s);   // a unit's first product starts O afresh
        ++n;
      }
    }
    tc::commit_w(drained);
  };

  if (warp < 4) {
    if (warp == 0 || warp == 2) {   // K with Q, and V
      const bool is_v = warp == 2;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      uint8_t* ring = is_v ? sv : sk;
      const CUtensorMap* map = is_v ? &maps.v : &maps.k;
      Walk w(p, place, cta);
      int g = 0, ends = 0;
      bool ok = true;
      // The page id of box `lane` of tile t, as the pool's coordinate.
      auto look_up = [&](const Cursor& at, int t) {
        const int key = t * TK + lane * box;
        int z = nowhere;
        if (lane < boxes && key < at.limit) {
          const int id = __ldg(p.table + (int64_t)at.s * p.table_width + (key >> p.page_shift));
          if (id >= 0 && id < p.pages) z = id * p.kv_heads + at.h;
          else if (!is_v && p.status) atomicOr(p.status + at.s, SVX_STATUS_BAD_PAGE);
        }
        return z;
      };
      int z = w.more() ? look_up(w.at, w.t0) : nowhere;
      while (ok && w.more()) {
        if (!is_v) {
          if (w.units && !wait_w(q_empty, (w.units - 1) & 1, abort_flag)) { ok = false; break; }
          const int nq = kChains == 2 ? live_tiles(p, w.at, tile_tokens) : 1;
          const uint32_t tile_bytes = C::atoms * 128 * tile_tokens * p.group;
          tc::expect_tx_w(q_full, nq * tile_bytes);
          for (int i = 0; i < nq; ++i)
            for (int a = 0; a < C::atoms; ++a)
              tc::tma_load_3d_w(sq + i * C::q_bytes + a * C::q_atom, &maps.q, a * 64, w.at.h * p.group,
                                w.at.q.row0 + w.at.j * p.unit_tokens + i * tile_tokens, q_full);
        }
        const Cursor at = w.at;
        const int t0 = w.t0, t1 = w.t1;
        w.next(p, place, gridDim.x);
        for (int t = t0; t < t1; ++t, ++g) {
          const int s = g % C::stages;
          if (g >= C::stages && !wait_w(empty + s, (g / C::stages - 1) & 1, abort_flag)) { ok = false; break; }
          const int left = at.q.len - t * TK;   // keys of the sequence from this tile on
          const bool end = is_v && left > 0 && left < TK && left % box != 0;
          uint64_t* bar = end ? v_end : full + s;
          uint8_t* dst = ring + s * C::k_bytes;
          tc::expect_tx_w(bar, C::k_bytes);
          for (int b = 0; b < boxes; ++b) {
            const int zb = __shfl_sync(0xffffffffu, z, b), row = (t * TK + b * box) & page_mask;
            for (int a = 0; a < C::atoms; ++a)
              tc::tma_load_3d_w(dst + a * C::k_atom + b * box * 128, map, a * 64, zb, row, bar);
          }
          if (end) {   // rows past the end may hold anything: zeros, then the tile is complete
            if (!wait_w(v_end, ends & 1, abort_flag)) {
              mbar_wait(v_end, ends & 1);
              ok = false;
              break;
            }
            ++ends;
            const int rows = box - left % box;   // to the end of the box
            for (int e = lane; e < C::atoms * rows * 8; e += 32) {
              const int a = e / (rows * 8), r = e % (rows * 8);
              *reinterpret_cast<uint4*>(dst + a * C::k_atom + left * 128 + r * 16) = make_uint4(0, 0, 0, 0);
            }
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(full + s);
          }
          if (t + 1 < t1) z = look_up(at, t + 1);
          else if (w.more()) z = look_up(w.at, w.t0);
        }
      }
      // Loads in flight end before the block does, also where an abort leaves nothing that waits for them.
      for (int u = max(0, g - C::stages); u < g; ++u) mbar_wait(full + u % C::stages, (u / C::stages) & 1);
      if (!is_v && w.units) mbar_wait(q_full, (w.units - 1) & 1);
    } else if (warp == 1 || kChains == 2) {   // warp 1: scores of query tile 0; warp 3: of query tile 1
      issue_all_scores(warp == 1 ? 0 : 1);
    } else {   // warp 3: O of the query tile
      issue_all_values(0);
    }
    // Teardown: the TMEM owner frees the columns once all warps are past their last TMEM access.
    tc::fence_before();
    __syncwarp();
    asm volatile("barrier.sync 1, %0;" ::"n"(kThreads) : "memory");
    if (warp == 1) {
      mbar_wait(drained, 0);
      __syncwarp();
      tc::fence_after();
      tc::tmem_dealloc(*tmem_slot, C::tmem_cols);
    }
    return;
  }

  if (warp >= 12) {   // warp 12: O of query tile 0; warp 13: of query tile 1
    issue_all_values(warp - 12);
    tc::fence_before();
    __syncwarp();
    asm volatile("barrier.arrive 1, %0;" ::"n"(kThreads) : "memory");
    return;
  }

  const int i = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
  const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
  const uint32_t to = tmem + lanes + C::o_col + 128 * i;
  const float sl2 = p.scale_log2;
  const bool in_tile = row < tile_tokens * p.group;
  int n0 = 0;
  bool ok = true;
  Walk w(p, place, cta);
  for (; ok && w.more(); w.next(p, place, gridDim.x)) {
    const Cursor& at = w.at;
    if (p.status && threadIdx.x == 128) {
      if (__ldg(p.lengths + at.s) != at.q.len) atomicOr(p.status + at.s, SVX_STATUS_BAD_PAGE);
    }
    if (idle(w, i)) continue;
    const int token = at.j * p.unit_tokens + i * tile_tokens + row / p.group;
    const bool live = in_tile && token < at.q.n;
    // Keys that this row sees; a dead row's result is not stored.
    const int limit = !live ? 0 : p.causal ? max(0, min(at.q.len, at.q.len - at.q.n + token + 1)) : at.q.len;
    const int least = __reduce_min_sync(0xffffffffu, live ? limit : 0x7fffffff);
    const bool warp_live = least != 0x7fffffff;
    float m_used = -INFINITY, l_run = 0.f;
    const int count = w.t1 - w.t0;
    int key0 = w.t0 * TK;
    for (int u = 0; u < count; ++u, key0 += TK) {
      const int n = n0 + u, buffer = n & 1;
      const uint32_t ts = tmem + lanes + C::s_col + 128 * i + 64 * buffer;
      if (!buffer_wait(s_full, i, n)) { ok = false; break; }
      if (!warp_live) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full + 2 * i + buffer);
        continue;
      }
      tc::fence_after();
      uint32_t r[2][32];
      tc::ld32(ts, r[0]);
      tc::ld32(ts + 32, r[1]);
      tc::wait_ld();
      if (key0 + TK > least) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (key0 + c * 32 + j >= limit) r[c][j] = __float_as_uint(-INFINITY);
      }
      float mc[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float a = __uint_as_float(r[c][0]), b = __uint_as_float(r[c][1]);
#pragma unroll
        for (int j = 2; j < 30; j += 4) {
          a = max3_nan(a, __uint_as_float(r[c][j]), __uint_as_float(r[c][j + 1]));
          b = max3_nan(b, __uint_as_float(r[c][j + 2]), __uint_as_float(r[c][j + 3]));
        }
        mc[c] = max3_nan(a, max2_nan(b, __uint_as_float(r[c][30])), __uint_as_float(r[c][31]));
      }
      const float mx = max2_nan(mc[0], mc[1]) * sl2;
      // Raise the exponent base only when the row's maximum outgrows it by more than 8 (warp-uniform rescale of O). A
      // NaN raises it too and stays: every weight of the row is NaN from then on.
      const bool raise = live && !(mx <= m_used + 8.f);
      const bool any_raise = __any_sync(0xffffffffu, raise);
      float alpha = 1.f;
      if (any_raise) {
        const float m_new = raise ? mx : m_used;
        alpha = m_used == m_new ? 1.f : tc::ex2(m_used - m_new);   // m_used = -inf: 0
        m_used = m_new;
      }
      const float base = m_used == -INFINITY ? 0.f : m_used - K::shift;
      const float2 scale2 = make_float2(sl2, sl2), nbase2 = make_float2(-base, -base);
      float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t packed[32];
#pragma unroll
      for (int j = 0; j < TK; j += 2) {
        const int c = j >> 5, jj = j & 31;
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c][jj]), __uint_as_float(r[c][jj + 1])), scale2, nbase2);
        const float2 e = ((j >> 1) & 7) < kPolyPairs ? exp2_poly<kChains == 2>(x) : make_float2(tc::ex2(x.x), tc::ex2(x.y));
        acc[(j >> 1) & 3] = __fadd2_rn(acc[(j >> 1) & 3], e);
        packed[j >> 1] = K::pack(e.x, e.y);
      }
      tc::st32(ts, packed);
      if (any_raise && u >= 1) {   // O holds the products of the earlier tiles once P(t - 1) V(t - 1) is done
        if (!buffer_wait(pv_done, i, n - 1)) { ok = false; break; }
        tc::fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          ld16(to + c, o);
          tc::wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          tc::st16(to + c, o);
        }
      }
      tc::wait_st();
      const float2 s01 = __fadd2_rn(acc[0], acc[1]), s23 = __fadd2_rn(acc[2], acc[3]);
      l_run = l_run * alpha + ((s01.x + s01.y) + (s23.x + s23.y));
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full + 2 * i + buffer);
    }
    if (ok) ok = buffer_wait(pv_done, i, n0 + count - 1);
    if (!ok) break;
    tc::fence_after();
    n0 += count;
    const bool whole = w.whole();
    // An infinite score makes the row NaN, as inf - inf does.
    if (m_used == INFINITY) l_run = __int_as_float(0x7fffffff);
    const bool none = m_used == -INFINITY;
    const float factor = none ? 0.f : whole ? 1.f / l_run : 1.f;
    if (warp_live) {
      const int64_t slot = partial_slot(cta, w.part);
      const int part_row = i * TQ + row;
      float4* part = reinterpret_cast<float4*>(p.partial_o) + slot * p.rows * (D / 4) + part_row;
      const int64_t row0 = (int64_t)(at.q.row0 + at.j * p.unit_tokens) * p.q_heads + at.h * p.group;
      const int out_row = live ? (token - at.j * p.unit_tokens) * p.q_heads + row % p.group : -1;
      uint8_t* mine = so + (warp - 4) * 32 * C::out_row;
      // Sixteen columns at a time, in a loop: unrolled, it cost the tile loop registers (8 windows of 1024 rows 184.6 us
      // against 182.0). A unit's end takes about 2 us, which the other chain or CTA fills in part.
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        ld16(to + c, o);
        tc::wait_ld();
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = none ? 0.f : __uint_as_float(o[j]) * factor;
        if (!whole) {   // neighbouring rows are neighbours in memory
          if (live) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              part[(c / 4 + k) * p.rows] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
          }
          continue;
        }
        // Through shared memory, so that the lanes of a row write its 64 or 128 bytes together. Pieces of 16 bytes are
        // swizzled: by the row for rows of 128 bytes, by every second row for rows of 64.
        auto place_of = [&](int r, int piece) {
          return reinterpret_cast<uint4*>(mine + r * C::out_row +
                                          ((kChains == 2 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3)) * 16));
        };
        const int piece0 = c % C::out_cols / 8;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *place_of(lane, piece0 + k) =
              make_uint4(K::pack(f[8 * k], f[8 * k + 1]), K::pack(f[8 * k + 2], f[8 * k + 3]),
                         K::pack(f[8 * k + 4], f[8 * k + 5]), K::pack(f[8 * k + 6], f[8 * k + 7]));
        if (piece0 + 2 < C::out_cols / 8 && c + 16 < D) continue;
        __syncwarp();
        const int shift = piece0 == 6 ? 3 : 2;   // log2 of the row's pieces: 8 or 4
#pragma unroll 4
        for (int k = 0; k < 1 << shift; ++k) {
          const int e = 32 * k + lane, r = e >> shift, piece = e & ((1 << shift) - 1);
          const int to_row = __shfl_sync(0xffffffffu, out_row, r);
          const uint4 x = *place_of(r, piece);
          if (to_row >= 0)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row0 + to_row) * D + c / C::out_cols * C::out_cols +
                                      piece * 8) = x;
        }
        __syncwarp();
      }
      if (live && !whole) p.partial_ml[slot * p.rows + part_row] = make_float2(m_used, l_run);
      if (live && whole && p.lse)
        p.lse[row0 + out_row] = none ? -INFINITY : (m_used - K::shift + log2f(l_run)) * 0.69314718056f;
    }
    if (threadIdx.x == 128 && ends_for_others(w.part, whole, w.t1 == at.tiles))
      p.join[cta] = Join{cta - place.first + 1, place.first, place.first_slot, at.q.row0 + at.j * p.unit_tokens,
                         min(p.unit_tokens, at.q.n - at.j * p.unit_tokens), at.h * p.group, p.group, 0};
    // O_i has been read; the next unit's first P V, which overwrites it, is issued only after this warpgroup's next
    // p_full arrival.
    tc::fence_before();
  }
  if (!ok && lane == 0) {
    atomicOr(&g_svx_paged_timeouts, SVX_STATUS_WAIT_TIMEOUT);
    if (p.status) atomicOr(p.status + w.at.s, SVX_STATUS_WAIT_TIMEOUT);
  }
  tc::fence_before();
  __syncwarp();
  asm volatile("barrier.arrive 1, %0;" ::"n"(kThreads) : "memory");
}

// The joining of a unit's parts (see join_kernel of the few rows), 32 rows x 32 columns at a time: a lane reads its row's
// columns of a part; neighbouring rows are neighbours in memory.
//
// Few parts: a warp a piece, written through shared memory. Many, as the units of a long sequence have (up to one for
// every CTA): four warps a piece share the parts, meet in shared memory, and each writes eight of the columns (2 sequences
// of 8 tokens x 8 heads of 128 over 12,000 keys: 22 us for the call against 39; with it alone, 8 windows of 1024 rows take
// 189 us against 185). Up to 4 parts are few: a boundary at 1 takes 63.8 us for 32 sequences of 5 tokens x 8 heads and 16.5
// for 2 of 8 x 4 over 2000 keys, at 2 61 and 14.8, at 4 60.5 and 14.6, at 8 63.2 and 18.1.
constexpr int kFewParts = 4;

template <typename T, int D>
__device__ __forceinline__ void join_few_parts(const Params& p, const Join& join, uint8_t* stages) {
  const int warp = warp_id(), lane = lane_id(), task = blockIdx.y * 8 + warp;
  uint8_t* stage = stages + warp * 32 * 64;
  const int r = task / (D / 32) * 32 + lane, c = task % (D / 32) * 32, in_tile = r % p.tile_rows;
  const int token = r / p.tile_rows * p.tile_tokens + in_tile / join.group;
  const bool live = r < p.rows && in_tile < p.tile_tokens * join.group && token < join.tokens;
  if (!__any_sync(0xffffffffu, live)) return;
  float top = -INFINITY, total = 0.f, f[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) f[j] = 0.f;
  if (live) {
    const float4* src = reinterpret_cast<const float4*>(p.partial_o) + c / 4 * p.rows + r;
#pragma unroll 2
    for (int i = 0; i < join.parts; ++i) {   // the loads of two parts are on their way together
      const float2 ml = p.partial_ml[join.slot(i) * p.rows + r];
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = src[join.slot(i) * p.rows * (D / 4) + k * p.rows];
      const float now = fmaxf(top, ml.x);
      const float old = top == now ? 1.f : tc::ex2(top - now), x = ml.x == now ? 1.f : tc::ex2(ml.x - now);
      top = now;
      total = fmaf(ml.y, x, total * old);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[4 * k] = fmaf(v[k].x, x, f[4 * k] * old);
        f[4 * k + 1] = fmaf(v[k].y, x, f[4 * k + 1] * old);
        f[4 * k + 2] = fmaf(v[k].z, x, f[4 * k + 2] * old);
        f[4 * k + 3] = fmaf(v[k].w, x, f[4 * k + 3] * old);
      }
    }
  }
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  const int64_t row0 = (int64_t)join.row * p.q_heads + join.head;
  const int out_row = live ? token * p.q_heads + in_tile % join.group : -1;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16)) =
        make_uint4(Kind<T>::pack(f[8 * k] * inverse, f[8 * k + 1] * inverse),
                   Kind<T>::pack(f[8 * k + 2] * inverse, f[8 * k + 3] * inverse),
                   Kind<T>::pack(f[8 * k + 4] * inverse, f[8 * k + 5] * inverse),
                   Kind<T>::pack(f[8 * k + 6] * inverse, f[8 * k + 7] * inverse));
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int q = 8 * k + lane / 4, piece = lane % 4, to_row = __shfl_sync(0xffffffffu, out_row, q);
    const uint4 x = *reinterpret_cast<const uint4*>(stage + q * 64 + ((piece ^ ((q >> 1) & 3)) * 16));
    if (to_row >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (row0 + to_row) * D + c + piece * 8) = x;
  }
  if (live && c == 0 && p.lse)
    p.lse[row0 + out_row] = total == 0.f ? -INFINITY : (top - Kind<T>::shift + log2f(total)) * 0.69314718056f;
}

template <typename T, int D>
__device__ __forceinline__ void join_many_parts(const Params& p, const Join& join, float4 (&s_f)[8][8][32], float2 (&s_ml)[8][32]) {
  const int warp = warp_id(), lane = lane_id(), share = warp % 4, task = blockIdx.y * 2 + warp / 4;
  const int r = task / (D / 32) * 32 + lane, c = task % (D / 32) * 32, in_tile = r % p.tile_rows;
  const int token = r / p.tile_rows * p.tile_tokens + in_tile / join.group;
  const bool live = r < p.rows && in_tile < p.tile_tokens * join.group && token < join.tokens;
  float top = -INFINITY, total = 0.f;
  float4 f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    const float4* src = reinterpret_cast<const float4*>(p.partial_o) + c / 4 * p.rows + r;
#pragma unroll 2
    for (int i = share; i < join.parts; i += 4) {   // the loads of two parts are on their way together
      const float2 ml = p.partial_ml[join.slot(i) * p.rows + r];
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = src[join.slot(i) * p.rows * (D / 4) + k * p.rows];
      const float now = fmaxf(top, ml.x);
      const float old = top == now ? 1.f : tc::ex2(top - now), x = ml.x == now ? 1.f : tc::ex2(ml.x - now);
      top = now;
      total = fmaf(ml.y, x, total * old);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k].x = fmaf(v[k].x, x, f[k].x * old);
        f[k].y = fmaf(v[k].y, x, f[k].y * old);
        f[k].z = fmaf(v[k].z, x, f[k].z * old);
        f[k].w = fmaf(v[k].w, x, f[k].w * old);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) s_f[warp][k][lane] = f[k];
  s_ml[warp][lane] = make_float2(top, total);
  __syncthreads();
  if (!live) return;
  const int w0 = warp - share;
  top = s_ml[w0][lane].x;
#pragma unroll
  for (int x = 1; x < 4; ++x) top = fmaxf(top, s_ml[w0 + x][lane].x);
  total = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float2 ml = s_ml[w0 + x][lane];
    const float y = ml.x == top ? 1.f : tc::ex2(ml.x - top);
    const float4 u = s_f[w0 + x][2 * share][lane], v = s_f[w0 + x][2 * share + 1][lane];
    total = fmaf(ml.y, y, total);
    a.x = fmaf(u.x, y, a.x); a.y = fmaf(u.y, y, a.y); a.z = fmaf(u.z, y, a.z); a.w = fmaf(u.w, y, a.w);
    b.x = fmaf(v.x, y, b.x); b.y = fmaf(v.y, y, b.y); b.z = fmaf(v.z, y, b.z); b.w = fmaf(v.w, y, b.w);
  }
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  const int64_t out_row = (int64_t)(join.row + token) * p.q_heads + join.head + in_tile % join.group;
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row * D + c + share * 8) =
      make_uint4(Kind<T>::pack(a.x * inverse, a.y * inverse), Kind<T>::pack(a.z * inverse, a.w * inverse),
                 Kind<T>::pack(b.x * inverse, b.y * inverse), Kind<T>::pack(b.z * inverse, b.w * inverse));
  if (c == 0 && share == 0 && p.lse)
    p.lse[out_row] = total == 0.f ? -INFINITY : (top - Kind<T>::shift + log2f(total)) * 0.69314718056f;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const Params p) {
  __shared__ float4 s_f[8][8][32];
  __shared__ float2 s_ml[8][32];
  grid_dependency_wait();
  const Join join = p.join[blockIdx.x];
  if (join.parts > kFewParts) join_many_parts<T, D>(p, join, s_f, s_ml);
  else if (join.parts) join_few_parts<T, D>(p, join, reinterpret_cast<uint8_t*>(s_f));
}

template <typename T, int D, int kChains>
int launch(const Maps& maps, const Params& p, int ctas, cudaStream_t stream) {
  using C = Tiles<D, kChains>;
  static PerDevice<int> ready;
  int unused;
  int rc = ready.get(&unused, [](int, int*) -> int {
    SVX_CHECK_CUDA(cudaFuncSetAttribute(chunk_kernel<T, D, kChains>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem));
    return SVX_OK;
  });
  if (!rc) rc = launch_dependent("chunk_kernel", chunk_kernel<T, D, kChains>, dim3(ctas), dim3(C::threads), C::smem, stream, maps, p);
  if (rc) return rc;
  return launch_dependent("chunk_join_kernel", chunk_join_kernel<T, D>, dim3(ctas, p.rows / 32 * (D / 32) / 2), dim3(256), 0, stream, p);
}

template <typename T>
int launch(const Maps& maps, const Params& p, int dim, int ctas, cudaStream_t stream) {
  const bool two = p.unit_tokens > p.tile_tokens;
  if (dim == 64) return two ? launch<T, 64, 2>(maps, p, ctas, stream) : launch<T, 64, 1>(maps, p, ctas, stream);
  if (dim == 96) return two ? launch<T, 96, 2>(maps, p, ctas, stream) : launch<T, 96, 1>(maps, p, ctas, stream);
  return two ? launch<T, 128, 2>(maps, p, ctas, stream) : launch<T, 128, 1>(maps, p, ctas, stream);
}

}  // namespace

int chunk_launch(const Params& p, int dtype, int dim, int ctas, cudaStream_t stream) {
  Maps maps;
  const int page = 1 << p.page_shift, box = page < TK ? page : TK, tile_tokens = p.tile_tokens;
  const uint64_t pools = (uint64_t)p.pages * p.kv_heads;
  int rc = make_map_3d(&maps.q, p.q, dim, p.q_heads, p.tokens, p.q_head * 2, p.q_token * 2, 64, tile_tokens,
                       CU_TENSOR_MAP_SWIZZLE_128B, p.group);
  if (!rc) rc = make_map_3d(&maps.k, p.k, dim, pools, page, (uint64_t)page * dim * 2, dim * 2, 64, box);
  if (!rc) rc = make_map_3d(&maps.v, p.v, dim, pools, page, (uint64_t)page * dim * 2, dim * 2, 64, box);
  if (rc) return rc;
  if (dtype == SVX_BF16) return launch<__nv_bfloat16>(maps, p, dim, ctas, stream);
  return launch<__half>(maps, p, dim, ctas, stream);
}

}  // namespace paged
}  // namespace svx
