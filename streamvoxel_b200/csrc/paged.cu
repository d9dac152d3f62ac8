// Attention of new tokens over a paged cache: the form for few query rows (decoding), the joining kernel, and the
// entry point that picks the form.
//
//   out[row] = softmax(scale q k^T) v over the keys that the row sees, kv head = head / group
//
// One pass over the keys with a running maximum m and sum l per row; o, m and l stay in fp32 registers:
//   m' = max(m, max s), o = o 2^(m - m') + p v, l = l 2^(m - m') + sum p, p = 2^(s - m')
// (s in log2 units). The weights p are rounded to the cache's type for the product with v, while l sums them
// unrounded: the rounding of each weight (at most 2^-8 bf16, 2^-11 fp16) is random and averages out over keys, and a row with
// one dominant key has p = 1 there, which is exact. For fp16, whose least step is 2^-24, weights are held 2^7 larger.
//
// Bound: the keys and values are read once for the whole group of query heads that share them, so a step with few rows
// is bound by memory. A group's rows are packed into one 16-row matrix tile (mma.sync m16n8k16; the tensor work is a
// small fraction of its rate, and tcgen05's 128-row tiles would be 7/8 padding). The line of all 64-key tiles of the
// batch (paged.cuh) is cut into equal runs, one per CTA: unequal lengths, one long sequence or many short ones all load
// the card evenly. Each of a CTA's four warps streams its own 16 keys of every tile through a private ring of cp.async
// stages, so the loop has no block barrier; the warps' parts of a unit are merged through shared memory at its end.
//
// Measured on B200 (bf16 unless said): 128 sequences of 40 to 16,384 keys, 8 kv heads of 128, 4 query heads each, pages of
// 16: 275 to 284 us, 5.6 TB/s; three of 90,000 to 131,072, 16 heads of 64 in fp16, pages of 128: 212 to 219 us, 6.1 TB/s; one
// of 4001 keys, 8 heads of 128: 11.7 us, of which 1.5 are the plan, 1.8 the first page ids, 1.3 the keys, 1.2 the merge and 3.5 the
// joining kernel with the gap before it.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace svx {

int check_cache(const svx_paged_cache* c, const char* who, int* shift) {
  const std::string at = std::string(who) + ": ";
  SVX_REQUIRE(c, at + "null cache");
  SVX_REQUIRE(c->dtype == SVX_BF16 || c->dtype == SVX_F16, at + "the cache must be bf16 or fp16");
  SVX_REQUIRE(c->pages > 0 && c->kv_heads > 0 && c->kv_heads <= 1024, at + "bad page or head count");
  SVX_REQUIRE(c->dim > 0 && c->dim % 8 == 0 && c->dim <= 1024, at + "dim must be a multiple of 8, at most 1024");
  SVX_REQUIRE(c->page >= 16 && c->page <= 1024 && (c->page & (c->page - 1)) == 0,
              at + "a page must hold 16, 32, .. 1024 keys");
  SVX_REQUIRE(c->sequences >= 0 && c->sequences <= (1 << 20), at + "bad sequence count");
  SVX_REQUIRE(c->table_width > 0 && (int64_t)c->table_width * c->page <= (1 << 30), at + "bad table width");
  SVX_REQUIRE(c->k && c->v && (!c->sequences || (c->table && c->lengths && c->offsets)), at + "null cache arrays");
  SVX_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) == 0,
              at + "pools must be 16-byte aligned");
  *shift = 0;
  while ((1 << *shift) < c->page) ++*shift;
  return SVX_OK;
}

namespace paged {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16;

template <typename T> struct Half;   // the two 16-bit types
template <> struct Half<__nv_bfloat16> {
  static constexpr float shift = 0.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Half<__half> {
  static constexpr float shift = 7.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes to shared memory, zeros where !take (the source is then not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0)
               : "memory");
}

template <int D> struct Shape {
  static constexpr int chunks = D / 8;                  // 16-byte pieces of a row
  static constexpr int row_bytes = (chunks + 1) * 16;   // odd in 16-byte units: ldmatrix rows fall into distinct banks
  static constexpr int stage_bytes = 2 * 16 * row_bytes;
  // CTAs of a SM and stages of a warp's ring: what keeps the most keys in flight within the registers (128, 168 and 220 a
  // thread) and shared memory.
  static constexpr int ctas_per_sm = D == 64 ? 4 : D == 96 ? 3 : 2;
  static constexpr int stages = D == 128 ? 3 : 2;
  static constexpr int merge_stride = D + 8;            // floats of a merged row: conflict-free for the fragments' layout
  static_assert(kRows * merge_stride * 4 <= stage_bytes, "a warp's part of a unit takes the place of a stage");
  static constexpr size_t smem = (size_t)kWarps * stages * stage_bytes;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, Shape<D>::ctas_per_sm) few_rows_kernel(const Params p) {
  using S = Shape<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ PlanShared plan_shared;
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  const int warp = warp_id(), lane = lane_id(), cta = blockIdx.x;
  const uint32_t ring = smem_addr(smem + warp * S::stages * S::stage_bytes);
  grid_launch_dependents();
  grid_dependency_wait();
  plan<kThreads, false>(p, cta, gridDim.x, plan_shared, nullptr);
  const Place& place = plan_shared.place;
  const int count = place.count;
  if (threadIdx.x == 0) p.join[cta].parts = 0;
  if (count <= 0) return;

  // The loading side: a cursor up to stages - 1 tiles ahead, with the next slice's page id already on its way.
  Cursor ahead;
  ahead.set(p, place);
  int ahead_t = place.t, issued = 0, page = 0;
  auto look_up = [&] {
    const int key = ahead_t * kTile + warp * 16;
    page = key < ahead.limit ? __ldg(p.table + (int64_t)ahead.s * p.table_width + (key >> p.page_shift)) : 0;
  };
  look_up();
  auto issue = [&] {
    if (issued < count) {
      const int key = ahead_t * kTile + warp * 16;
      int valid = max(0, min(16, ahead.limit - key));
      if (page < 0 || page >= p.pages) {
        if (p.status && lane == 0) atomicOr(p.status + ahead.s, SVX_STATUS_BAD_PAGE);
        page = 0;
        valid = 0;
      }
      const int head = ahead.h / p.blocks;
      const int64_t row = (((int64_t)page * p.kv_heads + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
      const T* k = static_cast<const T*>(p.k) + row * D;
      const T* v = static_cast<const T*>(p.v) + row * D;
      const uint32_t stage = ring + issued % S::stages * S::stage_bytes;
#pragma unroll
      for (int i = 0; i < S::chunks / 2; ++i) {
        const int e = lane + 32 * i, r = e / S::chunks, c = e % S::chunks;
        copy16(stage + r * S::row_bytes + c * 16, k + r * D + c * 8, r < valid);
      }
#pragma unroll
      for (int i = 0; i < S::chunks / 2; ++i) {
        const int e = lane + 32 * i, r = e / S::chunks, c = e % S::chunks;
        copy16(stage + 16 * S::row_bytes + r * S::row_bytes + c * 16, v + r * D + c * 8, r < valid);
      }
      ++issued;
      if (++ahead_t == ahead.tiles) {
        ahead_t = 0;
        ahead.next(p);
      }
      if (issued < count) look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < S::stages - 1; ++i) issue();

  Cursor at;
  at.set(p, place);
  int t = place.t, segment = 0;
  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2], l[2];
  int limit[2];
  auto start_unit = [&] {
    if (threadIdx.x == 0 && p.status) {
      const int raw = __ldg(p.lengths + at.s);
      if (raw != at.q.len) atomicOr(p.status + at.s, SVX_STATUS_BAD_PAGE);
    }
    const int g0 = at.h % p.blocks * p.group_part, part = min(p.group_part, p.group - g0);
    const int token0 = at.j * p.unit_tokens, tokens = min(p.unit_tokens, at.q.n - token0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = lane / 4 + 8 * u, token = r / part;
      const bool live = token < tokens;
      limit[u] = !live ? 0 : p.causal ? max(0, min(at.q.len, at.q.len - at.q.n + token0 + token + 1)) : at.q.len;
      const T* q = static_cast<const T*>(p.q) + (int64_t)(at.q.row0 + token0 + token) * p.q_token +
                   (int64_t)(at.h / p.blocks * p.group + g0 + r - token * part) * p.q_head + lane % 4 * 2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][u] = live ? __ldg(reinterpret_cast<const unsigned int*>(q + kk * 16)) : 0u;
        qf[kk][u + 2] = live ? __ldg(reinterpret_cast<const unsigned int*>(q + kk * 16 + 8)) : 0u;
      }
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  };
  start_unit();
  clear();
  for (int i = 0; i < count; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::stages - 2) : "memory");
    __syncwarp();
    issue();   // into the stage read last time round
    const uint32_t stage = ring + i % S::stages * S::stage_bytes;

    // S = Q K^T: K's rows are the columns of the product. Lanes 0-15 address keys 0-7, 16-31 keys 8-15; every other
    // eight the second half of 16 dims.
    float s[2][4] = {};
    const uint32_t k_at = stage + ((lane & 7) + (lane >> 4) * 8) * S::row_bytes + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t b[4];
      ldmatrix4(b, k_at + kk * 32);
      Half<T>::mma(s[0], qf[kk], b[0], b[1]);
      Half<T>::mma(s[1], qf[kk], b[2], b[3]);
    }
    const int key0 = t * kTile + warp * 16 + lane % 4 * 2;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float& x = s[nt][e];
        x = key0 + nt * 8 + (e & 1) < limit[e >> 1] ? x * p.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], x);
      }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 1));
      top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 2));
    }
    const bool grows = top[0] > m[0] || top[1] > m[1];
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float now = fmaxf(m[u], top[u]);
        const float f = m[u] == now ? 1.f : exp2_approx(m[u] - now);   // m = -inf: 0
        m[u] = now;
        l[u] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * u] *= f;
          o[d][2 * u + 1] *= f;
        }
      }
    }
    float w[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float base = m[u] == -INFINITY ? 0.f : m[u] - Half<T>::shift;   // a row without keys so far: weights 0
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = exp2_approx(s[nt][2 * u + e] - base);
          w[nt][2 * u + e] = x;
          l[u] += x;
        }
    }
    const uint32_t a[4] = {Half<T>::pack(w[0][0], w[0][1]), Half<T>::pack(w[0][2], w[0][3]),
                           Half<T>::pack(w[1][0], w[1][1]), Half<T>::pack(w[1][2], w[1][3])};
    const uint32_t v_at = stage + 16 * S::row_bytes + (lane & 15) * S::row_bytes + (lane >> 4) * 16;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t b[4];
      ldmatrix4_trans(b, v_at + d * 32);
      Half<T>::mma(o[2 * d], a, b[0], b[1]);
      Half<T>::mma(o[2 * d + 1], a, b[2], b[3]);
    }
    ++t;
    if (t < at.tiles && i + 1 < count) continue;

    // The unit's end, or the run's: merge the warps' parts, with the next unit's queries on their way.
    const bool whole = (segment || place.t == 0) && t == at.tiles;
    const bool ends_others = ends_for_others(segment, whole, t == at.tiles);
    const int64_t slot = partial_slot(cta, segment);
    const int g0 = at.h % p.blocks * p.group_part, part = min(p.group_part, p.group - g0);
    const int token0 = at.j * p.unit_tokens, tokens = min(p.unit_tokens, at.q.n - token0);
    const int row0 = at.q.row0 + token0, head0 = at.h / p.blocks * p.group + g0;
    if (i + 1 < count) {
      at.next(p);
      start_unit();
    }
    // Each warp leaves its part in the stage that it has just read, which is not loaded again before the second barrier.
    float* mine = reinterpret_cast<float*>(smem + (warp * S::stages + i % S::stages) * S::stage_bytes);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = lane / 4 + 8 * u;
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      if (lane % 4 == 0) {
        s_m[warp][r] = m[u];
        s_l[warp][r] = l[u];
      }
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(mine + r * S::merge_stride + d * 8 + lane % 4 * 2) = make_float2(o[d][2 * u], o[d][2 * u + 1]);
    }
    __syncthreads();
    // One row and four of every 32 columns a thread.
    const int r = threadIdx.x / 8, c = threadIdx.x % 8 * 4;
    float top_r = s_m[0][r], sum_r = 0.f, f[kWarps];
#pragma unroll
    for (int x = 1; x < kWarps; ++x) top_r = fmaxf(top_r, s_m[x][r]);
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      f[x] = s_m[x][r] == top_r ? 1.f : exp2_approx(s_m[x][r] - top_r);
      sum_r += s_l[x][r] * f[x];
    }
    const bool live = r < tokens * part;
    const int64_t out_row = (int64_t)(row0 + r / part) * p.q_heads + head0 + r % part;
    const float inverse = sum_r == 0.f ? 0.f : 1.f / sum_r;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float4 v = *reinterpret_cast<const float4*>(smem + (x * S::stages + i % S::stages) * S::stage_bytes +
                                                          (r * S::merge_stride + k * 32 + c) * 4);
        sum.x = fmaf(v.x, f[x], sum.x); sum.y = fmaf(v.y, f[x], sum.y);
        sum.z = fmaf(v.z, f[x], sum.z); sum.w = fmaf(v.w, f[x], sum.w);
      }
      // A row without keys: its weights of 0 have made NaN of infinite values that other rows of the unit see.
      if (sum_r == 0.f) sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!whole) {
        *reinterpret_cast<float4*>(p.partial_o + (slot * p.rows + r) * D + k * 32 + c) = sum;
      } else if (live) {
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + out_row * D + k * 32 + c) =
            make_uint2(Half<T>::pack(sum.x * inverse, sum.y * inverse), Half<T>::pack(sum.z * inverse, sum.w * inverse));
      }
    }
    __syncthreads();
    if (threadIdx.x % 8 == 0) {
      if (!whole) {
        p.partial_ml[slot * p.rows + r] = make_float2(top_r, sum_r);
      } else if (live && p.lse) {
        p.lse[out_row] = sum_r == 0.f ? -INFINITY : (top_r - Half<T>::shift + log2f(sum_r)) * 0.69314718056f;
      }
    }
    if (threadIdx.x == 0 && ends_others)
      p.join[cta] = Join{cta - place.first + 1, place.first, place.first_slot, row0, tokens, head0, part, 0};
    ++segment;
    t = 0;
    clear();
  }
}

// Joins a unit's parts: o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m). Block (c, y): the unit that CTA c ended, rows 2 y and
// 2 y + 1, four warps a row that share its parts (up to one for every CTA). Reads the partial sums once; they are in L2.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  grid_dependency_wait();
  const Join join = p.join[blockIdx.x];
  if (!join.parts) return;
  constexpr int kWarpsRow = 4, rows = 8 / kWarpsRow;
  const int warp = warp_id(), lane = lane_id(), share = warp % kWarpsRow;
  const int r = blockIdx.y * rows + warp / kWarpsRow, token = r / join.group;
  const bool live = token < join.tokens;
  auto slot = [&](int i) { return join.slot(i) * p.rows + r; };
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, total = 0.f;
  if (live) {
    for (int i0 = share; i0 < join.parts; i0 += 32 * kWarpsRow) {
      const int i = i0 + kWarpsRow * lane, here = min(32, (join.parts - i0 + kWarpsRow - 1) / kWarpsRow);   // this warp's parts
      float2 ml = make_float2(-INFINITY, 0.f);
      if (i < join.parts) ml = p.partial_ml[slot(i)];
      // Eight parts' columns are on their way at a time, the first of them with the bases.
      float4 v[8];
      auto load = [&](int x0) {
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (x0 + x < here && lane < D / 4)
            v[x] = *reinterpret_cast<const float4*>(p.partial_o + slot(i0 + kWarpsRow * (x0 + x)) * D + 4 * lane);
      };
      load(0);
      float now = ml.x;
#pragma unroll
      for (int d = 16; d; d >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
      now = fmaxf(now, top);
      const float old = top == now ? 1.f : exp2_approx(top - now);
      const float f = ml.x == now ? 1.f : exp2_approx(ml.x - now);
      float add = ml.y * f;
#pragma unroll
      for (int d = 16; d; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
      total = total * old + add;
      sum.x *= old; sum.y *= old; sum.z *= old; sum.w *= old;
      top = now;
      for (int x0 = 0;;) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float fx = __shfl_sync(0xffffffffu, f, (x0 + x) & 31);
          if (x0 + x < here && lane < D / 4) {
            sum.x = fmaf(v[x].x, fx, sum.x); sum.y = fmaf(v[x].y, fx, sum.y);
            sum.z = fmaf(v[x].z, fx, sum.z); sum.w = fmaf(v[x].w, fx, sum.w);
          }
        }
        x0 += 8;
        if (x0 >= here) break;
        load(x0);
      }
    }
  }
  __shared__ float4 s_o[8][32];
  __shared__ float2 s_ml[8];
  s_o[warp][lane] = sum;
  if (lane == 0) s_ml[warp] = make_float2(top, total);
  __syncthreads();
  if (share) return;
#pragma unroll
  for (int x = 1; x < kWarpsRow; ++x) {
    const float2 other = s_ml[warp + x];
    const float4 v = s_o[warp + x][lane];
    const float now = fmaxf(top, other.x);
    const float f = top == now ? 1.f : exp2_approx(top - now), g = other.x == now ? 1.f : exp2_approx(other.x - now);
    total = total * f + other.y * g;
    sum.x = sum.x * f + v.x * g; sum.y = sum.y * f + v.y * g;
    sum.z = sum.z * f + v.z * g; sum.w = sum.w * f + v.w * g;
    top = now;
  }
  if (!live) return;
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  const int64_t out_row = (int64_t)(join.row + token) * p.q_heads + join.head + r % join.group;
  if (lane < D / 4)
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + out_row * D + 4 * lane) =
        make_uint2(Half<T>::pack(sum.x * inverse, sum.y * inverse), Half<T>::pack(sum.z * inverse, sum.w * inverse));
  if (lane == 0 && p.lse)
    p.lse[out_row] = total == 0.f ? -INFINITY : (top - Half<T>::shift + log2f(total)) * 0.69314718056f;
}

int sm_count(int* sms) {
  static PerDevice<int> per_device;
  return per_device.get(sms, [](int device, int* count) -> int {
    SVX_CHECK_CUDA(cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device));
    return SVX_OK;
  });
}

template <typename T, int D>
int few_rows_launch(const Params& p, int ctas, cudaStream_t stream) {
  static PerDevice<int> ready;
  int unused;
  const int rc = ready.get(&unused, [](int, int*) -> int {
    SVX_CHECK_CUDA(cudaFuncSetAttribute(few_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<D>::smem));
    return SVX_OK;
  });
  if (rc) return rc;
  return launch_dependent("few_rows_kernel", few_rows_kernel<T, D>, dim3(ctas), dim3(kThreads), Shape<D>::smem, stream, p);
}

// How a call is divided: set from its shape alone, so that the workspace's size and the launch agree.
struct Division {
  bool chunk;   // the form for many rows
  int group_part, blocks, unit_tokens, tile_tokens, tile_rows, rows, ctas, min_tiles;
};

int divide(int tokens, int sequences, int group, int dim, int max_query, bool chunk_fits, Division* d) {
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  // Rows for each key: of the longest chunk where the caller knows it, else of the mean one.
  const int64_t query = max_query > 0 ? std::min(max_query, tokens) : (tokens + sequences - 1) / std::max(sequences, 1);
  // With 17 to 32 rows the few-rows form reads the keys twice: 92 us against 60 for 32 sequences of 300 to 12,000 keys, 4 kv
  // heads of 128; 17 against 21 for two such sequences, where latency counts.
  d->chunk = chunk_fits && query * group > kRows && group <= 128;
  if (d->chunk) {
    d->group_part = group;
    d->blocks = 1;
    d->tile_tokens = 128 / group;
    // Query tiles of a unit, and then one or two CTAs a SM. Two share the keys' way to the SM (16 chunks of 512 tokens x 4
    // heads of 128 over 4000 keys: 530 us against 673); one wastes less on chunks that fit a tile (32 of 5
    // tokens x 8 heads of 128: 62 us against 83). Where the longest chunk is far above the mean, most sequences are short
    // and leave half of a two-tile CTA idle, even beside one long chunk. One tile against two, group 4 of 128 unless said:
    //   mean of at most 3 tiles: 8192 tokens and 255 single ones 965 us against 1107, 4 x 2000 and 200 single 639 against
    //   706, 64 sequences of one or 300 204 against 241, 16 of 1 to 2000 64 against 76; but 2000 and 31 single 184 against 150;
    //   3 to 8 tiles: 100 of 1 to 700 tokens 648 against 598, 100 of 1 to 2048 1550 against 1389, 2 x 2000 and 30 single
    //   (group 8) 218 against 189, 24 of 1 to 700 159 against 171; with 64-wide heads, which load half as much for each
    //   product, 64 of 1 to 300 (group 6) 136 against 161, 24 of 1 to 700 90 against 101;
    //   above: 16 of 1 to 2000, 52 tiles in the mean (group 6 of 64), 592 against 577; 128-wide, 37 tiles, 1044 against 893.
    const int64_t mean = tokens / std::max(sequences, 1);
    const bool skewed = max_query > 0 && 4 * mean <= query && mean <= (dim > 96 ? 3 : 8) * d->tile_tokens;
    const int tiles = query > d->tile_tokens && !skewed ? 2 : 1;
    d->unit_tokens = tiles * d->tile_tokens;
    d->tile_rows = 128;
    d->rows = 128 * tiles;
    d->ctas = sms * (3 - tiles);
    d->min_tiles = 4;
  } else {
    d->group_part = std::min(group, kRows);
    d->blocks = (group + kRows - 1) / kRows;
    d->unit_tokens = d->tile_tokens = kRows / d->group_part;
    d->tile_rows = d->rows = kRows;
    d->ctas = sms * (dim == 64 ? Shape<64>::ctas_per_sm : dim == 96 ? Shape<96>::ctas_per_sm : Shape<128>::ctas_per_sm);
    d->min_tiles = 2;
  }
  return SVX_OK;
}

size_t workspace_bytes(const Division& d, int dim) {
  return (size_t)d.ctas * (sizeof(Join) + 2 * (size_t)d.rows * (dim * sizeof(float) + sizeof(float2)));
}

template <typename T, int D>
int launch_all(const Params& p, const Division& d, int dtype, cudaStream_t stream) {
  if (d.chunk) return chunk_launch(p, dtype, D, d.ctas, stream);
  if (const int rc = few_rows_launch<T, D>(p, d.ctas, stream)) return rc;
  return launch_dependent("join_kernel", join_kernel<T, D>, dim3(d.ctas, d.rows / 2), dim3(256), 0, stream, p);
}

template <typename T>
int launch_all(const Params& p, const Division& d, int dtype, int dim, cudaStream_t stream) {
  if (dim == 64) return launch_all<T, 64>(p, d, dtype, stream);
  if (dim == 96) return launch_all<T, 96>(p, d, dtype, stream);
  return launch_all<T, 128>(p, d, dtype, stream);
}

int check_attention(int tokens, int q_heads, int kv_heads, int dim) {
  SVX_REQUIRE(dim == 64 || dim == 96 || dim == 128, "svx_paged_attention: dim must be 64, 96 or 128");
  SVX_REQUIRE(kv_heads > 0 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 4096,
              "svx_paged_attention: the query heads must be a multiple of the cache's");
  SVX_REQUIRE(tokens >= 0, "svx_paged_attention: bad token count");
  return SVX_OK;
}

}  // namespace
}  // namespace paged
}  // namespace svx

using namespace svx;

extern "C" size_t svx_paged_attention_workspace_bytes(int tokens, int sequences, int q_heads, int kv_heads, int dim,
                                                      int max_query) {
  if (sequences < 0 || paged::check_attention(tokens, q_heads, kv_heads, dim)) return 0;
  paged::Division d;
  if (paged::divide(tokens, sequences, q_heads / kv_heads, dim, max_query, true, &d)) return 0;
  return paged::workspace_bytes(d, dim);
}

extern "C" int svx_paged_attention(const svx_paged_cache* cache, const void* q, int64_t q_token_stride,
                                   int64_t q_head_stride, int tokens, int q_heads, int causal, float scale, void* out,
                                   float* lse, int max_query, void* workspace, void* stream) {
  int shift = 0;
  if (const int rc = check_cache(cache, "svx_paged_attention", &shift)) return rc;
  if (const int rc = paged::check_attention(tokens, q_heads, cache->kv_heads, cache->dim)) return rc;
  SVX_REQUIRE(scale > 0.f && scale <= 1e30f, "svx_paged_attention: scale must be positive and finite");
  if (!tokens || !cache->sequences) return SVX_OK;
  SVX_REQUIRE(q && out && workspace, "svx_paged_attention: null arguments");
  if (tokens == 1) q_token_stride = (int64_t)q_heads * cache->dim;   // one token, one head: any stride will do
  if (q_heads == 1) q_head_stride = cache->dim;
  SVX_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0,
              "svx_paged_attention: strides of q must be multiples of 8 elements");
  SVX_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0,
              "svx_paged_attention: operands must be 16-byte aligned");
  paged::Division d;
  // The form for many rows reads through tensor maps, whose strides are positive and whose coordinates have 32 bits; the
  // other one takes everything, and less workspace.
  const bool fits = q_token_stride > 0 && q_head_stride > 0 && (int64_t)cache->pages * cache->kv_heads < INT32_MAX;
  if (const int rc = paged::divide(tokens, cache->sequences, q_heads / cache->kv_heads, cache->dim, max_query, fits, &d)) return rc;
  paged::Params p{};
  p.q = q;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.k = cache->k;
  p.v = cache->v;
  p.table = cache->table;
  p.lengths = cache->lengths;
  p.offsets = cache->offsets;
  p.out = out;
  p.lse = lse;
  p.status = cache->status;
  const size_t rows = 2 * (size_t)d.ctas * d.rows;
  p.partial_o = static_cast<float*>(workspace);
  p.partial_ml = reinterpret_cast<float2*>(p.partial_o + rows * cache->dim);
  p.join = reinterpret_cast<paged::Join*>(p.partial_ml + rows);
  p.tokens = tokens;
  p.sequences = cache->sequences;
  p.q_heads = q_heads;
  p.kv_heads = cache->kv_heads;
  p.group = q_heads / cache->kv_heads;
  p.page_shift = shift;
  p.pages = cache->pages;
  p.table_width = cache->table_width;
  p.causal = causal != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.unit_tokens = d.unit_tokens;
  p.blocks = d.blocks;
  p.group_part = d.group_part;
  p.tile_tokens = d.tile_tokens;
  p.tile_rows = d.tile_rows;
  p.rows = d.rows;
  p.min_tiles = d.min_tiles;
  if (cache->dtype == SVX_BF16)
    return paged::launch_all<__nv_bfloat16>(p, d, cache->dtype, cache->dim, as_stream(stream));
  return paged::launch_all<__half>(p, d, cache->dtype, cache->dim, as_stream(stream));
}
