// Rotary positions by themselves (svx_rope) and on the way into a paged cache (svx_paged_append).
//
// Each pair (a, b) of a head's first `rot` values turns by the angle position * inv_freq[pair]:
//   (a, b) -> scale * (a cos - b sin, a sin + b cos)
// and the values past `rot` are copied. The backward pass is the transposed turn, the same kernel with the sine's sign
// flipped. Interleaved pairs are (2j, 2j + 1), half pairs (j, j + rot / 2); with several position axes the pairs are
// split evenly among them, axis-major (the axial rotation of the GEMM epilogue).
//
// Both operators are one pass over their rows and bound by memory once the rows outgrow L2, if they spend few instructions
// and keep many loads in flight. A warp takes a token (or, of few tokens, a share of one): it sets off its first rows' loads
// of 16 bytes a lane, then looks up the token's place in the cache and computes its cosines and sines, once for all heads,
// which hides that chain of small loads behind the rows; no step waits for another warp. The angle is formed in float64
// and reduced to an eighth of a turn there (positions of a million lose 2e-2 of a radian in 32 bits), the rest is fp32; a
// value is rounded to its own type once.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace svx {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxPairs = 256;

// Rows to move: [tokens][heads][dim] with strides in elements.
struct Rows {
  const void* src;
  void* dst;             // q: strided like src; k, v: the pool
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;
};

struct MoveParams {
  Rows q, k, v;               // q (or svx_rope's x) and k turn, v is copied; k and v go to the pages
  const double* inv_freq;     // null: nothing turns
  const void* positions;      // null: the token's position in the cache
  int position_type, axes, pairs, layout, inverse;
  float scale;
  int tokens, dim;
  int parts;                  // warps of a token
  int items;                  // of a head, see move_rows_kernel
  int step_heads, step_items; // 32 * parts items on, in heads and items
  // cache
  const int32_t *table, *lengths, *offsets;
  uint32_t* status;
  int sequences, table_width, pages, page_shift;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float f);
template <> __device__ __forceinline__ float from_f32<float>(float f) { return f; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }
template <> __device__ __forceinline__ __half from_f32<__half>(float f) { return __float2half_rn(f); }

// N values: one of them, or 16 bytes as words (two 16-bit values or one fp32 value a word).
template <typename T, int N> struct Pack { uint4 w; };
template <typename T> struct Pack<T, 1> { T v; };

__device__ __forceinline__ float2 unpack(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack(__nv_bfloat16, float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ uint32_t pack(__half, float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
  return d;
}

// (f, g) turned by the angle with cosine c and sine s.
__device__ __forceinline__ float2 turned(float f, float g, float c, float s) {
  return make_float2(f * c - g * s, f * s + g * c);
}

// Whole pairs within a vector; cs: their (cos, sin).
template <typename T>
__device__ __forceinline__ void turn_inside(uint4& a, const float2* cs) {
  const float4 x = reinterpret_cast<const float4*>(cs)[0];
  if constexpr (sizeof(T) == 4) {
    const float2 u = turned(__uint_as_float(a.x), __uint_as_float(a.y), x.x, x.y);
    const float2 v = turned(__uint_as_float(a.z), __uint_as_float(a.w), x.z, x.w);
    a = make_uint4(__float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(v.x), __float_as_uint(v.y));
  } else {
    const float4 y = reinterpret_cast<const float4*>(cs)[1];
    auto word = [](uint32_t w, float c, float s) {
      const float2 f = unpack(T(), w), u = turned(f.x, f.y, c, s);
      return pack(T(), u.x, u.y);
    };
    a = make_uint4(word(a.x, x.x, x.y), word(a.y, x.z, x.w), word(a.z, y.x, y.y), word(a.w, y.z, y.w));
  }
}

// Pairs across two vectors.
template <typename T>
__device__ __forceinline__ void turn_across(uint4& a, uint4& b, const float2* cs) {
  if constexpr (sizeof(T) == 4) {
    auto word = [](uint32_t& f, uint32_t& g, float2 t) {
      const float2 u = turned(__uint_as_float(f), __uint_as_float(g), t.x, t.y);
      f = __float_as_uint(u.x);
      g = __float_as_uint(u.y);
    };
    word(a.x, b.x, cs[0]);
    word(a.y, b.y, cs[1]);
    word(a.z, b.z, cs[2]);
    word(a.w, b.w, cs[3]);
  } else {
    auto word = [](uint32_t& f, uint32_t& g, float4 t) {
      const float2 x = unpack(T(), f), y = unpack(T(), g);
      const float2 u = turned(x.x, y.x, t.x, t.y), v = turned(x.y, y.y, t.z, t.w);
      f = pack(T(), u.x, v.x);
      g = pack(T(), u.y, v.y);
    };
    const float4* at = reinterpret_cast<const float4*>(cs);
    word(a.x, b.x, at[0]);
    word(a.y, b.y, at[1]);
    word(a.z, b.z, at[2]);
    word(a.w, b.w, at[3]);
  }
}

// (cos, sin) of 2 pi turns. The turns are reduced to [-1/8, 1/8] in float64, then sine and cosine are their Taylor series up
// to x^9 and x^10 (|x| <= pi / 4: the next terms are under 2e-9), and the quarter turns swap and negate them. Turns from
// 2^49 on, whose eighths float64 does not hold, are reduced to a turn first: the angle means nothing there, but the pair
// still turns (beyond |x| = pi / 4 the series grow without limit).
__device__ __forceinline__ float2 cos_sin_turns(double turns) {
  if ((__double2hiint(turns) & 0x7fffffff) >= (1023 + 49) << 20) turns -= rint(turns);
  // Adding 1.5 * 2^52 rounds to a whole number, which then stands in the low bits (|turns| < 2^49); a rounding and a
  // conversion to integers would take the slow conversion pipe.
  const double sum = fma(4.0, turns, 6755399441055744.0), quarters = sum - 6755399441055744.0;
  const float x = (float)(fma(-0.25, quarters, turns) * 6.283185307179586477);
  const int k = __double2loint(sum) & 3;
  const float z = x * x;
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  const float cs = k & 1 ? s : c, sn = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -cs : cs, k >= 2 ? -sn : sn);
}

// An item of a head is N values, or N and their N partners (kPaired): vectors of the interleaved layout hold whole pairs,
// those of the half layout and single values (N = 1, the form for any dim, stride and alignment) come with a partner.
// Items past the turned values are N values without a partner.
template <typename T, int N, bool kPaired>
struct Items {
  using P = Pack<T, N>;
  const MoveParams& p;
  int turning, rot, partner, first_head, first_item;

  __device__ __forceinline__ Items(const MoveParams& p_, int start) : p(p_) {
    rot = p.inv_freq ? 2 * p.pairs : 0;
    turning = kPaired ? rot / (2 * N) : rot / N;
    partner = p.layout == SVX_ROPE_HALF ? p.pairs : 1;
    first_head = start / p.items;
    first_item = start - first_head * p.items;
  }
  __device__ __forceinline__ int value(int item) const {   // the first value of an item
    if (!kPaired) return item * N;
    if (item >= turning) return rot + (item - turning) * N;
    return N == 1 && p.layout != SVX_ROPE_HALF ? 2 * item : item * N;
  }
  __device__ __forceinline__ void advance(int* head, int* item) const {
    *head += p.step_heads;
    *item += p.step_items;
    if (*item >= p.items) {
      *item -= p.items;
      ++*head;
    }
  }
  __device__ __forceinline__ void load(const T* src, int item, P* a, P* b) const {
    *a = *reinterpret_cast<const P*>(src);
    if (kPaired && item < turning) *b = *reinterpret_cast<const P*>(src + partner);
  }
  __device__ __forceinline__ void turn(const float2* angles, int item, P* a, P* b) const {
    if (item >= turning) return;
    if constexpr (N == 1) {
      const float2 cs = angles[item], u = turned(to_f32(a->v), to_f32(b->v), cs.x, cs.y);
      a->v = from_f32<T>(u.x);
      b->v = from_f32<T>(u.y);
    } else if constexpr (kPaired) {
      turn_across<T>(a->w, b->w, angles + item * N);
    } else {
      turn_inside<T>(a->w, angles + item * (N / 2));
    }
  }
  __device__ __forceinline__ void store(T* dst, int item, const P& a, const P& b) const {
    *reinterpret_cast<P*>(dst) = a;
    if (kPaired && item < turning) *reinterpret_cast<P*>(dst + partner) = b;
  }
};

template <typename T, int N, bool kPaired, bool kPaged>
__global__ void __launch_bounds__(kThreads) move_rows_kernel(const MoveParams p) {
  // Items of a lane in flight, of q alone and of k and v together. Three of q keep 40 to 48 registers a thread, and with
  // them 40 warps a SM (8192 tokens x 16 heads x 96: 11.4 us; six items 12.2, 40 registers enforced 11.4; 16384 x 32 x 128
  // of halves: 45 us, 6.0 TB/s). Of k and v, fewer registers than it takes cost more than warps bring (39 us against 50).
  constexpr int kQ = kPaged ? (kPaired ? 1 : 2) : 3, kKv = kPaired ? 2 : 3;
  __shared__ __align__(16) float2 s_turn[kWarps][kMaxPairs];   // (cos, sin) * scale
  using P = Pack<T, N>;
  grid_launch_dependents();
  grid_dependency_wait();
  const int unit = blockIdx.x * kWarps + warp_id(), lane = lane_id();
  const int t = unit / p.parts, part = unit - t * p.parts;
  if (t >= p.tokens) return;
  const Items<T, N, kPaired> items(p, lane + 32 * part);
  const T* q_src = static_cast<const T*>(p.q.src) + (int64_t)t * p.q.src_token;
  T* q_dst = static_cast<T*>(p.q.dst) + (int64_t)t * p.q.dst_token;
  const T* k_src = static_cast<const T*>(p.k.src) + (int64_t)t * p.k.src_token;
  const T* v_src = static_cast<const T*>(p.v.src) + (int64_t)t * p.v.src_token;

  P qa[kQ], qb[kPaired ? kQ : 1], ka[kKv], kb[kPaired ? kKv : 1], va[kKv], vb[kPaired ? kKv : 1];
  auto load_q = [&](int head, int item) {
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      if (head < p.q.heads)
        items.load(q_src + (int64_t)head * p.q.src_head + items.value(item), item, qa + u, qb + (kPaired ? u : 0));
      items.advance(&head, &item);
    }
  };
  auto load_kv = [&](int head, int item) {
#pragma unroll
    for (int u = 0; u < kKv; ++u) {
      if (head < p.k.heads) {
        const int value = items.value(item);
        items.load(k_src + (int64_t)head * p.k.src_head + value, item, ka + u, kb + (kPaired ? u : 0));
        items.load(v_src + (int64_t)head * p.v.src_head + value, item, va + u, vb + (kPaired ? u : 0));
      }
      items.advance(&head, &item);
    }
  };
  if (kPaged) load_kv(items.first_head, items.first_item);
  load_q(items.first_head, items.first_item);

  int place = 0;       // the token's position in the cache
  int64_t row = -1;    // the row of its key in head 0 of its page, -1: not stored
  if (kPaged) {
    // The token's sequence is the count of sequence ends at or before it; every lane's loads are independent.
    int count = 0;
    for (int i = lane; i < p.sequences; i += 32) count += __ldg(p.offsets + i + 1) <= t;
    const int s = __reduce_add_sync(0xffffffffu, count);
    if (s >= p.sequences) return;
    const int begin = __ldg(p.offsets + s), end = __ldg(p.offsets + s + 1), length = __ldg(p.lengths + s);
    if (t < begin) return;
    const int64_t at = (int64_t)length - end + t;
    bool ok = at >= 0 && at < ((int64_t)p.table_width << p.page_shift);
    place = (int)max((int64_t)-(1 << 30), min(at, (int64_t)1 << 30));
    if (ok) {
      const int page = __ldg(p.table + (int64_t)s * p.table_width + (at >> p.page_shift));
      ok = page >= 0 && page < p.pages;
      if (ok) row = ((int64_t)page * p.k.heads << p.page_shift) + (at & ((1 << p.page_shift) - 1));
    }
    if (!ok && p.status && lane == 0 && part == 0) atomicOr(p.status + s, SVX_STATUS_BAD_PAGE);
  }
  float2* angles = s_turn[warp_id()];
  if (p.inv_freq) {
    const int per_axis = p.pairs / p.axes;
    for (int j = lane; j < p.pairs; j += 32) {
      double position = place;
      if (p.positions) {
        int64_t e = (int64_t)t * p.axes;
        for (int a = per_axis; a <= j; a += per_axis) ++e;   // the pair's axis
        position = p.position_type == SVX_I64   ? (double)static_cast<const int64_t*>(p.positions)[e]
                   : p.position_type == SVX_I32 ? (double)static_cast<const int32_t*>(p.positions)[e]
                                                : (double)static_cast<const float*>(p.positions)[e];
      }
      const float2 cs = cos_sin_turns(position * p.inv_freq[j] * 0.15915494309189533577);   // 1 / (2 pi)
      angles[j] = make_float2(cs.x * p.scale, (p.inverse ? -cs.y : cs.y) * p.scale);
    }
    __syncwarp();
  }

  if (kPaged && row >= 0) {
    T* k_dst = static_cast<T*>(p.k.dst) + row * p.dim;
    T* v_dst = static_cast<T*>(p.v.dst) + row * p.dim;
    const int64_t head_stride = (int64_t)p.dim << p.page_shift;
    int head = items.first_head, item = items.first_item;
    while (head < p.k.heads) {
#pragma unroll
      for (int u = 0; u < kKv; ++u) {
        if (head < p.k.heads) {
          const int64_t offset = head * head_stride + items.value(item);
          constexpr int second = kPaired ? 1 : 0;
          items.turn(angles, item, ka + u, kb + u * second);
          items.store(k_dst + offset, item, ka[u], kb[u * second]);
          items.store(v_dst + offset, item, va[u], vb[u * second]);
        }
        items.advance(&head, &item);
      }
      if (head < p.k.heads) load_kv(head, item);
    }
  }
  int head = items.first_head, item = items.first_item;
  while (head < p.q.heads) {
#pragma unroll
    for (int u = 0; u < kQ; ++u) {
      if (head < p.q.heads) {
        constexpr int second = kPaired ? 1 : 0;
        items.turn(angles, item, qa + u, qb + u * second);
        items.store(q_dst + (int64_t)head * p.q.dst_head + items.value(item), item, qa[u], qb[u * second]);
      }
      items.advance(&head, &item);
    }
    if (head < p.q.heads) load_q(head, item);
  }
}

// Whether rows can be moved in whole vectors of n elements.
bool whole(const Rows& r, int n, size_t size) {
  if (!r.heads) return true;
  const uintptr_t at = reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst);
  return at % (n * size) == 0 && r.src_token % n == 0 && r.src_head % n == 0 && r.dst_token % n == 0 &&
         r.dst_head % n == 0;
}

template <typename T, bool kPaged>
int launch_move(MoveParams p, cudaStream_t stream) {
  constexpr int n = 16 / sizeof(T);
  const bool half = p.layout == SVX_ROPE_HALF && p.inv_freq;
  const bool wide = p.dim % n == 0 && (!p.inv_freq || (half ? p.pairs % n == 0 : 2 * p.pairs % n == 0)) &&
                    whole(p.q, n, sizeof(T)) && whole(p.k, n, sizeof(T)) && whole(p.v, n, sizeof(T));
  const int width = wide ? n : 1, rot = p.inv_freq ? 2 * p.pairs : 0;
  p.items = (!wide || half ? rot / (2 * width) : rot / width) + (p.dim - rot) / width;
  // Warps of a token: one, or as many as there is work for while they are fewer than 16 a SM.
  const int64_t items = (int64_t)std::max(p.q.heads, p.k.heads) * p.items;
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>((items + 31) / 32, 2368 / p.tokens));
  p.step_heads = 32 * p.parts / p.items;
  p.step_items = 32 * p.parts % p.items;
  const int64_t units = (int64_t)p.tokens * p.parts;
  const dim3 grid((unsigned)((units + kWarps - 1) / kWarps));
  auto kernel = !wide ? move_rows_kernel<T, 1, true, kPaged>
                : half ? move_rows_kernel<T, n, true, kPaged> : move_rows_kernel<T, n, false, kPaged>;
  return launch_dependent("move_rows_kernel", kernel, grid, dim3(kThreads), 0, stream, p);
}

int take_rotary(const svx_rotary* r, int dim, MoveParams* p) {
  SVX_REQUIRE(r->inv_freq, "rotary: inv_freq is missing");
  SVX_REQUIRE(r->rot > 0 && r->rot % 2 == 0 && r->rot <= dim, "rotary: rot must be even, positive and at most dim");
  SVX_REQUIRE(r->rot <= 2 * kMaxPairs, "rotary: rot must be at most 512");
  SVX_REQUIRE(r->axes >= 1 && (r->rot / 2) % r->axes == 0, "rotary: the axes must share the pairs evenly");
  SVX_REQUIRE(r->layout == SVX_ROPE_INTERLEAVED || r->layout == SVX_ROPE_HALF, "rotary: unknown layout");
  SVX_REQUIRE(!r->positions || r->position_type == SVX_F32 || r->position_type == SVX_I32 || r->position_type == SVX_I64,
              "rotary: positions must be int32, int64 or fp32");
  SVX_REQUIRE(r->positions || r->axes == 1, "rotary: several axes need positions");
  p->inv_freq = r->inv_freq;
  p->positions = r->positions;
  p->position_type = r->position_type;
  p->axes = r->axes;
  p->pairs = r->rot / 2;
  p->layout = r->layout;
  p->scale = r->scale;
  return SVX_OK;
}

}  // namespace
}  // namespace svx

using namespace svx;

extern "C" int svx_rope(const void* x, int dtype, int64_t x_token_stride, int64_t x_head_stride, void* out,
                        int64_t out_token_stride, int64_t out_head_stride, int tokens, int heads, int dim,
                        const svx_rotary* rotary, int inverse, void* stream) {
  SVX_REQUIRE(dtype == SVX_F32 || dtype == SVX_BF16 || dtype == SVX_F16, "svx_rope: rows must be fp32, bf16 or fp16");
  SVX_REQUIRE(tokens >= 0 && heads > 0 && dim > 0 && heads <= (1 << 20) && dim <= (1 << 20) &&
                  (int64_t)heads * dim <= (1 << 24),
              "svx_rope: bad shape");
  if (!tokens) return SVX_OK;
  SVX_REQUIRE(rotary && rotary->positions, "svx_rope: positions are missing");
  MoveParams p{};
  if (const int rc = take_rotary(rotary, dim, &p)) return rc;
  SVX_REQUIRE(x && out, "svx_rope: null rows");
  p.q = Rows{x, out, x_token_stride, x_head_stride, out_token_stride, out_head_stride, heads};
  p.inverse = inverse != 0;
  p.tokens = tokens;
  p.dim = dim;
  if (dtype == SVX_BF16) return launch_move<__nv_bfloat16, false>(p, as_stream(stream));
  if (dtype == SVX_F16) return launch_move<__half, false>(p, as_stream(stream));
  return launch_move<float, false>(p, as_stream(stream));
}

extern "C" int svx_paged_append(const svx_paged_cache* cache, const void* k, int64_t k_token_stride,
                                int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                int tokens, const svx_rotary* rotary, const void* q, int64_t q_token_stride,
                                int64_t q_head_stride, int q_heads, void* q_out, void* stream) {
  int shift = 0;
  if (const int rc = check_cache(cache, "svx_paged_append", &shift)) return rc;
  SVX_REQUIRE(tokens >= 0, "svx_paged_append: bad token count");
  if (!tokens || !cache->sequences) return SVX_OK;
  SVX_REQUIRE(!q || (q_heads > 0 && q_heads <= 4096 && rotary), "svx_paged_append: q needs heads and a rotary");
  MoveParams p{};
  if (rotary)
    if (const int rc = take_rotary(rotary, cache->dim, &p)) return rc;
  SVX_REQUIRE(k && v && (!q || q_out), "svx_paged_append: null rows");
  if (q) p.q = Rows{q, q_out, q_token_stride, q_head_stride, (int64_t)q_heads * cache->dim, cache->dim, q_heads};
  p.k = Rows{k, cache->k, k_token_stride, k_head_stride, 0, 0, cache->kv_heads};
  p.v = Rows{v, cache->v, v_token_stride, v_head_stride, 0, 0, cache->kv_heads};
  p.tokens = tokens;
  p.dim = cache->dim;
  p.table = cache->table;
  p.lengths = cache->lengths;
  p.offsets = cache->offsets;
  p.status = cache->status;
  p.sequences = cache->sequences;
  p.table_width = cache->table_width;
  p.pages = cache->pages;
  p.page_shift = shift;
  if (cache->dtype == SVX_BF16) return launch_move<__nv_bfloat16, true>(p, as_stream(stream));
  return launch_move<__half, true>(p, as_stream(stream));
}
