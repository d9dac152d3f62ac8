// Rotary positions by themselves (svx_rope) and on the way into a paged cache (svx_paged_append).
//
// Each pair (a, b) of a head's first `rot` values turns by the angle position * inv_freq[pair]:
//   (a, b) -> scale * (a cos - b sin, a sin + b cos)
// and the values past `rot` are copied. The backward pass is the transposed turn, the same kernel with the sine's sign
// flipped. Interleaved pairs are (2j, 2j + 1), half pairs (j, j + rot / 2); with several position axes the pairs are
// split evenly among them, axis-major (the axial rotation of the GEMM epilogue).
//
// Both operators are one pass over their rows and bound by memory once the rows outgrow L2. A CTA takes a few tokens:
// it first computes the tokens' cosines and sines into shared memory, once for all heads, then moves 16-byte vectors.
// The angle is formed in float64 and reduced to a fraction of a turn there (positions of a million lose 2e-2 of a
// radian in 32 bits), the rest is fp32; a value is rounded to its own type once.
#include "common.cuh"
#include "paged.cuh"

namespace svx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTile = kThreads / 32;   // tokens of a CTA: a warp looks up each token's sequence
constexpr int kMaxPairs = 256;

// One source of rows: [tokens][heads][dim] with strides in elements; the destination likewise, or the cache's pages.
struct Rows {
  const void* src;
  void* dst;
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;
};

struct MoveParams {
  Rows q, k, v;               // q (or svx_rope's x) and k turn, v is copied; k and v go to the pages
  const double* inv_freq;     // null: nothing turns
  const void* positions;      // null: the token's position in the cache
  int position_type, axes, pairs, layout, inverse;
  float scale;
  int tokens, dim, tile;
  // cache (sequences == 0: none)
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

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// N = 1 is the form for any dim, stride and alignment; N = 16 bytes' worth needs all of them in whole vectors.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) move_rows_kernel(const MoveParams p) {
  __shared__ float2 s_turn[kMaxTile * kMaxPairs];   // (cos, sin) * scale, indexed [token][pair]
  __shared__ int64_t s_row[kMaxTile];      // row of the token's key in head 0 of its page, -1: not stored
  __shared__ int s_at[kMaxTile];           // position in the cache
  __shared__ int s_live[kMaxTile];         // 0: the token belongs to no sequence
  using P = Pack<T, N>;
  grid_launch_dependents();
  grid_dependency_wait();
  const int token0 = blockIdx.x * p.tile, tile = min(p.tile, p.tokens - token0);
  if (p.sequences) {
    const int w = warp_id();
    if (w < tile) {
      const int t = token0 + w;
      // The token's sequence is the count of sequence ends at or before it; every lane's loads are independent.
      int count = 0;
      for (int i = lane_id(); i < p.sequences; i += 32) count += __ldg(p.offsets + i + 1) <= t;
      const int s = __reduce_add_sync(0xffffffffu, count);
      if (lane_id() == 0) {
        int at = 0;
        int64_t row = -1;
        bool live = false;
        if (s < p.sequences) {
          const int first = p.offsets[s], end = p.offsets[s + 1];
          live = t >= first;
          if (live) {
            const int64_t place = (int64_t)p.lengths[s] - end + t;
            bool ok = place >= 0 && place < ((int64_t)p.table_width << p.page_shift);
            at = (int)max((int64_t)-(1 << 30), min(place, (int64_t)1 << 30));
            if (ok && p.k.heads) {
              const int page = p.table[(int64_t)s * p.table_width + (place >> p.page_shift)];
              ok = page >= 0 && page < p.pages;
              if (ok) row = ((int64_t)page * p.k.heads << p.page_shift) + (place & ((1 << p.page_shift) - 1));
            }
            if (!ok && p.status) atomicOr(p.status + s, SVX_STATUS_BAD_PAGE);
          }
        }
        s_at[w] = at;
        s_row[w] = row;
        s_live[w] = live;
      }
    }
    __syncthreads();
  }
  if (p.inv_freq) {
    const int per_axis = p.pairs / p.axes;
    for (int i = threadIdx.x; i < tile * p.pairs; i += kThreads) {
      const int w = i / p.pairs, j = i - w * p.pairs;
      double position;
      if (!p.positions) {
        position = s_at[w];
      } else {
        const int64_t e = (int64_t)(token0 + w) * p.axes + j / per_axis;
        position = p.position_type == SVX_I64   ? (double)static_cast<const int64_t*>(p.positions)[e]
                   : p.position_type == SVX_I32 ? (double)static_cast<const int32_t*>(p.positions)[e]
                                                : (double)static_cast<const float*>(p.positions)[e];
      }
      double turns = position * p.inv_freq[j] * 0.15915494309189533577;   // 1 / (2 pi)
      turns -= rint(turns);
      // The fraction of a turn as the nearest float and a first-order correction for what that drops.
      const float near = (float)turns, rest = (float)(turns - (double)near) * 6.2831853f;
      float sn, cs;
      sincospif(2.f * near, &sn, &cs);
      const float c = fmaf(-rest, sn, cs), s = fmaf(rest, cs, sn);
      s_turn[i] = make_float2(c * p.scale, (p.inverse ? -s : s) * p.scale);
    }
    __syncthreads();
  }
  // Items of a token: for each head its vectors; of the half layout the first rot / 2 values' items carry their
  // partners with them. `plain` items are copied.
  const bool half = p.layout == SVX_ROPE_HALF && p.inv_freq;
  const int turning = p.inv_freq ? (N == 1 || half ? p.pairs / (N == 1 ? 1 : N) : 2 * p.pairs / N) : 0;
  const int plain = (p.dim - (p.inv_freq ? 2 * p.pairs : 0)) / N;
  const int per_turned = turning + plain, per_copied = p.dim / N;
  const int n_turned = (p.q.heads + p.k.heads) * per_turned, per_token = n_turned + p.v.heads * per_copied;
  for (int i = threadIdx.x; i < tile * per_token; i += kThreads) {
    const int w = i / per_token;
    int r = i - w * per_token;
    const bool copied = r >= n_turned;
    int head, item;
    if (copied) {
      r -= n_turned;
      head = r / per_copied;
      item = r - head * per_copied;
    } else {
      head = r / per_turned;
      item = r - head * per_turned;
    }
    if (p.sequences && !s_live[w]) continue;
    const int64_t t = token0 + w;
    const bool is_k = !copied && head >= p.q.heads;
    const T* src;
    T* dst;
    if (copied || is_k) {
      if (is_k) head -= p.q.heads;
      if (s_row[w] < 0) continue;
      const int64_t row = s_row[w] + ((int64_t)head << p.page_shift);
      src = static_cast<const T*>(copied ? p.v.src : p.k.src) + t * (copied ? p.v.src_token : p.k.src_token) +
            head * (copied ? p.v.src_head : p.k.src_head);
      dst = static_cast<T*>(copied ? p.v.dst : p.k.dst) + row * p.dim;
    } else {
      src = static_cast<const T*>(p.q.src) + t * p.q.src_token + head * p.q.src_head;
      dst = static_cast<T*>(p.q.dst) + t * p.q.dst_token + head * p.q.dst_head;
    }
    const float2* turn = s_turn + w * p.pairs;
    if (copied || item >= turning) {
      const int e = copied ? item * N : p.dim - (per_turned - item) * N;
      *reinterpret_cast<P*>(dst + e) = *reinterpret_cast<const P*>(src + e);
    } else if (N == 1 || half) {
      const int a = half ? item * N : 2 * item, b = half ? a + p.pairs : a + 1;
      const P x = *reinterpret_cast<const P*>(src + a), y = *reinterpret_cast<const P*>(src + b);
      P u, v;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 cs = turn[item * N + e];
        const float f = to_f32(x.v[e]), g = to_f32(y.v[e]);
        u.v[e] = from_f32<T>(f * cs.x - g * cs.y);
        v.v[e] = from_f32<T>(f * cs.y + g * cs.x);
      }
      *reinterpret_cast<P*>(dst + a) = u;
      *reinterpret_cast<P*>(dst + b) = v;
    } else {
      const P x = *reinterpret_cast<const P*>(src + item * N);
      P u;
#pragma unroll
      for (int e = 0; e + 1 < N; e += 2) {
        const float2 cs = turn[(item * N + e) / 2];
        const float f = to_f32(x.v[e]), g = to_f32(x.v[e + 1]);
        u.v[e] = from_f32<T>(f * cs.x - g * cs.y);
        u.v[e + 1] = from_f32<T>(f * cs.y + g * cs.x);
      }
      *reinterpret_cast<P*>(dst + item * N) = u;
    }
  }
}

// Whether rows can be moved in whole vectors of n elements.
bool whole(const Rows& r, int n, size_t size) {
  if (!r.heads) return true;
  const uintptr_t at = reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst);
  return at % (n * size) == 0 && r.src_token % n == 0 && r.src_head % n == 0 && r.dst_token % n == 0 &&
         r.dst_head % n == 0;
}

template <typename T>
int launch_move(MoveParams p, cudaStream_t stream) {
  constexpr int n = 16 / sizeof(T);
  const bool half = p.layout == SVX_ROPE_HALF;
  const bool wide = p.dim % n == 0 && (!p.inv_freq || (half ? p.pairs % n == 0 : 2 * p.pairs % n == 0)) &&
                    whole(p.q, n, sizeof(T)) && whole(p.k, n, sizeof(T)) && whole(p.v, n, sizeof(T));
  // Tokens of a CTA: about four vectors a thread, but no fewer CTAs than two for each SM.
  const int64_t vectors = (int64_t)(p.q.heads + p.k.heads + p.v.heads) * p.dim / (wide ? n : 2);
  int tile = (int)(4 * kThreads / (vectors > 0 ? vectors : 1));
  tile = tile < 1 ? 1 : tile > kMaxTile ? kMaxTile : tile;
  while (tile > 1 && p.tokens / tile < 296) tile >>= 1;
  p.tile = tile;
  const dim3 grid((p.tokens + tile - 1) / tile);
  if (wide) return launch_dependent("move_rows_kernel", move_rows_kernel<T, n>, grid, dim3(kThreads), 0, stream, p);
  return launch_dependent("move_rows_kernel", move_rows_kernel<T, 1>, grid, dim3(kThreads), 0, stream, p);
}

int launch_move(const MoveParams& p, int dtype, cudaStream_t stream) {
  if (dtype == SVX_BF16) return launch_move<__nv_bfloat16>(p, stream);
  if (dtype == SVX_F16) return launch_move<__half>(p, stream);
  return launch_move<float>(p, stream);
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
  return launch_move(p, dtype, as_stream(stream));
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
  return launch_move(p, cache->dtype, as_stream(stream));
}
