// Attention of draft trees over a paged cache: the pieces that its kernels share.
//
//   out[r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q_r . k_j - max),  j over the positions
//   that row r sees: the context (all of it) and the tree nodes of its mask.
//
// Work is cut the same way by every kernel: a unit is (sequence, row tile, cached head), a row
// tile BM of the n G query vectors that share the head (vector R is node R / G, head R % G of the
// group), so each K/V byte is read once per row tile whatever G is. A unit has ceil(len / BN)
// key tiles; the tiles of all units form one line, and CTA c takes `per` of them in a row, so
// ragged batches and single long caches load every SM alike. A CTA that holds all tiles of a
// unit writes its rows; where a unit spans CTAs each writes a partial (running maximum, sum,
// unnormalised output) and a second kernel joins them in order (no atomics, so equal calls give
// equal bits).
#pragma once
#include "pp_paged.cuh"

namespace pp {

struct TreeArgs {
  PagedView c;  // the layer
  BatchView b;
  const void* q;
  void* out;
  float* lse;
  int64_t q_stride;  // elements
  const uint32_t* mask;
  int32_t mask_words, nh, G;
  float scale;
  float* part;      // [2 * ctas][BM][DP] outputs, then [2 * ctas][BM] (max, sum)
  int32_t ctas;     // CTAs that the line of tiles is cut over
  int32_t min_per;  // least tiles of a CTA
  uint32_t* err;
};

// A sequence whose lengths do not fit its table is left out.
__device__ __forceinline__ bool bad_sequence(const TreeArgs& a, int n, int len) {
  return n < 0 || len < n || (int64_t)len > (int64_t)a.b.table_stride * a.c.page.d;
}

// prefix[b] = tiles before sequence b on the line; prefix[batch] = all. By the whole CTA
// (NT threads), scan: NT / 32 words of shared memory.
template <int BM, int BN, int NT>
__device__ __forceinline__ void tile_prefix(const TreeArgs& a, int64_t* prefix, int64_t* scan,
                                            bool report) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.b.batch;
  const int each = (B + NT - 1) / NT, b0 = tid * each, b1 = min(B, b0 + each);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = a.b.cu_rows[b + 1] - a.b.cu_rows[b], len = a.b.kv_len[b];
    prefix[b] = sum;  // inside this thread's share
    if (bad_sequence(a, n, len)) {
      if (report && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
    } else if (n > 0) {
      const int64_t rts = ((int64_t)n * a.G + BM - 1) / BM;
      sum += rts * a.c.n_kv * ((len + BN - 1) / BN);
    }
  }
  int64_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) scan[warp] = inc;
  __syncthreads();
  int64_t before = inc - sum;
  for (int w = 0; w < warp; ++w) before += scan[w];
  for (int b = b0; b < b1; ++b) prefix[b] += before;
  if (tid == NT - 1) prefix[B] = before + sum;
  __syncthreads();
}

// The tiles of one CTA inside one unit.
struct Segment {
  int32_t b, h, rt;           // unit
  int32_t t0, t1, tiles;      // key tiles [t0, t1) of `tiles`
  int32_t row0, n, len, ctx;  // first row of the sequence, nodes, positions, context positions
  int64_t unit0;              // place of the unit's first tile on the line
};
template <int BM, int BN>
__device__ __forceinline__ Segment segment_at(const TreeArgs& a, const int64_t* prefix, int64_t w,
                                              int64_t end) {
  int lo = 0, hi = a.b.batch;  // last b with prefix[b] <= w: the one with tiles, as w < prefix[b + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= w) lo = mid;
    else hi = mid;
  }
  Segment s;
  s.b = lo;
  s.row0 = a.b.cu_rows[lo];
  s.n = a.b.cu_rows[lo + 1] - s.row0;
  s.len = a.b.kv_len[lo];
  s.ctx = s.len - s.n;
  s.tiles = (s.len + BN - 1) / BN;
  const int64_t off = w - prefix[lo], unit = off / s.tiles;
  s.t0 = (int)(off - unit * s.tiles);
  s.rt = (int)(unit / a.c.n_kv);
  s.h = (int)(unit - (int64_t)s.rt * a.c.n_kv);
  s.t1 = (int)min((int64_t)s.tiles, s.t0 + (end - w));
  s.unit0 = w - s.t0;
  return s;
}
__device__ __forceinline__ int64_t tiles_per_cta(const TreeArgs& a, int64_t total) {
  const int64_t even = (total + a.ctas - 1) / a.ctas;
  return even > a.min_per ? even : a.min_per;
}

// Whether row (sequence row i) sees node j (0 <= j < n).
__device__ __forceinline__ bool sees_node(const TreeArgs& a, int row, int i, int j) {
  if (!a.mask) return j <= i;
  const int w = j >> 5;
  return w < a.mask_words && (__ldg(a.mask + (int64_t)row * a.mask_words + w) >> (j & 31) & 1u);
}
// Whether a row without any probability mass sees something (its scores were all -inf: 0 / 0) or
// nothing (zeros).
__device__ __forceinline__ bool sees_any(const TreeArgs& a, int row, int n, int ctx) {
  if (ctx > 0 || !a.mask) return true;
  for (int w = 0; w < a.mask_words && 32 * w < n; ++w) {
    uint32_t m = a.mask[(int64_t)row * a.mask_words + w];
    if (32 * w + 32 > n) m &= (1u << (n - 32 * w)) - 1u;
    if (m) return true;
  }
  return false;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(read ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Softmax in base 2 (scores carry log2 e) for the 16-bit types, in base e for F32, where the
// product with log2 e would round a large score.
template <typename T>
__device__ __forceinline__ float soft_exp(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ float soft_scale(float scale) {
  return sizeof(T) == 4 ? scale : scale * 1.44269504088896341f;
}
template <typename T>
__device__ __forceinline__ float soft_lse(float m, float l) {
  return (sizeof(T) == 4 ? m : m * 0.69314718055994531f) + logf(l);
}

// Joins the partials of a unit: CTA (c, y) of the grid looks at the unit whose last tile CTA c of
// the line held, if others held its earlier ones, and joins rows y * 4 + warp, + 4 * gridDim.y, ...
// of it, a warp per row, lane l the dims l * 4 .. (float4), partial after partial.
template <typename T, int DP, int BM, int BN>
__global__ void __launch_bounds__(128) pp_tree_join_kernel(const TreeArgs a) {
  extern __shared__ int64_t s_prefix[];
  __shared__ int64_t scan[4];
  pdl_wait();
  tile_prefix<BM, BN, 128>(a, s_prefix, scan, false);
  const int64_t total = s_prefix[a.b.batch], per = tiles_per_cta(a, total);
  const int64_t c = blockIdx.x, w = c * per, end = min(total, w + per);
  if (w >= total) return;
  const Segment s = segment_at<BM, BN>(a, s_prefix, w, end);
  if (s.t0 == 0 || s.t1 != s.tiles) return;
  const int64_t c0 = s.unit0 / per;
  const int64_t first = c0 * per == s.unit0 ? 2 * c0 : 2 * c0 + 1;
  const int parts = (int)(c - c0) + 1;
  const float2* ml = (const float2*)(a.part + (int64_t)2 * a.ctas * BM * DP);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = min(BM, s.n * a.G - s.rt * BM);
  const int D = a.c.head_dim;
  for (int r = blockIdx.y * 4 + warp; r < rows; r += 4 * gridDim.y) {
    const int R = s.rt * BM + r, i = R / a.G, row = s.row0 + i;
    const int head = s.h * a.G + (R - i * a.G);
    auto slot = [&](int p) { return p == 0 ? first : 2 * (c0 + p); };
    float mx = -INFINITY;
    for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, ml[slot(p) * BM + r].x);
    mx = warp_max(mx);
    const float base = mx == -INFINITY ? 0.f : mx;
    float acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = 0.f;
    float l = 0.f;
    for (int p0 = 0; p0 < parts; p0 += 32) {
      float wgt = 0.f;
      if (p0 + lane < parts) {
        const float2 v = ml[slot(p0 + lane) * BM + r];
        wgt = soft_exp<T>(v.x - base);
        l += v.y * wgt;
      }
      const int m = min(32, parts - p0);
#pragma unroll 4
      for (int p = 0; p < m; ++p) {
        const float f = __shfl_sync(0xffffffffu, wgt, p);
        const float* o = a.part + (slot(p0 + p) * BM + r) * DP;
        if constexpr (DP >= 128) {
#pragma unroll
          for (int q = 0; q < DP / 128; ++q) {
            const float4 v = __ldcg((const float4*)(o + q * 128 + 4 * lane));
            acc[4 * q] += v.x * f;
            acc[4 * q + 1] += v.y * f;
            acc[4 * q + 2] += v.z * f;
            acc[4 * q + 3] += v.w * f;
          }
        } else {
          const float2 v = __ldcg((const float2*)(o + 2 * lane));
          acc[0] += v.x * f;
          acc[1] += v.y * f;
        }
      }
    }
    l = warp_sum(l);
    const bool empty = l == 0.f && !sees_any(a, row, s.n, s.ctx);
    T* out = (T*)a.out + ((int64_t)row * a.nh + head) * D;
    constexpr int V = DP >= 128 ? 4 : 2;
#pragma unroll
    for (int q = 0; q < DP / 32; ++q) {
      const int d = (q / V) * 32 * V + V * lane + q % V;
      if (d < D) out[d] = Elem<T>::put(empty ? 0.f : acc[q] / l);
    }
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<T>(mx, l);
  }
}

}  // namespace pp
