// pp_tree_attention: the kernels for few query vectors over caches of 16-bit types (mma.sync: the bytes
// of the cache bound it) and for F32 caches (CUDA cores), the choice of kernel and the entry point. The
// kernel for many query vectors is in pp_tree_tc.cu, the work split and the join in pp_tree_attn.cuh.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_attn.cuh"
#include "pp_tree_attn.cuh"
#include "pp_tree_plan.cuh"

using namespace pp;

namespace pp {

// ---- 16-bit caches, few query vectors --------------------------------------------------------
constexpr int kTreeThreads = 128;
constexpr int kTreeBN = kTreeTile<__half>;
// The bounds below were measured with 8 cached heads of 128 and hold for other heads and dims unmeasured.
// Caches of up to so many tiles are never cut, which saves the join's launch, about 1 us (one decoded
// row, 8 heads, narrow: 256 positions 8.0 us whole against 8.6, 512 11.9 against 9.4; F32: 64 positions
// 6.8 against 7.4, 128 10.9 against 7.2; 240 vectors, tcgen05: 128 positions 10.9 against 11.9).
constexpr int kWholeNarrow = 4, kWholeTc = 2, kWholeF32 = 2;
// Longer ones are not where that loads the fullest CTA with at most a quarter and so many tiles, or six
// times the equal share, more (fullest CTA whole against equal share; ragged trees of 61 nodes, 8 heads,
// tcgen05: 64 against 44 tiles 97 us against 108, 16 against 12 35 against 54, 8 against 2 18.8
// against 23.1, 8 against 1 17.8 against 15.3, 24 against 5 36 against 30, 64 against 32 105 against 80; decoded rows,
// narrow: 17 against 13 27.2 against 28.9, 4 against 1 9.5 against 10.7, 16 against 6 21.3 against 17.5;
// F32: 3 against 2 14.0 against 14.4, 10 against 7 35.9 against 31.6).
constexpr uint32_t kSlackNarrow = 3, kSlackTc = 12, kSlackF32 = 1;
// More than 8 query vectors a head, the narrow kernel takes in tiles of 8, reading K and V again for
// each from L2; it starts faster and its tiles are quicker, so it still leads up to this many of its
// tiles a CTA (32 vectors, 8 heads, narrow against tcgen05: 2056 positions 14.0 us against 17.3, 4104 18.1
// against 21.1, 8200 24.6 against 23.8, 16392 40.7 against 30.5, 32 x 2056 102 against 64).
constexpr uint64_t kNarrowTiles = 12;

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                     uint32_t b1) {
  mma_bf16_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two values as one register of T (a in the low half), and what their rounding left over.
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) {
  return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16;
}
__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16;
}
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const T ah = Elem<T>::put(a), bh = Elem<T>::put(b);
  hi = pack2(ah, bh);
  lo = pack2(Elem<T>::put(a - Elem<T>::get(ah)), Elem<T>::put(b - Elem<T>::get(bh)));
}
// The narrow kernel's shared memory: a ring of NS stages for each of the four warps, 16 rows of K and
// of V as 64-dim blocks [16 rows][128 bytes], the 16-byte unit u of row r at u ^ (r & 7).
template <int DP>
struct NarrowCfg {
  static constexpr int BM = 8, KW = 16, NS = DP == 256 ? 2 : 3, kPerSm = DP == 256 ? 1 : 2;
  static constexpr int kTile = KW * DP * 2, kStage = 2 * kTile, kRing = 4 * NS * kStage;
  static constexpr int kOPitch = DP + 4;
  static_assert(4 * BM * (kOPitch * 4 + 8) <= kRing, "the warps' outputs take the ring's place");
  // Nothing is static, so that the dynamic part starts on the 1024 bytes that the swizzle counts from.
  static constexpr int kBars = 4 * NS * 8 + 12 * (kTreeThreads / 32);
  static size_t smem(int batch) { return kRing + kBars + prefix_bytes(batch); }
};
// Byte offset of 16-byte unit u (dims 8 u ..) of row r in a tile of it.
__device__ __forceinline__ int narrow_unit(int r, int u) { return (u >> 3) * 2048 + r * 128 + (((u & 7) ^ (r & 7)) << 4); }

// A warp's 16 rows of K and V by 16-byte copies, for pages that boxes do not fit.
template <int DP>
__device__ __forceinline__ void narrow_copy(const TreeArgs& a, const RowFetch<16>& f, uint8_t* kd, int lane) {
  constexpr int UR = DP / 8, RP = 32 / UR;
  const int u = lane % UR, sub = lane / UR;
#pragma unroll 4
  for (int i = 0; i < 16 / RP; ++i) {
    const int l = i * RP + sub;
    const int64_t off = f.row(a, l);
    const bool read = off >= 0 && 8 * u < a.c.head_dim;
    const int64_t at = read ? off + 16 * u : 0;
    cp_async16(kd + narrow_unit(l, u), a.c.k + at, read);
    cp_async16(kd + NarrowCfg<DP>::kTile + narrow_unit(l, u), a.c.v + at, read);
  }
}

// Up to 8 query vectors of a cached head in a row tile (a decoded token with G <= 8): keys are the
// products' M dimension and the vectors N, S^T = K Q^T and O^T = V^T P^T on mma.sync, half the
// products and half the accumulators of a 16-row tile; at 8 rows the cache's bytes bound it, not the
// tensor cores. A warp fetches (TMA, 16-row boxes) and consumes its own 16 keys of every 64-key
// tile, so the loop has no CTA barrier. P^T turns from S^T's layout to an operand's by movmatrix; it is
// carried as two parts of the cache's type, hi + lo, for one alone would add as much error as the
// rounding of the output. 64 decoded rows over 4096 to 8192 positions, 8 heads of 128, BF16, pages of 16:
// 250 to 254 us for 1.63 GB, 6.4 to 6.5 TB/s, what a copy reaches; one row over 131072: 93 us, 5.8.
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
template <typename T, int DP>
__global__ void __launch_bounds__(kTreeThreads, NarrowCfg<DP>::kPerSm)
    pp_tree_narrow_kernel(const TreeArgs a, const __grid_constant__ TreeMaps maps) {
  using C = NarrowCfg<DP>;
  constexpr int BM = 8, BN = kTreeBN, NS = C::NS, KS = DP / 16, NB = DP / 64;
  extern __shared__ __align__(1024) uint8_t narrow_smem[];
  uint8_t* sm = narrow_smem;
  uint64_t* full = (uint64_t*)(sm + C::kRing);  // [4][NS]
  uint32_t* scan = (uint32_t*)(full + 4 * NS);
  uint32_t* prefix = scan + 3 * (kTreeThreads / 32);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t4 = lane & 3;
  const int D = a.c.head_dim;
  const float sc = soft_scale<T>(a.scale);
  const bool tma = maps.box != 0;
  uint8_t* ring = sm + warp * NS * C::kStage;  // the warp's
  uint64_t* bar = full + warp * NS;
  if (smem_u32(sm) & 1023u) {  // cannot be; the caller is told
    if (tid == 0 && a.err) atomicOr(a.err, PAGED_TIMEOUT);
    return;
  }
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  pdl_launch_dependents();
  const Line line = cut_line<BN, kTreeThreads>(a, __builtin_ctz(BM), prefix, true, scan, blockIdx.x == 0);
  uint32_t begin, end;
  cta_range(line, blockIdx.x, begin, end);
  RingCursor use;  // the stage of the next tile to consume
  bool ok = true;

  for (uint32_t w = begin; w < end;) {
    const Segment s = segment_at<BN>(a, line, prefix, w, end);
    const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
    RowFetch<16> rows;
    BoxPlace box;
    // Where tile t's rows are, a tile ahead of their copies.
    auto look = [&](int t) {
      const int idx = t * BN + warp * 16;
      if (tma) box.look(a, s, table, idx, t < s.t1);
      else rows.look(a, s, table, idx, t < s.t1, lane);
    };
    look(s.t0);
    // Q^T fragments: vector g4, dims 16 ks + 2 t4 and + 8.
    uint32_t qb[KS][2];
    {
      const int R = s.rt * BM + g4, i = (int)a.by_g.div((uint32_t)R);
      const bool in = R < s.n * a.G;
      const T* q = (const T*)a.q + (int64_t)(s.row0 + (in ? i : 0)) * a.q_stride + (int64_t)(s.h * a.G + (in ? R - i * a.G : 0)) * D + 2 * t4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qb[ks][e] = in && 16 * ks + 8 * e < D ? *(const uint32_t*)(q + 16 * ks + 8 * e) : 0u;
    }
    // The thread's two vectors: 2 t4 and 2 t4 + 1.
    const int i0 = (int)a.by_g.div((uint32_t)(s.rt * BM + 2 * t4)), i1 = (int)a.by_g.div((uint32_t)(s.rt * BM + 2 * t4 + 1));
    float o[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    // ldmatrix rows of the lane: K as [16 keys][16 dims], V the same, transposed.
    const int kr = lane & 15, ku = lane >> 4, vr = (lane & 7) + ((lane >> 4) << 3), vu = (lane >> 3) & 1;
    uint32_t found = 0;  // non-finite values of V were taken out of the products

    uint32_t into = use.slot;  // the stage that the next fetched tile takes
    for (int t = s.t0 - (NS - 1); t < s.t1; ++t) {
      if (t >= s.t0) {
        if (tma) {
          if (!warp_wait(&bar[use.slot], use.phase)) {
            ok = false;
            break;
          }
        } else {
          cp_async_wait<NS - 2>();
        }
      }
      __syncwarp();
      // Tile t + NS - 1 into the stage that tile t - 1 has left. A stage that ordinary loads have read
      // is handed to the copy engine by the proxy fence.
      const bool more = t + NS - 1 < s.t1;
      if (tma) {
        if (more) {
          if (elect_one()) {
            fence_async();
            mbar_arrive_expect_tx(&bar[into], C::kStage);
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i)
              tma_box(ring + into * C::kStage + i * 2048, i < NB ? &maps.k : &maps.v, &bar[into], maps, 64 * (i % NB),
                      s.h, box.row, box.page);
          }
          __syncwarp();
        }
      } else {
        if (more) narrow_copy<DP>(a, rows, ring + into * C::kStage, lane);
        cp_async_commit();
      }
      if (more) {
        into = into + 1 == NS ? 0 : into + 1;
        look(t + NS);
      }
      if (t < s.t0) continue;
      const uint8_t* kt = ring + use.slot * C::kStage;
      uint8_t* vt = ring + use.slot * C::kStage + C::kTile;
      const int j0 = t * BN + warp * 16;
      use.next(NS);

      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};  // even and odd k steps
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {  // dims past the head's are zero in Q
        uint32_t kf[4];
        ldmatrix_x4a(kf, kt + narrow_unit(kr, 2 * ks + ku));
        mma16<T>(ks & 1 ? y : x, kf, qb[ks][0], qb[ks][1]);
      }
      // Element e: key g4 + 8 (e >> 1), vector 2 t4 + (e & 1).
      const bool tree = j0 + 16 > s.ctx;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (x[e] + y[e]) * sc;
      if (tree) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int node = j0 + g4 + 8 * (e >> 1) - s.ctx, i = e & 1 ? i1 : i0;
          if (node >= 0 && (node >= s.n || i >= s.n || !sees_node(a, s.row0 + i, i, node))) x[e] = -INFINITY;
        }
      }
      float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1)
#pragma unroll
        for (int q = 0; q < 2; ++q) mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], sh));
      // The old base serves until a score passes its maximum by more than the lag: P stays small enough,
      // and the output need not be rescaled at every small step.
      const bool grown = soft_outgrown<T>(mx[0], m[0]) || soft_outgrown<T>(mx[1], m[1]);
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float mn = fmaxf(m[q], soft_base<T>(mx[q]));
          const float alpha = soft_exp<T>(m[q] - (mn == -INFINITY ? 0.f : mn));
          m[q] = mn;
          l[q] *= alpha;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            o[k][q] *= alpha;
            o[k][q + 2] *= alpha;
          }
        }
      }
      const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = soft_exp<T>(x[e] - base[e & 1]);
        l[e & 1] += x[e];
      }
      // Positions past the end hold whatever their page did: zeros there. And a V that some row is
      // blind to must not count even where it is not finite (0 * NaN): such values leave the tile
      // here and come back, for the rows that see them, with the output.
      const bool blind = tree && (a.mask || s.n > 1);
      if (blind || j0 + 16 > s.len) {
#pragma unroll 1
        for (int e = lane; e < 16 * (DP / 8); e += 32) {
          uint4* p = (uint4*)(vt + e * 16);
          uint4 v = *p;
          uint32_t bad[4] = {~0u, ~0u, ~0u, ~0u};
          if (j0 + ((e >> 3) & 15) < s.len) {
            bad[0] = nonfinite_halves<T>(v.x);
            bad[1] = nonfinite_halves<T>(v.y);
            bad[2] = nonfinite_halves<T>(v.z);
            bad[3] = nonfinite_halves<T>(v.w);
            if (!blind || !(bad[0] | bad[1] | bad[2] | bad[3])) continue;
            found = 1;
          }
          *p = make_uint4(v.x & ~bad[0], v.y & ~bad[1], v.z & ~bad[2], v.w & ~bad[3]);
        }
        __syncwarp();
      }
      // P is carried as hi + lo parts: rounded to T alone it would add as much error as the rounding
      // of the output.
      uint32_t ph[2], pl[2];
      split2<T>(x[0], x[1], ph[0], pl[0]);
      split2<T>(x[2], x[3], ph[1], pl[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ph[e] = movmatrix(ph[e]);
        pl[e] = movmatrix(pl[e]);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t vf[4];
        ldmatrix_x4_trans(vf, vt + narrow_unit(vr, 2 * k + vu));
        mma16<T>(o[k], vf, ph[0], ph[1]);
        mma16<T>(o[k], vf, pl[0], pl[1]);
      }
    }
    if (!tma) cp_async_wait<0>();
    const bool dirty = __syncthreads_or(found != 0);
    if (__syncthreads_or(!ok)) break;  // else the rings are free
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) l[q] += __shfl_xor_sync(0xffffffffu, l[q], sh);
    // Outputs [warp][8][DP + 4] and (max, sum) [warp][8] of the warps in the rings' place.
    float* os = (float*)sm;
    float2* ml = (float2*)(sm + 4 * BM * C::kOPitch * 4);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        os[(warp * BM + 2 * t4 + (e & 1)) * C::kOPitch + 16 * k + g4 + 8 * (e >> 1)] = o[k][e];
    if (g4 == 0) {
      ml[warp * BM + 2 * t4] = make_float2(m[0], l[0]);
      ml[warp * BM + 2 * t4 + 1] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (w == begin ? 0 : 1);
    const int live = min(BM, s.n * a.G - s.rt * BM);
    if (dirty) {  // into the output of the warp with the row's largest base, whose weight below is 1
      add_nonfinite<T>(a, s, live, max(s.ctx & ~15, s.t0 * BN), min(s.len, s.t1 * BN), tid, kTreeThreads,
                       [&](int r, int d) -> float& {
                         int k = 0;
                         for (int j = 1; j < 4; ++j)
                           if (ml[j * BM + r].x > ml[k * BM + r].x) k = j;
                         return os[(k * BM + r) * C::kOPitch + d];
                       });
      __syncthreads();
    }
#pragma unroll 1
    for (int e = tid; e < live * (DP / 8); e += kTreeThreads) {
      const int r = e / (DP / 8), u = e % (DP / 8), R = s.rt * BM + r, i = (int)a.by_g.div((uint32_t)R);
      float top = ml[r].x;
#pragma unroll
      for (int k = 1; k < 4; ++k) top = fmaxf(top, ml[k * BM + r].x);
      const float tb = top == -INFINITY ? 0.f : top;
      float sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = ml[k * BM + r];
        const float wgt = soft_exp<T>(v.x - tb);
        sum += v.y * wgt;
        const float* src = os + (k * BM + r) * C::kOPitch + 8 * u;
#pragma unroll
        for (int d = 0; d < 8; ++d) f[d] += src[d] * wgt;
      }
      if (whole) {
        const int row = s.row0 + i, head = s.h * a.G + R - i * a.G;
        const bool empty = sum == 0.f && !sees_any(a, row, s.n, s.ctx);
        const float inv = 1.f / sum;
#pragma unroll
        for (int d = 0; d < 8; ++d) f[d] = empty ? 0.f : f[d] * inv;
        if (8 * u < D) store8((T*)a.out + ((int64_t)row * a.nh + head) * D + 8 * u, f);
        if (a.lse && u == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<T>(top, sum);
      } else {
        store_n<float, 8>(a.part + (slot * BM + r) * DP + 8 * u, f);
        if (u == 0) a.part_ml[slot * BM + r] = make_float2(top, sum);
      }
    }
    fence_async();    // the rings go back to the copy engine
    __syncthreads();
    w += s.step;
  }
  if (!ok) {
    // Let the copies in flight land before the shared memory is released: at most one a stage.
    if (tma)
      for (int i = 0; i < NS; ++i) warp_wait(&bar[use.slot], use.phase), use.next(NS);
    if (lane == 0 && a.err) atomicOr(a.err, PAGED_TIMEOUT);
  }
}

// ---- F32 caches ----------------------------------------------------------------------------
// CUDA cores: the F32 products and sums of the definition. (Three tensor-core products of split halves
// would come near F32, and many vectors a head would gain by them: not built.) BM query vectors (4 for a decoded token,
// 16 else), 32-key tiles, four warps. Scores: warp w the rows w BM / 4 .., lane = key, so the softmax
// of a row stays in its warp; output: thread = dim, all rows. One row over 42 positions, 16 heads on 8:
// 7.0 us, the chain of launch, lengths, page and rows; 48 rows over 515 to 1030: 83 us, 3.7 TB/s, 64 over
// 2048 to 4096: 366 us, 4.5 TB/s, the multiply-adds and their shared-memory operands. Trees read K and V
// again for every 16 vectors: 16 of 61 nodes over 2048 to 4096 positions 4.5 ms, 11 TFLOP/s.
constexpr int kTreeFBN = kTreeTile<float>, kTreeFStages = 2;
template <int DP, int BM>
struct TreeFCfg {
  static constexpr int P = DP + 4;  // row pitch: 16-byte columns of consecutive rows in other banks
  static constexpr int PP = BM + 4;  // pitch of the probabilities' rows
  static constexpr int kTile = kTreeFBN * P * 4, kStage = 2 * kTile;
  static constexpr int kQ = BM * P * 4, kP = kTreeFBN * PP * 4, kRows = 2 * BM * 4;
  static constexpr int kPerSm = DP <= 64 ? 5 : DP <= 128 ? 3 : 1;
  static size_t smem(int batch) {
    return kTreeFStages * kStage + kQ + kP + kRows + prefix_bytes(batch);
  }
};

template <int DP, int BM>
__global__ void __launch_bounds__(kTreeThreads) pp_tree_f32_kernel(const TreeArgs a) {
  using C = TreeFCfg<DP, BM>;
  constexpr int BN = kTreeFBN, NS = kTreeFStages, P = C::P, PP = C::PP, UR = DP / 4, RW = BM / 4;
  constexpr int DT = DP <= 128 ? 1 : DP / 128;  // dims of a thread: tid, tid + 128
  extern __shared__ __align__(128) uint8_t f32_smem[];
  uint8_t* sm = f32_smem;
  uint8_t* ring = sm;
  float* qs = (float*)(sm + NS * C::kStage);
  float* pt = qs + BM * P;  // [key][PP]
  float* al_s = pt + BN * PP;
  uint32_t* vis_s = (uint32_t*)(al_s + BM);
  uint32_t* prefix = vis_s + BM;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, D = a.c.head_dim;

  pdl_launch_dependents();
  const Line line = cut_line<BN, kTreeThreads>(a, __builtin_ctz(BM), prefix, true, (uint32_t*)ring, blockIdx.x == 0);
  uint32_t begin, end;
  cta_range(line, blockIdx.x, begin, end);

  for (uint32_t w = begin; w < end;) {
    const Segment s = segment_at<BN>(a, line, prefix, w, end);
    const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
    const int NR = s.n * a.G;
    RowFetch<8> ahead;  // a warp fetches 8 rows of every tile
    auto look = [&](int t) { ahead.look(a, s, table, t * BN + warp * 8, t < s.t1, lane); };
    auto fetch = [&](int stage) {
      uint8_t* kd = ring + stage * C::kStage;
#pragma unroll 4
      for (int i = 0; i < 8 * UR / 32; ++i) {
        const int e = lane + 32 * i, l = e / UR, u = e % UR, r = warp * 8 + l;
        const int64_t off = ahead.row(a, l);
        const bool read = off >= 0 && 4 * u < D;
        const int64_t at = read ? off + 16 * u : 0;
        cp_async16(kd + (r * P + 4 * u) * 4, a.c.k + at, read);
        cp_async16(kd + C::kTile + (r * P + 4 * u) * 4, a.c.v + at, read);
      }
    };
    look(s.t0);
    fetch(0);
    cp_async_commit();
    look(s.t0 + 1);
#pragma unroll 2
    for (int e = tid; e < BM * UR; e += kTreeThreads) {
      const int r = e / UR, u = e % UR, R = s.rt * BM + r;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (R < NR && 4 * u < D) {
        const int i = (int)a.by_g.div((uint32_t)R);
        v = *(const float4*)((const float*)a.q + (int64_t)(s.row0 + i) * a.q_stride +
                             (int64_t)(s.h * a.G + R - i * a.G) * D + 4 * u);
      }
      *(float4*)(qs + r * P + 4 * u) = v;
    }
    float m[RW], l[RW];  // of the warp's rows
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    float acc[DT][BM];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < BM; ++r) acc[d][r] = 0.f;

    for (int t = s.t0; t < s.t1; ++t) {
      const int stage = (t - s.t0) % NS;
      if (t + 1 < s.t1) fetch((t + 1 - s.t0) % NS);
      cp_async_commit();
      look(t + 2);
      cp_async_wait<1>();
      __syncthreads();
      const float* kt = (const float*)(ring + stage * C::kStage) + lane * P;
      const float* vt = (const float*)(ring + stage * C::kStage + C::kTile);
      const float* qw = qs + warp * RW * P;
      float x[RW][2];
#pragma unroll
      for (int r = 0; r < RW; ++r) x[r][0] = x[r][1] = 0.f;
#pragma unroll 8
      for (int d = 0; d < D; d += 4) {
        const float4 k = *(const float4*)(kt + d);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float4 q = *(const float4*)(qw + r * P + d);
          x[r][0] += q.x * k.x;
          x[r][1] += q.y * k.y;
          x[r][0] += q.z * k.z;
          x[r][1] += q.w * k.w;
        }
      }
      const int node = t * BN + lane - s.ctx;
      const bool tree = (t + 1) * BN > s.ctx;
      float v[RW], mn[RW];
      uint32_t seen[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        bool see = true;
        if (tree && node >= 0) {
          const int i = (int)a.by_g.div((uint32_t)(s.rt * BM + warp * RW + r));
          see = node < s.n && i < s.n && sees_node(a, s.row0 + i, i, node);
        }
        v[r] = see ? (x[r][0] + x[r][1]) * a.scale : -INFINITY;
        mn[r] = v[r];
        seen[r] = tree ? __ballot_sync(0xffffffffu, see) : 0u;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int r = 0; r < RW; ++r) mn[r] = fmaxf(mn[r], __shfl_xor_sync(0xffffffffu, mn[r], o));
      float p[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        mn[r] = fmaxf(mn[r], m[r]);
        const float base = mn[r] == -INFINITY ? 0.f : mn[r];
        p[r] = expf(v[r] - base);
        const float alpha = expf(m[r] - base);
        m[r] = mn[r];
        l[r] = l[r] * alpha + p[r];  // this lane's keys
        if (lane == 0) {
          al_s[warp * RW + r] = alpha;
          vis_s[warp * RW + r] = seen[r];
        }
      }
      if constexpr (RW == 4) *(float4*)(pt + lane * PP + 4 * warp) = make_float4(p[0], p[1], p[2], p[3]);
      else pt[lane * PP + warp] = p[0];
      __syncthreads();
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int dim = tid + 128 * d;
        if (dim >= D) break;
#pragma unroll
        for (int r = 0; r < BM; ++r) acc[d][r] *= al_s[r];
        // A V that a row does not see must not count for it even where it is not finite (0 * NaN):
        // such a value is added for the rows that see it and leaves the tile.
        if (tree && (a.mask || s.n > 1)) {
          float* column = (float*)vt + dim;
          uint32_t odd = 0;
#pragma unroll 8
          for (int k = 0; k < BN; ++k) odd |= (uint32_t)!isfinite(column[k * P]) << k;
#pragma unroll 1
          for (; odd; odd &= odd - 1) {
            const int k = __ffs(odd) - 1;
            const float v1 = column[k * P];
#pragma unroll
            for (int r = 0; r < BM; ++r)
              if (vis_s[r] >> k & 1u) acc[d][r] += pt[k * PP + r] * v1;
            column[k * P] = 0.f;
          }
        }
#pragma unroll 8
        for (int k = 0; k < BN; ++k) {
          const float v1 = vt[k * P + dim];
#pragma unroll
          for (int r = 0; r < BM; r += 4) {
            const float4 pr = *(const float4*)(pt + k * PP + r);
            acc[d][r] += pr.x * v1;
            acc[d][r + 1] += pr.y * v1;
            acc[d][r + 2] += pr.z * v1;
            acc[d][r + 3] += pr.w * v1;
          }
        }
      }
      __syncthreads();  // the stage and the probabilities are free
    }
    cp_async_wait<0>();
    // (max, sum) of every row, through the probabilities' space.
    float2* ml = (float2*)pt;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      l[r] = warp_sum(l[r]);
      if (lane == 0) ml[warp * RW + r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (w == begin ? 0 : 1);
#pragma unroll
    for (int r = 0; r < BM; ++r) {
      const int R = s.rt * BM + r;
      if (R >= NR) break;
      const int i = (int)a.by_g.div((uint32_t)R), row = s.row0 + i, head = s.h * a.G + R - i * a.G;
      const float2 v = ml[r];
      if (whole) {
        const bool empty = v.y == 0.f && !sees_any(a, row, s.n, s.ctx);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (tid + 128 * d < D)
            ((float*)a.out)[((int64_t)row * a.nh + head) * D + tid + 128 * d] = empty ? 0.f : acc[d][r] / v.y;
        if (a.lse && tid == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<float>(v.x, v.y);
      } else {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (tid + 128 * d < DP) a.part[(slot * BM + r) * DP + tid + 128 * d] = acc[d][r];
        if (tid == 0) a.part_ml[slot * BM + r] = v;
      }
    }
    __syncthreads();
    w += s.step;
  }
}

// ---- host ----------------------------------------------------------------------------------
// Which kernel and how many CTAs, by the query vectors that share a cached head.
struct TreePlan {
  int dp, bm, bn, ctas;
  bool tc, whole;
  uint64_t work;
};
inline TreePlan tree_plan(const pp_paged_cache& c, const pp_paged_batch& b, uint32_t n_heads, int sms) {
  TreePlan p;
  p.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const uint64_t G = n_heads / c.n_kv_heads, vectors = (uint64_t)(b.max_rows ? b.max_rows : 1) * G;
  uint64_t per_sm = 2;
  p.tc = false;
  if (c.dtype == PP_F32) {
    p.bm = vectors <= 4 ? 4 : 16;
    p.bn = kTreeFBN;
    per_sm = p.dp == 64 ? 5 : p.dp == 128 ? 3 : 1;
  } else {
    if (p.dp == 256) per_sm = 1;
    const uint64_t tiles8 = (vectors + 7) / 8 * b.batch * c.n_kv_heads * (((uint64_t)b.max_len + kTreeBN - 1) / kTreeBN);
    p.tc = vectors > 8 && tiles8 > kNarrowTiles * per_sm * sms;
    p.bm = p.tc ? 128 : 8;
    p.bn = kTreeBN;
  }
  const uint64_t units = ((uint64_t)b.rows * G / p.bm + b.batch) * c.n_kv_heads;
  p.whole = b.max_len <= (uint32_t)p.bn * (c.dtype == PP_F32 ? kWholeF32 : p.tc ? kWholeTc : kWholeNarrow);
  const uint64_t tiles = units * (p.whole ? 1 : ((uint64_t)b.max_len + p.bn - 1) / p.bn + 1);
  const uint64_t most = (uint64_t)sms * per_sm;
  p.ctas = (int)(tiles < most ? (tiles ? tiles : 1) : most);
  p.work = 2ull * p.ctas * p.bm * (p.dp + 2) * 4;
  return p;
}

// Tensor maps of the layer's K and V, boxes of least .. most rows; box 0 (16-byte copies then) where they do not fit.
inline TreeMaps tree_maps(const pp_paged_cache& c, const PagedView& v, int least, int most) noexcept {
  TreeMaps m = {};
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (Encode)p;
  }();
  if (!encode || c.dtype == PP_F32 || c.page_size % least) return m;
  int box = most;
  while (c.page_size % box) box >>= 1;
  // Heads, rows and pages by ascending stride; a dimension of one element takes any stride.
  struct Dim {
    uint64_t size, stride;
    int what;
  } d[3] = {{c.n_kv_heads, (uint64_t)v.head_bytes, 0}, {c.page_size, (uint64_t)v.row_bytes, 1},
            {c.n_pages, (uint64_t)v.page_bytes, 2}};
  for (Dim& x : d) {
    if (x.size == 1) x.stride = (uint64_t)c.head_dim * 2;
    if (x.stride >= (1ull << 40)) return m;
  }
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (d[j].stride > d[j + 1].stride) {
        const Dim t = d[j];
        d[j] = d[j + 1];
        d[j + 1] = t;
      }
  cuuint64_t size[4] = {c.head_dim}, stride[3];
  cuuint32_t box_dim[4] = {64, 1, 1, 1}, one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i) {
    size[i + 1] = d[i].size;
    stride[i] = d[i].stride;
    if (d[i].what == 0) m.at_head = i + 1;
    else if (d[i].what == 1) m.at_row = i + 1, box_dim[i + 1] = box;
    else m.at_page = i + 1;
  }
  const CUtensorMapDataType t = c.dtype == PP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  for (int i = 0; i < 2; ++i)
    if (encode(i ? &m.v : &m.k, t, 4, i ? v.v : v.k, size, stride, box_dim, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return m;
  m.box = box;
  return m;
}

template <typename T, int DP>
pp_status run_tree_narrow(const TreeArgs& a, const TreeMaps& m, cudaStream_t st) {
  const pp_status r = launch_tree<pp_tree_narrow_kernel<T, DP>>(a, kTreeThreads, NarrowCfg<DP>::smem(a.b.batch), st, m);
  if (r != PP_OK || a.whole) return r;
  return launch_join<T, DP>(a, st);
}
template <typename T>
pp_status run_tree_16(const TreeArgs& a, const TreeMaps& m, int dp, cudaStream_t st) {
  if (dp == 64) return run_tree_narrow<T, 64>(a, m, st);
  if (dp == 128) return run_tree_narrow<T, 128>(a, m, st);
  return run_tree_narrow<T, 256>(a, m, st);
}
template <int DP, int BM>
pp_status run_tree_f32_rows(const TreeArgs& a, cudaStream_t st) {
  const pp_status r = launch_tree<pp_tree_f32_kernel<DP, BM>>(a, kTreeThreads, TreeFCfg<DP, BM>::smem(a.b.batch), st);
  if (r != PP_OK || a.whole) return r;
  return launch_join<float, DP>(a, st);
}
template <int DP>
pp_status run_tree_f32(const TreeArgs& a, cudaStream_t st) {
  return a.bm == 4 ? run_tree_f32_rows<DP, 4>(a, st) : run_tree_f32_rows<DP, 16>(a, st);
}

inline const char* tree_problem(const pp_paged_cache* c, const pp_paged_batch* b, uint32_t n_heads) {
  if (const char* m = cache_problem(c)) return m;
  if (const char* m = batch_problem(b)) return m;
  if (n_heads == 0 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 1024)
    return "n_heads must be a multiple of n_kv_heads, at most 1024 times it";
  if (b->max_rows > (uint32_t)kTreeMostRows) return "max_rows out of range";
  // The line of tiles is counted in 32 bits, whatever the device's lengths turn out to be.
  const uint64_t G = n_heads / c->n_kv_heads;
  const uint64_t units = ((uint64_t)b->rows * G / 4 + b->batch) * c->n_kv_heads;
  const uint64_t longest = (uint64_t)b->table_stride * c->page_size;
  if (longest > kTreeMostPositions) return "a page table of more than 2^31 - 4096 positions";
  if (units * (longest / 32 + 1) > 0x7fffffffull) return "rows times positions out of range";
  return nullptr;
}

}  // namespace pp

extern "C" uint64_t pp_tree_attention_work_bytes(const pp_paged_cache* cache, const pp_paged_batch* batch,
                                                 uint32_t n_heads) {
  if (const char* m = tree_problem(cache, batch, n_heads)) {
    paged_fail(PP_E_INVALID, m);
    return 0;
  }
  const int found = sm_count(cache->cuda_device), sms = found ? found : 148;
  return tree_plan(*cache, *batch, n_heads, sms).work;
}

extern "C" pp_status pp_tree_attention(const pp_paged_cache* cache, const pp_paged_batch* batch,
                                       const pp_tree_query* q, void* work, uint64_t work_bytes,
                                       uint32_t* err, void* stream) {
  if (!q) return paged_fail(PP_E_INVALID, "null query");
  if (const char* m = tree_problem(cache, batch, q->n_heads)) return paged_fail(PP_E_INVALID, m);
  if (!q->q || !q->out || !work) return paged_fail(PP_E_INVALID, "null argument");
  if (q->layer >= cache->layers) return paged_fail(PP_E_INVALID, "layer outside the cache");
  const int e = dtype_bytes(cache->dtype);
  if ((uintptr_t)q->q % 16 || (uintptr_t)q->out % 16 || q->q_stride % (16 / e))
    return paged_fail(PP_E_INVALID, "q, its row stride and out must be multiples of 16 bytes");
  if (batch->rows > 1 && q->q_stride < (int64_t)q->n_heads * cache->head_dim)
    return paged_fail(PP_E_INVALID, "q_stride shorter than a row");
  if (q->mask && (q->mask_words == 0 || q->mask_words > 32768))
    return paged_fail(PP_E_INVALID, "mask_words must be 1..32768 with a mask");
  if (q->out == q->q) return paged_fail(PP_E_INVALID, "out must not be q");
  DeviceScope dev(cache->cuda_device);
  const int sms = dev.ok ? sm_count(cache->cuda_device) : 0;
  if (!sms) return paged_fail(PP_E_CUDA, "cannot use the cache's device");
  const TreePlan p = tree_plan(*cache, *batch, q->n_heads, sms);
  if ((uintptr_t)work % 16 || work_bytes < p.work)
    return paged_fail(PP_E_INVALID, "work must be 16-byte aligned and pp_tree_attention_work_bytes long");
  if (batch->rows == 0) return PP_OK;
  TreeArgs a = {};
  a.c = paged_view(*cache, q->layer);
  a.b = batch_view(*batch);
  a.q = q->q;
  a.out = q->out;
  a.lse = q->lse;
  a.q_stride = q->q_stride;
  a.mask = q->mask;
  a.mask_words = (int32_t)q->mask_words;
  a.nh = (int32_t)q->n_heads;
  a.G = (int32_t)(q->n_heads / cache->n_kv_heads);
  a.scale = q->scale;
  a.by_g = FastDiv((uint32_t)a.G);
  a.by_kv = FastDiv(cache->n_kv_heads);
  a.bm = p.bm;
  a.part = (float*)work;
  a.part_ml = (float2*)(a.part + 2ll * p.ctas * p.bm * p.dp);
  a.ctas = p.ctas;
  a.whole = p.whole;
  a.slack = cache->dtype == PP_F32 ? kSlackF32 : p.tc ? kSlackTc : kSlackNarrow;
  a.dev = cache->cuda_device;
  a.err = err;
  const cudaStream_t st = (cudaStream_t)stream;
  if (cache->dtype == PP_F32) {
    if (p.dp == 64) return run_tree_f32<64>(a, st);
    if (p.dp == 128) return run_tree_f32<128>(a, st);
    return run_tree_f32<256>(a, st);
  }
  const TreeMaps m = tree_maps(*cache, a.c, p.tc ? 8 : 16, p.tc ? 64 : 16);
  if (p.tc) return run_tree_tc(a, m, cache->dtype, p.dp, st);
  if (cache->dtype == PP_BF16) return run_tree_16<__nv_bfloat16>(a, m, p.dp, st);
  return run_tree_16<__half>(a, m, p.dp, st);
}
