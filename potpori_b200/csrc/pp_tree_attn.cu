// pp_tree_attention: the kernels for caches of 16-bit types (mma.sync) and of F32 (CUDA cores),
// and the entry point. The work split and the join of partials are in pp_tree_attn.cuh.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_attn.cuh"
#include "pp_tree_attn.cuh"
#include "pp_tree_plan.cuh"

using namespace pp;

namespace pp {

// ---- 16-bit caches -------------------------------------------------------------------------
// CTA of 4 warps: WM warps over the rows (16 each), 4 / WM over the keys of a 64-key tile, each
// with its own running maximum, sum and output, joined in shared memory when the unit's segment
// ends. Q stays in registers; K and V tiles come through a ring of NS stages by 16-byte
// asynchronous copies, each row from wherever its page is. With WM = 1 (up to 16 query vectors, a
// decoded token or a short chain) a warp fetches and consumes its own 16 keys of every tile and
// the loop has no CTA barrier.
constexpr int kTreeThreads = 128;
constexpr int kTreeBN = 64;
constexpr uint64_t kTreeTcAbove = 32;  // more query vectors of a head than this: pp_tree_tc.cu

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
// Exponent all ones in either half of a register of T.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t v) {
  constexpr uint32_t E = sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  return ((v & E) == E ? 0xffffu : 0u) | ((v >> 16 & E) == E ? 0xffff0000u : 0u);
}

template <int DP, int WM>
struct TreeCfg {
  static constexpr int WN = 4 / WM, BM = 16 * WM, BN = kTreeBN, KW = BN / WN;
  static constexpr int NS = DP == 256 ? 2 : 3;
  static constexpr int kRow = DP * 2, kTile = BN * kRow, kStage = 2 * kTile;
  static constexpr int kOPitch = DP + 4;
  static constexpr int kQ = BM * kRow;
  static constexpr int kOut = 4 * 16 * kOPitch * 4 + 4 * 16 * 8;  // outputs and (max, sum) of 4 warps
  static constexpr int kRing = NS * kStage > kOut ? NS * kStage : kOut;
  static constexpr size_t smem(int batch) { return kRing + kQ + 8 * (size_t)(batch + 1); }
};

template <typename T, int DP, int WM>
__global__ void __launch_bounds__(kTreeThreads) pp_tree_mma_kernel(const TreeArgs a) {
  using C = TreeCfg<DP, WM>;
  constexpr int WN = C::WN, BM = C::BM, BN = C::BN, KW = C::KW, NS = C::NS, RB = C::kRow;
  constexpr int UR = DP / 8;  // 16-byte units of a row
  extern __shared__ __align__(128) uint8_t sm[];
  uint8_t* ring = sm;
  uint8_t* qs = sm + C::kRing;
  int64_t* prefix = (int64_t*)(qs + C::kQ);
  __shared__ int64_t scan[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wn = warp / WM, g4 = lane >> 2, t4 = lane & 3;
  const int D = a.c.head_dim;
  const float sc = soft_scale<T>(a.scale);

  pdl_launch_dependents();
  tile_prefix<BM, BN, kTreeThreads>(a, prefix, scan, blockIdx.x == 0);
  const int64_t total = prefix[a.b.batch], per = tiles_per_cta(a, total);
  const int64_t begin = blockIdx.x * per, end = min(total, begin + per);

  for (int64_t w = begin; w < end;) {
    const Segment s = segment_at<BM, BN>(a, prefix, w, end);
    const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
    const int NR = s.n * a.G;

    // A warp fetches 16 rows of every tile (with WM = 1 those that it consumes). Lane l < 16 looks
    // row l's page up a tile ahead of the copies, so that no copy waits for the page table.
    auto look = [&](int t) -> int64_t {
      const int idx = t * BN + warp * 16 + (lane & 15);
      if (t >= s.t1 || idx >= s.len) return -1;
      const int64_t off = paged_offset(a.c, table, a.b.table_stride, idx);
      if (off < 0) {
        if (a.err && lane < 16) atomicOr(a.err, PAGED_BAD_PAGE);
        return -1;
      }
      return off + (int64_t)s.h * a.c.head_bytes;
    };
    auto load_tile = [&](int stage, int64_t mine) {
      constexpr int RP = 32 / UR;
      const int u = lane % UR, sub = lane / UR;
      uint8_t* kd = ring + stage * C::kStage;
#pragma unroll
      for (int i = 0; i < 16 / RP; ++i) {
        const int l = i * RP + sub, r = warp * 16 + l;
        const int64_t off = __shfl_sync(0xffffffffu, mine, l);
        const bool read = off >= 0 && 8 * u < D;
        const int64_t at = read ? off + 16 * u : 0;
        const int dst = r * RB + ((u ^ (r & 7)) << 4);
        cp_async16(kd + dst, a.c.k + at, read);
        cp_async16(kd + C::kTile + dst, a.c.v + at, read);
      }
    };
    auto sync = [&] {
      if constexpr (WM == 1) __syncwarp();
      else __syncthreads();
    };

#pragma unroll
    for (int i = 0; i < NS - 1; ++i) {
      if (s.t0 + i < s.t1) load_tile(i, look(s.t0 + i));
      cp_async_commit();
    }
    int64_t ahead = look(s.t0 + NS - 1);
    // Queries: BM rows, zero past the unit's.
    for (int e = tid; e < BM * UR; e += kTreeThreads) {
      const int r = e / UR, u = e % UR, R = s.rt * BM + r;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (R < NR && 8 * u < D) {
        const int i = R / a.G;
        v = *(const uint4*)((const T*)a.q + (int64_t)(s.row0 + i) * a.q_stride +
                            (int64_t)(s.h * a.G + R - i * a.G) * D + 8 * u);
      }
      *(uint4*)(qs + r * RB + ((u ^ (r & 7)) << 4)) = v;
    }
    __syncthreads();
    constexpr bool kQReg = DP <= 128;
    uint32_t qa[kQReg ? DP / 16 : 1][4];
    const int qrow = wm * 16 + (lane & 15);
    const uint8_t* qp = qs + qrow * RB;
    if constexpr (kQReg) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
        ldmatrix_x4a(qa[ks], qp + (((2 * ks + (lane >> 4)) ^ (qrow & 7)) << 4));
    }
    // The thread's two rows: g4 and g4 + 8 of the warp's 16.
    const int RA = s.rt * BM + wm * 16 + g4, RBw = RA + 8;
    const int iA = RA / a.G, iB = RBw / a.G;

    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float mrow[2] = {-INFINITY, -INFINITY}, lrow[2] = {0.f, 0.f};

    for (int t = s.t0; t < s.t1; ++t) {
      const int stage = (t - s.t0) % NS;
      cp_async_wait<NS - 2>();
      sync();
      if (t + NS - 1 < s.t1) load_tile((t - s.t0 + NS - 1) % NS, ahead);
      cp_async_commit();
      ahead = look(t + NS);
      const uint8_t* kt = ring + stage * C::kStage;
      const uint8_t* vt = kt + C::kTile;
      const int kb = wn * KW;

      float x[KW / 8][4];
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        if (16 * ks >= D) break;
        uint32_t qf[4];
        if constexpr (kQReg) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[e] = qa[ks][e];
        } else {
          ldmatrix_x4a(qf, qp + (((2 * ks + (lane >> 4)) ^ (qrow & 7)) << 4));
        }
#pragma unroll
        for (int np = 0; np < KW / 16; ++np) {
          const int r = kb + 16 * np + (lane & 7) + ((lane >> 4) << 3);
          uint32_t kf[4];
          ldmatrix_x4a(kf, kt + r * RB + (((2 * ks + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
          mma16<T>(x[2 * np], qf, kf[0], kf[1]);
          mma16<T>(x[2 * np + 1], qf, kf[2], kf[3]);
        }
      }
      // Scale; mask where the tile reaches past the context.
      const int j0 = t * BN + kb;
      const bool tree = j0 + KW > s.ctx;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < KW / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = x[j][e] * sc;
          if (tree) {
            const int node = j0 + 8 * j + 2 * t4 + (e & 1) - s.ctx;
            const int i = e < 2 ? iA : iB;
            if (node >= 0 && (node >= s.n || i >= s.n || !sees_node(a, s.row0 + i, i, node))) v = -INFINITY;
          }
          x[j][e] = v;
          mx[e >> 1] = fmaxf(mx[e >> 1], v);
        }
      float base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        const float mn = fmaxf(mrow[i], mx[i]);
        base[i] = mn == -INFINITY ? 0.f : mn;
        const float alpha = soft_exp<T>(mrow[i] - base[i]);
        mrow[i] = mn;
        lrow[i] *= alpha;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * i] *= alpha;
          o[n][2 * i + 1] *= alpha;
        }
      }
#pragma unroll
      for (int j = 0; j < KW / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = soft_exp<T>(x[j][e] - base[e >> 1]);
          lrow[e >> 1] += x[j][e];
        }
      // Hidden nodes: their V must not count even where it is not finite (0 * NaN). Look for such
      // values only where some row can be blind to a node.
      bool dirty = false;
      if (tree && (a.mask || s.n > 1)) {
        uint32_t found = 0;
        for (int e = lane; e < KW * UR; e += 32) {
          const uint4 v = *(const uint4*)(vt + kb * RB + e * 16);
          found |= nonfinite_halves<T>(v.x) | nonfinite_halves<T>(v.y) | nonfinite_halves<T>(v.z) | nonfinite_halves<T>(v.w);
        }
        dirty = __any_sync(0xffffffffu, found != 0);
      }
      // O += P V. P is carried as hi + lo parts: rounded to T alone it would add as much error as
      // the rounding of the output.
#pragma unroll
      for (int ks = 0; ks < KW / 16; ++ks) {
        uint32_t ph[4], pl[4];
        split2<T>(x[2 * ks][0], x[2 * ks][1], ph[0], pl[0]);
        split2<T>(x[2 * ks][2], x[2 * ks][3], ph[1], pl[1]);
        split2<T>(x[2 * ks + 1][0], x[2 * ks + 1][1], ph[2], pl[2]);
        split2<T>(x[2 * ks + 1][2], x[2 * ks + 1][3], ph[3], pl[3]);
        const int r = kb + 16 * ks + (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
        for (int dp = 0; dp < DP / 16; ++dp) {
          if (16 * dp >= D) break;
          uint32_t vf[4];
          ldmatrix_x4_trans(vf, vt + r * RB + (((2 * dp + (lane >> 4)) ^ (r & 7)) << 4));
          if (dirty) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[e] &= ~nonfinite_halves<T>(vf[e]);
          }
          mma16<T>(o[2 * dp], ph, vf[0], vf[1]);
          mma16<T>(o[2 * dp + 1], ph, vf[2], vf[3]);
          mma16<T>(o[2 * dp], pl, vf[0], vf[1]);
          mma16<T>(o[2 * dp + 1], pl, vf[2], vf[3]);
        }
      }
      if (dirty) {  // the non-finite values of V, for the rows that see them
#pragma unroll
        for (int j = 0; j < KW / 8; ++j)
          for (int k8 = 0; k8 < 8; ++k8) {
            const int r = kb + 8 * j + k8, node = t * BN + r - s.ctx;
            const int from = (lane & ~3) | (k8 >> 1);
            const float a0 = __shfl_sync(0xffffffffu, x[j][0], from), a1 = __shfl_sync(0xffffffffu, x[j][1], from);
            const float b0 = __shfl_sync(0xffffffffu, x[j][2], from), b1 = __shfl_sync(0xffffffffu, x[j][3], from);
            const float p0 = k8 & 1 ? a1 : a0, p1 = k8 & 1 ? b1 : b0;
            if (node >= s.n) continue;
            const bool seeA = node < 0 || (iA < s.n && sees_node(a, s.row0 + iA, iA, node));
            const bool seeB = node < 0 || (iB < s.n && sees_node(a, s.row0 + iB, iB, node));
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              const uint32_t v = *(const uint32_t*)(vt + r * RB + ((n ^ (r & 7)) << 4) + 4 * t4);
              const uint32_t bad = nonfinite_halves<T>(v);
              T e2[2];
              *(uint32_t*)e2 = v;
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                if (!(bad >> (16 * q) & 1u)) continue;
                if (seeA) o[n][q] += p0 * Elem<T>::get(e2[q]);
                if (seeB) o[n][2 + q] += p1 * Elem<T>::get(e2[q]);
              }
            }
          }
      }
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring is free
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lrow[i] += __shfl_xor_sync(0xffffffffu, lrow[i], 1);
      lrow[i] += __shfl_xor_sync(0xffffffffu, lrow[i], 2);
    }
    // Outputs [wn][BM][DP + 4] and (max, sum) [wn][BM] of the warps.
    float* os = (float*)ring;
    float2* ml = (float2*)(ring + 4 * 16 * C::kOPitch * 4);
    {
      float* o0 = os + (size_t)(wn * BM + wm * 16 + g4) * C::kOPitch + 2 * t4;
      float* o1 = o0 + 8 * C::kOPitch;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        *(float2*)(o0 + 8 * n) = make_float2(o[n][0], o[n][1]);
        *(float2*)(o1 + 8 * n) = make_float2(o[n][2], o[n][3]);
      }
      if (t4 == 0) {
        ml[wn * BM + wm * 16 + g4] = make_float2(mrow[0], lrow[0]);
        ml[wn * BM + wm * 16 + g4 + 8] = make_float2(mrow[1], lrow[1]);
      }
    }
    __syncthreads();
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (w == begin ? 0 : 1);
    const int rows = min(BM, NR - s.rt * BM);
    for (int e = tid; e < rows * UR; e += kTreeThreads) {
      const int r = e / UR, u = e % UR, R = s.rt * BM + r, i = R / a.G;
      float m = ml[r].x;
#pragma unroll
      for (int k = 1; k < WN; ++k) m = fmaxf(m, ml[k * BM + r].x);
      const float mb = m == -INFINITY ? 0.f : m;
      float l = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WN; ++k) {
        const float2 v = ml[k * BM + r];
        const float wgt = WN == 1 ? 1.f : soft_exp<T>(v.x - mb);
        l += v.y * wgt;
        const float* src = os + (size_t)(k * BM + r) * C::kOPitch + 8 * u;
#pragma unroll
        for (int d = 0; d < 8; ++d) f[d] += src[d] * wgt;
      }
      if (whole) {
        const int row = s.row0 + i, head = s.h * a.G + R - i * a.G;
        const bool empty = l == 0.f && !sees_any(a, row, s.n, s.ctx);
#pragma unroll
        for (int d = 0; d < 8; ++d) f[d] = empty ? 0.f : f[d] / l;
        if (8 * u < D) store8((T*)a.out + ((int64_t)row * a.nh + head) * D + 8 * u, f);
        if (a.lse && u == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<T>(m, l);
      } else {
        float* dst = a.part + (slot * BM + r) * DP + 8 * u;
        *(float4*)dst = make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        if (u == 0) ((float2*)(a.part + (int64_t)2 * a.ctas * BM * DP))[slot * BM + r] = make_float2(m, l);
      }
    }
    __syncthreads();  // the ring may be filled again
    w += s.t1 - s.t0;
  }
}

// ---- F32 caches ----------------------------------------------------------------------------
// CUDA cores: on these tensor cores three products of split halves would be needed to keep F32,
// at the rate of an F32 multiply-add and with a worse sum. 16 query vectors, 32-key tiles.
constexpr int kTreeFBM = 16, kTreeFBN = 32, kTreeFStages = 2;
template <int DP>
struct TreeFCfg {
  static constexpr int P = DP + 4;  // row pitch: 16-byte columns of consecutive rows in other banks
  static constexpr int kTile = kTreeFBN * P * 4, kStage = 2 * kTile;
  static constexpr int kQ = kTreeFBM * P * 4;
  static constexpr int kS = kTreeFBM * 33 * 4, kP = kTreeFBN * kTreeFBM * 4, kRows = 5 * kTreeFBM * 4;
  static constexpr size_t smem(int batch) {
    return kTreeFStages * kStage + kQ + kP + kS + kRows + 8 * (size_t)(batch + 1) + 16;
  }
};

template <int DP>
__global__ void __launch_bounds__(kTreeThreads) pp_tree_f32_kernel(const TreeArgs a) {
  using C = TreeFCfg<DP>;
  constexpr int BM = kTreeFBM, BN = kTreeFBN, NS = kTreeFStages, P = C::P, UR = DP / 4;
  constexpr int DT = DP <= 128 ? 1 : DP / 128;  // dims of a thread: tid, tid + 128
  extern __shared__ __align__(128) uint8_t sm[];
  uint8_t* ring = sm;
  float* qs = (float*)(sm + NS * C::kStage);
  float* pt = qs + BM * P;        // [key][row]
  float* ss = pt + BN * BM;       // [row][33]
  float* m_s = ss + BM * 33;
  float* l_s = m_s + BM;
  float* al_s = l_s + BM;
  float* base_s = al_s + BM;
  uint32_t* vis_s = (uint32_t*)(base_s + BM);
  int64_t* prefix = (int64_t*)(((uintptr_t)(vis_s + BM) + 7) & ~(uintptr_t)7);
  __shared__ int64_t scan[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, D = a.c.head_dim;

  pdl_launch_dependents();
  tile_prefix<BM, BN, kTreeThreads>(a, prefix, scan, blockIdx.x == 0);
  const int64_t total = prefix[a.b.batch], per = tiles_per_cta(a, total);
  const int64_t begin = blockIdx.x * per, end = min(total, begin + per);

  for (int64_t w = begin; w < end;) {
    const Segment s = segment_at<BM, BN>(a, prefix, w, end);
    const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
    const int NR = s.n * a.G;
    auto load_tile = [&](int t, int stage) {
      constexpr int RP = kTreeThreads / UR;
      const int u = tid % UR;
      uint8_t* kd = ring + stage * C::kStage;
#pragma unroll
      for (int i = 0; i < BN / RP; ++i) {
        const int r = i * RP + tid / UR, idx = t * BN + r;
        int64_t off = -1;
        if (idx < s.len) {
          off = paged_offset(a.c, table, a.b.table_stride, idx);
          if (off < 0 && a.err && u == 0) atomicOr(a.err, PAGED_BAD_PAGE);
        }
        const bool read = off >= 0 && 4 * u < D;
        const int64_t at = read ? off + (int64_t)s.h * a.c.head_bytes + 16 * u : 0;
        cp_async16(kd + (r * P + 4 * u) * 4, a.c.k + at, read);
        cp_async16(kd + C::kTile + (r * P + 4 * u) * 4, a.c.v + at, read);
      }
    };
    load_tile(s.t0, 0);
    cp_async_commit();
    for (int e = tid; e < BM * UR; e += kTreeThreads) {
      const int r = e / UR, u = e % UR, R = s.rt * BM + r;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (R < NR && 4 * u < D) {
        const int i = R / a.G;
        v = *(const float4*)((const float*)a.q + (int64_t)(s.row0 + i) * a.q_stride +
                             (int64_t)(s.h * a.G + R - i * a.G) * D + 4 * u);
      }
      *(float4*)(qs + r * P + 4 * u) = v;
    }
    if (tid < BM) {
      m_s[tid] = -INFINITY;
      l_s[tid] = 0.f;
    }
    float acc[DT][BM];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < BM; ++r) acc[d][r] = 0.f;

    for (int t = s.t0; t < s.t1; ++t) {
      const int stage = (t - s.t0) % NS;
      if (t + 1 < s.t1) load_tile(t + 1, (t + 1 - s.t0) % NS);
      cp_async_commit();
      cp_async_wait<1>();
      __syncthreads();
      const float* kt = (const float*)(ring + stage * C::kStage);
      const float* vt = (const float*)(ring + stage * C::kStage + C::kTile);
      {  // scores: keys kk, kk + 16 by rows rr, rr + 8
        const int kk = tid & 15, rr = tid >> 4;
        float x[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
          const float4 k0 = *(const float4*)(kt + kk * P + d), k1 = *(const float4*)(kt + (kk + 16) * P + d);
          const float4 q0 = *(const float4*)(qs + rr * P + d), q1 = *(const float4*)(qs + (rr + 8) * P + d);
          x[0][0] += q0.x * k0.x + q0.y * k0.y + q0.z * k0.z + q0.w * k0.w;
          x[0][1] += q0.x * k1.x + q0.y * k1.y + q0.z * k1.z + q0.w * k1.w;
          x[1][0] += q1.x * k0.x + q1.y * k0.y + q1.z * k0.z + q1.w * k0.w;
          x[1][1] += q1.x * k1.x + q1.y * k1.y + q1.z * k1.z + q1.w * k1.w;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) ss[(rr + 8 * i) * 33 + kk + 16 * k] = x[i][k];
      }
      __syncthreads();
      // Softmax: warp w the rows 4 w .. 4 w + 3, lane = key.
      const int node = t * BN + lane - s.ctx;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 4 * warp + q, i = (s.rt * BM + r) / a.G;
        const bool see = node < 0 || (node < s.n && i < s.n && sees_node(a, s.row0 + i, i, node));
        const float v = see ? ss[r * 33 + lane] * a.scale : -INFINITY;
        const float mo = m_s[r], mn = fmaxf(mo, warp_max(v)), base = mn == -INFINITY ? 0.f : mn;
        const float p = expf(v - base);
        const float sum = warp_sum(p);
        const uint32_t seen = __ballot_sync(0xffffffffu, see);
        pt[lane * BM + r] = p;
        if (lane == 0) {
          const float alpha = expf(mo - base);
          m_s[r] = mn;
          l_s[r] = l_s[r] * alpha + sum;
          al_s[r] = alpha;
          vis_s[r] = seen;
        }
      }
      __syncthreads();
      const bool tree = (t + 1) * BN > s.ctx;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int dim = tid + 128 * d;
        if (dim >= D) break;
#pragma unroll
        for (int r = 0; r < BM; ++r) acc[d][r] *= al_s[r];
        if (!tree) {
#pragma unroll 4
          for (int k = 0; k < BN; ++k) {
            const float v = vt[k * P + dim];
#pragma unroll
            for (int r = 0; r < BM; r += 4) {
              const float4 p = *(const float4*)(pt + k * BM + r);
              acc[d][r] += p.x * v;
              acc[d][r + 1] += p.y * v;
              acc[d][r + 2] += p.z * v;
              acc[d][r + 3] += p.w * v;
            }
          }
        } else {  // an unseen V must not count even where it is not finite
          const int keys = min(BN, s.len - t * BN);
          for (int k = 0; k < keys; ++k) {
            const float v = vt[k * P + dim];
#pragma unroll
            for (int r = 0; r < BM; ++r)
              if (vis_s[r] >> k & 1u) acc[d][r] += pt[k * BM + r] * v;
          }
        }
      }
      __syncthreads();  // the stage, scores and probabilities are free
    }
    cp_async_wait<0>();
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (w == begin ? 0 : 1);
#pragma unroll
    for (int r = 0; r < BM; ++r) {
      const int R = s.rt * BM + r;
      if (R >= NR) break;
      const int i = R / a.G, row = s.row0 + i, head = s.h * a.G + R - i * a.G;
      const float m = m_s[r], l = l_s[r];
      if (whole) {
        const bool empty = l == 0.f && !sees_any(a, row, s.n, s.ctx);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (tid + 128 * d < D)
            ((float*)a.out)[((int64_t)row * a.nh + head) * D + tid + 128 * d] = empty ? 0.f : acc[d][r] / l;
        if (a.lse && tid == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<float>(m, l);
      } else {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (tid + 128 * d < DP) a.part[(slot * BM + r) * DP + tid + 128 * d] = acc[d][r];
        if (tid == 0) ((float2*)(a.part + (int64_t)2 * a.ctas * BM * DP))[slot * BM + r] = make_float2(m, l);
      }
    }
    __syncthreads();
    w += s.t1 - s.t0;
  }
}

// ---- host ----------------------------------------------------------------------------------
// Which kernel and how many CTAs, by the query vectors that share a cached head.
struct TreePlan {
  int dp, bm, bn, ctas;
  bool tc;
  uint64_t work;
};
inline TreePlan tree_plan(const pp_paged_cache& c, const pp_paged_batch& b, uint32_t n_heads, int sms, bool tc_ok) {
  TreePlan p;
  p.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const uint64_t G = n_heads / c.n_kv_heads, vectors = (uint64_t)(b.max_rows ? b.max_rows : 1) * G;
  p.tc = tc_ok && c.dtype != PP_F32 && vectors > kTreeTcAbove;
  if (c.dtype == PP_F32) {
    p.bm = kTreeFBM;
    p.bn = kTreeFBN;
  } else {
    p.bm = p.tc ? 128 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : 64;
    p.bn = kTreeBN;
  }
  const uint64_t units = ((uint64_t)b.rows * G / p.bm + b.batch) * c.n_kv_heads;
  const uint64_t tiles = units * (((uint64_t)b.max_len + p.bn - 1) / p.bn + 1);
  const uint64_t most = (uint64_t)sms * (p.dp == 256 ? 1 : 2);
  p.ctas = (int)(tiles < most ? (tiles ? tiles : 1) : most);
  p.work = 2ull * p.ctas * p.bm * (p.dp + 2) * 4;
  return p;
}

template <typename T, int DP, int WM>
pp_status run_tree_mma(const TreeArgs& a, cudaStream_t st) {
  using C = TreeCfg<DP, WM>;
  const pp_status r = launch_tree(pp_tree_mma_kernel<T, DP, WM>, a, kTreeThreads, C::smem(a.b.batch), st);
  if (r != PP_OK || a.ctas == 1) return r;
  return launch_join(pp_tree_join_kernel<T, DP, C::BM, C::BN>, a, C::BM, st);
}
template <typename T, int DP>
pp_status run_tree_rows(const TreeArgs& a, int bm, cudaStream_t st) {
  if (bm == 16) return run_tree_mma<T, DP, 1>(a, st);
  if (bm == 32) return run_tree_mma<T, DP, 2>(a, st);
  return run_tree_mma<T, DP, 4>(a, st);
}
template <typename T>
pp_status run_tree_16(const TreeArgs& a, int dp, int bm, cudaStream_t st) {
  if (dp == 64) return run_tree_rows<T, 64>(a, bm, st);
  if (dp == 128) return run_tree_rows<T, 128>(a, bm, st);
  return run_tree_rows<T, 256>(a, bm, st);
}
template <int DP>
pp_status run_tree_f32(const TreeArgs& a, cudaStream_t st) {
  const pp_status r = launch_tree(pp_tree_f32_kernel<DP>, a, kTreeThreads, TreeFCfg<DP>::smem(a.b.batch), st);
  if (r != PP_OK || a.ctas == 1) return r;
  return launch_join(pp_tree_join_kernel<float, DP, kTreeFBM, kTreeFBN>, a, kTreeFBM, st);
}

inline const char* tree_problem(const pp_paged_cache* c, const pp_paged_batch* b, uint32_t n_heads) {
  if (const char* m = cache_problem(c)) return m;
  if (const char* m = batch_problem(b)) return m;
  if (n_heads == 0 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 1024)
    return "n_heads must be a multiple of n_kv_heads, at most 1024 times it";
  if (b->max_rows > (1u << 20)) return "max_rows out of range";
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
  // Enough for either kernel: which one runs also depends on the query.
  const uint64_t x = tree_plan(*cache, *batch, n_heads, sms, true).work;
  const uint64_t y = tree_plan(*cache, *batch, n_heads, sms, false).work;
  return x > y ? x : y;
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
  // The tcgen05 kernel takes the maximum before the scale.
  const TreePlan p = tree_plan(*cache, *batch, q->n_heads, sms, q->scale > 0.f);
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
  a.part = (float*)work;
  a.ctas = p.ctas;
  a.min_per = 1;
  a.err = err;
  const cudaStream_t st = (cudaStream_t)stream;
  if (cache->dtype == PP_F32) {
    if (p.dp == 64) return run_tree_f32<64>(a, st);
    if (p.dp == 128) return run_tree_f32<128>(a, st);
    return run_tree_f32<256>(a, st);
  }
  if (p.tc) return run_tree_tc(a, cache->dtype, p.dp, st);
  if (cache->dtype == PP_BF16) return run_tree_16<__nv_bfloat16>(a, p.dp, p.bm, st);
  return run_tree_16<__half>(a, p.dp, p.bm, st);
}
