// Tree attention on the 5th-generation tensor cores (tcgen05, accumulators in TMEM): the kernel
// of pp_tree_attention for 16-bit caches when many query vectors share a cached head (a tree, or
// a chunk of a wide group). Row tiles of 128 vectors, key tiles of 64; the work split is
// pp_tree_attn.cuh's.
//
// One CTA, 224 threads, two CTAs on an SM (one at head_dim 256), so that one's softmax runs under
// the other's products:
//  * warps 4 and 5, producers: the K and V tiles by TMA, in boxes of 8 to 64 rows of one page and 64
//    dims, into a ring of tile-sized slots, in the order in which the products need them (K0, K1, V0,
//    K2, V1, ...). A box costs some 54 clocks whatever its size (the trees below: pages of 64
//    positions 92 to 98 us, 32 92, 16 122, 24, in boxes of 8, 165; 7, row by row, 279).
//    A slot holds 64-dim blocks of 64 rows x 128 bytes, the 16-byte unit u of row r at u ^ (r & 7):
//    read K-major it is the B operand of Q K^T, read MN-major the B operand of P V. Where pages are
//    not multiples of 8 positions, warps 4 and 5 fetch row by row with 16-byte asynchronous copies.
//  * warp 6, one thread: S = Q K^T (128 x 64, both operands in shared memory) and O += P V (P in
//    TMEM), each returned by a commit on an mbarrier. S has two places, and P takes its S's: S of a
//    tile is issued while the softmax works on the tile before, when the product of the one before
//    that is complete.
//  * warps 0-3, softmax: thread = row = TMEM lane. S of the row into 64 registers; mask; running
//    maximum; then, 32 columns at a time from TMEM again (no spills that way), exp2 and P. The output in
//    TMEM is rescaled only when a row's maximum has grown by more than 2^kSoftLag (until then the old base
//    serves: P stays in range and the sums are F32), so after the first tiles hardly ever. At the end of a
//    segment the rows leave from TMEM.
// P is carried as two parts of the cache's type, hi + lo, and both multiply V: rounded to one part
// it would add as much error as the rounding of the output.
// What bounds it: a tile's way through the softmax. Of 2000 to 2200 clocks a tile and CTA (two CTAs on
// the SM) 950 to 1150 are the exponentials and the two parts of P (64 exponentials a thread are 512 clocks
// of the SM's special units, and the other CTA wants them too), 250 to 380 the maximum, 470 to 570 the wait for S,
// whose products share the tensor core, about half busy, with the other CTA's. Left out one by one, on
// trial, neither half of the products nor the exponentials nor memory gave more than 5 %; two softmax
// warps a row were slower. 16 ragged trees of 61 nodes over 2048 to 4096 positions, 8 heads of 128, F16:
// 92 us replayed on a cool card, 545 TFLOP/s, 109 to 114 call after call at the power cap; one tree of
// 24 over 131072, BF16: 107 to 113 us, 4.8 TB/s, of which the tiles run at 6.5 TB/s, and 127 to 137.
// With heads of 256 the trees of 61 take 216 us (464 TFLOP/s), of 64 85.
// Every wait is bounded; one that expires sets bit 4 of the caller's error word, and the CTA still
// lets its copies and products land and frees its TMEM before it leaves.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_tree_attn.cuh"
#include "pp_tree_plan.cuh"

using namespace pp;

namespace pp {

constexpr int kTcThreads = 224;  // 7 warps: 14 on an SM leave 128 registers a thread
constexpr int kTcBM = 128, kTcBN = kTreeTile<__half>;
constexpr int kTcLag = 3;  // items a producer keeps in flight behind the one it issues

template <int DP>
struct TcCfg {
  static constexpr int kQ = kTcBM * DP * 2;
  static constexpr int kItem = kTcBN * DP * 2;  // a K or V tile
  static constexpr int kTurn = 4 * 4096;        // rows on their way out, 4 KB a softmax warp
  static constexpr int kSlots = DP == 64 ? 8 : 4;
  static constexpr int kPerSm = DP == 256 ? 1 : 2;
  static constexpr int kCols = DP == 256 ? 512 : 256;  // TMEM: O [DP], twice S or P [64]
  static constexpr int kBars = 192;
  // Two CTAs share 228 KB less 1 KB each: at head_dim 128 that leaves 1 KB beside Q, four slots and
  // the turn buffer, for the barriers and the prefix of up to 196 sequences; above, an SM
  // holds one CTA (trees of 24 over 300 to 600: 190 sequences 128 us, 210 197). (More slots than four
  // only lengthen every other load's way through memory: at the card's rate 148 x 2 x 64 KB in flight
  // are 3 us already.)
  static size_t smem(int batch) { return kQ + kTurn + kSlots * (size_t)kItem + kBars + prefix_bytes(batch); }
};

struct TcBars {
  uint64_t full[8], free[8];
  uint64_t q_full, s_full[2], p_full[2], pv_done, end;
  uint32_t tmem, dirty;
};
static_assert(sizeof(TcBars) <= 192, "barriers");

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// Descriptor of a SWIZZLE_128B operand: the low word holds its address / 16 and, MN-major, the bytes
// / 16 between its 64-element blocks; the high word 1024 bytes between 8-row atoms, version, swizzle.
// One thread issues every product, so what it computes per product counts: the words are kept and
// stepped by constants.
constexpr uint32_t kTcDescHi = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ constexpr uint32_t tc_lead(uint32_t bytes) { return (bytes >> 4) << 16; }
// kind::f16, F32 accumulator, A and B both of T, M = 128, N = n, B MN-major when mn.
template <typename T>
__device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool mn) {
  constexpr uint32_t t = __is_same(T, __half) ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kTcDescHi)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kTcDescHi)
      : "memory");
}
// 32 columns of the thread's lane.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t* r = (uint32_t*)v;
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 bits: which of the positions j0 .. j0 + 63 row i (array row `row`) sees.
__device__ __forceinline__ uint64_t seen64(const TreeArgs& a, const Segment& s, int row, int i, int j0) {
  const int node0 = j0 - s.ctx;  // may be negative: context
  const int skip = node0 < 0 ? -node0 : 0;
  if (skip >= 64) return ~0ull;
  const int first = node0 < 0 ? 0 : node0;
  uint64_t m = 0;
  if (i < s.n) {
    if (a.mask) {
      const uint32_t* w = a.mask + (int64_t)row * a.mask_words;
      const int k = first >> 5, sh = first & 31;
      const uint64_t w0 = k < a.mask_words ? w[k] : 0u, w1 = k + 1 < a.mask_words ? w[k + 1] : 0u,
                     w2 = k + 2 < a.mask_words ? w[k + 2] : 0u;
      m = (w0 | w1 << 32) >> sh;
      if (sh) m |= w2 << (64 - sh);
    } else if (i >= first) {
      m = i - first >= 63 ? ~0ull : (1ull << (i - first + 1)) - 1;
    }
    const int left = s.n - first;  // nodes from `first` on
    if (left < 64) m &= left <= 0 ? 0ull : (1ull << left) - 1;
  }
  return skip ? m << skip | ((1ull << skip) - 1) : m;
}

__device__ __forceinline__ uint32_t tc_pack(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&v;
}
__device__ __forceinline__ uint32_t tc_pack(float a, float b, __half*) {
  const __half2 v = __floats2half2_rn(a, b);
  return *(const uint32_t*)&v;
}
__device__ __forceinline__ float2 tc_unpack(uint32_t v, __nv_bfloat16*) { return make_float2(bf16lo(v), bf16hi(v)); }
__device__ __forceinline__ float2 tc_unpack(uint32_t v, __half*) { return __half22float2(*(const __half2*)&v); }

template <typename T, int DP>
__global__ void __launch_bounds__(kTcThreads, TcCfg<DP>::kPerSm) pp_tree_tc_kernel(const TreeArgs a, const __grid_constant__ TreeMaps maps) {
  using C = TcCfg<DP>;
  constexpr int BM = kTcBM, BN = kTcBN, UR = DP / 8, slots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t tc_smem[];
  uint8_t* sm = tc_smem;
  uint8_t* qs = sm;
  uint8_t* ring = sm + C::kQ + C::kTurn;
  TcBars* bars = (TcBars*)(ring + (size_t)slots * C::kItem);
  uint32_t* prefix = (uint32_t*)((uint8_t*)bars + C::kBars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = a.c.head_dim;
  if (smem_u32(sm) & 1023u) {  // cannot be (nothing is static); the caller is told
    if (tid == 0 && a.err) atomicOr(a.err, PAGED_TIMEOUT);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < slots; ++i) {
      mbar_init(&bars->full[i], maps.box && DP == 64 ? 1 : 2);
      mbar_init(&bars->free[i], 1);
    }
    mbar_init(&bars->q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
    }
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->end, 1);
    bars->dirty = 0;
    fence_barrier_init();
  }
  if (warp == 6) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)),
                 "r"(C::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_launch_dependents();
  tc_fence_before();
  const Line line = cut_line<BN, kTcThreads>(a, __builtin_ctz(BM), prefix, true, (uint32_t*)qs, blockIdx.x == 0);  // with CTA barriers
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const uint32_t tO = tmem, tS = tmem + DP;  // S of phase q at tS + 64 (q & 1), and its P in its place
  uint32_t begin, end;
  cta_range(line, blockIdx.x, begin, end);
  bool ok = true;

  constexpr int kFetchers = DP == 64 ? 1 : 2;  // warps that fetch by TMA, each its share of the dims
  if (warp >= 4 && warp < 4 + kFetchers && maps.box) {
    // ---- producers, by TMA: lane g looks row group g of a tile up (box rows, one page)
    constexpr int NB = DP / 64 / kFetchers;
    const int i0 = (warp - 4) * NB;  // 64-dim blocks i0 .. i0 + NB - 1
    const int groups = BN / maps.box;
    int n = 0;
    RingCursor rc;
    for (uint32_t w = begin; w < end && ok;) {
      const Segment s = segment_at<BN>(a, line, prefix, w, end);
      const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
      const int cnt = s.t1 - s.t0;
      // Places of tile i (V's turn), i + 1 (K's) and i + 2, looked up ahead of their copies.
      BoxPlace prev, cur, next;
      auto look = [&](BoxPlace& f, int i) { f.look(a, s, table, (s.t0 + i) * BN + lane * maps.box, i < cnt && lane < groups); };
      look(cur, 0);
      look(next, 1);
      prev = cur;
      for (int j = 0; j < 2 * cnt; ++j, ++n) {
        const bool isv = j == 2 * cnt - 1 || (j > 0 && !(j & 1));
        const int slot = rc.slot;
        if (n >= slots && !warp_wait(&bars->free[slot], rc.phase ^ 1u)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + (size_t)slot * C::kItem;
        if (elect_one()) mbar_arrive_expect_tx(&bars->full[slot], C::kItem / kFetchers);
        __syncwarp();
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
          const int page = __shfl_sync(0xffffffffu, isv ? prev.page : cur.page, g);
          const int row = __shfl_sync(0xffffffffu, isv ? prev.row : cur.row, g);
          if (elect_one())
#pragma unroll
            for (int i = 0; i < NB; ++i)
              tma_box(dst + (i0 + i) * (BN * 128) + g * maps.box * 128, isv ? &maps.v : &maps.k, &bars->full[slot], maps, 64 * (i0 + i),
                      s.h, row, page);
          __syncwarp();
        }
        rc.next(slots);
        if (j == 0 || isv) {
          prev = cur;
          cur = next;
          look(next, j / 2 + 2);
        }
      }
      w += s.step;
    }
    if (!ok)  // let the copies in flight land
      for (int i = n > slots ? n - slots : 0; i < n; ++i) warp_wait(&bars->full[i % slots], (uint32_t)(i / slots) & 1u);
  } else if ((warp == 4 || warp == 5) && !maps.box) {
    // ---- producers: warp pw the rows 32 pw .. + 31 of every tile
    const int pw = warp - 4;
    constexpr int RPP = 32 / UR;  // rows of one pass of a warp
    const int u = lane % UR, sub = lane / UR;
    int n = 0;
    RingCursor rc, done;
    for (uint32_t w = begin; w < end && ok;) {
      const Segment s = segment_at<BN>(a, line, prefix, w, end);
      const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
      const int cnt = s.t1 - s.t0;
      // Rows of tile i (V's turn), i + 1 (K's) and i + 2, looked up ahead of their copies.
      RowFetch<32> prev, cur, next;
      auto look = [&](RowFetch<32>& f, int i) { f.look(a, s, table, (s.t0 + i) * BN + pw * 32, i < cnt, lane); };
      look(cur, 0);
      look(next, 1);
      prev = cur;
      for (int j = 0; j < 2 * cnt; ++j, ++n) {
        const bool isv = j == 2 * cnt - 1 || (j > 0 && !(j & 1));
        const int slot = rc.slot;
        if (n >= slots && !warp_wait(&bars->free[slot], rc.phase ^ 1u)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + (size_t)slot * C::kItem;
        const uint8_t* base = isv ? a.c.v : a.c.k;
#pragma unroll 4
        for (int q = 0; q < 32 / RPP; ++q) {
          const int l = q * RPP + sub, r = pw * 32 + l;
          const int64_t off = isv ? prev.row(a, l) : cur.row(a, l);
          const bool read = off >= 0 && 8 * u < D;
          cp_async16(dst + (u >> 3) * (BN * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4), base + (read ? off + 16 * u : 0), read);
        }
        cp_async_commit();
        rc.next(slots);
        if (j == 0 || isv) {
          prev = cur;
          cur = next;
          look(next, j / 2 + 2);
        }
        if (n >= kTcLag) {
          cp_async_wait<kTcLag>();
          fence_async();
          warp_arrive(&bars->full[done.slot], lane);
          done.next(slots);
        }
      }
      w += s.step;
    }
    cp_async_wait<0>();
    fence_async();
    for (int i = n > kTcLag ? n - kTcLag : 0; i < n; ++i) {
      warp_arrive(&bars->full[done.slot], lane);
      done.next(slots);
    }
  } else if (warp == 6) {
    // ---- products: the warp waits together, one lane issues
    {
      constexpr uint32_t iqk = tc_idesc<T>(BN, false), ipv = tc_idesc<T>(DP, true);
      const uint32_t qa = (smem_u32(qs) >> 4) | tc_lead(16), ring_a = smem_u32(ring) >> 4;
      RingCursor rc;
      uint32_t q = 0, tiles = 0;  // phases of s_full and tiles so far
      uint32_t seg = 0;
      auto take = [&]() -> bool { return warp_wait(&bars->full[rc.slot], rc.phase); };
      for (uint32_t w = begin; w < end && ok;) {
        const Segment s = segment_at<BN>(a, line, prefix, w, end);
        const int cnt = s.t1 - s.t0;
        if (!warp_wait(&bars->q_full, seg)) {
          ok = false;
          break;
        }
        // Step i issues S of tile i + 1, then O of tile i. A segment has two phases of s_full more than
        // tiles: the first one's commit tells that the product before the last is complete, the second
        // one's that the last is.
        for (int i = -1; i < cnt; ++i, ++q) {
          // S of tile i + 1 takes the place of P of tile i - 1, whose product must be complete.
          if (i >= 1 && !warp_wait(&bars->pv_done, (tiles - 1) & 1u)) {
            ok = false;
            break;
          }
          if (i + 1 < cnt) {  // S = Q K^T from the ring's next item; dims past the head's are zero
            if (!take()) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t ka = (ring_a + rc.slot * (C::kItem >> 4)) | tc_lead(16), to = tS + 64 * (q & 1u);
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < DP / 16; ++ks)
                tc_mma_ss(to, qa + (ks >> 2) * (BM * 8) + (ks & 3) * 2, ka + (ks >> 2) * (BN * 8) + (ks & 3) * 2, iqk, ks != 0);
              tc_commit(&bars->s_full[q & 1u]);
              tc_commit(&bars->free[rc.slot]);
            }
            __syncwarp();
            rc.next(slots);
          } else {
            if (elect_one()) tc_commit(&bars->s_full[q & 1u]);
            __syncwarp();
          }
          if (i < 0) continue;
          if (!take() || !warp_wait(&bars->p_full[tiles & 1u], (tiles >> 1) & 1u)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t va = (ring_a + rc.slot * (C::kItem >> 4)) | tc_lead(BN * 128), tP = tS + 64 * (~q & 1u);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks) {
              tc_mma_ts(tO, tP + 32 * (ks >> 1) + 8 * (ks & 1), va + ks * 128, ipv, ks == 0 ? i : 1u);
              tc_mma_ts(tO, tP + 32 * (ks >> 1) + 8 * (ks & 1) + 16, va + ks * 128, ipv, 1u);
            }
            tc_commit(&bars->pv_done);
            tc_commit(&bars->free[rc.slot]);
          }
          __syncwarp();
          rc.next(slots);
          ++tiles;
        }
        if (!ok || !warp_wait(&bars->pv_done, (tiles - 1) & 1u)) {
          ok = false;
          break;
        }
        if (elect_one()) tc_commit(&bars->s_full[q & 1u]);
        __syncwarp();
        ++q;
        seg ^= 1u;
        w += s.step;
      }
      if (elect_one()) tc_commit(&bars->end);
      __syncwarp();
      warp_wait(&bars->end, 0);  // no product of this CTA runs when TMEM is freed
    }
  } else if (warp < 4) {
    // ---- softmax
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    // The maximum is taken before the scale, so the scale must be positive: another sign, or zero,
    // goes into the scores.
    const float sc = a.scale == 0.f ? 1.f : soft_scale<T>(fabsf(a.scale));
    // A segment's queries into Q's space, zero past the unit's: asynchronous copies, the next
    // segment's on their way while this one's rows leave.
    auto fetch_q = [&](const Segment& f) {
      const int nr = f.n * a.G;
#pragma unroll 4
      for (int e = tid; e < BM * UR; e += 128) {
        const int r = e / UR, u = e % UR, Rq = f.rt * BM + r;
        const bool read = Rq < nr && 8 * u < D;
        const int iq = (int)a.by_g.div((uint32_t)(read ? Rq : 0));
        const T* src = (const T*)a.q + (read ? (int64_t)(f.row0 + iq) * a.q_stride + (int64_t)(f.h * a.G + Rq - iq * a.G) * D + 8 * u : 0);
        cp_async16(qs + (u >> 3) * (BM * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4), src, read);
      }
      cp_async_commit();
    };
    Segment s;
    if (begin < end) {
      s = segment_at<BN>(a, line, prefix, begin, end);
      fetch_q(s);
    }
    int n0 = 0;  // items before this segment
    uint32_t q = 0, tiles = 0, seg = 0;  // phases of s_full, tiles so far
    for (uint32_t w = begin; w < end && ok;) {
      const int cnt = s.t1 - s.t0, NR = s.n * a.G;
      cp_async_wait<0>();
      fence_async();
      warp_arrive(&bars->q_full, lane);

      const int R = s.rt * BM + tid, i = (int)a.by_g.div((uint32_t)R), row = s.row0 + i;
      const bool idle = s.rt * BM + warp * 32 >= NR;
      // Tiles of context alone, which most are, come first and need nothing but the softmax: one test.
      const int plain = idle || a.scale <= 0.f ? 0 : s.ctx / BN - s.t0;
      float m = -INFINITY, high = -INFINITY, l = 0.f;  // base, maximum and sum of the row
      for (int t = 0; t < cnt; ++t, ++q, ++tiles) {
        if (!warp_wait(&bars->s_full[q & 1u], (q >> 1) & 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float x[2][32];
        const uint32_t at = tS + 64 * (q & 1u) + lanes;
        tc_ld32(at, x[0]);
        tc_ld32(at + 32, x[1]);
        tc_wait_ld();
        if (__builtin_expect(t >= plain, 0)) {
          const int j0 = (s.t0 + t) * BN;
          const bool tree = j0 + BN > s.ctx;
          const bool blind = tree && (a.mask || s.n > 1);
          if (blind || j0 + BN > s.len) {
            // Positions past the end hold whatever their page did: zeros there. And a V that some row
            // is blind to must not count even where it is not finite (0 * NaN): such values leave the
            // tile here and come back, for the rows that see them, with the output. The slot stays
            // until this tile's product, which waits for p_full.
            const int item = n0 + (t == cnt - 1 ? 2 * cnt - 1 : 2 * t + 2), slot = item % slots;
            if (!warp_wait(&bars->full[slot], (uint32_t)(item / slots) & 1u)) {
              ok = false;
              break;
            }
            uint32_t found = 0;
#pragma unroll 4
            for (int e = tid; e < BN * UR; e += 128) {
              uint4* p = (uint4*)(ring + (size_t)slot * C::kItem + e * 16);
              if (j0 + ((e >> 3) & (BN - 1)) >= s.len) {
                *p = make_uint4(0u, 0u, 0u, 0u);
              } else if (blind) {
                const uint4 v = *p;
                const uint32_t b0 = nonfinite_halves<T>(v.x), b1 = nonfinite_halves<T>(v.y), b2 = nonfinite_halves<T>(v.z), b3 = nonfinite_halves<T>(v.w);
                if (b0 | b1 | b2 | b3) {
                  found = 1;
                  *p = make_uint4(v.x & ~b0, v.y & ~b1, v.z & ~b2, v.w & ~b3);
                }
              }
            }
            if (found) bars->dirty = seg + 1;
            fence_async();
          }
          if (idle) {  // no row of the warp is in the unit: its P may be anything
            tc_fence_before();
            warp_arrive(&bars->p_full[tiles & 1u], lane);
            continue;
          }
          if (a.scale <= 0.f) {
            const float by = a.scale < 0.f ? -1.f : 0.f;
#pragma unroll
            for (int k = 0; k < 64; ++k) x[k >> 5][k & 31] *= by;
          }
          if (tree) {
            const uint64_t see = seen64(a, s, row, i, j0);
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (!(see >> k & 1u)) x[k >> 5][k & 31] = -INFINITY;
          }
          tc_st32(at, *(const uint32_t(*)[32])x[0]);
          tc_st32(at + 32, *(const uint32_t(*)[32])x[1]);
          tc_wait_st();
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 64; ++k) top[k & 3] = fmaxf(top[k & 3], x[k >> 5][k & 31]);
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        // scale > 0; rounded up for F16, as no exponent below may pass what this one says
        high = fmaxf(high, __is_same(T, __half) ? __fmul_ru(most, sc) : most * sc);
        float alpha = 1.f;
        const bool rescale = __any_sync(0xffffffffu, soft_outgrown<T>(high, m));
        if (rescale) {  // all of the warp's rows to their maxima, so that the next time is further off
          const float mn = fmaxf(m, soft_base<T>(high));
          alpha = soft_exp<T>(m - (mn == -INFINITY ? 0.f : mn));
          m = mn;
          l *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;
        // P over S: of each 32 keys 16 columns of high parts, 16 of low ones. Two elements an
        // instruction where there is one for F32 pairs.
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float xc[32];
          uint32_t p[32];
          tc_ld32(at + c, xc);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 y = __ffma2_rn(make_float2(xc[2 * k], xc[2 * k + 1]), make_float2(sc, sc), make_float2(-base, -base));
            const float2 v = make_float2(soft_exp<T>(y.x), soft_exp<T>(y.y));
            sum = __fadd2_rn(sum, v);
            p[k] = tc_pack(v.x, v.y, (T*)nullptr);
            const float2 h = tc_unpack(p[k], (T*)nullptr);
            const float2 rest = __fadd2_rn(v, make_float2(-h.x, -h.y));
            p[16 + k] = tc_pack(rest.x, rest.y, (T*)nullptr);
          }
          tc_st32(at + c, p);
        }
        l += sum.x + sum.y;
        if (rescale && t > 0) {
          // The next phase comes when the product of the tile before this one is complete.
          if (!warp_wait(&bars->s_full[~q & 1u], ((q + 1) >> 1) & 1u)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            float o[32];
            tc_ld32(tO + lanes + c, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= alpha;
            tc_st32(tO + lanes + c, *(const uint32_t(*)[32])o);
          }
        }
        tc_wait_st();
        tc_fence_before();
        warp_arrive(&bars->p_full[tiles & 1u], lane);
      }
      // Every product with Q and into O is complete after the segment's last phase.
      if (!ok || !warp_wait(&bars->s_full[q & 1u], (q >> 1) & 1u) ||
          !warp_wait(&bars->s_full[~q & 1u], ((q + 1) >> 1) & 1u)) {
        ok = false;
        break;
      }
      q += 2;
      tc_fence_after();
      // Every softmax thread's mark of this segment is visible once all have handed their last P on;
      // the next segment's come after all have passed here (its first S waits for all of Q).
      if (!warp_wait(&bars->p_full[~tiles & 1u], ((tiles - 1) >> 1) & 1u)) {
        ok = false;
        break;
      }
      // The next segment's queries may come.
      Segment following = s;
      if (w + s.step < end) {
        following = segment_at<BN>(a, line, prefix, w + s.step, end);
        fetch_q(following);
      }
      const bool dirty = *(volatile uint32_t*)&bars->dirty == seg + 1;
      const bool whole = s.t0 == 0 && s.t1 == s.tiles, live = R < NR;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (w == begin ? 0 : 1);
      const int head = s.h * a.G + R - i * a.G;
      const bool empty = live && l == 0.f && !sees_any(a, row, s.n, s.ctx);
      const float inv = 1.f / l;
      if (dirty) {  // column after column in TMEM: a value is the same for every lane of the warp
#pragma unroll 1
        for (int j = max(s.ctx & ~(BN - 1), s.t0 * BN); j < min(s.len, s.t1 * BN); ++j) {
          const int64_t off = paged_offset(a.c, a.b.table + (int64_t)s.b * a.b.table_stride, a.b.table_stride, j);
          if (off < 0) continue;
          const bool see = live && (j < s.ctx || sees_node(a, row, i, j - s.ctx));
          const T* src = (const T*)(a.c.v + off + (int64_t)s.h * a.c.head_bytes);
#pragma unroll 1
          for (int d = 0; d < D; ++d) {
            const float f = Elem<T>::get(src[d]);
            if (isfinite(f)) continue;
            uint32_t col;
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(col) : "r"(tO + lanes + d) : "memory");
            tc_wait_ld();
            col = __float_as_uint(__uint_as_float(col) + (see ? f : 0.f));
            asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(tO + lanes + d), "r"(col) : "memory");
            tc_wait_st();
          }
        }
      }
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        tc_ld32(tO + lanes + c, o);
        tc_wait_ld();
        // A lane holds a row, so its stores would scatter over 32 rows: the warp's rows pass through
        // shared memory and leave 128 bytes of a row at a time. Unit v of row r sits at v ^ (r & 7).
        uint8_t* turn = sm + C::kQ + warp * 4096;
        if (whole) {
          const uint32_t half = (c >> 5 & 1) * 4;  // 64 dims of T fill the 128 bytes
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = empty ? 0.f : o[k + q] * inv;
            store8((T*)(turn + lane * 128 + (((half + k / 8) ^ (lane & 7)) << 4)), f);
          }
          if (!half && c + 32 < DP) continue;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *(float4*)(turn + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
        __syncwarp();
        const int v = lane & 7;
#pragma unroll 4
        for (int k = 0; k < 8; ++k) {
          const int r = 4 * k + (lane >> 3), Rr = s.rt * BM + warp * 32 + r;
          const uint4 x = *(const uint4*)(turn + r * 128 + ((v ^ (r & 7)) << 4));
          if (Rr >= NR) continue;
          if (whole) {
            const int d = (c & ~63) + 8 * v, ir = (int)a.by_g.div((uint32_t)Rr);
            if (d < D)
              *(uint4*)((T*)a.out + ((int64_t)(s.row0 + ir) * a.nh + s.h * a.G + Rr - ir * a.G) * D + d) = x;
          } else {
            *(uint4*)(a.part + (slot * BM + warp * 32 + r) * DP + c + 4 * v) = x;
          }
        }
        __syncwarp();
      }
      if (live && whole && a.lse) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<T>(m, l);
      if (live && !whole) a.part_ml[slot * BM + tid] = make_float2(m, l);
      tc_fence_before();  // O may be overwritten after the next p_full
      ++seg;
      n0 += 2 * cnt;
      w += s.step;
      s = following;
    }
  }
  if (!ok && a.err) atomicOr(a.err, PAGED_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 6) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols));
  }
}

template <typename T, int DP>
static pp_status run_tc(const TreeArgs& a, const TreeMaps& m, cudaStream_t st) {
  using C = TcCfg<DP>;
  const int B = a.b.batch;
  const pp_status r = launch_tree<pp_tree_tc_kernel<T, DP>>(a, kTcThreads, C::smem(B), st, m);
  if (r != PP_OK || a.whole) return r;
  return launch_join<T, DP>(a, st);
}
template <typename T>
static pp_status run_tc_dim(const TreeArgs& a, const TreeMaps& m, int dp, cudaStream_t st) {
  if (dp == 64) return run_tc<T, 64>(a, m, st);
  if (dp == 128) return run_tc<T, 128>(a, m, st);
  return run_tc<T, 256>(a, m, st);
}
pp_status run_tree_tc(const TreeArgs& a, const TreeMaps& m, uint32_t dtype, int dp, cudaStream_t st) {
  return dtype == PP_BF16 ? run_tc_dim<__nv_bfloat16>(a, m, dp, st) : run_tc_dim<__half>(a, m, dp, st);
}

}  // namespace pp
