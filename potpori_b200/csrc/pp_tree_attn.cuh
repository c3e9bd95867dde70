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
// unit writes its rows; where a unit spans CTAs each writes a partial (the weights' base, their sum,
// unnormalised output) and a second kernel joins them in order (no atomics, so equal calls give
// equal bits).
// Lengths are read on the device, so a captured call follows new ones. What every call pays beside its
// tiles: 1 to 2 us from the launch to the cut, 2 to 4 until the first keys are there, 3 to 5 for the
// partials' way out and 3 to 8 for the join.
#pragma once
#include "pp_paged.cuh"

namespace pp {

// Keys of a tile, of the attention's kernels and of the join.
template <typename T>
constexpr int kTreeTile = sizeof(T) == 4 ? 32 : 64;
constexpr int kTreeMostRows = 1 << 20;  // of a sequence: times the group they stay below 2^31
// Of a page table: places are counted in 32 bits, a few tiles past a sequence's end among them.
constexpr uint64_t kTreeMostPositions = (1ull << 31) - 4096;

struct TreeArgs {
  PagedView c;  // the layer
  BatchView b;
  const void* q;
  void* out;
  float* lse;
  int64_t q_stride;  // elements
  const uint32_t* mask;
  int32_t mask_words, nh, G;
  FastDiv by_g, by_kv;  // by G, by the cached heads
  float scale;
  float* part;      // [2 * ctas][BM][DP] outputs
  float2* part_ml;  // [2 * ctas][BM] (base of the weights, sum)
  int32_t ctas;     // CTAs that the line of tiles is cut over
  int32_t bm;       // rows of a tile
  int32_t whole;    // units are never cut (short caches): no partials, no join
  uint32_t slack;   // see cut_line
  int32_t dev;
  uint32_t* err;
};

// A sequence whose rows do not fit the arrays or whose lengths do not fit its table is left out.
__device__ __forceinline__ bool bad_sequence(const TreeArgs& a, int first, int n, int len) {
  return n < 0 || n > kTreeMostRows || first < 0 || first > a.b.rows - n || len < n || (int64_t)len > (int64_t)a.b.table_stride * a.c.page.d;
}

// Sequences up to which a line may be put in order.
constexpr int kOrderMost = 64;
inline size_t prefix_bytes(int batch) { return 4 * ((size_t)batch + 1 + (batch <= kOrderMost ? batch : 0)); }

// The line of tiles, and how it is cut: CTA c takes the places [c per, (c + 1) per).
struct Line {
  uint32_t places, per;
  bool whole;  // a place is a unit, none is cut
  const uint32_t* order;  // the sequences by falling length; null: as they come
};
// prefix[b] = places before sequence b on the line; prefix[batch] = all. A CTA takes equal shares of
// the tiles, unless whole units load the fullest CTA with at most a quarter and `slack` tiles (or 6
// times the share) more: cutting units costs second segments and the join, and keeps every SM's CTAs in
// each other's way to the end. With `sort` whole units of long sequences come first where each unit has
// a CTA of its own, so that they start on empty SMs and the short ones fill up (16 ragged trees of 61
// nodes over 2048 to 4096 positions: 91.1 us against 92.7); `batch` words behind prefix then. By the
// whole CTA (NT threads); a tile has 1 << bm_log rows; scan: 3 NT / 32 words of shared memory.
template <int BN, int NT>
__device__ __forceinline__ Line cut_line(const TreeArgs& a, int bm_log, uint32_t* prefix, bool sort, uint32_t* scan,
                                         bool report) {
  constexpr int W = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.b.batch;
  uint32_t* order = prefix + B + 1;
  // Units of a sequence, and its tiles
  auto units_of = [&](int b, uint32_t& tiles, bool report) {
    const int first = a.b.cu_rows[b], n = a.b.cu_rows[b + 1] - first, len = a.b.kv_len[b];
    tiles = 0;
    if (bad_sequence(a, first, n, len)) {
      if (report && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
      return 0u;
    }
    if (n == 0) return 0u;
    tiles = (len + BN - 1) / BN;
    return ((((uint32_t)n * a.G - 1) >> bm_log) + 1) * a.c.n_kv;
  };
  auto cut = [&](uint32_t units, uint32_t tiles, uint32_t longest) {
    Line l = {};
    l.whole = true;
    l.places = units;
    l.per = max((units + a.ctas - 1) / a.ctas, 1u);
    if (!a.whole) {
      const uint32_t per = max((tiles + a.ctas - 1) / a.ctas, 1u);
      const uint64_t slack = a.slack < 6ull * per ? a.slack : 6ull * per;
      if ((uint64_t)l.per * longest > (uint64_t)per + per / 4 + slack) l = Line{tiles, per, false, nullptr};
    }
    return l;
  };
  if (B == 1) {  // the usual decode: no scan
    uint32_t tiles;
    const uint32_t units = units_of(0, tiles, report && tid == 0);
    const Line l = cut(units, units * tiles, tiles);
    if (tid == 0) {
      prefix[0] = 0;
      prefix[1] = l.places;
    }
    __syncthreads();
    return l;
  }
  const int each = (B + NT - 1) / NT, b0 = min(B, tid * each), b1 = min(B, b0 + each);
  uint32_t units = 0, tiles = 0, longest = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    uint32_t t;
    const uint32_t u = units_of(b, t, report);
    units += u;
    tiles += u * t;
    longest = max(longest, t);
  }
  const uint32_t mine = longest;  // of a lone sequence: its tiles
  uint32_t iu = units, it = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t vu = __shfl_up_sync(0xffffffffu, iu, o), vt = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) iu += vu, it += vt;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) scan[warp] = iu, scan[W + warp] = it, scan[2 * W + warp] = longest;
  __syncthreads();
  uint32_t bu = iu - units, bt = it - tiles, su = 0, st = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == warp) bu += su, bt += st;
    su += scan[w], st += scan[W + w];
    longest = max(longest, scan[2 * W + w]);
  }
  Line l = cut(su, st, longest);
  if (sort && l.whole && !a.whole && l.per == 1 && B <= kOrderMost) {  // a thread has one sequence
    const uint32_t own = mine;
    if (tid < B) prefix[tid] = own, order[tid] = units;
    __syncthreads();
    uint32_t rank = 0, before = 0;
#pragma unroll 4
    for (int b = 0; b < B; ++b) {
      const uint32_t t = prefix[b];
      if (t > own || (t == own && b < tid)) ++rank, before += order[b];
    }
    __syncthreads();
    if (tid < B) prefix[rank] = before, order[rank] = (uint32_t)tid;
    if (tid == 0) prefix[B] = l.places;
    __syncthreads();
    l.order = order;
    return l;
  }
  uint32_t at = l.whole ? bu : bt;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    uint32_t t;
    const uint32_t u = units_of(b, t, false);
    prefix[b] = at;
    at += l.whole ? u : u * t;
  }
  if (tid == 0) prefix[B] = l.places;
  __syncthreads();
  return l;
}

// The tiles of one CTA inside one unit.
struct Segment {
  int32_t b, h, rt;           // unit
  int32_t t0, t1, tiles;      // key tiles [t0, t1) of `tiles`
  int32_t row0, n, len, ctx;  // first row of the sequence, nodes, positions, context positions
  uint32_t unit0;             // place of the unit's first tile on the line
  uint32_t step;              // places on the line that the segment takes
};
template <int BN>
__device__ __forceinline__ Segment segment_at(const TreeArgs& a, const Line& line, const uint32_t* prefix, uint32_t w,
                                              uint32_t end) {
  int lo = 0, hi = a.b.batch;  // last b with prefix[b] <= w: the one with tiles, as w < prefix[b + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= w) lo = mid;
    else hi = mid;
  }
  const uint32_t off = w - prefix[lo];
  if (line.order) lo = (int)line.order[lo];
  Segment s;
  s.b = lo;
  s.row0 = a.b.cu_rows[lo];
  s.n = a.b.cu_rows[lo + 1] - s.row0;
  s.len = a.b.kv_len[lo];
  s.ctx = s.len - s.n;
  s.tiles = (s.len + BN - 1) / BN;
  const uint32_t unit = line.whole ? off : off / (uint32_t)s.tiles;
  s.t0 = line.whole ? 0 : (int)(off - unit * s.tiles);
  s.rt = (int)a.by_kv.div(unit);
  s.h = (int)(unit - (uint32_t)s.rt * a.c.n_kv);
  s.t1 = line.whole ? s.tiles : (int)min((uint32_t)s.tiles, s.t0 + (end - w));
  s.unit0 = w - s.t0;
  s.step = line.whole ? 1 : s.t1 - s.t0;
  return s;
}
// Range of the line that CTA `cta` takes.
__device__ __forceinline__ void cta_range(const Line& line, uint32_t cta, uint32_t& begin, uint32_t& end) {
  begin = min((uint64_t)cta * line.per, (uint64_t)line.places);
  end = min(begin + line.per, line.places);
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

// Place in a ring of item after item: slot and the parity of its use (a division by a run-time slot
// count would cost more than a product's issue).
struct RingCursor {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int slots) {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// K and V of the layer as tensor maps (TMA), for 16-bit caches with pages of a multiple of 8
// positions (16 for the narrow kernel): 64-dim boxes of `box` rows of one page, 128-byte swizzled. Dimension 0 is the head's dim;
// heads, rows and pages are the dimensions at_head, at_row and at_page in order of their strides.
// A box at page n_pages is out of range and reads zeros: so do absent pages.
struct TreeMaps {
  CUtensorMap k, v;
  int32_t box;  // rows of a box; 0: no maps, 16-byte copies instead
  int32_t at_head, at_row, at_page;
};
__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, uint64_t* bar, const TreeMaps& m,
                                        int32_t x, int32_t head, int32_t row, int32_t page) {
  const int32_t c1 = m.at_head == 1 ? head : m.at_row == 1 ? row : page;
  const int32_t c2 = m.at_head == 2 ? head : m.at_row == 2 ? row : page;
  const int32_t c3 = m.at_head == 3 ? head : m.at_row == 3 ? row : page;
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
// Page and row in it of position idx (a multiple of the box's rows); page n_pages where there is
// nothing to read.
struct BoxPlace {
  int32_t page, row;
  __device__ __forceinline__ void look(const TreeArgs& a, const Segment& s, const int32_t* table, int idx, bool in_range) {
    page = a.c.n_pages;
    row = 0;
    if (!in_range || idx >= s.len) return;
    const uint32_t p = a.c.page.div((uint32_t)idx);
    const int32_t id = __ldg(table + p);  // p is within the table: idx < len
    if ((uint32_t)id < (uint32_t)a.c.n_pages) {
      page = id;
      row = idx - (int)(p * a.c.page.d);
    } else if (a.err) {
      atomicOr(a.err, PAGED_BAD_PAGE);
    }
  }
};

// Exponent all ones in either half of a register of T.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t v) {
  constexpr uint32_t E = __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  return ((v & E) == E ? 0xffffu : 0u) | ((v >> 16 & E) == E ? 0xffff0000u : 0u);
}
// True in one lane of the (converged) warp. Products and TMA copies take their operands from uniform
// registers: behind this branch, of values that the whole warp holds alike, the compiler needs no
// loop over the lanes to get them there.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// One arrival for the warp, after all its lanes' work.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// Bounded wait of a whole warp: the same answer in every lane, so that a warp leaves together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A warp's fetch of ROWS consecutive positions of a tile (one K and V row of the head each): where
// the rows are is looked up a tile ahead of the copies. With pages of a multiple of ROWS positions
// they are evenly spaced in one page and one lookup serves all; else lane l looks row l up.
template <int ROWS>
struct RowFetch {
  int64_t off;  // of row 0, or of row `lane`; -1: none
  int left;     // rows before the sequence's end
  __device__ __forceinline__ void look(const TreeArgs& a, const Segment& s, const int32_t* table, int idx0,
                                       bool in_range, int lane) {
    off = -1;
    left = in_range ? s.len - idx0 : 0;
    if (left <= 0) return;
    const bool even = a.c.page.d % ROWS == 0;
    const int idx = even ? idx0 : idx0 + lane % ROWS;
    if (idx >= s.len) return;
    off = paged_offset(a.c, table, a.b.table_stride, idx);
    if (off < 0) {
      if (a.err) atomicOr(a.err, PAGED_BAD_PAGE);
      return;
    }
    off += (int64_t)s.h * a.c.head_bytes;
  }
  // Offset of row l (warp-collective), -1 where there is nothing to read.
  __device__ __forceinline__ int64_t row(const TreeArgs& a, int l) const {
    if (a.c.page.d % ROWS == 0) return off >= 0 && l < left ? off + l * a.c.row_bytes : -1;
    return __shfl_sync(0xffffffffu, off, l);
  }
};

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
// Weights of the 16-bit types are P = 2^(x - m) for a base m, which is the maximum less kSoftShift and
// may lag behind it by kSoftLag before it is followed. Two F16 parts end at 2^-25 whatever their sum
// is: with P of 1 at the maximum, a weight below 2^-25 of it would be lost to the product though not to
// the sum (one key 17.5 nats above 131071 keys that make up the output: zeros, or 0.3 % off). With 2^13 and
// a lag of 2.75, P stays below F16's 65504 and a weight's error within 2^-38 of the maximum. BF16 has
// F32's range: no shift, and a lag of 8. (A small lag costs rescales: 16 ragged trees of 61 nodes over
// 2048 to 4096 positions take 95.0 us, with a lag of 8 93.5, over 512 to 1024 34.5 against 32.6.) A base is rounded up and a bound down, so that P keeps below the
// limit where scores are so large that they are sparse, too.
template <typename T>
constexpr float kSoftShift = __is_same(T, __half) ? 13.f : 0.f;
template <typename T>
constexpr float kSoftLag = __is_same(T, __half) ? 2.75f : 8.f;
template <typename T>
__device__ __forceinline__ float soft_base(float high) {
  return __is_same(T, __half) ? __fadd_ru(high, -kSoftShift<T>) : high;
}
// Whether a base of m no longer serves scores of up to high.
template <typename T>
__device__ __forceinline__ bool soft_outgrown(float high, float m) {
  return high > __fadd_rd(m, kSoftShift<T> + kSoftLag<T>);
}
// Log of a sum l of weights of base m.
template <typename T>
__device__ __forceinline__ float soft_lse(float m, float l) {
  return (sizeof(T) == 4 ? m : m * 0.69314718055994531f) + logf(l);
}

// Adds the non-finite values of V at the positions [j0, j1), the tree's and those of the context that
// share its first tile, to the outputs that see them: the kernels' products saw zeros in their place.
// o(r, d) is the output of vector r of the tile, dim d; its weight there must be positive, so that the
// sum is what the value is. By NT threads over (vector, dim); kept small, it hardly ever runs.
template <typename T, typename O>
__device__ __forceinline__ void add_nonfinite(const TreeArgs& a, const Segment& s, int rows, int j0, int j1, int tid, int nt, O o) {
  const int D = a.c.head_dim;
  const int32_t* table = a.b.table + (int64_t)s.b * a.b.table_stride;
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    const int64_t off = paged_offset(a.c, table, a.b.table_stride, j);
    if (off < 0) continue;
    const T* v = (const T*)(a.c.v + off + (int64_t)s.h * a.c.head_bytes);
#pragma unroll 1
    for (int e = tid; e < rows * D; e += nt) {
      const int r = e / D, d = e - r * D;
      const float f = Elem<T>::get(v[d]);
      if (isfinite(f)) continue;
      const int i = (int)a.by_g.div((uint32_t)(s.rt * a.bm + r));
      if (j < s.ctx || sees_node(a, s.row0 + i, i, j - s.ctx)) o(r, d) += f;
    }
  }
}

// Joins the partials of the units that the line was cut in. A CTA of the attention whose first
// segment ends a unit that it did not begin stands for that unit. Items are spread over a grid of any
// size; 16 lanes take a row, DP / 16 dims each: of a unit with few partials an item is 8 rows, of one
// with many a row, its partials dealt to the 8 groups. What the units are follows from the lengths
// alone, so it is found while the attention's last CTAs still run: only the partials are waited for,
// and read once, with a running maximum (with descriptors left by the attention and a pass for the
// maximum first, the 37 partials of a tree of 24 over 131072 positions took 12 us behind the last CTA,
// now 3 to 7; they are 20 MB from L2).
constexpr int kJoinMany = 8;
struct JoinUnit {
  int32_t parts, rows;  // partials (0: no unit), rows of the tile
  int32_t first_slot, cta;  // slot of the first partial; the others are 2 * (cta + p)
  int32_t row0, vec0, head0, n, ctx;  // first array row, vector of row 0, first head, nodes, context
};
template <int BN>
__device__ __forceinline__ JoinUnit join_unit(const TreeArgs& a, const Line& line, int bm_log, const uint32_t* prefix,
                                              uint32_t cta) {
  JoinUnit u = {};
  uint32_t begin, end;
  cta_range(line, cta, begin, end);
  if (line.whole || begin >= end) return u;
  const Segment s = segment_at<BN>(a, line, prefix, begin, end);
  if (s.t0 == 0 || s.t1 < s.tiles) return u;
  const uint32_t c0 = s.unit0 / line.per;
  u.parts = (int)(cta - c0) + 1;
  u.vec0 = s.rt << bm_log;
  u.rows = min(1 << bm_log, s.n * a.G - u.vec0);
  u.first_slot = (int)(c0 * line.per == s.unit0 ? 2 * c0 : 2 * c0 + 1);
  u.cta = (int)c0;
  u.row0 = s.row0;
  u.head0 = s.h * a.G;
  u.n = s.n;
  u.ctx = s.ctx;
  return u;
}

template <typename T, int DP>
__global__ void __launch_bounds__(128) pp_tree_join_kernel(const TreeArgs a) {
  constexpr int V = DP / 16, BN = kTreeTile<T>;
  extern __shared__ uint32_t s_items[];  // [ctas + 1] items before each CTA's unit, then [batch + 1]
  __shared__ uint32_t scan[12];
  __shared__ float s_acc[8][DP];
  __shared__ float2 s_ml[8];
  uint32_t* prefix = s_items + a.ctas + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = tid >> 4, l16 = tid & 15;
  const int each = (a.ctas + 127) / 128, c0 = min(a.ctas, tid * each), c1 = min(a.ctas, c0 + each);
  const int bm_log = 31 - __clz(a.bm);
  const Line line = cut_line<BN, 128>(a, bm_log, prefix, false, scan, false);
  {
    uint32_t sum = 0;
#pragma unroll 1
    for (int c = c0; c < c1; ++c) {
      const JoinUnit u = join_unit<BN>(a, line, bm_log, prefix, c);
      s_items[c] = sum;
      if (u.parts > 0) sum += u.parts > kJoinMany ? u.rows : (u.rows + 7) / 8;
    }
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    uint32_t before = inc - sum;
#pragma unroll 1
    for (int w = 0; w < warp; ++w) before += scan[w];
#pragma unroll 1
    for (int c = c0; c < c1; ++c) s_items[c] += before;
    if (tid == 127) s_items[a.ctas] = before + sum;
    __syncthreads();
  }
  const uint32_t total = s_items[a.ctas];
  bool waited = false;
#pragma unroll 1
  for (uint32_t item = blockIdx.x;; item += gridDim.x) {
    JoinUnit u = {};
    int at = 0;
    if (item < total) {
      int lo = 0, hi = a.ctas;
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_items[mid] <= item) lo = mid;
        else hi = mid;
      }
      u = join_unit<BN>(a, line, bm_log, prefix, lo);
      at = (int)(item - s_items[lo]);
    }
    if (!waited) pdl_wait();  // by every CTA: the stream goes on when all of this grid's have ended
    waited = true;
    if (item >= total) break;
    const bool many = u.parts > kJoinMany;
    const int r = many ? at : at * 8 + grp;
    const bool live = r < u.rows;
    const int parts = live ? u.parts : 0;
    float acc[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < V; ++d) acc[d] = 0.f;
    auto add = [&](float pm, float pl, const float* x) {  // one more partial, in order
      const float mx = fmaxf(m, pm), base = mx == -INFINITY ? 0.f : mx;
      const float fa = soft_exp<T>(m - base), fp = soft_exp<T>(pm - base);
      m = mx;
      l = l * fa + pl * fp;
#pragma unroll
      for (int d = 0; d < V; ++d) acc[d] = acc[d] * fa + x[d] * fp;
    };
#pragma unroll 4
    for (int p = many ? grp : 0; p < parts; p += many ? 8 : 1) {
      const int64_t slot = (int64_t)(p == 0 ? u.first_slot : 2 * (u.cta + p)) * a.bm + r;
      const float2 ml = __ldcg(&a.part_ml[slot]);
      const float* o = a.part + slot * DP + V * l16;
      float x[V];
#pragma unroll
      for (int d = 0; d < V; d += 4) {
        const float4 v = __ldcg((const float4*)(o + d));
        x[d] = v.x;
        x[d + 1] = v.y;
        x[d + 2] = v.z;
        x[d + 3] = v.w;
      }
      add(ml.x, ml.y, x);
    }
    if (many) {  // the groups' shares, in order
#pragma unroll
      for (int d = 0; d < V; ++d) s_acc[grp][V * l16 + d] = acc[d];
      if (l16 == 0) s_ml[grp] = make_float2(m, l);
      __syncthreads();
      if (grp == 0) {
#pragma unroll 1
        for (int g = 1; g < 8; ++g) add(s_ml[g].x, s_ml[g].y, &s_acc[g][V * l16]);
      }
      __syncthreads();
    }
    if (!live || (many && grp > 0)) continue;
    const int R = u.vec0 + r, i = (int)a.by_g.div((uint32_t)R), row = u.row0 + i, head = u.head0 + (R - i * a.G);
    const bool empty = l == 0.f && !sees_any(a, row, u.n, u.ctx);
    const float inv = 1.f / l;
#pragma unroll
    for (int d = 0; d < V; ++d) acc[d] = empty ? 0.f : acc[d] * inv;
    T* out = (T*)a.out + ((int64_t)row * a.nh + head) * a.c.head_dim + V * l16;
    if constexpr (V == 4) {
      if (4 * l16 < a.c.head_dim) store_n<T, 4>(out, acc);
    } else {
#pragma unroll
      for (int d = 0; d < V; d += 8)
        if (V * l16 + d < a.c.head_dim) store_n<T, 8>(out + d, acc + d);
    }
    if (a.lse && l16 == 0) a.lse[(int64_t)row * a.nh + head] = empty ? -INFINITY : soft_lse<T>(m, l);
  }
}

}  // namespace pp
