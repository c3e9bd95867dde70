// Row movers of the paged K/V cache: appending rotated rows (pp_paged_append), committing the
// accepted path of a draft tree (pp_tree_commit) and reordering the states of beams
// (pp_beam_reorder). All are bound by the bytes they move; the small calls by the chain of
// dependent loads from a row to its page.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_paged.cuh"

using namespace pp;

namespace pp {

// ---- append -------------------------------------------------------------------------------
struct AppendArgs {
  PagedView c;
  BatchView b;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  int64_t q_stride, k_stride, v_stride;  // elements
  const int32_t* positions;
  const double* inv_freq;
  const float* q_norm;
  const float* k_norm;
  float eps;
  int32_t nh, rot, interleaved;
  int32_t tph;  // lanes per head: 8, 16 or 32, 8 dims each
  uint32_t* err;
};

constexpr int kAppendThreads = 128, kAppendAnyThreads = 256;

// cos and sin of position * inv_freq. The angle in turns is formed in 64 bits and reduced to
// (-0.5, 0.5] before it is rounded, so the error stays near 2^-24 of a turn up to positions of
// 2^31 (in 32 bits position 131072 would be off by 2^-7 radians already).
__device__ __forceinline__ float2 rotation(int32_t pos, double inv_freq) {
  double turns = (double)pos * inv_freq * 0.15915494309189533577;
  turns -= rint(turns);
  float s, c;
  sincospif((float)(2.0 * turns), &s, &c);
  return make_float2(c, s);
}

// (a, b) turned by the angle of r = (cos, sin).
__device__ __forceinline__ void turn(float& a, float& b, float2 r) {
  const float a0 = a, b0 = b;
  a = a0 * r.x - b0 * r.y;
  b = b0 * r.x + a0 * r.y;
}

// Where row t goes: its sequence, cache index and page, by a warp. `report`: this warp marks a bad one.
// Rows of nobody, and of a sequence whose rows do not fit the arrays or whose length does not fit its
// table, are left out whole, q too.
struct RowPlace {
  int64_t offset;  // -1: no valid page
  int32_t live, pos;
};
__device__ __forceinline__ RowPlace place_row(const AppendArgs& a, int t, int lane, bool report) {
  const int given = a.positions ? a.positions[t] : 0;
  const int b = find_sequence(a.b.cu_rows, a.b.batch, t, lane);
  RowPlace r = {-1, 0, 0};
  if (b >= 0) {
    const int first = a.b.cu_rows[b], n = a.b.cu_rows[b + 1] - first, len = a.b.kv_len[b];
    const int64_t room = (int64_t)a.b.table_stride * a.c.page.d;
    if (first >= 0 && n > t - first && n <= a.b.rows - first && len >= n && len <= room) {
      const int index = len - n + (t - first);
      r.live = 1;
      r.pos = a.positions ? given : index;
      r.offset = paged_offset(a.c, a.b.table + (int64_t)b * a.b.table_stride, a.b.table_stride, index);
    }
    if (r.offset < 0 && report && lane == 0 && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
  }
  return r;
}

// A CTA of one to four warps per row and share of its heads: one warp finds the row's place, all form
// its rotary_dim / 2 angles once. tph lanes take a head, 8 dims each, as two runs of 4: of the
// rotated dims lane j holds both halves' run j, so that a pair never leaves its lane, of the others 8
// in a row (interleaved pairs: all dims 8 in a row). A lane's first head is on its way before the
// row's place is known, the next one while this one leaves; more of them in flight, or more CTAs on an
// SM, gained nothing (6400 rows of 48 heads: 48.8 us at 64 registers, 49.5 with three heads ahead, 50.2
// with two, 53.8 at 32 registers: 4.8 TB/s of the 6.5 that a copy reaches).
template <typename TI, typename TC>
__global__ void __launch_bounds__(kAppendThreads, 8) pp_append_kernel(const AppendArgs a) {
  __shared__ float2 cs[128];
  __shared__ RowPlace s_place;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  const int D = a.c.head_dim, K = a.c.n_kv, heads = a.nh + 2 * K;
  const int per = 32 / a.tph, j = lane % a.tph;
  const bool dims = 8 * j < D, turns = 8 * j < a.rot;
  const int d0 = turns && !a.interleaved ? 4 * j : 8 * j;
  const int d1 = turns && !a.interleaved ? a.rot / 2 + 4 * j : 8 * j + 4;
  const int share = blockIdx.y * (blockDim.x >> 5) + warp, step = per * gridDim.y * (blockDim.x >> 5);
  int slot = share * per + lane / a.tph;
  const float inv_dim = 1.f / (float)D;
  float x[8];
  auto fetch = [&](int h) {
    if (h >= heads || !dims) return;
    const TI* src;
    if (h < a.nh) src = (const TI*)a.q + (int64_t)t * a.q_stride + h * D;
    else if (h < a.nh + K) src = (const TI*)a.k + (int64_t)t * a.k_stride + (h - a.nh) * D;
    else src = (const TI*)a.v + (int64_t)t * a.v_stride + (h - a.nh - K) * D;
    load_n<TI, 4>(src + d0, x);
    load_n<TI, 4>(src + d1, x + 4);
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  fetch(slot);
  if (warp == 0) {
    const RowPlace p = place_row(a, t, lane, blockIdx.y == 0);
    if (lane == 0) s_place = p;
  }
  __syncthreads();
  const RowPlace place = s_place;
  if (!place.live) return;
  for (int i = threadIdx.x; i < a.rot / 2; i += blockDim.x) cs[i] = rotation(place.pos, a.inv_freq[i]);
  __syncthreads();
  float2 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = turns ? cs[4 * j + i] : make_float2(1.f, 0.f);

  const float* held = nullptr;  // the norm's weights in wv
  float wv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wv[i] = 0.f;

#pragma unroll 1
  for (int s0 = share * per; s0 < heads; s0 += step, slot += step) {  // s0: the warp's first, so it stays together
    const bool live = slot < heads && dims, isq = slot < a.nh, isv = slot >= a.nh + K;
    const float* w = isq ? a.q_norm : isv ? nullptr : a.k_norm;
    if (a.q_norm || a.k_norm) {  // per-head RMSNorm; the sum of squares over the head's lanes
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      for (int o = a.tph >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && w) {
        if (w != held) {
          held = w;
          load_n<float, 4>(w + d0, wv);
          load_n<float, 4>(w + d1, wv + 4);
        }
        const float inv = rsqrtf(ss * inv_dim + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wv[i];
      }
    }
    if (turns && !isv) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(x[2 * i], x[2 * i + 1], r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(x[i], x[4 + i], r[i]);
      }
    }
    if (live && (isq || place.offset >= 0)) {
      const int hk = isv ? slot - a.nh - K : slot - a.nh;
      TC* dst = isq ? (TC*)a.q_out + ((int64_t)t * a.nh + slot) * D
                    : (TC*)((isv ? a.c.v : a.c.k) + place.offset + (int64_t)hk * a.c.head_bytes);
      store_n<TC, 4>(dst + d0, x);
      store_n<TC, 4>(dst + d1, x + 4);
    }
    fetch(slot + step);
  }
}

// The same for rows whose pointers, strides or rotation do not fit 8-element units: a warp per
// head, lane l the dims l, l + 32, ...
template <typename TI, typename TC>
__global__ void __launch_bounds__(kAppendAnyThreads) pp_append_any_kernel(const AppendArgs a) {
  __shared__ float2 cs[128];
  __shared__ RowPlace place;
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = a.c.head_dim, K = a.c.n_kv, heads = a.nh + 2 * K;
  if (warp == 0) {
    const RowPlace p = place_row(a, t, lane, blockIdx.y == 0);
    if (lane == 0) place = p;
  }
  __syncthreads();
  if (!place.live) return;
  if (a.inv_freq && tid < a.rot / 2) cs[tid] = rotation(place.pos, a.inv_freq[tid]);
  __syncthreads();
  for (int slot = blockIdx.y * 8 + warp; slot < heads; slot += 8 * gridDim.y) {
    const bool isq = slot < a.nh, isv = slot >= a.nh + K;
    const TI* src = isq ? (const TI*)a.q + (int64_t)t * a.q_stride + (int64_t)slot * D
                  : isv ? (const TI*)a.v + (int64_t)t * a.v_stride + (int64_t)(slot - a.nh - K) * D
                        : (const TI*)a.k + (int64_t)t * a.k_stride + (int64_t)(slot - a.nh) * D;
    const float* w = isv ? nullptr : isq ? a.q_norm : a.k_norm;
    const int rot = a.inv_freq && !isv ? a.rot : 0;
    float x[8], p[8];  // a dim and its rotation partner
    float ss = 0.f;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const int e = lane + 32 * m;
      const int pe = e >= rot ? e : a.interleaved ? e ^ 1 : e < rot / 2 ? e + rot / 2 : e - rot / 2;
      x[m] = e < D ? Elem<TI>::get(src[e]) : 0.f;
      p[m] = e < rot ? Elem<TI>::get(src[pe]) : 0.f;
      ss += x[m] * x[m];
    }
    const float rms = sqrtf(warp_sum(ss) / (float)D + a.eps);  // also: every load before a store
    int64_t off = 0;
    uint8_t* row = nullptr;
    if (!isq) {
      if (place.offset < 0) continue;
      off = place.offset + (int64_t)(isv ? slot - a.nh - K : slot - a.nh) * a.c.head_bytes;
      row = (isv ? a.c.v : a.c.k) + off;
    } else {
      row = (uint8_t*)((TC*)a.q_out + ((int64_t)t * a.nh + slot) * D);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const int e = lane + 32 * m;
      if (e >= D) continue;
      float y = x[m];
      if (w) y = y / rms * w[e];
      if (e < rot) {
        const bool head_of_pair = a.interleaved ? !(e & 1) : e < rot / 2;
        const int pe = a.interleaved ? e ^ 1 : head_of_pair ? e + rot / 2 : e - rot / 2;
        const float2 r = cs[a.interleaved ? e / 2 : head_of_pair ? e : pe];
        float o = p[m];
        if (w) o = o / rms * w[pe];
        y = head_of_pair ? y * r.x - o * r.y : y * r.x + o * r.y;
      }
      ((TC*)row)[e] = Elem<TC>::put(y);
    }
  }
}

// ---- commit -------------------------------------------------------------------------------
struct CommitArgs {
  PagedView c;  // layer 0
  BatchView b;
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* picks;
  int32_t* path;
  int32_t* accepted;
  int32_t* correction;
  int32_t* new_len;
  int32_t path_stride, max_rows, units;  // units: 16-byte units of a row of one head
  uint32_t* err;
};
constexpr int kCommitThreads = 128;
constexpr int kCommitMaxRows = 1024;
constexpr int kCommitBatch = 8;  // rows a thread holds between its loads and its stores

// Grid (slices of the 2 * layers planes, batch). Every CTA walks its sequence's tree itself (a
// few hundred cycles) and moves the path's rows in its planes. A thread keeps one 16-byte unit of
// a row and moves it down row after row: the rows before the first gap stay, and as path[d] >= d
// and both ascend, a row is written only after every row that it covers has been read. 64 trees,
// 36 layers, 61 MB: 22 us over changing caches, 2.8 TB/s (17 to 19 over the same one again and again),
// for every plane's CTA walks the tree again and nine of them fill an SM; one tree of 8, 28 layers: 3.7
// to 4.3 us, the chain from the tokens to the pages.
__global__ void __launch_bounds__(kCommitThreads) pp_tree_commit_kernel(const CommitArgs a) {
  __shared__ int32_t follow[kCommitMaxRows];  // the node that continues a path ending here
  __shared__ int32_t path[kCommitMaxRows];
  __shared__ int64_t from[kCommitMaxRows], to[kCommitMaxRows];
  __shared__ int32_t s_count;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int first = a.b.cu_rows[b], n = a.b.cu_rows[b + 1] - first, len = a.b.kv_len[b];
  const bool lead = blockIdx.x == 0;
  const bool bad = n < 0 || n > a.max_rows || len < n || first < 0 || first > a.b.rows - n ||
                   (int64_t)len > (int64_t)a.b.table_stride * a.c.page.d;
  if (n <= 0 || bad) {
    if (lead) {
      for (int d = tid; d < a.path_stride; d += kCommitThreads) a.path[(int64_t)b * a.path_stride + d] = -1;
      if (tid == 0) {
        a.accepted[b] = 0;
        a.correction[b] = -1;
        a.new_len[b] = len;
        if (bad && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
      }
    }
    return;
  }
  for (int i = tid; i < n; i += kCommitThreads) follow[i] = n;
  __syncthreads();
  for (int i = 1 + tid; i < n; i += kCommitThreads) {
    const int p = a.parents[first + i];
    if (p >= 0 && p < i && a.tokens[first + i] == a.picks[first + p]) atomicMin(&follow[p], i);
  }
  __syncthreads();
  if (tid == 0) {
    int count = 0;
    for (int node = 0; node < n; node = follow[node]) path[count++] = node;
    s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  const int32_t* table = a.b.table + (int64_t)b * a.b.table_stride;
  for (int d = tid; d < count; d += kCommitThreads) {
    const int base = len - n;
    const bool moves = path[d] != d;
    from[d] = moves ? paged_offset(a.c, table, a.b.table_stride, base + path[d]) : -1;
    to[d] = moves ? paged_offset(a.c, table, a.b.table_stride, base + d) : -1;
    if (moves && (from[d] < 0 || to[d] < 0)) {
      from[d] = to[d] = -1;
      if (lead && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
    }
  }
  if (lead) {
    for (int d = tid; d < a.path_stride; d += kCommitThreads)
      a.path[(int64_t)b * a.path_stride + d] = d < count ? path[d] : -1;
    if (tid == 0) {
      a.accepted[b] = count - 1;
      a.correction[b] = a.picks[first + path[count - 1]];
      a.new_len[b] = len - n + count;
    }
  }
  __syncthreads();
  int gap = 0;  // the first row that moves
  while (gap < count && path[gap] == gap) ++gap;
  if (gap == count) return;
  const int per_row = a.c.n_kv * a.units;
  for (int plane = blockIdx.x; plane < 2 * a.c.layers; plane += gridDim.x) {
    uint8_t* base = (plane & 1 ? a.c.v : a.c.k) + (int64_t)(plane >> 1) * a.c.layer_bytes;
    for (int u = tid; u < per_row; u += kCommitThreads) {
      const int h = u / a.units;
      uint8_t* col = base + (int64_t)h * a.c.head_bytes + (int64_t)(u - h * a.units) * 16;
      for (int d0 = gap; d0 < count; d0 += kCommitBatch) {
        uint4 hold[kCommitBatch];
#pragma unroll
        for (int i = 0; i < kCommitBatch; ++i)
          if (d0 + i < count && from[d0 + i] >= 0) hold[i] = *(const uint4*)(col + from[d0 + i]);
#pragma unroll
        for (int i = 0; i < kCommitBatch; ++i)
          if (d0 + i < count && from[d0 + i] >= 0) *(uint4*)(col + to[d0 + i]) = hold[i];
      }
    }
  }
}

// ---- beam reorder -------------------------------------------------------------------------
struct ReorderArgs {
  PagedView c;  // layer 0
  const int32_t* table;
  const int32_t* len;
  const int32_t* beams;
  const int32_t* spare;
  int32_t* new_table;
  int32_t* new_len;
  int32_t* taken;
  int32_t old_beams, new_beams, stride, units;
  uint32_t* err;
};
constexpr int kReorderThreads = 128;
constexpr int kReorderBatch = 4;  // units a lane holds between its loads and its stores

// Grid (slices of the 2 * layers planes, new beams, groups). Only beams that take their spare
// page copy: lanes over the 16-byte units of a row, warps over the rows, four loads before
// their stores. 32 x 8 beams, 36 layers: 73 to 76 us for 400 to 450 MB read and written, 5.5 to 5.9 TB/s;
// 4 beams, 28 layers: 3.9 us.
__global__ void __launch_bounds__(kReorderThreads) pp_beam_reorder_kernel(const ReorderArgs a) {
  const int j = blockIdx.y, g = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t* mine = a.beams + (int64_t)g * a.new_beams;
  const int64_t out = (int64_t)g * a.new_beams + j;
  const int p = mine[j];
  const bool lead = blockIdx.x == 0, known = p >= 0 && p < a.old_beams;
  const int64_t src = (int64_t)g * a.old_beams + (known ? p : 0);
  const int len = known ? a.len[src] : 0;
  bool elder = false;  // an earlier child of the same beam
  for (int i = tid; i < j; i += kReorderThreads) elder |= mine[i] == p;
  const bool again = __syncthreads_or(elder);
  bool bad = (!known && p != -1) || len < 0 || (int64_t)len > (int64_t)a.stride * a.c.page.d;
  const int last = bad ? 0 : (int)a.c.page.div((uint32_t)len);
  const int part = bad ? 0 : len - last * (int)a.c.page.d;
  const bool take = known && !bad && again && part > 0;
  int from = -1, to = -1;
  if (take) {
    from = a.table[src * a.stride + last];
    to = a.spare[out];
    if ((uint32_t)from >= (uint32_t)a.c.n_pages || (uint32_t)to >= (uint32_t)a.c.n_pages) {
      bad = true;
      from = -1;
    }
  }
  if (lead) {
    for (int e = tid; e < a.stride; e += kReorderThreads)
      a.new_table[out * a.stride + e] =
          !known ? -1 : take && e == last ? to : a.table[src * a.stride + e];
    if (tid == 0) {
      a.new_len[out] = len;
      a.taken[out] = take ? 1 : 0;
      if (bad && a.err) atomicOr(a.err, PAGED_BAD_PAGE);
    }
  }
  if (from < 0) return;
  const int per_row = a.c.n_kv * a.units;
  for (int plane = blockIdx.x; plane < 2 * a.c.layers; plane += gridDim.x) {
    uint8_t* base = (plane & 1 ? a.c.v : a.c.k) + (int64_t)(plane >> 1) * a.c.layer_bytes;
    const uint8_t* sp = base + (int64_t)from * a.c.page_bytes;
    uint8_t* dp = base + (int64_t)to * a.c.page_bytes;
    for (int u = lane; u < per_row; u += 32) {
      const int h = u / a.units;
      const int64_t col = (int64_t)h * a.c.head_bytes + (int64_t)(u - h * a.units) * 16;
      for (int r0 = warp; r0 < part; r0 += kReorderBatch * kReorderThreads / 32) {
        uint4 hold[kReorderBatch];
#pragma unroll
        for (int i = 0; i < kReorderBatch; ++i)
          if (r0 + i * kReorderThreads / 32 < part)
            hold[i] = *(const uint4*)(sp + col + (int64_t)(r0 + i * kReorderThreads / 32) * a.c.row_bytes);
#pragma unroll
        for (int i = 0; i < kReorderBatch; ++i)
          if (r0 + i * kReorderThreads / 32 < part)
            *(uint4*)(dp + col + (int64_t)(r0 + i * kReorderThreads / 32) * a.c.row_bytes) = hold[i];
      }
    }
  }
}

template <typename TI, typename TC>
void launch_append(const AppendArgs& a, bool vec, int rows, cudaStream_t st, int sms) {
  const int heads = a.nh + 2 * a.c.n_kv;
  if (vec) {
    // Up to four warps a row, with equal numbers of passes. Few rows: over several CTAs, a pass a warp at
    // the least, as long as the warps do not pass eight an SM.
    const int per = 32 / a.tph, passes = (heads + per - 1) / per;
    const int rounds = (passes + 3) / 4, warps = (passes + rounds - 1) / rounds;
    int y = rounds;
    while (y > 1 && (int64_t)rows * y * warps > 8 * (int64_t)sms) y = (y + 1) / 2;
    pp_append_kernel<TI, TC><<<dim3(rows, y), 32 * warps, 0, st>>>(a);
    return;
  }
  int y = (heads + 7) / 8;
  while (y > 1 && (int64_t)rows * y > 2 * (int64_t)sms) --y;
  pp_append_any_kernel<TI, TC><<<dim3(rows, y), kAppendAnyThreads, 0, st>>>(a);
}
template <typename TI>
void launch_append_to(const AppendArgs& a, uint32_t cache, bool vec, int rows, cudaStream_t st,
                      int sms) {
  if (cache == PP_F32) launch_append<TI, float>(a, vec, rows, st, sms);
  else if (cache == PP_BF16) launch_append<TI, __nv_bfloat16>(a, vec, rows, st, sms);
  else launch_append<TI, __half>(a, vec, rows, st, sms);
}

}  // namespace pp

extern "C" pp_status pp_paged_append(const pp_paged_cache* cache, const pp_paged_batch* batch,
                                     const pp_append_rows* r, uint32_t* err, void* stream) {
  if (const char* m = cache_problem(cache)) return paged_fail(PP_E_INVALID, m);
  if (const char* m = batch_problem(batch)) return paged_fail(PP_E_INVALID, m);
  if (!r || !r->k || !r->v) return paged_fail(PP_E_INVALID, "null rows");
  if (r->dtype != PP_F32 && r->dtype != PP_BF16 && r->dtype != PP_F16)
    return paged_fail(PP_E_INVALID, "the rows' dtype must be PP_F32, PP_BF16 or PP_F16");
  if ((r->q != nullptr) != (r->q_out != nullptr))
    return paged_fail(PP_E_INVALID, "q and q_out come together");
  if (r->q && (r->n_heads == 0 || r->n_heads > 4096))
    return paged_fail(PP_E_INVALID, "n_heads must be 1..4096 with q");
  if (r->layer >= cache->layers) return paged_fail(PP_E_INVALID, "layer outside the cache");
  const int64_t D = cache->head_dim, K = cache->n_kv_heads;
  const int nh = r->q ? (int)r->n_heads : 0;
  if (r->inv_freq && (r->rotary_dim == 0 || r->rotary_dim % 2 || r->rotary_dim > D))
    return paged_fail(PP_E_INVALID, "rotary_dim must be even and within head_dim");
  if (batch->rows > 1 && (r->k_stride < K * D || r->v_stride < K * D || (nh && r->q_stride < nh * D)))
    return paged_fail(PP_E_INVALID, "row strides shorter than the rows");
  const int e = dtype_bytes(r->dtype);
  const uintptr_t natural = (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->q;
  if (natural % e || (uintptr_t)r->q_out % dtype_bytes(cache->dtype))
    return paged_fail(PP_E_INVALID, "rows must be aligned to their element");
  if (r->q_out == r->q && r->q && (r->dtype != cache->dtype || (batch->rows > 1 && r->q_stride != nh * D)))
    return paged_fail(PP_E_INVALID, "q_out may be q only with equal types and adjacent rows");
  if (r->q_out && (r->q_out == r->k || r->q_out == r->v)) return paged_fail(PP_E_INVALID, "q_out must not be k or v");
  if (batch->rows == 0) return PP_OK;
  DeviceScope dev(cache->cuda_device);
  const int sms = dev.ok ? sm_count(cache->cuda_device) : 0;
  if (!sms) return paged_fail(PP_E_CUDA, "cannot use the cache's device");
  AppendArgs a = {};
  a.c = paged_view(*cache, r->layer);
  a.b = batch_view(*batch);
  a.q = r->q;
  a.k = r->k;
  a.v = r->v;
  a.q_out = r->q_out;
  a.q_stride = r->q_stride;
  a.k_stride = r->k_stride;
  a.v_stride = r->v_stride;
  a.positions = r->positions;
  a.inv_freq = r->inv_freq;
  a.q_norm = r->q_norm;
  a.k_norm = r->k_norm;
  a.eps = r->eps;
  a.nh = nh;
  a.rot = r->inv_freq ? (int)r->rotary_dim : 0;
  a.interleaved = r->interleaved != 0;
  a.tph = D <= 64 ? 8 : D <= 128 ? 16 : 32;
  a.err = err;
  const int64_t unit = 16 / e;
  const bool vec = (natural | (uintptr_t)r->q_out) % 16 == 0 && r->k_stride % unit == 0 &&
                   r->v_stride % unit == 0 && (!nh || r->q_stride % unit == 0) &&
                   a.rot % 8 == 0 &&
                   ((uintptr_t)r->q_norm | (uintptr_t)r->k_norm) % 16 == 0;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rows = (int)batch->rows;
  if (r->dtype == PP_F32) launch_append_to<float>(a, cache->dtype, vec, rows, st, sms);
  else if (r->dtype == PP_BF16) launch_append_to<__nv_bfloat16>(a, cache->dtype, vec, rows, st, sms);
  else launch_append_to<__half>(a, cache->dtype, vec, rows, st, sms);
  return launch_status("pp_paged_append");
}

extern "C" pp_status pp_tree_commit(const pp_paged_cache* cache, const pp_paged_batch* batch,
                                    const int32_t* tokens, const int32_t* parents,
                                    const int32_t* picks, int32_t* path, uint32_t path_stride,
                                    int32_t* accepted, int32_t* correction, int32_t* new_len,
                                    uint32_t* err, void* stream) {
  if (const char* m = cache_problem(cache)) return paged_fail(PP_E_INVALID, m);
  if (const char* m = batch_problem(batch)) return paged_fail(PP_E_INVALID, m);
  if (!tokens || !parents || !picks || !path || !accepted || !correction || !new_len)
    return paged_fail(PP_E_INVALID, "null argument");
  if (batch->max_rows > (uint32_t)kCommitMaxRows)
    return paged_fail(PP_E_UNSUPPORTED, "trees of more than 1024 nodes");
  if (path_stride < batch->max_rows || path_stride == 0 || path_stride > (1u << 24))
    return paged_fail(PP_E_INVALID, "path_stride must be at least max_rows and 1");
  const int32_t* const inputs[] = {tokens, parents, picks, batch->kv_len, batch->cu_rows, batch->page_table};
  for (const int32_t* in : inputs)  // which every CTA of a sequence reads
    if (in == path || in == accepted || in == correction || in == new_len)
      return paged_fail(PP_E_INVALID, "outputs must not be inputs (tokens, parents, picks, kv_len, cu_rows, the table)");
  DeviceScope dev(cache->cuda_device);
  const int sms = dev.ok ? sm_count(cache->cuda_device) : 0;
  if (!sms) return paged_fail(PP_E_CUDA, "cannot use the cache's device");
  CommitArgs a = {};
  a.c = paged_view(*cache, 0);
  a.b = batch_view(*batch);
  a.tokens = tokens;
  a.parents = parents;
  a.picks = picks;
  a.path = path;
  a.accepted = accepted;
  a.correction = correction;
  a.new_len = new_len;
  a.path_stride = (int32_t)path_stride;
  a.max_rows = (int32_t)batch->max_rows;
  a.units = (int32_t)(cache->head_dim * dtype_bytes(cache->dtype) / 16);
  a.err = err;
  const dim3 grid(2 * cache->layers, batch->batch);
  pp_tree_commit_kernel<<<grid, kCommitThreads, 0, (cudaStream_t)stream>>>(a);
  return launch_status("pp_tree_commit");
}

extern "C" pp_status pp_beam_reorder(const pp_paged_cache* cache, const int32_t* table,
                                     const int32_t* len, uint32_t groups, uint32_t old_beams,
                                     uint32_t new_beams, uint32_t table_stride,
                                     const int32_t* beams, const int32_t* spare,
                                     int32_t* new_table, int32_t* new_len, int32_t* taken,
                                     uint32_t* err, void* stream) {
  if (const char* m = cache_problem(cache)) return paged_fail(PP_E_INVALID, m);
  if (!table || !len || !beams || !spare || !new_table || !new_len || !taken)
    return paged_fail(PP_E_INVALID, "null argument");
  if (groups == 0 || groups > 65535 || old_beams == 0 || old_beams > 65535 || new_beams == 0 ||
      new_beams > 65535 || table_stride == 0 || table_stride > 0x7fffffffu)
    return paged_fail(PP_E_INVALID, "groups, beams and the table's width must be positive, at most 65535 beams and groups");
  const int32_t* const inputs[] = {table, len, beams, spare};
  for (const int32_t* in : inputs)
    if (in == new_table || in == new_len || in == taken)
      return paged_fail(PP_E_INVALID, "outputs must not be the inputs");
  DeviceScope dev(cache->cuda_device);
  const int sms = dev.ok ? sm_count(cache->cuda_device) : 0;
  if (!sms) return paged_fail(PP_E_CUDA, "cannot use the cache's device");
  ReorderArgs a = {};
  a.c = paged_view(*cache, 0);
  a.table = table;
  a.len = len;
  a.beams = beams;
  a.spare = spare;
  a.new_table = new_table;
  a.new_len = new_len;
  a.taken = taken;
  a.old_beams = (int32_t)old_beams;
  a.new_beams = (int32_t)new_beams;
  a.stride = (int32_t)table_stride;
  a.units = (int32_t)(cache->head_dim * dtype_bytes(cache->dtype) / 16);
  a.err = err;
  const dim3 grid(2 * cache->layers, new_beams, groups);
  pp_beam_reorder_kernel<<<grid, kReorderThreads, 0, (cudaStream_t)stream>>>(a);
  return launch_status("pp_beam_reorder");
}
