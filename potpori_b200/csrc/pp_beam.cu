// Beam search's selection (pp_beam_select): the k best of score + logit - lse over the beams and
// the vocabulary of every group, where lse = log sum exp of the beam's logits.
//
// Within a beam the order of the candidates is the order of its logits, so one pass over the
// logits is enough: pp_beam_rows_kernel reads each logit once and leaves, per slice of a row, its
// maximum, the sum of exp(logit - maximum) and the k largest (logit, token) pairs in order;
// pp_beam_merge_kernel joins the slices of a row and then the rows of a group. The pair is one
// 64-bit key, the logit's bits in ascending order above the inverted token, so keys are distinct,
// the order is total (ties to the lower token) and the result is the same on every run. A slice's
// sum is F32 (lse is good to about 2^-21); the sum over the slices, lse, the values and their comparisons
// are 64-bit, so that two candidates of a beam keep the order of their logits.
// 256 rows of 151936 F32 logits: 37 us with the merge, 4.2 TB/s (a slice is loaded, then worked on: its
// CTA's loads rest meanwhile); 4 rows of BF16 8.4 us, launches and the merge's chain of dependent steps.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_paged.cuh"

using namespace pp;

namespace pp {

constexpr int kBeamMax = 64;         // beams, k
constexpr int kBeamList = 1024;      // keys of a slice at or above its bound
constexpr int kMergeWarps = 16;
constexpr int kCursors = 4;          // slices a merging lane walks at once
constexpr size_t kMergeSmem = 160 * 1024;

// Of one slice of a row.
struct SliceSum {
  float max;
  float sum;  // of exp(logit - max); NaN where a logit was NaN or +inf
};

struct BeamArgs {
  const void* logits;
  int64_t row_stride;
  const float* scores;
  const uint8_t* finished;
  int32_t pad, beams, vocab, k, slices, staged;
  SliceSum* sums;   // [rows][slices]
  uint64_t* keys;   // [rows][slices][k], descending, 0 behind the last
  float* out_scores;
  int32_t* out_beams;
  int32_t* out_tokens;
  uint32_t* err;
};

// Bits of a float in the order of its value (-0 and +0 equal); 0 is below every finite value.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// 0 stands for "no candidate": the key of a logit of -inf.
__device__ __forceinline__ uint64_t beam_key(float v, uint32_t token) {
  return v == -INFINITY ? 0ull : (uint64_t)ordered(v) << 32 | (uint32_t)~token;
}

__device__ __forceinline__ uint64_t warp_max_u64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}

// One slice of one row: grid (slices, rows); a thread holds PER logits, in 16-byte units adjacent
// over the NT threads. A bound that at least k logits reach: the k-th largest among the maxima of G >= k
// groups (G = 32: lane l of all warps; G = NT: every thread). Logits at or above the bound, k and a
// few more, are gathered as keys and put in order by counting. Only where more than kBeamList logits
// are equal at the bound (a slice of constants) are the k best found one by one.
template <typename T, int G, int PER, int NT>
__global__ void __launch_bounds__(NT) pp_beam_rows_kernel(const BeamArgs a) {
  constexpr int W = NT / 32, V = 16 / (int)sizeof(T), U = PER / V, SLICE = NT * PER;
  __shared__ uint32_t s_top[NT];
  __shared__ SliceSum s_part[W];
  __shared__ int s_n;
  __shared__ uint64_t s_keys[kBeamList];
  __shared__ uint64_t s_pick[W];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.y;
  const int64_t slice = row * a.slices + blockIdx.x;
  const int first = blockIdx.x * SLICE, n = min(SLICE, a.vocab - first);
  pdl_launch_dependents();
  if (a.finished && a.finished[row]) return;  // its one candidate needs no logits
  const T* src = (const T*)a.logits + row * a.row_stride + first;

  float x[PER];
  const bool wide = ((uintptr_t)src & 15) == 0;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int e = (i * NT + tid) * V;
    if (wide && e + V <= n) {
      const uint4 raw = __ldcs((const uint4*)(src + e));
      const T* p = (const T*)&raw;
#pragma unroll
      for (int q = 0; q < V; ++q) x[i * V + q] = Elem<T>::get(p[q]);
    } else {
#pragma unroll
      for (int q = 0; q < V; ++q) x[i * V + q] = e + q < n ? Elem<T>::get(src[e + q]) : -INFINITY;
    }
  }
  auto token = [&](int i) { return (uint32_t)(first + ((i / V) * NT + tid) * V + i % V); };

  float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < PER; ++i) part[i & 3] = fmaxf(part[i & 3], x[i]);
  const float mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const uint32_t top = mx == -INFINITY ? 0u : ordered(mx);
  s_top[tid] = top;
  if (tid == 0) s_n = 0;
  // The warp's sum, about its own maximum: F32 over the thread's few and the 32 lanes. The difference
  // x - max is what is multiplied by log2 e, so the large terms are the exact ones. NaN or +inf
  // among the logits make it NaN.
  const uint32_t wt = __reduce_max_sync(0xffffffffu, top);
  const float wm = wt ? from_ordered(wt) : 0.f;
  float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    const float2 d = __fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(-wm, -wm));
    const float2 e = __fmul2_rn(d, make_float2(1.44269504088896341f, 1.44269504088896341f));
    float2 y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(e.y));
    sums[i >> 1 & 1] = __fadd2_rn(sums[i >> 1 & 1], y);
  }
  const float ws = warp_sum((sums[0].x + sums[0].y) + (sums[1].x + sums[1].y));
  if (lane == 0) s_part[warp] = SliceSum{wt ? wm : -INFINITY, ws};
  __syncthreads();
  if (tid == 0) {
    float m = s_part[0].max, t = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, s_part[w].max);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < W; ++w) t += s_part[w].max == -INFINITY ? s_part[w].sum : s_part[w].sum * expf(s_part[w].max - base);
    a.sums[slice] = SliceSum{m, t};
  }
  // The bound, by every warp for itself: k rounds of the largest of the groups' maxima.
  uint32_t bound = 0;
  if constexpr (G == 32) {
    uint32_t g = s_top[lane];
#pragma unroll
    for (int w = 1; w < W; ++w) g = max(g, s_top[32 * w + lane]);
    for (int i = 0; i < a.k; ++i) {
      bound = __reduce_max_sync(0xffffffffu, g);
      const uint32_t at = __ballot_sync(0xffffffffu, g == bound);
      if (lane == __ffs(at) - 1) g = 0;
    }
  } else {
    uint32_t g[W];
#pragma unroll
    for (int w = 0; w < W; ++w) g[w] = s_top[32 * w + lane];
    for (int i = 0; i < a.k; ++i) {
      uint32_t most = g[0];
#pragma unroll
      for (int w = 1; w < W; ++w) most = max(most, g[w]);
      bound = __reduce_max_sync(0xffffffffu, most);
      const uint32_t at = __ballot_sync(0xffffffffu, most == bound);
      if (lane == __ffs(at) - 1) {
        bool gone = false;
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (!gone && g[w] == bound) {
            g[w] = 0;
            gone = true;
          }
      }
    }
  }
  if (top && top >= bound) {
    // Few threads come here, each for few of its logits: those are read again rather than picked out
    // of the registers, which keeps the code short.
    const float at_least = bound ? from_ordered(bound) : -INFINITY;
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mask |= (uint32_t)(x[i] >= at_least) << i;
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      const uint32_t tok = token(i);
      if (tok >= (uint32_t)(first + n)) continue;  // past the row: -inf in the register
      const uint64_t key = beam_key(Elem<T>::get(src[tok - first]), tok);
      if (!key) continue;
      const int at = atomicAdd(&s_n, 1);
      if (at < kBeamList) s_keys[at] = key;
    }
  }
  __syncthreads();
  const int cnt = s_n;
  uint64_t* out = a.keys + slice * a.k;
  if (cnt <= kBeamList) {
    for (int i = tid; i < cnt; i += NT) {
      const uint64_t mine = s_keys[i];
      int rank = 0;
      for (int g = 0; g < cnt; ++g) rank += s_keys[g] > mine;
      if (rank < a.k) out[rank] = mine;
    }
    for (int i = cnt + tid; i < a.k; i += NT) out[i] = 0;
  } else {
    uint64_t last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < a.k; ++r) {
      uint64_t best = 0;
#pragma unroll 1
      for (int e = tid; e < n; e += NT) {
        const uint64_t key = beam_key(Elem<T>::get(src[e]), (uint32_t)(first + e));
        if (key < last && key > best) best = key;
      }
      best = warp_max_u64(best);
      if (lane == 0) s_pick[warp] = best;
      __syncthreads();
      last = s_pick[0];
#pragma unroll
      for (int w = 1; w < W; ++w) last = max(last, s_pick[w]);
      if (tid == 0) out[r] = last;
      __syncthreads();
    }
  }
}

// A double's bits in the order of its value.
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// One group: a warp per beam joins the beam's slices (lane l the slices l, l + 32, ...; k rounds
// of "largest head key, popped"), then one warp joins the beams the same way on the values.
__global__ void __launch_bounds__(32 * kMergeWarps) pp_beam_merge_kernel(const BeamArgs a) {
  extern __shared__ uint64_t s_rows[];  // [beams][k] keys, [beams] lse, [warps][slices][k] copies
  double* s_lse = (double*)(s_rows + a.beams * a.k);
  uint64_t* s_stage = (uint64_t*)(s_lse + a.beams);
  __shared__ int s_state[kBeamMax];  // 0 candidates from logits, 1 finished, 2 out
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int64_t g = blockIdx.x;
  pdl_wait();
  for (int b = warp; b < a.beams; b += warps) {
    const int64_t row = g * a.beams + b;
    const float score = a.scores[row];
    const bool fin = a.finished && a.finished[row];
    bool bad = !(score < INFINITY);
    double lse = 0;
    const uint64_t* keys = a.keys + row * a.slices * a.k;
    if (!fin) {
      // A copy of the row's keys in shared memory where it fits (a pop then waits for shared memory,
      // not for L2), on its way while lse is formed.
      if (a.staged) {
        uint64_t* mine = s_stage + (int64_t)warp * a.slices * a.k;
        for (int i = lane; i < a.slices * a.k; i += 32)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(mine + i)), "l"(keys + i) : "memory");
        keys = mine;
      }
      const SliceSum* sums = a.sums + row * a.slices;
      float m = -INFINITY;
      for (int s = lane; s < a.slices; s += 32) m = fmaxf(m, __ldcg((const float2*)&sums[s]).x);
      m = warp_max(m);
      double sum = 0;
      for (int s = lane; s < a.slices; s += 32) {
        const float2 t = __ldcg((const float2*)&sums[s]);
        sum += t.x == -INFINITY ? (double)t.y : (double)t.y * exp((double)t.x - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      bad |= isnan(sum);
      lse = (double)m + log(sum);
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
    if (bad && lane == 0 && a.err) atomicOr(a.err, PAGED_NONFINITE);
    const int state = bad || score == -INFINITY ? 2 : fin ? 1 : 0;
    if (lane == 0) {
      s_state[b] = state;
      s_lse[b] = lse;
    }
    if (state != 0) continue;
    // The row's k best keys.
    if (a.slices <= 32 * kCursors) {
      int at[kCursors] = {};
      uint64_t head[kCursors];
#pragma unroll
      for (int c = 0; c < kCursors; ++c)
        head[c] = lane + 32 * c < a.slices ? keys[(int64_t)(lane + 32 * c) * a.k] : 0;
      for (int i = 0; i < a.k; ++i) {
        uint64_t most = head[0];
#pragma unroll
        for (int c = 1; c < kCursors; ++c) most = max(most, head[c]);
        const uint64_t top = warp_max_u64(most);
        if (lane == 0) s_rows[b * a.k + i] = top;
        if (top && most == top) {
#pragma unroll
          for (int c = 0; c < kCursors; ++c)
            if (head[c] == top) {
              ++at[c];
              head[c] = at[c] < a.k ? keys[(int64_t)(lane + 32 * c) * a.k + at[c]] : 0;
            }
        }
      }
    } else {
      // A vocabulary of very many slices: round after round the largest key below the last one.
      uint64_t last = ~0ull;
      for (int i = 0; i < a.k; ++i) {
        uint64_t head = 0;
        for (int s = lane; s < a.slices; s += 32)
          for (int q = 0; q < a.k; ++q) {
            const uint64_t key = keys[(int64_t)s * a.k + q];
            if (key < last) {
              head = max(head, key);
              break;
            }
          }
        last = last ? warp_max_u64(head) : 0;
        if (lane == 0) s_rows[b * a.k + i] = last;
      }
    }
    __syncwarp();  // the copy may be overwritten by the warp's next beam
  }
  __syncthreads();
  if (warp != 0) return;
  // Lane l: beams l and l + 32.
  int at[2] = {0, 0};
  auto value = [&](int b, int i, double& v) -> bool {  // candidate i of beam b
    if (b >= a.beams || i >= a.k) return false;
    const double score = a.scores[g * a.beams + b];
    if (s_state[b] == 1) {
      v = score;
      return i == 0;
    }
    if (s_state[b] == 2) return false;
    const uint64_t key = s_rows[b * a.k + i];
    v = score + ((double)from_ordered((uint32_t)(key >> 32)) - s_lse[b]);
    return key != 0;
  };
  uint64_t head[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    double v;
    head[q] = value(lane + 32 * q, 0, v) ? ordered64(v) : 0;
  }
  for (int i = 0; i < a.k; ++i) {
    const uint64_t top = warp_max_u64(max(head[0], head[1]));
    // Ties: the lowest beam.
    const uint32_t lo = __ballot_sync(0xffffffffu, head[0] == top), hi = __ballot_sync(0xffffffffu, head[1] == top);
    const int b = !top ? -1 : lo ? __ffs(lo) - 1 : 32 + __ffs(hi) - 1;
    if (b < 0 ? lane == 0 : lane == (b & 31)) {
      const int64_t o = g * a.k + i;
      if (b < 0) {
        a.out_scores[o] = -INFINITY;
        a.out_beams[o] = -1;
        a.out_tokens[o] = -1;
      } else {
        const int q = b >> 5;
        double v = 0;
        const int c = q ? at[1] : at[0];
        value(b, c, v);
        a.out_scores[o] = (float)v;
        a.out_beams[o] = b;
        a.out_tokens[o] = s_state[b] == 1 ? a.pad : (int32_t)~(uint32_t)s_rows[b * a.k + c];
        const uint64_t next = value(b, c + 1, v) ? ordered64(v) : 0;
        if (q) {
          at[1] = c + 1;
          head[1] = next;
        } else {
          at[0] = c + 1;
          head[0] = next;
        }
      }
    }
    __syncwarp();
  }
}

constexpr uint32_t kSliceLarge = 128 * 32, kSliceSmall = 256 * 8;
// Slices of 4096 logits, 32 of each of 128 threads; where those are not four an SM, of 2048, 8 of each
// of 256, so that more warps share the work (256 rows of 151936: 38.3 us, of 8192 logits by 256 threads
// 43, of 2048 78; 4 rows: 9.0 us in 2048s, 11.9 in 4096s).
inline bool beam_wide(uint32_t groups, uint32_t beams, uint32_t vocab, int sms) {
  return (uint64_t)groups * beams * ((vocab + kSliceLarge - 1) / kSliceLarge) >= 4ull * sms;
}
struct BeamWork {
  uint64_t sums, keys, total;
  uint32_t slices;
  BeamWork(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k, bool wide) {
    const uint64_t rows = (uint64_t)groups * beams;
    const uint32_t size = wide ? kSliceLarge : kSliceSmall;
    slices = (uint32_t)(((uint64_t)vocab + size - 1) / size);
    sums = 0;
    keys = rows * slices * sizeof(SliceSum);
    total = keys + rows * slices * k * 8;
  }
};

template <typename T, int PER, int NT>
void launch_rows(const BeamArgs& a, dim3 grid, cudaStream_t st) {
  // Up to 16 of a slice: 32 groups; above, a group per thread.
  if (a.k <= 16) pp_beam_rows_kernel<T, 32, PER, NT><<<grid, NT, 0, st>>>(a);
  else pp_beam_rows_kernel<T, NT, PER, NT><<<grid, NT, 0, st>>>(a);
}
template <typename T>
void launch_rows(const BeamArgs& a, bool wide, dim3 grid, cudaStream_t st) {
  if (wide) launch_rows<T, 32, 128>(a, grid, st);
  else launch_rows<T, 8, 256>(a, grid, st);
}

}  // namespace pp

extern "C" uint64_t pp_beam_select_work_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k) {
  return BeamWork(groups, beams, vocab, k, false).total;  // the smaller slices need more, whatever the device
}

extern "C" pp_status pp_beam_select(const void* logits, pp_dtype dtype, int64_t row_stride,
                                    const float* scores, const uint8_t* finished, int32_t pad,
                                    uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k,
                                    float* out_scores, int32_t* out_beams, int32_t* out_tokens,
                                    void* work, uint64_t work_bytes, uint32_t* err,
                                    int32_t cuda_device, void* stream) {
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !work)
    return paged_fail(PP_E_INVALID, "null argument");
  if (dtype != PP_F32 && dtype != PP_BF16 && dtype != PP_F16)
    return paged_fail(PP_E_INVALID, "the logits' dtype must be PP_F32, PP_BF16 or PP_F16");
  if (groups == 0 || beams == 0 || beams > (uint32_t)kBeamMax || k == 0 || k > (uint32_t)kBeamMax)
    return paged_fail(PP_E_INVALID, "groups, beams and k must be positive, beams and k at most 64");
  if (vocab == 0 || vocab > (1u << 24)) return paged_fail(PP_E_INVALID, "vocab must be 1..2^24");
  if ((uint64_t)groups * beams > 65535) return paged_fail(PP_E_INVALID, "more than 65535 beams in all");
  if (row_stride < (int64_t)vocab && (uint64_t)groups * beams > 1)
    return paged_fail(PP_E_INVALID, "row_stride shorter than the vocabulary");
  if ((uintptr_t)logits % dtype_bytes(dtype)) return paged_fail(PP_E_INVALID, "misaligned logits");
  if ((uintptr_t)work % 16 || work_bytes < pp_beam_select_work_bytes(groups, beams, vocab, k))
    return paged_fail(PP_E_INVALID, "work must be 16-byte aligned and pp_beam_select_work_bytes long");
  if (out_scores == scores) return paged_fail(PP_E_INVALID, "out_scores must not be scores");
  DeviceScope dev(cuda_device);
  const int sms = dev.ok ? sm_count(cuda_device) : 0;
  if (!sms) return paged_fail(PP_E_CUDA, "cannot use the device");
  const bool wide = beam_wide(groups, beams, vocab, sms);
  const BeamWork w(groups, beams, vocab, k, wide);
  BeamArgs a = {};
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.pad = pad;
  a.beams = (int32_t)beams;
  a.vocab = (int32_t)vocab;
  a.k = (int32_t)k;
  a.slices = (int32_t)w.slices;
  a.sums = (SliceSum*)((uint8_t*)work + w.sums);
  a.keys = (uint64_t*)((uint8_t*)work + w.keys);
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  a.err = err;
  const cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(a.slices, groups * beams);
  if (dtype == PP_F32) launch_rows<float>(a, wide, grid, st);
  else if (dtype == PP_BF16) launch_rows<__nv_bfloat16>(a, wide, grid, st);
  else launch_rows<__half>(a, wide, grid, st);
  const pp_status r = launch_status("pp_beam_select");
  if (r != PP_OK) return r;
  const size_t base = (size_t)beams * k * 8 + (size_t)beams * 8, copy = (size_t)a.slices * k * 8;
  int warps = (int)(beams < (uint32_t)kMergeWarps ? beams : kMergeWarps);
  while (warps > 1 && base + warps * copy > kMergeSmem) --warps;
  a.staged = base + warps * copy <= kMergeSmem;
  if (!a.staged) warps = (int)(beams < (uint32_t)kMergeWarps ? beams : kMergeWarps);
  const size_t smem = base + (a.staged ? warps * copy : 0);
  static bool done[64] = {};
  if (!reserve_smem(pp_beam_merge_kernel, (int)kMergeSmem, cuda_device, done))
    return PP_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, pp_beam_merge_kernel, (const BeamArgs)a) != cudaSuccess)
    return launch_status("pp_beam_select merge");
  return PP_OK;
}
