// Beam search's selection (pp_beam_select): the k best of score + logit - lse over the beams and
// the vocabulary of every group, where lse = log sum exp of the beam's logits.
//
// Within a beam the order of the candidates is the order of its logits, so one pass over the
// logits is enough: pp_beam_rows_kernel reads each logit once and leaves, per slice of a row, its
// maximum, the sum of exp(logit - maximum) and the k largest (logit, token) pairs in order;
// pp_beam_merge_kernel joins the slices of a row and then the rows of a group. The pair is one
// 64-bit key, the logit's bits in ascending order above the inverted token, so keys are distinct,
// the order is total (ties to the lower token) and the result is the same on every run. A slice's
// sum is F32 over the few elements of a thread and 64-bit above that; lse, the values and their
// comparisons are 64-bit, so that two candidates a rounding apart keep their order.
#include <cuda_runtime.h>

#include "../../include/potpori_b200.h"
#include "pp_paged.cuh"

using namespace pp;

namespace pp {

constexpr int kBeamThreads = 256;
constexpr int kBeamPer = 16;                            // logits a thread holds
constexpr int kBeamSlice = kBeamThreads * kBeamPer;     // logits of a slice
constexpr int kBeamMax = 64;                            // beams, k
constexpr int kMergeWarps = 16;
constexpr int kCursors = 4;                             // slices a merging lane walks at once
constexpr size_t kMergeSmem = 160 * 1024;
constexpr int kBeamHeapMax = 2048;                      // keys of a slice at or above its bound

// Of one slice of a row.
struct SliceSum {
  double sum;  // of exp(logit - max)
  float max;
  int32_t bad;  // NaN or +inf seen
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

// One slice of one row: grid (slices, rows). A bound that at least k keys reach: the slice is cut
// into G >= k groups, and the k-th largest of the groups' largest keys has k keys at or above it.
// Keys at or above the bound (k plus a few, at most kBeamHeapMax as they lie in k groups) are
// gathered and put in order by counting.
template <typename T, int G>
__global__ void __launch_bounds__(kBeamThreads) pp_beam_rows_kernel(const BeamArgs a) {
  __shared__ float s_max[kBeamThreads / 32];
  __shared__ double s_sum[kBeamThreads / 32];
  __shared__ int s_bad[kBeamThreads / 32];
  __shared__ uint64_t s_group[G];
  __shared__ uint64_t s_bound;
  __shared__ int s_n;
  __shared__ uint64_t s_keys[kBeamHeapMax];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.y;
  const int64_t slice = row * a.slices + blockIdx.x;
  const int first = blockIdx.x * kBeamSlice, n = min(kBeamSlice, a.vocab - first);
  pdl_launch_dependents();
  if (a.finished && a.finished[row]) return;  // its one candidate needs no logits
  const T* src = (const T*)a.logits + row * a.row_stride + first;

  // Thread t holds elements [e0(i), e0(i) + V) for unit i, units V wide and adjacent over threads.
  constexpr int V = 16 / (int)sizeof(T), U = kBeamPer / V;
  float x[kBeamPer];
  const bool wide = ((uintptr_t)src & 15) == 0;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int e = (i * kBeamThreads + tid) * V;
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
  auto token = [&](int i) { return (uint32_t)(first + ((i / V) * kBeamThreads + tid) * V + i % V); };

  float mx = -INFINITY;
  int best = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) {
    bad |= !(x[i] < INFINITY);  // NaN and +inf
    if (x[i] > mx) {
      mx = x[i];
      best = i;
    }
  }
  uint64_t key = 0;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i)
    if (i == best) key = beam_key(mx, token(i));
  const float wm = warp_max(mx);
  const uint32_t any_bad = __ballot_sync(0xffffffffu, bad);
  if (lane == 0) {
    s_max[warp] = wm;
    s_bad[warp] = any_bad != 0;
  }
  // Groups: all the elements of G threads' worth each; group g = threads g, g + G, ...
  if (tid < G) s_group[tid] = 0;
  if (tid == 0) s_n = 0;
  __syncthreads();
  if (G == kBeamThreads) s_group[tid & (G - 1)] = key;
  else atomicMax((unsigned long long*)&s_group[tid & (G - 1)], (unsigned long long)key);
  float bm = s_max[0];
  int bb = s_bad[0];
#pragma unroll
  for (int w = 1; w < kBeamThreads / 32; ++w) {
    bm = fmaxf(bm, s_max[w]);
    bb |= s_bad[w];
  }
  // exp over the thread's elements; -inf everywhere (or a bad row, which is dropped) adds nothing.
  float sum = 0.f;
  if (bm > -INFINITY && !bb) {
#pragma unroll
    for (int i = 0; i < kBeamPer; ++i) sum += expf(x[i] - bm);
  }
  double ds = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ds += __shfl_xor_sync(0xffffffffu, ds, o);
  if (lane == 0) s_sum[warp] = ds;
  __syncthreads();
  if (tid == 0) {
    double t = 0;
    for (int w = 0; w < kBeamThreads / 32; ++w) t += s_sum[w];
    a.sums[slice] = SliceSum{t, bm, bb};
  }
  // The bound: a group key's rank is the number of larger ones.
  if (tid < G) {
    const uint64_t mine = s_group[tid];
    int rank = 0;
    for (int g = 0; g < G; ++g) {
      const uint64_t other = s_group[g];
      rank += other > mine || (other == mine && g < tid);
    }
    if (rank == a.k - 1) s_bound = mine;
  }
  __syncthreads();
  const uint64_t bound = s_bound;
  const uint32_t bound_hi = (uint32_t)(bound >> 32);
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) {
    if (x[i] == -INFINITY || ordered(x[i]) < bound_hi) continue;
    const uint64_t c = beam_key(x[i], token(i));
    if (c >= bound) {
      const int at = atomicAdd(&s_n, 1);
      if (at < kBeamHeapMax) s_keys[at] = c;
    }
  }
  __syncthreads();
  const int cnt = min(s_n, kBeamHeapMax);
  uint64_t* out = a.keys + slice * a.k;
  for (int i = tid; i < cnt; i += kBeamThreads) {
    const uint64_t mine = s_keys[i];
    int rank = 0;
    for (int g = 0; g < cnt; ++g) rank += s_keys[g] > mine;
    if (rank < a.k) out[rank] = mine;
  }
  for (int i = cnt + tid; i < a.k; i += kBeamThreads) out[i] = 0;
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
    double m = -INFINITY, sum = 0;
    if (!fin) {
      int nf = 0;
      for (int s = lane; s < a.slices; s += 32) {
        const SliceSum t = a.sums[row * a.slices + s];
        nf |= t.bad;
        if (!t.bad && t.sum > 0) {
          const double nm = fmax(m, (double)t.max);
          sum = sum * exp(m - nm) + t.sum * exp((double)t.max - nm);
          m = nm;
        }
      }
      bad |= __any_sync(0xffffffffu, nf);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
        const double nm = fmax(m, om);
        if (nm > -INFINITY) sum = sum * exp(m - nm) + os * exp(om - nm);
        m = nm;
      }
    }
    if (bad && lane == 0 && a.err) atomicOr(a.err, PAGED_NONFINITE);
    const int state = bad || score == -INFINITY ? 2 : fin ? 1 : 0;
    if (lane == 0) {
      s_state[b] = state;
      s_lse[b] = state == 0 ? m + log(sum) : 0.0;
    }
    if (state != 0) continue;
    // The row's k best keys, from a copy in shared memory where it fits (a pop then waits for
    // shared memory, not for L2).
    const uint64_t* keys = a.keys + row * a.slices * a.k;
    if (a.staged) {
      uint64_t* mine = s_stage + (int64_t)warp * a.slices * a.k;
      for (int i = lane; i < a.slices * a.k; i += 32) mine[i] = keys[i];
      __syncwarp();
      keys = mine;
    }
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

struct BeamWork {
  uint64_t sums, keys, total;
  BeamWork(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k) {
    const uint64_t slices = (vocab + (uint64_t)kBeamSlice - 1) / kBeamSlice, rows = (uint64_t)groups * beams;
    sums = 0;
    keys = rows * slices * sizeof(SliceSum);
    total = keys + rows * slices * k * 8;
  }
};

template <typename T>
void launch_rows(const BeamArgs& a, dim3 grid, cudaStream_t st) {
  // Up to 16 of a slice: 32 groups; above, a group per thread.
  if (a.k <= 16) pp_beam_rows_kernel<T, 32><<<grid, kBeamThreads, 0, st>>>(a);
  else pp_beam_rows_kernel<T, kBeamThreads><<<grid, kBeamThreads, 0, st>>>(a);
}

}  // namespace pp

extern "C" uint64_t pp_beam_select_work_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k) {
  return BeamWork(groups, beams, vocab, k).total;
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
  const BeamWork w(groups, beams, vocab, k);
  if ((uintptr_t)work % 16 || work_bytes < w.total)
    return paged_fail(PP_E_INVALID, "work must be 16-byte aligned and pp_beam_select_work_bytes long");
  DeviceScope dev(cuda_device);
  if (!dev.ok) return paged_fail(PP_E_CUDA, "cannot use the device");
  BeamArgs a = {};
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.pad = pad;
  a.beams = (int32_t)beams;
  a.vocab = (int32_t)vocab;
  a.k = (int32_t)k;
  a.slices = (int32_t)((vocab + kBeamSlice - 1) / kBeamSlice);
  a.sums = (SliceSum*)((uint8_t*)work + w.sums);
  a.keys = (uint64_t*)((uint8_t*)work + w.keys);
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  a.err = err;
  const cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(a.slices, groups * beams);
  if (dtype == PP_F32) launch_rows<float>(a, grid, st);
  else if (dtype == PP_BF16) launch_rows<__nv_bfloat16>(a, grid, st);
  else launch_rows<__half>(a, grid, st);
  const pp_status r = launch_status("pp_beam_select");
  if (r != PP_OK) return r;
  const size_t base = (size_t)beams * k * 8 + (size_t)beams * 8, copy = (size_t)a.slices * k * 8;
  int warps = (int)(beams < (uint32_t)kMergeWarps ? beams : kMergeWarps);
  while (warps > 1 && base + warps * copy > kMergeSmem) --warps;
  a.staged = base + warps * copy <= kMergeSmem;
  if (!a.staged) warps = (int)(beams < (uint32_t)kMergeWarps ? beams : kMergeWarps);
  const size_t smem = base + (a.staged ? warps * copy : 0);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(pp_beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)kMergeSmem) != cudaSuccess)
    return paged_fail(PP_E_CUDA, "cannot reserve the merge's shared memory");
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
