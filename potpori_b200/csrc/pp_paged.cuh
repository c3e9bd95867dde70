// What the operators over a paged K/V cache share: host checks of the descriptors, the device
// switch, and the device side's page addressing and element types.
//
// A cache holds, per layer, n_pages pages of page_size positions; position s of sequence b is
// row s % page_size of page page_table[b][s / page_size], and K (V) element (layer, page, row,
// head, dim) sits at base + layer * layer_stride + page * page_stride + row * row_stride +
// head * head_stride + dim. Offsets are 64-bit throughout: a long cache passes 2^31 elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdio>

#include "../../include/potpori_b200.h"
#include "pp_common.cuh"

namespace pp {

// ---- host ---------------------------------------------------------------------------------
inline pp_status paged_fail(pp_status st, const char* msg) noexcept {
  try {
    set_global_error(msg);
  } catch (...) {  // no memory for the message: the status still tells
  }
  return st;
}

// Makes `dev` current for the call and puts the caller's device back.
struct DeviceScope {
  int prev = -1;
  bool ok = false;
  explicit DeviceScope(int dev) noexcept {
    if (cudaGetDevice(&prev) != cudaSuccess) return;
    if (prev == dev) {
      ok = true;
      prev = -1;
      return;
    }
    ok = cudaSetDevice(dev) == cudaSuccess;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

inline int dtype_bytes(uint32_t t) { return t == PP_F32 ? 4 : 2; }

inline int sm_count(int dev) noexcept {
  static int n[64] = {};
  if (dev < 0 || dev >= 64) return 0;
  if (!n[dev]) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    n[dev] = v;
  }
  return n[dev];
}

// Lets `kernel` take up to `bytes` of dynamic shared memory on the current device, once per device
// (`done`: one flag per device of this kernel).
template <typename K>
inline bool reserve_smem(K kernel, int bytes, int dev, bool (&done)[64]) noexcept {
  if (dev < 0 || dev >= 64) return false;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      char msg[160];
      snprintf(msg, sizeof msg, "cannot reserve a kernel's shared memory: %s", cudaGetErrorString(e));
      paged_fail(PP_E_CUDA, msg);
      return false;
    }
    done[dev] = true;
  }
  return true;
}
constexpr int kMaxSmem = 232448;  // 227 KB: the most a CTA can have

// The rules every paged operator shares; nullptr when the descriptor can be run.
inline const char* cache_problem(const pp_paged_cache* c) noexcept {
  if (!c || !c->k || !c->v) return "null cache";
  if (c->dtype != PP_F32 && c->dtype != PP_BF16 && c->dtype != PP_F16)
    return "the cache's dtype must be PP_F32, PP_BF16 or PP_F16";
  if (c->layers == 0 || c->n_pages == 0 || c->page_size == 0 || c->n_kv_heads == 0)
    return "empty cache";
  if (c->n_pages > 0x7fffffffu || c->page_size > (1u << 20) || c->layers > 4096 ||
      c->n_kv_heads > 4096)
    return "cache sizes out of range";
  if (c->head_dim == 0 || c->head_dim % 8 || c->head_dim > 256)
    return "head_dim must be a multiple of 8 up to 256";
  const int64_t unit = 16 / dtype_bytes(c->dtype);
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || c->page_stride % unit ||
      c->row_stride % unit || c->head_stride % unit || c->layer_stride % unit)
    return "cache pointers and strides must be multiples of 16 bytes";
  if (c->row_stride < 0 || c->head_stride < 0 || c->page_stride < 0 || c->layer_stride < 0)
    return "cache strides must not be negative";
  const int64_t d = c->head_dim;
  if ((c->page_size > 1 && c->row_stride < d) || (c->n_kv_heads > 1 && c->head_stride < d) ||
      (c->n_pages > 1 && c->page_stride < d) || (c->layers > 1 && c->layer_stride < d))
    return "rows of the cache overlap";
  return nullptr;
}
inline const char* batch_problem(const pp_paged_batch* b) noexcept {
  if (!b || !b->cu_rows || !b->kv_len || !b->page_table) return "null batch";
  if (b->batch == 0 || b->batch > 4096) return "batch must be 1..4096 sequences";
  if (b->table_stride == 0 || b->table_stride > 0x7fffffffu) return "empty page table";
  if (b->rows > (1u << 24)) return "rows out of range";
  return nullptr;
}

inline pp_status launch_status(const char* what) noexcept {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return PP_OK;
  char msg[160];
  snprintf(msg, sizeof msg, "%s launch: %s", what, cudaGetErrorString(e));
  return paged_fail(PP_E_CUDA, msg);
}

// ---- device -------------------------------------------------------------------------------
// n / d for n < 2^31 by one multiplication (round-up method: q = (t + (n - t) / 2) >> (l - 1)
// with t the high half of n * m).
struct FastDiv {
  uint32_t d, m, s1, s2;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t div) : d(div) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < div) ++l;
    m = (uint32_t)((((1ull << 32) * ((1ull << l) - div)) / div) + 1);
    s1 = l < 1 ? l : 1;
    s2 = l < 1 ? 0 : l - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    const uint32_t t = __umulhi(m, n);
    return (t + ((n - t) >> s1)) >> s2;
  }
};

// One layer of a cache as the kernels take it.
struct PagedView {
  uint8_t* k;
  uint8_t* v;
  int64_t page_bytes, row_bytes, head_bytes, layer_bytes;
  int32_t n_pages, n_kv, head_dim, layers;
  FastDiv page;  // by page_size
};
inline PagedView paged_view(const pp_paged_cache& c, uint32_t layer) {
  const int64_t e = dtype_bytes(c.dtype);
  PagedView v;
  v.k = (uint8_t*)c.k + (int64_t)layer * c.layer_stride * e;
  v.v = (uint8_t*)c.v + (int64_t)layer * c.layer_stride * e;
  v.page_bytes = c.page_stride * e;
  v.row_bytes = c.row_stride * e;
  v.head_bytes = c.head_stride * e;
  v.layer_bytes = c.layer_stride * e;
  v.n_pages = (int32_t)c.n_pages;
  v.n_kv = (int32_t)c.n_kv_heads;
  v.head_dim = (int32_t)c.head_dim;
  v.layers = (int32_t)c.layers;
  v.page = FastDiv(c.page_size);
  return v;
}
struct BatchView {
  const int32_t* cu_rows;
  const int32_t* kv_len;
  const int32_t* table;
  int32_t batch, rows, table_stride;
};
inline BatchView batch_view(const pp_paged_batch& b) {
  return BatchView{b.cu_rows, b.kv_len, b.page_table, (int32_t)b.batch, (int32_t)b.rows,
                   (int32_t)b.table_stride};
}

// Byte offset of position `index` (head 0) in a layer's K or V, or -1 where the table has no
// valid page for it.
__device__ __forceinline__ int64_t paged_offset(const PagedView& c, const int32_t* table_row,
                                                int32_t table_stride, int32_t index) {
  if (index < 0) return -1;
  const uint32_t p = c.page.div((uint32_t)index);
  if (p >= (uint32_t)table_stride) return -1;
  const int32_t page = __ldg(table_row + p);
  if ((uint32_t)page >= (uint32_t)c.n_pages) return -1;
  return (int64_t)page * c.page_bytes + (int64_t)((uint32_t)index - p * c.page.d) * c.row_bytes;
}

// Sequence that holds row t: the last b with cu_rows[b] <= t. By one warp: every round narrows
// the range 32-fold. -1 when t is past the last sequence's rows.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, int t, int lane) {
  int lo = 0, n = batch + 1;  // the answer is the last index in [lo, lo + n) with cu <= t
  while (true) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool le = at < n && cu[lo + at] <= t;
    const uint32_t votes = __ballot_sync(0xffffffffu, le);
    if (!votes) return -1;
    const int last = 31 - __clz(votes);
    lo += last * step;
    n = min(step, n - last * step);
    if (step == 1) break;
  }
  return lo < batch ? lo : -1;
}

// Bits of the caller's error word.
enum : uint32_t { PAGED_BAD_PAGE = 1u, PAGED_NONFINITE = 2u, PAGED_TIMEOUT = 4u };

// Element types: load one as F32, store one rounded to nearest even.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// N consecutive elements (N * sizeof(T) a multiple of 8 bytes, aligned to the smaller of that and
// 16) as F32.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float* f) {
  alignas(16) T v[N];
  if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) ((uint4*)v)[i] = ((const uint4*)p)[i];
  } else {
    *(uint2*)v = *(const uint2*)p;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = Elem<T>::get(v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float* f) {
  alignas(16) T v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = Elem<T>::put(f[i]);
  if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) ((uint4*)p)[i] = ((const uint4*)v)[i];
  } else {
    *(uint2*)p = *(const uint2*)v;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  store_n<T, 8>(p, f);
}

}  // namespace pp
