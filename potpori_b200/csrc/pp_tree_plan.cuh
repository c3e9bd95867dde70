// Launches of the tree attention's kernels.
#pragma once
#include "pp_tree_attn.cuh"

namespace pp {

template <typename K, typename... Extra>
pp_status launch_tree(K kernel, const TreeArgs& a, int threads, size_t smem, cudaStream_t st, Extra... extra) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return paged_fail(PP_E_CUDA, "cannot reserve the attention's shared memory");
  kernel<<<a.ctas, threads, smem, st>>>(a, extra...);
  return launch_status("pp_tree_attention");
}

// The join starts while the last CTAs of the attention still run and waits for them on the device.
// Rows over gridDim.y, as far as one wave of CTAs goes.
template <typename K>
pp_status launch_join(K kernel, const TreeArgs& a, int bm, cudaStream_t st) {
  int y = bm / 4;
  while (y > 1 && (int64_t)y * a.ctas > 148 * 16) y >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.ctas, y);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 8 * (size_t)(a.b.batch + 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, (const TreeArgs)a) != cudaSuccess)
    return launch_status("pp_tree_attention join");
  return PP_OK;
}

// pp_tree_tc.cu
pp_status run_tree_tc(const TreeArgs& a, uint32_t dtype, int dp, cudaStream_t st);

}  // namespace pp
