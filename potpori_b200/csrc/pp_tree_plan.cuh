// Launches of the tree attention's kernels.
#pragma once
#include "pp_tree_attn.cuh"

namespace pp {

template <auto kernel, typename... Extra>
pp_status launch_tree(const TreeArgs& a, int threads, size_t smem, cudaStream_t st, Extra... extra) {
  static bool done[64] = {};
  if (!reserve_smem(kernel, kMaxSmem, a.dev, done))
    return PP_E_CUDA;
  kernel<<<a.ctas, threads, smem, st>>>(a, extra...);
  return launch_status("pp_tree_attention");
}

// The join starts while the last CTAs of the attention still run and waits for them on the device.
template <typename T, int DP>
pp_status launch_join(const TreeArgs& a, cudaStream_t st) {
  const int items = a.ctas * a.bm, most = 8 * sm_count(a.dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(items < most ? items : most);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 4 * (size_t)(a.ctas + 1 + a.b.batch + 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, pp_tree_join_kernel<T, DP>, (const TreeArgs)a) != cudaSuccess)
    return launch_status("pp_tree_attention join");
  return PP_OK;
}

// pp_tree_tc.cu
pp_status run_tree_tc(const TreeArgs& a, const TreeMaps& m, uint32_t dtype, int dp, cudaStream_t st);

}  // namespace pp
