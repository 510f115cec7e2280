// gemm_lora.cuh — parameters of the projection with low-rank adapters.
#pragma once

#include "../../include/snapjudge_b200.h"
#include "common.cuh"

namespace sjb {

struct GemmLora {
  const bf16 *X, *W, *A, *B;  // [M, K], [N, K], [n_adapters, R, K], [n_adapters, N, R]
  const float *scale, *bias;  // [n_adapters] or null, [N] or null
  bf16* C;
  int64_t ldx, ldc;
  int M, N, K, R, act, n_adapters;
  int n_blocks, n_slabs, max_slabs;  // max_slabs: of any one block
  const int32_t* rows;    // plan: adapter of each row
  const int2* blocks;     // plan: first slab (a multiple of 4) and slabs of each block
  const int2* slabs;      // plan: (adapter, sixteen)
  int unit;               // slabs that one load of B takes: 4, 2 or 1
};

// tcgen05 kernels (gemm_lora_tc.cu); U: n_slabs / 4 x 256 x 64 bf16 of workspace.
bool gemm_lora_tc_supported(const GemmLora& p);
cudaError_t gemm_lora_tc(const GemmLora& p, void* U, cudaStream_t st);
// One kernel for few rows (gemm_lora_small.cu), same shapes; no workspace.
bool gemm_lora_small_runs(const GemmLora& p);
cudaError_t gemm_lora_small(const GemmLora& p, cudaStream_t st);
// As attn_tc_take_status, for these kernels.
cudaError_t gemm_lora_take_status(int* code);

// Kernels on CUDA cores for every shape and alignment; U: M x R bf16 of workspace.
cudaError_t gemm_lora_simt(const GemmLora& p, void* U, cudaStream_t st);

}  // namespace sjb
