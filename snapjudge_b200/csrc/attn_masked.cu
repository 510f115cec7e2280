// attn_masked.cu — attention with score caps, distance biases and document /
// prefix masks: the entry point, and the kernel on CUDA cores that takes every
// shape.
//
// One warp per (query row, head).  The row's visible keys are two intervals
// from the plan; the warp walks them 32 keys at a time (lane = key), with one
// running maximum and sum per row, so masked keys and values are never read.
#include "../../include/snapjudge_b200.h"
#include "attn_masked.cuh"
#include "common.cuh"
#include "kernels.h"

namespace sjb {
namespace {

constexpr int kWarps = 4;

__global__ void __launch_bounds__(32 * kWarps) attn_masked_simt_kernel(AttnMasked p) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= (int64_t)p.n_rows * p.H) return;
  const int row = (int)(w / p.H), h = (int)(w % p.H);
  float o[4];
  attn_masked_row(p, row, h, lane, o);
  bf16* out = p.O + (int64_t)row * p.ldo + (int64_t)h * p.Dh;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < p.Dh) out[lane + 32 * c] = __float2bfloat16(o[c]);
}

}  // namespace

cudaError_t attn_masked_simt(const AttnMasked& p, cudaStream_t st) {
  const int64_t warps = (int64_t)p.n_rows * p.H;
  const int64_t blocks = (warps + kWarps - 1) / kWarps;
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  attn_masked_simt_kernel<<<(unsigned)blocks, 32 * kWarps, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace sjb

namespace {
int bad(const char* m) {
  sjb::set_last_error(m);
  return SJ_ERR_INVALID;
}
}  // namespace

extern "C" {

int64_t sj_attn_masked_workspace(const sj_attn_plan_info* info, int H, int Hkv, int Dh) {
  if (!info || H <= 0 || Hkv <= 0 || H % Hkv || Dh < 1 || Dh > 128) {
    bad("bad attention shape");
    return -1;
  }
  return 0;
}

int sj_attn_masked(const sj_attn_masked_args* a, const sj_attn_plan_info* info,
                   const int32_t* plan, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!a || !info) return bad("null attention argument");
  if (a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv)
    return bad("H must be a positive multiple of Hkv");
  if (a->Dh < 1 || a->Dh > 128) return bad("head_dim must be 1 to 128");
  if (!(a->softcap >= 0.f) || a->softcap > 3.0e38f) return bad("softcap must be finite and >= 0");
  if (a->scale != a->scale || a->scale > 3.0e38f || a->scale < -3.0e38f)
    return bad("scale must be finite");
  if (a->rel_bias && (a->rel_max < 0 || a->rel_max > 0x3fffffff))
    return bad("rel_max must not be negative");
  if (info->n_rows == 0) return SJ_OK;
  if (a->ldq < (int64_t)a->H * a->Dh || a->ldo < (int64_t)a->H * a->Dh ||
      a->ldk < (int64_t)a->Hkv * a->Dh || a->ldv < (int64_t)a->Hkv * a->Dh)
    return bad("a row pitch is smaller than its row");
  if (!a->q || !a->k || !a->v || !a->O || !plan) return bad("null attention operand");
  const int64_t need = sj_attn_masked_workspace(info, a->H, a->Hkv, a->Dh);
  if (workspace_bytes < need || (need > 0 && !workspace)) return bad("the workspace is too small");
  sjb::AttnMasked p = sjb::attn_masked_params(*a, *info, plan);
  const auto st = static_cast<cudaStream_t>(stream);
  const cudaError_t rc = sjb::attn_masked_tc_supported(p) ? sjb::attn_masked_tc(p, st)
                                                          : sjb::attn_masked_simt(p, st);
  if (rc == cudaSuccess) return SJ_OK;
  sjb::set_last_error(std::string("snapjudge CUDA: attn_masked: ") + cudaGetErrorString(rc));
  return SJ_ERR_CUDA;
}

}  // extern "C"
