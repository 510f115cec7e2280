// lora_plan.cu — sj_lora_plan: which adapters the rows of a batch use (host code).
//
// The plan holds
//   rows    the adapter of each row (-1: none);
//   blocks  2 words for each block of 256 rows: the first of its slabs, a multiple
//           of 4, and how many it has;
//   slabs   2 words each: an adapter that a row of the block uses, and which
//           16 of its ranks (adapters in the order of their first row); filled up
//           to a multiple of 4 in each block.
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/snapjudge_b200.h"
#include "kernels.h"

namespace {

int bad(const char* m) {
  sjb::set_last_error(m);
  return SJ_ERR_INVALID;
}

int make_plan(const int32_t* cu, int B, const int32_t* ids, int n_adapters, int rank,
              int32_t* plan, int64_t plan_len, sj_lora_plan_info* info) {
  if (B < 0) return bad("negative batch");
  if (n_adapters < 0) return bad("negative number of adapters");
  if (rank < 1 || rank > 1024) return bad("rank must be 1 to 1024");
  if (!cu || (B > 0 && !ids)) return bad("null plan argument");
  if (cu[0] != 0) return bad("cu_seqlens[0] must be 0");
  for (int b = 0; b < B; ++b) {
    if (cu[b + 1] < cu[b]) return bad("cu_seqlens must be non-decreasing");
    if (ids[b] < -1 || ids[b] >= n_adapters)
      return bad("an adapter number is not in -1 .. n_adapters - 1");
  }
  const int M = cu[B];
  const int per = (rank + 15) / 16;
  const int nb = (int)(((long long)M + 255) / 256);
  std::vector<int32_t> slabs, blocks((size_t)nb * 2, 0);
  std::vector<int> seen((size_t)n_adapters, -1);  // last block that listed the adapter
  int32_t most = 0;
  for (int k = 0, b = 0; k < nb; ++k) {
    const int r1 = std::min<long long>(M, 256ll * (k + 1));
    blocks[2 * k] = (int32_t)(slabs.size() / 2);
    while (b > 0 && cu[b] > 256 * k) --b;
    for (; b < B && cu[b] < r1; ++b) {
      if (cu[b + 1] <= 256 * k || cu[b + 1] == cu[b]) continue;
      const int a = ids[b];
      if (a < 0 || seen[a] == k) continue;
      seen[a] = k;
      for (int s = 0; s < per; ++s) {
        slabs.push_back(a);
        slabs.push_back(s);
      }
    }
    if (slabs.size() / 2 > 0x7ffff0) return bad("the batch needs too many adapter blocks");
    blocks[2 * k + 1] = (int32_t)(slabs.size() / 2) - blocks[2 * k];
    most = std::max(most, blocks[2 * k + 1]);
    slabs.resize((slabs.size() + 7) / 8 * 8, 0);
  }
  info->M = M;
  info->rank = rank;
  info->n_adapters = n_adapters;
  info->n_blocks = nb;
  info->n_slabs = (int32_t)(slabs.size() / 2);
  info->max_slabs = most;
  info->off_blocks = ((long long)M + 3) / 4 * 4;
  info->off_slabs = info->off_blocks + (2ll * nb + 3) / 4 * 4;
  info->plan_len = info->off_slabs + (long long)slabs.size();
  if (!plan) return SJ_OK;
  if (plan_len < info->plan_len) return bad("the plan's memory is too small");
  std::fill(plan, plan + info->plan_len, 0);
  for (int b = 0; b < B; ++b) std::fill(plan + cu[b], plan + cu[b + 1], ids[b]);
  std::copy(blocks.begin(), blocks.end(), plan + info->off_blocks);
  std::copy(slabs.begin(), slabs.end(), plan + info->off_slabs);
  return SJ_OK;
}

}  // namespace

extern "C" int sj_lora_plan(const int32_t* cu_seqlens_host, int B, const int32_t* ids,
                            int n_adapters, int rank, int32_t* plan, int64_t plan_len,
                            sj_lora_plan_info* info) {
  if (!info) return bad("null plan argument");
  try {
    return make_plan(cu_seqlens_host, B, ids, n_adapters, rank, plan, plan_len, info);
  } catch (const std::bad_alloc&) {
    return bad("out of host memory for the plan");
  }
}
