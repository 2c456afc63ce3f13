// Arguments of one paged attention call, shared by the C ABI and the kernels.
#pragma once
#include "paged.cuh"

namespace ak {
namespace paged {

struct AttnArgs {
  PagedLists l;
  const void *q, *k, *v;
  void* o;
  int H, Hkv, G, D;  // G = H / Hkv query heads per key/value head
  int causal, dtype;
  float scale_log2;  // sm_scale * log2(e)
  int64_t qs[2], os[2];    // {token, head}
  int64_t kcs[3], vcs[3];  // {page, head, slot}
};

// Keys that the i-th new token of a sequence sees.
AK_D int visible_keys(const SeqRange& r, int i, int causal) {
  return causal ? max(r.kv_len - r.n + i + 1, 0) : r.kv_len;
}

}  // namespace paged
}  // namespace ak
