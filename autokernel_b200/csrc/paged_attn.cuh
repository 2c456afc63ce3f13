// Arguments of one paged attention call, shared by the C ABI and the kernels.
#pragma once
#include "paged.cuh"
#include "sm100.cuh"

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

// Weights P = exp2(score scale log2e - r), of which the matrix units take 16 bits, against a reference r of
// their row that cancels in O / l.  r moves when a block's largest score passes it by more than
// kShift + kLag, and is then put kShift below that score, so the largest weight so far is at least
// 2^kShift and at most 2^(kShift + kLag).  bf16 has the exponents of fp32: no shift.  fp16 weights
// are kept at the top of its range, where 2^15 is the largest power: below 2^-14 they lose bits
// (2^-25 each), so a weight under 2^-(14 + kShift) of its row's largest is off by up to
// 2^-(25 + kShift) of that (20,000 keys 26 below a key whose value is 0 lost 1.3% of their output
// without the shift).  A smaller lag leaves more room and moves r, and with it O, more often: prompts
// of 4096 + 3700 tokens, 32 heads of 128, take 354 us with a lag of 8 or 4, 373 with 2 and 387
// with 0; with scores four times as wide 373, 382, 384 and 387.
template <int DT>
struct Weight {
  static constexpr float kShift = DT == AK_F16 ? 11.f : 0.f;
  static constexpr float kLag = DT == AK_F16 ? 4.f : 8.f;
  // Scores are fp32, and so is r.  From 2^23 on its steps are 1 and more: fp16 scores are rounded up to
  // it, so that no weight passes 2^15, and up to kLimit the largest one is at least 1 (in bf16,
  // between 2^-64 and 2^72).  A row whose largest score lies beyond, on either side, is NaN: its weights
  // would be infinite or all 0, and its scores have lost what tells them apart.  Scores below -kLimit
  // beside larger ones weigh 0.
  static constexpr float kLimit = DT == AK_F16 ? 134217728.f : 2147483648.f;  // 2^27, 2^31
  static constexpr float kFar = -3.4028235e38f;  // r of a row of which only scores below -kLimit were seen
  // the largest score of a block, scaled
  static AK_D float top(float score, float scale_log2) {
    return DT == AK_F16 ? __fmul_ru(score, scale_log2) : __fmul_rn(score, scale_log2);
  }
  // whether a block with this top moves r, and where to (r = -inf: nothing has been seen yet)
  static AK_D bool moves(float top, float r) { return top - r > kShift + kLag; }
  static AK_D float reference(float top) {
    return fabsf(top) < kLimit ? __fsub_ru(top, kShift) : top < 0.f ? kFar : __int_as_float(0x7fffffff);
  }
  // what is subtracted from scores: with no r to subtract, the exponential of what was seen is 0
  static AK_D float base(float r) { return r <= kFar ? 0.f : r; }
  // a row's sum of weights, from that sum and r over all of its keys
  static AK_D float total(float sum, float r) { return r == kFar ? __int_as_float(0x7fffffff) : sum; }
};

// paged_decode.cu: tiles of 16 query rows, each of which reads all of its keys; paged_chunk.cu: two tensor-core
// tiles of 128.  Either takes any lists; paged_attn.cu chooses.
int run_decode(const AttnArgs& a, void* ws, cudaStream_t st);
size_t decode_workspace(int D);
int run_chunk(const AttnArgs& a, void* ws, cudaStream_t st);
size_t chunk_workspace(int D);

inline int gcd_int(int x, int y) {
  while (y) {
    const int r = x % y;
    x = y;
    y = r;
  }
  return x;
}

// 4-D map over a cache [pages, heads, slots, D]: boxes of `box` slots x 64 elements of one page.
inline bool cache_tmap(CUtensorMap* m, const AttnArgs& a, const void* base, const int64_t* st,
                       int box) {
  const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)a.l.page_size, (uint64_t)a.Hkv,
                            (uint64_t)a.l.num_pages};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i)  // a dim of one element may carry any stride
    strides[i] = (uint64_t)(dims[i + 1] > 1 ? st[2 - i] : a.D) * 2;
  const uint32_t b[4] = {64, (uint32_t)box, 1, 1};
  return make_tmap(m, a.dtype, 4, base, dims, strides, b);
}

// The same cache as [pages, heads, D / 64, slots, 64]: one box is `box` slots of a page with all of D,
// chunk after chunk, so that one copy brings what cache_tmap's maps bring in D / 64.
inline bool cache_tmap_5d(CUtensorMap* m, const AttnArgs& a, const void* base, const int64_t* st,
                          int box) {
  const uint64_t dims[5] = {64, (uint64_t)a.l.page_size, (uint64_t)a.D / 64, (uint64_t)a.Hkv,
                            (uint64_t)a.l.num_pages};
  const uint64_t strides[4] = {(uint64_t)(a.l.page_size > 1 ? st[2] : a.D) * 2, 128,
                               (uint64_t)(a.Hkv > 1 ? st[1] : a.D) * 2,
                               (uint64_t)(a.l.num_pages > 1 ? st[0] : a.D) * 2};
  const uint32_t b[5] = {64, (uint32_t)box, (uint32_t)a.D / 64, 1, 1};
  return make_tmap(m, a.dtype, 5, base, dims, strides, b);
}

// Launch a kernel that may begin while its predecessor on the stream finishes (it waits for it
// with griddepcontrol.wait before it reads what that one wrote).
template <class... P, class... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    set_error("paged_attention: launch failed: %s", cudaGetErrorString(e));
    return AK_ERR_LAUNCH;
  }
  return AK_OK;
}

}  // namespace paged
}  // namespace ak
