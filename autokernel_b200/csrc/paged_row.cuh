// One row of attention (a token and a query head) by a whole CTA, key by key: any type, head dimension,
// stride and page size.
#pragma once
#include "paged_attn.cuh"

namespace ak {
namespace paged {

// Shared memory for it, of the kernel's own: what a function declares counts for every kernel of its file.
template <int NI, int THREADS>
struct RowScratch {
  static constexpr int GROUPS = THREADS / 8, WARPS = THREADS / 32;
  static_assert(GROUPS <= 32, "a warp joins the groups");
  float m[GROUPS], l[GROUPS];
  float o[WARPS][8 * NI];
};

// Row of the t-th new token of sequence b and of query head h; D <= 8 NI.  Groups of eight lanes each take
// every (THREADS / 8)th key with a running maximum and sum of their own, and are joined through
// shared memory at the end, so nothing is exchanged while keys are read.  The eight lanes split the
// head dimension (element lane + 8 i), which coalesces to whole 32-byte sectors in fp32 at any
// alignment.
template <int DT, int NI, int THREADS>
AK_D void row_by_cta(const AttnArgs& a, int b, const SeqRange& r, int t, int h, RowScratch<NI, THREADS>& sh) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int GROUPS = THREADS / 8, WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hk = h / a.G;
  const int sub = lane & 7, grp = threadIdx.x >> 3;
  const int vis = visible_keys(r, t, a.causal);

  float q[NI], o[NI];
  const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(r.begin + t) * a.qs[0] + h * a.qs[1];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int d = sub + 8 * i;
    q[i] = d < a.D ? E::to_f(qp[d]) : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, sum = 0.f;
  bool missing = false;
  for (int j = grp; j < vis; j += GROUPS) {
    const int pi = j / a.l.page_size, slot = j - pi * a.l.page_size;
    const int page = page_of(a.l, b, pi);
    if (page < 0) {
      missing = true;
      break;
    }
    const T* kp = reinterpret_cast<const T*>(a.k) + page * a.kcs[0] + hk * a.kcs[1] + slot * a.kcs[2];
    const T* vp = reinterpret_cast<const T*>(a.v) + page * a.vcs[0] + hk * a.vcs[1] + slot * a.vcs[2];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int d = sub + 8 * i;
      if (d < a.D) s = fmaf(q[i], E::to_f(kp[d]), s);
    }
    const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) s += __shfl_xor_sync(mask, s, x);
    const float mn = fmaxf(m, s);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f((m - ref) * a.scale_log2), p = exp2f((s - ref) * a.scale_log2);
    m = mn;
    sum = sum * alpha + p;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int d = sub + 8 * i;
      if (d < a.D) o[i] = fmaf(p, E::to_f(vp[d]), o[i] * alpha);
    }
  }
  missing = __syncthreads_or(missing);  // (also behind the last row's reads of what follows)

  // join the groups
  if (sub == 0) {
    sh.m[grp] = m;
    sh.l[grp] = sum;
  }
  __syncthreads();
  const float mine = lane < GROUPS ? sh.m[lane] : -INFINITY;
  const float top = warp_max(mine);
  const float ref = top == -INFINITY ? 0.f : top;
  const float total = warp_sum((lane < GROUPS ? sh.l[lane] : 0.f) * exp2f((mine - ref) * a.scale_log2));
  const float w = exp2f((m - ref) * a.scale_log2);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float x = o[i] * w;
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    x += __shfl_xor_sync(0xffffffffu, x, 16);
    if (lane < 8) sh.o[warp][sub + 8 * i] = x;
  }
  __syncthreads();
  T* op = reinterpret_cast<T*>(a.o) + (int64_t)(r.begin + t) * a.os[0] + h * a.os[1];
  for (int d = threadIdx.x; d < a.D; d += THREADS) {
    float x = 0.f;
#pragma unroll
    for (int y = 0; y < WARPS; ++y) x += sh.o[y][d];
    op[d] = E::from_f(missing ? __int_as_float(0x7fffffff) : total == 0.f ? 0.f : x / total);
  }
}

}  // namespace paged
}  // namespace ak
