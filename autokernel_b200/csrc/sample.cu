// Sampling one token per row of logits with temperature, top-k, top-p and min-p from given
// uniform numbers.  In 64 bits, over the row's alive entries (not NaN, not -inf):
//   w_i = exp((x_i - max x) / T); order: x descending, index ascending;
//   kept = the first min(k, n_p, n_m) of that order, where n_p counts the entries whose
//   predecessors' weights sum to less than p * (the weight of the first k), and n_m the w_i >= min_p;
//   token = the lowest index whose kept weights up to it sum to more than u * (the kept weight).
// T <= 0: the largest logit, lowest index.  No alive entry: -1.
//
// The kept set is always the front of the order, so it is given by a key tau and the number of
// entries equal to tau that belong to it (those of lowest index): keys are the logits' bits made
// monotone, and tau is found by bisection over counts (top-k) and weights (top-p).
#include "ak_common.cuh"

namespace ak {
namespace {

struct SampleArgs {
  const void* x;
  const float* u;
  const float *t_row, *p_row, *m_row;  // settings of each row, or null
  const int32_t* k_row;
  float t, p, m;                       // settings of all rows otherwise
  int k;
  int64_t* out;
  int64_t rows, ld;
  int vocab;
};

// Monotone key of a logit: larger logit, larger key; -0 and +0 share one; NaN and -inf are 0.
template <int DT>
struct Key;
template <>
struct Key<AK_F32> {
  using Bits = uint32_t;
  static constexpr uint32_t kLowest = 0x00800000u;  // of the lowest finite value
  static AK_D uint32_t of(uint32_t u) {
    if ((u << 1) == 0) u = 0;
    if ((u & 0x7fffffffu) > 0x7f800000u || u == 0xff800000u) return 0;
    return (u >> 31) ? ~u : u | 0x80000000u;
  }
  static AK_D float value(uint32_t k) {
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
  }
};
template <int DT>
struct Key16 {
  using Bits = uint16_t;
  static constexpr uint32_t kInf = DT == AK_F16 ? 0x7c00u : 0x7f80u;
  static constexpr uint32_t kLowest = DT == AK_F16 ? 0x0400u : 0x0080u;
  static AK_D uint32_t of(uint32_t u) {
    if ((u & 0x7fffu) == 0) u = 0;
    if ((u & 0x7fffu) > kInf || u == (kInf | 0x8000u)) return 0;
    return (u & 0x8000u) ? ~u & 0xffffu : u | 0x8000u;
  }
  static AK_D float value(uint32_t k) {
    const uint16_t b = (uint16_t)((k & 0x8000u) ? k & 0x7fffu : ~k);
    return Elem<DT>::to_f(*reinterpret_cast<const typename Elem<DT>::T*>(&b));
  }
};
template <>
struct Key<AK_F16> : Key16<AK_F16> {};
template <>
struct Key<AK_BF16> : Key16<AK_BF16> {};

template <int DT>
struct Weight {
  uint32_t top;
  double max, t;
  AK_D double operator()(uint32_t key) const {
    if (key == 0) return 0.0;
    if (key == top) return 1.0;
    return exp(((double)Key<DT>::value(key) - max) / t);
  }
};

template <int DT>
__global__ void __launch_bounds__(512) sample_kernel(const SampleArgs a) {
  using K = Key<DT>;
  const int64_t row = blockIdx.x;
  const typename K::Bits* x = reinterpret_cast<const typename K::Bits*>(a.x) + row * a.ld;
  const int n = a.vocab, tid = threadIdx.x, nt = blockDim.x;
  __shared__ double s_red[32];
  __shared__ double s_scan[512];
  __shared__ int s_ties[512];

  auto count = [&](uint32_t above) {  // entries with key > above
    int c = 0;
    for (int i = tid; i < n; i += nt) c += K::of(x[i]) > above;
    return (int64_t)block_sum_d((double)c, s_red);
  };

  uint32_t top = 0;
  for (int i = tid; i < n; i += nt) top = max(top, K::of(x[i]));
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  __syncthreads();
  if ((tid & 31) == 0) s_ties[tid >> 5] = (int)top;
  __syncthreads();
  for (int i = 0; i < nt / 32; ++i) top = max(top, (uint32_t)s_ties[i]);
  __syncthreads();
  if (top == 0) {
    if (tid == 0) a.out[row] = -1;
    return;
  }

  const float tf = a.t_row ? a.t_row[row] : a.t, pf = a.p_row ? a.p_row[row] : a.p;
  const float mf = a.m_row ? a.m_row[row] : a.m;
  const int kf = a.k_row ? a.k_row[row] : a.k;
  const bool greedy = !(tf > 0.f);
  const Weight<DT> w{top, (double)K::value(top), greedy ? 1.0 : (double)tf};
  const double p = pf, m = mf > 0.f ? fmin((double)mf, 1.0) : 0.0;
  const int64_t alive = count(0);

  // top-k: tau is the k-th largest key, `ties` of its entries are kept
  uint32_t tau = K::kLowest;
  int64_t ties = n;
  if (greedy || !(pf > 0.f)) {
    tau = top;
    ties = 1;
  } else {
    if (kf > 0 && kf < alive) {
      uint32_t lo = K::kLowest - 1, hi = top;  // count(> lo) >= k > count(> hi)
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (count(mid) >= kf) lo = mid; else hi = mid;
      }
      tau = hi;
      ties = kf - count(hi);
    }
    if (pf < 1.f) {
      auto mass = [&](uint32_t above) {  // weight of the entries with key > above
        double c = 0.0;
        for (int i = tid; i < n; i += nt) {
          const uint32_t key = K::of(x[i]);
          if (key > above) c += w(key);
        }
        return block_sum_d(c, s_red);
      };
      const double wt = w(tau);
      const double at = (double)(count(tau - 1) - count(tau));
      const double target = p * (mass(tau) + wt * fmin((double)ties, at));
      uint32_t lo = tau - 1, hi = top;  // mass(> hi) < target <= mass(> lo) or lo below tau
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (mass(mid) >= target) lo = mid; else hi = mid;
      }
      const double above = mass(hi), wh = w(hi);
      const int64_t limit = hi == tau ? ties : n;
      int64_t c = wh > 0.0 ? (int64_t)fmin(ceil((target - above) / wh), (double)n) : n;
      while (c > 1 && !(above + (double)(c - 1) * wh < target)) --c;
      while (c < n && above + (double)c * wh < target) ++c;
      tau = hi;
      ties = c < 1 ? 1 : (c < limit ? c : limit);
    }
  }

  // token: prefix sums over runs of consecutive entries, one run per thread
  const int run = (n + nt - 1) / nt;
  const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
  int eq = 0;
  for (int i = i0; i < i1; ++i) eq += K::of(x[i]) == tau;
  s_ties[tid] = eq;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < tid; ++i) before += s_ties[i];
  double sum = 0.0;
  int seen = before;
  for (int i = i0; i < i1; ++i) {
    const uint32_t key = K::of(x[i]);
    if (key < tau || (key == tau && seen++ >= ties)) continue;
    const double v = w(key);
    if (v >= m) sum += v;
  }
  s_scan[tid] = sum;
  __syncthreads();
  double start = 0.0, total = 0.0;
  for (int i = 0; i < nt; ++i) {
    if (i == tid) start = total;
    total += s_scan[i];
  }
  float uf = a.u[row];
  uf = uf > 0.f ? fminf(uf, 0.99999994f) : 0.f;
  const double goal = (double)uf * total;
  if (start <= goal && goal < start + sum) {
    double c = 0.0;
    seen = before;
    for (int i = i0; i < i1; ++i) {
      const uint32_t key = K::of(x[i]);
      if (key < tau || (key == tau && seen++ >= ties)) continue;
      const double v = w(key);
      if (v >= m) c += v;
      if (start + c > goal) {
        a.out[row] = i;
        break;
      }
    }
  }
}

}  // namespace
}  // namespace ak

using namespace ak;

extern "C" int ak_sample(const void* logits, const float* u, int64_t rows, int64_t vocab,
                         int64_t ld, int dtype, const float* temperatures, const int32_t* top_ks,
                         const float* top_ps, const float* min_ps, float temperature,
                         int32_t top_k, float top_p, float min_p, int64_t* out, void* stream) {
  AK_REQUIRE(dtype_ok(dtype), AK_ERR_DTYPE, "unsupported dtype %d", dtype);
  AK_REQUIRE(rows >= 0 && vocab > 0 && vocab < (1LL << 30) && rows < (1LL << 31) &&
                 ld >= 0,  // rows are only read, so they may overlap
             AK_ERR_SHAPE, "bad shape");
  if (rows == 0) return AK_OK;
  AK_REQUIRE(logits && u && out, AK_ERR_ARG, "null pointer");
  SampleArgs a{logits, u, temperatures, top_ps, min_ps, top_ks, temperature, top_p,
               min_p,  top_k, out, rows, ld, (int)vocab};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AK_F32: sample_kernel<AK_F32><<<(unsigned)rows, 512, 0, st>>>(a); break;
    case AK_F16: sample_kernel<AK_F16><<<(unsigned)rows, 512, 0, st>>>(a); break;
    default: sample_kernel<AK_BF16><<<(unsigned)rows, 512, 0, st>>>(a);
  }
  return launch_status("sample");
}
