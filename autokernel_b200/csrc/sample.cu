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

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

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
    const double d = ((double)Key<DT>::value(key) - max) / t;
    return d == d ? exp(d) : 0.0;  // (largest logit and temperature both infinite)
  }
};

// Cuts by bisection over keys: `count(key)` entries and `mass(key)` weight lie above a key.
// top-k: the key of the k-th entry; `ties` of its entries belong to the first k.
template <int DT, class Count>
AK_D uint32_t cut_by_count(Count count, uint32_t top, int64_t k, int64_t& ties) {
  uint32_t lo = Key<DT>::kLowest - 1, hi = top;  // count(lo) >= k > count(hi)
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (count(mid) >= k) lo = mid; else hi = mid;
  }
  ties = k - count(hi);
  return hi;
}
// top-p of the entries above tau and the first `ties` equal to it.
template <int DT, class Count, class Mass>
AK_D uint32_t cut_by_weight(Count count, Mass mass, const Weight<DT>& w, uint32_t top, uint32_t tau,
                            double p, int64_t n, int64_t& ties) {
  const double wt = w(tau);
  const double at = (double)(count(tau - 1) - count(tau));
  const double target = p * (mass(tau) + wt * fmin((double)ties, at));
  uint32_t lo = tau - 1, hi = top;  // mass(hi) < target <= mass(lo), or lo below tau
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (mass(mid) >= target) lo = mid; else hi = mid;
  }
  // the entries equal to hi whose predecessors weigh less than the target
  const double above = mass(hi), wh = w(hi);
  const int64_t limit = hi == tau ? ties : n;
  int64_t c = wh > 0.0 ? (int64_t)fmin(ceil((target - above) / wh), (double)n) : n;
  while (c > 1 && !(above + (double)(c - 1) * wh < target)) --c;
  while (c < n && above + (double)c * wh < target) ++c;
  ties = c < 1 ? 1 : (c < limit ? c : limit);
  return hi;
}

// A row of any length, read again in every pass; for rows that a cluster cannot hold.
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

  uint32_t tau = K::kLowest;
  int64_t ties = n;
  if (greedy || !(pf > 0.f)) {
    tau = top;
    ties = 1;
  } else {
    if (kf > 0 && kf < alive) tau = cut_by_count<DT>(count, top, kf, ties);
    if (pf < 1.f) {
      auto mass = [&](uint32_t above) {  // weight of the entries with key > above
        double c = 0.0;
        for (int i = tid; i < n; i += nt) {
          const uint32_t key = K::of(x[i]);
          if (key > above) c += w(key);
        }
        return block_sum_d(c, s_red);
      };
      tau = cut_by_weight<DT>(count, mass, w, top, tau, p, n, ties);
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

// ------------------------------------------------------------------ the row in a cluster
// One cluster of C CTAs per row (C up to 8), which keep it in shared memory, each thread reading only
// the 16-byte vectors it fetched, so logits come from memory once:
//   1  the largest key
//   2  (top-k or top-p) a histogram over max - x, 1536 bins of T / 48: counts, and weights as 64-bit
//      fixed point (2^-45, so sums do not depend on their order); the bin where the cut falls is
//      found by a scan, its few entries are gathered, sorted and cut exactly
//   3  kept weights per run of 32 vectors, then the run, the lane and the entry that u falls in
// Rows whose cut lies outside the bins or in a crowded bin (equal logits) are cut by bisection
// over keys instead.
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1536, kList = 1024;
constexpr int kMaxSlice = 160 * 1024;                  // bytes of a row per CTA
constexpr int kMaxRuns = kMaxSlice / 16 / 32 + kWarps;  // runs of 32 vectors
constexpr double kFixed = 35184372088832.0;            // 2^45: 2^18 weights of 1 fit 64 bits
constexpr int kMaxVocab = 1 << 18;

struct Hist {
  unsigned long long mass[kBins];
  uint32_t count[kBins];
};
struct List {
  uint32_t key[kList], idx[kList], key_sorted[kList], idx_sorted[kList];
  double weight[kList];
};
struct Shared {
  union {
    Hist h;   // this CTA's
    List list;  // the leader's, once the histograms are added up
  };
  Hist all;   // the leader's: of all CTAs
  unsigned long long rest, rest_all;  // weight outside the bins
  double run[kMaxRuns];
  double red[kWarps], total, above, target;
  unsigned long long scan[kWarps];
  uint32_t top, found, need;
  int n_list, bin, regather, bisect_k, bisect_p;
  uint32_t tau, last;  // cut: keys above tau, and those equal to it up to index `last`
};

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) sample_cluster_kernel(const SampleArgs a) {
  using K = Key<DT>;
  using Bits = typename K::Bits;
  constexpr int VEC = Elem<DT>::kVec;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Shared& lead = *cluster.map_shared_rank(&s, 0);

  const float tf = a.t_row ? a.t_row[row] : a.t, pf = a.p_row ? a.p_row[row] : a.p;
  const float mf = a.m_row ? a.m_row[row] : a.m;
  const int kf = a.k_row ? a.k_row[row] : a.k;

  // load: vectors start on 16-byte boundaries, so the first and the last may hold entries that are
  // not the row's; those become NaN, which no pass counts
  uint4* const slice = reinterpret_cast<uint4*>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
  int nv = 0, first, per;  // vectors of this thread; index of entry 0 of its first one; vectors of the CTA
  {
    const Bits* x = reinterpret_cast<const Bits*>(a.x) + row * a.ld;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(Bits));
    per = ((a.vocab + mis + VEC - 1) / VEC + C - 1) / C;
    first = (rank * per + tid) * VEC - mis;
    for (int j = tid; j < per; j += kThreads, ++nv) {
      const int i = first + nv * kThreads * VEC;
      if (i >= 0 && i + VEC <= a.vocab) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(slice + j)),
                     "l"(x + i)
                     : "memory");
      } else {
        uint4 raw = make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (i + e >= 0 && i + e < a.vocab) reinterpret_cast<Bits*>(&raw)[e] = x[i + e];
        slice[j] = raw;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  const int rounds = (per + kThreads - 1) / kThreads;
  auto index = [&](int v, int e) { return first + v * kThreads * VEC + e; };
  auto keys_of = [&](int v, uint32_t* key) {
    const uint4 raw = slice[v * kThreads + tid];
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      key[e] = VEC == 4 ? K::of(word[e]) : K::of((e & 1) ? word[e / 2] >> 16 : word[e / 2] & 0xffffu);
  };
  // f(key, index) for every entry of this thread
  auto each = [&](auto f) {
#pragma unroll 1
    for (int v = 0; v < nv; ++v) {
      uint32_t key[VEC];
      keys_of(v, key);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(key[e], index(v, e));
    }
  };

  // 1: the largest key of the row
  uint32_t top = 0;
  each([&](uint32_t key, int) { top = max(top, key); });
  top = __reduce_max_sync(0xffffffffu, top);
  if (tid == 0) {
    s.top = 0;
    s.found = 0xffffffffu;
    s.rest = 0;
    s.n_list = s.bisect_k = s.bisect_p = s.regather = 0;
  }
  __syncthreads();
  if (lane == 0) atomicMax(&s.top, top);
  cluster.sync();
  for (int i = 0; i < C; ++i) top = max(top, cluster.map_shared_rank(&s, i)->top);
  if (top == 0) {
    if (rank == 0 && tid == 0) a.out[row] = -1;
    cluster.sync();  // no CTA leaves while another may read its memory
    return;
  }

  const bool first_only = !(tf > 0.f) || !(pf > 0.f) || kf == 1;
  if (first_only) {
    uint32_t at = 0xffffffffu;
    each([&](uint32_t key, int i) {
      if (key == top) at = min(at, (uint32_t)i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0 && at != 0xffffffffu) atomicMin(&lead.found, at);
    cluster.sync();
    if (rank == 0 && tid == 0) a.out[row] = s.found;
    return;
  }

  const Weight<DT> w{top, (double)K::value(top), (double)tf};
  const double p = pf, m = mf > 0.f ? fmin((double)mf, 1.0) : 0.0;
  const bool cut_p = pf < 1.f;
  const bool cut_k = kf > 0 && kf < a.vocab;

  // bin of an entry: monotone in x, kBins when outside
  const float maxf_ = K::value(top), inv = kBins / fminf(fmaxf(32.f * tf, 16.f), 64.f);
  auto bin_of = [&](uint32_t key) {
    if (key == top) return 0;
    const float b = (maxf_ - K::value(key)) * inv;
    return b < (float)kBins ? (int)b : kBins;
  };
  // sum over the cluster, the same in every thread; a fixed order
  auto cluster_sum = [&](double v) {
    v = warp_sum_d(v);
    __syncthreads();
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int i = 0; i < kWarps; ++i) t += s.red[i];
      s.total = t;
    }
    cluster.sync();
    double t = 0.0;
    for (int i = 0; i < C; ++i) t += cluster.map_shared_rank(&s, i)->total;
    cluster.sync();
    return t;
  };

  uint32_t tau = 0, last = 0xffffffffu;
  if (cut_k || cut_p) {
    for (int i = tid; i < kBins; i += kThreads) {
      s.h.mass[i] = 0;
      s.h.count[i] = 0;
    }
    __syncthreads();
    double rest = 0.0;
    each([&](uint32_t key, int) {
      if (key == 0) return;
      const int b = bin_of(key);
      if (b < kBins) {
        if (cut_k) atomicAdd(&s.h.count[b], 1u);
        if (cut_p) atomicAdd(&s.h.mass[b], __double2ull_rn(w(key) * kFixed));
      } else if (cut_p) {
        rest += w(key);
      }
    });
    if (cut_p) {
      rest = warp_sum_d(rest);
      if (lane == 0) atomicAdd(&s.rest, __double2ull_rn(rest * kFixed));
    }
    cluster.sync();
    // each CTA adds up its share of the bins and hands it to the leader
    const int share = kBins / C;
    for (int i = rank * share + tid; i < (rank + 1) * share; i += kThreads) {
      unsigned long long ms = 0;
      uint32_t cs = 0;
      for (int c = 0; c < C; ++c) {
        const Shared& o = *cluster.map_shared_rank(&s, c);
        if (cut_p) ms += o.h.mass[i];
        if (cut_k) cs += o.h.count[i];
      }
      lead.all.mass[i] = ms;
      lead.all.count[i] = cs;
    }
    if (rank == 0 && tid == 0) {
      unsigned long long t = 0;
      for (int c = 0; c < C; ++c) t += cluster.map_shared_rank(&s, c)->rest;
      s.rest_all = t;
    }
    cluster.sync();

    // sums before this thread's bins (leader)
    constexpr int PER = kBins / kThreads;
    auto scan = [&](unsigned long long v) {
      unsigned long long inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      __syncthreads();
      if (lane == 31) s.scan[warp] = inc;
      __syncthreads();
      unsigned long long before = inc - v;
      for (int i = 0; i < warp; ++i) before += s.scan[i];
      return before;
    };
    // the entries of the leader's bin, of all CTAs, sorted into its list; too many: *crowded
    auto gather = [&](int* crowded) {
      const int bin = lead.bin;
      each([&](uint32_t key, int i) {
        if (key == 0 || bin_of(key) != bin) return;
        const int at = atomicAdd(&lead.n_list, 1);
        if (at < kList) {
          lead.list.key[at] = key;
          lead.list.idx[at] = i;
        }
      });
      cluster.sync();
      if (rank == 0) {
        List& t = s.list;
        const int n = s.n_list;
        if (n > kList) {
          if (tid == 0) *crowded = 1;
        } else {
          for (int i = tid; i < n; i += kThreads) {
            const uint32_t key = t.key[i], idx = t.idx[i];
            int before = 0;
            for (int j = 0; j < n; ++j) before += t.key[j] > key || (t.key[j] == key && t.idx[j] < idx);
            t.key_sorted[before] = key;
            t.idx_sorted[before] = idx;
            t.weight[before] = w(key);
          }
        }
        __syncthreads();
      }
    };

    // The leader's decisions are read by the others only behind the next cluster.sync, and a field is
    // written again only behind a later one.
    bool by_bisection = false;
    if (cut_k) {
      if (rank == 0) {
        uint32_t c[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += c[i] = s.all.count[tid * PER + i];
        uint32_t before = (uint32_t)scan(mine);
        if (tid == kThreads - 1 && before + mine < (uint32_t)kf) s.bisect_k = 1;  // outside the bins
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (before < (uint32_t)kf && before + c[i] >= (uint32_t)kf) {
            s.bin = tid * PER + i;
            s.need = kf - before;
          }
          before += c[i];
        }
      }
      cluster.sync();
      if (!lead.bisect_k) {
        cluster.sync();  // (gather may raise it)
        gather(&s.bisect_k);
      }
      if (rank == 0 && !s.bisect_k) {  // the first s.need of the list are kept
        if (cut_p) {
          // weight of the first k: the bins above and the kept entries
          unsigned long long ms = 0;
          for (int i = tid; i < s.bin; i += kThreads) ms += s.all.mass[i];
          double d = (double)ms / kFixed;
          for (int i = tid; i < (int)s.need; i += kThreads) d += s.list.weight[i];
          d = warp_sum_d(d);
          if (lane == 0) s.red[warp] = d;
          __syncthreads();
          if (tid == 0) {
            double t = 0.0;
            for (int i = 0; i < kWarps; ++i) t += s.red[i];
            s.target = p * t;
          }
        }
        if (tid == 0) {
          s.tau = s.list.key_sorted[s.need - 1];
          s.last = s.list.idx_sorted[s.need - 1];
        }
        __syncthreads();
      }
      cluster.sync();
      by_bisection = lead.bisect_k;
    }
    if (cut_p && !by_bisection) {
      if (rank == 0) {
        const int k_bin = cut_k ? s.bin : kBins;  // its list is there already
        unsigned long long c[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += c[i] = s.all.mass[tid * PER + i];
        unsigned long long before = scan(mine);
        if (!cut_k && tid == kThreads - 1) {
          const double in = (double)(before + mine) / kFixed;
          s.target = p * (in + (double)s.rest_all / kFixed);
          if (in < s.target) s.bisect_p = 1;  // outside the bins
        }
        __syncthreads();
        const double target = s.target;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int b = tid * PER + i;
          const double lo = (double)before / kFixed, hi = (double)(before + c[i]) / kFixed;
          if (b < k_bin && lo < target && hi >= target) {
            s.bin = b;
            s.above = lo;
            s.need = kList;
            s.n_list = 0;
            s.regather = 1;
          }
          if (b == k_bin && lo < target) s.above = lo;
          before += c[i];
        }
      }
      cluster.sync();
      const bool again = lead.regather && !lead.bisect_p;
      cluster.sync();  // (gather may raise it)
      if (again) gather(&s.bisect_p);
      if (rank == 0 && !s.bisect_p) {
        if (warp == 0) {
          // entries kept: those whose predecessors weigh less than the target
          const int n = min(s.n_list, (int)s.need);
          double run = s.above;
          int kept = 0;
          for (int base = 0; base < n; base += 32) {
            double inc = base + lane < n ? s.list.weight[base + lane] : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += y;
            }
            const double prev = __shfl_up_sync(0xffffffffu, inc, 1);
            const bool in = base + lane < n && run + (lane ? prev : 0.0) < s.target;
            kept += __popc(__ballot_sync(0xffffffffu, in));
            run += __shfl_sync(0xffffffffu, inc, 31);
          }
          if (lane == 0) {
            kept = max(kept, 1);
            s.tau = s.list.key_sorted[kept - 1];
            s.last = s.list.idx_sorted[kept - 1];
          }
        }
        __syncthreads();
      }
      cluster.sync();
      by_bisection = lead.bisect_p;
    }
    if (!by_bisection) {
      tau = lead.tau;
      last = lead.last;
    } else {
      auto count = [&](uint32_t above) {
        int c = 0;
        each([&](uint32_t key, int) { c += key > above; });
        return (int64_t)cluster_sum((double)c);
      };
      auto mass = [&](uint32_t above) {
        double c = 0.0;
        each([&](uint32_t key, int) {
          if (key > above) c += w(key);
        });
        return cluster_sum(c);
      };
      const int64_t alive = count(0);
      int64_t ties = a.vocab;
      tau = K::kLowest;
      if (cut_k && kf < alive) tau = cut_by_count<DT>(count, top, kf, ties);
      if (cut_p) tau = cut_by_weight<DT>(count, mass, w, top, tau, p, a.vocab, ties);
      int lo = 0, hi = a.vocab;  // entries equal to tau below index lo: fewer than ties; below hi: enough
      while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        int c = 0;
        each([&](uint32_t key, int i) { c += key == tau && i < mid; });
        if ((int64_t)cluster_sum((double)c) >= ties) hi = mid; else lo = mid;
      }
      last = hi - 1;
    }
  }

  // 3: kept weights up to and with each run of 32 vectors (a warp's v-th), in index order
  auto kept = [&](uint32_t key, int i) {
    if (key == 0 || key < tau || (key == tau && (uint32_t)i > last)) return 0.0;
    const double x = w(key);
    return x >= m ? x : 0.0;
  };
  const int most = (rounds * kWarps + 31) / 32 * 32;  // runs, padded to whole warps
  for (int i = tid; i < most; i += kThreads) s.run[i] = 0.0;
  __syncthreads();
#pragma unroll 1
  for (int v = 0; v < rounds; ++v) {
    double t = 0.0;
    if (v < nv) {
      uint32_t key[VEC];
      keys_of(v, key);
#pragma unroll
      for (int e = 0; e < VEC; ++e) t += kept(key[e], index(v, e));
    }
    t = warp_sum_d(t);
    if (lane == 0) s.run[v * kWarps + warp] = t;
  }
  __syncthreads();
  if (warp == 0) {
    double carry = 0.0;
    for (int base = 0; base < most; base += 32) {
      double inc = s.run[base + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      inc += carry;
      s.run[base + lane] = inc;
      carry = __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) s.total = carry;
  }
  cluster.sync();
  double start = 0.0, total = 0.0;
  for (int i = 0; i < C; ++i) {
    if (i == rank) start = total;
    total += cluster.map_shared_rank(&s, i)->total;
  }
  float uf = a.u[row];
  uf = uf > 0.f ? fminf(uf, 0.99999994f) : 0.f;
  const double goal = (double)uf * total;
  // the CTAs' stretches [start, start + total) share their borders' very values: one holds the goal
  if (warp == 0 && start <= goal && goal < start + s.total) {
    double here = goal - start;
    int run = -1;
    for (int base = 0; base < most && run < 0; base += 32) {
      const unsigned hit = __ballot_sync(0xffffffffu, s.run[base + lane] > here);
      if (hit) run = base + __ffs(hit) - 1;
    }
    if (run < 0) {  // (by rounding alone) the last run with any weight
      run = 0;
      for (int i = 1; i < most; ++i)
        if (s.run[i] > s.run[i - 1]) run = i;
    }
    here -= run ? s.run[run - 1] : 0.0;
    // this warp reads the run's vectors in the place of the warp that owns them
    const int j = run * 32 + lane, v0 = j * VEC + first - tid * VEC;
    double part[VEC], t = 0.0;
    const uint4 raw = j < per ? slice[j] : make_uint4(~0u, ~0u, ~0u, ~0u);
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t key = VEC == 4 ? K::of(word[e]) : K::of((e & 1) ? word[e / 2] >> 16 : word[e / 2] & 0xffffu);
      t += part[e] = kept(key, v0 + e);
    }
    double inc = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const unsigned some = __ballot_sync(0xffffffffu, t > 0.0);
    const unsigned hit = __ballot_sync(0xffffffffu, t > 0.0 && inc > here);
    if (lane == (hit ? __ffs(hit) - 1 : 31 - __clz(some))) {
      here -= inc - t;
      double c = 0.0;
      int at = 0;
      bool done = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (done || !(part[e] > 0.0)) continue;
        c += part[e];
        at = e;
        done = c > here;
      }
      a.out[row] = v0 + at;
    }
  }
  cluster.sync();  // no CTA leaves while another may read its memory
}

template <int DT>
int run_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int VEC = Elem<DT>::kVec;
  const int64_t vectors = (a.vocab + VEC - 1) / VEC + 1;
  const int sms = device_info().sm_count;
  auto slice = [&](int c) { return (vectors + c - 1) / c * 16; };
  // Larger clusters while a slice is large enough to keep a second CTA off the SM, or while SMs would
  // stay empty and every thread still has a vector.
  int c = 1;
  while (c < 8 && (slice(c) > 48 * 1024 || (a.rows * c < sms && slice(c) > kThreads * 16))) c *= 2;
  if (slice(c) > kMaxSlice || a.vocab > kMaxVocab) {
    sample_kernel<DT><<<(unsigned)a.rows, 512, 0, st>>>(a);
    return launch_status("sample");
  }
  constexpr size_t fixed = (sizeof(Shared) + 15) / 16 * 16;
  const cudaError_t attr = smem_optin<sample_cluster_kernel<DT>>((int)(fixed + kMaxSlice));
  AK_REQUIRE(attr == cudaSuccess, AK_ERR_LAUNCH, "sample smem attribute: %s", cudaGetErrorString(attr));
  AK_REQUIRE(a.rows * c < (1LL << 31), AK_ERR_SHAPE, "too many rows");
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = c;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = fixed + (size_t)slice(c);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_cluster_kernel<DT>, a);
  AK_REQUIRE(e == cudaSuccess, AK_ERR_LAUNCH, "sample: launch failed: %s", cudaGetErrorString(e));
  return AK_OK;
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
    case AK_F32: return run_sample<AK_F32>(a, st);
    case AK_F16: return run_sample<AK_F16>(a, st);
    default: return run_sample<AK_BF16>(a, st);
  }
}
