// Sampling one token per row of logits with temperature, top-k, top-p and min-p from given
// uniform numbers.  In 64 bits, over the row's alive entries (not NaN, not -inf):
//   w_i = exp((x_i - max x) / T); order: x descending, index ascending;
//   kept = the first min(k, n_p, n_m) of that order, where n_p counts the entries whose
//   predecessors' weights sum to less than p * (the weight of the first k), and n_m the w_i >= min_p;
//   token = the lowest index whose kept weights up to it sum to more than u * (the kept weight).
// T <= 0: the largest logit, lowest index.  No alive entry: -1.  With a largest logit of +inf only
// the entries equal to it are alive.
//
// The kept set is the front of the order, so it is given by the rank of its last entry: a 64-bit
// number, the logit's bits made monotone above the inverted index.
#include "ak_common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace ak {
namespace {

using u64 = unsigned long long;

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

struct Settings {
  float t, p;
  double m;  // smallest weight that is kept
  int k;
  double u;
  bool first_only;
};
AK_D Settings settings_of(const SampleArgs& a, int64_t row) {
  Settings s;
  s.t = a.t_row ? a.t_row[row] : a.t;
  s.p = a.p_row ? a.p_row[row] : a.p;
  s.k = a.k_row ? a.k_row[row] : a.k;
  const float m = a.m_row ? a.m_row[row] : a.m, u = a.u[row];
  s.m = m > 0.f ? fmin((double)m, 1.0) : 0.0;
  s.u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  s.first_only = !(s.t > 0.f) || !(s.p > 0.f) || s.k == 1;
  if (s.k <= 0 || s.k >= a.vocab) s.k = 0;
  return s;
}

// Alive entries are floats above -inf; a dead one is NaN or -inf.
AK_D bool alive(float x) { return x > -INFINITY; }
// Monotone bits of an alive logit, never 0; -0 and +0 are one.
AK_D uint32_t key_of(float x) {
  const uint32_t u = x == 0.f ? 0u : __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
AK_D float value_of(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
AK_D u64 rank_of(float x, int i) { return (u64)key_of(x) << 32 | (uint32_t)~i; }
constexpr u64 kAll = 1ull << 32;  // below the rank of every alive entry

// Sums over a row of any length, one CTA, the row read again in every pass: for rows that a cluster
// cannot hold.  The cuts are found by bisection over ranks.
template <int DT>
__global__ void __launch_bounds__(512) sample_kernel(const SampleArgs a) {
  using E = Elem<DT>;
  const int64_t row = blockIdx.x;
  const typename E::T* x = reinterpret_cast<const typename E::T*>(a.x) + row * a.ld;
  const int n = a.vocab, tid = threadIdx.x, nt = blockDim.x;
  __shared__ double s_red[32], s_scan[512];
  __shared__ u64 s_top;
  const Settings set = settings_of(a, row);
  if (tid == 0) s_top = 0;
  __syncthreads();
  u64 top = 0;  // the first entry's rank
  for (int i = tid; i < n; i += nt) {
    const float f = E::to_f(x[i]);
    if (alive(f)) top = max(top, rank_of(f, i));
  }
  atomicMax(&s_top, top);
  __syncthreads();
  top = s_top;
  if (top == 0 || set.first_only) {
    if (tid == 0) a.out[row] = top ? (int64_t)(uint32_t)~(uint32_t)top : -1;
    return;
  }
  const float max_ = value_of((uint32_t)(top >> 32));
  const double rate = 1.4426950408889634 / (double)set.t;
  auto w = [&](float f) {
    return f == max_ ? 1.0 : max_ == INFINITY ? 0.0 : exp2(((double)f - (double)max_) * rate);
  };
  auto count = [&](u64 from) {  // entries of rank `from` and above
    int c = 0;
    for (int i = tid; i < n; i += nt) {
      const float f = E::to_f(x[i]);
      c += alive(f) && rank_of(f, i) >= from;
    }
    return block_sum_d((double)c, s_red);
  };
  auto mass = [&](u64 from) {
    double c = 0.0;
    for (int i = tid; i < n; i += nt) {
      const float f = E::to_f(x[i]);
      if (alive(f) && rank_of(f, i) >= from) c += w(f);
    }
    return block_sum_d(c, s_red);
  };
  u64 least = kAll;  // the smallest rank that is kept
  if (set.k && count(least) > (double)set.k) {
    u64 lo = kAll, hi = top;  // count(lo) > k >= count(hi)
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      if (count(mid) > (double)set.k) lo = mid; else hi = mid;
    }
    least = hi;
  }
  if (set.p < 1.f) {
    // the smallest rank above which less than the target lies
    const double target = (double)set.p * mass(least);
    u64 lo = least - 1, hi = top;  // mass above lo >= target (or nothing is left), above hi less
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      if (mass(mid + 1) >= target) lo = mid; else hi = mid;
    }
    least = max(least, hi);
  }
  // token: sums over runs of consecutive entries, one run per thread
  const int run = (n + nt - 1) / nt;
  const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
  auto kept = [&](int i) {
    const float f = E::to_f(x[i]);
    if (!alive(f) || rank_of(f, i) < least) return 0.0;
    const double v = w(f);
    return v >= set.m ? v : 0.0;
  };
  double sum = 0.0;
  for (int i = i0; i < i1; ++i) sum += kept(i);
  s_scan[tid] = sum;
  __syncthreads();
  double start = 0.0, total = 0.0;
  for (int i = 0; i < nt; ++i) {
    if (i == tid) start = total;
    total += s_scan[i];
  }
  const double goal = set.u * total;
  if (start <= goal && goal < start + sum) {
    double c = 0.0;
    for (int i = i0; i < i1; ++i) {
      c += kept(i);
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
//   1  the largest logit
//   2  top-k: a histogram of counts over max - x (1535 bins of T / 48 and one for what lies beyond)
//      gives the bin that holds the k-th entry; its entries, when they are few, are gathered,
//      sorted and cut, and what is not kept dies.  A crowded bin is divided again by the bits of the
//      rank.
//   3  top-p: what top-k left, when it is few, is gathered and sorted at once.  Otherwise
//      the histogram of counts and mean places tells a small stretch of logits that holds the cut;
//      one pass sums every weight exactly (64-bit floating point above and below the stretch, fixed
//      point, 2^-45, in 1536 bins of the stretch, where no order of additions matters), and the
//      stretch is cut like top-k's bin.  A cut outside of the stretch costs one more pass.
//   4  kept weights per run of 32 vectors, then the run, the lane and the entry that u falls in
//
// Bound by 64-bit exponentials and the passes' synchronisation rather than by memory: 192 rows of 131072
// fp32 logits, top-p 0.9, take 296 us (341 GB/s of logits; a CTA's sums of 64-bit weights are a quarter of it,
// the histograms' merges and the leader's searches a third); 256 rows of 32000 in bf16 with settings of
// their own 78 us; one row with top-k and top-p 20 us, about ten cluster barriers and a launch.  256 rows of
// 32000: temperature alone 36 us, top-k 50 34 us, greedy 9.
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1536, kList = 128, kNear = 2048;
constexpr int kMaxSlice = 160 * 1024;                   // bytes of a row per CTA
constexpr int kMaxRuns = kMaxSlice / 16 / 32 + kWarps;  // runs of 32 vectors
constexpr double kFixed = 35184372088832.0;             // 2^45: 2^18 weights of 1 fit 64 bits
constexpr int kMaxVocab = 1 << 18;

// A 64-bit atomic addition in shared memory takes about 70 cycles a warp (measured, without
// conflicts), a 32-bit one 0.75: fixed-point weights (up to 2^45) are added in three digits of 15
// bits, whose sums over a slice (at most 2^17 entries) fit 32 bits.
struct Bins {
  uint32_t digit[3][kBins], count[kBins];
};
struct Shared {
  Bins h;  // this CTA's; then, in the leader's, of all CTAs with the weight in digits 0 and 1
  u64 list[kList], sorted[kList];
  double weight[kList];
  uint32_t near[kNear];  // this CTA's entries (numbers within the slice) in top-p's stretch
  int n_near;
  double run[kMaxRuns];
  double red[kWarps], total, above_w, below_w;
  u64 scan[kWarps], scan2[kWarps];
  u64 hi, lo;  // largest and smallest rank of this CTA's entries in the bin
  uint32_t found;
  float top[kWarps], max_;
  // the leader's decisions
  u64 above, goal, cut;  // what lies above the bin; where the place is; its rank
  double real_goal;      // top-p's, before it is rounded up
  uint32_t in_bin;
  int bin, n_list, next;
  float f_hi, f_lo;  // the stretch that holds top-p's cut
};
enum Step { kCount, kWeigh, kSums, kDivide, kGather };

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) sample_cluster_kernel(const __grid_constant__ SampleArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VEC = E::kVec;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  uint4* const slice = reinterpret_cast<uint4*>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Shared& lead = *cluster.map_shared_rank(&s, 0);
  auto peer = [&](int c) -> Shared& { return *cluster.map_shared_rank(&s, c); };
  auto sync = [&] {
    if (C > 1) cluster.sync(); else __syncthreads();
  };

  // load: vectors start on 16-byte boundaries, so the first and the last may hold entries that are
  // not the row's; those become NaN, which is dead
  int nv = 0, first, per;  // this thread's vectors; index of its first entry; the CTA's vectors
  {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
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
          if (i + e >= 0 && i + e < a.vocab) reinterpret_cast<T*>(&raw)[e] = x[i + e];
        slice[j] = raw;
      }
    }
    if (tid == 0) s.found = 0xffffffffu;
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  const Settings set = settings_of(a, row);
  const int rounds = (per + kThreads - 1) / kThreads;
  auto unpack = [](const uint4& raw, float* f) {
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = E::to_f(t[e]);
  };

  // 1: the largest logit (a maximum skips NaN)
  float max_ = -INFINITY;
#pragma unroll 2
  for (int v = 0; v < nv; ++v) {
    const uint4 raw = slice[v * kThreads + tid];
    float f[VEC];
    unpack(raw, f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) max_ = fmaxf(max_, f[e]);
  }
  max_ = warp_max(max_);
  if (lane == 0) s.top[warp] = max_;
  __syncthreads();
  max_ = warp_max(s.top[lane & (kWarps - 1)]);
  if (C > 1) {
    if (tid == 0) s.max_ = max_;
    cluster.sync();
    for (int c = 0; c < C; ++c) max_ = fmaxf(max_, peer(c).max_);
  }
  if (!alive(max_)) {
    if (rank == 0 && tid == 0) a.out[row] = -1;
    if (C > 1) cluster.sync();  // no CTA leaves while another may read its memory
    return;
  }

  // The code below is kept small (each pass exists once, and what few entries need runs in a loop of
  // its own): a row passes through it once, and waiting for instructions cost more than the work.
  auto index = [&](int v, int e) { return first + v * kThreads * VEC + e; };
  auto load = [&](int v, float* f) {
    const uint4 raw = slice[v * kThreads + tid];
    unpack(raw, f);
  };
  auto entry = [&](int j, int e) {  // entry e of the CTA's vector j
    return E::to_f(reinterpret_cast<const T*>(slice)[j * VEC + e]);
  };
  // every entry becomes value(entry, index): -inf to die
  auto kill = [&](auto value) {
#pragma unroll 1
    for (int v = 0; v < nv; ++v) {
      float f[VEC];
      load(v, f);
      uint4 raw;
#pragma unroll
      for (int e = 0; e < VEC; ++e) reinterpret_cast<T*>(&raw)[e] = E::from_f(value(f[e], index(v, e)));
      slice[v * kThreads + tid] = raw;
    }
  };
  if (max_ == INFINITY) {  // only the infinite entries count, all alike
    kill([](float f, int) { return f == INFINITY ? 0.f : -INFINITY; });
    max_ = 0.f;
  }

  if (set.first_only) {
    uint32_t at = 0xffffffffu;
#pragma unroll 1
    for (int v = 0; v < nv; ++v) {
      float f[VEC];
      load(v, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (f[e] == max_) at = min(at, (uint32_t)index(v, e));
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0 && at != 0xffffffffu) atomicMin(&lead.found, at);
    sync();
    if (rank == 0 && tid == 0) a.out[row] = s.found;
    return;
  }

  const double rate = 1.4426950408889634 / (double)set.t, top_d = max_;
  auto w = [&](float f) { return exp2(((double)f - top_d) * rate); };
  // an entry of weight w to bin b; round(w 2^45) is in the low bits of a sum with 2^52
  auto add = [&](int b, double w) {
    const u64 x = __double_as_longlong(fma(w, kFixed, 4503599627370496.0)) - 0x4330000000000000ll;
    atomicAdd(&s.h.count[b], 1u);
    atomicAdd(&s.h.digit[0][b], (uint32_t)x & 0x7fffu);
    atomicAdd(&s.h.digit[1][b], (uint32_t)(x >> 15) & 0x7fffu);
    atomicAdd(&s.h.digit[2][b], (uint32_t)(x >> 30));
  };
  // place of an entry in units of a bin, monotone in x; entries beyond the bins share the last one
  const float per_bin = (kBins - 1) / fminf(fmaxf(32.f * set.t, 16.f), 64.f);
  auto units = [&](float f) { return fminf(__fmul_rn(__fsub_rn(max_, f), per_bin), (float)(kBins - 1)); };
  // kept: entries above `cut_f`, and those equal to it up to index `cut_i`; at first all alive ones
  float cut_f = -INFINITY;
  int cut_i = -1;
  auto keep = [&](float f, int i) { return f > cut_f || (f == cut_f && i <= cut_i); };

  bool summed = false;  // s.run has the weights above f_hi, where top-p's cut is not
  float f_hi = 0.f, f_lo = 0.f;
#pragma unroll 1
  for (int top_p = 0; top_p < 2; ++top_p) {
    if (top_p ? !(set.p < 1.f) : !set.k) continue;
    // What top-k left for top-p, when it is few, is one bin.
    const bool whole = top_p && set.k && set.k <= kList;
    enum { kUnits, kStretch, kRanks, kOne } by = whole ? kOne : kUnits;
    float scale = 0.f;
    u64 hi = 0, lo = 0;
    int shift = 0, bin = 0;
    Step step = kCount;
    bool estimate = top_p;  // the first histogram tells where to look
    auto bin_of = [&](float f, int i) {  // of an alive entry, or -1
      if (by == kUnits) return (int)units(f);
      if (by == kOne) return 0;
      if (!(f <= f_hi && f >= f_lo)) return -1;
      if (by == kStretch) return min((int)((f_hi - f) * scale), kBins - 1);
      const u64 r = rank_of(f, i);
      return r >= lo && r <= hi ? (int)((hi - r) >> shift) : -1;
    };
    auto add_all = [&] {
#pragma unroll 1
      for (int v = 0; v < nv; ++v)
#pragma unroll 1
        for (int e = 0; e < VEC; ++e) {
          const float f = entry(v * kThreads + tid, e);
          const int b = alive(f) ? bin_of(f, index(v, e)) : -1;
          if (b >= 0) add(b, w(f));
        }
    };
    if (whole) {
      if (rank == 0 && tid == 0) s.n_list = 0;
      sync();
    }
    while (!whole) {
      for (int i = tid; i < kBins; i += kThreads)
        s.h.digit[0][i] = s.h.digit[1][i] = s.h.digit[2][i] = s.h.count[i] = 0;
      if (tid == 0 && step == kSums) s.n_near = 0;
      if (tid == 0 && estimate) {  // all of the row, should no bin of the estimate weigh anything
        s.f_hi = max_;
        s.f_lo = -3.4028235e38f;
      }
      __syncthreads();
      if (step == kSums) {  // every weight: above the stretch, in its bins, below it
        double below = 0.0;
#pragma unroll 1
        for (int v = 0; v < rounds; ++v) {
          double above = 0.0;
          if (v < nv) {
            float f[VEC];
            load(v, f);
            unsigned some = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {  // no branch: the chains of operations overlap
              const double x = w(f[e]);
              if (f[e] > f_hi) above += x;
              if (f[e] < f_lo) below += x;
              some |= (unsigned)(f[e] <= f_hi && f[e] >= f_lo) << e;
            }
            while (some) {  // their bins come later, from all threads at once
              const int at = atomicAdd(&s.n_near, 1);
              if (at < kNear) s.near[at] = (v * kThreads + tid) * VEC + __ffs(some) - 1;
              some &= some - 1;
            }
          }
          above = warp_sum_d(above);
          if (lane == 0) s.run[v * kWarps + warp] = above;
        }
        if (!(below >= 0.0)) {  // T = inf: a dead entry's x is NaN, any other's 1 (a test of each x cost 2%)
          below = 0.0;
#pragma unroll 1
          for (int j = tid; j < nv * kThreads; j += kThreads)
#pragma unroll 1
            for (int e = 0; e < VEC; ++e) below += alive(entry(j, e)) && entry(j, e) < f_lo;
        }
        below = warp_sum_d(below);
        if (lane == 0) s.red[warp] = below;
        __syncthreads();
        if (s.n_near <= kNear) {
          for (int i = tid; i < s.n_near; i += kThreads) {
            const float f = entry(s.near[i] / VEC, s.near[i] % VEC);
            add(bin_of(f, 0), w(f));
          }
        } else {
          add_all();
        }
        if (warp == 0) {
          double t = 0.0;
          for (int i = lane; i < rounds * kWarps; i += 32) t += s.run[i];
          t = warp_sum_d(t);
          const double y = warp_sum_d(lane < kWarps ? s.red[lane] : 0.0);
          if (lane == 0) {
            s.above_w = t;
            s.below_w = y;
          }
        }
      } else if (step == kCount && by == kUnits) {
#pragma unroll 1
        for (int v = 0; v < nv; ++v) {
          float f[VEC];
          load(v, f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (!alive(f[e])) continue;
            const float u = units(f[e]);
            const int b = (int)u;
            atomicAdd(&s.h.count[b], 1u);
            if (top_p) atomicAdd(&s.h.digit[0][b], (uint32_t)((u - (float)b) * 256.f));  // where in the bin
          }
        }
      } else {
        add_all();
      }
      // the leader's bins from every CTA's; each CTA adds up its share of them
      sync();
      const int share = kBins / C;
      const bool counts = step == kCount && by == kUnits;  // (digit 0 is a sum of places then)
      if (C > 1 || !counts) {
        for (int i = rank * share + tid; i < (rank + 1) * share; i += kThreads) {
          u64 ms = 0;
          uint32_t cs = 0;
#pragma unroll 4
          for (int c = 0; c < C; ++c) {
            const Bins& h = peer(c).h;
            cs += h.count[i];
            if (top_p) ms += h.digit[0][i];
            if (!counts) ms += ((u64)h.digit[1][i] << 15) + ((u64)h.digit[2][i] << 30);
          }
          lead.h.count[i] = cs;
          lead.h.digit[0][i] = (uint32_t)ms;
          lead.h.digit[1][i] = (uint32_t)(ms >> 32);
        }
      }
      sync();
      // The leader's decision, read by the others behind the next sync and changed behind a later one:
      // the bin where the goal (a number of entries, or fixed-point weight) is reached.
      if (rank == 0) {
        constexpr int PER = kBins / kThreads;
        u64 c[PER], mine = 0, inc, above = 0, goal, all = 0;
        double real = 0.0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int b = tid * PER + i;
          if (estimate) {
            // as if a bin's entries all were at their mean place
            const double n = s.h.count[b], mean = n > 0.0 ? (s.h.digit[0][b] / n + 0.5) / 256.0 : 0.0;
            c[i] = (u64)(n * exp2(-(b + mean) / per_bin * rate) * kFixed);
          } else {
            c[i] = !top_p ? s.h.count[b] : s.h.digit[0][b] | (u64)s.h.digit[1][b] << 32;
          }
          mine += c[i];
        }
        inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        if (lane == 31) s.scan[warp] = inc;
        __syncthreads();
        u64 before = inc - mine;
        for (int i = 0; i < kWarps; ++i) {
          if (i < warp) before += s.scan[i];
          all += s.scan[i];
        }
        if (by == kRanks) {
          above = s.above;
          goal = s.goal;
          real = s.real_goal;
        } else if (!top_p) {
          goal = min((u64)set.k, all);
        } else {
          double beside = 0.0;
          if (step == kSums) {
            for (int i = 0; i < C; ++i) beside += peer(i).above_w;
            above = (u64)(beside * kFixed);
            for (int i = 0; i < C; ++i) beside += peer(i).below_w;
          }
          real = (double)set.p * (beside * kFixed + (double)all);
          goal = max((u64)ceil(real), 1ull);
        }
        __syncthreads();  // everyone has read s.above and s.goal
        before += above;
        // With bins of w times T, entries about their mean place weigh up to w^2 / 8 more than at it
        // and the places' rounding moves them by up to w / 512: 1e-4 of all at w = 1 / 48.
        const double wide = 1.0 / ((double)per_bin * set.t);
        const double slack = wide * (0.5 * wide + 1.0 / 256.0) * (double)all;
        const u64 goal0 = (u64)max((double)goal - slack, 1.0);
        const u64 goal1 = min((u64)min((double)goal + slack, (double)all), all);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int b = tid * PER + i;
          const u64 up_to = before + c[i];
          if (!estimate) {
            if (before < goal && up_to >= goal) {
              s.above = before;
              s.bin = b;
              s.in_bin = s.h.count[b];
            }
          } else {
            if (before < goal0 && up_to >= goal0) s.f_hi = b == 0 ? max_ : max_ - b / per_bin;
            if (before < goal1 && up_to >= goal1) s.f_lo = b == kBins - 1 ? -3.4028235e38f : max_ - (b + 1) / per_bin;
          }
          before = up_to;
        }
        __syncthreads();
        if (tid == 0) {
          s.goal = goal;
          s.real_goal = real;
          s.n_list = 0;
          s.next = estimate                                 ? kSums
                   : goal <= above || goal > above + all    ? kWeigh  // the estimate was off
                   : s.in_bin <= (uint32_t)kList            ? kGather
                                                            : kDivide;
        }
      }
      sync();
      step = (Step)lead.next;
      bin = lead.bin;
      estimate = false;
      if (step == kGather) break;
      if (step == kSums) {
        f_hi = lead.f_hi;
        f_lo = lead.f_lo;
        scale = (float)kBins / fmaxf(f_hi - f_lo, 1e-30f);
        by = kStretch;
        summed = true;
      } else if (step == kWeigh) {
        by = kUnits;
        summed = false;
      } else {  // kDivide: the bin's range of ranks
        u64 a_hi = 0, a_lo = ~0ull;
#pragma unroll 1
        for (int v = 0; v < nv; ++v)
#pragma unroll 1
          for (int e = 0; e < VEC; ++e) {
            const float f = entry(v * kThreads + tid, e);
            if (!alive(f) || bin_of(f, index(v, e)) != bin) continue;
            const u64 r = rank_of(f, index(v, e));
            a_hi = max(a_hi, r);
            a_lo = min(a_lo, r);
          }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          a_hi = max(a_hi, __shfl_xor_sync(0xffffffffu, a_hi, o));
          a_lo = min(a_lo, __shfl_xor_sync(0xffffffffu, a_lo, o));
        }
        if (lane == 0) {
          s.scan[warp] = a_hi;
          s.scan2[warp] = a_lo;
        }
        __syncthreads();
        if (tid == 0) {
          for (int i = 1; i < kWarps; ++i) {
            a_hi = max(a_hi, s.scan[i]);
            a_lo = min(a_lo, s.scan2[i]);
          }
          s.hi = a_hi;
          s.lo = a_lo;
        }
        sync();
        hi = 0;
        lo = ~0ull;
        for (int c = 0; c < C; ++c) {
          hi = max(hi, peer(c).hi);
          lo = min(lo, peer(c).lo);
        }
        if (!summed) {  // (the stretch stays as it is)
          f_hi = value_of((uint32_t)(hi >> 32));
          f_lo = value_of((uint32_t)(lo >> 32));
        }
        by = kRanks;
        shift = max(64 - __clzll((long long)(hi - lo)) - 10, 0);  // at most 1024 bins
        step = top_p ? kWeigh : kCount;
      }
    }
    // the bin's few entries, to the leader's list; few others pass the first comparison
    const float g_hi = by == kOne ? INFINITY : by != kUnits ? f_hi : max_ - (bin - 0.5f) / per_bin;
    const float g_lo = by == kOne || (by == kUnits && bin == kBins - 1) ? -INFINITY
                       : by != kUnits                                   ? f_lo
                                                                        : max_ - (bin + 1.5f) / per_bin;
    auto offer = [&](int j, int e) {
      const float f = entry(j, e);
      const int i = first + (j - tid) * VEC + e;
      if (bin_of(f, i) == bin) lead.list[atomicAdd(&lead.n_list, 1)] = rank_of(f, i);
    };
    const bool listed = summed && s.n_near <= kNear;
    if (listed)
      for (int i = tid; i < s.n_near; i += kThreads) offer(s.near[i] / VEC, s.near[i] % VEC);
#pragma unroll 1
    for (int v = 0; v < nv && !listed; ++v) {
      float f[VEC];
      load(v, f);
      unsigned some = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) some |= (unsigned)(f[e] <= g_hi && f[e] >= g_lo && alive(f[e])) << e;
      while (some) {
        offer(v * kThreads + tid, __ffs(some) - 1);
        some &= some - 1;
      }
    }
    sync();
    if (rank == 0) {  // sorted, and cut at the goal
      const int n = s.n_list;
      if (tid < n) {
        const u64 r = s.list[tid];
        int before = 0;
        for (int j = 0; j < n; ++j) before += s.list[j] > r;
        s.sorted[before] = r;
        if (top_p) s.weight[before] = w(value_of((uint32_t)(r >> 32))) * kFixed;
      }
      __syncthreads();
      if (!top_p) {
        if (tid == 0) s.cut = s.sorted[s.goal - s.above - 1];
      } else if (warp == 0) {  // the last entry whose predecessors weigh less than the goal
        double run = whole ? 0.0 : (double)s.above, goal = s.real_goal;
        if (whole) {
          double t = 0.0;
          for (int i = lane; i < n; i += 32) t += s.weight[i];
          goal = (double)set.p * warp_sum_d(t);
        }
        int kept = 0;
#pragma unroll 1
        for (int at = 0; at < n; at += 32) {
          double inc = at + lane < n ? s.weight[at + lane] : 0.0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
          }
          const double prev = __shfl_up_sync(0xffffffffu, inc, 1);
          const bool in = at + lane < n && run + (lane ? prev : 0.0) < goal;
          kept += __popc(__ballot_sync(0xffffffffu, in));
          run += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) s.cut = s.sorted[max(kept, 1) - 1];
      }
    }
    sync();
    cut_f = value_of((uint32_t)(lead.cut >> 32));
    cut_i = (int)~(uint32_t)lead.cut;
    if (!top_p) kill([&](float f, int i) { return keep(f, i) ? f : -INFINITY; });
  }

  // 4: kept weights up to and with each run of 32 vectors (a warp's v-th), in index order
  summed = summed && set.m == 0.0;  // the stretch of the cut adds to the sums above it
  const float most = summed ? f_hi : INFINITY;
  const int runs = (rounds * kWarps + 31) / 32 * 32;  // padded to whole warps
  if (tid < runs - rounds * kWarps) s.run[rounds * kWarps + tid] = 0.0;
#pragma unroll 1
  for (int v = 0; v < rounds; ++v) {
    double t = 0.0;
    if (v < nv) {
      float f[VEC];
      load(v, f);
      unsigned some = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        some |= (unsigned)(f[e] >= cut_f && f[e] <= most && keep(f[e], index(v, e))) << e;
      if (__popc(some) > 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const double x = w(f[e]);
          t += (some >> e & 1) && x >= set.m ? x : 0.0;
        }
      } else if (some) {
        const double x = w(entry(v * kThreads + tid, __ffs(some) - 1));
        t = x >= set.m ? x : 0.0;
      }
    }
    if (__any_sync(0xffffffffu, t != 0.0)) {
      t = warp_sum_d(t);
      if (lane == 0) s.run[v * kWarps + warp] = summed ? s.run[v * kWarps + warp] + t : t;
    } else if (lane == 0 && !summed) {
      s.run[v * kWarps + warp] = 0.0;
    }
  }
  __syncthreads();
  if (warp == 0) {
    double carry = 0.0;
#pragma unroll 1
    for (int at = 0; at < runs; at += 32) {
      double inc = s.run[at + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      inc += carry;
      s.run[at + lane] = inc;
      carry = __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) s.total = carry;
  }
  sync();
  if (warp == 0) {
    double start = 0.0, total = 0.0;
    for (int c = 0; c < C; ++c) {
      if (c == rank) start = total;
      total += peer(c).total;
    }
    const double goal = set.u * total;
    // the CTAs' stretches [start, start + total) share their borders' very values: one holds the goal
    if (start <= goal && goal < start + s.total) {
      double here = goal - start;
      int run = -1;
#pragma unroll 1
      for (int at = 0; at < runs && run < 0; at += 32) {
        const unsigned hit = __ballot_sync(0xffffffffu, s.run[at + lane] > here);
        if (hit) run = at + __ffs(hit) - 1;
      }
      if (run < 0) {  // (by rounding alone) the last run with any weight
        run = 0;
        for (int i = 1; i < runs; ++i)
          if (s.run[i] > s.run[i - 1]) run = i;
      }
      here -= run ? s.run[run - 1] : 0.0;
      const int j = run * 32 + lane, i0 = first + (j - tid) * VEC;
      auto kept = [&](int e) {
        const float f = entry(j, e);
        const double x = keep(f, i0 + e) ? w(f) : 0.0;
        return x >= set.m ? x : 0.0;
      };
      double t = 0.0;
      if (j < per)
#pragma unroll 1
        for (int e = 0; e < VEC; ++e) t += kept(e);
      double inc = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned some = __ballot_sync(0xffffffffu, t > 0.0);
      const unsigned hit = __ballot_sync(0xffffffffu, t > 0.0 && inc > here);
      if (some && lane == (hit ? __ffs(hit) - 1 : 31 - __clz(some))) {
        here -= inc - t;
        double c = 0.0;
        int at = 0;
#pragma unroll 1
        for (int e = 0; e < VEC; ++e) {
          const double x = kept(e);
          c += x;
          if (x > 0.0) at = e;
          if (x > 0.0 && c > here) break;
        }
        a.out[row] = i0 + at;
      }
    }
  }
  if (C > 1) cluster.sync();  // no CTA leaves while another may read its memory
}

template <int DT>
int run_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int VEC = Elem<DT>::kVec;
  const int64_t vectors = (a.vocab + VEC - 1) / VEC + 1;
  const int sms = device_info().sm_count;
  auto slice = [&](int c) { return (vectors + c - 1) / c * 16; };
  // The smallest cluster whose slices leave room for a second CTA on the SM; larger while SMs would
  // stay empty and every thread still has a vector.
  int c = 1;
  while (c < 8 && (slice(c) > 66 * 1024 || (a.rows * c < sms && slice(c) > kThreads * 16))) c *= 2;
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
