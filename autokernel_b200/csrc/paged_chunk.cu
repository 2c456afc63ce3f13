// Paged attention of chunks of new tokens for sm_100a: 16-bit types, D 64 or 128.
//
// Bound by the tensor cores for long chunks (4 D flops per row and visible key) and by reading the
// keys for short ones.  A work item is two tiles of up to 128 query rows of one key/value head;
// row r of a tile is token r / G, head r % G of the group, so grouped heads share every key that
// is read and short chunks still fill the 128 rows.  The keys of an item are walked in blocks of
// 128, and the line of paged_sched.cuh gives every CTA (one per SM) the same number of keys, over item
// boundaries and inside items: one long prompt occupies the whole GPU.
//
// 320 threads:
//   warp 0      TMA producer: Q of each segment (3-D map [N, H, D], boxes of {128 / G tokens, G
//               heads, 64}), then a 2-stage ring of {K, V} blocks gathered page by page (a box
//               is gcd(page_size, 128) slots of a page)
//   warp 1      TMEM allocator and MMA issuer (S = Q K^T, O += P V with P from TMEM)
//   warps 2..5  softmax and epilogue of tile 0, one thread per query row; warps 6..9 of tile 1
// While one tile is in its softmax the tensor core works on the other.  P is rounded to 16 bits
// once, as the matrix unit takes it; maximum, sum and output are fp32.  Slots of the last page
// behind the last visible key may hold anything, NaN included: the producer zeroes their V rows
// before the matrix unit sees them (their scores are masked).
#include "paged_sched.cuh"

namespace ak {
namespace paged {

using namespace sm100;

namespace chunk {

constexpr int BQ = 128, BKV = 128, THREADS = 320;
constexpr int CHUNK_BYTES = 128 * 64 * 2;  // 128 rows x 64 16-bit elements
constexpr int ROWS = 2 * BQ;               // rows of an item

template <int D>
struct Cfg {
  static constexpr int NC = D / 64;
  static constexpr int TILE_BYTES = NC * CHUNK_BYTES;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * TILE_BYTES;
  static constexpr int V_OFF = K_OFF + 2 * TILE_BYTES;
  static constexpr int SMEM = V_OFF + 2 * TILE_BYTES + 1024;
  static constexpr int TMEM_TILE = 256;  // S (128) + O (<= 128)
  static constexpr int PART = ROWS * (D + 2);  // floats of a part: O as [D / 4][ROWS] float4, m, l
};

struct Params {
  TileRule rule;
  int tt;   // tokens per tile: 128 / G
  int box;  // slots per TMA box
  uint32_t idesc_qk, idesc_pv;
  float* ws;
};

// Key blocks of the segment that tile x takes, as an end: [blk0, end).  A tile whose tokens lie
// behind the sequence takes none; under the causal mask tile 0 may stop before tile 1.
struct Ends {
  int e[2];
  int lead;  // the tile that takes every block
};
AK_D Ends ends_of(const AttnArgs& a, const Params& p, const Segment& s) {
  Ends x;
  const bool two = s.t_lo + p.tt < s.t_hi;
  x.lead = two ? 1 : 0;
  x.e[1] = two ? s.blk1 : s.blk0;
  x.e[0] = s.blk1;
  if (two && a.causal) {
    const int hi = min(visible_keys(s.r, s.t_lo + p.tt - 1, 1), capacity(a.l));
    x.e[0] = max(s.blk0, min(s.blk1, (hi + BKV - 1) / BKV));
  }
  return x;
}

template <int DT, int D>
__global__ void __launch_bounds__(THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const __grid_constant__ AttnArgs a,
                 const __grid_constant__ Params p) {
  using C = Cfg<D>;
  using E = Elem<DT>;
  using T = typename E::T;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  __shared__ uint64_t q_full, q_empty, k_full[2], v_full[2], kv_empty[2], s_full[2], p_full[2],
      o_done[2], o_free[2], v_land;
  __shared__ int s_bad[2];  // first key of the block in a ring slot that has no page
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&v_land, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 4);
    }
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  const Line line = find_piece(a, p.rule, blockIdx.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* abort_p = &abort_flag;
  Walker walk(a, p.rule, line, blockIdx.x);
  Segment s;

  if (warp == 0) {  // ------------------------------------------------------- TMA producer
    const int boxes = BKV / p.box;
    int g = 0, nq = 0, nv = 0;  // ring slots, Q loads and tail blocks so far
    bool ok = true;
    while (ok && walk.next(s)) {
      if (s.blk0 == s.blk1) continue;  // no keys: nothing to load
      const Ends ends = ends_of(a, p, s);
      PageFeed feed;
      feed.start(a, s, s.blk0 * boxes, p.box);
      for (int blk = s.blk0; blk < s.blk1; ++blk, ++g) {
        const int st = g & 1;
        feed.reach(a, s, blk * boxes, p.box);
        if (blk == s.blk0) {
          ok = nq == 0 || mbar_wait(&q_empty, (nq - 1) & 1, abort_p);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) {
            mbar_expect_tx(&q_full, (1 + ends.lead) * C::NC * p.tt * a.G * 128);
            for (int x = 0; x <= ends.lead; ++x)
              for (int c = 0; c < C::NC; ++c)
                tma_load_3d(smem + C::Q_OFF + x * C::TILE_BYTES + c * CHUNK_BYTES, &tq, &q_full,
                            c * 64, s.h * a.G, s.r.begin + s.t_lo + x * p.tt);
          }
          ++nq;
        }
        ok = mbar_wait(&kv_empty[st], ((g >> 1) & 1) ^ 1, abort_p);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        // slots of a loaded page behind the last visible key: V must read as zeros there
        const int live = s.kv_hi - blk * BKV;
        const bool tail = live < BKV && live % p.box != 0;
        uint64_t* v_bar = tail ? &v_land : &v_full[st];
        const int bad = feed.missing(a.l, blk * boxes, boxes);
        for (int i = 0; i < boxes; ++i) {
          int page, slot;
          feed.get(a.l, blk * boxes + i, page, slot);
          if (lane == 0) {
            uint8_t* dst = smem + st * C::TILE_BYTES + i * p.box * 128;
#pragma unroll
            for (int c = 0; c < C::NC; ++c) {
              tma_load_4d(dst + C::K_OFF + c * CHUNK_BYTES, &tk, &k_full[st], c * 64, slot, s.h, page);
              tma_load_4d(dst + C::V_OFF + c * CHUNK_BYTES, &tv, v_bar, c * 64, slot, s.h, page);
            }
          }
        }
        if (lane == 0) {  // the phases cannot end before these arrivals
          s_bad[st] = bad;
          mbar_expect_tx(&k_full[st], C::TILE_BYTES);
          mbar_expect_tx(v_bar, C::TILE_BYTES);
        }
        __syncwarp();
        if (tail) {
          ok = mbar_wait(&v_land, nv++ & 1, abort_p);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          const int rows = (live + p.box - 1) / p.box * p.box - live;
          for (int i = lane; i < rows * 8 * C::NC; i += 32) {
            const int c = i / (rows * 8), j = i - c * rows * 8;
            *reinterpret_cast<uint4*>(smem + C::V_OFF + st * C::TILE_BYTES + c * CHUNK_BYTES +
                                      live * 128 + j * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
        }
      }
    }
    if (*abort_p && lane == 0) {  // giving up: wait for the copies in flight
      drain_ring(k_full, 2, g);
      drain_ring(v_full, 2, g);
      if (nq) drain_ring(&q_full, 1, nq);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // ------------------------------------------------------ MMA issuer
      const uint32_t sq = smem_u32(smem + C::Q_OFF);
      const uint32_t sk = smem_u32(smem + C::K_OFF);
      const uint32_t sv = smem_u32(smem + C::V_OFF);
      auto qk = [&](int x, int st) {  // S_x = Q_x K_st^T
        const uint32_t d = tmem + x * C::TMEM_TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * CHUNK_BYTES + (kk & 3) * 32;
          umma_ss(d, desc_kmajor(sq + x * C::TILE_BYTES + off),
                  desc_kmajor(sk + st * C::TILE_BYTES + off), p.idesc_qk, kk > 0);
        }
      };
      auto pv = [&](int x, int st, bool acc) {  // O_x += P_x V_st
        const uint32_t d = tmem + x * C::TMEM_TILE + 128;
        const uint32_t pa = tmem + x * C::TMEM_TILE;
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk)
          umma_ts(d, pa + kk * 8,
                  desc_mnmajor(sv + st * C::TILE_BYTES + kk * 16 * 128, CHUNK_BYTES), p.idesc_pv,
                  (acc || kk > 0) ? 1 : 0);
      };
      int g = 0, nq = 0;
      int cnt[2] = {0, 0};   // key blocks processed so far by each tile (S / P phases)
      int used[2] = {0, 0};  // segments in which each tile had blocks (O phases)
      bool ok = true;
      while (ok && walk.next(s)) {
        if (s.blk0 == s.blk1) continue;
        const Ends ends = ends_of(a, p, s);
        const int lead = ends.lead;
        if (!mbar_wait(&q_full, nq++ & 1, abort_p) ||
            !mbar_wait(&k_full[g & 1], (g >> 1) & 1, abort_p))
          break;
        tc_fence_after();
        // S of both tiles for the first block (the previous segment's P V, issued earlier, has
        // read S by the time the tensor core gets here)
        for (int x = 0; x < 2; ++x)
          if (s.blk0 < ends.e[x]) {
            qk(x, g & 1);
            umma_commit(&s_full[x]);
          }
        if (s.blk1 - s.blk0 == 1) umma_commit(&q_empty);  // that was the last read of Q
        for (int j = s.blk0; ok && j < s.blk1; ++j, ++g) {
          const int st = g & 1;
          bool v_ready = false, k_ready = false;
          for (int x = 0; x < 2 && ok; ++x) {
            if (j >= ends.e[x]) continue;
            if (!mbar_wait(&p_full[x], cnt[x] & 1, abort_p)) { ok = false; break; }
            // a segment's first P V overwrites O: the tile's last epilogue must have read it
            if (j == s.blk0 && used[x] > 0 && !mbar_wait(&o_free[x], (used[x] - 1) & 1, abort_p)) {
              ok = false;
              break;
            }
            if (!v_ready && !mbar_wait(&v_full[st], (g >> 1) & 1, abort_p)) { ok = false; break; }
            v_ready = true;
            tc_fence_after();
            pv(x, st, j > s.blk0);
            ++cnt[x];
            if (x == lead) umma_commit(&kv_empty[st]);
            if (j == ends.e[x] - 1) {
              umma_commit(&o_done[x]);
              ++used[x];
            } else {
              const int ng = g + 1;
              if (!k_ready && !mbar_wait(&k_full[ng & 1], (ng >> 1) & 1, abort_p)) { ok = false; break; }
              k_ready = true;
              tc_fence_after();
              qk(x, ng & 1);
              umma_commit(&s_full[x]);
              if (x == lead && j + 2 == s.blk1) umma_commit(&q_empty);
            }
          }
        }
      }
    }
  } else {  // ---------------------------------------------------------- softmax / epilogue
    const int x = (warp - 2) >> 2;
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + x * C::TMEM_TILE + lane_base;
    const uint32_t t_o = t_s + 128;
    const int cap = capacity(a.l);
    bool ok = true;
    int cnt = 0, used = 0, g = 0;
    while (ok && walk.next(s)) {
      const Ends ends = ends_of(a, p, s);
      const int tok = s.t_lo + x * p.tt + row / a.G;
      const bool valid = row < p.tt * a.G && tok < s.t_hi;
      const int vis = valid ? visible_keys(s.r, tok, a.causal) : 0;
      float m_ref = -INFINITY, l = 0.f;
      int bad = cap;
      const int g0 = g;
      g += s.blk1 - s.blk0;
      for (int j = s.blk0; j < ends.e[x]; ++j, ++cnt) {
        const bool w = mbar_wait(&s_full[x], cnt & 1, abort_p);
        if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
        tc_fence_after();
        bad = min(bad, s_bad[(g0 + j - s.blk0) & 1]);
        const int kmax = vis - j * BKV;  // keys below this are visible to the row
        uint32_t r[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, r + c * 32);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_regs_ready(r + c * 32);
        if (!__all_sync(0xffffffffu, kmax >= BKV)) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= kmax) r[i] = __float_as_uint(-INFINITY);
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mx[q] = fmax3(mx[q], __uint_as_float(r[i + 2 * q]), __uint_as_float(r[i + 2 * q + 1]));
        const float bmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
        // the reference maximum moves only when a block raises it by more than 8 (log2)
        float alpha = 1.f;
        if (bmax > m_ref + 8.f) {
          if (m_ref != -INFINITY) alpha = ex2_approx(m_ref - bmax);
          m_ref = bmax;
        }
        l *= alpha;
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) {
            uint32_t o[8];
            tmem_ld8(t_o + c * 8, o);
            tmem_wait_ld();
            tmem_regs_ready8(o);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st8(t_o + c * 8, o);
          }
          tmem_wait_st();
        }
        const float mr = m_ref == -INFINITY ? 0.f : m_ref;
        float2 sum2[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 e = ffma2_bcast(__uint_as_float(r[c * 16 + 2 * i]),
                                         __uint_as_float(r[c * 16 + 2 * i + 1]), a.scale_log2, -mr);
            const float u = ex2_approx(e.x), v = ex2_approx(e.y);
            fadd2_acc(sum2[i & 1], u, v);
            if constexpr (DT == AK_BF16) {
              __nv_bfloat162 h = __floats2bfloat162_rn(u, v);
              pk[i] = *reinterpret_cast<uint32_t*>(&h);
            } else {
              __half2 h = __floats2half2_rn(u, v);
              pk[i] = *reinterpret_cast<uint32_t*>(&h);
            }
          }
          tmem_st8(t_s + c * 8, pk);
        }
        l += (sum2[0].x + sum2[1].x) + (sum2[0].y + sum2[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (!ok) break;
      const bool took = s.blk0 < ends.e[x];  // the tile has an O
      if (took) {
        const bool w = mbar_wait(&o_done[x], used & 1, abort_p);
        if (!__all_sync(0xffffffffu, w)) break;
        tc_fence_after();
        ++used;
      }
      if (vis > bad) l = __int_as_float(0x7fffffff);  // a key that the row sees has no page
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* orow = reinterpret_cast<T*>(a.o) + (int64_t)(s.r.begin + tok) * a.os[0] +
                (int64_t)(s.h * a.G + row % a.G) * a.os[1];
      float* part = p.ws + ((int64_t)blockIdx.x * 2 + s.slot) * C::PART;
      const int prow = x * BQ + row;
      bool odd = false;  // a result that is not finite
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        __syncwarp();
        if (took) {
          tmem_ld32(t_o + c * 32, r);
          tmem_wait_ld();
          tmem_regs_ready(r);
          if (c == D / 32 - 1) {  // O has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[x]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
        if (!valid) continue;
        if (s.whole) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 raw;
            T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float y = l == 0.f ? 0.f : __uint_as_float(r[q * 8 + i]) * inv;
              odd |= !(fabsf(y) <= 3.4028235e38f);
              e[i] = E::from_f(y);
            }
            reinterpret_cast<uint4*>(orow + c * 32)[q] = raw;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            __stcg(reinterpret_cast<uint4*>(part) + (c * 8 + q) * ROWS + prow,
                   make_uint4(r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]));
        }
      }
      if (!s.whole && valid) {
        part[ROWS * D + prow] = m_ref;
        part[ROWS * D + ROWS + prow] = l;
      }
      // rows whose result is not finite although their weights are, beside keys hidden from them
      unsigned again = __ballot_sync(0xffffffffu, odd && fabsf(l) <= 3.4028235e38f && vis < s.kv_hi);
      while (again) {
        const int i = __ffs(again) - 1, rr = quarter * 32 + i;
        again &= again - 1;
        const int t = s.t_lo + x * p.tt + rr / a.G;
        __syncwarp();
        if (hidden_not_finite<DT>(a, s.b, s.h, visible_keys(s.r, t, a.causal), s.kv_hi))
          row_by_key<DT>(a, s.b, s.r, t, s.h * a.G + rr % a.G);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the item that boundary blockIdx.x + 1 cuts first.  One thread per row, 32
// rows per CTA and four threads along D.
template <int DT, int D>
__global__ void __launch_bounds__(128)
    chunk_join_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Params p) {
  using C = Cfg<D>;
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int V = D / 16;  // float4 of a row per thread
  __shared__ int s_slot[kParts];
  __shared__ int s_whole, s_again;
  if (threadIdx.x == 0) s_whole = s_again = 0;
  Line line;
  const Parts parts = find_parts(a, p.rule, line);
  wait_for_parts();
  if (parts.n == 0) return;
  const Segment& s = parts.s;
  const int lane = threadIdx.x & 31, part_d = threadIdx.x >> 5;
  const int prow = blockIdx.y * 32 + lane, x = prow / BQ, row = prow % BQ;
  const int tok = s.t_lo + x * p.tt + row / a.G;
  const bool valid = row < p.tt * a.G && tok < s.t_hi;
  float top = -INFINITY, sum = 0.f;
  float4 acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < parts.n; i0 += kParts) {
    const int n = min(kParts, parts.n - i0);
    __syncthreads();
    if (threadIdx.x < n) {
      bool whole;
      s_slot[threadIdx.x] = part_slot(a, p.rule, line, parts, i0 + threadIdx.x, whole);
      if (whole) s_whole = 1;
    }
    __syncthreads();
    if (s_whole) return;  // written by the CTA that has all of it
    if (!valid) continue;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      if (s_slot[i] < 0) continue;
      const float* part = p.ws + (int64_t)s_slot[i] * C::PART;
      float4 v[V];
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = __ldcg(reinterpret_cast<const float4*>(part) + (part_d * V + k) * ROWS + prow);
      const float m = __ldcg(part + ROWS * D + prow), l = __ldcg(part + ROWS * D + ROWS + prow);
      const float mn = fmaxf(top, m), ref = mn == -INFINITY ? 0.f : mn;
      const float f0 = ex2_approx(top - ref), f1 = ex2_approx(m - ref);
      top = mn;
      sum = sum * f0 + l * f1;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        acc[k].x = acc[k].x * f0 + v[k].x * f1;
        acc[k].y = acc[k].y * f0 + v[k].y * f1;
        acc[k].z = acc[k].z * f0 + v[k].z * f1;
        acc[k].w = acc[k].w * f0 + v[k].w * f1;
      }
    }
  }
  bool odd = false;
  if (valid) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* orow = reinterpret_cast<T*>(a.o) + (int64_t)(s.r.begin + tok) * a.os[0] +
              (int64_t)(s.h * a.G + row % a.G) * a.os[1] + part_d * (D / 4);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
      const float* f = reinterpret_cast<const float*>(&acc[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float o = sum == 0.f ? 0.f : f[k] * inv;
        odd |= !(fabsf(o) <= 3.4028235e38f);
        e[k] = E::from_f(o);
      }
      reinterpret_cast<uint4*>(orow)[i / 2] = raw;
    }
  }
  odd = odd && fabsf(sum) <= 3.4028235e38f && visible_keys(s.r, tok, a.causal) < s.kv_hi;
  if (odd) atomicOr(&s_again, 1 << lane);
  __syncthreads();
  for (int i = part_d; i < 32 && s_again; i += 4) {
    if (!(s_again >> i & 1)) continue;
    const int rr = blockIdx.y * 32 + i - x * BQ, t = s.t_lo + x * p.tt + rr / a.G;
    if (hidden_not_finite<DT>(a, s.b, s.h, visible_keys(s.r, t, a.causal), s.kv_hi))
      row_by_key<DT>(a, s.b, s.r, t, s.h * a.G + rr % a.G);
  }
}

template <int DT, int D>
static int launch(const AttnArgs& a, float* ws, cudaStream_t st) {
  Params p{};
  p.tt = BQ / a.G;
  p.box = gcd_int(a.l.page_size, BKV);
  p.rule = TileRule{0, 2 * p.tt, 7, 128, 512, device_info().sm_count, 1};
  const int fmt = DT == AK_BF16 ? 1 : 0;
  p.idesc_qk = idesc_f16(fmt, BQ, BKV, false, false);
  p.idesc_pv = idesc_f16(fmt, BQ, D, false, true);
  p.ws = ws;
  CUtensorMap tq, tk, tv;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)a.H, (uint64_t)a.l.N};
  const uint64_t strides[2] = {(uint64_t)(a.H > 1 ? a.qs[1] : D) * 2,
                               (uint64_t)(a.l.N > 1 ? a.qs[0] : D) * 2};
  const uint32_t box[3] = {64, (uint32_t)a.G, (uint32_t)p.tt};
  if (!make_tmap(&tq, DT, 3, a.q, dims, strides, box) || !cache_tmap(&tk, a, a.k, a.kcs, p.box) ||
      !cache_tmap(&tv, a, a.v, a.vcs, p.box))
    return AK_ERR_LAUNCH;
  const cudaError_t attr = smem_optin<chunk_kernel<DT, D>>(Cfg<D>::SMEM);
  AK_REQUIRE(attr == cudaSuccess, AK_ERR_LAUNCH, "paged_attention smem attribute: %s",
             cudaGetErrorString(attr));
  const int pieces = p.rule.ctas;
  chunk_kernel<DT, D><<<pieces, THREADS, Cfg<D>::SMEM, st>>>(tq, tk, tv, a, p);
  const int rc = launch_status("paged_attention");
  if (rc || pieces < 2) return rc;
  return launch_after(chunk_join_kernel<DT, D>, dim3(pieces - 1, ROWS / 32), 128, st, a, p);
}

}  // namespace chunk

size_t chunk_workspace(int D) {
  return 2 * (size_t)device_info().sm_count * chunk::ROWS * (D + 2) * sizeof(float);
}

int run_chunk(const AttnArgs& a, void* ws, cudaStream_t st) {
  float* f = reinterpret_cast<float*>(ws);
  if (a.dtype == AK_BF16)
    return a.D == 128 ? chunk::launch<AK_BF16, 128>(a, f, st) : chunk::launch<AK_BF16, 64>(a, f, st);
  return a.D == 128 ? chunk::launch<AK_F16, 128>(a, f, st) : chunk::launch<AK_F16, 64>(a, f, st);
}

}  // namespace paged
}  // namespace ak
