// Paged attention of chunks of new tokens for sm_100a: 16-bit types, D 64 or 128.
//
// Bound by the tensor cores for long chunks (4 D flops per row and visible key) and by reading the
// keys for short ones.  A work item is two tiles of up to 128 query rows of one key/value head;
// row r of a tile is token r / G, head r % G of the group, so grouped heads share every key that
// is read and short chunks still fill the 128 rows.  The keys of an item are walked in blocks of
// 128, and the line of paged_sched.cuh gives every CTA (one per SM) the same number of keys, over item
// boundaries and inside items: one long prompt occupies the whole GPU.
//
// 352 threads:
//   warp 0      walks the line and posts its segments; TMA producer of Q (3-D map [N, H, D], boxes of
//               {128 / G tokens, G heads, 64}) and of a 2-stage ring of K blocks, gathered page by
//               page (a box is gcd(page_size, 128) slots of a page)
//   warp 10     TMA producer of a 2-stage ring of V blocks
//   warp 1      TMEM allocator and MMA issuer (S = Q K^T, O += P V with P from TMEM)
//   warps 2..5  softmax and epilogue of tile 0, one thread per query row; warps 6..9 of tile 1
// While one tile is in its softmax the tensor core works on the other.  An item of one tile is split
// instead: tile 0's threads take its even key blocks and tile 1's its odd ones, with a maximum, sum
// and output of their own, and tile 0's threads join the two in the epilogue (a warp reads the
// TMEM lanes of its quarter of either tile).
//
// Measured: two prompts of 4096 and 3700 tokens, 32 heads of 128, bf16, pages of 64: 339 us, 736 TFLOP/s
// (360 to 371 us when called without a pause, where the clock gives way; a block's softmax takes longer than its
// two products, and a segment's start and end, which nothing overlaps, cost several us).  501 tokens on 7600
// keys, 32 heads over 8: 89 us, 720 TFLOP/s.  24 sequences of up to 96 tokens on up to 1500 keys, 12 heads
// of 64: 57 us, where reading the keys alone would take 10: 288 tiles of a few blocks each, whose starts and
// ends bound it.  What runs once per segment or block row (masks, the epilogue) is kept short: its
// instructions are not at hand when their turn comes (unrolled over a row's registers they took 380, 99 and
// 60 us, where the loops took 350, 91 and 56).
//
// P is rounded to 16 bits once, as the matrix unit takes it; reference, sum and output are fp32.  A second
// term of P, as the decoding kernel has it, would be half as much matrix work again, and as many more
// conversions and stores for the softmax threads, which bound the kernel.  Without it the relative error of
// the chunk above is 2.3e-3 in bf16, where exact results rounded once have 1.7e-3.
// Slots of the last page behind the last visible key may hold anything, NaN included: the
// producer zeroes their V rows before the matrix unit sees them (their scores are masked).
#include "attn_softmax.cuh"
#include "paged_sched.cuh"

namespace ak {
namespace paged {

using namespace sm100;

namespace chunk {

constexpr int BQ = 128, BKV = 128, THREADS = 352;
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
  Cutting* cuts;  // one per piece, behind the parts
  // Two per piece: whether rows of its whole items, and of the item that the boundary behind it cuts first, are
  // to be looked at again.
  int2* marks;
};

// A segment and what each tile does in it.  Tile x takes key blocks first[x], first[x] + step, ...
// below end[x]: both take all of theirs (under the causal mask tile 0 may stop before tile 1, even
// before it has begun), or a lone tile's blocks are split between them, or tile 1 takes none.
struct Posted {
  Segment s;
  int part;  // workspace slot of its part; negative: there are no more segments
  int two, split, step;
  int first[2], end[2];
  int bad;   // first key without a page of the blocks that have been loaded so far
};
AK_D void plan(const AttnArgs& a, const Params& p, Posted& x) {
  const Segment& s = x.s;
  x.two = s.t_lo + p.tt < s.t_hi;
  x.split = !x.two && s.blk1 - s.blk0 >= 2;
  x.step = x.split ? 2 : 1;
  x.first[0] = s.blk0;
  x.first[1] = s.blk0 + x.split;
  x.end[0] = s.blk1;
  x.end[1] = x.two || x.split ? s.blk1 : s.blk0;
  if (x.two && a.causal) {
    const int hi = min(visible_keys(s.r, s.t_lo + p.tt - 1, 1), capacity(a.l));
    x.end[0] = max(s.blk0, min(s.blk1, (hi + BKV - 1) / BKV));
  }
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
  constexpr int POSTS = 4;
  __shared__ uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2],
      p_full[2], o_done[2], o_free[2], v_land, ml_full, ml_free, post_full[POSTS], post_empty[POSTS];
  __shared__ Posted s_post[POSTS];
  __shared__ float2 s_ml[BQ];  // a split tile's second maximum and sum
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&v_land, 1);
    mbar_init(&ml_full, 4);
    mbar_init(&ml_free, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 4);
    }
    for (int i = 0; i < POSTS; ++i) {
      mbar_init(&post_full[i], 1);
      mbar_init(&post_empty[i], 10);  // the V producer, the MMA issuer and eight softmax warps
    }
    abort_flag = 0;
    p.marks[blockIdx.x] = make_int2(0, 0);
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
  // the n-th segment, or null when there is none (or another role gave up); released when done with
  auto segment = [&](int n) -> const Posted* {
    return mbar_wait(&post_full[n % POSTS], (n / POSTS) & 1, abort_p) && s_post[n % POSTS].part >= 0
               ? &s_post[n % POSTS]
               : nullptr;
  };
  const int boxes = BKV / p.box;

  if (warp == 0) {  // ----------------------------------------------- segments, Q and K
    Walker walk(a, p.rule, line, blockIdx.x);
    Posted x;
    int g = 0, nq = 0, posted = 0;  // K blocks, Q loads and segments so far
    auto post = [&]() -> bool {
      bool ok = mbar_wait(&post_empty[posted % POSTS], ((posted / POSTS) & 1) ^ 1, abort_p);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && lane == 0) {
        s_post[posted % POSTS] = x;
        mbar_arrive(&post_full[posted % POSTS]);
      }
      __syncwarp();
      ++posted;
      return ok;
    };
    bool ok = true;
    while (ok && walk.next(x.s)) {
      const Segment& s = x.s;
      x.part = 2 * blockIdx.x + s.slot;
      x.bad = 0x7fffffff;
      plan(a, p, x);
      ok = post();
      if (!ok || s.blk0 == s.blk1) continue;  // no keys: nothing to load
      PageFeed feed;
      feed.start(a, s, s.blk0 * boxes, p.box);
      ok = nq == 0 || mbar_wait(&q_empty, (nq - 1) & 1, abort_p);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      if (lane == 0) {
        mbar_expect_tx(&q_full, (1 + x.two) * C::NC * p.tt * a.G * 128);
        for (int t = 0; t <= x.two; ++t)
          for (int c = 0; c < C::NC; ++c)
            tma_load_3d(smem + C::Q_OFF + t * C::TILE_BYTES + c * CHUNK_BYTES, &tq, &q_full, c * 64,
                        s.h * a.G, s.r.begin + s.t_lo + t * p.tt);
      }
      ++nq;
      for (int blk = s.blk0; blk < s.blk1; ++blk, ++g) {
        const int st = g & 1;
        feed.reach(a, s, blk * boxes, p.box);
        ok = mbar_wait(&k_empty[st], ((g >> 1) & 1) ^ 1, abort_p);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        x.bad = min(x.bad, feed.missing(a.l, blk * boxes, boxes));
        for (int i = 0; i < boxes; ++i) {
          int page, slot;
          feed.get(a.l, blk * boxes + i, page, slot);
          if (lane == 0)
#pragma unroll
            for (int c = 0; c < C::NC; ++c)
              tma_load_4d(smem + C::K_OFF + st * C::TILE_BYTES + i * p.box * 128 + c * CHUNK_BYTES, &tk,
                          &k_full[st], c * 64, slot, s.h, page);
        }
        if (lane == 0) {  // the phase cannot end before this arrival
          s_post[(posted - 1) % POSTS].bad = x.bad;
          mbar_expect_tx(&k_full[st], C::TILE_BYTES);
        }
      }
    }
    x.part = -1;
    if (ok) post();
    if (lane == 0) p.cuts[blockIdx.x] = cutting_of(walk, line);
    if (*abort_p && lane == 0) {  // giving up: wait for the copies in flight
      drain_ring(k_full, 2, g);
      if (nq) drain_ring(&q_full, 1, nq);
    }
  } else if (warp == 10) {  // ------------------------------------------------------- V
    int g = 0, nv = 0;  // V blocks and tail blocks so far
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const Posted* x = segment(n);
      x = __all_sync(0xffffffffu, x != nullptr) ? x : nullptr;
      if (!x) break;
      const Segment s = x->s;
      __syncwarp();
      if (lane == 0) mbar_arrive(&post_empty[n % POSTS]);
      PageFeed feed;
      if (s.blk0 < s.blk1) feed.start(a, s, s.blk0 * boxes, p.box);
      for (int blk = s.blk0; blk < s.blk1; ++blk, ++g) {
        const int st = g & 1;
        feed.reach(a, s, blk * boxes, p.box);
        ok = mbar_wait(&v_empty[st], ((g >> 1) & 1) ^ 1, abort_p);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        // slots of a loaded page behind the last visible key: V must read as zeros there
        const int live = s.kv_hi - blk * BKV;
        const bool tail = live < BKV && live % p.box != 0;
        uint64_t* v_bar = tail ? &v_land : &v_full[st];
        for (int i = 0; i < boxes; ++i) {
          int page, slot;
          feed.get(a.l, blk * boxes + i, page, slot);
          if (lane == 0)
#pragma unroll
            for (int c = 0; c < C::NC; ++c)
              tma_load_4d(smem + C::V_OFF + st * C::TILE_BYTES + i * p.box * 128 + c * CHUNK_BYTES, &tv,
                          v_bar, c * 64, slot, s.h, page);
        }
        if (lane == 0) mbar_expect_tx(v_bar, C::TILE_BYTES);
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
    if (*abort_p && lane == 0) {
      drain_ring(v_full, 2, g);
      if (nv) drain_ring(&v_land, 1, nv);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // ------------------------------------------------------ MMA issuer
      const uint32_t sq = smem_u32(smem + C::Q_OFF);
      const uint32_t sk = smem_u32(smem + C::K_OFF);
      const uint32_t sv = smem_u32(smem + C::V_OFF);
      // (tile numbers below are constants of unrolled loops: this thread's arithmetic is on the way of
      // every product)
      auto qk = [&](int x, uint32_t q, int st) {  // S_x = Q K_st^T
        const uint32_t d = tmem + x * C::TMEM_TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * CHUNK_BYTES + (kk & 3) * 32;
          umma_ss(d, desc_kmajor(q + off),
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
      int g = 0, nq = 0;     // blocks before the segment, segments with blocks
      int kw = 0;            // K blocks that have been waited for
      int cnt[2] = {0, 0};   // key blocks processed so far by each tile (S / P phases)
      int used[2] = {0, 0};  // segments in which each tile had blocks (O phases)
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const Posted* post = segment(n);
        if (!post) break;
        const int blk0 = post->s.blk0, blk1 = post->s.blk1;
        const int two = post->two, split = post->split, step = post->step;
        const int first[2] = {post->first[0], post->first[1]}, end[2] = {post->end[0], post->end[1]};
        mbar_arrive(&post_empty[n % POSTS]);
        if (blk0 == blk1) continue;
        const uint32_t q1 = two ? sq + C::TILE_BYTES : sq;  // what tile 1 multiplies
        // S of tile x for block j, once K_j is there; a block's last reader frees it
        auto score = [&](int x, int j) -> bool {
          const int at = g + j - blk0;
          while (kw <= at) {
            if (!mbar_wait(&k_full[kw & 1], (kw >> 1) & 1, abort_p)) return false;
            ++kw;
          }
          tc_fence_after();
          qk(x, x ? q1 : sq, at & 1);
          umma_commit(&s_full[x]);
          if (!two || x == 1) umma_commit(&k_empty[at & 1]);
          if ((!two || x == 1) && j == blk1 - 1) umma_commit(&q_empty);  // the last read of Q
          return true;
        };
        if (!mbar_wait(&q_full, nq++ & 1, abort_p)) break;
        // (the previous segment's P V, issued earlier, have read S by the time the tensor core gets here)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (ok && first[x] < end[x]) ok = score(x, first[x]);
        for (int j = blk0; ok && j < blk1; ++j) {
          const int st = (g + j - blk0) & 1;
          bool v_ready = false;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!ok || j >= end[x] || (split && ((j - blk0) & 1) != x)) continue;
            if (!mbar_wait(&p_full[x], cnt[x] & 1, abort_p)) { ok = false; continue; }
            // a segment's first P V overwrites O: the tile's last epilogue must have read it
            if (j == first[x] && used[x] > 0 && !mbar_wait(&o_free[x], (used[x] - 1) & 1, abort_p)) {
              ok = false;
              continue;
            }
            if (!v_ready && !mbar_wait(&v_full[st], ((g + j - blk0) >> 1) & 1, abort_p)) { ok = false; continue; }
            v_ready = true;
            tc_fence_after();
            pv(x, st, j > first[x]);
            ++cnt[x];
            if (!two || x == 1) umma_commit(&v_empty[st]);
            if (j + step >= end[x]) {
              umma_commit(&o_done[x]);
              ++used[x];
            } else {
              ok = score(x, j + step);
            }
          }
        }
        g += blk1 - blk0;
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
    int cnt = 0, n_split = 0;
    int used[2] = {0, 0};  // segments in which each tile had blocks
    for (int n = 0; ok; ++n) {
      const Posted* post = segment(n);
      if (!__all_sync(0xffffffffu, post != nullptr)) break;
      int vis;  // keys that this thread's row sees; what else is known of the row is looked up again in
      {         // the epilogue: the loop needs every register
        const int tok = post->s.t_lo + (post->split ? 0 : x) * p.tt + row / a.G;
        // (a row of no token sees all: what it computes goes nowhere, and it masks nothing)
        vis = row < p.tt * a.G && tok < post->s.t_hi ? visible_keys(post->s.r, tok, a.causal) : 0x7fffffff;
      }
      float m_ref = -INFINITY, l = 0.f;
      const int step = post->step, end = post->end[x];
      for (int j = post->first[x]; j < end; j += step, ++cnt) {
        const bool w = mbar_wait(&s_full[x], cnt & 1, abort_p);
        if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
        tc_fence_after();
        const int kmax = vis - j * BKV;  // keys below this are visible to the row
        if (!__all_sync(0xffffffffu, kmax >= BKV)) {  // few blocks: masked in TMEM, where code is short
#pragma unroll 1
          for (int c = 0; c < BKV; c += 8) {
            if (__all_sync(0xffffffffu, kmax >= c + 8)) continue;
            uint32_t y[8];
            tmem_ld8(t_s + c, y);
            tmem_wait_ld();
            tmem_regs_ready8(y);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i >= kmax) y[i] = __float_as_uint(-INFINITY);
            tmem_st8(t_s + c, y);
          }
          tmem_wait_st();
        }
        uint32_t r[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, r + c * 32);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_regs_ready(r + c * 32);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mx[q] = fmax3(mx[q], __uint_as_float(r[i + 2 * q]), __uint_as_float(r[i + 2 * q + 1]));
        const float bmax = Weight<DT>::top(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), a.scale_log2);
        float alpha = 1.f;
        if (Weight<DT>::moves(bmax, m_ref)) {
          const float r = Weight<DT>::reference(bmax);
          if (m_ref != -INFINITY) alpha = ex2_approx(m_ref - r);
          m_ref = r;
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
        const float mr = Weight<DT>::base(m_ref);
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
      const Segment& s = post->s;
      const bool split = post->split;
      const int tile = split ? 0 : x;
      const int tok = s.t_lo + tile * p.tt + row / a.G;
      const bool valid = row < p.tt * a.G && tok < s.t_hi;
      // (blocks loaded since then, if any, hold no key that this tile's rows see)
      if (vis > min(post->bad, cap)) l = __int_as_float(0x7fffffff);  // a key that the row sees has no page
      const bool took[2] = {post->first[0] < post->end[0], post->first[1] < post->end[1]};
      bool w = true;
      if (split && x == 1) {  // its output is joined by tile 0's threads
        w = n_split == 0 || mbar_wait(&ml_free, (n_split - 1) & 1, abort_p);
        if (!__all_sync(0xffffffffu, w)) break;
        s_ml[row] = make_float2(m_ref, l);
        ++n_split;
        ++used[0];
        ++used[1];
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ml_full);
          mbar_arrive(&post_empty[n % POSTS]);
        }
        continue;
      }
      if (took[x]) w = mbar_wait(&o_done[x], used[x] & 1, abort_p);
      float f0 = 1.f, f1 = 0.f;  // weights of the tile's output and of the second one of a split
      if (split) {
        w = w && mbar_wait(&o_done[1], used[1] & 1, abort_p) && mbar_wait(&ml_full, n_split & 1, abort_p);
        const float2 ml = s_ml[row];
        const float mn = fmaxf(m_ref, ml.x), ref = mn == -INFINITY ? 0.f : mn;
        f0 = ex2_approx(m_ref - ref);
        f1 = ex2_approx(ml.x - ref);
        l = l * f0 + ml.y * f1;
        m_ref = mn;
        ++n_split;
      }
      if (!__all_sync(0xffffffffu, w)) break;
      if (split && lane == 0) mbar_arrive(&ml_free);
      tc_fence_after();
      used[0] += took[0];
      used[1] += took[1];
      if (s.whole) l = Weight<DT>::total(l, m_ref);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* orow = reinterpret_cast<T*>(a.o) + (int64_t)(s.r.begin + tok) * a.os[0] +
                (int64_t)(s.h * a.G + row % a.G) * a.os[1];
      float* part = p.ws + (int64_t)post->part * C::PART;
      const int prow = x * BQ + row;
      float odd = 0.f;  // NaN once a result is not finite
#pragma unroll 1
      for (int c = 0; c < D / 8; ++c) {
        uint32_t r[8];
        __syncwarp();
        if (took[x]) {
          tmem_ld8(t_o + c * 8, r);
          if (split) {
            uint32_t r1[8];
            tmem_ld8(t_o + C::TMEM_TILE + c * 8, r1);
            tmem_wait_ld();
            tmem_regs_ready8(r);
            tmem_regs_ready8(r1);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              r[i] = __float_as_uint(__uint_as_float(r[i]) * f0 + __uint_as_float(r1[i]) * f1);
          } else {
            tmem_wait_ld();
            tmem_regs_ready8(r);
          }
          if (c == D / 8 - 1) {  // O has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&o_free[x]);
              if (split) mbar_arrive(&o_free[1]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = 0;
        }
        if (s.whole) {
          uint32_t e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y0 = __uint_as_float(r[2 * i]) * inv, y1 = __uint_as_float(r[2 * i + 1]) * inv;
            odd = fmaf(y0, 0.f, fmaf(y1, 0.f, odd));
            e[i] = attn_sm::pack2<DT>(y0, y1);
          }
          if (valid) reinterpret_cast<uint4*>(orow)[c] = make_uint4(e[0], e[1], e[2], e[3]);
        } else if (valid) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            __stcg(reinterpret_cast<uint4*>(part) + (c * 2 + q) * ROWS + prow,
                   make_uint4(r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]));
        }
      }
      if (!s.whole && valid) {
        part[ROWS * D + prow] = m_ref;
        part[ROWS * D + ROWS + prow] = l;
      }
      // rows whose result is not finite although their weights are, beside keys hidden from them
      if (odd != 0.f && valid && fabsf(l) <= 3.4028235e38f && vis < s.kv_hi) p.marks[blockIdx.x].x = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&post_empty[n % POSTS]);
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
  __shared__ int s_whole;
  if (threadIdx.x == 0) s_whole = 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Line line;
  wait_for_parts();
  const Parts parts = parts_of(a, p.rule, p.cuts[blockIdx.x], line);
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
    sum = Weight<DT>::total(sum, top);
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
  if (odd && fabsf(sum) <= 3.4028235e38f && visible_keys(s.r, tok, a.causal) < s.kv_hi) p.marks[blockIdx.x].y = 1;
}

// Looks again at rows of the items that are marked, in a launch of its own: within the joining kernel that code,
// although it hardly ever runs, cost a call 4 to 10 us; here 2, if it is a function that is called (8 inlined).
template <int DT, int D>
__device__ __noinline__ void look_again_at_items(const AttnArgs& a, const Params& p, int2 marked, AgainScratch<D>& sh) {
  Parts parts;
  Line line;
  if (marked.y) parts = parts_of(a, p.rule, p.cuts[blockIdx.x], line);
  look_again<DT, D>(a, p.rule, parts.s, marked.y, marked.x, blockIdx.x, blockIdx.y * 32, blockIdx.y * 32 + 32, sh);
}
template <int DT, int D>
__global__ void __launch_bounds__(128)
    chunk_again_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Params p) {
  __shared__ AgainScratch<D> scratch;
  wait_for_parts();
  const int2 marked = __ldcg(p.marks + blockIdx.x);
  if (marked.x || marked.y) look_again_at_items<DT, D>(a, p, marked, scratch);
}

template <int DT, int D>
static int launch(const AttnArgs& a, float* ws, cudaStream_t st) {
  Params p{};
  p.tt = BQ / a.G;
  p.box = gcd_int(a.l.page_size, BKV);
  p.rule = TileRule{0, 2 * p.tt, 7, 128, 320, 512, device_info().sm_count, 1};
  const int fmt = DT == AK_BF16 ? 1 : 0;
  p.idesc_qk = idesc_f16(fmt, BQ, BKV, false, false);
  p.idesc_pv = idesc_f16(fmt, BQ, D, false, true);
  p.ws = ws;
  p.cuts = reinterpret_cast<Cutting*>(ws + 2 * (size_t)device_info().sm_count * Cfg<D>::PART);
  p.marks = reinterpret_cast<int2*>(p.cuts + device_info().sm_count);
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
  if (rc) return rc;
  const int joined = pieces < 2 ? AK_OK : launch_after(chunk_join_kernel<DT, D>, dim3(pieces - 1, ROWS / 32), 128, st, a, p);
  if (joined) return joined;
  return launch_after(chunk_again_kernel<DT, D>, dim3(pieces, ROWS / 32), 128, st, a, p);
}

}  // namespace chunk

size_t chunk_workspace(int D) {
  return (size_t)device_info().sm_count * (2 * chunk::ROWS * (D + 2) * sizeof(float) + sizeof(Cutting) + sizeof(int2));
}

int run_chunk(const AttnArgs& a, void* ws, cudaStream_t st) {
  float* f = reinterpret_cast<float*>(ws);
  if (a.dtype == AK_BF16)
    return a.D == 128 ? chunk::launch<AK_BF16, 128>(a, f, st) : chunk::launch<AK_BF16, 64>(a, f, st);
  return a.D == 128 ? chunk::launch<AK_F16, 128>(a, f, st) : chunk::launch<AK_F16, 64>(a, f, st);
}

}  // namespace paged
}  // namespace ak
