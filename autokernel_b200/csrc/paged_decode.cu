// Paged attention of few query rows per sequence (decoding) for sm_100a: 16-bit types, D 64 or 128.
//
// Bound by reading the live keys and values once (4 D bytes per key and key/value head in 16-bit
// types); the matrix work is small, so it runs on warp-level MMAs whose operands come from shared
// memory, and everything else serves keeping loads in flight.  A tile is 16 query rows: the
// heads of one key/value head's group (and the next tokens) share every key that is read.
//   warps 0..3  TMA producers of a ring of {K, V} blocks of 64 keys, gathered page by page (a box is
//               gcd(page_size, 64) slots of one page; 128-byte swizzle): K and V, even and odd
//               boxes.  One warp's copies leave about 140 cycles apart whatever their size, so a
//               single producer took 1140 cycles for a block of 16-slot pages, more than the 700
//               that HBM needs, and a table load per block cost it 2000 (the batch below took 309 us
//               so; 235 with four producers that fetch 32 page numbers at a time)
//   warps 4..11 two groups of four take alternate blocks, a warp 16 keys of its block, each with
//               its own reference (Weight), sum and output, joined through shared memory per segment
// One CTA per SM; the line of paged_sched.cuh gives each the same number of keys.
//
// Measured: 64 sequences of 300 to 8100 keys, 32 heads over 8 of 128, fp16, pages of 16: 194 us, 5.69 TB/s
// (87% of a plain copy's rate).  One sequence of 2011 keys, 32 heads of 128: 22.5 us, where the rate
// alone would take 5: the rest is latency, of the launch, of the lists and page numbers before the
// first copy can leave (2 us), of one ring fill and two joins per CTA and of the joining kernel (2 us).
//
// The weights P (Weight) are split into two 16-bit terms for P V, P = hi + lo: the matrix units have
// time to spare here.  In bf16 that keeps 16 bits of every P; in fp16 22, or what lies above 2^-25,
// where P's largest is 2^11 at least.  What is left is the rounding of the result.
#include "paged_sched.cuh"
#include "sm100.cuh"

namespace ak {
namespace paged {

using namespace sm100;

constexpr int kRows = 16, kBlk = 64, kWarps = 8, kProducers = 4, kThreads = 32 * (kWarps + kProducers);

template <int D>
struct DecodeCfg {
  static constexpr int NC = D / 64;
  static constexpr int HALF = kBlk * D * 2;      // K or V of one block
  static constexpr int STAGE = 2 * HALF;
  // Even: then a ring slot always belongs to the same group of consumer warps, which waits for each of
  // its phases in turn.  (A group that came to a slot every other phase could take the phase
  // before last, whose parity is the same, for the one it waits for.)
  static constexpr int STAGES = 192 * 1024 / STAGE;
  static_assert(STAGES % 2 == 0, "a ring slot must belong to one group");
  static constexpr int O_OFF = STAGES * STAGE;   // float [4][16][D]
  static constexpr int SMEM = O_OFF + kWarps / 2 * kRows * D * 4 + 1024;
};

// Rounds of pieces (paged_sched.cuh) where the tables could name a long line: four times the shortest share,
// since what they name is twice what is there or more in a batch of mixed lengths, and single pieces are the
// better ones for even lengths (159 : 170 us at 12,000 keys an SM).  Where the line turns out shorter, it is cut
// into single pieces, and the spare CTAs only cost their cancellation.  Fewer than 4 (sequence, head) pairs for 3
// SMs are cut into more parts by rounds than these gain: 160 pairs of 11,000 keys 162 : 183 us, 24 of 74,000 166 : 215.
static TileRule decode_rule(const AttnArgs& a) {
  const int ctas = device_info().sm_count;
  const int64_t pairs = (int64_t)a.l.B * a.Hkv;
  const double tiles = (double)a.l.B + (double)a.l.N * a.G / kRows;
  const double keys = tiles * a.Hkv * ((double)a.l.max_pages * a.l.page_size + 64);
  return TileRule{kRows, 0, 6, 64, 0, 256, ctas, keys / ctas >= 4 * kLongPiece && 3 * pairs >= 4 * ctas ? kRounds : 1};
}

static size_t decode_part_floats(int D) { return (size_t)kRows * (D + 2); }

template <int DT>
AK_D void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (DT == AK_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
AK_D void ldmatrix4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
AK_D void ldmatrix4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// (a, b) as 16-bit pairs hi + lo
template <int DT>
AK_D void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  if constexpr (DT == AK_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

AK_D void group_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }
AK_D bool group_all(bool x) {  // of all consumer warps
  int y;
  asm volatile("{.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.and.pred q, 1, %2, p;\nselp.s32 %0, 1, 0, q;}"
               : "=r"(y)
               : "r"((int)x), "n"(32 * kWarps)
               : "memory");
  return y;
}

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ AttnArgs a, const TileRule rule, int box,
                  float* ws) {
  using C = DecodeCfg<D>;
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int NF = D / 8;  // n8 tiles of the output
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* s_o = reinterpret_cast<float*>(smem + C::O_OFF);
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES];
  __shared__ int s_bad[C::STAGES];  // first key of the block without a page
  __shared__ float s_m[kWarps / 2][kRows], s_l[kWarps / 2][kRows];
  __shared__ int s_badw[kWarps];
  __shared__ int abort_flag, s_stop;
  // Segments, from the first producer to all other warps: finding one takes about 1000 cycles, so it is
  // done once and ahead of time.  part < 0: there are no more.
  struct Posted {
    Segment s;
    int part;  // workspace slot of its part
  };
  constexpr int POSTS = 4;
  __shared__ Posted s_post[POSTS];
  __shared__ uint64_t post_full[POSTS], post_empty[POSTS], next_full;
  __shared__ __align__(16) uint4 s_next;  // answer to the request for another piece
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (rule.rounds == 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    mbar_init(&next_full, 1);
    for (int i = 0; i < POSTS; ++i) {
      mbar_init(&post_full[i], 1);
      mbar_init(&post_empty[i], kWarps + kProducers - 1);
    }
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], kProducers);
      mbar_init(&empty[i], 4);
    }
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  Line line = find_piece(a, rule, blockIdx.x);
  __syncthreads();
  volatile int* abort_p = &abort_flag;
  int* const marks = reinterpret_cast<int*>(ws + 2 * (int64_t)gridDim.x * (kRows * (D + 2)));  // one per piece
  int g = 0;  // ring slots used so far
  // the n-th segment: null when there is none (or another warp gave up); free it when done with it
  auto segment = [&](int n) -> const Posted* {
    const bool got = mbar_wait(&post_full[n % POSTS], (n / POSTS) & 1, abort_p);
    return __all_sync(0xffffffffu, got) && s_post[n % POSTS].part >= 0 ? &s_post[n % POSTS] : nullptr;
  };
  auto release = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&post_empty[n % POSTS]);
  };

  if (warp < kProducers) {  // ------------------------------------------- TMA producers
    const int boxes = kBlk / box;
    const CUtensorMap* map = (warp & 1) ? &tv : &tk;
    const int i0 = warp >> 1, mine = (boxes - i0 + 1) / 2;  // boxes i0, i0 + 2, ...
    uint8_t* const dst = smem + ((warp & 1) ? C::HALF : 0);
    auto load = [&](const Segment& s) {
      PageFeed feed;
      if (s.blk0 < s.blk1) feed.start(a, s, s.blk0 * boxes, box);
      for (int blk = s.blk0; blk < s.blk1; ++blk, ++g) {
        const int st = g % C::STAGES;
        feed.reach(a, s, blk * boxes, box);
        const bool ok = mbar_wait(&empty[st], ((g / C::STAGES) & 1) ^ 1, abort_p);
        if (!__all_sync(0xffffffffu, ok)) return false;
        const int bad = warp == 0 ? feed.missing(a.l, blk * boxes, boxes) : 0;
        for (int i = i0; i < boxes; i += 2) {
          int page, slot;
          feed.get(a.l, blk * boxes + i, page, slot);
          if (lane == 0)
            tma_load_5d(dst + st * C::STAGE + i * (C::NC * box * 128), map, &full[st], 0, slot, 0, s.h, page);
        }
        if (lane == 0) {  // the phase cannot end before these arrivals, so `bad` is there with the data
          if (warp == 0) s_bad[st] = bad;
          if (mine) mbar_expect_tx(&full[st], mine * C::NC * box * 128); else mbar_arrive(&full[st]);
        }
      }
      return true;
    };
    if (warp == 0) {  // walks the line, posts its segments and asks for further pieces
      int piece = blockIdx.x, posted = 0, asked = 0;
      Walker walk(a, rule, line, piece);
      Segment s;
      auto post = [&](int part) {
        const bool ok = mbar_wait(&post_empty[posted % POSTS], ((posted / POSTS) & 1) ^ 1, abort_p);
        if (!__all_sync(0xffffffffu, ok)) return false;
        if (lane == 0) {
          s_post[posted % POSTS].s = s;
          s_post[posted % POSTS].part = part;
          mbar_arrive(&post_full[posted % POSTS]);
        }
        __syncwarp();
        ++posted;
        return true;
      };
      bool ok = true;
      while (ok) {
        if (lane == 0) marks[piece] = 0;  // (the consumers may set it once a segment is posted)
        while (ok && walk.next(s)) ok = post(2 * piece + s.slot) && load(s);
        if (!ok || rule.rounds == 1) break;
        if (lane == 0) {
          mbar_expect_tx(&next_full, 16);
          clc_try_cancel(&s_next, &next_full);
        }
        ok = mbar_wait(&next_full, asked++ & 1, abort_p);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {  // giving up: the answer still lands
          if (lane == 0) drain_ring(&next_full, 1, asked);
          break;
        }
        piece = clc_answer(&s_next);
        fence_proxy_async();
        __syncwarp();
        if (piece < 0) break;
        move_to_piece(a, rule, line, piece);
        walk.go(line, piece);
      }
      if (ok) post(-1);
      // nothing is left to launch: the join may
      if (rule.rounds > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
      // giving up: the copies in flight still land in this CTA's shared memory
      if (*abort_p && lane == 0) drain_ring(full, C::STAGES, g);
    } else {
      for (int n = 0;; ++n) {
        const Posted* p = segment(n);
        if (!p || !load(p->s)) break;
        release(n);
      }
    }
  } else {  // ---------------------------------------------------------------- consumers
    const int cw = warp - kProducers, grp = cw >> 2, k16 = (cw & 3) * 16;  // the warp's keys of its blocks
    const int r0 = lane >> 2, cq = 2 * (lane & 3);
    const uint32_t ring = smem_u32(smem);
    // a block lies box by box: [64 / box][D / 64][box slots][128 bytes]
    const uint32_t chunk = box * 128;
    auto row_at = [&](int row) { return (uint32_t)(row / box * (C::NC * box) + row % box) * 128; };
    const uint32_t krow[2] = {row_at(k16 + (lane & 7)), row_at(k16 + 8 + (lane & 7))};
    const uint32_t vrow = row_at(k16 + (lane & 15));
    const int cap = capacity(a.l);
    uint32_t q[D / 16][4];
    int vis[2];
    // this lane's part of a segment's queries and what its two rows see
    auto load_q = [&](const Segment& s) {
      const int row0 = s.tile * kRows, nr = min(kRows, s.r.n * a.G - row0);
      const T* qrow[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = min(r0 + 8 * i, nr - 1);
        const int t = (row0 + rr) / a.G, hg = (row0 + rr) % a.G;
        qrow[i] = reinterpret_cast<const T*>(a.q) + (int64_t)(s.r.begin + t) * a.qs[0] +
                  (int64_t)(s.h * a.G + hg) * a.qs[1];
        vis[i] = visible_keys(s.r, t, a.causal);
      }
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[kk][i] = __ldg(reinterpret_cast<const unsigned int*>(qrow[i & 1] + kk * 16 + cq + (i >> 1) * 8));
    };
    const Posted* now = segment(0);
    bool ok = group_all(now != nullptr);  // all of them meet in the loop, or none
    if (ok) load_q(now->s);
    for (int n_seg = 0; ok && now; ++n_seg) {
      const Segment& s = now->s;
      const int row0 = s.tile * kRows;
      const int nr = min(kRows, s.r.n * a.G - row0);
      float o[NF][4];
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      int bad = cap;
      // every row of the tile sees keys below this
      const int vis_all = visible_keys(s.r, s.t_lo, a.causal);
      const int blk0 = s.blk0, blk1 = s.blk1, kv_hi = s.kv_hi;
      for (int blk = blk0 + ((g & 1) != grp); blk < blk1; blk += 2) {
        const int at = g + blk - blk0, st = at % C::STAGES;
        const bool got = mbar_wait(&full[st], (at / C::STAGES) & 1, abort_p);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        bad = min(bad, s_bad[st]);
        const uint32_t kbase = ring + st * C::STAGE, vbase = kbase + C::HALF;
        const int key0 = blk * kBlk + k16;
        // S = Q K^T for 16 keys
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[n][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {  // 32 dims a load
          const int unit = (kk & 1) * 4 + (lane >> 3);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t kf[4];
            ldmatrix4(kf, kbase + krow[n] + (kk >> 1) * chunk + ((unit ^ (lane & 7)) << 4));
            mma16816<DT>(sc[n], q[2 * kk], kf[0], kf[1]);
            mma16816<DT>(sc[n], q[2 * kk + 1], kf[2], kf[3]);
          }
        }
        if (key0 + 16 > vis_all) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (key0 + n * 8 + cq + (j & 1) >= vis[j >> 1]) sc[n][j] = -INFINITY;
        }
        // m: the reference of the weights (Weight)
        float alpha[2];
        bool move = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          x = Weight<DT>::top(x, a.scale_log2);
          alpha[i] = 1.f;
          if (Weight<DT>::moves(x, m[i])) {
            x = Weight<DT>::reference(x);
            alpha[i] = m[i] == -INFINITY ? 0.f : ex2_approx(m[i] - x);
            m[i] = x;
            move = true;
          }
        }
        if (__any_sync(0xffffffffu, move)) {
          l[0] *= alpha[0];
          l[1] *= alpha[1];
#pragma unroll
          for (int i = 0; i < NF; ++i) {
            o[i][0] *= alpha[0];
            o[i][1] *= alpha[0];
            o[i][2] *= alpha[1];
            o[i][3] *= alpha[1];
          }
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float ref = Weight<DT>::base(m[i]);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float x = ex2_approx(fmaf(sc[n][2 * i], a.scale_log2, -ref));
            const float y = ex2_approx(fmaf(sc[n][2 * i + 1], a.scale_log2, -ref));
            l[i] += x + y;
            split2<DT>(x, y, ph[2 * n + i], pl[2 * n + i]);
          }
        }
        // O += P V; keys behind the last visible one count as 0 whatever their slots hold
        uint32_t mask[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int k = key0 + 8 * i + cq;
          mask[i] = k + 1 < kv_hi ? 0xffffffffu : k < kv_hi ? 0x0000ffffu : 0u;
        }
#pragma unroll
        for (int n = 0; n < NF / 2; ++n) {  // 16 dims a load
          const int unit = (n & 3) * 2 + (lane >> 4);
          uint32_t vf[4];
          ldmatrix4t(vf, vbase + vrow + (n >> 2) * chunk + ((unit ^ (lane & 7)) << 4));
          vf[0] &= mask[0];
          vf[1] &= mask[1];
          vf[2] &= mask[0];
          vf[3] &= mask[1];
          mma16816<DT>(o[2 * n], ph, vf[0], vf[1]);
          mma16816<DT>(o[2 * n + 1], ph, vf[2], vf[3]);
          mma16816<DT>(o[2 * n], pl, vf[0], vf[1]);
          mma16816<DT>(o[2 * n + 1], pl, vf[2], vf[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      g += blk1 - blk0;
      // the next segment's queries are on their way while this one is put together
      const Posted* next = segment(n_seg + 1);
      if (next) load_q(next->s);
      // join the eight warps: the second group's into the first's registers, then those four
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      const int w4 = cw & 3;
      auto put = [&] {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = r0 + 8 * i;
          if (row >= nr) continue;
          if ((lane & 3) == 0) {
            s_m[w4][row] = m[i];
            s_l[w4][row] = l[i];
          }
#pragma unroll
          for (int n = 0; n < NF; ++n)
            *reinterpret_cast<float2*>(s_o + (w4 * kRows + row) * D + ((n * 8 + cq) ^ ((row & 7) * 8))) =
                make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
      };
      if (grp == 1) put();
      group_sync();
      if (grp == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = r0 + 8 * i;
          if (row >= nr) continue;
          const float m1 = s_m[w4][row], mn = fmaxf(m[i], m1), ref = mn == -INFINITY ? 0.f : mn;
          const float f0 = ex2_approx(m[i] - ref), f1 = ex2_approx(m1 - ref);
          // Which group has the even blocks hangs on the pieces its CTA took before, so the two change places
          // from call to call: products and sum are rounded apart, which gives the same bits either way.
          l[i] = __fadd_rn(__fmul_rn(l[i], f0), __fmul_rn(s_l[w4][row], f1));
          m[i] = mn;
#pragma unroll
          for (int n = 0; n < NF; ++n) {
            const float2 x = *reinterpret_cast<const float2*>(s_o + (w4 * kRows + row) * D +
                                                              ((n * 8 + cq) ^ ((row & 7) * 8)));
            o[n][2 * i] = __fadd_rn(__fmul_rn(o[n][2 * i], f0), __fmul_rn(x.x, f1));
            o[n][2 * i + 1] = __fadd_rn(__fmul_rn(o[n][2 * i + 1], f0), __fmul_rn(x.y, f1));
          }
        }
        __syncwarp();  // a row's four lanes have read its m and l
        put();
      }
      if (lane == 0) s_badw[cw] = bad;
      // a warp that gave up still meets the others here; the results no longer count then
      group_sync();
      int first_bad = cap;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) first_bad = min(first_bad, s_badw[w]);
      const bool again = a.causal && s.t_hi - s.t_lo > 1;  // rows of the tile hide keys from one another
      float* part = ws + (int64_t)now->part * (kRows * (D + 2));
      for (int e = threadIdx.x - 32 * kProducers; e < nr * D; e += 32 * kWarps) {
        const int row = e / D, d = e % D;
        float top = s_m[0][row];
#pragma unroll
        for (int w = 1; w < kWarps / 2; ++w) top = fmaxf(top, s_m[w][row]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps / 2; ++w) {
          const float f = ex2_approx(s_m[w][row] - ref);
          sum = fmaf(s_l[w][row], f, sum);
          x = fmaf(s_o[(w * kRows + row) * D + (d ^ ((row & 7) * 8))], f, x);
        }
        const int t = (row0 + row) / a.G, hg = (row0 + row) % a.G;
        const int v = visible_keys(s.r, t, a.causal);
        if (v > first_bad) sum = __int_as_float(0x7fffffff);
        if (s.whole) {
          sum = Weight<DT>::total(sum, top);
          const float y = sum == 0.f ? 0.f : x / sum;
          if (again && !(fabsf(y) <= 3.4028235e38f) && fabsf(sum) <= 3.4028235e38f && v < s.kv_hi)
            marks[now->part >> 1] = 1;
          reinterpret_cast<T*>(a.o)[(int64_t)(s.r.begin + t) * a.os[0] +
                                    (int64_t)(s.h * a.G + hg) * a.os[1] + d] = E::from_f(y);
        } else {
          part[row * D + d] = x;
          if (d == 0) {
            part[kRows * D + row] = top;
            part[kRows * D + kRows + row] = sum;
          }
        }
      }
      if (threadIdx.x == 32 * kProducers) s_stop = *abort_p;  // one reading, so that all warps leave together
      group_sync();
      ok = !s_stop;
      release(n_seg);
      now = next;
    }
  }
}

// Joins the parts of the tile that boundary blockIdx.x + 1 cuts first, every output element from
// independent loads, and looks again at the rows of piece blockIdx.x if it is marked.
template <int DT, int D>
__global__ void __launch_bounds__(128, 5)  // (a block per piece of five rounds at once)
    decode_join_kernel(const __grid_constant__ AttnArgs a, const TileRule rule, const float* ws) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int PART = kRows * (D + 2), U = 6;
  __shared__ int s_slot[kParts];
  __shared__ int s_whole, s_again;
  __shared__ AgainScratch<D> s_look;
  if (threadIdx.x == 0) s_whole = s_again = 0;
  Line line;
  const Parts p = find_parts(a, rule, line);
  auto slots = [&](int i0) {  // of parts i0 .. i0 + kParts - 1
    __syncthreads();
    if (threadIdx.x < min(kParts, p.n - i0)) {
      bool whole;
      s_slot[threadIdx.x] = part_slot(a, rule, line, p, i0 + threadIdx.x, whole);
      if (whole) s_whole = 1;
    }
    __syncthreads();
  };
  if (p.n) slots(0);
  wait_for_parts();
  const int marked = __ldcg(reinterpret_cast<const int*>(ws + 2 * (int64_t)gridDim.x * PART) + blockIdx.x);
  const Segment& s = p.s;
  const int row0 = s.tile * kRows;
  // (none, or one that a CTA has all of and has written)
  const int nr = p.n == 0 || s_whole ? 0 : min(kRows, s.r.n * a.G - row0);
#pragma unroll 1
  for (int at = 0; at < nr * D; at += 128) {
    const int e = at + threadIdx.x, row = e / D, d = e % D;
    float x = 0.f, sum = 0.f, top = -INFINITY;
    for (int i0 = 0; i0 < p.n; i0 += kParts) {
      const int n = min(kParts, p.n - i0);
      if (p.n > kParts) slots(i0);
      if (row >= nr) continue;
      for (int i = 0; i < n; i += U) {
        float m[U], l[U], y[U], mx = top;
#pragma unroll
        for (int u = 0; u < U; ++u) {  // all loads first
          const bool in = i + u < n && s_slot[i + u] >= 0;
          const float* part = ws + (int64_t)(in ? s_slot[i + u] : 0) * PART;
          m[u] = in ? __ldcg(part + kRows * D + row) : -INFINITY;
          l[u] = in ? __ldcg(part + kRows * D + kRows + row) : 0.f;
          y[u] = in ? __ldcg(part + e) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, m[u]);
        const float ref = mx == -INFINITY ? 0.f : mx, old = ex2_approx(top - ref);
        x *= old;
        sum *= old;
        top = mx;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float w = ex2_approx(m[u] - ref);
          x = fmaf(y[u], w, x);
          sum = fmaf(l[u], w, sum);
        }
      }
    }
    if (row >= nr) break;
    const float l = Weight<DT>::total(sum, top), out = l == 0.f ? 0.f : x / l;
    const int t = (row0 + row) / a.G, hg = (row0 + row) % a.G;
    if (!(fabsf(out) <= 3.4028235e38f) && fabsf(l) <= 3.4028235e38f &&
        visible_keys(s.r, t, a.causal) < s.kv_hi)
      s_again = 1;
    reinterpret_cast<T*>(a.o)[(int64_t)(s.r.begin + t) * a.os[0] +
                              (int64_t)(s.h * a.G + hg) * a.os[1] + d] = E::from_f(out);
  }
  __syncthreads();
  look_again<DT, D>(a, rule, s, s_again, marked, blockIdx.x, 0, kRows, s_look);
}

template <int DT, int D>
static int launch_decode(const AttnArgs& a, float* ws, cudaStream_t st) {
  const int box = gcd_int(a.l.page_size, kBlk);
  CUtensorMap tk, tv;
  if (!cache_tmap_5d(&tk, a, a.k, a.kcs, box) || !cache_tmap_5d(&tv, a, a.v, a.vcs, box))
    return AK_ERR_LAUNCH;
  const cudaError_t attr = smem_optin<decode_kernel<DT, D>>(DecodeCfg<D>::SMEM);
  AK_REQUIRE(attr == cudaSuccess, AK_ERR_LAUNCH, "paged_attention smem attribute: %s",
             cudaGetErrorString(attr));
  const TileRule rule = decode_rule(a);
  const int pieces = rule.ctas * rule.rounds;
  decode_kernel<DT, D><<<pieces, kThreads, DecodeCfg<D>::SMEM, st>>>(tk, tv, a, rule, box, ws);
  const int rc = launch_status("paged_attention");
  if (rc) return rc;
  return launch_after(decode_join_kernel<DT, D>, dim3(pieces), 128, st, a, rule, (const float*)ws);
}

size_t decode_workspace(int D) {
  return (size_t)device_info().sm_count * kRounds * (2 * decode_part_floats(D) * sizeof(float) + sizeof(int));
}

int run_decode(const AttnArgs& a, void* ws, cudaStream_t st) {
  float* f = reinterpret_cast<float*>(ws);
  if (a.dtype == AK_BF16)
    return a.D == 128 ? launch_decode<AK_BF16, 128>(a, f, st) : launch_decode<AK_BF16, 64>(a, f, st);
  return a.D == 128 ? launch_decode<AK_F16, 128>(a, f, st) : launch_decode<AK_F16, 64>(a, f, st);
}

}  // namespace paged
}  // namespace ak
