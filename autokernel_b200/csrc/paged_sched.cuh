// How the paged attention kernels share their work out.
//
// A tile is a run of one sequence's query rows for one key/value head; its work is its keys.  All
// tiles are laid end to end on one line (sequence, head, tile), each as long as its keys plus a
// constant for its prologue and epilogue, and the line is cut into one equal piece per CTA: every
// SM gets the same number of keys whatever the lengths are, and no host code has to know them.  A
// piece may end inside a tile.  Such a tile's parts go to the workspace, at most two per piece (its
// first and its last segment), and a second kernel joins them in the line's order, so results do
// not depend on timing.
//
// Equal pieces do not take equal time when memory is the bound: decoding 64 sequences of up to 8K
// keys, the first of 148 CTAs was done after 164 us and the last after 215; many short tiles take longer
// than their keys say.  Long lines are therefore cut into five rounds of pieces, 32, 16, 8, 5 and 3 64ths
// of an equal share, and a CTA that is done takes the next piece that has not begun (the hardware's
// cancellation of a CTA that waits to be launched hands its number over).  Decoding, 32 heads of 128, us, single
// pieces : rounds (of 46, 8, 5, 3, 2 / 54, 4, 3, 2, 1 64ths):
//   over 8, 64 x 300..8100 keys  204 : 196 (198 / 213)    over 32, 16 x 300..8000  211 : 184 (184 / 189)
//   over 8, 512 x 100..2000      590 : 431 (448 / 513)    over 8, 2048 x 50..600  1238 : 924 (946 / 1086)
//   over 8, 64 x 4000            179 : 187 (188 / 193)    over 8, 3 x 74000        166 : 215 (few tiles, many parts)
#pragma once
#include "paged_row.cuh"

namespace ak {
namespace paged {

// Rule by which a kernel cuts a sequence's tokens into tiles.
struct TileRule {
  int rows;    // query rows (token, head of the group) per tile, when tiles are cut by rows; or 0
  int tokens;  // tokens per tile otherwise
  int shift;   // log2 of the keys per block
  int over;    // cost of a tile beside its keys, in keys
  int lone;    // more of it for a sequence of at most half a tile's tokens, whose blocks go faster
  int64_t min_piece;  // shortest piece of the line that a CTA gets
  int ctas;           // CTAs that run at once
  int rounds;         // kRounds: a long line may be cut into rounds of pieces; or 1
};

// A sequence on the line: tile i of a head is base + slope * (i + 1) long, the last one `last`.
struct SeqCost {
  int tiles;
  int64_t base, slope, last;
  AK_D int64_t prefix(int64_t i) const { return i * base + slope * (i * (i + 1) / 2); }
  AK_D int64_t total() const { return tiles ? prefix(tiles - 1) + last : 0; }
  AK_D int64_t cost(int i) const { return i == tiles - 1 ? last : base + slope * (i + 1); }
  AK_D int find(int64_t y) const {  // tile that holds point y
    int lo = 0, hi = tiles;         // prefix(lo) <= y < prefix(hi) or the end
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (prefix(mid) <= y) lo = mid; else hi = mid;
    }
    return lo;
  }
};

AK_D int capacity(const PagedLists& l) {  // keys that a table row can name
  const int64_t c = (int64_t)l.max_pages * l.page_size;
  return c < 0x7fffffff ? (int)c : 0x7fffffff;
}

AK_D SeqCost seq_cost(const AttnArgs& a, const TileRule& t, const SeqRange& r) {
  SeqCost c{0, 0, 0, 0};
  if (r.n == 0) return c;
  const int kv = min(r.kv_len, capacity(a.l));
  if (t.rows) {
    c.tiles = (r.n * a.G + t.rows - 1) / t.rows;  // (N G < 2^31)
    c.base = c.last = (int64_t)kv + t.over;
  } else {
    c.tiles = (r.n + t.tokens - 1) / t.tokens;
    const int over = t.over + (2 * r.n <= t.tokens ? t.lone : 0);
    if (a.causal) {
      c.base = (int64_t)max(kv - r.n, 0) + over;
      c.slope = t.tokens;
      c.last = c.base + r.n;
    } else {
      c.base = c.last = (int64_t)kv + over;
    }
  }
  return c;
}

// A CTA's part of one tile: key blocks [blk0, blk1) of the tile's nb.
struct Segment {
  SeqRange r;
  int b, h, tile;
  int t_lo, t_hi;  // the tile's tokens within the sequence
  int kv_hi;       // keys that its last token sees (and the table can name)
  int blk0, blk1, nb;
  bool whole;      // the whole tile: its result is final
  int slot;        // workspace slot of a part: 0 for the CTA's first segment, 1 for its last
};

// The tile's tokens, keys and blocks; z0, z1 on the tile's own stretch of the line.
AK_D void set_blocks(const AttnArgs& a, const TileRule& t, int64_t cost, int64_t z0, int64_t z1,
                     Segment& s) {
  if (t.rows) {
    const int r0 = s.tile * t.rows, r1 = min(r0 + t.rows, s.r.n * a.G);  // (N G < 2^31)
    s.t_lo = r0 / a.G;
    s.t_hi = (r1 - 1) / a.G + 1;
  } else {
    s.t_lo = s.tile * t.tokens;
    s.t_hi = min(s.t_lo + t.tokens, s.r.n);
  }
  s.kv_hi = min(visible_keys(s.r, s.t_hi - 1, a.causal), capacity(a.l));
  s.nb = (int)(((int64_t)s.kv_hi + (1 << t.shift) - 1) >> t.shift);
  auto block = [&](int64_t z) {
    return z >= cost ? s.nb : (int)min((int64_t)s.nb, (z + (1 << t.shift) / 2) >> t.shift);
  };
  s.blk0 = block(z0);
  s.blk1 = block(z1);
  s.whole = s.blk0 == 0 && s.blk1 == s.nb;
}

// How a line is cut into pieces.
constexpr int kRounds = 5;
constexpr int64_t kLongPiece = 4096;  // shortest equal share that is worth rounds (3000: 64 : 76, 66 : 77 us)
struct Cut {
  int64_t unit;  // a piece of round r is size(r) units long
  int ctas;
  bool rounds;
  // 32, 16, 8, 5, 3 of 64
  AK_D static int size(int r) { return r == 0 ? 32 : r == 1 ? 16 : r == 2 ? 8 : r == 3 ? 5 : 3; }
  AK_D static int before(int r) { return r == 0 ? 0 : r == 1 ? 32 : r == 2 ? 48 : r == 3 ? 56 : r == 4 ? 61 : 64; }
  AK_D int64_t start(int piece) const {
    if (!rounds) return piece * unit;
    const int r = piece / ctas;
    return ((int64_t)ctas * before(r) + (int64_t)(piece - r * ctas) * size(r)) * unit;
  }
  AK_D int holds(int64_t x) const {  // the piece that holds point x
    const int64_t y = x / unit;
    if (!rounds) return (int)y;
    int r = 0;
    while (r < kRounds - 1 && y >= (int64_t)ctas * before(r + 1)) ++r;
    return r * ctas + (int)((y - (int64_t)ctas * before(r)) / size(r));
  }
};

// The line, how it is cut, and one of its pieces.
struct Line {
  Cut cut;
  int64_t total;
  int64_t x;      // the piece's start, or -1: there is no such piece
  int b;          // sequence that holds x
  int64_t b_at;   // where that sequence starts
};

AK_D int64_t line_cost(const AttnArgs& a, const TileRule& t, int64_t b) {
  return b < a.l.B ? a.Hkv * seq_cost(a, t, seq_range(a.l, (int)b)).total() : (int64_t)0;
}

// Another piece, for a whole warp: 32 sequences at a time.
AK_D void move_to_piece(const AttnArgs& a, const TileRule& t, Line& line, int piece) {
  const int lane = threadIdx.x & 31;
  line.x = line.cut.start(piece);
  if (line.x >= line.total) {
    line.x = -1;
    return;
  }
  int64_t run = 0;
  for (int64_t base = 0; base < a.l.B; base += 32) {
    const int64_t v = line_cost(a, t, base + lane);
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const int64_t at = run + inc - v;
    const unsigned hit = __ballot_sync(0xffffffffu, line.x >= at && line.x < at + v);
    if (hit) {
      line.b = (int)base + __ffs(hit) - 1;
      line.b_at = __shfl_sync(0xffffffffu, at, __ffs(hit) - 1);
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  line.x = -1;
}

// Run by the whole CTA, whose threads each take one sequence at a time.
AK_D Line find_piece(const AttnArgs& a, const TileRule& t, int piece) {
  __shared__ int64_t s_warp[32], s_at;
  __shared__ int s_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  auto cost_of = [&](int64_t b) { return line_cost(a, t, b); };
  // sum of the values before this thread's, and of all
  auto scan = [&](int64_t v, int64_t& all) {
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int64_t part = lane < nw ? s_warp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, part, o);
      if (lane >= o) part += y;
    }
    all = __shfl_sync(0xffffffffu, part, 31);
    const int64_t up_to = __shfl_sync(0xffffffffu, part, warp);
    return up_to - __shfl_sync(0xffffffffu, inc, 31) + inc - v;
  };
  Line line;
  const int64_t first = cost_of(threadIdx.x);
  int64_t at = scan(first, line.total);  // all there is, up to as many sequences as threads
  if (a.l.B > (int)blockDim.x) {
    int64_t more = 0, all;
    for (int64_t b = (int64_t)threadIdx.x + blockDim.x; b < a.l.B; b += blockDim.x) more += cost_of(b);
    __syncthreads();
    scan(more, all);
    line.total += all;
  }
  line.cut.ctas = t.ctas;
  line.cut.unit = max((line.total + t.ctas - 1) / t.ctas, t.min_piece);
  line.cut.rounds = t.rounds > 1 && line.cut.unit >= kLongPiece;
  if (line.cut.rounds) line.cut.unit = (line.cut.unit + 63) / 64;
  line.x = line.cut.start(piece);
  if (line.x >= line.total) {
    line.x = -1;
    return line;
  }
  int64_t v = first, run = 0;
  for (int64_t base = 0; base < a.l.B; base += blockDim.x) {
    if (base) {
      int64_t all;
      v = cost_of(base + threadIdx.x);
      __syncthreads();
      at = run + scan(v, all);
      run += all;
    } else if (a.l.B > (int)blockDim.x) {
      run = __syncthreads_or(0);  // (all have read s_warp)
      int64_t all;
      at = scan(v, all);
      run = all;
    }
    const bool mine = line.x >= at && line.x < at + v;
    if (mine) {
      s_b = (int)(base + threadIdx.x);
      s_at = at;
    }
    if (__syncthreads_or(mine)) {
      line.b = s_b;
      line.b_at = s_at;
      return line;
    }
  }
  line.x = -1;  // (not reached while nobody writes the lists)
  return line;
}

// Walks the segments of one piece, in order.
struct Walker {
  const AttnArgs& a;
  const TileRule& t;
  int64_t x, start, end, b_at;
  int b, loaded;
  SeqRange r;
  SeqCost c;
  int64_t head;  // length of one head of sequence b
  // the last tile that was come to, and where it lies on the line
  int last_b, last_h, last_tile;
  int64_t last_at, last_cost;

  AK_D Walker(const AttnArgs& a_, const TileRule& t_, const Line& line, int piece)
      : a(a_), t(t_), head(0), last_b(-1), last_h(0), last_tile(0), last_at(0), last_cost(0) {
    go(line, piece);
  }
  AK_D void go(const Line& line, int piece) {
    x = start = line.x;
    end = line.x < 0 ? x : min(line.cut.start(piece + 1), line.total);
    b_at = line.b_at;
    b = line.b;
    loaded = -1;
  }
  AK_D bool next(Segment& s) {
    while (x < end) {
      if (loaded != b) {
        r = seq_range(a.l, b);
        c = seq_cost(a, t, r);
        head = c.total();
        loaded = b;
      }
      if (x >= b_at + head * a.Hkv) {
        b_at += head * a.Hkv;
        if (++b >= a.l.B) return false;
        continue;
      }
      int64_t y = x - b_at;
      s.h = (int)(y / head);
      y -= s.h * head;
      s.r = r;
      s.b = b;
      s.tile = c.find(y);
      const int64_t cost = c.cost(s.tile), z0 = y - c.prefix(s.tile);
      last_b = b;
      last_h = s.h;
      last_tile = s.tile;
      last_at = x - z0;
      last_cost = cost;
      const int64_t z1 = min(cost, z0 + (end - x));
      s.slot = x == start ? 0 : 1;
      x += z1 - z0;
      set_blocks(a, t, cost, z0, z1, s);
      if (s.nb == 0) {
        if (z0 == 0) return true;  // no keys at all: its first part writes the zeros
      } else if (s.blk0 < s.blk1) {
        return true;
      }
    }
    return false;
  }
};

// ------------------------------------------------------------------ joining a tile's parts

// The predecessor on the stream has written its parts: every block of a join waits, also one that
// has nothing to join.
AK_D void wait_for_parts() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The parts of the tile that boundary blockIdx.x + 1 between two pieces cuts first, for a whole CTA.
struct Parts {
  Segment s;        // the tile
  int n;            // parts there are: none if the boundary is not the tile's first, or one CTA had it all
  int64_t at, cost;
  int first;        // piece of part 0
};
constexpr int kParts = 32;  // parts looked at in one go

AK_D Parts find_parts(const AttnArgs& a, const TileRule& t, Line& line) {
  Parts p;
  p.n = 0;
  const int c = blockIdx.x + 1;
  line = find_piece(a, t, c);
  if (line.x < 0) return p;
  p.s.b = line.b;
  p.s.r = seq_range(a.l, line.b);
  const SeqCost sc = seq_cost(a, t, p.s.r);
  const int64_t head = sc.total();
  int64_t y = line.x - line.b_at;
  p.s.h = (int)(y / head);
  y -= p.s.h * head;
  p.s.tile = sc.find(y);
  p.at = line.x - (y - sc.prefix(p.s.tile));
  p.cost = sc.cost(p.s.tile);
  if (p.at == line.x || p.at < line.cut.start(c - 1)) return p;  // not the tile's first boundary
  set_blocks(a, t, p.cost, 0, p.cost, p.s);
  p.first = c - 1;
  if (p.s.nb) p.n = line.cut.holds(p.at + p.cost - 1) - (c - 1) + 1;
  return p;
}

// What the join at boundary c has to know, left by the CTA of piece c - 1 (where join blocks find no
// room beside the main kernel, looking for it there would come after it).
struct Cutting {
  int b, h, tile, valid;
  int64_t at, cost, unit;
};
// of the last tile that a piece [start, end) came to
AK_D Cutting cutting_of(const Walker& w, const Line& line) {
  const bool first = w.last_b >= 0 && w.last_at >= w.start && w.last_at + w.last_cost > w.end;
  return Cutting{w.last_b, w.last_h, w.last_tile, first, w.last_at, w.last_cost, line.cut.unit};
}
AK_D Parts parts_of(const AttnArgs& a, const TileRule& t, const Cutting& k, Line& line) {
  Parts p;
  p.n = 0;
  if (!k.valid) return p;
  line.cut = Cut{k.unit, t.ctas, false};
  p.s.b = k.b;
  p.s.h = k.h;
  p.s.tile = k.tile;
  p.s.r = seq_range(a.l, k.b);
  p.at = k.at;
  p.cost = k.cost;
  p.first = blockIdx.x;
  set_blocks(a, t, p.cost, 0, p.cost, p.s);
  if (p.s.nb) p.n = line.cut.holds(p.at + p.cost - 1) - p.first + 1;
  return p;
}

// Workspace slot (2 * piece + which) of part i, or -1 when it holds no block; *whole when it holds all.
AK_D int part_slot(const AttnArgs& a, const TileRule& t, const Line& line, const Parts& p, int i, bool& whole) {
  Segment s = p.s;
  const int64_t from = line.cut.start(p.first + i), to = line.cut.start(p.first + i + 1);
  set_blocks(a, t, p.cost, max(from - p.at, (int64_t)0), min(p.cost, to - p.at), s);
  whole = s.whole;
  return s.blk0 < s.blk1 ? 2 * (p.first + i) + (from >= p.at ? 0 : 1) : -1;
}

// Page numbers of consecutive boxes of a tile's keys, for a whole warp: 32 are loaded at once and the
// next 32 while those are used (a load per block, used at once, bounded the producer: about 2000
// cycles a block).  Nothing touches a loaded number before its box is asked for.
struct PageFeed {
  int raw, slot, key;                 // this lane's box of the current 32: table entry, slot, first key
  int next_raw, next_slot, next_key;
  int base;                           // first box of the current 32
  AK_D void fetch(const AttnArgs& a, const Segment& s, int first, int box, int& r, int& sl, int& k) {
    const int64_t at = ((int64_t)first + (threadIdx.x & 31)) * box;
    r = -2;  // behind the last key
    k = 0x7fffffff;
    sl = 0;
    if (at < s.kv_hi) {
      k = (int)at;
      const int i = k / a.l.page_size;
      sl = k - i * a.l.page_size;
      r = __ldg(a.l.page_table + (int64_t)s.b * a.l.table_ld + i);  // kv_hi is within the table
    }
  }
  AK_D void start(const AttnArgs& a, const Segment& s, int first, int box) {
    base = first;
    fetch(a, s, first, box, raw, slot, key);
    fetch(a, s, first + 32, box, next_raw, next_slot, next_key);
  }
  // makes box i (at most 32 behind the last one asked for) current
  AK_D void reach(const AttnArgs& a, const Segment& s, int i, int box) {
    if (i < base + 32) return;
    base += 32;
    raw = next_raw;
    slot = next_slot;
    key = next_key;
    fetch(a, s, base + 32, box, next_raw, next_slot, next_key);
  }
  // page and slot of box i: a page that does not exist (and slot 0) where the key has none
  AK_D void get(const PagedLists& l, int i, int& page, int& slot_) const {
    const bool ok = (unsigned)raw < (unsigned)l.num_pages;
    page = __shfl_sync(0xffffffffu, ok ? raw : l.num_pages, i - base);
    slot_ = __shfl_sync(0xffffffffu, ok ? slot : 0, i - base);
  }
  // first key of boxes [i, i + n) that the tile needs and that has no page
  AK_D int missing(const PagedLists& l, int i, int n) const {
    const int lane = threadIdx.x & 31;
    const bool bad = (unsigned)raw >= (unsigned)l.num_pages && lane >= i - base && lane < i - base + n;
    return __reduce_min_sync(0xffffffffu, bad ? key : 0x7fffffff);
  }
};

// ------------------------------------------------------------------ rows that get a second look
// The matrix instructions multiply a hidden key's value by a weight of 0, which is NaN when the
// value is not finite.  A row whose result is not finite although its sum of weights is, and that
// shares its tile with keys hidden from it, is looked at again: if a hidden value may be the cause,
// the row is computed from its visible keys alone.  Going through a long context key by key takes
// milliseconds, so that never happens in a kernel whose warps wait for one another (they give up after
// two seconds): the main kernels only mark the piece, and a kernel that comes after them and waits for
// nothing within does the rows (200 rows of 200,000 keys: 1.4 s).

template <int D>
struct AgainScratch {
  int last;
  RowScratch<D / 8, 128> row;
};

// The last key of [lo, hi) whose value is not finite, or -1; for a whole CTA.  16-bit types.
template <int DT, int D>
AK_D int last_not_finite(const AttnArgs& a, int b, int hk, int lo, int hi, int& s_last) {
  using E = Elem<DT>;
  using T = typename E::T;
  if (threadIdx.x == 0) s_last = -1;
  __syncthreads();
  constexpr int VECS = D / 8;
  int last = -1;
  for (int i = threadIdx.x; i < (hi - lo) * VECS; i += blockDim.x) {  // (as many keys as a tile has tokens)
    const int j = lo + i / VECS;
    const int page = page_of(a.l, b, j / a.l.page_size);
    if (page < 0) continue;
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(
        reinterpret_cast<const T*>(a.v) + page * a.vcs[0] + hk * a.vcs[1] + (j % a.l.page_size) * a.vcs[2] + i % VECS * 8));
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad |= !(fabsf(E::to_f(reinterpret_cast<const T*>(&raw)[e])) <= 3.4028235e38f);
    if (bad) last = j;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if ((threadIdx.x & 31) == 0) atomicMax(&s_last, last);
  __syncthreads();
  return s_last;
}

// Rows [i0, i1) of tile s, by a CTA of 128 threads.
template <int DT, int D>
AK_D void look_again_at_tile(const AttnArgs& a, const TileRule& rule, const Segment& s, int i0, int i1,
                             AgainScratch<D>& sh) {
  using T = typename Elem<DT>::T;
  const int last = last_not_finite<DT, D>(a, s.b, s.h, visible_keys(s.r, s.t_lo, a.causal), s.kv_hi, sh.last);
  __syncthreads();  // (before the next tile's search)
  for (int i = i0; i < i1 && last >= 0; ++i) {
    int t, hg;
    bool valid;
    if (rule.rows) {  // rows follow one another
      const int row = s.tile * rule.rows + i;
      t = row / a.G;
      hg = row % a.G;
      valid = t < s.t_hi;
    } else {  // two tiles of rule.tokens / 2 tokens
      const int tt = rule.tokens / 2, row = i % 128;
      t = s.t_lo + i / 128 * tt + row / a.G;
      hg = row % a.G;
      valid = row < tt * a.G && t < s.t_hi;
    }
    if (!valid || visible_keys(s.r, t, a.causal) > last) continue;
    const T* o = reinterpret_cast<const T*>(a.o) + (int64_t)(s.r.begin + t) * a.os[0] + (int64_t)(s.h * a.G + hg) * a.os[1];
    const bool bad = threadIdx.x < D && !(fabsf(Elem<DT>::to_f(o[threadIdx.x])) <= 3.4028235e38f);
    if (__syncthreads_or(bad)) row_by_cta<DT, D / 8, 128>(a, s.b, s.r, t, s.h * a.G + hg, sh.row);
  }
}

// Those rows of tile s (if `again`) and of every tile that piece `piece` has all of (if `marked`).
template <int DT, int D>
AK_D void look_again(const AttnArgs& a, const TileRule& rule, Segment s, bool again, bool marked, int piece, int i0,
                     int i1, AgainScratch<D>& sh) {
  if (!again && !marked) return;
  Line line;
  line.x = -1;
  if (marked) line = find_piece(a, rule, piece);
  Walker walk(a, rule, line, piece);
  while (again || walk.next(s)) {
    if (again || (s.whole && s.nb && a.causal && s.t_hi - s.t_lo > 1)) look_again_at_tile<DT, D>(a, rule, s, i0, i1, sh);
    again = false;
  }
}

}  // namespace paged
}  // namespace ak
