// Appending keys and values to a paged cache with the rotary position embedding on the way
// (interleaved pairs, the math of reference.py:63-69 with fp32 tables and one rounding, as
// models/llama_7b.py:40-48 rotates):
//   cache_k[page, h, slot] = rot(k[t, h], p),  cache_v[page, h, slot] = v[t, h],
//   q_out[t, h] = rot(q[t, h], p)   for token t at position p.
//
// Bound by bytes: each of q, k, v is read once and written once, the rotation is six fp32
// operations a pair.  One CTA takes one token (or a slice of its heads when there are few tokens);
// a thread owns one 16-byte vector of the head dimension and walks the heads, so a thread's cos
// and sin are loaded once for all of them, and the data loads, which need nothing but the token's
// number, are in flight while the token's sequence and page are looked up.
//
// Measured, 32 + 2 x 32 heads of 128, bf16: 12,750 tokens in 108 us, 5.9 TB/s (90% of a plain copy's
// rate; 129 us before k, v and q had loops of their own, which leaves 64 registers and four CTAs per
// SM); one token 4.1 us, a launch and the dependent loads of its place.
#include "paged.cuh"

#include <type_traits>

namespace ak {
namespace {

struct AppendArgs {
  PagedLists l;
  const void *k, *v, *q;
  void *k_cache, *v_cache, *q_out;
  const float *cos, *sin;  // [positions, D / 2], or null: no rotation
  int H, Hkv, D, positions;
  int64_t ks[2], vs[2], qs[2], os[2];  // {token, head}
  int64_t kcs[3], vcs[3];              // {page, head, slot}
};

// Where token t goes.  page < 0: stored nowhere; seq < 0: the token belongs to no sequence.
struct Place {
  int seq, pos, page, slot;
};

AK_D Place place_of(const PagedLists& l, int t) {
  Place w{-1, 0, -1, 0};
  const int b = seq_of_token_warp(l, t);
  if (b < 0 || b >= l.B) return w;
  const SeqRange r = seq_range(l, b);
  if (t < r.begin || t >= r.begin + r.n) return w;
  w.seq = b;
  w.pos = r.kv_len - r.n + (t - r.begin);
  if (w.pos < 0) return w;
  const int i = w.pos / l.page_size;
  w.slot = w.pos - i * l.page_size;
  w.page = page_of(l, b, i);
  return w;
}

template <int DT>
__global__ void __launch_bounds__(256, 4) append_vec_kernel(const __grid_constant__ AppendArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VEC = E::kVec, P = VEC / 2;
  constexpr int U = 2;  // vectors of each tensor in flight per thread
  const int vph = a.D / VEC;
  const int dv = threadIdx.x % vph, h0 = blockIdx.y * (blockDim.x / vph) + threadIdx.x / vph;
  const int step = gridDim.y * (blockDim.x / vph);  // this thread's heads: h0, h0 + step, ...
  const int t = blockIdx.x;
  const T* kp = reinterpret_cast<const T*>(a.k) + t * a.ks[0] + dv * VEC;
  const T* vp = reinterpret_cast<const T*>(a.v) + t * a.vs[0] + dv * VEC;
  const T* qp = reinterpret_cast<const T*>(a.q) + t * a.qs[0] + dv * VEC;
  auto at = [](const T* p, int64_t off) { return __ldcs(reinterpret_cast<const uint4*>(p + off)); };
  const int H = a.q ? a.H : 0;

  uint4 k[U], v[U], q[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * step;
    if (h < a.Hkv) k[u] = at(kp, h * a.ks[1]);
    if (h < a.Hkv) v[u] = at(vp, h * a.vs[1]);
    if (h < H) q[u] = at(qp, h * a.qs[1]);
  }

  __shared__ Place s_place;
  if (threadIdx.x < 32) {
    const Place w = place_of(a.l, t);
    if (threadIdx.x == 0) s_place = w;
  }
  __syncthreads();
  const Place w = s_place;
  if (w.seq < 0) return;  // behind the last sequence: left as it is

  float c[P], s[P];
  if (a.cos) {
    const bool in = (unsigned)w.pos < (unsigned)a.positions;  // no angle is known elsewhere: NaN
    const int64_t off = in ? (int64_t)w.pos * (a.D / 2) + dv * P : 0;
    using V = typename std::conditional<P == 4, float4, float2>::type;
    const V cv = __ldg(reinterpret_cast<const V*>(a.cos + off));
    const V sv = __ldg(reinterpret_cast<const V*>(a.sin + off));
#pragma unroll
    for (int i = 0; i < P; ++i) {
      c[i] = in ? reinterpret_cast<const float*>(&cv)[i] : __int_as_float(0x7fffffff);
      s[i] = in ? reinterpret_cast<const float*>(&sv)[i] : __int_as_float(0x7fffffff);
    }
  }
  auto turned = [&](uint4 x) {
    if (!a.cos) return x;
    T* e = reinterpret_cast<T*>(&x);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float x1 = E::to_f(e[2 * i]), x2 = E::to_f(e[2 * i + 1]);
      e[2 * i] = E::from_f(fmaf(x1, c[i], -x2 * s[i]));
      e[2 * i + 1] = E::from_f(fmaf(x1, s[i], x2 * c[i]));
    }
    return x;
  };
  if (w.page >= 0) {
    T* kd = reinterpret_cast<T*>(a.k_cache) + w.page * a.kcs[0] + w.slot * a.kcs[2] + dv * VEC;
    T* vd = reinterpret_cast<T*>(a.v_cache) + w.page * a.vcs[0] + w.slot * a.vcs[2] + dv * VEC;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * step;
      if (h >= a.Hkv) break;
      *reinterpret_cast<uint4*>(kd + h * a.kcs[1]) = turned(k[u]);
      *reinterpret_cast<uint4*>(vd + h * a.vcs[1]) = v[u];
    }
    for (int h = h0 + U * step; h < a.Hkv; h += step) {
      const uint4 x = at(kp, h * a.ks[1]), y = at(vp, h * a.vs[1]);
      *reinterpret_cast<uint4*>(kd + h * a.kcs[1]) = turned(x);
      *reinterpret_cast<uint4*>(vd + h * a.vcs[1]) = y;
    }
  }
  T* qd = reinterpret_cast<T*>(a.q_out) + t * a.os[0] + dv * VEC;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * step;
    if (h < H) *reinterpret_cast<uint4*>(qd + h * a.os[1]) = turned(q[u]);
  }
  for (int h = h0 + U * step; h < H; h += step)
    *reinterpret_cast<uint4*>(qd + h * a.os[1]) = turned(at(qp, h * a.qs[1]));
}

// Any even head dimension, stride and alignment: one thread per pair.
template <int DT>
__global__ void __launch_bounds__(256) append_scalar_kernel(const __grid_constant__ AppendArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  const int t = blockIdx.x;
  __shared__ Place s_place;
  if (threadIdx.x < 32) {
    const Place w = place_of(a.l, t);
    if (threadIdx.x == 0) s_place = w;
  }
  __syncthreads();
  const Place w = s_place;
  if (w.seq < 0) return;
  const int half = a.D / 2, heads = 2 * a.Hkv + (a.q ? a.H : 0);
  const bool in = (unsigned)w.pos < (unsigned)a.positions;
  for (int64_t g = threadIdx.x; g < (int64_t)heads * half; g += blockDim.x) {
    const int h = (int)(g / half), i = (int)(g - (int64_t)h * half);
    const T* src;
    T* dst;
    bool rot = a.cos != nullptr;
    if (h < 2 * a.Hkv && w.page < 0) continue;
    if (h < a.Hkv) {
      src = reinterpret_cast<const T*>(a.k) + t * a.ks[0] + h * a.ks[1];
      dst = reinterpret_cast<T*>(a.k_cache) + w.page * a.kcs[0] + h * a.kcs[1] + w.slot * a.kcs[2];
    } else if (h < 2 * a.Hkv) {
      src = reinterpret_cast<const T*>(a.v) + t * a.vs[0] + (h - a.Hkv) * a.vs[1];
      dst = reinterpret_cast<T*>(a.v_cache) + w.page * a.vcs[0] + (h - a.Hkv) * a.vcs[1] +
            w.slot * a.vcs[2];
      rot = false;
    } else {
      src = reinterpret_cast<const T*>(a.q) + t * a.qs[0] + (h - 2 * a.Hkv) * a.qs[1];
      dst = reinterpret_cast<T*>(a.q_out) + t * a.os[0] + (h - 2 * a.Hkv) * a.os[1];
    }
    const T e0 = src[2 * i], e1 = src[2 * i + 1];
    if (rot) {
      const float c = in ? a.cos[(int64_t)w.pos * half + i] : __int_as_float(0x7fffffff);
      const float s = in ? a.sin[(int64_t)w.pos * half + i] : __int_as_float(0x7fffffff);
      const float x1 = E::to_f(e0), x2 = E::to_f(e1);
      dst[2 * i] = E::from_f(fmaf(x1, c, -x2 * s));
      dst[2 * i + 1] = E::from_f(fmaf(x1, s, x2 * c));
    } else {
      dst[2 * i] = e0;
      dst[2 * i + 1] = e1;
    }
  }
}

bool multiple(const int64_t* s, int n, int64_t of) {
  for (int i = 0; i < n; ++i)
    if (s[i] % of) return false;
  return true;
}

template <int DT>
int run_append(const AppendArgs& a, cudaStream_t st) {
  constexpr int VEC = Elem<DT>::kVec;
  bool vec = a.D % VEC == 0 && a.D / VEC <= 256 && aligned16(a.k) && aligned16(a.v) &&
             aligned16(a.k_cache) && aligned16(a.v_cache) && multiple(a.ks, 2, VEC) &&
             multiple(a.vs, 2, VEC) && multiple(a.kcs, 3, VEC) && multiple(a.vcs, 3, VEC);
  if (a.q)
    vec = vec && aligned16(a.q) && aligned16(a.q_out) && multiple(a.qs, 2, VEC) &&
          multiple(a.os, 2, VEC);
  // a row of the tables is D / 2 floats, so every vector's piece is aligned with the first
  vec = vec && aligned16(a.cos) && aligned16(a.sin);
  if (!vec) {
    append_scalar_kernel<DT><<<a.l.N, 256, 0, st>>>(a);
    return launch_status("paged_append");
  }
  const int vph = a.D / VEC;
  const int threads = vph * (256 / vph);
  const int most = a.q && a.H > a.Hkv ? a.H : a.Hkv, at_once = threads / vph;
  // few tokens: their heads spread over more CTAs, until every SM has one
  int split = 1;
  while (split * at_once < most && (int64_t)a.l.N * split < device_info().sm_count) ++split;
  append_vec_kernel<DT><<<dim3((unsigned)a.l.N, (unsigned)split), threads, 0, st>>>(a);
  return launch_status("paged_append");
}

}  // namespace
}  // namespace ak

using namespace ak;

extern "C" int ak_paged_append(const void* k, const void* v, const void* q, void* q_out,
                               void* k_cache, void* v_cache, const int32_t* page_table,
                               const int32_t* cu_q, const int32_t* kv_lens, const float* cos,
                               const float* sin, int64_t N, int64_t B, int64_t H, int64_t Hkv,
                               int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages,
                               int64_t table_ld, int64_t positions, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* q_strides,
                               const int64_t* q_out_strides, const int64_t* k_cache_strides,
                               const int64_t* v_cache_strides, int dtype, void* stream) {
  AK_REQUIRE(dtype_ok(dtype), AK_ERR_DTYPE, "unsupported dtype %d", dtype);
  AK_REQUIRE(N >= 0 && B >= 0 && Hkv > 0 && D > 0 && num_pages >= 0 && page_size > 0 &&
                 max_pages >= 0 && table_ld >= 0 && positions >= 0,
             AK_ERR_SHAPE, "bad shape");
  AK_REQUIRE(D % 2 == 0, AK_ERR_SHAPE, "head_dim must be even, got %lld", (long long)D);
  AK_REQUIRE(N < (1LL << 31) && B < (1LL << 31) - 64 && H < (1LL << 24) && Hkv < (1LL << 24) &&
                 D <= 65536 && num_pages < (1LL << 31) && page_size < (1LL << 31) &&
                 max_pages < (1LL << 31) && positions < (1LL << 31),
             AK_ERR_SHAPE, "dimension too large");
  AK_REQUIRE(!q || H > 0, AK_ERR_SHAPE, "q given with %lld heads", (long long)H);
  AK_REQUIRE((cos == nullptr) == (sin == nullptr), AK_ERR_ARG, "cos and sin go together");
  AK_REQUIRE(!cos || positions > 0, AK_ERR_SHAPE, "cos and sin hold no position");
  if (N == 0 || B == 0) return AK_OK;
  AK_REQUIRE(k && v && cu_q && kv_lens && k_strides && v_strides && k_cache_strides && v_cache_strides &&
                 ((k_cache && v_cache) || num_pages == 0) && (page_table || max_pages == 0),
             AK_ERR_ARG, "null pointer");
  AK_REQUIRE(!q || (q_out && q_strides && q_out_strides), AK_ERR_ARG, "q without q_out");
  const int64_t cache[3] = {num_pages, Hkv, page_size}, tokens[2] = {N, H};
  AK_REQUIRE(num_pages == 0 || (k_cache != v_cache && !may_overlap(cache, k_cache_strides, 3, D) &&
                                !may_overlap(cache, v_cache_strides, 3, D)),
             AK_ERR_ARG, "the caches overlap each other or themselves");
  AK_REQUIRE(!q || !may_overlap(tokens, q_out_strides, 2, D), AK_ERR_ARG, "q_out overlaps itself");
  AK_REQUIRE(!q || (q_out != k && q_out != v && q_out != k_cache && q_out != v_cache &&
                    (q_out != q || (q_strides[0] == q_out_strides[0] && q_strides[1] == q_out_strides[1]))),
             AK_ERR_ARG, "q_out overlaps another tensor (it may only be q itself)");
  AppendArgs a{};
  a.l = PagedLists{page_table, cu_q,           kv_lens,        table_ld,      (int)N,
                   (int)B,     (int)max_pages, (int)num_pages, (int)page_size};
  a.k = k; a.v = v; a.q = q;
  a.k_cache = k_cache; a.v_cache = v_cache; a.q_out = q_out;
  a.cos = cos; a.sin = sin;
  a.H = (int)H; a.Hkv = (int)Hkv; a.D = (int)D; a.positions = (int)positions;
  for (int i = 0; i < 2; ++i) {
    a.ks[i] = k_strides[i];
    a.vs[i] = v_strides[i];
    a.qs[i] = q ? q_strides[i] : 0;
    a.os[i] = q ? q_out_strides[i] : 0;
  }
  for (int i = 0; i < 3; ++i) {
    a.kcs[i] = k_cache_strides[i];
    a.vcs[i] = v_cache_strides[i];
  }
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AK_F32: return run_append<AK_F32>(a, st);
    case AK_F16: return run_append<AK_F16>(a, st);
    default: return run_append<AK_BF16>(a, st);
  }
}
