// Attention of packed new tokens over a paged key/value cache: entry point and the SIMT kernel
// that takes every type, head dimension, stride and page size.
//
//   o[t, h] = sum_{j < vis(t)} softmax_j(scale q[t, h] . K[j, h / G]) V[j, h / G],  G = H / Hkv,
//   vis(t) = position(t) + 1 (causal) or kv_lens[b].
// A row that sees no key is 0.  A row that would see a key without a page (paged.cuh) is NaN.
#include "paged_row.cuh"

namespace ak {
namespace paged {

// One CTA per (token, head): keys are read again by every token and head of a group.  Measured, fp32, 32 heads over
// 8 of 128: one token on 2011 keys 160 us (its bytes would take 2.5), 64 of them on 300 to 4100 keys 1.73 ms
// (0.18), a chunk of 501 on 3501 keys 12.2 ms; bf16, heads of 80: 0.11, 1.03 and 7.9 ms.
template <int DT, int NI>
__global__ void __launch_bounds__(256) simt_kernel(const AttnArgs a) {
  const int t = blockIdx.x;
  __shared__ int s_seq;
  __shared__ RowScratch<NI, 256> scratch;
  if (threadIdx.x < 32) {
    const int b = seq_of_token_warp(a.l, t);
    if (threadIdx.x == 0) s_seq = b;
  }
  __syncthreads();
  const int b = s_seq;
  if (b < 0 || b >= a.l.B) return;
  const SeqRange r = seq_range(a.l, b);
  if (t < r.begin || t >= r.begin + r.n) return;
  row_by_cta<DT, NI, 256>(a, b, r, t - r.begin, blockIdx.y, scratch);
}

template <int DT>
static int run_simt(const AttnArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.l.N, (unsigned)a.H);
  if (a.D <= 64)
    simt_kernel<DT, 8><<<grid, 256, 0, st>>>(a);
  else if (a.D <= 128)
    simt_kernel<DT, 16><<<grid, 256, 0, st>>>(a);
  else
    simt_kernel<DT, 32><<<grid, 256, 0, st>>>(a);
  return launch_status("paged_attention");
}

// The tensor-core kernels read pages by TMA (16-byte multiples, boxes of at least the eight slots of a
// swizzle atom) and lay all tiles on one 64-bit line.
static bool tc_ok(const AttnArgs& a) {
  if (force_simt() || a.dtype == AK_F32 || (a.D != 64 && a.D != 128) || a.l.page_size % 8 || a.G > 128)
    return false;
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.o)) return false;
  if (a.l.num_pages == 0 || (int64_t)a.l.N * a.G >= (1LL << 31)) return false;
  auto ok = [](int64_t size, int64_t stride) {
    return size <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1LL << 38));
  };
  const int64_t cache[3] = {a.l.num_pages, a.Hkv, a.l.page_size}, tokens[2] = {a.l.N, a.H};
  for (int i = 0; i < 3; ++i)
    if (!ok(cache[i], a.kcs[i]) || !ok(cache[i], a.vcs[i])) return false;
  for (int i = 0; i < 2; ++i)
    if (!ok(tokens[i], a.qs[i]) || !ok(tokens[i], a.os[i])) return false;
  // (the line of lists that give every sequence all tokens fits too)
  const double keys = (double)a.l.max_pages * a.l.page_size;
  if (((double)a.l.N * a.G + 1) * a.l.B * a.Hkv *
          ((keys < 2147483647.0 ? keys : 2147483647.0) + a.l.N + 1024) > 4e18)
    return false;
  return device_info().cc_major == 10;
}

// The decoding kernel for few query rows a sequence and key/value head, on average: its tiles of 16 rows each
// read all keys and are put together row by row, where the chunk kernel's 256 rows read them once.  Rows
// are what the host knows (N G / B); how they spread over the sequences it does not.  Measured, us, decoding
// kernel : chunk kernel, heads of 128, bf16:
//   rows 1   64 x 300..8100 keys, 32 heads   645 : 938       1 x 2000, 32 heads          22 : 31
//   rows 4   the same, 32 over 8 heads       197 : 253       16 x 300..8000, 32 over 8   80 : 79
//   rows 8   128 x 300..4000, 32 over 8      222 : 306       1 x 4000, 32 over 8         40 : 30
//   rows 16  64 x 300..8100, 32 over 2       121 : 81        1 x 4000, 32 over 2         59 : 28
// Between 5 and 9 rows the joins at the ends of pieces decide: the decoding kernel is ahead where an SM has two
// (sequence, head) pairs or more, whose loads hide them (48 x 300..8000, 32 over 8: 173 : 195; 50..500: 57 : 53).
// One sequence of two tokens among 63 of one (32 over 8) is 197 : 254; 63 and a chunk of 512, 32 heads, 9
// rows, 711 : 1338.  A call with room for 64 sequences that holds one chunk of 64 tokens is the worst of it,
// 72 : 35 (nothing the host sees tells it from 64 of one).
static bool few_rows(int64_t N, int64_t B, int64_t G, int64_t Hkv) {
  return N * G <= 5 * B || (N * G <= 9 * B && B * Hkv >= 2 * (int64_t)device_info().sm_count);
}

}  // namespace paged
}  // namespace ak

using namespace ak;

extern "C" size_t ak_paged_attention_workspace_size(int64_t N, int64_t B, int64_t H, int64_t Hkv,
                                                    int64_t D, int dtype) {
  if (dtype == AK_F32 || (D != 64 && D != 128) || Hkv <= 0) return 0;
  return paged::few_rows(N, B, H / Hkv, Hkv) ? paged::decode_workspace((int)D) : paged::chunk_workspace((int)D);
}

extern "C" int ak_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                                  void* out, const int32_t* page_table, const int32_t* cu_q,
                                  const int32_t* kv_lens, int64_t N, int64_t B, int64_t H,
                                  int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                                  int64_t max_pages, int64_t table_ld, const int64_t* q_strides,
                                  const int64_t* out_strides, const int64_t* k_cache_strides,
                                  const int64_t* v_cache_strides, int causal, float sm_scale,
                                  int dtype, void* workspace, size_t ws_bytes, void* stream) {
  AK_REQUIRE(dtype_ok(dtype), AK_ERR_DTYPE, "unsupported dtype %d", dtype);
  AK_REQUIRE(N >= 0 && B >= 0 && H > 0 && Hkv > 0 && D > 0 && num_pages >= 0 && page_size > 0 &&
                 max_pages >= 0 && table_ld >= 0,
             AK_ERR_SHAPE, "bad shape");
  AK_REQUIRE(H % Hkv == 0, AK_ERR_SHAPE, "query heads %lld not a multiple of kv heads %lld",
             (long long)H, (long long)Hkv);
  AK_REQUIRE(D <= 256, AK_ERR_SHAPE, "head_dim %lld exceeds 256", (long long)D);
  AK_REQUIRE(N < (1LL << 31) && B < (1LL << 31) - 64 && H <= 65535 && num_pages < (1LL << 31) &&
                 page_size < (1LL << 31) && max_pages < (1LL << 31),
             AK_ERR_SHAPE, "dimension too large");
  AK_REQUIRE(sm_scale > 0.f && sm_scale <= 2.3e38f, AK_ERR_ARG,  // (times log2(e) it must be finite too)
             "sm_scale must be positive and finite");
  if (N == 0 || B == 0) return AK_OK;
  AK_REQUIRE(q && out && cu_q && kv_lens && q_strides && out_strides && k_cache_strides && v_cache_strides &&
                 ((k_cache && v_cache) || num_pages == 0) && (page_table || max_pages == 0),
             AK_ERR_ARG, "null pointer");
  const int64_t tokens[2] = {N, H};
  AK_REQUIRE(!may_overlap(tokens, out_strides, 2, D), AK_ERR_ARG, "out overlaps itself");
  AK_REQUIRE(out != q && out != k_cache && out != v_cache, AK_ERR_ARG, "out overlaps an input");
  const size_t need = ak_paged_attention_workspace_size(N, B, H, Hkv, D, dtype);
  AK_REQUIRE(need == 0 || (workspace && aligned16(workspace) && ws_bytes >= need), AK_ERR_ARG,
             "workspace of %zu bytes (16-byte aligned) needed, %zu given", need, ws_bytes);
  paged::AttnArgs a{};
  a.l = PagedLists{page_table, cu_q,           kv_lens,        table_ld,      (int)N,
                   (int)B,     (int)max_pages, (int)num_pages, (int)page_size};
  a.q = q; a.k = k_cache; a.v = v_cache; a.o = out;
  a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv); a.D = (int)D;
  a.causal = causal;
  a.dtype = dtype;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q_strides[i];
    a.os[i] = out_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    a.kcs[i] = k_cache_strides[i];
    a.vcs[i] = v_cache_strides[i];
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (paged::tc_ok(a))
    return paged::few_rows(N, B, a.G, Hkv) ? paged::run_decode(a, workspace, st) : paged::run_chunk(a, workspace, st);
  switch (dtype) {
    case AK_F32: return paged::run_simt<AK_F32>(a, st);
    case AK_F16: return paged::run_simt<AK_F16>(a, st);
    default: return paged::run_simt<AK_BF16>(a, st);
  }
}
