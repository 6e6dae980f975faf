// Attention over a paged key-value cache: one new token per sequence
// (zs_paged_decode_attention) and packed new tokens (zs_paged_prompt_attention).
//
// o = sum_k softmax_k(q . K_k * scale) V_k over the keys k <= p of the query's
// sequence (p its position, p - k < window where a window is given), with an
// optional sink logit q . k_sink * scale whose value is zero and an optional
// sigmoid gate on o.  A row that sees no key is zero, its log-sum-exp the sink
// logit or -inf.
#include "zs_common.cuh"

namespace zs {
namespace paged {

struct AttnArgs {
  const void* q;               // [tokens, H, hd] rows of ldq elements
  int64_t ldq;
  const void* k_pages;         // [num_pages, Hkv, page, hd]
  const void* v_pages;
  int64_t page_stride;
  int64_t num_pages;
  const int* block_table;      // [num_seqs, max_pages] rows of bt_ld
  int64_t bt_ld;
  int max_pages;
  const int* seq_lens;         // [num_seqs] tokens in the cache, the new ones included
  const int* cu;               // [num_seqs + 1] first token of each sequence (null: one token each)
  int num_seqs;
  int64_t tokens;
  int H, Hkv, page;
  int window;                  // 0: none
  float scale, scale_log2;
  const void* k_sink;          // nullable [H, hd]
  int sink_dtype;
  const void* gate;            // nullable [tokens, H] rows of ldg elements
  int64_t ldg;
  void* o;                     // [tokens, H, hd] packed
  float* lse;                  // nullable [tokens, H]
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == ZS_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == ZS_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

// A sequence's length, no longer than its row of the block table.
__device__ __forceinline__ int cut_length(const AttnArgs& a, int seq) {
  const int len = __ldg(a.seq_lens + seq), cap = a.max_pages * a.page;
  if (len > cap) record_error(ZS_DEVERR_INDEX);
  return len > cap ? cap : len;
}

// Plain form: one block per (token, head), four warps over the keys, an online
// softmax per warp, joined at the end.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const AttnArgs a) {
  constexpr int E = HD / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][HD];
  const int64_t tok = blockIdx.x;
  const int h = blockIdx.y, hk = h / (a.H / a.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int seq = (int)tok;
  int64_t pos;
  if (a.cu != nullptr) {
    seq = sequence_of(a.cu, a.num_seqs, (int)tok);
    if (seq < 0) {                     // a row of no sequence: zero
      for (int e = threadIdx.x; e < HD; e += 128) reinterpret_cast<T*>(a.o)[(tok * a.H + h) * HD + e] = from_f32<T>(0.f);
      if (a.lse != nullptr && threadIdx.x == 0) a.lse[tok * a.H + h] = -INFINITY;
      return;
    }
    pos = (int64_t)cut_length(a, seq) - a.cu[seq + 1] + tok;
  } else {
    pos = (int64_t)cut_length(a, seq) - 1;
  }
  const T* q = reinterpret_cast<const T*>(a.q) + tok * a.ldq + (int64_t)h * HD;
  float qv[E], ov[E];
  float m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    qv[e] = to_f32(q[lane * E + e]);
    ov[e] = 0.f;
  }
  if (a.k_sink != nullptr && warp == 0) {
    float dot = 0.f;
    for (int e = 0; e < E; ++e) dot = fmaf(qv[e], load_any(a.k_sink, a.sink_dtype, (int64_t)h * HD + lane * E + e), dot);
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    m = dot * a.scale;
    l = 1.f;
  }
  const int64_t first = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  for (int64_t k = first + warp; k <= pos; k += 4) {
    const int pg = a.block_table[seq * a.bt_ld + k / a.page];
    if (pg < 0 || pg >= a.num_pages) {
      if (lane == 0) record_error(ZS_DEVERR_INDEX);
    }
    const bool ok = pg >= 0 && pg < a.num_pages;
    const int64_t at = (ok ? pg : 0) * a.page_stride + ((int64_t)hk * a.page + k % a.page) * HD + lane * E;
    float dot = 0.f;
    for (int e = 0; e < E; ++e)
      dot = fmaf(qv[e], ok ? to_f32(reinterpret_cast<const T*>(a.k_pages)[at + e]) : 0.f, dot);
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float s = dot * a.scale, mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
    l = l * f + p;
    for (int e = 0; e < E; ++e)
      ov[e] = ov[e] * f + p * (ok ? to_f32(reinterpret_cast<const T*>(a.v_pages)[at + e]) : 0.f);
    m = mn;
  }
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = ov[e];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  if (threadIdx.x < HD) {
    float mx = -INFINITY;
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, s_m[w]);
    float lt = 0.f, o = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - mx);
      lt += f * s_l[w];
      o += f * s_o[w][threadIdx.x];
    }
    float inv = lt > 0.f ? 1.f / lt : 0.f;
    if (a.gate != nullptr)
      inv *= 1.f / (1.f + expf(-to_f32(reinterpret_cast<const T*>(a.gate)[tok * a.ldg + h])));
    reinterpret_cast<T*>(a.o)[(tok * a.H + h) * HD + threadIdx.x] = from_f32<T>(o * inv);
    if (a.lse != nullptr && threadIdx.x == 0) a.lse[tok * a.H + h] = lt > 0.f ? mx + logf(lt) : -INFINITY;
  }
}

}  // namespace paged
}  // namespace zs

using namespace zs;

static int attn_args(paged::AttnArgs& a, const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                     int64_t page_stride, int64_t num_pages, const int* block_table, int64_t bt_ld, int max_pages,
                     const int* seq_lens, const int* cu, int num_seqs, int64_t tokens, int H, int Hkv, int hd, int page,
                     int window, float scale, const void* k_sink, int sink_dtype, const void* gate, int64_t ldg,
                     void* o, float* lse, int dtype) {
  const int rc = pages_ok(k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens, num_seqs,
                          tokens, H, Hkv, hd, page, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(q && o, ZS_ERR_ARG);
  ZS_REQUIRE(window >= 0 && ldq >= (int64_t)H * hd && (gate == nullptr || ldg >= H), ZS_ERR_SHAPE);
  ZS_REQUIRE(ldq % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) == 0, ZS_ERR_ALIGN);
  ZS_REQUIRE(k_sink == nullptr || sink_dtype == ZS_F32 || sink_dtype == ZS_BF16 || sink_dtype == ZS_F16, ZS_ERR_DTYPE);
  a.q = q;
  a.ldq = ldq;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.page_stride = page_stride;
  a.num_pages = num_pages;
  a.block_table = block_table;
  a.bt_ld = bt_ld;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.cu = cu;
  a.num_seqs = num_seqs;
  a.tokens = tokens;
  a.H = H;
  a.Hkv = Hkv;
  a.page = page;
  a.window = window;
  a.scale = scale;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.k_sink = k_sink;
  a.sink_dtype = sink_dtype;
  a.gate = gate;
  a.ldg = ldg;
  a.o = o;
  a.lse = lse;
  return ZS_OK;
}

static int launch_plain(const paged::AttnArgs& a, int hd, int dtype, cudaStream_t stream) {
  const dim3 grid((unsigned)a.tokens, (unsigned)a.H);
  if (dtype == ZS_BF16) {
    if (hd == 128) paged::paged_attn_kernel<__nv_bfloat16, 128><<<grid, 128, 0, stream>>>(a);
    else paged::paged_attn_kernel<__nv_bfloat16, 64><<<grid, 128, 0, stream>>>(a);
  } else {
    if (hd == 128) paged::paged_attn_kernel<__half, 128><<<grid, 128, 0, stream>>>(a);
    else paged::paged_attn_kernel<__half, 64><<<grid, 128, 0, stream>>>(a);
  }
  ZS_CUDA_TRY(cudaGetLastError());
  return ZS_OK;
}

extern "C" size_t zs_paged_decode_workspace(int num_seqs, int H, int Hkv, int hd) {
  (void)num_seqs, (void)H, (void)Hkv, (void)hd;
  return 16;
}

extern "C" int zs_paged_decode_attention(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                         int64_t page_stride, int64_t num_pages, const int* block_table,
                                         int64_t bt_ld, int max_pages, const int* seq_lens, int num_seqs, int H,
                                         int Hkv, int hd, int page, int window, float scale, const void* k_sink,
                                         int sink_dtype, const void* gate, int64_t ldg, void* o, float* lse, int dtype,
                                         void* workspace, size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  paged::AttnArgs a;
  const int rc = attn_args(a, q, ldq, k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens,
                           nullptr, num_seqs, num_seqs, H, Hkv, hd, page, window, scale, k_sink, sink_dtype, gate, ldg,
                           o, lse, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(workspace && workspace_bytes >= zs_paged_decode_workspace(num_seqs, H, Hkv, hd), ZS_ERR_WORKSPACE);
  ZS_BIND(q);
  return launch_plain(a, hd, dtype, stream);
}

extern "C" int zs_paged_prompt_attention(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                         int64_t page_stride, int64_t num_pages, const int* block_table,
                                         int64_t bt_ld, int max_pages, const int* seq_lens, const int* cu_seqlens,
                                         int num_seqs, int64_t tokens, int H, int Hkv, int hd, int page, int window,
                                         float scale, const void* k_sink, int sink_dtype, const void* gate,
                                         int64_t ldg, void* o, float* lse, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  ZS_REQUIRE(cu_seqlens, ZS_ERR_ARG);
  paged::AttnArgs a;
  const int rc = attn_args(a, q, ldq, k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens,
                           cu_seqlens, num_seqs, tokens, H, Hkv, hd, page, window, scale, k_sink, sink_dtype, gate,
                           ldg, o, lse, dtype);
  if (rc != ZS_OK) return rc;
  ZS_BIND(q);
  return launch_plain(a, hd, dtype, stream);
}
