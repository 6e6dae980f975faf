// Paged key-value cache: storing new tokens in pages, and the page bookkeeping
// (extend, fork, free, compact, copy).
//
// Layout: k_pages / v_pages [num_pages, Hkv, page, hd], the last three
// dimensions packed, so one head's tokens of a page are one contiguous run
// (page * hd elements).  A sequence is a slot: a row of int32 page ids in the
// block table and its length; ref_count counts the rows that hold a page.
#include "zs_common.cuh"

namespace zs {
namespace paged {

// Tokens of a sequence: positions rounded up to a tile stay below 2^31.
constexpr int64_t MAX_TOKENS = ((int64_t)1 << 31) - 256;

// ------------------------------------------------------------------ element helpers

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_f(type v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ type from_f(float a, float b) { return __floats2bfloat162_rn(a, b); }
};
template <>
struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 to_f(type v) { return __half22float2(v); }
  static __device__ __forceinline__ type from_f(float a, float b) { return __floats2half2_rn(a, b); }
};

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const typename Pair<T>::type p = Pair<T>::from_f(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The sequence of packed token t: the last s with cu[s] <= t (empty sequences
// in between hold no token); -1 when t lies before cu[0] or from cu[n] on.  A
// whole warp asks together: each round of the search reads 32 entries at once.
__device__ __forceinline__ int sequence_of(const int* cu, int n, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, w = n + 1;                   // the last entry <= t is one of cu[lo .. lo + w)
  while (true) {
    const int step = (w + 31) / 32, i = lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, i < w && __ldg(cu + lo + i) <= t);
    if (below == 0) return -1;             // only when t < cu[0]
    const int j = (31 - __clz(below)) * step;
    lo += j;
    w = min(step, w - j);
    if (step == 1) break;
  }
  return lo < n ? lo : -1;
}

// ---------------------------------------------------------------------------- append

struct AppendArgs {
  const void* x;             // [tokens, >= (H + 2 Hkv) hd] rows of ldx elements: q heads, k heads, v heads
  int64_t ldx;
  const float* wq;           // nullable pair: norm gains (1 + w)
  const float* wk;
  float eps;
  const float* cos;          // [table_rows, rot] rows of table_ld floats
  const float* sin;
  int64_t table_ld;
  int64_t table_rows;
  int rot;
  const int* block_table;
  int64_t bt_ld;
  int max_pages;
  const int* seq_lens;
  const int* cu;             // nullable: token t is sequence t's one new token
  int num_seqs;
  int64_t tokens;
  int H, Hkv, page, page_shift;
  int64_t num_pages;
  void* k_pages;
  void* v_pages;
  int64_t page_stride;       // elements between pages
  void* q_out;               // [tokens, H, hd] packed
  int parts;                 // warps per token
};

// A warp holds 256 / hd head rows at a time; a lane has four columns of a row's
// first half and the same four of its second half (8-byte accesses, whole
// sectors), so it owns both members of the pairs that rotate.  A warp owns one
// of `parts` shares of a token's rows.  Each projected value is read once and
// written once, and what bounds that is loads in flight and issue slots: the first
// rows are asked for before the token's sequence and page are looked up, and cos and
// sin are read once per token.  21K prompt tokens of 16 + 2 * 4 heads of 128: 51 us,
// 4.9 TB/s in and out (75 % of a copy; DRAM itself is busy 46 % of that time, half of
// what is written being in L2 still at the end, and 65 % of the issue slots are used);
// blocks of four warps, because 28 warps fit an SM then (256 threads, 24 warps: 58 us).
template <typename T>
__device__ __forceinline__ void unpack4(const uint2& u, float* v) {
  const float2 a = Pair<T>::to_f(*reinterpret_cast<const typename Pair<T>::type*>(&u.x));
  const float2 b = Pair<T>::to_f(*reinterpret_cast<const typename Pair<T>::type*>(&u.y));
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
template <typename T>
__device__ __forceinline__ uint2 pack4(const float* v) {
  const typename Pair<T>::type a = Pair<T>::from_f(v[0], v[1]), b = Pair<T>::from_f(v[2], v[3]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <typename T, int HD>
__global__ void __launch_bounds__(128, 7) paged_append_kernel(const AppendArgs a) {
  constexpr int LPR = HD / 8;          // lanes per row
  constexpr int RPW = 32 / LPR;        // rows per warp pass
  constexpr int AHEAD = 4;             // passes loaded together
  const int lane = threadIdx.x & 31;
  const int rl = lane % LPR, rs = lane / LPR;
  const int64_t tok = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tok >= a.tokens) return;
  const int part = blockIdx.y;
  const int rows = a.H + 2 * a.Hkv, turned = a.H + a.Hkv;
  const int stride = a.parts * RPW;
  const T* x = reinterpret_cast<const T*>(a.x) + tok * a.ldx + rl * 4;
  uint2 lo[AHEAD], hi[AHEAD];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int r = r0 + u * stride + rs;
      lo[u] = hi[u] = make_uint2(0, 0);
      if (r < rows) {
        lo[u] = __ldcs(reinterpret_cast<const uint2*>(x + r * HD));
        hi[u] = __ldcs(reinterpret_cast<const uint2*>(x + r * HD + HD / 2));
      }
    }
  };
  load(part * RPW);

  int seq = (int)tok;
  int64_t pos = -1;
  if (a.cu != nullptr) {
    seq = sequence_of(a.cu, a.num_seqs, (int)tok);
    if (seq >= 0) pos = (int64_t)__ldg(a.seq_lens + seq) - __ldg(a.cu + seq + 1) + tok;
  } else {
    pos = (int64_t)__ldg(a.seq_lens + seq) - 1;
  }
  int page = -1;
  bool live = pos >= 0;                // no sequence or a negative position: zero q, nothing stored
  if (live) {
    if (pos < (int64_t)a.max_pages * a.page && (a.rot == 0 || pos < a.table_rows))   // below 2^31
      page = __ldg(a.block_table + seq * a.bt_ld + ((int)pos >> a.page_shift));
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0 && part == 0) record_error(ZS_DEVERR_INDEX);
      live = false;
    }
  }
  const int pairs = live ? min(a.rot - rl * 4, 4) : 0;   // pairs of this lane that rotate
  float cs[4], sn[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cs[e] = e < pairs ? __ldg(a.cos + pos * a.table_ld + rl * 4 + e) : 1.f;
    sn[e] = e < pairs ? __ldg(a.sin + pos * a.table_ld + rl * 4 + e) : 0.f;
  }
  T* q = reinterpret_cast<T*>(a.q_out) + tok * (int64_t)a.H * HD + rl * 4;
  const int64_t at = live ? page * a.page_stride + ((int)pos & (a.page - 1)) * HD + rl * 4 : 0;
  T* kp = reinterpret_cast<T*>(a.k_pages) + at;
  T* vp = reinterpret_cast<T*>(a.v_pages) + at;
  for (int r0 = part * RPW; r0 < rows; r0 += AHEAD * stride) {
    if (r0 != part * RPW) load(r0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int rb = r0 + u * stride;
      if (rb >= rows) break;
      const int r = rb + rs;
      if (rb < turned) {                         // the warp has a query or key row
        float v[8];
        unpack4<T>(lo[u], v);
        unpack4<T>(hi[u], v + 4);
        if (a.wq != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
#pragma unroll
          for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
          const float rstd = rsqrtf(ss / (float)HD + a.eps);
          const float* w = (r < a.H ? a.wq : a.wk) + rl * 4;
          const float4 w0 = __ldg(reinterpret_cast<const float4*>(w));
          const float4 w1 = __ldg(reinterpret_cast<const float4*>(w + HD / 2));
          const float g[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (v[e] * rstd) * (1.0f + g[e]);
        }
        if (pairs > 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e < pairs) {
              const float x1 = v[e], x2 = v[4 + e];
              v[e] = x1 * cs[e] - x2 * sn[e];
              v[4 + e] = x2 * cs[e] + x1 * sn[e];
            }
          }
        }
        if (r < turned) {                        // values keep their bits
          lo[u] = pack4<T>(v);
          hi[u] = pack4<T>(v + 4);
        }
      }
      if (r >= rows) continue;
      T* dst;
      if (r < a.H) {
        dst = q + r * HD;
        if (!live) lo[u] = hi[u] = make_uint2(0, 0);
      } else {
        if (!live) continue;
        dst = r < turned ? kp + (int64_t)(r - a.H) * a.page * HD : vp + (int64_t)(r - turned) * a.page * HD;
      }
      *reinterpret_cast<uint2*>(dst) = lo[u];
      *reinterpret_cast<uint2*>(dst + HD / 2) = hi[u];
    }
  }
}

// ------------------------------------------------------------------- page bookkeeping
//
// The plan kernels run in one block: requests are served in order and take the
// lowest-numbered free pages, so every result is a function of the tables
// alone.  Page data moves in kv_apply_kernel, which reads the plan's list of
// (from, to, rows); the lists name free pages as targets only, so no copy
// reads what another writes.

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_SLOTS = 8192;           // slots whose marks fit the plan's shared memory
constexpr int PLAN_CELLS = 8192;           // table cells that one block rewrites as fast as a grid launched for them

struct Plan {              // device workspace of a call, all int32
  int* count;              // number of moves
  int* from;               // [moves]
  int* to;
  int* rows;
  int* off;                // [n] first free page of request i in free_pages, -1: request refused
  int* len;                // [n] length of the source before the call
  int* first;              // [max_seqs] lowest request that names the slot
  int* free_pages;         // [num_pages] free pages in ascending order (as many as needed)
  int* map;                // [num_pages] new number of a moved page
  int* snap;               // [n, max_pages] source rows before the call
};

// Exclusive scan of one int per thread over the block; total in *sum.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += o;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const int before = warp ? s_warp[warp - 1] : 0;
  *sum = s_warp[31];
  __syncthreads();
  return before + inc - v;
}

// The lowest `want` free pages into list; returns how many there are (<= want).
__device__ __forceinline__ int find_free(const int* ref, int64_t P, int want, int* list, int* s_warp) {
  constexpr int PER = 8;
  int have = 0;
  for (int64_t base = 0; base < P && have < want; base += (int64_t)PLAN_THREADS * PER) {
    const int64_t p0 = base + (int64_t)threadIdx.x * PER;
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (p0 + e < P && ref[p0 + e] == 0) mask |= 1u << e;
    int sum;
    int at = have + block_scan(__popc(mask), s_warp, &sum);
    for (; mask; mask &= mask - 1, ++at)
      if (at < want) list[at] = (int)(p0 + __ffs(mask) - 1);
    have += sum;
  }
  __syncthreads();
  return have < want ? have : want;
}

// first[slot] = the lowest request that names the slot (requests out of range name none)
__device__ __forceinline__ void mark_first(const int* slots, int n, int max_seqs, int* first) {
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
    if ((unsigned)slots[i] < (unsigned)max_seqs) first[slots[i]] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
    if ((unsigned)slots[i] < (unsigned)max_seqs) atomicMin(first + slots[i], i);
  __syncthreads();
}

// One more or one less holder of a page; a page id out of range is recorded and left alone.
__device__ __forceinline__ void hold(const zs_kv_cache& c, int page, int by) {
  if ((unsigned)page < (unsigned)c.num_pages)
    atomicAdd(c.ref_count + page, by);
  else
    record_error(ZS_DEVERR_INDEX);
}

// Each request's number of new pages (need_of(i), -1: refused) scanned in
// order into plan.off; the pages found; requests past them refused.
template <typename F>
__device__ __forceinline__ void allot(const zs_kv_cache& c, const Plan& p, int n, F need_of, int* s_warp) {
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    const int need = i < n ? min(need_of(i), (int)c.num_pages + 1) : 0;
    int sum;
    // 32 bits hold the sums: a request counts at most num_pages + 1 <= 2000001 pages, a
    // block of requests 1024 times that, and the running total stops past the pool
    const int at = total + block_scan(need > 0 ? need : 0, s_warp, &sum);
    if (i < n) p.off[i] = need < 0 ? -1 : at;
    total = total > (int)c.num_pages - sum ? (int)c.num_pages + 1 : total + sum;
  }
  __syncthreads();
  const int want = total > (int)c.num_pages ? (int)c.num_pages : total;
  const int have = find_free(c.ref_count, c.num_pages, want, p.free_pages, s_warp);
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int need = need_of(i);
    if (need > 0 && (p.off[i] > have || need > have - p.off[i])) {
      p.off[i] = -1;
      record_error(ZS_DEVERR_CACHE_FULL);
    }
  }
  __syncthreads();
}

__global__ void __launch_bounds__(PLAN_THREADS) kv_extend_kernel(const zs_kv_cache c, Plan p,
                                                                 const int* slots, const int* tokens, int n) {
  __shared__ int s_warp[32], s_first[PLAN_SLOTS];
  if (c.max_seqs <= PLAN_SLOTS) p.first = s_first;
  mark_first(slots, n, c.max_seqs, p.first);
  auto need_of = [&](int i) -> int {
    const int s = slots[i], t = tokens[i];
    if ((unsigned)s >= (unsigned)c.max_seqs || t < 0 || p.first[s] != i) return -1;
    const int len = c.seq_lens[s];
    const int64_t end = (int64_t)len + t;
    if (len < 0 || end > (int64_t)c.max_pages * c.page_size) return -1;
    return (int)((end + c.page_size - 1) / c.page_size) - (len + c.page_size - 1) / c.page_size;
  };
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int s = slots[i], t = tokens[i];
    if ((unsigned)s >= (unsigned)c.max_seqs || t < 0 || p.first[s] != i || c.seq_lens[s] < 0)
      record_error(ZS_DEVERR_INDEX);
    else if ((int64_t)c.seq_lens[s] + t > (int64_t)c.max_pages * c.page_size)
      record_error(ZS_DEVERR_CACHE_FULL);
  }
  allot(c, p, n, need_of, s_warp);
  // A thread writes a request's first pages, a warp the many of a prompt (a warp for every request: 64 slots
  // by a token 6.4 us instead of 4.4, 1000 slots 33 instead of 10).
  constexpr int FEW = 2;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int off = p.off[i];
    if (off < 0) continue;
    const int s = slots[i], len = c.seq_lens[s], need = need_of(i);
    const int old = (len + c.page_size - 1) / c.page_size;
    for (int j = 0; j < min(need, FEW); ++j) {
      const int pg = p.free_pages[off + j];
      c.block_table[(int64_t)s * c.max_pages + old + j] = pg;
      c.ref_count[pg] = 1;
    }
    p.len[i] = need;
    p.rows[i] = old;
    c.seq_lens[s] = len + tokens[i];
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += PLAN_THREADS / 32) {
    const int off = p.off[i];
    if (off < 0 || p.len[i] <= FEW) continue;
    int* row = c.block_table + (int64_t)slots[i] * c.max_pages + p.rows[i];
    for (int j = FEW + lane; j < p.len[i]; j += 32) {
      const int pg = p.free_pages[off + j];
      row[j] = pg;
      c.ref_count[pg] = 1;
    }
  }
}

// Request i's cell j: the new row's page (the source's whole pages, then a page of its own
// for the partial one), kept until every source row is read; the counts of what the
// request holds and lets go.
__device__ __forceinline__ void fork_cell(const zs_kv_cache& c, const Plan& p, const int* src, const int* dst, int i,
                                          int j) {
  const int full = p.len[i] / c.page_size;
  const int old = c.block_table[(int64_t)dst[i] * c.max_pages + j];
  int pg = -1;
  if (j < full)
    pg = c.block_table[(int64_t)src[i] * c.max_pages + j];
  else if (j == full && p.len[i] % c.page_size)
    pg = p.free_pages[p.off[i]];
  if (j <= full && (pg >= 0 || j < full)) hold(c, pg, 1);
  p.snap[(int64_t)i * c.max_pages + j] = pg;
  if (old != -1) hold(c, old, -1);
}

__global__ void __launch_bounds__(PLAN_THREADS) kv_fork_plan_kernel(const zs_kv_cache c, Plan p,
                                                                    const int* src, const int* dst, int n,
                                                                    int rows_here) {
  __shared__ int s_warp[32], s_first[PLAN_SLOTS];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (c.max_seqs <= PLAN_SLOTS) p.first = s_first;
  mark_first(dst, n, c.max_seqs, p.first);
  auto need_of = [&](int i) -> int {
    const int s = src[i], d = dst[i];
    if ((unsigned)s >= (unsigned)c.max_seqs || (unsigned)d >= (unsigned)c.max_seqs || p.first[d] != i) return -1;
    if (s == d) return -1;                                  // stays as it is
    const int len = c.seq_lens[s];
    if (len < 0 || len > c.max_pages * c.page_size) return -1;
    return len % c.page_size ? 1 : 0;
  };
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int s = src[i], d = dst[i];
    const bool ok = (unsigned)s < (unsigned)c.max_seqs && (unsigned)d < (unsigned)c.max_seqs;
    if (!ok || p.first[d] != i) record_error(ZS_DEVERR_INDEX);
    p.len[i] = ok ? c.seq_lens[s] : 0;
    if (p.len[i] < 0 || p.len[i] > c.max_pages * c.page_size) record_error(ZS_DEVERR_INDEX);
  }
  allot(c, p, n, need_of, s_warp);
  int moves = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    bool mv = i < n && p.off[i] >= 0 && p.len[i] % c.page_size;
    const int last = mv ? c.block_table[(int64_t)src[i] * c.max_pages + p.len[i] / c.page_size] : 0;
    if ((unsigned)last >= (unsigned)c.num_pages) {          // a table that is not the cache's own
      record_error(ZS_DEVERR_INDEX);
      mv = false;
    }
    int sum;
    const int at = moves + block_scan(mv ? 1 : 0, s_warp, &sum);
    if (mv) {
      p.from[at] = last;
      p.to[at] = p.free_pages[p.off[i]];
      p.rows[at] = p.len[i] % c.page_size;
    }
    moves += sum;
  }
  if (threadIdx.x == 0) *p.count = moves;
  if (!rows_here) return;
  for (int e = threadIdx.x; e < n * c.max_pages; e += PLAN_THREADS) {
    const int i = e / c.max_pages;
    if (p.off[i] >= 0) fork_cell(c, p, src, dst, i, e - i * c.max_pages);
  }
}

// The same cells from a grid, block i request i.
__global__ void __launch_bounds__(256) kv_fork_rows_kernel(const zs_kv_cache c, const Plan p, const int* src,
                                                           const int* dst) {
  const int i = blockIdx.x;
  if (p.off[i] < 0) return;
  for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) fork_cell(c, p, src, dst, i, j);
}

__global__ void __launch_bounds__(128) kv_free_kernel(const zs_kv_cache c, const int* slots) {
  __shared__ int s_len;
  const int s = slots[blockIdx.x];
  if ((unsigned)s >= (unsigned)c.max_seqs) {
    if (threadIdx.x == 0) record_error(ZS_DEVERR_INDEX);
    return;
  }
  // a slot named twice is freed by whichever block takes its length
  if (threadIdx.x == 0) s_len = atomicExch(c.seq_lens + s, 0);
  __syncthreads();
  if (s_len == 0) return;
  for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) {
    int* e = c.block_table + (int64_t)s * c.max_pages + j;
    if (*e != -1) {
      hold(c, *e, -1);
      *e = -1;
    }
  }
}

__global__ void __launch_bounds__(PLAN_THREADS) kv_compact_plan_kernel(const zs_kv_cache c, const Plan p) {
  __shared__ int s_warp[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int PER = 8;
  const int64_t P = c.num_pages;
  auto used_mask = [&](int64_t p0) -> uint32_t {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (p0 + e < P && c.ref_count[p0 + e] != 0) m |= 1u << e;
    return m;
  };
  int mine = 0, U;
  for (int64_t base = 0; base < P; base += (int64_t)PLAN_THREADS * PER)
    mine += __popc(used_mask(base + (int64_t)threadIdx.x * PER));
  block_scan(mine, s_warp, &U);
  // holes below U in ascending order are the targets, used pages from U on the sources
  int holes = 0, movers = 0;
  for (int64_t base = 0; base < P; base += (int64_t)PLAN_THREADS * PER) {
    const int64_t p0 = base + (int64_t)threadIdx.x * PER;
    const uint32_t used = used_mask(p0);
    uint32_t hole = 0, mover = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int64_t pg = p0 + e;
      if (pg >= P) break;
      const bool u = used >> e & 1;
      if (pg < U && !u) hole |= 1u << e;
      if (pg >= U && u) mover |= 1u << e;
      p.map[pg] = (int)pg;
    }
    int sh, sm;
    int ah = holes + block_scan(__popc(hole), s_warp, &sh);
    int am = movers + block_scan(__popc(mover), s_warp, &sm);
    for (; hole; hole &= hole - 1, ++ah) p.to[ah] = (int)(p0 + __ffs(hole) - 1);
    for (; mover; mover &= mover - 1, ++am) p.from[am] = (int)(p0 + __ffs(mover) - 1);
    holes += sh;
    movers += sm;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += PLAN_THREADS) {
    p.rows[i] = c.page_size;
    p.map[p.from[i]] = p.to[i];
    c.ref_count[p.to[i]] = c.ref_count[p.from[i]];
    c.ref_count[p.from[i]] = 0;
  }
  if (threadIdx.x == 0) {
    *p.count = movers;
    p.off[0] = U;
  }
}

// Moves given by the caller: pages out of range, a target named twice (the
// first stands) and a target that is also a source are refused.
__global__ void __launch_bounds__(PLAN_THREADS) kv_copy_plan_kernel(const zs_kv_cache c, const Plan p, const int* src,
                                                                    const int* dst, int n) {
  __shared__ int s_warp[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const unsigned P = (unsigned)c.num_pages;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    if ((unsigned)src[i] < P) p.map[src[i]] = 0;
    if ((unsigned)dst[i] < P) {
      p.map[dst[i]] = 0;
      p.free_pages[dst[i]] = 0x7fffffff;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    if ((unsigned)src[i] < P) p.map[src[i]] = 1;              // a source
    if ((unsigned)dst[i] < P) atomicMin(p.free_pages + dst[i], i);
  }
  __syncthreads();
  int moves = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    bool mv = false;
    if (i < n) {
      const bool ok = (unsigned)src[i] < P && (unsigned)dst[i] < P && p.free_pages[dst[i]] == i && p.map[dst[i]] == 0;
      const bool same = (unsigned)src[i] < P && src[i] == dst[i];
      mv = ok && !same;
      if (!ok && !same) record_error(ZS_DEVERR_INDEX);
    }
    int sum;
    const int at = moves + block_scan(mv ? 1 : 0, s_warp, &sum);
    if (mv) {
      p.from[at] = src[i];
      p.to[at] = dst[i];
      p.rows[at] = c.page_size;
    }
    moves += sum;
  }
  if (threadIdx.x == 0) *p.count = moves;
}

// What follows a plan: the tables rewritten (FORK: the new rows; COMPACT: moved pages
// renamed), then the page data.  One work item: one head's filled rows of one page of one
// layer's keys or values, a contiguous run of rows * hd elements.  HBM-bound: read once,
// written once.  Launched while the plan still runs; waits for its end.  Eight blocks of 32
// registers an SM, all resident, no division per item (five of 48 registers with 64-bit divisions: fork of 32 beams
// over 16 layers 21.6 us instead of 20.9; about 10 of them do not grow with the bytes, the rest
// moves at 6.5 TB/s).  Compaction of 48 sequences in 8 layers: 136 us, 5.5 TB/s.
enum { AFTER_COPY, AFTER_FORK, AFTER_COMPACT };

template <int AFTER>
__global__ void __launch_bounds__(256, 8) kv_apply_kernel(const zs_kv_cache c, const Plan p, const int* dst, int n) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, all = (int64_t)gridDim.x * blockDim.x;
  if (AFTER == AFTER_FORK) {
    for (int64_t e = me; e < (int64_t)n * c.max_pages; e += all) {
      const int i = (int)(e / c.max_pages);
      if (p.off[i] < 0) continue;
      const int j = (int)(e - (int64_t)i * c.max_pages);
      c.block_table[(int64_t)dst[i] * c.max_pages + j] = p.snap[e];
      if (j == 0) c.seq_lens[dst[i]] = p.len[i];
    }
  }
  if (AFTER == AFTER_COMPACT) {
    const int U = p.off[0];
    for (int64_t e = me; e < (int64_t)c.max_seqs * c.max_pages; e += all) {
      const int pg = c.block_table[e];
      if (pg >= U && pg < c.num_pages) c.block_table[e] = p.map[pg];
    }
  }
  const int64_t run = (int64_t)c.page_size * c.head_dim / 8;        // 16-byte words of a whole run
  const int64_t page = run * c.n_kv_heads;
  const int per = 2 * c.n_layers * c.n_kv_heads, count = *p.count;   // items of a move
  uint4* kv = reinterpret_cast<uint4*>(c.kv);
  int m = blockIdx.x / per, rest = blockIdx.x % per;
  const int dm = gridDim.x / per, dr = gridDim.x % per;
  while (m < count) {
    const int slab = rest / c.n_kv_heads, h = rest - slab * c.n_kv_heads;
    const uint4* from = kv + (slab * (int64_t)c.num_pages + p.from[m]) * page + h * run;
    uint4* to = kv + (slab * (int64_t)c.num_pages + p.to[m]) * page + h * run;
    const int words = p.rows[m] * (c.head_dim / 8);
    for (int w = threadIdx.x; w < words; w += 4 * 256) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w + e * 256 < words) v[e] = from[w + e * 256];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w + e * 256 < words) to[w + e * 256] = v[e];
    }
    m += dm;
    rest += dr;
    if (rest >= per) rest -= per, ++m;
  }
}

static int cache_ok(const zs_kv_cache* c) {
  ZS_REQUIRE(c && c->kv && c->block_table && c->seq_lens && c->ref_count, ZS_ERR_ARG);
  ZS_REQUIRE(c->num_pages >= 1 && c->num_pages <= 2000000 && c->n_layers >= 1 && c->n_kv_heads >= 1 &&
                 c->max_seqs >= 1 && c->max_pages >= 1,
             ZS_ERR_SHAPE);
  ZS_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128, ZS_ERR_SHAPE);
  ZS_REQUIRE((int64_t)c->max_pages * c->page_size <= MAX_TOKENS, ZS_ERR_SHAPE);
  ZS_REQUIRE(c->head_dim == 64 || c->head_dim == 128, ZS_ERR_SHAPE);
  ZS_REQUIRE((reinterpret_cast<uintptr_t>(c->kv) & 15) == 0, ZS_ERR_ALIGN);
  return ZS_OK;
}

static Plan carve(const zs_kv_cache& c, int64_t n, void* ws) {
  Plan p;
  int* at = reinterpret_cast<int*>((reinterpret_cast<uintptr_t>(ws) + 15) & ~uintptr_t(15));
  auto take = [&](int64_t k) {
    int* r = at;
    at += (k + 3) & ~int64_t(3);
    return r;
  };
  const int64_t moves = n > c.num_pages ? n : c.num_pages;
  p.count = take(1);
  p.from = take(moves);
  p.to = take(moves);
  p.rows = take(moves);
  p.off = take(n + 1);
  p.len = take(n);
  p.first = take(c.max_seqs);
  p.free_pages = take(c.num_pages);
  p.map = take(c.num_pages);
  p.snap = take(n * c.max_pages);
  return p;
}

}  // namespace paged
}  // namespace zs

using namespace zs;

extern "C" size_t zs_kv_workspace(const zs_kv_cache* c, int64_t n) {
  if (c == nullptr || n < 0) return 0;
  const int64_t moves = n > c->num_pages ? n : c->num_pages;
  return (size_t)(3 * moves + 2 * n + c->max_seqs + 2 * c->num_pages + n * c->max_pages + 64) * sizeof(int) + 64;
}

#define ZS_KV_ENTER(n)                                                        \
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);                   \
  {                                                                           \
    const int rc_ = paged::cache_ok(c);                                       \
    if (rc_ != ZS_OK) return rc_;                                             \
  }                                                                           \
  ZS_REQUIRE((n) >= 0 && (n) < (1 << 24), ZS_ERR_SHAPE);                      \
  ZS_REQUIRE(workspace && workspace_bytes >= zs_kv_workspace(c, n), ZS_ERR_WORKSPACE); \
  ZS_BIND(c->kv);                                                             \
  const paged::Plan p = paged::carve(*c, n, workspace)

// A kernel that may be scheduled while the one before it in the stream still runs (it waits for
// that one's end itself).
template <typename... P, typename... A>
static int launch_after(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  ZS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
  return ZS_OK;
}

template <int AFTER>
static int launch_apply(const zs_kv_cache& c, const paged::Plan& p, const int* dst, int64_t n, cudaStream_t stream) {
  return launch_after(paged::kv_apply_kernel<AFTER>, dim3(num_sms() * 8), dim3(256), stream, c, p, dst, (int)n);
}

extern "C" int zs_kv_extend(const zs_kv_cache* c, const int* slots, const int* tokens, int64_t n, void* workspace,
                            size_t workspace_bytes, void* stream_) {
  ZS_KV_ENTER(n);
  if (n == 0) return ZS_OK;
  ZS_REQUIRE(slots && tokens, ZS_ERR_ARG);
  paged::kv_extend_kernel<<<1, paged::PLAN_THREADS, 0, stream>>>(*c, p, slots, tokens, (int)n);
  ZS_CUDA_TRY(cudaGetLastError());
  return ZS_OK;
}

extern "C" int zs_kv_fork(const zs_kv_cache* c, const int* src, const int* dst, int64_t n, void* workspace,
                          size_t workspace_bytes, void* stream_) {
  ZS_KV_ENTER(n);
  if (n == 0) return ZS_OK;
  ZS_REQUIRE(src && dst, ZS_ERR_ARG);
  const bool rows_here = n * c->max_pages <= paged::PLAN_CELLS;
  paged::kv_fork_plan_kernel<<<1, paged::PLAN_THREADS, 0, stream>>>(*c, p, src, dst, (int)n, rows_here ? 1 : 0);
  ZS_CUDA_TRY(cudaGetLastError());
  if (!rows_here) {
    paged::kv_fork_rows_kernel<<<(unsigned)n, 256, 0, stream>>>(*c, p, src, dst);
    ZS_CUDA_TRY(cudaGetLastError());
  }
  return launch_apply<paged::AFTER_FORK>(*c, p, dst, n, stream);
}

extern "C" int zs_kv_free(const zs_kv_cache* c, const int* slots, int64_t n, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = paged::cache_ok(c);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(n >= 0 && n < (1 << 24), ZS_ERR_SHAPE);
  if (n == 0) return ZS_OK;
  ZS_REQUIRE(slots, ZS_ERR_ARG);
  ZS_BIND(c->kv);
  paged::kv_free_kernel<<<(unsigned)n, 128, 0, stream>>>(*c, slots);
  ZS_CUDA_TRY(cudaGetLastError());
  return ZS_OK;
}

extern "C" int zs_kv_compact(const zs_kv_cache* c, void* workspace, size_t workspace_bytes, void* stream_) {
  ZS_KV_ENTER(0);
  paged::kv_compact_plan_kernel<<<1, paged::PLAN_THREADS, 0, stream>>>(*c, p);
  ZS_CUDA_TRY(cudaGetLastError());
  return launch_apply<paged::AFTER_COMPACT>(*c, p, nullptr, 0, stream);
}

extern "C" int zs_kv_copy_pages(const zs_kv_cache* c, const int* src, const int* dst, int64_t n, void* workspace,
                                size_t workspace_bytes, void* stream_) {
  ZS_KV_ENTER(n);
  if (n == 0) return ZS_OK;
  ZS_REQUIRE(src && dst, ZS_ERR_ARG);
  paged::kv_copy_plan_kernel<<<1, paged::PLAN_THREADS, 0, stream>>>(*c, p, src, dst, (int)n);
  ZS_CUDA_TRY(cudaGetLastError());
  return launch_apply<paged::AFTER_COPY>(*c, p, nullptr, 0, stream);
}

// Checks shared by the operators that read or write one layer's pages.
static int pages_ok(const void* k_pages, const void* v_pages, int64_t page_stride, int64_t num_pages,
                    const int* block_table, int64_t bt_ld, int max_pages, const int* seq_lens, int num_seqs,
                    int64_t tokens, int H, int Hkv, int hd, int page, int dtype) {
  ZS_REQUIRE(k_pages && v_pages && block_table && seq_lens, ZS_ERR_ARG);
  ZS_REQUIRE(dtype == ZS_BF16 || dtype == ZS_F16, ZS_ERR_DTYPE);
  ZS_REQUIRE(hd == 64 || hd == 128, ZS_ERR_SHAPE);
  ZS_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, ZS_ERR_SHAPE);
  ZS_REQUIRE(H >= 1 && Hkv >= 1 && H % Hkv == 0 && H <= 65535, ZS_ERR_SHAPE);
  ZS_REQUIRE(num_seqs >= 1 && tokens >= 1 && tokens < (int64_t)1 << 31 && num_pages >= 1 &&
                 num_pages < (int64_t)1 << 30 && max_pages >= 1 && (int64_t)max_pages * page <= paged::MAX_TOKENS,
             ZS_ERR_SHAPE);
  ZS_REQUIRE(bt_ld >= max_pages, ZS_ERR_SHAPE);
  ZS_REQUIRE(page_stride >= (int64_t)Hkv * page * hd && page_stride % 8 == 0, ZS_ERR_LAYOUT);
  ZS_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, ZS_ERR_ALIGN);
  return ZS_OK;
}

extern "C" int zs_paged_append(const void* qkv, int64_t ld, const float* q_weight, const float* k_weight, float eps,
                               const float* cos, const float* sin, int64_t table_ld, int64_t table_rows, int rot,
                               void* k_pages, void* v_pages, int64_t page_stride, int64_t num_pages,
                               const int* block_table, int64_t bt_ld, int max_pages, const int* seq_lens,
                               const int* cu_seqlens, int num_seqs, int64_t tokens, int H, int Hkv, int hd, int page,
                               void* q_out, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = pages_ok(k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens, num_seqs,
                    tokens, H, Hkv, hd, page, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(qkv && q_out && (q_weight == nullptr) == (k_weight == nullptr), ZS_ERR_ARG);
  ZS_REQUIRE(rot >= 0 && rot <= hd / 2, ZS_ERR_SHAPE);
  ZS_REQUIRE(rot == 0 || (cos && sin), ZS_ERR_ARG);
  ZS_REQUIRE(rot == 0 || (table_ld >= rot && table_rows >= 1), ZS_ERR_SHAPE);
  ZS_REQUIRE(ld >= (int64_t)(H + 2 * Hkv) * hd, ZS_ERR_SHAPE);
  ZS_REQUIRE(cu_seqlens != nullptr || tokens == num_seqs, ZS_ERR_SHAPE);
  ZS_REQUIRE(ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
                              reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight)) & 15) == 0,
             ZS_ERR_ALIGN);
  ZS_BIND(qkv);
  paged::AppendArgs a;
  a.x = qkv;
  a.ldx = ld;
  a.wq = q_weight;
  a.wk = k_weight;
  a.eps = eps;
  a.cos = cos;
  a.sin = sin;
  a.table_ld = table_ld;
  a.table_rows = table_rows;
  a.rot = rot;
  a.block_table = block_table;
  a.bt_ld = bt_ld;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.cu = cu_seqlens;
  a.num_seqs = num_seqs;
  a.tokens = tokens;
  a.H = H;
  a.Hkv = Hkv;
  a.page = page;
  a.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  a.num_pages = num_pages;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.page_stride = page_stride;
  a.q_out = q_out;
  const int rpw = 256 / hd, passes = (H + 2 * Hkv + rpw - 1) / rpw;
  // A share of a token's rows repeats the lookups, so a token is shared out only while there are fewer
  // than 32 warps an SM: 21K prompt tokens of 24 rows take 58 us with one warp a token, 63 to 69 us with three.
  a.parts = 1;
  while (a.parts < passes && tokens * a.parts * 2 <= (int64_t)num_sms() * 32) a.parts *= 2;
  if (a.parts > passes) a.parts = passes;
  const dim3 blocks((unsigned)((tokens + 3) / 4), (unsigned)a.parts);
  if (dtype == ZS_BF16) {
    if (hd == 128)
      paged::paged_append_kernel<__nv_bfloat16, 128><<<blocks, 128, 0, stream>>>(a);
    else
      paged::paged_append_kernel<__nv_bfloat16, 64><<<blocks, 128, 0, stream>>>(a);
  } else {
    if (hd == 128)
      paged::paged_append_kernel<__half, 128><<<blocks, 128, 0, stream>>>(a);
    else
      paged::paged_append_kernel<__half, 64><<<blocks, 128, 0, stream>>>(a);
  }
  ZS_CUDA_TRY(cudaGetLastError());
  return ZS_OK;
}
