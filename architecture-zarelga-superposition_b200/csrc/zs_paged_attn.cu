// Attention over a paged key-value cache: one new token per sequence
// (zs_paged_decode_attention) and packed new tokens (zs_paged_prompt_attention).
//
// o = sum_k softmax_k(q . K_k * scale) V_k over the keys k <= p of the query's
// sequence (p its position, p - k < window where a window is given), with an
// optional sink logit q . k_sink * scale whose value is zero and an optional
// sigmoid gate on o.  A row that sees no key is zero, its log-sum-exp the sink
// logit or -inf.
#include "zs_common.cuh"
#include "zs_paged_plan.cuh"

#include <atomic>
#include <type_traits>

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
  float scale_log2;            // softmax scale * log2(e)
  const float* k_sink;         // nullable [H, hd]
  const void* gate;            // nullable [tokens, H] rows of ldg elements
  int64_t ldg;
  void* o;                     // [tokens, H, hd] packed
  float* lse;                  // nullable [tokens, H]
};

// A sequence's length, no longer than its row of the block table.
__device__ __forceinline__ int cut_length(const AttnArgs& a, int seq) {
  const int len = __ldg(a.seq_lens + seq), cap = a.max_pages * a.page;
  if (len > cap) record_error(ZS_DEVERR_INDEX);
  return length_within(len, cap);
}

// ------------------------------------------------------------------------ decode
//
// One token per sequence: the cache is read once and hardly anything is computed, so the
// kernel is bound by HBM.  The work is the list of 16 KiB key tiles of every unit (sequence,
// key head, block of 16 query heads), in that order, cut into equal runs, one per block: a
// batch of sequences of any lengths loads every SM alike.  A unit counts OVER steps more than
// it has tiles, because its start and end (queries in, rows out) cost as much as that many.
// A block walks its run, and whatever part of a unit ends in it is finished there; parts of
// one that several blocks share go to the workspace (at most two per block, the run's first
// and last) and paged_join_kernel adds them in the order of the blocks.
//
// Warp 4 loads the pages of a tile with TMA (128-byte swizzle) into a ring of stages; warps
// 0-3 each take a quarter of its keys: S = Q K^T and O += P V by mma.sync with the group's query heads
// as the 16 rows, P straight from the accumulators of S, and a running (max, sum, O) of their
// own, joined through shared memory when a part ends.  mma.sync, not tcgen05: a 128-row tile
// would hold 1 to 16 rows of work, and the products are a tenth of the time of the loads.
//
// 64 sequences of 30K to 32K tokens, 16/4 heads of 128: 610 us, 6.7 TB/s (a copy reaches 6.56); 32 of 1 to
// 4096 tokens, 12/4 heads: 30 us, of which 20 are the bytes, 3.4 the start to the first load.

constexpr int DEC_MAX_BLOCKS = 320;       // two per SM
constexpr int DEC_ROWS = 16;              // query heads per block of rows
constexpr int DEC_LDO = 40;               // floats per row of the join buffer (32 + padding against bank conflicts)

// A row's weights are P = 2^(S - m) of a reference m (log2 units) that every earlier sum of the row is kept
// relative to, in f32.  P goes to the second product in the cache's type, since V is held in it and both operands
// have one type; that is half a step of each weight.  In bf16, which has f32's range, m follows the running maximum:
// raised when a tile's largest S passes it by more than 8, so that O is rescaled rarely.  f16 has bits for
// weights from 2^-14 to 2^15 only, so there m follows the tile: the largest P of a tile is kept between 2^7 and 2^15,
// up and down (one key may take nearly all the weight with a value of nothing, and the many others still add up).
// What f16 rounds away of a tile of n keys is then at most n 2^-25 / 2^7 of its largest weight.  Not below 2^-40
// of the row's largest weight: the sums relative to m stay far from f32's end.  Against a running maximum in f16 too:
// 129 decode windows of 512 23.8 us instead of 23.5, six prompt chunks after prefixes 47.5 instead of 47.1.
template <typename T>
struct RowRef {
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static constexpr float AT = F16 ? 11.f : 0.f;          // log2 of the largest P where m is set
  static constexpr float UP = F16 ? 15.f : 8.f, DOWN = 7.f, DEEP = 40.f;
  float m = -INFINITY, top = -INFINITY;                  // top: the largest S so far (f16)
  // A tile whose largest S is mx: whether m moves, and then what the sums so far are multiplied by.
  __device__ __forceinline__ bool move(float mx, float* f) {
    float to = mx;
    bool go = mx > m + UP;
    if (F16) {
      top = fmaxf(top, mx);
      to = fmaxf(mx, top - DEEP);
      go = go || (mx != -INFINITY && to < m + DOWN);
    }
    *f = 1.f;
    if (!go) return false;
    to -= AT;
    *f = m == -INFINITY ? 0.f : attn::fast_exp2(m - to);
    m = to;
    return true;
  }
};

template <int HD>
struct DecSmem {
  static constexpr int TILE = HD == 128 ? 64 : 128;             // keys per tile
  // Steps of a unit's start and end, measured over 0 to 6: 32 sequences of 1 to 4096 tokens of 12/4
  // heads of 128 take 42.5 us without, 33.1, 32.0, 31.7 and 32.3 us with 1 to 4; 129 windows of
  // 512 of 16/4 heads of 64 take 23.4 us with 1 and 23.9 to 24.4 us with 2 to 6.
  static constexpr int OVER = HD == 128 ? 3 : 1;
  static constexpr int STAGES = 3;
  static constexpr int MAT = TILE * HD * 2;                     // K or V of one tile
  static constexpr int STAGE = 2 * MAT;
  static constexpr int OFF_O = STAGES * STAGE;                  // [4 warps][16 rows][32 columns] f32, padded rows
  static constexpr int OFF_ML = OFF_O + 4 * DEC_ROWS * DEC_LDO * 4;  // max and sum [2][4][16]
  static constexpr int OFF_BAR = OFF_ML + 2 * 4 * DEC_ROWS * 4;
  static constexpr int OFF_MISC = OFF_BAR + 2 * STAGES * 8;
  static constexpr int TOTAL = OFF_MISC + 64;
  static constexpr int ALLOC = TOTAL + 1024;
};

// Partial results: [block][2] of O [rows][HD] and (max, sum) [rows], rows = min(group, 16).
__host__ __device__ __forceinline__ int part_rows(int G) { return G < DEC_ROWS ? (G + 1) & ~1 : DEC_ROWS; }
__host__ __device__ __forceinline__ int64_t part_floats(int hd, int rows) { return (int64_t)rows * (hd + 2); }

struct Span {              // the key tiles of a sequence
  int len, first_key, first_tile, tiles;
};
template <int TILE>
__device__ __forceinline__ Span span_of(const AttnArgs& a, int seq) {
  Span s;
  s.len = cut_length(a, seq);
  s.first_key = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
  s.first_tile = s.first_key / TILE;
  // an empty sequence has one tile with no key in it, so that its rows are written
  s.tiles = max((s.len + TILE - 1) / TILE - s.first_tile, 1);
  return s;
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Barrier of the four product warps; whether any thread's flag was set, the same answer for all.
__device__ __forceinline__ bool consumer_any(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)flag)
      : "memory");
  return r != 0;
}

// 3-D tiled TMA load: c0 in elements, c1 row inside the page, c2 page.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// The sink's logit of query head h (log2 units), summed over LANES neighbouring lanes that call
// together (all of the warp's lanes call).
template <typename T, int HD, int LANES>
__device__ __forceinline__ float sink_logit(const AttnArgs& a, int64_t tok, int h) {
  const int part = threadIdx.x & (LANES - 1);
  const T* q = reinterpret_cast<const T*>(a.q) + tok * a.ldq + (int64_t)h * HD;
  float dot = 0.f;
#pragma unroll
  for (int c = part * 4; c < HD; c += LANES * 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(q + c);
    const float2 f0 = Pair<T>::to_f(*reinterpret_cast<const typename Pair<T>::type*>(&x.x));
    const float2 f1 = Pair<T>::to_f(*reinterpret_cast<const typename Pair<T>::type*>(&x.y));
    const float4 v = __ldg(reinterpret_cast<const float4*>(a.k_sink + (int64_t)h * HD + c));
    dot = fmaf(f0.x, v.x, dot);
    dot = fmaf(f0.y, v.y, dot);
    dot = fmaf(f1.x, v.z, dot);
    dot = fmaf(f1.y, v.w, dot);
  }
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
  return dot * a.scale_log2;
}

template <typename T>
__device__ __forceinline__ float gate_of(const AttnArgs& a, int64_t tok, int h) {
  if (a.gate == nullptr) return 1.f;
  return 1.f / (1.f + expf(-to_f32(reinterpret_cast<const T*>(a.gate)[tok * a.ldg + h])));
}

// Four columns of a finished row: the sink joined, the sum divided out, the gate applied.
template <typename T, int HD>
__device__ __forceinline__ void finish_row(const AttnArgs& a, int64_t tok, int h, int col, float m, float l,
                                           const float (&o)[4], float z, float gate, bool write_lse) {
  float f = 1.f;
  if (a.k_sink != nullptr) {
    const float mt = fmaxf(m, z);
    f = m == -INFINITY ? 0.f : exp2f(m - mt);
    l = l * f + exp2f(z - mt);
    m = mt;
  }
  const float inv = gate * (l > 0.f ? f / l : (l != l ? l : 0.f));
  const typename Pair<T>::type v[2] = {Pair<T>::from_f(o[0] * inv, o[1] * inv), Pair<T>::from_f(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.o) + (tok * a.H + h) * HD + col) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&v[0]), *reinterpret_cast<const uint32_t*>(&v[1]));
  if (write_lse && a.lse != nullptr) a.lse[tok * a.H + h] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : (l != l ? l : -INFINITY);
}

// The steps 0 .. all - 1 cut into nb runs, the first `more` of them one step longer.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
struct Runs {
  int64_t nb, size, more;
  __device__ __forceinline__ Runs(int64_t all, int blocks) {
    nb = all < blocks ? all : blocks;
    size = quotient(all, nb);
    more = all - size * nb;
  }
  __device__ __forceinline__ int64_t begin(int64_t b) const { return b * size + min(b, more); }
  __device__ __forceinline__ int64_t block_of(int64_t t) const {
    const int64_t edge = more * (size + 1);
    return t < edge ? quotient(t, size + 1) : more + quotient(t - edge, size);
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(160, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const AttnArgs a, float* parts) {
  using L = DecSmem<HD>;
  constexpr int ATOMS = HD / 64, TILE = L::TILE, OVER = L::OVER;
  constexpr int KS = HD / 16;              // k-steps of S
  constexpr int KEYS = TILE / 4;           // keys of a warp
  constexpr int NT = KEYS / 8;
  constexpr int FEW = 512 / HD;            // rows that go out in one pass
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + L::STAGES;
  int64_t* s_run = reinterpret_cast<int64_t*>(smem + L::OFF_MISC);   // tiles in all, then tiles before s_seq
  int* s_seq = reinterpret_cast<int*>(smem + L::OFF_MISC + 16);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 20);
  int64_t* s_warp = reinterpret_cast<int64_t*>(smem + L::OFF_O);     // scratch of the count below

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.Hkv;
  const int blocks_g = (G + DEC_ROWS - 1) / DEC_ROWS;
  const int units = a.Hkv * blocks_g;      // per sequence
  const int prows = part_rows(G);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    *s_abort = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 128) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Count the tiles: thread t those of a contiguous share of the sequences.
  const int per = (a.num_seqs + 159) / 160;
  const int q0 = min(a.num_seqs, (int)threadIdx.x * per), q1 = min(a.num_seqs, q0 + per);
  int64_t mine = 0;
  for (int s = q0; s < q1; ++s) mine += span_of<TILE>(a, s).tiles + OVER;
  int64_t inc = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int64_t before = inc - mine, total = 0;
  for (int w = 0; w < 5; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  const int64_t all = total * units;
  const Runs runs(all, (int)gridDim.x);
  const int64_t begin = runs.begin(blockIdx.x), end = runs.begin(blockIdx.x + 1);
  const bool works = blockIdx.x < runs.nb;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the join waits for this grid's end itself
  {
    int64_t at = before;
    for (int s = q0; s < q1; ++s) {
      const int n = span_of<TILE>(a, s).tiles + OVER;
      if (works && begin >= at * units && begin < (at + n) * units) {
        *s_seq = s;
        s_run[1] = at;
      }
      at += n;
    }
  }
  __syncthreads();
  if (!works) return;

  // The run as parts: unit (seq, unit), its tiles [tile, tile + n).
  int seq = *s_seq, unit, at;              // at: step of the unit, its first OVER steps are no tiles
  Span sp = span_of<TILE>(a, seq);
  {
    const int64_t rest = begin - s_run[1] * units;
    unit = (int)quotient(rest, sp.tiles + OVER);
    at = (int)(rest - (int64_t)unit * (sp.tiles + OVER));
  }
  int64_t left = end - begin;
  int tile = 0, n = 0;
  auto advance_unit = [&]() {              // past a unit that is done (a run that ends in one stays)
    if (at < sp.tiles + OVER) return;
    at = 0;
    if (++unit < units) return;
    unit = 0;
    if (++seq < a.num_seqs) sp = span_of<TILE>(a, seq);
  };
  // the next part with a tile in it; false at the end of the run
  auto next_part = [&]() -> bool {
    while (left > 0) {
      const int steps = (int)min((int64_t)(sp.tiles + OVER - at), left);
      tile = max(at - OVER, 0);
      n = at + steps - OVER - tile;
      left -= steps;
      at += steps;
      if (n > 0) return true;
      advance_unit();
    }
    return false;
  };

  if (warp == 4) {
    // ---------------------------------------------------------------- loads
    const int rows = min(a.page, TILE);                // rows per box
    const int per_tile = TILE / rows;                  // pages of a tile
    const int boxes = per_tile * ATOMS * 2;            // lane = (page, atom, K or V)
    const int pg = lane / (2 * ATOMS), atom = (lane >> 1) % ATOMS, kv = lane & 1;
    int it = 0;
    uint32_t issued = 0, par = 0;
    bool ok = true;
    while (ok && next_part()) {
      const int hk = unit / blocks_g;
      for (int j = 0; j < n; ++j, ++it) {
        const int st = it % L::STAGES;
        const int key = (sp.first_tile + tile + j) * TILE + pg * rows;
        int page = (int)a.num_pages;                   // past the pool: TMA fills zeros
        if (lane < boxes && key < sp.len && key + rows > sp.first_key) {
          page = __ldg(a.block_table + seq * a.bt_ld + key / a.page);
          if ((unsigned)page >= (unsigned)a.num_pages) {
            record_error(ZS_DEVERR_INDEX);
            page = (int)a.num_pages;
          }
        }
        if (!warp_wait(&empty[st], ((it / L::STAGES) & 1) ^ 1, s_abort, ZS_DEVERR_TIMEOUT_PRODUCER)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[st], L::STAGE);
        __syncwarp();
        if (lane < boxes)
          tma_load_3d(smem + st * L::STAGE + kv * L::MAT + atom * (TILE * 128) + pg * rows * 128, kv ? &tmV : &tmK,
                      &full[st], atom * 64, hk * a.page + key % a.page, page);
        issued |= 1u << st;
        par = (par & ~(1u << st)) | ((uint32_t)((it / L::STAGES) & 1) << st);
      }
      advance_unit();
    }
    for (int s = 0; s < L::STAGES; ++s)                // copies in flight land before the warp leaves
      if (issued >> s & 1) mbar_wait(&full[s], par >> s & 1, nullptr, ZS_DEVERR_TIMEOUT_DRAIN);
    return;
  }

  // ------------------------------------------------------------------ products
  const int r4 = lane >> 2, c4 = lane & 3;
  float* s_o = reinterpret_cast<float*>(smem + L::OFF_O);
  float* s_m = reinterpret_cast<float*>(smem + L::OFF_ML);
  float* s_l = s_m + 4 * DEC_ROWS;
  uint32_t qf[KS][4];
  float o[HD / 8][4];
  RowRef<T> ref[2];
  float l[2];
  int it = 0;
  bool first = true;                                   // the part begins with the block's run
  while (next_part()) {
    const int hk = unit / blocks_g, g0 = (unit - hk * blocks_g) * DEC_ROWS;
    const int h0 = hk * G + g0, nrow = min(DEC_ROWS, G - g0);
    const bool whole = n == sp.tiles;
    {
      const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)seq * a.ldq + (int64_t)h0 * HD + c4 * 2;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int qr = r4 + (x & 1) * 8;
          qf[kk][x] = qr < nrow ? *reinterpret_cast<const uint32_t*>(q + qr * HD + kk * 16 + (x >> 1) * 8) : 0u;
        }
    }
    // asked for here, used when the part ends
    const int mine = h0 + min((int)threadIdx.x / (nrow <= FEW ? HD / 4 : 8), nrow - 1);   // this thread's row going out
    float z = 0.f;
    if (whole && a.k_sink != nullptr)
      z = nrow <= FEW ? sink_logit<T, HD, HD / 4>(a, seq, mine) : sink_logit<T, HD, 8>(a, seq, mine);
    const float gate = whole ? gate_of<T>(a, seq, mine) : 1.f;
#pragma unroll
    for (int c = 0; c < HD / 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][e] = 0.f;
    ref[0] = ref[1] = RowRef<T>();
    l[0] = l[1] = 0.f;
    for (int j = 0; j < n; ++j, ++it) {
      const int st = it % L::STAGES;
      const int key0 = (sp.first_tile + tile + j) * TILE + warp * KEYS;
      if (!warp_wait(&full[st], (it / L::STAGES) & 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE)) break;
      const uint32_t kb = smem_u32(smem + st * L::STAGE), vb = kb + L::MAT;
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        const int ch = kk * 2 + ((lane >> 3) & 1);     // 16-byte chunk of the row
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          const int krow = warp * KEYS + t * 8 + (lane >> 4) * 8 + (lane & 7);
          uint32_t b[4];
          ldsm_x4(kb + (ch >> 3) * (TILE * 128) + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4), b);
          mma_16816<T>(s[t], qf[kk], b[0], b[1]);
          mma_16816<T>(s[t + 1], qf[kk], b[2], b[3]);
        }
      }
      const bool edge = key0 + KEYS > sp.len || key0 < sp.first_key;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[t][e] *= a.scale_log2;
          if (edge) {
            const int k = key0 + t * 8 + c4 * 2 + (e & 1);
            if (k >= sp.len || k < sp.first_key) s[t][e] = -INFINITY;
          }
        }
      float f[2];
      bool grow = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
        for (int t = 1; t < NT; ++t) mx = fmaxf(mx, fmaxf(s[t][2 * r], s[t][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (ref[r].move(mx, &f[r])) {
          l[r] *= f[r];
          grow = true;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          o[c][0] *= f[0];
          o[c][1] *= f[0];
          o[c][2] *= f[1];
          o[c][3] *= f[1];
        }
      }
      // P in the cache's type, its sum in f32 before the rounding
      uint32_t p[NT / 2][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mu = ref[r].m == -INFINITY ? 0.f : ref[r].m;
          const float e0 = attn::fast_exp2(s[t][2 * r] - mu), e1 = attn::fast_exp2(s[t][2 * r + 1] - mu);
          l[r] += e0 + e1;
          const typename Pair<T>::type pp = Pair<T>::from_f(e0, e1);
          p[t / 2][(t & 1) * 2 + r] = *reinterpret_cast<const uint32_t*>(&pp);
        }
#pragma unroll
      for (int ks = 0; ks < NT / 2; ++ks) {
        const int vrow = warp * KEYS + ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};   // values of keys that are not seen count as zero
        if (edge) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int k = key0 + ks * 16 + t * 8 + c4 * 2;
            keep[t] = (k < sp.len && k >= sp.first_key ? 0xffffu : 0u) |
                      (k + 1 < sp.len && k + 1 >= sp.first_key ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int c = 0; c < HD / 8; c += 2) {
          const int ch = c + (lane >> 4);
          uint32_t b[4];
          ldsm_x4_t(vb + (ch >> 3) * (TILE * 128) + vrow * 128 + (((ch & 7) ^ (vrow & 7)) << 4), b);
          if (edge) {
            b[0] &= keep[0];
            b[1] &= keep[1];
            b[2] &= keep[0];
            b[3] &= keep[1];
          }
          mma_16816<T>(o[c], p[ks], b[0], b[1]);
          mma_16816<T>(o[c + 1], p[ks], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    // ------------------------------------------------------------- the part's end
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c4 == 0) {
        s_m[warp * DEC_ROWS + r4 + r * 8] = ref[r].m;
        s_l[warp * DEC_ROWS + r4 + r * 8] = l[r];
      }
    }
    float* part = parts + ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * part_floats(HD, prows);
    // COLS columns at a time through the buffer [4 warps][rows][COLS]: a group of few heads goes
    // out in one pass, 16 in HD / 32
    bool stop = false;
    auto emit = [&](auto cols) {
      constexpr int COLS = decltype(cols)::value, ROWS = 512 / COLS, LD = COLS + 8;
      const int row = threadIdx.x / (COLS / 4), col = threadIdx.x % (COLS / 4) * 4;
#pragma unroll
      for (int ps = 0; ps < HD / COLS; ++ps) {
#pragma unroll
        for (int c = 0; c < COLS / 8; ++c) {
          const float(&oc)[4] = o[ps * (COLS / 8) + c];
          float* dst = s_o + (warp * ROWS + r4) * LD + c * 8 + c4 * 2;
          if (ROWS >= 8 || r4 < ROWS) *reinterpret_cast<float2*>(dst) = make_float2(oc[0], oc[1]);
          if (ROWS > 8) *reinterpret_cast<float2*>(dst + 8 * LD) = make_float2(oc[2], oc[3]);
        }
        consumer_any(false);
        float mt = -INFINITY, lt = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) mt = fmaxf(mt, s_m[w * DEC_ROWS + row]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mw = s_m[w * DEC_ROWS + row];
          const float fw = mw == -INFINITY ? 0.f : exp2f(mw - mt);
          lt = fmaf(fw, s_l[w * DEC_ROWS + row], lt);
          const float4 x = *reinterpret_cast<const float4*>(s_o + (w * ROWS + row) * LD + col);
          acc[0] = fmaf(fw, x.x, acc[0]);
          acc[1] = fmaf(fw, x.y, acc[1]);
          acc[2] = fmaf(fw, x.z, acc[2]);
          acc[3] = fmaf(fw, x.w, acc[3]);
        }
        if (row < nrow) {
          if (whole) {
            finish_row<T, HD>(a, seq, h0 + row, ps * COLS + col, mt, lt, acc, z, gate, ps == 0 && col == 0);
          } else {
            *reinterpret_cast<float4*>(part + row * HD + ps * COLS + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (ps == 0 && col == 0) *reinterpret_cast<float2*>(part + prows * HD + row * 2) = make_float2(mt, lt);
          }
        }
        stop = consumer_any(*s_abort);                 // also: the buffer may be written again
      }
    };
    if (nrow <= FEW) emit(std::integral_constant<int, HD>());
    else emit(std::integral_constant<int, 32>());
    if (stop) return;
    advance_unit();
    first = false;
  }
}

// Block (sequence, unit): the sum of its parts, where more than one block of the decode
// kernel had a part of it.  A warp takes a row (four columns a lane) or, when the rows are
// few, one of several shares of a row's parts; it keeps four parts' loads in flight.
constexpr int JOIN_WARPS = 8;

template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const AttnArgs a, const float* parts,
                                                                     int decode_blocks) {
  constexpr int SUB = 128 / HD;            // parts side by side in a warp
  constexpr int OVER = DecSmem<HD>::OVER, TILE = DecSmem<HD>::TILE;
  __shared__ float s_o[JOIN_WARPS][HD], s_ml[JOIN_WARPS][2];
  __shared__ int64_t s_n[JOIN_WARPS][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.Hkv;
  const int blocks_g = (G + DEC_ROWS - 1) / DEC_ROWS;
  const int units = a.Hkv * blocks_g, prows = part_rows(G);
  const int seq = blockIdx.x, unit = blockIdx.y;
  const int hk = unit / blocks_g, g0 = (unit - hk * blocks_g) * DEC_ROWS;
  const int h0 = hk * G + g0, nrow = min(DEC_ROWS, G - g0);
  // all that does not come from the decode kernel, before its end
  int64_t before = 0, total = 0;
  for (int s = threadIdx.x; s < a.num_seqs; s += JOIN_WARPS * 32) {
    const int n = span_of<TILE>(a, s).tiles + OVER;
    total += n;
    if (s < seq) before += n;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, off);
    total += __shfl_xor_sync(0xffffffffu, total, off);
  }
  if (lane == 0) {
    s_n[warp][0] = before;
    s_n[warp][1] = total;
  }
  const int steps = span_of<TILE>(a, seq).tiles + OVER;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) {
    before += s_n[w][0];
    total += s_n[w][1];
  }
  const Runs runs(total * units, decode_blocks);
  const int64_t t0 = before * units + (int64_t)unit * steps + OVER, t1 = t0 + steps - OVER - 1;   // its first and last tile
  const int b0 = (int)runs.block_of(t0), b1 = (int)runs.block_of(t1);
  // every block waits, also one with nothing to join: what follows this grid in the stream follows the
  // decode kernel only through it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (b0 == b1) return;
  // a block's first part lies in its slot 0; the first block's part may come after another one
  const int shift = runs.begin(b0) < t0 - OVER ? 1 : 0;
  const int shares = nrow >= JOIN_WARPS ? 1 : JOIN_WARPS / nrow;
  const int share = warp % shares, sub = lane / (HD / 4), col = (lane % (HD / 4)) * 4;
  for (int row = warp / shares; row < nrow; row += JOIN_WARPS / shares) {
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int step = shares * SUB;
    for (int b = b0 + share * SUB + sub; b <= b1; b += 4 * step) {
      float4 o[4];
      float2 ml[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int bb = b + e * step;
        ml[e] = make_float2(-INFINITY, 0.f);
        o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (bb <= b1) {
          const float* part = parts + ((int64_t)bb * 2 + (bb == b0 ? shift : 0)) * part_floats(HD, prows);
          ml[e] = *reinterpret_cast<const float2*>(part + prows * HD + row * 2);
          o[e] = *reinterpret_cast<const float4*>(part + row * HD + col);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mt = fmaxf(m, ml[e].x);
        const float f = m == -INFINITY ? 0.f : exp2f(m - mt), fe = ml[e].x == -INFINITY ? 0.f : exp2f(ml[e].x - mt);
        l = l * f + ml[e].y * fe;
        acc[0] = acc[0] * f + o[e].x * fe;
        acc[1] = acc[1] * f + o[e].y * fe;
        acc[2] = acc[2] * f + o[e].z * fe;
        acc[3] = acc[3] * f + o[e].w * fe;
        m = mt;
      }
    }
    if (SUB == 2) {                        // the two halves of the warp, the lower first
      const float mo = __shfl_xor_sync(0xffffffffu, m, 16), lo = __shfl_xor_sync(0xffffffffu, l, 16);
      const float mt = fmaxf(m, mo);
      const float f = m == -INFINITY ? 0.f : exp2f(m - mt), fo = mo == -INFINITY ? 0.f : exp2f(mo - mt);
      l = l * f + lo * fo;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = acc[e] * f + __shfl_xor_sync(0xffffffffu, acc[e], 16) * fo;
      m = mt;
    }
    if (shares > 1) {                      // then every warp is here once
      if (sub == 0) *reinterpret_cast<float4*>(&s_o[warp][col]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (lane == 0) {
        s_ml[warp][0] = m;
        s_ml[warp][1] = l;
      }
    } else {
      const int h = h0 + row;
      const float z = a.k_sink != nullptr ? sink_logit<T, HD, 32>(a, seq, h) : 0.f;
      if (sub == 0) finish_row<T, HD>(a, seq, h, col, m, l, acc, z, gate_of<T>(a, seq, h), col == 0);
    }
  }
  if (shares == 1) return;
  __syncthreads();
  const int row = warp / shares;
  if (share != 0 || row >= nrow) return;
  const int h = h0 + row;
  const float z = a.k_sink != nullptr ? sink_logit<T, HD, 32>(a, seq, h) : 0.f;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int w = warp; w < warp + shares; ++w) m = fmaxf(m, s_ml[w][0]);
  for (int w = warp; w < warp + shares; ++w) {
    const float f = s_ml[w][0] == -INFINITY ? 0.f : exp2f(s_ml[w][0] - m);
    l = fmaf(f, s_ml[w][1], l);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, s_o[w][col + e], acc[e]);
  }
  if (sub == 0) finish_row<T, HD>(a, seq, h, col, m, l, acc, z, gate_of<T>(a, seq, h), col == 0);
}

// ------------------------------------------------------------------------ prompt
//
// Packed new tokens on the 5th-generation tensor cores.  The query heads of one key head share
// its keys, so a row is a (token, head of the group) pair: a tile of 128 rows is 128 / G tokens
// (short chunks after long prefixes fill it too), and a block is two such tiles of one
// sequence and key head.  As in the decode kernel the work is a list of steps, one per key tile of a
// block (and PT_OVER for its start and end), cut on the device into equal runs, one per persistent
// CTA: prompts of any lengths load every SM alike, and few rows after a long prefix are split over
// its length.  Blocks that a cut goes through leave parts in the workspace, which
// paged_prompt_join_kernel adds in the order of the CTAs.  The loads of the next block run while
// the rows of the last one go out.
//
//   warp 0      TMA: both Q tiles, then K and V of 128 keys, page by page, into a ring of slots
//   warp 1      MMA: per key tile and query tile t, O_t += P_t V (P from tensor memory, the first
//               half of its keys as soon as that half is there), then S_t = Q_t K^T
//   warps 2, 3  rows of no sequence (zero); the sink logits of query tiles 0 and 1
//   warps 4..7  softmax of query tile 0, warps 8..11 of query tile 1: one row per thread; S from
//               tensor memory, reference and sum (RowRef), P in the cache's type over S's first 64
//               columns, at the end the row out
// TMEM columns: S_t / P_t at t * 128, O_t at 256 + t * hd.  P is rounded to the cache's type because the
// products take 16-bit operands; its sum is taken in f32 before that.
//
// One prompt of 32768 tokens, 16/4 heads of 128: 4.01 to 4.16 ms by the clock, 1097 to 1057 TFLOP/s (65 to 62 % of a
// cuBLAS burst).  Bound by
// the chain of a query tile: of 3850 cycles for a step of both tiles, softmax takes 2000, products and
// waits 1700 to 1800, and the two tiles overlap each other's; pure products would take 2100.

constexpr int PT_ROWS = 128;              // rows of a query tile
constexpr int PT_KEYS = 128;              // keys of a key tile
constexpr int PT_THREADS = 384;
// Registers: launched with 168 a thread (384 * 168 = 64512); the first four warps give back what
// the softmax warps, which hold a whole row of S, take: 128 * (104 + 2 * 200) = 64512.
constexpr int PT_REGS_AUX = 104, PT_REGS_SOFTMAX = 200;
constexpr int PT_PLAN = 256;              // threads that count the work
// Steps of a block's start and end, and of the shortest run (where that leaves no block without a CTA).
// Measured (2, 6), (4, 6), (6, 10), (4, 16), (8, 16): nine packed prompts of 5 to 4096 tokens 225, 220, 225,
// 220, 236 us; three of 300 to 800 tokens 39.8, 35.7, 39.5, 42.0, 38.2 us.
constexpr int PT_OVER = 4;
constexpr int PT_LEAST = 6;
constexpr int PT_MAX_CTAS = 160;

// One lane of the converged warp; the compiler keeps what the branch computes in uniform registers,
// where the tensor instructions want their descriptors.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)::"memory");
  return r != 0;
}
// Products with the descriptors' low words as arguments (address and leading offset; the high word,
// stride 1024 bytes and 128-byte swizzle, is the same for all): one addition per operand and step.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* p, uint32_t lead) {
  return (smem_u32(p) >> 4 & 0x3FFF) | (lead >> 4) << 16;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "n"(DESC_HI), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "n"(DESC_HI), "r"(idesc), "r"(acc)
      : "memory");
}

template <int HD>
struct PromptSmem {
  static constexpr int TILE = 128 * HD * 2;
  static constexpr int SLOTS = HD == 128 ? 5 : 8;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_PLAN = OFF_KV;                // scratch of the count, before the first load
  static constexpr int OFF_PART = OFF_KV + SLOTS * TILE; // parts published by the loading warp (64 bytes each)
  static constexpr int OFF_CUT = OFF_PART + 4 * 64;
  static constexpr int OFF_Z = OFF_CUT + 32;             // sink logits of the query tiles' rows
  static constexpr int OFF_BAR = OFF_Z + 2 * 128 * 4;
  // q_full[2], q_empty[2], kv_full[SLOTS], kv_empty[SLOTS], s_full[2], p_half[2], p_full[2], o_done[2], o_free[2],
  // z_full[2], z_free[2], part_full[4], part_empty[4], done
  static constexpr int NBAR = 4 + 2 * SLOTS + 23;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int TOTAL = OFF_MISC + 16;
  static constexpr int ALLOC = TOTAL + 1024;
};

struct PromptBlock {
  int tok0;                // packed row of the block's first token
  int left;                // tokens of the sequence from there on
  int pos0;                // position of the first token
  int len;                 // tokens in the cache (cut)
  int floor;               // no query of the sequence sees a key before this one
  int lo[2], cnt[2];       // key tiles of the two query tiles
  int first, tiles;        // of both: one range (a window reaches back at least to the token itself)
};

// Packed row i of cu_seqlens, inside the rows there are.
__device__ __forceinline__ int cut_row(const AttnArgs& a, int i) {
  return min(max(__ldg(a.cu + i), 0), (int)a.tokens);
}
// Blocks of a sequence.
__device__ __forceinline__ int blocks_of(const AttnArgs& a, int seq, int per) {
  const int n = cut_row(a, seq + 1) - cut_row(a, seq);
  return n > 0 ? (n + per - 1) / per : 0;
}
__device__ __forceinline__ PromptBlock block_at(const AttnArgs& a, int seq, int blk, int tpt) {
  PromptBlock b;
  const int first = cut_row(a, seq), n = cut_row(a, seq + 1) - first, skip = blk * 2 * tpt;
  b.tok0 = first + skip;
  b.left = n - skip;
  b.len = cut_length(a, seq);
  b.pos0 = b.len - n + skip;
  b.floor = first_seen(b.len - n, a.window);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const KeyTiles k = key_tiles<PT_KEYS>(b.pos0 + t * tpt, min(b.left - t * tpt, tpt), a.window);
    b.lo[t] = k.lo;
    b.cnt[t] = k.cnt;
  }
  b.first = b.cnt[0] > 0 ? b.lo[0] : b.lo[1];
  const int end = b.cnt[1] > 0 ? b.lo[1] + b.cnt[1] : b.lo[0] + b.cnt[0];
  b.tiles = b.cnt[0] + b.cnt[1] > 0 ? end - b.first : 0;
  return b;
}
// A block without a key still counts one, so that its rows are written.
__device__ __forceinline__ int steps_of(const PromptBlock& b) { return PT_OVER + max(b.tiles, 1); }

// A run of steps as parts of blocks: key tiles [b.first, b.first + b.tiles) of block (seq, blk) of
// key head hk, the two query tiles' ranges cut to them.
struct PromptRun {
  int part_seq, part_hk;
  int seq, blk, hk, at;    // at: step of the block, its first PT_OVER steps are no tiles
  int64_t left;
  int tpt;
  bool first, starts, ends;   // the part is the run's first one, holds its block's first tile, its last one
  PromptBlock b;
  bool begun;

  __device__ __forceinline__ bool next(const AttnArgs& a) {
    first = !begun;
    while (left > 0) {
      b = block_at(a, seq, blk, tpt);
      part_seq = seq;
      part_hk = hk;
      const int all = steps_of(b), steps = (int)min((int64_t)(all - at), left);
      const int tile = max(at - PT_OVER, 0), n = at + steps - PT_OVER - tile;
      left -= steps;
      at += steps;
      const bool done = at == all;
      if (done) {                                        // the block after it
        at = 0;
        ++blk;
        while (left > 0 && blk >= blocks_of(a, seq, 2 * tpt)) {
          blk = 0;
          if (++seq == a.num_seqs) {
            seq = 0;
            ++hk;
          }
        }
      }
      if (n <= 0) continue;
      starts = tile == 0;
      ends = done;
      if (b.tiles > 0) {
        b.first += tile;
        b.tiles = n;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int end = min(b.lo[t] + b.cnt[t], b.first + n);
          b.lo[t] = max(b.lo[t], b.first);
          b.cnt[t] = max(end - b.lo[t], 0);
        }
      }
      begun = true;
      return true;
    }
    return false;
  }
};

// A part as the loading warp publishes it to the others.
struct PromptPart {
  int live;                // 0: the run has ended
  int hk, tok0, left, pos0, len, floor;
  int lo[2], cnt[2], first, tiles;
  int flags;               // 1: the run's first part, 2: holds its block's first tile, 4: its last one
};
constexpr int PT_PARTS = 4;

// Parts in the workspace: per CTA and slot (0: the run's first part, 1: its last) the two query tiles'
// O [hd / 4][128 rows] of four columns, then (max, sum, sink logit) [128 rows]; per CTA what the
// join has to know.
__host__ __device__ constexpr int64_t prompt_part_floats(int hd) { return (int64_t)2 * PT_ROWS * (hd + 4); }
struct PromptCut {
  int cut, cont;           // the run's last part does not end its block; its first one does not start it
  int single;              // both are the same part
  int slot, hk, tok0, left, pad;
};

// Exclusive scan over the PT_PLAN threads of warps 4 .. 11.
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* s, int64_t* sum) {
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - 4;
  int64_t inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  if (lane == 31) s[warp] = inc;
  asm volatile("bar.sync 1, 256;" ::: "memory");
  int64_t before = inc - v, all = 0;
#pragma unroll
  for (int w = 0; w < PT_PLAN / 32; ++w) {
    if (w < warp) before += s[w];
    all += s[w];
  }
  asm volatile("bar.sync 1, 256;" ::: "memory");
  *sum = all;
  return before;
}

// This CTA's run, found by warps 4 .. 11: blocks counted over groups of sequences, steps over groups of blocks.
__device__ __forceinline__ void plan_run(const AttnArgs& a, int tpt, uint8_t* scratch, PromptRun* out) {
  int64_t* s = reinterpret_cast<int64_t*>(scratch);
  int64_t* sums = s + PT_PLAN / 32;                      // blocks before each group
  const int g = threadIdx.x - 128, per = 2 * tpt;
  const int group = (a.num_seqs + PT_PLAN - 1) / PT_PLAN;
  int64_t mine = 0, blocks, steps;
  for (int q = g * group; q < min(a.num_seqs, (g + 1) * group); ++q) mine += blocks_of(a, q, per);
  sums[g] = plan_scan(mine, s, &blocks);
  asm volatile("bar.sync 1, 256;" ::: "memory");
  const int64_t b0 = blocks * g / PT_PLAN, b1 = blocks * (g + 1) / PT_PLAN;
  int seq = 0, blk = 0;
  if (b0 < b1) {                                         // block b0: its group, then its sequence
    int lo = 0, hi = PT_PLAN;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] <= b0) lo = mid; else hi = mid;
    }
    seq = lo * group;
    int64_t rest = b0 - sums[lo];
    for (int n; rest >= (n = blocks_of(a, seq, per)); ++seq) rest -= n;
    blk = (int)rest;
  }
  const int seq0 = seq, blk0 = blk;
  mine = 0;
  for (int64_t b = b0; b < b1; ++b) {
    while (blk >= blocks_of(a, seq, per)) ++seq, blk = 0;
    mine += steps_of(block_at(a, seq, blk++, tpt));
  }
  const int64_t before = plan_scan(mine, s, &steps);
  if (g == 0) out->left = 0;
  asm volatile("bar.sync 1, 256;" ::: "memory");
  if (steps == 0) return;                                // no packed row
  // no run so short that its start and end cost more than it holds, unless blocks are that short
  const int64_t all = steps * a.Hkv, want = max(all / PT_LEAST, blocks * a.Hkv);
  const Runs runs(all, (int)min(want, (int64_t)gridDim.x));
  if (blockIdx.x >= runs.nb) return;
  const int64_t begin = runs.begin(blockIdx.x);
  const int64_t hk = quotient(begin, steps), r = begin - hk * steps;
  if (r < before || r >= before + mine) return;
  int64_t at = r - before;
  seq = seq0, blk = blk0;
  while (true) {
    while (blk >= blocks_of(a, seq, per)) ++seq, blk = 0;
    const int n = steps_of(block_at(a, seq, blk, tpt));
    if (at < n) break;
    at -= n;
    ++blk;
  }
  out->seq = seq;
  out->blk = blk;
  out->hk = (int)hk;
  out->at = (int)at;
  out->left = runs.begin(blockIdx.x + 1) - begin;
}

template <typename T, int HD>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const AttnArgs a, float* parts, PromptCut* cuts) {
  using L = PromptSmem<HD>;
  constexpr int SLOTS = L::SLOTS;
  constexpr int ATOMS = HD / 64, ATOM = 128 * 128;       // 128 rows of 128 bytes
  constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0 : 1;
  constexpr uint32_t IDESC_S = idesc_f16(128, 128, FMT, 0, 0);
  constexpr uint32_t IDESC_PV = idesc_f16(128, HD, FMT, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PromptRun* s_run = reinterpret_cast<PromptRun*>(smem + L::OFF_PART);    // seq .. left of it, before the first part
  PromptPart* s_part = reinterpret_cast<PromptPart*>(smem + L::OFF_PART);
  float* s_z = reinterpret_cast<float*>(smem + L::OFF_Z);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_empty = q_full + 2;
  uint64_t* kv_full = q_empty + 2;
  uint64_t* kv_empty = kv_full + SLOTS;
  uint64_t* s_full = kv_empty + SLOTS;
  uint64_t* p_half = s_full + 2;
  uint64_t* p_full = p_half + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  uint64_t* z_full = o_free + 2;
  uint64_t* z_free = z_full + 2;
  uint64_t* part_full = z_free + 2;
  uint64_t* part_empty = part_full + PT_PARTS;
  uint64_t* done = part_empty + PT_PARTS;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.Hkv;
  const int tpt = PT_ROWS / G;                           // tokens of a tile; a block has two

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 2);                         // its last product, and its sink logits
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&z_full[t], 1);
      mbar_init(&z_free[t], 4);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < PT_PARTS; ++s) {
      mbar_init(&part_full[s], 1);
      mbar_init(&part_empty[s], 11);                     // products, sink logits, softmax
    }
    mbar_init(done, 1);
    *s_abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the join waits for this grid's end itself
  if (warp >= 4) {
    plan_run(a, tpt, smem + L::OFF_PLAN, s_run);
    fence_proxy_async_smem();                            // the scratch is written by the copy engine next
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // The next part, for a warp other than the loading one.
  uint32_t part_n = 0;
  auto next_part = [&](PromptPart& b) -> bool {
    const int sl = part_n % PT_PARTS;
    if (!warp_wait(&part_full[sl], part_n / PT_PARTS & 1, s_abort, ZS_DEVERR_TIMEOUT_PRODUCER)) return false;
    b = s_part[sl];
    __syncwarp();
    if (lane == 0) mbar_arrive(&part_empty[sl]);
    ++part_n;
    return b.live != 0;
  };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_REGS_AUX));
  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    const int rows = min(a.page, PT_KEYS), boxes = PT_KEYS / rows * ATOMS;   // lane = (page, atom)
    const int pg = lane / ATOMS, atom = lane % ATOMS;
    uint32_t issued = 0, par = 0, q_n[2] = {0, 0};
    int item = 0;
    bool ok = true;
    PromptRun run;
    run.seq = s_run->seq;
    run.blk = s_run->blk;
    run.hk = s_run->hk;
    run.at = s_run->at;
    run.left = s_run->left;
    run.tpt = tpt;
    run.begun = false;
    __syncwarp();
    while (ok) {
      const bool live = run.next(a);
      const PromptBlock& b = run.b;
      const int sl = part_n % PT_PARTS;
      ok = warp_wait(&part_empty[sl], part_n / PT_PARTS & 1 ^ 1, s_abort, ZS_DEVERR_TIMEOUT_PRODUCER);
      if (!ok) break;
      if (lane == 0) {
        PromptPart& o = s_part[sl];
        o.live = live ? 1 : 0;
        o.hk = run.part_hk;
        o.tok0 = b.tok0;
        o.left = b.left;
        o.pos0 = b.pos0;
        o.len = b.len;
        o.floor = b.floor;
        o.lo[0] = b.lo[0];
        o.lo[1] = b.lo[1];
        o.cnt[0] = b.cnt[0];
        o.cnt[1] = b.cnt[1];
        o.first = b.first;
        o.tiles = b.tiles;
        o.flags = (run.first ? 1 : 0) | (run.starts ? 2 : 0) | (run.ends ? 4 : 0);
        mbar_arrive(&part_full[sl]);
      }
      ++part_n;
      if (!live) break;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || b.cnt[t] == 0) continue;
        ok = warp_wait(&q_empty[t], (q_n[t] & 1) ^ 1, s_abort, ZS_DEVERR_TIMEOUT_PRODUCER);
        if (!ok) continue;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[t], G * tpt * HD * 2);
#pragma unroll
          for (int at = 0; at < ATOMS; ++at)
            tma_load_3d(smem + L::OFF_Q + t * L::TILE + at * ATOM, &tmQ, &q_full[t], at * 64, run.part_hk * G,
                        b.tok0 + t * tpt);
        }
        ++q_n[t];
      }
      if (b.cnt[0] + b.cnt[1] == 0) continue;
      for (int j = b.first; ok && j < b.first + b.tiles; ++j) {
        const int key = j * PT_KEYS + pg * rows;
        int page = (int)a.num_pages;                     // past the pool: TMA fills zeros
        if (lane < boxes && key < b.len && key + rows > b.floor) {
          page = __ldg(a.block_table + run.part_seq * a.bt_ld + key / a.page);
          if ((unsigned)page >= (unsigned)a.num_pages) {
            record_error(ZS_DEVERR_INDEX);
            page = (int)a.num_pages;
          }
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++item) {
          const int st = item % SLOTS;
          if (!warp_wait(&kv_empty[st], ((item / SLOTS) & 1) ^ 1, s_abort, ZS_DEVERR_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], L::TILE);
          __syncwarp();
          if (lane < boxes)
            tma_load_3d(smem + L::OFF_KV + st * L::TILE + atom * ATOM + pg * rows * 128, kv ? &tmV : &tmK, &kv_full[st],
                        atom * 64, run.part_hk * a.page + key % a.page, page);
          issued |= 1u << st;
          par = (par & ~(1u << st)) | ((uint32_t)((item / SLOTS) & 1) << st);
        }
      }
    }
    // copies in flight land before the CTA leaves
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (q_n[t] > 0) mbar_wait(&q_full[t], (q_n[t] - 1) & 1, nullptr, ZS_DEVERR_TIMEOUT_DRAIN);
    for (int s = 0; s < SLOTS; ++s)
      if (issued & (1u << s)) mbar_wait(&kv_full[s], (par >> s) & 1, nullptr, ZS_DEVERR_TIMEOUT_DRAIN);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ products
    bool ok = true, issued_any = false;
    int item = 0;                // of the ring: the block's first K
    uint32_t q_n[2] = {0, 0};    // Q tiles waited for
    uint32_t p_n[2] = {0, 0};    // P tiles waited for
    uint32_t b_n[2] = {0, 0};    // blocks begun, per query tile
    const uint32_t q_lo = desc_lo(smem + L::OFF_Q, 16), k_lo = desc_lo(smem + L::OFF_KV, 16),
                   v_lo = desc_lo(smem + L::OFF_KV, ATOM);
    auto ready = [&](int it) -> bool {
      return warp_wait(&kv_full[it % SLOTS], (it / SLOTS) & 1, s_abort, ZS_DEVERR_TIMEOUT_MMA);
    };
    PromptPart b;
    while (ok && next_part(b)) {
      if (b.cnt[0] + b.cnt[1] == 0) continue;
      const int ulo = b.first, uhi = b.first + b.tiles - 1;
      const int end[2] = {b.lo[0] + b.cnt[0], b.lo[1] + b.cnt[1]};
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (ok && b.cnt[t] > 0) ok = warp_wait(&q_full[t], q_n[t]++ & 1, s_abort, ZS_DEVERR_TIMEOUT_MMA);
      ok = ok && ready(item);
      // Step j: per query tile O_t += P_t V_{j-1}, then S_t = Q_t K_j; what step j + 1 reads is waited for
      // between the two query tiles, where the tensor pipe has work queued.
      int ks = item % SLOTS, vs = 0;
      for (int j = ulo; ok && j <= uhi + 1; ++j) {
        int ks_next = 0, vs_next = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (ok && j - 1 >= b.lo[t] && j - 1 < end[t]) {
            // the block's first product overwrites O: the last block's rows must be out
            const bool fresh = j - 1 == b.lo[t];
            if (fresh) ok = warp_wait(&o_free[t], (b_n[t]++ & 1) ^ 1, s_abort, ZS_DEVERR_TIMEOUT_MMA);
            const uint32_t va = v_lo + vs * (L::TILE >> 4);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              ok = ok && warp_wait(hf == 0 ? &p_half[t] : &p_full[t], p_n[t] & 1, s_abort, ZS_DEVERR_TIMEOUT_MMA);
              tc_fence_after();
              if (ok && elect_one()) {
#pragma unroll
                for (int kk = hf * 4; kk < hf * 4 + 4; ++kk)
                  mma_ts(tmem + 256 + t * HD, tmem + t * 128 + kk * 8, va + kk * (2048 >> 4), IDESC_PV,
                         kk > 0 ? 1u : (fresh ? 0u : 1u));
                if (hf == 1 && j == end[t]) tc_commit(&o_done[t]);
              }
              __syncwarp();
            }
            ++p_n[t];
          }
          if (ok && j >= b.lo[t] && j < end[t]) {
            tc_fence_after();
            if (elect_one()) {
              const uint32_t qa = q_lo + t * (L::TILE >> 4), ka = k_lo + ks * (L::TILE >> 4);
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const uint32_t off = (kk / 4) * (ATOM >> 4) + (kk % 4) * (32 >> 4);
                mma_ss(tmem + t * 128, qa + off, ka + off, IDESC_S, kk > 0 ? 1u : 0u);
              }
              tc_commit(&s_full[t]);
              if (j + 1 == end[t]) tc_commit(&q_empty[t]);     // the block's last use of this Q
            }
            issued_any = true;
            __syncwarp();
          }
          if (t == 1 && elect_one()) {                         // both query tiles have read these
            if (j <= uhi) tc_commit(&kv_empty[ks]);
            if (j > ulo) tc_commit(&kv_empty[vs]);
          }
          if (t == 0 && ok) {
            if (j <= uhi) {
              vs_next = (item + 1) % SLOTS;
              ok = ready(item + 1);
              // Values of keys that no query sees (behind the sequence, before every window) count as zero,
              // whatever lies there: 0 * NaN would reach every row.
              const int k0 = j * PT_KEYS;
              if (k0 + PT_KEYS > b.len || k0 < b.floor) {
                uint8_t* v = smem + L::OFF_KV + vs_next * L::TILE;
                for (int r = 0; r < PT_KEYS; ++r) {
                  if (k0 + r < b.len && k0 + r >= b.floor) continue;
                  if (lane < 8 * ATOMS)
                    *reinterpret_cast<uint4*>(v + (lane >> 3) * ATOM + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            if (j < uhi) {
              ks_next = (item + 2) % SLOTS;
              ok = ok && ready(item + 2);
            }
          }
        }
        ks = ks_next;
        vs = vs_next;
        if (j <= uhi) item += 2;
      }
    }
    if (issued_any) {                                    // what was issued ends before the warp leaves
      if (elect_one()) {
        tc_commit(done);
        mbar_wait(done, 0, nullptr, ZS_DEVERR_TIMEOUT_DRAIN);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ rows of no sequence, sink logits of tile t
    const int t = warp - 2;
    const int64_t end = cut_row(a, a.num_seqs), begin = cut_row(a, 0);
    const int64_t me = (int64_t)blockIdx.x * 64 + threadIdx.x - 64, all = (int64_t)gridDim.x * 64;
    const int64_t words = (int64_t)a.H * (HD / 8);
    for (int64_t e = me; e < a.tokens * words; e += all) {
      const int64_t tok = e / words;
      if (tok >= begin && tok < end) {
        e += (end - 1 - tok) * words / all * all;        // on to the rows behind the sequences
        continue;
      }
      reinterpret_cast<uint4*>(a.o)[e] = make_uint4(0, 0, 0, 0);
      if (a.lse != nullptr && e % (HD / 8) == 0) a.lse[e / (HD / 8)] = -INFINITY;
    }
    __syncwarp();
    uint32_t q_n = 0, z_n = 0;
    bool ok = true;
    PromptPart b;
    while (ok && next_part(b)) {
      const int tokens = min(b.left - t * tpt, tpt);
      if (tokens <= 0) continue;
      const bool loaded = (t == 0 ? b.cnt[0] : b.cnt[1]) > 0;
      if (loaded) ok = warp_wait(&q_full[t], q_n++ & 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      if (a.k_sink != nullptr && loaded) {
        // Q K_sink^T by mma.sync, 16 rows by 8 heads at a time, from which each row takes its own head's
        // column; the f32 sink as the sum of two values of Q's type (2^-17 of it is lost in bf16, 2^-22 in
        // f16), which f16 has the range for once a head's sink is brought to below 2^14 by a power of two.
        // Little code: what runs once a part is fetched anew each time, a few cycles an instruction.
        ok = warp_wait(&z_free[t], (z_n++ & 1) ^ 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE);
        if (!ok) break;
        const uint32_t qt = smem_u32(smem + L::OFF_Q + t * L::TILE);
        const int r4 = lane >> 2, c4 = lane & 3, inv = 65536 / G + 1;   // r / G == r * inv >> 16 for r < 128
#pragma unroll 1
        for (int g0 = 0; g0 < G; g0 += 8) {
          uint32_t hi[HD / 16][2], lo[HD / 16][2];
          const float* sink = a.k_sink + (int64_t)(b.hk * G + min(g0 + r4, G - 1)) * HD + c4 * 2;
          float up = 1.f, down[2] = {1.f, 1.f};          // the power of two; its inverse for this lane's columns
          if (std::is_same<T, __half>::value) {
            float big = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 8; ++kk) {
              const float2 f = __ldg(reinterpret_cast<const float2*>(sink + kk * 8));
              big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int e = min(267 - (__float_as_int(big) >> 23), 253);
            up = __int_as_float(e << 23);
#pragma unroll
            for (int x = 0; x < 2; ++x)
              down[x] = __shfl_sync(0xffffffffu, __int_as_float((254 - e) << 23), (c4 * 2 + x) * 4);
          }
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float2 f = __ldg(reinterpret_cast<const float2*>(sink + kk * 16 + x * 8));
              f.x *= up;
              f.y *= up;
              const typename Pair<T>::type h2 = Pair<T>::from_f(f.x, f.y);
              const float2 g2 = Pair<T>::to_f(h2);
              const typename Pair<T>::type l2 = Pair<T>::from_f(f.x - g2.x, f.y - g2.y);
              hi[kk][x] = *reinterpret_cast<const uint32_t*>(&h2);
              lo[kk][x] = *reinterpret_cast<const uint32_t*>(&l2);
            }
#pragma unroll 1
          for (int r0 = 0; r0 < G * tokens; r0 += 16) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            const int row = r0 + (lane & 15);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const int ch = kk * 2 + (lane >> 4);
              uint32_t q4[4];
              ldsm_x4(qt + (ch >> 3) * ATOM + row * 128 + (((ch & 7) ^ (row & 7)) << 4), q4);
              mma_16816<T>(acc, q4, hi[kk][0], hi[kk][1]);
              mma_16816<T>(acc, q4, lo[kk][0], lo[kk][1]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int r = r0 + r4 + x * 8, g = r - (r * inv >> 16) * G - g0;
              if (g >> 1 == c4) s_z[t * PT_ROWS + r] = g & 1 ? acc[x * 2 + 1] * down[1] : acc[x * 2] * down[0];
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&z_full[t]);
      }
      __syncwarp();
      if (loaded && lane == 0) mbar_arrive(&q_empty[t]);
    }
  }
  } else {
    // ------------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_REGS_SOFTMAX));
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;                   // this thread's row
    const int tr = r / G, g = r - tr * G;                // its token in the tile, its head in the group
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t ts = tmem + lane_base + t * 128, to = tmem + lane_base + 256 + t * HD;
    const uint64_t scale2 = attn::pack2(__float_as_uint(a.scale_log2), __float_as_uint(a.scale_log2));
    uint32_t s_n = 0, b_n = 0, z_n = 0;
    bool ok = true;
    PromptCut* cut = reinterpret_cast<PromptCut*>(smem + L::OFF_CUT);   // one thread's: what the join has to know
    if (threadIdx.x == 128) *cut = PromptCut{0, 0, 0, 0, 0, 0, 0, 0};
    PromptPart b;
    while (ok && next_part(b)) {
      if (threadIdx.x == 128) {
        if (b.flags & 1) cut->cont = b.flags & 2 ? 0 : 1;
        cut->cut = b.flags & 4 ? 0 : 1;
        cut->single = b.flags & 1;
        cut->slot = b.flags & 1 ? 0 : 1;
        cut->hk = b.hk;
        cut->tok0 = b.tok0;
        cut->left = b.left;
      }
      const int tokens = min(b.left - t * tpt, tpt);     // of the tile
      if (tokens <= 0) continue;
      const bool valid = tr < tokens;
      const int p0 = b.pos0 + t * tpt, p = p0 + tr;      // the tile's first position, the row's
      const int h = b.hk * G + g;
      const int64_t tok = (int64_t)b.tok0 + t * tpt + tr;
      const float gate = valid ? gate_of<T>(a, tok, h) : 1.f;   // asked for here, used when the part ends
      const int n = t == 0 ? b.cnt[0] : b.cnt[1], lo = t == 0 ? b.lo[0] : b.lo[1];
      RowRef<T> ref;
      float l = 0.f;
      for (int uu = 0; uu < n; ++uu) {
        const int k0 = (lo + uu) * PT_KEYS;
        if (!warp_wait(&s_full[t], s_n & 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        ++s_n;
        tc_fence_after();
        uint32_t sr[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[c * 32]));
        tc_wait_ld();
        const bool edge = k0 + PT_KEYS - 1 > p0 || (a.window > 0 && p0 + tokens - 1 - k0 >= a.window);
        if (edge) {
          const int k1 = p - k0;                                         // last and first visible column
          const int kf = a.window > 0 ? p - (a.window - 1) - k0 : 0;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c > k1 || c < kf) sr[c] = __float_as_uint(-INFINITY);
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 128; c += 8) {
          mx0 = attn::fmax3(mx0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          mx1 = attn::fmax3(mx1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
          mx2 = attn::fmax3(mx2, __uint_as_float(sr[c + 4]), __uint_as_float(sr[c + 5]));
          mx3 = attn::fmax3(mx3, __uint_as_float(sr[c + 6]), __uint_as_float(sr[c + 7]));
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * a.scale_log2;
        float f;
        const bool need = ref.move(mx, &f);
        if (need) l *= f;
        // O_t holds every earlier product of the block (this S_t was issued after them)
        if (uu >= 1 && __any_sync(0xffffffffu, need)) {
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(to + c * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            attn::tmem_st_32x32b_x32(to + c * 32, o);
          }
        }
        const float mu = ref.m == -INFINITY ? 0.f : ref.m;   // nothing seen so far: every P is exp2(-inf)
        const uint64_t negm = attn::pack2(__float_as_uint(-mu), __float_as_uint(-mu));
        uint64_t acc0 = 0, acc1 = 0;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t pw[32];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const int c = hf * 64 + 2 * x;
            float e0, e1, e2, e3;
            attn::unpack2(attn::ffma2(attn::pack2(sr[c], sr[c + 1]), scale2, negm), e0, e1);
            attn::unpack2(attn::ffma2(attn::pack2(sr[c + 2], sr[c + 3]), scale2, negm), e2, e3);
            e0 = attn::fast_exp2(e0);
            e1 = attn::fast_exp2(e1);
            e2 = attn::fast_exp2(e2);
            e3 = attn::fast_exp2(e3);
            acc0 = attn::fadd2(acc0, attn::pack2(__float_as_uint(e0), __float_as_uint(e1)));
            acc1 = attn::fadd2(acc1, attn::pack2(__float_as_uint(e2), __float_as_uint(e3)));
            const typename Pair<T>::type p01 = Pair<T>::from_f(e0, e1), p23 = Pair<T>::from_f(e2, e3);
            pw[x] = *reinterpret_cast<const uint32_t*>(&p01);
            pw[x + 1] = *reinterpret_cast<const uint32_t*>(&p23);
          }
          attn::tmem_st_32x32b_x32(ts + hf * 32, pw);
          attn::tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(hf == 0 ? &p_half[t] : &p_full[t]);
        }
        float a0, a1, a2, a3;
        attn::unpack2(acc0, a0, a1);
        attn::unpack2(acc1, a2, a3);
        l += (a0 + a1) + (a2 + a3);
      }
      if (!ok) break;
      float m = ref.m, z = 0.f;
      if (a.k_sink != nullptr && n == 0) {               // its Q is not loaded
        if (valid) {
          const T* q = reinterpret_cast<const T*>(a.q) + tok * a.ldq + (int64_t)h * HD;
#pragma unroll 1
          for (int c = 0; c < HD; ++c) z = fmaf(to_f32(q[c]), __ldg(a.k_sink + (int64_t)h * HD + c), z);
          z *= a.scale_log2;
        }
      } else if (a.k_sink != nullptr) {
        if (!warp_wait(&z_full[t], z_n++ & 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        z = s_z[t * PT_ROWS + r] * a.scale_log2;
        __syncwarp();
        if (lane == 0) mbar_arrive(&z_free[t]);
      }
      const bool whole = (b.flags & 6) == 6;
      float inv = 1.f;
      T* out = reinterpret_cast<T*>(a.o) + (tok * a.H + h) * HD;
      float4* part = reinterpret_cast<float4*>(parts + ((int64_t)blockIdx.x * 2 + (b.flags & 1 ? 0 : 1)) * prompt_part_floats(HD)) +
                     t * PT_ROWS * (HD / 4 + 1) + r;
      if (whole) {
        float f = 1.f;
        if (a.k_sink != nullptr) {
          const float mt = fmaxf(m, z);
          f = m == -INFINITY ? 0.f : attn::fast_exp2(m - mt);
          l = l * f + attn::fast_exp2(z - mt);
          m = mt;
        }
        inv = l > 0.f ? f / l : (l != l ? l : 0.f);
        if (valid) {
          inv *= gate;
          if (a.lse != nullptr)
            a.lse[tok * a.H + h] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : (l != l ? l : -INFINITY);
        }
      } else {
        part[PT_ROWS * (HD / 4)] = make_float4(m, l, z, 0.f);
      }
      if (n == 0) {                                      // no key for any row of the tile
        if (valid && whole)
          for (int c = 0; c < HD; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
        continue;
      }
      if (!warp_wait(&o_done[t], b_n & 1, s_abort, ZS_DEVERR_TIMEOUT_EPILOGUE)) {
        ok = false;
        break;
      }
      ++b_n;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(to + c * 32, o);
        tc_wait_ld();
        if (!whole) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            part[(c * 8 + x) * PT_ROWS] = make_float4(__uint_as_float(o[x * 4]), __uint_as_float(o[x * 4 + 1]),
                                                      __uint_as_float(o[x * 4 + 2]), __uint_as_float(o[x * 4 + 3]));
        } else if (valid) {
          uint4* dst = reinterpret_cast<uint4*>(out + c * 32);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float v[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) v[y] = __uint_as_float(o[x * 8 + y]) * inv;
            dst[x] = pack8<T>(v);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[t]);
    }
    if (threadIdx.x == 128) cuts[blockIdx.x] = *cut;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Block (c, query tile, 32 columns): the block that the cut behind CTA c goes through, unless an
// earlier cut does too; its parts in the order of the CTAs, a row per thread.
template <typename T, int HD>
__global__ void __launch_bounds__(PT_ROWS) paged_prompt_join_kernel(const AttnArgs a, const float* parts,
                                                                    const PromptCut* cuts, int ctas) {
  const int c = blockIdx.x, t = blockIdx.y, col = blockIdx.z * 32, r = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PromptCut cut = cuts[c];
  if (!cut.cut || (cut.single && cut.cont)) return;
  const int G = a.H / a.Hkv, tpt = PT_ROWS / G, tr = r / G;
  if (tr >= min(cut.left - t * tpt, tpt)) return;        // no row of the block
  const int h = cut.hk * G + r - tr * G;
  const int64_t tok = (int64_t)cut.tok0 + t * tpt + tr;
  float m = -INFINITY, l = 0.f, z = 0.f, acc[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) acc[e] = 0.f;
  for (int b = c, slot = cut.slot; b < ctas; ++b, slot = 0) {
    const float4* part = reinterpret_cast<const float4*>(parts + ((int64_t)b * 2 + slot) * prompt_part_floats(HD)) +
                         t * PT_ROWS * (HD / 4 + 1) + r;
    const float4 ml = part[PT_ROWS * (HD / 4)];
    float4 o[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = part[(col / 4 + x) * PT_ROWS];
    z = ml.z;
    if (ml.x != -INFINITY || ml.y != 0.f) {              // a part in which the row sees no key has no O
      const float mt = fmaxf(m, ml.x);
      const float f = m == -INFINITY ? 0.f : exp2f(m - mt), fb = ml.x == -INFINITY ? 1.f : exp2f(ml.x - mt);
      l = l * f + ml.y * fb;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        acc[x * 4] = acc[x * 4] * f + o[x].x * fb;
        acc[x * 4 + 1] = acc[x * 4 + 1] * f + o[x].y * fb;
        acc[x * 4 + 2] = acc[x * 4 + 2] * f + o[x].z * fb;
        acc[x * 4 + 3] = acc[x * 4 + 3] * f + o[x].w * fb;
      }
      m = mt;
    }
    if (b > c && !(cuts[b].cut && cuts[b].single)) break;   // it ends here
  }
  const float gate = gate_of<T>(a, tok, h);
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const float v[4] = {acc[x * 4], acc[x * 4 + 1], acc[x * 4 + 2], acc[x * 4 + 3]};
    finish_row<T, HD>(a, tok, h, col + x * 4, m, l, v, z, gate, col + x == 0);
  }
}

}  // namespace paged
}  // namespace zs

using namespace zs;

static int attn_args(paged::AttnArgs& a, const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                     int64_t page_stride, int64_t num_pages, const int* block_table, int64_t bt_ld, int max_pages,
                     const int* seq_lens, const int* cu, int num_seqs, int64_t tokens, int H, int Hkv, int hd, int page,
                     int window, float scale, const float* k_sink, const void* gate, int64_t ldg,
                     void* o, float* lse, int dtype) {
  const int rc = pages_ok(k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens, num_seqs,
                          tokens, H, Hkv, hd, page, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(q && o, ZS_ERR_ARG);
  ZS_REQUIRE(scale >= 0.f, ZS_ERR_ARG);                // the running maximum is of S, then scaled
  ZS_REQUIRE(window >= 0 && ldq >= (int64_t)H * hd && (gate == nullptr || ldg >= H), ZS_ERR_SHAPE);
  ZS_REQUIRE(ldq % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) == 0, ZS_ERR_ALIGN);
  ZS_REQUIRE((reinterpret_cast<uintptr_t>(k_sink) & 15) == 0, ZS_ERR_ALIGN);
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
  a.window = paged::window_within(window, (int64_t)max_pages * page);
  // At least the smallest normal number, which makes every finite logit next to nothing as a scale of zero does:
  // masked scores are -inf before they are scaled, and -inf * 0 is NaN.
  a.scale_log2 = fmaxf(scale * 1.4426950408889634f, 1.17549435e-38f);
  a.k_sink = k_sink;
  a.gate = gate;
  a.ldg = ldg;
  a.o = o;
  a.lse = lse;
  return ZS_OK;
}

// 3-D tensor map of 16-bit elements [n2][n1][hd] with element strides ld2 and ld1, boxes of
// box2 x box1 rows of 64 elements, 128-byte swizzle.
static int make_tmap3(CUtensorMap* m, const void* base, int dtype, int hd, int64_t n1, int64_t n2, int64_t ld1,
                      int64_t ld2, int box1, int box2) {
  auto fn = encode_fn();
  if (fn == nullptr) return ZS_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)n1, (cuuint64_t)n2};
  cuuint64_t strides[2] = {(cuuint64_t)ld1 * 2, (cuuint64_t)ld2 * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box1, (cuuint32_t)box2};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = fn(m, dtype == ZS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    zs_last_cuda_error_ref() = 100000 + (int)r;
    return ZS_ERR_CUDA;
  }
  return ZS_OK;
}

// Pages of one layer's keys or values: rows [Hkv * page] of a page, boxes of one page's rows.
static int make_page_tmap(CUtensorMap* m, const void* base, int dtype, int hd, int64_t rows, int64_t pages,
                          int64_t page_stride, int box_rows) {
  return make_tmap3(m, base, dtype, hd, rows, pages, hd, page_stride, box_rows, 1);
}

// Shared memory beyond the default for a kernel, asked for once per device.
template <auto KERNEL>
static int allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  ZS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1)) return ZS_OK;
  ZS_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return ZS_OK;
}

template <typename T, int HD>
static int launch_decode(const paged::AttnArgs& a, int dtype, void* workspace, cudaStream_t stream) {
  using L = paged::DecSmem<HD>;
  CUtensorMap tk, tv;
  const int box = a.page < L::TILE ? a.page : L::TILE;
  int rc = make_page_tmap(&tk, a.k_pages, dtype, HD, (int64_t)a.Hkv * a.page, a.num_pages, a.page_stride, box);
  if (rc != ZS_OK) return rc;
  rc = make_page_tmap(&tv, a.v_pages, dtype, HD, (int64_t)a.Hkv * a.page, a.num_pages, a.page_stride, box);
  if (rc != ZS_OK) return rc;
  // no more blocks than tiles that the table (or the window) leaves room for
  const int G = a.H / a.Hkv, units = a.Hkv * ((G + paged::DEC_ROWS - 1) / paged::DEC_ROWS);
  int64_t most = ((int64_t)a.max_pages * a.page + L::TILE - 1) / L::TILE;
  if (a.window > 0) most = min(most, ((int64_t)a.window + L::TILE - 2) / L::TILE + 1);
  const int64_t all = (most + L::OVER) * a.num_seqs * units;
  const int resident = 2 * num_sms() < paged::DEC_MAX_BLOCKS ? 2 * num_sms() : paged::DEC_MAX_BLOCKS;
  const int blocks = (int)(all < resident ? all : resident);
  float* parts = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  rc = allow_smem<paged::paged_decode_kernel<T, HD>>(L::ALLOC);
  if (rc != ZS_OK) return rc;
  paged::paged_decode_kernel<T, HD><<<blocks, 160, L::ALLOC, stream>>>(tk, tv, a, parts);
  ZS_CUDA_TRY(cudaGetLastError());
  if (most == 1) return ZS_OK;                         // nothing can be split
  return launch_after(paged::paged_join_kernel<T, HD>, dim3((unsigned)a.num_seqs, (unsigned)units),
                      dim3(paged::JOIN_WARPS * 32), stream, a, parts, blocks);
}

extern "C" size_t zs_paged_decode_workspace(int num_seqs, int H, int Hkv, int hd) {
  if (num_seqs < 0 || hd < 0 || Hkv < 1) return 0;
  return (size_t)(paged::DEC_MAX_BLOCKS * 2 * paged::part_floats(hd, paged::part_rows(H / Hkv)) * 4 + 64);
}

extern "C" int zs_paged_decode_attention(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                         int64_t page_stride, int64_t num_pages, const int* block_table,
                                         int64_t bt_ld, int max_pages, const int* seq_lens, int num_seqs, int H,
                                         int Hkv, int hd, int page, int window, float scale, const float* k_sink,
                                         const void* gate, int64_t ldg, void* o, float* lse, int dtype,
                                         void* workspace, size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  paged::AttnArgs a;
  const int rc = attn_args(a, q, ldq, k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens,
                           nullptr, num_seqs, num_seqs, H, Hkv, hd, page, window, scale, k_sink, gate, ldg,
                           o, lse, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(workspace && workspace_bytes >= zs_paged_decode_workspace(num_seqs, H, Hkv, hd), ZS_ERR_WORKSPACE);
  ZS_BIND(q);
  if (dtype == ZS_BF16)
    return hd == 128 ? launch_decode<__nv_bfloat16, 128>(a, dtype, workspace, stream)
                     : launch_decode<__nv_bfloat16, 64>(a, dtype, workspace, stream);
  return hd == 128 ? launch_decode<__half, 128>(a, dtype, workspace, stream)
                   : launch_decode<__half, 64>(a, dtype, workspace, stream);
}

// CTAs for as many steps as the packed rows and the tables leave room for.
static int prompt_ctas(int64_t tokens, int num_seqs, int H, int Hkv, int max_pages, int page, int window) {
  const int per = 2 * (paged::PT_ROWS / (H / Hkv));
  const int64_t blocks = (tokens / per + num_seqs) * Hkv;
  int64_t tiles = ((int64_t)max_pages * page + paged::PT_KEYS - 1) / paged::PT_KEYS;
  if (window > 0 && ((int64_t)window + per) / paged::PT_KEYS + 2 < tiles) tiles = ((int64_t)window + per) / paged::PT_KEYS + 2;
  int64_t want = blocks * (tiles + paged::PT_OVER) / paged::PT_LEAST;
  if (want < blocks) want = blocks;
  int sms = num_sms();
  if (sms > paged::PT_MAX_CTAS) sms = paged::PT_MAX_CTAS;
  return (int)(want < sms ? want : sms);
}

extern "C" size_t zs_paged_prompt_workspace(int64_t tokens, int num_seqs, int H, int Hkv, int hd, int max_pages,
                                            int page, int window) {
  if (tokens < 1 || num_seqs < 1 || Hkv < 1 || H / Hkv < 1 || H / Hkv > paged::PT_ROWS) return 0;
  const size_t ctas = (size_t)prompt_ctas(tokens, num_seqs, H, Hkv, max_pages, page, window);
  return ctas * (2 * paged::prompt_part_floats(hd) * 4 + sizeof(paged::PromptCut)) + 512;
}

template <typename T, int HD>
static int launch_prompt(const paged::AttnArgs& a, int dtype, void* workspace, cudaStream_t stream) {
  using L = paged::PromptSmem<HD>;
  const int G = a.H / a.Hkv, tpt = paged::PT_ROWS / G, box = a.page < paged::PT_KEYS ? a.page : paged::PT_KEYS;
  CUtensorMap tq, tk, tv;
  int rc = make_tmap3(&tq, a.q, dtype, HD, a.H, a.tokens, HD, a.ldq, G, tpt);
  if (rc != ZS_OK) return rc;
  rc = make_page_tmap(&tk, a.k_pages, dtype, HD, (int64_t)a.Hkv * a.page, a.num_pages, a.page_stride, box);
  if (rc != ZS_OK) return rc;
  rc = make_page_tmap(&tv, a.v_pages, dtype, HD, (int64_t)a.Hkv * a.page, a.num_pages, a.page_stride, box);
  if (rc != ZS_OK) return rc;
  const int grid = prompt_ctas(a.tokens, a.num_seqs, a.H, a.Hkv, a.max_pages, a.page, a.window);
  float* parts = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  paged::PromptCut* cuts = reinterpret_cast<paged::PromptCut*>(parts + grid * 2 * paged::prompt_part_floats(HD));
  rc = allow_smem<paged::paged_prompt_kernel<T, HD>>(L::ALLOC);
  if (rc != ZS_OK) return rc;
  paged::paged_prompt_kernel<T, HD><<<grid, paged::PT_THREADS, L::ALLOC, stream>>>(tq, tk, tv, a, parts, cuts);
  ZS_CUDA_TRY(cudaGetLastError());
  if (grid > 1 && (int64_t)a.max_pages * a.page > paged::PT_KEYS)      // else no block has a second tile to cut at
    return launch_after(paged::paged_prompt_join_kernel<T, HD>, dim3(grid - 1, 2, HD / 32), dim3(paged::PT_ROWS), stream, a,
                        parts, cuts, grid);
  return ZS_OK;
}

extern "C" int zs_paged_prompt_attention(const void* q, int64_t ldq, const void* k_pages, const void* v_pages,
                                         int64_t page_stride, int64_t num_pages, const int* block_table,
                                         int64_t bt_ld, int max_pages, const int* seq_lens, const int* cu_seqlens,
                                         int num_seqs, int64_t tokens, int H, int Hkv, int hd, int page, int window,
                                         float scale, const float* k_sink, const void* gate,
                                         int64_t ldg, void* o, float* lse, int dtype, void* workspace,
                                         size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  ZS_REQUIRE(cu_seqlens, ZS_ERR_ARG);
  paged::AttnArgs a;
  const int rc = attn_args(a, q, ldq, k_pages, v_pages, page_stride, num_pages, block_table, bt_ld, max_pages, seq_lens,
                           cu_seqlens, num_seqs, tokens, H, Hkv, hd, page, window, scale, k_sink, gate,
                           ldg, o, lse, dtype);
  if (rc != ZS_OK) return rc;
  ZS_REQUIRE(H / Hkv <= paged::PT_ROWS, ZS_ERR_SHAPE);
  ZS_REQUIRE(workspace, ZS_ERR_WORKSPACE);
  ZS_BIND(q);
  ZS_REQUIRE(workspace_bytes >= zs_paged_prompt_workspace(tokens, num_seqs, H, Hkv, hd, max_pages, page, window),
             ZS_ERR_WORKSPACE);
  if (dtype == ZS_BF16)
    return hd == 128 ? launch_prompt<__nv_bfloat16, 128>(a, dtype, workspace, stream)
                     : launch_prompt<__nv_bfloat16, 64>(a, dtype, workspace, stream);
  return hd == 128 ? launch_prompt<__half, 128>(a, dtype, workspace, stream) : launch_prompt<__half, 64>(a, dtype, workspace, stream);
}
