// Attention of a chunk of new tokens over a paged cache (8-bit or bf16 pages) and
// over itself, bidirectional, causal or causal between blocks.
//
// Segment s has n cached rows in pages and L new rows whose K / V are
// given in bf16.  New row t sees every cached row and the new rows j < vis(t):
//   vis(t) = L                                  mask_block = 0
//   vis(t) = min(L, ((n + t) / b + 1) * b - n)  mask_block = b >= 1 (1: causal)
// so only tiles of new rows ever need a mask that differs from row to row.
//
// "M rows" pack the g = Hq / Hkv query heads of a KV head: M row m is token m / g,
// head hkv * g + m % g; every K / V byte that is read serves all of them.
//
//   * chunk_rows_kernel (few M rows: single tokens, blocks): each of a workgroup's
//     four or eight wavefronts takes 32-key tiles of its own, by DMA into its own LDS.  No
//     wavefront waits for another until the states are merged at the end.
//   * chunk_tile_kernel (many M rows: pieces of prompts): 64-key tiles of K and V in LDS,
//     in bf16, shared by the workgroup's wavefronts of 32 M rows each; 8-bit rows are
//     converted once, on their way into LDS.
//   * long key ranges are split over workgroups; chunk_combine_kernel joins the parts.
#include "attn_tile.h"
#include "quant.h"

#include <algorithm>
#include <type_traits>

namespace dllm {

struct ChunkArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const uint8_t* kc;      // cache: records (8-bit) or bf16 rows [pages * 256][Hkv][128]
  const uint8_t* vc;
  float* ws;
  int64_t q_stride, k_stride, v_stride, o_stride;
  int64_t cache_rows;     // rows of the cache, whole pages
  int max_q, max_cached;
  int g;
  int mask_block;
  float scale_log2;
};

constexpr int kTileKeys = 32;   // keys of a wavefront's tile (chunk_rows_kernel)
constexpr int kBigTile = 64;    // keys of a workgroup's tile (chunk_tile_kernel)
constexpr int kMaxSplitTiles = 62 * kPageRows / kTileKeys;  // chunk_rows_kernel: at most 63 pages, one a lane
constexpr int64_t kMaxParts = (int64_t)1 << 30;             // bytes of parts (workspace) in a launch
constexpr int64_t kMaxBlocks = (int64_t)1 << 22;            // workgroups of a launch: 2^32 threads is HIP's limit

// A segment: new rows' first row and count, cached rows.
struct Segment {
  int row0, len, cached;
};

// New rows that new row t sees.  With r = n % b, the end of t's block is
// ((r + t) / b + 1) b - r: divisions of 32 bits (one of 64 is over a hundred
// instructions, and every wavefront starts with some).
__device__ __forceinline__ int visible(const Segment& g, int t, int mask_block) {
  if (mask_block == 0) return g.len;
  if (mask_block == 1) return min(g.len, t + 1);
  const uint32_t b = (uint32_t)mask_block, r = (uint32_t)g.cached % b;
  const uint32_t blocks = (r + (uint32_t)t) / b + 1;  // r < 2^31, t < 2^30
  return (int)min((uint64_t)g.len, (uint64_t)blocks * b - r);
}

// Splits that hold keys of the M tile whose last token is `last` (at least one).  The
// rows form deals the cached tiles alone, the new rows belonging to the last split; the
// tile form the cached tiles and those of the new rows that the M tile sees.
template <bool TILE>
__device__ __forceinline__ int splits_of(const ChunkArgs& a, int max_split, int tiles_per_split, const Segment& g,
                                         int last) {
  if (max_split == 1) return 1;
  int tiles;
  if (TILE)
    tiles = (g.cached + kBigTile - 1) / kBigTile + (visible(g, last, a.mask_block) + kBigTile - 1) / kBigTile;
  else
    tiles = (g.cached + kTileKeys - 1) / kTileKeys;
  return max(1, (int)((uint32_t)(tiles + tiles_per_split - 1) / (uint32_t)tiles_per_split));
}

// The tables and the launch's geometry come as leading scalar arguments (14 dwords): the
// library is built with kernel argument preloading, so they are in SGPRs when a wave
// starts instead of a load away -- a load that queues behind the keys that
// workgroups which started earlier are already streaming.
#define CHUNK_PARAMS                                                                                            \
  const int32_t *__restrict__ cu, const int32_t *__restrict__ seg_ids, const int32_t *__restrict__ lens,       \
      const int32_t *__restrict__ table, int chunk_pages, int logical_blocks, int mtiles, int max_split,       \
      int tiles_per_split, int Hkv, ChunkArgs a
// chunk_pages: the XCD interleave's chunk (1 .. 4) + 16 x whether the splits turn (work_of) +
// 32 x the page table's row length.

// A workgroup's work: one M tile and split of one (segment, KV head), M tiles fastest.
// Every segment has max_split splits; those past its end stop at once.
// (Numbering only the work that exists, by a prefix sum over the segments in every
// workgroup, made the first loads wait for another one: 32 ragged single tokens, 28/4
// heads, 25.4 -> 26 to 30 us.)
struct Work {
  int s, hkv, split, mt;
};
// r % n, and r / n left in r; a division is some twenty instructions at the start of
// every wavefront, and n is often one.
__device__ __forceinline__ int take(uint32_t& r, int n) {
  if (n == 1) return 0;
  const uint32_t x = r, q = x / (uint32_t)n;
  r = q;
  return (int)(x - q * (uint32_t)n);
}
// Workgroup L runs on XCD L % 8 and there on shader engine L / 8 % 4.  Of sequences with
// very different lengths most have only their first splits: with max_split a multiple of
// 32 those of all sequences would meet on one engine.  `turn`: split 0 of group (segment, KV
// head) i stands i / P places later, modulo max_split, P groups being what it takes for
// i * max_split to come back to the same engine.  (16 x 8 rows behind 100 - 8000, 28/4
// heads, 16 parts: 52.9 -> 30.6 us; 8 tokens behind 64 - 4000, 32 heads, 4 parts 34.2 -> 23.7.  Where
// all splits exist it is 1 - 3 % slower: one token behind 131071 27.2 and 27.7.)
__device__ __forceinline__ Work work_of(int L, int mtiles, int max_split, int Hkv, bool turn) {
  Work w;
  uint32_t r = (uint32_t)L;
  w.mt = take(r, mtiles);
  w.split = take(r, max_split);
  if (turn) {
    uint32_t t = r >> (5 - min(5, __builtin_ctz((uint32_t)max_split)));
    w.split -= take(t, max_split);
    if (w.split < 0) w.split += max_split;
  }
  w.hkv = take(r, Hkv);
  w.s = (int)r;
  return w;
}
// The place of a workgroup's part: M tiles fastest, then splits, KV heads, segments.
__device__ __forceinline__ int part_of(const Work& w, int mtiles, int max_split, int Hkv) {
  return ((w.s * Hkv + w.hkv) * max_split + w.split) * mtiles + w.mt;
}
__device__ __forceinline__ int block_of(int chunk_pages) {
  const int chunk = chunk_pages & 15;
  return chunk == 1 ? (int)blockIdx.x : xcd_remap(blockIdx.x, chunk);
}
// Token of M row m (m >= 0).
__device__ __forceinline__ int token_of(int m, int g) { return (int)((uint32_t)m / (uint32_t)g); }
// The M tile of a workgroup of the tile form.  The last M tiles, which see the most keys
// under a causal mask, come first, but first and last in turn from one 256 workgroups (one
// a CU) to the next, so that a CU's workgroups come out even: 8192 new rows, 32 heads,
// 819 -> 678 us.  Splits, which are even by themselves, leave the order alone.
__device__ __forceinline__ int tile_of(const Work& w, int L, int mtiles, int max_split) {
  return max_split == 1 && ((L - w.mt) >> 8 & 1) ? w.mt : mtiles - 1 - w.mt;
}
__device__ __forceinline__ Segment segment(const ChunkArgs& a, const int32_t* cu, const int32_t* seg_ids,
                                           const int32_t* lens, int s) {
  Segment g;
  const int id = seg_ids ? seg_ids[s] : s;
  int c0 = cu[id], c1 = cu[id + 1], n = lens[s];
  // These and the arguments are waited for once: loaded where they are first used, they
  // would make a chain of four loads at the start of every workgroup.  (This, the short
  // divisions and the waits below: one token behind 32 rows 5.85 -> 4.7 us, behind 511 10.1
  // -> 8.6, 32 ragged ones, 28/4 heads, 25.0 -> 22.7.)
  asm volatile(""
               : "+s"(c0), "+s"(c1), "+s"(n)
               : "s"(a.q), "s"(a.k), "s"(a.v), "s"(a.o), "s"(a.kc), "s"(a.vc), "s"(a.ws), "s"(a.q_stride),
                 "s"(a.k_stride), "s"(a.v_stride), "s"(a.o_stride), "s"(a.cache_rows));
  g.row0 = c0;
  // no more than the launch was sized for
  g.len = min(max(c1 - c0, 0), a.max_q);
  g.cached = min(max(n, 0), a.max_cached);
  return g;
}

// The part of M row `row` (of BM) of workgroup L: 128 floats, and the row's m and l
// behind all parts.
template <int BM>
__device__ __forceinline__ float* part_o(const ChunkArgs& a, int L, int row) {
  return a.ws + ((int64_t)L * BM + row) * HD;
}
template <int BM>
__device__ __forceinline__ float* part_ml(const ChunkArgs& a, int logical_blocks, int L, int row) {
  return a.ws + (int64_t)logical_blocks * BM * HD + ((int64_t)L * BM + row) * 2;
}

__device__ __forceinline__ float row_max4(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  x = pair_max32(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float row_sum4(float x) {
  x = pair_sum32(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// ---------------------------------------------------------------------------
// Few M rows.  Per wavefront and 32-key tile, with 16x16x32 MFMAs:
//   S^T[16 keys x 16 rows] = K . Q^T   two key halves u, four steps of 32 d each
//   O^T[16 d x 16 rows]   += V^T . P^T eight d blocks, one step of 32 keys
// Lane (c = l % 16, g4 = l / 16) holds K row 16 u + c and, in the results, M row c:
// scores of keys 16 u + 4 g4 + i, outputs d = 16 dt + 4 g4 + i.  A contraction does
// not depend on the order of its index, so the four lanes of a K row each take
// whole 16-byte pieces of it (8-bit: piece p covers d = 64 p + 16 g4 .. + 15, two
// steps; bf16: step s covers d = 32 s + 8 g4 .. + 7), Q^T is loaded in the same
// order, and P^T is fed to the second product as it stands: its index (g4, i) is
// key 4 g4 + i for i < 4 and 16 + 4 g4 + i - 4 otherwise, which V^T follows.
//
// K and V come by DMA into two stages of the wavefront's own LDS, as they are (8-bit
// rows with their scale bytes), so that two tiles -- 16 KiB in 8 bits -- are in flight
// without registers, and no wavefront waits for another.  8-bit codes become bf16
// on their way from LDS into the operands: K with its row's scale, which is part of
// the conversion; V^T, whose operand holds eight keys of one d
// (ds_read_b64_tr_b8: in a group of 16 lanes lane 2k + h supplies bytes 8 h .. 8 h + 7
// of row k of an 8 x 16 block and lane n receives column n), without: the powers of two
// are multiplied onto P instead, which commutes with its rounding (a V row of 2^127 may
// overflow there where only its larger elements would in f32).
//
// Bound by memory where workgroups fill the card (one token behind 131071, 28/4 heads: 23.8
// us, 5.7 TB/s; 16 ragged tokens over bf16 pages, 32 heads: 133 us, 6.0 TB/s), by what a
// CU takes in where there is one a CU (8 x 32 rows behind 608 - 1216, 32 heads, 18 us), by
// the chain start - lengths - first tile - turns - merge where there are few keys.
//
// Chunks of 16 bytes are XOR-swizzled inside a row, so that the lanes of a read phase
// fall on different banks:
//   8-bit K, V [32][128 B]  chunk ^ (row / 2 & 7) ^ 4 (row / 16)
//   bf16 K [32][256 B]      chunk ^ (row & 15)
//   bf16 V [32][256 B]      chunk ^ 2 (row & 7)
template <bool FP8>
struct RowsTile {
  static constexpr int kRow = FP8 ? kQuantD : 2 * HD;
  static constexpr int kV = kTileKeys * kRow;      // offset of V in a stage
  static constexpr int kScales = 2 * kV;           // K's 32 scale bytes, then V's
  static constexpr int kStage = FP8 ? kScales + 256 : kScales;
  static constexpr int kDma = kV / 1024;           // instructions of one matrix
  static constexpr int kOps = 2 * kDma + (FP8 ? 1 : 0);
};

// Floats of a wavefront's parked O (rows of 128 + 4, which spreads them over the
// banks), and bytes of a workgroup's LDS: the stages, later the parked O, m and l.
constexpr int park_floats(int nb) { return 16 * nb * 132; }
template <int NB, bool FP8, int NW>
constexpr int rows_lds() {
  constexpr int stages = NW * 2 * RowsTile<FP8>::kStage, park = NW * (park_floats(NB) + 2 * 16 * NB) * 4;
  return stages > park ? stages : park;
}

template <int NB>
struct RowState {
  f32x4_t o[NB][8];
  float m[NB], l[NB];  // reference maximum (log2 domain), this lane's part of the row sum
};

template <int NB>
__device__ __forceinline__ void rows_init(RowState<NB>& st) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int t = 0; t < 8; ++t) st.o[b][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    st.m[b] = -INFINITY;
    st.l[b] = 0.f;
  }
}

// Online softmax of one 32-key tile of one row block; p, times the keys' V scales
// where SCALED, comes back as the B operand.
template <bool SCALED>
__device__ __forceinline__ bf16x8_t rows_softmax(const f32x4_t (&s)[2], f32x4_t (&o)[8], float& m, float& l, float c,
                                                 const float (&vs)[8]) {
  float mx = s[0][0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
  mx = row_max4(mx) * c;
  const bool need = mx > m + kLazy;  // m = -inf: any finite score
  if (__builtin_amdgcn_ballot_w64(need)) {
    const float mn = need ? mx : m;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= alpha;
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] *= alpha;
    m = mn;
  }
  const float neg = m == -INFINITY ? 0.f : -m;
  u32x4_t pk;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w >> 1][(2 * w) & 3], c, neg));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w >> 1][(2 * w + 1) & 3], c, neg));
    const uint32_t r = cvt_pk_bf16(p0, p1);
    l = add_bf16x2(r, l);  // the rounded numerators, as the product uses them
    pk[w] = SCALED ? cvt_pk_bf16(p0 * vs[2 * w], p1 * vs[2 * w + 1]) : r;
  }
  return as_bf16x8(pk);
}

// NaN or infinity among eight bf16 values; the same values with those as zeros.
__device__ __forceinline__ bool has_nonfinite(u32x4_t x) {
  bool r = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) r |= (x[w] & 0x7f80u) == 0x7f80u || (x[w] & 0x7f800000u) == 0x7f800000u;
  return r;
}
__device__ __forceinline__ u32x4_t finite_part(u32x4_t x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if ((x[w] & 0x7f80u) == 0x7f80u) x[w] &= 0xffff0000u;
    if ((x[w] & 0x7f800000u) == 0x7f800000u) x[w] &= 0xffffu;
  }
  return x;
}

// LDS of one wavefront is read by other lanes than wrote it: nothing may move across.
__device__ __forceinline__ void wave_lds_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// The V^T codes of a tile, eight d blocks (one asm block with its own wait: the
// builtin would wait for the DMA of the next tiles as well).  vb: this lane's address
// for block 0; block dt is at vb ^ 16 dt.
__device__ __forceinline__ void v_codes(const uint8_t* vb_ptr, u32x2_t (&r)[8]) {
  const uint32_t vb = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)vb_ptr;
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8\n"
      "ds_read_b64_tr_b8 %1, %9\n"
      "ds_read_b64_tr_b8 %2, %10\n"
      "ds_read_b64_tr_b8 %3, %11\n"
      "ds_read_b64_tr_b8 %4, %12\n"
      "ds_read_b64_tr_b8 %5, %13\n"
      "ds_read_b64_tr_b8 %6, %14\n"
      "ds_read_b64_tr_b8 %7, %15\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(vb), "v"(vb ^ 16u), "v"(vb ^ 32u), "v"(vb ^ 48u), "v"(vb ^ 64u), "v"(vb ^ 80u), "v"(vb ^ 96u), "v"(vb ^ 112u)
      : "memory");
}
// The same for bf16 rows: blocks at vb ^ 32 dt, keys 16 .. 31 4 KiB further; output 2 dt + half.
__device__ __forceinline__ void v_rows(const uint8_t* vb_ptr, u32x2_t (&r)[16]) {
  const uint32_t vb = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)vb_ptr;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n"
      "ds_read_b64_tr_b16 %1, %16 offset:4096\n"
      "ds_read_b64_tr_b16 %2, %17\n"
      "ds_read_b64_tr_b16 %3, %17 offset:4096\n"
      "ds_read_b64_tr_b16 %4, %18\n"
      "ds_read_b64_tr_b16 %5, %18 offset:4096\n"
      "ds_read_b64_tr_b16 %6, %19\n"
      "ds_read_b64_tr_b16 %7, %19 offset:4096\n"
      "ds_read_b64_tr_b16 %8, %20\n"
      "ds_read_b64_tr_b16 %9, %20 offset:4096\n"
      "ds_read_b64_tr_b16 %10, %21\n"
      "ds_read_b64_tr_b16 %11, %21 offset:4096\n"
      "ds_read_b64_tr_b16 %12, %22\n"
      "ds_read_b64_tr_b16 %13, %22 offset:4096\n"
      "ds_read_b64_tr_b16 %14, %23\n"
      "ds_read_b64_tr_b16 %15, %23 offset:4096\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
      : "v"(vb), "v"(vb ^ 32u), "v"(vb ^ 64u), "v"(vb ^ 96u), "v"(vb ^ 128u), "v"(vb ^ 160u), "v"(vb ^ 192u), "v"(vb ^ 224u)
      : "memory");
}

// NW: wavefronts.  ONE: one M tile, so nothing else reads the keys and the loads are streaming ones (64
// tokens behind 2000, 32 heads: 192 -> 171 us; with seven M tiles, 16 x 32 rows, 28/4
// heads, they take 21.2, ordinary ones 19.8).
template <int NB, bool FP8, bool ONE, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_rows_kernel(CHUNK_PARAMS) {
  constexpr int AUX = ONE ? kStreamAux : 0;
  using T = RowsTile<FP8>;
  constexpr int BM = 16 * NB;
  constexpr int PARK = park_floats(NB);
  extern __shared__ __attribute__((aligned(16))) float lds[];  // rows_lds() bytes
  const int L = block_of(chunk_pages);
  if (L >= logical_blocks) return;
  const int max_pages = chunk_pages >> 5;
  const Work wk = work_of(L, mtiles, max_split, Hkv, chunk_pages & 16);
  const int s = wk.s, hkv = wk.hkv, split = wk.split;
  const int lane = threadIdx.x & 63;
  const int t_begin = split * tiles_per_split;
  // Page ids of the split, one a lane (a split spans at most 63): a tile's loads
  // then wait for no load of their own.  Their address needs no other load either.
  const int pg0 = t_begin * kTileKeys / kPageRows;
  int page_reg = max_pages > 0 ? table[(int64_t)s * max_pages + min(pg0 + lane, max_pages - 1)] : -1;
  const Segment sg = segment(a, cu, seg_ids, lens, s);
  const uint32_t n_pages = (uint32_t)min(a.cache_rows >> 8, (int64_t)1 << 23);
  const int g = a.g;
  const int M = sg.len * g;
  const int m_base = wk.mt * BM;
  if (m_base >= M) return;
  const int ns = splits_of<false>(a, max_split, tiles_per_split, sg, sg.len - 1);
  if (split >= ns) return;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  uint8_t* const my = reinterpret_cast<uint8_t*>(lds) + wave * 2 * T::kStage;

  const int tiles = (sg.cached + kTileKeys - 1) / kTileKeys;
  const int t_end = n_pages ? min(tiles, t_begin + tiles_per_split) : t_begin;  // no cache: nothing to read
  const uint32_t bf_row = (uint32_t)(Hkv * HD * 2);

  // The page ids, sent for first, have arrived when the lengths have.  Waited for here,
  // alone: at their first use the compiler would wait for all that is in flight by then.
  asm volatile("" : "+v"(page_reg));

  // ---- Q^T operands and the rows' limits ------------------------------------
  bf16x8_t qf[NB][4];
  int lim[NB];  // new rows that M row m_base + 16 b + col sees
  {
    const uint32_t qS = (uint32_t)(a.q_stride * 2);
    const uint32_t qbytes = (uint32_t)sg.len * qS;
    const __amdgpu_buffer_rsrc_t qrs = make_rsrc(a.q + (int64_t)sg.row0 * a.q_stride, qbytes);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int m = m_base + 16 * b + col;
      const int tok = token_of(m, g);
      lim[b] = visible(sg, min(tok, sg.len - 1), a.mask_block);
      const uint32_t base = m < M ? (uint32_t)tok * qS + (uint32_t)((hkv * g + m - tok * g) * HD) * 2u : qbytes;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const uint32_t off = FP8 ? (uint32_t)((st >> 1) * 128 + g4 * 32 + (st & 1) * 16) : (uint32_t)(st * 64 + g4 * 16);
        qf[b][st] = as_bf16x8(bload(qrs, base == qbytes ? qbytes : base + off, 0u));
      }
    }
  }

  // page of tile t, or -1: outside the cache, its rows are left out
  auto page_of = [&](int t) -> int {
    const int pg = t * kTileKeys / kPageRows;
    const int pid = __builtin_amdgcn_readlane(page_reg, (pg - pg0) & 63);
    return pg < max_pages && (uint32_t)pid < n_pages ? pid : -1;
  };
  // DMA of cached tile t into a stage; rows past the cached length, and all rows of a
  // page outside the cache, arrive as zeros through the buffer's bound.
  auto issue = [&](uint8_t* stage, int t, bool exists = true) {
    const int pid = page_of(t);
    const int row0 = t * kTileKeys & (kPageRows - 1);
    const int rows = pid < 0 || !exists ? 0 : min(sg.cached - t * kTileKeys, kTileKeys);
    if constexpr (FP8) {
      const int64_t rec = ((int64_t)max(pid, 0) * Hkv + hkv) * kRecord;
      const __amdgpu_buffer_rsrc_t krs = make_rsrc(a.kc + rec + row0 * kQuantD, (uint32_t)rows * kQuantD);
      const __amdgpu_buffer_rsrc_t vrs = make_rsrc(a.vc + rec + row0 * kQuantD, (uint32_t)rows * kQuantD);
      // lane l of instruction j: row 8 j + l / 8, physical chunk l % 8
      const uint32_t row = (uint32_t)((lane >> 3) * kQuantD), ch = (uint32_t)((lane & 7) ^ (lane >> 4)) * 16;
#pragma unroll
      for (int j = 0; j < T::kDma; ++j) {
        const uint32_t off = (uint32_t)(j * 1024) + row + (ch ^ (uint32_t)(j == 1 || j == 2 ? 64 : 0));
        dma16<AUX>(krs, stage + j * 1024, off);
        dma16<AUX>(vrs, stage + T::kV + j * 1024, off);
      }
      // lanes 0 .. 7: K's scale bytes, 8 .. 15: V's (the others repeat them)
      const uint8_t* sp = (lane & 8 ? a.vc : a.kc) + rec + kScaleOff + row0 + (lane & 7) * 4;
      // (in asm: after the builtin, which the compiler takes for an access that ends out of
      // order, it waits for all that is in flight wherever it waits for anything.  A write of
      // m0 is one wait state ahead of its use by such a load.)
      const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)(stage + T::kScales);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                   :
                   : "s"(to), "v"(sp)
                   : "m0", "memory");
    } else {
      const int64_t off0 = ((int64_t)max(pid, 0) * kPageRows + row0) * bf_row + hkv * HD * 2;
      const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * bf_row + HD * 2 : 0u;
      const __amdgpu_buffer_rsrc_t krs = make_rsrc(a.kc + off0, bytes), vrs = make_rsrc(a.vc + off0, bytes);
#pragma unroll
      for (int j = 0; j < T::kDma; ++j) {  // lane l: row 4 j + l / 16, physical chunk l % 16
        const int row = 4 * j + g4;
        dma16<AUX>(krs, stage + j * 1024, (uint32_t)row * bf_row + (uint32_t)((col ^ (row & 15)) * 16));
        dma16<AUX>(vrs, stage + T::kV + j * 1024, (uint32_t)row * bf_row + (uint32_t)((col ^ (2 * (row & 7))) * 16));
      }
    }
  };

  RowState<NB> st;
  rows_init(st);
  const float c = a.scale_log2;
  // this lane's transposing reads: bf16 rows, row 4 g4 + col / 4, chunk (col & 3) / 2 of a
  // 32-byte block; 8-bit rows, row 4 g4 + k or 16 + 4 g4 + k - 4 with k = col / 2, half col & 1
  const int row16 = 4 * g4 + (col >> 2);
  const uint32_t vb16 = (uint32_t)(row16 * 256 + ((((col & 3) >> 1) ^ (2 * (row16 & 7))) * 16) + 8 * (col & 1));
  const int k8 = col >> 1, row8 = k8 < 4 ? 4 * g4 + k8 : 12 + 4 * g4 + k8;
  const uint32_t vb8 = (uint32_t)(row8 * 128 + ((((row8 >> 1) & 7) ^ (4 * (row8 >> 4))) * 16) + 8 * (col & 1));

  // S^T of a tile whose K fragments of half u are keys(u, .), hide() its keys, softmax.
  auto scores = [&](auto&& keys, auto&& hide, const float (&vs)[8], auto scaled, bf16x8_t (&pf)[NB]) {
    f32x4_t sc[NB][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      bf16x8_t kf[4];
      keys(u, kf);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        sc[b][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4)
          sc[b][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[k4], qf[b][k4], sc[b][u], 0, 0, 0);
      }
    }
    hide(sc);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      pf[b] = rows_softmax<decltype(scaled)::value>(sc[b], st.o[b], st.m[b], st.l[b], c, vs);
  };
  auto add_bf16_rows = [&](const uint8_t* vtile, const bf16x8_t (&pf)[NB]) {
    u32x2_t x[16];
    v_rows(vtile + vb16, x);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        st.o[b][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            as_bf16x8(u32x4_t{x[2 * dt][0], x[2 * dt][1], x[2 * dt + 1][0], x[2 * dt + 1][1]}), pf[b], st.o[b][dt], 0, 0, 0);
  };

  auto compute_tile = [&](const uint8_t* stage, int t) {
    const int left = page_of(t) < 0 ? 0 : sg.cached - t * kTileKeys;
    const uint32_t bad = left >= kTileKeys ? 0u : ~0u << left;  // keys to leave out
    u32x4_t kx[2][FP8 ? 2 : 4];
    float ks[2] = {0.f, 0.f}, vs[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (FP8) {
        const uint32_t sw = (uint32_t)(((col >> 1) & 7) ^ (4 * u));
#pragma unroll
        for (int p = 0; p < 2; ++p)
          kx[u][p] = *reinterpret_cast<const u32x4_t*>(stage + (16 * u + col) * 128 + (((4 * p + g4) ^ sw) * 16));
        ks[u] = scale_of(stage[T::kScales + 16 * u + col]);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(stage + T::kScales + 32 + 16 * u + 4 * g4);
        vs[4 * u] = __uint_as_float((w << 23) & 0x7f800000u);
        vs[4 * u + 1] = __uint_as_float((w << 15) & 0x7f800000u);
        vs[4 * u + 2] = __uint_as_float((w << 7) & 0x7f800000u);
        vs[4 * u + 3] = __uint_as_float((w >> 1) & 0x7f800000u);
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p)
          kx[u][p] = *reinterpret_cast<const u32x4_t*>(stage + (16 * u + col) * 256 + (((4 * p + g4) ^ col) * 16));
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[4 * u + i] = 1.f;
      }
    }
    auto keys = [&](int u, bf16x8_t (&kf)[4]) {
#pragma unroll
      for (int p = 0; p < (FP8 ? 2 : 4); ++p) {
        if constexpr (FP8) {
          kf[2 * p] = as_bf16x8(dequant8(u32x2_t{kx[u][p][0], kx[u][p][1]}, ks[u]));
          kf[2 * p + 1] = as_bf16x8(dequant8(u32x2_t{kx[u][p][2], kx[u][p][3]}, ks[u]));
        } else {
          kf[p] = as_bf16x8(kx[u][p]);
        }
      }
    };
    auto hide = [&](f32x4_t (&sc)[NB][2]) {
      if (bad) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((bad >> (16 * u + 4 * g4 + i)) & 1u) {
#pragma unroll
              for (int b = 0; b < NB; ++b) sc[b][u][i] = -INFINITY;
              vs[4 * u + i] = 0.f;  // the scale byte of a row that does not exist may be anything
            }
      }
    };
    bf16x8_t pf[NB];
    scores(keys, hide, vs, std::integral_constant<bool, FP8>(), pf);
    if constexpr (FP8) {
      u32x2_t x[8];
      v_codes(stage + T::kV + vb8, x);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const bf16x8_t af = as_bf16x8(dequant8(x[dt], 1.f));
#pragma unroll
        for (int b = 0; b < NB; ++b)
          st.o[b][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, pf[b], st.o[b][dt], 0, 0, 0);
      }
    } else {
      add_bf16_rows(stage + T::kV, pf);
    }
  };

  // ---- new rows (the last split's), bf16 from k / v ------------------------------
  // Before the cached tiles: their loads are among the first, beside the first tile's DMA.
  const int n = max(0, (t_end - t_begin - wave + NW - 1) / NW);  // this wavefront's cached tiles
  const int first = t_begin + wave;
  bool fixed = false;
  const uint32_t vS = (uint32_t)(a.v_stride * 2), vb = (uint32_t)(sg.len - 1) * vS + HD * 2;
  const __amdgpu_buffer_rsrc_t vrs = make_rsrc(a.v + (int64_t)sg.row0 * a.v_stride + hkv * HD, vb);
  const int turn = max(t_end - t_begin, 0);
  if (n > 0) issue(my, first);
  if (split == ns - 1) {
    const uint32_t kS = (uint32_t)(a.k_stride * 2), kb = (uint32_t)(sg.len - 1) * kS + HD * 2;
    const __amdgpu_buffer_rsrc_t krs = make_rsrc(a.k + (int64_t)sg.row0 * a.k_stride + hkv * HD, kb);
    // the furthest new row that any of this workgroup's rows sees
    const int last = min(m_base + BM, M) - 1;
    const int see = visible(sg, token_of(last, g), a.mask_block);
    const int new_tiles = (see + kTileKeys - 1) / kTileKeys;
    for (int t = (wave - turn) & (NW - 1); t < new_tiles; t += NW) {
      bf16x8_t kx[2][4];
      u32x4_t vx[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // rows that do not exist start past the bound and arrive as zeros
        const uint32_t row = (uint32_t)min(t * kTileKeys + 16 * u + col, sg.len);
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const uint32_t off = FP8 ? (uint32_t)((k4 >> 1) * 128 + g4 * 32 + (k4 & 1) * 16) : (uint32_t)(k4 * 64 + g4 * 16);
          kx[u][k4] = as_bf16x8(bload(krs, row * kS + off, 0u));
          vx[u][k4] = bload(vrs, row * vS + (uint32_t)(k4 * 64 + g4 * 16), 0u);
        }
      }
      // A NaN or infinity in a V row that some M row does not see would reach that row
      // as 0 * V.  Such elements (rare) are multiplied as zeros and added at the end
      // to the rows that see them.
      bool odd = false;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int p = 0; p < 4; ++p) odd |= has_nonfinite(vx[u][p]);
      const bool fix = __builtin_amdgcn_ballot_w64(odd) != 0;
      if (fix) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int p = 0; p < 4; ++p) vx[u][p] = finite_part(vx[u][p]);
      }
      // V in bf16, as a tile of bf16 rows, where the second stage will be
      wave_lds_fence();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int row = 16 * u + col;
          *reinterpret_cast<u32x4_t*>(my + T::kStage + row * 256 + (((4 * p + g4) ^ (2 * (row & 7))) * 16)) = vx[u][p];
        }
      wave_lds_fence();
      auto keys = [&](int u, bf16x8_t (&kf)[4]) {
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) kf[k4] = kx[u][k4];
      };
      auto hide = [&](f32x4_t (&sc)[NB][2]) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (t * kTileKeys + 16 * u + 4 * g4 + i >= lim[b]) sc[b][u][i] = -INFINITY;
      };
      const float one[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
      bf16x8_t pf[NB];
      scores(keys, hide, one, std::false_type(), pf);
      add_bf16_rows(my + T::kStage, pf);
      fixed |= fix;
    }
  }

  // ---- cached tiles: this wavefront takes every NW-th, two in flight ----------------
  if (n > 0) {
    wave_lds_fence();  // the new rows' V has been read
    issue(my + T::kStage, first + NW, n > 1);  // no second tile: as many operations, all zeros
    // Q has landed, both tiles may be in flight.  (Where the compiler has to join paths with
    // different operations, it waits for the tiles as well.)
    vm_wait<2 * T::kOps>();
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) asm volatile("" : "+v"(qf[b][k4]));
    for (int i = 0; i < n; ++i) {
      if (i + 1 < n)
        vm_wait<T::kOps>();
      else
        vm_wait<0>();
      uint8_t* const stage = my + (i & 1) * T::kStage;
      compute_tile(stage, first + NW * i);
      wave_lds_fence();  // the tile's reads end before its stage is filled again
      if (i + 2 < n) issue(stage, first + NW * (i + 2));
    }
  }

  if (fixed) {
#pragma unroll 1
    for (int j = 0; j < sg.len; ++j) {
      if ((((j / kTileKeys) + turn - wave) & (NW - 1)) != 0) continue;  // a key of another wavefront
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const u32x2_t w = __builtin_bit_cast(
            u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(vrs, (int)((uint32_t)j * vS + (uint32_t)(32 * dt + 8 * g4)), 0, 0));
#pragma unroll
        for (int b = 0; b < NB; ++b)
          if (j < lim[b]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
              if ((h & 0x7f80u) == 0x7f80u) st.o[b][dt][i] += bf16_bits_to_f32(h);
            }
          }
      }
    }
  }

  // ---- merge of the wavefronts -----------------------------------------------------
  float* const ml = lds + NW * PARK;
  __syncthreads();  // the stages are free
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float lt = row_sum4(st.l[b]);
    if (g4 == 0) {
      ml[(wave * 2) * BM + 16 * b + col] = st.m[b];
      ml[(wave * 2 + 1) * BM + 16 * b + col] = lt;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      *reinterpret_cast<f32x4_t*>(lds + wave * PARK + (16 * b + col) * 132 + 16 * dt + 4 * g4) = st.o[b][dt];
  }
  __syncthreads();
  constexpr int TPR = 64 * NW / BM;  // threads of a row
  constexpr int DPT = HD / TPR;      // d positions of a thread
  const int row = tid / TPR, d0 = (tid % TPR) * 4;  // d0 + 4 TPR j
  const int m = m_base + row;
  if (m >= M) return;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) mx = fmaxf(mx, ml[(w * 2) * BM + row]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float f[NW], lsum = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float mw = ml[(w * 2) * BM + row];
    f[w] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mu);
    lsum += ml[(w * 2 + 1) * BM + row] * f[w];
  }
  const int tok = token_of(m, g), head = hkv * g + (m - tok * g);
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  const int part = part_of(wk, mtiles, max_split, Hkv);
#pragma unroll
  for (int j = 0; j < DPT / 4; ++j) {
    const int d = d0 + 4 * TPR * j;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (f[w] == 0.f) continue;  // a wavefront without keys
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(lds + w * PARK + row * 132 + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += x[e] * f[w];
    }
    if (ns == 1) {
      const u32x2_t w2 = {cvt_pk_bf16(acc[0] * inv, acc[1] * inv), cvt_pk_bf16(acc[2] * inv, acc[3] * inv)};
      *reinterpret_cast<u32x2_t*>(a.o + (int64_t)(sg.row0 + tok) * a.o_stride + head * HD + d) = w2;
    } else {
      *reinterpret_cast<f32x4_t*>(part_o<BM>(a, part, row) + d) = acc;
    }
  }
  if (ns > 1 && d0 == 0) {
    float* const pml = part_ml<BM>(a, logical_blocks, part, row);
    pml[0] = mx;
    pml[1] = lsum;
  }
}

// ---------------------------------------------------------------------------
// Many M rows: four wavefronts of 32 M rows share 64-key tiles of K and V in LDS
// (bf16, the swizzled layout of attn_tile.h), two stages.  The tile sequence is the
// cached rows' tiles, then those of the new rows.  While a tile is computed, the next one
// is on its way: bf16 rows by DMA into the other stage; 8-bit rows into registers (32
// bytes a thread and matrix), converted and written to the other stage after the
// products -- once per workgroup, not once per wavefront.  Two workgroups fit a CU, so
// that one computes while the other one waits at its barrier (eight wavefronts in one
// workgroup: 2048 rows behind 6144 cached, 32 heads, 289 against 296 us, but 8 ragged
// pieces, 28/4 heads, 147 against 139, 5 ragged ones, 32 heads, 212 against 199).
// The bf16 form also runs into what a CU takes in, 32 KB a tile and workgroup; V reads
// in one block that leaves the next tile's loads in flight were no faster.
//
// Bound by the matrix pipe and what its two wavefronts a SIMD do not overlap, and by
// power: 2048 rows behind 6144, 32 heads, 8-bit, 275 us back to back with changing inputs, 875
// TFLOP/s, the pipe busy 43 % of the time (bf16 50 %); 2 x 4096 bidirectional rows in bf16 1006.
constexpr int kTileRows = 128;
constexpr int kTileStage = 2 * kBigTile * 256;
template <bool FP8>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_tile_kernel(CHUNK_PARAMS) {
  constexpr int TK = kBigTile;
  constexpr int BM = kTileRows;
  constexpr int DMA = TK * 256 / 1024 / 4;   // DMA instructions of one matrix, tile and wavefront
  constexpr int PER = TK * 8 / 256;          // 8-bit rows: 16-byte pieces of one matrix and thread
  extern __shared__ __attribute__((aligned(16))) float lds_f[];
  uint8_t* const lds = reinterpret_cast<uint8_t*>(lds_f);  // two stages
  const int L = block_of(chunk_pages);
  if (L >= logical_blocks) return;
  const int max_pages = chunk_pages >> 5;
  const Work wk = work_of(L, mtiles, max_split, Hkv, false);
  const int s = wk.s, hkv = wk.hkv;
  const Segment sg = segment(a, cu, seg_ids, lens, s);
  const int g = a.g;
  const int M = sg.len * g;
  const int m_base = tile_of(wk, L, mtiles, max_split) * BM;
  if (m_base >= M) return;
  const int tok_first = token_of(m_base, g), tok_last = token_of(min(m_base + BM, M) - 1, g);
  const int ns = splits_of<true>(a, max_split, tiles_per_split, sg, tok_last);
  if (wk.split >= ns) return;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int lrow = lane & 31, hl = lane >> 5;
  const int rl = lane >> 4, P = lane & 15;

  const int t_cached = (sg.cached + TK - 1) / TK;
  const int see_first = visible(sg, tok_first, a.mask_block);
  const int t_all = t_cached + (visible(sg, tok_last, a.mask_block) + TK - 1) / TK;
  const int t0 = wk.split * tiles_per_split, t1 = min(t_all, t0 + tiles_per_split);
  const int c1 = min(t1, t_cached);          // cached tiles t0 .. c1 - 1, then new ones
  const uint32_t n_pages = (uint32_t)min(a.cache_rows >> 8, (int64_t)1 << 23);
  const int32_t* const pages = table + (int64_t)s * max_pages;
  const uint32_t bf_row = (uint32_t)(Hkv * HD * 2);

  // Page ids, one a lane: a tile's loads wait for no load of their own (with a scalar
  // load of the id in every turn the loop took 10 % longer).  Every 64 pages the next ones.
  int pg0 = t0 * TK / kPageRows, page_reg = -1;
  auto fetch_pages = [&](int pg) {
    pg0 = pg;
    page_reg = pages[min(pg0 + lane, max_pages - 1)];
  };
  if (n_pages > 0 && t0 < c1) fetch_pages(pg0);
  // `rows` rows (none: zeros) of kb / vb with strides kr / vr to a stage
  auto dma_rows = [&](uint8_t* stage, const void* kb, const void* vb, int rows, uint32_t kr, uint32_t vr) {
    const __amdgpu_buffer_rsrc_t krs = make_rsrc(kb, rows > 0 ? (uint32_t)(rows - 1) * kr + HD * 2 : 0u);
    const __amdgpu_buffer_rsrc_t vrs = make_rsrc(vb, rows > 0 ? (uint32_t)(rows - 1) * vr + HD * 2 : 0u);
#pragma unroll
    for (int j = 0; j < DMA; ++j) {
      const int q = DMA * wave + j;
      const uint32_t row = (uint32_t)(4 * q + rl);
      dma16(krs, stage + q * 1024, row * kr + (uint32_t)((P ^ ((4 * q + rl) & 15)) * 16));
      dma16(vrs, stage + TK * 256 + q * 1024, row * vr + (uint32_t)((P ^ (4 * rl)) * 16));
    }
  };
  auto issue_new = [&](uint8_t* stage, int t) {
    const int j0 = (t - t_cached) * TK;
    dma_rows(stage, a.k + (int64_t)(sg.row0 + j0) * a.k_stride + hkv * HD,
             a.v + (int64_t)(sg.row0 + j0) * a.v_stride + hkv * HD, sg.len - j0, (uint32_t)(a.k_stride * 2),
             (uint32_t)(a.v_stride * 2));
  };
  u32x4_t kx[PER], vx[PER];
  uint32_t ksc[PER], vsc[PER];
  // Cached tile t on its way to `stage` (8-bit rows: to registers); false where its
  // page is outside the cache.
  auto issue_cached = [&](uint8_t* stage, int t) -> bool {
    const int pg = t * TK / kPageRows;
    if (n_pages > 0 && pg - pg0 >= 64) fetch_pages(pg);
    int pid = __builtin_amdgcn_readlane(page_reg, pg - pg0);
    const bool ok = pg < max_pages && (uint32_t)pid < n_pages;
    pid = ok ? pid : 0;
    const int row0 = t * TK & (kPageRows - 1);
    const int rows = ok ? min(sg.cached - t * TK, TK) : 0;
    if constexpr (FP8) {
      const int64_t rec = ((int64_t)pid * Hkv + hkv) * kRecord + row0 * kQuantD;
      const __amdgpu_buffer_rsrc_t krs = make_rsrc(a.kc + rec, (uint32_t)rows * kQuantD);
      const __amdgpu_buffer_rsrc_t vrs = make_rsrc(a.vc + rec, (uint32_t)rows * kQuantD);
      const int64_t sc = ((int64_t)pid * Hkv + hkv) * kRecord + kScaleOff + row0;
      const __amdgpu_buffer_rsrc_t ksr = make_rsrc(a.kc + sc, (uint32_t)rows), vsr = make_rsrc(a.vc + sc, (uint32_t)rows);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int piece = i * 256 + tid;
        kx[i] = bload(krs, (uint32_t)piece * 16u, 0u);
        vx[i] = bload(vrs, (uint32_t)piece * 16u, 0u);
        // a row that does not exist: byte 0, which scales its zeros by 2^-127
        ksc[i] = __builtin_amdgcn_raw_buffer_load_b8(ksr, piece >> 3, 0, 0);
        vsc[i] = __builtin_amdgcn_raw_buffer_load_b8(vsr, piece >> 3, 0, 0);
      }
    } else {
      const int64_t off = ((int64_t)pid * kPageRows + row0) * bf_row + hkv * HD * 2;
      dma_rows(stage, a.kc + off, a.vc + off, rows, bf_row, bf_row);
    }
    return ok;
  };
  auto put = [&](uint8_t* stage) {
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int piece = i * 256 + tid, row = piece >> 3, ch = (piece & 7) * 2;
        const float ks = scale_of(ksc[i]), vs = scale_of(vsc[i]);
        uint8_t* const kr = stage + row * 256;
        uint8_t* const vr = stage + TK * 256 + row * 256;
        st128(kr + ((ch ^ (row & 15)) * 16), dequant8(u32x2_t{kx[i][0], kx[i][1]}, ks));
        st128(kr + (((ch + 1) ^ (row & 15)) * 16), dequant8(u32x2_t{kx[i][2], kx[i][3]}, ks));
        st128(vr + ((ch ^ (4 * (row & 3))) * 16), dequant8(u32x2_t{vx[i][0], vx[i][1]}, vs));
        st128(vr + (((ch + 1) ^ (4 * (row & 3))) * 16), dequant8(u32x2_t{vx[i][2], vx[i][3]}, vs));
      }
    }
  };

  bf16x8_t qf[8];
  const int m_lane = m_base + wave * 32 + lrow;
  const int lim = visible(sg, min(token_of(m_lane, g), sg.len - 1), a.mask_block);
  {
    const uint32_t qS = (uint32_t)(a.q_stride * 2);
    const uint32_t qbytes = (uint32_t)sg.len * qS;
    const __amdgpu_buffer_rsrc_t qrs = make_rsrc(a.q + (int64_t)sg.row0 * a.q_stride, qbytes);
    const int tok = token_of(m_lane, g);
    const bool ok = m_lane < M;
    const uint32_t qoff = (uint32_t)tok * qS + (uint32_t)((hkv * g + m_lane - tok * g) * HD + hl * 8) * 2u;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) qf[kk] = as_bf16x8(bload(qrs, ok ? qoff + (uint32_t)kk * 32u : qbytes, 0u));
  }
  // of this wavefront's rows: the least and the most that any sees
  const int lim_lo = __builtin_amdgcn_readfirstlane(
      visible(sg, min(token_of(m_base + wave * 32, g), sg.len - 1), a.mask_block));
  const int lim_hi =
      __builtin_amdgcn_readfirstlane(visible(sg, token_of(min(m_base + wave * 32 + 32, M) - 1, g), a.mask_block));
  const bool live = m_base + wave * 32 < M;

  DenseAddr ad;
  dense_addr(ad, lane, 0u, 0u);
  DenseState<1> st;
  dense_state_init(st);
  const float c = a.scale_log2;

  // One tile: scores, the keys from `valid` on hidden unless all are seen, softmax, V.
  // (One instance of it for all tiles: three -- whole cached tiles, the last one, new
  // ones -- spilled registers.)
  auto compute = [&](const uint8_t* cur, bool whole, int valid) {
    f32x16_t sacc[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[b][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const bf16x8_t af =
            as_bf16x8(*reinterpret_cast<const u32x4_t*>(cur + b * 32 * 256 + (ad.kbase ^ (uint32_t)(32 * kk))));
        sacc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, qf[kk], sacc[b], 0, 0, 0);
      }
    if (!whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (b * 32 + 8 * (i >> 2) + 4 * hl + (i & 3) >= valid) sacc[b][i] = -INFINITY;
    }
    bf16x8_t pf[4];
    dense_softmax<2, false>(sacc, st.oacc[0], st.m_run[0], st.l_run[0], st.thr[0], st.neg_m[0], pf, c, TK, 0, hl);
#pragma unroll
    for (int cch = 0; cch < 4; ++cch)
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const uint8_t* vp = cur + TK * 256 + (ad.vbase ^ (uint32_t)(64 * db)) + cch * 16 * 256;
        const u32x2_t x0 = ds_read_tr16(vp), x1 = ds_read_tr16(vp + 8 * 256);
        st.oacc[0][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(u32x4_t{x0[0], x0[1], x1[0], x1[1]}),
                                                                 pf[cch], st.oacc[0][db], 0, 0, 0);
      }
  };
  auto stage_of = [&](int t) { return lds + ((t - t0) & 1) * kTileStage; };
  auto tile_done = [&] {  // every wavefront's part of the next tile has arrived, this one's stage is free
    vm_wait<0>();
    __syncthreads();
  };

  bool ok = true;  // whether the page of the tile at hand is in the cache
  if (t0 < c1) {
    ok = issue_cached(stage_of(t0), t0);
    put(stage_of(t0));
    tile_done();
  } else if (t0 < t1) {
    issue_new(stage_of(t0), t0);
    tile_done();
  }
  // Q is waited for here: the compiler would else do so in every turn, and with it for
  // the next tile's loads (8192 new rows, 32 heads, 8-bit, 684 -> 662 us).
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) asm volatile("" : : "v"(qf[kk]));
  bool fixed = false;
  for (int t = t0; t < t1; ++t) {
    uint8_t* const cur = stage_of(t);
    uint8_t* const nxt = stage_of(t + 1);
    bool next_ok = true;
    if (t + 1 < c1)
      next_ok = issue_cached(nxt, t + 1);
    else if (t + 1 < t1)
      issue_new(nxt, t + 1);
    bool run = live && ok, whole;
    int valid;
    if (t < c1) {
      valid = sg.cached - t * TK;
      whole = valid >= TK;
    } else {
      const int j0 = (t - t_cached) * TK;
      valid = lim - j0;
      whole = lim_lo - j0 >= TK;
      run = run && lim_hi > j0;
      if (see_first - j0 < TK && see_first < sg.len) {
        // Some M row of the workgroup does not see all of the tile: a NaN or infinity in V
        // would reach it as 0 * V.  Every wavefront looks through the whole tile, so all agree;
        // such elements are multiplied as zeros and added at the end to the rows that see them.
        bool odd = false;
#pragma unroll 4
        for (int i = 0; i < TK * 256 / 1024; ++i)
          odd |= has_nonfinite(*reinterpret_cast<const u32x4_t*>(cur + TK * 256 + i * 1024 + lane * 16));
        if (__builtin_amdgcn_ballot_w64(odd)) {
          fixed = true;
          __syncthreads();
#pragma unroll 1
          for (int i = wave; i < TK * 256 / 1024; i += 4) {
            u32x4_t* const p = reinterpret_cast<u32x4_t*>(cur + TK * 256 + i * 1024 + lane * 16);
            *p = finite_part(*p);
          }
          __syncthreads();
        }
      }
    }
    if (run) compute(cur, whole, valid);
    if (t + 1 < c1) put(nxt);
    ok = next_ok;
    if (t + 1 < t1) tile_done();
  }
  if (fixed) {
    const uint16_t* const vnew = a.v + (int64_t)sg.row0 * a.v_stride + hkv * HD;
    const int end = min((t1 - t_cached) * TK, sg.len);
#pragma unroll 1
    for (int j = max(t0 - t_cached, 0) * TK; j < end; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * (i >> 2) + 8 * (i & 3) + 4 * hl;
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(vnew + (int64_t)j * a.v_stride + d);
        if (j < lim) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
            if ((h & 0x7f80u) == 0x7f80u) st.oacc[0][i >> 2][4 * (i & 3) + e] += bf16_bits_to_f32(h);
          }
        }
      }
  }

  const float l_tot = pair_sum32(st.l_run[0]);
  if (ns > 1) {
    if (m_lane < M) {
      float* const po = part_o<BM>(a, L, wave * 32 + lrow);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * (i >> 2) + 8 * (i & 3) + 4 * hl;
        *reinterpret_cast<f32x4_t*>(po + d) =
            f32x4_t{st.oacc[0][i >> 2][4 * (i & 3)], st.oacc[0][i >> 2][4 * (i & 3) + 1],
                    st.oacc[0][i >> 2][4 * (i & 3) + 2], st.oacc[0][i >> 2][4 * (i & 3) + 3]};
      }
      if (hl == 0) {
        float* const pml = part_ml<BM>(a, logical_blocks, L, wave * 32 + lrow);
        pml[0] = st.m_run[0];
        pml[1] = l_tot;
      }
    }
    return;
  }
  const float inv = l_tot != 0.f ? 1.f / l_tot : 0.f;
  __syncthreads();  // every wavefront is done with the stages
  uint8_t* const ot = lds + wave * 8192;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const u32x2_t w = {cvt_pk_bf16(st.oacc[0][db][4 * rq] * inv, st.oacc[0][db][4 * rq + 1] * inv),
                         cvt_pk_bf16(st.oacc[0][db][4 * rq + 2] * inv, st.oacc[0][db][4 * rq + 3] * inv)};
      *reinterpret_cast<u32x2_t*>(ot + lrow * 256 + (((4 * db + rq) ^ (lrow & 15)) * 16) + 8 * hl) = w;
    }
  wave_lds_fence();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = 4 * j + rl, m = m_base + wave * 32 + row;
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(ot + row * 256 + ((P ^ (row & 15)) * 16));
    if (m < M) {
      const int tok = token_of(m, g);
      st128(a.o + (int64_t)(sg.row0 + tok) * a.o_stride + (hkv * g + m - tok * g) * HD + P * 8, v);
    }
  }
}

// Joins the parts of every (segment, KV head, M row) whose keys were split.  G groups of
// 32 threads (four d each) share a row's parts, each taking every G-th, so that a row
// of many parts is one round of loads rather than a long chain (28 rows of 128 parts: 39 us
// with one group, 3.8 with eight).  Bound by its launch and that round: 3 - 4 us (32 x
// 28 rows of up to 8 parts 3.9).
template <int BM, bool TILE, int G>
__global__ __launch_bounds__(256) void chunk_combine_kernel(CHUNK_PARAMS) {
  static_assert(G == 1 || G == 8, "a workgroup holds eight rows or one");
  __shared__ f32x4_t part[G > 1 ? 256 : 1];
  __shared__ float part_s[G > 1 ? 16 : 1];
  const int grp = threadIdx.x >> 5;
  const int sub = grp % G;
  const int d0 = (threadIdx.x & 31) * 4;
  // grid: rows of the largest segment, KV heads, segments
  const int mrow = blockIdx.x * (8 / G) + grp / G;
  const int hkv = blockIdx.y, s = blockIdx.z;
  const int mt = mrow / BM, row = mrow % BM;
  if (mt >= mtiles) return;
  // part p of this row: workgroup L0 + p * mtiles (the tile form counts its M tiles from the last)
  const int L0 = (s * Hkv + hkv) * max_split * mtiles + (TILE ? mtiles - 1 - mt : mt);
  // A round of eight parts; those past the end, which hold anything, are left out after.
  f32x4_t x[8];
  float pm[8], pl[8];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = L0 + min(p0 + i * G, max_split - 1) * mtiles;
      x[i] = *reinterpret_cast<const f32x4_t*>(part_o<BM>(a, at, row) + d0);
      const float* const ml = part_ml<BM>(a, logical_blocks, at, row);
      pm[i] = ml[0];
      pl[i] = ml[1];
    }
  };
  fetch(sub);  // before the lengths that tell how many there are
  const Segment sg = segment(a, cu, seg_ids, lens, s);
  const int M = sg.len * a.g;
  const int parts = splits_of<TILE>(a, max_split, tiles_per_split, sg,
                                    TILE ? token_of(min((mt + 1) * BM, max(M, 1)) - 1, a.g) : 0);
  float mx = -INFINITY, l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = sub;;) {
    float top = mx;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (p0 + i * G >= parts) {
        pm[i] = -INFINITY;
        pl[i] = 0.f;
      }
      top = fmaxf(top, pm[i]);
    }
    const float mu = top == -INFINITY ? 0.f : top;
    const float w0 = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mu);
    l *= w0;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= w0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = pm[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm[i] - mu);
      l += pl[i] * w;  // a part of NaN scores alone has no maximum: its NaN stays in the sum
      if (w != 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += x[i][e] * w;
      }
    }
    mx = top;
    p0 += 8 * G;
    if (p0 >= parts) break;
    fetch(p0);
  }
  if constexpr (G > 1) {
    part[threadIdx.x] = acc;
    if ((threadIdx.x & 31) == 0) {
      part_s[2 * sub] = mx;
      part_s[2 * sub + 1] = l;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < G; ++i) top = fmaxf(top, part_s[2 * i]);
    const float tu = top == -INFINITY ? 0.f : top;
    l = 0.f;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float w = part_s[2 * i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(part_s[2 * i] - tu);
      l += part_s[2 * i + 1] * w;
      const f32x4_t x = part[32 * i + (threadIdx.x & 31)];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += x[e] * w;
    }
  }
  if (mrow >= M || parts == 1 || sub) return;  // one part: its workgroup wrote the row
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int tok = token_of(mrow, a.g), head = hkv * a.g + (mrow - tok * a.g);
  const u32x2_t w2 = {cvt_pk_bf16(acc[0] * inv, acc[1] * inv), cvt_pk_bf16(acc[2] * inv, acc[3] * inv)};
  *reinterpret_cast<u32x2_t*>(a.o + (int64_t)(sg.row0 + tok) * a.o_stride + head * HD + d0) = w2;
}

// ---- launch plan ---------------------------------------------------------------------
struct ChunkPlan {
  bool tile_form;
  int nb;                        // chunk_rows_kernel: 16-row blocks
  int bm;                        // M rows of a workgroup
  int max_split, tiles_per_split;
  bool turn;                     // rows form: the splits turn (work_of)
  int mtiles;                    // of the largest segment
  int run;                       // segments of a launch
  int64_t logical;               // its workgroups
};
// total_q / total_cached: the segments' sums, or an upper bound of them.
static ChunkPlan chunk_plan(int64_t n_seg, int max_q, int max_cached, int64_t total_q, int64_t total_cached, int Hq,
                            int Hkv) {
  ChunkPlan p = {};
  const int64_t g = Hq / Hkv, rows = max_q * g;
  // Tiles of 128 rows pay where they fill the card, three workgroups on four CUs, or where
  // there are many of them; otherwise the rows form, whose wavefronts share the keys.
  // 32/32 heads, rows / tiles in us: 8 x 100 rows behind 2000 84 / 75, 4 x 256 behind
  // 1000 59 / 51, but 1 x 300 behind 1000 31 / 38, 1 x 130 behind 500 16 / 20; 28/4 heads,
  // 1 x 1000 behind 1000 83 / 55, but 16 x 32 behind 384 - 1280 25 / 39, 4 x 100 behind 700 21 / 31.
  p.tile_form = rows > 1024 || (rows > 64 && n_seg * Hkv * ((rows + 127) / 128) >= 192);
  p.nb = rows <= 16 ? 1 : 2;
  p.bm = p.tile_form ? kTileRows : 16 * p.nb;
  p.mtiles = (int)((rows + p.bm - 1) / p.bm);
  // M tiles and tiles of all segments, at most
  const int64_t all_m = std::min(n_seg * p.mtiles, total_q * g / p.bm + n_seg);
  const int64_t key = p.tile_form ? kBigTile : kTileKeys;
  const int64_t tiles = (max_cached + key - 1) / key + (p.tile_form ? (max_q + key - 1) / key : 0);
  const int64_t all_t =
      std::min(n_seg * tiles, p.tile_form ? (total_cached + total_q + 2 * (key - 1) * n_seg) / key
                                          : (total_cached + (key - 1) * n_seg) / key);
  // Rows form: keys are split where that shortens the longest workgroup to two thirds.
  // Every workgroup pays for its start and the joining (8 x 32 rows behind 608 - 1216,
  // 32/32 heads, 256 workgroups: 20 us, split in two 30), and few keys are not split: the
  // joining takes 3 us, a turn of the wavefronts 0.8 (one token, 32 heads, whole / in parts:
  // behind 511 7.4 / 8.8, behind 767 8.4 / 9.3, behind 900 10.0 / 8.3).
  // As many parts as give every CU one workgroup where the sequences fill 0.7 or more of
  // the keys that they would all have at the longest one's length (one token behind 131071,
  // 28/4 heads: 256 workgroups 29.6 us, 384 34, 512 31; tokens, 28/4 heads, these parts / those of
  // the rule below: 16 behind 4000 18.2 / 20.3, behind 1600 - 4000 16.1 / 16.8, 12 behind 1200 -
  // 3000 12.8 / 13.1, 4 behind 3200 - 8000 12.4 / 13.9).  Three parts where whole ones would leave a third
  // of the CUs idle (5 tokens, 32 heads, bf16: behind 3565 54.1 whole, 53.1 in three, behind 1070 - 3565
  // 50.3 and 43.7; with several M tiles, 11 x 16 rows behind 3909, 28/4 heads, 30.5 and 37.8).
  // Where they fill 0.6 or less, parts of the longer ones even the card out: 384 workgroups, half
  // a part each lost to the last ones, 256 with many sequences, of 12 tiles at least, and none
  // of over half the longest (the same two: 32 tokens behind 512 - 4096 21.6 / 19.7, 32 behind 64 - 8192
  // 33 / 22.4, 64 behind 100 - 8000 53 / 37, 8 behind 64 - 4000, 32 heads, 30 / 24, one behind 15000 among
  // 256 behind 500 99 / 42; 8 behind 150 - 1500, 32 heads, whole 15.8, in two 18.3).  In between, the part
  // length goes over from the one to the other.
  const int64_t groups = all_m * Hkv;  // (M tile, KV head) pairs, each with its own parts
  const double work = (double)groups * (double)all_t / (double)n_seg;
  int64_t tps;
  if (p.tile_form) {
    // The work dealt to two workgroups a CU, whose phases overlap, if that halves the longest
    // and pays.  In us: a tile takes 1.7 in a workgroup that has its CU to itself, 2.4 in
    // one of two, a part of 128 rows 0.027 for its way through memory, the joining 3.  (256
    // workgroups of 20 tiles, 4 x 256 rows behind 1000, 32 heads: 44 us whole, 52 in two
    // parts; 220 of 112, 1000 rows behind 6144, 28/4 heads: 176 whole, 148 in three.)
    tps = std::max<int64_t>((int64_t)(work / 512 + 0.999), 4);
    const double parts = std::min((double)groups * (double)((tiles + tps - 1) / tps),
                                  work / (double)tps + 0.5 * (double)groups);
    const double whole = (groups <= 256 ? 1.7 : 2.4) * (double)tiles;
    if (tps * 2 > tiles || tiles <= 8 || whole < 2.4 * (double)tps + 3 + 0.027 * parts) tps = tiles;
  } else {
    const double fill = tiles ? (double)all_t / ((double)n_seg * (double)tiles) : 1;
    int64_t parts = std::max<int64_t>(1, 256 / groups);
    if (parts == 1 && p.mtiles == 1 && groups * 3 <= 512 && tiles >= 96) parts = 3;
    const double even = (double)std::max<int64_t>((tiles + parts - 1) / parts, 4);
    const double uneven = std::max(work / std::max(384 - 0.5 * (double)groups, 256.), 12.);
    const double to_even = std::min(std::max((fill - 0.6) * 10, 0.), 1.);
    tps = (int64_t)(uneven + to_even * (even - uneven) + 0.999);
    p.turn = to_even < 1;
    if ((double)tps > (double)tiles * (3 + to_even) / 6 || tiles <= (groups > 128 ? 32 : 24)) tps = tiles;
  }
  if (!p.tile_form) tps = std::min<int64_t>((tps + 3) / 4 * 4, kMaxSplitTiles);
  if (tps < 1) tps = 1;
  // Every segment of a launch has room for the parts that the one with the most rows and
  // the one with the most keys have together: a piece of a prompt among many single tokens
  // would ask for tens of gigabytes (2048 rows behind 131072 and 63 tokens behind 500,
  // 28/4 heads: 65).  So the segments are launched in runs, one after the other, that
  // use the same workspace; a run that fills it has over sixteen thousand workgroups.
  const int64_t part = Hkv * (int64_t)p.mtiles * p.bm * (HD + 2) * (int64_t)sizeof(float);  // of all rows of a segment
  const int64_t most = std::max<int64_t>(1, kMaxParts / part);
  if ((tiles + tps - 1) / tps > most) {
    tps = (tiles + most - 1) / most;
    if (!p.tile_form) tps = std::min<int64_t>((tps + 3) / 4 * 4, kMaxSplitTiles);
  }
  if (tps > 0x3fffffff) tps = 0x3fffffff;
  p.tiles_per_split = (int)tps;
  p.max_split = (int)std::max<int64_t>(1, (tiles + tps - 1) / tps);
  const int64_t blocks = Hkv * (int64_t)p.mtiles * p.max_split;  // of a segment
  int64_t run = std::min(n_seg, kMaxBlocks / blocks);
  if (p.max_split > 1) run = std::min(run, kMaxParts / (part * p.max_split));
  run = std::max<int64_t>(run, 1);
  const int64_t runs = (n_seg + run - 1) / run;
  p.run = (int)((n_seg + runs - 1) / runs);
  p.logical = p.run * blocks;
  return p;
}
static size_t chunk_ws(const ChunkPlan& p) {
  return p.max_split <= 1 ? 0 : (size_t)p.logical * p.bm * (HD + 2) * sizeof(float);
}

}  // namespace dllm

using namespace dllm;

static bool chunk_sizes_ok(int n_seg, int max_q, int max_cached, int64_t total_q, int64_t total_cached, int Hq, int Hkv,
                           int D) {
  return D == HD && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && n_seg >= 0 && max_q >= 0 && max_cached >= 0 && total_q >= 0 &&
         total_cached >= 0 && max_cached <= 0x7fffffff - 64 && (int64_t)max_q * (Hq / Hkv) <= (1 << 30);
}
// Sums that are not given, or beyond what the largest segment allows.
static int64_t chunk_total(int64_t total, int n_seg, int most) {
  const int64_t bound = (int64_t)n_seg * most;
  return total > 0 && total < bound ? total : bound;
}

extern "C" size_t dllm_attn_chunk_workspace_size(int n_seg, int max_q, int max_cached, int64_t total_q,
                                                 int64_t total_cached, int Hq, int Hkv, int D) {
  if (!chunk_sizes_ok(n_seg, max_q, max_cached, total_q, total_cached, Hq, Hkv, D) || n_seg == 0 || max_q == 0) return 0;
  return chunk_ws(chunk_plan(n_seg, max_q, max_cached, chunk_total(total_q, n_seg, max_q),
                             chunk_total(total_cached, n_seg, max_cached), Hq, Hkv));
}

static int chunk_grid(int64_t logical, int mtiles, int* chunk) {
  // The M tiles of a (segment, KV head) read the same keys: next to each other on one XCD,
  // but no more than four, which would give one XCD the longest work (8 ragged
  // pieces, 28/4 heads: chunks of 16 156 us, 4 140; 8192 new rows, 32 heads, 662 and 678).
  *chunk = std::min(mtiles, 4);
  const int64_t grain = 8 * (int64_t)*chunk;
  return (int)((logical + grain - 1) / grain * grain);
}

extern "C" int dllm_attn_chunk_launch_shape(int n_seg, int max_q, int max_cached, int64_t total_q, int64_t total_cached,
                                            int Hq, int Hkv, int D, int* rows, int* n_split, int* grid) {
  if (!chunk_sizes_ok(n_seg, max_q, max_cached, total_q, total_cached, Hq, Hkv, D))
    return fail(DLLM_ERR_INVALID_ARG, "dllm_attn_chunk_launch_shape: unsupported sizes");
  ChunkPlan p = {};
  int chunk, blocks = 0;
  if (n_seg > 0 && max_q > 0) {
    p = chunk_plan(n_seg, max_q, max_cached, chunk_total(total_q, n_seg, max_q),
                   chunk_total(total_cached, n_seg, max_cached), Hq, Hkv);
    blocks = p.logical > kMaxBlocks ? 0 : chunk_grid(p.logical, p.mtiles, &chunk);
  }
  if (rows) *rows = p.bm;
  if (n_split) *n_split = p.max_split;
  if (grid) *grid = blocks;
  return DLLM_OK;
}

extern "C" int dllm_attn_chunk_paged_fwd(const dllm_bf16* q, const dllm_bf16* k, const dllm_bf16* v, dllm_bf16* o,
                                         const int32_t* cu, const int32_t* seg_ids, int n_seg, int max_q, int max_cached,
                                         int64_t total_q, int64_t total_cached, const void* k_cache,
                                         const void* v_cache, int cache_type, int num_pages,
                                         const int32_t* page_table, int max_pages, const int32_t* cached_len,
                                         int mask_block, int Hq, int Hkv, int D, int64_t q_stride, int64_t k_stride,
                                         int64_t v_stride, int64_t o_stride, float softmax_scale, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  const char* name = "dllm_attn_chunk_paged_fwd";
  set_error("");
  int rc = common_checks(name, q, k, v, o, Hq, Hkv, D, q_stride, k_stride, v_stride, o_stride);
  if (rc) return rc;
  if (n_seg < 0 || max_q < 0 || max_cached < 0 || mask_block < 0 || max_pages < 0 || total_q < 0 ||
      total_cached < 0)
    return fail(DLLM_ERR_INVALID_ARG, "%s: negative size", name);
  if (cache_type != DLLM_CACHE_BF16 && cache_type != DLLM_CACHE_FP8)
    return fail(DLLM_ERR_INVALID_ARG, "%s: cache type %d", name, cache_type);
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY))
    return fail(DLLM_ERR_INVALID_ARG, "%s: softmax_scale must be positive and finite", name);
  if (n_seg == 0 || max_q == 0) return DLLM_OK;
  if (!chunk_sizes_ok(n_seg, max_q, max_cached, total_q, total_cached, Hq, Hkv, D))
    return fail(DLLM_ERR_UNSUPPORTED, "%s: %d new rows of %d query heads per KV head, %d cached", name, max_q, Hq / Hkv,
                max_cached);
  if (num_pages < 0 || num_pages > (1 << 23)) return fail(DLLM_ERR_INVALID_ARG, "%s: %d pages", name, num_pages);
  if (!cu || !cached_len) return fail(DLLM_ERR_INVALID_ARG, "%s: null cu / lengths", name);
  const int64_t kvs = k_stride > v_stride ? k_stride : v_stride;
  if ((int64_t)max_q * (q_stride > kvs ? q_stride : kvs) * 2 + 4096 >= ((int64_t)1 << 32))
    return fail(DLLM_ERR_UNSUPPORTED, "%s: a segment spans more than 4 GiB of q / k / v", name);
  if (cache_type == DLLM_CACHE_BF16 && (int64_t)Hkv * HD * 2 * kPageRows >= ((int64_t)1 << 31))
    return fail(DLLM_ERR_UNSUPPORTED, "%s: %d KV heads", name, Hkv);
  if (max_cached > 0 && num_pages > 0) {
    if (!k_cache || !v_cache || !page_table || max_pages == 0)
      return fail(DLLM_ERR_INVALID_ARG, "%s: null cache / page table", name);
    if (!aligned16(k_cache) || !aligned16(v_cache))
      return fail(DLLM_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", name);
  }
  if ((int64_t)n_seg * max_pages >= ((int64_t)1 << 31) || max_pages >= (1 << 26))
    return fail(DLLM_ERR_INVALID_ARG, "%s: page table too large", name);
  ChunkArgs a = {};
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.kc = reinterpret_cast<const uint8_t*>(k_cache);
  a.vc = reinterpret_cast<const uint8_t*>(v_cache);
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.o_stride = o_stride;
  a.cache_rows = (int64_t)num_pages * kPageRows;
  a.max_q = max_q; a.max_cached = max_cached;
  a.g = Hq / Hkv;
  a.mask_block = mask_block;
  a.scale_log2 = softmax_scale * kLog2e;
  const ChunkPlan p = chunk_plan(n_seg, max_q, max_cached, chunk_total(total_q, n_seg, max_q),
                                 chunk_total(total_cached, n_seg, max_cached), Hq, Hkv);
  if (p.logical > kMaxBlocks || n_seg > 65535 || Hkv > 65535)
    return fail(DLLM_ERR_INVALID_ARG, "%s: problem too large", name);
  const size_t need = chunk_ws(p);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return fail(DLLM_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", name, need,
                  workspace ? workspace_bytes : (size_t)0);
    if (!aligned16(workspace)) return fail(DLLM_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name);
    a.ws = reinterpret_cast<float*>(workspace);
  }
  int chunk;
  const int chunk_pages_row = max_cached > 0 && num_pages > 0 ? max_pages : 0;
  const bool fp8 = cache_type == DLLM_CACHE_FP8;
  // Few workgroups of some length: eight wavefronts each, which halves the turns (and takes a
  // CU's LDS, so 8-bit rows only).  One token behind 511 rows, 32 heads, 8.5 -> 7.4 us, behind
  // 767 10.1 -> 8.5, 128 rows behind 4000 29.9 -> 26.9; not where a workgroup a CU streams from
  // memory (4 tokens behind 2000 18.6, 18.8), nor for 32 rows of few keys, whose merge is
  // longer (32 behind 300 10.0, 10.4).
  const bool eight = fp8 && p.logical <= (p.mtiles > 1 ? 256 : 192) && p.tiles_per_split > (p.nb == 1 ? 4 : 12);
  for (int s0 = 0; s0 < n_seg; s0 += p.run) {
    const int segs = std::min(p.run, n_seg - s0);
    const int logical = (int)(p.logical / p.run * segs);
    const int grid = chunk_grid(logical, p.mtiles, &chunk);
    const int chunk_pages = chunk + (p.turn && p.max_split > 1 ? 16 : 0) + 32 * chunk_pages_row;
    auto start = [&](auto kern, dim3 blocks, int threads, int lds_bytes) {
      kern<<<blocks, dim3((unsigned)threads), lds_bytes, reinterpret_cast<hipStream_t>(stream)>>>(
          seg_ids ? cu : cu + s0, seg_ids ? seg_ids + s0 : nullptr, cached_len + s0,
          page_table + (int64_t)s0 * chunk_pages_row, chunk_pages, logical, p.mtiles, p.max_split, p.tiles_per_split, Hkv,
          a);
      return check_launch(name);
    };
    auto launch = [&](auto kern, int lds_bytes, int threads = 256) -> int {
      int e = set_lds(kern, lds_bytes, name);
      if (e) return e;
      return start(kern, dim3((unsigned)grid), threads, lds_bytes);
    };
    if (p.tile_form)
      rc = launch(fp8 ? chunk_tile_kernel<true> : chunk_tile_kernel<false>, 2 * kTileStage);
    else if (eight)
      rc = p.nb == 1 ? launch(chunk_rows_kernel<1, true, true, 8>, rows_lds<1, true, 8>(), 512)
           : p.mtiles == 1 ? launch(chunk_rows_kernel<2, true, true, 8>, rows_lds<2, true, 8>(), 512)
                           : launch(chunk_rows_kernel<2, true, false, 8>, rows_lds<2, true, 8>(), 512);
    else if (p.nb == 1)  // at most 16 rows
      rc = fp8 ? launch(chunk_rows_kernel<1, true, true, 4>, rows_lds<1, true, 4>())
               : launch(chunk_rows_kernel<1, false, true, 4>, rows_lds<1, false, 4>());
    else if (p.mtiles == 1)
      rc = fp8 ? launch(chunk_rows_kernel<2, true, true, 4>, rows_lds<2, true, 4>())
               : launch(chunk_rows_kernel<2, false, true, 4>, rows_lds<2, false, 4>());
    else
      rc = fp8 ? launch(chunk_rows_kernel<2, true, false, 4>, rows_lds<2, true, 4>())
               : launch(chunk_rows_kernel<2, false, false, 4>, rows_lds<2, false, 4>());
    if (rc || p.max_split == 1) {
      if (rc) return rc;
      continue;
    }
    auto join = [&](auto one, auto eight) {
      const bool many = p.max_split > 8;
      const int64_t rows = (int64_t)max_q * a.g;
      return start(many ? eight : one, dim3((unsigned)(many ? rows : (rows + 7) / 8), (unsigned)Hkv, (unsigned)segs), 256,
                   0);
    };
    if (p.tile_form)
      rc = join(chunk_combine_kernel<kTileRows, true, 1>, chunk_combine_kernel<kTileRows, true, 8>);
    else
      rc = p.nb == 1 ? join(chunk_combine_kernel<16, false, 1>, chunk_combine_kernel<16, false, 8>)
                     : join(chunk_combine_kernel<32, false, 1>, chunk_combine_kernel<32, false, 8>);
    if (rc) return rc;
  }
  return DLLM_OK;
}
