// What the attention kernels share: the XCD block map, the LDS tile layout with
// its operand reads, the online softmax of a 32-row block over one key tile, and
// the host-side checks of the entry points.
#pragma once

#include "common.h"

#include <math.h>

namespace dllm {

constexpr int HD = 128;       // the head dim these kernels handle

// Work-groups are dispatched round-robin over the 8 XCDs (XCD = b % 8), and
// each XCD has its own L2.  Logical blocks are dealt to the XCDs in chunks of
// `ch` consecutive ones, chunk j to XCD j % 8, so the blocks of a chunk (the
// m-tiles of one (segment, head), which read the same K/V) share an L2, while
// every XCD gets an even share of every part of the batch.  Handing each XCD
// one contiguous eighth instead left ragged batches unbalanced: with 16
// segments of 410..1245 tokens the busiest XCD held 1.6x the mean work
// (those 16 segments, 28 query / 4 KV heads: 226 -> 172 us with chunks of
// 4).  The grid must be a multiple of 8 * ch; the map is then a bijection
// onto [0, grid).
__device__ __forceinline__ int xcd_remap(int b, int ch) {
  const int x = b & 7, i = b >> 3;
  const int j = i / ch;
  return (j * 8 + x) * ch + (i - j * ch);
}

// Running softmax state of one wavefront (M row = lane % 32).  The reference
// maximum m_run (log2 domain) is only raised when a new score exceeds it by
// more than kLazy, so most tiles skip rescaling O; probabilities then stay
// below 2^kLazy, well inside the bf16 / fp32 range.
constexpr float kLazy = 8.0f;

// ---------------------------------------------------------------------------
// Key tiles of the dense form (K3a): K and V go HBM -> LDS by buffer DMA
// (buffer_load_dwordx4 ... lds, no VGPR staging); the V^T MFMA operand is
// read with the transposing LDS read ds_read_b64_tr_b16.
//
// LDS per stage (2 stages): K [64 keys][256 B] then V [64 keys][256 B], no
// padding; 16-byte chunks are XOR-swizzled inside a row so the MFMA operand
// reads are bank-conflict free:
//   K: physical chunk = logical chunk ^ (row & 15)
//   V: physical chunk = logical chunk ^ (4 * (row & 3))
// One DMA instruction writes 1 KiB = 4 rows; lane L of it carries row
// 4q + L/16, physical chunk L%16.
//
// ds_read_b64_tr_b16 (gfx950): in each group of 16 lanes, lane 4k+c supplies
// 8 bytes = elements [4c, 4c+4) of row k of a 4 x 16 block; lane n receives
// column n (rows 0..3).  With rows = keys and columns = head-dim positions
// this yields 4 consecutive keys of one d: half of a V^T A-operand fragment.
typedef short i16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2_t ds_read_tr16(const uint8_t* p) {
  const i16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4_t*)(const_cast<uint8_t*>(p)));
  return __builtin_bit_cast(u32x2_t, v);
}

// Per-lane LDS / DMA offsets.  The swizzles make every per-kk (K) and per-db
// (V) read offset a XOR of one base with a compile-time constant:
//   K read, kk:  lrow*256 + ((2kk + hl) ^ (lrow & 15))*16 = kbase ^ (32 kk)
//   V read, db:  (4hl + k)*256 + (4(db ^ k) + 2 dhalf + c/2)*16 + 8(c&1) = vbase ^ (64 db)
// A DMA instruction q writes tile rows R = 4q + L/16 (L = lane), physical
// chunk P = L % 16, i.e. global chunk P ^ (R & 15) (K) or P ^ 4(R & 3) (V):
//   K: (L/16)*kS + ((P ^ (L/16)) * 16 ^ 64 (q & 3))      V: (L/16)*vS + (P ^ 4(L/16))*16
// (the XOR acts on the chunk offset alone, the row offset is added after it)
struct DenseAddr {
  uint32_t kbase, vbase;
  uint32_t kdma_row, kdma_chunk, vdma;
};

__device__ __forceinline__ void dense_addr(DenseAddr& ad, int lane, uint32_t kS, uint32_t vS) {
  const int rl = lane >> 4, P = lane & 15;
  ad.kdma_row = (uint32_t)rl * kS;
  ad.kdma_chunk = (uint32_t)((P ^ rl) * 16);
  ad.vdma = (uint32_t)rl * vS + (uint32_t)((P ^ (4 * rl)) * 16);
  const int lrow = lane & 31, hl = lane >> 5;
  ad.kbase = (uint32_t)(lrow * 256 + ((hl ^ (lrow & 15)) * 16));
  const int dhalf = (lane >> 4) & 1, k = (lane & 15) >> 2, c = lane & 3;
  ad.vbase = (uint32_t)((4 * hl + k) * 256 + (4 * k + 2 * dhalf + (c >> 1)) * 16 + 8 * (c & 1));
}

// Softmax state of NQ query blocks (32 M rows each) of one wavefront.
// thr = m_run + kLazy and neg_m = -m_run (0 while m_run is -inf) change only
// when m_run does, so the per-tile test and exponent need no extra VALU work.
template <int NQ>
struct DenseState {
  f32x16_t oacc[NQ][4];
  float m_run[NQ];
  float l_run[NQ];
  float thr[NQ];
  float neg_m[NQ];
};

template <int NQ>
__device__ __forceinline__ void dense_state_init(DenseState<NQ>& st) {
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.oacc[q][db][i] = 0.f;
    st.m_run[q] = -INFINITY;
    st.l_run[q] = 0.f;
    st.thr[q] = -INFINITY;
    st.neg_m[q] = 0.f;
  }
}

// Raises the reference maximum of the rows whose tile maximum mx exceeds it by
// more than kLazy, and rescales their state.
__device__ __forceinline__ void dense_raise_max(float mx, f32x16_t (&oacc)[4], float& m_run, float& l_run, float& thr,
                                                float& neg_m) {
  const bool need = mx > thr;
  if (__builtin_amdgcn_ballot_w64(need)) {
    const float m_new = need ? mx : m_run;
    const float alpha = (m_run == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[db][i] *= alpha;
    m_run = m_new;
    thr = m_run + kLazy;
    neg_m = (m_run == -INFINITY) ? 0.f : -m_run;
  }
}

// Online-softmax update of one query block from its two S^T key blocks;
// returns the packed P^T fragments (B operands of O^T += V^T P^T).
template <int KB, bool MASK>
__device__ __forceinline__ void dense_softmax(f32x16_t (&sacc)[KB], f32x16_t (&oacc)[4], float& m_run, float& l_run,
                                              float& thr, float& neg_m, bf16x8_t (&pf)[2 * KB], float c, int k_valid,
                                              uint64_t bad, int hl) {
  float mx = -INFINITY;
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (MASK) {
        const int key = b * 32 + 8 * (i >> 2) + 4 * hl + (i & 3);
        if (key >= k_valid || ((bad >> key) & 1ull)) sacc[b][i] = -INFINITY;
      }
      mx = fmaxf(mx, sacc[b][i]);
    }
  mx = pair_max32(mx) * c;
  dense_raise_max(mx, oacc, m_run, l_run, thr, neg_m);
  // The row sum adds the bf16-rounded numerators, the same values the O^T
  // product consumes; two partial sums (one starting from l_run) keep the
  // dependent chain short.
  float psum[2] = {l_run, 0.f};
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4_t pk;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[b][8 * j + 2 * w], c, neg_m));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[b][8 * j + 2 * w + 1], c, neg_m));
        pk[w] = cvt_pk_bf16(p0, p1);
        psum[w & 1] = add_bf16x2(pk[w], psum[w & 1]);
      }
      pf[2 * b + j] = as_bf16x8(pk);
    }
  l_run = psum[0] + psum[1];
}

// One key tile (TK keys) for one wavefront owning NQ query blocks: every K
// and V^T operand fragment read from LDS feeds NQ MFMAs.
// V^T operands of one 32-key block for callers whose tiles arrive by
// global_load_lds: the compiler makes every transposing-read builtin wait for
// all such DMA still in flight (it cannot tell the tiles apart), which would
// drain the next tile's prefetch.  The 16 reads are one asm block that ends
// with its own lgkmcnt(0) wait, so its outputs are complete when it returns.
// Read (c, d, h) -- key chunk c, d block d, half h -- is at
// vbase ^ 64 d + 4096 c + 2048 h; output index (4 c + d) * 2 + h.
__device__ __forceinline__ void v_operands_untracked(const uint8_t* Vs, const DenseAddr& ad, u32x2_t (&r)[16]) {
  uint32_t b[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
    b[d] = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)(Vs + (ad.vbase ^ (uint32_t)(64 * d)));
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n"
      "ds_read_b64_tr_b16 %1, %16 offset:2048\n"
      "ds_read_b64_tr_b16 %2, %17\n"
      "ds_read_b64_tr_b16 %3, %17 offset:2048\n"
      "ds_read_b64_tr_b16 %4, %18\n"
      "ds_read_b64_tr_b16 %5, %18 offset:2048\n"
      "ds_read_b64_tr_b16 %6, %19\n"
      "ds_read_b64_tr_b16 %7, %19 offset:2048\n"
      "ds_read_b64_tr_b16 %8, %16 offset:4096\n"
      "ds_read_b64_tr_b16 %9, %16 offset:6144\n"
      "ds_read_b64_tr_b16 %10, %17 offset:4096\n"
      "ds_read_b64_tr_b16 %11, %17 offset:6144\n"
      "ds_read_b64_tr_b16 %12, %18 offset:4096\n"
      "ds_read_b64_tr_b16 %13, %18 offset:6144\n"
      "ds_read_b64_tr_b16 %14, %19 offset:4096\n"
      "ds_read_b64_tr_b16 %15, %19 offset:6144\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]),
        "=&v"(r[15])
      : "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3])
      : "memory");
}

// The same for NDB d blocks from vb (vbase with the first block's 64 d XORed in);
// output index (NDB c + d) * 2 + h.
template <int NDB>
__device__ __forceinline__ void v_operands_blocks(const uint8_t* Vs, uint32_t vb, u32x2_t (&r)[4 * NDB]) {
  static_assert(NDB == 1 || NDB == 2, "d blocks");
  const uint32_t b0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)(Vs + vb);
  if constexpr (NDB == 1) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n"
        "ds_read_b64_tr_b16 %1, %4 offset:2048\n"
        "ds_read_b64_tr_b16 %2, %4 offset:4096\n"
        "ds_read_b64_tr_b16 %3, %4 offset:6144\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(b0)
        : "memory");
  } else {
    const uint32_t b1 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)(Vs + (vb ^ 64u));
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n"
        "ds_read_b64_tr_b16 %1, %8 offset:2048\n"
        "ds_read_b64_tr_b16 %2, %9\n"
        "ds_read_b64_tr_b16 %3, %9 offset:2048\n"
        "ds_read_b64_tr_b16 %4, %8 offset:4096\n"
        "ds_read_b64_tr_b16 %5, %8 offset:6144\n"
        "ds_read_b64_tr_b16 %6, %9 offset:4096\n"
        "ds_read_b64_tr_b16 %7, %9 offset:6144\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(b0), "v"(b1)
        : "memory");
  }
}

template <int NQ, int TK, bool MASK, bool UNTRACKED_V = false>
__device__ __forceinline__ void dense_tile(const uint8_t* Ks, const uint8_t* Vs, const DenseAddr& ad,
                                           const bf16x8_t (&qf)[NQ][8], DenseState<NQ>& st, float c, int k_valid,
                                           uint64_t bad = 0) {
  constexpr int KB = TK / 32;  // key blocks of 32 per tile
  const int lane = threadIdx.x & 63;
  const int hl = lane >> 5;
  // kk outer, key block inner: the KB*NQ accumulators form independent MFMA
  // chains that interleave instead of one chain waiting on itself.  Each
  // S^T block is one chain over the head dimension: the wavefronts sharing
  // a SIMD interleave their chains, and splitting the reduction over two
  // partial accumulators (to lengthen the chain count) costs 16 VALU adds per
  // tile to merge them -- 2-5 % slower at every measured shape, since the
  // softmax VALU work rivals the MFMA work.
  f32x16_t sacc[NQ][KB];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[q][b][i] = 0.f;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const bf16x8_t af =
          as_bf16x8(*reinterpret_cast<const u32x4_t*>(Ks + b * 32 * 256 + (ad.kbase ^ (uint32_t)(32 * kk))));
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        sacc[q][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, qf[q][kk], sacc[q][b], 0, 0, 0);
    }
  }
  bf16x8_t pf[NQ][2 * KB];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    dense_softmax<KB, MASK>(sacc[q], st.oacc[q], st.m_run[q], st.l_run[q], st.thr[q], st.neg_m[q], pf[q], c, k_valid,
                            bad, hl);
  if constexpr (UNTRACKED_V) {
    static_assert(KB == 1, "one 32-key block per call");
    u32x2_t r[16];
    v_operands_untracked(Vs, ad, r);
#pragma unroll
    for (int cch = 0; cch < 2; ++cch)
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const u32x2_t lo = r[(4 * cch + db) * 2], hi = r[(4 * cch + db) * 2 + 1];
        const bf16x8_t af = as_bf16x8(u32x4_t{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
        for (int q = 0; q < NQ; ++q)
          st.oacc[q][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, pf[q][cch], st.oacc[q][db], 0, 0, 0);
      }
    return;
  }
  // key chunk outer, d block inner: 4*NQ independent accumulator chains.
#pragma unroll
  for (int cch = 0; cch < 2 * KB; ++cch) {
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      const uint8_t* vp = Vs + (ad.vbase ^ (uint32_t)(64 * db)) + cch * 16 * 256;
      const u32x2_t lo = ds_read_tr16(vp);
      const u32x2_t hi = ds_read_tr16(vp + 8 * 256);
      u32x4_t a4 = {lo[0], lo[1], hi[0], hi[1]};
      const bf16x8_t af = as_bf16x8(a4);
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        st.oacc[q][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, pf[q][cch], st.oacc[q][db], 0, 0, 0);
    }
  }
}

static const float kLog2e = 1.4426950408889634f;

static int common_checks(const char* name, const void* q, const void* k, const void* v, const void* o, int Hq,
                         int Hkv, int D, int64_t qs, int64_t ks, int64_t vs, int64_t os) {
  if (D != HD) return fail(DLLM_ERR_UNSUPPORTED, "%s: head_dim %d not supported (the kernels handle 128)", name, D);
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return fail(DLLM_ERR_INVALID_ARG, "%s: Hq=%d must be a positive multiple of Hkv=%d", name, Hq, Hkv);
  if (!q || !k || !v || !o) return fail(DLLM_ERR_INVALID_ARG, "%s: null tensor pointer", name);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return fail(DLLM_ERR_INVALID_ARG, "%s: q/k/v/o must be 16-byte aligned", name);
  if (qs % 8 || ks % 8 || vs % 8 || os % 8)
    return fail(DLLM_ERR_INVALID_ARG, "%s: token strides must be multiples of 8 elements", name);
  if (qs < (int64_t)Hq * D || os < (int64_t)Hq * D || ks < (int64_t)Hkv * D || vs < (int64_t)Hkv * D)
    return fail(DLLM_ERR_INVALID_ARG, "%s: token stride smaller than a token row", name);
  return DLLM_OK;
}

// Raise a kernel's dynamic-LDS limit (once per kernel and device; a thread
// remembers the devices of each kernel of a type as bits).
template <typename KernelFn>
static int set_lds(KernelFn fn, int bytes, const char* name) {
  constexpr int kKernels = 24;  // of one type: the block-cached form has twelve
  static thread_local const void* done[kKernels];
  static thread_local uint64_t done_dev[kKernels];
  static thread_local int n_done = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = -1;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  const void* key = reinterpret_cast<const void*>(fn);
  int i = 0;
  while (i < n_done && done[i] != key) ++i;
  if (i < n_done && (done_dev[i] & bit)) return DLLM_OK;
  hipError_t e = hipFuncSetAttribute(key, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return fail(DLLM_ERR_HIP, "%s: hipFuncSetAttribute(LDS %d B): %s", name, bytes, hipGetErrorString(e));
  if (i < kKernels) {
    done[i] = key;
    done_dev[i] |= bit;
    if (i == n_done) ++n_done;
  }
  return DLLM_OK;
}

}  // namespace dllm
