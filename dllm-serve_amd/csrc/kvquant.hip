// Quantising KV-cache scatter and its read-back (the 8-bit counterpart of
// kvcache.hip; row format in quant.h).
//
// Sixteen lanes carry one (token, KV head) row of K and of V, eight elements each:
// one 16-byte load, the row's maximum by four cross-lane steps, one 8-byte store
// (the sixteen lanes write a whole 128-byte line), and one lane's scale byte.  The
// reverse reads 8 bytes and the scale and writes 16.  Both are bound by memory: 512
// bytes per row of K and V on one side, 258 on the other.  10240 tokens of 32 heads: store
// 46.2 us, load 45.8, 5.5 TB/s each, above the 5.1 of a plain copy; 512 tokens of 4
// heads 2.3 us each, the launch.  Two or four rows in flight a lane group were no faster.
#include "quant.h"

namespace dllm {

// Leading scalar arguments (13 dwords): the library is built with kernel argument
// preloading, so a wave's first loads wait for no load of their addresses.
//   slot, k, v   slots; token rows (read by the store, written by the load)
//   rows         n_tok * Hkv
//   chunk        consecutive workgroups of an XCD
//   *_stride     elements
//   kp, vp       pages
#define QUANT_PARAMS                                                                                     \
  const int32_t *__restrict__ slots, uint16_t *__restrict__ k, uint16_t *__restrict__ v, int rows, int Hkv, \
      int chunk, int64_t k_stride, int64_t v_stride, uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, int64_t n_slots

template <bool VEC>
__device__ __forceinline__ u32x4_t ld_row8(const uint16_t* p) {
  if constexpr (VEC) return ld128_stream(p);
  u32x4_t r;
#pragma unroll
  for (int w = 0; w < 4; ++w) r[w] = (uint32_t)p[2 * w] | ((uint32_t)p[2 * w + 1] << 16);
  return r;
}
template <bool VEC>
__device__ __forceinline__ void st_row8(uint16_t* p, u32x4_t x) {
  if constexpr (VEC) {
    st128(p, x);
  } else {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      p[2 * w] = (uint16_t)x[w];
      p[2 * w + 1] = (uint16_t)(x[w] >> 16);
    }
  }
}

// Sixteen lanes a row; a workgroup takes 16 consecutive (token, head) rows.
template <bool VEC>
__global__ __launch_bounds__(256) void kv_quant_store(QUANT_PARAMS) {
  const int L = (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3);
  const int lane16 = threadIdx.x & 15;
  const int row = L * 16 + (threadIdx.x >> 4);
  int64_t slot = -1;
  int head = 0;
  u32x4_t kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
  if (row < rows) {
    const int tok = (int)((uint32_t)row / (uint32_t)Hkv);
    head = row - tok * Hkv;
    const int64_t e = (int64_t)head * kQuantD + lane16 * 8;
    slot = slots[tok];
    kx = ld_row8<VEC>(k + (int64_t)tok * k_stride + e);
    vx = ld_row8<VEC>(v + (int64_t)tok * v_stride + e);
  }
  uint32_t kb, vb;
  const u32x2_t kc = quant_row16(kx, kb);  // every lane is here
  const u32x2_t vc = quant_row16(vx, vb);
  if (slot < 0 || slot >= n_slots) return;
  const int64_t rec = record_off((uint32_t)slot, Hkv, head);
  const int r = (int)(slot & (kPageRows - 1));
  *reinterpret_cast<u32x2_t*>(kp + rec + r * kQuantD + lane16 * 8) = kc;
  *reinterpret_cast<u32x2_t*>(vp + rec + r * kQuantD + lane16 * 8) = vc;
  if (lane16 == 0) {
    kp[rec + kScaleOff + r] = (uint8_t)kb;
    vp[rec + kScaleOff + r] = (uint8_t)vb;
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void kv_quant_load(QUANT_PARAMS) {
  const int L = (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3);
  const int lane16 = threadIdx.x & 15;
  const int row = L * 16 + (threadIdx.x >> 4);
  if (row >= rows) return;
  const int tok = (int)((uint32_t)row / (uint32_t)Hkv);
  const int head = row - tok * Hkv;
  const int64_t slot = slots[tok];
  if (slot < 0 || slot >= n_slots) return;
  const int64_t e = (int64_t)head * kQuantD + lane16 * 8;
  const int64_t rec = record_off((uint32_t)slot, Hkv, head);
  const int r = (int)(slot & (kPageRows - 1));
  const u32x2_t kc = *reinterpret_cast<const u32x2_t*>(kp + rec + r * kQuantD + lane16 * 8);
  const u32x2_t vc = *reinterpret_cast<const u32x2_t*>(vp + rec + r * kQuantD + lane16 * 8);
  const uint32_t kb = kp[rec + kScaleOff + r], vb = vp[rec + kScaleOff + r];
  st_row8<VEC>(k + (int64_t)tok * k_stride + e, dequant8(kc, scale_of(kb)));
  st_row8<VEC>(v + (int64_t)tok * v_stride + e, dequant8(vc, scale_of(vb)));
}

template <bool STORE>
static int kv_quant(const char* name, uint16_t* k, int64_t ks, uint16_t* v, int64_t vs, uint8_t* kp, uint8_t* vp,
                    int64_t num_pages, const int32_t* slot, int n_tok, int Hkv, int D, void* stream) {
  set_error("");
  if (D != kQuantD) return fail(DLLM_ERR_UNSUPPORTED, "%s: head_dim %d not supported (the kernels handle 128)", name, D);
  if (n_tok < 0 || Hkv <= 0 || num_pages < 0 || num_pages > ((int64_t)1 << 23))
    return fail(DLLM_ERR_INVALID_ARG, "%s: bad sizes n_tok=%d Hkv=%d num_pages=%lld (at most 2^23 pages)", name, n_tok,
                Hkv, (long long)num_pages);
  if (n_tok == 0 || num_pages == 0) return DLLM_OK;  // without pages every slot is outside the cache
  if (!k || !v || !kp || !vp || !slot) return fail(DLLM_ERR_INVALID_ARG, "%s: null pointer", name);
  if (ks < (int64_t)Hkv * D || vs < (int64_t)Hkv * D)
    return fail(DLLM_ERR_INVALID_ARG, "%s: token stride (%lld, %lld) smaller than a token row of %lld", name,
                (long long)ks, (long long)vs, (long long)Hkv * D);
  if (!aligned16(kp) || !aligned16(vp)) return fail(DLLM_ERR_INVALID_ARG, "%s: pages must be 16-byte aligned", name);
  // sixteen threads a row, and HIP launches fewer than 2^32
  if ((int64_t)n_tok * Hkv >= ((int64_t)1 << 28) - 128)
    return fail(DLLM_ERR_UNSUPPORTED, "%s: %d tokens of %d KV heads in one call", name, n_tok, Hkv);
  const bool vec = ks % 8 == 0 && vs % 8 == 0 && aligned16(k) && aligned16(v);
  const int rows = n_tok * Hkv;
  const int64_t blocks = ((int64_t)rows + 15) / 16;
  // consecutive workgroups on one XCD: the scale bytes of a page's rows share lines
  const int chunk = (int)((blocks + 7) / 8);
  auto kern = STORE ? (vec ? kv_quant_store<true> : kv_quant_store<false>)
                    : (vec ? kv_quant_load<true> : kv_quant_load<false>);
  kern<<<dim3((unsigned)chunk * 8), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      slot, k, v, rows, Hkv, chunk, ks, vs, kp, vp, num_pages * kPageRows);
  return check_launch(name);
}

}  // namespace dllm

extern "C" size_t dllm_quant_page_bytes(int D) { return D == dllm::kQuantD ? dllm::kRecord : 0; }

extern "C" int dllm_store_kvcache_fp8(const dllm_bf16* key, int64_t key_stride_tok, const dllm_bf16* value,
                                      int64_t value_stride_tok, uint8_t* k_pages, uint8_t* v_pages, int64_t num_pages,
                                      const int32_t* slot_mapping, int n_tok, int Hkv, int D, void* stream) {
  return dllm::kv_quant<true>("dllm_store_kvcache_fp8", const_cast<dllm_bf16*>(key), key_stride_tok,
                              const_cast<dllm_bf16*>(value), value_stride_tok, k_pages, v_pages, num_pages,
                              slot_mapping, n_tok, Hkv, D, stream);
}

extern "C" int dllm_load_kvcache_fp8(dllm_bf16* key, int64_t key_stride_tok, dllm_bf16* value, int64_t value_stride_tok,
                                     const uint8_t* k_pages, const uint8_t* v_pages, int64_t num_pages,
                                     const int32_t* slot_mapping, int n_tok, int Hkv, int D, void* stream) {
  return dllm::kv_quant<false>("dllm_load_kvcache_fp8", key, key_stride_tok, value, value_stride_tok,
                               const_cast<uint8_t*>(k_pages), const_cast<uint8_t*>(v_pages), num_pages, slot_mapping,
                               n_tok, Hkv, D, stream);
}
