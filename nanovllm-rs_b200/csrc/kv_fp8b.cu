// Block-scaled FP8 (e4m3) KV pool: reading rows back, and the attention entry
// point over such a pool.  (The pool is filled by rope_append.cu.)
//
// No counterpart in the reference, whose pool is in the model dtype
// (nanovllm_rs/src/engine/model_runner.rs:286-303).  The format differs from
// the row-scaled e4m3 pool of kv_fp8.cu in its scales: one power of two per 16
// slots and kv head instead of an f32 per row, so scales are 1/16 of the bytes,
// a tile's scales are one 64-byte copy, and scaling is exact everywhere.
#include <algorithm>

#include "common.cuh"

namespace nvkv {
namespace {

constexpr int kBD = 128;  // head_dim
constexpr int kBBlock = NVKV_FP8B_BLOCK;

__device__ __forceinline__ void e4m3x4_f32(uint32_t w, float* f) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const float2 a = DT<__half>::to_f2(lo), b = DT<__half>::to_f2(hi);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

// two values of code * scale in the dtype
template <typename T>
__device__ __forceinline__ uint32_t pack_value(float a, float b) {
  return DT<T>::from_f2(saturate<T>(a), saturate<T>(b));
}

// 8 codes times their scale -> 8 values.
template <typename T>
__device__ __forceinline__ void store_values(T* dst, const uint2 w, float s) {
  float f[8];
  e4m3x4_f32(w.x, f);
  e4m3x4_f32(w.y, f + 4);
  *reinterpret_cast<uint4*>(dst) =
      make_uint4(pack_value<T>(f[0] * s, f[1] * s), pack_value<T>(f[2] * s, f[3] * s),
                 pack_value<T>(f[4] * s, f[5] * s), pack_value<T>(f[6] * s, f[7] * s));
}

// Rows slots[i], bound by HBM: `lanes` (16 or 32) lanes of a warp take one slot's
// K and V rows, 8 codes a lane (8-byte loads, 16-byte stores, both without gaps),
// up to four steps in flight.  16384 slots x 8 heads (100 MB, 15 us of traffic):
// 15.2 us, 17.7 with slots in random order; 28.3 us with a thread per 8 codes and
// 64-bit index divisions, 24.0 us with 16 codes a lane (its 16-byte stores leave gaps).
constexpr int kLoadFlight = 4;
template <typename T>
__global__ void __launch_bounds__(256)
    load_kvcache_fp8b_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                             const float* __restrict__ scale, const int64_t* __restrict__ slots,
                             int64_t n, int hkv, int lanes, int64_t num_slots, int page,
                             T* __restrict__ k_out, T* __restrict__ v_out, int* err) {
  const int lane = threadIdx.x & 31, l = lane & (lanes - 1);
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / lanes);
  const int per = page / kBBlock, chunks = hkv * (kBD / 8);
  const int64_t row = (int64_t)hkv * kBD;
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes; i < n;
       i += step) {
    int64_t slot = slots[i];
    if (slot >= num_slots) {
      if (l == 0) record_error(err, NVKV_DEVERR_SLOT_RANGE);
      slot = -1;
    }
    const int64_t blk = slot / kBBlock, pg = blk / per;
    const float* sc = scale + (pg * hkv * per + (blk - pg * per)) * 2;
    for (int c0 = l; c0 < chunks; c0 += lanes * kLoadFlight) {
      uint2 k[kLoadFlight], v[kLoadFlight];
      float2 s[kLoadFlight];
#pragma unroll
      for (int f = 0; f < kLoadFlight; ++f) {
        const int c = c0 + f * lanes;
        k[f] = v[f] = make_uint2(0, 0);
        s[f] = make_float2(0.f, 0.f);
        if (c < chunks && slot >= 0) {
          k[f] = *reinterpret_cast<const uint2*>(k_cache + slot * row + c * 8);
          v[f] = *reinterpret_cast<const uint2*>(v_cache + slot * row + c * 8);
          s[f] = *reinterpret_cast<const float2*>(sc + (c / (kBD / 8)) * per * 2);
        }
      }
#pragma unroll
      for (int f = 0; f < kLoadFlight; ++f) {
        const int c = c0 + f * lanes;
        if (c < chunks) {
          store_values(k_out + i * row + c * 8, k[f], s[f].x);
          store_values(v_out + i * row + c * 8, v[f], s[f].y);
        }
      }
    }
  }
}

// Dequantises kDeqKeys keys of prompt blockIdx.x into rows cu_kd[b] + j of kbuf /
// vbuf ([rows, Hkv, 128] in the dtype), a key's K and V rows by `lanes` lanes as
// above.
constexpr int kDeqKeys = 32;
template <typename T>
__global__ void __launch_bounds__(256)
    dequant_prompt_fp8b_kernel(const uint8_t* __restrict__ k_cache,
                               const uint8_t* __restrict__ v_cache, const float* __restrict__ scale,
                               const uint32_t* __restrict__ cu_kd,
                               const uint32_t* __restrict__ block_tables, int64_t bt_stride,
                               int64_t num_blocks, int page, int hkv, int lanes,
                               T* __restrict__ kbuf, T* __restrict__ vbuf, int* err) {
  pdl_wait();
  const int b = blockIdx.x;
  const uint32_t ks = cu_kd[b];
  const int len = (int)(cu_kd[b + 1] - ks);
  for (int64_t jj = (int64_t)blockIdx.y * kDeqKeys; jj < len; jj += (int64_t)gridDim.y * kDeqKeys) {
    const int j0 = (int)jj;
    // page_size is a multiple of 128: the keys share a page
    uint32_t pg = block_tables[(int64_t)b * bt_stride + j0 / page];
    if ((int64_t)pg >= num_blocks) {
      if (threadIdx.x == 0) record_error(err, NVKV_DEVERR_BLOCK_RANGE);
      pg = 0;
    }
    const int per = page / kBBlock, off = j0 % page, l = threadIdx.x & (lanes - 1);
    const int n = min(kDeqKeys, len - j0), chunks = hkv * (kBD / 8);
    const int64_t row = (int64_t)hkv * kBD;
    for (int j = threadIdx.x / lanes; j < n; j += blockDim.x / lanes) {
      const int64_t src = ((int64_t)pg * page + off + j) * row, dst = (int64_t)(ks + j0 + j) * row;
      const float* sc = scale + ((int64_t)pg * hkv * per + (off + j) / kBBlock) * 2;
      for (int c0 = l; c0 < chunks; c0 += lanes * kLoadFlight) {
        uint2 k[kLoadFlight], v[kLoadFlight];
        float2 s[kLoadFlight];
#pragma unroll
        for (int f = 0; f < kLoadFlight; ++f) {
          const int c = c0 + f * lanes;
          if (c < chunks) {
            k[f] = *reinterpret_cast<const uint2*>(k_cache + src + c * 8);
            v[f] = *reinterpret_cast<const uint2*>(v_cache + src + c * 8);
            s[f] = *reinterpret_cast<const float2*>(sc + (c / (kBD / 8)) * per * 2);
          }
        }
#pragma unroll
        for (int f = 0; f < kLoadFlight; ++f) {
          const int c = c0 + f * lanes;
          if (c < chunks) {
            store_values(kbuf + dst + c * 8, k[f], s[f].x);
            store_values(vbuf + dst + c * 8, v[f], s[f].y);
          }
        }
      }
    }
  }
}

// Query rows a sequence may have on the decode kernel: all sequences of a batch
// whose longest fits, else single rows only.
int short_rows(int hq, int hkv, int max_q) {
  return (int64_t)max_q * (hq / hkv) <= kFp8bMaxRows ? max_q : 1;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Workspace: the decode kernel's partials and, at the same place (it is done
// with them by then), the prefill kernel's region; for prompts then cu_kd
// [num_seqs + 1] and their dequantised K and V rows.
struct Layout {
  size_t base, cu_kd, kbuf, vbuf, total;
};
Layout layout(int num_seqs, int hq, int hkv, int max_q, int max_k, int64_t prompt_rows) {
  Layout L = {0, 0, 0, 0, 0};
  if (num_seqs <= 0 || max_q <= 0) return L;
  const int cap = short_rows(hq, hkv, max_q);
  L.base = decode_fp8b_bytes(hq, hkv, cap);
  L.total = L.base;
  if (cap == max_q) return L;
  L.base = std::max(L.base, attention_workspace_bytes(num_seqs, hq, hkv, max_q, max_k));
  L.cu_kd = align256(L.base);
  L.kbuf = align256(L.cu_kd + ((size_t)num_seqs + 1) * 4);
  const size_t rows = (size_t)prompt_rows * hkv * kBD * 2;
  L.vbuf = align256(L.kbuf + rows);
  L.total = L.vbuf + rows;
  return L;
}

}  // namespace
}  // namespace nvkv

extern "C" int nvkv_load_kvcache_fp8b(const void* k_cache, const void* v_cache,
                                      const float* kv_scale, const int64_t* slots,
                                      int64_t num_slots, int num_kv_heads, int head_dim,
                                      int64_t num_blocks, int page_size, void* k_out, void* v_out,
                                      int dtype, nvkv_stream_t stream) {
  NVKV_RANGE("nvkv_load_kvcache_fp8b");
  using namespace nvkv;
  clear_error();
  if (dtype != NVKV_DTYPE_BF16 && dtype != NVKV_DTYPE_F16)
    return set_error(NVKV_ERR_UNSUPPORTED, "load_kvcache_fp8b: output dtype must be bf16/f16");
  if (head_dim != kBD) return set_error(NVKV_ERR_UNSUPPORTED, "load_kvcache_fp8b: head_dim 128");
  if (num_slots < 0 || num_kv_heads <= 0 || num_kv_heads > 65536 || num_blocks <= 0 ||
      page_size <= 0 || num_blocks > INT64_MAX / page_size / ((int64_t)num_kv_heads * kBD))
    return set_error(NVKV_ERR_INVALID_ARG, "load_kvcache_fp8b: bad sizes");
  if (page_size % kBBlock)
    return set_error(NVKV_ERR_UNSUPPORTED, "load_kvcache_fp8b: page_size must be a multiple of 16");
  if (num_slots == 0) return NVKV_OK;
  if (!k_cache || !v_cache || !kv_scale || !slots || !k_out || !v_out)
    return set_error(NVKV_ERR_INVALID_ARG, "load_kvcache_fp8b: null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out) ||
      ((uintptr_t)kv_scale & 7u) || ((uintptr_t)slots & 7u))
    return set_error(NVKV_ERR_ALIGNMENT,
                     "load_kvcache_fp8b: caches and outputs 16-byte, scales and slots 8-byte aligned");
  const uint64_t out_bytes = (uint64_t)num_slots * num_kv_heads * kBD * 2;
  const uint64_t pool = (uint64_t)num_blocks * page_size * num_kv_heads * kBD;
  bool meet = spans_meet(k_out, out_bytes, v_out, out_bytes);
  for (const void* o : {k_out, v_out})
    meet |= spans_meet(o, out_bytes, k_cache, pool) || spans_meet(o, out_bytes, v_cache, pool) ||
            spans_meet(o, out_bytes, kv_scale, pool / (kBBlock * kBD) * 8) ||
            spans_meet(o, out_bytes, slots, (uint64_t)num_slots * 8);
  if (meet)
    return set_error(NVKV_ERR_INVALID_ARG,
                     "load_kvcache_fp8b: an output overlaps another, the pool or the slots");
  const int lanes = num_kv_heads == 1 ? 16 : 32;  // 16 chunks of 8 codes a head
  const int64_t rows = 256 / lanes;                // a CTA's
  const unsigned blocks = (unsigned)std::min<int64_t>((num_slots + rows - 1) / rows, 148 * 16);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const auto* k = static_cast<const uint8_t*>(k_cache);
  const auto* v = static_cast<const uint8_t*>(v_cache);
  int* err = device_error_word();
  if (dtype == NVKV_DTYPE_BF16)
    load_kvcache_fp8b_kernel<<<blocks, 256, 0, s>>>(
        k, v, kv_scale, slots, num_slots, num_kv_heads, lanes, num_blocks * page_size, page_size,
        static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), err);
  else
    load_kvcache_fp8b_kernel<<<blocks, 256, 0, s>>>(
        k, v, kv_scale, slots, num_slots, num_kv_heads, lanes, num_blocks * page_size, page_size,
        static_cast<__half*>(k_out), static_cast<__half*>(v_out), err);
  return check_cuda(cudaGetLastError(), "load_kvcache_fp8b launch");
}

extern "C" int nvkv_paged_attention_fp8b_workspace_size(int num_seqs, int num_q_heads,
                                                        int num_kv_heads, int head_dim,
                                                        int max_seqlen_q, int max_seqlen_k,
                                                        int64_t prompt_kv_tokens, size_t* bytes) {
  using namespace nvkv;
  clear_error();
  if (!bytes) return set_error(NVKV_ERR_INVALID_ARG, "fp8b workspace_size: null output");
  int rc = validate_shapes(num_seqs, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads,
                           head_dim);
  if (rc) return rc;
  if (prompt_kv_tokens < 0 || prompt_kv_tokens > 0x7fffffffLL)
    return set_error(NVKV_ERR_INVALID_ARG, "fp8b workspace_size: bad prompt_kv_tokens");
  *bytes = layout(num_seqs, num_q_heads, num_kv_heads, max_seqlen_q, max_seqlen_k,
                  prompt_kv_tokens)
               .total;
  return NVKV_OK;
}

extern "C" int nvkv_paged_attention_fp8b(
    const void* q, int64_t q_stride, int64_t num_q_tokens, const void* k_cache,
    const void* v_cache, const float* kv_scale, int64_t num_blocks, void* out,
    const uint32_t* cu_seqlens_q, const uint32_t* cu_seqlens_k, const uint32_t* block_tables,
    int64_t block_table_stride, int num_seqs, int max_seqlen_q, int max_seqlen_k,
    int num_q_heads, int num_kv_heads, int head_dim, int page_size, float softmax_scale,
    int causal, int64_t prompt_kv_tokens, void* workspace, size_t workspace_bytes, int dtype,
    nvkv_stream_t stream) {
  NVKV_RANGE("nvkv_paged_attention_fp8b");
  using namespace nvkv;
  clear_error();
  if (dtype != NVKV_DTYPE_BF16 && dtype != NVKV_DTYPE_F16)
    return set_error(NVKV_ERR_UNSUPPORTED, "paged_attention_fp8b: q/out dtype must be bf16/f16");
  int rc = validate_shapes(num_seqs, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads,
                           head_dim);
  if (rc) return rc;
  if (num_q_tokens < 0 || num_q_tokens > 0x7fffffffLL || prompt_kv_tokens < 0 ||
      prompt_kv_tokens > 0x7fffffffLL)
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: bad num_q_tokens / prompt rows");
  if (num_seqs == 0 || max_seqlen_q == 0 || num_q_tokens == 0) return NVKV_OK;
  if (!q || !k_cache || !v_cache || !kv_scale || !out || !cu_seqlens_q || !cu_seqlens_k ||
      !block_tables)
    return set_error(NVKV_ERR_INVALID_ARG,
                     "paged_attention_fp8b: null pointer (the pool is paged: block_tables)");
  if (num_blocks <= 0 || page_size <= 0 || page_size % 128 != 0)
    return set_error(NVKV_ERR_UNSUPPORTED,
                     "paged_attention_fp8b: page_size must be a positive multiple of 128");
  if (block_table_stride < ((int64_t)max_seqlen_k + page_size - 1) / page_size)
    return set_error(NVKV_ERR_INVALID_ARG,
                     "paged_attention_fp8b: block_table_stride < blocks needed by max_seqlen_k");
  if (num_blocks > 0x7fffffffLL / page_size || max_seqlen_k > 1 << 30)
    return set_error(NVKV_ERR_UNSUPPORTED,
                     "paged_attention_fp8b: more than 2^31 cache rows or 2^30 keys a sequence");
  if (q_stride < (int64_t)num_q_heads * head_dim || q_stride % 8 != 0 || !aligned16(q) ||
      !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(kv_scale))
    return set_error(NVKV_ERR_ALIGNMENT, "paged_attention_fp8b: misaligned buffer or stride");
  if (((uintptr_t)cu_seqlens_q | (uintptr_t)cu_seqlens_k | (uintptr_t)block_tables) & 3u)
    return set_error(NVKV_ERR_ALIGNMENT, "paged_attention_fp8b: metadata must be 4-byte aligned");
  if (!(softmax_scale > 0.f) || softmax_scale > 3e38f)
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: softmax_scale must be > 0");
  const int64_t q_row = (int64_t)num_q_heads * head_dim;
  if (rows_clash(q, q_stride, q_row, out, q_row, q_row, num_q_tokens))
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: out overlaps q without being it");
  const int cap = short_rows(num_q_heads, num_kv_heads, max_seqlen_q);
  const bool prompts = cap < max_seqlen_q;
  if (prompts && prompt_kv_tokens == 0)
    return set_error(NVKV_ERR_INVALID_ARG,
                     "paged_attention_fp8b: max_seqlen_q * Hq / Hkv > 32 needs prompt_kv_tokens >= "
                     "the prompts' total k_len");
  const Layout L = layout(num_seqs, num_q_heads, num_kv_heads, max_seqlen_q, max_seqlen_k,
                          prompt_kv_tokens);
  if (L.total > 0 && (!workspace || workspace_bytes < L.total || !aligned16(workspace)))
    return set_error(NVKV_ERR_WORKSPACE, "paged_attention_fp8b: workspace missing or too small "
                                         "(need " + std::to_string(L.total) + " bytes)");
  const uint64_t pool = (uint64_t)num_blocks * page_size * num_kv_heads * kBD;
  const uint64_t cu_bytes = ((uint64_t)num_seqs + 1) * 4, out_bytes = (uint64_t)num_q_tokens * q_row * 2;
  const Span kc = {k_cache, pool}, vc = {v_cache, pool}, sc = {kv_scale, pool / (kBBlock * kBD) * 8};
  const Span cq = {cu_seqlens_q, cu_bytes}, ck = {cu_seqlens_k, cu_bytes};
  const Span bt = {block_tables, ((uint64_t)(num_seqs - 1) * block_table_stride +
                                  ((int64_t)max_seqlen_k + page_size - 1) / page_size) * 4};
  if (spans_meet(out, out_bytes, {kc, vc, sc, cq, ck, bt}))
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: out overlaps the pool or metadata");
  if (spans_meet(workspace, L.total,
                 {{q, (uint64_t)((num_q_tokens - 1) * q_stride + q_row) * 2}, {out, out_bytes}, kc, vc,
                  sc, cq, ck, bt}))
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: the workspace overlaps a buffer");
  AttnArgs a;
  a.q = q;
  a.q_stride = q_stride;
  a.num_q_rows = num_q_tokens;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.num_blocks = num_blocks;
  a.kv_stride = (int64_t)num_kv_heads * head_dim;  // one byte a code
  a.out = out;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.num_seqs = num_seqs;
  a.max_q = max_seqlen_q;
  a.max_k = max_seqlen_k;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.d = head_dim;
  a.page = page_size;
  a.scale = softmax_scale;
  a.causal = causal ? 1 : 0;
  a.ws = workspace;
  a.ws_bytes = workspace_bytes;
  a.dtype = dtype;
  a.stream = reinterpret_cast<cudaStream_t>(stream);
  a.k_scale = kv_scale;
  if (!prompts) return launch_decode_fp8b(a, cap, true);
  // single rows on the decode kernel; the others' keys are dequantised (their row
  // offsets come first, beside the decode grid) for the contiguous prefill
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint32_t* cu_kd = reinterpret_cast<uint32_t*>(ws + L.cu_kd);
  rc = launch_prompt_rows(cu_seqlens_q, cu_seqlens_k, num_seqs, max_seqlen_k, prompt_kv_tokens,
                          cu_kd, a.stream);
  if (!rc) rc = launch_decode_fp8b(a, cap, false);
  if (rc) return rc;
  const dim3 grid((unsigned)num_seqs,
                  (unsigned)std::min(65535, (max_seqlen_k - 1) / kDeqKeys + 1));
  const int lanes = num_kv_heads == 1 ? 16 : 32;
  const auto* k8 = static_cast<const uint8_t*>(k_cache);
  const auto* v8 = static_cast<const uint8_t*>(v_cache);
  int* err = device_error_word();
  if (dtype == NVKV_DTYPE_BF16)
    rc = launch_pdl(dequant_prompt_fp8b_kernel<__nv_bfloat16>, grid, dim3(256), 0, a.stream,
                    "fp8b dequant launch", k8, v8, kv_scale, (const uint32_t*)cu_kd, block_tables,
                    block_table_stride, num_blocks, page_size, num_kv_heads, lanes,
                    reinterpret_cast<__nv_bfloat16*>(ws + L.kbuf),
                    reinterpret_cast<__nv_bfloat16*>(ws + L.vbuf), err);
  else
    rc = launch_pdl(dequant_prompt_fp8b_kernel<__half>, grid, dim3(256), 0, a.stream,
                    "fp8b dequant launch", k8, v8, kv_scale, (const uint32_t*)cu_kd, block_tables,
                    block_table_stride, num_blocks, page_size, num_kv_heads, lanes,
                    reinterpret_cast<__half*>(ws + L.kbuf), reinterpret_cast<__half*>(ws + L.vbuf),
                    err);
  if (rc) return rc;
  AttnArgs c = a;
  c.k_cache = ws + L.kbuf;
  c.v_cache = ws + L.vbuf;
  c.k_scale = nullptr;
  c.block_tables = nullptr;
  c.bt_stride = 0;
  c.num_blocks = prompt_kv_tokens;
  c.cu_k = cu_kd;
  return launch_paged_prefill(c);
}
