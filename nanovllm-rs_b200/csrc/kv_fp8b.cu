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

// two values of code * scale in the dtype; f16 saturates (a code's rounding may
// have carried a value past 65504)
template <typename T>
__device__ __forceinline__ uint32_t pack_value(float a, float b) {
  if (std::is_same<T, __half>::value) {
    a = a != a ? a : fminf(fmaxf(a, -65504.f), 65504.f);
    b = b != b ? b : fminf(fmaxf(b, -65504.f), 65504.f);
  }
  return DT<T>::from_f2(a, b);
}

// Rows slots[i]: a thread takes 8 codes (8-byte load, 16-byte store).
template <typename T>
__global__ void __launch_bounds__(256)
    load_kvcache_fp8b_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                             const float* __restrict__ scale, const int64_t* __restrict__ slots,
                             int64_t n, int hkv, int64_t num_slots, int page, T* __restrict__ k_out,
                             T* __restrict__ v_out, int* err) {
  const int per_row = hkv * (kBD / 8);
  const int64_t total = n * per_row * 2;
  const int per = page / kBBlock;
  for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < total;
       u += (int64_t)gridDim.x * blockDim.x) {
    const int64_t kvrow = u / per_row;
    const int c = (int)(u - kvrow * per_row);
    const int kv = (int)(kvrow & 1);
    const int64_t i = kvrow >> 1;
    const int64_t slot = slots[i];
    const int h = c / (kBD / 8);
    uint4 o = make_uint4(0, 0, 0, 0);
    if (slot >= num_slots) {
      if (c == 0) record_error(err, NVKV_DEVERR_SLOT_RANGE);
    } else if (slot >= 0) {
      const uint2 w = *reinterpret_cast<const uint2*>((kv ? v_cache : k_cache) +
                                                      slot * hkv * kBD + (int64_t)c * 8);
      const int64_t blk = slot / kBBlock;
      const float s = scale[(((blk / per) * hkv + h) * per + blk % per) * 2 + kv];
      float f[8];
      e4m3x4_f32(w.x, f);
      e4m3x4_f32(w.y, f + 4);
      o = make_uint4(pack_value<T>(f[0] * s, f[1] * s), pack_value<T>(f[2] * s, f[3] * s),
                     pack_value<T>(f[4] * s, f[5] * s), pack_value<T>(f[6] * s, f[7] * s));
    }
    *reinterpret_cast<uint4*>((kv ? v_out : k_out) + (i * per_row + c) * 8) = o;
  }
}

// Attention, the plain way: a CTA per (query row, kv head), its four warps over
// the keys, f32 online softmax, one query head after the other.
struct SimpleParams {
  const void* q;
  int64_t q_stride, num_q_rows;
  const uint8_t *k, *v;
  const float* scale;
  void* out;
  const uint32_t *cu_q, *cu_k, *bt;
  int64_t bt_stride, num_blocks;
  int num_seqs, max_k, hq, hkv, page, causal;
  float sm;
  int* err;
};

template <typename T>
__global__ void __launch_bounds__(128) attend_fp8b_kernel(const SimpleParams p) {
  __shared__ float so[4][kBD], sm_m[4], sm_l[4];
  const uint32_t row = blockIdx.x;
  const int kvh = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = p.num_seqs;  // the sequence of this row: cu_q[lo] <= row < cu_q[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.cu_q[mid] <= row) lo = mid;
    else hi = mid;
  }
  const uint32_t q0 = p.cu_q[lo], q1 = p.cu_q[lo + 1];
  if (row < q0 || row >= q1) return;
  const int q_len = (int)(q1 - q0), k_len = (int)(p.cu_k[lo + 1] - p.cu_k[lo]);
  const bool bad = k_len > p.max_k || (int64_t)q1 > p.num_q_rows || (q_len > 1 && k_len < q_len);
  if (bad || k_len <= 0) {
    if (threadIdx.x == 0) record_error(p.err, NVKV_DEVERR_SEQLEN);
    if (bad) return;
  }
  const int see = p.causal ? min(k_len, (int)(row - q0) + k_len - q_len + 1) : k_len;
  const int g = p.hq / p.hkv, per = p.page / kBBlock;
  for (int h = 0; h < g; ++h) {
    const T* qr = static_cast<const T*>(p.q) + row * p.q_stride + (int64_t)(kvh * g + h) * kBD;
    const uint2 raw = *reinterpret_cast<const uint2*>(qr + 4 * lane);
    const float2 qa = DT<T>::to_f2(raw.x), qb = DT<T>::to_f2(raw.y);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = warp; j < see; j += 4) {
      uint32_t pg = p.bt[lo * p.bt_stride + j / p.page];
      if ((int64_t)pg >= p.num_blocks) {
        if (lane == 0) record_error(p.err, NVKV_DEVERR_BLOCK_RANGE);
        pg = 0;
      }
      const int off = j % p.page;
      const int64_t at = (((int64_t)pg * p.page + off) * p.hkv + kvh) * kBD + 4 * lane;
      const float2 s2 = *reinterpret_cast<const float2*>(
          p.scale + (((int64_t)pg * p.hkv + kvh) * per + off / kBBlock) * 2);
      float kf[4], vf[4];
      e4m3x4_f32(*reinterpret_cast<const uint32_t*>(p.k + at), kf);
      e4m3x4_f32(*reinterpret_cast<const uint32_t*>(p.v + at), vf);
      float s = qa.x * kf[0] + qa.y * kf[1] + qb.x * kf[2] + qb.y * kf[3];
#pragma unroll
      for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= s2.x * p.sm;
      const float mn = fmaxf(m, s);
      const float al = exp2f(m - mn), e = exp2f(s - mn);
      m = mn;
      l = l * al + e;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = o[i] * al + e * (vf[i] * s2.y);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) so[warp][4 * lane + i] = o[i];
    if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
    __syncthreads();
    float mx = -INFINITY;
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm_m[w]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float acc = 0.f, ls = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(sm_m[w] - mu);
      acc += so[w][threadIdx.x] * f;
      ls += sm_l[w] * f;
    }
    static_cast<T*>(p.out)[((int64_t)row * p.hq + kvh * g + h) * kBD + threadIdx.x] =
        DT<T>::from_f(ls == 0.f ? 0.f : acc / ls);
  }
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
      page_size <= 0)
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
  const int64_t units = num_slots * num_kv_heads * (kBD / 8) * 2;
  const unsigned blocks = (unsigned)std::min<int64_t>((units + 255) / 256, 148 * 8 * 4);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const auto* k = static_cast<const uint8_t*>(k_cache);
  const auto* v = static_cast<const uint8_t*>(v_cache);
  int* err = device_error_word();
  if (dtype == NVKV_DTYPE_BF16)
    load_kvcache_fp8b_kernel<<<blocks, 256, 0, s>>>(
        k, v, kv_scale, slots, num_slots, num_kv_heads, num_blocks * page_size, page_size,
        static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), err);
  else
    load_kvcache_fp8b_kernel<<<blocks, 256, 0, s>>>(
        k, v, kv_scale, slots, num_slots, num_kv_heads, num_blocks * page_size, page_size,
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
  *bytes = 0;
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
  if (num_blocks > 0x7fffffffLL / page_size)
    return set_error(NVKV_ERR_UNSUPPORTED, "paged_attention_fp8b: more than 2^31 cache rows");
  if (q_stride < (int64_t)num_q_heads * head_dim || q_stride % 8 != 0 || !aligned16(q) ||
      !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(kv_scale))
    return set_error(NVKV_ERR_ALIGNMENT, "paged_attention_fp8b: misaligned buffer or stride");
  if (((uintptr_t)cu_seqlens_q | (uintptr_t)cu_seqlens_k | (uintptr_t)block_tables) & 3u)
    return set_error(NVKV_ERR_ALIGNMENT, "paged_attention_fp8b: metadata must be 4-byte aligned");
  if (!(softmax_scale > 0.f) || softmax_scale > 3e38f)
    return set_error(NVKV_ERR_INVALID_ARG, "paged_attention_fp8b: softmax_scale must be > 0");
  SimpleParams p;
  p.q = q;
  p.q_stride = q_stride;
  p.num_q_rows = num_q_tokens;
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.scale = kv_scale;
  p.out = out;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.bt = block_tables;
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.num_seqs = num_seqs;
  p.max_k = max_seqlen_k;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.page = page_size;
  p.causal = causal ? 1 : 0;
  p.sm = softmax_scale * 1.4426950408889634f;
  p.err = device_error_word();
  const dim3 grid((unsigned)num_q_tokens, (unsigned)num_kv_heads);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVKV_DTYPE_BF16) attend_fp8b_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else attend_fp8b_kernel<__half><<<grid, 128, 0, s>>>(p);
  return check_cuda(cudaGetLastError(), "paged_attention_fp8b launch");
}
