// Append to a paged KV cache with the rotation on the way (nvkv_rope_append):
// per-head RMSNorm (optional), rotary positions, and the store of K and V into
// the model-dtype pool or the block-scaled e4m3 pool, in one launch.
//
// Mathematics (fp8b pool).  With the rows x of a block of 16 slots and one kv
// head (K and V apart): e = max(e_kept, least e >= -100 with amax <= 448 2^e),
// code = e4m3(x 2^-e); rows that the block already held move by code' =
// e4m3(code 2^(e_kept - e)).  K is normalised and rotated in f64 and reaches
// e4m3 by ONE rounding (to f32 by rounding to odd, which the conversion to four
// significant bits cannot tell from the exact value), so the codes are a
// function of the formulas and not of the f32 arithmetic's order, and tests
// compare them bit by bit.  q and the dtype pool use f32 and round once.
//
// Layout.  A CTA of 8 warps owns a window of W tokens: the cos / sin of those
// tokens (and of the up to 15 that follow in the last one's block) go to shared
// memory once; then warps take q rows (one per warp, lane l holds dims 4l ..
// 4l + 3, pair partners meet by a shuffle) and K / V units.  A unit is one run
// (the call's tokens of one block), one kv head, K or V: the warp holds all of
// its up to 16 rows in registers (64 values a lane), so the maximum, the scale
// and the codes come from one read.  The run belongs to the window of its first
// token.  W = 1 for a decode step (a CTA per token: latency), up to 16 for
// prompts.  Bound by HBM for prompts (read qkv, write q and codes).
#include <algorithm>
#include <type_traits>

#include "rope_angle.cuh"

namespace nvkv {
namespace {

constexpr int kApD = 128;
constexpr int kApBlock = NVKV_FP8B_BLOCK;
constexpr int kApThreads = 256;
constexpr int kApWarps = kApThreads / 32;
constexpr int kApMaxWindow = 16;
constexpr int kApTable = kApMaxWindow + kApBlock - 1;  // tokens a table can hold
constexpr int kApMinE = -100;

struct AppendParams {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  int64_t num_tokens;
  int hq, hkv, half, inter, window;
  const int64_t* positions;
  const double* inv_freq;
  double a;
  const void *q_w, *k_w;
  float eps;
  void* q_out;
  void *k_cache, *v_cache;
  float* scale;
  const int64_t* slots;
  int64_t num_slots;
  int page;
  int* err;
};

// f64 -> f32 rounded to odd: toward zero, the last bit set if anything was cut.
__device__ __forceinline__ float f32_odd(double x) {
  const float f = __double2float_rz(x);
  return (double)f == x || x != x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// least e >= -100 with amax <= 448 * 2^e = 1.75 * 2^(e + 8)
__device__ __forceinline__ int block_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return max(kApMinE, (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u));
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ void e4m3x4_f32(uint32_t w, float* f) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const float2 a = DT<__half>::to_f2(lo), b = DT<__half>::to_f2(hi);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

template <typename R>
struct CS;
template <>
struct CS<float> {
  using V = float2;
};
template <>
struct CS<double> {
  using V = double2;
};

// Lane l's four dims 4l .. 4l + 3 of one head row, normalised (w != null) and
// rotated by the table row cs, in R arithmetic.  Full warp.
template <typename T, typename R, typename C>
__device__ __forceinline__ void norm_rotate(const uint2 raw, const T* w, float eps, const C* cs,
                                            int half, bool inter, int lane, R (&x)[4]) {
  const float2 p0 = DT<T>::to_f2(raw.x), p1 = DT<T>::to_f2(raw.y);
  x[0] = p0.x, x[1] = p0.y, x[2] = p1.x, x[3] = p1.y;
  if (w) {
    R ss = (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    const R inv = (R)1 / sqrt(ss / (R)kApD + (R)eps);
    const uint2 wr = *reinterpret_cast<const uint2*>(w + 4 * lane);
    const float2 w0 = DT<T>::to_f2(wr.x), w1 = DT<T>::to_f2(wr.y);
    x[0] = x[0] * inv * (R)w0.x;
    x[1] = x[1] * inv * (R)w0.y;
    x[2] = x[2] * inv * (R)w1.x;
    x[3] = x[3] * inv * (R)w1.y;
  }
  if (inter) {
    if (4 * lane < 2 * half) {
      const C c0 = cs[2 * lane], c1 = cs[2 * lane + 1];
      const R a = x[0], b = x[2];
      x[0] = a * (R)c0.x - x[1] * (R)c0.y;
      x[1] = x[1] * (R)c0.x + a * (R)c0.y;
      x[2] = b * (R)c1.x - x[3] * (R)c1.y;
      x[3] = x[3] * (R)c1.x + b * (R)c1.y;
    }
  } else {
    const int step = half >> 2;  // lanes between a pair's halves
    const bool lo = lane < step, in = lane < 2 * step;
    const int peer = lo ? lane + step : in ? lane - step : lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const R y = __shfl_sync(0xffffffffu, x[i], peer);
      if (in) {
        const C c = cs[4 * (lo ? lane : peer) + i];
        x[i] = lo ? x[i] * (R)c.x - y * (R)c.y : x[i] * (R)c.x + y * (R)c.y;
      }
    }
  }
}

template <typename T, bool kF8>
__global__ void __launch_bounds__(kApThreads) rope_append_kernel(const AppendParams p) {
  using R = typename std::conditional<kF8, double, float>::type;  // K's arithmetic
  using C = typename CS<R>::V;
  extern __shared__ __align__(16) uint8_t smem[];
  C* cs = reinterpret_cast<C*>(smem);  // [table tokens][half]
  __shared__ int64_t slot_s[kApTable + 1];  // slots of tokens w0 - 1 ..
  __shared__ int lead_s[kApMaxWindow], len_s[kApMaxWindow], nrun_s, ntab_s;
  const int64_t w0 = (int64_t)blockIdx.x * p.window;
  const int n = (int)min((int64_t)p.window, p.num_tokens - w0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // no memory access before this: the launch may overlap the kernel before it
  pdl_wait();
  if (warp == 0) {
    const int64_t t = w0 - 1 + lane;  // lane 0: the token before the window
    int64_t s = -1;
    if (t >= 0 && t < p.num_tokens && lane <= n + kApBlock - 1) {
      s = p.slots[t];
      if (s >= p.num_slots) {
        if (lane >= 1 && lane <= n) record_error(p.err, NVKV_DEVERR_SLOT_RANGE);
        s = -1;
      }
    }
    slot_s[lane] = s;
    if (kF8) {
      const int64_t before = __shfl_up_sync(0xffffffffu, s, 1);
      const bool same = lane > 0 && s >= 0 && before >= 0 && s / kApBlock == before / kApBlock;
      const bool bad = same && s <= before;
      const uint32_t joins = __ballot_sync(0xffffffffu, same && !bad);  // continues a run
      const bool in = lane >= 1 && lane <= n;
      if (bad && in) record_error(p.err, NVKV_DEVERR_SLOT_ORDER);
      const uint32_t leads = __ballot_sync(0xffffffffu, in && s >= 0 && !same);
      // tokens from here on that continue this lane's run
      const uint32_t after = lane < 31 ? ~(joins >> (lane + 1)) : ~0u;
      const int len = 1 + (__ffs(after) - 1);
      if (leads >> lane & 1) {
        const int r = __popc(leads & ((1u << lane) - 1));
        lead_s[r] = lane - 1;
        len_s[r] = len;
      }
      const int last = leads ? 31 - __clz(leads) : 0;
      const int end = last ? __shfl_sync(0xffffffffu, lane - 1 + len, last) : 0;
      if (lane == 0) {
        nrun_s = __popc(leads);
        ntab_s = max(n, end);
      }
    } else if (lane == 0) {
      nrun_s = 0;
      ntab_s = n;
    }
  }
  __syncthreads();
  const int ntab = ntab_s;
  for (int i = tid; i < ntab * p.half; i += kApThreads) {
    const int64_t pos = p.positions[w0 + i / p.half];
    const double f = p.inv_freq[i % p.half];
    if constexpr (kF8) cs[i] = rope_cs64(pos, f, p.a);
    else cs[i] = rope_cs(pos, f, (float)p.a);
  }
  __syncthreads();

  const bool inter = p.inter != 0;
  // q rows
  const T* qw = static_cast<const T*>(p.q_w);
  const T* kw = static_cast<const T*>(p.k_w);
  for (int u = warp; u < n * p.hq; u += kApWarps) {
    const int t = u / p.hq, h = u % p.hq;
    const T* src = static_cast<const T*>(p.q) + (w0 + t) * p.q_stride + (int64_t)h * kApD;
    float x[4];
    norm_rotate<T>(*reinterpret_cast<const uint2*>(src + 4 * lane), qw, p.eps, cs + t * p.half,
                   p.half, inter, lane, x);
    T* dst = static_cast<T*>(p.q_out) + ((w0 + t) * p.hq + h) * kApD;
    *reinterpret_cast<uint2*>(dst + 4 * lane) =
        make_uint2(DT<T>::from_f2(x[0], x[1]), DT<T>::from_f2(x[2], x[3]));
  }

  if constexpr (!kF8) {
    for (int u = warp; u < n * p.hkv * 2; u += kApWarps) {
      const int kv = u & 1, t = (u >> 1) / p.hkv, h = (u >> 1) % p.hkv;
      const int64_t slot = slot_s[t + 1];
      if (slot < 0) continue;
      const T* src = kv ? static_cast<const T*>(p.v) + (w0 + t) * p.v_stride
                        : static_cast<const T*>(p.k) + (w0 + t) * p.k_stride;
      uint2 raw = *reinterpret_cast<const uint2*>(src + (int64_t)h * kApD + 4 * lane);
      if (!kv) {
        float x[4];
        norm_rotate<T>(raw, kw, p.eps, cs + t * p.half, p.half, inter, lane, x);
        raw = make_uint2(DT<T>::from_f2(x[0], x[1]), DT<T>::from_f2(x[2], x[3]));
      }
      T* dst = static_cast<T*>(kv ? p.v_cache : p.k_cache) + (slot * p.hkv + h) * kApD;
      *reinterpret_cast<uint2*>(dst + 4 * lane) = raw;
    }
  } else {
    for (int u = warp; u < nrun_s * p.hkv * 2; u += kApWarps) {
      const int kv = u & 1, r = (u >> 1) / p.hkv, h = (u >> 1) % p.hkv;
      const int t = lead_s[r], len = len_s[r];
      const int64_t slot0 = slot_s[t + 1];
      const int64_t blk = slot0 / kApBlock;
      const int low = (int)(slot0 % kApBlock);
      const int per = p.page / kApBlock;
      float* sp = p.scale + (((blk / per) * p.hkv + h) * per + blk % per) * 2 + kv;
      const float old = low ? *sp : 0.f;
      const T* src = (kv ? static_cast<const T*>(p.v) + (w0 + t) * p.v_stride
                         : static_cast<const T*>(p.k) + (w0 + t) * p.k_stride) +
                     (int64_t)h * kApD + 4 * lane;
      const int64_t stride = kv ? p.v_stride : p.k_stride;
      float x[kApBlock][4];
      uint2 raw[kApBlock];
#pragma unroll
      for (int j = 0; j < kApBlock; ++j)
        if (j < len) raw[j] = *reinterpret_cast<const uint2*>(src + j * stride);
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < kApBlock; ++j) {
        if (j < len) {
          if (kv) {
            const float2 a = DT<T>::to_f2(raw[j].x), b = DT<T>::to_f2(raw[j].y);
            x[j][0] = a.x, x[j][1] = a.y, x[j][2] = b.x, x[j][3] = b.y;
          } else {
            R y[4];
            norm_rotate<T>(raw[j], kw, p.eps, cs + (t + j) * p.half, p.half, inter, lane, y);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = f32_odd(y[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float m = fabsf(x[j][i]);
            amax = fmaxf(amax, m < INFINITY ? m : 0.f);
          }
        }
      }
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) amax = warp_max_xor(amax, m);
      const int e_old = max(kApMinE, (int)(__float_as_uint(old) >> 23 & 0xffu) - 127);
      int e = block_exp(amax);
      if (low) e = max(e, e_old);
      const float inv = pow2i(-e);
      uint8_t* cache = static_cast<uint8_t*>(kv ? p.v_cache : p.k_cache);
      uint8_t* base = cache + (blk * kApBlock * p.hkv + h) * kApD + 4 * lane;
      const int64_t row = (int64_t)p.hkv * kApD;
#pragma unroll
      for (int j = 0; j < kApBlock; ++j)
        if (j < len)
          *reinterpret_cast<uint32_t*>(base + (slot_s[t + 1 + j] % kApBlock) * row) =
              e4m3x4(x[j][0] * inv, x[j][1] * inv, x[j][2] * inv, x[j][3] * inv);
      if (e > e_old && low) {  // the kept rows move to the larger scale
        const float f = pow2i(max(e_old - e, -126));
        for (int j = 0; j < low; ++j) {
          uint32_t* c = reinterpret_cast<uint32_t*>(base + j * row);
          float y[4];
          e4m3x4_f32(*c, y);
          *c = e4m3x4(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
        }
      }
      if (lane == 0 && (!low || e > e_old)) *sp = pow2i(e);
    }
  }
}

}  // namespace
}  // namespace nvkv

extern "C" int nvkv_rope_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                const void* v, int64_t v_stride, int64_t num_tokens,
                                int num_q_heads, int num_kv_heads, int head_dim,
                                const int64_t* positions, const double* inv_freq, int rot_dim,
                                double attn_factor, int interleaved, const void* q_norm_w,
                                const void* k_norm_w, float eps, void* q_out, void* k_cache,
                                void* v_cache, float* kv_scale, const int64_t* slot_mapping,
                                int64_t num_blocks, int page_size, int dtype,
                                nvkv_stream_t stream) {
  NVKV_RANGE("nvkv_rope_append");
  using namespace nvkv;
  clear_error();
  if (dtype != NVKV_DTYPE_BF16 && dtype != NVKV_DTYPE_F16)
    return set_error(NVKV_ERR_UNSUPPORTED, "rope_append: unsupported dtype (bf16/f16 only)");
  if (head_dim != kApD) return set_error(NVKV_ERR_UNSUPPORTED, "rope_append: head_dim must be 128");
  if (rot_dim <= 0 || rot_dim > kApD || rot_dim % 8)
    return set_error(NVKV_ERR_UNSUPPORTED, "rope_append: rot_dim must be a multiple of 8 up to 128");
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads <= 0 || num_q_heads > 65536 ||
      num_kv_heads > 65536 || num_blocks <= 0 || page_size <= 0)
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: bad sizes");
  if (kv_scale && page_size % kApBlock)
    return set_error(NVKV_ERR_UNSUPPORTED, "rope_append: page_size must be a multiple of 16");
  if (num_tokens == 0) return NVKV_OK;
  if (!k || !v || !positions || !inv_freq || !k_cache || !v_cache || !slot_mapping ||
      (num_q_heads && (!q || !q_out)))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: null pointer");
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: pass both norm weights or neither");
  const int64_t qr = (int64_t)num_q_heads * kApD, kr = (int64_t)num_kv_heads * kApD;
  if ((num_q_heads && q_stride < qr) || k_stride < kr || v_stride < kr)
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: a token stride is smaller than a row");
  if (!num_q_heads) q = q_out = nullptr;
  const uintptr_t m8 = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out |
                       (uintptr_t)q_norm_w | (uintptr_t)k_norm_w | (uintptr_t)positions |
                       (uintptr_t)inv_freq | (uintptr_t)slot_mapping |
                       (uintptr_t)(((num_q_heads ? q_stride : 0) | k_stride | v_stride) * 2);
  if ((m8 & 7u) || !aligned16(k_cache) || !aligned16(v_cache) || ((uintptr_t)kv_scale & 7u))
    return set_error(NVKV_ERR_ALIGNMENT,
                     "rope_append: rows, weights and metadata 8-byte, caches 16-byte aligned");
  if (q_out && (q_out == k || q_out == v || rows_clash(q, q_stride, qr, q_out, qr, qr, num_tokens) ||
                rows_clash(k, k_stride, kr, q_out, qr, qr, num_tokens) ||
                rows_clash(v, v_stride, kr, q_out, qr, qr, num_tokens)))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: q_out overlaps an input without being q");
  AppendParams p;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.num_tokens = num_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.half = rot_dim / 2;
  p.inter = interleaved ? 1 : 0;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.a = attn_factor;
  p.q_w = q_norm_w;
  p.k_w = k_norm_w;
  p.eps = eps;
  p.q_out = q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.scale = kv_scale;
  p.slots = slot_mapping;
  p.num_slots = num_blocks * page_size;
  p.page = page_size;
  p.err = device_error_word();
  p.window = (int)std::min<int64_t>(kApMaxWindow, std::max<int64_t>(1, num_tokens / (148 * 4)));
  const int64_t ctas = (num_tokens + p.window - 1) / p.window;
  if (ctas > 0x7fffffffLL) return set_error(NVKV_ERR_INVALID_ARG, "rope_append: too many tokens");
  const int table = kv_scale ? p.window + kApBlock - 1 : p.window;
  const size_t smem = (size_t)table * p.half * (kv_scale ? sizeof(double2) : sizeof(float2));
  const dim3 grid((unsigned)ctas), block(kApThreads);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVKV_DTYPE_BF16)
    return kv_scale ? launch_pdl(rope_append_kernel<__nv_bfloat16, true>, grid, block, smem, s,
                                 "rope_append launch", p)
                    : launch_pdl(rope_append_kernel<__nv_bfloat16, false>, grid, block, smem, s,
                                 "rope_append launch", p);
  return kv_scale ? launch_pdl(rope_append_kernel<__half, true>, grid, block, smem, s,
                               "rope_append launch", p)
                  : launch_pdl(rope_append_kernel<__half, false>, grid, block, smem, s,
                               "rope_append launch", p);
}
