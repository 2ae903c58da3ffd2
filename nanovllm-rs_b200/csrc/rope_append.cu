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
// tokens go to shared memory once (f32 for q; f64 for the tokens of the runs,
// up to 15 of them past the window); then warps take q rows and K / V units,
// every pair in one lane.  A unit is one run (the call's tokens of one block),
// one kv head, K or V: the warp holds all of its up to 16 rows in registers (64
// values a lane), so the maximum, the scale and the codes come from one read.
// The run belongs to the window of its first token.  W = 1 for a decode step (a CTA per token: latency), up to 16 for
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

// A lane's dims of a rotated row: the chunks x[a], x[a + 1] and x[b], x[b + 1],
// chosen so that every pair sits in one lane: pairs 2 lane and 2 lane + 1 of
// either layout while lane < half / 2, dims that pass through behind them.
struct LaneDims {
  int a, b;
  bool rot;
};
__device__ __forceinline__ LaneDims lane_dims(int lane, int half, bool inter) {
  LaneDims d;
  d.rot = lane < half / 2;
  d.a = d.rot && !inter ? 2 * lane : 4 * lane;  // half: pass-through dims 4 lane .. are >= 2 half
  d.b = d.rot && !inter ? half + 2 * lane : 4 * lane + 2;
  return d;
}

template <typename T, typename R>
__device__ __forceinline__ void to_vals(uint32_t a, uint32_t b, R (&x)[4]) {
  const float2 u = DT<T>::to_f2(a), v = DT<T>::to_f2(b);
  x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
}

// x rotated by the lane's two pairs' (cos, sin)
template <typename R, typename C>
__device__ __forceinline__ void rotate(R (&x)[4], const C c0, const C c1, bool inter) {
  const R p = x[0], q = inter ? x[1] : x[2], r = inter ? x[2] : x[1], s = x[3];
  const R y0 = p * c0.x - q * c0.y, y1 = q * c0.x + p * c0.y;
  const R y2 = r * c1.x - s * c1.y, y3 = s * c1.x + r * c1.y;
  x[0] = y0;
  x[1] = inter ? y1 : y2;
  x[2] = inter ? y2 : y1;
  x[3] = y3;
}

// Sums over the warp of N values a lane (N = 4 or 8): halving exchanges leave
// row j's sum in the lanes with j in their upper bits (9 shuffles for 8 rows
// instead of 40); row_lane(j) is one of them.
template <int N>
__device__ __forceinline__ int row_lane(int j) {
  return N == 8 ? ((j >> 2) & 1) << 4 | ((j >> 1) & 1) << 3 | (j & 1) << 2
                : ((j >> 1) & 1) << 4 | (j & 1) << 3;
}
template <int N, typename R>
__device__ __forceinline__ R row_sums(R (&v)[N], int lane) {
  int m = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int j = 0; j < n / 2; ++j) {
      const R keep = up ? v[j + n / 2] : v[j], give = up ? v[j] : v[j + n / 2];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, give, m);
    }
  }
#pragma unroll
  for (; m >= 1; m >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
  return v[0];
}

// Up to N head rows (128 apart) of one token: norm, rotation, one rounding.
template <typename T, int N>
__device__ __forceinline__ void rows_f32(const T* src, T* dst, int n, const T* w, float eps,
                                         const float2* cs, const LaneDims d, bool inter, int lane) {
  uint32_t ra[N], rb[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const T* s = src + (j < n ? j : 0) * kApD;
    ra[j] = *reinterpret_cast<const uint32_t*>(s + d.a);
    rb[j] = *reinterpret_cast<const uint32_t*>(s + d.b);
  }
  const float2 c0 = d.rot ? cs[2 * lane] : make_float2(1.f, 0.f);
  const float2 c1 = d.rot ? cs[2 * lane + 1] : make_float2(1.f, 0.f);
  float inv = 1.f, wv[4] = {1.f, 1.f, 1.f, 1.f};
  if (w) {
    to_vals<T>(*reinterpret_cast<const uint32_t*>(w + d.a),
               *reinterpret_cast<const uint32_t*>(w + d.b), wv);
    float ss[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float x[4];
      to_vals<T>(ra[j], rb[j], x);
      ss[j] = (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]);
    }
    inv = 1.f / sqrtf(row_sums<N>(ss, lane) * (1.f / kApD) + eps);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float x[4];
    to_vals<T>(ra[j], rb[j], x);
    if (w) {
      const float f = __shfl_sync(0xffffffffu, inv, row_lane<N>(j));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = x[i] * f * wv[i];
    }
    if (d.rot) rotate(x, c0, c1, inter);
    if (j < n) {
      *reinterpret_cast<uint32_t*>(dst + j * kApD + d.a) = DT<T>::from_f2(x[0], x[1]);
      *reinterpret_cast<uint32_t*>(dst + j * kApD + d.b) = DT<T>::from_f2(x[2], x[3]);
    }
  }
}

// K rows j0 .. j0 + 7 of a run in f64: x[j] becomes the normalised, rotated
// value rounded to odd.
template <typename T>
__device__ __forceinline__ void k_rows_f64(float (&x)[8][4], int n, const T* w, float eps,
                                           const double2* cs, int half, const LaneDims d,
                                           bool inter, int lane) {
  double inv = 1.0, wv[4];
  if (w) {
    to_vals<T>(*reinterpret_cast<const uint32_t*>(w + d.a),
               *reinterpret_cast<const uint32_t*>(w + d.b), wv);
    double ss[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss[j] = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss[j] = fma((double)x[j][i], (double)x[j][i], ss[j]);
    }
    inv = rsqrt(row_sums<8>(ss, lane) * (1.0 / kApD) + (double)eps);  // for this lane's row
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < n) {
      double y[4] = {x[j][0], x[j][1], x[j][2], x[j][3]};
      if (w) {
        const double f = __shfl_sync(0xffffffffu, inv, row_lane<8>(j));
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] * f * wv[i];
      }
      if (d.rot) rotate(y, cs[j * half + 2 * lane], cs[j * half + 2 * lane + 1], inter);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = f32_odd(y[i]);
    }
  }
}

// kWide: windows of several tokens (8 rows in flight a warp); else a decode
// step's single tokens (4, so that eight warps share 32 heads).
template <typename T, bool kF8, bool kWide>
__global__ void __launch_bounds__(kApThreads, 2) rope_append_kernel(const AppendParams p) {
  constexpr int kRows = kWide ? 8 : 4;
  extern __shared__ __align__(16) uint8_t smem[];
  double2* cs64 = reinterpret_cast<double2*>(smem);  // [run tokens][half], fp8b pool
  float2* cs = reinterpret_cast<float2*>(
      smem + (kF8 ? (size_t)(p.window + kApBlock - 1) * p.half * sizeof(double2) : 0));
  __shared__ int64_t slot_s[kApTable + 1];  // slots of tokens w0 - 1 ..
  __shared__ int lead_s[kApMaxWindow], len_s[kApMaxWindow], nrun_s, from_s, to_s;
  const int64_t w0 = (int64_t)blockIdx.x * p.window;
  const int n = (int)min((int64_t)p.window, p.num_tokens - w0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();  // nothing is read or written before: the launch may overlap the kernel before it
  for (int i = tid; i < n * p.half; i += kApThreads)
    cs[i] = rope_cs(p.positions[w0 + i / p.half], p.inv_freq[i % p.half], (float)p.a);
  if (warp == kApWarps - 1) {
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
      const int len = __ffs(after);
      if (leads >> lane & 1) {
        const int r = __popc(leads & ((1u << lane) - 1));
        lead_s[r] = lane - 1;
        len_s[r] = len;
      }
      const int last = leads ? 31 - __clz(leads) : 0;
      const int end = __shfl_sync(0xffffffffu, lane - 1 + len, last);
      if (lane == 0) {
        nrun_s = __popc(leads);
        from_s = leads ? __ffs(leads) - 2 : 0;  // tokens that the runs span
        to_s = leads ? end : 0;
      }
    }
  }
  __syncthreads();

  const bool inter = p.inter != 0;
  const LaneDims d = lane_dims(lane, p.half, inter);
  const T* qw = static_cast<const T*>(p.q_w);
  const T* kw = static_cast<const T*>(p.k_w);
  if (kF8) {
    const int from = from_s, to = to_s;
    for (int i = tid; i < (to - from) * p.half; i += kApThreads)
      cs64[from * p.half + i] = rope_cs64(p.positions[w0 + from + i / p.half],
                                          p.inv_freq[i % p.half], p.a);
  }

  // q rows (and K rows of the dtype pool): kRows heads of a token a step
  const int qb = (p.hq + kRows - 1) / kRows, kb = kF8 ? 0 : (p.hkv + kRows - 1) / kRows;
  for (int u = warp; u < n * (qb + kb); u += kApWarps) {
    const int t = u / (qb + kb), c = u % (qb + kb);
    if (c < qb) {
      const int h = c * kRows;
      rows_f32<T, kRows>(static_cast<const T*>(p.q) + (w0 + t) * p.q_stride + (int64_t)h * kApD,
                         static_cast<T*>(p.q_out) + ((w0 + t) * p.hq + h) * kApD,
                         min(kRows, p.hq - h), qw, p.eps, cs + t * p.half, d, inter, lane);
    } else {
      const int h = (c - qb) * kRows;
      const int64_t slot = slot_s[t + 1];
      if (slot >= 0)
        rows_f32<T, kRows>(static_cast<const T*>(p.k) + (w0 + t) * p.k_stride + (int64_t)h * kApD,
                           static_cast<T*>(p.k_cache) + (slot * p.hkv + h) * kApD,
                           min(kRows, p.hkv - h), kw, p.eps, cs + t * p.half, d, inter, lane);
    }
  }

  if constexpr (!kF8) {
    for (int u = warp; u < n * p.hkv; u += kApWarps) {
      const int t = u / p.hkv, h = u % p.hkv;
      const int64_t slot = slot_s[t + 1];
      if (slot < 0) continue;
      const T* src = static_cast<const T*>(p.v) + (w0 + t) * p.v_stride + (int64_t)h * kApD;
      T* dst = static_cast<T*>(p.v_cache) + (slot * p.hkv + h) * kApD;
      *reinterpret_cast<uint2*>(dst + 4 * lane) = *reinterpret_cast<const uint2*>(src + 4 * lane);
    }
  } else {
    __syncthreads();  // the f64 table
    const int per = p.page / kApBlock, nk = nrun_s * p.hkv;
    const int64_t row = (int64_t)p.hkv * kApD;
    for (int u = warp; u < 2 * nk; u += kApWarps) {
      const int kv = u >= nk, uu = kv ? u - nk : u;
      const int r = uu / p.hkv, h = uu % p.hkv;
      const int t = lead_s[r], len = len_s[r];
      const int64_t blk = slot_s[t + 1] / kApBlock;
      const int low = (int)(slot_s[t + 1] % kApBlock);
      float* sp = p.scale + (((blk / per) * p.hkv + h) * per + blk % per) * 2 + kv;
      const float old = low ? *sp : 0.f;
      const int64_t stride = kv ? p.v_stride : p.k_stride;
      const T* src = (kv ? static_cast<const T*>(p.v) : static_cast<const T*>(p.k)) +
                     (w0 + t) * stride + (int64_t)h * kApD;
      // V's rows are not rotated: four neighbouring dims a lane
      const int da = kv ? 4 * lane : d.a, db = kv ? 4 * lane + 2 : d.b;
      float x[2][8][4];
      float amax = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (8 * g < len) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const T* s = src + (8 * g + j < len ? 8 * g + j : 0) * stride;
            to_vals<T>(*reinterpret_cast<const uint32_t*>(s + da),
                       *reinterpret_cast<const uint32_t*>(s + db), x[g][j]);
          }
          if (!kv)
            k_rows_f64<T>(x[g], len - 8 * g, kw, p.eps, cs64 + (t + 8 * g) * p.half, p.half, d,
                          inter, lane);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (8 * g + j < len) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float m = fabsf(x[g][j][i]);
                amax = fmaxf(amax, m < INFINITY ? m : 0.f);
              }
            }
        }
      }
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) amax = warp_max_xor(amax, m);
      const int e_old = max(kApMinE, (int)(__float_as_uint(old) >> 23 & 0xffu) - 127);
      int e = block_exp(amax);
      if (low) e = max(e, e_old);
      const float inv = pow2i(-e);
      uint8_t* base = static_cast<uint8_t*>(kv ? p.v_cache : p.k_cache) +
                      (blk * kApBlock * p.hkv + h) * kApD;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (8 * g + j < len) {
            uint8_t* c = base + (slot_s[t + 1 + 8 * g + j] % kApBlock) * row;
            const float* y = x[g][j];
            const uint32_t w = e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
            *reinterpret_cast<uint16_t*>(c + da) = (uint16_t)w;
            *reinterpret_cast<uint16_t*>(c + db) = (uint16_t)(w >> 16);
          }
        }
      }
      if (e > e_old && low) {  // the kept rows move to the larger scale
        const float f = pow2i(max(e_old - e, -126));
#pragma unroll 4
        for (int j = 0; j < low; ++j) {
          uint32_t* c = reinterpret_cast<uint32_t*>(base + j * row + 4 * lane);
          float y[4];
          e4m3x4_f32(*c, y);
          *c = e4m3x4(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
        }
      }
      if (lane == 0 && (!low || e > e_old)) *sp = pow2i(e);
    }
  }
}

template <typename T>
int launch_append(const AppendParams& p, dim3 grid, size_t smem, cudaStream_t s) {
  const bool f8 = p.scale != nullptr, wide = p.window > 1;
  auto kern = f8 ? (wide ? rope_append_kernel<T, true, true> : rope_append_kernel<T, true, false>)
                 : (wide ? rope_append_kernel<T, false, true> : rope_append_kernel<T, false, false>);
  return launch_pdl(kern, grid, dim3(kApThreads), smem, s, "rope_append launch", p);
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
  const size_t smem = (size_t)p.half * (p.window * sizeof(float2) +
                                        (kv_scale ? (p.window + kApBlock - 1) * sizeof(double2) : 0));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == NVKV_DTYPE_BF16 ? launch_append<__nv_bfloat16>(p, dim3((unsigned)ctas), smem, s)
                                  : launch_append<__half>(p, dim3((unsigned)ctas), smem, s);
}
