// Rotary positions as an operator of its own (nvkv_rope), with the
// frequencies of long contexts (nvkv_rope_frequencies).
//
// The reference rotates whole heads in the half layout with plain frequencies
// (nanovllm_rs/src/layers/rotary_embedding.rs:11-70); nvkv_qknorm_rope keeps
// that form and its rounding points.  This one takes both pair layouts, a
// rotated part of the head, any frequencies and an attention factor:
//   half:         pairs (x[i], x[i + r/2]),   interleaved: (x[2i], x[2i + 1])
//   y0 = a (x0 cos - x1 sin), y1 = a (x1 cos + x0 sin), i < r/2;
//   dims r .. head_dim - 1 pass through.
// f32 arithmetic, one rounding to the dtype at the end.
//
// Bound by HBM: every row is read and written once.  A CTA takes a window of
// tokens; it puts their cos / sin (f64 angles, rope_angle.cuh) into shared
// memory once for all heads, then each thread keeps one 16-byte unit of one
// head (half layout: two 8-element vectors, r/2 apart; interleaved: one
// vector of four pairs; a vector behind r: a copy) and walks the window's
// tokens, two of them in flight.  Where r, the head size, a stride or an
// address do not allow 16-byte vectors, a unit is a single pair.
#include <math.h>

#include <algorithm>

#include "rope_angle.cuh"

namespace nvkv {
namespace {

struct RopeParams {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_stride, k_stride, qo_stride, ko_stride;
  int64_t num_tokens;
  int hq, heads, d, half;  // half = rot / 2
  int rot_units, units;    // units of a head: the rotated ones, then the copied ones
  int window;
  const int64_t* positions;
  const double* inv_freq;
  float a;
};

// Tokens in flight per thread, and CTAs of one wave.  Measured at 16384 tokens,
// 32 + 8 heads of 128 (51 us of traffic): 4 in flight (126 registers) 68.9 us, 2
// in flight 61.0 / 57.7 / 63.5 / 58.8 us with 3 / 4 / 5 / 6 CTAs an SM.
constexpr int kRopeFlight = 2;
constexpr int kRopeThreads = 448;
constexpr int kRopeWave = 148 * 4;
constexpr int kRopeMaxWindow = 32;

// VEC = 8: 16-byte units; 1: single pairs / elements.
template <typename T, int VEC, bool kInter>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  // (cos, sin) of two pairs a float4: [window][VEC / 2 or 1][rotated units], so
  // that neighbouring units read neighbouring words (8-byte entries for VEC = 1)
  extern __shared__ __align__(16) float2 cs[];
  constexpr int kPairs = VEC == 1 ? 1 : kInter ? 4 : 8;  // pairs of a unit
  const int64_t t0 = (int64_t)blockIdx.x * p.window;
  const int n = (int)min((int64_t)p.window, p.num_tokens - t0);
  const int nthr = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = tid; i < n * p.half; i += nthr) {
    const int t = i / p.half, pr = i % p.half, u = pr / kPairs, w = pr % kPairs;
    cs[t * p.half + (VEC == 1 ? pr : ((w >> 1) * p.rot_units + u) * 2 + (w & 1))] =
        rope_cs(p.positions[t0 + t], p.inv_freq[pr], p.a);
  }
  __syncthreads();
  using V = typename std::conditional<VEC == 8, uint4, uint16_t>::type;
  for (int u = threadIdx.x; u < p.units; u += blockDim.x) {
    const bool rot = u < p.rot_units;
    const bool two = rot && (!kInter || VEC == 1);  // a second vector / element
    const int e0 = rot ? (kInter && VEC == 1 ? 2 * u : u * VEC)
                       : 2 * p.half + (u - p.rot_units) * VEC;
    const int e1 = kInter ? e0 + 1 : e0 + p.half;
    for (int h = threadIdx.y; h < p.heads; h += blockDim.y) {
      const bool is_q = h < p.hq;
      const int64_t ho = (int64_t)(is_q ? h : h - p.hq) * p.d;
      const int64_t is = is_q ? p.q_stride : p.k_stride, os = is_q ? p.qo_stride : p.ko_stride;
      const T* src = static_cast<const T*>(is_q ? p.q : p.k) + t0 * is + ho;
      T* dst = static_cast<T*>(is_q ? p.q_out : p.k_out) + t0 * os + ho;
      for (int j = 0; j < n; j += kRopeFlight) {
        V a[kRopeFlight], b[kRopeFlight];
#pragma unroll
        for (int f = 0; f < kRopeFlight; ++f)
          if (j + f < n) {
            a[f] = *reinterpret_cast<const V*>(src + (j + f) * is + e0);
            if (two) b[f] = *reinterpret_cast<const V*>(src + (j + f) * is + e1);
          }
#pragma unroll
        for (int f = 0; f < kRopeFlight; ++f) {
          if (j + f >= n) break;
          if (rot) {
            const float2* c = cs + (j + f) * p.half + (VEC == 1 ? u : 2 * u);
            if constexpr (VEC == 1) {
              const float x0 = DT<T>::to_f(*reinterpret_cast<T*>(&a[f]));
              const float x1 = DT<T>::to_f(*reinterpret_cast<T*>(&b[f]));
              const T y0 = DT<T>::from_f(x0 * c[0].x - x1 * c[0].y);
              const T y1 = DT<T>::from_f(x1 * c[0].x + x0 * c[0].y);
              a[f] = *reinterpret_cast<const V*>(&y0);
              b[f] = *reinterpret_cast<const V*>(&y1);
            } else {
              uint32_t* wa = reinterpret_cast<uint32_t*>(&a[f]);
              uint32_t* wb = reinterpret_cast<uint32_t*>(&b[f]);
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                // pairs 2w, 2w + 1 of the unit (interleaved: pair w, half of an entry)
                const float4 r = *reinterpret_cast<const float4*>(
                    c + (kInter ? w >> 1 : w) * 2 * p.rot_units);
                if (kInter) {
                  const float2 x = DT<T>::to_f2(wa[w]);
                  const float cc = w & 1 ? r.z : r.x, ss = w & 1 ? r.w : r.y;
                  wa[w] = DT<T>::from_f2(x.x * cc - x.y * ss, x.y * cc + x.x * ss);
                } else {
                  const float2 x = DT<T>::to_f2(wa[w]), y = DT<T>::to_f2(wb[w]);
                  wa[w] = DT<T>::from_f2(x.x * r.x - y.x * r.y, x.y * r.z - y.y * r.w);
                  wb[w] = DT<T>::from_f2(y.x * r.x + x.x * r.y, y.y * r.z + x.y * r.w);
                }
              }
            }
          }
          *reinterpret_cast<V*>(dst + (j + f) * os + e0) = a[f];
          if (two) *reinterpret_cast<V*>(dst + (j + f) * os + e1) = b[f];
        }
      }
    }
  }
}

template <typename T>
void launch_rope(const RopeParams& p, bool vec, bool inter, dim3 grid, dim3 block, size_t smem,
                 cudaStream_t s) {
  if (vec && inter) rope_kernel<T, 8, true><<<grid, block, smem, s>>>(p);
  else if (vec) rope_kernel<T, 8, false><<<grid, block, smem, s>>>(p);
  else if (inter) rope_kernel<T, 1, true><<<grid, block, smem, s>>>(p);
  else rope_kernel<T, 1, false><<<grid, block, smem, s>>>(p);
}

}  // namespace

bool rows_clash(const void* a, int64_t a_stride, int64_t a_row, const void* b, int64_t b_stride,
                int64_t b_row, int64_t tokens) {
  if (!a || !b || tokens <= 0 || (a == b && (a_stride == b_stride || tokens == 1))) return false;
  uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  const uintptr_t xe = x + (uintptr_t)((tokens - 1) * a_stride + a_row) * 2;
  const uintptr_t ye = y + (uintptr_t)((tokens - 1) * b_stride + b_row) * 2;
  if (x >= ye || y >= xe) return false;
  if (a_stride != b_stride || tokens == 1) return true;
  // rows of one stride may interleave without touching (slices of one fused buffer)
  const uintptr_t st = (uintptr_t)a_stride * 2;
  const uintptr_t off = x >= y ? (x - y) % st : st - 1 - (y - x - 1) % st;  // a's start in b's rows
  return !(off >= (uintptr_t)b_row * 2 && off + (uintptr_t)a_row * 2 <= st);
}

}  // namespace nvkv

extern "C" int nvkv_rope_frequencies(int rot_dim, double theta, const nvkv_rope_scaling* scaling,
                                     double* inv_freq, double* attn_factor) {
  using namespace nvkv;
  clear_error();
  if (rot_dim <= 0 || rot_dim % 2 || !(theta > 0.0) || !isfinite(theta) || !inv_freq ||
      !attn_factor)
    return set_error(NVKV_ERR_INVALID_ARG,
                     "rope_frequencies: rot_dim even and > 0, theta > 0, outputs not null");
  const int type = scaling ? scaling->type : NVKV_ROPE_PLAIN;
  const double f = scaling ? scaling->factor : 1.0;
  const double two_pi = 6.283185307179586476925;
  if (type < NVKV_ROPE_PLAIN || type > NVKV_ROPE_BANDS)
    return set_error(NVKV_ERR_UNSUPPORTED, "rope_frequencies: unknown scaling type");
  if (type != NVKV_ROPE_PLAIN && !(f >= 1.0 && isfinite(f)))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_frequencies: factor must be >= 1");
  const bool by_length = type == NVKV_ROPE_YARN || type == NVKV_ROPE_BANDS;
  if (by_length && scaling->original_max_position <= 0)
    return set_error(NVKV_ERR_INVALID_ARG, "rope_frequencies: original_max_position must be > 0");
  const double orig = by_length ? (double)scaling->original_max_position : 0.0;
  double base = theta, lo = 0.0, hi = 0.0;
  *attn_factor = 1.0;
  if (type == NVKV_ROPE_NTK && rot_dim > 2) base = theta * pow(f, rot_dim / (double)(rot_dim - 2));
  if (type == NVKV_ROPE_YARN) {
    const double bf = scaling->beta_fast, bs = scaling->beta_slow;
    if (!(bf >= bs && bs > 0.0) || theta <= 1.0)
      return set_error(NVKV_ERR_INVALID_ARG,
                       "rope_frequencies: YARN needs beta_fast >= beta_slow > 0 and theta > 1");
    // the pair that makes `turns` turns over the original context
    auto pair_of = [&](double turns) {
      return rot_dim * log(orig / (turns * two_pi)) / (2.0 * log(theta));
    };
    lo = std::max(floor(pair_of(bf)), 0.0);
    hi = std::min(ceil(pair_of(bs)), rot_dim - 1.0);
    *attn_factor = 0.1 * log(f) + 1.0;
  }
  if (type == NVKV_ROPE_BANDS &&
      !(scaling->high_freq_factor > scaling->low_freq_factor && scaling->low_freq_factor > 0.0))
    return set_error(NVKV_ERR_INVALID_ARG,
                     "rope_frequencies: high_freq_factor > low_freq_factor > 0");
  if (scaling && scaling->attention_factor > 0.0) *attn_factor = scaling->attention_factor;
  for (int i = 0; i < rot_dim / 2; ++i) {
    const double x = pow(base, -2.0 * i / rot_dim);
    if (type == NVKV_ROPE_LINEAR) {
      inv_freq[i] = x / f;
    } else if (by_length) {
      double keep;  // share of the unscaled frequency
      if (type == NVKV_ROPE_YARN)
        keep = 1.0 - std::min(std::max((i - lo) / std::max(hi - lo, 1e-3), 0.0), 1.0);
      else
        keep = std::min(std::max((orig * x / two_pi - scaling->low_freq_factor) /
                                     (scaling->high_freq_factor - scaling->low_freq_factor), 0.0),
                        1.0);
      inv_freq[i] = x / f * (1.0 - keep) + x * keep;
    } else {
      inv_freq[i] = x;
    }
  }
  return NVKV_OK;
}

extern "C" int nvkv_rope(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                         void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride,
                         int64_t num_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                         const int64_t* positions, const double* inv_freq, int rot_dim,
                         double attn_factor, int interleaved, int dtype, nvkv_stream_t stream) {
  NVKV_RANGE("nvkv_rope");
  using namespace nvkv;
  clear_error();
  if (dtype != NVKV_DTYPE_BF16 && dtype != NVKV_DTYPE_F16)
    return set_error(NVKV_ERR_UNSUPPORTED, "rope: unsupported dtype (bf16/f16 only)");
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || num_q_heads + num_kv_heads <= 0 ||
      num_q_heads > 65536 || num_kv_heads > 65536)
    return set_error(NVKV_ERR_INVALID_ARG, "rope: bad sizes");
  if (head_dim <= 0 || head_dim > 1024 || rot_dim <= 0 || rot_dim % 2 || rot_dim > head_dim)
    return set_error(NVKV_ERR_UNSUPPORTED,
                     "rope: head_dim up to 1024, rot_dim even and at most head_dim");
  if (num_tokens == 0) return NVKV_OK;
  const int64_t qr = (int64_t)num_q_heads * head_dim, kr = (int64_t)num_kv_heads * head_dim;
  if (!positions || !inv_freq || (num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out)))
    return set_error(NVKV_ERR_INVALID_ARG, "rope: null pointer");
  if ((num_q_heads && (q_stride < qr || q_out_stride < qr)) ||
      (num_kv_heads && (k_stride < kr || k_out_stride < kr)))
    return set_error(NVKV_ERR_INVALID_ARG, "rope: a token stride is smaller than a row");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out) & 1u ||
      ((uintptr_t)positions | (uintptr_t)inv_freq) & 7u)
    return set_error(NVKV_ERR_ALIGNMENT, "rope: rows 2-byte, positions / inv_freq 8-byte aligned");
  const bool in_place = (!num_q_heads || q == q_out) && (!num_kv_heads || k == k_out);
  // an output may be its own input; any other overlap would be read after it is written
  if (!num_q_heads) q = q_out = nullptr;
  if (!num_kv_heads) k = k_out = nullptr;
  if (rows_clash(q, q_stride, qr, q_out, q_out_stride, qr, num_tokens) ||
      rows_clash(k, k_stride, kr, k_out, k_out_stride, kr, num_tokens))
    return set_error(NVKV_ERR_INVALID_ARG, "rope: an output overlaps its input without being it");
  if ((q_out && (q_out == k || q_out == k_out || k_out == q)) ||
      rows_clash(q_out, q_out_stride, qr, k, k_stride, kr, num_tokens) ||
      rows_clash(k_out, k_out_stride, kr, q, q_stride, qr, num_tokens) ||
      rows_clash(q_out, q_out_stride, qr, k_out, k_out_stride, kr, num_tokens))
    return set_error(NVKV_ERR_INVALID_ARG, "rope: q's and k's rows overlap");
  const Span pos = {positions, (uint64_t)num_tokens * 8}, freq = {inv_freq, (uint64_t)rot_dim * 4};
  if (spans_meet(q_out, (uint64_t)((num_tokens - 1) * q_out_stride + qr) * 2, {pos, freq}) ||
      spans_meet(k_out, (uint64_t)((num_tokens - 1) * k_out_stride + kr) * 2, {pos, freq}))
    return set_error(NVKV_ERR_INVALID_ARG, "rope: an output overlaps positions or inv_freq");
  RopeParams p;
  p.q = q;
  p.k = k;
  p.q_out = q_out;
  p.k_out = k_out;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.qo_stride = q_out_stride;
  p.ko_stride = k_out_stride;
  p.num_tokens = num_tokens;
  p.hq = num_q_heads;
  p.heads = num_q_heads + num_kv_heads;
  p.d = head_dim;
  p.half = rot_dim / 2;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.a = (float)attn_factor;
  const bool inter = interleaved != 0;
  const uintptr_t m = (uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out |
                      (uintptr_t)(num_q_heads ? (q_stride | q_out_stride) * 2 : 0) |
                      (uintptr_t)(num_kv_heads ? (k_stride | k_out_stride) * 2 : 0);
  const bool vec = (m & 15u) == 0 && head_dim % 8 == 0 && rot_dim % (inter ? 8 : 16) == 0;
  p.rot_units = vec ? rot_dim / (inter ? 8 : 16) : rot_dim / 2;
  const int copies = in_place ? 0 : (head_dim - rot_dim) / (vec ? 8 : 1);
  p.units = p.rot_units + copies;
  // One wave of CTAs: a CTA costs two dependent loads, the table and a barrier
  // before it streams (the same 16384 tokens with four in flight: windows of 1 / 2
  // / 4 / 8 tokens 237 / 140 / 93 / 75 us).
  // (the table of a window stays below the 48 KB that need no opt-in)
  p.window = (int)std::min<int64_t>(std::min(kRopeMaxWindow, 48 * 1024 / (p.half * 8)),
                                    (num_tokens + kRopeWave - 1) / kRopeWave);
  const int bx = std::min(p.units, 64);
  const int rounds = (p.heads * bx + 383) / 384;
  const int by = (p.heads + rounds - 1) / rounds;  // bx * by < 384 + bx
  const int64_t ctas = (num_tokens + p.window - 1) / p.window;
  if (ctas > 0x7fffffffLL) return set_error(NVKV_ERR_INVALID_ARG, "rope: too many tokens");
  const size_t smem = (size_t)p.window * p.half * sizeof(float2);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVKV_DTYPE_BF16)
    launch_rope<__nv_bfloat16>(p, vec, inter, dim3((unsigned)ctas), dim3(bx, by), smem, s);
  else
    launch_rope<__half>(p, vec, inter, dim3((unsigned)ctas), dim3(bx, by), smem, s);
  return check_cuda(cudaGetLastError(), "rope launch");
}
