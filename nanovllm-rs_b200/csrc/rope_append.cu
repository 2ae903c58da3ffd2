// Append to a paged KV cache with the rotation on the way (nvkv_rope_append):
// per-head RMSNorm (optional), rotary positions, and the store of K and V into
// the model-dtype pool or the block-scaled e4m3 pool, in one launch.
//
// Mathematics (fp8b pool).  With the rows x of a block of 16 slots and one kv
// head (K and V apart): e = max(e_kept, least e >= -100 with amax <= 448 2^e),
// code = e4m3(x 2^-e); rows that the block already held move by code' =
// e4m3(code 2^(e_kept - e)).  K is normalised and rotated in f64 and reaches
// e4m3 by ONE rounding (to f32 by rounding to odd, which the conversion to four
// significant bits cannot tell from the f64 value), so the codes are a function of
// the formulas and not of the f32 arithmetic's order, and tests compare them bit
// by bit.  q and the dtype pool use f32 and round once.
//
// Layout.  A CTA of 8 warps owns a window of W tokens: the cos / sin of those
// tokens (and of the up to 15 that follow in the last run) go to shared memory
// once; then warps take q rows and K / V units, every pair in one lane.  A unit is
// one run (the call's tokens of one block), one kv head, K or V: its warps hold all
// of its up to 16 rows in registers, so the maximum, the scale and the codes come
// from one read.  The run belongs to the window of its first token.  W = 1 for a
// decode step (a CTA per token: latency), up to 16 for prompts.
//
// Least traffic for prompts: qkv read, q and codes written.  16 x 1024 tokens of
// 32 + 8 + 8 heads (369 MB, 56 us): 89 us with norms, 83 without, 4.1-4.5 TB/s.  It
// waits for rows: 80 registers leave 20 warps an SM, each of which loads its rows and
// only then computes (half of the issue slots taken, f64 at 6 % of its pipe).  Up to
// some 4700 tokens a window has 2 to 7 tokens and as many of the eight warps the q
// rows: with norms 1184 tokens 24.6 us, 2400 28.2, 4096 33.6 (4.1, 8.3 and 14.1 us of
// traffic).  A step of 256 tokens (10 MB): 5.5-6.2 us, the chain of slot, kept rows,
// maximum and codes.  (K in f32 with an error bound, f64 where it leaves a code
// undecided: 121 and 17 us; q and K / V in blocks of their own: 121.)
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

// f64 -> f32 rounded to odd: toward zero, the last bit set if anything was cut
// (the low 29 bits, in f32's normal range; below it every code is 0 either way).
__device__ __forceinline__ float f32_odd(double x) {
  const uint32_t cut = (uint32_t)__double2loint(x) & 0x1fffffffu;
  return __uint_as_float(__float_as_uint(__double2float_rz(x)) | (cut ? 1u : 0u));
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

// Packed two-lane f32 arithmetic (sm_100): one instruction for two values.
__device__ __forceinline__ uint64_t pk(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpk(uint64_t r) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Half a warp takes a head row, 8 dims a lane in two chunks of four: x[a ..
// a + 3] and x[b .. b + 3].  While sub = lane % 16 < half / 4 they are pairs
// 4 sub .. 4 sub + 3 of either layout; the lanes behind pass their dims through.
struct LaneDims {
  int a, b;
  bool rot;
};
template <bool kInter>
__device__ __forceinline__ LaneDims lane_dims(int sub, int half) {
  LaneDims d;
  d.rot = sub < half / 4;
  d.a = d.rot && !kInter ? 4 * sub : 8 * sub;  // (8 sub >= 2 half behind the rotated part)
  d.b = d.rot && !kInter ? half + 4 * sub : 8 * sub + 4;
  return d;
}

// The eight values as pair partners: X = first members, Y = second ones, of
// pairs 4 sub .. 4 sub + 3 (for lanes that pass through: any fixed order).
template <typename T, bool kInter, typename R>
__device__ __forceinline__ void to_pairs(const uint2 wa, const uint2 wb, R (&x)[4], R (&y)[4]) {
  const float2 a0 = DT<T>::to_f2(wa.x), a1 = DT<T>::to_f2(wa.y);
  const float2 b0 = DT<T>::to_f2(wb.x), b1 = DT<T>::to_f2(wb.y);
  if (kInter) {
    x[0] = a0.x, y[0] = a0.y, x[1] = a1.x, y[1] = a1.y;
    x[2] = b0.x, y[2] = b0.y, x[3] = b1.x, y[3] = b1.y;
  } else {
    x[0] = a0.x, x[1] = a0.y, x[2] = a1.x, x[3] = a1.y;
    y[0] = b0.x, y[1] = b0.y, y[2] = b1.x, y[3] = b1.y;
  }
}

// Sums over half a warp of N values a lane: halving exchanges leave value j's
// sum in the lanes whose upper bits spell j (8 shuffles for 8 values, not 32).
template <int N>
__device__ __forceinline__ int sum_lane(int j, int lane) {
  return (lane & 16) | j * (16 / N);
}
template <int N, typename R>
__device__ __forceinline__ R half_sums(R (&v)[N], int lane) {
  int m = 8;
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

// A token's rotation with the norm's weights folded in, for the lane's four
// pairs: y0 = inv (x0 A - x1 B), y1 = inv (x1 C + x0 E); packed by two pairs.
struct Coef {
  uint64_t a[2], b[2], c[2], e[2];
};
template <typename T, bool kInter>
__device__ __forceinline__ Coef token_coef(const float2* cs, const T* w, const LaneDims d, int sub) {
  float wx[4] = {1.f, 1.f, 1.f, 1.f}, wy[4] = {1.f, 1.f, 1.f, 1.f};
  if (w)
    to_pairs<T, kInter>(*reinterpret_cast<const uint2*>(w + d.a),
                        *reinterpret_cast<const uint2*>(w + d.b), wx, wy);
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (d.rot) {
    const float4 p0 = *reinterpret_cast<const float4*>(cs + 4 * sub);
    const float4 p1 = *reinterpret_cast<const float4*>(cs + 4 * sub + 2);
    c[0] = p0.x, s[0] = p0.y, c[1] = p0.z, s[1] = p0.w;
    c[2] = p1.x, s[2] = p1.y, c[3] = p1.z, s[3] = p1.w;
  }
  Coef f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f.a[i] = pk(wx[2 * i] * c[2 * i], wx[2 * i + 1] * c[2 * i + 1]);
    f.b[i] = pk(-wy[2 * i] * s[2 * i], -wy[2 * i + 1] * s[2 * i + 1]);
    f.c[i] = pk(wy[2 * i] * c[2 * i], wy[2 * i + 1] * c[2 * i + 1]);
    f.e[i] = pk(wx[2 * i] * s[2 * i], wx[2 * i + 1] * s[2 * i + 1]);
  }
  return f;
}

// Up to 2 N head rows (128 apart) of one token: norm, rotation, one rounding.
template <typename T, int N, bool kInter>
__device__ __forceinline__ void rows_f32(const T* src, T* dst, int n, bool norm, float eps,
                                         const Coef& f, const LaneDims d, int lane) {
  const int grp = lane >> 4;
  float x[N][4], y[N][4];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const T* s = src + (2 * j + grp < n ? 2 * j + grp : 0) * kApD;
    to_pairs<T, kInter>(*reinterpret_cast<const uint2*>(s + d.a),
                        *reinterpret_cast<const uint2*>(s + d.b), x[j], y[j]);
  }
  float inv = 1.f;
  if (norm) {
    float ss[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      uint64_t q = mul2(pk(x[j][0], x[j][1]), pk(x[j][0], x[j][1]));
      q = fma2(pk(x[j][2], x[j][3]), pk(x[j][2], x[j][3]), q);
      q = fma2(pk(y[j][0], y[j][1]), pk(y[j][0], y[j][1]), q);
      q = fma2(pk(y[j][2], y[j][3]), pk(y[j][2], y[j][3]), q);
      ss[j] = unpk(q).x + unpk(q).y;
    }
    inv = 1.f / sqrtf(half_sums<N>(ss, lane) * (1.f / kApD) + eps);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float g = norm ? __shfl_sync(0xffffffffu, inv, sum_lane<N>(j, lane)) : 1.f;
    const uint64_t g2 = pk(g, g);
    float2 ox[2], oy[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t X = pk(x[j][2 * i], x[j][2 * i + 1]), Y = pk(y[j][2 * i], y[j][2 * i + 1]);
      uint64_t u = mul2(X, f.a[i]), v = mul2(Y, f.c[i]);
      if (d.rot) {
        u = fma2(Y, f.b[i], u);
        v = fma2(X, f.e[i], v);
      }
      if (norm) {
        u = mul2(u, g2);
        v = mul2(v, g2);
      }
      ox[i] = unpk(u);
      oy[i] = unpk(v);
    }
    if (2 * j + grp < n) {
      T* t = dst + (2 * j + grp) * kApD;
      uint2 wa, wb;
      if (kInter) {
        wa = make_uint2(DT<T>::from_f2(ox[0].x, oy[0].x), DT<T>::from_f2(ox[0].y, oy[0].y));
        wb = make_uint2(DT<T>::from_f2(ox[1].x, oy[1].x), DT<T>::from_f2(ox[1].y, oy[1].y));
      } else {
        wa = make_uint2(DT<T>::from_f2(ox[0].x, ox[0].y), DT<T>::from_f2(ox[1].x, ox[1].y));
        wb = make_uint2(DT<T>::from_f2(oy[0].x, oy[0].y), DT<T>::from_f2(oy[1].x, oy[1].y));
      }
      *reinterpret_cast<uint2*>(t + d.a) = wa;
      *reinterpret_cast<uint2*>(t + d.b) = wb;
    }
  }
}

// A barrier of warps 2 i and 2 i + 1.
__device__ __forceinline__ void pair_barrier(int warp) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
}

// One run of one kv head.  Of a warp's rows, row 2 j + lane / 16 sits in x[j] /
// y[j] (values as pairs for K, eight neighbouring dims for V); rows past the run
// repeat its row 0 and are not stored.
struct Unit {
  uint8_t* base;  // the block's row 0, this head
  float* scale;
  const int64_t* slot;  // shared: the run's slots
  int len, low, row0;
  int64_t row;  // bytes between rows
};

// The warp's largest finite |value|.
template <int N>
__device__ __forceinline__ float warp_amax(const float (&x)[N][4], const float (&y)[N][4]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = max(m, max(__float_as_uint(x[j][i]) & 0x7fffffffu, __float_as_uint(y[j][i]) & 0x7fffffffu));
  m = __reduce_max_sync(0xffffffffu, m);
  if (m >= 0x7f800000u) {  // an infinity or NaN among them: leave those out
    m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(x[j][i]) & 0x7fffffffu;
        const uint32_t b = __float_as_uint(y[j][i]) & 0x7fffffffu;
        m = max(m, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
      }
    m = __reduce_max_sync(0xffffffffu, m);
  }
  return __uint_as_float(m);
}

// Codes of a warp's rows once the block's largest value is known; the warp of row
// 0 also moves kept rows and writes the scale.  kFull: a whole block, 16 rows.
template <int N, bool kFull>
__device__ __forceinline__ void encode_rows(const float (&x)[N][4], const float (&y)[N][4],
                                            const Unit& u, float old, float amax, int da, int db,
                                            bool inter, int lane) {
  const int grp = lane >> 4;
  const int e_old = max(kApMinE, (int)(__float_as_uint(old) >> 23 & 0xffu) - 127);
  int e = block_exp(amax);
  if (!kFull && u.low) e = max(e, e_old);
  const float inv = pow2i(-e);
  uint8_t* c = u.base + (kFull ? (u.row0 + grp) * u.row : 0);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int r = u.row0 + 2 * j + grp;
    uint32_t wa, wb;
    if (inter) {
      wa = e4m3x4(x[j][0] * inv, y[j][0] * inv, x[j][1] * inv, y[j][1] * inv);
      wb = e4m3x4(x[j][2] * inv, y[j][2] * inv, x[j][3] * inv, y[j][3] * inv);
    } else {
      wa = e4m3x4(x[j][0] * inv, x[j][1] * inv, x[j][2] * inv, x[j][3] * inv);
      wb = e4m3x4(y[j][0] * inv, y[j][1] * inv, y[j][2] * inv, y[j][3] * inv);
    }
    if (kFull || r < u.len) {
      if (!kFull) c = u.base + (u.slot[r] % kApBlock) * u.row;
      *reinterpret_cast<uint32_t*>(c + da) = wa;
      *reinterpret_cast<uint32_t*>(c + db) = wb;
    }
    if (kFull) c += 2 * u.row;
  }
  if (u.row0 == 0) {
    if (!kFull && e > e_old && u.low) {
      const float f = pow2i(max(e_old - e, -126));
#pragma unroll 4
      for (int j = 0; j < u.low; ++j) {
        uint32_t* k = reinterpret_cast<uint32_t*>(u.base + j * u.row + 4 * lane);
        float v[4];
        e4m3x4_f32(*k, v);
        *k = e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
      }
    }
    if (lane == 0 && (kFull || !u.low || e > e_old)) *u.scale = pow2i(e);
  }
}

// A warp's rows of a run as pairs (x, y); rows past it repeat its row 0, row
// pairs past it are zero and count for nothing in the maximum.
template <typename T, int N, bool kFull, bool kInter>
__device__ __forceinline__ void load_rows(float (&x)[N][4], float (&y)[N][4], const T* src,
                                          int64_t stride, const Unit& u, int pairs, int da, int db,
                                          int grp) {
  const T* s = src + (kFull ? (u.row0 + grp) * stride : 0);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (kFull || j < pairs) {
      if (!kFull) {
        const int r = u.row0 + 2 * j + grp;
        s = src + (r < u.len ? r : 0) * stride;
      }
      to_pairs<T, kInter>(*reinterpret_cast<const uint2*>(s + da),
                          *reinterpret_cast<const uint2*>(s + db), x[j], y[j]);
      if (kFull) s += 2 * stride;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[j][c] = y[j][c] = 0.f;
    }
  }
}

// K rows in f64: norm, rotation, rounding to odd.  cs: the f64 table at the run's
// first token.
template <typename T, int N, bool kFull, bool kInter>
__device__ __forceinline__ void k_rows(float (&x)[N][4], float (&y)[N][4], const Unit& u,
                                       int pairs, const T* w, float eps, const double2* cs,
                                       int half, const LaneDims d, int lane) {
  const int sub = lane & 15, grp = lane >> 4;
  double inv = 1.0;
  float wx[4] = {1.f, 1.f, 1.f, 1.f}, wy[4] = {1.f, 1.f, 1.f, 1.f};
  if (w) {
    to_pairs<T, kInter>(*reinterpret_cast<const uint2*>(w + d.a),
                        *reinterpret_cast<const uint2*>(w + d.b), wx, wy);
    double ss[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      ss[j] = 0.0;
      if (kFull || j < pairs) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          ss[j] = fma((double)x[j][c], (double)x[j][c], ss[j]);
          ss[j] = fma((double)y[j][c], (double)y[j][c], ss[j]);
        }
      }
    }
    inv = rsqrt(half_sums<N>(ss, lane) * (1.0 / kApD) + (double)eps);
  }
  const double2* c64 = cs + (kFull ? (u.row0 + grp) * half : 0) + sub;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (kFull || j < pairs) {
      const double g = w ? __shfl_sync(0xffffffffu, inv, sum_lane<N>(j, lane)) : 1.0;
      if (!kFull) {
        const int r = u.row0 + 2 * j + grp;
        c64 = cs + (r < u.len ? r : 0) * half + sub;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        double a = x[j][c], b = y[j][c];
        if (w) {
          a *= (double)wx[c];
          b *= (double)wy[c];
        }
        if (d.rot) {
          const double2 k = c64[c * (half / 4)];
          const double a1 = a * k.x - b * k.y;
          b = b * k.x + a * k.y;
          a = a1;
        }
        x[j][c] = f32_odd(a * g);
        y[j][c] = f32_odd(b * g);
      }
    }
    if (kFull) c64 += 2 * half;
  }
}

// One unit: a run and kv head, K and (kWide) V.
template <typename T, int N, bool kWide, bool kFull, bool kInter>
__device__ __forceinline__ void unit(const AppendParams& p, Unit u, const T* ks, const T* vs,
                                     float* scale, int64_t block0, bool only_v, const double2* cs,
                                     const LaneDims d, float (*duo)[2], int warp, int lane) {
  const int sub = lane & 15, grp = lane >> 4, va = 8 * sub;  // V: eight neighbouring dims a lane
  const int pairs = max(1, (u.len - u.row0 + 1) / 2);        // row pairs in use
  float x[N][4], y[N][4], old_k = 0.f, old_v = 0.f;
  if (!kFull && u.low) old_k = scale[0], old_v = scale[1];
  if (only_v) {
    load_rows<T, N, kFull, false>(x, y, vs, p.v_stride, u, pairs, va, va + 4, grp);
  } else {
    load_rows<T, N, kFull, kInter>(x, y, ks, p.k_stride, u, pairs, d.a, d.b, grp);
    k_rows<T, N, kFull, kInter>(x, y, u, pairs, static_cast<const T*>(p.k_w), p.eps, cs, p.half, d,
                                lane);
  }
  float amax = warp_amax(x, y);
  if (kWide) {  // the other warp's; its scale has been read by the first barrier
    if (lane == 0) duo[warp][0] = amax;
    pair_barrier(warp);
    amax = fmaxf(amax, duo[warp ^ 1][0]);
  }
  u.base = static_cast<uint8_t*>(only_v ? p.v_cache : p.k_cache) + block0;
  u.scale = scale + (only_v ? 1 : 0);
  encode_rows<N, kFull>(x, y, u, only_v ? old_v : old_k, amax, only_v ? va : d.a,
                        only_v ? va + 4 : d.b, kInter && !only_v, lane);
  if (kWide) {
    load_rows<T, N, kFull, false>(x, y, vs, p.v_stride, u, pairs, va, va + 4, grp);
    float vmax = warp_amax(x, y);
    if (lane == 0) duo[warp][1] = vmax;
    pair_barrier(warp);
    vmax = fmaxf(vmax, duo[warp ^ 1][1]);
    u.base = static_cast<uint8_t*>(p.v_cache) + block0;
    u.scale = scale + 1;
    encode_rows<N, kFull>(x, y, u, old_v, vmax, va, va + 4, false, lane);
  }
}

// kWide: windows of several tokens (8 rows in flight a warp, two warps a run:
// registers for three CTAs an SM); else a decode step's single tokens (4 rows in
// flight, so that eight warps share 32 heads, and a warp a run, mostly one row).
template <typename T, bool kF8, bool kWide, bool kInter>
__global__ void __launch_bounds__(kApThreads, kWide ? 3 : 2)
    rope_append_kernel(const AppendParams p) {
  constexpr int kN = kWide ? 4 : 2, kRows = 2 * kN;
  constexpr int kM = kWide ? 4 : 8;  // row pairs of a warp's part of a run
  extern __shared__ __align__(16) uint8_t smem[];
  // f64 (cos, sin) of the run tokens, [token][pair % 4][pair / 4]: lanes read
  // neighbouring entries; then f32 ones, [token][half]
  double2* cs64 = reinterpret_cast<double2*>(smem);
  float2* cs = reinterpret_cast<float2*>(
      smem + (kF8 ? (size_t)(p.window + kApBlock - 1) * p.half * sizeof(double2) : 0));
  __shared__ int64_t slot_s[kApTable + 1];  // slots of tokens w0 - 1 ..
  __shared__ int lead_s[kApMaxWindow], len_s[kApMaxWindow], nrun_s, to_s;
  __shared__ float duo_s[kApWarps][2];
  const int64_t w0 = (int64_t)blockIdx.x * p.window;
  const int n = (int)min((int64_t)p.window, p.num_tokens - w0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane & 15;
  const LaneDims d = lane_dims<kInter>(sub, p.half);
  const T* qw = static_cast<const T*>(p.q_w);
  const T* kw = static_cast<const T*>(p.k_w);
  pdl_wait();  // nothing is read or written before: the launch may overlap the kernel before it
  // tables: a thread keeps one pair, 4 tokens a step
  const int pr = tid % 64;
  const double fr = pr < p.half ? p.inv_freq[pr] : 0.0;
  auto table = [&](int from, int to) {
    if (pr >= p.half) return;
    for (int t = from + tid / 64; t < to; t += kApThreads / 64) {
      if constexpr (kF8) {
        const double2 c = rope_cs64(p.positions[w0 + t], fr, p.a);
        cs64[t * p.half + (pr & 3) * (p.half / 4) + (pr >> 2)] = c;
        if (t < n) cs[t * p.half + pr] = make_float2((float)c.x, (float)c.y);
      } else {
        cs[t * p.half + pr] = rope_cs(p.positions[w0 + t], fr, (float)p.a);
      }
    }
  };
  table(0, n);
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
        to_s = leads ? end : 0;  // behind the last run's last token
      }
    }
  }
  __syncthreads();
  if (kF8) table(n, to_s);  // the last run may go on behind the window

  // rows of single tokens: a warp per token when the window is wide, else a few
  // heads of the token
  const int parts = kWide ? 1 : kApWarps, part = kWide ? 0 : warp;
  {
    for (int t = kWide ? warp : 0; t < n; t += kWide ? kApWarps : 1) {
      const int64_t tok = w0 + t;
      const Coef f = token_coef<T, kInter>(cs + t * p.half, qw, d, sub);
      for (int h = part * kRows; h < p.hq; h += parts * kRows)
        rows_f32<T, kN, kInter>(static_cast<const T*>(p.q) + tok * p.q_stride + (int64_t)h * kApD,
                                static_cast<T*>(p.q_out) + (tok * p.hq + h) * kApD,
                                min(kRows, p.hq - h), qw != nullptr, p.eps, f, d, lane);
    }
  }
  if constexpr (!kF8) {
    for (int t = kWide ? warp : 0; t < n; t += kWide ? kApWarps : 1) {
      const int64_t tok = w0 + t, slot = slot_s[t + 1];
      if (slot < 0) continue;
      const Coef f = token_coef<T, kInter>(cs + t * p.half, kw, d, sub);
      for (int h = part * kRows; h < p.hkv; h += parts * kRows)
        rows_f32<T, kN, kInter>(static_cast<const T*>(p.k) + tok * p.k_stride + (int64_t)h * kApD,
                                static_cast<T*>(p.k_cache) + (slot * p.hkv + h) * kApD,
                                min(kRows, p.hkv - h), kw != nullptr, p.eps, f, d, lane);
      const T* src = static_cast<const T*>(p.v) + tok * p.v_stride;
      T* dst = static_cast<T*>(p.v_cache) + slot * p.hkv * kApD;
#pragma unroll 4
      for (int c = part * 32 + lane; c < p.hkv * 32; c += parts * 32)
        *reinterpret_cast<uint2*>(dst + 4 * c) = *reinterpret_cast<const uint2*>(src + 4 * c);
    }
  } else {
    __syncthreads();  // the f64 table
    // units: (run, kv head), K then V by a pair of warps, or K and V apart by
    // single warps
    const int per = p.page / kApBlock, nu = nrun_s * p.hkv;
    for (int i = kWide ? warp >> 1 : warp; i < (kWide ? nu : 2 * nu);
         i += kWide ? kApWarps / 2 : kApWarps) {
      const bool only_v = !kWide && i >= nu;
      const int r = (only_v ? i - nu : i) / p.hkv, h = (only_v ? i - nu : i) % p.hkv;
      const int t = lead_s[r];
      Unit u;
      u.slot = slot_s + t + 1;
      u.len = len_s[r];
      u.row0 = kWide ? (warp & 1) * 8 : 0;
      const int64_t blk = u.slot[0] / kApBlock;
      u.low = (int)(u.slot[0] % kApBlock);
      u.row = (int64_t)p.hkv * kApD;
      const int64_t block0 = (blk * kApBlock * p.hkv + h) * kApD;
      float* scale = p.scale + (((blk / per) * p.hkv + h) * per + blk % per) * 2;
      const T* ks = static_cast<const T*>(p.k) + (w0 + t) * p.k_stride + (int64_t)h * kApD;
      const T* vs = static_cast<const T*>(p.v) + (w0 + t) * p.v_stride + (int64_t)h * kApD;
      const double2* c64 = cs64 + t * p.half;
      if (kWide && u.len == kApBlock)
        unit<T, kM, kWide, true, kInter>(p, u, ks, vs, scale, block0, false, c64, d, duo_s, warp,
                                         lane);
      else if (!kWide && u.len <= 2)  // a decode step's: one row pair
        unit<T, 1, kWide, false, kInter>(p, u, ks, vs, scale, block0, only_v, c64, d, duo_s, warp,
                                         lane);
      else
        unit<T, kM, kWide, false, kInter>(p, u, ks, vs, scale, block0, only_v, c64, d, duo_s, warp,
                                          lane);
    }
  }
}

template <typename T, bool kF8, bool kInter>
int launch_append(const AppendParams& p, dim3 grid, size_t smem, cudaStream_t s) {
  return launch_pdl(p.window > 1 ? rope_append_kernel<T, kF8, true, kInter>
                                 : rope_append_kernel<T, kF8, false, kInter>,
                    grid, dim3(kApThreads), smem, s, "rope_append launch", p);
}
template <typename T>
int launch_append(const AppendParams& p, dim3 grid, size_t smem, cudaStream_t s) {
  if (p.scale)
    return p.inter ? launch_append<T, true, true>(p, grid, smem, s)
                   : launch_append<T, true, false>(p, grid, smem, s);
  return p.inter ? launch_append<T, false, true>(p, grid, smem, s)
                 : launch_append<T, false, false>(p, grid, smem, s);
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
      num_kv_heads > 65536 || num_blocks <= 0 || page_size <= 0 ||
      num_blocks > INT64_MAX / page_size / ((int64_t)num_kv_heads * kApD * 2))
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
  const uint64_t pool = (uint64_t)num_blocks * page_size * kr * (kv_scale ? 1 : 2);
  const uint64_t k_bytes = (uint64_t)((num_tokens - 1) * k_stride + kr) * 2;
  const uint64_t v_bytes = (uint64_t)((num_tokens - 1) * v_stride + kr) * 2;
  const uint64_t q_bytes = q ? (uint64_t)((num_tokens - 1) * q_stride + qr) * 2 : 0;
  const uint64_t scales = pool / (kApBlock * kApD) * 8, qo_bytes = (uint64_t)num_tokens * qr * 2;
  const Span pos = {positions, (uint64_t)num_tokens * 8}, freq = {inv_freq, (uint64_t)rot_dim * 4};
  const Span slot = {slot_mapping, (uint64_t)num_tokens * 8};
  const Span qw = {q_norm_w, kApD * 2}, kw = {k_norm_w, kApD * 2};
  // what the call writes: q_out (whose own input rows are checked above), the caches
  // and the scales
  if (spans_meet(q_out, qo_bytes, {pos, freq, slot, qw, kw}))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: q_out overlaps metadata or weights");
  for (const Span& w : {Span{k_cache, pool}, Span{v_cache, pool}, Span{kv_scale, scales}})
    if (spans_meet(w.p, w.bytes, {{q, q_bytes}, {k, k_bytes}, {v, v_bytes}, {q_out, qo_bytes}, pos,
                                  freq, slot, qw, kw}))
      return set_error(NVKV_ERR_INVALID_ARG,
                       "rope_append: an input or q_out overlaps a cache or its scales");
  if (spans_meet(k_cache, pool, v_cache, pool) ||
      spans_meet(kv_scale, scales, {{k_cache, pool}, {v_cache, pool}}))
    return set_error(NVKV_ERR_INVALID_ARG, "rope_append: k_cache, v_cache and kv_scale overlap");
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
  // Two forms (see the kernel).  Block scales gain from two tokens a CTA on (32 + 8 + 8
  // heads, norms, single tokens / windows: 1184 tokens 26.1 / 24.6 us, 2400 39.1 / 28.2),
  // the dtype pool, whose warps then take whole tokens, from three (1184: 16.5 / 23.4,
  // 1800: 24.6 / 24.7, 2400: 31.6 / 26.4).
  if (!kv_scale && p.window < 3) p.window = 1;
  const int64_t ctas = (num_tokens + p.window - 1) / p.window;
  if (ctas > 0x7fffffffLL) return set_error(NVKV_ERR_INVALID_ARG, "rope_append: too many tokens");
  const size_t smem = (size_t)p.half * (p.window * sizeof(float2) +
                                        (kv_scale ? (p.window + kApBlock - 1) * sizeof(double2) : 0));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == NVKV_DTYPE_BF16 ? launch_append<__nv_bfloat16>(p, dim3((unsigned)ctas), smem, s)
                                  : launch_append<__half>(p, dim3((unsigned)ctas), smem, s);
}
