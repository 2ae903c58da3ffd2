// Decode attention over the block-scaled e4m3 pool, on tcgen05 (sequences of a
// few query tokens: rows = q_len x (Hq / Hkv) <= 32).
//
// A CTA streams a sequence's keys for one kv head, 128 keys a tile, and serves all
// its rows, so every code leaves HBM once.  Both products run on the tensor cores with the
// codes exactly as TMA put them into shared memory -- nothing is converted:
//   S^T [128 keys x rows] = K codes (A, K-major) . Q^T (B)
//   O^T [128 dims x rows] += V codes^T (A, MN-major) . P^T (B)
// Q enters as three e4m3 pieces, the weights P as four, every piece the e4m3
// rounding of what the ones before left over.  The pieces are extra columns of B
// (the tensor core's N has room), and are joined in f32 with their weights where
// the columns are read.
//
// A compute thread owns one key of the tile (one TMEM lane) and up to 8 of its
// rows: it joins its scores S, multiplies by the key block's K scale, and forms z =
// S + ev, ev = log2(V scale), so a weight 2^(z - M) already carries the value's scale
// and O needs none; the row sum takes the scale back out (an exact power of two).  M
// is a row's maximum of z over the CTA's keys, to within a headroom: one barrier with
// a reduced flag a tile says whether any score has left it; only then are maxima
// joined (redux.sync in a warp, shared memory over the four) and O rescaled in TMEM.
// Weights leave as 8- or 16-byte stores (N-major B operand).
//
// V scales may lie 2^220 apart (a block of zero values has the least one), and a key
// whose z is 126 below M would be flushed to 0 before the row sum could take its scale
// back out.  So the exponential of a key whose ev is more than kBelow below E, the
// largest ev so far to within kAbove, is taken 2^d higher, d = E - kBelow - ev, and the
// weight multiplied by 2^-d: weights are as before, and what the sum (in units of
// 2^(M - E)) can lose is below 2^(kBelow + kAbove - 126) = 2^-62 of a row's largest.
// The sum itself holds rows whose keys of large values weigh down to 2^-126 of the
// others.  (A second maximum and exponential, of S alone, for every key: 16 rows 86
// us against 80, 32 rows 82 against 77; a branch to them from the first tile that
// needs it: 82 and 78.)
//
//   G warpgroups  compute, G = 1, or rows / 8 for 16 and 32 rows (a warp has TMEM
//              lanes 32 (w % 4) ..): the chain of a tile, not its issue, sets their
//              pace, so rows go side by side
//   a warp     TMA producer: K and V code tiles (SWIZZLE_128B) and the tile's
//              64 bytes of scales, an mbarrier ring
//   a warp     TMEM allocation and every tcgen05.mma, one thread, in the order
//              S(0), S(1), O(0), S(2), O(1), ...: a tile's scores are computed
//              while the tile before it is in the softmax
//   two warps  the next sequence's Q pieces
//
// Work.  One wave of persistent CTAs, a group of Hkv neighbours (one per kv head)
// for each share of the batch: the sequences' tiles, one after the other, are cut
// into equal shares wherever the cuts fall, so every SM has the same number of
// tiles whatever the lengths, and ring, tensor memory and barriers are set up
// once.  (A CTA per (split, head, sequence) lost ~6 us of its 14 to its start and
// end.)  A share's whole sequences are written out; of a sequence that a cut goes
// through, each CTA leaves f32 partials and a base-2 log-sum-exp in the workspace
// (at most two per CTA), and combine_fp8b_kernel joins them.  Where the sequences are about
// as many as the shares and not far from equal, each is a share, uncut.
//
// Bound by HBM up to 8 rows where sequences are long: 2 x 128 bytes of codes + 0.5 of
// scales a key and kv head.  256 sequences of ~1290 keys, 32 / 8 heads (681 MB): 115.1
// us, 5.9 TB/s of the 6.55 that a copy reaches; the same loads without products 96 us.
// 64 x 32768 keys, 8 / 1 heads: 90-91.5 us, 5.9-6.0 TB/s.  With 8 rows and 512-4096
// keys (64 sequences, 8 kv heads, 305 MB) 62.9 us, 4.8 TB/s: the tile's chain and the
// parts' ends show.  16 rows (64 x 2000 keys, 32 / 8 heads, 4 queries each, 267 MB):
// 80.5 us, bound by the tile's chain of scores, weights and the issue of 8 products; 32
// rows (32 / 4 heads, 136 MB): 77.  Earlier forms at 16 rows: one warpgroup for all 87,
// and 2 CTAs of 2 stages instead of one of 6 then 85 (but 31.5 against 30.6 at 64 x
// 3000 keys of one head).
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "tcgen05.cuh"

namespace nvkv {
namespace {

constexpr int kBD = 128;
constexpr int kBTile = 128;                   // keys a tile
constexpr int kBCode = kBTile * kBD;          // 16 KB of codes
constexpr int kBStage = 2 * kBCode;           // K, V
constexpr int kBScale = kBTile / NVKV_FP8B_BLOCK * 2;  // floats of a tile's scales
constexpr float kLog2e_ = 1.4426950408889634f;
// Q and the weights P as sums of e4m3 pieces, x = c0 + 2^-5 c1 + 2^-10 c2 + ...,
// every piece the e4m3 rounding of what the ones before left over (at most 8 of a
// value below 256, so 32 times it fits again): 4 more bits each.
constexpr int kQPieces = 3, kPPieces = 4;
constexpr float kPiece1 = 1.f / 32.f, kPiece2 = 1.f / 1024.f, kPiece3 = 1.f / 32768.f;
// M is kept until a row's maximum passes it by this much (weights then reach 2^3):
// rescaling O waits for the product before it, and with M exact more than half of
// the first ten tiles of random scores did so.  Weights enter the pieces times
// 2^(8 - 3), so that the largest is 256; a weight down to 2^-17 of the largest
// keeps 12 bits.  (Three pieces, which the same number of columns would do for 4
// and 8 rows, keep 9 bits at 2^-15: too few where one key takes nearly all of the
// weight and the answer lies in the others.)
constexpr float kHeadroom = 3.f;
constexpr int kWeightLog2 = 5;
// Maxima of no keys yet: finite, so that the score of a hidden key, -inf, less it is -inf.
constexpr float kNoMax = -3e38f;
constexpr int kBelow = 48, kAbove = 16;

// Rows a CTA serves, padded: 4, 8, 16 or 32; its resources by that.
template <int HP>
struct Cfg {
  static constexpr int kCols = (kQPieces * HP + 15) / 16 * 16;  // pieces as B columns
  static constexpr int kPCols = kPPieces * HP;
  // compute warpgroups, each with its rows of a tile
  static constexpr int kGroups = HP <= 8 ? 1 : HP / 8, kRows = HP / kGroups;
  static constexpr int kThreads = 128 * kGroups + 128;
  static constexpr int kCtasPerSm = HP <= 8 ? 2 : 1;
  static constexpr int kStages = HP <= 8 ? 3 : HP == 16 ? 6 : 5;
  static constexpr int kQBytes = kCols * 128;
  // from the first Q buffer to the second: at 8 rows the 8 unused columns of the
  // first may be the second's rows (their scores are never read), so that two CTAs fit
  static constexpr int kQStride = HP == 8 ? 3 * HP * 128 : kQBytes;
  static constexpr int kPBytes = kPCols * 128;  // one of two buffers
  static constexpr int kUsed = 2 * kCols + kPCols;  // tensor-memory columns: two S, one O
  static constexpr int kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static constexpr int kOffQ = kStages * kBStage;
  static constexpr int kOffP = (kOffQ + kQStride + kQBytes + 1023) / 1024 * 1024;
  static constexpr int kOffScale = kOffP + 2 * kPBytes;
  static constexpr int kOffRed = kOffScale + kStages * kBScale * 4;  // [4][HP] maxima, sums
  static constexpr int kOffRow = kOffRed + 4 * HP * 4;           // [2][HP] factors, [HP] limits
  static constexpr int kOffBar = kOffRow + 3 * HP * 4;
  static constexpr int kBars = 2 * kStages + 11;
  static constexpr int kSmem = kOffBar + kBars * 8 + 16 + 1024;
  static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "decode fp8b: CTAs per SM");
  static_assert(kCtasPerSm * kTmem <= 512, "decode fp8b: tensor memory per SM");
};

struct Params {
  const void* q;
  int64_t q_stride;
  void* out;
  const uint32_t *cu_q, *cu_k, *block_tables;
  int64_t bt_stride, num_blocks, num_q_rows;
  const float* scale;
  int num_seqs, hq, hkv, group, groups, page, max_k, q_cap, all, causal;
  float scale_log2;
  // partials: slot 2 cta (a sequence that began in an earlier share) and 2 cta + 1
  // (one that goes on in a later share)
  int2* ws_desc;         // [2 ctas] {sequence or -1, 1: the sequence's last part}
  float *ws_lse, *ws_o;  // [2 ctas][q_cap * group] (x 128)
  int* err;
};

// A sequence as the kernel sees it.
struct Seq {
  uint32_t q0;
  int q_len, k_len, tiles;
};
// tiles = 0: nothing to do (another kernel's, or malformed: *err then gets a code
// if it is not null).  zero: rows without keys, whose output is 0.
__device__ __forceinline__ Seq read_seq(const Params& p, int b, int* err, bool* zero) {
  Seq s;
  s.q0 = p.cu_q[b];
  s.q_len = (int)(p.cu_q[b + 1] - s.q0);
  s.k_len = (int)(p.cu_k[b + 1] - p.cu_k[b]);
  s.tiles = 0;
  const bool other = s.q_len < 0 || s.q_len > p.q_cap;
  if (s.q_len == 0 || (other && !p.all)) return s;
  if (other || s.k_len > p.max_k || (int64_t)s.q0 + s.q_len > p.num_q_rows ||
      (s.q_len > 1 && s.k_len < s.q_len)) {
    if (err) record_error(err, NVKV_DEVERR_SEQLEN);
    return s;
  }
  if (s.k_len <= 0) {
    if (err) record_error(err, NVKV_DEVERR_SEQLEN);
    if (zero) *zero = true;
    return s;
  }
  s.tiles = (s.k_len + kBTile - 1) / kBTile;
  return s;
}

// A warp's walk over the share's sequences: lane i holds sequence base + i.
struct Cursor {
  Seq mine;
  int base, b, t, left;  // sequence, its first tile here, tiles left of the share
  __device__ __forceinline__ void fill(const Params& p, int lane) {
    base = b;
    mine.tiles = 0;
    if (b + lane < p.num_seqs) mine = read_seq(p, b + lane, nullptr, nullptr);
  }
  __device__ __forceinline__ void start(const Params& p, int b0, int t0, int n, int lane) {
    b = b0;
    t = t0;
    left = n;
    fill(p, lane);
  }
  // the next part: false when the share is done
  __device__ __forceinline__ bool next(const Params& p, Seq& s, int& n, int lane) {
    if (left <= 0) return false;
    for (;;) {
      if (b - base >= 32) fill(p, lane);
      s.tiles = __shfl_sync(0xffffffffu, mine.tiles, b - base);
      if (s.tiles > 0 || b >= p.num_seqs) break;
      ++b;
    }
    s.q0 = __shfl_sync(0xffffffffu, mine.q0, b - base);
    s.q_len = __shfl_sync(0xffffffffu, mine.q_len, b - base);
    s.k_len = __shfl_sync(0xffffffffu, mine.k_len, b - base);
    n = min(s.tiles - t, left);
    left -= n;
    return n > 0;
  }
  __device__ __forceinline__ void advance() {
    ++b;
    t = 0;
  }
};

// Shared-memory descriptors as two words: the low one holds the address (in 16
// bytes, so moving on within shared memory is one 32-bit add) and LBO, the high
// one SBO, the version bit and the layout (2: SWIZZLE_128B, 0: none).
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) {
  return (saddr >> 4) | ((lbo >> 4) << 16);
}
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo, uint32_t layout) {
  return (sbo >> 4) | (1u << 14) | (layout << 29);
}
// kind::f8f6f4, e4m3 x e4m3, f32 accumulate, M = 128
__host__ __device__ constexpr uint32_t idesc_f8(int n, uint32_t a_mn, uint32_t b_mn) {
  return (1u << 4) | (a_mn << 15) | (b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                       uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
// A wait that has mostly ended already: one test (a try_wait may suspend the
// thread, and took ~220 cycles even on a finished phase), then the bounded wait.
__device__ __forceinline__ bool mbar_ready(uint64_t* bar, uint32_t parity, int* err) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, ok)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}
// One lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// The barrier of a compute warpgroup
__device__ __forceinline__ void bar_compute(int g) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
}
// and returning whether any thread's flag was set.
__device__ __forceinline__ bool bar_compute_any(int g, bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)flag), "r"(1 + g)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// n (4 or 8) consecutive f32 columns of this thread's TMEM lane
template <int n>
__device__ __forceinline__ void tmem_ldn(uint32_t a, float* v) {
  static_assert(n == 4 || n == 8, "tmem_ldn");
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  if constexpr (n == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(a));
}

// e4m3 codes of (a, b), low byte a
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 a;\n\tcvt.u16.u32 a, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}"
      : "=r"(h)
      : "r"(w));
  return DT<__half>::to_f2(h);
}
// Four values (0 <= |x| <= 256) as N pieces: w[p] = the codes of piece p.
template <int N>
__device__ __forceinline__ void pieces4(float a, float b, float c, float d, uint32_t (&w)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const uint32_t lo = e4m3x2(a, b), hi = e4m3x2(c, d);
    w[p] = lo | (hi << 16);
    if (p < N - 1) {
      const float2 x = e4m3x2_f32(lo), y = e4m3x2_f32(hi);
      a = (a - x.x) * 32.f;
      b = (b - x.y) * 32.f;
      c = (c - y.x) * 32.f;
      d = (d - y.y) * 32.f;
    }
  }
}

// The rows' queries as B of the first product: row p HP + r of Q (128 bytes,
// SWIZZLE_128B) holds piece p of q row r times a power of two that puts the
// row's largest |q| into [128, 256); rowf[r] undoes it (times the softmax
// scale).  Rows past `rows` are zero.  Two warps (w = 0, 1).
template <typename T, int HP>
__device__ __forceinline__ void load_q(const Params& p, uint32_t q0, int kvh, int rows,
                                       uint8_t* sq, float* rowf, int w, int lane) {
#pragma unroll 4
  for (int r = w; r < HP; r += 2) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const T* src = static_cast<const T*>(p.q) + (int64_t)(q0 + r / p.group) * p.q_stride +
                     (int64_t)(kvh * p.group + r % p.group) * kBD + 4 * lane;
      const uint2 raw = *reinterpret_cast<const uint2*>(src);
      const float2 u = DT<T>::to_f2(raw.x), v = DT<T>::to_f2(raw.y);
      x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
    }
    float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    m = redux_max(m);
    const int e = (int)(__float_as_uint(m) >> 23);
    const int sh = m > 0.f ? min(127, 134 - e) : 0;  // m 2^sh in [128, 256)
    const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // an infinite query gives NaN, as its scores would
      x[i] = fabsf(x[i]) < INFINITY ? x[i] * up : __int_as_float(0x7fffffff);
    uint32_t c[kQPieces];
    pieces4(x[0], x[1], x[2], x[3], c);
#pragma unroll
    for (int pc = 0; pc < kQPieces; ++pc) {
      const int n = pc * HP + r;
      *reinterpret_cast<uint32_t*>(sq + n * 128 + (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4) =
          c[pc];
    }
    if (lane == 0) rowf[r] = __uint_as_float((uint32_t)(127 - sh) << 23) * p.scale_log2;
  }
}

template <typename T, int HP>
__global__ void __launch_bounds__(Cfg<HP>::kThreads, Cfg<HP>::kCtasPerSm)
    decode_fp8b_kernel(const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const Params p) {
  using C = Cfg<HP>;
  constexpr int kStages = C::kStages, kCols = C::kCols, kThreads = C::kThreads, R = C::kRows;
  constexpr int kTma = 4 * C::kGroups, kMma = kTma + 1, kLoadQ = kTma + 2;  // warps
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem + C::kOffQ;
  uint8_t* sp = smem + C::kOffP;
  float* ssc = reinterpret_cast<float*>(smem + C::kOffScale);
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  float* rowf = reinterpret_cast<float*>(smem + C::kOffRow);
  int* rowlim = reinterpret_cast<int*>(rowf + 2 * HP);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + kStages;
  uint64_t* s_full = empty + kStages;  // [2] scores of a tile are in TMEM
  uint64_t* p_full = s_full + 2;       // [2] scores read, weights in shared memory, O rescaled
  uint64_t* o_done = p_full + 2;       // [2] the tile's O product has finished
  uint64_t* q_full = o_done + 2;       // [2] a sequence's Q pieces and row factors
  uint64_t* q_empty = q_full + 2;      // [2] its last scores are done, its factors read
  uint64_t* drain = q_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int tops[kThreads / 32];
  __shared__ int start_b, start_t;
  __shared__ int4 top_ev[C::kGroups];  // the four warps' largest ev

  const int cta = blockIdx.x, share = cta / p.hkv, kvh = cta % p.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == kTma * 32) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 128 * C::kGroups);
      mbar_init(&o_done[x], 1);
      mbar_init(&q_full[x], 64);
      mbar_init(&q_empty[x], 128 * C::kGroups + 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < (C::kQStride + C::kQBytes) / 16; i += kThreads)  // the unused columns
    *reinterpret_cast<uint4*>(sq + i * 16) = make_uint4(0, 0, 0, 0);
  pdl_wait();  // inputs may come from the kernel before this one

  // ---- this CTA's share of the tiles: [lo, hi) of their total ----
  const int each = (p.num_seqs + kThreads - 1) / kThreads;  // sequences a thread
  const int b_lo = threadIdx.x * each, b_hi = min(b_lo + each, p.num_seqs);
  int64_t mine = 0;
  int top = 0;  // tiles of the longest sequence
  for (int b = b_lo; b < b_hi; ++b) {
    bool zero = false;
    const Seq s = read_seq(p, b, cta == 0 ? p.err : nullptr, &zero);
    mine += s.tiles;
    top = max(top, s.tiles);
    if (zero && share == 0)
      for (int r = 0; r < s.q_len * p.group; ++r) {
        uint4* o = reinterpret_cast<uint4*>(
            static_cast<T*>(p.out) +
            ((int64_t)(s.q0 + r / p.group) * p.hq + kvh * p.group + r % p.group) * kBD);
        for (int i = 0; i < kBD / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
      }
  }
  int64_t upto = mine;  // inclusive prefix sum over the threads
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += v;
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 31) sums[warp] = upto, tops[warp] = top;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
    top = max(top, tops[w]);
  }
  const int64_t used = min((int64_t)p.groups, total);  // shares of at least a tile
  if (threadIdx.x < 2) p.ws_desc[2 * cta + threadIdx.x] = make_int2(-1, 0);
  // Sequences that nearly fill the shares by their number, the longest at most 8 tiles
  // above an equal share, get a share each: no cuts, no parts to join.  One head, 4
  // rows, cut / a share each: 256 x 1280 keys (extra 1 tile) 24.6 / 21.4 us, 200 x 4096
  // (10) 42.5 / 40.6, 148 x 2048 (8) 21.3 / 21.2, 148 x 4096 (16) 33.0 / 34.3, 20 x 640
  // (4, few sequences) 10.2 / 10.2.
  const bool apart = p.num_seqs <= p.groups && 2 * p.num_seqs >= p.groups &&
                     top * used <= total + 8 * used;
  if (share >= (apart ? p.num_seqs : used)) return;
  int64_t lo = 0, hi = 0;
  if (apart) {
    const int n = read_seq(p, share, nullptr, nullptr).tiles;
    if (n == 0) return;
    hi = n;
    if (threadIdx.x == 0) start_b = share, start_t = 0;
  } else {
    lo = total * share / used;
    hi = total * (share + 1) / used;
    if (upto - mine <= lo && lo < upto) {  // the thread whose sequences hold the first tile
      int64_t at = upto - mine;
      for (int b = b_lo;; ++b) {
        const int n = read_seq(p, b, nullptr, nullptr).tiles;
        if (lo < at + n) {
          start_b = b;
          start_t = (int)(lo - at);
          break;
        }
        at += n;
      }
    }
  }
  if (warp == kMma) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  fence_async_smem();  // Q's zeros
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // only now, with this CTA's tensor memory in hand, may the next grid start
  pdl_launch_dependents();
  Cursor cur;
  cur.start(p, start_b, start_t, (int)(hi - lo), lane);
  Seq sq_info;
  int n_tiles;

  if (warp == kTma) {
    // ------------------------------ TMA producer ------------------------------
    int it = 0, go = 1;
    while (go && cur.next(p, sq_info, n_tiles, lane)) {
      const uint32_t* row_bt = p.block_tables + (int64_t)cur.b * p.bt_stride;
      int base = cur.t * kBTile / p.page;  // page of lane 0's entry
      uint32_t ent = base + lane < p.bt_stride ? __ldg(row_bt + base + lane) : 0u;
      for (int i = 0; i < n_tiles; ++i, ++it) {
        const int s = it % kStages;
        const int j0 = (cur.t + i) * kBTile;
        const int pg = j0 / p.page;
        if (pg >= base + 32) {  // warp-uniform: the next 32 entries
          base = pg;
          ent = base + lane < p.bt_stride ? __ldg(row_bt + base + lane) : 0u;
        }
        uint32_t page = __shfl_sync(0xffffffffu, ent, pg - base);
        if ((int64_t)page >= p.num_blocks) {  // recorded; read as page 0 so that the rest finishes
          if (lane == 0) record_error(p.err, NVKV_DEVERR_BLOCK_RANGE);
          page = 0;
        }
        if (lane == 0) {
          go = it < kStages || mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, p.err);
          if (go) {
            const int off = j0 - pg * p.page;
            const int row = (int)((int64_t)page * p.page + off);
            uint8_t* st = smem + s * kBStage;
            mbar_arrive_expect_tx(&full[s], kBStage + kBScale * 4);
            tma_load_3d(st, &tmap_k, &full[s], 0, kvh, row);
            tma_load_3d(st + kBCode, &tmap_v, &full[s], 0, kvh, row);
            bulk_load(ssc + s * kBScale,
                      p.scale + (((int64_t)page * p.hkv + kvh) * (p.page / NVKV_FP8B_BLOCK) +
                                 off / NVKV_FP8B_BLOCK) * 2,
                      kBScale * 4, &full[s]);
          }
        }
        go = __shfl_sync(0xffffffffu, go, 0);
        if (!go) break;
      }
      cur.advance();
    }
    if (!go && lane == 0)  // given up: wait for the copies in flight
      for (int i = max(0, it - kStages); i < it; ++i)
        mbar_wait(&full[i % kStages], (i / kStages) & 1, p.err);
  } else if (warp == kMma) {
    // ------------------------------- MMA issuer -------------------------------
    // The whole warp walks the loop, one lane issues: the loop is the critical path
    // of a tile, so descriptors move by 32-bit adds and ring positions by compares.
    constexpr uint32_t id_s = idesc_f8(kCols, 0, 0), id_o = idesc_f8(C::kPCols, 1, 1);
    constexpr uint32_t hi128 = desc_hi(1024, 2), hi_p = desc_hi(2048, 0);
    const uint32_t k0 = desc_lo(smem_u32(smem), 16), v0 = k0 + (kBCode >> 4);
    const uint32_t p0 = desc_lo(smem_u32(sp), 128);
    uint32_t s_st = 0, s_ph = 0, o_st = 0;  // ring positions of the S and O products
    int it = 0, part = 0;
    bool ok = true;
    uint32_t more = 0;  // 0: tile it - 1 was its part's first
    // O += V^T . P of tile it - 1: 32 keys a step
    auto issue_o = [&] {
      const uint32_t x = (uint32_t)(it - 1) & 1u;
      ok = ok && mbar_ready(&p_full[x], ((uint32_t)(it - 1) >> 1) & 1u, p.err);
      if (!ok) return;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t v = v0 + o_st * (kBStage >> 4), pb = p0 + x * (C::kPBytes >> 4);
#pragma unroll
        for (uint32_t kk = 0; kk < 4; ++kk)
          mma_f8(tmem + 2 * kCols, v + kk * (32 * 128 >> 4), hi128, pb + kk * (512 >> 4), hi_p, id_o,
                 kk > 0 ? 1u : more);
        tc_commit(&o_done[x]);
        tc_commit(&empty[o_st]);
      }
      __syncwarp();
      o_st = o_st + 1 == kStages ? 0 : o_st + 1;
    };
    for (; cur.next(p, sq_info, n_tiles, lane); ++part, cur.advance()) {
      const int qb = part & 1;
      const uint32_t q = desc_lo(smem_u32(sq + qb * C::kQStride), 16);
      ok = ok && mbar_ready(&q_full[qb], (part >> 1) & 1, p.err);
      for (int i = 0; i < n_tiles; ++i, ++it) {
        ok = ok && mbar_ready(&full[s_st], s_ph, p.err);
        if (ok) {  // S(it): K-major codes, 32 dims a step
          tc_fence_after();
          if (elect_one()) {
            const uint32_t k = k0 + s_st * (kBStage >> 4);
#pragma unroll
            for (uint32_t kk = 0; kk < 4; ++kk)
              mma_f8(tmem + (it & 1) * kCols, k + kk * 2, hi128, q + kk * 2, hi128, id_s, kk > 0);
            tc_commit(&s_full[it & 1]);
            if (i == n_tiles - 1) tc_commit(&q_empty[qb]);
          }
          __syncwarp();
          s_st = s_st + 1 == kStages ? 0 : s_st + 1;
          s_ph ^= s_st == 0 ? 1u : 0u;
        }
        if (it > 0) issue_o();
        more = i > 0 ? 1u : 0u;
      }
    }
    issue_o();
    if (!ok && elect_one()) {  // given up: let the products in flight finish before the memory goes
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr);
    }
  } else if (warp >= kLoadQ) {
    // -------------------------------- Q loaders --------------------------------
    int part = 0;
    bool ok = true;
    while (cur.next(p, sq_info, n_tiles, lane)) {
      const int qb = part & 1;
      if (part >= 2)
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&q_empty[qb], ((part >> 1) & 1) ^ 1,
                                                     p.err));
      if (ok) {
        load_q<T, HP>(p, sq_info.q0, kvh, sq_info.q_len * p.group, sq + qb * C::kQStride,
                      rowf + qb * HP, warp - kLoadQ, lane);
        fence_async_smem();
        mbar_arrive(&q_full[qb]);
      }
      ++part;
      cur.advance();
    }
  } else {
    // ------------------------------ compute warps ------------------------------
    const int grp = C::kGroups == 1 ? 0 : warp / 4, wg = warp % 4, r0 = grp * R;  // rows r0 ..
    const uint32_t lane_addr = tmem + ((uint32_t)(wg * 32) << 16);
    const int key = threadIdx.x % 128;  // this thread's key of a tile, and its dim of O
    bool alive = true;
    int it = 0, part = 0, st = 0;  // st, st_ph: ring position
    uint32_t st_ph = 0;
    for (; cur.next(p, sq_info, n_tiles, lane); ++part, cur.advance()) {
    const int qb = part & 1;
    const int rows = sq_info.q_len * p.group, k_len = sq_info.k_len;
    const uint32_t q0 = sq_info.q0;
    if (key < R) {
      const int r = r0 + key;
      rowlim[r] = r >= rows ? -1 : p.causal ? k_len - sq_info.q_len + r / p.group : k_len - 1;
    }
    // a wait that runs out is not repeated, but the warp stays in step with the
    // others' barriers to the end of the share
    alive = alive && __all_sync(0xffffffffu,
                                mbar_wait(&q_full[qb], (part >> 1) & 1, p.err));
    bar_compute(grp);  // rowlim
    float M[R], l[R], rf_r[R];  // (unused rows: no score passes infinity, every weight is 0)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = r0 + r < rows ? kNoMax : INFINITY;
      l[r] = 0.f;
      rf_r[r] = rowf[qb * HP + r0 + r];
    }
    const int seen = p.causal ? k_len - sq_info.q_len + 1 : k_len;  // keys that every row sees
    int E = -100;
    for (int i = 0; i < n_tiles; ++i, ++it) {
      const int s = st, x = it & 1;
      alive = alive && mbar_ready(&s_full[x], (it >> 1) & 1, p.err) &&
              mbar_ready(&full[s], st_ph, p.err);
      st = st + 1 == kStages ? 0 : st + 1;
      st_ph ^= st == 0 ? 1u : 0u;
      tc_fence_after();
      const float2 sc = *reinterpret_cast<const float2*>(ssc + s * kBScale +
                                                         key / NVKV_FP8B_BLOCK * 2);
      const float ks = sc.x;
      // log2 of the V scale, a power of two (a cleared pool's 0 counts as the least; a
      // key past the end may have a stale block's)
      const int j = (cur.t + i) * kBTile + key;
      const int ev = j < k_len ? min(max((int)(__float_as_uint(sc.y) >> 23 & 0xffu) - 127, -100), 120)
                               : E;
      int d = max(E - kBelow - ev, 0);
      float z[R];  // (+ d)
      const uint32_t cs = lane_addr + x * kCols + r0;
      if constexpr (R == 4) {
        float a[16];
        tmem_ld16(cs, a);
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < 4; ++r)
          z[r] = a[r] + a[4 + r] * kPiece1 + a[8 + r] * kPiece2;
      } else {
        float a0[8], a1[8], a2[8];
        tmem_ldn<8>(cs, a0);
        tmem_ldn<8>(cs + HP, a1);
        tmem_ldn<8>(cs + 2 * HP, a2);
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < 8; ++r)
          z[r] = a0[r] + a1[r] * kPiece1 + a2[r] * kPiece2;
      }
      float top = ev > E + kAbove ? INFINITY : -INFINITY;
#pragma unroll
      for (int r = 0; r < R; ++r) z[r] = z[r] * (rf_r[r] * ks) + (float)(ev + d);
      if ((cur.t + i + 1) * kBTile > seen) {
#pragma unroll
        for (int r = 0; r < R; ++r) z[r] = j <= rowlim[r0 + r] ? z[r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) top = fmaxf(top, z[r] - M[r]);
      if (bar_compute_any(grp, top > kHeadroom)) {
        // new maxima: of the warp's keys, lane r keeping row r's, then of the four warps'
        float mine = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m = redux_max(z[r] - (float)d);
          if (lane == r) mine = m;
        }
        if (lane < R) red[wg * HP + r0 + lane] = mine;
        const int warp_ev = __reduce_max_sync(0xffffffffu, ev);
        if (lane == 0) reinterpret_cast<int*>(&top_ev[grp])[wg] = warp_ev;
        bar_compute(grp);
        const int4 te = top_ev[grp];
        const int up_e = max(max(max(te.x, te.y), max(te.z, te.w)) - E, 0);
        const float fac_e = ex2_mufu((float)min(up_e, 126));
        float fac[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float* x = red + r0 + r;
          const float m = fmaxf(fmaxf(x[0], x[HP]), fmaxf(x[2 * HP], x[3 * HP]));
          const bool up = m > M[r] + kHeadroom;
          fac[r] = up ? ex2_mufu(M[r] - m) : 1.f;
          l[r] *= up ? ex2_mufu(M[r] - m + (float)up_e) : fac_e;
          M[r] = up ? m : M[r];
        }
        E += up_e;
        const int more = max(E - kBelow - ev, 0) - d;
        d += more;
#pragma unroll
        for (int r = 0; r < R; ++r) z[r] += (float)more;
        bar_compute(grp);  // (the next exchange may be the next tile's)
        if (i > 0) {  // O is in units of 2^M
          alive = alive && mbar_ready(&o_done[x ^ 1], ((it - 1) >> 1) & 1, p.err);
          tc_fence_after();
#pragma unroll 1
          for (int pc = 0; pc < kPPieces; ++pc) {
            const uint32_t a = lane_addr + 2 * kCols + pc * HP + r0;
            float o[R];
            tmem_ldn<R>(a, o);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] *= fac[r];
            const uint32_t* w = reinterpret_cast<const uint32_t*>(o);
            if constexpr (R == 4)
              asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a),
                           "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                           : "memory");
            else
              asm volatile(
                  "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(
                      a),
                  "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                  "r"(w[7])
                  : "memory");
          }
          tmem_wait_st();
        }
      }
      // weights, scaled for the pieces; the row sums without the V scale
      const float unscale = pow2(E - ev - d), weight = pow2(max(kWeightLog2 - d, -126));
      uint32_t w[kPPieces * R / 4];
#pragma unroll
      for (int c = 0; c < R; c += 4) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = ex2_mufu(z[c + r] - M[c + r]);
          l[c + r] += e[r] * unscale;
          e[r] *= weight;
        }
        uint32_t pw[kPPieces];
        pieces4(e[0], e[1], e[2], e[3], pw);
#pragma unroll
        for (int pc = 0; pc < kPPieces; ++pc) w[(pc * R + c) / 4] = pw[pc];
      }
      if (it >= 2)  // this buffer's last reader
        alive = alive && mbar_ready(&o_done[x], ((it - 2) >> 1) & 1, p.err);
      uint8_t* dst = sp + x * C::kPBytes + key * 16;
      if constexpr (C::kGroups == 1) {
#pragma unroll
        for (int nb = 0; nb < C::kPCols / 16; ++nb)
          *reinterpret_cast<uint4*>(dst + nb * 2048) =
              make_uint4(w[4 * nb], w[4 * nb + 1], w[4 * nb + 2], w[4 * nb + 3]);
      } else {  // piece pc of these eight rows is half of a block of 16 columns
#pragma unroll
        for (int pc = 0; pc < kPPieces; ++pc) {
          const int n = pc * HP + r0;
          *reinterpret_cast<uint2*>(dst + n / 16 * 2048 + n % 16) = make_uint2(w[2 * pc], w[2 * pc + 1]);
        }
      }
      if (grp == 0 && j >= k_len) {  // a key past the end: its V row may hold NaN codes, and 0 x NaN is NaN
        uint8_t* vr = smem + s * kBStage + kBCode + key * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vr + c * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_async_smem();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }

    mbar_arrive(&q_empty[qb]);  // this part's row factors have been read

    // ------------------------------- epilogue -------------------------------
    alive = alive && __all_sync(0xffffffffu, mbar_wait(&o_done[(it - 1) & 1],
                                                       ((it - 1) >> 1) & 1, p.err));
    tc_fence_after();
    // row sums: of the warp, each step of the first ones halving the rows a lane
    // keeps, then of the four warps; lane r goes on with row r
    int m = 16;
#pragma unroll
    for (int half = R / 2; half >= 1; half >>= 1, m >>= 1) {
      const bool up = lane & m;
#pragma unroll
      for (int r = 0; r < half; ++r) {
        const float send = up ? l[r] : l[r + half], keep = up ? l[r + half] : l[r];
        l[r] = keep + __shfl_xor_sync(0xffffffffu, send, m);
      }
    }
    for (; m >= 1; m >>= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], m);
    if (lane % (32 / R) == 0) red[wg * HP + r0 + lane / (32 / R)] = l[0];
    bar_compute(grp);  // (the next part's first one is before the next write to red)
    const bool whole = n_tiles == sq_info.tiles;
    const int slot = 2 * cta + (cur.t == 0 ? 1 : 0);
    if (!whole && threadIdx.x == 0)
      p.ws_desc[slot] = make_int2(alive ? cur.b : -1, cur.t + n_tiles == sq_info.tiles);
    const int r_ = r0 + lane % R;
    float ls = red[r_] + red[HP + r_] + red[2 * HP + r_] + red[3 * HP + r_];
    ls = ls > FLT_MAX ? FLT_MAX : ls;
    const float inv = ls == 0.f ? 0.f : pow2(E - kWeightLog2) / ls;
    int64_t at = (int64_t)slot * (p.q_cap * p.group) + r_;
    if (whole) {
      at = (int64_t)(q0 + r_ / p.group) * p.hq + kvh * p.group + r_ % p.group;
    } else if (wg == 0 && lane < R && r_ < rows && alive) {
      float Mr = -INFINITY;
#pragma unroll
      for (int r = 0; r < R; ++r) Mr = r == lane ? M[r] : Mr;
      p.ws_lse[at] = ls == 0.f ? -INFINITY : Mr - (float)E + log2f(ls);
    }
    // four rows a step, their chains side by side; not unrolled, as this runs once a
    // part and mostly from a cold instruction cache
#pragma unroll 1
    for (int c = 0; c < R && r0 + c < rows; c += 4) {
      float o[kPPieces][4], val[4];
      int64_t to[4];
#pragma unroll
      for (int pc = 0; pc < kPPieces; ++pc) tmem_ldn<4>(lane_addr + 2 * kCols + pc * HP + r0 + c, o[pc]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        val[i] = __shfl_sync(0xffffffffu, inv, c + i);
        to[i] = __shfl_sync(0xffffffffu, at, c + i) * kBD + key;
      }
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        val[i] = val[i] == 0.f ? 0.f : (o[0][i] + o[1][i] * kPiece1 + o[2][i] * kPiece2 +
                                        o[3][i] * kPiece3) * val[i];
      const int n = alive ? rows - r0 - c : 0;
      if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) static_cast<T*>(p.out)[to[i]] = DT<T>::from_f(saturate<T>(val[i]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) p.ws_o[to[i]] = saturate<float>(val[i]);
      }
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) {
    __syncwarp();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// Joins the parts of a sequence that the shares' cuts go through: block (cta, row)
// starts from the CTA whose share holds the sequence's first part, follows the
// next shares' first parts up to the last one, and weighs them by 2^(lse - max).
// Lane i looks at the i-th part after the first; 32 parts a step.
template <typename T>
__global__ void __launch_bounds__(kBD) combine_fp8b_kernel(const Params p) {
  pdl_wait();
  const int cta = blockIdx.x, r = blockIdx.y, kvh = cta % p.hkv, lane = threadIdx.x & 31;
  const int ctas = p.groups * p.hkv, cap = p.q_cap * p.group;
  const int b = p.ws_desc[2 * cta + 1].x;
  if (b < 0) return;
  const uint32_t q0 = p.cu_q[b];
  if (r >= (int)(p.cu_q[b + 1] - q0) * p.group) return;
  float mx = p.ws_lse[(int64_t)(2 * cta + 1) * cap + r], wsum = mx == -INFINITY ? 0.f : 1.f;
  float acc = wsum * p.ws_o[((int64_t)(2 * cta + 1) * cap + r) * kBD + threadIdx.x];
  for (int first = cta + p.hkv;; first += 32 * p.hkv) {
    const int c = first + lane * p.hkv;
    const int2 d = c < ctas ? p.ws_desc[2 * c] : make_int2(-1, 0);
    const uint32_t mine = __ballot_sync(0xffffffffu, d.x == b);
    const uint32_t last = __ballot_sync(0xffffffffu, d.x == b && d.y);
    // parts of this step: up to the last one, or as far as they go without a gap
    const int n = last ? __ffs(last) : min(32, __ffs(~mine) - 1 < 0 ? 32 : __ffs(~mine) - 1);
    const float lse = lane < n ? p.ws_lse[(int64_t)(2 * c) * cap + r] : -INFINITY;
    float m = lse;
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) m = warp_max_xor(m, x);
    m = fmaxf(m, mx);
    const float mu = m == -INFINITY ? 0.f : m;
    const float old = exp2f(mx - mu), w = exp2f(lse - mu);
    mx = m;
    wsum *= old;
    acc *= old;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      wsum += wi;
      acc += wi * p.ws_o[((int64_t)(2 * (first + i * p.hkv)) * cap + r) * kBD + threadIdx.x];
    }
    if (last || n < 32) break;
  }
  const int64_t at = (int64_t)(q0 + r / p.group) * p.hq + kvh * p.group + r % p.group;
  static_cast<T*>(p.out)[at * kBD + threadIdx.x] =
      DT<T>::from_f(saturate<T>(wsum == 0.f ? 0.f : acc / wsum));
}

int padded_rows(int rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

// Shares of the batch: one resident wave of CTAs, a share being Hkv of them.
int shares(int hkv, int rows) {
  return std::max(1, 148 * (padded_rows(rows) <= 8 ? 2 : 1) / hkv);
}
// Workspace: descriptors, log-sum-exps and partial rows of every CTA's two slots.
struct Partials {
  size_t lse, o, total;
};
Partials partials(int hq, int hkv, int q_cap) {
  const size_t slots = 2 * (size_t)shares(hkv, q_cap * (hq / hkv)) * hkv;
  const size_t rows = slots * q_cap * (hq / hkv);
  Partials w;
  w.lse = (slots * sizeof(int2) + 15) & ~size_t(15);
  w.o = (w.lse + rows * sizeof(float) + 15) & ~size_t(15);
  w.total = w.o + rows * kBD * sizeof(float);
  return w;
}

template <typename T, int HP>
int launch(const AttnArgs& a, const Params& p, const CUtensorMap& mk, const CUtensorMap& mv) {
  auto kern = decode_fp8b_kernel<T, HP>;
  static unsigned long long done = 0;
  int rc = ensure_smem_attr((const void*)kern, Cfg<HP>::kSmem, &done);
  if (!rc)
    rc = launch_pdl(kern, dim3(p.groups * a.hkv), dim3(Cfg<HP>::kThreads), Cfg<HP>::kSmem, a.stream,
                    "decode fp8b launch", mk, mv, p);
  if (!rc)
    rc = launch_pdl(combine_fp8b_kernel<T>, dim3(p.groups * a.hkv, p.q_cap * p.group), dim3(kBD), 0,
                    a.stream, "combine fp8b launch", p);
  return rc;
}
template <typename T>
int launch_rows(int rows, const AttnArgs& a, const Params& p, const CUtensorMap& mk,
                const CUtensorMap& mv) {
  switch (padded_rows(rows)) {
    case 4: return launch<T, 4>(a, p, mk, mv);
    case 8: return launch<T, 8>(a, p, mk, mv);
    case 16: return launch<T, 16>(a, p, mk, mv);
    default: return launch<T, 32>(a, p, mk, mv);
  }
}

}  // namespace

size_t decode_fp8b_bytes(int hq, int hkv, int q_cap) { return partials(hq, hkv, q_cap).total; }

int launch_decode_fp8b(const AttnArgs& a, int q_cap, bool all) {
  CUtensorMap mk, mv;
  int rc = encode_kv_tensor_map_u8(&mk, a.k_cache, kBD, a.hkv, a.num_blocks * a.page, a.kv_stride,
                                   kBTile);
  if (!rc)
    rc = encode_kv_tensor_map_u8(&mv, a.v_cache, kBD, a.hkv, a.num_blocks * a.page, a.kv_stride,
                                 kBTile);
  if (rc) return rc;
  Params p;
  p.q = a.q;
  p.q_stride = a.q_stride;
  p.out = a.out;
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.block_tables = a.block_tables;
  p.bt_stride = a.bt_stride;
  p.num_blocks = a.num_blocks;
  p.num_q_rows = a.num_q_rows;
  p.scale = a.k_scale;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  p.page = a.page;
  p.max_k = a.max_k;
  p.q_cap = q_cap;
  p.all = all ? 1 : 0;
  p.causal = a.causal;
  p.scale_log2 = a.scale * kLog2e_;
  p.err = device_error_word();
  p.num_seqs = a.num_seqs;
  p.groups = shares(a.hkv, q_cap * p.group);
  const Partials w = partials(a.hq, a.hkv, q_cap);
  uint8_t* ws = static_cast<uint8_t*>(a.ws);
  p.ws_desc = reinterpret_cast<int2*>(ws);
  p.ws_lse = reinterpret_cast<float*>(ws + w.lse);
  p.ws_o = reinterpret_cast<float*>(ws + w.o);
  return a.dtype == NVKV_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(q_cap * p.group, a, p, mk, mv)
                                    : launch_rows<__half>(q_cap * p.group, a, p, mk, mv);
}

}  // namespace nvkv
