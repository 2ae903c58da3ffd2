// Decode attention over the block-scaled e4m3 pool, on tcgen05 (sequences of a
// few query tokens: rows = q_len x (Hq / Hkv) <= 32).
//
// Work item = (split, kv head, sequence): a CTA streams one chunk of one
// sequence's keys for one kv head, 128 keys a tile, and serves all its rows, so
// every code leaves HBM once.  Both products run on the tensor cores with the
// codes exactly as TMA put them into shared memory -- nothing is converted:
//   S^T [128 keys x rows] = K codes (A, K-major) . Q^T (B)
//   O^T [128 dims x rows] += V codes^T (A, MN-major) . P^T (B)
// Q and the weights P enter as THREE e4m3 pieces each, x = c0 + 2^-5 c1 +
// 2^-10 c2, every piece the e4m3 rounding of what the ones before left over
// (c0's error is at most 8 of a value below 256, so 32 times it fits again);
// together they hold 12 significant bits.  The pieces are extra columns of B
// (the tensor core's N has room: 3 x rows), and are joined in f32 with their
// weights where the columns are read.
//
// A compute thread owns one key of the tile (one TMEM lane): it joins its
// scores, multiplies by the key block's K scale, and forms z = S + log2(V
// scale), so a weight 2^(z - M) already carries the value's scale and O needs
// none; the row sum takes the scale back out (an exact power of two).  M is the
// running maximum of z per row over the CTA's keys: warp maxima by redux.sync,
// joined over the four warps through shared memory with one named barrier a
// tile.  When M grows the threads rescale O in TMEM.  Weights leave as one or
// more 16-byte stores a thread (N-major B operand).
//
//   warps 0-3  compute (TMEM lanes 32 w .. 32 w + 31)
//   warp 4     TMA producer: K and V code tiles (SWIZZLE_128B) and the tile's
//              64 bytes of scales, an mbarrier ring
//   warp 5     TMEM allocation and every tcgen05.mma, one thread, in the order
//              S(0), S(1), O(0), S(2), O(1), ...: a tile's scores are computed
//              while the tile before it is in the softmax
//
// Bound by HBM: 2 x 128 bytes of codes + 0.5 of scales a key and kv head; per
// tile the compute warps issue ~700 instructions for 32 KB.
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
constexpr int kBThreads = 192;
constexpr float kLog2e_ = 1.4426950408889634f;
constexpr float kPiece1 = 1.f / 32.f, kPiece2 = 1.f / 1024.f;  // weights of pieces 1 and 2

// Rows a CTA serves, padded: 4, 8, 16 or 32; its resources by that.
template <int HP>
struct Cfg {
  static constexpr int kCols = (3 * HP + 15) / 16 * 16;       // pieces as B columns
  static constexpr int kCtasPerSm = HP <= 8 ? 2 : 1;
  static constexpr int kStages = HP <= 8 ? 3 : HP == 16 ? 6 : 5;
  static constexpr int kQBytes = kCols * 128;
  static constexpr int kPBytes = kCols * 128;                 // one of two buffers
  static constexpr int kTmem = 3 * kCols <= 64 ? 64 : 3 * kCols <= 128 ? 128
                               : 3 * kCols <= 256 ? 256 : 512;
  static constexpr int kOffQ = kStages * kBStage;
  static constexpr int kOffP = kOffQ + kQBytes;
  static constexpr int kOffScale = kOffP + 2 * kPBytes;
  static constexpr int kOffRed = kOffScale + kStages * kBScale * 4;  // [2][4][HP] maxima
  static constexpr int kOffRow = kOffRed + 2 * 4 * HP * 4;           // [HP] factor, [HP] limit
  static constexpr int kOffBar = kOffRow + 2 * HP * 4;
  static constexpr int kBars = 2 * kStages + 8;
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
  int hq, hkv, group, page, chunk, max_k, max_splits, q_cap, all, causal;
  float scale_log2;
  float *ws_o, *ws_lse;  // [B][splits][hkv][q_cap * group] (x 128)
  int* err;
};

__device__ __forceinline__ uint64_t sdesc_plain(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// kind::f8f6f4, e4m3 x e4m3, f32 accumulate, M = 128
__host__ __device__ constexpr uint32_t idesc_f8(int n, uint32_t a_mn, uint32_t b_mn) {
  return (1u << 4) | (a_mn << 15) | (b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// n (4, 8, 16) consecutive f32 columns of this thread's TMEM lane
template <int n>
__device__ __forceinline__ void tmem_ldn(uint32_t a, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  if constexpr (n == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
  else if constexpr (n == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(a));
  else
    tmem_ld16(a, v);
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
// Four values (0 <= |x| <= 256) as three pieces: w[p] = the codes of piece p.
__device__ __forceinline__ void pieces4(float a, float b, float c, float d, uint32_t (&w)[3]) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const uint32_t lo = e4m3x2(a, b), hi = e4m3x2(c, d);
    w[p] = lo | (hi << 16);
    if (p < 2) {
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
// scale).  Missing rows are zero.
template <typename T, int HP>
__device__ __forceinline__ void load_q(const Params& p, uint32_t q0, int kvh, int rows,
                                       uint8_t* sq, float* rowf, int warp, int lane) {
  constexpr int kCols = Cfg<HP>::kCols;
  for (int i = threadIdx.x; i < kCols * 8; i += 128)
    *reinterpret_cast<uint4*>(sq + i * 16) = make_uint4(0, 0, 0, 0);
  bar_compute();
  for (int r = warp; r < HP; r += 4) {
    if (r >= rows) {
      if (lane == 0) rowf[r] = 0.f;
      continue;
    }
    const T* src = static_cast<const T*>(p.q) + (int64_t)(q0 + r / p.group) * p.q_stride +
                   (int64_t)(kvh * p.group + r % p.group) * kBD + 4 * lane;
    const uint2 raw = *reinterpret_cast<const uint2*>(src);
    const float2 u = DT<T>::to_f2(raw.x), v = DT<T>::to_f2(raw.y);
    float x[4] = {u.x, u.y, v.x, v.y};
    float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    m = redux_max(m);
    const int e = (int)(__float_as_uint(m) >> 23);
    const int sh = m > 0.f ? min(127, 134 - e) : 0;  // m 2^sh in [128, 256)
    const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // an infinite query gives NaN, as its scores would
      x[i] = fabsf(x[i]) < INFINITY ? x[i] * up : __int_as_float(0x7fffffff);
    uint32_t w[3];
    pieces4(x[0], x[1], x[2], x[3], w);
#pragma unroll
    for (int pc = 0; pc < 3; ++pc) {
      const int n = pc * HP + r;
      *reinterpret_cast<uint32_t*>(sq + n * 128 + (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4) =
          w[pc];
    }
    if (lane == 0) rowf[r] = __uint_as_float((uint32_t)(127 - sh) << 23) * p.scale_log2;
  }
}

template <typename T, int HP>
__global__ void __launch_bounds__(kBThreads, Cfg<HP>::kCtasPerSm)
    decode_fp8b_kernel(const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const Params p) {
  using C = Cfg<HP>;
  constexpr int kStages = C::kStages, kCols = C::kCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem + C::kOffQ;
  uint8_t* sp = smem + C::kOffP;
  float* ssc = reinterpret_cast<float*>(smem + C::kOffScale);
  float* red = reinterpret_cast<float*>(smem + C::kOffRed);
  float* rowf = reinterpret_cast<float*>(smem + C::kOffRow);
  int* rowlim = reinterpret_cast<int*>(rowf + HP);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + kStages;
  uint64_t* s_full = empty + kStages;  // [2] scores of a tile are in TMEM
  uint64_t* p_full = s_full + 2;       // [2] scores read, weights in shared memory, O rescaled
  uint64_t* o_done = p_full + 2;       // [2] the tile's O product has finished
  uint64_t* q_full = o_done + 2;
  uint64_t* drain = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 128) {
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
      mbar_init(&p_full[x], 128);
      mbar_init(&o_done[x], 1);
    }
    mbar_init(q_full, 128);
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  pdl_wait();  // inputs may come from the kernel before this one

  // the chunk's first 32 block-table entries, beside the lengths (in the row:
  // split * chunk < the plan's bound <= page * bt_stride)
  const int pg_first = (int)((int64_t)split * p.chunk / p.page);
  uint32_t ent = 0;
  if (warp == 4 && pg_first + lane < p.bt_stride)
    ent = __ldg(p.block_tables + (int64_t)b * p.bt_stride + pg_first + lane);
  const uint32_t q0 = p.cu_q[b];
  const int q_len = (int)(p.cu_q[b + 1] - q0);
  const int k_len = (int)(p.cu_k[b + 1] - p.cu_k[b]);
  if (q_len == 0) return;
  const bool other = q_len < 0 || q_len > p.q_cap;
  if (other && !p.all) return;  // the prefill kernel's
  const int nsplit = k_len > 0 ? (k_len + p.chunk - 1) / p.chunk : 1;
  if (other || k_len > p.max_k || (int64_t)q0 + q_len > p.num_q_rows ||
      (q_len > 1 && k_len < q_len)) {
    if (threadIdx.x == 0) record_error(p.err, NVKV_DEVERR_SEQLEN);
    return;
  }
  if (split >= nsplit) return;
  if (k_len <= 0 && threadIdx.x == 0) record_error(p.err, NVKV_DEVERR_SEQLEN);
  const int tok0 = split * p.chunk;
  const int tok1 = min(k_len, tok0 + p.chunk);
  const int ntiles = tok1 > tok0 ? (tok1 - tok0 + kBTile - 1) / kBTile : 0;
  const int rows = q_len * p.group;
  if (warp == 5) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // only now, with this CTA's tensor memory in hand, may the next grid start
  pdl_launch_dependents();

  if (warp == 4) {
    // ------------------------------ TMA producer ------------------------------
    int base = 0;  // chunk page of lane 0's entry
    int it = 0, go = 1;
    for (; it < ntiles; ++it) {
      const int s = it % kStages;
      const int j0 = tok0 + it * kBTile;
      const int pi = j0 / p.page - pg_first;
      if (pi >= base + 32) {  // warp-uniform: the next 32 entries
        base += 32;
        const int pg = pg_first + base + lane;
        ent = pg < p.bt_stride ? __ldg(p.block_tables + (int64_t)b * p.bt_stride + pg) : 0u;
      }
      uint32_t page = __shfl_sync(0xffffffffu, ent, pi - base);
      if ((int64_t)page >= p.num_blocks) {  // recorded; read as page 0 so that the rest finishes
        if (lane == 0) record_error(p.err, NVKV_DEVERR_BLOCK_RANGE);
        page = 0;
      }
      if (lane == 0) {
        go = it < kStages || mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, p.err);
        if (go) {
          const int off = j0 % p.page;
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
    if (!go && lane == 0)  // given up: wait for the copies in flight
      for (int i = max(0, it - kStages); i < it; ++i)
        mbar_wait(&full[i % kStages], (i / kStages) & 1, p.err);
  } else if (warp == 5) {
    // ------------------------------- MMA issuer -------------------------------
    if (lane == 0 && ntiles > 0) {
      constexpr uint32_t id_s = idesc_f8(kCols, 0, 0), id_o = idesc_f8(kCols, 1, 1);
      const uint32_t tiles = smem_u32(smem), aq = smem_u32(sq), ap = smem_u32(sp);
      bool ok = mbar_wait(q_full, 0, p.err);
      int it = 0;
      for (; ok && it <= ntiles; ++it) {
        if (it < ntiles) {  // S(it): K-major codes, 32 dims a step
          ok = mbar_wait(&full[it % kStages], (it / kStages) & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ak = tiles + (it % kStages) * kBStage;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8(tmem + (it & 1) * kCols, sdesc(ak + kk * 32, 16, 1024),
                   sdesc(aq + kk * 32, 16, 1024), id_s, kk > 0);
          tc_commit(&s_full[it & 1]);
        }
        if (it > 0) {  // O += V^T . P of the tile before: 32 keys a step
          const int o = it - 1;
          ok = mbar_wait(&p_full[o & 1], (o >> 1) & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t av = tiles + (o % kStages) * kBStage + kBCode;
          const uint32_t pb = ap + (o & 1) * C::kPBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8(tmem + 2 * kCols, sdesc(av + kk * 32 * 128, 16, 1024),
                   sdesc_plain(pb + kk * 512, 128, 2048), id_o, o > 0 || kk > 0);
          tc_commit(&o_done[o & 1]);
          tc_commit(&empty[o % kStages]);
        }
      }
      if (!ok) {  // given up: let the products in flight finish before the memory goes
        tc_commit(drain);
        mbar_wait(drain, 0, nullptr);
      }
    }
  } else {
    // ------------------------------ compute warps ------------------------------
    const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
    const int key = threadIdx.x;  // this thread's key of a tile, and its dim of O
    if (threadIdx.x < HP) {
      const int r = threadIdx.x;
      rowlim[r] = r >= rows ? -1 : p.causal ? k_len - q_len + r / p.group : k_len - 1;
    }
    load_q<T, HP>(p, q0, kvh, rows, sq, rowf, warp, lane);
    fence_async_smem();
    mbar_arrive(q_full);
    bar_compute();  // rowf, rowlim
    float M[HP], l[HP];
#pragma unroll
    for (int r = 0; r < HP; ++r) M[r] = -INFINITY, l[r] = 0.f;
    bool alive = true;
    for (int it = 0; it < ntiles; ++it) {
      const int s = it % kStages, x = it & 1;
      // a wait that runs out is not repeated, but the warp stays in step with the
      // others' barriers to the end of the loop
      alive = alive && __all_sync(0xffffffffu, mbar_wait(&full[s], (it / kStages) & 1, p.err) &&
                                                   mbar_wait(&s_full[x], (it >> 1) & 1, p.err));
      tc_fence_after();
      const float2 sc = *reinterpret_cast<const float2*>(ssc + s * kBScale +
                                                         key / NVKV_FP8B_BLOCK * 2);
      const float ks = sc.x;
      // log2 of the V scale, a power of two (a cleared pool's 0 counts as the least;
      // the upper bound keeps a stale block's NaN out of the masked sums)
      const int ev = min(max((int)(__float_as_uint(sc.y) >> 23 & 0xffu) - 127, -100), 120);
      const int j = tok0 + it * kBTile + key;
      float z[HP];
      const uint32_t cs = lane_addr + x * kCols;
      if constexpr (HP == 4) {
        float a[16];
        tmem_ld16(cs, a);
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < 4; ++r)
          z[r] = a[r] + a[4 + r] * kPiece1 + a[8 + r] * kPiece2;
      } else {
#pragma unroll
        for (int c = 0; c < HP; c += 8) {
          float a0[8], a1[8], a2[8];
          tmem_ldn<8>(cs + c, a0);
          tmem_ldn<8>(cs + HP + c, a1);
          tmem_ldn<8>(cs + 2 * HP + c, a2);
          tmem_wait_ld();
#pragma unroll
          for (int r = 0; r < 8; ++r)
            z[c + r] = a0[r] + a1[r] * kPiece1 + a2[r] * kPiece2;
        }
      }
      float mine = -INFINITY;  // lane r: the warp's maximum of row r
#pragma unroll
      for (int r = 0; r < HP; ++r) {
        z[r] = j <= rowlim[r] ? z[r] * (rowf[r] * ks) + (float)ev : -INFINITY;
        const float m = redux_max(z[r]);
        if (lane == r) mine = m;
      }
      float* rd = red + x * 4 * HP;
      if (lane < HP) rd[warp * HP + lane] = mine;
      bar_compute();
      float fac[HP];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < HP; ++r) {
        const float m = fmaxf(fmaxf(rd[r], rd[HP + r]), fmaxf(rd[2 * HP + r], rd[3 * HP + r]));
        fac[r] = 1.f;
        if (m > M[r]) {
          fac[r] = ex2_mufu(M[r] - m);
          M[r] = m;
          grew = true;
        }
      }
      if (grew) {
#pragma unroll
        for (int r = 0; r < HP; ++r) l[r] *= fac[r];
        if (it > 0) {  // O is in units of 2^M
          alive = alive && __all_sync(0xffffffffu,
                                      mbar_wait(&o_done[x ^ 1], ((it - 1) >> 1) & 1, p.err));
          tc_fence_after();
          constexpr int n = HP == 4 ? 4 : 8;
#pragma unroll
          for (int pc = 0; pc < 3; ++pc)
#pragma unroll
            for (int c = 0; c < HP; c += n) {
              const uint32_t a = lane_addr + 2 * kCols + pc * HP + c;
              float o[n];
              tmem_ldn<n>(a, o);
              tmem_wait_ld();
#pragma unroll
              for (int r = 0; r < n; ++r) o[r] *= fac[c + r];
              const uint32_t* w = reinterpret_cast<const uint32_t*>(o);
              if constexpr (n == 4)
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
      // weights, times 256 for the pieces; the row sums without the V scale
      const float unscale = __uint_as_float((uint32_t)(127 - ev) << 23);
      uint32_t w[kCols / 4];
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) w[i] = 0u;
#pragma unroll
      for (int c = 0; c < HP; c += 4) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float m = M[c + r] == -INFINITY ? 0.f : M[c + r];
          e[r] = ex2_mufu(z[c + r] - m);
          l[c + r] += e[r] * unscale;
          e[r] *= 256.f;
        }
        uint32_t pw[3];
        pieces4(e[0], e[1], e[2], e[3], pw);
#pragma unroll
        for (int pc = 0; pc < 3; ++pc) w[(pc * HP + c) / 4] = pw[pc];
      }
      if (it >= 2)  // this buffer's last reader
        alive = alive &&
                __all_sync(0xffffffffu, mbar_wait(&o_done[x], ((it - 2) >> 1) & 1, p.err));
      uint8_t* dst = sp + x * C::kPBytes + key * 16;
#pragma unroll
      for (int nb = 0; nb < kCols / 16; ++nb)
        *reinterpret_cast<uint4*>(dst + nb * 2048) =
            make_uint4(w[4 * nb], w[4 * nb + 1], w[4 * nb + 2], w[4 * nb + 3]);
      if (j >= tok1) {  // a key past the end: its V row may hold NaN codes, and 0 x NaN is NaN
        uint8_t* vr = smem + s * kBStage + kBCode + key * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vr + c * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_async_smem();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }

    // ------------------------------- epilogue -------------------------------
    if (alive && ntiles > 0)
      alive = __all_sync(0xffffffffu, mbar_wait(&o_done[(ntiles - 1) & 1],
                                                ((ntiles - 1) >> 1) & 1, p.err));
    tc_fence_after();
    bar_compute();  // the last tile's maxima have been read
#pragma unroll
    for (int r = 0; r < HP; ++r) {
      float v = l[r];
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
      if (lane == 0) red[warp * HP + r] = v;
    }
    bar_compute();
    constexpr int n = HP == 4 ? 4 : 8;
    for (int c = 0; c < HP; c += n) {
      float o[3][n];
#pragma unroll
      for (int pc = 0; pc < 3; ++pc) tmem_ldn<n>(lane_addr + 2 * kCols + pc * HP + c, o[pc]);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int r = c + i;
        if (r >= rows || !alive) continue;
        const float ls = red[r] + red[HP + r] + red[2 * HP + r] + red[3 * HP + r];
        const float acc = (o[0][i] + o[1][i] * kPiece1 + o[2][i] * kPiece2) *
                          (1.f / 256.f);
        const float val = ls == 0.f ? 0.f : acc / ls;
        if (nsplit == 1) {
          const int64_t at = (int64_t)(q0 + r / p.group) * p.hq + kvh * p.group + r % p.group;
          static_cast<T*>(p.out)[at * kBD + key] = DT<T>::from_f(val);
        } else {
          const int64_t at =
              (((int64_t)b * p.max_splits + split) * p.hkv + kvh) * (p.q_cap * p.group) + r;
          p.ws_o[at * kBD + key] = val;
          float Mr = -INFINITY;
#pragma unroll
          for (int k = 0; k < HP; ++k) Mr = k == r ? M[k] : Mr;
          if (key == 0) p.ws_lse[at] = ls == 0.f ? -INFINITY : Mr + log2f(ls);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) {
    __syncwarp();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// Joins the splits of one (sequence, row): weights 2^(lse - max lse).
template <typename T>
__global__ void __launch_bounds__(kBD) combine_fp8b_kernel(const Params p) {
  pdl_wait();
  const int cap = p.q_cap * p.group;
  const int kvh = blockIdx.x / cap, r = blockIdx.x % cap, b = blockIdx.y;
  const uint32_t q0 = p.cu_q[b];
  const int q_len = (int)(p.cu_q[b + 1] - q0);
  const int k_len = (int)(p.cu_k[b + 1] - p.cu_k[b]);
  const int nsplit = k_len > 0 ? (k_len + p.chunk - 1) / p.chunk : 1;
  // the decode grid wrote no partials for these
  if (nsplit <= 1 || q_len <= 0 || q_len > p.q_cap || r >= q_len * p.group || k_len > p.max_k ||
      (int64_t)q0 + q_len > p.num_q_rows || (q_len > 1 && k_len < q_len))
    return;
  const int64_t step = (int64_t)p.hkv * cap;
  const int64_t base = (int64_t)b * p.max_splits * step + (int64_t)kvh * cap + r;
  float mx = -INFINITY;
  for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, p.ws_lse[base + s * step]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float wsum = 0.f, acc = 0.f;
#pragma unroll 4
  for (int s = 0; s < nsplit; ++s) {
    const float w = exp2f(p.ws_lse[base + s * step] - mu);
    wsum += w;
    acc += w * p.ws_o[(base + s * step) * kBD + threadIdx.x];
  }
  const int64_t at = (int64_t)(q0 + r / p.group) * p.hq + kvh * p.group + r % p.group;
  static_cast<T*>(p.out)[at * kBD + threadIdx.x] = DT<T>::from_f(wsum == 0.f ? 0.f : acc / wsum);
}

int padded_rows(int rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

// Split plan: as many CTAs as ~3 resident waves, chunks of at least 6 tiles;
// nothing is split when one CTA per (sequence, kv head) fills most of a wave and
// no sequence is long.
void plan(int num_seqs, int hkv, int max_k, int rows, int* chunk, int* max_splits) {
  const int per_sm = padded_rows(rows) <= 8 ? 2 : 1;
  const int tiles = max_k > 0 ? (max_k + kBTile - 1) / kBTile : 1;
  const int64_t items = (int64_t)num_seqs * hkv, wave = 148 * per_sm;
  int splits = (int)((3 * wave + items - 1) / items);
  splits = std::min(splits, (tiles + 5) / 6);
  if (items * 5 >= wave * 4 && tiles <= 24) splits = 1;
  splits = std::max(splits, 1);
  const int per = (tiles + splits - 1) / splits;
  *chunk = per * kBTile;
  *max_splits = (tiles + per - 1) / per;
}

template <typename T, int HP>
int launch(const AttnArgs& a, const Params& p, const CUtensorMap& mk, const CUtensorMap& mv) {
  auto kern = decode_fp8b_kernel<T, HP>;
  static unsigned long long done = 0;
  int rc = ensure_smem_attr((const void*)kern, Cfg<HP>::kSmem, &done);
  if (!rc)
    rc = launch_pdl(kern, dim3(p.max_splits, a.hkv, a.num_seqs), dim3(kBThreads), Cfg<HP>::kSmem,
                    a.stream, "decode fp8b launch", mk, mv, p);
  if (!rc && p.max_splits > 1)
    rc = launch_pdl(combine_fp8b_kernel<T>, dim3(a.hkv * p.q_cap * p.group, a.num_seqs),
                    dim3(kBD), 0, a.stream, "combine fp8b launch", p);
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

size_t decode_fp8b_bytes(int num_seqs, int hq, int hkv, int max_k, int q_cap) {
  int chunk, splits;
  plan(num_seqs, hkv, max_k, q_cap * (hq / hkv), &chunk, &splits);
  if (splits <= 1) return 0;
  const size_t n = (size_t)num_seqs * splits * hq * q_cap;
  return n * (kBD + 1) * sizeof(float);
}

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
  plan(a.num_seqs, a.hkv, a.max_k, q_cap * p.group, &p.chunk, &p.max_splits);
  p.ws_o = static_cast<float*>(a.ws);
  p.ws_lse = p.ws_o + (size_t)a.num_seqs * p.max_splits * a.hq * q_cap * kBD;
  return a.dtype == NVKV_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(q_cap * p.group, a, p, mk, mv)
                                    : launch_rows<__half>(q_cap * p.group, a, p, mk, mv);
}

}  // namespace nvkv
