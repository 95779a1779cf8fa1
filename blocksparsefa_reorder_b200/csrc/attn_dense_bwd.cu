// Gradient of cross attention (attn_dense.cu) for sm_100a: bf16 / fp16, head
// dim 64 or 128, key / value heads shared by groups of query heads, padded keys.
//
//   P = 2^(s scale_log2 - lse),  dP = dO V^T,  dS = P o (dP - Delta)
//   dQ = sm_scale dS K,  dK = sm_scale sum_g dS^T Q,  dV = sum_g P^T dO
// with Delta = rowsum(dO o O) and the sums over the query heads g of a key /
// value head.  No atomics: every gradient row is written by one CTA.
// fp16: dS of a long row is about dO / keys, below what fp16 resolves (2^-24)
// already for dO of 2^-8.  So it is held times the power of two that brings the
// largest |dO| of the rows summed up, found by the Delta kernel, into [4, 8) (dO of
// N(0, 1): 1), which dQ and dK take off again in fp32.  (2 x 16 heads x 2048 x
// 4096 x 128 in fp16 387 us, 386 without; 3 x 6 heads x 777 x 1531 x 64 40, 39 without.
// One maximum a group by atomics, behind a memset: 394 and 50.)  The same for P on
// its way to dV: at most 1 but for rounding, it is held times 2^12, so that a key
// of little weight in every row keeps its sum (an exponent's offset; no cost).
//
// Bound by the tensor cores: dQ needs three products of a 128 x 128 tile (S,
// dP, dS K), dK / dV four.  Both kinds of CTA keep them fed by the order in
// which the MMA warp issues:
//  * dQ: S two tiles ahead in two buffers; once dS_j is written, dP_j+1, then
//    dQ += dS_j K_j, then S_j+2.  The exponentials of tile j+1 run under dP_j+1;
//  * dK / dV: P_i^T ready -> dV += P_i^T dO_i, S_i+1^T (over P_i); dS_i^T ready
//    -> dK += dS_i^T Q_i, dP_i+1^T (over dS_i).  The exponentials of step i+1
//    run under the last two.
// Roles of a CTA: warp 0 TMA producer (one thread), warp 1 MMA issue (the whole
// warp, one elected lane: see attn_dense.cu), warpgroups 1 and 2 elementwise: a row is shared by two threads, one of each warpgroup, with 64
// of the tile's 128 columns, so that each 16-bit result lies over columns its
// own thread has read (columns 0-31 and 64-95 of the score buffer).
// Measured: 2 x 16 heads x 2048 x 4096 x 128 375 us (917 TF/s of the five
// products, seven being computed); 24 tokens of 4 heads over 4000 states 71 us.
// Every wait is bounded; a timeout sets BSA_DEVERR_TIMEOUT and all roles drain.
#include <cudaTypedefs.h>

#include "common.cuh"
#include "dense.h"
#include "internal.h"
#include "softmax.cuh"

namespace bsa {

namespace {

constexpr int kThreadsB = 384;

struct DBwdParams {
  int B, H, Hk, G, M, N;
  // A query tile holds mt tokens of gh heads of a group (a divisor of G), the
  // tokens fastest: nm along the tokens, q_tiles in all for a key / value head.
  int mt, gh, nm, q_tiles, k_tiles;
  int qb_mul, kb_mul, vb_mul, db_mul;  // 0: the tensor's batch stride is 0
  const void* lens;
  int lens_i64;
  float scale_log2, sm_scale;
  const float* lse;    // [B, H, M]
  const float* delta;  // [B, H, M]
  // largest |dout| of every max_rows rows of a head group, [B, Hk, maxima], or null: dS as it is
  const float* dout_max;
  int max_rows, maxima;
  uint8_t *dq, *dk, *dv;
  int64_t dq_b, dq_h, dq_n, dk_b, dk_h, dk_n, dv_b, dv_h, dv_n;
  int32_t* err;
  uint64_t wait_ns;
};

template <int D>
struct DBwdCfg {
  static constexpr int NCHUNK = D / 64;
  static constexpr int CHUNK = 128 * 128;
  static constexpr int TILE = 128 * D * 2;
  // Stages of the two streamed tensors: the first (K, resp. Q) is held until
  // the step's last product, the second until its first.
  static constexpr int SA = D == 128 ? 3 : 5, SB = D == 128 ? 2 : 5;
  static constexpr int BAR_BYTES = 256;
  static constexpr int STATS = 2 * 2 * 128 * 4;
  static constexpr int SMEM = (2 + SA + SB) * TILE + BAR_BYTES + STATS;
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert((2 * (SA + SB) + 8) * 8 + 8 <= BAR_BYTES, "barriers");
};

__device__ __forceinline__ int bwd_len(const DBwdParams& p, int b) {
  if (!p.lens) return p.N;
  const int64_t l = p.lens_i64 ? __ldg(static_cast<const int64_t*>(p.lens) + b)
                               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.lens) + b));
  if (l < 0 || l > p.N) set_err(p.err, BSA_DEVERR_COORD);
  return static_cast<int>(l < 0 ? 0 : l > p.N ? p.N : l);
}

// Row `rl` of query tile t of a group: its head of the group and token; false
// where the tile has no such row.
__device__ __forceinline__ bool query_of(const DBwdParams& p, int t, int rl, int& g, int& m) {
  const int gi = t / p.nm, q = rl / p.mt;
  m = (t - gi * p.nm) * p.mt + rl - q * p.mt;
  g = gi * p.gh + q;
  return q < p.gh && m < p.M;
}

// What dS is held times (see above) for a largest |dO| of the given bits; 1 where
// it is zero or not finite.
__device__ __forceinline__ float ds_scale(uint32_t bits) {
  if (bits == 0u || bits >= 0x7F800000u) return 1.f;
  return __uint_as_float((2 * 127 + 2 - (bits >> 23)) << 23);  // (an fp16 value is a normal fp32 one)
}

// -lse as the exponent's offset; a row without any weight (lse -inf) and a row
// past the end get P = 0.
__device__ __forceinline__ float neg_lse_of(const DBwdParams& p, bool in, int64_t i) {
  const float l = in ? __ldg(&p.lse[i]) : -INFINITY;
  return l == -INFINITY ? -INFINITY : -l;
}

// Half of an accumulator's columns (this thread's D / 2 of one row) times
// `scale`, as 16-bit values; `row`: the row's place, `keep`: whether it is
// stored, `zero`: as zeros.  8 lanes write 128 bytes of a row at D = 128.
template <int D, bool BF16>
__device__ __forceinline__ void store_half_row(uint32_t base, int half, float scale, uint8_t* row, bool keep, bool zero) {
  const int lane = threadIdx.x & 31;
  uint4 x[8];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t a[32];
    tmem_ld32(base + half * (D / 2) + c * 32, a);
    tmem_wait_ld32(a);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint4& v = x[c * 4 + g];
      v.x = pack2<BF16>(__uint_as_float(a[8 * g + 0]) * scale, __uint_as_float(a[8 * g + 1]) * scale);
      v.y = pack2<BF16>(__uint_as_float(a[8 * g + 2]) * scale, __uint_as_float(a[8 * g + 3]) * scale);
      v.z = pack2<BF16>(__uint_as_float(a[8 * g + 4]) * scale, __uint_as_float(a[8 * g + 5]) * scale);
      v.w = pack2<BF16>(__uint_as_float(a[8 * g + 6]) * scale, __uint_as_float(a[8 * g + 7]) * scale);
      if (zero) v = make_uint4(0, 0, 0, 0);
    }
  }
  if constexpr (D == 128) {
    transpose_pieces<8>(x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int from = (lane & 24) + k;
      uint8_t* dst = shfl_ptr(row, from);
      const bool st = __shfl_sync(0xffffffffu, static_cast<int>(keep), from) != 0;
      if (st) *reinterpret_cast<uint4*>(dst + half * D + (lane & 7) * 16) = x[k];
    }
  } else if (keep) {
#pragma unroll
    for (int g = 0; g < 4; ++g) reinterpret_cast<uint4*>(row)[half * 4 + g] = x[g];
  }
}

template <int D>
__device__ __forceinline__ void zero_half_row(int half, uint8_t* row) {
#pragma unroll
  for (int g = 0; g < D / 16; ++g) reinterpret_cast<uint4*>(row)[half * (D / 16) + g] = make_uint4(0, 0, 0, 0);
}

// Two exponentials, on the FMA pipe or on the special function unit: half of
// them each way, as a step's 64 a thread keep the unit busy for 1,024 cycles.
__device__ __forceinline__ void ex2_pair(uint64_t x, bool fma, float& p0, float& p1) {
  if (fma) {
    f32x2_unpack(ex2_fma_x2(x), p0, p1);
  } else {
    float x0, x1;
    f32x2_unpack(x, x0, x1);
    p0 = ex2_approx(x0);
    p1 = ex2_approx(x1);
  }
}

// dP - Delta of two columns, times what dS is held times (Delta has it in it).
template <bool BF16>
__device__ __forceinline__ uint64_t dp_minus(uint32_t dp0, uint32_t dp1, uint64_t held2, uint64_t neg_delta2) {
  const uint64_t dp = f32x2_pack(__uint_as_float(dp0), __uint_as_float(dp1));
  return BF16 ? f32x2_add(dp, neg_delta2) : f32x2_fma(dp, held2, neg_delta2);
}

// C (+)= A B^T of two 128 x D shared-memory tiles (K-major descriptors)
template <int D>
__device__ __forceinline__ void mma_abt(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const int off = (kk >> 2) * (DBwdCfg<D>::CHUNK >> 4) + (kk & 3) * 2;
    tc_mma_ss(d, a + off, b + off, idesc, kk > 0 ? 1u : 0u);
  }
}
// C (+)= A B of a 128 x 128 16-bit A in tensor memory (columns 0-31 and
// 64-95) and a 128 x D shared-memory tile (MN-major descriptor)
template <int D>
__device__ __forceinline__ void mma_ab(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool first) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    tc_mma_ts(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b + kk * (16 * 128 >> 4), idesc, (first && kk == 0) ? 0u : 1u);
}
__device__ __forceinline__ uint64_t k_major(const void* t) { return make_sw128_desc(smem_u32(t), 16, 1024); }
__device__ __forceinline__ uint64_t mn_major(const void* t) { return make_sw128_desc(smem_u32(t), 128 * 128, 1024); }

// ---------------------------------------------------------------------------
// dQ: one CTA per query tile, over the key tiles.
// TMEM: S_j / dS_j [128 (j & 1), +128), dP [256, 384), dQ [384, 384 + D).
// ---------------------------------------------------------------------------
template <int D, bool BF16>
__device__ void dq_tile(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const CUtensorMap& tmDO,
                        const DBwdParams& p, uint8_t* smem, int item) {
  using C = DBwdCfg<D>;
  constexpr int SA = C::SA, SB = C::SB;
  uint8_t* sQ = smem;
  uint8_t* sDO = sQ + C::TILE;
  uint8_t* sK = sDO + C::TILE;      // [SA]
  uint8_t* sV = sK + SA * C::TILE;  // [SB]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + SB * C::TILE);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;          // [SA]
  uint64_t* k_empty = k_full + SA;      // [SA] dQ_j (its last reader) completed
  uint64_t* v_full = k_empty + SA;      // [SB]
  uint64_t* v_empty = v_full + SB;      // [SB] dP_j completed
  uint64_t* s_full = v_empty + SB;      // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = dp_full + 1;        // 8 elementwise warps
  uint64_t* done = ds_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int bh = item / p.q_tiles, t = item - bh * p.q_tiles;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < SA; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < SB; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 8);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  constexpr uint32_t kDP = 256, kDQ = 384;
  const int len = bwd_len(p, b);
  const int n = (len + 127) / 128;
  auto wait = [&](uint64_t* bar, int k) { return mbar_wait(bar, k & 1, abort_flag, p.err, p.wait_ns); };
  auto wait_all = [&](uint64_t* bar, int k) { return __all_sync(0xffffffffu, wait(bar, k)) != 0; };

  if (warp == 0 && lane == 0 && n > 0) {
    // ------------------------------------------------------------- producer
    mbar_arrive_expect_tx(q_full, 2 * C::NCHUNK * p.mt * p.gh * 128);
    const int gi = t / p.nm, m0 = (t - gi * p.nm) * p.mt, h0 = hk * p.G + gi * p.gh;
    for (int c = 0; c < C::NCHUNK; ++c) {
      tma_load_4d(sQ + c * C::CHUNK, &tmQ, q_full, c * 64, m0, h0, b * p.qb_mul);
      tma_load_4d(sDO + c * C::CHUNK, &tmDO, q_full, c * 64, m0, h0, b * p.db_mul);
    }
    int nk = 0, nv = 0;  // loads issued
    for (int j = 0; j < n; ++j) {
      const int a = j % SA, v = j % SB;
      if (j >= SA && !wait(&k_empty[a], j / SA - 1)) break;
      mbar_arrive_expect_tx(&k_full[a], C::TILE);
      for (int c = 0; c < C::NCHUNK; ++c)
        tma_load_4d(sK + a * C::TILE + c * C::CHUNK, &tmK, &k_full[a], c * 64, j * 128, hk, b * p.kb_mul);
      ++nk;
      if (j >= SB && !wait(&v_empty[v], j / SB - 1)) break;
      mbar_arrive_expect_tx(&v_full[v], C::TILE);
      for (int c = 0; c < C::NCHUNK; ++c)
        tma_load_4d(sV + v * C::TILE + c * C::CHUNK, &tmV, &v_full[v], c * 64, j * 128, hk, b * p.vb_mul);
      ++nv;
    }
    mbar_wait(q_full, 0, nullptr, nullptr, p.wait_ns);
    for (int i = nk > SA ? nk - SA : 0; i < nk; ++i) mbar_wait(&k_full[i % SA], (i / SA) & 1, nullptr, nullptr, p.wait_ns);
    for (int i = nv > SB ? nv - SB : 0; i < nv; ++i) mbar_wait(&v_full[i % SB], (i / SB) & 1, nullptr, nullptr, p.wait_ns);
  } else if (warp == 1 && n > 0) {
    // -------------------- MMA issue (whole warp, one elected lane: see attn_dense.cu)
    constexpr uint32_t idesc_s = make_idesc_f16(BF16, 128, 128, false, false);
    constexpr uint32_t idesc_dq = make_idesc_f16(BF16, 128, D, false, true);
    constexpr int TS = C::TILE >> 4;
    const uint64_t qd = k_major(sQ), dod = k_major(sDO), kd = k_major(sK), vd = k_major(sV), kmn = mn_major(sK);
    bool ok = wait_all(q_full, 0);
    auto issue_s = [&](int j) {
      const int st = j % SA;
      if (!(ok = ok && wait_all(&k_full[st], j / SA))) return;
      tc_fence_after();
      if (elect_one()) {
        mma_abt<D>(tmem + (j & 1) * 128, qd, kd + st * TS, idesc_s);
        tc_commit(&s_full[j & 1]);
      }
      __syncwarp();
    };
    auto issue_dp = [&](int j) {
      const int st = j % SB;
      if (!(ok = ok && wait_all(&v_full[st], j / SB))) return;
      tc_fence_after();
      if (elect_one()) {
        mma_abt<D>(tmem + kDP, dod, vd + st * TS, idesc_s);
        tc_commit(dp_full);
        tc_commit(&v_empty[st]);
      }
      __syncwarp();
    };
    if (ok) issue_s(0);
    if (ok) issue_dp(0);
    if (ok && n > 1) issue_s(1);
    for (int j = 0; ok && j < n; ++j) {
      if (!(ok = wait_all(ds_ready, j))) break;
      tc_fence_after();
      // dP's buffer is free (dS_j is written): step j+1 can go on
      if (j + 1 < n) issue_dp(j + 1);
      if (!ok) break;
      if (elect_one()) {
        mma_ab<D>(tmem + kDQ, tmem + (j & 1) * 128, kmn + (j % SA) * TS, idesc_dq, j == 0);
        tc_commit(&k_empty[j % SA]);
      }
      __syncwarp();
      // over dS_j, which dQ_j (issued before) has read
      if (j + 2 < n) issue_s(j + 2);
    }
    if (elect_one()) {
      tc_commit(done);
      mbar_wait(done, 0, nullptr, nullptr, p.wait_ns);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------- elementwise, epilogue
    const int q4 = warp & 3, half = (warp - 4) >> 2;
    const int row = q4 * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    int g, m;
    const bool live = query_of(p, t, row, g, m);
    const int h = hk * p.G + g;
    uint8_t* orow = p.dq + 2 * (b * p.dq_b + h * p.dq_h + static_cast<int64_t>(m) * p.dq_n);
    if (n == 0) {
      if (live) zero_half_row<D>(half, orow);
    } else {
      const int64_t ri = (static_cast<int64_t>(b) * p.H + h) * p.M + m;
      const float neg_lse = neg_lse_of(p, live, ri);
      const float dlt = live ? __ldg(&p.delta[ri]) : 0.f;
      const uint64_t sc2 = f32x2_pack(p.scale_log2, p.scale_log2), nl2 = f32x2_pack(neg_lse, neg_lse);
      // (a row of dQ may have a scale of its own: the maximum of the rows around it)
      float held = 1.f;
      if (!BF16 && p.dout_max && live)
        held = ds_scale(__ldg(reinterpret_cast<const uint32_t*>(p.dout_max) + static_cast<int64_t>(bh) * p.maxima +
                              (static_cast<int64_t>(g) * p.M + m) / p.max_rows));
      const uint64_t held2 = f32x2_pack(held, held), nd2 = f32x2_pack(-dlt * held, -dlt * held);
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const uint32_t s_col = (j & 1) * 128 + half * 64;
        const int valid = len - j * 128 - half * 64;  // keys of this thread's columns
        if (!(ok = ok && wait_all(&s_full[j & 1], j >> 1))) break;
        tc_fence_after();
        float pv[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sv[32];
          tmem_ld32(lane_base + s_col + c * 32, sv);
          tmem_wait_ld32(sv);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const uint64_t x = f32x2_fma(f32x2_pack(__uint_as_float(sv[k]), __uint_as_float(sv[k + 1])), sc2, nl2);
            ex2_pair(x, (k & 2) != 0, pv[c * 32 + k], pv[c * 32 + k + 1]);
          }
        }
        if (!(ok = wait_all(dp_full, j))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t dp[32], ds[16];
          tmem_ld32(lane_base + kDP + half * 64 + c * 32, dp);
          tmem_wait_ld32(dp);
          if (valid < 64) {
            // keys past the length: dS = 0, whatever their scores and values are
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c * 32 + k >= valid) pv[c * 32 + k] = 0.f, dp[k] = 0u;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const uint64_t g = dp_minus<BF16>(dp[k], dp[k + 1], held2, nd2);
            float g0, g1;
            f32x2_unpack(g, g0, g1);
            ds[k / 2] = pack2<BF16>(pv[c * 32 + k] * g0, pv[c * 32 + k + 1] * g1);
          }
          tmem_st16(lane_base + s_col + c * 16, ds);
        }
        tmem_wait_st();
        if (j == n - 1 && (len & 127)) {
          // K rows past the length: zero before dS K may start, for dS = 0 times
          // what lies there (S_j, the tile's other reader, is complete)
          uint8_t* kt = sK + (j % SA) * C::TILE;
          for (int x = (len & 127) * 8 + (threadIdx.x - 128); x < 128 * 8; x += 256) {
#pragma unroll
            for (int c = 0; c < C::NCHUNK; ++c)
              *reinterpret_cast<uint4*>(kt + c * C::CHUNK + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
      }
      ok = ok && wait_all(done, 0);
      if (ok) {
        tc_fence_after();
        store_half_row<D, BF16>(lane_base + kDQ, half, p.sm_scale / held, orow, live, false);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// dK, dV: one CTA per 128 keys of one key / value head, over the query tiles of
// every query head that shares it.
// TMEM: S^T / P^T [0, 128), dP^T / dS^T [128, 256), dV [256, 256 + D), dK
// [256 + D, 256 + 2D).
// ---------------------------------------------------------------------------
template <int D, bool BF16>
__device__ void dkdv_tile(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const CUtensorMap& tmDO,
                          const DBwdParams& p, uint8_t* smem, int item) {
  using C = DBwdCfg<D>;
  constexpr int SA = C::SA, SB = C::SB;
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::TILE;
  uint8_t* sQ = sV + C::TILE;        // [SA]
  uint8_t* sDO = sQ + SA * C::TILE;  // [SB]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sDO + SB * C::TILE);
  float* col_lse = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + C::BAR_BYTES);  // [2][128]
  float* col_dlt = col_lse + 256;                                                                 // [2][128]
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;          // [SA]
  uint64_t* q_empty = q_full + SA;      // [SA] dK_i (its last reader) completed
  uint64_t* do_full = q_empty + SA;     // [SB]
  uint64_t* do_empty = do_full + SB;    // [SB] dV_i completed (dP_i was issued before)
  uint64_t* s_full = do_empty + SB;
  uint64_t* dp_full = s_full + 1;
  uint64_t* p_ready = dp_full + 1;      // 8 elementwise warps wrote P^T
  uint64_t* ds_ready = p_ready + 1;     // 8 elementwise warps wrote dS^T
  uint64_t* done = ds_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int bh = item / p.k_tiles, t = item - bh * p.k_tiles;
  const int b = bh / p.Hk, hk = bh - b * p.Hk;

  // Rows of a tile that no load fills: zero in every stage, so that their P = 0
  // and dS = 0 meet finite values in the sums over the queries.
  for (int x = p.mt * p.gh * 8 + threadIdx.x; x < 128 * 8; x += kThreadsB)
    for (int st = 0; st < SA + SB; ++st)
      for (int c = 0; c < C::NCHUNK; ++c)
        *reinterpret_cast<uint4*>(sQ + st * C::TILE + c * C::CHUNK + x * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < SA; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < SB; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 8);
    mbar_init(ds_ready, 8);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  const int len = bwd_len(p, b);
  const int n = t * 128 < len ? p.q_tiles : 0;  // steps: query tiles of the whole group
  auto wait = [&](uint64_t* bar, int k) { return mbar_wait(bar, k & 1, abort_flag, p.err, p.wait_ns); };
  auto wait_all = [&](uint64_t* bar, int k) { return __all_sync(0xffffffffu, wait(bar, k)) != 0; };

  if (warp == 0 && lane == 0 && n > 0) {
    // ------------------------------------------------------------- producer
    mbar_arrive_expect_tx(kv_full, 2 * C::TILE);
    for (int c = 0; c < C::NCHUNK; ++c) {
      tma_load_4d(sK + c * C::CHUNK, &tmK, kv_full, c * 64, t * 128, hk, b * p.kb_mul);
      tma_load_4d(sV + c * C::CHUNK, &tmV, kv_full, c * 64, t * 128, hk, b * p.vb_mul);
    }
    int nq = 0, nd = 0;  // loads issued
    for (int i = 0; i < n; ++i) {
      const int a = i % SA, o = i % SB;
      const int gi = i / p.nm, m0 = (i - gi * p.nm) * p.mt, h0 = hk * p.G + gi * p.gh;
      const int bytes = C::NCHUNK * p.mt * p.gh * 128;
      if (i >= SA && !wait(&q_empty[a], i / SA - 1)) break;
      mbar_arrive_expect_tx(&q_full[a], bytes);
      for (int c = 0; c < C::NCHUNK; ++c)
        tma_load_4d(sQ + a * C::TILE + c * C::CHUNK, &tmQ, &q_full[a], c * 64, m0, h0, b * p.qb_mul);
      ++nq;
      if (i >= SB && !wait(&do_empty[o], i / SB - 1)) break;
      mbar_arrive_expect_tx(&do_full[o], bytes);
      for (int c = 0; c < C::NCHUNK; ++c)
        tma_load_4d(sDO + o * C::TILE + c * C::CHUNK, &tmDO, &do_full[o], c * 64, m0, h0, b * p.db_mul);
      ++nd;
    }
    mbar_wait(kv_full, 0, nullptr, nullptr, p.wait_ns);
    for (int k = nq > SA ? nq - SA : 0; k < nq; ++k) mbar_wait(&q_full[k % SA], (k / SA) & 1, nullptr, nullptr, p.wait_ns);
    for (int k = nd > SB ? nd - SB : 0; k < nd; ++k) mbar_wait(&do_full[k % SB], (k / SB) & 1, nullptr, nullptr, p.wait_ns);
  } else if (warp == 1 && n > 0) {
    // -------------------- MMA issue (whole warp, one elected lane: see attn_dense.cu)
    constexpr uint32_t idesc_s = make_idesc_f16(BF16, 128, 128, false, false);
    constexpr uint32_t idesc_acc = make_idesc_f16(BF16, 128, D, false, true);
    constexpr int TS = C::TILE >> 4;
    const uint64_t kd = k_major(sK), vd = k_major(sV), qd = k_major(sQ), dod = k_major(sDO);
    const uint64_t qmn = mn_major(sQ), domn = mn_major(sDO);
    bool ok = wait_all(kv_full, 0);
    auto issue_s = [&](int i) {
      if (!(ok = ok && wait_all(&q_full[i % SA], i / SA))) return;
      tc_fence_after();
      if (elect_one()) {
        mma_abt<D>(tmem, kd, qd + (i % SA) * TS, idesc_s);
        tc_commit(s_full);
      }
      __syncwarp();
    };
    auto issue_dp = [&](int i) {
      if (!(ok = ok && wait_all(&do_full[i % SB], i / SB))) return;
      tc_fence_after();
      if (elect_one()) {
        mma_abt<D>(tmem + 128, vd, dod + (i % SB) * TS, idesc_s);
        tc_commit(dp_full);
      }
      __syncwarp();
    };
    if (ok) issue_s(0);
    if (ok) issue_dp(0);
    for (int i = 0; ok && i < n; ++i) {
      if (!(ok = wait_all(p_ready, i))) break;
      tc_fence_after();
      if (elect_one()) {
        mma_ab<D>(tmem + 256, tmem, domn + (i % SB) * TS, idesc_acc, i == 0);
        tc_commit(&do_empty[i % SB]);
      }
      __syncwarp();
      if (i + 1 < n) issue_s(i + 1);  // over P_i^T, which dV_i has read
      if (!(ok = ok && wait_all(ds_ready, i))) break;
      tc_fence_after();
      if (elect_one()) {
        mma_ab<D>(tmem + 256 + D, tmem + 128, qmn + (i % SA) * TS, idesc_acc, i == 0);
        tc_commit(&q_empty[i % SA]);
      }
      __syncwarp();
      if (i + 1 < n) issue_dp(i + 1);  // over dS_i^T
    }
    if (elect_one()) {
      tc_commit(done);
      mbar_wait(done, 0, nullptr, nullptr, p.wait_ns);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------- elementwise, epilogue
    const int q4 = warp & 3, half = (warp - 4) >> 2;
    const int row = q4 * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const int krow = t * 128 + row;
    const bool live = krow < p.N;
    uint8_t* krow_out = p.dk + 2 * (b * p.dk_b + hk * p.dk_h + static_cast<int64_t>(krow) * p.dk_n);
    uint8_t* vrow_out = p.dv + 2 * (b * p.dv_b + hk * p.dv_h + static_cast<int64_t>(krow) * p.dv_n);
    if (n == 0) {
      if (live) {
        zero_half_row<D>(half, krow_out);
        zero_half_row<D>(half, vrow_out);
      }
    } else {
      const uint64_t sc2 = f32x2_pack(p.scale_log2, p.scale_log2);
      float held = 1.f;
      if (!BF16 && p.dout_max) {
        const uint32_t* tops = reinterpret_cast<const uint32_t*>(p.dout_max) + static_cast<int64_t>(bh) * p.maxima;
        uint32_t top = 0;
#pragma unroll 8
        for (int i = lane; i < p.maxima; i += 32) top = max(top, __ldg(tops + i));
        held = ds_scale(__reduce_max_sync(0xffffffffu, top));
      }
      // P comes with 2^kHeldP in it, which dS takes off with dP - Delta
      constexpr float kHeldP = BF16 ? 0.f : 12.f, kTakeP = BF16 ? 1.f : 1.f / 4096.f;
      const float held_p = held * kTakeP;
      const uint64_t held2 = f32x2_pack(held_p, held_p);
      // the first warpgroup stages -lse, the second -Delta (scaled), of the step's 128
      // query rows; the value of the next step is fetched a step ahead
      auto fetch = [&](int i) -> float {
        int g, m;
        const bool in = query_of(p, i, row, g, m);
        const int64_t at = (static_cast<int64_t>(b) * p.H + hk * p.G + g) * p.M + m;
        return half == 0 ? neg_lse_of(p, in, at) + kHeldP : (in ? -__ldg(&p.delta[at]) * held_p : 0.f);
      };
      float next = fetch(0);
      bool ok = true;
      for (int i = 0; i < n; ++i) {
        const float* lb = col_lse + (i & 1) * 128 + half * 64;
        const float* db = col_dlt + (i & 1) * 128 + half * 64;
        (half == 0 ? col_lse : col_dlt)[(i & 1) * 128 + row] = next;
        if (i + 1 < n) next = fetch(i + 1);
        // (a warp whose wait failed keeps taking part in this barrier, which
        // has no time limit, and skips the rest of each step)
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (!(ok = ok && wait_all(s_full, i))) continue;
        tc_fence_after();
        float pv[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sv[32], pt[16];
          tmem_ld32(lane_base + half * 64 + c * 32, sv);
          tmem_wait_ld32(sv);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 nl = *reinterpret_cast<const float2*>(lb + c * 32 + k);
            const uint64_t x =
                f32x2_fma(f32x2_pack(__uint_as_float(sv[k]), __uint_as_float(sv[k + 1])), sc2, f32x2_pack(nl.x, nl.y));
            ex2_pair(x, (k & 2) != 0, pv[c * 32 + k], pv[c * 32 + k + 1]);
            pt[k / 2] = pack2<BF16>(pv[c * 32 + k], pv[c * 32 + k + 1]);
          }
          tmem_st16(lane_base + half * 64 + c * 16, pt);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        if (!(ok = wait_all(dp_full, i))) continue;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t dp[32], ds[16];
          tmem_ld32(lane_base + 128 + half * 64 + c * 32, dp);
          tmem_wait_ld32(dp);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 nd = *reinterpret_cast<const float2*>(db + c * 32 + k);
            const uint64_t g = dp_minus<BF16>(dp[k], dp[k + 1], held2, f32x2_pack(nd.x, nd.y));
            float g0, g1;
            f32x2_unpack(g, g0, g1);
            ds[k / 2] = pack2<BF16>(pv[c * 32 + k] * g0, pv[c * 32 + k + 1] * g1);
          }
          tmem_st16(lane_base + 128 + half * 64 + c * 16, ds);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
      }
      ok = ok && wait_all(done, 0);
      if (ok) {
        tc_fence_after();
        // keys past the length have no gradient
        const bool zero = krow >= len;
        store_half_row<D, BF16>(lane_base + 256, half, kTakeP, vrow_out, live, zero);
        store_half_row<D, BF16>(lane_base + 256 + D, half, p.sm_scale / held, krow_out, live, zero);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One launch for both: the dK / dV tiles first (the longer ones), then dQ.
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreadsB, 1)
    dense_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                     const __grid_constant__ DBwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) set_err(p.err, BSA_DEVERR_ALIGN);
    return;
  }
  const int kv_items = p.B * p.Hk * p.k_tiles;
  const int item = static_cast<int>(blockIdx.x);
  if (item < kv_items)
    dkdv_tile<D, BF16>(tmQ, tmK, tmV, tmDO, p, smem, item);
  else
    dq_tile<D, BF16>(tmQ, tmK, tmV, tmDO, p, smem, item - kv_items);
}

template <int D, bool BF16>
int launch_t(const bsa_cross_bwd_args* a, float* dout_max, cudaStream_t st) {
  using C = DBwdCfg<D>;
  auto kern = dense_bwd_kernel<D, BF16>;
  int r;
  if ((r = opt_in_smem(reinterpret_cast<const void*>(kern), C::SMEM))) return r;
  DBwdParams p{};
  CUtensorMap mq, mk{}, mv{}, mdo;
  // The tile shape with the fewest query tiles (8 tokens of 8 heads in one tile
  // instead of eight): the tokens in equal parts, then heads that divide a group.
  const int G = a->H / a->Hk;
  p.q_tiles = INT32_MAX;
  for (int parts = (a->M + 127) / 128, tries = 0; tries < 8 && parts <= a->M; ++parts, ++tries) {
    const int mt = a->M >= 128 && tries == 0 ? 128 : (a->M + parts - 1) / parts;
    int gh = 128 / mt < G ? 128 / mt : G;
    while (G % gh) --gh;
    const int nm = (a->M + mt - 1) / mt;
    if (static_cast<int64_t>(nm) * (G / gh) >= p.q_tiles) continue;
    p.mt = mt, p.gh = gh, p.nm = nm, p.q_tiles = nm * (G / gh);
  }
  if ((r = map_of(&mq, a->q, a->B, a->H, a->M, D, BF16, &p.qb_mul, p.mt, p.gh))) return r;
  if ((r = map_of(&mdo, a->dout, a->B, a->H, a->M, D, BF16, &p.db_mul, p.mt, p.gh))) return r;
  if (a->N > 0) {
    if ((r = map_of(&mk, a->k, a->B, a->Hk, a->N, D, BF16, &p.kb_mul))) return r;
    if ((r = map_of(&mv, a->v, a->B, a->Hk, a->N, D, BF16, &p.vb_mul))) return r;
  }
  if (BF16) dout_max = nullptr;
  if ((r = launch_bwd_delta(a->o, a->o_rest, a->dout, a->delta, a->B, a->H, a->M, D, BF16, st, dout_max, G))) return r;
  p.B = a->B, p.H = a->H, p.Hk = a->Hk, p.G = G, p.M = a->M, p.N = a->N;
  p.k_tiles = (a->N + 127) / 128;
  p.lens = a->k_lens;
  p.lens_i64 = a->lens_dtype == BSA_INDEX_I64;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.sm_scale = a->sm_scale;
  p.lse = a->lse;
  p.delta = a->delta;
  p.dout_max = dout_max;
  p.max_rows = bwd_delta_rows(D);
  p.maxima = static_cast<int>((static_cast<int64_t>(G) * a->M + p.max_rows - 1) / p.max_rows);
  p.dq = static_cast<uint8_t*>(a->dq.data), p.dq_b = a->dq.stride_b, p.dq_h = a->dq.stride_h, p.dq_n = a->dq.stride_n;
  p.dk = static_cast<uint8_t*>(a->dk.data), p.dk_b = a->dk.stride_b, p.dk_h = a->dk.stride_h, p.dk_n = a->dk.stride_n;
  p.dv = static_cast<uint8_t*>(a->dv.data), p.dv_b = a->dv.stride_b, p.dv_h = a->dv.stride_h, p.dv_n = a->dv.stride_n;
  p.err = a->err_flag;
  p.wait_ns = kWaitNs;
  const int64_t items =
      static_cast<int64_t>(p.B) * p.Hk * (static_cast<int64_t>(p.k_tiles) + p.q_tiles);
  if (items > INT32_MAX) return BSA_ERR_UNSUPPORTED;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items));
  cfg.blockDim = dim3(kThreadsB);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, mdo, p));
  return BSA_OK;
}

}  // namespace

int cross_bwd_validate(const bsa_cross_bwd_args* a) {
  if (!a) return BSA_ERR_INVALID_ARG;
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->M <= 0 || a->N < 0 || a->D <= 0) return BSA_ERR_INVALID_ARG;
  if (a->dtype != BSA_DTYPE_F16 && a->dtype != BSA_DTYPE_BF16) return BSA_ERR_DTYPE;
  if (a->H % a->Hk) return BSA_ERR_SHAPE;
  if (a->D != 64 && a->D != 128) return BSA_ERR_UNSUPPORTED;
  if (!(a->sm_scale > 0.f) || !(a->sm_scale < INFINITY)) return BSA_ERR_UNSUPPORTED;
  if (!a->lse || !a->delta) return BSA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->o_rest) % 16) return BSA_ERR_ALIGNMENT;
  if (static_cast<int64_t>(a->B) * a->H * a->M > INT32_MAX / 2 || a->N > INT32_MAX / 2) return BSA_ERR_UNSUPPORTED;
  const bsa_tensor4d* qs[] = {&a->q, &a->o, &a->dout, &a->dq};
  const bsa_tensor4d* ks[] = {&a->k, &a->v, &a->dk, &a->dv};
  for (int i = 0; i < 4; ++i) {
    if (!qs[i]->data) return BSA_ERR_INVALID_ARG;
    if (!aligned(*qs[i], a->B, a->H, a->M)) return BSA_ERR_ALIGNMENT;
    if (a->N == 0) continue;
    if (!ks[i]->data || ks[i]->stride_b < 0) return BSA_ERR_INVALID_ARG;
    if (!aligned(*ks[i], a->B, a->Hk, a->N)) return BSA_ERR_ALIGNMENT;
  }
  if (a->k_lens && a->lens_dtype != BSA_INDEX_I32 && a->lens_dtype != BSA_INDEX_I64) return BSA_ERR_DTYPE;
  return BSA_OK;
}

int launch_cross_bwd(const bsa_cross_bwd_args* a, float* dout_max, cudaStream_t st) {
  const bool bf = a->dtype == BSA_DTYPE_BF16;
  if (a->D == 128) return bf ? launch_t<128, true>(a, dout_max, st) : launch_t<128, false>(a, dout_max, st);
  return bf ? launch_t<64, true>(a, dout_max, st) : launch_t<64, false>(a, dout_max, st);
}

}  // namespace bsa
