// Attention of at most 8 rows a key / value head (16 on short ranges): one
// decoding step of cross attention, and the own keys of a sequence behind a
// shared prefix.  bf16 / fp16, head dim 64 or 128.
//
// Bound by the bytes of K and V (a row costs 4 D flops for 4 D bytes of them,
// and 16 rows still leave the tensor cores idle), so this kernel is built
// around loads: every warp takes 16 keys at a time on its own, reads their K
// and V rows straight into registers in the order the matrix instructions want
// them (16-byte loads, full sectors), and waits for nobody until the end.  16
// warps an SM keep about 100 KB in flight, where 45 KB cover the latency.
// tcgen05 would pad the rows to 128 and pass every tile between four roles: 256
// units of 1 row x 211 to 1,500 keys took 37 us there and take 17 us here (floor
// 8.6), 32 units of 4 rows x 65,536 keys 169 us, 6.3 TB/s.
//
// Per 16 keys, with mma.sync m16n8k16 (the keys, then the dims, as the m axis,
// so that 8 rows fill the n axis):
//   S^T = K Q^T,  p = 2^(s scale - m),  O^T += V^T P^T
// Lane (g, c) = (lane / 4, lane % 4) holds K rows g and g + 8 in pieces of 8
// dims (the order of the contracted dims is free as long as Q's is the same),
// and V rows 2c, 2c + 1, 2c + 8, 2c + 9 in pieces of 8 dims, which byte
// permutes pair up along the keys; P^T's operand is S^T's accumulator through
// movmatrix.  The reference point m of a row moves only when a score exceeds it
// by the slack, which one vote tells (softmax.cuh).  The warps' sums are joined
// in shared memory in a fixed order, behind a shared prefix together with the
// prefix kernel's partial results.
#include "common.cuh"
#include "dense.h"
#include "internal.h"
#include "softmax.cuh"

namespace bsa {

namespace {

constexpr int kWarpsF = 8;
constexpr int kThreadsF = kWarpsF * 32;

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 16 bytes, or zeros where `ok` is false (keys past the length: they may not
// be read, and 0 x NaN would reach O).
__device__ __forceinline__ uint4 load16(const uint8_t* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Element e of two rows' 8-element pieces as a pair.
__device__ __forceinline__ uint32_t pair_at(const uint4& lo, const uint4& hi, int e) {
  return __byte_perm(word(lo, e >> 1), word(hi, e >> 1), (e & 1) ? 0x7632 : 0x5410);
}

// OTHER: joins the other source's partial results too.
template <int D, bool BF16, int NR, bool OTHER>
__global__ void __launch_bounds__(kThreadsF, NR == 1 ? 2 : 1) attn_few_kernel(const __grid_constant__ FewParams p) {
  constexpr int KP = D / 32;  // 16-byte pieces of a K row a lane holds
  constexpr int VP = D / 64;  // and of a V row
  constexpr int MT = D / 16;  // m tiles of O^T
  constexpr int ROWS = 8 * NR;
  constexpr int UB = 128 / D;
  constexpr float kSlack = BF16 ? 30.f : 14.f;  // log2: p stays below 2^30 (bf16), 2^14 (fp16)
  extern __shared__ __align__(16) float fsm[];
  float* sm_o = fsm;                          // [kWarpsF][ROWS][D]
  float* sm_m = sm_o + kWarpsF * ROWS * D;    // [kWarpsF][ROWS]
  float* sm_l = sm_m + kWarpsF * ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int unit = blockIdx.x / p.splits, split = blockIdx.x - unit * p.splits;
  // Behind the kernel of the call's other source there is nothing to wait for
  // (that kernel waited for what the inputs need before it let this one start),
  // but the end of this grid has to mean the end of both for the join, so it
  // waits last.
  if (!p.late) grid_dependency_wait();
  allow_dependents();
  const int b = p.shared_kv ? 0 : unit / p.Hk, hk = p.shared_kv ? unit : unit - b * p.Hk;
  int len = p.keys;
  if (p.lens) {
    const int64_t l = p.lens_i64 ? __ldg(static_cast<const int64_t*>(p.lens) + b)
                                 : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.lens) + b));
    if (l < 0 || l > p.keys) {
      if (threadIdx.x == 0) set_err(p.err, BSA_DEVERR_COORD);
    }
    len = static_cast<int>(l < 0 ? 0 : l > p.keys ? p.keys : l);
  }
  const int k0 = split * p.chunk, k1 = min(len, k0 + p.chunk);

  // (sequence, head, token) of row r of the unit
  auto row_of = [&](int r, int& rb, int& rh, int& rm) {
    const int sg = r / p.M;
    rm = r - sg * p.M;
    const int sq = sg / p.G;
    rh = hk * p.G + (sg - sq * p.G);
    rb = p.shared_kv ? sq : b;
  };

  float acc[NR][MT][4];
  float m_run[NR][2], l_run[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
    m_run[n][0] = m_run[n][1] = -INFINITY;
    l_run[n][0] = l_run[n][1] = 0.f;
  }

  if (k0 + warp * 16 * UB < k1) {
    uint4 qf[NR][KP];
    int limit[NR][2];  // keys that rows 2c, 2c + 1 see
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = n * 8 + g;
      int rb, rh, rm;
      row_of(r < p.rows ? r : 0, rb, rh, rm);
      const uint8_t* src = p.q + 2 * (rb * p.qs_b + rh * p.qs_h + rm * p.qs_n + c * 8);
#pragma unroll
      for (int i = 0; i < KP; ++i) qf[n][i] = load16(src + i * 64, r < p.rows);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = n * 8 + 2 * c + e;
        limit[n][e] = rr >= p.rows ? 0 : p.causal ? max(0, len - (p.M - 1 - rr % p.M)) : len;
      }
    }
    const uint8_t* kb = p.k + 2 * (b * p.ks_b + hk * p.ks_h + c * 8);
    const uint8_t* vb = p.v + 2 * (b * p.vs_b + hk * p.vs_h + g * 8);
    // UB blocks of 16 keys at a time: at D = 64 two, for the same bytes in flight
    for (int key0 = k0 + warp * 16 * UB; key0 < k1; key0 += kWarpsF * 16 * UB) {
      const bool whole = key0 + 16 * UB <= k1;
      uint4 kfs[UB][2][KP], vfs[UB][4][VP];
#pragma unroll
      for (int u = 0; u < UB; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = key0 + u * 16 + g + 8 * h;
          const uint8_t* src = kb + 2 * (row * p.ks_n);
#pragma unroll
          for (int i = 0; i < KP; ++i) kfs[u][h][i] = load16(src + i * 64, whole || row < k1);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int row = key0 + u * 16 + 2 * c + (h & 1) + 8 * (h >> 1);
          const uint8_t* src = vb + 2 * (row * p.vs_n);
#pragma unroll
          for (int i = 0; i < VP; ++i) vfs[u][h][i] = load16(src + i * 128, whole || row < k1);
        }
      }
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        const int key = key0 + u * 16;
        const uint4 (&kf)[2][KP] = kfs[u];
        const uint4 (&vf)[4][VP] = vfs[u];
        uint32_t pt[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KP; ++i) {
            mma_16816<BF16>(s, kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, qf[n][i].x, qf[n][i].y);
            mma_16816<BF16>(s, kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, qf[n][i].z, qf[n][i].w);
          }
          // s[2 h + e]: key g + 8 h, row 2c + e
          float x[4];
          bool over = false;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int e = t & 1;
            x[t] = key + g + 8 * (t >> 1) < limit[n][e] ? s[t] * p.scale_log2 : -INFINITY;
            over = over || (x[t] - m_run[n][e] > kSlack);
          }
          if (__any_sync(0xffffffffu, over)) {
            // a new reference point, from the block's max of each row, over the 8 lanes that hold its keys
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(x[e], x[2 + e]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              mx = fmaxf(mx - ref_below<BF16>(), m_run[n][e]);
              const float alpha = mx == -INFINITY ? 1.f : ex2_approx(m_run[n][e] - mx);
              m_run[n][e] = mx;
              l_run[n][e] *= alpha;
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                acc[n][j][e] *= alpha;
                acc[n][j][2 + e] *= alpha;
              }
            }
          }
          float pr[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int e = t & 1;
            pr[t] = ex2_approx(x[t] - (m_run[n][e] == -INFINITY ? 0.f : m_run[n][e]));
            l_run[n][e] += pr[t];
          }
          pt[n][0] = movmatrix_trans(pack2<BF16>(pr[0], pr[1]));
          pt[n][1] = movmatrix_trans(pack2<BF16>(pr[2], pr[3]));
        }
        // m tile j: rows g and g + 8 are dims g 8 + j and 64 + g 8 + j (D 128), g 8 + 2j and g 8 + 2j + 1 (D 64)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int e0 = VP == 2 ? j : 2 * j, e1 = VP == 2 ? j : 2 * j + 1, hi = VP - 1;
          const uint32_t a0 = pair_at(vf[0][0], vf[1][0], e0), a1 = pair_at(vf[0][hi], vf[1][hi], e1);
          const uint32_t a2 = pair_at(vf[2][0], vf[3][0], e0), a3 = pair_at(vf[2][hi], vf[3][hi], e1);
#pragma unroll
          for (int n = 0; n < NR; ++n) mma_16816<BF16>(acc[n][j], a0, a1, a2, a3, pt[n][0], pt[n][1]);
        }
      }
    }
  }
  // The other source's partial results, every eighth of a row to each warp, as if
  // they were keys of weight 2^lse: a lane takes the dims its accumulators hold.
  if constexpr (OTHER) {
    grid_dependency_wait();
    constexpr int KU = 2 * UB;  // in flight
    const int64_t row0 = static_cast<int64_t>(hk) * p.other_rows + static_cast<int64_t>(b) * p.G * p.M;
    for (int k = warp; k < p.other_splits; k += kWarpsF * KU) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float l[KU][2];
        float4 f[KU][2][2 * VP];
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + 2 * c + e, kk = k + u * kWarpsF;
            const bool there = r < p.rows && kk < p.other_splits;
            const int64_t at = there ? (row0 + r) * p.other_splits + kk : 0;
            l[u][e] = there ? __ldcg(p.other_lse + at) : -INFINITY;
            const float4* src = reinterpret_cast<const float4*>(p.other_o + at * D + g * 8);
#pragma unroll
            for (int i = 0; i < 2 * VP; ++i)  // (a partial result without keys is only its lse)
              f[u][e][i] = l[u][e] != -INFINITY ? __ldcg(src + (i >> 1) * 16 + (i & 1)) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (l[u][e] == -INFINITY) continue;
            const float mx = fmaxf(m_run[n][e], l[u][e]);
            const float alpha = ex2_approx(m_run[n][e] - mx), w = ex2_approx(l[u][e] - mx);
            m_run[n][e] = mx;
            l_run[n][e] = fmaf(l_run[n][e], alpha, g == 0 ? w : 0.f);  // (summed over the lanes g below)
#pragma unroll
            for (int i = 0; i < 2 * VP; ++i) {
              const float4 x = f[u][e][i];
              const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                // element 8 (i / 2) + 4 (i % 2) + t of the lane's dims
                const int j = VP == 2 ? 4 * (i & 1) + t : 2 * i + (t >> 1), h = VP == 2 ? i >> 1 : t & 1;
                acc[n][j][2 * h + e] = fmaf(acc[n][j][2 * h + e], alpha, w * xs[t]);
              }
            }
          }
      }
    }
  }
  // ------------------------------------------------ join the warps
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[n][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = n * 8 + 2 * c + e;
      if (g == 0) {
        sm_m[warp * ROWS + r] = m_run[n][e];
        sm_l[warp * ROWS + r] = l;
      }
      float* dst = sm_o + (warp * ROWS + r) * D + g * 8;
      if constexpr (VP == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < MT; j += 4)
            *reinterpret_cast<float4*>(dst + h * 64 + j) = make_float4(acc[n][j][2 * h + e], acc[n][j + 1][2 * h + e],
                                                                       acc[n][j + 2][2 * h + e], acc[n][j + 3][2 * h + e]);
      } else {
#pragma unroll
        for (int j = 0; j < MT; j += 2)
          *reinterpret_cast<float4*>(dst + 2 * j) =
              make_float4(acc[n][j][e], acc[n][j][2 + e], acc[n][j + 1][e], acc[n][j + 1][2 + e]);
      }
    }
  __syncthreads();
  constexpr int PER = D / 8;  // threads of a row, 8 columns each
  for (int t = threadIdx.x; t < p.rows * PER; t += kThreadsF) {
    const int r = t / PER, col = (t - r * PER) * 8;
    float mx = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < kWarpsF; ++w) {
      mx = fmaxf(mx, sm_m[w * ROWS + r]);
      nan = nan || isnan(sm_l[w * ROWS + r]);
    }
    float sum = 0.f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarpsF; ++w) {
      const float l = sm_l[w * ROWS + r];
      if (l == 0.f) continue;  // this warp saw no key of the row
      const float f = ex2_approx(sm_m[w * ROWS + r] - mx);
      sum = fmaf(f, l, sum);
      const float4* src = reinterpret_cast<const float4*>(sm_o + (w * ROWS + r) * D + col);
      const float4 u = src[0], v = src[1];
      o[0] = fmaf(f, u.x, o[0]), o[1] = fmaf(f, u.y, o[1]), o[2] = fmaf(f, u.z, o[2]), o[3] = fmaf(f, u.w, o[3]);
      o[4] = fmaf(f, v.x, o[4]), o[5] = fmaf(f, v.y, o[5]), o[6] = fmaf(f, v.z, o[6]), o[7] = fmaf(f, v.w, o[7]);
    }
    const float inv = nan ? NAN : sum > 0.f ? 1.f / sum : 0.f;
    const float lse = nan ? NAN : sum > 0.f ? mx + log2f(sum) : -INFINITY;
    if (p.part_o) {
      const int64_t slot = (static_cast<int64_t>(unit) * p.rows + r) * p.splits + split;
      float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D + col);
      dst[0] = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      dst[1] = make_float4(o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv);
      if (col == 0) p.part_lse[slot] = lse;
    } else {
      int rb, rh, rm;
      row_of(r, rb, rh, rm);
      uint4 x;
      x.x = pack2<BF16>(o[0] * inv, o[1] * inv);
      x.y = pack2<BF16>(o[2] * inv, o[3] * inv);
      x.z = pack2<BF16>(o[4] * inv, o[5] * inv);
      x.w = pack2<BF16>(o[6] * inv, o[7] * inv);
      const int64_t at = 2 * (rb * p.os_b + rh * p.os_h + rm * p.os_n + col);
      *reinterpret_cast<uint4*>(p.o + at) = x;
      if (p.o_rest) {
        x.x = pack2_rest<BF16>(o[0] * inv, o[1] * inv, x.x);
        x.y = pack2_rest<BF16>(o[2] * inv, o[3] * inv, x.y);
        x.z = pack2_rest<BF16>(o[4] * inv, o[5] * inv, x.z);
        x.w = pack2_rest<BF16>(o[6] * inv, o[7] * inv, x.w);
        *reinterpret_cast<uint4*>(p.o_rest + at) = x;
      }
      if (col == 0 && p.lse) p.lse[(static_cast<int64_t>(rb) * p.H + rh) * p.M + rm] = lse;
    }
  }
  if (!OTHER && p.late) grid_dependency_wait();
}

template <int D, bool BF16, int NR, bool OTHER>
int launch_t(const FewParams& p, cudaStream_t st) {
  constexpr int smem = kWarpsF * 8 * NR * (D + 2) * static_cast<int>(sizeof(float));
  auto kern = attn_few_kernel<D, BF16, NR, OTHER>;
  int rc = opt_in_smem(reinterpret_cast<const void*>(kern), smem);
  if (rc) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.units * p.splits));
  cfg.blockDim = dim3(kThreadsF);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  return BSA_OK;
}

}  // namespace

int launch_attn_few(const FewParams& p, int D, bool bf16, cudaStream_t st) {
#define BSA_FEW_CASE(D_, BF_, NR_) \
  if (D == D_ && bf16 == BF_ && (p.rows > 8 ? 2 : 1) == NR_) \
    return p.other_o ? launch_t<D_, BF_, NR_, true>(p, st) : launch_t<D_, BF_, NR_, false>(p, st);
  BSA_FEW_CASE(128, true, 1)
  BSA_FEW_CASE(128, true, 2)
  BSA_FEW_CASE(128, false, 1)
  BSA_FEW_CASE(128, false, 2)
  BSA_FEW_CASE(64, true, 1)
  BSA_FEW_CASE(64, true, 2)
  BSA_FEW_CASE(64, false, 1)
  BSA_FEW_CASE(64, false, 2)
#undef BSA_FEW_CASE
  return BSA_ERR_UNSUPPORTED;
}

}  // namespace bsa
