// Root-mean-square norm of every query and key head and the rotation of its
// token's position, in one pass, and the gradient of both.
//
//   forward   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R(pos) (n o w)
//   backward  t = R(-pos) dy,  dw = sum over rows of t o n,
//             dx = r (u - n mean(u o n)),  u = t o w
// R(pos) turns the pairs of the row's first R dimensions by the angles whose
// cosines and sines the caller's table holds at row `pos`: pairs (i, i + R/2),
// or neighbours (2i, 2i + 1).  The remaining dimensions only get the norm.
// Sums, the norm and the rotation are fp32; y and dx are rounded once.
//
// Bound by memory: each row is read and written once (backward: x and dy read,
// dx written).  A row belongs to D / 8 neighbouring lanes, 8 elements (one or
// two 16-byte accesses) each, so the mean square takes log2(D / 8) shuffles
// and a pair's other half is one shuffle away (or in the same lane).  A fp32
// table row is twice as long as a 16-bit row of the same D, so a lane group
// keeps its token's angles in registers and walks over the token's heads.
// Measured: 16,384 tokens of 32 heads x 128, bf16, 53 us (5.2 TB/s), of 20
// heads x 64, fp16, gradient 33 us; 4,593 tokens of 15 heads x 128, fp32, 18 us,
// gradient 26 us.
#include "common.cuh"
#include "internal.h"
#include "softmax.cuh"

namespace bsa {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxD = 256;

// One tensor pair of the call (queries or keys).
struct RopeSide {
  const uint8_t* x;
  uint8_t* y;         // forward: output; backward: dx
  const uint8_t* dy;  // backward only
  const void* w;      // [D] or null (ones)
  int64_t xs_b, xs_h, xs_n, ys_b, ys_h, ys_n, ds_b, ds_h, ds_n;
  int heads;
};

struct RopeParams {
  RopeSide side[2];
  int N, D, R;
  int64_t tokens;  // B * N
  const float* cos;
  const float* sin;
  int64_t table_stride;
  int table_len;
  const void* pos;  // null: the token's index
  int pos_i64;
  int64_t pos_stride_b;
  int w_f32;
  float eps;
  int chunk;       // heads per block row
  int q_chunks;    // block rows of the queries; the rest are the keys'
  float* partial;  // backward: [blocks][2][D] sums of dw
  int32_t* err;
};

template <typename T>
struct Vec8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const uint8_t* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
// Read once and not again: the line goes first when the cache needs room.  (The
// gradient, with three streams: 37.4 -> 33.5 us and, fp32, 30.2 -> 26.3; the
// forward is 1 us slower with it at 16,384 tokens x 32 heads.)
template <typename T>
__device__ __forceinline__ Vec8<T> load8_once(const uint8_t* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ Vec8<T> zero8() {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = make_uint4(0, 0, 0, 0);
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T>& r, float (&f)[8]) {
  const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(t[i]);
}
template <typename T>
__device__ __forceinline__ void store8(uint8_t* p, const float (&f)[8]) {
  Vec8<T> r;
  T* t = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(f[i]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.v[i];
}

// The 8 elements as pairs for the paired fp32 instructions: with scalar ones the
// kernels were bound by issue slots (73 % of them busy at 54 % of the memory rate).
__device__ __forceinline__ void pairs8(const float (&f)[8], uint64_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = f32x2_pack(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ float pair_sum(uint64_t p) {
  float a, b;
  f32x2_unpack(p, a, b);
  return a + b;
}
template <typename T>
__device__ __forceinline__ void store_pairs(uint8_t* p, const uint64_t (&y)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f32x2_unpack(y[i], f[2 * i], f[2 * i + 1]);
  store8<T>(p, f);
}

template <int LPR>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// What a lane keeps of its token: the cosine and signed sine of each of its
// elements (y_i = x_i c_i + partner_i s_i), and where the partner is.
struct Turn {
  float c[8], s[8];
  int partner;  // lane of the pair's other half
  bool on;      // this lane's elements are rotated
};

// The other halves of a row's pairs: from the lane's own values, or from the
// partner lane's, shuffled as they were loaded (a 16-bit pair a shuffle).
template <typename T, bool IL>
__device__ __forceinline__ void other_half(const Vec8<T>& raw, const float (&x)[8], int partner, float (&o)[8]) {
  if constexpr (IL) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = x[i ^ 1];
  } else {
    Vec8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
      r.v[i].x = __shfl_sync(0xffffffffu, raw.v[i].x, partner);
      r.v[i].y = __shfl_sync(0xffffffffu, raw.v[i].y, partner);
      r.v[i].z = __shfl_sync(0xffffffffu, raw.v[i].z, partner);
      r.v[i].w = __shfl_sync(0xffffffffu, raw.v[i].w, partner);
    }
    unpack8<T>(r, o);
  }
}

// The angles of element group `l` (8 elements) at table row `pos`.
template <bool IL>
__device__ __forceinline__ void load_turn(const RopeParams& p, int l, int lane, int64_t pos, bool valid, Turn& t) {
  const int half = p.R >> 1;
  t.on = valid && l * 8 < p.R;
  t.partner = lane;
#pragma unroll
  for (int i = 0; i < 8; ++i) t.c[i] = 1.f, t.s[i] = 0.f;
  if constexpr (!IL) {
    // partner lanes are the same whatever the position, so that all lanes take part in the shuffles
    if (l * 8 < p.R) t.partner = l * 8 < half ? lane + half / 8 : lane - half / 8;
  }
  if (!t.on) return;
  if constexpr (IL) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + pos * p.table_stride + l * 4));
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + pos * p.table_stride + l * 4));
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) t.c[i] = cc[i / 2], t.s[i] = (i & 1) ? ss[i / 2] : -ss[i / 2];
  } else {
    const bool second = l * 8 >= half;
    const int64_t at = pos * p.table_stride + (second ? l * 8 - half : l * 8);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + at) + k);
      const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + at) + k);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) t.c[4 * k + i] = cc[i], t.s[4 * k + i] = second ? ss[i] : -ss[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int l, bool in, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = !in || !w ? 1.f
                     : (w_f32 ? __ldg(static_cast<const float*>(w) + l * 8 + i)
                              : to_f32(static_cast<const T*>(w)[l * 8 + i]));
}

// The token's position: table row, and whether it lies in the table.
__device__ __forceinline__ bool token_pos(const RopeParams& p, int64_t b, int64_t n, int64_t& pos) {
  pos = n;
  if (p.pos) {
    const int64_t i = b * p.pos_stride_b + n;
    pos = p.pos_i64 ? __ldg(static_cast<const int64_t*>(p.pos) + i)
                    : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.pos) + i));
  }
  return p.R == 0 || (pos >= 0 && pos < p.table_len);
}

// U rows (heads of one token) are in flight while U are computed: loads of the
// first ones go out before the position and its table row are known, and four
// blocks an SM keep 64 KB on the way.  (16 + 16 heads x 16,384 tokens x 128, bf16,
// 277 MB: 65 us with the loads behind the table and three blocks an SM.)
template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kThreads, 4) rope_fwd_kernel(const RopeParams p) {
  constexpr int U = sizeof(T) == 4 ? 1 : 2;
  constexpr int E = sizeof(T);
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * (kThreads / LPR) + threadIdx.x / LPR;
  const bool keys = static_cast<int>(blockIdx.y) >= p.q_chunks;
  const RopeSide& sd = p.side[keys ? 1 : 0];
  const int h0 = (static_cast<int>(blockIdx.y) - (keys ? p.q_chunks : 0)) * p.chunk;
  const int h1 = min(h0 + p.chunk, sd.heads);
  const bool live = token < p.tokens;
  const bool in = live && l * 8 < p.D;
  const int64_t b = live ? token / p.N : 0, n = live ? token - b * p.N : 0;
  const uint8_t* xp = sd.x + E * (b * sd.xs_b + n * sd.xs_n + l * 8);
  uint8_t* yp = sd.y + E * (b * sd.ys_b + n * sd.ys_n + l * 8);
  Vec8<T> next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = in && h0 + u < h1 ? load8<T>(xp + E * ((h0 + u) * sd.xs_h)) : zero8<T>();
  int64_t pos = 0;
  const bool valid = live && token_pos(p, b, n, pos);
  if (live && !valid && l == 0) set_err(p.err, BSA_DEVERR_COORD);
  Turn t;
  load_turn<IL>(p, l, lane, pos, valid, t);
  // y = r (x o A + other half o B): weights and angles in one factor each
  float A[8], B[8];
  load_weight<T>(sd.w, p.w_f32, l, in, A);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    B[i] = t.s[i] * (IL ? A[i ^ 1] : __shfl_sync(0xffffffffu, A[i], t.partner));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) A[i] *= t.c[i];
  uint64_t A2[4], B2[4];
  pairs8(A, A2);
  pairs8(B, B2);
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int64_t xstep = E * sd.xs_h, ystep = E * sd.ys_h;
  const uint8_t* xn = xp + E * ((h0 + U) * sd.xs_h);
  yp += E * (h0 * sd.ys_h);
  for (int h = h0; h < h1; h += U) {
    Vec8<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = next[u];
      next[u] = in && h + U + u < h1 ? load8<T>(xn) : zero8<T>();
      xn += xstep;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8], o[8];
      uint64_t x2[4], o2[4];
      unpack8<T>(raw[u], x);
      pairs8(x, x2);
      uint64_t s2 = f32x2_mul(x2[0], x2[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) s2 = f32x2_fma(x2[i], x2[i], s2);
      const float ss = group_sum<LPR>(pair_sum(s2));
      // (a position outside the table: NaN rather than a row that looks right)
      const float r = valid ? rsqrtf(fmaf(ss, inv_d, p.eps)) : NAN;
      const uint64_t r2 = f32x2_pack(r, r);
      other_half<T, IL>(raw[u], x, t.partner, o);
      pairs8(o, o2);
      if (t.on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x2[i] = f32x2_mul(r2, f32x2_fma(x2[i], A2[i], f32x2_mul(o2[i], B2[i])));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x2[i] = f32x2_mul(r2, f32x2_mul(x2[i], A2[i]));
      }
      if (in && h + u < h1) store_pairs<T>(yp, x2);
      yp += ystep;
    }
  }
}

// Backward: a block walks over tokens (grid-stride), each lane group over the
// heads of one side, and keeps its 8 columns' sums of dw in registers; the
// block adds its groups in a fixed order and writes one row of `partial`.
// grid.y: 0 = queries, 1 = keys.
template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kThreads, 3) rope_bwd_kernel(const RopeParams p) {
  constexpr int E = sizeof(T);
  constexpr int GP = kThreads / LPR;
  __shared__ float sums[GP][LPR * 8 + 4];
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const RopeSide& sd = p.side[blockIdx.y];
  const bool cols = l * 8 < p.D;
  float w[8];
  uint64_t w2[4], dw2[4] = {0, 0, 0, 0};
  load_weight<T>(sd.w, p.w_f32, l, cols, w);
  pairs8(w, w2);
  const int64_t xstep = E * sd.xs_h, dstep = E * sd.ds_h, ystep = E * sd.ys_h;
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int chunks = (sd.heads + p.chunk - 1) / p.chunk;
  const int64_t items = p.tokens * chunks;
  // whole blocks stay in the loop together (the shuffles name every lane)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * GP; base < items; base += static_cast<int64_t>(gridDim.x) * GP) {
    const int64_t item = base + threadIdx.x / LPR;
    const bool live = item < items;
    // neighbouring lane groups take neighbouring tokens of one chunk of heads
    const int64_t ck = live ? item / p.tokens : 0, token = live ? item - ck * p.tokens : 0;
    const int64_t b = token / p.N, n = token - b * p.N;
    const int h0 = static_cast<int>(ck) * p.chunk, h1 = min(h0 + p.chunk, sd.heads);
    const bool in = live && cols;
    const uint8_t* xp = sd.x + E * (b * sd.xs_b + n * sd.xs_n + h0 * sd.xs_h + l * 8);
    const uint8_t* dp = sd.dy + E * (b * sd.ds_b + n * sd.ds_n + h0 * sd.ds_h + l * 8);
    uint8_t* yp = sd.y + E * (b * sd.ys_b + n * sd.ys_n + h0 * sd.ys_h + l * 8);
    Vec8<T> nx = in ? load8_once<T>(xp) : zero8<T>();
    Vec8<T> nd = in ? load8_once<T>(dp) : zero8<T>();
    int64_t pos = 0;
    const bool valid = live && token_pos(p, b, n, pos);
    if (live && !valid && l == 0) set_err(p.err, BSA_DEVERR_COORD);
    Turn t;
    load_turn<IL>(p, l, lane, pos, valid, t);
    // (turned back: the sines with their signs the other way)
    uint64_t c2[4], s2[4];
    pairs8(t.c, c2);
#pragma unroll
    for (int i = 0; i < 4; ++i) s2[i] = f32x2_pack(-t.s[2 * i], -t.s[2 * i + 1]);
    for (int hh = 0; hh < p.chunk; ++hh) {
      const int h = h0 + hh;
      const Vec8<T> rx = nx, rd = nd;
      const bool more = in && hh + 1 < p.chunk && h + 1 < h1;
      xp += xstep, dp += dstep;
      nx = more ? load8_once<T>(xp) : zero8<T>();
      nd = more ? load8_once<T>(dp) : zero8<T>();
      float x[8], g[8], o[8];
      uint64_t x2[4], g2[4], o2[4];
      unpack8<T>(rx, x);
      unpack8<T>(rd, g);
      pairs8(x, x2);
      pairs8(g, g2);
      other_half<T, IL>(rd, g, t.partner, o);
      pairs8(o, o2);
      if (t.on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g2[i] = f32x2_fma(g2[i], c2[i], f32x2_mul(o2[i], s2[i]));
      }
      uint64_t ss2 = f32x2_mul(x2[0], x2[0]), u2[4], dot2 = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i) ss2 = f32x2_fma(x2[i], x2[i], ss2);
        u2[i] = f32x2_mul(g2[i], w2[i]);
        dot2 = f32x2_fma(u2[i], x2[i], dot2);
      }
      const float ss = group_sum<LPR>(pair_sum(ss2));
      const float dot = group_sum<LPR>(pair_sum(dot2));
      const bool ok = in && h < h1;
      // (a row that is not there adds 0 to dw, whatever eps is)
      const float r = ok ? (valid ? rsqrtf(fmaf(ss, inv_d, p.eps)) : NAN) : 0.f;
      const float m = -dot * r * inv_d;  // -mean(u o n)
      const uint64_t r2 = f32x2_pack(r, r), m2 = f32x2_pack(m, m);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t n2 = f32x2_mul(x2[i], r2);
        dw2[i] = f32x2_fma(g2[i], n2, dw2[i]);
        x2[i] = f32x2_mul(r2, f32x2_fma(n2, m2, u2[i]));
      }
      if (ok) store_pairs<T>(yp, x2);
      yp += ystep;
    }
  }
  if (!p.partial) return;
  const int g = threadIdx.x / LPR;
#pragma unroll
  for (int i = 0; i < 4; ++i) f32x2_unpack(dw2[i], sums[g][l * 8 + 2 * i], sums[g][l * 8 + 2 * i + 1]);
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kThreads) {
    float a = 0.f;
#pragma unroll 8
    for (int k = 0; k < GP; ++k) a += sums[k][c];
    p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + blockIdx.y) * p.D + c] = a;
  }
}

// dw[side][c] = sum over blocks of partial[block][side][c]: 32 columns a
// block, 32 warps over the rows, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) rope_dw_kernel(const float* partial, int blocks, int D, int w_f32, void* dwq,
                                                       void* dwk) {
  __shared__ float s[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 32 + lane, side = blockIdx.y;
  void* dw = side ? dwk : dwq;
  if (!dw) return;
  float a = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int r = warp; r < blocks; r += 32) a += partial[(static_cast<int64_t>(r) * 2 + side) * D + c];
  }
  s[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][lane];
    if (w_f32)
      static_cast<float*>(dw)[c] = t;
    else
      static_cast<T*>(dw)[c] = from_f32<T>(t);
  }
}

int lanes_per_row(int D) {
  int l = 2;
  while (l * 8 < D) l *= 2;
  return l;
}

template <typename T, bool IL>
int dispatch(const RopeParams& p, int lpr, dim3 grid, bool bwd, cudaStream_t st) {
  switch (lpr) {
#define BSA_ROPE_CASE(L_)                                             \
  case L_:                                                            \
    if (bwd)                                                          \
      rope_bwd_kernel<T, L_, IL><<<grid, kThreads, 0, st>>>(p);       \
    else                                                              \
      rope_fwd_kernel<T, L_, IL><<<grid, kThreads, 0, st>>>(p);       \
    break;
    BSA_ROPE_CASE(2)
    BSA_ROPE_CASE(4)
    BSA_ROPE_CASE(8)
    BSA_ROPE_CASE(16)
    BSA_ROPE_CASE(32)
#undef BSA_ROPE_CASE
    default: return BSA_ERR_UNSUPPORTED;
  }
  BSA_CUDA_CHECK(cudaGetLastError());
  return BSA_OK;
}

int dispatch_type(const RopeParams& p, int dtype, int lpr, bool il, dim3 grid, bool bwd, cudaStream_t st) {
  switch (dtype) {
    case BSA_DTYPE_F32: return il ? dispatch<float, true>(p, lpr, grid, bwd, st) : dispatch<float, false>(p, lpr, grid, bwd, st);
    case BSA_DTYPE_F16: return il ? dispatch<__half, true>(p, lpr, grid, bwd, st) : dispatch<__half, false>(p, lpr, grid, bwd, st);
    default:
      return il ? dispatch<__nv_bfloat16, true>(p, lpr, grid, bwd, st) : dispatch<__nv_bfloat16, false>(p, lpr, grid, bwd, st);
  }
}

// Rows that 16-byte accesses can take: the base and every stride of a
// dimension longer than one.
bool rows_aligned(const bsa_tensor4d& t, int B, int H, int N, int eb) {
  return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && (B == 1 || t.stride_b * eb % 16 == 0) &&
         (H == 1 || t.stride_h * eb % 16 == 0) && (N == 1 || t.stride_n * eb % 16 == 0);
}

int validate(const bsa_rope_args* a, bool bwd) {
  if (!a) return BSA_ERR_INVALID_ARG;
  if (a->B <= 0 || a->H < 0 || a->Hk < 0 || (a->H == 0 && a->Hk == 0) || a->N <= 0 || a->D <= 0) return BSA_ERR_INVALID_ARG;
  const int eb = dtype_bytes(a->dtype);
  if (!eb) return BSA_ERR_DTYPE;
  if (a->D % 8 || a->D > kMaxD || a->R < 0 || a->R > a->D || a->R % 16) return BSA_ERR_UNSUPPORTED;
  if (a->H > 65535 || a->Hk > 65535) return BSA_ERR_UNSUPPORTED;
  if (a->weight_dtype != BSA_DTYPE_F32 && a->weight_dtype != a->dtype) return BSA_ERR_DTYPE;
  if (!(a->eps >= 0.f)) return BSA_ERR_INVALID_ARG;
  if (a->R > 0) {
    if (!a->cos || !a->sin || a->table_len <= 0) return BSA_ERR_INVALID_ARG;
    if (a->table_stride < a->R / 2) return BSA_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(a->cos) % 16 || reinterpret_cast<uintptr_t>(a->sin) % 16 || a->table_stride % 4)
      return BSA_ERR_ALIGNMENT;
    if (a->positions && a->pos_dtype != BSA_INDEX_I32 && a->pos_dtype != BSA_INDEX_I64) return BSA_ERR_DTYPE;
  }
  for (int s = 0; s < 2; ++s) {
    const int heads = s ? a->Hk : a->H;
    if (!heads) continue;
    const bsa_tensor4d* ts[] = {s ? &a->k : &a->q, s ? &a->k_out : &a->q_out, s ? &a->dk_out : &a->dq_out};
    for (int i = 0; i < (bwd ? 3 : 2); ++i) {
      if (!ts[i]->data) return BSA_ERR_INVALID_ARG;
      if (!rows_aligned(*ts[i], a->B, heads, a->N, eb)) return BSA_ERR_ALIGNMENT;
    }
  }
  return BSA_OK;
}

RopeParams params(const bsa_rope_args* a) {
  RopeParams p{};
  for (int s = 0; s < 2; ++s) {
    const bsa_tensor4d &x = s ? a->k : a->q, &y = s ? a->k_out : a->q_out, &d = s ? a->dk_out : a->dq_out;
    RopeSide& sd = p.side[s];
    sd.x = static_cast<const uint8_t*>(x.data), sd.xs_b = x.stride_b, sd.xs_h = x.stride_h, sd.xs_n = x.stride_n;
    sd.y = static_cast<uint8_t*>(y.data), sd.ys_b = y.stride_b, sd.ys_h = y.stride_h, sd.ys_n = y.stride_n;
    sd.dy = static_cast<const uint8_t*>(d.data), sd.ds_b = d.stride_b, sd.ds_h = d.stride_h, sd.ds_n = d.stride_n;
    sd.w = s ? a->k_weight : a->q_weight;
    sd.heads = s ? a->Hk : a->H;
  }
  p.N = a->N, p.D = a->D, p.R = a->R;
  p.tokens = static_cast<int64_t>(a->B) * a->N;
  p.cos = a->cos, p.sin = a->sin, p.table_stride = a->table_stride, p.table_len = a->table_len;
  p.pos = a->positions, p.pos_i64 = a->pos_dtype == BSA_INDEX_I64, p.pos_stride_b = a->pos_stride_b;
  p.w_f32 = a->weight_dtype == BSA_DTYPE_F32;
  p.eps = a->eps;
  p.err = a->err_flag;
  return p;
}

// Blocks of the backward, which each write one row of partial sums: the token
// and head-chunk items, at most four blocks of a side for every SM.
int bwd_blocks(const bsa_rope_args* a) {
  const int gp = kThreads / lanes_per_row(a->D);
  const int64_t heads = a->H > a->Hk ? a->H : a->Hk;
  const int64_t items = static_cast<int64_t>(a->B) * a->N * ((heads + 3) / 4);
  const int64_t need = (items + gp - 1) / gp;
  return static_cast<int>(need < 4 * 148 ? need : 4 * 148);
}

}  // namespace

int launch_rope_fwd(const bsa_rope_args* a, cudaStream_t st) {
  const int rc = validate(a, false);
  if (rc) return rc;
  RopeParams p = params(a);
  const int lpr = lanes_per_row(a->D), gp = kThreads / lpr;
  const int64_t gx = (p.tokens + gp - 1) / gp;
  if (gx > INT32_MAX) return BSA_ERR_UNSUPPORTED;
  // Heads a lane group walks over: as many as share its angles while the grid
  // still fills the SMs.
  p.chunk = 16;
  auto rows = [&](int c) { return (a->H + c - 1) / c + (a->Hk + c - 1) / c; };
  while (p.chunk > 1 && gx * rows(p.chunk) < 148 * 8) p.chunk /= 2;
  while (rows(p.chunk) > 65535) p.chunk *= 2;
  p.q_chunks = (a->H + p.chunk - 1) / p.chunk;
  return dispatch_type(p, a->dtype, lpr, a->interleaved != 0, dim3(static_cast<unsigned>(gx), rows(p.chunk)), false, st);
}

size_t rope_bwd_workspace(const bsa_rope_args* a) { return static_cast<size_t>(bwd_blocks(a)) * 2 * a->D * sizeof(float); }

int rope_validate(const bsa_rope_args* a, bool bwd) { return validate(a, bwd); }

int launch_rope_bwd(const bsa_rope_args* a, void* workspace, size_t bytes, cudaStream_t st) {
  const int rc = validate(a, true);
  if (rc) return rc;
  RopeParams p = params(a);
  const bool sums = a->dq_weight || a->dk_weight;
  if (sums && (!workspace || bytes < rope_bwd_workspace(a))) return BSA_ERR_WORKSPACE;
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  p.chunk = 4;
  const int blocks = bwd_blocks(a), lpr = lanes_per_row(a->D);
  int r = dispatch_type(p, a->dtype, lpr, a->interleaved != 0, dim3(blocks, 2), true, st);
  if (r || !sums) return r;
  const dim3 grid((a->D + 31) / 32, 2);
  if (a->dtype == BSA_DTYPE_F16)
    rope_dw_kernel<__half><<<grid, 1024, 0, st>>>(p.partial, blocks, a->D, p.w_f32, a->dq_weight, a->dk_weight);
  else
    rope_dw_kernel<__nv_bfloat16><<<grid, 1024, 0, st>>>(p.partial, blocks, a->D, p.w_f32, a->dq_weight, a->dk_weight);
  BSA_CUDA_CHECK(cudaGetLastError());
  return BSA_OK;
}

}  // namespace bsa
