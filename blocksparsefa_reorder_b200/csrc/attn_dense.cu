// Attention over contiguous key ranges for sm_100a: cross attention (queries
// of one length, keys of another, padded per sequence, key / value heads
// shared by groups of query heads) and attention of a batch behind a shared
// prefix.  bf16 / fp16, head dim 64 or 128.
//
//   o = sum_j p_j v_j / l,  p_j = 2^(s_j scale - m),  l = sum_j p_j,
//   lse = m + log2 l,       s_j = q . k_j for the keys j the row may see
//
// A unit is one key / value head of one sequence, with the rows of every query
// head that shares it; in the shared prefix one unit holds the rows of all
// sequences, so that its keys are read once for the whole batch.  An item is
// one row tile of a unit times one range of key tiles (128 keys each); items
// are dealt to the persistent CTAs round robin.  Where few items would leave
// SMs idle the host splits the keys, and partial results (normalised o in fp32
// and its lse) are joined by attn_join_kernel:
//   m = max_i lse_i,  w_i = 2^(lse_i - m),  o = sum w_i o_i / sum w_i.
//
// A CTA runs two streams, each with its own softmax warpgroup, S and O
// columns in tensor memory:
//  * a tile of two subtiles (up to 128 rows each): stream s takes subtile s, and
//    both read each K / V tile once from shared memory;
//  * a unit of one subtile: both streams hold the same rows, stream s takes the
//    key tiles of parity s, and the epilogue joins the two.
// A subtile is a box of tokens x query heads x sequences, one TMA load.
// While one stream's softmax runs, the tensor cores work for the other.
// Per stream: S_i = Q K_i^T into TMEM, softmax (one row a thread) writes P_i as
// 16-bit pairs over S_i, then O += P_i V_i, then S_i+1; so S_i+1 seen complete
// means PV_i complete, and the softmax may rescale O and hand back the stages
// of V_i and K_i+1 without any further commit.
// Roles: warp 0 TMA producer; warp 1 issues tcgen05.mma (whole warp, one elected
// lane: with the operands in uniform registers a group of 8 takes 230 cycles to
// issue, from a diverged thread 560); warpgroups 1, 2 softmax of streams 0, 1;
// warpgroup 3 epilogue.
//
// Bound: 4 rows keys D flops against the tensor rate and, row by row, the 16
// exponentials a clock of an SM (as many cycles as the products at D = 128);
// with few rows the bytes of K and V.  Measured: 37 heads x 1024 rows x 16,384
// keys x 128 255 us (1,247 TF/s), D = 64 215 us; 16 heads x 4096 rows x 16,384
// keys 482 us (256 items over 148 SMs); 256 rows x 8 heads x 32,768 shared keys
// 46 us, of which 27 us are steps.
//
// Keys behind a sequence's length take no part: their scores are replaced, and
// their V rows are zeroed in shared memory (0 x NaN would reach O).
// Every wait is bounded; a timeout sets BSA_DEVERR_TIMEOUT and all roles drain.
#include <cudaTypedefs.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "dense.h"
#include "internal.h"
#include "softmax.cuh"

namespace bsa {

namespace {

constexpr int kThreadsD = 512;
constexpr int kSmemLimitD = 232448;
// setmaxnreg split: issue / two softmax / epilogue warpgroups, of a launch with 128 a thread
constexpr int kRegsLaunchD = 128;
constexpr int kRegsIssueD = 64;
constexpr int kRegsSoftmaxD = 168;
constexpr int kRegsEpilogueD = 112;
constexpr int kRegsSplitD = kRegsIssueD + 2 * kRegsSoftmaxD + kRegsEpilogueD;
static_assert(128 * kRegsSplitD <= kThreadsD * kRegsLaunchD, "register split");

// One source of keys.  Row r of a unit is query (sequence, head, token):
// r = (seq * G + g) * M + m.  Its rows lie in subtiles of mt tokens x gh heads x
// nb sequences, the tokens fastest.
struct DensePart {
  int rows;        // of a unit: seqs * G * M
  int seqs;        // sequences of a unit
  int mt, gh, nb;  // a subtile's tokens, heads, sequences
  int nm, ng;      // subtiles along the tokens and the heads of a unit
  int subs;        // subtiles of a unit
  int tiles;       // row tiles of a unit: two subtiles each (dual: one)
  int splits;      // key ranges
  int chunk;       // key tiles of a range
  int keys;        // keys the tensors hold
  int items;       // units * tiles * splits
  int shared_kv;   // a unit's keys serve every sequence (units: Hk, else B * Hk)
  int dual;        // one subtile: both streams run over its rows
  int kb_mul;      // 0: K / V batch stride 0 (one copy for the batch)
  int vb_mul;
  int qb_mul;      // 0: the queries' batch stride is 0
  int causal;      // query m of M sees keys below len - (M - 1 - m)
  const void* lens;  // [B] valid keys, or null (all)
  float* part_o;   // partial results, or null: this part is the whole result
  float* part_lse;
};

struct DenseParams {
  DensePart part[2];
  int nparts;
  int B, H, Hk, G, M;
  int lens_i64;
  uint8_t* o;
  uint8_t* o_rest;  // optional, laid out as o: what rounding left
  int64_t os_b, os_h, os_n;
  float* lse;
  float scale_log2;
  int32_t* err;
  uint64_t wait_ns;
};

template <int D>
struct DenseCfg {
  static constexpr int NCHUNK = D / 64;
  static constexpr int CHUNK = 128 * 128;   // 64 columns of 128 rows, 128-byte swizzle
  static constexpr int TILE = 128 * D * 2;
  static constexpr int SLOTS = D == 128 ? 5 : 12;
  static constexpr int BAR_BYTES = 512;
  static constexpr int STATS = 2 * 2 * 128 * 4;  // [stream][m, l][row]
  static constexpr int SMEM = (2 + SLOTS) * TILE + BAR_BYTES + STATS;
  static constexpr int O_COL = 256;  // S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [256+D, 256+2D)
  static_assert(SMEM <= kSmemLimitD, "shared memory budget");
  static_assert((2 * SLOTS + 18) * 8 + 8 <= BAR_BYTES, "barriers");
};

// One item as every role derives it from its number.
struct Item {
  int part, unit, split;
  int nk;       // key tiles to do
  int k0;       // first key
  int len;      // valid keys of the unit (all its sequences alike, but for causal rows)
  int sub0;     // first subtile
  int nsub;     // 1 or 2
  int b, hk;    // K / V coordinates (b: of the only sequence)
  bool dual;
};

__device__ __forceinline__ int clamp_len(const DenseParams& p, const DensePart& pt, int b) {
  if (!pt.lens) return pt.keys;
  const int64_t l = p.lens_i64 ? __ldg(static_cast<const int64_t*>(pt.lens) + b)
                               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(pt.lens) + b));
  if (l < 0 || l > pt.keys) set_err(p.err, BSA_DEVERR_COORD);
  return static_cast<int>(l < 0 ? 0 : l > pt.keys ? pt.keys : l);
}

__device__ __forceinline__ void get_item(const DenseParams& p, int w, Item& it) {
  it.part = w >= p.part[0].items ? 1 : 0;
  const DensePart& pt = p.part[it.part];
  w -= it.part ? p.part[0].items : 0;
  const int per_unit = pt.tiles * pt.splits;
  it.unit = w / per_unit;
  w -= it.unit * per_unit;
  it.split = w / pt.tiles;  // neighbouring CTAs: the same keys, so K / V come from L2
  const int tile = w - it.split * pt.tiles;
  it.dual = pt.dual != 0;
  it.sub0 = 2 * tile;
  it.nsub = min(2, pt.subs - it.sub0);
  if (pt.shared_kv) {
    it.b = 0;
    it.hk = it.unit;
    it.len = pt.keys;
  } else {
    it.b = it.unit / p.Hk;
    it.hk = it.unit - it.b * p.Hk;
    it.len = clamp_len(p, pt, it.b);
  }
  it.k0 = it.split * pt.chunk * 128;
  const int left = it.len - it.k0;
  it.nk = left <= 0 ? 0 : min(pt.chunk, (left + 127) / 128);
}

// First token, head (of the group) and sequence (of the unit) of a subtile.
__device__ __forceinline__ void origin_of(const DensePart& pt, int sub, int& m0, int& g0, int& s0) {
  const int q = sub / pt.nm, r = q / pt.ng;
  m0 = (sub - q * pt.nm) * pt.mt;
  g0 = (q - r * pt.ng) * pt.gh;
  s0 = r * pt.nb;
}

// Row `rl` of subtile `sub`: its head of the group, token and sequence of the
// unit; false where the subtile has no such row.
__device__ __forceinline__ bool row_of(const DenseParams& p, const DensePart& pt, int sub, int rl, int& sq, int& g, int& m) {
  int m0, g0, s0;
  origin_of(pt, sub, m0, g0, s0);
  const int q = rl / pt.mt, r = q / pt.gh;
  m = m0 + rl - q * pt.mt;
  g = g0 + q - r * pt.gh;
  sq = s0 + r;
  return r < pt.nb && m < p.M && g < p.G && sq < pt.seqs;
}

// Stage positions of K_t and V_t in the item's sequence of 2 nk loads (the
// order in which the MMA warp needs them).
__device__ __forceinline__ int k_at(const Item& it, int t) { return it.dual ? (t ? 2 * t - 1 : 0) : 2 * t; }
__device__ __forceinline__ int v_at(const Item& it, int t) {
  return it.dual ? min(2 * t + 2, 2 * it.nk - 1) : 2 * t + 1;
}
// steps of stream s, and the key tile of its i-th step
__device__ __forceinline__ int steps_of(const Item& it, int s) {
  return it.dual ? (it.nk - s + 1) / 2 : (s < it.nsub ? it.nk : 0);
}
__device__ __forceinline__ int tile_of(const Item& it, int s, int i) { return it.dual ? 2 * i + s : i; }

// A stage of the K / V ring and its phase.
template <int SL>
struct Ring {
  int st = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++st == SL) st = 0, ph ^= 1;
  }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreadsD, 1)
    attn_dense_kernel(const __grid_constant__ CUtensorMap tmQ0, const __grid_constant__ CUtensorMap tmK0,
                      const __grid_constant__ CUtensorMap tmV0, const __grid_constant__ CUtensorMap tmQ1,
                      const __grid_constant__ CUtensorMap tmK1, const __grid_constant__ CUtensorMap tmV1, const __grid_constant__ DenseParams p) {
  using C = DenseCfg<D>;
  constexpr int SL = C::SLOTS;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) set_err(p.err, BSA_DEVERR_ALIGN);
    return;
  }
  uint8_t* sQ = smem;                // [2][TILE]
  uint8_t* sKV = sQ + 2 * C::TILE;   // [SLOTS][TILE]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + SL * C::TILE);
  float* stats = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + C::BAR_BYTES);
  uint64_t* full = bars;                  // [SLOTS] tile landed
  uint64_t* empty = full + SL;            // [SLOTS] its last reader completed
  uint64_t* q_full = empty + SL;
  uint64_t* q_empty = q_full + 1;         // the item's last S completed
  uint64_t* s_full = q_empty + 1;         // [2] by stream
  uint64_t* p_ready = s_full + 2;         // [2] 4 softmax warps wrote P
  uint64_t* o_final = p_ready + 2;        // [2] the item's last PV completed
  uint64_t* o_empty = o_final + 2;        // [2] 4 epilogue warps read O
  uint64_t* stats_ready = o_empty + 2;    // [2] 4 softmax warps wrote (m, l)
  uint64_t* stats_empty = stats_ready + 2;  // [2] 4 epilogue warps read them
  uint64_t* drain = stats_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // warp-uniform for the compiler too
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < SL; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_final[i], 1);
      mbar_init(&o_empty[i], 4);
      mbar_init(&stats_ready[i], 4);
      mbar_init(&stats_empty[i], 4);
    }
    mbar_init(drain, 1);
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
  // set-up above touched this CTA's shared and tensor memory alone
  grid_dependency_wait();

  const int total = p.part[0].items + p.part[1].items;
  auto wait = [&](uint64_t* bar, int n) { return mbar_wait(bar, n & 1, abort_flag, p.err, p.wait_ns); };
  auto wait_all = [&](uint64_t* bar, int n) { return __all_sync(0xffffffffu, wait(bar, n)) != 0; };

  if (warp < 4) {
    regs_dec<kRegsIssueD>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ producer
      tma_prefetch_desc(&tmQ0);
      if (p.part[0].keys > 0) {  // (without keys there is no map of them)
        tma_prefetch_desc(&tmK0);
        tma_prefetch_desc(&tmV0);
      }
      int c = 0;      // loads so far
      int nq = 0;     // non-empty items so far
      bool ok = true;
      for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
        Item it;
        get_item(p, w, it);
        if (it.nk == 0) continue;
        const DensePart& pt = p.part[it.part];
        const CUtensorMap* mk = it.part ? &tmK1 : &tmK0;
        const CUtensorMap* mv = it.part ? &tmV1 : &tmV0;
        auto load = [&](bool is_v, int t) {
          const int st = c % SL;
          if (c >= SL && !wait(&empty[st], c / SL - 1)) return false;
          mbar_arrive_expect_tx(&full[st], C::TILE);
          const int cb = it.b * (is_v ? pt.vb_mul : pt.kb_mul);
          for (int ch = 0; ch < C::NCHUNK; ++ch)
            tma_load_4d(sKV + st * C::TILE + ch * C::CHUNK, is_v ? mv : mk, &full[st], ch * 64, it.k0 + t * 128, it.hk,
                        cb);
          ++c;
          return true;
        };
        if (!(ok = load(false, 0))) break;
        if (it.dual && it.nk > 1 && !(ok = load(false, 1))) break;
        if (nq > 0 && !(ok = wait(q_empty, nq - 1))) break;
        const int box = pt.mt * pt.gh * pt.nb * 128;  // bytes of one 64-column chunk
        mbar_arrive_expect_tx(q_full, it.nsub * C::NCHUNK * box);
        for (int s = 0; s < it.nsub; ++s) {
          int m0, g0, s0;
          origin_of(pt, it.sub0 + s, m0, g0, s0);
          const int qb = (pt.shared_kv ? s0 : it.b) * pt.qb_mul;
          for (int ch = 0; ch < C::NCHUNK; ++ch)
            tma_load_4d(sQ + s * C::TILE + ch * C::CHUNK, it.part ? &tmQ1 : &tmQ0, q_full, ch * 64, m0,
                        it.hk * p.G + g0, qb);
        }
        ++nq;
        const int ahead = it.dual ? 2 : 1;
        for (int t = 0; ok && t < it.nk; ++t) {
          ok = load(true, t);
          if (ok && t + ahead < it.nk) ok = load(false, t + ahead);
        }
      }
      // the next kernel of the stream may set itself up
      allow_dependents();
      // every load issued lands before the CTA exits
      for (int i = c > SL ? c - SL : 0; i < c; ++i) mbar_wait(&full[i % SL], (i / SL) & 1, nullptr, nullptr, p.wait_ns);
      if (nq > 0) mbar_wait(q_full, (nq - 1) & 1, nullptr, nullptr, p.wait_ns);
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issue
      // The whole warp, one elected lane, with nothing between the MMAs but
      // adding to descriptors: a group of 8 occupies the tensor cores for 512
      // cycles, and they queue about half of one, so an issuer slower than that
      // leaves them idle.
      constexpr uint32_t idesc_qk = make_idesc_f16(BF16, 128, 128, false, false);
      constexpr uint32_t idesc_pv = make_idesc_f16(BF16, 128, D, false, true);
      const uint64_t qd = make_sw128_desc(smem_u32(sQ), 16, 1024);
      const uint64_t kd = make_sw128_desc(smem_u32(sKV), 16, 1024);
      const uint64_t vd = make_sw128_desc(smem_u32(sKV), C::CHUNK, 1024);
      Ring<SL> ring;
      int nq = 0;           // non-empty items so far
      // by stream: P tiles consumed, items whose O it wrote
      int np0 = 0, np1 = 0, no0 = 0, no1 = 0;
      bool ok = true;
      auto landed = [&](const Ring<SL>& r) {
        return ok = ok && __all_sync(0xffffffffu, mbar_wait(&full[r.st], r.ph, abort_flag, p.err, p.wait_ns));
      };
      for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
        Item it;
        get_item(p, w, it);
        if (it.nk == 0) continue;
        const int n0 = steps_of(it, 0), n1 = steps_of(it, 1);
        const bool dual = it.dual;
        const int last_s = dual ? (it.nk - 1) & 1 : (n1 ? 1 : 0);  // stream of the item's last S and PV
        if (!(ok = wait_all(q_full, nq))) break;
        ++nq;
        Ring<SL> k, v;
        auto take = [&](Ring<SL>& r) {
          r = ring;
          ring.next();
          return landed(r);
        };
        // Step i of stream 0, then of stream 1: P_i V_i, S_i+1 (i = -1: the
        // first S).  The loads are taken in the order they were issued; the
        // second reader of a shared tile finds it landed.
        for (int i = -1; ok && i < n0; ++i) {
#pragma unroll 1
          for (int s = 0; ok && s < 2; ++s) {
            const int n = s ? n1 : n0;
            if (i >= 0 && i < n) {
              const bool last = i == n - 1;
              if ((s == 0 || dual) && !take(v)) break;
              const int np = s ? np1 : np0, no = s ? no1 : no0;
              if (i == 0 && no > 0 && !(ok = wait_all(&o_empty[s], no - 1))) break;
              if (!(ok = wait_all(&p_ready[s], np))) break;
              (s ? np1 : np0) += 1;
              (s ? no1 : no0) += last ? 1 : 0;
              tc_fence_after();
              const uint64_t b = vd + v.st * (C::TILE >> 4);
              const uint32_t st = tmem + s * 128, ot = tmem + C::O_COL + s * D;
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                  tc_mma_ts(ot, st + kk * 8, b + kk * (16 * 128 >> 4), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
                if (last) {
                  tc_commit(&o_final[s]);
                  // no later S of this stream tells the softmax that V is free
                  if (dual || s == last_s) tc_commit(&empty[v.st]);
                }
              }
              __syncwarp();
            }
            if (i + 1 < n) {
              if ((s == 0 || dual) && !take(k)) break;
              tc_fence_after();
              const uint64_t a = qd + (dual ? 0 : s * (C::TILE >> 4)), b = kd + k.st * (C::TILE >> 4);
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const int off = (kk >> 2) * (C::CHUNK >> 4) + (kk & 3) * 2;  // 32 bytes inside a chunk's rows
                  tc_mma_ss(tmem + s * 128, a + off, b + off, idesc_qk, kk > 0 ? 1u : 0u);
                }
                tc_commit(&s_full[s]);
                if (i + 2 == n && s == last_s) tc_commit(q_empty);
              }
              __syncwarp();
            }
          }
        }
      }
      if (elect_one()) {
        tc_commit(drain);
        mbar_wait(drain, 0, nullptr, nullptr, p.wait_ns);
      }
      __syncwarp();
    }
  } else if (warp < 12) {
    regs_inc<kRegsSoftmaxD>();
    // ---------------------------------------------------------------- softmax
    const int s = (warp - 4) >> 2;  // stream
    const int q4 = warp & 3;        // TMEM lane quarter
    const int row = q4 * 32 + lane;
    const uint32_t s_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16) + s * 128;
    const uint32_t o_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16) + C::O_COL + s * D;
    int c0 = 0;   // loads of earlier items
    int ns = 0;   // S tiles of this stream so far
    int ni = 0;   // items of this stream so far
    bool ok = true;
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      Item it;
      get_item(p, w, it);
      if (it.nk == 0) continue;
      const int n = steps_of(it, s);
      if (n == 0) {
        c0 += 2 * it.nk;
        continue;
      }
      const DensePart& pt = p.part[it.part];
      const bool releases = it.dual || it.nsub == 1 || s == 1;  // last reader of the shared tiles
      int kst = (c0 + k_at(it, tile_of(it, s, 0))) % SL;  // stage of the step's K; its V of the step before is one below
      // a warp without rows only keeps the barriers going
      const bool any_rows = q4 * 32 < pt.mt * pt.gh * pt.nb;
      int sq, g, m;
      int limit = row_of(p, pt, it.sub0 + (it.dual ? 0 : s), row, sq, g, m) ? it.len : 0;  // keys this row sees
      if (pt.causal) limit = max(0, limit - (p.M - 1 - m));
      float m_run = -INFINITY, l_run = 0.f;
      for (int i = 0; i < n; ++i, ++ns) {
        if (!(ok = ok && wait_all(&s_full[s], ns))) continue;
        tc_fence_after();
        const int t = tile_of(it, s, i);
        // S_i complete, and with it the PV of the step before: K_i and V_i-1 are free
        if (lane == 0 && releases) {
          if (q4 == 0) mbar_arrive(&empty[kst]);
          if (q4 == 1 && i > 0) mbar_arrive(&empty[kst ? kst - 1 : SL - 1]);
        }
        kst += it.dual ? (t ? 4 : 3) : 2;
        kst -= kst >= SL ? SL : 0;
        if (any_rows) {
          const int valid = limit - (it.k0 + t * 128);  // keys of this tile the row sees
          const bool mask = __any_sync(0xffffffffu, valid < 128);
          auto load = [&](int ch, uint32_t (&v)[32]) {
            tmem_ld32(s_base + ch * 32, v);
            tmem_wait_ld32(v);
            if (mask) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (ch * 32 + k >= valid) v[k] = __float_as_uint(-INFINITY);
            }
          };
          auto reference = [&]() {  // from the tile's max
            float mx = -INFINITY;
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t v[32];
              load(ch, v);
              mx = fmaxf(mx, row_max<32>(v));
            }
            return mx * p.scale_log2 - ref_below<BF16>();
          };
          uint32_t pr[64];
          auto exps = [&](auto cut) {  // cut: some keys of the tile are masked
            // a row that has seen nothing yet keeps m = -inf: its exponentials are 2^(-inf - 0) = 0
            const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
            float sum = 0.f;
            uint32_t buf[2][32];
            tmem_ld32(s_base, buf[0]);
            tmem_wait_ld32(buf[0]);
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              // the next 32 columns come while these are exponentiated
              uint32_t (&v)[32] = buf[ch & 1];
              uint32_t pp[16];
              if (ch < 3) tmem_ld32(s_base + (ch + 1) * 32, buf[(ch + 1) & 1]);
              if constexpr (decltype(cut)::value) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (ch * 32 + k >= valid) v[k] = __float_as_uint(-INFINITY);
              }
              sum += exp_block<32, BF16>(v, pp, p.scale_log2, neg_m);
#pragma unroll
              for (int k = 0; k < 16; ++k) pr[ch * 16 + k] = pp[k];
              if (ch < 3) tmem_wait_ld32(buf[(ch + 1) & 1]);
            }
            return sum;
          };
          // The reference point is the max of the row's first seen tile, and
          // moves only when a tile's sum passes the slack (softmax.cuh): a score
          // any amount above it gives inf.  (On the special function unit alone,
          // and whole tiles without the masking: 37 heads x 1024 rows x 16,384 keys
          // take 255 us at D = 128, 215 at 64; a quarter of the exponentials on the
          // FMA pipe, clamped to give inf there too, 267 and 229; the masking in
          // every tile 256 and 238.)
          if (__any_sync(0xffffffffu, m_run == -INFINITY && valid > 0)) {
            const float mx = reference();
            if (m_run == -INFINITY) m_run = mx;
          }
          float ls = mask ? exps(std::true_type{}) : exps(std::false_type{});
          if (__any_sync(0xffffffffu, !(ls <= ref_slack<BF16>()))) {
            const float m_new = fmaxf(m_run, reference());
            const float alpha = m_new == -INFINITY ? 1.f : ex2_approx(m_run - m_new);
            l_run *= alpha;
            m_run = m_new;
            ls = exps(std::true_type{});
            if (i > 0) {
#pragma unroll
              for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t v[32];
                tmem_ld32(o_base + ch * 32, v);
                tmem_wait_ld32(v);
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * alpha);
                tmem_st32(o_base + ch * 32, v);
              }
            }
          }
          l_run += ls;
          tmem_st32(s_base, pr);
          tmem_st32(s_base + 32, pr + 32);
          tmem_wait_st();
        }
        const int tail = it.len - (it.k0 + t * 128);
        if (tail < 128 && (it.dual || s == 0)) {
          // V rows past the length: zero before P V may start (a row is 128
          // bytes of each chunk, whatever its swizzle).  This stage's earlier
          // use was over before S_i, so the phase waited for is this load's.
          const int at = c0 + v_at(it, t);
          if (!(ok = wait_all(&full[at % SL], at / SL))) continue;
          uint8_t* vt = sKV + (at % SL) * C::TILE;
          for (int x = tail * 8 + row; x < 128 * 8; x += 128) {
#pragma unroll
            for (int ch = 0; ch < C::NCHUNK; ++ch)
              *reinterpret_cast<uint4*>(vt + ch * C::CHUNK + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[s]);
      }
      if (ni > 0) ok = ok && wait_all(&stats_empty[s], ni - 1);
      ++ni;
      stats[s * 256 + row] = m_run;
      stats[s * 256 + 128 + row] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&stats_ready[s]);
      c0 += 2 * it.nk;
    }
  } else {
    regs_dec<kRegsEpilogueD>();
    // --------------------------------------------------------------- epilogue
    const int q4 = warp & 3;
    const int row = q4 * 32 + lane;
    const uint32_t o_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16) + C::O_COL;
    int ni[2] = {0, 0};
    bool ok = true;
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      Item it;
      get_item(p, w, it);
      const DensePart& pt = p.part[it.part];
      const int nst = it.nk == 0 ? 0 : (steps_of(it, 1) > 0 ? 2 : 1);  // streams with an O
      const int passes = it.dual ? 1 : it.nsub;
      // this thread's rows' places in the result or in the partial results (null:
      // no such row) and their lse's, found while the item is computed
      auto place = [&](int ps, uint8_t*& dst, float*& dst_lse) {
        int sq, g, mm;
        const bool in = row_of(p, pt, it.sub0 + ps, row, sq, g, mm);
        const int b = pt.shared_kv ? sq : it.b, h = it.hk * p.G + g;
        const int64_t slot =
            (static_cast<int64_t>(it.unit) * pt.rows + (static_cast<int64_t>(sq) * p.G + g) * p.M + mm) * pt.splits + it.split;
        dst = !in          ? nullptr
              : pt.part_o ? reinterpret_cast<uint8_t*>(pt.part_o + slot * D)
                          : p.o + 2 * (b * p.os_b + h * p.os_h + mm * p.os_n);
        dst_lse = !in          ? nullptr
                  : pt.part_o ? pt.part_lse + slot
                  : p.lse     ? p.lse + (static_cast<int64_t>(b) * p.H + h) * p.M + mm
                              : nullptr;
      };
      uint8_t *dst0, *dst1 = nullptr;
      float *lse0, *lse1 = nullptr;
      place(0, dst0, lse0);
      if (passes > 1) place(1, dst1, lse1);
      for (int ps = 0; ps < passes; ++ps) {
        // streams whose O make up this pass's rows: [first, last)
        const int first = it.dual ? 0 : ps, last = it.nk == 0 ? first : (it.dual ? nst : ps + 1);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        for (int s = first; s < last; ++s) {
          ok = ok && wait_all(&stats_ready[s], ni[s]);
          if (ok) {
            m[s - first] = stats[s * 256 + row];
            l[s - first] = stats[s * 256 + 128 + row];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&stats_empty[s]);
          ok = ok && wait_all(&o_final[s], ni[s]);
          ++ni[s];
        }
        if (ok) tc_fence_after();
        // weights of the streams' sums: 2^(m_s - max) / l, 0 for a stream without any key
        const float mx = fmaxf(l[0] > 0.f ? m[0] : -INFINITY, l[1] > 0.f ? m[1] : -INFINITY);
        float f0 = l[0] > 0.f ? ex2_approx(m[0] - mx) : 0.f;
        float f1 = l[1] > 0.f ? ex2_approx(m[1] - mx) : 0.f;
        const float lt = f0 * l[0] + f1 * l[1];
        // (a sum that is NaN stays NaN: l > 0 is false only for 0 and NaN)
        const bool nan = isnan(l[0]) || isnan(l[1]);
        const float inv = nan ? NAN : (lt > 0.f ? 1.f / lt : 0.f);
        f0 *= inv;
        f1 *= inv;
        const float lse = nan ? NAN : (lt > 0.f ? mx + log2f(lt) : -INFINITY);
        uint8_t* const mine = ok ? (ps ? dst1 : dst0) : nullptr;
        float* const mine_lse = ps ? lse1 : lse0;
        if (ok && mine_lse) *mine_lse = lse;
        const bool have = it.nk > 0;
        if (have || !pt.part_o) {  // (a partial result without keys is only its lse)
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t v[32];
            if (have) {
              tmem_ld32(o_base + first * D + ch * 32, v);
              tmem_wait_ld32(v);
            }
#pragma unroll
            for (int k = 0; k < 32; ++k)
              v[k] = have && (l[0] > 0.f || nan) ? __float_as_uint(__uint_as_float(v[k]) * f0) : 0u;
            if (last - first == 2) {
              uint32_t u[32];
              tmem_ld32(o_base + D + ch * 32, u);
              tmem_wait_ld32(u);
              if (l[1] > 0.f) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  v[k] = __float_as_uint(fmaf(__uint_as_float(u[k]), f1, __uint_as_float(v[k])));
              }
            }
            if (have && ch == D / 32 - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0)
                for (int s = first; s < last; ++s) mbar_arrive(&o_empty[s]);
            }
            // 32 columns: 8 pieces of 16 bytes in fp32, 4 in 16 bits
            if (pt.part_o) {
              uint4 x[8];
#pragma unroll
              for (int g = 0; g < 8; ++g) x[g] = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
              transpose_pieces<8>(x);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int from = (lane & 24) + k;
                uint8_t* dst = shfl_ptr(mine, from);
                if (dst) *reinterpret_cast<uint4*>(dst + ch * 128 + (lane & 7) * 16) = x[k];
              }
            } else {
              // once for o and, where asked for, once for what its rounding left
#pragma unroll 1
              for (int turn = 0; turn < (p.o_rest ? 2 : 1); ++turn) {
                const int64_t to = turn ? p.o_rest - p.o : 0;
                uint4 x[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  uint32_t* y = reinterpret_cast<uint32_t*>(&x[g]);
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    float& lo = reinterpret_cast<float&>(v[8 * g + 2 * k]);
                    float& hi = reinterpret_cast<float&>(v[8 * g + 2 * k + 1]);
                    y[k] = pack2<BF16>(lo, hi);
                    float a, b;
                    unpack2<BF16>(y[k], a, b);
                    lo -= a, hi -= b;
                  }
                }
                transpose_pieces<4>(x);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int from = (lane & 28) + k;
                  uint8_t* dst = shfl_ptr(mine, from);
                  if (dst) *reinterpret_cast<uint4*>(dst + to + ch * 64 + (lane & 3) * 16) = x[k];
                }
              }
            }
          }
        }
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
// Joins the partial results of an output row: W warps a row, each D / 32
// columns a lane over every W-th partial result.  One whose lse is -inf saw no
// key and its o is not read.  W = 8 from eight partial results a row on
// (128 rows of 37: 5 us, with one warp a row 20 us), else 1.
// ---------------------------------------------------------------------------
struct JoinSrc {
  const float* o;
  const float* lse;
  int splits, rows, shared_kv;
};
struct JoinParams {
  JoinSrc src[2];
  int B, H, Hk, G, M;
  uint8_t* o;
  uint8_t* o_rest;
  int64_t os_b, os_h, os_n;
  float* lse;
};

template <int D, bool BF16, int W>
__global__ void __launch_bounds__(256) attn_join_kernel(const JoinParams p) {
  constexpr int V = D / 32;
  __shared__ float part[W == 1 ? 1 : W][D + 1];
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  if (row >= static_cast<int64_t>(p.B) * p.H * p.M) return;  // (W = 8: never)
  const int m = static_cast<int>(row % p.M);
  const int64_t bh = row / p.M;
  const int h = static_cast<int>(bh % p.H), b = static_cast<int>(bh / p.H);
  const int hk = h / p.G, g = h - hk * p.G;
  const float *ls[2], *os[2];
  int n[2];
  float mx = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const JoinSrc sr = p.src[s];
    const int64_t r = sr.shared_kv ? static_cast<int64_t>(hk) * sr.rows + (static_cast<int64_t>(b) * p.G + g) * p.M + m
                                   : (static_cast<int64_t>(b) * p.Hk + hk) * sr.rows + g * p.M + m;
    n[s] = sr.splits;
    ls[s] = sr.lse + r * sr.splits;
    os[s] = sr.o + r * sr.splits * D + lane * V;
    for (int k = lane; k < n[s]; k += 32) {
      const float l = ls[s][k];
      nan = nan || isnan(l);
      mx = fmaxf(mx, l);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  if (__any_sync(0xffffffffu, nan)) mx = NAN;
  float sum = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll 4
    for (int k = W == 1 ? 0 : warp; k < n[s]; k += W) {
      const float l = ls[s][k];
      const bool any = l != -INFINITY;
      const float* src = os[s] + static_cast<int64_t>(k) * D;
      float x[V];
      if constexpr (V == 4) {
        const float4 f = any ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
      } else {
        const float2 f = any ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
        x[0] = f.x, x[1] = f.y;
      }
      const float wt = any ? ex2_approx(l - mx) : 0.f;
      sum += wt;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(wt, x[i], acc[i]);
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) part[warp][lane * V + i] = acc[i];
    if (lane == 0) part[warp][D] = sum;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      sum += part[w][D];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += part[w][lane * V + i];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = 2 * (b * p.os_b + h * p.os_h + m * p.os_n + lane * V);
  uint32_t x[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) x[i] = pack2<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  auto store = [&](uint8_t* dst) {
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(x[0], x[1]);
    else
      *reinterpret_cast<uint32_t*>(dst) = x[0];
  };
  store(p.o + at);
  if (p.o_rest) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) x[i] = pack2_rest<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv, x[i]);
    store(p.o_rest + at);
  }
  if (lane == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : mx + log2f(sum);
}

// ---------------------------------------------------------------------------
// Host: splitting, workspace, launch.
// ---------------------------------------------------------------------------
constexpr int kSMs = 148;

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

struct DenseCall {
  int B, H, Hk, M, D, dtype;
  bsa_tensor4d q, o;
  int n;                      // sources of keys
  bsa_tensor4d k[2], v[2];
  int keys[2];
  bool shared_kv[2], causal[2];
  const void* lens[2];
  int lens_dtype;
  float sm_scale;
  float* lse;
  void* o_rest;
  int32_t* err;
};

// How one source is computed.
struct Source {
  bool few;                   // attn_few.cu
  bool dual;                  // both streams over the same rows
  int units, rows, seqs;
  int mt, gh, nb, nm, ng, subs, tiles;  // as in DensePart
  int splits, chunk;          // key ranges; key tiles (few: keys) of each
  size_t o_off, lse_off;      // partial results in the workspace
};
struct DensePlan {
  Source s[2];
  bool join;   // attn_join_kernel joins the partial results
  bool fused;  // the second source's few-rows kernel joins the first one's
  bool partial(int i) const { return join || (fused && i == 0); }
  size_t total;
};

Source source_of(const DenseCall& c, int i) {
  Source s{};
  const int G = c.H / c.Hk;
  s.seqs = c.shared_kv[i] ? c.B : 1;
  s.units = c.shared_kv[i] ? c.Hk : c.B * c.Hk;
  s.rows = s.seqs * G * c.M;
  // 9 to 16 rows leave the few-rows kernel half the warps an SM: it wins on
  // short ranges only (16 rows, 64 x 8 units of 512 keys 39 us against 48; 4 x 8
  // units of 65,536 keys 199 against 181).
  s.few = s.rows <= kFewRows / 2 || (s.rows <= kFewRows && c.keys[i] <= 8192);
  // The subtile shape with the fewest subtiles: the tokens in equal parts of at
  // most 128, as many heads as fit beside them, then as many sequences.
  s.subs = INT32_MAX;
  for (int parts = (c.M + 127) / 128, tries = 0; tries < 8 && parts <= c.M; ++parts, ++tries) {
    const int mt = c.M >= 128 && tries == 0 ? 128 : (c.M + parts - 1) / parts;
    const int gh = 128 / mt < G ? 128 / mt : G;
    const int fit = 128 / (mt * gh);
    const int nb = gh < G || (c.B > 1 && c.q.stride_b == 0) ? 1 : fit < s.seqs ? fit : s.seqs;
    const int nm = (c.M + mt - 1) / mt, ng = (G + gh - 1) / gh, ns = (s.seqs + nb - 1) / nb;
    if (static_cast<int64_t>(nm) * ng * ns >= s.subs) continue;
    s.mt = mt, s.gh = gh, s.nb = nb, s.nm = nm, s.ng = ng, s.subs = nm * ng * ns;
  }
  s.dual = s.subs == 1;
  s.tiles = (s.subs + 1) / 2;
  s.splits = 1;
  return s;
}

// The few-rows kernel: two CTAs an SM, whose time is their bytes.  Where the
// units alone do not fill the SMs, or a range is so long that ragged lengths
// would leave some of them busy alone at the end, the keys are split into about
// eight ranges an SM of at least 256 keys (a warp's share is then two blocks of
// 16).  (4 x 8 units of 4 rows x 65,536 keys: 4, 8, 16, 32 ranges an SM 173,
// 169, 176, 190 us, of 16,000 to 65,536 keys 133, 117, 115, 124 us; 256 units of
// 1,500 keys: one range 19 us, two and a join 27 us.)
void split_few(Source* s, int keys) {
  s->chunk = keys > 0 ? keys : 1;
  if (s->units < kSMs || keys > 8192) {
    const int64_t c = (static_cast<int64_t>(keys) * s->units + 8 * kSMs - 1) / (8 * kSMs);
    s->chunk = static_cast<int>(c < 256 ? 256 : (c + 127) / 128 * 128);
  }
  s->splits = keys > 0 ? (keys + s->chunk - 1) / s->chunk : 1;
}

// The tensor-core kernel: one CTA an SM.  A step (one key tile of 256 rows, or
// two of 128 rows) takes about 1.9 us, an item 4 us beside its steps, the join
// 3 us and the partial results' way through memory.  The number of ranges is
// the one of least
//   waves x longest item + join
// (16 heads x 4096 rows x 16,384 keys, 256 items: whole 507 us, halves 560 us;
// 8 units of 256 rows x 32,768 keys and their own keys: ranges of 12, 16, 24
// tiles 105, 93, 100 us, the rule's 94 us.)
void split_dense(Source* s, const int* keys, int n, int D, bool must_join) {
  int longest = 0;
  for (int i = 0; i < n; ++i)
    if (!s[i].few && (keys[i] + 127) / 128 > longest) longest = (keys[i] + 127) / 128;
  int best = longest > 0 ? longest : 1;
  double best_cost = 1e30;
  const int most = longest < 128 ? longest : 128;
  for (int k = 1; k <= most; ++k) {
    const int c = (longest + k - 1) / k;
    double work = 0, top = 0, bytes = 0, items = 0;
    for (int i = 0; i < n; ++i) {
      if (s[i].few) continue;
      const int nk = (keys[i] + 127) / 128;
      const int sp = nk ? (nk + c - 1) / c : 1;
      const double per = static_cast<double>(s[i].units) * s[i].tiles * sp;
      const int len = nk < c ? nk : c;
      const double t = 1.9 * (s[i].dual ? (len + 1) / 2 : len) + 4.0;
      work += per * t;
      items += per;
      top = t > top ? t : top;
      bytes += static_cast<double>(s[i].units) * s[i].rows * sp * D * 8.0;
    }
    if (items > 2.0e9) break;
    double cost = static_cast<double>(static_cast<int64_t>(work / (kSMs * top) + 0.999)) * top;
    if (k > 1 || must_join) cost += 3.0 + bytes / 5.0e6;
    if (cost < best_cost) best_cost = cost, best = c;
  }
  for (int i = 0; i < n; ++i) {
    if (s[i].few) continue;
    const int nk = (keys[i] + 127) / 128;
    s[i].chunk = best;
    s[i].splits = nk ? (nk + best - 1) / best : 1;
  }
}

DensePlan plan_of(const DenseCall& c) {
  DensePlan pl{};
  bool dense = false;
  for (int i = 0; i < c.n; ++i) {
    pl.s[i] = source_of(c, i);
    if (pl.s[i].few)
      split_few(&pl.s[i], c.keys[i]);
    else
      dense = true;
  }
  if (dense) split_dense(pl.s, c.keys, c.n, c.D, c.n > 1);
  // The second source's kernel joins the first one's partial results with its own
  // where it has all of a row's keys and its warps have at most four each to join
  // (64 sequences behind 32,768 keys, 18 ranges: 73 us against 80 with a third
  // kernel; one sequence, whose 8 CTAs would join 148 ranges: 45 against 41).
  pl.fused = c.n > 1 && pl.s[1].few && pl.s[1].splits == 1 && pl.s[0].splits <= 32;
  pl.join = !pl.fused && (c.n > 1 || pl.s[0].splits > 1);
  size_t off = 0;
  for (int i = 0; i < c.n; ++i) {
    if (!pl.partial(i)) continue;
    const size_t rows = static_cast<size_t>(pl.s[i].units) * pl.s[i].rows * pl.s[i].splits;
    pl.s[i].o_off = off;
    off += round256(rows * c.D * sizeof(float));
    pl.s[i].lse_off = off;
    off += round256(rows * sizeof(float));
  }
  pl.total = off;
  return pl;
}

cudaLaunchConfig_t config(unsigned grid, int threads, int smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

float* part_o(const Source& s, uint8_t* ws) { return reinterpret_cast<float*>(ws + s.o_off); }
float* part_lse(const Source& s, uint8_t* ws) { return reinterpret_cast<float*>(ws + s.lse_off); }

int launch_few(const DenseCall& c, const DensePlan& pl, int i, bool late, uint8_t* ws, cudaStream_t st) {
  const Source& s = pl.s[i];
  FewParams p{};
  p.units = s.units, p.rows = s.rows, p.splits = s.splits, p.chunk = s.chunk, p.keys = c.keys[i];
  p.shared_kv = c.shared_kv[i], p.causal = c.causal[i];
  p.H = c.H, p.Hk = c.Hk, p.G = c.H / c.Hk, p.M = c.M;
  p.lens = c.lens[i], p.lens_i64 = c.lens_dtype == BSA_INDEX_I64;
  p.q = static_cast<const uint8_t*>(c.q.data);
  p.k = static_cast<const uint8_t*>(c.k[i].data);
  p.v = static_cast<const uint8_t*>(c.v[i].data);
  p.qs_b = c.q.stride_b, p.qs_h = c.q.stride_h, p.qs_n = c.q.stride_n;
  p.ks_b = c.k[i].stride_b, p.ks_h = c.k[i].stride_h, p.ks_n = c.k[i].stride_n;
  p.vs_b = c.v[i].stride_b, p.vs_h = c.v[i].stride_h, p.vs_n = c.v[i].stride_n;
  p.o = static_cast<uint8_t*>(c.o.data);
  p.os_b = c.o.stride_b, p.os_h = c.o.stride_h, p.os_n = c.o.stride_n;
  p.lse = c.lse;
  p.o_rest = static_cast<uint8_t*>(c.o_rest);
  if (pl.partial(i)) p.part_o = part_o(s, ws), p.part_lse = part_lse(s, ws);
  if (pl.fused && i == 1) {
    const Source& other = pl.s[0];
    p.other_o = part_o(other, ws), p.other_lse = part_lse(other, ws);
    p.other_splits = other.splits, p.other_rows = other.rows;
  }
  p.scale_log2 = c.sm_scale * 1.4426950408889634f;
  p.late = late;
  p.err = c.err;
  return launch_attn_few(p, c.D, c.dtype == BSA_DTYPE_BF16, st);
}

template <int D, bool BF16>
int launch_dense(const DenseCall& c, const DensePlan& pl, uint8_t* ws, cudaStream_t st) {
  using C = DenseCfg<D>;
  auto kern = attn_dense_kernel<D, BF16>;
  static std::atomic<int> checked{0};  // 1 ok, 2 too few registers
  if (!checked.load(std::memory_order_relaxed)) {
    cudaFuncAttributes fa;
    BSA_CUDA_CHECK(cudaFuncGetAttributes(&fa, kern));
    // with fewer registers at launch the split's increases would never be granted
    checked.store(fa.numRegs * kThreadsD >= 128 * kRegsSplitD ? 1 : 2);
  }
  if (checked.load(std::memory_order_relaxed) != 1) return BSA_ERR_UNSUPPORTED;
  int r;
  if ((r = opt_in_smem(reinterpret_cast<const void*>(kern), C::SMEM))) return r;
  DenseParams p{};
  CUtensorMap mq[2] = {}, mk[2] = {}, mv[2] = {};
  for (int i = 0; i < c.n; ++i) {
    const Source& s = pl.s[i];
    if (s.few) continue;
    const int j = p.nparts++;
    DensePart& pt = p.part[j];
    pt.rows = s.rows, pt.seqs = s.seqs;
    pt.mt = s.mt, pt.gh = s.gh, pt.nb = s.nb, pt.nm = s.nm, pt.ng = s.ng, pt.subs = s.subs;
    pt.tiles = s.tiles;
    pt.dual = s.dual;
    pt.splits = s.splits;
    pt.chunk = s.chunk;
    pt.keys = c.keys[i];
    pt.items = s.units * s.tiles * s.splits;
    pt.shared_kv = c.shared_kv[i];
    pt.causal = c.causal[i];
    pt.lens = c.lens[i];
    if (pl.partial(i)) pt.part_o = part_o(s, ws), pt.part_lse = part_lse(s, ws);
    if ((r = map_of(&mq[j], c.q, c.B, c.H, c.M, D, BF16, &pt.qb_mul, s.mt, s.gh, s.nb))) return r;
    if (!c.keys[i]) continue;  // no key tile is ever loaded
    const int kb = c.shared_kv[i] ? 1 : c.B;
    if ((r = map_of(&mk[j], c.k[i], kb, c.Hk, c.keys[i], D, BF16, &pt.kb_mul))) return r;
    if ((r = map_of(&mv[j], c.v[i], kb, c.Hk, c.keys[i], D, BF16, &pt.vb_mul))) return r;
  }
  p.B = c.B, p.H = c.H, p.Hk = c.Hk, p.G = c.H / c.Hk, p.M = c.M;
  p.lens_i64 = c.lens_dtype == BSA_INDEX_I64;
  p.o = static_cast<uint8_t*>(c.o.data);
  p.os_b = c.o.stride_b, p.os_h = c.o.stride_h, p.os_n = c.o.stride_n;
  p.lse = c.lse;
  p.o_rest = static_cast<uint8_t*>(c.o_rest);
  p.scale_log2 = c.sm_scale * 1.4426950408889634f;
  p.err = c.err;
  p.wait_ns = kWaitNs;
  const int total = p.part[0].items + p.part[1].items;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(total < kSMs ? total : kSMs, kThreadsD, C::SMEM, st, attr);
  BSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, mq[0], mk[0], mv[0], mq[1], mk[1], mv[1], p));
  return BSA_OK;
}

template <int D, bool BF16>
int launch_all(const DenseCall& c, const DensePlan& pl, uint8_t* ws, cudaStream_t st) {
  int r;
  bool dense = false;
  for (int i = 0; i < c.n; ++i) dense = dense || !pl.s[i].few;
  if (dense && (r = launch_dense<D, BF16>(c, pl, ws, st))) return r;
  bool late = dense;
  for (int i = 0; i < c.n; ++i) {
    if (!pl.s[i].few) continue;
    if ((r = launch_few(c, pl, i, late, ws, st))) return r;
    late = true;
  }
  if (!pl.join) return BSA_OK;
  JoinParams j{};  // (an absent second source has no partial results)
  for (int i = 0; i < c.n; ++i) {
    j.src[i].o = part_o(pl.s[i], ws);
    j.src[i].lse = part_lse(pl.s[i], ws);
    j.src[i].splits = pl.s[i].splits;
    j.src[i].rows = pl.s[i].rows;
    j.src[i].shared_kv = c.shared_kv[i];
  }
  j.B = c.B, j.H = c.H, j.Hk = c.Hk, j.G = c.H / c.Hk, j.M = c.M;
  j.o = static_cast<uint8_t*>(c.o.data);
  j.os_b = c.o.stride_b, j.os_h = c.o.stride_h, j.os_n = c.o.stride_n;
  j.lse = c.lse;
  j.o_rest = static_cast<uint8_t*>(c.o_rest);
  const int64_t rows = static_cast<int64_t>(c.B) * c.H * c.M;
  cudaLaunchAttribute attr[1];
  if (pl.s[0].splits + (c.n > 1 ? pl.s[1].splits : 0) >= 8) {
    const cudaLaunchConfig_t cfg = config(static_cast<unsigned>(rows), 256, 0, st, attr);
    BSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, attn_join_kernel<D, BF16, 8>, j));
  } else {
    const cudaLaunchConfig_t cfg = config(static_cast<unsigned>((rows + 7) / 8), 256, 0, st, attr);
    BSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, attn_join_kernel<D, BF16, 1>, j));
  }
  return BSA_OK;
}

// Checks common to both operators; the sources' keys may be zero.
int validate(const DenseCall& c) {
  if (c.B <= 0 || c.H <= 0 || c.Hk <= 0 || c.M <= 0 || c.D <= 0) return BSA_ERR_INVALID_ARG;
  if (c.dtype != BSA_DTYPE_F16 && c.dtype != BSA_DTYPE_BF16) return BSA_ERR_DTYPE;
  if (c.H % c.Hk) return BSA_ERR_SHAPE;
  if (c.D != 64 && c.D != 128) return BSA_ERR_UNSUPPORTED;
  if (!(c.sm_scale > 0.f) || !(c.sm_scale < INFINITY)) return BSA_ERR_UNSUPPORTED;
  if (!c.q.data || !c.o.data) return BSA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(c.o_rest) % 16) return BSA_ERR_ALIGNMENT;
  // row and item numbers are 32-bit
  if (static_cast<int64_t>(c.B) * c.H * c.M > INT32_MAX / 2) return BSA_ERR_UNSUPPORTED;
  if (!aligned(c.q, c.B, c.H, c.M) || !aligned(c.o, c.B, c.H, c.M)) return BSA_ERR_ALIGNMENT;
  for (int i = 0; i < c.n; ++i) {
    if (c.keys[i] < 0) return BSA_ERR_INVALID_ARG;
    // key numbers are 32-bit, with a range's length added
    if (c.keys[i] > INT32_MAX / 2) return BSA_ERR_UNSUPPORTED;
    if (!c.keys[i]) continue;
    if (!c.k[i].data || !c.v[i].data) return BSA_ERR_INVALID_ARG;
    const int kb = c.shared_kv[i] ? 1 : c.B;
    const bsa_tensor4d* ts[] = {&c.k[i], &c.v[i]};
    for (const bsa_tensor4d* t : ts) {
      if (t->stride_b < 0 || t->stride_h < 0 || t->stride_n < 0) return BSA_ERR_INVALID_ARG;
      if (!aligned(*t, kb, c.Hk, c.keys[i])) return BSA_ERR_ALIGNMENT;
    }
    if (c.lens[i] && c.lens_dtype != BSA_INDEX_I32 && c.lens_dtype != BSA_INDEX_I64) return BSA_ERR_DTYPE;
  }
  return BSA_OK;
}

DenseCall call_of(const bsa_cross_args* a) {
  DenseCall c{};
  c.B = a->B, c.H = a->H, c.Hk = a->Hk, c.M = a->M, c.D = a->D, c.dtype = a->dtype;
  c.q = a->q, c.o = a->o;
  c.n = 1;
  c.k[0] = a->k, c.v[0] = a->v, c.keys[0] = a->N;
  c.lens[0] = a->k_lens, c.lens_dtype = a->lens_dtype;
  c.sm_scale = a->sm_scale, c.lse = a->lse, c.o_rest = a->o_rest, c.err = a->err_flag;
  return c;
}

DenseCall call_of(const bsa_prefix_args* a) {
  DenseCall c{};
  c.B = a->B, c.H = a->H, c.Hk = a->Hk, c.M = a->T, c.D = a->D, c.dtype = a->dtype;
  c.q = a->q, c.o = a->o;
  c.n = 2;
  c.k[0] = a->k_prefix, c.v[0] = a->v_prefix, c.keys[0] = a->P, c.shared_kv[0] = true;
  c.k[1] = a->k, c.v[1] = a->v, c.keys[1] = a->C, c.lens[1] = a->lens, c.causal[1] = a->T > 1;
  c.lens_dtype = a->lens_dtype;
  c.sm_scale = a->sm_scale, c.lse = a->lse, c.err = a->err_flag;
  return c;
}

// (the caller checked that `ws` holds plan_of(c).total bytes)
int run(const DenseCall& c, void* ws, cudaStream_t st) {
  if (reinterpret_cast<uintptr_t>(ws) % 16) return BSA_ERR_ALIGNMENT;
  const DensePlan pl = plan_of(c);
  uint8_t* w = static_cast<uint8_t*>(ws);
  const bool bf = c.dtype == BSA_DTYPE_BF16;
  if (c.D == 128) return bf ? launch_all<128, true>(c, pl, w, st) : launch_all<128, false>(c, pl, w, st);
  return bf ? launch_all<64, true>(c, pl, w, st) : launch_all<64, false>(c, pl, w, st);
}

}  // namespace

int cross_validate(const bsa_cross_args* a) { return a ? validate(call_of(a)) : BSA_ERR_INVALID_ARG; }
size_t cross_workspace(const bsa_cross_args* a) { return plan_of(call_of(a)).total; }
int launch_cross(const bsa_cross_args* a, void* ws, cudaStream_t st) { return run(call_of(a), ws, st); }
int prefix_validate(const bsa_prefix_args* a) { return a ? validate(call_of(a)) : BSA_ERR_INVALID_ARG; }
size_t prefix_workspace(const bsa_prefix_args* a) { return plan_of(call_of(a)).total; }
int launch_prefix(const bsa_prefix_args* a, void* ws, cudaStream_t st) { return run(call_of(a), ws, st); }

}  // namespace bsa
