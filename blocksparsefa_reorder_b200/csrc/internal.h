// Launchers shared between the translation units of the library.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/bsattn_b200.h"

namespace bsa {

// Element size in bytes of a bsa_dtype (0 when invalid).
inline int dtype_bytes(int dt) {
  return dt == BSA_DTYPE_F32 ? 4 : (dt == BSA_DTYPE_F16 || dt == BSA_DTYPE_BF16) ? 2 : 0;
}

inline int tiles_per_row(int nb, int block) { return (nb * block + 127) / 128; }

// preprocess.cu
int launch_plan_count(const uint8_t* mask, int64_t sb, int64_t sh, int64_t srow, int mask_b, int mask_h, int nb,
                      int block, int32_t* counts, cudaStream_t st);
int launch_plan_scan(const int32_t* counts, int64_t n, int32_t* tile_ptr, cudaStream_t st);
int launch_plan_fill(const uint8_t* mask, int64_t sb, int64_t sh, int64_t srow, int mask_b, int mask_h, int nb,
                     int block, const int32_t* tile_ptr, int32_t* tile_col, cudaStream_t st);
// Bits of a permutation check (ceil(n / 32) words) and the check itself:
// zeroes `scratch`, then sets BSA_DEVERR_PERM_RANGE / _DUP in `err`.
size_t perm_check_bytes(int64_t n);
int launch_perm_check(const void* perm, int perm_dtype, int64_t n, void* scratch, int32_t* err, cudaStream_t st);
int launch_permute_rows(bsa_tensor4d dst, bsa_tensor4d src, int B, int H, int N, int row_elems, int elt_bytes,
                        const void* perm, int perm_dtype, int inverse, int32_t* err, cudaStream_t st);

// attn_simt.cu
int launch_attn_simt(const bsa_fwd_args* a, cudaStream_t st);
// The backward kernels (attn_bwd.cu): Delta, dQ, dK / dV; arguments validated.
int launch_attn_bwd(const bsa_bwd_args* a, cudaStream_t st);
// Delta = rowsum(dout o (o + rest)) per query row, contiguous fp32 [B, H, N] (D 64
// / 128); rest (optional, laid out as o): what o's rounding left; dout_max
// (optional): receives the largest |dout| of every bwd_delta_rows(D) rows of a group
// of G heads, [B, H / G, ceil(G N / those rows)].
int bwd_delta_rows(int D);
int launch_bwd_delta(const bsa_tensor4d& o, const void* rest, const bsa_tensor4d& dout, float* delta, int B, int H, int N, int D,
                     bool bf16, cudaStream_t st, float* dout_max = nullptr, int G = 1);

// tma_maps.cu: whether the tcgen05 path takes these arguments (bf16 / fp16,
// D 64 or 128, BLOCK 64 or 128, 16-byte-aligned rows), and the 4-D TMA map
// over a [B, H, N, D] 16-bit tensor, box 64 x rows (x heads x batch), 128-byte
// swizzle.
bool attn_tc_supported(const bsa_fwd_args* a);
int make_tensor_map_4d(CUtensorMap* m, const bsa_tensor4d& t, int B, int H, int N, int D, bool bf16, int rows,
                       int box_h = 1, int box_b = 1);

// attn_tcp.cu: the persistent tcgen05 attention forward
// q_perm (optional, bsa_index_dtype perm_dtype): gather Q rows from and
// scatter O / lse rows to q_perm[row] inside the kernel.
int launch_attn_tcp(const bsa_fwd_args* a, cudaStream_t st, const void* q_perm = nullptr,
                    int perm_dtype = BSA_INDEX_I64);
// Arms the timeout test for the next launch_attn_tcp call (see
// bsa_test_arm_wait_timeout).
int arm_test_wait_timeout(uint32_t wait_us);

// qk_norm_rope.cu: norm and rotation of query / key heads, and its gradient
// (each launcher validates its arguments).
int rope_validate(const bsa_rope_args* a, bool bwd);
int launch_rope_fwd(const bsa_rope_args* a, cudaStream_t st);
size_t rope_bwd_workspace(const bsa_rope_args* a);
int launch_rope_bwd(const bsa_rope_args* a, void* workspace, size_t bytes, cudaStream_t st);

// attn_dense.cu: attention over contiguous key ranges (arguments and workspace
// checked by the caller with the *_validate and *_workspace functions).
int cross_validate(const bsa_cross_args* a);
size_t cross_workspace(const bsa_cross_args* a);
int launch_cross(const bsa_cross_args* a, void* workspace, cudaStream_t st);
int prefix_validate(const bsa_prefix_args* a);
size_t prefix_workspace(const bsa_prefix_args* a);
int launch_prefix(const bsa_prefix_args* a, void* workspace, cudaStream_t st);
// attn_dense_bwd.cu: gradient of cross attention
int cross_bwd_validate(const bsa_cross_bwd_args* a);
int launch_cross_bwd(const bsa_cross_bwd_args* a, float* dout_max, cudaStream_t st);

}  // namespace bsa

#define BSA_CUDA_CHECK(expr)                    \
  do {                                          \
    cudaError_t e_ = (expr);                    \
    if (e_ != cudaSuccess) return BSA_ERR_CUDA; \
  } while (0)
