// What the kernels of attention over contiguous key ranges share
// (attn_dense.cu, attn_few.cu, attn_dense_bwd.cu).
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "internal.h"

namespace bsa {

// The kernel for at most kFewRows rows of a unit (attn_few.cu).  Row r of a
// unit is query (sequence, head, token): r = (seq * G + g) * M + m.
constexpr int kFewRows = 16;
struct FewParams {
  int units;      // shared_kv: Hk, else B * Hk
  int rows;       // of a unit
  int splits;     // key ranges
  int chunk;      // keys of a range
  int keys;       // keys the tensors hold
  int shared_kv;  // the unit's keys serve every sequence
  int causal;     // query m of M sees keys below len - (M - 1 - m)
  int H, Hk, G, M;
  const void* lens;  // [B] valid keys, or null
  int lens_i64;
  const uint8_t *q, *k, *v;
  int64_t qs_b, qs_h, qs_n, ks_b, ks_h, ks_n, vs_b, vs_h, vs_n;
  uint8_t* o;
  int64_t os_b, os_h, os_n;
  uint8_t* o_rest;  // optional, laid out as o: what rounding left
  float* lse;
  float* part_o;  // partial results, or null: this is the whole result
  float* part_lse;
  // Partial results of the same rows from the other source's kernel of the call,
  // to be joined here (null: none): row b G M + r of shared unit hk.
  const float* other_o;
  const float* other_lse;
  int other_splits, other_rows;
  float scale_log2;
  int late;       // launched behind the other source's kernel of the same call: see attn_few.cu
  int32_t* err;
};
int launch_attn_few(const FewParams& p, int D, bool bf16, cudaStream_t st);

// A tensor map's batch dimension of 1 where the batch shares one copy.
inline int map_of(CUtensorMap* m, bsa_tensor4d t, int B, int H, int N, int D, bool bf16, int* mul, int rows = 128, int heads = 1,
           int batch = 1) {
  const bool one = B == 1 || t.stride_b == 0;
  *mul = one ? 0 : 1;
  // a dimension of length 1 has no stride of its own
  if (one) t.stride_b = 8;
  if (H == 1) t.stride_h = 8;
  if (N == 1) t.stride_n = 8;
  return make_tensor_map_4d(m, t, one ? 1 : B, H, N, D, bf16, rows, heads, batch);
}

// Rows that 16-byte accesses and tensor maps can take.
inline bool aligned(const bsa_tensor4d& t, int B, int H, int N) {
  return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && (B == 1 || t.stride_b * 2 % 16 == 0) &&
         (H == 1 || t.stride_h * 2 % 16 == 0) && (N == 1 || t.stride_n * 2 % 16 == 0);
}

// The dynamic shared memory opt-in of a kernel, once per device.
inline int opt_in_smem(const void* kern, int bytes) {
  if (bytes <= 48 * 1024) return BSA_OK;
  constexpr int kSlots = 32;
  static std::atomic<const void*> done[64][kSlots] = {};
  int dev = 0;
  BSA_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return BSA_ERR_DEVICE;
  for (int i = 0; i < kSlots; ++i) {
    const void* k = done[dev][i].load(std::memory_order_acquire);
    if (k == kern) return BSA_OK;
    if (k) continue;
    BSA_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev][i].compare_exchange_strong(k, kern);
    return BSA_OK;
  }
  BSA_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return BSA_OK;
}

}  // namespace bsa
