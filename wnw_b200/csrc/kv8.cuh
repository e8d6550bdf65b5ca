// The 8-bit paged cache's record layout and code conversions, shared by its
// append and its decode attention.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace wnw {

constexpr int kKv8Block = WNW_KV8_BLOCK;

template <int D>
struct Kv8Rec {
  static constexpr int kCodes = 2 * kKv8Block * D;        // keys, then values
  static constexpr int kUsed = kCodes + 16;               // + the two scales (16-byte copies)
  static constexpr int64_t kStride = kCodes + WNW_KV8_PAD;
};

// largest magnitude of a code
template <int CODE>
__host__ __device__ constexpr float kv8_top() {
  return CODE == WNW_KV8_E4M3 ? 448.f : 127.f;
}

// Once a device: lets a kernel take `bytes` of dynamic shared memory
// (`configured`: a bit a device, of the kernel's own).
template <typename K>
wnw_status raise_smem_limit(std::atomic<uint64_t>& configured, K kernel, int bytes) {
  int dev = 0;
  WNW_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (configured.load(std::memory_order_acquire) & bit) return WNW_OK;
  WNW_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  configured.fetch_or(bit, std::memory_order_release);
  return WNW_OK;
}

inline wnw_status check_kv8_store(const wnw_kv8_store& s) {
  WNW_CHECK_ARG(s.dtype == WNW_BF16 || s.dtype == WNW_F16, "the 8-bit cache serves bf16 and fp16 models (dtype %d)",
                s.dtype);
  WNW_CHECK_ARG(s.head_dim == 64 || s.head_dim == 128, "head_dim %d not compiled (64, 128)", s.head_dim);
  WNW_CHECK_ARG(s.code == WNW_KV8_E4M3 || s.code == WNW_KV8_INT8, "unknown code %d", s.code);
  WNW_CHECK_ARG(s.num_segs > 0 && s.num_pages >= 0 && s.max_pages >= 0, "bad segment or page counts");
  WNW_CHECK_ARG(s.page_blocks >= 1 && s.page_blocks <= 64 && (s.page_blocks & (s.page_blocks - 1)) == 0,
                "page_blocks %d: a power of two up to 64", s.page_blocks);
  WNW_CHECK_ARG(s.num_pages < (int64_t(1) << 31) && s.num_pages * s.page_blocks < (int64_t(1) << 31),
                "2^31 blocks or more");
  WNW_CHECK_ARG(int64_t(s.max_pages) * s.page_blocks * kKv8Block < (int64_t(1) << 31), "2^31 tokens a segment or more");
  WNW_CHECK_ARG((s.pool || s.num_pages == 0) && (s.page_table || s.max_pages == 0) && s.tail_k && s.tail_v && s.err,
                "null pointer argument");
  WNW_CHECK_ARG(aligned16(s.pool) && aligned16(s.tail_k) && aligned16(s.tail_v),
                "pool and tails must be 16-byte aligned");
  return WNW_OK;
}

}  // namespace wnw
