// Shared by the attention translation units: bounded device waits with their
// error words, and the tensor maps of (B, seq, heads, 64) bf16 tensors.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "vlak_device.cuh"
#include "vlak_internal.h"

namespace vlak {

// Device error word of the including translation unit (all of them are read by
// vlak_device_error_read). Used when a launch has no host-mapped error word
// (see host_error_word).
static __device__ int g_device_error = 0;

namespace {

// Records a failed wait where the host can see it: in the process's
// host-mapped error word when the launch has one (read without any device
// synchronization by vlak_device_error_poll, which the torch ops call on
// entry), else in the device error word.
__device__ __forceinline__ void publish_device_error(int* host_err, int code) {
  if (host_err != nullptr) {
    *reinterpret_cast<volatile int*>(host_err) = code;
    __threadfence_system();
  } else {
    atomicCAS(&g_device_error, 0, code);
  }
}

// Reads and clears the device error word of the including translation unit.
inline int take_device_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(int));
  if (e != cudaSuccess) return set_cuda_error("vlak_device_error_read", e);
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  return e == cudaSuccess ? VLAK_OK : set_cuda_error("vlak_device_error_read", e);
}

constexpr uint64_t kWaitLimitNs = 1000ull * 1000ull * 1000ull;  // 1 s per wait

// Bounded parity wait; `abort_flag` (shared) short-circuits the other
// waiters of the CTA once one of them has given up. kMode selects the probe:
// 0 try_wait with a suspend-time hint (a waiting warp yields its issue slots),
// 1 try_wait with the hardware's own time limit, 2 test_wait (pure polling,
// lowest wake-up latency, for waits on the critical hand-off path).
template <int kMode = 0>
__device__ __forceinline__ bool probe(uint64_t* bar, uint32_t parity) {
  if (kMode == 2) return mbar_test_wait(bar, parity);
  if (kMode == 1) return mbar_try_wait(bar, parity);
  return mbar_try_wait_suspend(bar, parity, 20000u);
}
template <int kMode = 0>
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity,
                                             volatile int* abort_flag,
                                             bool honour_abort = true) {
  // the elapsed time is checked every 64 probes
  if (probe<kMode>(bar, parity)) return true;
  uint64_t t0;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (uint32_t it = 1;; ++it) {
    if (probe<kMode>(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (honour_abort && *abort_flag) return false;
      uint64_t t;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t - t0 > kWaitLimitNs) {
        // reported by the CTA's thread 0 once every role has drained
        *abort_flag = 1;
        return false;
      }
    }
  }
}

// Zero rows [lo, hi) of a tile of 128-byte rows in shared memory, by a whole
// warp, before this warp's next MMA reads it (the tile's copy has completed).
__device__ __forceinline__ void clear_rows(uint8_t* tile, int lo, int hi) {
  if (lo >= hi) return;
  for (int i = lo * 8 + (threadIdx.x & 31); i < hi * 8; i += 32)
    reinterpret_cast<uint4*>(tile)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// Tensor map of dims (64, d1, d2, d3) with element strides s1..s3 and box
// (64, box1, box2, 1), rows in the 128-byte swizzle.
inline int encode_map(CUtensorMap* map, const void* base, int64_t d1, int64_t d2, int64_t d3,
               int64_t s1, int64_t s2, int64_t s3, uint32_t box1, uint32_t box2,
               const char* name) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return set_error(VLAK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  // a size-1 dimension is never stepped over; give it a harmless stride
  auto fix = [](int64_t size, int64_t stride_bytes, int64_t fallback) {
    return size == 1 ? fallback : stride_bytes;
  };
  const int64_t b1 = fix(d1, s1 * 2, 128);
  const int64_t b2 = fix(d2, s2 * 2, b1 * d1);
  const int64_t b3 = fix(d3, s3 * 2, b2 * d2);
  cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(d1), static_cast<cuuint64_t>(d2),
                        static_cast<cuuint64_t>(d3)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(b1), static_cast<cuuint64_t>(b2),
                           static_cast<cuuint64_t>(b3)};
  cuuint32_t box[4] = {64, box1, box2, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
                   box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT,
                      "fused_attention_gqa: cannot describe %s to TMA (CUresult %d); strides "
                      "must be multiples of 8 elements and the layout addressable",
                      name, static_cast<int>(r));
  return VLAK_OK;
}

}  // namespace
}  // namespace vlak
