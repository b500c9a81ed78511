// llm_ops.cuh -- what the batched serving ops (prompt attention, 8-bit cache, logits) share: element types, packed
// sequences, reporting of bad device-side indices.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace simp {

constexpr int SCRATCH_KV8_PART = 16;   // partial results of a split cache attention
constexpr int SCRATCH_KV8_COUNT = 17;  // its arrival counters (zero between calls)
constexpr int SCRATCH_ARGMAX = 18;     // row keys and arrival counters of logits_process (zero between calls)

constexpr int SCRATCH_ATTN_PACK = 19;  // padded or split copies of q, k, v

constexpr int STATUS_BAD_BLOCK = 3, STATUS_BAD_RANGE = 4;

// The calling thread's current device is the library's for the duration of a call (a host thread that never set one
// starts on device 0, and a stream takes launches only from its own device).
struct DeviceScope {
  int was = -1;
  DeviceScope() {
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != ctx().device && cudaSetDevice(ctx().device) == cudaSuccess) was = cur;
  }
  ~DeviceScope() {
    if (was >= 0) cudaSetDevice(was);
  }
};

inline bool dtype_ok(int dtype) { return dtype == SIMP_DTYPE_F32 || dtype == SIMP_DTYPE_F16 || dtype == SIMP_DTYPE_BF16; }
inline size_t dtype_size(int dtype) { return dtype == SIMP_DTYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of an array whose type is known at run time only (prologues and epilogues).
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == SIMP_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SIMP_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int dtype) {
  if (dtype == SIMP_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == SIMP_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void report_status(int* status, int code, int detail) {
  if (atomicCAS(status, 0, code) == 0) status[1] = detail;
}

// Rows [begin, end) of sequence s by an array of offsets; false (and reported) unless 0 <= begin <= end <= total.
__device__ __forceinline__ bool seq_range(const int32_t* off, int s, int64_t total, int* status, int& begin, int& end) {
  begin = __ldg(off + s);
  end = __ldg(off + s + 1);
  if (begin >= 0 && begin <= end && int64_t(end) <= total) return true;
  report_status(status, STATUS_BAD_RANGE, s);
  begin = end = 0;
  return false;
}

// Finds the sequence and the place in it of work unit u when sequence s has count(s) units (called by a whole warp;
// every lane gets the result).  32 sequences are looked at together, so a batch of 64 costs two rounds.  False: u lies
// behind the last unit.  With `weight`, up to 32 sequences are taken in the order of falling weight: blocks start in the
// order of their numbers, and long work that starts last ends alone.
struct NoWeight {};
template <typename Count, typename Weight = NoWeight>
__device__ __forceinline__ bool find_unit(int64_t u, int n_seqs, Count count, int& seq, int& place, Weight weight = Weight()) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    int c = s0 + lane < n_seqs ? count(s0 + lane) : 0, which = lane;
    if constexpr (!std::is_same_v<Weight, NoWeight>) {
      if (n_seqs > 1 && n_seqs <= 32) {
        // weight and lane in one word, sorted by comparators at distances k / 2, k / 4 .. 1 of runs of k = 2, 4 .. 32 (Batcher's
        // bitonic network): falling weight, equal ones by their numbers, lanes behind the last sequence at the end
        uint32_t key = (lane < n_seqs ? uint32_t(min(max(weight(lane), 0) + 1, (1 << 27) - 1)) << 5 : 0u) | uint32_t(31 - lane);
        const uint32_t head = __shfl_sync(0xffffffffu, key, 0) >> 5;
        if (!__all_sync(0xffffffffu, lane >= n_seqs || key >> 5 == head)) {
#pragma unroll
          for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
            for (int d = k >> 1; d > 0; d >>= 1) {
              const uint32_t o = __shfl_xor_sync(0xffffffffu, key, d);
              const bool larger = ((lane & d) == 0) == ((lane & k) == 0);
              key = larger ? max(key, o) : min(key, o);
            }
          which = 31 - int(key & 31u);
          c = __shfl_sync(0xffffffffu, c, which);
        }
      }
    }
    int64_t upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const unsigned in = __ballot_sync(0xffffffffu, u < upto);
    if (in) {
      const int l = __ffs(in) - 1;
      seq = s0 + __shfl_sync(0xffffffffu, which, l);
      place = int(u - __shfl_sync(0xffffffffu, upto - c, l));
      return true;
    }
    u -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
#endif

}  // namespace simp
