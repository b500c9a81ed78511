// logits.cu -- what stands between logits and the next token: penalties for repeated tokens, biases, grammar masks, and
// the greedy choice.
//
// Bound by HBM: each logit is read once and written once.  The history of a row is counted in shared memory, per segment
// of the vocabulary: a block owns one segment of one row, requests its logits first, then walks the row's history (a few
// kilobytes that stay in L2) and counts the tokens of its segment while the logits arrive.  No counts in global memory,
// nothing to clear, and integer atomics, so results do not depend on their order.
#include <algorithm>
#include <climits>

#include "llm_ops.cuh"

namespace simp {

struct LogitsArgs {
  const void* in;
  void* out;
  int64_t stride;
  int vocab, rows;
  simp_logits_rules r;
  int32_t* best;
  unsigned long long* key;   // per row: largest (ordered value, ~index); 0 between calls
  int* arrived;              // per row; 0 between calls
  int* status;
};

constexpr int LG_THREADS = 256;

// Larger floats have larger keys, equal ones the larger key at the lower index.  Never 0, and only asked for values above
// -infinity.
__device__ __forceinline__ unsigned long long logit_key(float v, int i) {
  uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);   // -0 and 0 are equal
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (static_cast<unsigned long long>(b) << 32) | (0xffffffffu - uint32_t(i));
}

// U: 16-byte vectors per thread; a block owns LG_THREADS * U * VEC tokens.
template <typename T, int U>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
  constexpr int VEC = 16 / sizeof(T), SEG = LG_THREADS * U * VEC;
  extern __shared__ __align__(16) int lg_smem[];
  __shared__ unsigned long long wbest[LG_THREADS / 32];
  const int row = blockIdx.y;
  const T* in = static_cast<const T*>(a.in) + row * a.stride;
  T* out = static_cast<T*>(a.out) + row * a.stride;
  // segments start on 16-byte boundaries of the input: token `base` may lie before the row, by less than a vector
  const int mis = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const int base = int(blockIdx.x) * SEG - mis;
  const bool st16 = (reinterpret_cast<uintptr_t>(out + base) & 15) == 0;
  T x[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v0 = base + (u * LG_THREADS + threadIdx.x) * VEC;
    if (v0 >= 0 && v0 + VEC <= a.vocab) {
      *reinterpret_cast<uint4*>(x[u]) = *reinterpret_cast<const uint4*>(in + v0);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (v0 + j >= 0 && v0 + j < a.vocab) x[u][j] = in[v0 + j];
    }
  }
  int* count = lg_smem;
  int* bias = lg_smem + (a.r.tokens ? SEG : 0);
  if (a.r.tokens || a.r.bias_tokens) {
    if (a.r.tokens)
      for (int i = 4 * threadIdx.x; i < SEG; i += 4 * LG_THREADS) *reinterpret_cast<int4*>(count + i) = make_int4(0, 0, 0, 0);
    if (a.r.bias_tokens)
      for (int i = 4 * threadIdx.x; i < SEG; i += 4 * LG_THREADS) *reinterpret_cast<int4*>(bias + i) = make_int4(-1, -1, -1, -1);
    __syncthreads();
    int b, e;
    const int first = max(base, 0), last = min(base + SEG, a.vocab);
    if (a.r.tokens && seq_range(a.r.token_offsets, row, a.r.n_tokens, a.status, b, e))
      for (int i = b + int(threadIdx.x); i < e; i += LG_THREADS) {
        const int id = __ldg(a.r.tokens + i);
        if (id >= first && id < last) atomicAdd(count + (id - base), 1);
      }
    if (a.r.bias_tokens && seq_range(a.r.bias_offsets, row, a.r.n_bias, a.status, b, e))
      for (int i = b + threadIdx.x; i < e; i += LG_THREADS) {
        const int id = __ldg(a.r.bias_tokens + i);
        if (id >= first && id < last) atomicMax(bias + (id - base), i);   // the last entry wins
      }
    __syncthreads();
  }
  const float rep = a.r.repetition ? __ldg(a.r.repetition + row) : 1.0f;
  const float freq = a.r.frequency ? __ldg(a.r.frequency + row) : 0.0f;
  const float pres = a.r.presence ? __ldg(a.r.presence + row) : 0.0f;
  const uint32_t* mask = a.r.allowed ? a.r.allowed + row * a.r.allowed_stride : nullptr;
  float top_v = -INFINITY;   // a thread's tokens ascend, so the first of equals stays
  int top_i = -1;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int l0 = (u * LG_THREADS + threadIdx.x) * VEC, v0 = base + l0;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = to_f32(x[u][j]);
    if (a.r.tokens) {
      int n[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j += 4) *reinterpret_cast<int4*>(n + j) = *reinterpret_cast<const int4*>(count + l0 + j);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (n[j] > 0) {   // separate roundings, so that the result does not hang on a contraction
          f[j] = f[j] > 0.0f ? __fdiv_rn(f[j], rep) : __fmul_rn(f[j], rep);
          f[j] = __fsub_rn(f[j], __fadd_rn(__fmul_rn(freq, float(n[j])), pres));
        }
    }
    if (a.r.bias_tokens) {
      int e[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j += 4) *reinterpret_cast<int4*>(e + j) = *reinterpret_cast<const int4*>(bias + l0 + j);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e[j] >= 0) f[j] = __fadd_rn(f[j], __ldg(a.r.bias_values + e[j]));
    }
    const bool whole = v0 >= 0 && v0 + VEC <= a.vocab;
    if (mask) {
      // a vector's bits lie in one word or two: 64 bits from the word of its first token on
      const int w0 = max(v0, 0) >> 5, w1 = min(w0 + 1, (a.vocab - 1) >> 5);
      if (v0 < a.vocab) {
        const uint32_t lo = __ldg(mask + w0), hi = __ldg(mask + w1);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int at = v0 + j - 32 * w0;   // negative before the row: that token is not written
          const uint32_t bit = at < 32 ? lo >> (at & 31) : hi >> (at & 31);
          if (!(bit & 1u)) f[j] = -INFINITY;
        }
      }
    }
    T y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      y[j] = from_f32<T>(f[j]);
      const float w = to_f32(y[j]);
      if (w > top_v && (whole || (v0 + j >= 0 && v0 + j < a.vocab))) {
        top_v = w;
        top_i = v0 + j;
      }
    }
    if (st16 && whole) {
      *reinterpret_cast<uint4*>(out + v0) = *reinterpret_cast<const uint4*>(y);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (v0 + j >= 0 && v0 + j < a.vocab) out[v0 + j] = y[j];
    }
  }
  if (!a.best) return;
  unsigned long long top = top_i >= 0 ? logit_key(top_v, top_i) : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, top, o);
    top = k > top ? k : top;
  }
  if ((threadIdx.x & 31) == 0) wbest[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < LG_THREADS / 32; ++w) top = wbest[w] > top ? wbest[w] : top;
  if (gridDim.x > 1) {
    if (top) atomicMax(a.key + row, top);
    __threadfence();
    if (atomicAdd(a.arrived + row, 1) != int(gridDim.x) - 1) return;
    __threadfence();
    top = atomicExch(a.key + row, 0ull);
    a.arrived[row] = 0;
  }
  a.best[row] = top ? int(0xffffffffu - uint32_t(top)) : -1;
}

template <typename T>
static int logits_launch(LogitsArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  // segments of 4 vectors per thread where that still gives every SM a few blocks, else of one
  const int64_t span = int64_t(a.vocab) + VEC - 1;
  const bool wide = cdiv(span, LG_THREADS * VEC * 4) * a.rows >= 2 * ctx().sm_count;
  const int seg = LG_THREADS * VEC * (wide ? 4 : 1);
  const dim3 grid(unsigned(cdiv(span, seg)), unsigned(a.rows));
  if (a.best && grid.x > 1) {
    // keys first, so that both arrays keep their alignment
    uint8_t* p = static_cast<uint8_t*>(scratch(size_t(65536) * 12, SCRATCH_ARGMAX, true));
    if (!p) return scratch_failed("logits_process");
    a.key = reinterpret_cast<unsigned long long*>(p);
    a.arrived = reinterpret_cast<int*>(p + size_t(65536) * 8);
  }
  const size_t smem = size_t(seg) * 4 * ((a.r.tokens ? 1 : 0) + (a.r.bias_tokens ? 1 : 0));
  auto kern = wide ? logits_kernel<T, 4> : logits_kernel<T, 1>;
  if (smem > 48 * 1024) SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  kern<<<grid, LG_THREADS, smem, ctx().stream>>>(a);
  SIMP_LAUNCH_CHECK();
  return SIMP_OK;
}

}  // namespace simp

using namespace simp;

SIMP_API int simp_gpu_logits_process(const void* logits_dev, void* out_dev, int64_t rows, int64_t vocab, int64_t row_stride,
                                     const simp_logits_rules* rules, int32_t* argmax_dev, int dtype) {
  SIMP_REQUIRE(dtype_ok(dtype), SIMP_ERR_ARG, "logits_process: unknown dtype %d", dtype);
  SIMP_REQUIRE(rows >= 0 && vocab >= 0, SIMP_ERR_ARG, "logits_process: negative size");
  SIMP_REQUIRE(rules, SIMP_ERR_ARG, "logits_process: rules is null");
  if (rows == 0) return SIMP_OK;
  SIMP_REQUIRE(vocab >= 1 && vocab <= (1 << 30) && rows <= 65535, SIMP_ERR_SHAPE, "logits_process: %lld rows of %lld (at most 65535 rows of 1 .. 2^30 tokens)",
               (long long)rows, (long long)vocab);
  SIMP_REQUIRE(logits_dev && out_dev, SIMP_ERR_ARG, "logits_process: null pointer");
  if (row_stride == 0) row_stride = vocab;
  SIMP_REQUIRE(row_stride >= vocab, SIMP_ERR_SHAPE, "logits_process: row_stride %lld is shorter than a row", (long long)row_stride);
  SIMP_REQUIRE(aligned_to(logits_dev, dtype_size(dtype)) && aligned_to(out_dev, dtype_size(dtype)), SIMP_ERR_ARG, "logits_process: misaligned pointer");
  const simp_logits_rules& r = *rules;
  SIMP_REQUIRE((r.tokens != nullptr) == (r.token_offsets != nullptr), SIMP_ERR_ARG, "logits_process: tokens and token_offsets go together");
  SIMP_REQUIRE(r.tokens || !(r.repetition || r.frequency || r.presence), SIMP_ERR_ARG, "logits_process: penalties need tokens");
  SIMP_REQUIRE((r.bias_tokens != nullptr) == (r.bias_values != nullptr) && (r.bias_tokens != nullptr) == (r.bias_offsets != nullptr),
               SIMP_ERR_ARG, "logits_process: bias_tokens, bias_values and bias_offsets go together");
  SIMP_REQUIRE(r.n_tokens >= 0 && r.n_tokens <= INT_MAX && r.n_bias >= 0 && r.n_bias <= INT_MAX, SIMP_ERR_ARG, "logits_process: bad length of a list");
  SIMP_REQUIRE(!r.allowed || r.allowed_stride == 0 || r.allowed_stride >= (vocab + 31) / 32, SIMP_ERR_SHAPE,
               "logits_process: allowed_stride %lld words for %lld tokens", (long long)r.allowed_stride, (long long)vocab);
  if (int rc = ensure_ready()) return rc;
  DeviceScope dev;
  LogitsArgs a{};
  a.in = logits_dev;
  a.out = out_dev;
  a.stride = row_stride;
  a.vocab = int(vocab);
  a.rows = int(rows);
  a.r = r;
  a.best = argmax_dev;
  a.status = ctx().dev_status;
  if (dtype == SIMP_DTYPE_F32) return logits_launch<float>(a);
  if (dtype == SIMP_DTYPE_F16) return logits_launch<__half>(a);
  return logits_launch<__nv_bfloat16>(a);
}
