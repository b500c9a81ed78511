// logits.cu -- what stands between logits and the next token: penalties for repeated tokens, biases, grammar masks, and
// the greedy choice.
//
// Bound by HBM: each logit is read once and written once.  A block owns a slice of one row's vocabulary.  The tokens of the
// row's history and biases are few: they are worked on first, one by one (counted in shared memory with integer atomics,
// so results do not depend on their order), while the slice's first logits are on their way; a bitmap then tells the pass
// over all logits which of them to replace.  (With the penalties in that pass its division ran for nearly every warp.)
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

// A thread has U 16-byte vectors in flight; a block works on NSUB times LG_THREADS * U * VEC tokens.
template <typename T, int U, int NSUB>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsArgs a) {
  constexpr int VEC = 16 / sizeof(T), SUB = LG_THREADS * U * VEC, SLICE = SUB * NSUB, LISTED = NSUB > 1 ? SLICE / 8 : 0;   // short slices: few entries each, and a step less to wait for
  extern __shared__ __align__(16) int lg_smem[];
  __shared__ unsigned long long wbest[LG_THREADS / 32];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const T* in = static_cast<const T*>(a.in) + row * a.stride;
  T* out = static_cast<T*>(a.out) + row * a.stride;
  // slices start on 16-byte boundaries of the input: token `base` may lie before the row, by less than a vector
  const int mis = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const int base = int(blockIdx.x) * SLICE - mis;
  const int first = max(base, 0), last = min(base + SLICE, a.vocab);
  const bool st16 = (reinterpret_cast<uintptr_t>(out + base) & 15) == 0;
  const uint32_t* mask = a.r.allowed ? a.r.allowed + row * a.r.allowed_stride : nullptr;
  const int words = (a.vocab - 1) >> 5;
  uint4 x[2][U];
  uint32_t mlo[2][U], mhi[2][U];   // a vector's mask bits lie in one word or two
  auto load = [&](int sub, uint4 (&v)[U], uint32_t (&lo)[U], uint32_t (&hi)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v0 = base + sub * SUB + (u * LG_THREADS + tid) * VEC;
      if (mask) {
        const int w0 = min(max(v0, 0) >> 5, words);
        lo[u] = __ldg(mask + w0);
        hi[u] = __ldg(mask + min(w0 + 1, words));
      }
      if (v0 >= 0 && v0 + VEC <= a.vocab) {
        v[u] = *reinterpret_cast<const uint4*>(in + v0);
      } else {
        T* e = reinterpret_cast<T*>(&v[u]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = v0 + j >= 0 && v0 + j < a.vocab ? in[v0 + j] : from_f32<T>(-INFINITY);
      }
    }
  };
  load(0, x[0], mlo[0], mhi[0]);
  // ---- the few: `changed` holds how often a token stands in the history, then its new logit, which a bit announces.  Loads of a step are issued together; each step is a round trip to L2 at most.
  int* changed = lg_smem;                                             // [SLICE]
  uint32_t* bits = reinterpret_cast<uint32_t*>(lg_smem + SLICE);      // [SLICE / 32]
  uint32_t* biased = bits + SLICE / 32;                               // [SLICE / 32]
  int* n_listed = lg_smem + SLICE + SLICE / 16;                       // the history's tokens in this slice, each once, so that
  uint16_t* listed = reinterpret_cast<uint16_t*>(n_listed + 4);       // warps work on whole lots of them: [LISTED]
  const bool sparse = a.r.tokens || a.r.bias_tokens;
  if (sparse) {
    int hb = 0, he = 0, bb = 0, be = 0;
    if (a.r.tokens) seq_range(a.r.token_offsets, row, a.r.n_tokens, a.status, hb, he);
    if (a.r.bias_tokens) seq_range(a.r.bias_offsets, row, a.r.n_bias, a.status, bb, be);
    constexpr int E = 8;   // history entries of a thread that stay in registers between the steps
    int ids[E];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int i = i0 + tid + k * LG_THREADS;
        const int id = i < he ? __ldg(a.r.tokens + i) : -1;
        ids[k] = id >= first && id < last ? id - base : -1;
      }
    };
    if (tid == 0) *n_listed = 0;
    fetch(hb);
    const int bias0 = a.r.bias_tokens && bb + tid < be ? __ldg(a.r.bias_tokens + bb + tid) : -1;
    for (int i = 4 * tid; i < SLICE + SLICE / 16; i += 4 * LG_THREADS) *reinterpret_cast<int4*>(lg_smem + i) = make_int4(0, 0, 0, 0);
    const float rep = a.r.repetition ? __ldg(a.r.repetition + row) : 1.0f;
    const float freq = a.r.frequency ? __ldg(a.r.frequency + row) : 0.0f;
    const float pres = a.r.presence ? __ldg(a.r.presence + row) : 0.0f;
    // their logits on the way to L2
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (ids[k] >= 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(in + base + ids[k]));
    if (bias0 >= first && bias0 < last) asm volatile("prefetch.global.L2 [%0];" ::"l"(in + bias0));
    __syncthreads();
    auto entry = [&](int i) {   // place in the slice of a bias entry's token, or -1
      const int id = i >= bb && i < be ? __ldg(a.r.bias_tokens + i) : -1;
      return id >= first && id < last ? id - base : -1;
    };
    bool twice = false;   // a token stands twice among the biases: rare, and its last entry counts
    for (int i = bb + tid; i < be; i += LG_THREADS)
      if (const int at = entry(i); at >= 0) {
        const uint32_t bit = 1u << (at & 31);
        twice = twice || (atomicOr(biased + (at >> 5), bit) & bit);
      }
    if (he > hb) {
      for (int i0 = hb;;) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          if (ids[k] < 0) continue;
          const bool first_of = atomicAdd(changed + ids[k], 1) == 0;
          if (LISTED > 0 && first_of) {
            if (const int at = atomicAdd(n_listed, 1); at < LISTED) listed[at] = uint16_t(ids[k]);
          }
          if (LISTED == 0 && !first_of) ids[k] = -1;
        }
        i0 += E * LG_THREADS;
        if (i0 >= he) break;
        fetch(i0);
      }
    }
    twice = __syncthreads_or(twice);
    auto penalise = [&](int id) {
      const float v = to_f32(in[base + id]);
      // separate roundings, so that the result does not hang on a contraction
      const float f = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      changed[id] = __float_as_int(__fsub_rn(f, __fadd_rn(__fmul_rn(freq, float(changed[id])), pres)));
    };
    if (LISTED == 0 && he - hb <= E * LG_THREADS) {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (ids[k] >= 0) {
          atomicOr(bits + (ids[k] >> 5), 1u << (ids[k] & 31));
          penalise(ids[k]);
        }
      __syncthreads();
    } else if (const int n = LISTED > 0 ? *n_listed : 1; n > LISTED) {   // too many to list: the first of a token's places in the history works for all
      for (int i = hb + tid; i < he; i += LG_THREADS) {
        int id = __ldg(a.r.tokens + i);
        if (id < first || id >= last) continue;
        id -= base;
        const uint32_t bit = 1u << (id & 31);
        if (!(atomicOr(bits + (id >> 5), bit) & bit)) penalise(id);
      }
      __syncthreads();
    } else if (n > 0) {
      for (int i = tid; i < n; i += LG_THREADS) {
        const int id = listed[i];
        atomicOr(bits + (id >> 5), 1u << (id & 31));
        penalise(id);
      }
      __syncthreads();
    }
    auto add = [&](int i, int at) {
      const uint32_t bit = 1u << (at & 31);
      const float raw = to_f32(in[base + at]), value = __ldg(a.r.bias_values + i);
      const bool held = atomicOr(bits + (at >> 5), bit) & bit;
      changed[at] = __float_as_int(__fadd_rn(held ? __int_as_float(changed[at]) : raw, value));
    };
    if (!twice) {
      for (int i = bb + tid; i < be; i += LG_THREADS)
        if (const int at = entry(i); at >= 0) add(i, at);
    } else if (tid < 32) {
      for (int w = lane; w < SLICE / 32; w += 32) biased[w] = 0u;
      __syncwarp();
      for (int i0 = be; i0 > bb; i0 -= 32) {   // from the last entry to the first: a token that is marked has had its own
        const int i = i0 - 1 - lane, at = entry(i);
        const unsigned same = __match_any_sync(0xffffffffu, at >= 0 ? at : -1 - lane);
        const uint32_t bit = 1u << (at & 31);
        if (at >= 0 && __ffs(same) - 1 == lane && !(atomicOr(biased + (at >> 5), bit) & bit)) add(i, at);
        __syncwarp();
      }
    }
    __syncthreads();
    // `out` may be `in`: nobody writes before every thread has read what it changes
  }
  // ---- all of them
  float top_v = -INFINITY;   // a thread's tokens ascend, so the first of equals stays
  int top_i = -1;
#pragma unroll
  for (int sub = 0; sub < NSUB; ++sub) {
    if (base + sub * SUB >= a.vocab) break;
    if (sub + 1 < NSUB) load(sub + 1, x[(sub + 1) & 1], mlo[(sub + 1) & 1], mhi[(sub + 1) & 1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l0 = sub * SUB + (u * LG_THREADS + tid) * VEC, v0 = base + l0;
      const T* raw = reinterpret_cast<const T*>(&x[sub & 1][u]);
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = to_f32(raw[j]);
      if (sparse) {
        const uint32_t b = bits[l0 >> 5] >> (l0 & 31);
        if (b & ((1u << VEC) - 1u)) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if ((b >> j) & 1u) f[j] = __int_as_float(changed[l0 + j]);
        }
      }
      const bool whole = v0 >= 0 && v0 + VEC <= a.vocab;
      if (mask) {
        const int shift = v0 - 32 * (max(v0, 0) >> 5);   // negative before the row: such tokens are not written
        const uint32_t lo = mlo[sub & 1][u], hi = mhi[sub & 1][u];
        const uint32_t m = shift >= 0 ? __funnelshift_r(lo, hi, shift) : lo << -shift;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!((m >> j) & 1u)) f[j] = -INFINITY;
      }
      uint4 packed;
      T* y = reinterpret_cast<T*>(&packed);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        y[j] = from_f32<T>(f[j]);
        const float w = to_f32(y[j]);
        if (w > top_v) {   // tokens outside the row were loaded as -infinity
          top_v = w;
          top_i = v0 + j;
        }
      }
      if (st16 && whole) {
        *reinterpret_cast<uint4*>(out + v0) = packed;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (v0 + j >= 0 && v0 + j < a.vocab) out[v0 + j] = y[j];
      }
    }
  }
  if (!a.best) return;
  unsigned long long top = top_i >= 0 ? logit_key(top_v, top_i) : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, top, o);
    top = k > top ? k : top;
  }
  if (lane == 0) wbest[tid >> 5] = top;
  __syncthreads();
  if (tid != 0) return;
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

template <typename T, int U, int NSUB>
static int logits_run(LogitsArgs& a) {
  constexpr int VEC = 16 / sizeof(T), SLICE = LG_THREADS * VEC * U * NSUB;
  const dim3 grid(unsigned(cdiv(int64_t(a.vocab) + VEC - 1, SLICE)), unsigned(a.rows));
  if (a.best && grid.x > 1) {
    // keys first, so that both arrays keep their alignment
    uint8_t* p = static_cast<uint8_t*>(scratch(size_t(65536) * 12, SCRATCH_ARGMAX, true));
    if (!p) return scratch_failed("logits_process");
    a.key = reinterpret_cast<unsigned long long*>(p);
    a.arrived = reinterpret_cast<int*>(p + size_t(65536) * 8);
  }
  const size_t smem = a.r.tokens || a.r.bias_tokens ? size_t(SLICE) * 4 + SLICE / 4 + 16 + SLICE / 4 : 0;
  auto kern = logits_kernel<T, U, NSUB>;
  if (smem > 32 * 1024) SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  SIMP_CUDA(launch_kernel(kern, grid, dim3(LG_THREADS), smem, ctx().stream, true, a));
  return SIMP_OK;
}

// Slices of 8192 tokens where that still gives every SM two blocks, else of 1024 (f32) or 2048.  200 rows of 128256 with
// histories of 2000: 55 us with 8192, 62 with 16384 (three blocks per SM), 66 with 4096 (histories read twice as often);
// without history and biases 36 us, 0.87 of the memory's rate.
template <typename T>
static int logits_launch(LogitsArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  if (cdiv(a.vocab, 8192) * a.rows >= 2 * ctx().sm_count) return logits_run<T, 2, 16 / VEC>(a);
  return logits_run<T, 1, 1>(a);
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
  SIMP_REQUIRE(r.n_tokens >= 0 && r.n_tokens <= (1 << 30) && r.n_bias >= 0 && r.n_bias <= (1 << 30), SIMP_ERR_ARG,
               "logits_process: a list's length is outside 0 .. 2^30");
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
