// attn_prompt.cu -- causal attention over prompts: packed sequences of different lengths, grouped heads.
//
// This file holds the entry point and the FFMA kernel.  Heads of up to 128 elements run on the tensor cores: f16 and bf16 in
// attn_prompt_tc.cu, f32 in attn_prompt_f32_tc.cu.  The FFMA kernel does what those cannot: scale <= 0 for 16-bit types,
// calls without keys or with more rows than their tensor maps address, and calls for which no scratch can be had (inside a
// recording that would have to grow it).
//
// FFMA kernel: one block per 64 queries of one head.  Scores of 64 keys at a time, the running maximum and sum of the softmax
// per row, one pass over K and V.  Bound by FFMA and the shared-memory loads that feed it: 32 heads of 100, 2048 f32 tokens
// 1010 us, where the tensor cores take 240.
#include <algorithm>
#include <climits>

#include "attn_prompt.cuh"

namespace simp {

constexpr int AP_BM = 64, AP_BN = 64, AP_THREADS = 128;

template <int DP>
constexpr size_t ap_smem() { return size_t(DP * AP_BM + DP * AP_BN + AP_BN * DP + AP_BN * AP_BM) * 4; }

// Thread (ty = tid / 8, tx = tid % 8): scores of rows 4 ty .. +3, keys 4 tx .. +3 and 32 + 4 tx .. +3; outputs of the same
// rows, elements 4 tx + 32 i.
template <typename T, int DP>
__global__ void __launch_bounds__(AP_THREADS) attn_prompt_f32_kernel(const AttnPromptArgs a) {
  extern __shared__ __align__(16) float ap_sm[];
  float* Qs = ap_sm;                    // [DP][BM]
  float* Ks = Qs + DP * AP_BM;          // [DP][BN]
  float* Vs = Ks + DP * AP_BN;          // [BN][DP]
  float* Ps = Vs + AP_BN * DP;          // [BN][BM]
  constexpr int OC = DP / 32;
  int seq, tile;
  auto count = [&](int s) {
    int b, e;
    return seq_range(a.q_off, s, a.total_q, a.status, b, e) ? (e - b + AP_BM - 1) / AP_BM : 0;
  };
  if (!find_unit(blockIdx.x, a.n_seqs, count, seq, tile)) return;
  int q0, q1, k0, k1;
  seq_range(a.q_off, seq, a.total_q, a.status, q0, q1);
  if (!seq_range(a.k_off, seq, a.total_k, a.status, k0, k1)) return;
  const int nq = q1 - q0, nk = k1 - k0;
  tile = (nq + AP_BM - 1) / AP_BM - 1 - tile;   // long rows first
  const int r0 = tile * AP_BM, h = blockIdx.y, kvh = h / a.rep, D = a.D;
  const int64_t shift = int64_t(nk) - nq;       // row i sees keys j <= i + shift
  const T* q = static_cast<const T*>(a.q) + int64_t(q0 + r0) * a.q_stride + int64_t(h) * D;
  const T* k = static_cast<const T*>(a.k) + int64_t(k0) * a.kv_stride + int64_t(kvh) * D;
  const T* v = static_cast<const T*>(a.v) + int64_t(k0) * a.kv_stride + int64_t(kvh) * D;
  T* out = static_cast<T*>(a.out) + int64_t(q0 + r0) * a.out_stride + int64_t(h) * D;
  const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7;
  const int rows = min(AP_BM, nq - r0);
  for (int i = tid; i < DP * AP_BM; i += AP_THREADS) {
    const int r = i / DP, d = i - r * DP;
    Qs[d * AP_BM + r] = r < rows && d < D ? to_f32(q[r * a.q_stride + d]) : 0.0f;
  }
  float o[4][4 * OC], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4 * OC; ++j) o[i][j] = 0.0f;
  }
  const int64_t see = min(int64_t(nk), int64_t(r0) + rows + shift);   // keys that the last row sees
  for (int64_t j0 = 0; j0 < see; j0 += AP_BN) {
    __syncthreads();
    const int keys = int(min(int64_t(AP_BN), see - j0));
    for (int i = tid; i < DP * AP_BN; i += AP_THREADS) {
      const int r = i / DP, d = i - r * DP;
      const bool in = r < keys && d < D;
      Ks[d * AP_BN + r] = in ? to_f32(k[(j0 + r) * a.kv_stride + d]) : 0.0f;
      Vs[r * DP + d] = in ? to_f32(v[(j0 + r) * a.kv_stride + d]) : 0.0f;
    }
    __syncthreads();
    float s[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < D; ++d) {
      const float4 qa = *reinterpret_cast<const float4*>(Qs + d * AP_BM + 4 * ty);
      const float4 ka = *reinterpret_cast<const float4*>(Ks + d * AP_BN + 4 * tx);
      const float4 kb = *reinterpret_cast<const float4*>(Ks + d * AP_BN + 32 + 4 * tx);
      const float qv[4] = {qa.x, qa.y, qa.z, qa.w}, kv[8] = {ka.x, ka.y, ka.z, ka.w, kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = fmaf(qv[i], kv[j], s[i][j]);
    }
    const bool edge = j0 + AP_BN > min(int64_t(nk), r0 + shift + 1);   // some row does not see some key of this tile
    float alpha[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t lim = min(int64_t(nk), r0 + 4 * ty + i + shift + 1) - j0;   // keys of the tile that row i sees
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = (j >> 2) * 32 + 4 * tx + (j & 3);
        s[i][j] = edge && key >= lim ? -INFINITY : s[i][j] * a.scale_log2;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float mn = fmaxf(m[i], top), base = mn == -INFINITY ? 0.0f : mn;
      alpha[i] = exp2f(m[i] - base);
      m[i] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        sum += s[i][j];
      }
      l[i] = fmaf(l[i], alpha[i], sum);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = (j >> 2) * 32 + 4 * tx + (j & 3);
      *reinterpret_cast<float4*>(Ps + key * AP_BM + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4 * OC; ++j) o[i][j] *= alpha[i];
    __syncwarp();   // the rows 4 ty .. of P are written and read by the same eight lanes
    if (edge) {
      // a key that a row does not see is left out, not multiplied by zero: it may be NaN or infinite
      for (int j = 0; j < keys; ++j) {
        const float4 pa = *reinterpret_cast<const float4*>(Ps + j * AP_BM + 4 * ty);
        const float pv[4] = {pa.x, pa.y, pa.z, pa.w};
#pragma unroll
        for (int c = 0; c < OC; ++c) {
          const float4 va = *reinterpret_cast<const float4*>(Vs + j * DP + 32 * c + 4 * tx);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pv[i] != 0.0f) {
              o[i][4 * c] = fmaf(pv[i], va.x, o[i][4 * c]);
              o[i][4 * c + 1] = fmaf(pv[i], va.y, o[i][4 * c + 1]);
              o[i][4 * c + 2] = fmaf(pv[i], va.z, o[i][4 * c + 2]);
              o[i][4 * c + 3] = fmaf(pv[i], va.w, o[i][4 * c + 3]);
            }
        }
      }
    } else {
#pragma unroll 4
      for (int j = 0; j < AP_BN; ++j) {
        const float4 pa = *reinterpret_cast<const float4*>(Ps + j * AP_BM + 4 * ty);
        const float pv[4] = {pa.x, pa.y, pa.z, pa.w};
#pragma unroll
        for (int c = 0; c < OC; ++c) {
          const float4 va = *reinterpret_cast<const float4*>(Vs + j * DP + 32 * c + 4 * tx);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[i][4 * c] = fmaf(pv[i], va.x, o[i][4 * c]);
            o[i][4 * c + 1] = fmaf(pv[i], va.y, o[i][4 * c + 1]);
            o[i][4 * c + 2] = fmaf(pv[i], va.z, o[i][4 * c + 2]);
            o[i][4 * c + 3] = fmaf(pv[i], va.w, o[i][4 * c + 3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int r = 4 * ty + i;
    if (r >= rows) continue;
#pragma unroll
    for (int j = 0; j < 4 * OC; ++j) {
      const int d = (j >> 2) * 32 + 4 * tx + (j & 3);
      if (d < D) out[r * a.out_stride + d] = from_f32<T>(l[i] == 0.0f ? 0.0f : o[i][j] / l[i]);
    }
  }
}

template <typename T, int DP>
static int ap_launch(const AttnPromptArgs& a) {
  auto kern = attn_prompt_f32_kernel<T, DP>;
  SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ap_smem<DP>())));
  const dim3 grid(unsigned(std::min(a.total_q, a.total_q / AP_BM + a.n_seqs)), unsigned(a.H));
  kern<<<grid, AP_THREADS, ap_smem<DP>(), ctx().stream>>>(a);
  SIMP_LAUNCH_CHECK();
  return SIMP_OK;
}
template <typename T>
static int ap_dispatch(const AttnPromptArgs& a) {
  return a.D <= 32 ? ap_launch<T, 32>(a) : a.D <= 64 ? ap_launch<T, 64>(a) : ap_launch<T, 128>(a);
}

}  // namespace simp

using namespace simp;

SIMP_API int simp_gpu_attn_prompt(const void* q_dev, const void* k_dev, const void* v_dev, void* out_dev, const int32_t* q_offsets_dev,
                                  const int32_t* k_offsets_dev, int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t n_heads,
                                  int64_t n_kv_heads, int64_t head_dim, int64_t q_stride, int64_t kv_stride, int64_t out_stride,
                                  float scale, int dtype) {
  SIMP_REQUIRE(dtype_ok(dtype), SIMP_ERR_ARG, "attn_prompt: unknown dtype %d", dtype);
  SIMP_REQUIRE(n_seqs >= 0 && total_q >= 0 && total_k >= 0, SIMP_ERR_ARG, "attn_prompt: negative size");
  SIMP_REQUIRE(head_dim >= 1 && head_dim <= 128, SIMP_ERR_SHAPE, "attn_prompt: head_dim %lld outside 1 .. 128", (long long)head_dim);
  SIMP_REQUIRE(n_heads >= 1 && n_kv_heads >= 1 && n_heads <= 65535 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128, SIMP_ERR_SHAPE,
               "attn_prompt: %lld query heads over %lld key/value heads", (long long)n_heads, (long long)n_kv_heads);
  if (n_seqs == 0 || total_q == 0) return SIMP_OK;
  SIMP_REQUIRE(n_seqs < INT_MAX && total_q <= INT_MAX && total_k <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many sequences or rows");
  SIMP_REQUIRE(q_dev && out_dev && q_offsets_dev && (total_k == 0 || (k_dev && v_dev)), SIMP_ERR_ARG, "attn_prompt: null pointer");
  SIMP_REQUIRE(k_offsets_dev || total_k == total_q, SIMP_ERR_SHAPE, "attn_prompt: %lld keys for %lld queries need k_offsets", (long long)total_k,
               (long long)total_q);
  if (q_stride == 0) q_stride = n_heads * head_dim;
  if (out_stride == 0) out_stride = n_heads * head_dim;
  if (kv_stride == 0) kv_stride = n_kv_heads * head_dim;
  SIMP_REQUIRE(q_stride >= n_heads * head_dim && out_stride >= n_heads * head_dim && kv_stride >= n_kv_heads * head_dim, SIMP_ERR_SHAPE,
               "attn_prompt: a stride is shorter than a row");
  const size_t es = dtype_size(dtype);
  SIMP_REQUIRE(aligned_to(q_dev, es) && aligned_to(k_dev, es) && aligned_to(v_dev, es) && aligned_to(out_dev, es), SIMP_ERR_ARG,
               "attn_prompt: misaligned pointer");
  if (int rc = ensure_ready()) return rc;
  DeviceScope dev;
  AttnPromptArgs a{};
  a.q = q_dev;
  a.k = k_dev;
  a.v = v_dev;
  a.out = out_dev;
  a.q_off = q_offsets_dev;
  a.k_off = k_offsets_dev ? k_offsets_dev : q_offsets_dev;
  a.total_q = total_q;
  a.total_k = total_k;
  a.q_stride = q_stride;
  a.kv_stride = kv_stride;
  a.out_stride = out_stride;
  a.n_seqs = int(n_seqs);
  a.H = int(n_heads);
  a.G = int(n_kv_heads);
  a.rep = int(n_heads / n_kv_heads);
  a.D = int(head_dim);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = ctx().dev_status;
  if (dtype == SIMP_DTYPE_F32) {
    if (int rc = attn_prompt_f32_tc(a); rc <= 0) return rc;
    return ap_dispatch<float>(a);
  }
  if (int rc = attn_prompt_tc(a, dtype); rc <= 0) return rc;
  if (dtype == SIMP_DTYPE_F16) return ap_dispatch<__half>(a);
  return ap_dispatch<__nv_bfloat16>(a);
}
