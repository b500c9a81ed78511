// attn_prompt_f32_tc.cu -- causal attention over packed prompts at f32 accuracy on the tcgen05 tensor cores.
//
// q, k and v are split into three bf16 planes each (x = h + m + l, 24 bits), and a product is the six plane products of
// relative size 2^-16 and above: l.h, h.l, m.m, m.h, h.m, h.h.  The tensor cores add into their f32 accumulators with
// truncation, so (1) the small products come first and only the last eighth or less of the additions is made at full
// size, and (2) the output of every tile of keys is a sum of its own, added to f32 registers with rounding: an
// accumulator kept over a long prompt would drift by 2e-8 per instruction.
//
// One block of 12 warps per row tile (128 rows: 128 / rep tokens x the rep heads that share a key/value head):
//   warp 0      TMA: the planes of K and V per tile of 64 keys (head sizes up to 64: 128), two stages of 48 KB each
//   warp 1      MMAs: S = Q K^T as soon as the softmax has read the S before; T = P V into a TMEM tile
//   warps 4-11  softmax, two threads per row; P in three planes to TMEM; T into registers (D / 2 each)
// The planes of Q lie in TMEM: from shared memory they would be read again for every product (6 KB per MMA of 32 cycles,
// where shared memory gives 128 bytes a cycle: 77 cycles were measured), and there would be no room for second stages.
// Per tile the tensor cores need 3072 cycles, the softmax about as many beside them.
//
// No plane product of an infinity or a NaN is right, and a zero weight does not hide them from an MMA (a tile may hold keys
// that some rows must not see, or rows of the next sequence).  The splitting pass leaves them out of the planes and marks
// the row and head; where anything is marked, scores of marked rows are computed again from the f32 tensors, and marked
// values that a row sees are added to its output at the end.  Whoever does not see them gets the same bits as without.
#include <algorithm>
#include <climits>

#include "attn_tc.cuh"

namespace simp {

constexpr int F3_THREADS = 384;

template <int D>
struct F3Shape {
  static constexpr int KEYS = D == 64 ? 128 : 64, ATOM = KEYS * 128;   // bytes of 64 elements of a tile's rows
  static constexpr int PLANE = KEYS * D * 2, STAGE = 3 * PLANE;
  static constexpr int BARS = 13;
  static constexpr size_t SMEM = 4 * size_t(STAGE) + BARS * 8 + 16 + 8 * 128 + 24;
  static constexpr uint32_t P = KEYS, T = P + 3 * KEYS / 2, Q = T + D;   // TMEM columns: S, three planes of P, T, three planes of Q
  static_assert(Q + 3 * D / 2 <= 512 && SMEM <= 232448, "");
};

struct F3Args {
  AttnPromptArgs a;
  int tpt;
  const uint16_t* q;   // planes [3][total_q][H][D]
  const int* any;   // set: some element is not finite; then the bytes of its row and head are set:
  const uint8_t *odd_q, *odd_k, *odd_v;
};

__device__ __forceinline__ uint32_t tmem_ld_1(uint32_t t) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(t) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_st_1(uint32_t t, uint32_t v) { asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(t), "r"(v) : "memory"); }

template <int D>
__global__ void __launch_bounds__(F3_THREADS, 1)
    attn_prompt_f32_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const F3Args p) {
  using Sh = F3Shape<D>;
  constexpr int KEYS = Sh::KEYS, MINE = KEYS / 2;   // keys of a tile, of a thread
  extern __shared__ __align__(1024) uint8_t f3_raw[];
  const uint32_t base = smem_u32(f3_raw), k_smem = base, v_smem = base + 2 * Sh::STAGE, bars = base + 4 * Sh::STAGE;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 16u + 8u * s; };
  auto v_full = [&](int s) { return bars + 32u + 8u * s; };
  auto v_empty = [&](int s) { return bars + 48u + 8u * s; };
  const uint32_t s_bar = bars + 64, s_read = bars + 72, p_bar = bars + 80, t_bar = bars + 88, q_bar = bars + 96;
  uint8_t* tail = f3_raw + 4 * Sh::STAGE + Sh::BARS * 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8);
  float* half_row = reinterpret_cast<float*>(tail + 16);   // [half][row]
  volatile int* found_unit = reinterpret_cast<volatile int*>(half_row + 2 * 128);   // found, place, q0, q1, k0, k1
  const AttnPromptArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {   // never: the declaration asks for it
    if (threadIdx.x == 0) report_status(a.status, 1, 70);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full(i), 1);
      mbar_init(k_empty(i), 1);
      mbar_init(v_full(i), 1);
      mbar_init(v_empty(i), 1);
    }
    mbar_init(s_bar, 1);
    mbar_init(s_read, 8);
    mbar_init(p_bar, 8);
    mbar_init(t_bar, 1);
    mbar_init(q_bar, 8);
    *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_launch_dependents();
  pdl_wait();
  // ---- which rows: found by one warp while the others prepare
  const int g = blockIdx.x % a.G;
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  if (warp == 0) {
    auto count = [&](int s) {
      int b, e;
      return seq_range(a.q_off, s, a.total_q, a.status, b, e) ? (e - b + p.tpt - 1) / p.tpt : 0;
    };
    auto keys_of = [&](int s) { return __ldg(a.k_off + s + 1) - __ldg(a.k_off + s); };
    int seq = 0, place = 0;
    bool found = find_unit(blockIdx.x / a.G, a.n_seqs, count, seq, place, keys_of);
    if (found) {
      seq_range(a.q_off, seq, a.total_q, a.status, q0, q1);
      found = seq_range(a.k_off, seq, a.total_k, a.status, k0, k1);
    }
    if (lane == 0) {
      found_unit[0] = found;
      found_unit[1] = place;
      found_unit[2] = q0;
      found_unit[3] = q1;
      found_unit[4] = k0;
      found_unit[5] = k1;
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);   // (all: one block per SM)
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  constexpr uint32_t tmem = 0;   // the block allocates every column
  if (!found_unit[0]) {
    if (warp == 1) tmem_dealloc(tmem, 512);
    return;
  }
  q0 = found_unit[2];
  q1 = found_unit[3];
  k0 = found_unit[4];
  k1 = found_unit[5];
  const int place = found_unit[1];
  const int nq = q1 - q0, nk = k1 - k0;
  const int r0 = ((nq + p.tpt - 1) / p.tpt - 1 - place) * p.tpt;   // the longest rows first
  const int64_t shift = int64_t(nk) - nq;
  auto sees = [&](int token) { return int(max(int64_t(0), min(int64_t(nk), token + shift + 1))); };
  const int n = (sees(min(r0 + p.tpt, nq) - 1) + KEYS - 1) / KEYS;

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0 && n > 0) {
      bool ok = true;
      auto tile = [&](const CUtensorMap* map, uint32_t dst, uint32_t full, uint32_t empty, int j) {
        ok = ok && wait_bar(empty, ((j >> 1) & 1) ^ 1, abort_flag, a.status, 71);
        if (!ok) return;
        mbar_arrive_expect_tx(full, Sh::STAGE);
        for (int s = 0; s < 3; ++s)
          for (int b = 0; b < D / 64; ++b)
            tma_load_3d(dst + (j & 1) * Sh::STAGE + s * Sh::PLANE + b * Sh::ATOM, map, full, 64 * b, g, int(s * a.total_k) + k0 + KEYS * j);
      };
      for (int j = 0; ok && j < n; ++j) {
        tile(&map_k, k_smem, k_full(j & 1), k_empty(j & 1), j);
        tile(&map_v, v_smem, v_full(j & 1), v_empty(j & 1), j);
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);   // let copies in flight land before the block retires
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMAs (the whole warp with the same values, one lane issues)
    constexpr uint32_t idesc_s = idesc_f16(true, KEYS, false);
    const int width = (a.D + 15) / 16;                        // steps of 16 elements that hold something
    const uint32_t idesc_t = idesc_f16(true, 16 * width, true);
    const bool leader = lane == 0;
    auto wait = [&](uint32_t bar, uint32_t phase, int site) {
      const bool ok = __all_sync(0xffffffffu, wait_bar(bar, phase, abort_flag, a.status, site));
      tc_fence_after_sync();
      return ok;
    };
    // planes of the two operands, small products first
    constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
    auto scores = [&](int j) {
      const uint64_t kd = make_smem_desc_sw128(k_smem, 16u, 1024u) + uint64_t((j & 1) * (Sh::STAGE / 16));
#pragma unroll
      for (int t = 0; t < 6; ++t)
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          mma_f16_ts(tmem, tmem + Sh::Q + uint32_t(D / 2) * PA[t] + 8u * s, kd + uint64_t(PB[t] * (Sh::PLANE / 16) + (s >> 2) * (Sh::ATOM / 16) + (s & 3) * 2),
                     idesc_s, t > 0 || s > 0, leader && s < width);
    };
    auto values = [&](int j) {
      const uint64_t vd = make_smem_desc_sw128(v_smem, uint32_t(Sh::ATOM), 1024u) + uint64_t((j & 1) * (Sh::STAGE / 16));   // 8 keys 1 KB apart
#pragma unroll
      for (int t = 0; t < 6; ++t)
#pragma unroll
        for (int s = 0; s < KEYS / 16; ++s)
          mma_f16_ts(tmem + Sh::T, tmem + Sh::P + uint32_t(KEYS / 2) * PA[t] + 8u * s, vd + uint64_t(PB[t] * (Sh::PLANE / 16) + s * 128), idesc_t, t > 0 || s > 0,
                     leader);
    };
    bool ok = true;
    if (n > 0) {
      ok = wait(q_bar, 0, 72) && wait(k_full(0), 0, 73);
      if (ok) {
        scores(0);
        if (leader) {
          mma_commit(s_bar);
          mma_commit(k_empty(0));
        }
      }
    }
    for (int j = 0; ok && j < n; ++j) {
      if (j + 1 < n) {
        ok = wait(k_full((j + 1) & 1), ((j + 1) >> 1) & 1, 74) && wait(s_read, j & 1, 75);
        if (!ok) break;
        scores(j + 1);
        if (leader) {
          mma_commit(s_bar);
          mma_commit(k_empty((j + 1) & 1));
        }
      }
      ok = wait(v_full(j & 1), (j >> 1) & 1, 76) && wait(p_bar, j & 1, 77);
      if (!ok) break;
      values(j);
      if (leader) {
        mma_commit(t_bar);
        mma_commit(v_empty(j & 1));
      }
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax and sums
    const int half = (warp - 4) >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_tmem = tmem + lanes + uint32_t(MINE) * half, t_tmem = tmem + Sh::T + lanes + uint32_t(D / 2) * half;
    const int token = r0 + row / a.rep, head = g * a.rep + row % a.rep;
    const bool mine = row < p.tpt * a.rep && token < nq;
    const int lim = mine ? sees(token) : 0;
    volatile float* to = half_row + half * 128 + row;
    volatile float* from = half_row + (half ^ 1) * 128 + row;
    // this row's planes of Q, half a row per thread, to TMEM (rows behind the sequence: zeros)
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t(q) * a.total_q + q0 + token) * a.H * D + int64_t(head) * D + (D / 2) * half);
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {   // 16 elements
        uint32_t w[8];
        const uint4 x = mine ? __ldg(src + 2 * h) : make_uint4(0u, 0u, 0u, 0u), y = mine ? __ldg(src + 2 * h + 1) : make_uint4(0u, 0u, 0u, 0u);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
        tmem_st_32x8(tmem + lanes + Sh::Q + uint32_t(D / 2) * q + uint32_t(D / 4) * half + 8u * h, w);
      }
    }
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_bar);
    const bool any = __ldcg(p.any) != 0, odd_row = any && mine && p.odd_q[int64_t(q0 + token) * a.H + head];
    float m = -INFINITY, l = 0.0f, o[D / 2];
#pragma unroll
    for (int i = 0; i < D / 2; ++i) o[i] = 0.0f;
    auto add_tile = [&](float alpha) {   // the tile's sum to the registers, then both to the new maximum
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        uint32_t t[16];
        tmem_ld_32x16(t_tmem + 16u * h, t);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[16 * h + i] = (o[16 * h + i] + __uint_as_float(t[i])) * alpha;
      }
    };
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = wait_bar(s_bar, j & 1, abort_flag, a.status, 78) && ok;
      tc_fence_after_sync();
      if (any) {   // rare: scores of rows that are not finite, by the f32 tensors
#pragma unroll 1
        for (int i = 0; i < MINE; ++i) {
          const int key = KEYS * j + MINE * half + i;
          uint32_t v = tmem_ld_1(s_tmem + i);
          tmem_ld_wait();
          if (key < lim && (odd_row || p.odd_k[int64_t(k0 + key) * a.G + g])) {
            const float* qr = static_cast<const float*>(a.q) + int64_t(q0 + token) * a.q_stride + int64_t(head) * a.D;
            const float* kr = static_cast<const float*>(a.k) + int64_t(k0 + key) * a.kv_stride + int64_t(g) * a.D;
            float d = 0.0f;
#pragma unroll 1
            for (int e = 0; e < a.D; ++e) d = fmaf(qr[e], kr[e], d);
            v = __float_as_uint(d);
          }
          __syncwarp();
          tmem_st_1(s_tmem + i, v);
        }
        tmem_st_wait();
      }
      uint32_t s[MINE];
#pragma unroll
      for (int h = 0; h < MINE / 32; ++h) tmem_ld_32x32(s_tmem + 32u * h, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * h));
      tmem_ld_wait();
      const int see = lim - KEYS * j - MINE * half;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const float y = i < see ? __uint_as_float(s[i]) * a.scale_log2 : -INFINITY;
        s[i] = __float_as_uint(y);
        top = fmaxf(top, y);
      }
      *to = top;
      tc_fence_before_sync();
      ok = all_of(1 + (warp & 3), 64, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive(s_read);
      const float mn = fmaxf(m, fmaxf(top, *from)), off = mn == -INFINITY ? 0.0f : mn;
      const float alpha = ex2(m - off);   // 0 for the first tile
      m = mn;
      float sum = 0.0f;
      uint32_t w[3][MINE / 2];
#pragma unroll
      for (int i = 0; i < MINE / 2; ++i) {
        const float e0 = ex2(__uint_as_float(s[2 * i]) - off), e1 = ex2(__uint_as_float(s[2 * i + 1]) - off);
        sum += e0 + e1;
        w[0][i] = pack2<true>(e0, e1);
        const float f0 = e0 - __uint_as_float(w[0][i] << 16), f1 = e1 - __uint_as_float(w[0][i] & 0xffff0000u);
        w[1][i] = pack2<true>(f0, f1);
        w[2][i] = pack2<true>(f0 - __uint_as_float(w[1][i] << 16), f1 - __uint_as_float(w[1][i] & 0xffff0000u));
      }
      if (j > 0) {   // the tile before: when it is done, its sum is taken and its P may be overwritten
        ok = __all_sync(0xffffffffu, wait_bar(t_bar, (j - 1) & 1, abort_flag, a.status, 79)) && ok;
        tc_fence_after_sync();
        add_tile(alpha);
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int h = 0; h < MINE / 32; ++h)
          tmem_st_32x16(tmem + lanes + Sh::P + uint32_t(KEYS / 2) * q + uint32_t(MINE / 2) * half + 16u * h, *reinterpret_cast<uint32_t(*)[16]>(w[q] + 16 * h));
      l = fmaf(l, alpha, sum);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_bar);
    }
    if (ok && n > 0) {
      ok = __all_sync(0xffffffffu, wait_bar(t_bar, (n - 1) & 1, abort_flag, a.status, 80));
      tc_fence_after_sync();
      add_tile(1.0f);
    }
    *to = l;
    ok = all_of(1 + (warp & 3), 64, ok);
    if (ok && mine) {
      l += *from;
      float* out = static_cast<float*>(a.out) + int64_t(q0 + token) * a.out_stride + int64_t(head) * a.D + (D / 2) * half;
      const int cols = a.D - (D / 2) * half;
      if (any)
#pragma unroll 1
        for (int key = 0; key < lim; ++key) {
          if (!p.odd_v[int64_t(k0 + key) * a.G + g]) continue;
          const float* v = static_cast<const float*>(a.v) + int64_t(k0 + key) * a.kv_stride + int64_t(g) * a.D + (D / 2) * half;
#pragma unroll
          for (int i = 0; i < D / 2; ++i)
            if (i < cols && !(fabsf(v[i]) <= 3.402823466e38f)) o[i] += v[i];
        }
      const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
      for (int i = 0; i < D / 2; i += 4) {
        float r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = l == 0.0f ? 0.0f : o[i + e] / l;
        if (vec && i + 4 <= cols) {
          *reinterpret_cast<float4*>(out + i) = make_float4(r[0], r[1], r[2], r[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < cols) out[i + e] = r[e];
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
static int f3_launch(F3Args p, const uint8_t* q, const uint8_t* k, const uint8_t* v) {
  const AttnPromptArgs& a = p.a;
  p.tpt = 128 / a.rep;
  p.q = reinterpret_cast<const uint16_t*>(q);
  CUtensorMap mk, mv;
  if (int rc = attn_tensor_map(&mk, true, k, 3 * a.total_k, a.G, D, int64_t(a.G) * D, 1, F3Shape<D>::KEYS)) return rc;
  if (int rc = attn_tensor_map(&mv, true, v, 3 * a.total_k, a.G, D, int64_t(a.G) * D, 1, F3Shape<D>::KEYS)) return rc;
  auto kern = attn_prompt_f32_tc_kernel<D>;
  SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(F3Shape<D>::SMEM)));
  const int64_t units = std::min(a.total_q, a.total_q / p.tpt + a.n_seqs) * a.G;
  SIMP_REQUIRE(units <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many rows and heads");
  SIMP_CUDA(launch_kernel(kern, dim3(unsigned(units)), dim3(F3_THREADS), F3Shape<D>::SMEM, ctx().stream, true, mk, mv, p));
  return SIMP_OK;
}

// 1: the call stays with the FFMA kernel (nothing was launched).
int attn_prompt_f32_tc(const AttnPromptArgs& a) {
  if (a.total_k == 0 || 3 * a.total_q > INT_MAX || 3 * a.total_k > INT_MAX) return 1;
  const int D = a.D <= 64 ? 64 : 128;
  const size_t nq = size_t(a.total_q) * a.H, nk = size_t(a.total_k) * a.G, pad = 16;
  uint8_t* s = static_cast<uint8_t*>(scratch((nq + 2 * nk) * D * 6 + 4 * pad + nq + 2 * nk, SCRATCH_ATTN_PACK));
  if (!s) return attn_no_scratch();
  uint8_t *q = s, *k = q + nq * D * 6, *v = k + nk * D * 6, *any = v + nk * D * 6, *oq = any + pad, *ok = oq + nq, *ov = ok + nk;
  F3Args p{};
  p.a = a;
  p.any = reinterpret_cast<const int*>(any);
  p.odd_q = oq;
  p.odd_k = ok;
  p.odd_v = ov;
  int* flag = reinterpret_cast<int*>(any);
  SIMP_CUDA(cudaMemsetAsync(flag, 0, 4, ctx().stream));
  const AttnPack of_q{a.q, q, oq, a.total_q, a.q_stride, a.H}, of_k{a.k, k, ok, a.total_k, a.kv_stride, a.G}, of_v{a.v, v, ov, a.total_k, a.kv_stride, a.G};
  if (int rc = attn_pack(true, of_q, of_k, of_v, a.D, D, flag)) return rc;
  return D == 64 ? f3_launch<64>(p, q, k, v) : f3_launch<128>(p, q, k, v);
}

}  // namespace simp
