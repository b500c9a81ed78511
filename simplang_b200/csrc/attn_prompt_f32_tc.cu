// attn_prompt_f32_tc.cu -- causal attention over packed prompts at f32 accuracy on the tcgen05 tensor cores.
//
// q, k and v are split into three bf16 planes each (x = h + m + l, 24 bits), and a product is the six plane products of
// relative size 2^-16 and above: l.h, h.l, m.m, m.h, h.m, h.h.  The tensor cores add into their f32 accumulators with
// truncation, so (1) the small products come first and only the last eighth or less of the additions is made at full
// size, and (2) the output of every tile of keys is a sum of its own, added to f32 registers with rounding: an
// accumulator kept over a long prompt would drift by 2e-8 per instruction.
//
// One block of 18 warps per row tile (128 rows: 128 / rep tokens x the rep heads that share a key/value head):
//   warp 0      TMA: the planes of K and V per tile of 128 keys (96 KB each for head sizes above 64)
//   warp 1      MMAs: S = Q K^T, then T = P V, into TMEM
//   warps 2-17  softmax, four threads per row; P in three planes to TMEM; T into registers (D / 4 each)
// The planes of Q lie in TMEM, where they take no shared memory (and are not read from it again for every product: 6 KB per
// MMA of 64 keys, where it gives 128 bytes a cycle).  That leaves no TMEM for a second S, so P replaces S and softmax and
// MMAs take turns; only T is added up while the next scores are multiplied.  The form before had tiles of 64 keys, whose S
// and P lay apart, and overlapped the two: an MMA of 64 keys takes no less time than one of 96 (50 cycles, 75 beside the
// softmax), so it lost more than it won (4 prompts of 2048, 32 heads of 128: 1180 us, and 1020 in this form; of 100: 1265 and 985).
// With Q through shared memory and whole rows written these take 930 and 905 us.
// A step of 128 keys takes 10700 cycles: 4200 S (48 MMAs, 64 cycles each when nothing loads), 2650 softmax (1024 of them
// exponentials), 3100 T, the rest hand-overs.  Loading V later, when no MMA runs, costs more than it gives (1085 us).
// Head sizes up to 64 have half the MMAs for S and keep T apart for each plane of V, which lets one MMA multiply a plane of P
// with up to three planes of V side by side (25 MMAs of up to 192 columns instead of 48 of 64, which take no less than 96).
//
// No plane product of an infinity or a NaN is right, and a zero weight does not hide them from an MMA (a tile may hold keys
// that some rows must not see, or rows of the next sequence).  The splitting pass leaves them out of the planes and marks
// the row and head; where anything is marked, scores of marked rows are computed again from the f32 tensors, and marked
// values that a row sees are added to its output at the end.  Whoever does not see them gets the same bits as without.
#include <algorithm>
#include <climits>

#include "attn_tc.cuh"

namespace simp {

constexpr int F3_THREADS = 576;   // (five warps on some scheduler: 96 registers a thread)

template <int D>
struct F3Shape {
  static constexpr int KEYS = 128, ATOM = KEYS * 128;   // bytes of 64 elements of a tile's rows
  static constexpr int PLANE = KEYS * D * 2, STAGE = 3 * PLANE;
  static constexpr int BARS = 9;
  static constexpr size_t SMEM = 2 * size_t(STAGE) + BARS * 8 + 16 + 16 * 128 + 24;
  // TMEM columns: S, which the planes of P replace (192: see place_of_p), T (head sizes up to 64: three), three planes of Q
  static constexpr uint32_t T = 192, Q = T + (D == 64 ? 3 * 64 : 128);
  static_assert(Q + 3 * D / 2 <= 512 && SMEM <= 232448, "");
};
// TMEM columns of P for 16 keys (step 0 .. 7 of a tile) and a plane.  S is 128 columns, P 192: a thread that takes the scores
// of its 32 keys frees 32 columns for 48 that it writes, and touches no column of the row's other threads.
__host__ __device__ constexpr uint32_t place_of_p(int step, int plane) {
  const int part = step >> 1, b = 3 * (step & 1) + plane;
  return b < 2 ? 128u + 16u * part + 8u * b : 32u * part + 8u * (b - 2);
}

struct F3Args {
  AttnPromptArgs a;
  int tpt;
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
    attn_prompt_f32_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const F3Args p) {
  using Sh = F3Shape<D>;
  constexpr int KEYS = Sh::KEYS, MINE = 32;   // keys of a tile, of a thread
  extern __shared__ __align__(1024) uint8_t f3_raw[];
  const uint32_t base = smem_u32(f3_raw), k_smem = base, v_smem = base + Sh::STAGE, bars = base + 2 * Sh::STAGE;
  auto k_full = [&](int plane) { return bars + 8u * plane; };
  const uint32_t v_full = bars + 24, s_bar = bars + 32, p_bar = bars + 40, t_bar = bars + 48, q_bar = bars + 56, q_full = bars + 64;
  uint8_t* tail = f3_raw + 2 * Sh::STAGE + Sh::BARS * 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8);
  float* part_row = reinterpret_cast<float*>(tail + 16);   // [part][row]
  volatile int* found_unit = reinterpret_cast<volatile int*>(part_row + 4 * 128);   // found, place, q0, q1, k0, k1
  const AttnPromptArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {   // never: the declaration asks for it
    if (threadIdx.x == 0) report_status(a.status, 1, 70);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(k_full(i), 1);
    mbar_init(v_full, 1);
    mbar_init(s_bar, 1);
    mbar_init(p_bar, 16);
    mbar_init(t_bar, 1);
    mbar_init(q_bar, 16);
    mbar_init(q_full, 1);
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
  const int keys = sees(min(r0 + p.tpt, nq) - 1), n = (keys + KEYS - 1) / KEYS;
  auto steps = [&](int j) { return min(KEYS, keys - KEYS * j + 15) >> 4; };   // of 16 keys in tile j that some row sees

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0 && n > 0) {
      bool ok = true;
      auto boxes = [&](int j) { return steps(j) > 4 ? 2 : 1; };   // of 64 keys
      auto plane = [&](const CUtensorMap* map, uint32_t dst, uint32_t full, int s, int j) {
        for (int b = 0; b < D / 64; ++b)
          for (int i = 0; i < boxes(j); ++i)
            tma_load_3d(dst + s * Sh::PLANE + b * Sh::ATOM + i * (Sh::ATOM / 2), map, full, 64 * b, g, int(s * a.total_k) + k0 + KEYS * j + 64 * i);
      };
      // Q first, where V(0) will lie; from there the softmax warps take it to TMEM
      const int rows = p.tpt * a.rep;
      mbar_arrive_expect_tx(q_full, 3 * (D / 64) * rows * 128);
      for (int s = 0; s < 3; ++s)
        for (int b = 0; b < D / 64; ++b)
          tma_load_3d(v_smem + s * Sh::PLANE + b * Sh::ATOM, &map_q, q_full, 64 * b, g * a.rep, int(s * a.total_q) + q0 + r0);
      for (int j = 0; ok && j < n; ++j) {
        ok = j == 0 || wait_bar(s_bar, (j - 1) & 1, abort_flag, a.status, 71);
        if (!ok) break;
        for (int i = 0; i < 3; ++i) {
          const int s = i == 0 ? 0 : 3 - i;   // as the products need them
          mbar_arrive_expect_tx(k_full(s), boxes(j) * (Sh::PLANE / 2));
          plane(&map_k, k_smem, k_full(s), s, j);
        }
        ok = j == 0 ? wait_bar(q_bar, 0, abort_flag, a.status, 83) : wait_bar(t_bar, (j - 1) & 1, abort_flag, a.status, 82);
        if (!ok) break;
        mbar_arrive_expect_tx(v_full, boxes(j) * (Sh::STAGE / 2));
        for (int s = 0; s < 3; ++s) plane(&map_v, v_smem, v_full, s, j);
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);   // let copies in flight land before the block retires
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMAs (the whole warp with the same values, one lane issues)
    const int width = (a.D + 15) / 16;   // steps of 16 elements that hold something
    const bool leader = lane == 0;
    auto wait = [&](uint32_t bar, uint32_t phase, int site) {
      const bool ok = __all_sync(0xffffffffu, wait_bar(bar, phase, abort_flag, a.status, site));
      tc_fence_after_sync();
      return ok;
    };
    // planes of the two operands, small products first
    constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
    auto scores = [&](int j) {
      const uint32_t idesc = idesc_f16(true, 16 * steps(j), false);
      const uint64_t kd = make_smem_desc_sw128(k_smem, 16u, 1024u);
#pragma unroll
      for (int t = 0; t < 6; ++t) {
        if (j == 0 && t < 3 && !wait(k_full(PB[t]), 0, 73)) return false;   // (later ones have been waited for)
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          if (s < D / 32 || s < width)   // (an MMA that is not issued still costs its instructions, about as much as one that is)
            mma_f16_ts(tmem, tmem + Sh::Q + uint32_t(D / 2) * PA[t] + 8u * s, kd + uint64_t(PB[t] * (Sh::PLANE / 16) + (s >> 2) * (Sh::ATOM / 16) + (s & 3) * 2),
                       idesc, t > 0 || s > 0, leader);
      }
      if (leader) mma_commit(s_bar);
      return true;
    };
    const uint64_t vd = make_smem_desc_sw128(v_smem, uint32_t(Sh::ATOM), 1024u);   // [key][element]: 8 keys 1 KB apart
    auto product = [&](int step, int pa, int pb, uint32_t idesc, bool acc, bool issue) {   // P plane pa, V planes pb ..
      mma_f16_ts(tmem + Sh::T + (D == 64 ? 64u * pb : 0u), tmem + place_of_p(step, pa), vd + uint64_t(pb * (Sh::PLANE / 16) + step * 128), idesc, acc, leader && issue);
    };
    auto values = [&](int j) {
      const int have = steps(j);
      if constexpr (D == 64) {   // planes of V side by side: what one plane of P is multiplied with takes one MMA
        constexpr uint32_t ONE = idesc_f16(true, 64, true), TWO = idesc_f16(true, 128, true), ALL = idesc_f16(true, 192, true);
#pragma unroll
        for (int s = 0; s < 8; ++s) product(s, 1, 0, TWO, s > 0, s < have);
#pragma unroll
        for (int s = 0; s < 8; ++s) product(s, 2, 0, ONE, true, s < have);
        product(0, 0, 2, ONE, false, true);   // begins the third sum
        product(0, 0, 0, TWO, true, true);
#pragma unroll
        for (int s = 1; s < 8; ++s) product(s, 0, 0, ALL, true, s < have);
      } else {
        const uint32_t idesc = idesc_f16(true, 16 * width, true);
#pragma unroll
        for (int t = 0; t < 6; ++t)
#pragma unroll
          for (int s = 0; s < 8; ++s) product(s, PA[t], PB[t], idesc, t > 0 || s > 0, s < have);
      }
      if (leader) mma_commit(t_bar);
    };
    bool ok = n == 0 || wait(q_bar, 0, 72);
    for (int j = 0; ok && j < n; ++j) {
      ok = scores(j);   // behind the products that read the P before: MMAs of one thread run in order
      ok = ok && wait(v_full, j & 1, 76);
      for (int s = 0; ok && j + 1 < n && s < 3; ++s) ok = wait(k_full(s), (j + 1) & 1, 74);   // here nothing waits for it
      ok = ok && wait(p_bar, j & 1, 77);
      if (ok) values(j);
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and sums
    const int part = (warp - 2) >> 2, row = 32 * (warp & 3) + lane;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_tmem = tmem + lanes + uint32_t(MINE) * part, t_tmem = tmem + Sh::T + lanes + uint32_t(D / 4) * part;
    const int token = r0 + row / a.rep, head = g * a.rep + row % a.rep;
    const bool mine = row < p.tpt * a.rep && token < nq;
    const int lim = mine ? sees(token) : 0;
    volatile float* to = part_row + part * 128 + row;
    volatile float* all = part_row + row;
    bool ok = n == 0 || wait_bar(q_full, 0, abort_flag, a.status, 84);
    // this row's planes of Q, a quarter of a row per thread, to TMEM (16-byte pieces of a row lie in the order of the 128-byte swizzle;
    // read row by row from global memory this took 8000 cycles, a sixth of a block of five steps)
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const int piece = D / 32 * part;   // of 8 elements
      const uint8_t* src = f3_raw + Sh::STAGE + q * Sh::PLANE + (piece >> 3) * Sh::ATOM + row * 128;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {   // 16 elements
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + ((((piece & 7) + 2 * h + e) ^ (row & 7)) << 4));
          w[4 * e] = x.x; w[4 * e + 1] = x.y; w[4 * e + 2] = x.z; w[4 * e + 3] = x.w;
        }
        tmem_st_32x8(tmem + lanes + Sh::Q + uint32_t(D / 2) * q + uint32_t(D / 8) * part + 8u * h, w);
      }
    }
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_bar);
    const bool any = __ldcg(p.any) != 0, odd_row = any && mine && p.odd_q[int64_t(q0 + token) * a.H + head];
    float m = -INFINITY, l = 0.0f, alpha = 0.0f, o[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; ++i) o[i] = 0.0f;
    auto add_tile = [&] {   // the sum of the last tile to the registers, which its maximum has not reached yet
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint32_t t[16];
        tmem_ld_32x16(t_tmem + 16u * h, t);
        if constexpr (D == 64) {
          uint32_t t1[16], t2[16];
          tmem_ld_32x16(t_tmem + 64u + 16u * h, t1);
          tmem_ld_32x16(t_tmem + 128u + 16u * h, t2);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = __float_as_uint(__uint_as_float(t[i]) + (__uint_as_float(t1[i]) + __uint_as_float(t2[i])));
        } else {
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[16 * h + i] = fmaf(o[16 * h + i], alpha, __uint_as_float(t[i]));
      }
    };
    const f2 c2 = pack_f2(a.scale_log2, a.scale_log2), none = 0;
    for (int j = 0; j < n; ++j) {
      if (j > 0) {   // while the scores are multiplied
        ok = __all_sync(0xffffffffu, wait_bar(t_bar, (j - 1) & 1, abort_flag, a.status, 79)) && ok;
        tc_fence_after_sync();
        add_tile();
      }
      ok = wait_bar(s_bar, j & 1, abort_flag, a.status, 78) && ok;
      tc_fence_after_sync();
      if (any) {   // rare: scores of rows that are not finite, by the f32 tensors
#pragma unroll 1
        for (int i = 0; i < MINE; ++i) {
          const int key = KEYS * j + MINE * part + i;
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
      const int see = lim - KEYS * j - MINE * part, chunks = steps(j) - 2 * part;   // of 16 keys
      const bool masked = __any_sync(0xffffffffu, see < MINE);
      const int most = masked ? __reduce_max_sync(0xffffffffu, see) : MINE;   // keys behind it no row of the warp sees
      float t[2] = {-INFINITY, -INFINITY};
      uint32_t s[MINE];
      tmem_ld_32x32(s_tmem, s);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < MINE; i += 2) {
        const f2 y = fma_f2(pack_f2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2, none);
        s[i] = uint32_t(y);
        s[i + 1] = uint32_t(y >> 32);
      }
      if (masked)
#pragma unroll
        for (int i = 0; i < MINE; ++i) s[i] = i < see ? s[i] : 0xff800000u;
#pragma unroll
      for (int i = 0; i < MINE; i += 2) t[(i >> 1) & 1] = max3(t[(i >> 1) & 1], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
      *to = fmaxf(t[0], t[1]);
      ok = all_of(1 + (warp & 3), 128, ok);
      if (!ok) break;
      const float top = fmaxf(max3(all[0], all[128], all[256]), all[384]);
      const float mn = fmaxf(m, top), off = mn == -INFINITY ? 0.0f : mn;
      alpha = ex2(m - off);   // 0 for the first tile
      m = mn;
      const f2 off2 = pack_f2(-off, -off), minus = pack_f2(-1.0f, -1.0f);
      f2 sum[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < 4; ++h) {   // 8 keys
        if ((h >> 1) >= chunks) break;
        uint32_t w[3][4];
        if (8 * h >= most) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[0][i] = w[1][i] = w[2][i] = 0u;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f2 y = add_f2(pack_f2(__uint_as_float(s[8 * h + 2 * i]), __uint_as_float(s[8 * h + 2 * i + 1])), off2);
            const f2 e = pack_f2(ex2(lo_f2(y)), ex2(hi_f2(y)));
            sum[i & 1] = add_f2(sum[i & 1], e);
            auto plane = [&](f2 x) { return pack2<true>(lo_f2(x), hi_f2(x)); };
            auto less = [&](f2 x, uint32_t p2) { return fma_f2(pack_f2(__uint_as_float(p2 << 16), __uint_as_float(p2 & 0xffff0000u)), minus, x); };   // exact
            w[0][i] = plane(e);
            const f2 f = less(e, w[0][i]);
            w[1][i] = plane(f);
            w[2][i] = plane(less(f, w[1][i]));
          }
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) tmem_st_32x4(tmem + lanes + place_of_p(2 * part + (h >> 1), q) + 4u * (h & 1), w[q]);
      }
      sum[0] = add_f2(sum[0], sum[1]);
      l = fmaf(l, alpha, lo_f2(sum[0]) + hi_f2(sum[0]));
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_bar);
    }
    if (ok && n > 0) {
      ok = __all_sync(0xffffffffu, wait_bar(t_bar, (n - 1) & 1, abort_flag, a.status, 80));
      tc_fence_after_sync();
      add_tile();
    }
    *to = l;
    ok = all_of(1 + (warp & 3), 128, ok);
    if (ok) {
      l = (all[0] + all[128]) + (all[256] + all[384]);
      const int cols = a.D - (D / 4) * part;
      if (any && mine)
#pragma unroll 1
        for (int key = 0; key < lim; ++key) {
          if (!p.odd_v[int64_t(k0 + key) * a.G + g]) continue;
          const float* v = static_cast<const float*>(a.v) + int64_t(k0 + key) * a.kv_stride + int64_t(g) * a.D + (D / 4) * part;
#pragma unroll
          for (int i = 0; i < D / 4; ++i)
            if (i < cols && !(fabsf(v[i]) <= 3.402823466e38f)) o[i] += v[i];
        }
      // By way of shared memory (K's place: every MMA is done), so that a warp writes whole rows: 16 bytes of 32 rows at a time
      // took 5000 cycles.  Rows there are 16 bytes apart in their banks.
      constexpr int PITCH = D + 4;
      float* rows = reinterpret_cast<float*>(f3_raw);
      static_assert(128 * PITCH * 4 <= Sh::STAGE, "");
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int i = 0; i < D / 4; i += 4) {
        float r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = l == 0.0f ? 0.0f : o[i + e] * inv;
        *reinterpret_cast<float4*>(rows + row * PITCH + (D / 4) * part + i) = make_float4(r[0], r[1], r[2], r[3]);
      }
      all_of(1 + (warp & 3), 128, true);
      const bool vec = a.D % 4 == 0 && a.out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
      const int first = 32 * (warp & 3) + 8 * part;
      int to_token = r0 + first / a.rep, to_head = first % a.rep;
#pragma unroll 1
      for (int at = first; at < min(first + 8, p.tpt * a.rep) && to_token < nq; ++at) {
        float* out = static_cast<float*>(a.out) + int64_t(q0 + to_token) * a.out_stride + int64_t(g * a.rep + to_head) * a.D;
        const float* from = rows + at * PITCH;
        if (vec) {
          if (4 * lane < a.D) *reinterpret_cast<float4*>(out + 4 * lane) = *reinterpret_cast<const float4*>(from + 4 * lane);
        } else {
          for (int d = lane; d < a.D; d += 32) out[d] = from[d];
        }
        if (++to_head == a.rep) to_head = 0, ++to_token;
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
  CUtensorMap mq, mk, mv;
  if (int rc = attn_tensor_map(&mq, true, q, 3 * a.total_q, a.H, D, int64_t(a.H) * D, a.rep, p.tpt)) return rc;
  if (int rc = attn_tensor_map(&mk, true, k, 3 * a.total_k, a.G, D, int64_t(a.G) * D, 1, 64)) return rc;
  if (int rc = attn_tensor_map(&mv, true, v, 3 * a.total_k, a.G, D, int64_t(a.G) * D, 1, 64)) return rc;
  auto kern = attn_prompt_f32_tc_kernel<D>;
  SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(F3Shape<D>::SMEM)));
  const int64_t units = std::min(a.total_q, a.total_q / p.tpt + a.n_seqs) * a.G;
  SIMP_REQUIRE(units <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many rows and heads");
  SIMP_CUDA(launch_kernel(kern, dim3(unsigned(units)), dim3(F3_THREADS), F3Shape<D>::SMEM, ctx().stream, true, mq, mk, mv, p));
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
