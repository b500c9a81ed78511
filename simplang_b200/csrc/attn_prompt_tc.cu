// attn_prompt_tc.cu -- causal attention over packed prompts on the tcgen05 tensor cores: f16 / bf16, head size 64 or 128.
//
// One block works on two row tiles ("A" and "B"; short prompts: one) of one key/value head of one sequence.  A row tile is 128 rows
// of the score matrix: 128 / rep consecutive tokens times the rep query heads that share the key/value head (row = token *
// rep + head), so grouped heads read K and V once, short prompts fill tiles and the causal edge is fine.  Roles:
//   warp 0          TMA: Q once, then K and V tiles of 128 keys through a ring of slots
//   warps 1, 2      issue the MMAs of tile A, of tile B: S = Q K^T (128 x 128, f32 in TMEM), O += P V with P read from TMEM.
//                   Issuing blocks while the tensor cores are busy, so one thread for both would leave them idle at its waits
//   warp 3          cleans the V tiles at the causal / ragged edge (see below)
//   warps 4-11, 12-19  softmax of tile A, of tile B: two threads per row, 64 keys each, which exchange their maxima
// P (16 bits) overwrites S in place: S_X(j + 1) is issued behind O_X += P_X(j) V(j) by the same thread, whose MMAs run in order.
// While the tensor cores work on one tile, the other tile's softmax runs: 2 x 128 x 128 x D MACs take 4 D cycles per tile and
// step, its 16384 exponentials 1024.  Measured for D = 128 (one prompt of 8192, 32 / 8 heads: 536 us, 1026 TFLOP/s, 0.63 of
// the measured rate): both tiles' steps take 3800 cycles, a tile's chain of 1700 softmax, 200 maxima, 100 P, 250 hand-over,
// 1250 MMAs and 250 hand-over back.  The tensor cores and the exponentials are each busy a little over half of the time; the
// softmax is held up by its two warps per scheduler issuing in order (exponentials in polynomial form on the FMA pipe cost
// more issue slots than they save: an eighth of them 564 us, a quarter 577).
//
// Softmax: the row's running maximum moves only when a tile exceeds it by more than 2^8 (weights are then at most 2^8, well
// inside f16), so O is rarely rescaled: it stays in TMEM.  S_X(j + 1) being complete implies that P_X(j) V(j) is, so the
// softmax warps may rescale O_X without another barrier.
//
// A weight of zero does not hide a NaN or an infinity from an MMA, and a tile may hold keys that some rows must not see:
// later tokens of the sequence, and rows of the NEXT sequence (or behind the last) where the sequence ends inside the tile.
// Warp 3 therefore zeroes, in the edge tiles only, V rows behind the sequence and every element that is not finite; a bit
// per such key tells the epilogue to add those elements (read again from global memory) to the rows that do see the key.
#include <algorithm>
#include <climits>
#include <cstring>
#include <type_traits>

#include "attn_tc.cuh"

namespace simp {

constexpr int W_LOAD = 0, W_MMA = 1, W_EDGE = 3;   // W_MMA: tile A, W_MMA + 1: tile B; 4 .. 19: softmax
constexpr int TC_EDGE = 4;   // edge tiles of a block: its rows see at most 255 keys more than its first row, so 3

// whether one of eight 16-bit elements is infinity or NaN: one more in the exponent then reaches the sign's place
template <bool BF16>
__device__ __forceinline__ bool any_odd(const uint4& w) {
  constexpr uint32_t E = BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = BF16 ? 0x00800080u : 0x04000400u;
  return ((((w.x & E) + ONE) | ((w.y & E) + ONE) | ((w.z & E) + ONE) | ((w.w & E) + ONE)) & 0x80008000u) != 0;
}
template <bool BF16>
__device__ __forceinline__ float to_16(uint16_t v) {
  return BF16 ? __uint_as_float(uint32_t(v) << 16) : __half2float(__ushort_as_half(v));
}

// TILES = 2: one block per SM, whose tiles take turns on the tensor cores.  TILES = 1: two blocks per SM, so that one works
// while the other starts, loads its first tiles or writes its output.
template <int D, int TILES>
struct TcShape {
  static constexpr int THREADS = 128 + 256 * TILES;
  static constexpr int TILE = 128 * D * 2;              // bytes of 128 rows
  static constexpr int SLOTS = TILES == 2 ? (D == 128 ? 5 : 8) : (D == 128 ? 2 : 4);
  static constexpr int BARS = 2 * SLOTS + 1 + 6 + TC_EDGE;
  static constexpr uint32_t TMEM = TILES == 2 ? 512 : 256, O = 128 * TILES;   // columns: S of each tile, then O of each
  // (1 KB of the SM's 228 belongs to the system for each block)
  static constexpr size_t SMEM = size_t(TILES + SLOTS) * TILE + BARS * 8 + 16 + TC_EDGE * 16 + 2 * TILES * 128 * 4 + 24;
  static_assert((3 - TILES) * (SMEM + 1024) <= 228 * 1024, "");
};

struct TcArgs {
  AttnPromptArgs a;
  int tpt;          // tokens per row tile
  const void* q;    // what the maps read: the caller's tensors, or copies padded to D elements per head
  const void* k;
  const void* v;
  int64_t q_stride, kv_stride;
  int chunk;        // elements of an output row that are written together: 8, 4 or 1, by its alignment and head size
};

// bits of the 16-bit halves of w that are infinity or NaN
template <bool BF16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}

template <bool BF16, int D, int TILES>
__global__ void __launch_bounds__(128 + 256 * TILES, 3 - TILES)
    attn_prompt_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const TcArgs p) {
  using Sh = TcShape<D, TILES>;
  extern __shared__ __align__(1024) uint8_t tc_raw[];   // swizzled tiles start on 1 KB boundaries
  const uint32_t base = smem_u32(tc_raw);
  const uint32_t q_smem = base, ring = base + TILES * Sh::TILE, bars = ring + Sh::SLOTS * Sh::TILE;
  uint8_t* generic = tc_raw;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (Sh::SLOTS + s); };
  const uint32_t q_bar = bars + 8u * (2 * Sh::SLOTS);
  auto s_bar = [&](int x) { return q_bar + 8u + 8u * x; };
  auto p_bar = [&](int x) { return q_bar + 24u + 8u * x; };
  auto o_bar = [&](int x) { return q_bar + 40u + 8u * x; };
  auto edge_bar = [&](int e) { return q_bar + 56u + 8u * e; };
  uint8_t* tail = generic + (bars - base) + Sh::BARS * 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8);
  uint32_t* odd_keys = reinterpret_cast<uint32_t*>(tail + 16);   // [TC_EDGE][4]: keys of edge tiles with an element that is not finite
  float* half_row = reinterpret_cast<float*>(tail + 16 + TC_EDGE * 16);   // [tile][half][row]: what the two threads of a row exchange
  volatile int* found_unit = reinterpret_cast<volatile int*>(half_row + 2 * TILES * 128);   // found, place, q0, q1, k0, k1
  const AttnPromptArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (base & 1023u) {   // never: the declaration asks for it
    if (threadIdx.x == 0) report_status(a.status, 1, 60);
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::SLOTS; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), TILES);
    }
    mbar_init(q_bar, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_bar(x), 1);
      mbar_init(p_bar(x), 9);
      mbar_init(o_bar(x), 1);
    }
    for (int e = 0; e < TC_EDGE; ++e) mbar_init(edge_bar(e), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < TC_EDGE * 4) odd_keys[threadIdx.x] = 0;

  pdl_launch_dependents();
  pdl_wait();
  // ---- which rows: found by one warp while the others prepare
  const int g = blockIdx.x % a.G;
  const int rows_cta = TILES * p.tpt;
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  if (warp == W_LOAD) {
    auto count = [&](int s) {
      int b, e;
      return seq_range(a.q_off, s, a.total_q, a.status, b, e) ? (e - b + rows_cta - 1) / rows_cta : 0;
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
  if (warp == W_MMA) {
    tmem_alloc(smem_u32(tmem_slot), Sh::TMEM);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = TILES == 2 ? 0u : *tmem_slot;   // a block that allocates every column starts at 0
  if (!found_unit[0]) {
    if (warp == W_MMA) tmem_dealloc(tmem, Sh::TMEM);
    return;
  }
  q0 = found_unit[2];
  q1 = found_unit[3];
  k0 = found_unit[4];
  k1 = found_unit[5];
  int place = found_unit[1];
  const int nq = q1 - q0, nk = k1 - k0;
  place = (nq + rows_cta - 1) / rows_cta - 1 - place;   // the longest rows first
  const int r0 = place * rows_cta;                      // first token of tile A
  const int64_t shift = int64_t(nk) - nq;               // token i sees keys j <= i + shift
  auto sees = [&](int token) { return int(max(int64_t(0), min(int64_t(nk), token + shift + 1))); };
  int n_x[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = r0 + x * p.tpt, last = min(first + p.tpt, nq) - 1;
    n_x[x] = x < TILES && first < nq ? (sees(last) + 127) >> 7 : 0;
  }
  const int n = max(n_x[0], n_x[1]);
  const int edge0 = sees(r0) >> 7;                      // tiles from here on hold a key that some row does not see

  // ------------------------------------------------------------------ MMAs of tile X
  // The whole warp runs this code with the same values and one lane issues; x, the TMEM columns (of a block that has all 512)
  // and the descriptors' bases are constants.  Operands of an MMA then live in uniform registers; from
  // general ones each costs several more instructions, and the warp shares its scheduler with the softmax of the other
  // tile, which leaves few slots (beside warps that issue nothing but FFMA an MMA took 113-130 cycles instead of 64).
  auto mma_role = [&](auto which) {
    constexpr int x = decltype(which)::value;
    const int mine = n_x[x], other = n_x[x ^ 1];
    const int steps = max(mine, other);
    const bool leader = lane == 0;
    auto wait = [&](uint32_t bar, uint32_t phase, int site) {
      const bool ok = __all_sync(0xffffffffu, wait_bar(bar, phase, abort_flag, a.status, site));
      tc_fence_after_sync();
      return ok;
    };
    auto commit = [&](uint32_t bar) {
      if (leader) mma_commit(bar);
    };
    constexpr uint32_t idesc_s = idesc_f16(BF16, 128, false), idesc_o = idesc_f16(BF16, D, true);
    const uint32_t s_tmem = tmem + 128u * x, o_tmem = tmem + Sh::O + uint32_t(D) * x;
    const uint64_t qd = make_smem_desc_sw128(q_smem + x * Sh::TILE, 16u, 1024u);
    const uint64_t ring_k = make_smem_desc_sw128(ring, 16u, 1024u);
    // V [key][element]: element-major operand, 64-element atoms 16 KB apart, 8 keys 1 KB apart
    const uint64_t ring_v = make_smem_desc_sw128(ring, 16384u, 1024u);
    auto scores = [&](int slot) {
      const uint64_t kd = ring_k + uint64_t(slot * (Sh::TILE / 16));
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {   // 16 elements = 32 bytes; the next 64 elements lie 16 KB further
        const uint64_t o = uint64_t((s >> 2) * 1024 + (s & 3) * 2);
        mma_f16_ss(s_tmem, qd + o, kd + o, idesc_s, s > 0, leader);
      }
    };
    auto values = [&](int slot, bool first) {
      const uint64_t vd = ring_v + uint64_t(slot * (Sh::TILE / 16));
#pragma unroll
      for (int s = 0; s < 8; ++s)          // 16 keys = 8 columns of P, 2 KB of V
        mma_f16_ts(o_tmem, s_tmem + 8u * s, vd + uint64_t(s * 128), idesc_o, !(first && s == 0), leader);
    };
    bool ok = true;
    int slot = 0;            // of K(j), then of V(j): slots are taken in the order K(0) V(0) K(1) ...
    uint32_t phase = 0;
    auto next = [&] {
      if (++slot == Sh::SLOTS) slot = 0, phase ^= 1u;
    };
    if (mine > 0) {
      ok = wait(q_bar, 0, 63) && wait(full_bar(0), 0, 62);
      if (ok) {
        scores(0);
        commit(s_bar(x));
        commit(empty_bar(0));
        if (leader && (x == 0 || other == 0)) mbar_arrive(p_bar(x));   // the first turn
      }
      next();
      for (int j = 0; ok && j < mine; ++j) {
        const bool more = j + 1 < mine;
        const int v_slot = slot;
        ok = wait(full_bar(v_slot), phase, 62);
        next();
        if (ok && more) ok = wait(full_bar(slot), phase, 62);
        // The weights are there and it is this tile's turn: A B A B ...  Were the tiles' MMAs mixed, both would end late and
        // both softmaxes run while the tensor cores idle.  The ninth arrival at the barrier is the other tile's thread
        // passing the turn on, or this one where the other tile has no such step.
        if (ok) ok = wait(p_bar(x), j & 1, 65);
        if (!ok) break;
        values(v_slot, j == 0);
        if (more) scores(slot);
        if (leader) {
          const int next = x == 0 ? j : j + 1;   // the other tile's step whose turn it is now, if there is one
          if (next < other) mbar_arrive(p_bar(x ^ 1));
          else if (more) mbar_arrive(p_bar(x));
        }
        commit(more ? s_bar(x) : o_bar(x));
        commit(empty_bar(v_slot));
        if (more) {
          commit(empty_bar(slot));
          next();
        }
      }
    }
    // slots that only the other tile works on
    for (int i = 2 * mine; ok && i < 2 * steps; ++i) {
      ok = wait(full_bar(slot), phase, 62);
      if (ok && leader) mbar_arrive(empty_bar(slot));
      next();
    }
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncwarp();
  };

  if (warp == W_LOAD) {
    // ------------------------------------------------------------------ loads
    if (lane == 0 && n > 0) {
      const int tiles = TILES == 2 && r0 + p.tpt < nq ? 2 : 1;
      const uint32_t box = uint32_t(p.tpt * a.rep) * 128u;
      mbar_arrive_expect_tx(q_bar, tiles * (D / 64) * box);
      for (int x = 0; x < tiles; ++x)
        for (int b = 0; b < D / 64; ++b)
          tma_load_3d(q_smem + x * Sh::TILE + b * 16384, &map_q, q_bar, 64 * b, g * a.rep, q0 + r0 + x * p.tpt);
      bool ok = true;
      for (int i = 0; ok && i < 2 * n; ++i) {
        const int s = i % Sh::SLOTS;
        if (!wait_bar(empty_bar(s), ((i / Sh::SLOTS) & 1) ^ 1, abort_flag, a.status, 61)) { ok = false; break; }
        const bool edge = (i & 1) && (i >> 1) >= edge0;   // lands for warp 3, which passes the slot on
        const uint32_t bar = edge ? edge_bar((i >> 1) - edge0) : full_bar(s);
        mbar_arrive_expect_tx(bar, Sh::TILE);
        for (int b = 0; b < D / 64; ++b)
          tma_load_3d(ring + s * Sh::TILE + b * 16384, i & 1 ? &map_v : &map_k, bar, 64 * b, g, k0 + 128 * (i >> 1));
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);   // let copies in flight land before the block retires
    }
    __syncwarp();
  } else if (warp == W_MMA) {
    mma_role(std::integral_constant<int, 0>());
  } else if (warp == W_MMA + 1) {
    if (TILES == 2) mma_role(std::integral_constant<int, 1>());
  } else if (warp == W_EDGE) {
    // ------------------------------------------------------------------ V at the edge
    for (int j = edge0; j < n; ++j) {
      const int i = 2 * j + 1;
      if (!wait_bar(edge_bar(j - edge0), 0, abort_flag, a.status, 66)) break;
      uint8_t* v = generic + TILES * Sh::TILE + (i % Sh::SLOTS) * Sh::TILE;
      const int keys = min(nk - 128 * j, 128);          // rows from here on are not the sequence's
      const int all_see = max(sees(r0) - 128 * j, 0);   // every row sees the keys before: nothing to hide
      // (the 128-byte swizzle moves 16-byte pieces inside a row only, so rows are found as if there were none)
#pragma unroll 1
      for (int b = 0; b < D / 64; ++b) {
        uint4* atom = reinterpret_cast<uint4*>(v + b * 16384);
#pragma unroll 1
        for (int c = 8 * keys + lane; c < 1024; c += 32) atom[c] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
        for (int c0 = 8 * all_see; c0 < 8 * keys; c0 += 256) {
          uint4 w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = c0 + 32 * e + lane < 8 * keys ? atom[c0 + 32 * e + lane] : make_uint4(0u, 0u, 0u, 0u);
          uint32_t found = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) found |= any_odd<BF16>(w[e]) ? 1u << e : 0u;
          if (found)
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
              if (!((found >> e) & 1u)) continue;
              const int c = c0 + 32 * e + lane, key = c >> 3;
              const uint4 o = atom[c];
              atom[c] = make_uint4(o.x & ~odd_halves<BF16>(o.x), o.y & ~odd_halves<BF16>(o.y), o.z & ~odd_halves<BF16>(o.z), o.w & ~odd_halves<BF16>(o.w));
              atomicOr(odd_keys + (j - edge0) * 4 + (key >> 5), 1u << (key & 31));
            }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full_bar(i % Sh::SLOTS));
    }
  } else {
    // ------------------------------------------------------------------ softmax
    const int x = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_tmem = tmem + 128u * x + lanes, o_tmem = tmem + Sh::O + uint32_t(D) * x + uint32_t(D / 2) * half + lanes;
    const int token = r0 + x * p.tpt + row / a.rep, head = g * a.rep + row % a.rep;
    const bool mine = row < p.tpt * a.rep && token < nq;
    const int lim = mine ? sees(token) : 0;
    const float c = a.scale_log2;
    volatile float* to = half_row + (2 * x + half) * 128 + row;
    volatile float* from = half_row + (2 * x + (half ^ 1)) * 128 + row;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const f2 c2 = pack_f2(c, c);
    for (int j = 0; j < n_x[x]; ++j) {
      ok = wait_bar(s_bar(x), j & 1, abort_flag, a.status, 67);
      tc_fence_after_sync();
      const int see = lim - 128 * j - 64 * half;
      const bool masked = __any_sync(0xffffffffu, see < 64);
      const int most = masked ? __reduce_max_sync(0xffffffffu, see) : 64;   // keys behind it no row of the warp sees
      // Weights relative to the maximum so far, and this tile's maximum beside them: the maximum nearly always stays, so the
      // exponentials need not wait for it.  Where it moves, once more with the new one; S is still there, P is not stored before
      // the row's two threads agree.
      for (int attempt = j == 0 ? -1 : 0;; attempt = 1) {
        if (attempt < 0) {   // the first tile: nothing to go by, so its maximum first
          float t[2] = {-INFINITY, -INFINITY};
          uint32_t s[2][16];
          tmem_ld_32x16(s_tmem + 64u * half, s[0]);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            tmem_ld_wait();
            if (h < 3) tmem_ld_32x16(s_tmem + 64u * half + 16u * (h + 1), s[(h + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float s0 = 16 * h + i < see ? __uint_as_float(s[h & 1][i]) : -INFINITY, s1 = 16 * h + i + 1 < see ? __uint_as_float(s[h & 1][i + 1]) : -INFINITY;
              t[h & 1] = max3(t[h & 1], s0, s1);
            }
          }
          const float top = fmaxf(t[0], t[1]);
          *to = top;
          ok = all_of(1 + 4 * x + (warp & 3), 64, ok);
          if (!ok) break;
          m = fmaxf(top, *from) * c;
          continue;
        }
        const float off = m == -INFINITY ? 0.0f : m;
        const f2 off2 = pack_f2(-off, -off);
        float t[2] = {-INFINITY, -INFINITY};
        f2 sum[2] = {0, 0};
        uint32_t s[2][16], w[32];   // 16 scores at a time, the next 16 on their way: room for exponentials in flight
        // Tiles that every row sees have a form without branches where heads of 64 leave the softmax alone on the critical path
        // (8192 tokens, 32 / 8 heads: 497 -> 465 us).  Heads of 128: 543 -> 526 us there, but 113 -> 118 for 16 prompts of 512
        // and 146 -> 149 for 8 of 1024, whose blocks go through the code of both forms for few tiles each.
        auto weigh = [&](auto all_seen) {
          constexpr bool ALL = decltype(all_seen)::value;
          tmem_ld_32x16(s_tmem + 64u * half, s[0]);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t(&v)[16] = s[h & 1];
            tmem_ld_wait();
            if (!ALL && 16 * h >= most) {
#pragma unroll
              for (int i = 0; i < 8; ++i) w[8 * h + i] = 0u;
              continue;
            }
            if (h < 3) tmem_ld_32x16(s_tmem + 64u * half + 16u * (h + 1), s[(h + 1) & 1]);
            if (!ALL && masked) {
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = 16 * h + i < see ? v[i] : 0xff800000u;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              t[i & 1] = max3(t[i & 1], __uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              const f2 y = fma_f2(pack_f2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), c2, off2);
              const f2 e = pack_f2(ex2(lo_f2(y)), ex2(hi_f2(y)));
              sum[i & 1] = add_f2(sum[i & 1], e);
              w[8 * h + i] = pack2<BF16>(lo_f2(e), hi_f2(e));
            }
          }
        };
        if constexpr (D == 64 && TILES == 2) {
          if (masked) weigh(std::false_type());
          else weigh(std::true_type());
        } else {
          weigh(std::false_type());
        }
        float top = fmaxf(t[0], t[1]);
        if (attempt == 0) *to = top;
        ok = all_of(1 + 4 * x + (warp & 3), 64, ok);   // behind this point both halves have read S
        if (!ok) break;
        if (attempt == 0) top = fmaxf(top, *from) * c;
        if (attempt == 0 && __any_sync(0xffffffffu, top > m + 8.0f)) {
          const float mn = fmaxf(m, top), alpha = m == mn ? 1.0f : ex2(m - mn);
          l *= alpha;
          m = mn;
          if (j > 0) {
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {   // this half's elements, 16 at a time
              uint32_t o[16];
              tmem_ld_32x16(o_tmem + 16u * h, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x16(o_tmem + 16u * h, o);
            }
          }
          continue;
        }
        tmem_st_32x32(s_tmem + 32u * half, w);
        sum[0] = add_f2(sum[0], sum[1]);
        l += lo_f2(sum[0]) + hi_f2(sum[0]);
        break;
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_bar(x));
    }
    if (ok && n_x[x] > 0) ok = wait_bar(o_bar(x), 0, abort_flag, a.status, 68);
    *to = l;
    ok = all_of(1 + 4 * x + (warp & 3), 64, ok);
    // Heads of 128 leave by way of shared memory (the place of this tile's Q, which no MMA reads any more), so that a warp writes
    // whole rows; 16-byte pieces of a row lie in another order per row, for the banks.  bf16, 32 / 8 heads: 64 prompts of 128
    // tokens 88 -> 80 us, 8 of 1024 144 -> 138.  Heads of 64, whose threads have 64 bytes in a row: 113 -> 117, so they do not.
    constexpr bool STAGED = D == 128;
    if (STAGED && ok && n > 0) ok = all_of(1 + 4 * x + (warp & 3), 64, wait_bar(q_bar, 0, abort_flag, a.status, 69));   // (a tile that sees nothing)
    if (ok) {
      tc_fence_after_sync();
      l += *from;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint8_t* const stage = generic + x * Sh::TILE;
      auto piece = [&](int r, int c) { return stage + r * (2 * D) + ((c ^ (r & 7)) << 4); };
      auto row_of = [&](int of, int h) { return static_cast<uint8_t*>(a.out) + (int64_t(q0 + of) * a.out_stride + int64_t(h) * a.D) * 2; };
      uint8_t* const out = row_of(token, head) + D * half;
      auto write = [&](uint8_t* at, const uint4& w, int left) {   // `left` elements from here to the head's end
        if (p.chunk == 8) {
          if (left > 0) *reinterpret_cast<uint4*>(at) = w;
        } else if (p.chunk == 4) {
          if (left > 0) *reinterpret_cast<uint2*>(at) = make_uint2(w.x, w.y);
          if (left > 4) *reinterpret_cast<uint2*>(at + 8) = make_uint2(w.z, w.w);
        } else {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(&w);
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (t < left) reinterpret_cast<uint16_t*>(at)[t] = e[t];
        }
      };
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint32_t o[32];
        if (n_x[x] > 0) {
          tmem_ld_32x32(o_tmem + 32u * h, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = l == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 w;
          w.x = pack2<BF16>(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1]));
          w.y = pack2<BF16>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]));
          w.z = pack2<BF16>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]));
          w.w = pack2<BF16>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
          if (STAGED) *reinterpret_cast<uint4*>(piece(row, D / 16 * half + 4 * h + i)) = w;
          else if (mine) write(out + 64 * h + 16 * i, w, a.D - ((D / 2) * half + 32 * h + 8 * i));
        }
        __syncwarp();
      }
      uint32_t odd = 0;
      for (int e = 0; e < TC_EDGE * 4; ++e) odd |= odd_keys[e];
      if (odd && mine) {   // rare: what the edge tiles' V has that is not finite, to the rows that see it
        const int cols = min(D / 2, a.D - (D / 2) * half);
#pragma unroll 1
        for (int key = 128 * edge0; key < lim; ++key) {
          if (!((odd_keys[(key - 128 * edge0) >> 5] >> (key & 31)) & 1u)) continue;
          const uint16_t* v = static_cast<const uint16_t*>(a.v) + int64_t(k0 + key) * a.kv_stride + int64_t(g) * a.D + (D / 2) * half;
#pragma unroll 1
          for (int i = 0; i < cols; ++i)
            if (odd_halves<BF16>(v[i]) & 0xffffu) {
              uint16_t& o16 = reinterpret_cast<uint16_t*>(STAGED ? piece(row, D / 16 * half + (i >> 3)) : out + 16 * (i >> 3))[i & 7];
              o16 = uint16_t(pack2<BF16>(to_16<BF16>(o16) + to_16<BF16>(v[i]), 0.0f));
            }
        }
      }
      if constexpr (STAGED) {
        all_of(1 + 4 * x + (warp & 3), 64, true);
        const int c = lane & 15;
        const uint32_t share = 65536u / uint32_t(a.rep) + 1u;   // r * share / 65536 is r / rep for r < 128
#pragma unroll 2
        for (int i = 0; i < 16; i += 2) {
          const int r = 32 * (warp & 3) + 16 * half + i + (lane >> 4), rt = int(uint32_t(r) * share >> 16), to_token = r0 + x * p.tpt + rt;
          if (r < p.tpt * a.rep && to_token < nq)
            write(row_of(to_token, g * a.rep + r - rt * a.rep) + 16 * c, *reinterpret_cast<const uint4*>(piece(r, c)), a.D - 8 * c);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, Sh::TMEM);
  }
}

int attn_tensor_map(CUtensorMap* map, bool bf16, const void* p, int64_t rows, int64_t heads, int D, int64_t stride, int box_heads, int box_rows) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode enc = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) sym = nullptr;
    return reinterpret_cast<Encode>(sym);
  }();
  SIMP_REQUIRE(enc != nullptr, SIMP_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(rows)};
  const cuuint64_t strides[2] = {cuuint64_t(D) * 2, cuuint64_t(stride) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_rows)}, one[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  SIMP_REQUIRE(r == CUDA_SUCCESS, SIMP_ERR_CUDA, "cuTensorMapEncodeTiled (attn_prompt) failed with CUresult %d", int(r));
  return SIMP_OK;
}

template <bool BF16, int D, int TILES>
static int tc_run(const TcArgs& p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv) {
  using Sh = TcShape<D, TILES>;
  const AttnPromptArgs& a = p.a;
  auto kern = attn_prompt_tc_kernel<BF16, D, TILES>;
  SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Sh::SMEM)));
  const int64_t units = std::min(a.total_q, a.total_q / (TILES * p.tpt) + a.n_seqs) * a.G;
  SIMP_REQUIRE(units <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many rows and heads");
  SIMP_CUDA(launch_kernel(kern, dim3(unsigned(units)), dim3(Sh::THREADS), Sh::SMEM, ctx().stream, true, mq, mk, mv, p));
  return SIMP_OK;
}
template <bool BF16, int D>
static int tc_launch(TcArgs p) {
  const AttnPromptArgs& a = p.a;
  p.tpt = 128 / a.rep;
  CUtensorMap mq, mk, mv;
  if (int rc = attn_tensor_map(&mq, BF16, p.q, a.total_q, a.H, D, p.q_stride, a.rep, p.tpt)) return rc;
  if (int rc = attn_tensor_map(&mk, BF16, p.k, a.total_k, a.G, D, p.kv_stride, 1, 128)) return rc;
  if (int rc = attn_tensor_map(&mv, BF16, p.v, a.total_k, a.G, D, p.kv_stride, 1, 128)) return rc;
  // Short prompts on one tile per block and two blocks per SM.  32/8 heads, us with one / two tiles: D = 64, 64 prompts of 128
  // tokens 64 / 76, 16 of 512 87 / 91, 4 of 2048 173 / 168; D = 128, 64 of 1 18 / 31, 64 of 128 82 / 91, 32 of 256 98 / 91.
  const bool brief = a.total_k < (D == 64 ? 2048 : 192) * int64_t(a.n_seqs);
  return brief ? tc_run<BF16, D, 1>(p, mq, mk, mv) : tc_run<BF16, D, 2>(p, mq, mk, mv);
}

// Rows to rows of heads padded to DP elements.  16-bit types are copied; f32 is split into three bf16 planes h + m + l (8 bits
// of mantissa each: exact, but for what lies below 2^-133), one behind the other.  Elements that are not finite have no
// place there: they are zeros in the planes, the byte of their row and head in `odd` is set, and *any.  A thread writes
// eight elements, the DP / 8 threads of a head are neighbours in a warp.  VEC: four elements lie together at a multiple of
// their size (D and strides multiples of 4, aligned pointers).
template <bool SPLIT, bool VEC>
__global__ void __launch_bounds__(256) attn_pack_kernel(const AttnPack q, const AttnPack k, const AttnPack v, unsigned blocks_q, unsigned blocks_k, int D,
                                                        int DP, int* any) {
  pdl_launch_dependents();
  pdl_wait();
  unsigned block = blockIdx.x;
  const AttnPack& t = block < blocks_q ? q : block < blocks_q + blocks_k ? k : v;
  block -= block < blocks_q ? 0 : block < blocks_q + blocks_k ? blocks_q : blocks_q + blocks_k;
  const void* __restrict__ src = t.src;
  uint16_t* __restrict__ dst = static_cast<uint16_t*>(t.dst);
  uint8_t* __restrict__ odd = t.odd;
  const int64_t rows = t.rows, stride = t.stride;
  const int heads = t.heads;
  const int64_t i = int64_t(block) * blockDim.x + threadIdx.x;   // eighth of a padded row
  const int eighths = DP / 8, per = heads * eighths;
  const int64_t row = i / per;
  const bool in = row < rows;
  const int at = int(i - row * per), head = at / eighths, d0 = 8 * (at % eighths);
  const int64_t from = row * stride + int64_t(head) * D + d0;
  const int n = in ? min(8, D - d0) : 0;
  using E = std::conditional_t<SPLIT, float, uint16_t>;
  using V4 = std::conditional_t<SPLIT, float4, uint2>;
  E e8[8];
  if (VEC) {   // n is 8, 4 or 0 or less
    V4 w[2] = {};
    if (n > 0) w[0] = __ldcs(reinterpret_cast<const V4*>(static_cast<const E*>(src) + from));
    if (n > 4) w[1] = __ldcs(reinterpret_cast<const V4*>(static_cast<const E*>(src) + from) + 1);
    memcpy(e8, w, sizeof(e8));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) e8[e] = e < n ? static_cast<const E*>(src)[from + e] : E(0);
  }
  uint4 out[3];
  uint16_t* h = reinterpret_cast<uint16_t*>(out);
  bool bad = false;
  if constexpr (SPLIT) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(e8[e]) & 0x7fffffffu);
    if (most < 0x7f7f8000u) {   // everything is finite and rounds to a finite bf16
      uint32_t* w = reinterpret_cast<uint32_t*>(out);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f2 minus = pack_f2(-1.0f, -1.0f);
        f2 x = pack_f2(e8[2 * e], e8[2 * e + 1]);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const uint32_t p = pack2<true>(lo_f2(x), hi_f2(x));
          w[4 * q + e] = p;
          if (q < 2) x = fma_f2(pack_f2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u)), minus, x);   // exact
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = e8[e];
        if (!(fabsf(x) <= 3.402823466e38f)) bad = true, x = 0.0f;
        uint16_t a = __bfloat16_as_ushort(__float2bfloat16_rn(x));
        if ((a & 0x7fffu) == 0x7f80u) --a;   // the largest f32 would round to infinity
        const float r = x - __uint_as_float(uint32_t(a) << 16);
        const __nv_bfloat16 b = __float2bfloat16_rn(r);
        h[e] = a;
        h[8 + e] = __bfloat16_as_ushort(b);
        h[16 + e] = __bfloat16_as_ushort(__float2bfloat16_rn(r - __bfloat162float(b)));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = e8[e];
  }
  if (in) {
    const int64_t plane = rows * per;
#pragma unroll
    for (int q = 0; q < (SPLIT ? 3 : 1); ++q) reinterpret_cast<uint4*>(dst)[q * plane + i] = out[q];
  }
  if (SPLIT) {
    const unsigned lanes = __ballot_sync(0xffffffffu, bad), lane = threadIdx.x & 31;
    if (in && lane % eighths == 0) {
      const bool mark = (lanes >> lane) & ((1u << eighths) - 1u);
      odd[row * heads + head] = mark;
      if (mark) atomicOr(any, 1);
    }
  }
}

int attn_pack(bool split, const AttnPack& q, const AttnPack& k, const AttnPack& v, int D, int DP, int* any) {
  auto blocks = [&](const AttnPack& t) { return cdiv(t.rows * t.heads * (DP / 8), 256); };
  const int64_t nq = blocks(q), nk = blocks(k);
  SIMP_REQUIRE(nq + 2 * nk <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many rows and heads");
  const size_t four = split ? 16 : 8;
  const bool vec = D % 4 == 0 && q.stride % 4 == 0 && k.stride % 4 == 0 && aligned_to(q.src, four) && aligned_to(k.src, four) && aligned_to(v.src, four);
  auto kern = split ? (vec ? attn_pack_kernel<true, true> : attn_pack_kernel<true, false>) : (vec ? attn_pack_kernel<false, true> : attn_pack_kernel<false, false>);
  SIMP_CUDA(launch_kernel(kern, dim3(unsigned(nq + 2 * nk)), dim3(256), 0, ctx().stream, true, q, k, v, unsigned(nq), unsigned(nk), D, DP, any));
  return SIMP_OK;
}

// 16-bit types on the tensor cores: a positive scale (the maximum of the scores is then the maximum of the scaled ones) and
// rows that TMA can address; others are copied into padded rows first (library scratch).  1: not taken.
int attn_prompt_tc(const AttnPromptArgs& a, int dtype) {
  if (dtype == SIMP_DTYPE_F32 || !(a.scale_log2 > 0.0f && a.scale_log2 <= 3.0e38f) || a.total_k == 0) return 1;
  const int D = a.D <= 64 ? 64 : 128;
  TcArgs p{};
  p.a = a;
  p.chunk = a.D % 8 == 0 && aligned_to(a.out, 16) && a.out_stride % 8 == 0 ? 8 : a.D % 4 == 0 && aligned_to(a.out, 8) && a.out_stride % 4 == 0 ? 4 : 1;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_stride = a.q_stride;
  p.kv_stride = a.kv_stride;
  if (a.D != D || !aligned_to(a.q, 16) || !aligned_to(a.k, 16) || !aligned_to(a.v, 16) || a.q_stride % 8 || a.kv_stride % 8) {
    const size_t nq = size_t(a.total_q) * a.H * D * 2, nk = size_t(a.total_k) * a.G * D * 2;
    uint8_t* s = static_cast<uint8_t*>(scratch(nq + 2 * nk, SCRATCH_ATTN_PACK));
    if (!s) return attn_no_scratch();
    p.q = s;
    p.k = s + nq;
    p.v = s + nq + nk;
    p.q_stride = int64_t(a.H) * D;
    p.kv_stride = int64_t(a.G) * D;
    const AttnPack of_q{a.q, s, nullptr, a.total_q, a.q_stride, a.H}, of_k{a.k, s + nq, nullptr, a.total_k, a.kv_stride, a.G};
    const AttnPack of_v{a.v, s + nq + nk, nullptr, a.total_k, a.kv_stride, a.G};
    if (int rc = attn_pack(false, of_q, of_k, of_v, a.D, D, nullptr)) return rc;
  }
  if (dtype == SIMP_DTYPE_BF16) return D == 64 ? tc_launch<true, 64>(p) : tc_launch<true, 128>(p);
  return D == 64 ? tc_launch<false, 64>(p) : tc_launch<false, 128>(p);
}

}  // namespace simp
