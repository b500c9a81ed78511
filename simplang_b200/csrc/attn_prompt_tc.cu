// attn_prompt_tc.cu -- causal attention over packed prompts on the tcgen05 tensor cores: f16 / bf16, head size 64 or 128.
//
// One block of 12 warps works on two row tiles ("A" and "B") of one key/value head of one sequence.  A row tile is 128 rows
// of the score matrix: 128 / rep consecutive tokens times the rep query heads that share the key/value head (row = token *
// rep + head), so grouped heads read K and V once, short prompts fill tiles and the causal edge is fine.  Roles:
//   warps 0-3, 4-7  softmax of tile A, of tile B: one thread per row
//   warp 8          TMA: Q once, then K and V tiles of 128 keys through a ring of slots
//   warp 9          issues the MMAs: S = Q K^T (128 x 128, f32 in TMEM), O += P V with P read from TMEM
//   warp 10         cleans the V tiles at the causal / ragged edge (see below)
// P (16 bits) overwrites S in place: S_X(j + 1) is issued behind O_X += P_X(j) V(j), and MMAs of one thread run in order.
// While the tensor cores work on one tile, the other tile's softmax runs: 2 x 128 x 128 x D MACs take 4 D cycles per tile and
// step, its 16384 exponentials 1024, so for D = 128 both are busy about half of the time.
//
// Softmax: the row's running maximum moves only when a tile exceeds it by more than 2^8 (weights are then at most 2^8, well
// inside f16), so O is rarely rescaled: it stays in TMEM.  S_X(j + 1) being complete implies that P_X(j) V(j) is, so the
// softmax warps may rescale O_X without another barrier.
//
// A weight of zero does not hide a NaN or an infinity from an MMA, and a tile may hold keys that some rows must not see:
// later tokens of the sequence, and rows of the NEXT sequence (or behind the last) where the sequence ends inside the tile.
// Warp 10 therefore zeroes, in the edge tiles only, V rows behind the sequence and every element that is not finite; a bit
// per such key tells the epilogue to add those elements (read again from global memory) to the rows that do see the key.
#include <cuda.h>
#include <algorithm>
#include <climits>

#include "attn_prompt.cuh"
#include "sm100_ptx.cuh"

namespace simp {
using namespace ptx;

constexpr int TC_THREADS = 384;
constexpr int TC_EDGE = 4;   // edge tiles of a block: its rows see at most 255 keys more than its first row, so 3

template <int D>
struct TcShape {
  static constexpr int TILE = 128 * D * 2;              // bytes of 128 rows
  static constexpr int SLOTS = D == 128 ? 5 : 8;
  static constexpr int BARS = 2 * SLOTS + 1 + 6 + TC_EDGE;
  static constexpr size_t SMEM = 1024 + size_t(2 + SLOTS) * TILE + BARS * 8 + 16 + TC_EDGE * 16;
};

struct TcArgs {
  AttnPromptArgs a;
  int tpt;          // tokens per row tile
  uint32_t idesc_s, idesc_o;
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(m),
               "r"(bar), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t t, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// bits of the 16-bit halves of w that are infinity or NaN
template <bool BF16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}

template <bool BF16, int D>
__global__ void __launch_bounds__(TC_THREADS, 1)
    attn_prompt_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const TcArgs p) {
  using Sh = TcShape<D>;
  extern __shared__ uint8_t tc_raw[];
  const uint32_t base = (smem_u32(tc_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = base, ring = base + 2 * Sh::TILE, bars = ring + Sh::SLOTS * Sh::TILE;
  uint8_t* generic = tc_raw + (base - smem_u32(tc_raw));
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
  const AttnPromptArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::SLOTS; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(q_bar, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_bar(x), 1);
      mbar_init(p_bar(x), 4);
      mbar_init(o_bar(x), 1);
    }
    for (int e = 0; e < TC_EDGE; ++e) mbar_init(edge_bar(e), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < TC_EDGE * 4) odd_keys[threadIdx.x] = 0;

  // ---- which rows (every warp finds them for itself)
  const int g = blockIdx.x % a.G;
  const int rows_cta = 2 * p.tpt;
  int seq = 0, place = 0, q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  auto count = [&](int s) {
    int b, e;
    return seq_range(a.q_off, s, a.total_q, a.status, b, e) ? (e - b + rows_cta - 1) / rows_cta : 0;
  };
  if (!find_unit(blockIdx.x / a.G, a.n_seqs, count, seq, place)) return;
  seq_range(a.q_off, seq, a.total_q, a.status, q0, q1);
  if (!seq_range(a.k_off, seq, a.total_k, a.status, k0, k1)) return;
  const int nq = q1 - q0, nk = k1 - k0;
  place = (nq + rows_cta - 1) / rows_cta - 1 - place;   // the longest rows first
  const int r0 = place * rows_cta;                      // first token of tile A
  const int64_t shift = int64_t(nk) - nq;               // token i sees keys j <= i + shift
  auto sees = [&](int token) { return int(max(int64_t(0), min(int64_t(nk), token + shift + 1))); };
  int n_x[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = r0 + x * p.tpt, last = min(first + p.tpt, nq) - 1;
    n_x[x] = first < nq ? (sees(last) + 127) >> 7 : 0;
  }
  const int n = max(n_x[0], n_x[1]);
  const int edge0 = sees(r0) >> 7;                      // tiles from here on hold a key that some row does not see

  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  if (warp == 8) {
    // ------------------------------------------------------------------ loads
    if (lane == 0 && n > 0) {
      const int tiles = r0 + p.tpt < nq ? 2 : 1;
      const uint32_t box = uint32_t(p.tpt * a.rep) * 128u;
      mbar_arrive_expect_tx(q_bar, tiles * (D / 64) * box);
      for (int x = 0; x < tiles; ++x)
        for (int b = 0; b < D / 64; ++b)
          tma_load_3d(q_smem + x * Sh::TILE + b * 16384, &map_q, q_bar, 64 * b, g * a.rep, q0 + r0 + x * p.tpt);
      bool ok = true;
      for (int i = 0; ok && i < 2 * n; ++i) {
        const int s = i % Sh::SLOTS;
        if (!mbar_wait(empty_bar(s), ((i / Sh::SLOTS) & 1) ^ 1, abort_flag, a.status, 61)) { ok = false; break; }
        const bool edge = (i & 1) && (i >> 1) >= edge0;   // lands for warp 10, which passes the slot on
        const uint32_t bar = edge ? edge_bar((i >> 1) - edge0) : full_bar(s);
        mbar_arrive_expect_tx(bar, Sh::TILE);
        for (int b = 0; b < D / 64; ++b)
          tma_load_3d(ring + s * Sh::TILE + b * 16384, i & 1 ? &map_v : &map_k, bar, 64 * b, g, k0 + 128 * (i >> 1));
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);   // let copies in flight land before the block retires
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMAs
    if (lane == 0 && n > 0) {
      auto wait = [&](uint32_t bar, uint32_t phase, int site) {
        const bool ok = mbar_wait(bar, phase, abort_flag, a.status, site);
        tc_fence_after_sync();
        return ok;
      };
      auto wait_slot = [&](int i) { return wait(full_bar(i % Sh::SLOTS), (i / Sh::SLOTS) & 1, 62); };
      auto scores = [&](int x, int j) {
        const uint64_t qd = make_smem_desc_sw128(q_smem + x * Sh::TILE, 16u, 1024u);
        const uint64_t kd = make_smem_desc_sw128(ring + (2 * j % Sh::SLOTS) * Sh::TILE, 16u, 1024u);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {   // 16 elements = 32 bytes; the next 64 elements lie 16 KB further
          const uint64_t o = uint64_t((s >> 2) * 1024 + (s & 3) * 2);
          mma_f16_ss(tmem + 128u * x, qd + o, kd + o, p.idesc_s, s > 0);
        }
      };
      auto values = [&](int x, int j) {
        // V [key][element]: element-major operand, 64-element atoms 16 KB apart, 8 keys 1 KB apart
        const uint64_t vd = make_smem_desc_sw128(ring + ((2 * j + 1) % Sh::SLOTS) * Sh::TILE, 16384u, 1024u);
#pragma unroll
        for (int s = 0; s < 8; ++s)          // 16 keys = 8 columns of P, 2 KB of V
          mma_f16_ts(tmem + 256u + uint32_t(D) * x, tmem + 128u * x + 8u * s, vd + uint64_t(s * 128), p.idesc_o, j > 0 || s > 0);
      };
      bool ok = wait(q_bar, 0, 63) && wait_slot(0);
      if (ok) {
        for (int x = 0; x < 2; ++x)
          if (n_x[x] > 0) {
            scores(x, 0);
            mma_commit(s_bar(x));
          }
        mma_commit(empty_bar(0));
      }
      for (int j = 0; ok && j < n; ++j) {
        ok = wait_slot(2 * j + 1);
        if (ok && j + 1 < n) ok = wait_slot(2 * j + 2);
        for (int x = 0; ok && x < 2; ++x) {
          if (j >= n_x[x]) continue;
          ok = wait(p_bar(x), j & 1, 65);
          if (!ok) break;
          values(x, j);
          if (j + 1 < n_x[x]) {
            scores(x, j + 1);
            mma_commit(s_bar(x));
          } else {
            mma_commit(o_bar(x));
          }
        }
        if (!ok) break;
        mma_commit(empty_bar((2 * j + 1) % Sh::SLOTS));
        if (j + 1 < n) mma_commit(empty_bar((2 * j + 2) % Sh::SLOTS));
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 10) {
    // ------------------------------------------------------------------ V at the edge
    for (int j = edge0; j < n; ++j) {
      const int i = 2 * j + 1;
      if (!mbar_wait(edge_bar(j - edge0), 0, abort_flag, a.status, 66)) break;
      uint8_t* v = generic + 2 * Sh::TILE + (i % Sh::SLOTS) * Sh::TILE;
      const int keys = nk - 128 * j;   // rows from here on are not the sequence's
      // (the 128-byte swizzle moves 16-byte pieces inside a row only, so rows are found as if there were none)
      for (int c = lane; c < Sh::TILE / 16; c += 32) {
        const int key = (c >> 3) & 127;
        uint4* at = reinterpret_cast<uint4*>(v) + c;
        uint4 w = *at;
        uint32_t m0 = odd_halves<BF16>(w.x), m1 = odd_halves<BF16>(w.y), m2 = odd_halves<BF16>(w.z), m3 = odd_halves<BF16>(w.w);
        if (key >= keys) {
          *at = make_uint4(0u, 0u, 0u, 0u);
        } else if (m0 | m1 | m2 | m3) {
          *at = make_uint4(w.x & ~m0, w.y & ~m1, w.z & ~m2, w.w & ~m3);
          atomicOr(odd_keys + (j - edge0) * 4 + (key >> 5), 1u << (key & 31));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full_bar(i % Sh::SLOTS));
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------------ softmax
    const int x = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
    const uint32_t s_tmem = tmem + 128u * x + lanes, o_tmem = tmem + 256u + uint32_t(D) * x + lanes;
    const int token = r0 + x * p.tpt + row / a.rep, head = g * a.rep + row % a.rep;
    const bool mine = row < p.tpt * a.rep && token < nq;
    const int lim = mine ? sees(token) : 0;
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < n_x[x]; ++j) {
      ok = mbar_wait(s_bar(x), j & 1, abort_flag, a.status, 67);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after_sync();
      float s[128];
#pragma unroll
      for (int h = 0; h < 4; ++h) tmem_ld_32x32(s_tmem + 32u * h, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * h));
      tmem_ld_wait();
      const int see = lim - 128 * j;
      if (__any_sync(0xffffffffu, see < 128)) {
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < see ? s[i] : -INFINITY;
      }
      float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < 128; i += 8) {
        t0 = fmaxf(t0, fmaxf(s[i], s[i + 1]));
        t1 = fmaxf(t1, fmaxf(s[i + 2], s[i + 3]));
        t2 = fmaxf(t2, fmaxf(s[i + 4], s[i + 5]));
        t3 = fmaxf(t3, fmaxf(s[i + 6], s[i + 7]));
      }
      const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * c;
      if (j == 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, top > m + 8.0f)) {
        const float mn = fmaxf(m, top), alpha = m == mn ? 1.0f : ex2(m - mn);
        l *= alpha;
        m = mn;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          tmem_ld_32x32(o_tmem + 32u * h, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32(o_tmem + 32u * h, o);
        }
      }
      const float off = m == -INFINITY ? 0.0f : m;
      float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float e0 = ex2(fmaf(s[64 * h + 2 * i], c, -off)), e1 = ex2(fmaf(s[64 * h + 2 * i + 1], c, -off));
          sum0 += e0;
          sum1 += e1;
          w[i] = pack2<BF16>(e0, e1);
        }
        tmem_st_32x32(s_tmem + 32u * h, w);
      }
      l += sum0 + sum1;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_bar(x));
    }
    if (ok && n_x[x] > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_bar(x), 0, abort_flag, a.status, 68));
    if (ok) {
      tc_fence_after_sync();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint8_t* out = static_cast<uint8_t*>(a.out) + (int64_t(q0 + token) * a.out_stride + int64_t(head) * D) * 2;
      uint32_t odd = 0;
      for (int e = 0; e < TC_EDGE * 4; ++e) odd |= odd_keys[e];
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        uint32_t o[32];
        if (n_x[x] > 0) {
          tmem_ld_32x32(o_tmem + 32u * h, o);
          tmem_ld_wait();
        }
        if (mine) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = l == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
          if (odd)   // rare: a key of an edge tile has elements that are not finite
            for (int key = 128 * edge0; key < lim; ++key)
              if ((odd_keys[(key - 128 * edge0) >> 5] >> (key & 31)) & 1u) {
                const uint16_t* v = static_cast<const uint16_t*>(a.v) + int64_t(k0 + key) * a.kv_stride + int64_t(g) * D + 32 * h;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (odd_halves<BF16>(v[i]) & 0xffffu) {
                    const float f = BF16 ? __uint_as_float(uint32_t(v[i]) << 16) : __half2float(__ushort_as_half(v[i]));
                    o[i] = __float_as_uint(__uint_as_float(o[i]) + f);
                  }
              }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 w;
            w.x = pack2<BF16>(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1]));
            w.y = pack2<BF16>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]));
            w.z = pack2<BF16>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]));
            w.w = pack2<BF16>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
            *reinterpret_cast<uint4*>(out + 64 * h + 16 * i) = w;
          }
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// [rows, heads, D] of 16-bit elements, rows a stride apart; boxes of 64 elements x box_heads x box_rows, 128-byte swizzle.
static int tc_map(CUtensorMap* map, bool bf16, const void* p, int64_t rows, int64_t heads, int D, int64_t stride, int box_heads, int box_rows) {
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

template <bool BF16, int D>
static int tc_launch(const AttnPromptArgs& a) {
  TcArgs p{};
  p.a = a;
  p.tpt = 128 / a.rep;
  // f32 accumulator; operand type; B of the second product is element-major
  const uint32_t type = (1u << 4) | (uint32_t(BF16) << 7) | (uint32_t(BF16) << 10) | (8u << 24);
  p.idesc_s = type | (uint32_t(128 >> 3) << 17);
  p.idesc_o = type | (1u << 16) | (uint32_t(D >> 3) << 17);
  CUtensorMap mq, mk, mv;
  if (int rc = tc_map(&mq, BF16, a.q, a.total_q, a.H, D, a.q_stride, a.rep, p.tpt)) return rc;
  if (int rc = tc_map(&mk, BF16, a.k, a.total_k, a.G, D, a.kv_stride, 1, 128)) return rc;
  if (int rc = tc_map(&mv, BF16, a.v, a.total_k, a.G, D, a.kv_stride, 1, 128)) return rc;
  auto kern = attn_prompt_tc_kernel<BF16, D>;
  SIMP_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(TcShape<D>::SMEM)));
  const int64_t units = std::min(a.total_q, a.total_q / (2 * p.tpt) + a.n_seqs) * a.G;
  SIMP_REQUIRE(units <= INT_MAX, SIMP_ERR_SHAPE, "attn_prompt: too many rows and heads");
  kern<<<unsigned(units), TC_THREADS, TcShape<D>::SMEM, ctx().stream>>>(mq, mk, mv, p);
  SIMP_LAUNCH_CHECK();
  return SIMP_OK;
}

// Whether the tensor-core kernel can take the call: head size, a positive scale (the maximum of the scores is then the
// maximum of the scaled ones), and rows that TMA can address.
bool attn_prompt_tc_takes(const AttnPromptArgs& a, int dtype) {
  return dtype != SIMP_DTYPE_F32 && (a.D == 64 || a.D == 128) && a.scale_log2 > 0.0f && a.scale_log2 <= 3.0e38f && a.total_k > 0 && aligned_to(a.q, 16) &&
         aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.out, 16) && a.q_stride % 8 == 0 && a.kv_stride % 8 == 0 && a.out_stride % 8 == 0;
}
int attn_prompt_tc(const AttnPromptArgs& a, int dtype) {
  if (dtype == SIMP_DTYPE_BF16) return a.D == 64 ? tc_launch<true, 64>(a) : tc_launch<true, 128>(a);
  return a.D == 64 ? tc_launch<false, 64>(a) : tc_launch<false, 128>(a);
}

}  // namespace simp
