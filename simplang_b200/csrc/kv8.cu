// kv8.cu -- the 8-bit key/value cache: writing rows into it, reading them back, attention of single tokens over it.
//
// A block holds `bt` tokens of one layer; per block and head one f32 scale.  K lies [token][pitch] (a score contracts
// over elements), V lies [token / 16][pitch][16 tokens] (an output contracts over tokens), so both are read as they are
// multiplied: as the s8 operand of warp-level integer MMAs, without a conversion or a transpose on the way.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "llm_ops.cuh"
#include "sm100_ptx.cuh"

namespace simp {

struct Kv8View {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  const int32_t* table;
  int64_t table_stride;
  int n_blocks, bt, G, D, pitch, shift;   // bt = 1 << shift
};

// ------------------------------------------------------------------------------------------------ write
// max|x| / 127, IEEE division; a subnormal step could not be divided by and stands for zeros.
__device__ __forceinline__ float kv8_step(float top) {
  const float s = __fdiv_rn(top, 127.0f);
  return s < FLT_MIN ? 0.0f : s;
}
__device__ __forceinline__ float kv8_magnitude(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.0f;   // NaN and infinities do not count
}
// x / s to the nearest integer, halves to even, exactly: the product with 1 / s is within one of it, and the remainder
// x - n s has no rounding error (n <= 127, |x - n s| < 2 s: a multiple of the smaller ulp that fits 24 bits), so it
// tells which side of a half x lies on.  A plain division would round quotients next to a half onto it.
// This is the general form; kv8_round4 takes the values that lie clear of halves, which are nearly all.
__device__ __forceinline__ uint32_t kv8_quantise(float x, float s, float inv) {
  if (s == 0.0f || x != x) return 0;
  if (fabsf(x) > FLT_MAX) return x > 0.0f ? 127u : uint32_t(-127) & 0xffu;
  float n = rintf(x * inv);
  const float r2 = 2.0f * fmaf(-n, s, x);
  if (r2 > s) n += 1.0f;
  else if (r2 < -s) n -= 1.0f;
  else if (fabsf(r2) == s && (int(n) & 1)) n += r2 > 0.0f ? 1.0f : -1.0f;
  return uint32_t(int(fminf(fmaxf(n, -127.0f), 127.0f))) & 0xffu;
}
// (out of line: it is rare, and what a block of few tokens waits for is its instructions)
__device__ __noinline__ uint32_t kv8_round4_general(float x0, float x1, float x2, float x3, float s, float inv) {
  return kv8_quantise(x0, s, inv) | kv8_quantise(x1, s, inv) << 8 | kv8_quantise(x2, s, inv) << 16 | kv8_quantise(x3, s, inv) << 24;
}
// Four values as four bytes.  Adding 1.5 * 2^23 rounds x / s to an integer that is then the sum's low byte; twice the exact
// remainder is below `sure` (s, or anything where s is a power of two: the product with 1 / s is then exact and rounded to
// even) where that integer is the nearest.  Above s it is off by one.  Quotients within rounding of a half are common
// (half of the largest value is 63.5), exact halves are not but for powers of two, whose blocks are full of them.
// `odd`: something in the block is not finite, or the step is 0.
__device__ __forceinline__ uint32_t kv8_round4(const float (&x)[4], float s, float inv, float sure, bool odd) {
  uint32_t b[4];
  float r2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fmaf(x[i], inv, 12582912.0f), r = fmaf(12582912.0f - t, s, x[i]);
    r2[i] = r + r;
    b[i] = __float_as_uint(t);
  }
  const float far = fmaxf(fmaxf(fabsf(r2[0]), fabsf(r2[1])), fmaxf(fabsf(r2[2]), fabsf(r2[3])));
  if (odd || !(far < sure)) {
    bool half = odd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      half = half || fabsf(r2[i]) == s;
      b[i] += uint32_t(r2[i] > s) - uint32_t(r2[i] < -s);
    }
    if (half) return kv8_round4_general(x[0], x[1], x[2], x[3], s, inv);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
__device__ __forceinline__ float kv8_sure(float s) { return __float_as_uint(s) & 0x007fffffu ? s : INFINITY; }
// A held integer to a larger step: q old / now to the nearest integer, halves to even, exactly.  q old is hi + lo; n is within one
// of the quotient and hi - n now has no rounding error, so their sum tells which side of a half the quotient lies on.
__device__ __forceinline__ uint32_t kv8_requantise(int q, float old, float now, float ratio) {
  const float x = float(q), hi = x * old, lo2 = 2.0f * fmaf(x, old, -hi);
  float n = rintf(x * ratio);
  const float r2 = 2.0f * fmaf(-n, now, hi);
  const float above = (r2 - now) + lo2, below = (r2 + now) + lo2;
  if (above > 0.0f || (above == 0.0f && (int(n) & 1))) n += 1.0f;
  else if (below < 0.0f || (below == 0.0f && (int(n) & 1))) n -= 1.0f;
  return uint32_t(int(n)) & 0xffu;
}

// The part of sequence s that lies in one block: unit = (sequence, block), found by find_unit.
struct Kv8Span {
  int seq, row0, a, b;   // packed row of place a of the block; places [a, b) are new
  int block;
};
__device__ __forceinline__ bool kv8_span(const Kv8View& c, int64_t unit, const int32_t* off, const int32_t* starts, int n_seqs,
                                         int64_t total, int* status, Kv8Span& sp) {
  const int64_t cap = c.table_stride * c.bt;
  auto count = [&](int s) {
    int q0, q1;
    if (!seq_range(off, s, total, status, q0, q1) || q0 == q1) return 0;
    const int64_t st = __ldg(starts + s), n = q1 - q0;
    if (st < 0 || st + n > cap) {
      report_status(status, STATUS_BAD_RANGE, s);
      return 0;
    }
    return int(((st + n - 1) >> c.shift) - (st >> c.shift)) + 1;
  };
  int place;
  if (!find_unit(unit, n_seqs, count, sp.seq, place)) return false;
  const int q0 = __ldg(off + sp.seq), n = __ldg(off + sp.seq + 1) - q0, st = __ldg(starts + sp.seq);
  const int64_t bi = (st >> c.shift) + place, p0 = bi << c.shift;
  sp.a = int(max(int64_t(st) - p0, int64_t(0)));
  sp.b = int(min(int64_t(st) + n - p0, int64_t(c.bt)));
  sp.row0 = int(q0 + (p0 + sp.a - st));
  sp.block = __ldg(c.table + sp.seq * c.table_stride + bi);
  if (sp.block < 0 || sp.block >= c.n_blocks) {
    if (threadIdx.x == 0) report_status(status, STATUS_BAD_BLOCK, sp.block);
    return false;
  }
  return true;
}

// A thread owns a patch of 16 tokens x 4 elements of K or of V: K leaves as words (a warp writes whole rows), V as 16-byte
// columns.  A block of threads per (sequence, cache block, head), for K and for V: bt / 16 x pitch / 4 patches.  Rows are
// read twice, for the maximum and for the values; the second time most come from L1.  Bound by these round trips: a call
// is hardly more than one wave of blocks (8192 bf16 rows of 8 heads x 128: 21 us, of 8 at the memory's rate; 26 with one
// block for K and V, 23 with 4 rows of the first pass in flight, 21 with 16).  Keeping patches in registers between the
// passes was tried: 254 registers, and code so long that fetching it took most of the time; 90 us.
// VEC: four elements lie together at a multiple of their size (head_dim a multiple of 4, aligned pointers and stride).
// Four elements as they are stored: what the maximum is taken of, two 16-bit ones at a time.
template <typename T> struct Kv8Raw;
template <> struct Kv8Raw<float> {
  uint32_t w[4];
  __device__ __forceinline__ void top(uint32_t& t) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) t = max(t, w[i] & 0x7fffffffu);
  }
  static __device__ __forceinline__ float magnitude(uint32_t t) { return __uint_as_float(t); }   // may be infinity or NaN
};
template <typename T> struct Kv8Raw {
  uint32_t w[2];
  __device__ __forceinline__ void top(uint32_t& t) const {
    asm("max.u16x2 %0, %0, %1;" : "+r"(t) : "r"(w[0] & 0x7fff7fffu));
    asm("max.u16x2 %0, %0, %1;" : "+r"(t) : "r"(w[1] & 0x7fff7fffu));
  }
  static __device__ __forceinline__ float magnitude(uint32_t t) {
    const uint16_t m = uint16_t(max(t & 0xffffu, t >> 16));
    return to_f32(reinterpret_cast<const T&>(m));
  }
};
template <typename T, bool VEC>
__device__ __forceinline__ Kv8Raw<T> kv8_raw4(const T* row, int d, int D) {
  Kv8Raw<T> r;
  if (VEC) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(r.w) = *reinterpret_cast<const uint4*>(row + d);
    else *reinterpret_cast<uint2*>(r.w) = *reinterpret_cast<const uint2*>(row + d);
  } else {
    T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = d + i < D ? row[d + i] : from_f32<T>(0.0f);
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void kv8_load4(const T* row, int d, int D, float (&x)[4]) {
  const Kv8Raw<T> r = kv8_raw4<T, VEC>(row, d, D);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(reinterpret_cast<const T*>(r.w)[i]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void kv8_store4(T* row, int d, int D, const float (&x)[4]) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + d) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      uint2 w;
      T* e = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(x[i]);
      *reinterpret_cast<uint2*>(row + d) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = from_f32<T>(x[i]);
  }
}

// The first `held` tokens of a patch from step `old` to the larger step `s`, four words of four at a time.  Their loads go ahead
// of the arithmetic: one byte after the other took 27 us where this takes 11 (one token for each of 48 sequences, blocks of 32
// tokens of 8 x 64, all growing).
__device__ __forceinline__ void kv8_grow(int8_t* to, bool is_v, int held, int pitch, float old, float s) {
  const float ratio = old / s;
  // K: a word is four elements of a token; V: four tokens of an element, and the others' bytes are written back as they are
  const int step = is_v ? 4 : pitch, words = is_v ? 16 : held;
#pragma unroll 1
  for (int j0 = 0; j0 < words; j0 += 4) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = j0 + j < words ? *reinterpret_cast<const uint32_t*>(to + (j0 + j) * step) : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = is_v ? held - 4 * j : 4;   // bytes of this word
      uint32_t r = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = (w[j] >> (8 * i)) & 0xffu;
        r |= (i < n ? kv8_requantise(int8_t(uint8_t(b)), old, s, ratio) : b) << (8 * i);
      }
      if (j0 + j < words) *reinterpret_cast<uint32_t*>(to + (j0 + j) * step) = r;
    }
  }
}

// (Blocks per SM by what long prompts take: 32768 f32 rows of 32 x 100 261 us with five, 273 with four; 262144 bf16 rows of
// 8 x 64 244 and 226.)
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 5 : 4) kv8_append_kernel(Kv8View c, const T* __restrict__ k, const T* __restrict__ v,
                                                         int64_t row_stride, const int32_t* __restrict__ off,
                                                         const int32_t* __restrict__ starts, int n_seqs, int64_t total, int* status) {
  __shared__ float tops[8];
  Kv8Span sp;
  pdl_launch_dependents();
  pdl_wait();
  if (!kv8_span(c, blockIdx.x, off, starts, n_seqs, total, status, sp)) return;
  const bool is_v = blockIdx.z;
  const int h = blockIdx.y, quads = c.pitch >> 2, g = threadIdx.x / quads, d = 4 * (threadIdx.x % quads);
  const int t0 = 16 * g, lo = max(sp.a - t0, 0), hi = g < (c.bt >> 4) ? min(sp.b - t0, 16) : 0;   // new tokens of the patch: [lo, hi)
  const bool some = d < c.D;   // pad elements are written as zeros
  const T* in = (is_v ? v : k) + (int64_t(sp.row0) + t0 - sp.a) * row_stride + int64_t(h) * c.D;
  const int64_t sc = int64_t(sp.block) * c.G + h;
  float* scale = (is_v ? c.vs : c.ks) + sc;
  const float old = sp.a ? *scale : 0.0f;
  uint32_t t = 0;
  if (some && lo == 0 && hi == 16) {
#pragma unroll 8
    for (int j = 0; j < 16; ++j) kv8_raw4<T, VEC>(in + j * row_stride, d, c.D).top(t);
  } else if (some) {
#pragma unroll 1
    for (int j = lo; j < hi; ++j) kv8_raw4<T, VEC>(in + j * row_stride, d, c.D).top(t);
  }
  float top = Kv8Raw<T>::magnitude(t);
  const bool odd = __syncthreads_or(!(top <= FLT_MAX));
  if (odd) {   // infinities and NaN do not count
    top = 0.0f;
#pragma unroll 1
    for (int j = lo; some && j < hi; ++j) {
      float x[4];
      kv8_load4<T, VEC>(in + j * row_stride, d, c.D, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, kv8_magnitude(x[i]));
    }
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < int(blockDim.x >> 5); ++i) top = fmaxf(top, tops[i]);
  const float s = fmaxf(kv8_step(top), old);
  if (threadIdx.x == 0) *scale = s;   // every thread has read the old one: it was loaded before the barrier
  if (g >= (c.bt >> 4)) return;
  const float inv = s > 0.0f ? 1.0f / s : 0.0f, sure = kv8_sure(s);
  const bool general = odd || s == 0.0f;
  int8_t* to = (is_v ? c.v : c.k) + sc * c.bt * c.pitch + (is_v ? (int64_t(g) * c.pitch + d) * 16 : int64_t(t0) * c.pitch + d);
  if (sp.a && s != old && lo > 0) kv8_grow(to, is_v, min(lo, 16), c.pitch, old, s);
  if (!is_v) {
#pragma unroll 4
    for (int j = lo; j < hi; ++j) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (some) kv8_load4<T, VEC>(in + j * row_stride, d, c.D, x);
      *reinterpret_cast<uint32_t*>(to + j * c.pitch) = kv8_round4(x, s, inv, sure, general);
    }
  } else if (lo == 0 && hi == 16) {
    uint32_t col[4][4];   // element, four words of four tokens
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (some) kv8_load4<T, VEC>(in + (4 * w + j) * row_stride, d, c.D, x);
        r[j] = kv8_round4(x, s, inv, sure, general);
      }
      // rows of four elements to columns of four tokens
      const uint32_t p0 = __byte_perm(r[0], r[1], 0x5140), p1 = __byte_perm(r[0], r[1], 0x7362);
      const uint32_t q0 = __byte_perm(r[2], r[3], 0x5140), q1 = __byte_perm(r[2], r[3], 0x7362);
      col[0][w] = __byte_perm(p0, q0, 0x5410);
      col[1][w] = __byte_perm(p0, q0, 0x7632);
      col[2][w] = __byte_perm(p1, q1, 0x5410);
      col[3][w] = __byte_perm(p1, q1, 0x7632);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(col[i][0], col[i][1], col[i][2], col[i][3]);
  } else {   // part of a column: byte by byte, what lies before and behind the new tokens stays
#pragma unroll 1
    for (int j = lo; j < hi; ++j) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (some) kv8_load4<T, VEC>(in + j * row_stride, d, c.D, x);
      const uint32_t r = kv8_round4(x, s, inv, sure, general);
#pragma unroll
      for (int i = 0; i < 4; ++i) to[16 * i + j] = int8_t(r >> (8 * i));
    }
  }
}

// ------------------------------------------------------------------------------------------------ read
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8View c, T* __restrict__ k, T* __restrict__ v, int64_t row_stride,
                                                       const int32_t* __restrict__ off, const int32_t* __restrict__ starts,
                                                       int n_seqs, int64_t total, int* status) {
  Kv8Span sp;
  pdl_launch_dependents();
  pdl_wait();
  if (!kv8_span(c, blockIdx.x, off, starts, n_seqs, total, status, sp)) return;
  const bool is_v = blockIdx.z;
  const int h = blockIdx.y, quads = c.pitch >> 2, g = threadIdx.x / quads, d = 4 * (threadIdx.x % quads);
  const int t0 = 16 * g, lo = max(sp.a - t0, 0), hi = g < (c.bt >> 4) ? min(sp.b - t0, 16) : 0;
  if (hi <= lo || d >= c.D) return;
  const int64_t sc = int64_t(sp.block) * c.G + h;
  const float s = __ldg((is_v ? c.vs : c.ks) + sc);
  T* out = (is_v ? v : k) + (int64_t(sp.row0) + t0 - sp.a) * row_stride + int64_t(h) * c.D;
  uint32_t w[16];   // four elements of token 4 t + j in word 4 j + t
  if (!is_v) {
    const int8_t* kb = c.k + (sc * c.bt + t0) * c.pitch + d;
#pragma unroll
    for (int j = 0; j < 16; ++j) w[4 * (j & 3) + (j >> 2)] = __ldcs(reinterpret_cast<const uint32_t*>(kb + j * c.pitch));
  } else {
    const uint4* vb = reinterpret_cast<const uint4*>(c.v + sc * c.bt * c.pitch) + int64_t(g) * c.pitch + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = __ldcs(vb + i);
#pragma unroll
    for (int t = 0; t < 4; ++t) {   // columns of four tokens to rows of four elements
      const uint32_t p0 = __byte_perm(w[t], w[4 + t], 0x5140), p1 = __byte_perm(w[t], w[4 + t], 0x7362);
      const uint32_t q0 = __byte_perm(w[8 + t], w[12 + t], 0x5140), q1 = __byte_perm(w[8 + t], w[12 + t], 0x7362);
      w[t] = __byte_perm(p0, q0, 0x5410);
      w[4 + t] = __byte_perm(p0, q0, 0x7632);
      w[8 + t] = __byte_perm(p1, q1, 0x5410);
      w[12 + t] = __byte_perm(p1, q1, 0x7632);
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (j < lo || j >= hi) continue;
    const uint32_t r = w[4 * (j & 3) + (j >> 2)];
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = float(int8_t(uint8_t(r >> (8 * i)))) * s;
    kv8_store4<T, VEC>(out + j * row_stride, d, c.D, x);
  }
}

// ------------------------------------------------------------------------------------------------ attention
// out = softmax(scale q . K) V for one token per sequence.  Bound by the cache's bytes, which bulk copies bring into a ring
// in shared memory and which go from there into the MMA operand registers as they are: mma.m16n8k32 with A = 16 tokens x 32 elements of K (s8) and B = the query,
// then A = 16 elements x 32 tokens of V (s8) and B = the softmax weights.  Queries and weights become integers of PLANES
// bytes (16 bits for 16-bit queries, 24 for f32: below the rounding of their own type), one byte plane per B column, so
// the heads of a group fill the eight columns (4 heads x 2 planes; the third planes of eight heads share one more) and
// the cache is read once for the whole group.  Integer products are exact; what is rounded is the query (relative to its
// largest element), the weights (relative to the largest of their 32 tokens) and f32 sums of at most a tile each.
//
// A warp owns tiles of 32 tokens.  MMA row <-> token is free to choose: lane (g = lane / 4, t = lane % 4) gets the scores
// of tokens 4g .. 4g+3 for head t, so softmax maxima are three shuffles, and the weights of a lane pack into one word per
// plane, which is what the second MMA's B operand wants after one more shuffle: nothing passes through shared memory.
// Scales multiply scores and weights, never the integers, so blocks of any size (16 and up) may meet in a tile.
struct AttnKv8Args {
  Kv8View c;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int32_t* lengths;
  float* part;        // [seq][kv head][group][chunk] x (heads x (pitch + 2))
  int* count;         // [seq][kv head][group]
  int* status;
  float scale_log2;   // scale * log2(e)
  int rep, max_len, chunk, max_chunks, dtype;
  bool cluster;       // the chunks of a (sequence, head group) are one thread-block cluster
};

constexpr int AK_WARPS = 4, AK_JOIN = 8;

__device__ __forceinline__ void mma_s8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// byte `b` of four integers as one word
template <int B> __device__ __forceinline__ uint32_t bytes_of(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
  constexpr uint32_t sel = B | ((4 + B) << 4);
  return __byte_perm(__byte_perm(x0, x1, sel), __byte_perm(x2, x3, sel), 0x5410);
}

// S = pitch / 32; PLANES = 2 (16-bit queries) or 3 (f32); NH = groups of four heads (1 or 2)
template <int S>
struct AttnKv8Ring {
  // Stages of a tile (K and V of 32 tokens, 64 bytes per element) per warp.  With two of 8 KB, four warps and three blocks
  // per SM have 96 KB on their way while as much is worked on, about twice what the memory's latency needs.
  static constexpr int STAGES = S >= 3 ? 2 : 4, STAGE = 64 * 32 * S;
  static constexpr size_t SMEM = size_t(AK_WARPS) * STAGES * STAGE;
};
template <int S, int PLANES, int NH>
__global__ void __launch_bounds__(AK_WARPS * 32) attn_kv8_kernel(const AttnKv8Args a) {
  constexpr int P = 32 * S, HEADS = 4 * NH, NT = NH + (PLANES == 3 ? 1 : 0), STEP = 32 * AK_WARPS;
  constexpr int STAGES = AttnKv8Ring<S>::STAGES, STAGE = AttnKv8Ring<S>::STAGE;
  constexpr float QMAX = float(127 << (8 * (PLANES - 1)));          // the top byte never overflows
  constexpr float PMAX = PLANES == 3 ? 16777215.0f : 65535.0f;
  extern __shared__ __align__(128) uint8_t ak_ring[];              // [warp][stage][K 32 x P, V 2 x P x 16]; at the end [warp][head][P] sums
  __shared__ __align__(16) int8_t qb[NT * 8][P];                   // byte planes, one row per B column
  __shared__ float qs[HEADS];
  __shared__ float om[AK_WARPS][HEADS], ol[AK_WARPS][HEADS];
  __shared__ __align__(8) float2 joined[HEADS];                    // this block's top and sum of each head
  __shared__ __align__(8) uint64_t bars[AK_WARPS][STAGES];
  __shared__ int last, abort_flag;
  const Kv8View& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n_groups = (a.rep + HEADS - 1) / HEADS;
  const int s = blockIdx.z, kvh = blockIdx.y / n_groups, hg = blockIdx.y % n_groups, chunk = blockIdx.x;
  const int h0 = kvh * a.rep + hg * HEADS, nh = min(HEADS, a.rep - hg * HEADS);
  const int64_t orow = s * a.out_stride + int64_t(h0) * c.D;
  const int32_t* table = c.table + s * c.table_stride;
  const int c0 = chunk * a.chunk, tile0 = c0 + 32 * warp;
  // Block numbers of a tile's two halves (tokens 0-15, 16-31), the first ones beside the length: a place below max_len has
  // an entry in the table.  Where the second half lies behind the sequence, the first half's block stands in.
  auto entries = [&](int tile, int limit, int& e0, int& e1) {
    e0 = __ldg(table + (tile >> c.shift));
    e1 = __ldg(table + ((tile + 16 < limit ? tile + 16 : tile) >> c.shift));
  };
  int e0 = 0, e1 = 0;
  pdl_launch_dependents();
  pdl_wait();
  if (tile0 < a.max_len) entries(tile0, a.max_len, e0, e1);
  const int len = __ldg(a.lengths + s);
  if (len < 0 || len > a.max_len) {
    if (threadIdx.x == 0) report_status(a.status, STATUS_BAD_RANGE, s);
    return;
  }
  const int n_chunks = (len + a.chunk - 1) / a.chunk;
  if (chunk >= n_chunks) {
    if (len == 0 && chunk == 0)
      for (int i = threadIdx.x; i < nh * c.D; i += blockDim.x) store_any(a.out, orow + i, 0.0f, a.dtype);
    if (a.cluster && n_chunks > 1) {   // the others' barriers
      ptx::cluster_sync_all();
      ptx::cluster_sync_all();
    }
    return;
  }
  const int c1 = min(len, c0 + a.chunk);
  const int64_t head_bytes = int64_t(c.bt) * P;
  uint8_t* mine = ak_ring + size_t(warp) * STAGES * STAGE;
  const uint32_t ring = ptx::smem_u32(mine);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0)
    for (int i = 0; i < STAGES; ++i) ptx::mbar_init(ptx::smem_u32(&bars[warp][i]), 1);
  ptx::fence_barrier_init();
  __syncwarp();
  // Requests a tile into a stage; returns this lane's scales (tokens 4 g ..: half g / 4) and whether its block is out of range.
  struct TileInfo {
    float ks, vs;
    bool bad;
  };
  auto request = [&](int tile, int stage, int b0, int b1) {
    const bool bad0 = b0 < 0 || b0 >= c.n_blocks, bad1 = tile + 16 < len && (b1 < 0 || b1 >= c.n_blocks);
    if (bad0 || bad1) {
      if (lane == 0) report_status(a.status, STATUS_BAD_BLOCK, bad0 ? b0 : b1);
    }
    if (bad0) b0 = 0;
    if (bad1 || tile + 16 >= len) b1 = b0;
    const int64_t at0 = int64_t(b0) * c.G + kvh, at1 = int64_t(b1) * c.G + kvh;
    if (lane == 0) {
      const uint32_t dst = ring + stage * STAGE, bar = ptx::smem_u32(&bars[warp][stage]);
      ptx::mbar_arrive_expect_tx(bar, STAGE);
      const int64_t off = int64_t(tile & (c.bt - 1)) * P;   // K rows and V groups of 16 tokens take the same bytes
      if (c.bt >= 32) {
        ptx::bulk_load(dst, c.k + at0 * head_bytes + off, 32 * P, bar);
        ptx::bulk_load(dst + 32 * P, c.v + at0 * head_bytes + off, 32 * P, bar);
      } else {
        ptx::bulk_load(dst, c.k + at0 * head_bytes, 16 * P, bar);
        ptx::bulk_load(dst + 16 * P, c.k + at1 * head_bytes, 16 * P, bar);
        ptx::bulk_load(dst + 32 * P, c.v + at0 * head_bytes, 16 * P, bar);
        ptx::bulk_load(dst + 48 * P, c.v + at1 * head_bytes, 16 * P, bar);
      }
    }
    const int64_t at = g & 4 ? at1 : at0;
    const bool bad = g & 4 ? bad1 : bad0;
    return TileInfo{__ldg(c.ks + at), bad ? 0.0f : __ldg(c.vs + at), bad};
  };
  TileInfo info[STAGES];
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    const int tile = tile0 + i * STEP;
    if (tile < c1) {
      if (i > 0) entries(tile, len, e0, e1);
      info[i] = request(tile, i, e0, e1);
    }
  }
  // ---- the query as byte planes
  for (int h = warp; h < HEADS; h += AK_WARPS) {
    float x[S], top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int d = lane + 32 * i;
      x[i] = h < nh && d < c.D ? load_any(a.q, s * a.q_stride + int64_t(h0 + h) * c.D + d, a.dtype) : 0.0f;
      top = fmaxf(top, fabsf(x[i]));
      odd = odd || !(fabsf(x[i]) <= FLT_MAX);
    }
    top = warp_max(top);
    odd = __any_sync(0xffffffffu, odd);
    if (odd) top = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      int n = top > 0.0f ? __float2int_rn(__fdiv_rn(x[i], top) * QMAX) : 0;
      const int lo = int(int8_t(n & 0xff));
      const int col = (h >> 2) * 8 + 2 * (h & 3), d = lane + 32 * i;
      if (PLANES == 3) {
        qb[NH * 8 + 2 * (h & 3) + (h >> 2)][d] = int8_t(lo);
        n = (n - lo) >> 8;
        const int mid = int(int8_t(n & 0xff));
        qb[col + 1][d] = int8_t(mid);
        qb[col][d] = int8_t((n - mid) >> 8);
      } else {
        qb[col + 1][d] = int8_t(lo);
        qb[col][d] = int8_t((n - lo) >> 8);
      }
    }
    if (PLANES == 3 && NH == 1)
      for (int i = 0; i < S; ++i) qb[8 + 2 * h + 1][lane + 32 * i] = 0;
    // a query that is not finite makes its head's result NaN
    if (lane == 0) qs[h] = odd ? __int_as_float(0x7fc00000) : top / QMAX * a.scale_log2;
  }
  __syncthreads();
  // B fragments: column g, elements 32 i + 8 t .. + 7 (the contraction order of the K words below)
  uint32_t qf[NT][S][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < S; ++i) {
      // S even: a 16-byte word covers two steps of a 64-element half; S odd: the last 32 elements by 8-byte words
      const int e = (i < (S & ~1)) ? 64 * (i >> 1) + 16 * t + 8 * (i & 1) : 32 * i + 8 * t;
      const uint2 w = *reinterpret_cast<const uint2*>(&qb[n * 8 + g][e]);
      qf[n][i][0] = w.x;
      qf[n][i][1] = w.y;
    }
  float hs[NH];   // this lane's heads: 4 n + t
#pragma unroll
  for (int n = 0; n < NH; ++n) hs[n] = qs[4 * n + t];

  float m[NH], l[NH], o[2 * S][NT][4];
#pragma unroll
  for (int n = 0; n < NH; ++n) m[n] = -INFINITY, l[n] = 0.0f;
#pragma unroll
  for (int i = 0; i < 2 * S; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][n][r] = 0.0f;

  uint32_t phase = 0;
  bool ok = true;
  for (int tile = tile0; ok && tile < c1;) {
#pragma unroll
    for (int stage = 0; stage < STAGES; ++stage, tile += STEP) {
      if (tile >= c1) break;
      const int next = tile + STAGES * STEP;
      if (next < c1) entries(next, len, e0, e1);   // arrive while this tile is worked on
      ok = ptx::mbar_wait(ptx::smem_u32(&bars[warp][stage]), phase, &abort_flag, a.status, 81);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const uint32_t kp = ring + stage * STAGE + 4 * g * P, vp = ring + stage * STAGE + 32 * P + (t >> 1) * (16 * P) + 8 * (t & 1) + 16 * g;
      const float k_step = info[stage].ks, v_step = info[stage].vs;
      const bool masked = info[stage].bad;
      // ---- scores
      int acc[2][NT][4];
#pragma unroll
      for (int mg = 0; mg < 2; ++mg) {
        uint32_t kw[2][2 * S];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int i = 0; i < S / 2; ++i) {
            const uint4 w = ptx::lds128(kp + (2 * mg + r) * P + 64 * i + 16 * t);
            kw[r][4 * i] = w.x; kw[r][4 * i + 1] = w.y; kw[r][4 * i + 2] = w.z; kw[r][4 * i + 3] = w.w;
          }
          if (S & 1) {
            const uint2 w = lds64(kp + (2 * mg + r) * P + 32 * (S - 1) + 8 * t);
            kw[r][2 * S - 2] = w.x; kw[r][2 * S - 1] = w.y;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[mg][n][r] = 0;
#pragma unroll
          for (int i = 0; i < S; ++i) mma_s8s8(acc[mg][n], kw[0][2 * i], kw[1][2 * i], kw[0][2 * i + 1], kw[1][2 * i + 1], qf[n][i][0], qf[n][i][1]);
        }
      }
      const float vs_top = fmaxf(v_step, __shfl_xor_sync(0xffffffffu, v_step, 16));
      const float vs_rel = vs_top > 0.0f ? v_step / vs_top : 0.0f;
      uint32_t pw[NH][PLANES];
      float fac[NH];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float sc[4], tm = -INFINITY;
        const float f = hs[n] * k_step;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int* x = acc[j >> 1][n] + 2 * (j & 1);
          float v = float(x[0] * 256 + x[1]);
          if (PLANES == 3) v = fmaf(v, 256.0f, float(acc[j >> 1][NT - 1][2 * (j & 1) + n]));
          sc[j] = tile + 4 * g + j < len && !masked ? v * f : -INFINITY;
          tm = fmaxf(tm, sc[j]);
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, x));
        const float mn = fmaxf(m[n], tm);
        const float alpha = m[n] == -INFINITY ? 0.0f : exp2f(m[n] - mn), beta = tm == -INFINITY ? 0.0f : exp2f(tm - mn);
        float sum = 0.0f;
        uint32_t pi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = sc[j] == -INFINITY ? 0.0f : exp2f(sc[j] - tm);
          sum += p;
          pi[j] = __float2uint_rn(p * vs_rel * PMAX);
        }
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
          l[n] *= alpha;
#pragma unroll
          for (int i = 0; i < 2 * S; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][n][r] *= alpha;
            if (PLANES == 3) {
              o[i][NT - 1][n] *= alpha;
              o[i][NT - 1][2 + n] *= alpha;
            }
          }
        }
        l[n] = fmaf(sum, beta, l[n]);
        m[n] = mn;
        fac[n] = beta * vs_top;
        if (PLANES == 3) {
          pw[n][0] = bytes_of<2>(pi[0], pi[1], pi[2], pi[3]);
          pw[n][1] = bytes_of<1>(pi[0], pi[1], pi[2], pi[3]);
          pw[n][PLANES - 1] = bytes_of<0>(pi[0], pi[1], pi[2], pi[3]);
        } else {
          pw[n][0] = bytes_of<1>(pi[0], pi[1], pi[2], pi[3]);
          pw[n][1] = bytes_of<0>(pi[0], pi[1], pi[2], pi[3]);
        }
      }
      // ---- weights to the B operand: column g = (head g / 2, plane g % 2), tokens 8 t .. 8 t + 7
      uint32_t pf[NT][2];
      const int src = 8 * t + (g >> 1);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const uint32_t hi = __shfl_sync(0xffffffffu, pw[n][0], src + 4 * b), lo = __shfl_sync(0xffffffffu, pw[n][1], src + 4 * b);
          pf[n][b] = g & 1 ? lo : hi;
        }
        if (PLANES == 3) {
          const uint32_t x = __shfl_sync(0xffffffffu, pw[0][PLANES - 1], src + 4 * b);
          const uint32_t y = NH == 2 ? __shfl_sync(0xffffffffu, pw[NH - 1][PLANES - 1], src + 4 * b) : 0u;
          pf[NT - 1][b] = g & 1 ? y : x;
        }
      }
      // ---- values
#pragma unroll
      for (int i = 0; i < 2 * S; ++i) {
        const uint2 v0 = lds64(vp + 256 * i), v1 = lds64(vp + 256 * i + 128);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          int d[4] = {0, 0, 0, 0};
          mma_s8u8(d, v0.x, v1.x, v0.y, v1.y, pf[n][0], pf[n][1]);
          const bool third = PLANES == 3 && n == NT - 1;
          const float f0 = third ? fac[0] : fac[n < NH ? n : 0], f1 = third ? fac[NH - 1] : f0;
          o[i][n][0] = fmaf(float(d[0]), f0, o[i][n][0]);
          o[i][n][1] = fmaf(float(d[1]), f1, o[i][n][1]);
          o[i][n][2] = fmaf(float(d[2]), f0, o[i][n][2]);
          o[i][n][3] = fmaf(float(d[3]), f1, o[i][n][3]);
        }
      }
      __syncwarp();   // every lane has read the stage
      if (next < c1) info[stage] = request(next, stage, e0, e1);
    }
    phase ^= 1u;
  }
  if (!ok)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);   // let copies in flight land
  // ---- planes together, warps together (the sums take the place of this warp's ring)
  float(*oacc)[P] = reinterpret_cast<float(*)[P]>(mine);
  __syncwarp();
#pragma unroll
  for (int n = 0; n < NH; ++n) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], x);
    const int h = 4 * n + t;
    if (g == 0) {
      om[warp][h] = m[n];
      ol[warp][h] = l[n];
    }
#pragma unroll
    for (int i = 0; i < 2 * S; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = fmaf(o[i][n][2 * r], 256.0f, o[i][n][2 * r + 1]);
        if (PLANES == 3) v = fmaf(v, 256.0f, o[i][NT - 1][2 * r + n]);
        oacc[h][16 * i + 8 * r + g] = v * (1.0f / PMAX);
      }
  }
  __syncthreads();
  // a part: top and sum of each head, then its P sums; 16-byte aligned
  constexpr int PART = HEADS * (P + 2);
  const int64_t slot = int64_t(s) * gridDim.y + blockIdx.y;
  float* part = a.part + (slot * a.max_chunks + chunk) * PART;
  auto finish = [&](int h, int d, float val, float den) {   // den is 0 where every block was out of range; NaN stays
    float r = den > 0.0f ? val / den : den;
    if (qs[h] != qs[h]) r = qs[h];
    if (d < c.D) store_any(a.out, orow + h * c.D + d, r, a.dtype);
  };
  for (int i = threadIdx.x; i < nh * P; i += blockDim.x) {
    const int h = i / P, d = i - h * P;
    float top = -INFINITY, den = 0.0f, val = 0.0f;
#pragma unroll
    for (int w = 0; w < AK_WARPS; ++w) top = fmaxf(top, om[w][h]);
#pragma unroll
    for (int w = 0; w < AK_WARPS; ++w) {
      const float f = om[w][h] == -INFINITY ? 0.0f : exp2f(om[w][h] - top);
      den = fmaf(ol[w][h], f, den);
      val = fmaf(reinterpret_cast<const float*>(ak_ring + size_t(w) * STAGES * STAGE)[h * P + d], f, val);
    }
    if (n_chunks == 1) {
      finish(h, d, val, den);
    } else if (a.cluster) {
      reinterpret_cast<float*>(ak_ring)[i] = val;   // (read by this thread only, above)
      if (d == 0) joined[h] = make_float2(top, den);
    } else {
      part[2 * HEADS + i] = val;
      if (d == 0) {
        part[2 * h] = top;
        part[2 * h + 1] = den;
      }
    }
  }
  if (n_chunks == 1) return;
  // ---- all chunks of this (sequence, head group), in their order, element i .. i + 3; part(x) is chunk x's
  auto join = [&](int i, auto part) {
    const int h = i / P, d = i - h * P;
    float top = -INFINITY, den = 0.0f;
    float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x0 = 0; x0 < n_chunks; x0 += AK_JOIN) {   // eight parts are requested together, their sum keeps its order
      float2 md[AK_JOIN];
      float4 v[AK_JOIN];
#pragma unroll
      for (int x = 0; x < AK_JOIN; ++x) {
        part(min(x0 + x, n_chunks - 1), h, i, md[x], v[x]);
        if (x0 + x >= n_chunks) md[x].x = -INFINITY;
      }
      float now = top;
#pragma unroll
      for (int x = 0; x < AK_JOIN; ++x) now = fmaxf(now, md[x].x);
      const float keep = top == -INFINITY ? 0.0f : exp2f(top - now);
      den *= keep;
      val = make_float4(val.x * keep, val.y * keep, val.z * keep, val.w * keep);
      top = now;
#pragma unroll
      for (int x = 0; x < AK_JOIN; ++x) {
        const float f = md[x].x == -INFINITY ? 0.0f : exp2f(md[x].x - top);
        den = fmaf(md[x].y, f, den);
        val = make_float4(fmaf(v[x].x, f, val.x), fmaf(v[x].y, f, val.y), fmaf(v[x].z, f, val.z), fmaf(v[x].w, f, val.w));
      }
    }
    finish(h, d, val.x, den);
    finish(h, d + 1, val.y, den);
    finish(h, d + 2, val.z, den);
    finish(h, d + 3, val.w, den);
  };
  if (a.cluster) {   // out of the blocks' shared memory, every block its share of the elements
    __syncwarp();
    ptx::cluster_sync_all();
    const uint32_t sums = ptx::smem_u32(ak_ring), heads = ptx::smem_u32(joined);
    for (int i = 4 * (threadIdx.x * n_chunks + chunk); i < nh * P; i += 4 * blockDim.x * n_chunks)
      join(i, [&](int x, int h, int at, float2& md, float4& v) {
        const uint32_t m2 = ptx::cluster_map(heads + 8 * h, x), v4 = ptx::cluster_map(sums + 4 * at, x);
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(md.x), "=f"(md.y) : "r"(m2));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(v4));
      });
    __syncwarp();
    ptx::cluster_sync_all();   // nobody leaves while another reads its memory
    return;
  }
  // out of global memory, by the chunk that arrives last
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.count + slot, 1) == n_chunks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* all = a.part + slot * a.max_chunks * PART;
  for (int i = 4 * threadIdx.x; i < nh * P; i += 4 * blockDim.x)
    join(i, [&](int x, int h, int at, float2& md, float4& v) {
      const float* p = all + int64_t(x) * PART;
      md = __ldcg(reinterpret_cast<const float2*>(p + 2 * h));
      v = __ldcg(reinterpret_cast<const float4*>(p + 2 * HEADS + at));
    });
  if (threadIdx.x == 0) a.count[slot] = 0;
}

template <int S, int PLANES>
static cudaError_t attn_kv8_launch(int nh, dim3 grid, cudaStream_t st, const AttnKv8Args& a) {
  auto kern = nh == 1 ? attn_kv8_kernel<S, PLANES, 1> : attn_kv8_kernel<S, PLANES, 2>;
  constexpr size_t smem = AttnKv8Ring<S>::SMEM;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)); e != cudaSuccess) return e;
  if (!a.cluster) return launch_kernel(kern, grid, dim3(AK_WARPS * 32), smem, st, true, a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(AK_WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = grid.x;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

// ------------------------------------------------------------------------------------------------ arguments
static int kv8_check(const char* who, const simp_kv8_cache* c, const int32_t* table, int64_t table_stride, Kv8View& v) {
  SIMP_REQUIRE(c, SIMP_ERR_ARG, "%s: cache is null", who);
  SIMP_REQUIRE(c->head_dim >= 1 && c->head_dim <= 128, SIMP_ERR_SHAPE, "%s: head_dim %lld outside 1 .. 128", who, (long long)c->head_dim);
  SIMP_REQUIRE(c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128, SIMP_ERR_SHAPE,
               "%s: block_tokens %lld is not 16, 32, 64 or 128", who, (long long)c->block_tokens);
  SIMP_REQUIRE(c->n_blocks >= 1 && c->n_blocks <= INT_MAX && c->n_kv_heads >= 1 && c->n_kv_heads <= 65535, SIMP_ERR_SHAPE,
               "%s: %lld blocks of %lld heads", who, (long long)c->n_blocks, (long long)c->n_kv_heads);
  SIMP_REQUIRE(c->k && c->v && c->k_scales && c->v_scales && table, SIMP_ERR_ARG, "%s: null pointer", who);
  SIMP_REQUIRE(aligned_to(c->k, 16) && aligned_to(c->v, 16), SIMP_ERR_ARG, "%s: the cache's k and v must be 16-byte aligned", who);
  SIMP_REQUIRE(table_stride >= 1 && table_stride <= INT_MAX / c->block_tokens, SIMP_ERR_SHAPE, "%s: table_stride %lld", who, (long long)table_stride);
  v = Kv8View{c->k, c->v, c->k_scales, c->v_scales, table, table_stride, int(c->n_blocks), int(c->block_tokens), int(c->n_kv_heads),
              int(c->head_dim), int((c->head_dim + 31) / 32 * 32), 31 - __builtin_clz(unsigned(c->block_tokens))};
  return SIMP_OK;
}

static int kv8_rows(const char* who, bool write, const simp_kv8_cache* cache, const int32_t* table, int64_t table_stride, void* k, void* v,
                    int64_t kv_stride, const int32_t* off, const int32_t* starts, int64_t n_seqs, int64_t total, int dtype) {
  Kv8View c;
  SIMP_REQUIRE(dtype_ok(dtype), SIMP_ERR_ARG, "%s: unknown dtype %d", who, dtype);
  SIMP_REQUIRE(n_seqs >= 0 && total >= 0, SIMP_ERR_ARG, "%s: negative size", who);
  if (int rc = kv8_check(who, cache, table, table_stride, c)) return rc;
  if (n_seqs == 0 || total == 0) return SIMP_OK;
  SIMP_REQUIRE(n_seqs < INT_MAX && total <= INT_MAX, SIMP_ERR_SHAPE, "%s: too many sequences or rows", who);
  SIMP_REQUIRE(k && v && off && starts, SIMP_ERR_ARG, "%s: null pointer", who);
  const int64_t row = int64_t(c.G) * c.D;
  if (kv_stride == 0) kv_stride = row;
  SIMP_REQUIRE(kv_stride >= row, SIMP_ERR_SHAPE, "%s: kv_stride %lld is shorter than a row", who, (long long)kv_stride);
  SIMP_REQUIRE(aligned_to(k, dtype_size(dtype)) && aligned_to(v, dtype_size(dtype)), SIMP_ERR_ARG, "%s: misaligned pointer", who);
  if (int rc = ensure_ready()) return rc;
  DeviceScope dev;
  cudaStream_t st = ctx().stream;
  // a sequence of n rows touches at most (n - 1) / bt + 2 blocks, and never more than n
  const dim3 grid(unsigned(std::min<int64_t>(total, total / c.bt + 2 * n_seqs)), unsigned(c.G), 2);   // z: K, V
  int* status = ctx().dev_status;
  const unsigned threads = unsigned((c.bt / 16 * (c.pitch / 4) + 31) / 32 * 32);
  const size_t four = 4 * dtype_size(dtype);
  const bool vec = c.D % 4 == 0 && kv_stride % 4 == 0 && aligned_to(k, four) && aligned_to(v, four);
  cudaError_t e = cudaSuccess;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    if (write) {
      auto kern = vec ? kv8_append_kernel<T, true> : kv8_append_kernel<T, false>;
      e = launch_kernel(kern, grid, dim3(threads), 0, st, true, c, static_cast<const T*>(k), static_cast<const T*>(v), kv_stride, off, starts, int(n_seqs), total, status);
    } else {
      auto kern = vec ? kv8_read_kernel<T, true> : kv8_read_kernel<T, false>;
      e = launch_kernel(kern, grid, dim3(threads), 0, st, true, c, static_cast<T*>(k), static_cast<T*>(v), kv_stride, off, starts, int(n_seqs), total, status);
    }
  };
  if (dtype == SIMP_DTYPE_F32) go(float());
  else if (dtype == SIMP_DTYPE_F16) go(__half());
  else go(__nv_bfloat16());
  SIMP_REQUIRE(e == cudaSuccess, SIMP_ERR_CUDA, "%s launch failed: %s", who, cudaGetErrorString(e));
  return SIMP_OK;
}

}  // namespace simp

using namespace simp;

SIMP_API int simp_gpu_kv8_append(const simp_kv8_cache* cache, const int32_t* block_table_dev, int64_t table_stride, const void* k_dev,
                                 const void* v_dev, int64_t kv_stride, const int32_t* offsets_dev, const int32_t* starts_dev,
                                 int64_t n_seqs, int64_t total, int dtype) {
  return kv8_rows("kv8_append", true, cache, block_table_dev, table_stride, const_cast<void*>(k_dev), const_cast<void*>(v_dev), kv_stride,
                  offsets_dev, starts_dev, n_seqs, total, dtype);
}

SIMP_API int simp_gpu_kv8_read(const simp_kv8_cache* cache, const int32_t* block_table_dev, int64_t table_stride, void* k_dev, void* v_dev,
                               int64_t kv_stride, const int32_t* offsets_dev, const int32_t* starts_dev, int64_t n_seqs, int64_t total,
                               int dtype) {
  return kv8_rows("kv8_read", false, cache, block_table_dev, table_stride, k_dev, v_dev, kv_stride, offsets_dev, starts_dev, n_seqs, total,
                  dtype);
}

SIMP_API int simp_gpu_attn_kv8(const simp_kv8_cache* cache, const int32_t* block_table_dev, int64_t table_stride, const void* q_dev,
                               void* out_dev, int64_t q_stride, int64_t out_stride, const int32_t* lengths_dev, int64_t n_seqs,
                               int64_t max_len, int64_t n_heads, float scale, int dtype) {
  AttnKv8Args a{};
  SIMP_REQUIRE(dtype_ok(dtype), SIMP_ERR_ARG, "attn_kv8: unknown dtype %d", dtype);
  SIMP_REQUIRE(n_seqs >= 0 && max_len >= 0, SIMP_ERR_ARG, "attn_kv8: negative size");
  if (int rc = kv8_check("attn_kv8", cache, block_table_dev, table_stride, a.c)) return rc;
  SIMP_REQUIRE(n_heads >= 1 && n_heads % a.c.G == 0 && n_heads <= 65535, SIMP_ERR_SHAPE, "attn_kv8: %lld query heads over %d key/value heads",
               (long long)n_heads, a.c.G);
  SIMP_REQUIRE(max_len <= table_stride * a.c.bt, SIMP_ERR_SHAPE, "attn_kv8: max_len %lld exceeds the table's %lld blocks of %d tokens",
               (long long)max_len, (long long)table_stride, a.c.bt);
  SIMP_REQUIRE(max_len <= (1 << 30), SIMP_ERR_SHAPE, "attn_kv8: max_len %lld exceeds 2^30", (long long)max_len);
  if (n_seqs == 0) return SIMP_OK;
  SIMP_REQUIRE(n_seqs <= 65535, SIMP_ERR_SHAPE, "attn_kv8: more than 65535 sequences");
  SIMP_REQUIRE(q_dev && out_dev && lengths_dev, SIMP_ERR_ARG, "attn_kv8: null pointer");
  const int64_t row = n_heads * a.c.D;
  if (q_stride == 0) q_stride = row;
  if (out_stride == 0) out_stride = row;
  SIMP_REQUIRE(q_stride >= row && out_stride >= row, SIMP_ERR_SHAPE, "attn_kv8: a stride is shorter than a row");
  SIMP_REQUIRE(aligned_to(q_dev, dtype_size(dtype)) && aligned_to(out_dev, dtype_size(dtype)), SIMP_ERR_ARG, "attn_kv8: misaligned pointer");
  if (int rc = ensure_ready()) return rc;
  DeviceScope dev;
  a.q = q_dev;
  a.out = out_dev;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.lengths = lengths_dev;
  a.status = ctx().dev_status;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.rep = int(n_heads / a.c.G);
  a.max_len = int(max_len);
  a.dtype = dtype;
  const int nh = a.rep > 4 ? 2 : 1;
  const int64_t groups = int64_t(a.c.G) * ((a.rep + 4 * nh - 1) / (4 * nh));
  const int64_t slots = n_seqs * groups;
  SIMP_REQUIRE(groups <= 65535, SIMP_ERR_SHAPE, "attn_kv8: too many heads");
  // Chunks of at least a tile per warp.  One sequence: as many blocks as run at once (three per SM; 131072 tokens, 8 x 128: 56 us
  // with 54 chunks, 67 with 109, 87 with 205).  Several, whose lengths differ: twice as many and none longer than 2048 tokens, so
  // that the longest does not end alone (64 sequences of up to 8097: 126 us, 135 in one chunk each, 131 with 1024).  But no more
  // than 32 (64 from 32768 tokens on), for the block that arrives last joins eight at a time: 16384 tokens of 1 x 128 with 8
  // query heads 19 us with 32, 23 with 64, 35 with 128; 131072 tokens 58, 45 and 93 (with 444).
  const int64_t least = 32 * AK_WARPS, waves = n_seqs == 1 ? 3 : 6, most = max_len < 32768 ? 32 : 64;
  const int64_t want = std::min(most, std::max<int64_t>(1, waves * int64_t(ctx().sm_count) / slots));
  a.chunk = int(std::max(least, cdiv(cdiv(std::max<int64_t>(max_len, 1), want), least) * least));
  if (n_seqs > 1) a.chunk = std::min(a.chunk, 2048);
  a.max_chunks = int(std::max<int64_t>(1, cdiv(max_len, a.chunk)));
  // Up to 4096 tokens where all blocks run at once: eight chunks at most, a cluster that joins them out of its shared memory,
  // which takes 1.3 us where global memory takes 2.8.  1024 tokens, 8 x 64: 6.2 -> 5.4 us, 2048: 7.7 -> 6.8, 4096: 9.8 -> 9.2, but
  // 8192: 11.1 -> 13.4.  (Clusters that do not all fit at once: 8 sequences of 1024, 8 x 64: 7.3 -> 11.8.)
  if (a.max_chunks > 1 && max_len <= 4096) {
    const int64_t share = cdiv(cdiv(max_len, AK_JOIN), least) * least, parts = cdiv(max_len, share);
    if (slots * parts <= 3 * int64_t(ctx().sm_count)) {
      a.cluster = true;
      a.chunk = int(share);
      a.max_chunks = int(parts);
    }
  }
  if (a.max_chunks > 1 && !a.cluster) {
    a.part = static_cast<float*>(scratch(size_t(slots) * a.max_chunks * 4 * nh * (a.c.pitch + 2) * 4, SCRATCH_KV8_PART));
    if (!a.part) return scratch_failed("attn_kv8");
    a.count = static_cast<int*>(scratch(size_t(slots) * 4, SCRATCH_KV8_COUNT, true));
    if (!a.count) return scratch_failed("attn_kv8");
  }
  const dim3 grid(unsigned(a.max_chunks), unsigned(groups), unsigned(n_seqs));
  cudaStream_t st = ctx().stream;
  const bool wide = dtype == SIMP_DTYPE_F32;
  cudaError_t e = cudaSuccess;
  switch (a.c.pitch / 32) {
    case 1: e = wide ? attn_kv8_launch<1, 3>(nh, grid, st, a) : attn_kv8_launch<1, 2>(nh, grid, st, a); break;
    case 2: e = wide ? attn_kv8_launch<2, 3>(nh, grid, st, a) : attn_kv8_launch<2, 2>(nh, grid, st, a); break;
    case 3: e = wide ? attn_kv8_launch<3, 3>(nh, grid, st, a) : attn_kv8_launch<3, 2>(nh, grid, st, a); break;
    default: e = wide ? attn_kv8_launch<4, 3>(nh, grid, st, a) : attn_kv8_launch<4, 2>(nh, grid, st, a); break;
  }
  SIMP_REQUIRE(e == cudaSuccess, SIMP_ERR_CUDA, "attn_kv8 launch failed: %s", cudaGetErrorString(e));
  return SIMP_OK;
}
