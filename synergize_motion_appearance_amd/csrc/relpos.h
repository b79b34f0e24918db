// What the forward and backward kernels of the attention with a relative position bias share (relpos_attn.hip, relpos_attn_bwd.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "smx.h"
#include "smx_common.h"
#include "bf16.h"

namespace relpos {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));        // (HIP's own uint4 is a struct: its copies kept staging registers in scratch memory)
typedef u32x4 u32x4a8 __attribute__((aligned(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MAP_MAX = 2049;         // entries of a bucket map
constexpr int TABLE_PAD = 96;         // entries a 64-key x 32-query tile can reach beyond the map's ends while it touches the map

// ---- fp32 operands on the half-precision matrix pipe ("f16x3") ----------------------------------------------------------------
// x = (h1 + h2) 2^-k with two IEEE halves: 22 significand bits; a product is h1 g1 + h1 g2 + h2 g1, the dropped h2 g2 is 2^-22 of it.  k brings the largest |x|
// that shares it to [2^14, 2^15): values down to 2^-16 of that keep all 22 bits, smaller ones are off by at most 2^-40 of it.  Rows that a wave keeps in
// registers are split there, each with a k of its own (own_rows).  Rows that are staged -- read by every block of the other side -- are split once, by a
// pass before: planes [B][heads][rows rounded up to 64][dh rounded up to 32] of h1 and of h2 with one k per 64 rows; keys that nobody may see,
// queries that see none and the columns from dh on are zeros.  Where a product sums over staged rows, the k of the tile joins the factor of the other operand (Unit).
struct Split {
  const float* src; long long bs; int ld, heads, rows, kv, flip;  // kv: rows of keys (masks and lengths apply); flip: odd rows negated
  _Float16* hi; _Float16* lo;                                   // planes
  float* inv;                                                   // [B][heads][tiles of 64] 2^-k
  const float* o;                                               // gradient rows: the output, for D_i = dO_i . o_i (dense, as src)
  float* dd;                                                    // [B][heads][rows rounded up to 64]
};

struct RP {
  const void* q; const void* k; const void* v; void* o;
  const float* table; const int* map; const uint8_t* mask; const int* kv_len;
  float* lse; const float* d_o; float* dq; float* dk; float* dv; float* dtable;
  long long q_bs, k_bs, v_bs, o_bs;
  int ldq, ldk, ldv, ldo;
  int B, H, Hkv, G, L, S, dh, map_lo, map_n, nb, causal, has_start, q_start;
  float scale;
  // keys that a query of the sample can see: with a causal rule none behind the last query's position
  __device__ __forceinline__ int keys(int b) const {
    const int n = kv_len ? max(0, min(kv_len[b], S)) : S;
    return causal && has_start ? max(0, min(n, q_start + L)) : n;
  }
  __device__ __forceinline__ int pos0(int n) const { return has_start ? q_start : n - L; }
  // backward: a query with no key left, by the forward's lse.  What it and its gradient hold must not meet the zeros of its weights
  __device__ __forceinline__ bool empty(int b, int h, int i) const { return lse[((long long)b * H + h) * L + i] == INFINITY; }
  __device__ __forceinline__ int entry(int delta) const { return max(0, min(delta - map_lo, map_n - 1)); }
};

static inline int up64(int n) { return (n + 63) & ~63; }
static inline int dhp(int dh) { return (dh + 31) / 32 * 32; }
static inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// the launchers of relpos_attn.hip
int check(const smx_relpos_desc* d, RP& p, bool bwd);
int64_t split_bytes(int B, int heads, int rows, int dh);        // planes and scales
char* split_setup(Split& s, char* ws, const float* src, long long bs, int ld, int B, int heads, int rows, int dh, bool kv);
int split_launch(const RP& p, const Split* s, int n, hipStream_t st);

// ---- matrix operands -----------------------------------------------------------------------------------------------------------
template <int NL>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (NL == 1) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
// c += a b over the levels, the smallest products first
template <int NL>
__device__ __forceinline__ f32x16 mfma_levels(const u32x4 (&a)[NL], const u32x4 (&b)[NL], f32x16 c) {
  if constexpr (NL == 2) {
    c = mfma<2>(a[1], b[0], c);
    c = mfma<2>(a[0], b[1], c);
  }
  return mfma<NL>(a[0], b[0], c);
}
// eight fp32, times w, -> two halves' fragments.  The second half is one v_fma_mix_f32 a value (v w - h1) and the rounding in pairs; a caller without
// a factor passes one(), a 1 that the compiler does not see as such: it would fall back to a conversion and a subtraction.
__device__ __forceinline__ float one() {
  float x = 1.f;
  asm volatile("" : "+s"(x));
  return x;
}
__device__ __forceinline__ void to_levels(const float* v, float w, u32x4 (&f)[2]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1];
    h[i] = cvt2_f16(a * w, b * w);
    l[i] = cvt2_f16(fmaf(a, w, -f16lo(h[i])), fmaf(b, w, -f16hi(h[i])));
  }
  f[0] = u32x4{h[0], h[1], h[2], h[3]};
  f[1] = u32x4{l[0], l[1], l[2], l[3]};
}
// the same for weights, whose first half is taken of v itself
__device__ __forceinline__ void to_halves(const float* v, float w1, u32x4 (&f)[2]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = cvt2_f16(v[2 * i], v[2 * i + 1]);
    l[i] = cvt2_f16(fmaf(v[2 * i], w1, -f16lo(h[i])), fmaf(v[2 * i + 1], w1, -f16hi(h[i])));
  }
  f[0] = u32x4{h[0], h[1], h[2], h[3]};
  f[1] = u32x4{l[0], l[1], l[2], l[3]};
}

// weights that meet values in bf16: two bf16 parts, together within 2^-16 of the weight (one, within 2^-8, would cost an output as much again as the rounding of
// the output itself; the row's sum takes the weights as they are)
__device__ __forceinline__ void to_bf16_parts(const float* v, u32x4 (&f)[2]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1];
    h[i] = cvt2_bf16(a, b);
    l[i] = cvt2_bf16(a - __uint_as_float(h[i] << 16), b - __uint_as_float(h[i] & 0xffff0000u));
  }
  f[0] = u32x4{h[0], h[1], h[2], h[3]};
  f[1] = u32x4{l[0], l[1], l[2], l[3]};
}

// lanes 0..31: bit k of a wave-uniform word, lanes 32..63: bit k + 4, as a select's lane mask (scalar work, one select a value)
__device__ __forceinline__ bool row_bit(unsigned long long word, int k) {
  const unsigned a = -(unsigned)((word >> k) & 1), b = -(unsigned)((word >> (k + 4)) & 1);
  return __builtin_amdgcn_inverse_ballot_w64((unsigned long long)b << 32 | a);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// a tile's row r of the 32x32 accumulator layout that a lane's register i holds: (i & 3) + 8 (i >> 2) + 4 (lane >> 5)
__device__ __forceinline__ constexpr int crow(int i) { return (i & 3) + 8 * (i >> 2); }

// Tiles in LDS: [row][DHP] 16-bit values, rows 16 bytes further apart than they are long: both the row fragments (16 B at row lane & 31) and the transposed
// reads (8 B at four rows by four columns a lane group) then fall on different banks.
template <int DHP> constexpr int ROWB = DHP * 2 + 16;

// operand fragment of 16 columns kk of the tile's row r0 + (lane & 31)
template <int DHP>
__device__ __forceinline__ u32x4 row_frag(const char* tile, int r0, int kk) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const u32x4*>(tile + (r0 + (lane & 31)) * ROWB<DHP> + kk * 32 + (lane >> 5) * 16);
}
// the transposed fragment: lane holds column 32 dt + (lane & 31) at the 16 rows from r0 on that an accumulator's eight registers hold
// (4 hh + 0..3 and 8 + 4 hh + 0..3): two transposing reads of 4 rows x 16 columns a lane group
template <int DHP>
__device__ __forceinline__ u32x4 col_frag(char* tile, int r0, int dt) {
  const int lane = threadIdx.x & 63, l = lane & 15;
  char* at = tile + (r0 + (lane >> 5) * 4 + (l >> 2)) * ROWB<DHP> + dt * 64 + ((lane >> 4) & 1) * 32 + (l & 3) * 8;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * ROWB<DHP>));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// the other 32 lanes' value
__device__ __forceinline__ float other_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^k and 2^-k for values up to m.  Nothing but zeros: 2^-k reads 0.  An infinity: 2^-k reads infinity, so that what its tile enters is no number -- with a
// finite one the other values of the tile would be lost without a sign.
__device__ __forceinline__ float pow2_of(float m, float& inv) {
  const int e = m > 0.f ? max((int)(__float_as_uint(m) >> 23), 15) - 127 : 14;     // floor(log2 m); 2^(14 - e) stays a normal number
  inv = m == 0.f ? 0.f : e == 128 ? INFINITY : __uint_as_float((unsigned)(e - 14 + 127) << 23);
  return __uint_as_float((unsigned)(14 - e + 127) << 23);
}

// 32 fp32 rows as fragments in registers: lane & 31 the row at x, columns 16 kk + 8 (lane >> 5) + 0..7; -> the row's 2^-k
template <int DHP>
__device__ __forceinline__ float own_rows(u32x4 (&f)[DHP / 16][2], const float* x, bool in, int dh) {
  float v[DHP / 16][8], m = 0.f, inv;
  const int hh = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int kk = 0; kk < DHP / 16; ++kk)
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const int d = kk * 16 + hh * 8 + i;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && d < dh) y = *reinterpret_cast<const float4*>(x + d);
      v[kk][i] = y.x; v[kk][i + 1] = y.y; v[kk][i + 2] = y.z; v[kk][i + 3] = y.w;
      m = fmaxf(m, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
    }
  const float sc = pow2_of(other_max(m), inv);
#pragma unroll
  for (int kk = 0; kk < DHP / 16; ++kk) {
    to_levels(v[kk], sc, f[kk]);
  }
  return inv;
}

// An accumulator that sums over staged rows is kept in units of a 2^-k.  A tile of larger values first brings it to its own (exactly: powers of two); a smaller
// one enters with the factor 2^log2w <= 1 on its other operand, down to 2^-8 (22 bits are still there: the factors' largest are 2^6 and more); below that
// the accumulator comes down to the tile, as rows that give the larger tile no weight must not lose the smaller one's bits -- by at most 2^60 from
// the largest, so that no sum leaves fp32's range.  A tile of zeros changes nothing.
struct Unit {
  int e = 0, most = 0;                                          // exponent bits of 2^-k and of the largest so far, wave-uniform; 0: none yet
  template <int N> __device__ __forceinline__ int enter(int t, f32x16 (&acc)[N]) {
    if (t == 0) return 0;
    most = max(most, t);
    if (t > e || t < e - 8) {
      const int to = max(t, most - 60);
      if (to != e) {
        const float r = __uint_as_float((unsigned)max(127 + e - to, 0) << 23);     // (the first tile: the accumulators are zeros)
        e = to;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[n][i] *= r;
      }
    }
    return max(t - e, -100);
  }
  __device__ __forceinline__ float inv() const { return __uint_as_float((unsigned)e << 23); }     // (0: no tile came)
};
// the exponent bits of a power of two that all lanes hold, and back
__device__ __forceinline__ int bits_of(float pow2) { return __builtin_amdgcn_readfirstlane(__float_as_uint(pow2) >> 23); }
__device__ __forceinline__ float pow2_bits(int e) { return __uint_as_float((unsigned)e << 23); }
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// keys (queries) a step: 64, or 32 where two operands of 128 columns in two halves each would not leave room for a second block on a CU
template <int DHP, int NL> constexpr int STEP = NL == 2 && DHP == 128 ? 32 : 64;

// Work order: consecutive block ids go to the 8 XCDs in turn; this gives each XCD a run of consecutive work items, so that the blocks that read the
// same keys share an L2.
__device__ __forceinline__ unsigned xcd_order(unsigned id, unsigned n) {
  const unsigned x = id & 7, s = id >> 3, q = n >> 3, r = n & 7;
  return x < r ? x * (q + 1) + s : r * (q + 1) + (x - r) * q + s;
}

// Which of a head's n blocks, and which of the heads, a block works on.  Blocks of one length: runs of heads by XCD.  With a causal rule a head's blocks differ, 0 the
// longest: all heads' longest go first (a chip that ends on long blocks waits for them: 1.3 waves a SIMD on average instead of 1.9), the heads of one XCD
// consecutive ones where they are a multiple of 8: 2 x 16 heads of 8192 x 8192 bf16 368 us instead of 405, 4096 x 4096 with its backward 1144 instead
// of 1235.  Ragged samples: heads in turn, so that no XCD has only the short ones (3 x 6 heads of 1311 and fewer keys: 63 us instead of 84).
struct Work { int i, head; };
__device__ __forceinline__ Work work_of(unsigned id, int n, int heads, int causal, bool ragged) {
  if (!causal && !ragged) { id = xcd_order(id, gridDim.x); return {(int)(id % n), (int)(id / n)}; }
  if (ragged || (heads & 7)) return {(int)(id / heads), (int)(id % heads)};
  const unsigned m = heads >> 3, s = id >> 3;
  return {(int)(s / m), (int)((id & 7) * m + s % m)};
}

// the head's bias in log2 units by map entry, TABLE_PAD more of its ends' values on both sides
__device__ __forceinline__ void fill_bias(float* lut, const RP& p, int h) {
  for (int t = threadIdx.x; t < p.map_n + 2 * TABLE_PAD; t += blockDim.x) {
    const int e = max(0, min(t - TABLE_PAD, p.map_n - 1));
    lut[t] = p.table[(long long)p.map[e] * p.H + h] * LOG2E;
  }
}

}  // namespace relpos
