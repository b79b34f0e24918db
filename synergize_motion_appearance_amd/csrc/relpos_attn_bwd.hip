// Attention with a learned relative position bias by buckets, backward (include/smx.h: smx_attention_relpos_bwd_f32):
//   D_i = sum_d dO_id o_id,  dS_ij = P_ij (dO_i . v_j - D_i),  dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij dO_i,  dtable[b][h] = sum of dS_ij over the pairs of bucket b
// P is computed again from q, k and the rows' lse (log2 units; +inf for a row with no key left, so that 2^{s - lse} is 0 there).  All products in the
// f16x3 arithmetic of relpos.h.  Two passes over the pairs, one that owns queries (dq, dtable) and one that owns keys (dk, dv): seven products
// instead of five, but no sum crosses blocks, so that nothing is atomic and results repeat bit for bit.
// The matrix cores cut the bits below an accumulator's last towards -inf (some 0.1 of its last bit on average): dP as a whole is a little low, D is not,
// and a bucket's sum over millions of pairs of mixed signs shows it (dtable off by 3e-6 to 5e-6 of its norm at 1024 x 1024).  V's odd rows enter with
// the opposite sign, so that the cuts of neighbouring keys cancel in every such sum.
#include "relpos.h"

namespace {
using namespace relpos;

struct Bwd {
  Split q, k, v, g;
  float* part;                                                   // [B][H][query blocks][map_n + 2 DPAD] sums of dS by distance
};
constexpr int DPAD = 64;                                         // entries a 32 x 32 tile reaches beyond the map's ends while it touches the map

// dS has no range known beforehand (it follows P, down to 2^-S and less): each column of the accumulators carries a power of two f of its own, chosen when the
// column's first |dS| arrive ([2^9, 2^10)) and again, exactly, when they outgrow a half.
template <int N>
__device__ __forceinline__ void follow(float top, float& f, f32x16 (&acc)[N]) {
  top = other_max(top);
  if (!__ballot(top * f > 32768.f)) return;
  if (top * f > 32768.f) {
    const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
    const float fn = __uint_as_float((unsigned)(9 - e + 127) << 23), r = fn / f;
    f = fn;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][i] *= r;
  }
}
constexpr float F0 = 1.2676506002282294e30f;                     // 2^100: before the first dS that is not zero

// stage TK rows of four planes (h1, h2 of two operands) through registers
template <int DHP, int NT>
struct Stage {
  static constexpr int TK = DHP == 128 ? 32 : 64, RB = ROWB<DHP>, PLANE = TK * RB, CPR = DHP / 8, NCH = TK * CPR / NT;
  u32x4 reg[4][NCH];
  __device__ __forceinline__ void load(const Split& x, const Split& y, long long at) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const long long e = at + (c * NT + threadIdx.x) * 8;
      reg[0][c] = *reinterpret_cast<const u32x4*>(x.hi + e); reg[1][c] = *reinterpret_cast<const u32x4*>(x.lo + e);
      reg[2][c] = *reinterpret_cast<const u32x4*>(y.hi + e); reg[3][c] = *reinterpret_cast<const u32x4*>(y.lo + e);
    }
  }
  __device__ __forceinline__ void store(char* sm) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int e = c * NT + threadIdx.x, off = e / CPR * RB + e % CPR * 16;
#pragma unroll
      for (int l = 0; l < 4; ++l) *reinterpret_cast<u32x4*>(sm + l * PLANE + off) = reg[l][c];
    }
  }
};

// fragments of 32 rows of an operand that stays in registers
template <int DHP>
__device__ __forceinline__ void own_rows(u32x4 (&f)[DHP / 16][2], const Split& s, long long row, bool in) {
  const long long at = row * DHP + ((threadIdx.x & 63) >> 5) * 8;
#pragma unroll
  for (int kk = 0; kk < DHP / 16; ++kk) {
    f[kk][0] = in ? *reinterpret_cast<const u32x4*>(s.hi + at + kk * 16) : u32x4{0, 0, 0, 0};
    f[kk][1] = in ? *reinterpret_cast<const u32x4*>(s.lo + at + kk * 16) : u32x4{0, 0, 0, 0};
  }
}

// 32 x 32 product of staged rows (planes at t, t + PLANE) with owned rows
template <int DHP>
__device__ __forceinline__ f32x16 rows_times(const char* t, int plane, int r0, const u32x4 (&own)[DHP / 16][2]) {
  f32x16 a = zero16();
#pragma unroll
  for (int kk = 0; kk < DHP / 16; ++kk) {
    const u32x4 f[2] = {row_frag<DHP>(t, r0, kk), row_frag<DHP>(t + plane, r0, kk)};
    a = mfma_levels<2>(f, own[kk], a);
  }
  return a;
}

// dq and the sums of dS by distance.  A wave: 32 queries as columns, K and V staged 64 keys at a time (32 for DHP = 128); S^T = K Q^T, dP^T = V dO^T, then
// dQ^T += K^T dS^T with dS^T from the registers.  dS by distance: in a tile that lies beyond the map's ends all pairs are of one entry, a
// lane adds its own; elsewhere lane t collects the tile's diagonal key - query = t - 31 through lane permutes, register by register, and adds it to the
// wave's table in LDS -- one lane an entry, tile after tile: a fixed order without atomics.
template <int DHP>
__global__ __launch_bounds__(256, DHP == 128 ? 1 : 2) void relpos_bwd_q_kernel(RP p, Bwd a) {
  using ST = Stage<DHP, 256>;
  constexpr int TK = ST::TK, NU = TK / 32, KS = DHP / 16, DT = DHP / 32;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  const int nent = p.map_n + 2 * DPAD;
  float* lut = reinterpret_cast<float*>(sm + 4 * ST::PLANE);
  float* dacc = lut + p.map_n + 2 * TABLE_PAD;                   // [4 waves][nent]
  __shared__ unsigned long long seen;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
  const int nq = (p.L + 127) / 128, up = (p.L + 63) & ~63;
  unsigned id = xcd_order(blockIdx.x, gridDim.x);
  const int qb = nq - 1 - id % nq;
  id /= nq;
  const int h = id % p.H, b = id / p.H, hk = h / p.G;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const int q0 = qb * 128 + wave * 32, qi = q0 + (lane & 31), pos = pos0 + qi;
  const int wlast = pos0 + min(q0 + 31, p.L - 1);
  const int kend = p.causal ? min(n, pos0 + min(qb * 128 + 127, p.L - 1) + 1) : n;
  const int ntiles = kend > 0 ? (kend + TK - 1) / TK : 0;
  const long long row = ((long long)b * p.H + h) * p.L + qi, prow = ((long long)b * p.H + h) * up + qi;

  fill_bias(lut, p, h);
  for (int t = threadIdx.x; t < 4 * nent; t += 256) dacc[t] = 0.f;
  dacc += wave * nent;
  const float first_bias = p.table[(long long)p.map[0] * p.H + h] * LOG2E, last_bias = p.table[(long long)p.map[p.map_n - 1] * p.H + h] * LOG2E;
  const int at2 = (b * p.Hkv + hk) * 2;
  const float inv_k = a.k.pow2[at2 + 1], inv_v = a.v.pow2[at2 + 1], inv_g = a.g.pow2[at2 + 1];
  const float sc = p.scale * LOG2E * a.q.pow2[at2 + 1] * inv_k;
  const float lse = qi < p.L ? p.lse[row] : INFINITY;
  const float D = qi < p.L ? a.g.dd[prow] * a.g.pow2[at2] * a.v.pow2[at2] : 0.f;       // in the units of dP's accumulators
  u32x4 qf[KS][2], gf[KS][2];
  own_rows<DHP>(qf, a.q, prow, qi < up);
  own_rows<DHP>(gf, a.g, prow, qi < up);
  f32x16 dq[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dq[t] = zero16();
  float f = F0, below = 0.f, above = 0.f;

  ST st;
  unsigned long long sreg = 0;
  const long long kv0 = ((long long)b * p.Hkv + hk) * ((p.S + 63) & ~63);
  auto load_tile = [&](int key0) {
    st.load(a.k, a.v, (kv0 + key0) * DHP);
    if (wave == 0) {
      const int key = key0 + lane;
      sreg = __ballot(lane < TK && key < n && !(p.mask && p.mask[(long long)b * p.S + key]));
    }
  };
  if (ntiles > 0) load_tile(0);
  const unsigned long long ALL = TK == 64 ? ~0ull : 0xffffffffull;
  for (int t = 0; t < ntiles; ++t) {
    const int key0 = t * TK;
    __syncthreads();                                             // the tile before has been read
    st.store(sm);
    if (threadIdx.x == 0) seen = sreg;
    __syncthreads();
    if (t + 1 < ntiles) load_tile(key0 + TK);
    const unsigned long long left = seen;
    if (!left || q0 >= p.L || (p.causal && key0 > wlast)) continue;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x16 s = rows_times<DHP>(sm, ST::PLANE, u * 32, qf);
      const f32x16 dp = rows_times<DHP>(sm + 2 * ST::PLANE, ST::PLANE, u * 32, gf);
      const int e0 = key0 + u * 32 - (pos0 + q0) - p.map_lo;     // entry of the tile's first key and first query; the others: + key - query
      const bool lo = e0 + 31 <= 0, hi = e0 - 31 >= p.map_n - 1;
      if (lo || hi) {
        const float c = (lo ? first_bias : last_bias) - lse;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, c));
      } else {
        const float* lp = lut + TABLE_PAD + e0 - (lane & 31) + 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, lp[crow(r)]) - lse);
      }
      if (left != ALL) {
        const unsigned long long mine = left >> (4 * hh + u * 32);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((mine >> crow(r)) & 1)) s[r] = 0.f;
      }
      if (p.causal && key0 + u * 32 + 31 > pos0 + q0) {
        const int d = key0 + u * 32 + 4 * hh - pos;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (d + crow(r) > 0) s[r] = 0.f;
      }
      float ds[16], top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) { ds[r] = s[r] * ((r & 1 ? -dp[r] : dp[r]) - D); top = fmaxf(top, fabsf(ds[r])); }
      if (lo || hi) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += ds[r];
        if (lo) below += sum; else above += sum;
      } else {
        float sum = 0.f;
        const int t0 = 31 - lane;                                // the diagonal's query in key row 0
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int q1 = t0 + crow(r), q2 = q1 + 4;              // lanes 0..31 hold key row crow(r), lanes 32..63 key row crow(r) + 4
          const float v1 = __uint_as_float(__builtin_amdgcn_ds_bpermute(q1 * 4, __float_as_uint(ds[r])));
          const float v2 = __uint_as_float(__builtin_amdgcn_ds_bpermute((q2 + 32) * 4, __float_as_uint(ds[r])));
          sum += (unsigned)q1 < 32u ? v1 : 0.f;
          sum += (unsigned)q2 < 32u ? v2 : 0.f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // another lane wrote this entry at the tile before
        __builtin_amdgcn_wave_barrier();
        dacc[DPAD + e0 + lane - 31] += sum;                      // (lane 63: no diagonal of its own, adds 0)
      }
      follow(top, f, dq);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4 pf[2];
        to_levels<2>(ds + 8 * g, pf);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 kf[2] = {col_frag<DHP>(sm, u * 32 + g * 16, d), col_frag<DHP>(sm + ST::PLANE, u * 32 + g * 16, d)};
          dq[d] = mfma_levels<2>(kf, pf, dq[d]);
        }
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { below += __shfl_xor(below, o, 64); above += __shfl_xor(above, o, 64); }
  __syncthreads();
  if (lane == 0) { dacc[DPAD] += below; dacc[DPAD + p.map_n - 1] += above; }
  __syncthreads();
  dacc -= wave * nent;
  float* part = a.part + (((long long)b * p.H + h) * nq + qb) * nent;
  for (int t = threadIdx.x; t < nent; t += 256) part[t] = ((dacc[t] + dacc[nent + t]) + (dacc[2 * nent + t] + dacc[3 * nent + t])) * inv_g * inv_v;
  if (qi >= p.L) return;
  const float w1 = inv_g * inv_k, w2 = inv_v * p.scale, fi = 1.f / f;
  float* DQ = p.dq + ((long long)b * p.L + qi) * p.H * p.dh + h * p.dh;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * hh;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dq[d][4 * g + e] * fi * w1 * w2;
      if (c < p.dh) *reinterpret_cast<float4*>(DQ + c) = make_float4(x[0], x[1], x[2], x[3]);
    }
}

// dk and dv.  A wave: 32 keys as columns; Q and dO of the heads that share them staged 64 queries at a time (32 for DHP = 128); S = Q K^T, dP = dO V^T,
// dV^T += dO^T P, dK^T += Q^T dS.  P carries 2^14.
template <int DHP>
__global__ __launch_bounds__(256, DHP == 128 ? 1 : 2) void relpos_bwd_kv_kernel(RP p, Bwd a) {
  using ST = Stage<DHP, 256>;
  constexpr int TQ = ST::TK, NU = TQ / 32, KS = DHP / 16, DT = DHP / 32;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  float* rl = reinterpret_cast<float*>(sm + 4 * ST::PLANE);      // the tile's lse - 14
  float* rd = rl + 64;                                           // and D
  float* lut = rd + 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
  const int nk = (p.S + 127) / 128, up = (p.L + 63) & ~63;
  unsigned id = xcd_order(blockIdx.x, gridDim.x);
  const int kb = id % nk;
  id /= nk;
  const int hk = id % p.Hkv, b = id / p.Hkv;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const int k0 = kb * 128 + wave * 32, key = k0 + (lane & 31);
  const int ups = (p.S + 63) & ~63;
  const long long krow = ((long long)b * p.Hkv + hk) * ups + key;
  const int at2 = (b * p.Hkv + hk) * 2;
  const float inv_q = a.q.pow2[at2 + 1], inv_v = a.v.pow2[at2 + 1], inv_g = a.g.pow2[at2 + 1], pg = a.g.pow2[at2], pv = a.v.pow2[at2];
  const float sc = p.scale * LOG2E * inv_q * a.k.pow2[at2 + 1];
  u32x4 kf[KS][2], vf[KS][2];
  own_rows<DHP>(kf, a.k, krow, key < ups);
  own_rows<DHP>(vf, a.v, krow, key < ups);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = zero16();
  float f = F0;
  const float sign = key & 1 ? -1.f : 1.f;                       // V's odd rows are negated
  // causal: the first query that stands at this block's first key or behind it
  const int t0 = p.causal ? max(0, kb * 128 - pos0) / TQ : 0, t1 = kb * 128 < n ? (p.L + TQ - 1) / TQ : 0;
  const int per = max(0, t1 - t0), ntiles = per * p.G;
  ST st;
  float lreg = 0.f, dreg = 0.f;
  auto load_tile = [&](int t) {
    const int h = hk * p.G + t / per, i0 = (t0 + t % per) * TQ, i = i0 + threadIdx.x;
    const long long r = (long long)b * p.H + h;
    st.load(a.q, a.g, (r * up + i0) * DHP);
    if (threadIdx.x < TQ) {
      lreg = i < p.L ? p.lse[r * p.L + i] - 14.f : INFINITY;
      dreg = i < p.L ? a.g.dd[r * up + i] * pg * pv : 0.f;
    }
  };
  if (ntiles > 0) load_tile(0);
  float first_bias = 0.f, last_bias = 0.f;
  for (int t = 0; t < ntiles; ++t) {
    const int h = hk * p.G + t / per, i0 = (t0 + t % per) * TQ;
    __syncthreads();
    st.store(sm);
    if (threadIdx.x < TQ) { rl[threadIdx.x] = lreg; rd[threadIdx.x] = dreg; }
    if (t % per == 0) {
      fill_bias(lut, p, h);
      first_bias = p.table[(long long)p.map[0] * p.H + h] * LOG2E;
      last_bias = p.table[(long long)p.map[p.map_n - 1] * p.H + h] * LOG2E;
    }
    __syncthreads();
    if (t + 1 < ntiles) load_tile(t + 1);
    if (k0 >= n || (p.causal && pos0 + i0 + TQ - 1 < k0)) continue;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x16 s = rows_times<DHP>(sm, ST::PLANE, u * 32, kf);
      const f32x16 dp = rows_times<DHP>(sm + 2 * ST::PLANE, ST::PLANE, u * 32, vf);
      float lv[16], dd[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(rl + u * 32 + 8 * g + 4 * hh), y = *reinterpret_cast<const float4*>(rd + u * 32 + 8 * g + 4 * hh);
        lv[4 * g] = x.x; lv[4 * g + 1] = x.y; lv[4 * g + 2] = x.z; lv[4 * g + 3] = x.w;
        dd[4 * g] = y.x; dd[4 * g + 1] = y.y; dd[4 * g + 2] = y.z; dd[4 * g + 3] = y.w;
      }
      const int q0 = pos0 + i0 + u * 32, e0 = k0 - q0 - p.map_lo;  // entry of the first key and the tile's first query; the others: + key - query
      if (e0 + 31 <= 0 || e0 - 31 >= p.map_n - 1) {
        const float c = e0 + 31 <= 0 ? first_bias : last_bias;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, c - lv[r]));
      } else {
        const float* lp = lut + TABLE_PAD + e0 + (lane & 31) - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, lp[-crow(r)] - lv[r]));
      }
      if (p.causal && k0 + 31 > q0) {
        const int d = key - q0 - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (d - crow(r) > 0) s[r] = 0.f;
      }
      float ds[16], top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) { ds[r] = s[r] * fmaf(dp[r], sign, -dd[r]); top = fmaxf(top, fabsf(ds[r])); }
      follow(top, f, dk);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4 pf[2], sf[2];
        const float e[8] = {s[8 * g], s[8 * g + 1], s[8 * g + 2], s[8 * g + 3], s[8 * g + 4], s[8 * g + 5], s[8 * g + 6], s[8 * g + 7]};
        to_levels<2>(e, pf);
        to_levels<2>(ds + 8 * g, sf);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 gt[2] = {col_frag<DHP>(sm + 2 * ST::PLANE, u * 32 + g * 16, d), col_frag<DHP>(sm + 3 * ST::PLANE, u * 32 + g * 16, d)};
          dv[d] = mfma_levels<2>(gt, pf, dv[d]);
          const u32x4 qt[2] = {col_frag<DHP>(sm, u * 32 + g * 16, d), col_frag<DHP>(sm + ST::PLANE, u * 32 + g * 16, d)};
          dk[d] = mfma_levels<2>(qt, sf, dk[d]);
        }
      }
    }
  }
  if (key >= p.S) return;
  const bool out = key >= n || (p.mask && p.mask[(long long)b * p.S + key]);       // nobody sees it: what its column holds is dropped
  const float w1 = inv_g * inv_q, w2 = inv_v * p.scale, fi = 0x1p-14f / f, wv = inv_g * 0x1p-14f;
  const long long at = ((long long)b * p.S + key) * p.Hkv * p.dh + hk * p.dh;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * hh;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { x[e] = out ? 0.f : dk[d][4 * g + e] * fi * w1 * w2; y[e] = out ? 0.f : dv[d][4 * g + e] * wv; }
      if (c < p.dh) {
        *reinterpret_cast<float4*>(p.dk + at + c) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p.dv + at + c) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
}

// dtable[bucket][h] += the distances of that bucket: a block a head, the query blocks' sums in four fixed runs, then bucket by bucket
__global__ __launch_bounds__(1024) void relpos_bwd_table_kernel(RP p, const float* __restrict__ part, int nq) {
  __shared__ float ent[4][MAP_MAX + 2 * DPAD];
  const int h = blockIdx.x, nent = p.map_n + 2 * DPAD, run = threadIdx.x >> 8;
  const long long rows = (long long)p.B * nq, r0 = rows * run / 4, r1 = rows * (run + 1) / 4;
  for (int e = threadIdx.x & 255; e < nent; e += 256) {
    float s = 0.f;
    for (long long r = r0; r < r1; ++r) s += part[((r / nq * p.H + h) * nq + r % nq) * nent + e];
    ent[run][e] = s;
  }
  __syncthreads();
  for (int bucket = threadIdx.x; bucket < p.nb; bucket += 1024) {
    float s = 0.f;
    for (int e = 0; e < nent; ++e)
      if (p.map[p.entry(e - DPAD + p.map_lo)] == bucket) s += (ent[0][e] + ent[1][e]) + (ent[2][e] + ent[3][e]);
    p.dtable[(long long)bucket * p.H + h] += s;
  }
}

template <int DHP>
int launch(const RP& p, const Bwd& a, hipStream_t st) {
  const int nq = (p.L + 127) / 128, nk = (p.S + 127) / 128;
  const long long qb = (long long)p.B * p.H * nq, kb = (long long)p.B * p.Hkv * nk;
  if (qb > 0x7fffffffLL || kb > 0x7fffffffLL) return SMX_EINVAL;
  const int planes = 4 * Stage<DHP, 256>::PLANE, lq = 4 * (p.map_n + 2 * TABLE_PAD + 4 * (p.map_n + 2 * DPAD)), lk = 4 * (128 + p.map_n + 2 * TABLE_PAD);
  SMX_HIP(smx_max_dynamic_lds((const void*)relpos_bwd_q_kernel<DHP>, planes + 4 * (MAP_MAX + 2 * TABLE_PAD + 4 * (MAP_MAX + 2 * DPAD))));
  SMX_HIP(smx_max_dynamic_lds((const void*)relpos_bwd_kv_kernel<DHP>, planes + 4 * (128 + MAP_MAX + 2 * TABLE_PAD)));
  SMX_LAUNCH(relpos_bwd_q_kernel<DHP>, dim3((unsigned)qb), dim3(256), planes + lq, st, p, a);
  SMX_LAUNCH(relpos_bwd_kv_kernel<DHP>, dim3((unsigned)kb), dim3(256), planes + lk, st, p, a);
  SMX_LAUNCH(relpos_bwd_table_kernel, dim3(p.H), dim3(1024), 0, st, p, (const float*)a.part, nq);
  return smx_launch_status();
}

int64_t part_bytes(const RP& p) { return ((int64_t)p.B * p.H * ((p.L + 127) / 128) * (p.map_n + 2 * DPAD) * 4 + 15) / 16 * 16; }

}  // namespace

extern "C" int64_t smx_attention_relpos_bwd_ws_bytes(const smx_relpos_desc* d) {
  RP p;
  if (check(d, p, true) != SMX_OK) return -1;
  return 2 * split_bytes(p.B, p.H, p.L, p.dh) + 2 * split_bytes(p.B, p.Hkv, p.S, p.dh) + part_bytes(p) + (int64_t)p.B * p.H * up64(p.L) * 4;
}

extern "C" int smx_attention_relpos_bwd_f32(const smx_relpos_desc* d, void* stream) {
  RP p;
  int rc = check(d, p, true);
  if (rc != SMX_OK) return rc;
  if (!d->ws || !aligned(d->ws, 16) || d->ws_bytes < smx_attention_relpos_bwd_ws_bytes(d) || p.H > 65535) return SMX_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  Bwd a;
  char* ws = (char*)d->ws;
  ws = split_setup(a.q, ws, (const float*)p.q, p.q_bs, p.ldq, p.B, p.H, p.G, p.L, p.dh, false);
  ws = split_setup(a.g, ws, p.d_o, (long long)p.L * p.H * p.dh, p.H * p.dh, p.B, p.H, p.G, p.L, p.dh, false);
  ws = split_setup(a.k, ws, (const float*)p.k, p.k_bs, p.ldk, p.B, p.Hkv, 1, p.S, p.dh, true);
  ws = split_setup(a.v, ws, (const float*)p.v, p.v_bs, p.ldv, p.B, p.Hkv, 1, p.S, p.dh, true);
  a.v.flip = 1;
  a.part = (float*)ws;
  a.g.o = (const float*)p.o;
  a.g.dd = (float*)(ws + part_bytes(p));
  const Split all[4] = {a.q, a.g, a.k, a.v};
  rc = split_launch(p, all, 4, st);
  if (rc != SMX_OK) return rc;
  switch (dhp(p.dh)) {
    case 32: return launch<32>(p, a, st);
    case 64: return launch<64>(p, a, st);
    default: return launch<128>(p, a, st);
  }
}
