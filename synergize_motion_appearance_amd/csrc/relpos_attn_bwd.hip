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
  float* part;                                                   // [B][H][query blocks * qparts][map_n + 2 DPAD] sums of dS by distance
  float* dqp; float* dkv;                                        // [qparts][B][L][H * dh] dq, [kparts][2][B][S][Hkv * dh] dk and dv, where the other side is split
  int qparts, kparts;
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
// A weight is computed again as 2^(s - lse), whose error is that of s: some 2^-23 |s|.  Where lse is large enough for that to count, s - lse is kept from
// passing 0: a weight above 1 would leave a half, and in the end fp32.  (No number stays none.)
__device__ __forceinline__ bool steep(float lse) { return fabsf(lse) > 0x1p20f && lse < INFINITY; }
__device__ __forceinline__ void at_most(f32x16& s, float top) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = s[r] > top ? top : s[r];
}
constexpr float F0 = 1.2676506002282294e30f;                     // 2^100: before the first dS that is not zero

// stage TK rows of four planes (h1, h2 of two operands) through registers
template <int DHP>
struct Stage {
  static constexpr int NT = 256, TK = STEP<DHP, 2>, RB = ROWB<DHP>, PLANE = TK * RB, CPR = DHP / 8, NCH = TK * CPR / NT;
  u32x4 reg[4][NCH];
  __device__ __forceinline__ void load(const Split& x, const Split& y, long long at) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const unsigned e = (c * NT + threadIdx.x) * 8;
      reg[0][c] = *reinterpret_cast<const u32x4*>(x.hi + at + e); reg[1][c] = *reinterpret_cast<const u32x4*>(x.lo + at + e);
      reg[2][c] = *reinterpret_cast<const u32x4*>(y.hi + at + e); reg[3][c] = *reinterpret_cast<const u32x4*>(y.lo + at + e);
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

// dq and the sums of dS by distance.  A wave: 32 queries as columns, K and V staged 64 or 32 keys at a time; S^T = K Q^T, dP^T = V dO^T, then
// dQ^T += K^T dS^T with dS^T from the registers.  dS by distance: in a tile that lies beyond the map's ends all pairs are of one entry, a
// lane adds its own; elsewhere lane t collects the tile's diagonal key - query = t - 31 through lane permutes, register by register, and adds it to the
// wave's table in LDS -- one lane an entry, tile after tile: a fixed order without atomics.
// Two waves a SIMD: 256 registers hold 32 queries' operands (Q, dO, dq) and a tile's S and dS (64 columns: 11 more go through scratch).  With so few, neither the
// matrix units (busy for 0.38 of the cycles) nor the vector units (0.34) are full: a wave waits for 0.35 of its time, for its tile's loads, LDS and
// barriers, and the causal blocks' lengths leave 1.6 waves a SIMD.  2 x 16 heads (4 kv) of 4096 x 4096 of 64, causal: 367 us, 281 TFLOP/s (0.67 of three
// half-precision products' rate); 4 x 8 heads of 1024 x 1024 of 32: 47 us, 137 TFLOP/s: 512 blocks of 8 tiles are one round of two a CU, 1.4
// waves a SIMD on average, which wait for 0.39 of their time.  One wave a SIMD without spills at 64 columns: 2% slower; three at 32: 20%;
// two waves a block: 30%; 64 queries a wave: 8% at 64 columns, 33% at 32.
template <int DHP>
__global__ __launch_bounds__(256, DHP >= 96 ? 1 : 2) void relpos_bwd_q_kernel(RP p, Bwd a) {
  using ST = Stage<DHP>;
  constexpr int TK = ST::TK, NU = TK / 32, KS = DHP / 16, DT = DHP / 32, NW = 4, NT = 256, QB = 128;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  const int nent = p.map_n + 2 * DPAD;
  float* lut = reinterpret_cast<float*>(sm + 4 * ST::PLANE);
  float* dacc = lut + p.map_n + 2 * TABLE_PAD;                   // [NW][nent]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
  const int nq = (p.L + QB - 1) / QB;
  const Work w = work_of(blockIdx.x, nq * a.qparts, p.B * p.H, p.causal, p.kv_len != nullptr);
  const int part = w.i % a.qparts, qb = nq - 1 - w.i / a.qparts;
  const int h = w.head % p.H, b = w.head / p.H, hk = h / p.G;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const int q0 = qb * QB + wave * 32, qi = q0 + (lane & 31), pos = pos0 + qi;
  const int wlast = pos0 + min(q0 + 31, p.L - 1);
  const int kend = p.causal ? min(n, pos0 + min(qb * QB + QB - 1, p.L - 1) + 1) : n;
  const int all = kend > 0 ? (kend + TK - 1) / TK : 0;
  const int first = (int)((long long)all * part / a.qparts), last = (int)((long long)all * (part + 1) / a.qparts);
  const bool live = qi < p.L;

  fill_bias(lut, p, h);
  for (int t = threadIdx.x; t < NW * nent; t += NT) dacc[t] = 0.f;
  dacc += wave * nent;
  const float first_bias = p.table[(long long)p.map[0] * p.H + h] * LOG2E, last_bias = p.table[(long long)p.map[p.map_n - 1] * p.H + h] * LOG2E;
  const float lse = live ? p.lse[((long long)b * p.H + h) * p.L + qi] : INFINITY;
  const bool sees = lse != INFINITY;                             // the query has a key (what it holds without one does not count)
  const bool is_steep = __ballot(steep(lse)) != 0;
  const float D = live ? a.g.dd[((long long)b * p.H + h) * ((p.L + 63) & ~63) + qi] : 0.f;
  u32x4 qf[KS][2], gf[KS][2];
  const float sq = p.scale * LOG2E * own_rows<DHP>(qf, (const float*)p.q + b * p.q_bs + (long long)qi * p.ldq + h * p.dh, sees, p.dh);
  const float sg = own_rows<DHP>(gf, p.d_o + ((long long)b * p.L + qi) * p.H * p.dh + h * p.dh, sees, p.dh);
  f32x16 dq[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dq[t] = zero16();
  float f = F0, below = 0.f, above = 0.f;
  Unit ku;

  ST st;
  unsigned long long nleft = 0;                                  // the next step's keys that are left, and the 2^-k of its tile
  float nik = 1.f, niv = 1.f;
  const long long tile0 = ((long long)b * p.Hkv + hk) * ((p.S + 63) >> 6);
  auto load_tile = [&](int key0) {
    st.load(a.k, a.v, (tile0 * 64 + key0) * DHP);
    const int key = key0 + lane;
    nleft = __ballot(lane < TK && key < n && !(p.mask && p.mask[(long long)b * p.S + key]));
    nik = a.k.inv[tile0 + (key0 >> 6)]; niv = a.v.inv[tile0 + (key0 >> 6)];
  };
  if (first < last) load_tile(first * TK);
  const unsigned long long ALL = TK == 64 ? ~0ull : 0xffffffffull;
  for (int t = first; t < last; ++t) {
    const int key0 = t * TK;
    __syncthreads();                                             // the tile before has been read
    st.store(sm);
    const unsigned long long left = nleft;
    const int ek = bits_of(nik);
    const float sc = sq * pow2_bits(ek), sp = sg * pow2_bits(bits_of(niv));
    __syncthreads();
    if (t + 1 < last) load_tile(key0 + TK);
    if (!left || q0 >= p.L || (p.causal && key0 > wlast)) continue;
    const float wk = exp2i(ku.enter(ek, dq));
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x16 s = rows_times<DHP>(sm, ST::PLANE, u * 32, qf);
      const f32x16 dp = rows_times<DHP>(sm + 2 * ST::PLANE, ST::PLANE, u * 32, gf);
      const int e0 = key0 + u * 32 - (pos0 + q0) - p.map_lo;     // entry of the tile's first key and first query; the others: + key - query
      const bool lo = e0 + 31 <= 0, hi = e0 - 31 >= p.map_n - 1;
      if (lo || hi) {
        const float c = (lo ? first_bias : last_bias) - lse;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc, c);
      } else {
        const float* lp = lut + TABLE_PAD + e0 - (lane & 31) + 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc, lp[crow(r)]) - lse;
      }
      if (is_steep) at_most(s, 0.f);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
      if (left != ALL) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = row_bit(left, u * 32 + crow(r)) ? s[r] : 0.f;
      }
      if (p.causal && key0 + u * 32 + 31 > pos0 + q0) {
        const int d = pos - (key0 + u * 32 + 4 * hh);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (d < crow(r)) s[r] = 0.f;
      }
      float ds[16], top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) { ds[r] = s[r] * fmaf(dp[r], r & 1 ? -sp : sp, -D); top = fmaxf(top, fabsf(ds[r])); }
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
      const float fk = f * wk;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4 pf[2];
        to_levels(ds + 8 * g, fk, pf);
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
  float* sums = a.part + ((((long long)b * p.H + h) * nq + qb) * a.qparts + part) * nent;
  for (int t = threadIdx.x; t < nent; t += NT) {
    float x = dacc[t];
#pragma unroll
    for (int y = 1; y < NW; ++y) x += dacc[y * nent + t];
    sums[t] = x;
  }
  if (!live) return;
  const float wq = ku.inv() * p.scale, fi = 1.f / f;
  float* DQ = (a.qparts > 1 ? a.dqp + (long long)part * p.B * p.L * p.H * p.dh : p.dq) + ((long long)b * p.L + qi) * p.H * p.dh + h * p.dh;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * hh;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dq[d][4 * g + e] * fi * wq;
      if (c < p.dh) *reinterpret_cast<float4*>(DQ + c) = make_float4(x[0], x[1], x[2], x[3]);
    }
}

// dk and dv.  A wave: 32 keys as columns; Q and dO of the heads that share them staged 64 or 32 queries at a time; S = Q K^T, dP = dO V^T, dV^T += dO^T P,
// dK^T += Q^T dS.  P carries 2^14, so that what is left of a weight is off by at most 2^-39.  The sizes above: 535 us, 257 TFLOP/s; 42 us, 206 TFLOP/s.  64 columns keep
// 33 registers in scratch (384 MB read, 129 written at the first size, 67 of them the parts' dk and dv) and wait for 0.57 of their time; matrix units 0.34, vector units 0.26.  65 columns and more
// run one wave a SIMD: 2 x 8 heads of 2048 x 2048 with the forward, 80 columns 470 us, 128 647.  Few key blocks: a part of their queries (tiles of all the
// heads) a block, joined by relpos_bwd_rest_kernel.
template <int DHP>
__global__ __launch_bounds__(256, DHP >= 96 ? 1 : 2) void relpos_bwd_kv_kernel(RP p, Bwd a) {
  using ST = Stage<DHP>;
  constexpr int TQ = ST::TK, NU = TQ / 32, KS = DHP / 16, DT = DHP / 32, KB = 128;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  float* rl = reinterpret_cast<float*>(sm + 4 * ST::PLANE);      // the tile's lse
  float* rd = rl + 64;                                           // and D
  int* flag = reinterpret_cast<int*>(rd + 64);                   // whether one of the tile's lse is steep
  float* lut = rd + 64 + 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
  const int nk = (p.S + KB - 1) / KB, qt = (p.L + 63) >> 6;
  const Work w = work_of(blockIdx.x, nk * a.kparts, p.B * p.Hkv, p.causal, p.kv_len != nullptr);
  const int part = w.i % a.kparts, kb = w.i / a.kparts;
  const int hk = w.head % p.Hkv, b = w.head / p.Hkv;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const int k0 = kb * KB + wave * 32, key = k0 + (lane & 31);
  const bool in = key < n && !(p.mask && p.mask[(long long)b * p.S + key]);
  u32x4 kf[KS][2], vf[KS][2];
  const float sk = p.scale * LOG2E * own_rows<DHP>(kf, (const float*)p.k + b * p.k_bs + (long long)key * p.ldk + hk * p.dh, in, p.dh);
  const float sv = own_rows<DHP>(vf, (const float*)p.v + b * p.v_bs + (long long)key * p.ldv + hk * p.dh, in, p.dh);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = zero16();
  float f = F0;
  Unit qu, gu;
  const float w1 = one();
  // causal: the first query that stands at this block's first key or behind it
  const int t0 = p.causal ? max(0, kb * KB - pos0) / TQ : 0, t1 = kb * KB < n ? (p.L + TQ - 1) / TQ : 0;
  const int per = max(0, t1 - t0);
  const long long all = (long long)per * p.G;
  const int first = (int)(all * part / a.kparts), last = (int)(all * (part + 1) / a.kparts);
  ST st;
  float lreg = 0.f, dreg = 0.f, niq = 1.f, nig = 1.f;            // the next tile's lse and D; its 2^-k
  auto load_tile = [&](int t) {
    const int i0 = (t0 + t % per) * TQ, i = i0 + threadIdx.x;
    const long long r = (long long)b * p.H + hk * p.G + t / per;
    st.load(a.q, a.g, (r * qt * 64 + i0) * DHP);
    if (threadIdx.x < TQ) {
      lreg = i < p.L ? p.lse[r * p.L + i] : INFINITY;
      dreg = i < p.L ? a.g.dd[r * qt * 64 + i] : 0.f;
    }
    niq = a.q.inv[r * qt + (i0 >> 6)]; nig = a.g.inv[r * qt + (i0 >> 6)];
  };
  if (first < last) load_tile(first);
  float first_bias = 0.f, last_bias = 0.f;
  for (int t = first; t < last; ++t) {
    const int h = hk * p.G + t / per, i0 = (t0 + t % per) * TQ;
    __syncthreads();
    st.store(sm);
    if (threadIdx.x < TQ) { rl[threadIdx.x] = lreg; rd[threadIdx.x] = dreg; }
    if (threadIdx.x < 64) *flag = __ballot(lane < TQ && steep(lreg)) != 0;
    if (t == first || t % per == 0) {
      fill_bias(lut, p, h);
      first_bias = p.table[(long long)p.map[0] * p.H + h] * LOG2E;
      last_bias = p.table[(long long)p.map[p.map_n - 1] * p.H + h] * LOG2E;
    }
    __syncthreads();
    const bool is_steep = __builtin_amdgcn_readfirstlane(*flag) != 0;
    const int eq = bits_of(niq), eg = bits_of(nig);
    const float sc = sk * pow2_bits(eq), sp = sv * pow2_bits(eg);
    if (t + 1 < last) load_tile(t + 1);
    if (k0 >= n || (p.causal && pos0 + i0 + TQ - 1 < k0)) continue;
    const int lp = 14 + gu.enter(eg, dv), lg = max(lp, 0);    // P carries 2^lg, in dv 2^lp: 2^-lp of a far smaller tile, times f, would leave fp32
    const float ig = exp2i(-lg), wq = exp2i(qu.enter(eq, dk)) * ig;
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
        const float c = (e0 + 31 <= 0 ? first_bias : last_bias) + lg;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc, c - lv[r]);
      } else {
        const float* bias = lut + TABLE_PAD + e0 + (lane & 31) - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc, bias[-crow(r)] - (lv[r] - lg));
      }
      if (is_steep) at_most(s, (float)lg);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
      if (p.causal && k0 + 31 > q0) {
        const int d = key - q0 - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (d > crow(r)) s[r] = 0.f;
      }
      float ds[16], top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) { ds[r] = s[r] * fmaf(dp[r], sp, -dd[r]); top = fmaxf(top, fabsf(ds[r])); }
      follow(top * ig, f, dk);
      const float fq = f * wq;
      if (lp < 0) {
        const float w = exp2i(lp);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= w;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4 pf[2], sf[2];
        const float e[8] = {s[8 * g], s[8 * g + 1], s[8 * g + 2], s[8 * g + 3], s[8 * g + 4], s[8 * g + 5], s[8 * g + 6], s[8 * g + 7]};
        to_halves(e, w1, pf);
        to_levels(ds + 8 * g, fq, sf);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 gt[2] = {col_frag<DHP>(sm + 2 * ST::PLANE, u * 32 + g * 16, d), col_frag<DHP>(sm + 3 * ST::PLANE, u * 32 + g * 16, d)};
          dv[d] = mfma_levels<2>(gt, pf, dv[d]);
          const u32x4 qt2[2] = {col_frag<DHP>(sm, u * 32 + g * 16, d), col_frag<DHP>(sm + ST::PLANE, u * 32 + g * 16, d)};
          dk[d] = mfma_levels<2>(qt2, sf, dk[d]);
        }
      }
    }
  }
  if (key >= p.S) return;
  const float wk = qu.inv() * p.scale, fi = 1.f / f, wv = gu.inv() * 0x1p-14f;
  const long long at = ((long long)b * p.S + key) * p.Hkv * p.dh + hk * p.dh, size = (long long)p.B * p.S * p.Hkv * p.dh;
  float* DK = a.kparts > 1 ? a.dkv + part * 2 * size : p.dk;
  float* DV = a.kparts > 1 ? a.dkv + (part * 2 + 1) * size : p.dv;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * hh;
      float x[4], y[4];                                          // a key that nobody sees: what its column holds is dropped
#pragma unroll
      for (int e = 0; e < 4; ++e) { x[e] = in ? dk[d][4 * g + e] * fi * wk : 0.f; y[e] = in ? dv[d][4 * g + e] * wv : 0.f; }
      if (c < p.dh) {
        *reinterpret_cast<float4*>(DK + at + c) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(DV + at + c) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
}

// What is left once the two passes are done, one launch: the first H blocks dtable, if it is wanted, the others gradients from their parts, in order (dq, dk, dv).
// dtable[bucket][h] += the distances of that bucket: the query blocks' sums in four fixed runs, then a wave a bucket.  Bound by its dependent loads on H blocks: 14 us after 4 x 8
// heads of 1024 x 1024.
struct Sum { const float* src; float* dst; long long size, step; int nparts, end; };      // end: running sum of blocks
struct Rest { Sum s[3]; const float* part; int rows, tables; };                          // rows: query blocks (and their parts) of a head and sample; tables: H or 0
__global__ __launch_bounds__(1024) void relpos_bwd_rest_kernel(RP p, Rest a) {
  __shared__ float ent[4][MAP_MAX + 2 * DPAD];
  __shared__ unsigned short of[MAP_MAX + 2 * DPAD];
  if ((int)blockIdx.x >= a.tables) {
    int id = blockIdx.x - a.tables, t = 0;
    while (id >= a.s[t].end) ++t;
    const Sum& s = a.s[t];
    const long long i = ((id - (t ? a.s[t - 1].end : 0)) * 1024LL + threadIdx.x) * 4;
    if (i >= s.size) return;
    float4 x = *reinterpret_cast<const float4*>(s.src + i);
#pragma unroll 4
    for (int n = 1; n < s.nparts; ++n) {
      const float4 y = *reinterpret_cast<const float4*>(s.src + n * s.step + i);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    *reinterpret_cast<float4*>(s.dst + i) = x;
    return;
  }
  const int h = blockIdx.x, nent = p.map_n + 2 * DPAD, run = threadIdx.x >> 8, lane = threadIdx.x & 63;
  const int rows = p.B * a.rows, r0 = (int)((long long)rows * run / 4), r1 = (int)((long long)rows * (run + 1) / 4);
  for (int e = threadIdx.x; e < nent; e += 1024) of[e] = (unsigned short)p.map[p.entry(e - DPAD + p.map_lo)];
  for (int e = threadIdx.x & 255; e < nent; e += 256) {
    float s = 0.f;
#pragma unroll 8
    for (int r = r0; r < r1; ++r) s += a.part[(((long long)(r / a.rows) * p.H + h) * a.rows + r % a.rows) * nent + e];
    ent[run][e] = s;
  }
  __syncthreads();
  for (int bucket = threadIdx.x >> 6; bucket < p.nb; bucket += 16) {
    float s = 0.f;
    for (int e = lane; e < nent; e += 64)
      if (of[e] == bucket) s += (ent[0][e] + ent[1][e]) + (ent[2][e] + ent[3][e]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) p.dtable[(long long)bucket * p.H + h] += s;
  }
}

// Parts: 256 CUs hold two blocks each at a time, and a wave alone on its SIMD waits through its own latencies, so fewer blocks than two a CU walk parts of
// the other side (none shorter than four tiles; their gradients are written and read once more).  With a causal rule blocks differ in length -- a first key meets all
// queries, a last one itself -- and four a CU are wanted.  In parts / not, forward and backward: 8 heads of 1024 x 1024 of 64, causal 110 / 196 us; 4 x 8 of 1024 x 1024 of 32
// 141 / 153; 2 x 8 of 2048 x 2048 of 64, causal 268 / 370.
struct Plan { int qparts, kparts; long long qblocks, kblocks; int64_t part, dd, dqp, dkv, total; };

int parts(long long base, long long tiles, bool causal) {
  const long long want = causal ? 1024 : 512;
  long long n = base >= want ? 1 : (want + base - 1) / base;
  if (n > tiles / 4) n = tiles / 4;
  return n < 1 ? 1 : n > 8 ? 8 : (int)n;
}

Plan plan(const RP& p) {
  Plan w;
  const long long nq = (p.L + 127) / 128, nk = (p.S + 127) / 128;
  w.qparts = parts(p.B * p.H * nq, (p.S + 63) / 64, p.causal);
  w.kparts = parts(p.B * p.Hkv * nk, (long long)p.G * ((p.L + 63) / 64), p.causal);
  w.qblocks = p.B * p.H * nq * w.qparts;
  w.kblocks = p.B * p.Hkv * nk * w.kparts;
  w.part = ((int64_t)w.qblocks * (p.map_n + 2 * DPAD) * 4 + 15) / 16 * 16;
  w.dd = (int64_t)p.B * p.H * up64(p.L) * 4;
  w.dqp = w.qparts > 1 ? (int64_t)w.qparts * p.B * p.L * p.H * p.dh * 4 : 0;
  w.dkv = w.kparts > 1 ? (int64_t)w.kparts * 2 * p.B * p.S * p.Hkv * p.dh * 4 : 0;
  w.total = 2 * split_bytes(p.B, p.H, p.L, p.dh) + 2 * split_bytes(p.B, p.Hkv, p.S, p.dh) + w.part + w.dd + w.dqp + w.dkv;
  return w;
}

template <int DHP>
int launch(const RP& p, const Bwd& a, const Plan& w, hipStream_t st) {
  const int planes = 4 * Stage<DHP>::PLANE, lq = 4 * (p.map_n + 2 * TABLE_PAD + 4 * (p.map_n + 2 * DPAD)), lk = 4 * (132 + p.map_n + 2 * TABLE_PAD);
  SMX_HIP(smx_max_dynamic_lds((const void*)relpos_bwd_q_kernel<DHP>, planes + 4 * (MAP_MAX + 2 * TABLE_PAD + 4 * (MAP_MAX + 2 * DPAD))));
  SMX_HIP(smx_max_dynamic_lds((const void*)relpos_bwd_kv_kernel<DHP>, planes + 4 * (132 + MAP_MAX + 2 * TABLE_PAD)));
  if (p.dq) SMX_LAUNCH(relpos_bwd_q_kernel<DHP>, dim3((unsigned)w.qblocks), dim3(256), planes + lq, st, p, a);
  if (p.dk) SMX_LAUNCH(relpos_bwd_kv_kernel<DHP>, dim3((unsigned)w.kblocks), dim3(256), planes + lk, st, p, a);
  return smx_launch_status();
}

}  // namespace

extern "C" int64_t smx_attention_relpos_bwd_ws_bytes(const smx_relpos_desc* d) {
  RP p;
  return check(d, p, true) == SMX_OK ? plan(p).total : -1;
}

extern "C" int smx_attention_relpos_bwd_f32(const smx_relpos_desc* d, void* stream) {
  RP p;
  int rc = check(d, p, true);
  if (rc != SMX_OK) return rc;
  const Plan w = plan(p);
  const long long sq = (long long)p.B * p.L * p.H * p.dh, sk = (long long)p.B * p.S * p.Hkv * p.dh;
  if (!d->ws || !aligned(d->ws, 16) || d->ws_bytes < w.total || w.qblocks > 0x7fffffffLL || w.kblocks > 0x7fffffffLL ||
      (sq + 2 * sk) / 4096 > 0x7ff00000LL - p.H) return SMX_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  Bwd a;
  char* ws = (char*)d->ws;
  ws = split_setup(a.q, ws, (const float*)p.q, p.q_bs, p.ldq, p.B, p.H, p.L, p.dh, false);
  ws = split_setup(a.g, ws, p.d_o, (long long)p.L * p.H * p.dh, p.H * p.dh, p.B, p.H, p.L, p.dh, false);
  ws = split_setup(a.k, ws, (const float*)p.k, p.k_bs, p.ldk, p.B, p.Hkv, p.S, p.dh, true);
  ws = split_setup(a.v, ws, (const float*)p.v, p.v_bs, p.ldv, p.B, p.Hkv, p.S, p.dh, true);
  a.v.flip = 1;
  a.part = (float*)ws;
  a.g.o = (const float*)p.o;
  a.g.dd = (float*)(ws + w.part);
  a.dqp = (float*)(ws + w.part + w.dd);
  a.dkv = (float*)(ws + w.part + w.dd + w.dqp);
  a.qparts = w.qparts; a.kparts = w.kparts;
  Split all[4] = {a.g};                                          // (D of its rows: both passes)
  int n = 1;
  if (p.dk) all[n++] = a.q;
  if (p.dq) { all[n++] = a.k; all[n++] = a.v; }
  rc = split_launch(p, all, n, st);
  if (rc != SMX_OK) return rc;
  switch (dhp(p.dh)) {
    case 32: rc = launch<32>(p, a, w, st); break;
    case 64: rc = launch<64>(p, a, w, st); break;
    case 96: rc = launch<96>(p, a, w, st); break;
    default: rc = launch<128>(p, a, w, st);
  }
  if (rc != SMX_OK) return rc;
  Rest u = {{{a.dqp, p.dq, p.dq && w.qparts > 1 ? sq : 0, sq, w.qparts, 0}, {a.dkv, p.dk, p.dk && w.kparts > 1 ? sk : 0, 2 * sk, w.kparts, 0},
             {a.dkv + sk, p.dv, p.dk && w.kparts > 1 ? sk : 0, 2 * sk, w.kparts, 0}}, a.part, (p.L + 127) / 128 * w.qparts, p.dtable ? p.H : 0};
  long long blocks = 0;
  for (Sum& x : u.s) { blocks += (x.size + 4095) / 4096; x.end = (int)blocks; }
  blocks += u.tables;
  if (blocks > 0x7fffffffLL) return SMX_EINVAL;
  if (!blocks) return rc;
  SMX_LAUNCH(relpos_bwd_rest_kernel, dim3((unsigned)blocks), dim3(1024), 0, st, p, u);
  return smx_launch_status();
}
