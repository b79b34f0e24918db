// Attention with a learned relative position bias by buckets, forward (include/smx.h: smx_attention_relpos):
//   s_ij = scale q_i . k_j + table[map[clamp(j - pos_i - map_lo)]][h],  P = softmax over the keys that are left,  o_i = sum_j P_ij v_j
// One pass over the keys with the running maximum and sum of the softmax, scores in log2 units.  Two kernels and what they need:
//   relpos_tile_kernel   queries in tiles of 32 a wave on the matrix cores (bf16 storage: bf16 products, weights in two parts; fp32 storage: f16x3, relpos.h)
//   relpos_token_kernel  a few queries per sample (decoding): bound by reading the cache, plain fp32 products on the vector units
//   relpos_join_kernel   joins the parts where the keys were split over blocks
//   relpos_split_kernel  the staged fp32 operands as two halves each
#include "relpos.h"

namespace relpos {

// ---- fp32 operands as halves (relpos.h: Split) ---------------------------------------------------------------------------------
struct Splits { Split s[4]; int end[4]; };                       // end: running sum of blocks

// 64 rows of one head -> both planes and their 2^-k; gradient rows: D_i = dO_i . o_i too.  Bound by memory: 2 x 38 x 1024 rows of 8 x 32, 159 MB with the planes,
// 26 us, 6.2 TB/s (much of it in the 256 MB of cache that all XCDs share).
template <int DHP>
__global__ __launch_bounds__(256) void relpos_split_kernel(RP p, Splits a) {
  __shared__ float red[4];
  int t = 0, id = blockIdx.x;
  while (id >= a.end[t]) ++t;
  const Split& s = a.s[t];
  id -= t ? a.end[t - 1] : 0;
  const int nt = (s.rows + 63) / 64, c = id % nt, h = id / nt % s.heads, b = id / nt / s.heads;
  const int n = s.kv ? min(p.keys(b), s.rows) : s.rows;
  constexpr int NI = DHP / 16;                                   // four threads a row, NI float4 each
  const int r = threadIdx.x >> 2, q = threadIdx.x & 3, row = c * 64 + r;
  const bool in = row < n && !(s.kv ? p.mask && p.mask[(long long)b * p.S + row] : p.empty(b, h, row));
  const long long at = b * s.bs + (long long)row * s.ld + h * p.dh, tile = ((long long)b * s.heads + h) * nt + c;
  float4 x[NI];
  float m = 0.f, D = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int d = (i * 4 + q) * 4;
    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in && d < p.dh) {
      x[i] = *reinterpret_cast<const float4*>(s.src + at + d);
      if (s.dd) { const float4 y = *reinterpret_cast<const float4*>(s.o + at + d); D += (x[i].x * y.x + x[i].y * y.y) + (x[i].z * y.z + x[i].w * y.w); }
    }
    m = fmaxf(m, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
  }
  if (s.dd) {
    D += __shfl_xor(D, 1, 64);
    D += __shfl_xor(D, 2, 64);
    if (q == 0) s.dd[tile * 64 + r] = D;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  float inv;
  float sc = pow2_of(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), inv);
  if (threadIdx.x == 0) s.inv[tile] = inv;
  if (s.flip && (r & 1)) sc = -sc;
  const long long out = (tile * 64 + r) * DHP;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const float4 y = make_float4(x[i].x * sc, x[i].y * sc, x[i].z * sc, x[i].w * sc);
    const uint2 h2 = make_uint2(cvt2_f16(y.x, y.y), cvt2_f16(y.z, y.w));
    const uint2 l2 = make_uint2(cvt2_f16(y.x - f16lo(h2.x), y.y - f16hi(h2.x)), cvt2_f16(y.z - f16lo(h2.y), y.w - f16hi(h2.y)));
    *reinterpret_cast<uint2*>(s.hi + out + (i * 4 + q) * 4) = h2;
    *reinterpret_cast<uint2*>(s.lo + out + (i * 4 + q) * 4) = l2;
  }
}

int64_t split_bytes(int B, int heads, int rows, int dh) {
  return (int64_t)B * heads * ((int64_t)up64(rows) * dhp(dh) * 4 + (up64(rows) / 64 + 3) / 4 * 16);
}

char* split_setup(Split& s, char* ws, const float* src, long long bs, int ld, int B, int heads, int rows, int dh, bool kv) {
  const int64_t plane = (int64_t)B * heads * up64(rows) * dhp(dh);
  s.src = src; s.bs = bs; s.ld = ld; s.heads = heads; s.rows = rows; s.kv = kv; s.flip = 0;
  s.hi = (_Float16*)ws; s.lo = s.hi + plane; s.inv = (float*)(s.lo + plane);
  s.o = nullptr; s.dd = nullptr;
  return ws + split_bytes(B, heads, rows, dh);
}

int split_launch(const RP& p, const Split* s, int n, hipStream_t st) {
  Splits a;
  long long nb = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < n) { a.s[i] = s[i]; nb += (long long)p.B * s[i].heads * (up64(s[i].rows) / 64); }
    if (nb > 0x7fffffffLL) return SMX_EINVAL;
    a.end[i] = (int)nb;
  }
  const dim3 grid((unsigned)nb), block(256);
  switch (dhp(p.dh)) {
    case 32: SMX_LAUNCH(relpos_split_kernel<32>, grid, block, 0, st, p, a); break;
    case 64: SMX_LAUNCH(relpos_split_kernel<64>, grid, block, 0, st, p, a); break;
    case 96: SMX_LAUNCH(relpos_split_kernel<96>, grid, block, 0, st, p, a); break;
    default: SMX_LAUNCH(relpos_split_kernel<128>, grid, block, 0, st, p, a);
  }
  return smx_launch_status();
}

int check(const smx_relpos_desc* d, RP& p, bool bwd) {
  if (!d || !d->q || !d->k || !d->v || !d->o || !d->table || !d->map) return SMX_EINVAL;
  if (d->B <= 0 || d->H <= 0 || d->Hkv <= 0 || d->H % d->Hkv || d->L <= 0 || d->S <= 0 || d->dh <= 0 || d->dh % 4 || d->dh > 128) return SMX_EINVAL;
  if ((long long)d->H * d->dh > (1 << 20) || (long long)d->B * d->H > (1 << 24) || d->L > (1 << 29) || d->S > (1 << 29)) return SMX_EINVAL;
  if (d->map_n <= 0 || d->map_n > MAP_MAX || d->map_lo > 0 || d->map_lo + d->map_n <= 0 || d->num_buckets <= 0 || d->num_buckets > 4096) return SMX_EINVAL;
  if (d->has_q_start && (d->q_start > (1 << 30) || d->q_start < -(1 << 30))) return SMX_EINVAL;
  if (!(d->scale == d->scale) || (d->bf16 != 0 && d->bf16 != 1) || (bwd && d->bf16)) return SMX_EINVAL;
  if (d->ldq < d->H * d->dh || d->ldk < d->Hkv * d->dh || d->ldv < d->Hkv * d->dh || d->ldo < d->H * d->dh) return SMX_EINVAL;
  if (d->ldq > (1 << 24) || d->ldk > (1 << 24) || d->ldv > (1 << 24) || d->ldo > (1 << 24)) return SMX_EINVAL;
  if ((d->ldq | d->ldk | d->ldv | d->ldo) % 4 || d->q_bs < 0 || d->k_bs < 0 || d->v_bs < 0 || d->o_bs < 0) return SMX_EINVAL;
  if (d->q_bs % 4 || d->k_bs % 4 || d->v_bs % 4 || d->o_bs % 4) return SMX_EINVAL;
  const int el = 4 * (d->bf16 ? 2 : 4);
  if (!aligned(d->q, el) || !aligned(d->k, el) || !aligned(d->v, el) || !aligned(d->o, el)) return SMX_EINVAL;
  if (bwd && (!d->d_o || !d->dq != !d->dtable || !d->dk != !d->dv || (!d->dq && !d->dk) || !d->lse || d->ldo != d->H * d->dh || d->o_bs != (int64_t)d->L * d->ldo)) return SMX_EINVAL;
  if (bwd && (!aligned(d->d_o, 16) || !aligned(d->dq, 16) || !aligned(d->dk, 16) || !aligned(d->dv, 16))) return SMX_EINVAL;
  p.q = d->q; p.k = d->k; p.v = d->v; p.o = d->o; p.table = d->table; p.map = d->map; p.mask = d->mask; p.kv_len = d->kv_len;
  p.lse = d->lse; p.d_o = d->d_o; p.dq = d->dq; p.dk = d->dk; p.dv = d->dv; p.dtable = d->dtable;
  p.q_bs = d->q_bs; p.k_bs = d->k_bs; p.v_bs = d->v_bs; p.o_bs = d->o_bs; p.ldq = d->ldq; p.ldk = d->ldk; p.ldv = d->ldv; p.ldo = d->ldo;
  p.B = d->B; p.H = d->H; p.Hkv = d->Hkv; p.G = d->H / d->Hkv; p.L = d->L; p.S = d->S; p.dh = d->dh;
  p.map_lo = d->map_lo; p.map_n = d->map_n; p.nb = d->num_buckets; p.causal = d->causal; p.has_start = d->has_q_start; p.q_start = d->q_start;
  p.scale = d->scale;
  return SMX_OK;
}

}  // namespace relpos

namespace {
using namespace relpos;

// ---- queries in tiles ----------------------------------------------------------------------------------------------------------
// two stages of keys in turn, one barrier a step; one where two would leave a CU with one block (fp32 storage, 65 to 96 columns: 106 KB).  8 x 16 heads of 1024 x 1024,
// one / two: fp32 32 columns 98 / 98 us, 64 148 / 148, 96 211 / 243, 128 (in steps of 32 keys) 279 / 279; bf16 64 columns (weights in one part) 62.6 / 61.8
template <int DHP, int NL> constexpr int BUFFERS = NL == 2 && DHP == 96 ? 1 : 2;

// where the operands come from: bf16 storage reads q / k / v themselves, fp32 storage q and the planes of k and v; parts: m, l [row][part], o
// [row][part][dh] when the keys are split
struct Src {
  Split k, v;
  int nparts, per;                    // parts of the keys, keys of a part (a multiple of 64)
  float* part_ml; float* part_o;
};

// A wave owns 32 queries as the columns of swapped products: S^T = K Q^T (a lane: one query, 16 of 32 keys), O^T += V^T P^T with P taken from the score
// registers as they are -- the transposing LDS reads fetch V's columns in the order of an accumulator's rows.  The statistics are lane-local but for one
// exchange between the two half waves.  The block's waves share the staged keys, the next tile's loads are in flight during the products.
// Weights are 2^(s - mo), mo finite and followed only when a row outgrows it by 2^8 (and at its first key): the scores leave the products through one fma,
// and P stays below 2^8 (fp32 storage: 2^14, below the largest half; its second half is then off by at most 2^-31 of the row's largest weight).
// The bias of a tile that lies beyond the map's ends is one number; other tiles read it per score from LDS.
// Bound by the vector units' work on the scores (bias, maximum, 2^x, sum, two parts: some 10 operations each) next to the matrix products, of which only part runs
// at the same time on 2 or 3 waves a SIMD.  2 x 16 heads (4 kv) of 8192 x 8192 of 64, causal, bf16: 465 us, 591 TFLOP/s; of the SIMDs' cycles the vector units are
// busy for 0.71, the matrix units for 0.40 (358 us with the weights in one bf16 part, the outputs' error then 1.3 times that of their own rounding).
// 38 x 8 heads of 1024 x 1024 of 32, fp32: 206 us with the split, 198 TFLOP/s of the formula's, 0.47 of what three half-precision products at a large matrix
// product's rate would take: vector 0.54, matrix 0.28, a quarter of the waves' time spent waiting, and 2432 blocks on 768 places are 3.2 rounds.
// Three waves a SIMD (bf16 up to 64 columns) against two, 8 x 16 heads of 1024 x 1024: 54.0 / 52.4 us for 32 columns, 75.7 / 76.4 for 64, where the long
// sequence takes 467 / 493.
// 64 queries a wave instead of 32: 221 us for 205 of that build.
template <int DHP, int NL>
__global__ __launch_bounds__(256, NL == 1 && DHP <= 64 ? 3 : 2) void relpos_tile_kernel(RP p, Src a) {
  constexpr int TK = STEP<DHP, NL>, NU = TK / 32, KS = DHP / 16, DT = DHP / 32, RB = ROWB<DHP>, NT = 256;
  constexpr int PLANE = TK * RB, STAGE = 2 * NL * PLANE;         // K levels, V levels
  constexpr int NBUF = BUFFERS<DHP, NL>;
  constexpr int CPR = DHP / 8, NCH = TK * CPR / NT;              // 16-byte chunks of a row; of a plane, a thread
  constexpr float PSH = NL == 2 ? 6.f : 0.f;
  extern __shared__ __attribute__((aligned(16))) char sm[];      // stages, bias
  float* lut = reinterpret_cast<float*>(sm + NBUF * STAGE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hh = lane >> 5;
  constexpr int QB = 128;
  const int nq = (p.L + QB - 1) / QB;
  const Work w = work_of(blockIdx.x, nq * a.nparts, p.B * p.H, p.causal, p.kv_len != nullptr);
  const int part = w.i % a.nparts, qb = nq - 1 - w.i / a.nparts;
  const int h = w.head % p.H, b = w.head / p.H, hk = h / p.G;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const int q0 = qb * QB + wave * 32, qi = q0 + (lane & 31), pos = pos0 + qi;
  const int wlast = pos0 + min(q0 + 31, p.L - 1);                // the wave's last position; none if q0 >= L
  int kend = p.causal ? min(n, pos0 + min(qb * QB + QB - 1, p.L - 1) + 1) : n;
  const int kbeg = a.nparts > 1 ? part * a.per : 0;
  if (a.nparts > 1) kend = min(kend, kbeg + a.per);
  const int ntiles = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;

  fill_bias(lut, p, h);
  const float first_bias = p.table[(long long)p.map[0] * p.H + h] * LOG2E, last_bias = p.table[(long long)p.map[p.map_n - 1] * p.H + h] * LOG2E;
  float sq = p.scale * LOG2E;
  u32x4 qf[KS][NL];
  if constexpr (NL == 2) {
    sq *= own_rows<DHP>(qf, (const float*)p.q + b * p.q_bs + (long long)qi * p.ldq + h * p.dh, qi < p.L, p.dh);
  } else {
    const bf16_t* Q = (const bf16_t*)p.q + b * p.q_bs + (long long)qi * p.ldq + h * p.dh;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const int d = kk * 16 + hh * 8;
      uint2 x = make_uint2(0, 0), y = make_uint2(0, 0);
      if (qi < p.L && d < p.dh) x = *reinterpret_cast<const uint2*>(Q + d);
      if (qi < p.L && d + 4 < p.dh) y = *reinterpret_cast<const uint2*>(Q + d + 4);
      qf[kk][0] = u32x4{x.x, x.y, y.x, y.y};
    }
  }

  u32x4 kreg[NL][NCH], vreg[NL][NCH];
  unsigned long long nleft = 0;                                  // the next step's keys that are left, and the 2^-k of its tile
  float nik = 1.f, niv = 1.f;
  const int tiles = (p.S + 63) >> 6;
  const long long tile0 = ((long long)b * p.Hkv + hk) * tiles;
  // a step's rows: a wave-uniform start and 32-bit places behind it (bf16: rows of at most 2^24 elements)
  unsigned ko[NCH], vo[NCH];
  bool cin[NCH];
  if constexpr (NL == 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const unsigned e = c * NT + threadIdx.x, d = e % CPR * 8;
      ko[c] = (e / CPR * p.ldk + d) * 2; vo[c] = (e / CPR * p.ldv + d) * 2;
      cin[c] = (int)d < p.dh;
    }
  }
  auto load_tile = [&](int key0) {
    if constexpr (NL == 2) {
      const long long at = (tile0 * 64 + key0) * DHP;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const unsigned e = (c * NT + threadIdx.x) * 8;
        kreg[0][c] = *reinterpret_cast<const u32x4*>(a.k.hi + at + e); kreg[1][c] = *reinterpret_cast<const u32x4*>(a.k.lo + at + e);
        vreg[0][c] = *reinterpret_cast<const u32x4*>(a.v.hi + at + e); vreg[1][c] = *reinterpret_cast<const u32x4*>(a.v.lo + at + e);
      }
    } else {
      const char* K = reinterpret_cast<const char*>((const bf16_t*)p.k + b * p.k_bs + (long long)key0 * p.ldk + hk * p.dh);
      const char* V = reinterpret_cast<const char*>((const bf16_t*)p.v + b * p.v_bs + (long long)key0 * p.ldv + hk * p.dh);
      if (key0 + TK <= n && !p.mask && p.dh % 8 == 0) {          // the usual step: nothing to look at
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          kreg[0][c] = vreg[0][c] = u32x4{0, 0, 0, 0};
          if (cin[c]) { kreg[0][c] = *reinterpret_cast<const u32x4a8*>(K + ko[c]); vreg[0][c] = *reinterpret_cast<const u32x4a8*>(V + vo[c]); }
        }
      } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int e = c * NT + threadIdx.x, key = key0 + e / CPR, d = e % CPR * 8;
          uint2 x = make_uint2(0, 0), y = x, z = x, w = x;
          if (key < n && !(p.mask && p.mask[(long long)b * p.S + key])) {      // what a left-out place holds must not meet a zero weight: zeros instead
            if (d < p.dh) { x = *reinterpret_cast<const uint2*>(K + ko[c]); z = *reinterpret_cast<const uint2*>(V + vo[c]); }
            if (d + 4 < p.dh) { y = *reinterpret_cast<const uint2*>(K + ko[c] + 8); w = *reinterpret_cast<const uint2*>(V + vo[c] + 8); }
          }
          kreg[0][c] = u32x4{x.x, x.y, y.x, y.y};
          vreg[0][c] = u32x4{z.x, z.y, w.x, w.y};
        }
      }
    }
    const int key = key0 + lane;
    nleft = __ballot(lane < TK && key < n && !(p.mask && p.mask[(long long)b * p.S + key]));
    if constexpr (NL == 2) { nik = a.k.inv[tile0 + (key0 >> 6)]; niv = a.v.inv[tile0 + (key0 >> 6)]; }
  };
  auto store_tile = [&](int buf) {
    char* st = sm + buf * STAGE;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int e = c * NT + threadIdx.x, off = e / CPR * RB + e % CPR * 16;
#pragma unroll
      for (int l = 0; l < NL; ++l) {
        *reinterpret_cast<u32x4*>(st + l * PLANE + off) = kreg[l][c];
        *reinterpret_cast<u32x4*>(st + (NL + l) * PLANE + off) = vreg[l][c];
      }
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = zero16();
  float mo = 0.f, l = 0.f;
  bool begun = false;                                            // the row has met a key
  Unit vu;
  const float w1 = one();
  const unsigned long long ALL = TK == 64 ? ~0ull : 0xffffffffull;
  if (ntiles > 0) { load_tile(kbeg); store_tile(0); }
  __syncthreads();
  for (int t = 0; t < ntiles; ++t) {
    const int buf = NBUF == 2 ? t & 1 : 0, key0 = kbeg + t * TK;
    const unsigned long long left = nleft;
    const int ek = bits_of(nik), ev = bits_of(niv);
    if (t + 1 < ntiles) load_tile(key0 + TK);
    char* st = sm + buf * STAGE;
    if (left && q0 < p.L && !(p.causal && key0 > wlast)) {
      float sc = sq;
      int lw = 0;
      if constexpr (NL == 2) {
        sc = sq * pow2_bits(ek);
        lw = vu.enter(ev, o);
      }
      f32x16 s[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u) s[u] = zero16();
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          u32x4 kf[NL];
#pragma unroll
          for (int x = 0; x < NL; ++x) kf[x] = row_frag<DHP>(st + x * PLANE, u * 32, kk);
          s[u] = mfma_levels<NL>(kf, qf[kk], s[u]);
        }
      const float kc = (float)lw - mo;
      const int e0 = key0 - (pos0 + q0) - p.map_lo;              // entry of the tile's first key and first query; the others: + key - query
      if (e0 + TK - 1 <= 0 || e0 - 31 >= p.map_n - 1) {
        const float c = (e0 + TK - 1 <= 0 ? first_bias : last_bias) + kc;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], sc, c);
      } else {
        const float* lp = lut + TABLE_PAD + e0 - (lane & 31) + 4 * hh;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], sc, lp[u * 32 + crow(r)]) + kc;
      }
      if (left != ALL) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = row_bit(left, u * 32 + crow(r)) ? s[u][r] : -INFINITY;
      }
      if (p.causal && key0 + TK - 1 > pos0 + q0) {
        const int d = pos - key0 - 4 * hh;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (d < u * 32 + crow(r)) s[u][r] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
      top = other_max(top) - (float)lw;                                 // s - mo of the row's largest score
      const bool first = !begun && top > -INFINITY;
      if (__ballot(first || top > PSH + 8.f)) {
        const float d = first ? top - PSH : top > PSH ? top - PSH : 0.f, al = begun ? __builtin_amdgcn_exp2f(-d) : 0.f;
        begun |= first;
        mo += d; l *= al;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] -= d;
#pragma unroll
        for (int x = 0; x < DT; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[x][r] *= al;
      }
      float lt = 0.f;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) { e[r] = __builtin_amdgcn_exp2f(s[u][r]); lt += e[r]; }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          u32x4 pf[2];
          if constexpr (NL == 2) to_halves(e + 8 * g, w1, pf);
          else to_bf16_parts(e + 8 * g, pf);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            u32x4 vf[NL];
#pragma unroll
            for (int x = 0; x < NL; ++x) vf[x] = col_frag<DHP>(st + (NL + x) * PLANE, u * 32 + g * 16, d);
            if constexpr (NL == 2) o[d] = mfma_levels<2>(vf, pf, o[d]);
            else { o[d] = mfma<1>(vf[0], pf[1], o[d]); o[d] = mfma<1>(vf[0], pf[0], o[d]); }
          }
        }
      }
      l = fmaf(lt, exp2i(-lw), l);
    }
    if (NBUF == 1) __syncthreads();
    if (t + 1 < ntiles) store_tile(NBUF == 2 ? buf ^ 1 : 0);
    __syncthreads();
  }
  if (qi >= p.L) return;
  l = other_sum(l);
  const float inv_v = NL == 2 ? vu.inv() : 1.f;
  const long long row = ((long long)b * p.H + h) * p.L + qi;
  if (a.nparts > 1) {
    float* O = a.part_o + (row * a.nparts + part) * p.dh;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + 8 * g + 4 * hh;
        if (c < p.dh) *reinterpret_cast<float4*>(O + c) = make_float4(o[d][4 * g] * inv_v, o[d][4 * g + 1] * inv_v, o[d][4 * g + 2] * inv_v, o[d][4 * g + 3] * inv_v);
      }
    if (hh == 0) *reinterpret_cast<float2*>(a.part_ml + (row * a.nparts + part) * 2) = make_float2(begun ? mo : -INFINITY, l);
    return;
  }
  const float il = l == 0.f ? 0.f : 1.f / l;                      // (0: no key left; a sum that is no number stays none.  inv_v / l could leave the normal numbers)
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * hh;
      const float4 w = make_float4(o[d][4 * g] * il * inv_v, o[d][4 * g + 1] * il * inv_v, o[d][4 * g + 2] * il * inv_v, o[d][4 * g + 3] * il * inv_v);
      if (c < p.dh) {
        if constexpr (NL == 2) St<float>::st4((float*)p.o + b * p.o_bs + (long long)qi * p.ldo + h * p.dh + c, w);
        else St<bf16_t>::st4((bf16_t*)p.o + b * p.o_bs + (long long)qi * p.ldo + h * p.dh + c, w);
      }
    }
  if (p.lse && hh == 0) p.lse[row] = l == 0.f ? INFINITY : mo + __log2f(l);
}

// ---- a few queries per sample ---------------------------------------------------------------------------------------------------
// A block takes a part of one (sample, kv head)'s keys for RT of its G * L query rows (as many passes over the keys as rows / 4, from the caches but the first).  LPK lanes hold a key's row, EPL values each, and the same columns of the
// RT queries and running outputs; every group of LPK lanes walks keys of its own, four a step, with a running maximum and sum of its own: the only
// exchanges are the LPK-lane sums of the scores.  The groups are joined through LDS at the end, the parts by relpos_join_kernel.  Bound by the keys' and values'
// bytes: 16 ragged samples of up to 32768 keys, 4 kv heads of 64 for 16, bf16, 411 MB: 105 us, 3.9 TB/s; for short caches by the launch and
// the caller's own work (8 samples of 300 keys: 12 us).
template <typename T, int EPL> struct Row;                       // EPL values as they lie in memory
template <> struct Row<float, 4> {
  typedef float Raw __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ void wide(Raw v, float (&f)[4]) { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
};
template <> struct Row<bf16_t, 4> {
  typedef unsigned Raw __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void wide(Raw v, float (&f)[4]) { const float4 x = unpack4(make_uint2(v.x, v.y)); f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; }
};
template <> struct Row<bf16_t, 8> {
  typedef unsigned Raw __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ void wide(Raw v, float (&f)[8]) { unpack8(make_uint4(v.x, v.y, v.z, v.w), f); }
};

template <int CTRL> __device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// sum over the LPK neighbouring lanes, in all of them
template <int LPK> __device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (LPK >= 2) x = dpp_add<0xB1>(x);                  // quad_perm 1 0 3 2
  if constexpr (LPK >= 4) x = dpp_add<0x4E>(x);                  // quad_perm 2 3 0 1
  if constexpr (LPK >= 8) x = dpp_add<0x141>(x);                 // row_half_mirror
  if constexpr (LPK >= 16) x = dpp_add<0x140>(x);                // row_mirror
  if constexpr (LPK >= 32) x += __shfl_xor(x, 16, 64);
  return x;
}

template <typename T, int EPL, int LPK, int RT>
__global__ __launch_bounds__(256) void relpos_token_kernel(RP p, Src a) {
  using R = Row<T, EPL>;
  using Raw = typename R::Raw;
  constexpr int GPB = 256 / LPK, U = 4;                          // groups of a block, keys a step
  extern __shared__ __attribute__((aligned(16))) char sm[];
  float* red = reinterpret_cast<float*>(sm);                     // [4 waves][RT][2 + LPK * EPL]
  const int sub = threadIdx.x % LPK, grp = threadIdx.x / LPK, c0 = sub * EPL;
  const int rows = p.G * p.L, nr = (rows + RT - 1) / RT;
  unsigned id = blockIdx.x;
  const int rc = id % nr; id /= nr;
  const int part = id % a.nparts; id /= a.nparts;
  const int hk = id % p.Hkv, b = id / p.Hkv;
  const int n = p.keys(b), pos0 = p.pos0(n);
  const bool in = c0 < p.dh;
  float q[RT][EPL], o[RT][EPL], m[RT], l[RT], fb[RT], lb[RT];
  int pos[RT], hd[RT];
  int pmax = -0x7fffffff, pmin = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = rc * RT + r, ok = row < rows, rr = ok ? row : 0;
    const int i = rr % p.L;
    hd[r] = hk * p.G + rr / p.L;
    pos[r] = pos0 + i;
    pmax = max(pmax, pos[r]); pmin = min(pmin, pos[r]);
    m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) { q[r][e] = 0.f; o[r][e] = 0.f; }
    if (in) R::wide(*reinterpret_cast<const Raw*>((const T*)p.q + b * p.q_bs + (long long)i * p.ldq + hd[r] * p.dh + c0), q[r]);
#pragma unroll
    for (int e = 0; e < EPL; ++e) q[r][e] *= p.scale * LOG2E;
    fb[r] = p.table[(long long)p.map[0] * p.H + hd[r]] * LOG2E;
    lb[r] = p.table[(long long)p.map[p.map_n - 1] * p.H + hd[r]] * LOG2E;
  }
  const int k0 = part * a.per, k1 = min(min(k0 + a.per, n), p.causal ? pmax + 1 : n);
  const T* K = (const T*)p.k + b * p.k_bs + hk * p.dh + c0;
  const T* V = (const T*)p.v + b * p.v_bs + hk * p.dh + c0;
  Raw kn[U], vn[U];                                              // the next step's keys and values, in flight during this one's sums
  unsigned okn = 0;
  auto load = [&](int j0) {
    okn = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * GPB + grp;
      kn[u] = Raw(0); vn[u] = Raw(0);
      if (j < k1 && !(p.mask && p.mask[(long long)b * p.S + j])) {
        okn |= 1u << u;
        if (in) {
          kn[u] = *reinterpret_cast<const Raw*>(K + (long long)j * p.ldk);
          vn[u] = *reinterpret_cast<const Raw*>(V + (long long)j * p.ldv);
        }
      }
    }
  };
  if (k0 < k1) load(k0);
  for (int j0 = k0; j0 < k1; j0 += GPB * U) {
    Raw kr[U], vr[U];
    const unsigned ok = okn;
#pragma unroll
    for (int u = 0; u < U; ++u) { kr[u] = kn[u]; vr[u] = vn[u]; }
    if (j0 + GPB * U < k1) load(j0 + GPB * U);
    // the step's keys all beyond one end of the map for all rows: the bias is one number a row
    const bool far_lo = j0 + GPB * U - 1 - pmin - p.map_lo <= 0, far_hi = j0 - pmax - p.map_lo >= p.map_n - 1;
    float s[RT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[EPL];
      R::wide(kr[u], kf);
      const int j = j0 + u * GPB + grp;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) x = fmaf(q[r][e], kf[e], x);
        x = lanes_sum<LPK>(x);
        const int delta = j - pos[r];
        x += far_lo ? fb[r] : far_hi ? lb[r] : p.table[(long long)p.map[p.entry(delta)] * p.H + hd[r]] * LOG2E;
        s[r][u] = (ok >> u & 1) && !(p.causal && delta > 0) ? x : -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float mn = fmaxf(m[r], fmaxf(fmaxf(s[r][0], s[r][1]), fmaxf(s[r][2], s[r][3])));
      const float mf = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m[r] - mf);
      m[r] = mn; l[r] *= al;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] *= al;
#pragma unroll
      for (int u = 0; u < U; ++u) { s[r][u] = __builtin_amdgcn_exp2f(s[r][u] - mf); l[r] += s[r][u]; }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vf[EPL];
      R::wide(vr[u], vf);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] = fmaf(s[r][u], vf[e], o[r][e]);
    }
  }
  // join the groups: first those of a wave, lane by lane, then the waves through LDS
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int x = LPK; x < 64; x <<= 1) {
      const float m2 = __shfl_xor(m[r], x, 64), l2 = __shfl_xor(l[r], x, 64), mn = fmaxf(m[r], m2);
      const float f1 = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - mn), f2 = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] = o[r][e] * f1 + __shfl_xor(o[r][e], x, 64) * f2;
      l[r] = l[r] * f1 + l2 * f2; m[r] = mn;
    }
  constexpr int W = LPK * EPL + 2;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane < LPK) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float* w = red + (wave * RT + r) * W;
#pragma unroll
      for (int e = 0; e < EPL; ++e) w[2 + c0 + e] = o[r][e];
      if (sub == 0) { w[0] = m[r]; w[1] = l[r]; }
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < RT * p.dh; t += 256) {
    const int r = t / p.dh, c = t - r * p.dh, row = rc * RT + r;
    if (row >= rows) break;
    float mm = -INFINITY, ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, red[(w * RT + r) * W]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(red[(w * RT + r) * W] - mm);
      ll += f * red[(w * RT + r) * W + 1]; oo += f * red[(w * RT + r) * W + 2 + c];
    }
    const int h = hk * p.G + row / p.L, i = row % p.L;
    const long long at = ((long long)b * p.H + h) * p.L + i;
    if (a.nparts > 1) {
      a.part_o[(at * a.nparts + part) * p.dh + c] = oo;
      if (c == 0) *reinterpret_cast<float2*>(a.part_ml + (at * a.nparts + part) * 2) = make_float2(mm, ll);
    } else {
      St<T>::st((T*)p.o + b * p.o_bs + (long long)i * p.ldo + h * p.dh + c, ll == 0.f ? 0.f : oo / ll);
      if (p.lse && c == 0) p.lse[at] = ll == 0.f ? INFINITY : mm + __log2f(ll);
    }
  }
}

// o = sum 2^(m_t - m) o_t / sum 2^(m_t - m) l_t over the parts.  8, 16 or 32 lanes hold a row's columns, four each; up to 8 parts go by one after the other and a
// wave has several rows, more are dealt to runs of lanes and joined by shuffles.  The lanes of a row first take a part each for m and the sum of l; the
// parts' rows follow with four loads in flight (one at a time, 128 parts of 16 rows took longer than the pass over the 67 MB of their keys).
template <typename T>
__global__ __launch_bounds__(256) void relpos_join_kernel(RP p, Src a) {
  const int lanes = p.dh <= 32 ? 8 : p.dh <= 64 ? 16 : 32, runs = a.nparts <= 8 ? 1 : 64 / lanes, per = lanes * runs, n = a.nparts;
  const int lane = threadIdx.x & 63, at = lane % per, run = at / lanes, c = lane % lanes * 4;
  const long long row = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (64 / per) + lane / per;
  if (row >= (long long)p.B * p.H * p.L) return;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * n;
  float m = -INFINITY;
  for (int s = at; s < n; s += per) m = fmaxf(m, ml[s].x);
  for (int o = 1; o < per; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float mf = m == -INFINITY ? 0.f : m;
  float l = 0.f, x = 0.f, y = 0.f, z = 0.f, w = 0.f;
  for (int s = at; s < n; s += per) { const float2 t = ml[s]; l += __builtin_amdgcn_exp2f(t.x - mf) * t.y; }
  for (int o = 1; o < per; o <<= 1) l += __shfl_xor(l, o, 64);
  if (c < p.dh) {
    const float* O = a.part_o + row * n * p.dh + c;
    for (int s0 = run; s0 < n; s0 += 4 * runs) {
      float f[4];
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = min(s0 + u * runs, n - 1);
        f[u] = ml[s].x;
        v[u] = *reinterpret_cast<const float4*>(O + (long long)s * p.dh);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (s0 + u * runs >= n) break;
        const float e = __builtin_amdgcn_exp2f(f[u] - mf);
        x += e * v[u].x; y += e * v[u].y; z += e * v[u].z; w += e * v[u].w;
      }
    }
  }
  for (int o = lanes; o < per; o <<= 1) { x += __shfl_xor(x, o, 64); y += __shfl_xor(y, o, 64); z += __shfl_xor(z, o, 64); w += __shfl_xor(w, o, 64); }
  if (run) return;
  const float il = l == 0.f ? 0.f : 1.f / l;
  const int i = (int)(row % p.L), h = (int)(row / p.L % p.H);
  const long long b = row / p.L / p.H;
  if (c < p.dh) St<T>::st4((T*)p.o + b * p.o_bs + (long long)i * p.ldo + h * p.dh + c, make_float4(x * il, y * il, z * il, w * il));
  if (p.lse && c == 0) p.lse[row] = l == 0.f ? INFINITY : m + __log2f(l);
}

// ---- which kernel, in how many parts ---------------------------------------------------------------------------------------------
struct Plan { bool token; int nparts, per, rt; long long blocks; int64_t split_ws, part_ws; };

// Which kernel.  The token kernel's time grows with the rows that share a key (four at a time), the tile kernel's does not up to 32 queries, but fp32 storage has
// its keys split first.  16 heads of 64, 4 x 4096 keys, us, token / tile: fp32 16 kv heads, 1 query 29 / 82, 4 42 / 82, 8 63 / 82, 32 269 / 86; 4 kv heads, 1 21 / 41, 2 26 / 41,
// 3 35 / 41, 4 42 / 41, 8 62 / 41; 1 kv head, 1 21 / 34, 2 28 / 33, 3 35 / 34.  bf16 16 kv heads, 1 query 20 / 22, 2 26 / 23, 3 33 / 23; 4 kv heads, 1 19 / 20, 2 21 / 19, 3 31 / 21.
// Likewise at 8 x 1024 keys of 32, 2 x 8192 of 128 and 32768 of 64.
Plan plan(const smx_relpos_desc* d, const RP& p) {
  Plan w;
  const long long rows = (long long)p.G * p.L;
  w.token = d->bf16 ? p.L == 1 : p.L <= 2 || (p.L <= 12 && rows <= 12);
  w.split_ws = 0;
  w.rt = rows >= 3 ? 4 : (int)rows;                                   // (8 at a time: 8 rows 110 us instead of 63)
  const long long base = w.token ? (long long)p.B * p.Hkv * ((rows + w.rt - 1) / w.rt) : (long long)p.B * p.H * ((p.L + 127) / 128);
  // parts of the keys from 513 keys on, none shorter than 256, until the chip's 256 CUs have two blocks each (the 32-column and the small bf16 kernels would hold three;
  // few queries, bound by the loads in flight: four).  Parts are cut from S, so that those behind a shorter sample's end have nothing to do.  In
  // parts / not, 8 heads of 64: 1024 queries on 4096 keys fp32 52 / 130 us, 128 on 8192 bf16 22 / 154, 1 on 4096 fp32 15 / 64
  long long np = ((w.token ? 1024 : 512) + base - 1) / base, most = p.S <= 512 ? 1 : (p.S + 255) / 256;
  if (np > most) np = most;
  w.per = (int)(((p.S + np - 1) / np + 63) / 64 * 64);
  w.nparts = (p.S + w.per - 1) / w.per;
  w.blocks = base * w.nparts;
  if (!w.token && !d->bf16) w.split_ws = 2 * split_bytes(p.B, p.Hkv, p.S, p.dh);
  w.part_ws = w.nparts > 1 ? (int64_t)p.B * p.H * p.L * w.nparts * (p.dh + 4) * 4 : 0;
  return w;
}

template <int DHP, int NL>
int tile_launch(const RP& p, const Src& a, const Plan& w, hipStream_t st) {
  const int fixed = BUFFERS<DHP, NL> * 2 * NL * STEP<DHP, NL> * ROWB<DHP>, lds = fixed + ((p.map_n + 2 * TABLE_PAD) * 4 + 15) / 16 * 16;
  SMX_HIP(smx_max_dynamic_lds((const void*)(relpos_tile_kernel<DHP, NL>), fixed + ((MAP_MAX + 2 * TABLE_PAD) * 4 + 15) / 16 * 16));
  SMX_LAUNCH((relpos_tile_kernel<DHP, NL>), dim3((unsigned)w.blocks), dim3(256), lds, st, p, a);
  return smx_launch_status();
}

template <typename T, int EPL, int LPK>
int token_launch(const RP& p, const Src& a, const Plan& w, hipStream_t st) {
  const int lds = 4 * w.rt * (LPK * EPL + 2) * 4;
  const dim3 grid((unsigned)w.blocks), block(256);
  if (w.rt == 4) SMX_LAUNCH((relpos_token_kernel<T, EPL, LPK, 4>), grid, block, lds, st, p, a);
  else if (w.rt == 2) SMX_LAUNCH((relpos_token_kernel<T, EPL, LPK, 2>), grid, block, lds, st, p, a);
  else SMX_LAUNCH((relpos_token_kernel<T, EPL, LPK, 1>), grid, block, lds, st, p, a);
  return smx_launch_status();
}

template <typename T, int EPL>
int token_width(const RP& p, const Src& a, const Plan& w, hipStream_t st) {
  if (p.dh <= 4 * EPL) return token_launch<T, EPL, 4>(p, a, w, st);
  if (p.dh <= 8 * EPL) return token_launch<T, EPL, 8>(p, a, w, st);
  if (p.dh <= 16 * EPL) return token_launch<T, EPL, 16>(p, a, w, st);
  return token_launch<T, EPL, 32>(p, a, w, st);
}

}  // namespace

extern "C" int64_t smx_attention_relpos_ws_bytes(const smx_relpos_desc* d) {
  RP p;
  if (check(d, p, false) != SMX_OK) return -1;
  const Plan w = plan(d, p);
  return w.split_ws + w.part_ws;
}

extern "C" int smx_attention_relpos(const smx_relpos_desc* d, void* stream) {
  RP p;
  int rc = check(d, p, false);
  if (rc != SMX_OK) return rc;
  const Plan w = plan(d, p);
  if (w.blocks > 0x7fffffffLL || (w.split_ws + w.part_ws && (!d->ws || !aligned(d->ws, 16) || d->ws_bytes < w.split_ws + w.part_ws))) return SMX_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  Src a{};
  a.nparts = w.nparts; a.per = w.per;
  char* ws = (char*)d->ws;
  if (w.part_ws) {
    a.part_o = (float*)(ws + w.split_ws);
    a.part_ml = a.part_o + (int64_t)p.B * p.H * p.L * w.nparts * p.dh;
  }
  if (w.token) {
    if (!d->bf16) rc = token_width<float, 4>(p, a, w, st);
    else if (p.dh % 8 == 0 && (p.ldq | p.ldk | p.ldv) % 8 == 0 && (p.q_bs | p.k_bs | p.v_bs) % 8 == 0 && aligned(p.q, 16) && aligned(p.k, 16) && aligned(p.v, 16))
      rc = token_width<bf16_t, 8>(p, a, w, st);
    else rc = token_width<bf16_t, 4>(p, a, w, st);
  } else {
    if (!d->bf16) {
      ws = split_setup(a.k, ws, (const float*)p.k, p.k_bs, p.ldk, p.B, p.Hkv, p.S, p.dh, true);
      ws = split_setup(a.v, ws, (const float*)p.v, p.v_bs, p.ldv, p.B, p.Hkv, p.S, p.dh, true);
      const Split both[2] = {a.k, a.v};
      rc = split_launch(p, both, 2, st);
      if (rc != SMX_OK) return rc;
    }
    switch (dhp(p.dh)) {
      case 32: rc = d->bf16 ? tile_launch<32, 1>(p, a, w, st) : tile_launch<32, 2>(p, a, w, st); break;
      case 64: rc = d->bf16 ? tile_launch<64, 1>(p, a, w, st) : tile_launch<64, 2>(p, a, w, st); break;
      case 96: rc = d->bf16 ? tile_launch<96, 1>(p, a, w, st) : tile_launch<96, 2>(p, a, w, st); break;
      default: rc = d->bf16 ? tile_launch<128, 1>(p, a, w, st) : tile_launch<128, 2>(p, a, w, st);
    }
  }
  if (rc != SMX_OK || w.nparts == 1) return rc;
  const int rows_a_block = 4 * (w.nparts <= 8 ? 64 / (p.dh <= 32 ? 8 : p.dh <= 64 ? 16 : 32) : 1);
  const long long nj = ((long long)p.B * p.H * p.L + rows_a_block - 1) / rows_a_block;
  if (nj > 0x7fffffffLL) return SMX_EINVAL;
  if (d->bf16) SMX_LAUNCH(relpos_join_kernel<bf16_t>, dim3((unsigned)nj), dim3(256), 0, st, p, a);
  else SMX_LAUNCH(relpos_join_kernel<float>, dim3((unsigned)nj), dim3(256), 0, st, p, a);
  return smx_launch_status();
}
