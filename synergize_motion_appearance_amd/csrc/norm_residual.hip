// The norms around a block, its gate and residual (include/smx.h: smx_norm_residual, smx_norm_residual_bwd_f32).
//   n = Norm(h),  x' = rs x + g n,  y = Norm(x')
// Backward, with c the gradient of x' (its own plus what comes back through y), hat = (v - mean) r the normalised rows:
//   NormBwd(g; v) = r (gamma g - mean(gamma g) - hat mean(gamma g hat))       (rms: without the middle term, mean = 0)
//   c = gx + NormBwd(gy; x'),  dx = rs c,  dn = g c,  dh = NormBwd(dn; h),  dgate = sum n c,  dgamma = sum g hat,  dbeta = sum g
// Bound by memory: forward reads x, h and writes x', y; backward reads x', h, gx, gy and writes dx, dh.  A large copy reaches 4.7 TB/s on this card.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <initializer_list>
#include "smx.h"
#include "smx_common.h"
#include "bf16.h"

namespace {

struct NRP {
  const void* x; const void* h; void* xo; void* y;
  const float* pg; const float* pb; const float* ng; const float* nb; const float* gate;
  const float* gx; const float* gy; float* dx; float* dh; float* part;
  long long T, per; int E, rms, nblk, rows, want; // want: which parameter sums; per: tokens of a gate row; nblk blocks of `rows` tokens walk each gate row's tokens
  float rs, eps;
};

// LPR lanes hold a row: lane `sub` the V columns of chunks sub, sub + LPR, ... (N of them); a block of BT threads BT / LPR rows at a time.  V is 16 bytes
// of the storage type.
template <int LPR>
struct Lanes {
  static constexpr int BT = LPR > 256 ? LPR : 256, RPB = BT / LPR, W = LPR / 64;
  int sub, row, turn = 0;
  float2* red;                                                    // [2][W], rows of more than a wave
  __device__ __forceinline__ Lanes(float2* r) : sub(threadIdx.x % LPR), row(threadIdx.x / LPR), red(r) {}
  // a row's sums of x and y, in all its lanes.  The two halves of `red` take turns: one barrier a sum
  __device__ __forceinline__ void sum(float& x, float& y) {
#pragma unroll
    for (int o = LPR < 64 ? LPR / 2 : 32; o > 0; o >>= 1) { x += __shfl_xor(x, o, 64); y += __shfl_xor(y, o, 64); }
    if constexpr (LPR > 64) {
      float2* r = red + turn * W;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = make_float2(x, y);
      __syncthreads();
      x = y = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) { x += r[w].x; y += r[w].y; }
    }
  }
};

// U: rows start anywhere and end inside a chunk.  The same 16-byte accesses then, which the card makes at any address of the type; a row's last chunk, of which
// not all columns are there, is read column by column -- or (S), where the next row is on its way while this one is summed and a branch would wait for it,
// from `back` columns before, and moved down once it has arrived, zeros behind it.  Forward and backward, us, all rows column by column / last chunks / S:
// 65536 x 250 183 / 258 / 168, 8192 x 1026 179 / 133 / 128, 2658 x 2470 175 / 90 / 126, 4096 x 4098 729 / 234 / 287 (S: more registers than two waves a SIMD have).
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u4u __attribute__((ext_vector_type(4), aligned(2)));
template <int V, bool S> __device__ __forceinline__ int back_of(int E, int c) { return S && E >= V ? max(0, c + V - E) : 0; }
template <typename TS, int V, bool U, bool S> __device__ __forceinline__ void ldr(const TS* row, int c, int E, float* f) {
  const TS* p = row + c - back_of<V, S>(E, c);
  if (U && (S ? E : E - c) < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < E - c ? St<TS>::ld(row + c + e) : 0.f;
  } else if constexpr (sizeof(TS) == 2) {
    float g[8];
    if constexpr (U) { const u4u x = *reinterpret_cast<const u4u*>(p); unpack8(make_uint4(x.x, x.y, x.z, x.w), g); }
    else unpack8(*reinterpret_cast<const uint4*>(p), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = g[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      if constexpr (U) { const f4u v = *reinterpret_cast<const f4u*>(p + e); f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w; }
      else { const float4 v = St<float>::ld4((const float*)p + e); f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w; }
    }
  }
}
template <int V, bool S> __device__ __forceinline__ void down(float* f, int back) {
  if (!S || !back) return;
#pragma unroll
  for (int b = 1; b < V; b <<= 1)
    if (back & b) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = e + b < V ? f[e + b] : 0.f;
    }
}
template <typename TS, int V, bool U> __device__ __forceinline__ void stv(TS* row, int c, int E, const float* f) {
  TS* p = row + c;
  if (U && E - c < V) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < E - c) St<TS>::st(p + e, f[e]);
  } else if constexpr (V == 8) {
    const float g[8] = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
    const uint4 x = pack8(g);
    if constexpr (U) *reinterpret_cast<u4u*>(p) = u4u{x.x, x.y, x.z, x.w};
    else *reinterpret_cast<uint4*>(p) = x;
  } else if constexpr (U) *reinterpret_cast<f4u*>(p) = f4u{f[0], f[1], f[2], f[3]};
  else St<TS>::st4(p, make_float4(f[0], f[1], f[2], f[3]));
}
// V fp32 parameters, `other` without them
template <int V, bool U, bool S> __device__ __forceinline__ void ldp(const float* p, int c, int E, float other, float* f) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = other;
  } else {
    ldr<float, V, U, S>(p, c, E, f);
    down<V, S>(f, back_of<V, S>(E, c));
  }
}

// mean and 1 / sqrt(var + eps) of two rows at a time (b unused: pass zeros): the sums first, then the squares of the deviations -- never a difference of
// squares
template <int NV, int LPR>
__device__ __forceinline__ void stats2(Lanes<LPR>& ln, const float (&a)[NV], const float (&b)[NV], const bool (&in)[NV], int E, int rms, float eps, float& ma, float& ra,
                                       float& mb, float& rb) {
  const float iE = 1.f / E;
  ma = mb = 0.f;
  if (!rms) {
#pragma unroll
    for (int k = 0; k < NV; ++k) { ma += a[k]; mb += b[k]; }
    ln.sum(ma, mb);
    ma *= iE; mb *= iE;
  }
  float qa = 0.f, qb = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) { const float x = in[k] ? a[k] - ma : 0.f, y = in[k] ? b[k] - mb : 0.f; qa = fmaf(x, x, qa); qb = fmaf(y, y, qb); }
  ln.sum(qa, qb);
  ra = 1.f / sqrtf(qa * iE + eps); rb = 1.f / sqrtf(qb * iE + eps);
}

// Forward: x and h are read once, x' and y written once; a row stays in its lanes' registers between the two norms.  With up to 8 columns a lane
// the parameters stay there too (five rows of fp32 against four of data: read again for every row they would be most of a CU's loads).
// 307200 x 256 bf16: 131 us, 4.8 TB/s; 15999 x 2048 fp32: 98 us, 5.4 TB/s; 8 x 4096 bf16: 11 us, the launch and the caller's own work.  Parameters read again for
// every row: 45 us instead of 43 at 65536 x 256 fp32.
template <typename TS, int V, int LPR, int N, bool U>
__global__ __launch_bounds__(Lanes<LPR>::BT) void norm_residual_kernel(NRP p) {
  constexpr int NV = N * V;
  constexpr bool HOLD = NV <= 8;
  __shared__ float2 red[2 * (LPR > 64 ? LPR / 64 : 1)];
  Lanes<LPR> ln(red);
  float pg[HOLD ? NV : 1], pb[HOLD ? NV : 1], ng[HOLD ? NV : 1], nb[HOLD ? NV : 1], gt[HOLD ? NV : 1];
  bool in[NV];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = (ln.sub + LPR * k) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) in[k * V + e] = c + (U ? e : 0) < p.E;
    if constexpr (HOLD)
      if (c < p.E) { ldp<V, U, false>(p.pg, c, p.E, 1.f, pg + k * V); ldp<V, U, false>(p.pb, c, p.E, 0.f, pb + k * V); ldp<V, U, false>(p.ng, c, p.E, 1.f, ng + k * V); ldp<V, U, false>(p.nb, c, p.E, 0.f, nb + k * V);
                     ldp<V, U, false>(p.per == p.T ? p.gate : nullptr, c, p.E, 1.f, gt + k * V); }
  }
  const bool same_gate = HOLD && p.per == p.T;
  for (long long t = blockIdx.x * (long long)Lanes<LPR>::RPB + ln.row; t < p.T; t += (long long)gridDim.x * Lanes<LPR>::RPB) {
    const long long at = t * p.E;
    const float* gate = p.gate ? p.gate + (p.per == p.T ? 0 : t / p.per * p.E) : nullptr;
    float x[NV], v[NV], zero[NV];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (ln.sub + LPR * k) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) x[k * V + e] = v[k * V + e] = zero[k * V + e] = 0.f;
      if (c < p.E) {
        ldr<TS, V, U, false>((const TS*)p.x + at, c, p.E, x + k * V); ldr<TS, V, U, false>((const TS*)p.h + at, c, p.E, v + k * V);
      }
    }
    float mean = 0.f, r = 1.f, m2, r2;
    if (p.pg) stats2<NV, LPR>(ln, v, zero, in, p.E, p.rms, p.eps, mean, r, m2, r2);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (ln.sub + LPR * k) * V;
      if (c < p.E) {
        float a[V], b[V], g[V];
        if constexpr (HOLD) {
#pragma unroll
          for (int e = 0; e < V; ++e) { a[e] = pg[k * V + e]; b[e] = pb[k * V + e]; g[e] = gt[k * V + e]; }
        } else { ldp<V, U, false>(p.pg, c, p.E, 1.f, a); ldp<V, U, false>(p.pb, c, p.E, 0.f, b); }
        if (!same_gate) ldp<V, U, false>(gate, c, p.E, 1.f, g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float n = fmaf((v[k * V + e] - mean) * r, a[e], b[e]);
          TS w;
          St<TS>::st(&w, fmaf(g[e], n, p.rs * x[k * V + e]));
          v[k * V + e] = St<TS>::ld(&w);             // y is the norm of what is stored
        }
        stv<TS, V, U>((TS*)p.xo + at, c, p.E, v + k * V);
      }
    }
    if (!p.y) continue;
    stats2<NV, LPR>(ln, v, zero, in, p.E, p.rms, p.eps, mean, r, m2, r2);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (ln.sub + LPR * k) * V;
      if (c < p.E) {
        float a[V], b[V];
        if constexpr (HOLD) {
#pragma unroll
          for (int e = 0; e < V; ++e) { a[e] = ng[k * V + e]; b[e] = nb[k * V + e]; }
        } else { ldp<V, U, false>(p.ng, c, p.E, 1.f, a); ldp<V, U, false>(p.nb, c, p.E, 0.f, b); }
#pragma unroll
        for (int e = 0; e < V; ++e) v[k * V + e] = fmaf((v[k * V + e] - mean) * r, a[e], b[e]);
        stv<TS, V, U>((TS*)p.y + at, c, p.E, v + k * V);
      }
    }
  }
}

// Backward: a block walks `rows` tokens of one gate row, each thread keeping its columns' five parameter sums in registers; the block's sums go to
// part [groups * nblk][5][E] (dpre gamma, dpre beta, dpost gamma, dpost beta, dgate; those that are wanted), norm_residual_sum_kernel adds the blocks.
// 15999 x 2048, six rows of fp32 a token, 786 MB: 189 us, 4.2 TB/s, with 7 us for the blocks' sums.
template <int V, int LPR, int N, bool U>
__global__ __launch_bounds__(Lanes<LPR>::BT) void norm_residual_bwd_kernel(NRP p) {
  constexpr int NV = N * V, BT = Lanes<LPR>::BT, RPB = Lanes<LPR>::RPB;
  __shared__ float2 red[2 * (LPR > 64 ? LPR / 64 : 1)];
  __shared__ float join[LPR > 64 ? 1 : 4 * LPR * NV];
  Lanes<LPR> ln(red);
  const long long g = blockIdx.x / p.nblk, blk = blockIdx.x - g * p.nblk;
  const float* gate = p.gate ? p.gate + g * p.E : nullptr;
  float a[5][NV];
  bool in[NV];
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int k = 0; k < NV; ++k) a[i][k] = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) in[k] = (ln.sub + LPR * (k / V)) * V + (U ? k % V : 0) < p.E;
  const long long t1 = g * p.per + min(p.per, (blk + 1) * (long long)p.rows);
  const float iE = 1.f / p.E;
  constexpr bool AHEAD = NV <= 8;                    // the next row is on its way during this one's sums (with the forward, 65536 x 256: 151 us instead of 194)
  constexpr bool SH = U && AHEAD;
  float row[2][4][NV];
  auto load = [&](float (&w)[4][NV], long long t) {
    const long long at = t * p.E;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int col = (ln.sub + LPR * k) * V;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][k * V + e] = 0.f;
      if (col < p.E) {
        ldr<float, V, U, SH>((const float*)p.h + at, col, p.E, w[1] + k * V);
        if (p.gx) ldr<float, V, U, SH>(p.gx + at, col, p.E, w[2] + k * V);
        if (p.gy) { ldr<float, V, U, SH>((const float*)p.xo + at, col, p.E, w[0] + k * V); ldr<float, V, U, SH>(p.gy + at, col, p.E, w[3] + k * V); }
      }
    }
  };
  long long t = g * p.per + blk * p.rows + ln.row;
  if (AHEAD && t < t1) load(row[1], t);
  for (; t < t1; t += RPB) {
    const long long at = t * p.E;
    float (&x)[NV] = row[0][0];
    float (&h)[NV] = row[0][1];
    float (&c)[NV] = row[0][2];
    float (&gy)[NV] = row[0][3];
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < NV; ++k) row[0][i][k] = row[1][i][k];
      if (t + RPB < t1) load(row[1], t + RPB);
    } else load(row[0], t);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int col = (ln.sub + LPR * k) * V;
#pragma unroll
      for (int i = 0; i < 4; ++i) down<V, SH>(row[0][i] + k * V, col < p.E ? back_of<V, SH>(p.E, col) : 0);
    }
    float mx, rx, mh, rh, s1 = 0.f, s2 = 0.f;
    stats2<NV, LPR>(ln, x, h, in, p.E, p.rms, p.eps, mx, rx, mh, rh);
    if (p.gy) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int col = (ln.sub + LPR * k) * V;
        float w[V];
        if (col < p.E) {
          ldp<V, U, SH>(p.ng, col, p.E, 1.f, w);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int i = k * V + e;
            const float hat = (x[i] - mx) * rx;
            a[0][i] = fmaf(gy[i], hat, a[0][i]); a[1][i] += gy[i];
            gy[i] *= w[e]; x[i] = hat;
            s1 += gy[i]; s2 = fmaf(gy[i], hat, s2);
          }
        }
      }
      ln.sum(s1, s2);
      s1 = p.rms ? 0.f : s1 * iE; s2 *= iE;
#pragma unroll
      for (int k = 0; k < NV; ++k) if (in[k]) c[k] = fmaf(rx, gy[k] - s1 - x[k] * s2, c[k]);
    }
    if (p.dx) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int col = (ln.sub + LPR * k) * V;
        float w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = p.rs * c[k * V + e];
        if (col < p.E) stv<float, V, U>(p.dx + at, col, p.E, w);
      }
    }
    s1 = s2 = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int col = (ln.sub + LPR * k) * V;
      float w[V], b[V], gt[V];
      if (col < p.E) {
        ldp<V, U, SH>(p.pg, col, p.E, 1.f, w); ldp<V, U, SH>(p.pb, col, p.E, 0.f, b); ldp<V, U, SH>(gate, col, p.E, 1.f, gt);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int i = k * V + e;
          if (!p.pg) { a[4][i] = fmaf(c[i], h[i], a[4][i]); c[i] *= gt[e]; continue; }
          const float hat = (h[i] - mh) * rh, dn = gt[e] * c[i];
          a[4][i] = fmaf(c[i], fmaf(hat, w[e], b[e]), a[4][i]);
          a[2][i] = fmaf(dn, hat, a[2][i]); a[3][i] += dn;
          c[i] = dn * w[e]; h[i] = hat;
          s1 += c[i]; s2 = fmaf(c[i], hat, s2);
        }
      }
    }
    if (p.pg) {
      ln.sum(s1, s2);
      s1 = p.rms ? 0.f : s1 * iE; s2 *= iE;
#pragma unroll
      for (int k = 0; k < NV; ++k) c[k] = rh * (c[k] - s1 - h[k] * s2);
    }
    if (p.dh) {
#pragma unroll
      for (int k = 0; k < N; ++k) { const int col = (ln.sub + LPR * k) * V; if (col < p.E) stv<float, V, U>(p.dh + at, col, p.E, c + k * V); }
    }
  }
  float* part = p.part + (long long)blockIdx.x * 5 * p.E;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    if (!(p.want >> i & 1)) continue;
    if constexpr (LPR > 64) {
#pragma unroll
      for (int k = 0; k < N; ++k) { const int col = (ln.sub + LPR * k) * V; if (col < p.E) stv<float, V, U>(part + (long long)i * p.E, col, p.E, a[i] + k * V); }
    } else {                                         // the rows of a wave by shuffles, its four waves through LDS
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) a[i][k] += __shfl_xor(a[i][k], o, 64);
      __syncthreads();
      if ((threadIdx.x & 63) < LPR) {
#pragma unroll
        for (int k = 0; k < NV; ++k) join[((threadIdx.x >> 6) * LPR + ln.sub) * NV + k] = a[i][k];
      }
      __syncthreads();
      for (int j = threadIdx.x; j < LPR * NV; j += BT) {
        const int col = (j / NV + LPR * (j % NV / V)) * V + j % V;
        if (col < p.E) part[(long long)i * p.E + col] = (join[j] + join[LPR * NV + j]) + (join[2 * LPR * NV + j] + join[3 * LPR * NV + j]);
      }
    }
  }
}

struct Outs { float* p[5]; };

// the blocks' sums in a fixed order: 32 columns by 32 runs of blocks a thread block; grid.y 0..3 the parameters (over all blocks), 4 + g the gate row g (over
// its own)
__global__ __launch_bounds__(1024) void norm_residual_sum_kernel(const float* __restrict__ part, Outs o, int E, long long nall, int nblk, int gate_acc, long long g0) {
  __shared__ float red[32][33];
  const int which = min((int)blockIdx.y, 4), cl = threadIdx.x & 31, run = threadIdx.x >> 5, e = blockIdx.x * 32 + cl;
  float* out = o.p[which];
  if (!out) return;
  const long long g = g0 + (int)blockIdx.y - which, n0 = which < 4 ? 0 : g * nblk, n1 = which < 4 ? nall : n0 + nblk;
  float s = 0.f;
  if (e < E) {
#pragma unroll 8
    for (long long n = n0 + run; n < n1; n += 32) s += part[(n * 5 + which) * E + e];
  }
  red[run][cl] = s;
  __syncthreads();
  if (run || e >= E) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += red[i][cl];
  if (which < 4) out[e] += s;
  else out[g * E + e] = gate_acc ? out[g * E + e] + s : s;
}

// Lanes a row and chunks a lane, by the row's 16-byte chunks: up to a wave's 64 lanes one chunk each, then up to 4
// a lane (256 chunks over 256 lanes with their barriers: 52 us instead of 44 at 16384 x 1024 fp32), then rows over a block -- of 256 threads for up to 1024
// chunks, 512 beyond, so that the backward's five sums of a thread's columns stay in registers up to 8192 columns.  Beyond, five sums of 32 columns next to the row
// do not fit (some 320 registers go through scratch): 1024 x 16384 404 us with the forward's 61, 2048 x 8192 202 with 67.
template <typename TS, int V, bool U, template <typename, int, int, int, bool> class K>
int by_width(const NRP& p, hipStream_t st) {
  const int n = smx_cdiv(p.E, V);
  if (n <= 8) return K<TS, V, 8, 1, U>::go(p, st);
  if (n <= 16) return K<TS, V, 16, 1, U>::go(p, st);
  if (n <= 32) return K<TS, V, 32, 1, U>::go(p, st);
  if (n <= 64) return K<TS, V, 64, 1, U>::go(p, st);
  if (n <= 128) return K<TS, V, 64, 2, U>::go(p, st);
  if (n <= 256) return K<TS, V, 64, 4, U>::go(p, st);
  if (n <= 512) return K<TS, V, 256, 2, U>::go(p, st);
  if (n <= 1024) return K<TS, V, 256, 4, U>::go(p, st);
  if (n <= 2048) return K<TS, V, 512, 4, U>::go(p, st);
  if constexpr (V == 4) return K<TS, V, 512, 8, U>::go(p, st);
  return SMX_EINVAL;
}

template <typename TS, int V, int LPR, int N, bool U> struct Fwd {
  static int go(const NRP& p, hipStream_t st) {
    const long long need = (p.T + Lanes<LPR>::RPB - 1) / Lanes<LPR>::RPB;
    SMX_LAUNCH((norm_residual_kernel<TS, V, LPR, N, U>), dim3((unsigned)(need < 4096 ? need : 4096)), dim3(Lanes<LPR>::BT), 0, st, p);
    return smx_launch_status();
  }
};
template <typename TS, int V, int LPR, int N, bool U> struct Bwd {
  static int go(const NRP& p, hipStream_t st) {
    SMX_LAUNCH((norm_residual_bwd_kernel<V, LPR, N, U>), dim3((unsigned)(p.T / p.per * p.nblk)), dim3(Lanes<LPR>::BT), 0, st, p);
    return smx_launch_status();
  }
};

// tokens a backward block walks: about 512 blocks (their sums are written and read once more), 256 of rows that take a block of 512 threads -- one a CU at a time
// --, but not fewer tokens than it has rows at a time.  Forward and backward with 256 / 512 / 1024 blocks: 65536 x 256 195 / 151 / 144 us, 8192 x 2048
// 177 / 148 / 158, 4096 x 4096 178 / 160 / 181, 2048 x 8192 194 / 218 / 234, 1024 x 16384 378 / 421 / 499.  A block ends with its gate row: with a row for every token
// a block has one token, and the blocks' sums are more than the tensors (5 T E floats): 65536 x 256 1709 us instead of 153.
int rows_of(long long T, long long per, int E) {
  const int want = E > 4096 ? 256 : 512;
  long long r = (T + want - 1) / want;
  const int at_a_time = E <= 32 ? 32 : E <= 64 ? 16 : E <= 128 ? 8 : E <= 1024 ? 4 : 1;
  if (r < at_a_time) r = at_a_time;
  if (r > per) r = per;
  return (int)r;
}

int check(const smx_norm_residual_desc* d, bool bwd) {
  if (!d || (!bwd && (!d->x || !d->pre_gamma != !d->y)) || !d->h || !d->xo || d->T <= 0 || d->groups <= 0 || d->T % d->groups || d->E <= 0 || d->E > 16384 || d->T > 0x7fffffffLL) return SMX_EINVAL;
  if ((d->post_beta && !d->post_gamma) || (d->pre_beta && !d->pre_gamma) || (d->groups > 1 && !d->gate)) return SMX_EINVAL;
  if (!(d->eps >= 0.f) || !(d->res_scale == d->res_scale) || (d->bf16 != 0 && d->bf16 != 1)) return SMX_EINVAL;
  return SMX_OK;
}

NRP params(const smx_norm_residual_desc* d) {
  NRP p;
  p.x = d->x; p.h = d->h; p.xo = d->xo; p.y = d->y; p.pg = d->post_gamma; p.pb = d->post_beta; p.ng = d->pre_gamma; p.nb = d->pre_beta; p.gate = d->gate;
  p.gx = d->gx; p.gy = d->gy; p.dx = d->dx; p.dh = d->dh; p.part = d->ws; p.T = d->T; p.per = d->T / d->groups; p.E = d->E; p.rms = d->rms != 0;
  p.rows = rows_of(d->T, p.per, d->E); p.nblk = smx_cdiv(p.per, p.rows); p.rs = d->res_scale; p.eps = d->eps;
  p.want = (d->dpre_gamma ? 1 : 0) | (d->dpre_beta ? 2 : 0) | (d->dpost_gamma ? 4 : 0) | (d->dpost_beta ? 8 : 0) | (d->dgate ? 16 : 0);
  return p;
}

// do all rows of these tensors start on 16 bytes?
bool wide(int E, int size, std::initializer_list<const void*> ps) {
  uintptr_t a = (uintptr_t)E * size;
  for (const void* p : ps) a |= (uintptr_t)p;
  return (a & 15) == 0;
}

}  // namespace

extern "C" int smx_norm_residual(const smx_norm_residual_desc* d, void* stream) {
  const int rc = check(d, false);
  if (rc != SMX_OK) return rc;
  const NRP p = params(d);
  hipStream_t st = (hipStream_t)stream;
  const bool w = wide(p.E, d->bf16 ? 2 : 4, {p.x, p.h, p.xo, p.y, p.pg, p.pb, p.ng, p.nb, p.gate});
  if (d->bf16) return w ? by_width<bf16_t, 8, false, Fwd>(p, st) : by_width<bf16_t, 8, true, Fwd>(p, st);
  return w ? by_width<float, 4, false, Fwd>(p, st) : by_width<float, 4, true, Fwd>(p, st);
}

extern "C" int64_t smx_norm_residual_bwd_ws_floats(int64_t T, int64_t groups, int E) {
  if (T <= 0 || groups <= 0 || T % groups || E <= 0 || E > 16384 || T > 0x7fffffffLL) return -1;
  return groups * smx_cdiv(T / groups, rows_of(T, T / groups, E)) * 5 * E;
}

extern "C" int smx_norm_residual_bwd_f32(const smx_norm_residual_desc* d, void* stream) {
  int rc = check(d, true);
  if (rc != SMX_OK) return rc;
  if (d->bf16 || (!d->gx && !d->gy) || (d->gy && !d->pre_gamma) || (d->dgate && !d->gate)) return SMX_EINVAL;
  if (d->dgate && !d->gate_accumulate && (d->dgate == d->dpre_gamma || d->dgate == d->dpre_beta || d->dgate == d->dpost_gamma || d->dgate == d->dpost_beta)) return SMX_EINVAL;
  if (((d->dpost_gamma || d->dpost_beta) && !d->post_gamma) || ((d->dpre_gamma || d->dpre_beta) && !d->pre_gamma)) return SMX_EINVAL;
  if (!d->ws || ((uintptr_t)d->ws & 15) || d->ws_floats < smx_norm_residual_bwd_ws_floats(d->T, d->groups, d->E)) return SMX_EINVAL;
  const NRP p = params(d);
  hipStream_t st = (hipStream_t)stream;
  rc = wide(p.E, 4, {p.h, p.xo, p.gx, p.gy, p.dx, p.dh, p.pg, p.pb, p.ng, p.nb, p.gate}) ? by_width<float, 4, false, Bwd>(p, st) : by_width<float, 4, true, Bwd>(p, st);
  if (rc != SMX_OK || !p.want) return rc;
  const Outs o = {{d->dpre_gamma, d->dpre_beta, d->dpost_gamma, d->dpost_beta, d->dgate}};
  bool shared = false;                               // one parameter in two places: its sums one launch after the other
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < i; ++j) shared |= o.p[i] && o.p[i] == o.p[j];
  for (int i = 0; shared && i < 4; ++i) {
    if (!o.p[i]) continue;
    Outs one = {{nullptr, nullptr, nullptr, nullptr, nullptr}};
    one.p[i] = o.p[i];
    SMX_LAUNCH(norm_residual_sum_kernel, dim3(smx_cdiv(p.E, 32), 4), dim3(1024), 0, st, (const float*)d->ws, one, p.E, (long long)d->groups * p.nblk, p.nblk, 0, 0LL);
  }
  if (shared && !d->dgate) return smx_launch_status();
  for (long long g0 = 0; g0 == 0 || (d->dgate && g0 < d->groups); g0 += 65000) {      // (a grid's y ends at 65535)
    Outs now = o;
    if (g0 || shared) now.p[0] = now.p[1] = now.p[2] = now.p[3] = nullptr;
    const long long left = d->groups - g0;
    SMX_LAUNCH(norm_residual_sum_kernel, dim3(smx_cdiv(p.E, 32), (unsigned)(d->dgate ? 4 + (left < 65000 ? left : 65000) : 4)), dim3(1024), 0, st, (const float*)d->ws, now,
               p.E, (long long)d->groups * p.nblk, p.nblk, (int)d->gate_accumulate, g0);
  }
  return smx_launch_status();
}
