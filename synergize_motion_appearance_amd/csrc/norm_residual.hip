// The norms around a block, its gate and residual (include/smx.h: smx_norm_residual, smx_norm_residual_bwd_f32).
//   n = Norm(h),  x' = rs x + g n,  y = Norm(x')
// Backward, with c the gradient of x' (its own plus what comes back through y), hat = (v - mean) r the normalised rows:
//   NormBwd(g; v) = r (gamma g - mean(gamma g) - hat mean(gamma g hat))       (rms: without the middle term, mean = 0)
//   c = gx + NormBwd(gy; x'),  dx = rs c,  dn = g c,  dh = NormBwd(dn; h),  dgate = sum n c,  dgamma = sum g hat,  dbeta = sum g
// Bound by memory: forward reads x, h and writes x', y; backward reads x', h, gx, gy and writes dx, dh.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "smx.h"
#include "smx_common.h"
#include "bf16.h"

namespace {

struct NRP {
  const void* x; const void* h; void* xo; void* y;
  const float* pg; const float* pb; const float* ng; const float* nb; const float* gate;
  const float* gx; const float* gy; float* dx; float* dh; float* part;
  long long T, per; int E, rms, nblk, rows;      // per: tokens of a gate row; nblk blocks of `rows` tokens walk each gate row's tokens
  float rs, eps;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// mean and 1 / sqrt(var + eps) of a row held as v[k] at columns threadIdx.x + 256 k
template <int N>
__device__ __forceinline__ void row_stats(const float (&v)[N], int E, int rms, float eps, float* red, float& mean, float& r) {
  float s = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int k = 0; k < N; ++k) s += v[k];
    mean = block_sum(s, red) / E;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) { const float d = (int)threadIdx.x + 256 * k < E ? v[k] - mean : 0.f; q += d * d; }
  r = 1.f / sqrtf(block_sum(q, red) / E + eps);
}

template <typename TS, int N>
__global__ __launch_bounds__(256) void norm_residual_kernel(NRP p) {
  __shared__ float red[4];
  const long long t = blockIdx.x, at = t * p.E;
  const float* gate = p.gate ? p.gate + t / p.per * p.E : nullptr;
  float v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) { const int c = threadIdx.x + 256 * k; v[k] = c < p.E ? St<TS>::ld((const TS*)p.h + at + c) : 0.f; }
  float mean, r;
  if (p.pg) {
    row_stats<N>(v, p.E, p.rms, p.eps, red, mean, r);
#pragma unroll
    for (int k = 0; k < N; ++k) { const int c = threadIdx.x + 256 * k; if (c < p.E) v[k] = (v[k] - mean) * r * p.pg[c] + (p.pb ? p.pb[c] : 0.f); }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = threadIdx.x + 256 * k;
    if (c < p.E) {
      TS w;
      St<TS>::st(&w, p.rs * St<TS>::ld((const TS*)p.x + at + c) + (gate ? gate[c] : 1.f) * v[k]);
      ((TS*)p.xo)[at + c] = w;
      v[k] = St<TS>::ld(&w);                       // y is the norm of what is stored
    }
  }
  if (!p.y) return;
  row_stats<N>(v, p.E, p.rms, p.eps, red, mean, r);
#pragma unroll
  for (int k = 0; k < N; ++k) { const int c = threadIdx.x + 256 * k; if (c < p.E) St<TS>::st((TS*)p.y + at + c, (v[k] - mean) * r * p.ng[c] + (p.nb ? p.nb[c] : 0.f)); }
}

// a block walks `rows` tokens of one gate row, keeping its columns' parameter sums in registers; part [groups][nblk][5][E]:
// dpre gamma, dpre beta, dpost gamma, dpost beta, dgate
template <int N>
__global__ __launch_bounds__(256) void norm_residual_bwd_kernel(NRP p) {
  __shared__ float red[4];
  const long long g = blockIdx.x / p.nblk, blk = blockIdx.x - g * p.nblk;
  const float* gate = p.gate ? p.gate + g * p.E : nullptr;
  float a[5][N];
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) a[i][k] = 0.f;
  const long long t1 = g * p.per + min(p.per, (blk + 1) * (long long)p.rows);
  for (long long t = g * p.per + blk * p.rows; t < t1; ++t) {
    const long long at = t * p.E;
    float v[N], c[N];
    float mean = 0.f, r = 1.f;
#pragma unroll
    for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; c[k] = e < p.E && p.gx ? p.gx[at + e] : 0.f; }
    if (p.gy) {
#pragma unroll
      for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; v[k] = e < p.E ? ((const float*)p.xo)[at + e] : 0.f; }
      row_stats<N>(v, p.E, p.rms, p.eps, red, mean, r);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int e = threadIdx.x + 256 * k;
        if (e < p.E) {
          const float gy = p.gy[at + e], hat = (v[k] - mean) * r, gw = gy * p.ng[e];
          a[0][k] += gy * hat; a[1][k] += gy;
          s1 += gw; s2 += gw * hat;
        }
      }
      s1 = p.rms ? 0.f : block_sum(s1, red) / p.E;
      s2 = block_sum(s2, red) / p.E;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int e = threadIdx.x + 256 * k;
        if (e < p.E) c[k] += r * (p.gy[at + e] * p.ng[e] - s1 - (v[k] - mean) * r * s2);
      }
    }
    if (p.dx) {
#pragma unroll
      for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; if (e < p.E) p.dx[at + e] = p.rs * c[k]; }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; v[k] = e < p.E ? ((const float*)p.h)[at + e] : 0.f; }
    if (!p.pg) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int e = threadIdx.x + 256 * k;
        if (e < p.E) { a[4][k] += v[k] * c[k]; if (p.dh) p.dh[at + e] = (gate ? gate[e] : 1.f) * c[k]; }
      }
      continue;
    }
    row_stats<N>(v, p.E, p.rms, p.eps, red, mean, r);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = threadIdx.x + 256 * k;
      if (e < p.E) {
        const float hat = (v[k] - mean) * r, dn = (gate ? gate[e] : 1.f) * c[k], gw = dn * p.pg[e];
        a[4][k] += c[k] * (hat * p.pg[e] + (p.pb ? p.pb[e] : 0.f));
        a[2][k] += dn * hat; a[3][k] += dn;
        s1 += gw; s2 += gw * hat;
        c[k] = gw; v[k] = hat;
      }
    }
    s1 = p.rms ? 0.f : block_sum(s1, red) / p.E;
    s2 = block_sum(s2, red) / p.E;
#pragma unroll
    for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; if (e < p.E && p.dh) p.dh[at + e] = r * (c[k] - s1 - v[k] * s2); }
  }
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) { const int e = threadIdx.x + 256 * k; if (e < p.E) p.part[((long long)blockIdx.x * 5 + i) * p.E + e] = a[i][k]; }
}

struct Outs { float* p[5]; };

// the blocks' sums in block order: grid.y 0..3 the parameters (over all blocks), 4 + g the gate row g (over its own)
__global__ __launch_bounds__(256) void norm_residual_sum_kernel(const float* __restrict__ part, Outs o, int E, long long nall, int nblk, int gate_acc) {
  const int e = blockIdx.x * 256 + threadIdx.x, which = min((int)blockIdx.y, 4);
  float* out = o.p[which];
  if (e >= E || !out) return;
  const long long g = (int)blockIdx.y - which, n0 = which < 4 ? 0 : g * nblk, n1 = which < 4 ? nall : n0 + nblk;
  float s = 0.f;
  for (long long n = n0; n < n1; ++n) s += part[(n * 5 + which) * E + e];
  if (which < 4) out[e] += s;
  else out[g * E + e] = gate_acc ? out[g * E + e] + s : s;
}

// tokens a block walks: enough blocks to fill the chip
int rows_of(long long T, long long per) {
  long long r = T / 1024;
  if (r < 1) r = 1;
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
  p.rows = rows_of(d->T, p.per); p.nblk = smx_cdiv(p.per, p.rows); p.rs = d->res_scale; p.eps = d->eps;
  return p;
}

template <typename TS>
int forward(const NRP& p, hipStream_t st) {
  const dim3 grid((unsigned)p.T), block(256);
  if (p.E <= 256) SMX_LAUNCH((norm_residual_kernel<TS, 1>), grid, block, 0, st, p);
  else if (p.E <= 1024) SMX_LAUNCH((norm_residual_kernel<TS, 4>), grid, block, 0, st, p);
  else if (p.E <= 4096) SMX_LAUNCH((norm_residual_kernel<TS, 16>), grid, block, 0, st, p);
  else SMX_LAUNCH((norm_residual_kernel<TS, 64>), grid, block, 0, st, p);
  return smx_launch_status();
}

}  // namespace

extern "C" int smx_norm_residual(const smx_norm_residual_desc* d, void* stream) {
  const int rc = check(d, false);
  if (rc != SMX_OK) return rc;
  const NRP p = params(d);
  return d->bf16 ? forward<bf16_t>(p, (hipStream_t)stream) : forward<float>(p, (hipStream_t)stream);
}

extern "C" int64_t smx_norm_residual_bwd_ws_floats(int64_t T, int64_t groups, int E) {
  if (T <= 0 || groups <= 0 || T % groups || E <= 0 || E > 16384 || T > 0x7fffffffLL) return -1;
  return groups * smx_cdiv(T / groups, rows_of(T, T / groups)) * 5 * E;
}

extern "C" int smx_norm_residual_bwd_f32(const smx_norm_residual_desc* d, void* stream) {
  const int rc = check(d, true);
  if (rc != SMX_OK) return rc;
  if (d->bf16 || (!d->gx && !d->gy) || (d->gy && !d->pre_gamma) || (d->dgate && !d->gate) || (d->groups > 65531 && d->dgate)) return SMX_EINVAL;
  if (((d->dpost_gamma || d->dpost_beta) && !d->post_gamma) || ((d->dpre_gamma || d->dpre_beta) && !d->pre_gamma)) return SMX_EINVAL;
  if (!d->ws || ((uintptr_t)d->ws & 15) || d->ws_floats < smx_norm_residual_bwd_ws_floats(d->T, d->groups, d->E)) return SMX_EINVAL;
  const NRP p = params(d);
  const long long nall = d->groups * p.nblk;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)nall), block(256);
  if (p.E <= 256) SMX_LAUNCH(norm_residual_bwd_kernel<1>, grid, block, 0, st, p);
  else if (p.E <= 1024) SMX_LAUNCH(norm_residual_bwd_kernel<4>, grid, block, 0, st, p);
  else if (p.E <= 4096) SMX_LAUNCH(norm_residual_bwd_kernel<16>, grid, block, 0, st, p);
  else SMX_LAUNCH(norm_residual_bwd_kernel<64>, grid, block, 0, st, p);
  const Outs o = {{d->dpre_gamma, d->dpre_beta, d->dpost_gamma, d->dpost_beta, d->dgate}};
  SMX_LAUNCH(norm_residual_sum_kernel, dim3(smx_cdiv(p.E, 256), (unsigned)(d->dgate ? 4 + d->groups : 4)), block, 0, st, (const float*)d->ws, o, p.E, nall,
             p.nblk, (int)d->gate_accumulate);
  return smx_launch_status();
}
