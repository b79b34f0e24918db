// Attention with a learned relative position bias by buckets, backward (include/smx.h: smx_attention_relpos_bwd_f32):
//   D_i = sum_d dO_id o_id,  dS_ij = P_ij (dO_i . v_j - D_i),  dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij dO_i,  dtable[b][h] = sum of dS_ij over the pairs of bucket b
// lse_i = log2 sum_j 2^{s_ij}, +inf for a row with no key left, so that 2^{s - lse} is 0 there.
#include "relpos.h"

namespace {
using namespace relpos;

// the log2-unit score of one pair, -inf where the key is not left
template <typename T>
__device__ __forceinline__ float score(const RP& p, const T* Q, const T* K, int b, int h, int j, int n, int pos) {
  const int delta = j - pos;
  if (j >= n || (p.causal && delta > 0) || (p.mask && p.mask[(long long)b * p.S + j])) return -INFINITY;
  const T* kr = K + (long long)j * p.ldk;
  float a = 0.f;
  for (int d = 0; d < p.dh; d += 4) {
    const float4 x = St<T>::ld4(Q + d), y = St<T>::ld4(kr + d);
    a += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
  }
  return (a * p.scale + p.table[(long long)p.map[p.entry(delta)] * p.H + h]) * LOG2E;
}

__device__ __forceinline__ float dot(const float* a, const float* b, int n) {
  float s = 0.f;
  for (int d = 0; d < n; d += 4) {
    const float4 x = St<float>::ld4(a + d), y = St<float>::ld4(b + d);
    s += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
  }
  return s;
}

// dq: one wave per query row; the row's D goes to `dd` for the other two kernels
__global__ __launch_bounds__(256) void relpos_bwd_q_kernel(RP p, float* __restrict__ dd) {
  const int lane = threadIdx.x & 63;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (row >= (long long)p.B * p.H * p.L) return;
  const int i = (int)(row % p.L), h = (int)(row / p.L % p.H), b = (int)(row / p.L / p.H), hk = h / p.G;
  const int n = p.keys(b), pos = p.pos0(n) + i;
  const float* Q = (const float*)p.q + b * p.q_bs + (long long)i * p.ldq + h * p.dh;
  const float* K = (const float*)p.k + b * p.k_bs + hk * p.dh;
  const float* V = (const float*)p.v + b * p.v_bs + hk * p.dh;
  const long long od = ((long long)b * p.L + i) * p.H * p.dh + h * p.dh;
  const float D = dot(p.d_o + od, (const float*)p.o + od, p.dh), lse = p.lse[row];
  float a0 = 0.f, a1 = 0.f;
  for (int j0 = 0; j0 < n; j0 += 64) {
    const float s = score<float>(p, Q, K, b, h, j0 + lane, n, pos);
    const float ds = s == -INFINITY ? 0.f : exp2f(s - lse) * (dot(p.d_o + od, V + (long long)(j0 + lane) * p.ldv, p.dh) - D);
    for (int t = 0; t < 64; ++t) {
      const float w = __shfl(ds, t, 64);
      if (w == 0.f) continue;
      const float* kr = K + (long long)(j0 + t) * p.ldk;
      if (lane < p.dh) a0 += w * kr[lane];
      if (lane + 64 < p.dh) a1 += w * kr[lane + 64];
    }
  }
  if (lane < p.dh) p.dq[od + lane] = a0 * p.scale;
  if (lane + 64 < p.dh) p.dq[od + lane + 64] = a1 * p.scale;
  if (lane == 0) dd[row] = D;
}

// dk, dv: one wave per key row, over the queries of the heads that share it
__global__ __launch_bounds__(256) void relpos_bwd_kv_kernel(RP p, const float* __restrict__ dd) {
  const int lane = threadIdx.x & 63;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (row >= (long long)p.B * p.Hkv * p.S) return;
  const int j = (int)(row % p.S), hk = (int)(row / p.S % p.Hkv), b = (int)(row / p.S / p.Hkv);
  const int n = p.keys(b);
  const float* K = (const float*)p.k + b * p.k_bs + hk * p.dh;
  const float* V = (const float*)p.v + b * p.v_bs + hk * p.dh;
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  if (j < n)
    for (int h = hk * p.G; h < (hk + 1) * p.G; ++h)
      for (int i0 = 0; i0 < p.L; i0 += 64) {
        const int i = i0 + lane;
        float pij = 0.f, ds = 0.f;
        if (i < p.L) {
          const long long r = ((long long)b * p.H + h) * p.L + i;
          const float s = score<float>(p, (const float*)p.q + b * p.q_bs + (long long)i * p.ldq + h * p.dh, K, b, h, j, n, p.pos0(n) + i);
          if (s != -INFINITY) {
            pij = exp2f(s - p.lse[r]);
            ds = pij * (dot(p.d_o + ((long long)b * p.L + i) * p.H * p.dh + h * p.dh, V + (long long)j * p.ldv, p.dh) - dd[r]);
          }
        }
        for (int t = 0; t < 64; ++t) {
          const float pt = __shfl(pij, t, 64), dt = __shfl(ds, t, 64);
          if (pt == 0.f) continue;
          const float* qr = (const float*)p.q + b * p.q_bs + (long long)(i0 + t) * p.ldq + h * p.dh;
          const float* gr = p.d_o + ((long long)b * p.L + i0 + t) * p.H * p.dh + h * p.dh;
          if (lane < p.dh) { k0 += dt * qr[lane]; v0 += pt * gr[lane]; }
          if (lane + 64 < p.dh) { k1 += dt * qr[lane + 64]; v1 += pt * gr[lane + 64]; }
        }
      }
  const long long od = ((long long)b * p.S + j) * p.Hkv * p.dh + hk * p.dh;
  if (lane < p.dh) { p.dk[od + lane] = k0 * p.scale; p.dv[od + lane] = v0; }
  if (lane + 64 < p.dh) { p.dk[od + lane + 64] = k1 * p.scale; p.dv[od + lane + 64] = v1; }
}

// sums of dS per (map entry, head): one block per pair of them, threads over the samples' queries whose key of that distance exists
// (the two ends of the map stand for all distances beyond them)
__global__ __launch_bounds__(256) void relpos_bwd_entry_kernel(RP p, const float* __restrict__ dd, float* __restrict__ part) {
  __shared__ float red[256];
  const int e = blockIdx.x, h = blockIdx.y, hk = h / p.G;
  float a = 0.f;
  for (int b = 0; b < p.B; ++b) {
    const int n = p.keys(b);
    const float* K = (const float*)p.k + b * p.k_bs + hk * p.dh;
    const float* V = (const float*)p.v + b * p.v_bs + hk * p.dh;
    for (int i = threadIdx.x; i < p.L; i += 256) {
      const int pos = p.pos0(n) + i;
      const long long r = ((long long)b * p.H + h) * p.L + i;
      int j0 = pos + p.map_lo + e, j1 = j0 + 1;
      if (e == 0) j0 = 0;
      if (e == p.map_n - 1) j1 = n;
      for (int j = max(j0, 0); j < min(j1, n); ++j) {
        const float s = score<float>(p, (const float*)p.q + b * p.q_bs + (long long)i * p.ldq + h * p.dh, K, b, h, j, n, pos);
        if (s != -INFINITY)
          a += exp2f(s - p.lse[r]) * (dot(p.d_o + ((long long)b * p.L + i) * p.H * p.dh + h * p.dh, V + (long long)j * p.ldv, p.dh) - dd[r]);
      }
    }
  }
  red[threadIdx.x] = a;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[(long long)h * p.map_n + e] = red[0];
}

// dtable[bucket][h] += the entries of that bucket
__global__ __launch_bounds__(256) void relpos_bwd_table_kernel(RP p, const float* __restrict__ part) {
  const int at = blockIdx.x * 256 + threadIdx.x;
  if (at >= p.nb * p.H) return;
  const int bucket = at / p.H, h = at - bucket * p.H;
  float a = 0.f;
  for (int e = 0; e < p.map_n; ++e)
    if (p.map[e] == bucket) a += part[(long long)h * p.map_n + e];
  p.dtable[at] += a;
}

}  // namespace

extern "C" int64_t smx_attention_relpos_bwd_ws_bytes(const smx_relpos_desc* d) {
  RP p;
  if (check(d, p, true) != SMX_OK) return -1;
  return 4 * ((int64_t)p.B * p.H * p.L + (int64_t)p.H * p.map_n);
}

extern "C" int smx_attention_relpos_bwd_f32(const smx_relpos_desc* d, void* stream) {
  RP p;
  const int rc = check(d, p, true);
  if (rc != SMX_OK) return rc;
  const long long qb = ((long long)p.B * p.H * p.L + 3) / 4, kb = ((long long)p.B * p.Hkv * p.S + 3) / 4;
  if (!d->ws || !aligned(d->ws, 16) || d->ws_bytes < smx_attention_relpos_bwd_ws_bytes(d) || qb > 0x7fffffffLL || kb > 0x7fffffffLL || p.H > 65535) return SMX_EINVAL;
  float* dd = (float*)d->ws;
  float* part = dd + (int64_t)p.B * p.H * p.L;
  hipStream_t st = (hipStream_t)stream;
  SMX_LAUNCH(relpos_bwd_q_kernel, dim3((unsigned)qb), dim3(256), 0, st, p, dd);
  SMX_LAUNCH(relpos_bwd_kv_kernel, dim3((unsigned)kb), dim3(256), 0, st, p, (const float*)dd);
  SMX_LAUNCH(relpos_bwd_entry_kernel, dim3(p.map_n, p.H), dim3(256), 0, st, p, (const float*)dd, part);
  SMX_LAUNCH(relpos_bwd_table_kernel, dim3(smx_cdiv((long long)p.nb * p.H, 256)), dim3(256), 0, st, p, (const float*)part);
  return smx_launch_status();
}
