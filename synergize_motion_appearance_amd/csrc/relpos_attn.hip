// Attention with a learned relative position bias by buckets (include/smx.h: smx_attention_relpos, smx_attention_relpos_bwd_f32).
//   s_ij = scale q_i . k_j + table[map[clamp(j - pos_i - map_lo)]][h],  P = softmax over the keys that are left,  o_i = sum_j P_ij v_j
//   D_i = sum_d dO_id o_id,  dS_ij = P_ij (dO_i . v_j - D_i),  dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij dO_i,  dtable[b][h] = sum of dS_ij over the pairs of bucket b
// Scores are kept in log2 units; lse_i = log2 sum_j 2^{s_ij}, +inf for a row with no key left, so that 2^{s - lse} is 0 there.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "smx.h"
#include "smx_common.h"
#include "bf16.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

struct RP {
  const void* q; const void* k; const void* v; void* o;
  const float* table; const int* map; const uint8_t* mask; const int* kv_len;
  float* lse; const float* d_o; float* dq; float* dk; float* dv; float* dtable;
  long long q_bs, k_bs, v_bs, o_bs;
  int ldq, ldk, ldv, ldo;
  int B, H, Hkv, G, L, S, dh, map_lo, map_n, nb, causal, has_start, q_start;
  float scale;
  __device__ __forceinline__ int keys(int b) const { return kv_len ? max(0, min(kv_len[b], S)) : S; }
  __device__ __forceinline__ int pos0(int n) const { return has_start ? q_start : n - L; }
  __device__ __forceinline__ int entry(int delta) const { return max(0, min(delta - map_lo, map_n - 1)); }
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

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

// one wave per query row: lane = key for the scores, lane = head column (two of them) for the output
template <typename T>
__global__ __launch_bounds__(256) void relpos_rows_kernel(RP p) {
  const int lane = threadIdx.x & 63;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (row >= (long long)p.B * p.H * p.L) return;
  const int i = (int)(row % p.L), h = (int)(row / p.L % p.H), b = (int)(row / p.L / p.H), hk = h / p.G;
  const int n = p.keys(b), pos = p.pos0(n) + i;
  const T* Q = (const T*)p.q + b * p.q_bs + (long long)i * p.ldq + h * p.dh;
  const T* K = (const T*)p.k + b * p.k_bs + hk * p.dh;
  const T* V = (const T*)p.v + b * p.v_bs + hk * p.dh;
  float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int j0 = 0; j0 < n; j0 += 64) {
    const float s = score<T>(p, Q, K, b, h, j0 + lane, n, pos);
    const float mn = fmaxf(m, wave_max(s));
    if (mn == -INFINITY) continue;
    const float al = exp2f(m - mn), e = exp2f(s - mn);
    l = l * al + wave_sum(e); a0 *= al; a1 *= al; m = mn;
    for (int t = 0; t < 64; ++t) {
      const float pt = __shfl(e, t, 64);
      if (pt == 0.f) continue;
      const T* vr = V + (long long)(j0 + t) * p.ldv;
      if (lane < p.dh) a0 += pt * St<T>::ld(vr + lane);
      if (lane + 64 < p.dh) a1 += pt * St<T>::ld(vr + lane + 64);
    }
  }
  T* O = (T*)p.o + b * p.o_bs + (long long)i * p.ldo + h * p.dh;
  const float il = l > 0.f ? 1.f / l : 0.f;
  if (lane < p.dh) St<T>::st(O + lane, a0 * il);
  if (lane + 64 < p.dh) St<T>::st(O + lane + 64, a1 * il);
  if (p.lse && lane == 0) p.lse[row] = l > 0.f ? m + log2f(l) : INFINITY;
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

bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// what both entry points ask of their arguments; fills RP
int check(const smx_relpos_desc* d, RP& p, bool bwd) {
  if (!d || !d->q || !d->k || !d->v || !d->o || !d->table || !d->map) return SMX_EINVAL;
  if (d->B <= 0 || d->H <= 0 || d->Hkv <= 0 || d->H % d->Hkv || d->L <= 0 || d->S <= 0 || d->dh <= 0 || d->dh % 4 || d->dh > 128) return SMX_EINVAL;
  if ((long long)d->H * d->dh > (1 << 20) || (long long)d->B * d->H > (1 << 24) || d->L > (1 << 30) || d->S > (1 << 30)) return SMX_EINVAL;
  if (d->map_n <= 0 || d->map_n > 2049 || d->map_lo > 0 || d->map_lo + d->map_n <= 0 || d->num_buckets <= 0 || d->num_buckets > 4096) return SMX_EINVAL;
  if (d->has_q_start && (d->q_start > (1 << 30) || d->q_start < -(1 << 30))) return SMX_EINVAL;
  if (!(d->scale == d->scale) || (d->bf16 != 0 && d->bf16 != 1) || (bwd && d->bf16)) return SMX_EINVAL;
  if (d->ldq < d->H * d->dh || d->ldk < d->Hkv * d->dh || d->ldv < d->Hkv * d->dh || d->ldo < d->H * d->dh) return SMX_EINVAL;
  if ((d->ldq | d->ldk | d->ldv | d->ldo) % 4 || d->q_bs < 0 || d->k_bs < 0 || d->v_bs < 0 || d->o_bs < 0) return SMX_EINVAL;
  if (d->q_bs % 4 || d->k_bs % 4 || d->v_bs % 4 || d->o_bs % 4) return SMX_EINVAL;
  const int el = 4 * (d->bf16 ? 2 : 4);
  if (!aligned(d->q, el) || !aligned(d->k, el) || !aligned(d->v, el) || !aligned(d->o, el)) return SMX_EINVAL;
  if (bwd && (!d->d_o || !d->dq || !d->dk || !d->dv || !d->dtable || !d->lse || d->ldo != d->H * d->dh || d->o_bs != (int64_t)d->L * d->ldo)) return SMX_EINVAL;
  if (bwd && (!aligned(d->d_o, 16) || !aligned(d->dq, 16) || !aligned(d->dk, 16) || !aligned(d->dv, 16))) return SMX_EINVAL;
  p.q = d->q; p.k = d->k; p.v = d->v; p.o = d->o; p.table = d->table; p.map = d->map; p.mask = d->mask; p.kv_len = d->kv_len;
  p.lse = d->lse; p.d_o = d->d_o; p.dq = d->dq; p.dk = d->dk; p.dv = d->dv; p.dtable = d->dtable;
  p.q_bs = d->q_bs; p.k_bs = d->k_bs; p.v_bs = d->v_bs; p.o_bs = d->o_bs; p.ldq = d->ldq; p.ldk = d->ldk; p.ldv = d->ldv; p.ldo = d->ldo;
  p.B = d->B; p.H = d->H; p.Hkv = d->Hkv; p.G = d->H / d->Hkv; p.L = d->L; p.S = d->S; p.dh = d->dh;
  p.map_lo = d->map_lo; p.map_n = d->map_n; p.nb = d->num_buckets; p.causal = d->causal; p.has_start = d->has_q_start; p.q_start = d->q_start;
  p.scale = d->scale;
  return SMX_OK;
}

}  // namespace

extern "C" int64_t smx_attention_relpos_ws_bytes(const smx_relpos_desc* d) {
  RP p;
  return check(d, p, false) == SMX_OK ? 0 : -1;
}

extern "C" int smx_attention_relpos(const smx_relpos_desc* d, void* stream) {
  RP p;
  const int rc = check(d, p, false);
  if (rc != SMX_OK) return rc;
  const long long blocks = ((long long)p.B * p.H * p.L + 3) / 4;
  if (blocks > 0x7fffffffLL) return SMX_EINVAL;
  if (d->bf16) SMX_LAUNCH(relpos_rows_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  else SMX_LAUNCH(relpos_rows_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  return smx_launch_status();
}

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
