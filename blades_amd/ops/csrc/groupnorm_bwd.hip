// Backward pass of the group normalisation: see groupnorm.h.
#include "groupnorm.h"

namespace {
using namespace groupnorm;

// g of one vector: gy behind the activation.  The gate byte or z, computed again, decides; z takes the residual again
// where the activation is smooth.
template <typename T, int VEC, int AK>
__device__ __forceinline__ void slope_vector(const Pack<T, VEC>& gy, const float (&xh)[VEC], size_t o, const T* res,
                                             const unsigned char* gate, const float (&ga)[VEC], const float (&be)[VEC], int act,
                                             float (&g)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) g[j] = to_f(gy.e[j]);
  if (AK <= 0) {
    if (act == 0) return;
  }
  if (AK <= 0 && gate != nullptr) {
    const unsigned m = gate[o / VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = (m >> j) & 1u ? g[j] : 0.f;
    return;
  }
  float z[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) z[j] = fmaf(xh[j], ga[j], be[j]);
  if (AK != 0 && res != nullptr) {
    const Pack<T, VEC> rv = *reinterpret_cast<const Pack<T, VEC>*>(res + o);
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[j] += to_f(rv.e[j]);
  }
  if (AK == 0 || (AK < 0 && act == 1)) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = z[j] <= 0.f ? 0.f : g[j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] *= act_slope<AK, sizeof(T) == 4>(z[j], act);
  }
}

template <typename T, int VEC, int NM>
__device__ __forceinline__ void bwd_vector(const float (&g)[VEC], const float (&xh)[VEC], size_t o, T* dx, T* dres,
                                           const float (&rs)[NM], const float (&ga)[VEC], const float (&m1)[NM],
                                           const float (&m2)[NM], bool through) {
  typedef Pack<T, VEC> V;
  if (dx != nullptr) {
    V w;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int m = NM == 1 ? 0 : j;
      from_f(rs[m] * (fmaf(g[j], ga[j], -m1[m]) - xh[j] * m2[m]), w.e[j]);
    }
    store_out(dx + o, w, through);
  }
  if (dres != nullptr) {
    V w;
#pragma unroll
    for (int j = 0; j < VEC; ++j) from_f(g[j], w.e[j]);
    store_out(dres + o, w, through);
  }
}

// Whole samples.  sums [N][C]: (A, B) of every sample and channel.
template <typename T, int VEC, int R, int NM, int AK>
__global__ __launch_bounds__(MAX_THREADS) void gn_bwd_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                                    const T* __restrict__ gy,
                                                                    const unsigned char* __restrict__ gate,
                                                                    const float* __restrict__ gamma,
                                                                    const float* __restrict__ beta,
                                                                    const float* __restrict__ mean,
                                                                    const float* __restrict__ rstd, T* __restrict__ dx,
                                                                    T* __restrict__ dres, float2* __restrict__ sums) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  const Place<VEC, NM> w(q);
  if (!w.here) return;
  V xr[R], gr[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.active && w.row + i * q.rows < w.pn) {
      xr[i] = *reinterpret_cast<const V*>(x + w.at + i * w.step);
      gr[i] = *reinterpret_cast<const V*>(gy + w.at + i * w.step);
    }
  float *ch = lds, *gam = ch + 2 * q.S, *stat = gam + q.S, *gsum = stat + 2 * w.Gs, *red = gsum + 2 * w.Gs;
  for (int c = threadIdx.x; c < q.S; c += blockDim.x)
    gam[c] = gamma ? gamma[w.client * q.gstride + w.slab * q.S + c] : 1.f;
  for (int g = threadIdx.x; g < w.Gs; g += blockDim.x) {
    const size_t o = (size_t)w.n * w.G + w.slab * w.Gs + g;
    stat[g] = mean[o]; stat[w.Gs + g] = rstd[o];
  }
  float mu[NM], rs[NM], m1[NM], m2[NM], ga[VEC], be[VEC];
  if (w.active) load_floats<VEC>(beta ? beta + w.client * q.bstride + w.c0 : nullptr, 0.f, be);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NM; ++j) {
    mu[j] = w.active ? stat[w.g[j]] : 0.f;
    rs[j] = w.active ? stat[w.Gs + w.g[j]] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) ga[j] = w.active ? gam[w.l * VEC + j] : 0.f;
  float v[2][VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[0][j] = v[1][j] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.active && w.row + i * q.rows < w.pn) {
      float g[VEC], xh[VEC];
      normed<T, VEC, NM>(xr[i], mu, rs, xh);
      slope_vector<T, VEC, AK>(gr[i], xh, w.at + i * w.step, res, gate, ga, be, q.act, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[0][j] += g[j];
        v[1][j] = fmaf(g[j], xh[j], v[1][j]);
      }
      if (sizeof(T) == 4) {  // (fp32: g replaces gy in its registers; a 16-bit type would round it)
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(g[j], gr[i].e[j]);
      }
    }
  slab_sums<2, VEC>(v, 1, q.S, q.tw_ch, q, w.l, w.row, w.active, red, ch);  // ch[0..S): A, ch[S..2S): B
  for (int c = threadIdx.x; c < q.S; c += blockDim.x)
    sums[(size_t)w.n * q.C + w.slab * q.S + c] = make_float2(ch[c], ch[q.S + c]);
  const int tw = q.tw_gr, e0 = threadIdx.x & (tw - 1);
  for (int g = threadIdx.x / tw; g < 2 * w.Gs; g += blockDim.x / tw) {
    const int k = g >= w.Gs, cb = (g - k * w.Gs) * q.D;
    float a = 0.f;
    for (int e = e0; e < q.D; e += tw) a = fmaf(gam[cb + e], ch[k * q.S + cb + e], a);
    for (int o = tw >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if (e0 == 0) gsum[g] = a;
  }
  __syncthreads();
  if (!w.active || (dx == nullptr && dres == nullptr)) return;
  const float inv = 1.f / ((float)q.P * (float)q.D);
#pragma unroll
  for (int j = 0; j < NM; ++j) { m1[j] = gsum[w.g[j]] * inv; m2[j] = gsum[w.Gs + w.g[j]] * inv; }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.row + i * q.rows < w.pn) {
      const size_t o = w.at + i * w.step;
      float g[VEC], xh[VEC];
      normed<T, VEC, NM>(xr[i], mu, rs, xh);
      if (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = to_f(gr[i].e[j]);
      } else {
        slope_vector<T, VEC, AK>(gr[i], xh, o, res, gate, ga, be, q.act, g);
      }
      bwd_vector<T, VEC, NM>(g, xh, o, dx, dres, rs, ga, m1, m2, q.through);
    }
}

// Pixel chunks.  APPLY false: part [N][nchunk][C], (A, B) of a chunk.  true: the second sweep, with the joined means [N][G].
template <typename T, int VEC, int NM, int AK, bool APPLY>
__global__ __launch_bounds__(MAX_THREADS) void gn_bwd_chunk_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                           const T* __restrict__ gy, const unsigned char* __restrict__ gate,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           T* __restrict__ dx, T* __restrict__ dres, float2* __restrict__ part,
                                                           const float2* __restrict__ means) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  const Place<VEC, NM> w(q);
  if (!w.here) return;
  float mu[NM], rs[NM], m1[NM], m2[NM], ga[VEC], be[VEC], v[2][VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[0][j] = v[1][j] = 0.f;
  if (w.active) {
#pragma unroll
    for (int j = 0; j < NM; ++j) {
      const size_t o = (size_t)w.n * w.G + w.slab * w.Gs + w.g[j];
      mu[j] = mean[o]; rs[j] = rstd[o];
      if (APPLY) { const float2 m = means[o]; m1[j] = m.x; m2[j] = m.y; }
    }
    load_floats<VEC>(gamma ? gamma + w.client * q.gstride + w.c0 : nullptr, 1.f, ga);
    load_floats<VEC>(beta ? beta + w.client * q.bstride + w.c0 : nullptr, 0.f, be);
    for (int p = w.row; p < w.pn; p += BLOCK * q.rows) {
      V xr[BLOCK], gr[BLOCK];
      const size_t o = w.at + (size_t)(p - w.row) * q.C;
#pragma unroll
      for (int i = 0; i < BLOCK; ++i)
        if (p + i * q.rows < w.pn) {
          xr[i] = *reinterpret_cast<const V*>(x + o + i * w.step);
          gr[i] = *reinterpret_cast<const V*>(gy + o + i * w.step);
        }
#pragma unroll
      for (int i = 0; i < BLOCK; ++i)
        if (p + i * q.rows < w.pn) {
          float g[VEC], xh[VEC];
          normed<T, VEC, NM>(xr[i], mu, rs, xh);
          slope_vector<T, VEC, AK>(gr[i], xh, o + i * w.step, res, gate, ga, be, q.act, g);
          if (APPLY) {
            bwd_vector<T, VEC, NM>(g, xh, o + i * w.step, dx, dres, rs, ga, m1, m2, q.through);
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              v[0][j] += g[j];
              v[1][j] = fmaf(g[j], xh[j], v[1][j]);
            }
          }
        }
    }
  }
  if (APPLY) return;
  float *ch = lds, *red = ch + 2 * q.S;
  slab_sums<2, VEC>(v, 1, q.S, q.tw_ch, q, w.l, w.row, w.active, red, ch);
  for (int c = threadIdx.x; c < q.S; c += blockDim.x)
    part[((size_t)w.n * q.nchunk + w.chunk) * q.C + w.slab * q.S + c] = make_float2(ch[c], ch[q.S + c]);
}

// The group means of the second sweep from the chunks' (A, B): one workgroup per (sample, group), fixed order.
__global__ __launch_bounds__(256) void gn_bwd_means_kernel(const float2* __restrict__ part, int n0, int C, int D, int P, int nchunk,
                                                           int per_client, const float* __restrict__ gamma, long gstride,
                                                           float2* __restrict__ means) {
  __shared__ double red[4][2];
  const int G = C / D, n = blockIdx.x / G, g = blockIdx.x - n * G;
  const float* gam = gamma ? gamma + ((n0 + n) / per_client) * gstride + g * D : nullptr;
  const float2* p = part + (size_t)n * nchunk * C + g * D;
  double a = 0.0, b = 0.0;
  for (long j = threadIdx.x; j < (long)nchunk * D; j += 256) {
    const long k = j / D;
    const int d = (int)(j - k * D);
    const float w = gam ? gam[d] : 1.f;
    const float2 e = p[k * C + d];
    a += (double)w * e.x; b += (double)w * e.y;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = a; red[threadIdx.x >> 6][1] = b; }
  __syncthreads();
  const double inv = 1.0 / ((double)P * D);
  if (threadIdx.x == 0)
    means[blockIdx.x] = make_float2((float)((red[0][0] + red[1][0] + red[2][0] + red[3][0]) * inv),
                                    (float)((red[0][1] + red[1][1] + red[2][1] + red[3][1]) * inv));
}

// dgamma / dbeta of a client: the (A, B) of its `per_client` rows (samples, or samples' chunks), 8 channels x 128 rows of
// threads a workgroup, fixed order (two channels x 512 rows, for few channels, are no faster: 6.4 us against 6.3 for 2064 rows
// of 64, 12 against 7 for 2048 rows of 512)
constexpr int AFF_THREADS = 1024, CH = 8;
__global__ __launch_bounds__(AFF_THREADS) void gn_affine_kernel(const float2* __restrict__ sums, int per_client, int C,
                                                                const float* __restrict__ coef, float* __restrict__ dg,
                                                                float* __restrict__ db, long ld, int accumulate) {
  constexpr int ROWS = AFF_THREADS / CH;
  __shared__ double red[ROWS][CH][2];
  const int chl = threadIdx.x % CH, r0 = threadIdx.x / CH, groups = (C + CH - 1) / CH;
  const int k = blockIdx.x / groups, ch = (blockIdx.x - k * groups) * CH + chl;
  double a = 0.0, b = 0.0;
  if (ch < C) {
    const float2* p = sums + (size_t)k * per_client * C + ch;
#pragma unroll 4
    for (int r = r0; r < per_client; r += ROWS) {
      const float2 e = p[(size_t)r * C];
      a += (double)e.x; b += (double)e.y;
    }
  }
  red[r0][chl][0] = a; red[r0][chl][1] = b;
  for (int o = ROWS / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (r0 < o) { red[r0][chl][0] += red[r0 + o][chl][0]; red[r0][chl][1] += red[r0 + o][chl][1]; }
  }
  if (r0 != 0 || ch >= C) return;
  const float s = coef ? coef[k] : 1.f;
  const float vg = s * (float)red[0][chl][1], vb = s * (float)red[0][chl][0];
  if (dg != nullptr) { float* p = dg + k * ld + ch; *p = accumulate ? *p + vg : vg; }
  if (db != nullptr) { float* p = db + k * ld + ch; *p = accumulate ? *p + vb : vb; }
}

template <typename T, int VEC, int NM, int AK>
int backward_t(const Plan& pl, const void* x, const void* res, const void* gy, const unsigned char* gate, const float* gamma,
               const float* beta, const float* mean, const float* rstd, void* dx, void* dres, float* ws, hipStream_t st) {
  const Geo& q = pl.q;
  const int G = q.C / q.D, N = q.N;
  float2* sums = (float2*)ws;                                         // [N][nchunk][C]
  float2* means = sums + (size_t)N * q.nchunk * q.C;                  // [piece][G], split plans alone
  const size_t per = (size_t)q.P * q.C;
  for (long n0 = 0; n0 < N; n0 += pl.piece) {
    Geo s = q;
    s.N = (int)(N - n0 < pl.piece ? N - n0 : pl.piece);
    s.first = (int)n0;
    const T *xp = (const T*)x + n0 * per, *gp = (const T*)gy + n0 * per, *rp = res ? (const T*)res + n0 * per : nullptr;
    const unsigned char* tp = gate ? gate + n0 * per / VEC : nullptr;
    T *dp = dx ? (T*)dx + n0 * per : nullptr, *ep = dres ? (T*)dres + n0 * per : nullptr;
    const float *mp = mean + n0 * G, *sp = rstd + n0 * G;
    const dim3 grid((unsigned)((s.N + 7) / 8 * 8) * q.nslab * q.nchunk), block(pl.threads);
    float2* part = sums + (size_t)n0 * q.nchunk * q.C;
    if (pl.split) {
      hipLaunchKernelGGL((gn_bwd_chunk_kernel<T, VEC, NM, AK, false>), grid, block, pl.lds, st, s, xp, rp, gp, tp, gamma, beta,
                         mp, sp, (T*)nullptr, (T*)nullptr, part, (const float2*)nullptr);
      if (dx == nullptr && dres == nullptr) continue;
      hipLaunchKernelGGL(gn_bwd_means_kernel, dim3((unsigned)s.N * G), dim3(256), 0, st, (const float2*)part, (int)n0, q.C, q.D,
                         q.P, q.nchunk, q.per_client, gamma, q.gstride, means);
      s.back = 1;
      hipLaunchKernelGGL((gn_bwd_chunk_kernel<T, VEC, NM, AK, true>), grid, block, 0, st, s, xp, rp, gp, tp, gamma, beta, mp, sp,
                         dp, ep, (float2*)nullptr, (const float2*)means);
      continue;
    }
#define GN_BWD(RR)                                                                                                         \
  hipLaunchKernelGGL((gn_bwd_kernel<T, VEC, RR, NM, AK>), grid, block, pl.lds, st, s, xp, rp, gp, tp, gamma, beta, mp, sp, dp, \
                     ep, part)
    switch (pl.R) {
      case 1: case 2: case 4: GN_BWD(4); break;
      case 8: GN_BWD(8); break;
      default:  // 16-bit types alone
        if constexpr (sizeof(T) == 2) GN_BWD(16);
    }
#undef GN_BWD
  }
  return 0;
}

}  // namespace

// dx / dres may be null.  dgamma / dbeta: rows of `ld` floats per client (an update matrix's rows or a [clients][C]
// tensor), scaled by coef[client] (null: 1) and added to what is there where `accumulate`; null: not wanted.
BLADES_API int blades_group_norm_backward(const void* x, const void* res, const void* gy, const void* gate, const float* gamma,
                                          const float* beta, const float* stats, void* dx, void* dres, const float* coef,
                                          float* dgamma, float* dbeta, long ld, int accumulate, float* ws, const Layer* p,
                                          hipStream_t st) {
  const Plan& pl = p->bwd;
  const Geo& q = pl.q;
  const int act = q.act;
  const unsigned char* gt = (const unsigned char*)gate;
  const float *mean = stats, *rstd = stats + (size_t)q.N * (q.C / q.D);
#define GN_B(T, V, M, K) backward_t<T, V, M, K>(pl, x, res, gy, gt, gamma, beta, mean, rstd, dx, dres, ws, st)
#define GN_BT(T)                                                                                  \
  if (p->vec == 1) GN_B(T, 1, 1, -1);                                                             \
  else if (act < 2) { if (pl.one) GN_B(T, 4, 1, 0); else GN_B(T, 4, 4, 0); }                      \
  else if (act == 2) { if (pl.one) GN_B(T, 4, 1, 2); else GN_B(T, 4, 4, 2); }                     \
  else { if (pl.one) GN_B(T, 4, 1, 3); else GN_B(T, 4, 4, 3); }
  if (p->dtype == 0) { GN_BT(float) }
  else if (p->dtype == 1) { GN_BT(Bf16) }
  else { GN_BT(Half) }
#undef GN_BT
#undef GN_B
  if (dgamma != nullptr || dbeta != nullptr) {
    // (samples times chunks stay below 2^24 + 2048: make_plan cuts samples only while there are fewer than 2048 workgroups)
    const long rows = (long)q.per_client * q.nchunk, clients = q.N / q.per_client;
    const int groups = cdiv(q.C, CH);
    const long most = ((1L << 32) - 1) / ((long)groups * AFF_THREADS);  // a grid counts its threads in 32 bits
    for (long k = 0; k < clients; k += most) {
      const long n = clients - k < most ? clients - k : most;
      hipLaunchKernelGGL(gn_affine_kernel, dim3((unsigned)(n * groups)), dim3(AFF_THREADS), 0, st,
                         (const float2*)ws + k * rows * q.C, (int)rows, q.C, coef ? coef + k : nullptr,
                         dgamma ? dgamma + k * ld : nullptr, dbeta ? dbeta + k * ld : nullptr, ld, accumulate);
    }
  }
  return 0;
}
