// Forward pass of the group normalisation: see groupnorm.h.
#include "groupnorm.h"

namespace {
using namespace groupnorm;

// y (and the ReLU's gate) of one vector
template <typename T, int VEC, int NM, int AK>
__device__ __forceinline__ void fwd_vector(const Pack<T, VEC>& x, size_t o, const T* res, T* y, unsigned char* gate,
                                           const float (&mu)[NM], const float (&rs)[NM], const float (&ga)[VEC],
                                           const float (&be)[VEC], int act, bool through) {
  typedef Pack<T, VEC> V;
  float z[VEC];
  normed<T, VEC, NM>(x, mu, rs, z);
#pragma unroll
  for (int j = 0; j < VEC; ++j) z[j] = fmaf(z[j], ga[j], be[j]);
  if (res != nullptr) {
    const V rv = *reinterpret_cast<const V*>(res + o);
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[j] += to_f(rv.e[j]);
  }
  if (gate != nullptr) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) m |= (z[j] <= 0.f ? 0u : 1u) << j;  // (a NaN's gate is open: it was passed on)
    gate[o / VEC] = (unsigned char)m;
  }
  V w;
#pragma unroll
  for (int j = 0; j < VEC; ++j) from_f(act_f<AK, sizeof(T) == 4>(z[j], act), w.e[j]);
  store_out(y + o, w, through);
}

// Whole samples.  R vectors a thread.
template <typename T, int VEC, int R, int NM, int AK>
__global__ __launch_bounds__(MAX_THREADS) void gn_fwd_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                                    const float* __restrict__ gamma,
                                                                    const float* __restrict__ beta, T* __restrict__ y,
                                                                    unsigned char* __restrict__ gate, float* __restrict__ mean,
                                                                    float* __restrict__ rstd) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  const Place<VEC, NM> w(q);
  if (!w.here) return;
  V xr[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.active && w.row + i * q.rows < w.pn) xr[i] = *reinterpret_cast<const V*>(x + w.at + i * w.step);
  float ga[VEC], be[VEC];
  if (w.active) {
    load_floats<VEC>(gamma ? gamma + w.client * q.gstride + w.c0 : nullptr, 1.f, ga);
    load_floats<VEC>(beta ? beta + w.client * q.bstride + w.c0 : nullptr, 0.f, be);
  }
  float *sum = lds, *sq = lds + w.Gs, *red = lds + 2 * w.Gs;
  const float inv = 1.f / ((float)w.pn * (float)q.D);
  const int gw = NM == 1 ? q.D / VEC : q.D;  // entries of a group in a pixel row
  float v[1][NM], mu[NM], rs[NM];
#pragma unroll
  for (int j = 0; j < NM; ++j) v[0][j] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.active && w.row + i * q.rows < w.pn)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[0][NM == 1 ? 0 : j] += to_f(xr[i].e[j]);
  slab_sums<1, NM>(v, gw, w.Gs, q.tw, q, w.l, w.row, w.active, red, sum);
#pragma unroll
  for (int j = 0; j < NM; ++j) { mu[j] = w.active ? sum[w.g[j]] * inv : 0.f; v[0][j] = 0.f; }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.active && w.row + i * q.rows < w.pn)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int m = NM == 1 ? 0 : j;
        const float d = to_f(xr[i].e[j]) - mu[m];
        v[0][m] = fmaf(d, d, v[0][m]);
      }
  slab_sums<1, NM>(v, gw, w.Gs, q.tw, q, w.l, w.row, w.active, red, sq);
  if (mean != nullptr)
    for (int g = threadIdx.x; g < w.Gs; g += blockDim.x) {
      const size_t o = (size_t)w.n * w.G + w.slab * w.Gs + g;
      mean[o] = sum[g] * inv;
      rstd[o] = 1.f / sqrtf(sq[g] * inv + q.eps);
    }
  if (!w.active) return;
#pragma unroll
  for (int j = 0; j < NM; ++j) rs[j] = 1.f / sqrtf(sq[w.g[j]] * inv + q.eps);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (w.row + i * q.rows < w.pn)
      fwd_vector<T, VEC, NM, AK>(xr[i], w.at + i * w.step, res, y, gate, mu, rs, ga, be, q.act, q.through);
}

// Pixel chunks, first sweep: (mean, M2) of a chunk.  A thread takes blocks of 4 vectors, centres each block's squares on
// the block's mean and joins blocks by Chan, Golub and LeVeque's update, so nothing cancels and nothing is read twice.
template <typename T, int VEC, int NM>
__global__ __launch_bounds__(MAX_THREADS) void gn_fwd_stats_kernel(Geo q, const T* __restrict__ x, float2* __restrict__ part) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  const Place<VEC, NM> w(q);
  if (!w.here) return;
  constexpr int E = NM == 1 ? VEC : 1;  // values a thread adds to one entry per vector
  float cnt = 0.f, mn[NM], m2[NM];
#pragma unroll
  for (int j = 0; j < NM; ++j) mn[j] = m2[j] = 0.f;
  if (w.active)
    for (int p = w.row; p < w.pn; p += BLOCK * q.rows) {
      V xr[BLOCK];
      const T* src = x + w.at + (size_t)(p - w.row) * q.C;
#pragma unroll
      for (int i = 0; i < BLOCK; ++i)
        if (p + i * q.rows < w.pn) xr[i] = *reinterpret_cast<const V*>(src + i * w.step);
      float s[NM], k = 0.f;
#pragma unroll
      for (int j = 0; j < NM; ++j) s[j] = 0.f;
#pragma unroll
      for (int i = 0; i < BLOCK; ++i)
        if (p + i * q.rows < w.pn) {
          k += E;
#pragma unroll
          for (int j = 0; j < VEC; ++j) s[NM == 1 ? 0 : j] += to_f(xr[i].e[j]);
        }
      const float ik = __builtin_amdgcn_rcpf(k), share = k * __builtin_amdgcn_rcpf(cnt + k);
      float d2[NM];
#pragma unroll
      for (int j = 0; j < NM; ++j) { s[j] *= ik; d2[j] = 0.f; }
      // (s is a centre near the block's mean; `k * ik` and the sums below make up for its rounding)
#pragma unroll
      for (int i = 0; i < BLOCK; ++i)
        if (p + i * q.rows < w.pn)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int m = NM == 1 ? 0 : j;
            const float d = to_f(xr[i].e[j]) - s[m];
            d2[m] = fmaf(d, d, d2[m]);
          }
#pragma unroll
      for (int j = 0; j < NM; ++j) {
        const float d = s[j] - mn[j];
        mn[j] = fmaf(d, share, mn[j]);
        m2[j] += fmaf(d * d, cnt * share, d2[j]);
      }
      cnt += k;
    }
  float *sum = lds, *sq = lds + w.Gs, *red = lds + 2 * w.Gs;
  const float inv = 1.f / ((float)w.pn * (float)q.D);
  const int gw = NM == 1 ? q.D / VEC : q.D;
  float v[1][NM];
#pragma unroll
  for (int j = 0; j < NM; ++j) v[0][j] = cnt * mn[j];
  slab_sums<1, NM>(v, gw, w.Gs, q.tw, q, w.l, w.row, w.active, red, sum);
#pragma unroll
  for (int j = 0; j < NM; ++j) {
    const float d = w.active ? mn[j] - sum[w.g[j]] * inv : 0.f;
    v[0][j] = fmaf(cnt * d, d, m2[j]);
  }
  slab_sums<1, NM>(v, gw, w.Gs, q.tw, q, w.l, w.row, w.active, red, sq);
  for (int g = threadIdx.x; g < w.Gs; g += blockDim.x)
    part[((size_t)w.n * q.nchunk + w.chunk) * w.G + w.slab * w.Gs + g] = make_float2(sum[g] * inv, sq[g]);
}

// second sweep
template <typename T, int VEC, int NM, int AK>
__global__ __launch_bounds__(MAX_THREADS) void gn_fwd_apply_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           T* __restrict__ y, unsigned char* __restrict__ gate,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd) {
  typedef Pack<T, VEC> V;
  const Place<VEC, NM> w(q);
  if (!w.here || !w.active) return;
  float mu[NM], rs[NM], ga[VEC], be[VEC];
#pragma unroll
  for (int j = 0; j < NM; ++j) {
    const size_t o = (size_t)w.n * w.G + w.slab * w.Gs + w.g[j];
    mu[j] = mean[o]; rs[j] = rstd[o];
  }
  load_floats<VEC>(gamma ? gamma + w.client * q.gstride + w.c0 : nullptr, 1.f, ga);
  load_floats<VEC>(beta ? beta + w.client * q.bstride + w.c0 : nullptr, 0.f, be);
  for (int p = w.row; p < w.pn; p += BLOCK * q.rows) {
    V xr[BLOCK];
    const size_t o = w.at + (size_t)(p - w.row) * q.C;
#pragma unroll
    for (int i = 0; i < BLOCK; ++i)
      if (p + i * q.rows < w.pn) xr[i] = *reinterpret_cast<const V*>(x + o + i * w.step);
#pragma unroll
    for (int i = 0; i < BLOCK; ++i)
      if (p + i * q.rows < w.pn)
        fwd_vector<T, VEC, NM, AK>(xr[i], o + i * w.step, res, y, gate, mu, rs, ga, be, q.act, q.through);
  }
}

// joins the chunks' (mean, M2): one wave per (sample, group), fixed order
__global__ __launch_bounds__(256) void gn_fwd_join_kernel(const float2* __restrict__ part, int n0, int cnt, int G, int D, int P,
                                                          int chunk, int nchunk, float eps, float* __restrict__ mean,
                                                          float* __restrict__ rstd) {
  const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= (long)cnt * G) return;
  const long n = i / G;
  const int g = (int)(i - n * G);
  const float2* p = part + (size_t)n * nchunk * G + g;
  double s = 0.0;
  for (int k = lane; k < nchunk; k += 64) s += (double)min(chunk, P - k * chunk) * p[(size_t)k * G].x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  const double m = s / P;
  double m2 = 0.0;
  for (int k = lane; k < nchunk; k += 64) {
    const float2 e = p[(size_t)k * G];
    const double d = (double)e.x - m;
    m2 += (double)e.y + (double)min(chunk, P - k * chunk) * D * d * d;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
  if (lane == 0) {
    const size_t o = (size_t)(n0 + n) * G + g;
    mean[o] = (float)m;
    rstd[o] = (float)(1.0 / sqrt(m2 / ((double)P * D) + (double)eps));
  }
}

template <typename T, int VEC, int NM, int AK>
int forward_t(const Plan& pl, const void* x, const void* res, const float* gamma, const float* beta, void* y, unsigned char* gate,
              float* mean, float* rstd, float* ws, hipStream_t st) {
  const Geo& q = pl.q;
  const int G = q.C / q.D, N = q.N;
  const size_t per = (size_t)q.P * q.C;
  for (long n0 = 0; n0 < N; n0 += pl.piece) {
    Geo s = q;
    s.N = (int)(N - n0 < pl.piece ? N - n0 : pl.piece);
    s.first = (int)n0;
    const T *xp = (const T*)x + n0 * per, *rp = res ? (const T*)res + n0 * per : nullptr;
    T* yp = (T*)y + n0 * per;
    unsigned char* tp = gate ? gate + n0 * per / VEC : nullptr;
    float *mp = mean ? mean + n0 * G : nullptr, *sp = rstd ? rstd + n0 * G : nullptr;
    const dim3 grid((unsigned)((s.N + 7) / 8 * 8) * q.nslab * q.nchunk), block(pl.threads);
    if (pl.split) {
      hipLaunchKernelGGL((gn_fwd_stats_kernel<T, VEC, NM>), grid, block, pl.lds, st, s, xp, (float2*)ws);
      hipLaunchKernelGGL(gn_fwd_join_kernel, dim3(cdiv((long)s.N * G, 4)), dim3(256), 0, st, (const float2*)ws, (int)n0, s.N, G,
                         q.D, q.P, q.chunk, q.nchunk, q.eps, mean, rstd);
      s.back = 1;
      hipLaunchKernelGGL((gn_fwd_apply_kernel<T, VEC, NM, AK>), grid, block, 0, st, s, xp, rp, gamma, beta, yp, tp, mp, sp);
      continue;
    }
#define GN_FWD(RR)                                                                                                          \
  hipLaunchKernelGGL((gn_fwd_kernel<T, VEC, RR, NM, AK>), grid, block, pl.lds, st, s, xp, rp, gamma, beta, yp, tp, mp, sp)
    switch (pl.R) {
      case 1: case 2: case 4: GN_FWD(4); break;
      case 8: GN_FWD(8); break;
      default: GN_FWD(16); break;
    }
#undef GN_FWD
  }
  return 0;
}

}  // namespace

BLADES_API long blades_group_norm_plan_size() { return sizeof(Layer); }

// What a layer's shape fixes.  dtype 0 fp32, 1 bf16, 2 fp16; vec: 4 channels per access, or 1 where C or an address does not
// allow it.  gamma / beta: stride from client to client in floats (0: shared).  act 0 none, 1 ReLU, 2 GELU, 3 SiLU.
// ws[2]: workspace bytes of the forward (0: a split sample's alone) and backward pass.
// Returns 2 where the shape is not supported (a group's channels exceed a workgroup).
BLADES_API int blades_group_norm_plan(Layer* p, long N, long P, int C, int G, float eps, int act, int per_client, long gstride,
                                      long bstride, int dtype, int vec, long* ws) {
  if (!valid(N, P, C, G, vec, dtype, per_client) || act < 0 || act > 3) return 1;
  p->dtype = dtype; p->vec = vec;
  for (int k = 0; k < 2; ++k) {
    Plan& pl = k ? p->bwd : p->fwd;
    if (!make_plan(pl, N, P, C, G, dtype == 0 ? 4 : 2, vec, k + 1, per_client)) return 2;
    pl.q.eps = eps; pl.q.act = act; pl.q.gstride = gstride; pl.q.bstride = bstride;
    pl.ws = k == 0 ? (pl.split ? pl.piece * pl.q.nchunk * G * 8 : 0)
                   : (N * pl.q.nchunk * C + (pl.split ? pl.piece * G : 0)) * 8;
    ws[k] = pl.ws;
  }
  return 0;
}

// gamma / beta: null or one vector (per client).  stats [2][N][G]: mean, 1 / std; null where neither a backward pass nor a
// workspace follows.  gate: one byte per vector, null: none.
BLADES_API int blades_group_norm_forward(const void* x, const void* res, const float* gamma, const float* beta, void* y,
                                         void* gate, float* stats, float* ws, const Layer* p, hipStream_t st) {
  const Plan& pl = p->fwd;
  const int act = pl.q.act;
  unsigned char* gt = (unsigned char*)gate;
  float *mean = stats, *rstd = stats ? stats + (size_t)pl.q.N * (pl.q.C / pl.q.D) : nullptr;
#define GN_F(T, V, M, K) return forward_t<T, V, M, K>(pl, x, res, gamma, beta, y, gt, mean, rstd, ws, st)
#define GN_FT(T)                                                                                  \
  if (p->vec == 1) GN_F(T, 1, 1, -1);                                                             \
  if (act < 2) { if (pl.one) GN_F(T, 4, 1, 0); GN_F(T, 4, 4, 0); }                                \
  if (act == 2) { if (pl.one) GN_F(T, 4, 1, 2); GN_F(T, 4, 4, 2); }                               \
  if (pl.one) GN_F(T, 4, 1, 3);                                                                   \
  GN_F(T, 4, 4, 3)
  if (p->dtype == 0) { GN_FT(float); }
  if (p->dtype == 1) { GN_FT(Bf16); }
  GN_FT(Half);
#undef GN_FT
#undef GN_F
}
