// Rotary positions with several axes (row and column of an image patch; time, height and width of a video one).
//
// The head dimension is cut into one section per axis (the rest passes through).  Pair i of the section of axis a, d_a wide,
// is the complex number x[2i] + j x[2i + 1]; it is turned by pos_a * base^(-2i / d_a) (inverse: by the negative angle,
// which is the gradient, a rotation's transpose).
//
// x [R][N][S][H][D] with any strides (D contiguous): slots s < rot of the packed projection are turned (q and k), the
// others copied (v).  A thread owns 16 bytes of the head dimension of one token: its two (four) angles are computed once,
// the turns (position times frequency in turns, reduced to an eighth) in 64 bits so that far positions keep theirs, sine
// and cosine by their Taylor polynomials in 32 bits, and used for all slots and heads of the token.
// Memory-bound: every byte is read and written once.
#include "common.h"

namespace {
constexpr int TPB = 256;
constexpr int MAX_PAIRS = 128;  // head dimension up to 256

struct Half { unsigned short v; };
struct Bf16 { unsigned short v; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(Bf16 v) { return __uint_as_float((unsigned)v.v << 16); }
__device__ __forceinline__ float to_f(Half v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f(float f, Bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ void from_f(float f, Half& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)f); }
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

struct Freq {
  double turns[MAX_PAIRS];         // base^(-2i / d_a) / 2 pi
  unsigned char axis[MAX_PAIRS];   // axis of the pair; 255: passes through
};

struct Shape {
  long R, N, sr, sn, ss, sh;       // samples, tokens; strides of x in elements (D: 1)
  int S, H, D, A, rot, slots;      // slots that are turned; slots that are walked (in place: the turned ones alone)
  long psr;                        // sample stride of the positions (0: shared)
  int pos_float, inverse;
};

// sine and cosine of a full turn's fraction
__device__ __forceinline__ void sincos_turns(double turns, float& s, float& c) {
  const double q = rint(turns * 4.0);
  const float a = (float)((turns - q * 0.25) * 6.283185307179586476925);  // |a| <= pi / 4 (+ rounding)
  const float b = a * a;
  // Taylor: the first terms left out are below 2^-27 for |a| <= pi / 4
  const float sa = fmaf(a * b, fmaf(b, fmaf(b, fmaf(b, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), a);
  const float ca = fmaf(b, fmaf(b, fmaf(b, fmaf(b, fmaf(b, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
  const int k = (int)((long long)q & 3);
  const float u = k & 1 ? ca : sa, v = k & 1 ? sa : ca;
  s = k & 2 ? -u : u;
  c = (k == 1 || k == 2) ? -v : v;
}

// gridDim.y workgroups share a token's S * H rows (`per` each) where there are few tokens.
template <typename T, int VEC>
__global__ __launch_bounds__(TPB) void rope_kernel(Freq f, Shape q, int per, const T* x, const void* __restrict__ pos, T* y) {
  typedef Pack<T, VEC> V;
  constexpr int U = 4;
  const int L = q.D / VEC;  // threads of a token
  const int r0 = blockIdx.y * per, r1 = min(r0 + per, q.slots * q.H);
  const bool turns = r0 < q.rot * q.H;
  const bool same = (const void*)x == (const void*)y;
  for (long i = (long)blockIdx.x * TPB + threadIdx.x; i < q.R * q.N * L; i += (long)gridDim.x * TPB) {
    const long token = i / L;
    const int l = (int)(i - token * L);
    const long r = token / q.N, n = token - r * q.N;
    const long xo = r * q.sr + n * q.sn + l * VEC;
    const size_t yo = (size_t)token * q.S * q.H * q.D + (size_t)l * VEC;
    float sn[VEC / 2], cs[VEC / 2];
    if (turns) {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const int pair = l * (VEC / 2) + j, a = f.axis[pair];
        sn[j] = 0.f; cs[j] = 1.f;
        if (a != 255) {
          const long o = r * q.psr + n * q.A + a;
          const double p = q.pos_float ? (double)static_cast<const float*>(pos)[o] : (double)static_cast<const long*>(pos)[o];
          sincos_turns(p * f.turns[pair], sn[j], cs[j]);
          if (q.inverse) sn[j] = -sn[j];
        }
      }
    }
    int s = r0 / q.H, h = r0 - s * q.H;
    for (int row = r0; row < r1; row += U) {
      V w[U];
      long at[U];
      bool turn[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        at[u] = xo + s * q.ss + h * q.sh;
        turn[u] = s < q.rot;
        if (row + u < r1) w[u] = *reinterpret_cast<const V*>(x + at[u]);
        if (++h == q.H) { h = 0; ++s; }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row + u < r1) {
          if (turn[u]) {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              const float a = to_f(w[u].e[2 * j]), b = to_f(w[u].e[2 * j + 1]);
              from_f(fmaf(a, cs[j], -b * sn[j]), w[u].e[2 * j]);
              from_f(fmaf(a, sn[j], b * cs[j]), w[u].e[2 * j + 1]);
            }
          }
          *reinterpret_cast<V*>(y + (same ? (size_t)at[u] : yo + (size_t)(row + u) * q.D)) = w[u];
        }
    }
  }
}
}  // namespace

// axes[A]: section widths (even, sum <= D).  y: contiguous [R][N][S][H][D], or x itself (then only the turned slots are
// touched).  dtype 0 fp32, 1 bf16, 2 fp16; vec: elements per access (16 bytes, or 2 where an address does not allow it).
BLADES_API int blades_rope_axes(const void* x, void* y, const void* pos, int pos_float, long psr, long R, long N, int S, int H,
                                int D, long sr, long sn, long ss, long sh, int rot, const int* axes, int A, double base,
                                int inverse, int dtype, int vec, hipStream_t st) {
  if (R < 1 || N < 1 || S < 1 || H < 1 || D < 2 || D > 2 * MAX_PAIRS || D % 2 || A < 1 || A > 8 || rot < 0 || rot > S) return 1;
  if (dtype < 0 || dtype > 2 || (vec != 2 && vec != (dtype == 0 ? 4 : 8)) || D % vec || !(base > 0.0)) return 1;
  Freq f;
  int pair = 0;
  for (int a = 0; a < A; ++a) {
    if (axes[a] < 2 || axes[a] % 2 || 2 * pair + axes[a] > D) return 1;
    for (int i = 0; i < axes[a] / 2; ++i, ++pair) {
      f.turns[pair] = pow(base, -2.0 * i / axes[a]) * 0.15915494309189533577;
      f.axis[pair] = (unsigned char)a;
    }
  }
  for (; pair < MAX_PAIRS; ++pair) { f.turns[pair] = 0.0; f.axis[pair] = 255; }
  const Shape q{R, N, sr, sn, ss, sh, S, H, D, A, rot, x == y ? rot : S, psr, pos_float, inverse};
  long blocks = (R * N * (D / vec) + TPB - 1) / TPB;
  if (blocks > (1L << 20)) blocks = 1L << 20;
  // a thread's rows: all of its token, fewer (at least 4 at a time) while the chip's 256 x 8 workgroups are not there
  const int rows = q.slots * H;
  if (rows == 0) return 0;
  int per = rows;
  while (per > 4 && blocks * ((rows + per - 1) / per) < 2048) per = (per + 1) / 2;
  const dim3 grid((unsigned)blocks, (unsigned)((rows + per - 1) / per)), block(TPB);
#define ROPE(T, V) hipLaunchKernelGGL((rope_kernel<T, V>), grid, block, 0, st, f, q, per, (const T*)x, pos, (T*)y)
  if (dtype == 0) { if (vec == 4) ROPE(float, 4); else ROPE(float, 2); }
  else if (dtype == 1) { if (vec == 8) ROPE(Bf16, 8); else ROPE(Bf16, 2); }
  else { if (vec == 8) ROPE(Half, 8); else ROPE(Half, 2); }
#undef ROPE
  return 0;
}
