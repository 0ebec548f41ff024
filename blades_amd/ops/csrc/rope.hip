// Rotary positions with several axes (row and column of an image patch; time, height and width of a video one).
//
// The head dimension is cut into one section per axis (the rest passes through).  Pair i of the section of axis a, d_a wide,
// is the complex number x[2i] + j x[2i + 1]; it is turned by pos_a * base^(-2i / d_a) (inverse: by the negative angle,
// which is the gradient, a rotation's transpose).
//
// x [R][N][S][H][D] with any strides (D contiguous): slots s < rot of the packed projection are turned (q and k), the
// others copied (v).  A thread owns 16 bytes of the head dimension of one token: while its first rows are on their way, its two
// (four) angles are computed, once for all its rows (slots and heads): the turns (position times frequency, reduced to an
// eighth) in 64 bits so that far positions keep theirs, sine and cosine by their Taylor polynomials in 32 bits.
// Memory-bound: every byte is read and written once.  Kernel times on average over training passes: 2048 x 64 x 3 x 2 x 64
// fp32 74 us (5.5 TB/s), 8 x 3136 x 3 x 6 x 64 bf16 with per-sample positions 23 (5.0; 19 without the angles).  (A workgroup that
// shares its tokens' angles through LDS and walks memory in order was slower, 95 against 73 us on the first: the index arithmetic
// of every vector and half the waves cost more than the angles.)
#include "common.h"
#include "layers_abi.h"

namespace rope {
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
  int pos_float, inverse, through;
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
  constexpr int U = 6;
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
    V w[U];
    long at[U];
    int s = r0 / q.H, h = r0 - s * q.H, turned[U];
    auto fetch = [&](int row) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        at[u] = xo + s * q.ss + h * q.sh;
        turned[u] = s < q.rot;
        if (row + u < r1) w[u] = *reinterpret_cast<const V*>(x + at[u]);
        if (++h == q.H) { h = 0; ++s; }
      }
    };
    fetch(r0);
    float sn[VEC / 2], cs[VEC / 2];
    bool still[VEC / 2];  // pairs that pass through: as they are (a turn by 0 would let an infinity into its neighbour)
    if (turns) {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const int pair = l * (VEC / 2) + j, a = f.axis[pair];
        sn[j] = 0.f; cs[j] = 1.f;
        still[j] = a == 255;
        if (!still[j]) {
          const long o = r * q.psr + n * q.A + a;
          const double p = q.pos_float ? (double)static_cast<const float*>(pos)[o] : (double)static_cast<const long*>(pos)[o];
          sincos_turns(p * f.turns[pair], sn[j], cs[j]);
          if (q.inverse) sn[j] = -sn[j];
        }
      }
    }
    for (int row = r0;;) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row + u < r1) {
          if (turned[u]) {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              const float a = to_f(w[u].e[2 * j]), b = to_f(w[u].e[2 * j + 1]);
              T ta, tb;
              from_f(fmaf(a, cs[j], -b * sn[j]), ta);
              from_f(fmaf(a, sn[j], b * cs[j]), tb);
              w[u].e[2 * j] = still[j] ? w[u].e[2 * j] : ta;
              w[u].e[2 * j + 1] = still[j] ? w[u].e[2 * j + 1] : tb;
            }
          }
          store_out(y + (same ? (size_t)at[u] : yo + (size_t)(row + u) * q.D), w[u], q.through);
        }
      row += U;
      if (row >= r1) break;
      fetch(row);
    }
  }
}

struct RopePlan {
  Freq f;
  Shape q;
  int dtype, vec, blocks, per, per_in_place;
};

// A thread's rows: all of its token, fewer (at least 4) while the chip's 256 x 8 workgroups are not there.
inline int rows_of(long blocks, int rows) {
  int per = rows;
  while (per > 4 && blocks * ((rows + per - 1) / per) < 2048) per = (per + 1) / 2;
  return per;
}
}  // namespace rope
using namespace rope;

BLADES_API long blades_rope_plan_size() { return sizeof(RopePlan); }

// What a layer's shape fixes.  axes[A]: section widths (even, sum <= D).  Strides of x in elements (D: 1).  dtype 0 fp32,
// 1 bf16, 2 fp16; vec: elements per access (16 bytes, or 2 where an address or a stride does not allow it).
BLADES_API int blades_rope_plan(RopePlan* p, int pos_float, long psr, long R, long N, int S, int H, int D, long sr, long sn,
                                long ss, long sh, int rot, const int* axes, int A, double base, int dtype, int vec) {
  if (R < 1 || N < 1 || S < 1 || H < 1 || D < 2 || D > 2 * MAX_PAIRS || D % 2 || A < 1 || A > 8 || rot < 0 || rot > S) return 1;
  if (dtype < 0 || dtype > 2 || (vec != 2 && vec != (dtype == 0 ? 4 : 8)) || D % vec || !(base > 0.0)) return 1;
  if ((double)S * H > 1e9) return 1;
  int pair = 0;
  for (int a = 0; a < A; ++a) {
    if (axes[a] < 2 || axes[a] % 2 || 2 * pair + axes[a] > D) return 1;
    for (int i = 0; i < axes[a] / 2; ++i, ++pair) {
      p->f.turns[pair] = pow(base, -2.0 * i / axes[a]) * 0.15915494309189533577;
      p->f.axis[pair] = (unsigned char)a;
    }
  }
  for (; pair < MAX_PAIRS; ++pair) { p->f.turns[pair] = 0.0; p->f.axis[pair] = 255; }
  // Outputs of up to 256 MB, the last-level cache, are stored past it.  Kernel times on average, stored past it against through
  // it: forward passes over one input / in a row of three with a product of equal size in front and behind.
  //   2048 x 64 x 3 x 2 x 64 fp32    62 : 79 / 203 : 217
  //   8 x 3136 x 3 x 6 x 64 bf16     23 : 24 /  59 :  59
  const long bytes = R * N * S * H * D * (dtype == 0 ? 4 : 2);
  p->q = Shape{R, N, sr, sn, ss, sh, S, H, D, A, rot, S, psr, pos_float, 0, bytes <= (256L << 20)};
  p->dtype = dtype; p->vec = vec;
  const long blocks = (R * N * (D / vec) + TPB - 1) / TPB;
  p->blocks = (int)(blocks > (1L << 20) ? 1L << 20 : blocks);
  p->per = rows_of(p->blocks, S * H);
  p->per_in_place = rows_of(p->blocks, rot * H);
  return 0;
}

// y: contiguous [R][N][S][H][D], or x itself (then only the turned slots are touched).
BLADES_API int blades_rope_axes(const void* x, void* y, const void* pos, const RopePlan* p, int inverse, hipStream_t st) {
  Shape q = p->q;
  q.inverse = inverse;
  if (x == y) q.slots = q.rot;
  const int rows = q.slots * q.H, per = x == y ? p->per_in_place : p->per;
  if (rows == 0) return 0;
  const dim3 grid((unsigned)p->blocks, (unsigned)((rows + per - 1) / per)), block(TPB);
  if (grid.y > 65535) return 1;
#define ROPE(T, V) hipLaunchKernelGGL((rope_kernel<T, V>), grid, block, 0, st, p->f, q, per, (const T*)x, pos, (T*)y)
  if (p->dtype == 0) { if (p->vec == 4) ROPE(float, 4); else ROPE(float, 2); }
  else if (p->dtype == 1) { if (p->vec == 8) ROPE(Bf16, 8); else ROPE(Bf16, 2); }
  else { if (p->vec == 8) ROPE(Half, 8); else ROPE(Half, 2); }
#undef ROPE
  return 0;
}
