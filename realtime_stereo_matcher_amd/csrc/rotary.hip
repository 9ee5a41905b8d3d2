// Rotary positions: the first R values of every head are R/2 pairs, and pair i of a token at
// position t is turned by the angle t f_i (f: R/2 frequencies, radians a position):
//   (u, w) -> a (u cos - w sin, w cos + u sin)
// "half": pair i is values i and i + R/2; "interleaved": values 2i and 2i + 1.  The values past R
// pass through.  The gradient is the turn by -t f_i.
//
// The angle is formed as a count of turns, t (f / 2 pi), in pairs of 64-bit numbers, and only its
// fraction, in [-1/2, 1/2], is rounded to fp32: any 64-bit position is turned as exactly as position
// 1, and no table of positions is kept or read.  A thread forms the sines of its pairs once and turns the
// same values of several heads with them, so the arithmetic hides behind the one read and one
// write of x that bound the operator: 4 x 8160 tokens, 16 heads of 128, 64 values turned, bf16: 267 MB
// in 54 us (4.9 TB/s, the rate of a large copy); 16 single tokens 4.2 us.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace smcv {
namespace rotary {

struct Args {
  const void* x;
  void* y;
  const void* pos;
  const double* freq;
  int64_t xs[3], ps;  // element strides of x (batch, token, head); of the positions' batches
  int64_t tokens;     // B * L
  int L, H, D, R;
  int cols;           // threads' columns of a head: rotated pieces, then pieces that pass through
  int turned;         // rotated pieces
  int par;            // heads taken side by side by different threads
  bool wide_pos;      // 64-bit positions
  float amp, sign;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec { T v[V]; };

// The fraction of (p + p0) f / (2 pi), for a p that 64 bits hold and a p0 that is small beside it.  f's
// turns are hi + lo, within 2^-105 of them; p hi is its rounding a and the rest e.  Each part's own
// fraction is exact, so what is lost is about 2^-53 and |p f| 2^-105.  (Twelve 64-bit operations more
// a pair than one product has; the copy still hides them.)  Nothing may be contracted here.
__device__ __forceinline__ float turned_part(double p, double p0, double f) {
#pragma clang fp contract(off)
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kRest = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double hi = f * kTurn, lo = fma(f, kRest, fma(f, kTurn, -hi));
  const double a = p * hi, e = fma(p, hi, -a), c = fma(p, lo, p0 * hi);
  const double t = (a - rint(a)) + ((e - rint(e)) + (c - rint(c)));
  return (float)(t - rint(t));
}

template <typename T, int V, bool HALF>
__global__ __launch_bounds__(256) void rotate(Args a) {
  const int64_t id = (int64_t)workgroup() * 256 + threadIdx.x;
  const int col = (int)(id % a.cols);
  const int64_t rest = id / a.cols;
  const int first = (int)(rest % a.par);
  const int64_t tok = rest / a.par;
  if (tok >= a.tokens) return;
  const int64_t b = tok / a.L;
  const int t = (int)(tok - b * a.L);
  const T* x = static_cast<const T*>(a.x) + b * a.xs[0] + t * a.xs[1];
  T* y = static_cast<T*>(a.y) + tok * a.H * a.D;
  using VT = Vec<T, V>;
  if (col >= a.turned) {
    const int d = a.R + (col - a.turned) * V;
#pragma unroll 4
    for (int h = first; h < a.H; h += a.par)
      *reinterpret_cast<VT*>(y + (int64_t)h * a.D + d) =
          *reinterpret_cast<const VT*>(x + h * a.xs[2] + d);
    return;
  }
  const int64_t at = b * a.ps + t;
  const int64_t pos = a.wide_pos ? static_cast<const int64_t*>(a.pos)[at] : static_cast<const int*>(a.pos)[at];
  // past 2^53 the last bits on their own, so that both parts are exact
  const int64_t last = ((uint64_t)pos + (1ull << 53)) >> 54 != 0 ? pos & 2047 : 0;
  const double p0 = (double)last, p1 = (double)(pos - last);
  // HALF: V pairs, one value of each in two vectors; interleaved: V/2 pairs side by side (V = 1:
  // a pair is two scalars in either layout)
  constexpr int P = HALF || V == 1 ? V : V / 2;
  float cs[P], sn[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    sincospif(2.f * turned_part(p1, p0, a.freq[col * P + p]), &sn[p], &cs[p]);
    cs[p] *= a.amp;
    sn[p] *= a.amp * a.sign;
  }
  if constexpr (HALF || V == 1) {
    const int d0 = HALF ? col * V : 2 * col, d1 = HALF ? d0 + a.R / 2 : d0 + 1;
#pragma unroll 4
    for (int h = first; h < a.H; h += a.par) {
      const T* xh = x + h * a.xs[2];
      T* yh = y + (int64_t)h * a.D;
      VT u = *reinterpret_cast<const VT*>(xh + d0), w = *reinterpret_cast<const VT*>(xh + d1);
#pragma unroll
      for (int p = 0; p < V; ++p) {
        const float uf = to_f(u.v[p]), wf = to_f(w.v[p]);
        u.v[p] = from_f<T>(fmaf(uf, cs[p], -(wf * sn[p])));
        w.v[p] = from_f<T>(fmaf(wf, cs[p], uf * sn[p]));
      }
      *reinterpret_cast<VT*>(yh + d0) = u;
      *reinterpret_cast<VT*>(yh + d1) = w;
    }
  } else {
    const int d = col * V;
#pragma unroll 4
    for (int h = first; h < a.H; h += a.par) {
      VT u = *reinterpret_cast<const VT*>(x + h * a.xs[2] + d);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float uf = to_f(u.v[2 * p]), wf = to_f(u.v[2 * p + 1]);
        u.v[2 * p] = from_f<T>(fmaf(uf, cs[p], -(wf * sn[p])));
        u.v[2 * p + 1] = from_f<T>(fmaf(wf, cs[p], uf * sn[p]));
      }
      *reinterpret_cast<VT*>(y + (int64_t)h * a.D + d) = u;
    }
  }
}

template <typename T, int V>
int launch(Args& a, bool half, hipStream_t st) {
  a.turned = half || V == 1 ? a.R / 2 / V : a.R / V;
  a.cols = a.turned + (a.D - a.R) / V;
  // heads side by side: all of them while the launch is short of threads (a few tokens), else so
  // many that each thread turns up to 4 heads with one set of sines
  const int64_t threads = a.tokens * a.cols;
  int64_t par = a.H;
  if (threads * a.H > (int64_t)256 * 2048) par = std::max<int64_t>(ceil_div(a.H, 4), std::min<int64_t>(a.H, ceil_div(256 * 2048, threads)));
  a.par = (int)par;
  const int64_t grid = ceil_div(threads * par, 256);
  if (grid > 0x7fffffffll) return fail(SM_EINVAL, "rotary: too many tokens");
  if (half)
    rotate<T, V, true><<<grid_of(grid), 256, 0, st>>>(a);
  else
    rotate<T, V, false><<<grid_of(grid), 256, 0, st>>>(a);
  return check_launch("rotary");
}

}  // namespace rotary

int rotary_entry(const void* x, const void* positions, const double* frequencies, void* y, int dtype,
                 int64_t B, int64_t L, int64_t H, int64_t D, int64_t R, const int64_t* x_strides,
                 int64_t position_stride, int flags, float amplitude, void* stream) {
  if (!valid_dtype(dtype)) return fail(SM_EDTYPE, "rotary: float32, float16 or bfloat16 only");
  if (B < 0 || L < 0 || H < 0 || D < 0) return fail(SM_EINVAL, "rotary: negative size");
  if (R < 2 || R % 2 != 0 || R > D)
    return fail(SM_EINVAL, "rotary: the rotated part must be an even number of values of the head");
  if (L >= (1ll << 31) || H >= (1 << 24) || D >= (1 << 24) || B >= (1ll << 31))
    return fail(SM_EINVAL, "rotary: size too large");
  if ((flags & ~7) != 0) return fail(SM_EINVAL, "rotary: unknown flags");
  rotary::Args a{};
  if (x_strides != nullptr) {
    for (int i = 0; i < 3; ++i) {
      if (x_strides[i] < 0) return fail(SM_EINVAL, "rotary: negative strides are not supported");
      a.xs[i] = x_strides[i];
    }
  } else {
    a.xs[0] = L * H * D;
    a.xs[1] = H * D;
    a.xs[2] = D;
  }
  if (position_stride < 0) return fail(SM_EINVAL, "rotary: negative strides are not supported");
  if (B == 0 || L == 0 || H == 0) return SM_OK;
  if (x == nullptr || y == nullptr || positions == nullptr || frequencies == nullptr)
    return fail(SM_EINVAL, "rotary: null pointer");
  a.x = x;
  a.y = y;
  a.pos = positions;
  a.freq = frequencies;
  a.ps = position_stride;
  a.tokens = B * L;
  a.L = (int)L;
  a.H = (int)H;
  a.D = (int)D;
  a.R = (int)R;
  a.wide_pos = (flags & SM_ROTARY_POS64) != 0;
  a.amp = amplitude;
  a.sign = (flags & SM_ROTARY_INVERSE) ? -1.f : 1.f;
  const bool half = (flags & SM_ROTARY_INTERLEAVED) == 0;
  // 16-byte pieces where every row, and each layout's first and second values, are aligned to them
  const int per = 16 / elem_size(dtype);
  bool wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0 &&
              D % per == 0 && R % per == 0 && (!half || R / 2 % per == 0);
  for (int i = 0; i < 3; ++i) wide = wide && a.xs[i] % per == 0;
  hipStream_t st = as_stream(stream);
  SM_DISPATCH_DTYPE(dtype, T, return wide ? rotary::launch<T, 16 / (int)sizeof(T)>(a, half, st)
                                          : rotary::launch<T, 1>(a, half, st));
  return SM_OK;
}

}  // namespace smcv
