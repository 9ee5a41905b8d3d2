// Root-mean-square norm of rows, with the residual's addition before it and, for serving, an output
// in 8 bits:
//   s = x + r (rounded to r's type: what the next layer adds to)   n = s / sqrt(mean s^2 + eps)
//   y = n w         or  q = e4m3(y / scale), scale = max |y| / 448 over the row or 128 values
// backward: with h = g w (g the gradient of y, z that of s),
//   ds = (h - n mean(h n)) / sqrt(mean s^2 + eps) + z        dw = sum over rows of g n
//
// Bound by memory: a row is read once into registers (8 neighbouring values a thread and step) and
// both its statistics and its outputs come from there.  Sums are fp32.  A row has 4 to 1024 threads,
// so that a wave holds whole rows of narrow maps and a workgroup one wide row.  518,400 rows of 64,
// bf16 with residual: forward 265 MB in 46 us, backward the same in 56 us and 6 us for the sum of dw;
// 32,760 rows of 5000, fp16 with a 32-bit stream, to e4m3: 1.8 GB in 359 us (5.0 TB/s;
// 350 with the codes' last two steps in 32 bits, which moved about one code in a million).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace smcv {
namespace rms {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

enum { kNone = 0, kSame = 1, kF32 = 2 };  // types of the residual and of the weight, against x's

struct Args {
  const void *x, *r, *w, *dy, *ds;
  void *y, *s, *q, *dx, *dr;
  float *scale, *part;
  int64_t rows, xs, rs, ys, zs;  // row strides of x, r, dy and ds (outputs are dense)
  int C, groups;
  int r_type, w_type;
  int vec;       // bits: which operands take 16-byte accesses
  float eps;
};

template <typename T>
__device__ __forceinline__ void get8(float (&v)[8], const T* p, int n, bool vec) {
  if (vec) {
    T t[8];
    if constexpr (sizeof(T) == 4) {
      const u32x4 a = reinterpret_cast<const u32x4*>(p)[0], b = reinterpret_cast<const u32x4*>(p)[1];
      __builtin_memcpy(t, &a, 16);
      __builtin_memcpy(t + 4, &b, 16);
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4*>(p);
      __builtin_memcpy(t, &a, 16);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f(t[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f(p[e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&v)[8], int n, bool vec) {
  if (vec) {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = from_f<T>(v[e]);
    u32x4 a[sizeof(T) * 8 / 16];
    __builtin_memcpy(a, t, sizeof(t));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) reinterpret_cast<u32x4*>(p)[i] = a[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = from_f<T>(v[e]);
  }
}
template <typename T>
__device__ __forceinline__ void get8_of(float (&v)[8], const void* base, int64_t at, int type, int n,
                                        bool vec) {
  if (type == kF32) get8(v, static_cast<const float*>(base) + at, n, vec);
  else get8(v, static_cast<const T*>(base) + at, n, vec);
}
template <typename T>
__device__ __forceinline__ void put8_of(void* base, int64_t at, int type, const float (&v)[8], int n,
                                        bool vec) {
  if (type == kF32) put8(static_cast<float*>(base) + at, v, n, vec);
  else put8(static_cast<T*>(base) + at, v, n, vec);
}

// the larger of two values that are not negative; NaN, whose bits are larger than infinity's, stays
__device__ __forceinline__ float larger(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// sums (or the maximum) over the TPR threads of a row; every thread receives the result.  Wide rows
// (TPR > 64) join their waves through `lds`, which the next call may use again at once: two slots,
// taken in turn.
template <int TPR, bool MAX, int N>
__device__ __forceinline__ void over_row(float (&v)[N], float* lds, int& slot) {
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = __shfl_xor(v[i], o);
      v[i] = MAX ? larger(v[i], u) : v[i] + u;
    }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* mine = lds + slot * W * 2;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) mine[i * W + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float u = mine[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) u = MAX ? larger(u, mine[i * W + w]) : u + mine[i * W + w];
      v[i] = u;
    }
  }
}

enum { kVecX = 1, kVecR = 2, kVecW = 4, kVecY = 8, kVecS = 16, kVecZ = 32, kVecD = 64, kVecDr = 128 };

template <typename T, int TPR, int NV, bool Q8>
__global__ __launch_bounds__((TPR > 256 ? TPR : 256)) void forward(Args a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kRowsWg = kThreads / TPR;
  __shared__ float lds[TPR > 64 ? 4 * TPR / 64 : 1];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)workgroup() * kRowsWg + threadIdx.x / TPR;
  const bool there = row < a.rows;
  float v[NV][8];
  float sq[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
    if (n > 0) {
      get8(v[k], static_cast<const T*>(a.x) + row * a.xs + c, n, a.vec & kVecX);
      if (a.r_type != kNone) {
        float r[8];
        get8_of<T>(r, a.r, row * a.rs + c, a.r_type, n, a.vec & kVecR);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[k][e] += r[e];
          // the stream is normalised as it is stored: its one rounding is part of the definition,
          // and the backward pass reads the same values
          if (a.r_type == kSame) v[k][e] = to_f(from_f<T>(v[k][e]));
        }
        put8_of<T>(a.s, row * a.C + c, a.r_type, v[k], n, a.vec & kVecS);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sq[0] = fmaf(v[k][e], v[k][e], sq[0]);
    }
  }
  over_row<TPR, false>(sq, lds, slot);
  const float inv = 1.f / sqrtf(sq[0] / (float)a.C + a.eps);
  float top[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
    top[k] = 0.f;
    if (n > 0) {
      float w[8];
      get8_of<T>(w, a.w, c, a.w_type, n, a.vec & kVecW);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (Q8) top[k] = larger(top[k], fabsf(v[k][e] * w[e]));
        else v[k][e] = v[k][e] * inv * w[e];
      }
      if constexpr (!Q8) put8(static_cast<T*>(a.y) + row * a.C + c, v[k], n, a.vec & kVecY);
    }
  }
  if constexpr (Q8) {
    auto over_group = [&](float (&m)[NV]) {
      if (a.groups == 1) {
#pragma unroll
        for (int k = 1; k < NV; ++k) m[0] = larger(m[0], m[k]);
        float one[1] = {m[0]};
        over_row<TPR, true>(one, lds, slot);
#pragma unroll
        for (int k = 0; k < NV; ++k) m[k] = one[0];
      } else {  // 128 values are 16 neighbouring threads' of one step (narrower rows: one group)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1)
#pragma unroll
          for (int k = 0; k < NV; ++k) m[k] = larger(m[k], __shfl_xor(m[k], o));
      }
    };
    float mine[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) mine[k] = top[k];
    over_group(top);
    // What the largest |s w| lost to its rounding, plus a unit (so that it is positive): of the values
    // that round to it, the largest.  Products of two 16-bit values are exact.
    float low[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) low[k] = 0.f;
    if (sizeof(T) == 4 || a.r_type == kF32 || a.w_type == kF32) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
        if (n <= 0 || mine[k] != top[k] || !(top[k] > 0x1p-60f && top[k] < INFINITY)) continue;
        float w[8];
        get8_of<T>(w, a.w, c, a.w_type, n, a.vec & kVecW);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = v[k][e] * w[e], lost = fmaf(v[k][e], w[e], -p);
          if (fabsf(p) == top[k]) low[k] = larger(low[k], top[k] * 0x1p-23f + (p < 0.f ? -lost : lost));
        }
      }
      over_group(low);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
      if (n <= 0) continue;
      // y / scale = s w 448 / max |s w|: the root cancels, and formed in 64 bits the value is rounded
      // once to 32 before it is rounded to 8, so no code on a border between two is left to chance
      const float most = top[k], y_most = most * inv;
      const float scale = y_most == 0.f ? 1.f : y_most / 448.f;
      const double by = 448.0 / (low[k] > 0.f ? (double)most + ((double)low[k] - (double)(most * 0x1p-23f)) : (double)most);
      float w[8];
      get8_of<T>(w, a.w, c, a.w_type, n, a.vec & kVecW);
      const int g = a.groups == 1 ? 0 : c / 128;
      if (a.groups == 1 ? c == 0 : c % 128 == 0) a.scale[row * a.groups + g] = scale;
      unsigned p[2];
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // NaN stays NaN
        z[e] = y_most == 0.f ? 0.f : (float)((double)v[k][e] * (double)w[e] * by);
        z[e] = z[e] > 448.f ? 448.f : z[e] < -448.f ? -448.f : z[e];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int u = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i], z[4 * i + 1], 0, false);
        p[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i + 2], z[4 * i + 3], u, true);
      }
      uint8_t* out = static_cast<uint8_t*>(a.q) + row * a.C + c;
      if (a.vec & kVecY) {
        *reinterpret_cast<u32x2*>(out) = u32x2{p[0], p[1]};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) out[e] = (uint8_t)(p[e >> 2] >> (8 * (e & 3)));
      }
    }
  }
}

// One workgroup takes every gridDim-th set of rows, keeps its share of dw in registers and leaves it
// in `part`; weight_sum adds the shares in their order, so the sum is the same on every run.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__((TPR > 256 ? TPR : 256)) void backward(Args a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kRowsWg = kThreads / TPR;
  __shared__ float lds[TPR > 64 ? 4 * TPR / 64 : 1];
  __shared__ float join[kRowsWg > 1 ? kThreads * 8 : 1];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  constexpr bool kKeep = TPR <= 256;  // the weights in registers (1024 threads have 128 each)
  float dw[NV][8], w[kKeep ? NV : 1][8];
  auto weights = [&](int k) {
    const int c = (k * TPR + t) * 8;
    if (c < a.C) get8_of<T>(w[kKeep ? k : 0], a.w, c, a.w_type, a.C - c, a.vec & kVecW);
  };
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = w[kKeep ? k : 0][e] = 0.f;
    if (kKeep) weights(k);
  }
  const int64_t sets = (a.rows + kRowsWg - 1) / kRowsWg;
  for (int64_t set = blockIdx.x; set < sets; set += gridDim.x) {
    const int64_t row = set * kRowsWg + threadIdx.x / TPR;
    const bool there = row < a.rows;
    float s[NV][8], h[NV][8], sums[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[k][e] = h[k][e] = 0.f;
      if (n > 0) {
        get8_of<T>(s[k], a.s, row * a.xs + c, a.r_type, n, a.vec & kVecS);
        get8(h[k], static_cast<const T*>(a.dy) + row * a.ys + c, n, a.vec & kVecY);
        if (!kKeep) weights(k);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sums[0] = fmaf(s[k][e], s[k][e], sums[0]);
          sums[1] = fmaf(h[k][e] * w[kKeep ? k : 0][e], s[k][e], sums[1]);
        }
      }
    }
    over_row<TPR, false>(sums, lds, slot);
    const float inv = 1.f / sqrtf(sums[0] / (float)a.C + a.eps);
    const float back = sums[1] / (float)a.C * inv * inv * inv;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * 8, n = there ? a.C - c : 0;
      if (n <= 0) continue;
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = 0.f;
      if (a.ds != nullptr) get8_of<T>(z, a.ds, row * a.zs + c, a.r_type, n, a.vec & kVecZ);
      if (!kKeep) weights(k);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[k][e] = fmaf(h[k][e] * inv, s[k][e], dw[k][e]);
        z[e] += h[k][e] * w[kKeep ? k : 0][e] * inv - s[k][e] * back;
      }
      put8(static_cast<T*>(a.dx) + row * a.C + c, z, n, a.vec & kVecD);
      if (a.dr != nullptr) put8(static_cast<float*>(a.dr) + row * a.C + c, z, n, a.vec & kVecDr);
    }
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * 8;
    if constexpr (kRowsWg > 1) {  // the workgroup's rows, in their order
      static_assert(NV == 1 || TPR >= 64, "narrow rows take one step");
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) join[threadIdx.x * 8 + e] = dw[k][e];
      __syncthreads();
      if (threadIdx.x < TPR)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float u = 0.f;
#pragma unroll 4
          for (int r = 0; r < kRowsWg; ++r) u += join[(r * TPR + threadIdx.x) * 8 + e];
          dw[k][e] = u;
        }
    }
    if (threadIdx.x < TPR)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < a.C) a.part[(int64_t)blockIdx.x * a.C + c + e] = dw[k][e];
  }
}

// dw = the sum of `n` rows of `part`: 64 columns a workgroup, its 16 waves a sixteenth of the rows each
template <typename TW>
__global__ __launch_bounds__(1024) void weight_sum(const float* part, int n, int C, TW* dw) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float u = 0.f;
  if (c < C)
#pragma unroll 4
    for (int i = wave; i < n; i += 16) u += part[(int64_t)i * C + c];
  lds[wave][lane] = u;
  __syncthreads();
  if (wave == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) u += lds[i][lane];
    dw[c] = from_f<TW>(u);
  }
}

constexpr int kMost = 65536;    // widest row
constexpr int kShares = 1024;   // at most so many workgroups share the sum of dw

int threads_per_row(int64_t C) {
  return C <= 32 ? 4 : C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 2048 ? 64 : C <= 8192 ? 256 : 1024;
}

int64_t shares(int64_t rows, int64_t C) {
  const int tpr = threads_per_row(C);
  const int per = tpr > 256 ? 1 : 256 / tpr;
  return std::min<int64_t>(ceil_div(rows, per), kShares);
}

#define SM_RMS_SHAPES(RUN)                                        \
  const int steps = (int)ceil_div(a.C, 8 * threads_per_row(a.C)); \
  switch (threads_per_row(a.C)) {                                 \
    case 4: RUN(4, 1)                                             \
    case 8: RUN(8, 1)                                             \
    case 16: RUN(16, 1)                                           \
    case 32: RUN(32, 1)                                           \
    case 64:                                                      \
      if (steps == 1) RUN(64, 1)                                  \
      if (steps == 2) RUN(64, 2)                                  \
      RUN(64, 4)                                                  \
    case 256:                                                     \
      if (steps <= 2) RUN(256, 2)                                 \
      if (steps == 3) RUN(256, 3)                                 \
      RUN(256, 4)                                                 \
    default:                                                      \
      if (steps <= 2) RUN(1024, 2)                                \
      if (steps <= 4) RUN(1024, 4)                                \
      RUN(1024, 8)                                                \
  }

template <typename T>
int launch_forward(const Args& a, bool q8, hipStream_t st) {
#define SM_RUN(TPR, NV)                                                                          \
  {                                                                                              \
    constexpr int threads = TPR > 256 ? TPR : 256;                                               \
    const dim3 grid = grid_of(ceil_div(a.rows, threads / TPR));                                  \
    if (q8) forward<T, TPR, NV, true><<<grid, threads, 0, st>>>(a);                              \
    else forward<T, TPR, NV, false><<<grid, threads, 0, st>>>(a);                                \
    return check_launch("rms_norm");                                                             \
  }
  SM_RMS_SHAPES(SM_RUN)
#undef SM_RUN
}

template <typename T>
int launch_backward(const Args& a, void* dw, hipStream_t st) {
  const int n = (int)shares(a.rows, a.C);
  auto rows = [&]() -> int {
#define SM_RUN(TPR, NV)                                                                  \
  {                                                                                      \
    backward<T, TPR, NV><<<dim3((unsigned)n), (TPR > 256 ? TPR : 256), 0, st>>>(a);      \
    return check_launch("rms_norm_backward");                                            \
  }
    SM_RMS_SHAPES(SM_RUN)
#undef SM_RUN
  };
  if (n > 0)
    if (const int rc = rows()) return rc;
  const dim3 grid((unsigned)ceil_div(a.C, 64));
  if (a.w_type == kF32) weight_sum<float><<<grid, 1024, 0, st>>>(a.part, n, a.C, static_cast<float*>(dw));
  else weight_sum<T><<<grid, 1024, 0, st>>>(a.part, n, a.C, static_cast<T*>(dw));
  return check_launch("rms_norm_backward weight");
}

// types of the residual stream and of the weight against x's; -1: not offered
int type_of(int dtype, int other) {
  return other == dtype ? kSame : other == SM_F32 ? kF32 : -1;
}
bool aligned(const void* p, int64_t stride, int64_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

int check(const char* what, int dtype, int64_t rows, int64_t C, float eps) {
  const std::string w(what);
  if (!valid_dtype(dtype)) return fail(SM_EDTYPE, w + ": float32, float16 or bfloat16 only");
  if (rows < 0 || C < 0) return fail(SM_EINVAL, w + ": negative size");
  if (C < 1 || C > kMost) return fail(SM_EINVAL, w + ": rows of 1 to 65536 values");
  if (rows >= (1ll << 31)) return fail(SM_EINVAL, w + ": 2^31 rows or more");
  if (!(eps >= 0.f) || eps > 3.4e38f) return fail(SM_EINVAL, w + ": eps must be finite and not negative");
  return SM_OK;
}

}  // namespace rms

int rms_norm_entry(const void* x, const void* residual, const void* weight, void* y, void* summed,
                   float* scales, int dtype, int res_dtype, int w_dtype, int64_t rows, int64_t C,
                   int64_t x_stride, int64_t r_stride, int64_t group, bool q8, float eps, void* stream) {
  using namespace rms;
  const char* what = q8 ? "rms_norm_e4m3" : "rms_norm";
  if (const int rc = rms::check(what, dtype, rows, C, eps)) return rc;
  Args a{};
  a.r_type = residual ? type_of(dtype, res_dtype) : kNone;
  a.w_type = type_of(dtype, w_dtype);
  if (a.r_type < 0 || a.w_type < 0)
    return fail(SM_EDTYPE, std::string(what) + ": residual and weight must have x's type or float32");
  if (q8 && group != 0 && group != 128)
    return fail(SM_EINVAL, "rms_norm_e4m3: a scale for each row (0) or each 128 values");
  if (x_stride < 0 || r_stride < 0) return fail(SM_EINVAL, std::string(what) + ": negative strides are not supported");
  if (rows == 0) return SM_OK;
  if (!x || !weight || !y || (residual && !summed) || (q8 && !scales))
    return fail(SM_EINVAL, std::string(what) + ": null pointer");
  const int es = elem_size(dtype), rsz = a.r_type == kF32 ? 4 : es;
  a.x = x;
  a.r = residual;
  a.w = weight;
  (q8 ? a.q : a.y) = y;
  a.s = summed;
  a.scale = scales;
  a.rows = rows;
  a.C = (int)C;
  a.xs = x_stride;
  a.rs = r_stride;
  a.groups = group == 0 ? 1 : (int)ceil_div(C, group);
  a.eps = eps;
  if (C % 8 == 0)
    a.vec = (aligned(x, x_stride, es) ? kVecX : 0) | (aligned(residual, r_stride, rsz) ? kVecR : 0) |
            (aligned(weight, 0, 1) ? kVecW : 0) |
            (reinterpret_cast<uintptr_t>(y) % (q8 ? 8 : 16) == 0 ? kVecY : 0) |
            (aligned(summed, C, rsz) ? kVecS : 0);
  SM_DISPATCH_DTYPE(dtype, T, return launch_forward<T>(a, q8, as_stream(stream)));
  return SM_OK;
}

int64_t rms_norm_workspace_bytes(int64_t rows, int64_t C) {
  if (rows <= 0 || C < 1 || C > rms::kMost) return 0;
  return rms::shares(rows, C) * C * 4;
}

int rms_norm_backward_entry(const void* summed, const void* weight, const void* dy, const void* dsummed,
                            void* dx, void* dresidual, void* dweight, int dtype, int s_dtype,
                            int w_dtype, int64_t rows, int64_t C, int64_t s_stride, int64_t dy_stride,
                            int64_t ds_stride, float eps, void* workspace, int64_t ws_bytes,
                            void* stream) {
  using namespace rms;
  const char* what = "rms_norm_backward";
  if (const int rc = rms::check(what, dtype, rows, C, eps)) return rc;
  Args a{};
  a.r_type = type_of(dtype, s_dtype);
  a.w_type = type_of(dtype, w_dtype);
  if (a.r_type < 0 || a.w_type < 0)
    return fail(SM_EDTYPE, "rms_norm_backward: stream and weight must have dy's type or float32");
  if (s_stride < 0 || dy_stride < 0 || ds_stride < 0)
    return fail(SM_EINVAL, "rms_norm_backward: negative strides are not supported");
  if (!dweight || (rows > 0 && (!summed || !weight || !dy || !dx)))
    return fail(SM_EINVAL, "rms_norm_backward: null pointer");
  if (dresidual && a.r_type != kF32)
    return fail(SM_EINVAL, "rms_norm_backward: a residual of x's type has x's gradient");
  if (rows > 0 && (workspace == nullptr || ws_bytes < rms_norm_workspace_bytes(rows, C)))
    return fail(SM_EINVAL, "rms_norm_backward: the workspace is smaller than "
                           "sm_rms_norm_backward_workspace_bytes()");
  if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
    return fail(SM_EINVAL, "rms_norm_backward: the workspace must be 4-byte aligned");
  const int es = elem_size(dtype), ss = a.r_type == kF32 ? 4 : es;
  a.w = weight;
  a.s = const_cast<void*>(summed);
  a.dy = dy;
  a.ds = dsummed;
  a.dx = dx;
  a.dr = dresidual;
  a.part = static_cast<float*>(workspace);
  a.rows = rows;
  a.C = (int)C;
  a.xs = s_stride;
  a.ys = dy_stride;
  a.zs = ds_stride;
  a.eps = eps;
  if (C % 8 == 0)
    a.vec = (aligned(weight, 0, 1) ? kVecW : 0) | (aligned(dy, dy_stride, es) ? kVecY : 0) |
            (aligned(summed, s_stride, ss) ? kVecS : 0) | (aligned(dsummed, ds_stride, ss) ? kVecZ : 0) |
            (aligned(dx, C, es) ? kVecD : 0) | (aligned(dresidual, C, 4) ? kVecDr : 0);
  SM_DISPATCH_DTYPE(dtype, T, return launch_backward<T>(a, dweight, as_stream(stream)));
  return SM_OK;
}

}  // namespace smcv
