// Cross attention, backward.  With p the weights (formed again from the saved logarithm of their
// sum), g the output's gradient and delta_i = sum_d g_id o_id:
//   dv_j = sum_i p_ij g_i      ds_ij = p_ij (g_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
// Two kernels, each with one side stationary in registers and the other streamed through LDS, so
// that every sum has one owner: no atomics, the same bits on every run, and the gradients of key
// heads shared by several query heads are summed in the owner's registers.  That forms the scores
// and their gradient twice (7 products where one kernel with atomic sums would have 5).  Bound by the
// matrix unit: 8160 x 8100 tokens, 16 heads, D=64, bf16: 1070 us for the 8 products that are executed
// in 16 bits, 1020 TFLOP/s.
//   attn_dq   a wave owns 32 query rows; writes dq, and per row delta and the logarithm in base 2.
//             In 16 bits g . o carries the rounding of o and of the weights that formed it, which
//             shifts a whole row of ds.  So the row's delta = sum_j p_ij (g_i . v_j) is summed in
//             fp32 beside the products for attn_dkv.  dq is formed with g . o and put right at the
//             end: exact ds sum to 0 over a row's keys, so what the rounded ones sum to, times
//             sum_j p_ij k_j (one product more, on the keys already read), is taken off.  That is
//             delta's error and, with it, the part of ds' own rounding that meets the keys' mean.
//   attn_dkv  a wave owns 32 keys; loops over the rows of all heads that share them
// fp16: ds would fall out of the type's range, so it enters its product with a power of two: one that
// brings the row's largest |g| into [1/2, 1) in attn_dq (a lane's scalar), the largest of the whole key
// head in attn_dkv, and about 2^8 more, since weights and values are mostly far below 1.  Where that
// passes the range (values of about 100 and more at large weights) the sum of the rounded ds is not
// finite: the workgroup forms its rows once more with 2^-8, which no finite input passes
// (|g . v - delta| <= 2 * 128 * 65504), and tells attn_dkv by the sign of its tile's maximum.  p enters
// dv times 2^14.  The factors are exact and are taken out of the fp32 sums at the end.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"

namespace smcv {
namespace attn {
namespace {

// How the waves of a workgroup share the work, by what the launch has to fill the card with:
//   kMany  four waves with 32 rows (dkv: keys) each
//   kSome  eight: two for each 32 rows, which take the even and the odd tiles of the other side
//   kFew   four (wide fp32: two) for the same 32 rows, which take the tiles in turn, each with its own
//          LDS and without barriers
// Waves that hold the same rows add their sums through LDS at the end, in one order.
enum { kMany = 0, kSome = 1, kFewRows = 2 };

template <typename T, int DP, int MODE> struct BCfg {
  static constexpr bool kWide = sizeof(T) == 4, kAlone = MODE == kFewRows;
  static constexpr int kTile = kWide || DP == 128 || kAlone ? 32 : 64;  // streamed rows
  static constexpr int kSets = kAlone ? 1 : 4;
  static constexpr int kParts = MODE == kMany ? 1 : MODE == kSome ? 2 : kWide && DP == 128 ? 2 : 4;
  static constexpr int kWaves = kSets * kParts, kThreads = 64 * kWaves, kTileRows = 32 * kSets;
  static constexpr int kCopiers = kAlone ? 64 : 256;  // threads that fetch a tile
  static constexpr int kTileBytes = kTile * DP * (int)sizeof(T);
  static constexpr int kBufQ = 2 * kTileBytes;         // keys and values
  static constexpr int kBufKv = 2 * kTileBytes + 512;  // rows, gradients, lse and delta
  static constexpr int kJoin = kParts > 1 ? kWaves * 32 * (DP + 4) * 4 : 0;
  static constexpr int kTilesQ = 2 * kBufQ * kParts;
  static constexpr int kMaskQ = 2 * kTile * 4 * kParts;  // 0 or -inf for each key of a buffer
  static constexpr int kFlagsQ = kJoin > kTilesQ + kMaskQ ? kJoin : kTilesQ + kMaskQ;  // fp16, two a wave
  static constexpr int kLdsQ = kFlagsQ + (std::is_same<T, __half>::value ? 2 * 4 * kWaves : 0);
  static constexpr int kLdsKv = kJoin > 2 * kBufKv * kParts ? kJoin : 2 * kBufKv * kParts;
  // waves a SIMD: two where the accumulators leave room for them
  static constexpr int kResident = kAlone || DP == 128 || (kWide && DP == 64) ? 1 : 2;
  static constexpr bool kHasSome = kWide ? DP <= 32 : DP <= 64;
};

// out(row of the workgroup, column, 4 values summed over the parts) for the waves' transposed results
template <typename T, int DP, int SETS, int PARTS, typename F>
__device__ __forceinline__ void join_columns(unsigned lds, int wave, int lane, int tid,
                                             const f32x16 (&acc)[DP / 32], F out) {
  constexpr int kPitch = (DP + 4) * 4, kWave = 32 * kPitch;
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
    lds_put(lds + wave * kWave + (lane & 31) * kPitch + column_at<T, DP>(i, lane >> 5) * 4,
            column_values<T, DP>(acc, i));
  __syncthreads();
  for (int p = tid; p < SETS * 32 * (DP / 4); p += SETS * PARTS * 64) {
    const int r = p / (DP / 4), d = 4 * (p % (DP / 4));
    const unsigned at = lds + (r >> 5) * kWave + (r & 31) * kPitch + d * 4;
    f32x4 v = lds_get<f32x4>(at);
#pragma unroll
    for (int w = 1; w < PARTS; ++w) {
      const f32x4 x = lds_get<f32x4>(at + w * SETS * kWave);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    out(r, d, v);
  }
}

// A wave's products go before the other waves' vector work where the loop is long enough for the
// waves to drift apart (4080 x 4080 tokens, 16 heads, D=64: 287 -> 276 us; wide heads, one wave a SIMD:
// 655 -> 664; D=32 198 -> 184, but its usual rows of 240, four tiles: 127 -> 131).
constexpr int kLongLoop = 8;
template <int DP> __device__ __forceinline__ void products_first(bool long_loop, bool on) {
  if constexpr (DP == 64)
    if (long_loop) {
      if (on) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
}

// the power of two that brings x into [1/2, 1), as an exponent; 0 for 0, infinities and NaN
__device__ __forceinline__ int down(float x) {
  const int e = (int)((__float_as_uint(x) >> 23) & 255);
  return e == 0 || e == 255 ? 0 : min(126 - e, 100);
}

// fp16: the powers of two that ds is formed with, first and once more
constexpr int kUpFirst = 8, kUpAgain = -8;

// whether `some` holds for a lane of the workgroup, the same answer for all its waves, once they are all
// here; `flags` is LDS that holds nothing else
template <int WAVES> __device__ __forceinline__ bool in_workgroup(bool some, unsigned flags, int wave, int lane) {
  const bool mine = __any(some);
  if (lane == 0) lds_put(flags + 4 * wave, (int)mine);
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any |= lds_get<int>(flags + 4 * w);
  return any != 0;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }  // not NaN either

template <typename T, int DP, bool KMASK, int MODE>
__global__ __launch_bounds__((BCfg<T, DP, MODE>::kThreads), (BCfg<T, DP, MODE>::kResident))
void attn_dq(Args a) {
  using C = BCfg<T, DP, MODE>;
  using TL = Tile<T, DP>;
  constexpr int KT = C::kTile, KB = KT / 32;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const unsigned id = xcd_id(a), bkv = a.by_row_tiles(id), b = a.by_kv(bkv);
  const int rt = id - bkv * a.row_tiles, kv = bkv - b * a.KV;
  const int set = C::kAlone ? 0 : wave & 3, part = C::kAlone ? wave : wave >> 2;
  const int ctid = C::kAlone ? lane : tid & 255, cwave0 = C::kAlone ? 0 : 64 * set;
  const int wg_row0 = rt * C::kTileRows, row0 = wg_row0 + 32 * set, row = row0 + (lane & 31);
  const int token = a.by_group(row), head = kv * a.G + row - token * a.G;
  const bool there = row < a.rows;

  Keys<KT, KMASK> keys(a, b, wg_row0, C::kTileRows);
  if (wg_row0 >= a.rows) keys.te = keys.tb;  // padding: its lse and delta alone

  const int64_t orow = (((int64_t)b * a.Lq + token) * a.H + head) * a.D;
  RowOps<T, DP> q, g;
  load_rows<T, DP>(q, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)token * a.qs[1] +
                          head * a.qs[2], there, half, a.D);
  load_rows<T, DP>(g, static_cast<const T*>(a.dout) + b * a.gs[0] + (int64_t)token * a.gs[1] +
                          head * a.gs[2], there, half, a.D);
  float delta = 0.f, most = 0.f;
  {
    RowOps<T, DP> o;
    load_rows<T, DP>(o, static_cast<const T*>(a.o) + orow, there, half, a.D);
#pragma unroll
    for (int s = 0; s < TL::kSteps; ++s)
#pragma unroll
      for (int e = 0; e < TL::kPer; ++e) {
        const float x = Mma<T>::get(g[s], e);
        delta = fmaf(x, Mma<T>::get(o[s], e), delta);
        most = fmaxf(most, fabsf(x));
      }
    delta = other_half_sum(delta);
    most = other_half_max(most);
  }
  const int64_t at = ((int64_t)b * a.KV + kv) * a.pad_rows + row;
  const float lse = there ? a.lse[((int64_t)b * a.KV + kv) * a.rows + row] : -INFINITY;
  // a row without keys, or past the end: +inf makes every weight that is formed from it 0
  const float lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
  if (half == 0 && part == 0) {
    a.row_lse[at] = lse2;
    if constexpr (sizeof(T) == 4) a.row_delta[at] = delta;
  }
  int shift = 0;
  if constexpr (kScaled) {
    float top = most;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
    if (lane == 0) lds_put(lds_addr(smem) + 4 * wave, top);
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 0; w < C::kSets; ++w) top = fmaxf(top, lds_get<float>(lds_addr(smem) + 4 * w));
      a.tile_max[((int64_t)b * a.KV + kv) * a.row_tiles + rt] = top;
    }
    __syncthreads();
    shift = down(most);
    delta = __builtin_ldexpf(delta, shift);
#pragma unroll
    for (int s = 0; s < TL::kSteps; ++s)
#pragma unroll
      for (int e = 0; e < TL::kPer; ++e)
        Mma<T>::put(g[s], e, __builtin_ldexpf(Mma<T>::get(g[s], e), shift));
  }

  const unsigned lds = lds_addr(smem) + part * 2 * C::kBufQ;
  const Reads<T, DP> from(lds, lane);
  const unsigned kb_row = (unsigned)a.ks[1] * sizeof(T), vb_row = (unsigned)a.vs[1] * sizeof(T);
  Stage<T, DP, KT, C::kCopiers> sk, sv;
  sk.init(ctid, a.D, [&](int r) { return r * kb_row; });
  sv.init(ctid, a.D, [&](int r) { return r * vb_row; });
  const uint64_t K = reinterpret_cast<uint64_t>(static_cast<const T*>(a.k) + b * a.ks[0] + kv * a.ks[2]);
  const uint64_t V = reinterpret_cast<uint64_t>(static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2]);
  const unsigned minus_inf = lds_addr(smem) + C::kTilesQ + part * 2 * KT * 4;
  auto put_mask = [&](int buf, uint64_t bits) {
    if (KMASK && cwave0 == 0 && lane < KT)
      lds_put(minus_inf + buf * KT * 4 + lane * 4, (bits >> lane) & 1 ? 0.f : -INFINITY);
  };
  auto copy = [&](int t, unsigned dst, uint64_t bits) {
    const uint64_t kp = K + (uint64_t)keys.first(t) * kb_row, vp = V + (uint64_t)keys.first(t) * vb_row;
    if (bits == keys.kAll) {
      sk.copy(kp, dst, cwave0);
      sv.copy(vp, dst + C::kTileBytes, cwave0);
    } else if (bits != 0) {
      sk.copy(kp, dst, cwave0, ctid, bits, kb_row);
      sv.copy(vp, dst + C::kTileBytes, cwave0, ctid, bits, vb_row);
    }
  };

  // dq, and (16-bit types) the weighted mean of the keys
  constexpr int N = sizeof(T) == 4 ? 1 : 2;
  f32x16 dq[N][DP / 32];
  float sum = 0.f;      // of p (g . v): delta again
  float rounded = 0.f;  // of ds as it enters the product
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[n][db][r] = 0.f;

  const bool long_loop = keys.te - keys.tb >= kLongLoop;
  int t = keys.tb + part;
  uint64_t bits = 0;
  int byte = 0;
  auto fetch_first = [&]() __attribute__((always_inline)) {
    if (t < keys.te) {
      bits = KMASK ? __ballot(keys.byte(t, lane)) : keys.by_length(t);
      copy(t, lds, bits);
      put_mask(0, bits);
    }
    if (KMASK) byte = keys.byte(t + C::kParts, lane);
  };
  fetch_first();
  int up = kScaled ? kUpFirst : 0;  // p, and with it ds and all sums, is formed times 2^up
  float from_lse = lse2 - (float)up;
  auto step = [&](auto buf) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(buf)::value * C::kBufQ;
    if (C::kAlone) wait_copies(); else publish();
    uint64_t next = 0;
    if (t + C::kParts < keys.te) {
      next = KMASK ? __ballot(byte) : keys.by_length(t + C::kParts);
      if (KMASK) byte = keys.byte(t + 2 * C::kParts, lane);
      copy(t + C::kParts, lds + (C::kBufQ - kBuf), next);
      put_mask(1 - decltype(buf)::value, next);
    }
    const uint64_t seen = bits;
    bits = next;
    if (seen == 0 || row0 >= a.rows) return;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const BandOf in(a, row0, keys.first(t) + 32 * kb, 32);
      const unsigned seen32 = (unsigned)(seen >> (32 * kb));
      if (!in.some || seen32 == 0) continue;
      f32x16 s;
      if constexpr (KMASK)
        s = mma_rows_masked<T, DP>(minus_inf + (decltype(buf)::value * KT + 32 * kb + 4 * half) * 4, from,
                                   kBuf, 32 * kb, q);
      else
        s = mma_rows<T, DP>(from, kBuf, 32 * kb, q);
      f32x16 ds[N];  // and the weights
      ds[0] = mma_rows<T, DP>(from, kBuf + C::kTileBytes, 32 * kb, g);
      const unsigned left = KMASK ? ~0u : seen32;
      if (!in.all || left != ~0u)
        mask_block(s, a.band > 0 ? band_bits(left, token - (keys.first(t) + 32 * kb), a.band) : left, half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -from_lse));
        if constexpr (N == 2) {
          sum = fmaf(p, ds[0][r], sum);
          ds[1][r] = p;
        }
        ds[0][r] = p * (ds[0][r] - delta);
      }
      if constexpr (N == 2)
#pragma unroll
        for (int r = 0; r < 16; r += 2) rounded = Mma<T>::add2(ds[0][r], ds[0][r + 1], rounded);
      products_first<DP>(long_loop, true);
      mma_transposed<T, DP, N>(dq, from, kBuf, 32 * kb, ds);
      products_first<DP>(long_loop, false);
    }
  };
  // every wave passes the same number of barriers: the parts' first tiles decide
  const int end = C::kAlone ? keys.te : keys.te + part;
  while (t < end) {
    step(std::integral_constant<int, 0>{});
    t += C::kParts;
    if (t >= end) break;
    step(std::integral_constant<int, 1>{});
    t += C::kParts;
  }
  const unsigned base = lds_addr(smem);
  // a ds past fp16's range has left the sum of the rounded ones infinite, or NaN
  if constexpr (kScaled)
    if (in_workgroup<C::kWaves>(!finite(rounded), base + C::kFlagsQ, wave, lane)) {
      up = kUpAgain;
      from_lse = lse2 - (float)up;
      sum = rounded = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) dq[n][db][r] = 0.f;
      t = keys.tb + part;
      fetch_first();
      while (t < end) {
        step(std::integral_constant<int, 0>{});
        t += C::kParts;
        if (t >= end) break;
        step(std::integral_constant<int, 1>{});
        t += C::kParts;
      }
    }
  if constexpr (C::kParts > 1) __syncthreads();
  if constexpr (N == 2) {
    sum = other_half_sum(sum);
    rounded = other_half_sum(rounded);
    if constexpr (C::kParts > 1) {
      const unsigned second = base + C::kWaves * 32 * 4;
      if (half == 0) {
        lds_put(base + (wave * 32 + lane) * 4, sum);
        lds_put(second + (wave * 32 + lane) * 4, rounded);
      }
      __syncthreads();
      sum = rounded = 0.f;
#pragma unroll
      for (int w = 0; w < C::kParts; ++w) {
        sum += lds_get<float>(base + ((w * C::kSets + set) * 32 + (lane & 31)) * 4);
        rounded += lds_get<float>(second + ((w * C::kSets + set) * 32 + (lane & 31)) * 4);
      }
      __syncthreads();
    }
    if constexpr (kScaled) {
      // attn_dkv forms ds with half the factor and the exact delta, and stays in range where this was
      // so here and delta's rounding moves ds by no more than 2^14
      const bool near = fabsf(sum - __builtin_ldexpf(delta, up)) <= 0x1p14f;
      if (in_workgroup<C::kWaves>(up == kUpAgain || !near, base + C::kFlagsQ + 4 * C::kWaves, wave, lane) && tid == 0) {
        float* top = a.tile_max + ((int64_t)b * a.KV + kv) * a.row_tiles + rt;
        *top = -*top;
      }
    }
    if (half == 0 && part == 0) a.row_delta[at] = __builtin_ldexpf(sum, -shift - up);
    const float off = __builtin_ldexpf(-rounded, -up);  // against weights that carry 2^up as well
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[0][db][r] = fmaf(off, dq[1][db][r], dq[0][db][r]);
  }
  const float by = __builtin_ldexpf(a.scale, -shift - up);
  if constexpr (C::kParts > 1) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[0][db][r] *= by;
    join_columns<T, DP, C::kSets, C::kParts>(base, wave, lane, tid, dq[0], [&](int r, int d, f32x4 v) {
      const int grow = wg_row0 + r, i = a.by_group(grow);
      if (grow < a.rows && d < a.D)
        store4<T>(static_cast<T*>(a.dq) + (((int64_t)b * a.Lq + i) * a.H + kv * a.G + grow - i * a.G) * a.D + d, v);
    });
  } else {
    if (!there) return;
    store_columns<T, DP>(static_cast<T*>(a.dq) + orow, dq[0], by, half, a.D);
  }
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__((BCfg<T, DP, MODE>::kThreads), (BCfg<T, DP, MODE>::kResident))
void attn_dkv(Args a) {
  using C = BCfg<T, DP, MODE>;
  constexpr int RT = C::kTile, RB = RT / 32;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  constexpr float kUp = kScaled ? 14.f : 0.f;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const unsigned id = xcd_id(a), bkv = a.by_key_tiles(id), b = a.by_kv(bkv);
  const int jt = id - bkv * a.key_tiles, kv = bkv - b * a.KV;
  const int set = C::kAlone ? 0 : wave & 3, part = C::kAlone ? wave : wave >> 2;
  const int ctid = C::kAlone ? lane : tid & 255, cwave0 = C::kAlone ? 0 : 64 * set;
  const int wg_j0 = jt * C::kTileRows, j0 = wg_j0 + 32 * set, j = j0 + (lane & 31);
  const int keys = a.lengths ? min(max(a.lengths[b], 0), a.Lk) : a.Lk;
  auto counts = [&](int key) {  // something may attend to the key
    return key < keys && (a.mask == nullptr || a.mask[(int64_t)b * a.Lk + key] != 0);
  };
  const bool there = counts(j);

  RowOps<T, DP> k, v;
  load_rows<T, DP>(k, static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)j * a.ks[1] +
                          kv * a.ks[2], there, half, a.D);
  load_rows<T, DP>(v, static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)j * a.vs[1] +
                          kv * a.vs[2], there, half, a.D);

  // rows of the heads that share these keys: all, or those whose band reaches them
  int64_t rlo = 0, rhi = a.rows;
  if (a.band > 0) {
    rlo = min((int64_t)a.rows, (int64_t)wg_j0 * a.G);
    rhi = min((int64_t)a.rows, ((int64_t)min(wg_j0 + C::kTileRows, a.Lk) - 1 + a.band) * a.G);
  }
  if (wg_j0 >= keys) rhi = rlo;  // nothing attends to them: their gradients are 0
  const int tb = (int)(rlo / RT), te = rhi > rlo ? (int)((rhi + RT - 1) / RT) : tb;

  const float* lse = a.row_lse + ((int64_t)b * a.KV + kv) * a.pad_rows;
  const float* delta = a.row_delta + ((int64_t)b * a.KV + kv) * a.pad_rows;
  int shift = 0;
  if constexpr (kScaled) {
    const float* tm = a.tile_max + ((int64_t)b * a.KV + kv) * a.row_tiles;
    float top = 0.f;
    bool far = false;
    for (int i = lane; i < a.row_tiles; i += 64) {
      top = fmaxf(top, fabsf(tm[i]));
      far |= tm[i] < 0.f;
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
    shift = __builtin_amdgcn_readfirstlane(down(top)) + (__any(far) ? kUpAgain : kUpFirst) - 1;
  }

  const unsigned lds = lds_addr(smem) + part * 2 * C::kBufKv;
  const Reads<T, DP> from(lds, lane);
  const uint64_t Q = reinterpret_cast<uint64_t>(static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)kv * a.G * a.qs[2]);
  const uint64_t GO = reinterpret_cast<uint64_t>(static_cast<const T*>(a.dout) + b * a.gs[0] + (int64_t)kv * a.G * a.gs[2]);
  // Row t RT + r is token (t RT + r) / G: where G divides RT the offsets from the tile's first token
  // are the same in every tile.
  const bool regular = (RT & (a.G - 1)) == 0 && (a.G & (a.G - 1)) == 0;
  auto row_at = [&](int row, int token0, const int64_t* st) -> unsigned {
    const int token = a.by_group(row), g = row - token * a.G;
    return ((token - token0) * (unsigned)st[1] + g * (unsigned)st[2]) * (unsigned)sizeof(T);
  };
  using SG = Stage<T, DP, RT, C::kCopiers>;
  SG sq, sg;
  sq.init(ctid, a.D, [&](int r) { return row_at(r, 0, a.qs); });
  sg.init(ctid, a.D, [&](int r) { return row_at(r, 0, a.gs); });
  auto copy = [&](int t, unsigned dst) {
    const int token0 = a.by_group(t * RT);
    const uint64_t qp = Q + (uint64_t)token0 * a.qs[1] * sizeof(T), gp = GO + (uint64_t)token0 * a.gs[1] * sizeof(T);
    if (regular && (t + 1) * RT <= a.rows) {
      sq.copy(qp, dst, cwave0);
      sg.copy(gp, dst + C::kTileBytes, cwave0);
    } else {  // rows past the end read the tile's first: their weights are 0
      auto at = [&](const int64_t* st) {
        return [=, &a](int it, unsigned o) {
          const int r = SG::row_of(it, ctid), row = t * RT + r;
          return o - row_at(r, 0, st) + row_at(row < a.rows ? row : t * RT, token0, st);
        };
      };
      sq.copy(qp, dst, cwave0, at(a.qs));
      sg.copy(gp, dst + C::kTileBytes, cwave0, at(a.gs));
    }
    // RT logarithms, then RT deltas (the rows are padded to whole tiles there)
    const uint64_t lp = reinterpret_cast<uint64_t>(lse + t * RT), dp = reinterpret_cast<uint64_t>(delta + t * RT);
    if ((C::kAlone || set == 0) && lane < RT) copy4(lp, lane * 4, dst + 2 * C::kTileBytes);
    if ((C::kAlone || set == 1) && lane < RT) copy4(dp, lane * 4, dst + 2 * C::kTileBytes + RT * 4);
  };

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;

  const bool long_loop = te - tb >= kLongLoop;
  int t = tb + part;
  if (t < te) copy(t, lds);
  auto step = [&](auto buf) __attribute__((always_inline)) {
    constexpr int kAt = decltype(buf)::value * C::kBufKv;
    if (C::kAlone) wait_copies(); else publish();
    if (t + C::kParts < te) copy(t + C::kParts, lds + (C::kBufKv - kAt));
    const unsigned st = lds + kAt + 2 * C::kTileBytes;
    if (j0 >= keys || t >= te) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      // row r is inside key j's band iff 0 <= r - j G < band G
      bool edge = false;
      if (a.band > 0) {
        const int64_t r0 = (int64_t)t * RT + 32 * rb, r1 = r0 + 31;
        const int64_t first = (int64_t)j0 * a.G, last = ((int64_t)j0 + 31 + a.band) * a.G - 1;
        if (r1 < first || r0 > last) continue;
        edge = r0 < (int64_t)(j0 + 31) * a.G || r1 >= ((int64_t)j0 + a.band) * a.G;
      }
      f32x16 p = mma_rows<T, DP>(from, kAt, 32 * rb, k);
      f32x16 ds = mma_rows<T, DP>(from, kAt + C::kTileBytes, 32 * rb, v);
      if (edge) {
        const int64_t first = (int64_t)j * a.G - ((int64_t)t * RT + 32 * rb);  // in the block
        const int64_t after = first + (int64_t)a.band * a.G;
        const unsigned upto = after >= 32 ? ~0u : after <= 0 ? 0u : (1u << after) - 1;
        const unsigned past = first <= 0 ? ~0u : first >= 32 ? 0u : ~0u << first;
        mask_block(p, upto & past, half);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = lds_get<f32x4>(st + (32 * rb + 8 * g + 4 * half) * 4);
        const f32x4 d4 = lds_get<f32x4>(st + RT * 4 + (32 * rb + 8 * g + 4 * half) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          // a masked score of -inf against +inf (a row without keys) is still -inf
          const float w = __builtin_amdgcn_exp2f(fmaf(p[r], a.c, -l4[e]));
          float x = w * (ds[r] - d4[e]);
          if constexpr (kScaled) {
            x = __builtin_ldexpf(x, shift);
            p[r] = __builtin_ldexpf(w, (int)kUp);
          } else {
            p[r] = w;
          }
          ds[r] = x;
        }
      }
      products_first<DP>(long_loop, true);
      mma_transposed<T, DP>(dv, from, kAt + C::kTileBytes, 32 * rb, p);
      mma_transposed<T, DP>(dk, from, kAt, 32 * rb, ds);
      products_first<DP>(long_loop, false);
    }
  };
  const int end = C::kAlone ? te : te + part;
  while (t < end) {
    step(std::integral_constant<int, 0>{});
    t += C::kParts;
    if (t >= end) break;
    step(std::integral_constant<int, 1>{});
    t += C::kParts;
  }
  // a key that nothing attends to gets 0, whatever the zero row that stood for it gave
  const float by_k = __builtin_ldexpf(a.scale, -shift), by_v = kScaled ? 0x1p-14f : 1.f;
  if constexpr (C::kParts > 1) {
    auto store = [&](void* to, float by) {
      return [&, to, by](int r, int d, f32x4 v) {
        const int key = wg_j0 + r;
        if (key >= a.Lk || d >= a.D) return;
        const bool some = counts(key);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = some ? v[e] * by : 0.f;
        store4<T>(static_cast<T*>(to) + (((int64_t)b * a.Lk + key) * a.KV + kv) * a.D + d, v);
      };
    };
    const unsigned base = lds_addr(smem);
    __syncthreads();
    join_columns<T, DP, C::kSets, C::kParts>(base, wave, lane, tid, dv, store(a.dv, by_v));
    __syncthreads();
    join_columns<T, DP, C::kSets, C::kParts>(base, wave, lane, tid, dk, store(a.dk, by_k));
  } else {
    if (j >= a.Lk) return;
    const int64_t out = (((int64_t)b * a.Lk + j) * a.KV + kv) * a.D;
    if (!there) {
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;
    }
    store_columns<T, DP>(static_cast<T*>(a.dv) + out, dv, by_v, half, a.D);
    store_columns<T, DP>(static_cast<T*>(a.dk) + out, dk, by_k, half, a.D);
  }
}

template <typename T, int DP, bool KMASK, int MODE>
int launch_dq(Args a, hipStream_t st) {
  using C = BCfg<T, DP, MODE>;
  static std::atomic<unsigned long long> done{0};
  const void* kern = reinterpret_cast<const void*>(&attn_dq<T, DP, KMASK, MODE>);
  if (const int rc = ensure_lds_limit(kern, C::kLdsQ, stream_device(st), done)) return rc;
  const int64_t grid = (int64_t)a.B * a.KV * a.row_tiles;
  return launch_all(a, grid, "cross_attention_backward dq", [&](dim3 part) {
    attn_dq<T, DP, KMASK, MODE><<<part, C::kThreads, C::kLdsQ, st>>>(a);
  });
}

template <typename T, int DP, int MODE>
int launch_dkv(Args a, hipStream_t st) {
  using C = BCfg<T, DP, MODE>;
  static std::atomic<unsigned long long> done{0};
  const void* kern = reinterpret_cast<const void*>(&attn_dkv<T, DP, MODE>);
  if (const int rc = ensure_lds_limit(kern, C::kLdsKv, stream_device(st), done)) return rc;
  a.key_tiles = (int)ceil_div(a.Lk, C::kTileRows);
  a.by_key_tiles = Divide(a.key_tiles);
  const int64_t grid = (int64_t)a.B * a.KV * a.key_tiles;
  return launch_all(a, grid, "cross_attention_backward dk, dv", [&](dim3 part) {
    attn_dkv<T, DP, MODE><<<part, C::kThreads, C::kLdsKv, st>>>(a);
  });
}

// `wgs`: workgroups of 128 rows.  Up to a quarter of the compute units: 32-row workgroups (8 x 255 x 301
// tokens, 4 heads over 2, fp32: both kernels 145 -> 45 us); up to one each: eight waves (2 x 1021 x 4093,
// 16 over 4, D=64: 230 -> 178 us), or up to half 32-row workgroups where eight waves do not fit
int mode_of(int64_t wgs, bool has_some, bool has_few) {
  if (!has_few) return kMany;
  if (wgs <= kCus / 4) return kFewRows;
  if (has_some) return wgs <= kCus ? kSome : kMany;
  return wgs <= kCus / 2 ? kFewRows : kMany;
}

template <typename T, int DP>
int launch(Args a, hipStream_t st) {
  const int64_t bkv = (int64_t)a.B * a.KV;
  if (bkv * (a.pad_rows / 32) > 0x7fffffffll || bkv * ceil_div(a.Lk, 32) > 0x7fffffffll)
    return fail(SM_EINVAL, "cross_attention_backward: too many row tiles");
  constexpr bool some = BCfg<T, DP, kMany>::kHasSome;
  a.row_tiles = a.pad_rows / kRows;
  if (a.row_tiles > 0) {
    const int mode = mode_of(bkv * a.row_tiles, some, true);
    if (mode == kFewRows) a.row_tiles = a.pad_rows / 32;
    a.by_row_tiles = Divide(a.row_tiles);
    const bool km = a.mask != nullptr;
    int rc = SM_OK;
    if (mode == kFewRows)
      rc = km ? launch_dq<T, DP, true, kFewRows>(a, st) : launch_dq<T, DP, false, kFewRows>(a, st);
    else if (mode == kMany)
      rc = km ? launch_dq<T, DP, true, kMany>(a, st) : launch_dq<T, DP, false, kMany>(a, st);
    else if constexpr (some)
      rc = km ? launch_dq<T, DP, true, kSome>(a, st) : launch_dq<T, DP, false, kSome>(a, st);
    if (rc) return rc;
  }
  if (a.Lk > 0 && bkv > 0) {
    // (32 wide fp32 keys in each of two waves would not fit their registers)
    constexpr bool few = sizeof(T) == 2 || DP < 128;
    const int mode = mode_of(bkv * ceil_div(a.Lk, kRows), some, few);
    if constexpr (few)
      if (mode == kFewRows) return launch_dkv<T, DP, kFewRows>(a, st);
    if (mode == kMany) return launch_dkv<T, DP, kMany>(a, st);
    if constexpr (some) return launch_dkv<T, DP, kSome>(a, st);
  }
  return SM_OK;
}

template <typename T>
int by_width(const Args& a, hipStream_t st) {
  if (a.D <= 32) return launch<T, 32>(a, st);
  if (a.D <= 64) return launch<T, 64>(a, st);
  return launch<T, 128>(a, st);
}

}  // namespace

// per row its logarithm and delta, and room for a maximum of each 32 rows
int64_t bwd_workspace_bytes(int64_t B, int64_t Lq, int64_t H, int64_t KV) {
  if (B <= 0 || Lq <= 0 || H <= 0 || KV <= 0 || H % KV != 0) return 0;
  const int64_t pad = ceil_div(Lq * (H / KV), kRows) * kRows;
  return B * KV * (2 * pad + pad / 32) * 4;
}

int bwd_entry(Args& a, int dtype, void* workspace, int64_t ws_bytes, hipStream_t st) {
  a.pad_rows = (int)(ceil_div(a.rows, kRows) * kRows);
  const int64_t n = (int64_t)a.B * a.KV * a.pad_rows;
  if (n > 0 && (workspace == nullptr || ws_bytes < (2 * n + n / 32) * 4))
    return fail(SM_EINVAL, "cross_attention_backward: the workspace is smaller than "
                           "sm_cross_attention_backward_workspace_bytes()");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(SM_EINVAL, "cross_attention_backward: the workspace must be 16-byte aligned");
  a.row_lse = static_cast<float*>(workspace);
  a.row_delta = a.row_lse + n;
  a.tile_max = a.row_delta + n;
  SM_DISPATCH_DTYPE(dtype, T, return by_width<T>(a, st));
  return SM_OK;
}

}  // namespace attn
}  // namespace smcv
