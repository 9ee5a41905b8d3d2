// Cross attention, forward: o_i = sum_j p_ij v_j, p = softmax over the keys j that token i may see.
//
// One pass over the keys with the running maximum m and sum l of each query's softmax: scores,
// weights and statistics stay in registers (attn_common.h has the layout), keys and values pass
// through LDS once a workgroup.  m is raised lazily: while a tile's scores exceed it by less than
// 2^8 in weight, the weights are formed against the old m and the accumulators are not rescaled
// (they are divided by l, formed against the same m, at the end; weights up to 2^8 lose nothing in
// any of the types).
//
// Bound by the matrix unit for wide heads (8160 x 8100 tokens, 16 heads, D=128, bf16: 530 us, 1020
// TFLOP/s; 455 us without any softmax work, which is what large library products reach too), by the
// exponentials and the other vector work for narrow ones (D=32: 212 us), by HBM for single tokens (four
// of 8 to 16 thousand keys, 8 key heads, D=128: 201 MB in 45 us).  Four waves of 32 rows: 64-row
// workgroups copy the keys too often (854 us at D=128), 256-row ones wait for each other (553 us, and
// 115 us instead of 92 for 540 rows of 960 in a band of 192).
#include <algorithm>
#include <type_traits>

#include "attn_common.h"

namespace smcv {
namespace attn {

namespace {

// How the waves of a workgroup share the work:
//   FEW       32 query rows (single tokens with shared heads, short launches): all waves hold the same
//             rows and take the key tiles in turn, each with its own LDS and without barriers
//   GROUPS    1: four waves, 32 rows each; 2: eight waves, 32 rows for each pair, which takes the even
//             and the odd key tiles
// Waves that hold the same rows join their sums and statistics through LDS at the end.
template <typename T, int DP, bool FEW, int GROUPS> struct Cfg {
  static constexpr int kTile = sizeof(T) == 4 ? 32 : (FEW && DP == 128) ? 32 : 64;  // keys
  static constexpr int kWaves = FEW ? (sizeof(T) == 4 && DP == 128 ? 2 : 4) : 4 * GROUPS;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kParts = FEW ? kWaves : GROUPS;  // of the keys
  static constexpr int kTileBytes = kTile * DP * (int)sizeof(T);
  static constexpr int kBufBytes = 2 * kTileBytes;  // keys and values
  // two buffers a part; the join needs a wave's sums and statistics each
  static constexpr int kTiles = 2 * kBufBytes * kParts;
  static constexpr int kMask = 2 * kTile * 4 * kParts;  // 0 or -inf for each key of a buffer
  static constexpr int kJoin = kParts > 1 ? kWaves * (32 * (DP + 4) * 4 + 256) : 0;
  static constexpr int kLds = kTiles + kMask > kJoin ? kTiles + kMask : kJoin;
};

constexpr float kLazy = 8.f;
// fp16 weights are formed times 2^7, so that with the lazy maximum they take the type's whole range (at
// most 2^15): each is rounded within 2^-32 of the largest, where 2^-25 each was lost, which 65 thousand
// keys far below one add up to 2e-3 of the output.  The sum of the weights carries the same factor.
template <typename T> constexpr float kWeightUp = std::is_same<T, __half>::value ? 7.f : 0.f;

template <typename T, int DP, bool KMASK, bool FEW, int GROUPS>
__global__ __launch_bounds__((Cfg<T, DP, FEW, GROUPS>::kThreads), (FEW || (sizeof(T) == 4 && DP == 128) ? 1 : 2))
void attn_fwd(Args a) {
  using C = Cfg<T, DP, FEW, GROUPS>;
  constexpr int KT = C::kTile, KB = KT / 32, kTileRows = FEW ? kFew : kRows;
  constexpr int kCopiers = FEW ? 64 : 256;  // threads that fetch a tile
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = FEW ? wave : wave >> 2;  // of the keys
  const int ctid = FEW ? lane : tid & 255, cwave0 = FEW ? 0 : (wave & 3) * 64;

  const unsigned id = xcd_id(a);
  // neighbours share the keys of a head, or (few rows) read the same tokens of neighbouring heads
  const unsigned u = FEW ? a.by_kv(id) : a.by_row_tiles(id);
  const int in_u = id - u * (FEW ? a.KV : a.row_tiles);
  const unsigned w = FEW ? a.by_row_tiles(u) : a.by_splits(u);
  const int in_w = u - w * (FEW ? a.row_tiles : a.splits);
  const unsigned b = FEW ? a.by_splits(w) : a.by_kv(w);
  const int in_b = w - b * (FEW ? a.splits : a.KV);
  const int rt = FEW ? in_w : in_u, split = FEW ? in_b : in_w, kv = FEW ? in_u : in_b;

  const int wg_row0 = rt * kTileRows;
  const int row0 = wg_row0 + (FEW ? 0 : 32 * (wave & 3));  // of this wave
  const int row = row0 + (lane & 31);                      // of this lane
  const int token = a.by_group(row), head = kv * a.G + row - token * a.G;
  const bool there = row < a.rows;

  Keys<KT, KMASK> keys(a, b, wg_row0, kTileRows);
  if (a.splits > 1) {
    const int per = (keys.te - keys.tb + a.splits - 1) / a.splits;
    keys.tb += split * per;
    keys.te = min(keys.te, keys.tb + per);
  }

  RowOps<T, DP> q;
  load_rows<T, DP>(q, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)token * a.qs[1] +
                          head * a.qs[2], there, half, a.D);

  const unsigned lds = lds_addr(smem) + part * 2 * C::kBufBytes;
  const Reads<T, DP> from(lds, lane);
  const unsigned kb_row = (unsigned)a.ks[1] * sizeof(T), vb_row = (unsigned)a.vs[1] * sizeof(T);
  Stage<T, DP, KT, kCopiers> sk, sv;
  sk.init(ctid, a.D, [&](int r) { return r * kb_row; });
  sv.init(ctid, a.D, [&](int r) { return r * vb_row; });
  const uint64_t K = reinterpret_cast<uint64_t>(static_cast<const T*>(a.k) + b * a.ks[0] + kv * a.ks[2]);
  const uint64_t V = reinterpret_cast<uint64_t>(static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2]);
  const unsigned minus_inf = lds_addr(smem) + C::kTiles + part * 2 * KT * 4;
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

  f32x16 o[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -INFINITY, l = 0.f;

  constexpr int kStep = C::kParts;
  int t = keys.tb + part;
  uint64_t bits = 0;
  int byte = 0;
  if (t < keys.te) {
    bits = KMASK ? __ballot(keys.byte(t, lane)) : keys.by_length(t);
    copy(t, lds, bits);
    put_mask(0, bits);
  }
  if (KMASK) byte = keys.byte(t + kStep, lane);

  auto step = [&](auto buf) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(buf)::value * C::kBufBytes;
    // this tile is in LDS, and nobody reads the other buffer any more
    if (FEW) wait_copies(); else publish();
    uint64_t next = 0;
    if (t + kStep < keys.te) {
      next = KMASK ? __ballot(byte) : keys.by_length(t + kStep);
      if (KMASK) byte = keys.byte(t + 2 * kStep, lane);
      copy(t + kStep, lds + (C::kBufBytes - kBuf), next);
      put_mask(1 - decltype(buf)::value, next);
    }
    const uint64_t seen = bits;
    bits = next;
    // (also a group's turn past the last tile, and a wave whose rows lie past the end)
    if (seen == 0 || row0 >= a.rows) return;
    const BandOf in(a, row0, keys.first(t), KT);
    if (!in.some) return;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      if constexpr (KMASK)
        s[kb] = mma_rows_masked<T, DP>(minus_inf + (decltype(buf)::value * KT + 32 * kb + 4 * half) * 4, from,
                                       kBuf, 32 * kb, q);
      else
        s[kb] = mma_rows<T, DP>(from, kBuf, 32 * kb, q);
    if (!in.all || (!KMASK && seen != keys.kAll))
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        unsigned w = KMASK ? ~0u : (unsigned)(seen >> (32 * kb));
        if (a.band > 0) w = band_bits(w, token - (keys.first(t) + 32 * kb), a.band);
        mask_block(s[kb], w, half);
      }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
    mx = other_half_max(mx);
    if (__any((mx - m) * a.c > kLazy)) {
      const float mn = fmaxf(m, mx);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
      l *= f;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= f;
      m = mn;
    }
    const float mc = m == -INFINITY ? 0.f : fmaf(m, a.c, -kWeightUp<T>);
    float part_l[2] = {0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], a.c, -mc));
        part_l[r & 1] += s[kb][r];
      }
    l += part_l[0] + part_l[1];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) mma_transposed<T, DP>(o, from, kBuf + C::kTileBytes, 32 * kb, s[kb]);
  };
  // every wave passes the same number of barriers: the groups' first tiles decide
  const int end = FEW ? keys.te : keys.te + part;
  while (t < end) {
    step(std::integral_constant<int, 0>{});
    t += kStep;
    if (t >= end) break;
    step(std::integral_constant<int, 1>{});
    t += kStep;
  }
  l = other_half_sum(l);

  if constexpr (C::kParts > 1) {
    // join the waves that hold the same rows: rows x DP partial sums and statistics of each wave
    constexpr int kPitch = (DP + 4) * 4, kWaveBytes = 32 * kPitch + 256;
    constexpr int kSets = FEW ? 1 : 4;  // of rows
    static_assert(C::kWaves * kWaveBytes == C::kJoin, "the join's LDS");
    const unsigned base = lds_addr(smem);
    __syncthreads();
    const unsigned mine = base + wave * kWaveBytes;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
      lds_put(mine + (lane & 31) * kPitch + column_at<T, DP>(i, half) * 4, column_values<T, DP>(o, i));
    if (half == 0) {
      lds_put(mine + 32 * kPitch + lane * 4, m);
      lds_put(mine + 32 * kPitch + 128 + lane * 4, l);
    }
    __syncthreads();
    for (int p = tid; p < kTileRows * (DP / 4); p += C::kThreads) {
      const int tr = p / (DP / 4), r = tr & 31, d = 4 * (p % (DP / 4)), grow = wg_row0 + tr;
      if (grow >= a.rows || d >= a.D) continue;
      const unsigned set = base + (tr >> 5) * kWaveBytes;
      float top = -INFINITY, mw[C::kParts];
#pragma unroll
      for (int w = 0; w < C::kParts; ++w) {
        mw[w] = lds_get<float>(set + w * kSets * kWaveBytes + 32 * kPitch + r * 4);
        top = fmaxf(top, mw[w]);
      }
      const float from_m = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < C::kParts; ++w) {
        const unsigned at = set + w * kSets * kWaveBytes;
        const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw[w] - from_m) * a.c);
        sum = fmaf(f, lds_get<float>(at + 32 * kPitch + 128 + r * 4), sum);
        const f32x4 x = lds_get<f32x4>(at + r * kPitch + d * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(f, x[e], v[e]);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= inv;
      const float lse = sum == 0.f ? -INFINITY : fmaf(from_m, a.c, __builtin_amdgcn_logf(sum) - kWeightUp<T>) * kLn2;
      const int64_t ra = ((int64_t)b * a.KV + kv) * a.rows + grow;
      if (a.splits > 1) {
        const int64_t ps = (int64_t)split * a.B * a.KV * a.rows + ra;
        *reinterpret_cast<f32x4*>(a.part_o + ps * a.D + d) = v;
        if (d == 0) a.part_l[ps] = lse;
      } else {
        const int i = a.by_group(grow);
        store4<T>(static_cast<T*>(a.out) + (((int64_t)b * a.Lq + i) * a.H + kv * a.G + grow - i * a.G) * a.D + d, v);
        if (d == 0 && a.lse) a.lse[ra] = lse;
      }
    }
  } else {
    if (!there) return;
    const int64_t at = ((int64_t)b * a.KV + kv) * a.rows + row;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float lse = l == 0.f ? -INFINITY : fmaf(m, a.c, __builtin_amdgcn_logf(l) - kWeightUp<T>) * kLn2;
    // wide fp32 rows alone split their keys in this shape: the others' launches of so few workgroups
    // have eight waves each (by_rows)
    if constexpr (sizeof(T) == 4 && DP == 128)
      if (a.splits > 1) {
        const int64_t ps = (int64_t)split * a.B * a.KV * a.rows + at;
        store_columns<T, DP, float>(a.part_o + ps * a.D, o, inv, half, a.D);
        if (half == 0) a.part_l[ps] = lse;
        return;
      }
    store_columns<T, DP>(static_cast<T*>(a.out) + (((int64_t)b * a.Lq + token) * a.H + head) * a.D,
                         o, inv, half, a.D);
    if (half == 0 && a.lse) a.lse[at] = lse;
  }
}

// The splits' outputs, each normalised over its own keys, weighted by their sums: one thread for 4
// values of a row.
template <typename T>
__global__ __launch_bounds__(256) void attn_join(Args a) {
  const int per = a.D / 4;
  const int64_t n = (int64_t)a.B * a.KV * a.rows;
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= n * per) return;
  const int64_t r = p / per;
  const int d = 4 * (int)(p % per);
  constexpr int kAtOnce = 8;  // splits whose loads are in flight together
  float top = -INFINITY, base = 0.f, sum = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += kAtOnce) {
    float l[kAtOnce];
    f32x4 x[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = (int64_t)min(s0 + i, a.splits - 1) * n + r;
      l[i] = a.part_l[at];
      x[i] = *reinterpret_cast<const f32x4*>(a.part_o + at * a.D + d);
    }
    float most = top;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (s0 + i >= a.splits) l[i] = -INFINITY;
      most = fmaxf(most, l[i]);
    }
    base = most == -INFINITY ? 0.f : most;
    const float keep = __builtin_amdgcn_exp2f((top - base) * kLog2e);
    top = most;
    sum *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= keep;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float w = __builtin_amdgcn_exp2f((l[i] - base) * kLog2e);
      sum += w;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(w, x[i][e], v[e]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= inv;
  const int row = (int)(r % a.rows), kv = (int)(r / a.rows % a.KV);
  const int64_t tok = r / a.rows / a.KV * a.Lq + row / a.G;
  store4<T>(static_cast<T*>(a.out) + (tok * a.H + kv * a.G + row % a.G) * a.D + d, v);
  if (d == 0 && a.lse) a.lse[r] = sum == 0.f ? -INFINITY : base + __builtin_amdgcn_logf(sum) * kLn2;
}

// 32-row workgroups whose waves split the keys: a single tile of rows, or a launch whose 128-row
// workgroups would fill no more than a quarter of the compute units
// (8 sequences of 255 rows, 301 keys, 4 heads over 2, fp32: 31 -> 14 us)
bool few_rows(int64_t B, int64_t KV, int64_t rows) {
  return rows <= kFew || B * KV * ceil_div(rows, kRows) <= kCus / 4;
}

template <typename T, int DP, bool KMASK, bool FEW, int GROUPS>
int launch(Args a, hipStream_t st) {
  using C = Cfg<T, DP, FEW, GROUPS>;
  static std::atomic<unsigned long long> done{0};
  const void* kern = reinterpret_cast<const void*>(&attn_fwd<T, DP, KMASK, FEW, GROUPS>);
  if (const int rc = ensure_lds_limit(kern, C::kLds, stream_device(st), done)) return rc;
  const int64_t grid = (int64_t)a.B * a.KV * a.splits * a.row_tiles;
  if (grid > 0x7fffffffll) return fail(SM_EINVAL, "cross_attention: too many row tiles");
  if (const int rc = launch_all(a, grid, "cross_attention", [&](dim3 part) {
        attn_fwd<T, DP, KMASK, FEW, GROUPS><<<part, C::kThreads, C::kLds, st>>>(a);
      })) return rc;
  if (a.splits > 1) {
    const int64_t n = (int64_t)a.B * a.KV * a.rows * (a.D / 4);
    attn_join<T><<<dim3((unsigned)ceil_div(n, 256)), 256, 0, st>>>(a);
    return check_launch("cross_attention join");
  }
  return SM_OK;
}

template <typename T, int DP, bool KMASK>
int by_rows(const Args& a, hipStream_t st) {
  if (few_rows(a.B, a.KV, a.rows)) return launch<T, DP, KMASK, true, 1>(a, st);
  // a launch that leaves a compute unit one workgroup gives it eight waves instead of four (wide fp32
  // rows need the registers of four): 2 x 1021 rows, 4093 keys, 16 heads over 4, D=64: 105 -> 73 us
  if constexpr (sizeof(T) == 2 || DP < 128) {
    const int64_t wgs = (int64_t)a.B * a.KV * a.splits * a.row_tiles;
    if (wgs <= kCus) return launch<T, DP, KMASK, false, 2>(a, st);
  }
  return launch<T, DP, KMASK, false, 1>(a, st);
}

template <typename T>
int by_width(const Args& a, hipStream_t st) {
  const bool km = a.mask != nullptr;
  if (a.D <= 32) return km ? by_rows<T, 32, true>(a, st) : by_rows<T, 32, false>(a, st);
  if (a.D <= 64) return km ? by_rows<T, 64, true>(a, st) : by_rows<T, 64, false>(a, st);
  return km ? by_rows<T, 128, true>(a, st) : by_rows<T, 128, false>(a, st);
}

// How many workgroups share the keys of one row tile: as many as fill the card's 256 compute units
// once, at least 256 keys each (below that the join costs more than the split gains).  Four single
// tokens with 8 key heads, 8 shares each: 49 us; 4 shares 66 us, 16 shares 53 us.
int split_count(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t KV) {
  const int64_t rows = Lq * (H / KV);
  const int64_t wgs = B * KV * ceil_div(rows, few_rows(B, KV, rows) ? kFew : kRows);
  const int64_t s = std::min<int64_t>(kCus / std::max<int64_t>(wgs, 1), Lk / 256);
  return (int)std::max<int64_t>(1, s);
}

}  // namespace

int check_problem(const char* what, int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                  int64_t KV, int64_t D, float scale, int64_t band) {
  const std::string w(what);
  if (!valid_dtype(dtype)) return fail(SM_EDTYPE, w + ": float32, float16 or bfloat16 only");
  if (B < 0 || Lq < 0 || Lk < 0 || H < 0 || KV < 0 || D < 0)
    return fail(SM_EINVAL, w + ": negative size");
  if (KV == 0 ? H != 0 : H % KV != 0)
    return fail(SM_EINVAL, w + ": the query heads must be a multiple of the key heads");
  if (D % 8 != 0 || D > 128 || D == 0)
    return fail(SM_EINVAL, w + ": the head width must be a multiple of 8, 8 to 128");
  if (Lk >= (1 << 30) || (KV > 0 && Lq >= (1 << 30) / std::max<int64_t>(1, H / KV)))
    return fail(SM_EINVAL, w + ": more than 2^30 rows or keys");
  if (B >= (1 << 30) || H >= (1 << 20)) return fail(SM_EINVAL, w + ": too many batches or heads");
  if ((double)B * (double)std::max(Lq * H, Lk * KV) * (double)D > 4e18)
    return fail(SM_EINVAL, w + ": tensors too large");
  if (!(scale > 0.f) || scale > 3.4e38f) return fail(SM_EINVAL, w + ": the scale must be positive and finite");
  if (band < 0 || band >= (1ll << 30)) return fail(SM_EINVAL, w + ": the band must be 0 (none) to 2^30 - 1");
  return SM_OK;
}

int read_strides3(const int64_t* s, int64_t L, int64_t H, int64_t D, int dtype, const void* base,
                  int64_t* out, int group, const char* name) {
  if (s == nullptr) {
    out[0] = L * H * D;
    out[1] = H * D;
    out[2] = D;
  } else {
    for (int i = 0; i < 3; ++i) out[i] = s[i];
  }
  const int per = 16 / elem_size(dtype);
  for (int i = 0; i < 3; ++i) {
    if (out[i] < 0) return fail(SM_EINVAL, std::string(name) + ": negative strides are not supported");
    if (out[i] % per != 0)
      return fail(SM_EINVAL, std::string(name) + ": strides must be multiples of 16 bytes");
  }
  if (group > 0) {
    const int64_t most = (1ll << 31) / elem_size(dtype);
    const bool far = out[1] >= most / 128 || (group > 1 && out[2] >= most / 2 / group) ||
                     (64 / group + 2) * out[1] + (group - 1) * out[2] >= most;
    if (far) return fail(SM_EINVAL, std::string(name) + ": tokens or heads too far apart");
  }
  if (reinterpret_cast<uintptr_t>(base) % 16 != 0)
    return fail(SM_EINVAL, std::string(name) + ": must be 16-byte aligned");
  return SM_OK;
}

int64_t fwd_workspace_bytes(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t KV, int64_t D) {
  if (B <= 0 || Lq <= 0 || Lk <= 0 || H <= 0 || KV <= 0 || D <= 0 || H % KV != 0) return 0;
  const int s = split_count(B, Lq, Lk, H, KV);
  return s > 1 ? (int64_t)s * B * H * Lq * (D + 1) * 4 : 0;
}

int fwd_entry(Args& a, int dtype, void* workspace, int64_t ws_bytes, hipStream_t st) {
  a.splits = split_count(a.B, a.Lq, a.Lk, a.H, a.KV);
  a.row_tiles = (int)ceil_div(a.rows, few_rows(a.B, a.KV, a.rows) ? kFew : kRows);
  if (a.splits > 1) {
    const int64_t n = (int64_t)a.splits * a.B * a.H * a.Lq;
    if (workspace == nullptr || ws_bytes < n * (a.D + 1) * 4)
      return fail(SM_EINVAL, "cross_attention: the workspace is smaller than "
                             "sm_cross_attention_workspace_bytes()");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(SM_EINVAL, "cross_attention: the workspace must be 16-byte aligned");
    a.part_o = static_cast<float*>(workspace);
    a.part_l = a.part_o + n * a.D;
  }
  a.by_row_tiles = Divide(a.row_tiles);
  a.by_splits = Divide(a.splits);
  SM_DISPATCH_DTYPE(dtype, T, return by_width<T>(a, st));
  return SM_OK;
}

}  // namespace attn
}  // namespace smcv
