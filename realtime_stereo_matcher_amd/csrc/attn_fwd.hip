// Cross attention, forward: o_i = sum_j p_ij v_j, p = softmax over the keys j that token i may see.
//
// One pass over the keys with the running maximum m and sum l of each query's softmax: scores,
// weights and statistics stay in registers (attn_common.h has the layout), keys and values pass
// through LDS once a workgroup.  m is raised lazily: while a tile's scores exceed it by less than
// 2^8 in weight, the weights are formed against the old m and the accumulators are not rescaled
// (they are divided by l, formed against the same m, at the end; weights up to 2^8 lose nothing in
// any of the types).
#include <algorithm>

#include "attn_common.h"

namespace smcv {
namespace attn {

namespace {

// FEW: at most 32 query rows (single tokens with shared heads): the waves hold the same rows and
// take the key tiles in turn, each with its own LDS, and join at the end.
template <typename T, int DP, bool FEW> struct Cfg {
  static constexpr int kTile = sizeof(T) == 4 ? 32 : (FEW && DP == 128) ? 32 : 64;  // keys
  static constexpr int kWaves = FEW && sizeof(T) == 4 && DP == 128 ? 2 : 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTileBytes = kTile * DP * (int)sizeof(T);
  static constexpr int kBufBytes = 2 * kTileBytes;  // keys and values
  static constexpr int kLds = 2 * kBufBytes * (FEW ? kWaves : 1);
};

constexpr float kLazy = 8.f;

template <typename T, int DP, bool KMASK, bool FEW>
__global__ __launch_bounds__((Cfg<T, DP, FEW>::kThreads), (FEW || sizeof(T) == 4 ? 1 : 2))
void attn_fwd(Args a) {
  using C = Cfg<T, DP, FEW>;
  using TL = Tile<T, DP>;
  using frag = Frag<T>;
  constexpr int KT = C::kTile, KB = KT / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  unsigned id = xcd_id();
  const int rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int kv = id % a.KV, b = id / a.KV;

  const int wg_row0 = rt * (FEW ? kFew : kRows);
  const int row0 = wg_row0 + (FEW ? 0 : 32 * wave);  // of this wave
  const int row = row0 + (lane & 31);                // of this lane
  const int token = row / a.G, head = kv * a.G + row % a.G;
  const bool there = row < a.rows;

  // key tiles of the workgroup: up to the sequence's length, inside the band of its rows, and of
  // those this split's share
  const int keys = key_count(a, b);
  int jlo = 0, jhi = keys;
  if (a.band > 0) {
    const int last = min(wg_row0 + (FEW ? kFew : kRows), a.rows) - 1;
    jlo = max(0, wg_row0 / a.G - a.band + 1);
    jhi = min(keys, last / a.G + 1);
  }
  int tb = jlo / KT, te = jhi > jlo ? (jhi + KT - 1) / KT : tb;
  if (a.splits > 1) {
    const int per = (te - tb + a.splits - 1) / a.splits;
    tb += split * per;
    te = min(te, tb + per);
  }

  const T* K = static_cast<const T*>(a.k) + b * a.ks[0] + kv * a.ks[2];
  const T* V = static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2];
  frag q[TL::kSteps];
  load_rows<T, DP>(q, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)token * a.qs[1] +
                          head * a.qs[2], there, half, a.D);

  const unsigned lds = lds_addr(smem) + (FEW ? wave * 2 * C::kBufBytes : 0);
  const uint8_t* mask = KMASK ? a.mask + (int64_t)b * a.Lk : nullptr;
  const int step = FEW ? C::kWaves : 1;

  // bit j: key j of the tile exists and is not masked
  auto mask_byte = [&](int t) -> int {
    const int j = t * KT + lane;
    return lane < KT && t < te && j < keys ? mask[j] : 0;
  };
  auto length_bits = [&](int t) -> uint64_t {
    const int n = keys - t * KT;
    return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
  };
  constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
  auto copy = [&](int t, unsigned dst, uint64_t bits) {
    auto ok = [&](int, int r) { return ((bits >> r) & 1) != 0; };
    if (FEW) {
      TL::template load<KT, 64>(K, a.ks[1], t * KT, dst, lane, a.D, ok);
      TL::template load<KT, 64>(V, a.vs[1], t * KT, dst + C::kTileBytes, lane, a.D, ok);
    } else {
      TL::template load<KT, C::kThreads>(K, a.ks[1], t * KT, dst, tid, a.D, ok);
      TL::template load<KT, C::kThreads>(V, a.vs[1], t * KT, dst + C::kTileBytes, tid, a.D, ok);
    }
  };

  f32x16 o[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -INFINITY, l = 0.f;

  int t = tb + (FEW ? wave : 0);
  uint64_t bits = 0;
  int byte = 0;
  if (t < te) {
    bits = KMASK ? __ballot(mask_byte(t)) : length_bits(t);
    if (KMASK) byte = mask_byte(t + step);
    copy(t, lds, bits);
  }
  for (int buf = 0; t < te; t += step, buf ^= 1) {
    // this tile is in LDS, and nobody reads the other buffer any more
    if (FEW) wait_copies(); else publish();
    uint64_t next = 0;
    if (t + step < te) {
      next = KMASK ? __ballot(byte) : length_bits(t + step);
      if (KMASK) byte = mask_byte(t + 2 * step);
      copy(t + step, lds + (buf ^ 1) * C::kBufBytes, next);
    }
    const unsigned kt = lds + buf * C::kBufBytes, vt = kt + C::kTileBytes;
    const uint64_t seen = bits & kAll;
    bits = next;
    bool edge = false;
    if (a.band > 0) {
      const int j0 = t * KT, j1 = j0 + KT - 1;
      const int i0 = row0 / a.G, i1 = min(row0 + 31, a.rows - 1) / a.G;
      if (j0 > i1 || j1 <= i0 - a.band) continue;  // outside this wave's band
      edge = j1 > i0 || j0 <= i1 - a.band;
    }
    if (seen == 0) continue;

    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = mma_rows<T, DP>(kt, 32 * kb, q, lane);
    if (seen != kAll) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const unsigned w = (unsigned)(seen >> (32 * kb)) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[kb][r] = (w >> (8 * (r >> 2) + (r & 3))) & 1 ? s[kb][r] : -INFINITY;
      }
    }
    if (edge) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int d = token - (t * KT + 32 * kb + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[kb][r] = (unsigned)(d - (8 * (r >> 2) + (r & 3))) < (unsigned)a.band ? s[kb][r] : -INFINITY;
      }
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
    const float mc = m == -INFINITY ? 0.f : m * a.c;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], a.c, -mc));
        l += s[kb][r];
      }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) mma_transposed<T, DP>(o, vt, 32 * kb, s[kb], lane);
  }
  l = other_half_sum(l);

  const int64_t at = ((int64_t)b * a.KV + kv) * a.rows + row;  // of this lane's row
  if constexpr (FEW) {
    // join the waves: rows x DP partial sums and the statistics of each wave
    constexpr int kPitch = (DP + 4) * 4, kWaveBytes = 32 * kPitch + 256;
    static_assert(C::kWaves * kWaveBytes <= C::kLds, "the join fits the tiles' LDS");
    __syncthreads();
    const unsigned mine = lds_addr(smem) + wave * kWaveBytes;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        lds_put(mine + (lane & 31) * kPitch + (32 * db + 8 * g + 4 * half) * 4,
                f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]});
    if (half == 0) {
      lds_put(mine + 32 * kPitch + lane * 4, m);
      lds_put(mine + 32 * kPitch + 128 + lane * 4, l);
    }
    __syncthreads();
    for (int p = tid; p < 32 * (DP / 4); p += C::kThreads) {
      const int r = p / (DP / 4), d = 4 * (p % (DP / 4)), grow = wg_row0 + r;
      if (grow >= a.rows || d >= a.D) continue;
      float top = -INFINITY, mw[C::kWaves];
#pragma unroll
      for (int w = 0; w < C::kWaves; ++w) {
        mw[w] = lds_get<float>(lds_addr(smem) + w * kWaveBytes + 32 * kPitch + r * 4);
        top = fmaxf(top, mw[w]);
      }
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < C::kWaves; ++w) {
        const unsigned from = lds_addr(smem) + w * kWaveBytes;
        const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw[w] - base) * a.c);
        sum = fmaf(f, lds_get<float>(from + 32 * kPitch + 128 + r * 4), sum);
        const f32x4 x = lds_get<f32x4>(from + r * kPitch + d * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(f, x[e], v[e]);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= inv;
      const float lse = sum == 0.f ? -INFINITY : fmaf(base, a.c, __builtin_amdgcn_logf(sum)) * kLn2;
      const int64_t ra = ((int64_t)b * a.KV + kv) * a.rows + grow;
      if (a.splits > 1) {
        const int64_t ps = (int64_t)split * a.B * a.KV * a.rows + ra;
        *reinterpret_cast<f32x4*>(a.part_o + ps * a.D + d) = v;
        if (d == 0) a.part_l[ps] = lse;
      } else {
        const int64_t tok = (int64_t)b * a.Lq + grow / a.G;
        store4<T>(static_cast<T*>(a.out) + (tok * a.H + kv * a.G + grow % a.G) * a.D + d, v);
        if (d == 0 && a.lse) a.lse[ra] = lse;
      }
    }
  } else {
    if (!there) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float lse = l == 0.f ? -INFINITY : fmaf(m, a.c, __builtin_amdgcn_logf(l)) * kLn2;
    if (a.splits > 1) {
      const int64_t ps = (int64_t)split * a.B * a.KV * a.rows + at;
      store_columns<float, DP>(a.part_o + ps * a.D, o, inv, half, a.D);
      if (half == 0) a.part_l[ps] = lse;
    } else {
      store_columns<T, DP>(static_cast<T*>(a.out) + (((int64_t)b * a.Lq + token) * a.H + head) * a.D,
                           o, inv, half, a.D);
      if (half == 0 && a.lse) a.lse[at] = lse;
    }
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
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_l[s * n + r]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f((a.part_l[s * n + r] - base) * kLog2e);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (s * n + r) * a.D + d);
    sum += w;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(w, x[e], v[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= inv;
  const int row = (int)(r % a.rows), kv = (int)(r / a.rows % a.KV);
  const int64_t tok = r / a.rows / a.KV * a.Lq + row / a.G;
  store4<T>(static_cast<T*>(a.out) + (tok * a.H + kv * a.G + row % a.G) * a.D + d, v);
  if (d == 0 && a.lse) a.lse[r] = sum == 0.f ? -INFINITY : base + __builtin_amdgcn_logf(sum) * kLn2;
}

template <typename T, int DP, bool KMASK, bool FEW>
int launch(const Args& a, hipStream_t st) {
  using C = Cfg<T, DP, FEW>;
  static std::atomic<unsigned long long> done{0};
  const void* kern = reinterpret_cast<const void*>(&attn_fwd<T, DP, KMASK, FEW>);
  if (const int rc = ensure_lds_limit(kern, C::kLds, stream_device(st), done)) return rc;
  const int64_t grid = (int64_t)a.B * a.KV * a.splits * a.row_tiles;
  if (grid > 0x7fffffffll) return fail(SM_EINVAL, "cross_attention: too many row tiles");
  attn_fwd<T, DP, KMASK, FEW><<<dim3((unsigned)grid), C::kThreads, C::kLds, st>>>(a);
  if (const int rc = check_launch("cross_attention")) return rc;
  if (a.splits > 1) {
    const int64_t n = (int64_t)a.B * a.KV * a.rows * (a.D / 4);
    attn_join<T><<<dim3((unsigned)ceil_div(n, 256)), 256, 0, st>>>(a);
    return check_launch("cross_attention join");
  }
  return SM_OK;
}

template <typename T>
int by_width(const Args& a, hipStream_t st) {
  const bool few = a.rows <= kFew, km = a.mask != nullptr;
#define SM_ATTN_WIDTH(DP)                                                            \
  return few ? (km ? launch<T, DP, true, true>(a, st) : launch<T, DP, false, true>(a, st)) \
             : (km ? launch<T, DP, true, false>(a, st) : launch<T, DP, false, false>(a, st));
  if (a.D <= 32) { SM_ATTN_WIDTH(32) }
  if (a.D <= 64) { SM_ATTN_WIDTH(64) }
  SM_ATTN_WIDTH(128)
#undef SM_ATTN_WIDTH
}

// How many workgroups share the keys of one row tile: as many as fill the card's 256 compute units
// once, at least 256 keys each (below that the join costs more than the split gains).
int split_count(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t KV) {
  const int64_t rows = Lq * (H / KV);
  const int64_t wgs = B * KV * ceil_div(rows, rows <= kFew ? kFew : kRows);
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
  if (!(scale > 0.f) || scale > 3.4e38f) return fail(SM_EINVAL, w + ": the scale must be positive and finite");
  if (band < 0 || band >= (1ll << 30)) return fail(SM_EINVAL, w + ": the band must be 0 (none) to 2^30 - 1");
  return SM_OK;
}

int read_strides3(const int64_t* s, int64_t L, int64_t H, int64_t D, int dtype, const void* base,
                  int64_t* out, const char* name) {
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
  a.row_tiles = (int)ceil_div(a.rows, a.rows <= kFew ? kFew : kRows);
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
  SM_DISPATCH_DTYPE(dtype, T, return by_width<T>(a, st));
  return SM_OK;
}

}  // namespace attn
}  // namespace smcv
