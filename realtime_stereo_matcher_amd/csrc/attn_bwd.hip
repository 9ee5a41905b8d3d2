// Cross attention, backward.  With p the weights (formed again from the saved logarithm of their
// sum), g the output's gradient and delta_i = sum_d g_id o_id:
//   dv_j = sum_i p_ij g_i      ds_ij = p_ij (g_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
// Two kernels, each with one side stationary in registers and the other streamed through LDS, so
// that every sum has one owner: no atomics, the same bits on every run, and the gradients of key
// heads shared by several query heads are summed in the owner's registers.  That forms the scores
// and their gradient twice (7 products where one kernel with atomic sums would have 5).
//   attn_dq   a wave owns 32 query rows; writes dq, and per row delta and the logarithm in base 2.
//             In 16 bits g . o carries the rounding of o and of the weights that formed it, which
//             shifts a whole row of ds.  So the row's delta = sum_j p_ij (g_i . v_j) is summed in
//             fp32 beside the products: attn_dkv takes that one, and dq, formed with g . o, is put
//             right at the end by the difference times sum_j p_ij k_j (one product more, on the
//             keys already read).
//   attn_dkv  a wave owns 32 keys; loops over the rows of all heads that share them
// fp16: ds would fall out of the type's range for small gradients, so g enters with a power of
// two: one that brings the row's largest |g| into [1/2, 1) in attn_dq (a lane's scalar), the
// largest of the whole key head in attn_dkv; p enters dv times 2^14.  The factors are exact and are
// taken out of the fp32 sums at the end.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"

namespace smcv {
namespace attn {
namespace {

template <typename T, int DP> struct BCfg {
  static constexpr int kTile = sizeof(T) == 4 || DP == 128 ? 32 : 64;  // streamed rows
  static constexpr int kTileBytes = kTile * DP * (int)sizeof(T);
  static constexpr int kLdsQ = 4 * kTileBytes;               // two buffers of keys and values
  static constexpr int kBuf = 2 * kTileBytes + 512;           // rows, gradients, lse and delta
  static constexpr int kLdsKv = 2 * kBuf;
};

// the power of two that brings x into [1/2, 1), as an exponent; 0 for 0, infinities and NaN
__device__ __forceinline__ int down(float x) {
  const int e = (int)((__float_as_uint(x) >> 23) & 255);
  return e == 0 || e == 255 ? 0 : min(126 - e, 100);
}

template <typename T, int DP, bool KMASK>
__global__ __launch_bounds__(256, (DP == 128 || sizeof(T) == 4 ? 1 : 2)) void attn_dq(Args a) {
  using C = BCfg<T, DP>;
  using TL = Tile<T, DP>;
  constexpr int KT = C::kTile, KB = KT / 32;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const unsigned id = xcd_id(), bkv = a.by_row_tiles(id), b = a.by_kv(bkv);
  const int rt = id - bkv * a.row_tiles, kv = bkv - b * a.KV;
  const int wg_row0 = rt * kRows, row0 = wg_row0 + 32 * wave, row = row0 + (lane & 31);
  const int token = a.by_group(row), head = kv * a.G + row - token * a.G;
  const bool there = row < a.rows;

  Keys<KT, KMASK> keys(a, b, wg_row0, kRows);

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
  const int64_t n_pad = (int64_t)a.row_tiles * kRows;
  const int64_t at = ((int64_t)b * a.KV + kv) * n_pad + row;
  const float lse = there ? a.lse[((int64_t)b * a.KV + kv) * a.rows + row] : -INFINITY;
  // a row without keys, or past the end: +inf makes every weight that is formed from it 0
  const float lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
  if (half == 0) {
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
      const unsigned at0 = lds_addr(smem);
      a.tile_max[((int64_t)b * a.KV + kv) * a.row_tiles + rt] =
          fmaxf(fmaxf(lds_get<float>(at0), lds_get<float>(at0 + 4)),
                fmaxf(lds_get<float>(at0 + 8), lds_get<float>(at0 + 12)));
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

  const unsigned lds = lds_addr(smem);
  const Reads<T, DP> from(lds, lane);
  const int wave0 = wave * 64;
  const unsigned kb_row = (unsigned)a.ks[1] * sizeof(T), vb_row = (unsigned)a.vs[1] * sizeof(T);
  Stage<T, DP, KT, 256> sk, sv;
  sk.init(tid, a.D, [&](int r) { return r * kb_row; });
  sv.init(tid, a.D, [&](int r) { return r * vb_row; });
  const uint64_t K = reinterpret_cast<uint64_t>(static_cast<const T*>(a.k) + b * a.ks[0] + kv * a.ks[2]);
  const uint64_t V = reinterpret_cast<uint64_t>(static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2]);
  auto copy = [&](int t, unsigned dst, uint64_t bits) {
    const uint64_t kp = K + (uint64_t)t * KT * kb_row, vp = V + (uint64_t)t * KT * vb_row;
    if (bits == keys.kAll) {
      sk.copy(kp, dst, wave0);
      sv.copy(vp, dst + C::kTileBytes, wave0);
    } else if (bits != 0) {
      sk.copy(kp, dst, wave0, tid, bits, kb_row);
      sv.copy(vp, dst + C::kTileBytes, wave0, tid, bits, vb_row);
    }
  };

  // dq, and (16-bit types) the weighted mean of the keys
  constexpr int N = sizeof(T) == 4 ? 1 : 2;
  f32x16 dq[N][DP / 32];
  float sum = 0.f;  // of p (g . v): delta again
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[n][db][r] = 0.f;

  int t = keys.tb;
  uint64_t bits = 0;
  int byte = 0;
  if (t < keys.te) {
    bits = KMASK ? __ballot(keys.byte(t, lane)) : keys.by_length(t);
    copy(t, lds, bits);
  }
  if (KMASK) byte = keys.byte(t + 1, lane);
  auto step = [&](auto buf) {
    constexpr int kBuf = decltype(buf)::value * 2 * C::kTileBytes;
    publish();
    uint64_t next = 0;
    if (t + 1 < keys.te) {
      next = KMASK ? __ballot(byte) : keys.by_length(t + 1);
      if (KMASK) byte = keys.byte(t + 2, lane);
      copy(t + 1, lds + (2 * C::kTileBytes - kBuf), next);
    }
    const uint64_t seen = bits;
    bits = next;
    if (seen == 0) return;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const BandOf in(a, row0, t * KT + 32 * kb, 32);
      const unsigned seen32 = (unsigned)(seen >> (32 * kb));
      if (!in.some || seen32 == 0) continue;
      f32x16 s = mma_rows<T, DP>(from, kBuf, 32 * kb, q);
      f32x16 ds[N];  // and the weights
      ds[0] = mma_rows<T, DP>(from, kBuf + C::kTileBytes, 32 * kb, g);
      if (!in.all || seen32 != ~0u)
        mask_block(s, a.band > 0 ? band_bits(seen32, token - (t * KT + 32 * kb), a.band) : seen32, half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse2));
        if constexpr (N == 2) {
          sum = fmaf(p, ds[0][r], sum);
          ds[1][r] = p;
        }
        ds[0][r] = p * (ds[0][r] - delta);
      }
      mma_transposed<T, DP, N>(dq, from, kBuf, 32 * kb, ds);
    }
  };
  while (t < keys.te) {
    step(std::integral_constant<int, 0>{});
    if (++t >= keys.te) break;
    step(std::integral_constant<int, 1>{});
    ++t;
  }
  if constexpr (N == 2) {
    sum = other_half_sum(sum);
    if (half == 0) a.row_delta[at] = __builtin_ldexpf(sum, -shift);
    delta -= sum;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[0][db][r] = fmaf(delta, dq[1][db][r], dq[0][db][r]);
  }
  if (!there) return;
  store_columns<T, DP>(static_cast<T*>(a.dq) + orow, dq[0], __builtin_ldexpf(a.scale, -shift), half, a.D);
}

template <typename T, int DP, bool KMASK>
__global__ __launch_bounds__(256, (DP == 128 || sizeof(T) == 4 ? 1 : 2)) void attn_dkv(Args a) {
  using C = BCfg<T, DP>;
  constexpr int RT = C::kTile, RB = RT / 32;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  constexpr float kUp = kScaled ? 14.f : 0.f;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const unsigned id = xcd_id(), bkv = a.by_key_tiles(id), b = a.by_kv(bkv);
  const int jt = id - bkv * a.key_tiles, kv = bkv - b * a.KV;
  const int wg_j0 = jt * kRows, j0 = wg_j0 + 32 * wave, j = j0 + (lane & 31);
  const int keys = a.lengths ? min(max(a.lengths[b], 0), a.Lk) : a.Lk;
  const bool there = j < keys && (!KMASK || a.mask[(int64_t)b * a.Lk + min(j, a.Lk - 1)] != 0);

  RowOps<T, DP> k, v;
  load_rows<T, DP>(k, static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)j * a.ks[1] +
                          kv * a.ks[2], there, half, a.D);
  load_rows<T, DP>(v, static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)j * a.vs[1] +
                          kv * a.vs[2], there, half, a.D);

  // rows of the heads that share these keys: all, or those whose band reaches them
  int64_t rlo = 0, rhi = a.rows;
  if (a.band > 0) {
    rlo = min((int64_t)a.rows, (int64_t)wg_j0 * a.G);
    rhi = min((int64_t)a.rows, ((int64_t)min(wg_j0 + kRows, a.Lk) - 1 + a.band) * a.G);
  }
  if (wg_j0 >= keys) rhi = rlo;  // nothing attends to them: their gradients are 0
  const int tb = (int)(rlo / RT), te = rhi > rlo ? (int)((rhi + RT - 1) / RT) : tb;

  const int64_t n_pad = (int64_t)a.row_tiles * kRows;
  const float* lse = a.row_lse + ((int64_t)b * a.KV + kv) * n_pad;
  const float* delta = a.row_delta + ((int64_t)b * a.KV + kv) * n_pad;
  int shift = 0;
  if constexpr (kScaled) {
    const float* tm = a.tile_max + ((int64_t)b * a.KV + kv) * a.row_tiles;
    float top = 0.f;
    for (int i = lane; i < a.row_tiles; i += 64) top = fmaxf(top, tm[i]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
    shift = __builtin_amdgcn_readfirstlane(down(top));
  }

  const unsigned lds = lds_addr(smem);
  const Reads<T, DP> from(lds, lane);
  const int wave0 = wave * 64;
  const uint64_t Q = reinterpret_cast<uint64_t>(static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)kv * a.G * a.qs[2]);
  const uint64_t GO = reinterpret_cast<uint64_t>(static_cast<const T*>(a.dout) + b * a.gs[0] + (int64_t)kv * a.G * a.gs[2]);
  // Row t RT + r is token (t RT + r) / G: where G divides RT the offsets from the tile's first token
  // are the same in every tile.
  const bool regular = (RT & (a.G - 1)) == 0 && (a.G & (a.G - 1)) == 0;
  auto row_at = [&](int row, int token0, const int64_t* st) -> unsigned {
    const int token = a.by_group(row), g = row - token * a.G;
    return ((token - token0) * (unsigned)st[1] + g * (unsigned)st[2]) * (unsigned)sizeof(T);
  };
  Stage<T, DP, RT, 256> sq, sg;
  sq.init(tid, a.D, [&](int r) { return row_at(r, 0, a.qs); });
  sg.init(tid, a.D, [&](int r) { return row_at(r, 0, a.gs); });
  auto copy = [&](int t, unsigned dst) {
    const int token0 = a.by_group(t * RT);
    const uint64_t qp = Q + (uint64_t)token0 * a.qs[1] * sizeof(T), gp = GO + (uint64_t)token0 * a.gs[1] * sizeof(T);
    if (regular && (t + 1) * RT <= a.rows) {
      sq.copy(qp, dst, wave0);
      sg.copy(gp, dst + C::kTileBytes, wave0);
    } else {  // rows past the end read the tile's first: their weights are 0
      auto at = [&](const int64_t* st) {
        return [=, &a](int it, unsigned o) {
          const int r = Stage<T, DP, RT, 256>::row_of(it, tid), row = t * RT + r;
          return o - row_at(r, 0, st) + row_at(row < a.rows ? row : t * RT, token0, st);
        };
      };
      sq.copy(qp, dst, wave0, at(a.qs));
      sg.copy(gp, dst + C::kTileBytes, wave0, at(a.gs));
    }
    // RT logarithms, then RT deltas (the rows are padded to whole tiles there)
    const uint64_t lp = reinterpret_cast<uint64_t>(lse + t * RT), dp = reinterpret_cast<uint64_t>(delta + t * RT);
    if (wave == 0 && lane < RT) copy4(lp, lane * 4, dst + 2 * C::kTileBytes);
    if (wave == 1 && lane < RT) copy4(dp, lane * 4, dst + 2 * C::kTileBytes + RT * 4);
  };

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;

  int t = tb;
  if (t < te) copy(t, lds);
  auto step = [&](auto buf) {
    constexpr int kAt = decltype(buf)::value * C::kBuf;
    publish();
    if (t + 1 < te) copy(t + 1, lds + (C::kBuf - kAt));
    const unsigned st = lds + kAt + 2 * C::kTileBytes;
    if (j0 >= keys) return;
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
      mma_transposed<T, DP>(dv, from, kAt + C::kTileBytes, 32 * rb, p);
      mma_transposed<T, DP>(dk, from, kAt, 32 * rb, ds);
    }
  };
  while (t < te) {
    step(std::integral_constant<int, 0>{});
    if (++t >= te) break;
    step(std::integral_constant<int, 1>{});
    ++t;
  }
  if (j >= a.Lk) return;
  const int64_t out = (((int64_t)b * a.Lk + j) * a.KV + kv) * a.D;
  if (!there) {  // 0 whatever the zero rows that stood for the key gave
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;
  }
  store_columns<T, DP>(static_cast<T*>(a.dv) + out, dv, kScaled ? 0x1p-14f : 1.f, half, a.D);
  store_columns<T, DP>(static_cast<T*>(a.dk) + out, dk, __builtin_ldexpf(a.scale, -shift), half, a.D);
}

template <typename T, int DP, bool KMASK>
int launch(const Args& a, hipStream_t st) {
  using C = BCfg<T, DP>;
  static std::atomic<unsigned long long> done_q{0}, done_kv{0};
  const int dev = stream_device(st);
  if (const int rc = ensure_lds_limit(reinterpret_cast<const void*>(&attn_dq<T, DP, KMASK>), C::kLdsQ, dev, done_q)) return rc;
  if (const int rc = ensure_lds_limit(reinterpret_cast<const void*>(&attn_dkv<T, DP, KMASK>), C::kLdsKv, dev, done_kv)) return rc;
  const int64_t bkv = (int64_t)a.B * a.KV, key_tiles = a.key_tiles;
  if (bkv * a.row_tiles > 0x7fffffffll || bkv * key_tiles > 0x7fffffffll)
    return fail(SM_EINVAL, "cross_attention_backward: too many row tiles");
  if (a.row_tiles > 0) {
    attn_dq<T, DP, KMASK><<<dim3((unsigned)(bkv * a.row_tiles)), 256, C::kLdsQ, st>>>(a);
    if (const int rc = check_launch("cross_attention_backward dq")) return rc;
  }
  if (key_tiles > 0) {
    attn_dkv<T, DP, KMASK><<<dim3((unsigned)(bkv * key_tiles)), 256, C::kLdsKv, st>>>(a);
    return check_launch("cross_attention_backward dk, dv");
  }
  return SM_OK;
}

template <typename T>
int by_width(const Args& a, hipStream_t st) {
  const bool km = a.mask != nullptr;
  if (a.D <= 32) return km ? launch<T, 32, true>(a, st) : launch<T, 32, false>(a, st);
  if (a.D <= 64) return km ? launch<T, 64, true>(a, st) : launch<T, 64, false>(a, st);
  return km ? launch<T, 128, true>(a, st) : launch<T, 128, false>(a, st);
}

}  // namespace

int64_t bwd_workspace_bytes(int64_t B, int64_t Lq, int64_t H, int64_t KV) {
  if (B <= 0 || Lq <= 0 || H <= 0 || KV <= 0 || H % KV != 0) return 0;
  const int64_t tiles = ceil_div(Lq * (H / KV), kRows);
  return B * KV * tiles * (2 * kRows + 1) * 4;
}

int bwd_entry(Args& a, int dtype, void* workspace, int64_t ws_bytes, hipStream_t st) {
  a.row_tiles = (int)ceil_div(a.rows, kRows);
  const int64_t n = (int64_t)a.B * a.KV * a.row_tiles;
  if (n > 0 && (workspace == nullptr || ws_bytes < n * (2 * kRows + 1) * 4))
    return fail(SM_EINVAL, "cross_attention_backward: the workspace is smaller than "
                           "sm_cross_attention_backward_workspace_bytes()");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(SM_EINVAL, "cross_attention_backward: the workspace must be 16-byte aligned");
  a.row_lse = static_cast<float*>(workspace);
  a.row_delta = a.row_lse + n * kRows;
  a.tile_max = a.row_delta + n * kRows;
  a.key_tiles = (int)ceil_div(a.Lk, kRows);
  a.by_row_tiles = Divide(a.row_tiles);
  a.by_key_tiles = Divide(a.key_tiles);
  SM_DISPATCH_DTYPE(dtype, T, return by_width<T>(a, st));
  return SM_OK;
}

}  // namespace attn
}  // namespace smcv
