// Shared pieces of the cross-attention kernels (attn_fwd.hip, attn_bwd.hip): the problem, the
// tiles in LDS and the matrix-instruction operands that are read from them.
//
// All products are formed transposed, so that a lane owns one COLUMN of every result.  With the
// 32x32 result layout (lane l, register r: row 8 (r/4) + 4 (l/32) + r%4, column l%32) a score block
// S^T = K Q^T leaves each lane 16 keys of one query: the softmax statistics are one scalar a lane,
// and the same registers, rounded, ARE the right operand of O^T += V^T P^T.  The contraction index
// of a product may be permuted if both operands agree, so the left operand is read with the order
// of keys that the result layout happens to have and no value crosses lanes.
#pragma once

#include "common.h"

namespace smcv {
namespace attn {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCus = 256;    // compute units of the MI355X: what a launch has to fill
constexpr int kRows = 128;   // query rows of a workgroup (32 a wave)
constexpr int kFew = 32;     // at most so many rows: the waves share the rows and split the keys

// n / d for 0 <= n < 2^31 by a multiplication (division by an invariant integer, Granlund and
// Montgomery 1994): with 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d) < 2^32 + 1, n m / 2^(31+l)
// exceeds n / d by less than 1 / d.
struct Divide {
  uint32_t m = 0, shift = 0;
  Divide() = default;
  explicit Divide(int64_t d) {
    d = d < 1 ? 1 : d;
    while ((int64_t(1) << shift) < d) ++shift;
    shift += 31;
    m = (uint32_t)(((uint64_t(1) << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int operator()(unsigned n) const { return (int)(((uint64_t)n * m) >> shift); }
};

struct Args {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float* lse;             // (B, KV, Lq * G), natural logarithm
  float *part_o, *part_l; // split keys: (splits, B, KV, rows, D) and (splits, B, KV, rows)
  float *row_lse, *row_delta;  // backward: (B, KV, padded rows)
  float* tile_max;        // backward, fp16: largest |dout| of each row tile, (B, KV, row tiles); negative
                          // where ds passed the type's range
  const int* lengths;     // (B) or null
  const uint8_t* mask;    // (B, Lk) or null
  int64_t qs[3], ks[3], vs[3], gs[3];  // element strides of batch, token and head
  int B, Lq, Lk, H, KV, G, D;
  int rows, row_tiles;    // Lq * G and its tiles: row r is token r / G, head kv * G + r % G
  int pad_rows;           // rows up to a multiple of 128 (backward)
  int band;               // > 0: key j is a candidate of token i iff 0 <= i - j < band
  int splits, key_tiles;  // shares of the keys; tiles of keys (backward)
  unsigned workgroups, first;  // of the problem; the launch's first
  Divide by_group, by_kv, by_row_tiles, by_splits, by_key_tiles;
  float scale, c;         // c = scale * log2(e): exp(scale x) = exp2(c x)
};

// ------------------------------------------------------------------------------------- operands
// 16-bit: a 32x32x16 step contracts 16 values, lane l holding 8 of column / row l%32.
template <typename T> struct Mma;
template <> struct Mma<__half> {
  using frag = h16x8;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ void put(frag& f, int e, float v) { f[e] = (_Float16)v; }
  static __device__ __forceinline__ float add2(float a, float b, float c) {  // rounded, summed in fp32
    typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(h16x2{(_Float16)a, (_Float16)b}, h16x2{1, 1}, c, false);
  }
  static __device__ __forceinline__ float get(const frag& f, int e) { return (float)f[e]; }
};
template <> struct Mma<bf16_t> {
  using frag = b16x8;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ void put(frag& f, int e, float v) { f[e] = (__bf16)v; }
  static __device__ __forceinline__ float add2(float a, float b, float c) {
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(b16x2{(__bf16)a, (__bf16)b}, b16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
  }
  static __device__ __forceinline__ float get(const frag& f, int e) { return (float)f[e]; }
};
// fp32: four 32x32x2 steps a 16-byte piece; step e contracts values 8c + e and 8c + 4 + e.
template <> struct Mma<float> {
  using frag = f32x4;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float get(const frag& f, int e) { return f[e]; }
};

template <typename T> using Frag = typename Mma<T>::frag;

// ---------------------------------------------------------------------------------- tiles in LDS
typedef __attribute__((address_space(3))) unsigned char lds_u8;
__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)(uintptr_t)(const lds_u8*)p;
}
template <typename V>
__device__ __forceinline__ V lds_get(unsigned addr) {
  return *reinterpret_cast<__attribute__((address_space(3))) V*>(addr);
}
template <typename V>
__device__ __forceinline__ void lds_put(unsigned addr, V v) {
  *reinterpret_cast<__attribute__((address_space(3))) V*>(addr) = v;
}
// 16 (4) bytes a lane, from a uniform base and a lane's offset, into LDS at a wave's base + 16 (4) *
// lane, without a register in between.  Inline, because the compiler would wait for every such copy
// in flight before each LDS read; the kernels wait themselves (wait_copies, publish) before a tile is
// read.
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)x) |
         (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
__device__ __forceinline__ void copy16(uint64_t base, unsigned off, unsigned dst) {
  base = uniform(base);
  dst = __builtin_amdgcn_readfirstlane(dst);
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "s"(base), "v"(off), "s"(dst)
      : "memory");
}
__device__ __forceinline__ void copy4(uint64_t base, unsigned off, unsigned dst) {
  base = uniform(base);
  dst = __builtin_amdgcn_readfirstlane(dst);
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %2, %1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "s"(base), "v"(off), "s"(dst)
      : "memory");
}
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ void publish() {  // this wave's copies done, then everyone's
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A tile of rows x DP values in LDS, in 16-byte pieces.  Piece `ch` of row `row` sits at
// ch ^ twist(row).  LDS serves 256 bytes a cycle: 16 lanes of a 16-byte read (16 rows, the same
// piece) or 32 lanes of a transposing read (4 rows, 64 bytes each), and the twist puts both on
// different banks whatever the rows' length (64 to 512 bytes).
template <typename T, int DP> struct Tile {
  static constexpr int kPer = 16 / (int)sizeof(T);
  static constexpr int kPieces = DP / kPer;  // of a row
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  static constexpr int kSteps = sizeof(T) == 4 ? DP / 8 : DP / 16;  // row-operand reads
  static __device__ __forceinline__ int twist(int row) {
    if constexpr (kRowBytes == 64) return (row >> 2) & 3;
    if constexpr (kRowBytes == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    if constexpr (sizeof(T) == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (((row >> 2) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1);
  }
};

// The copies of a tile of ROWS rows by NT threads: a lane's offset in each instruction, from the
// tile's first row.  Pieces past the head's width read its first piece: finite values that meet
// zeros in the other operand, or columns that are not stored.
template <typename T, int DP, int ROWS, int NT> struct Stage {
  using TL = Tile<T, DP>;
  static constexpr int kTotal = ROWS * TL::kPieces, kN = (kTotal + NT - 1) / NT;
  static_assert(kTotal % 64 == 0, "whole wave instructions");
  unsigned off[kN];
  static __device__ __forceinline__ int row_of(int it, int tid) { return (it * NT + tid) / TL::kPieces; }
  template <typename F> __device__ __forceinline__ void init(int tid, int D, F row_offset) {
#pragma unroll
    for (int it = 0; it < kN; ++it) {
      const int row = row_of(it, tid), ch = ((it * NT + tid) % TL::kPieces) ^ TL::twist(row);
      off[it] = row_offset(row) + (ch * TL::kPer < D ? ch * 16 : 0);
    }
  }
  // `adjust(it, offset)`: the offset to read instead
  template <typename F>
  __device__ __forceinline__ void copy(uint64_t base, unsigned dst, int wave0, F adjust) const {
#pragma unroll
    for (int it = 0; it < kN; ++it) {
      if (kTotal % NT != 0 && it * NT + wave0 >= kTotal) break;
      copy16(base, adjust(it, off[it]), dst + (it * NT + wave0) * 16);
    }
  }
  __device__ __forceinline__ void copy(uint64_t base, unsigned dst, int wave0) const {
    copy(base, dst, wave0, [](int, unsigned o) { return o; });
  }
  // Rows whose bit is clear (past the end, masked) read the tile's first row whose bit is set: the
  // scores they give are replaced by -inf, and their values are finite if that row's are.
  __device__ __forceinline__ void copy(uint64_t base, unsigned dst, int wave0, int tid, uint64_t bits,
                                       unsigned row_bytes) const {
    const int first = __builtin_ctzll(bits);
    copy(base, dst, wave0, [&](int it, unsigned o) {
      const int row = row_of(it, tid);
      return (bits >> row) & 1 ? o : o + (unsigned)((first - row) * (int)row_bytes);
    });
  }
};

// A wave's reads of tiles whose LDS addresses differ by constants: the lane's part of every address
// (a twist is an exclusive or, so each piece has its own) is formed once.
template <typename T, int DP> struct Reads {
  using TL = Tile<T, DP>;
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kRowRegs = TL::kSteps < 8 ? TL::kSteps : 8;  // twists are less than 16 pieces
  typedef float Columns __attribute__((ext_vector_type(DP / 32)));  // fp32: one of each block
  unsigned row[kRowRegs], col[kWide ? 8 : DP / 16];
  __device__ __forceinline__ Reads(unsigned lds, int lane) {
    const int half = lane >> 5, r = lane & 31;
#pragma unroll
    for (int c = 0; c < kRowRegs; ++c)
      row[c] = lds + r * TL::kRowBytes + ((2 * c + half) ^ TL::twist(r)) * 16;
    if constexpr (kWide) {
      // lane m's columns are the DP / 32 neighbours from (DP / 32) m on, one of each block
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int q = 8 * (u >> 2) + 4 * half + (u & 3), at = r * (DP / 8);
        col[u] = lds + q * TL::kRowBytes + (((at >> 4) ^ TL::twist(q)) << 4) + (at & 15);
      }
    } else {
      // ds_read_tr16_b64: in each 16 lanes, lane i receives column i of the 4 x 16 values whose row
      // j the lanes 4j .. 4j+3 address
      const int g = (lane >> 4) & 1, l16 = lane & 15;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int q = 8 * u + 4 * half + (l16 >> 2);
          col[2 * db + u] = lds + q * TL::kRowBytes +
                            ((4 * db + 2 * g + ((l16 & 3) >> 1)) ^ TL::twist(q)) * 16 + (l16 & 1) * 8;
        }
    }
  }
  // left operand with the tile's rows as its rows: rows row0 .. row0+31 (row0 a multiple of 32), step c
  __device__ __forceinline__ Frag<T> rows(int tile, int row0, int c) const {
    return lds_get<Frag<T>>(row[c % kRowRegs] + (tile + row0 * TL::kRowBytes + c / kRowRegs * 256));
  }
  // the same transposed, 16-bit: rows row0 + 16 s .. + 15 as the contraction of column block db
  __device__ __forceinline__ Frag<T> columns(int tile, int row0, int s, int db) const {
    static_assert(!kWide, "16-bit types");
    typedef __attribute__((address_space(3))) s16x4 lds_s4;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const unsigned at = tile + (row0 + 16 * s) * TL::kRowBytes;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(col[2 * db] + at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4*>(col[2 * db + 1] + at));
    const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<T>, both);
  }
  // fp32: the lane's columns of row `row0` + 8 (r/4) + 4 half + r%4
  __device__ __forceinline__ Columns columns(int tile, int row0, int r) const {
    static_assert(kWide, "fp32");
    return lds_get<Columns>(col[r & 7] + (tile + (row0 + 16 * (r >> 3)) * TL::kRowBytes));
  }
};

// A lane's part of a transposed result, as DP / 8 vectors of 4 neighbouring columns of its row.
template <typename T, int DP>
__device__ __forceinline__ int column_at(int i, int half) {
  if constexpr (sizeof(T) == 4 && DP > 32) {  // the order of Reads::columns
    const int r = DP == 64 ? 2 * i : i;
    return (DP / 32) * (8 * (r >> 2) + 4 * half + (r & 3));
  }
  return 32 * (i >> 2) + 8 * (i & 3) + 4 * half;
}
template <typename T, int DP>
__device__ __forceinline__ f32x4 column_values(const f32x16 (&acc)[DP / 32], int i) {
  if constexpr (sizeof(T) == 4 && DP == 128) return f32x4{acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
  if constexpr (sizeof(T) == 4 && DP == 64)
    return f32x4{acc[0][2 * i], acc[1][2 * i], acc[0][2 * i + 1], acc[1][2 * i + 1]};
  const f32x16& b = acc[i >> 2];
  const int g = 4 * (i & 3);
  return f32x4{b[g], b[g + 1], b[g + 2], b[g + 3]};
}

// acc[n][db] += (tile rows row0 .. row0+31, transposed) * block[n], where a block holds a 32x32
// result (tile rows x lane columns): values of the tile's column are the rows of the product.  N
// products share the reads of the tile.
template <typename T, int DP, int N>
__device__ __forceinline__ void mma_transposed(f32x16 (&acc)[N][DP / 32], const Reads<T, DP>& from,
                                               int tile, int row0, const f32x16 (&block)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const auto a = from.columns(tile, row0, r);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n][db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[db], block[n][r], acc[n][db], 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Frag<T> p[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) Mma<T>::put(p[n], e, block[n][8 * s + e]);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        const Frag<T> a = from.columns(tile, row0, s, db);
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n][db] = Mma<T>::mma(a, p[n], acc[n][db]);
      }
    }
  }
}
template <typename T, int DP>
__device__ __forceinline__ void mma_transposed(f32x16 (&acc)[DP / 32], const Reads<T, DP>& from, int tile,
                                               int row0, const f32x16& block) {
  mma_transposed<T, DP, 1>(reinterpret_cast<f32x16(&)[1][DP / 32]>(acc), from, tile, row0,
                           reinterpret_cast<const f32x16(&)[1]>(block));
}

// a row in registers, as the right operand of all steps over its values
template <typename T, int DP> using RowOps = Frag<T>[Tile<T, DP>::kSteps];

// right operand of one row (a query or a key) a lane, straight from global memory
template <typename T, int DP>
__device__ __forceinline__ void load_rows(RowOps<T, DP>& f, const T* row, bool there, int half, int D) {
  using TL = Tile<T, DP>;
#pragma unroll
  for (int s = 0; s < TL::kSteps; ++s) {
    const int d = (2 * s + half) * TL::kPer;
    u32x4 v = {0, 0, 0, 0};
    if (there && d < D) v = *reinterpret_cast<const u32x4*>(row + d);
    f[s] = __builtin_bit_cast(Frag<T>, v);
  }
}

// the next N instructions of the kinds in MASK, for the compiler's schedule (left to itself it reads
// each operand just before its product and waits for LDS every time)
constexpr int kMatrix = 0x008, kLdsRead = 0x100;
template <int MASK, int N> __device__ __forceinline__ void order() {
  __builtin_amdgcn_sched_group_barrier(MASK, N, 0);
}

// the tile's rows row0 .. row0+31 times the lanes' columns, added to `s` (which READS LDS reads form)
template <typename T, int DP, int READS>
__device__ __forceinline__ f32x16 mma_rows_to(f32x16 s, const Reads<T, DP>& from, int tile, int row0,
                                              const RowOps<T, DP>& f) {
#pragma unroll
  for (int c = 0; c < Tile<T, DP>::kSteps; ++c) s = Mma<T>::mma(from.rows(tile, row0, c), f[c], s);
  constexpr int kSteps = Tile<T, DP>::kSteps, kEarly = kSteps < 4 ? kSteps : 4;
  order<kLdsRead, kEarly + READS>();
#pragma unroll
  for (int c = 0; c < kSteps; ++c) {
    order<kMatrix, sizeof(T) == 4 ? 4 : 1>();
    if (c + kEarly < kSteps) order<kLdsRead, 1>();
  }
  return s;
}

template <typename T, int DP>
__device__ __forceinline__ f32x16 mma_rows(const Reads<T, DP>& from, int tile, int row0,
                                           const RowOps<T, DP>& f) {
  f32x16 zero;
#pragma unroll
  for (int r = 0; r < 16; ++r) zero[r] = 0.f;
  return mma_rows_to<T, DP, 0>(zero, from, tile, row0, f);
}
// The same for masked keys, from 0 for a key that counts and -inf for another: rows of `at`, from the
// lane's half on.  A masked row of the tile holds a finite copy of another, so its score is -inf without
// vector work (2 x 1021 x 4093 tokens, 16 heads over 4, D=64, bf16, with holes: forward 71 -> 61 us against
// two bit operations a score; 540 x 960 x 960, 2 heads of 32, fp16: backward 772 -> 727 us).
template <typename T, int DP>
__device__ __forceinline__ f32x16 mma_rows_masked(unsigned at, const Reads<T, DP>& from, int tile, int row0,
                                                  const RowOps<T, DP>& f) {
  f32x16 s;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 x = lds_get<f32x4>(at + 32 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * g + e] = x[e];
  }
  return mma_rows_to<T, DP, 4>(s, from, tile, row0, f);
}

// The keys of a 32-key block that the lane's token may see, bit j for key j: those that exist and are
// not masked (`there`, the same for every lane) and, if there is a band, 0 <= ahead - j < band with
// ahead = token - the block's first key.
__device__ __forceinline__ unsigned band_bits(unsigned there, int ahead, int band) {
  const int lo = ahead - band + 1;  // first key inside
  const unsigned upto = ahead < 0 ? 0u : ahead >= 31 ? ~0u : (2u << ahead) - 1;
  const unsigned from = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
  return there & upto & from;
}
// scores of keys whose bit is clear: -inf.  A lane holds keys 8 (r/4) + 4 half + r%4.  (Two bit
// operations a score: a compare and a select cost a wait between them.)
__device__ __forceinline__ void mask_block(f32x16& s, unsigned bits, int half) {
  const int w = (int)(bits >> (4 * half));
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const unsigned keep = (unsigned)((w << (31 - (8 * (r >> 2) + (r & 3)))) >> 31);
    s[r] = __uint_as_float((keep & __float_as_uint(s[r])) | (~keep & 0xff800000u));
  }
}
// whether a block of keys from j0 on touches (`some`), or lies inside (`all`), the band of the 32 rows
// from row0 on
struct BandOf {
  bool some, all;
  __device__ __forceinline__ BandOf(const Args& a, int row0, int j0, int n) : some(true), all(true) {
    if (a.band > 0) {
      const int i0 = a.by_group(row0), i1 = max(i0, a.by_group(min(row0 + 31, a.rows - 1))), j1 = j0 + n - 1;
      some = j0 <= i1 && j1 > i0 - a.band;
      all = j1 <= i0 && j0 > i1 - a.band;
    }
  }
};

// The key tiles of a row tile: which there are, and which keys of each count.  The first begins at the
// first key inside the band of the row tile's first row, so that the waves' bands cover few tiles.
template <int KT, bool KMASK> struct Keys {
  static constexpr uint64_t kAll = KT == 64 ? ~0ull : 0xffffffffull;
  const uint8_t* mask;
  int keys, lo, tb, te;
  __device__ __forceinline__ Keys(const Args& a, int b, int first_row, int tile_rows)
      : mask(KMASK ? a.mask + (int64_t)b * a.Lk : nullptr),
        keys(a.lengths ? min(max(a.lengths[b], 0), a.Lk) : a.Lk) {
    int hi = keys;
    lo = tb = 0;
    if (a.band > 0) {  // the keys inside the band of some row
      const int last = min(first_row + tile_rows, a.rows) - 1;
      lo = max(0, a.by_group(first_row) - a.band + 1);
      hi = min(keys, a.by_group(last) + 1);
    }
    te = hi > lo ? (hi - lo + KT - 1) / KT : 0;
  }
  __device__ __forceinline__ int first(int t) const { return lo + t * KT; }
  __device__ __forceinline__ int byte(int t, int lane) const {
    const int j = first(t) + lane;
    return lane < KT && t < te && j < keys ? mask[j] : 0;
  }
  __device__ __forceinline__ uint64_t by_length(int t) const {
    const int n = keys - first(t);
    return n >= KT ? kAll : n <= 0 ? 0ull : (1ull << n) - 1;
  }
};

// both halves of the wave see both halves' values
__device__ __forceinline__ float other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T> __device__ __forceinline__ void store4(T* p, f32x4 v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(p) = v;
  } else {
    Frag<T> f = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) Mma<T>::put(f, e, v[e]);
    const u32x4 u = __builtin_bit_cast(u32x4, f);
    *reinterpret_cast<u32x2*>(p) = u32x2{u[0], u[1]};
  }
}

// a lane's column of the transposed result of type-T operands to its row in memory (S: stored type)
template <typename T, int DP, typename S = T>
__device__ __forceinline__ void store_columns(S* row, const f32x16 (&acc)[DP / 32], float by,
                                              int half, int D) {
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
    const int d = column_at<T, DP>(i, half);
    if (d < D) store4<S>(row + d, column_values<T, DP>(acc, i) * by);
  }
}

// Workgroups go to the 8 XCDs in turn; neighbours in `id` share keys and values, so each XCD gets
// a contiguous share of the ids (its L2 then serves the re-reads).
__device__ __forceinline__ unsigned xcd_id(const Args& a) {
  const unsigned n = a.workgroups, at = a.first + blockIdx.x, x = at & 7, per = n >> 3, more = n & 7;
  return x * per + min(x, more) + (at >> 3);
}
// `n` workgroups of up to 1024 threads, in launches of fewer than 2^32 threads (more wrap without an error).
// Not a second side of the grid: that needs an exit for ids past the last, before which the kernels'
// arguments are not loaded (backward of 2 x 1021 x 4093 tokens, 16 heads over 4, D=64: 156 us against 154).
template <typename F> int launch_all(Args& a, int64_t n, const char* what, F launch) {
  constexpr int64_t kMost = 1 << 21;
  a.workgroups = (unsigned)n;
  for (int64_t first = 0; first < n; first += kMost) {
    a.first = (unsigned)first;
    launch(dim3((unsigned)(n - first < kMost ? n - first : kMost)));
    if (const int rc = check_launch(what)) return rc;
  }
  return SM_OK;
}

int64_t fwd_workspace_bytes(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t KV, int64_t D);
int64_t bwd_workspace_bytes(int64_t B, int64_t Lq, int64_t H, int64_t KV);
int check_problem(const char* what, int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                  int64_t KV, int64_t D, float scale, int64_t band);
// `group` > 0: tiles of 64 rows, `group` heads side by side, are copied by 32-bit offsets from their
// first token
int read_strides3(const int64_t* s, int64_t L, int64_t H, int64_t D, int dtype, const void* base,
                  int64_t* out, int group, const char* name);
int fwd_entry(Args& a, int dtype, void* workspace, int64_t ws_bytes, hipStream_t st);
int bwd_entry(Args& a, int dtype, void* workspace, int64_t ws_bytes, hipStream_t st);

}  // namespace attn
}  // namespace smcv
