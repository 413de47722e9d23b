// Tiles of bf16 rows in LDS and the MFMA operands read from them, shared by the attention kernels over key ranges.
//
// A tile is R rows (tokens) x DH channels as they lie in memory; it is written by LDS-DMA, lane-linear, and read in two
// ways: as rows (16 bytes = 8 channels of one token: operand with the channel along k) and transposed with
// ds_read_b64_tr_b16 (8 tokens of one channel: operand with the token along k).  So neither K / V nor Q / dO need a
// channel-major copy in memory.  The 16-byte slots of a row are XOR-swizzled so that both kinds of reads touch every bank
// once: 16 rows x one slot, and 4 rows x 4 neighbouring slots.
#pragma once
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

template <int DH>
struct Tile {
  static constexpr int CPR = DH / 8;           // 16-byte chunks per row
  static constexpr int ROW = DH * 2;           // bytes per row
  static constexpr int KS = DH / 16;           // 16-deep MFMA steps over the channels
  static constexpr int DT = DH / 32;           // 32-channel tiles

  // Distinct read offsets a lane keeps: at widths that are no multiple of 64 the swizzle stays within 64-byte groups, so the
  // offset of a later step is an earlier one's plus an immediate
  static constexpr int RK = DH % 64 == 0 ? KS : 2, CD = DH % 64 == 0 ? DT : 1;
  static __device__ __forceinline__ int row_at(const int (&r)[RK], int ks) { return RK == KS ? r[ks] : r[ks & 1] + 64 * (ks >> 1); }
  static __device__ __forceinline__ int col_at(const int (&c)[CD], int dt) { return CD == DT ? c[dt] : c[0] + 64 * dt; }

  // 256 bytes of banks hold 256 / ROW rows: the swizzle supplies the bits that the row offset does not
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (DH % 128 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (DH % 64 == 0) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
  }
  // where this thread's chunks lie in a tile of R rows: row | byte column << 16.  Row and column rather than byte offsets: one
  // set serves operands of any row stride.  Channels from D on: row R, which is past the end of every tile
  template <int NI, int R>
  static __device__ __forceinline__ void places(int t, int threads, int D, unsigned (&place)[NI]) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int idx = i * threads + t, row = idx / CPR, c = (idx % CPR) ^ swz(row);
      place[i] = c * 8 < D ? (unsigned)row | (unsigned)c << 20 : (unsigned)R;
    }
  }
  // stages rows [row0, min(row0 + R, end)) of src; rows from `end` on read as zeros.  `wave` is wave-uniform
  template <int NI, int R>
  static __device__ __forceinline__ void stage(const bf16_t* src, int64_t row0, int end, int ld, int D, const unsigned (&place)[NI],
                                               int wave, int waves, char* dst) {
    const int rows = min(R, end - (int)row0);
    const int bytes = ((rows - 1) * ld + D) * 2;
    const bf16_t* base = src + row0 * ld;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      // (one 24-bit multiply-add: rows of at most 2^23 bytes, below 2^31 in all; a chunk past the last row, or of row R, is past `bytes`)
      const unsigned off = __umul24(place[i] & 0xffffu, (unsigned)ld * 2u) + (place[i] >> 16);
      buffer_lds16(base, bytes, off, 0, dst + (i * waves + wave) * 1024);
    }
  }
  // operand with the channel along k: row `row`, channels 16 ks + 8 h .. + 7
  static __device__ __forceinline__ int row_off(int row, int ks, int h) { return row * ROW + (((2 * ks + h) ^ swz(row)) << 4); }
  static __device__ __forceinline__ bf16x8 row_frag(const char* tile, int off) { return *(const bf16x8*)(tile + off); }
  // operand with the token along k: channels 32 dt + (lane & 31), tokens 8 h .. 8 h + 7 (+ 16 m: add 16 m ROW): offsets of the
  // two transposing reads
  static __device__ __forceinline__ void col_off(int lane, int dt, int& lo, int& hi) {
    const int l = lane & 15, h = lane >> 5, b = (lane >> 4) & 1;
    const int ra = 8 * h + (l >> 2), rb = ra + 4, ch = 4 * dt + 2 * b + ((l & 3) >> 1);
    lo = ra * ROW + 16 * (ch ^ swz(ra)) + 8 * (l & 1);
    hi = rb * ROW + 16 * (ch ^ swz(rb)) + 8 * (l & 1);
  }
  static __device__ __forceinline__ bf16x8 col_frag(const char* tile, int lo, int hi) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tile + lo));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tile + hi));
    const s16x8 v = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return __builtin_bit_cast(bf16x8, v);
  }
};

// lane (r, h) <- X[row][16 ks + 8 h .. + 7], zero from channel D on
template <int KS>
__device__ __forceinline__ void load_frags(const bf16_t* row, int h, int D, bf16x8 (&f)[KS]) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    if (16 * ks + 8 * h < D) f[ks] = *(const bf16x8*)(row + 16 * ks + 8 * h);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) f[ks][e] = (__bf16)0.f;
  }
}

// An accumulator column (32 rows of k over the lane pair l, l + 32, in fours) as two 8-deep operand slices per lane: after the
// bf16 pack the pair swaps halves, so a lane holds rows 16 ss + 8 h .. + 7
__device__ __forceinline__ void pack_column(const float (&p)[16], bf16x8 (&f)[2]) {
#pragma unroll
  for (int ss = 0; ss < 2; ++ss) {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (__bf16)p[8 * ss + e];
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    const auto s0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const u32x4 x = {s0[0], s1[0], s0[1], s1[1]};
    f[ss] = __builtin_bit_cast(bf16x8, x);
  }
}

// Masked places hold 0 in one operand, and 0 * inf or 0 * NaN in the other would poison a sum that must not see them.  The walks
// scan each tile that has masked places (a few instructions per 16 bytes, and such tiles are few); where one holds a value that
// is not finite the whole walk is done again in a second form, whose masked tiles multiply the finite values alone and learn
// from a product of indicators (not finite x seen) which sums become NaN: seen by the mask, for a weight may be 0 at a place that
// is seen.  The first form carries none of that: with both in one loop the registers spilled and the tile loads were waited for
// at once (2.5 x slower).  Finite sums are the same bits whatever the masked places hold.
struct Plain { static constexpr bool guard = false; };
struct Guarded { static constexpr bool guard = true; };

template <int BYTES>
__device__ __forceinline__ bool tile_not_finite(const char* tile, int lane) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < BYTES / 1024; ++i) {
    const u32x4 w = *(const u32x4*)(tile + i * 1024 + lane * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) a |= (w[e] & 0x7f807f80u) + 0x00800080u;     // carries out of an exponent of all ones
  }
  return __builtin_amdgcn_ballot_w64((a & 0x80008000u) != 0) != 0;
}
// an operand's finite values, and ones where it holds others
__device__ __forceinline__ void split_finite(bf16x8 a, bf16x8& fin, bf16x8& ind) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool ok = (__builtin_bit_cast(uint16_t, (__bf16)a[e]) & 0x7f80) != 0x7f80;
    fin[e] = ok ? (__bf16)a[e] : (__bf16)0.f;
    ind[e] = ok ? (__bf16)0.f : (__bf16)1.f;
  }
}
// acc += a b over a's finite values; hit: how many of the others are `seen` (ones and zeros in b's layout)
__device__ __forceinline__ void mfma_guarded(bf16x8 a, bf16x8 b, bf16x8 seen, f32x16& acc, f32x16& hit) {
  bf16x8 fin, ind;
  split_finite(a, fin, ind);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fin, b, acc, 0, 0, 0);
  hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ind, seen, hit, 0, 0, 0);
}
__device__ __forceinline__ void poison(f32x16& acc, const f32x16& hit) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (hit[e] > 0.f) acc[e] = __builtin_nanf("");
}

// row of accumulator element e in lane half h
__device__ __forceinline__ constexpr int acc_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// What turns a product q.k into the exponent (base 2) of the softmax:
//   cap:  C tanh(scale q.k / cap), C = cap log2(e), tanh(x) = 1 - 2 / (exp(2 x) + 1)        bias: - slope |distance|
// Without a cap the scaling is left to the fused multiply-add that subtracts the maximum.
// The difference is off by a few half steps of C: 1e-5 at caps of 50, 2.5e-5 at 128, but 2e-4 at 1000 and 0.13 at 10^6.  From
// CAP_FAR on, arguments below 1/4 take tanh's series instead, whose next term is below 2^-26 of it: a few half steps of the score.
struct ScoreMap {
  float mul;        // factor still to be applied to a mapped score (scale * log2(e), or 1 when it is already in that unit)
  float scale;      // scale * log2(e)
  float cap_in;     // 2 scale log2(e) / cap
  float cap_out;    // cap log2(e); 0: no cap
  float cap_u;      // scale / cap
  float slope;      // factor of the slopes, in the units that the bias is added in
  int biased;
};
constexpr float CAP_FAR = 128.f;

// C tanh(scale s / cap), and x with 1 - tanh^2 = 4 x (1 - x)
template <bool FAR>
__device__ __forceinline__ float capped(const ScoreMap& m, float s, float& x) {
  x = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * m.cap_in) + 1.f);
  const float v = fmaf(-2.f * m.cap_out, x, m.cap_out);
  if constexpr (!FAR) return v;
  const float u = s * m.cap_u, t = u * u;
  float g = 62.f / 2835.f;
  g = fmaf(g, t, -17.f / 315.f);
  g = fmaf(g, t, 2.f / 15.f);
  g = fmaf(g, t, -1.f / 3.f);
  g = fmaf(g, t, 1.f);
  return fabsf(u) < 0.25f ? s * m.scale * g : v;
}

// a scale, a cap and what the kernels take from them: finite, and no number that f32 holds in fewer bits
inline bool score_map(float scale, float cap, ScoreMap& m) {
  const float log2e = 1.4426950408889634f, tiny = 1.17549435e-38f, huge = 0x1p126f;
  if (!(scale >= tiny && scale <= huge) || !(cap == 0.f || (cap >= tiny && cap <= huge))) return false;
  m.scale = scale * log2e;
  m.cap_in = cap > 0.f ? 2.f * scale * log2e / cap : 0.f;
  m.cap_out = cap * log2e;
  m.cap_u = cap > 0.f ? scale / cap : 0.f;
  return m.cap_in <= huge;
}

}  // namespace
