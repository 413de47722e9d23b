// RMS norm of every query / key head and the rotation by the token's position, one pass, forward and backward.
//
//   xh = x * rsqrt(mean(x^2) + eps)      y = R(pos) (w * xh)        (mean over the D channels of one head)
//   g  = R(pos)^T dy     dw = sum over tokens and heads of g * xh     dx = rsqrt(..) * (g w - xh * mean(g w xh))
//
// R rotates `rot` leading channels in pairs: (j, j + rot/2), or (2j, 2j+1) when `interleaved`; pair j takes its angle from
// axis j / F of the token's position (F = rot / 2 / axes) and column j mod F of the table of cosines and sines.  The
// angles' far positions lose bits in f32, so the table is built once, in 64 bits, on the host side.
//
// Bound by memory: 4 bytes per element forward, 6 backward (bf16) and some 10 / 25 operations.  A head is held by
// L = 2^k lanes, each with the TWO chunks of VEC channels that the rotation pairs up, so the rotation needs no exchange
// between lanes and the norm a log2(L)-step butterfly.  The lanes of a group walk heads of ONE token, so its cosines and
// sines are read once and stay in registers; the next head is loaded, and kept as it lies in memory, while one is worked on.
// All statistics and gradient sums are f32; each output is rounded once.
// Measured in a trace, 4 x 4096 tokens, 20 + 20 heads of 64, bf16: 30 us forward (168 MB, 5.6 TB/s; a copy reaches 4.9), 63 us backward
// (252 MB, 4.0 TB/s) and 4 us for the weights' gradients (both backward kernels 56 us when a graph replays them); a few tokens: 4.5 us, a launch's latency.
#include "common.h"

namespace {

constexpr int NR_THREADS = 256;
constexpr int NR_HEADS = 4;        // heads per lane group and token where there are many tokens

struct NormRope {
  const void *x[2], *w[2], *dy[2];
  void* y[2];                      // forward: outputs; backward: dx
  const float2* table;             // [P][F] (cos, sin)
  const int32_t* pos;              // [tokens][axes]
  float* partial;                  // backward: [grid][2][D]
  int64_t sx[2], sdy[2], sy[2];    // batch strides (elements)
  int ldx[2], lddy[2], ldy[2];     // token strides
  int H[2];
  int D, rot, axes, F, P, tokens, N, w_f32, w_wide, wide, gpt;
  float eps;
};

// one chunk as it lies in memory: kept packed until it is used, so that many fit in flight
template <typename T, int VEC>
struct Chunk {
  static constexpr int WORDS = VEC * sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const u32x4 a = *(const u32x4*)((const uint32_t*)p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i + e] = a[e];
      }
    } else {
      const uint2 a = *(const uint2*)p;
      w[0] = a.x;
      w[1] = a.y;
    }
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) {
    // opaque to the compiler: it would unpack at the load, and carry a head in flight in twice the registers
#pragma unroll
    for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (sizeof(T) == 4) v[e] = __builtin_bit_cast(float, w[e]);
      else v[e] = __builtin_bit_cast(float, (e & 1) ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void nr_store(T* p, const float (&v)[VEC]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *(f32x4*)(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else if constexpr (VEC == 8) {
    u16x8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a.v[e] = f2bf(v[e]);
    *(u16x8*)p = a;
  } else {
    u16x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e) a.v[e] = f2bf(v[e]);
    *(u16x4*)p = a;
  }
}

// The two chunks of unit u (channel offsets; -1: none).  Paired halves: units below rot / 2 / VEC hold the chunks that
// the rotation combines; the others, and every unit of the interleaved form, two neighbouring chunks.
template <int VEC, bool INTER>
__device__ __forceinline__ void nr_chunks(int u, int D, int rot, int& a, int& b, bool& turns_a, bool& turns_b) {
  const int h = INTER ? 0 : rot / 2 / VEC;
  if (u < h) {
    a = u * VEC;
    b = a + rot / 2;
    turns_a = turns_b = true;
    return;
  }
  a = (2 * u) * VEC;               // paired halves: 2 h chunks precede, units h, h+1, ... take the rest two by two
  b = a + VEC;
  if (a >= D) a = -1;
  if (b >= D) b = -1;
  turns_a = INTER && a >= 0 && a < rot;
  turns_b = INTER && b >= 0 && b < rot;
}

// cosine / sine of `n` = N pairs from pair j0 on.  A position outside the table: NaN, never a silent wrong angle.
// Pairs of one axis lie next to each other in the table (wide: 16-byte loads); a chunk may also cross axes.
template <int N>
__device__ __forceinline__ void nr_pairs(const NormRope& d, int64_t token, int j0, float* c, float* s) {
  const int32_t* pos = d.pos + token * d.axes;
  if (d.wide) {
    const int ax = j0 / d.F, p = pos[ax], pc = min(max(p, 0), d.P - 1);
    const f32x4* row = (const f32x4*)(d.table + (int64_t)pc * d.F + (j0 - ax * d.F));
    const float bad = pc == p ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const f32x4 v = row[e / 2];
      c[e] = v[0] + bad;
      s[e] = v[1] + bad;
      c[e + 1] = v[2] + bad;
      s[e + 1] = v[3] + bad;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int j = j0 + e, ax = j / d.F, p = pos[ax], pc = min(max(p, 0), d.P - 1);
      const float2 v = d.table[(int64_t)pc * d.F + (j - ax * d.F)];
      const float bad = pc == p ? 0.f : __builtin_nanf("");
      c[e] = v.x + bad;
      s[e] = v.y + bad;
    }
  }
}

// of the lane's chunks: VEC pairs for two chunks that the rotation combines, VEC / 2 per chunk when interleaved
template <int VEC, bool INTER>
__device__ __forceinline__ void nr_angles(const NormRope& d, int64_t token, int a, int b, bool ta, bool tb, float (&c)[VEC],
                                          float (&s)[VEC]) {
  if constexpr (INTER) {
    if (ta) nr_pairs<VEC / 2>(d, token, a / 2, c, s);
    if (tb) nr_pairs<VEC / 2>(d, token, b / 2, c + VEC / 2, s + VEC / 2);
  } else {
    if (ta) nr_pairs<VEC>(d, token, a, c, s);
  }
}

// rotate (va, vb) by the angle (sign = 1) or back (sign = -1)
template <int VEC, bool INTER>
__device__ __forceinline__ void nr_rotate(float (&va)[VEC], float (&vb)[VEC], const float (&c)[VEC], const float (&s)[VEC], bool ta,
                                          bool tb, float sign) {
  if constexpr (INTER) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float ca = c[e / 2], sa = sign * s[e / 2], cb = c[VEC / 2 + e / 2], sb = sign * s[VEC / 2 + e / 2];
      const float x0 = va[e], x1 = va[e + 1], y0 = vb[e], y1 = vb[e + 1];
      if (ta) {
        va[e] = x0 * ca - x1 * sa;
        va[e + 1] = x1 * ca + x0 * sa;
      }
      if (tb) {
        vb[e] = y0 * cb - y1 * sb;
        vb[e + 1] = y1 * cb + y0 * sb;
      }
    }
  } else if (ta) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x0 = va[e], x1 = vb[e];
      va[e] = x0 * c[e] - x1 * (sign * s[e]);
      vb[e] = x1 * c[e] + x0 * (sign * s[e]);
    }
  }
}

// sum over L neighbouring lanes, on the vector ALU's lane permutes: quad swaps, then mirrors inside 8 and 16 lanes (by then all
// lanes of a quad, or half, hold the same sum); an LDS permute per step would be the longest part of a head's chain
template <int CTRL>
__device__ __forceinline__ float nr_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float nr_sum(float v) {
  if constexpr (L >= 2) v = nr_dpp<0xb1>(v);      // quad_perm [1, 0, 3, 2]
  if constexpr (L >= 4) v = nr_dpp<0x4e>(v);      // quad_perm [2, 3, 0, 1]
  if constexpr (L >= 8) v = nr_dpp<0x141>(v);     // row_half_mirror
  if constexpr (L >= 16) v = nr_dpp<0x140>(v);    // row_mirror
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// the hardware's reciprocal root: off by one step of f32 where an exactly rounded one is off by half, which only the f32 form's
// outputs can show, and a fifth of its instructions.  It takes subnormal arguments for zeros, so those are scaled
__device__ __forceinline__ float nr_rsq(float v) {
  const bool tiny = v < 0x1p-126f;
  const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p24f : v);
  return tiny ? r * 0x1p12f : r;
}

// blockIdx.y: 0 the queries, 1 the keys
template <typename T, int VEC, bool INTER, int L, bool BWD>
__global__ __launch_bounds__(NR_THREADS) void norm_rope_kernel(NormRope d) {
  constexpr int GROUPS = NR_THREADS / L;
  const int t = threadIdx.x, u = t % L, group = t / L, z = blockIdx.y;
  const int tpb = GROUPS / d.gpt;                       // tokens per block and step
  const int sub = group % d.gpt;                        // this group's first head
  const int H = d.H[z];
  int ca, cb;
  bool ta, tb;
  nr_chunks<VEC, INTER>(u, d.D, d.rot, ca, cb, ta, tb);
  const int pa = ca < 0 ? 0 : ca, pb = cb < 0 ? 0 : cb; // idle chunks read channel 0 and count as zeros

  const void* weight = d.w[z];
  float wa[VEC], wb[VEC], dwa[VEC], dwb[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    wa[e] = wb[e] = 1.f;
    dwa[e] = dwb[e] = 0.f;
  }
  if (weight) {
    if (d.w_wide && d.w_f32) {
      Chunk<float, VEC> c;
      c.load((const float*)weight + pa);
      c.get(wa);
      c.load((const float*)weight + pb);
      c.get(wb);
    } else if (d.w_wide) {
      Chunk<bf16_t, VEC> c;
      c.load((const bf16_t*)weight + pa);
      c.get(wa);
      c.load((const bf16_t*)weight + pb);
      c.get(wb);
    } else {                       // a parameter's slot in a flat buffer need not start on 16 bytes
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        wa[e] = d.w_f32 ? ((const float*)weight)[pa + e] : bf2f(((const bf16_t*)weight)[pa + e]);
        wb[e] = d.w_f32 ? ((const float*)weight)[pb + e] : bf2f(((const bf16_t*)weight)[pb + e]);
      }
    }
  }
  const float inv_d = 1.f / (float)d.D;

  for (int64_t t0 = (int64_t)blockIdx.x * tpb; H > 0 && t0 < d.tokens; t0 += (int64_t)gridDim.x * tpb) {
    const int64_t token = t0 + group / d.gpt;
    const bool live = token < d.tokens;                 // groups past the end keep step with the butterflies, reading token 0
    const int64_t tk = live ? token : 0;
    const int64_t bb = tk / d.N, nn = tk - bb * d.N;
    const T* xr = (const T*)d.x[z] + bb * d.sx[z] + nn * d.ldx[z];
    const T* gr = BWD ? (const T*)d.dy[z] + bb * d.sdy[z] + nn * d.lddy[z] : nullptr;
    T* yr = (T*)d.y[z] + bb * d.sy[z] + nn * d.ldy[z];
    struct Head {
      Chunk<T, VEC> xa, xb, ga, gb;
    };
    auto load = [&](int h) __attribute__((always_inline)) {
      Head r;
      r.xa.load(xr + h * d.D + pa);
      r.xb.load(xr + h * d.D + pb);
      if constexpr (BWD) {
        r.ga.load(gr + h * d.D + pa);
        r.gb.load(gr + h * d.D + pb);
      }
      return r;
    };
    if (sub >= H) continue;                             // more groups than heads
    Head next = load(sub);                              // in flight while the angles are fetched
    float c[VEC], s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) c[e] = s[e] = 0.f;
    nr_angles<VEC, INTER>(d, tk, ca, cb, ta, tb, c, s);
#pragma unroll 1
    for (int h = sub; h < H; h += d.gpt) {
        Head now = next;
        if (h + d.gpt < H) next = load(h + d.gpt);      // in flight under this head's arithmetic
        float va[VEC], vb[VEC], qa = 0.f, qb = 0.f;
        now.xa.get(va);
        now.xb.get(vb);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          qa = fmaf(va[e], va[e], qa);
          qb = fmaf(vb[e], vb[e], qb);
        }
        // (a select, not a product: what an idle lane reads twice may be infinite)
        const float ms = nr_sum<L>((ca < 0 ? 0.f : qa) + (cb < 0 ? 0.f : qb)) * inv_d;
        const float rstd = nr_rsq(ms + d.eps);
        if constexpr (!BWD) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            va[e] = va[e] * rstd * wa[e];
            vb[e] = vb[e] * rstd * wb[e];
          }
          nr_rotate<VEC, INTER>(va, vb, c, s, ta, tb, 1.f);
        } else {
          float ua[VEC], ub[VEC], da = 0.f, db = 0.f;
          now.ga.get(ua);
          now.gb.get(ub);
          nr_rotate<VEC, INTER>(ua, ub, c, s, ta, tb, -1.f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            va[e] *= rstd;
            vb[e] *= rstd;
            if (live) {
              dwa[e] = fmaf(ua[e], va[e], dwa[e]);
              dwb[e] = fmaf(ub[e], vb[e], dwb[e]);
            }
            ua[e] *= wa[e];
            ub[e] *= wb[e];
            da = fmaf(ua[e], va[e], da);
            db = fmaf(ub[e], vb[e], db);
          }
          const float m = nr_sum<L>((ca < 0 ? 0.f : da) + (cb < 0 ? 0.f : db)) * inv_d;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            va[e] = rstd * (ua[e] - va[e] * m);
            vb[e] = rstd * (ub[e] - vb[e] * m);
          }
        }
        if (live && ca >= 0) nr_store<T, VEC>(yr + h * d.D + ca, va);
        if (live && cb >= 0) nr_store<T, VEC>(yr + h * d.D + cb, vb);
    }
  }

  if constexpr (BWD) {
    // the groups' sums of one block, in a fixed order: butterflies over the groups of a wave, then its four waves
    __shared__ float part[NR_THREADS / 64][256];
    const int wave = t >> 6;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float a = dwa[e], b = dwb[e];
#pragma unroll
      for (int o = L; o < 64; o <<= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
      }
      if ((t & 63) < L) {
        if (ca >= 0) part[wave][ca + e] = a;
        if (cb >= 0) part[wave][cb + e] = b;
      }
    }
    __syncthreads();
    for (int i = t; i < d.D; i += NR_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < NR_THREADS / 64; ++k) v += part[k][i];
      d.partial[((int64_t)blockIdx.x * 2 + z) * d.D + i] = v;
    }
  }
}

// dw[z][ch] = sum over blocks of partial[block][z][ch]: 16 columns per workgroup, 64 strips of blocks added in order
__global__ __launch_bounds__(1024) void norm_rope_dw_kernel(const float* __restrict__ partial, int blocks, int D, void* dwq, void* dwk,
                                                           int out_f32) {
  __shared__ float sums[64][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), strip = threadIdx.x >> 4;
  float v = 0.f;
  if (col < 2 * D)
#pragma unroll 8
    for (int b = strip; b < blocks; b += 64) v += partial[(int64_t)b * 2 * D + col];
  sums[strip][threadIdx.x & 15] = v;
  __syncthreads();
  if (strip == 0 && col < 2 * D) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 64; ++k) a += sums[k][threadIdx.x];
    void* dst = col < D ? dwq : dwk;
    if (!dst) return;
    const int ch = col < D ? col : col - D;
    if (out_f32) ((float*)dst)[ch] = a;
    else ((bf16_t*)dst)[ch] = f2bf(a);
  }
}

int nr_vec(int D, int rot, int interleaved) { return interleaved || (rot / 2) % 8 == 0 ? 8 : 4; }

int nr_lanes(int D, int vec) {
  const int units = (D / vec + 1) / 2;
  int l = 1;
  while (l < units) l <<= 1;
  return l;
}

// blocks of a launch: each reads the weights once (and, backward, writes 2 D partial sums), so a few per CU walk the tokens
int nr_blocks(int tokens, int tpb, int limit) {
  const int64_t need = ((int64_t)tokens + tpb - 1) / tpb;
  return (int)(need < limit ? need : limit);
}

constexpr int NR_BLOCKS = 2048, NR_BWD_BLOCKS = 1024;   // of the queries, and of the keys

template <typename T, int VEC, bool INTER, bool BWD>
void nr_launch(NormRope& d, int L, int blocks, hipStream_t s) {
#define NR(l) hipLaunchKernelGGL((norm_rope_kernel<T, VEC, INTER, l, BWD>), dim3(blocks, 2), dim3(NR_THREADS), 0, s, d)
  switch (L) {
    case 1: NR(1); break;
    case 2: NR(2); break;
    case 4: NR(4); break;
    case 8: NR(8); break;
    case 16: NR(16); break;
    default: NR(32); break;
  }
#undef NR
}

int nr_run(NormRope& d, int f32, int interleaved, bool bwd, hipStream_t s) {
  const int vec = nr_vec(d.D, d.rot, interleaved), L = nr_lanes(d.D, vec), groups = NR_THREADS / L;
  // lane groups per token: with many tokens four or five heads per group, so that the token's angles are read once for several
  // heads; with few tokens as many groups as there are heads.  20 + 20 heads of 64, two axes, one head per group against four,
  // forward / backward, replayed from a graph: 8 tokens 3.7 / 7.7 us against 4.6 / 8.9, 400 tokens 4.4 / 9.6 against 4.9 / 9.4, 1600 9.1 / 23.7 against
  // 6.5 / 12.4, 16384 44 / 81 against 31 / 57
  const int heads = d.H[0] > d.H[1] ? d.H[0] : d.H[1];
  const int per = (int64_t)d.tokens * heads >= 16384 ? NR_HEADS : 1;
  int gpt = 1;
  while (gpt < groups && gpt * per < heads) gpt <<= 1;
  d.gpt = gpt;
  d.wide = d.rot > 0 && d.F % (interleaved ? vec / 2 : vec) == 0 && lbmk_aligned(d.table, 16);
  const int blocks = nr_blocks(d.tokens, groups / gpt, bwd ? NR_BWD_BLOCKS : NR_BLOCKS);
#define NR_T(T)                                                        \
  do {                                                                 \
    if (interleaved) {                                                 \
      if (bwd) nr_launch<T, 8, true, true>(d, L, blocks, s);           \
      else nr_launch<T, 8, true, false>(d, L, blocks, s);              \
    } else if (vec == 8) {                                             \
      if (bwd) nr_launch<T, 8, false, true>(d, L, blocks, s);          \
      else nr_launch<T, 8, false, false>(d, L, blocks, s);             \
    } else {                                                           \
      if (bwd) nr_launch<T, 4, false, true>(d, L, blocks, s);          \
      else nr_launch<T, 4, false, false>(d, L, blocks, s);             \
    }                                                                  \
  } while (0)
  if (f32) NR_T(float);
  else NR_T(bf16_t);
#undef NR_T
  return blocks;
}

int nr_check(const lbmk_norm_rope_desc* p, bool bwd) {
  LBMK_REQUIRE(p, "norm_rope: null descriptor");
  LBMK_REQUIRE(p->D >= 8 && p->D <= 256 && p->D % 8 == 0, "norm_rope: head_dim %d (8 ... 256, a multiple of 8)", p->D);
  LBMK_REQUIRE(p->rot >= 0 && p->rot <= p->D && p->rot % 8 == 0, "norm_rope: %d rotated channels of %d (a multiple of 8)", p->rot, p->D);
  LBMK_REQUIRE(p->B >= 0 && p->N >= 0 && (int64_t)p->B * p->N < (1ll << 31), "norm_rope: batch %d, tokens %d", p->B, p->N);
  LBMK_REQUIRE(p->Hq >= 0 && p->Hk >= 0 && p->Hq <= 65536 && p->Hk <= 65536, "norm_rope: heads %d, %d", p->Hq, p->Hk);
  if (p->rot > 0) {
    LBMK_REQUIRE(p->axes >= 1 && (p->rot / 2) % p->axes == 0, "norm_rope: %d pairs over %d axes", p->rot / 2, p->axes);
  }
  const int row = p->f32 ? 4 : 8;
  const void* ptr[6] = {p->q, p->k, p->q_out, p->k_out, p->dq_out, p->dk_out};
  const int ld[6] = {p->ldq, p->ldk, p->ldqo, p->ldko, p->lddq, p->lddk};
  const int64_t st[6] = {p->sq, p->sk, p->sqo, p->sko, p->sdq, p->sdk};
  LBMK_REQUIRE(p->eps >= 0.f, "norm_rope: eps %g", (double)p->eps);
  const int we = p->w_f32 ? 4 : 2;
  LBMK_REQUIRE((!p->wq || lbmk_aligned(p->wq, we)) && (!p->wk || lbmk_aligned(p->wk, we)), "norm_rope: misaligned weight");
  if ((int64_t)p->B * p->N == 0) return LBMK_OK;      // nothing is read: the pointers may be null
  if (p->rot > 0) {
    LBMK_REQUIRE(p->table && p->pos && p->positions > 0, "norm_rope: rotation without a table or positions");
    LBMK_REQUIRE(lbmk_aligned(p->table, 8) && lbmk_aligned(p->pos, 4), "norm_rope: misaligned table or positions");
  }
  for (int i = 0; i < (bwd ? 6 : 4); ++i) {
    const int H = i % 2 ? p->Hk : p->Hq;
    if (H == 0) continue;
    LBMK_REQUIRE(ptr[i], "norm_rope: null pointer");
    LBMK_REQUIRE(lbmk_aligned(ptr[i], 16) && ld[i] % row == 0 && st[i] % row == 0, "norm_rope: rows must start on 16 bytes");
    LBMK_REQUIRE(p->N <= 1 || ld[i] >= H * p->D, "norm_rope: token stride %d below %d heads of %d", ld[i], H, p->D);
    LBMK_REQUIRE(p->B <= 1 || st[i] >= 0, "norm_rope: negative batch stride");
  }
  return LBMK_OK;
}

NormRope nr_desc(const lbmk_norm_rope_desc* p) {
  NormRope d = {};
  d.x[0] = p->q; d.x[1] = p->k;
  d.w[0] = p->wq; d.w[1] = p->wk;
  d.y[0] = p->q_out; d.y[1] = p->k_out;
  d.dy[0] = p->dq_out; d.dy[1] = p->dk_out;
  d.table = (const float2*)p->table;
  d.pos = p->pos;
  d.sx[0] = p->sq; d.sx[1] = p->sk; d.sy[0] = p->sqo; d.sy[1] = p->sko; d.sdy[0] = p->sdq; d.sdy[1] = p->sdk;
  d.ldx[0] = p->ldq; d.ldx[1] = p->ldk; d.ldy[0] = p->ldqo; d.ldy[1] = p->ldko; d.lddy[0] = p->lddq; d.lddy[1] = p->lddk;
  d.H[0] = p->Hq; d.H[1] = p->Hk;
  d.D = p->D; d.rot = p->rot; d.axes = p->rot ? p->axes : 1; d.F = p->rot ? p->rot / 2 / p->axes : 1;
  d.P = p->positions; d.tokens = p->B * p->N; d.N = p->N > 0 ? p->N : 1; d.w_f32 = p->w_f32; d.eps = p->eps;
  d.w_wide = (!p->wq || lbmk_aligned(p->wq, 16)) && (!p->wk || lbmk_aligned(p->wk, 16));
  return d;
}

}  // namespace

extern "C" int64_t lbmk_norm_rope_bwd_scratch_floats(int D) { return D > 0 ? (int64_t)NR_BWD_BLOCKS * 2 * D : 0; }

extern "C" int lbmk_norm_rope(const lbmk_norm_rope_desc* p, void* stream) {
  const int rc = nr_check(p, false);
  if (rc != LBMK_OK) return rc;
  if ((int64_t)p->B * p->N == 0 || p->Hq + p->Hk == 0) return LBMK_OK;
  NormRope d = nr_desc(p);
  nr_run(d, p->f32, p->interleaved, false, (hipStream_t)stream);
  return lbmk_check_launch("norm_rope");
}

extern "C" int lbmk_norm_rope_bwd(const lbmk_norm_rope_desc* p, float* scratch, void* dwq, void* dwk, void* stream) {
  const int rc = nr_check(p, true);
  if (rc != LBMK_OK) return rc;
  LBMK_REQUIRE(scratch && lbmk_aligned(scratch, 4), "norm_rope_bwd: no scratch");
  hipStream_t s = (hipStream_t)stream;
  int blocks = 0;
  if ((int64_t)p->B * p->N > 0 && p->Hq + p->Hk > 0) {
    NormRope d = nr_desc(p);
    d.partial = scratch;
    blocks = nr_run(d, p->f32, p->interleaved, true, s);
  }
  if (dwq || dwk)
    hipLaunchKernelGGL(norm_rope_dw_kernel, dim3((2 * p->D + 15) / 16), dim3(1024), 0, s, scratch, blocks, p->D, dwq, dwk, p->w_f32);
  return lbmk_check_launch("norm_rope_bwd");
}
