// Attention in which every query sees one interval [lo, hi) of keys: documents packed into a row, prefixes, causal and
// windowed masks, padded batches; scores optionally capped by a tanh and biased by the distance; grouped key heads.
//
//   s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i + Nk - Nq - j|      p_i = softmax over j in [lo_i, hi_i)      o_i = p_i V
// An empty interval gives a row of zeros.  Backward, with p recomputed from the rows' log-sum-exp and delta_i = dO_i.O_i:
//   dV = P^T dO    dP = dO V^T    dS = P (dP - delta) (1 - tanh^2) scale    dQ = dS K    dK = dS^T Q
//
// Same formulation as the unmasked kernels: scores are produced transposed to the operand that they feed next
// (S^T = K Q^T, the query on the lane), so the exponentiated tile goes from registers into the next product, and a
// row's statistics live in one lane pair.  Unlike those, every operand is read as it lies in memory (attn_tile.h).
// A workgroup of 4 waves owns 128 rows, 32 per wave, and walks only the keys between the first and the last that one of its
// rows sees; a wave skips a 64-key tile none of its rows sees and leaves out the comparisons where all of them see all of it.
// No atomics: results do not change from run to run.
//
// Bound by the vector ALU beside the matrix cores: a score costs 4 D operations of matrix work forward, and an exp2 (a quarter of
// the rate), a fused multiply-add, a maximum, an addition and half a conversion of vector work, as long again at 64 channels; the
// tiles come from L2.  Counted over 2 x 4096 tokens, 20 heads of 64, matrix / vector units busy: forward 35 / 61 % of the cycles, dQ
// 44 / 69, dK and dV 39 / 43; with a cap 23 / 81, 28 / 84, 26 / 67.  Short or uneven walks leave CUs without work instead: 69 ... 83 %
// of the cycles with some over a prefix or 7 documents, 56 ... 61 % over short causal documents.  Measured, 2 x 4096 tokens, 20 heads of 64: all keys 207 us forward (830 TFLOP/s), 715 us backward (600 TFLOP/s of its
// 5 products); causal 122 (700) and 386 us.  8 heads of 128, causal: 102 us (670), 366 us.  (A library product of 8192^3 reaches 1380 TFLOP/s on the same card.)
#include "attn_tile.h"

namespace {

constexpr int RB = 128;   // rows (queries or keys) of a workgroup
constexpr int TB = 64;    // tokens per tile of the walked operand

// How a product becomes a score: as it is; with a bias, which the product's accumulators start from (two operations per score instead
// of three); capped (and then biased where slopes are given).  A kernel of its own for each: as uniform branches in one kernel they
// cost registers and scheduling.  2 x 4096 tokens, 20 heads of 64, forward / backward, one kernel against three: plain 207 / 740 us
// against 207 / 715, with a bias 234 / 779 against 214 / 725, with a cap 286 / 1004 against 281 / 971; 8 heads of 128, causal, 104 / 394
// against 102 / 366.  (Forward, causal, plain, 64 channels alone gets slower, 117 -> 122 us.)
// Caps above CAP_FAR (attn_tile.h) in a fourth: the same shapes 289 / 1006 us with a cap of 50, 471 / 1290 with one of 500; 8 heads of
// 128, all keys, 186 / 821 against 237 / 961.
constexpr int LINEAR = 0, BIASED = 1, CAPPED = 2, CAPPED_FAR = 3;

typedef __attribute__((address_space(3))) char* lds_ptr;

struct Ranged {
  const bf16_t *q, *k, *v, *dout;
  bf16_t *o, *rest, *dq, *dk, *dv;     // rest: [B][Nq][H * D], what rounding took from o
  float *lse, *delta, *part;          // part: f32 [2][splits][B][Nk][Hk * D] when splits > 1
  const int32_t* ranges;              // [B][Nq][2] or null: every key
  const float* slopes;                // [H]
  int4* tiles;                        // [B][2 ceil(Nq / 64)] smallest lo, largest hi, largest lo, smallest hi of 32 queries
  int64_t sq, sk, sv, so, sg;         // batch strides
  int ldq, ldk, ldv, ldo, ldg;
  int B, H, Hk, Nq, Nk, D, blocks, parts, splits, cus, ordered, snake;
  float scale;
  ScoreMap map;
};

// a kernel's arguments by the address of its argument segment: a function that it calls reads them there (scalar loads) instead of
// taking a copy on the stack
__device__ __forceinline__ const Ranged& kernel_args(uint64_t at) {
  const uint64_t p = (uint64_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
  return *(const Ranged*)(const __attribute__((address_space(4))) Ranged*)p;
}

// lowest start of a running maximum: below every score that matters, and finite, so that a row that has seen nothing yet
// needs no special case (its exponents are -inf, its sums 0)
constexpr float M_NONE = -3.0e38f;

__device__ __forceinline__ int2 row_range(const Ranged& a, int b, int q) {
  if (!a.ranges) return make_int2(0, a.Nk);
  const int2 r = *(const int2*)(a.ranges + ((int64_t)b * a.Nq + q) * 2);
  return make_int2(max(r.x, 0), min(r.y, a.Nk));
}

// Which (row of the batch, block of queries, part, head) a workgroup takes.
//
// Two parts per block of queries: part 1 takes the queries whose keys start behind those of the block's first query, part 0 the
// others.  A block across two documents would walk the keys of both, one half of it idle in each, and it alone would set the
// kernel's time; as two parts it does not (9001 keys in 7 documents, 10 heads of 64, in one part: 106 us instead of 67, 3000
// keys with 4 heads of 160 63 instead of 32).  Under a causal mask every query is of part 0, and part 1 ends at once (2 ... 3 us of a short call).
//
// Documents and causal masks give the blocks very different numbers of keys, and a launch is often no more workgroups than the
// chip holds at once: in any fixed order some CUs get three long ones and others three short ones.  So, over long rows and with up
// to 512 items (order_blocks), every workgroup ranks them by the span of keys that a few of their queries see (ties by index: a
// permutation, whatever the ranges are) and takes the item of its own rank: the longest first.  Where the chip holds the whole
// launch at once (snake), every other round of CUs backwards, so that a CU with a long one gets a short one beside it; otherwise
// the next longest goes to the CU that is done first, as it should.
// (All LDS of a kernel is one array: with a second object the compiler waits for the tile loads in flight before it reads it.)
constexpr int ORDER_ITEMS = 512;
__device__ __forceinline__ void block_of(const Ranged& a, int* key, int& b, int& qb, int& part, int& head) {
  const int items = a.B * a.blocks * a.parts, total = items * a.H;
  int id = blockIdx.x;
  part = 0;
  if (a.ordered) {
    int& taken = key[ORDER_ITEMS];
    const int round = id / a.cus, first = round * a.cus;
    if (a.snake && (round & 1) && first + a.cus <= total) id = first + a.cus - 1 - (id - first);
    const int half = a.B * a.blocks;                    // items from here on: part 1
    for (int t = threadIdx.x; t < items; t += 256) {
      const int it = t >= half ? t - half : t, tb = it / a.blocks, r0 = (it - tb * a.blocks) * RB, r1 = min(r0 + RB, a.Nq) - 1;
      int lo = a.Nk, hi = 0;
      const int at[3] = {r0, (r0 + r1) >> 1, r1};
      int2 r[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) r[i] = row_range(a, tb, at[i]);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const bool in = r[i].x < r[i].y && (a.parts == 1 || (r[i].x >= r[0].y) == (t >= half));
        lo = in ? min(lo, r[i].x) : lo;
        hi = in ? max(hi, r[i].y) : hi;
      }
      key[t] = (min(max(hi - lo, 0) >> 5, (1 << 21) - 1) << 9) + (ORDER_ITEMS - 1 - t);
    }
    const int padded = (items + 15) & ~15;
    for (int t = items + (int)threadIdx.x; t < padded; t += 256) key[t] = -1;
    __syncthreads();
    for (int t = threadIdx.x; t < items; t += 256) {
      const int mine = key[t];
      int rank = 0;
      for (int i = 0; i < padded; i += 16) {
        int4 k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *(const int4*)(key + i + 4 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) rank += (k[j].x > mine) + (k[j].y > mine) + (k[j].z > mine) + (k[j].w > mine);
      }
      if (rank == id / a.H) taken = t;
    }
    __syncthreads();
    // (bounded: ranges that another stream changes meanwhile are no permutation, and must not lead out of the operands)
    const int item = min(max(__builtin_amdgcn_readfirstlane(taken), 0), items - 1);
    part = item >= half;
    const int it = part ? item - half : item;
    b = it / a.blocks;
    qb = it - b * a.blocks;
    head = id % a.H;
  } else {      // the last rows first: with a causal mask they have the most keys
    const int hb = id % (a.H * a.B), at = id / (a.H * a.B);
    part = at >= a.blocks;
    qb = a.blocks - 1 - (part ? at - a.blocks : at);
    b = hb / a.H;
    head = hb - b * a.H;
  }
  // (uniform, and the compiler has to know: it would loop over the lanes' tile descriptors)
  b = __builtin_amdgcn_readfirstlane(b);
  qb = __builtin_amdgcn_readfirstlane(qb);
  part = __builtin_amdgcn_readfirstlane(part);
  head = __builtin_amdgcn_readfirstlane(head);
}

// whether query row `range` belongs to this part of the block that starts with query `first`
__device__ __forceinline__ bool of_part(const Ranged& a, int b, int first, int part, int2 range) {
  return a.parts == 1 || (range.x >= row_range(a, b, first).y) == (part != 0);
}

// the walked interval of a workgroup and what its waves need to know about theirs
struct Walk {
  int begin, end;            // keys that some row of the workgroup sees
  int lo_min, hi_max;        // of this wave's rows (an empty row: none)
  int lo_max, hi_min;        // keys that all of them see
  bool any;                  // some row is this workgroup's
};

// `mine`: the row is this workgroup's (another part's counts as one that is not there)
__device__ __forceinline__ Walk walk_of(int2 r, bool mine, int wave, int* sm) {
  const bool empty = r.x >= r.y;
  Walk w;
  w.lo_min = wave_min_i(empty || !mine ? 0x7fffffff : r.x);
  w.hi_max = wave_max_i(empty || !mine ? 0 : r.y);
  w.lo_max = wave_max_i(!mine ? 0 : empty ? 0x7fffffff : r.x);
  w.hi_min = wave_min_i(!mine ? 0x7fffffff : empty ? 0 : r.y);
  const bool some = __builtin_amdgcn_ballot_w64(mine) != 0;
  if ((threadIdx.x & 63) == 0) {
    sm[wave] = w.lo_min;
    sm[4 + wave] = w.hi_max;
    sm[8 + wave] = some;
  }
  __syncthreads();
  w.begin = __builtin_amdgcn_readfirstlane(min(min(sm[0], sm[1]), min(sm[2], sm[3])));
  w.end = __builtin_amdgcn_readfirstlane(max(max(sm[4], sm[5]), max(sm[6], sm[7])));
  w.any = __builtin_amdgcn_readfirstlane(sm[8] | sm[9] | sm[10] | sm[11]) != 0;
  return w;
}

// whether a wave of the workgroup says so (and every wave is done with what it did before).  The last barrier: a wave that has
// the answer starts the second walk, whose walk_of writes the same words, and a wave that had not read them yet would take its
// own way out, its share of the tiles unstaged.
__device__ __forceinline__ bool any_wave(bool x, int wave, int* sm) {
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[wave] = x;
  __syncthreads();
  const bool any = __builtin_amdgcn_readfirstlane(sm[0] | sm[1] | sm[2] | sm[3]) != 0;
  __syncthreads();
  return any;
}

template <int DH, int KS, int MAP, class Form>
__device__ __forceinline__ bool ranged_fwd_body(const Ranged& a, char* smem) {
  constexpr bool GUARD = Form::guard;
  using T = Tile<DH>;
  constexpr int DT = T::DT, NI = T::CPR / 4, STAGE = 2 * TB * T::ROW;
  int* span = (int*)(smem + 2 * STAGE);

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 31, h = lane >> 5;
  int b, qb, part, head;
  block_of(a, (int*)smem, b, qb, part, head);
  const int khead = head / (a.H / a.Hk);
  const int q0 = qb * RB + wave * 32, q = q0 + r, qr = min(q, a.Nq - 1);

  const int2 range = row_range(a, b, qr);
  const bool mine = of_part(a, b, qb * RB, part, range);
  const Walk w = walk_of(range, mine, wave, span);
  if (!w.any) return false;
  const bf16_t* K = a.k + b * a.sk + (int64_t)khead * a.D;
  const bf16_t* V = a.v + b * a.sv + (int64_t)khead * a.D;

  bf16x8 qf[KS];
  load_frags<KS>(a.q + b * a.sq + (int64_t)qr * a.ldq + (int64_t)head * a.D, h, a.D, qf);
  const float slope = MAP != LINEAR && a.map.biased ? a.slopes[head] * a.map.slope : 0.f;
  const int pos = qr + a.Nk - a.Nq;
  const unsigned len = mine ? (unsigned)max(range.y - range.x, 0) : 0u;

  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m_run = M_NONE, l_run = 0.f;
  // the maximum may lag behind a row's by 2^LAG: p <= 256, and the accumulators are rescaled a few times per row, not per tile
  constexpr float LAG = 8.f;

  unsigned place[NI];
  T::template places<NI, TB>(t, 256, a.D, place);
  int kr[T::RK], clo[T::CD], chi[T::CD];
#pragma unroll
  for (int ks = 0; ks < T::RK; ++ks) kr[ks] = T::row_off(r, ks, h);
#pragma unroll
  for (int dt = 0; dt < T::CD; ++dt) T::col_off(lane, dt, clo[dt], chi[dt]);

  auto stage = [&](int kv0, char* buf) __attribute__((always_inline)) {
    T::template stage<NI, TB>(K, kv0, w.end, a.ldk, a.D, place, wave, 4, buf);
    T::template stage<NI, TB>(V, kv0, w.end, a.ldv, a.D, place, wave, 4, buf + TB * T::ROW);
  };
  bool bad = false;                  // a masked tile holds values that are not finite, and the sums are worth nothing
  if (w.begin < w.end) stage(w.begin, smem);
  int cur = 0;
  for (int kv0 = w.begin; kv0 < w.end; kv0 += TB) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                 // the tile is in place, and every wave is done with the other buffer
    const char* sK = smem + cur * STAGE;
    const char* sV = sK + TB * T::ROW;
    cur ^= 1;
    if (kv0 + TB < w.end) stage(kv0 + TB, smem + cur * STAGE);
    if (w.lo_min >= kv0 + TB || w.hi_max <= kv0) continue;       // no row of this wave sees the tile
    const bool masked = w.lo_max > kv0 || w.hi_min < kv0 + TB;

    f32x16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      auto product = [&](const f32x16& from) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sK + kt * 32 * T::ROW, T::row_at(kr, ks)), qf[ks], ks == 0 ? from : s[kt], 0, 0, 0);
      };
      if constexpr (MAP == BIASED) {
        f32x16 c;
        const float d0 = (float)(pos - kv0 - 4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] = -slope * fabsf(d0 - (float)(32 * kt + acc_row(e, 0)));
        product(c);
      } else {
        product(zero);
      }
    }
    if constexpr (MAP >= CAPPED) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x;
          s[kt][e] = capped<MAP == CAPPED_FAR>(a.map, s[kt][e], x);
        }
      if (a.map.biased) {
        asm volatile("" ::: "memory");
        const float d0 = (float)(pos - kv0 - 4 * h);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kt][e] = fmaf(-slope, fabsf(d0 - (float)(32 * kt + acc_row(e, 0))), s[kt][e]);
      }
    }
    if (masked) {
      asm volatile("" ::: "memory");           // (keeps the uniform condition a branch)
      const unsigned k0 = (unsigned)(kv0 + 4 * h - range.x);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + (unsigned)(32 * kt + acc_row(e, 0)) >= len) s[kt][e] = -INFINITY;
    }
    // ---- online softmax: a row is the lane pair (l, l + 32) ----
    float mx = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)          // a tree of three-input maxima
#pragma unroll
      for (int e = kt == 0 ? 1 : 0; e + 1 < 16; e += 2) mx = fmaxf(fmaxf(mx, s[kt][e]), s[kt][e + 1]);
    mx = fmaxf(mx, s[0][15]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.map.mul;
    if (__builtin_amdgcn_ballot_w64(mx > m_run + LAG) != 0) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
      m_run = m_new;
    }
    const float nm = -m_run;
    float ps0 = 0.f, ps1 = 0.f;
    bf16x8 pf[2][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float p[16];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(s[kt][e], a.map.mul, nm));
        p[e + 1] = __builtin_amdgcn_exp2f(fmaf(s[kt][e + 1], a.map.mul, nm));
        ps0 += p[e];
        ps1 += p[e + 1];
      }
      pack_column(p, pf[kt]);       // bf16 operand of P V: half a step per probability, of random sign over the keys
    }
    l_run += ps0 + ps1;

    if (GUARD && masked) {
      bf16x8 seen[2][2];
      const unsigned k0 = (unsigned)(kv0 + 4 * h - range.x);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        float one[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) one[e] = k0 + (unsigned)(32 * kt + acc_row(e, 0)) < len ? 1.f : 0.f;
        pack_column(one, seen[kt]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x16 hit = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 4; ++m)
          mfma_guarded(T::col_frag(sV + 16 * m * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[m >> 1][m & 1], seen[m >> 1][m & 1], o[dt], hit);
        poison(o[dt], hit);
      }
      continue;
    }
    if (!GUARD && masked) bad |= tile_not_finite<TB * T::ROW>(sV, lane);
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::col_frag(sV + 16 * m * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[m >> 1][m & 1], o[dt], 0, 0, 0);
  }
  if (!GUARD && any_wave(bad, wave, span)) return true;

  const float l = l_run + __shfl_xor(l_run, 32, 64);
  const bool none = range.x >= range.y;
  const float inv = none ? 0.f : 1.0f / l;
  if (q < a.Nq && mine) {
    if (a.lse && h == 0) a.lse[((int64_t)b * a.H + head) * a.Nq + q] = none ? INFINITY : m_run + __builtin_amdgcn_logf(l);
    bf16_t* op = a.o + b * a.so + (int64_t)q * a.ldo + (int64_t)head * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * dt + 8 * g + 4 * h;
        if (c < a.D) {
          u16x4 ov, rv;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = none ? 0.f : o[dt][4 * g + e] * inv;
            ov.v[e] = f2bf(v);
            rv.v[e] = f2bf(v - bf2f(ov.v[e]));
          }
          *(u16x4*)(op + c) = ov;
          if (a.rest) *(u16x4*)(a.rest + (((int64_t)b * a.Nq + q) * a.H + head) * a.D + c) = rv;
        }
      }
  }
  return false;
}

// the walk again, guarded: a call, so that its registers are not the kernel's
template <int DH, int KS, int MAP>
__device__ __attribute__((noinline)) void ranged_fwd_again(uint64_t args, lds_ptr smem) {
  ranged_fwd_body<DH, KS, MAP, Guarded>(kernel_args(args), (char*)smem);
}

// (the series of the far caps does not fit a third of the registers: 1033 instead of 471 us, 2 x 4096 tokens, 20 heads of 64)
template <int DH, int KS, int MAP>
__global__ __launch_bounds__(256, DH <= 96 && MAP != CAPPED_FAR ? 3 : DH <= 128 ? 2 : 1) void ranged_fwd_kernel(const Ranged a) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (2 * TB * Tile<DH>::ROW) + 64];
  if (ranged_fwd_body<DH, KS, MAP, Plain>(a, smem)) ranged_fwd_again<DH, KS, MAP>((uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr(), (lds_ptr)smem);
}

template <int DT>
__device__ __forceinline__ void put_rows(bf16_t* op, const f32x16 (&acc)[DT], float mul, int h, int D) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * dt + 8 * g + 4 * h;
      if (c < D) {
        u16x4 ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) ov.v[e] = f2bf(acc[dt][4 * g + e] * mul);
        *(u16x4*)(op + c) = ov;
      }
    }
}

template <int DT>
__device__ __forceinline__ void put_rows_f32(float* op, const f32x16 (&acc)[DT], float mul, int h, int D) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * dt + 8 * g + 4 * h;
      if (c < D) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[dt][4 * g + e] * mul;
        *(f32x4*)(op + c) = v;
      }
    }
}

// Two backward kernels, dQ by blocks of queries and dK / dV by blocks of keys: S and dP are formed in both, and dS K twice (dS as two
// operands), eight products instead of five, but no atomics and no f32 partial sums of dQ, and each operand that an owner keeps stays in registers.  About as long as each other (2 x 2111 tokens,
// causal documents, 20 over 5 heads of 64: 55 and 57 us).
//
// dQ and delta; also writes, for the second kernel, what the ranges of each 32 queries have in common
template <int DH, int KS, int MAP, class Form>
__device__ __forceinline__ bool ranged_bwd_dq_body(const Ranged& a, char* smem) {
  constexpr bool GUARD = Form::guard;
  using T = Tile<DH>;
  constexpr int DT = T::DT, NI = T::CPR / 4, STAGE = 2 * TB * T::ROW;
  int* span = (int*)(smem + 2 * STAGE);

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 31, h = lane >> 5;
  int b, qb, part, head;
  block_of(a, (int*)smem, b, qb, part, head);
  const int khead = head / (a.H / a.Hk);
  const int q0 = qb * RB + wave * 32, q = q0 + r, qr = min(q, a.Nq - 1);

  const int2 range = row_range(a, b, qr);
  const int groups = (a.Nq + TB - 1) / TB * 2;            // of 32 queries, the last one empty where they are an odd number
  if (a.ranges && head == 0 && part == 0 && q0 / 32 < groups) {
    const bool none = range.x >= range.y || q0 >= a.Nq;
    const int4 all = make_int4(wave_min_i(none ? 0x7fffffff : range.x), wave_max_i(none ? 0 : range.y), wave_max_i(none ? 0x7fffffff : range.x),
                               wave_min_i(none ? 0 : range.y));
    if (lane == 0) a.tiles[(int64_t)b * groups + q0 / 32] = all;
  }
  const bool mine = of_part(a, b, qb * RB, part, range);
  const Walk w = walk_of(range, mine, wave, span);
  if (!w.any) return false;
  const bf16_t* K = a.k + b * a.sk + (int64_t)khead * a.D;
  const bf16_t* V = a.v + b * a.sv + (int64_t)khead * a.D;

  bf16x8 qf[KS], gf[KS];
  load_frags<KS>(a.q + b * a.sq + (int64_t)qr * a.ldq + (int64_t)head * a.D, h, a.D, qf);
  load_frags<KS>(a.dout + b * a.sg + (int64_t)qr * a.ldg + (int64_t)head * a.D, h, a.D, gf);
  const int64_t stat = ((int64_t)b * a.H + head) * a.Nq + qr;
  float delta = 0.f;
  {
    bf16x8 of[KS];
    load_frags<KS>(a.o + b * a.so + (int64_t)qr * a.ldo + (int64_t)head * a.D, h, a.D, of);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[ks][e], (float)of[ks][e], delta);
    if (a.rest) {      // dS = P (dP - delta) cancels: the half step of o would be the largest error of dQ and dK
      load_frags<KS>(a.rest + (((int64_t)b * a.Nq + qr) * a.H + head) * a.D, h, a.D, of);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[ks][e], (float)of[ks][e], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (q < a.Nq && mine && h == 0) a.delta[stat] = delta;
  }
  const float nl = -a.lse[stat];
  const float slope = MAP != LINEAR && a.map.biased ? a.slopes[head] * a.map.slope : 0.f;
  const int pos = qr + a.Nk - a.Nq;
  const unsigned len = mine ? (unsigned)max(range.y - range.x, 0) : 0u;

  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  unsigned place[NI];
  T::template places<NI, TB>(t, 256, a.D, place);
  int kr[T::RK], clo[T::CD], chi[T::CD];
#pragma unroll
  for (int ks = 0; ks < T::RK; ++ks) kr[ks] = T::row_off(r, ks, h);
#pragma unroll
  for (int dt = 0; dt < T::CD; ++dt) T::col_off(lane, dt, clo[dt], chi[dt]);

  auto stage = [&](int kv0, char* buf) __attribute__((always_inline)) {
    T::template stage<NI, TB>(K, kv0, w.end, a.ldk, a.D, place, wave, 4, buf);
    T::template stage<NI, TB>(V, kv0, w.end, a.ldv, a.D, place, wave, 4, buf + TB * T::ROW);
  };
  bool bad = false;
  if (w.begin < w.end) stage(w.begin, smem);
  int cur = 0;
  for (int kv0 = w.begin; kv0 < w.end; kv0 += TB) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const char* sK = smem + cur * STAGE;
    const char* sV = sK + TB * T::ROW;
    cur ^= 1;
    if (kv0 + TB < w.end) stage(kv0 + TB, smem + cur * STAGE);
    if (w.lo_min >= kv0 + TB || w.hi_max <= kv0) continue;
    const bool masked = w.lo_max > kv0 || w.hi_min < kv0 + TB;
    if (!GUARD && masked) bad |= tile_not_finite<TB * T::ROW>(sK, lane);

#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      f32x16 s, dp;
      const float d0 = (float)(pos - kv0 - 32 * kt - 4 * h);
      auto product = [&](const f32x16& from) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sK + kt * 32 * T::ROW, T::row_at(kr, ks)), qf[ks], ks == 0 ? from : s, 0, 0, 0);
      };
      if constexpr (MAP == BIASED) {
        f32x16 c;
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] = -slope * fabsf(d0 - (float)acc_row(e, 0));
        product(c);
      } else {
        product(zero);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sV + kt * 32 * T::ROW, T::row_at(kr, ks)), gf[ks], ks == 0 ? zero : dp, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] -= delta;
      if constexpr (MAP >= CAPPED) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x;
          s[e] = capped<MAP == CAPPED_FAR>(a.map, s[e], x);
          dp[e] *= 4.f * x * (1.f - x);                       // 1 - tanh^2
        }
        if (a.map.biased) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 - (float)acc_row(e, 0)), s[e]);
        }
      }
      float ds[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) ds[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.map.mul, nl)) * dp[e];
      if (masked) {
        asm volatile("" ::: "memory");
        const unsigned k0 = (unsigned)(kv0 + 32 * kt + 4 * h - range.x);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + (unsigned)acc_row(e, 0) >= len) ds[e] = 0.f;
      }
      // dS as the sum of two bf16 operands: rounded to one, its half steps are as large an error of dQ as dQ's own rounding
      // (relative to 64 bits 2.5e-3 against 1.8e-3).  The second product costs 3 ... 12 % of the whole backward pass.
      bf16x8 df[2], dl[2];
      pack_column(ds, df);
#pragma unroll
      for (int e = 0; e < 16; ++e) ds[e] -= (float)(__bf16)ds[e];
      pack_column(ds, dl);
      const char* sk = sK + 32 * kt * T::ROW;
      if (GUARD && masked) {
        bf16x8 seen[2];
        float one[16];
        const unsigned k0 = (unsigned)(kv0 + 32 * kt + 4 * h - range.x);
#pragma unroll
        for (int e = 0; e < 16; ++e) one[e] = k0 + (unsigned)acc_row(e, 0) < len ? 1.f : 0.f;
        pack_column(one, seen);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x16 hit = zero;
#pragma unroll
          for (int ss = 0; ss < 2; ++ss) {
            bf16x8 fin, ind;
            split_finite(T::col_frag(sk + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), fin, ind);
            acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fin, dl[ss], acc[dt], 0, 0, 0);
            acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fin, df[ss], acc[dt], 0, 0, 0);
            hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ind, seen[ss], hit, 0, 0, 0);
          }
          poison(acc[dt], hit);
        }
        continue;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          const bf16x8 kc = T::col_frag(sk + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt));
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kc, dl[ss], acc[dt], 0, 0, 0);
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kc, df[ss], acc[dt], 0, 0, 0);
        }
    }
  }
  if (!GUARD && any_wave(bad, wave, span)) return true;
  if (q < a.Nq && mine) put_rows<DT>(a.dq + ((int64_t)b * a.Nq + q) * a.H * a.D + (int64_t)head * a.D, acc, a.scale, h, a.D);
  return false;
}

// the walk again, guarded: a call, so that its registers are not the kernel's
template <int DH, int KS, int MAP>
__device__ __attribute__((noinline)) void ranged_bwd_dq_again(uint64_t args, lds_ptr smem) {
  ranged_bwd_dq_body<DH, KS, MAP, Guarded>(kernel_args(args), (char*)smem);
}

template <int DH, int KS, int MAP>
__global__ __launch_bounds__(256, DH <= 64 ? 3 : DH <= 96 ? 2 : 1) void ranged_bwd_dq_kernel(const Ranged a) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (2 * TB * Tile<DH>::ROW) + 64];
  if (ranged_bwd_dq_body<DH, KS, MAP, Plain>(a, smem)) ranged_bwd_dq_again<DH, KS, MAP>((uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr(), (lds_ptr)smem);
}

// Which (row of the batch, block of keys, key head, part of the walk) a workgroup of the key kernel takes: as block_of, ranked by
// the number of 32-query groups that see the block, which the first kernel has summarised.
constexpr int ORDER_GROUPS = 4096;
__device__ __forceinline__ void keys_of(const Ranged& a, char* smem, int& b, int& kb, int& khead, int& cut) {
  const int blocks = (a.Nk + RB - 1) / RB, items = a.B * blocks, total = items * a.Hk * a.splits;
  int id = blockIdx.x;
  if (a.ordered) {
    const int nsub = (a.Nq + TB - 1) / TB * 2;
    int2* span = (int2*)smem;
    int* key = (int*)(smem + ORDER_GROUPS * 8 - (ORDER_ITEMS / 2 + 16) * 4);
    int& taken = key[ORDER_ITEMS / 2];
    const int round = id / a.cus, first = round * a.cus;
    if (a.snake && (round & 1) && first + a.cus <= total) id = first + a.cus - 1 - (id - first);
    for (int i = threadIdx.x; i < a.B * nsub; i += 256) {
      const int4 x = a.tiles[i];
      span[i] = make_int2(x.x, x.y);
    }
    __syncthreads();
    const int t = threadIdx.x;
    int mine = -1;
    if (t < items) {
      const int tb = t / blocks, k0 = (t - tb * blocks) * RB, k1 = min(k0 + RB, a.Nk);
      int n = 0;
#pragma unroll 8
      for (int i = 0; i < nsub; ++i) {
        const int2 x = span[tb * nsub + i];
        n += x.x < k1 && x.y > k0;
      }
      mine = (n << 8) + (ORDER_ITEMS / 2 - 1 - t);
    }
    key[t] = mine;                        // (behind the spans: there are at most ORDER_GROUPS - 256)
    __syncthreads();
    if (t < items) {
      int rank = 0;
      for (int i = 0; i < items; i += 16) {
        int4 k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *(const int4*)(key + i + 4 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) rank += (k[j].x > mine) + (k[j].y > mine) + (k[j].z > mine) + (k[j].w > mine);
      }
      if (rank == id / (a.Hk * a.splits)) taken = t;
    }
    __syncthreads();
    const int item = min(max(__builtin_amdgcn_readfirstlane(taken), 0), items - 1), rest = id % (a.Hk * a.splits);
    __syncthreads();                      // (the tiles go over it)
    b = item / blocks;
    kb = item - b * blocks;
    khead = rest % a.Hk;
    cut = rest / a.Hk;
  } else {      // the first keys first: with a causal mask most queries see them
    const int per = a.Hk * a.B * a.splits, rest = id % per;
    kb = id / per;
    cut = rest / (a.Hk * a.B);
    b = rest / a.Hk % a.B;
    khead = rest % a.Hk;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  kb = __builtin_amdgcn_readfirstlane(kb);
  khead = __builtin_amdgcn_readfirstlane(khead);
  cut = __builtin_amdgcn_readfirstlane(cut);
}

// dK and dV of 128 keys (four products per tile, and dS and P as operands, one bf16 each: half a step per weight, of random sign over
// the queries; a second operand for each, as dQ has for dS, would cost two products more.  dK and dV are 2.3 ... 2.5e-3 of their norm
// off, where their own rounding is 1.7e-3): walks the query tiles of every head that shares the key head.  With few workgroups the walk is cut
// into `splits` parts whose sums are added afterwards in their order.
template <int DH, int KS, int MAP, class Form>
__device__ __forceinline__ bool ranged_bwd_dkv_body(const Ranged& a, char* smem) {
  constexpr bool GUARD = Form::guard;
  using T = Tile<DH>;
  constexpr int DT = T::DT, NI = T::CPR / 4, STAGE = 2 * TB * T::ROW + 4 * TB * 4;
  int* span = (int*)(smem + 2 * STAGE);

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int group = a.H / a.Hk;
  int b, kb, khead, cut;
  keys_of(a, smem, b, kb, khead, cut);
  const int k0 = kb * RB, kw = k0 + wave * 32, key = kw + r, kc = min(key, a.Nk - 1);
  const int kend = min(k0 + RB, a.Nk);

  bf16x8 kf[KS], vf[KS];
  load_frags<KS>(a.k + b * a.sk + (int64_t)kc * a.ldk + (int64_t)khead * a.D, h, a.D, kf);
  load_frags<KS>(a.v + b * a.sv + (int64_t)kc * a.ldv + (int64_t)khead * a.D, h, a.D, vf);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[i][e] = dv[i][e] = 0.f;

  unsigned place[NI];
  T::template places<NI, TB>(t, 256, a.D, place);
  int rr[T::RK], clo[T::CD], chi[T::CD];
#pragma unroll
  for (int ks = 0; ks < T::RK; ++ks) rr[ks] = T::row_off(r, ks, h);
#pragma unroll
  for (int dt = 0; dt < T::CD; ++dt) T::col_off(lane, dt, clo[dt], chi[dt]);

  const int nqt = (a.Nq + TB - 1) / TB;
  // the summaries of a tile's two groups of 32 queries, by scalar loads (uniform, and written by the kernel before)
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  typedef const __attribute__((address_space(4))) i32x4* summary_t;
  const bool ranged = a.ranges != nullptr;
  const summary_t tiles = (summary_t)(uintptr_t)(a.tiles + (int64_t)b * 2 * nqt);
  const int4* lane_tiles = a.tiles + (int64_t)b * 2 * nqt;
  struct Seen {
    i32x4 u[2];
  };
  auto summary = [&](int qt) __attribute__((always_inline)) {
    Seen x = {};
    if (ranged) {
      x.u[0] = tiles[2 * qt];
      x.u[1] = tiles[2 * qt + 1];
    }
    return x;
  };
  // whether some of the 64 queries sees one of this workgroup's keys
  auto sees = [&](const Seen& x) __attribute__((always_inline)) {
    return !ranged || (min(x.u[0][0], x.u[1][0]) < kend && max(x.u[0][1], x.u[1][1]) > k0);
  };
  auto lane_sees = [&](int i) __attribute__((always_inline)) {
    if (i >= nqt) return false;
    if (!ranged) return true;
    const int4 x = lane_tiles[2 * (nqt - 1 - i)], y = lane_tiles[2 * (nqt - 1 - i) + 1];
    return min(x.x, y.x) < kend && max(x.y, y.y) > k0;
  };
  // a unit of work is a tile of one of the group's heads; each head's tiles are taken from the last one on: under a causal mask
  // the workgroups of a head all see the last tiles, and so read them at the same time.  The parts get equal numbers of the tiles
  // that see these keys: the first of this part, and how many
  struct Unit {
    int head, tile;
  };
  Unit first = {0, nqt - 1};
  int units;
  {
    int count = 0;
    for (int t0 = 0; t0 < nqt; t0 += 64)
      count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane_sees(t0 + lane)));
    const int64_t all = (int64_t)group * count;
    const int u0 = (int)(all * cut / a.splits);
    units = (int)(all * (cut + 1) / a.splits) - u0;
    if (units > 0) {
      int skip = u0 % count;
      for (int t0 = 0;; t0 += 64) {
        uint64_t m = __builtin_amdgcn_ballot_w64(lane_sees(t0 + lane));
        const int c = __builtin_popcountll(m);
        if (skip >= c) {
          skip -= c;
          continue;
        }
        for (; skip > 0; --skip) m &= m - 1;
        first.head = u0 / count;
        first.tile = nqt - 1 - (t0 + __builtin_ctzll(m));
        break;
      }
    }
    first.head = __builtin_amdgcn_readfirstlane(first.head);
    first.tile = __builtin_amdgcn_readfirstlane(first.tile);
    units = __builtin_amdgcn_readfirstlane(units);
  }
  auto behind = [&](Unit u) __attribute__((always_inline)) {
    const bool wrap = u.tile == 0;
    return Unit{u.head + wrap, wrap ? nqt - 1 : u.tile - 1};
  };
  // from unit i on (there is one), the first that sees the keys; x: its summaries
  auto settle = [&](Unit& i, Seen& x) __attribute__((always_inline)) {
    while (!sees(x)) {
      i = behind(i);
      x = summary(i.tile);
    }
  };
  // row statistics, one kind per wave: lse and delta of the head, first and last key of the batch row's queries
  const bf16_t* qh = a.q + b * a.sq + (int64_t)khead * group * a.D;
  const bf16_t* gh = a.dout + b * a.sg + (int64_t)khead * group * a.D;
  const int stat_row = wave < 2 ? 4 : 8;                 // bytes per query
  const int64_t stat_head = wave < 2 ? (int64_t)a.Nq * 4 : 0;
  const char* stat = wave < 2 ? (const char*)((wave == 0 ? a.lse : a.delta) + ((int64_t)b * a.H + khead * group) * a.Nq)
                              : (const char*)(a.ranges + (int64_t)b * a.Nq * 2);
  const unsigned stat_lane = (unsigned)(lane * stat_row + (wave == 3 ? 4 : 0));
  const bool stat_wanted = wave < 2 || ranged;
  auto stage = [&](Unit i, char* buf) __attribute__((always_inline)) {
    const int q0 = i.tile * TB;
    T::template stage<NI, TB>(qh + (int64_t)i.head * a.D, q0, a.Nq, a.ldq, a.D, place, wave, 4, buf);
    T::template stage<NI, TB>(gh + (int64_t)i.head * a.D, q0, a.Nq, a.ldg, a.D, place, wave, 4, buf + TB * T::ROW);
    // rows past the end read zeros
    if (stat_wanted)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc((void*)(stat + i.head * stat_head + (int64_t)q0 * stat_row), 0, min(TB, a.Nq - q0) * stat_row, 0x00020000),
          (__attribute__((address_space(3))) void*)(buf + 2 * TB * T::ROW + wave * TB * 4), 4, stat_lane, 0, 0, 0);
  };

  bool bad = false;
  int cur = 0, head = -1;
  Unit i = first, j = behind(first);
  float slope = 0.f;
  Seen x = {}, y = {};
  if (units > 0) {
    stage(i, smem);
    x = summary(i.tile);
    if (units > 1) {
      y = summary(j.tile);
      settle(j, y);
    }
  }
  for (int left = units; left > 0; --left) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const char* sQ = smem + cur * STAGE;
    const char* sG = sQ + TB * T::ROW;
    const float* sL = (const float*)(sG + TB * T::ROW);
    cur ^= 1;
    if (left > 1) stage(j, smem + cur * STAGE);
    const int qt = i.tile;
    if (MAP != LINEAR && a.map.biased && head != i.head) slope = a.slopes[khead * group + i.head] * a.map.slope;
    head = i.head;
    const Seen now = x;
    i = j;
    x = y;
    j = behind(j);
    if (left > 2) y = summary(j.tile);                  // used after this tile's products

#pragma unroll
    for (int u = 0; u < 2; ++u) {
      bool masked = false;
      if (ranged) {
        if (now.u[u][0] >= kw + 32 || now.u[u][1] <= kw) continue;      // none of these queries sees a key of this wave
        masked = now.u[u][2] > kw || now.u[u][3] < kw + 32;
      }
      const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      f32x16 s, dp;
      const float d0 = (float)(qt * TB + 32 * u + 4 * h + a.Nk - a.Nq - kc);
      auto product = [&](const f32x16& from) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sQ + u * 32 * T::ROW, T::row_at(rr, ks)), kf[ks], ks == 0 ? from : s, 0, 0, 0);
      };
      if constexpr (MAP == BIASED) {
        f32x16 c;
#pragma unroll
        for (int e = 0; e < 16; ++e) c[e] = -slope * fabsf(d0 + (float)acc_row(e, 0));
        product(c);
      } else {
        product(zero);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sG + u * 32 * T::ROW, T::row_at(rr, ks)), vf[ks], ks == 0 ? zero : dp, 0, 0, 0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = *(const f32x4*)(sL + TB + 32 * u + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * g + e] -= d4[e];
      }
      if constexpr (MAP >= CAPPED) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x;
          s[e] = capped<MAP == CAPPED_FAR>(a.map, s[e], x);
          dp[e] *= 4.f * x * (1.f - x);
        }
        if (a.map.biased) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 + (float)acc_row(e, 0)), s[e]);
        }
      }
      float p[16], ds[16], one[16];       // one: 1 where a row sees the key
      if constexpr (GUARD)
#pragma unroll
        for (int e = 0; e < 16; ++e) one[e] = 1.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = *(const f32x4*)(sL + 32 * u + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.map.mul, -l4[e]));
          ds[4 * g + e] = p[4 * g + e] * dp[4 * g + e];
        }
      }
      if (masked) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 lo = *(const int4*)(sL + 2 * TB + 32 * u + 8 * g + 4 * h);
          const int4 hi = *(const int4*)(sL + 3 * TB + 32 * u + 8 * g + 4 * h);
          const int l[4] = {lo.x, lo.y, lo.z, lo.w}, g4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (kc < l[e] || kc >= g4[e]) {
              p[4 * g + e] = ds[4 * g + e] = 0.f;
              if constexpr (GUARD) one[4 * g + e] = 0.f;
            }
        }
      }
      if (qt * TB + 32 * u + 32 > a.Nq) {      // rows past the end: their statistics read as zeros, and a bias may make p infinite
        asm volatile("" ::: "memory");
        const int past = a.Nq - (qt * TB + 32 * u + 4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (acc_row(e, 0) >= past) {
            p[e] = ds[e] = 0.f;
            if constexpr (GUARD) one[e] = 0.f;
          }
      }
      bf16x8 pf[2], df[2];
      pack_column(p, pf);
      pack_column(ds, df);
      const char* sq = sQ + 32 * u * T::ROW;
      const char* sg = sG + 32 * u * T::ROW;
      if (GUARD && masked) {
        bf16x8 seen[2];
        pack_column(one, seen);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          f32x16 hq = zero, hg = zero;
#pragma unroll
          for (int ss = 0; ss < 2; ++ss) {
            mfma_guarded(T::col_frag(sg + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[ss], seen[ss], dv[dt], hg);
            mfma_guarded(T::col_frag(sq + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), df[ss], seen[ss], dk[dt], hq);
          }
          poison(dv[dt], hg);
          poison(dk[dt], hq);
        }
        continue;
      }
      if (!GUARD && masked) bad |= tile_not_finite<32 * T::ROW>(sq, lane) | tile_not_finite<32 * T::ROW>(sg, lane);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::col_frag(sg + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[ss], dv[dt], 0, 0, 0);
          dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::col_frag(sq + 16 * ss * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), df[ss], dk[dt], 0, 0, 0);
        }
      }
    }
    if (left > 2) settle(j, y);
  }
  if (!GUARD && any_wave(bad, wave, span)) return true;
  if (key < a.Nk) {
    const int64_t at = ((int64_t)b * a.Nk + key) * a.Hk * a.D + (int64_t)khead * a.D;
    if (a.splits > 1) {
      const int64_t all = (int64_t)a.B * a.Nk * a.Hk * a.D;
      put_rows_f32<DT>(a.part + (int64_t)cut * all + at, dk, a.scale, h, a.D);
      put_rows_f32<DT>(a.part + (int64_t)(a.splits + cut) * all + at, dv, 1.f, h, a.D);
    } else {
      put_rows<DT>(a.dk + at, dk, a.scale, h, a.D);
      put_rows<DT>(a.dv + at, dv, 1.f, h, a.D);
    }
  }
  return false;
}

// the walk again, guarded: a call, so that its registers are not the kernel's
template <int DH, int KS, int MAP>
__device__ __attribute__((noinline)) void ranged_bwd_dkv_again(uint64_t args, lds_ptr smem) {
  ranged_bwd_dkv_body<DH, KS, MAP, Guarded>(kernel_args(args), (char*)smem);
}

template <int DH, int KS, int MAP>
__global__ __launch_bounds__(256, DH <= 96 ? 2 : 1) void ranged_bwd_dkv_kernel(const Ranged a) {
  __shared__ __attribute__((aligned(16))) char smem[2 * (2 * TB * Tile<DH>::ROW + 4 * TB * 4) + 64];
  if (ranged_bwd_dkv_body<DH, KS, MAP, Plain>(a, smem)) ranged_bwd_dkv_again<DH, KS, MAP>((uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr(), (lds_ptr)smem);
}

// The interval of keys that each query of a packed, padded or generated batch sees (see lbmk_key_ranges)
__global__ __launch_bounds__(256) void key_ranges_kernel(int32_t* out, const int32_t* offsets, const int32_t* prefix, const int32_t* lens,
                                                         int B, int Nq, int Nk, int docs, int64_t so, int causal, int window) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)B * Nq) return;
  const int b = (int)(i / Nq), pos = (int)(i - (int64_t)b * Nq) + Nk - Nq;
  int lo = 0, hi = lens ? min(max(lens[b], 0), Nk) : Nk;
  if (offsets) {
    // the document: the last offset at or below the position (offsets ascend; a search over anything else still ends)
    const int32_t* o = offsets + b * so;
    int l = 0, r = docs;                    // o[l] <= pos < o[r] once found
    if (pos < o[0] || pos >= o[docs]) {
      lo = hi = 0;                          // padding in front of the first or behind the last document
    } else {
      while (r - l > 1) {
        const int m = (l + r) >> 1;
        if (o[m] <= pos) l = m;
        else r = m;
      }
      lo = max(o[l], 0);
      hi = min(hi, o[r]);
    }
  }
  int last = causal ? pos + 1 : hi;
  if (prefix) last = max(last, min(lo, Nk) + min(max(prefix[b], 0), Nk));      // the first tokens (of each document) are seen by all
  hi = min(hi, last);
  if (window > 0) lo = max(lo, pos + 1 - window);
  if (pos < 0 || lo >= hi) lo = hi = 0;
  *(int2*)(out + 2 * i) = make_int2(lo, hi);
}

int pad_head(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 160; }

// parts of the key kernel's walk: enough workgroups for every CU to hold its fill (two of up to 96 channels, one wider).  Where
// ranges make the walks unequal and they are long, twice as many, so that the next part goes to the CU that is done first.  A part
// costs its f32 sums (8 bytes per element of dK and dV written and read): never more than eight, none below eight tiles.
// Measured, the whole backward pass without any cut against with: 2 x 2111 tokens causal, 20 over 5 heads of 64, 317 -> 159 us, 4096
// causal, 8 over 2 heads, 583 -> 195 us; the doubling: the documents of 9001 tokens 320 -> 282 us, 2 x 4096 with a prefix 328 -> 302.
int dkv_splits(bool ranged, int B, int H, int Hk, int Nq, int Nk, int D) {
  const int64_t blocks = (int64_t)((Nk + RB - 1) / RB) * Hk * B, work = (int64_t)(H / Hk) * ((Nq + TB - 1) / TB);
  const int64_t slots = (D <= 96 ? 2ll : 1ll) * lbmk_num_cus();
  if (blocks <= 0) return 1;
  int64_t s = (slots + blocks - 1) / blocks;
  if (ranged && blocks * s < 2 * slots && work / s >= 64) s *= 2;
  if (s > work / 8) s = work / 8;
  return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

// workgroups of the row kernels that fit a CU (their launch bounds)
int fwd_occupancy(int DHP, bool far) { return DHP <= 96 && !far ? 3 : DHP <= 128 ? 2 : 1; }
int dq_occupancy(int DHP) { return DHP <= 64 ? 3 : DHP <= 96 ? 2 : 1; }

// Ranked workgroups: few enough for the order to matter and for the ranking to be cheap, and walks long enough to pay for it (every
// workgroup ranks before it starts, 2 ... 4 us).  Both sides measured, index order -> ranked, forward and backward us: unequal
// documents, 9001 keys in 7, 10 heads of 64 86 -> 72 and 300 -> 278, 8 heads of 128 119 -> 93 and 524 -> 476; 12000 in 9, 8 of 64
// 86 -> 73 and 327 -> 292; 6000 in 5, 10 of 64 55 -> 44 and 208 -> 178; 4600 in 5, 16 of 64 50 -> 40 and 187 -> 165.  It loses where
// the launch is small or the spans fall evenly: 4200 in 6, 4 heads of 80 29 -> 32 and 98 -> 104, 8000 in 3 causal, 8 of 64 77 -> 80
// and 254 -> 258; up to 4096 keys it gains little: 3500 in 5, 10 of 64 30 -> 29 and 108 -> 106 (2 x 2111, 20 heads, causal
// documents: 26 -> 30 forward).
constexpr int ORDER_KEYS = 4096;
bool order_pays(const Ranged& a, int64_t n) { return a.ranges && a.Nk > ORDER_KEYS && n <= 4ll * a.cus; }
void order_blocks(Ranged& a, int occupancy) {
  const int64_t n = (int64_t)a.blocks * a.H * a.B;
  a.ordered = order_pays(a, n) && (int64_t)a.B * a.blocks * a.parts <= ORDER_ITEMS;
  a.snake = n <= (int64_t)occupancy * a.cus;
}

int ranged_check(const lbmk_ranged_attn_desc* p, bool bwd) {
  LBMK_REQUIRE(p, "ranged_attn: null descriptor");
  LBMK_REQUIRE(p->D >= 8 && p->D <= 160 && p->D % 8 == 0, "ranged_attn: head_dim %d (8 ... 160, a multiple of 8)", p->D);
  LBMK_REQUIRE(p->H > 0 && p->Hk > 0 && p->H % p->Hk == 0, "ranged_attn: %d heads over %d key heads", p->H, p->Hk);
  LBMK_REQUIRE(p->B >= 0 && p->Nq >= 0 && p->Nk >= 0, "ranged_attn: negative sizes");
  LBMK_REQUIRE(2ll * p->B * p->H * ((p->Nq + RB - 1) / RB) < (1ll << 31) && 8ll * p->B * p->Hk * ((p->Nk + RB - 1) / RB) < (1ll << 31) &&
                   p->Nq < (1 << 30) && p->Nk < (1 << 30) && (int64_t)(p->H / p->Hk) * ((p->Nq + TB - 1) / TB) < (1ll << 31),
               "ranged_attn: sizes");
  ScoreMap map;
  LBMK_REQUIRE(score_map(p->scale, p->cap, map), "ranged_attn: scale %g, cap %g", (double)p->scale, (double)p->cap);
  if (p->B == 0 || p->Nq == 0) return LBMK_OK;
  const void* ptr[8] = {p->q, p->o, p->dout, p->dq, p->k, p->v, p->dk, p->dv};
  const int ld[8] = {p->ldq, p->ldo, p->ldg, 0, p->ldk, p->ldv, 0, 0};
  const int64_t st[8] = {p->sq, p->so, p->sg, 0, p->sk, p->sv, 0, 0};
  for (int i = 0; i < 8; ++i) {
    if (!bwd && (i == 2 || i == 3 || i >= 6)) continue;
    if (i >= 4 && p->Nk == 0) continue;
    LBMK_REQUIRE(ptr[i] && lbmk_aligned(ptr[i], 16), "ranged_attn: null or misaligned pointer (rows start on 16 bytes)");
    if (i == 3 || i >= 6) continue;
    const int64_t wide = (int64_t)(i < 4 ? p->H : p->Hk) * p->D;
    LBMK_REQUIRE(ld[i] % 8 == 0 && ld[i] >= wide && ld[i] <= (1 << 22) && st[i] % 8 == 0 && st[i] >= 0, "ranged_attn: row stride %d, batch stride %lld",
                 ld[i], (long long)st[i]);
  }
  LBMK_REQUIRE(!p->ranges || lbmk_aligned(p->ranges, 8), "ranged_attn: misaligned ranges");
  LBMK_REQUIRE(!p->slopes || lbmk_aligned(p->slopes, 4), "ranged_attn: misaligned slopes");
  LBMK_REQUIRE(!p->rest || lbmk_aligned(p->rest, 16), "ranged_attn: misaligned rest");
  if (bwd) LBMK_REQUIRE(p->lse && p->scratch && lbmk_aligned(p->scratch, 16), "ranged_attn_bwd: no log-sum-exp or scratch");
  return LBMK_OK;
}

Ranged ranged_args(const lbmk_ranged_attn_desc* p) {
  Ranged a = {};
  a.q = (const bf16_t*)p->q; a.k = (const bf16_t*)p->k; a.v = (const bf16_t*)p->v; a.dout = (const bf16_t*)p->dout;
  a.o = (bf16_t*)p->o; a.dq = (bf16_t*)p->dq; a.dk = (bf16_t*)p->dk; a.dv = (bf16_t*)p->dv;
  a.lse = p->lse;
  a.rest = (bf16_t*)p->rest;
  a.ranges = p->ranges;
  a.slopes = p->slopes;
  a.sq = p->sq; a.sk = p->sk; a.sv = p->sv; a.so = p->so; a.sg = p->sg;
  a.ldq = p->ldq; a.ldk = p->ldk; a.ldv = p->ldv; a.ldo = p->ldo; a.ldg = p->ldg;
  a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.Nq = p->Nq; a.Nk = p->Nk; a.D = p->D;
  a.splits = 1;
  a.parts = p->ranges ? 2 : 1;
  a.cus = lbmk_num_cus();
  a.scale = p->scale;
  score_map(p->scale, p->cap, a.map);
  a.map.biased = p->slopes != nullptr;
  // without a cap the bias is in units of q.k: the product starts from it
  a.map.slope = p->cap > 0.f ? 1.4426950408889634f : 1.f / p->scale;
  a.map.mul = p->cap > 0.f ? 1.f : a.map.scale;
  return a;
}

// padded head width, and 16-channel steps of the products over the channels: heads of up to 80 leave out the sixth (2 x 4096 tokens,
// 8 heads of 80 with a prefix: 100 -> 86 us forward, 290 -> 280 backward; a third instead of four steps for 40 gains nothing)
#define BY_HEAD(D, LAUNCH, MAP)           \
  switch (((D) + 15) / 16) {              \
    case 1: case 2: LAUNCH(32, 2, MAP); break; \
    case 3: case 4: LAUNCH(64, 4, MAP); break; \
    case 5: LAUNCH(96, 5, MAP); break;         \
    case 6: LAUNCH(96, 6, MAP); break;         \
    case 7: case 8: LAUNCH(128, 8, MAP); break; \
    default: LAUNCH(160, 10, MAP); break;      \
  }
#define BY_MAP(LAUNCH)                                              \
  if (p->cap > CAP_FAR) { BY_HEAD(a.D, LAUNCH, CAPPED_FAR) }        \
  else if (p->cap > 0.f) { BY_HEAD(a.D, LAUNCH, CAPPED) }           \
  else if (a.map.biased) { BY_HEAD(a.D, LAUNCH, BIASED) }           \
  else { BY_HEAD(a.D, LAUNCH, LINEAR) }

__global__ __launch_bounds__(256) void sum_splits_kernel(const float* __restrict__ part, bf16_t* dk, bf16_t* dv, int64_t n, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;       // n is a multiple of 8
  if (i >= 2 * n) return;
  const bool second = i >= n;
  const float* p = part + (second ? (int64_t)splits * n + (i - n) : i);
  f32x4 v = *(const f32x4*)p;
  for (int s = 1; s < splits; ++s) v += *(const f32x4*)(p + (int64_t)s * n);
  u16x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o.v[e] = f2bf(v[e]);
  *(u16x4*)((second ? dv : dk) + (second ? i - n : i)) = o;
}

}  // namespace

extern "C" int lbmk_key_ranges(int32_t* ranges, const int32_t* doc_offsets, int docs, int64_t doc_stride, const int32_t* prefix,
                               const int32_t* lens, int B, int Nq, int Nk, int causal, int window, void* stream) {
  LBMK_REQUIRE(B >= 0 && Nq >= 0 && Nk >= 0 && Nq < (1 << 30) && Nk < (1 << 30) && window >= 0 && (int64_t)B * Nq < (1ll << 38), "key_ranges: sizes");
  if (B == 0 || Nq == 0) return LBMK_OK;
  LBMK_REQUIRE(ranges && lbmk_aligned(ranges, 8), "key_ranges: null or misaligned output");
  LBMK_REQUIRE(!doc_offsets || docs >= 1, "key_ranges: %d documents", docs);
  hipLaunchKernelGGL(key_ranges_kernel, dim3((unsigned)(((int64_t)B * Nq + 255) / 256)), dim3(256), 0, (hipStream_t)stream, ranges, doc_offsets, prefix,
                     lens, B, Nq, Nk, docs, doc_stride, causal, window);
  return lbmk_check_launch("key_ranges");
}

extern "C" int lbmk_ranged_attn(const lbmk_ranged_attn_desc* p, void* stream) {
  const int rc = ranged_check(p, false);
  if (rc != LBMK_OK) return rc;
  if (p->B == 0 || p->Nq == 0) return LBMK_OK;
  Ranged a = ranged_args(p);
  hipStream_t s = (hipStream_t)stream;
  a.blocks = (a.Nq + RB - 1) / RB;
  order_blocks(a, fwd_occupancy(pad_head(a.D), p->cap > CAP_FAR));
#define FWD(DHP, KSP, MAPP) hipLaunchKernelGGL((ranged_fwd_kernel<DHP, KSP, MAPP>), dim3((unsigned)((int64_t)a.blocks * a.parts * a.H * a.B)), dim3(256), 0, s, a)
  BY_MAP(FWD)
#undef FWD
  return lbmk_check_launch("ranged_attn");
}

// delta [B][H][Nq], the summaries of the queries' ranges, and the parts of the key kernel
extern "C" int64_t lbmk_ranged_attn_bwd_scratch_floats(int B, int H, int Hk, int Nq, int Nk, int D, int ranged) {
  if (B <= 0 || H <= 0 || Hk <= 0 || Nq <= 0 || H % Hk) return 0;
  const int64_t delta = ((int64_t)B * H * Nq + 3) / 4 * 4, tiles = (int64_t)B * ((Nq + TB - 1) / TB) * 8;
  const int splits = dkv_splits(ranged != 0, B, H, Hk, Nq, Nk, D);
  return delta + tiles + (splits > 1 ? 2ll * splits * B * Nk * Hk * D : 0);
}

extern "C" int lbmk_ranged_attn_bwd(const lbmk_ranged_attn_desc* p, void* stream) {
  const int rc = ranged_check(p, true);
  if (rc != LBMK_OK) return rc;
  if (p->B == 0 || p->Nq == 0) return LBMK_OK;
  Ranged a = ranged_args(p);
  a.delta = p->scratch;
  a.tiles = (int4*)(p->scratch + ((int64_t)a.B * a.H * a.Nq + 3) / 4 * 4);
  hipStream_t s = (hipStream_t)stream;
  a.blocks = (a.Nq + RB - 1) / RB;
  order_blocks(a, dq_occupancy(pad_head(a.D)));
#define DQ(DHP, KSP, MAPP) hipLaunchKernelGGL((ranged_bwd_dq_kernel<DHP, KSP, MAPP>), dim3((unsigned)((int64_t)a.blocks * a.parts * a.H * a.B)), dim3(256), 0, s, a)
  BY_MAP(DQ)
#undef DQ
  if (a.Nk > 0) {
    a.splits = dkv_splits(a.ranges != nullptr, a.B, a.H, a.Hk, a.Nq, a.Nk, a.D);
    const int64_t kblocks = (a.Nk + RB - 1) / RB, n = kblocks * a.Hk * a.B * a.splits;
    // (32 KB of LDS for the queries' spans: a stage pair of the narrowest heads is smaller)
    a.ordered = order_pays(a, n / 2) && a.D > 32 && kblocks * a.B <= ORDER_ITEMS / 2 && (int64_t)a.B * ((a.Nq + TB - 1) / TB) * 2 <= ORDER_GROUPS - 256;
    a.snake = n <= (a.D <= 96 ? 2ll : 1ll) * a.cus;
    a.part = (float*)(a.tiles + (int64_t)a.B * ((a.Nq + TB - 1) / TB) * 2);
#define DKV(DHP, KSP, MAPP) hipLaunchKernelGGL((ranged_bwd_dkv_kernel<DHP, KSP, MAPP>), dim3((unsigned)((int64_t)((a.Nk + RB - 1) / RB) * a.Hk * a.B * a.splits)), dim3(256), 0, s, a)
    BY_MAP(DKV)
#undef DKV
    if (a.splits > 1) {
      const int64_t all = (int64_t)a.B * a.Nk * a.Hk * a.D;
      hipLaunchKernelGGL(sum_splits_kernel, dim3((unsigned)((2 * all / 4 + 255) / 256)), dim3(256), 0, s, a.part, a.dk, a.dv, all, a.splits);
    }
  }
  return lbmk_check_launch("ranged_attn_bwd");
}
