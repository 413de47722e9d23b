// Attention of a few new tokens over a cache of keys and values: the single-token form of the attention over key ranges
// (same score: tanh cap, distance bias; grouped key heads; optional window).
//
// One new token reads its whole cache once and multiplies it by a handful of rows, so the cache's bytes are the floor and
// there are too few rows to fill the chip: the keys are split.  A workgroup takes the rows that share a key head (new
// tokens x heads of the group, 32 per block) and one part of the keys; its 4 waves walk 32-key tiles of their own, each with
// its own double buffer in LDS and no barrier in the loop, the next tile in flight under the products of this one.  The
// waves' sums are joined in LDS, the parts' by a second kernel, in a fixed order.  The part's length follows the request's
// length on the device: the host needs no copy of the lengths, and parts are equal whatever the cache's capacity.
//
// Bound by memory: 64 requests of up to 8191 keys, 5 key heads of 64: 355 MB in 71 + 5 us (5.0 TB/s in the first kernel; a copy
// reaches 4.9); one request of 16000 keys (20 MB, by then in the last-level cache) 7.5 + 4.5 us: two launches' latencies.
#include "attn_tile.h"

namespace {

constexpr int CT = 32;            // keys per tile
constexpr int SPLIT_MAX = 64;

struct Cached {
  const bf16_t *q, *k, *v;
  bf16_t* o;
  float* part_o;                  // [splits][rows][D]
  float2* part_ml;                // [splits][rows]
  const int32_t* lens;            // [B]
  const float* slopes;
  int64_t sq, sk, sv;
  int ldq, ldk, ldv;
  int B, H, Hk, n, cap_rows, D, splits, window, rows, row_blocks;
  ScoreMap map;
};

constexpr float M_NONE = -3.0e38f;

// the keys [x, y) that new token tok of request b sees
__device__ __forceinline__ int2 seen_by(const Cached& a, int b, int tok) {
  const int pos = min(max(a.lens[b], 0), a.cap_rows) - a.n + tok;       // its place in the cache
  return make_int2(a.window > 0 ? max(pos + 1 - a.window, 0) : 0, max(pos + 1, 0));
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int DH>
__global__ __launch_bounds__(256) void cached_attn_kernel(const Cached a) {
  using T = Tile<DH>;
  constexpr int KS = T::KS, DT = T::DT, NI = T::CPR / 2, TILE = CT * T::ROW, WAVE = 4 * TILE;
  // per wave two stages of (K tile, V tile); the join reuses it: 4 waves x (DH x 33 sums, 32 maxima, 32 row sums)
  constexpr int JOIN = 4 * (DH * 33 + 64) * 4;
  __shared__ __attribute__((aligned(16))) char smem[4 * WAVE > JOIN ? 4 * WAVE : JOIN];
  float (*sm_m)[32] = (float (*)[32])(smem + 4 * DH * 33 * 4), (*sm_l)[32] = sm_m + 4;

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int group = a.H / a.Hk;
  const int rb = blockIdx.x % a.row_blocks, hb = blockIdx.x / a.row_blocks;
  const int b = hb / a.Hk, khead = hb - b * a.Hk;
  const int R = a.n * group, row = rb * 32 + r, rc = min(row, R - 1);
  const int tok = rc / group, head = khead * group + rc - tok * group;

  const int2 range = seen_by(a, __builtin_amdgcn_readfirstlane(b), tok);
  const int lo = range.x, hi = range.y, pos = hi - 1;     // (a token in front of the cache's start sees nothing: its position does not matter)
  const unsigned seen = (unsigned)max(hi - lo, 0);
  // keys that some row of the block sees (the last row's token is the newest), and this part of them
  const int k_begin = wave_min_i(lo), k_end = wave_max_i(hi), all_lo = wave_max_i(lo), all_hi = wave_min_i(hi);
  const int total = max(k_end - k_begin, 0);
  const int chunk = ((total + a.splits - 1) / a.splits + 4 * CT - 1) / (4 * CT) * (4 * CT);
  const int64_t at = (int64_t)chunk * blockIdx.y;
  const int c0 = at < total ? k_begin + (int)at : k_end, c1 = min(c0 + chunk, k_end);

  const bf16_t* K = a.k + b * a.sk + (int64_t)khead * a.D;
  const bf16_t* V = a.v + b * a.sv + (int64_t)khead * a.D;
  bf16x8 qf[KS];
  load_frags<KS>(a.q + b * a.sq + (int64_t)tok * a.ldq + (int64_t)head * a.D, h, a.D, qf);
  const float slope = a.map.biased ? a.slopes[head] * a.map.slope : 0.f;

  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float m_run = M_NONE, l_run = 0.f;
  constexpr float LAG = 8.f;

  unsigned place[NI];
  T::template places<NI, CT>(lane, 64, a.D, place);
  int kr[T::RK], clo[T::CD], chi[T::CD];
#pragma unroll
  for (int ks = 0; ks < T::RK; ++ks) kr[ks] = T::row_off(r, ks, h);
#pragma unroll
  for (int dt = 0; dt < T::CD; ++dt) T::col_off(lane, dt, clo[dt], chi[dt]);
  char* mine = smem + wave * WAVE;
  auto stage = [&](int kv0, int buf) __attribute__((always_inline)) {
    T::template stage<NI, CT>(K, kv0, c1, a.ldk, a.D, place, 0, 1, mine + buf * 2 * TILE);
    T::template stage<NI, CT>(V, kv0, c1, a.ldv, a.D, place, 0, 1, mine + buf * 2 * TILE + TILE);
  };

  // a wave walks alone, so it alone repeats its walk where masked places held values that are not finite
  auto walk = [&](auto form) __attribute__((always_inline)) {
  constexpr bool GUARD = decltype(form)::guard;
  bool bad = false;
  int kv0 = c0 + wave * CT, cur = 0;
  if (kv0 < c1) stage(kv0, 0);
  for (; kv0 < c1; kv0 += 4 * CT) {
    if (kv0 + 4 * CT < c1) {
      stage(kv0 + 4 * CT, cur ^ 1);
      wait_loads<2 * NI>();            // this tile's loads are the older ones
    } else {
      wait_loads<0>();
    }
    const char* sK = mine + cur * 2 * TILE;
    const char* sV = sK + TILE;
    cur ^= 1;
    const bool masked = all_lo > kv0 || all_hi < kv0 + CT;

    f32x16 s;
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::row_frag(sK, T::row_at(kr, ks)), qf[ks], ks == 0 ? zero : s, 0, 0, 0);
    if (a.map.cap_out != 0.f) {
      asm volatile("" ::: "memory");
      float x;
      if (a.map.cap_out <= CAP_FAR * 1.4426950408889634f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = capped<false>(a.map, s[e], x);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = capped<true>(a.map, s[e], x);
      }
    }
    if (a.map.biased) {
      asm volatile("" ::: "memory");
      const float f = a.map.cap_out != 0.f ? 1.f : a.map.scale;
      const float d0 = (float)(pos - kv0 - 4 * h);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(d0 - (float)acc_row(e, 0)), s[e] * f);
    }
    if (masked) {
      asm volatile("" ::: "memory");
      const unsigned k0 = (unsigned)(kv0 + 4 * h - lo);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (k0 + (unsigned)acc_row(e, 0) >= seen) s[e] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 15; e += 2) mx = fmaxf(fmaxf(mx, s[e]), s[e + 1]);
    mx = fmaxf(mx, s[15]);
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
    float p[16], ps = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.map.mul, -m_run));
      ps += p[e];
    }
    l_run += ps;
    bf16x8 pf[2];
    pack_column(p, pf);

    if (GUARD && masked) {
      bf16x8 visible[2];
      float one[16];
      const unsigned k0 = (unsigned)(kv0 + 4 * h - lo);
#pragma unroll
      for (int e = 0; e < 16; ++e) one[e] = k0 + (unsigned)acc_row(e, 0) < seen ? 1.f : 0.f;
      pack_column(one, visible);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x16 hit = zero;
#pragma unroll
        for (int m = 0; m < 2; ++m) mfma_guarded(T::col_frag(sV + 16 * m * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[m], visible[m], o[dt], hit);
        poison(o[dt], hit);
      }
      continue;
    }
    if (!GUARD && masked) bad |= tile_not_finite<TILE>(sV, lane);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int m = 0; m < 2; ++m)
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(T::col_frag(sV + 16 * m * T::ROW, T::col_at(clo, dt), T::col_at(chi, dt)), pf[m], o[dt], 0, 0, 0);
  }
  return bad;
  };
  if (walk(Plain())) {
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    m_run = M_NONE;
    l_run = 0.f;
    walk(Guarded());
  }

  // ---- join the four waves ----
  l_run += __shfl_xor(l_run, 32, 64);
  __syncthreads();                       // every wave is done with its tiles
  float* so = (float*)smem + wave * DH * 33;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) so[(32 * dt + acc_row(e, h)) * 33 + r] = o[dt][e];
  if (h == 0) {
    sm_m[wave][r] = m_run;
    sm_l[wave][r] = l_run;
  }
  __syncthreads();
  const float* all = (const float*)smem;
  for (int i = t; i < 32 * DH; i += 256) {
    const int jr = i / DH, c = i - jr * DH, out_row = rb * 32 + jr;
    if (out_row >= R || c >= a.D) continue;
    const int2 keys = seen_by(a, b, out_row / group);
    const bool none = keys.x >= keys.y;
    float m = M_NONE, l = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, sm_m[w][jr]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w][jr] - m);
      l = fmaf(f, sm_l[w][jr], l);
      v = fmaf(f, all[(w * DH + c) * 33 + jr], v);
    }
    if (a.splits == 1) {
      const int ot = out_row / group, oh = khead * group + out_row - ot * group;
      a.o[((int64_t)b * a.n + ot) * a.H * a.D + (int64_t)oh * a.D + c] = f2bf(none ? 0.f : v / l);
    } else {
      const int64_t g = (int64_t)blockIdx.y * a.rows + (int64_t)hb * R + out_row;
      a.part_o[g * a.D + c] = v;
      if (c == 0) a.part_ml[g] = make_float2(m, l);
    }
  }
}

// one workgroup per row: its 4 waves take every fourth part, 64 channels at a time
__global__ __launch_bounds__(256) void cached_join_kernel(const Cached a) {
  __shared__ float ws[SPLIT_MAX], sv[4][64];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const float2 ml = lane < a.splits ? a.part_ml[(int64_t)lane * a.rows + row] : make_float2(M_NONE, 0.f);
  const float m = wave_max(ml.x);
  const float f = __builtin_amdgcn_exp2f(ml.x - m);
  const float l = wave_sum(f * ml.y);
  if (wave == 0) ws[lane] = f;
  __syncthreads();
  const int group = a.H / a.Hk, R = a.n * group;
  const int hb = (int)(row / R), i = (int)(row - (int64_t)hb * R), b = hb / a.Hk, khead = hb - b * a.Hk;
  const int tok = i / group, head = khead * group + i - tok * group;
  const int2 keys = seen_by(a, b, tok);
  const bool none = keys.x >= keys.y;
  for (int c0 = 0; c0 < a.D; c0 += 64) {
    const int c = c0 + lane;
    float v = 0.f;
    if (c < a.D)
#pragma unroll 4
      for (int s = wave; s < a.splits; s += 4) v = fmaf(ws[s], a.part_o[((int64_t)s * a.rows + row) * a.D + c], v);
    sv[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < a.D) {
      v = (sv[0][lane] + sv[1][lane]) + (sv[2][lane] + sv[3][lane]);
      a.o[((int64_t)b * a.n + tok) * a.H * a.D + (int64_t)head * a.D + c] = f2bf(none ? 0.f : v / l);
    }
    __syncthreads();
  }
}

int cache_pad(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 160; }

// parts of the keys: some four workgroups per CU over all requests, of at least 256 keys of a full cache each.  One / two / four per
// CU, 20 over 5 heads: 64 requests of 2000 ... 8200 keys, heads of 64 97 / 91 / 84 us, of 96 160 / 146 / 141, of 128 175 / 167 / 162
// (5.0 TB/s), of 160 251 / 228 / 217; 8 requests of 1200 ... 4000 keys, 64 12.3 / 12.5 / 15.4, 128 21.3 / 23.5 / 25.5, 160 27 / 30 / 30;
// one of 16000, 64 10.9 / 10.9 / 10.9, 128 17.5 / 22.8 / 22.6.  The rule is the many requests': from 72 channels on LDS holds one
// workgroup per CU, and few requests would be 6 ... 30 % faster with one.
int cache_splits(int B, int H, int Hk, int n, int cap_rows) {
  const int64_t blocks = (int64_t)B * Hk * (((int64_t)n * (H / Hk) + 31) / 32);
  int64_t s = (4ll * lbmk_num_cus() + blocks - 1) / (blocks > 0 ? blocks : 1);
  const int64_t most = cap_rows / 256;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s > SPLIT_MAX ? SPLIT_MAX : s);
}

}  // namespace

extern "C" int64_t lbmk_cached_attn_scratch_floats(int B, int H, int Hk, int n, int cap_rows, int D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || n <= 0 || H % Hk || cap_rows <= 0) return 0;
  const int s = cache_splits(B, H, Hk, n, cap_rows);
  return s > 1 ? (int64_t)s * B * H * n * (D + 2) : 0;
}

extern "C" int lbmk_cached_attn(const lbmk_cached_attn_desc* p, void* stream) {
  LBMK_REQUIRE(p, "cached_attn: null descriptor");
  LBMK_REQUIRE(p->D >= 8 && p->D <= 160 && p->D % 8 == 0, "cached_attn: head_dim %d (8 ... 160, a multiple of 8)", p->D);
  LBMK_REQUIRE(p->H > 0 && p->Hk > 0 && p->H % p->Hk == 0, "cached_attn: %d heads over %d key heads", p->H, p->Hk);
  LBMK_REQUIRE(p->B >= 0 && p->n >= 0 && p->cap_rows >= 0 && p->cap_rows < (1 << 30) && p->window >= 0, "cached_attn: sizes");
  LBMK_REQUIRE((int64_t)p->B * p->H * p->n < (1ll << 31) && (int64_t)p->n * (p->H / p->Hk) < (1 << 30), "cached_attn: too many rows");
  Cached a = {};
  LBMK_REQUIRE(score_map(p->scale, p->cap, a.map), "cached_attn: scale %g, cap %g", (double)p->scale, (double)p->cap);
  if (p->B == 0 || p->n == 0) return LBMK_OK;
  LBMK_REQUIRE(p->q && p->o && p->lens && (p->cap_rows == 0 || (p->k && p->v)), "cached_attn: null pointer");
  LBMK_REQUIRE(lbmk_aligned(p->q, 16) && lbmk_aligned(p->k, 16) && lbmk_aligned(p->v, 16) && lbmk_aligned(p->o, 2) && lbmk_aligned(p->lens, 4) &&
                   (!p->slopes || lbmk_aligned(p->slopes, 4)), "cached_attn: misaligned pointer (rows start on 16 bytes)");
  const int ld[3] = {p->ldq, p->ldk, p->ldv};
  const int64_t st[3] = {p->sq, p->sk, p->sv};
  for (int i = 0; i < 3; ++i)
    LBMK_REQUIRE(ld[i] % 8 == 0 && ld[i] >= (i ? p->Hk : p->H) * p->D && ld[i] <= (1 << 22) && st[i] % 8 == 0 && st[i] >= 0,
                 "cached_attn: row stride %d, batch stride %lld", ld[i], (long long)st[i]);
  a.q = (const bf16_t*)p->q; a.k = (const bf16_t*)p->k; a.v = (const bf16_t*)p->v; a.o = (bf16_t*)p->o;
  a.lens = p->lens; a.slopes = p->slopes;
  a.sq = p->sq; a.sk = p->sk; a.sv = p->sv; a.ldq = p->ldq; a.ldk = p->ldk; a.ldv = p->ldv;
  a.B = p->B; a.H = p->H; a.Hk = p->Hk; a.n = p->n; a.cap_rows = p->cap_rows; a.D = p->D; a.window = p->window;
  a.rows = p->B * p->H * p->n;
  a.row_blocks = (p->n * (p->H / p->Hk) + 31) / 32;
  a.splits = cache_splits(p->B, p->H, p->Hk, p->n, p->cap_rows);
  if (a.splits > 1) {
    LBMK_REQUIRE(p->scratch && lbmk_aligned(p->scratch, 8), "cached_attn: no scratch");
    a.part_ml = (float2*)p->scratch;
    a.part_o = p->scratch + 2ll * a.splits * a.rows;
  }
  a.map.biased = p->slopes != nullptr;
  a.map.slope = 1.4426950408889634f;
  a.map.mul = p->cap > 0.f || p->slopes ? 1.f : a.map.scale;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * a.row_blocks), a.splits);
#define CACHED(DHP) hipLaunchKernelGGL((cached_attn_kernel<DHP>), grid, dim3(256), 0, s, a)
  switch (cache_pad(a.D)) {
    case 32: CACHED(32); break;
    case 64: CACHED(64); break;
    case 96: CACHED(96); break;
    case 128: CACHED(128); break;
    default: CACHED(160); break;
  }
#undef CACHED
  if (a.splits > 1) hipLaunchKernelGGL(cached_join_kernel, dim3(a.rows), dim3(256), 0, s, a);
  return lbmk_check_launch("cached_attn");
}
