// A projection shared by many requests, each with a low-rank adapter of its own (or none):
//
//   y[m] = x[m] W^T + bias + t[m] B_a^T          t[m] = s_a x[m] A_a^T          a = index[request of row m]
//
// The factor products are a few per cent of the shared one, so what costs is reading x again and every launch.  Two steps:
//   * adapter_down: t, bf16 (its half step is relative to the adapter's own share of y).  16 or 32 rows x 32 ranks per workgroup on
//     v_mfma_f32_16x16x32_bf16, both operands K-contiguous and read straight into registers; the eight waves of a workgroup
//     split K and are joined in LDS in a fixed order, because there are too few row groups to fill the chip otherwise.
//   * the shared product with t B_a^T added to its accumulators before the one rounding of y: many rows in lbmk_igemm
//     (lr_* fields), few rows here: the weight's bytes are the floor, so a workgroup of 8 waves takes
//     16 output columns of 64 rows, its waves split K, and W goes from memory into MFMA operands without LDS.
// Measured: 16 requests of one token, 1280 -> 1280, rank 16: 5.4 + 5.8 us, of which the weight's 3.3 MB are 0.7: latency of two
// launches.  8 x 1024 rows, 1280 -> 3840, rank 32: adapter_down 7.7 us (8.7 in a trace; 21 MB of x; the factor, 80 KB, is read from
// L2 by each of 256 workgroups), the whole call 86.5 ... 90.5, the shared product alone 75.5.
#include "common.h"

namespace {

__device__ __forceinline__ bf16x8 zero8() {
  const u32x4 z = {0u, 0u, 0u, 0u};
  return __builtin_bit_cast(bf16x8, z);
}

// waves over K; groups of 16 ranks that share one reading of x (one group per workgroup: 12.3 us instead of 10.6 at rank 32)
constexpr int DOWN_WAVES = 8, DOWN_GROUPS = 2;

// RG: groups of 16 rows that share one reading of the factor.  grid: (columns of t / 32, ceil(rows / (16 RG)) * requests)
template <int RG>
__global__ __launch_bounds__(64 * DOWN_WAVES) void adapter_down_kernel(const bf16_t* __restrict__ x, const bf16_t* __restrict__ down,
                                                                      const int32_t* __restrict__ index, const float* __restrict__ scaling,
                                                                      bf16_t* __restrict__ t, int rows, int K, int64_t ldx, int rank, int tk,
                                                                      int count) {
  __shared__ f32x4 part[DOWN_WAVES][RG * DOWN_GROUPS][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int blocks = (rows + 16 * RG - 1) / (16 * RG), request = blockIdx.y / blocks, m0 = (blockIdx.y - request * blocks) * 16 * RG, r0 = blockIdx.x * 32;
  const int a = index[request];
  if ((unsigned)a >= (unsigned)count) return;                  // no adapter: nobody reads these rows of t
  const bf16_t *xr[RG], *dr[DOWN_GROUPS];
#pragma unroll
  for (int i = 0; i < RG; ++i) xr[i] = x + ((int64_t)request * rows + min(m0 + 16 * i + lr, rows - 1)) * ldx + 8 * lq;
#pragma unroll
  for (int g = 0; g < DOWN_GROUPS; ++g) dr[g] = down + ((int64_t)a * rank + min(r0 + 16 * g + lr, rank - 1)) * K + 8 * lq;
  // K in chunks of 32: an equal, contiguous share per wave
  const int chunks = (K + 31) / 32, per = (chunks + DOWN_WAVES - 1) / DOWN_WAVES;
  const int c0 = wave * per, c1 = min(c0 + per, chunks);
  f32x4 acc[RG][DOWN_GROUPS];
#pragma unroll
  for (int i = 0; i < RG; ++i)
#pragma unroll
    for (int g = 0; g < DOWN_GROUPS; ++g) acc[i][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 5
  for (int c = c0; c < c1; ++c) {
    const bool in = 32 * c + 8 * lq < K;                       // K % 8 == 0
    bf16x8 fx[RG];
#pragma unroll
    for (int i = 0; i < RG; ++i) fx[i] = in ? *(const bf16x8*)(xr[i] + 32 * c) : zero8();
#pragma unroll
    for (int g = 0; g < DOWN_GROUPS; ++g) {
      const bf16x8 fd = in ? *(const bf16x8*)(dr[g] + 32 * c) : zero8();
#pragma unroll
      for (int i = 0; i < RG; ++i) acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fd, fx[i], acc[i][g], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < RG; ++i)
#pragma unroll
    for (int g = 0; g < DOWN_GROUPS; ++g) part[wave][i * DOWN_GROUPS + g][lane] = acc[i][g];
  __syncthreads();
  const float s = scaling ? scaling[a] : 1.f;
  // a wave joins one group of ranks at a time.  Lane: row m0 + 16 i + lr, ranks 4 lq .. + 3 of the group; ranks from `rank` on are zeros
  for (int j = wave; j < RG * DOWN_GROUPS; j += DOWN_WAVES) {
    const int m = m0 + 16 * (j / DOWN_GROUPS) + lr, n = r0 + 16 * (j % DOWN_GROUPS) + 4 * lq;
    if (m >= rows) continue;
    f32x4 v = part[0][j][lane];
#pragma unroll
    for (int w = 1; w < DOWN_WAVES; ++w) v += part[w][j][lane];
    u16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = f2bf(n + e < rank ? v[e] * s : 0.f);
    *(u16x4*)(t + ((int64_t)request * rows + m) * tk + n) = o;
  }
}

constexpr int FEW_WAVES = 8, FEW_ROWS = 64;       // rows of a workgroup

// MT: row groups of 16.  grid: (ceil(N / 16), ceil(M / 64))
template <int MT>
__global__ __launch_bounds__(64 * FEW_WAVES) void adapter_few_kernel(const bf16_t* __restrict__ x, const bf16_t* __restrict__ w,
                                                                   const float* __restrict__ bias, const bf16_t* __restrict__ t,
                                                                   const bf16_t* __restrict__ up, const int32_t* __restrict__ index,
                                                                   bf16_t* __restrict__ y, int M, int rows, int N, int K, int64_t ldx, int ldw,
                                                                   int64_t ldy, int rank, int tk, int count) {
  __shared__ f32x4 part[FEW_WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lq = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * FEW_ROWS;
  const bf16_t* wr = w + (int64_t)min(n0 + lr, N - 1) * ldw + 8 * lq;
  const bf16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = x + (int64_t)min(m0 + 16 * i + lr, M - 1) * ldx + 8 * lq;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = (K + 31) / 32;
  // the waves take chunks in turn: eight of them read 512 consecutive bytes of each row of W
#pragma unroll 4
  for (int c = wave; c < chunks; c += FEW_WAVES) {
    const bool in = 32 * c + 8 * lq < K;
    const bf16x8 fw = in ? *(const bf16x8*)(wr + 32 * c) : zero8();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const bf16x8 fx = in ? *(const bf16x8*)(xr[i] + 32 * c) : zero8();
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, fx, acc[i], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  // output (m, n): four neighbouring columns per thread, as they lie in the accumulators
  for (int o = threadIdx.x; o < MT * 64; o += 64 * FEW_WAVES) {
    const int i = o >> 6, l = o & 63, m = m0 + 16 * i + (l & 15), n = n0 + 4 * (l >> 4);
    if (m >= M || n >= N) continue;                            // N % 4 == 0
    f32x4 v = part[0][i][l];
#pragma unroll
    for (int k = 1; k < FEW_WAVES; ++k) v += part[k][i][l];
    if (bias)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bias[n + e];
    const int a = index[m / rows];
    if ((unsigned)a < (unsigned)count) {
      const bf16_t* tr = t + (int64_t)m * tk;
      const bf16_t* ur = up + ((int64_t)a * N + n) * rank;
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      if ((rank & 7) == 0) {
        for (int k = 0; k < rank; k += 8) {
          const u16x8 tv = *(const u16x8*)(tr + k);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u16x8 uv = *(const u16x8*)(ur + (int64_t)e * rank + k);
#pragma unroll
            for (int q = 0; q < 8; ++q) d[e] = fmaf(bf2f(tv.v[q]), bf2f(uv.v[q]), d[e]);
          }
        }
      } else {
        for (int k = 0; k < rank; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = fmaf(bf2f(tr[k]), bf2f(ur[(int64_t)e * rank + k]), d[e]);
      }
      v += d;
    }
    u16x4 ov;
#pragma unroll
    for (int e = 0; e < 4; ++e) ov.v[e] = f2bf(v[e]);
    *(u16x4*)(y + (int64_t)m * ldy + n) = ov;
  }
}

}  // namespace

extern "C" int lbmk_adapter_down(const void* x, const void* down, const int32_t* index, const float* scaling, void* t, int requests,
                                 int rows, int K, int64_t ldx, int rank, int tk, int count, void* stream) {
  LBMK_REQUIRE(requests >= 0 && rows >= 0 && K > 0 && K % 8 == 0 && rank > 0 && rank <= 256 && count > 0, "adapter_down: sizes");
  LBMK_REQUIRE(tk % 32 == 0 && tk >= rank && tk - rank < 32, "adapter_down: t has %d columns for rank %d (rounded up to 32)", tk, rank);
  if (requests == 0 || rows == 0) return LBMK_OK;
  LBMK_REQUIRE(x && down && index && t && lbmk_aligned(x, 16) && lbmk_aligned(down, 16) && lbmk_aligned(t, 16) && lbmk_aligned(index, 4) &&
                   (!scaling || lbmk_aligned(scaling, 4)), "adapter_down: null or misaligned pointer");
  LBMK_REQUIRE(ldx % 8 == 0 && ldx >= K, "adapter_down: row stride %lld", (long long)ldx);
  const int64_t groups = (int64_t)requests * ((rows + 15) / 16);
  LBMK_REQUIRE(groups < (1ll << 31) && (int64_t)requests * rows < (1ll << 31), "adapter_down: too many rows");
  // (grid.y carries the row groups and is limited to 65535: larger batches go in slices of whole requests)
  // Two groups of rows per workgroup read the factor half as often, where that still leaves two workgroups per CU.  One against two,
  // with eight waves: 8 requests of 1024 rows, K 1280, rank 32: 9.6 / 7.7 us; 2 of 4096, 640, 64: 9.7 / 7.6; 4 of 1024, 640, 16: 4.0 /
  // 4.5; 20 of 33, 2560, 16: 8.0 / 10.3.  (Four groups: 10.1 us for the first.  Four waves: single tokens of K 1280 4.7 us instead of 4.3.)
  const int rg = (int64_t)requests * ((rows + 15) / 16) >= 2ll * lbmk_num_cus() && rows > 16 ? 2 : 1, per = (rows + 16 * rg - 1) / (16 * rg), most = 65535 / per;
  LBMK_REQUIRE(most > 0, "adapter_down: %d rows per request (at most %d)", rows, 65535 * 16);
  for (int r = 0; r < requests; r += most) {
    const int n = requests - r < most ? requests - r : most;
#define DOWN(RG)                                                                                                                          \
  hipLaunchKernelGGL((adapter_down_kernel<RG>), dim3(tk / 32, n * per), dim3(64 * DOWN_WAVES), 0, (hipStream_t)stream,                     \
                     (const bf16_t*)x + (int64_t)r * rows * ldx, (const bf16_t*)down, index + r, scaling, (bf16_t*)t + (int64_t)r * rows * tk, rows, K, \
                     ldx, rank, tk, count)
    if (rg > 1) DOWN(2);
    else DOWN(1);
#undef DOWN
  }
  return lbmk_check_launch("adapter_down");
}

// Both sides measured, the call with lbmk_igemm against the one with the few-rows kernel (layers 1280 -> 1280, 640 -> 5120,
// 2560 -> 640, rank 16): 128 rows, of 8, 16 or 32 per request: 18 ... 30 us against 15 ... 23; 256 rows, of 4: 23 / 22 / 33
// against 20 / 25 / 23, of 16: 19 / 18 / 29 against 21 / 25 / 24.  A tile of lbmk_igemm takes one step of its factor loop per
// request in it, so single rows cost it most: 512 of them 44 / 44 / 61 against 29 / 50 / 39, 1024 48 / 92 / 65 against 52 / 85 / 56.
extern "C" int lbmk_adapter_few_suits(int requests, int rows) {
  const int64_t M = (int64_t)requests * rows;
  return M <= 128 || (rows <= 2 && M <= 512);
}

extern "C" int lbmk_adapter_linear_few(const void* x, const void* w, const float* bias, const void* t, const void* up, const int32_t* index,
                                       void* y, int requests, int rows, int N, int K, int64_t ldx, int ldw, int64_t ldy, int rank, int tk, int count,
                                       void* stream) {
  LBMK_REQUIRE(requests >= 0 && rows >= 0 && (int64_t)requests * rows <= 65535 * FEW_ROWS, "adapter_linear_few: %d requests of %d rows (at most %d rows)",
               requests, rows, 65535 * FEW_ROWS);
  LBMK_REQUIRE(N > 0 && N % 4 == 0 && K > 0 && K % 8 == 0 && rank > 0 && rank <= 256 && count > 0 && tk % 32 == 0 && tk >= rank, "adapter_linear_few: sizes");
  if (requests == 0 || rows == 0) return LBMK_OK;
  LBMK_REQUIRE(x && w && t && up && index && y && lbmk_aligned(x, 16) && lbmk_aligned(w, 16) && lbmk_aligned(t, 16) &&
                   lbmk_aligned(up, rank % 8 == 0 ? 16 : 2) && lbmk_aligned(index, 4) && lbmk_aligned(y, 8) && (!bias || lbmk_aligned(bias, 4)),
               "adapter_linear_few: null or misaligned pointer");
  LBMK_REQUIRE(ldx % 8 == 0 && ldx >= K && ldw % 8 == 0 && ldw >= K && ldy % 4 == 0 && ldy >= N, "adapter_linear_few: row strides");
  const int M = requests * rows;
#define FEW(MT)                                                                                                                    \
  hipLaunchKernelGGL((adapter_few_kernel<MT>), dim3((N + 15) / 16, (M + FEW_ROWS - 1) / FEW_ROWS), dim3(64 * FEW_WAVES), 0, (hipStream_t)stream, (const bf16_t*)x, \
                     (const bf16_t*)w, bias, (const bf16_t*)t, (const bf16_t*)up, index, (bf16_t*)y, M, rows, N, K, ldx, ldw, ldy, rank, tk, count)
  switch ((M + 15) / 16) {
    case 1: FEW(1); break;
    case 2: FEW(2); break;
    case 3: FEW(3); break;
    default: FEW(4); break;
  }
#undef FEW
  return lbmk_check_launch("adapter_linear_few");
}
