// Gated feed-forward projection, for MI355X (gfx950):
//
//   g = x Wg^T, u = x Wu^T (x [M, D]; Wg, Wu [F, D], the contraction index
//   contiguous),  h = a(g) u,   a one of
//     silu    g s(g)
//     gelu    g s(2 sqrt(2 / pi) (g + 0.044715 g^3))    (the tanh form)
//     sigmoid s(g),                                      s(z) = 1 / (1 + e^-z)
//   and the elementwise part of its backward, from dh and g and u in fp32, either
//   computed again or kept by the forward:
//     dg = dh u a'(g),  du = dh a(g),  written as [dg | du] [M, 2F].
//
// Both products of one output meet in one lane's accumulators, so h (or
// [dg | du]) is all that has to be written, and the values that meet are fp32:
// the one rounding is that of the output.
//
// [dg | du] is rounded to bf16 because the products that follow, with the weights
// and with x, run on the bf16 matrix cores; in two bf16 parts or in fp32 they would
// cost twice the operations and more.  So dx, dWg and dWu carry two roundings:
// 2-norm 2.35e-3 off the formula where one rounding of the result is 1.66e-3 (37 429 x
// 512 -> 2 048, 8 192 x 4 096 -> 10 240 and every size measured).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "hstu_common.h"
#include "hstu_mi355x.h"

namespace {
using namespace hstu;

enum Act { kSilu = 0, kGelu = 1, kSigmoid = 2 };
constexpr float kGelu1 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGelu3 = 0.044715f;

// a(g), and a'(g) with DERIV.  1 - s(z) is taken as e^-z s(z), which keeps the
// digits that a subtraction from 1 would lose.  Where e^-z passes 2^126, s is 0
// (its value is under 2^-126, and g may be anything); gelu's cubic is taken at 64
// at the most, where s is 0 or 1 in fp32 and the cube still a number.
template <int KIND, bool DERIV>
__device__ __forceinline__ void act(float g, float& a, float& da) {
  float z = g, dz = 1.f;
  if constexpr (KIND == kGelu) {
    const float c = __builtin_fabsf(g) > 64.f ? __builtin_copysignf(64.f, g) : g;  // NaN stays
    const float q = kGelu3 * c * c;
    z = kGelu1 * __builtin_fmaf(q, c, c);
    dz = kGelu1 * __builtin_fmaf(3.f, q, 1.f);
  }
  const float t = -kLog2e * z;
  const float e = __builtin_amdgcn_exp2f(t > 126.f ? 126.f : t);
  float s = __builtin_amdgcn_rcpf(1.f + e);
  s = t > 126.f ? 0.f : s;
  a = KIND == kSigmoid ? s : g * s;
  if constexpr (DERIV) {
    const float d = e * s * s;  // s (1 - s)
    da = KIND == kSigmoid ? d : KIND == kSilu ? __builtin_fmaf(g, d, s) : __builtin_fmaf(g * d, dz, s);
  }
}
// f with the activation as a constant: a branch in every value would keep their
// chains of exponential and reciprocal from overlapping
template <typename F>
__device__ __forceinline__ void by_act(int kind, F&& f) {
  if (kind == kSilu) f(std::integral_constant<int, kSilu>{});
  else if (kind == kGelu) f(std::integral_constant<int, kGelu>{});
  else f(std::integral_constant<int, kSigmoid>{});
}

struct GatedParams {
  const uint8_t* x;
  const uint8_t* wg;
  const uint8_t* wu;
  int64_t ldx, ldwg, ldwu;  // bytes
  const float* xs;          // e4m3: scales of x (one, or one a row), of Wg and Wu (one, or one a row of theirs)
  const float* gs;
  const float* us;
  int xs_row, gs_row, us_row;
  const uint16_t* dh;  // backward
  int64_t lddh;        // elements
  uint16_t* out;       // h [M, F], or [dg | du] [M, 2F]
  float* keep;         // [g | u] [M, 2F] contiguous, or null
  int64_t ldo;         // elements
  int M, F, K;         // K = D in bytes
  int act;
  int tiles_m;
};

__device__ __forceinline__ float bf16f(uint32_t b16) { return __builtin_bit_cast(float, b16 << 16); }

template <int N>
using Bf16s = typename std::conditional<N == 8, u32x4, u32x2>::type;
// N (4 or 8) consecutive values of dh from column n of row m on
template <int N>
__device__ __forceinline__ Bf16s<N> load_dh(const GatedParams& p, int m, int n) {
  return *(const Bf16s<N>*)(p.dh + (int64_t)m * p.lddh + n);
}
// N consecutive outputs from column n of row m on, from their products (and d, their dh).
template <int KIND, bool BWD, int N>
__device__ __forceinline__ void gated_store(const GatedParams& p, int m, int n, const float (&g)[N],
                                            const float (&u)[N], Bf16s<N> d) {
  using Vec = Bf16s<N>;
  Vec o0, o1;
  if constexpr (!BWD) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      float a0, a1, unused;
      act<KIND, false>(g[2 * j], a0, unused);
      act<KIND, false>(g[2 * j + 1], a1, unused);
      o0[j] = pack_bf16(a0 * u[2 * j], a1 * u[2 * j + 1]);
    }
    *(Vec*)(p.out + (int64_t)m * p.ldo + n) = o0;
    if (p.keep) {
      float* k = p.keep + (int64_t)m * 2 * p.F + n;
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        *(f32x4*)(k + i) = f32x4{g[i], g[i + 1], g[i + 2], g[i + 3]};
        *(f32x4*)(k + p.F + i) = f32x4{u[i], u[i + 1], u[i + 2], u[i + 3]};
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const float d0 = bf16f(d[j] & 0xffffu), d1 = __builtin_bit_cast(float, d[j] & 0xffff0000u);
      float a0, a1, b0, b1;
      act<KIND, true>(g[2 * j], a0, b0);
      act<KIND, true>(g[2 * j + 1], a1, b1);
      o0[j] = pack_bf16(d0 * u[2 * j] * b0, d1 * u[2 * j + 1] * b1);
      o1[j] = pack_bf16(d0 * a0, d1 * a1);
    }
    uint16_t* o = p.out + (int64_t)m * p.ldo + n;
    *(Vec*)o = o0;
    *(Vec*)(o + p.F) = o1;
  }
}

// ---------------------------------------------------------------- row form
// Few rows: the weights' bytes are the time.  A workgroup owns 16 columns of all
// (at most 16 MB) rows; its WAVES waves take one contiguous piece of the contraction each, with the
// operands going from memory to registers as the MFMA takes them (lane (li, q): bytes
// 32 q .. 32 q + 31 of each 128 of row li, so both of its loads hit one line), and
// meet in LDS: wave b sums row block b over the waves in order.
// Measured (us, M x D x F): 8 x 2 048 x 4 096, 34 MB of weights, 8.0 (4.2 TB/s), e4m3 5.5; 1 x
// 4 096 x 10 240, 168 MB, 30-34 (5.0-5.6 TB/s, the rate of a large copy), e4m3 15.7; 16 x 512 x
// 2 048 4.2, e4m3 3.4.  The second with 64-byte pieces 37.4, with eight waves 37.6.
template <bool F8, int MB, int WAVES, bool BWD>
__global__ void __launch_bounds__(64 * WAVES) gated_rows_kernel(GatedParams p) {
  constexpr int STEP = 128, LB = STEP / 4;  // bytes of a row, and of a lane
  __shared__ f32x4 part[WAVES][2 * MB][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint8_t* gp = p.wg + (int64_t)(n0 + li) * p.ldwg + LB * q;
  const uint8_t* up = p.wu + (int64_t)(n0 + li) * p.ldwu + LB * q;
  const uint8_t* xp[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xp[b] = p.x + (int64_t)min(16 * b + li, p.M - 1) * p.ldx + LB * q;
  f32x4 ag[MB], au[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) ag[b] = au[b] = zero4();
  const int steps = p.K / STEP, each = (steps + WAVES - 1) / WAVES;
  const int k_end = min((wave + 1) * each, steps) * STEP;
#pragma unroll 2
  for (int k = wave * each * STEP; k < k_end; k += STEP) {
    if constexpr (F8) {
      const i32x8 g = cat8(*(const u32x4*)(gp + k), *(const u32x4*)(gp + k + 16));
      const i32x8 u = cat8(*(const u32x4*)(up + k), *(const u32x4*)(up + k + 16));
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const i32x8 x = cat8(*(const u32x4*)(xp[b] + k), *(const u32x4*)(xp[b] + k + 16));
        ag[b] = mfma_fp8(g, x, ag[b]);
        au[b] = mfma_fp8(u, x, au[b]);
      }
    } else {
      const u32x4 g0 = *(const u32x4*)(gp + k), g1 = *(const u32x4*)(gp + k + 16);
      const u32x4 u0 = *(const u32x4*)(up + k), u1 = *(const u32x4*)(up + k + 16);
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const u32x4 x0 = *(const u32x4*)(xp[b] + k), x1 = *(const u32x4*)(xp[b] + k + 16);
        ag[b] = mfma_bf16(g1, x1, mfma_bf16(g0, x0, ag[b]));
        au[b] = mfma_bf16(u1, x1, mfma_bf16(u0, x0, au[b]));
      }
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) part[wave][2 * b][lane] = ag[b], part[wave][2 * b + 1][lane] = au[b];
  __syncthreads();
  if (wave >= MB) return;
  const int b = wave, m = 16 * b + li, n = n0 + 4 * q;
  if (m >= p.M) return;
  f32x4 tg = part[0][2 * b][lane], tu = part[0][2 * b + 1][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) tg += part[w][2 * b][lane], tu += part[w][2 * b + 1][lane];
  float g[4], u[4];
  const float xs = F8 ? p.xs[p.xs_row ? m : 0] : 1.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    g[e] = tg[e];
    u[e] = tu[e];
    if constexpr (F8) {
      g[e] *= xs * p.gs[p.gs_row ? n + e : 0];
      u[e] *= xs * p.us[p.us_row ? n + e : 0];
    }
  }
  by_act(p.act, [&](auto k) { gated_store<decltype(k)::value, BWD, 4>(p, m, n, g, u, BWD ? load_dh<4>(p, m, n) : u32x2{}); });
}

// ---------------------------------------------------------------- middle form
// Some hundred rows: 128 x 128 tiles leave most CUs idle and one tile's serial
// k-steps are the time.  This form takes 64 rows x 32 columns of h (64 x 64 of
// products, 4 waves of 32 rows x 16 columns, two workgroups per CU) through a ring of
// four 16 KiB stages, three k-steps' loads in flight, one barrier a step.  W rows of a
// wave in LDS: 16 gate rows, then the 16 up rows of the same columns, permuted so
// that a lane holds both products of eight (bf16) or four (e4m3) columns.
// Bound by what its tiles read from L2, 16 KiB a k-step each (256 rows x 2 048 -> 5 632: 704
// tiles, 369 MB), in 1.4 rounds of the chip's places.  Measured (us, rows at D = 2 048, F =
// 5 632, bf16 / e4m3): 7 11.5 / 7.2, 64 11.9 / 8.0, 128 14.8 / 10.0, 256 24.2 / 15.1; the
// weights' bytes are 9.0 / 4.5.
constexpr int kFewStages = 4, kFewStage = 2 * 64 * 128;

template <bool F8, bool BWD>
__global__ void __launch_bounds__(kThreads, 2) gated_few_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kFewStages][kFewStage];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  // an XCD runs a contiguous range of column panels: its L2 holds its share of the weights and all of x
  const int tiles_m = (p.M + 63) / 64, total = tiles_m * (p.F / 32), per_xcd = (total + 7) / 8;
  const int t = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (t >= min((((int)blockIdx.x & 7) + 1) * per_xcd, total)) return;
  const int nt = t / tiles_m, mt = t - nt * tiles_m;
  const int m0 = mt * 64, n0 = nt * 32, mrows = min(64, p.M - m0);
  const int wm = 32 * (wave >> 1), wn = wave & 1;
  const int nk = p.K >> 7;
  const int li = lane & 15, q = lane >> 4, lr = lane & 31, h = lane >> 5;

  // wave w fills rows 16 w .. 16 w + 15 of both operands' stages: W rows of one matrix
  uint32_t av[2], wv[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = 64 * (2 * wave + j) + lane, r = s >> 3, i = r & 15;
    const uint32_t pos = (uint32_t)(((s & 7) ^ wide_swz(r)) * 16);
    const int col = 16 * (wave >> 1) + (F8 ? i : 8 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3));
    av[j] = (uint32_t)r * (uint32_t)p.ldx + pos;
    wv[j] = (uint32_t)col * (uint32_t)(wave & 1 ? p.ldwu : p.ldwg) + pos;
  }
  const i32x4 ars = rsrc_sgprs(p.x + (int64_t)m0 * p.ldx, (uint32_t)((mrows - 1) * p.ldx + p.K));
  const int64_t ldw = wave & 1 ? p.ldwu : p.ldwg;
  const i32x4 wrs = rsrc_sgprs((wave & 1 ? p.wu : p.wg) + (int64_t)n0 * ldw, (uint32_t)(31 * ldw + p.K));
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&ring[0][0];
  auto issue = [&](int s) {  // four loads of this wave
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring0 + (uint32_t)((s % kFewStages) * kFewStage + 2048 * wave));
#pragma unroll
    for (int j = 0; j < 2; ++j) dma_to_lds(dst + 1024 * j, av[j], ars, (uint32_t)(128 * s));
#pragma unroll
    for (int j = 0; j < 2; ++j) dma_to_lds(dst + kFewStage / 2 + 1024 * j, wv[j], wrs, (uint32_t)(128 * s));
  };
  for (int s = 0; s < min(kFewStages - 1, nk); ++s) issue(s);

  f32x4 acc4[2][2];  // e4m3: [row block][gate, up]
  f32x16 acc16;      // bf16: gate, then up
#pragma unroll
  for (int i = 0; i < 4; ++i) acc4[i >> 1][i & 1] = zero4();
#pragma unroll
  for (int r = 0; r < 16; ++r) acc16[r] = 0.f;
  auto kstep = [&](int s, auto vm_c) {
    // step s has landed when only the later steps' loads are outstanding; the barrier
    // also frees step s - 1's stage for step s + 3
    dma_barrier<decltype(vm_c)::value>();
    if (s + kFewStages - 1 < nk) issue(s + kFewStages - 1);
    const uint8_t* sa = ring[s % kFewStages] + wm * 128;
    const uint8_t* sw = ring[s % kFewStages] + kFewStage / 2 + wn * 32 * 128;
    if constexpr (!F8) {
      u32x4 a[4], w[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        a[kk] = lds_ld128(sa + lr * 128 + (((2 * kk + h) ^ wide_swz(wm + lr)) * 16));
        w[kk] = lds_ld128(sw + lr * 128 + (((2 * kk + h) ^ wide_swz(32 * wn + lr)) * 16));
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) acc16 = mfma32_bf16(w[kk], a[kk], acc16);
    } else {
      i32x8 a[2], w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 16 * i + li;
        a[i] = cat8(lds_ld128(sa + r * 128 + ((q ^ wide_swz(wm + r)) * 16)),
                    lds_ld128(sa + r * 128 + (((q + 4) ^ wide_swz(wm + r)) * 16)));
        w[i] = cat8(lds_ld128(sw + r * 128 + ((q ^ wide_swz(32 * wn + r)) * 16)),
                    lds_ld128(sw + r * 128 + (((q + 4) ^ wide_swz(32 * wn + r)) * 16)));
      }
#pragma unroll
      for (int ms = 0; ms < 2; ++ms)
#pragma unroll
        for (int ns = 0; ns < 2; ++ns) acc4[ms][ns] = mfma_fp8(w[ns], a[ms], acc4[ms][ns]);
    }
  };
  for (int s = 0; s < nk - 2; ++s) kstep(s, std::integral_constant<int, 8>{});
  if (nk >= 2) kstep(nk - 2, std::integral_constant<int, 4>{});
  kstep(nk - 1, std::integral_constant<int, 0>{});

  if constexpr (!F8) {
    const int r = wm + lr;
    if (r >= mrows) return;
    float g[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = acc16[e], u[e] = acc16[8 + e];
    const int n = n0 + 16 * wn + 8 * h;
    by_act(p.act, [&](auto k) { gated_store<decltype(k)::value, BWD, 8>(p, m0 + r, n, g, u, BWD ? load_dh<8>(p, m0 + r, n) : u32x4{}); });
  } else {
    const int n = n0 + 16 * wn + 4 * q;
#pragma unroll
    for (int ms = 0; ms < 2; ++ms) {
      const int r = wm + 16 * ms + li;
      if (r >= mrows) continue;
      const float xs = p.xs[p.xs_row ? m0 + r : 0];
      float g[4], u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = acc4[ms][0][e] * (xs * p.gs[p.gs_row ? n + e : 0]);
        u[e] = acc4[ms][1][e] * (xs * p.us[p.us_row ? n + e : 0]);
      }
      by_act(p.act, [&](auto k) { gated_store<decltype(k)::value, BWD, 4>(p, m0 + r, n, g, u, BWD ? load_dh<4>(p, m0 + r, n) : u32x2{}); });
    }
  }
}

// ---------------------------------------------------------------- tile form, bf16
// Bound by the matrix cores.  128 rows x 128 columns of h a workgroup, so 128 x 256 of
// products: the projection GEMM's two-workgroup form (ring of five 16 KiB slots, exact waits on
// inline LDS DMAs) with W0 the tile's gate rows and W1 its up rows.  Wave w owns all
// 128 rows and columns 32 w .. 32 w + 31 of both products, so a lane's
// accumulators of one output pair up in registers and the epilogue is local.
// W rows are permuted in LDS so that a lane holds runs of eight columns.
// The MFMA is v_mfma_f32_16x16x32_bf16, which takes less power than 32x32x16 for the same
// bytes (M x D -> F, us, 32x32x16 / 16x16x32: 8 192 x 4 096 -> 10 240 1 091 / 1 037, 37 429 x
// 1 024 -> 4 096 558 / 540, 37 429 x 512 -> 2 048 161 / 165).  Now 1 025, 513 and 154-162: 1.34, 1.22
// and 1.0 PFLOP/s, where a large library product reaches 1.42.  With g and u kept 8 192 x
// 4 096 -> 10 240 takes 1 130-1 260; the backward's computation of 37 429 x 512 -> 2 048 197-215.
// Tiles of 256 rows in one workgroup, with a third less to load, were 4 % faster at D =
// 4 096 and 7 % slower at D = 1 024.
// The epilogue has no branch on the activation inside, and the backward's has all of a
// lane's dh in flight first (each row block waited for its own: 37 429 x 512 -> 2 048 253
// -> 205-215 us, the forward 170 -> 162; e4m3 111 -> 99).
template <bool BWD>
__global__ void __launch_bounds__(kDuoThreads, 2) gated_tile_kernel(GatedParams p, int per_xcd) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kDuoSlots][kDuoItem];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  int mt, nt;
  if (!tile_of(p.tiles_m, p.F / 128, per_xcd, mt, nt)) return;
  const int m0 = mt * 128, n0 = nt * 128, mrows = min(128, p.M - m0);
  const int nk = p.K >> 7;

  uint32_t av[4], wv[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int q = 64 * (4 * wave + j) + lane, r = q >> 3, i = r & 31;
    av[j] = (uint32_t)r * (uint32_t)p.ldx + (uint32_t)(((q & 7) ^ wide_swz(r)) * 16);
    // W blocks of 32 rows all in one swizzle (a wave reads one block of each product)
    const uint32_t pos = (uint32_t)(((q & 7) ^ wide_swz(i)) * 16);
    const int col = (r & ~31) + 8 * ((i & 15) >> 2) + 4 * (i >> 4) + (i & 3);  // a lane: 8 consecutive columns
    wv[0][j] = (uint32_t)col * (uint32_t)p.ldwg + pos;
    wv[1][j] = (uint32_t)col * (uint32_t)p.ldwu + pos;
  }
  // rows past M read as zero
  const i32x4 ars = rsrc_sgprs(p.x + (int64_t)m0 * p.ldx, (uint32_t)((mrows - 1) * p.ldx + p.K));
  const i32x4 grs = rsrc_sgprs(p.wg + (int64_t)n0 * p.ldwg, (uint32_t)(127 * p.ldwg + p.K));
  const i32x4 urs = rsrc_sgprs(p.wu + (int64_t)n0 * p.ldwu, (uint32_t)(127 * p.ldwu + p.K));
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&ring[0][0];
  auto issue = [&](int it) {  // item it: k-step it / 3; 0 x, 1 gate, 2 up
    const int s = it / 3, kind = it - 3 * s;
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring0 + (uint32_t)((it % kDuoSlots) * kDuoItem + 4096 * wave));
    if (kind == 0) duo_dma4(dst, av, ars, (uint32_t)(s * 128));
    else if (kind == 1) duo_dma4(dst, wv[0], grs, (uint32_t)(s * 128));
    else duo_dma4(dst, wv[1], urs, (uint32_t)(s * 128));
  };
  for (int it = 0; it < 5; ++it) issue(it);  // D % 256: at least four k-steps

  const int li = lane & 15, q = lane >> 4;
  // chunks q and q + 4 of row li; in odd 32-row blocks of x the two trade places
  uint32_t rd[2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) rd[kk] = li * 128 + (((4 * kk + q) ^ wide_swz(li)) * 16);
  const uint32_t w_off = 4096 * wave;

  f32x4 acc[8][4];
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[m][nb] = zero4();
  auto kstep = [&](int s, auto items_c) {
    constexpr int ITEMS = decltype(items_c)::value;
    if constexpr (ITEMS == 0) dma_barrier<0>();
    else dma_barrier<8>();
    const uint8_t* sa = ring[(3 * s) % kDuoSlots];
    u32x4 w[4][2], a[8][2];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      const uint8_t* sw = ring[(3 * s + 1 + (nb >> 1)) % kDuoSlots] + w_off + 2048 * (nb & 1);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) w[nb][kk] = lds_ld128(sw + rd[kk]);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) a[m][kk] = lds_ld128(sa + 2048 * m + rd[m & 2 ? kk ^ 1 : kk]);
    pc_barrier_lds();  // every wave has read step s: its three slots are free
    const uint32_t ka = (uint32_t)(128 * (s + 2)), kw1 = (uint32_t)(128 * (s + 1));
    uint32_t dst[3];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
      dst[k] = __builtin_amdgcn_readfirstlane(ring0 + (uint32_t)(((3 * s + 5 + k) % kDuoSlots) * kDuoItem + 4096 * wave));
    static_for<64>([&](auto nc) {
      constexpr int n = decltype(nc)::value, kk = n >> 5, m = (n >> 2) & 7, nb = n & 3;
      acc[m][nb] = mfma_bf16(w[nb][kk], a[m][kk], acc[m][nb]);
      if constexpr (n % 4 == 3 && n / 4 < 4 * ITEMS) {  // items 3 s + 5 (up), 3 s + 6 (x), 3 s + 7 (gate)
        constexpr int i = n / 4, k = i >> 2, j = i & 3;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (k == 0) dma_to_lds(dst[0] + 1024 * j, wv[1][j], urs, kw1);
        else if constexpr (k == 1) dma_to_lds(dst[1] + 1024 * j, av[j], ars, ka);
        else dma_to_lds(dst[2] + 1024 * j, wv[0][j], grs, ka);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  for (int s = 0; s < nk - 2; ++s) kstep(s, std::integral_constant<int, 3>{});
  kstep(nk - 2, std::integral_constant<int, 1>{});
  kstep(nk - 1, std::integral_constant<int, 0>{});

  // lane: rows m0 + 16 mb + li, columns n0 + 32 wave + 8 q + (0..7) of both products
  const int cl = n0 + 32 * wave + 8 * q;
  u32x4 dh[8];
#pragma unroll
  for (int mb = 0; mb < 8; ++mb) {  // all in flight before the first is used
    dh[mb] = u32x4{};
    if constexpr (BWD) dh[mb] = load_dh<8>(p, m0 + min(16 * mb + li, mrows - 1), cl);
  }
  __builtin_amdgcn_sched_barrier(0);
  by_act(p.act, [&](auto k) {
#pragma unroll
    for (int mb = 0; mb < 8; ++mb) {
      const int r = 16 * mb + li;
      if (r >= mrows) continue;
      float g[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = acc[mb][e >> 2][e & 3], u[e] = acc[mb][2 + (e >> 2)][e & 3];
      gated_store<decltype(k)::value, BWD, 8>(p, m0 + r, cl, g, u, dh[mb]);
    }
  });
}

// ---------------------------------------------------------------- tile form, e4m3
// The same tile, ring and items on rows of e4m3 (a k-step is 128 elements) with
// v_mfma_f32_16x16x128_f8f6f4: 16-row blocks 0, 1 of a wave's weights are gate
// rows, 2, 3 up rows.  Measured: 37 429 x 1 024 -> 4 096 302-314 us, 2.0 PFLOP/s, in eight
// k-steps a tile (a large library product 2.63).
// The instruction (in every form) takes eight consecutive products together and cuts each
// toward zero at 2^-13 of 2^(the largest's two exponents); these sums meet in fp32.  With
// random operands that moves 2 % of the outputs to the next bf16 value, and the 2-norm
// off the formula from 1.6589e-3 to 1.6590e-3.
__global__ void __launch_bounds__(kDuoThreads, 2) gated_tile_fp8_kernel(GatedParams p, int per_xcd) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kDuoSlots][kDuoItem];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  int mt, nt;
  if (!tile_of(p.tiles_m, p.F / 128, per_xcd, mt, nt)) return;
  const int m0 = mt * 128, n0 = nt * 128, mrows = min(128, p.M - m0);
  const int nk = p.K >> 7;  // at least two

  uint32_t av[4], wv[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int q = 64 * (4 * wave + j) + lane, r = q >> 3, i = r & 31;
    av[j] = (uint32_t)r * (uint32_t)p.ldx + (uint32_t)(((q & 7) ^ wide_swz(r)) * 16);
    const uint32_t pos = (uint32_t)(((q & 7) ^ wide_swz(i)) * 16);
    const int col = (r & ~31) + 8 * ((i & 15) >> 2) + 4 * (i >> 4) + (i & 3);  // a lane: 8 consecutive columns
    wv[0][j] = (uint32_t)col * (uint32_t)p.ldwg + pos;
    wv[1][j] = (uint32_t)col * (uint32_t)p.ldwu + pos;
  }
  const i32x4 ars = rsrc_sgprs(p.x + (int64_t)m0 * p.ldx, (uint32_t)((mrows - 1) * p.ldx + p.K));
  const i32x4 grs = rsrc_sgprs(p.wg + (int64_t)n0 * p.ldwg, (uint32_t)(127 * p.ldwg + p.K));
  const i32x4 urs = rsrc_sgprs(p.wu + (int64_t)n0 * p.ldwu, (uint32_t)(127 * p.ldwu + p.K));
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&ring[0][0];
  auto issue = [&](int it) {  // item it: k-step it / 3; 0 x, 1 gate, 2 up
    const int s = it / 3, kind = it - 3 * s;
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring0 + (uint32_t)((it % kDuoSlots) * kDuoItem + 4096 * wave));
    if (kind == 0) duo_dma4(dst, av, ars, (uint32_t)(s * 128));
    else if (kind == 1) duo_dma4(dst, wv[0], grs, (uint32_t)(s * 128));
    else duo_dma4(dst, wv[1], urs, (uint32_t)(s * 128));
  };
  for (int it = 0; it < 5; ++it) issue(it);

  const int li = lane & 15, q = lane >> 4;
  // chunks q and q + 4 of row li; in odd 32-row blocks of x the two trade places
  const uint32_t rd0 = li * 128 + ((q ^ wide_swz(li)) * 16), rd1 = li * 128 + (((q + 4) ^ wide_swz(li)) * 16);
  const uint32_t w_off = 4096 * wave;
  const int cl = n0 + 32 * wave + 8 * q;  // the lane's columns: cl + 4 (ns % 2) + (0..3)
  f32x4 gsv[2], usv[2];
  float sav[8];
  auto load_consts = [&]() {
    const BufRsrc gsr = make_rsrc(p.gs, p.gs_row ? (uint32_t)p.F * 4u : 4u);
    const BufRsrc usr = make_rsrc(p.us, p.us_row ? (uint32_t)p.F * 4u : 4u);
    const BufRsrc xsr = make_rsrc(p.xs + (p.xs_row ? m0 : 0), p.xs_row ? (uint32_t)mrows * 4u : 4u);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (p.gs_row) gsv[i] = __builtin_bit_cast(f32x4, buf_ld128(gsr, (uint32_t)(cl + 4 * i) * 4u, 0));
      else gsv[i] = zero4() + buf_ldf(gsr, 0, 0);
      if (p.us_row) usv[i] = __builtin_bit_cast(f32x4, buf_ld128(usr, (uint32_t)(cl + 4 * i) * 4u, 0));
      else usv[i] = zero4() + buf_ldf(usr, 0, 0);
    }
#pragma unroll
    for (int ms = 0; ms < 8; ++ms) sav[ms] = buf_ldf(xsr, p.xs_row ? (uint32_t)(16 * ms + li) * 4u : 0u, 0);
  };

  f32x4 acc[8][4];
  auto mfma_rows = [&](const i32x8 (&w)[4], const i32x8 (&a)[4], int ms0, bool first) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ns = 0; ns < 4; ++ns) acc[ms0 + i][ns] = mfma_fp8(w[ns], a[i], first ? zero4() : acc[ms0 + i][ns]);
  };
  auto read_a = [&](const uint8_t* st, int ms0, i32x8 (&a)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ms = ms0 + i;
      a[i] = cat8(lds_ld128(st + (ms & 2 ? rd1 : rd0) + 2048 * ms), lds_ld128(st + (ms & 2 ? rd0 : rd1) + 2048 * ms));
    }
  };
  auto kstep = [&](int s, auto first_c, auto last_c) {
    constexpr bool FIRST = decltype(first_c)::value, LAST = decltype(last_c)::value;
    if constexpr (LAST) dma_barrier<0>();
    else dma_barrier<8>();
    const uint8_t* sa = ring[(3 * s) % kDuoSlots];
    i32x8 w[4], a0[4], a1[4];
#pragma unroll
    for (int ns = 0; ns < 4; ++ns) {
      const uint8_t* sw = ring[(3 * s + 1 + (ns >> 1)) % kDuoSlots] + w_off + 2048 * (ns & 1);
      w[ns] = cat8(lds_ld128(sw + rd0), lds_ld128(sw + rd1));
    }
    read_a(sa, 0, a0);
    mfma_rows(w, a0, 0, FIRST);
    read_a(sa, 4, a1);
    pc_barrier_lds();  // every wave has read step s: its three slots are free
    if constexpr (LAST) {
      load_consts();
    } else {
#pragma unroll
      for (int k = 5; k < 8; ++k)
        if (3 * s + k < 3 * nk) issue(3 * s + k);
    }
    mfma_rows(w, a1, 4, FIRST);
  };
  kstep(0, std::true_type{}, std::false_type{});
  for (int s = 1; s < nk - 1; ++s) kstep(s, std::false_type{}, std::false_type{});
  kstep(nk - 1, std::false_type{}, std::true_type{});

  by_act(p.act, [&](auto k) {
#pragma unroll
    for (int ms = 0; ms < 8; ++ms) {
      const int r = 16 * ms + li;
      if (r >= mrows) continue;
      float g[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = acc[ms][e >> 2][e & 3] * (sav[ms] * gsv[e >> 2][e & 3]);
        u[e] = acc[ms][2 + (e >> 2)][e & 3] * (sav[ms] * usv[e >> 2][e & 3]);
      }
      gated_store<decltype(k)::value, false, 8>(p, m0 + r, cl, g, u, u32x4{});
    }
  });
}

// ---------------------------------------------------------------- backward from kept g and u
// Memory alone bounds it: 10 bytes in and 4 out a value.  A thread takes eight
// consecutive columns.  8 192 x 10 240 (1.17 GB) 247-253 us, 4.7 TB/s.
struct KeptArgs {
  const uint16_t* dh;
  const float* keep;
  uint16_t* out;
  int64_t lddh, ldo;  // elements
  int64_t rows;
  int F, act;
};
__global__ void __launch_bounds__(256) gated_kept_kernel(KeptArgs a) {
  const int chunks = a.F / 8;
  const int64_t total = a.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / chunks;
    const int n = (int)(i - m * chunks) * 8;
    const float* k = a.keep + m * 2 * a.F + n;
    const u32x4 d = *(const u32x4*)(a.dh + m * a.lddh + n);
    const f32x4 gv[2] = {*(const f32x4*)k, *(const f32x4*)(k + 4)};
    const f32x4 uv[2] = {*(const f32x4*)(k + a.F), *(const f32x4*)(k + a.F + 4)};
    u32x4 o0, o1;
    by_act(a.act, [&](auto kind) {
      constexpr int K = decltype(kind)::value;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = d[j];
        const float d0 = bf16f(w & 0xffffu), d1 = __builtin_bit_cast(float, w & 0xffff0000u);
        float a0, a1, b0, b1;
        act<K, true>(gv[j >> 1][2 * (j & 1)], a0, b0);
        act<K, true>(gv[j >> 1][2 * (j & 1) + 1], a1, b1);
        o0[j] = pack_bf16(d0 * uv[j >> 1][2 * (j & 1)] * b0, d1 * uv[j >> 1][2 * (j & 1) + 1] * b1);
        o1[j] = pack_bf16(d0 * a0, d1 * a1);
      }
    });
    uint16_t* o = a.out + m * a.ldo + n;
    *(u32x4*)o = o0;
    *(u32x4*)(o + a.F) = o1;
  }
}

// The weights side by side with the contraction index of dx = [dg | du] [Wg; Wu]
// contiguous: out[d][f] = Wg[f][d], out[d][F + f] = Wu[f][d].  64 x 64 tiles through
// LDS (pitch 66 elements: both the row and the column accesses spread over the
// banks), 16-byte loads and stores; bound by memory: two of 10 240 x 4 096 (336 MB)
// 57-60 us, 5.7 TB/s.
__global__ void __launch_bounds__(256) gated_transpose_kernel(const uint16_t* wg, const uint16_t* wu, int64_t ldg,
                                                              int64_t ldu, int F, uint16_t* out, int64_t ldo) {
  __shared__ uint16_t tile[64 * 66];
  const int half = blockIdx.z, f0 = blockIdx.x * 64, d0 = blockIdx.y * 64;
  const uint16_t* w = half ? wu : wg;
  const int64_t ld = half ? ldu : ldg;
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const u32x4 v = *(const u32x4*)(w + (int64_t)(f0 + r + 32 * k) * ld + d0 + c);
    uint32_t* t = (uint32_t*)(tile + (r + 32 * k) * 66 + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = tile[(c + 2 * j) * 66 + r + 32 * k], hi = tile[(c + 2 * j + 1) * 66 + r + 32 * k];
      v[j] = lo | hi << 16;
    }
    *(u32x4*)(out + (int64_t)(d0 + r + 32 * k) * ldo + (int64_t)half * F + f0 + c) = u32x4{v[0], v[1], v[2], v[3]};
  }
}

// Which form.  Rows: 16 columns a workgroup, so F / 16 of them; few rows with at most
// one a CU, or with many.  Between, 256 < F / 16 <= 512, half of the CUs have two
// while the middle form's F / 32 tiles have a CU each (us, rows / middle, 8 rows:
// D = 2 048, F = 4 096 7.3 / 10.5, 5 632 11.8 / 10.7, 8 192 13.3 / 12.2, 10 240 19.3 / 22.4;
// D = 512, F = 2 048 4.0 / 4.9).  Its two row blocks serve narrow weights (D = 2 048, F =
// 4 096, 24 rows 9.0 / 10.3, D = 512, F = 2 048, 64 rows 5.4 / 4.7).
// Middle: up to 1.5 rounds of the chip's 512 places (us, middle / 128 x 128 tiles:
// 704 tiles 23.3 / 29.7, 1 056 34.6 / 30.0, 1 280 86.7 / 72.8; e4m3 14.0 / 20.2, 21.3 /
// 20.5), and e4m3 rows of one k-step.
bool rows_form(int M, int F) { return F <= 4096 ? M <= 32 : F > 8192 && M <= 16; }
constexpr int kFewMaxTiles = 768;

template <bool F8, bool BWD>
int launch_gated(GatedParams p, hipStream_t stream) {
  if (rows_form(p.M, p.F)) {
    constexpr int W = 4;
    const dim3 grid(p.F / 16), block(64 * W);
    if (p.M <= 16) hipLaunchKernelGGL((gated_rows_kernel<F8, 1, W, BWD>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gated_rows_kernel<F8, 2, W, BWD>), grid, block, 0, stream, p);
    return (int)hipGetLastError();
  }
  const int64_t few = ((int64_t)p.M + 63) / 64 * (p.F / 32), big = ((int64_t)p.M + 127) / 128 * (p.F / 128);
  if (few <= kFewMaxTiles || p.K < 256) {
    if (few >= (1 << 30)) return HSTU_E_UNSUPPORTED;
    hipLaunchKernelGGL((gated_few_kernel<F8, BWD>), dim3((unsigned)((few + 7) / 8 * 8)), dim3(kThreads), 0, stream, p);
    return (int)hipGetLastError();
  }
  if (big >= (1 << 30)) return HSTU_E_UNSUPPORTED;
  p.tiles_m = (p.M + 127) / 128;
  const int per_xcd = (int)((big + 7) / 8);
  if constexpr (F8) hipLaunchKernelGGL(gated_tile_fp8_kernel, dim3(8 * per_xcd), dim3(kDuoThreads), 0, stream, p, per_xcd);
  else hipLaunchKernelGGL((gated_tile_kernel<BWD>), dim3(8 * per_xcd), dim3(kDuoThreads), 0, stream, p, per_xcd);
  return (int)hipGetLastError();
}

// arguments that the three entry points share
int check(const GatedParams& p, int es, int D, int kmul) {
  if (p.M < 0 || p.F <= 0 || D <= 0 || p.act < kSilu || p.act > kSigmoid) return HSTU_E_BAD_ARG;
  if (p.ldx < (int64_t)D * es || p.ldwg < (int64_t)D * es || p.ldwu < (int64_t)D * es) return HSTU_E_BAD_ARG;
  if (p.M > 0 && (!p.x || !p.wg || !p.wu || !p.out)) return HSTU_E_BAD_ARG;
  if (p.F % 128 || D % kmul) return HSTU_E_UNSUPPORTED;
  // 32-bit offsets of a tile's rows
  if ((p.ldx | p.ldwg | p.ldwu) >> 24 || (int64_t)D * es >= (1 << 24)) return HSTU_E_UNSUPPORTED;
  if (((uintptr_t)p.x | (uintptr_t)p.wg | (uintptr_t)p.wu | (uintptr_t)p.out) % 16 ||
      (p.ldx | p.ldwg | p.ldwu) % 16 || p.ldo % 8)
    return HSTU_E_UNSUPPORTED;
  return 0;
}

}  // namespace

extern "C" int hstu_gated_fwd(const void* x, int64_t ldx, const void* w_gate, int64_t ldg, const void* w_up,
                              int64_t ldu, int M, int F, int D, int activation, void* h, int64_t ldh,
                              float* keep, hipStream_t stream) {
  GatedParams p{};
  p.keep = keep;
  if ((uintptr_t)keep % 16) return HSTU_E_UNSUPPORTED;
  p.x = (const uint8_t*)x;
  p.wg = (const uint8_t*)w_gate;
  p.wu = (const uint8_t*)w_up;
  p.ldx = 2 * ldx;
  p.ldwg = 2 * ldg;
  p.ldwu = 2 * ldu;
  p.out = (uint16_t*)h;
  p.ldo = ldh;
  p.M = M;
  p.F = F;
  p.K = 2 * D;
  p.act = activation;
  if (ldh < F) return HSTU_E_BAD_ARG;
  const int st = check(p, 2, D, 256);
  if (st != 0 || M == 0) return st;
  return launch_gated<false, false>(p, stream);
}

extern "C" int hstu_gated_bwd(const void* dh, int64_t lddh, const void* x, int64_t ldx, const void* w_gate,
                              int64_t ldg, const void* w_up, int64_t ldu, int M, int F, int D, int activation,
                              void* dgu, int64_t lddgu, hipStream_t stream) {
  GatedParams p{};
  p.x = (const uint8_t*)x;
  p.wg = (const uint8_t*)w_gate;
  p.wu = (const uint8_t*)w_up;
  p.ldx = 2 * ldx;
  p.ldwg = 2 * ldg;
  p.ldwu = 2 * ldu;
  p.dh = (const uint16_t*)dh;
  p.lddh = lddh;
  p.out = (uint16_t*)dgu;
  p.ldo = lddgu;
  p.M = M;
  p.F = F;
  p.K = 2 * D;
  p.act = activation;
  if (lddh < F || lddgu < 2 * (int64_t)F || (M > 0 && !dh)) return HSTU_E_BAD_ARG;
  const int st = check(p, 2, D, 256);
  if (st != 0 || M == 0) return st;
  if ((uintptr_t)dh % 16 || lddh % 8) return HSTU_E_UNSUPPORTED;
  return launch_gated<false, true>(p, stream);
}

extern "C" int hstu_gated_fwd_fp8(const void* x, int64_t ldx, const float* x_scale, int x_scale_mode,
                                  const void* w_gate, int64_t ldg, const float* gate_scale, int gate_scale_mode,
                                  const void* w_up, int64_t ldu, const float* up_scale, int up_scale_mode, int M, int F,
                                  int D, int activation, void* h, int64_t ldh, hipStream_t stream) {
  GatedParams p{};
  p.x = (const uint8_t*)x;
  p.wg = (const uint8_t*)w_gate;
  p.wu = (const uint8_t*)w_up;
  p.ldx = ldx;
  p.ldwg = ldg;
  p.ldwu = ldu;
  p.xs = x_scale;
  p.gs = gate_scale;
  p.us = up_scale;
  p.xs_row = x_scale_mode != 0;
  p.gs_row = gate_scale_mode != 0;
  p.us_row = up_scale_mode != 0;
  p.out = (uint16_t*)h;
  p.ldo = ldh;
  p.M = M;
  p.F = F;
  p.K = D;
  p.act = activation;
  if (ldh < F || (M > 0 && (!x_scale || !gate_scale || !up_scale))) return HSTU_E_BAD_ARG;
  const int st = check(p, 1, D, 128);
  if (st != 0 || M == 0) return st;
  if (((uintptr_t)x_scale | (uintptr_t)gate_scale | (uintptr_t)up_scale) % 4) return HSTU_E_UNSUPPORTED;
  return launch_gated<true, false>(p, stream);
}

extern "C" int hstu_gated_bwd_kept(const void* dh, int64_t lddh, const float* keep, int64_t rows, int F, int activation,
                                   void* dgu, int64_t lddgu, hipStream_t stream) {
  if (rows < 0 || F <= 0 || lddh < F || lddgu < 2 * (int64_t)F || activation < kSilu || activation > kSigmoid)
    return HSTU_E_BAD_ARG;
  if (rows > 0 && (!dh || !keep || !dgu)) return HSTU_E_BAD_ARG;
  if (F % 8 || ((uintptr_t)dh | (uintptr_t)keep | (uintptr_t)dgu) % 16 || lddh % 8 || lddgu % 8) return HSTU_E_UNSUPPORTED;
  if (rows == 0) return 0;
  const KeptArgs a{(const uint16_t*)dh, keep, (uint16_t*)dgu, lddh, lddgu, rows, F, activation};
  const int64_t blocks = std::min<int64_t>((rows * (F / 8) + 255) / 256, 8192);
  hipLaunchKernelGGL(gated_kept_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

extern "C" int hstu_gated_transpose(const void* w_gate, int64_t ldg, const void* w_up, int64_t ldu, int F, int D, void* out,
                                    int64_t ldo, hipStream_t stream) {
  if (F <= 0 || D <= 0 || ldg < D || ldu < D || ldo < 2 * (int64_t)F || !w_gate || !w_up || !out) return HSTU_E_BAD_ARG;
  if (F % 64 || D % 64 || D / 64 > 65535 || ((uintptr_t)w_gate | (uintptr_t)w_up | (uintptr_t)out) % 16 || ldg % 8 ||
      ldu % 8 || ldo % 8)
    return HSTU_E_UNSUPPORTED;
  hipLaunchKernelGGL(gated_transpose_kernel, dim3(F / 64, D / 64, 2), dim3(256), 0, stream, (const uint16_t*)w_gate,
                     (const uint16_t*)w_up, ldg, ldu, F, (uint16_t*)out, ldo);
  return (int)hipGetLastError();
}
