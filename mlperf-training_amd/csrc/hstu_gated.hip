// Gated feed-forward projection, for MI355X (gfx950):
//
//   g = x Wg^T, u = x Wu^T (x [M, D]; Wg, Wu [F, D], the contraction index
//   contiguous),  h = a(g) u,   a one of
//     silu    g s(g)
//     gelu    g s(2 sqrt(2 / pi) (g + 0.044715 g^3))    (the tanh form)
//     sigmoid s(g),                                      s(z) = 1 / (1 + e^-z)
//   and the elementwise part of its backward from dh, g and u computed again:
//     dg = dh u a'(g),  du = dh a(g),  written as [dg | du] [M, 2F].
//
// Both products of one output meet in one lane's accumulators, so nothing of
// [M, F] but h (or [dg | du]) is written, and the values that meet are fp32:
// the one rounding is that of the output.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "hstu_common.h"
#include "hstu_mi355x.h"

namespace {
using namespace hstu;

enum Act { kSilu = 0, kGelu = 1, kSigmoid = 2 };
constexpr float kGelu1 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGelu3 = 0.044715f;

// a(g), and a'(g) with DERIV.  1 - s(z) is taken as e^-z s(z), which keeps the
// digits that a subtraction from 1 would lose; e^-z is held below 2^126, so
// that s stays a normal number.
template <bool DERIV>
__device__ __forceinline__ void act(int kind, float g, float& a, float& da) {
  float z = g, dz = 1.f;
  if (kind == kGelu) {
    const float q = kGelu3 * g * g;
    z = kGelu1 * __builtin_fmaf(q, g, g);
    dz = kGelu1 * __builtin_fmaf(3.f, q, 1.f);
  }
  float t = -kLog2e * z;
  t = t > 126.f ? 126.f : t;  // NaN stays
  const float e = __builtin_amdgcn_exp2f(t), s = __builtin_amdgcn_rcpf(1.f + e);
  a = kind == kSigmoid ? s : g * s;
  if constexpr (DERIV) {
    const float d = e * s * s;  // s (1 - s)
    da = kind == kSigmoid ? d : __builtin_fmaf(g * d, dz, s);
  }
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
  int64_t ldo;         // elements
  int M, F, K;         // K = D in bytes
  int act;
};

__device__ __forceinline__ float bf16f(uint32_t b16) { return __builtin_bit_cast(float, b16 << 16); }

// Four consecutive outputs (columns n .. n + 3 of row m) from their products.
template <bool BWD>
__device__ __forceinline__ void gated_store4(const GatedParams& p, int m, int n, const float (&g)[4],
                                             const float (&u)[4]) {
  if constexpr (!BWD) {
    float h[4], unused;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a;
      act<false>(p.act, g[e], a, unused);
      h[e] = a * u[e];
    }
    *(u32x2*)(p.out + (int64_t)m * p.ldo + n) = u32x2{pack_bf16(h[0], h[1]), pack_bf16(h[2], h[3])};
  } else {
    const u32x2 d = *(const u32x2*)(p.dh + (int64_t)m * p.lddh + n);
    float dg[4], du[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float dh = bf16f(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu);
      float a, da;
      act<true>(p.act, g[e], a, da);
      dg[e] = dh * u[e] * da;
      du[e] = dh * a;
    }
    uint16_t* o = p.out + (int64_t)m * p.ldo + n;
    *(u32x2*)o = u32x2{pack_bf16(dg[0], dg[1]), pack_bf16(dg[2], dg[3])};
    *(u32x2*)(o + p.F) = u32x2{pack_bf16(du[0], du[1]), pack_bf16(du[2], du[3])};
  }
}

// Row form: a workgroup owns 16 columns and 16 MB rows, its four waves split
// the contraction and meet in LDS in wave order.  Operands go from memory to
// registers as the MFMA takes them: lane (li, q) reads 16 (bf16) or 32 (e4m3)
// contiguous bytes of row li.
template <bool F8, int MB, bool BWD>
__global__ void __launch_bounds__(kThreads) gated_rows_kernel(GatedParams p) {
  constexpr int STEP = F8 ? 128 : 64;  // bytes of a row per MFMA
  constexpr int LB = STEP / 4;         // bytes of a lane
  __shared__ f32x4 part[3][2 * MB][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, q = lane >> 4;
  const int nt = p.F / 16, mt = blockIdx.x / nt, n0 = (blockIdx.x - mt * nt) * 16, m0 = mt * 16 * MB;
  const uint8_t* gp = p.wg + (int64_t)(n0 + li) * p.ldwg + LB * q;
  const uint8_t* up = p.wu + (int64_t)(n0 + li) * p.ldwu + LB * q;
  const uint8_t* xp[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) xp[b] = p.x + (int64_t)min(m0 + 16 * b + li, p.M - 1) * p.ldx + LB * q;
  f32x4 ag[MB], au[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) ag[b] = au[b] = zero4();
#pragma unroll 4
  for (int k = wave * STEP; k < p.K; k += 4 * STEP) {
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
      const u32x4 g = *(const u32x4*)(gp + k), u = *(const u32x4*)(up + k);
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const u32x4 x = *(const u32x4*)(xp[b] + k);
        ag[b] = mfma_bf16(g, x, ag[b]);
        au[b] = mfma_bf16(u, x, au[b]);
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int b = 0; b < MB; ++b) part[wave - 1][2 * b][lane] = ag[b], part[wave - 1][2 * b + 1][lane] = au[b];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int b = 0; b < MB; ++b) {
#pragma unroll
    for (int w = 0; w < 3; ++w) ag[b] += part[w][2 * b][lane], au[b] += part[w][2 * b + 1][lane];
    const int m = m0 + 16 * b + li, n = n0 + 4 * q;
    if (m >= p.M) continue;
    float g[4], u[4];
    const float xs = F8 ? p.xs[p.xs_row ? m : 0] : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = ag[b][e];
      u[e] = au[b][e];
      if constexpr (F8) {
        g[e] *= xs * p.gs[p.gs_row ? n + e : 0];
        u[e] *= xs * p.us[p.us_row ? n + e : 0];
      }
    }
    gated_store4<BWD>(p, m, n, g, u);
  }
}

template <bool F8, bool BWD>
int launch_gated(const GatedParams& p, hipStream_t stream) {
  const int mb = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
  const int64_t tiles = ((int64_t)p.M + 16 * mb - 1) / (16 * mb) * (p.F / 16);
  if (tiles >= ((int64_t)1 << 31)) return HSTU_E_UNSUPPORTED;
  const dim3 grid((unsigned)tiles);
  if (mb == 1) hipLaunchKernelGGL((gated_rows_kernel<F8, 1, BWD>), grid, dim3(kThreads), 0, stream, p);
  else if (mb == 2) hipLaunchKernelGGL((gated_rows_kernel<F8, 2, BWD>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((gated_rows_kernel<F8, 4, BWD>), grid, dim3(kThreads), 0, stream, p);
  return (int)hipGetLastError();
}

// arguments that the three entry points share
int check(const GatedParams& p, int es, int D, int kmul) {
  if (p.M < 0 || p.F <= 0 || D <= 0 || p.act < kSilu || p.act > kSigmoid) return HSTU_E_BAD_ARG;
  if (p.ldx < (int64_t)D * es || p.ldwg < (int64_t)D * es || p.ldwu < (int64_t)D * es) return HSTU_E_BAD_ARG;
  if (p.M > 0 && (!p.x || !p.wg || !p.wu || !p.out)) return HSTU_E_BAD_ARG;
  if (p.F % 128 || D % kmul) return HSTU_E_UNSUPPORTED;
  if (((uintptr_t)p.x | (uintptr_t)p.wg | (uintptr_t)p.wu | (uintptr_t)p.out) % 16 ||
      (p.ldx | p.ldwg | p.ldwu) % 16 || p.ldo % 8)
    return HSTU_E_UNSUPPORTED;
  return 0;
}

}  // namespace

extern "C" int hstu_gated_fwd(const void* x, int64_t ldx, const void* w_gate, int64_t ldg, const void* w_up,
                              int64_t ldu, int M, int F, int D, int activation, void* h, int64_t ldh,
                              hipStream_t stream) {
  GatedParams p{};
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
