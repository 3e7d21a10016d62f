// RMS norm with the residual's addition, forward and backward, for MI355X (gfx950).
//
//   h    = round(x + residual)                    (h = x without a residual)
//   rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * w
//   y in the input's type, or e4m3(clamp(y / s, +-448)) with the row's own
//   s = max|y| / 448 (1 / 448 for a row of zeros) or one given scale.
//   backward, c = w dy, xhat = h rstd:
//   dx = rstd (c - xhat mean(c xhat)) + dh,  dw = sum over rows of dy xhat
//
// The norm is of the rounded h, the one that is returned and that the backward
// has: its gradients are then those of the function that was computed.  Sums
// and statistics are fp32 throughout.
//
// What bounds it: memory (about one operation a byte).  So a row is read once
// and stays in registers between its statistics and its output: a group of G
// threads owns a row, NV chunks of 8 consecutive values a thread.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "hstu_common.h"
#include "hstu_mi355x.h"

namespace {
using namespace hstu;

template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ float dpp_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROW_MASK, 0xf, true));
}
// sum, and largest magnitude (as its bits, so that a NaN is the largest; lanes without
// a source read 0), over the wave
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_move<0x111>(v);
  v += dpp_move<0x112>(v);
  v += dpp_move<0x114>(v);
  v += dpp_move<0x118>(v);
  v += dpp_move<0x142, 0xa>(v);
  v += dpp_move<0x143, 0xc>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xf, true));
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
  v = dpp_max<0x111>(v);
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142, 0xa>(v);
  v = dpp_max<0x143, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Eight consecutive values of a row from element c0 on.  VEC: whole and 16-byte
// aligned; else one by one, those from D on as zeros.
template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const uint8_t* row, int c0, int D, float (&v)[8]) {
  if constexpr (VEC && F32) {
    const f32x4* p = (const f32x4*)(row + 4 * (int64_t)c0);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else if constexpr (VEC) {
    const u32x4 a = *(const u32x4*)(row + 2 * (int64_t)c0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __builtin_bit_cast(float, a[e] << 16);
      v[2 * e + 1] = __builtin_bit_cast(float, a[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
      if (c0 + e < D)
        v[e] = F32 ? ((const float*)row)[c0 + e] : __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[c0 + e] << 16);
    }
  }
}
// The same in two parts, so that a row's loads can be issued before its turn.
// Without VEC the second part loads.
template <bool F32, bool VEC>
struct Raw8 {
  u32x4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t* row, int c0) {
    if constexpr (VEC) {
      const u32x4* p = (const u32x4*)(row + (F32 ? 4 : 2) * (int64_t)c0);
      v[0] = p[0];
      if constexpr (F32) v[1] = p[1];
    }
  }
  __device__ __forceinline__ void get(const uint8_t* row, int c0, int D, float (&o)[8]) const {
    if constexpr (!VEC) {
      load8<F32, false>(row, c0, D, o);
    } else if constexpr (F32) {
      const f32x4 a = __builtin_bit_cast(f32x4, v[0]), b = __builtin_bit_cast(f32x4, v[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = a[e], o[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = v[0][e];
        o[2 * e] = __builtin_bit_cast(float, x << 16);
        o[2 * e + 1] = __builtin_bit_cast(float, x & 0xffff0000u);
      }
    }
  }
};
template <bool F32, bool VEC>
__device__ __forceinline__ void store8(uint8_t* row, int c0, int D, const float (&v)[8]) {
  if constexpr (VEC && F32) {
    f32x4* p = (f32x4*)(row + 4 * (int64_t)c0);
    p[0] = f32x4{v[0], v[1], v[2], v[3]};
    p[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else if constexpr (VEC) {
    *(u32x4*)(row + 2 * (int64_t)c0) =
        u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < D) {
        if constexpr (F32) ((float*)row)[c0 + e] = v[e];
        else ((uint16_t*)row)[c0 + e] = to_bf16(v[e]);
      }
  }
}
__device__ __forceinline__ float sat_e4m3(float q) {  // NaN stays NaN
  return q != q ? q : __builtin_fminf(__builtin_fmaxf(q, -448.f), 448.f);
}
template <bool VEC>
__device__ __forceinline__ void store8_e4m3(uint8_t* row, int c0, int D, const float (&q)[8]) {
  const uint32_t lo = pack_fp8x4(q[0], q[1], q[2], q[3]), hi = pack_fp8x4(q[4], q[5], q[6], q[7]);
  if constexpr (VEC) {
    *(u32x2*)(row + c0) = u32x2{lo, hi};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < D) row[c0 + e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
  }
}

struct FwdArgs {
  const uint8_t* x;
  const uint8_t* res;  // or null
  const uint8_t* w;
  uint8_t* h;  // with a residual
  uint8_t* y;
  int64_t ldx, ldr, ldh, ldy;  // bytes
  const float* scale_in;       // e4m3: the given scale, or null (the row's own, to scale_out)
  float* scale_out;
  float* rstd;  // or null
  int64_t rows;
  int D, w_f32;
  float eps, inv_d;
};

// A block of BLOCK threads is BLOCK / G row groups; every group walks the same
// number of rows, so that the barriers of a group of several waves are the
// block's.  Measured: 162 251 x 512 bf16 with residual to e4m3 (581 MB) 108 us, 5.4 TB/s;
// 37 429 x 512 bf16 with residual (153 MB) 26-30 us; 4 099 x 5 120 fp32 (168 MB) 33-39 us;
// a large copy runs at 5.1 TB/s.  One row of 2 048 2.6 us, a launch's own time.
// Without VEC (rows not 16-byte aligned, D % 8) every lane makes eight accesses of one
// element where it makes one of 16 bytes, and these requests bound it, forward and
// backward (bf16 with residual; aligned / not): 37 429 x 512 / 513 23.5 / 78 us, its e4m3
// 24 / 85, its backward 26 / 93; 162 251 x 512 / 509 117 / 407, backward 138 / 401.
template <bool F32, bool VEC, int G, int NV, int BLOCK, bool OUT8>
__global__ void __launch_bounds__(BLOCK) rms_fwd_kernel(FwdArgs a) {
  constexpr int GROUPS = BLOCK / G, WPG = G / 64;
  __shared__ float red[2][GROUPS][WPG][2];
  const int group = threadIdx.x / G, tg = threadIdx.x % G, wg = tg >> 6;
  float w[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = 8 * (tg + G * i);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = 0.f;
    if (c0 < a.D) {
      if (a.w_f32) load8<true, VEC>(a.w, c0, a.D, w[i]);
      else load8<false, VEC>(a.w, c0, a.D, w[i]);
    }
  }
  const float given = OUT8 && a.scale_in ? a.scale_in[0] : 0.f;
  int par = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < a.rows; r0 += (int64_t)gridDim.x * GROUPS, par ^= 1) {
    const int64_t row = r0 + group;
    const bool live = row < a.rows;
    float h[NV][8];
    float ss = 0.f;
    uint32_t top = 0;  // bits of max|h w|
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = 8 * (tg + G * i);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = 0.f;
      if (!live || c0 >= a.D) continue;
      load8<F32, VEC>(a.x + row * a.ldx, c0, a.D, h[i]);
      if (a.res) {
        float r[8];
        load8<F32, VEC>(a.res + row * a.ldr, c0, a.D, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[i][e] += r[e];
          if constexpr (!F32) h[i][e] = (float)(__bf16)h[i][e];
        }
        store8<F32, VEC>(a.h + row * a.ldh, c0, a.D, h[i]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = __builtin_fmaf(h[i][e], h[i][e], ss);
        if constexpr (OUT8) top = max(top, magnitude(h[i][e] * w[i][e]));
      }
    }
    ss = wave_sum(ss);
    if constexpr (OUT8) top = wave_top(top);
    if constexpr (WPG > 1) {
      if ((tg & 63) == 0) red[par][group][wg][0] = ss, red[par][group][wg][1] = __builtin_bit_cast(float, top);
      __syncthreads();  // two copies: the next row's sums do not meet this row's readers
      ss = 0.f;
      top = 0;
#pragma unroll
      for (int k = 0; k < WPG; ++k) ss += red[par][group][k][0], top = max(top, magnitude(red[par][group][k][1]));
    }
    if (!live) continue;
    const float rstd = __builtin_amdgcn_rsqf(ss * a.inv_d + a.eps);
    if (a.rstd && tg == 0) a.rstd[row] = rstd;
    float s = 1.f, is = 1.f, up = 1.f, den = 1.f;
    if constexpr (OUT8) {
      // max|y| as max|h w| rstd: one reduction for both statistics
      const float m = __builtin_bit_cast(float, top) * rstd;
      s = a.scale_in ? given : m > 0.f ? m / 448.f : m == 0.f ? 1.f / 448.f : m;  // NaN stays
      // y / s as (y up) / den: 1 / s would overflow for a small s (2^64 in both), and an
      // infinite one has no reciprocal to correct with (y 0: zeros, NaN for an infinite y)
      const bool far = __builtin_fabsf(s) == __builtin_huge_valf();
      up = __builtin_fabsf(s) < 0x1p-100f ? 0x1p64f : far ? 0.f : 1.f;
      den = far ? 1.f : s * up;
      is = 1.f / den;
      if (!a.scale_in && tg == 0) a.scale_out[row] = s;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = 8 * (tg + G * i);
      if (c0 >= a.D) continue;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = h[i][e] * rstd * w[i][e];
        if constexpr (OUT8) y[e] = sat_e4m3(div_by(y[e] * up, den, is));
      }
      if constexpr (OUT8) store8_e4m3<VEC>(a.y + row * a.ldy, c0, a.D, y);
      else store8<F32, VEC>(a.y + row * a.ldy, c0, a.D, y);
    }
  }
}

struct BwdArgs {
  const uint8_t* dy;
  const uint8_t* h;
  const uint8_t* dh;  // or null
  const uint8_t* w;
  const float* rstd;
  uint8_t* dx;
  int64_t lddy, ldh, lddh, lddx;  // bytes
  float* part;                    // [blocks][D]: each block's sum of dy xhat
  int64_t rows;
  int D, w_f32;
  float inv_d;
};

// The same groups, over at most as many blocks as the chip holds at a time: each
// keeps its columns' share of dw in registers over all of its rows and writes it
// once, so that dw costs blocks x D x 8 bytes and no second pass over the rows.
// Measured: 37 429 x 512 bf16 with dh (153 MB) 27-29 us, 5.3-5.7 TB/s; 4 099 x 5 120 fp32
// (252 MB) 44-45 us, 5.6 TB/s; rms_dw_kernel 4 us more.
template <bool F32, bool VEC, int G, int NV, int BLOCK>
__global__ void __launch_bounds__(BLOCK) rms_bwd_kernel(BwdArgs a) {
  constexpr int GROUPS = BLOCK / G, WPG = G / 64;
  __shared__ float red[2][GROUPS][WPG];
  extern __shared__ __attribute__((aligned(16))) float fold[];  // [GROUPS][D] with several groups
  const int group = threadIdx.x / G, tg = threadIdx.x % G, wg = tg >> 6;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = 8 * (tg + G * i);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = dw[i][e] = 0.f;
    if (c0 < a.D) {
      if (a.w_f32) load8<true, VEC>(a.w, c0, a.D, w[i]);
      else load8<false, VEC>(a.w, c0, a.D, w[i]);
    }
  }
  // AHEAD: a row's operands are loaded while the row before it is worked on (a
  // block with one row at a time otherwise waits for each; measured with the
  // blocks of bwd_blocks, 4 099 x 5 120 fp32 61.0 -> 53.2 us, 8 192 x 4 096 bf16 63.8 ->
  // 59.5; rows of one wave overlap by themselves, 162 251 x 512 123.7 -> 128.2)
  constexpr bool AHEAD = G == 256 || G == 512;
  Raw8<F32, VEC> hr[NV], yr[NV], dr[NV];
  float rn = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    rn = a.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = 8 * (tg + G * i);
      if (c0 >= a.D) continue;
      hr[i].load(a.h + row * a.ldh, c0);
      yr[i].load(a.dy + row * a.lddy, c0);
      if (a.dh) dr[i].load(a.dh + row * a.lddh, c0);
    }
  };
  if constexpr (AHEAD) fetch((int64_t)blockIdx.x * GROUPS + group);
  int par = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < a.rows; r0 += (int64_t)gridDim.x * GROUPS, par ^= 1) {
    const int64_t row = r0 + group;
    const bool live = row < a.rows;
    float h[NV][8], dy[NV][8], d[NV][8];
    float m = 0.f;
    if constexpr (!AHEAD) fetch(row);
    const float rstd = live ? rn : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = 8 * (tg + G * i);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = dy[i][e] = d[i][e] = 0.f;
      if (!live || c0 >= a.D) continue;
      hr[i].get(a.h + row * a.ldh, c0, a.D, h[i]);
      yr[i].get(a.dy + row * a.lddy, c0, a.D, dy[i]);
      if constexpr (AHEAD) {
        if (a.dh) dr[i].get(a.dh + row * a.lddh, c0, a.D, d[i]);
      }
    }
    if constexpr (AHEAD) fetch(row + (int64_t)gridDim.x * GROUPS);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] *= rstd;  // xhat
        dw[i][e] = __builtin_fmaf(dy[i][e], h[i][e], dw[i][e]);
        dy[i][e] *= w[i][e];  // c
        m = __builtin_fmaf(dy[i][e], h[i][e], m);
      }
    m = wave_sum(m);
    if constexpr (WPG > 1) {
      if ((tg & 63) == 0) red[par][group][wg] = m;
      __syncthreads();
      m = 0.f;
#pragma unroll
      for (int k = 0; k < WPG; ++k) m += red[par][group][k];
    }
    if (!live) continue;
    m *= a.inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = 8 * (tg + G * i);
      if (c0 >= a.D) continue;
      float dx[8];
      if constexpr (!AHEAD) {
        if (a.dh) dr[i].get(a.dh + row * a.lddh, c0, a.D, d[i]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) dx[e] = __builtin_fmaf(rstd, __builtin_fmaf(-h[i][e], m, dy[i][e]), d[i][e]);
      store8<F32, VEC>(a.dx + row * a.lddx, c0, a.D, dx);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.D;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = 8 * (tg + G * i) + e;
        if (c < a.D) part[c] = dw[i][e];
      }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = 8 * (tg + G * i) + e;
        if (c < a.D) fold[group * a.D + c] = dw[i][e];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += BLOCK) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) t += fold[k * a.D + c];
      part[c] = t;
    }
  }
}

// dw[c] = sum of the blocks' partials, in a fixed order: a workgroup owns 16
// columns, its 64 row lanes sum every 64th partial, four loads in flight, then
// those sums.  Few columns a workgroup, because the time is the chain of loads.
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float* __restrict__ part, int blocks, int D, void* dw,
                                                      int f32) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, c = blockIdx.x * 16 + cl, k = threadIdx.x >> 4;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < D) {
    int b = k;
    for (; b + 192 < blocks; b += 256)
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] += part[(int64_t)(b + 64 * j) * D + c];
    for (; b < blocks; b += 64) t[0] += part[(int64_t)b * D + c];
  }
  red[k][cl] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  // 64 sums -> 4 (a wave's 16 columns x 4) -> 1
  if (threadIdx.x < 64) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += red[16 * k + j][cl];
    red[16 * k][cl] = s;
  }
  __syncthreads();
  if (threadIdx.x < 16 && c < D) {
    const float s = (red[0][cl] + red[16][cl]) + (red[32][cl] + red[48][cl]);
    if (f32) ((float*)dw)[c] = s;
    else ((uint16_t*)dw)[c] = to_bf16(s);
  }
}

constexpr int kMaxD = 16384;
// row groups of a backward block: 8 or 16 waves, whose sums for dw meet in 32 KiB of LDS
int bwd_groups(int D) { return D <= 512 ? 16 : D <= 1024 ? 8 : 1; }
// as many as the chip holds at a time: their sums are written and read again
int bwd_blocks(int64_t rows, int D) {
  const int groups = bwd_groups(D);
  return (int)std::min<int64_t>((rows + groups - 1) / groups, D <= 1024 ? 512 : D <= 4096 ? 768 : 256);
}

template <template <bool, bool, int, int> class L, bool F32, bool VEC, typename... A>
void by_width(int D, A... args) {
  if (D <= 512) L<F32, VEC, 64, 1>::go(args...);
  else if (D <= 1024) L<F32, VEC, 64, 2>::go(args...);
  else if (D <= 2048) L<F32, VEC, 256, 1>::go(args...);
  else if (D <= 4096) L<F32, VEC, 256, 2>::go(args...);
  else if (D <= 8192) L<F32, VEC, 512, 2>::go(args...);
  else L<F32, VEC, 1024, 2>::go(args...);
}
template <bool F32, bool VEC, int G, int NV>
struct Fwd {
  static void go(const FwdArgs& a, bool out8, hipStream_t stream) {
    constexpr int BLOCK = G < 256 ? 256 : G;
    const int64_t blocks = std::min<int64_t>((a.rows * G + BLOCK - 1) / BLOCK, 256 * 2048 / BLOCK);
    if (out8)
      hipLaunchKernelGGL((rms_fwd_kernel<F32, VEC, G, NV, BLOCK, true>), dim3((unsigned)blocks), dim3(BLOCK), 0, stream, a);
    else
      hipLaunchKernelGGL((rms_fwd_kernel<F32, VEC, G, NV, BLOCK, false>), dim3((unsigned)blocks), dim3(BLOCK), 0, stream, a);
  }
};
template <bool F32, bool VEC, int G, int NV>
struct Bwd {
  static void go(const BwdArgs& a, int blocks, hipStream_t stream) {
    constexpr int GROUPS = G > 64 ? 1 : NV == 1 ? 16 : 8, BLOCK = GROUPS * G;
    hipLaunchKernelGGL((rms_bwd_kernel<F32, VEC, G, NV, BLOCK>), dim3((unsigned)blocks), dim3(BLOCK),
                       GROUPS > 1 ? GROUPS * a.D * 4 : 0, stream, a);
  }
};
template <template <bool, bool, int, int> class L, typename... A>
void by_type(bool f32, bool vec, int D, A... args) {
  if (f32 && vec) by_width<L, true, true>(D, args...);
  else if (f32) by_width<L, true, false>(D, args...);
  else if (vec) by_width<L, false, true>(D, args...);
  else by_width<L, false, false>(D, args...);
}

bool aligned16(const void* p, int64_t ld_bytes) { return (uintptr_t)p % 16 == 0 && ld_bytes % 16 == 0; }
// element alignment, which every access needs
bool aligned_es(const void* p, int es) { return (uintptr_t)p % es == 0; }
// Whether rows of `a` (wa bytes each, lda apart) and of `b` share a byte.  Rows of one
// stride may interleave (columns of one wide buffer); of two strides their whole
// ranges have to be apart.
bool share(const void* pa, int64_t lda, int64_t wa, const void* pb, int64_t ldb, int64_t wb, int64_t rows) {
  const int64_t a = (int64_t)(uintptr_t)pa, b = (int64_t)(uintptr_t)pb;
  if (a + (rows - 1) * lda + wa <= b || b + (rows - 1) * ldb + wb <= a) return false;
  if (lda != ldb || rows == 1) return true;
  const int64_t d = ((b - a) % lda + lda) % lda;  // where b's rows begin within a's
  return d < wa || d + wb > lda;
}

}  // namespace

extern "C" int hstu_rms_norm_fwd(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                 const void* weight, int param_dtype, float eps, int64_t rows, int D, void* h,
                                 int64_t ldh, void* y, int64_t ldy, int out_dtype, const float* scale_in,
                                 float* scale_out, float* rstd, hipStream_t stream) {
  const bool f32 = dtype == HSTU_DTYPE_FP32, out8 = out_dtype == HSTU_DTYPE_FP8_E4M3;
  if (!f32 && dtype != HSTU_DTYPE_BF16) return HSTU_E_BAD_ARG;
  if (!out8 && out_dtype != dtype) return HSTU_E_BAD_ARG;
  if (param_dtype != HSTU_DTYPE_BF16 && param_dtype != HSTU_DTYPE_FP32) return HSTU_E_BAD_ARG;
  if (rows < 0 || D <= 0 || ldx < D || ldy < D || (residual && (ldr < D || ldh < D))) return HSTU_E_BAD_ARG;
  if (rows == 0) return 0;
  if (!x || !weight || !y || (residual && !h) || (out8 && !scale_in == !scale_out)) return HSTU_E_BAD_ARG;
  if (D > kMaxD) return HSTU_E_UNSUPPORTED;
  const int es = f32 ? 4 : 2, ws = param_dtype == HSTU_DTYPE_FP32 ? 4 : 2;
  if (!aligned_es(x, es) || !aligned_es(residual, es) || !aligned_es(weight, ws) || !aligned_es(h, es) ||
      !aligned_es(y, out8 ? 1 : es))
    return HSTU_E_UNSUPPORTED;
  FwdArgs a{};
  a.x = (const uint8_t*)x;
  a.res = (const uint8_t*)residual;
  a.w = (const uint8_t*)weight;
  a.h = (uint8_t*)h;
  a.y = (uint8_t*)y;
  a.ldx = ldx * es;
  a.ldr = ldr * es;
  a.ldh = ldh * es;
  a.ldy = ldy * (out8 ? 1 : es);
  a.scale_in = scale_in;
  a.scale_out = scale_out;
  a.rstd = rstd;
  a.rows = rows;
  a.D = D;
  a.w_f32 = ws == 4;
  a.eps = eps;
  a.inv_d = 1.f / (float)D;
  // Row groups run in any order, so an output may lie on an input only where each
  // row lies on itself: the same address, stride and type.  e4m3 rows are shorter.
  const int64_t in_w = (int64_t)D * es, y_w = out8 ? D : in_w;
  auto clash = [&](const void* out, int64_t ldo, int64_t wo, const void* in, int64_t ldi) {
    return share(out, ldo, wo, in, ldi, in_w, rows) && !(out == in && ldo == ldi && wo == in_w);
  };
  if (clash(y, a.ldy, y_w, x, a.ldx)) return HSTU_E_BAD_ARG;
  if (residual && (clash(y, a.ldy, y_w, residual, a.ldr) || clash(h, a.ldh, in_w, x, a.ldx) ||
                   clash(h, a.ldh, in_w, residual, a.ldr) || share(y, a.ldy, y_w, h, a.ldh, in_w, rows)))
    return HSTU_E_BAD_ARG;
  const bool vec = D % 8 == 0 && aligned16(x, a.ldx) && aligned16(weight, 0) &&
                   (!residual || (aligned16(residual, a.ldr) && aligned16(h, a.ldh))) &&
                   (out8 ? (uintptr_t)y % 8 == 0 && a.ldy % 8 == 0 : aligned16(y, a.ldy));
  by_type<Fwd>(f32, vec, D, a, out8, stream);
  return (int)hipGetLastError();
}

extern "C" int64_t hstu_rms_norm_bwd_workspace_bytes(int64_t rows, int D) {
  if (rows < 0 || D <= 0 || D > kMaxD) return -1;
  return (int64_t)std::max(1, bwd_blocks(rows, D)) * D * 4;
}

extern "C" int hstu_rms_norm_bwd(int dtype, const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* dh,
                                 int64_t lddh, const void* weight, int param_dtype, const float* rstd, int64_t rows,
                                 int D, void* dx, int64_t lddx, void* dweight, int dweight_dtype, void* workspace,
                                 int64_t workspace_bytes, hipStream_t stream) {
  const bool f32 = dtype == HSTU_DTYPE_FP32;
  if (!f32 && dtype != HSTU_DTYPE_BF16) return HSTU_E_BAD_ARG;
  if ((param_dtype != HSTU_DTYPE_BF16 && param_dtype != HSTU_DTYPE_FP32) ||
      (dweight_dtype != HSTU_DTYPE_BF16 && dweight_dtype != HSTU_DTYPE_FP32))
    return HSTU_E_BAD_ARG;
  if (rows < 0 || D <= 0 || lddy < D || ldh < D || lddx < D || (dh && lddh < D) || !dweight) return HSTU_E_BAD_ARG;
  if (D > kMaxD) return HSTU_E_UNSUPPORTED;
  if (rows > 0 && (!dy || !h || !weight || !rstd || !dx)) return HSTU_E_BAD_ARG;
  if (!workspace || workspace_bytes < hstu_rms_norm_bwd_workspace_bytes(rows, D)) return HSTU_E_BAD_ARG;
  const int es = f32 ? 4 : 2, ws = param_dtype == HSTU_DTYPE_FP32 ? 4 : 2;
  if (!aligned_es(dy, es) || !aligned_es(h, es) || !aligned_es(dh, es) || !aligned_es(weight, ws) ||
      !aligned_es(dx, es) || !aligned_es(rstd, 4) || (uintptr_t)workspace % 16 ||
      !aligned_es(dweight, dweight_dtype == HSTU_DTYPE_FP32 ? 4 : 2))
    return HSTU_E_UNSUPPORTED;
  const int blocks = bwd_blocks(rows, D);
  if (rows > 0) {
    BwdArgs a{};
    a.dy = (const uint8_t*)dy;
    a.h = (const uint8_t*)h;
    a.dh = (const uint8_t*)dh;
    a.w = (const uint8_t*)weight;
    a.rstd = rstd;
    a.dx = (uint8_t*)dx;
    a.lddy = lddy * es;
    a.ldh = ldh * es;
    a.lddh = lddh * es;
    a.lddx = lddx * es;
    a.part = (float*)workspace;
    a.rows = rows;
    a.D = D;
    a.w_f32 = ws == 4;
    a.inv_d = 1.f / (float)D;
    const bool vec = D % 8 == 0 && aligned16(dy, a.lddy) && aligned16(h, a.ldh) && aligned16(weight, 0) &&
                     aligned16(dx, a.lddx) && (!dh || aligned16(dh, a.lddh));
    by_type<Bwd>(f32, vec, D, a, blocks, stream);
  }
  hipLaunchKernelGGL(rms_dw_kernel, dim3((unsigned)((D + 15) / 16)), dim3(1024), 0, stream, (const float*)workspace,
                     blocks, D, dweight, dweight_dtype == HSTU_DTYPE_FP32 ? 1 : 0);
  return (int)hipGetLastError();
}
