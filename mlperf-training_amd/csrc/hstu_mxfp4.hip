// Microscaled 4-bit floating point (OCP MX: e2m1 values, one E8M0 scale for 32
// consecutive values of a row): quantisation, its inverse, and the product of
// two quantised matrices, for MI355X (gfx950).
//
//   E = max(floor(log2 max|v|) - 2, -127) of a block (2 is e2m1's largest
//   exponent), scale byte E + 127; code = nearest e2m1 (0, .5, 1, 1.5, 2, 3, 4,
//   6) of v 2^-E, ties to the even code, at most 6.  A block of zeros has byte 0,
//   one with an infinity or NaN byte 255 and stands for NaN.  Codes lie two a
//   byte, the even column in the low half.
//   C[m][n] = sum_k A[m][k] W[n][k] [+ bias[n]] [+ residual[m][n]], A [M, K] and W
//   [N, K] in this format: the matrix cores scale each block of the products'
//   sum, which is kept in fp32.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "hstu_common.h"
#include "hstu_mi355x.h"

namespace {
using namespace hstu;

__device__ __forceinline__ float bf16f(uint32_t b16) { return __builtin_bit_cast(float, b16 << 16); }

// ---------------------------------------------------------------- quantisation
// maximum over the four lanes of a quad
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}
// Scale byte from the exponent field of a block's largest magnitude (255: it is
// infinite or NaN), and the float whose exponent the conversions divide by: 2^E
// (they use the exponent field alone, so byte 0 is 2^-127 there too).
__device__ __forceinline__ uint32_t mx_byte(uint32_t field) { return field == 255u ? 255u : field >= 2u ? field - 2u : 0u; }
__device__ __forceinline__ float mx_divisor(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Largest magnitude of bf16 pairs, as 16-bit integers (NaN above infinity)
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 mag_max(u16x2 top, uint32_t x) {
  return __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t field_of(u16x2 top) { return (uint32_t)max(top[0], top[1]) >> 7; }
// Eight bf16 -> eight codes (round to nearest even, at most 6)
__device__ __forceinline__ uint32_t mx_codes8(u32x4 v, float divisor) {
  const uint32_t x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, x0), divisor, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, x1), divisor, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, x2), divisor, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, x3), divisor, 3);
}
// Eight values of a lane, the block being those of its quad -> codes, scale byte
__device__ __forceinline__ uint32_t mx_encode8(u32x4 v, uint32_t& byte) {
  u16x2 top = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) top = mag_max(top, v[j]);
  byte = mx_byte(quad_max(field_of(top)));
  const uint32_t w = mx_codes8(v, mx_divisor(byte));
  return byte == 255u ? 0u : w;
}
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
  byte = mx_byte(quad_max(top >> 23));
  const float d = mx_divisor(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], d, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], d, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], d, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], d, 3);
  return byte == 255u ? 0u : w;
}
// A whole block, 32 bf16 of one lane
__device__ __forceinline__ u32x4 mx_encode32(const u32x4* x, uint32_t& byte) {
  const u32x4 v0 = x[0], v1 = x[1], v2 = x[2], v3 = x[3];
  u16x2 top = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) top = mag_max(mag_max(mag_max(mag_max(top, v0[j]), v1[j]), v2[j]), v3[j]);
  byte = mx_byte(field_of(top));
  const float d = mx_divisor(byte);
  return u32x4{mx_codes8(v0, d), mx_codes8(v1, d), mx_codes8(v2, d), mx_codes8(v3, d)};
}

struct QuantArgs {
  const uint8_t* x;
  int64_t ldx;  // bytes
  int64_t rows;
  int chunks;  // chunks of 8 values in a row
  uint8_t* codes;
  uint8_t* scales;
};

// A lane takes 8 consecutive values; a quad is a block, so a block's maximum is two
// lane exchanges and the accesses of a wave are whole lines.  VEC: 16-byte aligned
// rows.  Bound by memory: 8 192 x 8 192 bf16 (170 MB) 32-36 us, 4.7-5.3 TB/s; 162 251 x 512
// (210 MB) 43-48; 2 048 x 5 632 fp32 (52 MB) 9.5.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(QuantArgs a) {
  const int64_t total = a.rows * a.chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / a.chunks;
    const int c = (int)(i - row * a.chunks);
    const uint8_t* src = a.x + row * a.ldx + (int64_t)c * (F32 ? 32 : 16);
    uint32_t byte, w;
    if constexpr (F32) {
      float v[8];
      if constexpr (VEC) {
        const f32x4 p = *(const f32x4*)src, q = *(const f32x4*)(src + 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = p[e], v[4 + e] = q[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ((const float*)src)[e];
      }
      w = mx_encode8(v, byte);
    } else {
      u32x4 v;
      if constexpr (VEC) {
        v = *(const u32x4*)src;
      } else {
        const uint16_t* h = (const uint16_t*)src;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (uint32_t)h[2 * e] | (uint32_t)h[2 * e + 1] << 16;
      }
      w = mx_encode8(v, byte);
    }
    ((uint32_t*)a.codes)[i] = w;
    if ((i & 3) == 0) a.scales[i >> 2] = (uint8_t)byte;
  }
}

// 2^(byte - 127); NaN for 255
__device__ __forceinline__ float mx_unit(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}
// Bound by memory: 162 251 x 512 to bf16 (210 MB) 32 us, 6.5 TB/s (the codes are in the
// caches that the quantisation left them in).
template <bool F32>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t total,
                                                            int chunks, uint8_t* out, int64_t ldo) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    const uint32_t w = codes[i];
    const float s = mx_unit(scales[i >> 2]);
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    const float v[8] = {p0[0] * s, p0[1] * s, p1[0] * s, p1[1] * s, p2[0] * s, p2[1] * s, p3[0] * s, p3[1] * s};
    uint8_t* dst = out + row * ldo + (int64_t)c * (F32 ? 32 : 16);
    if constexpr (F32) {
      *(f32x4*)dst = f32x4{v[0], v[1], v[2], v[3]};
      *(f32x4*)(dst + 16) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      *(u32x4*)dst = u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    }
  }
}

// ---------------------------------------------------------------- product
struct MxParams {
  const uint8_t* A;
  const uint8_t* W;
  const uint8_t* as;
  const uint8_t* ws;
  int64_t lda, ldw, ldas, ldws;  // bytes
  const void* bias;              // [N], bf16 or fp32, or null
  const uint16_t* resid;         // bf16 or null
  uint16_t* C;
  int64_t ldr, ldc;  // elements
  int M, N, K;
  int bias_f32;
};

// e2m1 x e2m1 (16x16x128) with E8M0 scales: lane (li, q) holds values 32 q .. 32 q
// + 31 of row li of each operand and, in byte 0 of its scale register, the
// scale of that block.
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 a, u32x4 b, f32x4 c, int sa, int sb) {
  const u32x4 z = {0u, 0u, 0u, 0u};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(cat8(a, z), cat8(b, z), c, 4, 4, 0, sa, 0, sb);
}

__device__ __forceinline__ void add8(u32x4 b, float (&v)[8]) {  // eight bf16
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = b[j];
    v[2 * j] += bf16f(x & 0xffffu);
    v[2 * j + 1] += __builtin_bit_cast(float, x & 0xffff0000u);
  }
}
// The bias of eight columns from n on: added as it is, fp32 or bf16
__device__ __forceinline__ void add_bias8(const MxParams& p, int n, float (&v)[8]) {
  if (p.bias_f32) {
    const f32x4* b = (const f32x4*)((const float*)p.bias + n);
    const f32x4 b0 = b[0], b1 = b[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += b0[e], v[4 + e] += b1[e];
  } else {
    add8(*(const u32x4*)((const uint16_t*)p.bias + n), v);
  }
}
// Four consecutive outputs of row m from column n on.
__device__ __forceinline__ void mx_store4(const MxParams& p, int m, int n, f32x4 v) {
  if (p.bias && p.bias_f32) {
    v += *(const f32x4*)((const float*)p.bias + n);
  } else if (p.bias) {
    const u32x2 b = *(const u32x2*)((const uint16_t*)p.bias + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bf16f(e & 1 ? b[e >> 1] >> 16 : b[e >> 1] & 0xffffu);
  }
  if (p.resid) {
    const u32x2 r = *(const u32x2*)(p.resid + (int64_t)m * p.ldr + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bf16f(e & 1 ? r[e >> 1] >> 16 : r[e >> 1] & 0xffffu);
  }
  *(u32x2*)(p.C + (int64_t)m * p.ldc + n) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
}

// Row form, for few rows, where the weights' bytes and the calls are the time (5 x 5 632
// against 2 048 outputs, 6.1 MB of weights, 6.2-7.3 us with the quantisation): 16 NB
// columns and 16 MB rows a workgroup, whose WAVES waves take one contiguous piece
// of the contraction each, operands going from memory to registers as the MFMA takes
// them, and meet in LDS, where the blocks are summed over the waves in order.
// A step is 256 values: lane (li, q) holds blocks 2 q and 2 q + 1 of row li, so its two
// loads hit one line; a last step of 128 takes block q.
// QUANT: A is bf16 and quantised here: a lane holds whole blocks, so their scales and
// codes need no other lane.  It costs 60 instructions a block, for every 16 NB
// columns again.
template <int MB, int NB, int WAVES, bool QUANT>
__global__ void __launch_bounds__(64 * WAVES) mx_rows_kernel(MxParams p) {
  __shared__ f32x4 part[WAVES][MB * NB][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, q = lane >> 4;
  const int nt = (p.N + 16 * NB - 1) / (16 * NB), mt = blockIdx.x / nt, n0 = (blockIdx.x - mt * nt) * 16 * NB;
  const int m0 = mt * 16 * MB;
  const uint8_t *wp[NB], *wsp[NB], *ap[MB], *asp[MB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {  // columns past N repeat the last
    const int row = min(n0 + 16 * n + li, p.N - 1);
    wp[n] = p.W + (int64_t)row * p.ldw;
    wsp[n] = p.ws + (int64_t)row * p.ldws;
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int m = min(m0 + 16 * b + li, p.M - 1);
    ap[b] = p.A + (int64_t)m * p.lda;
    asp[b] = QUANT ? nullptr : p.as + (int64_t)m * p.ldas;
  }
  f32x4 acc[MB][NB];
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[b][n] = zero4();
  // block `blk` of the contraction against that of the other lanes' q
  auto block = [&](int blk, const u32x4 (&w)[NB], const int (&ws)[NB]) {
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      u32x4 a;
      uint32_t as;
      if constexpr (QUANT) {
        a = mx_encode32((const u32x4*)(ap[b] + 64 * blk), as);
      } else {
        a = *(const u32x4*)(ap[b] + 16 * blk);
        as = asp[b][blk];
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[b][n] = mfma_mx4(w[n], a, acc[b][n], ws[n], (int)as);
    }
  };
  const int steps = p.K / 256, each = (steps + WAVES - 1) / WAVES, s_end = min((wave + 1) * each, steps);
#pragma unroll 2
  for (int s = wave * each; s < s_end; ++s) {
    const int blk = 8 * s + 2 * q;
    u32x4 w0[NB], w1[NB];
    int ws0[NB], ws1[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      w0[n] = *(const u32x4*)(wp[n] + 16 * blk);
      w1[n] = *(const u32x4*)(wp[n] + 16 * blk + 16);
      const int both = *(const uint16_t*)(wsp[n] + blk);
      ws0[n] = both & 255;
      ws1[n] = both >> 8;
    }
    block(blk, w0, ws0);
    block(blk + 1, w1, ws1);
  }
  if ((p.K & 255) && wave == WAVES - 1) {
    const int blk = 8 * steps + q;
    u32x4 w0[NB];
    int ws0[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) w0[n] = *(const u32x4*)(wp[n] + 16 * blk), ws0[n] = wsp[n][blk];
    block(blk, w0, ws0);
  }
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int n = 0; n < NB; ++n) part[wave][b * NB + n][lane] = acc[b][n];
  __syncthreads();
  if (wave >= MB * NB) return;
  const int m = m0 + 16 * (wave / NB) + li, n = n0 + 16 * (wave % NB) + 4 * q;
  if (m >= p.M || n >= p.N) return;
  f32x4 t = part[0][wave][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) t += part[w][wave][lane];
  mx_store4(p, m, n, t);
}

template <int BYTE>
__device__ __forceinline__ f32x16 mfma32_mx4(u32x4 a, u32x4 b, f32x16 c, int sa, int sb) {
  const u32x4 z = {0u, 0u, 0u, 0u};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(cat8(a, z), cat8(b, z), c, 4, 4, BYTE, sa, BYTE, sb);
}

// Middle form, for some hundred rows: 64 x 64 outputs a workgroup of 4 waves (32 x 32
// each), two workgroups per CU, a ring of four 16 KiB steps (256 values of k) with
// three steps' loads in flight and one barrier a step; scales of two steps at a time
// in a ring of four.  Fragments, scale bytes and the last half step as in the tile
// form below.  Bound by what its tiles read from L2, 16 KiB a step each (256 x 8 192 x 8 192:
// 512 tiles, 268 MB).  Measured (us, rows at K = N = 8 192): 64 12.8, 256 21.6, 512 38.3, where
// the weights' bytes are 7.0.
constexpr int kMxFewStages = 4, kMxFewStage = 2 * 64 * 128, kMxFewScales = 4 * 1024;
__global__ void __launch_bounds__(kThreads, 2) mx_few_kernel(MxParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kMxFewStages][kMxFewStage];
  __shared__ __attribute__((aligned(1024))) uint8_t sring[4][kMxFewScales];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int tiles_m = (p.M + 63) / 64, total = tiles_m * ((p.N + 63) / 64), per_xcd = (total + 7) / 8;
  const int t = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (t >= min((((int)blockIdx.x & 7) + 1) * per_xcd, total)) return;
  const int nt = t / tiles_m, mt = t - nt * tiles_m;
  const int m0 = mt * 64, n0 = nt * 64, mrows = min(64, p.M - m0), ncols = min(64, p.N - n0);
  const int wm = 32 * (wave >> 1), wn = 32 * (wave & 1);
  const int S = (p.K + 255) >> 8;
  const int lr = lane & 31, h = lane >> 5;
  auto column = [](int r) {  // output column (in the tile) of LDS row r of W
    const int i = r & 31;
    return (r & ~31) + duo32_col((i >> 2) & 1, 4 * (i >> 3) + (i & 3));
  };
  // wave w fills rows 16 w .. 16 w + 15 of both operands, and the scales of 32 rows:
  // A's (waves 0, 1) or W's (2, 3), each twice in its KiB
  uint32_t av[2], wv[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = 64 * (2 * wave + j) + lane, r = s >> 3;
    const uint32_t pos = (uint32_t)(((s & 7) ^ ((r >> 1) & 7)) * 16);
    av[j] = (uint32_t)r * (uint32_t)p.lda + pos;
    wv[j] = (uint32_t)column(r) * (uint32_t)p.ldw + pos;
  }
  const bool sw_wave = wave >= 2;
  const int sr = 32 * (wave & 1) + lr;
  const uint32_t sv = sw_wave ? (uint32_t)column(sr) * (uint32_t)p.ldws : (uint32_t)sr * (uint32_t)p.ldas;
  // rows past M and N read as zero (code 0, scale byte 0)
  const i32x4 ars = rsrc_sgprs(p.A + (int64_t)m0 * p.lda, (uint32_t)((mrows - 1) * p.lda + p.K / 2));
  const i32x4 wrs = rsrc_sgprs(p.W + (int64_t)n0 * p.ldw, (uint32_t)((ncols - 1) * p.ldw + p.K / 2));
  const i32x4 srs = rsrc_sgprs(sw_wave ? p.ws + (int64_t)n0 * p.ldws : p.as + (int64_t)m0 * p.ldas,
                               sw_wave ? (uint32_t)((ncols - 1) * p.ldws + p.K / 32) : (uint32_t)((mrows - 1) * p.ldas + p.K / 32));
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&ring[0][0];
  const uint32_t sring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&sring[0][0];
  auto issue = [&](int s) {  // four loads of this wave, five in an even step
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring0 + (uint32_t)((s % kMxFewStages) * kMxFewStage + 2048 * wave));
    if ((s & 1) == 0)
      dma_to_lds(__builtin_amdgcn_readfirstlane(sring0 + (uint32_t)(((s >> 1) & 3) * kMxFewScales + 1024 * wave)), sv, srs,
                 (uint32_t)(8 * s));
#pragma unroll
    for (int j = 0; j < 2; ++j) dma_to_lds(dst + 1024 * j, av[j], ars, (uint32_t)(128 * s));
#pragma unroll
    for (int j = 0; j < 2; ++j) dma_to_lds(dst + kMxFewStage / 2 + 1024 * j, wv[j], wrs, (uint32_t)(128 * s));
  };
  for (int s = 0; s < min(kMxFewStages - 1, S); ++s) issue(s);

  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  const uint32_t rd = lr * 128 + (((4 * h) ^ ((lr >> 1) & 7)) * 16);  // chunk 4 h + kk at rd ^ 16 kk
  auto kstep = [&](int s, auto vm_c, bool half) {
    // Step s has landed when only the two later steps' loads are outstanding (nine);
    // the barrier also frees step s - 1's place for step s + 3.
    dma_barrier<decltype(vm_c)::value>();
    if (s + kMxFewStages - 1 < S) issue(s + kMxFewStages - 1);
    const uint8_t* sa = ring[s % kMxFewStages] + wm * 128;
    const uint8_t* sw = ring[s % kMxFewStages] + kMxFewStage / 2 + wn * 128;
    const uint8_t* sc = sring[(s >> 1) & 3] + 16 * lr + 8 * (s & 1) + 4 * h;
    u32x4 a[4], w[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      a[kk] = lds_ld128(sa + (rd ^ (16 * kk)));
      w[kk] = lds_ld128(sw + (rd ^ (16 * kk)));
    }
    int as = *(const int*)(sc + 1024 * (wave >> 1)), ws = *(const int*)(sc + 2048 + 1024 * (wave & 1));
    if (half && h == 1) {  // a last step of 128 values: half 1 has none
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) w[kk] = u32x4{0u, 0u, 0u, 0u};
      as = ws = 0;
    }
    acc = mfma32_mx4<0>(w[0], a[0], acc, ws, as);
    acc = mfma32_mx4<1>(w[1], a[1], acc, ws, as);
    acc = mfma32_mx4<2>(w[2], a[2], acc, ws, as);
    acc = mfma32_mx4<3>(w[3], a[3], acc, ws, as);
  };
  for (int s = 0; s < S - 2; ++s) kstep(s, std::integral_constant<int, 9>{}, false);
  if (S >= 2) kstep(S - 2, std::integral_constant<int, 4>{}, false);
  kstep(S - 1, std::integral_constant<int, 0>{}, (p.K & 255) != 0);

  // lane: row m0 + wm + lr, columns n0 + wn + 16 run + 8 h + (0..7)
  const int m = m0 + wm + lr;
  if (m >= p.M) return;
#pragma unroll
  for (int run = 0; run < 2; ++run) {
    const int c = n0 + wn + 16 * run + 8 * h;
    if (c >= p.N) continue;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = acc[8 * run + e];
    if (p.bias) add_bias8(p, c, o);
    if (p.resid) add8(*(const u32x4*)(p.resid + (int64_t)m * p.ldr + c), o);
    *(u32x4*)(p.C + (int64_t)m * p.ldc + c) =
        u32x4{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7])};
  }
}

// Tile form: 256 x 256 outputs a workgroup of 8 waves (2 x 4 of 128 x 64, 4 x 2
// accumulators of 32 x 32), v_mfma_scale_f32_32x32x64_f8f6f4.
//  * A step is 256 values of k, 128 bytes of each row: 64 KiB, in a ring of two,
//    filled by LDS DMA (inline assembly, explicit waits).  Whole 128-byte lines
//    halve the requests to L2 that 64-byte pieces make.  A row's scales come 16
//    bytes (two steps) at a time, because every row of them is a line of its own.
//  * Fragments roll: while step s's MFMAs run, each register whose last MFMA is
//    issued takes the same fragment of step s + 1.  So step s's place in the ring
//    is free when step s begins, step s + 2's loads go there, and have until step
//    s + 1 begins to land: one barrier a step, which finds the operands read.
//  * Lane half h takes chunks (16 bytes, one block) 4 h .. 4 h + 3 of its row for a
//    step's four MFMAs, so one dword holds its scale bytes and the byte is the
//    instruction's selector.  In a last step of 128 values half 1 has none: its
//    W codes and scales are cleared in registers.
//  * Chunk c of LDS row r lies at c ^ ((r >> 1) & 7): 16 consecutive rows read one
//    chunk each from 16 distinct bank groups.  W rows are permuted in LDS so that a
//    lane holds runs of eight columns.
// Measured: 8 192^3 282-330 us, 3.3-3.9 PFLOP/s (a large library product in e4m3 2.6;
// the instruction alone 6.5 from registers of random codes, the power limit, 9.9 of
// zeros).  Without its MFMAs 206 us, without its loads 235; a workgroup has the CU's LDS
// to itself, so nothing runs under its epilogue.  43 registers are spilled: four are read
// back in the main loop's two steps, the rest around the epilogue.
constexpr int kMxThreads = 512;
constexpr int kMxTile = 256;
constexpr int kMxOperand = kMxTile * 128;    // 32 KiB
constexpr int kMxStage = 2 * kMxOperand;     // A, W
constexpr int kMxScales = 2 * kMxTile * 16;  // 16 bytes for each row of A and W: two steps
constexpr int kMxLds = 2 * kMxStage + 2 * kMxScales;

__global__ void __launch_bounds__(kMxThreads, 2) mx_tile_kernel(MxParams p, int tiles_m, int tiles_n, int per_xcd) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  int mt, nt;
  if (!tile_of(tiles_m, tiles_n, per_xcd, mt, nt)) return;
  const int m0 = mt * kMxTile, n0 = nt * kMxTile;
  const int mrows = min(kMxTile, p.M - m0), ncols = min(kMxTile, p.N - n0);
  const int S = (p.K + 255) >> 8;

  // rows past M and N read as zero (code 0, scale byte 0)
  const i32x4 ars = rsrc_sgprs(p.A + (int64_t)m0 * p.lda, (uint32_t)((mrows - 1) * p.lda + p.K / 2));
  const i32x4 wrs = rsrc_sgprs(p.W + (int64_t)n0 * p.ldw, (uint32_t)((ncols - 1) * p.ldw + p.K / 2));
  // waves 0-3 load A's scales, 4-7 W's: 16 bytes of 64 rows each
  const bool sw_wave = wave >= 4;
  const i32x4 srs = rsrc_sgprs(sw_wave ? p.ws + (int64_t)n0 * p.ldws : p.as + (int64_t)m0 * p.ldas,
                               sw_wave ? (uint32_t)((ncols - 1) * p.ldws + p.K / 32) : (uint32_t)((mrows - 1) * p.ldas + p.K / 32));
  auto column = [](int r) {  // output column (in the tile) of LDS row r of W
    const int i = r & 31;
    return (r & ~31) + duo32_col((i >> 2) & 1, 4 * (i >> 3) + (i & 3));
  };
  // chunk 4 wave + j of 8 LDS rows; j and j + 2 are 16 rows of memory apart
  uint32_t av[2], wv[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int q = 64 * (4 * wave + j) + lane, r = q >> 3;
    const uint32_t pos = (uint32_t)(((q & 7) ^ ((r >> 1) & 7)) * 16);
    av[j] = (uint32_t)r * (uint32_t)p.lda + pos;
    wv[j] = (uint32_t)column(r) * (uint32_t)p.ldw + pos;
  }
  const int sr = 64 * (wave & 3) + lane;
  const uint32_t sv = sw_wave ? (uint32_t)column(sr) * (uint32_t)p.ldws : (uint32_t)sr * (uint32_t)p.ldas;
  const uint32_t lds0 =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)smem);
  // load i (0 .. 7) of this wave for step s; the scales of steps 2 q and 2 q + 1
  auto load = [&](int s, auto i_c) {
    constexpr int i = decltype(i_c)::value, j = i & 3;
    const uint32_t dst = lds0 + (uint32_t)((s & 1) * kMxStage) + 1024u * (uint32_t)(4 * wave + j);
    if constexpr (i < 4) dma_to_lds(dst, av[j & 1], ars, (uint32_t)(128 * s) + (j >> 1) * 16u * (uint32_t)p.lda);
    else dma_to_lds(dst + kMxOperand, wv[j & 1], wrs, (uint32_t)(128 * s) + (j >> 1) * 16u * (uint32_t)p.ldw);
  };
  auto load_scales = [&](int q) {
    dma_to_lds(lds0 + 2 * kMxStage + (uint32_t)((q & 1) * kMxScales) + 1024u * (uint32_t)wave, sv, srs, (uint32_t)(16 * q));
  };

  const int lr = lane & 31, h = lane >> 5, wm = wave >> 2, wn = wave & 3;
  // chunk 4 h + kk of row lr is at rd ^ 16 kk, its scales at rs
  const uint32_t rd = lr * 128 + (((4 * h) ^ ((lr >> 1) & 7)) * 16), rs = 16 * lr + 4 * h;
  const uint32_t a_off = 128 * 128 * wm, w_off = kMxOperand + 64 * 128 * wn;
  const uint32_t as_off = 2 * kMxStage + 16 * 128 * wm, ws_off = 2 * kMxStage + 16 * (kMxTile + 64 * wn);

  u32x4 a[4][4], w[2][4];
  int sa[4], sw[2];
  // fragments of the step at (f, q): its place in the ring, that of its scales
  auto read_a = [&](uint32_t f, uint32_t q, int mb) {
    const uint32_t at = f + a_off + rd;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) a[mb][kk] = lds_ld128(smem + (at ^ (16 * kk)) + 4096 * mb);
    sa[mb] = *(const int*)(smem + q + as_off + rs + 512 * mb);
  };
  auto read_w = [&](uint32_t f, int nb, int kk) { w[nb][kk] = lds_ld128(smem + ((f + w_off + rd) ^ (16 * kk)) + 4096 * nb); };
  auto read_ws = [&](uint32_t q, int nb) { sw[nb] = *(const int*)(smem + q + ws_off + rs + 512 * nb); };
  auto place = [](int s) { return (uint32_t)((s & 1) * kMxStage); };
  auto scale_place = [](int s) { return (uint32_t)(((s >> 1) & 1) * kMxScales + 8 * (s & 1)); };
  f32x16 acc[4][2];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[mb][nb][r] = 0.f;

  static_for<8>([&](auto i_c) { load(0, i_c); });
  load_scales(0);
  if (S > 1) {
    static_for<8>([&](auto i_c) { load(1, i_c); });
    dma_barrier<8>();
  } else {
    dma_barrier<0>();
  }
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) read_w(0, nb, kk);
    read_ws(0, nb);
  }
#pragma unroll
  for (int mb = 0; mb < 4; ++mb) read_a(0, 0, mb);

  // step s; NEXT: there is a step s + 1, which has landed; MORE: and a step s + 2
  // to load, spread between the MFMAs (an even one with the scales of two)
  auto step = [&](int s, auto next_c, auto more_c, auto even_c) {
    constexpr bool NEXT = decltype(next_c)::value, MORE = decltype(more_c)::value, EVEN = decltype(even_c)::value;
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), which the barrier has seen to: tells the compiler
    const uint32_t f = place(s + 1), q = scale_place(s + 1);
    __builtin_amdgcn_sched_barrier(0);
    static_for<16>([&](auto n_c) {
      constexpr int n = decltype(n_c)::value, mb = n >> 2, kk = n & 3;
      static_for<2>([&](auto nb_c) {
        constexpr int nb = decltype(nb_c)::value;
        acc[mb][nb] = mfma32_mx4<kk>(w[nb][kk], a[mb][kk], acc[mb][nb], sw[nb], sa[mb]);
        if constexpr (NEXT && mb == 3) {
          read_w(f, nb, kk);
          if constexpr (kk == 3) read_ws(q, nb);
        }
      });
      if constexpr (NEXT && kk == 3) read_a(f, q, mb);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MORE && EVEN && n == 0) load_scales((s + 2) >> 1);
      if constexpr (MORE && n < 4) {
        load(s + 2, std::integral_constant<int, 2 * n>{});
        load(s + 2, std::integral_constant<int, 2 * n + 1>{});
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  using No = std::false_type;
  using Yes = std::true_type;
  int s = 0;
  for (; s + 3 < S; s += 2) {  // no branches inside: the compiler would move MFMAs across them
    dma_barrier<0>();
    step(s, Yes{}, Yes{}, Yes{});
    dma_barrier<0>();
    step(s + 1, Yes{}, Yes{}, No{});
  }
  if (s + 2 < S) {
    dma_barrier<0>();
    step(s, Yes{}, Yes{}, Yes{});
    ++s;
  }
  if (s + 1 < S) {
    dma_barrier<0>();
    step(s, Yes{}, No{}, No{});
  }
  if ((p.K & 255) && h == 1) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) w[nb][kk] = u32x4{0u, 0u, 0u, 0u};
      sw[nb] = 0;
    }
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) sa[mb] = 0;
  }
  step(S - 1, No{}, No{}, No{});

  // The lane's outputs, rows 32 mb + lr and columns 32 nb + 16 run + 8 h + (0..7) of the
  // wave's 128 x 64, go through LDS (chunk c of row r at c ^ ((r >> 1) & 7) of the wave's
  // 16 KiB), so that a store writes whole lines of 8 rows; the residual
  // comes the same way.  Straight from the registers they are 32-byte pieces of 32 rows
  // (us, pieces / lines: 8 192^3 290 / 282, with a residual 401 / 363, 37 429 x 2 048 x 512 (M x N
  // x K) 74 / 56 and 158 / 113; 2 600 x 2 576 x 768 12.5 / 13.2).
  // A wave's lanes read what others of its lanes wrote: wave_lds_order() between the two.
  dma_barrier<0>();  // every wave has read its last fragments
  int le = lane;
  asm volatile("" : "+v"(le));  // what follows is computed here, not kept in registers over the loop
  const int r8 = le >> 3, wrow = m0 + 128 * wm, wcol = n0 + 64 * wn, c8 = wcol + 8 * (le & 7);
  const uint32_t mine = 128 * 128 * wave;
  // row 8 j + r8, chunk le % 8; and row 32 mb + le % 32, chunk 4 nb + 2 run + le / 32
  auto line_at = [&](int j) { return (mine + 128 * r8 + (((le & 7) ^ (r8 >> 1)) * 16)) ^ (64 * (j & 1)); };
  auto out_at = [&](int nb, int run) {
    return (mine + 128 * (le & 31) + (((le >> 5) ^ ((le >> 1) & 7)) * 16)) ^ (64 * nb + 32 * run);
  };
  if (p.resid) {
    const uint16_t* from = p.resid + min(c8, p.N - 8);
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      u32x4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = *(const u32x4*)(from + (int64_t)min(wrow + 8 * (i + j) + r8, p.M - 1) * p.ldr);
#pragma unroll
      for (int j = 0; j < 8; ++j) *(u32x4*)(smem + line_at(i + j) + 1024 * (i + j)) = v[j];
    }
    wave_lds_order();
  }
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int run = 0; run < 2; ++run) {
      const int c = wcol + 32 * nb + 16 * run + 8 * (le >> 5);
      float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p.bias && c < p.N) add_bias8(p, c, b);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        u32x4* at = (u32x4*)(smem + out_at(nb, run) + 4096 * mb);
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = acc[mb][nb][8 * run + e] + b[e];
        if (p.resid) add8(*at, o);
        *at = u32x4{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7])};
      }
    }
  wave_lds_order();
  if (c8 >= p.N) return;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int m = wrow + 8 * j + r8;
    if (m < p.M) *(u32x4*)(p.C + (int64_t)m * p.ldc + c8) = *(const u32x4*)(smem + line_at(j) + 1024 * j);
  }
}

// the tile form's LDS limit, once a device
hipError_t set_mx_lds() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? (uint64_t)1 << dev : 0;
  if (e != hipSuccess || (done.load() & bit)) return e;
  e = hipFuncSetAttribute((const void*)mx_tile_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kMxLds);
  if (e == hipSuccess) done.fetch_or(bit);
  return e;
}

}  // namespace

extern "C" int hstu_mxfp4_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int cols, void* codes,
                                   void* scales, hipStream_t stream) {
  const bool f32 = dtype == HSTU_DTYPE_FP32;
  if ((!f32 && dtype != HSTU_DTYPE_BF16) || rows < 0 || cols <= 0 || ldx < cols) return HSTU_E_BAD_ARG;
  if (rows > 0 && (!x || !codes || !scales)) return HSTU_E_BAD_ARG;
  const int es = f32 ? 4 : 2;
  if (cols % 32 || (uintptr_t)x % es || (uintptr_t)codes % 4) return HSTU_E_UNSUPPORTED;
  if (rows == 0) return 0;
  QuantArgs a{(const uint8_t*)x, ldx * es, rows, cols / 8, (uint8_t*)codes, (uint8_t*)scales};
  const bool vec = (uintptr_t)x % 16 == 0 && a.ldx % 16 == 0;
  const dim3 grid((unsigned)std::min<int64_t>((rows * a.chunks + 255) / 256, 4096)), block(256);
  if (f32 && vec) hipLaunchKernelGGL((mx_quantize_kernel<true, true>), grid, block, 0, stream, a);
  else if (f32) hipLaunchKernelGGL((mx_quantize_kernel<true, false>), grid, block, 0, stream, a);
  else if (vec) hipLaunchKernelGGL((mx_quantize_kernel<false, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((mx_quantize_kernel<false, false>), grid, block, 0, stream, a);
  return (int)hipGetLastError();
}

extern "C" int hstu_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int cols, int out_dtype,
                                     void* out, int64_t ldo, hipStream_t stream) {
  const bool f32 = out_dtype == HSTU_DTYPE_FP32;
  if ((!f32 && out_dtype != HSTU_DTYPE_BF16) || rows < 0 || cols <= 0 || ldo < cols) return HSTU_E_BAD_ARG;
  if (rows > 0 && (!codes || !scales || !out)) return HSTU_E_BAD_ARG;
  const int es = f32 ? 4 : 2;
  if (cols % 32 || (uintptr_t)codes % 4 || (uintptr_t)out % 16 || (ldo * es) % 16) return HSTU_E_UNSUPPORTED;
  if (rows == 0) return 0;
  const int64_t total = rows * (cols / 8);
  const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 4096)), block(256);
  if (f32)
    hipLaunchKernelGGL((mx_dequantize_kernel<true>), grid, block, 0, stream, (const uint32_t*)codes,
                       (const uint8_t*)scales, total, cols / 8, (uint8_t*)out, ldo * es);
  else
    hipLaunchKernelGGL((mx_dequantize_kernel<false>), grid, block, 0, stream, (const uint32_t*)codes,
                       (const uint8_t*)scales, total, cols / 8, (uint8_t*)out, ldo * es);
  return (int)hipGetLastError();
}

namespace {
// Rows: up to 16, and up to 32 for narrow outputs, where a middle tile's serial steps
// would be the time on a few CUs (us, rows / middle, M x K x N: 32 x 8 192 x 1 024 9.9 /
// 12.0, 32 x 5 632 x 2 048 7.0 / 9.0, 16 x 5 632 x 2 048 5.2 / 8.9; 32 x 2 048 x 5 632 6.3 /
// 4.9, 32 x 8 192 x 8 192 18.9 / 12.0).  Middle: up to three rounds of the chip's 512
// places (us, middle / 256 x 256 tiles: 1 024 tiles 36.9 / 52.7, 1 408 16.7 / 18.3, 2 048
// 23.8 / 19.9 and 78.2 / 59.0).
bool mx_rows_form(int M, int N) { return M <= 16 || (M <= 32 && N <= 2048); }
constexpr int kMxFewTiles = 1536;
int check_product(const MxParams& p, bool quant) {
  if (p.M < 0 || p.N <= 0 || p.K <= 0 || p.ldw < p.K / 2 || p.ldws < p.K / 32 || p.ldc < p.N || (p.resid && p.ldr < p.N) ||
      (quant ? p.lda < 2 * (int64_t)p.K : p.lda < p.K / 2 || p.ldas < p.K / 32))
    return HSTU_E_BAD_ARG;
  if (p.M > 0 && (!p.A || !p.W || !p.ws || !p.C || (!quant && !p.as))) return HSTU_E_BAD_ARG;
  if (p.N % 16 || p.K % 128) return HSTU_E_UNSUPPORTED;
  if (((uintptr_t)p.A | (uintptr_t)p.W | (uintptr_t)p.C | (uintptr_t)p.resid | (uintptr_t)p.bias) % 16 ||
      (p.lda | p.ldw) % 16 || ((uintptr_t)p.as | (uintptr_t)p.ws) % 4 || (p.ldas | p.ldws) % 4 || p.ldc % 8 ||
      (p.resid && p.ldr % 8))
    return HSTU_E_UNSUPPORTED;
  // 32-bit offsets of a tile's rows
  if ((p.lda | p.ldw | p.ldas | p.ldws) >> 23) return HSTU_E_UNSUPPORTED;
  return 0;
}
template <int MB, int NB, bool QUANT>
int launch_rows(const MxParams& p, hipStream_t stream) {
  constexpr int W = 8;
  static_assert(MB * NB <= W, "a wave joins each block");
  const int64_t tiles = ((int64_t)p.M + 16 * MB - 1) / (16 * MB) * ((p.N + 16 * NB - 1) / (16 * NB));
  if (tiles >= ((int64_t)1 << 31)) return HSTU_E_UNSUPPORTED;
  hipLaunchKernelGGL((mx_rows_kernel<MB, NB, W, QUANT>), dim3((unsigned)tiles), dim3(64 * W), 0, stream, p);
  return (int)hipGetLastError();
}
}  // namespace

namespace {
int gemm(const MxParams& p, hipStream_t stream) {
  const int st = check_product(p, false);
  if (st != 0 || p.M == 0) return st;
  if (mx_rows_form(p.M, p.N)) return p.M <= 16 ? launch_rows<1, 1, false>(p, stream) : launch_rows<2, 1, false>(p, stream);
  const int64_t few = ((int64_t)p.M + 63) / 64 * ((p.N + 63) / 64);
  const int64_t tiles_m = ((int64_t)p.M + kMxTile - 1) / kMxTile, tiles_n = (p.N + kMxTile - 1) / kMxTile;
  if (few <= kMxFewTiles) {
    hipLaunchKernelGGL(mx_few_kernel, dim3((unsigned)((few + 7) / 8 * 8)), dim3(kThreads), 0, stream, p);
    return (int)hipGetLastError();
  }
  if (tiles_m * tiles_n >= (1 << 30)) return HSTU_E_UNSUPPORTED;
  hipError_t e = set_mx_lds();
  if (e != hipSuccess) return (int)e;
  const int per_xcd = (int)((tiles_m * tiles_n + 7) / 8);
  hipLaunchKernelGGL(mx_tile_kernel, dim3(8 * per_xcd), dim3(kMxThreads), kMxLds, stream, p, (int)tiles_m, (int)tiles_n,
                     per_xcd);
  return (int)hipGetLastError();
}
int linear_rows(const MxParams& p, hipStream_t stream) {
  const int st = check_product(p, true);
  if (st != 0 || p.M == 0) return st;
  // Two column blocks a workgroup where that still leaves one for every CU: half of
  // the quantisation (us, one / two: 8 x 8 192 x 8 192 (M x K x N) 17.7 / 13.0, 16 x
  // 2 048 x 8 192 8.2 / 6.6; 16 x 4 096 x 4 096 8.3 / 9.5, 5 x 5 632 x 2 048 6.9 / 8.2).
  return p.N >= 8192 ? launch_rows<1, 2, true>(p, stream) : launch_rows<1, 1, true>(p, stream);
}
MxParams product(const void* A, int64_t lda, const void* a_scale, int64_t ldas, const void* W, int64_t ldw,
                 const void* w_scale, int64_t ldws, const void* bias, int bias_f32, const void* residual, int64_t ldr,
                 void* C, int64_t ldc, int M, int N, int K) {
  return MxParams{(const uint8_t*)A, (const uint8_t*)W, (const uint8_t*)a_scale, (const uint8_t*)w_scale, lda, ldw, ldas,
                  ldws, bias, (const uint16_t*)residual, (uint16_t*)C, ldr, ldc, M, N, K, bias_f32};
}
}  // namespace

extern "C" int hstu_mxfp4_gemm(const void* A, int64_t lda, const void* a_scale, int64_t ldas, const void* W,
                               int64_t ldw, const void* w_scale, int64_t ldws, const void* bias, const void* residual,
                               int64_t ldr, void* C, int64_t ldc, int M, int N, int K, hipStream_t stream) {
  return gemm(product(A, lda, a_scale, ldas, W, ldw, w_scale, ldws, bias, 0, residual, ldr, C, ldc, M, N, K), stream);
}

extern "C" int hstu_mxfp4_gemm_bias_fp32(const void* A, int64_t lda, const void* a_scale, int64_t ldas, const void* W,
                               int64_t ldw, const void* w_scale, int64_t ldws, const float* bias, const void* residual,
                               int64_t ldr, void* C, int64_t ldc, int M, int N, int K, hipStream_t stream) {
  return gemm(product(A, lda, a_scale, ldas, W, ldw, w_scale, ldws, bias, 1, residual, ldr, C, ldc, M, N, K), stream);
}

extern "C" int hstu_mxfp4_linear_rows(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* w_scale,
                                      int64_t ldws, const void* bias, const void* residual, int64_t ldr, void* C,
                                      int64_t ldc, int M, int N, int K, hipStream_t stream) {
  return linear_rows(product(x, 2 * ldx, nullptr, 0, W, ldw, w_scale, ldws, bias, 0, residual, ldr, C, ldc, M, N, K),
                     stream);
}

extern "C" int hstu_mxfp4_linear_rows_bias_fp32(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* w_scale,
                                      int64_t ldws, const float* bias, const void* residual, int64_t ldr, void* C,
                                      int64_t ldc, int M, int N, int K, hipStream_t stream) {
  return linear_rows(product(x, 2 * ldx, nullptr, 0, W, ldw, w_scale, ldws, bias, 1, residual, ldr, C, ldc, M, N, K),
                     stream);
}
