// Matrix-core and per-head helpers shared by the layer-by-layer engine (layers_kernel.hip) and the
// persistent batched decode kernel (batch_kernel.hip) on MI355X (gfx950).
//
// MFMA operand layout (v_mfma_f32_16x16x32_bf16; lane l, i = l % 16, g = l / 16): A[i][8g + j] and
// B[8g + j][i] for j = 0..7 (8 bf16 = 16 bytes per lane), accumulator C[4g + j][i] for j = 0..3.
// Both operands are read as 16-byte chunks of K-contiguous rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mk_device.h"

namespace mkp {
using namespace mk;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr int D = 128, HQ = 16, HKV = 8;
constexpr float EPS = 1e-6f;
constexpr float ATT_SCALE = 0.08838834764831845f;  // 128 ** -0.5

__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                 0, 0, 0);
}

// hi = bf16(v), lo = bf16(v - hi) of 8 values, as two 16-byte chunks
__device__ __forceinline__ void split8(const float* v, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    h[q] = pack_bf16x2(v[2 * q], v[2 * q + 1]);
    l[q] = pack_bf16x2(v[2 * q] - bf16_lo(h[q]), v[2 * q + 1] - bf16_hi(h[q]));
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ void unpack8(uint4 w, float (&v)[8]) {
  v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
  v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
}

// Greedy key of a logit: (order-preserving bf16 of the logit) << 32 | ~idx, so that the maximum key
// is the largest bf16-rounded logit and, among equal ones, the lowest index
// (/root/reference/model.py:97 takes torch's argmax of the logits).
__device__ __forceinline__ u64 argmax_key(float logit, int idx) {
  uint32_t u = (uint32_t)f32_to_bf16(logit) << 16;
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((u64)u << 32) | (0xffffffffu - (uint32_t)idx);
}

// Per-head RMSNorm + rotate-half RoPE of 8 dims of one head row held by a 16-lane row (lane t: dims
// 8t..8t+7; the RoPE partner of dim d is d +- 64, in lane t ^ 8), as the decode kernel applies them
// (/root/reference/megakernel.cu:490-630, 548-555).
__device__ __forceinline__ void head_norm_rope(float (&v)[8], const float (&wn)[8], const float (&cs)[8],
                                               const float (&sn)[8], int t) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
  const float rs = rsqrtf(row16_sum(ss) / (float)D + EPS);
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = v[i] * rs * wn[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float pr = dpp<0x128>(u[i]);  // row_ror:8 inside the 16-lane row: lane t ^ 8
    v[i] = t < 8 ? u[i] * cs[i] - pr * sn[i] : u[i] * cs[i] + pr * sn[i];
  }
}

// Fragment-major layout of a bf16 activation matrix with K columns (K a multiple of 32), the A
// operand of gemm_kernel: 16-row x 32-column blocks of 1 KB, block (m / 16, k / 32) at KB offset
// (m / 16) * (K / 32) + k / 32; inside a block, MFMA lane l = (m % 16) + 16 * ((k % 32) / 8) holds
// the 16 bytes of columns [8 ((k % 32) / 8), +8). A wave reads one operand fragment as 1 KB of
// consecutive bytes. Buffers in this layout hold whole row tiles (operand_rows); rows past M are never
// written, and the sums they produce are never stored.
__device__ __forceinline__ size_t frag_off(int m, int k, int K) {
  return ((((size_t)(m >> 4) * (K >> 5) + (k >> 5)) * 64 + ((k >> 3) & 3) * 16 + (m & 15)) << 3) + (k & 7);
}

// Activation operand of the skinny products in fragment order ("skinny fragments", used by the
// batched decode): for column block cb (sequences 8 cb .. 8 cb + 7) and K block kb (32 inputs), one
// 1 KB fragment holding, at lane l, MFMA column li = l % 16 (sequence 8 cb + li / 2, bf16 hi part for
// even li, lo for odd) and inputs 32 kb + 8 (l / 16) .. + 8. A wave then loads a whole B operand as
// 1 KB of consecutive bytes. In row order (B rows of ldx elements, hi and lo in two arrays) each lane
// of such a load reads 16 bytes of a different row, and the vector cache takes one access per lane:
// at 64 sequences that was the skinny products' bound (rocprof at 64 sequences: ~64 L1 accesses per
// load instruction, TA address stalls). Rows past the batch are never written; their columns of the
// products are never read.
// Column-block major: the K blocks of one column block are adjacent. (K-block major, the column blocks of
// one K block adjacent, measured on MI355X from 9 to 64 sequences and 16 to 256 prompt tokens at both
// widths: within 0.4% either way, but 131 tokens 1,612 -> 1,634 us, 40 at 1.7B 1,740 -> 1,754.)
__host__ __device__ inline int skf_blocks(int B) { return (B + 7) / 8; }
__host__ __device__ inline size_t skf_frag(int cb, int kb, int K) { return (size_t)cb * (K >> 5) + kb; }
__host__ __device__ inline size_t skf_off(int b, int k, int part, int K) {
  const int cb = b >> 3, li = 2 * (b & 7) + part, kb = k >> 5, lg = (k & 31) >> 3;
  return ((skf_frag(cb, kb, K) * 64 + lg * 16 + li) << 3) + (k & 7);
}

}  // namespace mkp
