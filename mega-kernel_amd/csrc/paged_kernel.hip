// A K/V cache of many sequences in one pool of pages, on MI355X (gfx950): rows quantised as they are written,
// read back, and the attention of each sequence's new token over its pages.
//
// Rows. A row is the 128 numbers of one position and K/V head. In bf16 pages it is rounded to bf16. In 8-bit
// pages it is e4m3 values and one power of two: the least 2^e (e >= -117) with max|x| <= 448 * 2^e. A power of
// two loses nothing against a finer scale (e4m3 keeps its relative precision over 2^15), x / 2^e is exact, so the
// only rounding is the value's own (2^-4 of it), and value * 2^e is exact in bf16, which the attention multiplies.
// A row with an infinity or NaN is NaN throughout. Writing and reading take a wave per position, 16 lanes to a row:
// bound by memory. Measured on MI355X, a write and a read: 14,992 fp32 rows of 8 heads into bf16 pages, and
// 16,492 read back (319 MB moved) 58 us, 5.5 TB/s, where a copy of 4 GiB runs at 4.8; one row to each of 8 sequences 3.6 and 3.3 us
// by the kernels' own times, a launch and three loads that wait for each other (begin, table, row).
//
// Attention. out[b][h] = sum over j < len[b] of softmax_j(q[b][h] . k[j][h / G] / sqrt(128)) v[j][h / G].
// A wave takes 32 keys of one (sequence, K/V head) at a time for up to 16 of its query heads, on the matrix cores
// and in registers alone (v_mfma_f32_16x16x32_bf16, lane l: n = l % 16, g = l / 16):
//   S^T = K . Q^T    keys as rows. Row m of half t is key 8 (m / 4) + 4 t + m % 4, so that lane l holds the scores
//                    of query n against keys 8 g .. 8 g + 7: maximum and sum take registers and two lane swaps;
//   O^T += V^T . P^T the lane's weights are the B operand as they stand (slots 8 g + j mean keys 8 g + j). For the A
//                    operand lane l loads dims 8 n .. 8 n + 7 of keys 8 g .. 8 g + 7, whole rows to 16 lanes, and
//                    swaps them into 8 fragments, the i-th of dims 8 n + i: an 8 x 8 transpose in registers.
//                    Lane l then holds dims 32 g .. 32 g + 31 of query n.
// K's loads for the next 32 keys leave when the scores are made, V's when its fragments are. At 2 queries to a K/V head
// 14 of the 16 columns are zero and the matrix cores are still idle most of the time: the read of the keys bounds it.
// Measured, bf16 queries of 16 heads on 8, both launches: 64 sequences of 900 to 4,095 keys in bf16 pages (655 MB) 120 us,
// 5.5 TB/s; 30,001 keys of one (123 MB) 30 us, 4.1 TB/s, of which 5 are the join; 64 of 64 to 960 in 8-bit pages (69 MB) 23.7 us;
// one of 300 keys 7.9 us: launch, cold code, and lengths, table and keys one after the other. Tiles through LDS would only
// add a trip: a wave's keys are its own, and no second wave reads them.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "mk_device.h"
#include "mk_layers.h"
#include "mk_scan.h"
#include "../../include/megakernel_amd.h"

namespace mkp {

constexpr int64_t ROWS_MAX = 1 << 25;  // of a call: 64 threads each, and a launch has less than 2^32
constexpr int CSEQ = 128;  // sequences per launch of the cache's kernels (their places travel as kernel arguments)
constexpr int MIN_BYTE = 10;  // e8m0 byte of 2^-117: the least e4m3 value times it is bf16's least normal number

struct PagePool {
  uint8_t *k, *v;          // bytes
  uint8_t *ks, *vs;        // scales (8-bit pages)
  int64_t page, head, row;  // bytes between pages, heads, rows
  int64_t spage, shead;
  const int32_t* tables;
  int64_t tstride;
  int tn, pages, shift;  // entries of a table, pages of the pool, log2 of the page size
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CacheArgs {
  PagePool p;
  const uint8_t *k, *v;  // written rows
  uint8_t *ok, *ov;      // read rows, bf16 [rows][heads][128]
  int64_t k_row, k_head, v_row, v_head;  // bytes
  const int32_t* begin;
  int64_t rows, out0;  // rows of this launch, the first of them
  int hkv, nseq, seq0;
  int ones;  // every sequence has one row
  int32_t first[CSEQ];  // each sequence's first row, from out0
};

// The sequence that row r (the same for the whole wave) belongs to: the last one that starts at or before it.
__device__ __forceinline__ int sequence_of(const CacheArgs& a, int lane, int64_t r) {
  if (a.ones) return (int)r;
  int n = 0;
#pragma unroll
  for (int i = 0; i < CSEQ / 64; ++i) {
    const int s = 64 * i + lane;
    n += __popcll(__builtin_amdgcn_ballot_w64(s < a.nseq && a.first[s] <= r));
  }
  return n - 1;
}

__device__ __forceinline__ uint32_t row16_max(uint32_t v) {  // over each 16 lanes
  auto step = [&](uint32_t o) { v = max(v, o); };
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));
  return v;
}

// Where the rows of position r's K/V heads are: in bytes from a pool's start, of values and of scales.
struct Spot {
  bool out;  // out of range
  int64_t at, sat;
};
__device__ __forceinline__ Spot spot_of(const CacheArgs& a, int s, int64_t r) {
  const int64_t pos = (int64_t)a.begin[a.seq0 + s] + (a.ones ? 0 : r - a.first[s]);
  Spot p{true, 0, 0};
  if (pos < 0 || (pos >> a.p.shift) >= a.p.tn) return p;
  const int page = a.p.tables[(a.seq0 + s) * a.p.tstride + (pos >> a.p.shift)];
  const int in = (int)(pos & ((1 << a.p.shift) - 1));
  p.out = (uint32_t)page >= (uint32_t)a.p.pages;
  p.at = page * a.p.page + in * a.p.row;
  p.sat = page * a.p.spage + in;
  return p;
}

// A wave to a position, 16 lanes to a row; the rows of k's heads, then of v's, 16 of them at a time. What a wave writes is
// loaded before its place is looked up. ONCE: past the L2s, where the rows are more than these hold. Measured on MI355X:
// 14,992 fp32 rows of 8 heads (123 MB) into bf16 pages and 16,492 read back 58 us with and 65 us without; 1,092 rows (9 MB,
// still in the L2s from call to call) 14.9 and 13.8.
template <bool FP32, bool E4M3, bool ONCE>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheArgs a) {
  const int lane = threadIdx.x & 63, t = lane & 15;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= a.rows) return;
  Spot p{true, 0, 0};
#pragma unroll 1
  for (int i0 = 0; i0 < 2 * a.hkv; i0 += 16) {
    uint4 w[4][FP32 ? 2 : 1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * k + (lane >> 4), h = i >= a.hkv ? i - a.hkv : i;
      const uint8_t* src = i >= a.hkv ? a.v + (a.out0 + r) * a.v_row + h * a.v_head : a.k + (a.out0 + r) * a.k_row + h * a.k_head;
#pragma unroll
      for (int e = 0; e < (FP32 ? 2 : 1); ++e) {
        w[k][e] = make_uint4(0, 0, 0, 0);
        if (i >= 2 * a.hkv) continue;
        const uint8_t* from = src + (FP32 ? 32 : 16) * t + 16 * e;
        if constexpr (ONCE) w[k][e] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from)));
        else w[k][e] = *reinterpret_cast<const uint4*>(from);
      }
    }
    if (i0 == 0) p = spot_of(a, sequence_of(a, lane, r), r);
    if (p.out) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * k + (lane >> 4), h = i >= a.hkv ? i - a.hkv : i;
      if (i >= 2 * a.hkv) continue;  // (all 16 lanes of a row)
      float x[8];
      if constexpr (FP32) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 z = __builtin_bit_cast(float4, w[k][e]);
          x[4 * e] = z.x; x[4 * e + 1] = z.y; x[4 * e + 2] = z.z; x[4 * e + 3] = z.w;
        }
      } else {
        unpack8(w[k][0], x);
      }
      uint8_t* dst = (i >= a.hkv ? a.p.v : a.p.k) + p.at + h * a.p.head;
      if constexpr (!E4M3) {
        if constexpr (FP32)
          w[k][0] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        *reinterpret_cast<uint4*>(dst + 16 * t) = w[k][0];
      } else {
        uint32_t m = 0;  // the largest magnitude's bits: NaN is above infinity is above the numbers
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
        m = row16_max(m);
        const bool bad = m >= 0x7f800000u;
        // m = 1.f * 2^(E - 127) <= 1.75 * 2^8 * 2^e
        const int byte = bad ? 255 : max(MIN_BYTE, (int)(m >> 23) - 8 + ((m & 0x7fffff) > 0x600000));
        const float inv = __uint_as_float((uint32_t)(254 - (bad ? 127 : byte)) << 23);
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, hi, true);
        *reinterpret_cast<uint2*>(dst + 8 * t) = bad ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : make_uint2(lo, hi);
        if (t == 0) ((i >= a.hkv ? a.p.vs : a.p.ks) + p.sat + h * a.p.shead)[0] = (uint8_t)byte;
      }
    }
  }
}

// Two e4m3 numbers (the low or high half of w) times a power of two, as bf16.
template <bool HIGH>
__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}
__device__ __forceinline__ uint4 bf16x8_of_e4m3(uint32_t a, uint32_t b, float scale) {
  return make_uint4(bf16_of_e4m3<false>(a, scale), bf16_of_e4m3<true>(a, scale), bf16_of_e4m3<false>(b, scale),
                    bf16_of_e4m3<true>(b, scale));
}
// What the conversion takes as a scale, of which it looks at the exponent alone: 0 is 2^-127, an infinity makes NaN.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// The number that the byte of a scale is.
__device__ __forceinline__ float unit_of(uint32_t byte) {
  return byte == 255 ? __builtin_nanf("") : byte == 0 ? 0x1p-127f : __uint_as_float(byte << 23);
}

template <bool E4M3>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheArgs a) {
  const int lane = threadIdx.x & 63, t = lane & 15;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= a.rows) return;
  const Spot p = spot_of(a, sequence_of(a, lane, r), r);
#pragma unroll 1
  for (int i0 = 0; i0 < 2 * a.hkv; i0 += 16) {
    typename std::conditional<E4M3, uint2, uint4>::type x[4];
    uint32_t byte[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * k + (lane >> 4), h = i >= a.hkv ? i - a.hkv : i;
      x[k] = {};
      byte[k] = 255;
      if (i >= 2 * a.hkv || p.out) continue;
      const uint8_t* src = (i >= a.hkv ? a.p.v : a.p.k) + p.at + h * a.p.head;
      if constexpr (E4M3) {
        x[k] = *reinterpret_cast<const uint2*>(src + 8 * t);
        byte[k] = ((i >= a.hkv ? a.p.vs : a.p.ks) + p.sat + h * a.p.shead)[0];
      } else {
        x[k] = *reinterpret_cast<const uint4*>(src + 16 * t);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 4 * k + (lane >> 4), h = i >= a.hkv ? i - a.hkv : i;
      if (i >= 2 * a.hkv) continue;
      u32x4 w = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};  // NaN
      if (!p.out) {
        uint4 y = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (!E4M3) y = x[k];
        else if (byte[k] != 255) y = bf16x8_of_e4m3(x[k].x, x[k].y, scale_of(byte[k]));
        w = u32x4{y.x, y.y, y.z, y.w};
      }
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>((i >= a.hkv ? a.ov : a.ok) + (((a.out0 + r) * a.hkv + h) * D) * 2 + 16 * t));
    }
  }
}

// -----------------------------------------------------------------------------------------------------------
// attention of one token per sequence
// -----------------------------------------------------------------------------------------------------------
constexpr int TK = 32;           // keys to a tile
constexpr int WAVES = 4;         // to a workgroup
constexpr int NQ = 16;           // queries to a unit: (sequence, K/V head, 16 of its query heads)
constexpr int OROW = D + 4;      // floats of a query's output in LDS
constexpr int PART = D + 2;      // floats of one query's partial result: sum, maximum, output
constexpr int SEQ_MAX = 4096;
// Workgroups that share the tiles out: two to a CU, as the registers of two waves to a SIMD allow. (With three waves of
// bf16 queries, on 168 registers: 64 sequences of 900 to 4,095 keys in bf16 pages 132 us instead of 121, as six registers
// spill; of 64 to 960 in 8-bit pages 23.1 instead of 23.9.)
constexpr int PAGED_WGS = 512;
constexpr size_t BASE_BYTES = ((SEQ_MAX + 1) * sizeof(double) + 255) & ~(size_t)255;
// Tiles that the start of a unit costs as much as: 1, 2 and 4 measure within 2% of each other from 1 to 256 sequences,
// except 8-bit pages of 8 keys, where 4 takes 25.8 us and 1 and 2 take 24.4.
constexpr int START = 2;

struct PagedArgs {
  PagePool p;
  const uint8_t* q;
  int64_t q_row, q_head;  // bytes
  uint8_t* out;
  const int32_t* lengths;
  float* part;   // [2 * PAGED_WGS][queries of a unit][PART]
  double* base;  // [nseq + 1]: the first place of each sequence's first unit, and `per`
  int nseq, hkv, g, gt;  // gt: units to a K/V head
  int64_t capacity;           // positions of a table
};

// Keys of sequence b; none if its length is out of range.
__device__ __forceinline__ int valid_length(const PagedArgs& a, int b) {
  const int n = a.lengths[b];
  return n > 0 && n <= a.capacity ? n : 0;
}

// How the work is shared out. Each unit with keys takes START + its tiles places in one row of all units, sequence by
// sequence, and every workgroup `per` places of the row, its waves a part each; the places before a unit's first tile
// stand for what a unit costs by itself (its queries, its first loads). Places are counted in doubles, exactly.
__device__ __forceinline__ double places_of(int length) { return length > 0 ? START + (length + TK - 1) / TK : 0; }
__device__ __forceinline__ double places_per(double total) {
  return fmax(floor((total + PAGED_WGS - 1) / PAGED_WGS), (double)WAVES);
}

// v as the sum of PARTS bf16 numbers, each the rounding of what the ones before it leave
template <int PARTS>
__device__ __forceinline__ void parts_of(const float (&v)[8], uint4 (&p)[PARTS]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int s = 0; s < PARTS; ++s) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (s + 1 < PARTS) {
        r[2 * i] -= bf16_lo(w[i]);
        r[2 * i + 1] -= bf16_hi(w[i]);
      }
    }
    p[s] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool E4M3>
struct Tile {
  uint4 k[2][E4M3 ? 2 : 4];
  typename std::conditional<E4M3, uint2, uint4>::type v[8];
  uint32_t ks[2], vs[2];  // bytes
};
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int i) { return w >> (8 * i) & 255; }

// One score in fp32 from the whole query: see the NaN of parts below.
template <bool E4M3>
__device__ __attribute__((noinline)) float whole_score(const uint8_t* k, float unit, const float* q) {
  float s = 0.f;
  for (int d = 0; d < D; ++d) {
    float x;
    if constexpr (E4M3) x = __builtin_amdgcn_cvt_f32_fp8((int)k[d], 0) * unit;
    else x = bf16_to_f32(reinterpret_cast<const uint16_t*>(k)[d]);
    s = fmaf(q[d], x, s);
  }
  return s;
}

// What a wave has of a unit that it did not do alone, in LDS: up to two to a wave, its first and its last unit.
struct Piece {
  int id, t0, t1, tiles;  // seq * units + unit; t0 == t1: none; the unit's tiles
  int row, nq;            // of the output's (sequence, head) rows, the unit's first; their number
};
struct PagedSmem {
  Piece piece[2 * WAVES];
  float m[2 * WAVES][NQ], l[2 * WAVES][NQ];
};

template <int QP>
__device__ __forceinline__ void store_out(uint8_t* out, int64_t at, float4 y) {  // 4 numbers of the output from at on
  if constexpr (QP == 1) *reinterpret_cast<uint2*>(out + 2 * at) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
  else *reinterpret_cast<float4*>(out + 4 * at) = y;
}

// A weight goes into its product in this many bf16 parts, 24 bits. (Two of them, 2^-17 of a weight lost: 64 sequences of 900 to
// 4,095 keys 0.3% faster in bf16 pages and 2.5% in 8-bit ones, but 0.2% of bf16 outputs round to another side.)
constexpr int PP = 3;

// E4M3: 8-bit pages. QP: bf16 parts of a query (1 for bf16 queries, 3 for fp32 ones).
// PG: 2, a tile lies in one page (8-bit pages: one look-up and one address for all scales, 22.7 us instead of 23.6 for 64
// sequences of 256 to 1,024 keys; bf16 pages gain nothing and take 1); 1, each 8 keys of it do; 0, pages are looked up key
// by key (13 sequences of 128 to 512 keys 10.5 us instead of 9.6, 8-bit pages of 8 keys 25.9 instead of 24.4).
// SPLIT: the tiles of all units are shared out evenly, a unit's parts joined by paged_join_kernel; else a workgroup takes a
// unit, a wave a run of its tiles.
template <bool E4M3, int QP, int PG, bool SPLIT>
__global__ void __launch_bounds__(64 * WAVES, 2) paged_attention_kernel(const PagedArgs a) {
  __shared__ PagedSmem sm;
  extern __shared__ __attribute__((aligned(16))) float outs[];  // [pieces][queries of a unit][OROW]
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int units = a.hkv * a.gt;  // of a sequence
  const int gmax = min(a.g, NQ);
  int b, u, len;       // sequence, unit of it, its keys
  double p = 0, left;  // places of the unit that are behind the wave, places that it has still to do
  // each wave its own two, which nobody else touches before the barrier behind the loop
  if (lane < 2) sm.piece[2 * w + lane].t0 = sm.piece[2 * w + lane].t1 = 0;
  if constexpr (SPLIT) {
    // Every wave for itself: a lane adds up `each` sequences, and the lane that the wave's first place falls to tells
    // the sequence, or (more than 64 of them) the 64 lanes look among its sequences.
    const int each = (a.nseq + 63) / 64;
    double mine = 0;
    int len0 = 0;
#pragma unroll 1
    for (int i = 0; i < each; ++i) {
      const int s = lane * each + i;
      len0 = s < a.nseq ? valid_length(a, s) : 0;
      mine += places_of(len0);
    }
    mine *= units;
    double upto = scan_wave(mine, plus<double>);
    const double total = at_lane(upto, 63);
    const double per = places_per(total), wper = floor((per + WAVES - 1) / WAVES);
    if (blockIdx.x == 0 && w == 0) {  // for the join
      double at = upto - mine;
#pragma unroll 1
      for (int i = 0; i < each; ++i) {
        const int s = lane * each + i;
        if (s < a.nseq) {
          a.base[s] = at;
          if (each > 1) at += places_of(valid_length(a, s)) * units;
        }
      }
      if (lane == 0) a.base[a.nseq] = per;
    }
    if (blockIdx.x * per >= total) return;
    const double lo = blockIdx.x * per + w * wper;
    left = fmin(fmin(wper, per - w * wper), total - lo);
    b = u = len = 0;
    if (left > 0) {
      int at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(lo < upto)) - 1;
      b = at;
      if (each > 1) {
        const double before = at_lane(upto - mine, at);
        const int s = at * each + lane;
        len0 = lane < each && s < a.nseq ? valid_length(a, s) : 0;
        mine = places_of(len0) * units;
        upto = before + scan_wave(mine, plus<double>);
        b = at * each;
        at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(lo < upto)) - 1;
        b += at;
      }
      len = at_lane(len0, at);
      const double cost = places_of(len), off = lo - at_lane(upto - mine, at);
      double q = floor(off / cost);
      if (q * cost > off) --q;
      u = __builtin_amdgcn_readfirstlane((int)q);
      p = off - q * cost;
    }
  } else {
    b = blockIdx.x / units;
    u = blockIdx.x % units;
    len = __builtin_amdgcn_readfirstlane(valid_length(a, b));
    const int T = (len + TK - 1) / TK, each = (T + WAVES - 1) / WAVES;
    p = START + min(T, w * each);
    left = min(each, T - min(T, w * each));
  }
  const int mask = (1 << a.p.shift) - 1;
  int piece = 2 * w;
#pragma unroll 1
  while (left > 0) {
    const int T = (len + TK - 1) / TK;
    const int t0 = __builtin_amdgcn_readfirstlane(max(0, (int)(p - START)));
    const int t1 = __builtin_amdgcn_readfirstlane((int)fmin((double)T, fmax(0.0, p + left - START)));
    if (t1 > t0) {
      const int kh = u / a.gt, h0 = kh * a.g + NQ * (u % a.gt), nq = min(NQ, a.g - NQ * (u % a.gt));
      const int32_t* table = a.p.tables + b * a.p.tstride;
      const uint8_t* kbase = a.p.k + kh * a.p.head;
      const uint8_t* vbase = a.p.v + kh * a.p.head;
      const uint8_t* ksb = E4M3 ? a.p.ks + kh * a.p.shead : nullptr;
      const uint8_t* vsb = E4M3 ? a.p.vs + kh * a.p.shead : nullptr;
      bool bad = false;

      // Places of keys, in bytes from a head's rows: a page's, or that of the first of 8 keys of the lane's (8 (n / 4) of
      // k, 8 g of v), and the rows' from there. In a unit's last tile a key past the last is the last one: its weight is
      // 0, and neither a row past the sequence's nor a page past its last is looked at.
      auto page_of = [&](int key) __attribute__((always_inline)) {
        int page = table[key >> a.p.shift];
        if ((uint32_t)page >= (uint32_t)a.p.pages) {
          bad = true;
          page = 0;
        }
        return page;
      };
      const int row = (int)a.p.row, gk = 8 * (n >> 2), gv = 8 * g;
      uint32_t rk[2], rv[8];  // PG 0: not used
      int64_t pk = 0, pv = 0, sk = 0, sv = 0;
      auto rows_from = [&](int last) __attribute__((always_inline)) {  // keys of the tile up to `last`
        const int k0 = PG == 2 ? 0 : min(gk, last & ~7), v0 = PG == 2 ? 0 : min(gv, last & ~7);
#pragma unroll
        for (int h = 0; h < 2; ++h) rk[h] = (uint32_t)((min(gk + 4 * h + (n & 3), last) - k0) * row + 16 * g);
#pragma unroll
        for (int j = 0; j < 8; ++j) rv[j] = (uint32_t)((min(gv + j, last) - v0) * row + (E4M3 ? 8 : 16) * n);
      };
      auto look_up = [&](int t) __attribute__((always_inline)) {
        if constexpr (PG == 2) {
          const int page = page_of(t * TK), in = t * TK & mask;
          pk = pv = page * a.p.page + in * a.p.row;
          sk = sv = page * a.p.spage + in;
        } else if constexpr (PG == 1) {
          const int last = min(TK, len - t * TK) - 1, k0 = t * TK + min(gk, last & ~7), v0 = t * TK + min(gv, last & ~7);
          const int page = page_of(k0), page2 = page_of(v0);
          pk = page * a.p.page + (k0 & mask) * a.p.row;
          pv = page2 * a.p.page + (v0 & mask) * a.p.row;
          sk = page * a.p.spage + (k0 & mask);
          sv = page2 * a.p.spage + (v0 & mask);
        }
        if (t * TK + TK > len) rows_from(len - t * TK - 1);
      };
      auto place = [&](int t, int kk, int64_t& at, int64_t& sat) __attribute__((always_inline)) {  // of any key
        const int key = min(t * TK + kk, len - 1), page = page_of(key);
        at = page * a.p.page + (key & mask) * a.p.row;
        sat = page * a.p.spage + (key & mask);
      };
      Tile<E4M3> x;
      auto load_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* from;
          if constexpr (PG == 0) {
            int64_t at, sat;
            place(t, gk + 4 * h + (n & 3), at, sat);
            from = kbase + at + 16 * g;
            if constexpr (E4M3) x.ks[h] = ksb[sat];
          } else {
            from = kbase + pk + rk[h];
          }
#pragma unroll
          for (int s = 0; s < (E4M3 ? 2 : 4); ++s) x.k[h][s] = *reinterpret_cast<const uint4*>(from + 64 * s);
        }
        if constexpr (E4M3 && PG > 0) {  // the 8 scales of the lane's 8 keys, of which it takes two
          const uint2 y = *reinterpret_cast<const uint2*>(ksb + sk + (PG == 2 ? gk : 0));
          x.ks[0] = byte_of(y.x, n & 3);
          x.ks[1] = byte_of(y.y, n & 3);
        }
      };
      auto load_v = [&](int t) __attribute__((always_inline)) {
        if constexpr (E4M3 && PG == 0) x.vs[0] = x.vs[1] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint8_t* from;
          if constexpr (PG == 0) {
            int64_t at, sat;
            place(t, gv + j, at, sat);
            from = vbase + at + (E4M3 ? 8 : 16) * n;
            if constexpr (E4M3) x.vs[j >> 2] |= (uint32_t)vsb[sat] << (8 * (j & 3));
          } else {
            from = vbase + pv + rv[j];
          }
          if constexpr (E4M3) x.v[j] = *reinterpret_cast<const uint2*>(from);
          else x.v[j] = *reinterpret_cast<const uint4*>(from);
        }
        if constexpr (E4M3 && PG > 0) {
          const uint2 y = *reinterpret_cast<const uint2*>(vsb + sv + (PG == 2 ? gv : 0));
          x.vs[0] = y.x;
          x.vs[1] = y.y;
        }
      };

      if constexpr (PG > 0) rows_from(TK - 1);
      // the queries as B operands: dims of step s at 8 lanes' width, as the keys' loads have them
      auto dim_of = [&](int s) { return E4M3 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
      uint4 qf[4][QP], raw[4][2];
      const uint8_t* qrow = a.q + b * a.q_row + (int64_t)(h0 + n) * a.q_head;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < (QP > 1 ? 2 : 1); ++h)
          raw[s][h] = n < nq ? *reinterpret_cast<const uint4*>(qrow + (QP > 1 ? 4 : 2) * dim_of(s) + 16 * h) : make_uint4(0, 0, 0, 0);
      look_up(t0);
      load_k(t0);
      load_v(t0);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if constexpr (QP == 1) {
          qf[s][0] = raw[s][0];
        } else {
          float y[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 z = __builtin_bit_cast(float4, raw[s][h]);
            y[4 * h] = z.x; y[4 * h + 1] = z.y; y[4 * h + 2] = z.z; y[4 * h + 3] = z.w;
          }
          parts_of<QP>(y, qf[s]);
        }
      }

      float m = -INFINITY, l = 0.f;
      f32x4 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int t = t0; t < t1; ++t) {
        // scores
        f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            uint4 f;
            if constexpr (E4M3) {
              const uint4 r = x.k[h][st >> 1];
              f = bf16x8_of_e4m3(st & 1 ? r.z : r.x, st & 1 ? r.w : r.y, scale_of(x.ks[h]));
            } else {
              f = x.k[h][st];
            }
#pragma unroll
            for (int i = 0; i < QP; ++i) s[h] = mfma(f, qf[st][i], s[h]);
          }
        if (t * TK + TK > len)  // keys past the last weigh nothing, whatever their scales have made of them
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (t * TK + 8 * g + j >= len) s[j >> 2][j & 3] = -INFINITY;
        if constexpr (QP > 1) {
          // Parts of a query may make NaN of an infinite key where the whole query makes an infinity: such scores are
          // made again, while the query's sum is not NaN already.
          bool again = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) again |= s[j >> 2][j & 3] != s[j >> 2][j & 3];
          if (__builtin_amdgcn_ballot_w64(again && n < nq && l == l)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              int64_t at, sat;
              place(t, 8 * g + j, at, sat);
              if (n < nq && l == l && s[j >> 2][j & 3] != s[j >> 2][j & 3])
                s[j >> 2][j & 3] = whole_score<E4M3>(kbase + at, E4M3 ? unit_of(ksb[sat]) : 1.f,
                                                     reinterpret_cast<const float*>(qrow));
            }
          }
        }
        if (t + 1 < t1) {
          look_up(t + 1);
          load_k(t + 1);
        }
        constexpr float C = ATT_SCALE * 1.4426950408889634f;  // weights are powers of two
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = s[j >> 2][j & 3] * C;
        float top = e[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, e[j]);
        top = xmax32(xmax16(top));
        if (__builtin_amdgcn_ballot_w64(top > m)) {
          const float up = fmaxf(m, top), f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
          m = up;
          l *= f;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __builtin_amdgcn_exp2f(e[j] - ref);
          l += e[j];
        }
        uint4 pf[PP];
        parts_of<PP>(e, pf);
        // values
        if constexpr (E4M3 && PG > 0)
          if (t * TK + TK > len)  // scales behind the last row may be anything
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (t * TK + gv + j >= len) x.vs[j >> 2] = (x.vs[j >> 2] & ~(255u << (8 * (j & 3)))) | 127u << (8 * (j & 3));
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // dims 8 n + 2 c and the next
          uint32_t r[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (E4M3) {
              const float sc = scale_of(byte_of(x.vs[j >> 2], j & 3));
              const uint32_t y = c < 2 ? x.v[j].x : x.v[j].y;
              r[j] = c & 1 ? bf16_of_e4m3<true>(y, sc) : bf16_of_e4m3<false>(y, sc);
            } else {
              r[j] = c == 0 ? x.v[j].x : c == 1 ? x.v[j].y : c == 2 ? x.v[j].z : x.v[j].w;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t f[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              f[q] = __builtin_amdgcn_perm(r[2 * q + 1], r[2 * q], h ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int k = 0; k < PP; ++k) o[2 * c + h] = mfma(make_uint4(f[0], f[1], f[2], f[3]), pf[k], o[2 * c + h]);
          }
        }
        if (t + 1 < t1) load_v(t + 1);
      }
      if (__builtin_amdgcn_ballot_w64(bad)) l = __builtin_nanf("");
      l = xsum32(xsum16(l));

      // the lane's dims 32 g + 8 r + i of query n: the output if the wave had the whole unit, else a piece of it
      const bool whole = t0 == 0 && t1 == T;
      const float inv = whole ? (l > 0.f ? 1.f / l : __builtin_nanf("")) : 1.f;  // no key of weight: NaN, as 0 / 0
      if (n < nq) {
        float* to = outs + (piece * gmax + n) * OROW + 32 * g;
        const int64_t at = ((int64_t)b * a.hkv * a.g + h0 + n) * D + 32 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 y = make_float4(o[i][r] * inv, o[i + 1][r] * inv, o[i + 2][r] * inv, o[i + 3][r] * inv);
            if (whole) store_out<QP>(a.out, at + 8 * r + i, y);
            else *reinterpret_cast<float4*>(to + 8 * r + i) = y;
          }
      }
      if (!whole) {
        if (g == 0) {
          sm.m[piece][n] = m;
          sm.l[piece][n] = l;
        }
        if (lane == 0) sm.piece[piece] = Piece{b * units + u, t0, t1, T, b * a.hkv * a.g + h0, nq};
        piece = 2 * w + 1;
      }
    }
    const double cost = places_of(len);
    left -= cost - p;
    p = 0;
    if (left > 0 && ++u == units) {
      u = 0;
      do ++b;
      while (b < a.nseq && valid_length(a, b) == 0);
      b = __builtin_amdgcn_readfirstlane(b);
      if (b >= a.nseq) break;
      len = __builtin_amdgcn_readfirstlane(valid_length(a, b));
    }
  }
  __syncthreads();

  // The pieces joined, unit by unit, by the wave that has the unit's first: what a query's weights refer to differs from
  // piece to piece. A unit that the workgroup had whole is done, others go to the join.
  const Piece y = sm.piece[min(lane, 2 * WAVES - 1)];  // lane e: piece e
  const uint32_t some = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 2 * WAVES && y.t0 != y.t1);
#pragma unroll 1
  for (int e0 = 2 * w; e0 < 2 * w + 2; ++e0) {
    if (!(some >> e0 & 1)) continue;
    const int id = __builtin_amdgcn_readlane(y.id, e0);
    const uint32_t run = some & (uint32_t)__builtin_amdgcn_ballot_w64(y.id == id);
    if (__ffs(run) - 1 != e0) continue;  // an earlier wave's
    const int t0 = __builtin_amdgcn_readlane(y.t0, e0), t1 = __builtin_amdgcn_readlane(y.t1, 31 - __clz(run));
    const bool whole = t0 == 0 && t1 == __builtin_amdgcn_readlane(y.tiles, e0);
    const int nq = __builtin_amdgcn_readlane(y.nq, e0), row = __builtin_amdgcn_readlane(y.row, e0);
#pragma unroll 1
    for (int i = lane; i < nq * (D / 4); i += 64) {
      const int qi = i / (D / 4), d = 4 * (i % (D / 4));
      float M = -INFINITY;
#pragma unroll 2
      for (int e = 0; e < 2 * WAVES; ++e) M = run >> e & 1 ? fmaxf(M, sm.m[e][qi]) : M;
      const float ref = M == -INFINITY ? 0.f : M;
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (uint32_t todo = run; todo; todo &= todo - 1) {
        const int e = __ffs(todo) - 1;
        const float f = __builtin_amdgcn_exp2f(sm.m[e][qi] - ref);
        const float4 z = *reinterpret_cast<const float4*>(outs + (e * gmax + qi) * OROW + d);
        sum += f * sm.l[e][qi];
        acc.x += f * z.x; acc.y += f * z.y; acc.z += f * z.z; acc.w += f * z.w;
      }
      if (whole) {
        const float inv = sum > 0.f ? 1.f / sum : __builtin_nanf("");
        store_out<QP>(a.out, (int64_t)(row + qi) * D + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      } else {
        float* to = a.part + ((int64_t)(2 * blockIdx.x + (t0 == 0)) * gmax + qi) * PART;
        if (d == 0) {
          to[0] = sum;
          to[1] = M;
        }
        *reinterpret_cast<float2*>(to + 2 + d) = make_float2(acc.x, acc.y);  // (PART is even: 8-byte aligned)
        *reinterpret_cast<float2*>(to + 4 + d) = make_float2(acc.z, acc.w);
      }
    }
  }
  if constexpr (!SPLIT)
    if (len == 0) {  // an empty sequence, or a length out of range
      const float y = a.lengths[b] == 0 ? 0.f : __builtin_nanf("");
      const int kh = u / a.gt, h0 = kh * a.g + NQ * (u % a.gt), nq = min(NQ, a.g - NQ * (u % a.gt));
      for (int i = tid; i < nq * (D / 4); i += 64 * WAVES)
        store_out<QP>(a.out, ((int64_t)b * a.hkv * a.g + h0) * D + 4 * i, make_float4(y, y, y, y));
    }
}

// Joins the parts of the units that more than one workgroup worked on, in their order: a workgroup to `take` pairs of
// (sequence, query head), a lane to look at each, and the whole of it to join the few that need it. The pairs of a workgroup lie
// far apart, as all heads of a long sequence need it (one of 8,000 keys among 256 short ones 19 us, 41 with neighbours). Sequences
// without keys get their answer here too.
template <bool FP32>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a, int take) {
  __shared__ __attribute__((aligned(16))) float acc[8][D];
  __shared__ float accl[8], accm[8];
  const int tid = threadIdx.x, lane = tid & 63;
  const int heads = a.hkv * a.g, gmax = min(a.g, NQ), step = gridDim.x, pairs = a.nseq * heads;
  int len = 0, w0 = 0, w1 = 0;
  bool some = false;
  auto pair_of = [&](int e) { return (int)blockIdx.x + e * step; };
  if (lane < take && pair_of(lane) < pairs) {
    const int b = pair_of(lane) / heads, h = pair_of(lane) % heads;
    len = valid_length(a, b);
    const double per = a.base[a.nseq], cost = places_of(len);
    const double u0 = a.base[b] + (h / a.g * a.gt + h % a.g / NQ) * cost;
    w0 = (int)floor((u0 + START) / per);
    w1 = (int)floor((u0 + cost - 1) / per);
    some = len > 0 && w0 != w1;
  }
  {  // sequences without keys, 16 lanes to a pair
    const int e = tid >> 4, item = pair_of(e), keys = __shfl(len, e);
    if (e < take && item < pairs && keys == 0) {
      const float y = a.lengths[item / heads] == 0 ? 0.f : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        store_out<FP32 ? 2 : 1>(a.out, (int64_t)item * D + 8 * (tid & 15) + i, make_float4(y, y, y, y));
    }
  }
#pragma unroll 1
  for (u64 todo = __builtin_amdgcn_ballot_w64(some); todo; todo &= todo - 1) {
    const int e = __ffsll(todo) - 1, item = pair_of(e);
    const int64_t at = (int64_t)item * D + tid;
    auto store = [&](float x) {
      if constexpr (FP32) reinterpret_cast<float*>(a.out)[at] = x;
      else reinterpret_cast<uint16_t*>(a.out)[at] = f32_to_bf16(x);
    };
    const int v1 = at_lane(w1, e), vs = at_lane(w0, e), qi = item % heads % a.g % NQ;
    auto slot = [&](int v) { return a.part + ((int64_t)(2 * v + (v == vs)) * gmax + qi) * PART; };
    // 32 lanes to a part, eight parts of a lane at a time, so that their loads are made together
    const int r = tid >> 5, d = 4 * (tid & 31);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f, M = -INFINITY;
#pragma unroll 1
    for (int v0 = vs + r; v0 <= v1; v0 += 64) {
      float2 ml[8], x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* p = slot(min(v0 + 8 * i, v1));
        ml[i] = *reinterpret_cast<const float2*>(p);
        x[i] = *reinterpret_cast<const float2*>(p + 2 + d);
        y[i] = *reinterpret_cast<const float2*>(p + 4 + d);
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, v0 + 8 * i <= v1 ? ml[i].y : -INFINITY);
      const float ref = top == -INFINITY ? 0.f : top, f0 = __builtin_amdgcn_exp2f(M - ref);
      M = top;
      sum *= f0;
      o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (v0 + 8 * i > v1) continue;
        const float f = __builtin_amdgcn_exp2f(ml[i].y - ref);
        sum += f * ml[i].x;
        o.x += f * x[i].x; o.y += f * x[i].y; o.z += f * y[i].x; o.w += f * y[i].y;
      }
    }
    *reinterpret_cast<float4*>(&acc[r][d]) = o;
    if (d == 0) {
      accl[r] = sum;
      accm[r] = M;
    }
    __syncthreads();
    if (tid < D) {
      M = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) M = fmaxf(M, accm[i]);
      const float ref = M == -INFINITY ? 0.f : M;
      float x = 0.f, all = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = __builtin_amdgcn_exp2f(accm[i] - ref);
        x += f * acc[i][tid];
        all += f * accl[i];
      }
      store(x * (all > 0.f ? 1.f / all : __builtin_nanf("")));
    }
    __syncthreads();
  }
}

static bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether the rows of `width` elements at these strides are places of their own.
static bool apart(int64_t width, std::initializer_list<std::pair<int64_t, int64_t>> dims) {  // (stride, count)
  std::pair<int64_t, int64_t> d[3];
  int n = 0;
  for (const auto& x : dims)
    if (x.second > 1) d[n++] = x;
  std::sort(d, d + n);
  for (int i = 0; i < n; ++i) {
    if (d[i].first < width) return false;
    width += d[i].first * (d[i].second - 1);
  }
  return true;
}

// The pool as the kernels take it; false where it is not one, or is to be written and has rows that overlap.
static bool pool_of(const mk_paged_cache* c, PagePool& p, bool written) {
  if (!c || !c->k_pages || !c->v_pages || c->k_pages == c->v_pages || !c->block_tables) return false;
  const bool e4m3 = c->k_scales || c->v_scales;
  if (e4m3 && (!c->k_scales || !c->v_scales || c->k_scales == c->v_scales)) return false;
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_pages < 1 || c->page_size < 1 || c->page_size > 4096 ||
      (c->page_size & (c->page_size - 1)) != 0 || c->num_seqs < 1 || c->table_entries < 1 || c->table_stride < 0 ||
      (int64_t)c->table_entries * c->page_size > 1 << 30)
    return false;
  const int64_t size = e4m3 ? 1 : 2, unit = 16 / size;
  for (int64_t s : {c->page_stride, c->head_stride, c->row_stride})
    if (s < 0 || s % unit != 0) return false;
  if (c->row_stride > (1 << 24)) return false;  // a page's rows are told apart by 32 bits
  if (!aligned_to(c->k_pages, 16) || !aligned_to(c->v_pages, 16) || !aligned_to(c->block_tables, 4)) return false;
  if (e4m3 && (c->scale_page_stride < 0 || c->scale_head_stride < 0)) return false;
  if (written) {
    if (!apart(D, {{c->page_stride, c->num_pages}, {c->head_stride, c->kv_heads}, {c->row_stride, c->page_size}})) return false;
    if (e4m3 && !apart(c->page_size, {{c->scale_page_stride, c->num_pages}, {c->scale_head_stride, c->kv_heads}})) return false;
  }
  p.k = static_cast<uint8_t*>(c->k_pages);
  p.v = static_cast<uint8_t*>(c->v_pages);
  p.ks = static_cast<uint8_t*>(c->k_scales);
  p.vs = static_cast<uint8_t*>(c->v_scales);
  p.page = c->page_stride * size;
  p.head = c->head_stride * size;
  p.row = c->row_stride * size;
  p.spage = c->scale_page_stride;
  p.shead = c->scale_head_stride;
  p.tables = c->block_tables;
  p.tstride = c->table_stride;
  p.tn = c->table_entries;
  p.pages = c->num_pages;
  p.shift = 0;
  while ((1 << p.shift) < c->page_size) ++p.shift;
  return true;
}

// The launches of a cache call: at most CSEQ sequences to each.
template <typename F>
static hipError_t cache_launches(CacheArgs& a, const int32_t* lengths, int num_seqs, F launch) {
  a.out0 = 0;
  for (int s = 0; s < num_seqs; s += CSEQ) {
    a.seq0 = s;
    a.nseq = std::min(CSEQ, num_seqs - s);
    int64_t at = 0;
    for (int i = 0; i < a.nseq; ++i) {
      a.first[i] = (int32_t)at;
      at += lengths[s + i];
    }
    a.rows = at;
    a.ones = 1;
    for (int i = 0; i < a.nseq; ++i) a.ones &= lengths[s + i] == 1;
    if (at == 0) continue;
    launch(dim3((unsigned)((at + 3) / 4)));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.out0 += at;
  }
  return hipSuccess;
}

// Rows in all; -1 where the lengths are not ones.
static int64_t rows_of(const int32_t* lengths, int num_seqs) {
  if (!lengths) return -1;
  int64_t total = 0;
  for (int i = 0; i < num_seqs; ++i) {
    if (lengths[i] < 0) return -1;
    total += lengths[i];
  }
  return total <= ROWS_MAX ? total : -1;
}

// Tables of at most 512 positions, 16 tiles to a unit, take one launch: four tiles to a wave at most. Measured, heads 16 / 8,
// bf16 pages, lengths even over capacity / 4 .. capacity, without and with the split: capacity 512 one sequence 6.4 and
// 8.5 us, 13 of them 9.6 and 10.7, 64 17.9 and 20.7, 256 63.0 and 65.4; capacity 1,024 one 13.2 and 8.9, 13 16.5 and 12.9,
// 64 30.6 and 33.2, 256 128 and 135, but 64 of which one is full and the others have up to 64 keys 14.7 and 10.7; capacity 768
// 64 23.2 and 26.7, 256 92 and 101, one full among 64 12.3 and 11.1.
static bool paged_split(int64_t capacity) { return capacity > 512; }

}  // namespace mkp

using namespace mkp;

extern "C" hipError_t mk_cache_write(const mk_paged_cache* cache, const void* k, int64_t k_row_stride,
                                     int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride,
                                     int rows_fp32, const int32_t* begin, const int32_t* lengths, hipStream_t stream) {
  CacheArgs a{};
  if (!pool_of(cache, a.p, true) || !begin) return hipErrorInvalidValue;
  const int64_t rows = rows_of(lengths, cache->num_seqs);
  if (rows < 0) return hipErrorInvalidValue;
  if (rows == 0) return hipSuccess;
  if (!k || !v || !aligned_to(k, 16) || !aligned_to(v, 16)) return hipErrorInvalidValue;
  const int size = rows_fp32 ? 4 : 2;
  for (int64_t s : {k_row_stride, k_head_stride, v_row_stride, v_head_stride})
    if (s < 0 || s % (16 / size) != 0) return hipErrorInvalidValue;
  a.k = static_cast<const uint8_t*>(k);
  a.v = static_cast<const uint8_t*>(v);
  a.k_row = k_row_stride * size;
  a.k_head = k_head_stride * size;
  a.v_row = v_row_stride * size;
  a.v_head = v_head_stride * size;
  a.begin = begin;
  a.hkv = cache->kv_heads;
  return cache_launches(a, lengths, cache->num_seqs, [&](dim3 grid) {
    const bool once = a.rows * a.hkv * (2 * D) * size > 32 << 20;
    auto go = [&](auto fp32, auto e4m3) {
      if (once) hipLaunchKernelGGL((cache_write_kernel<fp32.value, e4m3.value, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((cache_write_kernel<fp32.value, e4m3.value, false>), grid, dim3(256), 0, stream, a);
    };
    if (rows_fp32) a.p.ks ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
    else a.p.ks ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
  });
}

extern "C" hipError_t mk_cache_read(const mk_paged_cache* cache, const int32_t* begin, const int32_t* lengths, void* k,
                                    void* v, hipStream_t stream) {
  CacheArgs a{};
  if (!pool_of(cache, a.p, false) || !begin) return hipErrorInvalidValue;
  const int64_t rows = rows_of(lengths, cache->num_seqs);
  if (rows < 0) return hipErrorInvalidValue;
  if (rows == 0) return hipSuccess;
  if (!k || !v || k == v || !aligned_to(k, 16) || !aligned_to(v, 16)) return hipErrorInvalidValue;
  a.ok = static_cast<uint8_t*>(k);
  a.ov = static_cast<uint8_t*>(v);
  a.begin = begin;
  a.hkv = cache->kv_heads;
  return cache_launches(a, lengths, cache->num_seqs, [&](dim3 grid) {
    if (a.p.ks) hipLaunchKernelGGL(cache_read_kernel<true>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(cache_read_kernel<false>, grid, dim3(256), 0, stream, a);
  });
}

extern "C" size_t mk_attention_paged_workspace_bytes(int q_heads, int kv_heads) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0) return 0;
  return BASE_BYTES + (((size_t)2 * PAGED_WGS * std::min(NQ, q_heads / kv_heads) * PART * sizeof(float) + 255) & ~(size_t)255);
}

// Up to this many pairs of (sequence, query head) the join takes a workgroup to each, then one to 16, as few of them need
// one. Measured, 1 and 16: 4,096 pairs 6.3 and 9.2 us, 8,192 9.8 and 6.3, 16,384 15.6 and 7.0, 65,536 49 and 7.5.
constexpr int JOIN_WGS = 4096;
template <bool E4M3, int QP, int PG>
static void launch_paged(const PagedArgs& a, hipStream_t stream) {
  const unsigned units = (unsigned)((int64_t)a.nseq * a.hkv * a.gt);
  const unsigned lds = 2 * WAVES * std::min(a.g, NQ) * OROW * sizeof(float);
  if (!paged_split(a.capacity)) {
    hipLaunchKernelGGL((paged_attention_kernel<E4M3, QP, PG, false>), dim3(units), dim3(64 * WAVES), lds, stream, a);
  } else {
    hipLaunchKernelGGL((paged_attention_kernel<E4M3, QP, PG, true>), dim3(PAGED_WGS), dim3(64 * WAVES), lds, stream, a);
    const int pairs = a.nseq * a.hkv * a.g, take = pairs > JOIN_WGS ? 16 : 1;
    hipLaunchKernelGGL(paged_join_kernel<(QP > 1)>, dim3((pairs + take - 1) / take), dim3(256), 0, stream, a, take);
  }
}

extern "C" hipError_t mk_attention_paged(const mk_paged_cache* cache, int q_heads, const void* q, int64_t q_row_stride,
                                         int64_t q_head_stride, int q_fp32, const int32_t* lengths, void* out,
                                         void* workspace, size_t workspace_bytes, hipStream_t stream) {
  PagedArgs a{};
  if (!pool_of(cache, a.p, false)) return hipErrorInvalidValue;
  const size_t need = mk_attention_paged_workspace_bytes(q_heads, cache->kv_heads);
  if (need == 0 || cache->num_seqs > SEQ_MAX || (int64_t)cache->num_seqs * q_heads > INT32_MAX / D) return hipErrorInvalidValue;
  if (!q || !out || !lengths || !workspace || workspace_bytes < need || !aligned_to(workspace, 256)) return hipErrorInvalidValue;
  if (!aligned_to(q, 16) || !aligned_to(out, 16)) return hipErrorInvalidValue;
  const int size = q_fp32 ? 4 : 2;
  for (int64_t s : {q_row_stride, q_head_stride})
    if (s < 0 || s % (16 / size) != 0) return hipErrorInvalidValue;
  a.q = static_cast<const uint8_t*>(q);
  a.q_row = q_row_stride * size;
  a.q_head = q_head_stride * size;
  a.out = static_cast<uint8_t*>(out);
  a.lengths = lengths;
  a.base = static_cast<double*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + BASE_BYTES);
  a.nseq = cache->num_seqs;
  a.hkv = cache->kv_heads;
  a.g = q_heads / cache->kv_heads;
  a.gt = (a.g + NQ - 1) / NQ;
  a.capacity = (int64_t)cache->table_entries * cache->page_size;
  // the keys of a tile that surely share a page, and scales that can be loaded 8 at a time
  int pg = a.p.ks && cache->page_size >= TK ? 2 : cache->page_size >= 8 ? 1 : 0;
  if (a.p.ks && (!aligned_to(a.p.ks, 8) || !aligned_to(a.p.vs, 8) || a.p.spage % 8 != 0 || a.p.shead % 8 != 0)) pg = 0;
  auto launch = [&](auto e4m3, auto qp) {
    if constexpr (e4m3.value)
      if (pg == 2) return launch_paged<true, qp.value, 2>(a, stream);
    if (pg == 1) launch_paged<e4m3.value, qp.value, 1>(a, stream);
    else launch_paged<e4m3.value, qp.value, 0>(a, stream);
  };
  constexpr std::integral_constant<int, 1> bf16;
  constexpr std::integral_constant<int, 3> fp32;
  if (a.p.ks) q_fp32 ? launch(std::true_type(), fp32) : launch(std::true_type(), bf16);
  else q_fp32 ? launch(std::false_type(), fp32) : launch(std::false_type(), bf16);
  return hipGetLastError();
}
