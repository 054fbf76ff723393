// Causal attention of packed sequences on MI355X (gfx950): the prompts of several sequences, one after
// the other in one array of rows, each attending to itself alone.
//
//   out[t][h] = sum over j <= t of softmax_j(q[t][h] . k[j][h / G] / sqrt(128)) v[j][h / G]
//
// for every token t of every sequence, j over the same sequence's tokens, G query heads on each K/V head.
//
// Tiles. The G query heads of a K/V head share its keys, so a sequence's queries of one K/V head are
// taken as len * G rows, row r = (token r / G, head r % G), whatever G is. A workgroup takes 128
// consecutive rows (on small grids 64 or 32), a wave 32 of them, and runs over the keys 64 or 32 at a time up to its
// last token's, where that pays with its waves in groups on different keys:
//   S^T = K . Q^T   (v_mfma_f32_32x32x16_bf16, keys as rows): lane l holds the scores of its one query
//                   l % 32 against keys 8 (j / 4) + 4 (l / 32) + j % 4, j = 0..15, of each 32-key half,
//                   so the running maximum takes registers and one lane swap, the sum registers alone;
//   O^T += V^T . P^T: the lane's own weights, rounded to bf16, are the B operand as they stand when the
//                   K slots of a 16-key step mean keys {4 g .. 4 g + 3, 8 + 4 g .. +3} (g = l / 32); the
//                   A operand is V read transposed from LDS (ds_read_b64_tr_b16) in the same order. The
//                   output's columns are the queries too: rescaling is one factor per lane.
// K and V tiles are staged through LDS, two deep. 32 rows to a wave rather than 64: the output and the scores of
// two tiles then stay in the 256 registers of two waves per SIMD (64 rows: 628 us where 32 took 372 then).
//
// Bound by the matrix cores and the exponentials beside them on long sequences: 8,192 + 4,096 + 1,801 tokens of 16
// heads on 8 take 362 us, 987 TFLOP/s of useful products (a library product of 16,384 cubed: 1,351), MFMA busy 47%
// and VALU issuing 40% of the time; 3,584 fp32 tokens 141 us, 1,120 TFLOP/s with the three products each. By
// memory and the blocks' first loads on short ones: 64 prompts of 64 to 960 tokens 150 us (2.7 TB/s, 580 TFLOP/s).
// By latency on few: 32 tokens 5.8 us, most of it the fetch of code and operands by one wave per SIMD.
//
// Rounding. Queries and weights are multiplied as PARTS bf16 numbers whose sum they are: 1 for bf16
// queries (a weight is then off by at most 2^-8 of itself, as the output is by its own rounding), 2 for
// the prefill's hi/lo pairs (2^-16), 3 for fp32 queries (2^-24). Scores, maximum, sum and output are fp32.
// One bf16 number per weight keeps the second product at one MFMA per fragment; outputs of bf16 queries are then
// 0.0017 to 0.0020 of their norm from 64 bits, 0.0015 to 0.0016 with weights of 32 bits (the output's own rounding).
//
// A masked key weighs nothing, whatever its value row holds: a tile that some query sees in part is looked
// over for infinities and NaN, and where it has any they are left out of the matrix product (0 times infinity would
// reach the others). Where weights are multiplied by parts, every tile is (a part may be 0 or negative where the
// weight is not). Behind the loop a block that left some out, or whose outputs are not finite, looks for those that
// each query sees: they are its output, also where fp32 holds their weight as 0.
// Keys stay as they are: an infinite one may give such queries a NaN where the formula has an infinity. The sum shows
// it, and the row is made again from whole queries (fp32 and hi/lo queries alone; nothing of it is in the loop).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <numeric>
#include <type_traits>
#include <vector>

#include "mk_batch.h"
#include "mk_device.h"
#include "mk_layers.h"
#include "mk_packed.h"
#include "../../include/megakernel_amd.h"

namespace mkp {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int PSEQ = 128;      // sequences per launch (their places travel as kernel arguments)

// Division by a number that the host knows: q = n / d for 0 <= n < 2^31 by a multiplication (the rounded-up
// reciprocal of d at 32 + ceil(log2 d) bits is off by less than 2^-31 of n / d).
struct DivBy {
  uint32_t d, mul, shift;
};
static DivBy div_by(uint32_t d) {
  uint32_t l = 0;
  while ((1u << l) < d) ++l;
  return {d, (uint32_t)(((1ull << (32 + l)) + d - 1) / d - (1ull << 32)), l};  // the multiplier's low 32 of 33 bits
}
__device__ __forceinline__ int div(uint32_t n, const DivBy& b) {
  return (int)((uint32_t)(((uint64_t)__umulhi(n, b.mul) + n) >> b.shift));
}
__device__ __forceinline__ int mod(uint32_t n, const DivBy& b) { return (int)(n - div(n, b) * b.d); }

struct PackedArgs {
  const void* q;       // PARTS 1: bf16, 2: the hi parts, 3: fp32
  const uint16_t* ql;  // PARTS 2: the lo parts
  const uint16_t *k, *v;
  void* out;           // PARTS 1: bf16 [rows][heads][128], 2: fragments, 3: fp32 [rows][heads][128]
  uint16_t* out_lo;    // PARTS 2: attn_out's `ol`
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // elements
  int64_t kv_seq;      // PARTS 2: elements between the sequences' caches
  DivBy by_hkv, by_g;
  int hkv, g, nseq, frag;
  int alone;  // sequences whose blocks come one sequence after another, before the others' in turn
  // the launch's sequences, longest first: see the kernel's order of blocks; first row, length, number
  int32_t first[PSEQ], row[PSEQ], len[PSEQ], seq[PSEQ];
};

__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// v as the sum of PARTS bf16 numbers, each the rounding of what the ones before it leave
template <int PARTS>
__device__ __forceinline__ void split_parts(const float (&v)[8], uint4 (&p)[PARTS]) {
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

// top bits of the two halves set where that bf16 is an infinity or NaN
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t finite_or_0(uint32_t w) {
  const uint32_t n = nonfinite2(w) >> 15;
  return w & ~(n * 0xFFFFu);
}

// Staged rows are padded so that fragment reads do not meet in a bank and every address is one base and
// an immediate: K by 16 bytes (16 lanes on 16 rows at one 16-byte chunk), V by 64 (a half wave of a
// transposed read takes 64 bytes of each of 4 rows).
constexpr int PKS = 2 * D + 16, PVS = 2 * D + 64;

template <int PK, int RG, int KS>
struct PackedSmem {
  struct Tiles {
    unsigned char k[2][PK * PKS];
    unsigned char v[2][PK * PVS];
  };
  union {
    Tiles tiles[KS];
    struct {  // the output blocks that a key group leaves to another, the maxima and sums, lane by lane
      float acc[KS > 1 ? KS : 1][KS > 1 ? RG : 1][KS == 4 ? 16 : 16 - 16 / KS + (KS == 1)][64][4];
      float m[KS][RG][64], l[KS][RG][64];
    } join;
  };
  int bad[KS * RG];  // per staging wave: an infinity or NaN taken out of a tile's values
};

// PK: keys per tile; RG: waves on different rows, 32 each; KS: groups of RG waves on different tiles
template <int PARTS, int PK, int RG, int KS>
__global__ void __launch_bounds__(64 * RG * KS, RG == 1 ? 1 : 2) packed_attention_kernel(const PackedArgs a) {
  constexpr int PR = 32 * RG;                      // rows per workgroup
  constexpr int PH = PK / 32, NX = PK / (4 * RG);  // 32-key halves of a tile, chunks of K that a lane stages
  __shared__ __attribute__((aligned(16))) PackedSmem<PK, RG, KS> sm;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = wave % RG, ks = wave / RG;   // key group ks takes tiles ks, KS + ks, ...
  const int col = lane & 31, g = lane >> 5;  // this lane's query and half of the K slots
  auto& tiles = sm.tiles[ks];
  // workgroup b: K/V head b % hkv (with 8 heads, a head's keys stay in one XCD's L2), query block b / hkv of
  // the launch's. The blocks of the first `alone` sequences come one sequence after another, the last block (the
  // most keys) first. The others' go by their number in their sequence, the highest first: with the sequences'
  // block counts n_0 >= n_1 >= ..., those above n_1 are sequence 0's, the next down to n_2 sequence 0's and 1's in
  // turn, and so on. first[i] blocks come before sequence i's, or before those of it and the ones in turn with it.
  // The tables are read whole, a lane an entry, and picked from with lane reads: arguments are far away, and
  // one round trip there costs as much as a tile.
  int tf[PSEQ / 64], tl[PSEQ / 64], tr[PSEQ / 64], ts[PSEQ / 64];
#pragma unroll
  for (int o = 0; o < PSEQ / 64; ++o) {
    tf[o] = a.first[64 * o + lane];
    tl[o] = a.len[64 * o + lane];
    tr[o] = a.row[64 * o + lane];
    ts[o] = PARTS == 2 ? a.seq[64 * o + lane] : 0;
  }
  asm volatile("" ::"s"(a.q), "s"(a.k), "s"(a.v), "s"(a.q_row), "s"(a.q_head), "s"(a.k_row), "s"(a.k_head),
               "s"(a.v_row), "s"(a.v_head), "s"(a.by_hkv.d), "s"(a.by_hkv.mul),
               "s"(a.by_hkv.shift), "s"(a.by_g.mul), "s"(a.by_g.shift), "s"(a.g), "s"(a.nseq),
               "s"(a.alone));  // the other arguments, all in the same trip
  auto pick = [&](const int (&t)[PSEQ / 64], int n) {
    int v = t[0];
#pragma unroll
    for (int o = 1; o < PSEQ / 64; ++o) v = n >= 64 * o ? t[o] : v;
    return __builtin_amdgcn_readlane(v, n & 63);
  };
  const int kh = mod(blockIdx.x, a.by_hkv), item = div(blockIdx.x, a.by_hkv);
  int pi = -1;
#pragma unroll
  for (int o = 0; o < PSEQ / 64; ++o)
    pi += __popcll(__builtin_amdgcn_ballot_w64(64 * o + lane < a.nseq && tf[o] <= item));
  const int at = item - pick(tf, pi), m = pi < a.alone ? 1 : pi - a.alone + 1;  // sequences in turn
  const int turn = m == 1 ? at : at / m, si = pi < a.alone ? pi : a.alone + at - turn * m;
  const int qb = (pick(tl, pi) * a.g + PR - 1) / PR - 1 - turn;
  const int len = pick(tl, si), row0 = pick(tr, si), rows = len * a.g;
  const int r0 = qb * PR + 32 * w, r = r0 + col;          // this wave's first row, this lane's row
  const int rc = min(r, rows - 1), tok = div(rc, a.by_g), hq = kh * a.g + (rc - tok * a.g);
  const int first = div(qb * PR, a.by_g), last = div(min(rows, (qb + 1) * PR) - 1, a.by_g);  // the block's tokens
  const int wfirst = div(r0, a.by_g), wlast = r0 < rows ? div(min(rows, r0 + 32) - 1, a.by_g) : -1;  // the wave's
  const int ntile = last / PK + 1, niter = (ntile + KS - 1) / KS;
  auto tile = [&](int i) { return KS * i + ks; };
  // its first key and value row: in the sequence's cache, or packed as the queries are
  const char* kbase = (const char*)(a.k + (PARTS == 2 ? pick(ts, si) * a.kv_seq : row0 * a.k_row) + kh * a.k_head);
  const char* vbase = (const char*)(a.v + (PARTS == 2 ? pick(ts, si) * a.kv_seq : row0 * a.v_row) + kh * a.v_head);

  // a key group's wave w stages rows PK / RG w .. of its tile, four to an instruction (lane l: chunk l % 16 of row
  // l / 16), through registers, where a later tile waits while this one is multiplied. Keys past the
  // block's last one are that one again (masked).
  const int srow = PK / RG * w + (lane >> 4), chunk = lane & 15;
  struct Tile {
    uint4 x[NX];
  };
  // Uniform bases, the lane's row on them as 32 bits. No branch, or the compiler waits for what is in flight where
  // its two sides meet.
  auto load = [&](Tile& d, const char* base, int64_t row, int i) __attribute__((always_inline)) {
    const int key = min(tile(i) * PK, last);
    const uint32_t rb = 2 * (uint32_t)row, o = srow * rb + 16 * chunk;
    const uint32_t end = min(last - key, PK - 1) * rb + 16 * chunk;
#pragma unroll
    for (int n = 0; n < NX; ++n)
      d.x[n] = ld_global16(reinterpret_cast<const uint4*>(base + key * (2 * row) + min(o + 4 * n * rb, end)));
  };
  // the same where the block has all of the tile's keys
  auto load_whole = [&](Tile& d, const char* base, int64_t row, int i) __attribute__((always_inline)) {
    const uint32_t o = srow * (2 * (uint32_t)row) + 16 * chunk;
#pragma unroll
    for (int n = 0; n < NX; ++n)
      d.x[n] = ld_global16(reinterpret_cast<const uint4*>(base + (tile(i) * PK + 4 * n) * (2 * row) + o));
  };
  auto store_k = [&](const Tile& d, int i) __attribute__((always_inline)) {
    unsigned char* p = tiles.k[i & 1] + srow * PKS + 16 * chunk;
#pragma unroll
    for (int n = 0; n < NX; ++n) *reinterpret_cast<uint4*>(p + 4 * n * PKS) = d.x[n];
  };
  auto store_v = [&](Tile& d, int i, bool whole = false) __attribute__((always_inline)) {
    // a tile that some query of the block sees in part, or that is multiplied by parts: finite values only
    if (PARTS > 1 || (!whole && tile(i) * PK + PK - 1 > first)) {
      uint32_t bad = 0;
#pragma unroll
      for (int n = 0; n < NX; ++n)
        bad |= nonfinite2(d.x[n].x) | nonfinite2(d.x[n].y) | nonfinite2(d.x[n].z) | nonfinite2(d.x[n].w);
      if (bad) {
        sm.bad[wave] = 1;
#pragma unroll
        for (int n = 0; n < NX; ++n)
          d.x[n] = make_uint4(finite_or_0(d.x[n].x), finite_or_0(d.x[n].y), finite_or_0(d.x[n].z),
                              finite_or_0(d.x[n].w));
      }
    }
    unsigned char* p = tiles.v[i & 1] + srow * PVS + 16 * chunk;
#pragma unroll
    for (int n = 0; n < NX; ++n) *reinterpret_cast<uint4*>(p + 4 * n * PVS) = d.x[n];
  };
  // The queries: a row's 256 bytes (or 2 times 256) by 16 lanes, and through LDS to the lanes whose B operand they
  // are. (Read by those directly, 16 bytes of 32 rows to an instruction, their addresses took longer than a tile.)
  // The key groups of a row group share the reading.
  constexpr int QP = PARTS == 1 ? 1 : 2;  // 256-byte pieces: hi and lo, or half a row of fp32 each
  const int qrow = 32 / KS * ks + (lane >> 4);  // among the wave's 32, and 4, 8 .. after it
  uint4 qx[QP][8 / KS];
  const int64_t qo = ((int64_t)(row0 + tok) * a.q_row + hq * a.q_head) * (PARTS == 3 ? 4 : 2);  // row `col`, bytes
#pragma unroll
  for (int n = 0; n < 8 / KS; ++n) {
    const int64_t o = (int64_t)((uint64_t)(uint32_t)__shfl((int)(qo >> 32), qrow + 4 * n) << 32 |
                                (uint32_t)__shfl((int)qo, qrow + 4 * n));
#pragma unroll
    for (int p = 0; p < QP; ++p)
      qx[p][n] = ld_global16(reinterpret_cast<const uint4*>((const char*)(PARTS == 2 && p ? a.ql : a.q) + o +
                                                            (PARTS == 3 ? 256 * p : 0) + 16 * chunk));
  }
  uint4 fq[PARTS][8];  // dims 16 s + 8 g .. +7 of row `col`
  Tile x;  // on the way to LDS: V of the next tile, then K of the one after it
  Tile v0;
  {
    Tile k0;  // (of a tile that the block does not have: its last key)
    load(k0, kbase, a.k_row, 0);
    load(v0, vbase, a.v_row, 0);
    if (lane == 0) sm.bad[wave] = 0;
    unsigned char* qs = reinterpret_cast<unsigned char*>(&sm.tiles);
    static_assert(sizeof(sm.tiles) >= PR * PKS);
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      if (p) __syncthreads();
#pragma unroll
      for (int n = 0; n < 8 / KS; ++n)
        *reinterpret_cast<uint4*>(qs + (32 * w + qrow + 4 * n) * PKS + 16 * chunk) = qx[p][n];
      __syncthreads();
      const unsigned char* row = qs + (32 * w + col) * PKS;
      if constexpr (PARTS == 3) {
#pragma unroll
        for (int s = 4 * p; s < 4 * p + 4; ++s) {
          const float4 x = *reinterpret_cast<const float4*>(row + 64 * (s & 3) + 32 * g);
          const float4 y = *reinterpret_cast<const float4*>(row + 64 * (s & 3) + 32 * g + 16);
          const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          uint4 part[PARTS];
          split_parts<PARTS>(f, part);
#pragma unroll
          for (int i = 0; i < PARTS; ++i) fq[i][s] = part[i];
        }
      } else {
#pragma unroll
        for (int s = 0; s < 8; ++s) fq[p][s] = *reinterpret_cast<const uint4*>(row + 32 * s + 16 * g);
      }
    }
    __syncthreads();
    store_k(k0, 0);
  }

  f32x16 acc[4];  // dims 32 b + 8 (j / 4) + 4 g + j % 4 of query `col`
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  // running maximum of the raw scores, the number that the exponents refer to (in their scale), this lane's half of
  // the sum
  float mrun = -INFINITY, mscaled = 0.f, lrun = 0.f;
  constexpr float C = ATT_SCALE * 1.4426950408889634f;

  // raw scores of the group's tile i
  typedef f32x16 Scores[PH];
  auto scores = [&](Scores& st, int i) __attribute__((always_inline)) {
    const unsigned char* kt = tiles.k[i & 1] + col * PKS + 16 * g;  // K row `col` at dims 8 g
#pragma unroll
    for (int h = 0; h < PH; ++h) st[h] = f32x16{};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint4 fk[PH];
#pragma unroll
      for (int h = 0; h < PH; ++h) fk[h] = *reinterpret_cast<const uint4*>(kt + 32 * h * PKS + 32 * s);
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int h = 0; h < PH; ++h) st[h] = mfma32(fk[h], fq[p][s], st[h]);
    }
  };
  // its mask, if some query of the wave sees it in part
  auto mask = [&](Scores& st, int i) __attribute__((always_inline)) {
    const int key = tile(i) * PK;
    if (key + PK - 1 > wfirst) {
#pragma unroll
      for (int h = 0; h < PH; ++h)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (key + 32 * h + 8 * (j >> 2) + 4 * g + (j & 3) > tok) st[h][j] = -INFINITY;
    }
  };
  // the running maximum with it
  float mnew = -INFINITY;
  auto maximum = [&](const Scores& st) __attribute__((always_inline)) {
    mnew = mrun;
#pragma unroll
    for (int h = 0; h < PH; ++h)
#pragma unroll
      for (int j = 0; j < 16; ++j) mnew = fmaxf(mnew, st[h][j]);
    mnew = xmax32(mnew);
  };
  // The output and the sum to a new reference, where the maximum has left the old one 2^8 behind: until then the
  // weights are up to 2^8 instead of 1, as exact in bf16 and fp32, and the 64 products (which some query of a wave
  // asks for in most tiles if each new maximum does) are saved: 8,192 + 4,096 + 1,801 tokens 375 -> 362 us, 3,584
  // fp32 tokens 148 -> 141.
  auto rescale = [&]() __attribute__((always_inline)) {
    const float mc = mnew * C;
    const bool first = mrun == -INFINITY;  // a query that has seen no key of weight so far
    const float ref = first ? (mnew == -INFINITY ? 0.f : mc) : mc > mscaled + 8.f ? mc : mscaled;
    mrun = mnew;
    if (__builtin_amdgcn_ballot_w64(ref != mscaled) != 0) {
      // exactly 1 where the reference holds; of what has no weight so far (and a first maximum far below 0 would
      // make of 0 times infinity) too
      const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(mscaled - ref);
      mscaled = ref;
      lrun *= alpha;
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] *= alpha;
    }
  };
  // half a tile's weights, in place of its scores, and their sum (of the rounded ones, where they are)
  auto weights = [&](f32x16& st) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 16; ++j) st[j] = __builtin_amdgcn_exp2f(fmaf(st[j], C, -mscaled));
    float sum = 0.f;
    if constexpr (PARTS == 1) {
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const bf16x2_t p = {(__bf16)st[j], (__bf16)st[j + 1]}, one = {(__bf16)1.f, (__bf16)1.f};
        sum = __builtin_amdgcn_fdot2_f32_bf16(p, one, sum, false);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) sum += st[j];
    }
    lrun += sum;
  };
  // O^T += V^T . P^T over keys 32 h .. 32 h + 31 of the tile
  auto output = [&](const f32x16& st, int i, int h) __attribute__((always_inline)) {
    // this lane's places: V row 4 g + l % 16 / 4 at dims 16 (l / 16 % 2) + 4 (l % 4)
    const unsigned char* vt =
        tiles.v[i & 1] + (4 * g + ((lane & 15) >> 2)) * PVS + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float pw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) pw[j] = st[8 * u + j];
      uint4 fp[PARTS];
      split_parts<PARTS>(pw, fp);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint2 x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          x[e] = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                         vt + (32 * h + 16 * u + 8 * e) * PVS + 64 * b)));
        const uint4 fv = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) acc[b] = mfma32(fv, fp[p], acc[b]);
      }
    }
  };

  // Tile i's weights are taken while the matrix cores make tile i + 1's scores. A place in LDS is written in
  // the step after the one that read it last (tile i + 1's V takes tile i - 1's, tile i + 2's K tile i's), so
  // one barrier a step is enough.
  Scores st, sn;
  Tile k1;
  const bool more = tile(1) < ntile;
  if (more) {
    load(k1, kbase, a.k_row, 1);
    load(x, vbase, a.v_row, 1);
  }
  __syncthreads();
  if (tile(0) * PK <= wlast) {
    scores(st, 0);
    mask(st, 0);
    maximum(st);
    mrun = mnew;  // what the first tile's rescaling would come to
    mscaled = mnew == -INFINITY ? 0.f : mnew * C;
  }
  store_v(v0, 0);
  if (more) store_k(k1, 1);
  __syncthreads();  // tile 0's scores made by every wave: tile 2's K takes its place in the first step
  int i = 0;
  // tiles whose next one the whole block sees, two before the last: no masks, no ends
  auto step = [&](Scores& st, Scores& sn, int i) __attribute__((always_inline)) {
    store_v(x, i + 1, true);
    load_whole(x, kbase, a.k_row, i + 2);
    rescale();
    scores(sn, i + 1);
#pragma unroll
    for (int h = 0; h < PH; ++h) weights(st[h]);
#pragma unroll
    for (int h = 0; h < PH; ++h) output(st[h], i, h);
    maximum(sn);
    store_k(x, i + 2);
    load_whole(x, vbase, a.v_row, i + 2);
    __syncthreads();
  };
  for (const int nfast = min((first + 1) / (PK * KS) - 1, (last + 1) / (PK * KS) - 2); i + 1 < nfast; i += 2) {
    step(st, sn, i);
    step(sn, st, i + 1);
  }
  for (; i < niter; ++i) {
    const bool next = tile(i + 1) < ntile, after = tile(i + 2) < ntile, seen = tile(i) * PK <= wlast;
    if (next) store_v(x, i + 1);
    if (after) load(x, kbase, a.k_row, i + 2);
    if (seen) {
      rescale();
      if (next) scores(sn, i + 1);
#pragma unroll
      for (int h = 0; h < PH; ++h) weights(st[h]);
    }
    if (after) {
      store_k(x, i + 2);
      load(x, vbase, a.v_row, i + 2);
    }
    if (seen) {
#pragma unroll
      for (int h = 0; h < PH; ++h) output(st[h], i, h);
    }
    if (seen && next) {
      mask(sn, i + 1);
      maximum(sn);
#pragma unroll
      for (int h = 0; h < PH; ++h) st[h] = sn[h];
    }
    __syncthreads();
  }
  // Each key group finishes 4 / KS of the four output blocks: it leaves its sums of the others in LDS, and
  // takes the other groups' of its own. (Of four groups each leaves all: picking its own among the registers is
  // more code, which a small grid's CUs fetch for the first time: 32 tokens 6.05 -> 5.80 us, 512 in fp32 16.3 -> 15.6.)
  constexpr int NB = 4 / KS;
  const int b0 = NB * ks;
  f32x16 out[NB];
  if constexpr (KS > 1) {
    int n = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (KS == 2 && b / NB == ks) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(sm.join.acc[ks][w][n + j][lane]) =
            make_float4(acc[b][4 * j], acc[b][4 * j + 1], acc[b][4 * j + 2], acc[b][4 * j + 3]);
      n += 4;
    }
    const float me = mrun == -INFINITY ? -INFINITY : mscaled;  // the exponents' scale that the sums refer to
    sm.join.m[ks][w][lane] = me;
    sm.join.l[ks][w][lane] = lrun;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (KS == 2) out[b] = ks ? acc[NB + b] : acc[b];
      else out[b] = f32x16{};
    }
    __syncthreads();
    float mc = me;
#pragma unroll
    for (int o = 0; o < KS; ++o) mc = fmaxf(mc, sm.join.m[o][w][lane]);
    if (mc == -INFINITY) mc = 0.f;
    const float own = KS == 2 ? __builtin_amdgcn_exp2f(me - mc) : 0.f;  // 0 for a group that saw no key
    lrun *= own;
#pragma unroll
    for (int b = 0; b < NB; ++b) out[b] *= own;
#pragma unroll
    for (int o = 0; o < KS; ++o) {
      if (KS == 2 && o == ks) continue;
      const float f = __builtin_amdgcn_exp2f(sm.join.m[o][w][lane] - mc);
      lrun = fmaf(f, sm.join.l[o][w][lane], lrun);
      const int n = 4 * (b0 - (KS == 2 && ks > o ? NB : 0));  // this group's first block among those that group o left
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(sm.join.acc[o][w][n + 4 * b + j][lane]);
          const float t[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) out[b][4 * j + e] = fmaf(f, t[e], out[b][4 * j + e]);
        }
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) out[b] = acc[b];
  }
  if constexpr (KS > 1) __syncthreads();  // what the groups left is read: its place takes the output rows
  if (r0 >= rows) return;
  float sum = xsum32(lrun);
  if constexpr (PARTS > 1) {
    // A query's part may be 0, or of the other sign, where the query is not (or an infinity, for one beyond bf16's
    // range), so on an infinite key component the parts' products are NaN where the query's is an infinity. Such a
    // score has made its row's sum NaN: these rows are made again from whole queries, key after key in fp32
    // (8,192 tokens with such a key in every row 16.5 ms, without 0.80).
    const bool again = sum != sum;
    if (__builtin_amdgcn_ballot_w64(again) != 0) {
      int c = col;
      asm volatile("" : "+v"(c));  // the query's place found again: kept, it would take registers of the loop above
      const int rq = min(r0 + c, rows - 1), tq = div(rq, a.by_g);
      const int64_t qo =
          ((int64_t)(row0 + tq) * a.q_row + (kh * a.g + (rq - tq * a.g)) * a.q_head) * (PARTS == 3 ? 4 : 2);
      float m = -INFINITY, l = 0.f;
      if (again)
#pragma unroll
        for (int b = 0; b < NB; ++b) out[b] = f32x16{};
      float qf[64];  // dims 16 s + 8 g + e of the query at 8 s + e
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const char* qp = (const char*)a.q + qo + (PARTS == 3 ? 64 * s + 32 * g : 32 * s + 16 * g);
        const uint4 x = *reinterpret_cast<const uint4*>(qp);
        const uint4 y =
            *reinterpret_cast<const uint4*>(PARTS == 3 ? qp + 16 : (const char*)a.ql + (qp - (const char*)a.q));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (PARTS == 3) qf[8 * s + e] = __uint_as_float(e < 4 ? xw[e] : yw[e - 4]);
          else qf[8 * s + e] = (e & 1 ? bf16_hi(xw[e / 2]) : bf16_lo(xw[e / 2])) +
                               (e & 1 ? bf16_hi(yw[e / 2]) : bf16_lo(yw[e / 2]));
        }
      }
#pragma unroll 1
      for (int key = 0; key <= wlast; ++key) {
        if (__builtin_amdgcn_ballot_w64(again && l == l) == 0) break;  // a NaN query or key leaves nothing to find
        float dot[8] = {};  // by the lane's 64 dims of query and key, the other half's beside them
        const char* kr = kbase + key * (2 * a.k_row) + 16 * g;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const uint4 k = *reinterpret_cast<const uint4*>(kr + 32 * s);
          const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dot[e] = fmaf(qf[8 * s + e], e & 1 ? bf16_hi(kw[e / 2]) : bf16_lo(kw[e / 2]), dot[e]);
        }
        const float score =
            xsum32(((dot[0] + dot[1]) + (dot[2] + dot[3])) + ((dot[4] + dot[5]) + (dot[6] + dot[7]))) * C;
        const bool seen = again && key <= tok;
        const float mn = seen ? fmaxf(m, score) : m, ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref);
        const float wt = seen ? __builtin_amdgcn_exp2f(score - ref) : 0.f;
        m = mn;
        l = fmaf(l, alpha, wt);
        const char* vr = vbase + key * (2 * a.v_row) + 64 * b0 + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint2 v = *reinterpret_cast<const uint2*>(vr + 64 * b + 16 * q);
            const uint32_t f[2] = {finite_or_0(v.x), finite_or_0(v.y)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              out[b][4 * q + j] = fmaf(wt, j & 1 ? bf16_hi(f[j / 2]) : bf16_lo(f[j / 2]), out[b][4 * q + j] * alpha);
          }
      }
      if (again) sum = l;
    }
  }
  // Infinite and NaN values: those that a query sees are what it gets, however small their weights. They were left out
  // of the tiles, or (one part, tiles that every query of the block sees) have gone through the products, from which
  // an output that they enter never comes out finite.
  int bad = 0;
#pragma unroll
  for (int n = 0; n < KS * RG; ++n) bad |= sm.bad[n];
  if constexpr (PARTS == 1) {
    float zero = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) zero = fmaf(out[b][j], 0.f, zero);
    bad |= zero != zero;
  }
  if (__builtin_amdgcn_ballot_w64(bad && sum == sum) != 0) {
    f32x16 seen[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) seen[b] = f32x16{};
    // 32 rows at a time, four to an instruction; the rare one that holds some, dim by dim (8,192 tokens behind an
    // infinite value 0.60 ms, without 0.30; fp32 1.0 and 0.80)
    int l16 = lane;
    asm volatile("" : "+v"(l16));  // so that nothing of it is made before the loop above, and kept there
#pragma unroll 1
    for (int k0 = 0; k0 <= wlast; k0 += 32) {
      uint32_t hit[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int key = min(k0 + 4 * n + (l16 >> 4), wlast);
        const uint4 x = *reinterpret_cast<const uint4*>(vbase + key * (2 * a.v_row) + 16 * (l16 & 15));
        hit[n] = nonfinite2(x.x) | nonfinite2(x.y) | nonfinite2(x.z) | nonfinite2(x.w);
      }
#pragma unroll 1
      for (int n = 0; n < 8; ++n) {
        uint32_t h = hit[0];
#pragma unroll
        for (int o = 1; o < 8; ++o) h = n == o ? hit[o] : h;
        const u64 any = __builtin_amdgcn_ballot_w64(h != 0);
        if (any == 0) continue;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 4 * n + e;
          if ((any >> (16 * e) & 0xffff) == 0 || key > wlast) continue;
          const uint16_t* vr = reinterpret_cast<const uint16_t*>(vbase + key * (2 * a.v_row)) + 32 * b0 + 4 * g;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float f = bf16_to_f32(vr[32 * b + 8 * q + j]);
                if (key <= tok && !(fabsf(f) < INFINITY)) seen[b][4 * q + j] += f;
              }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) out[b][j] = bad && seen[b][j] != 0.f ? seen[b][j] : out[b][j];
  }

  // the output's columns are queries: 8 dims of one query per lane after a swap between the wave's halves
  const float inv = sum > 0.f ? 1.f / sum : __builtin_nanf("");  // no key of weight: NaN, as 0 / 0
  auto dims8 = [&](int b, int q, float (&o)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(out[b][4 * q + j] * inv),
                                                      __float_as_uint(out[b][4 * q + 4 + j] * inv), false, false);
      o[j] = __uint_as_float(x[0]);
      o[4 + j] = __uint_as_float(x[1]);
    }
  };
  if constexpr (PARTS == 2) {  // attn_out's two fragment orders (layers_kernel.hip)
    const int64_t m = row0 + tok;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        float o[8];
        dims8(b, q, o);
        if (r >= rows) continue;
        uint4 p[PARTS];
        split_parts<PARTS>(o, p);
        const int kk = hq * D + 32 * (b0 + b) + 8 * (q + g);
        uint16_t* hi = (uint16_t*)a.out;
        *reinterpret_cast<uint4*>(hi + (a.frag == 2 ? skf_off(m, kk, 0, HQ * D) : frag_off(m, kk, HQ * D))) = p[0];
        *reinterpret_cast<uint4*>(a.frag == 2 ? hi + skf_off(m, kk, 1, HQ * D)
                                              : a.out_lo + frag_off(m, kk, HQ * D)) = p[1];
      }
  } else {
    // Through the wave's own 32 padded rows of LDS, so that a store instruction writes whole lines, BB bytes of
    // a row at a time, past the L2s. Measured over one set of inputs again and again (some 5 us less than with inputs
    // that change from call to call, as the header's figures are) and before the later steps: 64 prompts 168 -> 158
    // us, 3,584 fp32 tokens 151 -> 148 (whole lines into the L2s 168 and 149, 32 bytes of 32 rows past them 192).
    constexpr int ES = PARTS == 1 ? 2 : 4, BB = 32 * NB * ES < 256 ? 32 * NB * ES : 256;
    constexpr int NP = BB / (32 * ES), LR = BB / 16;  // output blocks at a time, lanes to a row
    static_assert(sizeof(sm.tiles) >= KS * RG * 32 * (BB + 16));
    unsigned char* ob = reinterpret_cast<unsigned char*>(&sm.tiles) + wave * 32 * (BB + 16);
#pragma unroll
    for (int pass = 0; pass < NB / NP; ++pass) {
#pragma unroll
      for (int b = 0; b < NP; ++b)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          float o[8];
          dims8(NP * pass + b, q, o);
          unsigned char* p = ob + col * (BB + 16) + ES * (32 * b + 8 * (q + g));
          if constexpr (PARTS == 1) {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                                      pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
          } else {
            *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<float4*>(p + 16) = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
      wave_sync();
#pragma unroll
      for (int n = 0; n < LR / 2; ++n) {
        const int orow = 64 / LR * n + lane / LR, ro = r0 + orow;
        const u32x4 x = *reinterpret_cast<const u32x4*>(ob + orow * (BB + 16) + 16 * (lane % LR));
        if (ro < rows) {
          const int t = div(ro, a.by_g);
          const int64_t at = (int64_t)(row0 + t) * (a.hkv * a.g) + kh * a.g + (ro - t * a.g);
          unsigned char* p = (unsigned char*)a.out + ES * (at * D + 32 * (b0 + NP * pass)) + 16 * (lane % LR);
          __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
        }
      }
      wave_sync();
    }
  }
}

}  // namespace mkp

using namespace mkp;

// The launches of a call: the sequences longest first, at most PSEQ of them to a launch (a block costs its
// keys, so the long chains start first and short ones fill the CUs that finish).
template <int PARTS, int PK>
static hipError_t launch_packed(PackedArgs& a, const int32_t* lengths, int num_seqs, hipStream_t stream) {
  a.by_hkv = div_by(a.hkv);
  a.by_g = div_by(a.g);
  try {
    std::vector<int32_t> order(num_seqs), row(num_seqs);
    std::iota(order.begin(), order.end(), 0);
    for (int i = 0, at = 0; i < num_seqs; at += lengths[i++]) row[i] = at;
    std::stable_sort(order.begin(), order.end(), [&](int32_t x, int32_t y) { return lengths[x] > lengths[y]; });
    for (int s = 0; s < num_seqs && lengths[order[s]] > 0;) {
      int n = 0;
      for (; n < PSEQ && s < num_seqs && lengths[order[s]] > 0; ++n, ++s) {
        const int i = order[s];
        a.row[n] = row[i];
        a.len[n] = lengths[i];
        a.seq[n] = i;
      }
      a.nseq = n;
      // the workgroups of blocks of pr rows, and each sequence's place among them
      auto places = [&](int pr) {
        auto count = [&](int i) { return i < n ? ((int64_t)a.len[i] * a.g + pr - 1) / pr : 0; };
        // Blocks of one sequence after another find its keys in the L2s; blocks in turn, the longest first, end
        // together. So in turn are the last sequences, as many as keep the 512 workgroups that run at once busy
        // for as long as the longest block before them lasts (in units of the keys of one block). Measured on
        // MI355X over one set of inputs again and again, us with all in turn / so / none in turn: 64 prompts of 64 to
        // 960 tokens 158 / 148 / 148, of 512 136 / 125 / 132, 24 of 1,024 151 / 145 / 153, 8 of 2,048 162 / 163 / 179
        // (16 query heads on 8, bf16).
        int64_t blocks = 0, rest = 0;
        a.alone = 0;
        for (int i = n - 1; i > 0 && a.alone == 0 && pr == 128; --i) {
          rest += count(i) * (count(i) + 1) / 2;
          if (rest * a.hkv >= 512 * count(i - 1)) a.alone = i;
        }
        for (int i = 0; i < n; ++i) {
          a.first[i] = (int32_t)blocks;
          blocks += i < a.alone ? count(i) : (count(i) - count(i + 1)) * (i - a.alone + 1);
        }
        return dim3((unsigned)(blocks * a.hkv));
      };
      // A causal grid lasts as long as its longest chain of keys, so where it leaves CUs idle the chains are shared
      // out among more waves: 32 rows to a workgroup and four key groups of one wave; 64 rows and four groups of
      // two, where one workgroup a CU takes all, or two in turn and chains are long; 64 rows and two groups, two
      // workgroups to a CU; 128 rows and two groups of four, two in turn on long chains; else 128 rows and one
      // group, two workgroups to a CU. Measured on MI355X (16 query heads on
      // 8), us. With 32 / 64 rows: bf16 256 tokens (128 workgroups of 32 rows) 9.0 / -, 400 (200) 11.6 / 10.5;
      // fp32 700 (352) 19.4 / 22.2, 800 (400) 23.7 / 24.0, 8 prompts of 100 (448) 15.0 / 11.2. With 64 rows / 128
      // and two groups: bf16 800 tokens (200 workgroups of 64 rows) 13.9 / 18.3, 1,500 (376) 21.5 / 28.2, 2,048
      // (512) 31.4 / 35.0, 2,500 (632) 48.5 / 43.5, 700 + 200 + 100 (264) 13.0 / 17.0; fp32 1,500 38.5 / 56.8, 2,048
      // 60 / 75. With 64 rows and four / two groups / 128 rows and two: bf16 3 of 600 (456) 16.8 / 14.4 / 15.8, 8 of
      // 256 (512) 13.8 / 9.7 / 10.8, 6 of 600 (912) 31 / 22.5 / 19.5 (one group); fp32 5 of 300 (400) 21.0 / 17.0 /
      // 18.8. With two / one key groups of 128 rows: bf16 3,584 tokens (448 workgroups) 67.6 / 83.3, 4 of 1,024
      // (512) 30.2 / 29.6, 8 of 512 (512) 21.8 / 18.5, 32 of 128 (512) 17.8 / 11.6; fp32 3,584 155 / 190, 5 of 768
      // (480) 48.9 / 50.7, 6 of 600 (480) 42.5 / 40.8, 32 of 128 27.2 / 20.8.
      // The first limit of fp32 goes by single prompts. On 257 to 384 workgroups of 32 rows it loses with chains below
      // about 300: 32 / 64 rows, fp32, 6 of 100 (336) 14.0 / 10.4, 16 of 48 (384) 14.0 / 9.7, 3 of 200 (312) 13.9 /
      // 12.2, 330 + 300 (320) 14.0 / 14.8, 700 (352) 18.5 / 21.3. The prefill's hi/lo instances go by fp32's limits.
      const int longest = a.len[0];
      dim3 grid = places(32);
      if (grid.x <= (PARTS > 1 ? 384 : 160)) {
        hipLaunchKernelGGL((packed_attention_kernel<PARTS, 32, 1, 4>), grid, dim3(256), 0, stream, a);
      } else if ((grid = places(64)).x <= (longest < 640 ? 256 : 512)) {
        hipLaunchKernelGGL((packed_attention_kernel<PARTS, 32, 2, 4>), grid, dim3(512), 0, stream, a);
      } else if (grid.x <= 512) {
        hipLaunchKernelGGL((packed_attention_kernel<PARTS, 32, 2, 2>), grid, dim3(256), 0, stream, a);
      } else if ((grid = places(128)).x <= 512 && longest >= (PARTS > 1 ? 768 : 1024)) {
        hipLaunchKernelGGL((packed_attention_kernel<PARTS, PK, 4, 2>), grid, dim3(512), 0, stream, a);
      } else {
        hipLaunchKernelGGL((packed_attention_kernel<PARTS, PK, 4, 1>), grid, dim3(256), 0, stream, a);
      }
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  } catch (const std::bad_alloc&) {
    return hipErrorOutOfMemory;
  }
  return hipSuccess;
}

hipError_t mkp_attention_prefill(const MkPackedPrefill& p, hipStream_t stream) {
  PackedArgs a{};
  a.q = p.qh;
  a.ql = p.ql;
  const int64_t layer = (int64_t)p.layer * HKV * p.max_seq * D;
  a.k = p.k_cache + layer;
  a.v = p.v_cache + layer;
  a.out = p.oh;
  a.out_lo = p.ol;
  a.q_row = HQ * D;
  a.q_head = D;
  a.k_row = a.v_row = D;
  a.k_head = a.v_head = (int64_t)p.max_seq * D;
  a.kv_seq = p.seq_stride;
  a.hkv = HKV;
  a.g = HQ / HKV;
  a.frag = p.frag;
  return launch_packed<2, 32>(a, p.lengths, p.num_seqs, stream);
}

extern "C" hipError_t mk_attention_packed(int q_heads, int kv_heads, const void* q, int64_t q_row_stride,
                                          int64_t q_head_stride, const void* k, int64_t k_row_stride,
                                          int64_t k_head_stride, const void* v, int64_t v_row_stride,
                                          int64_t v_head_stride, const int32_t* lengths, int num_seqs, int q_fp32,
                                          void* out, hipStream_t stream) {
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || num_seqs < 0 || (num_seqs > 0 && !lengths))
    return hipErrorInvalidValue;
  int64_t total = 0;
  for (int i = 0; i < num_seqs; ++i) {
    if (lengths[i] < 0) return hipErrorInvalidValue;
    total += lengths[i];
  }
  // rows of a K/V head and workgroups are counted in 32 bits
  if (total * q_heads > INT32_MAX - 255) return hipErrorInvalidValue;
  if (total == 0) return hipSuccess;
  if (!q || !k || !v || !out) return hipErrorInvalidValue;
  for (const void* p : {q, k, v, (const void*)out})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return hipErrorInvalidValue;
  const int unit = q_fp32 ? 4 : 8;  // elements of 16 bytes
  for (int64_t s : {q_row_stride, q_head_stride})
    if (s < 0 || s % unit != 0) return hipErrorInvalidValue;
  for (int64_t s : {k_row_stride, k_head_stride, v_row_stride, v_head_stride})
    if (s < 0 || s % 8 != 0) return hipErrorInvalidValue;
  if (std::max(k_row_stride, v_row_stride) > 1 << 24) return hipErrorInvalidValue;  // a tile's offsets are 32 bits
  PackedArgs a{};
  a.q = q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.out = out;
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.hkv = kv_heads;
  a.g = q_heads / kv_heads;
  return q_fp32 ? launch_packed<3, 32>(a, lengths, num_seqs, stream)
                : launch_packed<1, 64>(a, lengths, num_seqs, stream);
}
