// Causal attention of packed sequences on MI355X (gfx950): the prompts of several sequences, one after
// the other in one array of rows, each attending to itself alone.
//
//   out[t][h] = sum over j <= t of softmax_j(q[t][h] . k[j][h / G] / sqrt(128)) v[j][h / G]
//
// for every token t of every sequence, j over the same sequence's tokens, G query heads on each K/V head.
//
// Tiles. The G query heads of a K/V head share its keys, so a sequence's queries of one K/V head are
// taken as len * G rows, row r = (token r / G, head r % G), whatever G is. A workgroup takes 128
// consecutive rows, a wave 32 of them, and runs over the keys 64 at a time up to its last token's:
//   S^T = K . Q^T   (v_mfma_f32_32x32x16_bf16, keys as rows): lane l holds the scores of its one query
//                   l % 32 against keys 8 (j / 4) + 4 (l / 32) + j % 4, j = 0..15, of each 32-key half,
//                   so the running maximum takes registers and one lane swap, the sum registers alone;
//   O^T += V^T . P^T: the lane's own weights, rounded to bf16, are the B operand as they stand when the
//                   K slots of a 16-key step mean keys {4 g .. 4 g + 3, 8 + 4 g .. +3} (g = l / 32); the
//                   A operand is V read transposed from LDS (ds_read_b64_tr_b16) in the same order. The
//                   output's columns are the queries too: rescaling is one factor per lane.
// K and V tiles are staged through LDS, two deep.
//
// Rounding. Queries and weights are multiplied as PARTS bf16 numbers whose sum they are: 1 for bf16
// queries (a weight is then off by at most 2^-8 of itself, as the output is by its own rounding), 2 for
// the prefill's hi/lo pairs (2^-16), 3 for fp32 queries (2^-24). Scores, maximum, sum and output are fp32.
//
// A masked key weighs nothing, whatever its value row holds: a tile that some query sees in part is looked
// over for infinities and NaN, and where it has any they are added outside the matrix product to the
// queries that see them (0 times infinity would reach the others).
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
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int PK = 64;         // keys per tile
constexpr int PW = 4;          // waves per workgroup
constexpr int PR = 32 * PW;    // rows per workgroup
constexpr int PSEQ = 128;      // sequences per launch (their places travel as kernel arguments)

struct PackedArgs {
  const void* q;       // PARTS 1: bf16, 2: the hi parts, 3: fp32
  const uint16_t* ql;  // PARTS 2: the lo parts
  const uint16_t *k, *v;
  void* out;           // PARTS 1: bf16 [rows][heads][128], 2: fragments, 3: fp32 [rows][heads][128]
  uint16_t* out_lo;    // PARTS 2: attn_out's `ol`
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // elements
  int64_t kv_seq;      // PARTS 2: elements between the sequences' caches
  int hkv, g, nseq, frag;
  // the launch's sequences, longest first: query blocks before them, first row, length, number
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

struct PackedSmem {
  unsigned char k[2][PK * PKS];
  unsigned char v[2][PK * PVS];
  int bad[PW];  // per staging wave: an infinity or NaN in a value row of a tile seen in part
};

template <int PARTS>
__global__ void __launch_bounds__(64 * PW, 2) packed_attention_kernel(const PackedArgs a) {
  __shared__ __attribute__((aligned(16))) PackedSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;  // this lane's query and half of the K slots
  // workgroup b: K/V head b % hkv (with 8 heads, a head's keys stay in one XCD's L2), query block b / hkv of
  // the launch, a sequence's last block (the most keys) first
  const int kh = blockIdx.x % a.hkv, item = blockIdx.x / a.hkv;
  int si = -1;
#pragma unroll
  for (int o = 0; o < PSEQ; o += 64)
    si += __popcll(__builtin_amdgcn_ballot_w64(o + lane < a.nseq && a.first[o + lane] <= item));
  const int len = a.len[si], row0 = a.row[si], rows = len * a.g;
  const int qb = (rows + PR - 1) / PR - 1 - (item - a.first[si]);
  const int r0 = qb * PR + 32 * w, r = r0 + col;          // this wave's first row, this lane's row
  const int rc = min(r, rows - 1), tok = rc / a.g, hq = kh * a.g + rc % a.g;
  const int last = (min(rows, (qb + 1) * PR) - 1) / a.g;  // the block's last token
  const int wlast = r0 < rows ? (min(rows, r0 + 32) - 1) / a.g : -1;
  const int ntile = last / PK + 1;
  // its first key and value row: in the sequence's cache, or packed as the queries are
  const uint16_t* kbase = a.k + (PARTS == 2 ? a.seq[si] * a.kv_seq : row0 * a.k_row) + kh * a.k_head;
  const uint16_t* vbase = a.v + (PARTS == 2 ? a.seq[si] * a.kv_seq : row0 * a.v_row) + kh * a.v_head;

  // wave w stages rows 16 w .. 16 w + 15 of a tile, four to an instruction (lane l: chunk l % 16 of row
  // l / 16), through registers, where the next tile waits while this one is multiplied. Keys past the
  // block's last one are that one again (masked).
  const int srow = 16 * w + (lane >> 4), chunk = lane & 15;
  struct Tile {
    uint4 k[4], v[4];
  };
  auto load = [&](Tile& x, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // the tile's first row as a uniform base, the lane's as 32 bits on it
      const uint32_t key = min(srow + 4 * i, last - t * PK);
      x.k[i] = ld_global16(reinterpret_cast<const uint4*>(
          reinterpret_cast<const char*>(kbase + (int64_t)(t * PK) * a.k_row) + (key * (2 * (uint32_t)a.k_row) + 16 * chunk)));
      x.v[i] = ld_global16(reinterpret_cast<const uint4*>(
          reinterpret_cast<const char*>(vbase + (int64_t)(t * PK) * a.v_row) + (key * (2 * (uint32_t)a.v_row) + 16 * chunk)));
    }
  };
  const int first = qb * PR / a.g;  // the block's first token
  auto store = [&](const Tile& x, int t) __attribute__((always_inline)) {
    const int buf = t & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = srow + 4 * i;
      *reinterpret_cast<uint4*>(sm.k[buf] + rr * PKS + 16 * chunk) = x.k[i];
      *reinterpret_cast<uint4*>(sm.v[buf] + rr * PVS + 16 * chunk) = x.v[i];
    }
    if (t * PK + PK - 1 > first) {  // a tile that some query of the block sees in part
      uint32_t n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        n |= nonfinite2(x.v[i].x) | nonfinite2(x.v[i].y) | nonfinite2(x.v[i].z) | nonfinite2(x.v[i].w);
      if (n) sm.bad[w] = 1;
    }
  };
  if (lane == 0) sm.bad[w] = 0;
  Tile x;
  load(x, 0);

  // the queries as the B operand: dims 16 s + 8 g .. +7 of row `col`
  uint4 fq[PARTS][8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int64_t o = (int64_t)(row0 + tok) * a.q_row + hq * a.q_head + 16 * s + 8 * g;
    if constexpr (PARTS == 3) {
      const float4 x = *reinterpret_cast<const float4*>((const float*)a.q + o);
      const float4 y = *reinterpret_cast<const float4*>((const float*)a.q + o + 4);
      const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      uint4 p[PARTS];
      split_parts<PARTS>(f, p);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) fq[i][s] = p[i];
    } else {
      fq[0][s] = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + o);
      if constexpr (PARTS == 2) fq[1][s] = *reinterpret_cast<const uint4*>(a.ql + o);
    }
  }

  f32x16 acc[4];  // dims 32 b + 8 (j / 4) + 4 g + j % 4 of query `col`
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  // running maximum of the raw scores, the same in the exponents' scale (rounded once: the weights and the
  // later rescaling refer to one number), this lane's half of the sum
  float mrun = -INFINITY, mscaled = 0.f, lrun = 0.f;
  constexpr float C = ATT_SCALE * 1.4426950408889634f;

  // one tile into the running softmax and the output. MASKED: some query of the block sees it in part
  auto consume = [&](int t, auto MASKED) __attribute__((always_inline)) {
    constexpr bool masked = decltype(MASKED)::value;
    const int k0 = t * PK, buf = t & 1;
    // this lane's places in the tile: K row `col` at dims 8 g, V row 4 g + l % 16 / 4 at dims 16 (l / 16 % 2) + 4 (l % 4)
    const unsigned char* kt = sm.k[buf] + col * PKS + 16 * g;
    const unsigned char* vt = sm.v[buf] + (4 * g + ((lane & 15) >> 2)) * PVS + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    f32x16 st[2];
    st[0] = f32x16{};
    st[1] = f32x16{};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint4 fk[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        fk[h] = *reinterpret_cast<const uint4*>(kt + 32 * h * PKS + 32 * s);
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) st[h] = mfma32(fk[h], fq[p][s], st[h]);
    }
    if constexpr (masked) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (k0 + 32 * h + 8 * (j >> 2) + 4 * g + (j & 3) > tok) st[h][j] = -INFINITY;
    }
    float m = mrun;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 16; ++j) m = fmaxf(m, st[h][j]);
    m = xmax32(m);
    const float mc = m == -INFINITY ? 0.f : m * C;  // a query that has seen no key of weight so far
    const float alpha = __builtin_amdgcn_exp2f(mscaled - mc);  // exactly 1 when the maximum holds
    mrun = m;
    mscaled = mc;
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        st[h][j] = __builtin_amdgcn_exp2f(fmaf(st[h][j], C, -mc));
        sum += st[h][j];
      }
    lrun = fmaf(lrun, alpha, sum);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] *= alpha;
    }
    auto weigh = [&](auto BAD) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float pw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pw[j] = st[u >> 1][8 * (u & 1) + j];
        uint4 fp[PARTS];
        split_parts<PARTS>(pw, fp);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint2 h[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            h[e] = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                           vt + (16 * u + 8 * e) * PVS + 64 * b)));
          }
          uint4 fv = make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
          if constexpr (decltype(BAD)::value)
            fv = make_uint4(finite_or_0(fv.x), finite_or_0(fv.y), finite_or_0(fv.z), finite_or_0(fv.w));
#pragma unroll
          for (int p = 0; p < PARTS; ++p) acc[b] = mfma32(fv, fp[p], acc[b]);
        }
      }
    };
    if (!masked || !(sm.bad[0] | sm.bad[1] | sm.bad[2] | sm.bad[3])) {  // the same for every lane
      weigh(std::false_type{});
    } else {
      weigh(std::true_type{});
      for (int key = 0; key < PK; ++key) {
        if (k0 + key > tok) break;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint2 x = *reinterpret_cast<const uint2*>(sm.v[buf] + key * PVS + 64 * b + 16 * q + 8 * g);
            const float f[4] = {bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!(fabsf(f[j]) < INFINITY)) acc[b][4 * q + j] += f[j];
          }
      }
    }
  };

  store(x, 0);
  __syncthreads();
  // the tiles that every query of the block sees whole, then the others
  const int nfull = min((first + 1) / PK, ntile - 1);
  for (int t = 0; t < nfull; ++t) {
    load(x, t + 1);
    consume(t, std::false_type{});
    store(x, t + 1);
    __syncthreads();  // tile t consumed by every wave, tile t + 1 staged
  }
  for (int t = nfull; t < ntile; ++t) {
    if (t + 1 < ntile) load(x, t + 1);
    if (t * PK <= wlast) consume(t, std::true_type{});
    if (t + 1 < ntile) store(x, t + 1);
    __syncthreads();
  }
  if (r0 >= rows) return;

  // the output's columns are queries: 8 dims of one query per lane after a swap between the wave's halves
  const float inv = 1.f / xsum32(lrun);
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
      float o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[b][4 * q + j] * inv),
                                                        __float_as_uint(acc[b][4 * q + 4 + j] * inv), false, false);
        o[j] = __uint_as_float(x[0]);
        o[4 + j] = __uint_as_float(x[1]);
      }
      if (r >= rows) continue;
      const int d = 32 * b + 8 * (q + g);
      const int64_t m = row0 + tok;
      if constexpr (PARTS == 1) {
        *reinterpret_cast<uint4*>((uint16_t*)a.out + (m * (a.hkv * a.g) + hq) * D + d) =
            make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                       pack_bf16x2(o[6], o[7]));
      } else if constexpr (PARTS == 2) {  // attn_out's two fragment orders (layers_kernel.hip)
        uint4 p[PARTS];
        split_parts<PARTS>(o, p);
        const int64_t kk = hq * D + d;
        uint16_t* out = (uint16_t*)a.out;
        *reinterpret_cast<uint4*>(out + (a.frag == 2 ? skf_off(m, kk, 0, HQ * D) : frag_off(m, kk, HQ * D))) = p[0];
        *reinterpret_cast<uint4*>(a.frag == 2 ? out + skf_off(m, kk, 1, HQ * D)
                                              : a.out_lo + frag_off(m, kk, HQ * D)) = p[1];
      } else {
        float4* p = reinterpret_cast<float4*>((float*)a.out + (m * (a.hkv * a.g) + hq) * D + d);
        p[0] = make_float4(o[0], o[1], o[2], o[3]);
        p[1] = make_float4(o[4], o[5], o[6], o[7]);
      }
    }
}

}  // namespace mkp

using namespace mkp;

// The launches of a call: the sequences longest first (a block costs its keys, so the long chains start
// first and short ones fill the CUs that finish), at most PSEQ of them to a launch.
template <int PARTS>
static hipError_t launch_packed(PackedArgs& a, const int32_t* lengths, int num_seqs, hipStream_t stream) {
  try {
    std::vector<int32_t> order(num_seqs), row(num_seqs);
    std::iota(order.begin(), order.end(), 0);
    for (int i = 0, at = 0; i < num_seqs; at += lengths[i++]) row[i] = at;
    std::stable_sort(order.begin(), order.end(), [&](int32_t x, int32_t y) { return lengths[x] > lengths[y]; });
    for (int s = 0; s < num_seqs && lengths[order[s]] > 0;) {
      int blocks = 0, n = 0;
      for (; n < PSEQ && s < num_seqs && lengths[order[s]] > 0; ++n, ++s) {
        const int i = order[s];
        a.first[n] = blocks;
        a.row[n] = row[i];
        a.len[n] = lengths[i];
        a.seq[n] = i;
        blocks += (int)(((int64_t)lengths[i] * a.g + PR - 1) / PR);
      }
      a.nseq = n;
      hipLaunchKernelGGL((packed_attention_kernel<PARTS>), dim3((unsigned)blocks * a.hkv), dim3(64 * PW), 0, stream, a);
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
  return launch_packed<2>(a, p.lengths, p.num_seqs, stream);
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
  if (total * q_heads > INT32_MAX - 2 * PR + 1) return hipErrorInvalidValue;
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
  return q_fp32 ? launch_packed<3>(a, lengths, num_seqs, stream) : launch_packed<1>(a, lengths, num_seqs, stream);
}
