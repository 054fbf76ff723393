// Beam search beside the batched decode, on MI355X (gfx950): the selection of each group's next beams
// from the decode's logits, and the reordering of the beams' K/V caches that follows from it.
//
// Selection. Rows of one group (`beams` consecutive ones) compete: candidate (row r, token v) has
//   score[r] + logit[r][v] - log(sum over u of exp(logit[r][u])),
// a finished row the one candidate (eos, score[r]), and the group's `beams` best go on. Within a row the
// order of the candidates is that of the logits, so it needs no arithmetic:
//   beam_chunk_kernel  a workgroup takes 8,192 logits of a row, a wave 2,048, all in registers: the sum of
//                      exp(logit - reference) to 2^-22, and their `beams` best (logit, token) as 64-bit keys;
//   beam_pick_kernel   a workgroup per group: a wave joins a row's sums (64 bits) and keys, then the group's
//                      beams^2 row bests are ranked by their scores in 64 bits, which tell apart any two
//                      candidates of one row and, between rows, what the sums' 2^-22 resolve.
// Bound by the read of the logits where there are many rows (8 x 8 beams of a vocabulary of 151,936, 38.9 MB in all:
// 17.6 us, 14.0 and 4.5 of them in the two kernels; 16.1 with plain fp32 sums), by launches and round trips where there
// are few (4 beams 9.4 us). 2,048 logits to a wave: 32 registers hold them, and 64 rows make 4,864 waves, one round on the chip.
// Equal candidates: the lower row first, within a row the larger logit, then the lower token.
//
// Reordering. new[b][p] = old[parents[b]][p] for the rows p of [begin[b], end[b]): a thread takes one 16-byte
// piece of one row of all the group's caches, loads every changed beam's parent before it stores any, and
// nobody else touches that piece: any map of a group onto itself, in place, each byte moved once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "mk_device.h"
#include "mk_layers.h"
#include "../../include/megakernel_amd.h"

namespace mkp {

constexpr int BEAMS_MAX = 16;
constexpr int BL = 2048;                 // logits per wave of the first kernel
constexpr int BC = 4 * BL;               // and per workgroup: a chunk
constexpr int BV_MAX = 1 << 20;          // vocabulary: BV_MAX / BC heads per row in LDS
constexpr int PICK_WAVES = 8;

// Key of (logit, token): larger for the larger logit, then the lower token; 0 is no candidate (a NaN's
// key is never used: its row's sum is NaN too).
__device__ __forceinline__ uint32_t order_bits(float x) {  // unsigned order is the numbers'
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 beam_key(float x, int v) {
  return ((u64)order_bits(x) << 32) | (0xffffffffu - (uint32_t)v);
}
__device__ __forceinline__ float key_logit(u64 k) { return from_order_bits((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_token(u64 k) { return (int)(0xffffffffu - (uint32_t)k); }

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  v = fmaxf(v, dpp<0x140>(v));
  return xmax32(xmax16(v));
}
__device__ __forceinline__ u64 wave_max_key(u64 k) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 x = __shfl_xor(k, o);
    k = k > x ? k : x;
  }
  return k;
}

__device__ __forceinline__ double join64(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const u64 u = __builtin_bit_cast(u64, v);
  return join64(__float_as_uint(dpp<CTRL>(__uint_as_float((uint32_t)u))),
                __float_as_uint(dpp<CTRL>(__uint_as_float((uint32_t)(u >> 32)))));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  v += dpp64<0x140>(v);
  u64 u = __builtin_bit_cast(u64, v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  v = join64(lo[0], hi[0]) + join64(lo[1], hi[1]);
  u = __builtin_bit_cast(u64, v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  return join64(lo[0], hi[0]) + join64(lo[1], hi[1]);
}

// A sum that refers to R, for the higher reference M (mostly the same one); a sum without a reference is 0, or NaN.
__device__ __forceinline__ double to_reference(double R, double sum, double M) {
  return R == M || R == -INFINITY ? sum : sum * exp(R - M);
}

struct BeamArgs {
  const float* logits;  // [rows][row_stride]
  int64_t row_stride;
  const float* scores;
  const uint8_t* finished;
  int rows, vocab, beams, eos, chunks;
  u64* cand;     // [rows][chunks][beams]
  double2* stat;  // [rows][chunks]: a reference R and the sum of exp(logit - R); -infinity: no logit above that
  int32_t *tokens, *parents;
  float* out_scores;
  uint8_t* out_finished;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any element

__global__ void __launch_bounds__(256) beam_chunk_kernel(const BeamArgs a) {
  __shared__ u64 list[64];
  __shared__ double sref[4], ssum[4];
  __shared__ uint32_t sbits[4];
  __shared__ u64 sbest[4];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.y, W = a.beams;
  const int v0 = blockIdx.x * BC + w * BL + 4 * lane;  // this lane's logits: v0 + 256 j + q
  const float* x = a.logits + row * a.row_stride;
  float f[BL / 64];
  // all loads at once; whether the row has ended is known by the time they arrive
  const bool ended = a.eos >= 0 && a.finished[row];
#pragma unroll
  for (int j = 0; j < BL / 256; ++j) {
    const int v = v0 + 256 * j;
    if (v + 3 < a.vocab) {
      const f4u t = *reinterpret_cast<const f4u*>(x + v);
#pragma unroll
      for (int q = 0; q < 4; ++q) f[4 * j + q] = t[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) f[4 * j + q] = v + q < a.vocab ? x[v + q] : -INFINITY;
    }
  }
  if (ended) return;  // its one candidate needs no logits
  auto token = [&](int i) { return v0 + 256 * (i >> 2) + (i & 3); };
  float lmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < BL / 64; ++i) lmax = fmaxf(lmax, f[i]);
  // A threshold that at least W lanes' maxima reach, and few others: the upper half of the W-th largest
  // maximum's bits (in an order that is the numbers'), bit by bit. The highest of the four waves' serves all.
  const uint32_t u = order_bits(lmax);
  uint32_t bits = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t more = bits | (1u << b);
    if (__popcll(__builtin_amdgcn_ballot_w64(u >= more)) >= W) bits = more;
  }
  // The sum of exp(logit - R) to 2^-22 of itself, also where all terms' roundings point one way (thousands of equal
  // logits). R is the maximum's next multiple of 32 towards 0, so the difference is exact (a rounded one is of a term
  // at least e^16 below the maximum). The product with log2 e keeps what its rounding leaves, c, for a sum of its own:
  // exp(d) = exp2(p) (1 + c log 2). Terms are off by exp2's step, 2^-23, and by half a one where two are added in fp32;
  // all else is in 64 bits. (With plain fp32 a floor of 151,936 equal logits under peaks was off by 2^-20.)
  constexpr float L = 1.4426950408889634f, L2 = (float)(1.4426950408889634 - (double)L);  // log2 e
  const float m = wave_max(lmax), ref = m == -INFINITY ? 0.f : 32.f * truncf(m * (1.f / 32));
  double sum = 0;
  float rest = 0.f;
#pragma unroll
  for (int i = 0; i < BL / 64; i += 2) {
    float e[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // e^-136 is 0 in fp32; -infinity would make c NaN, NaN stays
      const float d = __builtin_elementwise_maximum(f[i + q] - ref, -136.f), p = d * L;
      const float c = fmaf(d, L2, fmaf(d, L, -p));
      e[q] = __builtin_amdgcn_exp2f(p);
      rest = fmaf(e[q], c, rest);
    }
    sum += e[0] + e[1];
  }
  sum = wave_sum64(fma((double)rest, 0.6931471805599453, sum));
  if (lane == 0) {
    sref[w] = m == -INFINITY ? -INFINITY : ref;
    ssum[w] = sum;
    sbits[w] = bits;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  bits = max(max(sbits[0], sbits[1]), max(sbits[2], sbits[3]));
  const float t = bits <= order_bits(-INFINITY) ? -INFINITY : from_order_bits(bits);
  uint32_t mine = 0;  // this lane's logits that reach it
#pragma unroll
  for (int i = 0; i < BL / 64; ++i)
    if (f[i] >= t) mine |= 1u << i;
  if (blockIdx.x * BC + (w + 1) * BL > a.vocab)
#pragma unroll
    for (int i = 0; i < BL / 64; ++i)
      if (token(i) >= a.vocab) mine &= ~(1u << i);
  while (mine) {
    const int v = token(__ffs(mine) - 1);
    mine &= mine - 1;
    const int at = atomicAdd(&count, 1);
    if (at >= 64) break;
    list[at] = beam_key(x[v], v);  // the logit again: cheaper than finding it among the registers
  }
  __syncthreads();
  const int64_t slot = (int64_t)row * a.chunks + blockIdx.x;
  u64* out = a.cand + slot * W;
  const int n = count;
  if (n <= 64) {  // a key's place is how many are larger
    if (w == 0) {
      const u64 key = lane < n ? list[lane] : 0;
      int place = 0;
      for (int i = 0; i < n; ++i) place += list[i] > key;
      if (lane < n && place < W) out[place] = key;
      if (lane >= n && lane < W) out[lane] = 0;  // fewer than W logits
    }
  } else {  // many equal logits: the largest key below the last one, W times
    u64 last = ~(u64)0;
    for (int k = 0; k < W; ++k) {
      u64 best = 0;
#pragma unroll 1
      for (int i = 0; i < BL / 64; ++i) {  // from memory: kept in registers, their keys would cost the others theirs
        const u64 key = token(i) < a.vocab ? beam_key(x[token(i)], token(i)) : 0;
        if (key < last && key > best) best = key;
      }
      best = wave_max_key(best);
      __syncthreads();
      if (lane == 0) sbest[w] = best;
      __syncthreads();
      last = max(max(sbest[0], sbest[1]), max(sbest[2], sbest[3]));
      if (tid == 0) out[k] = last;
    }
  }
  if (tid == 0) {
    const double R = fmax(fmax(sref[0], sref[1]), fmax(sref[2], sref[3]));
    double s = 0;
#pragma unroll
    for (int o = 0; o < 4; ++o) s += to_reference(sref[o], ssum[o], R);
    a.stat[slot] = make_double2(R, s);
  }
}

__global__ void __launch_bounds__(64 * PICK_WAVES) beam_pick_kernel(const BeamArgs a) {
  constexpr int NL = BV_MAX / BC / 64, NK = BEAMS_MAX * BEAMS_MAX / 64;  // chunks, and a group's candidates, per lane
  constexpr int KL = 4;
  __shared__ __attribute__((aligned(16))) u64 heads[PICK_WAVES][64 * NL];
  __shared__ __attribute__((aligned(16))) u64 near[PICK_WAVES][64 * NK];
  __shared__ u64 least[PICK_WAVES];
  __shared__ double score[64 * NK];  // NaN: no candidate
  __shared__ int token[64 * NK];
  __shared__ int state[BEAMS_MAX];  // 1: the row has failed, 2: it had ended
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int W = a.beams, W2 = W * W, first = blockIdx.x * W;
  for (int r = w; r < W; r += PICK_WAVES) {
    const int row = first + r;
    const int64_t s0 = (int64_t)row * a.chunks;
    // what the row needs, in one trip: the chunks' sums and best keys, NL to a lane, and its keys, KL to a lane (of
    // the few rows that have more, the others below); an ended row has none that mean anything
    double2 st[NL];
    u64 head[NL], own[KL];
    const int keys = a.chunks * W;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int i = 64 * n + lane;
      st[n] = make_double2(-INFINITY, 0);
      head[n] = 0;
      if (i < a.chunks) {
        st[n] = a.stat[s0 + i];
        head[n] = a.cand[(s0 + i) * W];
      }
    }
#pragma unroll
    for (int n = 0; n < KL; ++n) own[n] = 64 * n + lane < keys ? a.cand[s0 * W + 64 * n + lane] : 0;
    const double base = a.scores[row];
    const bool bad = !(base < INFINITY), ended = a.eos >= 0 && a.finished[row];  // bad: NaN or +infinity
    if (lane < W) score[r * W + lane] = __builtin_nan("");
    if (ended) {
      if (lane == 0) {
        score[r * W] = base;
        token[r * W] = a.eos;
        state[r] = 2 + bad;
      }
      continue;
    }
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      m = fmaxf(m, (float)st[n].x);
      heads[w][64 * n + lane] = head[n];
    }
    if (lane == 0) least[w] = 0;
    wave_sync();
    // The W-th best of the chunks' best keys: none but keys that reach it are among the row's W best. (No two keys
    // are the same but those of no logit, 0. A failed row's keys may be anything.)
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      if (64 * n >= a.chunks) break;
      int rank = 0;
#pragma unroll 2
      for (int j = 0; j < a.chunks; j += 4)  // places past the last chunk hold 0
#pragma unroll
        for (int q = 0; q < 4; ++q) rank += heads[w][j + q] > head[n];
      if (head[n] != 0 && rank == W - 1) least[w] = head[n];
    }
    // log of the row's sum
    m = wave_max(m);
    double sum = 0;
#pragma unroll
    for (int n = 0; n < NL; ++n) sum += to_reference(st[n].x, st[n].y, m);
    sum = wave_sum64(sum);
    const double lsum = log(sum);  // beside its reference: together they would lose it in a row of the lowest numbers
    if (lane == 0) state[r] = bad || sum != sum;
    wave_sync();
    // the keys that reach it: W at least (if there are as many), W a chunk of W chunks at most
    const u64 low = least[w];
    int n = 0;
    auto keep = [&](u64 key) {
      const u64 all = __builtin_amdgcn_ballot_w64(key != 0 && key >= low);
      const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
      if (key != 0 && key >= low && at < 64 * NK) near[w][at] = key;
      n += __popcll(all);
    };
#pragma unroll
    for (int i = 0; i < KL; ++i)
      if (64 * i < keys) keep(own[i]);
    for (int e = 64 * KL + lane; e - lane < keys; e += 64) keep(e < keys ? a.cand[s0 * W + e] : 0);
    n = min(n, 64 * NK);
    if (lane < 8 && n + lane < 64 * NK) near[w][n + lane] = 0;
    wave_sync();
    for (int e = lane; e < n; e += 64) {
      const u64 key = near[w][e];
      int place = 0;
      for (int j = 0; j < n; j += 8)
#pragma unroll
        for (int q = 0; q < 8; ++q) place += near[w][j + q] > key;
      if (place < W) {
        const float x = key_logit(key);
        score[r * W + place] = x == -INFINITY ? -INFINITY : base + (((double)x - m) - lsum);
        token[r * W + place] = key_token(key);
      }
    }
    wave_sync();  // the next row's keys take the same places
  }
  __syncthreads();
  const int mine = lane < W ? state[lane] : 0;
  const u64 over = __builtin_amdgcn_ballot_w64(mine & 2);
  const bool fail = __builtin_amdgcn_ballot_w64(mine & 1) != 0;
  if (fail) {  // every beam of the group shows it
    if (tid < W) {
      a.tokens[first + tid] = -1;
      a.parents[first + tid] = first + tid;
      a.out_scores[first + tid] = __builtin_nanf("");
      a.out_finished[first + tid] = over >> tid & 1;
    }
    return;
  }
  // The group's candidates by score, equal ones by row and place: eight lanes count for one candidate how many
  // come before it.
  for (int c0 = 0; c0 < W2; c0 += 64 * PICK_WAVES / 8) {
    const int c = c0 + tid / 8, cc = min(c, W2 - 1);
    const double s = score[cc];
    int before = 0;
#pragma unroll 4
    for (int e = tid & 7; e < W2; e += 8) before += score[e] > s || (score[e] == s && e < cc);
    before += __builtin_amdgcn_update_dpp(0, before, 0xB1, 0xf, 0xf, false);
    before += __builtin_amdgcn_update_dpp(0, before, 0x4E, 0xf, 0xf, false);
    before += __builtin_amdgcn_update_dpp(0, before, 0x141, 0xf, 0xf, false);
    if (c < W2 && s == s && before < W && (tid & 7) == 0) {
      const int at = first + before, r = c / W, t = token[c];
      a.tokens[at] = t;
      a.parents[at] = first + r;
      a.out_scores[at] = (float)s;
      a.out_finished[at] = a.eos >= 0 && (t == a.eos || (over >> r & 1));
    }
  }
}

struct ReorderArgs {
  uint16_t *k, *v;
  const int32_t *parents, *begin, *end;
  int beams, max_seq, slabs;  // slabs: (layer, head) pairs
  int64_t seq;                // elements of one sequence's cache
};

// Workgroup (x, g): steps x, x + gridDim.x, ... of group g; a step is 16 rows of one (cache, layer, head).
// Bound by memory. Measured on MI355X: 8 groups of 8 beams, 400 positions, half of the beams replaced (2.94 GB
// read and written) 570 us, 5.15 TB/s (a device copy: 5.04); 5 of 3, 301 positions (345 MB) 62.5 us, 5.5 TB/s. The
// non-temporal hint on the stores and 8,192 workgroups instead of the 2,048 that are resident are 627 -> 570 us; for
// one group (4 beams, 128 positions, 59 MB from the L2s and the memory-side cache, 10.5 us) more than 2,048
// find no steps: 12.3 us.
template <int W>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
  const int g0 = blockIdx.y * a.beams;
  int from[W], lo[W], hi[W], p0 = INT32_MAX, p1 = 0;
#pragma unroll
  for (int b = 0; b < W; ++b) {
    from[b] = 0;
    lo[b] = hi[b] = 0;
    if (b < a.beams) {
      const uint32_t p = (uint32_t)a.parents[g0 + b] - (uint32_t)g0;  // any entry outside the group is large
      if (p < (uint32_t)a.beams && p != (uint32_t)b) {
        from[b] = (int)p;
        lo[b] = max(a.begin[g0 + b], 0);
        hi[b] = min(a.end[g0 + b], a.max_seq);
        if (lo[b] < hi[b]) {
          p0 = min(p0, lo[b]);
          p1 = max(p1, hi[b]);
        }
      }
    }
  }
  if (p0 >= p1) return;
  const int chunks = (p1 - p0 + 15) / 16;
  const int steps = 2 * a.slabs * chunks;
  const int rr = threadIdx.x >> 4, e = 8 * (threadIdx.x & 15);
  for (int s = blockIdx.x; s < steps; s += gridDim.x) {
    const int slab = s / chunks, row = p0 + 16 * (s % chunks) + rr;
    uint16_t* base = (slab < a.slabs ? a.k : a.v) + g0 * a.seq +
                     ((int64_t)(slab < a.slabs ? slab : slab - a.slabs) * a.max_seq + row) * D + e;
    u32x4 x[W];
#pragma unroll
    for (int b = 0; b < W; ++b) {
      x[b] = u32x4{0, 0, 0, 0};
      if (row >= lo[b] && row < hi[b]) x[b] = *reinterpret_cast<const u32x4*>(base + from[b] * a.seq);
    }
#pragma unroll
    for (int b = 0; b < W; ++b)
      if (row >= lo[b] && row < hi[b]) __builtin_nontemporal_store(x[b], reinterpret_cast<u32x4*>(base + b * a.seq));
  }
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace mkp

using namespace mkp;

extern "C" size_t mk_beam_select_workspace_bytes(int rows, int vocab, int beams) {
  if (rows < 1 || vocab < 1 || vocab > BV_MAX || beams < 1 || beams > BEAMS_MAX) return 0;
  const size_t slots = (size_t)rows * ((vocab + BC - 1) / BC);
  return align256(slots * beams * sizeof(u64)) + align256(slots * sizeof(double2));
}

extern "C" hipError_t mk_beam_select(int rows, int vocab, int beams, const float* logits, int64_t row_stride,
                                     const float* scores, const uint8_t* finished, int eos, int32_t* tokens,
                                     int32_t* parents, float* out_scores, uint8_t* out_finished, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
  const size_t need = mk_beam_select_workspace_bytes(rows, vocab, beams);
  if (need == 0 || rows % beams != 0 || rows > 65535) return hipErrorInvalidValue;
  if (!logits || !scores || !finished || !tokens || !parents || !out_scores || !out_finished || !workspace)
    return hipErrorInvalidValue;
  if (row_stride < 0 || eos < -1 || eos >= vocab) return hipErrorInvalidValue;
  if (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return hipErrorInvalidValue;
  BeamArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.rows = rows;
  a.vocab = vocab;
  a.beams = beams;
  a.eos = eos;
  a.chunks = (vocab + BC - 1) / BC;
  a.cand = static_cast<u64*>(workspace);
  a.stat = reinterpret_cast<double2*>(static_cast<char*>(workspace) +
                                     align256((size_t)rows * a.chunks * beams * sizeof(u64)));
  a.tokens = tokens;
  a.parents = parents;
  a.out_scores = out_scores;
  a.out_finished = out_finished;
  hipLaunchKernelGGL(beam_chunk_kernel, dim3(a.chunks, rows), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(beam_pick_kernel, dim3(rows / beams), dim3(64 * PICK_WAVES), 0, stream, a);
  return hipGetLastError();
}

extern "C" hipError_t mk_beam_reorder(int num_layers, int rows, int beams, int max_seq_len, void* k_cache, void* v_cache,
                                      const int32_t* parents, const int32_t* begin, const int32_t* end,
                                      hipStream_t stream) {
  if (num_layers < 1 || max_seq_len < 1 || beams < 1 || beams > BEAMS_MAX || rows < 1 || rows % beams != 0 ||
      rows / beams > 65535)
    return hipErrorInvalidValue;
  if ((int64_t)num_layers * HKV * 2 * (((int64_t)max_seq_len + 15) / 16) > INT32_MAX - 8192)  // steps, counted in 32 bits
    return hipErrorInvalidValue;
  if (!k_cache || !v_cache || k_cache == v_cache || !parents || !begin || !end) return hipErrorInvalidValue;
  for (const void* p : {(const void*)k_cache, (const void*)v_cache})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return hipErrorInvalidValue;
  if (beams == 1) return hipSuccess;  // a lone beam is its own parent
  ReorderArgs a{};
  a.k = static_cast<uint16_t*>(k_cache);
  a.v = static_cast<uint16_t*>(v_cache);
  a.parents = parents;
  a.begin = begin;
  a.end = end;
  a.beams = beams;
  a.max_seq = max_seq_len;
  a.slabs = num_layers * HKV;
  a.seq = (int64_t)a.slabs * max_seq_len * D;
  const int groups = rows / beams, wgs = std::max(1, std::min(2048, 8192 / groups));
  const dim3 grid(std::min(wgs, 2 * a.slabs * ((max_seq_len + 15) / 16)), groups);
  if (beams <= 2) hipLaunchKernelGGL(beam_reorder_kernel<2>, grid, dim3(256), 0, stream, a);
  else if (beams <= 4) hipLaunchKernelGGL(beam_reorder_kernel<4>, grid, dim3(256), 0, stream, a);
  else if (beams <= 8) hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}
