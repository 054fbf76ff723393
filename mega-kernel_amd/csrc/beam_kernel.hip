// Beam search beside the batched decode, on MI355X (gfx950): the selection of each group's next beams
// from the decode's logits, and the reordering of the beams' K/V caches that follows from it.
//
// Selection. Rows of one group (`beams` consecutive ones) compete: candidate (row r, token v) has
//   score[r] + logit[r][v] - log(sum over u of exp(logit[r][u])),
// a finished row the one candidate (eos, score[r]), and the group's `beams` best go on. Within a row the
// order of the candidates is that of the logits, so it needs no arithmetic:
//   beam_chunk_kernel  a wave takes 2,048 logits of a row, all in registers: their maximum, the sum of
//                      exp(logit - maximum), and their `beams` best (logit, token) as 64-bit keys, best first;
//   beam_pick_kernel   a workgroup per group: a wave joins a row's sums (64 bits) and keys, then the group's
//                      beams^2 row bests are ranked by their scores in 64 bits, which tell apart any two
//                      candidates of one row and, between rows, what the fp32 sums resolve.
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
constexpr int BC = 2048;                 // logits per wave
constexpr int BV_MAX = 1 << 20;          // vocabulary: BV_MAX / BC heads per row in LDS
constexpr int PICK_WAVES = 8;

// Key of (logit, token): larger for the larger logit, then the lower token; 0 is no candidate (a NaN's
// key is never used: its row's sum is NaN too).
__device__ __forceinline__ u64 beam_key(float x, int v) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return ((u64)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32) | (0xffffffffu - (uint32_t)v);
}
__device__ __forceinline__ float key_logit(u64 k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
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

// LDS that one lane of a wave wrote and another reads
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct BeamArgs {
  const float* logits;  // [rows][row_stride]
  int64_t row_stride;
  const float* scores;
  const uint8_t* finished;
  int rows, vocab, beams, eos, chunks;
  u64* cand;     // [rows][chunks][beams]
  float2* stat;  // [rows][chunks]: maximum, sum of exp(logit - maximum)
  int32_t *tokens, *parents;
  float* out_scores;
  uint8_t* out_finished;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any element

__global__ void __launch_bounds__(256) beam_chunk_kernel(const BeamArgs a) {
  __shared__ u64 list[4][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x * 4 + w, row = blockIdx.y;
  if (chunk >= a.chunks) return;
  if (a.eos >= 0 && a.finished[row]) return;  // its one candidate needs no logits
  const float* x = a.logits + row * a.row_stride;
  const int v0 = chunk * BC + 4 * lane;  // this lane's logits: v0 + 256 j + q
  float f[BC / 64];
  if ((chunk + 1) * BC <= a.vocab) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const f4u t = *reinterpret_cast<const f4u*>(x + v0 + 256 * j);
#pragma unroll
      for (int q = 0; q < 4; ++q) f[4 * j + q] = t[q];
    }
  } else {
#pragma unroll
    for (int i = 0; i < BC / 64; ++i) {
      const int v = v0 + 256 * (i >> 2) + (i & 3);
      f[i] = v < a.vocab ? x[v] : -INFINITY;
    }
  }
  float lmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < BC / 64; ++i) lmax = fmaxf(lmax, f[i]);
  const float m = wave_max(lmax), mc = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < BC / 64; ++i) sum += __builtin_amdgcn_exp2f((f[i] - mc) * 1.4426950408889634f);
  sum = wave_sum(sum);
  const int64_t slot = (int64_t)row * a.chunks + chunk;
  if (lane == 0) a.stat[slot] = make_float2(m, sum);

  // The `beams`-th largest of the lanes' maxima: at least `beams` logits reach it, and few more.
  float t = m, left = lmax;
  for (int k = 0; k < a.beams; ++k) {
    t = wave_max(left);
    const u64 at = __builtin_amdgcn_ballot_w64(left == t);
    if (lane == (at ? __ffsll((unsigned long long)at) - 1 : -1)) left = -INFINITY;  // one of the lanes that hold it
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < BC / 64; ++i) {
    const int v = v0 + 256 * (i >> 2) + (i & 3);
    const bool in = f[i] >= t && v < a.vocab;
    const u64 all = __builtin_amdgcn_ballot_w64(in);
    if (all) {
      const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
      if (in && at < 64) list[w][at] = beam_key(f[i], v);
      n += __popcll(all);
    }
  }
  wave_sync();
  u64* out = a.cand + slot * a.beams;
  if (n <= 64) {  // the lane's place among them is how many are larger
    const u64 key = lane < n ? list[w][lane] : 0;
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += list[w][i] > key;
    if (lane < n && rank < a.beams) out[rank] = key;
    if (lane >= n && lane < a.beams) out[lane] = 0;
  } else {  // many equal logits: the largest key below the last one, `beams` times
    u64 last = ~(u64)0;
    for (int k = 0; k < a.beams; ++k) {
      u64 best = 0;
#pragma unroll
      for (int i = 0; i < BC / 64; ++i) {
        const int v = v0 + 256 * (i >> 2) + (i & 3);
        const u64 key = v < a.vocab ? beam_key(f[i], v) : 0;
        if (key < last && key > best) best = key;
      }
      last = wave_max_key(best);
      if (lane == 0) out[k] = last;
    }
  }
}

__global__ void __launch_bounds__(64 * PICK_WAVES) beam_pick_kernel(const BeamArgs a) {
  __shared__ u64 heads[PICK_WAVES][BV_MAX / BC];
  __shared__ u64 near[PICK_WAVES][BEAMS_MAX * BEAMS_MAX];
  __shared__ int sel[PICK_WAVES][BEAMS_MAX];
  __shared__ double score[BEAMS_MAX * BEAMS_MAX];
  __shared__ int token[BEAMS_MAX * BEAMS_MAX];  // -1: no candidate
  __shared__ int failed[BEAMS_MAX];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int W = a.beams, first = blockIdx.x * W;
  for (int r = w; r < W; r += PICK_WAVES) {
    const int row = first + r;
    const double base = a.scores[row];
    const bool bad = !(base < INFINITY);  // NaN or +infinity
    if (lane < W) token[r * W + lane] = -1;
    if (a.eos >= 0 && a.finished[row]) {
      if (lane == 0) {
        score[r * W] = base;
        token[r * W] = a.eos;
        failed[r] = bad;
      }
      continue;
    }
    const int64_t s0 = (int64_t)row * a.chunks;
    // log of the row's sum, in 64 bits over the chunks' sums
    float m = -INFINITY;
    for (int i = lane; i < a.chunks; i += 64) {
      m = fmaxf(m, a.stat[s0 + i].x);
      heads[w][i] = a.cand[(s0 + i) * W];
    }
    if (lane < W) sel[w][lane] = 0;  // a failed row may have fewer chunks with a key
    wave_sync();
    m = wave_max(m);
    double sum = 0;
    for (int i = lane; i < a.chunks; i += 64) {
      const float2 s = a.stat[s0 + i];
      sum += s.x == -INFINITY ? (double)s.y : (double)s.y * exp((double)s.x - (double)m);  // s.y: 0, or NaN
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    const double lse = (double)m + log(sum);
    if (lane == 0) failed[r] = bad || sum != sum;
    // the W chunks with the best first keys hold the row's W best keys
    for (int i = lane; i < a.chunks; i += 64) {
      const u64 key = heads[w][i];
      int rank = 0;
      for (int j = 0; j < a.chunks; ++j) rank += heads[w][j] > key;
      if (rank < W) sel[w][rank] = i;  // keys differ, but for the empty ones: a chunk always has a candidate
    }
    wave_sync();
    const int nsel = min(W, a.chunks);
    for (int e = lane; e < nsel * W; e += 64) near[w][e] = a.cand[(s0 + sel[w][e / W]) * W + e % W];
    wave_sync();
    for (int e = lane; e < nsel * W; e += 64) {
      const u64 key = near[w][e];
      if (key == 0) continue;
      int rank = 0;
      for (int j = 0; j < nsel * W; ++j) rank += near[w][j] > key;
      if (rank < W) {
        const float x = key_logit(key);
        score[r * W + rank] = x == -INFINITY ? -INFINITY : base + ((double)x - lse);
        token[r * W + rank] = key_token(key);
      }
    }
    wave_sync();  // the next row's keys take the same places
  }
  __syncthreads();
  bool fail = false;
  for (int r = 0; r < W; ++r) fail |= failed[r] != 0;
  if (tid >= W * W) return;
  const int r = tid / W;
  if (fail) {  // every beam of the group shows it
    if (tid % W == 0) {
      a.tokens[first + r] = -1;
      a.parents[first + r] = first + r;
      a.out_scores[first + r] = __builtin_nanf("");
      a.out_finished[first + r] = a.eos >= 0 ? a.finished[first + r] : 0;
    }
    return;
  }
  if (token[tid] < 0) return;
  const double s = score[tid];
  int rank = 0;
  for (int j = 0; j < W * W; ++j) rank += token[j] >= 0 && (score[j] > s || (score[j] == s && j < tid));
  if (rank < W) {
    a.tokens[first + rank] = token[tid];
    a.parents[first + rank] = first + r;
    a.out_scores[first + rank] = (float)s;
    a.out_finished[first + rank] = a.eos >= 0 && (token[tid] == a.eos || a.finished[first + r]);
  }
}

struct ReorderArgs {
  uint16_t *k, *v;
  const int32_t *parents, *begin, *end;
  int beams, max_seq, slabs;  // slabs: (layer, head) pairs
  int64_t seq;                // elements of one sequence's cache
};

// Workgroup (x, g): steps x, x + gridDim.x, ... of group g; a step is 16 rows of one (cache, layer, head).
template <int W>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
  const int g0 = blockIdx.y * a.beams;
  int from[W], lo[W], hi[W], p0 = INT32_MAX, p1 = 0;
#pragma unroll
  for (int b = 0; b < W; ++b) {
    from[b] = 0;
    lo[b] = hi[b] = 0;
    if (b < a.beams) {
      const int p = a.parents[g0 + b] - g0;
      if (p >= 0 && p < a.beams && p != b) {
        from[b] = p;
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
      if (row >= lo[b] && row < hi[b]) *reinterpret_cast<u32x4*>(base + b * a.seq) = x[b];
  }
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace mkp

using namespace mkp;

extern "C" size_t mk_beam_select_workspace_bytes(int rows, int vocab, int beams) {
  if (rows < 1 || vocab < 1 || vocab > BV_MAX || beams < 1 || beams > BEAMS_MAX) return 0;
  const size_t slots = (size_t)rows * ((vocab + BC - 1) / BC);
  return align256(slots * beams * sizeof(u64)) + align256(slots * sizeof(float2));
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
  a.stat = reinterpret_cast<float2*>(static_cast<char*>(workspace) +
                                     align256((size_t)rows * a.chunks * beams * sizeof(u64)));
  a.tokens = tokens;
  a.parents = parents;
  a.out_scores = out_scores;
  a.out_finished = out_finished;
  hipLaunchKernelGGL(beam_chunk_kernel, dim3((a.chunks + 3) / 4, rows), dim3(256), 0, stream, a);
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
  if ((int64_t)num_layers * HKV * 2 * ((max_seq_len + 15) / 16) > INT32_MAX) return hipErrorInvalidValue;
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
  const int groups = rows / beams, wgs = std::max(1, 2048 / groups);
  const dim3 grid(std::min(wgs, 2 * a.slabs * ((max_seq_len + 15) / 16)), groups);
  if (beams <= 2) hipLaunchKernelGGL(beam_reorder_kernel<2>, grid, dim3(256), 0, stream, a);
  else if (beams <= 4) hipLaunchKernelGGL(beam_reorder_kernel<4>, grid, dim3(256), 0, stream, a);
  else if (beams <= 8) hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}
