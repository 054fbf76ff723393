// Sampling from the logits with temperature, top-k, top-p and min-p and a given random number a row, on MI355X
// (gfx950). With w = exp((x - max) / T):
//   candidates  the top_k largest logits; of these, in order, the fewest whose w reach top_p of their sum; of these
//               those with w >= min_p. Equal logits: the lower token first. All three are one cut (x, token) in the
//               order of the logits;
//   answer      the first token of the vocabulary at which the running sum of the candidates' w exceeds u times
//               their whole sum.
// The answer is a whole number that a border may decide, so sums are exact ones of w rounded to 2^-36 of itself, and two
// sums within SAME of each other count as equal: 5 of 10 equal logits reach half of them, and do not exceed it.
//
// Bins, 11 to a factor of 2. p = x * 11 log2(e) / T falls into bin floor(p), the same for equal logits wherever they
// are, and within its bin w is 2^((p - floor(p)) / 11), a polynomial on [1, 1.066), kept as a whole number of 2^-36: a
// bin's sum is a sum of whole numbers, the same in any order, and its weight that sum times 2^(bin / 11). Its number of
// logits shares the 64 bits, so that a logit is one atomic addition in LDS: 8,192 logits leave 36 bits behind the point, 12 more
// than the logits, the numbers u and top_p themselves have. More would take a second addition for the number.
//   sample_chunk_kernel  a workgroup takes 8,192 logits of a row from registers into 512 bins (a factor of 2^46) below
//                        their maximum (what lies lower is a tail of its own), and lists the logits of the first bins,
//                        up to 256 of them in all;
//   sample_pick_kernel   a workgroup per row. Where its borders lie among the listed logits it bins these, finds the
//                        bin that a border falls into, sorts that bin's logits, and sums the kept ones chunk by chunk.
//                        Where a border lies deeper it joins the chunks' bins instead and gathers the border's bin from
//                        the row, by its logits' bins in a byte each (narrowing it first where it holds more than 4,096). The
//                        answer is looked for among the 8,192 logits of its chunk. Without any filter the chunks' sums are all
//                        that is needed.
// How deep a border lies is up to the logits: of normal ones of deviation 2 with two dozen peaks, top-p 0.9 at T 0.8 goes below
// the lists in a third of the rows, 0.95 at T 1 in nearly all (40,000 of 151,936 tokens kept), a top-k of 50 in none.
// The logits are read once and the chunk of the answer, or its listed logits, again. Measured on MI355X: one row of 151,936 22
// to 25 us, 9 of them the first kernel, a chain of seven barriers, and 13 to 15 the second; with a border deeper than the lists
// 37 to 45, 28 and more of them the second kernel's one workgroup (the gather by codes, the sort, the chunks' sums).
// 64 rows (39 MB) 53 to 54 us with such borders among them: 24 us of the first kernel, which the 64-bit
// products and whole-number atomics of the weights bound (its read alone takes 8 us), and the deepest row's second.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "mk_device.h"
#include "mk_layers.h"
#include "mk_scan.h"
#include "../../include/megakernel_amd.h"

namespace mkp {

constexpr int ST = 1024;            // threads of the second kernel
constexpr int SW = ST / 64;
constexpr int SC = 8192;            // logits of a chunk
constexpr int SV_MAX = 1 << 20;
constexpr int SCH = SV_MAX / SC;    // chunks of a row at most
constexpr int NB = 512;             // bins; the last one is the tail
constexpr int RES = 11;             // bins to a factor of 2
constexpr int FIX = 36;             // bits behind the point of a weight within its bin
constexpr double ONE = (double)(1ull << FIX);
constexpr int CNT = 50;             // a bin's number of logits, at most 8,192, from this bit on
constexpr u64 SUM_MASK = (1ull << CNT) - 1;
constexpr double SAME = 1.0 / (1ull << 42);
constexpr int CAP = 4096;           // logits of a bin that are taken together: what LDS holds
constexpr int RANKED = 256;         // logits that are sorted by counting, four threads of the 1,024 to each
constexpr int SUB = 2048;           // narrower bins of a bin that holds more
constexpr int LISTED = 4;           // listed logits of a row per thread
constexpr int LIST_MAX = 256;       // and of a chunk, a multiple of 64 (above 64 chunks, 524,288 logits, none: all borders
                                    // are deep ones)

typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any element

struct SampleStat {
  double ref;    // the bin of the chunk's maximum; -infinity: no finite logit
  double total;  // its weights, in units of 2^(ref / 11)
  double tail;   // those below the bins
  u64 key;       // the largest logit, the lowest token of equal ones; all bits set: the chunk has a NaN or +infinity
  int32_t tail_count, number;
  int32_t depth;  // bins 0 .. depth are listed in full; NB: all logits are
};

struct SampleArgs {
  const float* logits;
  int64_t row_stride;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprobs;
  int vocab, chunks, list;  // list: logits listed of a chunk
  SampleStat* stat;  // [rows][chunks]
  u64* bins;         // [rows][chunks][NB]
  u64* listed;       // [rows][chunks][list], filled up with 0
  uint8_t* codes;    // [rows][chunks][SC]: half of each logit's bin, of rows whose border may lie deeper
};

// No weight is above 1: a larger min_p leaves the likeliest token alone, the lowest of equal ones, as a top_k of 1 does.
__device__ __forceinline__ int top_k_under(float min_p, int top_k) { return min_p > 1.f ? 1 : top_k; }

__device__ __forceinline__ uint32_t logit_order(float x) {  // unsigned order is the numbers'
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 logit_key(float x, int v) { return (u64)logit_order(x) << 32 | (0xffffffffu - (uint32_t)v); }
__device__ __forceinline__ float key_x(u64 key) { return logit_of((uint32_t)(key >> 32)); }
__device__ __forceinline__ int key_v(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

// How logits at a temperature fall into bins: c bins per logit. `in` is 1, or 0 where bins are so small (p above 2^45)
// that different logits lie thousands of bins apart and p has too few digits behind the point: any place in the bin
// serves.
struct Scale {
  double c, in;
};
__device__ __forceinline__ Scale scale_of_row(float T, double top) {
  Scale s;
  s.c = RES * 1.4426950408889634 / (double)T;
  s.in = fabs(top * s.c) < 0x1p45 ? 1.0 : 0.0;
  return s;
}
// Bins from the largest logit's down to which there are weights, a factor of 2^1000: what lies lower is 0, everywhere, so that a
// chunk whose sum is not 0 has a logit that is drawn, and no weight is too small for a double's full precision.
constexpr double DEEPEST = 1000 * RES;
// 2^(-k / RES) for a whole number k >= 0, to 2^-51 of itself
__device__ __forceinline__ double bin_weight(double k) {
  if (!(k <= DEEPEST)) return 0;
  const double q = floor(k * (1.0 / RES) + 1.0 / (2 * RES));
  const int i = (int)(k - q * RES);  // its powers of 2: 2^(-2^b / 11)
  double y = i & 1 ? 0x1.e0bb8d64fdb5ap-1 : 1.0;
  y *= i & 2 ? 0x1.c35fedd14b862p-1 : 1.0;
  y *= i & 4 ? 0x1.8ded91f0e72eep-1 : 1.0;
  y *= i & 8 ? 0x1.3545598e5c232p-1 : 1.0;
  return ldexp(y, -(int)q);
}
// log x to 2^-48 of itself: 2 artanh((m - 1) / (m + 1)) of the mantissa m in [0.7, 1.42)
__device__ __forceinline__ double log64(double x) {
  int e;
  double m = frexp(x, &e);
  if (m < 0.70710678) {
    m *= 2;
    --e;
  }
  const double t = (m - 1) / (m + 1), q = t * t;
  double y = 1.0 / 21;
#pragma unroll
  for (int k = 19; k >= 3; k -= 2) y = fma(y, q, 1.0 / k);
  return fma((double)e, 0.6931471805599453, 2 * fma(t * q, y, t));
}
// 2^(f / 11) for the place f in [0, 1] of a logit in its bin fl, in whole numbers of 2^-FIX: the series, whose next
// term is below 2^-40, behind 2^16, where a double's last bit is 2^-36.
__device__ __forceinline__ u64 fixed_in_bin(float x, const Scale& s, double fl) {
  constexpr double A = 0.6931471805599453 / RES, BIG = 1 << (52 - FIX);
  const double f = fma((double)x, s.c, -fl) * s.in;
  double y = A * A * A * A * A * A / 720;
  y = fma(y, f, A * A * A * A * A / 120);
  y = fma(y, f, A * A * A * A / 24);
  y = fma(y, f, A * A * A / 6);
  y = fma(y, f, A * A / 2);
  y = fma(y, f, A);
  return __builtin_bit_cast(u64, fma(y, f, 1 + BIG)) - __builtin_bit_cast(u64, BIG);
}
// 2^((p - ref) / 11) to fp32's accuracy: the tail's weights, below 2^-46 of the largest. `fl` is floor(p), a logit's bin, which alone
// decides where weights end, as it does for chunks.
__device__ __forceinline__ double tail_weight(double p, double fl, double ref) {
  if (!(ref - fl <= DEEPEST)) return 0;
  const double t = (p - ref) * (1.0 / RES), n = floor(t);
  return ldexp((double)__builtin_amdgcn_exp2f((float)(t - n)), (int)n);
}
// the bin of floor(p) below `ref`, the tail's for all from there on
__device__ __forceinline__ int bin_of(double ref, double fl) {
  const double k = ref - fl;
  return k < NB - 1 ? (int)k : NB - 1;
}

// The second kernel runs each of its instructions a few times at most, and what takes its time beside the loads is the
// fetch of cold code. So its loops are not unrolled: eight numbers in registers turn round instead.
__device__ __forceinline__ void turn(float (&f)[8]) {
  const float x = f[0];
#pragma unroll
  for (int i = 0; i < 7; ++i) f[i] = f[i + 1];
  f[7] = x;
}

// W waves to a chunk's 8,192 logits.
template <int W>
__global__ void __launch_bounds__(64 * W) sample_chunk_kernel(const SampleArgs a) {
  constexpr int N = SC / (64 * W), PB = (NB + 64 * W - 1) / (64 * W);  // logits and bins to a thread
  __shared__ u64 bins[NB];
  __shared__ u64 skey[W];
  __shared__ double stail[W], stotal[W];
  __shared__ int32_t stc[W], scan[W];
  __shared__ int sdepth;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.y, v0 = blockIdx.x * SC + 64 * N * w + 4 * lane;  // this lane's logits: v0 + 256 j + q
  const float* x = a.logits + row * a.row_stride;
  float f[N];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const int v = v0 + 256 * j;
    if (v + 3 < a.vocab) {
      const f4a t = *reinterpret_cast<const f4a*>(x + v);
#pragma unroll
      for (int q = 0; q < 4; ++q) f[4 * j + q] = t[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) f[4 * j + q] = v + q < a.vocab ? x[v + q] : -INFINITY;
    }
  }
  const float T = a.temperature[row];
  const float top_p = a.top_p[row], min_p = a.min_p[row];
  const int top_k = top_k_under(min_p, a.top_k[row]);
  const bool filtered = top_k > 0 || !(top_p >= 1.f) || min_p > 0.f;
  for (int i = tid; i < NB; i += 64 * W) bins[i] = 0;
  if (tid == 0) sdepth = -1;
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m = fmaxf(m, f[i]);
    bad |= !(f[i] < INFINITY);  // NaN too
  }
  int at = 0;
  if (T == 0.f)  // nobody else asks for the token
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
      if (f[i] == m) at = v0 + 256 * (i >> 2) + (i & 3);
  u64 key = max_over_wave(bad ? ~(u64)0 : logit_key(m, at));
  if (lane == 0) skey[w] = key;
  __syncthreads();
  key = max_over_wave(skey[lane & (W - 1)]);
  const float top = key_x(key);  // NaN, where all bits are set
  const int64_t slot = (int64_t)row * a.chunks + blockIdx.x;
  const Scale s = scale_of_row(T, top);
  SampleStat out{};
  out.ref = top == -INFINITY ? -INFINITY : floor((double)top * s.c);
  out.key = key;
  out.depth = NB;
  if (!(T > 0.f) || !(top > -INFINITY)) {  // the likeliest, no number, or an answer that has failed
    if (filtered) {
      for (int i = tid; i < NB; i += 64 * W) a.bins[slot * NB + i] = 0;
      for (int i = tid; i < a.list; i += 64 * W) a.listed[slot * a.list + i] = 0;
    }
    if (tid == 0) a.stat[slot] = out;
    return;
  }
  if (min_p > 0.f && top_p >= 1.f) {  // what min_p leaves out against the chunk's maximum nobody asks for
    const float low = (float)((double)top + (double)T * log64(fmin((double)min_p, 1.0)));
    const float lim = low - fmaxf(fabsf(low) * 0x1p-22f, 1e-37f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = f[i] >= lim ? f[i] : -INFINITY;
  }
  const bool coded = filtered && (top_k <= 0 || top_k > a.list);
  uint32_t* codes = reinterpret_cast<uint32_t*>(a.codes + slot * SC + 64 * N * w + 4 * lane);
  double tail = 0;
  int tc = 0;
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    uint32_t code = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = 4 * j + q;
      const double p = (double)f[i] * s.c, fl = floor(p);
      const int bin = bin_of(out.ref, fl);
      if (bin < NB - 1) {
        atomicAdd(&bins[bin], fixed_in_bin(f[i], s, fl) + (1ull << CNT));
      } else if (f[i] > -INFINITY) {
        tail += tail_weight(p, fl, out.ref);
        ++tc;
      }
      code |= (uint32_t)(bin >> 1) << (8 * q);
    }
    if (coded) codes[64 * j] = code;
  }
  if (__builtin_amdgcn_ballot_w64(tc > 0)) {
    tail = sum_over_wave(tail);
    tc = sum_over_wave(tc);
  }
  if (lane == 0) {
    stail[w] = tail;
    stc[w] = tc;
  }
  __syncthreads();
  // the bins' weights and numbers, PB to a thread
  u64 b[PB];
  double weight = 0;
  int number = 0, all;
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int j = PB * tid + i;
    b[i] = j < NB ? bins[j] : 0;
    weight += (double)(b[i] & SUM_MASK) / ONE * bin_weight(j);
    number += (int)(b[i] >> CNT);
  }
  weight = sum_over_wave(weight);
  if (lane == 0) stotal[w] = weight;
  int upto = block_before<W>(number, scan, all);  // (stotal is written behind it)
#pragma unroll 1
  for (int i = 0; i < W; ++i) {
    out.tail += stail[i];
    out.tail_count += stc[i];
    out.total += stotal[i];
  }
  out.total += out.tail;
  out.number = all + out.tail_count;
  if (filtered) {
    // the bins that the list holds in full
    int in = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int j = PB * tid + i;
      upto += (int)(b[i] >> CNT);
      if (j < NB) a.bins[slot * NB + j] = b[i];
      in += __popcll(__builtin_amdgcn_ballot_w64(j < NB - 1 && upto <= a.list));
    }
    if (lane == 0 && in) atomicAdd(&sdepth, in);
    __syncthreads();
    out.depth = out.number <= a.list ? NB : sdepth;
    // their logits, in the threads' order: first those that cannot be lower, to a part of a bin
    // (their bins decide as they did above: beyond 2^53 the number of the bin that is next to `ref` is `ref` again)
    const float lim = out.depth == NB ? -INFINITY : (float)fmax((out.ref - out.depth - 0.5) / s.c, -3.4028234663852886e38);
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine = mine + mine + (f[i] >= lim && f[i] > -INFINITY);
    uint32_t keep = 0;
    for (uint32_t todo = mine; todo;) {
      const int e = 31 - __clz(todo);
      todo &= ~(1u << e);
      const int i = N - 1 - e;
      const float y = x[v0 + 256 * (i >> 2) + (i & 3)];  // again: cheaper than finding it among the registers
      if (bin_of(out.ref, floor((double)y * s.c)) <= out.depth) keep |= 1u << e;
    }
    int n;
    int to = block_before<W>((int)__popc(keep), scan, n);
    while (keep) {
      const int e = 31 - __clz(keep);
      keep &= ~(1u << e);
      const int i = N - 1 - e, v = v0 + 256 * (i >> 2) + (i & 3);
      a.listed[slot * a.list + to++] = logit_key(x[v], v);
    }
    for (int i = n + tid; i < a.list; i += 64 * W) a.listed[slot * a.list + i] = 0;
  }
  if (tid == 0) a.stat[slot] = out;
}

// The least u32 in [lo, hi] for which `test`, false up to some number and true from there on, is true (hi, if none
// below it is), by all lanes of a wave: 64 numbers around a guess as a rule decide, else 64 places at a time.
template <typename F>
__device__ __forceinline__ uint32_t least_true(uint32_t lo, uint32_t hi, uint32_t guess, F test) {
  const int lane = threadIdx.x & 63;
  uint64_t a = max(lo, min(hi, max(guess, 32u) - 32)), n = 63;
  bool near = true;
#pragma unroll 1
  while (n > 0) {  // the answer lies in [a, a + n], once it is not near
    const uint64_t step = (n + 63) / 64, end = min((uint64_t)hi, a + n);
    const uint64_t at = near ? a + lane : a + (lane + 1) * step - 1;  // is it at or before there?
    const u64 hit = __builtin_amdgcn_ballot_w64(at >= (near ? (uint64_t)hi : end) || test((uint32_t)min((uint64_t)hi, at)));
    const int first = hit ? __ffsll(hit) - 1 : 64;
    if (near) {
      near = false;
      if (hit && (first > 0 || a == lo)) return (uint32_t)min((uint64_t)hi, a + first);
      a = lo;
      n = hi - lo;
    } else {
      a = min(end, a + first * step);
      n = min(step - 1, end - a);
    }
  }
  return (uint32_t)a;
}

// A row's border: kept are bins 0 .. bin - 1 and, of bin `bin`, all (part false) or the logits above x and those
// equal to it up to token i.
struct Cut {
  int bin;
  bool part;
  float x;
  int token;
  __device__ __forceinline__ bool keeps(int j, float y, int v) const {
    return j < bin || (j == bin && (!part || y > x || (y == x && v <= token)));
  }
};

// What the threads of a row share.
struct PickSmem {
  double et[NB];        // 2^(-j / 11)
  double upto[NB];      // weights of bins 0 .. j
  int32_t cupto[NB];    // their logits
  int32_t delta[SCH];   // bins of the row above the chunk's first (at most 2^20)
  double scale[SCH], csum[SCH];
  u64 part[SCH];        // kept weights of the border's bin, by chunk
  u64 lkey[LISTED * ST];  // the listed logits; where a border lies deeper, no longer needed
  u64 lbin[LISTED * ST];  // their bins, above LBIN, and weights in their bins
  u64 list[CAP];  // logits of a bin
  union {
    u64 bins[NB];
    u64 sub[SUB];  // numbers and sums of narrower bins
    struct {
      u64 sum[SUB];
      uint32_t count[SUB];
    } many;
    struct {
      u64 raw[RANKED], key[RANKED];
    } sort;
    double lsum[LISTED * SW];  // kept weights of 64 listed logits each
    struct {
      uint32_t map[SC / 32];
      int mapped[SC / 32], token[LIST_MAX];
      double inorder[LIST_MAX];
    };
  };
  double wsum[SW];
  int32_t wcount[SW];
  u64 wfix[SW], wfix2[SW];
  int first, last;  // of the answer's candidates
  int found, border, n, above, depth, number;
  u64 sum, key;
  uint32_t klo, khi;
  double z, goal;
  Cut cut;
};
__device__ __forceinline__ PickSmem& smem() {
  __shared__ PickSmem s;
  return s;
}
constexpr int LBIN = 40;

struct Row {
  const float* x;
  int vocab;
  Scale s;
  double ref;  // the bin of the largest
  uint32_t ktop, kmin;
};

__device__ __forceinline__ double weight_below(int j) { return j > 0 ? smem().upto[j - 1] : 0.0; }
__device__ __forceinline__ int number_below(int j) { return j > 0 ? smem().cupto[j - 1] : 0; }
// The bin that a border falls into: the first one up to which there are `rank` logits (by_rank), or, of those that have any,
// weights of `goal`; the last one if none is. (Running sums are added up in orders of their own: a bin without logits may have
// a larger one than the bins around it, by the last digit.)
__device__ __forceinline__ int border_bin(bool by_rank, int rank, double goal) {
  PickSmem& sm = smem();
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) sm.border = NB - 1;
  __syncthreads();
  if (tid < NB) {
    const int n = sm.cupto[tid];
    const u64 hit = __builtin_amdgcn_ballot_w64(by_rank ? n >= rank : n > number_below(tid) && sm.upto[tid] >= goal);
    if (hit && lane == __ffsll(hit) - 1) atomicMin(&sm.border, tid);
  }
  __syncthreads();
  return sm.border;
}

// The weight of a logit of the row's bin j, in 2^-FIX of 2^(-j / 11).
__device__ __forceinline__ u64 fixed_weight(const Scale& s, double ref, float x, int j) {
  const double p = (double)x * s.c, fl = floor(p);
  if (j == NB - 1) return (u64)(tail_weight(p, fl, ref) * (ONE / smem().et[NB - 1]));
  return fixed_in_bin(x, s, fl);
}

// The border among sm.list, n <= CAP logits of bin j: the first of them, in order, at which their number reaches `rank`
// (by_rank), or their sum reaches `goal` (in 2^-FIX of the bin's unit; the last of `most` logits, if none of them does),
// `above` and `sabove` being those of the bin before the list. Into sm.key, and the sum up to it into sm.sum.
// The range of the keys is narrowed, SUB bins at a time, to the few that are sorted.
__device__ __forceinline__ void border_in_list(int n, int j, double c, double in, double ref, bool by_rank,
                                                         int rank, double goal, int most, int above, u64 sabove) {
  PickSmem& sm = smem();
  const int tid = threadIdx.x;
  const Scale s = {c, in};
  const int size = n;
  auto reached = [&](int number, u64 sum) { return by_rank ? number >= rank : (double)sum >= goal || number >= most; };
  u64 lo = 0, hi = ~(u64)0;
  if (n > RANKED) {  // the list's own range
    u64 l = ~(u64)0, h = 0;
#pragma unroll 1
    for (int i = tid; i < size; i += ST) {
      l = min(l, sm.list[i]);
      h = max(h, sm.list[i]);
    }
    h = max_over_wave(h);
    l = ~max_over_wave(~l);
    __syncthreads();
    if ((tid & 63) == 0) {
      sm.wfix[tid >> 6] = h;
      sm.wfix2[tid >> 6] = l;
    }
    __syncthreads();
    hi = max_over_wave(sm.wfix[tid & (SW - 1)]);
    lo = ~max_over_wave(~sm.wfix2[tid & (SW - 1)]);
  }
#pragma unroll 1
  while (n > RANKED) {
    const int bits = 64 - __clzll((hi - lo) | 1), shift = max(0, bits - 11);
    __syncthreads();
    for (int i = tid; i < SUB; i += ST) sm.sub[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < size; i += ST) {
      const u64 k = sm.list[i];
      if (k >= lo && k <= hi) atomicAdd(&sm.sub[(hi - k) >> shift], fixed_weight(s, ref, key_x(k), j) + (1ull << CNT));
    }
    __syncthreads();
    const u64 b0 = sm.sub[2 * tid], b1 = sm.sub[2 * tid + 1];
    u64 all;
    const u64 before = block_before<SW>(b0 + b1, sm.wfix, all);
    const int c0 = above + (int)(before >> CNT);
    const u64 s0 = sabove + (before & SUM_MASK);
    const int c1 = c0 + (int)(b0 >> CNT), c2 = c1 + (int)(b1 >> CNT);
    const u64 s1 = s0 + (b0 & SUM_MASK), s2 = s1 + (b1 & SUM_MASK);
    // the one bin where it is reached, the last one with any logits if nowhere
    const int end = above + n;
    const bool r0 = c0 > above && (reached(c0, s0) || c0 == end), r1 = c1 > above && (reached(c1, s1) || c1 == end);
    const bool r2 = c2 > above && (reached(c2, s2) || c2 == end);
    if (!r0 && r2) {
      sm.found = r1 ? 2 * tid : 2 * tid + 1;
      sm.n = (int)((r1 ? b0 : b1) >> CNT);
      sm.above = r1 ? c0 : c1;
      sm.sum = r1 ? s0 : s1;
    }
    __syncthreads();
    n = sm.n;
    above = sm.above;
    sabove = sm.sum;
    hi -= (u64)sm.found << shift;
    const u64 width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
  }
  // the rest sorted: a key's place is how many are larger, four lanes to a key
  __syncthreads();
  if (tid == 0) sm.n = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < size; i += ST) {
    const u64 k = sm.list[i];
    if (k >= lo && k <= hi) {
      const int at = atomicAdd(&sm.n, 1);
      if (at < RANKED) sm.sort.raw[at] = k;
    }
  }
  __syncthreads();
  {
    const int i = tid >> 2;
    const u64 k = i < n ? sm.sort.raw[i] : 0;
    int place = 0;
    if (i < n)
#pragma unroll 4
      for (int e = tid & 3; e < n; e += 4) place += sm.sort.raw[e] > k;
    place += __shfl_xor(place, 1);
    place += __shfl_xor(place, 2);
    if (i < n && (tid & 3) == 0) sm.sort.key[place] = k;
  }
  __syncthreads();
  const u64 k = tid < n ? sm.sort.key[tid] : 0, mine = tid < n ? fixed_weight(s, ref, key_x(k), j) : 0;
  u64 all;
  const u64 before = sabove + block_before<SW>(mine, sm.wfix, all);
  if (tid < n && (tid == 0 || !reached(above + tid, before)) && (tid == n - 1 || reached(above + tid + 1, before + mine))) {
    sm.key = k;
    sm.sum = before + mine;
  }
  __syncthreads();
}

// -----------------------------------------------------------------------------------------------------------
// Borders that lie deeper than the listed logits: from the chunks' bins and the row's logits.
// -----------------------------------------------------------------------------------------------------------

// fn(logit, token) for every logit of the row whose order's number lies in [lo, hi], by the whole workgroup. 32 logits
// to a thread are compared as numbers (both zeros are one, with one place in the order); the few that pass are read again.
template <typename F>
__device__ __forceinline__ void sweep(const Row& r, uint32_t lo, uint32_t hi, F fn) {
  const int tid = threadIdx.x;
  const float flo = logit_of(lo), fhi = logit_of(hi);
#pragma unroll 1
  for (int base = 0; base < r.vocab; base += 8 * 4 * ST) {
    float f[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int v = base + 4 * ST * j + 4 * tid;
      if (v + 3 < r.vocab) {
        const f4a t = *reinterpret_cast<const f4a*>(r.x + v);
#pragma unroll
        for (int q = 0; q < 4; ++q) f[j][q] = t[q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) f[j][q] = v + q < r.vocab ? r.x[v + q] : -INFINITY;
      }
    }
    uint32_t mask = 0;  // the first logit in the highest bit
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) mask = mask + mask + (__builtin_amdgcn_fmed3f(f[j][q], flo, fhi) == f[j][q]);
#pragma unroll 1
    while (mask) {
      const int e = __clz(mask), v = base + 4 * ST * (e >> 2) + 4 * tid + (e & 3);
      mask &= ~(0x80000000u >> e);
      const float x = r.x[v];
      const uint32_t o = logit_order(x);
      if (o >= lo && o <= hi) fn(x, v);
    }
  }
}

__device__ __forceinline__ u64 fixed_weight(const Row& r, float x, int j) { return fixed_weight(r.s, r.ref, x, j); }

// The order's numbers of bin j's logits, by two waves.
__device__ __forceinline__ void bin_range(const Row& r, int j) {
  PickSmem& sm = smem();
  __syncthreads();
  if (threadIdx.x < 128) {
    const bool high = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double b = r.ref - j + high;  // the least logit of bin j, or of the one above
    uint32_t k = high ? r.ktop + 1 : r.kmin;
    if (high ? j > 0 : j < NB - 1) {
      const float guess = (float)fmin(fmax(b / r.s.c, -3.4028234663852886e38), (double)logit_of(r.ktop));
      k = least_true(r.kmin, r.ktop, logit_order(guess), [&](uint32_t o) { return floor((double)logit_of(o) * r.s.c) >= b; });
    }
    if ((threadIdx.x & 63) == 0) {
      if (high) sm.khi = k - 1;
      else sm.klo = k;
    }
  }
  __syncthreads();
}

// Gathers the logits of the order's numbers [klo, khi], at most CAP.
__device__ __forceinline__ void gather(const Row& r, uint32_t klo, uint32_t khi) {
  PickSmem& sm = smem();
  __syncthreads();
  if (threadIdx.x == 0) sm.n = 0;
  __syncthreads();
  sweep(r, klo, khi, [&](float x, int v) {
    const int at = atomicAdd(&sm.n, 1);
    if (at < CAP) sm.list[at] = logit_key(x, v);
  });
  __syncthreads();
}

// Gathers the logits of bin j, not the tail's, from `low` on, at most CAP, by the codes: 16 of them to a load. False if too
// many others have their code.
__device__ __forceinline__ bool gather_bin(const Row& r, const uint8_t* codes, int chunks, int j, float low) {
  PickSmem& sm = smem();
  int* maybe = reinterpret_cast<int*>(sm.lkey);
  static_assert(sizeof(sm.lkey) >= 2 * CAP * sizeof(int));
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) sm.n = sm.found = 0;
  __syncthreads();
  const double fl = r.ref - j;
  const int units = chunks * (SC / 16);
#pragma unroll 1
  for (int base = 0; base < units; base += 5 * ST) {
    uint4 q[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int at = base + i * ST + tid;
      q[i] = at < units ? *reinterpret_cast<const uint4*>(codes + (int64_t)16 * at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int at = base + i * ST + tid, k = j - sm.delta[min(at / (SC / 16), chunks - 1)];  // the chunk's bin
      if (at >= units || k < 0) continue;
      const uint32_t code = (uint32_t)(k >> 1) * 0x01010101u, w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
      uint32_t mask = 0;  // bit 8 byte + word: a byte that is the code
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t y = w[e] ^ code, z = ~(((y & 0x7f7f7f7fu) + 0x7f7f7f7fu) | y) & 0x80808080u;
        mask |= z >> (7 - e);
      }
#pragma unroll 1
      while (mask) {
        const int bit = __ffs(mask) - 1, v = 16 * at + 4 * (bit & 7) + (bit >> 3);
        mask &= mask - 1;
        const int to = atomicAdd(&sm.found, 1);
        if (to < 2 * CAP) maybe[to] = v;
      }
    }
  }
  __syncthreads();
  const int all = sm.found;
  if (all > 2 * CAP) return false;
#pragma unroll 4
  for (int i = tid; i < all; i += ST) {
    const int v = maybe[i];
    const float x = v < r.vocab ? r.x[v] : -INFINITY;
    if (floor((double)x * r.s.c) == fl && x >= low) {
      const int to = atomicAdd(&sm.n, 1);
      if (to < CAP) sm.list[to] = logit_key(x, v);
    }
  }
  __syncthreads();
  return true;
}

// Finds the border within bin j, which has `count` logits: the first of them, in order, at which their number reaches
// `rank` (by_rank), or their sum reaches `goal` (in 2^-FIX of the bin's unit; the last of `most` logits, if none of
// them does). Returns the sum up to it. `low`: the count may leave out logits below it, which the first kernel has dropped
// for min_p; a border among these is put at `low`. held: how many of the bin's logits from `low` on sm.list then
// holds, all of them, or -1.
__device__ __forceinline__ u64 border_in_bin(const Row& r, const uint8_t* codes, int chunks, int j, int count, bool by_rank,
                                             int rank, double goal, int most, float low, Cut& cut, int& held) {
  PickSmem& sm = smem();
  const int tid = threadIdx.x;
  int n = count, above = 0;  // logits in [klo, khi], and of the bin above khi
  u64 sabove = 0;
  held = -1;
  if (!(count <= CAP && j < NB - 1 && codes && gather_bin(r, codes, chunks, j, low))) {
    bin_range(r, j);
    uint32_t klo = sm.klo, khi = sm.khi;
    if (count <= CAP) klo = max(klo, logit_order(low));
    auto reached = [&](int number, u64 sum) { return by_rank ? number >= rank : (double)sum >= goal || number >= most; };
    while (n > CAP && klo < khi) {  // narrow: SUB bins of the order's numbers, the first of the order first
      int shift = 0;
      while (((khi - klo) >> shift) >= SUB) ++shift;
      __syncthreads();
      for (int i = tid; i < SUB; i += ST) {
        sm.many.sum[i] = 0;
        sm.many.count[i] = 0;
      }
      __syncthreads();
      sweep(r, klo, khi, [&](float x, int) {
        const uint32_t b = (khi - logit_order(x)) >> shift;
        atomicAdd(&sm.many.count[b], 1u);
        atomicAdd(&sm.many.sum[b], fixed_weight(r, x, j));
      });
      __syncthreads();
      const int c0 = (int)sm.many.count[2 * tid], c1 = (int)sm.many.count[2 * tid + 1];
      const u64 s0 = sm.many.sum[2 * tid], s1 = sm.many.sum[2 * tid + 1];
      int call;
      u64 sall;
      int cb = above + block_before<SW>(c0 + c1, sm.wcount, call);
      u64 sb = sabove + block_before<SW>(s0 + s1, sm.wfix, sall);
      // the one place where it is reached, at the end of the range if nowhere before
      const int lastb = (int)((khi - klo) >> shift);
      const bool r0 = reached(cb + c0, sb + s0) || 2 * tid >= lastb, r1 = reached(cb + c0 + c1, sb + s0 + s1) || 2 * tid + 1 >= lastb;
      const bool rb = tid > 0 && (reached(cb, sb) || 2 * tid - 1 >= lastb);
      if (!rb && r1) {
        sm.found = r0 ? 2 * tid : 2 * tid + 1;
        sm.n = r0 ? c0 : c1;
        sm.above = r0 ? cb : cb + c0;
        sm.sum = r0 ? sb : sb + s0;
      }
      __syncthreads();
      n = sm.n;
      above = sm.above;
      sabove = sm.sum;
      const uint32_t hi = khi - ((uint32_t)sm.found << shift), width = (1u << shift) - 1;
      klo = hi - klo > width ? hi - width : klo;
      khi = hi;
      __syncthreads();
    }
    if (n > CAP) {  // equal logits: so many of them, the lowest tokens
      const float x = logit_of(khi);
      const u64 w = fixed_weight(r, x, j);
      int take;
      if (by_rank) {
        take = rank - above;
      } else {
        take = w ? (int)fmin(ceil((goal - (double)sabove) / (double)w), (double)n) : n;
        take = min(take, most - above);
      }
      take = max(1, min(take, n));
      // the token of the take-th: tokens in their order, a piece of 4 to a thread
      int seen = 0;
      if (tid == 0) sm.found = 0;
      for (int base = 0; base < r.vocab && seen < take; base += 4 * ST) {
        int mine = 0, all;
        for (int q = 0; q < 4; ++q) {
          const int v = base + 4 * tid + q;
          mine += v < r.vocab && r.x[v] == x;
        }
        int before = seen + block_before<SW>(mine, sm.wcount, all);
        if (before < take && before + mine >= take)
          for (int q = 0; q < 4; ++q) {
            const int v = base + 4 * tid + q;
            if (v < r.vocab && r.x[v] == x && ++before == take) sm.found = v;
          }
        seen += all;
      }
      __syncthreads();
      cut = {j, true, x, sm.found};
      return sabove + (u64)take * w;
    }
    gather(r, klo, khi);
  }
  if (count <= CAP) {
    n = held = sm.n;
    if (by_rank ? rank > n : n == 0) {
      cut = {j, true, low, INT32_MAX};
      return 0;
    }
  }
  border_in_list(n, j, r.s.c, r.s.in, r.ref, by_rank, rank, goal, most, above, sabove);
  cut = {j, true, key_x(sm.key), key_v(sm.key)};
  return sm.sum;
}

// The border by all filters, one of which has to leave something out, into sm.cut, and the chunks' sums of what is kept, into
// sm.csum.
__device__ __forceinline__ void deep_cut(const u64* bins, const SampleStat* stat,
                                                   const uint8_t* codes, int chunks, const float* x,
                                                   int vocab, double c, double in, double ref, uint32_t ktop, int number,
                                                   double whole, int top_k, float top_p, float xm, int jm) {
  PickSmem& sm = smem();
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Row r = {x, vocab, {c, in}, ref, ktop, logit_order(-3.4028234663852886e38f)};
  __syncthreads();
  // the chunks' bins joined, a wave to a chunk
  for (int i = tid; i < NB; i += ST) {
    sm.many.sum[i] = 0;
    sm.many.count[i] = 0;
  }
  __syncthreads();
  int tn = 0;
#pragma unroll 1
  for (int k = w; k < chunks; k += SW) {
    const int d = sm.delta[k];
    const double f = sm.scale[k];
    u64 b[NB / 64];
#pragma unroll
    for (int i = 0; i < NB / 64; ++i) b[i] = bins[k * NB + 64 * i + lane];
    double t = 0;
#pragma unroll
    for (int i = 0; i < NB / 64; ++i) {
      const int j = 64 * i + lane;
      if (j + d < NB - 1) {
        if (b[i]) {
          atomicAdd(&sm.many.sum[j + d], b[i] & SUM_MASK);
          atomicAdd(&sm.many.count[j + d], (uint32_t)(b[i] >> CNT));
        }
      } else if (j < NB - 1) {  // in the row's tail
        t += (double)(b[i] & SUM_MASK) / ONE * (sm.et[j] * f);
        tn += (int)(b[i] >> CNT);
      }
    }
    t = sum_over_wave(t);
    if (lane == 0) {
      sm.csum[k] = t + stat[k].tail * f;
      tn += stat[k].tail_count;
    }
  }
  if (tid == 0) sm.n = 0;
  __syncthreads();
  tn = sum_over_wave(tn);
  if (lane == 0) atomicAdd(&sm.n, tn);
  double t = (lane < chunks ? sm.csum[lane] : 0) + (64 + lane < chunks ? sm.csum[64 + lane] : 0);
  t = sum_over_wave(t);
  __syncthreads();
  {
    double weight = 0, wall;
    int n = 0, call;
    if (tid < NB) {
      n = tid < NB - 1 ? (int)sm.many.count[tid] : sm.n;
      weight = tid < NB - 1 ? (double)sm.many.sum[tid] / ONE * sm.et[tid] : t;
    }
    const double upto = block_upto<SW>(weight, sm.wsum, wall);
    const int cupto = block_upto<SW>(n, sm.wcount, call);
    if (tid < NB) {
      sm.upto[tid] = upto;
      sm.cupto[tid] = cupto;
    }
    __syncthreads();  // min_p's border alone is looked for without another one
  }
  Cut cut = {NB - 1, false, 0.f, 0};
  const float low = top_p >= 1.f && jm < NB ? xm : -3.4028234663852886e38f;  // the first kernel may have dropped those below
  int kept = number, holds = -1, held = -1;  // candidates; the bin whose logits the list holds, and their number
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const bool by_rank = pass == 0;
    if (by_rank ? top_k <= 0 || top_k >= number : !(top_p < 1.f)) continue;
    const double goal = (double)top_p * whole * (1 - SAME);
    const int j = min(cut.bin, border_bin(by_rank, top_k, goal));
    const int n = sm.cupto[j] - number_below(j);
    const u64 s = border_in_bin(r, codes, chunks, j, n, by_rank, top_k - number_below(j), (goal - weight_below(j)) / sm.et[j] * ONE,
                                min(n, kept - number_below(j)), low, cut, held);
    holds = held >= 0 ? j : -1;
    if (by_rank) {
      kept = top_k;
      whole = weight_below(j) + (double)s / ONE * sm.et[j];
    }
  }
  if (jm < cut.bin || (jm == cut.bin && (!cut.part || xm > cut.x))) cut = {jm, true, xm, INT32_MAX};
  if (tid == 0) sm.cut = cut;
  // The kept weights of the border's bin. One of the tail that is no whole number of its unit is marked, so that its chunk has a
  // sum above 0.
  constexpr u64 MARK = 1ull << 63;  // above all sums: 2^20 weights below 2^37
  {
    const int j = cut.bin, n = sm.cupto[j] - number_below(j);
    auto add = [&](float y, int v) {
      if (!cut.keeps(j, y, v)) return;
      const u64 f = fixed_weight(r, y, j);
      if (f > 0) atomicAdd(&sm.part[v / SC], f);
      else if (r.ref - floor((double)y * r.s.c) <= DEEPEST) atomicOr(&sm.part[v / SC], MARK);
    };
    if (n <= CAP) {
      if (holds != j) {
        if (j == NB - 1 || !codes || !gather_bin(r, codes, chunks, j, cut.x)) {
          bin_range(r, j);
          gather(r, max(sm.klo, logit_order(cut.x)), sm.khi);
        }
        held = sm.n;
      }
      for (int i = tid; i < held; i += ST) add(key_x(sm.list[i]), key_v(sm.list[i]));
    } else {
      bin_range(r, j);
      sweep(r, logit_order(cut.x), sm.khi, add);
    }
  }
  __syncthreads();
  for (int k = w; k < chunks; k += SW) {
    const int d = sm.delta[k];
    double s = 0;
#pragma unroll
    for (int i = 0; i < NB / 64; ++i) {
      const int j = 64 * i + lane;
      const u64 b = bins[k * NB + j];
      if (j < NB - 1 && j + d < cut.bin) s += (double)(b & SUM_MASK) / ONE * (sm.et[j] * sm.scale[k]);
    }
    s = sum_over_wave(s);
    const u64 part = sm.part[k];
    if (lane == 0) sm.csum[k] = s + (double)(part & ~MARK) / ONE * sm.et[cut.bin] + (part & MARK ? 0x1p-1000 : 0);
  }
}

__global__ void __launch_bounds__(ST) sample_pick_kernel(const SampleArgs a) {
  PickSmem& sm = smem();
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x, chunks = a.chunks;
  const int64_t s0 = (int64_t)row * chunks;
  const float T = a.temperature[row], u = a.uniforms[row], top_p = a.top_p[row], min_p = a.min_p[row];
  const int top_k = top_k_under(min_p, a.top_k[row]);
  const bool filtered = top_k > 0 || !(top_p >= 1.f) || min_p > 0.f;
  u64 key = 0;
  SampleStat st{};
  const int ci = tid - NB;  // the threads behind the bins' take a chunk each
  if (ci >= 0 && ci < chunks) st = a.stat[s0 + ci];
  if (lane < chunks) key = a.stat[s0 + lane].key;
  if (64 + lane < chunks) key = max(key, a.stat[s0 + 64 + lane].key);
  if (filtered)
#pragma unroll
    for (int i = 0; i < LISTED; ++i)
      sm.lkey[i * ST + tid] = i * ST + tid < chunks * a.list ? a.listed[s0 * a.list + i * ST + tid] : 0;
  key = max_over_wave(key);
  const float top = key_x(key);  // NaN for a row that has failed
  if (!(top > -INFINITY) || !(T >= 0.f && T < INFINITY) || u != u || top_p != top_p || min_p != min_p || T == 0.f) {
    if (tid == 0) {
      const bool likeliest = T == 0.f && top > -INFINITY && u == u && top_p == top_p && min_p == min_p;
      a.tokens[row] = likeliest ? key_v(key) : -1;
      if (a.logprobs) a.logprobs[row] = likeliest ? 0.f : __builtin_nanf("");
    }
    return;
  }
  const float* x = a.logits + row * a.row_stride;
  const Scale sc = scale_of_row(T, top);
  const double ref = floor((double)top * sc.c);
  if (tid == 0) {
    sm.depth = NB - 2;
    sm.number = 0;
  }
  const double d = ref - st.ref;
  const double y = bin_weight(tid < NB ? tid : d);
  if (tid < NB) {
    sm.et[tid] = y;
    sm.bins[tid] = 0;
  }
  __syncthreads();
  if (ci >= 0 && ci < chunks) {
    const int delta = d < (1 << 20) ? (int)d : 1 << 20;  // (-infinity: no finite logit, no weight)
    sm.delta[ci] = delta;
    sm.scale[ci] = y;
    sm.csum[ci] = st.total * y;
    sm.part[ci] = 0;
    if (st.depth < NB) atomicMin(&sm.depth, st.depth + delta);
    atomicAdd(&sm.number, st.number);
  }
  __syncthreads();

  Cut cut = {NB - 1, false, 0.f, 0};
  bool from_list = false;  // what is kept is listed, its weights in sm.lbin
  if (filtered) {
    const int number = sm.number, depth = sm.depth;
    double whole = (lane < chunks ? sm.csum[lane] : 0) + (64 + lane < chunks ? sm.csum[64 + lane] : 0);
    whole = sum_over_wave(whole);
    // the listed logits' bins: the row's, as far down as `depth`
#pragma unroll 1
    for (int i = tid; i < LISTED * ST; i += ST) {
      const u64 k = sm.lkey[i];
      u64 packed = (u64)NB << LBIN;  // none
      if (k) {
        const float y = key_x(k);
        const double fl = floor((double)y * sc.c);
        const int j = bin_of(ref, fl);
        const u64 f = fixed_in_bin(y, sc, fl);
        if (j <= depth) {
          packed = (u64)j << LBIN | f;
          atomicAdd(&sm.bins[j], f + (1ull << CNT));
        }
      }
      sm.lbin[i] = packed;
    }
    __syncthreads();
    {
      const u64 b = tid < NB - 1 ? sm.bins[tid] : 0;
      const double weight = tid < NB ? (double)(b & SUM_MASK) / ONE * sm.et[tid] : 0;
      double all;
      int call;
      const double upto = block_upto<SW>(weight, sm.wsum, all);
      const int cupto = block_upto<SW>((int)(b >> CNT), sm.wcount, call);
      if (tid < NB) {
        sm.upto[tid] = upto;
        sm.cupto[tid] = cupto;
      }
    }
    // the least logit with w >= min_p, and its bin
    float xm = 0;
    int jm = NB;
    const uint32_t ktop = (uint32_t)(key >> 32);
    if (min_p > 0.f) {
      const double y = (double)top + (double)T * log64(fmin((double)min_p, 1.0));
      xm = fmaxf((float)y, -3.4028234663852886e38f);
      if ((double)xm < y) xm = logit_of(logit_order(xm) + 1);  // rounded up
      jm = bin_of(ref, floor((double)xm * sc.c));
    }
    // the borders among the listed logits: by number, then by weight
    int kept = number;
    bool deep = false;
    double sum = whole;  // the candidates'
#pragma unroll 1
    for (int pass = 0; pass < 2 && !deep; ++pass) {
      const bool by_rank = pass == 0;
      if (by_rank ? top_k <= 0 || top_k >= number : !(top_p < 1.f)) continue;
      const double goal = (double)top_p * sum * (1 - SAME);
      const int j = min(cut.bin, border_bin(by_rank, top_k, goal));
      const int n = sm.cupto[j] - number_below(j);
      if (j > depth) {
        deep = true;
        break;
      }
      if (tid == 0) sm.n = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < LISTED * ST; i += ST)
        if ((int)(sm.lbin[i] >> LBIN) == j) sm.list[atomicAdd(&sm.n, 1)] = sm.lkey[i];
      __syncthreads();
      border_in_list(n, j, sc.c, sc.in, ref, by_rank, top_k - number_below(j), (goal - weight_below(j)) / sm.et[j] * ONE,
                     min(n, kept - number_below(j)), 0, 0);
      cut = {j, true, key_x(sm.key), key_v(sm.key)};
      if (by_rank) {
        kept = top_k;
        sum = weight_below(j) + (double)sm.sum / ONE * sm.et[j];
      }
      __syncthreads();
    }
    if (!deep) {
      if (jm < cut.bin || (jm == cut.bin && (!cut.part || xm > cut.x))) cut = {jm, true, xm, INT32_MAX};
      deep = cut.part && cut.bin > depth;
    }
    if (deep) {
      deep_cut(a.bins + s0 * NB, a.stat + s0, top_k <= 0 || top_k > a.list ? a.codes + s0 * SC : nullptr, chunks, x, a.vocab,
               sc.c, sc.in, ref, ktop, number, whole, top_k, top_p, xm, jm);
      __syncthreads();
      cut = sm.cut;
    } else if (cut.part) {  // the chunks' sums of what is kept: all of it is listed, a wave's 64 are of one chunk
      from_list = true;
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < LISTED * ST; i += ST) {
        const u64 k = sm.lkey[i], b = sm.lbin[i];
        const int j = (int)(b >> LBIN);
        double s = 0;
        if (j < NB && cut.keeps(j, key_x(k), key_v(k))) s = (double)(b & ((1ull << LBIN) - 1)) / ONE * sm.et[j];
        sm.lbin[i] = __builtin_bit_cast(u64, s);
        if (__builtin_amdgcn_ballot_w64(s > 0)) s = sum_over_wave(s);
        if (lane == 0) sm.lsum[i / 64] = s;
      }
      __syncthreads();
      if (tid < chunks) {
        const int n = a.list / 64;
        double s = 0;
#pragma unroll 1
        for (int i = 0; i < n; ++i) s += sm.lsum[tid * n + i];
        sm.csum[tid] = s;
      }
    }
    __syncthreads();
  }

  // the chunk of the answer: the first one whose running sum exceeds u times the whole
  if (w == 0) {
    const double c0 = 2 * lane < chunks ? sm.csum[2 * lane] : 0, c1 = 2 * lane + 1 < chunks ? sm.csum[2 * lane + 1] : 0;
    const double run = scan_wave(c0 + c1, plus<double>);
    const double z = at_lane(run, 63), goal = fmax((double)u, 0.0) * z * (1 + SAME);
    double before = __shfl_up(run, 1);
    if (lane == 0) before = 0;
    const bool h0 = c0 > 0 && before + c0 > goal, h1 = c1 > 0 && run > goal;
    const u64 hit = __builtin_amdgcn_ballot_w64(h0 || h1), some = __builtin_amdgcn_ballot_w64(c0 > 0 || c1 > 0);
    const int at = hit ? __ffsll(hit) - 1 : 63 - __clzll(some);  // none: the last one with any weight
    if (lane == at) {
      const bool second = hit ? !h0 : c1 > 0;
      sm.found = 2 * lane + second;
      sm.goal = fmax(goal - (second ? before + c0 : before), 0.0);  // (the sums before it may have been rounded up)
      sm.z = z;
      sm.first = INT32_MAX;
      sm.last = -1;
    }
  }
  __syncthreads();
  const double goal = sm.goal, z = sm.z;
  if (from_list) {  // the kept logits of the chunk in the order of their tokens: a bit map tells each its place
    const int i = sm.found * a.list + tid, first = sm.found * SC;
    double weight = tid < a.list ? __builtin_bit_cast(double, sm.lbin[i]) : 0;
    const int v = tid < a.list ? key_v(sm.lkey[i]) : 0, off = weight > 0 ? v - first : 0;
    if (tid < SC / 32) sm.map[tid] = 0;
    __syncthreads();
    if (weight > 0) atomicOr(&sm.map[off >> 5], 1u << (off & 31));
    __syncthreads();
    const uint32_t bits = tid < SC / 32 ? sm.map[tid] : 0;
    int n;
    const int place = block_before<SW>((int)__popc(bits), sm.wcount, n);
    if (tid < SC / 32) sm.mapped[tid] = place;
    __syncthreads();
    if (weight > 0) {
      const int at = sm.mapped[off >> 5] + __popc(sm.map[off >> 5] & ((1u << (off & 31)) - 1));
      sm.inorder[at] = weight;
      sm.token[at] = v;
    }
    __syncthreads();
    weight = tid < n ? sm.inorder[tid] : 0;
    double all;
    // the first one whose running sum exceeds the goal, the last one if none does
    const u64 hit = __builtin_amdgcn_ballot_w64(block_upto<SW>(weight, sm.wsum, all) > goal && tid < n);
    if (hit && lane == __ffsll(hit) - 1) atomicMin(&sm.first, tid);
    __syncthreads();
    if (tid == min(sm.first, n - 1)) {
      a.tokens[row] = sm.token[tid];
      if (a.logprobs) a.logprobs[row] = (float)fmin(log64(weight / z), 0.0);
    }
    return;
  }
  // the answer among the chunk's logits, eight to a thread
  const int v0 = sm.found * SC + 8 * tid;
  float f[8];
  if (v0 + 7 < a.vocab) {
    const f4a y0 = *reinterpret_cast<const f4a*>(x + v0), y1 = *reinterpret_cast<const f4a*>(x + v0 + 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[q] = y0[q];
      f[4 + q] = y1[q];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = v0 + q < a.vocab ? x[v0 + q] : -INFINITY;
  }
  // a thread's sum and its last logit of any weight, then, by the waves that the answer may be in, the first logit with which
  // the running sum exceeds the goal; the row's last one of any weight if none does
  double* weights = reinterpret_cast<double*>(sm.lkey) + tid;  // (and on into lbin)
  static_assert(sizeof(sm.lkey) + sizeof(sm.lbin) >= SC * sizeof(double));
  double mine = 0, all, waves;
  int last = -1;
#pragma unroll 1
  for (int q = 0; q < 8; ++q) {
    const double p = (double)f[0] * sc.c, fl = floor(p);
    const int j = bin_of(ref, fl);
    double s = 0;
    if (f[0] > -INFINITY && cut.keeps(j, f[0], v0 + q))
      s = j < NB - 1 ? (double)fixed_in_bin(f[0], sc, fl) / ONE * sm.et[j] : tail_weight(p, fl, ref);
    weights[q * ST] = s;
    mine += s;
    last = s > 0 ? v0 + q : last;
    turn(f);
  }
  const double upto = block_upto<SW>(mine, sm.wsum, all, waves);
  double run = __shfl_up(upto, 1);
  if (lane == 0) run = waves;
  const u64 some = __builtin_amdgcn_ballot_w64(last >= 0);
  if (some && lane == 63 - __clzll(some)) atomicMax(&sm.last, last);
  // Sums in another order may differ in their last digits: a little more than the thread that has it, so that one of these has
  // it wherever the goal is below all of them.
  const bool here = mine > 0 && (run + mine) * (1 + SAME) > goal && run * (1 - SAME) <= goal;
  int hit = INT32_MAX;
  if (__builtin_amdgcn_ballot_w64(here)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const double s = weights[q * ST];
      run += s;
      if (here && s > 0 && run > goal) hit = min(hit, v0 + q);
    }
  }
  if (hit < INT32_MAX) atomicMin(&sm.first, hit);
  __syncthreads();
  const int v = sm.first < INT32_MAX ? sm.first : sm.last;
  if (v >= v0 && v < v0 + 8) {
    a.tokens[row] = v;
    if (a.logprobs) a.logprobs[row] = (float)fmin(log64(weights[(v - v0) * ST] / z), 0.0);
  }
}

static size_t sample_align(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace mkp

using namespace mkp;

extern "C" size_t mk_sample_workspace_bytes(int rows, int vocab) {
  if (rows < 1 || rows > 65535 || vocab < 1 || vocab > SV_MAX) return 0;
  const size_t slots = (size_t)rows * ((vocab + SC - 1) / SC);
  return sample_align(slots * sizeof(SampleStat)) + slots * ((NB + LIST_MAX) * sizeof(u64) + SC);
}

extern "C" hipError_t mk_sample(int rows, int vocab, const float* logits, int64_t row_stride, const float* uniforms,
                                const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                int32_t* tokens, float* logprobs, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
  const size_t need = mk_sample_workspace_bytes(rows, vocab);
  if (need == 0 || row_stride < 0) return hipErrorInvalidValue;
  if (!logits || !uniforms || !temperature || !top_k || !top_p || !min_p || !tokens || !workspace) return hipErrorInvalidValue;
  if (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return hipErrorInvalidValue;
  SampleArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.vocab = vocab;
  a.chunks = (vocab + SC - 1) / SC;
  const size_t slots = (size_t)rows * a.chunks;
  char* ws = static_cast<char*>(workspace);
  a.stat = reinterpret_cast<SampleStat*>(ws);
  a.list = std::min(LIST_MAX, LISTED * ST / a.chunks & ~63);
  a.bins = reinterpret_cast<u64*>(ws + sample_align(slots * sizeof(SampleStat)));
  a.listed = a.bins + slots * NB;
  a.codes = reinterpret_cast<uint8_t*>(a.listed + slots * LIST_MAX);
  const dim3 grid(a.chunks, rows);
  // A workgroup of 16 waves to a CU at most; beyond that, smaller ones overlap better. Measured on MI355X, top 50 of 0.95, 16
  // waves and 4: 151,936 logits (19 chunks) 1 row 25.0 and 26.6 us, 13 rows 26.0 and 27.7, 20 rows 29.8 and 28.8, 64 rows
  // 45.6 and 37.9; 32,000 (4 chunks) 64 rows 23.2 and 24.6, 128 rows 27.9 and 26.6. (8 waves: within 1% of 4 at 64 rows.)
  if ((int64_t)a.chunks * rows <= 256) hipLaunchKernelGGL(sample_chunk_kernel<16>, grid, dim3(1024), 0, stream, a);
  else hipLaunchKernelGGL(sample_chunk_kernel<4>, grid, dim3(256), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(rows), dim3(ST), 0, stream, a);
  return hipGetLastError();
}
