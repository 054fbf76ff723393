// Sampling from the logits with temperature, top-k, top-p and min-p and a given random number a row, on MI355X
// (gfx950). With w = exp((x - max) / T):
//   candidates  the top_k largest logits; of these, in order, the fewest whose w reach top_p of their sum; of these
//               those with w >= min_p. Equal logits: the lower token first. All three are one cut (x, token) in the
//               order of the logits;
//   answer      the first token of the vocabulary at which the running sum of the candidates' w exceeds u times
//               their whole sum.
// The answer is a whole number that a border may decide, so sums are exact ones of w rounded to 2^-43 of itself, and two
// sums within SAME of each other count as equal: 5 of 10 equal logits reach half of them, and do not exceed it.
//
// Bins. p = x * 16 / T falls into bin floor(p), the same for equal logits wherever they are, and within its bin
// w is exp((p - floor(p)) / 16), a polynomial on [1, 1.065), kept as a whole number of 2^-43: a bin's sum is a sum of
// whole numbers, the same in any order, and its weight that sum times exp(bin / 16).
//   sample_chunk_kernel  a workgroup takes 8,192 logits of a row from registers into 512 bins (32 in units of T) below
//                        their maximum: number and sum of each; what lies lower is a tail of its own;
//   sample_pick_kernel   a workgroup per row joins the chunks' bins, finds the bin that a border falls into, gathers
//                        and sorts that bin's logits (narrowing it first where it holds more than 4,096), takes the
//                        chunks' sums from their bins, and looks for the answer among the 8,192 logits of its chunk.
// No logit but those of the border's bin and of the answer's chunk is looked at twice in full.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mk_device.h"
#include "mk_layers.h"
#include "../../include/megakernel_amd.h"

namespace mkp {

constexpr int SL = 2048;            // logits per wave of the first kernel
constexpr int SC = 4 * SL;          // and per workgroup: a chunk
constexpr int SV_MAX = 1 << 20;
constexpr int SCH = SV_MAX / SC;    // chunks of a row at most
constexpr int NB = 512;             // bins; the last one is the tail
constexpr double RES = 16;          // bins per unit of x / T
constexpr int FIX = 43;             // bits behind the point of a weight within its bin
constexpr double SAME = 1.0 / (1ull << 42);
constexpr int CAP = 4096;           // logits that are sorted
constexpr int SUB = 2048;           // narrower bins of a bin that holds more
constexpr int PT = 1024;            // threads of the second kernel

typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any element

struct SampleStat {
  double ref;   // the bin of the chunk's maximum; -infinity: no finite logit
  double tail;  // the weights below the bins, in units of exp(ref / 16)
  u64 key;      // the largest logit, the lowest token of equal ones
  int32_t tail_count, bad;
};

struct SampleArgs {
  const float* logits;
  int64_t row_stride;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprobs;
  int vocab, chunks;
  SampleStat* stat;  // [rows][chunks]
  u64* sum;          // [rows][chunks][NB]
  uint32_t* count;   // [rows][chunks][NB]
};

__device__ __forceinline__ uint32_t logit_order(float x) {  // unsigned order is the numbers'
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 logit_key(float x, int v) { return (u64)logit_order(x) << 32 | (0xffffffffu - (uint32_t)v); }
__device__ __forceinline__ int token_of(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

__device__ __forceinline__ double sum_over_wave(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// exp(f / 16) for f in [0, 1]: the series about 1/32, whose next term is below 2^-47
__device__ __forceinline__ double exp_in_bin(double f) {
  constexpr double A = 1.0 / 16, E = 1.0317434074991028;  // exp(1/32)
  const double g = f - 0.5;
  double y = E * A * A * A * A * A * A / 720;
  y = fma(y, g, E * A * A * A * A * A / 120);
  y = fma(y, g, E * A * A * A * A / 24);
  y = fma(y, g, E * A * A * A / 6);
  y = fma(y, g, E * A * A / 2);
  y = fma(y, g, E * A);
  return fma(y, g, E);
}
// the same as a whole number of 2^-FIX
__device__ __forceinline__ u64 fixed_in_bin(double f) {
  const u64 b = __builtin_bit_cast(u64, exp_in_bin(f));  // in [1, 2)
  return (((b & 0xfffffffffffffull) | 1ull << 52) + (1ull << (51 - FIX))) >> (52 - FIX);
}
// The place of a logit in its bin. Above 2^53 p has no digits behind the point, and different logits lie in bins far
// from each other's: any number serves.
__device__ __forceinline__ double in_bin(float x, double c, double fl) {
  return fmin(fmax(fma((double)x, c, -fl), 0.0), 1.0);
}
// exp(t / 16) for t <= 0 to fp32's accuracy, over the doubles' range: the tail's weights, below exp(-31) of the largest
__device__ __forceinline__ double exp_tail(double t) {
  const double p = t * (1.4426950408889634 / RES), n = floor(fmax(p, -1100.0));
  return ldexp((double)__builtin_amdgcn_exp2f((float)fmax(p - n, 0.0)), (int)n);
}

__global__ void __launch_bounds__(256) sample_chunk_kernel(const SampleArgs a) {
  __shared__ u64 sum[NB];
  __shared__ uint32_t count[NB];
  __shared__ u64 skey[4];
  __shared__ double stail[4];
  __shared__ int sbad[4], stc[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.y, v0 = blockIdx.x * SC + w * SL + 4 * lane;  // this lane's logits: v0 + 256 j + q
  const float* x = a.logits + row * a.row_stride;
  const float T = a.temperature[row];
  float f[SL / 64];
#pragma unroll
  for (int j = 0; j < SL / 256; ++j) {
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
  for (int i = tid; i < NB; i += 256) {
    sum[i] = 0;
    count[i] = 0;
  }
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < SL / 64; ++i) {
    m = fmaxf(m, f[i]);
    bad |= !(f[i] < INFINITY);  // NaN too
  }
  int at = INT32_MAX;
#pragma unroll
  for (int i = SL / 64 - 1; i >= 0; --i)
    if (f[i] == m) at = v0 + 256 * (i >> 2) + (i & 3);
  u64 key = logit_key(m, min(at, SV_MAX));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 y = __shfl_xor(key, o);
    key = key > y ? key : y;
  }
  if (lane == 0) skey[w] = key;
  const bool wbad = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (lane == 0) sbad[w] = wbad;
  __syncthreads();
  key = max(max(skey[0], skey[1]), max(skey[2], skey[3]));
  const float top = logit_of((uint32_t)(key >> 32));
  const bool empty = top == -INFINITY;
  const double c = RES / (double)T;
  const double ref = empty ? -INFINITY : floor((double)top * c);
  double tail = 0;
  int tc = 0;
  if (T > 0.f && !empty) {
#pragma unroll
    for (int i = 0; i < SL / 64; ++i) {
      const double p = (double)f[i] * c, fl = floor(p);
      const double k = ref - fl;
      if (k < NB - 1) {
        atomicAdd(&sum[(int)k], fixed_in_bin(in_bin(f[i], c, fl)));
        atomicAdd(&count[(int)k], 1u);
      } else if (f[i] > -INFINITY) {
        tail += exp_tail(p - ref);
        ++tc;
      }
    }
  }
  tail = sum_over_wave(tail);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) tc += __shfl_xor(tc, o);
  if (lane == 0) {
    stail[w] = tail;
    stc[w] = tc;
  }
  __syncthreads();
  const int64_t slot = (int64_t)row * a.chunks + blockIdx.x;
  for (int i = tid; i < NB; i += 256) {
    a.sum[slot * NB + i] = sum[i];
    a.count[slot * NB + i] = count[i];
  }
  if (tid == 0) {
    SampleStat s;
    s.ref = ref;
    s.tail = (stail[0] + stail[1]) + (stail[2] + stail[3]);
    s.key = key;
    s.tail_count = stc[0] + stc[1] + stc[2] + stc[3];
    s.bad = sbad[0] | sbad[1] | sbad[2] | sbad[3];
    a.stat[slot] = s;
  }
}

// The least u32 in [lo, hi] for which `test`, false up to some number and true from there on, is true (hi, if none
// below it is): by all lanes of a wave, 64 places at a time.
template <typename F>
__device__ __forceinline__ uint32_t least_true(uint32_t lo, uint32_t hi, F test) {
  const int lane = threadIdx.x & 63;
  uint64_t a = lo, n = (uint64_t)hi - lo;  // the answer lies in [a, a + n]
  while (n > 0) {
    const uint64_t step = (n + 63) / 64;  // places a + step - 1, a + 2 step - 1, ...: is it at or before there?
    const uint64_t at = a + (lane + 1) * step - 1;
    const u64 hit = __builtin_amdgcn_ballot_w64(at >= a + n || test((uint32_t)at));
    const int first = hit ? __ffsll(hit) - 1 : 64;
    const uint64_t end = a + n;
    a += first * step;
    n = min((uint64_t)(step - 1), end - a);
    if (a > end) { a = end; n = 0; }
  }
  return (uint32_t)a;
}

struct PickSmem {
  double et[NB];        // exp(-j / 16)
  double upto[NB];      // weights of bins 0 .. j
  int32_t cupto[NB];    // their logits
  int32_t delta[SCH];   // bins of the row above the chunk's first (at most 2^20)
  double scale[SCH], ref[SCH], tail[SCH], csum[SCH];
  int32_t tcount[SCH];
  u64 part[SCH];        // kept weights of the border's bin, by chunk
  union {
    u64 list[CAP];
    struct {
      u64 sum[SUB];
      uint32_t count[SUB];
    } sub;
    struct {
      u64 sum[NB];
      int32_t count[NB];
      double tail[PT / 64];
      int32_t tcount[PT / 64];
    } half;
  };
  double wsum[PT / 64];
  int32_t wcount[PT / 64];
  u64 wfix[PT / 64];
  int found, n, last;
  uint32_t klo, khi;
  double w0;
};

// Sums over the threads before this one and over all (numbers that commute exactly, or in the threads' order).
template <typename V>
__device__ __forceinline__ V block_before(V v, V* lds, V& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  V x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) lds[w] = x;
  __syncthreads();
  V before = 0, all = 0;
  for (int i = 0; i < PT / 64; ++i) {
    if (i == w) before = all;
    all += lds[i];
  }
  total = all;
  return before + (x - v);
}

// A row's border: kept are bins 0 .. bin - 1 and, of bin `bin`, all (part false) or the logits above x and those
// equal to it up to token i.
struct Cut {
  int bin;
  bool part;
  float x;
  int token;
};

struct Row {
  const float* x;
  int vocab, chunks;
  double c, ref;  // bins per logit; the bin of the largest
  uint32_t ktop, kmin;
};

// fn(logit, token) for every logit of the row whose order's number lies in [lo, hi], by the whole workgroup.
template <typename F>
__device__ __forceinline__ void sweep(const Row& r, uint32_t lo, uint32_t hi, F fn) {
  const int tid = threadIdx.x;
  for (int base = 0; base < r.vocab; base += 8 * 4 * PT) {
    float f[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int v = base + 4 * PT * j + 4 * tid;
      if (v + 3 < r.vocab) {
        const f4a t = *reinterpret_cast<const f4a*>(r.x + v);
#pragma unroll
        for (int q = 0; q < 4; ++q) f[j][q] = t[q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) f[j][q] = v + q < r.vocab ? r.x[v + q] : -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t o = logit_order(f[j][q]);  // not the numbers: -0 and 0 are one number, and one place alone
        if (o >= lo && o <= hi) fn(f[j][q], base + 4 * PT * j + 4 * tid + q);
      }
  }
}

// The weight of a logit of bin j (the row's), in 2^-FIX of exp(-j / 16).
__device__ __forceinline__ u64 fixed_weight(const Row& r, float x, int j) {
  const double p = (double)x * r.c, fl = floor(p);
  if (j == NB - 1) return (u64)(exp_tail(p - r.ref + (NB - 1)) * (double)(1ull << FIX));
  return fixed_in_bin(in_bin(x, r.c, fl));
}

// The order's numbers of bin j's logits, by wave 0.
__device__ __forceinline__ void bin_range(const Row& r, int j, PickSmem& sm) {
  if (threadIdx.x < 64) {
    auto from = [&](double b) {  // the least logit of bin b or above
      return least_true(r.kmin, r.ktop, [&](uint32_t k) { return floor((double)logit_of(k) * r.c) >= b; });
    };
    const uint32_t lo = j == NB - 1 ? r.kmin : from(r.ref - j);
    const uint32_t hi = j == 0 ? r.ktop : from(r.ref - (j - 1)) - 1;
    if (threadIdx.x == 0) {
      sm.klo = lo;
      sm.khi = hi;
    }
  }
  __syncthreads();
}

// Gathers the logits of the order's numbers [klo, khi] (n <= CAP of them) and sorts them, the first of the order first.
__device__ __forceinline__ void gather(const Row& r, uint32_t klo, uint32_t khi, int n, PickSmem& sm) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) sm.n = 0;
  __syncthreads();
  sweep(r, klo, khi, [&](float x, int v) {
    const int at = atomicAdd(&sm.n, 1);
    if (at < CAP) sm.list[at] = logit_key(x, v);
  });
  __syncthreads();
  const int got = min(sm.n, CAP);  // n
  int size = 64;
  while (size < max(n, got)) size *= 2;
  for (int i = got + tid; i < size; i += PT) sm.list[i] = 0;
  __syncthreads();
  if (size <= 256) {  // a key's place is how many are larger: four lanes to a key
    const int i = tid >> 2;
    u64 key = 0;
    int place = 0;
    if (i < n) {
      key = sm.list[i];
      for (int e = tid & 3; e < n; e += 4) place += sm.list[e] > key;
    }
    place += __shfl_xor(place, 1);
    place += __shfl_xor(place, 2);
    __syncthreads();
    if (i < n && (tid & 3) == 0) sm.list[place] = key;
    __syncthreads();
    return;
  }
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int p = tid; p < size / 2; p += PT) {
        const int lo = 2 * p - (p & (j - 1)), hi = lo + j;
        const u64 a = sm.list[lo], b = sm.list[hi];
        if ((a < b) == ((lo & k) == 0)) {
          sm.list[lo] = b;
          sm.list[hi] = a;
        }
      }
      __syncthreads();
    }
}

// Finds the border within bin j: the first of its logits, in order, at which their number reaches `rank` (by_rank), or
// their sum reaches `goal` (in 2^-FIX of the bin's unit; the last of `most` logits, if none of them does). Returns
// the sum up to it. Leaves the list of the whole bin where it holds no more than CAP (listed).
__device__ u64 border_in_bin(const Row& r, int j, int count, bool by_rank, int rank, double goal, int most, bool& listed,
                             Cut& cut, PickSmem& sm) {
  const int tid = threadIdx.x;
  bin_range(r, j, sm);
  uint32_t klo = sm.klo, khi = sm.khi;
  int n = count, above = 0;  // logits in [klo, khi], and of the bin above khi
  u64 sabove = 0;
  listed = n <= CAP;
  while (n > CAP && klo < khi) {  // narrow: SUB bins of the order's numbers, the first of the order first
    int shift = 0;
    while (((khi - klo) >> shift) >= SUB) ++shift;
    __syncthreads();
    for (int i = tid; i < SUB; i += PT) {
      sm.sub.sum[i] = 0;
      sm.sub.count[i] = 0;
    }
    if (tid == 0) sm.found = SUB - 1;
    __syncthreads();
    sweep(r, klo, khi, [&](float x, int) {
      const uint32_t b = (khi - logit_order(x)) >> shift;
      atomicAdd(&sm.sub.count[b], 1u);
      atomicAdd(&sm.sub.sum[b], fixed_weight(r, x, j));
    });
    __syncthreads();
    int c0 = (int)sm.sub.count[2 * tid], c1 = (int)sm.sub.count[2 * tid + 1], call;
    u64 s0 = sm.sub.sum[2 * tid], s1 = sm.sub.sum[2 * tid + 1], sall;
    const int cb = above + block_before<int32_t>(c0 + c1, sm.wcount, call);
    const u64 sb = sabove + block_before<u64>(s0 + s1, sm.wfix, sall);
    auto reached = [&](int number, u64 sum) { return by_rank ? number >= rank : (double)sum >= goal || number >= most; };
    if (reached(cb + c0, sb + s0)) atomicMin(&sm.found, 2 * tid);
    else if (reached(cb + c0 + c1, sb + s0 + s1)) atomicMin(&sm.found, 2 * tid + 1);
    __syncthreads();
    const int b = min(sm.found, (int)((khi - klo) >> shift));
    if (tid == b / 2) {
      sm.n = b & 1 ? c1 : c0;
      sm.last = b & 1 ? cb + c0 : cb;
      sm.wfix[0] = b & 1 ? sb + s0 : sb;
    }
    __syncthreads();
    n = sm.n;
    above = sm.last;
    sabove = sm.wfix[0];
    const uint32_t top = khi - ((uint32_t)b << shift);
    const uint32_t width = (1u << shift) - 1;
    klo = top - klo > width ? top - width : klo;
    khi = top;
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
    for (int base = 0; base < r.vocab && seen < take; base += 4 * PT) {
      int mine = 0, all;
      for (int q = 0; q < 4; ++q) {
        const int v = base + 4 * tid + q;
        mine += v < r.vocab && r.x[v] == x;
      }
      int before = seen + block_before<int32_t>(mine, sm.wcount, all);
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
  gather(r, klo, khi, n, sm);
  // running sums of the sorted logits, four to a thread
  u64 s[4], mine = 0, all;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * tid + q;
    s[q] = i < n ? fixed_weight(r, logit_of((uint32_t)(sm.list[i] >> 32)), j) : 0;
    mine += s[q];
  }
  if (tid == 0) sm.found = max(0, min(n, most - above) - 1);
  u64 run = sabove + block_before<u64>(mine, sm.wfix, all);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * tid + q;
    run += s[q];
    s[q] = run;
    if (i < n && (by_rank ? above + i + 1 >= rank : (double)run >= goal)) atomicMin(&sm.found, i);
  }
  __syncthreads();
  const int at = sm.found;
  if (tid == at / 4) sm.wfix[0] = at % 4 == 0 ? s[0] : at % 4 == 1 ? s[1] : at % 4 == 2 ? s[2] : s[3];
  const u64 key = sm.list[at];
  __syncthreads();
  cut = {j, true, logit_of((uint32_t)(key >> 32)), token_of(key)};
  return sm.wfix[0];
}

__global__ void __launch_bounds__(PT) sample_pick_kernel(const SampleArgs a) {
  __shared__ PickSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x, chunks = a.chunks;
  const int64_t s0 = (int64_t)row * chunks;
  const float T = a.temperature[row], u = a.uniforms[row], top_p = a.top_p[row], min_p = a.min_p[row];
  const int top_k = a.top_k[row];
  auto answer = [&](int token, float logprob) {
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = logprob;
  };
  // the row's maximum, and what is wrong with it
  u64 key = 0;
  int bad = 0;
  double ref = -INFINITY;
  for (int i = lane; i < chunks; i += 64) {  // every wave for itself
    const SampleStat s = a.stat[s0 + i];
    key = key > s.key ? key : s.key;
    bad |= s.bad;
    ref = fmax(ref, s.ref);
    if (w == 0) {
      sm.ref[i] = s.ref;
      sm.tail[i] = s.tail;
      sm.tcount[i] = s.tail_count;
      sm.part[i] = 0;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 y = __shfl_xor(key, o);
    key = key > y ? key : y;
    bad |= __shfl_xor(bad, o);
    ref = fmax(ref, __shfl_xor(ref, o));
  }
  const float top = logit_of((uint32_t)(key >> 32));
  if (bad || top == -INFINITY || !(T >= 0.f && T < INFINITY) || u != u || top_p != top_p || min_p != min_p) {
    if (tid == 0) answer(-1, __builtin_nanf(""));
    return;
  }
  if (T == 0.f) {
    if (tid == 0) answer(token_of(key), 0.f);
    return;
  }
  Row r;
  r.x = a.logits + row * a.row_stride;
  r.vocab = a.vocab;
  r.chunks = chunks;
  r.c = RES / (double)T;
  r.ref = ref;
  r.ktop = (uint32_t)(key >> 32);
  r.kmin = logit_order(-3.4028234663852886e38f);
  if (tid < NB) sm.et[tid] = exp(-tid / RES);
  __syncthreads();
  if (tid < chunks) {
    const double d = ref - sm.ref[tid];
    sm.delta[tid] = d < (1 << 20) ? (int)d : 1 << 20;
    sm.scale[tid] = exp(-d / RES);
  }
  __syncthreads();

  // the chunks' bins joined: two threads to a bin
  {
    constexpr double UNIT = 1.0 / (double)(1ull << FIX);
    const int j = tid % NB, half = tid / NB;
    u64 s = 0;
    int n = 0, tn = 0;
    double t = 0;
    for (int c = half; c < chunks; c += PT / NB) {
      const int d = sm.delta[c];
      if (j >= d && j - d < NB - 1) {
        s += a.sum[(s0 + c) * NB + j - d];
        n += (int)a.count[(s0 + c) * NB + j - d];
      }
      if (j < NB - 1 && j + d >= NB - 1) {  // the chunk's bin lies in the row's tail
        t += (double)a.sum[(s0 + c) * NB + j] * UNIT * (sm.et[j] * sm.scale[c]);
        tn += (int)a.count[(s0 + c) * NB + j];
      }
      if (j == NB - 1) {
        t += sm.tail[c] * sm.scale[c];
        tn += sm.tcount[c];
      }
    }
    t = sum_over_wave(t);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) tn += __shfl_xor(tn, o);
    if (lane == 0) {
      sm.half.tail[w] = t;
      sm.half.tcount[w] = tn;
    }
    if (half) {
      sm.half.sum[j] = s;
      sm.half.count[j] = n;
    }
    __syncthreads();
    double weight = 0;
    if (!half) {
      s += sm.half.sum[j];
      n += sm.half.count[j];
      weight = (double)s * UNIT * sm.et[j];
      if (j == NB - 1) {
        weight = 0;
        n = 0;
        for (int i = 0; i < PT / 64; ++i) {
          weight += sm.half.tail[i];
          n += sm.half.tcount[i];
        }
      }
    } else {
      n = 0;
    }
    double all;
    int call;
    const double wb = block_before<double>(weight, sm.wsum, all);
    const int cb = block_before<int32_t>(n, sm.wcount, call);
    if (!half) {
      sm.upto[j] = wb + weight;
      sm.cupto[j] = cb + n;
    }
    __syncthreads();
  }
  const int number = sm.cupto[NB - 1];
  constexpr double ONE = (double)(1ull << FIX);
  auto below = [&](int j) { return j > 0 ? sm.upto[j - 1] : 0.0; };
  auto cbelow = [&](int j) { return j > 0 ? sm.cupto[j - 1] : 0; };
  auto first_bin = [&](auto test) {  // the first bin that passes, the last one if none does
    __syncthreads();
    if (tid == 0) sm.found = NB - 1;
    __syncthreads();
    if (tid < NB && test(tid)) atomicMin(&sm.found, tid);
    __syncthreads();
    return sm.found;
  };

  Cut cut = {NB - 1, false, 0.f, 0};
  double whole = sm.upto[NB - 1];  // the candidates' sum
  int listed = -1, kept = number;  // the bin whose logits the list holds; candidates
  if (top_k > 0 && top_k < number) {
    const int j = first_bin([&](int i) { return sm.cupto[i] >= top_k; });
    const int rank = top_k - cbelow(j), n = sm.cupto[j] - cbelow(j);
    kept = top_k;
    if (rank == n) {
      cut.bin = j;
      whole = sm.upto[j];
    } else {
      bool l;
      const u64 s = border_in_bin(r, j, n, true, rank, 0, INT32_MAX, l, cut, sm);
      listed = l ? j : -1;
      whole = below(j) + (double)s / ONE * sm.et[j];
    }
  }
  if (top_p < 1.f) {
    const double goal = (double)top_p * whole * (1 - SAME);
    const int j = min(cut.bin, first_bin([&](int i) { return sm.cupto[i] > 0 && sm.upto[i] >= goal; }));
    const int n = sm.cupto[j] - cbelow(j);
    bool l;
    border_in_bin(r, j, n, false, 0, (goal - below(j)) / sm.et[j] * ONE, min(n, kept - cbelow(j)), l, cut, sm);
    listed = l ? j : -1;
  }
  if (min_p > 0.f) {
    // the least logit with w >= min_p, and its bin
    if (tid < 64) {
      const double lim = fmin((double)min_p, 1.0);
      const uint32_t k = least_true(r.kmin, r.ktop, [&](uint32_t o) {
        return exp(((double)logit_of(o) - (double)top) / (double)T) >= lim;
      });
      if (tid == 0) sm.klo = k;
    }
    __syncthreads();
    const float x = logit_of(sm.klo);
    const double d = ref - floor((double)x * r.c);
    const int j = d < NB - 1 ? (int)d : NB - 1;
    if (j < cut.bin || (j == cut.bin && (!cut.part || x > cut.x))) cut = {j, true, x, INT32_MAX};
  }

  // the kept weights of the border's bin, by chunk
  if (cut.part) {
    const int j = cut.bin, n = sm.cupto[j] - cbelow(j);
    if (n <= CAP) {
      if (listed != j) {
        bin_range(r, j, sm);
        gather(r, sm.klo, sm.khi, n, sm);
      }
      for (int i = tid; i < n; i += PT) {
        const float x = logit_of((uint32_t)(sm.list[i] >> 32));
        const int v = token_of(sm.list[i]);
        if (x > cut.x || (x == cut.x && v <= cut.token)) atomicAdd(&sm.part[v / SC], fixed_weight(r, x, j));
      }
    } else {
      bin_range(r, j, sm);
      sweep(r, logit_order(cut.x), sm.khi, [&](float x, int v) {
        if (x > cut.x || v <= cut.token) atomicAdd(&sm.part[v / SC], fixed_weight(r, x, j));
      });
    }
  }
  __syncthreads();

  // the chunks' sums: a wave to a chunk
  const int full = cut.part ? cut.bin : cut.bin + 1;  // bins kept in full
  for (int c = w; c < chunks; c += PT / 64) {
    const int d = sm.delta[c];
    double s = 0;
    for (int j = lane; j < NB - 1; j += 64)
      if (full == NB || j + d < full) s += (double)a.sum[(s0 + c) * NB + j] / ONE * (sm.et[j] * sm.scale[c]);
    s = sum_over_wave(s);
    if (full == NB) s += sm.tail[c] * sm.scale[c];
    if (cut.part) s += (double)sm.part[c] / ONE * sm.et[cut.bin];
    if (lane == 0) sm.csum[c] = s;
  }
  __syncthreads();
  if (tid == 0) {
    double z = 0;
    for (int c = 0; c < chunks; ++c) z += sm.csum[c];
    const double goal = (double)u * z * (1 + SAME);
    double before = 0;
    int at = 0;
    double at_before = 0;
    for (int c = 0; c < chunks; ++c) {
      if (sm.csum[c] > 0) {
        at = c;
        at_before = before;
        if (before + sm.csum[c] > goal) break;
      }
      before += sm.csum[c];
    }
    sm.found = at;
    sm.w0 = goal - at_before;
    sm.upto[0] = z;
    sm.n = INT32_MAX;
    sm.last = -1;
  }
  __syncthreads();
  // the answer among the chunk's logits, eight to a thread
  const int v0 = sm.found * SC + 8 * tid;
  const double goal = sm.w0, z = sm.upto[0];
  double s[8], mine = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float x = v0 + q < a.vocab ? r.x[v0 + q] : -INFINITY;
    const double fl = floor((double)x * r.c), d = ref - fl;
    double weight = 0;
    if (x > -INFINITY) {
      const int j = d < NB - 1 ? (int)d : NB - 1;
      if (j < full || (cut.part && j == cut.bin && (x > cut.x || (x == cut.x && v0 + q <= cut.token))))
        weight = j < NB - 1 ? exp_in_bin(in_bin(x, r.c, fl)) * sm.et[j] : exp_tail((double)x * r.c - ref);
    }
    s[q] = weight;
    mine += weight;
  }
  double all;
  double run = block_before<double>(mine, sm.wsum, all);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    run += s[q];
    if (s[q] > 0) {
      if (run > goal) atomicMin(&sm.n, v0 + q);
      atomicMax(&sm.last, v0 + q);
    }
  }
  __syncthreads();
  const int v = sm.n < INT32_MAX ? sm.n : sm.last;
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if (v0 + q == v) answer(v, (float)fmin(log(s[q]) - log(z), 0.0));
}

static size_t sample_align(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace mkp

using namespace mkp;

extern "C" size_t mk_sample_workspace_bytes(int rows, int vocab) {
  if (rows < 1 || rows > 65535 || vocab < 1 || vocab > SV_MAX) return 0;
  const size_t slots = (size_t)rows * ((vocab + SC - 1) / SC);
  return sample_align(slots * sizeof(SampleStat)) + slots * NB * (sizeof(u64) + sizeof(uint32_t));
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
  a.sum = reinterpret_cast<u64*>(ws + sample_align(slots * sizeof(SampleStat)));
  a.count = reinterpret_cast<uint32_t*>(a.sum + slots * NB);
  hipLaunchKernelGGL(sample_chunk_kernel, dim3(a.chunks, rows), dim3(256), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(rows), dim3(PT), 0, stream, a);
  return hipGetLastError();
}
