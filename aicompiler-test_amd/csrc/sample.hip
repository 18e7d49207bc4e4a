// A token per row of logits [rows, vocabulary] by temperature, top-k, top-p and
// min-p from a given random number, and its probability.
//
// With m = max x and w_i = exp((x_i - m) / temperature), tokens ranked by logit
// (equals by the lower index):
//   top-k keeps the first k; top-p, of these, each one before which less than
//   top_p of their sum lies; min-p, of these, those with w >= min_p;
// the token is the first kept one, in the order of the vocabulary, at which the
// running sum passes u times the sum of all kept.
//
// Sums must come out alike in every run, and close enough that a draw next to a border
// falls on its right side: a weight is 2^a with a in 64 bits, and sums are of 64-bit
// integers (multiples of 2^-scale of the greatest weight), in any order, or of 64-bit
// floats, in a fixed one.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>

// (a lambda that is not inlined keeps what it refers to in memory)
#define TMC_INLINE __attribute__((always_inline))

namespace tmc {
namespace {

typedef unsigned long long u64;

// What a block of a shared row leaves to the last of them.
struct SampleRecord {
  u64 best;    // greatest rank key
  double sum;  // of weights, relative to its greatest logit
};

struct SampleParams {
  const void* logits;
  const float* temperature;  // [rows] each, or null
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;
  int32_t* tokens;
  float* probability;  // or null
  long stride;
  int rows, vocab;
  int scale;            // integer weights are multiples of 2^-scale
  int count, walk;      // blocks a row, parts of a row that each takes
  SampleRecord* parts;  // of shared rows: [rows][count]
  u64* bins;            // [rows][count][kBins]
  int* arrivals;        // [rows], kCounterStride apart
};

// Below it a temperature counts as 0: the most probable token.
constexpr float kColdest = 1.0f / 65536.0f;

// log2 of the least weight that counts: what lies below it, of 2^20 tokens, is less
// than half the distance of two 24-bit random numbers near 1.
constexpr double kFaintest = -44.0;
constexpr int64_t kMostTokens = 1 << 20;

// A logit and its index as one number, the higher ranked greater (-0 as +0; no
// NaN).
__device__ __forceinline__ u64 rank_key(float v, int index) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);
  const unsigned order = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)order << 32 | (unsigned)~index;
}
__device__ __forceinline__ int key_index(u64 key) { return (int)~(unsigned)key; }
__device__ __forceinline__ float key_value(u64 key) {
  const unsigned order = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

struct Settings {
  double heat;   // log2(e) / temperature; 0: take the most probable token
  double least;  // log2 of min_p
  float share;   // top_p, 1 for all
  double uniform;
  int most;      // top_k, the vocabulary for all
};
__device__ __forceinline__ Settings settings_of(const SampleParams& p, int row) {
  const float t = p.temperature ? p.temperature[row] : 1.0f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float share = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p ? p.min_p[row] : 0.0f;
  Settings s;
  const double u = p.uniforms[row];
  s.uniform = u > 0.0 ? fmin(u, 1.0) : 0.0;  // (NaN: 0)
  s.heat = t >= kColdest ? 1.4426950408889634 / (double)t : 0.0;
  if (t == INFINITY) s.heat = 0x1p-1000;  // equal weights
  s.least = least > 0.0f ? log2((double)fminf(least, 1.0f)) : -INFINITY;
  s.share = share < 1.0f ? fmaxf(share, 0.0f) : 1.0f;
  s.most = k > 0 && k < p.vocab ? k : p.vocab;
  return s;
}

// ------------------------------------------------------------ shared by both ways
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

constexpr int kDigits = 256;
// A row's tokens are looked at bin by bin: 1/16 octave of the weight each, down to
// kFaintest.
constexpr int kBinsOctave = 16, kBins = 44 * kBinsOctave;
static_assert(kFaintest == -44.0, "bins down to the least weight");
constexpr int kMostKept = 2048, kMostTopK = 1024;  // tokens in the list, top_k that goes by it
constexpr int kMostGroups = 4096;                  // sums of a wave's loads in a block's part

template <int THREADS> struct SampleScratch {
  u64 hist[kBins > kDigits ? kBins : kDigits];
  u64 keys[kMostKept];
  double groups[kMostGroups];
  double wave[THREADS / kWave];
  u64 words[THREADS / kWave];
  double value;
  u64 found64, below;
  int found, count, last;
};

template <int THREADS>
__device__ __forceinline__ u64 block_sum_u64(u64 v, SampleScratch<THREADS>& s) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) s.words[threadIdx.x / kWave] = v;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) sum += s.words[w];
  return sum;
}
template <int THREADS>
__device__ __forceinline__ u64 block_max_u64(u64 v, SampleScratch<THREADS>& s) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v = max(v, (u64)__shfl_xor(v, off, kWave));
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) s.words[threadIdx.x / kWave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) v = max(v, s.words[w]);
  return v;
}

// 2^a for a <= 0: Taylor's series of e^z, |z| <= ln 2 / 2, up to z^11: its rest is below
// 2^-47 of it.
__device__ __forceinline__ double exp2_of(double a) {
  const double n = rint(a), z = (a - n) * 0.6931471805599453;
  double s = 1.0 / 39916800.0;
  s = fma(s, z, 1.0 / 3628800.0);
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, 1.0 / 40320.0);
  s = fma(s, z, 1.0 / 5040.0);
  s = fma(s, z, 1.0 / 720.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, 1.0 / 24.0);
  s = fma(s, z, 1.0 / 6.0);
  s = fma(s, z, 0.5);
  s = fma(s, z, 1.0);
  s = fma(s, z, 1.0);
  return ldexp(s, (int)n);
}

// ------------------------------------------------------------ any row
// The key at which the running cost, from the highest ranked down, reaches
// `target` (at least 1 and at most all of it): digit by digit, a histogram of the
// costs of the keys that agree so far.
template <int THREADS, typename EACH>
__device__ u64 cut_at(u64 target, SampleScratch<THREADS>& s, const EACH& each) {
  u64 prefix = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += THREADS) s.hist[d] = 0;
    __syncthreads();
    each([&](u64 key, u64 cost) {
      if (shift == 56 || key >> (shift + 8) == prefix >> (shift + 8))
        atomicAdd(&s.hist[key >> shift & 255], cost);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 above = 0;
      int d = kDigits - 1;
      while (d > 0 && above + s.hist[d] < target) above += s.hist[d--];
      s.found64 = d;
      s.below = target - above;
    }
    __syncthreads();
    prefix |= s.found64 << shift;
    target = s.below;
  }
  return prefix;
}

// A row by one block, whatever it holds, pass after pass over memory: weights as
// integers, cuts by their digits.  20 to 40 us a pass of a row of 32000, 5 to 25
// passes.
template <typename T, int THREADS>
__device__ void row_by_digits(const SampleParams& p, int row, const Settings& set,
                              SampleScratch<THREADS>& s) {
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  // ---- the most probable token
  u64 best = 0;
  for (int i = threadIdx.x; i < p.vocab; i += THREADS) {
    const float v = (float)x[i];
    if (v == v) best = max(best, rank_key(v, i));
  }
  best = block_max_u64<THREADS>(best, s);
  const float top = key_value(best);
  if (set.heat == 0.0 || best == 0 || top == -INFINITY) {
    if (threadIdx.x == 0) {
      p.tokens[row] = best ? key_index(best) : -1;
      if (p.probability)
        p.probability[row] = set.heat == 0.0 && best ? 1.0f : __builtin_nanf("");
    }
    return;
  }
  const double unit = ldexp(1.0, p.scale);
  auto weight = [&](float v) -> u64 {
    if (v == top) return (u64)unit;
    if (!(v > -INFINITY) || top == INFINITY) return 0;
    const double a = ((double)v - (double)top) * set.heat;
    return a >= kFaintest ? max((u64)rint(exp2_of(a) * unit), (u64)1) : 0;
  };
  u64 cut = 0;
  auto kept = [&](float v, int i) -> u64 {
    const u64 w = weight(v);
    return w && rank_key(v, i) >= cut ? w : 0;
  };
  if (set.most < p.vocab) {
    auto each = [&](auto&& take) {
      for (int i = threadIdx.x; i < p.vocab; i += THREADS) {
        const float v = (float)x[i];
        if (weight(v)) take(rank_key(v, i), 1);
      }
    };
    u64 count = 0;
    each([&](u64, u64 one) { count += one; });
    if (block_sum_u64<THREADS>(count, s) > (u64)set.most) cut = cut_at<THREADS>((u64)set.most, s, each);
  }
  if (set.share < 1.0f) {
    auto each = [&](auto&& take) {
      for (int i = threadIdx.x; i < p.vocab; i += THREADS) {
        const float v = (float)x[i];
        if (const u64 w = kept(v, i)) take(rank_key(v, i), w);
      }
    };
    u64 sum = 0;
    each([&](u64, u64 w) { sum += w; });
    sum = block_sum_u64<THREADS>(sum, s);
    const u64 target = max((u64)1, min(sum, (u64)ceil((double)set.share * (double)sum)));
    cut = max(cut, cut_at<THREADS>(target, s, each));
  }
  auto final_weight = [&](int i) -> u64 {
    const float v = (float)x[i];
    if (v != top && !(((double)v - (double)top) * set.heat >= set.least)) return 0;
    return kept(v, i);
  };
  u64 sum = 0;
  for (int i = threadIdx.x; i < p.vocab; i += THREADS) sum += final_weight(i);
  sum = block_sum_u64<THREADS>(sum, s);
  const u64 target = min(sum - 1, (u64)(set.uniform * (double)sum));
  // ---- the first kept token at which the running sum passes the target
  u64 before = 0;
  for (int at = 0;; at += THREADS) {
    const int i = at + threadIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const u64 w = i < p.vocab ? final_weight(i) : 0;
    u64 run = w;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const u64 other = __shfl_up(run, off, kWave);
      if (lane >= off) run += other;
    }
    __syncthreads();
    if (lane == kWave - 1) s.words[wave] = run;
    __syncthreads();
    u64 all = 0;
    run += before;
#pragma unroll
    for (int v = 0; v < THREADS / kWave; ++v) {
      if (v < wave) run += s.words[v];
      all += s.words[v];
    }
    if (w && run > target && run - w <= target) {
      p.tokens[row] = i;
      if (p.probability) p.probability[row] = (float)((double)w / (double)sum);
    }
    before += all;
    if (before > target) break;
  }
}

// ------------------------------------------------------------ rows in registers
// A block takes a row, or, where rows are few, a part of one; the last of a row's blocks
// to arrive goes on with the row.  With the part's logits in registers:
//   - the maximum;
//   - for top-k and top-p, the tokens' number or weight in each bin, in LDS, and from
//     these the bin in which the cut falls: its tokens (for top-k those above it too)
//     are collected and sorted, which gives the cut exactly;
//   - the sums of the kept weights of every 64 lanes' tokens, and of these the 64 that
//     hold the number drawn.
// Bins are of absolute logits, so that those of several blocks fit together.  Sums of
// bins are of integers, all others are in a fixed order: the result does not depend
// on which thread comes first.  Rows that this does not fit (more than kMostKept tokens
// to collect, as in flat rows or with many equals; infinities; a top_k above kMostTopK)
// go to row_by_digits().

// The thread's EACH consecutive values and their sum.
template <int EACH, typename VALUE>
__device__ __forceinline__ double take_values(double (&v)[EACH], const VALUE& value) {
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) sum += v[e] = value((int)threadIdx.x * EACH + e);
  return sum;
}

// Inclusive and exclusive sums over the block's threads, in their order; `all`: of all.
template <int THREADS>
__device__ __forceinline__ double block_scan(double v, SampleScratch<THREADS>& s, double& before,
                                             double& all) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double other = __shfl_up(v, off, kWave);
    if (lane >= off) v += other;
  }
  __syncthreads();
  if (lane == kWave - 1) s.wave[wave] = v;
  __syncthreads();
  double base = 0.0;
  all = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) {
    if (w == wave) base = all;
    all += s.wave[w];
  }
  v += base;
  before = __shfl_up(v, 1, kWave);
  if (lane == 0) before = base;
  return v;
}

// Of `count` values, EACH consecutive ones a thread, the first that is not 0 and at which
// the running sum passes `target` (STRICT) or reaches it, the last that is not 0
// where none does; `before`: the sum before it.  -1: all are 0.
template <int THREADS, bool STRICT, int EACH>
__device__ __forceinline__ int find_in(const double (&v)[EACH], double target, double& before,
                                       SampleScratch<THREADS>& s) {
  double sum = 0.0, base, all;
#pragma unroll
  for (int e = 0; e < EACH; ++e) sum += v[e];
  block_scan<THREADS>(sum, s, base, all);
  if (threadIdx.x == 0) {
    s.found = 0x7fffffff;
    s.last = -1;
  }
  __syncthreads();
  int mine = 0x7fffffff, last = -1;
  double run = base, at = 0.0, at_last = 0.0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const double next = run + v[e];
    if (v[e] > 0.0) {
      const int i = (int)threadIdx.x * EACH + e;
      if ((STRICT ? next > target : next >= target) && mine == 0x7fffffff) {
        mine = i;
        at = run;
      }
      last = i;
      at_last = run;
    }
    run = next;
  }
  if (mine != 0x7fffffff) atomicMin(&s.found, mine);
  if (last >= 0) atomicMax(&s.last, last);
  __syncthreads();
  const bool some = s.found != 0x7fffffff;
  const int found = some ? s.found : s.last;
  if (some ? mine == found : last == found && last >= 0) s.value = some ? at : at_last;
  __syncthreads();
  before = s.value;
  return found;
}

// n keys in falling order (0 behind them up to a power of two).
template <int THREADS>
__device__ __forceinline__ void sort_keys(u64* keys, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + (int)threadIdx.x; i < size; i += THREADS) keys[i] = 0;
  for (int span = 2; span <= size; span <<= 1)
    for (int step = span >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int low = 2 * i - (i & (step - 1)), high = low + step;
        const u64 a = keys[low], b = keys[high];
        if ((a < b) == ((low & span) == 0)) {
          keys[low] = b;
          keys[high] = a;
        }
      }
    }
  __syncthreads();
}

template <typename T, int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
  constexpr int WAVES = THREADS / kWave, VEC = 16 / (int)sizeof(T), LOADS = EACH / VEC;
  constexpr int PART = THREADS * EACH, KEPT = (kMostKept + THREADS - 1) / THREADS;
  constexpr int BINS = (kBins + THREADS - 1) / THREADS;  // bins a thread
  typedef T vec __attribute__((ext_vector_type(VEC)));
  typedef vec unaligned __attribute__((aligned(sizeof(T))));  // rows start at any element
  __shared__ SampleScratch<THREADS> s;
  const int split = blockIdx.x % p.count, row = blockIdx.x / p.count;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  const Settings set = settings_of(p, row);
  const double heat16 = set.heat * kBinsOctave;
  const bool shared = p.count > 1;

  // ---- a part of the row: load i of lane l of wave w holds the VEC tokens from
  // ((i WAVES + w) 64 + l) VEC on, so that order is the vocabulary's
  float v[EACH];
  auto fetch = [&](int at, int end) TMC_INLINE {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int from = at + (i * THREADS + (int)threadIdx.x) * VEC;
      if (from + VEC <= end) {
        const vec in = *reinterpret_cast<const unaligned*>(x + from);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i * VEC + e] = (float)in[e];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          v[i * VEC + e] = from + e < end ? (float)x[from + e] : __builtin_nanf("");
      }
    }
  };
  auto place = [&](int at, int i) TMC_INLINE {
    return at + (i / VEC * THREADS + (int)threadIdx.x) * VEC + i % VEC;
  };
  // take(part's start) for every part of [begin, end), its logits in v
  int held = -1;  // start of the part in v
  auto parts = [&](int begin, int end, auto&& take) TMC_INLINE {
    for (int at = begin; at < end; at += PART) {
      if (at != held) fetch(at, end);
      held = at;
      take(at);
    }
  };
  const int begin = split * p.walk * PART, end = min(p.vocab, begin + p.walk * PART);

  // ---- the block's greatest
  float most = -INFINITY;  // (NaN left out)
  parts(begin, end, [&](int) TMC_INLINE {
#pragma unroll
    for (int i = 0; i < EACH; ++i) most = fmaxf(most, v[i]);
  });
  u64 best = 0;
  if (set.heat == 0.0) {  // with its token
    parts(begin, end, [&](int at) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (v[i] == most) best = max(best, rank_key(v[i], place(at, i)));
    });
  } else {
    best = most == -INFINITY ? 0 : rank_key(most, 0);
  }
  best = block_max_u64<THREADS>(best, s);
  // a row (part) without a logit above -inf, and infinities: by digits
  float top = best ? key_value(best) : -INFINITY;
  bool odd = !(fabsf(top) < INFINITY) || (set.most < p.vocab && set.most > kMostTopK);

  // ---- what the row's settings need of it
  enum { kGreedy, kList, kBin, kSum } way =
      set.heat == 0.0 ? kGreedy
      : set.most < p.vocab ? kList
      : set.share < 1.0f || (shared && set.least > kFaintest) ? kBin : kSum;
  auto bin_of = [&](float x) TMC_INLINE { return floor((double)x * heat16); };
  double first_bin = bin_of(top);  // of the greatest
  const double unit = 0x1p43;
  if (!odd && (way == kList || way == kBin)) {
    for (int i = threadIdx.x; i < kBins; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    parts(begin, end, [&](int) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const double bin = first_bin - bin_of(v[i]);  // (NaN: in none)
        if (bin < (double)kBins) {
          u64 cost = 1;
          if (way == kBin)
            cost = (u64)rint(exp2_of(fmax(((double)v[i] - (double)top) * set.heat, -60.0)) * unit);
          atomicAdd(&s.hist[(int)bin], cost);
        }
      }
    });
    __syncthreads();
  }
  // Weight of a token, 0 for one that is not kept: below the last that counts, or ranked
  // below `cut`.
  const double faintest = fmax(set.least, kFaintest);
  u64 cut = 0;
  auto weight = [&](float x, int at) TMC_INLINE -> double {
    const double a = ((double)x - (double)top) * set.heat;
    return a >= faintest && rank_key(x, at) >= cut ? exp2_of(a) : 0.0;
  };
  // the sums of every 64 lanes' loads, in their order, and of all
  auto sum_groups = [&](int begin, int end) TMC_INLINE {
    parts(begin, end, [&](int at) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += weight(v[i * VEC + e], place(at, i * VEC + e));
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
        if (lane == 0) s.groups[((at - begin) / PART * LOADS + i) * WAVES + wave] = sum;
      }
    });
    __syncthreads();
  };
  auto say = [&](int token, double share) TMC_INLINE {
    p.tokens[row] = token;
    if (p.probability) p.probability[row] = (float)share;
  };
  // The token of [begin, end) whose weight the running sum, `before` ahead of it, passes
  // u times the sum `total` with (total < 0: that of these tokens).
  auto draw = [&](int begin, int end, double before, double total) TMC_INLINE {
    sum_groups(begin, end);
    const int groups = (end - begin + PART - 1) / PART * LOADS * WAVES;
    constexpr int kEach = kMostGroups / THREADS;
    auto group = [&](int g) TMC_INLINE { return g < groups ? s.groups[g] : 0.0; };
    double mine[kEach], base, here;
    block_scan<THREADS>(take_values(mine, group), s, base, here);
    if (total < 0.0) total = here;
    double target = set.uniform * total - before;
    const int g = find_in<THREADS, true>(mine, target, before, s);
    if (g < 0 || wave != 0) return;  // (the first wave goes on with the group)
    target -= before;
    const int at = begin + (g / (LOADS * WAVES)) * PART +
                   ((g / WAVES % LOADS) * THREADS + g % WAVES * kWave + lane) * VEC;
    double w[VEC], sum = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[e] = at + e < end ? weight((float)x[at + e], at + e) : 0.0;
      sum += w[e];
    }
    double run = sum;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const double other = __shfl_up(run, off, kWave);
      if (lane >= off) run += other;
    }
    double ahead = __shfl_up(run, 1, kWave);
    if (lane == 0) ahead = 0.0;
    // (the last that is kept where sums of another order fall short)
    const u64 some = __builtin_amdgcn_ballot_w64(sum > 0.0);
    const u64 past = __builtin_amdgcn_ballot_w64(sum > 0.0 && run > target);
    if (some == 0 || lane != (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some))) return;
    int token = -1;
    double share = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (w[e] > 0.0 && !(token >= 0 && ahead > target)) {
        token = at + e;
        share = w[e];
      }
      ahead += w[e];
    }
    say(token, share / total);
  };
  // The tokens of [begin, end) in bins [from, to] into the list; false: too many.
  auto collect = [&](int begin, int end, int from, int to) TMC_INLINE -> bool {
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    parts(begin, end, [&](int at) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const double bin = first_bin - bin_of(v[i]);
        if (bin >= (double)from && bin <= (double)to) {
          const int slot = atomicAdd(&s.count, 1);
          if (slot < kMostKept) s.keys[slot] = rank_key(v[i], place(at, i));
        }
      }
    });
    __syncthreads();
    return s.count <= kMostKept;
  };
  auto listed = [&](int i, int n) TMC_INLINE {  // weight of the list's token i
    if (i >= n) return 0.0;
    const double a = ((double)key_value(s.keys[i]) - (double)top) * set.heat;
    return a >= kFaintest ? exp2_of(a) : 0.0;
  };
  // The draw from the sorted list, its first `most` tokens.
  auto draw_list = [&](int n) TMC_INLINE {
    n = min(n, set.most);
    double before, total;
    double w[KEPT];
    block_scan<THREADS>(take_values(w, [&](int i) { return listed(i, n); }), s, before, total);
    // kept: those of which less than the share lies before
    const double limit = set.share < 1.0f ? (double)set.share * total : INFINITY;
    int kept = 0;
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = (int)threadIdx.x * KEPT + e;
      const double a = i < n ? ((double)key_value(s.keys[i]) - (double)top) * set.heat : -INFINITY;
      kept += i == 0 || (w[e] > 0.0 && before < limit && a >= set.least);
      before += w[e];
    }
    n = (int)block_sum_u64<THREADS>((u64)kept, s);
    // by index, each with its rank behind
    u64 index[KEPT];
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = (int)threadIdx.x * KEPT + e;
      index[e] = i < n ? s.keys[i] & 0xFFFFFFFFull : 0;  // (~index: the lowest first)
      s.groups[i] = w[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = (int)threadIdx.x * KEPT + e;
      if (i < n) s.keys[i] = index[e] << 32 | (unsigned)i;
    }
    sort_keys<THREADS>(s.keys, n);
    auto value = [&](int i) TMC_INLINE { return i < n ? s.groups[(unsigned)s.keys[i]] : 0.0; };
    block_scan<THREADS>(take_values(w, value), s, before, total);
    const int i = find_in<THREADS, true>(w, set.uniform * total, before, s);
    if (threadIdx.x == 0) say((int)~(unsigned)(s.keys[i] >> 32), value(i) / total);
  };
  // The bin in which top-p or min-p cuts, of this thread's sums of the bins and their
  // sum; its tokens decide.  False: too many of them.
  auto cut_bin = [&](const double (&v)[BINS], double sum, int& bin) -> bool {
    double before, total, above;
    block_scan<THREADS>(sum, s, before, total);
    const double limit = set.share < 1.0f ? (double)set.share * total : INFINITY;
    bin = find_in<THREADS, false>(v, limit, above, s);
    // min-p: the bin of the least logit that it keeps, or the one before (a quotient may
    // be off by its last bit): the tokens of both are looked at
    const double least = first_bin - bin_of((float)((double)top + faintest / set.heat)) - 1.0;
    int from = bin, to = bin;
    if (set.least > kFaintest && least < (double)bin) {
      from = max((int)least, 0);
      to = min(bin, (int)least + 2);
    }
    if (!collect(0, p.vocab, from, to)) return false;
    const int n = s.count;
    sort_keys<THREADS>(s.keys, n);
    // the sum before the list
    if (from != bin) {
      double run = before;
#pragma unroll
      for (int e = 0; e < BINS; ++e) {
        if ((int)threadIdx.x * BINS + e == from) s.value = run;
        run += v[e];
      }
      __syncthreads();
      above = s.value;
    }
    bin = from;
    double w[KEPT], ahead, all;
    block_scan<THREADS>(take_values(w, [&](int i) { return listed(i, n); }), s, ahead, all);
    int kept = 0;
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = (int)threadIdx.x * KEPT + e;
      const double a = i < n ? ((double)key_value(s.keys[i]) - (double)top) * set.heat : -INFINITY;
      kept += w[e] > 0.0 && above + ahead < limit && a >= set.least;
      ahead += w[e];
    }
    kept = (int)block_sum_u64<THREADS>((u64)kept, s);
    if (from == 0) kept = max(kept, 1);  // the most probable token
    // None kept: the cut is between the list and the bins before it (without a list it is
    // min-p's, which weight() applies).
    cut = kept > 0 ? s.keys[kept - 1] : n == 0 ? 0 : s.keys[0] + 1;
    s.count = kept;
    return true;
  };

  // ---- the row's blocks together: every word at agent scope, completed before the
  // arrival is counted; the last of them goes on
  auto put = [](auto* to, auto value) TMC_INLINE {
    __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto get = [](const auto* from) TMC_INLINE {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  SampleRecord* records = p.parts + (size_t)row * p.count;
  u64* bins = p.bins + (size_t)row * p.count * kBins;
  if (shared) {
    double sum = 0.0;
    if (way == kSum && !odd) {
      sum_groups(begin, end);
      const int groups = (end - begin + PART - 1) / PART * LOADS * WAVES;
      double mine = 0.0, before;
      for (int g = threadIdx.x; g < groups; g += THREADS) mine += s.groups[g];
      block_scan<THREADS>(mine, s, before, sum);
    }
    if (threadIdx.x == 0) {
      put(&records[split].best, best);
      put(&records[split].sum, sum);
    }
    if (!odd && (way == kList || way == kBin))
      for (int i = threadIdx.x; i < kBins; i += THREADS)
        put(bins + (size_t)split * kBins + i, s.hist[i]);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
      s.last = __hip_atomic_fetch_add(p.arrivals + row * kCounterStride, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == p.count - 1;
    __syncthreads();
    const bool last = s.last;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) put(p.arrivals + row * kCounterStride, 0);
    best = 0;
    odd = set.most < p.vocab && set.most > kMostTopK;
    for (int b = threadIdx.x; b < p.count; b += THREADS) {
      const u64 other = get(&records[b].best);
      best = max(best, other);
      odd |= other && !(fabsf(key_value(other)) < INFINITY);
    }
    odd = __syncthreads_or(odd);
    best = block_max_u64<THREADS>(best, s);
    top = best ? key_value(best) : -INFINITY;
    first_bin = bin_of(top);
  }
  if (way == kGreedy && best) {
    if (threadIdx.x == 0) say(key_index(best), 1.0);
    return;
  }
  // A block's factor: its greatest weight.  Its bins are so many behind the row's.  (A
  // block of -inf alone put none, and is passed over.)
  auto high_of = [&](int b) TMC_INLINE {
    const u64 other = get(&records[b].best);
    return other ? key_value(other) : -INFINITY;
  };
  auto factor_of = [&](float high) TMC_INLINE {
    const double a = ((double)high - (double)top) * set.heat;
    return a >= kFaintest ? exp2_of(a) : 0.0;
  };
  bool done = best != 0 && !odd;
  int bin = 0;
  if (done && way != kSum) {
    // the row's bins, block after block
    double mine[BINS], all = 0.0;
#pragma unroll
    for (int e = 0; e < BINS; ++e) mine[e] = 0.0;
    for (int b = 0; b < p.count; ++b) {
      const float high = shared ? high_of(b) : top;
      const double behind = first_bin - bin_of(high);
      if (!(behind < (double)kBins)) continue;
      const double scale = way == kBin ? factor_of(high) * (1.0 / unit) : 1.0;
#pragma unroll
      for (int e = 0; e < BINS; ++e) {
        const int i = (int)threadIdx.x * BINS + e - (int)behind;
        if (i >= 0 && i + (int)behind < kBins)
          mine[e] += scale * (double)(shared ? get(bins + (size_t)b * kBins + i) : s.hist[i]);
      }
    }
#pragma unroll
    for (int e = 0; e < BINS; ++e) all += mine[e];
    if (way == kList) {
      double before;
      bin = find_in<THREADS, false>(mine, (double)set.most, before, s);
    } else {
      done = cut_bin(mine, all, bin);
    }
    if (way == kList) {
      done = collect(0, p.vocab, 0, bin);
      if (done) {
        const int n = s.count;
        sort_keys<THREADS>(s.keys, n);
        draw_list(n);
        return;
      }
    }
  }
  if (!done) {
    row_by_digits<T, THREADS>(p, row, set, s);
    return;
  }
  int draw_begin = 0, draw_end = p.vocab;
  double before = 0.0, total = -1.0;
  if (shared) {
    // what each block keeps: its bins before the list, and its tokens of the list
    double* s_block = s.groups;
    const int kept = s.count, span = p.walk * PART;
    for (int b = wave; b < p.count; b += WAVES) {
      const float high = high_of(b);
      const double behind = first_bin - bin_of(high);
      double sum = 0.0;
      if (way == kSum) {
        sum = lane == 0 ? factor_of(high) * get(&records[b].sum) : 0.0;
      } else {
        if (behind < (double)bin) {
          const double scale = factor_of(high) * (1.0 / unit);
          for (int i = lane; i + (int)behind < bin; i += kWave)
            sum += scale * (double)get(bins + (size_t)b * kBins + i);
        }
        for (int i = lane; i < kept; i += kWave)
          if (key_index(s.keys[i]) / span == b) sum += listed(i, kept);
      }
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
      if (lane == 0) s_block[b] = sum;
    }
    __syncthreads();
    constexpr int kEach = (kSharedRows + THREADS - 1) / THREADS;  // blocks of a row, at most
    double mine[kEach], base;
    const double sum = take_values(mine, [&](int b) { return b < p.count ? s_block[b] : 0.0; });
    block_scan<THREADS>(sum, s, base, total);
    const int b = find_in<THREADS, true>(mine, set.uniform * total, before, s);
    __syncthreads();
    draw_begin = b * span;
    draw_end = min(p.vocab, draw_begin + span);
  }
  draw(draw_begin, draw_end, before, total);
}

bool sample_shape(int64_t rows, int64_t vocabulary) {
  return rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary <= kMostTokens;
}

// How rows are shared out.  A block of 1024 threads holds a row of up to 32768 in its
// registers, one of 256 up to 8192.  Where rows are few, blocks of 8192 share one, up to
// kFill of them together.
constexpr int64_t kFill = 512, kFewRows = 192;
static_assert(kFill <= kSharedRows, "every shared row has its counter");
struct SamplePlan {
  int threads, each, walk, count;
};
SamplePlan sample_plan(int64_t rows, int64_t vocabulary) {
  SamplePlan plan{1024, 32, 1, 1};
  if (vocabulary <= 8192) {
    plan.threads = 256;
  } else if (rows < kFewRows) {
    const int64_t parts = (vocabulary + 8191) / 8192, blocks = std::min(parts, kFill / rows);
    plan.each = 8;
    plan.walk = (int)((parts + blocks - 1) / blocks);
    plan.count = (int)((parts + plan.walk - 1) / plan.walk);
    return plan;
  }
  const int64_t span = (int64_t)plan.threads * plan.each;
  plan.walk = (int)((vocabulary + span - 1) / span);
  return plan;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_sample_workspace_bytes(int64_t rows, int64_t vocabulary) {
  if (!sample_shape(rows, vocabulary)) return 0;
  const int64_t count = sample_plan(rows, vocabulary).count;
  return count == 1 ? 0
                    : kCounterBytes + (size_t)(rows * count) *
                                          (sizeof(SampleRecord) + kBins * sizeof(u64));
}

extern "C" int tmc_sample(const void* logits, int dtype, int64_t row_stride,
                          const float* temperature, const int32_t* top_k, const float* top_p,
                          const float* min_p, const float* uniforms, int32_t* tokens,
                          float* probability, int64_t rows, int64_t vocabulary, void* workspace,
                          size_t workspace_bytes, void* stream) {
  TMC_REQUIRE(logits && uniforms && tokens, "Sample: null device pointer.");
  TMC_REQUIRE(dtype == TMC_F32 || dtype == TMC_F16, "Sample: logits must be f32 or f16.");
  TMC_REQUIRE(sample_shape(rows, vocabulary) && row_stride >= vocabulary &&
                  row_stride < (1LL << 36),
              "Sample: invalid shape.");
  TMC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == TMC_F32 ? 4 : 2) == 0,
              "Sample: logits must be aligned to their elements.");
  const size_t need = tmc_sample_workspace_bytes(rows, vocabulary);
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "Sample: workspace is smaller than tmc_sample_workspace_bytes() or not 16-byte "
              "aligned.");
  SampleParams p{};
  p.logits = logits;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.uniforms = uniforms;
  p.tokens = tokens;
  p.probability = probability;
  p.stride = (long)row_stride;
  p.rows = (int)rows;
  p.vocab = (int)vocabulary;
  // a sum of `vocabulary` weights fits 64 bits
  int bits = 0;
  while (((int64_t)1 << bits) < vocabulary) ++bits;
  p.scale = std::min(52, 63 - bits);
  const SamplePlan plan = sample_plan(rows, vocabulary);
  p.walk = plan.walk;
  p.count = plan.count;
  if (need) {
    p.arrivals = static_cast<int*>(workspace);
    p.parts = reinterpret_cast<SampleRecord*>(static_cast<char*>(workspace) + kCounterBytes);
    p.bins = reinterpret_cast<u64*>(p.parts + rows * plan.count);
  }
  const dim3 grid((unsigned)(rows * plan.count));
  const hipStream_t s = as_stream(stream);
#define TMC_SAMPLE(TYPE, THREADS, EACH) \
  hipLaunchKernelGGL((sample_kernel<TYPE, THREADS, EACH>), grid, dim3(THREADS), 0, s, p)
#define TMC_SAMPLE_PLAN(TYPE)                              \
  if (plan.threads == 256) TMC_SAMPLE(TYPE, 256, 32);      \
  else if (plan.each == 32) TMC_SAMPLE(TYPE, 1024, 32);    \
  else TMC_SAMPLE(TYPE, 1024, 8)
  if (dtype == TMC_F32) {
    TMC_SAMPLE_PLAN(float);
  } else {
    TMC_SAMPLE_PLAN(half_t);
  }
#undef TMC_SAMPLE_PLAN
#undef TMC_SAMPLE
  return check_launch("sample_kernel");
}
