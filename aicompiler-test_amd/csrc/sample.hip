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
#include <type_traits>

// (a lambda that is not inlined keeps what it refers to in memory)
#define TMC_INLINE __attribute__((always_inline))

namespace tmc {
namespace {

typedef unsigned long long u64;

// What the blocks of a shared row find out together in the first launch.
struct SampleRow {
  u64 best;         // greatest rank key
  float low, high;  // the logits in the list: from low on, below high
  int odd;          // to be done by digits
  int least;        // the list is where min-p cuts, see bounds()
  int listed;       // in the second launch: tokens in the list so far
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
  int vocab;
  int scale;            // integer weights are multiples of 2^-scale
  int count, walk;      // blocks a row, parts of a row that each takes
  // of shared rows
  SampleRow* records;   // [rows]
  u64* blocks;          // [rows][count]: greatest rank keys, then sums of weights
  u64* sums;            // [rows][count][walk]: the kept weights of every part
  u64* lists;           // [rows][kMostKept]
  float* bins;          // [rows][count][kBins]: their running sums
  int* arrivals;        // [rows], kCounterStride apart
};

constexpr int kMostBlocks = 512;  // of a row

// Below it a temperature counts as 0: the most probable token.
constexpr float kColdest = 1.0f / 65536.0f;

// log2 of the least weight that counts: what lies below it, of 2^20 tokens, is less
// than the distance of two 24-bit random numbers near 1.
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
  s.least = least > 0.0f ? log2((double)fminf(least, 1.0f)) : -INFINITY;
  if (t == INFINITY) {  // equal weights, of which min-p takes none
    s.heat = 0x1p-1000;
    s.least = -INFINITY;
  }
  s.share = share < 1.0f ? fmaxf(share, 0.0f) : 1.0f;
  s.most = k > 0 && k < p.vocab ? k : p.vocab;
  return s;
}

// ------------------------------------------------------------ shared by both ways
// v of the lane that the row operation CTRL names, 0 where it names none.
template <int CTRL, int ROWS, typename TYPE> __device__ __forceinline__ TYPE lane_move(TYPE v) {
  const u64 b = __builtin_bit_cast(u64, v);
  const unsigned low = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xf, false);
  const unsigned high = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(TYPE, (u64)high << 32 | low);
}
// Running sums (or maxima) over the lanes: of rows of 16, then of all.
template <typename TYPE, typename JOIN>
__device__ __forceinline__ TYPE wave_scan(TYPE v, const JOIN& join) {
  v = join(v, lane_move<0x111, 0xf>(v));  // the lane 1, 2, 4 and 8 before
  v = join(v, lane_move<0x112, 0xf>(v));
  v = join(v, lane_move<0x114, 0xf>(v));
  v = join(v, lane_move<0x118, 0xf>(v));
  v = join(v, lane_move<0x142, 0xa>(v));  // the last of the row before, in every other row
  v = join(v, lane_move<0x143, 0xc>(v));  // the last of the lower half, in the upper
  return v;
}
template <typename TYPE> __device__ __forceinline__ TYPE wave_scan(TYPE v) {
  return wave_scan(v, [](TYPE a, TYPE b) TMC_INLINE { return a + b; });
}

constexpr int kDigits = 256;
// A row's tokens are looked at bin by bin: 1/16 octave of the weight each, down to
// kFaintest.
constexpr int kBinsOctave = 16, kBins = 44 * kBinsOctave;
// Bins are numbered in fp32: below this number, and kBins further down, exactly.
constexpr float kMostLevel = 0x1p23f;
static_assert(kFaintest == -44.0, "bins down to the least weight");
// Tokens in the list, as many as let four blocks into LDS, and the top_k that goes by it.
constexpr int kMostKept = 2048, kMostTopK = 1024;
constexpr int kMostGroups = 512;                   // sums of a block's parts
constexpr int kCoarse = 32;  // bins of a coarse step, and at most steps
static_assert(kMostBlocks <= kMostGroups, "a sum a block");
static_assert(kBins % kCoarse == 0 && kBins / kCoarse <= kCoarse, "two steps to a bin");

template <int THREADS> struct SampleScratch {
  u64 hist[kBins > 2 * kDigits ? (kBins + 1) / 2 : kDigits];  // (bins: of 32 bits)
  u64 keys[kMostKept];
  u64 groups[kMostGroups];  // (of a shared row first what its blocks keep of the list)
  u64 words[THREADS / kWave];
  double levels[kCoarse];
  double value;  // (or an integer)
  u64 found64;
  int found, last, small;
};

template <int THREADS>
__device__ __forceinline__ u64 block_sum_u64(u64 v, SampleScratch<THREADS>& s) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) s.words[threadIdx.x / kWave] = v;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) sum += s.words[w];
  return sum;
}
template <int THREADS>
__device__ __forceinline__ u64 block_max_u64(u64 v, SampleScratch<THREADS>& s) {
  v = wave_scan(v, [](u64 a, u64 b) TMC_INLINE { return max(a, b); });
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) s.words[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) v = max(v, s.words[w]);
  return v;
}

// 2^a for a <= 0: Taylor's series of e^z, |z| <= ln 2 / 2, up to z^11: its rest is below
// 2^-46.6 of it.
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

// ------------------------------------------------------------ rows in registers
// With a part of the row at a time in registers:
//   - the maximum;
//   - for top-k and top-p, the tokens' number or weight in each bin, in LDS, and from
//     these the bins in which the cut falls;
//   - the tokens of these bins (for top-k those above too) into a list, and the sums of
//     the weights before them, of every part; in the list the cut is found exactly;
//   - the part that holds the number drawn, and in it the token.
// One 64-bit exponential a token: the bins' weights are of 32 bits, and say only which
// tokens to list.  Where these are more than kMostKept, their bins are cut into 64 each and
// the last two steps are done again (not with min-p, whose cut may be another bin's).
//
// Where rows are few, several blocks share one, in two launches: the first ends with the
// bins, of which the last of a row's blocks to arrive finds the list's bounds; in the
// second each block sums and lists its own tokens, and the last goes on with the row.
// (In one launch the last block has to read the whole row again by itself: 30 us of 91
// for 64 rows of 128000, in two launches 60.)
//
// Measured (32-bit logits, top-k and top-p, warm caches): one row of 32000 30 us, a
// chain of some thirty steps that each wait for the one before; 1024 rows of 32003 with
// mixed settings 100 us, 1.3 TB/s: 32 us the maximum, which reads the logits from memory,
// 10 us the bins, 38 us the exponentials (some 35 64-bit operations a token), 20 us the
// list and the draw.  64 rows of 128000 fp16 tokens 57 us: 18 us the first launch.
//
// Bins are of absolute logits, so that those of several blocks fit together; finer ones of
// logits less the greatest of theirs.  Weights are integers: the result does not depend on
// which thread comes first.  Rows that this does not fit go to row_by_digits(), 0.5 ms a
// row of 32000 and 1.8 to 2.1 ms one of 128000, 3.5 to 4.1 ms 64 of these:
//   - long runs of equals at the cut, infinities, a top_k above kMostTopK;
//   - more than kMostKept tokens in the cut's bins, with a min-p;
//   - a greatest logit of 3.6e5 temperatures and more (kMostLevel bins);
//   - a run of equals so close to top-p's border that the bins took the wrong one, which the
//     exact sums of the listed tokens tell.

// The thread's EACH consecutive values and their sum.
template <int EACH, typename TYPE, typename VALUE>
__device__ __forceinline__ TYPE take_values(TYPE (&v)[EACH], const VALUE& value) {
  TYPE sum = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) sum += v[e] = value((int)threadIdx.x * EACH + e);
  return sum;
}

// Inclusive and exclusive sums over the block's threads, in their order; `all`: of all.
template <int THREADS, typename TYPE>
__device__ __forceinline__ TYPE block_scan(TYPE v, SampleScratch<THREADS>& s, TYPE& before,
                                           TYPE& all) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  TYPE* words = reinterpret_cast<TYPE*>(s.words);
  v = wave_scan(v);
  __syncthreads();
  if (lane == kWave - 1) words[wave] = v;
  __syncthreads();
  TYPE base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) {
    if (w == wave) base = all;
    all += words[w];
  }
  before = base + lane_move<0x138, 0xf>(v);  // the lane before
  return base + v;
}

// Of values, EACH consecutive ones a thread, with `base` the sum before the thread's: the
// first that is not 0 and at which the running sum passes `target` (STRICT) or
// reaches it, the last that is not 0 where none does; `before`: the sum before it.  -1:
// all are 0.
template <int THREADS, bool STRICT, int EACH, typename TYPE>
__device__ __forceinline__ int find_in(const TYPE (&v)[EACH], TYPE base, TYPE target, TYPE& before,
                                       SampleScratch<THREADS>& s) {
  TYPE* value = reinterpret_cast<TYPE*>(&s.value);
  if (threadIdx.x == 0) {
    s.found = 0x7fffffff;
    s.last = -1;
  }
  __syncthreads();
  int mine = 0x7fffffff, last = -1;
  TYPE run = base, at = 0, at_last = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const TYPE next = run + v[e];
    if (v[e] > 0) {
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
  if (some ? mine == found : last == found && last >= 0) *value = some ? at : at_last;
  __syncthreads();
  before = *value;
  return found;
}

// The key of the list s.keys[0 ... n), all in [low, high], at which the running cost, from
// the highest ranked down, reaches `target` (at least 1); 0 where all of it does not.
// `cost` gives that of a place.  The list's range of keys is cut into 256, then that of the
// part with the target, until a wave can take the rest: for logits that are not equal,
// once or twice.
template <int THREADS, typename COST>
__device__ __forceinline__ u64 select_key(int n, u64 low, u64 high, u64 target,
                                          SampleScratch<THREADS>& s, const COST& cost) {
  static_assert(THREADS == kDigits, "a digit a thread");
  const int lane = threadIdx.x & (kWave - 1);
  u64* hist = s.hist;
  for (;;) {
    // the keys in [low, high], by their first eight bits above `low`
    const int bits = 64 - __clzll((high - low) | 1), shift = max(0, bits - 8);
    __syncthreads();
    hist[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.small = 0;
    __syncthreads();
    int here = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const u64 key = s.keys[i];
      if (key >= low && key <= high) {
        atomicAdd(&hist[255 - ((key - low) >> shift)], cost(i));
        ++here;
      }
    }
    const int left = (int)block_sum_u64<THREADS>((u64)here, s);
    if (left <= kWave) break;
    const u64 mine[1] = {hist[threadIdx.x]};
    u64 base, all, before;
    block_scan<THREADS>(mine[0], s, base, all);
    if (all < target) return 0;
    const int digit = find_in<THREADS, false>(mine, base, target, before, s);
    target -= before;
    if (shift == 0) return low + (255 - digit);
    low += (u64)(255 - digit) << shift;
    high = min(high, low + (((u64)1 << shift) - 1));
  }
  // up to 64 keys: each lane sums what ranks above its own
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 key = s.keys[i];
    if (key < low || key > high) continue;
    const int slot = atomicAdd(&s.small, 1);
    hist[slot] = key;
    hist[kWave + slot] = cost(i);
  }
  if (threadIdx.x == 0) s.found64 = 0;
  __syncthreads();
  const int few = s.small;
  if ((int)threadIdx.x < few) {
    const u64 key = hist[lane], own = hist[kWave + lane];
    u64 run = 0;
    for (int o = 0; o < few; ++o)
      if (hist[o] >= key) run += hist[kWave + o];
    if (run >= target && run - own < target) s.found64 = key;
  }
  __syncthreads();
  const u64 found = s.found64;
  __syncthreads();
  return found;
}

// ------------------------------------------------------------ any row
// The key at which the running cost, from the highest ranked down, reaches
// `target` (at least 1 and at most all of it): digit by digit, a histogram of the
// costs of the keys that agree so far.
template <int THREADS, typename EACH>
__device__ __forceinline__ u64 cut_at(u64 target, SampleScratch<THREADS>& s, const EACH& each) {
  static_assert(THREADS == kDigits, "a digit a thread");
  u64 prefix = 0;
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    s.hist[threadIdx.x] = 0;
    __syncthreads();
    each([&](u64 key, u64 cost) TMC_INLINE {
      if (shift < 56 && key >> (shift + 8) != prefix >> (shift + 8)) return;
      // (rows of equals: one lane for all that are alike)
      const unsigned digit = (unsigned)(key >> shift) & 255u;
      const u64 here = __ballot(true);
      const bool alike = digit == (unsigned)__builtin_amdgcn_readfirstlane(digit) &&
                         cost == ((u64)(unsigned)__builtin_amdgcn_readfirstlane((int)(cost >> 32)) << 32 |
                                  (unsigned)__builtin_amdgcn_readfirstlane((int)cost));
      if (__ballot(alike) != here) atomicAdd(&s.hist[digit], cost);
      else if ((threadIdx.x & (kWave - 1)) == __builtin_ctzll(here))
        atomicAdd(&s.hist[digit], cost * __popcll(here));
    });
    __syncthreads();
    const u64 mine[1] = {s.hist[kDigits - 1 - threadIdx.x]};
    u64 base, all, before;
    block_scan<THREADS>(mine[0], s, base, all);
    const int digit = kDigits - 1 - find_in<THREADS, false>(mine, base, target, before, s);
    prefix |= (u64)digit << shift;
    target -= before;
  }
  return prefix;
}

// A row by one block, whatever it holds, pass after pass over memory: weights as
// integers, cuts by their digits, up to 21 passes.
template <typename T, int THREADS>
__device__ __forceinline__ void row_by_digits(const SampleParams& p, int row, const Settings& set,
                                              SampleScratch<THREADS>& s) {
  constexpr int AHEAD = 4;  // loads in flight
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  // take(logit, index) of the tokens of [begin, end); NaN behind them
  auto tokens = [&](int begin, int end, auto&& take) TMC_INLINE {
#pragma unroll 1
    for (int at = begin + (int)threadIdx.x; at - (int)threadIdx.x < end; at += AHEAD * THREADS) {
      float v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        v[j] = at + j * THREADS < end ? (float)x[at + j * THREADS] : __builtin_nanf("");
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) take(v[j], at + j * THREADS);
    }
  };
  // ---- the most probable token
  u64 best = 0;
  tokens(0, p.vocab, [&](float v, int i) TMC_INLINE {
    if (v == v) best = max(best, rank_key(v, i));
  });
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
  auto weight = [&](float v) TMC_INLINE -> u64 {
    if (v == top) return (u64)unit;
    if (!(v > -INFINITY) || top == INFINITY) return 0;
    const double a = ((double)v - (double)top) * set.heat;
    return a >= kFaintest ? max((u64)rint(exp2_of(a) * unit), (u64)1) : 0;
  };
  u64 cut = 0;
  // top-k, then top-p
#pragma unroll 1
  for (int step = set.most < p.vocab ? 0 : 1; step < (set.share < 1.0f ? 2 : 1); ++step) {
    auto each = [&](auto&& take) TMC_INLINE {
      tokens(0, p.vocab, [&](float v, int i) TMC_INLINE {
        const u64 w = weight(v), key = rank_key(v, i);
        if (w && key >= cut) take(key, step == 0 ? (u64)1 : w);
      });
    };
    u64 sum = 0;
    each([&](u64, u64 cost) TMC_INLINE { sum += cost; });
    sum = block_sum_u64<THREADS>(sum, s);
    u64 target = (u64)set.most;
    if (step == 1) target = max((u64)1, min(sum, (u64)ceil((double)set.share * (double)sum)));
    else if (sum <= target) continue;
    cut = max(cut, cut_at<THREADS>(target, s, each));
  }
  auto kept = [&](float v, int i) TMC_INLINE -> u64 {
    if (v != top && !(((double)v - (double)top) * set.heat >= set.least)) return 0;
    const u64 w = weight(v);
    return w && rank_key(v, i) >= cut ? w : 0;
  };
  u64 sum = 0;
  tokens(0, p.vocab, [&](float v, int i) TMC_INLINE { sum += kept(v, i); });
  sum = block_sum_u64<THREADS>(sum, s);
  const u64 target = min(sum - 1, (u64)(set.uniform * (double)sum));
  // ---- the first kept token at which the running sum passes the target: among 16 loads a
  // thread, then among one
  u64 before = 0;
  int begin = 0;
#pragma unroll 1
  for (int span = 16 * THREADS; span >= THREADS; span /= 16)
#pragma unroll 1
    for (;; begin += span) {
      u64 own = 0;
      tokens(begin, min(p.vocab, begin + span), [&](float v, int i) TMC_INLINE { own += kept(v, i); });
      own = block_sum_u64<THREADS>(own, s);
      if (before + own > target || begin + span >= p.vocab) break;
      before += own;
    }
  const int at = begin + (int)threadIdx.x;
  const u64 w[1] = {at < p.vocab ? kept((float)x[at], at) : 0};
  u64 base, all, ahead;
  block_scan<THREADS>(w[0], s, base, all);
  const int index = find_in<THREADS, true>(w, base, target - before, ahead, s);
  if ((int)threadIdx.x == index) {
    p.tokens[row] = at;
    if (p.probability) p.probability[row] = (float)((double)w[0] / (double)sum);
  }
}

// ------------------------------------------------------------ the kernel
// STAGE: 0 for a row of one block, 1 and 2 for the launches of shared rows.  Four blocks a
// CU, as many as LDS holds: without the bound the loop over finer bins takes registers
// from them (1024 rows 121 us for 108).
template <typename T, int THREADS, int EACH, int STAGE>
__global__ __launch_bounds__(THREADS, 4) void sample_kernel(SampleParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), LOADS = EACH / VEC;
  constexpr int PART = THREADS * EACH;
  constexpr int BINS = (kBins + THREADS - 1) / THREADS;  // bins a thread
  constexpr bool SHARED = STAGE > 0;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  typedef vec unaligned __attribute__((aligned(sizeof(T))));  // rows start at any element
  __shared__ SampleScratch<THREADS> s;
  __shared__ double factors[STAGE == 1 ? kMostBlocks : 1];  // of a row's blocks: the greatest weight,
  __shared__ u64 costs[STAGE == 1 ? 1 : kMostKept];         // of the list's keys
  __shared__ float highs[STAGE == 1 ? kMostBlocks : 1];     // the greatest logit
  const int split = SHARED ? blockIdx.x % p.count : 0, row = SHARED ? blockIdx.x / p.count : blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;

  // ---- a part of the row, EACH tokens a thread, so that order is the vocabulary's
  auto load = [&](int from, int end) TMC_INLINE -> vec {
    if (from + VEC <= end) return *reinterpret_cast<const unaligned*>(x + from);
    vec in;
#pragma unroll
    for (int e = 0; e < VEC; ++e) in[e] = from + e < end ? x[from + e] : (T)__builtin_nanf("");
    return in;
  };
  float v[EACH];
  int held = -1;  // start of the part in v
  auto fetch = [&](int at, int end) TMC_INLINE {
    if (at == held) return;
    vec in[LOADS];
    const int from = at + (int)threadIdx.x * EACH;
    if (at + PART <= end) {  // (for all threads: the loads are in flight together)
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        in[i] = *reinterpret_cast<const unaligned*>(x + from + i * VEC);
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) in[i] = load(from + i * VEC, end);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = (float)in[i / VEC][i % VEC];
    held = at;
  };
  // What a pass computes of each logit it computes anew: kept for the next pass it would
  // take more registers than there are.
  float top = 0.0f, first_bin = 0.0f;
  // take(part's start) for every part of [begin, end), its logits in v
  auto parts = [&](int begin, int end, auto&& take) TMC_INLINE {
    for (int at = begin; at < end; at += PART) {
      fetch(at, end);
      asm volatile("" : "+v"(top), "+v"(first_bin));
      take(at);
    }
  };
  auto place = [&](int at, int i) TMC_INLINE {
    return at + (int)threadIdx.x * EACH + i;
  };
  const int span = p.walk * PART;  // of a block
  int begin = split * span, end = SHARED ? min(p.vocab, begin + span) : p.vocab;
  SampleRow* record = p.records + row;

  // ---- the greatest, of the block or (known already) of the row
  u64 best = 0;
  fetch(begin, end);
  const Settings set = settings_of(p, row);
  if (STAGE == 2) {
    best = record->best;
  } else {
    float most = -INFINITY;  // (NaN left out)
    parts(begin, end, [&](int) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i) most = fmaxf(most, v[i]);
    });
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
  }
  top = best ? key_value(best) : -INFINITY;
  const float heat = (float)set.heat;
  float octave = kBinsOctave, per_bin = heat * octave;  // bins an octave, and a logit
  // what has no bins, and long lists: by digits.  (A block of a shared row whose logits are
  // far below the row's is passed over: its bins need a number, no exact one.)
  auto is_odd = [&](float top, float most) TMC_INLINE {
    return !(fabsf(top * per_bin) < most) || !(fabsf(top) < INFINITY);
  };
  bool odd = STAGE == 2 ? record->odd
                        : is_odd(top, SHARED ? INFINITY : kMostLevel) ||
                              (set.most < p.vocab && set.most > kMostTopK);

  // ---- what the row's settings need of it
  enum { kGreedy, kList, kBin, kSum } way = set.heat == 0.0         ? kGreedy
                                            : set.most < p.vocab    ? kList
                                            : set.share < 1.0f      ? kBin
                                                                    : kSum;
  // A token's bin, counted down from the greatest's (NaN: none).  Levels are of logits less
  // `origin`: 0, or in finer bins the logit that these begin with, so that they are exact for
  // logits of any size.
  float origin = 0.0f;
  auto level_of = [&](float x) TMC_INLINE { return floorf((x - origin) * per_bin); };
  first_bin = level_of(top);
  auto bin_of = [&](float x) TMC_INLINE { return first_bin - level_of(x); };
  auto octaves = [&](float x) TMC_INLINE { return ((double)x - (double)top) * set.heat; };
  // 2^octaves in multiples of 2^-43: the last bits of that and 512.
  constexpr double kUnit = 0x1p43;
  auto integer = [&](double a) TMC_INLINE -> u64 {
    return __builtin_bit_cast(u64, exp2_of(a) + 512.0) - __builtin_bit_cast(u64, 512.0);
  };
  // The tokens of [low, roof) in bins counted from that of `ref`: numbers, or weights
  // relative to the bin's in units of 2^-11 (a sum of 2^20 tokens fits).  Returns how many of
  // the thread's are above.
  unsigned* rough = reinterpret_cast<unsigned*>(s.hist);
  float low = -INFINITY, roof = INFINITY, ref = top;
  auto fill_bins = [&]() TMC_INLINE -> int {
    for (int i = threadIdx.x; i < kBins; i += THREADS) rough[i] = 0;
    __syncthreads();
    const float width = 1.0f / octave;  // (a power of two)
    int above = 0;
    parts(begin, end, [&](int) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const float bin = bin_of(v[i]);
        if (v[i] >= roof) ++above;
        else if (v[i] >= low && bin < (float)kBins) {
          unsigned cost = 1;
          if (way == kBin)
            cost = (unsigned)__fmaf_rn(fast_exp2(__fmaf_rn(v[i] - ref, heat, bin * width)), 0x1p11f,
                                       0.5f);
          atomicAdd(&rough[(int)bin], cost);
        }
      }
    });
    __syncthreads();
    return above;
  };
  if (STAGE < 2 && !odd && (way == kList || way == kBin)) fill_bins();
  // The thread's bins, and the sum of all before them.
  auto take_bins = [&](double (&mine)[BINS], double& base, double& all) TMC_INLINE {
    const double sum = take_values(mine, [&](int i) TMC_INLINE {
      const double scale = way == kBin ? (double)fast_exp2((float)-i / octave) : 1.0;
      return i < kBins ? scale * (double)rough[i] : 0.0;
    });
    block_scan<THREADS>(sum, s, base, all);
  };
  // Of a token: what it weighs, 0 for one that is not kept: below the last that counts, or
  // ranked below `cut`.
  const double faintest = fmax(set.least, kFaintest);
  u64 cut = 0;
  auto weight = [&](float x, int at) TMC_INLINE -> u64 {
    const double a = octaves(x);
    return a >= faintest && rank_key(x, at) >= cut ? integer(a) : 0;
  };
  auto say = [&](int token, double share) TMC_INLINE {
    p.tokens[row] = token;
    if (p.probability) p.probability[row] = (float)share;
  };
  // The least logit of a level from `low` on: 64 of the remaining floats at a time, in
  // their order, from -inf (which has none) up.
  auto least_of = [&](float low) TMC_INLINE -> float {
    constexpr u64 kFirst = 0x007FFFFFull, kLast = 0xFF800000ull;  // keys of -inf and inf
    u64 below = kFirst;
#pragma unroll
    for (int shift = 30; shift >= 0; shift -= 6) {
      const u64 at = below + ((u64)lane << shift);
      const bool less = at <= kLast && !(level_of(key_value(at << 32)) >= low);
      below += (u64)max(__popcll(__ballot(less)) - 1, 0) << shift;
    }
    return key_value((below + 1) << 32);
  };
  // Tokens into the list: each wave its own, by index, then all of them together.
  constexpr int WAVES = THREADS / kWave, OWN = 2 * kMostKept / WAVES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  unsigned* queue = reinterpret_cast<unsigned*>(s.keys) + wave * OWN;
  int queued = 0;  // of this wave
  auto collect = [&](bool take, int token) TMC_INLINE {
    const u64 takes = __ballot(take);
    if (takes == 0) return;
    const int slot = queued + __builtin_amdgcn_mbcnt_hi((unsigned)(takes >> 32),
                                                        __builtin_amdgcn_mbcnt_lo((unsigned)takes, 0));
    if (take && slot < OWN) queue[slot] = (unsigned)token;
    queued += __popcll(takes);
  };
  // Returns how many there are, above kMostKept where they are too many.
  auto collected = [&]() TMC_INLINE -> int {
    constexpr int KEPT = kMostKept / THREADS;
    int* counts = reinterpret_cast<int*>(s.words);
    __syncthreads();
    if (lane == 0) counts[wave] = queued;
    __syncthreads();
    int n = 0, ends[WAVES];
    bool fits = true;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      fits &= counts[w] <= OWN;
      ends[w] = n += counts[w];
    }
    if (!fits || n > kMostKept) return kMostKept + 1;
    u64 keys[KEPT];
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = e * THREADS + (int)threadIdx.x;
      keys[e] = 0;
      if (i >= n) continue;
      int slot = i;
#pragma unroll
      for (int w = 1; w < WAVES; ++w)
        if (i >= ends[w - 1]) slot = w * OWN + i - ends[w - 1];
      const int token = (int)reinterpret_cast<const unsigned*>(s.keys)[slot];
      keys[e] = rank_key((float)x[token], token);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < KEPT; ++e) {
      const int i = e * THREADS + (int)threadIdx.x;
      if (i < n) s.keys[i] = keys[e];
    }
    __syncthreads();
    return n;
  };
  float high = 0.0f;  // the list's logits: from low on, below high
  // The sums of the block's parts: of the tokens from the logit `high` on (all, where none
  // are listed) that min-p keeps; those from `low` on and below `high` into the list.
  // Returns the sum of all tokens' weights, of this thread (0 where none are listed).
  u64* groups = s.groups;
  auto sum_groups = [&](auto lists) TMC_INLINE -> u64 {
    u64 all = 0;
    for (int g = threadIdx.x; g < kMostGroups; g += THREADS) groups[g] = 0;
    __syncthreads();
    parts(begin, end, [&](int at) TMC_INLINE {
      u64 sum = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const double a = octaves(v[i]);
        const u64 w = integer(fmax(a, -60.0));  // (below 2^-44, and of NaN: 0)
        if (lists) all += w;
        if ((!lists || v[i] >= high) && a >= faintest) sum += w;
        if (lists) collect(v[i] >= low && v[i] < high, place(at, i));
      }
      sum = wave_scan(sum);
      if (lane == kWave - 1 && sum) atomicAdd(&groups[(at - begin) / PART], sum);
    });
    __syncthreads();
    return all;
  };
  auto count_groups = [&](int tokens) TMC_INLINE { return (tokens + PART - 1) / PART; };

  // The bins [from, to] that are listed: that in which the running sum, `above` before it and
  // `reached` with it, reaches its aim, and its neighbours where the border is nearer than
  // rough sums are exact (half a unit of a token's 2^11 and more, and as much of the aim); or,
  // where min-p ends before them, the bins around the least logit that it keeps.
  bool by_least = false;  // the latter
  auto bounds = [&](int bin, double above, double reached, double aim, double all) TMC_INLINE {
    int from = 0, to = bin;
    if (way == kBin) {
      const double near = 6e-4 * all;
      from = max(0, bin - (aim - above < near));
      to = bin + (reached - aim < near);
      const float least = bin_of((float)((double)top + faintest / set.heat)) - 1.0f;
      by_least = set.least > kFaintest && least < (float)from;
      if (by_least) {
        from = max((int)least, 0);
        to = min(to, (int)least + 2);
      }
    }
    low = least_of(first_bin - (float)to);
    high = from > 0 ? least_of(first_bin - (float)from + 1.0f) : roof;
  };

  // ---- the row's blocks together: every word at agent scope, completed before the
  // arrival is counted; the last of them goes on
  auto put = [](auto* to, auto value) TMC_INLINE {
    __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto get = [](const auto* from) TMC_INLINE {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto arrive = [&]() TMC_INLINE -> bool {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      int* count = p.arrivals + row * kCounterStride;
      s.last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               p.count - 1;
      if (s.last) put(count, 0);
    }
    __syncthreads();
    const bool last = s.last;
    __syncthreads();
    return last;
  };
  u64* blocks = p.blocks + (size_t)row * p.count;
  if constexpr (STAGE == 1) {
    float* bins = p.bins + (size_t)row * p.count * kBins;
    if (!odd && (way == kList || way == kBin)) {
      double mine[BINS], base, all;
      take_bins(mine, base, all);
#pragma unroll
      for (int e = 0; e < BINS; ++e) {
        const int i = (int)threadIdx.x * BINS + e;
        base += mine[e];
        if (i < kBins) put(bins + (size_t)split * kBins + i, (float)base);
      }
    }
    if (threadIdx.x == 0) put(blocks + split, best);
    if (!arrive()) return;
    best = 0;
    odd = set.most < p.vocab && set.most > kMostTopK;
    for (int b = threadIdx.x; b < p.count; b += THREADS) {
      const u64 other = get(blocks + b);
      highs[b] = other ? key_value(other) : -INFINITY;  // (of -inf alone: no bins, passed over)
      best = max(best, other);
      odd |= other && is_odd(highs[b], INFINITY);
    }
    odd = __syncthreads_or(odd);
    best = block_max_u64<THREADS>(best, s);
    odd |= best == 0;
    top = best ? key_value(best) : -INFINITY;
    odd |= is_odd(top, kMostLevel);
    first_bin = level_of(top);
    if (way == kGreedy && best) {
      odd = false;
      if (threadIdx.x == 0) say(key_index(best), 1.0);
    }
    if (!odd && (way == kList || way == kBin)) {
      double sum = 0.0, base, all;
      for (int b = threadIdx.x; b < p.count; b += THREADS) {
        const double a = octaves(highs[b]);
        factors[b] = way == kList ? 1.0 : a >= kFaintest ? exp2_of(a) : 0.0;
        sum += highs[b] > -INFINITY ? factors[b] * (double)get(bins + (size_t)b * kBins + kBins - 1) : 0.0;
      }
      block_scan<THREADS>(sum, s, base, all);
      // The running sum of the row's bins up to bin i: of this thread's share of its blocks,
      // every `step`-th.
      auto merged = [&](int i, int first, int step) TMC_INLINE -> double {
        constexpr int kAhead = 4;  // blocks at once
        double sum = 0.0;
        for (int b0 = first; b0 < p.count; b0 += kAhead * step) {
          float in[kAhead];
          double factor[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int b = min(b0 + u * step, p.count - 1);
            const float behind = bin_of(highs[b]);
            const bool here = b0 + u * step < p.count && behind <= (float)i;
            in[u] = get(bins + (size_t)(here ? b : split) * kBins + (here ? i - (int)behind : 0));
            factor[u] = here ? factors[b] : 0.0;
          }
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (factor[u] > 0.0) sum += factor[u] * (double)in[u];
        }
        return sum;
      };
      // in two steps: the coarse ones' running sums, then those of one's bins
      const double aim = way == kList ? (double)set.most : (double)set.share * all;
      constexpr int LANES = THREADS / kCoarse;
      int first = 0;
      double above = 0.0, reached = 0.0;
#pragma unroll 1
      for (int step = kCoarse; step >= 1; step /= kCoarse) {
        const int point = (int)threadIdx.x / LANES, i = first + (point + 1) * step - 1;
        double mine = i < kBins ? merged(i, (int)threadIdx.x % LANES, LANES) : 0.0;
#pragma unroll
        for (int off = 1; off < LANES; off <<= 1) mine += __shfl_xor(mine, off, kWave);
        __syncthreads();
        if (threadIdx.x % LANES == 0) s.levels[point] = i < kBins ? mine : INFINITY;
        __syncthreads();
        int at = 0;
        while (at < kCoarse - 1 && s.levels[at] < aim) ++at;
        if (at > 0) above = s.levels[at - 1];
        reached = s.levels[at];
        first = min(first + at * step, kBins - step);
      }
      bounds(first, above, reached, aim, all);
    }
    if (threadIdx.x == 0) *record = {best, low, high, odd, by_least, 0};
    return;
  }
  if (STAGE == 2) {
    if (odd && split > 0) return;
    if (!odd && way == kGreedy) return;
    low = record->low;
    high = record->high;
    by_least = record->least;
  }
  auto by_bins = [&]() TMC_INLINE -> bool {
    bool done = best != 0 && !odd;
    if (way == kGreedy && best) {
      if (threadIdx.x == 0) say(key_index(best), 1.0);
      return true;
    }
    u64 weights = 0;  // of all tokens, this thread's
    if (done) {
      // the bins' running sum reaches `aim`: the list's bounds
      auto find_bounds = [&](double aim, bool share) TMC_INLINE {
        double mine[BINS], base, all, above;
        take_bins(mine, base, all);
        if (share) aim *= all;
        const int bin = max(find_in<THREADS, false>(mine, base, aim, above, s), 0);
        const double scale = way == kBin ? (double)fast_exp2((float)-bin / octave) : 1.0;
        bounds(bin, above, above + scale * rough[bin], aim, all);
      };
      if (STAGE == 0 && way != kSum)
        find_bounds(way == kList ? (double)set.most : (double)set.share, way == kBin);
      if (way == kList) {
        parts(begin, end, [&](int at) TMC_INLINE {
#pragma unroll
          for (int i = 0; i < EACH; ++i) collect(v[i] >= low, place(at, i));
        });
      } else if (way == kBin) {
        weights = sum_groups(std::true_type());
      } else {
        sum_groups(std::false_type());
      }
      int n = way == kSum ? 0 : collected();
      if constexpr (STAGE == 2) {
        // its tokens and sums to the row's
        u64* list = p.lists + (size_t)row * kMostKept;
        u64* sums = p.sums + (size_t)row * p.count * p.walk;
        if (n > 0) {
          if (threadIdx.x == 0)
            s.found = __hip_atomic_fetch_add(&record->listed, n, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT);
          __syncthreads();
          const int first = s.found;
          for (int i = threadIdx.x; i < n && n <= kMostKept && first + i < kMostKept; i += THREADS)
            put(list + first + i, s.keys[i]);
        }
        if (way != kList)
          for (int g = threadIdx.x; g < p.walk; g += THREADS) put(sums + split * p.walk + g, groups[g]);
        weights = block_sum_u64<THREADS>(weights, s);
        if (threadIdx.x == 0) put(blocks + split, weights);
        if (!arrive()) return true;
        n = get(&record->listed);
        weights = 0;
        for (int b = threadIdx.x; b < p.count; b += THREADS) weights += get(blocks + b);
        if (way != kList)
          for (int g = threadIdx.x; g < count_groups(p.vocab); g += THREADS) groups[g] = get(sums + g);
        for (int i = threadIdx.x; i < min(n, kMostKept); i += THREADS) s.keys[i] = get(list + i);
        __syncthreads();
      }
      // too many: those bins in 64 finer ones each, as long as that tells tokens apart
#pragma unroll 1
      for (int level = 0; level < 3 && n > kMostKept && !(set.least > kFaintest); ++level) {
        double aim = 0.0;
        roof = way == kBin ? high : least_of(level_of(low) + 1.0f);
        // (the greatest logit below the roof: where logits are far apart next to the bins' width
        // the roof itself is many bins away)
        ref = fminf(key_value(rank_key(roof, 0) - (1ull << 32)), top);
        if (way == kBin) {
          u64 mine = 0;
          for (int g = threadIdx.x; g < count_groups(p.vocab); g += THREADS) mine += groups[g];
          const u64 total = block_sum_u64<THREADS>(weights, s), ahead = block_sum_u64<THREADS>(mine, s);
          aim = ((double)set.share * (double)total - (double)ahead) * (0x1p11 / kUnit) /
                exp2_of(octaves(ref));
        }
        octave *= 64.0f;
        per_bin = heat * octave;
        origin = ref;
        first_bin = level_of(ref);
        begin = 0;
        end = p.vocab;
        queued = 0;
        const int above = fill_bins();
        if (way == kList) aim = (double)set.most - (double)block_sum_u64<THREADS>((u64)above, s);
        find_bounds(aim, false);
        if (way == kList) {
          parts(begin, end, [&](int at) TMC_INLINE {
#pragma unroll
            for (int i = 0; i < EACH; ++i) collect(v[i] >= low, place(at, i));
          });
        } else {
          weights = sum_groups(std::true_type());
        }
        n = collected();
      }
      done = n <= kMostKept;
      double limit = INFINITY;  // top-p: tokens before which less than that lies stay
      double above = 0.0;       // the sum before the list
      if (done && way != kSum) {
        __syncthreads();
        u64 low = ~0ull, high = 0;  // of the list's keys
        for (int i = threadIdx.x; i < n; i += THREADS) {
          const u64 key = s.keys[i];
          low = min(low, key);
          high = max(high, key);
          const double a = octaves(key_value(key));
          costs[i] = a >= kFaintest ? integer(a) : 0;
        }
        high = block_max_u64<THREADS>(high, s);
        low = ~block_max_u64<THREADS>(~low, s);
        if (way == kBin) {
          // exact sums: of all, and of what lies before the list
          u64 before, total, ahead;
          block_scan<THREADS>(weights, s, before, total);
          limit = (double)set.share * ((double)total * (1.0 / kUnit));
          u64 mine = 0;
          for (int g = threadIdx.x; g < count_groups(p.vocab); g += THREADS) mine += groups[g];
          block_scan<THREADS>(mine, s, before, ahead);
          above = (double)ahead * (1.0 / kUnit);
          // the bins said that the cut is in the list (or, where min-p ends before it, in it or
          // behind it): the tokens must bear it out
          u64 sum = 0, all;
          for (int i = threadIdx.x; i < n; i += THREADS) sum += costs[i];
          block_scan<THREADS>(sum, s, before, all);
          const double listed = (double)all * (1.0 / kUnit);
          done = (above == 0.0 || above < limit) &&
                 (by_least || (n > 0 && above + listed >= limit));
        }
        // top-k, then top-p: (in a loop, for one copy of its code)
#pragma unroll 1
        for (int step = way == kList ? 0 : 1; step < 2 && n > 0 && done; ++step) {
          u64 target = (u64)set.most;
          if (step == 0) {
            cut = low;  // (nothing behind the list)
            if (n <= set.most) continue;
          } else {
            if (set.share == 1.0f) break;
            cut = max(cut, low);
            if (way == kList) {
              u64 sum = 0, before, all;
              for (int i = threadIdx.x; i < n; i += THREADS)
                if (s.keys[i] >= cut) sum += costs[i];
              block_scan<THREADS>(sum, s, before, all);
              limit = (double)set.share * ((double)all * (1.0 / kUnit));
            }
            // (the most probable token stays)
            target = (u64)fmax(ceil((limit - above) * kUnit), 1.0);
          }
          cut = max(cut, select_key<THREADS>(n, low, high, target, s, [&](int i) TMC_INLINE {
                      return step == 0 ? (u64)1 : costs[i];
                    }));
        }
        // the list's kept tokens to the sums of their parts
        if (way == kList)
          for (int g = threadIdx.x; g < kMostGroups; g += THREADS) groups[g] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += THREADS) {
          const u64 key = s.keys[i];
          const double a = octaves(key_value(key));
          if (key >= cut && a >= faintest) atomicAdd(&groups[key_index(key) / PART], costs[i]);
        }
        __syncthreads();
      }
    }
    if (!done) return false;

    // ---- the draw
    constexpr int SUMS = kMostGroups / THREADS;  // a thread
    const int n = count_groups(p.vocab);
    u64 mine[SUMS], base, all, before;
    const u64 sum = take_values(mine, [&](int g) TMC_INLINE { return g < n ? groups[g] : 0ull; });
    block_scan<THREADS>(sum, s, base, all);
    if (all == 0) return false;
    u64 aim = min((u64)(set.uniform * (double)all), all - 1);
    const int g = find_in<THREADS, true>(mine, base, aim, before, s);
    if (g < 0) return false;
    aim -= before;
    u64 w[EACH], own = 0, part;
    parts(g * PART, min(p.vocab, (g + 1) * PART), [&](int at) TMC_INLINE {
#pragma unroll
      for (int i = 0; i < EACH; ++i) own += w[i] = weight(v[i], place(at, i));
    });
    block_scan<THREADS>(own, s, before, part);
    const int index = find_in<THREADS, true>(w, before, aim, before, s);
    if (index < 0) return false;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if ((int)threadIdx.x * EACH + i == index) say(g * PART + index, (double)w[i] / (double)all);
    return true;
  };
  if (!by_bins()) row_by_digits<T, THREADS>(p, row, set, s);
}

bool sample_shape(int64_t rows, int64_t vocabulary) {
  return rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary <= kMostTokens;
}

// How rows are shared out: a block a row, or, below kFewRows rows, blocks of 4096 tokens, up
// to kFill of them together.  fp16 rows of 32000 and of 128000 tokens, shared and not:
// 16 rows 33 and 54, 42 and 150 us; 256 rows 52 and 59, 112 and 180 us; 511 rows 71 and
// 72, 190 and 224 us.  kFill 512: 134 us for 256 rows of 128000 for 112, 2048: 68 us for 256
// rows of 32000 for 52.
constexpr int kThreads = 256, kEach = 8;
constexpr int64_t kFill = 1024, kFewRows = 512;
static_assert(kFewRows <= kSharedRows, "every shared row has its counter");
static_assert(kMostTokens / (kThreads * kEach) <= kMostGroups, "a sum a part");
struct SamplePlan {
  int walk, count;
};
SamplePlan sample_plan(int64_t rows, int64_t vocabulary) {
  const int64_t part = kThreads * kEach, parts = (vocabulary + part - 1) / part;
  int64_t blocks = 1;
  if (rows < kFewRows)
    blocks = std::max<int64_t>(
        1, std::min({(parts + 1) / 2, kFill / rows, (int64_t)kMostBlocks}));
  SamplePlan plan;
  plan.walk = (int)((parts + blocks - 1) / blocks);
  plan.count = (int)((parts + plan.walk - 1) / plan.walk);
  return plan;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_sample_workspace_bytes(int64_t rows, int64_t vocabulary) {
  if (!sample_shape(rows, vocabulary)) return 0;
  const SamplePlan plan = sample_plan(rows, vocabulary);
  const size_t block = sizeof(u64) * (1 + plan.walk) + sizeof(float) * kBins;
  return plan.count == 1 ? 0
                         : kCounterBytes + (size_t)rows * (sizeof(SampleRow) + plan.count * block +
                                                           kMostKept * sizeof(u64));
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
    p.records = reinterpret_cast<SampleRow*>(static_cast<char*>(workspace) + kCounterBytes);
    p.lists = reinterpret_cast<u64*>(p.records + rows);
    p.blocks = p.lists + rows * kMostKept;
    p.sums = p.blocks + rows * plan.count;
    p.bins = reinterpret_cast<float*>(p.sums + rows * plan.count * plan.walk);
  }
  const bool full = dtype == TMC_F32;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * plan.count)), dim3(kThreads), 0,
                       as_stream(stream), p);
  };
  if (plan.count == 1) {
    launch(full ? sample_kernel<float, kThreads, kEach, 0> : sample_kernel<half_t, kThreads, kEach, 0>);
  } else {
    launch(full ? sample_kernel<float, kThreads, kEach, 1> : sample_kernel<half_t, kThreads, kEach, 1>);
    launch(full ? sample_kernel<float, kThreads, kEach, 2> : sample_kernel<half_t, kThreads, kEach, 2>);
  }
  return check_launch("sample_kernel");
}
