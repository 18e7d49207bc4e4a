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
// Sums must come out alike whatever the order of their terms, and close enough
// that a draw next to a border falls on its right side: a weight is 2^a with a in
// 64 bits, rounded to a multiple of 2^-scale of the greatest, and sums are of
// 64-bit integers.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>

namespace tmc {
namespace {

typedef unsigned long long u64;

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
  int scale;           // weights are multiples of 2^-scale
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
  float uniform;
  int most;      // top_k, the vocabulary for all
};
__device__ __forceinline__ Settings settings_of(const SampleParams& p, int row) {
  const float t = p.temperature ? p.temperature[row] : 1.0f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float share = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p ? p.min_p[row] : 0.0f;
  Settings s;
  s.uniform = p.uniforms[row];
  s.heat = t >= kColdest ? 1.4426950408889634 / (double)t : 0.0;
  if (t == INFINITY) s.heat = 0x1p-1000;  // equal weights
  s.least = least > 0.0f ? log2((double)fminf(least, 1.0f)) : -INFINITY;
  s.share = share < 1.0f ? fmaxf(share, 0.0f) : 1.0f;
  s.most = k > 0 && k < p.vocab ? k : p.vocab;
  return s;
}

// ------------------------------------------------------------ a block a row
constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / kWave, kDigits = 256;

struct RowScratch {
  u64 hist[kDigits];
  u64 wave[kRowWaves];
  u64 found, below;
};

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
__device__ __forceinline__ u64 block_sum_u64(u64 v, RowScratch& s) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) s.wave[threadIdx.x / kWave] = v;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) sum += s.wave[w];
  return sum;
}

// The key at which the running cost, from the highest ranked down, reaches
// `target` (at least 1 and at most all of it): digit by digit, a histogram of the
// costs of the keys that agree so far.
template <typename EACH>
__device__ u64 cut_at(u64 target, RowScratch& s, const EACH& each) {
  u64 prefix = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < kDigits) s.hist[threadIdx.x] = 0;
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
      s.found = d;
      s.below = target - above;
    }
    __syncthreads();
    prefix |= s.found << shift;
    target = s.below;
  }
  return prefix;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleParams p) {
  __shared__ RowScratch s;
  const int row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  const Settings set = settings_of(p, row);
  // ---- the most probable token
  u64 best = 0;
  for (int i = threadIdx.x; i < p.vocab; i += kRowThreads) {
    const float v = (float)x[i];
    if (v == v) best = max(best, rank_key(v, i));
  }
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) best = max(best, (u64)__shfl_xor(best, off, kWave));
  if ((threadIdx.x & (kWave - 1)) == 0) s.wave[threadIdx.x / kWave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) best = max(best, s.wave[w]);
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
    return a >= kFaintest ? max((u64)rint(exp2(a) * unit), (u64)1) : 0;
  };
  u64 cut = 0;
  auto kept = [&](float v, int i) -> u64 {
    const u64 w = weight(v);
    return w && rank_key(v, i) >= cut ? w : 0;
  };
  if (set.most < p.vocab) {
    auto each = [&](auto&& take) {
      for (int i = threadIdx.x; i < p.vocab; i += kRowThreads) {
        const float v = (float)x[i];
        if (weight(v)) take(rank_key(v, i), 1);
      }
    };
    u64 count = 0;
    each([&](u64, u64 one) { count += one; });
    if (block_sum_u64(count, s) > (u64)set.most) cut = cut_at((u64)set.most, s, each);
  }
  if (set.share < 1.0f) {
    auto each = [&](auto&& take) {
      for (int i = threadIdx.x; i < p.vocab; i += kRowThreads) {
        const float v = (float)x[i];
        if (const u64 w = kept(v, i)) take(rank_key(v, i), w);
      }
    };
    u64 sum = 0;
    each([&](u64, u64 w) { sum += w; });
    sum = block_sum_u64(sum, s);
    const u64 target = max((u64)1, min(sum, (u64)ceil((double)set.share * (double)sum)));
    cut = max(cut, cut_at(target, s, each));
  }
  auto final_weight = [&](int i) -> u64 {
    const float v = (float)x[i];
    if (v != top && !(((double)v - (double)top) * set.heat >= set.least)) return 0;
    return kept(v, i);
  };
  u64 sum = 0;
  for (int i = threadIdx.x; i < p.vocab; i += kRowThreads) sum += final_weight(i);
  sum = block_sum_u64(sum, s);
  const double u = set.uniform > 0.0f ? (double)set.uniform : 0.0;
  const u64 target = u < 1.0 ? min(sum - 1, (u64)(u * (double)sum)) : sum - 1;
  // ---- the first kept token at which the running sum passes the target
  u64 before = 0;
  for (int at = 0;; at += kRowThreads) {
    const int i = at + threadIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const u64 w = i < p.vocab ? final_weight(i) : 0;
    u64 run = w;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const u64 other = __shfl_up(run, off, kWave);
      if (lane >= off) run += other;
    }
    __syncthreads();
    if (lane == kWave - 1) s.wave[wave] = run;
    __syncthreads();
    u64 all = 0;
    run += before;
#pragma unroll
    for (int v = 0; v < kRowWaves; ++v) {
      if (v < wave) run += s.wave[v];
      all += s.wave[v];
    }
    if (w && run > target && run - w <= target) {
      p.tokens[row] = i;
      if (p.probability) p.probability[row] = (float)((double)w / (double)sum);
    }
    before += all;
    if (before > target) break;
  }
}

bool sample_shape(int64_t rows, int64_t vocabulary) {
  return rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary <= kMostTokens;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_sample_workspace_bytes(int64_t rows, int64_t vocabulary) {
  if (!sample_shape(rows, vocabulary)) return 0;
  return 0;
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
  const hipStream_t s = as_stream(stream);
  if (dtype == TMC_F32)
    hipLaunchKernelGGL((sample_row_kernel<float>), dim3((unsigned)rows), dim3(kRowThreads), 0, s, p);
  else
    hipLaunchKernelGGL((sample_row_kernel<half_t>), dim3((unsigned)rows), dim3(kRowThreads), 0, s, p);
  return check_launch("sample_row_kernel");
}
