// Log probabilities of given tokens, the entropy of every row and its most
// probable tokens, from logits [rows, vocabulary].
//
// With m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(t) = x[t] - m - log S,   entropy = log S - T / S.
// A logit of -inf adds nothing to S or T.  The alternatives come in the greedy
// order of tmc_argmax_f32 (the greater first, equals by the lower index, NaN
// never).
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>

namespace tmc {
namespace {

constexpr int kTopMax = 64;
constexpr int kLpThreads = 256;

struct LogprobParams {
  const void* logits;
  const int32_t* tokens;  // may be null: no given tokens
  float* logprob;
  float* entropy;  // may be null
  int32_t* top_tokens;
  float* top_logprobs;
  long stride;
  int rows, vocab, top;
};

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(LogprobParams p) {
  __shared__ double s_s[kLpThreads / kWave], s_t[kLpThreads / kWave];
  __shared__ float s_a[kLpThreads / kWave];
  __shared__ int s_i[kLpThreads / kWave];
  const int row = blockIdx.x, wave = threadIdx.x / kWave;
  const bool first = threadIdx.x % kWave == 0;
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) m = fmaxf(m, to_float<T>(x[i]));
  m = cross_max<1>(m);
  if (first) s_a[wave] = m;
  __syncthreads();
  for (int w = 0; w < kLpThreads / kWave; ++w) m = fmaxf(m, s_a[w]);
  __syncthreads();
  // sums in 64 bits: equal terms in a long fp32 sum round the same way each time
  double s = 0.0, t = 0.0;
  for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
    const float d = to_float<T>(x[i]) - m, e = expf(d);
    s += e;
    t += e == 0.0f ? 0.0f : e * d;
  }
  for (int off = 1; off < kWave; off <<= 1) {
    s += __shfl_xor(s, off, kWave);
    t += __shfl_xor(t, off, kWave);
  }
  if (first) {
    s_s[wave] = s;
    s_t[wave] = t;
  }
  __syncthreads();
  s = t = 0.0;
  for (int w = 0; w < kLpThreads / kWave; ++w) {
    s += s_s[w];
    t += s_t[w];
  }
  const float log_s = logf((float)s);
  if (threadIdx.x == 0) {
    if (p.entropy) p.entropy[row] = log_s - (float)(t / s);
    if (p.tokens) {
      const int token = p.tokens[row];
      if (token >= 0 && token < p.vocab) p.logprob[row] = to_float<T>(x[token]) - m - log_s;
    }
  }
  // one alternative a round: the best of those behind the previous one
  float above = INFINITY;
  int after = -1;
  bool any = false;
  for (int k = 0; k < p.top; ++k) {
    float best = -INFINITY;
    int which = -1;
    for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
      const float v = to_float<T>(x[i]);
      const bool behind = !any || v < above || (v == above && i > after);
      if (behind && argmax_better(v, i, best, which)) {
        best = v;
        which = i;
      }
    }
    argmax_wave(best, which);
    __syncthreads();
    if (first) {
      s_a[wave] = best;
      s_i[wave] = which;
    }
    __syncthreads();
    for (int w = 0; w < kLpThreads / kWave; ++w)
      if (argmax_better(s_a[w], s_i[w], best, which)) {
        best = s_a[w];
        which = s_i[w];
      }
    if (threadIdx.x == 0) {
      p.top_tokens[(size_t)row * p.top + k] = which;
      p.top_logprobs[(size_t)row * p.top + k] = which < 0 ? -INFINITY : best - m - log_s;
    }
    above = which < 0 ? -INFINITY : best;
    after = which < 0 ? p.vocab : which;
    any = true;
  }
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_logprobs_workspace_bytes(int64_t rows, int64_t vocabulary, int64_t top) {
  return 0;
}

extern "C" int tmc_logprobs(const void* logits, int dtype, int64_t row_stride,
                            const int32_t* tokens, float* logprob, float* entropy,
                            int32_t* top_tokens, float* top_logprobs, int64_t rows,
                            int64_t vocabulary, int64_t top, void* workspace,
                            size_t workspace_bytes, void* stream) {
  TMC_REQUIRE(logits, "Log probabilities: null device pointer.");
  TMC_REQUIRE(dtype == TMC_F32 || dtype == TMC_F16,
              "Log probabilities: logits must be f32 or f16.");
  TMC_REQUIRE(rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary < (1LL << 28) &&
                  row_stride >= vocabulary && row_stride < (1LL << 40),
              "Log probabilities: invalid shape.");
  TMC_REQUIRE(top >= 0 && top <= kTopMax && top <= vocabulary,
              "Log probabilities: top must be in [0, 64] and within the vocabulary.");
  TMC_REQUIRE(!tokens == !logprob, "Log probabilities: tokens and logprob go together.");
  TMC_REQUIRE(!top || (top_tokens && top_logprobs),
              "Log probabilities: null pointer for the alternatives.");
  TMC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == TMC_F32 ? 4 : 2) == 0,
              "Log probabilities: logits must be aligned to their elements.");
  const size_t need = tmc_logprobs_workspace_bytes(rows, vocabulary, top);
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "Log probabilities: workspace is smaller than tmc_logprobs_workspace_bytes().");
  LogprobParams p{};
  p.logits = logits;
  p.tokens = tokens;
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_tokens = top_tokens;
  p.top_logprobs = top_logprobs;
  p.stride = (long)row_stride;
  p.rows = (int)rows;
  p.vocab = (int)vocabulary;
  p.top = (int)top;
  if (dtype == TMC_F32)
    hipLaunchKernelGGL((logprobs_kernel<float>), dim3((unsigned)rows), dim3(kLpThreads), 0,
                       as_stream(stream), p);
  else
    hipLaunchKernelGGL((logprobs_kernel<half_t>), dim3((unsigned)rows), dim3(kLpThreads), 0,
                       as_stream(stream), p);
  return check_launch("logprobs_kernel");
}
