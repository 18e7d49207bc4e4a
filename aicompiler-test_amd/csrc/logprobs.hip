// Log probabilities of given tokens, the entropy of every row and its most
// probable tokens, from logits [rows, vocabulary].
//
// With m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(t) = x[t] - m - log S,   entropy = log S - T / S.
// A logit of -inf adds nothing to S or T.  The alternatives come in the greedy
// order of tmc_argmax_f32 (the greater first, equals by the lower index, NaN
// never).
//
// Bound by reading the logits once.  A row is cut into parts, one block each;
// a wave holds its elements of the part in registers, so the maximum, the sums
// and the alternatives are three passes over registers, not over memory.  The
// last block of a row to arrive joins the parts in their order.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>

namespace tmc {
namespace {

constexpr int kTopMax = 64;
constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / kWave;
constexpr size_t kLpCounterBytes = 64u << 10;
// Candidates a block ranks; one with more (many equal logits) picks its best
// one by one.
constexpr int kCandidates = 256;
constexpr long long kNoKey = (long long)0x8000000000000000ull;

struct LogprobParams {
  const void* logits;
  const int32_t* tokens;  // may be null: no given tokens
  float* logprob;
  float* entropy;  // may be null
  int32_t* top_tokens;
  float* top_logprobs;
  float* parts;   // [rows][count](m, S, T), then [rows][count][top] values, then indices
  int* arrivals;  // [rows]
  long stride;
  int rows, vocab, top;
  int count;      // parts a row
};

// A logit and its index as one number, greater in the greedy order first: the
// float's bits in the order of its value (-0 as +0; no NaN), then the lower
// index.
__device__ __forceinline__ long long key_of(float v, int index) {
  const int b = __builtin_bit_cast(int, v + 0.0f);
  const int order = b >= 0 ? b : b ^ 0x7FFFFFFF;
  return ((long long)order << 32) | (unsigned)~index;
}
__device__ __forceinline__ float key_value(long long key) {
  const int order = (int)(key >> 32);
  return __builtin_bit_cast(float, order >= 0 ? order : order ^ 0x7FFFFFFF);
}
__device__ __forceinline__ int key_index(long long key) { return (int)~(unsigned)key; }

// Wave-wide maximum in every lane, by exchanges inside registers.
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kDppQuadSwap1>(v));
  v = fmaxf(v, dpp<kDppQuadSwap2>(v));
  v = fmaxf(v, dpp<kDppRowHalfMirror>(v));
  v = fmaxf(v, dpp<kDppRowMirror>(v));
  return fmaxf(fmaxf(readlane(v, 0), readlane(v, 16)), fmaxf(readlane(v, 32), readlane(v, 48)));
}

// (m, S, T) of two sets of logits together.  S and T are relative to m.
struct Mass {
  float m;
  double s, t;
  __device__ __forceinline__ void add(float om, double os, double ot) {
    const float next = fmaxf(m, om);
    if (next == -INFINITY) {  // two empty sets (their NaNs stay)
      s += os;
      t += ot;
      return;
    }
    const double da = (double)m - next, db = (double)om - next;
    // an empty set weighs nothing; 0 * inf must not arise
    const double ea = m == -INFINITY ? 0.0 : (double)expf((float)da);
    const double eb = om == -INFINITY ? 0.0 : (double)expf((float)db);
    t = (m == -INFINITY ? t : ea * (t + s * da)) + (om == -INFINITY ? ot : eb * (ot + os * db));
    s = (m == -INFINITY ? s : ea * s) + (om == -INFINITY ? os : eb * os);
    m = next;
  }
};

// The best `top` of `count` distinct keys (at most kCandidates) to the places their rank
// gives them, the rest of the places empty.  Ends with a barrier.
__device__ __forceinline__ void rank_keys(const long long* keys, int count, int top,
                                          long long* out) {
  const int me = threadIdx.x;
  if (me < top) out[me] = kNoKey;
  __syncthreads();
  const long long mine = me < count ? keys[me] : kNoKey;
  if (mine != kNoKey) {
    int rank = 0, o = 0;
    for (; o + 8 <= count; o += 8)
#pragma unroll
      for (int u = 0; u < 8; ++u) rank += keys[o + u] > mine ? 1 : 0;
    for (; o < count; ++o) rank += keys[o] > mine ? 1 : 0;
    if (rank < top) out[rank] = mine;
  }
  __syncthreads();
}

// EACH: elements a lane holds; a part is kLpThreads * EACH elements.
template <typename T, int EACH>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(LogprobParams p) {
  constexpr int VEC = 16 / (int)sizeof(T);  // elements a load
  constexpr int LOADS = EACH / VEC;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  // rows start anywhere on an element boundary
  typedef vec unaligned __attribute__((aligned(sizeof(T))));
  static_assert(kCandidates == kLpThreads, "a thread a candidate");
  __shared__ __align__(16) long long s_keys[kCandidates];
  __shared__ __align__(16) long long s_best[kTopMax];
  __shared__ float s_m[kLpWaves], s_bound[kLpWaves];
  __shared__ double s_s[kLpWaves], s_t[kLpWaves];
  __shared__ int s_reach[kLpWaves], s_found, s_last;
  const int part = blockIdx.x % p.count, row = blockIdx.x / p.count;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  // the wave's elements: loads of 64 lanes x VEC, load after load
  const int base = part * (kLpThreads * EACH) + wave * (kWave * EACH) + lane * VEC;
  float v[EACH];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int at = base + i * kWave * VEC;
    if (at + VEC <= p.vocab) {
      const vec in = *reinterpret_cast<const unaligned*>(x + at);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = (float)in[e];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        v[i * VEC + e] = at + e < p.vocab ? (float)x[at + e] : -INFINITY;
    }
  }
  float mine = -INFINITY;  // the lane's greatest (NaN left out)
#pragma unroll
  for (int i = 0; i < EACH; ++i) mine = fmaxf(mine, v[i]);
  const float m = wave_max(mine);
  // A wave of -inf or nothing adds nothing; its NaNs spoil the sums all the same.
  const float shift = m == -INFINITY ? 0.0f : m;
  float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f}, t4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float d = v[i] - shift, e = fast_exp2(d * 1.44269504f);
    s4[i & 3] += e;
    t4[i & 3] += e == 0.0f ? 0.0f : e * d;
  }
  // 32 bits over at most 8 + 2 + 4 additions, 64 above
  const float s16 = group_sum<16>((s4[0] + s4[1]) + (s4[2] + s4[3]));
  const float t16 = group_sum<16>((t4[0] + t4[1]) + (t4[2] + t4[3]));
  double s = 0.0, t = 0.0;
#pragma unroll
  for (int r = 0; r < kWave; r += 16) {
    s += readlane(s16, r);
    t += readlane(t16, r);
  }
  // ---- a bound that at least `top` of the block's elements reach, from the
  // lanes' greatest: each wave finds what its share of them reach
  const int top = p.top;
  const int part_at = part * (kLpThreads * EACH);
  if (top > 0) {
    // waves whose lanes all hold elements
    const int full = min(kLpWaves, (p.vocab - part_at + kWave * (EACH - VEC)) / (kWave * EACH));
    const int need = full > 0 ? (top + full - 1) / full : top;
    float rest = mine, bound = -INFINITY;
    int reach = 0;
    while (reach < need) {
      const float most = wave_max(rest);
      if (most == -INFINITY) {
        bound = -INFINITY;
        break;
      }
      bound = most;
      reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(rest == most));
      if (rest == most) rest = -INFINITY;
    }
    if (lane == 0) {
      s_bound[wave] = bound;
      s_reach[wave] = reach;
    }
  }
  if (lane == 0) {
    s_m[wave] = m;
    s_s[wave] = s;
    s_t[wave] = t;
  }
  if (threadIdx.x == 0) s_found = 0;
  __syncthreads();
  Mass mass{s_m[0], s_s[0], s_t[0]};
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) mass.add(s_m[w], s_s[w], s_t[w]);
  if (top > 0) {
    float bound = -INFINITY;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
      int reach = 0;
#pragma unroll
      for (int u = 0; u < kLpWaves; ++u) reach += s_bound[u] >= s_bound[w] ? s_reach[u] : 0;
      if (reach >= top) bound = fmaxf(bound, s_bound[w]);
    }
    // ---- the elements that reach it
    if (m >= bound) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = base + i / VEC * kWave * VEC + i % VEC;
        const bool in = v[i] >= bound && at < p.vocab;  // a NaN never
        if (__builtin_amdgcn_ballot_w64(in) != 0 && in) {
          const int place = atomicAdd(&s_found, 1);
          if (place < kCandidates) s_keys[place] = key_of(v[i], at);
        }
      }
    }
    __syncthreads();
    const int found = s_found;
    if (found <= kCandidates) {
      rank_keys(s_keys, found, top, s_best);
    } else {
      // too many: one a round, the best behind the one before
      long long last = 0x7FFFFFFFFFFFFFFFll;
      for (int k = 0; k < top; ++k) {
        long long best = kNoKey;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int at = base + i / VEC * kWave * VEC + i % VEC;
          const long long key = key_of(v[i], at);
          if (at < p.vocab && v[i] == v[i] && key < last && key > best) best = key;
        }
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
          const long long other = __shfl_xor(best, off, kWave);
          best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) s_keys[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) best = s_keys[w] > best ? s_keys[w] : best;
        if (threadIdx.x == 0) s_best[k] = best;
        last = best;
      }
      __syncthreads();
    }
  }

  // ---- the row's blocks together
  if (p.count > 1) {
    const size_t slots = (size_t)p.rows * p.count, slot = (size_t)row * p.count + part;
    double* sums = reinterpret_cast<double*>(p.parts);            // [slots][2]
    long long* keys = reinterpret_cast<long long*>(sums + 2 * slots);  // [slots][top]
    float* maxima = reinterpret_cast<float*>(keys + slots * top);
    // every word at agent scope, completed before the arrival is counted
    if (threadIdx.x == 0) {
      __hip_atomic_store(sums + 2 * slot, mass.s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * slot + 1, mass.t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(maxima + slot, mass.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((int)threadIdx.x < top)
      __hip_atomic_store(keys + slot * top + threadIdx.x, s_best[threadIdx.x], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      s_last = __hip_atomic_fetch_add(p.arrivals + row, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == p.count - 1;
      s_found = 0;
    }
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0)
      __hip_atomic_store(p.arrivals + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const size_t first = (size_t)row * p.count;
    // lane by lane over the parts, then over the lanes: the same order each time
    Mass all{-INFINITY, 0.0, 0.0};
    long long bound = kNoKey;  // the greatest of the parts' last keys: `top` keys reach it
    for (int i = lane; i < p.count; i += kWave) {
      all.add(__hip_atomic_load(maxima + first + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
              __hip_atomic_load(sums + 2 * (first + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
              __hip_atomic_load(sums + 2 * (first + i) + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      if (top > 0) {
        const long long key = __hip_atomic_load(keys + (first + i) * top + top - 1,
                                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        bound = key > bound ? key : bound;
      }
    }
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const float om = __shfl_xor(all.m, off, kWave);
      const double os = __shfl_xor(all.s, off, kWave), ot = __shfl_xor(all.t, off, kWave);
      all.add(om, os, ot);
      const long long other = __shfl_xor(bound, off, kWave);
      bound = other > bound ? other : bound;
    }
    mass = all;
    if (top > 0) {
      const int total = p.count * top;
      const long long* from = keys + first * top;
      for (int i = threadIdx.x; i < total; i += kLpThreads) {
        const long long key =
            __hip_atomic_load(from + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (key != kNoKey && key >= bound) {
          const int place = atomicAdd(&s_found, 1);
          if (place < kCandidates) s_keys[place] = key;
        }
      }
      __syncthreads();
      if (s_found <= kCandidates) {
        rank_keys(s_keys, s_found, top, s_best);
      } else {
        // the best so far and the next keys, as many as fit
        constexpr int kNext = kCandidates - kTopMax;
        if ((int)threadIdx.x < top) s_best[threadIdx.x] = kNoKey;
        __syncthreads();
        for (int at = 0; at < total; at += kNext) {
          const int n = min(kNext, total - at), i = threadIdx.x;
          if (i < top) s_keys[i] = s_best[i];
          if (i < n)
            s_keys[top + i] =
                __hip_atomic_load(from + at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __syncthreads();
          rank_keys(s_keys, top + n, top, s_best);
        }
      }
    }
  }

  // ---- the row
  // -inf alone: 0 / 0, a NaN as the other rows without a distribution
  const float log_s = mass.m == -INFINITY ? __builtin_nanf("") : logf((float)mass.s);
  if (threadIdx.x == 0) {
    if (p.entropy) p.entropy[row] = log_s - (float)(mass.t / mass.s);
    if (p.tokens) {
      const int token = p.tokens[row];
      if (token >= 0 && token < p.vocab) p.logprob[row] = (float)x[token] - mass.m - log_s;
    }
  }
  if ((int)threadIdx.x < top) {
    const long long key = s_best[threadIdx.x];
    const size_t to = (size_t)row * top + threadIdx.x;
    p.top_tokens[to] = key == kNoKey ? -1 : key_index(key);
    p.top_logprobs[to] = key == kNoKey ? -INFINITY : key_value(key) - mass.m - log_s;
  }
}

// Elements a lane holds: 8 where the rows are too few to fill the chip, else 32.
int each_of(int64_t rows, int64_t vocabulary) {
  return rows * ((vocabulary + 32 * kLpThreads - 1) / (32 * kLpThreads)) < 512 ? 8 : 32;
}
int64_t parts_of(int64_t rows, int64_t vocabulary) {
  const int64_t span = (int64_t)kLpThreads * each_of(rows, vocabulary);
  return (vocabulary + span - 1) / span;
}
bool logprob_shape(int64_t rows, int64_t vocabulary, int64_t top) {
  return rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary < (1LL << 28) && top >= 0 &&
         top <= kTopMax && top <= vocabulary && rows * parts_of(rows, vocabulary) < (1LL << 31);
}
size_t logprob_counter_bytes(int64_t rows) {
  return std::max(kLpCounterBytes, (size_t)(rows * 4 + 255) / 256 * 256);
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_logprobs_workspace_bytes(int64_t rows, int64_t vocabulary, int64_t top) {
  if (!logprob_shape(rows, vocabulary, top)) return 0;
  const int64_t parts = parts_of(rows, vocabulary);
  return parts == 1 ? 0 : logprob_counter_bytes(rows) + (size_t)(rows * parts) * (20 + 8 * top);
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
                  row_stride >= vocabulary && row_stride < (1LL << 36),
              "Log probabilities: invalid shape.");
  TMC_REQUIRE(top >= 0 && top <= kTopMax && top <= vocabulary,
              "Log probabilities: top must be in [0, 64] and within the vocabulary.");
  TMC_REQUIRE(logprob_shape(rows, vocabulary, top), "Log probabilities: invalid shape.");
  TMC_REQUIRE(!tokens == !logprob, "Log probabilities: tokens and logprob go together.");
  TMC_REQUIRE(!top || (top_tokens && top_logprobs),
              "Log probabilities: null pointer for the alternatives.");
  TMC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == TMC_F32 ? 4 : 2) == 0,
              "Log probabilities: logits must be aligned to their elements.");
  const size_t need = tmc_logprobs_workspace_bytes(rows, vocabulary, top);
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "Log probabilities: workspace is smaller than tmc_logprobs_workspace_bytes() or not "
              "16-byte aligned.");
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
  p.count = (int)parts_of(rows, vocabulary);
  if (need) {
    p.arrivals = static_cast<int*>(workspace);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + logprob_counter_bytes(rows));
  }
  const dim3 grid((unsigned)(rows * p.count));
  const hipStream_t s = as_stream(stream);
#define TMC_LP(TYPE, EACH) \
  hipLaunchKernelGGL((logprobs_kernel<TYPE, EACH>), grid, dim3(kLpThreads), 0, s, p)
  const bool few = each_of(rows, vocabulary) == 8;
  if (dtype == TMC_F32) {
    if (few) TMC_LP(float, 8); else TMC_LP(float, 32);
  } else {
    if (few) TMC_LP(half_t, 8); else TMC_LP(half_t, 32);
  }
#undef TMC_LP
  return check_launch("logprobs_kernel");
}
