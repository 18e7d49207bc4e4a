// Log probabilities of given tokens, the entropy of every row and its most
// probable tokens, from logits [rows, vocabulary].
//
// With m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(t) = x[t] - m - log S,   entropy = log S - T / S.
// A logit of -inf adds nothing to S or T.  The alternatives come in the greedy
// order of tmc_argmax_f32 (the greater first, equals by the lower index, NaN
// never).
//
// Bound by reading the logits once.  A block holds a part of a row in
// registers at a time, so the maximum, the sums and the alternatives are three
// passes over registers, not over memory, while the next part is on its way.
// Each wave keeps the candidates for the alternatives that it meets, without
// waiting for the others; they are ranked together at the row's end.
// Where several blocks share a row, the last to arrive joins them in their
// order.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>

namespace tmc {
namespace {

constexpr int kTopMax = 64;
constexpr int kLpThreads = 256;
constexpr int kWaveKeys = 128;           // candidates a wave holds
static_assert(kTopMax + kWave <= kWaveKeys, "a wave's best and a round of new ones fit its list");
constexpr long long kNoKey = (long long)0x8000000000000000ull;

struct LogprobParams {
  const void* logits;
  const int32_t* tokens;  // may be null: no given tokens
  float* logprob;
  float* entropy;  // may be null
  int32_t* top_tokens;
  float* top_logprobs;
  // of shared rows: [rows][count] (S, T) in fp64, [rows][count][top] keys, [rows][count] m
  float* parts;
  int* arrivals;  // [rows], kCounterStride apart
  long stride;
  int rows, vocab, top;
  int count;      // blocks a row
  int walk;       // parts a block
};

// A logit and its index as one number, greater in the greedy order first: the
// float's bits in the order of its value (-0 as +0; no NaN), then the lower
// index.
__device__ __forceinline__ long long key_of(float v, int index) {
  const int b = __builtin_bit_cast(int, v + 0.0f);
  const int order = b ^ (b >> 31 & 0x7FFFFFFF);
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

// What a set of logits with maximum m and sums s, t (relative to m) adds to the
// sums relative to `high` >= m: nothing when it is empty (m = -inf), but for
// the NaNs that an empty maximum hides.
__device__ __forceinline__ void add_mass(float m, double s, double t, float high, double& sum_s,
                                         double& sum_t) {
  const float d = m == -INFINITY ? 0.0f : m - high;
  const double e = (double)fast_exp2(d * 1.44269504f);
  sum_s += e * s;
  sum_t += e == 0.0 ? 0.0 : e * (t + s * (double)d);
}

// The best `top` of `count` distinct keys (at most THREADS) to the places their rank
// gives them, the rest of the places empty.  Up to 64 keys: four threads a key.
// Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void rank_keys(const long long* keys, int count, int top,
                                          long long* out) {
  const bool few = count * 4 <= THREADS;
  const int me = few ? threadIdx.x >> 2 : threadIdx.x, step = few ? 4 : 1;
  if ((int)threadIdx.x < top) out[threadIdx.x] = kNoKey;
  __syncthreads();
  const long long mine = me < count ? keys[me] : kNoKey;
  int rank = 0, o = few ? threadIdx.x & 3 : 0;
  for (; o + 7 * step < count; o += 8 * step)
#pragma unroll
    for (int u = 0; u < 8; ++u) rank += keys[o + u * step] > mine ? 1 : 0;
  for (; o < count; o += step) rank += keys[o] > mine ? 1 : 0;
  if (few) {
    rank += __shfl_xor(rank, 1, kWave);
    rank += __shfl_xor(rank, 2, kWave);
  }
  if (mine != kNoKey && rank < top) out[rank] = mine;
  __syncthreads();
}

// The candidates of one wave, in LDS that only it touches: every key above
// `floor`, behind which at least `top` keys of the block's row are known to lie.
struct WaveKeys {
  long long* list;
  int held;
  float floor_v;
  long long floor;

  // A key a lane, where `in`; there is room for them.
  __device__ __forceinline__ void add(long long key, bool in) {
    const unsigned long long mask = __builtin_amdgcn_ballot_w64(in);
    const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32),
                                                 __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
    if (in) list[held + before] = key;
    held += __builtin_popcountll(mask);
  }
  // The best `top`, in order; the last of them is then the floor.
  __device__ __forceinline__ void keep_best(int top) {
    const int lane = threadIdx.x & (kWave - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const long long a = lane < held ? list[lane] : kNoKey;
    const long long b = lane + kWave < held ? list[lane + kWave] : kNoKey;
    int rank_a = 0, rank_b = 0;
    for (int o = 0; o < held; ++o) {
      const long long other = list[o];
      rank_a += other > a ? 1 : 0;
      rank_b += other > b ? 1 : 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (a != kNoKey && rank_a < top) list[rank_a] = a;
    if (b != kNoKey && rank_b < top) list[rank_b] = b;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    held = min(held, top);
    if (held == top) {
      floor = list[top - 1];
      floor_v = key_value(floor);
    }
  }
};

// EACH: elements a lane holds; a part is THREADS * EACH elements.  A block
// walks `walk` parts of its row, the next one's loads in flight.
template <typename T, int EACH, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(LogprobParams p) {
  constexpr int WAVES = THREADS / kWave;
  static_assert(WAVES * kTopMax <= THREADS, "the waves' best fit a ranking");
  constexpr int VEC = 16 / (int)sizeof(T);  // elements a load
  constexpr int LOADS = EACH / VEC;
  constexpr int PART = THREADS * EACH;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  // rows start anywhere on an element boundary
  typedef vec unaligned __attribute__((aligned(sizeof(T))));
  __shared__ __align__(16) long long s_lists[WAVES][kWaveKeys];
  __shared__ __align__(16) long long s_keys[THREADS];
  __shared__ __align__(16) long long s_best[kTopMax];
  __shared__ float s_m[WAVES], s_bound[WAVES];
  __shared__ double s_s[WAVES], s_t[WAVES];
  __shared__ int s_reach[WAVES], s_held[WAVES], s_found, s_last;
  const int split = blockIdx.x % p.count, row = blockIdx.x / p.count;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const T* x = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  const int begin = split * p.walk * PART, end = min(p.vocab, begin + p.walk * PART);
  const int top = p.top;
  // the wave's elements of a part: loads of 64 lanes x VEC, load after load
  const int own = wave * (kWave * EACH) + lane * VEC;
  auto fetch = [&](int part_at, vec (&in)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = part_at + own + i * kWave * VEC;
      if (at + VEC <= end) {
        in[i] = *reinterpret_cast<const unaligned*>(x + at);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) in[i][e] = at + e < end ? x[at + e] : (T)-INFINITY;
      }
    }
  };
  // the lane's own maximum and sums (relative to it)
  float m = -INFINITY, s = 0.0f, t = 0.0f;
  WaveKeys best{s_lists[wave], 0, -INFINITY, kNoKey};
  vec next[LOADS];
  fetch(begin, next);
  // the given token's logit comes beside the row's, not at the end
  const int token = p.tokens ? p.tokens[row] : -1;
  const bool known = token >= 0 && token < p.vocab;
  const float given = known ? (float)x[token] : 0.0f;
  for (int part_at = begin; part_at < end; part_at += PART) {
    float v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = (float)next[i / VEC][i % VEC];
    if (part_at + PART < end) fetch(part_at + PART, next);
    float mine = -INFINITY;  // (NaN left out)
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine = fmaxf(mine, v[i]);
    {
      // A lane of -inf adds nothing; its NaNs spoil the sums all the same.
      const float high = fmaxf(m, mine), shift = high == -INFINITY ? 0.0f : high;
      if (m != -INFINITY && m != high) {
        const float d = m - high, e = fast_exp2(d * 1.44269504f);
        t = e == 0.0f ? 0.0f : e * (t + s * d);
        s *= e;
      }
      m = high;
      float s4[4] = {s, 0.0f, 0.0f, 0.0f}, t4[4] = {t, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const float d = v[i] - shift, e = fast_exp2(d * 1.44269504f);
        s4[i & 3] += e;
        // (finite: 0 times it is 0; a NaN is in e)
        t4[i & 3] = __fmaf_rn(e, fmaxf(d, -1e30f), t4[i & 3]);
      }
      s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      t = (t4[0] + t4[1]) + (t4[2] + t4[3]);
    }
    if (top == 0) continue;

    // ---- a bound that at least `top` of the first part's elements reach, from the
    // lanes' greatest: each wave finds what its share of them reaches
    if (part_at == begin) {
      // waves whose lanes all hold elements
      const int full = min(WAVES, (end - part_at + kWave * (EACH - VEC)) / (kWave * EACH));
      const int need = full > 0 ? (top + full - 1) / full : top;
      float rest = mine, most = -INFINITY;
      int reach = 0;
      while (reach < need) {
        const float now = wave_max(rest);
        most = now;
        if (now == -INFINITY) break;
        reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(rest == now));
        if (rest == now) rest = -INFINITY;
      }
      if (lane == 0) {
        s_bound[wave] = most;
        s_reach[wave] = reach;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        int total = 0;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) total += s_bound[u] >= s_bound[w] ? s_reach[u] : 0;
        if (total >= top) best.floor_v = fmaxf(best.floor_v, s_bound[w]);
      }
    }
    // ---- the elements that reach it: no other wave is waited for
    const int lanes = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine >= best.floor_v));
    if (lanes != 0) {
      auto place = [&](int i) { return part_at + own + i / VEC * kWave * VEC + i % VEC; };
      int more = lanes * EACH;  // at most
      if (best.held + more > kWaveKeys) {
        more = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= best.floor_v));
      }
      if (best.held + more <= kWaveKeys && best.floor == kNoKey && best.floor_v != -INFINITY) {
        // (what lies past the end is -inf)
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const bool in = v[i] >= best.floor_v;  // (a NaN never)
          if (__builtin_amdgcn_ballot_w64(in) != 0) best.add(key_of(v[i], place(i)), in);
        }
      } else {  // no bound, or many (equal logits, say): the best of them now and then
#pragma clang loop unroll(disable)
        for (int i = 0; i < EACH; ++i) {
          if (best.held > kWaveKeys - kWave) best.keep_best(top);
          const long long key = key_of(v[0], place(i));
          best.add(key, v[0] >= best.floor_v && place(i) < end && key > best.floor);
#pragma unroll
          for (int e = 0; e + 1 < EACH; ++e) v[e] = v[e + 1];
        }
      }
    }
  }
  if (top > 0) {
    // ---- the waves' candidates together
    if (lane == 0) s_held[wave] = best.held;
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += s_held[w];
    if (total > THREADS) {  // the same in every thread
      best.keep_best(top);      // (of fewer than that, nothing changes but their order)
      __syncthreads();
      if (lane == 0) s_held[wave] = best.held;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) total += s_held[w];
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w) before += w < wave ? s_held[w] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = lane; i < best.held; i += kWave) s_keys[before + i] = best.list[i];
    __syncthreads();
    rank_keys<THREADS>(s_keys, total, top, s_best);
  }
  {
    // the lanes of a row of 16 in 32 bits, rows and waves in 64
    const float high = wave_max(m);
    const float e = m == -INFINITY ? 1.0f : fast_exp2((m - high) * 1.44269504f);
    const float d = m == -INFINITY ? 0.0f : m - high;
    const float s16 = group_sum<16>(e * s);
    const float t16 = group_sum<16>(e == 0.0f ? 0.0f : e * (t + s * d));
    double sw = 0.0, tw = 0.0;
#pragma unroll
    for (int r = 0; r < kWave; r += 16) {
      sw += readlane(s16, r);
      tw += readlane(t16, r);
    }
    if (lane == 0) {
      s_m[wave] = high;
      s_s[wave] = sw;
      s_t[wave] = tw;
    }
  }
  __syncthreads();
  float row_m = s_m[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) row_m = fmaxf(row_m, s_m[w]);
  double row_s = 0.0, row_t = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) add_mass(s_m[w], s_s[w], s_t[w], row_m, row_s, row_t);

  // ---- the row's blocks together
  if (THREADS == kLpThreads && p.count > 1) {
    const size_t slots = (size_t)p.rows * p.count, slot = (size_t)row * p.count + split;
    double* sums = reinterpret_cast<double*>(p.parts);            // [slots][2]
    long long* keys = reinterpret_cast<long long*>(sums + 2 * slots);  // [slots][top]
    float* maxima = reinterpret_cast<float*>(keys + slots * top);
    // every word at agent scope, completed before the arrival is counted
    if (threadIdx.x == 0) {
      __hip_atomic_store(sums + 2 * slot, row_s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * slot + 1, row_t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(maxima + slot, row_m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((int)threadIdx.x < top)
      __hip_atomic_store(keys + slot * top + threadIdx.x, s_best[threadIdx.x], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      s_last = __hip_atomic_fetch_add(p.arrivals + row * kCounterStride, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == p.count - 1;
      s_found = 0;
    }
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0)
      __hip_atomic_store(p.arrivals + row * kCounterStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const size_t first = (size_t)row * p.count;
    // What the first round of each of the steps below needs, in flight at once.
    const size_t here = first + min(lane, p.count - 1);
    const float part_m = __hip_atomic_load(maxima + here, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double part_s = __hip_atomic_load(sums + 2 * here, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double part_t =
        __hip_atomic_load(sums + 2 * here + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int total = p.count * top;
    const long long* from = keys + first * top;
    constexpr int kAhead = 4;  // keys a thread loads at once
    long long key[kAhead];
    auto load_keys = [&](int i) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        key[u] = __hip_atomic_load(from + min(i + u * THREADS, total - 1), __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
    };
    if (top > 0) load_keys(threadIdx.x);
    // each wave by itself: the maximum, then the sums relative to it, lane by
    // lane over the parts and then over the lanes: the same order each time
    row_m = lane < p.count ? part_m : -INFINITY;
    for (int i = lane + kWave; i < p.count; i += kWave)
      row_m = fmaxf(row_m, __hip_atomic_load(maxima + first + i, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT));
    // A bound that at least `top` keys reach: where `deep` parts are needed to
    // give `top` keys with their best `each` ones, the deep-th greatest of the
    // parts' each-th keys.
    const int some = min(p.count, THREADS), each = (top + some - 1) / some;
    if (top > 0 && (int)threadIdx.x < some)
      s_keys[threadIdx.x] = __hip_atomic_load(keys + (first + threadIdx.x) * top + each - 1,
                                              __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    row_m = wave_max(row_m);
    row_s = row_t = 0.0;
    if (lane < p.count) add_mass(part_m, part_s, part_t, row_m, row_s, row_t);
    for (int i = lane + kWave; i < p.count; i += kWave)
      add_mass(__hip_atomic_load(maxima + first + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
               __hip_atomic_load(sums + 2 * (first + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
               __hip_atomic_load(sums + 2 * (first + i) + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
               row_m, row_s, row_t);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      row_s += __shfl_xor(row_s, off, kWave);
      row_t += __shfl_xor(row_t, off, kWave);
    }
    if (top > 0) {
      const int deep = (top + each - 1) / each;  // at most `some`
      if (threadIdx.x == 0) s_best[0] = kNoKey;
      __syncthreads();
      if ((int)threadIdx.x < some) {
        const long long mine = s_keys[threadIdx.x];
        int rank = 0;
        for (int o = 0; o < some; ++o) rank += s_keys[o] > mine ? 1 : 0;
        if (rank == deep - 1 && mine != kNoKey) s_best[0] = mine;  // keys are distinct
      }
      __syncthreads();
      const long long bound = s_best[0];
      __syncthreads();
      for (int i = threadIdx.x; i < total; i += kAhead * THREADS) {
        if (i != (int)threadIdx.x) load_keys(i);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i + u * THREADS < total && key[u] != kNoKey && key[u] >= bound) {
            const int place = atomicAdd(&s_found, 1);
            if (place < THREADS) s_keys[place] = key[u];
          }
      }
      __syncthreads();
      if (s_found <= THREADS) {
        rank_keys<THREADS>(s_keys, s_found, top, s_best);
      } else {
        // the best so far and the next keys, as many as fit
        constexpr int kNext = THREADS > kTopMax ? THREADS - kTopMax : 1;
        if ((int)threadIdx.x < top) s_best[threadIdx.x] = kNoKey;
        __syncthreads();
        for (int at = 0; at < total; at += kNext) {
          const int n = min(kNext, total - at), i = threadIdx.x;
          if (i < top) s_keys[i] = s_best[i];
          if (i < n)
            s_keys[top + i] =
                __hip_atomic_load(from + at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __syncthreads();
          rank_keys<THREADS>(s_keys, top + n, top, s_best);
        }
      }
    }
  }

  // ---- the row
  // -inf alone: 0 / 0, a NaN as the other rows without a distribution
  const float log_s = row_m == -INFINITY ? __builtin_nanf("") : logf((float)row_s);
  if (threadIdx.x == 0) {
    if (p.entropy) p.entropy[row] = log_s - (float)row_t / (float)row_s;
    if (known) p.logprob[row] = given - row_m - log_s;
  }
  if ((int)threadIdx.x < top) {
    const long long key = s_best[threadIdx.x];
    const size_t to = (size_t)row * top + threadIdx.x;
    p.top_tokens[to] = key == kNoKey ? -1 : key_index(key);
    p.top_logprobs[to] = key == kNoKey ? -INFINITY : key_value(key) - row_m - log_s;
  }
}

// How a row is shared out: threads a block, elements a lane holds, parts a block,
// blocks a row.  Short rows take a wave each, which waits for no other: 3578 rows,
// 10 alternatives, of 130 21.4 us in blocks of four waves, 9.1 in one, of 1000 21.8 and
// 10.3, of 2000 20.8 and 14.9, of 4000 21.5 and 20.4; 600 rows of 1000 8.0 and 6.1, of
// 4000 7.4 and 12.8; 300 rows of 1000 5.9 and 6.0, of 2000 5.8 and 7.9; 1000 of 2000 8.3
// and 8.2, of 3000 8.4 and 11.0.  (From 1000 to 2047 rows of 1025 to 2048 the rule takes
// blocks where waves are as fast or faster: 1500 of 2000 10.2 and 8.9, 2047 of 1500 13.8
// and 8.9.)
// Rows in the hundreds take a block each; fewer are cut until there are kFill
// blocks or parts run out, the fewest rows into small parts.  MI355X, fp32:
// 2048 rows of 32003, 5 alternatives 55 us with 16 elements a lane, 60 with 8;
// without alternatives 48 to 51 (5.1 to 5.5 TB/s; a large copy moves 5.2); in fp16, half
// the bytes, 46 and 40.  16 rows of 32000,
// 20 alternatives 9.6 us from 16 blocks a row; 64 rows 12.3 us from 8 blocks a
// row, 12.7 from 4, 17.4 from 2; 200 rows 18.4 from 3, 27.9 from one.  Twice the
// blocks where each would walk more than 4 parts: 186 rows of 121000 36 us in 3
// blocks a row, 30 in 6 (400 rows of 32000 in 2 and 3 blocks 18.7 and 19.4).  Many rows
// are bound by the vector ALUs and the memory alike, few by the latency of the
// steps: logits, bound, ranks, arrival, join.
constexpr int64_t kFill = 512, kNarrow = 1024;
static_assert(kFill <= kSharedRows, "every shared row has its counter");
struct LogprobPlan {
  int threads, each, walk, count;
};
LogprobPlan logprob_plan(int64_t rows, int64_t vocabulary) {
  LogprobPlan plan{kLpThreads, 16, 1, 1};
  if (vocabulary <= (rows < 2048 ? kNarrow : 2 * kNarrow)) {
    plan.threads = kWave;
    plan.walk = (int)((vocabulary + 16 * kWave - 1) / (16 * kWave));
    return plan;
  }
  if (rows * ((vocabulary + 16 * kLpThreads - 1) / (16 * kLpThreads)) < kFill) plan.each = 8;
  const int64_t span = (int64_t)kLpThreads * plan.each, parts = (vocabulary + span - 1) / span;
  int64_t blocks = std::min(parts, std::max<int64_t>(1, (kFill + rows - 1) / rows));
  if (rows < kFill && parts > 4 * blocks) blocks *= 2;
  plan.walk = (int)((parts + blocks - 1) / blocks);
  plan.count = (int)((parts + plan.walk - 1) / plan.walk);
  return plan;
}
bool logprob_shape(int64_t rows, int64_t vocabulary, int64_t top) {
  return rows > 0 && rows < (1LL << 24) && vocabulary > 0 && vocabulary < (1LL << 28) && top >= 0 &&
         top <= kTopMax && top <= vocabulary;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" size_t tmc_logprobs_workspace_bytes(int64_t rows, int64_t vocabulary, int64_t top) {
  if (!logprob_shape(rows, vocabulary, top)) return 0;
  const int64_t parts = logprob_plan(rows, vocabulary).count;
  return parts == 1 ? 0 : kCounterBytes + (size_t)(rows * parts) * (20 + 8 * top);
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
  const LogprobPlan plan = logprob_plan(rows, vocabulary);
  p.walk = plan.walk;
  p.count = plan.count;
  if (need) {
    p.arrivals = static_cast<int*>(workspace);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  }
  const dim3 grid((unsigned)(rows * p.count));
  const hipStream_t s = as_stream(stream);
#define TMC_LP(TYPE, EACH, THREADS) \
  hipLaunchKernelGGL((logprobs_kernel<TYPE, EACH, THREADS>), grid, dim3(THREADS), 0, s, p)
#define TMC_LP_PLAN(TYPE)                                \
  if (plan.threads == kWave) TMC_LP(TYPE, 16, kWave);    \
  else if (plan.each == 8) TMC_LP(TYPE, 8, kLpThreads);  \
  else TMC_LP(TYPE, 16, kLpThreads)
  if (dtype == TMC_F32) {
    TMC_LP_PLAN(float);
  } else {
    TMC_LP_PLAN(half_t);
  }
#undef TMC_LP_PLAN
#undef TMC_LP
  return check_launch("logprobs_kernel");
}
