// Attention with a sliding window and sinks over a paged cache, gfx950.
//
// Query token at position p = valid - 1 sees the positions i <= p that lie in
// its window (i > p - window) or among the first `sinks` ones:
//   out = sum_i w_i v_i / sum_i w_i,  w_i = exp(q . k_i / sqrt(D) - max).
// The visible positions are [0, min(sinks, begin)) and [begin, valid) with
// begin = max(0, valid - window): pages between the two parts are never
// looked up, so a server may have given them back.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tmc {
namespace {

struct WindowParams {
  const half_t* q;       // [rows][q_heads][D]
  const half_t* k;       // pools [pages][kv_heads][page_size][D] at the strides
  const half_t* v;
  half_t* out;
  const int32_t* valid;      // [rows]
  const int32_t* tables;     // [table_rows][max_pages]
  const int32_t* row_table;  // table row of each row; null: its own (decode) or row 0 (one table)
  const int32_t* active;     // may be null: all rows
  long page_stride, head_stride;
  int pool_pages, rows, table_rows, q_heads, kv_heads, group, dim;
  int page_size, max_pages;
  unsigned page_magic;   // pos / page_size = (pos * magic >> 32) >> shift for pos < 2^31;
  int page_shift;        // magic 0: page_size 1
  int window, sinks;
  int own_table;         // row r reads table row r
  long out_pass;         // > 0: packed activation order, elements per 16-row pass
  float scale_log2;      // log2(e) / sqrt(D)
};

__device__ __forceinline__ int window_page(const WindowParams& p, int pos) {
  const int q = (int)(__umulhi((unsigned)pos, p.page_magic) >> p.page_shift);
  return p.page_magic ? q : pos;
}
__device__ __forceinline__ bool window_page_ok(const WindowParams& p, int page) {
  return page >= 0 && page < p.pool_pages;
}
__device__ __forceinline__ int window_begin(const WindowParams& p, int valid) {
  return max(0, valid - p.window);
}
// Table row of a query row, -1 when it has none.
__device__ __forceinline__ int window_table(const WindowParams& p, int row) {
  const int t = p.row_table ? p.row_table[row] : p.own_table ? row : 0;
  return t >= 0 && t < p.table_rows ? t : -1;
}
// Element of out for a row and a column (query head * D + d), see
// TMC_LAYOUT_Y_PACKED.
__device__ __forceinline__ size_t window_out(const WindowParams& p, int row, int col) {
  if (p.out_pass <= 0) return (size_t)row * p.q_heads * p.dim + col;
  return (size_t)(row >> 4) * p.out_pass +
         ((size_t)(col >> 5) * 64 + (row & 15) + 16 * ((col & 31) >> 3)) * 8 + (col & 7);
}

// ------------------------------------------------------------ any geometry
// One wave per (row, query head): 64 visible positions at a time, one per
// lane for the scores (whole K rows in 16-byte chunks), then lanes over the
// dims for P V.  Online softmax in fp32.  For the head dims that the matrix
// core kernels do not take, pools of 64 GiB, and chunks past the token form of
// more than 64 query heads a kv head; at 128 dims it takes 45 us where they
// take 7 (one request of 300 positions, 32 heads) and 8.3 ms where they take
// 91 us (2048 tokens, window 2048).  512 tokens over 1024 positions, 8 kv heads: 23 us
// at 128 dims, 0.85 ms at 96, 1.9 at 256; 71 query heads of 64 dims on one kv head
// 1.6 ms.  Bound by the latency of its loads: with a branch before each of them it
// took 2 to 5 times as long.
constexpr int kPlainMaxDim = 256;

struct PlainScratch {  // of one wave
  __align__(16) half_t q[kPlainMaxDim];
  float weight[kWave];
  long at[kWave];
};

// One (row, query head), whose length and table row are valid.  DIM: the head dim
// where it is known, else 0.  Loads have no branch between them: columns past the
// head dim and places without a row read the last column and the pool's first
// row, whatever they hold, and are not used.
template <int DIM>
__device__ __forceinline__ void plain_row_inline(const WindowParams& p, int row, int head,
                                                 PlainScratch& scratch) {
  constexpr int TILES = (DIM ? DIM : kPlainMaxDim) / kWave;
  constexpr int kAhead = 8;  // chunks of K, rows of V loaded at once
  const int lane = threadIdx.x & (kWave - 1);
  const int valid = p.valid[row];
  const int32_t* table = p.tables + (size_t)window_table(p, row) * p.max_pages;
  const int kvh = head / p.group, d = DIM ? DIM : p.dim;
  const half_t* q = p.q + ((size_t)row * p.q_heads + head) * d;
  for (int i = lane; i < d; i += kWave) scratch.q[i] = q[i];
  const int begin = window_begin(p, valid), first = min(p.sinks, begin);
  const int count = first + valid - begin;
  float m = -INFINITY, sum = 0.0f, o[TILES] = {};
  int column[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) column[t] = min(lane + t * kWave, d - 1);
  bool bad = false;
  for (int u0 = 0; u0 < count; u0 += kWave) {
    const int u = u0 + lane, pos = u < first ? u : begin + u - first;
    float score = -INFINITY;
    long at = -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (u < count) {
      const int slot = window_page(p, pos), page = table[slot];
      if (window_page_ok(p, page)) {
        at = (long)page * p.page_stride + (long)kvh * p.head_stride +
             (long)(pos - slot * p.page_size) * d;
        float dot = 0.0f;
#pragma unroll kAhead
        for (int c = 0; c < d; c += 8)
          dot = dot8(load_h8(scratch.q + c), load_h8(p.k + at + c), dot);
        score = dot * p.scale_log2;
      } else {
        bad = true;
      }
    }
    const float next = fmaxf(m, cross_max<1>(score));
    const float alpha = next == -INFINITY ? 1.0f : fast_exp2(m - next);
    const float w = score == -INFINITY ? 0.0f : fast_exp2(score - next);
    m = next;
    sum = sum * alpha + w;
    scratch.weight[lane] = w;
    scratch.at[lane] = at;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] *= alpha;
    const int live = min(kWave, count - u0);
    for (int i = 0; i < live; i += kAhead) {
      half_t v[kAhead][TILES];
      bool here[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const long from = scratch.at[i + a];
        here[a] = from >= 0;
#pragma unroll
        for (int t = 0; t < TILES; ++t) v[a][t] = p.v[max(from, 0L) + column[t]];
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const float wa = scratch.weight[i + a];
#pragma unroll
        for (int t = 0; t < TILES; ++t) o[t] += here[a] ? wa * (float)v[a][t] : 0.0f;
      }
    }
  }
  if (__any(bad)) return;
  sum = cross_sum<1>(sum);
#pragma unroll
  for (int t = 0; t < TILES; ++t)
    if (lane + t * kWave < d)
      p.out[window_out(p, row, head * d + lane + t * kWave)] = (half_t)(o[t] / sum);
}
template <int DIM>
__device__ __noinline__ void plain_row(WindowParams p, int row, int head, PlainScratch& scratch) {
  plain_row_inline<DIM>(p, row, head, scratch);
}

__global__ __launch_bounds__(kWave) void window_plain_kernel(WindowParams p) {
  __shared__ PlainScratch scratch;
  const int row = blockIdx.x, head = blockIdx.y;
  if (row >= (p.active ? min(p.active[0], p.rows) : p.rows)) return;
  const int valid = p.valid[row];
  if (valid < 1 || valid > p.page_size * p.max_pages || window_table(p, row) < 0) return;
  plain_row_inline<0>(p, row, head, scratch);
}

// ------------------------------------------------------------ one token a request
// D = 64 and 128.  A step is 32 (D = 64) or 16 visible positions of one
// (request, kv head) row; kv heads of more than 16 query heads make a row for
// every 16 or fewer of them.  A row is a block's, or, where rows are few, shared
// by up to `parts` blocks in even shares of about kDecodeLeast steps or more; each
// writes a partial (max, sum, weighted) to the workspace and the last one to
// arrive joins them, in block order.
//
// Inside a block its 8, 4 or 1 waves take the steps of a share in turn.  Each wave has a
// ring of STAGES steps in LDS that only it touches, filled by 16-byte loads
// straight to LDS: no barrier, no register holds a load in flight, and a
// stage is reloaded as soon as its operands are in registers.  K and V rows lie
// in LDS as in their pages, 16-byte chunks (K) and 32-byte units (V) swizzled
// by the row so that the operand reads spread over the banks.  A position that
// does not exist reads a zero row.  Scores S^T = K Q^T (16 positions x 16
// heads) leave lane (head j, group g) with positions 4g .. 4g+3, the order in
// which O^T = V^T P^T wants its weights; V^T comes from transposing LDS reads.
//
// Bound by reading K and V: 64 requests, 8 kv heads of 128 dims, window 2048, 516
// MB: 90 us, 5.7 TB/s (a large copy moves 5.2).  Two blocks of 64 KiB rings a CU
// rather than one of 128 KiB with steps twice as long (103 us).  Few rows are bound by latency: lengths,
// pages, K and V, and at the join stores, arrival and loads, 3 to 4 us of it.
constexpr int kDecodeCus = 256;  // of an MI355X
constexpr int kDecodeLeast = 8, kDecodeAlone = 20;
static_assert(kDecodeCus <= kSharedRows, "every shared row has its counter");

// Blocks that share a row of `steps`, of at most `parts`.
__host__ __device__ inline int decode_shares(int64_t steps, int64_t parts) {
  const int64_t shares = steps <= kDecodeAlone ? (steps > 0) : (steps + kDecodeLeast - 1) / kDecodeLeast;
  return (int)(shares < parts ? shares : parts);
}
struct DecodePlan {
  float* slots;   // [rows][kv_heads][splits][parts][heads][D + 2]
  int* arrivals;  // [rows][kv_heads][splits], kCounterStride apart
  int parts, splits, heads;
};

static __device__ __align__(16) unsigned s_zero_row[4];  // what absent positions read

// A matrix product's result may be read by vector instructions only some wait
// states later.  The compiler puts them in within a block of code, but hipcc
// 7.2 left them out where a branch follows the product: the scores' maximum
// was then taken of old registers.
template <typename T> __device__ __forceinline__ void settle(T& result) {
  asm volatile("s_nop 15" : "+v"(result));
}

template <int N> __device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Maximum over lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ float max_of_groups(float v) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const unsigned a0 = a[0], a1 = a[1];
  v = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const unsigned y = __builtin_bit_cast(unsigned, v);
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// The operands of one step out of LDS, waits included: the compiler would let
// such reads wait for every load to LDS in flight.
template <int D, int STEP, int OFFSET, int PAGE_OFFSET>
__device__ __forceinline__ void read_keys(const unsigned (&at)[D / 32], unsigned page_at,
                                          h8 (&k)[STEP / 16][D / 32], int& page) {
  static_assert((D == 128 && STEP == 16) || (D == 64 && STEP == 32), "four operands a step");
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b32 %4, %9 offset:%11\n\t"
        "ds_read_b128 %0, %5 offset:%10\n\tds_read_b128 %1, %6 offset:%10\n\t"
        "ds_read_b128 %2, %7 offset:%10\n\tds_read_b128 %3, %8 offset:%10\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(page)
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(page_at), "n"(OFFSET),
          "n"(PAGE_OFFSET)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b32 %4, %7 offset:%10\n\t"
        "ds_read_b128 %0, %5 offset:%8\n\tds_read_b128 %1, %6 offset:%8\n\t"
        "ds_read_b128 %2, %5 offset:%9\n\tds_read_b128 %3, %6 offset:%9\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(page)
        : "v"(at[0]), "v"(at[1]), "v"(page_at), "n"(OFFSET), "n"(OFFSET + 32 * D),
          "n"(PAGE_OFFSET)
        : "memory");
  }
}

// V^T, lane (j, g): dims 16 t + j, positions 4g .. 4g+3 of the step's first 16
// (v[0]) and, D = 64, of its last 16 (v[1]).
template <int D, int STEP, int OFFSET>
__device__ __forceinline__ void read_values(const unsigned (&at)[D / 16], h4 (&v)[STEP / 16][D / 16]) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
        "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
        "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
        "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[0][4]),
          "=&v"(v[0][5]), "=&v"(v[0][6]), "=&v"(v[0][7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
          "v"(at[7]), "n"(OFFSET)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %10 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]),
          "=&v"(v[1][1]), "=&v"(v[1][2]), "=&v"(v[1][3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(OFFSET), "n"(OFFSET + 32 * D)
        : "memory");
  }
}

// Weights are stored 2^kRaiseLog times their value in fp16 (the greatest is
// 2^kRaiseLog itself): weights down to 2^-29 of the greatest keep their 11
// bits, and the sum takes the rounded ones, so the factor cancels.  fp16 is
// what the matrix cores multiply with V's type; what the rounding left as a
// second operand (22 bits) would double the products of P V.  An output is off
// by up to 2^-11 of the mean of |v| for it, beside the 2^-11 of its own fp16: the
// error against 64 bits is 1.2 to 1.4 times that of fp32 weights (2.5e-4 to
// 2.9e-4 of the outputs' norm, 2.1e-4 of which is their fp16).
constexpr float kRaiseLog = 15.0f;
constexpr unsigned kNoUnit = 0xFFFFFFFFu;

// Two floats that other blocks read, and two of theirs: at agent scope.
__device__ __forceinline__ void store_pair(float* to, float a, float b) {
  const float2 v = {a, b};
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(to),
                     __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_pair(const float* from) {
  return __builtin_bit_cast(
      float2, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(from),
                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
// Two dims of an output; whether one of them is a NaN.
__device__ __forceinline__ bool put_pair(const WindowParams& p, int row, int col, float a, float b) {
  *reinterpret_cast<h2*>(p.out + window_out(p, row, col)) = h2{(half_t)a, (half_t)b};
  return !(a == a) | !(b == b);
}

// A greatest score that is infinite, as where all are NaN or -inf, leaves no
// result but NaN, with weights of any type.
__device__ __forceinline__ bool finite(float top) { return fabsf(top) < INFINITY; }

// Visible positions of a row of length `valid`, in steps.
template <int STEP>
__device__ __forceinline__ int steps_of(const WindowParams& p, int valid, bool active) {
  if (!active || valid < 1 || valid > p.page_size * p.max_pages) return 0;
  const int begin = window_begin(p, valid);
  return (min(p.sinks, begin) + valid - begin + STEP - 1) / STEP;
}

template <int D, int STEP, int STAGES, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void window_decode_kernel(WindowParams p,
                                                                         DecodePlan plan) {
  constexpr int KS = D / 32, DT = D / 16, CH = D / 8, TILES = STEP / 16;
  constexpr int RPL = kWave / CH, LOADS = STEP / RPL;  // rows a load, loads of K (of V) a step
  constexpr int STAGE = 2 * STEP * D;                  // halves
  constexpr int THREADS = WAVES * kWave;
  __shared__ __align__(16) half_t s_ring[WAVES * STAGES * STAGE];
  __shared__ int s_pages[WAVES * STAGES * kWave];
  __shared__ int s_last;
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) const void global_void;
  static_assert(sizeof(s_ring) >= WAVES * 16 * (D + 2) * sizeof(float),
                "the waves' results fit the ring");

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int j = lane & 15, g = lane >> 4;
  const int active = p.active ? min(p.active[0], p.rows) : p.rows;

  // ---- this block's steps [first_step, last_step) of its row
  const int unit = blockIdx.x / plan.parts, part = blockIdx.x - unit * plan.parts;
  const int pair = unit / plan.splits, split = unit - pair * plan.splits;
  const int row = pair / p.kv_heads, kvh = pair - row * p.kv_heads;
  const int first_head = kvh * p.group + split * plan.heads;
  const int heads = min(plan.heads, p.group - split * plan.heads);
  const int valid = p.valid[row];
  const int table_row = window_table(p, row);
  const int steps = steps_of<STEP>(p, valid, row < active && table_row >= 0);
  const int shares = decode_shares(steps, plan.parts);
  if (part >= shares) return;
  const int even = steps / shares, over = steps - even * shares;
  const int first_step = part * even + min(part, over);
  const int last_step = first_step + even + (part < over);

  // ---- LDS places: loads are linear (lane l: row l / CH, slot l % CH)
  half_t* ring = s_ring + wave * STAGES * STAGE;
  unsigned key_at[KS], value_at[DT];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    key_at[s] = lds_address(ring) +
                (unsigned)(j * D * 2 + (((4 * s + g) ^ (D == 128 ? j : (j >> 1) & 7)) << 4));
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int R = 4 * g + (j >> 2), unit = t ^ (D == 128 ? R & 7 : (R >> 1) & 3);
    value_at[t] = lds_address(ring) + (unsigned)(STEP * D * 2 + R * D * 2 + (unit << 5) + ((j & 3) << 3));
  }
  int* pages = s_pages + wave * STAGES * kWave;
  const unsigned page_at = lds_address(pages + lane);
  const char* zero = reinterpret_cast<const char*>(s_zero_row);

  const int begin = window_begin(p, valid), sinks = min(p.sinks, begin);
  const int count = sinks + valid - begin;
  const int32_t* table = p.tables + (size_t)table_row * p.max_pages;
  const unsigned head_unit = (unsigned)((size_t)kvh * p.head_stride / 8);
  h8 qb[KS];
  {
    const half_t* q = p.q + ((size_t)row * p.q_heads + first_head + min(j, heads - 1)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = load_h8(q + 32 * s + 8 * g);
  }
  f4 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, lsum = 0.0f;
  int bad = 0;

  // Table slot of the position that lane (l & 31) stands for in a step (past
  // the end: of the last one) and its row in that page.
  auto locate = [&](int step, int& slot_row) -> const int32_t* {
    const int u = min(step * STEP + (lane & (STEP - 1)), count - 1);
    const int pos = u < sinks ? u : begin + u - sinks;
    const int slot = window_page(p, pos);
    slot_row = pos - slot * p.page_size;
    return table + slot;
  };
  // 16-byte unit where that position's row starts, kNoUnit when it has none
  auto place = [&](int step, int page, int slot_row) -> unsigned {
    const bool ok = window_page_ok(p, page);
    bad |= !ok;
    return ok && step * STEP + (lane & (STEP - 1)) < count
               ? (unsigned)page * (unsigned)(p.page_stride / 8) + head_unit +
                     (unsigned)(slot_row * CH)
               : kNoUnit;
  };
  // K and V rows of a step, and the pages of the step that follows it in the
  // stage: those too by loads to LDS, so that no load the compiler could wait
  // for mixes with the ones in flight.
  auto issue = [&](unsigned unit, const int32_t* next, int stage) {
    half_t* to = ring + stage * STAGE;
    __builtin_amdgcn_global_load_lds((global_void*)next, (lds_void*)(pages + stage * kWave), 4, 0, 0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int R = RPL * i + lane / CH, slot = lane % CH;
      const unsigned row_unit = (unsigned)__shfl((int)unit, R, kWave);
      const unsigned kc = slot ^ (D == 128 ? R & 15 : (R >> 1) & 7);
      const unsigned vc = (((slot >> 1) ^ (D == 128 ? R & 7 : (R >> 1) & 3)) << 1) | (slot & 1);
      const bool here = row_unit != kNoUnit;
      const char* ka = here ? reinterpret_cast<const char*>(p.k) + (size_t)(row_unit + kc) * 16 : zero;
      const char* va = here ? reinterpret_cast<const char*>(p.v) + (size_t)(row_unit + vc) * 16 : zero;
      __builtin_amdgcn_global_load_lds((global_void*)ka, (lds_void*)(to + RPL * i * D), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_void*)va, (lds_void*)(to + (STEP + RPL * i) * D),
                                       16, 0, 0);
    }
  };
  auto consume = [&](int step, const h8 (&k)[TILES][KS], const h4 (&v)[TILES][DT]) {
    f4 sc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      sc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s)
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][s], qb[s], sc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) settle(sc[t]);
    const int left = count - step * STEP;  // positions of the step that exist
    if (left < STEP)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * t + 4 * g + r >= left) sc[t][r] = -INFINITY;
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
    if constexpr (TILES == 2)
      top = fmaxf(top, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    top = max_of_groups(top) * p.scale_log2;
    if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
      const float next = fmaxf(m, top);
      const float alpha = next == m ? 1.0f : fast_exp2(m - next);
      m = next;
      lsum *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] *= alpha;
    }
    const float shift = m == -INFINITY ? 0.0f : m - kRaiseLog;
    h4 w[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        w[t][r] = (half_t)fast_exp2(__fmaf_rn(sc[t][r], p.scale_log2, -shift));
      const h2 ones = {(half_t)1.0f, (half_t)1.0f};
      lsum = __builtin_amdgcn_fdot2(__builtin_shufflevector(w[t], w[t], 0, 1), ones, lsum, false);
      lsum = __builtin_amdgcn_fdot2(__builtin_shufflevector(w[t], w[t], 2, 3), ones, lsum, false);
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      if constexpr (TILES == 2)
        o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            __builtin_shufflevector(v[0][t], v[1][t], 0, 1, 2, 3, 4, 5, 6, 7),
            __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7), o[t], 0, 0, 0);
      else
        o[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(v[0][t], w[0], o[t], 0, 0, 0);
    }
  };

  // ---- the wave's steps: every WAVES-th of the part
  const int mine = first_step + wave;
  int slot_row[STAGES];  // of the step that a stage takes next
  {
    int first_page[STAGES], first_row[STAGES];
#pragma unroll
    for (int st = 0; st < STAGES; ++st)
      first_page[st] = *locate(mine + st * WAVES, first_row[st]);
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
      const int32_t* next = locate(mine + (STAGES + st) * WAVES, slot_row[st]);
      if (mine + st * WAVES < last_step)
        issue(place(mine + st * WAVES, first_page[st], first_row[st]), next, st);
    }
  }
  // One step out of its stage, and the stage loaded again.  BODY: every step
  // that is waited for or loaded exists.
  auto turn = [&](auto stage, auto body, int step) {
    constexpr int ST = decltype(stage)::value;
    constexpr bool BODY = decltype(body)::value;
    const int again = step + STAGES * WAVES;
    if (BODY || step + (STAGES - 1) * WAVES < last_step)
      wait_loads<(2 * LOADS + 1) * (STAGES - 1)>();
    else
      wait_loads<0>();
    h8 k[TILES][KS];
    h4 v[TILES][DT];
    int page;
    read_keys<D, STEP, ST * STAGE * 2, ST * kWave * 4>(key_at, page_at, k, page);
    read_values<D, STEP, ST * STAGE * 2>(value_at, v);
    if (BODY || again < last_step) {
      const unsigned unit = place(again, page, slot_row[ST]);
      issue(unit, locate(again + STAGES * WAVES, slot_row[ST]), ST);
    }
    consume(step, k, v);
  };
  auto round = [&](auto body, int step) {
    constexpr bool BODY = decltype(body)::value;
    turn(std::integral_constant<int, 0>{}, body, step);
    if constexpr (STAGES > 1)
      if (BODY || step + WAVES < last_step)
        turn(std::integral_constant<int, 1>{}, body, step + WAVES);
    if constexpr (STAGES > 2)
      if (BODY || step + 2 * WAVES < last_step)
        turn(std::integral_constant<int, 2>{}, body, step + 2 * WAVES);
    if constexpr (STAGES > 3)
      if (BODY || step + 3 * WAVES < last_step)
        turn(std::integral_constant<int, 3>{}, body, step + 3 * WAVES);
  };
  int step = mine;
  for (; step + (2 * STAGES - 1) * WAVES < last_step; step += STAGES * WAVES)
    round(std::true_type{}, step);
  for (; step < last_step; step += STAGES * WAVES) round(std::false_type{}, step);

  // ---- the waves meet in LDS (the ring: every load into it has landed)
  lsum = cross_sum<16>(lsum);
  bad = __syncthreads_or(bad);
  float* s_max = reinterpret_cast<float*>(s_ring);  // [waves][16]
  float* s_sum = s_max + WAVES * 16;
  float* s_out = s_sum + WAVES * 16;         // [waves][heads][D]
  if (j < heads) {
    if (g == 0) {
      s_max[wave * 16 + j] = m;
      s_sum[wave * 16 + j] = lsum;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<f4*>(s_out + (size_t)(wave * heads + j) * D + 16 * t + 4 * g) = o[t];
  }
  __syncthreads();
  const bool whole = shares == 1;
  const size_t slot_floats = (size_t)plan.heads * (D + 2);
  float* slots = plan.slots + (size_t)unit * plan.parts * slot_floats;
  // two dims a thread
  unsigned again = 0;  // heads with a NaN among the dims that this thread put
  for (int i = threadIdx.x; i < heads * (D / 2); i += THREADS) {
    const int head = i / (D / 2), d = i % (D / 2) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_max[w * 16 + head]);
    float sum = 0.0f, val0 = 0.0f, val1 = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float high = s_max[w * 16 + head];
      const float scale = high == -INFINITY ? 0.0f : fast_exp2(high - top);
      sum += scale * s_sum[w * 16 + head];
      const float2 part = *reinterpret_cast<const float2*>(
          s_out + (size_t)(w * heads + head) * D + d);
      val0 += scale * part.x;
      val1 += scale * part.y;
    }
    if (whole) {
      if (!bad && put_pair(p, row, (first_head + head) * D + d, val0 / sum, val1 / sum) &&
          finite(top))
        again |= 1u << head;
    } else {
      float* out = slots + part * slot_floats + (size_t)head * (D + 2);
      store_pair(out + d, val0, val1);
      if (d == 0) store_pair(out + D, top, bad ? -1.0f : sum);
    }
  }
  if (!whole) {
    // the last of the row's blocks joins the partials, in block order (every
    // word is written and read at agent scope; the stores have completed
    // before the arrival is counted)
    int* counter = plan.arrivals + unit * kCounterStride;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               shares - 1;
    __syncthreads();
    if (s_last) {
      if (threadIdx.x == 0)
        __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      for (int i = threadIdx.x; i < heads * (D / 2); i += THREADS) {
        const int head = i / (D / 2), d = i % (D / 2) * 2;
        float top = -INFINITY, sum = 0.0f, val0 = 0.0f, val1 = 0.0f;
        bool spoiled = false;
        constexpr int kAhead = 16;  // partials loaded at once
        for (int b = 0; b < shares; b += kAhead) {
          float2 x[kAhead], y[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const float* in = slots + min(b + u, shares - 1) * slot_floats + (size_t)head * (D + 2);
            x[u] = load_pair(in + d);
            y[u] = load_pair(in + D);
          }
          float next = top;
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (b + u < shares) {
              spoiled |= y[u].y < 0.0f;
              next = fmaxf(next, y[u].x);
            }
          const float a = top == -INFINITY ? 0.0f : fast_exp2(top - next);
          sum *= a;
          val0 *= a;
          val1 *= a;
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (b + u < shares) {
              const float c = y[u].x == -INFINITY ? 0.0f : fast_exp2(y[u].x - next);
              sum += y[u].y * c;
              val0 += x[u].x * c;
              val1 += x[u].y * c;
            }
          top = next;
        }
        if (!spoiled && put_pair(p, row, (first_head + head) * D + d, val0 / sum, val1 / sum) &&
            finite(top))
          again |= 1u << head;
      }
    }
  }
  // A weight that fp16 rounds to 0 times an infinity of V, or one past its range
  // (scores of 2^24 and more, whose fp32 maximum is several powers of two off),
  // is a NaN that weights of fp32 do not give: such heads are done again with
  // those, by the wave that put them, in LDS behind what the waves met in.  (0.2 ms
  // for the heads of 2048 positions; nothing where none is.)
  unsigned long long waiting = __builtin_amdgcn_ballot_w64(again != 0);
  if (waiting) {
    unsigned todo = 0;
    for (; waiting; waiting &= waiting - 1)
      todo |= (unsigned)__shfl((int)again, __builtin_ctzll(waiting), kWave);
    constexpr int kMet = WAVES * 16 * (D + 2) * (int)sizeof(float);
    static_assert(kMet % 16 == 0 && kMet + sizeof(PlainScratch) * WAVES <= sizeof(s_ring),
                  "a scratch for every wave");
    PlainScratch& scratch =
        reinterpret_cast<PlainScratch*>(reinterpret_cast<char*>(s_ring) + kMet)[wave];
    __builtin_amdgcn_s_waitcnt(0);  // the NaNs are stored
    for (; todo; todo &= todo - 1)
      plain_row_inline<D>(p, row, first_head + __builtin_ctz(todo), scratch);
  }
}

// ------------------------------------------------------------ a chunk of rows
// D = 64 and 128.  One block of 8 waves per (kv head, tile of query vectors =
// tokens x query heads of that kv head).  A wave holds 32 vectors on
// v_mfma_f32_32x32x16_f16: S^T = K Q^T (32 positions x 32 vectors) leaves lane
// (vector, half) with the positions 8 (r / 4) + 4 half + r % 4, the order in
// which O^T = V^T P^T takes its weights.  Two waves a SIMD: one's softmax runs
// beside the other's products.
//
// PG = 1: the waves hold 8 x 32 vectors and all take the 64 positions of a
// stage.  PG = 2 (4): they hold 4 (2) x 32 vectors and take a half (quarter) of
// the 64 (128) positions of a stage each; the partials join at the end.  K and V go
// through registers, loaded one stage ahead of the LDS one; one barrier a
// stage.
//
// Bound by the products, the softmax and the LDS together: 2048 tokens, 32 heads
// of 128 dims, window 2048: 91 us, 760 TFLOP/s; matrix cores, vector ALUs and LDS
// are busy 37, 42 and 44% of the time, the products with loads alone take 78 us.
// Measured and no faster: 4 waves of 64 vectors with the products of one tile
// beside the softmax of the other (130), opposite phases or priorities for the
// two waves of a SIMD, loads placed among the products, K read a step ahead.
//
// A tile's positions are those that any of its tokens sees, sinks first.
// Positions that a vector does not see are masked in the steps where that can
// be; steps that none of a wave's vectors sees are left out.  Rows of several
// requests in a tile are done run by run: 256 rows over 1024 positions, 8 kv heads,
// 22 us as one request, 25 as 16, 339 as 256 (186 as a decode batch).
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kChunkWaves = 8;

// A new maximum moves the weights' scale only when it is kLag above the one in
// use, so a wave seldom rescales its sums; weights are then at most
// 2^(kChunkRaise + kLag) in fp16 and keep 11 bits down to 2^-24 of that scale (fp16
// for the reason that kRaiseLog states).
constexpr float kLag = 5.0f, kChunkRaise = 10.0f;

__device__ __forceinline__ unsigned opaque(unsigned v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The least of lanes 0 ... 31 (32 ... 63 hold the same), in all lanes.
__device__ __forceinline__ int least_of_half(int v) {
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x121, 0xF, 0xF, false));  // row_ror 1, 2, 4, 8
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x122, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x124, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x128, 0xF, 0xF, false));
  return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}

template <int D, int PG>
__global__ __launch_bounds__(kChunkWaves * kWave, 2) void window_chunk_kernel(WindowParams p,
                                                                              int tiles,
                                                                              int tokens_per_tile) {
  constexpr int KS = D / 16, DT = D / 32, CH = D / 8;
  constexpr int WAVES = kChunkWaves, THREADS = WAVES * kWave, VG = WAVES / PG;
  constexpr int SPAN = PG == 1 ? 64 : 32 * PG;        // positions a stage
  constexpr int OWN = SPAN / WAVES;                   // rows of a stage a wave loads
  constexpr int RPL = kWave / CH, LOADS = OWN / RPL;  // rows a load, loads of K (of V)
  constexpr int STAGE = 2 * SPAN * D;                 // halves: K rows, V rows
  static_assert(LOADS >= 1 && 2 * STAGE >= WAVES * 32 * D, "results fit the stages");
  constexpr int PER = SPAN / kWave, TURNS = WAVES / PER;  // waves that find a stage's rows
  __shared__ __align__(256) half_t s_kv[2 * STAGE];
  __shared__ unsigned s_units[4][SPAN];  // 16-byte units where the rows of four stages start
  __shared__ int s_run, s_low, s_high;
  __shared__ float s_max[WAVES][32], s_sum[WAVES][32];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int vg = wave % VG, pg = wave / VG;
  const int col = lane & 31, half = lane >> 5;
  // the tiles of one kv head stay on one XCD, whose L2 then holds its pages
  int kvh, tile;
  if (p.kv_heads % 8 == 0) {
    const int xcd = blockIdx.x % 8, r = blockIdx.x / 8;
    kvh = xcd + 8 * (r / tiles);
    tile = tiles - 1 - r % tiles;
  } else {
    kvh = blockIdx.x / tiles;
    tile = tiles - 1 - blockIdx.x % tiles;
  }
  const int active = p.active ? min(p.active[0], p.rows) : p.rows;
  const int t0 = tile * tokens_per_tile, tokens = min(tokens_per_tile, active - t0);
  const unsigned head_unit = (unsigned)((size_t)kvh * p.head_stride / 8);
  const int capacity = p.page_size * p.max_pages;
  // this lane's vector
  const int token = (32 * vg + col) / p.group, row = t0 + token;
  const int head = kvh * p.group + 32 * vg + col - token * p.group;
  const int any_row = min(row, p.rows - 1);  // one that exists
  const int row_len = p.valid[any_row];
  h8 qb[KS];
  {
    const half_t* q = p.q + ((size_t)any_row * p.q_heads + head) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = load_h8(q + 16 * s + 8 * half);
  }

  for (int run = 0; run < tokens;) {
    // ---- the run of tokens [run, run_end) of one request
    const int table_row = window_table(p, t0 + run);
    if (threadIdx.x == 0) {
      s_run = tokens;
      s_low = 0x7fffffff;
      s_high = 0;
    }
    __syncthreads();
    if (p.row_table) {
      int other = tokens;
      for (int t = run + 1 + (int)threadIdx.x; t < tokens; t += THREADS)
        if (window_table(p, t0 + t) != table_row) other = min(other, t);
      if (other < tokens) atomicMin(&s_run, other);
      __syncthreads();
    }
    const int run_end = s_run, run_at = run;
    run = run_end;
    int len = 0;
    if (table_row >= 0 && token >= run_at && token < run_end) {
      len = row_len < 1 || row_len > capacity ? 0 : row_len;
    }
    const int from = len > 0 ? window_begin(p, len) : 0x7fffffff;
    // the wave's extremes, then the tile's
    int min_len = len > 0 ? len : 0x7fffffff, max_len = len, min_from = from,
        max_from = len > 0 ? from : 0;
    min_len = least_of_half(min_len);
    max_len = -least_of_half(-max_len);
    min_from = least_of_half(min_from);
    max_from = -least_of_half(-max_from);
    if (lane == 0 && max_len > 0) {
      atomicMin(&s_low, min_from);
      atomicMax(&s_high, max_len);
    }
    __syncthreads();
    const int low = s_low, high = s_high;
    if (high == 0) {
      __syncthreads();
      continue;
    }
    const int32_t* table = p.tables + (size_t)table_row * p.max_pages;
    const int sinks = min(p.sinks, low), gap = low - sinks;
    const int count = high - gap;  // positions of the tile: u < sinks, then u + gap

    // ---- loads.  The waves take turns to find a stage's rows: their table entries
    // four stages ahead, their units three ahead.  Places past the end take the
    // last position's row and positions without a page page 0's: such scores are
    // masked, or their vectors not stored.
    int bad = 0, page = 0, slot_row = 0;
    auto my_turn = [&](int stage) { return stage % TURNS == wave / PER; };
    const int turn_row = wave % PER * kWave + lane;
    auto look_up = [&](int stage) {
      const int u = min(stage * SPAN + turn_row, count - 1);
      const int pos = u < sinks ? u : u + gap;
      const int at = window_page(p, pos);
      slot_row = pos - at * p.page_size;
      page = table[at];
    };
    auto put_units = [&](int stage) {
      const bool ok = window_page_ok(p, page);
      bad |= !ok;
      s_units[stage % 4][turn_row] = (unsigned)(ok ? page : 0) * (unsigned)(p.page_stride / 8) +
                                     head_unit + (unsigned)(slot_row * CH);
    };
    const int own_row = OWN * wave + lane / CH, slot = lane % CH;
    // 16-byte chunk of its row that a lane loads; RPL i changes other bits of the row
    const unsigned key_chunk = slot ^ (D == 128 ? own_row & 15 : (own_row >> 1) & 7);
    const unsigned value_chunk =
        (((slot >> 1) ^ (D == 128 ? own_row & 7 : (own_row >> 1) & 3)) << 1) | (slot & 1);
    h8 kr[LOADS], vr[LOADS];
    auto load = [&](int stage) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const unsigned unit = s_units[stage % 4][own_row + RPL * i];
        const unsigned kx = D == 128 ? RPL * i & 15 : (RPL * i >> 1) & 7;
        const unsigned vx = (D == 128 ? RPL * i & 7 : (RPL * i >> 1) & 3) << 1;
        kr[i] = *reinterpret_cast<const h8*>(reinterpret_cast<const char*>(p.k) +
                                             (size_t)(unit + (key_chunk ^ kx)) * 16);
        vr[i] = *reinterpret_cast<const h8*>(reinterpret_cast<const char*>(p.v) +
                                             (size_t)(unit + (value_chunk ^ vx)) * 16);
      }
    };
    auto store = [&](half_t* buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int at = (OWN * wave + RPL * i) * D + 8 * lane;
        *reinterpret_cast<h8*>(buf + at) = kr[i];
        *reinterpret_cast<h8*>(buf + SPAN * D + at) = vr[i];
      }
    };
    const int stages = (count + SPAN - 1) / SPAN;
#pragma unroll
    for (int stage = 0; stage < 4; ++stage)
      if (my_turn(stage)) {
        look_up(stage);
        if (stage < 3) put_units(stage);
      }
    __syncthreads();
    load(0);

    f16v o[DT];
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;

    // ---- one step of 32 positions: rows R0 ... of a stage, u0 ... of the tile.
    // V's operands are read before the weights are computed (the fences keep
    // the reads there), into the registers that K's have left.  Rows start at
    // multiples of 128 bytes, so the swizzled chunk is an exclusive or on the
    // address; the addresses are rebuilt in every step (opaque()), not kept in
    // registers that the step has no room for.
    typedef __fp16 v4fp16 __attribute__((__vector_size__(8)));
    typedef __attribute__((address_space(3))) v4fp16 lds_v4;
    typedef const __attribute__((address_space(3))) h8 lds_h8;
    h8 k[KS], va[2][DT];
    const unsigned key_at =
        lds_address(s_kv) +
        (unsigned)(col * D * 2 + ((half ^ (D == 128 ? col & 15 : (col >> 1) & 7)) << 4));
    const int value_row = 4 * half + ((lane & 15) >> 2);
    const unsigned value_at =
        lds_address(s_kv) +
        (unsigned)((SPAN + value_row) * D * 2 +
                   ((((lane >> 4) & 1) ^ (D == 128 ? value_row & 7 : (value_row >> 1) & 3)) << 5) +
                   ((lane & 3) << 3));
    auto read_keys = [&](unsigned buf, int R0) {
      const unsigned at = opaque(key_at) + buf + (unsigned)(R0 * D * 2);
#pragma unroll
      for (int s = 0; s < KS; ++s) k[s] = *(lds_h8*)(uintptr_t)(at ^ (unsigned)(s << 5));
    };
    auto read_values = [&](unsigned buf, int R0) {
      const unsigned at = opaque(value_at) + buf + (unsigned)(R0 * D * 2);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          h4 part[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            part[h] = __builtin_bit_cast(
                h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4*)(uintptr_t)(
                        (at ^ (unsigned)(t << 6)) + (unsigned)((16 * c + 8 * h) * D * 2))));
          va[c][t] = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    // Position of place u of the tile.
    auto position = [&](int u) { return u < sinks ? u : u + gap; };
    // Steps that some of the wave's vectors see, and those of which all of them
    // see all.
    const int sink_steps = (int)((min((long)p.sinks, (long)count) + 31) / 32);
    const int live_from = (min_from - gap) / 32, live_to = (max_len - gap + 31) / 32;
    const int clear_from = (max_from - gap + 31) / 32, clear_to = (min_len - gap) / 32;
    auto seen = [&](int step) {
      return (step < sink_steps || step >= live_from) && step < live_to && max_len > 0;
    };
    f16v sc;
    auto scores = [&]() {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[s], qb[s], sc, 0, 0, 0);
    };
    h8 w[2];
    // out of sight: positions from the length on and [p.sinks, from)
    const unsigned hidden = (unsigned)max(0, min(from, 0x7ffffffe) - p.sinks);
    auto weigh = [&](int step) {
      settle(sc);
      if (step < clear_from || step >= clear_to) {
        const int first = 32 * step + 4 * (int)opaque(half);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int pos = position(first + 8 * (e >> 2) + (e & 3));
          const int away = (pos >= len) | ((unsigned)(pos - p.sinks) < hidden);
          sc[e] = away ? -INFINITY : sc[e];
        }
      }
      float top = sc[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
      const unsigned x = __builtin_bit_cast(unsigned, top);
      const auto sw = __builtin_amdgcn_permlane32_swap(x, x, false, false);
      const unsigned s0 = sw[0], s1 = sw[1];
      top = fmaxf(__builtin_bit_cast(float, s0), __builtin_bit_cast(float, s1)) * p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(top > m + kLag) != 0) {
        const float next_m = top > m + kLag ? top : m;
        const float alpha = next_m == m ? 1.0f : fast_exp2(m - next_m);
        m = next_m;
        sum *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= alpha;
      }
      const float shift = m == -INFINITY ? 0.0f : m - kChunkRaise;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[e >> 3][e & 7] = (half_t)fast_exp2(__fmaf_rn(sc[e], p.scale_log2, -shift));
      const h8 ones = {(half_t)1.0f, (half_t)1.0f, (half_t)1.0f, (half_t)1.0f,
                       (half_t)1.0f, (half_t)1.0f, (half_t)1.0f, (half_t)1.0f};
      sum = dot8(w[0], ones, dot8(w[1], ones, sum));
    };
    auto add_values = [&]() {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t)
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[c][t], w[c], o[t], 0, 0, 0);
    };

    // ---- the stages
    store(s_kv);
    load(1);
    for (int i = 0; i < stages; ++i) {
      const unsigned buf = (unsigned)((i & 1) * STAGE * 2);
      // stage i and the units of stage i + 2 are in LDS, stage i - 1 has been read
      lds_barrier();
      store(s_kv + ((i + 1) & 1) * STAGE);
      load(i + 2);
      if (my_turn(i + 3)) put_units(i + 3);
      if (my_turn(i + 4)) look_up(i + 4);
#pragma unroll
      for (int s = 0; s < (PG > 1 ? 1 : 2); ++s) {
        const int R0 = PG > 1 ? 32 * pg : 32 * s, step = i * (SPAN / 32) + R0 / 32;
        if (!seen(step)) continue;
        read_keys(buf, R0);
        __builtin_amdgcn_sched_barrier(0);
        scores();
        __builtin_amdgcn_sched_barrier(0);
        read_values(buf, R0);
        __builtin_amdgcn_sched_barrier(0);
        weigh(step);
        add_values();
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- join and store
    bad = __syncthreads_or(bad);
    sum += __shfl_xor(sum, 32, kWave);
    if (bad && len > 0) {  // some position of the tile has no page: one of this vector's?
      const int sink_end = min(p.sinks, from);
      bool whole = true;
      for (int i = 0; i * (long)p.page_size < sink_end; ++i) whole &= window_page_ok(p, table[i]);
      for (int i = window_page(p, from); i <= window_page(p, len - 1); ++i)
        whole &= window_page_ok(p, table[i]);
      if (!whole) len = 0;
    }
    float scale = 1.0f / sum, top = m;
    bool nan = false;  // in what this lane stored of its vector
    if constexpr (PG > 1) {
      if (half == 0) {
        s_max[wave][col] = m;
        s_sum[wave][col] = sum;
      }
      __syncthreads();
      float total = 0.0f;
#pragma unroll
      for (int g = 0; g < PG; ++g) top = fmaxf(top, s_max[g * VG + vg][col]);
#pragma unroll
      for (int g = 0; g < PG; ++g) {
        const float other = s_max[g * VG + vg][col];
        total += other == -INFINITY ? 0.0f : fast_exp2(other - top) * s_sum[g * VG + vg][col];
      }
      scale = m == -INFINITY ? 0.0f : fast_exp2(m - top) / total;
      // the groups' sums in fp32, as many 32-dim tiles a pass as fit: group pg
      // finishes EPG of a tile's elements (element e: dim 8 (e / 4) + 4 half + e % 4)
      float* hand = reinterpret_cast<float*>(s_kv);
      constexpr int kTile = 16 * kWave, EPG = 16 / PG;
      constexpr int FIT = (int)(sizeof(s_kv) / (sizeof(float) * WAVES * kTile));
      constexpr int TILES = FIT < DT ? FIT : DT;
      static_assert(TILES > 0 && DT % TILES == 0, "a pass fits");
#pragma unroll
      for (int first = 0; first < DT; first += TILES) {
        if (first) __syncthreads();
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            hand[(wave * TILES + t) * kTile + e * kWave + lane] = o[first + t][e] * scale;
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int part = 0; part < EPG / 4; ++part) {
            const int quad = pg * (EPG / 4) + part;
            float val[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < PG; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                val[e] += hand[((g * VG + vg) * TILES + t) * kTile + (4 * quad + e) * kWave + lane];
            if (len > 0)
              *reinterpret_cast<h4*>(p.out + ((size_t)row * p.q_heads + head) * D +
                                     32 * (first + t) + 8 * quad + 4 * half) =
                  h4{(half_t)val[0], (half_t)val[1], (half_t)val[2], (half_t)val[3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) nan |= !(val[e] == val[e]);
          }
      }
    } else {
      // rows through LDS (16-byte chunks swizzled by the row), so that whole
      // rows are stored: lane l then holds chunk l % CH of row l / CH
      half_t* rows = s_kv + wave * 32 * D;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          o[t][e] *= scale;
          nan |= !(o[t][e] == o[t][e]);
        }
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<h4*>(rows + col * D + (((4 * t + e) ^ (col & (CH - 1))) << 3) + 4 * half) =
              h4{(half_t)o[t][4 * e], (half_t)o[t][4 * e + 1], (half_t)o[t][4 * e + 2],
                 (half_t)o[t][4 * e + 3]};
      __builtin_amdgcn_wave_barrier();
      const int put = len > 0 ? row * p.q_heads + head : -1;
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) {
        const int R = RPL * i + lane / CH;
        const int to = __shfl(put, R, kWave);
        const h8 val = *reinterpret_cast<const h8*>(rows + R * D + ((slot ^ (R & (CH - 1))) << 3));
        if (to >= 0) *reinterpret_cast<h8*>(p.out + (size_t)to * D + 8 * slot) = val;
      }
    }
    // A weight of 0 times an infinity or NaN of V that the vector does not see
    // (another one of the tile does) is a NaN, and so is what weights past the
    // range of fp16 leave, or none at all (scores of 2^24 and more, whose fp32
    // maximum is several powers of two off): such vectors are done again, one at a
    // time, over their own positions alone and with weights of fp32.
    nan &= len > 0 && finite(top);
    if (__syncthreads_or(nan)) {
      unsigned long long again = __builtin_amdgcn_ballot_w64(nan);
      again = (again | again >> 32) & 0xFFFFFFFFull;
      PlainScratch& scratch = reinterpret_cast<PlainScratch*>(s_kv)[wave];
      static_assert(sizeof(PlainScratch) * WAVES <= sizeof(s_kv), "a scratch for every wave");
      while (again) {
        const int from_lane = __builtin_ctzll(again);
        again &= again - 1;
        plain_row<D>(p, __shfl(row, from_lane, kWave), __shfl(head, from_lane, kWave), scratch);
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ host
int window_params(WindowParams& p, const char* what, const void* q, const void* key_pool,
                  const void* value_pool, const int32_t* valid, const int32_t* tables, void* out,
                  int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                  int64_t page_size, int64_t max_pages, int64_t pool_pages, int64_t page_stride,
                  int64_t head_stride, int64_t window, int64_t sinks) {
  const std::string name = std::string(what) + ": ";
  TMC_REQUIRE(q && key_pool && value_pool && valid && tables && out, name + "null device pointer.");
  TMC_REQUIRE(head_dim >= 8 && head_dim <= kPlainMaxDim && head_dim % 8 == 0,
              name + "head_dim must be a multiple of 8 up to 256.");
  TMC_REQUIRE(rows > 0 && rows < (1LL << 24) && q_heads > 0 && kv_heads > 0 &&
                  q_heads < 65536 && q_heads % kv_heads == 0,
              name + "invalid rows or heads.");
  TMC_REQUIRE(page_size > 0 && max_pages > 0 && page_size < (1LL << 30) &&
                  max_pages < (1LL << 30) && page_size * max_pages < (1LL << 30) &&
                  pool_pages > 0 && pool_pages < (1LL << 31),
              name + "invalid page geometry.");
  TMC_REQUIRE(page_stride % 8 == 0 && head_stride % 8 == 0 && page_stride < (1LL << 40) &&
                  head_stride < (1LL << 40) && head_stride >= page_size * head_dim &&
                  page_stride >= (kv_heads - 1) * head_stride + page_size * head_dim,
              name + "strides must be multiples of 8 elements, the head stride hold a head's page "
                     "rows and the page stride every kv head.");
  TMC_REQUIRE(aligned16(q) && aligned16(key_pool) && aligned16(value_pool) && aligned16(out),
              name + "q, K, V and out must be 16-byte aligned.");
  TMC_REQUIRE(window >= 1 && sinks >= 0, name + "window must be at least 1 and sinks at least 0.");
  p = WindowParams{};
  p.q = static_cast<const half_t*>(q);
  p.k = static_cast<const half_t*>(key_pool);
  p.v = static_cast<const half_t*>(value_pool);
  p.out = static_cast<half_t*>(out);
  p.valid = valid;
  p.tables = tables;
  p.page_stride = (long)page_stride;
  p.head_stride = (long)head_stride;
  p.pool_pages = (int)pool_pages;
  p.rows = (int)rows;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads);
  p.dim = (int)head_dim;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages;
  if (page_size > 1) {
    // magic = floor(2^(31 + s) / d) + 1 with d <= 2^s: magic d - 2^(31 + s) is
    // in (0, 2^s], so the quotient is exact below 2^31
    int s = 1;
    while (((int64_t)1 << s) < page_size) ++s;
    p.page_magic = (unsigned)(((uint64_t)1 << (31 + s)) / (uint64_t)page_size + 1);
    p.page_shift = s - 1;
  }
  const int64_t capacity = page_size * max_pages;
  p.window = (int)std::min(window, capacity);
  p.sinks = (int)std::min(sinks, capacity);
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
  return 0;
}

int launch_plain(const WindowParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(window_plain_kernel, dim3((unsigned)p.rows, (unsigned)p.q_heads), dim3(kWave),
                     0, stream, p);
  return check_launch("window_plain_kernel");
}

}  // namespace
}  // namespace tmc

using namespace tmc;

namespace tmc {
namespace {
// The shapes window_decode_kernel takes; the others run window_plain_kernel.
bool decode_shape(int64_t head_dim) {
  return head_dim == 64 || head_dim == 128;
}
// Query heads of one kv head beyond 16 are done 16 or fewer at a time, as if
// they had a kv head each.
int64_t decode_splits(int64_t q_heads, int64_t kv_heads) {
  return (q_heads / kv_heads + 15) / 16;
}
// Steps of a row that sees as much as it can.
int64_t decode_steps(int64_t head_dim, int64_t capacity, int64_t window, int64_t sinks) {
  const int64_t step = head_dim == 128 ? 16 : 32;
  const int64_t seen = std::min(capacity, std::min(window, capacity) + std::min(sinks, capacity));
  return (seen + step - 1) / step;
}
// Blocks a row, one of `units`: as many as give every CU one, twice that where
// shares are then long (rows of unlike lengths), while a full row leaves each
// kDecodeLeast steps, and not more than the square root of the steps: a step
// takes about as long as one more partial at the join (0.16 and 0.22 us at 4
// query heads of 128 dims), which takes 16 at a time.  Rows of up to
// kDecodeAlone steps are a block's.  us, 8 kv heads of 128 dims.  One request,
// shared and alone: 320 positions (20 steps) 7.8 and 7.1, 384 8.1 and 7.7, 512 8.1
// and 8.6, 1024 8.4 and 11.9, 4096 11.5 and 33, 8192 13.9 (15.0 in 32 parts, 23
// in 64) and 60; of 64 dims 512 (16 steps) 7.2 and 6.4, 768 7.2 and 7.4, 1024 7.3
// and 8.4.  16 requests up to 4096, window 1024: 16.4 in 2 parts (the rule's), 15.4
// in 1, 17.3 in 4; window 4096 34.6 in 4 (the rule's), 37 in 2, 50 in 1; 32
// requests, window 1024, 25.4 in 1 (the rule's), 28.9 in 2.  The lengths are not
// known here: with 256 rows and more none is shared, and a batch of 32 with one row
// of 8192 takes 57, active alone 59, where one request takes 12.
int decode_parts(int64_t units, int64_t head_dim, int64_t capacity, int64_t window,
                 int64_t sinks) {
  const int64_t steps = decode_steps(head_dim, capacity, window, sinks);
  int64_t most = (kDecodeCus + units - 1) / units;
  if (most > 1 && steps / most > 96) most *= 2;
  const int parts =
      decode_shares(steps, std::min(most, (int64_t)std::ceil(std::sqrt((double)steps))));
  return parts > 16 ? parts / 16 * 16 : parts;
}
int launch_decode(const WindowParams& p, const DecodePlan& plan, unsigned blocks,
                  hipStream_t stream) {
  // Eight waves (two a SIMD) where there is a block a CU, four where there are two,
  // and a wave a block where there are more, which then come and go one by one.
  // us, one request, 4 waves and 8: 8192 positions 14.2 and 13.9, 300 positions of
  // 32 kv heads 7.7 and 7.1 (four stages a ring instead: 14.6 and 7.4).  8 kv heads
  // of 128 dims, 8 waves, 4 and 1: 64 requests, window 256 19.6, 15.5 and 15.9; 96,
  // window 128 20.2, 16.1 and 13.1; 250, window 128 53, 36 and 29; 96, window 2048
  // 140, 137 and 138.
#define TMC_DECODE(DIM, STEP, WAVES)                                                             \
  hipLaunchKernelGGL((window_decode_kernel<DIM, STEP, 2, WAVES>), dim3(blocks), dim3(WAVES * kWave), \
                     0, stream, p, plan)
#define TMC_DECODE_WAVES(DIM, STEP)                   \
  if (blocks <= kDecodeCus) TMC_DECODE(DIM, STEP, 8); \
  else if (blocks <= 2 * kDecodeCus) TMC_DECODE(DIM, STEP, 4); \
  else TMC_DECODE(DIM, STEP, 1)
  if (p.dim == 128) {
    TMC_DECODE_WAVES(128, 16);
  } else {
    TMC_DECODE_WAVES(64, 32);
  }
#undef TMC_DECODE_WAVES
#undef TMC_DECODE
  return check_launch("window_decode_kernel");
}
}  // namespace
}  // namespace tmc

extern "C" size_t tmc_window_attention_workspace_bytes(int64_t batch, int64_t q_heads,
                                                       int64_t kv_heads, int64_t head_dim,
                                                       int64_t capacity, int64_t window,
                                                       int64_t sinks) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || capacity <= 0 || q_heads % kv_heads ||
      window < 1 || sinks < 0 || !decode_shape(head_dim))
    return 0;
  const int64_t splits = decode_splits(q_heads, kv_heads), units = batch * kv_heads * splits;
  const int parts = decode_parts(units, head_dim, capacity, window, sinks);
  const int64_t heads = (q_heads / kv_heads + splits - 1) / splits;
  return parts < 2 ? 0
                   : kCounterBytes +
                         (size_t)units * parts * heads * (head_dim + 2) * sizeof(float);
}

extern "C" int tmc_window_decode_attention(
    const void* q, const void* key_pool, const void* value_pool, const int32_t* valid_lengths,
    const int32_t* block_tables, const int32_t* active_count, void* out, int dtype,
    int64_t max_batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
    int64_t max_pages, int64_t pool_pages, int64_t page_stride, int64_t head_stride,
    int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, int layout,
    void* stream) {
  TMC_REQUIRE(dtype == TMC_F16, "Window attention: the gfx950 kernel stores K/V in fp16.");
  WindowParams p;
  if (window_params(p, "Window attention", q, key_pool, value_pool, valid_lengths, block_tables,
                    out, max_batch, q_heads, kv_heads, head_dim, page_size, max_pages, pool_pages,
                    page_stride, head_stride, window, sinks))
    return 1;
  TMC_REQUIRE(max_batch < 65536, "Window attention: max_batch must be below 65536.");
  TMC_REQUIRE(layout == 0 || layout == TMC_LAYOUT_Y_PACKED,
              "Window attention: layout must be 0 or TMC_LAYOUT_Y_PACKED.");
  const size_t need = tmc_window_attention_workspace_bytes(
      max_batch, q_heads, kv_heads, head_dim, page_size * max_pages, window, sinks);
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "Window attention: workspace is smaller than "
              "tmc_window_attention_workspace_bytes() or not 16-byte aligned.");
  p.active = active_count;
  p.table_rows = p.rows;
  p.own_table = 1;
  if (layout) p.out_pass = (long)((q_heads * head_dim + 31) / 32) * 512;
  // 16-byte units of the pools are counted in 32 bits: below 64 GiB each
  if (!decode_shape(head_dim) ||
      (uint64_t)pool_pages * (uint64_t)page_stride / 8 >= 0xFFFFFFFFull)
    return launch_plain(p, as_stream(stream));
  DecodePlan plan{};
  plan.splits = (int)decode_splits(q_heads, kv_heads);
  const int64_t units = max_batch * kv_heads * plan.splits;
  plan.heads = (p.group + plan.splits - 1) / plan.splits;
  plan.parts = decode_parts(units, head_dim, page_size * max_pages, window, sinks);
  const unsigned blocks = (unsigned)(units * plan.parts);
  if (need) {
    plan.arrivals = static_cast<int*>(workspace);
    plan.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                          kCounterBytes);
  }
  return launch_decode(p, plan, blocks, as_stream(stream));
}

extern "C" int tmc_window_prefill_attention_f16(
    const void* q, const void* key_pool, const void* value_pool, const int32_t* valid_lengths,
    const int32_t* block_tables, const int32_t* row_table, int64_t table_rows,
    const int32_t* active_count, void* out, int64_t rows, int64_t q_heads, int64_t kv_heads,
    int64_t head_dim, int64_t page_size, int64_t max_pages, int64_t pool_pages,
    int64_t page_stride, int64_t head_stride, int64_t window, int64_t sinks, void* stream) {
  WindowParams p;
  if (window_params(p, "Window prefill attention", q, key_pool, value_pool, valid_lengths,
                    block_tables, out, rows, q_heads, kv_heads, head_dim, page_size, max_pages,
                    pool_pages, page_stride, head_stride, window, sinks))
    return 1;
  TMC_REQUIRE(active_count, "Window prefill attention: null active count.");
  TMC_REQUIRE(table_rows >= 1 && (row_table || table_rows == 1) && table_rows < (1LL << 24),
              "Window prefill attention: table_rows must be 1 without a row table, else at "
              "least 1.");
  p.active = active_count;
  p.row_table = row_table;
  p.table_rows = (int)table_rows;
  if (!decode_shape(head_dim) || (uint64_t)pool_pages * (uint64_t)page_stride / 8 >= 0xFFFFFFFFull)
    return launch_plain(p, as_stream(stream));
  // Few tokens, or short windows: each token as if it were a request of its own.  us,
  // in tiles and here, 32 query heads.  8 kv heads of 128 dims: one token over 300
  // positions 12.0 and 7.1, over 1024 20.5 and 12.1, 32 over 4096 54 and 35, 32 over 20
  // 9.3 and 5.3; 64 over 100 9.8 and 6.8, over 1024 20.8 and 20.7, over 4096 53 and 67;
  // 256 over 20 9.9 and 7.5, over 100 10.4 and 12.5.  Of 64 dims: 64 over 300 8.7 and
  // 7.6, over 1024 13.8 and 13.3; 128 over 300 8.7 and 11.0.  32 kv heads of 128: 16
  // over 300 11.7 and 9.6, over 4096 54 and 68; 32 over 20 8.7 and 5.2, over 300 12.3
  // and 16.6, and over 100 10.6 and 8.7, where the rule takes the tiles.
  const int64_t splits = decode_splits(q_heads, kv_heads), units = rows * kv_heads * splits;
  const int64_t steps = decode_steps(head_dim, page_size * max_pages, window, sinks);
  if (units <= kDecodeCus || (units <= 2 * kDecodeCus && steps <= 64) || units * steps <= 4096) {
    DecodePlan plan{};
    plan.parts = 1;
    plan.splits = (int)splits;
    plan.heads = (int)((p.group + splits - 1) / splits);
    return launch_decode(p, plan, (unsigned)units, as_stream(stream));
  }
  if (p.group > 64) return launch_plain(p, as_stream(stream));
  // A block a CU: tiles of 256 vectors, or of 128 or 64, whose waves share the
  // positions, while there are few.  us for tiles of 64, 128 and 256, 32 heads of 128
  // dims, window 2048: 512 tokens 37, 51 and 79, 768 67, 52 and 79, 1024 67, 55 and 79,
  // 1280 98, 100 and 80, 2048 132, 107 and 93; over 8 kv heads 512 tokens 35, 46 and 70,
  // 1024 64, 50 and 71, 1280 95, 91 and 72.
  const int64_t wide = (rows + 256 / p.group - 1) / (256 / p.group) * kv_heads;
  const int vectors = wide <= 64 ? 64 : wide <= 128 ? 128 : 256;
  const int tokens = vectors / p.group;
  const int tiles = (int)((rows + tokens - 1) / tokens);
  const dim3 grid((unsigned)(tiles * kv_heads)), block(kChunkWaves * kWave);
#define TMC_CHUNK(DIM, PG)                                                                        \
  hipLaunchKernelGGL((window_chunk_kernel<DIM, PG>), grid, block, 0, as_stream(stream), p, tiles, \
                     tokens)
#define TMC_CHUNK_VECTORS(DIM)                  \
  if (vectors == 64) TMC_CHUNK(DIM, 4);         \
  else if (vectors == 128) TMC_CHUNK(DIM, 2);   \
  else TMC_CHUNK(DIM, 1)
  if (head_dim == 128) {
    TMC_CHUNK_VECTORS(128);
  } else {
    TMC_CHUNK_VECTORS(64);
  }
#undef TMC_CHUNK_VECTORS
#undef TMC_CHUNK
  return check_launch("window_chunk_kernel");
}
