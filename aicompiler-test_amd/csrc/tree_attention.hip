// Attention of trees of drafted tokens over a paged cache, gfx950.
//
// Node i of request r, with `cached` positions before its tree, sees [0, cached)
// and position cached + j for every bit j < count of its mask:
//   out = sum_s w_s v_s / sum_s w_s,  w_s = exp(q . k_s / sqrt(D) - max),
// and zeros where it sees nothing.
#include "attention_device.hpp"
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tmc {
namespace {

struct TreeParams {
  const half_t* q;          // [batch][nodes][q_heads][D]
  const half_t* k;          // pools [pages][kv_heads][page_size][D] at the strides
  const half_t* v;
  half_t* out;              // [batch][nodes][q_heads][D]
  const int32_t* cached;    // [batch]
  const uint32_t* masks;    // [batch][nodes][words]
  const int32_t* counts;    // [batch] or null: all nodes
  const int32_t* tables;    // [batch][max_pages]
  const int32_t* active;    // or null: all requests
  long page_stride, head_stride;
  int pool_pages, batch, nodes, words, q_heads, kv_heads, group, dim;
  int page_size, max_pages;
  PageDivide divide;
  float scale_log2;         // log2(e) / sqrt(D)
};

// A request: its cached positions and the nodes of its tree, -1 for a request to
// be left alone.
struct Request {
  int cached, count;
};
__device__ __forceinline__ Request request_of(const TreeParams& p, int r) {
  const int active = p.active ? p.active[0] : p.batch;
  const int cached = p.cached[r];
  const int count = p.counts ? min(p.counts[r], p.nodes) : p.nodes;
  const bool whole = r < active && count > 0 && cached >= 0 &&
                     (long)cached + count <= (long)p.page_size * p.max_pages;
  return Request{cached, whole ? count : -1};
}
__device__ __forceinline__ bool tree_page_ok(const TreeParams& p, int page) {
  return page >= 0 && page < p.pool_pages;
}

// ------------------------------------------------------------ any geometry
// One wave per (node, query head): 64 positions at a time, one per lane for the
// scores (whole K rows in 16-byte chunks), then lanes over the dims for P V.
constexpr int kPlainMaxDim = 256;

struct PlainScratch {  // of one wave
  __align__(16) half_t q[kPlainMaxDim];
  float weight[kWave];
  long at[kWave];
};

template <int DIM>
__device__ __forceinline__ void plain_node(const TreeParams& p, int r, const Request& request,
                                           int node, int head, PlainScratch& scratch) {
  constexpr int TILES = (DIM ? DIM : kPlainMaxDim) / kWave;
  constexpr int kAhead = 8;  // chunks of K, rows of V loaded at once
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t* table = p.tables + (size_t)r * p.max_pages;
  const int kvh = head / p.group, d = DIM ? DIM : p.dim;
  const size_t row = (size_t)r * p.nodes + node;
  const half_t* q = p.q + (row * p.q_heads + head) * d;
  const uint32_t* mask = p.masks + row * p.words;
  for (int i = lane; i < d; i += kWave) scratch.q[i] = q[i];
  const int count = request.cached + request.count;
  float m = -INFINITY, sum = 0.0f, o[TILES] = {};
  int column[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) column[t] = min(lane + t * kWave, d - 1);
  bool bad = false, any = false;
  for (int u0 = 0; u0 < count; u0 += kWave) {
    const int pos = u0 + lane;
    float score = -INFINITY;
    long at = -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (pos < count) {
      const int slot = p.divide(pos), page = table[slot];
      const int bit = pos - request.cached;
      const bool sees = bit < 0 || (mask[bit >> 5] >> (bit & 31) & 1);
      if (!tree_page_ok(p, page)) {
        bad = true;
      } else if (sees) {
        any = true;
        at = (long)page * p.page_stride + (long)kvh * p.head_stride +
             (long)(pos - slot * p.page_size) * d;
        float dot = 0.0f;
#pragma unroll kAhead
        for (int c = 0; c < d; c += 8)
          dot = dot8(load_h8(scratch.q + c), load_h8(p.k + at + c), dot);
        score = dot * p.scale_log2;
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
  any = __any(any);
  sum = cross_sum<1>(sum);
#pragma unroll
  for (int t = 0; t < TILES; ++t)
    if (lane + t * kWave < d)
      p.out[(row * p.q_heads + head) * d + lane + t * kWave] =
          any ? (half_t)(o[t] / sum) : (half_t)0.0f;
}

__global__ __launch_bounds__(kWave) void tree_plain_kernel(TreeParams p) {
  __shared__ PlainScratch scratch;
  const int r = blockIdx.x / p.nodes, node = blockIdx.x - r * p.nodes;
  const Request request = request_of(p, r);
  if (node >= request.count) return;
  plain_node<0>(p, r, request, node, blockIdx.y, scratch);
}

// ------------------------------------------------------------ matrix cores
// D = 64 and 128.  A unit is a (request, kv head) with up to 64 of its query
// vectors (nodes x query heads of that kv head, in C tiles of 16); a step is 32 of
// its positions.  A unit's steps are a block's, or shared by several; the last of
// these to arrive joins their partials, in block order.
//
// The block's waves take the steps of a share in turn, each over a ring of two
// steps in LDS that only it touches, filled by 16-byte loads straight to LDS: no
// barrier, no register holds a load in flight, and a stage is loaded again as soon
// as its operands are in registers.  K and V rows lie in LDS as in their pages,
// 16-byte chunks (K) and 32-byte units (V) swizzled by the row so that the operand
// reads spread over the banks.  A position that does not exist reads a zero row.
// Scores S^T = K Q^T leave lane (vector j, group g) with positions 4g .. 4g+3 of
// both halves of the step, the order in which O^T = V^T P^T wants its weights; V^T
// comes from transposing LDS reads.  K and V are read from LDS once for all C
// tiles.
//
// Only steps that reach into the tree look at masks: 32 bits of a node's mask for
// the 32 positions.
constexpr int kTreeStep = 32, kTreeStages = 2, kTreeWaves = 4;
constexpr int kTreeCus = 256;                          // of an MI355X
constexpr int kTreeLeast = 8, kTreeAlone = 10;         // steps
constexpr int kTreeTiles = 4;                          // tiles of 16 vectors a wave holds, at most

struct TreePlan {
  float* slots;   // [units][parts][16 C][D + 2]
  int* arrivals;  // [units], kCounterStride apart
  int parts, tiles, items;
  float per_step;  // steps a share for each step of all requests
};

// Weights are stored 2^kRaise times their value in fp16 and a new maximum moves
// their scale only when it is kLag above the one in use, so a wave seldom rescales
// its sums: weights are at most 2^(kRaise + kLag) and keep 11 bits down to 2^-24 of
// that scale.  fp16 is what the matrix cores multiply with V's type; the sum takes
// the rounded weights, so an output is off by up to 2^-11 of the mean of |v| for it,
// beside the 2^-11 of its own fp16.
constexpr float kLag = 5.0f, kRaise = 10.0f;
constexpr unsigned kNoUnit = 0xFFFFFFFFu;

// The operands of one step out of LDS, waits included: the compiler would let
// such reads wait for every load to LDS in flight.
template <int D, int OFFSET, int PAGE_OFFSET>
__device__ __forceinline__ void read_keys(const unsigned (&at)[D / 32], unsigned page_at,
                                          h8 (&k)[2][D / 32], int& page) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b32 %8, %13 offset:%16\n\t"
        "ds_read_b128 %0, %9 offset:%14\n\tds_read_b128 %1, %10 offset:%14\n\t"
        "ds_read_b128 %2, %11 offset:%14\n\tds_read_b128 %3, %12 offset:%14\n\t"
        "ds_read_b128 %4, %9 offset:%15\n\tds_read_b128 %5, %10 offset:%15\n\t"
        "ds_read_b128 %6, %11 offset:%15\n\tds_read_b128 %7, %12 offset:%15\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]),
          "=&v"(k[1][1]), "=&v"(k[1][2]), "=&v"(k[1][3]), "=&v"(page)
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(page_at), "n"(OFFSET),
          "n"(OFFSET + 32 * D), "n"(PAGE_OFFSET)
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
// (v[0]) and of its last 16 (v[1]).
template <int D, int OFFSET>
__device__ __forceinline__ void read_values(const unsigned (&at)[D / 16], h4 (&v)[2][D / 16]) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %1, %17 offset:%24\n\t"
        "ds_read_b64_tr_b16 %2, %18 offset:%24\n\tds_read_b64_tr_b16 %3, %19 offset:%24\n\t"
        "ds_read_b64_tr_b16 %4, %20 offset:%24\n\tds_read_b64_tr_b16 %5, %21 offset:%24\n\t"
        "ds_read_b64_tr_b16 %6, %22 offset:%24\n\tds_read_b64_tr_b16 %7, %23 offset:%24\n\t"
        "ds_read_b64_tr_b16 %8, %16 offset:%25\n\tds_read_b64_tr_b16 %9, %17 offset:%25\n\t"
        "ds_read_b64_tr_b16 %10, %18 offset:%25\n\tds_read_b64_tr_b16 %11, %19 offset:%25\n\t"
        "ds_read_b64_tr_b16 %12, %20 offset:%25\n\tds_read_b64_tr_b16 %13, %21 offset:%25\n\t"
        "ds_read_b64_tr_b16 %14, %22 offset:%25\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[0][4]),
          "=&v"(v[0][5]), "=&v"(v[0][6]), "=&v"(v[0][7]), "=&v"(v[1][0]), "=&v"(v[1][1]),
          "=&v"(v[1][2]), "=&v"(v[1][3]), "=&v"(v[1][4]), "=&v"(v[1][5]), "=&v"(v[1][6]),
          "=&v"(v[1][7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
          "v"(at[7]), "n"(OFFSET), "n"(OFFSET + 32 * D)
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

// A vector's products read by vector instructions: see settle().
template <int C> __device__ __forceinline__ void settle_all(f4 (&sc)[C][2]) {
#pragma unroll
  for (int c = 0; c + 1 < C; ++c) asm volatile("" : "+v"(sc[c][0]), "+v"(sc[c][1]));
  if constexpr (C == 1)
    asm volatile("s_nop 15" : "+v"(sc[0][0]), "+v"(sc[0][1]));
  else if constexpr (C == 2)
    asm volatile("s_nop 15" : "+v"(sc[0][0]), "+v"(sc[0][1]), "+v"(sc[1][0]), "+v"(sc[1][1]));
  else if constexpr (C == 3)
    asm volatile("s_nop 15" : "+v"(sc[0][0]), "+v"(sc[0][1]), "+v"(sc[1][0]), "+v"(sc[1][1]),
                              "+v"(sc[2][0]), "+v"(sc[2][1]));
  else
    asm volatile("s_nop 15" : "+v"(sc[0][0]), "+v"(sc[0][1]), "+v"(sc[1][0]), "+v"(sc[1][1]),
                              "+v"(sc[2][0]), "+v"(sc[2][1]), "+v"(sc[3][0]), "+v"(sc[3][1]));
}

// Bits [from, from + 32) of a node's mask: ones before the tree, zeros behind it.
__device__ __forceinline__ unsigned mask_window(const uint32_t* mask, int count, int from) {
  auto word = [&](int w) -> unsigned {
    const int left = count - 32 * w;
    if (w < 0) return ~0u;
    if (left <= 0) return 0u;
    return mask[w] & (left >= 32 ? ~0u : (1u << left) - 1u);
  };
  const int w = from >> 5, shift = from & 31;
  const unsigned low = word(w);
  return shift ? low >> shift | word(w + 1) << (32 - shift) : low;
}
__device__ __forceinline__ bool sees_nothing(const TreeParams& p, const Request& request,
                                             const uint32_t* mask) {
  unsigned any = request.cached > 0;
  for (int w = 0; 32 * w < request.count; ++w) any |= mask_window(mask, request.count, 32 * w);
  return any == 0;
}
__device__ __forceinline__ int steps_of(const Request& r) {
  return r.count > 0 ? (r.cached + r.count + kTreeStep - 1) / kTreeStep : 0;
}

template <int D, int C>
__global__ __launch_bounds__(kTreeWaves * kWave, D == 128 ? 1 : 2) void tree_attention_kernel(
    TreeParams p, TreePlan plan) {
  constexpr int STEP = kTreeStep, STAGES = kTreeStages, WAVES = kTreeWaves, NV = 16 * C;
  constexpr int KS = D / 32, DT = D / 16, CH = D / 8;
  constexpr int RPL = kWave / CH, LOADS = STEP / RPL;  // rows a load, loads of K (of V) a step
  constexpr int STAGE = 2 * STEP * D;                  // halves
  constexpr int THREADS = WAVES * kWave;
  constexpr int ROW = D + 4;                           // floats of a vector's sums in LDS
  constexpr int RING_BYTES = WAVES * STAGES * STAGE * 2, MET_BYTES = WAVES * NV * ROW * 4;
  __shared__ __align__(16) char s_space[RING_BYTES > MET_BYTES ? RING_BYTES : MET_BYTES];
  __shared__ int s_pages[WAVES * STAGES * kWave];
  __shared__ float s_max[WAVES][NV], s_sum[WAVES][NV];
  __shared__ int s_last;
  __shared__ float s_total[WAVES];
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) const void global_void;
  static_assert(sizeof(PlainScratch) * WAVES <= sizeof(s_space), "a scratch for every wave");

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int j = lane & 15, g = lane >> 4;

  // ---- this block: the tiles of one item (request, kv head, part) on one XCD, whose
  // L2 then holds its pages
  const int rest = blockIdx.x / 8, item = rest / plan.tiles * 8 + blockIdx.x % 8;
  const int tile = rest % plan.tiles;
  if (item >= plan.items) return;
  const int pair = item / plan.parts, part = item - pair * plan.parts;
  const int r = pair / p.kv_heads, kvh = pair - r * p.kv_heads;
  const int unit = pair * plan.tiles + tile;
  const Request request = request_of(p, r);
  const int first_vec = tile * NV, vecs = min(NV, request.count * p.group - first_vec);
  int steps = steps_of(request), shares = 1;
  if (plan.parts > 1) {
    // Shares of about as many steps each, over all requests, as give every CU its
    // own, and of kTreeLeast or more.
    float total = 0.0f;
    for (int i = threadIdx.x; i < p.batch; i += THREADS) total += steps_of(request_of(p, i));
    total = wave_sum(total);
    if (lane == 0) s_total[wave] = total;
    __syncthreads();
    total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    const int share = max(kTreeLeast, (int)(total * plan.per_step) + 1);
    if (steps > kTreeAlone) shares = min(plan.parts, (steps + share - 1) / share);
  }
  if (vecs <= 0 || part >= shares) return;
  const int even = steps / shares, over = steps - even * shares;
  const int first_step = part * even + min(part, over);
  const int last_step = first_step + even + (part < over);

  // ---- LDS places: loads are linear (lane l: row l / CH, slot l % CH)
  half_t* ring = reinterpret_cast<half_t*>(s_space) + wave * STAGES * STAGE;
  unsigned key_at[KS], value_at[DT];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    key_at[s] = lds_address(ring) +
                (unsigned)(j * D * 2 + (((4 * s + g) ^ (D == 128 ? j : (j >> 1) & 7)) << 4));
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int R = 4 * g + (j >> 2), place = t ^ (D == 128 ? R & 7 : (R >> 1) & 3);
    value_at[t] =
        lds_address(ring) + (unsigned)(STEP * D * 2 + R * D * 2 + (place << 5) + ((j & 3) << 3));
  }
  int* pages = s_pages + wave * STAGES * kWave;
  const unsigned page_at = lds_address(pages + lane);
  const char* zero = reinterpret_cast<const char*>(s_zero_row);

  const int count = request.cached + request.count;  // positions
  const int32_t* table = p.tables + (size_t)r * p.max_pages;
  const unsigned head_unit = (unsigned)((size_t)kvh * p.head_stride / 8);
  h8 qb[C][KS];
  int row[C];  // of q, out and the masks
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int vec = first_vec + min(16 * c + j, vecs - 1), node = vec / p.group;
    row[c] = r * p.nodes + node;
    const half_t* q =
        p.q + ((size_t)row[c] * p.q_heads + kvh * p.group + (vec - node * p.group)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[c][s] = load_h8(q + 32 * s + 8 * g);
  }
  f4 o[C][DT];
  float m[C], lsum[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    m[c] = -INFINITY;
    lsum[c] = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[c][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  int bad = 0;

  // Table slot of the position that lane (l & 31) stands for in a step (past the
  // end: of the last one) and its row in that page.
  auto locate = [&](int step, int& slot_row) -> const int32_t* {
    const int pos = min(step * STEP + (lane & (STEP - 1)), count - 1);
    const int slot = p.divide(pos);
    slot_row = pos - slot * p.page_size;
    return table + slot;
  };
  // 16-byte unit where that position's row starts, kNoUnit when it has none
  auto place = [&](int step, int page, int slot_row) -> unsigned {
    const bool ok = tree_page_ok(p, page);
    bad |= !ok;
    return ok && step * STEP + (lane & (STEP - 1)) < count
               ? (unsigned)page * (unsigned)(p.page_stride / 8) + head_unit +
                     (unsigned)(slot_row * CH)
               : kNoUnit;
  };
  // K and V rows of a step, and the pages of the step that follows it in the
  // stage: those too by loads to LDS, so that no load the compiler could wait for
  // mixes with the ones in flight.
  auto issue = [&](unsigned first, const int32_t* next, int stage) {
    half_t* to = ring + stage * STAGE;
    __builtin_amdgcn_global_load_lds((global_void*)next, (lds_void*)(pages + stage * kWave), 4, 0, 0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int R = RPL * i + lane / CH, slot = lane % CH;
      const unsigned row_unit = (unsigned)__shfl((int)first, R, kWave);
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
  auto consume = [&](int step, const h8 (&k)[2][KS], const h4 (&v)[2][DT]) {
    f4 sc[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[c][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
          sc[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][s], qb[c][s], sc[c][t], 0, 0, 0);
      }
    settle_all<C>(sc);
    if (step * STEP + STEP > request.cached) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const unsigned sees = mask_window(p.masks + (size_t)row[c] * p.words, request.count,
                                          step * STEP - request.cached) >> (4 * g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(sees >> (16 * t + e) & 1)) sc[c][t][e] = -INFINITY;
      }
    }
    float top[C];
    bool grows = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      top[c] = fmaxf(fmaxf(fmaxf(sc[c][0][0], sc[c][0][1]), fmaxf(sc[c][0][2], sc[c][0][3])),
                     fmaxf(fmaxf(sc[c][1][0], sc[c][1][1]), fmaxf(sc[c][1][2], sc[c][1][3])));
      top[c] = max_of_groups(top[c]) * p.scale_log2;
      grows |= top[c] > m[c] + kLag;
    }
    if (__builtin_amdgcn_ballot_w64(grows) != 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float next = top[c] > m[c] + kLag ? top[c] : m[c];
        const float alpha = next == m[c] ? 1.0f : fast_exp2(m[c] - next);
        m[c] = next;
        lsum[c] *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[c][t] *= alpha;
      }
    }
    h8 w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float shift = m[c] == -INFINITY ? 0.0f : m[c] - kRaise;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[c][e] = (half_t)fast_exp2(__fmaf_rn(sc[c][e >> 2][e & 3], p.scale_log2, -shift));
      const h8 ones = {(half_t)1.0f, (half_t)1.0f, (half_t)1.0f, (half_t)1.0f,
                       (half_t)1.0f, (half_t)1.0f, (half_t)1.0f, (half_t)1.0f};
      lsum[c] = dot8(w[c], ones, lsum[c]);
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const h8 vt = __builtin_shufflevector(v[0][t], v[1][t], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int c = 0; c < C; ++c)
        o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, w[c], o[c][t], 0, 0, 0);
    }
  };

  // ---- the wave's steps: every WAVES-th of the share
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
  // One step out of its stage, and the stage loaded again.  BODY: every step that is
  // waited for or loaded exists.
  auto turn = [&](auto stage, auto body, int step) {
    constexpr int ST = decltype(stage)::value;
    constexpr bool BODY = decltype(body)::value;
    const int again = step + STAGES * WAVES;
    if (BODY || step + (STAGES - 1) * WAVES < last_step)
      wait_loads<(2 * LOADS + 1) * (STAGES - 1)>();
    else
      wait_loads<0>();
    h8 k[2][KS];
    h4 v[2][DT];
    int page;
    read_keys<D, ST * STAGE * 2, ST * kWave * 4>(key_at, page_at, k, page);
    read_values<D, ST * STAGE * 2>(value_at, v);
    if (BODY || again < last_step) {
      const unsigned first = place(again, page, slot_row[ST]);
      issue(first, locate(again + STAGES * WAVES, slot_row[ST]), ST);
    }
    consume(step, k, v);
  };
  static_assert(STAGES == 2, "a round is two turns");
  int step = mine;
  for (; step + (2 * STAGES - 1) * WAVES < last_step; step += STAGES * WAVES) {
    turn(std::integral_constant<int, 0>{}, std::true_type{}, step);
    turn(std::integral_constant<int, 1>{}, std::true_type{}, step + WAVES);
  }
  for (; step < last_step; step += STAGES * WAVES) {
    turn(std::integral_constant<int, 0>{}, std::false_type{}, step);
    if (step + WAVES < last_step)
      turn(std::integral_constant<int, 1>{}, std::false_type{}, step + WAVES);
  }

  // ---- the waves meet in LDS (the rings: every load into them has landed)
  bad = __syncthreads_or(bad);
  float* s_out = reinterpret_cast<float*>(s_space);  // [waves][NV][ROW]
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float sum = cross_sum<16>(lsum[c]);
    if (g == 0) {
      s_max[wave][16 * c + j] = m[c];
      s_sum[wave][16 * c + j] = sum;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<f4*>(s_out + (size_t)(wave * NV + 16 * c + j) * ROW + 16 * t + 4 * g) =
          o[c][t];
  }
  __syncthreads();
  // Two dims of an output; whether it is to be done again, see below.
  auto put = [&](int vec, int d, float top, float sum, float a, float b) -> bool {
    const int node = (first_vec + vec) / p.group;
    const size_t at = (size_t)r * p.nodes + node;
    if (top == -INFINITY && sees_nothing(p, request, p.masks + at * p.words)) {
      a = b = 0.0f;
      sum = 1.0f;
    }
    a /= sum;
    b /= sum;
    *reinterpret_cast<h2*>(p.out + (at * p.q_heads + kvh * p.group +
                                    (first_vec + vec - node * p.group)) * D + d) =
        h2{(half_t)a, (half_t)b};
    return (!(a == a) | !(b == b)) && finite(top);
  };
  const bool whole = shares == 1;
  constexpr size_t SLOT = (size_t)NV * (D + 2);
  float* slots = plan.slots + (size_t)unit * plan.parts * SLOT;
  unsigned long long again = 0;  // vectors with a NaN among the dims that this thread put
  for (int i = threadIdx.x; i < vecs * (D / 2); i += THREADS) {
    const int vec = i / (D / 2), d = i % (D / 2) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_max[w][vec]);
    float sum = 0.0f, val0 = 0.0f, val1 = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float high = s_max[w][vec];
      // (a wave that saw nothing has no weights, but NaN where it met one of V)
      const float scale = high == -INFINITY ? 0.0f : fast_exp2(high - top);
      const float2 mine = *reinterpret_cast<const float2*>(s_out + (size_t)(w * NV + vec) * ROW + d);
      sum += scale * s_sum[w][vec];
      val0 += scale * mine.x;
      val1 += scale * mine.y;
    }
    if (whole) {
      if (!bad && put(vec, d, top, sum, val0, val1)) again |= 1ull << vec;
    } else {
      float* out = slots + part * SLOT + (size_t)vec * (D + 2);
      store_pair(out + d, val0, val1);
      if (d == 0) store_pair(out + D, top, bad ? -1.0f : sum);
    }
  }
  if (!whole) {
    // the last of the unit's blocks joins the partials, in block order (every word
    // is written and read at agent scope; the stores have completed before the
    // arrival is counted)
    int* counter = plan.arrivals + unit * kCounterStride;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               shares - 1;
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0)
      __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = threadIdx.x; i < vecs * (D / 2); i += THREADS) {
      const int vec = i / (D / 2), d = i % (D / 2) * 2;
      float top = -INFINITY, sum = 0.0f, val0 = 0.0f, val1 = 0.0f;
      bool spoiled = false;
      constexpr int kAhead = 8;  // partials loaded at once
      for (int b = 0; b < shares; b += kAhead) {
        float2 x[kAhead], y[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float* in = slots + min(b + u, shares - 1) * SLOT + (size_t)vec * (D + 2);
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
            const float scale = y[u].x == -INFINITY ? 0.0f : fast_exp2(y[u].x - next);
            sum += y[u].y * scale;
            val0 += x[u].x * scale;
            val1 += x[u].y * scale;
          }
        top = next;
      }
      if (!spoiled && put(vec, d, top, sum, val0, val1)) again |= 1ull << vec;
    }
  }
  // A weight of 0 times an infinity or NaN of V that the node does not see (another
  // one of the tile does), a weight that fp16 rounds to 0 times an infinity, and
  // weights past its range (scores of 2^24 and more, whose fp32 maximum is several
  // powers of two off) give a NaN that weights of fp32 over a node's own positions
  // do not: such vectors are done again with those, one at a time.
  if (__syncthreads_or(again != 0)) {
    unsigned long long todo = 0, waiting = __builtin_amdgcn_ballot_w64(again != 0);
    for (; waiting; waiting &= waiting - 1)
      todo |= __shfl(again, __builtin_ctzll(waiting), kWave);
    PlainScratch& scratch = reinterpret_cast<PlainScratch*>(s_space)[wave];
    __builtin_amdgcn_s_waitcnt(0);  // the NaNs are stored
    for (; todo; todo &= todo - 1) {
      const int vec = first_vec + __builtin_ctzll(todo), node = vec / p.group;
      plain_node<D>(p, r, request, node, kvh * p.group + (vec - node * p.group), scratch);
    }
  }
}

int tree_params(TreeParams& p, const void* q, const void* key_pool, const void* value_pool,
                const int32_t* cached, const uint32_t* masks, const int32_t* tables, void* out,
                int64_t batch, int64_t nodes, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                int64_t page_size, int64_t max_pages, int64_t pool_pages, int64_t page_stride,
                int64_t head_stride) {
  TMC_REQUIRE(q && key_pool && value_pool && cached && masks && tables && out,
              "Tree attention: null device pointer.");
  TMC_REQUIRE(head_dim >= 8 && head_dim <= kPlainMaxDim && head_dim % 8 == 0,
              "Tree attention: head_dim must be a multiple of 8 up to 256.");
  TMC_REQUIRE(batch > 0 && batch < 65536 && nodes > 0 && nodes <= kTreeMost,
              "Tree attention: batch must be in [1, 65535] and nodes in [1, 256].");
  TMC_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads < 65536 && q_heads % kv_heads == 0,
              "Tree attention: invalid heads.");
  TMC_REQUIRE(page_size > 0 && max_pages > 0 && page_size < (1LL << 30) &&
                  max_pages < (1LL << 30) && page_size * max_pages < (1LL << 30) &&
                  pool_pages > 0 && pool_pages < (1LL << 31),
              "Tree attention: invalid page geometry.");
  TMC_REQUIRE(page_stride % 8 == 0 && head_stride % 8 == 0 && page_stride < (1LL << 40) &&
                  head_stride < (1LL << 40) && head_stride >= page_size * head_dim &&
                  page_stride >= (kv_heads - 1) * head_stride + page_size * head_dim,
              "Tree attention: strides must be multiples of 8 elements, the head stride hold a "
              "head's page rows and the page stride every kv head.");
  TMC_REQUIRE(aligned16(q) && aligned16(key_pool) && aligned16(value_pool) && aligned16(out),
              "Tree attention: q, K, V and out must be 16-byte aligned.");
  p = TreeParams{};
  p.q = static_cast<const half_t*>(q);
  p.k = static_cast<const half_t*>(key_pool);
  p.v = static_cast<const half_t*>(value_pool);
  p.out = static_cast<half_t*>(out);
  p.cached = cached;
  p.masks = masks;
  p.tables = tables;
  p.page_stride = (long)page_stride;
  p.head_stride = (long)head_stride;
  p.pool_pages = (int)pool_pages;
  p.batch = (int)batch;
  p.nodes = (int)nodes;
  p.words = (int)((nodes + 31) / 32);
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads);
  p.dim = (int)head_dim;
  p.page_size = (int)page_size;
  p.max_pages = (int)max_pages;
  p.divide = PageDivide::by(page_size);
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
  return 0;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

namespace tmc {
namespace {
// The shapes tree_attention_kernel takes; the others run tree_plain_kernel.
bool tree_shape(int64_t head_dim) { return head_dim == 64 || head_dim == 128; }

struct TreeLayout {
  int tiles, columns, parts;  // columns: tiles of 16 vectors a block holds
  int64_t units;
};
TreeLayout tree_layout(int64_t batch, int64_t nodes, int64_t q_heads, int64_t kv_heads,
                       int64_t capacity) {
  TreeLayout l{};
  const int64_t vectors = nodes * (q_heads / kv_heads), most = 16 * kTreeTiles;
  l.tiles = (int)((vectors + most - 1) / most);
  l.columns = (int)((vectors + 16 * l.tiles - 1) / (16 * l.tiles));
  l.units = batch * kv_heads * l.tiles;
  const int64_t steps = (capacity + kTreeStep - 1) / kTreeStep;
  l.parts = 1;
  if (l.units <= kTreeCus && steps > kTreeAlone)
    l.parts = (int)std::max<int64_t>(
        1, std::min((steps + kTreeLeast - 1) / kTreeLeast, (kTreeCus + l.units - 1) / l.units));
  return l;
}
}  // namespace
}  // namespace tmc

extern "C" size_t tmc_tree_attention_workspace_bytes(int64_t batch, int64_t nodes, int64_t q_heads,
                                                     int64_t kv_heads, int64_t head_dim,
                                                     int64_t capacity) {
  if (batch <= 0 || batch >= 65536 || nodes <= 0 || nodes > kTreeMost || q_heads <= 0 ||
      q_heads >= 65536 || kv_heads <= 0 || q_heads % kv_heads || capacity <= 0 ||
      capacity >= (1LL << 30) || !tree_shape(head_dim))
    return 0;
  const TreeLayout l = tree_layout(batch, nodes, q_heads, kv_heads, capacity);
  return l.parts < 2 ? 0
                     : kCounterBytes + (size_t)l.units * l.parts * (16 * l.columns) *
                                           (head_dim + 2) * sizeof(float);
}

extern "C" int tmc_tree_attention(const void* q, const void* key_pool, const void* value_pool,
                                  const int32_t* cached_lengths, const uint32_t* masks,
                                  const int32_t* counts, const int32_t* block_tables,
                                  const int32_t* active_count, void* out, int dtype,
                                  int64_t batch, int64_t nodes, int64_t q_heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t page_size, int64_t max_pages,
                                  int64_t pool_pages, int64_t page_stride, int64_t head_stride,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  TMC_REQUIRE(dtype == TMC_F16, "Tree attention: the gfx950 kernel stores K/V in fp16.");
  TreeParams p;
  if (tree_params(p, q, key_pool, value_pool, cached_lengths, masks, block_tables, out, batch,
                  nodes, q_heads, kv_heads, head_dim, page_size, max_pages, pool_pages,
                  page_stride, head_stride))
    return 1;
  const size_t need = tmc_tree_attention_workspace_bytes(batch, nodes, q_heads, kv_heads, head_dim,
                                                         page_size * max_pages);
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "Tree attention: workspace is smaller than tmc_tree_attention_workspace_bytes() or "
              "not 16-byte aligned.");
  p.counts = counts;
  p.active = active_count;
  const hipStream_t s = as_stream(stream);
  const TreeLayout l = tree_layout(batch, nodes, q_heads, kv_heads, page_size * max_pages);
  const int64_t items = batch * kv_heads * l.parts;
  const int64_t blocks = (items + 7) / 8 * 8 * l.tiles;
  // 16-byte units of the pools are counted in 32 bits: below 64 GiB each
  if (!tree_shape(head_dim) || (uint64_t)pool_pages * (uint64_t)page_stride / 8 >= 0xFFFFFFFFull ||
      blocks >= (1LL << 31)) {
    hipLaunchKernelGGL(tree_plain_kernel, dim3((unsigned)(batch * nodes), (unsigned)q_heads),
                       dim3(kWave), 0, s, p);
    return check_launch("tree_plain_kernel");
  }
  TreePlan plan{};
  plan.parts = l.parts;
  plan.tiles = l.tiles;
  plan.items = (int)items;
  plan.per_step = (float)(kv_heads * l.tiles) / (float)kTreeCus;
  if (need) {
    plan.arrivals = static_cast<int*>(workspace);
    plan.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  }
#define TMC_TREE(DIM, COLUMNS)                                                              \
  case COLUMNS:                                                                             \
    hipLaunchKernelGGL((tree_attention_kernel<DIM, COLUMNS>), dim3((unsigned)blocks),       \
                       dim3(kTreeWaves * kWave), 0, s, p, plan);                            \
    break
#define TMC_TREE_COLUMNS(DIM) \
  switch (l.columns) {        \
    TMC_TREE(DIM, 1);         \
    TMC_TREE(DIM, 2);         \
    TMC_TREE(DIM, 3);         \
    default:                  \
    TMC_TREE(DIM, 4);         \
  }
  if (head_dim == 128) {
    TMC_TREE_COLUMNS(128)
  } else {
    TMC_TREE_COLUMNS(64)
  }
#undef TMC_TREE_COLUMNS
#undef TMC_TREE
  return check_launch("tree_attention_kernel");
}
