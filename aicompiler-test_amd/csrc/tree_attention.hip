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

// A value that the compiler knows nothing of: what follows from it is computed where it is
// used, not kept in registers around the loops before.
__device__ __forceinline__ unsigned opaque(unsigned v) {
  asm volatile("" : "+v"(v));
  return v;
}

// ------------------------------------------------------------ any geometry
// One wave per (node, query head): 64 positions at a time, one per lane for the
// scores (whole K rows in 16-byte chunks), then lanes over the dims for P V.  Every node
// reads all of K and V: 8 requests of up to 2000 positions with 24 nodes, 32 heads and
// head dim 96 543 us, where the kernels below take 28 us for head dim 128.
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
  const int lane = (int)opaque(threadIdx.x) & (kWave - 1);
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

// ------------------------------------------------------------ few vectors
// D = 64 and 128.  A unit is a (request, kv head) with up to 32 of its query
// vectors (nodes x query heads of that kv head, in C tiles of 16); a step is 32 of
// its positions.  A unit's steps are a block's, or shared by several; the last of
// these to arrive joins their partials, in block order.
//
// The block's waves take the steps of a share in turn, each over a ring of two
// (D = 128) or four steps in LDS that only it touches, filled by 16-byte loads straight to
// LDS: no barrier, no register holds a load in flight, and a stage is loaded again as soon
// as its operands are in registers.  K and V rows lie in LDS as in their pages,
// 16-byte chunks (K) and 32-byte units (V) swizzled by the row so that the operand
// reads spread over the banks.  A position that does not exist reads a zero row.
// Scores S^T = K Q^T leave lane (vector j, group g) with positions 4g .. 4g+3 of
// both halves of the step, the order in which O^T = V^T P^T wants its weights; V^T
// comes from transposing LDS reads.  K and V are read from LDS once for all C
// tiles.
//
// Only steps that reach into the tree look at masks, 32 bits of a node's for the 32
// positions.
//
// Bound by the loads of K and V: 32 requests of 2048 positions with 8 nodes, 8 K/V heads of
// 128 dims and 32 vectors each 56 us, 4.8 TB/s; 16 requests of 65 to 4096 positions with
// 16 and 32 vectors 37 and 42 us (26 of loads at the rate of a large copy, the rest
// beginnings and joins).  One request of 300: 11 us of latencies, with one vector a
// head 8.
constexpr int kTreeStep = 32, kTreeWaves = 4;
constexpr int kTreeCus = 256;     // of an MI355X
constexpr int kTreePieces = 512;  // of a unit, at most
constexpr int kTreeSurvey = 256;  // requests of a batch whose steps are shared out

struct TreePlan {
  float* slots;   // [2 blocks][tiles][vectors][D + 4]
  int* arrivals;  // [units], kCounterStride apart; null: tree_join_kernel joins
  int tiles, blocks;  // blocks a tile
  int split;          // steps are shared out evenly; else a block takes whole units
  int least, alone;   // steps of a block, at least, and of requests that are not split
  int lead;           // steps that beginning a unit takes as long as
};

// Weights are stored 2^kRaise times their value in fp16 and a new maximum moves
// their scale only when it is kLag above the one in use, so a wave seldom rescales
// its sums: weights are at most 2^(kRaise + kLag) and keep 11 bits down to 2^-24 of
// that scale.  fp16 is what the matrix cores multiply with V's type; the sum takes
// the rounded weights, so an output is off by up to 2^-11 of the mean of |v| for it,
// beside the 2^-11 of its own fp16.
constexpr float kLag = 5.0f, kRaise = 10.0f;
constexpr unsigned kNoUnit = 0xFFFFFFFFu;

// The operands of one step of 32 positions, D = 128, out of LDS, waits included (D = 64:
// read_keys, read_values).
__device__ __forceinline__ void read_step_keys(const unsigned (&at)[4], unsigned page_at,
                                               h8 (&k)[2][4], int& page) {
  asm volatile(
      "ds_read_b32 %8, %13\n\t"
      "ds_read_b128 %0, %9\n\tds_read_b128 %1, %10\n\tds_read_b128 %2, %11\n\t"
      "ds_read_b128 %3, %12\n\t"
      "ds_read_b128 %4, %9 offset:4096\n\tds_read_b128 %5, %10 offset:4096\n\t"
      "ds_read_b128 %6, %11 offset:4096\n\tds_read_b128 %7, %12 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]),
        "=&v"(k[1][1]), "=&v"(k[1][2]), "=&v"(k[1][3]), "=&v"(page)
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(page_at)
      : "memory");
}
__device__ __forceinline__ void read_step_values(const unsigned (&at)[8], h4 (&v)[2][8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %17\n\t"
      "ds_read_b64_tr_b16 %2, %18\n\tds_read_b64_tr_b16 %3, %19\n\t"
      "ds_read_b64_tr_b16 %4, %20\n\tds_read_b64_tr_b16 %5, %21\n\t"
      "ds_read_b64_tr_b16 %6, %22\n\tds_read_b64_tr_b16 %7, %23\n\t"
      "ds_read_b64_tr_b16 %8, %16 offset:4096\n\tds_read_b64_tr_b16 %9, %17 offset:4096\n\t"
      "ds_read_b64_tr_b16 %10, %18 offset:4096\n\tds_read_b64_tr_b16 %11, %19 offset:4096\n\t"
      "ds_read_b64_tr_b16 %12, %20 offset:4096\n\tds_read_b64_tr_b16 %13, %21 offset:4096\n\t"
      "ds_read_b64_tr_b16 %14, %22 offset:4096\n\tds_read_b64_tr_b16 %15, %23 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[0][4]),
        "=&v"(v[0][5]), "=&v"(v[0][6]), "=&v"(v[0][7]), "=&v"(v[1][0]), "=&v"(v[1][1]),
        "=&v"(v[1][2]), "=&v"(v[1][3]), "=&v"(v[1][4]), "=&v"(v[1][5]), "=&v"(v[1][6]),
        "=&v"(v[1][7])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
        "v"(at[7])
      : "memory");
}

// The products of N tiles, see settle(): one wait for all.
template <int N> __device__ __forceinline__ void settle_all(f4 (&sc)[N]) {
  static_assert(N == 2 || N == 4, "the operands of one instruction");
  if constexpr (N == 2)
    asm volatile("s_nop 15" : "+v"(sc[0]), "+v"(sc[1]));
  else
    asm volatile("s_nop 15" : "+v"(sc[0]), "+v"(sc[1]), "+v"(sc[2]), "+v"(sc[3]));
}

// Bits [from, from + 32) of a node's mask: ones before the tree, zeros behind it.
// (Words that do not exist read one that does: no branch before a load.)
__device__ __forceinline__ unsigned mask_window(const uint32_t* mask, int count, int from) {
  const int w = from >> 5, last = (count - 1) >> 5, shift = from & 31;
  auto word = [&](unsigned x, int w) -> unsigned {
    const int left = count - 32 * w;
    const unsigned some = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u;
    return w < 0 ? ~0u : x & some;
  };
  const unsigned a = mask[max(0, min(w, last))], b = mask[max(0, min(w + 1, last))];
  const unsigned low = word(a, w), high = word(b, w + 1);
  return shift ? low >> shift | high << (32 - shift) : low;
}
__device__ __forceinline__ bool sees_nothing(const TreeParams& p, const Request& request,
                                             const uint32_t* mask) {
  unsigned any = request.cached > 0;
  for (int w = 0; 32 * w < request.count; ++w) any |= mask_window(mask, request.count, 32 * w);
  return any == 0;
}
template <int STEP> __device__ __forceinline__ int steps_of(const Request& r) {
  return r.count > 0 ? (r.cached + r.count + STEP - 1) / STEP : 0;
}

// What a block does next: steps [first, last) of one unit for `vecs` query vectors from
// first_vec on.  A unit whose steps are not all one block's is in pieces, each with a
// slot of the workspace: slot 2 b is of a piece that block b begins with, 2 b + 1 of
// the one that it ends with.
struct Part {
  Request request;
  int r, kvh, unit, tile, first_vec, vecs, steps, first, last;
  int pieces, piece, first_block, first_slot;
  __device__ __forceinline__ int slot(int piece) const {
    return piece == 0 ? first_slot : 2 * (first_block + piece);
  }
};

// The steps of all (request, kv head) pairs, request by request, cut into even runs of
// `chunk`, one a block (of each tile): every block has as much to do, however
// unlike the lengths.  A pair counts plan.lead steps more, before its own, for what it
// takes to begin and end it (a block with many short requests took 2.4 times as long
// as the others without).  With plan.split 0, or where no request has more than plan.alone
// steps, blocks take whole units, one after the other.
struct SurveySpace {
  int ends[kTreeSurvey];
  Request request[kTreeSurvey];
};
// Pieces whose factors fit a space of so many bytes, see join().
template <int COUNT> constexpr int pieces_in(size_t bytes) {
  return (int)(bytes / (COUNT * sizeof(float2)));
}
template <int NV, int STEP> struct Survey {
  const TreeParams& p;
  const TreePlan& plan;
  int* s_ends;         // [kTreeSurvey] in LDS: end of each request's run
  Request* s_request;  // [kTreeSurvey]
  int chunk;           // 0: whole units
  int total;

  // No unit is in more than `pieces` pieces.  (Every wave writes the same values to LDS.)
  __device__ __forceinline__ Survey(const TreeParams& p_, const TreePlan& plan_, SurveySpace& s,
                                    int pieces)
      : p(p_), plan(plan_), s_ends(s.ends), s_request(s.request), chunk(0),
        total(p_.batch * p_.kv_heads) {
    if (!plan.split) return;
    const int lane = threadIdx.x & (kWave - 1);
    int sum = 0, most = 0;
    for (int r0 = 0; r0 < p.batch; r0 += kWave) {
      const int r = r0 + lane;
      const Request request = request_of(p, min(r, p.batch - 1));
      const int steps = r < p.batch ? steps_of<STEP>(request) : 0;
      most = max(most, steps);
      int run = steps ? (steps + plan.lead) * p.kv_heads : 0;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const int other = __shfl_up(run, off, kWave);
        if (lane >= off) run += other;
      }
      s_ends[r] = sum + run;
      s_request[r] = request;
      sum += __builtin_amdgcn_readlane(run, kWave - 1);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) most = max(most, __shfl_xor(most, off, kWave));
    most = __builtin_amdgcn_readfirstlane(most);
    if (most <= plan.alone) return;
    total = sum;
    // (a unit of n steps is in up to n / chunk rounded up and one more)
    chunk = max(max(plan.least, (sum + plan.blocks - 1) / plan.blocks),
                (most + pieces - 2) / (pieces - 1));
  }
  __device__ __forceinline__ int begin(int block) const { return chunk ? block * chunk : block; }
  __device__ __forceinline__ int end(int block) const {
    return chunk ? min(total, (block + 1) * chunk) : total;
  }
  // The unit at `at`, a step of the pairs or a pair; its steps from there on, up to `to`
  // (none where that is in its lead).  Returns where the next one begins.
  __device__ __forceinline__ int part(Part& part, int at, int to) const {
    int before = 0;
    if (chunk) {
      const int lane = threadIdx.x & (kWave - 1);
      int r = 0;
      for (int r0 = 0; r0 < p.batch; r0 += kWave)
        r += __builtin_popcountll(
            __builtin_amdgcn_ballot_w64(r0 + lane < p.batch && s_ends[r0 + lane] <= at));
      part.r = r;
      before = __builtin_amdgcn_readfirstlane(r ? s_ends[r - 1] : 0);
      part.request = Request{__builtin_amdgcn_readfirstlane(s_request[r].cached),
                             __builtin_amdgcn_readfirstlane(s_request[r].count)};
    } else {
      part.r = at / p.kv_heads;
      part.request = request_of(p, part.r);
    }
    part.steps = steps_of<STEP>(part.request);
    part.first = 0;
    part.last = part.steps;
    part.pieces = 1;
    part.piece = part.first_block = part.first_slot = 0;
    int next = at + plan.blocks;
    part.kvh = at - part.r * p.kv_heads;
    if (chunk) {
      const int pair = part.steps + plan.lead;
      part.kvh = (at - before) / pair;
      const int begins = before + part.kvh * pair + plan.lead;  // of its own steps
      next = min(to, begins + part.steps);
      part.first = max(0, at - begins);
      part.last = next - begins;
      part.first_block = begins / chunk;
      part.pieces = (begins + part.steps - 1) / chunk - part.first_block + 1;
      part.piece = max(at, begins) / chunk - part.first_block;
      part.first_slot = 2 * part.first_block + (begins != part.first_block * chunk);
    }
    part.unit = (part.r * p.kv_heads + part.kvh) * plan.tiles + part.tile;
    part.first_vec = part.tile * NV;
    part.vecs = min(NV, part.request.count * p.group - part.first_vec);
    return next;
  }
};

// Blocks of the same steps, one a tile, on one XCD, whose L2 then holds their pages.
__device__ __forceinline__ int block_of(const TreePlan& plan, int& tile) {
  const int rest = blockIdx.x / 8;
  tile = rest % plan.tiles;
  return rest / plan.tiles * 8 + blockIdx.x % 8;
}

// Where the outputs of a block's vectors begin and their greatest score.
constexpr long kNowhere = -1;  // of a request to be left alone
template <int NV> struct Outputs {
  long at[NV];  // -2 less that for a node that sees nothing: zeros
  float top[NV];
};
template <int D>
__device__ __forceinline__ long output_of(const TreeParams& p, const Part& at, int vec, float top) {
  const int node = (at.first_vec + vec) / p.group;
  const size_t row = (size_t)at.r * p.nodes + node;
  const long to =
      (long)((row * p.q_heads + at.kvh * p.group + (at.first_vec + vec - node * p.group)) * D);
  return top == -INFINITY && sees_nothing(p, at.request, p.masks + row * p.words) ? -2 - to : to;
}
// Four dims of an output; whether the vector is to be done again, see redo().
__device__ __forceinline__ bool put(const TreeParams& p, long at, float top, int d, f4 x) {
  if (at == kNowhere) return false;
  if (at < 0) {
    at = -2 - at;
    x = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  *reinterpret_cast<h4*>(p.out + at + d) =
      h4{(half_t)x[0], (half_t)x[1], (half_t)x[2], (half_t)x[3]};
  return (!(x[0] == x[0]) | !(x[1] == x[1]) | !(x[2] == x[2]) | !(x[3] == x[3])) && finite(top);
}

// A slot holds the sums of NV vectors [D], each with its maximum and sum of weights
// behind.
template <int D> constexpr int slot_row() { return D + 4; }
template <bool AGENT> __device__ __forceinline__ f4 load_four(const float* from) {
  if constexpr (!AGENT) return *reinterpret_cast<const f4*>(from);
  const float2 a = load_pair(from), b = load_pair(from + 2);
  return f4{a.x, a.y, b.x, b.y};
}

// `count` vectors of a unit from first_vec on, out of its pieces, joined in their order,
// by all threads.  First the pieces' maxima and sums of weights, LANES threads a
// vector, which leave each piece's factor in LDS; then four dims a thread.  AGENT: the
// slots were written in this launch.  The bits of redo().
template <int D, int NV, int COUNT, int THREADS, bool AGENT>
__device__ __forceinline__ unsigned join(const TreeParams& p, const TreePlan& plan, const Part& at,
                                         int first_vec, int count, char* s_space,
                                         Outputs<COUNT>& s_outputs) {
  const int thread = (int)opaque(threadIdx.x);
  constexpr int ROW = slot_row<D>();
  constexpr int LANES = THREADS / COUNT < kWave ? THREADS / COUNT : kWave;
  float2* s_factor = reinterpret_cast<float2*>(s_space);  // [pieces][COUNT]: (maximum, sum)
  auto slot = [&](int piece) {
    return plan.slots + (((size_t)at.slot(piece) * plan.tiles + at.tile) * NV + first_vec) * ROW;
  };
  {
    const int vec = thread / LANES, lane = thread % LANES;
    float top = -INFINITY, sum = 0.0f;
    if (vec < count) {
      for (int b = lane; b < at.pieces; b += LANES) {
        const float* from = slot(b) + (size_t)vec * ROW + D;
        const float2 y = AGENT ? load_pair(from) : *reinterpret_cast<const float2*>(from);
        s_factor[b * COUNT + vec] = y;
        top = fmaxf(top, y.x);
      }
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
      bool spoiled = false;
      for (int b = lane; b < at.pieces; b += LANES) {
        const float2 y = s_factor[b * COUNT + vec];
        spoiled |= y.y < 0.0f;
        const float scale = y.x == -INFINITY ? 0.0f : fast_exp2(y.x - top);
        sum += y.y * scale;
        s_factor[b * COUNT + vec].x = scale;
      }
      if (spoiled) sum = -1.0f;
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) {
        const float other = __shfl_xor(sum, off, kWave);
        sum = sum < 0.0f || other < 0.0f ? -1.0f : sum + other;
      }
      const float whole = 1.0f / sum;
      for (int b = lane; b < at.pieces; b += LANES) s_factor[b * COUNT + vec].x *= whole;
      if (lane == 0) {
        s_outputs.at[vec] = sum < 0.0f ? kNowhere : output_of<D>(p, at, first_vec + vec, top);
        s_outputs.top[vec] = top;
      }
    }
  }
  __syncthreads();
  unsigned again = 0, bit = 1;
  constexpr int kTurns = COUNT * (D / 4) > THREADS ? 2 : 1, kAhead = kTurns > 1 ? 4 : 12;
  const int items = count * (D / 4);
  for (int i = thread; i < items; i += kTurns * THREADS, bit <<= kTurns) {
    f4 val[kTurns] = {};
    for (int b = 0; b < at.pieces; b += kAhead) {
      f4 x[kTurns][kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float* from = slot(min(b + u, at.pieces - 1));
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
          const int place = min(i + t * THREADS, items - 1);
          x[t][u] = load_four<AGENT>(from + (size_t)(place / (D / 4)) * ROW + place % (D / 4) * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (b + u < at.pieces)
#pragma unroll
          for (int t = 0; t < kTurns; ++t)
            val[t] += s_factor[(b + u) * COUNT + min(i + t * THREADS, items - 1) / (D / 4)].x *
                      x[t][u];
    }
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int place = i + t * THREADS, vec = place / (D / 4);
      if (place < items && put(p, s_outputs.at[vec], s_outputs.top[vec], place % (D / 4) * 4, val[t]))
        again |= bit << t;
    }
  }
  return again;
}

// A weight of 0 times an infinity or NaN of V that the node does not see (another one of
// the tile does), a weight that fp16 rounds to 0 times an infinity, and weights past
// its range (scores of 2^24 and more, whose fp32 maximum is several powers of two
// off) give a NaN that weights of fp32 over a node's own positions do not: such
// vectors are done again with those, one at a time, by the wave that put them.  Bit t
// of `again`: this thread's dims of vector first + (t * THREADS + thread) / (D / 4).
template <int D, int THREADS>
__device__ __forceinline__ void redo(const TreeParams& p, const Part& at, unsigned again, int first,
                                     char* s_space) {
  const int thread = (int)opaque(threadIdx.x);
  if (__syncthreads_or(again != 0)) {
    PlainScratch& scratch = reinterpret_cast<PlainScratch*>(s_space)[thread / kWave];
    __builtin_amdgcn_s_waitcnt(0);  // the NaNs are stored
    constexpr int SIDE = D / 4;     // lanes of a vector
    static_assert(SIDE < kWave, "a vector is a wave's");
    first += (thread & ~(kWave - 1)) / SIDE;
    for (int turn = 0; turn < 32; ++turn) {
      const unsigned long long lanes = __builtin_amdgcn_ballot_w64(again >> turn & 1);
      if (lanes == 0) continue;
      for (int side = 0; side < kWave / SIDE; ++side) {
        if (!(lanes >> (side * SIDE) & ((1ull << SIDE) - 1))) continue;
        const int vec = at.first_vec + first + turn * (THREADS / SIDE) + side, node = vec / p.group;
        plain_node<D>(p, at.r, at.request, node, at.kvh * p.group + (vec - node * p.group), scratch);
      }
    }
  }
}

// GROUPS partial results of NV vectors lie in LDS: sums [GROUPS][NV][D + 4], maxima and
// sums of weights [GROUPS][NV].  They are joined and stored as outputs, or in the
// piece's slot; with arrival counters the last of a unit's pieces joins them all.
template <int D, int NV, int GROUPS, int THREADS>
__device__ __forceinline__ void finish(const TreeParams& p, const TreePlan& plan, const Part& at,
                                       char* s_space, float* s_max, const float* s_sum, int bad) {
  const int thread = (int)opaque(threadIdx.x);
  constexpr int ROW = slot_row<D>();
  static_assert(NV <= THREADS && NV * (D / 4) / THREADS <= 32, "a thread a vector, a bit a turn");
  static_assert(sizeof(PlainScratch) * (THREADS / kWave) <= NV * ROW * 4 * GROUPS,
                "a scratch for every wave");
  __shared__ Outputs<NV> s_outputs;
  __shared__ int s_last;
  const float* s_out = reinterpret_cast<const float*>(s_space);
  const bool whole = at.pieces == 1;
  float* slot = plan.slots + ((size_t)at.slot(at.piece) * plan.tiles + at.tile) * NV * ROW;
  if (thread < at.vecs) {
    const int vec = thread;
    float top = -INFINITY, sum = 0.0f, scale[GROUPS];
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) top = fmaxf(top, s_max[w * NV + vec]);
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) {
      const float high = s_max[w * NV + vec];
      scale[w] = high == -INFINITY ? 0.0f : fast_exp2(high - top);
      sum += scale[w] * s_sum[w * NV + vec];
    }
    const float part = whole ? 1.0f / sum : 1.0f;
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) s_max[w * NV + vec] = scale[w] * part;  // the group's factor
    if (whole) {
      s_outputs.at[vec] = bad ? kNowhere : output_of<D>(p, at, vec, top);
      s_outputs.top[vec] = top;
    } else {
      float* to = slot + (size_t)vec * ROW + D;
      const float mass = bad ? -1.0f : sum;
      if (plan.arrivals) store_pair(to, top, mass);
      else *reinterpret_cast<float2*>(to) = float2{top, mass};
    }
  }
  __syncthreads();
  unsigned again = 0, bit = 1;
  for (int i = thread; i < at.vecs * (D / 4); i += THREADS, bit <<= 1) {
    const int vec = i / (D / 4), d = i % (D / 4) * 4;
    f4 val = {};
#pragma unroll
    for (int w = 0; w < GROUPS; ++w)
      val += s_max[w * NV + vec] *
             *reinterpret_cast<const f4*>(s_out + (size_t)(w * NV + vec) * ROW + d);
    float* to = slot + (size_t)vec * ROW + d;
    if (whole) {
      if (put(p, s_outputs.at[vec], s_outputs.top[vec], d, val)) again |= bit;
    } else if (plan.arrivals) {
      store_pair(to, val[0], val[1]);
      store_pair(to + 2, val[2], val[3]);
    } else {
      *reinterpret_cast<f4*>(to) = val;
    }
  }
  if (!whole) {
    if (!plan.arrivals) return;
    // every word is written and read at agent scope; the stores have completed before
    // the arrival is counted
    int* counter = plan.arrivals + at.unit * kCounterStride;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (thread == 0)
      s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               at.pieces - 1;
    __syncthreads();
    if (!s_last) return;
    if (thread == 0)
      __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    again = join<D, NV, NV, THREADS, true>(p, plan, at, 0, at.vecs, s_space, s_outputs);
    __syncthreads();
  }
  redo<D, THREADS>(p, at, again, 0, s_space);
}

template <int D, int C>
__global__ __launch_bounds__(kTreeWaves * kWave, 1) void tree_ring_kernel(
    TreeParams p, TreePlan plan) {
  constexpr int STEP = kTreeStep, STAGES = D == 128 ? 2 : 4, WAVES = kTreeWaves, NV = 16 * C;
  constexpr int KS = D / 32, DT = D / 16, CH = D / 8, TILES = STEP / 16;
  static_assert(TILES == 2, "a step is the depth of one product with V");
  constexpr int RPL = kWave / CH, LOADS = STEP / RPL;  // rows a load, loads of K (of V) a step
  constexpr int STAGE = 2 * STEP * D;                  // halves
  constexpr int THREADS = WAVES * kWave;
  constexpr int ROW = D + 4;                           // floats of a vector's sums in LDS
  constexpr int RING_BYTES = WAVES * STAGES * STAGE * 2, MET_BYTES = WAVES * NV * ROW * 4;
  __shared__ __align__(16) char s_space[RING_BYTES > MET_BYTES ? RING_BYTES : MET_BYTES];
  __shared__ int s_pages[WAVES * STAGES * kWave];
  __shared__ float s_max[WAVES * NV], s_sum[WAVES * NV];
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) const void global_void;

  __shared__ SurveySpace s_survey;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int j = lane & 15, g = lane >> 4;
  Part at;
  const int block = block_of(plan, at.tile);
  const Survey<NV, STEP> survey(p, plan, s_survey,
                                plan.arrivals ? pieces_in<NV>(sizeof(s_space)) : kTreePieces);
  const int end = survey.end(block);
  for (int next = survey.begin(block); next < end;) {
  next = survey.part(at, next, end);
  if (at.vecs <= 0 || at.last <= at.first) continue;
  const Request request = at.request;
  const int r = at.r, kvh = at.kvh, first_vec = at.first_vec, vecs = at.vecs;
  const int first_step = at.first, last_step = at.last;

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
  const int tree_step = request.cached / STEP;  // the first that reaches into the tree
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

  // Table entry of the position that lane l % STEP stands for in a step (past the end:
  // of the last one).
  auto position = [&](int step) { return min(step * STEP + (lane & (STEP - 1)), count - 1); };
  auto entry = [&](int step) { return table + p.divide(position(step)); };
  // 16-byte unit where that position's row starts, kNoUnit when it has none
  auto place = [&](int step, int page) -> unsigned {
    const bool ok = tree_page_ok(p, page);
    bad |= !ok;
    const int pos = position(step), slot_row = pos - p.divide(pos) * p.page_size;
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
    unsigned units[LOADS];  // (one wait for all)
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      units[i] = (unsigned)__builtin_amdgcn_ds_bpermute((RPL * i + lane / CH) * 4, (int)first);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int R = RPL * i + lane / CH, slot = lane % CH;
      const unsigned row_unit = units[i];
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
  auto consume = [&](auto masked, int step, const h8 (&k)[TILES][KS], const h4 (&v)[TILES][DT]) {
    f4 sc[C * TILES];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        f4& to = sc[c * TILES + t];
        to = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
          to = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][s], qb[c][s], to, 0, 0, 0);
      }
    settle_all(sc);
    if constexpr (decltype(masked)::value) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const unsigned bits = mask_window(p.masks + (size_t)row[c] * p.words, request.count,
                                          step * STEP - request.cached) >> (4 * g);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(bits >> (16 * t + e) & 1)) sc[c * TILES + t][e] = -INFINITY;
      }
    }
    float top[C];
    bool grows = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      top[c] = -INFINITY;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const f4 x = sc[c * TILES + t];
        top[c] = fmaxf(top[c], fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
      }
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
    h4 w[C][TILES];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float shift = m[c] == -INFINITY ? 0.0f : m[c] - kRaise;
      const h2 ones = {(half_t)1.0f, (half_t)1.0f};
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[c][t][e] = (half_t)fast_exp2(__fmaf_rn(sc[c * TILES + t][e], p.scale_log2, -shift));
        const h4 x = w[c][t];
        lsum[c] = __builtin_amdgcn_fdot2(__builtin_shufflevector(x, x, 0, 1), ones, lsum[c], false);
        lsum[c] = __builtin_amdgcn_fdot2(__builtin_shufflevector(x, x, 2, 3), ones, lsum[c], false);
      }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c)
        o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            __builtin_shufflevector(v[0][t], v[1][t], 0, 1, 2, 3, 4, 5, 6, 7),
            __builtin_shufflevector(w[c][0], w[c][1], 0, 1, 2, 3, 4, 5, 6, 7), o[c][t], 0, 0, 0);
  };

  // ---- the wave's steps: every WAVES-th of the piece
  const int mine = first_step + wave;
  {
    int page[STAGES];
#pragma unroll
    for (int st = 0; st < STAGES; ++st) page[st] = *entry(mine + st * WAVES);
#pragma unroll
    for (int st = 0; st < STAGES; ++st)
      if (mine + st * WAVES < last_step)
        issue(place(mine + st * WAVES, page[st]), entry(mine + (STAGES + st) * WAVES), st);
  }
  constexpr int FLIGHT = 2 * LOADS + 1;  // loads of a step
  static_assert(STAGES == 2 || STAGES == 4, "the waits below");
  int stage = 0;
  for (int step = mine; step < last_step; step += WAVES, stage = (stage + 1) % STAGES) {
    // the step's own loads are the oldest of those in flight
    const int later = last_step - 1 - step;
    if (STAGES > 2 && later >= 3 * WAVES) wait_loads<STAGES == 2 ? 0 : 3 * FLIGHT>();
    else if (STAGES > 2 && later >= 2 * WAVES) wait_loads<STAGES == 2 ? 0 : 2 * FLIGHT>();
    else if (later >= WAVES) wait_loads<FLIGHT>();
    else wait_loads<0>();
    h8 k[TILES][KS];
    h4 v[TILES][DT];
    int page;
    unsigned keys[KS], values[DT];
#pragma unroll
    for (int s = 0; s < KS; ++s) keys[s] = key_at[s] + (unsigned)(stage * STAGE * 2);
#pragma unroll
    for (int t = 0; t < DT; ++t) values[t] = value_at[t] + (unsigned)(stage * STAGE * 2);
    if constexpr (D == 128) {
      read_step_keys(keys, page_at + (unsigned)(stage * kWave * 4), k, page);
      read_step_values(values, v);
    } else {
      read_keys<D, STEP, 0, 0>(keys, page_at + (unsigned)(stage * kWave * 4), k, page);
      read_values<D, STEP, 0>(values, v);
    }
    const int again = step + STAGES * WAVES;
    if (again < last_step) issue(place(again, page), entry(again + STAGES * WAVES), stage);
    if (step < tree_step)
      consume(std::false_type{}, step, k, v);
    else
      consume(std::true_type{}, step, k, v);
  }

  // ---- the waves meet in LDS (the rings: every load into them has landed)
  bad = __syncthreads_or(bad);
  float* s_out = reinterpret_cast<float*>(s_space);  // [waves][NV][ROW]
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float sum = cross_sum<16>(lsum[c]);
    if (g == 0) {
      s_max[wave * NV + 16 * c + j] = m[c];
      s_sum[wave * NV + 16 * c + j] = sum;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<f4*>(s_out + (size_t)(wave * NV + 16 * c + j) * ROW + 16 * t + 4 * g) =
          o[c][t];
  }
  __syncthreads();
  finish<D, NV, WAVES, THREADS>(p, plan, at, s_space, s_max, s_sum, bad);
  __syncthreads();
  }
}

// ------------------------------------------------------------ many vectors
// D = 64 and 128.  A unit is a (request, kv head) with up to 32 VG of its query
// vectors; each wave holds 32 vectors on v_mfma_f32_32x32x16_f16, VG groups of
// vectors, and PG groups of waves take a stage's 32-position steps: S^T = K Q^T (32
// positions x 32 vectors) leaves lane (vector, half) with the positions 8 (r / 4) +
// 4 half + r % 4, the order in which O^T = V^T P^T takes its weights.  Two waves a
// SIMD: one's softmax runs beside the other's products.  K and V go through
// registers, loaded one stage ahead of the LDS one; one barrier a stage.
//
// 8 requests of 1000 to 8000 positions with 64 nodes and 32 K/V heads of 128 dims 137 us,
// 4.4 TB/s: the loads.  One of 100000 positions with 240 vectors for each of 8 K/V heads
// 150 us, 660 TFLOP/s of products (a large library product reaches 1300) at 2.7 TB/s:
// bound by the waves' issue, of which softmax has as much as the products.
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kWideSpan = 64;  // positions a stage

template <int D, int VG, int PG>
__global__ __launch_bounds__(VG * PG * kWave, 2) void tree_wide_kernel(TreeParams p, TreePlan plan) {
  constexpr int KS = D / 16, DT = D / 32, CH = D / 8;
  constexpr int WAVES = VG * PG, THREADS = WAVES * kWave, NV = 32 * VG;
  constexpr int SPAN = kWideSpan;
  static_assert(PG == 1 || SPAN == 32 * PG, "a step of every stage a group, or all");
  constexpr int OWN = SPAN / WAVES;                   // rows of a stage a wave loads
  constexpr int RPL = kWave / CH, LOADS = OWN / RPL;  // rows a load, loads of K (of V)
  constexpr int STAGE = 2 * SPAN * D;                 // halves: K rows, V rows
  constexpr int ROW = D + 4;
  constexpr int KV_BYTES = 2 * STAGE * 2, MET_BYTES = WAVES * 32 * ROW * 4;
  constexpr int PER = SPAN / kWave, TURNS = WAVES / PER;  // waves that find a stage's rows
  static_assert(LOADS >= 1, "a wave loads whole rows");
  __shared__ __align__(256) char s_space[KV_BYTES > MET_BYTES ? KV_BYTES : MET_BYTES];
  __shared__ unsigned s_units[4][SPAN];  // 16-byte units where the rows of four stages start
  __shared__ float s_max[PG * NV], s_sum[PG * NV];
  half_t* s_kv = reinterpret_cast<half_t*>(s_space);

  __shared__ SurveySpace s_survey;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  Part at;
  const int block = block_of(plan, at.tile);
  const Survey<NV, SPAN> survey(p, plan, s_survey,
                                plan.arrivals ? pieces_in<NV>(sizeof(s_space)) : kTreePieces);
  const int end = survey.end(block);
  for (int next = survey.begin(block); next < end;) {
  next = survey.part(at, next, end);
  if (at.vecs <= 0 || at.last <= at.first) continue;
  const Request request = at.request;
  const int vg = wave % VG, pg = wave / VG;
  const int col = lane & 31, half = lane >> 5;
  const unsigned head_unit = (unsigned)((size_t)at.kvh * p.head_stride / 8);
  const int32_t* table = p.tables + (size_t)at.r * p.max_pages;
  const int count = request.cached + request.count;  // positions
  const int first = at.first, stages = at.last - at.first;
  // this lane's vector
  const bool busy = 32 * vg < at.vecs;
  const int vec = at.first_vec + min(32 * vg + col, at.vecs - 1), node = vec / p.group;
  const int row = at.r * p.nodes + node;
  const uint32_t* mask = p.masks + (size_t)row * p.words;
  h8 qb[KS];
  {
    const half_t* q = p.q + ((size_t)row * p.q_heads + at.kvh * p.group + (vec - node * p.group)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = load_h8(q + 16 * s + 8 * half);
  }

  // ---- loads.  The waves take turns to find a stage's rows: their table entries
  // four stages ahead, their units three ahead.  Places past the end take the last
  // position's row and positions without a page page 0's: such scores are masked, or
  // their request not stored.
  int bad = 0, page = 0, slot_row = 0;
  auto my_turn = [&](int stage) { return stage % TURNS == wave / PER; };
  const int turn_row = wave % PER * kWave + lane;
  auto look_up = [&](int stage) {
    const int pos = min((first + stage) * SPAN + turn_row, count - 1);
    const int index = p.divide(pos);
    slot_row = pos - index * p.page_size;
    page = table[index];
  };
  auto put_units = [&](int stage) {
    const bool ok = tree_page_ok(p, page);
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
  auto load = [&](int stage, h8 (&kr)[LOADS], h8 (&vr)[LOADS]) {
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
      const int to = (OWN * wave + RPL * i) * D + 8 * lane;
      *reinterpret_cast<h8*>(buf + to) = kr[i];
      *reinterpret_cast<h8*>(buf + SPAN * D + to) = vr[i];
    }
  };
#pragma unroll
  for (int stage = 0; stage < 4; ++stage)
    if (my_turn(stage)) {
      look_up(stage);
      if (stage < 3) put_units(stage);
    }
  __syncthreads();
  load(0, kr, vr);
  {
    h8 kn[LOADS], vn[LOADS];  // both first stages in flight at once
    load(1, kn, vn);
    store(s_kv);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      kr[i] = kn[i];
      vr[i] = vn[i];
    }
  }

  f16v o[DT];
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;

  // ---- one step of 32 positions: rows R0 ... of a stage.  V's operands are read before
  // the weights are computed (the fences keep the reads there), into the registers
  // that K's have left.  Rows start at multiples of 128 bytes, so the swizzled chunk
  // is an exclusive or on the address; the addresses are rebuilt in every step
  // (opaque()), not kept in registers that the step has no room for.
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
    const unsigned from = opaque(key_at) + buf + (unsigned)(R0 * D * 2);
#pragma unroll
    for (int s = 0; s < KS; ++s) k[s] = *(lds_h8*)(uintptr_t)(from ^ (unsigned)(s << 5));
  };
  auto read_values = [&](unsigned buf, int R0) {
    const unsigned from = opaque(value_at) + buf + (unsigned)(R0 * D * 2);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        h4 part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          part[h] = __builtin_bit_cast(
              h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4*)(uintptr_t)(
                      (from ^ (unsigned)(t << 6)) + (unsigned)((16 * c + 8 * h) * D * 2))));
        va[c][t] = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
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
  auto weigh = [&](int from) {  // of positions from ... from + 31
    settle(sc);
    if (from + 32 > request.cached) {
      const unsigned sees =
          mask_window(mask, request.count, from - request.cached) >> (4 * half);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(sees >> (8 * (e >> 2) + (e & 3)) & 1)) sc[e] = -INFINITY;
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
    const float shift = m == -INFINITY ? 0.0f : m - kRaise;
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
  for (int i = 0; i < stages; ++i) {
    const unsigned buf = (unsigned)((i & 1) * STAGE * 2);
    // stage i and the units of stage i + 2 are in LDS, stage i - 1 has been read
    lds_barrier();
    store(s_kv + ((i + 1) & 1) * STAGE);
    load(i + 2, kr, vr);
    if (my_turn(i + 3)) put_units(i + 3);
    if (my_turn(i + 4)) look_up(i + 4);
#pragma unroll
    for (int s = 0; s < (PG > 1 ? 1 : 2); ++s) {
      const int R0 = PG > 1 ? 32 * pg : 32 * s, from = (first + i) * SPAN + R0;
      if (from >= count || !busy) continue;
      read_keys(buf, R0);
      __builtin_amdgcn_sched_barrier(0);
      scores();
      __builtin_amdgcn_sched_barrier(0);
      read_values(buf, R0);
      __builtin_amdgcn_sched_barrier(0);
      weigh(from);
      add_values();
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // ---- the waves meet in LDS
  bad = __syncthreads_or(bad);
  sum += __shfl_xor(sum, 32, kWave);
  const int place = wave * 32 + col;  // group pg of vector 32 vg + col
  if (half == 0) {
    s_max[place] = m;
    s_sum[place] = sum;
  }
  float* s_out = reinterpret_cast<float*>(s_space) + (size_t)place * ROW;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<f4*>(s_out + 32 * t + 8 * e + 4 * half) =
          f4{o[t][4 * e], o[t][4 * e + 1], o[t][4 * e + 2], o[t][4 * e + 3]};
  __syncthreads();
  finish<D, NV, PG, THREADS>(p, plan, at, s_space, s_max, s_sum, bad);
  __syncthreads();
  }
}

// The units of tree_wide_kernel that are in pieces, kJoinThreads / (D / 4) vectors a
// block.
constexpr int kJoinThreads = 256;
template <int D, int NV>
__global__ __launch_bounds__(kJoinThreads) void tree_join_kernel(TreeParams p, TreePlan plan) {
  constexpr int VECS = kJoinThreads / (D / 4), GROUPS = NV / VECS;
  constexpr int SPACE = kTreePieces * VECS * (int)sizeof(float2);
  static_assert(pieces_in<VECS>(SPACE) == kTreePieces, "every piece's factor has its place");
  static_assert(sizeof(PlainScratch) * (kJoinThreads / kWave) <= SPACE, "a scratch for every wave");
  __shared__ __align__(16) char s_space[SPACE];
  __shared__ Outputs<VECS> s_outputs;
  __shared__ SurveySpace s_survey;
  Part at;
  const int group = blockIdx.x % GROUPS, rest = blockIdx.x / GROUPS;
  at.tile = rest % plan.tiles;
  const int pair = rest / plan.tiles, r = pair / p.kv_heads;
  const Survey<NV, kWideSpan> survey(p, plan, s_survey, kTreePieces);
  const int steps = steps_of<kWideSpan>(request_of(p, r));
  if (survey.chunk == 0 || steps == 0) return;
  const int begins = (r ? s_survey.ends[r - 1] : 0) + (pair - r * p.kv_heads) * (steps + plan.lead);
  survey.part(at, __builtin_amdgcn_readfirstlane(begins), survey.total);
  if (at.pieces < 2 || group * VECS >= at.vecs) return;
  const unsigned again = join<D, NV, VECS, kJoinThreads, false>(
      p, plan, at, group * VECS, min(VECS, at.vecs - group * VECS), s_space, s_outputs);
  __syncthreads();
  redo<D, kJoinThreads>(p, at, again, group * VECS, s_space);
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
// The shapes tree_ring_kernel and tree_wide_kernel take; the others run tree_plain_kernel.
bool tree_shape(int64_t head_dim) { return head_dim == 64 || head_dim == 128; }

// The tiles whose pieces tree_join_kernel joins; of the others a unit's last block does.
bool has_join(int64_t head_dim, int vectors) {
  return vectors == 64 || (vectors == 256 && head_dim == 128);
}

// How a launch is shared out: query vectors a block, tiles of so many of a (request,
// kv head), blocks a tile, and whether steps are shared out.
struct TreeLayout {
  int vectors, tiles, blocks, least, alone, lead;
  bool split, arrivals;  // arrivals: the last piece of a unit joins them
};
TreeLayout tree_layout(int64_t batch, int64_t nodes, int64_t q_heads, int64_t kv_heads,
                       int64_t head_dim, int64_t capacity) {
  TreeLayout l{};
  const int64_t vectors = nodes * (q_heads / kv_heads), pairs = batch * kv_heads;
  int resident;  // blocks that share the steps
  // Sharing costs some 10 us of lookups and joins: requests up to `alone` steps go whole, up
  // to so many positions that half the CUs take as long.  Whole and shared: 4 requests of 400
  // positions with 32 vectors 12.6 and 15.6 us, of 1400 23.5 and 19.1; 24 requests 16.5 and
  // 27.6, 33.2 and 42.1; with 256 vectors 4 of 1400 54 and 32, 24 of 1400 62 and 94
  // (but 16 of 1400, which go whole, 59 and 51).
  const bool many = pairs >= kTreeCus / 2;
  if (vectors <= 32) {
    l.vectors = vectors <= 16 ? 16 : 32;
    l.least = 8;
    l.alone = many ? 48 : 20;
    l.lead = 12;
    resident = kTreeCus;
  } else {
    // Shared out, a block's partials cost as much as some steps, and tiles of 64 vectors have
    // the fewest.  For head dim 128 and much to read, one tile of up to 256 vectors reads K
    // and V once: 4 requests of 1400 and 8000 positions with 256 vectors 32 and 64 us, in
    // tiles of 64 32 and 79; 12 of up to 3000 65 and 62; one of 100000 with 240 153 and 195
    // (but 4 of 1400 with 256 vectors for each of 32 K/V heads 81 and 59).
    // Head dim 64 has half the work a vector: 16 requests of up to 4096 with 256 vectors 52
    // us in tiles of 64, 55 in one of 256; one of 100000 113 and 146.
    // One tile of 64 on one block a CU: 16 requests of up to 4096 with 64 vectors 47 us, on two
    // 48; 24 of up to 2000 with head dim 64 25 and 30.
    const bool one = vectors <= 64;
    l.vectors = one || head_dim == 64 || pairs * ((capacity + kWideSpan - 1) / kWideSpan) <= 12 * kTreeCus
                    ? 64 : 256;
    l.least = 4;
    l.alone = !many ? (one ? 9 : 7) : one || head_dim == 128 ? 24 : 16;
    l.lead = 8;
    resident = one || l.vectors == 256 ? kTreeCus : 2 * kTreeCus;
  }
  const auto share = [&]() {
    const int step = l.vectors <= 32 ? kTreeStep : kWideSpan;
    const int64_t steps = (capacity + step - 1) / step;
    l.tiles = (int)((vectors + l.vectors - 1) / l.vectors);
    return batch <= kTreeSurvey && pairs * l.tiles <= kSharedRows && steps > l.alone &&
           pairs * (steps + l.lead) < (1LL << 30);
  };
  l.split = share();
  if (vectors > 64 && (!l.split || pairs >= 2 * kTreeCus)) {
    // mostly whole units: wide blocks do the same work in less time, but not on vectors that
    // are not there (64 requests of 1000 positions with 128 vectors: tiles of 64 85 us, of
    // 128 69, of 256 82; with 256 vectors 152, 124 and 117)
    const int64_t cost64 = (vectors + 63) / 64 * 64 * 7, cost128 = (vectors + 127) / 128 * 128 * 6,
                  cost256 = (vectors + 255) / 256 * 256 * 5;
    l.vectors = cost64 < std::min(cost128, cost256) ? 64 : cost128 < cost256 ? 128 : 256;
    resident = l.vectors == 256 && head_dim == 128 ? kTreeCus : 2 * kTreeCus;
    l.split = share();
  }
  // a multiple of the XCDs, no more than are resident
  l.blocks = (int)(l.split ? std::max(resident / l.tiles / 8 * 8, 8) : (pairs + 7) / 8 * 8);
  // A unit's last block joins two pieces sooner than another launch does, but not more (8
  // requests of 8000 positions with 256 vectors 135 and 115 us, 16 of them 205 and 207).
  // Tiles of 128, and of 256 for head dim 64, are for many pairs or many tiles, and have no
  // other launch, nor have those of up to 32.
  l.arrivals = !has_join(head_dim, l.vectors) || l.blocks <= 2 * pairs;
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
  const TreeLayout l = tree_layout(batch, nodes, q_heads, kv_heads, head_dim, capacity);
  return l.split ? kCounterBytes + (size_t)2 * l.blocks * l.tiles * l.vectors * (head_dim + 4) *
                                       sizeof(float)
                 : 0;
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
  const TreeLayout l =
      tree_layout(batch, nodes, q_heads, kv_heads, head_dim, page_size * max_pages);
  TMC_REQUIRE(!l.split || l.arrivals || has_join(head_dim, l.vectors),
              "Tree attention: no kernel joins these tiles.");
  const int64_t blocks = (int64_t)l.blocks * l.tiles;
  // 16-byte units of the pools are counted in 32 bits: below 64 GiB each
  if (!tree_shape(head_dim) || (uint64_t)pool_pages * (uint64_t)page_stride / 8 >= 0xFFFFFFFFull ||
      batch * kv_heads >= (1LL << 30) || blocks >= (1LL << 31)) {
    hipLaunchKernelGGL(tree_plain_kernel, dim3((unsigned)(batch * nodes), (unsigned)q_heads),
                       dim3(kWave), 0, s, p);
    return check_launch("tree_plain_kernel");
  }
  TreePlan plan{};
  plan.tiles = l.tiles;
  plan.blocks = l.blocks;
  plan.split = l.split;
  plan.least = l.least;
  plan.alone = l.alone;
  plan.lead = l.lead;
  if (need) {
    if (l.arrivals) plan.arrivals = static_cast<int*>(workspace);
    plan.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  }
#define TMC_TREE_RING(DIM, C)                                                               \
  hipLaunchKernelGGL((tree_ring_kernel<DIM, C>), dim3((unsigned)blocks),                    \
                     dim3(kTreeWaves * kWave), 0, s, p, plan)
#define TMC_TREE_WIDE(DIM, VG, PG)                                               \
  hipLaunchKernelGGL((tree_wide_kernel<DIM, VG, PG>), dim3((unsigned)blocks),    \
                     dim3(VG * PG * kWave), 0, s, p, plan)
#define TMC_TREE_JOIN(DIM, NV)                                                   \
  hipLaunchKernelGGL((tree_join_kernel<DIM, NV>),                                \
                     dim3((unsigned)(batch * kv_heads * l.tiles * NV * (DIM / 4) / kJoinThreads)), \
                     dim3(kJoinThreads), 0, s, p, plan)
#define TMC_TREE_VECTORS(DIM)                        \
  if (l.vectors == 16) TMC_TREE_RING(DIM, 1);        \
  else if (l.vectors == 32) TMC_TREE_RING(DIM, 2);   \
  else if (l.vectors == 64) TMC_TREE_WIDE(DIM, 2, 2); \
  else if (l.vectors == 128) TMC_TREE_WIDE(DIM, 4, 1); \
  else TMC_TREE_WIDE(DIM, 8, 1)
  if (head_dim == 128) {
    TMC_TREE_VECTORS(128);
  } else {
    TMC_TREE_VECTORS(64);
  }
#undef TMC_TREE_VECTORS
#undef TMC_TREE_WIDE
#undef TMC_TREE_RING
  if (check_launch(l.vectors <= 32 ? "tree_ring_kernel" : "tree_wide_kernel")) return 1;
  if (!l.split || l.arrivals) return 0;
  // has_join()
  if (head_dim == 64) TMC_TREE_JOIN(64, 64);
  else if (l.vectors == 64) TMC_TREE_JOIN(128, 64);
  else TMC_TREE_JOIN(128, 256);
#undef TMC_TREE_JOIN
  return check_launch("tree_join_kernel");
}
