// Attention of trees of drafted tokens over a paged cache, gfx950.
//
// Node i of request r, with `cached` positions before its tree, sees [0, cached)
// and position cached + j for every bit j < count of its mask:
//   out = sum_s w_s v_s / sum_s w_s,  w_s = exp(q . k_s / sqrt(D) - max),
// and zeros where it sees nothing.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <cmath>

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

extern "C" size_t tmc_tree_attention_workspace_bytes(int64_t batch, int64_t nodes, int64_t q_heads,
                                                     int64_t kv_heads, int64_t head_dim,
                                                     int64_t capacity) {
  return 0;
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
  p.counts = counts;
  p.active = active_count;
  hipLaunchKernelGGL(tree_plain_kernel, dim3((unsigned)(batch * nodes), (unsigned)q_heads),
                     dim3(kWave), 0, as_stream(stream), p);
  return check_launch("tree_plain_kernel");
}
