// Trees of drafted tokens beside a paged cache: what each node sees, its K and V
// into the cache, the branch that the sampled tokens agree with, and its K and
// V moved up.
//
// A tree has up to kTreeMost nodes.  Node i's parent is an earlier node; a parent
// outside [0, i) makes it a root.  Node i of a request with `cached` positions
// lies in slot cached + i and at position cached + depth(i).
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>

namespace tmc {
namespace {

__device__ __forceinline__ int tree_count(const int32_t* counts, int request, int nodes) {
  return counts ? max(0, min(counts[request], nodes)) : nodes;
}

// ------------------------------------------------------------ masks and depths
// mask(i) = mask(parent(i)) | 1 << i, depth(i) = depth(parent(i)) + 1.  A block a
// tree, a thread a node: ancestors known so far are joined with those of the last
// of them, so a chain of n takes log2 n turns, not n.  2.3 us for a tree, 3.6 for 64 of 32
// nodes: launch and latencies.
__global__ __launch_bounds__(kTreeMost) void tree_layout_kernel(const int32_t* __restrict__ parents,
                                                                const int32_t* __restrict__ counts,
                                                                uint32_t* __restrict__ masks,
                                                                int32_t* __restrict__ depths,
                                                                int nodes, int words) {
  __shared__ uint32_t s_mask[2][kTreeWords][kTreeMost];
  __shared__ int s_up[2][kTreeMost];
  const int request = blockIdx.x, i = threadIdx.x;
  const size_t node = (size_t)request * nodes + i;
  const bool here = i < nodes;
  int up = here ? parents[node] : -1;
  const int count = tree_count(counts, request, nodes);
  if (up < 0 || up >= i) up = -1;
  uint32_t mask[kTreeWords];
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) mask[w] = w == i >> 5 ? 1u << (i & 31) : 0u;
  int turn = 0;
  while (__syncthreads_or(up >= 0)) {
    s_up[turn][i] = up;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) s_mask[turn][w][i] = mask[w];
    __syncthreads();
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) mask[w] |= s_mask[turn][w][up];
      up = s_up[turn][up];
    }
    turn ^= 1;
  }
  if (!here || i >= count) return;
  int depth = -1;
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) {
    depth += __popc(mask[w]);
    if (w < words) masks[node * words + w] = mask[w];
  }
  depths[node] = depth;
}

// ------------------------------------------------------------ rotation and append
// tmc_decode_rope_append with a position and a slot of a node's own: bits as there.
struct TreeAppend {
  const float* cosine;      // [positions][head_dim / 2]
  const float* sine;
  const int32_t* cached;    // [batch]
  const int32_t* depths;    // [batch][nodes]
  const int32_t* counts;    // [batch] or null
  const int32_t* tables;    // [batch][max_pages]
  const int32_t* active;    // or null
  int batch, nodes, q_heads, kv_heads, head_dim, page_size, max_pages, pool_pages;
  long positions;
  PageDivide by_row, by_nodes, by_head, by_page;  // by a row's units, and so on
};

// EACH adjacent elements of one head a thread: 8 in 16-byte loads and stores, else
// a pair.  64 trees of 32 nodes (32 + 2 x 8 heads of 128): 7.8 us, 3.1 TB/s for 24 MB; a
// tree of 8 nodes 3.2 us.  Indices by products: with divisions, and angles by single
// words, 12.4 us.
template <typename T, int EACH>
__global__ __launch_bounds__(256) void tree_append_kernel(const T* __restrict__ qkv,
                                                          T* __restrict__ q_out,
                                                          T* __restrict__ k_pool,
                                                          T* __restrict__ v_pool, TreeAppend p) {
  typedef T vec __attribute__((ext_vector_type(EACH)));
  const int width = (p.q_heads + 2 * p.kv_heads) * p.head_dim;
  const unsigned id = blockIdx.x * 256u + threadIdx.x;  // below 2^31; of elements, below 2^32
  const int node = p.by_row((int)id);
  if (node >= p.batch * p.nodes) return;
  const int request = p.by_nodes(node), i = node - request * p.nodes;
  const int column = (int)(EACH * id - (unsigned)node * (unsigned)width);
  // everything that depends on nothing, in flight at once
  const int active = p.active ? p.active[0] : p.batch;
  const int cached = p.cached[request], depth = p.depths[node];
  const int count = tree_count(p.counts, request, p.nodes);
  const vec x = *reinterpret_cast<const vec*>(qkv + (size_t)node * width + column);
  const long slot = (long)cached + i, position = (long)cached + depth;
  if (request >= active || i >= count || cached < 0 || position < 0 || position >= p.positions ||
      slot >= (long)p.page_size * p.max_pages)
    return;
  const int q_width = p.q_heads * p.head_dim, kv_width = p.kv_heads * p.head_dim;
  vec y = x;
  if (column < q_width + kv_width) {
    const int feature = column - p.by_head(column) * p.head_dim;
    const size_t at = (size_t)position * (p.head_dim / 2) + feature / 2;
    typedef float angles __attribute__((ext_vector_type(EACH / 2), aligned(4)));
    const angles cosine = *reinterpret_cast<const angles*>(p.cosine + at);
    const angles sine = *reinterpret_cast<const angles*>(p.sine + at);
#pragma unroll
    for (int e = 0; e < EACH; e += 2) {
      float even, odd;
      rotate_pair(to_float<T>(x[e]), to_float<T>(x[e + 1]), cosine[e / 2], sine[e / 2], even, odd);
      // fp32 first, then the storage type, as the other rotations round
      asm volatile("" : "+v"(even), "+v"(odd));
      y[e] = from_float<T>(even);
      y[e + 1] = from_float<T>(odd);
    }
  }
  if (column < q_width) {
    *reinterpret_cast<vec*>(q_out + (size_t)node * q_width + column) = y;
    return;
  }
  const int index = p.by_page((int)slot);
  const int page = p.tables[(size_t)request * p.max_pages + index];
  if (page < 0 || page >= p.pool_pages) return;
  const bool key = column < q_width + kv_width;
  const int feature = column - q_width - (key ? 0 : kv_width), head = p.by_head(feature);
  *reinterpret_cast<vec*>((key ? k_pool : v_pool) +
                          (((size_t)page * p.kv_heads + head) * p.page_size +
                           ((int)slot - index * p.page_size)) * p.head_dim +
                          (feature - head * p.head_dim)) = y;
}

// ------------------------------------------------------------ the branch kept
// From node 0 to the child whose drafted token is the one chosen at its parent
// (the lowest of several), as long as there is one.  A wave a tree, four nodes a
// lane in registers: a step is a read of the chosen token and ballots.  2.5 us for a
// tree of 8 nodes, 4.2 us for 64 of 32: launch and latencies.
constexpr int kNodesLane = kTreeMost / kWave;
struct TreeAccept {
  const int32_t* drafted;  // [batch][nodes]
  const int32_t* parents;
  const int32_t* chosen;
  const int32_t* counts;   // [batch] or null
  const int32_t* active;   // or null
  const int32_t* cached;   // [batch] or null
  int32_t* path;           // [batch][nodes]
  int32_t* accepted;       // [batch]
  int32_t* emitted;        // [batch][nodes]
  int32_t* new_lengths;    // [batch] or null
  int batch, nodes;
};

__global__ __launch_bounds__(kWave) void tree_accept_kernel(TreeAccept p) {
  __shared__ int s_chosen[kTreeMost], s_path[kTreeMost];
  const int request = blockIdx.x, lane = threadIdx.x;
  const size_t first = (size_t)request * p.nodes;
  const int active = p.active ? p.active[0] : p.batch;
  const int cached = p.cached ? p.cached[request] : 0;
  const int count = request < active ? tree_count(p.counts, request, p.nodes) : 0;
  int parent[kNodesLane], token[kNodesLane];
#pragma unroll
  for (int r = 0; r < kNodesLane; ++r) {
    const int i = r * kWave + lane;
    const bool here = i < p.nodes;
    parent[r] = here ? p.parents[first + i] : -1;
    token[r] = here ? p.drafted[first + i] : 0;
    s_chosen[i] = here ? p.chosen[first + i] : 0;
    if (i >= count || parent[r] >= i) parent[r] = -1;
  }
  __syncthreads();
  int at = count > 0 ? 0 : -1, taken = 0;
  while (at >= 0) {  // ever greater nodes
    const int pick = s_chosen[at];
    if (lane == 0) s_path[taken] = at;
    ++taken;
    int next = -1;
#pragma unroll
    for (int r = kNodesLane - 1; r >= 0; --r) {
      const unsigned long long fits =
          __builtin_amdgcn_ballot_w64(parent[r] == at && token[r] == pick);
      if (fits) next = r * kWave + __builtin_ctzll(fits);
    }
    at = next;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kNodesLane; ++r) {
    const int i = r * kWave + lane;
    if (i >= p.nodes) break;
    const int node = i < taken ? s_path[i] : -1;
    p.path[first + i] = node;
    p.emitted[first + i] = i < taken ? s_chosen[node] : -1;
  }
  if (lane == 0) {
    p.accepted[request] = taken;
    if (p.new_lengths) p.new_lengths[request] = cached + taken;
  }
}

// ------------------------------------------------------------ K and V moved up
// Slot cached + path[s] to slot cached + s, for every step s.  Paths increase, so
// path[s] >= s, no later step reads what an earlier one wrote, and steps before
// the first with path[s] != s have nothing to move.  A thread owns a unit of a
// (layer, head), of K and of V, and takes the steps in order, kKeepAhead loads before
// their stores, so that nobody else is waited for.  64 requests, 32 layers, up to 8
// steps: 10 us, latencies of path, table, page and store one after the other; step by
// step and K and V apart it took 23 us.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kKeepPools = 128;  // pool pairs per launch (kernel arguments)
constexpr int kKeepAhead = 8, kKeepThreads = 128;

struct TreeKeep {
  void* key[kKeepPools];
  void* value[kKeepPools];
  const int32_t* tables;    // [pools][batch][max_pages]
  const int32_t* cached;    // [batch]
  const int32_t* path;      // [batch][nodes]
  const int32_t* accepted;  // [batch]
  int batch, nodes, heads, page_size, max_pages, pool_pages, row_units;
  long page_stride, head_stride;  // units
  PageDivide by_row, by_page;
};

template <typename UNIT>
__global__ __launch_bounds__(kKeepThreads) void tree_keep_kernel(TreeKeep p) {
  const int request = blockIdx.x, pool = blockIdx.y;
  const int column = (int)blockIdx.z * kKeepThreads + threadIdx.x;
  const int head = p.by_row(column);
  const int32_t* path = p.path + (size_t)request * p.nodes;
  const int taken = min(p.accepted[request], p.nodes), cached = p.cached[request];
  if (head >= p.heads || cached < 0) return;
  const int32_t* table = p.tables + ((size_t)pool * p.batch + request) * p.max_pages;
  const long capacity = (long)p.page_size * p.max_pages;
  const size_t own = (size_t)head * p.head_stride + (column - head * p.row_units);
  UNIT* const base[2] = {static_cast<UNIT*>(p.key[pool]) + own,
                         static_cast<UNIT*>(p.value[pool]) + own};
  int last = -1;  // node of the step before
  for (int s0 = 0; s0 < taken; s0 += kKeepAhead) {
    // (every load of a stage in flight at once: those of steps that move nothing from a
    // place that is there)
    int node[kKeepAhead], row[2][kKeepAhead], page[2][kKeepAhead];
    bool moves[kKeepAhead];
    UNIT held[2][kKeepAhead];
#pragma unroll
    for (int a = 0; a < kKeepAhead; ++a) node[a] = path[min(s0 + a, p.nodes - 1)];
#pragma unroll
    for (int a = 0; a < kKeepAhead; ++a) {
      const int s = s0 + a;
      // (a list that does not increase ends where it does not)
      last = s < taken && node[a] > last && node[a] < p.nodes ? node[a] : p.nodes;
      moves[a] = last != p.nodes && node[a] != s && (long)cached + node[a] < capacity;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const int slot = moves[a] ? cached + (side ? s : node[a]) : 0, index = p.by_page(slot);
        row[side][a] = slot - index * p.page_size;
        page[side][a] = table[index];
      }
    }
#pragma unroll
    for (int a = 0; a < kKeepAhead; ++a) {
#pragma unroll
      for (int side = 0; side < 2; ++side)
        moves[a] = moves[a] && page[side][a] >= 0 && page[side][a] < p.pool_pages;
      const size_t from = moves[a] ? (size_t)page[0][a] * p.page_stride +
                                         (size_t)row[0][a] * p.row_units
                                   : 0;
      held[0][a] = base[0][from];
      held[1][a] = base[1][from];
    }
#pragma unroll
    for (int a = 0; a < kKeepAhead; ++a) {
      if (!moves[a]) continue;
      const size_t to = (size_t)page[1][a] * p.page_stride + (size_t)row[1][a] * p.row_units;
      base[0][to] = held[0][a];
      base[1][to] = held[1][a];
    }
  }
}

bool tree_shape(int64_t batch, int64_t nodes) {
  return batch > 0 && batch < 65536 && nodes > 0 && nodes <= kTreeMost;
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" int tmc_tree_layout(const int32_t* parents, const int32_t* counts, uint32_t* masks,
                               int32_t* depths, int64_t batch, int64_t nodes, void* stream) {
  TMC_REQUIRE(parents && masks && depths, "Tree layout: null device pointer.");
  TMC_REQUIRE(tree_shape(batch, nodes),
              "Tree layout: batch must be in [1, 65535] and nodes in [1, 256].");
  const unsigned threads = (unsigned)((nodes + kWave - 1) / kWave * kWave);
  hipLaunchKernelGGL(tree_layout_kernel, dim3((unsigned)batch), dim3(threads), 0,
                     as_stream(stream), parents, counts, masks, depths, (int)nodes,
                     (int)((nodes + 31) / 32));
  return check_launch("tree_layout_kernel");
}

extern "C" int tmc_tree_rope_append(const void* qkv, const float* cosine, const float* sine,
                                    int64_t positions, const int32_t* cached_lengths,
                                    const int32_t* depths, const int32_t* counts,
                                    const int32_t* block_tables, const int32_t* active_count,
                                    void* q_out, void* key_pool, void* value_pool, int dtype,
                                    int64_t batch, int64_t nodes, int64_t q_heads,
                                    int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                    int64_t max_pages, int64_t pool_pages, void* stream) {
  TMC_REQUIRE(qkv && cosine && sine && cached_lengths && depths && block_tables && q_out &&
                  key_pool && value_pool,
              "Tree append: null device pointer.");
  TMC_REQUIRE(dtype == TMC_F16 || dtype == TMC_F32, "Tree append: dtype must be f16 or f32.");
  TMC_REQUIRE(tree_shape(batch, nodes),
              "Tree append: batch must be in [1, 65535] and nodes in [1, 256].");
  TMC_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads < 65536 && q_heads % kv_heads == 0 &&
                  head_dim > 0 && head_dim % 2 == 0 && head_dim <= 1024 && positions > 0,
              "Tree append: invalid heads or rotation table.");
  TMC_REQUIRE(page_size > 0 && max_pages > 0 && page_size < (1LL << 30) &&
                  max_pages < (1LL << 30) && page_size * max_pages < (1LL << 30) &&
                  pool_pages > 0 && pool_pages < (1LL << 31),
              "Tree append: invalid page geometry.");
  const int64_t width = (q_heads + 2 * kv_heads) * head_dim;
  TMC_REQUIRE(batch * nodes * (width / 2) < (1LL << 31), "Tree append: too many elements.");
  const uintptr_t size = dtype == TMC_F16 ? 2 : 4;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
                         reinterpret_cast<uintptr_t>(key_pool) |
                         reinterpret_cast<uintptr_t>(value_pool);
  TMC_REQUIRE(bits % (2 * size) == 0, "Tree append: buffers must be aligned to two elements.");
  const int each = dtype == TMC_F16 && head_dim % 8 == 0 && bits % 16 == 0 ? 8 : 2;
  TreeAppend p{cosine,     sine,         cached_lengths, depths,        counts,         block_tables,
               active_count, (int)batch, (int)nodes,     (int)q_heads,  (int)kv_heads,  (int)head_dim,
               (int)page_size, (int)max_pages, (int)pool_pages, (long)positions,
               PageDivide::by(width / each), PageDivide::by(nodes), PageDivide::by(head_dim),
               PageDivide::by(page_size)};
#define TMC_TREE_APPEND(TYPE, EACH)                                                             \
  hipLaunchKernelGGL((tree_append_kernel<TYPE, EACH>),                                          \
                     dim3((unsigned)((batch * nodes * (width / EACH) + 255) / 256)), dim3(256), \
                     0, as_stream(stream), static_cast<const TYPE*>(qkv),                       \
                     static_cast<TYPE*>(q_out), static_cast<TYPE*>(key_pool),                   \
                     static_cast<TYPE*>(value_pool), p)
  if (dtype == TMC_F32) TMC_TREE_APPEND(float, 2);
  else if (each == 8) TMC_TREE_APPEND(half_t, 8);
  else TMC_TREE_APPEND(half_t, 2);
#undef TMC_TREE_APPEND
  return check_launch("tree_append_kernel");
}

extern "C" int tmc_tree_accept(const int32_t* drafted, const int32_t* parents,
                               const int32_t* chosen, const int32_t* counts,
                               const int32_t* active_count, const int32_t* cached_lengths,
                               int32_t* path, int32_t* accepted, int32_t* emitted,
                               int32_t* new_lengths, int64_t batch, int64_t nodes, void* stream) {
  TMC_REQUIRE(drafted && parents && chosen && path && accepted && emitted,
              "Tree accept: null device pointer.");
  TMC_REQUIRE(!new_lengths || cached_lengths, "Tree accept: new lengths need the cached ones.");
  TMC_REQUIRE(tree_shape(batch, nodes),
              "Tree accept: batch must be in [1, 65535] and nodes in [1, 256].");
  const TreeAccept p{drafted, parents,  chosen,  counts,      active_count, cached_lengths,
                     path,    accepted, emitted, new_lengths, (int)batch,   (int)nodes};
  hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)batch), dim3(kWave), 0, as_stream(stream), p);
  return check_launch("tree_accept_kernel");
}

extern "C" int tmc_tree_keep(void* const* key_pools, void* const* value_pools, int64_t pools,
                             const int32_t* block_tables, const int32_t* cached_lengths,
                             const int32_t* path, const int32_t* accepted, int dtype,
                             int64_t batch, int64_t nodes, int64_t heads, int64_t head_dim,
                             int64_t page_size, int64_t max_pages, int64_t pool_pages,
                             int64_t page_stride, int64_t head_stride, void* stream) {
  TMC_REQUIRE(key_pools && value_pools && block_tables && cached_lengths && path && accepted,
              "Tree keep: null pointer.");
  TMC_REQUIRE(dtype == TMC_F16 || dtype == TMC_F32 || dtype == TMC_BF16,
              "Tree keep: dtype must be f16, bf16 or f32.");
  TMC_REQUIRE(tree_shape(batch, nodes),
              "Tree keep: batch must be in [1, 65535] and nodes in [1, 256].");
  TMC_REQUIRE(pools > 0 && pools < (1LL << 20) && heads > 0 && heads < (1LL << 16) &&
                  head_dim > 0 && head_dim <= 1024,
              "Tree keep: invalid pools, heads or head_dim.");
  TMC_REQUIRE(page_size > 0 && max_pages > 0 && page_size < (1LL << 30) &&
                  max_pages < (1LL << 30) && page_size * max_pages < (1LL << 30) &&
                  pool_pages > 0 && pool_pages < (1LL << 31),
              "Tree keep: invalid page geometry.");
  TMC_REQUIRE(page_stride < (1LL << 40) && head_stride < (1LL << 40) &&
                  head_stride >= page_size * head_dim &&
                  page_stride >= (heads - 1) * head_stride + page_size * head_dim,
              "Tree keep: the head stride must hold a head's page rows and the page stride every "
              "head.");
  const int size = dtype == TMC_F32 ? 4 : 2;
  uintptr_t bits = (uintptr_t)(head_dim * size) | (uintptr_t)(page_stride * size) |
                   (uintptr_t)(head_stride * size);
  for (int64_t i = 0; i < pools; ++i) {
    TMC_REQUIRE(key_pools[i] && value_pools[i], "Tree keep: null pool pointer.");
    bits |= reinterpret_cast<uintptr_t>(key_pools[i]) | reinterpret_cast<uintptr_t>(value_pools[i]);
  }
  TMC_REQUIRE(bits % size == 0, "Tree keep: pools must be aligned to their elements.");
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
  const int64_t columns = heads * head_dim * size / unit;
  const int64_t parts = (columns + kKeepThreads - 1) / kKeepThreads;
  TMC_REQUIRE(parts < 65536, "Tree keep: too many heads.");
  for (int64_t first = 0; first < pools; first += kKeepPools) {
    const int here = (int)std::min<int64_t>(kKeepPools, pools - first);
    TreeKeep p{};
    for (int i = 0; i < here; ++i) {
      p.key[i] = key_pools[first + i];
      p.value[i] = value_pools[first + i];
    }
    p.tables = block_tables + first * batch * max_pages;
    p.cached = cached_lengths;
    p.path = path;
    p.accepted = accepted;
    p.batch = (int)batch;
    p.nodes = (int)nodes;
    p.heads = (int)heads;
    p.page_size = (int)page_size;
    p.max_pages = (int)max_pages;
    p.pool_pages = (int)pool_pages;
    p.row_units = (int)(head_dim * size / unit);
    p.by_row = PageDivide::by(p.row_units);
    p.by_page = PageDivide::by(page_size);
    p.page_stride = (long)page_stride * size / unit;
    p.head_stride = (long)head_stride * size / unit;
    const dim3 grid((unsigned)batch, (unsigned)here, (unsigned)parts);
    const hipStream_t s = as_stream(stream);
    if (unit == 16)
      hipLaunchKernelGGL((tree_keep_kernel<u32x4>), grid, dim3(kKeepThreads), 0, s, p);
    else if (unit == 4)
      hipLaunchKernelGGL((tree_keep_kernel<uint32_t>), grid, dim3(kKeepThreads), 0, s, p);
    else
      hipLaunchKernelGGL((tree_keep_kernel<uint16_t>), grid, dim3(kKeepThreads), 0, s, p);
    if (check_launch("tree_keep_kernel")) return 1;
  }
  return 0;
}
