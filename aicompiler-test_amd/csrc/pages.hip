// Pages of a paged cache copied inside their pools, and the block tables that
// follow them: forking a request (its children share its full pages and get a
// copy of the partly filled last one) and compacting a fragmented pool.
#include "tmc_abi.hpp"
#include "tmc_device.hpp"

#include <algorithm>
#include <exception>
#include <set>
#include <utility>

namespace tmc {
namespace {

constexpr int kMovePools = 128;  // pool pairs per launch (kernel arguments)

struct MoveParams {
  void* key[kMovePools];
  void* value[kMovePools];
  const int4* moves;  // (pool, source page, destination page, positions)
  int first_pool, pools, pool_pages, heads, page_size;
  long page_bytes, head_bytes;  // strides
  int row_bytes;                // one head's position
  int parts, head_blocks;       // blocks a head, or blocks the heads share
};

// One block per (move, K or V, about kMoveUnits of the page: a part of one head's
// positions, or every head_blocks-th head), in units of UNIT bytes: pure copying,
// bound by memory, so a thread copies unit by unit (eight loads ahead of their
// stores took 1.5 times as long over a large pool).  Four copies each of 8
// requests' last pages in 32 layers, 8 MB read and 32 written: 12 us, against 8 at a large copy's
// rate; a quarter of 1 GiB of pools compacted: 104 us, 5.2 TB/s, that rate.  Pages
// of 256 positions, 8 heads of 128: 13 us where a block a page took 40; pages of
// 32 positions, 32 heads, compacted: 10 us where two blocks a page took 17.
// Pages of one position, 32 heads, forked: 13 us where a head at a time took 30.
constexpr int kMoveUnits = 1024;
template <typename UNIT>
__global__ __launch_bounds__(256) void move_pages_kernel(MoveParams p) {
  const int4 m = p.moves[blockIdx.x];
  const int from = m.y, to = m.z, count = m.w;
  if (m.x < p.first_pool || m.x - p.first_pool >= p.pools || from < 0 ||
      from >= p.pool_pages || to < 0 || to >= p.pool_pages || from == to || count < 1 ||
      count > p.page_size)
    return;
  const int pool = m.x - p.first_pool;
  char* base = static_cast<char*>(blockIdx.y ? p.value[pool] : p.key[pool]);
  const char* src = base + (size_t)from * p.page_bytes;
  char* dst = base + (size_t)to * p.page_bytes;
  const unsigned run = (unsigned)((long)count * p.row_bytes / (int)sizeof(UNIT));  // units a head
  const int part = blockIdx.z / p.head_blocks;
  // threads a head: short runs of several heads are copied side by side
  const unsigned wide = min(run, 256u), at_once = 256u / wide;
  const unsigned mine = threadIdx.x / wide, lane = threadIdx.x - mine * wide;
  if (mine >= at_once) return;
  for (unsigned h = blockIdx.z - part * p.head_blocks + mine * p.head_blocks; h < (unsigned)p.heads;
       h += at_once * p.head_blocks) {
    const UNIT* s = reinterpret_cast<const UNIT*>(src + (size_t)h * p.head_bytes);
    UNIT* d = reinterpret_cast<UNIT*>(dst + (size_t)h * p.head_bytes);
    for (unsigned first = part * kMoveUnits; first < run; first += p.parts * kMoveUnits)
      for (unsigned u = first + lane; u < min(first + kMoveUnits, run); u += wide) d[u] = s[u];
  }
}

struct TableParams {
  const int32_t* tables;   // [layers][table_rows][max_pages]
  const int32_t* parents;  // [rows] or null: row r itself
  const int32_t* remap;    // [layers][pool_pages] or null
  const int32_t* slots;    // [rows] or null
  const int32_t* tails;    // [layers][rows]
  int32_t* out;            // [layers][rows][max_pages]
  int table_rows, rows, max_pages, pool_pages;
  size_t entries;
};

__global__ __launch_bounds__(256) void rebuild_tables_kernel(TableParams p) {
  for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < p.entries;
       e += (size_t)gridDim.x * 256) {
    const size_t line = e / (unsigned)p.max_pages;
    const int slot = (int)(e - line * p.max_pages);
    const size_t layer = line / (unsigned)p.rows;
    const int row = (int)(line - layer * p.rows);
    const int parent = p.parents ? p.parents[row] : row;
    int page = -1;
    if (parent >= 0 && parent < p.table_rows)
      page = p.tables[(layer * p.table_rows + parent) * p.max_pages + slot];
    if (p.remap && page >= 0 && page < p.pool_pages) page = p.remap[layer * p.pool_pages + page];
    if (p.slots && p.slots[row] == slot) page = p.tails[line];
    p.out[e] = page;
  }
}

int element_bytes_of(int dtype) { return dtype == TMC_F16 || dtype == TMC_BF16 ? 2 : 4; }

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" int tmc_check_page_moves(const int32_t* moves, int64_t count, int64_t pools,
                                    int64_t pool_pages, int64_t page_size) {
  TMC_REQUIRE(moves || count == 0, "Page moves: null pointer.");
  TMC_REQUIRE(count >= 0 && pools > 0 && pool_pages > 0 && page_size > 0,
              "Page moves: invalid shape.");
  try {
    std::set<std::pair<int32_t, int32_t>> sources, targets;
    for (int64_t i = 0; i < count; ++i) {
      const int32_t *m = moves + 4 * i, pool = m[0], from = m[1], to = m[2], positions = m[3];
      const std::string which = "Page moves: move " + std::to_string(i);
      TMC_REQUIRE(pool >= 0 && pool < pools && from >= 0 && from < pool_pages && to >= 0 &&
                      to < pool_pages,
                  which + " names a pool or page that does not exist.");
      TMC_REQUIRE(positions >= 1 && positions <= page_size,
                  which + " must copy 1 to page_size positions.");
      TMC_REQUIRE(targets.insert({pool, to}).second, which + " writes a page that another move writes.");
      sources.insert({pool, from});
    }
    for (const auto& t : targets)
      TMC_REQUIRE(!sources.count(t), "Page moves: page " + std::to_string(t.second) + " of pool " +
                                         std::to_string(t.first) + " is both read and written.");
  } catch (const std::exception& e) {  // out of memory
    TMC_REQUIRE(false, std::string("Page moves: ") + e.what());
  }
  return 0;
}

extern "C" int tmc_move_pages(void* const* key_pools, void* const* value_pools, int64_t pools,
                              const int32_t* moves, int64_t count, int dtype, int64_t pool_pages,
                              int64_t heads, int64_t page_size, int64_t head_dim,
                              int64_t page_stride, int64_t head_stride, void* stream) {
  TMC_REQUIRE(key_pools && value_pools && moves, "Move pages: null pointer.");
  TMC_REQUIRE(dtype == TMC_F16 || dtype == TMC_F32 || dtype == TMC_BF16,
              "Move pages: dtype must be f16, bf16 or f32.");
  TMC_REQUIRE(pools > 0 && pools < (1LL << 20) && count >= 0 && count < (1LL << 24) &&
                  pool_pages > 0 && pool_pages < (1LL << 31) && heads > 0 && heads < (1LL << 20) &&
                  page_size > 0 && page_size < (1LL << 24) && head_dim > 0 &&
                  head_dim < (1LL << 16) && page_size * head_dim < (1LL << 29),
              "Move pages: invalid shape.");
  TMC_REQUIRE(page_stride < (1LL << 40) && head_stride < (1LL << 40) &&
                  head_stride >= page_size * head_dim &&
                  page_stride >= (heads - 1) * head_stride + page_size * head_dim,
              "Move pages: the head stride must hold a head's page rows and the page stride every "
              "head.");
  const int size = element_bytes_of(dtype);
  TMC_REQUIRE((reinterpret_cast<uintptr_t>(moves) & 15) == 0,
              "Move pages: moves must be 16-byte aligned.");
  uintptr_t bits = (uintptr_t)(head_dim * size) | (uintptr_t)(page_stride * size) |
                   (uintptr_t)(head_stride * size);
  for (int64_t i = 0; i < pools; ++i) {
    TMC_REQUIRE(key_pools[i] && value_pools[i], "Move pages: null pool pointer.");
    bits |= reinterpret_cast<uintptr_t>(key_pools[i]) | reinterpret_cast<uintptr_t>(value_pools[i]);
  }
  TMC_REQUIRE(bits % size == 0, "Move pages: pools must be aligned to their elements.");
  if (count == 0) return 0;
  const hipStream_t s = as_stream(stream);
  for (int64_t first = 0; first < pools; first += kMovePools) {
    MoveParams p{};
    p.first_pool = (int)first;
    p.pools = (int)std::min<int64_t>(kMovePools, pools - first);
    for (int i = 0; i < p.pools; ++i) {
      p.key[i] = key_pools[first + i];
      p.value[i] = value_pools[first + i];
    }
    p.moves = reinterpret_cast<const int4*>(moves);
    p.pool_pages = (int)pool_pages;
    p.heads = (int)heads;
    p.page_size = (int)page_size;
    p.page_bytes = (long)page_stride * size;
    p.head_bytes = (long)head_stride * size;
    p.row_bytes = (int)head_dim * size;
    const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
    const int64_t units = page_size * p.row_bytes / unit;  // a head's
    p.parts = (int)std::min<int64_t>((units + kMoveUnits - 1) / kMoveUnits, 64);
    const int64_t together = std::max<int64_t>(kMoveUnits / units, 1);  // heads a block
    p.head_blocks = (int)std::min<int64_t>((heads + together - 1) / together, 512);
    const dim3 grid((unsigned)count, 2, (unsigned)(p.parts * p.head_blocks));
    if (bits % 16 == 0)
      hipLaunchKernelGGL((move_pages_kernel<uint4>), grid, dim3(256), 0, s, p);
    else if (bits % 4 == 0)
      hipLaunchKernelGGL((move_pages_kernel<uint32_t>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((move_pages_kernel<uint16_t>), grid, dim3(256), 0, s, p);
    if (check_launch("move_pages_kernel")) return 1;
  }
  return 0;
}

extern "C" int tmc_rebuild_tables(const int32_t* tables, const int32_t* parents,
                                  const int32_t* remap, const int32_t* tail_slots,
                                  const int32_t* tails, int32_t* out, int64_t layers,
                                  int64_t table_rows, int64_t rows, int64_t max_pages,
                                  int64_t pool_pages, void* stream) {
  TMC_REQUIRE(tables && out, "Rebuild tables: null device pointer.");
  TMC_REQUIRE(!tail_slots == !tails, "Rebuild tables: tail slots and tails go together.");
  const int64_t most = 1LL << 24;
  TMC_REQUIRE(layers > 0 && layers < most && table_rows > 0 && table_rows < most && rows > 0 &&
                  rows < most && max_pages > 0 && max_pages < (1LL << 30) && pool_pages > 0 &&
                  pool_pages < (1LL << 31) && rows * max_pages < (1LL << 40) / layers &&
                  table_rows * max_pages < (1LL << 40) / layers,
              "Rebuild tables: invalid shape.");
  TMC_REQUIRE(parents || rows == table_rows,
              "Rebuild tables: without parents the rows are those of the tables.");
  const char *from = reinterpret_cast<const char*>(tables), *to = reinterpret_cast<char*>(out);
  const int64_t from_bytes = layers * table_rows * max_pages * 4,
                to_bytes = layers * rows * max_pages * 4;
  TMC_REQUIRE((!parents && from == to) || from + from_bytes <= to || to + to_bytes <= from,
              "Rebuild tables: out may be the tables themselves (without parents), else it must "
              "not overlap them.");
  TableParams p{};
  p.tables = tables;
  p.parents = parents;
  p.remap = remap;
  p.slots = tail_slots;
  p.tails = tails;
  p.out = out;
  p.table_rows = (int)table_rows;
  p.rows = (int)rows;
  p.max_pages = (int)max_pages;
  p.pool_pages = (int)pool_pages;
  p.entries = (size_t)(layers * rows * max_pages);
  const unsigned blocks = (unsigned)std::min<size_t>((p.entries + 255) / 256, 8192);
  hipLaunchKernelGGL(rebuild_tables_kernel, dim3(blocks), dim3(256), 0, as_stream(stream), p);
  return check_launch("rebuild_tables_kernel");
}
