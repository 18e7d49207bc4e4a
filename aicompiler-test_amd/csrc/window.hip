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
  int page_size, max_pages, page_shift;
  int window, sinks;
  int own_table;         // row r reads table row r
  long out_pass;         // > 0: packed activation order, elements per 16-row pass
  float scale_log2;      // log2(e) / sqrt(D)
};

__device__ __forceinline__ int window_page(const WindowParams& p, int pos) {
  return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
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
// dims for P V.  Online softmax in fp32.
constexpr int kPlainMaxDim = 256;

__global__ __launch_bounds__(kWave) void window_plain_kernel(WindowParams p) {
  __shared__ __align__(16) half_t s_q[kPlainMaxDim];
  __shared__ float s_p[kWave];
  __shared__ long s_at[kWave];
  const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y;
  if (row >= (p.active ? min(p.active[0], p.rows) : p.rows)) return;
  const int valid = p.valid[row], table_row = window_table(p, row);
  if (valid < 1 || valid > p.page_size * p.max_pages || table_row < 0) return;
  const int32_t* table = p.tables + (size_t)table_row * p.max_pages;
  const int kvh = head / p.group, d = p.dim;
  const half_t* q = p.q + ((size_t)row * p.q_heads + head) * d;
  for (int i = lane; i < d; i += kWave) s_q[i] = q[i];
  const int begin = window_begin(p, valid), first = min(p.sinks, begin);
  const int count = first + valid - begin;
  float m = -INFINITY, sum = 0.0f, o[kPlainMaxDim / kWave] = {};
  bool bad = false;
  __syncthreads();
  for (int u0 = 0; u0 < count; u0 += kWave) {
    const int u = u0 + lane, pos = u < first ? u : begin + u - first;
    float score = -INFINITY;
    long at = -1;
    if (u < count) {
      const int slot = window_page(p, pos), page = table[slot];
      if (window_page_ok(p, page)) {
        at = (long)page * p.page_stride + (long)kvh * p.head_stride +
             (long)(pos - slot * p.page_size) * d;
        float dot = 0.0f;
        for (int c = 0; c < d; c += 8)
          dot = dot8(load_h8(s_q + c), load_h8(p.k + at + c), dot);
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
    s_p[lane] = w;
    s_at[lane] = at;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kPlainMaxDim / kWave; ++t) o[t] *= alpha;
    const int live = min(kWave, count - u0);
    for (int i = 0; i < live; ++i) {
      const long from = s_at[i];
      const float wi = s_p[i];
      if (from < 0) continue;
#pragma unroll
      for (int t = 0; t < kPlainMaxDim / kWave; ++t)
        if (lane + t * kWave < d) o[t] += wi * (float)p.v[from + lane + t * kWave];
    }
    __syncthreads();
  }
  if (__any(bad)) return;
  sum = cross_sum<1>(sum);
#pragma unroll
  for (int t = 0; t < kPlainMaxDim / kWave; ++t)
    if (lane + t * kWave < d)
      p.out[window_out(p, row, head * d + lane + t * kWave)] = (half_t)(o[t] / sum);
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
  p.page_shift = -1;
  for (int b = 0; b < 30; ++b)
    if (page_size == (int64_t)1 << b) p.page_shift = b;
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

extern "C" size_t tmc_window_attention_workspace_bytes(int64_t batch, int64_t q_heads,
                                                       int64_t kv_heads, int64_t head_dim,
                                                       int64_t capacity, int64_t window,
                                                       int64_t sinks) {
  return 0;
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
  TMC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "Window attention: workspace is smaller than "
              "tmc_window_attention_workspace_bytes().");
  p.active = active_count;
  p.table_rows = p.rows;
  p.own_table = 1;
  if (layout) p.out_pass = (long)((q_heads * head_dim + 31) / 32) * 512;
  return launch_plain(p, as_stream(stream));
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
  return launch_plain(p, as_stream(stream));
}
