// Entry points of the paged attention (paged_attention.h has the kernel and its reasons).
#include "paged_attention.h"

namespace pvsg {

// Caches of up to so many tiles are not split: each has a workgroup of its own (and waits once a tile for its memory, 1.2 us).  Measured both
// ways with 4 heads, 2 / 25 / 100 ragged sequences, us split and joined against whole:
//   f32 over f32, heads of 128 (64 keys a tile: 512 positions)   up to  400  14.5 / 15.8 / 26.3  against 13.9 / 15.0 / 26.2,  700  14.8 / 16.7 / 41.4  against 19.3 / 20.3 / 43.8
//   bf16 over bf16, heads of 128 (128 keys: 1024 positions)      up to  700  11.9 / 13.2 / 23.6  against 11.1 / 12.2 / 21.1, 1500  12.5 / 16.3 / 42.1  against 17.8 / 18.9 / 45.5
//   f32 over e4m3, heads of 128 (128 keys)                       up to 1000  13.7 / 14.8 / 22.5  against 13.1 / 14.1 / 20.4, 1500  13.8 / 15.3 / 25.7  against 17.0 / 18.1 / 27.9
//   bf16 over e4m3, heads of 64 (128 keys)                       up to 1000  11.8 / 12.2 / 19.2  against 11.4 / 11.8 / 16.1, 1500  12.0 / 12.9 / 20.6  against 15.0 / 15.7 / 20.8
//   f32 over f32, heads of 32 (128 keys)                         up to 1000  12.5 / 13.6 / 21.3  against 12.0 / 12.8 / 19.5, 1500  12.7 / 13.9 / 25.2  against 15.9 / 16.8 / 25.6
//   16 new tokens, bf16 over bf16, heads of 128                  up to 1000  15.7 / 17.3 / 36.1  against 14.2 / 15.3 / 31.4, 1500  15.8 / 18.3 / 47.4  against 18.3 / 19.4 / 47.4
constexpr int PA_SHORT = 8;

// 16-row tiles a wave carries: two where there are more rows than one tile holds and the accumulators of two (of f32 rows: three-part queries
// or single columns of two) fit.  Rows past that walk the cache again: 100 x up to 5000 x 4 x 128, 16 and 32 new tokens, f32 over f32 211 and
// 324 us, over bf16 116 and 173, over e4m3 72 and 102.
static int pa_tiles(int rows, int dim, int row_type) { return rows > 16 && dim <= (row_type == KV_F32 ? 64 : 128) ? 2 : 1; }

// How the work is shared out: rows of a tile group, groups, and how many workgroups take equal stretches (0: one each)
struct PaPlan {
  int tiles, row_groups, workgroups;
  long long units;
  size_t part_o, part_ml;                // floats of the workspace
};
static PaPlan pa_plan(const pvsg_kv_pages& p, int B, int T, int q_heads, int row_type, int table_width, long long max_len) {
  PaPlan s{};
  const int rows = T * (q_heads / p.heads);
  s.tiles = pa_tiles(rows, p.dim, row_type);
  s.row_groups = (rows + 16 * s.tiles - 1) / (16 * s.tiles);
  s.units = (long long)B * p.heads * s.row_groups;
  const long long capacity = (long long)table_width * p.page_size, longest = max_len > 0 && max_len < capacity ? max_len : capacity;
  const int dim = pa_dim(p.dim);
  auto tile = [&](bool split) { return PA_WAVES * 16 * pa_blocks(row_type, p.type, dim, s.tiles, split); };
  const int blocks = pa_blocks(row_type, p.type, dim, s.tiles, true), part = pa_part_cost(blocks);
  if (longest <= (long long)PA_SHORT * tile(false) || s.units * (capacity / tile(true) + 1 + part) >= (1ll << 31)) return s;     // (the list is counted in 32 bits)
  const long long tiles = (longest + tile(true) - 1) / tile(true);
  static_assert(256 * pa_per_cu(32, 1, 2) <= PVSG_PAGED_ATTENTION_COUNTERS, "a counter for each workgroup");
  const long long room = 256 * pa_per_cu(dim, s.tiles, blocks), work = (s.units * (tiles + part) + part + PA_GRAIN - 1) / (part + PA_GRAIN);
  s.workgroups = (int)(work < room ? work : room);
  const size_t rows_of = (size_t)2 * s.workgroups * 16 * s.tiles;
  s.part_o = rows_of * p.dim, s.part_ml = rows_of * 2;
  return s;
}

}  // namespace pvsg

extern "C" long long pvsg_paged_attention_workspace_bytes(const pvsg_kv_pages* pages, int B, int T, int q_heads, int row_type, int table_width,
                                                          long long max_len) {
  using namespace pvsg;
  if (!pages || pages->heads <= 0 || pages->dim <= 0 || B <= 0 || T <= 0 || q_heads < pages->heads || table_width <= 0) return 0;
  const PaPlan s = pa_plan(*pages, B, T, q_heads, row_type, table_width, max_len);
  return (long long)(s.part_o + s.part_ml) * 4;
}

extern "C" int pvsg_paged_attention(const pvsg_kv_pages* pages, const void* q, long long q_seq_stride, long long q_token_stride,
                                    long long q_head_stride, void* out, int row_type, const int* table, long long table_stride, int table_width,
                                    const int* lens, const int* new_lens, const uint8_t* padding, long long padding_stride, int padding_width,
                                    int B, int T, int q_heads, float scale, int causal, long long max_len, void* workspace, uint32_t* counters, void* stream) {
  using namespace pvsg;
  if (const int rc = kv_check_pages("pvsg_paged_attention", pages, table, table_stride, table_width, lens, B)) return rc;
  PVSG_REQUIRE(q && out, "pvsg_paged_attention: null pointer");
  PVSG_REQUIRE(row_type >= KV_F32 && row_type <= KV_F16, "pvsg_paged_attention: row type %d", row_type);
  PVSG_REQUIRE(row_type == KV_F32 || row_type == pages->type || kv_scaled(pages->type), "pvsg_paged_attention: rows of type %d over a pool of type %d", row_type, pages->type);
  const long long rb = kv_bytes(row_type);
  PVSG_REQUIRE(((q_seq_stride | q_token_stride | q_head_stride) * rb) % 16 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0, "pvsg_paged_attention: rows are not 16-byte aligned");
  PVSG_REQUIRE(T >= 0 && T <= PA_MAX_T, "pvsg_paged_attention: %d new tokens (at most %d)", T, PA_MAX_T);
  PVSG_REQUIRE(q_heads > 0 && q_heads % pages->heads == 0 && q_heads / pages->heads <= 1024, "pvsg_paged_attention: %d query heads over %d key heads", q_heads, pages->heads);
  PVSG_REQUIRE(!padding || (padding_width >= 0 && padding_stride >= 0), "pvsg_paged_attention: bad padding mask");
  if (B == 0 || T == 0) return PVSG_OK;
  const PaPlan s = pa_plan(*pages, B, T, q_heads, row_type, table_width, max_len);
  PVSG_REQUIRE(s.workgroups == 0 || (workspace && counters && (((uintptr_t)workspace & 15) | ((uintptr_t)counters & 3)) == 0),
               "pvsg_paged_attention: workspace %p and counters %p, %lld bytes are needed", workspace, static_cast<void*>(counters),
               (long long)(s.part_o + s.part_ml) * 4);
  PVSG_REQUIRE(s.workgroups || s.units < KV_MAX_BLOCKS, "pvsg_paged_attention: %lld parts are too many for one launch", s.units);
  PagedAttn a{};
  a.p = *pages;
  a.q = static_cast<const unsigned char*>(q), a.out = static_cast<unsigned char*>(out);
  a.table = table, a.lens = lens, a.new_lens = new_lens, a.padding = padding;
  a.q_seq = q_seq_stride * rb, a.q_token = q_token_stride * rb, a.q_head = q_head_stride * rb;
  a.table_stride = table_stride, a.padding_stride = padding_stride;
  a.scale_log2e = scale * 1.44269504088896340736f;
  a.width = table_width, a.padding_width = padding_width;
  while ((1 << a.page_shift) < pages->page_size) ++a.page_shift;
  a.B = B, a.T = T, a.q_heads = q_heads, a.group = q_heads / pages->heads, a.rows = T * a.group, a.row_groups = s.row_groups, a.causal = causal;
  a.workgroups = s.workgroups;
  if (s.workgroups) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + s.part_o;
    a.arrived = counters;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  (row_type == KV_F32 ? pa_run_f32 : row_type == KV_BF16 ? pa_run_bf16 : pa_run_f16)(a, s.tiles, (unsigned)(s.workgroups ? s.workgroups : s.units), st);
  PVSG_LAUNCH_CHECK("pvsg_paged_attention");
  return PVSG_OK;
}
