// Entry points of the paged attention (paged_attention.h has the kernel and its reasons).
#include "paged_attention.h"

namespace pvsg {

// Caches of up to so many tiles are not split: each has a workgroup of its own.  Measured over 4 .. 800 (sequence, key head)s of bf16
// heads of 128: at 700 positions (6 tiles) 11.0 - 37.8 us so and 13.5 - 42.8 us split and joined, at 1000 (8) 13.5 - 50 and 13.7 -
// 53.7, at 1500 (12) 17.6 - 70 and 13.5 - 71: the wait for a tile's memory, 1.2 us, is paid once a tile.
constexpr int PA_SHORT = 8;

// 16-row tiles a wave carries: two where there are more rows than one tile holds and the accumulators of two fit
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
