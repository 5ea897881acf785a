// Entry points of the paged attention (paged_attention.h has the kernel and its reasons) and the join of its splits.
#include "paged_attention.h"

namespace pvsg {

// The join: one workgroup per query row, dim / 4 threads across a partial and the others down the splits.
template <int RT>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const PagedAttn a) {
  const long long row = blockIdx.x;
  const int b = (int)(row / ((long long)a.T * a.q_heads)), t = (int)(row / a.q_heads % a.T);
  const KvSpan span = kv_span(a.lens, a.new_lens, b, a.T, a.width << a.page_shift);
  const int n = t < span.fresh ? (int)min((long long)a.splits, ((long long)span.there + a.chunk - 1) / a.chunk) : 0;
  const int D = a.p.dim, d4 = D / 4, down = 256 / d4;
  const int x = threadIdx.x % d4, s0 = threadIdx.x / d4;
  const float* ml = a.part_ml + row * a.splits * 2;
  float top = -INFINITY;
  for (int s = threadIdx.x & 63; s < n; s += 64) top = fmaxf(top, ml[2 * s]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (s0 < down) {
    for (int s = s0; s < n; s += down) {
      const float2 p = *reinterpret_cast<const float2*>(ml + 2 * s);
      const float w = __builtin_amdgcn_exp2f(p.x - ref);
      const float4 v = ld4(a.part_o + (row * a.splits + s) * D + 4 * x);
      sum += w * p.y;
      o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
    }
  }
  __shared__ __align__(16) float s_o[256][4];
  __shared__ float s_l[256];
  st4(s_o[threadIdx.x], o);
  s_l[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x < (unsigned)d4) {
    for (int s = 1; s < down; ++s) {
      const float4 v = ld4(s_o[s * d4 + x]);
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
      sum += s_l[s * d4 + x];
    }
    const bool some = !(sum == 0.f);
    const float y[4] = {some ? o.x / sum : 0.f, some ? o.y / sum : 0.f, some ? o.z / sum : 0.f, some ? o.w / sum : 0.f};
    pa_store_row4<RT>(a.out, row * D + 4 * x, y);
  }
}

// 16-row tiles a wave carries: two where there are more rows than one tile holds and the accumulators of two fit
static int pa_tiles(int rows, int dim, int row_type) { return rows > 16 && dim <= (row_type == KV_F32 ? 64 : 128) ? 2 : 1; }

}  // namespace pvsg

extern "C" int pvsg_paged_attention_splits(int B, int T, int q_heads, int kv_heads, int dim, int row_type, long long max_len) {
  using namespace pvsg;
  if (B <= 0 || T <= 0 || kv_heads <= 0 || q_heads < kv_heads || max_len <= 0) return 1;
  const int rows = T * (q_heads / kv_heads), per = 16 * pa_tiles(rows, dim, row_type);
  const long long units = (long long)B * kv_heads * ((rows + per - 1) / per);
  const long long tiles = (max_len + 127) / 128;                    // one 32-key tile for each wave
  long long n = (2048 + units - 1) / units;
  n = n < tiles ? n : tiles;
  return (int)(n < 1 ? 1 : n > 512 ? 512 : n);
}

extern "C" int pvsg_paged_attention(const pvsg_kv_pages* pages, const void* q, long long q_seq_stride, long long q_token_stride,
                                    long long q_head_stride, void* out, int row_type, const int* table, long long table_stride, int table_width,
                                    const int* lens, const int* new_lens, const uint8_t* padding, long long padding_stride, int padding_width,
                                    int B, int T, int q_heads, float scale, int causal, long long max_len, int splits, void* workspace, void* stream) {
  using namespace pvsg;
  if (const int rc = kv_check_pages("pvsg_paged_attention", pages, table, table_stride, table_width, lens, B)) return rc;
  PVSG_REQUIRE(q && out, "pvsg_paged_attention: null pointer");
  PVSG_REQUIRE(row_type >= KV_F32 && row_type <= KV_F16, "pvsg_paged_attention: row type %d", row_type);
  PVSG_REQUIRE(row_type == KV_F32 || row_type == pages->type || kv_scaled(pages->type), "pvsg_paged_attention: rows of type %d over a pool of type %d", row_type, pages->type);
  const long long rb = kv_bytes(row_type);
  PVSG_REQUIRE(((q_seq_stride | q_token_stride | q_head_stride) * rb) % 16 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0, "pvsg_paged_attention: rows are not 16-byte aligned");
  PVSG_REQUIRE(T >= 0 && T <= PA_MAX_T, "pvsg_paged_attention: %d new tokens (at most %d)", T, PA_MAX_T);
  PVSG_REQUIRE(q_heads > 0 && q_heads % pages->heads == 0 && q_heads / pages->heads <= 1024, "pvsg_paged_attention: %d query heads over %d key heads", q_heads, pages->heads);
  PVSG_REQUIRE(splits >= 1 && splits <= 512 && (splits == 1 || (workspace && ((uintptr_t)workspace & 15) == 0)), "pvsg_paged_attention: %d splits, workspace %p", splits, workspace);
  PVSG_REQUIRE(!padding || (padding_width >= 0 && padding_stride >= 0), "pvsg_paged_attention: bad padding mask");
  if (B == 0 || T == 0) return PVSG_OK;
  PagedAttn a{};
  a.p = *pages;
  a.q = static_cast<const unsigned char*>(q), a.out = static_cast<unsigned char*>(out);
  a.table = table, a.lens = lens, a.new_lens = new_lens, a.padding = padding;
  a.q_seq = q_seq_stride * rb, a.q_token = q_token_stride * rb, a.q_head = q_head_stride * rb;
  a.table_stride = table_stride, a.padding_stride = padding_stride;
  a.scale_log2e = scale * 1.44269504088896340736f;
  a.width = table_width, a.padding_width = padding_width;
  while ((1 << a.page_shift) < pages->page_size) ++a.page_shift;
  a.B = B, a.T = T, a.q_heads = q_heads, a.group = q_heads / pages->heads, a.rows = T * a.group, a.splits = splits, a.causal = causal;
  const int tiles = pa_tiles(a.rows, pages->dim, row_type);
  a.row_groups = (a.rows + 16 * tiles - 1) / (16 * tiles);
  const long long capacity = (long long)table_width * pages->page_size;
  const long long longest = max_len > 0 && max_len < capacity ? max_len : capacity;
  const long long share = ((longest + splits - 1) / splits + 127) / 128 * 128;
  a.chunk = (int)(share < PA_MAX_CHUNK ? share : PA_MAX_CHUNK);
  const long long total = (long long)B * T * q_heads;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o ? a.part_o + total * splits * pages->dim : nullptr;
  long long units = (long long)B * pages->heads * splits;
  if (a.row_groups > 1) units = (units + 7) / 8 * 8 * a.row_groups;
  PVSG_REQUIRE(units < (1ll << 31) && total < (1ll << 31), "pvsg_paged_attention: too many rows for one launch");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned blocks = (unsigned)units;
  (row_type == KV_F32 ? pa_run_f32 : row_type == KV_BF16 ? pa_run_bf16 : pa_run_f16)(a, tiles, blocks, st);
  PVSG_LAUNCH_CHECK("pvsg_paged_attention");
  if (splits > 1) {
    if (row_type == KV_F32) hipLaunchKernelGGL((paged_attention_join_kernel<KV_F32>), dim3((unsigned)total), dim3(256), 0, st, a);
    else if (row_type == KV_BF16) hipLaunchKernelGGL((paged_attention_join_kernel<KV_BF16>), dim3((unsigned)total), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attention_join_kernel<KV_F16>), dim3((unsigned)total), dim3(256), 0, st, a);
    PVSG_LAUNCH_CHECK("pvsg_paged_attention");
  }
  return PVSG_OK;
}
