// f32 rows (paged_attention.h)
#include "paged_attention.h"

void pvsg::pa_run_f32(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream) {
  switch (a.p.type) {
    case KV_F32: pa_launch<KV_F32, KV_F32>(a, tiles, blocks, stream); break;
    case KV_BF16: pa_launch<KV_F32, KV_BF16>(a, tiles, blocks, stream); break;
    case KV_F16: pa_launch<KV_F32, KV_F16>(a, tiles, blocks, stream); break;
    case KV_E4M3: pa_launch<KV_F32, KV_E4M3>(a, tiles, blocks, stream); break;
    default: pa_launch<KV_F32, KV_I8>(a, tiles, blocks, stream);
  }
}
