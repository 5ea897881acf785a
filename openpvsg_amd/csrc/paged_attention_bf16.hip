// bf16 rows (paged_attention.h)
#include "paged_attention.h"

void pvsg::pa_run_bf16(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream) {
  switch (a.p.type) {
    case KV_BF16: pa_launch<KV_BF16, KV_BF16>(a, tiles, blocks, stream); break;
    case KV_E4M3: pa_launch<KV_BF16, KV_E4M3>(a, tiles, blocks, stream); break;
    default: pa_launch<KV_BF16, KV_I8>(a, tiles, blocks, stream);
  }
}
