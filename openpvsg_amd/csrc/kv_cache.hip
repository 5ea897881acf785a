// Writing a paged key/value pool (quantising on the way) and reading it back dense.
//
// Both are one pass over the rows and bound by memory: a row is 2 * dim elements in one type in, the same in another out, and
// a scale.  A lane holds 8 elements of a row's K and of its V, so a row is next_pow2(dim/8) lanes: 16 at dim 128, four rows to a
// wave, and the row's maximum needs log2 of that in lane exchanges and no LDS.  The 8 elements are one run, or where one side is f32
// two runs of 4, a row's lanes apart: every access is then dense over the lanes.
//
// Measured: 16 x 4096 rows of 8 x 128 bf16 into int8 86.9 us, 4.7 TB/s (a copy of as many bytes: 5.0-5.3); 100 histories of up to 900 rows
// of 4 x 128 bf16 read back as f32 88.5 us, 5.2 TB/s; 100 x 1 row of 4 x 128 f32 into bf16 2.9 us, the latency of lens -> page id -> store.
#include "kv_pages.h"

namespace pvsg {

int kv_check_pages(const char* who, const pvsg_kv_pages* p, const int* table, long long table_stride, int table_width, const int* lens, int B) {
  PVSG_REQUIRE(p && p->k && p->v && table && lens, "%s: null pointer", who);
  PVSG_REQUIRE(p->type >= KV_F32 && p->type <= KV_I8, "%s: pool type %d", who, p->type);
  PVSG_REQUIRE(p->num_pages > 0 && p->heads > 0 && p->heads <= 65535, "%s: %d pages, %d heads", who, p->num_pages, p->heads);
  PVSG_REQUIRE(p->page_size >= 8 && p->page_size <= 65536 && (p->page_size & (p->page_size - 1)) == 0, "%s: page_size %d is no power of two in [8, 65536]", who, p->page_size);
  PVSG_REQUIRE(p->dim >= 16 && p->dim <= 256 && p->dim % 16 == 0, "%s: dim %d is no multiple of 16 up to 256", who, p->dim);
  const long long unit = 16 / kv_bytes(p->type);
  PVSG_REQUIRE(p->page_stride % unit == 0 && p->head_stride % unit == 0 && p->slot_stride % unit == 0 && (((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0,
               "%s: the pool's rows are not 16-byte aligned", who);
  PVSG_REQUIRE(p->page_stride >= 0 && p->head_stride >= 0 && p->slot_stride >= p->dim, "%s: bad pool strides", who);
  if (kv_scaled(p->type)) {
    PVSG_REQUIRE(p->k_scale && p->v_scale, "%s: an 8-bit pool needs its scales", who);
    PVSG_REQUIRE(p->scale_page_stride % 4 == 0 && p->scale_head_stride % 4 == 0 && (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 15) == 0,
                 "%s: the scales are not 16-byte aligned", who);
  }
  PVSG_REQUIRE(B >= 0 && B <= 65535, "%s: %d sequences (at most 65535)", who, B);
  PVSG_REQUIRE(table_width > 0 && table_stride >= 0 && (long long)table_width * p->page_size <= (1ll << 30), "%s: table of %d pages of %d (positions stay below 2^30)", who,
               table_width, p->page_size);
  return PVSG_OK;
}

struct KvAppend {
  pvsg_kv_pages p;
  const unsigned char *k, *v;
  long long seq_stride, token_stride, head_stride;   // bytes
  const int* table;
  long long table_stride;
  const int *lens, *new_lens;
  int width, T, page_shift, lanes_shift, run_shift;
};

constexpr float KV_TINY = 1.17549435e-38f;           // 2^-126: keeps x / s finite where the row is all zeros or denormal

// x / s for the numbers of a row, correctly rounded: a multiplication by 1/s alone would put values that lie next to a border
// between two codes on its other side.  With y = 1/s correctly rounded, each step q + (x - q s) y takes a q a few units in the last
// place off to one half off, and the second one to the nearest (Markstein's theorem: y the nearest to 1/s, q within one unit, the
// remainder exact by fma).  Five operations, where the division's own sequence takes about ten (measured: 100 -> 89 us for
// 16 x 4096 rows of 8 x 128 bf16 into int8).  Over- and underflow cannot come between: 2^-126 <= s <= 2^128 / 127 and |x / s| <= 448 (1 +
// 2^-22), and a q below the normal range is code 0 either way.
struct KvScale {
  float s, y;
  bool odd;                              // a row of the wave whose scale is no finite number: the division itself
};
__device__ __forceinline__ float kv_quotient(float x, const KvScale& k) {
  if (k.odd) return x / k.s;
  float q = x * k.y;
  q = __builtin_fmaf(__builtin_fmaf(-q, k.s, x), k.y, q);
  return __builtin_fmaf(__builtin_fmaf(-q, k.s, x), k.y, q);
}

// eight f32 -> the row's stored words
template <int CT>
__device__ __forceinline__ void kv_encode8(const float* x, const KvScale& k, unsigned* w) {
  if constexpr (CT == KV_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __builtin_bit_cast(unsigned, x[i]);
  } else if constexpr (CT == KV_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = kv_pack_bf16(x[2 * i], x[2 * i + 1]);
  } else if constexpr (CT == KV_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = kv_pack_f16(x[2 * i], x[2 * i + 1]);
  } else {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = kv_quotient(x[i], k);
    if constexpr (CT == KV_E4M3) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], lo, true);
      }
    } else {
      // |q| <= 127 (1 + 2^-22): added to 1.5 * 2^23 it is rounded to a whole number, ties to even, whose low byte is the code.
      // In a row with a NaN or infinity q is 0 or NaN; a NaN is made 0 first, and the row's scale reads it back as NaN.
      unsigned u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = __builtin_bit_cast(unsigned, (k.odd && q[i] != q[i] ? 0.f : q[i]) + 12582912.f);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x0c0c0400u), __builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0400u), 0x05040100u);
    }
  }
}

constexpr int kv_run(int row_type, int pool_type) { return row_type == KV_F32 || pool_type == KV_F32 ? 4 : 8; }

// this lane's 8 elements of a row that starts at `row`, dim of them in all
template <int TYPE, int RUN>
__device__ __forceinline__ void kv_load_run(unsigned (&w)[kv_bytes(TYPE) * 2], const unsigned char* row, int sub, int lanes, int dim) {
#pragma unroll
  for (int i = 0; i < 8 / RUN; ++i) {
    const int d = RUN * (sub + i * lanes);
    if (d < dim) kv_load_once<RUN * kv_bytes(TYPE)>(&w[i * RUN * kv_bytes(TYPE) / 4], row + d * kv_bytes(TYPE));
  }
}
template <int TYPE, int RUN, bool ONCE>
__device__ __forceinline__ void kv_store_run(unsigned char* row, const unsigned (&w)[kv_bytes(TYPE) * 2], int sub, int lanes, int dim) {
#pragma unroll
  for (int i = 0; i < 8 / RUN; ++i) {
    const int d = RUN * (sub + i * lanes);
    if (d < dim) kv_store<RUN * kv_bytes(TYPE), ONCE>(row + d * kv_bytes(TYPE), &w[i * RUN * kv_bytes(TYPE) / 4]);
  }
}

template <int RT, int CT>
__device__ __forceinline__ void kv_append_row(const unsigned (&raw)[kv_bytes(RT) * 2], unsigned char* dst, float* scale, int sub, int lanes, int dim, bool live) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = kv_elem<RT>(raw, i);
  KvScale k = {1.f, 1.f, false};
  if constexpr (kv_scaled(CT)) {
    // the maximum of the magnitudes' bits: a NaN is above infinity is above every number, so a row that holds one has a scale
    // of NaN or infinity
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu);
    for (int o = lanes >> 1; o >= 1; o >>= 1) a = max(a, (unsigned)__shfl_xor((int)a, o));
    const float m = __builtin_bit_cast(float, a);
    k.s = m * (CT == KV_E4M3 ? 1.f / 448.f : 1.f / 127.f);
    k.s = k.s < KV_TINY ? KV_TINY : k.s;               // a NaN stays
    k.y = 1.f / k.s;
    k.odd = __any(!(k.s < INFINITY));
    if (live && sub == 0) *scale = k.s;
  }
  unsigned w[kv_bytes(CT) * 2];
  kv_encode8<CT>(x, k, w);
  if (live) kv_store_run<CT, kv_run(RT, CT), false>(dst, w, sub, lanes, dim);
}

template <int RT, int CT>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppend a) {
  constexpr int RB = kv_bytes(RT), CB = kv_bytes(CT);
  const int b = blockIdx.y;
  const int lanes = 1 << a.lanes_shift;
  const int sub = threadIdx.x & (lanes - 1);
  // runs of 2^run_shift tokens of one head, so that a workgroup's scales lie together: 4-byte pieces of one line from many
  // workgroups, each behind another L2, cost as much as the codes (measured at 16 x 4096 rows into int8: 93 -> 86 us)
  const unsigned r = (blockIdx.x << (8 - a.lanes_shift)) + (threadIdx.x >> a.lanes_shift), run = r >> a.run_shift;
  const unsigned t = ((run / a.p.heads) << a.run_shift) + (r & ((1u << a.run_shift) - 1)), h = run % a.p.heads;
  // the rows are asked for before the lengths and the page id are there: a row that turns out not to be real is not written
  unsigned kr[RB * 2] = {}, vr[RB * 2] = {};
  if ((int)t < a.T) {
    const long long src = b * a.seq_stride + (long long)t * a.token_stride + (long long)h * a.head_stride;
    kv_load_run<RT, kv_run(RT, CT)>(kr, a.k + src, sub, lanes, a.p.dim);
    kv_load_run<RT, kv_run(RT, CT)>(vr, a.v + src, sub, lanes, a.p.dim);
  }
  const KvSpan span = kv_span(a.lens, a.new_lens, b, a.T, a.width << a.page_shift);
  bool live = (int)t < span.fresh;
  const int pos = live ? span.len - span.fresh + (int)t : 0;
  int page = 0;
  if (live) {
    page = pos < span.there ? a.table[(long long)b * a.table_stride + (pos >> a.page_shift)] : -1;
    if ((unsigned)page >= (unsigned)a.p.num_pages) {
      live = false;
      page = 0;
      if (sub == 0) kv_fault(a.p.faults, 1);
    }
  }
  const int slot = pos & (a.p.page_size - 1);
  const long long dst = ((long long)page * a.p.page_stride + (long long)h * a.p.head_stride + (long long)slot * a.p.slot_stride) * CB;
  const long long sc = (long long)page * a.p.scale_page_stride + (long long)h * a.p.scale_head_stride + slot;
  kv_append_row<RT, CT>(kr, static_cast<unsigned char*>(a.p.k) + dst, a.p.k_scale + sc, sub, lanes, a.p.dim, live);
  kv_append_row<RT, CT>(vr, static_cast<unsigned char*>(a.p.v) + dst, a.p.v_scale + sc, sub, lanes, a.p.dim, live);
}

struct KvRead {
  pvsg_kv_pages p;
  unsigned char *k, *v;
  const int* table;
  long long table_stride;
  const int* lens;
  int width, start, length, page_shift, lanes_shift;
};

template <int RT, int CT>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvRead a) {
  constexpr int RB = kv_bytes(RT), CB = kv_bytes(CT), RUN = kv_run(RT, CT);
  const int b = blockIdx.y;
  const int lanes = 1 << a.lanes_shift, sub = threadIdx.x & (lanes - 1);
  const unsigned r = (blockIdx.x << (8 - a.lanes_shift)) + (threadIdx.x >> a.lanes_shift), t = r / a.p.heads, h = r % a.p.heads;
  if ((int)t >= a.length) return;
  const KvSpan span = kv_span(a.lens, nullptr, b, 0, a.width << a.page_shift);
  const long long pos = a.start + (long long)t;
  unsigned kw[CB * 2] = {}, vw[CB * 2] = {};
  float ks = 0.f, vs = 0.f;
  if (pos < span.len) {
    const int page = pos < span.there ? a.table[(long long)b * a.table_stride + (pos >> a.page_shift)] : -1;
    if ((unsigned)page < (unsigned)a.p.num_pages) {
      const int slot = (int)pos & (a.p.page_size - 1);
      const long long src = ((long long)page * a.p.page_stride + (long long)h * a.p.head_stride + (long long)slot * a.p.slot_stride) * CB;
      kv_load_run<CT, RUN>(kw, static_cast<const unsigned char*>(a.p.k) + src, sub, lanes, a.p.dim);
      kv_load_run<CT, RUN>(vw, static_cast<const unsigned char*>(a.p.v) + src, sub, lanes, a.p.dim);
      if constexpr (kv_scaled(CT)) {
        const long long sc = (long long)page * a.p.scale_page_stride + (long long)h * a.p.scale_head_stride + slot;
        ks = a.p.k_scale[sc], vs = a.p.v_scale[sc];
      }
    } else if (sub == 0) {
      kv_fault(a.p.faults, 2);
    }
  }
  const long long dst = ((long long)b * a.length * a.p.heads + r) * a.p.dim * RB;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const unsigned* w = which ? vw : kw;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = kv_elem<CT>(w, i);
      if constexpr (kv_scaled(CT)) x[i] *= which ? vs : ks;
    }
    unsigned o[RB * 2];
    kv_encode8<RT>(x, KvScale{1.f, 1.f, false}, o);
    kv_store_run<RT, RUN, true>((which ? a.v : a.k) + dst, o, sub, lanes, a.p.dim);
  }
}

static int kv_log2(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

template <int RT, int CT, class A>
static void kv_launch(const A& a, dim3 grid, hipStream_t stream) {
  if constexpr (__is_same(A, KvAppend)) {
    hipLaunchKernelGGL((kv_append_kernel<RT, CT>), grid, dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((kv_read_kernel<RT, CT>), grid, dim3(256), 0, stream, a);
  }
}
template <int RT, class A>
static void kv_launch(const A& a, dim3 grid, hipStream_t stream) {
  switch (a.p.type) {
    case KV_F32: kv_launch<RT, KV_F32>(a, grid, stream); break;
    case KV_BF16: kv_launch<RT, KV_BF16>(a, grid, stream); break;
    case KV_F16: kv_launch<RT, KV_F16>(a, grid, stream); break;
    case KV_E4M3: kv_launch<RT, KV_E4M3>(a, grid, stream); break;
    default: kv_launch<RT, KV_I8>(a, grid, stream);
  }
}
template <class A>
static void kv_launch(int row_type, const A& a, dim3 grid, hipStream_t stream) {
  switch (row_type) {
    case KV_F32: kv_launch<KV_F32>(a, grid, stream); break;
    case KV_BF16: kv_launch<KV_BF16>(a, grid, stream); break;
    default: kv_launch<KV_F16>(a, grid, stream);
  }
}

}  // namespace pvsg

extern "C" int pvsg_kv_append(const pvsg_kv_pages* pages, const void* k, const void* v, int row_type, long long seq_stride,
                              long long token_stride, long long head_stride, const int* table, long long table_stride, int table_width,
                              const int* lens, const int* new_lens, int B, int T, void* stream) {
  using namespace pvsg;
  if (const int rc = kv_check_pages("pvsg_kv_append", pages, table, table_stride, table_width, lens, B)) return rc;
  PVSG_REQUIRE(k && v, "pvsg_kv_append: null pointer");
  PVSG_REQUIRE(row_type >= KV_F32 && row_type <= KV_F16, "pvsg_kv_append: row type %d", row_type);
  const long long rb = kv_bytes(row_type);
  PVSG_REQUIRE(((seq_stride | token_stride | head_stride) * rb) % 16 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, "pvsg_kv_append: rows are not 16-byte aligned");
  PVSG_REQUIRE(T >= 0, "pvsg_kv_append: %d tokens", T);
  if (B == 0 || T == 0) return PVSG_OK;
  KvAppend a{*pages, static_cast<const unsigned char*>(k), static_cast<const unsigned char*>(v), seq_stride * rb, token_stride * rb, head_stride * rb,
             table, table_stride, lens, new_lens, table_width, T, kv_log2(pages->page_size), kv_log2(pages->dim / 8), 0};
  while ((2 << a.run_shift) <= T && a.run_shift < 8 - a.lanes_shift) ++a.run_shift;
  const long long rows = (((long long)T + (1 << a.run_shift) - 1) >> a.run_shift << a.run_shift) * pages->heads, blocks = ((rows << a.lanes_shift) + 255) / 256;
  PVSG_REQUIRE(rows < (1ll << 31) - 256 && blocks < KV_MAX_BLOCKS, "pvsg_kv_append: %d tokens of %d heads are too many for one launch", T, pages->heads);
  kv_launch(row_type, a, dim3((unsigned)blocks, (unsigned)B), static_cast<hipStream_t>(stream));
  PVSG_LAUNCH_CHECK("pvsg_kv_append");
  return PVSG_OK;
}

extern "C" int pvsg_kv_read(const pvsg_kv_pages* pages, void* k_out, void* v_out, int out_type, const int* table, long long table_stride,
                            int table_width, const int* lens, int B, int start, int length, void* stream) {
  using namespace pvsg;
  if (const int rc = kv_check_pages("pvsg_kv_read", pages, table, table_stride, table_width, lens, B)) return rc;
  PVSG_REQUIRE(k_out && v_out && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "pvsg_kv_read: null or misaligned output");
  PVSG_REQUIRE(out_type >= KV_F32 && out_type <= KV_F16, "pvsg_kv_read: output type %d", out_type);
  PVSG_REQUIRE(start >= 0 && length >= 0, "pvsg_kv_read: positions %d + %d", start, length);
  if (B == 0 || length == 0) return PVSG_OK;
  KvRead a{*pages, static_cast<unsigned char*>(k_out), static_cast<unsigned char*>(v_out), table, table_stride, lens, table_width, start, length,
           kv_log2(pages->page_size), kv_log2(pages->dim / 8)};
  const long long rows = (long long)length * pages->heads, blocks = ((rows << a.lanes_shift) + 255) / 256;
  PVSG_REQUIRE(rows < (1ll << 31) - 256 && blocks < KV_MAX_BLOCKS, "pvsg_kv_read: %d positions of %d heads are too many for one launch", length, pages->heads);
  kv_launch(out_type, a, dim3((unsigned)blocks, (unsigned)B), static_cast<hipStream_t>(stream));
  PVSG_LAUNCH_CHECK("pvsg_kv_read");
  return PVSG_OK;
}
