// Attention of 1..32 new tokens per sequence over a paged key/value pool, split over the cache's length and joined.
//
//   o = sum_p softmax(scale * q . k_p) v_p,  one pass over the keys with a running maximum m and sum l per row; 0 where l is 0: a row
//   that sees nothing, or only logits of -infinity (which leave m there).
//
// The T * (q_heads / kv_heads) query rows that share a key head make 16-row tiles.  A wave walks the cache in tiles of KEYS keys and
// feeds the matrix cores straight from global memory, with no LDS between: keys are the A operand of S^T = K Q^T (a lane's part of
// a row is dense in memory), and S^T leaves the pipe with a lane holding 4 keys of one query row -- which is the B operand of
// O^T = V^T P^T as it stands, so P never moves.  For V^T a lane loads the same columns of several keys and pairs them by
// byte permutes (16-bit products take 8 keys a lane; f32 products take one, and need no permutes).  Four waves take every
// fourth tile and meet in LDS at the end.
//
// Sequences differ in length, and only the device knows by how much.  So the tiles of all of them are one list, and as many
// workgroups as the card holds each take an equal stretch of it: each finds its stretch by a scan over the lengths.  A (sequence, key
// head, row group) that lies in several stretches leaves (m, l, O) of each, and whoever comes last joins them, in the stretches' order.  Where
// no cache is longer than a few tiles there is nothing to even out, and each has a workgroup of its own and no join.
//
// Rounding: 16-bit rows multiply in their own type, exact products in f32 sums; 8-bit codes convert to it exactly and their
// scales multiply S and P in f32.  P goes to the matrix cores as three bf16 parts over a bf16 or 8-bit pool (the 24 bits of f32), as two f16
// parts over a f16 one (22, see LIFT).  One part alone adds an error as large as the rounding of the result itself; two of bf16
// hold 16 bits, which shows where values cancel, and save little (100 x up to 5000 x 4 x 128 e4m3, 32 new tokens: 78.7 us, three parts
// 79.8; 64 x 8192 x 8 heads of 64 int8 119.1 and 122.8; 8 x 65536 bf16 361 both).  (P carries the scale of
// V's codes: rows whose scale is below 2^-100 lose bits, since bf16 ends at 2^-133.)  f32 rows over a bf16 or 8-bit pool go as three bf16 parts too.  At
// the matrix cores' peak three 16-bit products take 3/16 of the time that the f32 ones would.  f32 rows over a f32 or f16 pool run on the f32
// products.
//
// Measured: 8 x 65536 x 8 key heads of 128 bf16 360 us, 5.95 TB/s, bound by HBM; 100 ragged caches of up to 900 x 4 x 128 f32 48 us,
// 3.85 TB/s: a stretch takes 5 us to its first keys (lengths, scan, page ids, queries: waits for memory that depend on each other)
// and 4 to be joined and counted, and with two workgroups on a CU that is covered in part; 100 of up to 5000 x 4 x 128 e4m3, 32 new
// tokens, 76 us, 3.6 TB/s, the waves as long in the softmax's instructions as in waits; the smallest call 6.5 us, five such waits.
#pragma once
#include "kv_pages.h"

#include <limits.h>

#include <type_traits>

namespace pvsg {

struct PagedAttn {
  pvsg_kv_pages p;
  const unsigned char* q;
  unsigned char* out;
  const int* table;
  const int *lens, *new_lens;
  const unsigned char* padding;
  float *part_o, *part_ml;
  long long q_seq, q_token, q_head;      // bytes
  long long table_stride, padding_stride;
  float scale_log2e;
  int width, padding_width, page_shift;
  int B, T, q_heads, group, rows, row_groups, causal;
  int workgroups;                        // how many share the tiles; 0: one for each (sequence, key head, row group)
  unsigned* arrived;                     // zeros, one for each: how many parts of a row are there
};

constexpr int PA_WAVES = 4;
constexpr int PA_CHUNK = 4096;           // keys whose pages are looked up at a time
constexpr int PA_GRAIN = 1;               // tiles that a workgroup takes at least
constexpr int PA_MAX_T = 32;

// The kernel reads its arguments where the launch left them, again for each part of its work: held in scalar registers
// throughout, they would push the loop's own values out of those (measured: 130 to 260 of them spilled).
typedef const __attribute__((address_space(4))) PagedAttn PagedAttnArgs;

// device memory that nothing writes while the kernel runs, read at a place that all threads share: by scalar loads
__device__ __forceinline__ const __attribute__((address_space(4))) int* pa_const(const int* p) {
  return (const __attribute__((address_space(4))) int*)p;
}

// whether rows of one type over a pool of another are multiplied in 16 bits
constexpr bool pa_16bit(int row, int pool) { return row != KV_F32 || pool == KV_BF16 || kv_scaled(pool); }
// the size class of a head
constexpr int pa_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// 16-key blocks of a wave's tile.  f32 products take one key at a time, so that a block of theirs is work enough.  Of heads of up to 64
// in 16 bits there is room for four beside the next tile's, and where the caches are long (`split`: the tiles are shared out) they
// save waits for memory: 64 x 8192 x 8 heads of 64 int8 130.9 -> 122.8 us, 20 ragged ones of up to 3000 x 8 bf16 19.9 -> 18.6.  Short ones go two
// blocks at a time, three workgroups to a CU: 100 of up to 900 positions x 8 int8 21.2 us, and 24.7 with four.
constexpr int pa_blocks(int row, int pool, int dim, int tiles, bool split) {
  return pa_16bit(row, pool) ? (split && tiles == 1 && row != KV_F32 && dim <= 64 ? 4 : 2) : dim <= 32 ? 2 : 1;
}
// what a part costs beside its tiles, in tiles (swept 1 .. 5)
constexpr int pa_part_cost(int blocks) { return blocks == 4 ? 1 : 3; }
// workgroups of a CU that the kernel's registers leave room for
constexpr int pa_per_cu(int dim, int tiles, int blocks) { return dim <= 64 ? (tiles == 1 && blocks < 4 ? 3 : 2) : dim <= 128 ? 2 : 1; }

// four packed 16-bit words (the 8 elements of one lane of a matrix product's operand)
template <int MT>
__device__ __forceinline__ f32x4 pa_mfma16(const unsigned (&a)[4], const unsigned (&b)[4], f32x4 c) {
  const kv_u32x4 av = {a[0], a[1], a[2], a[3]}, bv = {b[0], b[1], b[2], b[3]};
  if constexpr (MT == KV_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv_bf16x8, av), __builtin_bit_cast(kv_bf16x8, bv), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv_f16x8, av), __builtin_bit_cast(kv_f16x8, bv), c, 0, 0, 0);
  }
}
template <int MT>
__device__ __forceinline__ unsigned pa_pack(float a, float b) {
  return MT == KV_BF16 ? kv_pack_bf16(a, b) : kv_pack_f16(a, b);
}
template <int MT>
__device__ __forceinline__ float pa_half(unsigned w, int i) {
  return MT == KV_BF16 ? kv_elem<KV_BF16>(&w, i) : kv_elem<KV_F16>(&w, i);
}
// bytes 2i, 2i+1 of an 8-bit word -> a packed 16-bit pair
template <int MT, int CT>
__device__ __forceinline__ unsigned pa_widen(unsigned w, bool hi) {
  if constexpr (CT == KV_E4M3) {
    if constexpr (MT == KV_BF16) {
      return __builtin_bit_cast(unsigned, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
    } else {
      return __builtin_bit_cast(unsigned, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    }
  } else {
    return pa_pack<MT>(kv_elem<KV_I8>(&w, hi ? 2 : 0), kv_elem<KV_I8>(&w, hi ? 3 : 1));
  }
}

// maximum / sum over the four 16-lane groups of a wave, in every lane
__device__ __forceinline__ float pa_max4(float x) {
  // swapping 16-lane rows of x with itself leaves rows 0 0 2 2 of x in one result and 1 1 3 3 in the other; then halves alike
  unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned r0 = r[0], r1 = r[1];
  x = fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
  u = __builtin_bit_cast(unsigned, x);
  const auto q = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned q0 = q[0], q1 = q[1];
  return fmaxf(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}
__device__ __forceinline__ float pa_sum4(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// sum over the lanes up to this one: inside the 16-lane rows by shifts, then the last lane of a row (of two rows) to the next
__device__ __forceinline__ unsigned pa_scan(unsigned x) {
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
  return x;
}

template <int RT>
__device__ __forceinline__ void pa_store_row4(unsigned char* out, long long at, const float (&x)[4]) {
  unsigned w[4];
  if constexpr (RT == KV_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, x[i]);
    kv_store<16>(out + at * 4, w);
  } else {
    w[0] = pa_pack<RT>(x[0], x[1]), w[1] = pa_pack<RT>(x[2], x[3]);
    kv_store<8>(out + at * 2, w);
  }
}

// A part's values go between workgroups of one launch: stored through and read past the caches that other workgroups do not share.
__device__ __forceinline__ float2 pa_get2(const float* p) {
  const unsigned long long u = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__builtin_bit_cast(float, (unsigned)u), __builtin_bit_cast(float, (unsigned)(u >> 32)));
}
__device__ __forceinline__ void pa_put2(float* p, float x, float y) {
  const unsigned long long u = __builtin_bit_cast(unsigned, x) | (unsigned long long)__builtin_bit_cast(unsigned, y) << 32;
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The parts that the stretches of workgroups first .. first + n - 1 left of the `tile_rows` rows at row0 of key head h: joined and written.
// dim / 4 threads across a row; of the groups of so many threads, `share` take one row's parts between them, so that few rows of
// many parts are read at once as well.  The parts come in the stretches' order, whoever joins them.
template <int RT>
__device__ void pa_join(PagedAttnArgs& a, int b, int h, int row0, int tile_rows, int first, int n, int fresh, float (*s_o)[4], float* s_m, float* s_l) {
  const int rows = min(tile_rows, a.rows - row0);
  const int D = a.p.dim, d4 = D / 4, groups = 256 / d4, x = threadIdx.x % d4, y = threadIdx.x / d4;
  const int share = max(1, min(groups / rows, n / 2)), at_once = groups / share;
  for (int r0 = 0; r0 < rows; r0 += at_once) {
    const int r = r0 + y / share, k0 = y % share;
    const bool mine = y < at_once * share && r < rows;
    // part k: what the first stretch left at its end, then what each later one left at its beginning
    float top = -INFINITY, sum = 0.f, o[4] = {};
    if (mine) {
#pragma unroll 4
      for (int k = k0; k < n; k += share) {
        const long long slot = (long long)(2 * (first + k) + (k == 0 ? 1 : 0)) * tile_rows + r;
        const float2 p = pa_get2(a.part_ml + 2 * slot);
        const float2 v = pa_get2(a.part_o + slot * D + 4 * x), u = pa_get2(a.part_o + slot * D + 4 * x + 2);
        const float up = fmaxf(top, p.x), ref = up == -INFINITY ? 0.f : up;
        const float keep = __builtin_amdgcn_exp2f(top - ref), w = __builtin_amdgcn_exp2f(p.x - ref);
        sum = sum * keep + w * p.y;
        o[0] = o[0] * keep + w * v.x, o[1] = o[1] * keep + w * v.y, o[2] = o[2] * keep + w * u.x, o[3] = o[3] * keep + w * u.y;
        top = up;
      }
    }
    if (share > 1) {
      __syncthreads();
      st4(s_o[threadIdx.x], make_float4(o[0], o[1], o[2], o[3]));
      s_m[threadIdx.x] = top, s_l[threadIdx.x] = sum;
      __syncthreads();
      if (mine && k0 == 0) {
        float up = top;
        for (int s = 1; s < share; ++s) up = fmaxf(up, s_m[threadIdx.x + s * d4]);
        const float ref = up == -INFINITY ? 0.f : up, keep = __builtin_amdgcn_exp2f(top - ref);
        sum *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= keep;
        for (int s = 1; s < share; ++s) {
          const float w = __builtin_amdgcn_exp2f(s_m[threadIdx.x + s * d4] - ref);
          const float4 v = ld4(s_o[threadIdx.x + s * d4]);
          sum += w * s_l[threadIdx.x + s * d4];
          o[0] += w * v.x, o[1] += w * v.y, o[2] += w * v.z, o[3] += w * v.w;
        }
      }
    }
    if (mine && k0 == 0) {
      const int t = (row0 + r) / a.group;
      const bool some = t < fresh && !(sum == 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = some ? o[i] / sum : 0.f;
      pa_store_row4<RT>(a.out, (((long long)b * a.T + t) * a.q_heads + h * a.group + (row0 + r) % a.group) * D + 4 * x, o);
    }
  }
}

// Rows r0 .. r1-1 of one (sequence, key head) over the keys lo .. hi-1, by plain sums, a key at a time: the fallback for values that are
// not finite.  buf: 3 * 256 floats of LDS; part_o / part_ml: where a part goes, null for the result itself.
template <int RT, int CT>
__device__ void pa_rows_alone(PagedAttnArgs& a, int b, int h, int lo, int hi, int r0, int r1, const KvSpan& span, float* part_o, float* part_ml, float* buf) {
  const int tid = threadIdx.x, D = a.p.dim;
  int* page_of = reinterpret_cast<int*>(buf);                       // -1: not seen
  float *z_of = buf + 256, *w_of = buf + 512;
  const int dq = min(tid, D - 1);                                   // this thread's column
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const int t = r / a.group, hq = h * a.group + r % a.group;
    const int lim = t >= span.fresh ? 0 : min(hi, a.causal ? min(span.len - span.fresh + t + 1, span.there) : span.there);
    const unsigned char* qr = a.q + b * a.q_seq + t * a.q_token + (long long)hq * a.q_head;
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll 1
    for (int p0 = lo; p0 < lim; p0 += 256) {
      const int p = p0 + tid;
      int page = -1;
      if (p < lim && (!a.padding || (p < a.padding_width && !a.padding[(long long)b * a.padding_stride + p]))) {
        page = a.table[(long long)b * a.table_stride + (p >> a.page_shift)];
        if ((unsigned)page >= (unsigned)a.p.num_pages) page = -1;
      }
      const int slot = p & (a.p.page_size - 1);
      float z = -INFINITY;
      if (page >= 0) {
        const long long at = (long long)page * a.p.page_stride + (long long)h * a.p.head_stride + (long long)slot * a.p.slot_stride;
        z = 0.f;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {
          unsigned kw[8], qw[8];
          kv_load<kv_bytes(CT) == 4 ? 16 : kv_bytes(CT) * 8>(kw, static_cast<const unsigned char*>(a.p.k) + (at + d) * kv_bytes(CT));
          if constexpr (kv_bytes(CT) == 4) kv_load<16>(kw + 4, static_cast<const unsigned char*>(a.p.k) + (at + d) * 4 + 16);
          kv_load<16>(qw, qr + d * kv_bytes(RT));
          if constexpr (kv_bytes(RT) == 4) kv_load<16>(qw + 4, qr + d * 4 + 16);
#pragma unroll
          for (int i = 0; i < 8; ++i) z += kv_elem<RT>(qw, i) * kv_elem<CT>(kw, i);
        }
        z *= a.scale_log2e;
        if constexpr (kv_scaled(CT)) z *= a.p.k_scale[(long long)page * a.p.scale_page_stride + (long long)h * a.p.scale_head_stride + slot];
      }
      __syncthreads();                                            // the last block's lists have been read
      page_of[tid] = page;
      z_of[tid] = z;
      __syncthreads();
      float up = top;
#pragma unroll 4
      for (int i = 0; i < 256; ++i) up = fmaxf(up, z_of[i]);
      const float ref = up == -INFINITY ? 0.f : up;
      const float shrink = __builtin_amdgcn_exp2f(top - ref);
      top = up;
      w_of[tid] = page < 0 ? 0.f : __builtin_amdgcn_exp2f(z - ref);
      __syncthreads();
      // (before anything was seen o and sum are 0, and shrink is 0 or 1)
      o *= shrink, sum *= shrink;
#pragma unroll 1
      for (int i = 0; i < min(256, lim - p0); ++i) {
        if (page_of[i] < 0) continue;
        const int si = (p0 + i) & (a.p.page_size - 1);
        const long long at = (long long)page_of[i] * a.p.page_stride + (long long)h * a.p.head_stride + (long long)si * a.p.slot_stride + dq;
        const unsigned char* src = static_cast<const unsigned char*>(a.p.v) + at * kv_bytes(CT);
        unsigned w[1];
        if constexpr (kv_bytes(CT) == 4) w[0] = *reinterpret_cast<const unsigned*>(src);
        else if constexpr (kv_bytes(CT) == 2) w[0] = *reinterpret_cast<const unsigned short*>(src);
        else w[0] = *src;
        float pv = w_of[i];
        sum += pv;
        if constexpr (kv_scaled(CT)) pv *= a.p.v_scale[(long long)page_of[i] * a.p.scale_page_stride + (long long)h * a.p.scale_head_stride + si];
        o += pv * kv_elem<CT>(w, 0);
      }
    }
    const long long row = ((long long)b * a.T + t) * a.q_heads + hq;
    if (tid < D) {
      if (part_o) {
        __hip_atomic_store(&part_o[(r - r0) * D + tid], o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0) pa_put2(part_ml + (r - r0) * 2, top, sum);
      } else {
        const float y = sum == 0.f ? 0.f : o / sum;
        if constexpr (RT == KV_F32) reinterpret_cast<float*>(a.out)[row * D + tid] = y;
        else reinterpret_cast<unsigned short*>(a.out)[row * D + tid] = (unsigned short)pa_pack<RT>(y, 0.f);
      }
    }
  }
}

// 16-bit parts that a f32 value is multiplied in: 3 of bf16 hold all its 24 bits
template <int PARTS, int MT>
__device__ __forceinline__ void pa_parts(float a, float b, unsigned (&w)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    w[i] = pa_pack<MT>(a, b);
    a -= pa_half<MT>(w[i], 0), b -= pa_half<MT>(w[i], 1);
  }
}

template <int RT, int CT, int DP, int NT, int KT, bool PADDED>
__global__ __launch_bounds__(64 * PA_WAVES, pa_per_cu(DP, NT, KT)) void paged_attention_kernel(const PagedAttn) {
  constexpr bool M16 = pa_16bit(RT, CT);
  constexpr int QK = RT == KV_F16 ? KV_F16 : KV_BF16, PV = CT == KV_F16 ? KV_F16 : KV_BF16;      // operand types of the 16-bit products
  constexpr int QL = RT == KV_F32 ? 3 : 1, PL = PV == KV_BF16 ? 3 : 2;
  constexpr int CB = kv_bytes(CT), RB = kv_bytes(RT);
  constexpr int KEYS = 16 * KT, PA_PART = pa_part_cost(KT);           // a wave's tile is KT blocks of 16 keys
  // keys: chunk i of a lane in 16-lane group g is columns i*4*KC + KC*g ...; values: column c*16*VC + VC*m + e for lane m
  constexpr int KC = 16 / CB < DP / 4 ? 16 / CB : DP / 4, NK = DP / (4 * KC), KW = KC * CB / 4;
  constexpr int VE = DP / 16, VC = 16 / CB < VE ? 16 / CB : VE, NV = VE / VC, VB = VC * CB, VW = (VB + 3) / 4;
  constexpr int QN = M16 ? DP / 32 : DP / 4;                        // steps of 8 packed columns, or single columns
  // f16 has no normal numbers below 2^-14 and nothing below 2^-25, and weights there count where the largest one's value does not.
  // So m is held 15 below the maximum: weights of up to 2^15, whose two f16 parts hold 22 bits down to 2^-29 of the largest one and
  // 2^-40 of it below.  O and l have the same factor, and (m, l, O) mean what they do without it.  (Maxima so large that their
  // f32 is not exact to a few units can make a weight infinite: such rows are computed again.)
  constexpr float LIFT = M16 && PV == KV_F16 ? 15.f : 0.f;
  static_assert(!M16 || KC % 8 == 0, "16-bit products take 8 columns a lane");

  __shared__ int s_page[PA_CHUNK / 8 + 1];
  __shared__ __align__(16) unsigned char s_hide[PADDED ? PA_CHUNK : 16];
  constexpr int OR = DP == 256 ? 8 : 16;                            // rows of a wave in LDS at a time
  __shared__ __align__(16) float s_o[PA_WAVES][OR][DP + 4];
  __shared__ float s_ml[PA_WAVES][16][2];

  constexpr int TILE = PA_WAVES * KEYS;
  PagedAttnArgs* args = (PagedAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  auto tiles_of = [](int len, int capacity) { return max((min(max(len, 0), capacity) + TILE - 1) / TILE, 1); };   // one at least, which writes the zeros

  // ---- this workgroup's stretch.  The list: for each sequence its (key head, row group)s one after the other, each of them PA_PART
  // entries that stand for what a part costs beside its tiles, then its tiles.  hr: the first one of sequence b that the stretch
  // meets, `at` the entry of it where the stretch begins, `left` how many entries it has.
  int b, hr, at, left, len;
  unsigned share = 0, more = 0, first = 0;                          // workgroup i takes `share` entries, and one more if i < more; the next of this one's
  const int each = args->p.heads * args->row_groups;
  if (PagedAttnArgs& a = *args; a.workgroups == 0) {
    b = blockIdx.x / each, hr = blockIdx.x % each, at = 0;
    len = pa_const(a.lens)[b];
    left = INT_MAX;
  } else {
    // every wave scans the lengths by itself: 64 lanes, `per` sequences each, the first four of them in registers
    const int lane = threadIdx.x & 63, per = (a.B + 63) / 64, b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B), capacity = a.width << a.page_shift;
    auto entries = [&](int n) { return (unsigned)(PA_PART + tiles_of(n, capacity)); };
    int lens[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) lens[k] = b0 + k < b1 ? a.lens[b0 + k] : 0;
    unsigned mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += b0 + k < b1 ? entries(lens[k]) : 0;
#pragma unroll 8
    for (int i = b0 + 4; i < b1; ++i) mine += entries(a.lens[i]);
    mine *= each;
    const unsigned upto = pa_scan(mine);
    const unsigned total = __builtin_amdgcn_readlane(upto, 63);
    const unsigned used = min((unsigned)a.workgroups, (total + PA_PART + PA_GRAIN - 1) / (PA_PART + PA_GRAIN));
    share = total / used, more = total - share * used;
    first = blockIdx.x * share + min(blockIdx.x, more);
    if (blockIdx.x >= used) return;
    left = share + (blockIdx.x < more ? 1 : 0);
    const int whose = __builtin_ctzll(__ballot(first < upto));      // the lane whose sequences the stretch begins in
    unsigned inside;
    if (per <= 4) {
      unsigned before = upto - mine;
      b = b0, len = lens[0];
      bool found = false;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const unsigned n = entries(lens[k]) * each;
        found |= b0 + k >= b1 - 1 || first < before + n;
        if (!found) before += n, b = b0 + k + 1, len = lens[k + 1];
      }
      b = __builtin_amdgcn_readlane(b, whose), len = __builtin_amdgcn_readlane(len, whose);
      inside = first - __builtin_amdgcn_readlane(before, whose);
    } else {
      // that lane's sequences, 64 at a time
      unsigned before = __builtin_amdgcn_readlane(upto - mine, whose);
      const int end = min((whose + 1) * per, a.B);
      for (b = whose * per;; b += 64) {
        const int mine_len = b + lane < end ? a.lens[b + lane] : 0;
        const unsigned n = b + lane < end ? entries(mine_len) * each : 0, sum = pa_scan(n);
        const unsigned long long here = __ballot(first < before + sum);
        if (here) {                                                 // (in the last 64 at the latest)
          const int l = __builtin_ctzll(here);
          b += l, len = __builtin_amdgcn_readlane(mine_len, l), inside = first - before - __builtin_amdgcn_readlane(sum - n, l);
          break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        if (b + 64 >= end) return;                                  // never: the lane's sequences hold `first`
      }
    }
    const unsigned n = PA_PART + tiles_of(len, capacity);
    hr = inside / n, at = inside - hr * n;
  }

#pragma unroll 1
  for (bool next_b = false; left > 0; at = 0, next_b = ++hr == each, b += next_b, hr = next_b ? 0 : hr) {
    int tid = threadIdx.x;
    asm volatile("" : "+s"(args), "+v"(tid));                        // (nothing made of these is kept from part to part)
    PagedAttnArgs& a = *args;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
    const int D = a.p.dim, page_mask = a.p.page_size - 1, capacity = a.width << a.page_shift;
    if (next_b) len = pa_const(a.lens)[b];
    const int tiles = tiles_of(len, capacity);
    int tile0 = 0, tile1 = tiles, first_wg = 0, last_wg = 0;          // workgroups that have the first and the last of the tiles
    if (a.workgroups) {
      const int end = min(PA_PART + tiles, at + left);
      tile0 = max(at - PA_PART, 0), tile1 = max(end - PA_PART, 0);
      const unsigned from = first - at;                             // where the row begins in the list
      left -= end - at, first += end - at;
      if (tile0 == tile1) continue;
      if (tile0 != 0 || tile1 != tiles) {
        auto holder = [&](unsigned entry) { return entry < more * (share + 1) ? entry / (share + 1) : more + (entry - more * (share + 1)) / share; };
        first_wg = holder(from + PA_PART), last_wg = holder(from + PA_PART + tiles - 1);
      }
    } else {
      left = 0;
    }
    float *part_o = nullptr, *part_ml = nullptr;
    if (tile0 != 0 || tile1 != tiles) {
      // a stretch has one part at most that begins inside a row's tiles and one that only ends inside
      const int slot = 2 * blockIdx.x + (tile0 == 0 ? 1 : 0);
      part_o = a.part_o + (long long)slot * (16 * NT) * D;
      part_ml = a.part_ml + (long long)slot * (16 * NT) * 2;
    }
    const int h = hr / a.row_groups, row0 = hr % a.row_groups * (16 * NT);
    const int fresh = a.new_lens ? pa_const(a.new_lens)[b] : a.T;

    // what depends on the length alone is asked for first: the page ids of the first keys, two a thread at most
    const int there = min(max(len, 0), capacity), key1 = (int)min((long long)tile1 * TILE, (long long)there);
    auto pages_of = [&](int c0) { return c0 < key1 ? ((min(c0 + PA_CHUNK, key1) - 1) >> a.page_shift) - (c0 >> a.page_shift) + 1 : 0; };
    auto page_at = [&](int c0, int i) { return a.table[(long long)b * a.table_stride + (c0 >> a.page_shift) + i]; };
    constexpr int PAGES = PA_CHUNK / 8 / (64 * PA_WAVES);
    int page_id[PAGES];
#pragma unroll
    for (int i = 0; i < PAGES; ++i) page_id[i] = tid + i * 64 * PA_WAVES < pages_of(tile0 * TILE) ? page_at(tile0 * TILE, tid + i * 64 * PA_WAVES) : 0;

    // query rows, in the operand layout
    unsigned qf[NT][QN * (M16 ? 4 * QL : 1)];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 16 + m, t = r / a.group, j = r % a.group;
      const unsigned char* qr = a.q + b * a.q_seq + t * a.q_token + (long long)(h * a.group + j) * a.q_head;
      constexpr int STEP = M16 ? 8 : 4;
#pragma unroll
      for (int i = 0; i < DP / 4 / STEP; ++i) {
        const int d = (i * STEP / KC) * 4 * KC + KC * g + i * STEP % KC;
        unsigned w[STEP * RB / 4] = {};
        if (r < a.rows && d < D) {
          kv_load<16>(w, qr + d * RB);
          if constexpr (STEP * RB == 32) kv_load<16>(w + 4, qr + d * RB + 16);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if constexpr (M16 && QL > 1) {
            unsigned part[QL];
            pa_parts<QL, QK>(kv_elem<RT>(w, 2 * x), kv_elem<RT>(w, 2 * x + 1), part);
#pragma unroll
            for (int l = 0; l < QL; ++l) qf[nt][(i * QL + l) * 4 + x] = part[l];
          } else {
            qf[nt][i * 4 + x] = w[x];
          }
        }
      }
    }

    const KvSpan span = kv_span_of(len, fresh, a.T, capacity);
    const int past = span.len - span.fresh;
    if (len > capacity && tid == 0) kv_fault(a.p.faults, 4);
    // what the first and the last real row of this group see, and each of this lane's
    const int t_lo = row0 / a.group, t_hi = min((min(row0 + 16 * NT, a.rows) - 1) / a.group, span.fresh - 1);
    const int most = min(t_lo < span.fresh ? (a.causal ? past + t_hi + 1 : there) : 0, key1);
    const int least = a.causal ? min(past + t_lo + 1, there) : there;
    int lim[NT];
    f32x4 acc[NT][VE];
    float mrow[NT], lrow[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 16 + m, t = r / a.group;
      lim[nt] = r >= a.rows || t >= span.fresh ? most : a.causal ? min(past + t + 1, there) : there;
      mrow[nt] = -INFINITY, lrow[nt] = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[nt][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const unsigned char* kbase = static_cast<const unsigned char*>(a.p.k) + (long long)h * a.p.head_stride * CB;
    const unsigned char* vbase = static_cast<const unsigned char*>(a.p.v) + (long long)h * a.p.head_stride * CB;

    // A tile's keys are loaded while the tile before is still in its softmax and its second product, its values while its own
    // first product runs: each goes to the registers that the tile before has just done with, so nothing is held twice.
    unsigned kw[KT][NK * KW], vw[KT * 4][NV * VW];
    unsigned seen = 0;                                                // bit s*4+j: this lane's key 16 s + 4 g + j is there
    float ks[KT][4], vs[KT][4];

    for (int c0 = tile0 * TILE; c0 < most; c0 += PA_CHUNK) {
      const int c1 = min(c0 + PA_CHUNK, most);
      const int first_page = c0 >> a.page_shift, pages = pages_of(c0);
      if (c0 > tile0 * TILE) {
        __syncthreads();                                              // the last keys' pages have been read
#pragma unroll
        for (int i = 0; i < PAGES; ++i) page_id[i] = tid + i * 64 * PA_WAVES < pages ? page_at(c0, tid + i * 64 * PA_WAVES) : 0;
      }
#pragma unroll
      for (int i = 0; i < PAGES; ++i) {
        const bool bad = (unsigned)page_id[i] >= (unsigned)a.p.num_pages;
        if (bad) kv_fault(a.p.faults, 4);
        if (tid + i * 64 * PA_WAVES < pages) s_page[tid + i * 64 * PA_WAVES] = bad ? -1 : page_id[i];
      }
      if constexpr (PADDED) {
        for (int i = tid; i < c1 - c0; i += 64 * PA_WAVES) {
          const int p = c0 + i;
          s_hide[i] = p < a.padding_width && !a.padding[(long long)b * a.padding_stride + p] ? 0 : 1;
        }
      }
      __syncthreads();

      // Keys past the end read their slot of the last page (in the pool, whatever it holds), keys of a bad page that of page 0;
      // neither is seen.
      auto load_k = [&](int k0) {
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          const int p = k0 + 16 * s + m;
          const int page = max(s_page[(min(p, c1 - 1) >> a.page_shift) - first_page], 0);
          const unsigned char* src = kbase + ((long long)page * a.p.page_stride + (long long)(p & page_mask) * a.p.slot_stride) * CB;
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            const int d = i * 4 * KC + KC * g;
            kv_load<KC * CB>(&kw[s][i * KW], src + (d < D ? d : 0) * CB);
          }
        }
      };
      auto load_v = [&](int k0) {
        seen = 0;
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          const int p = k0 + 16 * s + 4 * g;                          // four keys of one page
          const int page = s_page[(min(p, c1 - 1) >> a.page_shift) - first_page], slot = p & page_mask;
          unsigned there = page >= 0 ? (1u << min(max(c1 - p, 0), 4)) - 1u : 0u;
          if constexpr (PADDED) {
            const unsigned x = ~*reinterpret_cast<const unsigned*>(&s_hide[p < c1 ? p - c0 : 0]);
            there &= (x & 1u) | (x >> 7 & 2u) | (x >> 14 & 4u) | (x >> 21 & 8u);
          }
          seen |= there << (4 * s);
          const unsigned char* src = vbase + ((long long)max(page, 0) * a.p.page_stride + (long long)slot * a.p.slot_stride) * CB;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int c = 0; c < NV; ++c) {
              const int d = c * 16 * VC + VC * m;
              kv_load<VB>(&vw[4 * s + j][c * VW], src + (long long)j * a.p.slot_stride * CB + (d < D ? d : 0) * CB);
            }
          }
          if constexpr (kv_scaled(CT)) {
            const long long at = (long long)max(page, 0) * a.p.scale_page_stride + (long long)h * a.p.scale_head_stride + slot;
            kv_load<16>(reinterpret_cast<unsigned*>(ks[s]), reinterpret_cast<const unsigned char*>(a.p.k_scale + at));
            kv_load<16>(reinterpret_cast<unsigned*>(vs[s]), reinterpret_cast<const unsigned char*>(a.p.v_scale + at));
          }
        }
      };

      // One tile, and the loads of the wave's next one where there is one: that is known to the compiler, since a wait for the
      // values in flight must not depend on a branch over the loads behind them.  (Columns of K past the row's end hold other columns
      // of it and meet zeros of Q; if those are not finite, neither is the result, see below.)
      auto tile = [&](int k0, auto more) {
        // ---- S^T = K Q^T
        f32x4 st[NT][KT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int s = 0; s < KT; ++s) st[nt][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KT; ++s) {
          if constexpr (M16) {
#pragma unroll
            for (int i = 0; i < QN; ++i) {
              unsigned kf[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) kf[x] = CB == 2 ? kw[s][i * 4 + x] : pa_widen<QK, CT>(kw[s][(i * 4 + x) / 2], x & 1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int l = 0; l < QL; ++l) {
                  const unsigned* qp = &qf[nt][(i * QL + l) * 4];
                  const unsigned qv[4] = {qp[0], qp[1], qp[2], qp[3]};
                  st[nt][s] = pa_mfma16<QK>(kf, qv, st[nt][s]);
                }
            }
          } else {
#pragma unroll
            for (int i = 0; i < QN; ++i) {
              const float kf = kv_elem<CT>(&kw[s][(i / KC) * KW], i % KC);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                st[nt][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf, __builtin_bit_cast(float, qf[nt][i]), st[nt][s], 0, 0, 0);
            }
          }
        }
        if constexpr (more.value) load_k(k0 + PA_WAVES * KEYS);

        // ---- softmax: base 2, scale * log2(e) folded into S
        const bool whole = !PADDED && k0 + KEYS <= least && __all(seen == (1u << (4 * KT)) - 1u);
        float pr[NT][KT * 4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float z[KT * 4], top = -INFINITY;
#pragma unroll
          for (int k = 0; k < KT * 4; ++k) {
            z[k] = st[nt][k >> 2][k & 3] * a.scale_log2e;
            if constexpr (kv_scaled(CT)) z[k] *= ks[k >> 2][k & 3];
          }
          if (!whole) {
#pragma unroll
            for (int k = 0; k < KT * 4; ++k) z[k] = ((seen >> k) & 1u) && k0 + 16 * (k >> 2) + 4 * g + (k & 3) < lim[nt] ? z[k] : -INFINITY;
          }
#pragma unroll
          for (int k = 0; k < KT * 4; ++k) top = fmaxf(top, z[k]);
          top = fmaxf(pa_max4(top) - LIFT, mrow[nt]);
          const float ref = top == -INFINITY ? 0.f : top;             // a row that has seen nothing yet
          if (__any(top > mrow[nt])) {
            const float shrink = __builtin_amdgcn_exp2f(mrow[nt] - ref);
            lrow[nt] *= shrink;
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[nt][e] *= shrink;
            mrow[nt] = top;
          }
#pragma unroll
          for (int k = 0; k < KT * 4; ++k) {
            pr[nt][k] = __builtin_amdgcn_exp2f(z[k] - ref);
            lrow[nt] += pr[nt][k];
          }
          if constexpr (kv_scaled(CT)) {
#pragma unroll
            for (int k = 0; k < KT * 4; ++k) pr[nt][k] *= vs[k >> 2][k & 3];
            if (!whole) {
#pragma unroll
              for (int k = 0; k < KT * 4; ++k) pr[nt][k] = z[k] != -INFINITY ? pr[nt][k] : 0.f;
            }
          }
        }
        if (!whole) {                                                 // a key that nobody sees must not meet the products
#pragma unroll
          for (int k = 0; k < KT * 4; ++k)
#pragma unroll
            for (int x = 0; x < NV * VW; ++x) vw[k][x] = (seen >> k) & 1u ? vw[k][x] : 0u;
        }

        // ---- O^T += V^T P^T
        if constexpr (M16) {
#pragma unroll
          for (int k0 = 0; k0 < KT * 4; k0 += 8) {                    // eight of this lane's keys at a time
            unsigned pf[NT][PL][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                unsigned part[PL];
                pa_parts<PL, PV>(pr[nt][k0 + 2 * x], pr[nt][k0 + 2 * x + 1], part);
#pragma unroll
                for (int l = 0; l < PL; ++l) pf[nt][l][x] = part[l];
              }
#pragma unroll
            for (int c = 0; c < NV; ++c) {
#pragma unroll
              for (int q4 = 0; q4 < (VC + 3) / 4; ++q4) {
                // four columns (a pair of words of 16-bit elements, a word of codes) of the keys -> one operand per column
                unsigned vf[4][4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  if constexpr (CB == 2) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                      if (4 * q4 + 2 * y < VC) {
                        const unsigned wa = vw[k0 + 2 * x][c * VW + 2 * q4 + y], wb = vw[k0 + 2 * x + 1][c * VW + 2 * q4 + y];
                        vf[2 * y][x] = __builtin_amdgcn_perm(wb, wa, 0x05040100u);
                        vf[2 * y + 1][x] = __builtin_amdgcn_perm(wb, wa, 0x07060302u);
                      }
                    }
                  } else {
                    const unsigned wa = vw[k0 + 2 * x][c * VW + q4], wb = vw[k0 + 2 * x + 1][c * VW + q4];
                    const unsigned t0 = __builtin_amdgcn_perm(wb, wa, 0x05010400u), t1 = __builtin_amdgcn_perm(wb, wa, 0x07030602u);
                    vf[0][x] = pa_widen<PV, CT>(t0, false);
                    vf[1][x] = pa_widen<PV, CT>(t0, true);
                    if (VC > 2) {
                      vf[2][x] = pa_widen<PV, CT>(t1, false);
                      vf[3][x] = pa_widen<PV, CT>(t1, true);
                    }
                  }
                }
                // (the parts of P one after the other over the columns: products that follow each other do not wait for each other)
#pragma unroll
                for (int l = 0; l < PL; ++l)
#pragma unroll
                  for (int y = 0; y < 4; ++y) {
                    if (4 * q4 + y < VC) {
#pragma unroll
                      for (int nt = 0; nt < NT; ++nt) acc[nt][c * VC + 4 * q4 + y] = pa_mfma16<PV>(vf[y], pf[nt][l], acc[nt][c * VC + 4 * q4 + y]);
                    }
                  }
              }
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KT * 4; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const float vf = kv_elem<CT>(&vw[k][(e / VC) * VW], e % VC);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[nt][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, pr[nt][k], acc[nt][e], 0, 0, 0);
            }
        }
        if constexpr (more.value) load_v(k0 + PA_WAVES * KEYS);
      };

      int k0 = c0 + wave * KEYS;
      if (k0 < c1) {
        load_k(k0);
        __builtin_amdgcn_sched_barrier(0);                            // keys first: the values are waited for later
        load_v(k0);
#pragma unroll 1
        for (; k0 + PA_WAVES * KEYS < c1; k0 += PA_WAVES * KEYS) tile(k0, std::true_type{});
        tile(k0, std::false_type{});
      }
    }

    // ---- the four waves' parts of each row
    bool off = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float l = pa_sum4(lrow[nt]);
#pragma unroll
      for (int half = 0; half < 16 / OR; ++half) {
        __syncthreads();
        if (g == 0) s_ml[wave][m][0] = mrow[nt], s_ml[wave][m][1] = l;
        if (m / OR == half) {
#pragma unroll
          for (int e = 0; e < VE; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) s_o[wave][m % OR][(e / VC) * 16 * VC + VC * (4 * g + j) + e % VC] = acc[nt][e][j];
        }
        __syncthreads();
        for (int i = tid; i < OR * (DP / 4); i += 64 * PA_WAVES) {
          const int ml = i / (DP / 4) + half * OR, d = (i % (DP / 4)) * 4;
          const int r = row0 + nt * 16 + ml, t = r / a.group;
          if (r >= a.rows || d >= D) continue;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < PA_WAVES; ++w) top = fmaxf(top, s_ml[w][ml][0]);
          const float ref = top == -INFINITY ? 0.f : top;
          float sum = 0.f, o[4] = {};
#pragma unroll
          for (int w = 0; w < PA_WAVES; ++w) {
            const float x = __builtin_amdgcn_exp2f(s_ml[w][ml][0] - ref);
            sum += x * s_ml[w][ml][1];
            const float4 v = ld4(&s_o[w][ml - half * OR][d]);
            // a wave whose keys this row does not see adds nothing (its O is zero: no 0 * infinity comes of it)
            o[0] += x * v.x, o[1] += x * v.y, o[2] += x * v.z, o[3] += x * v.w;
          }
          const long long row = ((long long)b * a.T + t) * a.q_heads + h * a.group + r % a.group;
          off |= t < span.fresh && !(__builtin_fabsf(o[0]) + __builtin_fabsf(o[1]) + __builtin_fabsf(o[2]) + __builtin_fabsf(o[3]) < INFINITY);
          if (part_o) {
            pa_put2(part_o + (nt * 16 + ml) * D + d, o[0], o[1]);
            pa_put2(part_o + (nt * 16 + ml) * D + d + 2, o[2], o[3]);
            if (d == 0) pa_put2(part_ml + (nt * 16 + ml) * 2, top, sum);
          } else {
            const bool some = t < span.fresh && !(sum == 0.f);
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = some ? o[x] / sum : 0.f;
            pa_store_row4<RT>(a.out, row * D + d, o);
          }
        }
      }
    }
    // What a row does not see must not reach it, but 0 * infinity and 0 * NaN do in a matrix product over shared values, and an
    // infinite value meets the rest of its P, which may be 0 or negative.  So where a result is not finite, the rows are
    // computed again, each from what it sees alone.  (The barrier also parts these rows' LDS from the next ones'.)
    if (__syncthreads_or(off)) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // what is stored above does not land on top of it
      __syncthreads();
      pa_rows_alone<RT, CT>(a, b, h, tile0 * TILE, most, row0, min(row0 + 16 * NT, a.rows), span, part_o, part_ml, &s_o[0][0][0]);
    }
    if (part_o) {
      // The last of a row's workgroups joins its parts.  Parts are stored through the caches that do not reach other workgroups, and
      // every store is complete before this one counts; a release at device scope would write back everything those caches hold
      // (measured: microseconds).  The counter is zero again for the next launch.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) {
        const unsigned n = last_wg - first_wg + 1;
        const bool last = __hip_atomic_fetch_add(&a.arrived[first_wg], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (last) __hip_atomic_store(&a.arrived[first_wg], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_page[0] = last;
      }
      __syncthreads();
      const bool last = s_page[0] != 0;
      __syncthreads();
      if (last) {
        float* buf = &s_o[0][0][0];
        pa_join<RT>(a, b, h, row0, 16 * NT, first_wg, last_wg - first_wg + 1, span.fresh, reinterpret_cast<float(*)[4]>(buf), buf + 1024, buf + 1280);
        __syncthreads();
      }
    }
  }
}

template <int RT, int CT, int DP, int NT, int KT>
static void pa_launch(const PagedAttn& a, unsigned blocks, hipStream_t stream) {
  if (a.padding) hipLaunchKernelGGL((paged_attention_kernel<RT, CT, DP, NT, KT, true>), dim3(blocks), dim3(64 * PA_WAVES), 0, stream, a);
  else hipLaunchKernelGGL((paged_attention_kernel<RT, CT, DP, NT, KT, false>), dim3(blocks), dim3(64 * PA_WAVES), 0, stream, a);
}
template <int RT, int CT, int DP, int NT>
static void pa_launch(const PagedAttn& a, unsigned blocks, hipStream_t stream) {
  a.workgroups ? pa_launch<RT, CT, DP, NT, pa_blocks(RT, CT, DP, NT, true)>(a, blocks, stream)
               : pa_launch<RT, CT, DP, NT, pa_blocks(RT, CT, DP, NT, false)>(a, blocks, stream);
}
template <int RT, int CT>
static void pa_launch(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream) {
  const int D = a.p.dim;
  if (D <= 32) tiles == 2 ? pa_launch<RT, CT, 32, 2>(a, blocks, stream) : pa_launch<RT, CT, 32, 1>(a, blocks, stream);
  else if (D <= 64) tiles == 2 ? pa_launch<RT, CT, 64, 2>(a, blocks, stream) : pa_launch<RT, CT, 64, 1>(a, blocks, stream);
  else if (D > 128) pa_launch<RT, CT, 256, 1>(a, blocks, stream);
  else if constexpr (RT == KV_F32) pa_launch<RT, CT, 128, 1>(a, blocks, stream);
  else tiles == 2 ? pa_launch<RT, CT, 128, 2>(a, blocks, stream) : pa_launch<RT, CT, 128, 1>(a, blocks, stream);
}

// one definition per row type, each in its own source file: the instantiations compile side by side
void pa_run_f32(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream);
void pa_run_bf16(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream);
void pa_run_f16(const PagedAttn& a, int tiles, unsigned blocks, hipStream_t stream);

}  // namespace pvsg
