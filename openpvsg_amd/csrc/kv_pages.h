// Paged key/value pools: what kv_cache.hip (write, read back) and paged_attention.hip share.
//
// A pool is K and V of (pages, heads, page_size, dim), element strides for the first three axes, the last one dense, and for
// the 8-bit types one f32 scale per row (pages, heads, page_size), slots dense.  Position p of sequence b is slot p % page_size
// of page table[b][p / page_size].  Page ids come from device memory, so the kernels check every one of them: an id outside the
// pool is never dereferenced, it sets a bit in the pool's `faults` word.
#pragma once
#include "../../include/openpvsg_hip.h"
#include "common.h"

namespace pvsg {

enum : int { KV_F32 = PVSG_TYPE_F32, KV_BF16 = PVSG_TYPE_BF16, KV_F16 = PVSG_TYPE_F16, KV_E4M3 = PVSG_TYPE_E4M3, KV_I8 = PVSG_TYPE_I8 };

constexpr int kv_bytes(int type) { return type == KV_F32 ? 4 : type == KV_BF16 || type == KV_F16 ? 2 : 1; }
constexpr bool kv_scaled(int type) { return type == KV_E4M3 || type == KV_I8; }

typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 kv_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned kv_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned kv_u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ unsigned kv_pack_bf16(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, kv_bf16x2));
}
__device__ __forceinline__ unsigned kv_pack_f16(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, kv_f16x2));
}

// element i (a constant once unrolled) of packed little-endian words, as f32: exact for every type
template <int TYPE>
__device__ __forceinline__ float kv_elem(const unsigned* w, int i) {
  if constexpr (TYPE == KV_F32) {
    return __builtin_bit_cast(float, w[i]);
  } else if constexpr (TYPE == KV_BF16) {
    return __builtin_bit_cast(float, (i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  } else if constexpr (TYPE == KV_F16) {
    return (float)__builtin_bit_cast(kv_f16x2, w[i >> 1])[i & 1];
  } else if constexpr (TYPE == KV_E4M3) {
    const int x = (int)w[i >> 2];
    switch (i & 3) {                       // the byte select is an immediate
      case 0: return __builtin_amdgcn_cvt_f32_fp8(x, 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8(x, 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8(x, 2);
      default: return __builtin_amdgcn_cvt_f32_fp8(x, 3);
    }
  } else {
    return (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// N bytes (a power of two, 2..16) between memory and words
template <int N>
__device__ __forceinline__ void kv_load(unsigned* w, const unsigned char* p) {
  if constexpr (N == 16) {
    const kv_u32x4 t = *reinterpret_cast<const kv_u32x4*>(p);
    w[0] = t[0], w[1] = t[1], w[2] = t[2], w[3] = t[3];
  } else if constexpr (N == 8) {
    const kv_u32x2 t = *reinterpret_cast<const kv_u32x2*>(p);
    w[0] = t[0], w[1] = t[1];
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  } else {
    w[0] = *reinterpret_cast<const unsigned short*>(p);
  }
}
// the same for what is read once (and below, ONCE, for what is written and not soon read): without room in L2 taken for it.
// Dense over a wave's lanes only: 16 bytes in every 32 this way took 1.6 times the time.
template <int N>
__device__ __forceinline__ void kv_load_once(unsigned* w, const unsigned char* p) {
  if constexpr (N == 16) {
    const kv_u32x4 t = __builtin_nontemporal_load(reinterpret_cast<const kv_u32x4*>(p));
    w[0] = t[0], w[1] = t[1], w[2] = t[2], w[3] = t[3];
  } else if constexpr (N == 8) {
    const kv_u32x2 t = __builtin_nontemporal_load(reinterpret_cast<const kv_u32x2*>(p));
    w[0] = t[0], w[1] = t[1];
  } else {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(p));
  }
}
template <int N, bool ONCE = false>
__device__ __forceinline__ void kv_store(unsigned char* p, const unsigned* w) {
  if constexpr (N == 16) {
    const kv_u32x4 t = {w[0], w[1], w[2], w[3]};
    if constexpr (ONCE) __builtin_nontemporal_store(t, reinterpret_cast<kv_u32x4*>(p));
    else *reinterpret_cast<kv_u32x4*>(p) = t;
  } else if constexpr (N == 8) {
    const kv_u32x2 t = {w[0], w[1]};
    if constexpr (ONCE) __builtin_nontemporal_store(t, reinterpret_cast<kv_u32x2*>(p));
    else *reinterpret_cast<kv_u32x2*>(p) = t;
  } else {
    *reinterpret_cast<unsigned*>(p) = w[0];
  }
}

// Positions of a sequence, from the device's lengths: `len` of them by its own count, `there` of them inside its table, the
// `fresh` last ones new in this call (at most T, and at most all).
struct KvSpan {
  int len, there, fresh;
};
__device__ __forceinline__ KvSpan kv_span_of(int len, int fresh, int T, int capacity) {
  KvSpan s;
  s.len = max(len, 0);
  s.there = min(s.len, capacity);
  s.fresh = min(max(min(fresh, T), 0), s.len);
  return s;
}
__device__ __forceinline__ KvSpan kv_span(const int* __restrict__ lens, const int* __restrict__ new_lens, int b, int T, int capacity) {
  return kv_span_of(lens[b], new_lens ? new_lens[b] : T, T, capacity);
}

__device__ __forceinline__ void kv_fault(int* faults, int bit) {
  if (faults) __hip_atomic_fetch_or(faults, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// a launch of 256-thread workgroups holds fewer than 2^32 threads
constexpr long long KV_MAX_BLOCKS = 1ll << 24;

// the checks every entry point makes of its pool
int kv_check_pages(const char* who, const pvsg_kv_pages* p, const int* table, long long table_stride, int table_width, const int* lens, int B);

}  // namespace pvsg
