// Element types, cache rows and reductions that the serving kernels share.
#pragma once
#include "common.h"

typedef uint32_t gm_u32x4a __attribute__((ext_vector_type(4), aligned(16)));
typedef __bf16 gm_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 gm_h8 __attribute__((ext_vector_type(8)));
typedef float gm_f32x16 __attribute__((ext_vector_type(16)));

// The two 16-bit types: bits <-> float (to nearest even) and their MFMAs.
template <int QT> struct GmT16;
template <> struct GmT16<GM_QTYPE_BF16> {
  using V8 = gm_bf8;
  using V2 = __bf16 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    V2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
  // c + both elements
  static __device__ __forceinline__ float add(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(V2, w), __builtin_bit_cast(V2, 0x3f803f80u), c, false);
  }
  static __device__ __forceinline__ gm_f32x4 mfma16(gm_u32x4 a, gm_u32x4 b, gm_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ gm_f32x16 mfma32(gm_u32x4 a, gm_u32x4 b, gm_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
};
template <> struct GmT16<GM_QTYPE_F16> {
  using V8 = gm_h8;
  using V2 = _Float16 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float lo(uint32_t w) { return gm_h2f(w & 0xffffu); }
  static __device__ __forceinline__ float hi(uint32_t w) { return gm_h2f(w >> 16); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    V2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float add(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(V2, w), __builtin_bit_cast(V2, 0x3c003c00u), c, false);
  }
  static __device__ __forceinline__ gm_f32x4 mfma16(gm_u32x4 a, gm_u32x4 b, gm_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ gm_f32x16 mfma32(gm_u32x4 a, gm_u32x4 b, gm_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
};

__host__ __device__ inline int gm_elem_bytes(int qtype) { return qtype == GM_QTYPE_F32 ? 4 : 2; }
inline bool gm_is_elem(int qtype) {
  return qtype == GM_QTYPE_F32 || qtype == GM_QTYPE_F16 || qtype == GM_QTYPE_BF16;
}
inline bool gm_is_t16(int qtype) { return qtype == GM_QTYPE_F16 || qtype == GM_QTYPE_BF16; }

// Element i of an array of `qtype` (uniform over the launch).
__device__ __forceinline__ float gm_elem(const void* p, int64_t i, int qtype) {
  if (qtype == GM_QTYPE_F32) return static_cast<const float*>(p)[i];
  const uint32_t w = static_cast<const uint16_t*>(p)[i];
  return qtype == GM_QTYPE_BF16 ? GmT16<GM_QTYPE_BF16>::lo(w) : GmT16<GM_QTYPE_F16>::lo(w);
}

// N (4 or 8) elements from i on; vec: their address is a multiple of N elements.
template <int N>
__device__ __forceinline__ void gm_load(const void* p, int64_t i, int qtype, bool vec, float (&v)[N]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = gm_elem(p, i + e, qtype);
    return;
  }
  if (qtype == GM_QTYPE_F32) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const gm_f32x4 x = *reinterpret_cast<const gm_f32x4*>(static_cast<const float*>(p) + i + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = x[e];
    }
    return;
  }
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const gm_u32x4 x = *reinterpret_cast<const gm_u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = x[e];
  } else {
    const gm_u32x2 x = *reinterpret_cast<const gm_u32x2*>(static_cast<const uint16_t*>(p) + i);
    w[0] = x[0];
    w[1] = x[1];
  }
#pragma unroll
  for (int e = 0; e < N / 2; ++e) {
    v[2 * e] = qtype == GM_QTYPE_BF16 ? GmT16<GM_QTYPE_BF16>::lo(w[e]) : GmT16<GM_QTYPE_F16>::lo(w[e]);
    v[2 * e + 1] = qtype == GM_QTYPE_BF16 ? GmT16<GM_QTYPE_BF16>::hi(w[e]) : GmT16<GM_QTYPE_F16>::hi(w[e]);
  }
}

// N (4 or 8) elements to an address that is a multiple of N elements, each
// rounded once, to nearest even.
template <int N>
__device__ __forceinline__ void gm_store(void* p, int64_t i, int qtype, const float (&v)[N]) {
  if (qtype == GM_QTYPE_F32) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h)
      *reinterpret_cast<gm_f32x4*>(static_cast<float*>(p) + i + 4 * h) =
          gm_f32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    return;
  }
  uint32_t w[N / 2];
#pragma unroll
  for (int e = 0; e < N / 2; ++e)
    w[e] = qtype == GM_QTYPE_BF16 ? GmT16<GM_QTYPE_BF16>::pack(v[2 * e], v[2 * e + 1])
                                  : GmT16<GM_QTYPE_F16>::pack(v[2 * e], v[2 * e + 1]);
  if constexpr (N == 8)
    *reinterpret_cast<gm_u32x4*>(static_cast<uint16_t*>(p) + i) = gm_u32x4{w[0], w[1], w[2], w[3]};
  else
    *reinterpret_cast<gm_u32x2*>(static_cast<uint16_t*>(p) + i) = gm_u32x2{w[0], w[1]};
}

// Whether rows of these strides (elements) start at multiples of 16 bytes.
inline bool gm_rows_aligned(const void* p, int qtype, int64_t st, int64_t sh) {
  const int64_t n = 16 / gm_elem_bytes(qtype);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st % n == 0 && sh % n == 0;
}

int gm_rope_append_run(const gm_rope_append_args* a, hipStream_t s);
size_t gm_paged_attn_ws(const gm_paged_attn_args* a);
int gm_paged_attn_run(const gm_paged_attn_args* a, uint8_t* ws, hipStream_t s);
int gm_prompt_attn_run(const gm_prompt_attn_args* a, hipStream_t s);
size_t gm_sample_ws(const gm_sample_args* a);
int gm_sample_run(const gm_sample_args* a, uint8_t* ws, hipStream_t s);
