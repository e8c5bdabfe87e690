// s2c_words_common.h -- element types and wave helpers of the word operators (s2c_vocab.hip, s2c_embed.hip).
#pragma once
#include "s2c_common.h"
#include "../../include/s2c_ops.h"
#include "../../include/s2c_words.h"

namespace s2c {

typedef unsigned short u16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// 16 bytes at any element boundary (global memory takes unaligned 16-byte accesses on gfx950)
template <int ES>
struct __attribute__((packed, aligned(ES))) Bytes16 { u32 w[4]; };
struct Raw { u32 w[4]; };

template <int DT> struct Elem;
template <> struct Elem<S2C_F32> {
  typedef float T;
  static constexpr int VEC = 4, ES = 4;
  static constexpr u32 NEG_INF = 0xFF800000u;
  // element e of a vector, given the word that holds it
  static __device__ __forceinline__ float of(u32 w, int) { return __builtin_bit_cast(float, w); }
  static __device__ __forceinline__ float at(const Raw &r, int e) { return of(r.w[e], e); }
  static __device__ __forceinline__ float load(const void *p, long long i) { return ((const float *)p)[i]; }
  static __device__ __forceinline__ void store(void *p, long long i, float v) { ((float *)p)[i] = v; }
  static __device__ __forceinline__ u32 bits(const void *p, long long i) { return ((const u32 *)p)[i]; }
  static __device__ __forceinline__ void put(Raw &r, int e, u32 b) { r.w[e] = b; }
  static __device__ __forceinline__ Raw pack(const float (&f)[4]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(u32, f[i]);
    return r;
  }
};
template <> struct Elem<S2C_BF16> {
  typedef u16 T;
  static constexpr int VEC = 8, ES = 2;
  static constexpr u32 NEG_INF = 0xFF80FF80u;
  static __device__ __forceinline__ float of(u32 w, int e) {
    return __builtin_bit_cast(float, (e & 1) ? (w & 0xFFFF0000u) : (w << 16));
  }
  static __device__ __forceinline__ float at(const Raw &r, int e) { return of(r.w[e >> 1], e); }
  static __device__ __forceinline__ float load(const void *p, long long i) {
    return __builtin_bit_cast(float, (u32)((const u16 *)p)[i] << 16);
  }
  static __device__ __forceinline__ void store(void *p, long long i, float v) { ((__bf16 *)p)[i] = (__bf16)v; }
  static __device__ __forceinline__ u32 bits(const void *p, long long i) { return ((const u16 *)p)[i]; }
  static __device__ __forceinline__ void put(Raw &r, int e, u32 b) {
    r.w[e >> 1] = (e & 1) ? ((r.w[e >> 1] & 0xFFFFu) | (b << 16)) : ((r.w[e >> 1] & 0xFFFF0000u) | b);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      r.w[i] = __builtin_bit_cast(u32, __builtin_convertvector(v, bf16x2));
    }
    return r;
  }
};
template <> struct Elem<S2C_F16> {
  typedef u16 T;
  static constexpr int VEC = 8, ES = 2;
  static constexpr u32 NEG_INF = 0xFC00FC00u;
  static __device__ __forceinline__ float of(u32 w, int e) {
    return (float)__builtin_bit_cast(_Float16, (u16)((e & 1) ? (w >> 16) : (w & 0xFFFFu)));
  }
  static __device__ __forceinline__ float at(const Raw &r, int e) { return of(r.w[e >> 1], e); }
  static __device__ __forceinline__ float load(const void *p, long long i) { return (float)((const _Float16 *)p)[i]; }
  static __device__ __forceinline__ void store(void *p, long long i, float v) { ((_Float16 *)p)[i] = (_Float16)v; }
  static __device__ __forceinline__ u32 bits(const void *p, long long i) { return ((const u16 *)p)[i]; }
  static __device__ __forceinline__ void put(Raw &r, int e, u32 b) { Elem<S2C_BF16>::put(r, e, b); }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      r.w[i] = __builtin_bit_cast(u32, __builtin_convertvector(v, f16x2));
    }
    return r;
  }
};

template <int DT>
__device__ __forceinline__ Raw load16(const void *p, long long i) {
  typedef Bytes16<Elem<DT>::ES> B;
  const B b = *reinterpret_cast<const B *>((const char *)p + i * Elem<DT>::ES);
  return Raw{{b.w[0], b.w[1], b.w[2], b.w[3]}};
}
template <int DT>
__device__ __forceinline__ void store16(void *p, long long i, const Raw &r) {
  typedef Bytes16<Elem<DT>::ES> B;
  B b = {{r.w[0], r.w[1], r.w[2], r.w[3]}};
  *reinterpret_cast<B *>((char *)p + i * Elem<DT>::ES) = b;
}

// a 16-byte aligned store that does not stay in the caches
__device__ __forceinline__ void store16_past_cache(void *p, long long byte, const Raw &r) {
  typedef u32 u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 v = {r.w[0], r.w[1], r.w[2], r.w[3]};
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>((char *)p + byte));
}

// element i of an array whose type is known at run time only
__device__ __forceinline__ float load_any(const void *p, long long i, int dt) {
  return dt == S2C_F32 ? Elem<S2C_F32>::load(p, i)
                       : dt == S2C_BF16 ? Elem<S2C_BF16>::load(p, i) : Elem<S2C_F16>::load(p, i);
}

// reductions over a wave: within rows of 16 lanes through DPP (no LDS round trips), then the four rows;
// always in the same order
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float lane_f32(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_f32<DPP_QUAD_1032>(v);
  v += dpp_f32<DPP_QUAD_2301>(v);
  v += dpp_f32<DPP_ROW_HALF_MIRROR>(v);
  v += dpp_f32<DPP_ROW_MIRROR>(v);
  return (lane_f32(v, 0) + lane_f32(v, 16)) + (lane_f32(v, 32) + lane_f32(v, 48));
}
// (a NaN is passed over, as fmaxf does)
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_f32<DPP_QUAD_1032>(v));
  v = fmaxf(v, dpp_f32<DPP_QUAD_2301>(v));
  v = fmaxf(v, dpp_f32<DPP_ROW_HALF_MIRROR>(v));
  v = fmaxf(v, dpp_f32<DPP_ROW_MIRROR>(v));
  return fmaxf(fmaxf(lane_f32(v, 0), lane_f32(v, 16)), fmaxf(lane_f32(v, 32), lane_f32(v, 48)));
}
// order LDS accesses of the lanes of ONE wave (its LDS operations execute in order; this keeps the
// compiler from moving them)
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace s2c
