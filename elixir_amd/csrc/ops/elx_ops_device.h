// Element codecs and memory access shared by the kernels of libelx_ops.so.
#ifndef ELX_OPS_DEVICE_H
#define ELX_OPS_DEVICE_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "elx_ops.h"

namespace elx_ops {

constexpr int kWave = 64;
constexpr uint32_t kLdsPerCu = 160u * 1024u;    // gfx950

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int D>
struct Elem;

template <>
struct Elem<ELX_F32> {
    typedef float scalar;
    typedef f32x4 vec4;
    static __device__ __forceinline__ float to_f32(float x) { return x; }
    static __device__ __forceinline__ float from_f32(float x) { return x; }
};

template <>
struct Elem<ELX_F16> {
    typedef uint16_t scalar;
    typedef u16x4 vec4;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
    // round to nearest even, overflow to infinity, subnormals kept
    static __device__ __forceinline__ uint16_t from_f32(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

template <>
struct Elem<ELX_BF16> {
    typedef uint16_t scalar;
    typedef u16x4 vec4;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
    // round to nearest even, NaN stays a quiet NaN
    static __device__ __forceinline__ uint16_t from_f32(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};

// Tile-local buffer addressing: a uniform base and extent, a 32-bit byte offset per lane; accesses beyond the extent
// read zero and write nothing.  AUX is the cache policy (2 non-temporal, 16 agent scope).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, 0x00020000);
}

template <typename V>
struct TileIo;

template <>
struct TileIo<f32x4> {
    template <int AUX>
    static __device__ __forceinline__ f32x4 load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, AUX));
    }
    template <int AUX>
    static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t off, f32x4 x) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, (int)off, 0, AUX);
    }
};

template <>
struct TileIo<u16x4> {
    template <int AUX>
    static __device__ __forceinline__ u16x4 load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
        return __builtin_bit_cast(u16x4, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, AUX));
    }
    template <int AUX>
    static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t off, u16x4 x) {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), r, (int)off, 0, AUX);
    }
};

template <>
struct TileIo<uint32_t> {
    template <int AUX>
    static __device__ __forceinline__ uint32_t load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
        return __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, AUX);
    }
    template <int AUX>
    static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t x) {
        __builtin_amdgcn_raw_buffer_store_b32(x, r, (int)off, 0, AUX);
    }
};

inline bool is_float_code(int d) { return d == ELX_F32 || d == ELX_F16 || d == ELX_BF16; }
inline uint32_t elem_size(int d) { return d == ELX_F32 ? 4u : 2u; }

}    // namespace elx_ops

#endif    // ELX_OPS_DEVICE_H
