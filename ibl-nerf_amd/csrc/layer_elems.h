// Eight neighbouring elements of a row in float32, bfloat16 or float16: loads and stores that stop at the row's end, conversions (dense_kernel.hip, lookup_kernel.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "layers.h"

namespace ibl {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int T> struct Bytes { static constexpr int v = T == LT_F32 ? 4 : 2; };

// (by value: __builtin_bit_cast of a vector's element reads element 0)
__device__ __forceinline__ float as_float(unsigned u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ unsigned as_bits(float f) { return __builtin_bit_cast(unsigned, f); }

__device__ __forceinline__ float half_float(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }

// eight consecutive elements of a row as they lie in memory: 16 bytes (16-bit types) or 32 (float32)
template <int T> struct Raw8 { u32x4 q[T == LT_F32 ? 2 : 1]; };

__device__ __forceinline__ u32x4 load16(const void* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);        // (rows of odd length: any alignment of the element type)
    return v;
}

template <int T> __device__ __forceinline__ Raw8<T> zero8() {
    Raw8<T> v;
    v.q[0] = u32x4{0, 0, 0, 0};
    if constexpr (T == LT_F32) v.q[1] = u32x4{0, 0, 0, 0};
    return v;
}

// columns c .. c + 7 of a row of `cols` elements; what lies beyond the row's end is zero and is not read
template <int T> __device__ __forceinline__ Raw8<T> load8(const char* row, int c, int cols) {
    Raw8<T> v = zero8<T>();
    if (c + 8 <= cols) {
        v.q[0] = load16(row + (size_t)c * Bytes<T>::v);
        if constexpr (T == LT_F32) v.q[1] = load16(row + (size_t)c * 4 + 16);
    } else if (c < cols) {
        if constexpr (T == LT_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) v.q[i >> 2][i & 3] = reinterpret_cast<const unsigned*>(row)[c + i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) v.q[0][i >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(row)[c + i] << (16 * (i & 1));
        }
    }
    return v;
}

// eight columns from c on, all of them there (straight code)
template <int T> __device__ __forceinline__ Raw8<T> load8_whole(const char* row, int c) {
    Raw8<T> v;
    v.q[0] = load16(row + (size_t)c * Bytes<T>::v);
    if constexpr (T == LT_F32) v.q[1] = load16(row + (size_t)c * 4 + 16);
    return v;
}

// the elements whose code byte is zero become zero (a select: what stands in a closed place, a NaN too, is gone)
template <int T> __device__ __forceinline__ void close8(Raw8<T>& v, u32x2 codes) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const unsigned c = codes[g];
        const unsigned t = ((c & 0x7f7f7f7fu) + 0x7f7f7f7fu) | c;      // bit 7 of each byte: that byte is not zero
        if constexpr (T == LT_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v.q[g][i] &= (unsigned)((int)(t << (24 - 8 * i)) >> 31);
        } else {
            const unsigned u = t << 8;                                 // v_perm selectors 8 .. 11: the sign of byte 1, 3 (second operand), 5, 7 (first) in all eight bits
            v.q[0][2 * g] &= __builtin_amdgcn_perm(t, u, 0x0a0a0808u);
            v.q[0][2 * g + 1] &= __builtin_amdgcn_perm(t, u, 0x0b0b0909u);
        }
    }
}

template <int T> __device__ __forceinline__ void to_floats(const Raw8<T>& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == LT_F32) f[i] = as_float(v.q[i >> 2][i & 3]);
        else if constexpr (T == LT_BF16) f[i] = as_float((i & 1) ? (v.q[0][i >> 1] & 0xffff0000u) : (v.q[0][i >> 1] << 16));
        else { const unsigned u = v.q[0][i >> 1]; f[i] = (float)__builtin_bit_cast(f16x2, u)[i & 1]; }
    }
}

// two floats rounded to nearest (even) in a 16-bit type
template <int T> __device__ __forceinline__ unsigned pack2(float a, float b) {
    const f32x2 x = {a, b};
    if constexpr (T == LT_BF16) return __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(x, f16x2));
}

template <int T> __device__ __forceinline__ Raw8<T> from_floats(const float (&f)[8]) {
    Raw8<T> v;
    if constexpr (T == LT_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.q[i >> 2][i & 3] = as_bits(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v.q[0][i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    return v;
}

template <int T> __device__ __forceinline__ void store8(char* row, int c, int cols, const Raw8<T>& v) {
    if (c + 8 <= cols) {
        __builtin_memcpy(row + (size_t)c * Bytes<T>::v, &v.q[0], 16);
        if constexpr (T == LT_F32) __builtin_memcpy(row + (size_t)c * 4 + 16, &v.q[1], 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < cols) {
                if constexpr (T == LT_F32) reinterpret_cast<unsigned*>(row)[c + i] = v.q[i >> 2][i & 3];
                else reinterpret_cast<unsigned short*>(row)[c + i] = (unsigned short)(v.q[0][i >> 1] >> (16 * (i & 1)));
            }
    }
}

}  // namespace

}  // namespace ibl
