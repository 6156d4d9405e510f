// policy_common.hpp — element types, exact splits into bfloat16 planes and matrix-core
// products shared by the policy's operators (libnavi_policy.so).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "navi_policy.h"

namespace navi_policy {

int set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

using f2 = float __attribute__((ext_vector_type(2)));
using f4 = float __attribute__((ext_vector_type(4)));
using u2 = uint32_t __attribute__((ext_vector_type(2)));
using u4 = uint32_t __attribute__((ext_vector_type(4)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using s4 = short __attribute__((ext_vector_type(4)));

struct bf16 {
    uint16_t bits;
};
struct f16 {
    _Float16 value;
};

__device__ inline uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ inline float float_of(uint32_t x) { return __builtin_bit_cast(float, x); }

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(bf16 x) { return float_of(static_cast<uint32_t>(x.bits) << 16); }
__device__ inline float to_float(f16 x) { return static_cast<float>(x.value); }

template <class E>
__device__ inline E from_float(float x);
template <>
__device__ inline float from_float<float>(float x) {
    return x;
}
template <>
__device__ inline bf16 from_float<bf16>(float x) {  // to nearest even, NaN kept (v_cvt_pk_bf16_f32)
    return bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(x))};
}
template <>
__device__ inline f16 from_float<f16>(float x) {
    return f16{static_cast<_Float16>(x)};
}

// A float32 is the sum of three bfloat16, each the rounding of what those before it leave (8 bits
// of its 24 and a sign), a float16's 11 bits fit two, so products of such planes on the matrix
// cores keep float32's precision at a third to a sixth of the bfloat16 rate: five to two times
// float32's own. (Numbers above 3.39e38, bfloat16's largest, count as infinite.)
template <class E>
inline constexpr int kPlanes = 3;
template <>
inline constexpr int kPlanes<bf16> = 1;
template <>
inline constexpr int kPlanes<f16> = 2;

// Two floats rounded to nearest as two bfloat16 (a in the low half; v_cvt_pk_bf16_f32).
__device__ inline uint32_t rounded_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf16x2));
}

// The planes of two floats; with N = 3 their sum is exact (a normal float's). Plane p's remainder
// is at most 2^-9 of the one before it, of either sign: cut off instead of rounded, it would be
// 2^-7 and always of the number's sign, and what products of planes leave out would add up.
template <int N>
__device__ inline void split_pair(float a, float b, uint32_t (&plane)[N]) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
        plane[p] = rounded_pair(a, b);
        if (p + 1 < N) {
            a -= float_of(plane[p] << 16);
            b -= float_of(plane[p] & 0xffff0000u);
        }
    }
}

// The wave's place in its workgroup, in a scalar register: matrix products run whatever the
// execution mask says, so a branch around them has to be one that the wave takes or not.
__device__ inline int wave_of_workgroup() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Eight floats of a lane as an operand of 16x16x32 products.
template <int N>
__device__ inline void split8(const float (&x)[8], u4 (&plane)[N]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t p[N];
        split_pair<N>(x[2 * j], x[2 * j + 1], p);
#pragma unroll
        for (int n = 0; n < N; ++n) plane[n][j] = p[n];
    }
}

template <int N>
__device__ inline void split8(f4 a, f4 b, u4 (&plane)[N]) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    split8<N>(x, plane);
}

// D += A B on the matrix cores, 16 x 32 by 32 x 16: lane l holds row (of A) or column (of B,
// C and D) l % 16; of A and B the eight numbers at 8 (l / 16) of the contracted axis (in any
// order that A and B share), of C and D rows 4 (l / 16) to 4 (l / 16) + 3.
__device__ inline f4 mfma(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// The product of two sums of planes, smallest terms first. Left out is the second plane of one
// times the third of the other, 2^-27 of the product each, and less.
template <int NA, int NB>
__device__ inline f4 mma(const u4 (&a)[NA], const u4 (&b)[NB], f4 c) {
#pragma unroll
    for (int s = (NA + NB - 2 < 2 ? NA + NB - 2 : 2); s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = mfma(a[i], b[s - i], c);
    return c;
}

// The products of several left operands with one right operand, term by term over all of them:
// a product waits for the one before it in the same sum, so neighbours are of different sums.
template <int kCount, int NA, int NB>
__device__ inline void mma_each(const u4 (&a)[kCount][NA], const u4 (&b)[NB], f4 (&c)[kCount]) {
#pragma unroll
    for (int s = (NA + NB - 2 < 2 ? NA + NB - 2 : 2); s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB)
#pragma unroll
                for (int n = 0; n < kCount; ++n) c[n] = mfma(a[n][i], b[s - i], c[n]);
}

// The same, each result transposed: the operands hold rows and columns alike, so exchanging them
// does. A lane then has row l % 16 of the result, columns 4 (l / 16) to 4 (l / 16) + 3.
template <int kCount, int NA, int NB>
__device__ inline void mma_each_transposed(const u4 (&a)[kCount][NA], const u4 (&b)[NB], f4 (&c)[kCount]) {
#pragma unroll
    for (int s = (NA + NB - 2 < 2 ? NA + NB - 2 : 2); s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB)
#pragma unroll
                for (int n = 0; n < kCount; ++n) c[n] = mfma(b[s - i], a[n][i], c[n]);
}

// 16x16x4 in float32: A's lane holds row l % 16, B's column l % 16, at l / 16 of the four.
__device__ inline f4 mfma_f32(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Four 16-bit numbers of a 4 x 16 block's column for each of 16 lanes; lane i of the 16 gives
// the address of row i / 4, columns 4 (i % 4) to 4 (i % 4) + 3.
__device__ inline u2 read_transposed(const uint16_t* lds) {
    using pointer = __attribute__((address_space(3))) s4*;
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pointer)(lds)));
}

// Buffer accesses: a scalar base and size and a lane's 32-bit offset; loads from kOutside or
// past the size give 0, stores there are dropped, so tails need no branches. The whole offset
// is the lane's: a scalar part beyond the size would turn the range check around (it compares
// the lane's part with the size less the scalar part, unsigned).
using Buffer = __amdgpu_buffer_rsrc_t;
constexpr uint32_t kOutside = 0x80000000u;  // (sizes and what is added to an offset are below 2^31)

__device__ inline Buffer buffer_of(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00020000);
}

template <class E>
__device__ inline E buffer_load(Buffer from, uint32_t offset) {
    if constexpr (sizeof(E) == 4)
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0));
    else
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b16(from, offset, 0, 0));
}

template <class E>
__device__ inline void buffer_store(Buffer to, uint32_t offset, E x) {
    if constexpr (sizeof(E) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), to, offset, 0, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), to, offset, 0, 0);
}

__device__ inline u4 buffer_load16(Buffer from, uint32_t offset) {
    return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0));
}

// Four numbers of a row in one store (the address a multiple of their bytes).
__device__ inline void buffer_store_four(Buffer to, uint32_t offset, const bf16 (&x)[4]) {
    __builtin_amdgcn_raw_buffer_store_b64(u2{x[0].bits | static_cast<uint32_t>(x[1].bits) << 16,
                                             x[2].bits | static_cast<uint32_t>(x[3].bits) << 16}, to, offset, 0, 0);
}
__device__ inline void buffer_store_four(Buffer to, uint32_t offset, const f16 (&x)[4]) {
    bf16 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i].bits = __builtin_bit_cast(uint16_t, x[i].value);
    buffer_store_four(to, offset, y);
}
__device__ inline void buffer_store_four(Buffer to, uint32_t offset, const float (&x)[4]) {
    __builtin_amdgcn_raw_buffer_store_b128(u4{bits_of(x[0]), bits_of(x[1]), bits_of(x[2]), bits_of(x[3])}, to, offset, 0, 0);
}

// Numbers of a row from `offset` bytes on: in 16-byte loads where rows are multiples of eight,
// else one by one, those from `valid` on as zeros.
template <class T, int kCount>
struct Part {
    static constexpr int kWords = kCount * sizeof(T) / 16;
    u4 words[kWords];

    __device__ void load(Buffer from, uint32_t offset, int valid, bool wide) {
        if (wide) {
            const uint32_t lane = valid > 0 ? offset : kOutside;
#pragma unroll
            for (int w = 0; w < kWords; ++w) words[w] = buffer_load16(from, lane + 16 * w);
            return;
        }
        uint32_t x[kCount];
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const T y = buffer_load<T>(from, i < valid ? offset + i * sizeof(T) : kOutside);
            if constexpr (sizeof(T) == 4)
                x[i] = bits_of(y);
            else
                x[i] = __builtin_bit_cast(uint16_t, y);
        }
#pragma unroll
        for (int i = 0; i < 4 * kWords; ++i)
            words[i / 4][i % 4] = sizeof(T) == 4 ? x[i] : x[2 * i % kCount] | x[(2 * i + 1) % kCount] << 16;
    }

    __device__ void floats(float (&x)[kCount]) const {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if constexpr (sizeof(T) == 4)
                x[i] = float_of(words[i / 4][i % 4]);
            else
                x[i] = to_float(__builtin_bit_cast(T, static_cast<uint16_t>(words[0][i / 2] >> (16 * (i % 2)))));
        }
    }
};

inline hipStream_t as_stream(void* stream) { return static_cast<hipStream_t>(stream); }

template <class... P>
bool aligned(int64_t bytes, const P*... p) {
    return ((reinterpret_cast<uintptr_t>(p) % bytes == 0) && ...);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace navi_policy
