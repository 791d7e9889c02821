// elements.h -- element types, matrix-core fragments and small device helpers of the training kernels (gfx950 only).
//
// A FRAGMENT is one 16-byte chunk per lane: lane (lr = lane & 15, lg = lane >> 4) holds 16 / sizeof(element) consecutive contraction
// indices of row lr, chunk lg. mma() multiplies an A fragment (16 rows) by a B fragment (16 columns) over KS contraction indices
// (16-bit types: one v_mfma_f32_16x16x32; fp32: four v_mfma_f32_16x16x4, chunk element e of the four lane groups in the e-th) and
// leaves D[row 4 lg + r][column lr] in register r of the lane. Any order of the contraction indices will do as long as A and B agree:
// an operand stored with its own index contiguous is read in the order that the transposing LDS read gives (read_cols), and a row-form
// operand beside it in the same order (read_row_chunk).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stddef.h>
#include "../../../include/atlas_train.h"

namespace atlas_train {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// 16, 8 and 4 bytes at the alignment of their elements: one access, whatever the address
typedef u4 __attribute__((aligned(2))) u4_any;
typedef u2 __attribute__((aligned(2))) u2_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;

static __device__ __forceinline__ float as_f(uint32_t u) { return __builtin_bit_cast(float, u); }
static __device__ __forceinline__ uint32_t as_u(float f) { return __builtin_bit_cast(uint32_t, f); }

struct F16 {
    typedef uint16_t elem;
    static constexpr int DT = ATLAS_TRAIN_F16, EPC = 8, KS = 32, TILES = 2;      // elements per chunk, contraction per mma, 16-row tiles per chunk
    static __device__ __forceinline__ float ld(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
    static __device__ __forceinline__ uint16_t st(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
    static __device__ __forceinline__ f4 mma(const u4& a, const u4& b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};
struct BF16 {
    typedef uint16_t elem;
    static constexpr int DT = ATLAS_TRAIN_BF16, EPC = 8, KS = 32, TILES = 2;
    static __device__ __forceinline__ float ld(uint16_t b) { return as_f((uint32_t)b << 16); }
    static __device__ __forceinline__ uint16_t st(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
    static __device__ __forceinline__ f4 mma(const u4& a, const u4& b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
};
struct F32 {
    typedef float elem;
    static constexpr int DT = ATLAS_TRAIN_F32, EPC = 4, KS = 16, TILES = 1;
    static __device__ __forceinline__ float ld(float b) { return b; }
    static __device__ __forceinline__ float st(float f) { return f; }
    static __device__ __forceinline__ f4 mma(const u4& a, const u4& b, f4 c) {
        const uint32_t a0 = a.x, a1 = a.y, a2 = a.z, a3 = a.w, b0 = b.x, b1 = b.y, b2 = b.z, b3 = b.w;
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f(a0), as_f(b0), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f(a1), as_f(b1), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f(a2), as_f(b2), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f(a3), as_f(b3), c, 0, 0, 0);
        return c;
    }
};

template <class T> static __device__ __forceinline__ void unpack(const u4& t, float (&v)[T::EPC]) {
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < T::EPC; ++i) {
        if constexpr (T::EPC == 4) v[i] = as_f(w[i]);
        else v[i] = T::ld((uint16_t)(w[i / 2] >> (16 * (i & 1))));
    }
}
// acc[a][b] += fa[a] x fb[b]. fp32: the four products of a step go round the accumulators, so that neighbours are independent (a dependent
// v_mfma_f32_16x16x4 waits 8 cycles more than the 32 it takes)
template <class T, int FA, int FB> static __device__ __forceinline__ void mma_block(const u4 (&fa)[FA], const u4 (&fb)[FB], f4 (&acc)[FA][FB]) {
    if constexpr (T::EPC == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int a = 0; a < FA; ++a) {
                const uint32_t x = fa[a][e];
#pragma unroll
                for (int b = 0; b < FB; ++b) {
                    const uint32_t y = fb[b][e];
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(as_f(x), as_f(y), acc[a][b], 0, 0, 0);
                }
            }
    } else {
#pragma unroll
        for (int a = 0; a < FA; ++a)
#pragma unroll
            for (int b = 0; b < FB; ++b) acc[a][b] = T::mma(fa[a], fb[b], acc[a][b]);
    }
}

// NV consecutive elements <-> floats; 8 or 16 bytes are one aligned vector access
template <class T, int NV> static __device__ __forceinline__ void load_n(const typename T::elem* p, float (&v)[NV]) {
    typedef typename T::elem E;
    if constexpr (sizeof(E) * NV == 16) {
        const u4 t = *(const u4*)p;
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (sizeof(E) == 4) v[i] = as_f(w[i]);
            else v[i] = T::ld((uint16_t)(w[i / 2] >> (16 * (i & 1))));
        }
    } else if constexpr (sizeof(E) * NV == 8) {
        const uint2 t = *(const uint2*)p;
        const uint32_t w[2] = {t.x, t.y};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (sizeof(E) == 4) v[i] = as_f(w[i]);
            else v[i] = T::ld((uint16_t)(w[i / 2] >> (16 * (i & 1))));
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = T::ld(p[i]);
    }
}
// two values -> one word, round to nearest even (one v_cvt_pk)
typedef float f2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
template <class T> static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f2 v = {a, b};
    if constexpr (T::DT == ATLAS_TRAIN_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
}
// four consecutive elements at any alignment
template <class T> static __device__ __forceinline__ void load4_any(const typename T::elem* p, float (&v)[4]) {
    if constexpr (T::EPC == 4) {
        const u4 t = *(const u4_any*)p;
        v[0] = as_f(t.x); v[1] = as_f(t.y); v[2] = as_f(t.z); v[3] = as_f(t.w);
    } else {
        const u2 t = *(const u2_any*)p;
        v[0] = T::ld((uint16_t)t.x); v[1] = T::ld((uint16_t)(t.x >> 16)); v[2] = T::ld((uint16_t)t.y); v[3] = T::ld((uint16_t)(t.y >> 16));
    }
}
template <class T> static __device__ __forceinline__ void store4_any(typename T::elem* p, const float (&v)[4]) {
    if constexpr (T::EPC == 4) *(u4_any*)p = (u4){as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])};
    else *(u2_any*)p = (u2){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
}
template <class T, int NV> static __device__ __forceinline__ void store_n(typename T::elem* p, const float (&v)[NV]) {
    typedef typename T::elem E;
    if constexpr (sizeof(E) * NV == 16) {
        if constexpr (sizeof(E) == 4) *(u4*)p = (u4){as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])};
        else *(u4*)p = (u4){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
    } else if constexpr (sizeof(E) * NV == 8 && sizeof(E) == 2) {
        *(uint2*)p = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) p[i] = T::st(v[i]);
    }
}

// a chunk of an operand in col form: column c0 + lr of rows r0 + 4 lg .. + 3 (16-bit: and of rows r0 + 16 + 4 lg .. + 3) of a row-major LDS tile.
// 16-bit: ds_read_b64_tr_b16 transposes inside a group of 16 lanes: lane s gives the address of row s >> 2, columns 4 (s & 3) .. + 3 and
// receives column s of the four rows. `tile` is a byte address in LDS, pitch in bytes.
template <class T> static __device__ __forceinline__ u4 read_cols(const unsigned char* tile, int pitch, int r0, int c0, int lr, int lg) {
    if constexpr (T::TILES == 1) {
        const float* p = (const float*)(tile + (r0 + 4 * lg) * pitch) + c0 + lr;
        const int q = pitch / 4;
        return (u4){as_u(p[0]), as_u(p[q]), as_u(p[2 * q]), as_u(p[3 * q])};
    } else {
        const unsigned char* p = tile + (r0 + 4 * lg + (lr >> 2)) * pitch + (c0 + 4 * (lr & 3)) * 2;
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)p);
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)(p + 16 * pitch));
        const uint2 a = __builtin_bit_cast(uint2, x), b = __builtin_bit_cast(uint2, y);
        return (u4){a.x, a.y, b.x, b.y};
    }
}

// a fragment of a row-form tile: the lane's own 16 bytes, or (beside an operand read by read_cols, 16-bit types) the two 8-byte pieces that hold the
// contraction indices 4 lg .. + 3 and 16 + 4 lg .. + 3 which that read enumerates
template <class T, bool BESIDE_COLS> static __device__ __forceinline__ u4 read_row_chunk(const unsigned char* row, int lg) {
    if constexpr (T::TILES == 2 && BESIDE_COLS) {
        const uint2 a = *(const uint2*)(row + 8 * lg), b = *(const uint2*)(row + 32 + 8 * lg);
        return (u4){a.x, a.y, b.x, b.y};
    } else return *(const u4*)(row + 16 * lg);
}

static __device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp, 2^-inf = 0
static __device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// ---- 8-bit codes (the header's definition) ----
// e of the group's power of two 2^e: the smallest with amax / 2^e <= 448 = 1.75 * 2^8. amax = 1.m * 2^E: e = E - 8, one more if 1.m > 1.75
static __device__ __forceinline__ int group_power(float amax) {
    const uint32_t b = as_u(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
    return e < -126 ? -126 : e > 120 ? 120 : e;
}
static __device__ __forceinline__ float power_of(int e) { return as_f((uint32_t)(e + 127) << 23); }     // -126 <= e <= 127
static __device__ __forceinline__ float finite_abs(float x) { const float a = fabsf(x); return a < __builtin_inff() ? a : 0.f; }     // NaN, inf: 0
// the e from which the code 256 stands for more than the type's largest finite value (2^16, 2^128): magnitudes end at the code below it, 240, there
template <class T> struct TopPower { static constexpr int E = 120; };
template <> struct TopPower<F16> { static constexpr int E = 8; };
// N values of a group -> N codes, four to a word, the first in the low byte. Scaled values end at 448 by the choice of e and NaN converts to NaN: nothing
// else to look at, unless there are infinities or the group is at the type's end (13 848 x 3 072 bf16: 18.0 us with a look at every value, 16.6 without).
static __device__ __forceinline__ float to_encode(float x, float inv, float cap) {
    return fabsf(x) < __builtin_inff() ? __builtin_amdgcn_fmed3f(x * inv, -cap, cap) : __builtin_nanf("");
}
// the power of a group of which this lane and the three lanes STEP, 2 STEP and 3 STEP away (by exclusive or) hold N values each; whether it has infinities
struct GroupPower { int e; bool infinities; };
template <int N, int STEP = 1> static __device__ __forceinline__ GroupPower group_power4(const float (&v)[N]) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]));
    top = fmaxf(top, __shfl_xor(top, STEP));
    top = fmaxf(top, __shfl_xor(top, 2 * STEP));
    if (top < __builtin_inff()) return {group_power(top), false};
    top = 0.f;                                                               // they do not count
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmaxf(top, finite_abs(v[j]));
    top = fmaxf(top, __shfl_xor(top, STEP));
    top = fmaxf(top, __shfl_xor(top, 2 * STEP));
    return {group_power(top), true};
}
template <int N> static __device__ __forceinline__ void encode(const float (&v)[N], GroupPower g, int top_power, uint32_t (&w)[N / 4]) {
    const float inv = power_of(-g.e), cap = g.e >= top_power ? 240.f : 448.f;
    if (g.e < top_power && !g.infinities) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inv, v[4 * i + 1] * inv, 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inv, v[4 * i + 3] * inv, x, true);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const int x = __builtin_amdgcn_cvt_pk_fp8_f32(to_encode(v[4 * i], inv, cap), to_encode(v[4 * i + 1], inv, cap), 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(to_encode(v[4 * i + 2], inv, cap), to_encode(v[4 * i + 3], inv, cap), x, true);
    }
}
static __device__ __forceinline__ void values4(uint32_t w, float s, float (&v)[4]) {
    v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s;
    v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s;
    v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s;
    v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s;
}

// ---- what a rounding to 16 bits left of a value, in a signed byte: the difference of the two floats' bits, in 1/128ths of half a step (0 where nothing is left; below
// fp16's 2^-14, whose steps are wider than its numbers' bits, what fits) ----
template <class T> struct Rest {
    static constexpr bool ON = sizeof(typename T::elem) == 2;
    static constexpr int SHIFT = T::DT == ATLAS_TRAIN_F16 ? 5 : 8;
    static __device__ __forceinline__ uint32_t code(float value, float rounded) {
        const int d = (int)(as_u(value) - as_u(rounded) + (1u << (SHIFT - 1))) >> SHIFT;
        return (uint32_t)(d < -128 ? -128 : d > 127 ? 127 : d) & 0xffu;
    }
    static __device__ __forceinline__ float value(float rounded, uint32_t codes, int byte) {
        return as_f(as_u(rounded) + ((uint32_t)__builtin_amdgcn_sbfe((int)codes, 8 * byte, 8) << SHIFT));
    }
};
// of four values that become two words
template <class T> static __device__ __forceinline__ uint32_t rest4(const float* v) {
    const uint32_t a = pack2<T>(v[0], v[1]), b = pack2<T>(v[2], v[3]);
    return Rest<T>::code(v[0], T::ld((uint16_t)a)) | Rest<T>::code(v[1], T::ld((uint16_t)(a >> 16))) << 8 | Rest<T>::code(v[2], T::ld((uint16_t)b)) << 16 |
           Rest<T>::code(v[3], T::ld((uint16_t)(b >> 16))) << 24;
}

// two codes (the low or the high half of a word) -> two values in the 16-bit type: gfx950's scaled conversion, the scale a power of two
template <class T, bool HIGH> static __device__ __forceinline__ uint32_t values2(uint32_t w, float s) {
    if constexpr (T::DT == ATLAS_TRAIN_F16) { const h2 v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, HIGH); return __builtin_bit_cast(uint32_t, v); }
    else { const b2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s, HIGH); return __builtin_bit_cast(uint32_t, v); }
}

// ---- GELU (exact erf form) and its derivative Phi(z) + z phi(z) ----
// tail = erfc(|z| / sqrt 2) = 2^P(|z| / sqrt 2), P a degree-8 polynomial without constant term fitted to log2 erfc on [0, 4] (the encoder's:
// |error of erf| <= 1.1e-7); Phi(z) = 1 - tail / 2 for z >= 0 and tail / 2 below, without cancellation. One v_exp_f32 and 9 multiply-adds where
// erfcf takes some 60 instructions and a branch: the dz pass of 13 848 x 3 072 fp16 went from 91 to 60 us with it.
static __device__ __forceinline__ float half_tail(float a /* |z| */) {
    float p = -2.83505892e-06f;                                               // the encoder's coefficients by powers of 1 / sqrt 2
    p = __builtin_fmaf(p, a, 3.93791197e-05f);
    p = __builtin_fmaf(p, a, -0.000186185687f);
    p = __builtin_fmaf(p, a, -0.000136926086f);
    p = __builtin_fmaf(p, a, 0.00706340978f);
    p = __builtin_fmaf(p, a, -0.0524961762f);
    p = __builtin_fmaf(p, a, -0.45920819f);
    p = __builtin_fmaf(p, a, -1.15110517f);
    return exp2_fast(__builtin_fmaf(p, a, -1.0f));
}
static __device__ __forceinline__ float gelu(float z) {                      // z Phi(z) = max(z, 0) - |z| tail / 2
    const float a = fabsf(z);
    return __builtin_fmaf(-fminf(a, 3e38f), half_tail(a), fmaxf(z, 0.f));     // (infinity times a tail of 0 is no number; a NaN comes through the tail)
}
static __device__ __forceinline__ float gelu_slope(float z) {
    const float h = half_tail(fabsf(z)), cdf = z >= 0.f ? 1.f - h : h, bounded = __builtin_amdgcn_fmed3f(z, -3e38f, 3e38f);     // (as above; a NaN comes through cdf)
    return __builtin_fmaf(bounded * 0.3989422804014327f, exp2_fast(z * z * -0.72134752044448170f), cdf);    // phi(z) = 2^(-z^2 log2(e) / 2) / sqrt(2 pi)
}

}  // namespace atlas_train
