// 8-bit activation checkpoints: the number format and its stand-alone kernels.
//
// Format: 32 channels of a row share one exponent e, the smallest with max|x| <= 127 * 2^e over the FINITE entries;
// an entry is the code rint(x / 2^e) (ties to even) in [-127, 127].  Codes are signed bytes (a conversion with a
// sign-extended byte operand reads one of four), exponents e + 127: the byte IS the exponent field of the float 2^e.
//   * every restored value code * 2^e has at most 7 significant bits, so it is exact in bf16 and (with the fp16 range
//     of e below) in fp16: a checkpoint can feed a matrix instruction without a second rounding;
//   * a power-of-two step costs up to one bit against a free scale (64..127 codes used on each side) and makes encode
//     and decode exact but for the one rounding to the code: error <= 2^e / 2 per entry;
//   * code -128 marks a non-finite entry: it comes back as NaN, its 31 neighbours are not touched.  A block that holds one
//     has the exponent byte 255 and its exponent in a second array, which is neither written nor read otherwise: readers
//     test one byte per block instead of every code;
//   * e is clamped to [-126, 122] (fp16: [-24, 10]).  At the upper end the code stops at +-63, where 64 would restore
//     to infinity; at the lower end 2^e stays a normal float (fp16: the spacing of its subnormals).
#pragma once
#include "common.hpp"
#include "../../include/sad.h"

namespace sad {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));     // dword-aligned 8-byte access
typedef unsigned u32h __attribute__((aligned(2)));                        // 2-byte-aligned 4-byte access
typedef unsigned u32x2w __attribute__((ext_vector_type(2), aligned(4)));  // dword-aligned 8-byte access

constexpr int C8_BLOCK = 32;                       // channels that share an exponent
constexpr unsigned C8_NONFINITE = 0x7f800000u;     // |bits| of the smallest non-finite float

template <int KIND> struct C8Range { static constexpr int lo = KIND == SAD_SRC_F16 ? -24 : -126, hi = KIND == SAD_SRC_F16 ? 10 : 122; };

// exponent byte of a block whose largest finite |x| has the bits `top`
template <int KIND>
__device__ __forceinline__ int c8_exponent(unsigned top) {
    // top = 1.m * 2^(E-127): 127 * 2^e reaches it from e = E - 133 on if 1.m <= 127/64, one later otherwise
    const int e = (int)(top >> 23) - 133 + 127 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    const int lo = C8Range<KIND>::lo + 127, hi = C8Range<KIND>::hi + 127;
    return e < lo ? lo : (e > hi ? hi : e);
}
__device__ __forceinline__ float c8_scale(int byte) { return __builtin_bit_cast(float, (unsigned)byte << 23); }
__device__ __forceinline__ float c8_inv_scale(int byte) { return __builtin_bit_cast(float, (unsigned)(254 - byte) << 23); }
__device__ __forceinline__ unsigned c8_abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }
// code of a finite x, as a byte; `cap` = 127, or 63 in a block at the upper exponent clamp.  x * 2^-e is exact or far
// below half a code, so this is the format's only rounding.
__device__ __forceinline__ unsigned c8_code(float x, float inv, float cap) {
    const float q = __builtin_amdgcn_fmed3f(__builtin_rintf(x * inv), -cap, cap);
    return (unsigned)(int)q & 0xffu;
}
constexpr unsigned C8_LOST = 0x80u;                // code of a non-finite entry
constexpr unsigned C8_MARK = 255u;                 // exponent byte of a block that holds one
// code N of w: one conversion with a sign-extended byte operand (from C++ the compiler makes two or three instructions)
template <int N>
__device__ __forceinline__ float c8_int(unsigned w) {
    float r;
    if constexpr (N == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(r) : "v"(w));
    if constexpr (N == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(r) : "v"(w));
    if constexpr (N == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(r) : "v"(w));
    if constexpr (N == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(r) : "v"(w));
    return r;
}
// ... times 2^e: exact
template <int N>
__device__ __forceinline__ float c8_value(unsigned w, float scale) { return c8_int<N>(w) * scale; }
template <int N>
__device__ __forceinline__ bool c8_is_lost(unsigned w) { return ((w >> (8 * N)) & 0xffu) == C8_LOST; }
template <int N>
__device__ __forceinline__ float c8_value_checked(unsigned w, float scale) {
    return c8_is_lost<N>(w) ? __builtin_nanf("") : c8_value<N>(w, scale);
}

// ---- element conversions ------------------------------------------------------------------------------------------
template <int KIND> struct Elem;
template <> struct Elem<SAD_SRC_F32> {
    static constexpr int bytes = 4;
    static __device__ __forceinline__ float load(const void* p, long long i) { return ((const float*)p)[i]; }
    static __device__ __forceinline__ void store(void* p, long long i, float v) { ((float*)p)[i] = v; }
};
template <> struct Elem<SAD_SRC_BF16> {
    static constexpr int bytes = 2;
    static __device__ __forceinline__ float load(const void* p, long long i) { return bf16_to_f32(((const bf16raw*)p)[i]); }
    static __device__ __forceinline__ void store(void* p, long long i, float v) { ((bf16raw*)p)[i] = f32_to_bf16(v); }
};
template <> struct Elem<SAD_SRC_F16> {
    static constexpr int bytes = 2;
    static __device__ __forceinline__ float load(const void* p, long long i) { return (float)((const _Float16*)p)[i]; }
    static __device__ __forceinline__ void store(void* p, long long i, float v) { ((_Float16*)p)[i] = (_Float16)v; }
};

// Rows of a [n0, n1, C] tensor with unit channel stride: row m = i0 * n1 + i1 starts at i0 * s0 + i1 * s1.
struct Rows2 {
    long long s0, s1;
    unsigned n1;
    __device__ __forceinline__ long long at(unsigned m) const {
        const unsigned i0 = m / n1, i1 = m - i0 * n1;
        return (long long)i0 * s0 + (long long)i1 * s1;
    }
};

// 16 consecutive elements of a row; those at or past C read as zero
template <int KIND>
__device__ __forceinline__ void c8_load16(float (&v)[16], const void* row, int c, int C) {
    if (c + 16 <= C) {
        if constexpr (KIND == SAD_SRC_F32) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 r = *(const f32x4u*)((const float*)row + c + 4 * q);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * q + i] = r[i];
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const u32x4 r = *(const u32x4h*)((const unsigned short*)row + c + 8 * q);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned short h = (unsigned short)(r[i >> 1] >> (16 * (i & 1)));
                    v[8 * q + i] = KIND == SAD_SRC_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = c + i < C ? Elem<KIND>::load(row, c + i) : 0.f;
    }
}

// Thread layout of both kernels: a thread holds 16 channels of a row, `per` = 2 * ceil(C / 32) threads cover a row, a
// workgroup holds `rpb` = max(1, 256 / per) rows; two neighbouring lanes share an exponent.  Bound by memory: 16-bit
// types move 3.03 bytes per element each way; [65536, 2048] bf16: save 84 us (4.9 TB/s), restore 68 us (6.0 TB/s).
template <int KIND>
__global__ __launch_bounds__(256) void k_ckpt8_save(int rows, int C, int per, int rpb, const void* __restrict__ x, Rows2 xr,
                                                   unsigned char* __restrict__ codes, unsigned char* __restrict__ exps,
                                                   unsigned char* __restrict__ marked) {
    const int r = (int)threadIdx.x / per, row = blockIdx.x * rpb + r;
    if (r >= rpb && rpb > 1) return;
    if (row >= rows) return;
    const char* xp = (const char*)x + xr.at((unsigned)row) * Elem<KIND>::bytes;
    for (int q = rpb > 1 ? (int)threadIdx.x - r * per : (int)threadIdx.x; q < per; q += 256) {
        float v[16];
        c8_load16<KIND>(v, xp, q * 16, C);
        unsigned top = 0u, all = 0u;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const unsigned b = c8_abs_bits(v[i]);
            all = all > b ? all : b;
        }
        top = all;
        if (all >= C8_NONFINITE) {
            top = 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const unsigned b = c8_abs_bits(v[i]);
                if (b < C8_NONFINITE && b > top) top = b;
            }
        }
        const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false);   // quad_perm [1,0,3,2]
        top = top > other ? top : other;
        const int e = c8_exponent<KIND>(top);
        const float inv = c8_inv_scale(e), cap = e == C8Range<KIND>::hi + 127 ? 63.f : 127.f;
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[k] |= c8_code(v[4 * k + i], inv, cap) << (8 * i);
        }
        const unsigned pair = (unsigned)__builtin_amdgcn_update_dpp(0, (int)all, 0xB1, 0xf, 0xf, false);
        const bool lost = all >= C8_NONFINITE || pair >= C8_NONFINITE;
        if (all >= C8_NONFINITE) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (c8_abs_bits(v[i]) >= C8_NONFINITE) w[i >> 2] = (w[i >> 2] & ~(0xffu << (8 * (i & 3)))) | (C8_LOST << (8 * (i & 3)));
        }
        *(u32x4*)(codes + ((long long)row * per + q) * 16) = w;
        if ((q & 1) == 0) {
            const long long at = (long long)row * (per >> 1) + (q >> 1);
            exps[at] = lost ? (unsigned char)C8_MARK : (unsigned char)e;
            if (lost) marked[at] = (unsigned char)e;
        }
    }
}

template <int KIND>
__global__ __launch_bounds__(256) void k_ckpt8_restore(int rows, int C, int per, int rpb, const unsigned char* __restrict__ codes,
                                                      const unsigned char* __restrict__ exps,
                                                      const unsigned char* __restrict__ marked, void* __restrict__ out) {
    const int r = (int)threadIdx.x / per, row = blockIdx.x * rpb + r;
    if (r >= rpb && rpb > 1) return;
    if (row >= rows) return;
    char* op = (char*)out + (long long)row * C * Elem<KIND>::bytes;
    for (int q = rpb > 1 ? (int)threadIdx.x - r * per : (int)threadIdx.x; q < per; q += 256) {
        const u32x4 w = *(const u32x4*)(codes + ((long long)row * per + q) * 16);
        const long long at = (long long)row * (per >> 1) + (q >> 1);
        const unsigned byte = exps[at];
        float v[16];
        if (byte != C8_MARK) {
            const float scale = c8_scale((int)byte);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[4 * k + 0] = c8_value<0>(w[k], scale);
                v[4 * k + 1] = c8_value<1>(w[k], scale);
                v[4 * k + 2] = c8_value<2>(w[k], scale);
                v[4 * k + 3] = c8_value<3>(w[k], scale);
            }
        } else {
            const float scale = c8_scale((int)marked[at]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[4 * k + 0] = c8_value_checked<0>(w[k], scale);
                v[4 * k + 1] = c8_value_checked<1>(w[k], scale);
                v[4 * k + 2] = c8_value_checked<2>(w[k], scale);
                v[4 * k + 3] = c8_value_checked<3>(w[k], scale);
            }
        }
        const int c = q * 16;
        if (c + 16 <= C) {
            if constexpr (KIND == SAD_SRC_F32) {
#pragma unroll
                for (int k = 0; k < 4; ++k) *(f32x4u*)((float*)op + c + 4 * k) = f32x4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    u32x4 o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = v[8 * k + 2 * i], b = v[8 * k + 2 * i + 1];
                        if constexpr (KIND == SAD_SRC_BF16) o[i] = pack_bf16x2(a, b);
                        else o[i] = (unsigned)__builtin_bit_cast(unsigned short, (_Float16)a) |
                                    ((unsigned)__builtin_bit_cast(unsigned short, (_Float16)b) << 16);
                    }
                    *(u32x4h*)((unsigned short*)op + c + 8 * k) = o;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (c + i < C) Elem<KIND>::store(op, c + i, v[i]);
        }
    }
}

}  // namespace sad
