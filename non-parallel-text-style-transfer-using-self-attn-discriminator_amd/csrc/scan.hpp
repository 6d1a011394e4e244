// Gated linear recurrence (functional.gated_scan): forward, backward, one-token step.
//
//   s_t = sigmoid(-f_t) = 1 - a_t ,  h_t = h_{t-1} + s_t (x_t - h_{t-1}) ,  y_t = sigmoid(o_t) h_t     (t < len)
//   g_t = dy_t sigmoid(o_t) + a_{t+1} g_{t+1} ,  dx_t = s_t g_t ,  df_t = a_t s_t g_t (h_{t-1} - x_t) ,
//   do_t = dy_t h_t so (1 - so) ,  dh0 = a_1 g_1
//
// The state is one number per channel and the recurrence is linear in it, so unlike the LSTM's it needs no exchange
// between channels (no hand-off between workgroups) and can be cut along time: a stretch of steps is the affine map
// h -> h - M h + v, with M = 1 - prod a.  M obeys the recurrence itself (x = 1, from 0), which keeps its relative error
// small where a is close to one; prod a rounded in fp32 would lose the long memories.  State and maps are fp32.
//
// Bound by memory: 16-bit types move 8 bytes per element forward and 14 backward (11.1 with 8-bit activations) against
// about 60 / 100 issue slots of arithmetic per element pair.  One wave owns 128 channels (two neighbours per lane: 4-byte
// loads, 256 contiguous bytes per row and part) of one sentence and walks over time in blocks of 16 steps; the loads of
// the next block (48 instructions, 12 KB per wave) are in flight while a block is computed.
//
// A training call keeps the state that enters each block (fp32, 1/4 byte per element and step): the backward pass walks
// the blocks from the last to the first, recomputes the 16 states of a block from its kept one in registers and needs
// no second pass over the sequence.
//
// Channels: lane l of a wave holds channels cc, cc + 1 with cc = min(c0, D - 2).  In the last wave of a row the lanes
// past the end repeat channels D-2, D-1 and store the same values to the same addresses, so no load or store is
// predicated and nothing is read past a row's part; odd D and any alignment run the same code.
#pragma once
#include "ckpt8.hpp"
#include "gemm_core.hpp"

namespace sad {

constexpr int SC_STEPS = 16;       // time steps of a block: states kept, loads in flight
constexpr int SC_CH = 128;         // channels of a wave
constexpr float SC_LOG2E = 1.4426950408889634f;

struct ScanP {
    int B, T, D, nblk, ncg;        // nblk = ceil(T / 16), ncg = ceil(D / 128)
    int reverse;
    int nchunk, cblk;              // time chunks per sentence, blocks per chunk
    const void* z; long long z_sb, z_st;
    const int* lengths;
    const float* h0;
    void* y; long long y_sb, y_st;
    float* h_last;
    float* kept;                   // [B][nblk][D]
    unsigned char* codes;          // [B][nblk][parts][D][16], steps in scan order
    unsigned char* exps;           // [B][nblk][parts][ceil(D/32)][16]
    const void* dy; long long dy_sb, dy_st;
    const float* dh_last;
    void* dz; long long dz_sb, dz_st;
    float* dh0;
    float* sums;                   // [B][nchunk][2][D]: (M, v) of a chunk, chunks in the order of the walk
};

// two neighbouring channels of one row
template <int KIND> struct Pair {
    typedef unsigned raw;
    static __device__ __forceinline__ raw load(const void* p) { return *(const u32h*)p; }
    static __device__ __forceinline__ raw zero() { return 0u; }
    static __device__ __forceinline__ f32x2 get(raw r) {
        if constexpr (KIND == SAD_SRC_BF16)
            return f32x2{__builtin_bit_cast(float, r << 16), __builtin_bit_cast(float, r & 0xffff0000u)};
        else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            const h2 h = __builtin_bit_cast(h2, r);
            return f32x2{(float)h[0], (float)h[1]};
        }
    }
    static __device__ __forceinline__ void store(void* p, f32x2 v) {
        if constexpr (KIND == SAD_SRC_BF16) *(u32h*)p = pack_bf16x2(v[0], v[1]);
        else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            *(u32h*)p = __builtin_bit_cast(unsigned, h2{(_Float16)v[0], (_Float16)v[1]});
        }
    }
};
template <> struct Pair<SAD_SRC_F32> {
    typedef f32x2 raw;
    static __device__ __forceinline__ raw load(const void* p) { return *(const f32x2u*)p; }
    static __device__ __forceinline__ raw zero() { return f32x2{0.f, 0.f}; }
    static __device__ __forceinline__ f32x2 get(raw r) { return r; }
    static __device__ __forceinline__ void store(void* p, f32x2 v) { *(f32x2u*)p = v; }
};

// sigmoid(-f); exp2's overflow to infinity gives the limit 0
__device__ __forceinline__ float sc_share(float f) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(SC_LOG2E * f)); }
// p = sigmoid(v) is given together with q = 1 - p at full relative precision: u = e^-v, q = u p where q is the small one
__device__ __forceinline__ void sc_gate(float v, float& p, float& q) {
    const float u = __builtin_amdgcn_exp2f(-SC_LOG2E * v);
    p = __builtin_amdgcn_rcpf(1.0f + u);
    q = p > 0.5f ? u * p : 1.0f - p;
}

// position of a wave
struct ScanAt {
    int b, cg, ord, cc, len, lo, hi;      // ord: chunk in the order of the walk; [lo, hi) its blocks
    bool valid;
};
// `backward`: the walk visits the chunks against the scan's direction
__device__ __forceinline__ ScanAt scan_at(const ScanP& p, bool backward) {
    ScanAt w;
    const int lane = threadIdx.x & 63;
    const unsigned id = blockIdx.x * (blockDim.x >> 6) + (unsigned)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned per = (unsigned)p.ncg * p.nchunk;
    w.b = (int)(id / per);
    const unsigned r = id - (unsigned)w.b * per;
    const int chunk = (int)(r / (unsigned)p.ncg);
    w.cg = (int)(r - (unsigned)chunk * p.ncg);
    w.valid = w.b < p.B;
    w.ord = (p.reverse != 0) != backward ? p.nchunk - 1 - chunk : chunk;
    const int c0 = w.cg * SC_CH + 2 * lane;
    w.cc = c0 < p.D - 2 ? c0 : p.D - 2;
    w.lo = chunk * p.cblk;
    w.hi = w.lo + p.cblk < p.nblk ? w.lo + p.cblk : p.nblk;
    int len = p.T;
    if (w.valid && p.lengths != nullptr) {
        len = __builtin_amdgcn_readfirstlane(p.lengths[w.b]);
        len = len < 0 ? 0 : (len > p.T ? p.T : len);
    }
    w.len = len;
    return w;
}

// (M, v) of every chunk in front of `ord` in the order of the walk, applied to the state h
__device__ __forceinline__ f32x2 scan_enter(const ScanP& p, const ScanAt& w, f32x2 h) {
    const float* q = p.sums + (long long)w.b * p.nchunk * 2 * p.D + w.cc;
    int k = 0;
    for (; k + 8 <= w.ord; k += 8) {
        f32x2 m[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = *(const f32x2u*)(q + (long long)(k + i) * 2 * p.D);
            v[i] = *(const f32x2u*)(q + (long long)(k + i) * 2 * p.D + p.D);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) h[e] = __builtin_fmaf(-m[i][e], h[e], h[e]) + v[i][e];
    }
    for (; k < w.ord; ++k) {
        const f32x2 m = *(const f32x2u*)(q + (long long)k * 2 * p.D), v = *(const f32x2u*)(q + (long long)k * 2 * p.D + p.D);
#pragma unroll
        for (int e = 0; e < 2; ++e) h[e] = __builtin_fmaf(-m[e], h[e], h[e]) + v[e];
    }
    return h;
}

// raw rows of one part of z (or of dy) in scan order; rows past the end of the tensor read the last one
template <int KIND>
__device__ __forceinline__ void sc_load_rows(typename Pair<KIND>::raw (&r)[SC_STEPS], const unsigned char* base, long long st, int kb,
                                             int T, int reverse) {
#pragma unroll
    for (int i = 0; i < SC_STEPS; ++i) {
        const int t = kb * SC_STEPS + (reverse ? SC_STEPS - 1 - i : i);
        r[i] = Pair<KIND>::load(base + (long long)(t < T ? t : T - 1) * st);
    }
}

// Codes of one row of one part: two values per lane, the 16 lanes of a DPP row share the exponent.
// `in0` / `in1`: this lane's entry belongs to the 32 channels of its 16 lanes
template <int KIND>
__device__ __forceinline__ void sc_encode(f32x2 v, bool in0, bool in1, unsigned& u0, unsigned& u1, unsigned& byte) {
    const unsigned b0 = in0 ? c8_abs_bits(v[0]) : 0u, b1 = in1 ? c8_abs_bits(v[1]) : 0u;
    auto row_max = [](unsigned m) {
        auto ror = [](unsigned x, auto c) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(c)::value, 0xf, 0xf, false); };
        unsigned t;
        t = ror(m, std::integral_constant<int, 0x128>{}); m = m > t ? m : t;      // row_ror:8
        t = ror(m, std::integral_constant<int, 0x124>{}); m = m > t ? m : t;
        t = ror(m, std::integral_constant<int, 0x122>{}); m = m > t ? m : t;
        t = ror(m, std::integral_constant<int, 0x121>{}); m = m > t ? m : t;
        return m;
    };
    unsigned top = row_max(b0 > b1 ? b0 : b1);
    const bool bad = __any(top >= C8_NONFINITE);
    if (bad) top = row_max((b0 < C8_NONFINITE ? b0 : 0u) > (b1 < C8_NONFINITE ? b1 : 0u) ? (b0 < C8_NONFINITE ? b0 : 0u)
                                                                                         : (b1 < C8_NONFINITE ? b1 : 0u));
    const int e = c8_exponent<KIND>(top);
    const float inv = c8_inv_scale(e), cap = e == C8Range<KIND>::hi + 127 ? 63.f : 127.f;
    u0 = c8_code(v[0], inv, cap);
    u1 = c8_code(v[1], inv, cap);
    if (bad) {
        if (c8_abs_bits(v[0]) >= C8_NONFINITE) u0 = C8_LOST;
        if (c8_abs_bits(v[1]) >= C8_NONFINITE) u1 = C8_LOST;
    }
    byte = (unsigned)e;
}

// Forward.  SAVE: 0 nothing, 1 the state entering each block, 2 that and the 8-bit codes of z.
template <int KIND, bool GATED, int SAVE>
__global__ __launch_bounds__(256) void k_scan_fwd(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at(p, false);
    if (!w.valid) return;
    const int lane = threadIdx.x & 63;
    const long long zst = p.z_st * EB, yst = p.y_st * EB;
    const unsigned char* zx = (const unsigned char*)p.z + (w.b * p.z_sb + w.cc) * EB;
    const unsigned char* zf = zx + (long long)p.D * EB;
    const unsigned char* zo = zf + (long long)p.D * EB;
    unsigned char* yp = (unsigned char*)p.y + (w.b * p.y_sb + w.cc) * EB;
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi;     // blocks that hold a valid step
    for (int kb = hi > w.lo ? hi : w.lo; kb < w.hi; ++kb)                                 // blocks behind the sentence
        for (int i = 0; i < SC_STEPS; ++i)
            if (kb * SC_STEPS + i < p.T) Pair<KIND>::store(yp + (long long)(kb * SC_STEPS + i) * yst, f32x2{0.f, 0.f});
    f32x2 h = p.h0 != nullptr ? (f32x2)*(const f32x2u*)(p.h0 + (long long)w.b * p.D + w.cc) : f32x2{0.f, 0.f};
    if (p.nchunk > 1) h = scan_enter(p, w, h);

    const int c0 = w.cg * SC_CH + 2 * lane;
    const bool own0 = c0 < p.D && w.cc == c0, own1 = c0 < p.D;      // the lane's own channels among (cc, cc + 1)
    raw nx[SC_STEPS], nf[SC_STEPS], no[SC_STEPS];
    auto issue = [&](int kb) {
        sc_load_rows<KIND>(nx, zx, zst, kb, p.T, p.reverse);
        sc_load_rows<KIND>(nf, zf, zst, kb, p.T, p.reverse);
        if constexpr (GATED) sc_load_rows<KIND>(no, zo, zst, kb, p.T, p.reverse);
    };
    const int n = hi - w.lo;
    if (n > 0) issue(p.reverse ? hi - 1 : w.lo);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? hi - 1 - it : w.lo + it;
        raw x[SC_STEPS], f[SC_STEPS], o[SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) {
            x[i] = nx[i];
            f[i] = nf[i];
            if constexpr (GATED) o[i] = no[i];
        }
        if (it + 1 < n) issue(p.reverse ? kb - 1 : kb + 1);
        if constexpr (SAVE > 0) *(f32x2u*)(p.kept + ((long long)w.b * p.nblk + kb) * p.D + w.cc) = h;
        unsigned code[SAVE == 2 ? PARTS : 1][2][4], eb[SAVE == 2 ? PARTS : 1][4];
        auto block = [&](auto full) {
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) {
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const bool ok = decltype(full)::value || t < w.len;
                const f32x2 xv = Pair<KIND>::get(x[i]), fv = Pair<KIND>::get(f[i]);
                f32x2 hn, ov;
#pragma unroll
                for (int e = 0; e < 2; ++e) hn[e] = __builtin_fmaf(sc_share(fv[e]), xv[e] - h[e], h[e]);
                if (ok) h = hn;                                     // uniform
                f32x2 yv = h;
                if constexpr (GATED) {
                    ov = Pair<KIND>::get(o[i]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) yv[e] = h[e] * sigmoidf_(ov[e]);
                }
                if (!ok) yv = f32x2{0.f, 0.f};
                if (decltype(full)::value || t < p.T) Pair<KIND>::store(yp + (long long)t * yst, yv);
                if constexpr (SAVE == 2) {
                    unsigned u0, u1, e;
                    auto put = [&](int q, f32x2 v) {
                        sc_encode<KIND>(v, own0, own1, u0, u1, e);
                        const int sh = 8 * (i & 3);
                        if ((i & 3) == 0) { code[q][0][i >> 2] = u0; code[q][1][i >> 2] = u1; eb[q][i >> 2] = e; }
                        else { code[q][0][i >> 2] |= u0 << sh; code[q][1][i >> 2] |= u1 << sh; eb[q][i >> 2] |= e << sh; }
                    };
                    put(0, xv);
                    put(1, fv);
                    if constexpr (GATED) put(2, ov);
                }
            }
        };
        if ((kb + 1) * SC_STEPS <= w.len) block(std::integral_constant<bool, true>{});
        else block(std::integral_constant<bool, false>{});
        if constexpr (SAVE == 2) {
            const int nb = (p.D + C8_BLOCK - 1) / C8_BLOCK;
            const long long tile = ((long long)w.b * p.nblk + kb) * PARTS;
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                unsigned char* cp = p.codes + ((tile + q) * p.D + w.cc) * SC_STEPS;
                if (own0) *(u32x4*)cp = u32x4{code[q][0][0], code[q][0][1], code[q][0][2], code[q][0][3]};
                if (own1) *(u32x4*)(cp + SC_STEPS) = u32x4{code[q][1][0], code[q][1][1], code[q][1][2], code[q][1][3]};
                if ((lane & 15) == 0 && own1)
                    *(u32x4*)(p.exps + ((tile + q) * nb + c0 / C8_BLOCK) * SC_STEPS) = u32x4{eb[q][0], eb[q][1], eb[q][2], eb[q][3]};
            }
        }
    }
    if (w.ord == p.nchunk - 1) *(f32x2u*)(p.h_last + (long long)w.b * p.D + w.cc) = h;
}

// (M, v) of one chunk, forward: the chunk's steps from the zero state.
template <int KIND>
__global__ __launch_bounds__(256) void k_scan_sum(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at(p, false);
    if (!w.valid || w.ord == p.nchunk - 1) return;                  // the last chunk's map is not needed
    const long long zst = p.z_st * EB;
    const unsigned char* zx = (const unsigned char*)p.z + (w.b * p.z_sb + w.cc) * EB;
    const unsigned char* zf = zx + (long long)p.D * EB;
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi, n = hi - w.lo;
    f32x2 h{0.f, 0.f}, m{0.f, 0.f};
    raw nx[SC_STEPS], nf[SC_STEPS];
    auto issue = [&](int kb) {
        sc_load_rows<KIND>(nx, zx, zst, kb, p.T, p.reverse);
        sc_load_rows<KIND>(nf, zf, zst, kb, p.T, p.reverse);
    };
    if (n > 0) issue(p.reverse ? hi - 1 : w.lo);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? hi - 1 - it : w.lo + it;
        raw x[SC_STEPS], f[SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) { x[i] = nx[i]; f[i] = nf[i]; }
        if (it + 1 < n) issue(p.reverse ? kb - 1 : kb + 1);
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) {
            const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
            const f32x2 xv = Pair<KIND>::get(x[i]), fv = Pair<KIND>::get(f[i]);
            if (t < w.len) {                                        // uniform
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float s = sc_share(fv[e]);
                    h[e] = __builtin_fmaf(s, xv[e] - h[e], h[e]);
                    m[e] = __builtin_fmaf(s, 1.0f - m[e], m[e]);
                }
            }
        }
    }
    float* q = p.sums + ((long long)w.b * p.nchunk + w.ord) * 2 * p.D + w.cc;
    *(f32x2u*)q = m;
    *(f32x2u*)(q + p.D) = h;
}

// What a block of the backward pass reads of z: the rows themselves, or codes and exponents.
template <int KIND, int PARTS, bool CODES> struct ScanIn;
template <int KIND, int PARTS> struct ScanIn<KIND, PARTS, false> {
    typename Pair<KIND>::raw r[PARTS][SC_STEPS];
    template <int Q> __device__ __forceinline__ void load(const ScanP& p, const ScanAt& w, int kb) {
        sc_load_rows<KIND>(r[Q], (const unsigned char*)p.z + (w.b * p.z_sb + w.cc + (long long)Q * p.D) * Elem<KIND>::bytes,
                           p.z_st * Elem<KIND>::bytes, kb, p.T, p.reverse);
    }
    template <int Q, int I> __device__ __forceinline__ f32x2 get() const { return Pair<KIND>::get(r[Q][I]); }
};
template <int KIND, int PARTS> struct ScanIn<KIND, PARTS, true> {
    u32x4 c[PARTS][2], e[PARTS][2];
    template <int Q> __device__ __forceinline__ void load(const ScanP& p, const ScanAt& w, int kb) {
        const int nb = (p.D + C8_BLOCK - 1) / C8_BLOCK;
        const long long tile = ((long long)w.b * p.nblk + kb) * PARTS + Q;
        const unsigned char* cp = p.codes + (tile * p.D + w.cc) * SC_STEPS;
        c[Q][0] = *(const u32x4*)cp;
        c[Q][1] = *(const u32x4*)(cp + SC_STEPS);
        const unsigned char* ep = p.exps + tile * nb * SC_STEPS;
        e[Q][1] = *(const u32x4*)(ep + (long long)((w.cc + 1) / C8_BLOCK) * SC_STEPS);
        e[Q][0] = e[Q][1];
        // channels D-2 and D-1 of the last lanes lie in different blocks of 32
        if (p.D % C8_BLOCK == 1) e[Q][0] = *(const u32x4*)(ep + (long long)(w.cc / C8_BLOCK) * SC_STEPS);
    }
    template <int Q, int I> __device__ __forceinline__ f32x2 get() const {
        f32x2 v;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float scale = c8_scale((e[Q][k][I >> 2] >> (8 * (I & 3))) & 0xffu);
            v[k] = c8_value_checked<I & 3>(c[Q][k][I >> 2], scale);
        }
        return v;
    }
};

// Backward.
template <int KIND, bool GATED, bool CODES>
__global__ __launch_bounds__(256) void k_scan_bwd(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at(p, true);
    if (!w.valid) return;
    const long long dyst = p.dy_st * EB, dzst = p.dz_st * EB;
    const unsigned char* dyp = (const unsigned char*)p.dy + (w.b * p.dy_sb + w.cc) * EB;
    unsigned char* gx = (unsigned char*)p.dz + (w.b * p.dz_sb + w.cc) * EB;
    unsigned char* gf = gx + (long long)p.D * EB;
    unsigned char* go = gf + (long long)p.D * EB;
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi, n = hi - w.lo;
    for (int kb = hi > w.lo ? hi : w.lo; kb < w.hi; ++kb)
        for (int i = 0; i < SC_STEPS; ++i) {
            const int t = kb * SC_STEPS + i;
            if (t < p.T) {
                Pair<KIND>::store(gx + t * dzst, f32x2{0.f, 0.f});
                Pair<KIND>::store(gf + t * dzst, f32x2{0.f, 0.f});
                if constexpr (GATED) Pair<KIND>::store(go + t * dzst, f32x2{0.f, 0.f});
            }
        }
    f32x2 carry = p.dh_last != nullptr ? (f32x2)*(const f32x2u*)(p.dh_last + (long long)w.b * p.D + w.cc) : f32x2{0.f, 0.f};
    if (p.nchunk > 1) carry = scan_enter(p, w, carry);

    ScanIn<KIND, PARTS, CODES> nin;
    raw ndy[SC_STEPS];
    f32x2 nh;
    auto issue = [&](int kb) {
        nh = *(const f32x2u*)(p.kept + ((long long)w.b * p.nblk + kb) * p.D + w.cc);
        nin.template load<0>(p, w, kb);
        nin.template load<1>(p, w, kb);
        if constexpr (GATED) nin.template load<2>(p, w, kb);
        if (p.dy != nullptr) sc_load_rows<KIND>(ndy, dyp, dyst, kb, p.T, p.reverse);
        else {
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) ndy[i] = Pair<KIND>::zero();
        }
    };
    if (n > 0) issue(p.reverse ? w.lo : hi - 1);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? w.lo + it : hi - 1 - it;
        const ScanIn<KIND, PARTS, CODES> in = nin;
        const f32x2 enter = nh;
        raw dy[SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) dy[i] = ndy[i];
        if (it + 1 < n) issue(p.reverse ? kb + 1 : kb - 1);
        auto block = [&](auto full) {
            f32x2 h[SC_STEPS], s[SC_STEPS];
            f32x2 hc = enter;
            static_for<SC_STEPS>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const f32x2 xv = in.template get<0, i>(), fv = in.template get<1, i>();
                f32x2 hn;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[i][e] = sc_share(fv[e]);
                    hn[e] = __builtin_fmaf(s[i][e], xv[e] - hc[e], hc[e]);
                }
                if (decltype(full)::value || t < w.len) hc = hn;    // uniform
                h[i] = hc;
            });
            static_for<SC_STEPS>([&](auto jc) {
                constexpr int i = SC_STEPS - 1 - decltype(jc)::value;
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const bool ok = decltype(full)::value || t < w.len;
                const f32x2 xv = in.template get<0, i>(), fv = in.template get<1, i>(), dyv = Pair<KIND>::get(dy[i]);
                f32x2 dx, df, dov, cn;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float hp = i == 0 ? enter[e] : h[i == 0 ? 0 : i - 1][e];
                    float dh = dyv[e];
                    if constexpr (GATED) {
                        float so, sq;
                        sc_gate(in.template get<2, i>()[e], so, sq);
                        dh *= so;
                        dov[e] = dh * h[i][e] * sq;
                    }
                    const float g = dh + carry[e], sv = s[i][e];
                    const float a = sv < 0.5f ? 1.0f - sv : __builtin_amdgcn_exp2f(SC_LOG2E * fv[e]) * sv;
                    dx[e] = sv * g;
                    df[e] = a * dx[e] * (hp - xv[e]);
                    cn[e] = __builtin_fmaf(-sv, g, g);
                }
                if (ok) carry = cn;                                 // uniform
                else dx = df = dov = f32x2{0.f, 0.f};
                if (decltype(full)::value || t < p.T) {
                    Pair<KIND>::store(gx + t * dzst, dx);
                    Pair<KIND>::store(gf + t * dzst, df);
                    if constexpr (GATED) Pair<KIND>::store(go + t * dzst, dov);
                }
            });
        };
        if ((kb + 1) * SC_STEPS <= w.len) block(std::integral_constant<bool, true>{});
        else block(std::integral_constant<bool, false>{});
    }
    if (p.dh0 != nullptr && w.ord == p.nchunk - 1) *(f32x2u*)(p.dh0 + (long long)w.b * p.D + w.cc) = carry;
}

// (M, v) of one chunk, backward: carry -> carry - M carry + v.
template <int KIND, bool GATED, bool CODES>
__global__ __launch_bounds__(256) void k_scan_bsum(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at(p, true);
    if (!w.valid || w.ord == p.nchunk - 1) return;
    const long long dyst = p.dy_st * EB;
    const unsigned char* dyp = (const unsigned char*)p.dy + (w.b * p.dy_sb + w.cc) * EB;
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi, n = hi - w.lo;
    f32x2 v{0.f, 0.f}, m{0.f, 0.f};
    ScanIn<KIND, PARTS, CODES> nin;
    raw ndy[SC_STEPS];
    auto issue = [&](int kb) {
        nin.template load<1>(p, w, kb);
        if constexpr (GATED) nin.template load<2>(p, w, kb);
        if (p.dy != nullptr) sc_load_rows<KIND>(ndy, dyp, dyst, kb, p.T, p.reverse);
        else {
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) ndy[i] = Pair<KIND>::zero();
        }
    };
    if (n > 0) issue(p.reverse ? w.lo : hi - 1);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? w.lo + it : hi - 1 - it;
        const ScanIn<KIND, PARTS, CODES> in = nin;
        raw dy[SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) dy[i] = ndy[i];
        if (it + 1 < n) issue(p.reverse ? kb + 1 : kb - 1);
        static_for<SC_STEPS>([&](auto jc) {
            constexpr int i = SC_STEPS - 1 - decltype(jc)::value;
            const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
            if (t < w.len) {                                        // uniform
                const f32x2 fv = in.template get<1, i>(), dyv = Pair<KIND>::get(dy[i]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float dh = dyv[e];
                    if constexpr (GATED) dh *= sigmoidf_(in.template get<2, i>()[e]);
                    const float s = sc_share(fv[e]), g = dh + v[e];
                    v[e] = __builtin_fmaf(-s, g, g);
                    m[e] = __builtin_fmaf(s, 1.0f - m[e], m[e]);
                }
            }
        });
    }
    float* q = p.sums + ((long long)w.b * p.nchunk + w.ord) * 2 * p.D + w.cc;
    *(f32x2u*)q = m;
    *(f32x2u*)(q + p.D) = v;
}

// One token.  `alive` (nullable): a sentence that has ended keeps its state and gives y = 0.  h_out may be h: every
// channel is read before it is written, by the lane that writes it (no channel is repeated here).
template <int KIND, bool GATED>
__global__ __launch_bounds__(256) void k_scan_step(int D, int per, const void* __restrict__ z, long long z_sb, const float* h, long long h_sb,
                                                  const unsigned char* __restrict__ alive, void* __restrict__ y, long long y_sb,
                                                  float* h_out, long long ho_sb) {
    const int b = blockIdx.x / per, c = (blockIdx.x - b * per) * 256 + threadIdx.x;     // per: workgroups of a sentence
    if (c >= D) return;
    const long long zo = (long long)b * z_sb + c;
    const float hp = h[(long long)b * h_sb + c];
    const float x = Elem<KIND>::load(z, zo), f = Elem<KIND>::load(z, zo + D);
    float hn = __builtin_fmaf(sc_share(f), x - hp, hp), yv = hn;
    if constexpr (GATED) yv *= sigmoidf_(Elem<KIND>::load(z, zo + 2ll * D));
    const bool live = alive == nullptr || alive[b] != 0;
    Elem<KIND>::store(y, (long long)b * y_sb + c, live ? yv : 0.f);
    h_out[(long long)b * ho_sb + c] = live ? hn : hp;
}

}  // namespace sad
