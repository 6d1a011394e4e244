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
// Where the sentences and channels alone do not fill the card, a first launch (k_scan_sum / k_scan_bsum) computes the maps
// of the time chunks: it reads x and f (backward: f, o, dy) once more than necessary.  A workgroup joins the maps of four
// neighbouring chunks, so that a wave of the main launch applies at most 15 + 1 of them to find its entering state.
//
// Bound by memory.  One wave owns 128 channels (two neighbours per lane: 4-byte loads, 256 contiguous bytes per row and part)
// of one sentence and walks over time in blocks of 16 steps; the loads of the next block (48 instructions, 12 KB per wave)
// are in flight while a block is computed.  16-bit types move 8 bytes per element forward (11 with 8-bit codes written) and
// 14 backward (11 with codes read).  Measured, bf16: [8, 4096, 2048] with 8-bit activations, forward 145 us = 5.2 TB/s of
// 754 MB, backward 159 us = 4.8 TB/s of 762 MB (a copy of 2 GB: 4.9 TB/s), their sums 83 and 86 us (3.3 TB/s);
// [1024, 32, 512] ragged, forward 28 us, backward 37 us; [64, 23, 512] ragged 6.6 and 10 us (latency of two blocks).
// Channel counts whose rows do not start on lines cost more, as a wave's 256 bytes then lie in three lines instead of two: a
// training call at [64, 500, 960] takes 171 us, at [64, 500, 1000] 207.
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
constexpr int SC_GROUP = 4;        // time chunks whose maps one workgroup joins
// how a block is computed: every step valid; every row inside the tensor, steps behind the sentence masked by selects; rows
// past the end of the tensor
constexpr int SC_FULL = 2, SC_INSIDE = 1, SC_EDGE = 0;
constexpr float SC_LOG2E = 1.4426950408889634f;

struct ScanP {
    int B, T, D, nblk, ncg;        // nblk = ceil(T / 16), ncg = ceil(D / 128)
    int reverse;
    int nchunk, cblk;              // time chunks per sentence, blocks per chunk
    int group, ngroup;             // chunks of a group (waves of a summing workgroup), groups per sentence
    const void* z; long long z_sb, z_st;
    const int* lengths;
    const float* h0;
    void* y; long long y_sb, y_st;
    float* h_last;
    float* kept;                   // [B][nblk][D]
    unsigned char* codes;          // [B][nblk][parts][D][16], steps in scan order
    unsigned char* exps;           // [B][nblk][parts][ceil(D/32)][16]
    unsigned* lost;                // [B][nblk][ncg]: does a wave's block hold a lost (non-finite) entry
    const void* dy; long long dy_sb, dy_st;
    const float* dh_last;
    void* dz; long long dz_sb, dz_st;
    float* dh0;
    float* sums;                   // [B][nchunk][2][D]: (M, v) of the chunks of its group in front of a chunk, in the order of
                                   // the walk; then [B][ngroup][2][D]: (M, v) of a group
};

// two neighbouring channels of one row
template <int KIND> struct Pair {
    typedef unsigned raw;
    static __device__ __forceinline__ raw load(const void* p) { return *(const u32h*)p; }
    static __device__ __forceinline__ raw zero() { return 0u; }
    // magnitudes as ordered integers, the first non-finite one, and the float such an integer stands for
    static constexpr unsigned nonfinite = KIND == SAD_SRC_BF16 ? 0x7f80u : 0x7c00u;
    static __device__ __forceinline__ unsigned mag(raw r, int e) { return e == 0 ? r & 0x7fffu : (r >> 16) & 0x7fffu; }
    static __device__ __forceinline__ float mag_value(unsigned m) {
        if constexpr (KIND == SAD_SRC_BF16) return __builtin_bit_cast(float, m << 16);
        else return (float)__builtin_bit_cast(_Float16, (unsigned short)m);
    }
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
    static constexpr unsigned nonfinite = C8_NONFINITE;
    static __device__ __forceinline__ unsigned mag(raw r, int e) { return c8_abs_bits(r[e]); }
    static __device__ __forceinline__ float mag_value(unsigned m) { return __builtin_bit_cast(float, m); }
    static __device__ __forceinline__ f32x2 get(raw r) { return r; }
    static __device__ __forceinline__ void store(void* p, f32x2 v) { *(f32x2u*)p = v; }
};

// sigmoid(-f); exp2's overflow to infinity gives the limit 0
__device__ __forceinline__ float sc_share(float f) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(SC_LOG2E * f)); }
// u = 2^arg with arg kept where 1 + u and u / (1 + u) are finite; a NaN stays one (minimum, not min).  With arg = log2 e f:
// 1 / (1 + u) = sigmoid(-f) and u / (1 + u) = sigmoid(f), neither a difference from one: both keep a relative error of at most
// (1.25 |f| + 8) 2^-24, most of it the rounding of the argument.
__device__ __forceinline__ float sc_odds(float arg) { return __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(arg, 126.0f)); }

// The part of a state (or of a carried gradient) that an update takes away from it, h - s h: an infinite one loses a finite
// amount and stays infinite, as in (1 - s) h; a NaN is one through the h that the update adds to.  One instruction in
// the chain of steps ([4, 8191, 512] fp16: 38.9 us with it, 38.0 without).  Computing a block again where a state turned
// NaN costs nothing otherwise, but the second form of the block rounds other channels' fp16 results differently.
__device__ __forceinline__ float sc_lose(float h) {
    constexpr float top = 3.402823466e38f;      // the largest float
    return __builtin_amdgcn_fmed3f(h, -top, top);
}

// position of a wave
struct ScanAt {
    int b, cg, ord, cc, len, lo, hi;      // ord: chunk in the order of the walk; [lo, hi) its blocks
    bool valid;
};
// `backward`: the walk visits the chunks against the scan's direction.  A workgroup holds neighbouring channel groups, or,
// where it sums, the chunks of one group.
template <bool SUMS>
__device__ __forceinline__ ScanAt scan_at(const ScanP& p, bool backward) {
    ScanAt w;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned per, r;
    if constexpr (SUMS) {
        per = (unsigned)p.ncg * p.ngroup;
        w.b = (int)(blockIdx.x / per);
        r = blockIdx.x - (unsigned)w.b * per;
        w.ord = (int)(r / (unsigned)p.ncg);
        w.cg = (int)(r - (unsigned)w.ord * p.ncg);
        w.ord = w.ord * p.group + wave;
        w.valid = w.ord < p.nchunk;
    } else {
        const unsigned id = blockIdx.x * (blockDim.x >> 6) + (unsigned)wave;
        per = (unsigned)p.ncg * p.nchunk;
        w.b = (int)(id / per);
        r = id - (unsigned)w.b * per;
        w.ord = (int)(r / (unsigned)p.ncg);
        w.cg = (int)(r - (unsigned)w.ord * p.ncg);
        w.valid = w.b < p.B;
    }
    const int chunk = (p.reverse != 0) != backward ? p.nchunk - 1 - w.ord : w.ord;
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

__device__ __forceinline__ void scan_apply(f32x2& h, f32x2 m, f32x2 v) {
#pragma unroll
    for (int e = 0; e < 2; ++e) h[e] = __builtin_fmaf(-m[e], sc_lose(h[e]), h[e]) + v[e];
}

// The state that enters a chunk: the maps of the groups in front of its group, then of its predecessors in the group.
__device__ __forceinline__ f32x2 scan_enter(const ScanP& p, const ScanAt& w, f32x2 h) {
    const long long D = p.D;
    const int g = w.ord / p.group;
    const float* q = p.sums + ((long long)p.B * p.nchunk + (long long)w.b * p.ngroup) * 2 * D + w.cc;
    const float* l = p.sums + ((long long)w.b * p.nchunk + w.ord) * 2 * D + w.cc;
    const f32x2 lm = *(const f32x2u*)l, lv = *(const f32x2u*)(l + D);
    int k = 0;
    for (; k + 8 <= g; k += 8) {
        f32x2 m[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = *(const f32x2u*)(q + (k + i) * 2 * D);
            v[i] = *(const f32x2u*)(q + (k + i) * 2 * D + D);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) scan_apply(h, m[i], v[i]);
    }
    if (k < g) {      // up to seven more; loads past the last group repeat it
        f32x2 m[7], v[7];
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            const int j = k + i < g ? k + i : g - 1;
            m[i] = *(const f32x2u*)(q + j * 2 * D);
            v[i] = *(const f32x2u*)(q + j * 2 * D + D);
        }
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (k + i < g) scan_apply(h, m[i], v[i]);               // uniform
    }
    scan_apply(h, lm, lv);
    return h;
}

// End of a summing workgroup: every wave brings the map of its chunk, and leaves that of its predecessors in the group; the
// last one leaves the whole group's.
__device__ __forceinline__ void scan_leave(const ScanP& p, const ScanAt& w, f32x2 m, f32x2 v) {
    __shared__ f32x2 maps[SC_GROUP][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    maps[wave][0][lane] = m;
    maps[wave][1][lane] = v;
    __syncthreads();
    // composition: h -> h - (m1 + m2 - m1 m2) h + (v1 - m2 v1 + v2)
    f32x2 pm{0.f, 0.f}, pv{0.f, 0.f};
    auto then = [&](f32x2 m2, f32x2 v2) {
        scan_apply(pv, m2, v2);
#pragma unroll
        for (int e = 0; e < 2; ++e) pm[e] = __builtin_fmaf(m2[e], 1.0f - pm[e], pm[e]);
    };
    for (int k = 0; k < wave; ++k) then(maps[k][0][lane], maps[k][1][lane]);
    if (w.valid) {
        float* q = p.sums + ((long long)w.b * p.nchunk + w.ord) * 2 * p.D + w.cc;
        *(f32x2u*)q = pm;
        *(f32x2u*)(q + p.D) = pv;
    }
    if (wave == p.group - 1) {
        then(m, v);
        float* q = p.sums + ((long long)p.B * p.nchunk + (long long)w.b * p.ngroup + w.ord / p.group) * 2 * p.D + w.cc;
        *(f32x2u*)q = pm;
        *(f32x2u*)(q + p.D) = pv;
    }
}

template <class F> __device__ __forceinline__ void sc_by_mode(int mode, F&& f) {
    if (mode == SC_FULL) f(std::integral_constant<int, SC_FULL>{});
    else if (mode == SC_INSIDE) f(std::integral_constant<int, SC_INSIDE>{});
    else f(std::integral_constant<int, SC_EDGE>{});
}
__device__ __forceinline__ int sc_mode(int kb, int len, int T) {
    return (kb + 1) * SC_STEPS <= len ? SC_FULL : ((kb + 1) * SC_STEPS <= T ? SC_INSIDE : SC_EDGE);
}
__device__ __forceinline__ f32x2 sc_select(bool c, f32x2 a, f32x2 b) { return f32x2{c ? a[0] : b[0], c ? a[1] : b[1]}; }

// A lane's 32-bit offset, opaque from here on: its zero extension then stays in the block of code that uses it, where
// scalar base + lane offset is one address operand; hoisted out of a loop it costs a 64-bit vector addition per access.
__device__ __forceinline__ unsigned sc_here(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Walk over the 16 rows of a block in scan order.  The row pointer is uniform (scalar registers), a lane adds its own
// 32-bit offset; rows past the end of the tensor repeat the last one.
struct RowWalk {
    const unsigned char* p;
    long long step;
    int t, dt, last;
    __device__ __forceinline__ RowWalk(const void* base, long long st, int kb, int T, int reverse) {
        t = kb * SC_STEPS + (reverse ? SC_STEPS - 1 : 0);
        dt = reverse ? -1 : 1;
        last = T - 1;
        step = reverse ? -st : st;
        p = (const unsigned char*)base + (long long)(t < T ? t : T - 1) * st;
    }
    __device__ __forceinline__ void next() {
        const bool move = dt < 0 ? t <= last : t < last;
        p += move ? step : 0;
        t += dt;
    }
};

template <int KIND, int Q0, int Q1, int PARTS>
__device__ __forceinline__ void sc_load_rows(typename Pair<KIND>::raw (&r)[PARTS][SC_STEPS], const void* base, long long st,
                                             const unsigned (&voff)[PARTS], int kb, int T, int reverse) {
    RowWalk w(base, st, kb, T, reverse);
    unsigned v[PARTS];
#pragma unroll
    for (int q = Q0; q < Q1; ++q) v[q] = sc_here(voff[q]);
#pragma unroll
    for (int i = 0; i < SC_STEPS; ++i) {
#pragma unroll
        for (int q = Q0; q < Q1; ++q) r[q][i] = Pair<KIND>::load(w.p + v[q]);
        w.next();
    }
}

// Largest of m[i] over the 16 lanes of a DPP row, for all 16 steps i at once: lane l gets the one of step l & 15.  Each
// level hands half of the steps to a partner lane and keeps the other half; the partners l^8, l^7, l^2, l^1 are the DPP
// controls row_ror:8, row_half_mirror and two quad permutations, and together reach every lane of the row.
__device__ __forceinline__ unsigned sc_row_max16(const unsigned (&m)[SC_STEPS], int lane) {
    auto meet = [](unsigned keep, unsigned send, auto ctrl) {
        const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)send, decltype(ctrl)::value, 0xf, 0xf, false);
        return keep > got ? keep : got;
    };
    unsigned a[8], b[4], c[2];
    const bool h8 = lane & 8, h4 = lane & 4, h2 = lane & 2, h1 = lane & 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = meet(h8 ? m[k + 8] : m[k], h8 ? m[k] : m[k + 8], std::integral_constant<int, 0x128>{});
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = meet(h4 ? a[k + 4] : a[k], h4 ? a[k] : a[k + 4], std::integral_constant<int, 0x141>{});
#pragma unroll
    for (int k = 0; k < 2; ++k) c[k] = meet(h2 ? b[k + 2] : b[k], h2 ? b[k] : b[k + 2], std::integral_constant<int, 0x4E>{});
    return meet(h1 ? c[1] : c[0], h1 ? c[0] : c[1], std::integral_constant<int, 0xB1>{});
}

// Codes of one part of a block: 16 steps of this lane's two channels, whose 16-lane row shares an exponent per step.
// in0 / in1: the lane's entry belongs to the 32 channels of its row.  code[e][j]: steps 4j .. 4j+3 of channel cc + e;
// `byte`: exponent of step lane & 15.  Returns whether an entry of the wave was lost.
template <int KIND>
__device__ __forceinline__ bool sc_encode(const typename Pair<KIND>::raw (&r)[SC_STEPS], bool in0, bool in1, int lane,
                                          unsigned (&code)[2][4], unsigned& byte) {
    typedef Pair<KIND> P;
    unsigned m[SC_STEPS];
#pragma unroll
    for (int i = 0; i < SC_STEPS; ++i) {
        const unsigned m0 = in0 ? P::mag(r[i], 0) : 0u, m1 = in1 ? P::mag(r[i], 1) : 0u;
        m[i] = m0 > m1 ? m0 : m1;
    }
    unsigned top = sc_row_max16(m, lane);
    const bool lost = __any(top >= P::nonfinite);
    if (lost) {
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) {
            const unsigned m0 = in0 && P::mag(r[i], 0) < P::nonfinite ? P::mag(r[i], 0) : 0u;
            const unsigned m1 = in1 && P::mag(r[i], 1) < P::nonfinite ? P::mag(r[i], 1) : 0u;
            m[i] = m0 > m1 ? m0 : m1;
        }
        top = sc_row_max16(m, lane);
    }
    const int ex = c8_exponent<KIND>(__builtin_bit_cast(unsigned, P::mag_value(top)));
    byte = (unsigned)ex;
    const float inv = c8_inv_scale(ex);
    const bool rare = lost || __any(ex == C8Range<KIND>::hi + 127);
    unsigned u[2][SC_STEPS];
    static_for<SC_STEPS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        // the exponent's reciprocal of step i from lane i of the row (row_newbcast)
        const float q = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, inv), 0x150 + i, 0xf, 0xf, false));
        const f32x2 v = P::get(r[i]);
        // x * 2^-e + 1.5 * 2^23: the sum's step is 1, so the one rounding is the code's (ties to even), and the low byte
        // of its bits is the code
#pragma unroll
        for (int e = 0; e < 2; ++e) u[e][i] = __builtin_bit_cast(unsigned, __builtin_fmaf(v[e], q, 12582912.0f));
        if (rare) {
            const float cap = q == c8_inv_scale(C8Range<KIND>::hi + 127) ? 63.f : 127.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) u[e][i] = P::mag(r[i], e) >= P::nonfinite ? C8_LOST : c8_code(v[e], q, cap);
        }
    });
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // v_perm_b32: selectors 0-3 take the second operand's bytes, 4-7 the first one's
            const unsigned lo = __builtin_amdgcn_perm(u[e][4 * j + 1], u[e][4 * j], 0x0c0c0400u);
            const unsigned hi = __builtin_amdgcn_perm(u[e][4 * j + 3], u[e][4 * j + 2], 0x04000c0cu);
            code[e][j] = lo | hi;
        }
    return lost;
}

// Forward.  SAVE: 0 nothing, 1 the state entering each block, 2 that and the 8-bit codes of z.
template <int KIND, bool GATED, int SAVE>
__global__ __launch_bounds__(256) void k_scan_fwd(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at<false>(p, false);
    if (!w.valid) return;
    const int lane = threadIdx.x & 63;
    const long long zst = p.z_st * EB, yst = p.y_st * EB;
    const unsigned char* zb = (const unsigned char*)p.z + w.b * p.z_sb * EB;
    unsigned char* yb = (unsigned char*)p.y + w.b * p.y_sb * EB;
    unsigned voff[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) voff[q] = (unsigned)(q * p.D + w.cc) * EB;
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi;     // blocks that hold a valid step
    for (int kb = hi > w.lo ? hi : w.lo; kb < w.hi; ++kb)                                 // blocks behind the sentence
        for (int i = 0; i < SC_STEPS; ++i)
            if (kb * SC_STEPS + i < p.T) Pair<KIND>::store(yb + (long long)(kb * SC_STEPS + i) * yst + voff[0], f32x2{0.f, 0.f});
    f32x2 h = p.h0 != nullptr ? (f32x2)*(const f32x2u*)(p.h0 + (long long)w.b * p.D + w.cc) : f32x2{0.f, 0.f};
    const int c0 = w.cg * SC_CH + 2 * lane;
    const bool own0 = c0 < p.D && w.cc == c0, own1 = c0 < p.D;      // the lane's own channels among (cc, cc + 1)
    raw nz[PARTS][SC_STEPS];
    const int n = hi - w.lo;
    if (n > 0) sc_load_rows<KIND, 0, PARTS>(nz, zb, zst, voff, p.reverse ? hi - 1 : w.lo, p.T, p.reverse);
    if (p.nchunk > 1) h = scan_enter(p, w, h);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? hi - 1 - it : w.lo + it;
        raw z[PARTS][SC_STEPS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) z[q][i] = nz[q][i];
        if (it + 1 < n) sc_load_rows<KIND, 0, PARTS>(nz, zb, zst, voff, p.reverse ? kb - 1 : kb + 1, p.T, p.reverse);
        if constexpr (SAVE > 0) *(f32x2u*)(p.kept + ((long long)w.b * p.nblk + kb) * p.D + w.cc) = h;
        if constexpr (SAVE == 2) {
            const int nb = (p.D + C8_BLOCK - 1) / C8_BLOCK;
            const long long tile = ((long long)w.b * p.nblk + kb) * PARTS;
            bool lost = false;
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                unsigned code[2][4], byte;
                lost |= sc_encode<KIND>(z[q], own0, own1, lane, code, byte);
                unsigned char* cp = p.codes + ((tile + q) * p.D + w.cc) * SC_STEPS;
                if (own0) *(u32x4*)cp = u32x4{code[0][0], code[0][1], code[0][2], code[0][3]};
                if (own1) *(u32x4*)(cp + SC_STEPS) = u32x4{code[1][0], code[1][1], code[1][2], code[1][3]};
                const int blk = (w.cg * SC_CH + (lane & 48) * 2) / C8_BLOCK;
                if (blk < nb) p.exps[((tile + q) * nb + blk) * SC_STEPS + (lane & 15)] = (unsigned char)byte;
            }
            if (lane == 0) p.lost[((long long)w.b * p.nblk + kb) * p.ncg + w.cg] = lost ? 1u : 0u;
        }
        sc_by_mode(sc_mode(kb, w.len, p.T), [&](auto mode) {
            constexpr int MODE = decltype(mode)::value;
            unsigned char* yr = yb + (long long)(kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 : 0)) * yst;
            const unsigned vy = sc_here(voff[0]);
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) {
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const bool ok = MODE == SC_FULL || t < w.len;
                const f32x2 xv = Pair<KIND>::get(z[0][i]), fv = Pair<KIND>::get(z[1][i]);
                f32x2 hn;
#pragma unroll
                for (int e = 0; e < 2; ++e) hn[e] = __builtin_fmaf(sc_share(fv[e]), xv[e] - sc_lose(h[e]), h[e]);
                h = sc_select(ok, hn, h);
                f32x2 yv = h;
                if constexpr (GATED) {
                    const f32x2 ov = Pair<KIND>::get(z[PARTS - 1][i]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) yv[e] = h[e] * sigmoidf_(ov[e]);
                }
                yv = sc_select(ok, yv, f32x2{0.f, 0.f});
                if (MODE != SC_EDGE || t < p.T) Pair<KIND>::store(yr + vy, yv);
                yr += p.reverse ? -yst : yst;
            }
        });
    }
    if (w.ord == p.nchunk - 1) *(f32x2u*)(p.h_last + (long long)w.b * p.D + w.cc) = h;
}

// (M, v) of one chunk, forward: the chunk's steps from the zero state.
template <int KIND>
__global__ __launch_bounds__(64 * SC_GROUP) void k_scan_sum(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at<true>(p, false);
    const long long zst = p.z_st * EB;
    const unsigned char* zb = (const unsigned char*)p.z + w.b * p.z_sb * EB;
    const unsigned voff[2] = {(unsigned)w.cc * EB, (unsigned)(p.D + w.cc) * EB};
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi;
    const int n = w.ord < p.nchunk - 1 ? hi - w.lo : 0;             // nothing follows the last chunk's map
    f32x2 h{0.f, 0.f}, m{0.f, 0.f};
    raw nz[2][SC_STEPS];
    if (n > 0) sc_load_rows<KIND, 0, 2>(nz, zb, zst, voff, p.reverse ? hi - 1 : w.lo, p.T, p.reverse);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? hi - 1 - it : w.lo + it;
        raw z[2][SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) { z[0][i] = nz[0][i]; z[1][i] = nz[1][i]; }
        if (it + 1 < n) sc_load_rows<KIND, 0, 2>(nz, zb, zst, voff, p.reverse ? kb - 1 : kb + 1, p.T, p.reverse);
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) {
            const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
            const f32x2 xv = Pair<KIND>::get(z[0][i]), fv = Pair<KIND>::get(z[1][i]);
            const bool ok = t < w.len;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float s = sc_share(fv[e]);
                h[e] = ok ? __builtin_fmaf(s, xv[e] - sc_lose(h[e]), h[e]) : h[e];
                m[e] = ok ? __builtin_fmaf(s, 1.0f - m[e], m[e]) : m[e];
            }
        }
    }
    scan_leave(p, w, m, h);
}

// What a block of the backward pass reads of z (parts Q0 ..): the rows themselves, or codes and exponents.
template <int KIND, int PARTS, bool CODES> struct ScanIn;
template <int KIND, int PARTS> struct ScanIn<KIND, PARTS, false> {
    typename Pair<KIND>::raw r[PARTS][SC_STEPS];
    template <int Q0, int Q1> __device__ __forceinline__ void load(const ScanP& p, const ScanAt& w, int kb) {
        constexpr int EB = Elem<KIND>::bytes;
        unsigned voff[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) voff[q] = (unsigned)(q * p.D + w.cc) * EB;
        sc_load_rows<KIND, Q0, Q1>(r, (const unsigned char*)p.z + w.b * p.z_sb * EB, p.z_st * EB, voff, kb, p.T, p.reverse);
    }
    __device__ __forceinline__ bool lost() const { return false; }
    // makes the compiler decode x and f again instead of keeping 64 decoded registers alive between two uses
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) asm volatile("" : "+v"(r[q][i]));
    }
    // c times part Q of step I, and x of step I less h
    template <int Q, int I, bool CHECKED> __device__ __forceinline__ f32x2 times(float c) const {
        const f32x2 v = Pair<KIND>::get(r[Q][I]);
        return f32x2{c * v[0], c * v[1]};
    }
    template <int I, bool CHECKED> __device__ __forceinline__ f32x2 x_less(f32x2 h) const {
        const f32x2 v = Pair<KIND>::get(r[0][I]);
        return f32x2{v[0] - h[0], v[1] - h[1]};
    }
};
template <int KIND, int PARTS> struct ScanIn<KIND, PARTS, true> {
    u32x4 c[PARTS][2], e[PARTS][2];
    unsigned flag;
    template <int Q0, int Q1> __device__ __forceinline__ void load(const ScanP& p, const ScanAt& w, int kb) {
        const int nb = (p.D + C8_BLOCK - 1) / C8_BLOCK;
        const long long blk = (long long)w.b * p.nblk + kb;
        if (Q0 < 2) flag = p.lost[blk * p.ncg + w.cg];
#pragma unroll
        for (int q = Q0; q < Q1; ++q) {
            const long long tile = blk * PARTS + q;
            const unsigned char* cp = p.codes + tile * p.D * SC_STEPS;
            c[q][0] = *(const u32x4*)(cp + (unsigned)w.cc * SC_STEPS);
            c[q][1] = *(const u32x4*)(cp + (unsigned)(w.cc + 1) * SC_STEPS);
            const unsigned char* ep = p.exps + tile * nb * SC_STEPS;
            e[q][1] = *(const u32x4*)(ep + (unsigned)((w.cc + 1) / C8_BLOCK) * SC_STEPS);
            e[q][0] = e[q][1];
            // channels D-2 and D-1 of the last lanes lie in different blocks of 32
            if (p.D % C8_BLOCK == 1) e[q][0] = *(const u32x4*)(ep + (unsigned)(w.cc / C8_BLOCK) * SC_STEPS);
        }
    }
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < 2; ++k) asm volatile("" : "+v"(c[q][k]), "+v"(e[q][k]));
    }
    __device__ __forceinline__ bool lost() const { return __builtin_amdgcn_readfirstlane(flag) != 0; }
    template <int Q, int I> __device__ __forceinline__ float scale(int k) const {
        return c8_scale((e[Q][k][I >> 2] >> (8 * (I & 3))) & 0xffu);
    }
    template <int Q, int I, bool CHECKED> __device__ __forceinline__ f32x2 times(float f) const {
        f32x2 v;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            v[k] = c8_int<I & 3>(c[Q][k][I >> 2]) * (scale<Q, I>(k) * f);       // the power of two moves freely: one rounding
            if (CHECKED && c8_is_lost<I & 3>(c[Q][k][I >> 2])) v[k] = __builtin_nanf("");
        }
        return v;
    }
    template <int I, bool CHECKED> __device__ __forceinline__ f32x2 x_less(f32x2 h) const {
        f32x2 v;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            v[k] = __builtin_fmaf(c8_int<I & 3>(c[0][k][I >> 2]), scale<0, I>(k), -h[k]);
            if (CHECKED && c8_is_lost<I & 3>(c[0][k][I >> 2])) v[k] = __builtin_nanf("");
        }
        return v;
    }
};

// Backward.
template <int KIND, bool GATED, bool CODES>
__global__ __launch_bounds__(256, 2) void k_scan_bwd(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at<false>(p, true);
    if (!w.valid) return;
    const long long dyst = p.dy_st * EB, dzst = p.dz_st * EB;
    const unsigned char* dyb = (const unsigned char*)p.dy + w.b * p.dy_sb * EB;
    unsigned char* gb = (unsigned char*)p.dz + w.b * p.dz_sb * EB;
    unsigned voff[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) voff[q] = (unsigned)(q * p.D + w.cc) * EB;
    const unsigned dyoff[1] = {voff[0]};
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi, n = hi - w.lo;
    for (int kb = hi > w.lo ? hi : w.lo; kb < w.hi; ++kb)
        for (int i = 0; i < SC_STEPS; ++i)
            if (kb * SC_STEPS + i < p.T) {
#pragma unroll
                for (int q = 0; q < PARTS; ++q) Pair<KIND>::store(gb + (long long)(kb * SC_STEPS + i) * dzst + voff[q], f32x2{0.f, 0.f});
            }
    f32x2 carry = p.dh_last != nullptr ? (f32x2)*(const f32x2u*)(p.dh_last + (long long)w.b * p.D + w.cc) : f32x2{0.f, 0.f};

    // x, f and the kept state of the next block are loaded behind the states of this one, o and dy of this block in front of
    // them: each load has one of the two passes over the block to arrive in, and at most 96 registers hold rows.
    ScanIn<KIND, PARTS, CODES> in, nin;
    f32x2 enter, nh;
    auto issue = [&](int kb) {
        nh = *(const f32x2u*)(p.kept + ((long long)w.b * p.nblk + kb) * p.D + w.cc);
        nin.template load<0, 2>(p, w, kb);
    };
    if (n > 0) issue(p.reverse ? w.lo : hi - 1);
    if (p.nchunk > 1) carry = scan_enter(p, w, carry);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? w.lo + it : hi - 1 - it;
        raw dy[1][SC_STEPS];
        in = nin;
        enter = nh;
        if constexpr (GATED) in.template load<2, PARTS>(p, w, kb);
        if (p.dy != nullptr) sc_load_rows<KIND, 0, 1>(dy, dyb, dyst, dyoff, kb, p.T, p.reverse);
        else {
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) dy[0][i] = Pair<KIND>::zero();
        }
        __builtin_amdgcn_sched_barrier(0);
        // lost entries are looked for in the slowest form only
        const int mode = in.lost() ? SC_EDGE : sc_mode(kb, w.len, p.T);
        f32x2 h[SC_STEPS], odds[SC_STEPS];                          // states; e^f
        auto states = [&](auto m) {
            constexpr int MODE = decltype(m)::value;
            f32x2 hc = enter;
            static_for<SC_STEPS>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const f32x2 fa = in.template times<1, i, MODE == SC_EDGE>(SC_LOG2E), xd = in.template x_less<i, MODE == SC_EDGE>(f32x2{sc_lose(hc[0]), sc_lose(hc[1])});
                f32x2 hn;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    odds[i][e] = sc_odds(fa[e]);
                    hn[e] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + odds[i][e]), xd[e], hc[e]);
                }
                hc = sc_select(MODE == SC_FULL || t < w.len, hn, hc);
                h[i] = hc;
            });
        };
        auto grads = [&](auto m) {
            constexpr int MODE = decltype(m)::value;
            unsigned char* gr = gb + (long long)(kb * SC_STEPS + (p.reverse ? 0 : SC_STEPS - 1)) * dzst;
            unsigned vg[PARTS];
#pragma unroll
            for (int q = 0; q < PARTS; ++q) vg[q] = sc_here(voff[q]);
            static_for<SC_STEPS>([&](auto jc) {
                constexpr int i = SC_STEPS - 1 - decltype(jc)::value;
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const bool ok = MODE == SC_FULL || t < w.len;
                const f32x2 hp = i == 0 ? enter : h[i == 0 ? 0 : i - 1], dyv = Pair<KIND>::get(dy[0][i]);
                const f32x2 xd = in.template x_less<i, MODE == SC_EDGE>(hp);
                f32x2 oa, dx, df, dov, cn;
                if constexpr (GATED) oa = in.template times<PARTS - 1, i, MODE == SC_EDGE>(-SC_LOG2E);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float dh = dyv[e];
                    if constexpr (GATED) {
                        const float u = sc_odds(oa[e]), so = __builtin_amdgcn_rcpf(1.0f + u);
                        dh *= so;
                        dov[e] = dh * h[i][e] * (u * so);
                    }
                    const float g = dh + carry[e], sv = __builtin_amdgcn_rcpf(1.0f + odds[i][e]);
                    dx[e] = sv * g;
                    df[e] = -(odds[i][e] * sv * dx[e]) * xd[e];
                    cn[e] = __builtin_fmaf(-sv, sc_lose(g), g);
                }
                const f32x2 none{0.f, 0.f};
                carry = sc_select(ok, cn, carry);
                dx = sc_select(ok, dx, none);
                df = sc_select(ok, df, none);
                if constexpr (GATED) dov = sc_select(ok, dov, none);
                if (MODE != SC_EDGE || t < p.T) {
                    Pair<KIND>::store(gr + vg[0], dx);
                    Pair<KIND>::store(gr + vg[1], df);
                    if constexpr (GATED) Pair<KIND>::store(gr + vg[PARTS - 1], dov);
                }
                gr += p.reverse ? dzst : -dzst;
            });
        };
        sc_by_mode(mode, states);
        __builtin_amdgcn_sched_barrier(0);
        in.forget();
        if (it + 1 < n) issue(p.reverse ? kb + 1 : kb - 1);
        sc_by_mode(mode, grads);
    }
    if (p.dh0 != nullptr && w.ord == p.nchunk - 1) *(f32x2u*)(p.dh0 + (long long)w.b * p.D + w.cc) = carry;
}

// (M, v) of one chunk, backward: carry -> carry - M carry + v.
template <int KIND, bool GATED, bool CODES>
__global__ __launch_bounds__(64 * SC_GROUP) void k_scan_bsum(ScanP p) {
    typedef typename Pair<KIND>::raw raw;
    constexpr int PARTS = GATED ? 3 : 2, EB = Elem<KIND>::bytes;
    const ScanAt w = scan_at<true>(p, true);
    const long long dyst = p.dy_st * EB;
    const unsigned char* dyb = (const unsigned char*)p.dy + w.b * p.dy_sb * EB;
    const unsigned dyoff[1] = {(unsigned)w.cc * EB};
    const int vhi = (w.len + SC_STEPS - 1) / SC_STEPS, hi = w.hi < vhi ? w.hi : vhi;
    const int n = w.ord < p.nchunk - 1 ? hi - w.lo : 0;
    f32x2 v{0.f, 0.f}, m{0.f, 0.f};
    ScanIn<KIND, PARTS, CODES> nin;
    raw ndy[1][SC_STEPS];
    auto issue = [&](int kb) {
        nin.template load<1, PARTS>(p, w, kb);
        if (p.dy != nullptr) sc_load_rows<KIND, 0, 1>(ndy, dyb, dyst, dyoff, kb, p.T, p.reverse);
        else {
#pragma unroll
            for (int i = 0; i < SC_STEPS; ++i) ndy[0][i] = Pair<KIND>::zero();
        }
    };
    if (n > 0) issue(p.reverse ? w.lo : hi - 1);
    for (int it = 0; it < n; ++it) {
        const int kb = p.reverse ? w.lo + it : hi - 1 - it;
        const ScanIn<KIND, PARTS, CODES> in = nin;
        raw dy[SC_STEPS];
#pragma unroll
        for (int i = 0; i < SC_STEPS; ++i) dy[i] = ndy[0][i];
        const bool checked = in.lost();
        if (it + 1 < n) issue(p.reverse ? kb + 1 : kb - 1);
        auto block = [&](auto chk) {
            constexpr bool CHECKED = decltype(chk)::value;
            static_for<SC_STEPS>([&](auto jc) {
                constexpr int i = SC_STEPS - 1 - decltype(jc)::value;
                const int t = kb * SC_STEPS + (p.reverse ? SC_STEPS - 1 - i : i);
                const bool ok = t < w.len;
                const f32x2 fa = in.template times<1, i, CHECKED>(SC_LOG2E), dyv = Pair<KIND>::get(dy[i]);
                f32x2 oa;
                if constexpr (GATED) oa = in.template times<PARTS - 1, i, CHECKED>(-SC_LOG2E);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float dh = dyv[e];
                    if constexpr (GATED) dh *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(oa[e]));
                    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(fa[e])), g = dh + v[e];
                    v[e] = ok ? __builtin_fmaf(-s, sc_lose(g), g) : v[e];
                    m[e] = ok ? __builtin_fmaf(s, 1.0f - m[e], m[e]) : m[e];
                }
            });
        };
        if constexpr (CODES) {
            if (checked) block(std::integral_constant<bool, true>{});
            else block(std::integral_constant<bool, false>{});
        } else block(std::integral_constant<bool, false>{});
    }
    scan_leave(p, w, m, v);
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
    float hn = __builtin_fmaf(sc_share(f), x - sc_lose(hp), hp), yv = hn;
    if constexpr (GATED) yv *= sigmoidf_(Elem<KIND>::load(z, zo + 2ll * D));
    const bool live = alive == nullptr || alive[b] != 0;
    Elem<KIND>::store(y, (long long)b * y_sb + c, live ? yv : 0.f);
    h_out[(long long)b * ho_sb + c] = live ? hn : hp;
}

}  // namespace sad
