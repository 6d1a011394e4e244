// Weight gradient of a linear layer from an 8-bit checkpoint of its input:
//
//   dW[n][k] = sum_m dY[m][n] X^[m][k] ,   db[n] = sum_m dY[m][n]           (m: token rows, the reduced index)
//
// X^ is decoded on its way into LDS; its values are exact in bf16 and fp16 (ckpt8.hpp), so the products are those of dY
// with the checkpoint and nothing is rounded but the fp32 sums.  dY in float32 is cut into three bf16 parts
// (8 + 8 + 8 significant bits, exact; infinities and the largest floats stay what they are), one matrix instruction each.  The workgroups of the first k
// tile also add up the columns of dY that pass through their registers: db.
//
// Both operands are stored with the reduced index slow, so fragments are read from LDS with the transposing read
// (tr_frag).  Token rows are split over workgroups where the output has few tiles; the partial tiles go to a slab and a
// second launch adds them in fixed order (no atomics: the result does not depend on scheduling).
//
// Pipeline: two LDS buffers, one barrier per stage of 64 rows.  While a stage is multiplied, the next one moves from
// registers (decoded) into the other buffer and the loads of the one after are issued, all in one instruction stream: a
// stage is cut into slices of one fragment of dY against all fragments of X^, and every slice carries its share of the
// fragment reads for the slices behind it, of the decoding and of the loads.  The compiler may not move instructions from
// slice to slice (sched_barrier): left alone it reads all fragments first and decodes last.
//
// Measured, bf16: [16384 rows, 6144, 2048] 460-510 us (412 GFLOP: 810-900 TFLOP/s; a large library product reaches 1337, the
// library's own dY^T X of this shape 943), matrix units busy 42 % of the cycles at a clock of 1.85-2.0 GHz under this load,
// LDS 30 %, vector instructions 36 %, no bank conflicts; four waves of 96 x 128 outputs instead of eight of 96 x 64 read less
// LDS but the compiler copies accumulators between register files (650 us).  [32768, 1536, 300]: 53 us and 8 us to
// join 21 splits (the library: 188 us).  Rows of dY that no single stride reaches (a time-major dY under a batch-major
// checkpoint) are read chunk by chunk behind the matrix loop: [64 x 500, 1536, 300] 61 us instead of 57.
#pragma once
#include "ckpt8.hpp"
#include "gemm_core.hpp"

namespace sad {

// Workgroup tile BN x BK outputs, W1 x W2 waves.
template <int KIND_, int BN_, int BK_, int W1_, int W2_> struct W8 {
    static constexpr int KIND = KIND_, BN = BN_, BK = BK_, W1 = W1_, W2 = W2_;
    static constexpr int BM = 64;                              // token rows per stage
    static constexpr int NT = 64 * W1 * W2;
    static constexpr int T1 = BN / W1 / 16, T2 = BK / W2 / 16; // 16x16 tiles of a wave
    static constexpr int PLANES = KIND == SAD_SRC_F32 ? 3 : 1; // bf16 / fp16 images of dY
    static constexpr int PA = BN * 2 + 32, PB = BK * 2 + 32;   // LDS row pitch in bytes: odd multiples of 32 (tr_frag)
    static constexpr int ABYTES = BM * PA, BUF = PLANES * ABYTES + BM * PB;
    static constexpr int LDS = 2 * BUF;
    // Chunks (8 entries of dY, 8 codes) of a thread: column blocks of 64, 8 threads to a row.  A thread's chunks then differ
    // by constants in LDS and by uniform steps in memory.
    static constexpr int AB = BN / 64, BB = BK / 64, R = NT / 8, NA = AB * BM / R, NB = BB * BM / R;
    static constexpr int SL = 2 * PLANES * T1;                 // slices of a stage
    static constexpr int UNITS = NA + NB;                      // pieces of staging work, spread over the slices
    static_assert(BN % 64 == 0 && BK % 64 == 0 && BM % R == 0, "staging must divide evenly");
    static_assert((BN / 16) % 2 == 0 && (BK / 16) % 2 == 0, "tile");
};

struct Wgrad8P {
    int M, N, K, Kp;              // Kp: K rounded up to 32 (pitch of the codes)
    const void* dy; Rows2 yr; int y_flat;      // y_flat: row m starts at m * yr.s1
    int fast_rows;                // rows in front of this one may be read in whole chunks of 8 columns
    const unsigned char* codes; const unsigned char* exps; const unsigned char* marked;
    float* out;                   // dW, or the slab of the splits: [splits][N * K + N], dW in front of db
    float* out_b;                 // db in it; NULL: no bias
    long long slab;               // floats of a split
    int tn, tk, splits, rows;     // tiles, row splits, rows per split (multiple of 64)
    int per_xcd;                  // workgroups per XCD
};

// 8 entries of dY as loaded
template <int KIND> struct DyChunk { u32x4 v; };
template <> struct DyChunk<SAD_SRC_F32> { f32x4 a, b; };

__device__ __forceinline__ unsigned c8_pack16(float a, float b, bool half) {
    if (half) return (unsigned)__builtin_bit_cast(unsigned short, (_Float16)a) | ((unsigned)__builtin_bit_cast(unsigned short, (_Float16)b) << 16);
    // the upper halves (bf16 values are exact in them)
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}

// Position and staging state of a workgroup; BIAS: it also sums the columns of dY.
template <class W, bool BIAS> struct Wgrad8 {
    static constexpr int KIND = W::KIND, EB = Elem<KIND>::bytes;
    const Wgrad8P& p;
    unsigned char* lds;
    int n0, k0, m_begin, m_end, split, lane, w1, w2;
    int aoff, boff;                              // LDS offsets of this thread's first chunks
    unsigned ag[W::AB], bg[W::BB], eg[W::BB];    // their offsets from the stage's first row in memory, per column block
    DyChunk<KIND> ra[W::NA];
    u32x2 rb[W::NB];
    unsigned re[W::NB];
    f32x4 acc[W::T1][W::T2];
    float sum[BIAS ? W::AB : 1][8];              // column sums of this thread's chunks
    int fa_off, fb_off;

    __device__ __forceinline__ Wgrad8(const Wgrad8P& p_, unsigned char* lds_) : p(p_), lds(lds_) {}
    // chunk i: column block i % AB (BB), row row() + i / AB * R
    __device__ __forceinline__ int row() const { return (int)threadIdx.x >> 3; }
    __device__ __forceinline__ int col() const { return ((int)threadIdx.x & 7) * 8; }
    static constexpr int a_lds(int i) { return (i % W::AB) * 128 + (i / W::AB) * W::R * W::PA; }
    static constexpr int b_lds(int i) { return (i % W::BB) * 128 + (i / W::BB) * W::R * W::PB; }

    __device__ __forceinline__ void init() {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        lane = threadIdx.x & 63; w1 = wave / W::W2; w2 = wave % W::W2;
        aoff = row() * W::PA + col() * 2;
        boff = W::PLANES * W::ABYTES + row() * W::PB + col() * 2;
        // chunks that lie past the last column read the first one (their products are not stored)
#pragma unroll
        for (int j = 0; j < W::AB; ++j) {
            const int c = n0 + 64 * j + col();
            ag[j] = (unsigned)(row() * (long long)p.yr.s1 + (c < p.N ? c : 0)) * EB;
        }
#pragma unroll
        for (int j = 0; j < W::BB; ++j) {
            const int c = k0 + 64 * j + col() < p.Kp ? k0 + 64 * j + col() : 0;
            bg[j] = (unsigned)(row() * p.Kp + c);
            eg[j] = (unsigned)(row() * (p.Kp / C8_BLOCK) + c / C8_BLOCK);
        }
        const int rowsel = 4 * (lane >> 4) + ((lane >> 2) & 3), p4 = (lane & 3) * 4;
        fa_off = rowsel * W::PA + (w1 * (W::BN / W::W1) + p4) * 2;
        fb_off = W::PLANES * W::ABYTES + rowsel * W::PB + (w2 * (W::BK / W::W2) + p4) * 2;
#pragma unroll
        for (int a = 0; a < W::T1; ++a)
#pragma unroll
            for (int b = 0; b < W::T2; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (BIAS) {
#pragma unroll
            for (int j = 0; j < W::AB; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) sum[j][k] = 0.f;
        }
    }
    // a stage all of whose chunks may be read whole
    __device__ __forceinline__ bool fast(int s) const {
        const int e = m_begin + (s + 1) * W::BM;
        return e <= p.fast_rows && e <= m_end;
    }
    __device__ __forceinline__ const unsigned char* a_base(int s) const { return (const unsigned char*)p.dy + (long long)(m_begin + s * W::BM) * p.yr.s1 * EB; }
    __device__ __forceinline__ const unsigned char* b_base(int s) const { return p.codes + (long long)(m_begin + s * W::BM) * p.Kp; }
    __device__ __forceinline__ const unsigned char* e_base(int s) const { return p.exps + (long long)(m_begin + s * W::BM) * (p.Kp / C8_BLOCK); }
    __device__ __forceinline__ static unsigned here(unsigned v) {      // keeps the zero extension beside the load (one address operand)
        asm volatile("" : "+v"(v));
        return v;
    }
    template <int I> __device__ __forceinline__ void load_a(const unsigned char* base) {
        const unsigned char* q = base + (long long)(I / W::AB) * W::R * p.yr.s1 * EB + here(ag[I % W::AB]);
        if constexpr (KIND == SAD_SRC_F32) {
            ra[I].a = *(const f32x4u*)q;
            ra[I].b = *(const f32x4u*)(q + 16);
        } else ra[I].v = *(const u32x4h*)q;
    }
    template <int I> __device__ __forceinline__ void load_b(const unsigned char* base, const unsigned char* ebase) {
        rb[I] = *(const u32x2*)(base + (long long)(I / W::BB) * W::R * p.Kp + here(bg[I % W::BB]));
        re[I] = *(ebase + (long long)(I / W::BB) * W::R * (p.Kp / C8_BLOCK) + here(eg[I % W::BB]));
    }
    __device__ __forceinline__ void load_fast(int s) {
        const unsigned char *a = a_base(s), *b = b_base(s), *e = e_base(s);
        // codes first, as in a stage: the wait for them in front of the next stage then leaves dY in flight
        static_for<W::NB>([&](auto i) { load_b<decltype(i)::value>(b, e); });
        __builtin_amdgcn_sched_barrier(0);
        static_for<W::NA>([&](auto i) { load_a<decltype(i)::value>(a); });
    }
    __device__ __forceinline__ void load_guarded(int s) {
        const int m0 = m_begin + s * W::BM;
#pragma unroll
        for (int i = 0; i < W::NA; ++i) {
            if constexpr (KIND == SAD_SRC_F32) ra[i].a = ra[i].b = f32x4{0.f, 0.f, 0.f, 0.f};
            else ra[i].v = u32x4{0u, 0u, 0u, 0u};
            const int m = m0 + row() + (i / W::AB) * W::R, c = n0 + col() + (i % W::AB) * 64;
            if (m < m_end) {
                const long long off = (p.y_flat ? (long long)m * p.yr.s1 : p.yr.at((unsigned)m)) + c;
                if constexpr (KIND == SAD_SRC_F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (c + j < p.N) ra[i].a[j] = ((const float*)p.dy)[off + j];
                        if (c + 4 + j < p.N) ra[i].b[j] = ((const float*)p.dy)[off + 4 + j];
                    }
                } else if (c + 8 <= p.N) ra[i].v = *(const u32x4h*)((const unsigned short*)p.dy + off);
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (c + j < p.N) ra[i].v[j >> 1] |= (unsigned)((const unsigned short*)p.dy)[off + j] << (16 * (j & 1));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < W::NB; ++i) {
            rb[i] = u32x2{0u, 0u};
            re[i] = 1u;
            if (m0 + row() + (i / W::BB) * W::R < m_end) {
                rb[i] = *(const u32x2*)(b_base(s) + (long long)(i / W::BB) * W::R * p.Kp + bg[i % W::BB]);
                re[i] = *(e_base(s) + (long long)(i / W::BB) * W::R * (p.Kp / C8_BLOCK) + eg[i % W::BB]);
            }
        }
    }
    __device__ __forceinline__ void load(int s) {
        if (fast(s)) load_fast(s);
        else load_guarded(s);
    }
    template <int I> __device__ __forceinline__ void put_a(unsigned char* buf) {
        unsigned char* at = buf + aoff + a_lds(I);
        if constexpr (KIND == SAD_SRC_F32) {
            float rest[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = j < 4 ? ra[I].a[j] : ra[I].b[j - 4];
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                u32x4 v;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // cut, not rounded: the largest floats round to infinity in bf16
                    v[j] = c8_pack16(rest[2 * j], rest[2 * j + 1], false);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float r = rest[2 * j + h], part = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, r) & 0xffff0000u);
                        // nothing is left of an infinity; a NaN, whose upper half may read as one, leaves a NaN
                        rest[2 * j + h] = q == 0 && __builtin_fabsf(r) == __builtin_inff() ? 0.f : r - part;
                    }
                }
                *(u32x4*)(at + q * W::ABYTES) = v;
            }
        } else *(u32x4*)at = ra[I].v;
        if constexpr (BIAS) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float v;
                if constexpr (KIND == SAD_SRC_F32) v = k < 4 ? ra[I].a[k] : ra[I].b[k - 4];
                else {
                    const unsigned short h = (unsigned short)(ra[I].v[k >> 1] >> (16 * (k & 1)));
                    v = KIND == SAD_SRC_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
                }
                sum[I % W::AB][k] += v;
            }
        }
    }
    template <int I> __device__ __forceinline__ void put_b(unsigned char* buf) {
        const float scale = c8_scale((int)re[I]);
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const unsigned w = rb[I][j];
            v[2 * j] = c8_pack16(c8_value<0>(w, scale), c8_value<1>(w, scale), KIND == SAD_SRC_F16);
            v[2 * j + 1] = c8_pack16(c8_value<2>(w, scale), c8_value<3>(w, scale), KIND == SAD_SRC_F16);
        }
        *(u32x4*)(buf + boff + b_lds(I)) = v;
    }
    __device__ __forceinline__ void put(unsigned char* buf) {
        static_for<W::NA>([&](auto i) { put_a<decltype(i)::value>(buf); });
        static_for<W::NB>([&](auto i) { put_b<decltype(i)::value>(buf); });
    }
    // does the stage in the registers hold a marked block (uniform)
    __device__ __forceinline__ bool marks() const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < W::NB; ++i) any |= re[i] == C8_MARK;
        return __any(any);
    }
    // Rare: the marked chunks of stage s, written again from memory with their own exponents and NaN for lost entries (by the
    // thread that wrote them before, so in order).
    __device__ __forceinline__ void repair(int s, unsigned char* buf) {
#pragma unroll
        for (int i = 0; i < W::NB; ++i) {
            const long long eat = (long long)(i / W::BB) * W::R * (p.Kp / C8_BLOCK) + eg[i % W::BB];
            if (m_begin + s * W::BM + row() + (i / W::BB) * W::R < m_end && *(e_base(s) + eat) == C8_MARK) {
                const u32x2 c = *(const u32x2*)(b_base(s) + (long long)(i / W::BB) * W::R * p.Kp + bg[i % W::BB]);
                const float scale = c8_scale((int)*(p.marked + (e_base(s) - p.exps) + eat));
                u32x4 v;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    v[2 * j] = c8_pack16(c8_value_checked<0>(c[j], scale), c8_value_checked<1>(c[j], scale), KIND == SAD_SRC_F16);
                    v[2 * j + 1] = c8_pack16(c8_value_checked<2>(c[j], scale), c8_value_checked<3>(c[j], scale), KIND == SAD_SRC_F16);
                }
                *(u32x4*)(buf + boff + b_lds(i)) = v;
            }
        }
    }
    __device__ __forceinline__ static f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
        if constexpr (KIND == SAD_SRC_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // slice = (ks * PLANES + plane) * T1 + a
    template <int S> __device__ __forceinline__ bf16x8 frag_a(const unsigned char* buf) const {
        constexpr int ks = S / (W::PLANES * W::T1), q = S / W::T1 % W::PLANES, a = S % W::T1;
        return tr_frag(buf + fa_off + q * W::ABYTES + ks * 32 * W::PA + a * 32, W::PA);
    }
    template <int KS, int B> __device__ __forceinline__ bf16x8 frag_b(const unsigned char* buf) const {
        return tr_frag(buf + fb_off + KS * 32 * W::PB + B * 32, W::PB);
    }
    // One stage out of `cur`.  FULL: the stage in the registers goes to `nxt`, and the stage `s_load` into the registers.
    template <bool FULL> __device__ __forceinline__ void stage(const unsigned char* cur, unsigned char* nxt, int s_load) {
        const unsigned char *ab = nullptr, *bb = nullptr, *eb = nullptr;
        if constexpr (FULL) { ab = a_base(s_load); bb = b_base(s_load); eb = e_base(s_load); }
        constexpr int HALF = W::SL / 2;
        bf16x8 fb[W::T2], fa[3];
        static_for<W::T2>([&](auto b) { fb[decltype(b)::value] = frag_b<0, decltype(b)::value>(cur); });
        fa[0] = frag_a<0>(cur);
        fa[1] = frag_a<1>(cur);
        static_for<W::SL>([&](auto sc) {
            constexpr int S = decltype(sc)::value, a = S % W::T1;
            if constexpr (S + 2 < W::SL) fa[(S + 2) % 3] = frag_a<S + 2>(cur);
            static_for<W::T2>([&](auto bc) {
                constexpr int b = decltype(bc)::value;
                acc[a][b] = mma(fa[S % 3], fb[b], acc[a][b]);
                if constexpr (S == HALF - 1) fb[b] = frag_b<1, b>(cur);      // in its last use's place
            });
            if constexpr (FULL) {          // the chunks of codes, then those of dY
                constexpr int u0 = (S * W::UNITS + W::SL - 1) / W::SL, u1 = ((S + 1) * W::UNITS + W::SL - 1) / W::SL;
                static_for<u1 - u0>([&](auto uc) {
                    constexpr int u = u0 + decltype(uc)::value;
                    if constexpr (u < W::NB) {
                        put_b<u>(nxt);
                        load_b<u>(bb, eb);
                    } else {
                        put_a<u - W::NB>(nxt);
                        load_a<u - W::NB>(ab);
                    }
                });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    __device__ __forceinline__ void run() {
        init();
        const int nst = (m_end - m_begin + W::BM - 1) / W::BM;
        const int whole = (p.fast_rows < m_end ? p.fast_rows : m_end) - m_begin;
        const int nfast = whole > 0 ? whole / W::BM : 0;                // stages that can be read in whole chunks
        int s = 0;
        if (nfast > 2) {
            load_fast(0);
            put(lds);
            if (marks()) repair(0, lds);
            load_fast(1);
            __syncthreads();
            for (; s + 2 < nfast; ++s) {
                unsigned char* nxt = lds + ((s + 1) & 1) * W::BUF;
                const bool marked = marks();
                stage<true>(lds + (s & 1) * W::BUF, nxt, s + 2);
                if (marked) repair(s + 1, nxt);
                __syncthreads();
            }
        } else {
            load(0);
            put(lds);
            if (marks()) repair(0, lds);
            if (nst > 1) load(1);
            __syncthreads();
        }
        for (; s < nst; ++s) {
            unsigned char* nxt = lds + ((s + 1) & 1) * W::BUF;
            if (s + 1 < nst) {
                put(nxt);
                if (marks()) repair(s + 1, nxt);
            }
            if (s + 2 < nst) load_guarded(s + 2);
            stage<false>(lds + (s & 1) * W::BUF, nullptr, 0);
            __syncthreads();
        }
        float* out = p.out + split * p.slab;
#pragma unroll
        for (int a = 0; a < W::T1; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + w1 * (W::BN / W::W1) + 16 * a + 4 * (lane >> 4) + e, k = k0 + w2 * (W::BK / W::W2) + (lane & 15);
                if (n < p.N) {
                    float* q = out + (long long)n * p.K + k;
#pragma unroll
                    for (int b = 0; b < W::T2; ++b)
                        if (k + 16 * b < p.K) q[16 * b] = acc[a][b][e];
                }
            }
        if constexpr (BIAS) {      // [row threads][columns] in LDS, then one thread per column
            float* red = (float*)lds;
#pragma unroll
            for (int j = 0; j < W::AB; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) red[row() * W::BN + 64 * j + col() + k] = sum[j][k];
            __syncthreads();
            if ((int)threadIdx.x < W::BN && n0 + (int)threadIdx.x < p.N) {
                float v = 0.f;
                for (int j = 0; j < W::R; ++j) v += red[j * W::BN + threadIdx.x];
                p.out_b[split * p.slab + n0 + threadIdx.x] = v;
            }
        }
    }
};

template <class W>
__global__ __launch_bounds__(W::NT) void k_wgrad8(Wgrad8P p) {
    extern __shared__ __align__(16) unsigned char lds[];
    // Consecutive workgroups go to the 8 XCDs in turn.  Each XCD takes a compact block of tiles (4 k tiles wide), so that
    // the rows its workgroups stream at the same time are shared in its L2.
    const int unit = (int)(blockIdx.x & 7) * p.per_xcd + (int)(blockIdx.x >> 3);
    const int tiles = p.tn * p.tk;
    if (unit >= tiles * p.splits) return;
    const int split = unit / tiles, o = unit - split * tiles;
    const int kg = o / (4 * p.tn), gw = p.tk - kg * 4 < 4 ? p.tk - kg * 4 : 4, r = o - kg * 4 * p.tn;
    const int n0 = (r / gw) * W::BN, k0 = (kg * 4 + r % gw) * W::BK, m0 = split * p.rows;
    auto go = [&](auto bias) {
        Wgrad8<W, decltype(bias)::value> g(p, lds);
        g.n0 = n0; g.k0 = k0; g.split = split; g.m_begin = m0;
        g.m_end = m0 + p.rows < p.M ? m0 + p.rows : p.M;
        g.run();
    };
    if (p.out_b != nullptr && k0 == 0) go(std::integral_constant<bool, true>{});
    else go(std::integral_constant<bool, false>{});
}

// Partial results of the row splits, added in their order: entries [0, nw) to dw, [nw, n) to db.
__global__ __launch_bounds__(256) void k_wgrad8_join(long long n, long long nw, int splits, long long slab, const float* __restrict__ part,
                                                    float* __restrict__ dw, float* __restrict__ db) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = part[i];
        for (int k = 1; k < splits; ++k) s += part[k * slab + i];
        if (i < nw) dw[i] = s;
        else db[i - nw] = s;
    }
}

}  // namespace sad
