// Weight gradient of a linear layer from an 8-bit checkpoint of its input:
//
//   dW[n][k] = sum_m dY[m][n] X^[m][k] ,   db[n] = sum_m dY[m][n]           (m: token rows, the reduced index)
//
// X^ is decoded on its way into LDS; its values are exact in bf16 and fp16 (ckpt8.hpp), so the products are those of dY
// with the checkpoint and nothing is rounded but the fp32 sums.  dY in float32 is split into three bf16 parts
// (8 + 8 + 8 significant bits, exact), one matrix instruction each.  db is one more column of ones for the matrix
// instructions of the workgroups of the first k tile.
//
// Both operands are stored with the reduced index slow, so fragments are read from LDS with the transposing read
// (tr_frag).  Token rows are split over workgroups where the output has few tiles; the partial tiles go to a slab and a
// second launch adds them in fixed order (no atomics: the result does not depend on scheduling).
//
// Pipeline, one barrier per stage of 64 rows: stage s is multiplied out of one LDS buffer while stage s + 1 moves from
// registers (decoded) into the other and the loads of stage s + 2 are issued.  Half of the waves stage first and multiply
// then, the other half the other way round, and each SIMD holds one of each: the decoding (vector) of one overlaps the
// matrix instructions of the other.
#pragma once
#include "ckpt8.hpp"
#include "gemm_core.hpp"

namespace sad {

// Workgroup tile BN x BK outputs, W1 x W2 waves.
template <int KIND_, int BN_, int BK_, int W1_, int W2_> struct W8 {
    static constexpr int KIND = KIND_, BN = BN_, BK = BK_, W1 = W1_, W2 = W2_;
    static constexpr int BM = 64;                              // token rows per stage
    static constexpr int NT = 64 * W1 * W2;
    static constexpr int T1 = BN / W1 / 16, T2 = BK / W2 / 16;
    static constexpr int PLANES = KIND == SAD_SRC_F32 ? 3 : 1; // bf16 / fp16 images of dY
    static constexpr int PA = BN * 2 + 32, PB = BK * 2 + 32;   // LDS row pitch in bytes: odd multiples of 32 (tr_frag)
    static constexpr int ABYTES = BM * PA, BUF = PLANES * ABYTES + BM * PB;
    static constexpr int LDS = 2 * BUF;
    static constexpr int CA = BN / 8, CB = BK / 16;            // chunks of a row: 8 entries of dY, 16 codes
    static constexpr int NA = BM * CA / NT, NB = BM * CB / NT; // chunks per thread
    static_assert(BM * CA % NT == 0 && BM * CB % NT == 0, "staging must divide evenly");
    static_assert(BN % (W1 * 16) == 0 && BK % (W2 * 16) == 0 && (BN / 16) % 2 == 0 && (BK / 16) % 2 == 0, "tile");
};

struct Wgrad8P {
    int M, N, K, Kp;              // Kp: K rounded up to 32 (pitch of the codes)
    const void* dy; Rows2 yr; int y_flat;      // y_flat: row m starts at m * yr.s1
    int fast_rows;                // rows in front of this one may be read in whole chunks of 8 columns
    const unsigned char* codes; const unsigned char* exps;
    float* out;                   // [splits][N][K], or dW itself when splits == 1
    float* out_b;                 // [splits][N] or db; NULL: no bias
    int tn, tk, splits, rows;     // tiles, row splits, rows per split (multiple of 64)
    int per_xcd;                  // workgroups per XCD
};

// 8 entries of dY as loaded
template <int KIND> struct DyChunk { u32x4 v; };
template <> struct DyChunk<SAD_SRC_F32> { f32x4 a, b; };

__device__ __forceinline__ unsigned c8_pack16(float a, float b, bool half) {
    if (half) return (unsigned)__builtin_bit_cast(unsigned short, (_Float16)a) | ((unsigned)__builtin_bit_cast(unsigned short, (_Float16)b) << 16);
    // exact in bf16: the upper halves
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}

template <class W>
__global__ __launch_bounds__(W::NT) void k_wgrad8(Wgrad8P p) {
    constexpr int KIND = W::KIND, EB = Elem<KIND>::bytes;
    extern __shared__ __align__(16) unsigned char lds[];
    // Consecutive workgroups go to the 8 XCDs in turn.  Each XCD takes a compact block of tiles (4 k tiles wide), so that
    // the rows its workgroups stream at the same time are shared in its L2.
    const int unit = (int)(blockIdx.x & 7) * p.per_xcd + (int)(blockIdx.x >> 3);
    const int tiles = p.tn * p.tk;
    if (unit >= tiles * p.splits) return;
    const int split = unit / tiles, o = unit - split * tiles;
    const int kg = o / (4 * p.tn), gw = p.tk - kg * 4 < 4 ? p.tk - kg * 4 : 4, r = o - kg * 4 * p.tn;
    const int n0 = (r / gw) * W::BN, k0 = (kg * 4 + r % gw) * W::BK;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w1 = wave / W::W2, w2 = wave % W::W2;
    const int m_begin = split * p.rows, m_end = m_begin + p.rows < p.M ? m_begin + p.rows : p.M;
    const int nst = (m_end - m_begin + W::BM - 1) / W::BM;
    const bool bias = p.out_b != nullptr && k0 == 0;

    // this thread's chunks of a stage
    int arow[W::NA], acol[W::NA], brow[W::NB], bcol[W::NB];
    const unsigned char* ap[W::NA];
    const unsigned char* bp[W::NB];
    const unsigned char* ep[W::NB];
#pragma unroll
    for (int i = 0; i < W::NA; ++i) {
        const int g = tid + i * W::NT;
        arow[i] = g / W::CA;
        acol[i] = (g - arow[i] * W::CA) * 8;
        // chunks that lie past the last column read the first one (their products are not stored)
        ap[i] = (const unsigned char*)p.dy + ((long long)(m_begin + arow[i]) * p.yr.s1 + (n0 + acol[i] < p.N ? n0 + acol[i] : 0)) * EB;
    }
#pragma unroll
    for (int i = 0; i < W::NB; ++i) {
        const int g = tid + i * W::NT;
        brow[i] = g / W::CB;
        bcol[i] = (g - brow[i] * W::CB) * 16;
        const int c = k0 + bcol[i] < p.Kp ? k0 + bcol[i] : 0;
        bp[i] = p.codes + (long long)(m_begin + brow[i]) * p.Kp + c;
        ep[i] = p.exps + (long long)(m_begin + brow[i]) * (p.Kp / C8_BLOCK) + c / C8_BLOCK;
    }
    const long long astep = (long long)W::BM * p.yr.s1 * EB, bstep = (long long)W::BM * p.Kp, estep = bstep / C8_BLOCK;

    DyChunk<KIND> ra[W::NA];
    u32x4 rb[W::NB];
    unsigned re[W::NB];
    auto issue = [&](int s) {
        const int m0 = m_begin + s * W::BM;
        if (m0 + W::BM <= p.fast_rows && m0 + W::BM <= m_end) {
#pragma unroll
            for (int i = 0; i < W::NA; ++i) {
                if constexpr (KIND == SAD_SRC_F32) {
                    ra[i].a = *(const f32x4u*)ap[i];
                    ra[i].b = *(const f32x4u*)(ap[i] + 16);
                } else ra[i].v = *(const u32x4h*)ap[i];
            }
#pragma unroll
            for (int i = 0; i < W::NB; ++i) {
                rb[i] = *(const u32x4*)bp[i];
                re[i] = *ep[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < W::NA; ++i) {
                if constexpr (KIND == SAD_SRC_F32) ra[i].a = ra[i].b = f32x4{0.f, 0.f, 0.f, 0.f};
                else ra[i].v = u32x4{0u, 0u, 0u, 0u};
                const int m = m0 + arow[i], c = n0 + acol[i];
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
                rb[i] = u32x4{0u, 0u, 0u, 0u};
                re[i] = 1u;
                if (m0 + brow[i] < m_end) {
                    rb[i] = *(const u32x4*)bp[i];
                    re[i] = *ep[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < W::NA; ++i) ap[i] += astep;
#pragma unroll
        for (int i = 0; i < W::NB; ++i) { bp[i] += bstep; ep[i] += estep; }
    };
    auto stage = [&](unsigned char* buf) {
#pragma unroll
        for (int i = 0; i < W::NA; ++i) {
            unsigned char* at = buf + arow[i] * W::PA + acol[i] * 2;
            if constexpr (KIND == SAD_SRC_F32) {
                float rest[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) rest[j] = j < 4 ? ra[i].a[j] : ra[i].b[j - 4];
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    u32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[j] = pack_bf16x2(rest[2 * j], rest[2 * j + 1]);
                        rest[2 * j] -= __builtin_bit_cast(float, v[j] << 16);
                        rest[2 * j + 1] -= __builtin_bit_cast(float, v[j] & 0xffff0000u);
                    }
                    *(u32x4*)(at + q * W::ABYTES) = v;
                }
            } else *(u32x4*)at = ra[i].v;
        }
#pragma unroll
        for (int i = 0; i < W::NB; ++i) {
            const float scale = c8_scale((int)re[i]);
            u32x4 v[2];
            float low = 0.f;                  // smallest code: -128 where an entry was lost
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned w = rb[i][j];
                const float c0 = c8_int<0>(w), c1 = c8_int<1>(w), c2 = c8_int<2>(w), c3 = c8_int<3>(w);
                low = fminf(fminf(low, c0), c1);
                low = fminf(fminf(low, c2), c3);
                v[j >> 1][(j & 1) * 2] = c8_pack16(c0 * scale, c1 * scale, KIND == SAD_SRC_F16);
                v[j >> 1][(j & 1) * 2 + 1] = c8_pack16(c2 * scale, c3 * scale, KIND == SAD_SRC_F16);
            }
            if (__any(low < -127.5f)) {       // a lost entry's NaN
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (((rb[i][j >> 2] >> (8 * (j & 3))) & 0xffu) == C8_LOST) v[j >> 3][(j >> 1) & 3] |= 0x7fffu << (16 * (j & 1));
            }
            unsigned char* at = buf + W::PLANES * W::ABYTES + brow[i] * W::PB + bcol[i] * 2;
            *(u32x4*)at = v[0];
            *(u32x4*)(at + 16) = v[1];
        }
    };

    f32x4 acc[W::T1][W::T2], accb[2];
#pragma unroll
    for (int a = 0; a < W::T1; ++a)
#pragma unroll
        for (int b = 0; b < W::T2; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    accb[0] = accb[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned one = KIND == SAD_SRC_F16 ? 0x3c003c00u : 0x3f803f80u;
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{one, one, one, one});
    auto mma = [](bf16x8 a, bf16x8 b, f32x4 c) {
        if constexpr (KIND == SAD_SRC_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    };
    const int rowsel = 4 * (lane >> 4) + ((lane >> 2) & 3), p4 = (lane & 3) * 4;
    const int aoff = rowsel * W::PA + (w1 * (W::BN / W::W1) + p4) * 2;
    const int boff = W::PLANES * W::ABYTES + rowsel * W::PB + (w2 * (W::BK / W::W2) + p4) * 2;
    auto multiply = [&](const unsigned char* buf) {
#pragma unroll
        for (int ks = 0; ks < W::BM / 32; ++ks) {
            bf16x8 fb[W::T2];
#pragma unroll
            for (int b = 0; b < W::T2; ++b) fb[b] = tr_frag(buf + boff + ks * 32 * W::PB + b * 32, W::PB);
#pragma unroll
            for (int q = 0; q < W::PLANES; ++q)
#pragma unroll
                for (int a = 0; a < W::T1; ++a) {
                    const bf16x8 fa = tr_frag(buf + aoff + q * W::ABYTES + ks * 32 * W::PA + a * 32, W::PA);
#pragma unroll
                    for (int b = 0; b < W::T2; ++b) acc[a][b] = mma(fa, fb[b], acc[a][b]);
                }
        }
        if (bias) {      // uniform: the waves of a row of the workgroup share its columns
#pragma unroll
            for (int ks = 0; ks < W::BM / 32; ++ks)
#pragma unroll
                for (int q = 0; q < W::PLANES; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (w2 + j * W::W2 < W::T1)
                            accb[j] = mma(tr_frag(buf + aoff + q * W::ABYTES + ks * 32 * W::PA + (w2 + j * W::W2) * 32, W::PA), ones, accb[j]);
        }
    };

    issue(0);
    stage(lds);
    if (nst > 1) issue(1);
    __syncthreads();
    const bool early = wave < W::W1 * W::W2 / 2;
    for (int s = 0; s < nst; ++s) {
        unsigned char* cur = lds + (s & 1) * W::BUF;
        unsigned char* nxt = lds + ((s + 1) & 1) * W::BUF;
        if (early && s + 1 < nst) {
            stage(nxt);
            if (s + 2 < nst) issue(s + 2);
        }
        __builtin_amdgcn_s_setprio(1);      // the SIMD's other wave is staging
        multiply(cur);
        __builtin_amdgcn_s_setprio(0);
        if (!early && s + 1 < nst) {
            stage(nxt);
            if (s + 2 < nst) issue(s + 2);
        }
        __syncthreads();
    }
    float* out = p.out + (long long)split * p.N * p.K;
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
    if (bias && (lane & 15) == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int a = w2 + j * W::W2, n = n0 + w1 * (W::BN / W::W1) + 16 * a + 4 * (lane >> 4) + e;
                if (a < W::T1 && n < p.N) p.out_b[(long long)split * p.N + n] = accb[j][e];
            }
    }
}

// Partial results of the row splits, added in their order: out[i] = sum_s part[s][i].
__global__ __launch_bounds__(256) void k_wgrad8_join(long long n, int splits, const float* __restrict__ part, float* __restrict__ out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = part[i];
        for (int k = 1; k < splits; ++k) s += part[(long long)k * n + i];
        out[i] = s;
    }
}

}  // namespace sad
