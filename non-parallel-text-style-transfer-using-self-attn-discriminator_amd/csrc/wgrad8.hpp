// Weight gradient of a linear layer from an 8-bit checkpoint of its input:
//
//   dW[n][k] = sum_m dY[m][n] X^[m][k] ,   db[n] = sum_m dY[m][n]           (m: token rows, the reduced index)
//
// X^ is decoded on its way into LDS; its values are exact in bf16 and fp16 (ckpt8.hpp), so the products are those of dY
// with the checkpoint and nothing is rounded but the fp32 sums.  dY in float32 is split into three bf16 parts
// (8 + 8 + 8 significant bits, exact), one matrix instruction each.
//
// Both operands are stored with the reduced index slow, so fragments are read from LDS with the transposing read
// (tr_frag).  Token rows are split over workgroups where the output has few tiles; the partial tiles go to a
// slab and a second launch adds them in fixed order (no atomics: the result does not depend on scheduling).
#pragma once
#include "ckpt8.hpp"
#include "gemm_core.hpp"

namespace sad {

constexpr int W8_BN = 128, W8_BK = 128, W8_BM = 64;        // outputs n, outputs k, token rows per stage
constexpr int W8_PITCH = W8_BN * 2 + 32;                   // LDS row pitch in bytes: odd multiple of 32 (tr_frag)
template <int KIND> struct W8 {
    static constexpr int PLANES = KIND == SAD_SRC_F32 ? 3 : 1;              // bf16 / fp16 images of dY
    static constexpr int LDS = W8_BM * W8_PITCH * (PLANES + 1);
};

struct Wgrad8P {
    int M, N, K, Kp;              // Kp: K rounded up to 32 (pitch of the codes)
    const void* dy; Rows2 yr; int y_flat;      // y_flat: row m starts at m * yr.s1
    const unsigned char* codes; const unsigned char* exps;
    float* out;                   // [splits][N][K], or dW itself when splits == 1
    float* out_b;                 // [splits][N] or db; NULL: no bias
    int tn, tk, splits, rows;     // tiles, row splits, rows per split (multiple of W8_BM)
};

// 8 columns of dY from c on, as loaded
template <int KIND> struct DyChunk { u32x4 v; };
template <> struct DyChunk<SAD_SRC_F32> { f32x4 a, b; };

template <int KIND>
__global__ __launch_bounds__(256) void k_wgrad8(Wgrad8P p) {
    constexpr int PLANES = W8<KIND>::PLANES, PLANE = W8_BM * W8_PITCH, CH = W8_BM * (W8_BN / 8) / 256;
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, w1 = wave >> 1, w2 = wave & 1;
    const int tile = blockIdx.x % (p.tn * p.tk), split = blockIdx.x / (p.tn * p.tk);
    const int n0 = (tile / p.tk) * W8_BN, k0 = (tile % p.tk) * W8_BK;
    const int m_begin = split * p.rows, m_end = m_begin + p.rows < p.M ? m_begin + p.rows : p.M;
    const int cc = tid & 15, rr = tid >> 4;                  // this thread's 8-column chunk and first row of a stage
    const int cn = n0 + cc * 8, ck = k0 + cc * 8;
    const int nfull = p.N - cn;                              // columns of dY left from cn on
    const bool kin = ck < p.Kp;
    DyChunk<KIND> ra[CH];
    u32x2 rb[CH];
    unsigned re[CH];
    f32x4 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};

    auto issue = [&](int m0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int m = m0 + rr + 16 * i;
            const bool ok = m < m_end;
            if constexpr (KIND == SAD_SRC_F32) ra[i].a = ra[i].b = f32x4{0.f, 0.f, 0.f, 0.f};
            else ra[i].v = u32x4{0u, 0u, 0u, 0u};
            rb[i] = u32x2{0u, 0u};
            re[i] = 1u;
            if (ok && nfull > 0) {
                const long long off = (p.y_flat ? (long long)m * p.yr.s1 : p.yr.at((unsigned)m)) + cn;
                if constexpr (KIND == SAD_SRC_F32) {
                    const float* q = (const float*)p.dy + off;
                    if (nfull >= 8) { ra[i].a = *(const f32x4u*)q; ra[i].b = *(const f32x4u*)(q + 4); }
                    else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float v = j < nfull ? q[j] : 0.f;
                            if (j < 4) ra[i].a[j] = v; else ra[i].b[j - 4] = v;
                        }
                    }
                } else {
                    const unsigned short* q = (const unsigned short*)p.dy + off;
                    if (nfull >= 8) ra[i].v = *(const u32x4h*)q;
                    else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const unsigned v = j < nfull ? q[j] : 0u;
                            ra[i].v[j >> 1] |= v << (16 * (j & 1));
                        }
                    }
                }
            }
            if (ok && kin) {
                rb[i] = *(const u32x2*)(p.codes + (long long)m * p.Kp + ck);
                re[i] = p.exps[(long long)m * (p.Kp / C8_BLOCK) + ck / C8_BLOCK];
            }
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            unsigned char* at = lds + (rr + 16 * i) * W8_PITCH + cc * 16;
            float v[8];
            if constexpr (KIND == SAD_SRC_F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = j < 4 ? ra[i].a[j] : ra[i].b[j - 4];
                float rest[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    u32x4 o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        o[j] = pack_bf16x2(rest[2 * j], rest[2 * j + 1]);
                        rest[2 * j] -= __builtin_bit_cast(float, o[j] << 16);
                        rest[2 * j + 1] -= __builtin_bit_cast(float, o[j] & 0xffff0000u);
                    }
                    *(u32x4*)(at + q * PLANE) = o;
                }
            } else {
                *(u32x4*)at = ra[i].v;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned short h = (unsigned short)(ra[i].v[j >> 1] >> (16 * (j & 1)));
                    v[j] = KIND == SAD_SRC_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) bias[j] += v[j];
            const float scale = c8_scale((int)re[i]);
            float x[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x[4 * j + 0] = c8_value_checked<0>(rb[i][j], scale);
                x[4 * j + 1] = c8_value_checked<1>(rb[i][j], scale);
                x[4 * j + 2] = c8_value_checked<2>(rb[i][j], scale);
                x[4 * j + 3] = c8_value_checked<3>(rb[i][j], scale);
            }
            u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (KIND == SAD_SRC_F16)
                    o[j] = (unsigned)__builtin_bit_cast(unsigned short, (_Float16)x[2 * j]) |
                           ((unsigned)__builtin_bit_cast(unsigned short, (_Float16)x[2 * j + 1]) << 16);
                else o[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
            }
            *(u32x4*)(at + PLANES * PLANE) = o;
        }
    };
    const int rowsel = 4 * (lane >> 4) + ((lane >> 2) & 3), p4 = (lane & 3) * 4;
    const unsigned char* abase = lds + rowsel * W8_PITCH + (w1 * 64 + p4) * 2;
    const unsigned char* bbase = lds + PLANES * PLANE + rowsel * W8_PITCH + (w2 * 64 + p4) * 2;
    issue(m_begin);
    for (int m0 = m_begin; m0 < m_end; m0 += W8_BM) {
        stage();
        __syncthreads();
        if (m0 + W8_BM < m_end) issue(m0 + W8_BM);
#pragma unroll
        for (int ks = 0; ks < W8_BM / 32; ++ks) {
            bf16x8 fb[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) fb[b] = tr_frag(bbase + ks * 32 * W8_PITCH + b * 32, W8_PITCH);
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const bf16x8 fa = tr_frag(abase + q * PLANE + ks * 32 * W8_PITCH + a * 32, W8_PITCH);
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if constexpr (KIND == SAD_SRC_F16)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fa), __builtin_bit_cast(f16x8, fb[b]),
                                                                               acc[a][b], 0, 0, 0);
                        else acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[b], acc[a][b], 0, 0, 0);
                    }
                }
        }
        __syncthreads();
    }
    float* out = p.out + (long long)split * p.N * p.K;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + w1 * 64 + 16 * a + 4 * (lane >> 4) + e, k = k0 + w2 * 64 + 16 * b + (lane & 15);
                if (n < p.N && k < p.K) out[(long long)n * p.K + k] = acc[a][b][e];
            }
    if (p.out_b != nullptr && k0 == 0) {
        float* red = (float*)lds;                           // [16 row groups][128 columns]
#pragma unroll
        for (int j = 0; j < 8; ++j) red[rr * W8_BN + cc * 8 + j] = bias[j];
        __syncthreads();
        if (tid < W8_BN && n0 + tid < p.N) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) s += red[j * W8_BN + tid];
            p.out_b[(long long)split * p.N + n0 + tid] = s;
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
