// C-ABI entry points of the gated linear recurrence and of the 8-bit activation checkpoints (include/sad.h).
// gfx950 only.  Nothing here allocates, frees or synchronises, and nothing needs zeroed workspaces.
#include "../../include/sad.h"
#include "host.hpp"
#include "scan.hpp"
#include "ckpt8.hpp"
#include "wgrad8.hpp"

#include <mutex>

using namespace sad;

namespace {

#define SAD_LAUNCHED(name)                                                                   \
    do {                                                                                     \
        hipError_t e__ = hipGetLastError();                                                  \
        if (e__ != hipSuccess) return set_error(-2, "%s: %s", name, hipGetErrorString(e__)); \
    } while (0)
#define SAD_NEED(ptr, name)                                             \
    do {                                                                \
        if ((ptr) == nullptr) return set_error(-1, "%s is NULL", name); \
    } while (0)

constexpr int MAX_GRID = 0x7fffffff;

bool known_kind(int kind) { return kind == SAD_SRC_F32 || kind == SAD_SRC_BF16 || kind == SAD_SRC_F16; }

// More than 64 KB of dynamic LDS have to be allowed once per kernel and device.
hipError_t allow_dynamic_lds(const void* kernel, int bytes) {
    static std::mutex mu;
    static const void* done[64][16];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    std::lock_guard<std::mutex> lock(mu);
    int i = 0;
    for (; i < 16 && done[dev][i] != nullptr; ++i)
        if (done[dev][i] == kernel) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && i < 16) done[dev][i] = kernel;
    return e;
}

// ---- scan ---------------------------------------------------------------------------------------------------------
// Time chunks of a sentence: one where the waves of all sentences and channel groups fill the card by themselves (bf16, uncut
// against cut: 800 waves of 300 steps, training 160 against 200 us, with 8-bit activations 216 against 238; 512 waves of 500
// steps 224 against 207 and 329 against 236), or where a sentence is so short that the second launch costs more than the cut
// saves.  Otherwise as many as give 2048 waves at
// most: what the backward kernel holds resident (two waves on each of 1024 SIMDs).  A training call at [8, 4096, 2048] with
// 8-bit activations, us: 525 with 8 chunks, 433 with 16, 453 with 32, 557 with 18 (2304 waves: a second round of 256).
int scan_chunks(int B, int T, int D) {
    const long long waves = (long long)B * ceil_div(D, SC_CH);
    const int nblk = ceil_div(T, SC_STEPS);
    if (waves >= 700 || nblk < 4) return 1;
    long long n = 2048 / waves;
    if (n > 64) n = 64;
    if (n > nblk) n = nblk;
    const int cblk = ceil_div(nblk, (int)n);
    return ceil_div(nblk, cblk);
}

int check_scan_dims(int B, int T, int D, int kind) {
    if (B < 1 || T < 1 || D < 2) return set_error(-1, "gated scan needs B >= 1, T >= 1, D >= 2 (B=%d T=%d D=%d)", B, T, D);
    if (D > (1 << 24) || T > (1 << 28)) return set_error(-1, "gated scan: D=%d or T=%d beyond the supported maximum", D, T);
    // one wave per sentence and 128 channels (more only where there are few): a launch holds fewer than 2^32 threads
    if (((long long)B * ceil_div(D, SC_CH) + 3) / 4 * 256 > 0xffffffffll) return set_error(-1, "gated scan: B=%d x D=%d beyond the supported maximum", B, D);
    if (!known_kind(kind)) return set_error(-1, "kind must be SAD_SRC_F32, SAD_SRC_BF16 or SAD_SRC_F16, got %d", kind);
    return 0;
}

ScanP scan_params(const sad_scan_args* a, void* workspace) {
    ScanP p{};
    p.B = a->B; p.T = a->T; p.D = a->D;
    p.nblk = ceil_div(a->T, SC_STEPS);
    p.ncg = ceil_div(a->D, SC_CH);
    p.reverse = a->reverse != 0;
    p.nchunk = scan_chunks(a->B, a->T, a->D);
    p.cblk = ceil_div(p.nblk, p.nchunk);
    p.z = a->z; p.z_sb = a->z_stride_b; p.z_st = a->z_stride_t;
    p.lengths = a->lengths;
    p.h0 = a->h0;
    p.y = a->y; p.y_sb = a->y_stride_b; p.y_st = a->y_stride_t;
    p.h_last = a->h_last;
    p.kept = a->kept;
    p.codes = (unsigned char*)a->codes;
    if (a->codes != nullptr) {
        const size_t tiles = (size_t)a->B * p.nblk * (a->gated ? 3 : 2);
        p.exps = p.codes + tiles * a->D * SC_STEPS;
        p.lost = (unsigned*)(p.exps + tiles * ceil_div(a->D, C8_BLOCK) * SC_STEPS);
    }
    p.dy = a->dy; p.dy_sb = a->dy_stride_b; p.dy_st = a->dy_stride_t;
    p.dh_last = a->dh_last;
    p.dz = a->dz; p.dz_sb = a->dz_stride_b; p.dz_st = a->dz_stride_t;
    p.dh0 = a->dh0;
    p.sums = (float*)workspace;
    p.group = p.nchunk < SC_GROUP ? p.nchunk : SC_GROUP;
    p.ngroup = ceil_div(p.nchunk, p.group);
    return p;
}

int scan_grid(const ScanP& p) { return (int)(((long long)p.B * p.ncg * p.nchunk + 3) / 4); }
int scan_sum_grid(const ScanP& p) { return p.B * p.ncg * p.ngroup; }

template <int KIND>
int launch_scan_fwd(const sad_scan_args* a, const ScanP& p, hipStream_t st) {
    const dim3 grid(scan_grid(p)), block(256);
    if (p.nchunk > 1) {
        hipLaunchKernelGGL((k_scan_sum<KIND>), dim3(scan_sum_grid(p)), dim3(64 * p.group), 0, st, p);
        SAD_LAUNCHED("k_scan_sum");
    }
    const int save = p.codes != nullptr ? 2 : (p.kept != nullptr ? 1 : 0);
#define SCAN_FWD(G, S) hipLaunchKernelGGL((k_scan_fwd<KIND, G, S>), grid, block, 0, st, p)
    if (a->gated) {
        if (save == 0) SCAN_FWD(true, 0);
        else if (save == 1) SCAN_FWD(true, 1);
        else SCAN_FWD(true, 2);
    } else {
        if (save == 0) SCAN_FWD(false, 0);
        else if (save == 1) SCAN_FWD(false, 1);
        else SCAN_FWD(false, 2);
    }
#undef SCAN_FWD
    SAD_LAUNCHED("k_scan_fwd");
    return 0;
}

template <int KIND, bool GATED, bool CODES>
int launch_scan_bwd(const ScanP& p, hipStream_t st) {
    const dim3 grid(scan_grid(p)), block(256);
    if (p.nchunk > 1) {
        hipLaunchKernelGGL((k_scan_bsum<KIND, GATED, CODES>), dim3(scan_sum_grid(p)), dim3(64 * p.group), 0, st, p);
        SAD_LAUNCHED("k_scan_bsum");
    }
    hipLaunchKernelGGL((k_scan_bwd<KIND, GATED, CODES>), grid, block, 0, st, p);
    SAD_LAUNCHED("k_scan_bwd");
    return 0;
}

template <int KIND>
int launch_scan_bwd(const sad_scan_args* a, const ScanP& p, hipStream_t st) {
    if (a->gated) return p.codes != nullptr ? launch_scan_bwd<KIND, true, true>(p, st) : launch_scan_bwd<KIND, true, false>(p, st);
    return p.codes != nullptr ? launch_scan_bwd<KIND, false, true>(p, st) : launch_scan_bwd<KIND, false, false>(p, st);
}

#define BY_KIND(kind, call)                                   \
    do {                                                      \
        if ((kind) == SAD_SRC_F32) { constexpr int KIND = SAD_SRC_F32; call; }        \
        else if ((kind) == SAD_SRC_BF16) { constexpr int KIND = SAD_SRC_BF16; call; } \
        else { constexpr int KIND = SAD_SRC_F16; call; }                              \
    } while (0)

// ---- checkpoints ----------------------------------------------------------------------------------------------------
int check_matrix(int64_t rows, int64_t C, int kind) {
    if (rows < 1 || C < 1) return set_error(-1, "rows and channels must be positive (rows=%lld C=%lld)", (long long)rows, (long long)C);
    if (rows > (1 << 30) || C > (1 << 24)) return set_error(-1, "rows=%lld or C=%lld beyond the supported maximum", (long long)rows, (long long)C);
    if (!known_kind(kind)) return set_error(-1, "kind must be SAD_SRC_F32, SAD_SRC_BF16 or SAD_SRC_F16, got %d", kind);
    return 0;
}

// ---- weight gradient --------------------------------------------------------------------------------------------------
// Tile and row splits by an estimate of the time: rounds of workgroups over the 256 CUs, each as long as its rows take at
// the tile's pace and a fixed start and end, and the slab of the splits, written and read once.  Paces measured in bf16 on
// [16384 rows, 6144, 2048]: 539 us with 256 x 256 tiles (192 of them), 487 with 192 x 256 (256), 664 with 128 x 320 (336, three
// splits), 738 with 128 x 128 (768); on [32768, 1536, 300] the same tiles take 71, 67, 55 and 100 us.
struct Split { int bn, bk, tn, tk, splits, rows; };
Split wgrad8_split(int64_t M, int64_t N, int64_t K, int kind) {
    struct Tile { int bn, bk; double us_per_row; };        // pace: time of a workgroup per token row, all CUs at work
    static const Tile wide[] = {{256, 256, 0.0325}, {192, 256, 0.0295}, {128, 320, 0.0285}, {128, 128, 0.0150}};
    static const Tile fp32[] = {{128, 128, 0.0400}};
    const Tile* t = kind == SAD_SRC_F32 ? fp32 : wide;
    const int nt = kind == SAD_SRC_F32 ? 1 : 4;
    Split best{};
    double best_us = 1e30;
    for (int i = 0; i < nt; ++i) {
        const int64_t tn = (N + t[i].bn - 1) / t[i].bn, tk = (K + t[i].bk - 1) / t[i].bk;
        for (int64_t n = 1; n <= 64; ++n) {
            int64_t rows = (M + n - 1) / n;
            rows = (rows + 63) / 64 * 64;
            const int64_t splits = (M + rows - 1) / rows;
            if (splits != n && n > 1) continue;
            if (n > 1 && rows < 256) break;
            const int64_t rounds = (tn * tk * splits + 255) / 256;
            const double us = rounds * (rows * t[i].us_per_row + 5.0) + (splits > 1 ? 3.0 + splits * 8.0 * N * K / 4.0e6 : 0.0);
            if (us < best_us) {
                best_us = us;
                best = Split{t[i].bn, t[i].bk, (int)tn, (int)tk, (int)splits, (int)rows};
            }
        }
    }
    return best;
}

template <int KIND, int BN, int BK, int W1, int W2>
int launch_wgrad8(const Wgrad8P& p, hipStream_t st) {
    typedef W8<KIND, BN, BK, W1, W2> W;
    if (allow_dynamic_lds((const void*)k_wgrad8<W>, W::LDS) != hipSuccess) return set_error(-2, "k_wgrad8: %d bytes of LDS refused", W::LDS);
    hipLaunchKernelGGL((k_wgrad8<W>), dim3(8u * p.per_xcd), dim3(W::NT), W::LDS, st, p);
    SAD_LAUNCHED("k_wgrad8");
    return 0;
}

template <int KIND>
int launch_wgrad8(const Wgrad8P& p, const Split& s, hipStream_t st) {
    if constexpr (KIND != SAD_SRC_F32) {
        if (s.bn == 256) return launch_wgrad8<KIND, 256, 256, 2, 4>(p, st);
        if (s.bn == 192) return launch_wgrad8<KIND, 192, 256, 2, 4>(p, st);
        if (s.bk == 320) return launch_wgrad8<KIND, 128, 320, 2, 4>(p, st);
    }
    return launch_wgrad8<KIND, 128, 128, 2, 2>(p, st);
}

}  // namespace

extern "C" {

size_t sad_gated_scan_workspace_bytes(int32_t B, int32_t T, int32_t D) {
    if (check_scan_dims(B, T, D, SAD_SRC_F32)) return 0;
    const int n = scan_chunks(B, T, D);
    return n > 1 ? (size_t)B * (n + ceil_div(n, n < SC_GROUP ? n : SC_GROUP)) * 2 * D * sizeof(float) : 16;
}

size_t sad_gated_scan_kept_bytes(int32_t B, int32_t T, int32_t D) {
    if (check_scan_dims(B, T, D, SAD_SRC_F32)) return 0;
    return (size_t)B * ceil_div(T, SC_STEPS) * D * sizeof(float);
}

size_t sad_gated_scan_codes_bytes(int32_t B, int32_t T, int32_t D, int32_t gated) {
    if (check_scan_dims(B, T, D, SAD_SRC_F32)) return 0;
    const size_t blocks = (size_t)B * ceil_div(T, SC_STEPS);
    return blocks * ((gated ? 3 : 2) * ((size_t)D + ceil_div(D, C8_BLOCK)) * SC_STEPS + ceil_div(D, SC_CH) * sizeof(unsigned));
}

int sad_gated_scan_fwd(const sad_scan_args* a, void* workspace, void* stream) {
    SAD_NEED(a, "args");
    if (check_scan_dims(a->B, a->T, a->D, a->kind)) return -1;
    SAD_NEED(a->z, "z");
    SAD_NEED(a->y, "y");
    SAD_NEED(a->h_last, "h_last");
    SAD_NEED(workspace, "workspace");
    if (a->codes != nullptr && a->kept == nullptr) return set_error(-1, "codes need kept");
    if ((size_t)a->codes % 16) return set_error(-1, "codes must be 16-byte aligned");
    const ScanP p = scan_params(a, workspace);
    BY_KIND(a->kind, return launch_scan_fwd<KIND>(a, p, (hipStream_t)stream));
}

int sad_gated_scan_bwd(const sad_scan_args* a, void* workspace, void* stream) {
    SAD_NEED(a, "args");
    if (check_scan_dims(a->B, a->T, a->D, a->kind)) return -1;
    if (a->z == nullptr && a->codes == nullptr) return set_error(-1, "need z or codes");
    SAD_NEED(a->kept, "kept");
    SAD_NEED(a->dz, "dz");
    SAD_NEED(workspace, "workspace");
    if ((size_t)a->codes % 16) return set_error(-1, "codes must be 16-byte aligned");
    const ScanP p = scan_params(a, workspace);
    BY_KIND(a->kind, return launch_scan_bwd<KIND>(a, p, (hipStream_t)stream));
}

int sad_gated_scan_step(int32_t B, int32_t D, int32_t kind, int32_t gated, const void* z, int64_t z_stride_b, const float* h,
                        int64_t h_stride_b, const uint8_t* alive, void* y, int64_t y_stride_b, float* h_out, int64_t h_out_stride_b,
                        void* stream) {
    if (B < 1 || D < 1) return set_error(-1, "B and D must be positive (B=%d D=%d)", B, D);
    const int per = ceil_div(D, 256);
    if ((int64_t)B * per > MAX_GRID) return set_error(-1, "B=%d x D=%d beyond the supported maximum", B, D);
    if (!known_kind(kind)) return set_error(-1, "kind must be SAD_SRC_F32, SAD_SRC_BF16 or SAD_SRC_F16, got %d", kind);
    SAD_NEED(z, "z");
    SAD_NEED(h, "h");
    SAD_NEED(y, "y");
    SAD_NEED(h_out, "h_out");
    const dim3 grid((unsigned)B * per);
#define SCAN_STEP(G)                                                                                                          \
    hipLaunchKernelGGL((k_scan_step<KIND, G>), grid, dim3(256), 0, (hipStream_t)stream, D, per, z, (long long)z_stride_b, h,   \
                       (long long)h_stride_b, alive, y, (long long)y_stride_b, h_out, (long long)h_out_stride_b)
    if (gated) BY_KIND(kind, SCAN_STEP(true));
    else BY_KIND(kind, SCAN_STEP(false));
#undef SCAN_STEP
    SAD_LAUNCHED("k_scan_step");
    return 0;
}

size_t sad_checkpoint8_bytes(int64_t rows, int64_t C) {
    if (check_matrix(rows, C, SAD_SRC_F32)) return 0;
    const size_t nb = (size_t)((C + C8_BLOCK - 1) / C8_BLOCK);
    return (size_t)rows * nb * (C8_BLOCK + 2);        // codes, exponents, exponents of marked blocks
}

int sad_checkpoint8_save(int64_t n0, int64_t n1, int64_t C, int32_t kind, const void* x, int64_t stride0, int64_t stride1,
                         void* saved, void* stream) {
    if (n0 < 1 || n1 < 1) return set_error(-1, "rows must be positive (%lld x %lld)", (long long)n0, (long long)n1);
    if (n0 > MAX_GRID || n1 > MAX_GRID) return set_error(-1, "rows beyond the supported maximum");
    const int64_t rows = n0 * n1;
    if (check_matrix(rows, C, kind)) return -1;
    SAD_NEED(x, "x");
    SAD_NEED(saved, "saved");
    if ((size_t)saved % 16) return set_error(-1, "saved must be 16-byte aligned");
    const int nb = (int)((C + C8_BLOCK - 1) / C8_BLOCK), per = 2 * nb, rpb = per < 256 ? 256 / per : 1;
    unsigned char* codes = (unsigned char*)saved;
    unsigned char* exps = codes + (size_t)rows * nb * C8_BLOCK;
    const Rows2 xr{stride0, stride1, (unsigned)n1};
    BY_KIND(kind, hipLaunchKernelGGL((k_ckpt8_save<KIND>), dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0, (hipStream_t)stream,
                                     (int)rows, (int)C, per, rpb, x, xr, codes, exps, exps + (size_t)rows * nb));
    SAD_LAUNCHED("k_ckpt8_save");
    return 0;
}

int sad_checkpoint8_restore(int64_t rows, int64_t C, int32_t kind, const void* saved, void* out, void* stream) {
    if (check_matrix(rows, C, kind)) return -1;
    SAD_NEED(saved, "saved");
    SAD_NEED(out, "out");
    if ((size_t)saved % 16) return set_error(-1, "saved must be 16-byte aligned");
    const int nb = (int)((C + C8_BLOCK - 1) / C8_BLOCK), per = 2 * nb, rpb = per < 256 ? 256 / per : 1;
    const unsigned char* codes = (const unsigned char*)saved;
    const unsigned char* exps = codes + (size_t)rows * nb * C8_BLOCK;
    BY_KIND(kind, hipLaunchKernelGGL((k_ckpt8_restore<KIND>), dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0,
                                     (hipStream_t)stream, (int)rows, (int)C, per, rpb, codes, exps, exps + (size_t)rows * nb, out));
    SAD_LAUNCHED("k_ckpt8_restore");
    return 0;
}

size_t sad_weight_grad8_workspace_bytes(int64_t rows, int64_t N, int64_t K, int32_t kind) {
    if (check_matrix(rows, K, kind) || check_matrix(rows, N, kind)) return 0;
    const Split s = wgrad8_split(rows, N, K, kind);
    return s.splits > 1 ? (size_t)s.splits * (N * K + N) * sizeof(float) : 16;
}

int sad_weight_grad8(int64_t n0, int64_t n1, int64_t N, int64_t K, int32_t kind, const void* dy, int64_t stride0, int64_t stride1,
                     const void* saved, float* dw, float* db, void* workspace, void* stream) {
    if (n0 < 1 || n1 < 1) return set_error(-1, "rows must be positive (%lld x %lld)", (long long)n0, (long long)n1);
    if (n0 > MAX_GRID || n1 > MAX_GRID) return set_error(-1, "rows beyond the supported maximum");
    const int64_t M = n0 * n1;
    if (check_matrix(M, K, kind) || check_matrix(M, N, kind)) return -1;
    SAD_NEED(dy, "dy");
    SAD_NEED(saved, "saved");
    SAD_NEED(dw, "dw");
    SAD_NEED(workspace, "workspace");
    if ((size_t)saved % 16) return set_error(-1, "saved must be 16-byte aligned");
    const Split s = wgrad8_split(M, N, K, kind);
    const int64_t groups = (int64_t)s.tn * s.tk * s.splits;
    if (groups > MAX_GRID) return set_error(-1, "N=%lld x K=%lld beyond the supported maximum", (long long)N, (long long)K);
    Wgrad8P p{};
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.Kp = (int)((K + C8_BLOCK - 1) / C8_BLOCK * C8_BLOCK);
    p.dy = dy;
    p.yr = Rows2{stride0, stride1, (unsigned)n1};
    p.y_flat = n0 == 1 || stride0 == n1 * stride1;
    // Chunks of 8 columns reach `over` entries past a row's end where N is no multiple of 8: memory of the rows behind, which
    // is there for all rows but the last few.
    const int64_t over = (8 - N % 8) % 8;
    p.fast_rows = !p.y_flat || stride1 > (1 << 22) ? 0 : (over == 0 ? (int)M : (stride1 > 0 ? (int)(M - (over + stride1 - 1) / stride1) : 0));
    p.codes = (const unsigned char*)saved;
    p.exps = p.codes + (size_t)M * p.Kp;
    p.marked = p.exps + (size_t)M * (p.Kp / C8_BLOCK);
    p.per_xcd = (int)((groups + 7) / 8);
    p.tn = s.tn; p.tk = s.tk; p.splits = s.splits; p.rows = s.rows;
    p.out = s.splits > 1 ? (float*)workspace : dw;
    p.out_b = db == nullptr ? nullptr : (s.splits > 1 ? p.out + N * K : db);
    p.slab = N * K + N;
    hipStream_t st = (hipStream_t)stream;
    int rc = 0;
    BY_KIND(kind, rc = launch_wgrad8<KIND>(p, s, st));
    if (rc != 0) return rc;
    if (s.splits > 1) {
        const long long n = db == nullptr ? (long long)N * K : p.slab, g = (n + 255) / 256;
        hipLaunchKernelGGL(k_wgrad8_join, dim3((unsigned)(g < 8192 ? g : 8192)), dim3(256), 0, st, n, (long long)N * K, s.splits, p.slab,
                           (const float*)workspace, dw, db);
        SAD_LAUNCHED("k_wgrad8_join");
    }
    return 0;
}

}  // extern "C"
