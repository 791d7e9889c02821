// gemm.h -- C[m][n] = sum_k A(m,k) B(k,n) on the matrix cores with the dense layer's epilogue, for one element type (gemm_{f16,bf16,f32}.hip).
//
// The product is computed transposed: B's columns (the layer's output features) are the A operand of the matrix instruction, A's rows (tokens)
// its B operand, so a lane ends up with four CONSECUTIVE output features of one token. P names the operand on the feature side, Q the one on the
// token side. Either may be stored with its contraction index contiguous ("row" form: a Linear weight, an activation in x W^T) or with its own
// index contiguous ("col" form: the weight in dz W; both operands in dz^T x). An LDS tile keeps the form it has in memory; row tiles are read
// with ds_read_b128, col tiles through the transposing read.
#pragma once
#include "elements.h"

namespace atlas_train {

struct GemmP {
    const unsigned char *p, *q;                 // feature side, token side
    int64_t ldp, ldq, ldc;                      // elements
    int m, n, k;
    const uint8_t *codes, *scales;              // P in 8 bits (col form), row stride ldp
    const unsigned char* bias;
    int act;
    unsigned char* save_z;
    uint8_t *save_codes, *save_scales;
    const uint8_t* keep;
    float keep_scale;
    const unsigned char* residual;
    int64_t ld_residual;
    unsigned char* c;
    float* part;                                // split product: [splits][m][n]
    int splits, k_per_split;                    // k_per_split: a multiple of the k-tile
    int tiles_n, tiles_m;
};

// four consecutive features n .. n + 3 of token m; `full`: all four exist and rows are aligned for vector access
template <class T> static __device__ __forceinline__ void epilogue4(const GemmP& g, const f4& acc, int m, int n, bool vec, const float (&z)[4]) {
    typedef typename T::elem E;
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = g.act ? gelu(z[r]) : z[r];
    if (vec) {
        if (g.save_z) store_n<T, 4>((E*)g.save_z + (int64_t)m * g.n + n, z);
        if (g.keep) {
            const uint32_t kw = *(const uint32_t*)(g.keep + (int64_t)m * g.n + n);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = (kw >> (8 * r)) & 0xffu ? y[r] * g.keep_scale : 0.f;
        }
        if (g.residual) {
            float x[4];
            load_n<T, 4>((const E*)g.residual + m * g.ld_residual + n, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] += x[r];
        }
        store_n<T, 4>((E*)g.c + m * g.ldc + n, y);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= g.n) continue;
            const int64_t at = (int64_t)m * g.n + n + r;
            if (g.save_z) ((E*)g.save_z)[at] = T::st(z[r]);
            if (g.keep) y[r] = g.keep[at] ? y[r] * g.keep_scale : 0.f;
            if (g.residual) y[r] += T::ld(((const E*)g.residual)[m * g.ld_residual + n + r]);
            ((E*)g.c)[m * g.ldc + n + r] = T::st(y[r]);
        }
    }
}
// the 32 features n0 .. n0 + 31 (a group of the 8-bit codes) of token m: two fragments of this lane and the three lanes 16, 32, 48 away
template <class T> static __device__ __forceinline__ void epilogue32(const GemmP& g, const f4& a0, const f4& a1, int m, int n0, int lg, bool vec) {
    typedef typename T::elem E;
    const bool row = m < g.m;
    const int n[2] = {n0 + 4 * lg, n0 + 16 + 4 * lg};
    float z[2][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) { z[0][r] = a0[r]; z[1][r] = a1[r]; }
    if (g.part) {
        if (!row) return;
        float* to = g.part + (int64_t)m * g.n;                               // (the caller has moved part to its split)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (n[h] + 4 <= g.n && (g.n & 3) == 0) *(f4*)(to + n[h]) = (f4){z[h][0], z[h][1], z[h][2], z[h][3]};
            else
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n[h] + r < g.n) to[n[h] + r] = z[h][r];
        }
        return;
    }
    if (g.bias) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[h][r] += n[h] + r < g.n ? T::ld(((const E*)g.bias)[n[h] + r]) : 0.f;
    }
    if (g.save_codes) {
        float top = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, n[h] + r < g.n ? finite_abs(z[h][r]) : 0.f);
        top = groups_max(top);
        if (row && n0 < g.n) {
            const int e = group_power(top);
            const int64_t ld = (g.n + 31) / 32 * 32;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = n[h] + r < g.n ? z[h][r] : 0.f;
                *(uint32_t*)(g.save_codes + m * ld + n[h]) = codes4(v[0], v[1], v[2], v[3], e, TopPower<F32>::E);
            }
            if (lg == 0) g.save_scales[m * (ld / 32) + n0 / 32] = (uint8_t)(e + 127);
        }
    }
    if (!row) return;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (n[h] < g.n) epilogue4<T>(g, h ? a1 : a0, m, n[h], vec && n[h] + 4 <= g.n, z[h]);
}
static __device__ __forceinline__ bool epilogue_vec(const GemmP& g, int size) {
    return (g.n & 3) == 0 && (g.ldc & 3) == 0 && (g.ld_residual & 3) == 0 &&
           (((uintptr_t)g.c | (uintptr_t)g.save_z | (uintptr_t)g.residual) & (4 * size - 1)) == 0 && ((uintptr_t)g.keep & 3) == 0;
}

// ---- any sizes, any alignment: 64 x 64 tiles, staged through registers ----
// 4 waves as 2 x 2, a wave 32 features x 32 tokens; the k-tile is two matrix steps (16-bit: 64, fp32: 32 indices).
// Element (i, k) of an operand lies at [i][k] (row form) or [k][i] (col form).
template <class T, bool PCOL, bool QCOL, bool CODES>
__global__ void __launch_bounds__(256) gemm_any_kernel(GemmP g) {
    typedef typename T::elem E;
    constexpr int SZ = (int)sizeof(E), BK = 2 * T::KS, R = 64;
    constexpr int PITCH_ROW = BK * SZ + 16, PITCH_COL = R * SZ + 16;
    constexpr int P_BYTES = PCOL ? BK * PITCH_COL : R * PITCH_ROW, Q_BYTES = QCOL ? BK * PITCH_COL : R * PITCH_ROW;
    __shared__ __attribute__((aligned(16))) unsigned char sp[P_BYTES], sq[Q_BYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const int n0 = (int)(blockIdx.x % g.tiles_n) * R, m0 = (int)(blockIdx.x / g.tiles_n) * R;
    const int split = blockIdx.y, kbeg = split * g.k_per_split, kend = g.k - kbeg < g.k_per_split ? g.k : kbeg + g.k_per_split;
    if (g.part) g.part += (int64_t)split * g.m * g.n;

    constexpr int EPC = 16 / SZ, NC = R * BK / EPC / 256;               // 16-byte chunks of one operand tile per thread
    const bool pv = (((uintptr_t)g.p | (uintptr_t)(g.ldp * SZ)) & 15) == 0, qv = (((uintptr_t)g.q | (uintptr_t)(g.ldq * SZ)) & 15) == 0;
    u4 xp[NC], xq[NC];
    // chunk i of this thread: rows of the tile as stored, `len` elements per row
    auto fetch = [&](const unsigned char* base, int64_t ld, bool col, bool vec, int i0, int lim, int k0, u4 (&x)[NC]) {
        const int cpr = (col ? R : BK) / EPC;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int id = i * 256 + (int)threadIdx.x, row = id / cpr, c = id % cpr * EPC;
            const int64_t r = col ? k0 + row : i0 + row, e = col ? i0 + c : k0 + c;      // row and element in memory
            const int64_t rlim = col ? kend : lim, elim = col ? lim : kend;
            x[i] = (u4){0, 0, 0, 0};
            if (r >= rlim || e >= elim) continue;
            const E* src = (const E*)base + r * ld + e;
            if (vec && e + EPC <= elim) x[i] = *(const u4*)src;
            else {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < EPC; ++j)
                    if (e + j < elim) {
                        if constexpr (SZ == 4) w[j] = as_u(src[j]);
                        else w[j / 2] |= (uint32_t)src[j] << (16 * (j & 1));
                    }
                x[i] = (u4){w[0], w[1], w[2], w[3]};
            }
        }
    };
    auto fetch_codes = [&](int i0, int k0, u4 (&x)[NC]) {               // P in col form: codes [k][ldp], ldp a multiple of 32
        constexpr int cpr = R / EPC;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int id = i * 256 + (int)threadIdx.x, row = id / cpr, c = i0 + id % cpr * EPC;
            const int64_t r = k0 + row;
            x[i] = (u4){0, 0, 0, 0};
            if (r >= kend || c >= g.n) continue;
            const float s = power_of((int)g.scales[r * (g.ldp / 32) + c / 32] - 127);
            float v[EPC];
#pragma unroll
            for (int j = 0; j < EPC; j += 4) values4(*(const uint32_t*)(g.codes + r * g.ldp + c + j), s, (float(&)[4])v[j]);
            if constexpr (SZ == 4) x[i] = (u4){as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])};
            else x[i] = (u4){pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
        }
    };
    auto put = [&](unsigned char* tile, bool col, const u4 (&x)[NC]) {
        const int cpr = (col ? R : BK) / EPC, pitch = col ? PITCH_COL : PITCH_ROW;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int id = i * 256 + (int)threadIdx.x;
            *(u4*)(tile + id / cpr * pitch + id % cpr * 16) = x[i];
        }
    };
    auto next = [&](int k0) {
        if constexpr (CODES) fetch_codes(n0, k0, xp); else fetch(g.p, g.ldp, PCOL, pv, n0, g.n, k0, xp);
        fetch(g.q, g.ldq, QCOL, qv, m0, g.m, k0, xq);
    };
    f4 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = (f4){0.f, 0.f, 0.f, 0.f};
    const int pi = (wave & 1) * 32, qi = (wave >> 1) * 32;
    if (kbeg < kend) next(kbeg);
    for (int k0 = kbeg; k0 < kend; k0 += BK) {
        __syncthreads();
        put(sp, PCOL, xp);
        put(sq, QCOL, xq);
        __syncthreads();
        if (k0 + BK < kend) next(k0 + BK);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u4 fp[2], fq[2];
            // (a col fragment enumerates the step's contraction indices as read_cols does: a row fragment beside it has to follow)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                if constexpr (PCOL) fp[a] = read_cols<T>(sp, PITCH_COL, s * T::KS, pi + 16 * a, lr, lg);
                else fp[a] = read_row_chunk<T, QCOL>(sp + (pi + 16 * a + lr) * PITCH_ROW + s * 64, lg);
                if constexpr (QCOL) fq[a] = read_cols<T>(sq, PITCH_COL, s * T::KS, qi + 16 * a, lr, lg);
                else fq[a] = read_row_chunk<T, PCOL>(sq + (qi + 16 * a + lr) * PITCH_ROW + s * 64, lg);
            }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) acc[a][b] = T::mma(fp[a], fq[b], acc[a][b]);
        }
    }
    const bool vec = epilogue_vec(g, SZ);
#pragma unroll
    for (int b = 0; b < 2; ++b) epilogue32<T>(g, acc[0][b], acc[1][b], m0 + qi + 16 * b + lr, n0 + pi, lg, vec);
}

// ---- launches ----
struct GemmPlan { int splits, k_per_split, tiles_m, tiles_n; };
template <class T> GemmPlan gemm_plan(int64_t m, int64_t n, int64_t k, bool may_split) {
    constexpr int BK = 2 * T::KS;
    GemmPlan pl;
    pl.tiles_m = (int)((m + 63) / 64);
    pl.tiles_n = (int)((n + 63) / 64);
    const int64_t tiles = (int64_t)pl.tiles_m * pl.tiles_n;
    int64_t s = 1;
    if (may_split && tiles < 1024) {                                    // fewer than four workgroups per CU: split k, no shorter than 8 k-tiles
        s = 1024 / (tiles > 0 ? tiles : 1);
        const int64_t most = (k + 8 * BK - 1) / (8 * BK);
        if (s > most) s = most;
        if (s > 64) s = 64;
        if (s < 1) s = 1;
    }
    const int64_t kt = (k + BK - 1) / BK, per = (kt + s - 1) / s;
    pl.k_per_split = (int)((per > 0 ? per : 1) * BK);
    pl.splits = (int)((k + pl.k_per_split - 1) / pl.k_per_split);
    if (pl.splits < 1) pl.splits = 1;
    return pl;
}

template <class T> int gemm_t(GemmP g, bool pcol, bool qcol, bool split, hipStream_t stream) {
    const GemmPlan pl = gemm_plan<T>(g.m, g.n, g.k, split);
    g.splits = pl.splits; g.k_per_split = pl.k_per_split; g.tiles_m = pl.tiles_m; g.tiles_n = pl.tiles_n;
    if (pl.splits == 1) g.part = nullptr;
    const dim3 grid((unsigned)(pl.tiles_m * pl.tiles_n), (unsigned)pl.splits);
    if (pcol && qcol) {
        if (g.codes) hipLaunchKernelGGL((gemm_any_kernel<T, true, true, true>), grid, dim3(256), 0, stream, g);
        else hipLaunchKernelGGL((gemm_any_kernel<T, true, true, false>), grid, dim3(256), 0, stream, g);
    } else if (pcol) hipLaunchKernelGGL((gemm_any_kernel<T, true, false, false>), grid, dim3(256), 0, stream, g);
    else if (qcol) return ATLAS_TRAIN_E_UNSUPPORTED;
    else hipLaunchKernelGGL((gemm_any_kernel<T, false, false, false>), grid, dim3(256), 0, stream, g);
    return (int)hipGetLastError();
}
template <class T> int gemm_splits(int64_t m, int64_t n, int64_t k, bool may_split) { return gemm_plan<T>(m, n, k, may_split).splits; }

}  // namespace atlas_train
