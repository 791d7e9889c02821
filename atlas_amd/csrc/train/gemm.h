// gemm.h -- C[m][n] = sum_k A(m,k) B(k,n) on the matrix cores with the dense layer's epilogue, for one element type (gemm_{f16,bf16,f32}.hip).
//
// The product is computed transposed: B's columns (the layer's output features) are the A operand of the matrix instruction, A's rows (tokens)
// its B operand, so a lane ends up with four CONSECUTIVE output features of one token. P names the operand on the feature side, Q the one on the
// token side. Either may be stored with its contraction index contiguous ("row" form: a Linear weight, an activation in x W^T) or with its own
// index contiguous ("col" form: the weight in dz W; both operands in dz^T x). An LDS tile keeps the form it has in memory; row tiles are read
// with ds_read_b128, col tiles through the transposing read.
#pragma once
#include <type_traits>
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

// The pre-activation is saved in the tensors' type (or 8 bits, from fp32): only the activation's slope is taken from it, whose error is at most 0.8 of z's; fp32 would
// take 170 MB more, there and back, of 13 848 x 3 072.
// four consecutive features n .. n + 3 of token m, at any alignment; fewer at a row's end
template <class T> static __device__ __forceinline__ void epilogue4(const GemmP& g, int m, int n, const float (&z)[4]) {
    typedef typename T::elem E;
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = g.act ? gelu(z[r]) : z[r];
    const int64_t at = (int64_t)m * g.n + n;
    if (n + 4 <= g.n) {
        if (g.save_z) store4_any<T>((E*)g.save_z + at, z);
        if (g.keep) {
            const uint32_t kw = *(const u32_any*)(g.keep + at);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = (kw >> (8 * r)) & 0xffu ? y[r] * g.keep_scale : 0.f;
        }
        if (g.residual) {
            float x[4];
            load4_any<T>((const E*)g.residual + m * g.ld_residual + n, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] += x[r];
        }
        store4_any<T>((E*)g.c + m * g.ldc + n, y);
    } else
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= g.n) continue;
            if (g.save_z) ((E*)g.save_z)[at + r] = T::st(z[r]);
            if (g.keep) y[r] = g.keep[at + r] ? y[r] * g.keep_scale : 0.f;
            if (g.residual) y[r] += T::ld(((const E*)g.residual)[m * g.ld_residual + n + r]);
            ((E*)g.c)[m * g.ldc + n + r] = T::st(y[r]);
        }
}
// the 32 features n0 .. n0 + 31 (a group of the 8-bit codes) of token m: two fragments of this lane and the three lanes 16, 32, 48 away
template <class T> static __device__ __forceinline__ void epilogue32(const GemmP& g, const f4& a0, const f4& a1, int m, int n0, int lg) {
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
            if (n[h] + 4 <= g.n) store4_any<F32>(to + n[h], z[h]);
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
        float v[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * h + r] = n[h] + r < g.n ? z[h][r] : 0.f;
        const GroupPower e = group_power4<8, 16>(v);
        if (row && n0 < g.n) {
            const int64_t ld = (g.n + 31) / 32 * 32;
            uint32_t w[2];
            encode<8>(v, e, TopPower<F32>::E, w);
#pragma unroll
            for (int h = 0; h < 2; ++h) *(uint32_t*)(g.save_codes + m * ld + n[h]) = w[h];
            if (lg == 0) g.save_scales[m * (ld / 32) + n0 / 32] = (uint8_t)(e.e + 127);
        }
    }
    if (!row) return;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (n[h] < g.n) epilogue4<T>(g, m, n[h], z[h]);
}

// ---- any sizes, any alignment: R x R tiles, staged through registers ----
// A CU takes in some 20 GB/s here, so what a small product costs is the bytes of one workgroup: the contraction is split over workgroups until the chip is
// full (41 x 768 x 768 bf16: 12 tiles in 12.7 us; 72 parts in 4.3 and their join in 4.6), never over more waves of the same workgroup (four groups of waves
// taking turns at the k-tiles of a tile: 11.8 us).
// 4 waves as 2 x 2, a wave R / 2 features x R / 2 tokens; R = 128 or 64 by estimated time (gemm_plan); the k-tile is two matrix steps (16-bit: 64, fp32: 32 indices).
// Element (i, k) of an operand lies at [i][k] (row form) or [k][i] (col form).
template <class T, bool PCOL, bool QCOL, bool CODES, int R>
__global__ void __launch_bounds__(256) gemm_any_kernel(GemmP g) {
    typedef typename T::elem E;
    constexpr int SZ = (int)sizeof(E), BK = 2 * T::KS, F = R / 32;
    constexpr int PITCH_ROW = BK * SZ + 16, PITCH_COL = R * SZ + 16;
    constexpr int P_BYTES = PCOL ? BK * PITCH_COL : R * PITCH_ROW, Q_BYTES = QCOL ? BK * PITCH_COL : R * PITCH_ROW;
    __shared__ __attribute__((aligned(16))) unsigned char sp[P_BYTES], sq[Q_BYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const int n0 = (int)(blockIdx.x % g.tiles_n) * R, m0 = (int)(blockIdx.x / g.tiles_n) * R;
    const int split = blockIdx.y, kbeg = split * g.k_per_split, kend = g.k - kbeg < g.k_per_split ? g.k : kbeg + g.k_per_split;
    if (g.part) g.part += (int64_t)split * g.m * g.n;

    constexpr int EPC = 16 / SZ, NC = R * BK / EPC / 256;               // 16-byte chunks of one operand tile per thread
    u4 xp[NC], xq[NC];
    // chunk i of this thread: rows of the tile as stored, `len` elements per row
    auto fetch = [&](const unsigned char* base, int64_t ld, bool col, int i0, int lim, int k0, u4 (&x)[NC]) {
        const int cpr = (col ? R : BK) / EPC;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int id = i * 256 + (int)threadIdx.x, row = id / cpr, c = id % cpr * EPC;
            const int64_t r = col ? k0 + row : i0 + row, e = col ? i0 + c : k0 + c;      // row and element in memory
            const int64_t rlim = col ? kend : lim, elim = col ? lim : kend;
            x[i] = (u4){0, 0, 0, 0};
            if (r >= rlim || e >= elim) continue;
            const E* src = (const E*)base + r * ld + e;
            if (e + EPC <= elim) x[i] = *(const u4_any*)src;
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
        if constexpr (CODES) fetch_codes(n0, k0, xp); else fetch(g.p, g.ldp, PCOL, n0, g.n, k0, xp);
        fetch(g.q, g.ldq, QCOL, m0, g.m, k0, xq);
    };
    f4 acc[F][F];
#pragma unroll
    for (int a = 0; a < F; ++a)
#pragma unroll
        for (int b = 0; b < F; ++b) acc[a][b] = (f4){0.f, 0.f, 0.f, 0.f};
    const int pi = (wave & 1) * (R / 2), qi = (wave >> 1) * (R / 2);
    if (kbeg < kend) next(kbeg);
    for (int k0 = kbeg; k0 < kend; k0 += BK) {
        __syncthreads();
        put(sp, PCOL, xp);
        put(sq, QCOL, xq);
        __syncthreads();
        if (k0 + BK < kend) next(k0 + BK);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u4 fp[F], fq[F];
            // (a col fragment enumerates the step's contraction indices as read_cols does: a row fragment beside it has to follow)
#pragma unroll
            for (int a = 0; a < F; ++a) {
                if constexpr (PCOL) fp[a] = read_cols<T>(sp, PITCH_COL, s * T::KS, pi + 16 * a, lr, lg);
                else fp[a] = read_row_chunk<T, QCOL>(sp + (pi + 16 * a + lr) * PITCH_ROW + s * 64, lg);
                if constexpr (QCOL) fq[a] = read_cols<T>(sq, PITCH_COL, s * T::KS, qi + 16 * a, lr, lg);
                else fq[a] = read_row_chunk<T, PCOL>(sq + (qi + 16 * a + lr) * PITCH_ROW + s * 64, lg);
            }
            mma_block<T, F, F>(fp, fq, acc);
        }
    }
#pragma unroll
    for (int b = 0; b < F; ++b)
#pragma unroll
        for (int a = 0; a < F; a += 2) epilogue32<T>(g, acc[a][b], acc[a + 1][b], m0 + qi + 16 * b + lr, n0 + pi + 16 * a, lg);
}

// ---- the bulk of the work: 256 x 256 tiles, both operands by LDS-DMA, the two waves of a SIMD in opposite phases ----
// 8 waves as 2 (features) x 4 (tokens), a wave 128 x 64: 8 x 4 fragments, 128 accumulator registers. (Or 256 features x 192 tokens, FB = 3, with tokens in row form:
// less work a byte, but where it saves a round of tiles over the 256 CUs, or fills them better, faster: 13 848 x 3 072 -> 768 fp16 78 us for 92, 9 000 x 768 -> 768
// bf16 29 for 35; 20 011 x 768 -> 3 072 with codes 177 for 173, so not there.) A k-tile is 128 bytes of contraction (two matrix steps):
// 32 KiB an operand, two stages: 128 KiB of LDS. Waves w and w + 4 share a SIMD: while one reads its 24 fragments of a k-tile, the other multiplies (64 matrix
// instructions), a barrier between the phases:
//     phase 2k     A reads tile k, then sends for tile k + 1          | B sends for tile k + 1, multiplies tile k - 1
//     phase 2k + 1 A multiplies tile k, then waits for its own pieces | B waits for its own pieces, reads tile k
// (pieces of tile k + 1 go where tile k - 1 was, which A left in phase 2k - 2 and B in phase 2k - 1). Bounds are the buffer descriptors': rows and
// contraction indices behind the end arrive as zeros.
// LDS images. Row form: 128-byte rows, 16-byte chunk c of row r at place c ^ ((r >> 1) & 7) (rows r and r + 1 lie in different halves of the banks). Col form: the contraction index is the row (512 or 1024 bytes of 256
// own indices); 16-bit: the 32-byte piece s of row r at place s ^ (r & 7), so that the eight rows a transposing read touches at once lie in
// different banks; fp32: the 64-byte piece s at place s ^ ((r >> 2) & 3). The swizzle is in the DMA's source address.
// What bounds it: a k-tile takes some 1.9 us where its products take 0.95 (61 441 x 3 072 -> 768 bf16: 282 us = 1.03 PFLOP/s); the matrix unit is busy 38 .. 53 % of a long
// product. The rest is the pieces' way: when a wave sends is what it comes down to. Sent before the reads instead of behind them (A) 337 us for 313 (in runs of a dozen
// launches), between the products (B) 347, with a touch of the lines a tile further ahead 346. Beside a col form the 8-byte reads of a row form conflict: 23 .. 32 % of the LDS
// cycles of dx, 40 % of dW from codes; products of two row forms or two col forms have no conflicts.
typedef __attribute__((address_space(3))) void* lds_ptr;
static constexpr int BIG = 256, STAGE = 32768, BIG_LDS = 4 * STAGE;

template <class T, bool COL, int PIECES /* of 1 KiB a wave sends for; a col form's tile has 4 */> struct BigOperand {
    static_assert(!COL || PIECES == 4, "256 own indices");
    typedef typename T::elem E;
    static constexpr int SZ = (int)sizeof(E), BK = 128 / SZ;
    const unsigned char* base;                  // element (i0, kbeg)
    int64_t bytes_left, step;                   // from base to the operand's end; advance of one k-tile
    uint32_t off, piece;                        // this lane's source offset of the wave's first piece; from one piece to the next
    int chunk;                                  // this lane's 16-byte chunk of a row, swizzled
    int krest;                                  // row form: contraction chunks left from base on
    __device__ __forceinline__ void init(const unsigned char* p, int64_t ld, int i0, int lim, int kbeg, int kend, int wave, int lane) {
        const int64_t ldb = ld * SZ;
        if constexpr (COL) {
            constexpr int RB = BIG * SZ, CPR = RB / 16, RPW = 4 * 64 / CPR;  // bytes and chunks of an LDS row, rows a wave sends for
            base = p + kbeg * ldb + (int64_t)i0 * SZ;
            bytes_left = (int64_t)(kend - kbeg - 1) * ldb + (int64_t)(lim - i0) * SZ;
            step = BK * ldb;
            const int r = wave * RPW + lane / CPR, c = lane % CPR;
            chunk = SZ == 2 ? c ^ ((r & 7) << 1) : c ^ (((r >> 2) & 3) << 2);
            off = (uint32_t)(r * ldb);
            piece = (uint32_t)(RPW / 4 * ldb);
            krest = 0;
        } else {
            base = p + i0 * ldb + (int64_t)kbeg * SZ;
            bytes_left = (int64_t)(lim - i0 - 1) * ldb + (int64_t)(kend - kbeg) * SZ;
            step = 128;
            chunk = (lane & 7) ^ (lane >> 4);
            off = (uint32_t)((wave * 8 * PIECES + (lane >> 3)) * ldb);
            piece = (uint32_t)(8 * ldb);
            krest = (kend - kbeg) * SZ / 16;
        }
    }
    // send for the next k-tile
    __device__ __forceinline__ void fetch(unsigned char* stage, int wave) {
        const int records = bytes_left < 0 ? 0 : bytes_left > 0x7fffffff ? 0x7fffffff : (int)bytes_left;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, records, 0x00020000);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            // 16-bit col form: piece i holds rows 2 i and 2 i + 1 of the wave's eight; row form: rows 8 i .. + 7
            const int c = COL ? (SZ == 2 ? chunk ^ (4 * i) : chunk) : chunk ^ (4 * ((wave * PIECES + i) & 1));
            const uint32_t first = !COL && c >= krest ? 0x80000000u : off;   // (what lies beyond the descriptor's reach arrives as zeros)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(stage + (wave * PIECES + i) * 1024), 16, (int)(first + i * piece + c * 16), 0, 0, 0);
        }
        base += step;
        bytes_left -= step;
        if constexpr (!COL) krest -= 8;
    }
};
// P in 8 bits (col form): a thread takes CPT consecutive codes of one contraction index (they share a power of two). They come by DMA into a place of the
// wave's own behind the stages -- held in registers across the matrix instructions they cost 49 spilled registers and twice the time (20 011 x 768 x 3 072 bf16:
// 222 us) -- and convert() leaves their values in the stage where a 16-bit operand's pieces would have to have landed.
template <class T> struct BigCodes {
    typedef typename T::elem E;
    static constexpr int SZ = (int)sizeof(E), BK = 128 / SZ, CPT = BK / 2, TPR = BIG / CPT, LDS = 512 * CPT;
    const uint8_t *codes, *scales;              // of contraction index kbeg, column i0
    int64_t ld, bytes_left, scales_left;
    uint32_t off;                               // this thread's codes and, / 32, its power of two
    uint32_t scale;
    static __device__ __forceinline__ int row() { return threadIdx.x / TPR; }
    static __device__ __forceinline__ int col() { return (int)(threadIdx.x % TPR) * CPT; }
    __device__ __forceinline__ void init(const GemmP& g, int i0, int kbeg, int kend) {
        ld = g.ldp;
        codes = g.codes + kbeg * ld + i0;
        scales = g.scales + kbeg * (ld / 32) + i0 / 32;
        bytes_left = (int64_t)(kend - kbeg - 1) * ld + (ld - i0);
        scales_left = (int64_t)(kend - kbeg - 1) * (ld / 32) + (ld - i0) / 32;
        off = (uint32_t)(row() * ld + col());
    }
    __device__ __forceinline__ void load(unsigned char* place) {             // place: the wave's
        const auto reach = [](int64_t n) { return n < 0 ? 0 : n > 0x7fffffff ? 0x7fffffff : (int)n; };
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)codes, 0, reach(bytes_left), 0x00020000);
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)scales, 0, reach(scales_left), 0x00020000);
        scale = __builtin_amdgcn_raw_buffer_load_b8(rc, (int)(off / 32), 0, 0);      // behind the end: 0, and its codes are 0
#pragma unroll
        for (int i = 0; i < CPT / 16; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(place + 1024 * i), 16, (int)(off + 16 * i), 0, 0, 0);
        codes += BK * ld;
        scales += BK * (ld / 32);
        bytes_left -= BK * ld;
        scales_left -= BK * (ld / 32);
    }
    __device__ __forceinline__ void convert(const unsigned char* place, unsigned char* stage) const {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const float s = as_f(scale << 23);
        const int r = row();
#pragma unroll
        for (int i = 0; i < CPT / 16; ++i) {
            const u4 x = *(const u4*)(place + 1024 * i + (threadIdx.x & 63) * 16);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int h = 0; h < SZ; ++h) {                                   // 16 codes: SZ chunks of 16 bytes
                const int c = (col() + 16 * i) * SZ / 16 + h, at = SZ == 2 ? c ^ ((r & 7) << 1) : c ^ (((r >> 2) & 3) << 2);
                u4 y;
                if constexpr (SZ == 2) y = (u4){values2<T, false>(w[2 * h], s), values2<T, true>(w[2 * h], s), values2<T, false>(w[2 * h + 1], s), values2<T, true>(w[2 * h + 1], s)};
                else {
                    float v[4];
                    values4(w[h], s, v);
                    y = (u4){as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])};
                }
                *(u4*)(stage + r * (BIG * SZ) + at * 16) = y;
            }
        }
    }
};
// this lane's LDS addresses of an operand's fragments and the reads; fragment f covers own indices i0 + 16 f .. + 15 (i0: the wave's, a multiple of 64)
template <class T, bool COL, bool BESIDE_COLS, int F> struct BigReader {
    static constexpr int SZ = (int)sizeof(typename T::elem);
    static constexpr int NA = COL ? F : BESIDE_COLS && SZ == 2 ? 4 : 2;
    const unsigned char* at[NA];
    __device__ __forceinline__ void init(const unsigned char* stage0, int i0, int lr, int lg) {
        if constexpr (COL && SZ == 2) {
            const int r = 4 * lg + (lr >> 2);
#pragma unroll
            for (int f = 0; f < F; ++f) at[f] = stage0 + r * 512 + (((i0 / 16 + f) ^ (r & 7)) * 32) + 8 * (lr & 3);
        } else if constexpr (COL) {
#pragma unroll
            for (int f = 0; f < F; ++f) at[f] = stage0 + 4 * lg * 1024 + (((i0 / 16 + f) ^ lg) * 64) + 4 * lr;
        } else if constexpr (BESIDE_COLS && SZ == 2) {                       // 8-byte pieces: indices 4 lg .. and 16 + 4 lg .. of each step
            const unsigned char* row = stage0 + (i0 + lr) * 128 + 8 * (lg & 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) at[j] = row + ((2 * j + (lg >> 1)) ^ (lr >> 1)) * 16;
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = stage0 + (i0 + lr) * 128 + ((4 * s + lg) ^ (lr >> 1)) * 16;
        }
    }
    template <int BUF> __device__ __forceinline__ void read(int s, u4 (&x)[F]) const {
#pragma unroll
        for (int f = 0; f < F; ++f) {
            if constexpr (COL && SZ == 2) {
                const unsigned char* p = at[f] + BUF * STAGE + s * 16384;
                const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)p));
                const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)(p + 8192)));
                x[f] = (u4){a.x, a.y, b.x, b.y};
            } else if constexpr (COL) {
                const float* p = (const float*)(at[f] + BUF * STAGE + s * 16384);
                x[f] = (u4){as_u(p[0]), as_u(p[256]), as_u(p[512]), as_u(p[768])};
            } else if constexpr (BESIDE_COLS && SZ == 2) {
                const uint2 a = *(const uint2*)(at[2 * s] + BUF * STAGE + f * 2048), b = *(const uint2*)(at[2 * s + 1] + BUF * STAGE + f * 2048);
                x[f] = (u4){a.x, a.y, b.x, b.y};
            } else x[f] = *(const u4*)(at[s] + BUF * STAGE + f * 2048);
        }
    }
};
#define PHASE_END() do { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); __builtin_amdgcn_sched_barrier(0); } while (0)

// what the epilogue of eight consecutive features of a token reads
template <class T> struct Ahead {
    u4 r[T::EPC == 8 ? 1 : 2];
    u2 k;
    __device__ __forceinline__ void load(const GemmP& g, int m, int n) {
        if (g.residual) {
            const typename T::elem* p = (const typename T::elem*)g.residual + m * g.ld_residual + n;
            r[0] = *(const u4*)p;
            if constexpr (T::EPC == 4) r[1] = *(const u4*)(p + 4);
        }
        if (g.keep) k = *(const u2*)(g.keep + (int64_t)m * g.n + n);
    }
};
// eight consecutive features n .. n + 7 of token m (both inside the result), aligned for vector access
template <class T> static __device__ __forceinline__ void epilogue8(const GemmP& g, int m, int n, float (&z)[8], const float (&bias)[8], const Ahead<T>& ahead) {
    typedef typename T::elem E;
    auto store8 = [](E* p, const float (&v)[8]) {
        if constexpr (sizeof(E) == 2) store_n<T, 8>(p, v);
        else { store_n<T, 4>(p, (const float(&)[4])v[0]); store_n<T, 4>(p + 4, (const float(&)[4])v[4]); }
    };
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] += bias[j];
    const int64_t at = (int64_t)m * g.n + n;
    if (g.save_codes) {                                                      // the group's 32 features are this lane's and three neighbours' (n is 8 times the lane in the row)
        const GroupPower e = group_power4<8>(z);
        uint32_t w[2];
        encode<8>(z, e, TopPower<F32>::E, w);
        const int64_t ld = (g.n + 31) / 32 * 32;
        *(uint2*)(g.save_codes + m * ld + n) = make_uint2(w[0], w[1]);
        if ((n & 31) == 0) g.save_scales[m * (ld / 32) + n / 32] = (uint8_t)(e.e + 127);
    }
    if (g.save_z) store8((E*)g.save_z + at, z);
    if (g.act)
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = gelu(z[j]);
    if (g.keep) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = ((j < 4 ? ahead.k.x : ahead.k.y) >> (8 * (j & 3))) & 0xffu ? z[j] * g.keep_scale : 0.f;
    }
    if (g.residual) {
        float t[8];
        unpack<T>(ahead.r[0], (float(&)[T::EPC])t[0]);
        if constexpr (T::EPC == 4) unpack<T>(ahead.r[1], (float(&)[T::EPC])t[4]);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] += t[j];
    }
    store8((E*)g.c + m * g.ldc + n, z);
}

template <class T> static __device__ __forceinline__ void load_bias8(const GemmP& g, int n, float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
    if (g.bias && n < g.n) {
        const typename T::elem* p = (const typename T::elem*)g.bias + n;
        unpack<T>(*(const u4*)p, (float(&)[T::EPC])b[0]);
        if constexpr (T::EPC == 4) unpack<T>(*(const u4*)(p + 4), (float(&)[T::EPC])b[4]);
    }
}

template <class T, bool PCOL, bool QCOL, bool CODES, int FB>
__global__ void __launch_bounds__(512) gemm_big_kernel(GemmP g) {
    constexpr int SZ = (int)sizeof(typename T::elem), BK = 128 / SZ, FA = 8;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // P0 | P1 | Q0 | Q1
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
    const bool second = wave >= 4;                                           // group B
    // unit -> (split, token tile, feature tile), feature tiles fastest; an XCD (workgroup id mod 8) takes consecutive units, which share operand tiles in its L2
    const int units = g.tiles_m * g.tiles_n * g.splits, per = (units + 7) / 8, u = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (u >= units || (int)(blockIdx.x >> 3) >= per) return;
    const int tn = u % g.tiles_n, tm = u / g.tiles_n % g.tiles_m, split = u / g.tiles_n / g.tiles_m;
    const int n0 = tn * BIG, m0 = tm * 64 * FB, kbeg = split * g.k_per_split, kend = g.k - kbeg < g.k_per_split ? g.k : kbeg + g.k_per_split;
    if (g.part) g.part += (int64_t)split * g.m * g.n;
    const int nk = (kend - kbeg + BK - 1) / BK;

    typename std::conditional<CODES, BigCodes<T>, BigOperand<T, PCOL, 4>>::type po;
    BigOperand<T, QCOL, FB> qo;
    if constexpr (CODES) po.init(g, n0, kbeg, kend); else po.init(g.p, g.ldp, n0, g.n, kbeg, kend, wave, lane);
    qo.init(g.q, g.ldq, m0, g.m, kbeg, kend, wave, lane);
    BigReader<T, PCOL, QCOL, FA> pr;
    BigReader<T, QCOL, PCOL, FB> qr;
    pr.init(smem, (wave >> 2) * 128, lr, lg);
    qr.init(smem + 2 * STAGE, (wave & 3) * 16 * FB, lr, lg);
    f4 acc[FA][FB];
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b) acc[a][b] = (f4){0.f, 0.f, 0.f, 0.f};

    auto fetch = [&](int buf) {
        if constexpr (CODES) po.load(smem + BIG_LDS + wave * (BigCodes<T>::LDS / 8)); else po.fetch(smem + buf * STAGE, wave);
        qo.fetch(smem + (2 + buf) * STAGE, wave);
    };
    fetch(0);
    if constexpr (CODES) po.convert(smem + BIG_LDS + wave * (BigCodes<T>::LDS / 8), smem);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    PHASE_END();
    if (second) {
        if (nk > 1) fetch(1);
        PHASE_END();
    }
    auto tile = [&](auto buf_, int kt) {
        constexpr int buf = decltype(buf_)::value;
        u4 fp0[FA], fq0[FB], fp1[FA], fq1[FB];
        if constexpr (CODES)
            if (second && kt + 1 < nk) { po.convert(smem + BIG_LDS + wave * (BigCodes<T>::LDS / 8), smem + (buf ^ 1) * STAGE); __builtin_amdgcn_sched_barrier(0); }
        pr.template read<buf>(0, fp0);
        qr.template read<buf>(0, fq0);
        pr.template read<buf>(1, fp1);
        qr.template read<buf>(1, fq1);
        if (!second) {
            if (kt + 1 < nk) { __builtin_amdgcn_sched_barrier(0); fetch(buf ^ 1); }
        } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        PHASE_END();
        if (second && kt + 2 < nk) fetch(buf);
        __builtin_amdgcn_sched_barrier(0);
        mma_block<T, FA, FB>(fp0, fq0, acc);
        mma_block<T, FA, FB>(fp1, fq1, acc);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (CODES)
            if (!second && kt + 1 < nk) po.convert(smem + BIG_LDS + wave * (BigCodes<T>::LDS / 8), smem + (buf ^ 1) * STAGE);
        if (!second) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        PHASE_END();
    };
    for (int kt = 0; kt < nk; kt += 2) {
        tile(std::integral_constant<int, 0>{}, kt);
        if (kt + 1 < nk) tile(std::integral_constant<int, 1>{}, kt + 1);
    }
    if (!second) PHASE_END();                                                // group A matches B's extra barrier: every fragment has been read

    // the result through LDS, 16 tokens x 128 features of a wave at a time in its own 8.25 KiB: lanes leave four consecutive features of 16 tokens and take
    // eight consecutive features of a token, so that stores (and the epilogue's loads) are whole rows of 256 bytes
    constexpr int PITCH = 128 * 4 + 16;
    unsigned char* mine = smem + wave * 16 * PITCH;
    const int nw = n0 + (wave >> 2) * 128, mw = m0 + (wave & 3) * 16 * FB, nl = nw + 8 * (lane & 15);
    float bias[8];
    load_bias8<T>(g, nl, bias);
    Ahead<T> ahead[2][4];                                                    // 16 tokens' residual and dropout are read while the 16 before them are written
    auto fetch_ahead = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = mw + 16 * b + 4 * i + (lane >> 4);
            if (m < g.m && nl < g.n) ahead[b & 1][i].load(g, m, nl);
        }
    };
    fetch_ahead(0);
#pragma unroll
    for (int b = 0; b < FB; ++b) {
        if (b + 1 < FB) fetch_ahead(b + 1);
#pragma unroll
        for (int a = 0; a < FA; ++a) *(f4*)(mine + lr * PITCH + (16 * a + 4 * lg) * 4) = acc[a][b];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 4 * i + (lane >> 4), m = mw + 16 * b + t;
            const float* row = (const float*)(mine + t * PITCH) + 8 * (lane & 15);
            const f4 x = *(const f4*)row, y = *(const f4*)(row + 4);
            float z[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            if (m < g.m && nl < g.n) {
                if (g.part) {
                    float* to = g.part + (int64_t)m * g.n + nl;
                    *(f4*)to = x;
                    *(f4*)(to + 4) = y;
                } else epilogue8<T>(g, m, nl, z, bias, ahead[b & 1][i]);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// ---- a split product's parts, summed in their order, and its epilogue ----
// VEC: eight features a thread (aligned rows; with codes to save, whole groups of 32), otherwise one
template <class T, bool VEC> __global__ void __launch_bounds__(256) gemm_join_kernel(GemmP g) {
    typedef typename T::elem E;
    constexpr int NV = VEC ? 8 : 1;
    const int per_row = g.n / NV;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, plane = (int64_t)g.m * g.n;
    if (i >= (int64_t)g.m * per_row) return;
    const int m = (int)(i / per_row), n = (int)(i - (int64_t)m * per_row) * NV;
    const float* from = g.part + (int64_t)m * g.n + n;
    float z[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) z[j] = 0.f;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
        if constexpr (VEC) {
            const f4 x = *(const f4*)(from + s * plane), y = *(const f4*)(from + s * plane + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { z[j] += x[j]; z[4 + j] += y[j]; }
        } else z[0] += from[s * plane];
    }
    if constexpr (VEC) {
        float bias[8];
        Ahead<T> ahead;
        load_bias8<T>(g, n, bias);
        ahead.load(g, m, n);
        epilogue8<T>(g, m, n, z, bias, ahead);
    }
    else {
        if (g.bias) z[0] += T::ld(((const E*)g.bias)[n]);
        const int64_t at = (int64_t)m * g.n + n;
        if (g.save_z) ((E*)g.save_z)[at] = T::st(z[0]);
        float y = g.act ? gelu(z[0]) : z[0];
        if (g.keep) y = g.keep[at] ? y * g.keep_scale : 0.f;
        if (g.residual) y += T::ld(((const E*)g.residual)[m * g.ld_residual + n]);
        ((E*)g.c)[m * g.ldc + n] = T::st(y);
    }
}

// ---- launches ----
struct GemmPlan { bool big; int tile, splits, k_per_split, tiles_m, tiles_n; };
// rows that can be written (and their epilogue's operands read) eight features at a time
template <class T> static bool rows_of_eight(const GemmP& g) {
    return (((uintptr_t)g.c | (uintptr_t)g.save_z | (uintptr_t)g.residual | (uintptr_t)g.bias) & 15) == 0 && ((uintptr_t)g.keep & 7) == 0 && g.n % 8 == 0 &&
           (g.ldc | g.ld_residual) % T::EPC == 0 && (!g.save_codes || g.n % 32 == 0);
}
// the big kernel takes 16-byte aligned rows of whole 16-byte chunks whose tiles stay within a descriptor's 2^31 bytes
template <class T> static bool big_fits(const GemmP& g, bool pcol, bool qcol) {
    constexpr int EPC = T::EPC;
    const bool operands = (((g.codes ? (uintptr_t)g.codes : (uintptr_t)g.p) | (uintptr_t)g.q) & 15) == 0 && (g.ldp | g.ldq) % EPC == 0;
    const bool contraction = (pcol && qcol) || g.k % EPC == 0, own = !qcol || g.m % EPC == 0;
    const bool reach = g.ldp >= (pcol ? g.n : g.k) && g.ldq >= (qcol ? g.m : g.k) && g.ldp < (1 << 21) && g.ldq < (1 << 21);
    return rows_of_eight<T>(g) && operands && contraction && own && reach;
}
// The kernel and the split of the contraction are those with the least estimated time: the workgroups that fall to the fullest CU, each so many k-tiles, and
// a join that writes and reads every part. Microseconds measured on the training sizes: `busy` of CU time per k-tile, `alone` where a workgroup has the CU
// to itself and only waits, `start` per tile. (13 848 x 3072 by 768 fp16: 219 tiles of 192 x 256, 78 us; 4001 x 1945 x 3001 fp32's weight gradient, 384 tiles
// of 128: unsplit 796 us, in two parts 533 and their join 18.)
struct GemmCost { double busy, alone, start; };
template <class T> GemmPlan gemm_plan(const GemmP& g, bool pcol, bool qcol) {
    constexpr bool WIDE = sizeof(typename T::elem) == 4;
    const GemmCost costs[4] = {{WIDE ? 10.0 : 1.9, WIDE ? 10.0 : 1.9, 6.0}, {WIDE ? 8.0 : 1.58, WIDE ? 8.0 : 1.58, 5.0}, {WIDE ? 2.8 : 1.8, 2.8, 3.0}, {WIDE ? 0.75 : 0.55, 1.2, 2.5}};
    const int tokens_of[4] = {256, 192, 128, 64}, features_of[4] = {256, 256, 128, 64};
    const bool big = big_fits<T>(g, pcol, qcol), join = rows_of_eight<T>(g) || !g.save_codes;     // (a join eight features at a time, or without groups of codes)
    const double part_us = (double)g.m * g.n * 8 / 4.5e6;
    GemmPlan best = {};
    double least = 0;
    for (int v = big ? 0 : 2; v < 4; ++v) {
        if (v == 1 && qcol) continue;
        const int tile = tokens_of[v], wide = features_of[v], bk = v < 2 ? 128 / (int)sizeof(typename T::elem) : 2 * T::KS;
        const int64_t tm = ((int64_t)g.m + tile - 1) / tile, tn = ((int64_t)g.n + wide - 1) / wide, tiles = tm * tn, kt = ((int64_t)g.k + bk - 1) / bk;
        for (int s : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
            if ((s > 1 && (!join || s > kt)) || tiles * s >= (1LL << 32) / (v < 2 ? 512 : 256)) break;       // (a launch takes less than 2^32 threads)
            const int64_t per = kt > 0 ? (kt + s - 1) / s : 0, rounds = (tiles * s + 255) / 256;
            double us = (double)rounds * (per * costs[v].busy + (v < 2 ? costs[v].start : 0));
            const double wait = per * costs[v].alone + costs[v].start;
            if (us < wait) us = wait;
            if (s > 1) us += 4.0 + s * part_us;
            if (best.tile && us >= least) continue;
            least = us;
            best.big = v < 2; best.tile = tile; best.tiles_m = (int)tm; best.tiles_n = (int)tn;
            best.k_per_split = (int)((per > 0 ? per : 1) * bk);
            best.splits = (int)(((int64_t)g.k + best.k_per_split - 1) / best.k_per_split);
            if (best.splits < 1) best.splits = 1;
        }
    }
    return best;
}

template <class T, bool PCOL, bool QCOL, bool CODES> static int gemm_launch(const GemmP& g, const GemmPlan& pl, hipStream_t stream) {
    if (pl.big) {
        auto kernel = gemm_big_kernel<T, PCOL, QCOL, CODES, 4>;
        if constexpr (!QCOL)
            if (pl.tile == 192) kernel = gemm_big_kernel<T, PCOL, QCOL, CODES, 3>;
        const int lds = BIG_LDS + (CODES ? BigCodes<T>::LDS : 0);
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return (int)e;
        const int64_t units = (int64_t)pl.tiles_m * pl.tiles_n * pl.splits;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((units + 7) / 8 * 8)), dim3(512), lds, stream, g);
    } else {
        const dim3 grid((unsigned)(pl.tiles_m * pl.tiles_n), (unsigned)pl.splits);
        if (pl.tile == 128) hipLaunchKernelGGL((gemm_any_kernel<T, PCOL, QCOL, CODES, 128>), grid, dim3(256), 0, stream, g);
        else hipLaunchKernelGGL((gemm_any_kernel<T, PCOL, QCOL, CODES, 64>), grid, dim3(256), 0, stream, g);
    }
    int rc = (int)hipGetLastError();
    if (rc || pl.splits == 1) return rc;
    const bool vec = rows_of_eight<T>(g);
    const int64_t threads = (int64_t)g.m * (vec ? g.n / 8 : g.n);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (vec) hipLaunchKernelGGL((gemm_join_kernel<T, true>), grid, dim3(256), 0, stream, g);
    else hipLaunchKernelGGL((gemm_join_kernel<T, false>), grid, dim3(256), 0, stream, g);
    return (int)hipGetLastError();
}
template <class T> int gemm_t(GemmP g, bool pcol, bool qcol, hipStream_t stream) {
    const GemmPlan pl = gemm_plan<T>(g, pcol, qcol);
    if (!pl.tile) return ATLAS_TRAIN_E_UNSUPPORTED;                          // more tiles than a launch takes
    g.splits = pl.splits; g.k_per_split = pl.k_per_split; g.tiles_m = pl.tiles_m; g.tiles_n = pl.tiles_n;
    if (pl.splits == 1) g.part = nullptr;
    if (pcol && qcol) return g.codes ? gemm_launch<T, true, true, true>(g, pl, stream) : gemm_launch<T, true, true, false>(g, pl, stream);
    if (pcol) return gemm_launch<T, true, false, false>(g, pl, stream);
    if (qcol) return ATLAS_TRAIN_E_UNSUPPORTED;
    return gemm_launch<T, false, false, false>(g, pl, stream);
}
template <class T> int gemm_splits(const GemmP& g, bool pcol, bool qcol) { return gemm_plan<T>(g, pcol, qcol).splits; }

}  // namespace atlas_train
