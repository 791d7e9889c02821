// attention.h -- attention over packed sequences, forward and backward, for one element type (attention_{f16,bf16,f32}.hip).
//
//   forward   S = scale q k^T; O = softmax(S) v in one pass over the keys with the running maximum and sum of the softmax; what is kept
//             for the backward pass is one float per row, lse = log2 sum 2^(S log2 e)
//   backward  P = 2^(S log2 e - lse) is recomputed. With M = keep * keep_scale and delta = rowsum(dO . O):
//             dS = P . (M . (dO v^T) - delta);  dq = scale dS k;  dk = scale dS^T q;  dv = (M . P)^T dO
//             dq_kernel owns query rows and walks the keys (and leaves delta); dkv_kernel owns keys and walks the query rows of every
//             query head that shares them. Each recomputes S and dO v^T (7 products instead of 5) and neither needs an atomic: the same
//             bits from call to call.
// All three are the same loop: a wave OWNS 16 * F rows whose vectors sit in registers as B fragments; tiles of 64 WALKED rows pass through
// LDS; the products with the walked rows as the A operand leave, in each lane, four consecutive walked rows of one owned row -- which is the
// B fragment layout of the second product, whose A operand is read out of the same row-major tile through the transposing LDS read. So scores
// and probabilities never leave their lane, and the statistics of an owned row are scalars of its lane.
#pragma once
#include "elements.h"

namespace atlas_train {

struct AttnP {
    const unsigned char *q, *k, *v, *dout;
    const unsigned char* out_in;                        // backward: the forward's output
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;      // in bytes
    const int32_t *q_offsets, *k_offsets;
    int64_t total_q, total_k;
    int batch, heads, kv_heads, dim, keep_cols;
    const uint8_t *key_mask, *keep;
    int64_t keep_row, keep_head;
    float scale, keep_scale;
    unsigned char *out, *dq, *dk, *dv;                  // out: forward only
    float *lse, *delta;
    int tiles;                                          // tiles of the longest sequence (launch size)
    int blocks;                                         // blocks that compute; those behind them clear the rows of no sequence
};

static constexpr int WALK = 64;                         // walked rows of one tile

template <class T, int DP> struct Geo {
    typedef typename T::elem E;
    static constexpr int SZ = (int)sizeof(E), CPR = DP * SZ / 16, RPP = 256 / CPR, NP = WALK / RPP, NKS = DP / T::KS, ND = DP / 16;
    // pitch of a tile's rows: 16 bytes more than the row (row reads of 16 lanes cover the banks)
    static constexpr int PITCH = DP * SZ + 16;
};

struct Seq { int64_t begin; int len; };
static __device__ __forceinline__ Seq sequence(const int32_t* offsets, int b, int64_t total) {
    int64_t lo = offsets[b], hi = offsets[b + 1];
    lo = lo < 0 ? 0 : lo > total ? total : lo;
    hi = hi < lo ? lo : hi > total ? total : hi;
    Seq s; s.begin = lo; s.len = (int)(hi - lo);
    return s;
}

// item -> (tile, head, sequence): consecutive items run on one XCD (workgroup g runs on XCD g mod 8), so the tiles of a head, which read the same
// walked rows, share an L2
struct Item { int tile, head, b; };
static __device__ __forceinline__ Item item_of(int bid, int blocks, int tiles, int heads) {
    const int per = blocks / 8;                         // blocks is a multiple of 8
    int i = (bid & 7) * per + (bid >> 3);
    Item t;
    t.tile = i % tiles; i /= tiles;
    t.head = i % heads;
    t.b = i / heads;
    return t;
}

// rows that belong to no sequence (in front of the first, behind the last) get zeros
static __device__ __forceinline__ void clear_gaps(unsigned char* out, int64_t row_bytes, const int32_t* offsets, int batch, int64_t total, int part, int parts) {
    int64_t first = offsets[0], last = offsets[batch];
    first = first < 0 ? 0 : first > total ? total : first;
    last = last < first ? first : last > total ? total : last;
    const int64_t n16 = row_bytes / 16, head = first * n16, all = head + (total - last) * n16;
    for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < all; i += (int64_t)parts * 256) {
        const int64_t at = i < head ? i : last * n16 + (i - head);
        *(u4*)(out + at * 16) = (u4){0, 0, 0, 0};
    }
}

// one walked tile (rows row0 .. row0 + 63 of a sequence of `len`) between global memory and LDS, through registers
template <class T, int DP> struct Tile {
    typedef Geo<T, DP> G;
    u4 x[G::NP];
    __device__ __forceinline__ void load(const unsigned char* base, int64_t row_bytes, int row0, int len, int dim) {
        const int c = (threadIdx.x % G::CPR), r = threadIdx.x / G::CPR;
#pragma unroll
        for (int i = 0; i < G::NP; ++i) {
            const int row = row0 + i * G::RPP + r;
            x[i] = (u4){0, 0, 0, 0};
            if (row < len && c * T::EPC < dim) x[i] = *(const u4*)(base + row * row_bytes + c * 16);
        }
    }
    // rows whose `live` entry is 0 are stored as zeros
    __device__ __forceinline__ void store(unsigned char* tile, const float* live) const {
        const int c = (threadIdx.x % G::CPR), r = threadIdx.x / G::CPR;
#pragma unroll
        for (int i = 0; i < G::NP; ++i) {
            const int row = i * G::RPP + r;
            const bool on = live == nullptr || live[row] != 0.f;
            *(u4*)(tile + row * G::PITCH + c * 16) = on ? x[i] : (u4){0, 0, 0, 0};
        }
    }
};

// the owned rows' vectors as B fragments, straight from global memory (zeros behind the end)
template <class T, int DP, int F> static __device__ __forceinline__ void load_owned(const unsigned char* base, int64_t row_bytes, int row0, int len, int dim,
                                                                                    int lr, int lg, u4 (&x)[F][Geo<T, DP>::NKS]) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int row = row0 + 16 * f + lr;
#pragma unroll
        for (int s = 0; s < Geo<T, DP>::NKS; ++s) {
            x[f][s] = (u4){0, 0, 0, 0};
            const int e = s * T::KS + lg * T::EPC;
            if (row < len && e < dim) x[f][s] = *(const u4*)(base + row * row_bytes + e * (int)sizeof(typename T::elem));
        }
    }
}

// t[a][f] = (walked rows 16 a .. + 15) x (owned rows of fragment f), contraction over the vectors' dimension
template <class T, int DP, int F, int A = WALK / 16>
static __device__ __forceinline__ void scores(const unsigned char* tile, const u4 (&own)[F][Geo<T, DP>::NKS], int lr, int lg, f4 (&t)[A][F], int a0 = 0) {
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
        for (int f = 0; f < F; ++f) t[a][f] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < Geo<T, DP>::NKS; ++s)
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const u4 w = *(const u4*)(tile + (16 * (a0 + a) + lr) * Geo<T, DP>::PITCH + (s * 4 + lg) * 16);
#pragma unroll
            for (int f = 0; f < F; ++f) t[a][f] = T::mma(w, own[f][s], t[a][f]);
        }
}
// acc[d][f] += (walked columns: dimension 16 d + ..) x t, contraction over the walked rows
template <class T, int DP, int F, int A = WALK / 16>
static __device__ __forceinline__ void gather(const unsigned char* tile, const f4 (&t)[A][F], int lr, int lg, f4 (&acc)[Geo<T, DP>::ND][F], int a0 = 0) {
    constexpr int S = T::TILES;
#pragma unroll
    for (int j = 0; j < A / S; ++j) {
        u4 p[F];
#pragma unroll
        for (int f = 0; f < F; ++f) p[f] = pack_chunk<T>(t[S * j][f], t[S * j + S - 1][f]);
#pragma unroll
        for (int d = 0; d < Geo<T, DP>::ND; ++d) {
            const u4 w = read_cols<T>(tile, Geo<T, DP>::PITCH, 16 * (a0 + S * j), 16 * d, lr, lg);
#pragma unroll
            for (int f = 0; f < F; ++f) acc[d][f] = T::mma(w, p[f], acc[d][f]);
        }
    }
}
// four consecutive dropout decisions of one query row, keys j .. j + 3 (bit i: keep key j + i); columns from `cols` on count as dropped
static __device__ __forceinline__ uint32_t keep4(const uint8_t* row, int j, int cols) {
    typedef uint32_t __attribute__((aligned(1))) u32_a1;
    if (j + 4 <= cols) {
        const uint32_t w = *(const u32_a1*)(row + j);
        return (w & 0xffu ? 1u : 0u) | (w & 0xff00u ? 2u : 0u) | (w & 0xff0000u ? 4u : 0u) | (w & 0xff000000u ? 8u : 0u);
    }
    uint32_t m = 0;
    for (int i = 0; i < 4; ++i)
        if (j + i < cols && row[j + i]) m |= 1u << i;
    return m;
}
template <class T, int DP, int F> static __device__ __forceinline__ void store_owned(unsigned char* base, int64_t row_bytes, int row0, int len, int dim, int lr, int lg,
                                                                                     const f4 (&acc)[Geo<T, DP>::ND][F], const float (&mul)[F]) {
    typedef typename T::elem E;
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int row = row0 + 16 * f + lr;
        if (row >= len) continue;
#pragma unroll
        for (int d = 0; d < Geo<T, DP>::ND; ++d) {
            const int e = 16 * d + 4 * lg;
            if (e >= dim) continue;
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = mul[f] == 0.f ? 0.f : acc[d][f][r] * mul[f];     // a row without keys is zeros, whatever was summed
            store_n<T, 4>((E*)(base + row * row_bytes) + e, o);
        }
    }
}

// ---- forward: owned = query rows, walked = keys ----
template <class T, int DP, int F, bool KEEP>
__global__ void __launch_bounds__(256) attention_forward_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.out, (int64_t)p.heads * p.dim * G::SZ, p.q_offsets, p.batch, p.total_q, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned char *sk = smem, *sv = smem + WALK * G::PITCH;
    float* live = (float*)(smem + 2 * WALK * G::PITCH);                      // 1: the key is visible
    const Item it = item_of(blockIdx.x, p.blocks, p.tiles, p.heads);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int kvh = it.head / (p.heads / p.kv_heads);
    const unsigned char* kb = p.k + ks.begin * p.k_row + kvh * p.k_head;
    const unsigned char* vb = p.v + ks.begin * p.v_row + kvh * p.v_head;
    const unsigned char* qb = p.q + sq.begin * p.q_row + it.head * p.q_head;
    const float c = p.scale * 1.4426950408889634f;                           // exponents in base 2
    for (int tile = it.tile; tile * 64 * F < sq.len; tile += p.tiles) {
        const int row0 = tile * 64 * F + wave * 16 * F;
        u4 own[F][G::NKS];
        load_owned<T, DP, F>(qb, p.q_row, row0, sq.len, p.dim, lr, lg, own);
        f4 acc[G::ND][F];
        float m[F], l[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            m[f] = -__builtin_inff(); l[f] = 0.f;
#pragma unroll
            for (int d = 0; d < G::ND; ++d) acc[d][f] = (f4){0.f, 0.f, 0.f, 0.f};
        }
        Tile<T, DP> tk, tv;
        float alive = 0.f;
        auto fetch = [&](int k0) {
            tk.load(kb, p.k_row, k0, ks.len, p.dim);
            tv.load(vb, p.v_row, k0, ks.len, p.dim);
            if (threadIdx.x < WALK) {
                const int key = k0 + threadIdx.x;
                alive = key < ks.len && (p.key_mask == nullptr || p.key_mask[ks.begin + key]) ? 1.f : 0.f;
            }
        };
        if (ks.len > 0) fetch(0);
        for (int k0 = 0; k0 < ks.len; k0 += WALK) {
            __syncthreads();                                                 // the tile before has been read
            if (threadIdx.x < WALK) live[threadIdx.x] = alive;
            if (p.key_mask) __syncthreads();
            tk.store(sk, p.key_mask ? live : nullptr);
            tv.store(sv, p.key_mask ? live : nullptr);
            __syncthreads();
            if (k0 + WALK < ks.len) fetch(k0 + WALK);
            f4 t[WALK / 16][F];
            scores<T, DP, F>(sk, own, lr, lg, t);
            if (p.key_mask != nullptr || k0 + WALK > ks.len) {
#pragma unroll
                for (int a = 0; a < WALK / 16; ++a) {
                    const f4 on = *(const f4*)(live + 16 * a + 4 * lg);
#pragma unroll
                    for (int f = 0; f < F; ++f)
#pragma unroll
                        for (int r = 0; r < 4; ++r) t[a][f][r] = on[r] != 0.f ? t[a][f][r] : -__builtin_inff();
                }
            }
#pragma unroll
            for (int f = 0; f < F; ++f) {
                float top = t[0][f][0];
#pragma unroll
                for (int a = 0; a < WALK / 16; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, t[a][f][r]);
                top = fmaxf(m[f], groups_max(top));
                if (__any(top > m[f])) {                                     // the running maximum moved for some row of this wave
                    const float base = top == -__builtin_inff() ? 0.f : top;
                    const float keep = exp2_fast((m[f] - base) * c);
                    l[f] *= keep;
#pragma unroll
                    for (int d = 0; d < G::ND; ++d) acc[d][f] *= keep;
                    m[f] = top;
                }
                const float off = m[f] == -__builtin_inff() ? 0.f : -m[f] * c;
#pragma unroll
                for (int a = 0; a < WALK / 16; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = exp2_fast(__builtin_fmaf(t[a][f][r], c, off));
                        t[a][f][r] = e;
                        l[f] += e;
                    }
                if constexpr (KEEP) {
                    const int row = row0 + 16 * f + lr;
                    if (row < sq.len) {
                        const uint8_t* kr = p.keep + (sq.begin + row) * p.keep_row + it.head * p.keep_head;
#pragma unroll
                        for (int a = 0; a < WALK / 16; ++a) {
                            const uint32_t bits = keep4(kr, k0 + 16 * a + 4 * lg, ks.len < p.keep_cols ? ks.len : p.keep_cols);
#pragma unroll
                            for (int r = 0; r < 4; ++r) t[a][f][r] = bits >> r & 1 ? t[a][f][r] : 0.f;
                        }
                    }
                }
            }
            gather<T, DP, F>(sv, t, lr, lg, acc);
        }
        float mul[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const float sum = groups_sum(l[f]);
            mul[f] = sum == 0.f ? 0.f : (KEEP ? p.keep_scale : 1.f) / sum;   // (scores that are NaN leave a NaN sum: no empty row)
            const int row = row0 + 16 * f + lr;
            if (lg == 0 && row < sq.len)
                p.lse[(int64_t)it.head * p.total_q + sq.begin + row] = sum == 0.f ? __builtin_inff() : __builtin_fmaf(m[f], c, log2f(sum));
        }
        const int64_t rb = (int64_t)p.heads * p.dim * G::SZ;
        store_owned<T, DP, F>(p.out + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lr, lg, acc, mul);
    }
}

// ---- backward, dq: owned = query rows, walked = keys; leaves delta for dkv_kernel ----
template <class T, int DP, int F, bool KEEP>
__global__ void __launch_bounds__(256) attention_dq_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.dq, (int64_t)p.heads * p.dim * G::SZ, p.q_offsets, p.batch, p.total_q, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned char *sk = smem, *sv = smem + WALK * G::PITCH;
    float* live = (float*)(smem + 2 * WALK * G::PITCH);
    const Item it = item_of(blockIdx.x, p.blocks, p.tiles, p.heads);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int kvh = it.head / (p.heads / p.kv_heads);
    const unsigned char* kb = p.k + ks.begin * p.k_row + kvh * p.k_head;
    const unsigned char* vb = p.v + ks.begin * p.v_row + kvh * p.v_head;
    const int64_t rb = (int64_t)p.heads * p.dim * G::SZ;
    const float c = p.scale * 1.4426950408889634f;
    for (int tile = it.tile; tile * 64 * F < sq.len; tile += p.tiles) {
        const int row0 = tile * 64 * F + wave * 16 * F;
        u4 own[F][G::NKS], dof[F][G::NKS];
        load_owned<T, DP, F>(p.q + sq.begin * p.q_row + it.head * p.q_head, p.q_row, row0, sq.len, p.dim, lr, lg, own);
        load_owned<T, DP, F>(p.dout + sq.begin * p.do_row + it.head * p.do_head, p.do_row, row0, sq.len, p.dim, lr, lg, dof);
        float lse[F], delta[F];
        {
            u4 of[F][G::NKS];
            load_owned<T, DP, F>(p.out_in + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lr, lg, of);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int row = row0 + 16 * f + lr;
                const int64_t at = (int64_t)it.head * p.total_q + sq.begin + row;
                lse[f] = row < sq.len ? p.lse[at] : __builtin_inff();
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < G::NKS; ++i) {
                    const uint32_t a[4] = {of[f][i].x, of[f][i].y, of[f][i].z, of[f][i].w}, b[4] = {dof[f][i].x, dof[f][i].y, dof[f][i].z, dof[f][i].w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (G::SZ == 4) s = __builtin_fmaf(as_f(a[w]), as_f(b[w]), s);
                        else {
                            s = __builtin_fmaf(T::ld((uint16_t)(a[w] & 0xffff)), T::ld((uint16_t)(b[w] & 0xffff)), s);
                            s = __builtin_fmaf(T::ld((uint16_t)(a[w] >> 16)), T::ld((uint16_t)(b[w] >> 16)), s);
                        }
                    }
                }
                s = groups_sum(s);
                const bool empty = lse[f] == __builtin_inff();               // nothing visible: q and dout of the row are not used
                delta[f] = empty ? 0.f : s;
                if (lg == 0 && row < sq.len) p.delta[at] = delta[f];
#pragma unroll
                for (int i = 0; i < G::NKS; ++i)
                    if (empty) { own[f][i] = (u4){0, 0, 0, 0}; dof[f][i] = (u4){0, 0, 0, 0}; }
            }
        }
        f4 acc[G::ND][F];
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int d = 0; d < G::ND; ++d) acc[d][f] = (f4){0.f, 0.f, 0.f, 0.f};
        Tile<T, DP> tk, tv;
        float alive = 0.f;
        auto fetch = [&](int k0) {
            tk.load(kb, p.k_row, k0, ks.len, p.dim);
            tv.load(vb, p.v_row, k0, ks.len, p.dim);
            if (threadIdx.x < WALK) {
                const int key = k0 + threadIdx.x;
                alive = key < ks.len && (p.key_mask == nullptr || p.key_mask[ks.begin + key]) ? 1.f : 0.f;
            }
        };
        if (ks.len > 0) fetch(0);
        for (int k0 = 0; k0 < ks.len; k0 += WALK) {
            __syncthreads();
            if (threadIdx.x < WALK) live[threadIdx.x] = alive;
            if (p.key_mask) __syncthreads();
            tk.store(sk, p.key_mask ? live : nullptr);
            tv.store(sv, p.key_mask ? live : nullptr);
            __syncthreads();
            if (k0 + WALK < ks.len) fetch(k0 + WALK);
            f4 t[WALK / 16][F], g[WALK / 16][F];
            scores<T, DP, F>(sk, own, lr, lg, t);
            scores<T, DP, F>(sv, dof, lr, lg, g);
            const bool ragged = p.key_mask != nullptr || k0 + WALK > ks.len;
#pragma unroll
            for (int a = 0; a < WALK / 16; ++a) {
                f4 on = {1.f, 1.f, 1.f, 1.f};
                if (ragged) on = *(const f4*)(live + 16 * a + 4 * lg);
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    uint32_t bits = 15;
                    if constexpr (KEEP) {
                        const int row = row0 + 16 * f + lr;
                        if (row < sq.len)
                            bits = keep4(p.keep + (sq.begin + row) * p.keep_row + it.head * p.keep_head, k0 + 16 * a + 4 * lg, ks.len < p.keep_cols ? ks.len : p.keep_cols);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = on[r] != 0.f ? exp2_fast(__builtin_fmaf(t[a][f][r], c, -lse[f])) : 0.f;
                        const float dp = KEEP ? (bits >> r & 1 ? g[a][f][r] * p.keep_scale : 0.f) : g[a][f][r];
                        t[a][f][r] = e * (dp - delta[f]);
                    }
                }
            }
            gather<T, DP, F>(sk, t, lr, lg, acc);
        }
        float mul[F];
#pragma unroll
        for (int f = 0; f < F; ++f) mul[f] = lse[f] == __builtin_inff() ? 0.f : p.scale;
        store_owned<T, DP, F>(p.dq + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lr, lg, acc, mul);
    }
}

// ---- backward, dk and dv: owned = keys, walked = the query rows of every query head that reads them ----
template <class T, int DP, int F, bool KEEP>
__global__ void __launch_bounds__(256) attention_dkv_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    const int64_t rb = (int64_t)p.kv_heads * p.dim * G::SZ;
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.dk, rb, p.k_offsets, p.batch, p.total_k, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        clear_gaps(p.dv, rb, p.k_offsets, p.batch, p.total_k, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned char *sq_t = smem, *sd_t = smem + WALK * G::PITCH;
    float* s_live = (float*)(smem + 2 * WALK * G::PITCH);                    // 1: the row has visible keys | lse | delta
    float *s_lse = s_live + WALK, *s_delta = s_lse + WALK;
    const Item it = item_of(blockIdx.x, p.blocks, p.tiles, p.kv_heads);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int group = p.heads / p.kv_heads;
    const float c = p.scale * 1.4426950408889634f;
    for (int tile = it.tile; tile * 64 * F < ks.len; tile += p.tiles) {
        const int row0 = tile * 64 * F + wave * 16 * F;
        u4 kf[F][G::NKS], vf[F][G::NKS];
        load_owned<T, DP, F>(p.k + ks.begin * p.k_row + it.head * p.k_head, p.k_row, row0, ks.len, p.dim, lr, lg, kf);
        load_owned<T, DP, F>(p.v + ks.begin * p.v_row + it.head * p.v_head, p.v_row, row0, ks.len, p.dim, lr, lg, vf);
        float vis[F];
        f4 dk[G::ND][F], dv[G::ND][F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int row = row0 + 16 * f + lr;
            vis[f] = row < ks.len && (p.key_mask == nullptr || p.key_mask[ks.begin + row]) ? 1.f : 0.f;
#pragma unroll
            for (int i = 0; i < G::NKS; ++i)
                if (vis[f] == 0.f) { kf[f][i] = (u4){0, 0, 0, 0}; vf[f][i] = (u4){0, 0, 0, 0}; }
#pragma unroll
            for (int d = 0; d < G::ND; ++d) { dk[d][f] = (f4){0.f, 0.f, 0.f, 0.f}; dv[d][f] = (f4){0.f, 0.f, 0.f, 0.f}; }
        }
        const int steps = (sq.len + WALK - 1) / WALK;                        // walked tiles of one query head
        Tile<T, DP> tq, td;
        float r_live = 0.f, r_lse = 0.f, r_delta = 0.f;
        auto fetch = [&](int i) {
            const int head = it.head * group + i / steps, q0 = (i % steps) * WALK;
            tq.load(p.q + sq.begin * p.q_row + head * p.q_head, p.q_row, q0, sq.len, p.dim);
            td.load(p.dout + sq.begin * p.do_row + head * p.do_head, p.do_row, q0, sq.len, p.dim);
            if (threadIdx.x < WALK) {
                const int row = q0 + threadIdx.x;
                const int64_t at = (int64_t)head * p.total_q + sq.begin + row;
                r_lse = row < sq.len ? p.lse[at] : __builtin_inff();
                r_delta = row < sq.len ? p.delta[at] : 0.f;
                r_live = r_lse == __builtin_inff() ? 0.f : 1.f;
            }
        };
        if (sq.len > 0) fetch(0);
        for (int i = 0; i < steps * group; ++i) {
            __syncthreads();
            if (threadIdx.x < WALK) { s_live[threadIdx.x] = r_live; s_lse[threadIdx.x] = r_lse; s_delta[threadIdx.x] = r_delta; }
            __syncthreads();
            tq.store(sq_t, s_live);
            td.store(sd_t, s_live);
            __syncthreads();
            if (i + 1 < steps * group) fetch(i + 1);
            const int head = it.head * group + i / steps, q0 = (i % steps) * WALK;
            f4 t[WALK / 16][F], g[WALK / 16][F];
            scores<T, DP, F>(sq_t, kf, lr, lg, t);
            scores<T, DP, F>(sd_t, vf, lr, lg, g);
#pragma unroll
            for (int a = 0; a < WALK / 16; ++a) {
                const f4 lse = *(const f4*)(s_lse + 16 * a + 4 * lg), delta = *(const f4*)(s_delta + 16 * a + 4 * lg);
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = vis[f] != 0.f ? exp2_fast(__builtin_fmaf(t[a][f][r], c, -lse[r])) : 0.f;
                        float kept = e, dp = g[a][f][r];
                        if constexpr (KEEP) {
                            const int qrow = q0 + 16 * a + 4 * lg + r, key = row0 + 16 * f + lr;
                            const bool on = qrow < sq.len && key < ks.len && key < p.keep_cols &&
                                            p.keep[(sq.begin + qrow) * p.keep_row + head * p.keep_head + key] != 0;
                            kept = on ? e : 0.f;
                            dp = on ? dp * p.keep_scale : 0.f;
                        }
                        t[a][f][r] = kept;
                        g[a][f][r] = e * (dp - delta[r]);
                    }
            }
            gather<T, DP, F>(sd_t, t, lr, lg, dv);
            gather<T, DP, F>(sq_t, g, lr, lg, dk);
        }
        float mk[F], mv[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            mk[f] = vis[f] != 0.f ? p.scale : 0.f;
            mv[f] = vis[f] != 0.f ? (KEEP ? p.keep_scale : 1.f) : 0.f;
        }
        store_owned<T, DP, F>(p.dk + ks.begin * rb + it.head * (p.dim * G::SZ), rb, row0, ks.len, p.dim, lr, lg, dk, mk);
        store_owned<T, DP, F>(p.dv + ks.begin * rb + it.head * (p.dim * G::SZ), rb, row0, ks.len, p.dim, lr, lg, dv, mv);
    }
}

// ---- launches ----
static inline int attention_blocks(AttnP& p, int64_t tiles, int heads) {
    const int64_t n = (tiles * heads * p.batch + 7) / 8 * 8;
    if (n > (1 << 30)) return -1;
    p.tiles = (int)tiles;
    p.blocks = (int)n;
    return 0;
}
static constexpr int GAP_BLOCKS = 8;                    // blocks that clear the rows of no sequence (usually there are none)

template <class K> static int attention_launch(K kernel, const AttnP& p, int lds, hipStream_t stream) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3(p.blocks + GAP_BLOCKS), dim3(256), lds, stream, p);
    return (int)hipGetLastError();
}

template <class T, int DP, bool KEEP> static int attention_forward_dp(AttnP p, int max_q, hipStream_t stream) {
    const int lds = 2 * WALK * Geo<T, DP>::PITCH + 4 * WALK;
    if (attention_blocks(p, (max_q + 63) / 64, p.heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    return attention_launch(attention_forward_kernel<T, DP, 1, KEEP>, p, lds, stream);
}
template <class T, int DP, bool KEEP> static int attention_backward_dp(AttnP p, int max_q, int max_k, hipStream_t stream) {
    const int lds = 2 * WALK * Geo<T, DP>::PITCH + 12 * WALK;
    if (attention_blocks(p, (max_q + 63) / 64, p.heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    int rc = attention_launch(attention_dq_kernel<T, DP, 1, KEEP>, p, lds, stream);
    if (rc) return rc;
    if (attention_blocks(p, (max_k + 63) / 64, p.kv_heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    return attention_launch(attention_dkv_kernel<T, DP, 1, KEEP>, p, lds, stream);
}

template <class T> int attention_forward_t(const AttnP& p, int max_q, hipStream_t s) {
    if (p.dim <= 64) return p.keep ? attention_forward_dp<T, 64, true>(p, max_q, s) : attention_forward_dp<T, 64, false>(p, max_q, s);
    return p.keep ? attention_forward_dp<T, 128, true>(p, max_q, s) : attention_forward_dp<T, 128, false>(p, max_q, s);
}
template <class T> int attention_backward_t(const AttnP& p, int max_q, int max_k, hipStream_t s) {
    if (p.dim <= 64) return p.keep ? attention_backward_dp<T, 64, true>(p, max_q, max_k, s) : attention_backward_dp<T, 64, false>(p, max_q, max_k, s);
    return p.keep ? attention_backward_dp<T, 128, true>(p, max_q, max_k, s) : attention_backward_dp<T, 128, false>(p, max_q, max_k, s);
}

}  // namespace atlas_train
