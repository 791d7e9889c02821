// attention.h -- attention over packed sequences, forward and backward, for one element type (attention_{f16,bf16,f32}.hip).
//
//   forward   S = scale q k^T; O = softmax(S) v in one pass over the keys with the running maximum and sum of the softmax; what is kept
//             for the backward pass is one float per row, lse = log2 sum 2^(S log2 e), and the dropout's decisions as bits
//   backward  P = 2^(S log2 e - lse) is recomputed. With M = keep * keep_scale and delta = rowsum(dO . O):
//             dS = P . (M . (dO v^T) - delta);  dq = scale dS k;  dk = scale dS^T q;  dv = (M . P)^T dO
//             dq_kernel owns query rows and walks the keys (and leaves delta); dkv_kernel owns keys and walks the query rows of every
//             query head that shares them. Each recomputes S and dO v^T (7 products instead of 5) and neither needs an atomic: the same
//             bits from call to call.
// All three are the same loop: a wave OWNS R rows (32; 16 in fp32, whose rows take twice the registers and time) whose vectors sit in registers as B fragments; tiles of WALKED rows pass through LDS
// (two buffers, one barrier a tile, the next tile on its way in registers); R x R products with the walked rows as the A operand leave, in each
// lane, runs of four consecutive walked rows of one owned row -- which is the B fragment layout of the second product, whose A operand is read out of
// the same row-major tile through the transposing LDS read. So scores and probabilities never leave their lane, and the statistics of an owned row
// are scalars of its lane and of the lanes R, 2 R .. away.
// P and dS are rounded once to the tensors' 16 bits where they become operands of the second products (half a unit of the last place of each, of either sign: it
// averages out over a row's keys; a gradient's error grows from one rounding's to some 1.45 of it, 0.0024 for 0.0017 in bf16). The running sum and lse are of the
// unrounded fp32 values. delta, whose error all dS of a row have, is of the output before its rounding, which comes along in a byte a value (Rest), and the largest P of
// a row is not rounded (Range): from the rounded output, dq and dk of rows that few keys dominate were off by 0.0064 for 0.0017 (bf16, scores of deviation 6 over 200
// keys; now 0.0024), of two keys by 0.0045 (now 0.0025). It costs 80 passages 3.5 us of 41 forward and 3 of 46 in dq, two sequences of 4000 tokens 11 of 675 a step.
// What bounds it: of two sequences of 4000 tokens the vector unit is busy 47 / 32 / 35 % of the time (forward, dq, dkv), the matrix unit 26 / 29 / 30 %, at 1.3 .. 1.7 waves
// a SIMD of the three or two that fit (the last round of workgroups is nearly empty): latency, and most of it the vector unit's. A score costs one v_exp_f32 (a quarter
// of the rate) and some five other instructions against 256 (forward, D = 64) matrix operations, so everything else is kept out of it: tiles come by buffer loads whose descriptor moves (no address arithmetic, no bounds branches),
// the running maximum is raised only when it grows (fp32: by 2^8), masks are looked at only where there are any.
#pragma once
#include <type_traits>
#include "elements.h"

namespace atlas_train {

struct AttnP {
    const unsigned char *q, *k, *v, *dout;
    const unsigned char* out_in;                        // backward: the forward's output
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;      // in bytes
    const int32_t *q_offsets, *k_offsets;
    int64_t total_q, total_k;
    int batch, heads, kv_heads, dim, keep_cols, keep_words;
    const uint8_t *key_mask, *keep;
    int64_t keep_row, keep_head;
    uint32_t* keep_bits;                                // [heads][total_q][keep_words]
    float scale, keep_scale;
    unsigned char *out, *dq, *dk, *dv;                  // out: forward only
    float *lse, *delta;
    uint8_t* out_rest;                                  // [total_q][heads][DP]: what rounding left of the output (16-bit types; or none)
    int tiles;                                          // tiles of the longest sequence (launch size)
    int blocks;                                         // blocks that compute; those behind them clear the rows of no sequence
    int splits;                                         // > 1: a walk is split into so many parts, whose sums go to `part` ([splits][rows][heads][dim]; dkv: dk's, then dv's)
    float* part;
    float2* part_stats;                                 // forward: [splits][heads][total_q], the exponent of 2 that its sums are relative to, and the sum
};

typedef float f16v __attribute__((ext_vector_type(16)));

// R x R products. A fragment is 16 bytes a lane: lane l holds row l % R, chunk l / R of a step of 16 * 64 / R bytes of contraction (16-bit: one
// v_mfma_f32_32x32x16; fp32: four v_mfma_f32_16x16x4). The result: register i of lane l is row 8 (i >> 2) + 4 (l / R) + (i & 3), column l % R.
template <class T> struct Square;
template <> struct Square<F16> {
    static constexpr int R = 32;
    typedef f16v Result;
    static __device__ __forceinline__ f16v mma(const u4& a, const u4& b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
};
template <> struct Square<BF16> {
    static constexpr int R = 32;
    typedef f16v Result;
    static __device__ __forceinline__ f16v mma(const u4& a, const u4& b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
};
template <> struct Square<F32> {
    static constexpr int R = 16;
    typedef f4 Result;
    static __device__ __forceinline__ f4 mma(const u4& a, const u4& b, f4 c) { return F32::mma(a, b, c); }
};
template <class T> using Result = typename Square<T>::Result;
template <class T> static __device__ __forceinline__ Result<T> zeros() {
    Result<T> z;
#pragma unroll
    for (int i = 0; i < Square<T>::R * Square<T>::R / 64; ++i) z[i] = 0.f;
    return z;
}
template <class T> static __device__ __forceinline__ float all_max(float x) {
#pragma unroll
    for (int o = Square<T>::R; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
template <class T> static __device__ __forceinline__ float all_sum(float x) {
#pragma unroll
    for (int o = Square<T>::R; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

template <class T, int DP> struct Geo {
    typedef typename T::elem E;
    static constexpr int R = Square<T>::R, NR = R * R / 64, LG = 64 / R;      // rows of a product, its result registers, lane groups
    static constexpr int SZ = (int)sizeof(E), ROW = DP * SZ, CPR = ROW / 16, NKS = CPR / LG, ND = DP / R;
    static constexpr int CH = T::EPC, NCH = NR / CH;                         // result registers that make a B chunk, chunks of a product; a chunk is 16 rows
    static constexpr int WALK = ROW >= 512 ? 32 : 64;                        // walked rows of a tile: two buffers of two tiles within 70 KiB
    // waves of a SIMD that the registers are held to; dkv owns two accumulators, key masks cost some
    static constexpr int WAVES = ROW <= 128 ? 3 : 2, WAVES_DKV = SZ == 2 && DP == 128 ? 1 : 2;
    // pitch: 16 bytes more than the row, so that the row reads of 16 lanes cover the banks
    static constexpr int PITCH = ROW + 16, TILE = WALK * PITCH, LDS = 4 * TILE;
};

struct Seq { int64_t begin; int len; };
static __device__ __forceinline__ Seq sequence(const int32_t* offsets, int b, int64_t total) {
    int64_t lo = __builtin_amdgcn_readfirstlane(offsets[b]), hi = __builtin_amdgcn_readfirstlane(offsets[b + 1]);
    lo = lo < 0 ? 0 : lo > total ? total : lo;
    hi = hi < lo ? lo : hi > total ? total : hi;
    Seq s; s.begin = lo; s.len = (int)(hi - lo);
    return s;
}

// workgroup -> (tile, part of the walk, head, sequence). Workgroup g runs on XCD g mod 8: the tiles of a head, which read the same walked rows, share an XCD and its L2;
// the parts and heads of a sequence are dealt over all XCDs, so that a long sequence does not load one of them (12 ragged sequences of 16 heads, fp32: an eighth
// of the items in order for each XCD took 807 us a step, dealt ones 664). Four heads at a time go tile by tile: their last tiles, often almost empty, come last
// and do not hold up full ones.
struct Item { int tile, split, head, b; };
static constexpr int DEAL = 4;
static __device__ __forceinline__ Item item_of(int bid, int tiles, int splits, int heads, int batch) {
    const int pairs = (splits * heads * batch + 7) / 8, whole = pairs / DEAL * DEAL;   // of an XCD; those that go four at a time
    int slot = bid >> 3, deal = DEAL, first = slot / (DEAL * tiles) * DEAL;
    if (first < whole) slot -= first * tiles;
    else { first = whole; slot -= whole * tiles; deal = pairs - whole; }
    const int part = (first + slot % deal) * 8 + (bid & 7), pair = part / splits;
    Item t;
    t.tile = slot / deal;
    t.split = part - pair * splits;
    t.head = pair % heads;
    t.b = pair / heads;
    return t;
}

// rows that belong to no sequence (in front of the first, behind the last) get zeros
static __device__ __forceinline__ void clear_gaps(unsigned char* out, int64_t row_bytes, const int32_t* offsets, int batch, int64_t total, int part, int parts) {
    int64_t first = offsets[0], last = offsets[batch];
    first = first < 0 ? 0 : first > total ? total : first;
    last = last < first ? first : last > total ? total : last;
    const int64_t n16 = row_bytes / 16, head = first * n16, all = head + (total - last) * n16;
    for (int64_t i = (int64_t)part * blockDim.x + threadIdx.x; i < all; i += (int64_t)parts * blockDim.x) {
        const int64_t at = i < head ? i : last * n16 + (i - head);
        *(u4*)(out + at * 16) = (u4){0, 0, 0, 0};
    }
}

// a buffer descriptor of rows [row0, len) of a sequence: what lies behind the last row's `dim` elements arrives as zeros
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const unsigned char* base, int64_t row_bytes, int row0, int len, int vec_bytes) {
    const int64_t left = row0 < len ? (int64_t)(len - row0 - 1) * row_bytes + vec_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (row0 < len ? (int64_t)row0 * row_bytes : 0)), 0, left > 0x7fffffff ? 0x7fffffff : (int)left, 0x00020000);
}

// one walked tile between global memory and LDS, through registers; NT threads
template <class T, int DP, int NT> struct Tile {
    typedef Geo<T, DP> G;
    static constexpr int RPP = NT / G::CPR, NP = G::WALK / RPP;              // rows of one pass of the threads, passes
    u4 x[NP];
    uint32_t off;                                                            // this thread's place in the first pass
    __device__ __forceinline__ void init(int64_t row_bytes, int dim) {
        const int c = threadIdx.x % G::CPR, r = threadIdx.x / G::CPR;
        off = c * T::EPC < dim ? (uint32_t)(r * row_bytes + c * 16) : 0x80000000u;
    }
    static __device__ __forceinline__ int row(int i) { return i * RPP + (int)threadIdx.x / G::CPR; }
    __device__ __forceinline__ void load(const unsigned char* base, int64_t row_bytes, int row0, int len, int dim) {
        const __amdgpu_buffer_rsrc_t rs = rows_from(base, row_bytes, row0, len, dim * G::SZ);
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + (uint32_t)(i * RPP) * (uint32_t)row_bytes), 0, 0));
    }
    __device__ __forceinline__ void store(unsigned char* tile) const {
#pragma unroll
        for (int i = 0; i < NP; ++i) *(u4*)(tile + row(i) * G::PITCH + (threadIdx.x % G::CPR) * 16) = x[i];
    }
    // rows whose `dead` bit (by pass) is set are stored as zeros: what a hidden row holds must not reach a product
    __device__ __forceinline__ void store_live(unsigned char* tile, uint32_t dead) const {
#pragma unroll
        for (int i = 0; i < NP; ++i) *(u4*)(tile + row(i) * G::PITCH + (threadIdx.x % G::CPR) * 16) = dead >> i & 1 ? (u4){0, 0, 0, 0} : x[i];
    }
};

// the owned rows' vectors as B fragments, straight from global memory (zeros behind the end)
template <class T, int DP> static __device__ __forceinline__ void load_owned(const unsigned char* base, int64_t row_bytes, int row0, int len, int dim, int lane,
                                                                             u4 (&x)[Geo<T, DP>::NKS]) {
    const int row = row0 + lane % Geo<T, DP>::R;
#pragma unroll
    for (int s = 0; s < Geo<T, DP>::NKS; ++s) {
        x[s] = (u4){0, 0, 0, 0};
        const int c = Geo<T, DP>::LG * s + lane / Geo<T, DP>::R;
        if (row < len && c * T::EPC < dim) x[s] = *(const u4*)(base + row * row_bytes + c * 16);
    }
}
// t + (walked rows R a ..) x (the owned rows), contraction over the vectors' dimension
template <class T, int DP> static __device__ __forceinline__ Result<T> scores(const unsigned char* tile, int a, const u4 (&own)[Geo<T, DP>::NKS], int lane, Result<T> t = zeros<T>()) {
    typedef Geo<T, DP> G;
    const unsigned char* p = tile + (G::R * a + lane % G::R) * G::PITCH + lane / G::R * 16;
#pragma unroll
    for (int s = 0; s < G::NKS; ++s) t = Square<T>::mma(*(const u4*)(p + 16 * G::LG * s), own[s], t);
    return t;
}
// acc[d] += (dimensions R d .. of the walked rows R a ..) x t, contraction over the walked rows. fp32: the 16 rows of a product are summed by themselves first. Sums of equal
// terms round one way, and a chain of them over the whole walk, four rows at a time, was off by 5e-5 of the result at 4096 keys, 2e-4 at 65 536
// (now 4e-6 and 1.4e-5; 12 ragged sequences with shared heads: 503 -> 518 us a step).
template <class T, int DP> static __device__ __forceinline__ void gather(const unsigned char* tile, int a, const Result<T>& t, int lane, Result<T> (&acc)[Geo<T, DP>::ND]) {
    typedef Geo<T, DP> G;
#pragma unroll
    for (int c = 0; c < G::NCH; ++c) {
        u4 p;
        if constexpr (T::TILES == 2) p = (u4){pack2<T>(t[8 * c], t[8 * c + 1]), pack2<T>(t[8 * c + 2], t[8 * c + 3]), pack2<T>(t[8 * c + 4], t[8 * c + 5]), pack2<T>(t[8 * c + 6], t[8 * c + 7])};
        else {
            const float a0 = t[4 * c], a1 = t[4 * c + 1], a2 = t[4 * c + 2], a3 = t[4 * c + 3];
            p = (u4){as_u(a0), as_u(a1), as_u(a2), as_u(a3)};
        }
        const int row = G::R * a + 16 * c + 4 * (lane / G::R);               // the lane's rows of the chunk: row .. + 3 (and, 16-bit, + 8 .. + 11)
#pragma unroll
        for (int d = 0; d < G::ND; ++d) {
            u4 w;
            if constexpr (T::TILES == 2) {
                const unsigned char* at = tile + (row + ((lane & 15) >> 2)) * G::PITCH + (32 * d + (lane & 16) + 4 * (lane & 3)) * 2;
                const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)at));
                const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(uintptr_t)(lds_byte*)(at + 8 * G::PITCH)));
                w = (u4){x.x, x.y, y.x, y.y};
            } else {
                const float* at = (const float*)(tile + row * G::PITCH) + G::R * d + lane % G::R;
                w = (u4){as_u(at[0]), as_u(at[G::PITCH / 4]), as_u(at[2 * (G::PITCH / 4)]), as_u(at[3 * (G::PITCH / 4)])};
            }
            if constexpr (T::TILES == 2) acc[d] = Square<T>::mma(w, p, acc[d]);
            else acc[d] += Square<T>::mma(w, p, zeros<T>());
        }
    }
}
template <class T, int DP> static __device__ __forceinline__ void store_owned(unsigned char* base, int64_t row_bytes, int row0, int len, int dim, int lane,
                                                                              const Result<T> (&acc)[Geo<T, DP>::ND], float mul) {
    typedef typename T::elem E;
    typedef Geo<T, DP> G;
    const int row = row0 + lane % G::R;
    if (row >= len) return;
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int c = 0; c < G::NR / 4; ++c) {
            const int e = G::R * d + 8 * c + 4 * (lane / G::R);
            if (e >= dim) continue;
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = mul == 0.f ? 0.f : acc[d][4 * c + r] * mul;     // a row without keys is zeros, whatever was summed
            store_n<T, 4>((E*)(base + row * row_bytes) + e, o);
        }
}

// what rounding leaves of the output, four dimensions a word. A lane has those at 8 c + 4 (lane / R) of every 32: the word's place is such that they are two runs here and,
// in the backward pass, where a lane has whole chunks of eight dimensions, one
template <class T, int DP> static __device__ __forceinline__ int rest_word(int d, int c, int group) { return ((c & 1) * 2 + group) * (2 * Geo<T, DP>::ND) + 2 * d + (c >> 1); }
template <class T, int DP> static __device__ __forceinline__ void store_rest(uint8_t* base, int64_t row_bytes, int row0, int len, int dim, int lane,
                                                                             const Result<T> (&acc)[Geo<T, DP>::ND], float mul) {
    typedef Geo<T, DP> G;
    constexpr int RUN = 2 * G::ND;
    const int row = row0 + lane % G::R;
    if (row >= len) return;
    uint32_t w[2][RUN];
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = mul == 0.f ? 0.f : acc[d][4 * c + r] * mul;
            w[c & 1][2 * d + (c >> 1)] = rest4<T>(o);
        }
#pragma unroll
    for (int odd = 0; odd < 2; ++odd)
#pragma unroll
        for (int i = 0; i < RUN; i += 4)
            *(u4*)(base + row * row_bytes + 4 * (rest_word<T, DP>(0, odd, lane / G::R) + i)) = (u4){w[odd][i], w[odd][i + 1], w[odd][i + 2], w[odd][i + 3]};
}

// one part's sums of the owned rows, fp32; of rows that count for nothing, zeros
template <class T, int DP> static __device__ __forceinline__ void store_part(float* base, int64_t row_elems, int row0, int len, int dim, int lane,
                                                                             const Result<T> (&acc)[Geo<T, DP>::ND], float mul) {
    typedef Geo<T, DP> G;
    const int row = row0 + lane % G::R;
    if (row >= len) return;
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int c = 0; c < G::NR / 4; ++c) {
            const int e = G::R * d + 8 * c + 4 * (lane / G::R);
            if (e >= dim) continue;
            f4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = mul == 0.f ? 0.f : acc[d][4 * c + r] * mul;
            *(f4*)(base + row * row_elems + e) = o;
        }
}
// fp16 ends at 2^16 and loses bits below 2^-14, where dS of long sequences lies: there the dS of an owned row (a column of products) are held times 2^lift, lift
// as large as their largest so far allows, lowered where one passes 2^15. (4000 keys, gradients of 0.003: dq off by 8.7e-4 of its norm without, 3.0e-4 with;
// and finite results where a dS passes 2^16. It costs dq 4 % and dkv 17 %: 289 -> 338 us, 2 sequences of 4000 tokens, 12 heads.)
// The largest of a product's values times 2^lift is looked at; returns whether some row's lift falls, by `down`.
// P is at most 1, and about 1 / keys: dkv's are held times 2^P15 from the exponent on, so that one of 2^-29 still has all its bits (dv of 262 144 keys off by 5.2e-3 of
// its norm without, by the roundings' 3e-4 with).
template <class T> struct Lift {
    static constexpr bool ON = T::DT == ATLAS_TRAIN_F16;
    static constexpr int P15 = ON ? 15 : 0;
    int lift = ON ? 24 : 0;
    __device__ __forceinline__ bool passed(const Result<T>& t, int& down) const {
        constexpr int NR = Square<T>::R * Square<T>::R / 64;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i) top = fmaxf(top, fabsf(t[i]));
        down = 0;
        if (!__any(top > 32768.f)) return false;
        top = all_max<T>(top);
        if (top > 32768.f && top < __builtin_inff()) down = (int)(as_u(top) >> 23) - 127 - 8;
        return true;
    }
    __device__ __forceinline__ float undo() const { return power_of(-lift); }
};
// The forward pass holds probabilities relative to the running maximum, which may lag by a factor of 2^LAG in fp32. In 16 bits it does not: a row's largest probability
// is then a power of 2, and what the others lost in rounding is all that delta is off by. fp16: times 2^SHIFT, so that those down to 2^-29 of the row's largest
// keep all their bits (65 535 keys of 2^-25.6 each beside a large one: lost without). The sum has the factor too; lse goes without.
template <class T> struct Range {
    static constexpr int SHIFT = T::DT == ATLAS_TRAIN_F16 ? 15 : 0;
    static constexpr float LAG = Rest<T>::ON ? 0.f : 8.f;
};
// this workgroup's run of `all` walked tiles
struct Run { int begin, end; };
static __device__ __forceinline__ Run run_of(int all, int split, int splits) {
    const int per = (all + splits - 1) / splits, begin = split * per;
    Run r;
    r.begin = begin < all ? begin : all;
    r.end = begin + per < all ? begin + per : all;
    return r;
}

// ---- dropout's decisions: 32 keys of one query row are a word, bit j for key j ----
// the R / 16 .. lanes of a wave that share a row read R / 2 bytes (0 or 1 each) of the row's 32 and exchange their bits; columns from `cols` on count as dropped
static __device__ __forceinline__ uint32_t nibble(uint32_t w) { w |= w >> 7; return (w | w >> 14) & 15u; }
template <int R> struct KeepBytes {
    static constexpr int N = R / 2;                     // keys of a lane
    uint32_t w[N / 4];
    __device__ __forceinline__ void load(const uint8_t* rows, uint32_t row, int j0, int cols, int lane) {
        const int j = j0 + N * (lane / R);
        const uint32_t at = row + (uint32_t)j;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = 0;
        if (j + N <= cols) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) w[i] = *(const u32_any*)(rows + at + 4 * i);
        } else
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (j + i < cols) w[i / 4] |= (uint32_t)rows[at + i] << (8 * (i & 3));
    }
    __device__ __forceinline__ uint32_t word(int lane) const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) m |= nibble(w[i]) << (4 * i);
        m <<= N * (lane / R);
#pragma unroll
        for (int o = R; o < 64; o <<= 1) m |= (uint32_t)__shfl_xor((int)m, o);
        return m;
    }
};
// register i of a result is walked row 8 (i >> 2) + (i & 3), shifted by the lane group's 4
static __device__ __forceinline__ constexpr int row_of(int i) { return 8 * (i >> 2) + (i & 3); }
// x where the word's bit is set, 0 (whatever x is) elsewhere
static __device__ __forceinline__ float kept(float x, uint32_t word, int bit) { return as_f(as_u(x) & (uint32_t)__builtin_amdgcn_sbfe((int)word, bit, 1)); }

// what is known about the rows of a walked tile of keys: for the staging threads which of their rows are hidden, for the others a live flag per row
template <class T, int DP, int NT> struct KeyMask {
    typedef Tile<T, DP, NT> TL;
    uint32_t dead;
    float alive;
    __device__ __forceinline__ void load(const uint8_t* mask, int row0, int len) {       // mask: of the sequence
        dead = 0;
#pragma unroll
        for (int i = 0; i < TL::NP; ++i) {
            const int r = row0 + TL::row(i);
            dead |= (r < len && mask[r] == 0 ? 1u : 0u) << i;
        }
        const int r = row0 + (int)threadIdx.x;
        alive = threadIdx.x < Geo<T, DP>::WALK && r < len && mask[r] ? 1.f : 0.f;
    }
};
// scores of keys that are hidden or behind the end become -inf
template <class T> static __device__ __forceinline__ void hide(Result<T>& t, const float* live /* of the product's rows */, int lane) {
    constexpr int R = Square<T>::R;
#pragma unroll
    for (int c = 0; c < R * R / 256; ++c) {
        const f4 on = *(const f4*)(live + 8 * c + 4 * (lane / R));
#pragma unroll
        for (int r = 0; r < 4; ++r) t[4 * c + r] = on[r] != 0.f ? t[4 * c + r] : -__builtin_inff();
    }
}
template <class T> static __device__ __forceinline__ void hide_behind(Result<T>& t, int left /* rows from the product's first on */, int lane) {
    constexpr int R = Square<T>::R;
    left -= 4 * (lane / R);
#pragma unroll
    for (int i = 0; i < R * R / 64; ++i) t[i] = 8 * (i >> 2) + (i & 3) < left ? t[i] : -__builtin_inff();
}

// ---- forward: owned = query rows, walked = keys ----
template <class T, int DP, int NW, bool KEEP, bool MASK>
__global__ void __launch_bounds__(NW * 64, (MASK ? 2 : Geo<T, DP>::WAVES)) attention_forward_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    constexpr int R = G::R, NR = G::NR, A = G::WALK / R, PER = 32 / R;       // products of a tile, products of a dropout word
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.out, (int64_t)p.heads * p.dim * G::SZ, p.q_offsets, p.batch, p.total_q, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // two buffers of k | v, two of live flags
    float* live = (float*)(smem + G::LDS);
    const Item it = item_of(blockIdx.x, p.tiles, p.splits, p.heads, p.batch);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int kvh = it.head / (p.heads / p.kv_heads);
    const unsigned char* kb = p.k + ks.begin * p.k_row + kvh * p.k_head;
    const unsigned char* vb = p.v + ks.begin * p.v_row + kvh * p.v_head;
    const unsigned char* qb = p.q + sq.begin * p.q_row + it.head * p.q_head;
    const float c = p.scale * 1.4426950408889634f;                           // exponents in base 2
    const Run run = run_of((ks.len + G::WALK - 1) / G::WALK, it.split, p.splits);
    const int kend = run.end * G::WALK < ks.len ? run.end * G::WALK : ks.len;
    Tile<T, DP, NW * 64> tk, tv;
    KeyMask<T, DP, NW * 64> km;
    tk.init(p.k_row, p.dim);
    tv.init(p.v_row, p.dim);
    auto fetch = [&](int k0) {
        tk.load(kb, p.k_row, k0, kend, p.dim);
        tv.load(vb, p.v_row, k0, kend, p.dim);
        if constexpr (MASK) km.load(p.key_mask + ks.begin, k0, kend);
    };
    for (int tile = it.tile; tile * R * NW < sq.len; tile += p.tiles) {
        const int row0 = (tile * NW + wave) * R, row = row0 + lane % R;
        u4 own[G::NKS];
        load_owned<T, DP>(qb, p.q_row, row0, sq.len, p.dim, lane, own);
        Result<T> acc[G::ND];
#pragma unroll
        for (int d = 0; d < G::ND; ++d) acc[d] = zeros<T>();
        float m = -__builtin_inff(), l = 0.f;
        KeepBytes<R> bytes[A / PER];                                         // dropout's decisions, on their way while the scores are made (80 passages: 43.6 us, so 40.9)
        uint32_t words[A / PER];
        const uint8_t* keep = KEEP ? p.keep + (sq.begin + row0) * p.keep_row + it.head * p.keep_head : nullptr;      // of the wave's first row
        uint32_t* keep_bits = KEEP && p.keep_bits ? p.keep_bits + ((int64_t)it.head * p.total_q + sq.begin + row0) * p.keep_words : nullptr;
        auto fetch_keep = [&](int k0) {
#pragma unroll
            for (int a = 0; a < A / PER; ++a)
                if (row < sq.len) bytes[a].load(keep, (uint32_t)(lane % R) * (uint32_t)p.keep_row, k0 + 32 * a, p.keep_cols, lane);
        };
        auto take_keep = [&](int k0) {
#pragma unroll
            for (int a = 0; a < A / PER; ++a) {
                const int j0 = k0 + 32 * a;
                words[a] = bytes[a].word(lane);
                if (keep_bits && lane < R && row < sq.len && j0 < p.keep_cols) keep_bits[(uint32_t)lane * (uint32_t)p.keep_words + (uint32_t)(j0 >> 5)] = words[a];
                words[a] >>= 4 * (lane / R);
            }
        };
        // one tile; PART: it ends behind the last key (its own code, so that whole tiles carry no trace of the check)
        auto step = [&](auto part, int k0, int buf) {
            constexpr bool PART = decltype(part)::value;
            unsigned char *sk = smem + buf * 2 * G::TILE, *sv = sk + G::TILE;
            float* on = live + buf * G::WALK;
            if constexpr (MASK) {
                if (threadIdx.x < G::WALK) on[threadIdx.x] = km.alive;
                tk.store_live(sk, km.dead);
                tv.store_live(sv, km.dead);
            } else {
                tk.store(sk);
                tv.store(sv);
            }
            __syncthreads();                                                 // (the buffer's last readers passed the barrier before)
            if (!PART && k0 + G::WALK < kend) fetch(k0 + G::WALK);
            if (row0 >= sq.len) return;                                      // no rows for this wave: it only helps to stage
            if constexpr (KEEP) fetch_keep(k0);
            Result<T> t[A];
#pragma unroll
            for (int a = 0; a < A; ++a) t[a] = scores<T, DP>(sk, a, own, lane);
            if constexpr (MASK) {
#pragma unroll
                for (int a = 0; a < A; ++a) hide<T>(t[a], on + R * a, lane);
            } else if constexpr (PART) {
#pragma unroll
                for (int a = 0; a < A; ++a) hide_behind<T>(t[a], kend - k0 - R * a, lane);
            }
            float top = t[0][0];
#pragma unroll
            for (int a = 0; a < A; ++a)
#pragma unroll
                for (int i = 0; i < NR; ++i) top = fmaxf(top, t[a][i]);
            // raised only where a probability would pass 2^LAG (or there was none yet), and where none does, the exchange between a row's lanes is skipped too (two sequences
            // of 4000 tokens, 12 heads: 187 us with it in every tile, 180 where a lag of 2^8 lets most tiles skip it)
            if (__any((top - m) * c > Range<T>::LAG)) {
                top = all_max<T>(top);
                const float next = fmaxf(m, top), base = next == -__builtin_inff() ? 0.f : next;
                const float less = exp2_fast((m - base) * c);
                l *= less;
#pragma unroll
                for (int d = 0; d < G::ND; ++d) acc[d] *= less;
                m = next;
            }
            const float off = m == -__builtin_inff() ? 0.f : (float)Range<T>::SHIFT - m * c;
            float tile_sum = 0.f;                                            // (by itself: as in gather)
            if constexpr (KEEP) take_keep(k0);
#pragma unroll
            for (int a = 0; a < A; ++a) {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    t[a][i] = exp2_fast(__builtin_fmaf(t[a][i], c, off));
                    tile_sum += t[a][i];
                }
                if constexpr (KEEP) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) t[a][i] = kept(t[a][i], words[a / PER], R * (a % PER) + row_of(i));
                }
                gather<T, DP>(sv, a, t[a], lane, acc);
            }
            l += tile_sum;
        };
        int k0 = run.begin * G::WALK, buf = 0;
        fetch(k0);
        for (; k0 + G::WALK <= kend; k0 += G::WALK, buf ^= 1) step(std::false_type{}, k0, buf);
        if (k0 < kend) step(std::true_type{}, k0, buf);
        const float sum = all_sum<T>(l);
        if (p.splits > 1) {
            const int64_t at = ((int64_t)it.split * p.total_q + sq.begin) * p.heads + it.head;
            store_part<T, DP>(p.part + at * p.dim, (int64_t)p.heads * p.dim, row0, sq.len, p.dim, lane, acc, 1.f);
            if (lane < R && row < sq.len)
                p.part_stats[((int64_t)it.split * p.heads + it.head) * p.total_q + sq.begin + row] = make_float2(m == -__builtin_inff() ? m : m * c - (float)Range<T>::SHIFT, sum);
            __syncthreads();
            continue;
        }
        const float mul = sum == 0.f ? 0.f : (KEEP ? p.keep_scale : 1.f) / sum;      // (scores that are NaN leave a NaN sum: no empty row)
        if (lane < R && row < sq.len)
            p.lse[(int64_t)it.head * p.total_q + sq.begin + row] = sum == 0.f ? __builtin_inff() : __builtin_fmaf(m, c, log2f(sum) - (float)Range<T>::SHIFT);
        const int64_t rb = (int64_t)p.heads * p.dim * G::SZ;
        store_owned<T, DP>(p.out + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lane, acc, mul);
        if constexpr (Rest<T>::ON)
            if (p.out_rest) store_rest<T, DP>(p.out_rest + (sq.begin * p.heads + it.head) * DP, (int64_t)p.heads * DP, row0, sq.len, p.dim, lane, acc, mul);
        __syncthreads();                                                     // the next round starts with the first buffer again
    }
}

// ---- backward, dq: owned = query rows, walked = keys; leaves delta for dkv_kernel ----
template <class T, int DP, int NW, bool KEEP, bool MASK>
__global__ void __launch_bounds__(NW * 64, (MASK ? 2 : Geo<T, DP>::WAVES)) attention_dq_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    constexpr int R = G::R, NR = G::NR, A = G::WALK / R, PER = 32 / R;       // products of a tile, products of a dropout word
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.dq, (int64_t)p.heads * p.dim * G::SZ, p.q_offsets, p.batch, p.total_q, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float* live = (float*)(smem + G::LDS);
    const Item it = item_of(blockIdx.x, p.tiles, p.splits, p.heads, p.batch);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int kvh = it.head / (p.heads / p.kv_heads);
    const unsigned char* kb = p.k + ks.begin * p.k_row + kvh * p.k_head;
    const unsigned char* vb = p.v + ks.begin * p.v_row + kvh * p.v_head;
    const int64_t rb = (int64_t)p.heads * p.dim * G::SZ;
    const float c = p.scale * 1.4426950408889634f;
    const Run run = run_of((ks.len + G::WALK - 1) / G::WALK, it.split, p.splits);
    const int kend = run.end * G::WALK < ks.len ? run.end * G::WALK : ks.len;
    Tile<T, DP, NW * 64> tk, tv;
    KeyMask<T, DP, NW * 64> km;
    tk.init(p.k_row, p.dim);
    tv.init(p.v_row, p.dim);
    auto fetch = [&](int k0) {
        tk.load(kb, p.k_row, k0, kend, p.dim);
        tv.load(vb, p.v_row, k0, kend, p.dim);
        if constexpr (MASK) km.load(p.key_mask + ks.begin, k0, kend);
    };
    for (int tile = it.tile; tile * R * NW < sq.len; tile += p.tiles) {
        const int row0 = (tile * NW + wave) * R, row = row0 + lane % R;
        const int64_t at = (int64_t)it.head * p.total_q + sq.begin + row;
        u4 own[G::NKS], dof[G::NKS];
        load_owned<T, DP>(p.q + sq.begin * p.q_row + it.head * p.q_head, p.q_row, row0, sq.len, p.dim, lane, own);
        load_owned<T, DP>(p.dout + sq.begin * p.do_row + it.head * p.do_head, p.do_row, row0, sq.len, p.dim, lane, dof);
        const float lse = row < sq.len ? p.lse[at] : __builtin_inff();
        const bool empty = lse == __builtin_inff();                          // nothing visible: q and dout of the row are not used
        float delta = 0.f;
        {
            u4 of[G::NKS], rest[G::NKS / 2];
            if constexpr (Rest<T>::ON) {
                const uint8_t* at = p.out_rest + ((sq.begin + row) * p.heads + it.head) * DP + 4 * rest_word<T, DP>(0, lane / R, 0);
#pragma unroll
                for (int i = 0; i < G::NKS / 2; ++i) rest[i] = p.out_rest && row < sq.len ? *(const u4*)(at + 16 * i) : (u4){0, 0, 0, 0};
            }
            load_owned<T, DP>(p.out_in + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lane, of);
#pragma unroll
            for (int i = 0; i < G::NKS; ++i) {
                float x[T::EPC], y[T::EPC];
                unpack<T>(of[i], x);
                if constexpr (Rest<T>::ON) {                                 // (the lane's dimensions 16 i + 8 (lane / R) .. + 7; those behind dim have no byte)
                    const bool in = 16 * i + 8 * (lane / R) < p.dim;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t w = rest[j / 4 * (G::NKS / 4) + i / 4][i & 3];
                        x[j] = Rest<T>::value(x[j], in ? w : 0u, j & 3);
                    }
                }
                unpack<T>(dof[i], y);
#pragma unroll
                for (int j = 0; j < T::EPC; ++j) delta = __builtin_fmaf(x[j], y[j], delta);
                if (empty) own[i] = dof[i] = (u4){0, 0, 0, 0};
            }
            delta = all_sum<T>(delta);
            if (empty) delta = 0.f;
            if (lane < R && row < sq.len && it.split == 0) p.delta[at] = delta;
        }
        Lift<T> lift;
        float neg_lse = -lse + (float)lift.lift;                             // (dS times 2^lift: in the exponent)
        const uint32_t* keep_bits = KEEP ? p.keep_bits + ((int64_t)it.head * p.total_q + sq.begin + row0) * p.keep_words : nullptr;      // of the wave's first row
        Result<T> acc[G::ND];
#pragma unroll
        for (int d = 0; d < G::ND; ++d) acc[d] = zeros<T>();
        auto step = [&](auto part, int k0, int buf) {
            constexpr bool PART = decltype(part)::value;
            unsigned char *sk = smem + buf * 2 * G::TILE, *sv = sk + G::TILE;
            float* on = live + buf * G::WALK;
            if constexpr (MASK) {
                if (threadIdx.x < G::WALK) on[threadIdx.x] = km.alive;
                tk.store_live(sk, km.dead);
                tv.store_live(sv, km.dead);
            } else {
                tk.store(sk);
                tv.store(sv);
            }
            uint32_t word[A / PER];
            if constexpr (KEEP) {
#pragma unroll
                for (int a = 0; a < A / PER; ++a) {
                    const int j0 = k0 + 32 * a;
                    word[a] = row < sq.len && j0 < p.keep_cols && j0 < kend ? keep_bits[(uint32_t)(lane % R) * (uint32_t)p.keep_words + (uint32_t)(j0 >> 5)] >> (4 * (lane / R)) : 0u;
                }
            }
            __syncthreads();
            if (!PART && k0 + G::WALK < kend) fetch(k0 + G::WALK);
            if (row0 >= sq.len) return;                                      // no rows for this wave: it only helps to stage
#pragma unroll
            for (int a = 0; a < A; ++a) {
                Result<T> t = scores<T, DP>(sk, a, own, lane);
                Result<T> g;                                                      // dP - delta: the product starts from -delta (with dropout, 0)
#pragma unroll
                for (int i = 0; i < NR; ++i) g[i] = KEEP ? 0.f : -delta;
                g = scores<T, DP>(sv, a, dof, lane, g);
                if constexpr (MASK) hide<T>(t, on + R * a, lane);
                else if constexpr (PART) hide_behind<T>(t, kend - k0 - R * a, lane);
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const float e = exp2_fast(__builtin_fmaf(t[i], c, neg_lse));
                    if constexpr (KEEP) t[i] = e * __builtin_fmaf(kept(g[i], word[a / PER], R * (a % PER) + row_of(i)), p.keep_scale, -delta);
                    else t[i] = e * g[i];
                }
                if constexpr (Lift<T>::ON) {
                    int down;
                    if (lift.passed(t, down)) {
                        const float less = power_of(-down);
                        t *= less;
#pragma unroll
                        for (int d = 0; d < G::ND; ++d) acc[d] *= less;
                        lift.lift -= down;
                        neg_lse -= (float)down;
                    }
                }
                gather<T, DP>(sk, a, t, lane, acc);
            }
        };
        int k0 = run.begin * G::WALK, buf = 0;
        fetch(k0);
        for (; k0 + G::WALK <= kend; k0 += G::WALK, buf ^= 1) step(std::false_type{}, k0, buf);
        if (k0 < kend) step(std::true_type{}, k0, buf);
        if (p.splits > 1)
            store_part<T, DP>(p.part + (((int64_t)it.split * p.total_q + sq.begin) * p.heads + it.head) * p.dim, (int64_t)p.heads * p.dim, row0, sq.len, p.dim, lane, acc, empty ? 0.f : lift.undo());
        else store_owned<T, DP>(p.dq + sq.begin * rb + it.head * (p.dim * G::SZ), rb, row0, sq.len, p.dim, lane, acc, empty ? 0.f : p.scale * lift.undo());
        __syncthreads();
    }
}

// ---- backward, dk and dv: owned = keys, walked = the query rows of every query head that reads them ----
// (a hidden key's column holds whatever its zeroed vectors give -- an infinite probability, even -- and is left out when the results are stored;
// columns do not meet)
template <class T, int DP, int NW, bool KEEP, bool MASK>
__global__ void __launch_bounds__(NW * 64, (Geo<T, DP>::WAVES_DKV)) attention_dkv_kernel(const AttnP p) {
    typedef Geo<T, DP> G;
    constexpr int R = G::R, NR = G::NR, A = G::WALK / R;                         // products of a tile
    const int64_t rb = (int64_t)p.kv_heads * p.dim * G::SZ;
    if ((int)blockIdx.x >= p.blocks) {
        clear_gaps(p.dk, rb, p.k_offsets, p.batch, p.total_k, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        clear_gaps(p.dv, rb, p.k_offsets, p.batch, p.total_k, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];     // two buffers of q | dout, of -lse (+ P15) | -delta, of dropout words [WORDS][WALK]
    constexpr int WORDS = NW * R / 32;                                       // dropout words of a walked row for the workgroup's keys
    float* stats = (float*)(smem + G::LDS);
    uint32_t* words = (uint32_t*)(stats + 4 * G::WALK);
    const Item it = item_of(blockIdx.x, p.tiles, p.splits, p.kv_heads, p.batch);
    if (it.b >= p.batch) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Seq sq = sequence(p.q_offsets, it.b, p.total_q), ks = sequence(p.k_offsets, it.b, p.total_k);
    const int group = p.heads / p.kv_heads, steps = (sq.len + G::WALK - 1) / G::WALK;    // walked tiles of one query head
    const Run run = run_of(group * steps, it.split, p.splits);
    const float c = p.scale * 1.4426950408889634f;
    for (int tile = it.tile; tile * R * NW < ks.len; tile += p.tiles) {
        const int row0 = (tile * NW + wave) * R, row = row0 + lane % R;
        u4 kf[G::NKS], vf[G::NKS];
        load_owned<T, DP>(p.k + ks.begin * p.k_row + it.head * p.k_head, p.k_row, row0, ks.len, p.dim, lane, kf);
        load_owned<T, DP>(p.v + ks.begin * p.v_row + it.head * p.v_head, p.v_row, row0, ks.len, p.dim, lane, vf);
        const bool seen = row < ks.len && (!MASK || p.key_mask[ks.begin + row]);
#pragma unroll
        for (int i = 0; i < G::NKS; ++i)
            if (!seen) kf[i] = vf[i] = (u4){0, 0, 0, 0};
        Result<T> dk[G::ND], dv[G::ND];
#pragma unroll
        for (int d = 0; d < G::ND; ++d) dk[d] = dv[d] = zeros<T>();
        Lift<T> lift;
        Tile<T, DP, NW * 64> tq, td;
        tq.init(p.q_row, p.dim);
        td.init(p.do_row, p.dim);
        float r_lse = 0.f, r_delta = 0.f;
        uint32_t r_word = 0, dead = 0;
        static_assert(WORDS * G::WALK <= NW * 64, "a thread holds one dropout word");
        auto fetch = [&](int head, int q0) {
            tq.load(p.q + sq.begin * p.q_row + head * p.q_head, p.q_row, q0, sq.len, p.dim);
            td.load(p.dout + sq.begin * p.do_row + head * p.do_head, p.do_row, q0, sq.len, p.dim);
            const int64_t at = (int64_t)head * p.total_q + sq.begin + q0;
            if (threadIdx.x < G::WALK) {
                const bool on = q0 + (int)threadIdx.x < sq.len;
                r_lse = on ? (float)Lift<T>::P15 - p.lse[at + threadIdx.x] : -__builtin_inff();
                r_delta = on ? -p.delta[at + threadIdx.x] : 0.f;
            }
            if constexpr (MASK) {                                            // only then can a row have nothing to see: its q and dout are not used
                dead = 0;
#pragma unroll
                for (int i = 0; i < Tile<T, DP, NW * 64>::NP; ++i) {
                    const int r = Tile<T, DP, NW * 64>::row(i);
                    dead |= (q0 + r < sq.len && p.lse[at + r] == __builtin_inff() ? 1u : 0u) << i;
                }
            }
            if constexpr (KEEP) {                                            // thread (w, r): keys 32 w .. of this workgroup, walked row r
                const int w = threadIdx.x / G::WALK, r = threadIdx.x % G::WALK, j0 = tile * NW * R + 32 * w;
                r_word = w < WORDS && q0 + r < sq.len && j0 < p.keep_cols && j0 < ks.len ? p.keep_bits[(at + r) * p.keep_words + (j0 >> 5)] : 0u;
            }
        };
        int buf = 0, h = steps > 0 ? run.begin / steps : 0, q0 = (run.begin - h * steps) * G::WALK;
        if (run.begin < run.end) fetch(it.head * group + h, q0);
        for (int i = run.begin; i < run.end; ++i, buf ^= 1) {
            unsigned char *sq_t = smem + buf * 2 * G::TILE, *sd_t = sq_t + G::TILE;
            float *s_lse = stats + buf * 2 * G::WALK, *s_delta = s_lse + G::WALK;
            uint32_t* s_word = words + buf * WORDS * G::WALK;
            if (threadIdx.x < G::WALK) { s_lse[threadIdx.x] = r_lse; s_delta[threadIdx.x] = r_delta; }
            if constexpr (KEEP)
                if (threadIdx.x < WORDS * G::WALK) s_word[threadIdx.x] = r_word;
            if constexpr (MASK) {
                tq.store_live(sq_t, dead);
                td.store_live(sd_t, dead);
            } else {
                tq.store(sq_t);
                td.store(sd_t);
            }
            __syncthreads();
            q0 += G::WALK;
            if (q0 >= sq.len) { q0 = 0; ++h; }
            if (i + 1 < run.end) fetch(it.head * group + h, q0);
#pragma unroll
            for (int a = 0; a < A; ++a) {
                Result<T> t = scores<T, DP>(sq_t, a, kf, lane), g;
                if constexpr (KEEP) g = zeros<T>();
                else                                                     // dP - delta: the product starts from -delta
#pragma unroll
                    for (int cc = 0; cc < NR / 4; ++cc) {
                        const f4 delta = *(const f4*)(s_delta + R * a + 8 * cc + 4 * (lane / R));
#pragma unroll
                        for (int r = 0; r < 4; ++r) g[4 * cc + r] = delta[r];
                    }
                g = scores<T, DP>(sd_t, a, vf, lane, g);
#pragma unroll
                for (int cc = 0; cc < NR / 4; ++cc) {
                    const int r4 = R * a + 8 * cc + 4 * (lane / R);
                    const f4 nl = *(const f4*)(s_lse + r4);
                    f4 delta = {0.f, 0.f, 0.f, 0.f};
                    u4 w = {0, 0, 0, 0};
                    if constexpr (KEEP) { delta = *(const f4*)(s_delta + r4); w = *(const u4*)(s_word + wave * R / 32 * G::WALK + r4); }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 4 * cc + r;
                        const float e = exp2_fast(__builtin_fmaf(t[i], c, nl[r]));
                        if constexpr (KEEP) {
                            const int bit = wave * R % 32 + lane % R;
                            t[i] = kept(e, w[r], bit);
                            g[i] = e * __builtin_fmaf(kept(g[i], w[r], bit), p.keep_scale, delta[r]);
                        } else {
                            t[i] = e;
                            g[i] *= e;
                        }
                    }
                }
                gather<T, DP>(sd_t, a, t, lane, dv);
                if constexpr (Lift<T>::ON) {
                    g *= power_of(lift.lift - Lift<T>::P15);                 // (they have P's already)
                    int down;
                    if (lift.passed(g, down)) {
                        const float less = power_of(-down);
                        g *= less;
#pragma unroll
                        for (int d = 0; d < G::ND; ++d) dk[d] *= less;
                        lift.lift -= down;
                    }
                }
                gather<T, DP>(sq_t, a, g, lane, dk);
            }
        }
        if (p.splits > 1) {
            const int64_t plane = p.total_k * p.kv_heads * p.dim, re = (int64_t)p.kv_heads * p.dim;
            float* to = p.part + it.split * plane + ks.begin * re + it.head * p.dim;
            store_part<T, DP>(to, re, row0, ks.len, p.dim, lane, dk, seen ? lift.undo() : 0.f);
            store_part<T, DP>(to + p.splits * plane, re, row0, ks.len, p.dim, lane, dv, seen ? power_of(-Lift<T>::P15) : 0.f);
            __syncthreads();
            continue;
        }
        store_owned<T, DP>(p.dk + ks.begin * rb + it.head * (p.dim * G::SZ), rb, row0, ks.len, p.dim, lane, dk, seen ? p.scale * lift.undo() : 0.f);
        store_owned<T, DP>(p.dv + ks.begin * rb + it.head * (p.dim * G::SZ), rb, row0, ks.len, p.dim, lane, dv, seen ? (KEEP ? p.keep_scale : 1.f) * power_of(-Lift<T>::P15) : 0.f);
        __syncthreads();
    }
}

// ---- a split walk's parts, joined in their order; eight dimensions a thread, rows of no sequence get zeros ----
// SOFTMAX: the parts' sums are of probabilities relative to the exponent in each part's statistics. Otherwise a plain sum, for one or two (blockIdx.y) results.
template <class T, bool SOFTMAX>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnP p, const int32_t* offsets, int64_t total, int heads, unsigned char* out0, float mul0,
                                                             unsigned char* out1, float mul1) {
    typedef typename T::elem E;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, plane = total * heads * p.dim;
    if (i * 8 >= plane) return;
    const int64_t at = i / (p.dim / 8), row = at / heads;                    // at: (row, head)
    const float* from = p.part + (blockIdx.y ? p.splits * plane : 0) + i * 8;
    E* out = (E*)(blockIdx.y ? out1 : out0) + i * 8;
    float o[8], mul = blockIdx.y ? mul1 : mul0;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.f;
    const bool in = row >= offsets[0] && row < offsets[p.batch];
    const float2* stats = nullptr;
    float top = -__builtin_inff(), sum = 0.f;
    if constexpr (SOFTMAX) {
        stats = p.part_stats + (at - row * heads) * total + row;
        if (in)
            for (int s = 0; s < p.splits; ++s) top = fmaxf(top, stats[s * heads * total].x);
        if (top == -__builtin_inff()) top = 0.f;                             // (no visible key: every sum is 0)
    }
    if (in)
        for (int s = 0; s < p.splits; ++s) {
            const f4 x = *(const f4*)(from + s * plane), y = *(const f4*)(from + s * plane + 4);
            float less = 1.f;
            if constexpr (SOFTMAX) {
                const float2 st = stats[s * heads * total];
                less = exp2_fast(st.x - top);
                sum = __builtin_fmaf(less, st.y, sum);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { o[j] = __builtin_fmaf(less, x[j], o[j]); o[4 + j] = __builtin_fmaf(less, y[j], o[4 + j]); }
        }
    if constexpr (SOFTMAX) {
        const bool none = !in || sum == 0.f;
        mul = none ? 0.f : mul0 / sum;
        if (in && i % (p.dim / 8) == 0) p.lse[(at - row * heads) * total + row] = none ? __builtin_inff() : top + log2f(sum);
        if (none)
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] *= mul;
    if constexpr (sizeof(E) == 2) store_n<T, 8>(out, o);
    else { store_n<T, 4>(out, (const float(&)[4])o[0]); store_n<T, 4>(out + 4, (const float(&)[4])o[4]); }
    if constexpr (SOFTMAX && Rest<T>::ON)
        if (p.out_rest) {                                                    // (places: those of the kernel's DP, which is 64 or 128)
            const int k = (int)(i % (p.dim / 8)), d = k >> 2, c = k & 3;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int word = p.dim <= 64 ? rest_word<T, 64>(d, c, g) : rest_word<T, 128>(d, c, g);
                *(uint32_t*)(p.out_rest + at * (p.dim <= 64 ? 64 : 128) + 4 * word) = rest4<T>(o + 4 * g);
            }
        }
}

// ---- launches ----
// Where the host knows the longest sequence badly, most of tiles x heads x sequences hold nothing: beyond 2^20 of them (four for each wave that the chip holds) a
// workgroup walks several tiles of its sequence.
static inline int attention_blocks(AttnP& p, int64_t tiles, int heads) {
    const int64_t pairs = ((int64_t)p.splits * heads * p.batch + 7) / 8 * 8;
    if (pairs > (1 << 23)) return -1;                                        // (a launch takes 2^32 threads)
    if (tiles * pairs > (1 << 20)) tiles = pairs < (1 << 20) ? (1 << 20) / pairs : 1;
    const int64_t n = tiles * pairs;
    p.tiles = (int)tiles;
    p.blocks = (int)n;
    return 0;
}
static constexpr int GAP_BLOCKS = 8;                    // blocks that clear the rows of no sequence (usually there are none)

// ---- how many workgroups share a walk ----
// A few long sequences, or a key head that many query heads read, make too few workgroups for 256 CUs: their walks are split, and a second launch joins the
// parts' fp32 sums. The number of parts is the one with the least estimated time, from microseconds measured: a walked tile where a workgroup has its CU to itself
// and where the CU is full, a workgroup's start and end, the join, and the parts, written and read. (us, unsplit and split with the join: one sequence
// of 4000 tokens, 2 heads of 64, bf16: forward 68 -> 29, dq 81 -> 33, dkv 105 -> 38; dkv of 4 sequences of 300 .. 500 tokens, 8 query heads on one key head: 99 -> 24; of
// 12 ragged ones, 16 heads on 4 of 128, fp32: 307 -> 235; forward of 512 and 300 tokens, 12 heads of 64: 12.7 -> 18.5, so not there.)
enum Walk { FORWARD, DQ, DKV };
template <class T, int DP> static int attention_splits(Walk w, const AttnP& p, int64_t max_q, int64_t max_k) {
    typedef Geo<T, DP> G;
    const double size = G::SZ == 4 ? 2.5 : DP / 64.0, alone = (w == FORWARD ? 0.95 : w == DQ ? 1.25 : 1.5) * size, full = (w == FORWARD ? 0.8 : w == DQ ? 1.0 : 1.25) * size;
    const int64_t owned = w == DKV ? max_k : max_q, walked = w == DKV ? max_q : max_k, heads = w == DKV ? p.kv_heads : p.heads;
    const int64_t own = (owned + 4 * G::R - 1) / (4 * G::R), pairs = heads * p.batch, tiles = (walked + G::WALK - 1) / G::WALK * (w == DKV ? p.heads / p.kv_heads : 1);
    const double part_us = (double)(w == DKV ? 2 * p.total_k * p.kv_heads : p.total_q * p.heads) * p.dim * 8 / 3e6;
    if (pairs == 0) return 1;                                                // no sequences: no walks, only rows to clear
    int best = 1;
    double least = 0;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (s > 1 && (s > tiles || own * pairs * s > 4096)) break;
        // an XCD has 32 CUs and the owned tiles of every eighth of pairs x parts
        const double per = (double)((tiles + s - 1) / s), rounds = (double)(((pairs * s + 7) / 8 * own + 31) / 32);
        double us = rounds * per * full;
        if (us < per * alone) us = per * alone;
        us += 5.0;
        if (s > 1) us += 5.0 + s * part_us;
        if (s == 1 || us < least) { least = us; best = s; }
    }
    return best;
}
static inline size_t attention_part_bytes(Walk w, const AttnP& p, int splits) {
    if (splits < 2) return 0;
    const size_t rows = w == DKV ? 2 * (size_t)p.total_k * p.kv_heads : (size_t)p.total_q * p.heads;
    return splits * rows * (p.dim * sizeof(float) + (w == FORWARD ? sizeof(float2) : 0));
}
static inline void attention_set_parts(Walk w, AttnP& p, int splits, void* ws) {
    p.splits = splits;
    p.part = splits > 1 ? (float*)ws : nullptr;
    p.part_stats = splits > 1 && w == FORWARD ? (float2*)((float*)ws + (size_t)splits * p.total_q * p.heads * p.dim) : nullptr;
}
template <class T, bool SOFTMAX> static int attention_join(const AttnP& p, const int32_t* offsets, int64_t total, int heads, unsigned char* out0, float mul0,
                                                           unsigned char* out1, float mul1, hipStream_t stream) {
    const int64_t threads = total * heads * (p.dim / 8);
    if (threads == 0) return 0;
    hipLaunchKernelGGL((attention_join_kernel<T, SOFTMAX>), dim3((unsigned)((threads + 255) / 256), out1 ? 2 : 1), dim3(256), 0, stream, p, offsets, total, heads, out0,
                       mul0, out1, mul1);
    return (int)hipGetLastError();
}

template <class K> static int attention_launch(K kernel, const AttnP& p, int threads, int lds, hipStream_t stream) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3(p.blocks + (p.splits > 1 ? 0 : GAP_BLOCKS)), dim3(threads), lds, stream, p);
    return (int)hipGetLastError();
}
static constexpr int NW = 4;                            // waves of a workgroup
template <class T, int DP, bool KEEP, bool MASK> static int attention_forward_dp(AttnP p, int max_q, int max_k, void* ws, hipStream_t stream) {
    typedef Geo<T, DP> G;
    attention_set_parts(FORWARD, p, attention_splits<T, DP>(FORWARD, p, max_q, max_k), ws);
    if (attention_blocks(p, (max_q + NW * G::R - 1) / (NW * G::R), p.heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    const int rc = attention_launch(attention_forward_kernel<T, DP, NW, KEEP, MASK>, p, NW * 64, G::LDS + 8 * G::WALK, stream);
    return rc || p.splits == 1 ? rc : attention_join<T, true>(p, p.q_offsets, p.total_q, p.heads, p.out, KEEP ? p.keep_scale : 1.f, nullptr, 0.f, stream);
}
template <class T, int DP, bool KEEP, bool MASK> static int attention_backward_dp(AttnP p, int max_q, int max_k, void* ws, hipStream_t stream) {
    typedef Geo<T, DP> G;
    attention_set_parts(DQ, p, attention_splits<T, DP>(DQ, p, max_q, max_k), ws);
    if (attention_blocks(p, (max_q + NW * G::R - 1) / (NW * G::R), p.heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    int rc = attention_launch(attention_dq_kernel<T, DP, NW, KEEP, MASK>, p, NW * 64, G::LDS + 8 * G::WALK, stream);
    if (!rc && p.splits > 1) rc = attention_join<T, false>(p, p.q_offsets, p.total_q, p.heads, p.dq, p.scale, nullptr, 0.f, stream);
    if (rc) return rc;
    attention_set_parts(DKV, p, attention_splits<T, DP>(DKV, p, max_q, max_k), ws);      // (dq's parts are done with)
    if (attention_blocks(p, (max_k + NW * G::R - 1) / (NW * G::R), p.kv_heads)) return ATLAS_TRAIN_E_UNSUPPORTED;
    rc = attention_launch(attention_dkv_kernel<T, DP, NW, KEEP, MASK>, p, NW * 64, G::LDS + 16 * G::WALK + (KEEP ? NW * G::R / 4 * G::WALK : 0), stream);
    return rc || p.splits == 1 ? rc : attention_join<T, false>(p, p.k_offsets, p.total_k, p.kv_heads, p.dk, p.scale, p.dv, KEEP ? p.keep_scale : 1.f, stream);
}
// dropout and key masks each cost instructions on every score: a call without them runs code without them
template <class T, int DP> static int attention_forward_m(const AttnP& p, int max_q, int max_k, void* ws, hipStream_t s) {
    if (p.key_mask) return p.keep ? attention_forward_dp<T, DP, true, true>(p, max_q, max_k, ws, s) : attention_forward_dp<T, DP, false, true>(p, max_q, max_k, ws, s);
    return p.keep ? attention_forward_dp<T, DP, true, false>(p, max_q, max_k, ws, s) : attention_forward_dp<T, DP, false, false>(p, max_q, max_k, ws, s);
}
template <class T, int DP> static int attention_backward_m(const AttnP& p, int max_q, int max_k, void* ws, hipStream_t s) {
    if (p.key_mask)
        return p.keep_bits ? attention_backward_dp<T, DP, true, true>(p, max_q, max_k, ws, s) : attention_backward_dp<T, DP, false, true>(p, max_q, max_k, ws, s);
    return p.keep_bits ? attention_backward_dp<T, DP, true, false>(p, max_q, max_k, ws, s) : attention_backward_dp<T, DP, false, false>(p, max_q, max_k, ws, s);
}
template <class T> int attention_forward_t(const AttnP& p, int max_q, int max_k, void* ws, hipStream_t s) {
    return p.dim <= 64 ? attention_forward_m<T, 64>(p, max_q, max_k, ws, s) : attention_forward_m<T, 128>(p, max_q, max_k, ws, s);
}
template <class T> int attention_backward_t(const AttnP& p, int max_q, int max_k, void* ws, hipStream_t s) {
    return p.dim <= 64 ? attention_backward_m<T, 64>(p, max_q, max_k, ws, s) : attention_backward_m<T, 128>(p, max_q, max_k, ws, s);
}
template <class T, int DP> static size_t attention_bytes_dp(const AttnP& p, int max_q, int max_k, bool backward) {
    const auto need = [&](Walk w) { return attention_part_bytes(w, p, attention_splits<T, DP>(w, p, max_q, max_k)); };
    if (!backward) return need(FORWARD);
    const size_t a = need(DQ), b = need(DKV);
    return a > b ? a : b;
}
template <class T> size_t attention_bytes(const AttnP& p, int max_q, int max_k, bool backward) {
    return p.dim <= 64 ? attention_bytes_dp<T, 64>(p, max_q, max_k, backward) : attention_bytes_dp<T, 128>(p, max_q, max_k, backward);
}

}  // namespace atlas_train
