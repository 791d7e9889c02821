// rows.hip -- the training kernels that are one pass over rows: 8-bit activations, the dense layer's dz and bias gradient, layer norm, and the sums of
// fp32 partial results; and the C entries of the whole library (include/atlas_train.h). Everything here is bound by the bytes it moves.
#include "attention.h"
#include "gemm.h"

namespace atlas_train {

static inline int64_t up32(int64_t n) { return (n + 31) / 32 * 32; }

// ---- 8-bit activations ----
// A thread takes 8 consecutive values, four threads a group of 32. x is read 16 bytes (16-bit types) or 32 bytes (fp32) at a time.
template <class T, bool VEC> __global__ void __launch_bounds__(256)
compress_kernel(const typename T::elem* __restrict__ x, int64_t ldx, int64_t m, int n, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int per_row = (n + 31) / 32 * 4;                                   // threads of a row
    const int64_t all = m * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int t = (int)(i - row * per_row), c = 8 * t;
        float v[8];
        if (VEC && c + 8 <= n) {
            float a[4], b[4];
            if constexpr (sizeof(typename T::elem) == 2) load_n<T, 8>(x + row * ldx + c, v);
            else {
                load_n<T, 4>(x + row * ldx + c, a); load_n<T, 4>(x + row * ldx + c + 4, b);
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
            }
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < n ? T::ld(x[row * ldx + c + j]) : 0.f;
        const GroupPower e = group_power4<8>(v);                                    // the group's four threads are in the loop together: 64 is a multiple of 4, and so is `all`
        uint32_t w[2];
        encode<8>(v, e, TopPower<T>::E, w);
        *(uint2*)(codes + row * (per_row * 8) + c) = make_uint2(w[0], w[1]);
        if ((t & 3) == 0) scales[row * (per_row / 4) + t / 4] = (uint8_t)(e.e + 127);
    }
}
template <class T, bool VEC> __global__ void __launch_bounds__(256)
decompress_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t m, int n, typename T::elem* __restrict__ out) {
    const int per_row = (n + 7) / 8, groups = (n + 31) / 32;
    const int64_t all = m * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int t = (int)(i - row * per_row), c = 8 * t;
        const uint2 w = *(const uint2*)(codes + row * groups * 32 + c);
        const float s = power_of((int)scales[row * groups + t / 4] - 127);
        float a[4], b[4];
        values4(w.x, s, a); values4(w.y, s, b);
        typename T::elem* to = out + row * n + c;
        if constexpr (VEC) {
            if constexpr (sizeof(typename T::elem) == 2) *(u4*)to = (u4){pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3])};
            else { store_n<T, 4>(to, a); store_n<T, 4>(to + 4, b); }
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < n) to[j] = T::st(j < 4 ? a[j & 3] : b[j & 3]);
    }
}

// ---- fp32 partial sums of columns -> element type: out[c] = sum over p of part[p][c], for one or two planes of parts ----
// 16 threads a column, each every 16th part, joined in a fixed order (one thread a column took 86 us
// for 341 x 768: a chain of dependent loads on three workgroups)
template <class T> __global__ void __launch_bounds__(256)
sum_many_parts_kernel(const float* __restrict__ part, int parts, int n, typename T::elem* __restrict__ out, typename T::elem* __restrict__ second) {
    if (blockIdx.y) { part += (int64_t)parts * n; out = second; }
    __shared__ float sh[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, c = blockIdx.x * 16 + tx;
    float s = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int p = ty; p < parts; p += 16) s += part[(int64_t)p * n + c];
    }
    sh[ty][tx] = s;
    __syncthreads();
    if (ty != 0 || c >= n) return;
    float t = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) t += sh[y][tx];
    out[c] = T::st(t);
}

// ---- sums over rows: a workgroup takes 128 columns (32 threads x 4) of a run of rows, 8 rows at a time ----
// (up to 64 rows in one run: 41 x 768 bf16 dz takes 6.1 us where three runs take 4.2 and their sum 2.4, and a launch of some 2 us of host time is saved)
static constexpr int COL_W = 128, ROWS_MIN = 16, PARTS_MAX = 512, ROWS_ALONE = 64;
static inline int column_parts(int64_t m, int n) {
    const int64_t strips = (n + COL_W - 1) / COL_W;
    int64_t p = 2048 / (strips > 0 ? strips : 1);
    const int64_t most = (m + ROWS_MIN - 1) / ROWS_MIN;
    if (p > most) p = most;
    if (p > PARTS_MAX) p = PARTS_MAX;
    return p < 1 || m <= ROWS_ALONE ? 1 : (int)p;
}
// (a lone part is the sum: it goes to the outputs `whole`)
template <class T, int NS> static __device__ __forceinline__ void strip_sums(float (&s)[NS][4], float* __restrict__ part, int64_t plane, int n, int c,
                                                                             typename T::elem* const (&whole)[NS]) {
    __shared__ float sh[8][NS * 4 * 32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < NS; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) sh[ty][(k * 4 + j) * 32 + tx] = s[k][j];
    __syncthreads();
    if (ty != 0) return;
#pragma unroll
    for (int k = 0; k < NS; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float t = 0.f;
#pragma unroll
            for (int y = 0; y < 8; ++y) t += sh[y][(k * 4 + j) * 32 + tx];
            if (c + j >= n) continue;
            if (gridDim.y == 1) whole[k][c + j] = T::st(t);
            else part[k * plane + (int64_t)blockIdx.y * n + c + j] = t;
        }
}
template <class T> static __device__ __forceinline__ void load4_guarded(const typename T::elem* p, int left, float (&v)[4]) {
    if (left >= 4) { load4_any<T>(p, v); return; }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? T::ld(p[j]) : 0.f;
}

// dz = dy * keep * act'(z) and its column sums. The sums are of the fp32 values; dz is rounded to the tensors' type, because it is an operand of the matrix instructions
// of dx and dW (each value by at most half a step, of either sign: dx and dW of 16 bits are off by 1.4 of their own rounding, bf16 0.0024 for 0.0017)
template <class T> __global__ void __launch_bounds__(256)
linear_dz_kernel(const typename T::elem* __restrict__ dy, int64_t ld_dy, const typename T::elem* __restrict__ z, const uint8_t* __restrict__ zc,
                 const uint8_t* __restrict__ zs, const uint8_t* __restrict__ keep, float keep_scale, int64_t m, int n, typename T::elem* __restrict__ dz,
                 float* __restrict__ part, typename T::elem* __restrict__ db) {
    const int c = blockIdx.x * COL_W + (threadIdx.x & 31) * 4, left = n - c;
    const int64_t per = (m + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < m ? r0 + per : m;
    const int groups = (n + 31) / 32;
    float s[1][4] = {{0.f, 0.f, 0.f, 0.f}};
    if (left > 0)
        for (int64_t r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
            float g[4];
            load4_guarded<T>(dy + r * ld_dy + c, left, g);
            if (keep) {
                const uint8_t* k = keep + r * n + c;
                if (left >= 4) {
                    const uint32_t w = *(const u32_any*)k;
#pragma unroll
                    for (int j = 0; j < 4; ++j) g[j] = w >> (8 * j) & 0xffu ? g[j] * keep_scale : 0.f;
                } else
#pragma unroll
                    for (int j = 0; j < 4; ++j) g[j] = j < left && k[j] ? g[j] * keep_scale : 0.f;
            }
            if (z || zc) {
                float v[4];
                if (zc) values4(*(const uint32_t*)(zc + r * groups * 32 + c), power_of((int)zs[r * groups + c / 32] - 127), v);
                else load4_guarded<T>(z + r * n + c, left, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] *= gelu_slope(v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0][j] += g[j];
            if (dz) {
                typename T::elem* to = dz + r * n + c;
                if (left >= 4) store4_any<T>(to, g);
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j < left) to[j] = T::st(g[j]);
            }
        }
    typename T::elem* const whole[1] = {db};
    if (db) strip_sums<T, 1>(s, part, 0, n, c, whole);
}

// ---- layer norm ----
// dx = r (g - mean(g) - (r x) mean(r g (x - mu))): the scale r of a row may be anything, r^3 leaves fp32 from r = 10^12.8 and 10^-12.6 on
// one wave per row; the row is read twice (statistics, then the result: the second time from the cache)
template <class T, bool VEC> __global__ void __launch_bounds__(256)
layer_norm_kernel(const typename T::elem* __restrict__ x, int64_t ldx, const typename T::elem* __restrict__ w, const typename T::elem* __restrict__ b, float eps,
                  int64_t m, int n, typename T::elem* __restrict__ y, float* __restrict__ stats) {
    constexpr int NV = VEC ? T::EPC : 1;
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < m; r += (int64_t)gridDim.x * 4) {
        const typename T::elem* xr = x + r * ldx;
        float s = 0.f, s2 = 0.f;
        for (int c = lane * NV; c < n; c += 64 * NV) {
            float v[NV];
            load_n<T, NV>(xr + c, v);
#pragma unroll
            for (int j = 0; j < NV; ++j) { s += v[j]; s2 = __builtin_fmaf(v[j], v[j], s2); }
        }
        s = wave_sum(s); s2 = wave_sum(s2);
        const float mu = s / (float)n, rs = 1.0f / sqrtf(s2 / (float)n + eps);
        if (lane == 0) *(float2*)(stats + 2 * r) = make_float2(mu, rs);
        for (int c = lane * NV; c < n; c += 64 * NV) {
            float v[NV], ww[NV], bb[NV];
            load_n<T, NV>(xr + c, v); load_n<T, NV>(w + c, ww); load_n<T, NV>(b + c, bb);
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = __builtin_fmaf(ww[j] * (v[j] - mu), rs, bb[j]);
            store_n<T, NV>(y + r * n + c, v);
        }
    }
}
template <class T, bool VEC> __global__ void __launch_bounds__(256)
layer_norm_dx_kernel(const typename T::elem* __restrict__ x, int64_t ldx, const typename T::elem* __restrict__ w, const float* __restrict__ stats,
                     const typename T::elem* __restrict__ dy, int64_t ldy, int64_t m, int n, typename T::elem* __restrict__ dx) {
    constexpr int NV = VEC ? T::EPC : 1;
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < m; r += (int64_t)gridDim.x * 4) {
        const typename T::elem *xr = x + r * ldx, *dr = dy + r * ldy;
        const float2 st = *(const float2*)(stats + 2 * r);
        float s = 0.f, s2 = 0.f;
        for (int c = lane * NV; c < n; c += 64 * NV) {
            float v[NV], ww[NV], d[NV];
            load_n<T, NV>(xr + c, v); load_n<T, NV>(w + c, ww); load_n<T, NV>(dr + c, d);
#pragma unroll
            for (int j = 0; j < NV; ++j) { const float g = ww[j] * d[j]; s += g; s2 = __builtin_fmaf(g, v[j] - st.x, s2); }
        }
        const float gm = wave_sum(s) / (float)n, gx = wave_sum(s2) / (float)n * st.y;
        for (int c = lane * NV; c < n; c += 64 * NV) {
            float v[NV], ww[NV], d[NV];
            load_n<T, NV>(xr + c, v); load_n<T, NV>(w + c, ww); load_n<T, NV>(dr + c, d);
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = st.y * __builtin_fmaf(-v[j] * st.y, gx, ww[j] * d[j] - gm);
            store_n<T, NV>(dx + r * n + c, v);
        }
    }
}
// both at once where a row fits the registers of a wave (n <= CH * 64 chunks): x and dy are read once; a wave walks rows and keeps the sums of its own
// columns, a workgroup joins its four waves' sums in a fixed order. Bound by memory: 61 441 x 768 bf16 in 64 us = 4.4 TB/s; without the prefetch of
// the next row 89 us, as two kernels (dx, then dw and db) 83 us
static constexpr int LN_BLOCKS = 1024;
static inline int layer_norm_parts(int64_t m) { return (int)(m / 16 < 1 ? 1 : m / 16 > LN_BLOCKS ? LN_BLOCKS : m / 16); }      // at least four rows a wave
template <class T, int CH> __global__ void __launch_bounds__(256)
layer_norm_backward_kernel(const typename T::elem* __restrict__ x, int64_t ldx, const typename T::elem* __restrict__ w, const float* __restrict__ stats,
                           const typename T::elem* __restrict__ dy, int64_t ldy, int64_t m, int n, typename T::elem* __restrict__ dx, float* __restrict__ part,
                           typename T::elem* __restrict__ dw, typename T::elem* __restrict__ db) {
    constexpr int NV = T::EPC;
    extern __shared__ float sh[];                                            // [4][2][n]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float ww[CH][NV], sw[CH][NV], sb[CH][NV];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = (i * 64 + lane) * NV;
#pragma unroll
        for (int j = 0; j < NV; ++j) ww[i][j] = sw[i][j] = sb[i][j] = 0.f;
        if (c < n) load_n<T, NV>(w + c, ww[i]);
    }
    u4 xn[CH], dn[CH];                                                       // the next row is on its way while this one is summed
    float2 sn = make_float2(0.f, 0.f);
    auto fetch = [&](int64_t r) {
        sn = *(const float2*)(stats + 2 * r);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = (i * 64 + lane) * NV;
            xn[i] = dn[i] = (u4){0, 0, 0, 0};
            if (c < n) { xn[i] = *(const u4*)(x + r * ldx + c); dn[i] = *(const u4*)(dy + r * ldy + c); }
        }
    };
    const int64_t step = (int64_t)gridDim.x * 4;
    int64_t r = (int64_t)blockIdx.x * 4 + wave;
    if (r < m) fetch(r);
    for (; r < m; r += step) {
        const float2 st = sn;
        float v[CH][NV], d[CH][NV], s = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) { unpack<T>(xn[i], v[i]); unpack<T>(dn[i], d[i]); }
        if (r + step < m) fetch(r + step);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NV; ++j) {                                   // (columns behind the row's end: w and dy are 0 there)
                const float g = ww[i][j] * d[i][j], cen = v[i][j] - st.x;
                s += g;
                s2 = __builtin_fmaf(g, cen, s2);
                sw[i][j] = __builtin_fmaf(d[i][j] * st.y, cen, sw[i][j]);
                sb[i][j] += d[i][j];
            }
        if (dx) {
            const float gm = wave_sum(s) / (float)n, gx = wave_sum(s2) / (float)n * st.y;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int c = (i * 64 + lane) * NV;
#pragma unroll
                for (int j = 0; j < NV; ++j) v[i][j] = st.y * __builtin_fmaf(-v[i][j] * st.y, gx, ww[i][j] * d[i][j] - gm);
                if (c < n) store_n<T, NV>(dx + r * n + c, v[i]);
            }
        }
    }
    if (!dw) return;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = (i * 64 + lane) * NV;
        if (c < n)
#pragma unroll
            for (int j = 0; j < NV; ++j) { sh[wave * 2 * n + c + j] = sw[i][j]; sh[(wave * 2 + 1) * n + c + j] = sb[i][j]; }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * n; c += 256) {                         // part: [2][blocks][n]
        const float t = (sh[c] + sh[2 * n + c]) + (sh[4 * n + c] + sh[6 * n + c]);
        if (gridDim.x == 1) (c < n ? dw : db - n)[c] = T::st(t);
        else part[c < n ? (int64_t)blockIdx.x * n + c : ((int64_t)gridDim.x + blockIdx.x) * n + c - n] = t;
    }
}

template <class T> __global__ void __launch_bounds__(256)
layer_norm_dwb_kernel(const typename T::elem* __restrict__ x, int64_t ldx, const float* __restrict__ stats, const typename T::elem* __restrict__ dy, int64_t ldy,
                      int64_t m, int n, float* __restrict__ part, typename T::elem* __restrict__ dw, typename T::elem* __restrict__ db) {
    const int c = blockIdx.x * COL_W + (threadIdx.x & 31) * 4, left = n - c;
    const int64_t per = (m + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < m ? r0 + per : m;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (left > 0)
        for (int64_t r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
            float v[4], d[4];
            const float2 st = *(const float2*)(stats + 2 * r);
            load4_guarded<T>(x + r * ldx + c, left, v);
            load4_guarded<T>(dy + r * ldy + c, left, d);
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[0][j] = __builtin_fmaf(d[j] * st.y, v[j] - st.x, s[0][j]); s[1][j] += d[j]; }
        }
    typename T::elem* const whole[2] = {dw, db};
    strip_sums<T, 2>(s, part, (int64_t)gridDim.y * n, n, c, whole);
}

// ---- host side ----
static inline bool aligned(const void* p, int64_t ld, int bytes_per_access, int size) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & (bytes_per_access - 1)) == 0; }
static inline unsigned capped(int64_t blocks, int64_t most) { return (unsigned)(blocks < 1 ? 1 : blocks > most ? most : blocks); }

template <class T> static int sum_columns(const float* part, int parts, int n, void* out, void* second, hipStream_t s) {
    typedef typename T::elem E;
    if (parts == 1) return 0;
    hipLaunchKernelGGL((sum_many_parts_kernel<T>), dim3((n + 15) / 16, second ? 2 : 1), dim3(256), 0, s, part, parts, n, (E*)out, (E*)second);
    return (int)hipGetLastError();
}
template <class T> static int compress_t(const void* x, int64_t ldx, int64_t m, int n, uint8_t* codes, uint8_t* scales, hipStream_t s) {
    typedef typename T::elem E;
    const unsigned blocks = capped((m * ((n + 31) / 32 * 4) + 255) / 256, 1 << 20);
    if (aligned(x, ldx, 16, sizeof(E))) hipLaunchKernelGGL((compress_kernel<T, true>), dim3(blocks), dim3(256), 0, s, (const E*)x, ldx, m, n, codes, scales);
    else hipLaunchKernelGGL((compress_kernel<T, false>), dim3(blocks), dim3(256), 0, s, (const E*)x, ldx, m, n, codes, scales);
    return (int)hipGetLastError();
}
template <class T> static int decompress_t(const uint8_t* codes, const uint8_t* scales, int64_t m, int n, void* out, hipStream_t s) {
    typedef typename T::elem E;
    const unsigned blocks = capped((m * ((n + 7) / 8) + 255) / 256, 1 << 20);
    if (n % 8 == 0 && ((uintptr_t)out & 15) == 0) hipLaunchKernelGGL((decompress_kernel<T, true>), dim3(blocks), dim3(256), 0, s, codes, scales, m, n, (E*)out);
    else hipLaunchKernelGGL((decompress_kernel<T, false>), dim3(blocks), dim3(256), 0, s, codes, scales, m, n, (E*)out);
    return (int)hipGetLastError();
}
template <class T> static int linear_dz_t(const void* dy, int64_t ld, const void* z, const uint8_t* zc, const uint8_t* zs, const uint8_t* keep, float ks, int64_t m, int n,
                                          void* dz, void* db, float* ws, hipStream_t s) {
    typedef typename T::elem E;
    const int parts = column_parts(m, n);
    hipLaunchKernelGGL((linear_dz_kernel<T>), dim3((n + COL_W - 1) / COL_W, parts), dim3(256), 0, s, (const E*)dy, ld, (const E*)z, zc, zs, keep, ks, m, n, (E*)dz,
                       ws, (E*)db);
    const int rc = (int)hipGetLastError();
    return rc || !db ? rc : sum_columns<T>(ws, parts, n, db, nullptr, s);
}
template <class T> static int ln_fwd_t(const void* x, int64_t ldx, const void* w, const void* b, float eps, int64_t m, int n, void* y, float* stats, hipStream_t s) {
    typedef typename T::elem E;
    const dim3 grid(capped((m + 3) / 4, 1 << 22));                           // (a launch takes 2^32 threads)
    if (n % T::EPC == 0 && aligned(x, ldx, 16, sizeof(E)) && (((uintptr_t)w | (uintptr_t)b | (uintptr_t)y) & 15) == 0)
        hipLaunchKernelGGL((layer_norm_kernel<T, true>), grid, dim3(256), 0, s, (const E*)x, ldx, (const E*)w, (const E*)b, eps, m, n, (E*)y, stats);
    else
        hipLaunchKernelGGL((layer_norm_kernel<T, false>), grid, dim3(256), 0, s, (const E*)x, ldx, (const E*)w, (const E*)b, eps, m, n, (E*)y, stats);
    return (int)hipGetLastError();
}
template <class T> static int ln_bwd_t(const void* x, int64_t ldx, const void* w, const float* stats, const void* dy, int64_t ldy, int64_t m, int n, void* dx, void* dw,
                                       void* db, float* ws, hipStream_t s) {
    typedef typename T::elem E;
    const int chunks = (n + 64 * T::EPC - 1) / (64 * T::EPC);
    if (m > 0 && chunks <= 4 && n % T::EPC == 0 && aligned(x, ldx, 16, sizeof(E)) && aligned(dy, ldy, 16, sizeof(E)) && (((uintptr_t)w | (uintptr_t)dx) & 15) == 0) {
        const int parts = layer_norm_parts(m);
        const dim3 grid(parts);
        const size_t lds = dw ? (size_t)8 * n * 4 : 0;
        if (chunks == 1) hipLaunchKernelGGL((layer_norm_backward_kernel<T, 1>), grid, dim3(256), lds, s, (const E*)x, ldx, (const E*)w, stats, (const E*)dy, ldy, m, n, (E*)dx, ws, (E*)dw, (E*)db);
        else if (chunks == 2) hipLaunchKernelGGL((layer_norm_backward_kernel<T, 2>), grid, dim3(256), lds, s, (const E*)x, ldx, (const E*)w, stats, (const E*)dy, ldy, m, n, (E*)dx, ws, (E*)dw, (E*)db);
        else hipLaunchKernelGGL((layer_norm_backward_kernel<T, 4>), grid, dim3(256), lds, s, (const E*)x, ldx, (const E*)w, stats, (const E*)dy, ldy, m, n, (E*)dx, ws, (E*)dw, (E*)db);
        const int rc = (int)hipGetLastError();
        return rc || !dw ? rc : sum_columns<T>(ws, parts, n, dw, db, s);
    }
    if (dx) {
        const dim3 grid(capped((m + 3) / 4, 1 << 22));
        if (m > 0) {
            if (n % T::EPC == 0 && aligned(x, ldx, 16, sizeof(E)) && aligned(dy, ldy, 16, sizeof(E)) && (((uintptr_t)w | (uintptr_t)dx) & 15) == 0)
                hipLaunchKernelGGL((layer_norm_dx_kernel<T, true>), grid, dim3(256), 0, s, (const E*)x, ldx, (const E*)w, stats, (const E*)dy, ldy, m, n, (E*)dx);
            else
                hipLaunchKernelGGL((layer_norm_dx_kernel<T, false>), grid, dim3(256), 0, s, (const E*)x, ldx, (const E*)w, stats, (const E*)dy, ldy, m, n, (E*)dx);
            if (int rc = (int)hipGetLastError()) return rc;
        }
    }
    if (!dw) return 0;
    const int parts = column_parts(m, n);
    hipLaunchKernelGGL((layer_norm_dwb_kernel<T>), dim3((n + COL_W - 1) / COL_W, parts), dim3(256), 0, s, (const E*)x, ldx, stats, (const E*)dy, ldy, m, n, ws, (E*)dw, (E*)db);
    const int rc = (int)hipGetLastError();
    return rc ? rc : sum_columns<T>(ws, parts, n, dw, db, s);
}

static inline bool known(int dtype) { return dtype == ATLAS_TRAIN_F16 || dtype == ATLAS_TRAIN_F32 || dtype == ATLAS_TRAIN_BF16; }
static inline int size_of(int dtype) { return dtype == ATLAS_TRAIN_F32 ? 4 : 2; }
#define BY_TYPE(dtype, call) ((dtype) == ATLAS_TRAIN_F16 ? call(F16) : (dtype) == ATLAS_TRAIN_BF16 ? call(BF16) : call(F32))

extern template int attention_forward_t<F16>(const AttnP&, int, int, void*, hipStream_t);
extern template int attention_forward_t<BF16>(const AttnP&, int, int, void*, hipStream_t);
extern template int attention_forward_t<F32>(const AttnP&, int, int, void*, hipStream_t);
extern template int attention_backward_t<F16>(const AttnP&, int, int, void*, hipStream_t);
extern template size_t attention_bytes<F16>(const AttnP&, int, int, bool);
extern template int attention_backward_t<BF16>(const AttnP&, int, int, void*, hipStream_t);
extern template size_t attention_bytes<BF16>(const AttnP&, int, int, bool);
extern template int attention_backward_t<F32>(const AttnP&, int, int, void*, hipStream_t);
extern template size_t attention_bytes<F32>(const AttnP&, int, int, bool);
extern template int gemm_t<F16>(GemmP, bool, bool, hipStream_t);
extern template int gemm_t<BF16>(GemmP, bool, bool, hipStream_t);
extern template int gemm_t<F32>(GemmP, bool, bool, hipStream_t);
extern template int gemm_splits<F16>(const GemmP&, bool, bool);
extern template int gemm_splits<BF16>(const GemmP&, bool, bool);
extern template int gemm_splits<F32>(const GemmP&, bool, bool);

// 0, or what is wrong with the arguments that both directions share
static int attention_params(const atlas_attention_args* a, bool backward, AttnP& p) {
    if (!a || !known(a->dtype) || a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->total_q < 0 || a->total_k < 0 || a->max_q < 0 ||
        a->max_k < 0 || !a->q_offsets || !a->k_offsets || !(a->scale > 0.f))
        return ATLAS_TRAIN_E_BADARG;
    if (a->dim <= 0 || a->dim % 8 || a->dim > 128 || a->total_q > 0x7fffff00 || a->total_k > 0x7fffff00) return ATLAS_TRAIN_E_UNSUPPORTED;
    const bool some_q = a->total_q > 0, some_k = a->total_k > 0;
    if ((some_q && (!a->q || !a->out || !a->lse)) || (some_k && (!a->k || !a->v))) return ATLAS_TRAIN_E_BADARG;
    if (backward && ((some_q && (!a->dout || !a->dq || !a->delta)) || (some_k && (!a->dk || !a->dv)))) return ATLAS_TRAIN_E_BADARG;
    if ((a->keep || a->keep_bits) && a->keep_cols < 0) return ATLAS_TRAIN_E_BADARG;
    const int64_t sz = size_of(a->dtype);
    const uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)(a->q_row * sz) | (uintptr_t)(a->q_head * sz) |
                           (uintptr_t)(a->k_row * sz) | (uintptr_t)(a->k_head * sz) | (uintptr_t)(a->v_row * sz) | (uintptr_t)(a->v_head * sz) |
                           (backward ? (uintptr_t)a->dout | (uintptr_t)(a->dout_row * sz) | (uintptr_t)(a->dout_head * sz) | (uintptr_t)a->dq | (uintptr_t)a->dk |
                                           (uintptr_t)a->dv : 0);
    if ((bits | (uintptr_t)a->out_rest) & 15) return ATLAS_TRAIN_E_BADARG;
    const int64_t reach = 1 << 24;                                          // a walked tile's rows within a buffer descriptor's 2^31 bytes
    const int64_t strides[4] = {a->q_row * sz, a->k_row * sz, a->v_row * sz, backward ? a->dout_row * sz : 0};
    for (int64_t s : strides)
        if (s < 0 || s >= reach) return ATLAS_TRAIN_E_UNSUPPORTED;
    if (a->keep && (a->keep_row < 0 || a->keep_row >= 1 << 26)) return ATLAS_TRAIN_E_UNSUPPORTED;      // a wave's rows by 32-bit offsets
    p.q = (const unsigned char*)a->q; p.k = (const unsigned char*)a->k; p.v = (const unsigned char*)a->v; p.dout = (const unsigned char*)a->dout;
    p.out_in = (const unsigned char*)a->out; p.out = (unsigned char*)a->out;
    p.q_row = a->q_row * sz; p.q_head = a->q_head * sz; p.k_row = a->k_row * sz; p.k_head = a->k_head * sz; p.v_row = a->v_row * sz; p.v_head = a->v_head * sz;
    p.do_row = a->dout_row * sz; p.do_head = a->dout_head * sz;
    p.q_offsets = a->q_offsets; p.k_offsets = a->k_offsets; p.total_q = a->total_q; p.total_k = a->total_k;
    p.batch = a->batch; p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->dim; p.keep_cols = a->keep_cols;
    p.key_mask = a->key_mask; p.keep = a->keep; p.keep_row = a->keep_row; p.keep_head = a->keep_head;
    p.keep_bits = a->keep_bits; p.keep_words = (a->keep_cols + 31) / 32;
    p.scale = a->scale; p.keep_scale = a->keep_scale;
    p.dq = (unsigned char*)a->dq; p.dk = (unsigned char*)a->dk; p.dv = (unsigned char*)a->dv; p.lse = a->lse; p.delta = a->delta; p.out_rest = size_of(a->dtype) == 2 ? a->out_rest : nullptr;
    p.tiles = p.blocks = 0;
    p.splits = 1;
    p.part = nullptr;
    p.part_stats = nullptr;
    return 0;
}
static int gemm_check(const atlas_gemm_args* a) {
    if (!a || !known(a->dtype) || a->m < 0 || a->n < 0 || a->k < 0 || a->a_layout < 0 || a->a_layout > 1 || a->b_layout < 0 || a->b_layout > 1 || a->act < 0 || a->act > 1)
        return ATLAS_TRAIN_E_BADARG;
    if (a->a_layout && !a->b_layout) return ATLAS_TRAIN_E_UNSUPPORTED;
    if (a->b_codes && (!a->a_layout || !a->b_scales || a->ldb % 32 || ((uintptr_t)a->b_codes & 15))) return ATLAS_TRAIN_E_BADARG;
    if (a->save_z_codes && (!a->save_z_scales || ((uintptr_t)a->save_z_codes & 15))) return ATLAS_TRAIN_E_BADARG;
    if (a->m && a->n && (!a->c || (a->k && (!a->a || (!a->b && !a->b_codes))))) return ATLAS_TRAIN_E_BADARG;
    return 0;
}
static GemmP gemm_params(const atlas_gemm_args* a) {
    GemmP g = {};
    g.p = (const unsigned char*)a->b; g.q = (const unsigned char*)a->a; g.ldp = a->ldb; g.ldq = a->lda; g.ldc = a->ldc;
    g.m = a->m; g.n = a->n; g.k = a->k; g.codes = a->b_codes; g.scales = a->b_scales;
    g.bias = (const unsigned char*)a->bias; g.act = a->act; g.save_z = (unsigned char*)a->save_z; g.save_codes = a->save_z_codes; g.save_scales = a->save_z_scales;
    g.keep = a->keep; g.keep_scale = a->keep_scale; g.residual = (const unsigned char*)a->residual; g.ld_residual = a->ld_residual; g.c = (unsigned char*)a->c;
    g.part = (float*)a->ws;
    return g;
}
static int gemm_parts(const atlas_gemm_args* a) {
    const GemmP g = gemm_params(a);
#define CALL(T) gemm_splits<T>(g, a->b_layout == 1, a->a_layout == 1)
    return BY_TYPE(a->dtype, CALL);
#undef CALL
}

static size_t attention_need(const atlas_attention_args* a, const AttnP& p, bool backward) {
    const int mq = a->max_q > 0 ? a->max_q : 1, mk = a->max_k > 0 ? a->max_k : 1;
#define CALL(T) attention_bytes<T>(p, mq, mk, backward)
    return BY_TYPE(a->dtype, CALL);
#undef CALL
}

}  // namespace atlas_train

using namespace atlas_train;

extern "C" {

int atlas_train_abi_version(void) { return ATLAS_TRAIN_ABI_VERSION; }

size_t atlas_attention_workspace_bytes(const atlas_attention_args* a, int backward) {
    AttnP p;
    return attention_params(a, backward, p) || (a->total_q == 0 && (!backward || a->total_k == 0)) ? 0 : attention_need(a, p, backward);
}
int atlas_attention_forward(const atlas_attention_args* a, void* stream) {
    AttnP p;
    if (int rc = attention_params(a, false, p)) return rc;
    if (a->total_q == 0) return 0;
    const size_t need = attention_need(a, p, false);
    if (need && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < need)) return ATLAS_TRAIN_E_WORKSPACE;
    const int mq = a->max_q > 0 ? a->max_q : 1, mk = a->max_k > 0 ? a->max_k : 1;
#define CALL(T) attention_forward_t<T>(p, mq, mk, a->ws, (hipStream_t)stream)
    return BY_TYPE(a->dtype, CALL);
#undef CALL
}
int atlas_attention_backward(const atlas_attention_args* a, void* stream) {
    AttnP p;
    if (int rc = attention_params(a, true, p)) return rc;
    if (a->total_q == 0 && a->total_k == 0) return 0;
    const size_t need = attention_need(a, p, true);
    if (need && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < need)) return ATLAS_TRAIN_E_WORKSPACE;
    const int mq = a->max_q > 0 ? a->max_q : 1, mk = a->max_k > 0 ? a->max_k : 1;
#define CALL(T) attention_backward_t<T>(p, mq, mk, a->ws, (hipStream_t)stream)
    return BY_TYPE(a->dtype, CALL);
#undef CALL
}

size_t atlas_gemm_workspace_bytes(const atlas_gemm_args* a) {
    if (gemm_check(a) || !a->m || !a->n) return 0;
    const int parts = gemm_parts(a);
    return parts > 1 ? (size_t)parts * a->m * a->n * 4 : 0;
}
int atlas_gemm(const atlas_gemm_args* a, void* stream) {
    if (int rc = gemm_check(a)) return rc;
    if (!a->m || !a->n) return 0;
    const int parts = gemm_parts(a);
    if (parts > 1 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < (size_t)parts * a->m * a->n * 4)) return ATLAS_TRAIN_E_WORKSPACE;
    const GemmP g = gemm_params(a);
#define CALL(T) gemm_t<T>(g, a->b_layout == 1, a->a_layout == 1, (hipStream_t)stream)
    return BY_TYPE(a->dtype, CALL);
#undef CALL
}

size_t atlas_linear_dz_workspace_bytes(int64_t m, int n) { return m < 0 || n <= 0 ? 0 : (size_t)column_parts(m, n) * n * 4; }
int atlas_linear_dz(const void* dy, int64_t ld_dy, const void* z, const uint8_t* z_codes, const uint8_t* z_scales, const uint8_t* keep, float keep_scale, int64_t m, int n,
                    int dtype, void* dz, void* db, void* ws, size_t ws_bytes, void* stream) {
    if (!known(dtype) || m < 0 || n < 0 || (m && n && !dy) || (z && z_codes) || (z_codes && !z_scales)) return ATLAS_TRAIN_E_BADARG;
    if (!n || (!dz && !db)) return 0;
    if (db && (!ws || ((uintptr_t)ws & 3) || ws_bytes < atlas_linear_dz_workspace_bytes(m, n))) return ATLAS_TRAIN_E_WORKSPACE;
#define CALL(T) linear_dz_t<T>(dy, ld_dy, z, z_codes, z_scales, keep, keep_scale, m, n, dz, db, (float*)ws, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

int atlas_compress(const void* x, int64_t ldx, int64_t m, int n, int dtype, uint8_t* codes, uint8_t* scales, void* stream) {
    if (!known(dtype) || m < 0 || n < 0) return ATLAS_TRAIN_E_BADARG;
    if (!m || !n) return 0;
    if (!x || !codes || !scales || ((uintptr_t)codes & 15)) return ATLAS_TRAIN_E_BADARG;
#define CALL(T) compress_t<T>(x, ldx, m, n, codes, scales, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}
int atlas_decompress(const uint8_t* codes, const uint8_t* scales, int64_t m, int n, int dtype, void* out, void* stream) {
    if (!known(dtype) || m < 0 || n < 0) return ATLAS_TRAIN_E_BADARG;
    if (!m || !n) return 0;
    if (!out || !codes || !scales || ((uintptr_t)codes & 15)) return ATLAS_TRAIN_E_BADARG;
#define CALL(T) decompress_t<T>(codes, scales, m, n, out, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

int atlas_layer_norm_forward(const void* x, int64_t ldx, const void* w, const void* b, float eps, int64_t m, int n, int dtype, void* y, float* stats, void* stream) {
    if (!known(dtype) || m < 0 || n < 0 || !(eps >= 0.f)) return ATLAS_TRAIN_E_BADARG;
    if (!m || !n) return 0;
    if (!x || !w || !b || !y || !stats || ((uintptr_t)stats & 7)) return ATLAS_TRAIN_E_BADARG;
#define CALL(T) ln_fwd_t<T>(x, ldx, w, b, eps, m, n, y, stats, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}
size_t atlas_layer_norm_workspace_bytes(int64_t m, int n) {
    if (m < 0 || n <= 0) return 0;
    const int a = column_parts(m, n), b = layer_norm_parts(m);
    return (size_t)(a > b ? a : b) * n * 8;
}
int atlas_layer_norm_backward(const void* x, int64_t ldx, const void* w, const float* stats, const void* dy, int64_t ld_dy, int64_t m, int n, int dtype, void* dx, void* dw,
                              void* db, void* ws, size_t ws_bytes, void* stream) {
    if (!known(dtype) || m < 0 || n < 0 || (!dw) != (!db) || (m && n && (!x || !w || !stats || !dy))) return ATLAS_TRAIN_E_BADARG;
    if (!n) return 0;
    if (dw && (!ws || ((uintptr_t)ws & 3) || ws_bytes < atlas_layer_norm_workspace_bytes(m, n))) return ATLAS_TRAIN_E_WORKSPACE;
#define CALL(T) ln_bwd_t<T>(x, ldx, w, stats, dy, ld_dy, m, n, dx, dw, db, (float*)ws, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

}  // extern "C"
