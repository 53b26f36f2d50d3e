// Layer norm over the last axis, forward and backward (include/lsdm_hip.h: lsdm_layer_norm, lsdm_layer_norm_backward), gfx950.
//
//   mu = mean x, var = mean (x - mu)^2, rstd = 1 / sqrt(var + eps), h = (x - mu) rstd, y = h w + b
//   g = dy w;  dx = rstd (g - mean g - h mean(g h));  dw = sum_rows dy h;  db = sum_rows dy
//
// Bound by HBM: forward reads x and writes y, backward reads dy and x (or h's 8-bit codes) and writes dx.  A row sits in the registers of NT
// threads (one pass over memory; the variance is taken around the mean, from registers), statistics and sums in fp32.  NT follows the width: 8
// threads for rows of up to 64 columns up to 1024 threads for 16384, so that a lane holds 8 or 16 values.  A work-group walks many rows: the
// parameters stay in registers, and the backward pass adds dw / db per lane over its rows and writes ONE partial row per work-group, joined in
// order by a second launch (no atomics: results do not depend on the schedule).
// A row is read and written in pieces of eight elements (ops.hpp), whatever its width and alignment.  (Beyond 8192 columns the backward kernel keeps up to five
// registers of a thread in scratch memory where the type is fp32 or the width odd.)
// Measured, bf16 (a copy runs at 4.9 TB/s): 32768 x 2048 forward 44.5 us (6.0 TB/s), backward 76 us (5.3), with h in 8 bits 57 and 65 us; 4928 x 771
// forward 7.5 us, backward 20; fp32 32768 x 2048 107 and 148 us.
#include <type_traits>

#include "ops.hpp"
#include "ops_launch.hpp"

namespace lsdm {
namespace ops {

// Sum / maximum over groups of W = 4 .. 64 neighbouring lanes, the result in all of them: within 16 lanes by DPP operands of the addition itself (quad
// permutes, then the mirrored half and full rows), across rows by the 16- and 32-lane swaps.  No LDS round trips (__shfl_xor is one per level).
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int W, class F>
__device__ __forceinline__ unsigned lanes_join(unsigned v, F f) {
    if constexpr (W >= 2) v = f(v, dpp<0xB1>(v));            // lanes 1 0 3 2
    if constexpr (W >= 4) v = f(v, dpp<0x4E>(v));            // lanes 2 3 0 1
    if constexpr (W >= 8) v = f(v, dpp<0x141>(v));           // mirrored within 8
    if constexpr (W >= 16) v = f(v, dpp<0x140>(v));          // mirrored within 16
    if constexpr (W >= 32) { const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false); v = f(r[0], r[1]); }
    if constexpr (W >= 64) { const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false); v = f(r[0], r[1]); }
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    return __builtin_bit_cast(float, lanes_join<W>(__builtin_bit_cast(unsigned, v), [](unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}
template <int W>
__device__ __forceinline__ unsigned lanes_max(unsigned v) { return lanes_join<W>(v, [](unsigned a, unsigned b) { return max(a, b); }); }

// over the NT threads of a row: both sums, or the sum and (MAX) the largest of values >= 0; red: one entry per wave of the work-group
template <int NT, bool MAX = false>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* red, int t) {
    constexpr int W = NT < 64 ? NT : 64;
    a = lanes_sum<W>(a);
    b = MAX ? __builtin_bit_cast(float, lanes_max<W>(__builtin_bit_cast(unsigned, b))) : lanes_sum<W>(b);
    if constexpr (NT > 64) {
        constexpr int NW = NT / 64;
        const int first = (t / NT) * NW;         // the row's waves
        wg_sync();                               // (the previous sums have been read)
        if ((t & 63) == 0) red[t >> 6] = make_float2(a, b);
        wg_sync();
        a = 0.0f; b = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) { a += red[first + i].x; b = MAX ? fmaxf(b, red[first + i].y) : b + red[first + i].y; }
    }
    return make_float2(a, b);
}

// lane l of a row's NT threads holds the pieces of 8 columns l, l + NT, ...  WHOLE: the width is a multiple of 8, so a piece is valid or not as one.
template <int NT>
__device__ __forceinline__ int col_of(int l, int i) { return (l + NT * i) * 8; }

// p: a row that exists (of D elements); n: D, or 0 where the values are not wanted.  The loads stand in no branch -- a lane without a whole piece reads
// the row's first one and drops it -- so that all of a row's are in flight together; only the piece cut short by the row's end takes a branch.
template <class T, int NT, int NV, bool WHOLE>
__device__ __forceinline__ void row_load(const T* p, int D, int n, int l, float (&v)[NV][8]) {
    typedef typename Piece<T>::frag frag;
    typedef typename Piece<T>::mem mem;
    constexpr int H = 8 * (int)sizeof(T) / 16;
    frag raw[NV][H];
    if (WHOLE || D >= 8) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = col_of<NT>(l, i), at = c + 8 <= n ? c : 0;
#pragma unroll
            for (int k = 0; k < H; ++k) raw[i][k] = *reinterpret_cast<const mem*>(p + at + k * (8 / H));
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const bool full = col_of<NT>(l, i) + 8 <= n;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = full ? (float)raw[i][j / (8 / H)][j % (8 / H)] : 0.0f;
    }
    if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = col_of<NT>(l, i);
            if (c < n && c + 8 > n) {
#pragma unroll
                for (int j = 0; j < 8; ++j) if (j < n - c) v[i][j] = (float)p[c + j];
            }
        }
    }
}
template <class T, int NT, int NV, bool WHOLE>
__device__ __forceinline__ void row_store(T* p, int D, int l, const float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = col_of<NT>(l, i);
        if (c < D) {
            if constexpr (WHOLE) store8<true>(p + c, v[i]); else store8n<true>(p + c, D - c, v[i]);
        }
    }
}

// the row's 8-bit checkpoint: a group of 32 columns is four lanes' pieces
template <int NT, int NV, bool WHOLE>
__device__ __forceinline__ void row_encode(const float (&h)[NV][8], int D, int l, signed char* codes, unsigned char* exps) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __builtin_bit_cast(unsigned, h[i][j]) & 0x7fffffffu);   // (order of the bit patterns: NaN is largest)
        const unsigned b = exp8_of_amax(__builtin_bit_cast(float, lanes_max<4>(m)));
        const float inv = exp8_inv(b);
        const int c = col_of<NT>(l, i);
        if (c < D) {
            unsigned q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = (unsigned)code8(h[i][j], inv) & 255u;
            store_codes(codes + c, WHOLE ? 8 : D - c, q);
            if ((l & 3) == 0) exps[c >> 5] = (unsigned char)b;
        }
    }
}
template <int NT, int NV, bool WHOLE>
__device__ __forceinline__ void row_decode(const signed char* codes, const unsigned char* exps, int D, int n, int l, float (&h)[NV][8]) {
    u32x2 w[NV];
    unsigned b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = col_of<NT>(l, i);
        b[i] = exps[c < n ? c >> 5 : 0];
        if (WHOLE || D >= 8) w[i] = *reinterpret_cast<const codes8*>(codes + (c + 8 <= n ? c : 0));
        if constexpr (!WHOLE) { if (c < n && c + 8 > n) w[i] = load_codes(codes + c, n - c); }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const bool any = col_of<NT>(l, i) < n;
        const float s = exp8_step(b[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = any ? (float)((int)(w[i][j >> 2] << (24 - 8 * (j & 3))) >> 24) * s : 0.0f;
    }
}

template <class T, int NT, int NV, bool WHOLE>
__device__ __forceinline__ void param_load(const void* p, int is_f32, float missing, int D, int l, float (&v)[NV][8]) {
    if (p && is_f32) return row_load<float, NT, NV, WHOLE>(static_cast<const float*>(p), D, D, l, v);
    if (p) return row_load<T, NT, NV, WHOLE>(static_cast<const T*>(p), D, D, l, v);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = missing;
}

// a / b, correctly rounded, from the rounded reciprocal of b
__device__ __forceinline__ float over(float a, float b, float inv_b) {
    const float q = a * inv_b;
    return fmaf(fmaf(-q, b, a), inv_b, q);
}

template <class T, int NT, int NV, bool WHOLE>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void norm_fwd_kernel(NormArgs a) {
    constexpr int THREADS = NT > 256 ? NT : 256, RPG = THREADS / NT;
    __shared__ float2 red[THREADS / 64];
    const int t = threadIdx.x, l = t % NT, D = a.D;
    float w[NV][8], b[NV][8];
    param_load<T, NT, NV, WHOLE>(a.w, a.param_f32, 1.0f, D, l, w);
    param_load<T, NT, NV, WHOLE>(a.b, a.param_f32, 0.0f, D, l, b);
    constexpr bool SCALED = !std::is_same<T, _Float16>::value;      // (fp16's squares stay in range)
    const float inv_d = 1.0f / (float)D, root_eps = sqrtf(a.eps), least = a.eps > 0.0f ? 0x1p-126f : 0.0f;
    // (the loop is uniform over the work-group, as its barriers need it: a group of threads without a row left works on zeros and stores nothing)
    for (long long r0 = (long long)blockIdx.x * RPG; r0 < a.rows; r0 += (long long)gridDim.x * RPG) {
        const long long r = r0 + t / NT;
        const bool live = r < a.rows;
        const long long rr = live ? r : a.rows - 1;
        float x[NV][8];
        row_load<T, NT, NV, WHOLE>(static_cast<const T*>(a.x) + rr * a.ldx, D, live ? D : 0, l, x);
        // The row is evaluated times 2^-e, the power of two that brings the larger of max |x| and sqrt(eps) into [1, 2): its squares stay in fp32's range for
        // all finite rows (unscaled they leave it from about 1e17 on, and below 1e-19 where eps does not cover them).  The scaling is exact, so ordinary rows
        // have the bits they have without it.  (The maximum costs bf16 2 .. 6 % of the time, fp32 nothing; a rare second pass over such rows instead cost more
        // in registers: 65536 x 512 bf16 23.0 us without, 24.5 with the maximum, 27 with a second pass.)
        float s = 0.0f, top = 0.0f;
        int e = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s = SCALED ? fmaf(x[i][j], 0x1p-15f, s) : s + x[i][j];      // (2^14 values: the sum stays in range as well)
                if constexpr (SCALED) top = fmaxf(top, fabsf(x[i][j]));
            }
        const float2 first = row_sum2<NT, SCALED>(s, top, red, t);
        float mu = over(first.x, (float)D, inv_d), q = 0.0f, eps = a.eps;
        if constexpr (SCALED) {
            e = min((int)(__builtin_bit_cast(unsigned, fmaxf(first.y, root_eps)) >> 23) - 127, 126);
            e = max(e, -126);
            mu = ldexpf(mu, 15 - e);
            eps = ldexpf(eps, -2 * e);
        }
        const float unit = SCALED ? __builtin_bit_cast(float, (unsigned)(127 - e) << 23) : 1.0f;
        // the mean's own rounding is taken out again: d = the mean of x - mu (a row without spread gives h = 0, not a last bit times 1 / sqrt(eps))
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[i][j] = fmaf(x[i][j], unit, col_of<NT>(l, i) + (WHOLE ? 0 : j) < D ? -mu : 0.0f);      // (columns beyond the row are 0 and stay 0)
                s += x[i][j];
                q = fmaf(x[i][j], x[i][j], q);
            }
        const float2 c = row_sum2<NT>(s, q, red, t);
        const float d = over(c.x, (float)D, inv_d);       // (to the last bit: equal values cancel also where eps is nothing next to them)
        const float scale = 1.0f / sqrtf(fmaxf(fmaxf(fmaf(c.y, inv_d, -d * d), 0.0f) + eps, least)), rstd = SCALED ? ldexpf(scale, -e) : scale;
        mu = SCALED ? ldexpf(mu + d, e) : mu + d;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = (x[i][j] - (col_of<NT>(l, i) + (WHOLE ? 0 : j) < D ? d : 0.0f)) * scale;
        if (a.mean && live && l == 0) a.mean[r] = mu;
        if (a.rstd && live && l == 0) a.rstd[r] = rstd;
        if (a.codes) row_encode<NT, NV, WHOLE>(x, live ? D : 0, l, a.codes + r * D, a.exps + r * ((D + 31) >> 5));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = fmaf(x[i][j], w[i][j], b[i][j]);
        row_store<T, NT, NV, WHOLE>(static_cast<T*>(a.y) + r * D, live ? D : 0, l, x);
    }
}

template <class T, int NT, int NV, bool WHOLE>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void norm_bwd_kernel(NormArgs a) {
    constexpr int THREADS = NT > 256 ? NT : 256, RPG = THREADS / NT, COLS = NT * NV * 8;
    __shared__ float2 red[THREADS / 64];
    __shared__ float join[RPG > 1 ? RPG : 1][RPG > 1 ? COLS + 1 : 1];
    const int t = threadIdx.x, l = t % NT, D = a.D;
    float w[NV][8], dw[NV][8], db[NV][8];
    param_load<T, NT, NV, WHOLE>(a.w, a.param_f32, 1.0f, D, l, w);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.0f;
    const float inv_d = 1.0f / (float)D;
    for (long long r0 = (long long)blockIdx.x * RPG; r0 < a.rows; r0 += (long long)gridDim.x * RPG) {       // (uniform, as above)
        const long long r = r0 + t / NT;
        const bool live = r < a.rows;
        const long long rr = live ? r : a.rows - 1;
        const int n = live ? D : 0;
        float g[NV][8], h[NV][8];
        row_load<T, NT, NV, WHOLE>(static_cast<const T*>(a.dy) + rr * a.lddy, D, n, l, g);
        const float rstd = a.rstd[rr];
        if (a.codes) {
            row_decode<NT, NV, WHOLE>(a.codes + rr * D, a.exps + rr * ((D + 31) >> 5), D, n, l, h);
        } else {
            row_load<T, NT, NV, WHOLE>(static_cast<const T*>(a.x) + rr * a.ldx, D, n, l, h);
            // (x - mu) rstd as (x / 2 - mu / 2) 2 rstd: the same bits, and the difference of two large values stays in range
            const float half = 0.5f * a.mean[rr], twice = 2.0f * rstd;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = fmaf(h[i][j], 0.5f, -half) * twice;        // (columns beyond the row: g = 0 there, so h does not matter)
        }
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
                db[i][j] += g[i][j];
                g[i][j] *= w[i][j];
                s += g[i][j];
                q = fmaf(g[i][j], h[i][j], q);
            }
        if (a.dx) {
            const float2 c = row_sum2<NT>(s, q, red, t);
            const float c1 = c.x * inv_d, c2 = c.y * inv_d;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) g[i][j] = rstd * (g[i][j] - c1 - h[i][j] * c2);
            row_store<T, NT, NV, WHOLE>(static_cast<T*>(a.dx) + r * D, n, l, g);
        }
    }
    if (!a.part) return;
    // one partial row of dw and of db per work-group
    float* out = a.part + (long long)blockIdx.x * 2 * D;
    if constexpr (RPG == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) { const int c = col_of<NT>(l, i) + j; if (c < D) { out[c] = dw[i][j]; out[D + c] = db[i][j]; } }
    } else {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            wg_sync();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) join[t / NT][col_of<NT>(l, i) + j] = which ? db[i][j] : dw[i][j];
            wg_sync();
            for (int c = t; c < D; c += THREADS) {
                float v = 0.0f;
#pragma unroll 8
                for (int k = 0; k < RPG; ++k) v += join[k][c];
                out[(long long)which * D + c] = v;
            }
        }
    }
}

// dw[c], db[c] = the sum over the work-groups' partial rows, in order
template <class T>
__global__ __launch_bounds__(256) void norm_join_kernel(const float* __restrict__ part, int groups, int D, void* dw, void* db, int param_f32) {
    __shared__ float red[16][17];
    const int cl = threadIdx.x & 15, q = threadIdx.x >> 4, c = (int)blockIdx.x * 16 + cl;      // c over the 2 D columns of a partial row
    float s = 0.0f;
    if (c < 2 * D)
#pragma unroll 8
        for (int k = q; k < groups; k += 16) s += part[(long long)k * 2 * D + c];
    red[q][cl] = s;
    wg_sync();
    if (q == 0 && c < 2 * D) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) v += red[k][cl];
        void* dst = c < D ? dw : db;
        if (dst) store_param<T>(dst, param_f32, c < D ? c : c - D, v);
    }
}

namespace {

// threads per row and pieces per thread for a width: up to 1024 columns a row stays within one wave (no barrier), beyond that 8 .. 16 values per lane
template <class F>
void by_width(int D, F go) {
    if (D <= 64) go(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    else if (D <= 128) go(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    else if (D <= 256) go(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
    else if (D <= 512) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (D <= 1024) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (D <= 2048) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{});
    else if (D <= 4096) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (D <= 8192) go(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}

template <class T, bool WHOLE>
void launch_norm_t(const NormArgs& a, int grid, bool backward, hipStream_t st) {
    by_width(a.D, [&](auto nt, auto nv) {
        constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
        const dim3 b(NT > 256 ? NT : 256);
        if (backward) hipLaunchKernelGGL((norm_bwd_kernel<T, NT, NV, WHOLE>), dim3(grid), b, 0, st, a);
        else hipLaunchKernelGGL((norm_fwd_kernel<T, NT, NV, WHOLE>), dim3(grid), b, 0, st, a);
    });
}

}  // namespace

int norm_threads(int D) {
    int r = 0;
    by_width(D, [&](auto nt, auto) { r = decltype(nt)::value > 256 ? decltype(nt)::value : 256; });
    return r;
}
int norm_rows_per_group(int D) {
    int r = 0;
    by_width(D, [&](auto nt, auto) { r = decltype(nt)::value > 256 ? 1 : 256 / decltype(nt)::value; });
    return r;
}

void launch_norm_join(int dtype, const float* part, int groups, int D, void* dw, void* db, int param_f32, hipStream_t st) {
    const dim3 grid((unsigned)((2 * D + 15) / 16));
    if (dtype == 0) hipLaunchKernelGGL((norm_join_kernel<float>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
    else if (dtype == 1) hipLaunchKernelGGL((norm_join_kernel<__bf16>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
    else hipLaunchKernelGGL((norm_join_kernel<_Float16>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
}

void launch_norm(int dtype, const NormArgs& a, int grid, bool backward, hipStream_t st) {
    const bool whole = a.D % 8 == 0;
    if (dtype == 0) whole ? launch_norm_t<float, true>(a, grid, backward, st) : launch_norm_t<float, false>(a, grid, backward, st);
    else if (dtype == 1) whole ? launch_norm_t<__bf16, true>(a, grid, backward, st) : launch_norm_t<__bf16, false>(a, grid, backward, st);
    else whole ? launch_norm_t<_Float16, true>(a, grid, backward, st) : launch_norm_t<_Float16, false>(a, grid, backward, st);
}

}  // namespace ops
}  // namespace lsdm
