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
// VEC: 16-byte pieces (a lane's columns are (lane + NT i) 8 + j); otherwise -- odd widths, unaligned rows -- single elements, lane-interleaved
// (column (8 i + j) NT + lane), which stays coalesced.
#include "ops.hpp"
#include "ops_launch.hpp"

namespace lsdm {
namespace ops {

template <int NT>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* red, int t) {
    constexpr int W = NT < 64 ? NT : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
    if constexpr (NT > 64) {
        constexpr int NW = NT / 64;
        wg_sync();                               // (the previous sums have been read)
        if ((t & 63) == 0) red[t >> 6] = make_float2(a, b);
        wg_sync();
        a = 0.0f; b = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) { a += red[i].x; b += red[i].y; }
    }
    return make_float2(a, b);
}

template <int NT, bool VEC>
__device__ __forceinline__ int col_of(int l, int i, int j) { return VEC ? (l + NT * i) * 8 + j : (i * 8 + j) * NT + l; }

template <class T, int NT, int NV, bool VEC>
__device__ __forceinline__ void row_load(const T* p, int D, int l, float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            if ((l + NT * i) * 8 < D) load8(p + (l + NT * i) * 8, v[i]);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) { const int c = col_of<NT, VEC>(l, i, j); v[i][j] = c < D ? (float)p[c] : 0.0f; }
        }
    }
}
template <class T, int NT, int NV, bool VEC>
__device__ __forceinline__ void row_store(T* p, int D, int l, const float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            if ((l + NT * i) * 8 < D) store8(p + (l + NT * i) * 8, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) { const int c = col_of<NT, VEC>(l, i, j); if (c < D) p[c] = (T)v[i][j]; }
        }
    }
}

// the row's 8-bit checkpoint: groups of 32 columns are four lanes' pieces (VEC) or 32 lanes' single elements
template <int NT, int NV, bool VEC>
__device__ __forceinline__ void row_encode(const float (&h)[NV][8], int D, int l, signed char* codes, unsigned char* exps) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __builtin_bit_cast(unsigned, h[i][j]) & 0x7fffffffu);   // (order of the bit patterns: NaN is largest)
            m = max(m, (unsigned)__shfl_xor((int)m, 1));
            m = max(m, (unsigned)__shfl_xor((int)m, 2));
            const unsigned b = exp8_of_amax(__builtin_bit_cast(float, m));
            const float inv = exp8_inv(b);
            const int c = (l + NT * i) * 8;
            if (c < D) {
                unsigned q[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = (unsigned)code8(h[i][j], inv) & 255u;
                *reinterpret_cast<u32x2*>(codes + c) = u32x2{q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24};
                if ((l & 3) == 0) exps[c >> 5] = (unsigned char)b;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = col_of<NT, VEC>(l, i, j);
                unsigned m = c < D ? __builtin_bit_cast(unsigned, h[i][j]) & 0x7fffffffu : 0u;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
                const unsigned b = exp8_of_amax(__builtin_bit_cast(float, m));
                if (c < D) {
                    codes[c] = (signed char)code8(h[i][j], exp8_inv(b));
                    if ((l & 31) == 0) exps[c >> 5] = (unsigned char)b;
                }
            }
        }
    }
}
template <int NT, int NV, bool VEC>
__device__ __forceinline__ void row_decode(const signed char* codes, const unsigned char* exps, int D, int l, float (&h)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            const int c = (l + NT * i) * 8;
            u32x2 w = {0, 0};
            float s = 0.0f;
            if (c < D) { w = *reinterpret_cast<const u32x2*>(codes + c); s = exp8_step(exps[c >> 5]); }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = (float)((int)(w[j >> 2] << (24 - 8 * (j & 3))) >> 24) * s;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = col_of<NT, VEC>(l, i, j);
                h[i][j] = c < D ? (float)codes[c] * exp8_step(exps[c >> 5]) : 0.0f;
            }
        }
    }
}

template <class T, int NT, int NV, bool VEC>
__device__ __forceinline__ void param_load(const void* p, int is_f32, float missing, int D, int l, float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) { const int c = col_of<NT, VEC>(l, i, j); v[i][j] = p && c < D ? param<T>(p, is_f32, c) : (c < D ? missing : 0.0f); }
}

template <class T, int NT, int NV, bool VEC>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void norm_fwd_kernel(NormArgs a) {
    constexpr int THREADS = NT > 256 ? NT : 256, RPG = THREADS / NT;
    __shared__ float2 red[NT > 64 ? NT / 64 : 1];
    const int t = threadIdx.x, l = t % NT, D = a.D;
    float w[NV][8], b[NV][8];
    param_load<T, NT, NV, VEC>(a.w, a.param_f32, 1.0f, D, l, w);
    param_load<T, NT, NV, VEC>(a.b, a.param_f32, 0.0f, D, l, b);
    const float inv_d = 1.0f / (float)D;
    // (a work-group of one row per NT <= 64 threads has no barrier: its rows end independently; with NT > 64 the loop is uniform)
    for (long long r = (long long)blockIdx.x * RPG + t / NT; r < a.rows; r += (long long)gridDim.x * RPG) {
        float x[NV][8];
        row_load<T, NT, NV, VEC>(static_cast<const T*>(a.x) + r * a.ldx, D, l, x);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += x[i][j];
        // the mean's own rounding is taken out again: d = the mean of x - mu (a row without spread gives h = 0, not a last bit times 1 / sqrt(eps))
        float mu = row_sum2<NT>(s, 0.0f, red, t).x / (float)D, q = 0.0f;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) { x[i][j] = col_of<NT, VEC>(l, i, j) < D ? x[i][j] - mu : 0.0f; s += x[i][j]; q = fmaf(x[i][j], x[i][j], q); }
        const float2 c = row_sum2<NT>(s, q, red, t);
        const float d = c.x * inv_d, rstd = 1.0f / sqrtf(fmaxf(fmaf(c.y, inv_d, -d * d), 0.0f) + a.eps);
        mu += d;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = col_of<NT, VEC>(l, i, j) < D ? (x[i][j] - d) * rstd : 0.0f;
        if (a.mean && l == 0) a.mean[r] = mu;
        if (a.rstd && l == 0) a.rstd[r] = rstd;
        if (a.codes) row_encode<NT, NV, VEC>(x, D, l, a.codes + r * D, a.exps + r * ((D + 31) >> 5));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = fmaf(x[i][j], w[i][j], b[i][j]);
        row_store<T, NT, NV, VEC>(static_cast<T*>(a.y) + r * D, D, l, x);
    }
}

template <class T, int NT, int NV, bool VEC>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void norm_bwd_kernel(NormArgs a) {
    constexpr int THREADS = NT > 256 ? NT : 256, RPG = THREADS / NT, COLS = NT * NV * 8;
    __shared__ float2 red[NT > 64 ? NT / 64 : 1];
    __shared__ float join[RPG > 1 ? RPG : 1][RPG > 1 ? COLS + 1 : 1];
    const int t = threadIdx.x, l = t % NT, D = a.D;
    float w[NV][8], dw[NV][8], db[NV][8];
    param_load<T, NT, NV, VEC>(a.w, a.param_f32, 1.0f, D, l, w);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.0f;
    const float inv_d = 1.0f / (float)D;
    for (long long r = (long long)blockIdx.x * RPG + t / NT; r < a.rows; r += (long long)gridDim.x * RPG) {
        float g[NV][8], h[NV][8];
        row_load<T, NT, NV, VEC>(static_cast<const T*>(a.dy) + r * a.lddy, D, l, g);
        const float rstd = a.rstd[r];
        if (a.codes) {
            row_decode<NT, NV, VEC>(a.codes + r * D, a.exps + r * ((D + 31) >> 5), D, l, h);
        } else {
            row_load<T, NT, NV, VEC>(static_cast<const T*>(a.x) + r * a.ldx, D, l, h);
            const float mu = a.mean[r];
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = col_of<NT, VEC>(l, i, j) < D ? (h[i][j] - mu) * rstd : 0.0f;
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
            row_store<T, NT, NV, VEC>(static_cast<T*>(a.dx) + r * D, D, l, g);
        }
    }
    if (!a.part) return;
    // one partial row of dw and of db per work-group
    float* out = a.part + (long long)blockIdx.x * 2 * D;
    if constexpr (RPG == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) { const int c = col_of<NT, VEC>(l, i, j); if (c < D) { out[c] = dw[i][j]; out[D + c] = db[i][j]; } }
    } else {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            wg_sync();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) join[t / NT][col_of<NT, VEC>(l, i, j)] = which ? db[i][j] : dw[i][j];
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

// threads per row and pieces per thread for a width: up to 1024 columns a row stays within one wave (no barrier), beyond that it is a work-group's
template <class T, bool VEC, class F>
void by_width(int D, F go) {
    if constexpr (VEC) {
        if (D <= 64) return go(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
        if (D <= 128) return go(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    }
    if (D <= 256) go(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
    else if (D <= 512) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (D <= 1024) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (D <= 2048) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (D <= 4096) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (D <= 8192) go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}

template <class T, bool VEC>
void launch_norm_tv(const NormArgs& a, int grid, bool backward, hipStream_t st) {
    by_width<T, VEC>(a.D, [&](auto nt, auto nv) {
        constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
        const dim3 b(NT > 256 ? NT : 256);
        if (backward) hipLaunchKernelGGL((norm_bwd_kernel<T, NT, NV, VEC>), dim3(grid), b, 0, st, a);
        else hipLaunchKernelGGL((norm_fwd_kernel<T, NT, NV, VEC>), dim3(grid), b, 0, st, a);
    });
}
template <class T>
void launch_norm_t(const NormArgs& a, bool vec, int grid, bool backward, hipStream_t st) {
    if (vec) launch_norm_tv<T, true>(a, grid, backward, st);
    else launch_norm_tv<T, false>(a, grid, backward, st);
}

}  // namespace

int norm_rows_per_group(int D, bool vec) {
    int r = 1;
    auto f = [&](auto nt, auto) { constexpr int NT = decltype(nt)::value; r = NT >= 256 ? 1 : 256 / NT; };
    if (vec) by_width<float, true>(D, f); else by_width<float, false>(D, f);
    return r;
}

void launch_norm_join(int dtype, const float* part, int groups, int D, void* dw, void* db, int param_f32, hipStream_t st) {
    const dim3 grid((unsigned)((2 * D + 15) / 16));
    if (dtype == 0) hipLaunchKernelGGL((norm_join_kernel<float>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
    else if (dtype == 1) hipLaunchKernelGGL((norm_join_kernel<__bf16>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
    else hipLaunchKernelGGL((norm_join_kernel<_Float16>), grid, dim3(256), 0, st, part, groups, D, dw, db, param_f32);
}

void launch_norm(int dtype, const NormArgs& a, bool vec, int grid, bool backward, hipStream_t st) {
    if (dtype == 0) launch_norm_t<float>(a, vec, grid, backward, st);
    else if (dtype == 1) launch_norm_t<__bf16>(a, vec, grid, backward, st);
    else launch_norm_t<_Float16>(a, vec, grid, backward, st);
}

}  // namespace ops
}  // namespace lsdm
