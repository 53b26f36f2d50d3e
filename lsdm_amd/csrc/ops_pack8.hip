// 8-bit activation checkpoints (ops.hpp: the format; include/lsdm_hip.h: lsdm_pack8, lsdm_unpack8), gfx950.  Bound by HBM: pack reads a value and
// writes 33/32 bytes, unpack the reverse.
//   wide rows (a multiple of 32 columns, 16-byte aligned): a thread owns 16 consecutive values, two threads share a group's maximum by one
//   cross-lane exchange; any other row: half a wave per group, a value per lane.
#include "ops.hpp"
#include "ops_launch.hpp"

namespace lsdm {
namespace ops {

template <class T>
__global__ __launch_bounds__(256) void pack8_wide_kernel(Pack8Args a, long long pieces, int ppr) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;                     // (pieces is even: both threads of a group are here or neither is)
    const long long r = i / ppr;
    const int c = (int)(i - r * ppr) * 16;
    float v[2][8];
    const T* p = static_cast<const T*>(a.x) + r * a.ldx + c;
    load8(p, v[0]);
    load8(p + 8, v[1]);
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = max(m, __builtin_bit_cast(unsigned, v[k >> 3][k & 7]) & 0x7fffffffu);
    m = max(m, (unsigned)__shfl_xor((int)m, 1));
    const unsigned b = exp8_of_amax(__builtin_bit_cast(float, m));
    const float inv = exp8_inv(b);
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        unsigned q = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) q |= ((unsigned)code8(v[(4 * k + j) >> 3][(4 * k + j) & 7], inv) & 255u) << (8 * j);
        w[k] = q;
    }
    *reinterpret_cast<u32x4*>(a.codes + i * 16) = w;
    if ((threadIdx.x & 1) == 0) a.exps[i >> 1] = (unsigned char)b;
}
template <class T>
__global__ __launch_bounds__(256) void unpack8_wide_kernel(Pack8Args a, long long pieces) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const u32x4 w = *reinterpret_cast<const u32x4*>(a.codes + i * 16);
    const float s = exp8_step(a.exps[i >> 1]);
    float v[2][8];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k >> 3][k & 7] = (float)((int)(w[k >> 2] << (24 - 8 * (k & 3))) >> 24) * s;
    T* p = static_cast<T*>(a.out) + i * 16;
    store8(p, v[0]);
    store8(p + 8, v[1]);
}
template <class T>
__global__ __launch_bounds__(256) void pack8_any_kernel(Pack8Args a, long long groups, int gpr) {
    const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
    if (g >= groups) return;
    const long long r = g / gpr;
    const int c = (int)(g - r * gpr) * 32 + (threadIdx.x & 31);
    const float x = c < a.D ? (float)static_cast<const T*>(a.x)[r * a.ldx + c] : 0.0f;
    unsigned m = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
    const unsigned b = exp8_of_amax(__builtin_bit_cast(float, m));
    if (c < a.D) a.codes[r * a.D + c] = (signed char)code8(x, exp8_inv(b));
    if ((threadIdx.x & 31) == 0) a.exps[g] = (unsigned char)b;
}
template <class T>
__global__ __launch_bounds__(256) void unpack8_any_kernel(Pack8Args a, long long total, int gpr) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const long long r = i / a.D;
    const int c = (int)(i - r * a.D);
    static_cast<T*>(a.out)[i] = (T)((float)a.codes[i] * exp8_step(a.exps[r * gpr + (c >> 5)]));
}

namespace {
unsigned blocks(long long threads) { return (unsigned)((threads + 255) / 256); }

template <class T>
void pack_t(const Pack8Args& a, bool wide, hipStream_t st) {
    const int gpr = (a.D + 31) / 32;
    if (wide) hipLaunchKernelGGL((pack8_wide_kernel<T>), dim3(blocks(a.rows * (a.D / 16))), dim3(256), 0, st, a, a.rows * (a.D / 16), a.D / 16);
    else hipLaunchKernelGGL((pack8_any_kernel<T>), dim3(blocks(a.rows * gpr * 32)), dim3(256), 0, st, a, a.rows * gpr, gpr);
}
template <class T>
void unpack_t(const Pack8Args& a, bool wide, hipStream_t st) {
    const int gpr = (a.D + 31) / 32;
    if (wide) hipLaunchKernelGGL((unpack8_wide_kernel<T>), dim3(blocks(a.rows * (a.D / 16))), dim3(256), 0, st, a, a.rows * (a.D / 16));
    else hipLaunchKernelGGL((unpack8_any_kernel<T>), dim3(blocks(a.rows * a.D)), dim3(256), 0, st, a, a.rows * a.D, gpr);
}
}  // namespace

void launch_pack8(int dtype, const Pack8Args& a, bool wide, hipStream_t st) {
    if (dtype == 0) pack_t<float>(a, wide, st);
    else if (dtype == 1) pack_t<__bf16>(a, wide, st);
    else pack_t<_Float16>(a, wide, st);
}
void launch_unpack8(int dtype, const Pack8Args& a, bool wide, hipStream_t st) {
    if (dtype == 0) unpack_t<float>(a, wide, st);
    else if (dtype == 1) unpack_t<__bf16>(a, wide, st);
    else unpack_t<_Float16>(a, wide, st);
}

}  // namespace ops
}  // namespace lsdm
