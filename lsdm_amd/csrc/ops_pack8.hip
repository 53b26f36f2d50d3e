// 8-bit activation checkpoints (ops.hpp: the format; include/lsdm_hip.h: lsdm_pack8, lsdm_unpack8), gfx950.  Bound by HBM: pack reads a value and
// writes 33/32 bytes, unpack the reverse.
// A thread owns 16 consecutive values of a row; two threads share a group and its maximum by one cross-lane exchange.
// Measured: 32768 x 2048 bf16 pack 31 us, unpack 32 us (6.6 TB/s, part of it out of the cache); fp32 59 and 91 us.
#include "ops.hpp"
#include "ops_launch.hpp"

namespace lsdm {
namespace ops {

// half: 16 columns, two to a group; hpr halves per row (an even number, the last may be cut short or empty)
template <class T>
__global__ __launch_bounds__(256) void pack8_kernel(Pack8Args a, long long halves, int hpr) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= halves) return;                     // (halves is even: both threads of a group are here or neither is)
    const long long r = i / hpr;
    const int h = (int)(i - r * hpr), c = h * 16, n = a.D - c;
    float v[2][8];
    const T* p = static_cast<const T*>(a.x) + r * a.ldx + c;
    if (n >= 16) {                               // (both pieces in one branch: two loads in flight)
        load8(p, v[0]);
        load8(p + 8, v[1]);
    } else {
        load8n(p, n, v[0]);
        load8n(p + 8, n - 8, v[1]);
    }
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = max(m, __builtin_bit_cast(unsigned, v[k >> 3][k & 7]) & 0x7fffffffu);
    m = max(m, (unsigned)__shfl_xor((int)m, 1));
    const unsigned b = exp8_of_amax(__builtin_bit_cast(float, m));
    const float inv = exp8_inv(b);
    unsigned q[2][8];
#pragma unroll
    for (int k = 0; k < 16; ++k) q[k >> 3][k & 7] = (unsigned)code8(v[k >> 3][k & 7], inv) & 255u;
    signed char* out = a.codes + r * a.D + c;
    if (n >= 16) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned* s = &q[k >> 1][4 * (k & 1)];
            w[k] = s[0] | s[1] << 8 | s[2] << 16 | s[3] << 24;
        }
        *reinterpret_cast<codes16*>(out) = w;
    } else {
        store_codes(out, n, q[0]);
        store_codes(out + 8, n - 8, q[1]);
    }
    if ((h & 1) == 0) a.exps[r * (hpr >> 1) + (h >> 1)] = (unsigned char)b;
}
template <class T>
__global__ __launch_bounds__(256) void unpack8_kernel(Pack8Args a, long long halves, int hpr) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= halves) return;
    const long long r = i / hpr;
    const int h = (int)(i - r * hpr), c = h * 16, n = a.D - c;
    if (n <= 0) return;
    const signed char* in = a.codes + r * a.D + c;
    u32x4 w;
    if (n >= 16) {
        w = *reinterpret_cast<const codes16*>(in);
    } else {
        const u32x2 w0 = load_codes(in, n), w1 = load_codes(in + 8, n - 8);
        w = u32x4{w0[0], w0[1], w1[0], w1[1]};
    }
    const float s = exp8_step(a.exps[r * (hpr >> 1) + (h >> 1)]);
    float v[2][8];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k >> 3][k & 7] = (float)((int)(w[k >> 2] << (24 - 8 * (k & 3))) >> 24) * s;
    T* p = static_cast<T*>(a.out) + r * a.D + c;
    store8n(p, n, v[0]);
    store8n(p + 8, n - 8, v[1]);
}

namespace {
template <class T>
void launch_t(const Pack8Args& a, bool pack, hipStream_t st) {
    const int hpr = (a.D + 31) / 32 * 2;
    const long long halves = a.rows * hpr;
    const dim3 grid((unsigned)((halves + 255) / 256));
    if (pack) hipLaunchKernelGGL((pack8_kernel<T>), grid, dim3(256), 0, st, a, halves, hpr);
    else hipLaunchKernelGGL((unpack8_kernel<T>), grid, dim3(256), 0, st, a, halves, hpr);
}
void launch(int dtype, const Pack8Args& a, bool pack, hipStream_t st) {
    if (dtype == 0) launch_t<float>(a, pack, st);
    else if (dtype == 1) launch_t<__bf16>(a, pack, st);
    else launch_t<_Float16>(a, pack, st);
}
}  // namespace

void launch_pack8(int dtype, const Pack8Args& a, hipStream_t st) { launch(dtype, a, true, st); }
void launch_unpack8(int dtype, const Pack8Args& a, hipStream_t st) { launch(dtype, a, false, st); }

}  // namespace ops
}  // namespace lsdm
