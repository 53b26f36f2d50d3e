// Shared pieces of the public operators (ops_gemm.hip, ops_norm.hip, ops_pack8.hip, ops_api.hip): element types, 8-element row pieces, the
// activations with their derivatives, the 8-bit checkpoint format, and the launchers the C entry points call.
#pragma once
#include "common.hpp"

namespace lsdm {
namespace ops {

typedef __bf16 bfrag __attribute__((ext_vector_type(8)));
typedef _Float16 hfrag __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

enum OpAct { OP_NONE = 0, OP_RELU, OP_GELU, OP_QUICK_GELU, OP_SILU, OP_SIGMOID, OP_TANH, OP_ACT_COUNT };

// Eight consecutive elements of a row as one memory access.  Rows of any width start anywhere, so the pieces are typed with the element's alignment:
// gfx950 takes 16-byte global accesses at any address (the compiler emits one instruction), and an odd width costs a misaligned line per wave
// instead of eight single-element accesses per piece.
template <class T> struct Piece;
template <> struct Piece<__bf16> { typedef bfrag frag; typedef bfrag mem __attribute__((aligned(2))); };
template <> struct Piece<_Float16> { typedef hfrag frag; typedef hfrag mem __attribute__((aligned(2))); };
template <> struct Piece<float> { typedef f32x4 frag; typedef f32x4 mem __attribute__((aligned(4))); };
typedef u32x2 codes8 __attribute__((aligned(1)));
typedef u32x4 codes16 __attribute__((aligned(1)));

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    typedef typename Piece<T>::mem mem;
    if constexpr (sizeof(T) == 2) {
        const typename Piece<T>::frag r = *reinterpret_cast<const mem*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
    } else {
        const f32x4 a = *reinterpret_cast<const mem*>(p), b = *reinterpret_cast<const mem*>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    }
}
// STREAM: 16-bit results that nothing reads soon are stored non-temporally (norms 5 .. 15 %, products 3 .. 10 % of the time at large sizes: the inputs
// keep the caches).  Not scratch memory that the next launch reads (its products lost 10 %), and not where a wave's store leaves gaps for a second one to
// fill, as the two halves of an fp32 piece do: such lines are written twice (unpack8: 32 -> 63 us in bf16, 89 -> 311 us in fp32 at 32768 x 2048).
template <bool STREAM = false, class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    typedef typename Piece<T>::frag frag;
    typedef typename Piece<T>::mem mem;
    constexpr int H = 8 * (int)sizeof(T) / 16;
#pragma unroll
    for (int k = 0; k < H; ++k) {
        frag r;
#pragma unroll
        for (int j = 0; j < 8 / H; ++j) r[j] = (T)v[k * (8 / H) + j];
        mem* q = reinterpret_cast<mem*>(p + k * (8 / H));
        if constexpr (STREAM && sizeof(T) == 2) __builtin_nontemporal_store(r, q); else *q = r;
    }
}
// a piece cut short by the row's end: n valid elements (n <= 0: none); the others read as 0 and are not written
template <class T>
__device__ __forceinline__ void load8n(const T* p, int n, float (&v)[8]) {
    if (n >= 8) return load8(p, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
}
template <bool STREAM = false, class T>
__device__ __forceinline__ void store8n(T* p, int n, const float (&v)[8]) {
    if (n >= 8) return store8<STREAM>(p, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = (T)v[j];
}
// eight bytes (codes), the same way
__device__ __forceinline__ u32x2 load_codes(const void* q, int n) {
    const unsigned char* p = static_cast<const unsigned char*>(q);
    if (n >= 8) return *reinterpret_cast<const codes8*>(p);
    u32x2 w = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) w[j >> 2] |= (unsigned)p[j] << (8 * (j & 3));
    return w;
}
__device__ __forceinline__ void store_codes(void* q, int n, const unsigned (&c)[8]) {
    unsigned char* p = static_cast<unsigned char*>(q);
    if (n >= 8) {
        *reinterpret_cast<codes8*>(p) = u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = (unsigned char)c[j];
}
// a parameter vector (bias, norm weight) is of the operand's type or fp32
template <class T>
__device__ __forceinline__ float param(const void* p, int is_f32, long long i) {
    return is_f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
template <class T>
__device__ __forceinline__ void store_param(void* p, int is_f32, long long i, float v) {
    if (is_f32) static_cast<float*>(p)[i] = v; else static_cast<T*>(p)[i] = (T)v;
}

// ---- activations: y = a(z) and, where asked for, d = a'(z) ----
// fp32 results use the libm functions; 16-bit results the hardware's exp2 and reciprocal (1 ulp each), and for gelu Abramowitz & Stegun 7.1.26 (|error| of
// Phi <= 1.5e-7, as in common.hpp); tanh is tanhf in every type.  Absolute error of the factors Phi and s <= 3e-7, of y = z Phi and z s |z| times that: in the
// far tail of 16-bit gelu the polynomial's own error shows (1 % of y at z = -8, where y = -5e-15).  No form subtracts from one what may be next to one: 1 - s
// is e s with e = exp(-c z) (its NaN at e = infinity, s = 0 gives way to 1), Phi of a negative z comes from erfc, 1 - tanh^2 from exp(-2 |z|); so fp32 values and
// derivatives keep their relative accuracy in saturation (a few ulp, plus z^2 ulp for gelu).  NaN stays NaN in y for every activation; relu'(NaN) = 0 (the
// comparison z > 0).
template <class T, int ACT>
__device__ __forceinline__ void act_one(float z, bool want, float& y, float& d) {
    constexpr bool fast = sizeof(T) == 2;
    if constexpr (ACT == OP_RELU) {
        y = z <= 0.0f ? 0.0f : z;
        d = z > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == OP_GELU && fast) {
        const float x = fabsf(z) * 0.70710678118654752440f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f)), ex = __expf(-x * x);
        float pl = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
        pl = fmaf(t, pl, 0.5f * 1.421413741f);
        pl = fmaf(t, pl, 0.5f * -0.284496736f);
        pl = fmaf(t, pl, 0.5f * 0.254829592f);
        const float q = pl * t * ex, phi = z < 0.0f ? q : 1.0f - q;
        y = z * phi;
        d = fmaf(z * 0.39894228040143267794f, ex, phi);
    } else if constexpr (ACT == OP_GELU) {
        const float phi = 0.5f * erfcf(z * -0.70710678118654752440f);
        y = z * phi;
        if (want) d = phi + z * 0.39894228040143267794f * expf(-0.5f * z * z);
    } else if constexpr (ACT == OP_QUICK_GELU || ACT == OP_SILU || ACT == OP_SIGMOID) {
        constexpr float c = ACT == OP_QUICK_GELU ? 1.702f : 1.0f;
        const float e = fast ? __expf(-(c * z)) : expf(-(c * z)), s = fast ? __builtin_amdgcn_rcpf(1.0f + e) : 1.0f / (1.0f + e), rest = fminf(e * s, 1.0f);
        y = ACT == OP_SIGMOID ? s : z * s;
        d = ACT == OP_SIGMOID ? s * rest : s * fmaf(c * z, rest, 1.0f);
    } else {
        y = tanhf(z);
        if (want) {
            const float e = fast ? __expf(-2.0f * fabsf(z)) : expf(-2.0f * fabsf(z)), r = fast ? __builtin_amdgcn_rcpf(1.0f + e) : 1.0f / (1.0f + e);
            d = 4.0f * e * r * r;
        }
    }
}
template <class T, int ACT>
__device__ __forceinline__ void act_each(const float (&z)[8], bool want, float (&y)[8], float (&d)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) act_one<T, ACT>(z[j], want, y[j], d[j]);
}
// one branch on the activation for eight values, whose chains of transcendentals then overlap
template <class T>
__device__ __forceinline__ void act8(int act, const float (&z)[8], bool want, float (&y)[8], float (&d)[8]) {
    switch (act) {
        case OP_RELU: act_each<T, OP_RELU>(z, want, y, d); break;
        case OP_GELU: act_each<T, OP_GELU>(z, want, y, d); break;
        case OP_QUICK_GELU: act_each<T, OP_QUICK_GELU>(z, want, y, d); break;
        case OP_SILU: act_each<T, OP_SILU>(z, want, y, d); break;
        case OP_SIGMOID: act_each<T, OP_SIGMOID>(z, want, y, d); break;
        default: act_each<T, OP_TANH>(z, want, y, d); break;
    }
}

// a'(z) is kept for the backward pass in 16 bits (bf16 and fp16 calls; fp32 calls keep fp32): the sign and C |a'|^(1/4) as a whole number, C = 31744; the
// largest |a'|, gelu's 1.13, is code 32722.  A value d is rounded by 2 d / (C d^(1/4)): 2^-14 relative near 1, 2^-13 at 2^-4, and 2^-8, half a step of bf16, at
// 2^-23; from 1/32 up a sixteenth (bf16) or a third (fp16) of half a step of the type itself, and no zero before 2^-64.  (Sign, 3 exponent and 12 mantissa
// bits, which ended at 2^-19, lost saturated derivatives.  Two square roots when written, three products when read: 16384 x 2048 -> 8192 with gelu, both passes,
// 1603 -> 1611 us.)
// 0 and 1 (relu) are exact, as C (1 / C) is in fp32.  0x7fff stands for NaN.
constexpr float kDeriv16 = 31744.0f;
__device__ __forceinline__ unsigned deriv_code16(float d) {
    const float v = fmaf(kDeriv16, __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(fabsf(d))), 0.5f);
    return (v < 32767.0f ? (unsigned)v : 0x7fffu) | ((__builtin_bit_cast(unsigned, d) >> 16) & 0x8000u);
}
__device__ __forceinline__ float deriv_value16(unsigned u) {
    const unsigned c = u & 0x7fffu;
    float v = (float)c * (1.0f / kDeriv16);
    v *= v;
    v *= v;
    return c == 0x7fffu ? __builtin_nanf("") : __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) | (u & 0x8000u) << 16);
}
// ... or, with an 8-bit checkpoint, in 8 bits: u = rint(192 a') + 32, codes 7 .. 249; 0 and 1 (relu) are exact, the error is at most 1/384.  Code 255
// stands for NaN.
__device__ __forceinline__ unsigned deriv_code8(float d) {
    const float u = fminf(fmaxf(rintf(192.0f * d) + 32.0f, 0.0f), 254.0f);
    return d != d ? 255u : (unsigned)u;
}
__device__ __forceinline__ float deriv_value8(unsigned u) {
    return u == 255u ? __builtin_nanf("") : (float)((int)u - 32) * (1.0f / 192.0f);
}
enum DerivForm { DERIV_NONE = 0, DERIV_F32 = 1, DERIV_16 = 2, DERIV_8 = 3 };

// ---- 8-bit checkpoint: groups of kGroup8 consecutive values of a row share a power-of-two step 2^e ----
// m = max |x| of the group, e = max(floor(log2 m) - 6, -126), q = clamp(rint(x 2^-e), +-127); stored: q (int8), e + 127 (uint8), 255 for a
// group that holds an infinity or a NaN (it decodes to NaN: a checkpoint never hides an overflow).  q 2^e has at most 7 significant bits, so it
// is exact in fp32, in bf16 and in the type the values came from (in fp16 what lies outside its range is not, if they came from another).
constexpr int kGroup8 = 32;
constexpr unsigned kNanExp8 = 255u;
__device__ __forceinline__ unsigned exp8_of_amax(float m) {        // m >= 0, NaN or inf for a non-finite group
    const int E = (int)(__builtin_bit_cast(unsigned, m) >> 23);     // biased exponent (0: zero or subnormal)
    return E == 255 ? kNanExp8 : (unsigned)(E - 6 > 1 ? E - 6 : 1);
}
__device__ __forceinline__ float exp8_step(unsigned b) { return b == kNanExp8 ? __builtin_nanf("") : __builtin_bit_cast(float, b << 23); }
// 2^-e: e + 127 in [1, 248] -> the reciprocal's biased exponent 254 - b is in [6, 253]; b = 255 gives 0 (the codes of such a group: 0, or -127 for the
// infinities and NaN themselves; nothing reads them as values)
__device__ __forceinline__ float exp8_inv(unsigned b) { return b == kNanExp8 ? 0.0f : __builtin_bit_cast(float, (254u - b) << 23); }
__device__ __forceinline__ int code8(float x, float inv) {
    const float v = rintf(x * inv);
    return (int)fminf(fmaxf(v, -127.0f), 127.0f);                   // (non-finite groups: inv = 0, and the NaN of inf * 0 becomes -127)
}

// ---- kernels' argument blocks and launchers ----
struct Epilogue {
    const void* bias = nullptr; int bias_f32 = 0;
    const void* res = nullptr; long long ldr = 0;
    void* out = nullptr; long long ldo = 0;
    void* deriv = nullptr; long long ldd = 0; int form = DERIV_NONE;   // a'(z) for the backward pass
    int act = OP_NONE;
    int stream = 0;                                                 // rows of out and deriv are made of whole 128-byte lines
};
struct GemmArgs {
    const void *A = nullptr, *B = nullptr;                          // C(m, n) = sum_k A(m, k) B(n, k)
    long long lda = 0, ldb = 0;                                     // row strides in elements
    int M = 0, N = 0, K = 0;
    int tiles_m = 0, tiles_n = 0, splits = 1, kchunk = 0;
    float* part = nullptr;                                          // splits > 1: (splits, M, N) partial sums
    Epilogue e;
    // work-groups behind the tiles' join column sums left by an earlier launch: out[c] = sum over the chunks of cs_part[chunk][c], in order
    int blocks = 0;                                                 // work-groups of the product itself
    const float* cs_part = nullptr; int cs_chunks = 0, cs_n = 0, cs_f32 = 0; void* cs_out = nullptr;
};

enum Layout { KK = 0, KM = 1, MM = 2 };                             // contraction axis contiguous in (A and B), (A only), (neither)

}  // namespace ops
}  // namespace lsdm
