// Matrix products of ops.linear (include/lsdm_hip.h: lsdm_linear, lsdm_linear_backward), gfx950.
//
//   forward   y = a(x W^T + b) + r          C(m, n) = sum_k A(m, k) B(n, k),  A = x, B = W: the contraction axis is contiguous in both   (KK)
//   dx        dz W                          A = dz, B(n, k) = W[k][n]: contiguous in A only                                               (KM)
//   dW        dz^T x                        A(m, k) = dz[k][m], B(n, k) = x[k][n]: contiguous in neither                                  (MM)
//
// One tile core for all three.  A work-group owns a BM x BN tile of C and walks k in steps of 128 bytes through two LDS buffers: both operand tiles come into
// LDS by LDS-DMA (16 bytes per lane, no registers), the next step's in flight while this one is multiplied.
//   16-bit: v_mfma_f32_16x16x32; a tile whose contraction axis is contiguous is read with ds_read_b128, the other kind with the transposing
//           ds_read_b64_tr_b16, so that no operand is ever transposed in memory.
//   fp32:   v_mfma_f32_32x32x2 (exact products, an fmaf chain).
// The products are evaluated as D[n][m] (the B tile is the instruction's first operand): a lane owns four consecutive n of one m, and the
// epilogue goes through LDS once so that a store instruction writes whole 128-byte lines.
// LDS-DMA writes lane l's 16 bytes at base + 16 l, so the bank swizzle is put into the GLOBAL address a lane reads (src_* below) and undone by
// the reader.  A lane whose k lies beyond the end reads 16 zero bytes (g_zero16); rows beyond the end are clamped to the last one, and their
// results are not stored.
// Measured (MI355X, back to back; the boxes differ by 5 %): 8192 x 4096 x 8256 bf16 KK 414 .. 440 us = 1.26 .. 1.34 PFLOP/s (a 16 KiB row stride, K = 8192,
// costs 15 %: the rows of a tile fall on the same channels), 16384 x 2048 x 8192 KM 429 .. 450 us = 1.22 .. 1.28 (490 in a pass, behind the launch that wrote dz),
// 8192 x 2048 x 8192 MM 206 .. 216 us = 1.27 .. 1.34; fp32 4096^3 KM 0.99 ms = 0.139.  Bound by the issue of the LDS copies next to the matrix instructions
// (SQ_VALU_MFMA_BUSY 57 % of the cycles); with all rows on one cache line the same loop reaches 1.38.
// 64-byte steps in three to five buffers, or two groups of waves half a period apart, measured 0 .. 15 % slower.
#include <algorithm>

#include "ops.hpp"
#include "ops_launch.hpp"

namespace lsdm {
namespace ops {

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __attribute__((aligned(16))) const unsigned g_zero16[4] = {0, 0, 0, 0};

template <class T> struct Mma;
template <> struct Mma<__bf16> {
    static constexpr int F = 16;                 // rows of a fragment
    typedef bfrag frag; typedef f32x4 acc;
    static constexpr int KI = 1;                 // instructions per fragment
    static __device__ __forceinline__ acc go(frag a, frag b, acc c, int) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<_Float16> {
    static constexpr int F = 16;
    typedef hfrag frag; typedef f32x4 acc;
    static constexpr int KI = 1;
    static __device__ __forceinline__ acc go(frag a, frag b, acc c, int) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {
    static constexpr int F = 32;
    typedef f32x4 frag; typedef f32x16 acc;      // a fragment is four k values, one per instruction
    static constexpr int KI = 4;
    static __device__ __forceinline__ acc go(frag a, frag b, acc c, int i) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0); }
};

// ---- LDS tiles ----------------------------------------------------------------------------------------------------------------
// A step is SB = 128 bytes of the contraction axis.
// KMAJOR: R rows of SB bytes, the 16-byte chunk c of row r at position c ^ swz(r).
// else:   SB / sizeof(T) rows (one per k) of R elements; a block of 16 columns (32 bytes, 16-bit types) or 32 columns (128 bytes, fp32) b of
//         row k at position b ^ swz(k).
// ds_read_b128 takes its 64 lanes in four passes over the 64 banks: lanes 0-3, 12-15, 20-27; 4-11, 16-19, 28-31; and the same 32 lanes further.
// The sixteen rows (fp32: chunks) of a pass fall into sixteen different 16-byte columns of the banks with these two forms (SQ_LDS_BANK_CONFLICT
// from 50 % of the LDS cycles with r & 7 and (r >> 2) & 3 to 0).
constexpr int SB = 128;
template <class T>
__device__ __forceinline__ int swz_k(int r) { return ((r >> 1) & 1) * 2 | ((r >> 3) & 1) * 4 | (sizeof(T) == 4 ? (r >> 4) & 1 : 0); }
template <class T, int R>
__device__ __forceinline__ int swz_m(int k) {
    if constexpr (sizeof(T) == 4) return (k >> 2) & 1;
    else if constexpr (R >= 128) return (k & 3) | ((k >> 3) & 1) << 2;
    else return ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
}

template <class T, int R, bool KMAJOR, int NW>
struct Loader {
    static constexpr int NI = R * SB / 1024 / NW;        // wave instructions (1 KB each) per wave and step
    static constexpr int EC = 16 / (int)sizeof(T), CPR = SB / 16;
    static_assert(R * SB % (1024 * NW) == 0, "whole instructions per wave");
    const char* src[NI];
    int kpos[NI];                                // this lane's k within the step
    long long step;

    __device__ __forceinline__ void init(const void* base, long long ld, int row0, int rows, int k0, int wave, int lane) {
        const T* p = static_cast<const T*>(base);
        step = KMAJOR ? SB : (long long)(SB / (int)sizeof(T)) * ld * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int q = wave * NI + i;
            if constexpr (KMAJOR) {
                const int r = q * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ swz_k<T>(r);
                const int gr = min(row0 + r, rows - 1);
                kpos[i] = c * EC;
                src[i] = reinterpret_cast<const char*>(p + (long long)gr * ld + k0 + c * EC);
            } else {
                constexpr int RB = R * (int)sizeof(T);
                const int o = q * 1024 + lane * 16, k = o / RB, pos = (o % RB) >> 4;
                const int c = sizeof(T) == 4 ? pos ^ (swz_m<T, R>(k) << 3) : (((pos >> 1) ^ swz_m<T, R>(k)) << 1 | (pos & 1));
                int col = row0 + c * EC;
                if (col >= rows) col = 0;        // (columns that no output uses: any valid address)
                kpos[i] = k;
                src[i] = reinterpret_cast<const char*>(p + (long long)(k0 + k) * ld + col);
            }
        }
    }
    // requests the step that starts kleft elements before the end of the contraction range
    __device__ __forceinline__ void issue(unsigned lds, int wave, int kleft) {
        constexpr int BK = SB / (int)sizeof(T);
        if (kleft >= BK) {
#pragma unroll
            for (int i = 0; i < NI; ++i) lds_dma16(src[i], lds + (wave * NI + i) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) lds_dma16(kpos[i] < kleft ? src[i] : reinterpret_cast<const char*>(g_zero16), lds + (wave * NI + i) * 1024);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) src[i] += step;
    }
};

// fragments of one wave: NF blocks of F rows starting at row0 of the tile
template <class T, int R, bool KMAJOR, int NF>
struct Reader {
    typedef Mma<T> MM_;
    typedef typename MM_::frag frag;
    static constexpr int RB = R * (int)sizeof(T);
    static constexpr int KS = sizeof(T) == 4 ? SB / 32 : SB / 64;      // sub-steps of a step (8 fp32 or 32 16-bit k each)
    int off[(KMAJOR && sizeof(T) == 2) || sizeof(T) == 4 ? KS : NF];
    int frow;                                              // (fp32, column tiles)
    __device__ __forceinline__ void init(int row0, int lane) {
        if constexpr (sizeof(T) == 2 && KMAJOR) {
            const int r = row0 + (lane & 15);
#pragma unroll
            for (int s = 0; s < KS; ++s) off[s] = r * SB + (((s * 4 + (lane >> 4)) ^ swz_k<T>(r)) << 4);
        } else if constexpr (sizeof(T) == 2) {
            const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < NF; ++i) off[i] = k * RB + ((((row0 >> 4) + i) ^ swz_m<T, R>(k)) << 5) + (lane & 3) * 8;
        } else if constexpr (KMAJOR) {
            const int r = row0 + (lane & 31);
#pragma unroll
            for (int s = 0; s < KS; ++s) off[s] = r * SB + (((2 * s + (lane >> 5)) ^ swz_k<T>(r)) << 4);
        } else {
            frow = row0;
        }
    }
    __device__ __forceinline__ frag get(const char* tile, int s, int i, int lane) const {
        if constexpr (sizeof(T) == 2 && KMAJOR) {
            return *reinterpret_cast<const frag*>(tile + off[s] + i * 16 * SB);
        } else if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4* lp;
            const char* p = tile + off[i] + s * 32 * RB;
            union { s16x4 h[2]; frag f; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * RB));
            return u.f;
        } else if constexpr (KMAJOR) {
            return *reinterpret_cast<const frag*>(tile + off[s] + i * 32 * SB);
        } else {
            const int h = lane >> 5, b = ((frow >> 5) + i) ^ h;           // swz_m(k) = (k >> 2) & 1 = h for k = 8 s + 4 h + j
            const char* p = tile + (8 * s + 4 * h) * RB + (b << 7) + (lane & 31) * 4;
            frag f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(p + j * RB);
            return f;
        }
    }
};

// ---- epilogue of eight consecutive outputs (row m, columns n ..) ----
template <class T>
__device__ __forceinline__ void epilogue8(const Epilogue& e, float (&z)[8], const float (&bias)[8], long long m, int n, int N) {
    const int cnt = min(8, N - n);
    if (cnt <= 0) return;
    const bool want = e.deriv != nullptr;
    float y[8], d[8], r[8];
    if (e.res) {
        const T* p = static_cast<const T*>(e.res) + m * e.ldr + n;
        load8n(p, cnt, r);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] += bias[j];
    if (e.act == OP_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = z[j];
    } else {
        act8<T>(e.act, z, want, y, d);
        if (want) {
            if (e.form == DERIV_8) {
                unsigned c[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) c[j] = deriv_code8(d[j]);
                store_codes(static_cast<unsigned char*>(e.deriv) + m * e.ldd + n, cnt, c);
            } else if constexpr (sizeof(T) == 2) {
                T v[8];                          // (the 16-bit form travels as T's bits)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __builtin_bit_cast(T, (unsigned short)deriv_code16(d[j]));
                T* p = static_cast<T*>(e.deriv) + m * e.ldd + n;
                if (cnt >= 8) {
                    typename Piece<T>::frag f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = v[j];
                    typename Piece<T>::mem* q = reinterpret_cast<typename Piece<T>::mem*>(p);
                    if (e.stream) __builtin_nontemporal_store(f, q); else *q = f;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (j < cnt) p[j] = v[j];
                }
            } else {
                store8n(static_cast<float*>(e.deriv) + m * e.ldd + n, cnt, d);
            }
        }
    }
    if (e.res) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] += r[j];
    }
    T* p = static_cast<T*>(e.out) + m * e.ldo + n;
    if (e.stream) store8n<true>(p, cnt, y); else store8n(p, cnt, y);
}
template <class T>
__device__ __forceinline__ void bias8(const Epilogue& e, int n, int N, float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = e.bias && n + j < N ? param<T>(e.bias, e.bias_f32, n + j) : 0.0f;
}

// out[c] = sum over the chunks of part[chunk][c]: 64 columns per work-group, its waves take every nw-th chunk, joined in order
template <class T>
__device__ __forceinline__ void colsum_join(const GemmArgs& g, int block, float* red) {
    const int t = threadIdx.x, c = block * 64 + (t & 63), q = t >> 6, nw = (int)blockDim.x >> 6;
    float s = 0.0f;
    if (c < g.cs_n)                              // (sixteen loads in flight: the products' tiles must not wait for this work-group)
#pragma unroll 4
        for (int k = q; k < g.cs_chunks; k += nw) s += g.cs_part[(long long)k * g.cs_n + c];
    red[t] = s;
    wg_sync();
    if (q == 0 && c < g.cs_n) {
        for (int k = 1; k < nw; ++k) s += red[k * 64 + t];
        store_param<T>(g.cs_out, g.cs_f32, c, s);
    }
}
template <class T>
__global__ __launch_bounds__(256) void colsum_join_kernel(GemmArgs g) {
    __shared__ float red[256];
    colsum_join<T>(g, (int)blockIdx.x, red);
}

// ---- the tile kernel ------------------------------------------------------------------------------------------------------------
template <class T, int BM, int BN, int WGM, int WGN, bool AKM, bool BKM, int WPE>
__global__ __launch_bounds__(64 * WGM * WGN, WPE) void gemm_kernel(GemmArgs g) {
    typedef Mma<T> MM_;
    constexpr int NW = WGM * WGN, TM = BM / WGM, TN = BN / WGN, F = MM_::F, FM = TM / F, FN = TN / F;
    constexpr int BK = SB / (int)sizeof(T), KS = Reader<T, BM, AKM, FM>::KS;
    constexpr int TA = BM * SB, TB = BN * SB, ST = TA + TB;
    constexpr int RW = TM < 64 ? TM : 64, PITCH = TN * 4 + 16, EPI = RW * PITCH;        // epilogue: RW rows of a wave's tile at a time, in fp32
    constexpr int BYTES = 2 * ST > EPI * NW ? 2 * ST : EPI * NW;
    __shared__ __attribute__((aligned(1024))) char lds[BYTES];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / WGN, wn = wave - wm * WGN;

    if ((int)blockIdx.x >= g.blocks) { colsum_join<T>(g, (int)blockIdx.x - g.blocks, reinterpret_cast<float*>(lds)); return; }

    // tiles in groups of 8 rows of tiles, an XCD walks a contiguous range: the tiles in flight on an XCD share their operands in its L2
    const int tiles = g.tiles_m * g.tiles_n;
    int v = xcd_remap((int)blockIdx.x, g.blocks);
    const int ks = v / tiles;
    v -= ks * tiles;
    const int per = 8 * g.tiles_n, grp = v / per, gm = min(8, g.tiles_m - grp * 8), in = v - grp * per;
    const int tm = grp * 8 + in % gm, tn = in / gm;
    const int m0 = tm * BM, n0 = tn * BN;
    const int k_lo = ks * g.kchunk, k_hi = min(g.K, k_lo + g.kchunk);
    const int nk = k_hi > k_lo ? (k_hi - k_lo + BK - 1) / BK : 0;

    Loader<T, BM, AKM, NW> la;
    Loader<T, BN, BKM, NW> lb;
    la.init(g.A, g.lda, m0, g.M, k_lo, wave, lane);
    lb.init(g.B, g.ldb, n0, g.N, k_lo, wave, lane);
    Reader<T, BM, AKM, FM> ra;
    Reader<T, BN, BKM, FN> rb;
    ra.init(wm * TM, lane);
    rb.init(wn * TN, lane);
    const unsigned base = lds_addr(lds);

    typename MM_::acc acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < (int)(sizeof(typename MM_::acc) / 4); ++r) acc[i][j][r] = 0.0f;

    auto issue = [&](int buf, int it) {
        la.issue(base + buf * ST, wave, k_hi - k_lo - it * BK);
        lb.issue(base + buf * ST + TA, wave, k_hi - k_lo - it * BK);
    };
    if (nk > 0) issue(0, 0);
    int buf = 0;
    for (int it = 0; it < nk; ++it) {
        lds_dma_wait();                          // this step's pieces have landed, for every wave behind the barrier
        wg_sync();
        if (it + 1 < nk) issue(buf ^ 1, it + 1); // into the buffer of step it - 1, which every wave has read
        const char* ta = lds + buf * ST;
        const char* tb = ta + TA;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            typename MM_::frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = rb.get(tb, s, j, lane);
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = ra.get(ta, s, i, lane);
#pragma unroll
            for (int q = 0; q < MM_::KI; ++q)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = MM_::go(fb[j], fa[i], acc[i][j], q);
        }
        if constexpr (sizeof(T) == 2 && (BM == 256 || (BM == 128 && !AKM))) {
            // The compiler's own order reads a fragment, waits for it and uses it; this one starts with the B fragments and two of A and keeps every later
            // read that far ahead of its use (256: KK 595 -> 573 us at 16384 x 2048 x 8192, KM 229 -> 214, MM 229 -> 211 at 8192 x 4096 x 4096; 128 MM 253 -> 236,
            // but 128 KK and KM 3 .. 5 % slower, 64 the same: not there).
            constexpr int RA = AKM ? 1 : 2, RB = BKM ? 1 : 2, READS = KS * (FM * RA + FN * RB), AHEAD = FN * RB + 2 * RA, MF = KS * FM * FN;
            constexpr int PERR = MF / (READS - AHEAD);
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);            // LDS reads
#pragma unroll
            for (int g = 0; g < READS - AHEAD; ++g) {
                __builtin_amdgcn_sched_group_barrier(0x8, PERR, 0);           // matrix instructions
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, MF - PERR * (READS - AHEAD), 0);
        }
        buf ^= 1;
    }

    // epilogue: the wave's tile through its own piece of LDS, RW rows at a time
    wg_sync();
    char* mine = lds + wave * EPI;
    constexpr int CPR = TN / 8, RPI = 64 / CPR;          // 8-column pieces per row, rows per wave instruction
    const int en = n0 + wn * TN + (lane % CPR) * 8;
    float bias[8];
    bias8<T>(g.e, en, g.N, bias);
#pragma unroll
    for (int half = 0; half < TM / RW; ++half) {
#pragma unroll
        for (int i = 0; i < RW / F; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const typename MM_::acc& a = acc[half * (RW / F) + i][j];
                if constexpr (F == 16) {
                    *reinterpret_cast<f32x4*>(mine + (i * 16 + (lane & 15)) * PITCH + (j * 16 + (lane >> 4) * 4) * 4) = a;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f32x4*>(mine + (i * 32 + (lane & 31)) * PITCH + (j * 32 + 8 * q + 4 * (lane >> 5)) * 4) =
                            f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                }
            }
        const int em = m0 + wm * TM + half * RW + lane / CPR;
#pragma unroll 1
        for (int r = 0; r < RW; r += RPI) {
            const int m = em + r;
            float z[8];
            const f32x4* zp = reinterpret_cast<const f32x4*>(mine + (r + lane / CPR) * PITCH + (lane % CPR) * 32);
            const f32x4 z0 = zp[0], z1 = zp[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) { z[j] = z0[j]; z[4 + j] = z1[j]; }
            if (m < g.M) {
                if (g.splits > 1) {
                    float* p = g.part + ((long long)ks * g.M + m) * g.N + en;
                    store8n(p, g.N - en, z);
                } else {
                    epilogue8<T>(g.e, z, bias, m, en, g.N);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// joins the partial sums of a split contraction, in order, and applies the epilogue: one thread per eight outputs of a row
template <class T>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs g, long long pieces, int ppr) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const long long m = i / ppr;
    const int n = (int)(i - m * ppr) * 8;
    float z[8] = {0, 0, 0, 0, 0, 0, 0, 0}, bias[8];
    bias8<T>(g.e, n, g.N, bias);
    const long long slab = (long long)g.M * g.N;
    const float* p = g.part + m * g.N + n;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
        float v[8];
        load8n(p + s * slab, g.N - n, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] += v[j];
    }
    epilogue8<T>(g.e, z, bias, m, n, g.N);
}

// ---- few rows: M <= 16 MB.  A work-group owns 16 columns; its waves split k and join through LDS.  W is read once, straight into fragments; any K and any
// alignment.  Small layers are bound by latency (1 x 512 -> 256 fp32: one launch of 3 us), one row of a wide one by W's read (bf16, W out of HBM: 1 x 8192 ->
// 8192 31.7 us = 4.2 TB/s, -> 32000 102 us = 5.1; fp32 60.5 us = 4.4 and 210 us = 5.0).  More rows are bound by reading x again in every work-group: 8192 -> 8192
// bf16 41 us with 16 rows, 83 with 64 (fp32 79 and 188). ----
template <class T>
__device__ __forceinline__ typename Mma<T>::frag row_frag(const T* p, int k, int K) {
    typename Mma<T>::frag f;
    constexpr int E = sizeof(T) == 4 ? 4 : 8;
    if (k + E <= K) return *reinterpret_cast<const typename Piece<T>::mem*>(p + k);
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = k + j < K ? p[k + j] : (T)0.0f;
    return f;
}
template <class T> struct RowMma {
    static __device__ __forceinline__ f32x4 go(typename Mma<T>::frag a, typename Mma<T>::frag b, f32x4 c) { return Mma<T>::go(a, b, c, 0); }
};
template <> struct RowMma<float> {
    static __device__ __forceinline__ f32x4 go(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};
template <class T, int MB>
__global__ __launch_bounds__(1024) void rows_kernel(GemmArgs g) {
    constexpr int E = sizeof(T) == 4 ? 4 : 8, KSTEP = 4 * E;        // k of one instruction group over the four 16-lane groups
    __shared__ float part[MB == 4 ? 8 : 16][MB * 16][16 + 4];        // (one slab per wave: launch_rows_t starts at most that many)
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, nw = (int)blockDim.x >> 6;
    const int n0 = (int)blockIdx.x * 16;
    const T* w = static_cast<const T*>(g.B) + (long long)min(n0 + (lane & 15), g.N - 1) * g.ldb;
    const T* x[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = static_cast<const T*>(g.A) + (long long)min(b * 16 + (lane & 15), g.M - 1) * g.lda;
    f32x4 acc[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (g.K + KSTEP - 1) / KSTEP;
    constexpr int U = MB >= 4 ? 2 : 4;
    const int kl = (lane >> 4) * E;
    for (int s0 = wave; s0 < steps; s0 += nw * U) {
        typename Mma<T>::frag fw[U], fx[U][MB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s0 + u * nw) * KSTEP + kl;
            fw[u] = row_frag<T>(w, k, g.K);
#pragma unroll
            for (int b = 0; b < MB; ++b) fx[u][b] = row_frag<T>(x[b], k, g.K);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[b] = RowMma<T>::go(fw[u], fx[u][b], acc[b]);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) *reinterpret_cast<f32x4*>(&part[wave][b * 16 + (lane & 15)][(lane >> 4) * 4]) = acc[b];
    wg_sync();
    if (t < MB * 32) {
        const int m = t >> 1, c = (t & 1) * 8;
        if (m < g.M) {
            float z[8] = {0, 0, 0, 0, 0, 0, 0, 0}, bias[8];
            for (int v = 0; v < nw; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] += part[v][m][c + j];
            bias8<T>(g.e, n0 + c, g.N, bias);
            epilogue8<T>(g.e, z, bias, m, n0 + c, g.N);
        }
    }
}

// ---- what the products need prepared, up to three jobs in one launch (blockIdx.z) ----
//   dst (rows, ldd) = src (rows, n) * d, or the values of an 8-bit checkpoint; columns n .. ldd - 1 are zeroed, so that rows no 16-byte load divides
//   become rows that one does.  part[blockIdx.y][c] = the work-group's sum of the fp32 products over its rows (a fixed order).
// Bound by HBM: each operand is read once, dst is written once (16384 x 8192 bf16 with a 16-bit a'(z): 178 us = 4.5 TB/s).
// one row's piece: v = the source's values times a'(z).  Whole pieces are loaded outside any branch on the lane, so that several rows' are in flight.
template <class T, bool WHOLE>
__device__ __forceinline__ void prep_piece(const PrepJob& a, long long r, int c0, int n, float (&v)[8]) {
    typedef typename Piece<T>::frag frag;
    typedef typename Piece<T>::mem mem;
    const long long at = r * a.n + c0;
    if (a.exps) {
        const unsigned char* q = static_cast<const unsigned char*>(a.src) + at;
        const u32x2 w = WHOLE ? *reinterpret_cast<const codes8*>(q) : load_codes(q, n);
        const float step = n > 0 ? exp8_step(a.exps[r * ((a.n + 31) >> 5) + (c0 >> 5)]) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)((int)(w[j >> 2] << (24 - 8 * (j & 3))) >> 24) * step;
    } else {
        const T* p = static_cast<const T*>(a.src) + r * a.lds + c0;
        if constexpr (WHOLE) load8(p, v); else load8n(p, n, v);
    }
    if (a.form == DERIV_NONE) return;
    float d[8];
    if (a.form == DERIV_8) {
        const unsigned char* q = static_cast<const unsigned char*>(a.deriv) + at;
        const u32x2 w = WHOLE ? *reinterpret_cast<const codes8*>(q) : load_codes(q, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = deriv_value8((w[j >> 2] >> (8 * (j & 3))) & 255u);
    } else if constexpr (sizeof(T) == 2) {
        const T* q = static_cast<const T*>(a.deriv) + at;
        if constexpr (WHOLE) {
            const frag f = *reinterpret_cast<const mem*>(q);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = deriv_value16(__builtin_bit_cast(unsigned short, (T)f[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = j < n ? deriv_value16(__builtin_bit_cast(unsigned short, q[j])) : 0.0f;
        }
    } else {
        const float* q = static_cast<const float*>(a.deriv) + at;
        if constexpr (WHOLE) load8(q, d); else load8n(q, n, d);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = WHOLE || j < n ? v[j] * d[j] : 0.0f;
}
template <class T>
__global__ __launch_bounds__(256) void prep_kernel(PrepArgs args) {
    const PrepJob& a = args.job[blockIdx.z];
    __shared__ float red[8][256 + 8];
    const int t = threadIdx.x, tc = t & 31, tr = t >> 5;
    const int c0 = ((int)blockIdx.x * 32 + tc) * 8;
    if ((int)blockIdx.y >= a.chunks || (long long)blockIdx.x * 256 >= (a.dst && a.ldd > a.n ? a.ldd : a.n)) return;      // (whole work-groups)
    const long long per = (a.rows + a.chunks - 1) / a.chunks, lo = (long long)blockIdx.y * per, hi = min(a.rows, lo + per);
    const int n = max(0, min(8, a.n - c0));
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    T* dst = static_cast<T*>(a.dst) + c0;
    if (n == 8) {
        long long r = lo + tr;
        for (; r + 24 < hi; r += 32) {
            float v[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) prep_piece<T, true>(a, r + 8 * u, c0, 8, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (a.dst) store8(dst + (r + 8 * u) * a.ldd, v[u]);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += v[u][j];
            }
        }
        for (; r < hi; r += 8) {
            float v[8];
            prep_piece<T, true>(a, r, c0, 8, v);
            if (a.dst) store8(dst + r * a.ldd, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
    } else if (n > 0 || (a.dst && c0 < a.ldd)) {
#pragma unroll 4
        for (long long r = lo + tr; r < hi; r += 8) {
            float v[8];
            prep_piece<T, false>(a, r, c0, n, v);
            if (a.dst) store8(dst + r * a.ldd, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[tr][tc * 8 + j] = s[j];
    wg_sync();
    const int c = (int)blockIdx.x * 256 + t;
    if (c < a.n) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += red[q][t];
        a.part[(long long)blockIdx.y * a.n + c] = v;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------
namespace {

template <class T, int BM, int BN, int WGM, int WGN, int WPE>
void launch_layout(const GemmArgs& g, int layout, unsigned grid, hipStream_t st) {
    const dim3 b(64 * WGM * WGN);
    if (layout == KK) hipLaunchKernelGGL((gemm_kernel<T, BM, BN, WGM, WGN, true, true, WPE>), dim3(grid), b, 0, st, g);
    else if (layout == KM) hipLaunchKernelGGL((gemm_kernel<T, BM, BN, WGM, WGN, true, false, WPE>), dim3(grid), b, 0, st, g);
    else hipLaunchKernelGGL((gemm_kernel<T, BM, BN, WGM, WGN, false, false, WPE>), dim3(grid), b, 0, st, g);
}

}  // namespace

template <class T>
void launch_gemm_t(const GemmPlan& p, GemmArgs g, int layout, hipStream_t st) {
    g.tiles_m = p.tiles_m; g.tiles_n = p.tiles_n; g.splits = p.splits; g.kchunk = p.kchunk;
    g.blocks = p.tiles_m * p.tiles_n * p.splits;
    const unsigned grid = (unsigned)(g.blocks + (g.cs_out ? (g.cs_n + 63) / 64 : 0));
    if constexpr (sizeof(T) == 2) {
        if (p.tile == 256) launch_layout<T, 256, 256, 2, 4, 2>(g, layout, grid, st);
        else if (p.tile < p.tile_n) launch_layout<T, 64, 128, 2, 2, 2>(g, layout, grid, st);
    }
    if (p.tile == 128) launch_layout<T, 128, 128, 2, 2, 2>(g, layout, grid, st);
    else if (p.tile_n == 64) launch_layout<T, 64, 64, 2, 2, 2>(g, layout, grid, st);
    if (p.splits > 1) {
        const int ppr = (g.N + 7) / 8;
        const long long pieces = (long long)g.M * ppr;
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, g, pieces, ppr);
    }
}

template <class T>
void launch_rows_t(const GemmArgs& g, hipStream_t st) {
    const dim3 grid((unsigned)((g.N + 15) / 16));
    constexpr int KSTEP = sizeof(T) == 4 ? 16 : 32;
    const int steps = (g.K + KSTEP - 1) / KSTEP;
    // waves of a work-group: enough that a wave's share of k is about one round of loads (four instruction groups), at most 16 (8 with four row
    // blocks: the slabs of the join)
    int nw = 1;
    while (nw < (g.M > 32 ? 8 : 16) && nw * 4 < steps) nw *= 2;
    const dim3 b(64 * nw);
    auto go = [&](auto mb) {
        constexpr int MB = decltype(mb)::value;
        // the join needs 32 MB threads
        const dim3 bb(b.x < 32 * MB ? 32 * MB : b.x);
        hipLaunchKernelGGL((rows_kernel<T, MB>), grid, bb, 0, st, g);
    };
    if (g.M <= 16) go(std::integral_constant<int, 1>{});
    else if (g.M <= 32) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
}

void launch_gemm(int dtype, const GemmPlan& p, const GemmArgs& g, int layout, hipStream_t st) {
    if (dtype == 0) launch_gemm_t<float>(p, g, layout, st);
    else if (dtype == 1) launch_gemm_t<__bf16>(p, g, layout, st);
    else launch_gemm_t<_Float16>(p, g, layout, st);
}
void launch_rows(int dtype, const GemmArgs& g, hipStream_t st) {
    if (dtype == 0) launch_rows_t<float>(g, st);
    else if (dtype == 1) launch_rows_t<__bf16>(g, st);
    else launch_rows_t<_Float16>(g, st);
}
void launch_prep(int dtype, const PrepArgs& a, int jobs, hipStream_t st) {
    unsigned x = 1, y = 1;
    for (int i = 0; i < jobs; ++i) {
        const long long cols = a.job[i].ldd > a.job[i].n ? a.job[i].ldd : a.job[i].n;
        x = std::max(x, (unsigned)((cols + 255) / 256));
        y = std::max(y, (unsigned)a.job[i].chunks);
    }
    const dim3 grid(x, y, (unsigned)jobs);
    if (dtype == 0) hipLaunchKernelGGL((prep_kernel<float>), grid, dim3(256), 0, st, a);
    else if (dtype == 1) hipLaunchKernelGGL((prep_kernel<__bf16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((prep_kernel<_Float16>), grid, dim3(256), 0, st, a);
}
void launch_colsum_join(int dtype, const GemmArgs& g, hipStream_t st) {
    const dim3 grid((unsigned)((g.cs_n + 63) / 64));
    if (dtype == 0) hipLaunchKernelGGL((colsum_join_kernel<float>), grid, dim3(256), 0, st, g);
    else if (dtype == 1) hipLaunchKernelGGL((colsum_join_kernel<__bf16>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((colsum_join_kernel<_Float16>), grid, dim3(256), 0, st, g);
}

}  // namespace ops
}  // namespace lsdm
