// Launchers of the public operators' kernels (host side of ops_gemm.hip, ops_norm.hip, ops_pack8.hip).
#pragma once
#include <type_traits>

#include "ops.hpp"

namespace lsdm {
namespace ops {

constexpr int kNormMaxWidth = 16384;      // (1024 threads, 16 values each)

struct GemmPlan { int tile = 0, tile_n = 0, tiles_m = 0, tiles_n = 0, splits = 1, kchunk = 0; };

struct PrepJob {
    const void* src = nullptr; long long lds = 0;
    const unsigned char* exps = nullptr;             // not NULL: src holds the codes of an 8-bit checkpoint (dense rows)
    const void* deriv = nullptr; int form = DERIV_NONE;               // dense rows
    void* dst = nullptr; long long ldd = 0;          // NULL: only the column sums; ldd a multiple of 8 elements, rows 16-byte aligned
    float* part = nullptr;                           // (chunks, n) column sums, or NULL
    long long rows = 0; int n = 0, chunks = 1;
};
struct PrepArgs { PrepJob job[3]; };

struct NormArgs {
    long long rows = 0; int D = 0; float eps = 0.0f;
    const void* x = nullptr; long long ldx = 0;
    const void *w = nullptr, *b = nullptr; int param_f32 = 0;
    void* y = nullptr;                               // (rows, D) dense
    float *mean = nullptr, *rstd = nullptr;          // (rows)
    signed char* codes = nullptr; unsigned char* exps = nullptr;      // 8-bit checkpoint of h: written by the forward pass, read by the backward
    const void* dy = nullptr; long long lddy = 0;
    void* dx = nullptr;                              // (rows, D) dense, or NULL
    float* part = nullptr;                           // (grid, 2, D) partial sums of dw and db, or NULL
};
struct Pack8Args {
    long long rows = 0; int D = 0;
    const void* x = nullptr; long long ldx = 0;
    signed char* codes = nullptr; unsigned char* exps = nullptr;      // (rows, D), (rows, ceil(D / 32))
    void* out = nullptr;                             // (rows, D) dense
};

void launch_gemm(int dtype, const GemmPlan& p, const GemmArgs& g, int layout, hipStream_t st);
void launch_rows(int dtype, const GemmArgs& g, hipStream_t st);
void launch_prep(int dtype, const PrepArgs& a, int jobs, hipStream_t st);
void launch_colsum_join(int dtype, const GemmArgs& g, hipStream_t st);
void launch_norm(int dtype, const NormArgs& a, int grid, bool backward, hipStream_t st);
void launch_norm_join(int dtype, const float* part, int groups, int D, void* dw, void* db, int param_f32, hipStream_t st);
int norm_threads(int D);                             // threads of a work-group of the norm kernels, and the rows it has in flight
int norm_rows_per_group(int D);
void launch_pack8(int dtype, const Pack8Args& a, hipStream_t st);
void launch_unpack8(int dtype, const Pack8Args& a, hipStream_t st);

}  // namespace ops
}  // namespace lsdm
