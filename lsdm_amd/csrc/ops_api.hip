// C entry points of the public operators (include/lsdm_hip.h: lsdm_linear*, lsdm_layer_norm*, lsdm_pack8, lsdm_unpack8): argument checks, the
// choice of a kernel variant, and the layout of the caller's scratch memory.  They need no context: any thread, any device, any stream; a
// failure's message is the calling thread's (lsdm_last_error(NULL)).
#include "../../include/lsdm_hip.h"

#include <cstdarg>
#include <cstdio>

#include "kernels.hpp"
#include "ops_launch.hpp"

using namespace lsdm;
using namespace lsdm::ops;

namespace {

int refuse(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_thread_error(buf);
    return code;
}

struct OnDevice {                                 // the entry point's device, the caller's restored on return
    int prev = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev == device) { ok = true; prev = -1; return; }
        ok = device >= 0 && hipSetDevice(device) == hipSuccess;
        if (!ok) { (void)hipGetLastError(); refuse(LSDM_ERR_HIP, "hipSetDevice(%d) failed", device); }
    }
    ~OnDevice() { if (prev >= 0) (void)hipSetDevice(prev); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LSDM_OK : refuse(LSDM_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr int64_t kMaxSize = (int64_t)1 << 30;
constexpr int64_t kMaxOut = (int64_t)1 << 25;     // rows of W: a launch's work-groups go with them, up to 1024 threads for every 16 of them
constexpr int kCUs = 256;                         // MI355X
constexpr int64_t kMaxThreads = (int64_t)1 << 31; // threads of a launch (the runtime takes fewer than 2^32; column-sum work-groups may come on top)
int esize(int dtype) { return dtype == LSDM_F32 ? 4 : 2; }
bool dtype_ok(int d) { return d == LSDM_F32 || d == LSDM_BF16 || d == LSDM_F16; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows of `width` elements `ld` apart whose 16-byte pieces are whole and aligned
bool rows16(const void* p, int64_t ld, int64_t width, int es) { return aligned16(p) && ld * es % 16 == 0 && width * es % 16 == 0; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// carves the caller's scratch memory; with base == NULL it only adds up
struct Carve {
    char* base;
    int64_t used = 0;
    void* take(int64_t bytes) {
        void* p = base ? base + used : nullptr;
        used += up(bytes, 256);
        return p;
    }
};

// Tile and split of C (M, N) with contraction K, by an estimate of the launch's time.  A tile kind keeps up to `resident` work-groups on a CU; a
// 128-byte step of the contraction takes max(alone, shared * n) us with n of them there, prologue and epilogue fixed + each * n us.  The grid runs
// in full rounds of 256 `resident` work-groups and a last, thinner one; a split contraction adds the join's launch and its traffic (the partial sums
// are written once and read once).  The constants are fitted to timed launches of every tile and 1 .. 32 splits in the three operand layouts (16 bits:
// 177 shapes log-uniform over 16 .. 16384; fp32: 35) of products WITHOUT activation and derivative: among those the estimate's choice is within 1 % of the best
// one in the mean, within 20 % at worst.  Without the 64 x 128 tile it would be 1.5 % (4928 x 2048 x 512: 22 -> 18 us, 704 x 1640 x 3952: 37 -> 25).  What an
// epilogue costs is not in the estimate, though it is a third of a large product with gelu and its derivative: 8192 x 1024 -> 4096 runs 114 us where 62 are
// expected, and another tile takes 98.
struct TileCost { int tile, tile_n, resident; float alone, shared, fixed, each; };
const TileCost kHalfTiles[] = {{256, 256, 1, 0.0f, 1.36f, 8.5f, 0.61f}, {128, 128, 2, 0.78f, 0.39f, 1.87f, 1.4f}, {64, 128, 3, 0.395f, 0.28f, 1.98f, 0.74f},
                               {64, 64, 5, 0.315f, 0.19f, 2.31f, 0.08f}};
const TileCost kSingleTiles[] = {{128, 128, 2, 0.40f, 1.61f, 4.9f, 0.13f}, {64, 64, 4, 0.52f, 0.49f, 0.06f, 0.09f}};
constexpr float kJoinLaunch = 2.6f, kJoinBytesPerUs = 3.6e6f;

GemmPlan plan(int64_t M, int64_t N, int64_t K, int dtype) {
    const bool f32 = dtype == LSDM_F32;
    const int bk = f32 ? 32 : 64, kinds = f32 ? 2 : 4;
    const int64_t steps = (K + bk - 1) / bk;
    GemmPlan best;
    float best_us = 0.0f;
    for (int i = 0; i < kinds; ++i) {
        const TileCost& k = f32 ? kSingleTiles[i] : kHalfTiles[i];
        const int64_t tm = (M + k.tile - 1) / k.tile, tn = (N + k.tile_n - 1) / k.tile_n;
        const int64_t most = kMaxThreads / (k.tile == 256 ? 512 : 256);
        if (tm * tn > most) continue;
        for (int s = 1; s <= 32; s = s < 4 ? s + 1 : s * 2) {
            if (s > 1 && (steps < 2 * s || tm * tn * s > most || M * ((N + 7) / 8) > kMaxThreads)) break;      // (the join: a thread per eight outputs)
            const int64_t per = (steps + s - 1) / s;
            if ((steps + per - 1) / per != s) continue;
            const int64_t groups = tm * tn * s, round = (int64_t)kCUs * k.resident, full = groups / round, rest = groups - full * round;
            auto cost = [&](float n) { return (float)per * (k.alone > k.shared * n ? k.alone : k.shared * n) + k.fixed + k.each * n; };
            float us = (float)full * cost((float)k.resident) + (rest ? cost((float)((rest + kCUs - 1) / kCUs)) : 0.0f);
            if (s > 1) us += kJoinLaunch + (float)(s + 1) * (float)M * (float)N * 4.0f / kJoinBytesPerUs;
            if (best.tile == 0 || us < best_us) {
                best_us = us;
                best.tile = k.tile; best.tile_n = k.tile_n; best.tiles_m = (int)tm; best.tiles_n = (int)tn; best.splits = s; best.kchunk = (int)(per * bk);
            }
        }
    }
    return best;
}

int64_t part_bytes(const GemmPlan& p, int64_t M, int64_t N) { return p.splits > 1 ? (int64_t)p.splits * M * N * 4 : 0; }

// row chunks of a preparation job: about 2048 work-groups in all with at least 32 rows each (four per thread, whose loads are in flight together); fewer
// rows where there would be less than a work-group for every CU.  The column sums' join reads one row per chunk.
int prep_chunks(int64_t rows, int64_t cols) {
    const int64_t cb = (cols + 255) / 256, most = (rows + 7) / 8;
    int64_t c = (rows + 31) / 32, fill = (kCUs + cb - 1) / cb;
    if (fill > most) fill = most;
    if (c < fill) c = fill;
    if (c > 2048 / cb) c = 2048 / cb;
    if (c > 1024) c = 1024;
    return c < 1 ? 1 : (int)c;
}

constexpr int64_t kFewRows = 64;                  // products with at most this many rows run on rows_kernel

struct Fwd { bool rows, xpad, wpad; GemmPlan p; void *x, *w; float* part; int64_t bytes; };
Fwd forward_layout(int dtype, int64_t M, int64_t N, int64_t K, bool x_ok, bool w_ok, void* ws) {
    Fwd f{};
    Carve c{static_cast<char*>(ws)};
    f.rows = M <= kFewRows;
    if (!f.rows) {
        const int64_t kp = up(K, 8);
        f.xpad = !x_ok; f.wpad = !w_ok;
        f.p = plan(M, N, K, dtype);
        if (f.xpad) f.x = c.take(M * kp * esize(dtype));
        if (f.wpad) f.w = c.take(N * kp * esize(dtype));
        f.part = static_cast<float*>(c.take(part_bytes(f.p, M, N)));
    }
    f.bytes = c.used;
    return f;
}

struct Bwd { bool dz, xpad, wpad; int chunks; int64_t ldz, kp; GemmPlan px, pw; void *z, *x, *w; float *cs, *partx, *partw; int64_t bytes; };
Bwd backward_layout(int dtype, int64_t M, int64_t N, int64_t K, bool dx, bool dw, bool db, bool deriv, bool codes, bool dy_ok, bool x_ok, bool w_ok,
                    void* ws) {
    Bwd b{};
    Carve c{static_cast<char*>(ws)};
    const int es = esize(dtype);
    b.kp = up(K, 8); b.ldz = up(N, 8);
    b.dz = (dx || dw) && (deriv || !dy_ok);
    b.xpad = dw && (codes || !x_ok);
    b.wpad = dx && !w_ok;
    b.chunks = prep_chunks(M, b.ldz);
    if (b.dz) b.z = c.take(M * b.ldz * es);
    if (db) b.cs = static_cast<float*>(c.take((int64_t)b.chunks * N * 4));
    if (b.xpad) b.x = c.take(M * b.kp * es);
    if (b.wpad) b.w = c.take(N * b.kp * es);
    if (dx) { b.px = plan(M, K, N, dtype); b.partx = static_cast<float*>(c.take(part_bytes(b.px, M, K))); }
    if (dw) { b.pw = plan(N, K, M, dtype); b.partw = static_cast<float*>(c.take(part_bytes(b.pw, N, K))); }
    b.bytes = c.used;
    return b;
}

// a job that copies rows of n elements into rows of ldd >= n, zero-padded
PrepJob padded(int dtype, const void* src, int64_t lds, int64_t rows, int64_t n, void* dst, int64_t ldd) {
    PrepJob j;
    j.src = src; j.lds = lds; j.dst = dst; j.ldd = ldd; j.rows = rows; j.n = (int)n; j.chunks = prep_chunks(rows, ldd);
    return j;
}
// rows made of whole 128-byte lines
bool whole_lines(const void* p, int64_t width, int es) { return ((uintptr_t)p & 127) == 0 && width * es % 128 == 0; }
int deriv_form(int dtype, int flags) { return flags & LSDM_OP_DERIV8 ? DERIV_8 : dtype == LSDM_F32 ? DERIV_F32 : DERIV_16; }

int check_linear(int dtype, int64_t M, int64_t N, int64_t K) {
    if (!dtype_ok(dtype)) return refuse(LSDM_ERR_ARG, "lsdm_linear: unknown dtype %d", dtype);
    if (M < 1 || N < 1 || K < 1 || M > kMaxSize || N > kMaxOut || K > kMaxSize)
        return refuse(LSDM_ERR_ARG, "lsdm_linear: sizes M = %lld, K = %lld must lie in [1, 2^30], N = %lld in [1, 2^25]", (long long)M, (long long)K, (long long)N);
    return LSDM_OK;
}

// Work-groups of the norm kernels.  Each loads the parameters once, and in the backward pass leaves one partial row of dw and db: enough threads on a
// CU to keep HBM busy, no more (backward, 32768 x 2048: bf16 1024 threads per CU 95 us, 512 of them 145 us, 1536 of them 101 us; fp32 512 of them
// 148 us, 1024 of them 157 us; forward 2048 and 4096 of them the same).
int norm_grid(int64_t rows, int D, bool backward, int es) {
    const int threads = norm_threads(D), rpg = norm_rows_per_group(D);
    const int64_t need = (rows + rpg - 1) / rpg, per_cu = (backward ? (es == 4 ? 512 : 1024) : 2048) / threads, cap = kCUs * (per_cu > 1 ? per_cu : 1);
    return (int)(need < cap ? need : cap);
}

}  // namespace

extern "C" {

int64_t lsdm_linear_workspace(int dtype, int flags, int64_t M, int64_t N, int64_t K) {
    if (check_linear(dtype, M, N, K) != LSDM_OK) return LSDM_ERR_ARG;
    const bool x_ok = !(flags & LSDM_OP_X_UNALIGNED), w_ok = !(flags & LSDM_OP_W_UNALIGNED);
    if (!(flags & LSDM_OP_BACKWARD)) return forward_layout(dtype, M, N, K, x_ok, w_ok, nullptr).bytes;
    return backward_layout(dtype, M, N, K, flags & LSDM_OP_DX, flags & LSDM_OP_DW, flags & LSDM_OP_DB, flags & LSDM_OP_DERIV, flags & LSDM_OP_CODES,
                           !(flags & LSDM_OP_DY_UNALIGNED), x_ok, w_ok, nullptr).bytes;
}

int64_t lsdm_linear_plan(int dtype, int64_t M, int64_t N, int64_t K) {
    if (check_linear(dtype, M, N, K) != LSDM_OK) return LSDM_ERR_ARG;
    const GemmPlan p = plan(M, N, K, dtype);
    return (int64_t)p.tile << 32 | (int64_t)p.tile_n << 16 | (p.tile ? p.splits : 0);
}

int lsdm_linear(int device, int dtype, int activation, int flags, int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* w, int64_t ldw,
                const void* bias, const void* residual, int64_t ldr, void* y, void* deriv, void* ws, int64_t ws_bytes, void* stream) {
    if (const int rc = check_linear(dtype, M, N, K)) return rc;
    if (activation < 0 || activation >= LSDM_ACT_COUNT) return refuse(LSDM_ERR_ARG, "lsdm_linear: unknown activation %d", activation);
    if (!x || !w || !y) return refuse(LSDM_ERR_ARG, "lsdm_linear: x, w and y must not be NULL");
    if (ldx < K || ldw < K || (residual && ldr < N)) return refuse(LSDM_ERR_ARG, "lsdm_linear: a row stride is shorter than its row");
    const int es = esize(dtype);
    const bool x_ok = rows16(x, ldx, K, es), w_ok = rows16(w, ldw, K, es);
    const Fwd f = forward_layout(dtype, M, N, K, x_ok, w_ok, ws);
    if (!f.rows && !f.p.tile) return refuse(LSDM_ERR_ARG, "lsdm_linear: the result has more tiles than a launch can hold");
    if (f.bytes > 0 && (!ws || ws_bytes < f.bytes || !aligned16(ws)))
        return refuse(LSDM_ERR_ARG, "lsdm_linear: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)ws_bytes, (long long)f.bytes);
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GemmArgs g;
    g.M = (int)M; g.N = (int)N; g.K = (int)K;
    g.A = x; g.lda = ldx; g.B = w; g.ldb = ldw;
    Epilogue& e = g.e;
    e.bias = bias; e.bias_f32 = flags & LSDM_OP_PARAM_F32 ? 1 : 0;
    e.res = residual; e.ldr = ldr;
    e.out = y; e.ldo = N;
    e.act = activation;
    if (activation != LSDM_ACT_NONE && deriv) { e.deriv = deriv; e.ldd = N; e.form = deriv_form(dtype, flags); }
    e.stream = whole_lines(y, N, es) && (!e.deriv || whole_lines(e.deriv, N, es));
    if (f.rows) {
        launch_rows(dtype, g, st);
        return launched("lsdm_linear");
    }
    const int64_t kp = up(K, 8);
    PrepArgs prep;
    int jobs = 0;
    if (f.xpad) { prep.job[jobs++] = padded(dtype, x, ldx, M, K, f.x, kp); g.A = f.x; g.lda = kp; }
    if (f.wpad) { prep.job[jobs++] = padded(dtype, w, ldw, N, K, f.w, kp); g.B = f.w; g.ldb = kp; }
    if (jobs) launch_prep(dtype, prep, jobs, st);
    g.part = f.part;
    launch_gemm(dtype, f.p, g, KK, st);
    return launched("lsdm_linear");
}

int lsdm_linear_backward(int device, int dtype, int flags, int64_t M, int64_t N, int64_t K, const void* dy, int64_t lddy, const void* deriv, const void* x,
                         int64_t ldx, const void* codes, const void* exps, const void* w, int64_t ldw, void* dx, void* dw, void* db, void* ws,
                         int64_t ws_bytes, void* stream) {
    if (const int rc = check_linear(dtype, M, N, K)) return rc;
    if (!dy || lddy < N) return refuse(LSDM_ERR_ARG, "lsdm_linear_backward: dy must not be NULL, its row stride not shorter than a row");
    if (dx && (!w || ldw < K)) return refuse(LSDM_ERR_ARG, "lsdm_linear_backward: dx needs w with a row stride of at least K");
    if (dw && !(codes ? exps != nullptr : x && ldx >= K)) return refuse(LSDM_ERR_ARG, "lsdm_linear_backward: dw needs x (row stride of at least K) or codes with exps");
    const int es = esize(dtype);
    const Bwd b = backward_layout(dtype, M, N, K, dx, dw, db, deriv, codes, rows16(dy, lddy, N, es), rows16(x, ldx, K, es), rows16(w, ldw, K, es), ws);
    if ((dx && !b.px.tile) || (dw && !b.pw.tile)) return refuse(LSDM_ERR_ARG, "lsdm_linear_backward: a gradient has more tiles than a launch can hold");
    if (b.bytes > 0 && (!ws || ws_bytes < b.bytes || !aligned16(ws)))
        return refuse(LSDM_ERR_ARG, "lsdm_linear_backward: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)ws_bytes, (long long)b.bytes);
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    hipStream_t st = static_cast<hipStream_t>(stream);
    // one launch prepares everything: dz = dy a'(z) with the column sums of its fp32 values, x from its 8-bit checkpoint, and rows that need padding.
    // dz is rounded to the operands' type: the matrix cores take both operands of a product in it, as an eager layer's backward pass does.  It puts a second
    // rounding beside the result's (bf16, 16384 x 2048 -> 8192 with gelu: dx and dw 2.35e-3 from 64 bits, 1.66e-3 if dz were kept in 32); dz as two bf16 terms
    // would take it out again and double both products, 900 us more in a pass of 1600.  Derivatives of 0 and 1 (relu, none) round nothing.
    PrepArgs prep;
    int jobs = 0;
    GemmArgs base;
    const void *z = dy, *xs = x, *ws_ = w;
    int64_t ldz = lddy, ldxs = ldx, ldws = ldw;
    if (b.dz || db) {
        PrepJob& j = prep.job[jobs++];
        j.src = dy; j.lds = lddy; j.deriv = deriv; j.form = deriv ? deriv_form(dtype, flags) : DERIV_NONE;
        j.rows = M; j.n = (int)N; j.chunks = b.chunks;
        if (b.dz) { j.dst = b.z; j.ldd = b.ldz; z = b.z; ldz = b.ldz; }
        j.part = b.cs;
    }
    if (b.xpad) {
        PrepJob& j = prep.job[jobs++];
        j = padded(dtype, codes ? codes : x, codes ? K : ldx, M, K, b.x, b.kp);
        if (codes) j.exps = static_cast<const unsigned char*>(exps);
        xs = b.x; ldxs = b.kp;
    }
    if (b.wpad) { prep.job[jobs++] = padded(dtype, w, ldw, N, K, b.w, b.kp); ws_ = b.w; ldws = b.kp; }
    if (jobs) launch_prep(dtype, prep, jobs, st);
    if (db) { base.cs_part = b.cs; base.cs_chunks = b.chunks; base.cs_n = (int)N; base.cs_out = db; base.cs_f32 = flags & LSDM_OP_PARAM_F32 ? 1 : 0; }
    if (!dx && !dw) {
        if (db) launch_colsum_join(dtype, base, st);
        return launched("lsdm_linear_backward");
    }
    if (dx) {
        GemmArgs g = base;                        // (the column sums are joined by the first product's launch)
        base = GemmArgs();
        g.M = (int)M; g.N = (int)K; g.K = (int)N;
        g.A = z; g.lda = ldz; g.B = ws_; g.ldb = ldws;
        g.part = b.partx;
        g.e.out = dx; g.e.ldo = K; g.e.stream = whole_lines(dx, K, es);
        launch_gemm(dtype, b.px, g, KM, st);
    }
    if (dw) {
        GemmArgs g = base;
        g.M = (int)N; g.N = (int)K; g.K = (int)M;
        g.A = z; g.lda = ldz; g.B = xs; g.ldb = ldxs;
        g.part = b.partw;
        g.e.out = dw; g.e.ldo = K; g.e.stream = whole_lines(dw, K, es);
        launch_gemm(dtype, b.pw, g, MM, st);
    }
    return launched("lsdm_linear_backward");
}

int64_t lsdm_layer_norm_workspace(int64_t rows, int64_t D) {
    if (rows < 1 || D < 1 || D > kNormMaxWidth) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm: rows >= 1 and a width in [1, %d] are needed", kNormMaxWidth);
    return (int64_t)norm_grid(rows, (int)D, true, 2) * 2 * D * 4;      // (16-bit calls have the larger grid)
}

static int check_norm(const char* who, int dtype, int64_t rows, int64_t D) {
    if (!dtype_ok(dtype)) return refuse(LSDM_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (rows < 1 || D < 1 || D > kNormMaxWidth) return refuse(LSDM_ERR_ARG, "%s: rows >= 1 and a width in [1, %d] are needed", who, kNormMaxWidth);
    return LSDM_OK;
}

int lsdm_layer_norm(int device, int dtype, int flags, int64_t rows, int64_t D, const void* x, int64_t ldx, const void* w, const void* b, float eps, void* y,
                    float* mean, float* rstd, void* codes, void* exps, void* stream) {
    if (const int rc = check_norm("lsdm_layer_norm", dtype, rows, D)) return rc;
    if (!x || !y || ldx < D) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm: x and y must not be NULL, the row stride not shorter than a row");
    if ((codes == nullptr) != (exps == nullptr)) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm: codes and exps come together");
    if (!(eps >= 0.0f)) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm: eps must be >= 0");
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    NormArgs a;
    a.rows = rows; a.D = (int)D; a.eps = eps; a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.param_f32 = flags & LSDM_OP_PARAM_F32 ? 1 : 0;
    a.y = y; a.mean = mean; a.rstd = rstd; a.codes = (signed char*)codes; a.exps = (unsigned char*)exps;
    launch_norm(dtype, a, norm_grid(rows, (int)D, false, esize(dtype)), false, static_cast<hipStream_t>(stream));
    return launched("lsdm_layer_norm");
}

int lsdm_layer_norm_backward(int device, int dtype, int flags, int64_t rows, int64_t D, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* codes,
                             const void* exps, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db, void* ws, int64_t ws_bytes,
                             void* stream) {
    if (const int rc = check_norm("lsdm_layer_norm_backward", dtype, rows, D)) return rc;
    if (!dy || lddy < D || !rstd) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm_backward: dy and rstd must not be NULL, the row stride not shorter than a row");
    if (!(codes ? exps != nullptr : x && mean && ldx >= D)) return refuse(LSDM_ERR_ARG, "lsdm_layer_norm_backward: x with mean, or codes with exps, are needed");
    const bool part = dw || db;
    const int64_t need = part ? lsdm_layer_norm_workspace(rows, D) : 0;
    if (part && (!ws || ws_bytes < need || !aligned16(ws)))
        return refuse(LSDM_ERR_ARG, "lsdm_layer_norm_backward: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)ws_bytes, (long long)need);
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    hipStream_t st = static_cast<hipStream_t>(stream);
    NormArgs a;
    a.rows = rows; a.D = (int)D; a.x = codes ? nullptr : x; a.ldx = ldx; a.w = w; a.param_f32 = flags & LSDM_OP_PARAM_F32 ? 1 : 0;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.codes = (signed char*)codes; a.exps = (unsigned char*)exps;
    a.dy = dy; a.lddy = lddy; a.dx = dx; a.part = part ? static_cast<float*>(ws) : nullptr;
    const int grid = norm_grid(rows, (int)D, true, esize(dtype));
    launch_norm(dtype, a, grid, true, st);
    if (part) launch_norm_join(dtype, a.part, grid, (int)D, dw, db, a.param_f32, st);
    return launched("lsdm_layer_norm_backward");
}

// two threads per group of 32 values
static bool pack8_sizes(int64_t rows, int64_t D) { return rows >= 1 && D >= 1 && D <= kMaxSize && rows <= kMaxThreads / ((D + 31) / 32 * 2); }

int lsdm_pack8(int device, int dtype, int64_t rows, int64_t D, const void* x, int64_t ldx, void* codes, void* exps, void* stream) {
    if (!dtype_ok(dtype) || !pack8_sizes(rows, D) || !x || !codes || !exps || ldx < D) return refuse(LSDM_ERR_ARG, "lsdm_pack8: bad argument");
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    Pack8Args a;
    a.rows = rows; a.D = (int)D; a.x = x; a.ldx = ldx; a.codes = (signed char*)codes; a.exps = (unsigned char*)exps;
    launch_pack8(dtype, a, static_cast<hipStream_t>(stream));
    return launched("lsdm_pack8");
}

int lsdm_unpack8(int device, int dtype, int64_t rows, int64_t D, const void* codes, const void* exps, void* out, void* stream) {
    if (!dtype_ok(dtype) || !pack8_sizes(rows, D) || !codes || !exps || !out) return refuse(LSDM_ERR_ARG, "lsdm_unpack8: bad argument");
    OnDevice dev(device);
    if (!dev.ok) return LSDM_ERR_HIP;
    Pack8Args a;
    a.rows = rows; a.D = (int)D; a.codes = (signed char*)codes; a.exps = (unsigned char*)exps; a.out = out;
    launch_unpack8(dtype, a, static_cast<hipStream_t>(stream));
    return launched("lsdm_unpack8");
}

}  // extern "C"
