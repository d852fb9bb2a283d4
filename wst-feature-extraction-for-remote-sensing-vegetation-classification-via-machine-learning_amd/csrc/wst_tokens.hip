// Layer norm and rotary positions on coefficient tokens (C ABI: include/wst_hip.h, "Token operators").
//
// Layer norm, for a row x of n values (a token's coefficients), mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps):
//   y  = (x - mu) r w + b
//   dx = r (g - mean(g) - h mean(g h)),  g = dy w,  h = (x - mu) r
//   dw = sum over rows of dy h,  db = sum over rows of dy
// Every variant computes mean, variance and all sums in float32 with the mean taken out before squaring, and rounds
// once when it stores. All are bound by memory: the forward pass reads x and writes y once.
//
// Rows lie in memory in one of two ways: "rows" (the n values adjacent) and "maps" (the points adjacent, as the
// scattering transform writes its maps: value k of point p at k * points + p).
#include <cmath>
#include <cstdarg>

#include "wst_tokens.h"

namespace wst_tok {

namespace {
thread_local char g_error[512] = "";
}

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? WST_OK : fail(WST_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace wst_tok

namespace {

using namespace wst_tok;

// ------------------------------------------------------------------------------------------ layer norm, rows
// Sums of NV values over the TPR threads of a row, to all of them. `slot` is LDS of (blockDim / 64) * NV floats.
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float* slot) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = wave_sum(v[i]);
    if constexpr (TPR > 64) {   // the row is the block
        const int w = threadIdx.x >> 6;
        __syncthreads();        // the slots' last readers are done
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) slot[w * NV + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < TPR / 64; ++k) s += slot[k * NV + i];
            v[i] = s;
        }
    }
}

struct NormArgs {
    int64_t rows, points;        // rows = batch * points
    int64_t n;
    int64_t sb, sp, sn;          // strides of x: batch, point, value
    int64_t db_, dp_, dn_;       // strides of dx
    int wdt;                     // type of w, b, dw, db
    float eps;
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *dbias;
    float *mean, *rstd;
    float *part;                 // (groups, 2, n) partial dw, db
    float *c;                    // (rows, 2): mean(g), mean(g h)
    int groups;
    int64_t first;               // this launch's first block (in_launches)
};

__device__ __forceinline__ int64_t row_at(const NormArgs& a, int64_t row, int64_t sb, int64_t sp) {
    if (a.points == a.rows) return row * sp;
    const int64_t b = row / a.points;
    return b * sb + (row - b * a.points) * sp;
}

template <int VEC, typename T, typename I>
__device__ __forceinline__ void load_part(const T* p, I col, I n, float (&v)[VEC]) {
    if (col + VEC <= n) {
        load<VEC>(p + col, v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = col + e < n ? static_cast<float>(p[col + e]) : 0.f;
    }
}
// the same, unconverted; WHOLE: n is a multiple of VEC
template <int VEC, bool WHOLE, typename T>
__device__ __forceinline__ Vec<T, VEC> load_raw(const T* p, int col, int n) {
    Vec<T, VEC> v{};
    if constexpr (WHOLE) {
        if (col < n) __builtin_memcpy(&v, p + col, sizeof(v));
    } else if (col + VEC <= n) {
        __builtin_memcpy(&v, p + col, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v.v[e] = col + e < n ? p[col + e] : static_cast<T>(0.f);
    }
    return v;
}
template <int VEC, typename T, typename I>
__device__ __forceinline__ void store_part(T* p, I col, I n, const float (&v)[VEC]) {
    if (col + VEC <= n) {
        store<VEC>(p + col, v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (col + e < n) p[col + e] = static_cast<T>(v[e]);
    }
}
template <int VEC, typename I>
__device__ __forceinline__ void load_w(const void* w, int wdt, float none, I col, I n, float (&v)[VEC]) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = none;
    } else if (col + VEC <= n) {
        load_as_n<VEC>(w, wdt, col, v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = col + e < n ? load_as(w, wdt, col + e) : 0.f;
    }
}

// One row per TPR threads, its values in registers (CH chunks of VEC a thread): x is read once. 32768 rows of 1024 in
// bfloat16: 30 us, 4.5 TB/s, of 4.9 that a large copy reaches.
template <typename Tx, typename Ty, int VEC, int CH, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_rows(NormArgs a) {
    __shared__ float slot[(TPR > 256 ? TPR : 256) / 64];
    const int t = threadIdx.x % TPR, n = static_cast<int>(a.n);
    const int64_t row = (a.first + blockIdx.x) * (blockDim.x / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;   // whole waves; with TPR > 64 the block is one row
    const Tx* x = static_cast<const Tx*>(a.x) + row_at(a, row, a.sb, a.sp);
    float v[CH][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_part<VEC>(x, (c * TPR + t) * VEC, n, v[c]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += v[c][e];
    }
    row_sum<TPR>(s, slot);
    const float count = static_cast<float>(n), mu = s[0] / count;   // divided: a constant row is its own mean
    s[0] = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = (c * TPR + t) * VEC + e < n ? v[c][e] - mu : 0.f;
            v[c][e] = d;
            s[0] += d * d;
        }
    row_sum<TPR>(s, slot);
    const float r = 1.f / sqrtf(s[0] / count + a.eps);
    Ty* y = static_cast<Ty*>(a.y) + row * a.n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + t) * VEC;
        if (col < n) {
            float w[VEC], b[VEC], o[VEC];
            load_w<VEC>(a.w, a.wdt, 1.f, col, n, w);
            load_w<VEC>(a.b, a.wdt, 0.f, col, n, b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = v[c][e] * r * w[e] + b[e];
            store_part<VEC>(y, col, n, o);
        }
    }
    if (t == 0 && a.mean) {
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
}

// Rows longer than the registers of a block: three sweeps, the second and third out of the caches.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(1024) void k_norm_long(NormArgs a) {
    __shared__ float slot[16];
    const int64_t row = a.first + blockIdx.x;
    const Tx* x = static_cast<const Tx*>(a.x) + row_at(a, row, a.sb, a.sp);
    float s[1] = {0.f};
    for (int64_t col = threadIdx.x * 4L; col < a.n; col += 4096) {
        float v[4];
        load_part<4>(x, col, a.n, v);
        s[0] += (v[0] + v[1]) + (v[2] + v[3]);
    }
    row_sum<1024>(s, slot);
    const float count = static_cast<float>(a.n), mu = s[0] / count;   // divided: a constant row's mean is itself
    s[0] = 0.f;
    for (int64_t col = threadIdx.x * 4L; col < a.n; col += 4096) {
        float v[4];
        load_part<4>(x, col, a.n, v);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < a.n) s[0] += (v[e] - mu) * (v[e] - mu);
    }
    row_sum<1024>(s, slot);
    const float r = 1.f / sqrtf(s[0] / count + a.eps);
    Ty* y = static_cast<Ty*>(a.y) + row * a.n;
    for (int64_t col = threadIdx.x * 4L; col < a.n; col += 4096) {
        float v[4], w[4], b[4];
        load_part<4>(x, col, a.n, v);
        load_w<4>(a.w, a.wdt, 1.f, col, a.n, w);
        load_w<4>(a.b, a.wdt, 0.f, col, a.n, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (v[e] - mu) * r * w[e] + b[e];
        store_part<4>(y, col, a.n, v);
    }
    if (threadIdx.x == 0 && a.mean) {
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
}

// Backward pass of rows: a block walks rows block, block + groups, ...; dx leaves at once, the thread's columns of dw
// and db stay in its registers until the block has added its waves' up and writes one partial row of each. The
// partials are added in a fixed order (k_norm_fold), so results repeat bit for bit. A wave has the next row's loads under
// way while it works on one; with a row in one piece of code for whole and for ragged chunks (not WHOLE) the compiler
// waits for them at once. 32768 rows of 1024 in bfloat16: 53 us, 3.8 TB/s (70 without the loads ahead).
template <typename Tx, typename Ty, int VEC, int CH, int TPR, bool WHOLE>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_bwd_rows(NormArgs a) {
    constexpr int kThreads = TPR > 256 ? TPR : 256, kRows = kThreads / TPR;
    __shared__ float slot[kThreads / 64 * 2];
    __shared__ float fold[kRows > 1 ? kRows * TPR * VEC : 1];
    const int n = static_cast<int>(a.n), t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float w[CH][VEC], dw[CH][VEC], db[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_w<VEC>(a.w, a.wdt, 1.f, (c * TPR + t) * VEC, n, w[c]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[c][e] = db[c][e] = 0.f;
    }
    const float count = static_cast<float>(n);
    // the next row is on its way, as it is in memory, while one is worked on
    Vec<Tx, VEC> xr[CH];
    Vec<Ty, VEC> gr[CH];
    float mu1 = 0.f, r1 = 0.f;
    auto fetch = [&](int64_t row) {
        const Tx* x = static_cast<const Tx*>(a.x) + row_at(a, row, a.sb, a.sp);
        const Ty* dy = static_cast<const Ty*>(a.dy) + row * a.n;
        mu1 = a.mean[row];
        r1 = a.rstd[row];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            xr[c] = load_raw<VEC, WHOLE>(x, (c * TPR + t) * VEC, n);
            gr[c] = load_raw<VEC, WHOLE>(dy, (c * TPR + t) * VEC, n);
        }
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub;
    if (row < a.rows) fetch(row);
    for (; row < a.rows; row += step) {
        const float mu = mu1, r = r1;
        float h[CH][VEC], g[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[c][e] = static_cast<float>(xr[c].v[e]);
                g[c][e] = static_cast<float>(gr[c].v[e]);
            }
        if (row + step < a.rows) fetch(row + step);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[c][e] = (c * TPR + t) * VEC + e < n ? (h[c][e] - mu) * r : 0.f;
                dw[c][e] += g[c][e] * h[c][e];
                db[c][e] += g[c][e];
                g[c][e] *= w[c][e];
                s[0] += g[c][e];
                s[1] += g[c][e] * h[c][e];
            }
        if (a.dx) {
            row_sum<TPR>(s, slot);
            const float c1 = s[0] / count, c2 = s[1] / count;
            Tx* dx = static_cast<Tx*>(a.dx) + row_at(a, row, a.db_, a.dp_);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * TPR + t) * VEC;
                if (col < n) {
                    float o[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o[e] = r * (g[c][e] - c1 - h[c][e] * c2);
                    store_part<VEC>(dx, col, n, o);
                }
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + t) * VEC;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = q ? db[c][e] : dw[c][e];
            if constexpr (kRows > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VEC; ++e) fold[(sub * TPR + t) * VEC + e] = o[e];
                __syncthreads();
                if (sub == 0)
#pragma unroll
                    for (int k = 1; k < kRows; ++k)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) o[e] += fold[(k * TPR + t) * VEC + e];
            }
            if (sub == 0 && col < n) store_part<VEC>(part + q * n, col, n, o);
        }
    }
}

// mean(g) and mean(g h) of rows longer than a block's registers.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(1024) void k_norm_bwd_long_sums(NormArgs a) {
    __shared__ float slot[32];
    const int64_t row = a.first + blockIdx.x;
    const Tx* x = static_cast<const Tx*>(a.x) + row_at(a, row, a.sb, a.sp);
    const Ty* dy = static_cast<const Ty*>(a.dy) + row * a.n;
    const float mu = a.mean[row], r = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int64_t col = threadIdx.x * 4L; col < a.n; col += 4096) {
        float h[4], g[4], w[4];
        load_part<4>(x, col, a.n, h);
        load_part<4>(dy, col, a.n, g);   // 0 beyond the row
        load_w<4>(a.w, a.wdt, 1.f, col, a.n, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            g[e] *= w[e];
            s[0] += g[e];
            s[1] += col + e < a.n ? g[e] * ((h[e] - mu) * r) : 0.f;
        }
    }
    row_sum<1024>(s, slot);
    if (threadIdx.x == 0) {
        a.c[2 * row] = s[0] / static_cast<float>(a.n);
        a.c[2 * row + 1] = s[1] / static_cast<float>(a.n);
    }
}

// dx and the partial dw, db of long rows: a thread keeps one column and walks the rows of its group.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(256) void k_norm_bwd_long_cols(NormArgs a) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (col >= a.n) return;
    const float w = a.w ? load_as(a.w, a.wdt, col) : 1.f;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float r = a.rstd[row];
        const float h = (static_cast<float>(static_cast<const Tx*>(a.x)[row_at(a, row, a.sb, a.sp) + col]) - a.mean[row]) * r;
        const float g = static_cast<float>(static_cast<const Ty*>(a.dy)[row * a.n + col]);
        dw += g * h;
        db += g;
        if (a.dx)
            static_cast<Tx*>(a.dx)[row_at(a, row, a.db_, a.dp_) + col] =
                static_cast<Tx>(r * (g * w - a.c[2 * row] - h * a.c[2 * row + 1]));
    }
    if (a.part) {
        float* part = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.n;
        part[col] = dw;
        part[a.n + col] = db;
    }
}

// Adds the groups' partial dw (blockIdx.y 0) and db (1): 32 columns a block, 32 threads a column, then over those.
__global__ __launch_bounds__(1024) void k_norm_fold(NormArgs a) {
    __shared__ float s[32][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
    const int64_t col = (a.first + blockIdx.x) * 32 + c;
    void* out = blockIdx.y ? a.dbias : a.dw;
    if (!out) return;
    float v = 0.f;
    if (col < a.n)
        for (int g = q; g < a.groups; g += 32) v += a.part[(static_cast<int64_t>(g) * 2 + blockIdx.y) * a.n + col];
    s[q][c] = v;
    __syncthreads();
    if (q == 0 && col < a.n) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += s[k][c];
        store_as(out, a.wdt, col, v);
    }
}

// ------------------------------------------------------------------------------------------ layer norm, maps
constexpr int kMapThreads = 512, kMapBig = 1024;
constexpr int kMapPts = 32;      // points of a block at most

// Copies columns [k0, k0 + nk) of the points [p0, p0 + np) of one batch entry into LDS, turned: tile[p][k], row
// stride ld. Global memory is read along the points (four at a time), LDS written so that the lanes of a wave, tp / 4
// fours of points by 256 / tp consecutive columns, fall on different banks: ld = 64 / tp modulo 16 (map_ld).
template <typename Tx>
__device__ __forceinline__ void load_tile(const Tx* x, int64_t sn, int tp, int np, int64_t k0, int nk, float* tile, int ld) {
    const int quads = tp >> 2;                      // 4 or 8: tp is 16 or kMapPts
    const int q = (threadIdx.x & (quads - 1)) * 4, step = blockDim.x / quads;
    for (int k = threadIdx.x / quads; k < nk; k += step) {
        const Tx* s = x + (k0 + k) * sn + q;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (q + 4 <= np) {
            load<4>(s, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (q + e < np) v[e] = static_cast<float>(s[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[(q + e) * ld + k] = v[e];
    }
}

// Values that a lane of a row in LDS stores at once: two of 16 bits or one of 32, so that reading LDS without bank
// conflicts and writing memory in whole lines go together whatever ld is.
template <typename Ty>
constexpr int kPack = sizeof(Ty) == 2 ? 2 : 1;

// A block takes tp points of one batch entry with all n values into LDS, then a wave takes its points' mean and variance
// out of LDS, and at last writes their rows whole, some columns at a time, with the weights of those columns in
// registers: one read of x. For n * 16 values that fit the LDS. PLAIN: weight and bias are there, in float32 (a branch on
// their type at every value took as many instructions as all else: 128 us then).
// 160 x 1024 points of 243 in float32: 77 us, 4.1 TB/s. 1024 x 16 points of 1251, bfloat16 out: 39 us, 3.1 TB/s: there a
// block's 80 KB of LDS leave room for two blocks a CU, which wait together for memory at their start.
template <typename Tx, typename Ty, bool PLAIN>
__global__ __launch_bounds__(kMapBig) void k_norm_maps(NormArgs a, int tp, int ld) {
    extern __shared__ float tile[];
    __shared__ float stat[2][kMapPts];
    const int64_t tiles = (a.points + tp - 1) / tp;
    const int64_t id = a.first + blockIdx.x, b = id / tiles, p0 = (id - b * tiles) * tp;
    const int np = static_cast<int>(a.points - p0 < tp ? a.points - p0 : tp), n = static_cast<int>(a.n);
    load_tile(static_cast<const Tx*>(a.x) + b * a.sb + p0, a.sn, tp, np, 0, n, tile, ld);
    __syncthreads();
    const int lane = threadIdx.x & 63, w0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const float count = static_cast<float>(n);
    const int64_t row0 = b * a.points + p0;
    for (int p = w0; p < np; p += waves) {
        const float* v = tile + p * ld + lane;
        float s = 0.f;
        int k = 0;
        for (; k + 512 <= n; k += 512)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[k + 64 * e];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + 64 * e + lane < n) s += v[k + 64 * e];
        const float mu = wave_sum(s) / count;
        s = 0.f;
        k = 0;
        for (; k + 512 <= n; k += 512)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = v[k + 64 * e] - mu;
                s = fmaf(d, d, s);
            }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + 64 * e + lane < n) {
                const float d = v[k + 64 * e] - mu;
                s = fmaf(d, d, s);
            }
        const float r = 1.f / sqrtf(wave_sum(s) / count + a.eps);
        if (lane == 0) {
            stat[0][p] = mu;
            stat[1][p] = r;
            if (a.mean) {
                a.mean[row0 + p] = mu;
                a.rstd[row0 + p] = r;
            }
        }
    }
    // a wave writes the rows whose statistics it took, so no barrier of the block
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int N = kPack<Ty>, C = 4;      // C chunks of 64 N columns at a time
    for (int k0 = lane * N; k0 < n; k0 += 64 * N * C) {
        float w[C][N], c[C][N];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int k = k0 + 64 * N * i;
            if constexpr (PLAIN) {
                load_part<N>(static_cast<const float*>(a.w), k, n, w[i]);
                load_part<N>(static_cast<const float*>(a.b), k, n, c[i]);
            } else {
                load_w<N>(a.w, a.wdt, 1.f, k, n, w[i]);
                load_w<N>(a.b, a.wdt, 0.f, k, n, c[i]);
            }
        }
        for (int p = w0; p < np; p += waves) {
            const float* v = tile + p * ld + k0;
            const float mu = stat[0][p], r = stat[1][p];
            Ty* y = static_cast<Ty*>(a.y) + (row0 + p) * a.n + k0;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                if (k0 + 64 * N * i >= n) break;
                float o[N];
#pragma unroll
                for (int e = 0; e < N; ++e) o[e] = (v[64 * N * i + e] - mu) * r * w[i][e] + c[i][e];
                store_part<N>(y + 64 * N * i, 0, n - k0 - 64 * N * i, o);
            }
        }
    }
}

constexpr int kPts = 16, kCols = 256, kLd = 260;   // tile of the sweeps over longer maps: 260 = 4 modulo 16

// Maps whose n * 16 values exceed the LDS (four bands, J=6, L=12: 8932): mean, variance and output in three sweeps over tiles of 256
// columns of 16 points, the later ones out of the caches.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(kMapThreads) void k_norm_maps_long(NormArgs a) {
    __shared__ float tile[kPts * kLd];
    const int64_t tiles = (a.points + kPts - 1) / kPts;
    const int64_t id = a.first + blockIdx.x, b = id / tiles, p0 = (id - b * tiles) * kPts;
    const int np = static_cast<int>(a.points - p0 < kPts ? a.points - p0 : kPts);
    const Tx* x = static_cast<const Tx*>(a.x) + b * a.sb + p0;
    const int lane = threadIdx.x & 63, w0 = threadIdx.x >> 6;   // a wave's points: w0 and w0 + 8
    const float count = static_cast<float>(a.n);
    float mu[2] = {0.f, 0.f}, s[2] = {0.f, 0.f}, r[2] = {0.f, 0.f};
    for (int sweep = 0; sweep < 3; ++sweep) {
        for (int64_t k0 = 0; k0 < a.n; k0 += kCols) {
            const int nk = static_cast<int>(a.n - k0 < kCols ? a.n - k0 : kCols);
            __syncthreads();
            load_tile(x, a.sn, kPts, np, k0, nk, tile, kLd);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = w0 + 8 * i;
                const float* v = tile + p * kLd;
                if (sweep < 2) {
                    for (int k = lane; k < nk; k += 64) s[i] += sweep ? (v[k] - mu[i]) * (v[k] - mu[i]) : v[k];
                } else if (p < np && lane * 4 < nk) {
                    float w[4], c[4], o[4];
                    load_w<4>(a.w, a.wdt, 1.f, k0 + lane * 4, a.n, w);
                    load_w<4>(a.b, a.wdt, 0.f, k0 + lane * 4, a.n, c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = (v[lane * 4 + e] - mu[i]) * r[i] * w[e] + c[e];
                    store_part<4>(static_cast<Ty*>(a.y) + (b * a.points + p0 + p) * a.n, k0 + lane * 4, a.n, o);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float t = wave_sum(s[i]) / count;
            if (sweep == 0) mu[i] = t;
            if (sweep == 1) r[i] = 1.f / sqrtf(t + a.eps);
            s[i] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t row = b * a.points + p0 + w0 + 8 * i;
        if (lane == 0 && w0 + 8 * i < np && a.mean) {
            a.mean[row] = mu[i];
            a.rstd[row] = r[i];
        }
    }
}

// mean(g) and mean(g h) of 16 points of a map, for the gradient of x.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(kMapThreads) void k_norm_bwd_maps_sums(NormArgs a) {
    __shared__ float tile[kPts * kLd];
    const int64_t tiles = (a.points + kPts - 1) / kPts;
    const int64_t id = a.first + blockIdx.x, b = id / tiles, p0 = (id - b * tiles) * kPts;
    const int np = static_cast<int>(a.points - p0 < kPts ? a.points - p0 : kPts);
    const Tx* x = static_cast<const Tx*>(a.x) + b * a.sb + p0;
    const int lane = threadIdx.x & 63, w0 = threadIdx.x >> 6;
    float s0[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f};
    for (int64_t k0 = 0; k0 < a.n; k0 += kCols) {
        const int nk = static_cast<int>(a.n - k0 < kCols ? a.n - k0 : kCols);
        __syncthreads();
        load_tile(x, a.sn, kPts, np, k0, nk, tile, kLd);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int p = w0 + 8 * i;
            if (p < np) {
                const int64_t row = b * a.points + p0 + p;
                const float mu = a.mean[row], r = a.rstd[row];
                const Ty* dy = static_cast<const Ty*>(a.dy) + row * a.n + k0;
                for (int k = lane; k < nk; k += 64) {
                    const float g = static_cast<float>(dy[k]) * (a.w ? load_as(a.w, a.wdt, k0 + k) : 1.f);
                    s0[i] += g;
                    s1[i] += g * ((tile[p * kLd + k] - mu) * r);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float t0 = wave_sum(s0[i]), t1 = wave_sum(s1[i]);
        if (lane == 0 && w0 + 8 * i < np) {
            const int64_t row = b * a.points + p0 + w0 + 8 * i;
            a.c[2 * row] = t0 / static_cast<float>(a.n);
            a.c[2 * row + 1] = t1 / static_cast<float>(a.n);
        }
    }
}

constexpr int kBCols = 512, kBLd = 516;      // 516 = 4 modulo 16

// dx and the partial dw, db of maps: a block keeps 512 columns and walks tiles of 16 points, a thread two columns and
// half of the points; the next tile of x and dy is on its way while one is worked on. No sums over n are needed here, so
// any n goes through the same tile. 1024 x 16 points of 1251, dy bfloat16, weight and bias alone: 40 us, 3.1 TB/s.
template <typename Tx, typename Ty>
__global__ __launch_bounds__(kMapThreads) void k_norm_bwd_maps(NormArgs a) {
    __shared__ float tile[kPts * kBLd];
    __shared__ float fold[2][kBCols];
    const int64_t k0 = static_cast<int64_t>(blockIdx.x) * kBCols;
    const int nk = static_cast<int>(a.n - k0 < kBCols ? a.n - k0 : kBCols);
    const int k = (threadIdx.x & 255) * 2, half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int64_t tiles = (a.points + kPts - 1) / kPts, all = a.rows / a.points * tiles;
    const bool mine = k < nk, pair = k + 1 < nk;
    const float w[2] = {a.w && mine ? load_as(a.w, a.wdt, k0 + k) : 1.f, a.w && pair ? load_as(a.w, a.wdt, k0 + k + 1) : 1.f};
    float dw[2] = {0.f, 0.f}, db[2] = {0.f, 0.f};
    // loading: a thread's four points q .. q + 3 of columns kq, kq + 128, ...
    const int q = (threadIdx.x & 3) * 4, kq = threadIdx.x >> 2;
    float xv[4][4];
    Vec<Ty, 2> gv[kPts / 2];
    auto fetch = [&](int64_t t) {
        const int64_t b = t / tiles, p0 = (t - b * tiles) * kPts;
        const int np = static_cast<int>(a.points - p0 < kPts ? a.points - p0 : kPts);
        const Tx* x = static_cast<const Tx*>(a.x) + b * a.sb + p0 + q + (k0 + kq) * a.sn;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (q + 4 <= np && kq + 128 * i < nk) {
                load<4>(x + 128 * i * a.sn, xv[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) xv[i][e] = q + e < np && kq + 128 * i < nk ? static_cast<float>(x[128 * i * a.sn + e]) : 0.f;
            }
        }
        const Ty* dy = static_cast<const Ty*>(a.dy) + (b * a.points + p0) * a.n + k0 + k;
#pragma unroll
        for (int i = 0; i < kPts / 2; ++i) {
            const int p = half * (kPts / 2) + i;
            if (p < np && pair) __builtin_memcpy(&gv[i], dy + p * a.n, sizeof(gv[i]));
            else gv[i] = Vec<Ty, 2>{{p < np && mine ? dy[p * a.n] : static_cast<Ty>(0.f), static_cast<Ty>(0.f)}};
        }
    };
    int64_t t = blockIdx.y;
    if (t < all) fetch(t);
    for (; t < all; t += gridDim.y) {
        const int64_t b = t / tiles, p0 = (t - b * tiles) * kPts;
        const int np = static_cast<int>(a.points - p0 < kPts ? a.points - p0 : kPts);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) tile[(q + e) * kBLd + kq + 128 * i] = xv[i][e];
        Vec<Ty, 2> now[kPts / 2];
#pragma unroll
        for (int i = 0; i < kPts / 2; ++i) now[i] = gv[i];
        __syncthreads();
        if (t + gridDim.y < all) fetch(t + gridDim.y);
        const int64_t row0 = b * a.points + p0;
#pragma unroll
        for (int i = 0; i < kPts / 2; ++i) {
            const int p = half * (kPts / 2) + i;
            if (p < np) {          // uniform
                const float r = a.rstd[row0 + p], mu = a.mean[row0 + p];
                float* v = tile + p * kBLd + k;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float h = (v[e] - mu) * r, g = static_cast<float>(now[i].v[e]);
                    dw[e] = fmaf(g, h, dw[e]);
                    db[e] += g;
                    if (a.dx) v[e] = r * (g * w[e] - a.c[2 * (row0 + p)] - h * a.c[2 * (row0 + p) + 1]);
                }
            }
        }
        if (a.dx) {
            __syncthreads();
            Tx* dx = static_cast<Tx*>(a.dx) + b * a.db_ + p0 * a.dp_;
            for (int i = threadIdx.x; i < kPts * nk; i += kMapThreads) {
                const int p = i & (kPts - 1), kk = i / kPts;
                if (p < np) dx[(k0 + kk) * a.dn_ + p * a.dp_] = static_cast<Tx>(tile[p * kBLd + kk]);
            }
        }
    }
    if (!a.part) return;
    if (half && mine) {
        fold[0][k] = dw[0];
        fold[1][k] = db[0];
        fold[0][k + 1] = dw[1];
        fold[1][k + 1] = db[1];
    }
    __syncthreads();
    if (!half && mine) {
        float* part = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.n + k0 + k;
        part[0] = dw[0] + fold[0][k];
        part[a.n] = db[0] + fold[1][k];
        if (pair) {
            part[1] = dw[1] + fold[0][k + 1];
            part[a.n + 1] = db[1] + fold[1][k + 1];
        }
    }
}

// ------------------------------------------------------------------------------------------ layer norm, host
template <typename T>
struct Tag {
    using type = T;
};
template <typename F>
int with_type(int dtype, F f) {
    if (dtype == WST_F32) return f(Tag<float>{});
    if (dtype == WST_BF16) return f(Tag<bf16>{});
    return f(Tag<f16>{});
}

bool type_ok(int t) { return t == WST_F32 || t == WST_BF16 || t == WST_F16; }

// Whether the values lie as maps: the points adjacent, the values of a point apart.
bool as_maps(const wst_norm_desc& d) { return d.x_stride_n != 1 && d.n > 1; }

int norm_check(const wst_norm_desc* d) {
    if (!d) return fail(WST_ERR_INVALID, "layer norm: descriptor is NULL");
    if (d->batch < 0 || d->points < 0 || d->n < 1) return fail(WST_ERR_INVALID, "layer norm: bad sizes (%lld, %lld, %lld)",
        static_cast<long long>(d->batch), static_cast<long long>(d->points), static_cast<long long>(d->n));
    if (!type_ok(d->x_dtype) || !type_ok(d->y_dtype) || !type_ok(d->w_dtype)) return fail(WST_ERR_INVALID, "layer norm: unknown type");
    if (!(d->eps >= 0.f)) return fail(WST_ERR_INVALID, "layer norm: eps must not be negative");
    if (as_maps(*d) && d->x_stride_point != 1 && d->points > 1)
        return fail(WST_ERR_INVALID, "layer norm: either the values or the points of x must be adjacent");
    const double rows = static_cast<double>(d->batch) * static_cast<double>(d->points);
    if (rows > 2147483647.0 || d->n > 2147483647LL) return fail(WST_ERR_UNSUPPORTED, "layer norm: more than 2^31 - 1 rows or values");
    return WST_OK;
}

NormArgs norm_args(const wst_norm_desc& d) {
    NormArgs a{};
    a.rows = d.batch * d.points;
    a.points = d.points;
    a.n = d.n;
    a.sb = d.x_stride_batch; a.sp = d.x_stride_point; a.sn = d.x_stride_n;
    a.db_ = d.dx_stride_batch; a.dp_ = d.dx_stride_point; a.dn_ = d.dx_stride_n;
    a.wdt = d.w_dtype;
    a.eps = d.eps;
    if (d.batch == 1) a.sb = a.db_ = 0;
    return a;
}

constexpr int kGroups = 512;                // partial rows of dw and db at most
constexpr int64_t kRegRows = 8192;          // longest rows whose backward pass keeps them in registers

// Partial rows that the backward pass makes, for its variant.
int norm_groups(const wst_norm_desc& d) {
    const int64_t rows = d.batch * d.points;
    if (as_maps(d)) {
        const int64_t tiles = d.batch * ((d.points + kPts - 1) / kPts), cols = (d.n + kBCols - 1) / kBCols;
        int64_t g = (1024 + cols - 1) / cols;                    // about four blocks a CU
        if (g > kGroups) g = kGroups;
        return static_cast<int>(g < tiles ? g : tiles);
    }
    if (d.n > kRegRows) return static_cast<int>(rows < 64 ? rows : 64);
    const int64_t blocks = d.n <= 1024 ? (rows + 3) / 4 : rows;  // four rows a block up to 1024 values
    return static_cast<int>(blocks < kGroups ? blocks : kGroups);
}

size_t norm_bytes(const wst_norm_desc& d) {
    const size_t rows = static_cast<size_t>(d.batch) * d.points;
    return (static_cast<size_t>(norm_groups(d)) * 2 * d.n + 2 * rows) * sizeof(float);
}

// A launch that asks for 2^32 threads or more is cut to what is left of them, without an error: calls with more blocks go in
// several launches.
template <typename F>
void in_launches(NormArgs a, int64_t blocks, int threads, F launch) {
    const int64_t most = (1LL << 31) / threads;
    for (; a.first < blocks; a.first += most)
        launch(a, static_cast<unsigned>(blocks - a.first < most ? blocks - a.first : most));
}

template <typename Tx, typename Ty>
void norm_rows(const NormArgs& args, hipStream_t st) {
    // one wave a row up to 2048 values, a block of 256 or 1024 threads up to 32768, three sweeps beyond
    const int chunks = static_cast<int>((args.n + 255) / 256);
    if (chunks <= 8) {
        const int per = args.rows >= 2048 ? 4 : 1;    // few rows: one to a block, so that they spread over the CUs
        in_launches(args, (args.rows + per - 1) / per, 64 * per, [&](const NormArgs& a, unsigned blocks) {
            const dim3 g(blocks), t(64 * per);
            if (chunks <= 1) k_norm_rows<Tx, Ty, 4, 1, 64><<<g, t, 0, st>>>(a);
            else if (chunks <= 2) k_norm_rows<Tx, Ty, 4, 2, 64><<<g, t, 0, st>>>(a);
            else if (chunks <= 4) k_norm_rows<Tx, Ty, 4, 4, 64><<<g, t, 0, st>>>(a);
            else k_norm_rows<Tx, Ty, 4, 8, 64><<<g, t, 0, st>>>(a);
        });
    } else if (args.n <= 8192) {
        in_launches(args, args.rows, 256, [&](const NormArgs& a, unsigned blocks) {
            k_norm_rows<Tx, Ty, 4, 8, 256><<<dim3(blocks), dim3(256), 0, st>>>(a);
        });
    } else {
        in_launches(args, args.rows, 1024, [&](const NormArgs& a, unsigned blocks) {
            if (a.n <= 32768) k_norm_rows<Tx, Ty, 4, 8, 1024><<<dim3(blocks), dim3(1024), 0, st>>>(a);
            else k_norm_long<Tx, Ty><<<dim3(blocks), dim3(1024), 0, st>>>(a);
        });
    }
}

constexpr int kLdsMax = 160 * 1024;

template <typename Tx, typename Ty>
int norm_maps(const NormArgs& args, hipStream_t st) {
    const int64_t batch = args.rows / args.points;
    // Points a block takes: 32 make whole lines of 128 bytes; fewer when there are no more, or when the block's share of
    // the LDS would leave less than two to a CU.
    // ld: n + 1 or more (a pair may end behind the last column), 64 / tp modulo 16
    auto map_ld = [&](int64_t tp) { return (args.n + 1 + 15 - 64 / tp) / 16 * 16 + 64 / tp; };
    int tp = kMapPts;
    while (tp > 16 && (tp / 2 >= args.points || tp * map_ld(tp) * 4 > kLdsMax / 2 - 512)) tp >>= 1;
    const int64_t ld = map_ld(tp), bytes = tp * ld * 4, tiles = (args.points + tp - 1) / tp;
    const int threads = bytes > kLdsMax / 4 ? kMapBig : kMapThreads;      // two blocks of sixteen waves, or four of eight
    if (bytes <= kLdsMax - 1024) {
        const bool plain = args.w && args.b && args.wdt == WST_F32;
        const void* kernel = plain ? reinterpret_cast<const void*>(&k_norm_maps<Tx, Ty, true>) : reinterpret_cast<const void*>(&k_norm_maps<Tx, Ty, false>);
        if (bytes > 64 * 1024 && hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMax - 1024) != hipSuccess)
            return launched("layer norm");
        in_launches(args, batch * tiles, threads, [&](const NormArgs& a, unsigned blocks) {
            if (plain) k_norm_maps<Tx, Ty, true><<<dim3(blocks), dim3(threads), bytes, st>>>(a, tp, static_cast<int>(ld));
            else k_norm_maps<Tx, Ty, false><<<dim3(blocks), dim3(threads), bytes, st>>>(a, tp, static_cast<int>(ld));
        });
    } else {
        in_launches(args, batch * ((args.points + kPts - 1) / kPts), kMapThreads, [&](const NormArgs& a, unsigned blocks) {
            k_norm_maps_long<Tx, Ty><<<dim3(blocks), dim3(kMapThreads), 0, st>>>(a);
        });
    }
    return WST_OK;
}

template <typename Tx, typename Ty, bool WHOLE>
void norm_bwd_regs(const NormArgs& a, hipStream_t st) {
    const int chunks = static_cast<int>((a.n + 255) / 256);
    const dim3 g(static_cast<unsigned>(a.groups));
    if (chunks <= 1) k_norm_bwd_rows<Tx, Ty, 4, 1, 64, WHOLE><<<g, dim3(256), 0, st>>>(a);
    else if (chunks <= 2) k_norm_bwd_rows<Tx, Ty, 4, 2, 64, WHOLE><<<g, dim3(256), 0, st>>>(a);
    else if (chunks <= 4) k_norm_bwd_rows<Tx, Ty, 4, 4, 64, WHOLE><<<g, dim3(256), 0, st>>>(a);
    else if (chunks <= 8) k_norm_bwd_rows<Tx, Ty, 4, 1, 512, WHOLE><<<g, dim3(512), 0, st>>>(a);
    else if (chunks <= 16) k_norm_bwd_rows<Tx, Ty, 4, 2, 512, WHOLE><<<g, dim3(512), 0, st>>>(a);
    else k_norm_bwd_rows<Tx, Ty, 4, 4, 512, WHOLE><<<g, dim3(512), 0, st>>>(a);
}

template <typename Tx, typename Ty>
void norm_bwd_rows(const NormArgs& a, hipStream_t st) {
    if (a.n <= kRegRows) {
        if (a.n % 4 == 0) norm_bwd_regs<Tx, Ty, true>(a, st);
        else norm_bwd_regs<Tx, Ty, false>(a, st);
    } else {
        if (a.dx)
            in_launches(a, a.rows, 1024, [&](const NormArgs& x, unsigned blocks) {
                k_norm_bwd_long_sums<Tx, Ty><<<dim3(blocks), dim3(1024), 0, st>>>(x);
            });
        k_norm_bwd_long_cols<Tx, Ty><<<dim3(static_cast<unsigned>((a.n + 255) / 256), a.groups), dim3(256), 0, st>>>(a);
    }
}

template <typename Tx, typename Ty>
void norm_bwd_maps(const NormArgs& a, hipStream_t st) {
    const int64_t tiles = a.rows / a.points * ((a.points + kPts - 1) / kPts);
    if (a.dx)
        in_launches(a, tiles, kMapThreads, [&](const NormArgs& x, unsigned blocks) {
            k_norm_bwd_maps_sums<Tx, Ty><<<dim3(blocks), dim3(kMapThreads), 0, st>>>(x);
        });
    k_norm_bwd_maps<Tx, Ty><<<dim3(static_cast<unsigned>((a.n + kBCols - 1) / kBCols), a.groups), dim3(kMapThreads), 0, st>>>(a);
}

// ------------------------------------------------------------------------------------------ rotary
// Pair p belongs to one axis; its angle is position * base^(-i / pairs of the axis). A turn is held as a fraction of
// a revolution: position * (frequency / 2 pi) in 64 bits less its whole part, so far positions lose nothing; the
// sine and cosine of what is left are taken in 32 bits. The angle depends on token and pair alone, so a thread
// computes it once and applies it to all its heads.
constexpr int kMaxPairs = WST_MAX_PAIRS;

struct RotaryTable {
    double rev[kMaxPairs];        // revolutions a step of position
    unsigned char axis[kMaxPairs];
};

struct RotaryArgs {
    const void* x[2];
    void* y[2];
    int64_t xs[2][3], ys[2][3];   // strides: batch, token, head
    int heads[2];
    int64_t tokens, rows;         // rows = batch * tokens
    const int32_t* pos;
    int64_t pos_sb;               // elements a batch entry of positions takes; 0 when shared
    int axes, pairs, dim, split;  // split: blocks that share a row's heads
    float sign;
};

constexpr int kRotPairs = 4;      // pairs a thread turns

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a, RotaryTable tab) {
    const int turned = (a.pairs + kRotPairs - 1) / kRotPairs;                       // units that turn pairs
    const int units = turned + (a.dim - 2 * a.pairs + 7) / 8;                       // and units that copy the rest
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = id / units;
    if (row >= a.rows) return;
    const int u = static_cast<int>(id - row * units);
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const int total = a.heads[0] + a.heads[1];
    float c[kRotPairs], s[kRotPairs];
    const int p0 = u * kRotPairs;
    if (u < turned) {
        const int32_t* pos = a.pos + b * a.pos_sb + t * a.axes;
#pragma unroll
        for (int i = 0; i < kRotPairs; ++i) {
            const int p = p0 + i < a.pairs ? p0 + i : a.pairs - 1;
            const double turn = static_cast<double>(pos[tab.axis[p]]) * tab.rev[p];
            sincospif(2.f * static_cast<float>(turn - rint(turn)), &s[i], &c[i]);
            s[i] *= a.sign;
        }
    }
    for (int h = blockIdx.y; h < total; h += a.split) {
        const int which = h >= a.heads[0];
        const int hh = which ? h - a.heads[0] : h;
        const T* x = static_cast<const T*>(a.x[which]) + b * a.xs[which][0] + t * a.xs[which][1] + hh * a.xs[which][2];
        T* y = static_cast<T*>(a.y[which]) + b * a.ys[which][0] + t * a.ys[which][1] + hh * a.ys[which][2];
        if (u >= turned) {
            const int d0 = 2 * a.pairs + (u - turned) * 8;
            if (d0 + 8 <= a.dim) {
                Vec<T, 8> v;
                __builtin_memcpy(&v, x + d0, sizeof(v));
                __builtin_memcpy(y + d0, &v, sizeof(v));
            } else {
                for (int d = d0; d < a.dim; ++d) y[d] = x[d];
            }
        } else if (p0 + kRotPairs <= a.pairs) {
            float x0[kRotPairs], x1[kRotPairs];
            if constexpr (INTER) {
                float v[2 * kRotPairs];
                load<2 * kRotPairs>(x + 2 * p0, v);
#pragma unroll
                for (int i = 0; i < kRotPairs; ++i) {
                    x0[i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
                    x1[i] = v[2 * i + 1] * c[i] + v[2 * i] * s[i];
                }
#pragma unroll
                for (int i = 0; i < kRotPairs; ++i) {
                    v[2 * i] = x0[i];
                    v[2 * i + 1] = x1[i];
                }
                store<2 * kRotPairs>(y + 2 * p0, v);
            } else {
                float y0[kRotPairs], y1[kRotPairs];
                load<kRotPairs>(x + p0, x0);
                load<kRotPairs>(x + a.pairs + p0, x1);
#pragma unroll
                for (int i = 0; i < kRotPairs; ++i) {
                    y0[i] = x0[i] * c[i] - x1[i] * s[i];
                    y1[i] = x1[i] * c[i] + x0[i] * s[i];
                }
                store<kRotPairs>(y + p0, y0);
                store<kRotPairs>(y + a.pairs + p0, y1);
            }
        } else {
            for (int i = 0; p0 + i < a.pairs; ++i) {
                const int p = p0 + i, i0 = INTER ? 2 * p : p, i1 = INTER ? 2 * p + 1 : p + a.pairs;
                // the loop's bound is below kRotPairs: c and s stay in registers through the selects
                const float cc = i == 0 ? c[0] : i == 1 ? c[1] : c[2], ss = i == 0 ? s[0] : i == 1 ? s[1] : s[2];
                const float x0 = static_cast<float>(x[i0]), x1 = static_cast<float>(x[i1]);
                y[i0] = static_cast<T>(x0 * cc - x1 * ss);
                y[i1] = static_cast<T>(x1 * cc + x0 * ss);
            }
        }
    }
}

}  // namespace

extern "C" {

const char* wst_tokens_last_error(void) { return wst_tok::g_error; }

int wst_layer_norm_forward(const wst_norm_desc* d, const void* x, const void* weight, const void* bias, void* y,
                           float* mean, float* rstd, void* stream) {
    if (const int e = norm_check(d)) return e;
    if (d->batch == 0 || d->points == 0) return WST_OK;
    if (!x || !y) return fail(WST_ERR_INVALID, "layer norm: input or output pointer is NULL");
    if (!mean != !rstd) return fail(WST_ERR_INVALID, "layer norm: mean and rstd go together");
    NormArgs a = norm_args(*d);
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int e = with_type(d->x_dtype, [&](auto tx) {
        return with_type(d->y_dtype, [&](auto ty) {
            using Tx = typename decltype(tx)::type;
            using Ty = typename decltype(ty)::type;
            if (as_maps(*d)) return norm_maps<Tx, Ty>(a, st);
            norm_rows<Tx, Ty>(a, st);
            return static_cast<int>(WST_OK);
        });
    });
    return e ? e : launched("layer norm");
}

int wst_layer_norm_workspace(const wst_norm_desc* d, size_t* bytes) {
    if (!bytes) return fail(WST_ERR_INVALID, "layer norm: bytes is NULL");
    if (const int e = norm_check(d)) return e;
    *bytes = d->batch && d->points ? norm_bytes(*d) : 0;
    return WST_OK;
}

int wst_layer_norm_backward(const wst_norm_desc* d, const void* x, const void* weight, const void* dy, const float* mean,
                            const float* rstd, void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                            void* stream) {
    if (const int e = norm_check(d)) return e;
    if (d->batch == 0 || d->points == 0) return fail(WST_ERR_INVALID, "layer norm: no rows, the weight's gradient is zero");
    if (!x || !dy || !mean || !rstd) return fail(WST_ERR_INVALID, "layer norm: an input pointer is NULL");
    if (dx && (as_maps(*d) ? d->dx_stride_point != 1 && d->points > 1 : d->dx_stride_n != 1 && d->n > 1))
        return fail(WST_ERR_INVALID, "layer norm: dx must lie as x does");
    if (!workspace || workspace_bytes < norm_bytes(*d)) return fail(WST_ERR_INVALID, "layer norm: workspace too small");
    if (!dx && !dweight && !dbias) return WST_OK;
    NormArgs a = norm_args(*d);
    a.x = x; a.w = weight; a.dy = dy; a.dx = dx; a.dw = dweight; a.dbias = dbias;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.groups = norm_groups(*d);
    a.part = dweight || dbias ? static_cast<float*>(workspace) : nullptr;
    a.c = static_cast<float*>(workspace) + static_cast<size_t>(a.groups) * 2 * d->n;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->x_dtype, [&](auto tx) {
        return with_type(d->y_dtype, [&](auto ty) {
            using Tx = typename decltype(tx)::type;
            using Ty = typename decltype(ty)::type;
            if (as_maps(*d)) norm_bwd_maps<Tx, Ty>(a, st);
            else norm_bwd_rows<Tx, Ty>(a, st);
            return 0;
        });
    });
    if (a.part)
        in_launches(a, (d->n + 31) / 32, 1024, [&](const NormArgs& x, unsigned blocks) {
            k_norm_fold<<<dim3(blocks, 2), dim3(1024), 0, st>>>(x);
        });
    return launched("layer norm backward");
}

int wst_rotary(const wst_rotary_desc* d, const void* q, void* q_out, const void* k, void* k_out, const int32_t* positions,
               void* stream) {
    if (!d) return fail(WST_ERR_INVALID, "rotary: descriptor is NULL");
    if (d->batch < 0 || d->tokens < 0 || d->dim < 1 || d->q_heads < 0 || d->k_heads < 0) return fail(WST_ERR_INVALID, "rotary: bad sizes");
    if (!type_ok(d->dtype)) return fail(WST_ERR_INVALID, "rotary: unknown type");
    if (d->axes < 1 || d->axes > WST_MAX_AXES) return fail(WST_ERR_INVALID, "rotary: 1 to %d axes, got %d", WST_MAX_AXES, d->axes);
    if (!(d->base > 0) || !std::isfinite(d->base)) return fail(WST_ERR_INVALID, "rotary: base must be positive");
    int64_t pairs = 0;
    for (int i = 0; i < d->axes; ++i) {
        if (d->sections[i] < 0) return fail(WST_ERR_INVALID, "rotary: negative section");
        pairs += d->sections[i];
    }
    if (2 * pairs > d->dim) return fail(WST_ERR_INVALID, "rotary: %lld pairs do not fit %d values", static_cast<long long>(pairs), d->dim);
    if (pairs > kMaxPairs) return fail(WST_ERR_UNSUPPORTED, "rotary: more than %d pairs", kMaxPairs);
    if (d->batch == 0 || d->tokens == 0 || d->q_heads + d->k_heads == 0) return WST_OK;
    if ((d->q_heads && (!q || !q_out)) || (d->k_heads && (!k || !k_out)) || !positions)
        return fail(WST_ERR_INVALID, "rotary: a pointer is NULL");
    RotaryTable tab{};
    int p = 0;
    for (int i = 0; i < d->axes; ++i)
        for (int j = 0; j < d->sections[i]; ++j, ++p) {
            tab.rev[p] = std::pow(d->base, -static_cast<double>(j) / d->sections[i]) / 6.283185307179586476925286766559;
            tab.axis[p] = static_cast<unsigned char>(i);
        }
    RotaryArgs a{};
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
    for (int i = 0; i < 3; ++i) {
        a.xs[0][i] = d->q_strides[i]; a.xs[1][i] = d->k_strides[i];
        a.ys[0][i] = d->q_out_strides[i]; a.ys[1][i] = d->k_out_strides[i];
    }
    a.heads[0] = d->q_heads; a.heads[1] = d->k_heads;
    a.tokens = d->tokens;
    a.rows = d->batch * d->tokens;
    a.pos = positions;
    a.pos_sb = d->positions_shared ? 0 : d->tokens * d->axes;
    a.axes = d->axes; a.pairs = static_cast<int>(pairs); a.dim = d->dim;
    a.sign = d->inverse ? -1.f : 1.f;
    const int units = (a.pairs + kRotPairs - 1) / kRotPairs + (a.dim - 2 * a.pairs + 7) / 8;
    const double blocks = std::ceil(static_cast<double>(a.rows) * units / 256.0);
    if (blocks * 256 >= 4294967296.0) return fail(WST_ERR_UNSUPPORTED, "rotary: too many tokens for one launch");
    // a thread walks all heads with one set of angles; few tokens: the heads are shared out over more blocks
    const int total = a.heads[0] + a.heads[1];
    int split = static_cast<int>(2048.0 / blocks);
    a.split = split < 1 ? 1 : split > total ? total : split;
    if (a.split > 65535) a.split = 65535;
    const dim3 g(static_cast<unsigned>(blocks), a.split);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    with_type(d->dtype, [&](auto tx) {
        using T = typename decltype(tx)::type;
        if (d->interleaved) k_rotary<T, true><<<g, dim3(256), 0, st>>>(a, tab);
        else k_rotary<T, false><<<g, dim3(256), 0, st>>>(a, tab);
        return 0;
    });
    return launched("rotary");
}

}  // extern "C"
