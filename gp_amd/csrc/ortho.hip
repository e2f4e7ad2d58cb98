// ortho.hip — orthogonalised update of a batch of matrices by Newton-Schulz products.
//
// X_0 = G / (|G|_F + eps);  step k:  A = X X^T,  X <- a X + (b A + c A A) X = p(X),  an odd polynomial that acts on the singular
// values alone: sigma -> a sigma + b sigma^3 + c sigma^5.  |G|_F >= sigma_max, so the singular values start in [0, 1].
// For matrices with more rows than columns the same is done with X^T X from the right: the products with the long side
// stay two, the square ones have the short side.
#include <algorithm>
#include <cmath>
#include "mm_tile.h"
#include "../../include/gpx.h"

namespace {

constexpr int kParts = 64;   // partial sums of squares per matrix

template <class T> __device__ __forceinline__ double as_double(T v) { return (double)v; }

// sums of squares in double: neither overflow nor loss for any float input, one order of addition
template <class T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const T* __restrict__ G, long ldg, long stride_g, int rows, int cols, double* __restrict__ part) {
    const T* g = G + blockIdx.y * stride_g;
    const long total = (long)rows * cols, per = (total + kParts - 1) / kParts;
    const long lo = blockIdx.x * per, hi = min(total, lo + per);
    double s = 0.0;
    for (long e = lo + threadIdx.x; e < hi; e += 256) {
        const double v = as_double(g[e / cols * ldg + e % cols]);
        s = fma(v, v, s);
    }
#pragma unroll
    for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, 64);
    __shared__ double ws[4];
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * kParts + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

template <class T, class O>
__global__ __launch_bounds__(256) void ortho_scale_kernel(const T* G, long ldg, long stride_g, int rows, int cols, const double* __restrict__ part,
                                                          double eps, O* X, long ldx, long stride_x) {
    double s = part[blockIdx.y * kParts + (threadIdx.x & 63)];
#pragma unroll
    for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, 64);
    const double norm = sqrt(s) + eps;
    const long total = (long)rows * cols;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        const long r = e / cols, c = e % cols;
        X[blockIdx.y * stride_x + r * ldx + c] = (O)(as_double(G[blockIdx.y * stride_g + r * ldg + c]) / norm);
    }
}

// D = c1 P Q^T + c2 E over a batch; W: type of the iterates (float, or double for double matrices)
struct OrthoArgs {
    const char* P; const char* Q; const char* E; char* D;
    long ldp, ldq, lde, ldd, sp, sq, se, sd;   // bytes
    int I, J, K;
    double c1, c2;
};
template <class W, class O, bool PKC, bool QKC>
__global__ __launch_bounds__(256, 2) void ortho_mm_kernel(const OrthoArgs g) {
    typedef mm::Tile<W, 128, 128, 2, 2, PKC, QKC> Tile;
    __shared__ __attribute__((aligned(128))) char lds[Tile::LDS];
    const int jt = (g.J + 127) / 128;
    const int i0 = (int)(blockIdx.x / jt) * 128, j0 = (int)(blockIdx.x % jt) * 128;
    typename Tile::OpP p = {g.P + blockIdx.y * g.sp + (PKC ? i0 * g.ldp : i0 * (long)sizeof(W)), g.ldp, min(g.I - i0, 128), g.K};
    typename Tile::OpQ q = {g.Q + blockIdx.y * g.sq + (QKC ? j0 * g.ldq : j0 * (long)sizeof(W)), g.ldq, min(g.J - j0, 128), g.K};
    Tile t;
    t.clear();
    t.run_staged(lds, p, q, g.K);
    const W c1 = (W)g.c1, c2 = (W)g.c2;
    t.each([&](int i, int j, const W* v, auto) {
        i += i0;
        j += j0;
        if (i >= g.I || j >= g.J) return;
        const W e = g.c2 != 0.0 ? c2 * reinterpret_cast<const W*>(g.E + blockIdx.y * g.se + i * g.lde)[j] : W(0);
        reinterpret_cast<O*>(g.D + blockIdx.y * g.sd + i * g.ldd)[j] = (O)(c1 * v[0] + e);
    });
}

struct OrthoWork {   // offsets in bytes
    long part, x[2], a, b, total;
};
OrthoWork ortho_work(int dtype, long batch, long rows, long cols) {
    const long w = dtype == GPX_F64 ? 8 : 4, s = std::min(rows, cols);
    auto up = [](long v) { return (v + 255) / 256 * 256; };
    OrthoWork o;
    o.part = 0;
    o.x[0] = up(batch * kParts * 8);
    o.x[1] = o.x[0] + up(batch * rows * cols * w);
    o.a = o.x[1] + up(batch * rows * cols * w);
    o.b = o.a + up(batch * s * s * w);
    o.total = o.b + up(batch * s * s * w);
    return o;
}

template <class W, class O, bool PKC, bool QKC> int launch(hipStream_t st, const OrthoArgs& g, int batch) {
    const long tiles = ((g.I + 127L) / 128) * ((g.J + 127L) / 128);
    ortho_mm_kernel<W, O, PKC, QKC><<<dim3((unsigned)tiles, (unsigned)batch), 256, 0, st>>>(g);
    HIP_TRY(hipGetLastError());
    return GPX_OK;
}

// rows x cols row-major (the column-major cols x rows of the C interface)
template <class T, class W>
int ortho_typed(hipStream_t st, int dtype, int batch, int rows, int cols, const T* G, long ldg, long stride_g, int steps, const double* coef,
                double eps, T* O, long ldo, long stride_o, char* work) {
    const OrthoWork o = ortho_work(dtype, batch, rows, cols);
    double* part = reinterpret_cast<double*>(work + o.part);
    ortho_norm_kernel<T><<<dim3(kParts, batch), 256, 0, st>>>(G, ldg, stride_g, rows, cols, part);
    HIP_TRY(hipGetLastError());
    const long total = (long)rows * cols;
    const dim3 grid((unsigned)std::min<long>((total + 1023) / 1024, 2048), (unsigned)batch);
    if (steps == 0) {
        ortho_scale_kernel<T, T><<<grid, 256, 0, st>>>(G, ldg, stride_g, rows, cols, part, eps, O, ldo, stride_o);
        HIP_TRY(hipGetLastError());
        return GPX_OK;
    }
    char* x[2] = {work + o.x[0], work + o.x[1]};
    char *a = work + o.a, *b = work + o.b;
    ortho_scale_kernel<T, W><<<grid, 256, 0, st>>>(G, ldg, stride_g, rows, cols, part, eps, reinterpret_cast<W*>(x[0]), cols, total);
    HIP_TRY(hipGetLastError());
    const bool tall = rows > cols;
    const int s = std::min(rows, cols), l = std::max(rows, cols);
    const long w = sizeof(W), ldx = cols * w, sx = total * w, lda = s * w, sa = (long)s * s * w;
    for (int k = 0; k < steps; ++k) {
        const double ca = coef[3 * k], cb = coef[3 * k + 1], cc = coef[3 * k + 2];
        char *from = x[k & 1], *to = x[~k & 1];
        OrthoArgs gram = {from, from, nullptr, a, ldx, ldx, 0, lda, sx, sx, 0, sa, s, s, l, 1.0, 0.0};
        int rc = tall ? launch<W, W, false, false>(st, gram, batch) : launch<W, W, true, true>(st, gram, batch);
        if (rc) return rc;
        OrthoArgs poly = {a, a, a, b, lda, lda, lda, lda, sa, sa, sa, sa, s, s, s, cc, cb};
        if ((rc = launch<W, W, true, true>(st, poly, batch))) return rc;
        const bool last = k + 1 == steps;
        const long ldd = last ? ldo * (long)sizeof(T) : ldx, sd = last ? stride_o * (long)sizeof(T) : sx;
        char* d = last ? reinterpret_cast<char*>(O) : to;
        OrthoArgs apply = tall ? OrthoArgs{from, b, from, d, ldx, lda, ldx, ldd, sx, sa, sx, sd, rows, cols, s, 1.0, ca}
                               : OrthoArgs{b, from, from, d, lda, ldx, ldx, ldd, sa, sx, sx, sd, rows, cols, s, 1.0, ca};
        if (tall) rc = last ? launch<W, T, true, true>(st, apply, batch) : launch<W, W, true, true>(st, apply, batch);
        else rc = last ? launch<W, T, true, false>(st, apply, batch) : launch<W, W, true, false>(st, apply, batch);
        if (rc) return rc;
    }
    return GPX_OK;
}

constexpr int kMaxSteps = 64;
constexpr long kMaxSide = 1L << 20;
const double kQuintic[3] = {3.4445, -4.7750, 2.0315};

bool sizes_ok(int dtype, int64_t batch, int64_t M, int64_t N) {
    return dtype >= GPX_F64 && dtype <= GPX_F16 && batch >= 0 && batch <= 65535 && M >= 0 && N >= 0 && M <= kMaxSide && N <= kMaxSide;
}

}  // namespace

extern "C" int gpx_orthogonalize_work(int dtype, int64_t batch, int64_t M, int64_t N, int64_t* work_bytes) {
    if (!work_bytes || !sizes_ok(dtype, batch, M, N)) return GPX_ERR_ARG;
    *work_bytes = batch && M && N ? ortho_work(dtype, batch, N, M).total : 0;
    return GPX_OK;
}

extern "C" int gpx_orthogonalize(int dtype, int64_t batch, int64_t M, int64_t N, const void* G, int64_t ldg, int64_t stride_g, int steps,
                                 const double* coef, double eps, void* O, int64_t ldo, int64_t stride_o, void* work, int64_t work_bytes,
                                 void* hip_stream) {
    if (!sizes_ok(dtype, batch, M, N) || steps < 0 || steps > kMaxSteps || !(eps > 0.0) || !std::isfinite(eps)) return GPX_ERR_ARG;
    if (ldg < M || ldo < M || stride_g < 0 || stride_o < 0) return GPX_ERR_ARG;
    if (batch == 0 || M == 0 || N == 0) return GPX_OK;
    if (batch > 1 && stride_o < (N - 1) * ldo + M) return GPX_ERR_ARG;   // results of two matrices would overlap
    if (!G || !O || !work) return GPX_ERR_ARG;
    const uintptr_t e = dtype == GPX_F64 ? 8 : dtype == GPX_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(G) % e || reinterpret_cast<uintptr_t>(O) % e || reinterpret_cast<uintptr_t>(work) % 16) return GPX_ERR_ARG;
    if (work_bytes < ortho_work(dtype, batch, N, M).total) return GPX_ERR_ARG;
    double table[3 * kMaxSteps];
    for (int k = 0; k < steps; ++k)
        for (int c = 0; c < 3; ++c) {
            table[3 * k + c] = coef ? coef[3 * k + c] : kQuintic[c];
            if (!std::isfinite(table[3 * k + c])) return GPX_ERR_ARG;
        }
    StreamDevice dev(static_cast<hipStream_t>(hip_stream));
    if (dev.status) return dev.status;
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    char* w = static_cast<char*>(work);
    const int b = (int)batch, r = (int)N, c = (int)M;
    switch (dtype) {
        case GPX_F64:
            return ortho_typed<double, double>(st, dtype, b, r, c, static_cast<const double*>(G), ldg, stride_g, steps, table, eps,
                                               static_cast<double*>(O), ldo, stride_o, w);
        case GPX_F32:
            return ortho_typed<float, float>(st, dtype, b, r, c, static_cast<const float*>(G), ldg, stride_g, steps, table, eps,
                                             static_cast<float*>(O), ldo, stride_o, w);
        case GPX_BF16:
            return ortho_typed<__bf16, float>(st, dtype, b, r, c, static_cast<const __bf16*>(G), ldg, stride_g, steps, table, eps,
                                              static_cast<__bf16*>(O), ldo, stride_o, w);
        default:
            return ortho_typed<_Float16, float>(st, dtype, b, r, c, static_cast<const _Float16*>(G), ldg, stride_g, steps, table, eps,
                                                static_cast<_Float16*>(O), ldo, stride_o, w);
    }
}
