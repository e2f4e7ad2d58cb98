// grouped.hip — matrix products grouped by expert with ragged numbers of rows, and the gradient of their weights.
//
// gpx_grouped_gemm: rows t of group g (offsets[g] <= t < offsets[g+1]):  y_t = alpha W_g x_t + beta y_t.
//   D(i, j) with i = row, j = output column: P = X (k contiguous), Q = W_g in either layout, so the input gradient
//   dX = dY W is the same call with the other layout flag.
// gpx_grouped_gemm_dw: C_g = alpha sum_{t in g} dy_t x_t^T + beta C_g: P = dY, Q = X, both with k (= rows t) strided.
//
// The offsets live on the device: the host never waits for them.  Every kernel clamps them to [0, T] and reads a
// decreasing pair as an empty group, so no value of theirs leads outside the buffers.
#include <type_traits>
#include "mm_tile.h"
#include "../../include/gpx.h"

namespace {

using mm::v4f;

struct GroupedArgs {
    const char* X; const char* W; char* Y;
    const int64_t* offsets;
    long ldx, ldw, stride_w, ldy;   // bytes
    long T;
    int groups, N, K;
    double alpha, beta;
    int vec;   // Y's rows allow 4-element stores
};

__device__ __forceinline__ long clamped(const int64_t* offsets, int g, long T) {
    const long o = offsets[g];
    return o < 0 ? 0 : o > T ? T : o;
}

struct RowTile { int group, rows; long row0; };   // rows of this tile; group < 0: no tile

// The tile number `t` in the order of the groups, ceil(rows / BM) tiles each.  One wave looks at 64 groups at a time: the
// tile counts, their running sum over the lanes, and the first lane whose sum passes t.
template <int BM> __device__ RowTile find_row_tile(const int64_t* offsets, int groups, long T, long t) {
    const int lane = threadIdx.x & 63;
    RowTile out = {-1, 0, 0};
    long before = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const int g = g0 + lane;
        long lo = 0, rows = 0;
        if (g < groups) {
            lo = clamped(offsets, g, T);
            const long hi = clamped(offsets, g + 1, T);
            rows = hi > lo ? hi - lo : 0;
        }
        const long tiles = (rows + BM - 1) / BM;
        long sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const long up = __shfl_up(sum, d, 64);
            if (lane >= d) sum += up;
        }
        const unsigned long long past = __ballot(before + sum > t);
        if (past) {
            const int src = __builtin_ctzll(past);
            const long mine = t - (before + sum - tiles);   // tile within the group
            out.group = g0 + src;
            const long m = __shfl(mine, src, 64);
            const long r = __shfl(rows, src, 64) - m * BM;
            out.rows = (int)(r < BM ? r : BM);
            out.row0 = __shfl(lo, src, 64) + m * BM;
            break;
        }
        before += __shfl(sum, 63, 64);
    }
    out.group = __builtin_amdgcn_readfirstlane(out.group);
    out.rows = __builtin_amdgcn_readfirstlane(out.rows);
    return out;
}

template <class O, class A, int CNT>
__device__ __forceinline__ void put(char* row, int j, int N, const A* v, A alpha, A beta, bool vec) {
    O* p = reinterpret_cast<O*>(row) + j;
    if (CNT == 4 && vec && j + 4 <= N) {
        union { O e[4]; int w[sizeof(O)]; } u;
        typedef int words __attribute__((ext_vector_type(sizeof(O) == 8 ? 4 : sizeof(O))));
        if (beta != A(0)) {
#pragma unroll
            for (int x = 0; x < 4; ++x) u.e[x] = (O)(alpha * v[x] + beta * (A)p[x]);
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) u.e[x] = (O)(alpha * v[x]);
        }
        words w;
#pragma unroll
        for (int x = 0; x < (int)sizeof(O); ++x) w[x] = u.w[x];
        *reinterpret_cast<words*>(p) = w;
        return;
    }
#pragma unroll
    for (int x = 0; x < CNT; ++x)
        if (j + x < N) p[x] = (O)(beta != A(0) ? alpha * v[x] + beta * (A)p[x] : alpha * v[x]);
}

template <class T, int BM, int BN, int WR, int WC, bool WKC, bool DIRECT>
__global__ __launch_bounds__(WR * WC * 64, 2) void grouped_kernel(const GroupedArgs g) {
    typedef mm::Tile<T, BM, BN, WR, WC, true, WKC> Tile;
    typedef typename Tile::one A;
    __shared__ __attribute__((aligned(128))) char lds[Tile::LDS];
    const int nt = (g.N + BN - 1) / BN;
    const RowTile rt = find_row_tile<BM>(g.offsets, g.groups, g.T, blockIdx.x / nt);
    if (rt.group < 0) return;
    const int n0 = (int)(blockIdx.x % nt) * BN;
    typename Tile::OpP p = {g.X + rt.row0 * g.ldx, g.ldx, rt.rows, g.K};
    typename Tile::OpQ q = {g.W + rt.group * g.stride_w + (WKC ? n0 * g.ldw : n0 * (long)sizeof(T)), g.ldw, min(g.N - n0, BN), g.K};
    Tile t;
    t.clear();
    if (DIRECT) t.run_direct(lds, p, q, g.K);
    else t.run_staged(lds, p, q, g.K);
    char* y = g.Y + rt.row0 * g.ldy;
    const A alpha = (A)g.alpha, beta = (A)g.beta;
    t.each([&](int i, int j, const A* v, auto cnt) {
        if (i < rt.rows) put<T, A, decltype(cnt)::value>(y + i * g.ldy, n0 + j, g.N, v, alpha, beta, g.vec);
    });
}

struct GroupedDwArgs {
    const char* X; const char* Z; char* C;   // Z: the gradient of the outputs
    const int64_t* offsets;
    long ldx, ldz, ldc, stride_c;   // bytes
    long T;
    int M, N;   // columns of X (contiguous in C) and of Z
    double alpha, beta;
    int vec;
};

// rows in whole, aligned 16-byte chunks: what a direct-to-LDS load needs
bool whole_chunks(const void* p, long ld_bytes, long stride_bytes, long extent, long elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0 && stride_bytes % 16 == 0 && extent * elem % 16 == 0;
}

template <class T, class O, int BM, int BN, int WR, int WC, bool DIRECT>
__global__ __launch_bounds__(WR * WC * 64, 2) void grouped_dw_kernel(const GroupedDwArgs g) {
    typedef mm::Tile<T, BM, BN, WR, WC, false, false> Tile;
    typedef typename Tile::one A;
    __shared__ __attribute__((aligned(128))) char lds[Tile::LDS];
    const int mt = (g.M + BN - 1) / BN;
    const int group = blockIdx.y;
    const int n0 = (int)(blockIdx.x / mt) * BM, m0 = (int)(blockIdx.x % mt) * BN;
    const long lo = clamped(g.offsets, group, g.T), hi = clamped(g.offsets, group + 1, g.T);
    const int rows = (int)(hi > lo ? hi - lo : 0);
    typename Tile::OpP p = {g.Z + lo * g.ldz + n0 * (long)sizeof(T), g.ldz, min(g.N - n0, BM), rows};
    typename Tile::OpQ q = {g.X + lo * g.ldx + m0 * (long)sizeof(T), g.ldx, min(g.M - m0, BN), rows};
    Tile t;
    t.clear();
    if (DIRECT) t.run_direct(lds, p, q, rows);
    else t.run_staged(lds, p, q, rows);
    char* c = g.C + group * g.stride_c + n0 * g.ldc;
    const A alpha = (A)g.alpha, beta = (A)g.beta;
    t.each([&](int i, int j, const A* v, auto cnt) {
        if (n0 + i < g.N) put<O, A, decltype(cnt)::value>(c + i * g.ldc, m0 + j, g.M, v, alpha, beta, g.vec);
    });
}

// A row-tile count that is never less than sum of ceil(rows / BM)
long row_tiles(long T, int groups, int BM) { return T / BM + (groups < T ? groups : T); }

template <class T, int BM, int BN, int WR, int WC> int grouped_launch(hipStream_t st, bool w_kc, bool direct, const GroupedArgs& g) {
    const long tiles = row_tiles(g.T, g.groups, BM) * ((g.N + BN - 1) / BN);
    if (tiles >= 1L << 31) return GPX_ERR_UNSUPPORTED;
    auto go = [&](auto kc, auto dir) {
        grouped_kernel<T, BM, BN, WR, WC, decltype(kc)::value, decltype(dir)::value><<<(unsigned)tiles, WR * WC * 64, 0, st>>>(g);
    };
    if (w_kc && direct) go(std::true_type{}, std::true_type{});
    else if (w_kc) go(std::true_type{}, std::false_type{});
    else if (direct) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
    HIP_TRY(hipGetLastError());
    return GPX_OK;
}
// 16-bit products: 256 x 256 tiles (one workgroup of 8 waves per CU, 128 KB of LDS) once they fill the chip, else 128 x 128
// (two workgroups of 4 waves per CU).  bf16, 8 x (4096 x 4096 x 7168): 1.17-1.23 PFLOP/s against 1.02-1.05; 8 groups of one
// row, N = 1024, K = 512: 17.5 us against 11.5.
bool tile256(long row_tiles256, long N) { return row_tiles256 * ((N + 255) / 256) >= 256; }

template <class T> int grouped_typed(hipStream_t st, bool w_kc, const GroupedArgs& g) {
    // rows of X (k contiguous) and of W in 16-byte chunks, lane offsets of one K step within the buffer resource
    const long wn = w_kc ? g.K : g.N;   // W's contiguous extent
    const bool direct = whole_chunks(g.X, g.ldx, 0, g.K, sizeof(T)) && whole_chunks(g.W, g.ldw, g.stride_w, wn, sizeof(T)) &&
                        256 * g.ldx < (long)mm::kRange && 256 * g.ldw < (long)mm::kRange;
    if constexpr (sizeof(T) == 2)
        if (tile256(g.T / 256 + g.groups / 2, g.N)) return grouped_launch<T, 256, 256, 2, 4>(st, w_kc, direct, g);
    return grouped_launch<T, 128, 128, 2, 2>(st, w_kc, direct, g);
}

template <class T, class O, int BM, int BN, int WR, int WC> int grouped_dw_launch(hipStream_t st, bool direct, const GroupedDwArgs& g, int groups) {
    const long tiles = (long)((g.N + BM - 1) / BM) * ((g.M + BN - 1) / BN);
    if (tiles >= 1L << 31) return GPX_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)tiles, (unsigned)groups);
    if (direct) grouped_dw_kernel<T, O, BM, BN, WR, WC, true><<<grid, WR * WC * 64, 0, st>>>(g);
    else grouped_dw_kernel<T, O, BM, BN, WR, WC, false><<<grid, WR * WC * 64, 0, st>>>(g);
    HIP_TRY(hipGetLastError());
    return GPX_OK;
}

template <class T, class O> int grouped_dw_typed(hipStream_t st, const GroupedDwArgs& g, int groups) {
    const bool direct = whole_chunks(g.X, g.ldx, 0, g.M, sizeof(T)) && whole_chunks(g.Z, g.ldz, 0, g.N, sizeof(T)) &&
                        64 * g.ldx < (long)mm::kRange && 64 * g.ldz < (long)mm::kRange;
    if constexpr (sizeof(T) == 2)
        if (tile256((long)groups * ((g.N + 255) / 256), g.M)) return grouped_dw_launch<T, O, 256, 256, 2, 4>(st, direct, g, groups);
    return grouped_dw_launch<T, O, 128, 128, 2, 2>(st, direct, g, groups);
}

constexpr long kMaxExtent = (1L << 31) - 1024;   // row, column and k numbers within one product are 32-bit
constexpr int kMaxGroups = 65535;

int elem_bytes(int dtype) { return dtype == GPX_F64 ? 8 : dtype == GPX_F32 ? 4 : dtype == GPX_BF16 || dtype == GPX_F16 ? 2 : 0; }
bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes != 0; }
bool rows4(const void* p, long ld_bytes, long stride_bytes, int elem) {   // 4-element vector stores
    const uintptr_t a = (uintptr_t)(elem == 8 ? 16 : 4 * elem);
    return reinterpret_cast<uintptr_t>(p) % a == 0 && ld_bytes % (long)a == 0 && stride_bytes % (long)a == 0;
}

}  // namespace

extern "C" int gpx_grouped_gemm(int dtype, int w_kc, int64_t groups, int64_t T, int64_t N, int64_t K, double alpha, const void* X,
                                int64_t ldx, const void* W, int64_t ldw, int64_t stride_w, const int64_t* offsets, double beta,
                                void* Y, int64_t ldy, void* hip_stream) {
    const int e = elem_bytes(dtype);
    if (!e || groups < 0 || groups > kMaxGroups || T < 0 || N < 0 || K < 0) return GPX_ERR_ARG;
    if (T > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return GPX_ERR_ARG;
    if (ldx < K || ldw < (w_kc ? K : N) || ldy < N || stride_w < 0) return GPX_ERR_ARG;
    if (groups == 0 || T == 0 || N == 0) return GPX_OK;   // no row of Y belongs to a group
    if (!Y || !offsets || (K > 0 && (!X || !W))) return GPX_ERR_ARG;
    if (misaligned(X, e) || misaligned(W, e) || misaligned(Y, e) || misaligned(offsets, 8)) return GPX_ERR_ARG;
    StreamDevice dev(static_cast<hipStream_t>(hip_stream));
    if (dev.status) return dev.status;
    GroupedArgs g = {static_cast<const char*>(X), static_cast<const char*>(W), static_cast<char*>(Y), offsets, ldx * e, ldw * e,
                     stride_w * e, ldy * e, T, (int)groups, (int)N, (int)K, alpha, beta, rows4(Y, ldy * e, 0, e)};
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    switch (dtype) {
        case GPX_F64: return grouped_typed<double>(st, w_kc != 0, g);
        case GPX_F32: return grouped_typed<float>(st, w_kc != 0, g);
        case GPX_BF16: return grouped_typed<__bf16>(st, w_kc != 0, g);
        default: return grouped_typed<_Float16>(st, w_kc != 0, g);
    }
}

extern "C" int gpx_grouped_gemm_dw(int dtype, int c_dtype, int64_t groups, int64_t T, int64_t M, int64_t N, double alpha,
                                   const void* X, int64_t ldx, const void* Z, int64_t ldz, const int64_t* offsets, double beta,
                                   void* C, int64_t ldc, int64_t stride_c, void* work, int64_t work_bytes, void* hip_stream) {
    const int e = elem_bytes(dtype), ec = elem_bytes(c_dtype);
    if (!e || !ec || (c_dtype != dtype && !(c_dtype == GPX_F32 && e == 2))) return GPX_ERR_ARG;
    if (groups < 0 || groups > kMaxGroups || T < 0 || M < 0 || N < 0 || T > kMaxExtent || M > kMaxExtent || N > kMaxExtent)
        return GPX_ERR_ARG;
    if (ldx < M || ldz < N || ldc < M || stride_c < 0 || work_bytes < 0) return GPX_ERR_ARG;
    if (groups == 0 || M == 0 || N == 0) return GPX_OK;
    if (groups > 1 && stride_c < (N - 1) * ldc + M) return GPX_ERR_ARG;   // results of two groups would overlap
    if (!C || !offsets || (T > 0 && (!X || !Z))) return GPX_ERR_ARG;
    if (misaligned(X, e) || misaligned(Z, e) || misaligned(C, ec) || misaligned(offsets, 8)) return GPX_ERR_ARG;
    StreamDevice dev(static_cast<hipStream_t>(hip_stream));
    if (dev.status) return dev.status;
    GroupedDwArgs g = {static_cast<const char*>(X), static_cast<const char*>(Z), static_cast<char*>(C), offsets, ldx * e, ldz * e,
                       ldc * ec, stride_c * ec, T, (int)M, (int)N, alpha, beta, rows4(C, ldc * ec, stride_c * ec, ec)};
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int n = (int)groups;
    switch (dtype) {
        case GPX_F64: return grouped_dw_typed<double, double>(st, g, n);
        case GPX_F32: return grouped_dw_typed<float, float>(st, g, n);
        case GPX_BF16: return c_dtype == GPX_F32 ? grouped_dw_typed<__bf16, float>(st, g, n) : grouped_dw_typed<__bf16, __bf16>(st, g, n);
        default: return c_dtype == GPX_F32 ? grouped_dw_typed<_Float16, float>(st, g, n) : grouped_dw_typed<_Float16, _Float16>(st, g, n);
    }
}

extern "C" int gpx_grouped_gemm_dw_work(int dtype, int64_t groups, int64_t T, int64_t M, int64_t N, int64_t* work_bytes) {
    if (!elem_bytes(dtype) || !work_bytes || groups < 0 || T < 0 || M < 0 || N < 0) return GPX_ERR_ARG;
    *work_bytes = 0;
    return GPX_OK;
}
