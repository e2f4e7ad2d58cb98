// ortho.hip — orthogonalised update of a batch of matrices by Newton-Schulz products.
//
// X_0 = G / (|G|_F + eps);  step k:  A = X X^T,  X <- a X + (b A + c A A) X = p(X),  an odd polynomial that acts on the singular
// values alone: sigma -> a sigma + b sigma^3 + c sigma^5.  |G|_F >= sigma_max, so the singular values start in [0, 1].
// For matrices with more rows than columns the same is done with X^T X from the right: the products with the long side
// stay two, the square ones have the short side.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "mm_tile.h"
#include "../../include/gpx.h"

namespace {

constexpr int kParts = 256;   // partial sums of squares per matrix, at most

template <class T> __device__ __forceinline__ double as_double(T v) { return (double)v; }

// Walks the runs of 8 neighbours of a rows x cols matrix, run number `first` and every `step`-th behind it, without a
// division per run: f(row, first column of the run).
template <class Body> __device__ __forceinline__ void each_run(int rows, int cols, long first, long step, Body&& f) {
    const int n8 = (cols + 7) / 8;
    long r = first / n8, dr = step / n8;
    int c = (int)(first % n8), dc = (int)(step % n8);
#pragma unroll 4
    while (r < rows) {
        f((int)r, c * 8);
        r += dr;
        c += dc;
        if (c >= n8) {
            c -= n8;
            ++r;
        }
    }
}
// v = the run at p, of which `count` elements exist
template <class T> __device__ __forceinline__ void load_run(const T* p, int count, T (&v)[8]) {
    if (count >= 8) {   // at any alignment
        __builtin_memcpy(v, p, sizeof v);
    } else {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = x < count ? p[x] : (T)0.0f;
    }
}

// Sums of squares in double: neither overflow nor loss for any narrower input, one order of addition.  Doubles take three sums, of
// values beyond 2^480, below 2^-480 and between, the outer ones scaled by 2^-600 and 2^600, and leave the root instead.
template <class T> struct Squares {
    double s;
    __device__ __forceinline__ void add(T v) { s = fma(as_double(v), as_double(v), s); }
    __device__ __forceinline__ void join(int d) { s += __shfl_xor(s, d, 64); }
    __device__ __forceinline__ void join(const Squares& o) { s += o.s; }
    __device__ __forceinline__ double part() const { return s; }
};
template <> struct Squares<double> {
    double s, large, little;
    __device__ __forceinline__ void add(double v) {
        const double a = fabs(v), b = a > 0x1p480 ? a * 0x1p-600 : a < 0x1p-480 ? a * 0x1p600 : a;
        const double q = b * b;   // (NaN goes between)
        if (a > 0x1p480) large += q;
        else if (a < 0x1p-480) little += q;
        else s += q;
    }
    __device__ __forceinline__ void join(int d) {
        s += __shfl_xor(s, d, 64);
        large += __shfl_xor(large, d, 64);
        little += __shfl_xor(little, d, 64);
    }
    __device__ __forceinline__ void join(const Squares& o) {
        s += o.s;
        large += o.large;
        little += o.little;
    }
    __device__ __forceinline__ double part() const {
        return hypot(hypot(sqrt(large) * 0x1p600, sqrt(s)), sqrt(little) * 0x1p-600);
    }
};

template <class T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const T* __restrict__ G, long ldg, long stride_g, int rows, int cols, double* __restrict__ part) {
    const T* g = G + blockIdx.y * stride_g;
    Squares<T> s = {};
    each_run(rows, cols, blockIdx.x * 256L + threadIdx.x, gridDim.x * 256L, [&](int r, int c) {
        T v[8];
        load_run(g + r * ldg + c, cols - c, v);
#pragma unroll
        for (int x = 0; x < 8; ++x) s.add(v[x]);
    });
#pragma unroll
    for (int d = 32; d; d /= 2) s.join(d);
    __shared__ Squares<T> ws[4];
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        Squares<T> a = ws[0], b = ws[2];
        a.join(ws[1]);
        b.join(ws[3]);
        a.join(b);
        part[blockIdx.y * (long)gridDim.x + blockIdx.x] = a.part();
    }
}

// the norm of one matrix of T from its partial sums (or roots), in every lane
template <class T> __device__ __forceinline__ double norm_of(const double* part, int parts) {
    double s = 0.0;
    if constexpr (__is_same(T, double)) {
        double most = 0.0;
        bool finite = true;
        for (int e = threadIdx.x & 63; e < parts; e += 64) {
            most = fmax(most, part[e]);
            finite = finite && isfinite(part[e]);
            s += part[e];
        }
#pragma unroll
        for (int d = 32; d; d /= 2) {
            most = fmax(most, __shfl_xor(most, d, 64));
            s += __shfl_xor(s, d, 64);
        }
        if (!__all(finite) || most == 0.0) return s;   // an infinity or NaN, or zero
        s = 0.0;
        for (int e = threadIdx.x & 63; e < parts; e += 64) s = fma(part[e] / most, part[e] / most, s);
#pragma unroll
        for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, 64);
        return most * sqrt(s);
    } else {
        for (int e = threadIdx.x & 63; e < parts; e += 64) s += part[e];
#pragma unroll
        for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, 64);
        return sqrt(s);
    }
}

// A positive factor of any size as mantissa and exponent: floats times it without overflow on the way, by the exact power of
// two first and one rounded product
struct Factor {
    double all;
    float mantissa;
    int exponent;
    __device__ explicit Factor(double v) : all(v) {
        exponent = isfinite(v) && v > 0.0 ? ilogb(v) : 0;
        mantissa = (float)ldexp(v, -exponent);
    }
    __device__ __forceinline__ float times(float v) const { return ldexpf(v, exponent) * mantissa; }
};

// steps == 0: the normalised matrix itself.  G and X may be the same buffer.
template <class T>
__global__ __launch_bounds__(256) void ortho_normalize_kernel(const T* G, long ldg, long stride_g, int rows, int cols, const double* __restrict__ part,
                                                              int parts, double eps, T* X, long ldx, long stride_x) {
    const double norm = norm_of<T>(part + blockIdx.y * (long)parts, parts) + eps;
    each_run(rows, cols, blockIdx.x * 256L + threadIdx.x, gridDim.x * 256L, [&](int r, int c) {
        T v[8];
        load_run(G + blockIdx.y * stride_g + r * ldg + c, cols - c, v);
        T* x = X + blockIdx.y * stride_x + r * ldx + c;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols) x[e] = (T)(as_double(v[e]) / norm);
    });
}

// ---- the iterates ------------------------------------------------------------------------------------------------
// Double matrices stay in double.  All others are iterated in the split format, two f16 planes under one power of two per
// matrix and step: 22 bits of every value, the accumulators and all sums in 32.  One f16 product is 16 times the rate of a
// product of floats here, the three that the split needs leave a factor of five.  The host bounds the singular values of
// every iterate from the coefficients and places the largest possible element at 2^15: nothing overflows, and the smallest
// step of the second plane is 2^-39 of that bound.
// The largest elements of A and of b A + c A A, their diagonals, are kept in floats beside the matrices (zero in them) and applied
// where the products' results are written.  Relative error of the result without and with that, f32: 16 x 208 in three steps
// 1.2e-6 and 3.3e-7 (products of floats: 5.7e-7), 300 x 2000 in six 2.5e-6 and 6.6e-7 (2.9e-6).  It costs 0.5 us of 21 for a small
// matrix, 0.8 % for one of 4096 x 4096.
// bf16 matrices take the same planes.  In one plane of 11 bits their products take half the time (16 of 1024 x 2816), but the
// result is then further from 64 bits than its own rounding (1.73e-3 against 1.66e-3).
template <class F> struct Iterate;
// v = h + l.  The compiler may form a converted product in one rounding and the product itself in two; h has to be one value
// for both planes (told apart at ties, the planes would disagree by a step of the first one).
__device__ __forceinline__ void split(float v, _Float16& h, _Float16& l) {
    unsigned bits = __builtin_bit_cast(unsigned short, (_Float16)v);
    asm("" : "+v"(bits));
    h = __builtin_bit_cast(_Float16, (unsigned short)bits);
    l = (_Float16)(v - (float)h);
}
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
// the same for two neighbours, without rounding what is left
__device__ __forceinline__ v2h split2(v2f v, v2f& left) {
    unsigned bits = __builtin_bit_cast(unsigned, __builtin_convertvector(v, v2h));
    asm("" : "+v"(bits));
    const v2h h = __builtin_bit_cast(v2h, bits);
    left[0] = v[0] - (float)h[0];
    left[1] = v[1] - (float)h[1];
    return h;
}
template <> struct Iterate<double> {
    static constexpr int PAD = 2;
    __device__ static void store(char* row, int j, double v) { reinterpret_cast<double*>(row)[j] = v; }
    __device__ static double load(const char* row, int j) { return reinterpret_cast<const double*>(row)[j]; }
    static long bytes(long cols) { return cols * 8; }
};
template <> struct Iterate<mm::Split> {
    static constexpr int PAD = 32;
    __device__ static long at(int j) { return (long)(j >> 5) * 64 + (j & 31); }
    __device__ static void store(char* row, int j, float v) {
        _Float16* p = reinterpret_cast<_Float16*>(row) + at(j);
        split(v, p[0], p[32]);
    }
    __device__ static float load(const char* row, int j) {
        const _Float16* p = reinterpret_cast<const _Float16*>(row) + at(j);
        return (float)p[0] + (float)p[32];
    }
    static long bytes(long cols) { return cols * 4; }
    // eight neighbours from column j on, j a multiple of 8
    __device__ static void store8(char* row, int j, const float (&v)[8]) {
        mm::v8h h, l;
#pragma unroll
        for (int x = 0; x < 8; x += 2) {
            v2f left;
            const v2h a = split2(v2f{v[x], v[x + 1]}, left), b = __builtin_convertvector(left, v2h);
            h[x] = a[0];
            h[x + 1] = a[1];
            l[x] = b[0];
            l[x + 1] = b[1];
        }
        _Float16* p = reinterpret_cast<_Float16*>(row) + at(j);
        *reinterpret_cast<mm::v8h*>(p) = h;
        *reinterpret_cast<mm::v8h*>(p + 32) = l;
    }
    __device__ static void add8(const char* row, int j, const float (&by)[8], float (&v)[8]) {   // v += by * row
        const _Float16* p = reinterpret_cast<const _Float16*>(row) + at(j);
        const mm::v8h h = *reinterpret_cast<const mm::v8h*>(p), l = *reinterpret_cast<const mm::v8h*>(p + 32);
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] += by[x] * ((float)h[x] + (float)l[x]);
    }
};
template <class F> int padded(int cols) { return (cols + Iterate<F>::PAD - 1) / Iterate<F>::PAD * Iterate<F>::PAD; }

template <class T, class F>
__global__ __launch_bounds__(256) void ortho_scale_kernel(const T* __restrict__ G, long ldg, long stride_g, int rows, int cols, int pcols,
                                                          const double* __restrict__ part, int parts, double eps, double scale, char* __restrict__ X,
                                                          long ldx, long stride_x) {
    const double norm = norm_of<T>(part + blockIdx.y * (long)parts, parts) + eps;
    const Factor by(scale / norm);
    each_run(rows, pcols, blockIdx.x * 256L + threadIdx.x, gridDim.x * 256L, [&](int r, int c) {
        T v[8];
        load_run(G + blockIdx.y * stride_g + r * ldg + c, cols - c, v);
        char* x = X + blockIdx.y * stride_x + r * ldx;
        if constexpr (!__is_same(F, double)) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = by.times((float)v[e]);
            Iterate<F>::store8(x, c, w);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < pcols) Iterate<F>::store(x, c + e, as_double(v[e]) * by.all);
        }
    });
}

// D = c1 P Q^T + c2 E over a batch, E and D in the format F, or (LAST) D in the type O of the result.
// SYM: D is symmetric; tiles on and below the diagonal are computed, and those below it stored on both sides.
// Not for doubles: every square matrix has its diagonal, in floats, beside it, and zeros in its place.  A symmetric product leaves its own
// in diag_out; the square of A + diag(d) is A A + (d_i + d_j) A_ij + d_i^2, and diag(d) X is added to the product with X, by the
// rows of D where the square matrix is on the left, by its columns where it is on the right (QKC).
struct OrthoArgs {
    const char* P; const char* Q; const char* E; char* D;
    long ldp, ldq, lde, ldd, sp, sq, se, sd;   // bytes
    int I, J, K, batch;
    double c1, c2;
    const float* diag; float* diag_out;        // min(rows, cols) per matrix
};
template <class F, class O, bool LAST, int B, int WR, int WC, int ST, int KG, bool PKC, bool QKC, bool SYM>
__global__ __launch_bounds__(WR * WC * 64 * KG, KG > 1 ? 4 : B * B / (WR * WC) > 128 * 64 ? 1 : 2) void ortho_mm_kernel(const OrthoArgs g) {
    typedef mm::Tile<F, B, B, WR, WC, PKC, QKC, ST, KG> Tile;
    typedef typename Tile::one one;
    constexpr int W = mm::Stored<F>::WIDE * (int)sizeof(typename Tile::T);   // bytes per value
    constexpr int WE = mm::Stored<F>::WIDE;
    constexpr int LDS = !Tile::SWAP && Tile::SLAB > Tile::LDS ? Tile::SLAB : Tile::LDS;
    __shared__ __attribute__((aligned(128))) char lds[LDS];
    // Bands of eight tile rows, column by column, matrix after matrix; XCD x takes the x-th eighth of every chunk of
    // workgroups that the chip holds at a time, so that its CUs share eight row panels and a few column panels in their L2.
    constexpr int CHUNK = B > 128 || KG > 1 ? 256 : 512;
    const int it = (g.I + B - 1) / B, jt = (g.J + B - 1) / B;
    const unsigned tiles = SYM ? it * (it + 1) / 2 : it * jt, all = tiles * g.batch, start = blockIdx.x / CHUNK * CHUNK;
    if (start >= all) return;
    const unsigned here = min((unsigned)CHUNK, all - start), xcd = blockIdx.x & 7;
    const unsigned nth = here * xcd / 8 + (blockIdx.x % CHUNK >> 3);
    if (nth >= here * (xcd + 1) / 8) return;
    const int mat = (start + nth) / tiles;
    int in = (start + nth) % tiles, ti, tj;
    if (SYM) {   // band b: 8 b whole columns, then the triangle on the diagonal, row by row
        int band = 0, high = min(8, it), size = high * (high + 1) / 2;
        while (in >= size) {
            in -= size;
            ++band;
            high = min(8, it - 8 * band);
            size = 8 * band * high + high * (high + 1) / 2;
        }
        if (in < 8 * band * high) {
            ti = 8 * band + in % high;
            tj = in / high;
        } else {
            int r = 0;
            in -= 8 * band * high;
            while (in > r) in -= ++r;
            ti = 8 * band + r;
            tj = 8 * band + in;
        }
    } else {
        const int band = in / (8 * jt), high = min(8, it - 8 * band);
        in -= band * 8 * jt;
        ti = 8 * band + in % high;
        tj = in / high;
    }
    const int i0 = ti * B, j0 = tj * B;
    const int Jp = (g.J + Iterate<F>::PAD - 1) / Iterate<F>::PAD * Iterate<F>::PAD, Ip = (g.I + Iterate<F>::PAD - 1) / Iterate<F>::PAD * Iterate<F>::PAD;
    typename Tile::OpP p = {g.P + mat * g.sp + (PKC ? i0 * g.ldp : i0 * (long)W), g.ldp, PKC ? min(g.I - i0, B) : min(Ip - i0, B) * WE, g.K};
    typename Tile::OpQ q = {g.Q + mat * g.sq + (QKC ? j0 * g.ldq : j0 * (long)W), g.ldq, QKC ? min(g.J - j0, B) : min(Jp - j0, B) * WE, g.K};
    Tile t;
    t.clear();
    const one c1 = (one)g.c1, c2 = (one)g.c2;
    constexpr bool DIAG = !__is_same(F, double);
    const float* diag = DIAG && g.diag ? g.diag + mat * (long)(SYM ? g.I : g.K) : nullptr;
    if constexpr (KG > 1) t.run_groups(lds, p, q, g.K);
    else t.run_direct(lds, p, q, g.K);
    const char* E = g.E + mat * g.se;
    char* D = g.D + mat * g.sd;
    if constexpr (!Tile::SWAP) {
        // Through LDS, one wave row of the tile at a time, so that planes are read and written in runs of 16 bytes, the mirrored
        // tile too (single elements from the accumulators: 90 us for a 256 x 256 tile, most of it the mirrored stores).
        float* slab = reinterpret_cast<float*>(lds);
        constexpr int NT = Tile::THREADS, R = Tile::SLAB_ROWS;
        float* diag_out = DIAG && SYM ? g.diag_out + mat * (long)g.I : nullptr;
        auto factors = [&](int i, int j, int exist, float (&by)[8]) {   // of E(i, j..j+7)
#pragma unroll
            for (int x = 0; x < 8; ++x) by[x] = 0.0f;
            if constexpr (DIAG && (SYM || QKC)) load_run(diag + j, exist, by);
            const float of_row = DIAG && (SYM || !QKC) ? diag[i] : 0.0f;
#pragma unroll
            for (int x = 0; x < 8; ++x) by[x] = DIAG ? c2 + c1 * (of_row + by[x]) : c2;
        };
        for (int pass = 0; pass < WR; ++pass) {
            const int ib = i0 + pass * R;
            constexpr int RUNS = R * (B / 8), TURNS = (RUNS + NT - 1) / NT;
            __syncthreads();
            t.to_slab(slab, pass);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < TURNS; ++n) {
                const int e = threadIdx.x + n * NT;
                if (RUNS % NT != 0 && e >= RUNS) continue;
                const int il = e / (B / 8), i = ib + il, jl = e % (B / 8) * 8, j = j0 + jl;
                if (i >= g.I || j >= Jp) continue;
                float v[8];
                const mm::v4f lo = *reinterpret_cast<const mm::v4f*>(slab + Tile::slab_at(il, jl)), hi = *reinterpret_cast<const mm::v4f*>(slab + Tile::slab_at(il, jl + 4));
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    v[x] = c1 * lo[x];
                    v[4 + x] = c1 * hi[x];
                }
                if (c2 != 0.0f || (DIAG && diag)) {
                    float by[8];
                    factors(i, j, g.J - j, by);
                    Iterate<F>::add8(E + i * g.lde, j, by, v);
                }
                if constexpr (DIAG && SYM) {
                    if (i >= j && i < j + 8) {
                        const float d = diag ? diag[i] : 0.0f;
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (i == j + x) {
                                diag_out[i] = v[x] + (c2 + c1 * d) * d;
                                v[x] = 0.0f;
                            }
                    }
                }
                if constexpr (LAST) {
                    O* d = reinterpret_cast<O*>(D + i * g.ldd) + j;
                    typedef O o8 __attribute__((ext_vector_type(8)));
                    if (j + 8 <= g.J) {   // at any alignment
                        o8 w;
#pragma unroll
                        for (int x = 0; x < 8; ++x) w[x] = (O)v[x];
                        asm volatile("" ::: "memory");   // keep the run in one piece
                        __builtin_memcpy(d, &w, sizeof w);
                        asm volatile("" ::: "memory");
                    } else {
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (j + x < g.J) d[x] = (O)v[x];
                    }
                } else {
                    Iterate<F>::store8(D + i * g.ldd, j, v);
                }
            }
            if (SYM && ti != tj) {   // D(j, i): E is symmetric to the bit, so both triangles are
                // eight lanes along i (128 bytes of a row of D, both planes twice), eight along j
                for (int e = threadIdx.x; e < B * ((R + 63) / 64 * 8); e += NT) {
                    const int jl = (e >> 3) % B, j = j0 + jl, il = ((e & 7) + (e >> 3) / B * 8) * 8, i = ib + il;
                    if (R % 64 != 0 && il >= R) continue;
                    if (j >= g.J || i >= Ip) continue;
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = c1 * slab[Tile::slab_at(il + x, jl)];
                    if (c2 != 0.0f || (DIAG && diag)) {
                        float by[8];
                        factors(j, i, g.I - i, by);
                        Iterate<F>::add8(E + j * g.lde, i, by, v);
                    }
                    Iterate<F>::store8(D + j * g.ldd, i, v);
                }
            }
        }
    } else {
        if (Tile::group() != 0) return;
        t.each([&](int i, int j, const one* v, auto) {
            i += i0;
            j += j0;
            if (i >= g.I || j >= (LAST ? g.J : Jp)) return;
            one d = c1 * v[0];
            if (c2 != one(0) && j < g.J) d += c2 * Iterate<F>::load(E + i * g.lde, j);
            if constexpr (LAST) {
                reinterpret_cast<O*>(D + i * g.ldd)[j] = (O)d;
            } else {
                Iterate<F>::store(D + i * g.ldd, j, d);
                if (SYM && ti != tj && j < g.J) Iterate<F>::store(D + j * g.ldd, i, d);
            }
        });
        if (SYM && ti != tj && i0 + B >= g.I) {   // the zeros behind the rows that the mirrored tile ends
            const int w = Ip - g.I;
            for (int e = threadIdx.x; e < w * B; e += WR * WC * 64)
                if (j0 + e / w < g.J) Iterate<F>::store(D + (j0 + e / w) * g.ldd, g.I + e % w, one(0));
        }
    }
}

struct OrthoWork {   // offsets and strides in bytes; rows of the iterates padded to whole blocks
    long part, x[2], a, b, diag[2], total;   // diag: of a and b
    long ldx, sx, lda, sa;
};
// Rows of a power of two of bytes would meet in few memory channels: the K step of a tile reads 128 bytes of every row.
template <class F> long row_bytes(int cols) {
    const long b = Iterate<F>::bytes(padded<F>(cols));
    return b % 1024 == 0 ? b + 128 : b;
}
long up256(long v) { return (v + 255) / 256 * 256; }
template <class F> long norm_runs(int rows, int cols) { return (long)rows * ((padded<F>(cols) + 7) / 8); }
template <class F> int norm_parts(int rows, int cols) { return (int)std::min<long>((norm_runs<F>(rows, cols) + 511) / 512, kParts); }
template <class F> OrthoWork ortho_work_of(long batch, int rows, int cols) {
    const int s = std::min(rows, cols);
    OrthoWork o;
    o.ldx = row_bytes<F>(cols);
    o.sx = o.ldx * rows;
    o.lda = row_bytes<F>(s);
    o.sa = o.lda * s;
    o.part = 0;
    o.x[0] = up256(batch * norm_parts<F>(rows, cols) * 8L);
    o.x[1] = o.x[0] + up256(batch * o.sx);
    o.a = o.x[1] + up256(batch * o.sx);
    o.b = o.a + up256(batch * o.sa);
    o.diag[0] = o.b + up256(batch * o.sa);
    o.diag[1] = o.diag[0] + (__is_same(F, double) ? 0 : up256(batch * s * 4));
    o.total = o.diag[1] + (o.diag[1] - o.diag[0]);
    return o;
}
// The tile of one product of split matrices, by the time it takes: rounds of workgroups over the 256 CUs, each of them K / 32
// steps and an epilogue.  us per step and per epilogue, measured with S = 4096 and 1024 matrices: 256 (one workgroup of 8 waves
// a CU) 2.3 / 20, 192 (one of 8) 1.65 / 10, 128 (two of 4; alone on its CU) 1.4 (0.85) / 8, 64 (two of 4, four LDS stages: a
// grid that does not fill the chip waits for memory more than for the matrix cores) 0.55 (0.36) / 4.  Rounds decide: the 136
// lower 256-tiles of a 4096 x 4096 Gram matrix take as long as all 256, its 253 lower 192-tiles 0.7 of that.
// Long sums on few 64-tiles: four groups of waves on one tile, 0.30 (0.13) / 6.5 (1024 x 1024: 235 -> 210 us in all, 300 x 2000: 205 -> 187).
enum TileChoice { TILE256, TILE128, TILE64, TILE64_GROUPS, TILE192 };
TileChoice choose_tile(bool sym, int I, int J, int K, int batch) {
    struct Cost { int b; double step, step_alone, rest; };
    static const Cost t[5] = {{256, 2.3, 2.3, 20.0}, {128, 1.4, 0.85, 8.0}, {64, 0.55, 0.36, 4.0}, {64, 0.30, 0.13, 6.5}, {192, 1.65, 1.65, 10.0}};
    int best = 0;
    double least = 1e300;
    for (int c = 0; c < 5; ++c) {
        const double it = (I + t[c].b - 1) / t[c].b, jt = (J + t[c].b - 1) / t[c].b;
        const double tiles = (sym ? it * (it + 1) / 2 : it * jt) * batch, slots = t[c].b >= 192 || c == TILE64_GROUPS ? 256.0 : 512.0;
        const double step = tiles <= 256.0 ? t[c].step_alone : t[c].step;
        const double cost = ceil(tiles / slots) * (step * ((K + 31) / 32) + t[c].rest);
        if (cost < least) {
            least = cost;
            best = c;
        }
    }
    return (TileChoice)best;
}

template <int V> using Int = std::integral_constant<int, V>;

// dry: only looks whether a launch takes so many workgroups (less than 2^32 work-items)
template <class F, class O, bool LAST, bool PKC, bool QKC, bool SYM> int launch(hipStream_t st, const OrthoArgs& g, int batch, bool dry) {
#define GO(B, R, C, S, G) go(Int<B>{}, Int<R>{}, Int<C>{}, Int<S>{}, Int<G>{})
    int rc = GPX_OK;
    auto go = [&](auto tile, auto wr, auto wc, auto stages, auto groups) {
        constexpr int B = decltype(tile)::value, WR = decltype(wr)::value, WC = decltype(wc)::value, ST = decltype(stages)::value, KG = decltype(groups)::value;
        const long it = (g.I + B - 1) / B, jt = (g.J + B - 1) / B;
        const long grid = ((SYM ? it * (it + 1) / 2 : it * jt) * batch + 7) / 8 * 8;   // as many for every XCD
        constexpr int threads = WR * WC * 64 * KG;
        if (grid * threads >= 1L << 32) rc = GPX_ERR_UNSUPPORTED;
        else if (!dry) ortho_mm_kernel<F, O, LAST, B, WR, WC, ST, KG, PKC, QKC, SYM><<<(unsigned)grid, threads, 0, st>>>(g);
    };
    if constexpr (!__is_same(F, double)) {
        const TileChoice c = choose_tile(SYM, g.I, g.J, g.K, batch);
        if (c == TILE256) GO(256, 2, 4, 2, 1);
        else if (c == TILE128) GO(128, 2, 2, 2, 1);
        else if (c == TILE64) GO(64, 2, 2, 4, 1);
        else if (c == TILE64_GROUPS) GO(64, 2, 2, 2, 4);
        else GO(192, 2, 4, 2, 1);
    } else {
        // doubles: 64 x 64 tiles cost 4 % on a full chip and are three to four times as many; 32 x 32 where these are few; where those
        // are few too, four groups of waves share a sum (512 x 512: 233 -> 193 us), or 16 single waves that of a 16 x 16 tile
        // (1296 x 264: 274 -> 150, 16 x 4000: 422 -> 143)
        const long it = (g.I + 63) / 64, jt = (g.J + 63) / 64;
        const long in = (g.I + 31) / 32, jn = (g.J + 31) / 32, small = (SYM ? in * (in + 1) / 2 : in * jn) * batch;
        const long im = (g.I + 15) / 16, jm = (g.J + 15) / 16, tiny = (SYM ? im * (im + 1) / 2 : im * jm) * batch;
        if ((SYM ? it * (it + 1) / 2 : it * jt) * batch >= 192) GO(64, 2, 2, 2, 1);
        else if (tiny <= 512 && g.K >= (tiny <= 256 ? 64 : 512)) GO(16, 1, 1, 2, 16);
        else if (small <= 256 && g.K >= 128) GO(32, 2, 2, 2, 4);
        else GO(32, 2, 2, 4, 1);
    }
#undef GO
    if (!dry) HIP_TRY(hipGetLastError());
    return rc;
}

// Largest |a s + b s^3 + c s^5| for 0 <= s <= top, a little above it: the ends and the zeros of the derivative
double largest_value(double a, double b, double c, double top) {
    auto p = [&](double s) { return fabs(s * (a + s * s * (b + c * s * s))); };
    double most = p(top);
    // a + 3 b u + 5 c u^2 = 0, u = s^2
    double u[2] = {-1.0, -1.0};
    if (c != 0.0) {
        const double disc = 9.0 * b * b - 20.0 * a * c;
        if (disc >= 0.0) {
            u[0] = (-3.0 * b + sqrt(disc)) / (10.0 * c);
            u[1] = (-3.0 * b - sqrt(disc)) / (10.0 * c);
        }
    } else if (b != 0.0) {
        u[0] = -a / (3.0 * b);
    }
    for (double v : u)
        if (v > 0.0 && v < top * top) most = std::max(most, p(sqrt(v)));
    return most;
}
double largest_quadratic(double b, double c, double top) {   // largest |b u + c u^2|, 0 <= u <= top
    double most = fabs(top * (b + c * top));
    if (c != 0.0) {
        const double u = -b / (2.0 * c);
        if (u > 0.0 && u < top) most = std::max(most, fabs(u * (b + c * u)));
    }
    return most;
}
// the factors of every step's three products, powers of two of the split format included
struct OrthoFactors { double start, gram[64], square[64], linear[64], apply[64], keep[64]; };
int place(double bound);
bool ortho_factors(bool scaled, int steps, const double* coef, OrthoFactors& f) {   // false: the iterates may leave 2^100
    constexpr double slack = 1.01;   // rounding may carry a singular value past the bound of the exact iterate
    double top = slack;              // of the singular values; |G|_F >= sigma_max
    int ex = scaled ? place(top) : 0;
    f.start = ldexp(1.0, ex);
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        top = std::max(top, 0x1p-100);
        const double next = slack * largest_value(a, b, c, top);
        if (scaled && !(std::max(next, top * largest_quadratic(b, c, top * top)) < 0x1p100)) return false;
        const int ea = scaled ? place(slack * top * top) : 0;
        // (no further below a than 2^-20: a X passes through accumulators in the square factor's scale)
        const int eb = scaled ? place(slack * std::max(largest_quadratic(b, c, top * top), fabs(a) * 0x1p-20)) : 0;
        const int en = scaled && k + 1 < steps ? place(next) : 0;
        f.gram[k] = ldexp(1.0, ea - 2 * ex);
        f.square[k] = ldexp(c, eb - 2 * ea);
        f.linear[k] = ldexp(b, eb - ea);
        f.apply[k] = ldexp(1.0, en - ex - eb);
        // a X is added to the finished sum: inside it, as a I in the square factor, every later addition of the sum would round
        // relative to a X (first steps, 4096 x 4096: error 4.2e-7 instead of 4e-8)
        f.keep[k] = ldexp(a, en - ex);
        top = next;
        ex = en;
    }
    return true;
}
// exponent of the power of two that places values of at most `bound` below 2^15
int place(double bound) { return bound > 0.0 ? 14 - std::ilogb(bound) : 14; }

// ---- small matrices: all steps in one workgroup -------------------------------------------------------------------------
// X (short side S as rows, padded to 32; long side L padded to 32) and A stay in LDS in the split format, rows 32 bytes longer
// than their values so that neighbouring rows do not share banks.  Per step: A = X X^T, one 16 x 16 tile per wave and turn;
// A <- b A + c A A from registers once every wave has read A; X <- a X + A X by blocks of 16 columns, each read whole into
// registers by the one wave that overwrites it.  What bounds it is latency: 15 short products behind barriers.
constexpr int kSmallWaves = 16, kSmallSide = 128, kSmallLds = 160 * 1024 - 1536;
struct OrthoSmallArgs {
    long ldg, stride_g, ldo, stride_o;   // elements
    int rows, cols, steps;
    double eps, scale;
    float gram[64], square[64], linear[64], apply[64], keep[64];   // factors of every step, powers of two included
};
constexpr int small_row(int values) { return values * 4 + 32; }
// Bytes of LDS (two: enough for a second X and A), or 0 where the matrix does not fit or one workgroup would need longer than the many of the general path:
// 0.9 us + 1.5 us per 10^6 of S S (2 L + S) a step (128 x 128: 10 us) against 13 us there, most of it three launches.
long small_lds(int rows, int cols, bool& two) {
    const long s = (std::min(rows, cols) + 31) / 32 * 32, l = (std::max(rows, cols) + 31) / 32 * 32;
    if (s > kSmallSide || l > (1 << 16) || s * s * (2 * l + s) > 6500000) return 0;
    const long one = s * (small_row((int)l) + small_row((int)s)), more = s == 32 ? kSmallWaves * 3 * 1024 : 0;
    two = 2 * one + more <= kSmallLds;
    return two ? 2 * one + more : one + more <= kSmallLds ? one + more : 0;
}
__device__ __forceinline__ mm::v4i small_frag_kc(const char* m, int ld, int row0, int k32, int lo, int lane) {
    return *reinterpret_cast<const mm::v4i*>(m + (row0 + (lane & 15)) * ld + k32 * 128 + lo * 64 + (lane >> 4) * 16);
}
__device__ __forceinline__ mm::v4i small_frag_strided(const char* m, int ld, int col0, int k32, int lo, int lane) {
    const int r = lane & 15, q = lane >> 4;
    const char* p = m + (k32 * 32 + 8 * q + (r >> 2)) * ld + (col0 >> 5) * 128 + (col0 & 16) * 2 + lo * 64 + (r & 3) * 8;
    typedef __attribute__((address_space(3))) mm::v4s lds4;
    union { mm::v4s h[2]; mm::v4i v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * ld));
    return u.v;
}
// the three products of the split format in accumulators of their own: no matrix instruction waits for the one before it
struct SmallAcc {
    mm::v4f a = {}, b = {}, c = {};
    __device__ __forceinline__ void add(mm::v4i qh, mm::v4i ql, mm::v4i ph, mm::v4i pl) {
        a = mm::mma<_Float16>(ql, ph, a);
        b = mm::mma<_Float16>(qh, pl, b);
        c = mm::mma<_Float16>(qh, ph, c);
    }
    __device__ __forceinline__ mm::v4f sum() const { return (a + b) + c; }
};
__device__ __forceinline__ void small_store4(char* row, int j, mm::v4f v) {   // j a multiple of 4
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    v4h h, l;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        _Float16 a, b;
        split(v[x], a, b);
        h[x] = a;
        l[x] = b;
    }
    char* p = row + (j >> 5) * 128 + (j & 31) * 2;
    *reinterpret_cast<v4h*>(p) = h;
    *reinterpret_cast<v4h*>(p + 64) = l;
}

__device__ __forceinline__ mm::v4f small_load4(const char* row, int j) {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    const char* p = row + (j >> 5) * 128 + (j & 31) * 2;
    const v4h h = *reinterpret_cast<const v4h*>(p), l = *reinterpret_cast<const v4h*>(p + 64);
    mm::v4f v;
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = (float)h[x] + (float)l[x];
    return v;
}

// the 16 x 16 tile c of a symmetric matrix into both of its places, its diagonal into diag
__device__ __forceinline__ void small_store_both(char* to, int ld, float* diag, int i0, int j0, mm::v4f c, int lane) {
    const int r = lane & 15, q = lane >> 4;
    if (i0 == j0) {
#pragma unroll
        for (int y = 0; y < 4; ++y)
            if (r == 4 * q + y) {
                diag[i0 + r] = c[y];
                c[y] = 0.0f;
            }
    }
    small_store4(to + (i0 + r) * ld, j0 + 4 * q, c);
    if (i0 != j0) {
#pragma unroll
        for (int y = 0; y < 4; ++y) Iterate<mm::Split>::store(to + (j0 + 4 * q + y) * ld, i0 + r, c[y]);
    }
}
// tile of square A A + linear A, `a` its tile of A.  A = A0 + diag(d): A A = A0 A0 + (d_i + d_j) A0, on the diagonal A0 A0 + d^2.
template <int NB> __device__ __forceinline__ mm::v4f small_square(const char* A, int ld, const float* d, int i0, int j0, mm::v4f a, float square, float linear, int lane) {
    const int r = lane & 15, q = lane >> 4;
    SmallAcc c;
#pragma unroll
    for (int k = 0; k < NB; ++k)
        c.add(small_frag_kc(A, ld, j0, k, 0, lane), small_frag_kc(A, ld, j0, k, 1, lane), small_frag_kc(A, ld, i0, k, 0, lane), small_frag_kc(A, ld, i0, k, 1, lane));
    const float di = d[i0 + r];
    const mm::v4f dj = *reinterpret_cast<const mm::v4f*>(d + j0 + 4 * q), sum = c.sum();
    mm::v4f b;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
        const float of_d = i0 + r == j0 + 4 * q + y ? di : di + dj[y];
        b[y] = sum[y] * square + a[y] * (linear + square * of_d);
    }
    return b;
}

// NB: blocks of 32 of the short side.  TWO: room for a second X and A, so that nobody waits before writing, and two waves can
// share a block of 16 columns (128 x 50: 21.6 -> 20.9 us, 300 of 128 x 128: 153 -> 126).
template <class T, int NB, bool TWO>
__global__ __launch_bounds__(kSmallWaves * 64) void ortho_small_kernel(const T* G, T* O, const OrthoSmallArgs g) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ double ws[kSmallWaves];
    __shared__ __attribute__((aligned(16))) float da[kSmallSide], db[kSmallSide];   // the diagonals, which A and B hold zeros for
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const bool tall = g.rows > g.cols;
    const int S = tall ? g.cols : g.rows, L = tall ? g.rows : g.cols;
    constexpr int Sp = NB * 32, NT = NB * 2, TILES = NT * (NT + 1) / 2, TURNS = (TILES + kSmallWaves - 1) / kSmallWaves;
    const int Lp = (L + 31) / 32 * 32;
    const int ldx = small_row(Lp), lda = small_row(Sp);
    char* X = lds;
    char* A = lds + (TWO ? 2L : 1L) * Sp * ldx;
    char* X2 = TWO ? lds + (long)Sp * ldx : X;
    char* B = TWO ? A + Sp * lda : A;
    G += blockIdx.x * g.stride_g;
    O += blockIdx.x * g.stride_o;
    double s = 0.0;
    T first[8];   // this thread's first run stays in registers
    bool held = false;
    each_run(g.rows, g.cols, threadIdx.x, kSmallWaves * 64, [&](int row, int c) {
        T v[8];
        load_run(G + row * g.ldg + c, g.cols - c, v);
#pragma unroll
        for (int x = 0; x < 8; ++x) s = fma(as_double(v[x]), as_double(v[x]), s);
        if (!held) {
#pragma unroll
            for (int x = 0; x < 8; ++x) first[x] = v[x];
            held = true;
        }
    });
#pragma unroll
    for (int d = 32; d; d /= 2) s += __shfl_xor(s, d, 64);
    if (lane == 0) ws[wave] = s;
    for (int e = threadIdx.x; e < (TWO ? 2 : 1) * Sp * ldx / 16; e += kSmallWaves * 64) reinterpret_cast<mm::v4i*>(X)[e] = mm::v4i{0, 0, 0, 0};
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) s += ws[w];
    const Factor by(g.scale / (sqrt(s) + g.eps));
    each_run(g.rows, g.cols, threadIdx.x, kSmallWaves * 64, [&](int row, int c) {
        T v[8];
        if (held) {
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = first[x];
            held = false;
        } else {
            load_run(G + row * g.ldg + c, g.cols - c, v);
        }
        if (tall) {
#pragma unroll
            for (int x = 0; x < 8; ++x)
                if (c + x < g.cols) Iterate<mm::Split>::store(X + (c + x) * ldx, row, by.times((float)v[x]));
        } else {
            float w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = by.times((float)v[x]);
            Iterate<mm::Split>::store8(X + row * ldx, c, w);
        }
    });
    __syncthreads();
    const int kx = Lp / 32;
    // this wave's tiles of the lower triangle
    int ti[TURNS], tj[TURNS];
#pragma unroll
    for (int x = 0; x < TURNS; ++x) {
        int t = wave + kSmallWaves * x, i = 0;
        while (t > i) t -= ++i;
        ti[x] = i * 16;
        tj[x] = t * 16;
    }
    auto store_both = [&](char* to, float* diag, int i0, int j0, mm::v4f c) { small_store_both(to, lda, diag, i0, j0, c, lane); };
    for (int step = 0; step < g.steps; ++step) {
        mm::v4f a[TURNS], b[TURNS];   // this wave's tiles of A and of the square factor
        if constexpr (NB == 1) {
            // three tiles: every wave takes each sixteenth block of k for all of them, the sums meet in LDS behind A
            mm::v4f* meet = reinterpret_cast<mm::v4f*>(A + (TWO ? 2 : 1) * Sp * lda);
            SmallAcc c[3];
            for (int k = wave; k < kx; k += kSmallWaves) {
                mm::v4i f[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo) f[h][lo] = small_frag_kc(X, ldx, 16 * h, k, lo, lane);
                c[0].add(f[0][0], f[0][1], f[0][0], f[0][1]);
                c[1].add(f[0][0], f[0][1], f[1][0], f[1][1]);
                c[2].add(f[1][0], f[1][1], f[1][0], f[1][1]);
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) meet[(wave * 3 + x) * 64 + lane] = c[x].sum();
            __syncthreads();
            if (wave < 3) {
                mm::v4f c = meet[wave * 64 + lane];
#pragma unroll
                for (int w = 1; w < kSmallWaves; ++w) c += meet[(w * 3 + wave) * 64 + lane];
                a[0] = c * g.gram[step];
                store_both(A, da, ti[0], tj[0], a[0]);
            }
        } else {
#pragma unroll
            for (int x = 0; x < TURNS; ++x) {
                if (wave + kSmallWaves * x >= TILES) break;
                SmallAcc c;
                for (int k = 0; k < kx; ++k)
                    c.add(small_frag_kc(X, ldx, tj[x], k, 0, lane), small_frag_kc(X, ldx, tj[x], k, 1, lane), small_frag_kc(X, ldx, ti[x], k, 0, lane),
                          small_frag_kc(X, ldx, ti[x], k, 1, lane));
                a[x] = c.sum() * g.gram[step];
                store_both(A, da, ti[x], tj[x], a[x]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            if (wave + kSmallWaves * x >= TILES) break;
            b[x] = small_square<NB>(A, lda, da, ti[x], tj[x], a[x], g.square[step], g.linear[step], lane);
            if (TWO) store_both(B, db, ti[x], tj[x], b[x]);
        }
        __syncthreads();
        if constexpr (!TWO) {
#pragma unroll
            for (int x = 0; x < TURNS; ++x) {
                if (wave + kSmallWaves * x >= TILES) break;
                store_both(B, db, ti[x], tj[x], b[x]);
            }
            __syncthreads();
        }
        const bool last = step + 1 == g.steps;
        mm::v4i next[NB][2];   // the block of the next turn is read while this one is multiplied
        auto read_block = [&](int j0) {
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                next[k][0] = small_frag_strided(X, ldx, j0, k, 0, lane);
                next[k][1] = small_frag_strided(X, ldx, j0, k, 1, lane);
            }
        };
        // two waves a block of columns, half of its rows each, where there are no more than 8 blocks
        const bool halves = TWO && Lp <= 128;
        const int first_block = halves ? wave >> 1 : wave, blocks = halves ? kSmallWaves / 2 : kSmallWaves;
        const int from = halves && (wave & 1) ? Sp / 2 : 0, to = halves && !(wave & 1) ? Sp / 2 : Sp;
        if (first_block * 16 < Lp) read_block(first_block * 16);
        for (int j0 = first_block * 16; j0 < Lp; j0 += blocks * 16) {
            mm::v4i qf[NB][2];
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                qf[k][0] = next[k][0];
                qf[k][1] = next[k][1];
            }
            if (j0 + blocks * 16 < Lp) read_block(j0 + blocks * 16);
#pragma unroll 2
            for (int i0 = from; i0 < to; i0 += 16) {
                SmallAcc acc;
#pragma unroll
                for (int k = 0; k < NB; ++k)
                    acc.add(qf[k][0], qf[k][1], small_frag_kc(B, lda, i0, k, 0, lane), small_frag_kc(B, lda, i0, k, 1, lane));
                const mm::v4f c = acc.sum() * g.apply[step] + small_load4(X + (i0 + r) * ldx, j0 + 4 * q) * (g.keep[step] + g.apply[step] * db[i0 + r]);
                if (last) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int i = i0 + r, j = j0 + 4 * q + y;
                        if (i < S && j < L) O[tall ? j * g.ldo + i : i * g.ldo + j] = (T)c[y];
                    }
                } else {
                    small_store4(X2 + (i0 + r) * ldx, j0 + 4 * q, c);
                }
            }
        }
        __syncthreads();
        if (TWO) {
            char* t = X;
            X = X2;
            X2 = t;
        }
    }
}

// ---- short sides up to 128 that one workgroup cannot hold: one launch a step ----------------------------------------------
// Every workgroup keeps LC columns of X, and the launch of a step does, for them: A from the sums of all chunks (in one order),
// the square factor (again in every workgroup: short products), X <- a X + (b A + c A A) X, and the chunk's part of the next X X^T.
// Launches and their short dependent products bound it: 3 a step on the general path.  f32: 50 x 1203 (8, three steps) 70 -> 38 us,
// 128 x 4096 237 -> 126, 16 x 2000 117 -> 34, 128 x 168 95 -> 75.
struct OrthoChunkArgs {
    long ldg, stride_g, ldo, stride_o;   // elements
    int rows, cols, chunks, parts;
    const double* part;                  // of the norm
    double eps, scale;
    char* X;                             // LDS images of the chunks
    const mm::v4f* in; mm::v4f* out;     // parts of X X^T: tiles of 16 x 16 as accumulators
    float gram, square, linear, apply, keep;
    bool first, last;                    // first: X_0 and its part only
};
template <int NB> struct Chunk {
    static constexpr int LC = NB <= 2 ? 256 : 128, S = NB * 32, NT = NB * 2, TILES = NT * (NT + 1) / 2;
    static constexpr int LDX = LC * 4 + 32, LDA = S * 4 + 32, IMAGE = S * LDX, LDS = IMAGE + S * LDA;
};
template <class T, int NB>
__global__ __launch_bounds__(kSmallWaves * 64) void ortho_chunk_kernel(const T* G, T* O, const OrthoChunkArgs g) {
    typedef Chunk<NB> K;
    constexpr int LC = K::LC, Sp = K::S, TILES = K::TILES, LDX = K::LDX, LDA = K::LDA, TURNS = (TILES + kSmallWaves - 1) / kSmallWaves;
    extern __shared__ __attribute__((aligned(128))) char lds[];
    __shared__ __attribute__((aligned(16))) float da[Sp], db[Sp];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int mat = blockIdx.x / g.chunks, c0 = blockIdx.x % g.chunks * LC;
    const bool tall = g.rows > g.cols;
    const int S = tall ? g.cols : g.rows, L = tall ? g.rows : g.cols, wide = min(L - c0, LC);
    char* X = lds;
    char* A = lds + K::IMAGE;
    mm::v4i* image = reinterpret_cast<mm::v4i*>(g.X + blockIdx.x * (long)K::IMAGE);
    int ti[TURNS], tj[TURNS];   // this wave's tiles of the lower triangle
#pragma unroll
    for (int x = 0; x < TURNS; ++x) {
        int t = wave + kSmallWaves * x, i = 0;
        while (t > i) t -= ++i;
        ti[x] = i * 16;
        tj[x] = t * 16;
    }
    if (g.first) {
        const Factor by(g.scale / (norm_of<T>(g.part + mat * (long)g.parts, g.parts) + g.eps));
        for (int e = threadIdx.x; e < K::IMAGE / 16; e += kSmallWaves * 64) reinterpret_cast<mm::v4i*>(X)[e] = mm::v4i{0, 0, 0, 0};
        __syncthreads();
        const T* from = G + mat * g.stride_g + (tall ? c0 * g.ldg : c0);
        const int have = tall ? g.cols : wide;   // columns
        each_run(tall ? wide : g.rows, have, threadIdx.x, kSmallWaves * 64, [&](int row, int c) {
            T v[8];
            load_run(from + row * g.ldg + c, have - c, v);
            if (tall) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (c + x < have) Iterate<mm::Split>::store(X + (c + x) * LDX, row, by.times((float)v[x]));
            } else {
                float w[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) w[x] = by.times((float)v[x]);
                Iterate<mm::Split>::store8(X + row * LDX, c, w);
            }
        });
    } else {
        for (int e = threadIdx.x; e < K::IMAGE / 16; e += kSmallWaves * 64) reinterpret_cast<mm::v4i*>(X)[e] = image[e];
        mm::v4f a[TURNS], b[TURNS];
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            const int t = wave + kSmallWaves * x;
            if (t >= TILES) break;
            a[x] = mm::v4f{};
            const mm::v4f* in = g.in + ((long)mat * g.chunks * TILES + t) * 64 + lane;
#pragma unroll 8
            for (int c = 0; c < g.chunks; ++c) a[x] += in[(long)c * TILES * 64];
            a[x] *= g.gram;
            small_store_both(A, LDA, da, ti[x], tj[x], a[x], lane);
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            if (wave + kSmallWaves * x >= TILES) break;
            b[x] = small_square<NB>(A, LDA, da, ti[x], tj[x], a[x], g.square, g.linear, lane);
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            if (wave + kSmallWaves * x >= TILES) break;
            small_store_both(A, LDA, db, ti[x], tj[x], b[x], lane);
        }
        // LC / 16 blocks of 16 columns: a wave each, or two with half of the rows each
        constexpr bool HALVES = LC / 16 < kSmallWaves;
        const int j0 = (HALVES ? wave >> 1 : wave) * 16, from = HALVES && (wave & 1) ? Sp / 2 : 0, to = HALVES && !(wave & 1) ? Sp / 2 : Sp;
        mm::v4i qf[NB][2];
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            qf[k][0] = small_frag_strided(X, LDX, j0, k, 0, lane);
            qf[k][1] = small_frag_strided(X, LDX, j0, k, 1, lane);
        }
        __syncthreads();   // the square factor is there, and every block is in registers
#pragma unroll 2
        for (int i0 = from; i0 < to; i0 += 16) {
            SmallAcc acc;
#pragma unroll
            for (int k = 0; k < NB; ++k) acc.add(qf[k][0], qf[k][1], small_frag_kc(A, LDA, i0, k, 0, lane), small_frag_kc(A, LDA, i0, k, 1, lane));
            const mm::v4f c = acc.sum() * g.apply + small_load4(X + (i0 + r) * LDX, j0 + 4 * q) * (g.keep + g.apply * db[i0 + r]);
            if (g.last) {
                T* o = O + mat * g.stride_o;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int i = i0 + r, j = c0 + j0 + 4 * q + y;
                    if (i < S && j < L) o[tall ? j * g.ldo + i : i * g.ldo + j] = (T)c[y];
                }
            } else {
                small_store4(X + (i0 + r) * LDX, j0 + 4 * q, c);
            }
        }
        if (g.last) return;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < TURNS; ++x) {
        const int t = wave + kSmallWaves * x;
        if (t >= TILES) break;
        SmallAcc c;
#pragma unroll
        for (int k = 0; k < LC / 32; ++k)
            c.add(small_frag_kc(X, LDX, tj[x], k, 0, lane), small_frag_kc(X, LDX, tj[x], k, 1, lane), small_frag_kc(X, LDX, ti[x], k, 0, lane),
                  small_frag_kc(X, LDX, ti[x], k, 1, lane));
        g.out[((long)blockIdx.x * TILES + t) * 64 + lane] = c.sum();
    }
    for (int e = threadIdx.x; e < K::IMAGE / 16; e += kSmallWaves * 64) image[e] = reinterpret_cast<mm::v4i*>(X)[e];
}

struct ChunkPlan { int chunks; long images, sums, total; };   // chunks 0: not this way.  bytes: images of X, one set of sums, workspace
template <int NB> ChunkPlan chunk_plan_of(long batch, int l, long part_bytes) {
    typedef Chunk<NB> K;
    const long chunks = (l + K::LC - 1) / K::LC;
    // Two rounds of workgroups pay for short sides up to 64 (f32 24 x 50 x 4000: 250 -> 140 us), not for longer ones (24 x 128 x 2048:
    // 212 -> 242); every workgroup reads all chunks' sums (1 x 128 x 8192, 2.4 MB: 371 -> 173).
    if (chunks * batch > (NB <= 2 ? 512 : 256) || chunks * K::TILES > 2400) return {0, 0, 0, 0};
    const long images = up256(batch * chunks * K::IMAGE), sums = batch * chunks * K::TILES * 1024L;
    return {(int)chunks, images, sums, part_bytes + images + 2 * sums};
}
ChunkPlan chunk_plan(long batch, int rows, int cols) {
    const int s = std::min(rows, cols), l = std::max(rows, cols);
    bool two;
    if (s > kSmallSide || small_lds(rows, cols, two)) return {0, 0, 0, 0};
    const long part = ortho_work_of<mm::Split>(batch, rows, cols).x[0];
    switch ((s + 31) / 32) {
        case 1: return chunk_plan_of<1>(batch, l, part);
        case 2: return chunk_plan_of<2>(batch, l, part);
        case 3: return chunk_plan_of<3>(batch, l, part);
        default: return chunk_plan_of<4>(batch, l, part);
    }
}

// bytes of workspace of the path that is taken
long ortho_work(int dtype, long batch, int rows, int cols) {
    if (dtype == GPX_F64) return ortho_work_of<double>(batch, rows, cols).total;
    const OrthoWork o = ortho_work_of<mm::Split>(batch, rows, cols);
    bool two;
    if (small_lds(rows, cols, two)) return o.x[0];   // the norms, for no steps at all
    const ChunkPlan plan = chunk_plan(batch, rows, cols);
    return plan.chunks ? plan.total : o.total;
}

// rows x cols row-major (the column-major cols x rows of the C interface)
template <class T, class F>
int ortho_typed(hipStream_t st, int batch, int rows, int cols, const T* G, long ldg, long stride_g, int steps, const double* coef, double eps,
                T* O, long ldo, long stride_o, char* work) {
    OrthoFactors f;
    if (!ortho_factors(!__is_same(F, double), steps, coef, f)) return GPX_ERR_ARG;
    if constexpr (!__is_same(F, double)) {
        bool two = false;
        const long bytes = small_lds(rows, cols, two);
        if (steps > 0 && bytes) {
            OrthoSmallArgs g = {ldg, stride_g, ldo, stride_o, rows, cols, steps, eps, f.start, {}, {}, {}, {}, {}};
            for (int k = 0; k < steps; ++k) {
                g.gram[k] = (float)f.gram[k];
                g.square[k] = (float)f.square[k];
                g.linear[k] = (float)f.linear[k];
                g.apply[k] = (float)f.apply[k];
                g.keep[k] = (float)f.keep[k];
            }
            const int nb = (std::min(rows, cols) + 31) / 32;
            auto go = [&](auto blocks) {
                constexpr int NB = decltype(blocks)::value;
                if (two) ortho_small_kernel<T, NB, true><<<batch, kSmallWaves * 64, (unsigned)bytes, st>>>(G, O, g);
                else ortho_small_kernel<T, NB, false><<<batch, kSmallWaves * 64, (unsigned)bytes, st>>>(G, O, g);
            };
            if (nb == 1) go(Int<1>{});
            else if (nb == 2) go(Int<2>{});
            else if (nb == 3) go(Int<3>{});
            else go(Int<4>{});
            HIP_TRY(hipGetLastError());
            return GPX_OK;
        }
    }
    const OrthoWork o = ortho_work_of<F>(batch, rows, cols);
    double* part = reinterpret_cast<double*>(work + o.part);
    const long runs = norm_runs<F>(rows, cols);
    const int parts = norm_parts<F>(rows, cols);
    char* x[2] = {work + o.x[0], work + o.x[1]};
    char *a = work + o.a, *b = work + o.b;
    float *da = reinterpret_cast<float*>(work + o.diag[0]), *db = reinterpret_cast<float*>(work + o.diag[1]);
    const bool tall = rows > cols;
    const int s = std::min(rows, cols), l = std::max(rows, cols);
    auto step = [&](int k, bool dry) -> int {
        char *from = x[k & 1], *to = x[~k & 1];
        const OrthoArgs gram = {from, from, from, a, o.ldx, o.ldx, 0, o.lda, o.sx, o.sx, 0, o.sa, s, s, l, batch, f.gram[k], 0.0, nullptr, da};
        int rc = tall ? launch<F, F, false, false, false, true>(st, gram, batch, dry) : launch<F, F, false, true, true, true>(st, gram, batch, dry);
        if (rc) return rc;
        const OrthoArgs poly = {a, a, a, b, o.lda, o.lda, o.lda, o.lda, o.sa, o.sa, o.sa, o.sa, s, s, s, batch,
                                f.square[k], f.linear[k], da, db};
        if ((rc = launch<F, F, false, true, true, true>(st, poly, batch, dry))) return rc;
        const bool last = k + 1 == steps;
        const long ldd = last ? ldo * (long)sizeof(T) : o.ldx, sd = last ? stride_o * (long)sizeof(T) : o.sx;
        char* d = last ? reinterpret_cast<char*>(O) : to;
        const OrthoArgs apply = tall ? OrthoArgs{from, b, from, d, o.ldx, o.lda, o.ldx, ldd, o.sx, o.sa, o.sx, sd, rows, cols, s, batch, f.apply[k], f.keep[k], db, nullptr}
                                     : OrthoArgs{b, from, from, d, o.lda, o.ldx, o.ldx, ldd, o.sa, o.sx, o.sx, sd, rows, cols, s, batch, f.apply[k], f.keep[k], db, nullptr};
        if (tall) rc = last ? launch<F, T, true, true, true, false>(st, apply, batch, dry) : launch<F, F, false, true, true, false>(st, apply, batch, dry);
        else rc = last ? launch<F, T, true, true, false, false>(st, apply, batch, dry) : launch<F, F, false, true, false, false>(st, apply, batch, dry);
        return rc;
    };
    const ChunkPlan plan = __is_same(F, double) ? ChunkPlan{} : chunk_plan(batch, rows, cols);
    if (steps > 0 && !plan.chunks)
        if (const int rc = step(0, true)) return rc;
    ortho_norm_kernel<T><<<dim3(parts, batch), 256, 0, st>>>(G, ldg, stride_g, rows, cols, part);
    HIP_TRY(hipGetLastError());
    const dim3 grid((unsigned)std::min<long>((runs + 255) / 256, 2048), (unsigned)batch);
    if constexpr (!__is_same(F, double)) {
        if (steps > 0 && plan.chunks) {
            char* images = work + o.x[0];
            mm::v4f* sums[2] = {reinterpret_cast<mm::v4f*>(images + plan.images), reinterpret_cast<mm::v4f*>(images + plan.images + plan.sums)};
            OrthoChunkArgs g = {ldg, stride_g, ldo, stride_o, rows, cols, plan.chunks, parts, part, eps, f.start, images};
            auto go = [&](auto blocks) {
                constexpr int NB = decltype(blocks)::value;
                for (int k = 0; k <= steps; ++k) {
                    g.in = sums[~k & 1];
                    g.out = sums[k & 1];
                    g.first = k == 0;
                    g.last = k == steps;
                    if (k > 0) {
                        g.gram = (float)f.gram[k - 1];
                        g.square = (float)f.square[k - 1];
                        g.linear = (float)f.linear[k - 1];
                        g.apply = (float)f.apply[k - 1];
                        g.keep = (float)f.keep[k - 1];
                    }
                    ortho_chunk_kernel<T, NB><<<batch * plan.chunks, kSmallWaves * 64, Chunk<NB>::LDS, st>>>(G, O, g);
                }
            };
            const int nb = (std::min(rows, cols) + 31) / 32;
            if (nb == 1) go(Int<1>{});
            else if (nb == 2) go(Int<2>{});
            else if (nb == 3) go(Int<3>{});
            else go(Int<4>{});
            HIP_TRY(hipGetLastError());
            return GPX_OK;
        }
    }
    if (steps == 0) {
        ortho_normalize_kernel<T><<<grid, 256, 0, st>>>(G, ldg, stride_g, rows, cols, part, parts, eps, O, ldo, stride_o);
        HIP_TRY(hipGetLastError());
        return GPX_OK;
    }
    ortho_scale_kernel<T, F><<<grid, 256, 0, st>>>(G, ldg, stride_g, rows, cols, padded<F>(cols), part, parts, eps, f.start, x[0], o.ldx, o.sx);
    HIP_TRY(hipGetLastError());
    for (int k = 0; k < steps; ++k)
        if (const int rc = step(k, false)) return rc;
    return GPX_OK;
}

constexpr int kMaxSteps = 64;
constexpr long kMaxSide = 1L << 20;
constexpr int64_t kMaxLd = 1L << 32, kMaxStride = 1L << 48;   // elements: in bytes they pass no 63 bits
constexpr double kLeastEps = 1e-300;                          // 2^15 / eps stays finite: a zero matrix gives zeros
const double kQuintic[3] = {3.4445, -4.7750, 2.0315};

bool sizes_ok(int dtype, int64_t batch, int64_t M, int64_t N) {
    return dtype >= GPX_F64 && dtype <= GPX_F16 && batch >= 0 && batch <= 65535 && M >= 0 && N >= 0 && M <= kMaxSide && N <= kMaxSide;
}

// 16-bit matrices with a side above 65536: 2 of 70000 x 1 in bf16 ended in a GPU fault, in kernels for one plane of 11 bits that are
// no longer here, and its cause was not found.  (f32 and f64 took that size.)
bool switched_off(int dtype, int64_t M, int64_t N) { return (dtype == GPX_BF16 || dtype == GPX_F16) && std::max(M, N) > 65536; }

}  // namespace

extern "C" int gpx_orthogonalize_work(int dtype, int64_t batch, int64_t M, int64_t N, int64_t* work_bytes) {
    if (!work_bytes || !sizes_ok(dtype, batch, M, N)) return GPX_ERR_ARG;
    if (batch && M && N && switched_off(dtype, M, N)) return GPX_ERR_ARG;
    *work_bytes = batch && M && N ? ortho_work(dtype, batch, (int)N, (int)M) : 0;
    return GPX_OK;
}

extern "C" int gpx_orthogonalize(int dtype, int64_t batch, int64_t M, int64_t N, const void* G, int64_t ldg, int64_t stride_g, int steps,
                                 const double* coef, double eps, void* O, int64_t ldo, int64_t stride_o, void* work, int64_t work_bytes,
                                 void* hip_stream) {
    if (!sizes_ok(dtype, batch, M, N) || steps < 0 || steps > kMaxSteps || !(eps >= kLeastEps) || !std::isfinite(eps)) return GPX_ERR_ARG;
    if (ldg < M || ldo < M || stride_g < 0 || stride_o < 0) return GPX_ERR_ARG;
    if (ldg > kMaxLd || ldo > kMaxLd || stride_g > kMaxStride || stride_o > kMaxStride) return GPX_ERR_ARG;
    const uintptr_t e = dtype == GPX_F64 ? 8 : dtype == GPX_F32 ? 4 : 2;
    const int64_t el = (int64_t)e;
    const ByteRows in = {G, batch, stride_g * el, N, ldg * el, M * el}, out = {O, batch, stride_o * el, N, ldo * el, M * el};
    if (!gpx_reaches(in) || !gpx_reaches(out)) return GPX_ERR_ARG;
    if (batch == 0 || M == 0 || N == 0) return GPX_OK;
    if (switched_off(dtype, M, N)) return GPX_ERR_ARG;
    if (batch > 1 && stride_o < (N - 1) * ldo + M) return GPX_ERR_ARG;   // results of two matrices would overlap
    if (!G || !O || !work) return GPX_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(G) % e || reinterpret_cast<uintptr_t>(O) % e || reinterpret_cast<uintptr_t>(work) % 16) return GPX_ERR_ARG;
    const int64_t need = ortho_work(dtype, batch, (int)N, (int)M);
    if (work_bytes < need) return GPX_ERR_ARG;
    const ByteRows room = {work, 1, 0, 1, 0, need};
    const bool in_place = G == O && (N == 1 || ldg == ldo) && (batch == 1 || stride_g == stride_o);
    if ((!in_place && gpx_share_bytes(in, out)) || gpx_share_bytes(room, in) || gpx_share_bytes(room, out)) return GPX_ERR_ARG;
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
            return ortho_typed<double, double>(st, b, r, c, static_cast<const double*>(G), ldg, stride_g, steps, table, eps,
                                               static_cast<double*>(O), ldo, stride_o, w);
        case GPX_F32:
            return ortho_typed<float, mm::Split>(st, b, r, c, static_cast<const float*>(G), ldg, stride_g, steps, table, eps,
                                             static_cast<float*>(O), ldo, stride_o, w);
        case GPX_BF16:
            return ortho_typed<__bf16, mm::Split>(st, b, r, c, static_cast<const __bf16*>(G), ldg, stride_g, steps, table, eps,
                                              static_cast<__bf16*>(O), ldo, stride_o, w);
        default:
            return ortho_typed<_Float16, mm::Split>(st, b, r, c, static_cast<const _Float16*>(G), ldg, stride_g, steps, table, eps,
                                                static_cast<_Float16*>(O), ldo, stride_o, w);
    }
}
