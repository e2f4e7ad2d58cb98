// grouped.hip — matrix products grouped by expert with ragged numbers of rows, and the gradient of their weights.
//
// gpx_grouped_gemm: rows t of group g (offsets[g] <= t < offsets[g+1]):  y_t = alpha W_g x_t + beta y_t.
//   D(i, j) with i = row, j = output column: P = X (k contiguous), Q = W_g in either layout, so the input gradient
//   dX = dY W is the same call with the other layout flag.
// gpx_grouped_gemm_dw: C_g = alpha sum_{t in g} dy_t x_t^T + beta C_g: P = dY, Q = X, both with k (= rows t) strided.
//
// The offsets live on the device: the host never waits for them.  Every kernel clamps them to [0, T] and reads a
// decreasing pair as an empty group, so no value of theirs leads outside the buffers.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "mm_tile.h"
#include "../../include/gpx.h"

namespace {

struct GroupedArgs {
    const char* X; const char* W; char* Y;
    const int64_t* offsets;
    long ldx, ldw, stride_w, ldy;   // bytes
    long T;
    int groups, N, K;
    double alpha, beta;
    int slots, most;   // see the two levels of tiles; 0: one
};

__device__ __forceinline__ long clamped(const int64_t* offsets, int g, long T) {
    const long o = offsets[g];
    return o < 0 ? 0 : o > T ? T : o;
}

struct RowTile { int group, rows; long row0; };   // rows of this tile; group < 0: no tile

// One wave looks at 64 groups at a time: rows of group g0 + lane, in tiles of `unit` rows, and the running sum of the tiles.
struct GroupScan {
    long lo, rows, tiles, sum;
    __device__ GroupScan(const int64_t* offsets, int groups, long T, int g0, unsigned unit) {
        const int lane = threadIdx.x & 63, g = g0 + lane;
        lo = rows = 0;
        if (g < groups) {
            lo = clamped(offsets, g, T);
            const long hi = clamped(offsets, g + 1, T);
            rows = hi > lo ? hi - lo : 0;
        }
        sum = tiles = ((unsigned)rows + unit - 1) / unit;   // T < 2^31
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const long up = __shfl_up(sum, d, 64);
            if (lane >= d) sum += up;
        }
    }
};

// row tile number t in the order of the groups; `first`: the scan of the first 64
__device__ RowTile row_tile(const GroupScan& first, const int64_t* offsets, int groups, long T, long t, unsigned unit) {
    long before = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const GroupScan s = g0 ? GroupScan(offsets, groups, T, g0, unit) : first;
        const unsigned long long past = __ballot(before + s.sum > t);
        if (past) {
            const int src = __builtin_ctzll(past);
            const long m = t - before - __shfl(s.sum - s.tiles, src, 64);   // tile within the group
            const long r = __shfl(s.rows, src, 64) - m * unit;
            RowTile out;
            out.group = __builtin_amdgcn_readfirstlane(g0 + src);
            out.rows = __builtin_amdgcn_readfirstlane((int)(r < unit ? r : unit));
            out.row0 = __shfl(s.lo, src, 64) + m * unit;
            return out;
        }
        before += __shfl(s.sum, 63, 64);
    }
    return {-1, 0, 0};
}

// The order of the tiles: row tiles in the order of the groups, ceil(rows / BM) each, cut into bands of eight; a band's tiles
// column by column.  That order is walked in chunks of CHUNK tiles, what the chip holds at a time, and since workgroups go
// round the 8 XCDs, XCD x takes the x-th eighth of every chunk: its CUs share 8 row panels and a few column panels in their L2,
// and all XCDs stay in one neighbourhood of X and W in the cache behind them.
//
// Two levels (slots > 0): what is left behind the last whole round of `slots` tiles, if it is no more than `most`, is done in
// tiles of half the rows and columns by a second launch (REST; the tiles of the first are 2 BM high then): a few large tiles
// would take the time of a whole round (bf16 4 x 2048 x 4096 x 2304: 194 -> 174 us,
// f32 5000 x 2000 x 2000: 356 -> 327).
template <int BM, int CHUNK, int HIGH = 8, bool REST = false>
__device__ RowTile find_tile(const int64_t* offsets, int groups, long T, int nt, int& col, int slots = 0, int most = 0) {
    constexpr int UNIT = REST ? 2 * BM : BM;
    const GroupScan first(offsets, groups, T, 0, UNIT);
    long total = __shfl(first.sum, 63, 64);
    for (int g0 = 64; g0 < groups; g0 += 64) total += __shfl(GroupScan(offsets, groups, T, g0, UNIT).sum, 63, 64);
    long all = total * nt, start = 0, last;
    const unsigned xcd = blockIdx.x & 7;
    if (slots) {
        const int left = (int)(all % slots);
        const bool two = left <= most && left < all;
        if (REST) {
            if (!two) return {-1, 0, 0};
            start = all - left;
        } else if (two) {
            all -= left;
        }
    }
    unsigned in_chunk;
    if (!REST) {
        start = (long)(blockIdx.x / CHUNK) * CHUNK;
        if (start >= all) return {-1, 0, 0};
        const unsigned here = (unsigned)min((long)CHUNK, all - start);
        in_chunk = here * xcd / 8 + (blockIdx.x % CHUNK >> 3);
        last = here * (xcd + 1) / 8;
    } else {   // four workgroups a tile
        const unsigned here = (unsigned)(all - start);
        in_chunk = here * xcd / 8 + (blockIdx.x >> 5);
        last = here * (xcd + 1) / 8;
    }
    if (in_chunk >= last) return {-1, 0, 0};
    const long o = start + in_chunk;
    const unsigned band = (unsigned)(o / (HIGH * nt)), in = (unsigned)(o - (long)band * HIGH * nt);
    const unsigned high = (unsigned)min((long)HIGH, total - (long)HIGH * band);
    col = __builtin_amdgcn_readfirstlane((int)(in / high));
    RowTile t = row_tile(first, offsets, groups, T, (long)HIGH * band + in % high, UNIT);
    if (REST) {
        const int down = blockIdx.x >> 4 & 1;
        col = 2 * col + (blockIdx.x >> 3 & 1);
        t.row0 += down * BM;
        t.rows = min(t.rows - down * BM, BM);
        if (t.rows <= 0) t.group = -1;
    }
    return t;
}

// p[0..R) (those j + x < N) = alpha v + beta p in the type O, R of them 16 bytes, at any alignment.  PAST: whole runs go past the
// caches (weight gradients, which nobody reads soon: 163 -> 142 us for 16 of 2816 x 2048; forward results, which somebody does,
// gain nothing).
template <class O, int R, bool PAST> __device__ __forceinline__ void put_run(char* row, int j, int N, const float (&v)[R], float alpha, float beta) {
    static_assert(R * sizeof(O) == 16, "16 bytes");
    O* p = reinterpret_cast<O*>(row) + j;
    union { O e[R]; mm::v4i w; } u;
    const bool whole = j + R <= N;
    if (beta != 0.0f) {
        if (whole) {
            __builtin_memcpy(&u.w, p, 16);
        } else {
#pragma unroll
            for (int x = 0; x < R; ++x) u.e[x] = j + x < N ? p[x] : (O)0.0f;
        }
#pragma unroll
        for (int x = 0; x < R; ++x) u.e[x] = (O)(alpha * v[x] + beta * (float)u.e[x]);
    } else {
#pragma unroll
        for (int x = 0; x < R; ++x) u.e[x] = (O)(alpha * v[x]);
    }
    if (whole) {
        // between fences: or the compiler takes what both branches store out of them, and the 16 bytes apart (165 -> 205 us for
        // 16 weight gradients of 2816 x 2048)
        asm volatile("" ::: "memory");
        typedef int v4iu __attribute__((ext_vector_type(4), aligned(1)));
        if (PAST) __builtin_nontemporal_store(u.w, reinterpret_cast<v4iu*>(p));
        else *reinterpret_cast<v4iu*>(p) = u.w;
        asm volatile("" ::: "memory");
    } else {
#pragma unroll
        for (int x = 0; x < R; ++x)
            if (j + x < N) p[x] = u.e[x];
    }
}

// the tile's result: rows x cols of it at `row0`, `ld` bytes apart
template <class O, bool PAST, class Tile>
__device__ __forceinline__ void store_tile(Tile& t, char* lds, char* row0, long ld, int rows, int cols, double alpha, double beta) {
    typedef typename Tile::one A;
    const A al = (A)alpha, be = (A)beta;
    if constexpr (Tile::SWAP) {   // 16 neighbouring lanes store 16 neighbouring columns
        if (Tile::group() != 0) return;
        t.each([&](int i, int j, const A* v, auto) {
            if (i >= rows || j >= cols) return;
            O* p = reinterpret_cast<O*>(row0 + i * ld) + j;
            *p = (O)(be != A(0) ? al * v[0] + be * (A)*p : al * v[0]);
        });
    } else {
        constexpr int R = 16 / (int)sizeof(O);
        t.template each_run<R>(lds, rows, cols, [&](int i, int j, const float (&v)[R]) { put_run<O, R, PAST>(row0 + i * ld, j, cols, v, al, be); });
    }
}

constexpr int kShortSub = 8;

template <class Tile> constexpr int tile_lds() { return Tile::SWAP || Tile::LDS > Tile::SLAB ? Tile::LDS : Tile::SLAB; }

template <class T, int BM, int BN, int WR, int WC, int ST, int KG, bool WKC, bool DIRECT, bool REST = false>
__global__ __launch_bounds__(WR * WC * 64 * KG, KG > 1 ? 4 : 2) void grouped_kernel(const GroupedArgs g) {
    typedef mm::Tile<T, BM, BN, WR, WC, true, WKC, ST, KG> Tile;
    __shared__ __attribute__((aligned(128))) char lds[tile_lds<Tile>()];
    int col = 0;
    constexpr int CHUNK = BM * BN > 128 * 128 || KG > 1 ? 256 : 512, WIDTH = REST ? 2 * BN : BN;
    const RowTile rt = find_tile<BM, CHUNK, 8, REST>(g.offsets, g.groups, g.T, (g.N + WIDTH - 1) / WIDTH, col, g.slots, g.most);
    const int n0 = col * BN, cols = min(g.N - n0, BN);
    if (rt.group < 0 || (REST && cols <= 0)) return;
    typename Tile::OpP p = {g.X + rt.row0 * g.ldx, g.ldx, rt.rows, g.K};
    typename Tile::OpQ q = {g.W + rt.group * g.stride_w + (WKC ? n0 * g.ldw : n0 * (long)sizeof(T)), g.ldw, cols, g.K};
    Tile t;
    t.clear();
    if constexpr (KG > 1) t.run_groups(lds, p, q, g.K);
    else if constexpr (DIRECT) t.run_direct(lds, p, q, g.K);
    else t.run_staged(lds, p, q, g.K);
    store_tile<T, false>(t, lds, g.Y + rt.row0 * g.ldy + n0 * (long)sizeof(T), g.ldy, rt.rows, cols, g.alpha, g.beta);
}

// Short k (at most 512 bytes of it: inputs of a few dozen dimensions) in floats and doubles, where the result is most of the
// traffic: one workgroup takes its 64 columns of W into registers for all of k (as fragments, once through LDS) and walks
// SUB tiles of 32 rows.  Per tile one wait and one barrier: the rows of the next tile arrive while this one is multiplied,
// and the stores of this one leave while the next is.  Four workgroups a CU (32 KB of LDS each): the products of one cover
// the waits of the others.  The columns of one group of rows go side by side over the chip (whole rows of the result at a
// time: 232 -> 192 us at d = 20, N = 2048 in double, 5.7 TB/s).  65536 rows, d = 50, N = 1024 in double, 12 groups: 178 us (floors: 97
// for the products, 85 for the result); as single 128-tiles 204, with W in LDS and so two workgroups a CU 193.
template <class T, bool WKC>
__global__ __launch_bounds__(256, 4) void grouped_short_kernel(const GroupedArgs g) {
    constexpr int BM = 32, BN = 64, SUB = kShortSub, MOST = 4;   // MOST: K steps
    typedef mm::Tile<T, BM, BN, 2, 2, true, WKC> Tile;
    typedef typename Tile::OpP OpP;
    typedef typename Tile::OpQ OpQ;
    constexpr int TI = Tile::TI, TJ = Tile::TJ;
    static_assert(2 * OpP::BYTES <= OpQ::BYTES, "the rows of two tiles take the place of W");
    __shared__ __attribute__((aligned(128))) char lds[MOST * OpQ::BYTES];
    int col = 0;
    const RowTile rt = find_tile<BM * SUB, 1024, 1>(g.offsets, g.groups, g.T, (g.N + BN - 1) / BN, col);
    if (rt.group < 0) return;
    const int n0 = col * BN, cols = min(g.N - n0, BN);
    const int steps = (g.K + OpP::BK - 1) / OpP::BK, last = g.K - (steps - 1) * OpP::BK;
    const int halves = last * 2 <= OpP::BK ? 1 : 2;   // of the last step
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = wave / 2 * (BM / 2), j0 = wave % 2 * (BN / 2);
    const unsigned at = (unsigned)reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)lds);
    const OpQ q = {g.W + rt.group * g.stride_w + (WKC ? n0 * g.ldw : n0 * (long)sizeof(T)), g.ldw, cols, g.K};
    for (int s = 0; s < steps; ++s) q.issue(at + s * OpQ::BYTES, q.lanes(s + 1 < steps ? OpQ::BK : last), s);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    mm::v4i w[MOST][2][TJ];
#pragma unroll
    for (int s = 0; s < MOST; ++s) {
        if (s >= steps) break;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int j = 0; j < TJ; ++j) w[s][kk][j] = mm::frag<T, BN, WKC>(lds + s * OpQ::BYTES, j0 + 16 * j, kk, lane);
    }
    const int tiles = (rt.rows + BM - 1) / BM;
    auto fetch = [&](int t) {
        const OpP p = {g.X + (rt.row0 + t * BM) * g.ldx, g.ldx, min(rt.rows - t * BM, BM), g.K};
        for (int s = 0; s < steps; ++s) p.issue(at + ((t & 1) * MOST + s) * OpP::BYTES, p.lanes(s + 1 < steps ? OpP::BK : last), s);
    };
    constexpr int STORES = TI * TJ * 4;   // of this wave, of a whole tile
    bool counted = false;                 // the stores behind the last fetch are exactly these
    const typename Tile::one alpha = (typename Tile::one)g.alpha;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // W is in every wave's registers
    fetch(0);
    if (tiles > 1) fetch(1);
    for (int t = 0; t < tiles; ++t) {
        const int rows = min(rt.rows - t * BM, BM);
        // Tile t is here.  Vector memory operations retire in order: the stores of tile t - 1 and the fetch of tile t + 1, issued
        // behind the fetch that is waited for, may stay on their way.
        if (!counted) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else if (steps == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(STORES + OpP::NL) : "memory");
        else if (steps == 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(STORES + 2 * OpP::NL) : "memory");
        else if (steps == 3) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(STORES + 3 * OpP::NL) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(STORES + 4 * OpP::NL) : "memory");
        Tile m;
        m.clear();
#pragma unroll
        for (int s = 0; s < MOST; ++s) {
            if (s >= steps) break;
            const char* sp = lds + ((t & 1) * MOST + s) * OpP::BYTES;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if (kk == 1 && s + 1 == steps && halves == 1) break;
#pragma unroll
                for (int i = 0; i < TI; ++i) {
                    const mm::v4i p = mm::frag<T, BM, true>(sp, i0 + 16 * i, kk, lane);
#pragma unroll
                    for (int j = 0; j < TJ; ++j) m.acc[i][j] = mm::mma<T>(p, w[s][kk][j], m.acc[i][j]);
                }
            }
        }
        char* y = g.Y + (rt.row0 + t * BM) * g.ldy + n0 * (long)sizeof(T);
        const bool whole = rows == BM && cols == BN && g.beta == 0.0;
        if (whole) {
            // one store instruction per element of a fragment, written out so that their number is known; past the L2, which
            // the result would only sweep
            const unsigned long long to = reinterpret_cast<unsigned long long>(y);
            unsigned long long base = (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)to) |
                                      (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(to >> 32)) << 32;
            mm::settle(base);
            m.each([=](int i, int j, const typename Tile::one* v, auto) {
                const unsigned long long at_y = base;
                const unsigned off = (unsigned)(i * g.ldy) + j * (unsigned)sizeof(T);
                const typename Tile::one o = alpha * v[0];   // (also what the matrix instruction's result has to pass before a store)
                if constexpr (sizeof(T) == 8) asm volatile("global_store_dwordx2 %0, %1, %2 nt" ::"v"(off), "v"(o), "s"(at_y) : "memory");
                else asm volatile("global_store_dword %0, %1, %2 nt" ::"v"(off), "v"(o), "s"(at_y) : "memory");
            });
        } else {
            store_tile<T, false>(m, lds, y, g.ldy, rows, cols, g.alpha, g.beta);
        }
        counted = whole && t + 2 < tiles;
        if (t + 2 < tiles) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // nobody reads tile t any more
            fetch(t + 2);
        }
    }
}

struct GroupedDwArgs {
    const char* X; const char* Z; char* C;   // Z: the gradient of the outputs
    const int64_t* offsets;
    long ldx, ldz, ldc, stride_c;   // bytes
    long T;
    int M, N;   // columns of X (contiguous in C) and of Z
    int groups;
    double alpha, beta;
    char* slabs;     // SPLIT: the sum over every part of `part_rows` rows, N x M each, in the accumulators' type
    int part_rows, parts;
};

// Up to 64 groups are taken by their rows, most first (equal ones in their order), so that what runs last on a nearly empty
// chip is short: 8 groups of 4096 to 12288 rows, m = 1024 in double: 2.13 -> 2.02 ms; 16 of 256 to 768, bf16: 174 -> 171 us.
__device__ int nth_group(const int64_t* offsets, int groups, long T, int n) {
    if (groups > 64) return n;
    const GroupScan s(offsets, groups, T, 0, 1);
    const int mine = (int)s.rows, lane = threadIdx.x & 63;
    int rank = 0;
    for (int h = 0; h < groups; ++h) {
        const int r = __builtin_amdgcn_readlane(mine, h);
        rank += r > mine || (r == mine && h < lane);
    }
    return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(lane < groups && rank == n)));
}

// SPLIT: few tiles and many rows.  The rows of every group are cut into parts, a workgroup sums one part into a slab of its own,
// and grouped_dw_join_kernel adds the slabs of a group in their order: the same bits in every run.
template <class T, class O, int B, int WR, int WC, int ST, bool DIRECT, bool SPLIT>
__global__ __launch_bounds__(WR * WC * 64, 2) void grouped_dw_kernel(const GroupedDwArgs g) {
    typedef mm::Tile<T, B, B, WR, WC, false, false, ST> Tile;
    typedef typename Tile::one A;
    __shared__ __attribute__((aligned(128))) char lds[tile_lds<Tile>()];
    const int mt = (g.M + B - 1) / B;
    const int n0 = (int)(blockIdx.x / mt) * B, m0 = (int)(blockIdx.x % mt) * B;
    long lo;
    int rows, group = 0;
    if (SPLIT) {
        const RowTile part = row_tile(GroupScan(g.offsets, g.groups, g.T, 0, g.part_rows), g.offsets, g.groups, g.T, blockIdx.y, g.part_rows);
        if (part.group < 0) return;
        lo = part.row0;
        rows = part.rows;
    } else {
        group = nth_group(g.offsets, g.groups, g.T, blockIdx.y);
        lo = clamped(g.offsets, group, g.T);
        const long hi = clamped(g.offsets, group + 1, g.T);
        rows = (int)(hi > lo ? hi - lo : 0);
    }
    typename Tile::OpP p = {g.Z + lo * g.ldz + n0 * (long)sizeof(T), g.ldz, min(g.N - n0, B), rows};
    typename Tile::OpQ q = {g.X + lo * g.ldx + m0 * (long)sizeof(T), g.ldx, min(g.M - m0, B), rows};
    Tile t;
    t.clear();
    if (DIRECT) t.run_direct(lds, p, q, rows);
    else t.run_staged(lds, p, q, rows);
    if (SPLIT) {
        const long ld = (long)g.M * sizeof(A);
        store_tile<A, false>(t, lds, g.slabs + (blockIdx.y * (long)g.N + n0) * ld + m0 * (long)sizeof(A), ld, p.rows, q.rows, 1.0, 0.0);
    } else {
        store_tile<O, true>(t, lds, g.C + group * g.stride_c + n0 * g.ldc + m0 * (long)sizeof(O), g.ldc, p.rows, q.rows, g.alpha, g.beta);
    }
}

template <class A, class O>
__global__ __launch_bounds__(256) void grouped_dw_join_kernel(const GroupedDwArgs g) {
    const int group = blockIdx.y;
    // parts before this group and in it
    long first = 0, mine = 0;
    for (int g0 = 0; g0 <= group; g0 += 64) {
        const GroupScan s(g.offsets, g.groups, g.T, g0, g.part_rows);
        const int last = min(group - g0, 63);
        first += __shfl(s.sum - (g0 + 63 >= group ? s.tiles : 0), last, 64);
        mine = __shfl(s.tiles, last, 64);
    }
    mine = min(mine, max(0L, g.parts - first));   // a wrong table may name more parts than there are slabs
    const long size = (long)g.N * g.M;
    const A* slab = reinterpret_cast<const A*>(g.slabs) + first * size;
    const A al = (A)g.alpha, be = (A)g.beta;
    for (long e = blockIdx.x * 256L + threadIdx.x; e < size; e += gridDim.x * 256L) {
        A s = A(0);
        for (long part = 0; part < mine; ++part) s += slab[part * size + e];
        O* c = reinterpret_cast<O*>(g.C + group * g.stride_c + e / g.M * g.ldc) + e % g.M;
        *c = (O)(be != A(0) ? al * s + be * (A)*c : al * s);
    }
}

// rows in whole, aligned 16-byte chunks: what a direct-to-LDS load needs
bool whole_chunks(const void* p, long ld_bytes, long stride_bytes, long extent, long elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0 && stride_bytes % 16 == 0 && extent * elem % 16 == 0;
}

template <int V> using Int = std::integral_constant<int, V>;

// What a launch takes: less than 2^32 work-items along x (the grids are rounded up to a multiple of 32 workgroups).
bool one_launch(long workgroups, int threads) { return (workgroups + 31) * threads < 1L << 32; }
// A row-tile count that is never less than sum of ceil(rows / BM)
long row_tiles(long T, int groups, int BM) { return T / BM + (groups < T ? groups : T); }

// Which tile: the one whose rounds over the 256 CUs take the least time, by the time of a K step (128 bytes of k) with the
// chip full and with one workgroup on a CU, and of prologue and epilogue.  us, measured on a full chip:
struct TileCost { int bm, bn, slots, threads; double step, alone, rest; };
constexpr TileCost kCost16[] = {
    {256, 256, 256, 512, 1.50, 1.50, 14.0},   // one workgroup of 8 waves a CU: 1.17-1.25 PFLOP/s on 8 x 4096 x 4096 x 7168
    {128, 128, 512, 256, 1.05, 0.52, 5.0},    // two of 4 waves: 1.00-1.07
    {64, 64, 512, 256, 0.38, 0.25, 2.3},      // two of 4 waves, four LDS stages: 0.63
    {32, 128, 512, 256, 0.43, 0.30, 2.0},     // a few rows a group, W in 256-byte runs (n contiguous): the read of W bounds it
    {32, 64, 768, 256, 0.36, 0.25, 2.0},      // the same, k contiguous: 5.5 TB/s on 32 x 2816 x 2048
    {32, 64, 256, 1024, 0.25, 0.10, 4.0},      // few tiles and long k: four groups of waves share the sum (one of 8192 x 8192: 40 -> 28 us)
    {64, 64, 256, 1024, 0.25, 0.11, 5.0},
    {32, 16, 256, 512, 0.12, 0.05, 4.0}};     // narrow ones, eight single waves
// 4-byte floats and doubles; the last two as above: four groups of four waves (8 groups of 2 rows, 1024 x 1024 in doubles: 35 -> 27 us),
// eight of one (30 rows, 512 x 8192 in floats, 512 x 4096 in doubles: 87 -> 32 us)
constexpr TileCost kCost32[] = {{128, 128, 512, 256, 3.30, 2.40, 3.0}, {64, 64, 256, 256, 0.52, 0.52, 1.0}, {32, 64, 256, 256, 0.32, 0.45, 1.0},
                                 {32, 64, 256, 1024, 0.36, 0.33, 2.5}, {32, 16, 256, 512, 0.18, 0.06, 3.0}};
constexpr TileCost kCost64[] = {{128, 128, 512, 256, 3.90, 2.20, 3.0}, {64, 64, 256, 256, 0.51, 0.51, 1.0}, {32, 64, 256, 256, 0.31, 0.45, 1.0},
                                 {32, 64, 256, 1024, 0.36, 0.33, 2.5}, {32, 16, 256, 512, 0.18, 0.06, 3.0}};
double tile_time(const TileCost& c, double tiles, double steps) {
    const double full = floor(tiles / c.slots), left = tiles - full * c.slots;
    return full * (c.step * steps + c.rest) + (left > 256.0 ? c.step * steps + c.rest : left > 0.0 ? c.alone * steps + c.rest : 0.0);
}

template <class T> int grouped_typed(hipStream_t st, bool w_kc, const GroupedArgs& g) {
    GroupedArgs a = g;
    // rows of X (k contiguous) and of W in 16-byte chunks, lane offsets of one K step within the buffer resource
    const long wn = w_kc ? g.K : g.N;   // W's contiguous extent
    const bool direct = whole_chunks(g.X, g.ldx, 0, g.K, sizeof(T)) && whole_chunks(g.W, g.ldw, g.stride_w, wn, sizeof(T)) &&
                        256 * g.ldx < (long)mm::kRange && 256 * g.ldw < (long)mm::kRange;
    const double busy = (double)std::min<long>(g.groups, g.T), steps = (double)((g.K * (long)sizeof(T) + 127) / 128);
    const TileCost* const costs = sizeof(T) == 2 ? kCost16 : sizeof(T) == 4 ? kCost32 : kCost64;
    const int large = sizeof(T) == 2 ? 2 : 1;   // tiles that the next of the table is half of, in both directions
    // whether so many tiles behind the last whole round are better done in the next smaller tile by a launch of their own, 5 us
    auto better = [&](int i, double left) { return tile_time(costs[i + 1], 4.0 * left, steps) + 5.0 < tile_time(costs[i], left, steps); };
    auto tiles_of = [&](const TileCost& c) {   // half a row tile of every group is empty on average
        return std::max(busy, g.T / (double)c.bm + 0.5 * busy) * ((g.N + c.bn - 1) / c.bn);
    };
    auto fits = [&](const TileCost& c) { return one_launch(row_tiles(g.T, g.groups, c.bm) * ((g.N + c.bn - 1L) / c.bn), c.threads); };
    auto time_of = [&](const TileCost& c) { return fits(c) ? tile_time(c, tiles_of(c), steps) : 1e300; };
    int rc = GPX_OK;
    auto go = [&](auto bm, auto bn, auto wr, auto wc, auto stages, auto kgroups, auto rest) {
        constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WR = decltype(wr)::value, WC = decltype(wc)::value, ST = decltype(stages)::value,
                      KG = decltype(kgroups)::value;
        constexpr bool REST = decltype(rest)::value != 0;
        const long tiles = REST ? 4L * a.most : row_tiles(g.T, g.groups, BM) * ((g.N + BN - 1L) / BN);
        constexpr int threads = WR * WC * 64 * KG;
        if (!one_launch(tiles, threads)) {
            rc = GPX_ERR_UNSUPPORTED;
            return;
        }
        const unsigned grid = (unsigned)((tiles + 31) / 32 * 32);   // as many for every XCD (REST: whole tiles)
        if (w_kc && direct) grouped_kernel<T, BM, BN, WR, WC, ST, KG, true, true, REST><<<grid, threads, 0, st>>>(a);
        else if (direct) grouped_kernel<T, BM, BN, WR, WC, ST, KG, false, true, REST><<<grid, threads, 0, st>>>(a);
        else if constexpr (BM == 256 || KG > 1 || REST) rc = GPX_ERR_STATE;   // (never chosen for rows that are not direct)
        else if (w_kc) grouped_kernel<T, BM, BN, WR, WC, 2, 1, true, false, REST><<<grid, threads, 0, st>>>(a);
        else grouped_kernel<T, BM, BN, WR, WC, 2, 1, false, false, REST><<<grid, threads, 0, st>>>(a);
    };
    // The tile, or the larger one whose rest is done in smaller ones, if that saves more than the estimates are good for (chosen
    // for any gain: 4 x 1000 x 2048 x 1000 in double 289 -> 297 us).
    auto levels = [&](int best) {
        if (!direct) return best;
        double least = 0.93 * time_of(costs[best]);
        for (int i = 0; i < large; ++i) {
            const double tiles = tiles_of(costs[i]), left = fmod(tiles, costs[i].slots);
            const double time = tile_time(costs[i], tiles - left, steps) + tile_time(costs[i + 1], 4.0 * left, steps) + 5.0;
            if (tiles < costs[i].slots || left < 1.0 || time >= least) continue;
            least = time;
            best = i;
            a.slots = costs[i].slots;
            a.most = 0;
            for (int n = 8; n < a.slots && better(i, n); n += 8) a.most = n;
        }
        return best;
    };
    constexpr Int<0> whole{};
    constexpr Int<1> rest{};
    // from: rows that have to pass through registers take 128-tiles at most (20000 x 1001 x 2003 in bf16: 166 us, 256-tiles 241)
    auto best_of = [&](const TileCost* c, int from, int n, int not_this) {
        int best = from;
        for (int i = from + 1; i < n; ++i)
            if (i != not_this && time_of(c[i]) < time_of(c[best])) best = i;
        return best;
    };
    if constexpr (sizeof(T) == 2) {
        switch (levels(best_of(kCost16, direct ? 0 : 1, direct ? 8 : 5, w_kc ? 3 : 4))) {
            case 0:
                go(Int<256>{}, Int<256>{}, Int<2>{}, Int<4>{}, Int<2>{}, Int<1>{}, whole);
                if (a.slots) go(Int<128>{}, Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<1>{}, rest);
                break;
            case 1:
                go(Int<128>{}, Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<1>{}, whole);
                if (a.slots) go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<4>{}, Int<1>{}, rest);
                break;
            case 2: go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<4>{}, Int<1>{}, whole); break;
            case 3: go(Int<32>{}, Int<128>{}, Int<1>{}, Int<4>{}, Int<4>{}, Int<1>{}, whole); break;
            case 4: go(Int<32>{}, Int<64>{}, Int<1>{}, Int<4>{}, Int<4>{}, Int<1>{}, whole); break;
            case 5: go(Int<32>{}, Int<64>{}, Int<1>{}, Int<4>{}, Int<3>{}, Int<4>{}, whole); break;
            case 6: go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<4>{}, whole); break;
            default: go(Int<32>{}, Int<16>{}, Int<1>{}, Int<1>{}, Int<3>{}, Int<8>{}, whole);
        }
    } else if (const long units = row_tiles(g.T, g.groups, 32 * kShortSub) * ((g.N + 63L) / 64);
               direct && g.K * (long)sizeof(T) <= 512 && 32 * g.ldy < (long)mm::kRange && g.K > 0 && units >= 512 && one_launch(units, 256)) {
        // (fewer workgroups than slots on the chip: no better than single tiles)
        const unsigned grid = (unsigned)((units + 7) / 8 * 8);
        if (w_kc) grouped_short_kernel<T, true><<<grid, 256, 0, st>>>(g);
        else grouped_short_kernel<T, false><<<grid, 256, 0, st>>>(g);
    } else {
        switch (levels(best_of(costs, 0, direct ? 5 : 3, -1))) {
            case 0:
                go(Int<128>{}, Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<1>{}, whole);
                if (a.slots) go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<1>{}, rest);
                break;
            case 1: go(Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<1>{}, whole); break;
            case 2: go(Int<32>{}, Int<64>{}, Int<1>{}, Int<4>{}, Int<4>{}, Int<1>{}, whole); break;
            case 3: go(Int<32>{}, Int<64>{}, Int<1>{}, Int<4>{}, Int<3>{}, Int<4>{}, whole); break;
            default: go(Int<32>{}, Int<16>{}, Int<1>{}, Int<1>{}, Int<3>{}, Int<8>{}, whole);
        }
    }
    if (rc) return rc;
    HIP_TRY(hipGetLastError());
    return GPX_OK;
}

// The weight gradient's tile and the rows of a part (0: not split), from sizes alone: the workspace follows from it.
struct DwPlan { int tile, part_rows; long parts; };
// (Whether it is split and into what does not depend on the results' type, so that the workspace does not either.)
DwPlan dw_plan(int elem, int c_elem, long groups, long T, long M, long N) {
    const TileCost* c = elem == 2 ? kCost16 : elem == 4 ? kCost32 : kCost64;
    const int sizes = elem == 2 ? 3 : 2;
    const double busy = (double)std::max<long>(1, std::min(groups, T)), per = 128.0 / elem, steps = std::max(1.0, ceil(T / busy / per));
    auto tiles = [&](int i) { return (double)((N + c[i].bn - 1) / c[i].bn) * ((M + c[i].bm - 1) / c[i].bm); };
    DwPlan best = {0, 0, 0};
    double least = 1e300;
    for (int i = 0; i < sizes; ++i) {
        // Groups of unequal rows leave the large tiles of floats and doubles unevenly over the CUs where each gets a few:
        // 512 tiles of 128 in double, groups of 4096 to 12288 rows: 2.39 ms, as 2048 tiles of 64: 2.02; equal groups: 1.97 and 2.06.
        const double uneven = elem > 2 && i == 0 && groups > 1 && tiles(i) * groups < 4.0 * c[i].slots ? 1.2 : 1.0;
        const double t = uneven * tile_time(c[i], tiles(i) * groups, steps);
        if (t < least) {
            least = t;
            best = {i, 0, 0};
        }
    }
    // Split: parts of at least 8 steps, as many as give the chip one round; the slabs are written and read once (4 TB/s) and
    // the second kernel costs 4 us more.
    for (int i = 0; i < sizes; ++i) {
        const double round = std::max(256.0, (double)c[i].slots) / tiles(i);
        const long rows = std::max<long>((long)(8 * per), ((long)ceil(T / std::max(1.0, round - 0.5 * busy)) + 63) / 64 * 64);
        if (rows * busy > 0.75 * T) continue;
        const long parts = T / rows + std::min(groups, T);
        const double each = std::max(c[i].alone, c[i].step / std::max(1.0, c[i].slots / 256.0));
        const double t = ceil(tiles(i) * (T / (double)rows + 0.5 * busy) / 256.0) * (each * rows / per + c[i].rest) +
                         4.0 + 2.0 * parts * (double)(M * N) * std::max(4, elem) / 4e6;
        if (t < 0.8 * least && rows < (1L << 30) && parts <= 65535) {
            least = t;
            best = {i, (int)rows, parts};
        }
    }
    // 16-bit rows, one pass: the stores of a round weigh more than its steps where the groups are short.  us a round besides the
    // steps, 16- and 32-bit results: 256-tiles 9 / 16, 128-tiles 3 / 10 (16 groups of 512 rows, 2816 x 2048: 125 / 165 and 119 / 193)
    if (elem == 2 && !best.part_rows) {
        const double wide = c_elem == 4 ? 7.0 : 0.0;
        TileCost t256 = c[0], t128 = c[1];
        t256.rest = 9.0 + wide;
        t128.step = 0.95;
        t128.rest = 3.0 + wide;
        const double a = tile_time(t256, tiles(0) * groups, steps), b = tile_time(t128, tiles(1) * groups, steps);
        if (best.tile < 2 || std::min(a, b) < least) best.tile = a < b ? 0 : 1;
    }
    return best;
}
long dw_work_bytes(const DwPlan& p, int elem, long M, long N) { return p.part_rows ? p.parts * M * N * std::max(4, elem) : 0; }

template <class T, class O> int grouped_dw_typed(hipStream_t st, const GroupedDwArgs& g, const DwPlan& plan) {
    const bool direct = whole_chunks(g.X, g.ldx, 0, g.M, sizeof(T)) && whole_chunks(g.Z, g.ldz, 0, g.N, sizeof(T)) &&
                        64 * g.ldx < (long)mm::kRange && 64 * g.ldz < (long)mm::kRange;
    int rc = GPX_OK;
    auto go = [&](auto bm, auto wr, auto wc, auto stages) {
        constexpr int B = decltype(bm)::value, WR = decltype(wr)::value, WC = decltype(wc)::value, ST = decltype(stages)::value;
        const long tiles = (long)((g.N + B - 1L) / B) * ((g.M + B - 1L) / B);
        if (!one_launch(tiles, WR * WC * 64)) {
            rc = GPX_ERR_UNSUPPORTED;
            return;
        }
        if (plan.part_rows) {
            const dim3 grid((unsigned)tiles, (unsigned)plan.parts);
            if (direct) grouped_dw_kernel<T, O, B, WR, WC, ST, true, true><<<grid, WR * WC * 64, 0, st>>>(g);
            else if constexpr (B == 256) rc = GPX_ERR_STATE;
            else grouped_dw_kernel<T, O, B, WR, WC, 2, false, true><<<grid, WR * WC * 64, 0, st>>>(g);
            const long size = (long)g.M * g.N;
            grouped_dw_join_kernel<typename mm::Acc<T>::one, O>
                <<<dim3((unsigned)std::min<long>((size + 255) / 256, 2048), (unsigned)g.groups), 256, 0, st>>>(g);
        } else {
            const dim3 grid((unsigned)tiles, (unsigned)g.groups);
            if (direct) grouped_dw_kernel<T, O, B, WR, WC, ST, true, false><<<grid, WR * WC * 64, 0, st>>>(g);
            else if constexpr (B == 256) rc = GPX_ERR_STATE;
            else grouped_dw_kernel<T, O, B, WR, WC, 2, false, false><<<grid, WR * WC * 64, 0, st>>>(g);
        }
    };
    if constexpr (sizeof(T) == 2) {
        if (plan.tile == 0 && direct) go(Int<256>{}, Int<2>{}, Int<4>{}, Int<2>{});
        else if (plan.tile <= 1) go(Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{});
        else go(Int<64>{}, Int<2>{}, Int<2>{}, Int<4>{});
    } else {
        if (plan.tile == 0) go(Int<128>{}, Int<2>{}, Int<2>{}, Int<2>{});
        else go(Int<64>{}, Int<2>{}, Int<2>{}, Int<2>{});
    }
    if (rc) return rc;
    HIP_TRY(hipGetLastError());
    return GPX_OK;
}

constexpr long kMaxExtent = (1L << 31) - 1024;   // row, column and k numbers within one product are 32-bit
constexpr int kMaxGroups = 65535;
constexpr int64_t kMaxLd = 1L << 32, kMaxStride = 1L << 48;   // elements: in bytes they pass no 63 bits

int elem_bytes(int dtype) { return dtype == GPX_F64 ? 8 : dtype == GPX_F32 ? 4 : dtype == GPX_BF16 || dtype == GPX_F16 ? 2 : 0; }
bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes != 0; }

}  // namespace

extern "C" int gpx_grouped_gemm(int dtype, int w_kc, int64_t groups, int64_t T, int64_t N, int64_t K, double alpha, const void* X,
                                int64_t ldx, const void* W, int64_t ldw, int64_t stride_w, const int64_t* offsets, double beta,
                                void* Y, int64_t ldy, void* hip_stream) {
    const int e = elem_bytes(dtype);
    if (!e || groups < 0 || groups > kMaxGroups || T < 0 || N < 0 || K < 0) return GPX_ERR_ARG;
    if (T > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return GPX_ERR_ARG;
    if (ldx < K || ldw < (w_kc ? K : N) || ldy < N || stride_w < 0) return GPX_ERR_ARG;
    if (ldx > kMaxLd || ldw > kMaxLd || ldy > kMaxLd || stride_w > kMaxStride) return GPX_ERR_ARG;
    const ByteRows x = {X, 1, 0, T, ldx * e, K * e}, y = {Y, 1, 0, T, ldy * e, N * e};
    const ByteRows w = {W, groups, stride_w * e, w_kc ? N : K, ldw * e, (w_kc ? K : N) * e}, table = {offsets, 1, 0, 1, 0, 8 * (groups + 1)};
    if (!gpx_reaches(x) || !gpx_reaches(y) || !gpx_reaches(w)) return GPX_ERR_ARG;
    if (groups == 0 || T == 0 || N == 0) return GPX_OK;   // no row of Y belongs to a group
    if (!Y || !offsets || (K > 0 && (!X || !W))) return GPX_ERR_ARG;
    if (misaligned(X, e) || misaligned(W, e) || misaligned(Y, e) || misaligned(offsets, 8)) return GPX_ERR_ARG;
    if (gpx_share_bytes(y, x) || gpx_share_bytes(y, w) || gpx_share_bytes(y, table)) return GPX_ERR_ARG;
    StreamDevice dev(static_cast<hipStream_t>(hip_stream));
    if (dev.status) return dev.status;
    GroupedArgs g = {static_cast<const char*>(X), static_cast<const char*>(W), static_cast<char*>(Y), offsets, ldx * e, ldw * e,
                     stride_w * e, ldy * e, T, (int)groups, (int)N, (int)K, alpha, beta, 0, 0};
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
    if (ldx > kMaxLd || ldz > kMaxLd || ldc > kMaxLd || stride_c > kMaxStride) return GPX_ERR_ARG;
    const ByteRows x = {X, 1, 0, T, ldx * e, M * e}, z = {Z, 1, 0, T, ldz * e, N * e}, c = {C, groups, stride_c * ec, N, ldc * ec, M * ec};
    const ByteRows table = {offsets, 1, 0, 1, 0, 8 * (groups + 1)};
    if (!gpx_reaches(x) || !gpx_reaches(z) || !gpx_reaches(c)) return GPX_ERR_ARG;
    if (groups == 0 || M == 0 || N == 0) return GPX_OK;
    if (groups > 1 && stride_c < (N - 1) * ldc + M) return GPX_ERR_ARG;   // results of two groups would overlap
    if (!C || !offsets || (T > 0 && (!X || !Z))) return GPX_ERR_ARG;
    if (misaligned(X, e) || misaligned(Z, e) || misaligned(C, ec) || misaligned(offsets, 8)) return GPX_ERR_ARG;
    const DwPlan plan = dw_plan(e, ec, groups, T, M, N);
    if (plan.part_rows && (!work || misaligned(work, 16) || work_bytes < dw_work_bytes(plan, e, M, N))) return GPX_ERR_ARG;
    const ByteRows w = {work, 1, 0, 1, 0, dw_work_bytes(plan, e, M, N)};
    if (gpx_share_bytes(c, x) || gpx_share_bytes(c, z) || gpx_share_bytes(c, table) || gpx_share_bytes(w, x) || gpx_share_bytes(w, z) ||
        gpx_share_bytes(w, c) || gpx_share_bytes(w, table))
        return GPX_ERR_ARG;
    StreamDevice dev(static_cast<hipStream_t>(hip_stream));
    if (dev.status) return dev.status;
    const GroupedDwArgs g = {static_cast<const char*>(X), static_cast<const char*>(Z), static_cast<char*>(C), offsets, ldx * e, ldz * e, ldc * ec,
                             stride_c * ec, T, (int)M, (int)N, (int)groups, alpha, beta,
                             static_cast<char*>(work), plan.part_rows, (int)plan.parts};
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    switch (dtype) {
        case GPX_F64: return grouped_dw_typed<double, double>(st, g, plan);
        case GPX_F32: return grouped_dw_typed<float, float>(st, g, plan);
        case GPX_BF16: return c_dtype == GPX_F32 ? grouped_dw_typed<__bf16, float>(st, g, plan) : grouped_dw_typed<__bf16, __bf16>(st, g, plan);
        default: return c_dtype == GPX_F32 ? grouped_dw_typed<_Float16, float>(st, g, plan) : grouped_dw_typed<_Float16, _Float16>(st, g, plan);
    }
}

extern "C" int gpx_grouped_gemm_dw_work(int dtype, int64_t groups, int64_t T, int64_t M, int64_t N, int64_t* work_bytes) {
    const int e = elem_bytes(dtype);
    if (!e || !work_bytes || groups < 0 || groups > kMaxGroups || T < 0 || M < 0 || N < 0 || T > kMaxExtent || M > kMaxExtent || N > kMaxExtent)
        return GPX_ERR_ARG;
    *work_bytes = groups && T && M && N ? dw_work_bytes(dw_plan(e, e, groups, T, M, N), e, M, N) : 0;
    return GPX_OK;
}
