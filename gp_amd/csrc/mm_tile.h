// mm_tile.h — one workgroup's output tile D = P Q^T on the matrix cores, for double, float, bf16 and f16 operands.
//
// D(i, j) = sum_k P(i, k) Q(j, k), i < BM, j < BN.  Either operand is stored with k contiguous (KC: element (i, k) at
// base + i*ld + k) or with its own index contiguous (base + k*ld + i).  Products of 16-bit elements and of floats are summed
// in 32 bits, those of doubles in 64: the accumulator of the matrix instruction, never narrower.
//
// LDS image of one K step: 128 bytes of k per row (BK = 16 doubles, 32 floats, 64 16-bit elements), always written in 16-byte
// chunks, chunk number = thread number, so that the image is the same whether a chunk arrives through registers or straight
// from memory.  KC operands: [row][8 chunks], chunk c of row r sits at c ^ (r & 7): the 16 rows that one fragment read
// touches would otherwise share one 128-byte bank window.  The others: [k][ROWS], blocks of 16 columns permuted by a function
// of k (strided_swizzle) for the same reason.  Fragments: lane l holds row l & 15 and the k group l >> 4 of its 16x16 tile;
// both operands use one assignment of k to lanes, so any assignment is right and the one that reads 16 contiguous bytes is taken.
// 16-bit operands with k strided are turned by the transposing LDS read (ds_read_b64_tr_b16: in each 16 lanes, lane n
// addresses 8 bytes of row n / 4 and receives column n of the 4 x 16 block).
#pragma once
#include "gpx_internal.h"

namespace mm {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <class T> struct Acc { typedef v4f vec; typedef float one; };
template <> struct Acc<double> { typedef v4d vec; typedef double one; };

template <class T> constexpr int chunk_elems() { return 16 / (int)sizeof(T); }
template <class T> constexpr int step_k() { return 128 / (int)sizeof(T); }

// ---- fragments: 16 rows x (64 bytes of k), one v4i per lane --------------------------------------------------------
template <class T> __device__ __forceinline__ int strided_swizzle(int k) {
    if (sizeof(T) == 8) return (k >> 1) & 1;   // the k groups 2q of one read: halves of the 256-byte bank window
    if (sizeof(T) == 4) return (k >> 2) & 3;   // the k groups 4q: quarters
    return (k & 3) | ((k >> 3) & 1) << 2;      // 32-byte blocks: rows k..k+3 of the k groups 8q
}

// of the block numbers of a row of `cols` elements: the permutation must stay within the row
template <class T> constexpr int swizzle_mask(int cols) {
    return sizeof(T) == 2 ? (cols / 16 % 8 == 0 ? 7 : cols / 16 % 4 == 0 ? 3 : cols / 16 % 2 == 0 ? 1 : 0)
                          : (cols / 16 % 4 == 0 ? 3 : cols / 16 % 2 == 0 ? 1 : 0);
}

template <class T, int ROWS, bool KC>
__device__ __forceinline__ v4i frag(const char* s, int row0, int kk, int lane) {
    const int r = lane & 15, q = lane >> 4;
    if constexpr (KC) {
        const int row = row0 + r;
        return *reinterpret_cast<const v4i*>(s + row * 128 + (((kk * 4 + q) ^ (row & 7)) << 4));
    } else if constexpr (sizeof(T) == 2) {
        constexpr int mask = swizzle_mask<T>(ROWS);
        const int k = kk * 32 + 8 * q + (r >> 2);
        const int b = (row0 >> 4) ^ (strided_swizzle<T>(k) & mask);
        const char* p = s + k * (ROWS * 2) + b * 32 + (r & 3) * 8;
        typedef __attribute__((address_space(3))) v4s lds4;
        union { v4s h[2]; v4i v; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * ROWS * 2));
        return u.v;
    } else {
        constexpr int E = chunk_elems<T>(), mask = swizzle_mask<T>(ROWS);
        const int k = kk * 4 * E + E * q;
        const int b = (row0 >> 4) ^ (strided_swizzle<T>(k) & mask);
        const T* p = reinterpret_cast<const T*>(s) + k * ROWS + b * 16 + r;
        union { T e[E]; v4i v; } u;
#pragma unroll
        for (int x = 0; x < E; ++x) u.e[x] = p[x * ROWS];
        return u.v;
    }
}

// Split format (mm::Split): a matrix of values known to 22 bits as two f16 planes, v = hi + lo, in blocks of 32 columns:
// element (r, c) has hi at r*ld + (c / 32)*64 + c % 32 and lo 32 elements behind it.  128 bytes are 32 values, so that a K step
// has the geometry of 16-bit operands: its two 64-byte halves are the two planes.  Rows end in zeros up to a whole block.
struct Split {};
template <int ROWS, bool KC>
__device__ __forceinline__ v4i frag_split(const char* s, int row0, int lo, int lane) {
    if constexpr (KC) return frag<_Float16, ROWS, true>(s, row0, lo, lane);
    const int r = lane & 15, q = lane >> 4;
    static_assert(swizzle_mask<_Float16>(2 * ROWS) == 7, "whole permutations");
    const int k = 8 * q + (r >> 2);
    const int b = ((row0 >> 5) * 4 + ((row0 >> 4) & 1) + 2 * lo) ^ strided_swizzle<_Float16>(k);
    const char* p = s + k * (ROWS * 4) + b * 32 + (r & 3) * 8;
    typedef __attribute__((address_space(3))) v4s lds4;
    union { v4s h[2]; v4i v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * ROWS * 4));
    return u.v;
}

// D += A B^T over the 64 bytes of k of the fragments.  The lane holds D rows (index of `a`) 4q + r (doubles: q + 4r),
// r = 0..3, and the column (index of `b`) lane & 15.
template <class T> __device__ __forceinline__ typename Acc<T>::vec mma(v4i a, v4i b, typename Acc<T>::vec c) {
    if constexpr (sizeof(T) == 8) {
        union { v4i v; double e[2]; } x{a}, y{b};
        c = __builtin_amdgcn_mfma_f64_16x16x4f64(x.e[0], y.e[0], c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f64_16x16x4f64(x.e[1], y.e[1], c, 0, 0, 0);
    } else if constexpr (sizeof(T) == 4) {
        union { v4i v; float e[4]; } x{a}, y{b};
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.e[s], y.e[s], c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, __bf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
}

// ---- one operand's tile of one K step, through registers: any alignment, any extent ---------------------------------
// `valid` elements of the 16 bytes at p may be read, the others are zero
template <class T> __device__ __forceinline__ v4i load_chunk(const char* p, int valid) {
    constexpr int E = chunk_elems<T>();
    v4i v = {0, 0, 0, 0};
    if (valid >= E) {
        __builtin_memcpy(&v, p, 16);
    } else if (valid > 0) {
        union { v4i v; T e[E]; } u;
        u.v = v;
#pragma unroll
        for (int x = 0; x < E; ++x)
            if (x < valid) u.e[x] = reinterpret_cast<const T*>(p)[x];
        v = u.v;
    }
    return v;
}

// Scalar registers that a vector instruction may have written (readfirstlane) must be five wait states old before a memory
// instruction reads them.  The compiler sees to that for its own instructions, not for those in inline assembly: the value
// passes through this between the two.
template <class S> __device__ __forceinline__ void settle(S& s) { asm volatile("s_nop 4" : "+s"(s)); }

constexpr unsigned kRange = 0x7fff0000u;     // bytes that the lane offsets of one K step may span (checked by the host)
constexpr unsigned kOutside = 0x7fff8000u;   // an offset behind them

// what a type is stored as, and the values of k in a step
template <class T> struct Stored { typedef T type; static constexpr int BK = step_k<T>(), WIDE = 1; static constexpr bool split = false; };
template <> struct Stored<Split> { typedef _Float16 type; static constexpr int BK = 32, WIDE = 2; static constexpr bool split = true; };

template <class F, int ROWS, bool KC, int NT> struct Operand {
    typedef typename Stored<F>::type T;
    static constexpr int E = chunk_elems<T>(), BK = Stored<F>::BK;
    static constexpr int COLS = ROWS * Stored<F>::WIDE;   // elements per k of an operand with k strided
    static constexpr int NL = ROWS * 8 / NT;   // chunks per thread
    static constexpr int BYTES = ROWS * 128;
    static_assert(ROWS * 8 % NT == 0 && (NT & (NT - 1)) == 0, "whole chunks per thread");
    __device__ static __forceinline__ int tid() { return threadIdx.x & (NT - 1); }   // of the K group
    const char* base;   // element (0, 0) of the tile's rows
    long ld;            // bytes between rows (KC) or between k (otherwise)
    int rows, K;        // rows of the tile (split, k strided: elements) and extent of k that exist

    __device__ __forceinline__ void place(int c, int& row, int& k) const {   // first element of chunk c
        if (KC) {
            row = c >> 3;
            k = ((c & 7) ^ (row & 7)) * E;
        } else {
            constexpr int PER = COLS / E;              // chunks per k
            constexpr int HB = 16 / E;                 // chunks per block of 16 columns
            constexpr int mask = swizzle_mask<T>(COLS);
            k = c / PER;
            const int slot = c % PER;
            row = ((slot / HB) ^ (strided_swizzle<T>(k) & mask)) * 16 + slot % HB * E;
        }
    }
    __device__ __forceinline__ void load(v4i (&r)[NL], int k0) const {
#pragma unroll
        for (int it = 0; it < NL; ++it) {
            int row, k;
            place(it * NT + tid(), row, k);
            k += k0;
            if (KC) r[it] = load_chunk<T>(base + row * ld + (long)k * sizeof(T), row < rows ? K - k : 0);
            else r[it] = load_chunk<T>(base + k * ld + (long)row * sizeof(T), k < K ? rows - row : 0);
        }
    }
    // The same for a step that has more than a step of k behind it: no tests.  Rows that do not exist read the last one
    // (their results are dropped); with k strided a run may end up to 15 bytes behind its row, in the rows of the next step.
    __device__ __forceinline__ void load_inside(v4i (&r)[NL], int k0) const {
#pragma unroll
        for (int it = 0; it < NL; ++it) {
            int row, k;
            place(it * NT + tid(), row, k);
            row = min(row, rows - 1);
            k += k0;
            const char* p = KC ? base + row * ld + (long)k * sizeof(T) : base + k * ld + (long)row * sizeof(T);
            __builtin_memcpy(&r[it], p, 16);
        }
    }
    // ---- straight from memory into LDS: 16-byte aligned rows whose contiguous extent is a multiple of E elements, so that
    // a chunk exists as a whole or not at all.  A chunk that does not exist gets an offset behind the resource's
    // range: the load returns zeros without touching memory.
    struct Lanes { unsigned off[NL]; };
    __device__ __forceinline__ Lanes lanes(int k_valid) const {   // of one K step that has k_valid values of k
        Lanes l;
#pragma unroll
        for (int it = 0; it < NL; ++it) {
            int row, k;
            place(it * NT + tid(), row, k);
            const unsigned at = KC ? (unsigned)(row * ld) + k * (unsigned)sizeof(T) : (unsigned)(k * ld) + row * (unsigned)sizeof(T);
            l.off[it] = row < rows && (k < k_valid || (KC && Stored<F>::split)) ? at : kOutside;
        }
        return l;
    }
    // ONCE: nobody else reads these bytes, they need not stay in a cache
    template <bool ONCE = false> __device__ __forceinline__ void issue(unsigned lds_addr, const Lanes& l, int step) const {
        const unsigned long long a = reinterpret_cast<unsigned long long>(base) + (unsigned long long)step * (KC ? 128 : BK * ld);
        v4i rsrc = {__builtin_amdgcn_readfirstlane((int)(unsigned)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)),
                    (int)kRange, 0x00027000};
        settle(rsrc);
        const unsigned wave_addr = __builtin_amdgcn_readfirstlane(lds_addr + (tid() >> 6) * 1024);
#pragma unroll
        for (int it = 0; it < NL; ++it)   // lane l of the wave writes the 16 bytes at M0 + 16 l
            if constexpr (ONCE)
                asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(l.off[it]), "s"(rsrc),
                             "s"(wave_addr + it * NT * 16)
                             : "memory");
            else
                asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(l.off[it]), "s"(rsrc),
                             "s"(wave_addr + it * NT * 16)
                             : "memory");
    }
    __device__ __forceinline__ void stash(char* s, const v4i (&r)[NL]) const {
#pragma unroll
        for (int it = 0; it < NL; ++it) *reinterpret_cast<v4i*>(s + (it * NT + tid()) * 16) = r[it];
    }
};

// ---- the tile ----------------------------------------------------------------------------------------------------
// Waves in a WR (rows i) x WC (columns j) grid; each owns TI x TJ fragments of 16.  SWAP: the accumulator's contiguous
// lanes run along j (doubles and floats: whole 64..128-byte runs per store); otherwise its four registers do (16-bit
// results: 8-byte stores instead of single elements).
template <class F, int BM, int BN, int WR, int WC, bool PKC, bool QKC, int STAGES = 2, int GROUPS = 1> struct Tile {
    typedef typename Stored<F>::type T;
    static constexpr int NT = WR * WC * 64;
    static constexpr int TI = BM / WR / 16, TJ = BN / WC / 16;
    static constexpr bool SWAP = sizeof(T) != 2;
    // a tile of 32 rows is mostly all the rows of its group: its Q is read once (32 groups of 2816 x 2048: 4.9 -> 5.5 TB/s)
    static constexpr bool ONCE = BM == 32;
    typedef Operand<F, BM, PKC, NT> OpP;
    typedef Operand<F, BN, QKC, NT> OpQ;
    typedef typename Acc<T>::vec vec;
    typedef typename Acc<T>::one one;
    static constexpr int STAGE = OpP::BYTES + OpQ::BYTES;
    static constexpr int LDS = STAGES * GROUPS * STAGE;
    static constexpr int THREADS = NT * GROUPS;
    __device__ static __forceinline__ int wave_id() { return (threadIdx.x & (NT - 1)) >> 6; }
    __device__ static __forceinline__ int group() { return GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT); }
    vec acc[TI][TJ];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = vec{};
    }
    // whether any of this wave's rows and columns exist: a ragged last tile costs the matrix cores only the wave rows it has
    __device__ __forceinline__ bool has_rows(int rows_p, int rows_q) const {
        const int wave = __builtin_amdgcn_readfirstlane(wave_id());
        return wave / WC * (BM / WR) < rows_p && wave % WC * (BN / WC) < rows_q;   // (split, k strided: twice the rows, never less)
    }
    // halves: 1 if the second 64 bytes of k are all zeros (the end of K)
    __device__ __forceinline__ void multiply(const char* sp, const char* sq, int halves = 2) {
        const int lane = threadIdx.x & 63, wave = wave_id();
        const int i0 = wave / WC * (BM / WR), j0 = wave % WC * (BN / WC);
        if constexpr (Stored<F>::split) {
            // (ph + pl)(qh + ql) without pl ql, which is 2^-22 of the product at most
            v4i qh[TJ], ql[TJ];
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                qh[j] = frag_split<BN, QKC>(sq, j0 + 16 * j, 0, lane);
                ql[j] = frag_split<BN, QKC>(sq, j0 + 16 * j, 1, lane);
            }
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                const v4i ph = frag_split<BM, PKC>(sp, i0 + 16 * i, 0, lane), pl = frag_split<BM, PKC>(sp, i0 + 16 * i, 1, lane);
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = mma<T>(ql[j], ph, acc[i][j]);
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = mma<T>(qh[j], pl, acc[i][j]);
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = mma<T>(qh[j], ph, acc[i][j]);
            }
            return;
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            if (kk >= halves) break;
            v4i fp[TI], fq[TJ];
#pragma unroll
            for (int i = 0; i < TI; ++i) fp[i] = frag<T, BM, PKC>(sp, i0 + 16 * i, kk, lane);
#pragma unroll
            for (int j = 0; j < TJ; ++j) fq[j] = frag<T, BN, QKC>(sq, j0 + 16 * j, kk, lane);
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = SWAP ? mma<T>(fp[i], fq[j], acc[i][j]) : mma<T>(fq[j], fp[i], acc[i][j]);
        }
    }
    // register-staged K loop: the chunks of step k + 1 are in flight while step k is multiplied, two LDS stages, one barrier
    __device__ __forceinline__ void run_staged(char* lds, const OpP& p, const OpQ& q, int K) {
        v4i rp[OpP::NL], rq[OpQ::NL];
        const int steps = (K + OpP::BK - 1) / OpP::BK;
        if (steps == 0) return;
        const bool busy = has_rows(p.rows, q.rows);
        auto load = [&](int s) {
            if ((s + 2) * OpP::BK <= K) {
                p.load_inside(rp, s * OpP::BK);
                q.load_inside(rq, s * OpP::BK);
            } else {
                p.load(rp, s * OpP::BK);
                q.load(rq, s * OpP::BK);
            }
        };
        load(0);
        for (int s = 0; s < steps; ++s) {
            char* st = lds + (s & 1) * STAGE;
            p.stash(st, rp);
            q.stash(st + OpP::BYTES, rq);
            if (s + 1 < steps) load(s + 1);
            __syncthreads();   // also: nobody reads the other stage any more when the next step writes it
            if (busy) multiply(st, st + OpP::BYTES);
        }
    }
    // K loop on direct loads, STAGES LDS stages: while step s is multiplied, steps s + 1 .. s + STAGES - 1 are on their way.
    __device__ __forceinline__ void run_direct(char* lds, const OpP& p, const OpQ& q, int K) {
        constexpr int BK = OpP::BK;
        constexpr int AHEAD = (STAGES - 2) * (OpP::NL + OpQ::NL);   // loads of this wave behind those of the step waited for
        const int full = K / BK, rest = K - full * BK, steps = full + (rest != 0);
        typename OpP::Lanes lp = p.lanes(BK);
        typename OpQ::Lanes lq = q.lanes(BK);
        const unsigned at = (unsigned)reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)lds);
        auto issue = [&](int s, int stage) {
            if (s >= full) {
                lp = p.lanes(rest);
                lq = q.lanes(rest);
            }
            p.issue(at + stage * STAGE, lp, s);
            q.template issue<ONCE>(at + stage * STAGE + OpP::BYTES, lq, s);
        };
        const bool busy = has_rows(p.rows, q.rows);
        for (int s = 0; s < STAGES - 1 && s < steps; ++s) issue(s, s);
        int stage = 0, into = STAGES - 1;   // of step s, of step s + STAGES - 1
        for (int s = 0; s < steps; ++s) {
            // this wave's part of step s has arrived, and it reads nothing of the stage that is overwritten next any more
            if (STAGES > 2 && s + STAGES - 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(AHEAD) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + STAGES - 1 < steps) issue(s + STAGES - 1, into);
            if (busy) multiply(lds + stage * STAGE, lds + stage * STAGE + OpP::BYTES, s >= full && rest * 2 <= BK ? 1 : 2);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            into = into + 1 == STAGES ? 0 : into + 1;
        }
    }
    // The same for few tiles with long sums: GROUPS sets of NT threads take the steps in turn, each with LDS stages of its own,
    // and add their accumulators at the end in one order, the sum in group 0.  A step of a 64-tile alone on its CU costs
    // 0.36 us, most of it waiting; four groups do four in 0.5 us.
    __device__ __forceinline__ void run_groups(char* lds, const OpP& p, const OpQ& q, int K) {
        static_assert(GROUPS > 1, "groups");
        constexpr int BK = OpP::BK, AHEAD = (STAGES - 2) * (OpP::NL + OpQ::NL);
        const int full = K / BK, rest = K - full * BK, steps = full + (rest != 0), turns = (steps + GROUPS - 1) / GROUPS, mine = group();
        const int own_turns = (steps - mine + GROUPS - 1) / GROUPS;   // (0 where steps <= mine)
        typename OpP::Lanes lp = p.lanes(BK);
        typename OpQ::Lanes lq = q.lanes(BK);
        char* own = lds + mine * STAGES * STAGE;
        const unsigned at = (unsigned)reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)own);
        auto issue = [&](int turn, int stage) {
            const int s = turn * GROUPS + mine;
            if (s >= steps) return;
            if (s >= full) {
                lp = p.lanes(rest);
                lq = q.lanes(rest);
            }
            p.issue(at + stage * STAGE, lp, s);
            q.template issue<ONCE>(at + stage * STAGE + OpP::BYTES, lq, s);
        };
        const bool busy = has_rows(p.rows, q.rows);
        for (int t = 0; t < STAGES - 1; ++t) issue(t, t);
        int stage = 0, into = STAGES - 1;
        for (int t = 0; t < turns; ++t) {
            if (STAGES > 2 && t + STAGES - 2 < own_turns) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(AHEAD) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            issue(t + STAGES - 1, into);
            const int s = t * GROUPS + mine;
            const char* st = own + stage * STAGE;
            if (busy && s < steps) multiply(st, st + OpP::BYTES, s >= full && rest * 2 <= BK ? 1 : 2);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            into = into + 1 == STAGES ? 0 : into + 1;
        }
        __syncthreads();
        vec* meet = reinterpret_cast<vec*>(lds);
        constexpr int EACH = TI * TJ * NT;
        static_assert((GROUPS - 1) * EACH * (int)sizeof(vec) <= LDS, "the accumulators take the place of the stages");
        if (mine > 0) {
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) meet[(mine - 1) * EACH + (i * TJ + j) * NT + (threadIdx.x & (NT - 1))] = acc[i][j];
        }
        __syncthreads();
        if (mine == 0) {
#pragma unroll
            for (int g = 0; g < GROUPS - 1; ++g)
#pragma unroll
                for (int i = 0; i < TI; ++i)
#pragma unroll
                    for (int j = 0; j < TJ; ++j) acc[i][j] += meet[g * EACH + (i * TJ + j) * NT + threadIdx.x];
        }
    }
    // The accumulators of wave row `pass` (BM / WR rows of the tile) as floats in LDS, rows of SLAB_LD: what an epilogue that
    // reads and writes whole 16-byte runs needs.  Between barriers of the caller.
    static constexpr int SLAB_ROWS = BM / WR, SLAB_LD = BN + 4, SLAB = SLAB_ROWS * SLAB_LD * 4;
    // groups of four columns permuted by the row, so that a column of eight-row runs does not meet in one bank
    __device__ static __forceinline__ int slab_at(int row, int col) { return row * SLAB_LD + (col ^ (row >> 3 & 7) << 2); }
    __device__ __forceinline__ void to_slab(float* slab, int pass) const {
        const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, q = lane >> 4;
        if (wave / WC != pass || group() != 0) return;
        const int j0 = wave % WC * (BN / WC);
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) *reinterpret_cast<v4f*>(slab + slab_at(16 * i + r, j0 + 16 * j + 4 * q)) = acc[i][j];
    }
    // Epilogue in whole runs: f(i, j, v) for every run of RUN columns j.. of row i, i < rows, j < cols (16-bit operands).  RUN
    // elements of the result are 16 bytes, so that neighbouring lanes store neighbouring 16 bytes.
    template <int RUN, class Put> __device__ __forceinline__ void each_run(char* lds, int rows, int cols, Put&& f) const {
        static_assert(!SWAP && (RUN == 4 || RUN == 8), "accumulators along j");
        float* slab = reinterpret_cast<float*>(lds);
        for (int pass = 0; pass < WR; ++pass) {
            const int ib = pass * SLAB_ROWS;
            if (ib >= rows) return;
            __syncthreads();
            to_slab(slab, pass);
            __syncthreads();
            for (int e = threadIdx.x; e < SLAB_ROWS * (BN / RUN); e += THREADS) {
                const int il = e / (BN / RUN), j = e % (BN / RUN) * RUN;
                if (ib + il >= rows || j >= cols) continue;
                union { v4f w[RUN / 4]; float v[RUN]; } u;
#pragma unroll
                for (int x = 0; x < RUN / 4; ++x) u.w[x] = *reinterpret_cast<const v4f*>(slab + slab_at(il, j + 4 * x));
                f(ib + il, j, u.v);
            }
        }
    }
    // f(i, j, value pointer, count): count consecutive columns j.. of row i of the tile
    template <class Put> __device__ __forceinline__ void each(Put&& f) {
        const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, q = lane >> 4;
        const int i0 = wave / WC * (BM / WR), j0 = wave % WC * (BN / WC);
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                if constexpr (SWAP) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        one v = acc[i][j][x];
                        f(i0 + 16 * i + (sizeof(T) == 8 ? q + 4 * x : 4 * q + x), j0 + 16 * j + r, &v, std::integral_constant<int, 1>{});
                    }
                } else {
                    one v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = acc[i][j][x];
                    f(i0 + 16 * i + r, j0 + 16 * j + 4 * q, v, std::integral_constant<int, 4>{});
                }
            }
    }
};

}  // namespace mm
