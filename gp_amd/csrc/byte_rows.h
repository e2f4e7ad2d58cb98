// byte_rows.h — host code: whether two strided operands of one call overlap.
#pragma once
#include <cstdint>
#include <initializer_list>

// Rows of a matrix or of a stack of them, in bytes: `width` bytes at base + m*stride + r*ld, m < mats, r < rows.
struct ByteRows {
    const void* base;
    int64_t mats, stride, rows, ld, width;
};
// Whether they reach less than 2^60 bytes from `base` on, so that no address of theirs wraps.
static inline bool gpx_reaches(const ByteRows& m) {
    return m.mats <= 0 || m.rows <= 0 || (m.mats - 1.0) * m.stride + (m.rows - 1.0) * m.ld + m.width < 0x1p60;
}
// Whether two of them, which do, are seen to share bytes.  Columns beside one another of one larger matrix do not, nor do row blocks beside one
// another of every matrix of a stack; where two leading dimensions or strides differ, only the
// first rows and ranges without gaps are judged.
static inline bool gpx_share_bytes(ByteRows a, ByteRows b) {
    if (a.mats <= 0 || a.rows <= 0 || a.width <= 0 || b.mats <= 0 || b.rows <= 0 || b.width <= 0) return false;
    if (a.stride == 0) a.mats = 1;
    if (b.stride == 0) b.mats = 1;
    if (a.mats == 1 || b.mats == 1 || a.stride != b.stride)   // a stack that is one matrix
        for (ByteRows* m : {&a, &b})
            if (m->mats > 1 && m->rows * m->ld == m->stride) {
                m->rows *= m->mats;
                m->mats = 1;
            }
    auto extent = [](const ByteRows& m) { return (m.rows - 1) * m.ld + m.width; };
    const int64_t ea = extent(a), eb = extent(b);
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.base), b0 = reinterpret_cast<uintptr_t>(b.base);
    if (a0 + (a.mats - 1) * a.stride + ea <= b0 || b0 + (b.mats - 1) * b.stride + eb <= a0) return false;
    const int64_t all = (int64_t)(b0 - a0);
    if (all < a.width && -all < b.width) return true;   // their first rows
    auto gapless = [](const ByteRows& m) { return m.rows == 1 || m.ld <= m.width; };
    auto one = [&](int64_t d) {   // one matrix of a, and one of b that begins d bytes behind it
        if (d >= ea || -d >= eb) return false;
        if (gapless(a) && gapless(b)) return true;
        const int64_t ld = a.rows > 1 ? a.ld : b.ld;
        if ((b.rows > 1 && b.ld != ld) || a.width > ld || b.width > ld) return false;
        const int64_t c = (d % ld + ld) % ld;
        return c < a.width || c + b.width > ld;
    };
    if (a.mats == 1 && b.mats == 1) return one(all);
    const int64_t s = a.mats > 1 ? a.stride : b.stride;
    if ((b.mats > 1 && b.stride != s) || ea > s || eb > s) return false;
    // matrix i of a and j of b are all + (j - i) s apart: the two such distances that their extents allow, if there are such i and j
    const int64_t d = (all % s + s) % s, k = (d - all) / s;
    auto exist = [&](int64_t k) { return k < b.mats && -k < a.mats; };
    return (exist(k) && one(d)) || (exist(k - 1) && one(d - s));
}
