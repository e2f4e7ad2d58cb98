// gpx_share_bytes against sets of bytes: never "shared" where no byte is, and always where the strides are equal.
#include <cstdio>
#include <cstdlib>
#include <set>
#include "../../gp_amd/csrc/byte_rows.h"

static std::set<long> bytes(const ByteRows& m) {
    std::set<long> s;
    for (long i = 0; i < m.mats; ++i)
        for (long r = 0; r < m.rows; ++r)
            for (long c = 0; c < m.width; ++c) s.insert((long)m.base + i * m.stride + r * m.ld + c);
    return s;
}
static bool meet(const ByteRows& a, const ByteRows& b) {
    const auto s = bytes(a), t = bytes(b);
    for (long v : s)
        if (t.count(v)) return true;
    return false;
}

int main() {
    srand(3);
    auto up_to = [](int n) { return rand() % (n + 1); };
    long shared = 0, apart = 0, missed = 0;
    for (int n = 0; n < 60000; ++n) {
        const long ld = 1 + up_to(11), stride = ld * (1 + up_to(5));
        ByteRows m[2];
        for (auto& v : m) {
            v.ld = n % 4 == 3 ? 1 + up_to(11) : ld;
            v.width = up_to((int)v.ld);
            v.rows = n % 2 ? 1 + up_to(5) : 1 + up_to((int)(stride / ld) - 1);
            v.mats = n % 3 ? 1 : 1 + up_to(3);
            v.stride = n % 2 ? up_to(40) : stride;
            v.base = reinterpret_cast<const void*>(1000L + up_to(120));
        }
        const bool real = meet(m[0], m[1]), said = gpx_share_bytes(m[0], m[1]);
        (real ? shared : apart)++;
        const bool fits = n % 4 != 3 && n % 2 == 0;   // equal strides, matrices that end before the next
        if (said != gpx_share_bytes(m[1], m[0]) || (fits ? said != real : n % 2 == 0 && said && !real)) {
            printf("case %d: shares %d, said %d\n", n, real, said);
            for (auto& v : m) printf("  base %ld mats %ld stride %ld rows %ld ld %ld width %ld\n", (long)v.base, (long)v.mats, (long)v.stride, (long)v.rows, (long)v.ld, (long)v.width);
            return 1;
        }
        // any strides: nothing apart is refused where the matrices of a stack end before the next
        auto ordered = [](const ByteRows& v) { return v.mats == 1 || v.stride == 0 || v.stride >= (v.rows - 1) * v.ld + v.width; };
        if (said && !real && ordered(m[0]) && ordered(m[1])) {
            printf("case %d refused\n", n);
            return 1;
        }
        missed += real && !said;
    }
    printf("shared %ld apart %ld missed %ld\n", shared, apart, missed);
    return shared > 5000 && apart > 5000 ? 0 : 1;
}
