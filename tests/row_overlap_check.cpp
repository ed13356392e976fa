// Rows that share memory (row_overlap.h) against a look at every pair of rows, over random layouts. Exit code 0: the same throughout, and both answers came up.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "../msnhnet_b200/csrc/row_overlap.h"

using namespace msnh;

static std::vector<int64_t> places(int64_t at, const Rows &r) {
    std::vector<int64_t> all;
    for (int64_t i = 0; i < r.n; ++i)
        for (int64_t j = 0; j < r.m; ++j) all.push_back(at + i * r.n_step + j * r.m_step);
    return all;
}

int main(int argc, char **argv) {
    std::mt19937 rng(argc > 1 ? std::atoi(argv[1]) : 1);
    const auto pick = [&](int low, int high) { return static_cast<int64_t>(std::uniform_int_distribution<int>(low, high)(rng)); };
    long alone[2] = {0, 0}, meet[2] = {0, 0};
    for (int k = 0; k < 300000; ++k) {
        const int64_t width = pick(1, 6), n = pick(0, 5), m = pick(0, 5);
        const int most = k % 2 ? 12 : 40;
        const Rows a(n, m, pick(0, most), pick(0, most), width), b = k % 3 ? a : Rows(n, m, pick(0, most), pick(0, most), width);
        const int64_t apart = pick(-90, 90);
        const auto pa = places(1000, a), pb = places(1000 + apart, b);
        bool own = false, both = false;
        for (size_t x = 0; x < pa.size(); ++x) {
            for (size_t y = 0; y < x; ++y) own |= std::abs(pa[x] - pa[y]) < width;
            for (size_t y = 0; y < pb.size(); ++y) both |= std::abs(pa[x] - pb[y]) < width;
        }
        if (rows_overlap(a) != own || rows_meet(reinterpret_cast<void *>(1000), a, reinterpret_cast<void *>(1000 + apart), b) != both) {
            std::printf("%ld x %ld rows of %ld, strides %ld %ld and %ld %ld, %ld apart: wrong\n", long(n), long(m), long(width), long(a.n_step), long(a.m_step), long(b.n_step), long(b.m_step), long(apart));
            return 1;
        }
        ++alone[own];
        ++meet[both];
    }
    // sizes whose products pass 64 bits
    const int64_t huge = int64_t(1) << 62;
    if (rows_overlap(Rows(huge, huge, huge, 1, huge)) != true || rows_overlap(Rows(3, 1 << 30, huge, 4096, 4096)) || rows_overlap(Rows(3, 2, 4096, huge, 4096))) return 2;
    std::printf("%ld %ld %ld %ld\n", alone[0], alone[1], meet[0], meet[1]);
    return alone[0] > 1000 && alone[1] > 1000 && meet[0] > 1000 && meet[1] > 1000 ? 0 : 3;
}
