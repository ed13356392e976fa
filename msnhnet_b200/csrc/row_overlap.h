// Whether rows that a call writes share memory, with each other or with rows of another tensor: [n][m] rows of `width` bytes with a stride for each
// of the two. Exact for any strides; where rows lie as usual, a few divisions.
#pragma once
#include <algorithm>
#include <cstdint>
#include <utility>

namespace msnh {

using Wide = __int128;                                           // (strides times counts of a caller may pass 64 bits)

struct Rows {
    int64_t n, m, n_step, m_step;                                // counts, strides in bytes
    int64_t width;
    // (a stride that no second row uses does not count)
    Rows(int64_t n_, int64_t m_, int64_t n_step_, int64_t m_step_, int64_t width_) : n(n_), m(m_), n_step(n_ > 1 ? n_step_ : 0), m_step(m_ > 1 ? m_step_ : 0), width(width_) {}
    Wide span() const { return static_cast<Wide>(n - 1) * n_step + static_cast<Wide>(m - 1) * m_step + width; }
};

inline Wide floor_div(Wide a, Wide b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); }

// Whether |at + i * n_step + j * m_step| < r's width for an i of [n_low, n_high] and a j of [m_low, m_high].
inline bool reaches(Wide at, const Rows &r, Wide n_low, Wide n_high, Wide m_low, Wide m_high) {
    Wide step = r.n_step, low = n_low, high = n_high, far = r.m_step, from = m_low, to = m_high;
    if (step > far) {
        std::swap(step, far);
        std::swap(low, from);
        std::swap(high, to);
    }
    if (low > high || from > to) return false;
    // by the larger stride to what the smaller one can bridge
    if (far > 0) {
        from = std::max(from, floor_div(-r.width - at - high * step, far) + 1);
        to = std::min(to, -floor_div(at + low * step - r.width, far) - 1);
    } else {
        to = from;
    }
    for (Wide j = from; j <= to; ++j) {
        const Wide rest = at + j * far;
        const Wide first = step > 0 ? std::max(low, floor_div(-r.width - rest, step) + 1) : low, last = step > 0 ? std::min(high, -floor_div(rest - r.width, step) - 1) : low;
        if (first <= last && (step > 0 || (rest < r.width && rest > -r.width))) return true;
    }
    return false;
}

// Whether two of the rows share a byte. (Strides below 0 are not looked at: they overlap by definition here.)
inline bool rows_overlap(const Rows &r) {
    if (r.n < 1 || r.m < 1) return false;
    if (r.n_step < 0 || r.m_step < 0) return true;
    // one side's rows behind one another, the other side's steps beyond them: as outputs lie mostly
    const bool n_outer = r.n_step >= r.m_step;
    const int64_t step = n_outer ? r.m_step : r.n_step, many = n_outer ? r.m : r.n, far = n_outer ? r.n_step : r.m_step, others = n_outer ? r.n : r.m;
    if ((many == 1 || step >= r.width) && (others == 1 || far >= static_cast<Wide>(many - 1) * step + r.width)) return false;
    return reaches(0, r, 1, r.n - 1, 1 - r.m, r.m - 1) || reaches(0, r, 0, 0, 1, r.m - 1);
}

// Whether a row of `a` at address a_at shares a byte with one of `b` at b_at (of the same counts and width).
inline bool rows_meet(const void *a_at, const Rows &a, const void *b_at, const Rows &b) {
    if (a.n < 1 || a.m < 1) return false;
    const Wide apart = static_cast<Wide>(reinterpret_cast<uintptr_t>(b_at)) - static_cast<Wide>(reinterpret_cast<uintptr_t>(a_at));
    if (apart >= a.span() || -apart >= b.span()) return false;
    if (a.n_step == b.n_step && a.m_step == b.m_step) return reaches(apart, a, 1 - a.n, a.n - 1, 1 - a.m, a.m - 1);
    for (int64_t i = 0; i < a.n; ++i)
        for (int64_t j = 0; j < a.m; ++j)
            if (reaches(apart - static_cast<Wide>(i) * a.n_step - static_cast<Wide>(j) * a.m_step, b, 0, b.n - 1, 0, b.m - 1)) return true;
    return false;
}

}  // namespace msnh
