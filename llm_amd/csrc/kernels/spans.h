// spans.h -- which memory a call's operands take up, for entry points that refuse outputs over their inputs (host code).
#pragma once
#include <stdint.h>

// What a call reads or writes: n3 x n2 planes of n1 rows of `row` bytes, and the first and last byte of all that
struct Span {
    int64_t row, n1, nb1, n2, nb2, n3, nb3;
    int64_t plane, nb[2], n[2];                       // bytes from a plane's first to its last; the planes' strides, the larger one first, and numbers
    uintptr_t low, end;
    Span(const void * at, int64_t row_bytes, int64_t n1_, int64_t nb1_, int64_t n2_, int64_t nb2_, int64_t n3_, int64_t nb3_)
        : row(at ? row_bytes : 0), n1(n1_), nb1(nb1_), n2(n2_), nb2(nb2_), n3(n3_), nb3(nb3_) {
        low = (uintptr_t)at + (nb1 < 0 ? (n1 - 1) * nb1 : 0) + (nb2 < 0 ? (n2 - 1) * nb2 : 0) + (nb3 < 0 ? (n3 - 1) * nb3 : 0);
        const int64_t s2 = nb2 < 0 ? -nb2 : nb2, s3 = nb3 < 0 ? -nb3 : nb3;
        plane = (n1 - 1) * (nb1 < 0 ? -nb1 : nb1) + row;
        const int big = n2 < 2 || (n3 > 1 && s3 >= s2) ? 0 : 1;
        n[big] = n3; nb[big] = s3; n[!big] = n2; nb[!big] = s2;
        end = row > 0 && n1 > 0 ? low + (n2 - 1) * s2 + (n3 - 1) * s3 + plane : low;
    }
    // the same rows in the same order (an operand that may be worked on in place)
    bool same(const Span & o) const {
        return low == o.low && row == o.row && n1 == o.n1 && n2 == o.n2 && n3 == o.n3 && (n1 == 1 || nb1 == o.nb1) && (n2 == 1 || nb2 == o.nb2) && (n3 == 1 || nb3 == o.nb3);
    }
    // rows that share bytes with one another (an expanded tensor's), or may: strides that do not nest
    bool folds() const {
        int64_t c[3] = {n1, n2, n3}, b[3] = {nb1 < 0 ? -nb1 : nb1, nb2 < 0 ? -nb2 : nb2, nb3 < 0 ? -nb3 : nb3}, size = row;
        if (row <= 0 || n1 < 1 || n2 < 1 || n3 < 1) return false;
        for (int k = 0; k < 3; k++) {                 // the dimension of the smallest stride that is left
            int at = -1;
            for (int i = 0; i < 3; i++) if (c[i] > 1 && (at < 0 || b[i] < b[at])) at = i;
            if (at < 0) return false;
            if (b[at] < size) return true;
            size += (c[at] - 1) * b[at];
            c[at] = 1;
        }
        return false;
    }
    bool apart(const Span & o) const { return end <= o.low || o.end <= low || end == low || o.end == o.low; }
};
// Can a byte belong to both, if not apart as wholes?  Never a wrong no.  Apart plane by plane (a cache and its copy take turns in memory), or as
// rows of one pitch that lie in each other's gaps (K and V side by side); anything less regular counts as a yes
static inline bool planes_meet(const Span & a, const Span & b) {
    // of n steps of `by` bytes, the first and last that begin less than `after` bytes behind a place and end, `size` bytes on, behind it
    struct Steps {
        int64_t first, last;
        Steps(int64_t n, int64_t by, int64_t place, int64_t after, int64_t size) {
            if (by == 0) { first = 0; last = 0 < place + after && size > place ? 0 : -1; return; }
            first = place - size < 0 ? 0 : (place - size) / by + 1;
            last = place + after <= 0 ? -1 : (place + after - 1) / by < n ? (place + after - 1) / by : n - 1;
        }
    };
    const bool pitch = a.nb1 == b.nb1 && a.nb1 >= a.row && a.nb1 >= b.row;
    int left = 1 << 18;                               // steps of the search
    for (int64_t i = 0; i < a.n[0]; i++)
        for (int64_t j = 0; j < a.n[1]; j++) {
            if (--left < 0) return true;
            const int64_t lo = (int64_t)(a.low + i * a.nb[0] + j * a.nb[1] - b.low);
            const Steps k(b.n[0], b.nb[0], lo, a.plane, (b.n[1] - 1) * b.nb[1] + b.plane);
            for (int64_t x = k.first; x <= k.last; x++) {
                if (--left < 0) return true;
                const Steps l(b.n[1], b.nb[1], lo - x * b.nb[0], a.plane, b.plane);
                for (int64_t y = l.first; y <= l.last; y++) {
                    if (!pitch || --left < 0) return true;
                    const int64_t d = (x * b.nb[0] + y * b.nb[1] - lo) % a.nb1, r = d < 0 ? d + a.nb1 : d;
                    if (r < a.row || a.nb1 - r < b.row) return true;
                }
            }
        }
    return false;
}
static inline bool spans_meet(const Span & a, const Span & b) { return !a.apart(b) && planes_meet(a, b); }
