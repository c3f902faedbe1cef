// rows.hpp — whether rows of two strided buffers meet in memory, exactly: column or token slices of one buffer that lie
// beside each other do not.  Host arithmetic only, in bytes.
#pragma once

#include <stdint.h>

namespace dc {
namespace host {

// batch x seq rows of `width` bytes: row (b, t) starts at p + b * batch_stride + t * token_stride (strides >= 0).
struct Rows {
    const void *p;
    int64_t batch, seq, batch_stride, token_stride, width;
};

inline bool no_rows(const Rows &r) { return !r.p || r.batch <= 0 || r.seq <= 0 || r.width <= 0; }
inline __int128 sequence_bytes(const Rows &r) { return (__int128)(r.seq - 1) * r.token_stride + r.width; }
inline __int128 all_bytes(const Rows &r) { return (__int128)(r.batch - 1) * r.batch_stride + sequence_bytes(r); }
inline __int128 floor_div(__int128 a, __int128 b) {  // b > 0
    const __int128 q = a / b;
    return q - (a % b < 0 ? 1 : 0);
}
// The whole numbers i of [lo, hi] with -before < at + i * stride < after (stride > 0, or lo == hi).
inline void cut(__int128 at, __int128 stride, __int128 before, __int128 after, int64_t &lo, int64_t &hi) {
    if (stride <= 0) {
        if (at >= after || at <= -before) hi = lo - 1;
        return;
    }
    const __int128 first = floor_div(-before - at, stride) + 1, last = -floor_div(at - after, stride) - 1;
    if (first > lo) lo = first > hi ? hi + 1 : (int64_t)first;
    if (last < hi) hi = last < lo ? lo - 1 : (int64_t)last;
}
// Whether a row of x's sequence and one of y's, which starts `at` bytes after it, meet.
inline bool sequences_meet(const Rows &x, const Rows &y, __int128 at) {
    if (at >= sequence_bytes(x) || at <= -sequence_bytes(y)) return false;
    if (x.seq == 1 && y.seq == 1) return true;
    if (x.token_stride == y.token_stride && x.seq == y.seq) {  // by the difference of the tokens
        int64_t lo = x.token_stride ? 1 - x.seq : 0, hi = x.token_stride ? x.seq - 1 : 0;
        cut(at, x.token_stride, y.width, x.width, lo, hi);
        return lo <= hi;
    }
    __int128 a = 0, b = at;
    for (int64_t i = 0, j = 0; i < x.seq && j < y.seq;) {
        if (a + x.width <= b) ++i, a += x.token_stride;
        else if (b + y.width <= a) ++j, b += y.token_stride;
        else return true;
    }
    return false;
}

// Whether any row of x and any row of y share a byte.
inline bool rows_meet(Rows x, Rows y) {
    if (no_rows(x) || no_rows(y)) return false;
    const __int128 at = (__int128)(intptr_t)y.p - (__int128)(intptr_t)x.p;
    if (at >= all_bytes(x) || at <= -all_bytes(y)) return false;
    if (x.batch_stride == 0) x.batch = 1;
    if (y.batch_stride == 0) y.batch = 1;
    if (x.batch == y.batch && x.batch_stride == y.batch_stride) {  // by the difference of the sequences
        int64_t lo = 1 - x.batch, hi = x.batch - 1;
        cut(at, x.batch_stride, sequence_bytes(y), sequence_bytes(x), lo, hi);
        for (int64_t d = lo; d <= hi; ++d)
            if (sequences_meet(x, y, at + (__int128)d * x.batch_stride)) return true;
        return false;
    }
    for (int64_t i = 0; i < x.batch; ++i) {
        const __int128 from = at - (__int128)i * x.batch_stride;
        int64_t lo = 0, hi = y.batch - 1;
        cut(from, y.batch_stride, sequence_bytes(y), sequence_bytes(x), lo, hi);
        for (int64_t d = lo; d <= hi; ++d)
            if (sequences_meet(x, y, from + (__int128)d * y.batch_stride)) return true;
    }
    return false;
}

// Whether two of its own rows share a byte: not a buffer to write to.
inline bool rows_fold(const Rows &r) {
    if (no_rows(r)) return false;
    if (r.seq > 1 && r.token_stride < r.width) return true;
    if (r.batch == 1) return false;
    if (r.batch_stride <= 0) return true;
    int64_t lo = 1, hi = r.batch - 1;
    cut(0, r.batch_stride, sequence_bytes(r), sequence_bytes(r), lo, hi);
    for (int64_t d = lo; d <= hi; ++d)
        if (sequences_meet(r, r, (__int128)d * r.batch_stride)) return true;
    return false;
}

// Whether n bytes at p meet any row of r.
inline bool rows_meet(const void *p, int64_t n, const Rows &r) { return rows_meet(Rows{p, 1, 1, 0, 0, n}, r); }

}  // namespace host
}  // namespace dc
