// Host-side checks of arguments: do two strided stacks of matrices share elements?
#pragma once
#include <stdint.h>

struct MatRange {                     // count matrices [rows][cols] of `size`-byte elements, row pitch ld, matrix stride `stride` (elements)
    uintptr_t at;
    int size;
    long stride, ld;
    int count; long rows; int cols;
    bool write; int item;
    long span() const { return (rows - 1) * ld + cols; }                                          // elements of one matrix, first to last
    uintptr_t end() const { return at + (uintptr_t)((count - 1) * stride + span()) * size; }
};

// May a and b share an element?  Exact for disjoint address ranges, for column blocks of one matrix (equal pitch, strides a multiple of it) and for
// stacks interleaved with one stride (the matrices of a block in one arena); other layouts whose ranges overlap count as shared.
inline bool ranges_meet(const MatRange& x, const MatRange& y) {
    const MatRange &a = x.at <= y.at ? x : y, &b = x.at <= y.at ? y : x;
    if (a.end() <= b.at) return false;
    const uintptr_t bytes = b.at - a.at;
    if (a.size != b.size || bytes % a.size) return true;
    const long delta = (long)(bytes / a.size);
    const bool by_rows_a = a.count == 1 || (a.ld > 0 && a.stride % a.ld == 0), by_rows_b = b.count == 1 || (b.ld > 0 && b.stride % b.ld == 0);
    if (a.ld == b.ld && a.ld > 0 && by_rows_a && by_rows_b) {
        const long c = delta % a.ld;
        if (c >= a.cols && c + b.cols <= a.ld) return false;
    }
    const long s = a.count > 1 ? a.stride : b.stride;
    if ((a.count > 1 || b.count > 1) && (b.count == 1 || b.stride == s) && s > 0) {
        const long d = delta % s;
        if (d >= a.span() && d + b.span() <= s) return false;
    }
    return true;
}

struct FlatRange { uintptr_t at; size_t bytes; };
inline bool ranges_meet(const FlatRange& x, const FlatRange& y) { return x.at < y.at + y.bytes && y.at < x.at + x.bytes; }
// One matrix and a contiguous piece of memory: exact, what lies between the rows is not the matrix's.
inline bool ranges_meet(const MatRange& m, const FlatRange& f) {
    if (f.at + f.bytes <= m.at || f.at >= m.end()) return false;
    if (f.at < m.at) return true;
    const size_t pitch = (size_t)m.ld * m.size, off = (f.at - m.at) % pitch;
    return off < (size_t)m.cols * m.size || off + f.bytes > pitch;
}
