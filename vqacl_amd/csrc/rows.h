// Host side: what a call is refused for before it is launched.
#pragma once

#define VLT5_MOST_THREADS 0xffffffffLL                   // of a grid in one dimension: the runtime counts them in 32 bits

// Do two sets of rows share a byte?  Asked where an output over an input would let one workgroup write what another has yet to read.
// n rows of `width` bytes, `stride` bytes apart (of one row the stride does not matter); rows of one set do not overlap each other
struct RowSpan {
    const void* at; long long n, stride, width;
};
static inline bool vlt5_rows_overlap(RowSpan a, RowSpan b) {
    typedef __int128 wide_t;                                                   // (the strides are a caller's)
    if (!a.at || !b.at || a.n <= 0 || b.n <= 0) return false;
    if (a.n == 1) a.stride = b.n == 1 ? a.width + b.width : b.stride;
    if (b.n == 1) b.stride = a.stride;
    const wide_t pa = (wide_t)(uintptr_t)a.at, pb = (wide_t)(uintptr_t)b.at;
    if (pa + (wide_t)(a.n - 1) * a.stride + a.width <= pb || pb + (wide_t)(b.n - 1) * b.stride + b.width <= pa) return false;
    if (a.stride == b.stride) {                                                // slices of one buffer: row i of a and row i + k of b are d + k * stride apart
        const wide_t d = pb - pa, s = a.stride, low = -d - b.width;            // the smallest k with d + k * stride > -b.width
        wide_t k = low / s - (low % s < 0) + 1;
        if (k < 1 - (wide_t)a.n) k = 1 - (wide_t)a.n;
        return k < b.n && d + k * s < a.width;
    }
    long long i = 0, j = 0;
    while (i < a.n && j < b.n) {
        const wide_t x = pa + (wide_t)i * a.stride, y = pb + (wide_t)j * b.stride;
        if (x + a.width <= y) ++i;
        else if (y + b.width <= x) ++j;
        else return true;
    }
    return false;
}
