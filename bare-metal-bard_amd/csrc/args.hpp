// What the entry points that return a status share in checking their
// arguments.
#pragma once

#include <stdint.h>
#include <stdio.h>

#include "../../include/nn.h"

namespace bmb {

// Prints why an entry point refuses its arguments; the caller returns -1.
inline int refuse(const char *entry, const char *why) {
    fprintf(stderr, "bmb: %s: %s\n", entry, why);
    return -1;
}

inline int element_size(int type) {
    return type == BMB_F32 ? 4 : type == BMB_F16 || type == BMB_BF16 ? 2 : 0;
}

// `rows` rows of `width` bytes, `stride` bytes apart (0 or at least width).
struct Rows {
    const void *p;
    long long stride, width;
};

// Whether a byte of one lies in the other. Rows of one stride may lie side by
// side (column ranges of one buffer); of two strides, one has to end before
// the other begins.
inline bool overlap(const Rows &a, const Rows &b, long long rows) {
    if (a.p == nullptr || b.p == nullptr || rows < 1) return false;
    const unsigned __int128 pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    const auto end = [&](unsigned __int128 p, const Rows &r) {
        return p + (unsigned __int128)(rows - 1) * r.stride + r.width;
    };
    if (end(pa, a) <= pb || end(pb, b) <= pa) return false;
    if (a.stride != b.stride || a.stride == 0 || rows == 1) return true;
    const long long d = (long long)((pb > pa ? pb - pa : pa - pb) % a.stride);
    const long long first = pb > pa ? a.width : b.width;
    const long long second = pb > pa ? b.width : a.width;
    return d < first || d + second > a.stride;
}

// The same rows: in place.
inline bool same(const Rows &a, const Rows &b, long long rows) {
    return a.p == b.p && a.width == b.width && (a.stride == b.stride || rows == 1);
}

}  // namespace bmb
