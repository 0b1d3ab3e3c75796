// Host-side checks of strided tensors at an entry point: outputs have a place of their own for every element and share memory with no other
// tensor of the call.
#pragma once
#include "common.h"

namespace xrl {

struct arg_t {
    const char* name;
    const void* p;                 // NULL: not given
    int bytes, dims;               // of an element; of the shape
    int64_t n[5], s[5];            // sizes and strides in elements, outermost first
    bool out;
};

static inline int64_t arg_span(const arg_t& a, int from) {
    int64_t v = 1;
    for (int i = from; i < a.dims; ++i) v += (a.n[i] - 1) * a.s[i];
    return v;
}
static inline bool arg_empty(const arg_t& a) {
    if (!a.p) return true;
    for (int i = 0; i < a.dims; ++i) if (a.n[i] == 0) return true;
    return false;
}

// strides, smallest first, each pass what the ones below it span
static inline bool arg_injective(const arg_t& a) {
    bool used[5] = {false, false, false, false, false};
    int64_t span = 1;
    for (;;) {
        int k = -1;
        for (int i = 0; i < a.dims; ++i)
            if (!used[i] && a.n[i] > 1 && (k < 0 || a.s[i] < a.s[k])) k = i;
        if (k < 0) return true;
        if (a.s[k] < span) return false;
        span += a.s[k] * (a.n[k] - 1);
        used[k] = true;
    }
}

// the two lie in one stretch of memory without a common element: slices of one wider row, the rows at the same pitch
static inline bool arg_interleaved(const arg_t& a, const arg_t& b) {
    if (a.dims != b.dims || a.bytes != b.bytes) return false;
    const int64_t diff = reinterpret_cast<const char*>(b.p) - reinterpret_cast<const char*>(a.p);
    if (diff % a.bytes) return false;
    for (int inner = a.dims - 1; inner >= 1; --inner) {              // dimensions [inner, dims) make up a slice
        int64_t pitch = 0;
        bool same = true;
        for (int i = 0; i < inner; ++i)
            if (a.n[i] > 1 || b.n[i] > 1) {
                same = same && a.s[i] == b.s[i];
                if (pitch == 0 || a.s[i] < pitch) pitch = a.s[i];
            }
        if (!same || pitch <= 0) continue;
        for (int i = 0; i < inner; ++i)
            if ((a.n[i] > 1 || b.n[i] > 1) && a.s[i] % pitch) same = false;
        if (!same) continue;
        int64_t off = (diff / a.bytes) % pitch;
        if (off < 0) off += pitch;
        if (off >= arg_span(a, inner) && off + arg_span(b, inner) <= pitch) return true;
    }
    return false;
}

static inline bool arg_same(const arg_t& a, const arg_t& b) {
    if (a.p != b.p || a.dims != b.dims || a.bytes != b.bytes) return false;
    for (int i = 0; i < a.dims; ++i)
        if (a.n[i] != b.n[i] || (a.n[i] > 1 && a.s[i] != b.s[i])) return false;
    return true;
}

// pairs: indices of an output and of the one other tensor that it may be
static inline int check_args(const arg_t* a, int count, const int (*pairs)[2], int n_pairs) {
    for (int i = 0; i < count; ++i) {
        if (arg_empty(a[i])) continue;
        for (int d = 0; d < a[i].dims; ++d)
            if (a[i].s[d] < 0) { set_error("invalid argument: negative strides of %s", a[i].name); return XRL_EINVAL; }
    }
    for (int i = 0; i < count; ++i) {
        if (!a[i].out || arg_empty(a[i])) continue;
        if (!arg_injective(a[i])) { set_error("invalid argument: elements of the output %s share memory", a[i].name); return XRL_EINVAL; }
        const char* lo = reinterpret_cast<const char*>(a[i].p);
        const char* hi = lo + arg_span(a[i], 0) * a[i].bytes;
        for (int j = 0; j < count; ++j) {
            if (j == i || (a[j].out && j < i) || arg_empty(a[j])) continue;
            const char* l2 = reinterpret_cast<const char*>(a[j].p);
            const char* h2 = l2 + arg_span(a[j], 0) * a[j].bytes;
            if (h2 <= lo || hi <= l2 || arg_interleaved(a[i], a[j])) continue;
            bool fine = false;
            for (int k = 0; k < n_pairs; ++k) fine = fine || (pairs[k][0] == i && pairs[k][1] == j && arg_same(a[i], a[j]));
            if (!fine) { set_error("invalid argument: %s and %s share memory", a[i].name, a[j].name); return XRL_EINVAL; }
        }
    }
    return XRL_OK;
}

}  // namespace xrl
