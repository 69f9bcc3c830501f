// okf_args.h -- checks of arguments that the entry points of attention, the cache and
// the layers around them share.
#pragma once
#include "okf_impl.h"

namespace okf_impl {

inline bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }

inline bool attn_type(int32_t t) { return t == F32 || t == F16 || t == BF16; }

// Runs f with a value of the element type t (attn_type).
template <class Fn>
void with_type(int32_t t, Fn f) {
    if (t == F32) f(float{});
    else if (t == F16) f(_Float16{});
    else f(__bf16{});
}

inline bool good_dim(uint32_t d) { return d >= 16 && d <= 256 && d % 16 == 0; }

// A row stride of 16-byte rows: `least` values when 0, else at least that and whole 16 bytes.
inline bool row_stride(uint64_t &st, uint64_t least, uint32_t size) {
    if (!st) st = least;
    return st >= least && st <= (1ull << 40) && st * size % 16 == 0;
}

// Whether `na` rows of `la` bytes, `sa` bytes apart, surely share no memory with `nb` rows of `lb`
// bytes, `sb` apart: apart as a whole, or as columns of rows of one stride.
inline bool rows_apart(const void *a, uint64_t sa, uint64_t la, uint64_t na, const void *b, uint64_t sb, uint64_t lb, uint64_t nb) {
    typedef unsigned __int128 wide;  // (rows and strides at their limits leave 64 bits)
    const uint64_t pa = (uint64_t)(uintptr_t)a, pb = (uint64_t)(uintptr_t)b;
    if (!na || !nb || pa + (wide)(na - 1) * sa + la <= pb || pb + (wide)(nb - 1) * sb + lb <= pa) return true;
    if (sa != sb) return false;
    const uint64_t d = pb >= pa ? (pb - pa) % sa : (sa - (pa - pb) % sa) % sa;
    return la <= d && d + lb <= sa;
}

}  // namespace okf_impl
