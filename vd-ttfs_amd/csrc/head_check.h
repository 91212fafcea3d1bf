// Argument checks, sizes and scratch shared by the entry points of the heads.
#pragma once

#include "head.h"

namespace vdttfs {

constexpr int kMaxTopK = 64, kMaxGroups = 64;
constexpr int64_t kMaxRows = 0x7fffffff;

inline int bad(const char* what, const char* why) { return set_error(VDTTFS_E_INVALID, "%s: %s", what, why); }

inline size_t elem_size(int elem) { return elem == VDTTFS_ELEM_BF16 || elem == VDTTFS_ELEM_F16 ? 2 : 4; }

inline int check_float_ptr(const char* what, const void* p, size_t align) {
    if (!p) return bad(what, "null buffer");
    if ((uintptr_t)p % align) return bad(what, "a float buffer is not aligned to its type");
    return VDTTFS_OK;
}

inline int check_in(const char* what, const void* x, int elem, int64_t ldx, int64_t rows, int cols) {
    if (elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_TIMES) return bad(what, "unknown input element type");
    if (rows < 0 || cols < 0) return bad(what, "negative size");
    if (rows > kMaxRows) return set_error(VDTTFS_E_UNSUPPORTED, "%s: 2^31 rows or more", what);
    if (ldx < cols) return bad(what, "leading dimension below the columns");
    if (rows > 0 && cols > 0) VD_TRY(check_float_ptr(what, x, elem_size(elem)));
    return VDTTFS_OK;
}

inline int check_out(const char* what, const void* out, int elem, int64_t ldo, int N) {
    if (elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_F16) return bad(what, "unknown output element type");
    if (ldo < N) return bad(what, "leading dimension below the columns");
    return check_float_ptr(what, out, elem_size(elem));
}

inline int check_channels(const char* what, int N) {
    if (N > VDTTFS_I8_MAX_N)
        return set_error(VDTTFS_E_UNSUPPORTED, "%s: %d output channels, at most %d", what, N, VDTTFS_I8_MAX_N);
    return VDTTFS_OK;
}

inline int check_mnk(const char* what, int64_t M, int N, int K) {
    if (M < 0 || N < 0 || K < 0) return bad(what, "negative size");
    if (M > kMaxRows) return set_error(VDTTFS_E_UNSUPPORTED, "%s: 2^31 rows or more", what);
    return check_channels(what, N);
}

// The context's scratch of these calls, at least `bytes`; a buffer whose
// address a captured graph holds is set aside until the context ends.
int head_scratch(vdttfs_ctx* ctx, size_t bytes, unsigned char** out);

// Parts of one scratch buffer, each on a 256-byte boundary.
struct Layout {
    size_t bytes = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) & ~size_t(255);
        return at;
    }
};

}  // namespace vdttfs
