// What the C ABI's files share: checks of arguments, and a caller's workspace cut into its parts.
#pragma once
#include "../../include/int4linear.h"

#include <cstddef>
#include <cstdint>

namespace int4linear {

// Row and column numbers are 32-bit in the kernels, rounded up to tiles; offsets are 64-bit.
constexpr int kMostRows = 1 << 30;

inline bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
inline bool is_type(int type) { return type == INT4LINEAR_OUT_F32 || type == INT4LINEAR_OUT_F16 || type == INT4LINEAR_OUT_BF16; }
inline size_t type_bytes(int type) { return type == INT4LINEAR_OUT_F32 ? 4 : 2; }

// A status for the first of some checks that fails.
struct Checks {
    int status = INT4LINEAR_OK;
    Checks &that(bool ok, int otherwise)
    {
        if (status == INT4LINEAR_OK && !ok)
            status = otherwise;
        return *this;
    }
    Checks &sizes(int a, int b, int c)
    {
        that(a >= 0 && b >= 0 && c >= 0, INT4LINEAR_ERR_SHAPE);
        return that(a <= kMostRows && b <= kMostRows && c <= kMostRows, INT4LINEAR_ERR_UNSUPPORTED);
    }
    // Elements between rows of `columns`.  (A negative number given as size_t is beyond all memory: rows would lie in front of the array.)
    Checks &apart(size_t ld, int columns)
    {
        return that(ld >= (size_t)(columns > 0 ? columns : 0) && ld <= (size_t)1 << 48, INT4LINEAR_ERR_SHAPE);
    }
    // An array the call reads or writes; `used`: it has elements.
    Checks &array(const void *p, size_t alignment, bool used)
    {
        that(!used || p, INT4LINEAR_ERR_NULL);
        return that(!used || aligned(p, alignment), INT4LINEAR_ERR_ALIGN);
    }
    Checks &optional(const void *p, size_t alignment) { return that(!p || aligned(p, alignment), INT4LINEAR_ERR_ALIGN); }
    Checks &matrix(const void *codes, const void *scales, int rows, int k)
    {
        array(codes, 16, rows > 0 && k > 0);
        return array(scales, 16, rows > 0 && k > 0);
    }
    explicit operator bool() const { return status == INT4LINEAR_OK; }
};

inline size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// The caller's workspace, handed out part by part in steps of 256 bytes; with a null base it only counts.
struct Parts {
    uint8_t *base;
    size_t used = 0;
    template <class T>
    T *take(size_t count)
    {
        T *p = base ? (T *)(base + used) : nullptr;
        used += up(count * sizeof(T), 256);
        return p;
    }
};

}  // namespace int4linear
