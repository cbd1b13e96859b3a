// Checks that the C ABI calls of the caches share (kv4.cpp, paged.cpp): extents of rows,
// buffers that a call writes, and the device that its kernels are launched on.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "vx_internal.h"

namespace vx {

// Kernels are launched with the context's device current; the caller's is put back.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        int now = device;
        if (hipGetDevice(&now) != hipSuccess) (void)hipGetLastError();
        if (now == device) return;
        was_ = now;
        (void)hipSetDevice(device);
    }
    ~OnDevice() {
        if (was_ >= 0) (void)hipSetDevice(was_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

  private:
    int was_ = -1;
};

// The end, in bytes, of `rows` rows of `width` floats at `base`: 2^38 rows of stride 2^32 need
// more than 64 bits, and count as more than any buffer holds.
inline uint64_t rows_end(uint64_t rows, uint32_t stride, uint32_t base, uint32_t width) {
    const unsigned __int128 end = ((unsigned __int128)(rows - 1u) * stride + base + width) * 4u;
    return end >> 64 ? UINT64_MAX : (uint64_t)end;
}

inline int check_rows(const vx_buf *b, uint64_t rows, uint32_t stride, uint32_t base, uint32_t width, const char *what) {
    if (stride < width) return fail(VX_ERR_SHAPE, "%s: stride %u is less than a row of %u", what, stride, width);
    return need_buf(b, rows_end(rows, stride, base, width), what);
}

inline bool aligned(uint32_t stride, uint32_t base) { return stride % 4u == 0 && base % 4u == 0; }

// Bytes [a, a_end) of one buffer and [b, b_end) of another share memory.
inline bool overlap(const vx_buf *x, uint64_t a, uint64_t a_end, const vx_buf *y, uint64_t b, uint64_t b_end) {
    const char *p = static_cast<const char *>(x->ptr), *q = static_cast<const char *>(y->ptr);
    return p + a < q + b_end && q + b < p + a_end;
}

// A buffer that a call writes, nullable ones among them, may share memory with no other of it:
// other workgroups read that, or write it.
inline int check_apart(const char *what, std::initializer_list<const vx_buf *> written,
                       std::initializer_list<const vx_buf *> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        if (!*w) continue;
        auto shares = [&](const vx_buf *b) { return b && overlap(*w, 0, (*w)->bytes, b, 0, b->bytes); };
        if (std::any_of(w + 1, written.end(), shares) || std::any_of(read.begin(), read.end(), shares))
            return fail(VX_ERR_INVALID_ARG, "%s: a buffer that is written is bound twice", what);
    }
    return VX_OK;
}

// Rows of two operands, where one is written: apart as a whole, or of one stride and side by side.
inline int check_rows_apart(const char *what, const vx_buf *x, uint32_t x_stride, uint32_t x_base, const vx_buf *y,
                            uint32_t y_stride, uint32_t y_base, uint64_t rows, uint32_t width) {
    if (!overlap(x, 4ull * x_base, rows_end(rows, x_stride, x_base, width), y, 4ull * y_base,
                 rows_end(rows, y_stride, y_base, width)))
        return VX_OK;
    if (x_stride == y_stride) {
        const int64_t stride = 4ll * x_stride, wide = 4ll * width;
        const int64_t off = (static_cast<const char *>(y->ptr) - static_cast<const char *>(x->ptr) + 4ll * y_base - 4ll * x_base) % stride;
        const int64_t ahead = off < 0 ? off + stride : off;   // of the next row of y from a row of x
        if (ahead >= wide && stride - ahead >= wide) return VX_OK;
    }
    return fail(VX_ERR_INVALID_ARG, "%s overlap", what);
}

}  // namespace vx
