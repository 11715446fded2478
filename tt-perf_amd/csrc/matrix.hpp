// matrix.hpp — the operators' checks of the matrices and arrays they are given.
#pragma once

#include <stdint.h>

#include <string>

#include "context.hpp"

namespace ttpi {

inline uint64_t elem_size(int dtype) { return dtype == TTP_DTYPE_BF16 ? 2 : 4; }

// A matrix's own fields (its shape is the caller's to compare).
inline int check_matrix(const ttp_matrix* m, const char* what) {
    const std::string name(what);
    if (!m) return fail(TTP_ERR_INVALID, name + ": null matrix");
    if (m->dtype != TTP_DTYPE_F32 && m->dtype != TTP_DTYPE_BF16)
        return fail(TTP_ERR_INVALID, name + ": dtype must be TTP_DTYPE_F32 or TTP_DTYPE_BF16");
    if (m->reserved) return fail(TTP_ERR_INVALID, name + ": reserved must be 0");
    if (!m->cols || m->cols >= (1ull << 31))
        return fail(TTP_ERR_RANGE, name + ": " + std::to_string(m->cols) +
                                       " columns; 1 to 2^31 - 1 are allowed");
    if (m->rows >= (1ull << 31))
        return fail(TTP_ERR_RANGE, name + ": " + std::to_string(m->rows) +
                                       " rows; at most 2^31 - 1 are allowed");
    if (m->stride < m->cols || m->stride >= (1ull << 32))
        return fail(TTP_ERR_RANGE, name + ": a row stride of " + std::to_string(m->stride) +
                                       " elements for " + std::to_string(m->cols) +
                                       " columns (at least those, less than 2^32)");
    return TTP_OK;
}

// What a call reads and writes, checked one by one as it is added, and against each other: what
// it writes overlaps nothing else of the call (but for a result in its input's place).
class Buffers {
  public:
    explicit Buffers(const ttp_ctx* c) : c_(c) {}

    // an array of n elements of `size` bytes
    int array(const void* p, uint64_t n, uint64_t size, const char* what, bool written) {
        if ((uintptr_t)p % size) return misaligned(what);
        const int rc = device_buffer(c_, p, n * size, what, &seen_);
        if (rc) return rc;
        return add({(uintptr_t)p, n * size, n * size, n * size, written, false, what});
    }

    // a matrix of `rows` x `cols`; it may be exactly `same_as` (a result in its input's place)
    int matrix(const ttp_matrix* m, uint64_t rows, uint64_t cols, const char* what, bool written,
               const ttp_matrix* same_as = nullptr) {
        const int rc0 = check_matrix(m, what);
        if (rc0) return rc0;
        if (m->rows != rows || m->cols != cols)
            return fail(TTP_ERR_RANGE, std::string(what) + " is " + std::to_string(m->rows) +
                                           " x " + std::to_string(m->cols) + ", not " +
                                           std::to_string(rows) + " x " + std::to_string(cols));
        const uint64_t size = elem_size(m->dtype);
        if ((uintptr_t)m->data % size) return misaligned(what);
        const uint64_t bytes = rows ? ((rows - 1) * m->stride + cols) * size : 0;
        const int rc = device_buffer(c_, m->data, bytes, what, &seen_);
        if (rc) return rc;
        const bool in_place = same_as && m->data == same_as->data &&
                              m->stride == same_as->stride && m->dtype == same_as->dtype;
        return add({(uintptr_t)m->data, bytes, m->stride * size, cols * size, written, in_place,
                    what});
    }

  private:
    struct Span {
        uintptr_t at;
        uint64_t bytes, pitch, width;  // of the whole, from row to row, of a row
        bool written, in_place;
        const char* what;
    };

    static int misaligned(const char* what) {
        return fail(TTP_ERR_INVALID, std::string(what) + " is not aligned to its elements");
    }

    static bool overlap(const Span& a, const Span& b) {
        if (!a.bytes || !b.bytes || a.at + a.bytes <= b.at || b.at + b.bytes <= a.at) return false;
        if (a.pitch == b.pitch) {  // columns of one wider matrix, side by side
            const int64_t pitch = (int64_t)a.pitch;
            const uint64_t d = (uint64_t)((((int64_t)(b.at - a.at)) % pitch + pitch) % pitch);
            if (d >= a.width && d + b.width <= a.pitch) return false;
        }
        return true;
    }

    int add(const Span& s) {
        for (int k = 0; k < n_; ++k) {
            const Span& o = spans_[k];
            if (!(s.written || o.written) || !overlap(s, o)) continue;
            if (s.in_place && !o.written && s.at == o.at && s.bytes == o.bytes) continue;
            return fail(TTP_ERR_INVALID, std::string(s.what) + " overlaps " + o.what);
        }
        if (n_ < kMax) spans_[n_++] = s;
        return TTP_OK;
    }

    static constexpr int kMax = 12;  // no call has more
    const ttp_ctx* c_;
    SeenAlloc seen_;
    Span spans_[kMax];
    int n_ = 0;
};

}  // namespace ttpi
