// What the kernels over a paged cache share: a batch's device arrays, read so that no value in them takes an address out of
// the rows, the table or the pool (what is beyond is cut, and sets a bit of the fault word).
#pragma once
#include "../../include/fusekit_hip.h"
#include "fk_device.hpp"

namespace fk {

struct PagedArgs {
    const uint32_t* row_start;
    const uint32_t* kv_len;
    const uint32_t* table;
    uint32_t table_stride, n_seqs, rows, max_rows, max_len;
    uint32_t n_pages, page_shift, n_kv;
    uint32_t* fault;
};

// Checks a batch and a pool and makes the argument block of them (host).
fk_status paged_args(const char* what, const fk_paged_batch* batch, const fk_page_pool* pool, PagedArgs* out);

// Whether rows of `a_width` and `b_width` values that lie `a_stride` and `b_stride` apart share a byte, `rows` of each: column blocks of one wider row
// do not (host).
inline bool rows_overlap(const uint16_t* a, size_t a_stride, size_t a_width, const uint16_t* b, size_t b_stride, size_t b_width, size_t rows) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b, a1 = a0 + 2 * ((rows - 1) * a_stride + a_width), b1 = b0 + 2 * ((rows - 1) * b_stride + b_width);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a_stride != b_stride) return true;
    const uintptr_t apart = a0 < b0 ? (b0 - a0) % (2 * a_stride) : (a0 - b0) % (2 * a_stride);   // of a row's start behind the other's
    return apart < 2 * (a0 < b0 ? a_width : b_width) || apart + 2 * (a0 < b0 ? b_width : a_width) > 2 * a_stride;
}

__device__ __forceinline__ void paged_fault(const PagedArgs& b, uint32_t bit) {
    if (b.fault) __hip_atomic_fetch_or(b.fault, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sequence `i` (below n_seqs): its first new row, how many, and its positions; `bad`: the bits that its values set.
struct PagedSeq {
    uint32_t row0, rows, len, bad;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& b, uint32_t i) {
    const uint32_t s0 = b.row_start[i], s1 = b.row_start[i + 1], raw = b.kv_len[i];
    PagedSeq s;
    s.bad = 0;
    s.row0 = s0 < b.rows ? s0 : b.rows;
    const uint32_t end = s1 < b.rows ? s1 : b.rows;
    s.rows = end > s.row0 ? end - s.row0 : 0u;
    s.rows = s.rows < b.max_rows ? s.rows : b.max_rows;
    if (s1 < s0 || s1 - s0 != s.rows) s.bad |= FK_PAGED_BAD_ROWS;
    s.len = raw < b.max_len ? raw : b.max_len;
    if (s.rows && (raw > b.max_len || raw < s.rows)) s.bad |= FK_PAGED_BAD_LENGTH;
    return s;
}

// The sequence that row `row` belongs to, or n_seqs: the number of ends at or below it, 64 of them with one request.  All of
// a wave's lanes call it with the same row.  (Starts that fall are found where the sequence is read.)
__device__ __forceinline__ uint32_t paged_seq_of(const PagedArgs& b, uint32_t row, uint32_t lane) {
    for (uint32_t at = 0; at < b.n_seqs; at += kWave) {
        const uint32_t i = at + lane < b.n_seqs ? at + lane : b.n_seqs - 1u;
        const unsigned long long below = __builtin_amdgcn_ballot_w64(b.row_start[i + 1] > row && at + lane < b.n_seqs);
        if (below) return at + (uint32_t)__builtin_ctzll(below);
    }
    return b.n_seqs;
}

// The page of a sequence's position (below its len), in the pool.
__device__ __forceinline__ uint32_t paged_page(const PagedArgs& b, uint32_t seq, uint32_t page_at, uint32_t& bad) {
    const uint32_t id = b.table[(size_t)seq * b.table_stride + page_at];
    if (id < b.n_pages) return id;
    bad |= FK_PAGED_BAD_PAGE;
    return 0u;
}

}  // namespace fk
