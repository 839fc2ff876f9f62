// A batch over a paged cache built on the device from the requests' lengths: row starts, lengths, page tables and the pool row of every new row, with the
// pages that are missing taken from a stack of free ones.
//
//     before = ceil(held / page_rows), after = ceil((held + new) / page_rows):   sequence i takes after - before pages, behind those of the sequences before it
#include <algorithm>

#include "fk_host.hpp"
#include "paged_device.hpp"

namespace fk {

struct ExtendArgs {
    const uint32_t* slot;       // null: sequence i is in slot i
    const uint32_t* new_rows;   // null: one each
    const uint32_t* lengths;
    uint32_t* lengths_out;
    uint32_t* tables;
    const uint32_t* free_pages;
    const uint32_t* n_free;
    uint32_t* n_free_out;
    uint32_t* counter;
    uint32_t* row_start;
    uint32_t* kv_len;
    uint32_t* page_table;
    uint32_t* row_slots;   // may be null
    uint32_t* fault;
    uint32_t n_slots, tables_stride, table_stride, n_seqs, rows, max_rows, max_len, n_pages, page_shift;
};

constexpr uint32_t kExtendThreads = 256, kExtendMost = 64;      // sequences of a block, at most
constexpr uint32_t kExtendSlots = 1u << 18;                     // a bit each in LDS

// Every block forms the sums over all sequences by itself, and then does those that are its own, a wave one at a time.  What the launch leaves for the
// next one (lengths, free pages) is written by the block that is the last to have read it, so that it may be written in place.
__global__ __launch_bounds__(kExtendThreads) void paged_extend_kernel(const ExtendArgs a) {
    extern __shared__ uint32_t named[];   // a bit for a slot, where slots are given
    struct Own {
        uint32_t slot, held, rows, row0, page0;
    };
    __shared__ Own own[kExtendMost];
    __shared__ uint64_t part[2][kExtendThreads / 64];
    __shared__ uint32_t bad_all, last;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, page_rows = 1u << a.page_shift;
    if (tid == 0) bad_all = 0;
    if (a.slot)
        for (uint32_t i = tid; i < (a.n_slots + 31u) / 32u; i += kExtendThreads) named[i] = 0;
    __syncthreads();
    const uint32_t n_free_raw = *a.n_free, n_free = n_free_raw < a.n_pages ? n_free_raw : a.n_pages;
    uint32_t bad = n_free_raw > a.n_pages ? FK_PAGED_BAD_PAGE : 0u;
    // a thread's sequences lie side by side
    const uint32_t per = (a.n_seqs + kExtendThreads - 1u) / kExtendThreads, first = tid * per < a.n_seqs ? tid * per : a.n_seqs, end = first + per < a.n_seqs ? first + per : a.n_seqs;
    struct Seq {
        uint32_t slot, held, rows, pages, bad;
    };
    auto read = [&](uint32_t i) {
        Seq s;
        s.bad = 0;
        s.slot = a.slot ? a.slot[i] : i;
        s.rows = a.new_rows ? a.new_rows[i] : 1u;
        if (s.slot >= a.n_slots) {
            s.slot = 0;
            s.bad = FK_PAGED_BAD_SLOT;
        }
        s.held = a.lengths[s.slot];
        if (s.rows > a.max_rows) {
            s.rows = 0;
            s.bad |= FK_PAGED_BAD_ROWS;
        }
        if (s.held > a.max_len || s.rows > a.max_len - s.held) {
            s.rows = 0;
            s.held = 0;
            s.bad |= FK_PAGED_BAD_LENGTH;
        }
        const uint32_t before = (s.held + page_rows - 1u) >> a.page_shift, after = (s.held + s.rows + page_rows - 1u) >> a.page_shift;
        s.pages = after - before;
        return s;
    };
    uint64_t rows = 0, pages = 0;
    for (uint32_t i = first; i < end; ++i) {
        const Seq s = read(i);
        bad |= s.bad;
        if (a.slot && !(s.bad & FK_PAGED_BAD_SLOT) && (atomicOr(&named[s.slot / 32u], 1u << s.slot % 32u) >> s.slot % 32u & 1u)) bad |= FK_PAGED_BAD_SLOT;   // named twice
        rows += s.rows;
        pages += s.pages;
    }
    uint64_t rows_upto = rows, pages_upto = pages;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t r = __shfl_up((unsigned long long)rows_upto, o, 64), p = __shfl_up((unsigned long long)pages_upto, o, 64);
        rows_upto += lane >= (uint32_t)o ? r : 0u;
        pages_upto += lane >= (uint32_t)o ? p : 0u;
    }
    if (lane == 63u) {
        part[0][wave] = rows_upto;
        part[1][wave] = pages_upto;
    }
    if (bad) atomicOr(&bad_all, bad);
    __syncthreads();
    uint64_t all_rows = 0, all_pages = 0;
#pragma unroll
    for (uint32_t w = 0; w < kExtendThreads / 64; ++w) {
        if (w < wave) {
            rows_upto += part[0][w];
            pages_upto += part[1][w];
        }
        all_rows += part[0][w];
        all_pages += part[1][w];
    }
    bad = bad_all;
    if (all_rows > a.rows) bad |= FK_PAGED_BAD_ROWS;
    if (all_pages > n_free) bad |= FK_PAGED_NO_PAGE;
    const bool ok = bad == 0;   // else nothing is taken, and no sequence has a new row
    if (bad && tid == 0 && blockIdx.x == 0 && a.fault) __hip_atomic_fetch_or(a.fault, bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    const uint32_t share = (a.n_seqs + gridDim.x - 1u) / gridDim.x, mine0 = blockIdx.x * share, mine1 = mine0 + share < a.n_seqs ? mine0 + share : a.n_seqs;
    const uint32_t n = mine0 < mine1 ? mine1 - mine0 : 0u;
    if (first < mine1 && end > mine0) {
        uint64_t r = rows_upto - rows, p = pages_upto - pages;
        for (uint32_t i = first; i < end && i < mine1; ++i) {
            const Seq s = read(i);
            if (i >= mine0) own[i - mine0] = Own{s.slot, s.held, ok ? s.rows : 0u, ok ? (uint32_t)r : 0u, (uint32_t)p};
            r += s.rows;
            p += s.pages;
        }
    }
    __syncthreads();
    // (lengths and n_free are read no more, but by the last block)
    if (tid == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1u ? 1u : 0u;
    uint32_t bad_page = 0;
    for (uint32_t i = wave; i < n; i += kExtendThreads / 64) {
        const Own s = own[i];
        const uint32_t seq = mine0 + i, before = (s.held + page_rows - 1u) >> a.page_shift, length = s.held + s.rows, after = (length + page_rows - 1u) >> a.page_shift;
        if (lane == 0) {
            a.row_start[seq] = s.row0;
            a.kv_len[seq] = ok ? length : 0u;
            if (seq + 1u == a.n_seqs) a.row_start[seq + 1u] = s.row0 + s.rows;
        }
        if (!ok) continue;
        uint32_t* const from = a.tables + (size_t)s.slot * a.tables_stride;
        uint32_t* const to = a.page_table + (size_t)seq * a.table_stride;
        auto page_at = [&](uint32_t c) {
            if (c < before) return from[c];
            const uint32_t id = a.free_pages[n_free - 1u - (s.page0 + (c - before))];
            if (id >= a.n_pages) bad_page = FK_PAGED_BAD_PAGE;
            return id;
        };
        for (uint32_t c = lane; c < after; c += 64u) {
            const uint32_t id = page_at(c);
            if (c >= before) from[c] = id;
            to[c] = id;
        }
        if (a.row_slots)
            for (uint32_t j = lane; j < s.rows; j += 64u) {
                const uint32_t pos = s.held + j;
                a.row_slots[s.row0 + j] = page_at(pos >> a.page_shift) * page_rows + (pos & (page_rows - 1u));
            }
    }
    if (bad_page && a.fault) __hip_atomic_fetch_or(a.fault, bad_page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (!last) return;
    if (tid == 0) {
        __hip_atomic_store(a.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *a.n_free_out = ok ? n_free - (uint32_t)all_pages : n_free_raw;
    }
    // (a sequence's own slot is written once: the slots are all different)
    if (a.lengths_out != a.lengths) {
        for (uint32_t i = tid; i < a.n_slots; i += kExtendThreads) a.lengths_out[i] = a.lengths[i];
        __syncthreads();
    }
    if (ok)
        for (uint32_t i = tid; i < a.n_seqs; i += kExtendThreads) {
            const uint32_t slot = a.slot ? a.slot[i] : i;
            a.lengths_out[slot] = a.lengths[slot] + (a.new_rows ? a.new_rows[i] : 1u);
        }
}

fk_status plan_paged_extend(const fk_paged_requests* q, const fk_paged_batch* b, uint32_t n_pages, uint32_t page_rows, uint32_t* row_slots, Launch* l) {
    if (!q || !b) return set_error(FK_ERR_INVALID, "paged_extend: null requests or batch");
    if (!q->lengths || !q->lengths_out || !q->tables || !q->free_pages || !q->n_free || !q->n_free_out || !q->counter || !b->row_start || !b->kv_len || !b->page_table)
        return set_error(FK_ERR_INVALID, "paged_extend: null pointer in the requests or the batch");
    if (q->n_slots == 0 || b->n_seqs == 0 || b->rows == 0 || b->max_rows == 0 || b->max_len == 0 || n_pages == 0)
        return set_error(FK_ERR_INVALID, "paged_extend: no slots, empty batch or no pages");
    if (b->max_rows > b->rows) return set_error(FK_ERR_INVALID, "paged_extend: max_rows exceeds the rows of the buffers");
    if (page_rows < 16 || page_rows > 1024 || (page_rows & (page_rows - 1))) return set_error(FK_ERR_UNSUPPORTED, "paged_extend: page_rows must be a power of two from 16 to 1024");
    if (b->max_len > 0x7fffffffu || b->rows > 0x7fffffffu) return set_error(FK_ERR_UNSUPPORTED, "paged_extend: batch too large");
    if (b->n_seqs > q->n_slots) return set_error(FK_ERR_INVALID, "paged_extend: more sequences than slots");
    if (q->n_slots > kExtendSlots) return set_error(FK_ERR_UNSUPPORTED, "paged_extend: up to 2^18 slots");
    const uint64_t most = ((uint64_t)b->max_len + page_rows - 1) / page_rows;
    if (most > b->table_stride || most > q->table_stride) return set_error(FK_ERR_INVALID, "paged_extend: max_len exceeds what a row of a page table holds");
    if (row_slots && (uint64_t)n_pages * page_rows > 0xffffffffull) return set_error(FK_ERR_UNSUPPORTED, "paged_extend: a pool of 2^32 rows or more has no slot map");
    const uintptr_t all = (uintptr_t)q->slot | (uintptr_t)q->new_rows | (uintptr_t)q->lengths | (uintptr_t)q->lengths_out | (uintptr_t)q->tables | (uintptr_t)q->free_pages |
                          (uintptr_t)q->n_free | (uintptr_t)q->n_free_out | (uintptr_t)q->counter | (uintptr_t)b->row_start | (uintptr_t)b->kv_len |
                          (uintptr_t)b->page_table | (uintptr_t)row_slots | (uintptr_t)b->fault;
    if (all & 3u) return set_error(FK_ERR_INVALID, "paged_extend: arrays must be 4-byte aligned");
    // what is written overlaps nothing else, but that lengths_out may be lengths and n_free_out n_free
    enum { READ, WRITTEN, LENGTHS, FREE };
    const struct {
        const void* at;
        uint64_t words;
        int kind;
        bool may_share;
    } spans[] = {{q->slot, b->n_seqs, READ, false}, {q->new_rows, b->n_seqs, READ, false}, {q->free_pages, n_pages, READ, false},
                 {q->lengths, q->n_slots, LENGTHS, true}, {q->lengths_out, q->n_slots, LENGTHS, true}, {q->n_free, 1, FREE, true}, {q->n_free_out, 1, FREE, true},
                 {q->tables, (uint64_t)q->n_slots * q->table_stride, WRITTEN, false}, {q->counter, 1, WRITTEN, false}, {b->row_start, b->n_seqs + 1ull, WRITTEN, false},
                 {b->kv_len, b->n_seqs, WRITTEN, false}, {b->page_table, (uint64_t)b->n_seqs * b->table_stride, WRITTEN, false},
                 {row_slots, b->rows, WRITTEN, false}, {b->fault, 1, WRITTEN, false}};
    for (const auto& x : spans)
        for (const auto& y : spans) {
            if (&x >= &y || !x.at || !y.at || (x.kind == READ && y.kind == READ)) continue;
            if (x.may_share && x.kind == y.kind && x.at == y.at) continue;
            if ((uintptr_t)x.at < (uintptr_t)y.at + 4 * y.words && (uintptr_t)y.at < (uintptr_t)x.at + 4 * x.words)
                return set_error(FK_ERR_INVALID, "paged_extend: an array that is written overlaps another");
        }
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    uint32_t shift = 4;
    while ((1u << shift) < page_rows) ++shift;
    ExtendArgs a{q->slot, q->new_rows, q->lengths, q->lengths_out, q->tables, q->free_pages, q->n_free, q->n_free_out, q->counter,
                 const_cast<uint32_t*>(b->row_start), const_cast<uint32_t*>(b->kv_len), const_cast<uint32_t*>(b->page_table), row_slots, b->fault,
                 q->n_slots, q->table_stride, b->table_stride, b->n_seqs, b->rows, b->max_rows, b->max_len, n_pages, shift};
    l->func = reinterpret_cast<const void*>(&paged_extend_kernel);
    l->grid = dim3(std::max(std::min((b->n_seqs + 3) / 4, (uint32_t)dev->cus), (b->n_seqs + kExtendMost - 1) / kExtendMost), 1, 1);
    l->block = dim3(kExtendThreads, 1, 1);
    l->shmem = q->slot ? (q->n_slots + 31) / 32 * 4 : 0;
    FK_TRY(raise_dynamic_lds(l->func, l->shmem));
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
