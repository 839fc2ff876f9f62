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

constexpr uint32_t kExtendKept = 4;                             // sequences that a thread has in hand
constexpr uint32_t kExtendMost = 64;                            // sequences of a block, at most
constexpr uint32_t kExtendSlots = 1u << 18;                     // a bit each in LDS
constexpr uint32_t kExtendFew = 64;                             // new rows of a sequence that one wave writes
constexpr uint32_t kExtendLots = 0x7fffffffu;                   // sums stop there: more than any batch or pool holds

// The sum of this lane's value and those before it, each up to kExtendLots: inside rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t extend_step(uint32_t v) {
    const uint32_t sum = v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    return sum < kExtendLots ? sum : kExtendLots;
}
__device__ __forceinline__ uint32_t extend_upto(uint32_t v) {
    v = extend_step<0x111, 0xF>(v);
    v = extend_step<0x112, 0xF>(v);
    v = extend_step<0x114, 0xF>(v);
    v = extend_step<0x118, 0xF>(v);
    v = extend_step<0x142, 0xA>(v);
    return extend_step<0x143, 0xC>(v);
}
__device__ __forceinline__ uint32_t extend_add(uint32_t a, uint32_t b) { return a + b < kExtendLots ? a + b : kExtendLots; }

// Every block forms the sums over all sequences by itself, four a thread at a time, and then does those that are its own, a wave one at a time: the copy of a row of
// page ids with 4 KB on their way, the new pages, and, all waves together, the rows of a chunk.  What the launch leaves for the next one (lengths, free
// pages) is written by the block that is the last to have read it, so that it may be written in place.
// Bound by trips to memory one after another: slots and rows (1 us), lengths (1.1), the sums (0.6 to 2.5), the longest row of ids (1.5 to 4.5), the last
// block's lengths (1).  One token 4.5 us, 256 tokens of up to 30000 positions in pages of 16 6.1, 1003 sequences of up to 60000 9.9 (5.7 MB, 0.6 TB/s), a chunk of 8192
// rows 9.1.  A row of ids with 16 KB on its way, or by the four waves together, took 10.2 and 11.4 of the 9.9.
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void paged_extend_kernel(const ExtendArgs a) {
    extern __shared__ uint32_t named[];   // a bit for a slot, where slots are given
    struct Own {
        uint32_t slot, held, rows, row0, page0;
    };
    __shared__ Own own[kExtendMost];
    __shared__ uint32_t part[2][2][THREADS / 64];
    __shared__ uint32_t bad_all, last;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), page_rows = 1u << a.page_shift;
    const uint32_t share = (a.n_seqs + gridDim.x - 1u) / gridDim.x, mine0 = blockIdx.x * share, mine1 = mine0 + share < a.n_seqs ? mine0 + share : a.n_seqs;
    const uint32_t n_free_raw = *a.n_free, n_free = n_free_raw < a.n_pages ? n_free_raw : a.n_pages;
    uint32_t bad = n_free_raw > a.n_pages ? FK_PAGED_BAD_PAGE : 0u;
    uint32_t all_rows = 0, all_pages = 0;
    uint32_t slot[kExtendKept], held[kExtendKept], rows[kExtendKept];
    for (uint32_t at = 0, turn = 0; at < a.n_seqs; at += THREADS * kExtendKept, turn ^= 1u) {
        const uint32_t first = at + tid * kExtendKept;
        uint32_t pages[kExtendKept];
#pragma unroll
        for (uint32_t u = 0; u < kExtendKept; ++u) {
            const uint32_t i = first + u < a.n_seqs ? first + u : a.n_seqs - 1u;
            slot[u] = a.slot ? a.slot[i] : i;
            rows[u] = a.new_rows ? a.new_rows[i] : 1u;
        }
#pragma unroll
        for (uint32_t u = 0; u < kExtendKept; ++u) held[u] = a.lengths[slot[u] < a.n_slots ? slot[u] : 0u];
        if (at == 0) {   // (while the first are on their way)
            if (tid == 0) bad_all = 0;
            if (a.slot)
                for (uint32_t i = tid; i < (a.n_slots + 31u) / 32u; i += THREADS) named[i] = 0;
            __syncthreads();
        }
        uint32_t my_rows = 0, my_pages = 0;
#pragma unroll
        for (uint32_t u = 0; u < kExtendKept; ++u) {
            const bool in = first + u < a.n_seqs;
            uint32_t wrong = slot[u] >= a.n_slots ? FK_PAGED_BAD_SLOT : 0u;
            if (rows[u] > a.max_rows) wrong |= FK_PAGED_BAD_ROWS;
            else if (held[u] > a.max_len || rows[u] > a.max_len - held[u]) wrong |= FK_PAGED_BAD_LENGTH;
            if (in && a.slot && slot[u] < a.n_slots && (atomicOr(&named[slot[u] / 32u], 1u << slot[u] % 32u) >> slot[u] % 32u & 1u)) wrong |= FK_PAGED_BAD_SLOT;   // named twice
            if (in) bad |= wrong;
            if (wrong || !in) slot[u] = held[u] = rows[u] = 0;
            pages[u] = ((held[u] + rows[u] + page_rows - 1u) >> a.page_shift) - ((held[u] + page_rows - 1u) >> a.page_shift);
            my_rows = extend_add(my_rows, rows[u]);
            my_pages = extend_add(my_pages, pages[u]);
        }
        uint32_t rows_upto = extend_upto(my_rows), pages_upto = extend_upto(my_pages);
        if (lane == 63u) {
            part[turn][0][wave] = rows_upto;
            part[turn][1][wave] = pages_upto;
        }
        __syncthreads();
        // (sums that have reached kExtendLots are not used)
        rows_upto += all_rows - my_rows;
        pages_upto += all_pages - my_pages;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            const uint32_t r = part[turn][0][w], p = part[turn][1][w];
            rows_upto += w < wave ? r : 0u;
            pages_upto += w < wave ? p : 0u;
            all_rows = extend_add(all_rows, r);
            all_pages = extend_add(all_pages, p);
        }
#pragma unroll
        for (uint32_t u = 0; u < kExtendKept; ++u) {
            if (first + u >= mine0 && first + u < mine1) own[first + u - mine0] = Own{slot[u], held[u], rows[u], rows_upto, pages_upto};
            rows_upto += rows[u];
            pages_upto += pages[u];
        }
    }
    if (bad) atomicOr(&bad_all, bad);
    __syncthreads();
    // (lengths and n_free are read no more, but by the last block)
    if (tid == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1u ? 1u : 0u;
    bad = bad_all;
    if (all_rows > a.rows) bad |= FK_PAGED_BAD_ROWS;
    if (all_pages > n_free) bad |= FK_PAGED_NO_PAGE;
    const bool ok = bad == 0;   // else nothing is taken, and no sequence has a new row
    if (bad && tid == 0 && blockIdx.x == 0 && a.fault) __hip_atomic_fetch_or(a.fault, bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    const uint32_t n = mine0 < mine1 ? mine1 - mine0 : 0u;
    uint32_t bad_page = 0;
    auto page_at = [&](const Own& s, uint32_t c) {   // page c of a sequence
        const uint32_t before = (s.held + page_rows - 1u) >> a.page_shift;
        if (c < before) return a.tables[(size_t)s.slot * a.tables_stride + c];
        const uint32_t id = a.free_pages[n_free - 1u - (s.page0 + (c - before))];
        if (id >= a.n_pages) bad_page = FK_PAGED_BAD_PAGE;
        return id;
    };
    auto row_slot = [&](const Own& s, uint32_t j) {
        const uint32_t pos = s.held + j;
        return page_at(s, pos >> a.page_shift) * page_rows + (pos & (page_rows - 1u));
    };
    for (uint32_t i = tid; i < n; i += THREADS) {
        const Own s = own[i];
        a.row_start[mine0 + i] = ok ? s.row0 : 0u;
        a.kv_len[mine0 + i] = ok ? s.held + s.rows : 0u;
        if (mine0 + i + 1u == a.n_seqs) a.row_start[a.n_seqs] = ok ? s.row0 + s.rows : 0u;
    }
    if (ok) {
        typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(4)));
        for (uint32_t i = wave; i < n; i += THREADS / 64) {
            const Own s = own[i];
            const uint32_t before = (s.held + page_rows - 1u) >> a.page_shift, after = (s.held + s.rows + page_rows - 1u) >> a.page_shift;
            uint32_t* const from = a.tables + (size_t)s.slot * a.tables_stride;
            uint32_t* const to = a.page_table + (size_t)(mine0 + i) * a.table_stride;
            const uint32_t quads = before / 4u;
            constexpr uint32_t AHEAD = 4;
            for (uint32_t q0 = lane; q0 < quads; q0 += 64u * AHEAD) {
                loose v[AHEAD];
#pragma unroll
                for (uint32_t u = 0; u < AHEAD; ++u) v[u] = *reinterpret_cast<const loose*>(from + 4u * (q0 + 64u * u < quads ? q0 + 64u * u : q0));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t u = 0; u < AHEAD; ++u)
                    if (q0 + 64u * u < quads) *reinterpret_cast<loose*>(to + 4u * (q0 + 64u * u)) = v[u];
            }
            for (uint32_t c = quads * 4u + lane; c < after; c += 64u) {
                const uint32_t id = page_at(s, c);
                if (c >= before) from[c] = id;
                to[c] = id;
            }
            if (a.row_slots && s.rows <= kExtendFew && lane < s.rows) a.row_slots[s.row0 + lane] = row_slot(s, lane);
        }
        if (a.row_slots)
            for (uint32_t i = 0; i < n; ++i) {
                const Own s = own[i];
                if (s.rows <= kExtendFew) continue;
                // (four rows lie in one page or two)
                const uint32_t quads = s.rows / 4u;
                constexpr uint32_t AHEAD = 2;
                for (uint32_t q0 = tid; q0 < quads; q0 += THREADS * AHEAD) {
                    uint32_t page[AHEAD][2];
#pragma unroll
                    for (uint32_t u = 0; u < AHEAD; ++u) {
                        const uint32_t q = q0 + THREADS * u < quads ? q0 + THREADS * u : q0, pos = s.held + 4u * q;
                        page[u][0] = page_at(s, pos >> a.page_shift);
                        page[u][1] = page_at(s, (pos + 3u) >> a.page_shift);
                    }
#pragma unroll
                    for (uint32_t u = 0; u < AHEAD; ++u) {
                        const uint32_t q = q0 + THREADS * u, pos = s.held + 4u * q;
                        loose v;
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) v[e] = page[u][(pos + e) >> a.page_shift != pos >> a.page_shift] * page_rows + ((pos + e) & (page_rows - 1u));
                        if (q < quads) *reinterpret_cast<loose*>(a.row_slots + s.row0 + 4u * q) = v;
                    }
                }
                for (uint32_t j = quads * 4u + tid; j < s.rows; j += THREADS) a.row_slots[s.row0 + j] = row_slot(s, j);
            }
    }
    if (bad_page && a.fault) __hip_atomic_fetch_or(a.fault, bad_page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (!last) return;
    if (tid == 0) {
        __hip_atomic_store(a.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *a.n_free_out = ok ? n_free - all_pages : n_free_raw;
    }
    auto mark = [&](uint32_t i) { return a.slot ? (named[i / 32u] >> i % 32u & 1u) != 0 : i < a.n_seqs; };   // (a faulty batch may not name all that it means: nothing changes)
    if (a.lengths_out != a.lengths)
#pragma unroll 4
        for (uint32_t i = tid; i < a.n_slots; i += THREADS)
            if (!ok || !mark(i)) a.lengths_out[i] = a.lengths[i];
    if (!ok) return;
    // (the slots are all different; the last ones' lengths are still in hand)
    const uint32_t in_hand = (a.n_seqs - 1u) / (THREADS * kExtendKept) * (THREADS * kExtendKept);
#pragma unroll
    for (uint32_t u = 0; u < kExtendKept; ++u)
        if (in_hand + tid * kExtendKept + u < a.n_seqs) a.lengths_out[slot[u]] = held[u] + rows[u];
#pragma unroll 4
    for (uint32_t i = tid; i < in_hand; i += THREADS) {
        const uint32_t at = a.slot ? a.slot[i] : i;
        a.lengths_out[at] = a.lengths[at] + (a.new_rows ? a.new_rows[i] : 1u);
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
    if (b->max_len > 0x7fffffffu || b->rows >= kExtendLots || n_pages >= kExtendLots) return set_error(FK_ERR_UNSUPPORTED, "paged_extend: batch too large");
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
    const bool many = b->n_seqs > 1024;   // (the sequences that 256 threads have in hand: 4096 of them in four turns 25 us, at once 15)
    l->func = many ? reinterpret_cast<const void*>(&paged_extend_kernel<1024>) : reinterpret_cast<const void*>(&paged_extend_kernel<256>);
    const uint32_t waves = many ? 16 : 4;
    l->grid = dim3(std::max(std::min((b->n_seqs + waves - 1) / waves, (uint32_t)dev->cus), (b->n_seqs + kExtendMost - 1) / kExtendMost), 1, 1);
    l->block = dim3(64 * waves, 1, 1);
    l->shmem = q->slot ? (q->n_slots + 31) / 32 * 4 : 0;
    FK_TRY(raise_dynamic_lds(l->func, l->shmem));
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
