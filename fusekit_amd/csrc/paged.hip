// Rotary positions and the append of new rows for sequences over a paged cache, and pages copied inside a pool.
#include <math.h>

#include <algorithm>
#include <new>

#include "fk_host.hpp"
#include "paged_device.hpp"

namespace fk {

fk_status paged_args(const char* what, const fk_paged_batch* b, const fk_page_pool* p, PagedArgs* out) {
    const std::string w = what;
    if (!b || !p) return set_error(FK_ERR_INVALID, w + ": null batch or pool");
    if (!b->row_start || !b->kv_len || !b->page_table || !p->k || !p->v) return set_error(FK_ERR_INVALID, w + ": null pointer in the batch or the pool");
    if (b->n_seqs == 0 || b->rows == 0 || b->max_rows == 0 || b->max_len == 0 || p->n_pages == 0 || p->n_kv == 0)
        return set_error(FK_ERR_INVALID, w + ": empty batch or pool");
    if (b->max_rows > b->rows) return set_error(FK_ERR_INVALID, w + ": max_rows exceeds the rows of the buffers");
    if (p->page_rows < 16 || p->page_rows > 1024 || (p->page_rows & (p->page_rows - 1)))
        return set_error(FK_ERR_UNSUPPORTED, w + ": page_rows must be a power of two from 16 to 1024");
    if (p->head_dim != 64 && p->head_dim != 128) return set_error(FK_ERR_UNSUPPORTED, w + ": head dimension 64 or 128");
    if (((uint64_t)b->max_len + p->page_rows - 1) / p->page_rows > b->table_stride)
        return set_error(FK_ERR_INVALID, w + ": max_len exceeds what a row of the page table holds");
    if (b->max_len > 0x7fffffffu || b->rows > 0x7fffffffu || b->n_seqs > 0x7fffffffu) return set_error(FK_ERR_UNSUPPORTED, w + ": batch too large");
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15u) return set_error(FK_ERR_INVALID, w + ": pages must be 16-byte aligned");
    if (((uintptr_t)b->row_start | (uintptr_t)b->kv_len | (uintptr_t)b->page_table | (uintptr_t)b->fault) & 3u)
        return set_error(FK_ERR_INVALID, w + ": the batch's arrays must be 4-byte aligned");
    uint32_t shift = 4;
    while ((1u << shift) < p->page_rows) ++shift;
    *out = PagedArgs{b->row_start, b->kv_len, b->page_table, b->table_stride, b->n_seqs, b->rows, b->max_rows, b->max_len,
                     p->n_pages, shift, p->n_kv, b->fault};
    return FK_OK;
}

// ---- rotary frequencies ----
// One thread a pair; the formulas are the header's, in 64 bits.
struct RopeFreqArgs {
    double* out;
    uint32_t pairs;
    int scaling;
    double theta, factor, low, high, trained, ramp_lo, ramp_hi;
};
__global__ __launch_bounds__(64) void rope_frequencies_kernel(const RopeFreqArgs a) {
    const double two_pi = 6.283185307179586476925;
    for (uint32_t i = threadIdx.x; i <= a.pairs; i += 64) {
        if (i == a.pairs) {
            a.out[i] = a.scaling == FK_ROPE_RAMP ? 0.1 * log(a.factor) + 1.0 : 1.0;
            continue;
        }
        double rev = pow(a.theta, -(double)i / (double)a.pairs) / two_pi;
        double keep = 1.0;   // how much of the unscaled frequency stays
        if (a.scaling == FK_ROPE_LINEAR) keep = 0.0;
        if (a.scaling == FK_ROPE_PARTS) keep = (a.trained * rev - a.low) / (a.high - a.low);
        if (a.scaling == FK_ROPE_RAMP) keep = 1.0 - ((double)i - a.ramp_lo) / fmax(a.ramp_hi - a.ramp_lo, 1e-3);
        keep = fmin(fmax(keep, 0.0), 1.0);
        a.out[i] = rev * (keep + (1.0 - keep) / a.factor);
    }
}

fk_status plan_rope_frequencies(uint32_t dims, double theta, int scaling, double factor, double low, double high, uint32_t trained,
                                double* out, Launch* l) {
    if (!out) return set_error(FK_ERR_INVALID, "rope frequencies: null pointer");
    if (dims == 0 || dims % 2) return set_error(FK_ERR_INVALID, "rope frequencies: dims must be even and not 0");
    if (!(theta > 1.0) || !std::isfinite(theta)) return set_error(FK_ERR_INVALID, "rope frequencies: theta must be above 1");
    if (scaling < FK_ROPE_PLAIN || scaling > FK_ROPE_RAMP) return set_error(FK_ERR_INVALID, "rope frequencies: unknown scaling");
    if (scaling == FK_ROPE_PLAIN) factor = 1.0;
    if (!(factor >= 1.0) || !std::isfinite(factor)) return set_error(FK_ERR_INVALID, "rope frequencies: factor must be at least 1");
    RopeFreqArgs a{out, dims / 2, scaling, theta, factor, low, high, (double)trained, 0.0, 0.0};
    if (scaling >= FK_ROPE_PARTS) {
        if (!(low > 0.0) || !(high > low) || !std::isfinite(high) || trained == 0)
            return set_error(FK_ERR_INVALID, "rope frequencies: 0 < low < high turns and a trained context");
        // the (fractional) pair that turns `t` times within the trained context
        auto pair_of = [&](double t) { return dims * log(trained / (t * 6.283185307179586476925)) / (2.0 * log(theta)); };
        a.ramp_lo = std::max(floor(pair_of(high)), 0.0);
        a.ramp_hi = std::min(ceil(pair_of(low)), (double)dims - 1.0);
    }
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    l->func = reinterpret_cast<const void*>(&rope_frequencies_kernel);
    l->grid = dim3(1, 1, 1);
    l->block = dim3(64, 1, 1);
    l->set_args(a);
    return FK_OK;
}

// ---- rotary positions, and k and v into the pages ----
struct RopePagedArgs {
    PagedArgs b;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;
    const uint16_t* q_norm;
    const uint16_t* k_norm;
    uint16_t* k_pages;
    uint16_t* v_pages;
    const double* freq;
    uint32_t q_stride, k_stride, v_stride, q_out_stride, n_heads, rope_dims;
    float eps;
};

// pair (x, y) -> (x c - y s, y c + x s) gain, the angle 2 pi frac(position * revolutions) -- its product in 64 bits, its fraction in fp32, so that it is off by
// 2^-24 of a turn at any position.  Before it x r w, r = 1 / sqrt(mean x^2 + eps), where a head norm is given; one rounding, at the store.
// A block a row: its position, page and D / 2 cosines and sines are found once for all heads.  A thread takes 16-byte pieces (8 dims), D / 8 lanes a
// head, and the piece it is paired with a second time, out of the cache.  Bound by the bytes, read and written once: 4015 rows of 32 + 2 x 8 heads x 128 in
// 23.5 us, 4.2 TB/s (a copy: 4.75); a single row 2.4 us.
template <int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_paged_store_kernel(const RopePagedArgs a) {
    constexpr uint32_t PIECES = D / 8;
    __shared__ float2 turn[D / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, row = blockIdx.x;
    const uint32_t seq = paged_seq_of(a.b, row, lane);
    if (seq >= a.b.n_seqs) return;   // behind the last sequence
    const PagedSeq s = paged_seq(a.b, seq);
    uint32_t bad = s.bad;
    const uint32_t place = row - s.row0;
    const bool live = row >= s.row0 && place < s.rows && s.len + place >= s.rows;
    const uint32_t pos = s.len + place - s.rows;
    uint32_t page = 0;
    if (live) page = paged_page(a.b, seq, pos >> a.b.page_shift, bad);
    if (bad && tid == 0) paged_fault(a.b, bad);
    if (!live) return;
    const uint32_t half = a.rope_dims / 2;
    if (tid < half) {
        // the angle in revolutions: 64 bits until only its fraction is left
        const double rev = (double)pos * a.freq[tid];
        const float part = (float)(rev - floor(rev)), gain = (float)a.freq[half];
        float sn, cs;
        sincospif(2.0f * part, &sn, &cs);
        turn[tid] = make_float2(cs * gain, sn * gain);
    }
    __syncthreads();
    const uint32_t heads = a.n_heads + 2u * a.b.n_kv, page_rows = 1u << a.b.page_shift, slot = pos & (page_rows - 1u);
    for (uint32_t i = tid; i < heads * PIECES; i += 256u) {
        const uint32_t head = i / PIECES, piece = i % PIECES;
        const bool is_q = head < a.n_heads, is_k = !is_q && head < a.n_heads + a.b.n_kv;
        const uint32_t kvh = is_q ? 0u : (head - a.n_heads) % a.b.n_kv;
        const uint16_t* src = is_q ? a.q + (size_t)row * a.q_stride + (size_t)head * D
                                   : is_k ? a.k + (size_t)row * a.k_stride + (size_t)kvh * D : a.v + (size_t)row * a.v_stride + (size_t)kvh * D;
        const size_t at = (((size_t)page * a.b.n_kv + kvh) * page_rows + slot) * D;
        uint16_t* dst = is_q ? a.q_out + (size_t)row * a.q_out_stride + (size_t)head * D : (is_k ? a.k_pages : a.v_pages) + at;
        const bool store = is_q || !(bad & FK_PAGED_BAD_PAGE);
        uint4 x = reinterpret_cast<const uint4*>(src)[piece];
        if (is_q || is_k) {
            const uint32_t d0 = piece * 8u;
            const bool rotated = d0 < a.rope_dims;
            const uint32_t other = INTERLEAVED || !rotated ? piece : (d0 < half ? piece + half / 8u : piece - half / 8u);
            const uint4 y = reinterpret_cast<const uint4*>(src)[other];
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
            float xf[8], yf[8], o[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                xf[2 * e] = bf16_lo(xw[e]);
                xf[2 * e + 1] = bf16_hi(xw[e]);
                yf[2 * e] = bf16_lo(yw[e]);
                yf[2 * e + 1] = bf16_hi(yw[e]);
            }
            const uint16_t* nw = is_q ? a.q_norm : a.k_norm;
            if (nw) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(xf[e], xf[e], ss);
                ss = group_sum(ss, (int)PIECES);
                const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    xf[e] = xf[e] * r * bf16_bits_to_f32(nw[d0 + e]);
                    yf[e] = yf[e] * r * bf16_bits_to_f32(nw[other * 8u + e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = xf[e];
            if (rotated) {
                if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 t = turn[piece * 4u + e];
                        o[2 * e] = xf[2 * e] * t.x - xf[2 * e + 1] * t.y;
                        o[2 * e + 1] = xf[2 * e + 1] * t.x + xf[2 * e] * t.y;
                    }
                } else {
                    const bool low = d0 < half;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 t = turn[(low ? d0 : d0 - half) + e];
                        o[e] = fmaf(xf[e], t.x, (low ? -yf[e] : yf[e]) * t.y);
                    }
                }
            }
            x = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        }
        if (store) reinterpret_cast<uint4*>(dst)[piece] = x;
    }
}

fk_status plan_rope_paged_store(const uint16_t* q, uint32_t q_stride, const uint16_t* k, uint32_t k_stride, const uint16_t* v, uint32_t v_stride,
                                uint16_t* q_out, uint32_t q_out_stride, uint32_t n_heads, const uint16_t* q_norm, const uint16_t* k_norm,
                                float eps, uint32_t rope_dims, int interleaved, const double* freq, const fk_paged_batch* batch,
                                const fk_page_pool* pool, Launch* l) {
    RopePagedArgs a;
    memset(&a, 0, sizeof(a));
    FK_TRY(paged_args("rope_paged_store", batch, pool, &a.b));
    const uint32_t D = pool->head_dim, n_kv = pool->n_kv;
    if (!q || !k || !v || !q_out) return set_error(FK_ERR_INVALID, "rope_paged_store: null pointer");
    if (n_heads == 0) return set_error(FK_ERR_INVALID, "rope_paged_store: no query heads");
    if (rope_dims % 16 || rope_dims > D) return set_error(FK_ERR_UNSUPPORTED, "rope_paged_store: rope_dims must be a multiple of 16 up to head_dim");
    if (rope_dims && !freq) return set_error(FK_ERR_INVALID, "rope_paged_store: null frequencies");
    if ((uintptr_t)freq & 7u) return set_error(FK_ERR_INVALID, "rope_paged_store: frequencies must be 8-byte aligned");
    if ((uint64_t)n_heads * D > 0xffffffffull || (uint64_t)n_kv * D > 0xffffffffull || (uint64_t)n_heads + 2ull * n_kv > 0x00ffffffull)
        return set_error(FK_ERR_UNSUPPORTED, "rope_paged_store: too many heads");
    if (q_stride < n_heads * D || q_out_stride < n_heads * D || k_stride < n_kv * D || v_stride < n_kv * D)
        return set_error(FK_ERR_INVALID, "rope_paged_store: a row stride is shorter than the row");
    if ((q_stride | q_out_stride | k_stride | v_stride) % 8) return set_error(FK_ERR_INVALID, "rope_paged_store: strides must be multiples of 8 elements");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & 15u)
        return set_error(FK_ERR_INVALID, "rope_paged_store: pointers must be 16-byte aligned");
    if (((uintptr_t)q_norm | (uintptr_t)k_norm) & 1u) return set_error(FK_ERR_INVALID, "rope_paged_store: norms must be 2-byte aligned");
    if (!(eps >= 0.f)) return set_error(FK_ERR_INVALID, "rope_paged_store: eps must not be negative");
    const size_t qw = (size_t)n_heads * D, kw = (size_t)n_kv * D;
    if (!(q_out == q && q_out_stride == q_stride) && rows_overlap(q, q_stride, qw, q_out, q_out_stride, qw, batch->rows))
        return set_error(FK_ERR_INVALID, "rope_paged_store: q_out must be q, with its stride, or not overlap it");
    if (rows_overlap(k, k_stride, kw, q_out, q_out_stride, qw, batch->rows) || rows_overlap(v, v_stride, kw, q_out, q_out_stride, qw, batch->rows))
        return set_error(FK_ERR_INVALID, "rope_paged_store: q_out overlaps k or v");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.q_norm = q_norm; a.k_norm = k_norm;
    a.k_pages = pool->k; a.v_pages = pool->v; a.freq = freq;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
    a.n_heads = n_heads; a.rope_dims = rope_dims; a.eps = eps;
    l->func = D == 64 ? (interleaved ? reinterpret_cast<const void*>(&rope_paged_store_kernel<64, true>) : reinterpret_cast<const void*>(&rope_paged_store_kernel<64, false>))
                      : (interleaved ? reinterpret_cast<const void*>(&rope_paged_store_kernel<128, true>) : reinterpret_cast<const void*>(&rope_paged_store_kernel<128, false>));
    l->grid = dim3(batch->rows, 1, 1);
    l->block = dim3(256, 1, 1);
    l->set_args(a);
    return FK_OK;
}

// ---- pages copied inside a pool ----
// The pairs travel in the kernel's argument block: no upload, and nothing for a caller to keep alive.  480 of them fill it.  A block for each page, plane
// and 4 KB, up to 64 a page and plane: four pages of 4 KB in 48 planes 2.5 us, 307 pages of 32 KB in 72 planes 285 us, 5.1 TB/s
// read and written (a copy of 4 GB: 4.75).
constexpr uint32_t kPagePairs = 480;
struct PagesCopyArgs {
    unsigned char* base;
    size_t plane_stride, page_bytes;
    uint32_t pairs[2 * kPagePairs];
};
__global__ __launch_bounds__(256) void pages_copy_kernel(const PagesCopyArgs a) {
    const uint32_t from = a.pairs[2 * blockIdx.x], to = a.pairs[2 * blockIdx.x + 1];
    unsigned char* plane = a.base + (size_t)blockIdx.y * a.plane_stride;
    const uint4* src = reinterpret_cast<const uint4*>(plane + (size_t)from * a.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(plane + (size_t)to * a.page_bytes);
    for (size_t i = (size_t)blockIdx.z * 256 + threadIdx.x; i < a.page_bytes / 16; i += (size_t)gridDim.z * 256) dst[i] = src[i];
}

fk_status run_pages_copy(void* base, uint32_t n_planes, size_t plane_stride, uint32_t n_pages, size_t page_bytes, const uint32_t* pairs,
                         uint32_t n_pairs, hipStream_t s) {
    if (n_pairs == 0) return FK_OK;
    if (!base || !pairs) return set_error(FK_ERR_INVALID, "pages_copy: null pointer");
    if (n_planes == 0 || n_pages == 0 || page_bytes == 0) return set_error(FK_ERR_INVALID, "pages_copy: empty pool");
    if (page_bytes % 16 || plane_stride % 16 || (uintptr_t)base % 16) return set_error(FK_ERR_INVALID, "pages_copy: base, page_bytes and plane_stride must be multiples of 16");
    if (page_bytes > SIZE_MAX / n_pages) return set_error(FK_ERR_UNSUPPORTED, "pages_copy: pool too large");
    if (n_planes > 1 && plane_stride < page_bytes * n_pages) return set_error(FK_ERR_INVALID, "pages_copy: planes overlap");
    if (n_planes > 65535) return set_error(FK_ERR_UNSUPPORTED, "pages_copy: more than 65535 planes");
    // what is read, then what is written, in order: a page that is written twice, or read and written, stands next to itself
    uint32_t* order = new (std::nothrow) uint32_t[(size_t)n_pairs * 2];
    if (!order) return set_error(FK_ERR_UNSUPPORTED, "pages_copy: out of host memory");
    const char* wrong = nullptr;
    for (uint32_t i = 0; i < n_pairs; ++i) {
        order[i] = pairs[2 * (size_t)i];
        order[(size_t)n_pairs + i] = pairs[2 * (size_t)i + 1];
        if (pairs[2 * (size_t)i] >= n_pages || pairs[2 * (size_t)i + 1] >= n_pages) wrong = "pages_copy: a page that the pool does not have";
    }
    std::sort(order, order + n_pairs);
    std::sort(order + n_pairs, order + 2 * (size_t)n_pairs);
    for (size_t i = 0, j = n_pairs; !wrong && j < 2 * (size_t)n_pairs; ++j) {
        if (j > n_pairs && order[j] == order[j - 1]) wrong = "pages_copy: a page is written twice";
        while (i < n_pairs && order[i] < order[j]) ++i;
        if (i < n_pairs && order[i] == order[j]) wrong = "pages_copy: a page is both read and written";
    }
    delete[] order;
    if (wrong) return set_error(FK_ERR_INVALID, wrong);
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    PagesCopyArgs a;
    a.base = static_cast<unsigned char*>(base);
    a.plane_stride = plane_stride;
    a.page_bytes = page_bytes;
    for (uint32_t at = 0; at < n_pairs; at += kPagePairs) {
        const uint32_t n = std::min(kPagePairs, n_pairs - at);
        memcpy(a.pairs, pairs + 2 * (size_t)at, (size_t)n * 8);
        const uint32_t parts = (uint32_t)std::min<size_t>((page_bytes / 16 + 255) / 256, 64);
        void* params[1] = {&a};
        FK_HIP(hipLaunchKernel(reinterpret_cast<const void*>(&pages_copy_kernel), dim3(n, n_planes, parts), dim3(256), params, 0, s));
    }
    return FK_OK;
}

}  // namespace fk
