// Attention of new rows -- chunks of prompts, single tokens, both in one batch -- over a paged cache.
//
//     out[r, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(x_j - max x),   x_j = c(q[r, h] . K[j] * scale),   max(0, p - window + 1) <= j <= p
//
// with p the row's position and c(x) = x, or softcap * tanh(x / softcap).
#include <math.h>

#include "fk_host.hpp"
#include "paged_device.hpp"

namespace fk {

// Probabilities carry this factor, which cancels: a sum of 2^24 of them times the type's largest values stays in fp32's range.
constexpr float kSmall = 0x1p-32f;

struct SdpaPagedArgs {
    PagedArgs b;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    uint32_t q_stride, out_stride, n_heads, group;
    uint32_t window;
    float scale, softcap;
};

// A wave a (row, head).  64 positions at a time: a lane forms one score, then the lanes share out the dims.
template <int D>
__global__ __launch_bounds__(64) void sdpa_paged_row_kernel(const SdpaPagedArgs a) {
    const uint32_t lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kvh = head / a.group;
    const uint32_t seq = paged_seq_of(a.b, row, lane);
    if (seq >= a.b.n_seqs) return;
    const PagedSeq s = paged_seq(a.b, seq);
    uint32_t bad = s.bad;
    if (bad && lane == 0) paged_fault(a.b, bad);
    const uint32_t place = row - s.row0;
    if (row < s.row0 || place >= s.rows) return;
    const uint32_t page_rows = 1u << a.b.page_shift;
    const uint32_t end = s.len + place + 1u > s.rows ? s.len + place + 1u - s.rows : 0u;   // positions up to the row's own
    const uint32_t first = a.window && end > a.window ? end - a.window : 0u;
    const uint16_t* qr = a.q + (size_t)row * a.q_stride + (size_t)head * D;
    constexpr int DL = D / 64;
    float m = -INFINITY, l = 0.f, o[DL];
#pragma unroll
    for (int i = 0; i < DL; ++i) o[i] = 0.f;
    for (uint32_t at = first; at < end; at += 64u) {
        const uint32_t pos = at + lane < end ? at + lane : end - 1u;
        const uint32_t page = paged_page(a.b, seq, pos >> a.b.page_shift, bad);
        const size_t base = (((size_t)page * a.b.n_kv + kvh) * page_rows + (pos & (page_rows - 1u))) * D;
        const uint4* kr = reinterpret_cast<const uint4*>(a.k + base);
        float x = 0.f;
        for (int i = 0; i < D / 8; ++i) {
            const uint4 kk = kr[i], qq = reinterpret_cast<const uint4*>(qr)[i];
            const uint32_t kw[4] = {kk.x, kk.y, kk.z, kk.w}, qw[4] = {qq.x, qq.y, qq.z, qq.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) x = fmaf(bf16_hi(kw[e]), bf16_hi(qw[e]), fmaf(bf16_lo(kw[e]), bf16_lo(qw[e]), x));
        }
        x *= a.scale;
        if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
        if (at + lane >= end) x = -INFINITY;
        const float m_new = fmaxf(m, wave_max(x)), ref = m_new == -INFINITY ? 0.f : m_new, alpha = expf(m - ref), p = expf(x - ref) * kSmall;
        l = l * alpha + wave_sum(p);
        m = m_new;
#pragma unroll
        for (int i = 0; i < DL; ++i) o[i] *= alpha;
        const uint32_t n = end - at < 64u ? end - at : 64u;
        for (uint32_t j = 0; j < n; ++j) {
            const float pj = __shfl(p, (int)j, 64);
            const size_t vb = __shfl((unsigned long long)base, (int)j, 64);
#pragma unroll
            for (int i = 0; i < DL; ++i) o[i] = fmaf(pj, bf16_bits_to_f32(a.v[vb + lane + 64u * i]), o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < DL; ++i)
        a.out[(size_t)row * a.out_stride + (size_t)head * D + lane + 64u * i] = (uint16_t)f32_to_bf16_bits(end > first ? o[i] / l : 0.f);
    if (__builtin_amdgcn_ballot_w64(bad != 0)) {
        if (bad) paged_fault(a.b, bad);
    }
}

fk_status sdpa_paged_workspace_bytes(uint32_t n_heads, uint32_t n_kv, uint32_t head_dim, uint32_t n_seqs, uint32_t rows, uint32_t max_len,
                                     size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "sdpa_paged workspace: null pointer");
    if (n_heads == 0 || n_kv == 0 || n_heads % n_kv || n_seqs == 0 || rows == 0 || max_len == 0)
        return set_error(FK_ERR_INVALID, "sdpa_paged workspace: empty shape, or n_heads not a multiple of n_kv");
    if (head_dim != 64 && head_dim != 128) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged workspace: head dimension 64 or 128");
    *bytes = 4096;
    return FK_OK;
}

fk_status plan_sdpa_paged(const uint16_t* q, uint32_t q_stride, uint16_t* out, uint32_t out_stride, uint32_t n_heads, float scale, float softcap,
                          uint32_t window, const fk_paged_batch* batch, const fk_page_pool* pool, void* workspace, size_t workspace_bytes, Launch* l) {
    SdpaPagedArgs a;
    memset(&a, 0, sizeof(a));
    FK_TRY(paged_args("sdpa_paged", batch, pool, &a.b));
    const uint32_t D = pool->head_dim, n_kv = pool->n_kv;
    if (!q || !out || !workspace) return set_error(FK_ERR_INVALID, "sdpa_paged: null pointer");
    if (n_heads == 0 || n_heads % n_kv) return set_error(FK_ERR_INVALID, "sdpa_paged: n_heads must be a multiple of n_kv");
    if (n_heads > 65535) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: too many heads");
    if (q_stride < n_heads * D || out_stride < n_heads * D) return set_error(FK_ERR_INVALID, "sdpa_paged: a row stride is shorter than the row");
    if ((q_stride | out_stride) % 8) return set_error(FK_ERR_INVALID, "sdpa_paged: strides must be multiples of 8 elements");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15u) return set_error(FK_ERR_INVALID, "sdpa_paged: pointers must be 16-byte aligned");
    if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(FK_ERR_INVALID, "sdpa_paged: scale must be positive");
    if (!(softcap >= 0.f) || !std::isfinite(softcap)) return set_error(FK_ERR_INVALID, "sdpa_paged: softcap must not be negative");
    size_t need = 0;
    FK_TRY(sdpa_paged_workspace_bytes(n_heads, n_kv, D, batch->n_seqs, batch->rows, batch->max_len, &need));
    if (workspace_bytes < need) return set_error(FK_ERR_INVALID, "sdpa_paged: workspace too small");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    a.q = q; a.k = pool->k; a.v = pool->v; a.out = out;
    a.q_stride = q_stride; a.out_stride = out_stride; a.n_heads = n_heads; a.group = n_heads / n_kv;
    a.window = window; a.scale = scale; a.softcap = softcap;
    l->func = D == 64 ? reinterpret_cast<const void*>(&sdpa_paged_row_kernel<64>) : reinterpret_cast<const void*>(&sdpa_paged_row_kernel<128>);
    l->grid = dim3(batch->rows, n_heads, 1);
    l->block = dim3(64, 1, 1);
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
