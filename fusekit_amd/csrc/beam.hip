// Beam search: the k best continuations of each group's beams, and state rows that follow the beams chosen.
//
//     total[b, t] = score[b] + logit[b, t] - lse[b],   lse[b] = m + log sum_t exp(logit[b, t] - m)
//
// The k best of a group in order, ties to the lower b * vocab + t.  Inside a row the order is that of the logits, so a row
// contributes only its k largest logits; rows are then compared in 64 bits.
#include <math.h>

#include "argmax_tail.hpp"
#include "fk_host.hpp"

namespace fk {

constexpr uint32_t kBeamMax = 64;

struct BeamArgs {
    const uint16_t* logits;
    size_t row_stride;
    const float* scores;
    const uint32_t* finished;
    uint32_t pad, groups, beams, vocab, k;
    float* out_scores;
    uint32_t* out_beams;
    uint32_t* out_tokens;
    double* base;      // [groups * beams]: score - lse
    uint64_t* best;    // [groups * beams][k]: (order of the logit << 32) | ~token, 0 where the row has no more
};

// a NaN counts as -inf; -0 as 0
__device__ __forceinline__ float beam_logit(uint32_t bits) {
    const float v = bf16_bits_to_f32(bits);
    return v != v ? -INFINITY : v + 0.0f;
}

__global__ __launch_bounds__(256) void beam_rows_kernel(const BeamArgs a) {
    __shared__ float red[8];
    __shared__ uint64_t win[4];
    __shared__ double part[4];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const uint16_t* x = a.logits + (size_t)row * a.row_stride;
    float m = -INFINITY;
    for (uint32_t t = tid; t < a.vocab; t += 256u) m = fmaxf(m, beam_logit(x[t]));
    m = block_max<256>(m, red);
    double sum = 0.0;
    for (uint32_t t = tid; t < a.vocab; t += 256u) sum += (double)expf(beam_logit(x[t]) - m);
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((tid & 63u) == 0) part[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) a.base[row] = (double)a.scores[row] - ((double)m + log((part[0] + part[1]) + (part[2] + part[3])));
    uint64_t last = ~0ull;
    for (uint32_t i = 0; i < a.k; ++i) {
        uint64_t best = 0;
        for (uint32_t t = tid; t < a.vocab; t += 256u) {
            const uint64_t c = ((uint64_t)order_key(beam_logit(x[t])) << 32) | (uint32_t)~t;
            if (c < last && c > best) best = c;
        }
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor(best, o, 64);
            best = other > best ? other : best;
        }
        if ((tid & 63u) == 0) win[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < 4; ++w) best = win[w] > best ? win[w] : best;
        __syncthreads();
        last = best;
        if (tid == 0) a.best[(size_t)row * a.k + i] = best;
        if (best == 0) last = 1;   // nothing is left: every further one is 0 too
    }
}

__device__ __forceinline__ float order_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// One wave a group.
__global__ __launch_bounds__(64) void beam_merge_kernel(const BeamArgs a) {
    __shared__ uint64_t chosen[kBeamMax];
    const uint32_t g = blockIdx.x, lane = threadIdx.x;
    const uint64_t vocab = a.vocab;
    double last = INFINITY;
    uint64_t last_at = 0;
    bool any = false;
    uint32_t n = 0;
    for (; n < a.k; ++n) {
        double best = -INFINITY;
        uint64_t at = ~0ull;
        for (uint32_t c = lane; c < a.beams * a.k; c += 64u) {
            const uint32_t b = c / a.k, row = g * a.beams + b;
            double v;
            uint32_t t;
            if (a.finished && a.finished[row]) {
                if (c % a.k) continue;
                v = a.scores[row];
                t = a.pad;
            } else {
                const uint64_t e = a.best[(size_t)row * a.k + c % a.k];
                if (!e) continue;
                v = a.base[row] + (double)order_value((uint32_t)(e >> 32));
                t = ~(uint32_t)e;
            }
            if (!(v > -INFINITY)) continue;
            const uint64_t flat = b * vocab + t;
            if (any && !(v < last || (v == last && flat > last_at))) continue;   // chosen before
            if (v > best || (v == best && flat < at)) {
                best = v;
                at = flat;
            }
        }
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(best, o, 64);
            const uint64_t oa = __shfl_xor(at, o, 64);
            if (ov > best || (ov == best && oa < at)) {
                best = ov;
                at = oa;
            }
        }
        if (at == ~0ull) break;
        last = best;
        last_at = at;
        any = true;
        if (lane == 0) {
            chosen[n] = at;
            a.out_scores[(size_t)g * a.k + n] = (float)best;
            a.out_beams[(size_t)g * a.k + n] = (uint32_t)(at / vocab);
            a.out_tokens[(size_t)g * a.k + n] = (uint32_t)(at % vocab);
        }
    }
    if (lane != 0) return;
    // nothing above -inf is left: the lowest places that were not chosen
    uint64_t at = 0;
    for (uint32_t found = n; n < a.k; ++n, ++at) {
        for (bool again = true; again;) {
            again = false;
            for (uint32_t i = 0; i < found; ++i)
                if (chosen[i] == at) {
                    ++at;
                    again = true;
                }
        }
        a.out_scores[(size_t)g * a.k + n] = -INFINITY;
        a.out_beams[(size_t)g * a.k + n] = (uint32_t)(at / vocab);
        a.out_tokens[(size_t)g * a.k + n] = (uint32_t)(at % vocab);
    }
}

fk_status beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k, size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "beam_select workspace: null pointer");
    if (groups == 0 || beams == 0 || vocab == 0 || k == 0) return set_error(FK_ERR_INVALID, "beam_select: empty shape");
    if (beams > kBeamMax || k > kBeamMax) return set_error(FK_ERR_UNSUPPORTED, "beam_select: beams and k up to 64");
    if ((uint64_t)groups * beams > 65535) return set_error(FK_ERR_UNSUPPORTED, "beam_select: more than 65535 beams in all groups");
    if (k > (uint64_t)beams * vocab) return set_error(FK_ERR_INVALID, "beam_select: k exceeds the continuations of a group");
    *bytes = (size_t)groups * beams * 8 * (1 + k);
    return FK_OK;
}

fk_status plan_beam_select(const uint16_t* logits, size_t row_stride, const float* scores, const uint32_t* finished, uint32_t pad_token, uint32_t groups,
                           uint32_t beams, uint32_t vocab, uint32_t k, float* out_scores, uint32_t* out_beams, uint32_t* out_tokens, void* workspace,
                           size_t workspace_bytes, Launch* l) {
    size_t need = 0;
    FK_TRY(beam_select_workspace_bytes(groups, beams, vocab, k, &need));
    if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !workspace) return set_error(FK_ERR_INVALID, "beam_select: null pointer");
    if (row_stride < vocab) return set_error(FK_ERR_INVALID, "beam_select: row_stride is shorter than the vocabulary");
    if (finished && pad_token >= vocab) return set_error(FK_ERR_INVALID, "beam_select: pad_token outside of the vocabulary");
    if ((uintptr_t)logits & 1u || ((uintptr_t)scores | (uintptr_t)finished | (uintptr_t)out_scores | (uintptr_t)out_beams | (uintptr_t)out_tokens) & 3u ||
        (uintptr_t)workspace & 15u)
        return set_error(FK_ERR_INVALID, "beam_select: logits must be 2-byte, the other arrays 4-byte and the workspace 16-byte aligned");
    if (workspace_bytes < need) return set_error(FK_ERR_INVALID, "beam_select: workspace too small");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    BeamArgs a{logits, row_stride, scores, finished, pad_token, groups, beams, vocab, k, out_scores, out_beams, out_tokens, nullptr, nullptr};
    a.base = static_cast<double*>(workspace);
    a.best = reinterpret_cast<uint64_t*>(a.base + (size_t)groups * beams);
    l->func = reinterpret_cast<const void*>(&beam_rows_kernel);
    l->grid = dim3(groups * beams, 1, 1);
    l->block = dim3(256, 1, 1);
    l->set_args(a);
    Launch m;
    m.func = reinterpret_cast<const void*>(&beam_merge_kernel);
    m.grid = dim3(groups, 1, 1);
    m.block = dim3(64, 1, 1);
    m.set_args(a);
    l->then.push_back(m);
    return FK_OK;
}

// ---- rows of state that follow the beams ----
// A thread takes one column of a group: it reads that column of every row before it writes one, so that src may be dst.
struct ReorderArgs {
    const void* src;
    void* dst;
    size_t columns;
    const uint32_t* parents;
    uint32_t beams, n_out;
};
template <typename T, uint32_t N>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const ReorderArgs a) {
    const size_t c = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.columns) return;
    const uint32_t g = blockIdx.y;
    const T* src = static_cast<const T*>(a.src) + (size_t)g * a.beams * a.columns + c;
    T* dst = static_cast<T*>(a.dst) + (size_t)g * a.n_out * a.columns + c;
    T v[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        if (i < a.n_out) {
            const uint32_t p = a.parents[(size_t)g * a.n_out + i];
            v[i] = src[(size_t)(p < a.beams ? p : a.beams - 1u) * a.columns];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
        if (i < a.n_out) dst[(size_t)i * a.columns] = v[i];
}

fk_status plan_beam_reorder(const void* src, void* dst, size_t row_bytes, const uint32_t* parents, uint32_t groups, uint32_t beams, uint32_t n_out, Launch* l) {
    if (!src || !dst || !parents) return set_error(FK_ERR_INVALID, "beam_reorder: null pointer");
    if (row_bytes == 0 || groups == 0 || beams == 0 || n_out == 0) return set_error(FK_ERR_INVALID, "beam_reorder: empty shape");
    if (beams > kBeamMax || n_out > kBeamMax) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: beams up to 64");
    if (groups > 65535) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: more than 65535 groups");
    if ((uintptr_t)parents & 3u) return set_error(FK_ERR_INVALID, "beam_reorder: parents must be 4-byte aligned");
    if (row_bytes > (SIZE_MAX >> 1) / ((size_t)groups * kBeamMax)) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: state too large");
    const uintptr_t s0 = (uintptr_t)src, d0 = (uintptr_t)dst, sn = (size_t)groups * beams * row_bytes, dn = (size_t)groups * n_out * row_bytes;
    if (s0 == d0 ? n_out != beams : (s0 < d0 + dn && d0 < s0 + sn))
        return set_error(FK_ERR_INVALID, "beam_reorder: src and dst must be one buffer with n_out == beams, or not overlap");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    const uint32_t width = (s0 | d0 | row_bytes) % 16 == 0 ? 16 : (s0 | d0 | row_bytes) % 4 == 0 ? 4 : 1;
    ReorderArgs a{src, dst, row_bytes / width, parents, beams, n_out};
    if ((a.columns + 255) / 256 > 0x7fffffffu) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: rows too long");
    l->func = width == 16 ? reinterpret_cast<const void*>(&beam_reorder_kernel<uint4, kBeamMax>)
              : width == 4 ? reinterpret_cast<const void*>(&beam_reorder_kernel<uint32_t, kBeamMax>) : reinterpret_cast<const void*>(&beam_reorder_kernel<uint8_t, kBeamMax>);
    l->grid = dim3((uint32_t)((a.columns + 255) / 256), groups, 1);
    l->block = dim3(256, 1, 1);
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
