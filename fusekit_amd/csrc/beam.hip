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

constexpr uint32_t kBeamMax = 64, kBeamGroups = 4096;
constexpr size_t kBeamCounterBytes = 4 * kBeamGroups;   // at the same place for every shape: a workspace serves one call after another

// One launch.  A block takes a piece of a row: it leaves the piece's largest logit, its sum of exponentials and its k largest logits in order; the
// block of a group that comes last forms lse and the k best of what all pieces left.  The pieces are cut by token, never by address: rows that
// hold the same values have the same sums wherever they lie, so that ties between beams stay ties.
//
// The k largest of a piece without sorting it: the k-th largest of the 256 threads' largest values is a bound that at least k values reach and few
// more (16 of 256: 17 on average); found by bisection over its 16 bits with ballots.  What reaches it is collected in LDS and ranked by counting.
// Only a piece full of ties has more than fit there: its k largest are then taken one by one.
struct BeamArgs {
    const uint16_t* logits;
    size_t row_stride;
    const float* scores;
    const uint32_t* finished;
    uint32_t pad, beams, vocab, k, pieces;
    float* out_scores;
    uint32_t* out_beams;
    uint32_t* out_tokens;
    uint32_t* arrived;   // [groups], zero before the first launch, left zero
    double* sums;        // [groups * beams][pieces]
    float* tops;         // [groups * beams][pieces]
    uint32_t* best;      // [groups * beams][pieces][k]: (order of the logit << 16) | (65535 - place in the piece), 0 where there are no more
};

constexpr uint32_t kBeamList = 512;   // candidates that fit in LDS

__device__ __forceinline__ double wave_sum_wide(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The largest bound that at least k of the block's 256 values reach, or 1 where fewer than k are not 0; `all`: LDS, 256 words.
template <int BITS, int LOW>
__device__ __forceinline__ uint32_t bound_of_best(uint32_t mine, uint32_t k, uint32_t* all) {
    const uint32_t lane = threadIdx.x & 63u;
    all[threadIdx.x] = mine;
    __syncthreads();
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = all[lane + 64u * i];
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = LOW + BITS - 1; bit >= LOW; --bit) {
        const uint32_t at = t | (1u << bit);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= at));
        if (n >= k) t = at;
    }
    return t ? t : 1u;
}

template <int VEC>   // 16-byte loads of a thread
__global__ __launch_bounds__(256) void beam_select_kernel(const BeamArgs a) {
    constexpr uint32_t PIECE = 2048u * VEC;
    typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));   // (rows of an odd length start anywhere)
    __shared__ uint32_t all[256];
    __shared__ uint32_t list[kBeamList];
    __shared__ double values[kBeamList], part[4], base[kBeamMax];
    __shared__ uint32_t n_list, flag;
    __shared__ float top[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t piece = blockIdx.x, row = blockIdx.y, g = row / a.beams, k = a.k;
    const uint32_t from = piece * PIECE, left = a.vocab - from;
    const bool over = a.finished && a.finished[row];   // (the same for the block)
    if (!over) {
        const uint16_t* x = a.logits + (size_t)row * a.row_stride + from;
        loose w[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const uint32_t at = ((uint32_t)i * 256u + tid) * 8u;
            if (at + 8u <= left) {
                w[i] = *reinterpret_cast<const loose*>(x + at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = at + 2u * e < left ? x[at + 2u * e] : 0xff80u, hi = at + 2u * e + 1u < left ? x[at + 2u * e + 1u] : 0xff80u;
                    w[i][e] = lo | hi << 16;
                }
            }
        }
        // (a NaN counts as -inf: the larger of the two)
        auto value = [&](int i, int e) { return fmaxf(e & 1 ? bf16_hi(w[i][e >> 1]) : bf16_lo(w[i][e >> 1]), -INFINITY); };
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, value(i, e));
        const float mw = wave_max(m), ref = mw == -INFINITY ? 0.f : mw;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float s8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s8[e] = __builtin_amdgcn_exp2f((value(i, e) - ref) * 1.44269504088896341f);
            sum += (double)((s8[0] + s8[1]) + (s8[2] + s8[3])) + (double)((s8[4] + s8[5]) + (s8[6] + s8[7]));
        }
        sum = wave_sum_wide(sum);
        if (lane == 0) {
            top[wave] = mw;
            part[wave] = sum;
        }
        if (tid == 0) n_list = 0;
        const uint32_t bound = bound_of_best<16, 16>(m == -INFINITY ? 0u : order_key(m + 0.0f), k, all);   // (-0 as 0)
        const float least = __uint_as_float(bound >= 0x80000000u ? (bound & 0x7fff0000u) : (~bound & 0xffff0000u));   // (bound 1: a NaN's pattern)
        const bool any = bound < 0x10000u;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = value(i, e);
                if (v > -INFINITY && (any || v >= least)) {
                    const uint32_t at = atomicAdd(&n_list, 1u);
                    if (at < kBeamList) list[at] = (order_key(v + 0.0f) & 0xffff0000u) | (0xffffu - (((uint32_t)i * 256u + tid) * 8u + e));
                }
            }
        __syncthreads();
        const uint32_t n = n_list;
        uint32_t* const out = a.best + ((size_t)row * a.pieces + piece) * k;
        if (n <= kBeamList) {
            for (uint32_t c = tid; c < n; c += 256u) {
                const uint32_t mine = list[c];
                uint32_t rank = 0;
                for (uint32_t o = 0; o < n; ++o) rank += list[o] > mine ? 1u : 0u;
                if (rank < k) __hip_atomic_store(&out[rank], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            for (uint32_t c = n + tid; c < k; c += 256u) __hip_atomic_store(&out[c], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else {
            uint32_t last = ~0u;
            for (uint32_t c = 0; c < k; ++c) {
                uint32_t best = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float v = value(i, e);
                        const uint32_t key = v > -INFINITY ? (order_key(v + 0.0f) & 0xffff0000u) | (0xffffu - (((uint32_t)i * 256u + tid) * 8u + e)) : 0u;
                        best = key < last && key > best ? key : best;
                    }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    const uint32_t other = __shfl_xor(best, o, 64);
                    best = other > best ? other : best;
                }
                __syncthreads();
                if (lane == 0) all[wave] = best;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 4; ++i) best = all[i] > best ? all[i] : best;
                if (tid == 0) __hip_atomic_store(&out[c], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = best;   // (0: nothing is left, and nothing is below it)
            }
        }
        if (tid == 0) {
            const float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), rt = mt == -INFINITY ? 0.f : mt;
            double s = 0.0;
            for (int i = 0; i < 4; ++i) s += part[i] * (double)__builtin_amdgcn_exp2f((top[i] - rt) * 1.44269504088896341f);
            const size_t at = (size_t)row * a.pieces + piece;
            __hip_atomic_store(&a.tops[at], mt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(reinterpret_cast<unsigned long long*>(&a.sums[at]), (unsigned long long)__double_as_longlong(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }

    // ---- the group's last block ----
    wait_memory_ops_done();
    __syncthreads();
    if (tid == 0) flag = atomicAdd(&a.arrived[g], 1u) == a.beams * a.pieces - 1u ? 1u : 0u;
    __syncthreads();
    if (!flag) return;
    if (tid == 0) {
        __hip_atomic_store(&a.arrived[g], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        n_list = 0;
    }
    for (uint32_t b = wave; b < a.beams; b += 4u) {
        const uint32_t r = g * a.beams + b;
        const float score = a.scores[r];
        if (a.finished && a.finished[r]) {
            if (lane == 0) base[b] = (double)score;
            continue;
        }
        float m = -INFINITY;
        for (uint32_t p = lane; p < a.pieces; p += 64u) m = fmaxf(m, __hip_atomic_load(&a.tops[(size_t)r * a.pieces + p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        m = wave_max(m);
        double s = 0.0;
        for (uint32_t p = lane; p < a.pieces; p += 64u) {
            const size_t at = (size_t)r * a.pieces + p;
            const float mp = __hip_atomic_load(&a.tops[at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const double sp = __longlong_as_double((long long)__hip_atomic_load(reinterpret_cast<unsigned long long*>(&a.sums[at]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            if (mp > -INFINITY) s += sp * exp((double)mp - (double)m);
        }
        s = wave_sum_wide(s);
        if (lane == 0) base[b] = (double)score - ((double)m + log(s));
    }
    __syncthreads();
    const uint32_t row_n = a.pieces * k, total = a.beams * row_n;
    const uint32_t* const group_best = a.best + (size_t)g * total;
    // candidate i of the group: its score and its place, or -inf
    auto candidate = [&](uint32_t i, uint32_t key, uint64_t& flat) {
        const uint32_t b = i / row_n, j = i - b * row_n;
        if (a.finished && a.finished[g * a.beams + b]) {
            flat = (uint64_t)b * a.vocab + a.pad;
            return j == 0 ? base[b] : (double)-INFINITY;
        }
        flat = (uint64_t)b * a.vocab + (j / k) * PIECE + (0xffffu - (key & 0xffffu));
        const uint32_t o = key & 0xffff0000u;
        const double v = base[b] + (double)__uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o & 0xffff0000u);
        return key && v > -INFINITY ? v : (double)-INFINITY;
    };
    constexpr uint32_t AHEAD = 8;
    auto load = [&](uint32_t i) { return i < total ? __hip_atomic_load(&group_best[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u; };
    // (of a finished row nothing was written: its keys are not looked at, whatever they are)
    uint32_t mine = 0;
    uint32_t kept[AHEAD];
    for (uint32_t at = 0; at < total; at += 256u * AHEAD) {
        uint32_t key[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) key[u] = load(at + u * 256u + tid);
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t i = at + u * 256u + tid;
            if (i >= total) continue;
            uint64_t flat;
            const double v = candidate(i, key[u], flat);
            if (v > -INFINITY) {
                const uint32_t o = order_key((float)v);
                mine = o > mine ? o : mine;
            }
        }
        if (at == 0) {
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) kept[u] = key[u];
        }
    }
    const uint32_t bound = bound_of_best<32, 0>(mine, k, all);
    auto collect = [&](uint32_t i, uint32_t key) {
        if (i >= total) return;
        uint64_t flat;
        const double v = candidate(i, key, flat);
        if (v > -INFINITY && order_key((float)v) >= bound) {
            const uint32_t at = atomicAdd(&n_list, 1u);
            if (at < kBeamList) {
                list[at] = i;
                values[at] = v;
            }
        }
    };
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; ++u) collect(u * 256u + tid, kept[u]);
    for (uint32_t i = 256u * AHEAD + tid; i < total; i += 256u) collect(i, load(i));
    __syncthreads();
    uint32_t n = n_list;
    auto put = [&](uint32_t at, double v, uint64_t flat) {
        a.out_scores[(size_t)g * k + at] = (float)v;
        a.out_beams[(size_t)g * k + at] = (uint32_t)(flat / a.vocab);
        a.out_tokens[(size_t)g * k + at] = (uint32_t)(flat % a.vocab);
    };
    if (n <= kBeamList) {
        // their places in LDS too, then each one's rank by counting
        __shared__ uint64_t flats[kBeamList];
        for (uint32_t c = tid; c < n; c += 256u) {
            uint64_t flat;
            candidate(list[c], load(list[c]), flat);
            flats[c] = flat;
        }
        __syncthreads();
        for (uint32_t c = tid; c < n; c += 256u) {
            const double v = values[c];
            const uint64_t flat = flats[c];
            uint32_t rank = 0;
            for (uint32_t o = 0; o < n; ++o) rank += values[o] > v || (values[o] == v && flats[o] < flat) ? 1u : 0u;
            if (rank < k) put(rank, v, flat);
        }
        if (n >= k || tid != 0) return;
        // fewer than k above -inf: the lowest places that are not among them
        uint64_t at = 0;
        for (uint32_t i = n; i < k; ++i, ++at) {
            for (bool again = true; again;) {
                again = false;
                for (uint32_t c = 0; c < n; ++c)
                    if (flats[c] == at) {
                        ++at;
                        again = true;
                    }
            }
            put(i, -INFINITY, at);
        }
        return;
    }
    // ties beyond the list: one by one
    double last = INFINITY;
    uint64_t last_at = 0;
    for (uint32_t c = 0; c < k; ++c) {
        double best = -INFINITY;
        uint64_t at = ~0ull;
        for (uint32_t i = tid; i < total; i += 256u) {
            uint64_t flat;
            const double v = candidate(i, load(i), flat);
            if (!(v > -INFINITY) || (c && !(v < last || (v == last && flat > last_at)))) continue;
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
        __syncthreads();
        if (lane == 0) {
            values[wave] = best;
            values[4 + wave] = __longlong_as_double((long long)at);
        }
        __syncthreads();
        for (int i = 0; i < 4; ++i) {
            const double ov = values[i];
            const uint64_t oa = (uint64_t)__double_as_longlong(values[4 + i]);
            if (ov > best || (ov == best && oa < at)) {
                best = ov;
                at = oa;
            }
        }
        last = best;
        last_at = at;
        if (tid == 0) put(c, best, at);   // (more than fit into the list: k of them exist)
    }
}

// Pieces of 8192 tokens where that makes two blocks a CU, else of 2048.
static uint32_t beam_piece(uint32_t groups, uint32_t beams, uint32_t vocab) { return (uint64_t)groups * beams * ((vocab + 8191u) / 8192u) >= 512u ? 8192u : 2048u; }

fk_status beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t k, size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "beam_select workspace: null pointer");
    if (groups == 0 || beams == 0 || vocab == 0 || k == 0) return set_error(FK_ERR_INVALID, "beam_select: empty shape");
    if (beams > kBeamMax || k > kBeamMax) return set_error(FK_ERR_UNSUPPORTED, "beam_select: beams and k up to 64");
    if (groups > kBeamGroups) return set_error(FK_ERR_UNSUPPORTED, "beam_select: more than 4096 groups");
    if ((uint64_t)groups * beams > 65535) return set_error(FK_ERR_UNSUPPORTED, "beam_select: more than 65535 beams in all groups");
    if (k > (uint64_t)beams * vocab) return set_error(FK_ERR_INVALID, "beam_select: k exceeds the continuations of a group");
    const size_t rows = (size_t)groups * beams, pieces = ((size_t)vocab + 2047) / 2048;   // (the smaller pieces, whichever are taken)
    if (pieces > 65535) return set_error(FK_ERR_UNSUPPORTED, "beam_select: vocabulary too large");
    *bytes = kBeamCounterBytes + rows * pieces * (12 + 4 * (size_t)k);
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
    const uint32_t piece = beam_piece(groups, beams, vocab), pieces = (vocab + piece - 1) / piece;
    const size_t rows = (size_t)groups * beams;
    BeamArgs a{logits, row_stride, scores, finished, pad_token, beams, vocab, k, pieces, out_scores, out_beams, out_tokens, nullptr, nullptr, nullptr, nullptr};
    a.arrived = static_cast<uint32_t*>(workspace);
    a.sums = reinterpret_cast<double*>(static_cast<unsigned char*>(workspace) + kBeamCounterBytes);
    a.tops = reinterpret_cast<float*>(a.sums + rows * pieces);
    a.best = reinterpret_cast<uint32_t*>(a.tops + rows * pieces);
    l->func = piece == 8192 ? reinterpret_cast<const void*>(&beam_select_kernel<4>) : reinterpret_cast<const void*>(&beam_select_kernel<1>);
    l->grid = dim3(pieces, (uint32_t)rows, 1);
    l->block = dim3(256, 1, 1);
    l->set_args(a);
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
