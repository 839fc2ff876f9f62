// Tokens drawn from rows of logits, each row with a temperature, top-k, top-p and min-p of its own, from given random numbers.
//
//     w_i = exp((x_i - max x) / T);   the tokens in the order of their logits, the largest first, ties to the lower token
//     of these the first top_k;   of what they weigh, W_k, the shortest run from the first on that weighs top_p W_k;   of that, those with w_i >= min_p
//     token: the first whose running sum is above u W, W the sum of what is left
//
// A bf16 row holds few distinct logits: its tokens are counted by logit, in LDS, and each weight is formed once, in 64 bits.  Weights are held as integers in
// units of 2^-shift of the largest, so that every sum is the same whatever the order and the cut of the row, and is off by half a unit a token at most.
#include <math.h>

#include <algorithm>

#include "fk_host.hpp"

namespace fk {

struct SampleArgs {
    const uint16_t* logits;
    size_t row_stride;
    const float* temperature;   // these four may be null
    const uint32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    uint32_t* tokens;
    float* logprobs;   // may be null
    uint32_t vocab;
    int shift;
};

constexpr uint32_t kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr uint32_t kSampleChunks = 165, kSampleBins = 64 * kSampleChunks;   // bins are looked at 64 at a time

// A logit's place among all that bf16 has, the largest first: 0 is infinity, kSampleRanks and more are not counted (-inf, NaN).
constexpr uint32_t kSampleRanks = 2 * 0x7f80;
__device__ __forceinline__ uint32_t sample_rank(uint32_t bits) {
    const uint32_t m = bits & 0x7fffu;
    if (m > 0x7f80u) return kSampleRanks;
    return bits & 0x8000u ? 0x7f80u + m : 0x7f80u - m;
}
__device__ __forceinline__ double sample_value(uint32_t rank) {
    return (double)__uint_as_float((rank < 0x7f80u ? 0x7f80u - rank : 0x8000u | (rank - 0x7f80u)) << 16);
}

struct SampleRow {
    double top, inv_t, unit;   // the largest logit, 1 / T, 2^shift
    bool infinite;             // the largest is infinity: what is equal to it weighs 1, everything else nothing
    __device__ __forceinline__ double weigh(uint32_t rank, double by) const { return infinite ? (rank == 0 ? 1.0 : 0.0) : exp((sample_value(rank) - top) * by); }
    __device__ __forceinline__ uint64_t weight(uint32_t rank) const { return (uint64_t)(weigh(rank, inv_t) * unit + 0.5); }
    __device__ __forceinline__ uint64_t plain(uint32_t rank) const { return (uint64_t)(weigh(rank, 1.0) * unit + 0.5); }   // at T = 1
};

__device__ __forceinline__ uint64_t lesser(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
    return v;
}
// The sum of this lane's and those before it.
template <typename T>
__device__ __forceinline__ T wave_upto(T v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T other = __shfl_up(v, o, 64);
        v += lane >= (uint32_t)o ? other : (T)0;
    }
    return v;
}

// Eight logits of a row from `at` on, a multiple of 8 below vocab; NaN behind its end (not counted).
__device__ __forceinline__ void sample_load(const uint16_t* x, uint32_t at, uint32_t vocab, uint32_t (&w)[4]) {
    typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));   // (rows of an odd length start anywhere)
    if (__builtin_expect(at + 8u <= vocab, 1)) {
        const loose v = *reinterpret_cast<const loose*>(x + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = at + 2u * e < vocab ? x[at + 2u * e] : 0x7fffu, hi = at + 2u * e + 1u < vocab ? x[at + 2u * e + 1u] : 0x7fffu;
            w[e] = lo | hi << 16;
        }
    }
}

// A block a row.  Its logits are counted in a window of kSampleBins ranks from the largest on; where the row goes on below, in another one.  The sums are
// walked three times, window by window: for W_k, for what is left, for the token.
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs a) {
    __shared__ uint32_t hist[kSampleBins], count[kSampleChunks];
    __shared__ uint64_t mass[kSampleChunks], plain[kSampleChunks];
    __shared__ uint32_t words[kSampleWaves], next, found_rank, found_place, over;
    __shared__ uint64_t sums[3];   // W_k, W, the plain sum
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, row = blockIdx.x;
    const uint16_t* const x = a.logits + (size_t)row * a.row_stride;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(t > 0.f);
    const uint32_t top_k = a.top_k ? a.top_k[row] : 0u, k = greedy ? 1u : top_k ? top_k : ~0u;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    float min_p = a.min_p ? a.min_p[row] : 0.f;
    min_p = min_p > 0.f ? fminf(min_p, 1.0f) : 0.f;
    const bool whole_p = !(top_p < 1.0f);

    // the largest
    uint32_t best = kSampleRanks;
    uint32_t w[4];
    for (uint32_t at = tid * 8u; at < a.vocab; at += kSampleThreads * 8u) {
        sample_load(x, at, a.vocab, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = sample_rank(w[e] & 0xffffu), hi = sample_rank(w[e] >> 16);
            best = min(best, min(lo, hi));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = min(best, (uint32_t)__shfl_xor((int)best, o, 64));
    if (lane == 0) words[wave] = best;
    __syncthreads();
    best = words[0];
#pragma unroll
    for (uint32_t i = 1; i < kSampleWaves; ++i) best = min(best, words[i]);
    if (best >= kSampleRanks) {   // nothing above -inf
        if (tid == 0) {
            a.tokens[row] = 0;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        return;
    }
    SampleRow r;
    r.infinite = best == 0;
    r.top = sample_value(best);
    r.inv_t = greedy ? 0.0 : 1.0 / (double)t;
    r.unit = (double)(1ull << a.shift);

    uint32_t built = ~0u;
    auto build = [&](uint32_t base) {
        if (built == base) return;
        built = base;
        for (uint32_t i = tid; i < kSampleBins; i += kSampleThreads) hist[i] = 0;
        if (tid == 0) next = kSampleRanks;
        __syncthreads();
        uint32_t below = kSampleRanks;
        for (uint32_t at = tid * 8u; at < a.vocab; at += kSampleThreads * 8u) {
            sample_load(x, at, a.vocab, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t rank = sample_rank(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu), bin = rank - base;
                if (bin < kSampleBins && rank < kSampleRanks) atomicAdd(&hist[bin], 1u);
                else if (rank > base) below = min(below, rank);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) below = min(below, (uint32_t)__shfl_xor((int)below, o, 64));
        if (lane == 0) atomicMin(&next, below);
        __syncthreads();
        for (uint32_t c = wave; c < kSampleChunks; c += kSampleWaves) {
            const uint32_t n = hist[c * 64u + lane];
            uint64_t m = 0, p = 0;
            uint32_t all = 0;
            if (__builtin_amdgcn_ballot_w64(n != 0)) {
                const uint32_t rank = base + c * 64u + lane;
                m = n ? n * r.weight(rank) : 0;
                p = a.logprobs && n ? n * r.plain(rank) : 0;
                all = (uint32_t)wave_sum_u64(n);
                m = wave_sum_u64(m);
                p = wave_sum_u64(p);
            }
            if (lane == 0) {
                count[c] = all;
                mass[c] = m;
                plain[c] = p;
            }
        }
        __syncthreads();
    };
    // Wave 0 walks a window's chunks, and of the first one that `whole(tokens, mass up to its end, its last rank)` does not take, the bins.  partial(tokens
    // before, mass before, count, rank) says how many of a bin's are taken; of the first bin that is not taken whole, `found` is told.
    uint64_t walked = 0, walked_mass = 0, walked_plain = 0;   // (wave 0's)
    auto walk = [&](uint32_t base, auto whole, auto partial, auto found) {
        if (wave != 0) return;
        for (uint32_t c0 = 0; c0 < kSampleChunks; c0 += 64u) {
            const uint32_t c = c0 + lane;
            const bool in = c < kSampleChunks;
            const uint64_t n = wave_upto((unsigned long long)(in ? count[c] : 0u), lane) + walked, m = wave_upto((unsigned long long)(in ? mass[c] : 0u), lane) + walked_mass;
            const bool stops = in && count[c] != 0 && !whole(n, m, base + c * 64u + 63u);
            const unsigned long long at = __builtin_amdgcn_ballot_w64(stops);
            const int last = at ? (int)__builtin_ctzll(at) : 63;
            const uint64_t before_n = __shfl((unsigned long long)(n - (in ? count[c] : 0u)), last, 64), before_m = __shfl((unsigned long long)(m - (in ? mass[c] : 0u)), last, 64);
            if (!at) {
                walked = __shfl((unsigned long long)n, 63, 64);
                walked_mass = __shfl((unsigned long long)m, 63, 64);
                continue;
            }
            const uint32_t bin = (c0 + (uint32_t)last) * 64u + lane, rank = base + bin, held = hist[bin];
            const uint64_t each = held ? r.weight(rank) : 0;
            const uint64_t bn = wave_upto((unsigned long long)held, lane) + before_n, bm = wave_upto((unsigned long long)(held * each), lane) + before_m;
            const uint64_t take = held ? partial(bn - held, bm - held * each, held, each) : 0;
            const unsigned long long cut = __builtin_amdgcn_ballot_w64(held != 0 && take < held);
            if (!cut) {   // (the chunk's last weight was below min_p, none of its logits' was)
                walked = __shfl((unsigned long long)bn, 63, 64);
                walked_mass = __shfl((unsigned long long)bm, 63, 64);
                // the chunks behind it, once more from here
                c0 = c0 + (uint32_t)last + 1u - 64u;
                continue;
            }
            if (lane == (uint32_t)__builtin_ctzll(cut)) {
                found(rank, take, bm - held * each + take * each);
                over = 1;
            }
            return;
        }
    };
    if (tid == 0) {
        sums[0] = sums[1] = sums[2] = 0;
        over = 0;
    }
    __syncthreads();
    // pass 0: W_k, and what everything weighs at T = 1; pass 1: W; pass 2: the token
    for (int pass = 0; pass < 3; ++pass) {
        if (pass == 0 && whole_p && !a.logprobs) continue;
        walked = walked_mass = 0;
        const uint64_t w_k = sums[0], limit = sums[1];
        const double need_real = (double)top_p * (double)w_k;
        const uint64_t need = whole_p ? ~0ull : top_p > 0.f ? (uint64_t)ceil(need_real) : 0u;
        const double least = (double)min_p * r.unit;
        const float uu = pass == 2 ? a.u[row] : 0.f;
        const double goal = uu > 0.f ? (double)uu * (double)limit : 0.0;
        const uint64_t target = goal < (double)limit ? lesser((uint64_t)goal, limit - 1u) : limit - 1u;
        __syncthreads();
        for (uint32_t base = best; base < kSampleRanks;) {
            build(base);
            if (pass == 0 && a.logprobs && wave == 0) {
                uint64_t p = 0;
                for (uint32_t c = lane; c < kSampleChunks; c += 64u) p += plain[c];
                walked_plain += wave_sum_u64(p);
            }
            if (pass == 0) {
                if (!over)
                    walk(base, [&](uint64_t n, uint64_t, uint32_t) { return n <= k; },
                         [&](uint64_t n, uint64_t, uint32_t held, uint64_t) { return n >= k ? (uint64_t)0 : lesser(held, k - n); },
                         [&](uint32_t, uint64_t, uint64_t m) { sums[0] = m; });
            } else if (pass == 1) {
                walk(base, [&](uint64_t n, uint64_t m, uint32_t rank) { return n <= k && m < need && (double)r.weight(rank < kSampleRanks ? rank : kSampleRanks - 1u) >= least; },
                     [&](uint64_t n, uint64_t m, uint32_t held, uint64_t each) {
                         uint64_t take = n >= k ? (uint64_t)0 : lesser(held, k - n);
                         if (m >= need) take = 0;
                         else if (each && need - m < take * each) take = (need - m + each - 1u) / each;
                         if ((double)each < least) take = 0;
                         if (n == 0 && take == 0) take = 1;   // the largest stays
                         return take;
                     },
                     [&](uint32_t, uint64_t, uint64_t m) { sums[1] = m; });
            } else {
                walk(base, [&](uint64_t, uint64_t m, uint32_t) { return m <= target; },
                     [&](uint64_t, uint64_t m, uint32_t held, uint64_t each) { return m > target ? (uint64_t)0 : each ? lesser(held, (target - m) / each) : (uint64_t)held; },
                     [&](uint32_t rank, uint64_t take, uint64_t) {
                         found_rank = rank;
                         found_place = (uint32_t)take;
                     });
            }
            __syncthreads();
            const uint32_t done = over, on = next;
            __syncthreads();
            if (done && !(pass == 0 && a.logprobs)) break;
            base = on;
            // (what weighs nothing from here on ends no sum)
            if (base < kSampleRanks && pass < 2 && r.weight(base) == 0 && (pass != 0 || !a.logprobs || r.plain(base) == 0)) break;
        }
        if (tid == 0 && pass < 2 && !over) sums[pass] = walked_mass;   // everything is in it
        if (tid == 0) {
            over = 0;
            if (pass == 0) sums[2] = walked_plain;
        }
        __syncthreads();
    }

    // the token: of those that hold the logit, in their order, the one at found_place
    const uint32_t rank = found_rank;
    uint32_t left = found_place;
    for (uint32_t at0 = 0; at0 < a.vocab; at0 += kSampleThreads * 8u) {
        const uint32_t at = at0 + tid * 8u;
        uint32_t here = 0;
        if (at < a.vocab) {
            sample_load(x, at, a.vocab, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) here |= sample_rank(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu) == rank ? 1u << e : 0u;
        }
        const uint32_t n = (uint32_t)__builtin_popcount(here), upto = wave_upto(n, lane);
        if (lane == 63u) words[wave] = upto;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (uint32_t i = 0; i < kSampleWaves; ++i) {
            before += i < wave ? words[i] : 0u;
            all += words[i];
        }
        before += upto - n;
        if (left >= before && left < before + n) {
            for (uint32_t i = left - before; i; --i) here &= here - 1u;
            a.tokens[row] = at + (uint32_t)__builtin_ctz(here);
        }
        if (left < all) break;
        left -= all;
        __syncthreads();
    }
    if (tid == 0 && a.logprobs) {
        const double v = r.infinite ? 0.0 : sample_value(rank) - r.top;
        a.logprobs[row] = (float)(v - log((double)sums[2] / r.unit));
    }
}

namespace {
constexpr uint32_t kSampleMostVocab = 1u << 24;
}

fk_status sample_workspace_bytes(uint32_t rows, uint32_t vocab, size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "sample workspace: null pointer");
    if (rows == 0 || vocab == 0) return set_error(FK_ERR_INVALID, "sample workspace: empty shape");
    if (vocab > kSampleMostVocab || rows > 65535) return set_error(FK_ERR_UNSUPPORTED, "sample workspace: up to 65535 rows of up to 2^24 logits");
    *bytes = 16;
    return FK_OK;
}

fk_status plan_sample(const uint16_t* logits, size_t row_stride, uint32_t rows, uint32_t vocab, const float* temperature, const uint32_t* top_k,
                      const float* top_p, const float* min_p, const float* u, uint32_t* tokens, float* logprobs, void* workspace, size_t workspace_bytes,
                      Launch* l) {
    if (!logits || !u || !tokens || !workspace) return set_error(FK_ERR_INVALID, "sample: null pointer");
    size_t need = 0;
    FK_TRY(sample_workspace_bytes(rows, vocab, &need));
    if (row_stride < vocab) return set_error(FK_ERR_INVALID, "sample: row stride shorter than the row");
    if (row_stride > SIZE_MAX / 2 / rows) return set_error(FK_ERR_UNSUPPORTED, "sample: row stride too large");
    if ((uintptr_t)logits & 1u) return set_error(FK_ERR_INVALID, "sample: logits must be 2-byte aligned");
    if (((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)u | (uintptr_t)tokens | (uintptr_t)logprobs) & 3u)
        return set_error(FK_ERR_INVALID, "sample: the rows' arrays must be 4-byte aligned");
    const uintptr_t one = 4 * (uintptr_t)rows;
    const struct { const void* at; uintptr_t bytes; } in[] = {{logits, 2 * ((rows - 1) * (uintptr_t)row_stride + vocab)}, {temperature, one}, {top_k, one}, {top_p, one},
                                                               {min_p, one}, {u, one}, {workspace, need}};
    auto meets = [](const void* a, uintptr_t an, const void* b, uintptr_t bn) { return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an; };
    for (const auto& i : in)
        if (meets(tokens, one, i.at, i.bytes) || meets(logprobs, one, i.at, i.bytes)) return set_error(FK_ERR_INVALID, "sample: an output overlaps an input or the workspace");
    if (meets(tokens, one, logprobs, one)) return set_error(FK_ERR_INVALID, "sample: tokens overlap logprobs");
    if ((uintptr_t)workspace & 15u) return set_error(FK_ERR_INVALID, "sample: workspace must be 16-byte aligned");
    if (workspace_bytes < need) return set_error(FK_ERR_INVALID, "sample: workspace too small");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    SampleArgs a{logits, row_stride, temperature, top_k, top_p, min_p, u, tokens, logprobs, vocab, 0};
    a.shift = 62;   // (a whole row of the largest weight stays below 2^63)
    while ((1ull << (62 - a.shift)) < vocab) --a.shift;
    l->func = reinterpret_cast<const void*>(&sample_kernel);
    l->grid = dim3(rows, 1, 1);
    l->block = dim3(kSampleThreads, 1, 1);
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
