// Tokens drawn from rows of logits, each row with a temperature, top-k, top-p and min-p of its own, from given random numbers.
//
//     w_i = exp((x_i - max x) / T);   the tokens in the order of their logits, the largest first, ties to the lower token
//     of these the first top_k;   of what they weigh, W_k, the shortest run from the first on that weighs top_p W_k;   of that, those with w_i >= min_p
//     token: the first whose running sum is above u W, W the sum of what is left
//
// A bf16 row holds few distinct logits: its tokens are counted by logit, in LDS, and each weight is formed once, in 64 bits.  Counts are whole numbers, so that
// everything behind them is the same whatever the order and the cut of the row.
#include <math.h>

#include <algorithm>

#include "fk_device.hpp"
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
    uint32_t* shared;  // [rows][kSampleShared], for rows of several pieces; zero before the first launch, left zero
    uint32_t vocab, pieces, piece;   // a piece: whole groups
    uint32_t group_shift;            // a group: 512 AHEAD << group_shift tokens
};

constexpr uint32_t kSampleGroups = 512;   // of a row, at most
constexpr uint32_t kSampleRanks = 2 * 0x7f80;

// A logit's place among all that bf16 has, the largest first: 0 is infinity, both zeros are one, kSampleRanks and more are not counted (-inf, NaN).
__device__ __forceinline__ uint32_t sample_rank(uint32_t bits) {
    const uint32_t m = bits & 0x7fffu;
    if (m > 0x7f80u) return kSampleRanks;
    return bits & 0x8000u ? 0x7f80u + m : 0x7f80u - m;
}
__device__ __forceinline__ uint32_t sample_bits(uint32_t rank) { return rank <= 0x7f80u ? 0x7f80u - rank : 0x8000u | (rank - 0x7f80u); }
__device__ __forceinline__ double sample_value(uint32_t rank) { return (double)__uint_as_float(sample_bits(rank) << 16); }

// Logits of a magnitude from 2^-32 up to 512, and zeros, have a bin each, in their order: the positive ones, zero, the negative ones.  Bins are dealt to the
// threads of a block in runs; zero and the negative ones start a run.
constexpr uint32_t kSampleLow = (127 - 32) * 128, kSampleSpan = 41 * 128, kSampleSizes = kSampleSpan / 128;
template <uint32_t THREADS>
struct SampleBins {
    static constexpr uint32_t run = (2 * kSampleSpan + 3 * THREADS / 64) / THREADS | 1u;   // an odd number: the lanes of a wave are in banks of their own
    static constexpr uint32_t zero = (kSampleSpan + run - 1) / run * run, negative = zero + run, all = THREADS * run;
    static_assert(negative + kSampleSpan <= all && run <= 32);
    // In LDS both signs lie by their magnitude, so that a place follows from a logit's bits in few instructions: zero, words that stay empty, the positive ones,
    // the negative ones, words that stay empty.
    static constexpr uint32_t positive_at = run, negative_at = run + kSampleSpan;
    __device__ static __forceinline__ uint32_t place(uint32_t bin) {
        return bin < zero ? positive_at + kSampleSpan - 1u - bin : bin < negative ? bin - zero : bin - negative + negative_at;
    }
    static_assert(positive_at + kSampleSpan - 1u >= zero - 1u && all - negative + negative_at <= all && 4 * all < 65536);
};
// What the blocks of one row share: counts, the groups' largest logits, then these words.
constexpr uint32_t kSampleMost = SampleBins<1024>::all, kSampleWords = kSampleMost + kSampleGroups, kSampleShared = kSampleWords + 32;
constexpr int kSampleNone = -0x10000;   // a group without a logit that has a bin
enum { kSampleArrived = 0, kSampleOdd = 1, kSampleLower = 2 };

// The sum of this lane's value and those before it: inside rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sample_moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double sample_moved(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)sample_moved<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | sample_moved<CTRL, ROWS>((uint32_t)b)));
}
template <uint32_t LANES = 64, typename T>   // (of the first LANES)
__device__ __forceinline__ T wave_upto(T v) {
    v += sample_moved<0x111, 0xF>(v);
    v += sample_moved<0x112, 0xF>(v);
    v += sample_moved<0x114, 0xF>(v);
    v += sample_moved<0x118, 0xF>(v);
    if constexpr (LANES > 16) v += sample_moved<0x142, 0xA>(v);
    if constexpr (LANES > 32) v += sample_moved<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }
__device__ __forceinline__ double of_lane(double v, uint32_t lane) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)of_lane((uint32_t)(b >> 32), lane) << 32 | of_lane((uint32_t)b, lane)));
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return of_lane(v, 63u); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sample_lesser(uint32_t v) { return min(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ int sample_greater(int v) { return max(v, __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xF, false)); }
__device__ __forceinline__ int wave_most(int v) {
    v = sample_greater<0x111, 0xF>(v);
    v = sample_greater<0x112, 0xF>(v);
    v = sample_greater<0x114, 0xF>(v);
    v = sample_greater<0x118, 0xF>(v);
    v = sample_greater<0x142, 0xA>(v);
    v = sample_greater<0x143, 0xC>(v);
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    v = sample_lesser<0x111, 0xF>(v);
    v = sample_lesser<0x112, 0xF>(v);
    v = sample_lesser<0x114, 0xF>(v);
    v = sample_lesser<0x118, 0xF>(v);
    v = sample_lesser<0x142, 0xA>(v);
    v = sample_lesser<0x143, 0xC>(v);
    return last_lane(v);
}

// 2^y for y up to 0; 2^f, |f| <= 1/2, by its series to the 11th power, off by 6e-15.
__device__ __forceinline__ double sample_exp2(double y) {
    const double n = rint(y), f = y - n, f2 = f * f, f4 = f2 * f2;
    const double a = fma(6.9314718055994531e-01, f, 1.0), b = fma(5.5504108664821580e-02, f, 2.4022650695910072e-01);   // ln(2)^k / k!
    const double c = fma(1.3333558146428443e-03, f, 9.6181291076284772e-03), d = fma(1.5252733804059841e-05, f, 1.5403530393381609e-04);
    const double e = fma(1.0178086009239701e-07, f, 1.3215486790144309e-06), g = fma(4.4455382718708116e-10, f, 7.0549116208011233e-09);
    return ldexp(fma(fma(fma(g, f2, e), f4, fma(d, f2, c)), f4, fma(b, f2, a)), (int)n);
}
constexpr double kSampleLog2E = 1.44269504088896340736;
// A row's weights, 2^((x - top) by).  (An infinity's difference from itself is none; beside one everything else weighs nothing.)
struct SampleRow {
    double top, by, least;   // the largest logit, log2 e / T, the smallest logit that min_p leaves
    __device__ __forceinline__ double weight_by(double value, double b) const { return sample_exp2(value == top ? 0.0 : fmax((value - top) * b, -2000.0)); }
    __device__ __forceinline__ double weight(double value) const { return weight_by(value, by); }
    __device__ __forceinline__ double plain(double value) const { return weight_by(value, kSampleLog2E); }   // at T = 1
};
constexpr double kSampleNothing = 0x1p-90;   // a weight below it is none: 2^24 of them are no part of a sum that starts with 1

// Eight logits of a row from `at` on, a multiple of 8 below vocab; -inf behind its end (not counted).
__device__ __forceinline__ void sample_load(const uint16_t* x, uint32_t at, uint32_t vocab, uint32_t (&w)[4]) {
    typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));   // (rows of an odd length start anywhere)
    if (__builtin_expect(at + 8u <= vocab, 1)) {
        const loose v = *reinterpret_cast<const loose*>(x + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = at + 2u * e < vocab ? x[at + 2u * e] : 0xff80u, hi = at + 2u * e + 1u < vocab ? x[at + 2u * e + 1u] : 0xff80u;
            w[e] = lo | hi << 16;
        }
    }
}

// One launch, a block for each piece of a row.  The piece's logits are counted in LDS; the blocks of a row add what they counted into its shared bins, and the
// last of them, or the only one, forms what each thread's run of bins holds and weighs, the sums up to each run, and from these, in up to three walks of one
// wave, the token's logit and its place among those that are equal to it; a last look at the groups of the row that hold one as large finds it.  A row that
// holds other logits (beyond 512, below 2^-32) is counted anew by that block in windows of as many ranks as there are bins, from the largest logit on.  (Logits
// of -512 and below that weigh nothing, as masks of the type's lowest value do, are no such others.)
// Many rows are bound by a CU's units, none of which works all the time: for a row of 152 000 tokens that spread as logits do its LDS takes 8 us (8 cycles a
// wave's atomic, two thirds of them bank conflicts), its vector instructions 10 and its share of the memory 15; 2000 rows 175 us (607 MB, 3.5 TB/s), 22 us a row
// on its CU.  Between 257 and 512 rows some CUs have two rows and others one: 389 rows 43 us from the last-level cache, 50 from memory (118 MB, 2.4 TB/s).  A
// single row is bound by steps that wait for each other: of 15 us for 151851 tokens the launch and the first bytes 3, the count 2.7, the pieces' meeting 2.5,
// the largest logit 0.6, the weights 2.5, three walks 3.2, the token 1.4.  Sums of fixed-point weights (5.3 for the weights' 2.5), sums by
// reductions over chunks of bins (5.3) and bins that are not empty dealt to lanes (5.4) were slower.
template <uint32_t THREADS, uint32_t AHEAD>   // requests of 16 bytes that a lane has in flight
__global__ __launch_bounds__(THREADS, 4) void sample_kernel(const SampleArgs a) {
    constexpr uint32_t WAVES = THREADS / 64, UNIT = 512 * AHEAD;   // tokens that a wave takes at a time
    constexpr uint32_t RUN = SampleBins<THREADS>::run, ZERO = SampleBins<THREADS>::zero, NEGATIVE = SampleBins<THREADS>::negative, BINS = SampleBins<THREADS>::all;
    static_assert(kSampleGroups <= THREADS && BINS <= kSampleMost);
    __shared__ uint32_t hist[BINS];
    __shared__ int most_of[kSampleGroups];          // of a group, its largest logit: its offset, for a negative one all bits inverted; zero as 0
    __shared__ uint32_t count_upto[THREADS];        // the tokens, and the weight, in a thread's bins and those before them in its wave
    __shared__ double mass_upto[THREADS];
    __shared__ uint32_t wave_n[WAVES];              // of a wave's bins
    __shared__ double wave_m[WAVES], wave_plain[WAVES], log_plain, reach;   // reach: how far below the largest min_p's border is
    __shared__ double ratio[2][kSampleSizes];       // of two weights, at T and at 1, whose logits of a size are next to each other
    __shared__ uint16_t list[kSampleGroups];
    __shared__ uint32_t words[WAVES], odd, lower, flag, next, best_word, found_rank, found_bin, found_place, found_held, of_wave[2][WAVES], over;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.y;
    const uint16_t* const x = a.logits + (size_t)row * a.row_stride;
    const uint32_t from = blockIdx.x * a.piece, left = a.vocab - from, to = from + (left < a.piece ? left : a.piece);

    // (asked for here, looked at behind the count)
    const float t_asked = a.temperature ? a.temperature[row] : 1.0f, p_asked = a.top_p ? a.top_p[row] : 1.0f, m_asked = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
    const uint32_t k_asked = a.top_k ? a.top_k[row] : 0u;

    // ---- the piece's logits, counted ----
    auto count_all = [&](uint32_t begin, uint32_t end, auto&& ready, auto&& each) __attribute__((always_inline)) {   // ready(): behind the first requests
        auto request = [&](uint32_t unit, uint32_t (&w)[AHEAD][4]) __attribute__((always_inline)) {   // (-inf behind the row)
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i) sample_load(x, unit + i * 512u + lane * 8u, a.vocab, w[i]);
        };
        // (a request of 16 bytes a lane is followed by the next before it is counted: 200 rows from memory 37 us without, 33 with; of four there are enough)
        constexpr bool TWO = AHEAD == 1;
        uint32_t w[AHEAD][4], behind[AHEAD][4];
        uint32_t unit = begin + wave * UNIT;   // (all of a wave's lanes)
        if (unit < end) request(unit, w);
        ready();
        while (unit < end) {
            const uint32_t next = unit + WAVES * UNIT;
            if (TWO && next < end) request(next, behind);
            each(unit, w);
            if (TWO)
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[i][e] = behind[i][e];
            else if (next < end) request(next, w);
            unit = next;
        }
    };
    double by = 0.0;
    uint32_t zeros = 0, others = 0, below = 0;   // this thread's zeros; whether it met another logit; of those of -512 and below how far the highest is above -inf (1: the type's lowest)
    auto ready = [&] {
        for (uint32_t i = tid * 4u; i < BINS; i += THREADS * 4u) *reinterpret_cast<uint4*>(&hist[i]) = make_uint4(0, 0, 0, 0);
        if (tid < kSampleGroups) most_of[tid] = kSampleNone;
        if (tid == 0) odd = lower = 0;
        by = kSampleLog2E / (t_asked > 0.f ? (double)t_asked : 1.0);
        if (tid < 2u * kSampleSizes) {
            const uint32_t size = tid < kSampleSizes ? tid : tid - kSampleSizes;
            const double apart = -(double)__uint_as_float((size + (kSampleLow >> 7) - 7u) << 23);
            ratio[tid < kSampleSizes ? 0 : 1][size] = sample_exp2(fmax(apart * (tid < kSampleSizes ? by : kSampleLog2E), -2000.0));
        }
        __syncthreads();
    };
    count_all(from, to, ready, [&](uint32_t unit, const uint32_t (&w)[AHEAD][4]) __attribute__((always_inline)) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        typedef short i16x2 __attribute__((ext_vector_type(2)));
        constexpr unsigned short TO_NEGATIVE = SampleBins<THREADS>::negative_at - SampleBins<THREADS>::positive_at;
        auto off_of = [](uint32_t pair) { return __builtin_bit_cast(u16x2, pair & 0x7fff7fffu) - (unsigned short)kSampleLow; };
        auto sign_of = [](uint32_t pair) { return __builtin_bit_cast(u16x2, __builtin_bit_cast(i16x2, pair) >> 15); };
        u16x2 furthest = {0, 0};
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) furthest = __builtin_elementwise_max(furthest, off_of(w[i][e]));
        unsigned char* const bytes = reinterpret_cast<unsigned char*>(&hist[SampleBins<THREADS>::positive_at]);
        auto places_of = [&](u16x2 off, u16x2 sign) { return __builtin_bit_cast(uint32_t, (off - sign * TO_NEGATIVE) << (unsigned short)2); };   // in bytes from there
        auto counted = [&](uint32_t place) { atomicAdd(reinterpret_cast<uint32_t*>(bytes + place), 1u); };
        i16x2 largest = {-0x8000, -0x8000};
        int most = kSampleNone;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(furthest[0] >= kSampleSpan || furthest[1] >= kSampleSpan) == 0, 1)) {
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u16x2 off = off_of(w[i][e]), sign = sign_of(w[i][e]);
                    largest = __builtin_elementwise_max(largest, __builtin_bit_cast(i16x2, off ^ sign));
                    const uint32_t places = places_of(off, sign);
                    counted(places & 0xffffu);
                    counted(places >> 16);
                }
        } else {   // some without a bin: masked ones, -inf or the type's lowest, most likely
            bool other = false, lowest = false;
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u16x2 off = off_of(w[i][e]), sign = sign_of(w[i][e]), masked = __builtin_bit_cast(u16x2, w[i][e]) + (unsigned short)0x81;   // 0xff7f, 0xff80: 0, 1
                    const i16x2 order = __builtin_bit_cast(i16x2, off ^ sign);
                    const uint32_t places = places_of(off, sign);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool in = off[h] < kSampleSpan;
                        if (in) counted(h ? places >> 16 : places & 0xffffu);
                        largest[h] = in && order[h] > largest[h] ? order[h] : largest[h];
                        other |= !in && masked[h] > 1;
                        lowest |= !in && masked[h] == 0;
                    }
                }
            below = lowest ? max(below, 1u) : below;
            if (__builtin_amdgcn_ballot_w64(other)) {
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t bits = e & 1 ? w[i][e / 2] >> 16 : w[i][e / 2] & 0xffffu, m = bits & 0x7fffu;
                        if (m - kSampleLow < kSampleSpan) continue;
                        if (m == 0) {
                            ++zeros;
                            most = max(most, 0);
                        } else if (m < 0x7f80u && bits >= 0x8000u && m >= kSampleLow) {
                            below = max(below, 0x7f80u - m);
                        } else if (m < 0x7f80u || bits == 0x7f80u) {
                            others = 1;
                        }
                    }
            }
        }
        const int order = largest[0] > largest[1] ? largest[0] : largest[1];
        most = order > -0x8000 ? max(most, order) : most;
        most = wave_most(most);
        if (lane == 0) atomicMax(&most_of[unit / UNIT >> a.group_shift], most);
    });
    if (zeros) atomicAdd(&hist[SampleBins<THREADS>::place(ZERO)], zeros);
    if (others) odd = 1;
    if (below) atomicMax(&lower, below);
    __syncthreads();

    auto borders = [&] {   // (while requests are on their way)
        if (tid == 128u) reach = (double)t_asked * log((double)fminf(m_asked, 1.0f));
    };
    // ---- the row's pieces meet ----
    uint32_t* const shared = a.shared + (size_t)row * kSampleShared;
    if (a.pieces > 1u) {
        uint32_t n[RUN];
#pragma unroll
        for (uint32_t i = 0; i < RUN; ++i) n[i] = hist[i * THREADS + tid];
#pragma unroll
        for (uint32_t i = 0; i < RUN; ++i)
            if (n[i]) __hip_atomic_fetch_add(&shared[i * THREADS + tid], n[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint32_t per_group = UNIT << a.group_shift;   // (a piece holds whole groups)
        if (tid >= from / per_group && tid < (to + per_group - 1u) / per_group)
            __hip_atomic_store(&shared[kSampleMost + tid], (uint32_t)most_of[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0 && odd) __hip_atomic_store(&shared[kSampleWords + kSampleOdd], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0 && lower) __hip_atomic_fetch_max(&shared[kSampleWords + kSampleLower], lower, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        borders();
        wait_memory_ops_done();
        __syncthreads();
        if (tid == 0) flag = atomicAdd(&shared[kSampleWords + kSampleArrived], 1u) == a.pieces - 1u ? 1u : 0u;
        __syncthreads();
        if (!flag) return;
        auto at_word = [&](uint32_t i) { return __hip_atomic_load(&shared[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
#pragma unroll
        for (uint32_t i = 0; i < RUN; ++i) n[i] = at_word(i * THREADS + tid);
        const uint32_t f = tid < kSampleGroups ? at_word(kSampleMost + tid) : 0u, o = at_word(kSampleWords + kSampleOdd), b = at_word(kSampleWords + kSampleLower);
        auto clear = [&](uint32_t i) { __hip_atomic_store(&shared[i], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
#pragma unroll
        for (uint32_t i = 0; i < RUN; ++i) {
            hist[i * THREADS + tid] = n[i];
            if (n[i]) clear(i * THREADS + tid);
        }
        if (tid < kSampleGroups) most_of[tid] = (int)f;   // (of groups behind the row: nothing that is looked at)
        if (tid == 0) {
            odd = o;
            lower = b;
        }
        __syncthreads();
        if (tid < 3) clear(kSampleWords + tid);
    } else {
        borders();
    }

    // ---- the largest logit ----
    const float t = t_asked, top_p = p_asked, min_p = m_asked > 0.f ? fminf(m_asked, 1.0f) : 0.f;
    const bool greedy = !(t > 0.f), whole_p = !(top_p < 1.0f);
    const uint32_t k = greedy ? 1u : k_asked ? k_asked : ~0u;
    auto rank_of = [&](uint32_t bin, uint32_t base) -> uint32_t {   // base: of a window; ~0: the bins by magnitude
        if (base != ~0u) return min(base + bin, kSampleRanks - 1u);
        return bin < ZERO ? bin + (0x7f80u + 1u - kSampleLow - kSampleSpan) : bin < NEGATIVE ? 0x7f80u : min(bin + (0x7f80u + kSampleLow - NEGATIVE), kSampleRanks - 1u);
    };
    const uint32_t per_group = UNIT << a.group_shift, groups = (a.vocab + per_group - 1u) / per_group;
    uint32_t best = kSampleRanks, top_bin;
    {
        int m = wave_most(tid < groups ? most_of[tid] : kSampleNone);
        if (lane == 0) words[wave] = (uint32_t)m;
        __syncthreads();
        m = (int)words[0];
#pragma unroll
        for (uint32_t i = 1; i < WAVES; ++i) m = max(m, (int)words[i]);
        // (0: zero, or 2^-32)
        top_bin = m == 0 && hist[SampleBins<THREADS>::positive_at] == 0 ? ZERO : m >= 0 ? kSampleSpan - 1u - (uint32_t)m : NEGATIVE + (uint32_t)~m;
        if (m != kSampleNone) best = rank_of(top_bin, ~0u);
    }
    SampleRow r;
    r.by = by;
    auto from_best = [&] {
        r.top = sample_value(best);
        r.least = min_p > 0.f && !greedy ? r.top + reach : -INFINITY;
    };
    from_best();
    bool windows = odd != 0;
    if (lower && !windows) {   // do any of -512 and below weigh something?
        const uint32_t rank = kSampleRanks - lower;
        windows = best >= kSampleRanks || r.weight(sample_value(rank)) > kSampleNothing || (a.logprobs && r.plain(sample_value(rank)) > kSampleNothing);
    }
    if (windows) {
        if (tid == 0) best_word = kSampleRanks;
        __syncthreads();
        uint32_t b = kSampleRanks;
        count_all(0, a.vocab, [] {}, [&](uint32_t, const uint32_t (&w)[AHEAD][4]) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) b = min(b, min(sample_rank(w[i][e] & 0xffffu), sample_rank(w[i][e] >> 16)));
        });
        b = wave_least(b);
        if (lane == 0) atomicMin(&best_word, b);
        __syncthreads();
        best = best_word;
        from_best();
    }
    if (best >= kSampleRanks) {   // nothing above -inf
        if (tid == 0) {
            a.tokens[row] = 0;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        return;
    }

    // ---- a window's sums: the tokens and the weight up to each thread's bins ----
    uint32_t total_n = 0, n_waves = 0;          // (wave 0's) of a window; a lane's: up to the end of that wave's bins
    double total_m = 0.0, m_waves = 0.0;
    auto weigh = [&](uint32_t base) {
        const uint32_t bin0 = tid * RUN;
        uint32_t all = 0;
        double m = 0.0, p = 0.0;
        if (base == ~0u) {
            // Logits of one size (a power of two) are 2^-7 of it apart: the weights of a run are that of its first one times powers of one ratio, beyond a border
            // of two sizes of another.  (Bins above the largest logit, and those that stand for none, are empty.)
            const bool positive = bin0 < ZERO;
            const uint32_t low0 = positive ? kSampleSpan - 2u - bin0 : bin0 - NEGATIVE;   // of the first two magnitudes, as offsets, the lower
            const uint32_t size0 = min(low0 >> 7, kSampleSizes - 1u), size1 = min((positive ? low0 - (RUN - 2u) : low0 + (RUN - 2u)) >> 7, kSampleSizes - 1u);
            const uint32_t border = positive ? (low0 & 127u) + 1u : 128u - (low0 & 127u);   // the steps of the first size
            const uint32_t above = top_bin > bin0 ? top_bin - bin0 : 0u;                    // the steps above the largest logit
            const double w0 = ratio[0][size0], w1 = ratio[0][size1], one0 = ratio[1][size0], one1 = ratio[1][size1];
            const double first = above ? r.top : sample_value(rank_of(bin0, base));
            const int at = (int)SampleBins<THREADS>::place(bin0), step = positive ? -1 : 1;
            uint32_t n[RUN];
#pragma unroll
            for (uint32_t i = 0; i < RUN; ++i) all += n[i] = hist[at + step * (int)i];
            if (__builtin_amdgcn_ballot_w64(all != 0)) {   // (of 82 sizes of both signs a row fills some 25)
                // (from the last one on: each sum times the ratio, and the next count)
                m = p = (double)n[RUN - 1u];
#pragma unroll
                for (int i = (int)RUN - 2; i >= 0; --i) {
                    const bool near = (uint32_t)i < border, over = (uint32_t)i < above;
                    m = fma(m, over ? 1.0 : near ? w0 : w1, (double)n[i]);
                    p = fma(p, over ? 1.0 : near ? one0 : one1, (double)n[i]);
                }
                m *= sample_exp2(fmax((first - r.top) * r.by, -2000.0));
                p *= sample_exp2(fmax((first - r.top) * kSampleLog2E, -2000.0));
            }
        } else {
#pragma unroll 1
            for (uint32_t i = 0; i < RUN; ++i) {
                const uint32_t n = hist[bin0 + i];
                if (!n) continue;
                const double v = sample_value(rank_of(bin0 + i, base));
                all += n;
                m = fma((double)n, r.weight(v), m);
                p = fma((double)n, r.plain(v), p);
            }
        }
        uint32_t n_upto = 0;
        double m_upto = 0.0, p_upto = 0.0;
        if (__builtin_amdgcn_ballot_w64(all != 0)) {
            n_upto = wave_upto(all);
            m_upto = wave_upto(m);
            p_upto = wave_upto(p);
        }
        count_upto[tid] = n_upto;
        mass_upto[tid] = m_upto;
        if (lane == 63u) {
            wave_n[wave] = n_upto;
            wave_m[wave] = m_upto;
            wave_plain[wave] = p_upto;
        }
        __syncthreads();
        if (wave == 0) {
            n_waves = wave_upto<WAVES>(lane < WAVES ? wave_n[lane] : 0u);
            m_waves = wave_upto<WAVES>(lane < WAVES ? wave_m[lane] : 0.0);
            total_n = of_lane(n_waves, WAVES - 1u);
            total_m = of_lane(m_waves, WAVES - 1u);
        }
    };
    // Wave 0 looks for the end of a run of tokens from the first on: at `most` tokens, where it weighs `goal`, or before a logit below `least`; the thread whose bins it
    // ends in is found in two steps.  True where it ends in this window; then `taken` is what it weighs and found_* the bin and how many of the bin it
    // takes.  `before`: it ends before the token that goes past the goal.
    uint32_t walked_n = 0;   // the windows before
    double walked_m = 0.0, taken = 0.0;
    auto walk = [&](uint32_t base, uint32_t most, double goal, double least, bool before) -> bool {
        auto ends = [&](uint32_t n, double m, uint32_t run) {   // what lies up to its end
            return n > most || m >= goal || (least > -INFINITY && sample_value(rank_of(run * RUN + RUN - 1u, base)) < least);
        };
        uint32_t from_run = 0;
#pragma unroll 1
        for (;;) {
            const unsigned long long waves = __builtin_amdgcn_ballot_w64(lane < WAVES && lane * 64u + 63u >= from_run && ends(walked_n + n_waves, walked_m + m_waves, lane * 64u + 63u));
            if (!waves) break;
            const uint32_t in_wave = (uint32_t)__builtin_ctzll(waves), at = in_wave * 64u + lane;
            const uint32_t n_at = walked_n + (in_wave ? of_lane(n_waves, in_wave - 1u) : 0u) + count_upto[at];
            const double m_at = walked_m + ((in_wave ? of_lane(m_waves, in_wave - 1u) : 0.0) + mass_upto[at]);
            // (rounded another way, the wave's end may be found short of the goal: its last run then)
            const unsigned long long runs = __builtin_amdgcn_ballot_w64(at >= from_run && (lane == 63u || ends(n_at, m_at, at)));
            const uint32_t in = (uint32_t)__builtin_ctzll(runs), run = in_wave * 64u + in;
            const uint32_t bin = run * RUN + lane, rank = rank_of(bin, base), held = lane < RUN ? hist[base == ~0u ? SampleBins<THREADS>::place(bin) : bin] : 0u;
            const double v = sample_value(rank), each = r.weight(v), all = held ? (double)held * each : 0.0;
            const uint32_t n = of_lane(n_at - count_upto[at], 0) + (in ? count_upto[run - 1u] : 0u) + wave_upto<RUN>(held) - held;
            const double m = of_lane(m_at - mass_upto[at], 0) + (in ? mass_upto[run - 1u] : 0.0) + (wave_upto<RUN>(all) - all);
            uint32_t take = n >= most ? 0u : min(held, most - n);
            if (m >= goal || v < least) {
                take = 0;
            } else if (m + take * each >= goal) {
                const double q = fmin((goal - m) / each, 16777216.0);
                take = min(take, (uint32_t)(before ? floor(q) : ceil(q)));
                if (before && take == held) take = held - 1u;   // (its last token is the one that goes past it)
            }
            if (n == 0 && take == 0 && !before) take = min(held, 1u);   // the largest stays
            const unsigned long long less = __builtin_amdgcn_ballot_w64(take < held);
            if (less) {
                const uint32_t who = (uint32_t)__builtin_ctzll(less);
                taken = of_lane(m + take * each, who);
                if (lane == who) {
                    found_rank = rank;
                    found_bin = bin;
                    found_place = take;
                    found_held = held;
                }
                wave_lds_order();
                return true;
            }
            // all of it is taken after all: the end is before the next token, wherever that is
            from_run = run + 1u;
            most = min(most, of_lane(n_at, in));
            goal = INFINITY;
            least = -INFINITY;
        }
        walked_n += total_n;
        walked_m += total_m;
        return false;
    };
    uint32_t built = kSampleRanks;
    auto build = [&](uint32_t base) {   // a window's bins, and in `next` the first rank behind it that the row holds
        if (built == base) return;
        built = base;
        for (uint32_t i = tid; i < BINS; i += THREADS) hist[i] = 0;
        if (tid == 0) next = kSampleRanks;
        __syncthreads();
        uint32_t behind = kSampleRanks;
        count_all(0, a.vocab, [] {}, [&](uint32_t, const uint32_t (&w)[AHEAD][4]) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t rank = sample_rank(e & 1 ? w[i][e / 2] >> 16 : w[i][e / 2] & 0xffffu), bin = rank - base;
                    if (bin < BINS && rank < kSampleRanks) atomicAdd(&hist[bin], 1u);
                    else if (rank > base) behind = min(behind, rank);
                }
        });
        behind = wave_least(behind);
        if (lane == 0) atomicMin(&next, behind);
        __syncthreads();
        weigh(base);
    };

    // ---- pass 0: W_k, and what the row weighs at T = 1; pass 1: W; pass 2: the token's logit, and its place among equal ones ----
    double w_k = 0.0, limit = 0.0, all_plain = 0.0;
    if (!windows) {
        weigh(~0u);
        if (wave == 1u && a.logprobs) {   // (while wave 0 goes on)
            const double all = of_lane(wave_upto<WAVES>(lane < WAVES ? wave_plain[lane] : 0.0), WAVES - 1u);
            if (lane == 0) log_plain = log(all);
        }
    }
#pragma unroll 1
    for (int pass = windows || wave == 0 ? 0 : 3; pass < 3; ++pass) {
        // the run that is looked for ends at `most` tokens, at a weight of `goal`, and at logits below `least`: taken up to (passes 0 and 1: the goal is
        // reached), or short of it (pass 2: the goal is passed)
        const uint32_t most = pass < 2 ? k : ~0u;
        const double least = pass == 1 ? r.least : -INFINITY;
        double goal = INFINITY;
        if (pass == 1 && !whole_p) goal = top_p > 0.f ? (double)top_p * w_k : 0.0;
        if (pass == 2)   // (above it: from the next number on)
            goal = __longlong_as_double(__double_as_longlong(u > 0.f ? (double)fminf(u, 0x1.fffffep-1f) * limit : 0.0) + 1);
        if (!windows && pass < 2 && ((pass == 0 && whole_p) || (k >= total_n && goal == INFINITY && least == -INFINITY))) {   // nothing is cut, or W_k not asked for
            (pass == 0 ? w_k : limit) = total_m;
            continue;
        }
        walked_n = 0;
        walked_m = 0.0;
        bool done = false;
        uint32_t base = windows ? best : ~0u;
#pragma unroll 1
        for (;;) {
            if (windows) build(base);
            if (windows && pass == 0) all_plain += of_lane(wave_upto<WAVES>(lane < WAVES ? wave_plain[lane] : 0.0), WAVES - 1u);
            if (!done && wave == 0) done = walk(base, most, goal, least, pass == 2);
            if (!windows) break;
            if (tid == 0) over = done ? 1u : 0u;
            __syncthreads();
            base = next;
            done = over != 0;
            __syncthreads();
            if (base >= kSampleRanks || (done && !(pass == 0 && a.logprobs))) break;
            // (what weighs nothing from here on ends no sum)
            if (pass < 2 && r.weight(sample_value(base)) <= kSampleNothing && (pass != 0 || !a.logprobs || r.plain(sample_value(base)) <= kSampleNothing)) break;
        }
        (pass == 0 ? w_k : limit) = done ? taken : walked_m;   // (wave 0's)
    }
    if (windows && tid == 0 && a.logprobs) log_plain = log(all_plain);
    __syncthreads();
    if (tid == 0 && a.logprobs) a.logprobs[row] = (float)((best == 0 ? 0.0 : sample_value(found_rank) - r.top) - log_plain);

    // ---- the token: of those that hold the logit, in their order, the one at found_place; looked for in the groups that hold one as large ----
    const uint32_t bin = found_bin, zero = found_rank == 0x7f80u, want = zero ? 0u : sample_bits(found_rank) * 0x10001u, mask = zero ? 0x7fff7fffu : ~0u;   // (both halves of a word)
    const int least_most = bin < ZERO ? (int)(kSampleSpan - 1u - bin) : bin < NEGATIVE ? 0 : ~(int)(bin - NEGATIVE);
    const bool may = tid < groups && (windows || most_of[tid] >= least_most);
    const unsigned long long may_all = __builtin_amdgcn_ballot_w64(may);
    if (lane == 0) words[wave] = (uint32_t)__builtin_popcountll(may_all);
    __syncthreads();
    uint32_t listed = 0, listed_before = 0;
#pragma unroll
    for (uint32_t i = 0; i < WAVES; ++i) {
        listed_before += i < wave ? words[i] : 0u;
        listed += words[i];
    }
    if (may) list[listed_before + (uint32_t)__builtin_popcountll(may_all & ((1ull << lane) - 1ull))] = (uint16_t)tid;
    __syncthreads();
    // (from the end that is nearer, if those that hold it lie as they fall: a logit that a whole row of 151851 holds took 17 us of the 55 of 389 rows from the
    // first one on; a round's requests ahead of the one that is counted do not fit the registers)
    const bool back = found_place > (found_held - 1u) / 2u;
    uint32_t place = back ? found_held - 1u - found_place : found_place;
    const uint32_t units = (listed << a.group_shift) * AHEAD, in = AHEAD << a.group_shift;   // of 512 tokens
    constexpr uint32_t UNITS = 8;                                                            // of a wave at a time
    auto at_unit = [&](uint32_t u) {   // this lane's first token of the u-th one
        const uint32_t unit = back ? units - 1u - u : u;
        return (uint32_t)list[unit / AHEAD >> a.group_shift] * (512u * in) + (unit & (in - 1u)) * 512u + lane * 8u;
    };
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    auto differ = [&](const uint32_t (&w)[4]) __attribute__((always_inline)) {   // of this lane's eight, in two halves
        u16x2 n = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) n += __builtin_elementwise_min(__builtin_bit_cast(u16x2, (w[e] & mask) ^ want), u16x2{1, 1});
        return n;
    };
#pragma unroll 1
    for (uint32_t unit0 = 0, turn = 0; unit0 < units; unit0 += WAVES * UNITS, turn ^= 1u) {
        const uint32_t mine0 = unit0 + wave * UNITS, mine = mine0 < units ? min(units - mine0, UNITS) : 0u;   // units of this wave
        uint32_t w[UNITS][4], all = 0;
        if (mine) {
#pragma unroll
            for (uint32_t i = 0; i < UNITS; ++i) {
                if (i < mine) sample_load(x, at_unit(mine0 + i), a.vocab, w[i]);
                else w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0xff80ff80u;
            }
            u16x2 other = {0, 0};
#pragma unroll
            for (uint32_t i = 0; i < UNITS; ++i) other += differ(w[i]);
            all = last_lane(wave_upto(8u * UNITS - other[0] - other[1]));
        }
        if (lane == 0) of_wave[turn][wave] = all;
        __syncthreads();
        uint32_t before = 0, every = 0;
#pragma unroll
        for (uint32_t i = 0; i < WAVES; ++i) {
            before += i < wave ? of_wave[turn][i] : 0u;
            every += of_wave[turn][i];
        }
        if (place >= before && place < before + all) {
            uint32_t skip = place - before;
#pragma unroll
            for (uint32_t i = 0; i < UNITS; ++i) {
                const u16x2 o = differ(w[i]);
                const uint32_t n = 8u - o[0] - o[1], upto = wave_upto(n), unit_all = last_lane(upto);
                if (skip < unit_all) {
                    const uint32_t first = back ? unit_all - 1u - skip : skip;
                    if (first >= upto - n && first < upto) {
                        uint32_t bits = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t d = (w[i][e] & mask) ^ want;
                            bits |= (d & 0xffffu ? 0u : 1u) << (2 * e) | (d >> 16 ? 0u : 2u) << (2 * e);
                        }
                        for (uint32_t o1 = first - (upto - n); o1; --o1) bits &= bits - 1u;
                        a.tokens[row] = at_unit(mine0 + i) + (uint32_t)__builtin_ctz(bits);
                    }
                    break;
                }
                skip -= unit_all;
            }
        }
        if (place < every) break;
        place -= every;
    }
}

namespace {

constexpr uint32_t kSampleMostVocab = 1u << 24;

// How a launch is cut.  Up to 256 rows (a CU each): blocks of 1024 threads, whose last steps are short, and rows of more than 32768 tokens in as many pieces as give
// every CU one block, 16 at most, of 8192 tokens at least.  us of 1, 16, 64 and 96 rows of some 151900 whole, in 2, 4, 8 and 16 pieces: 23.3, 20.2, 17.7, 16.5,
// 15.6; 24.6, 21.4, 18.7, 17.9, 18.2; 28.1, 25.8, 24.4, 40.1, 64.5; 28.3, 26.4, 37.5, 52.9, 87.6; of 1 and 128 rows of 32000 whole and in 4 15.2, 15.3; 19.3, 33.9.
// More rows: blocks of 512 threads, two on a CU, one of which counts while the other is at its last steps: 389 rows of 151851 55 us (1024 threads: 66), 512 of
// 32000 23 (35).  Those whole: their bins meet in memory, 389 rows in 1 to 4 pieces 49, 63, 57 and 86 us.  (All before the token was looked for from the nearer end.)
constexpr uint32_t kSampleWide = 256, kSampleWhole = 32768, kSampleMostPieces = 16, kSampleLeastPiece = 8192;
struct SamplePlan {
    uint32_t pieces, piece, group_shift;
    bool wide;
};
SamplePlan sample_plan(uint32_t rows, uint32_t vocab) {
    SamplePlan p;
    p.wide = rows <= kSampleWide;
    const uint32_t least_group = p.wide ? 512 : 2048;
    p.group_shift = 0;
    while ((uint64_t)(least_group << p.group_shift) * kSampleGroups < vocab) ++p.group_shift;
    const uint32_t group = least_group << p.group_shift, want = vocab <= kSampleWhole ? 1 : std::max(1u, std::min(kSampleWide / rows, kSampleMostPieces));
    const uint32_t piece = std::max((vocab + want - 1) / want, kSampleLeastPiece);
    p.piece = (piece + group - 1) / group * group;
    p.pieces = (vocab + p.piece - 1) / p.piece;
    return p;
}

}  // namespace

fk_status sample_workspace_bytes(uint32_t rows, uint32_t vocab, size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "sample workspace: null pointer");
    if (rows == 0 || vocab == 0) return set_error(FK_ERR_INVALID, "sample workspace: empty shape");
    if (vocab > kSampleMostVocab || rows > 65535) return set_error(FK_ERR_UNSUPPORTED, "sample workspace: up to 65535 rows of up to 2^24 logits");
    *bytes = sample_plan(rows, vocab).pieces > 1 ? (size_t)rows * kSampleShared * 4 : 16;
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
    const SamplePlan p = sample_plan(rows, vocab);
    SampleArgs a{logits, row_stride, temperature, top_k, top_p, min_p, u, tokens, logprobs, static_cast<uint32_t*>(workspace), vocab, p.pieces, p.piece, p.group_shift};
    l->func = p.wide ? reinterpret_cast<const void*>(&sample_kernel<1024, 1>) : reinterpret_cast<const void*>(&sample_kernel<512, 4>);
    l->grid = dim3(p.pieces, rows, 1);
    l->block = dim3(p.wide ? 1024 : 512, 1, 1);
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
