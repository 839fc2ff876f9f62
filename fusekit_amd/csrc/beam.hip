// Beam search: the k best continuations of each group's beams, and state rows that follow the beams chosen.
//
//     total[b, t] = score[b] - log sum_t exp(logit[b, t] - m) + (logit[b, t] - m),   m the largest logit of row b
//
// (the differences first: logits of any size, a mask of the type's lowest value among them, lose nothing by it).
// The k best of a group in order, ties to the lower b * vocab + t.  Inside a row the order is that of the logits, so a row
// contributes only its k largest logits; rows are then compared in 64 bits.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "argmax_tail.hpp"
#include "fk_host.hpp"

namespace fk {

constexpr uint32_t kBeamMax = 64, kBeamGroups = 4096;
// A group's counter has a line of its own: atomics on one line follow one another, also on different words of it (2432 arrivals of 16 groups in
// one line: 18 us).  They lie at the same place for every shape: a workspace serves one call after another.
constexpr uint32_t kBeamCounterStep = 32;
constexpr size_t kBeamCounterBytes = (size_t)4 * kBeamCounterStep * kBeamGroups;

// One launch.  A block takes a piece of a row: it leaves the piece's largest logit, its sum of exponentials and its k largest logits in order; the
// block of a group that comes last forms the rows' sums and the k best of what all pieces left.  The pieces are cut by token, never by address: rows that
// hold the same values have the same sums wherever they lie, so that ties between beams stay ties.
//
// The k largest of a piece without sorting it: the k-th largest of the maxima of 64 (beyond k = 24: 256) parts of it is a bound that at least k
// values reach and few more; found by bisection over its 16 bits with ballots.  What reaches it is collected in LDS and ranked by counting.
// Only a piece full of ties has more than fit there: its k largest are then taken one by one (all but one token in a thousand at bf16's lowest value: 16 x 8
// rows of 151851 102 us for 21, 4 of 32000 13 for 9; masked with -inf, which is not collected, as without a mask).  Logits are compared two at a time as 16-bit
// integers: with a negative one's magnitude negated, bf16 values are in order (and -0 is 0).
//
// 16 x 8 rows of 151851 in 21 us, 1.85 TB/s.  A block waits for its piece (3 us while all ask at once), then for the bound, the list and the counter after
// one another (another 3); 2432 blocks are one round of 2048 and a fifth of a second, and the last group's merge is 5 us.  4 rows of 32000 in 9 us: 4 to
// the last arrival, 5 of merge.  Pieces of 4096, 6144, 8192, 10240, 12288 and 16384 tokens take 27, 22, 21, 22, 23 and 37 us of the former; of
// 8192 instead of 2048 10.3 us of the latter.
struct BeamArgs {
    const uint16_t* logits;
    size_t row_stride;
    const float* scores;
    const uint32_t* finished;
    uint32_t pad, beams, vocab, k, pieces;
    float* out_scores;
    uint32_t* out_beams;
    uint32_t* out_tokens;
    uint32_t* arrived;   // [groups][kBeamCounterStep], zero before the first launch, left zero
    double* sums;        // [groups * beams][pieces]
    float* tops;         // [groups * beams][pieces]
    uint32_t* best;      // [groups * beams][pieces][k]: (order of the logit << 16) | (65535 - place in the piece), 0 where there are no more
};

constexpr uint32_t kBeamList = 512, kBeamPart = kBeamList / 4;   // candidates that fit in LDS, of a wave
constexpr float kBeamLog2E = 1.44269504088896341f;
typedef short i16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ double wave_sum_wide(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Two logits as integers in their order; the float that an order stands for; the smallest order above -inf.
__device__ __forceinline__ i16x2_t beam_order(uint32_t w) {
    const i16x2_t x = __builtin_bit_cast(i16x2_t, w), s = x >> 15;
    return (x ^ (s & 0x7fff)) - s;
}
__device__ __forceinline__ float beam_value(int order) { return __uint_as_float((uint32_t)(order < 0 ? 0x8000 | -order : order) << 16); }
constexpr int kBeamLeast = -0x7f80 + 1;

// A bound that at least k of what the block's threads hold reach, the k-th largest of their `mine` or of the maxima of four of them (k up to 24), or
// 0 where fewer than k are not 0; its bits below LOW are not looked for.  `all`: LDS, 256 words.
template <int BITS, int LOW>
__device__ __forceinline__ uint32_t bound_of_best(uint32_t mine, uint32_t k, uint32_t* all) {
    const uint32_t lane = threadIdx.x & 63u;
    all[threadIdx.x] = mine;
    __syncthreads();
    uint32_t v[4], t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = all[lane + 64u * i];
    auto count = [&](uint32_t x, uint32_t at) { return (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(x >= at)); };
    if (__builtin_expect(k <= 24u, 1)) {
        const uint32_t a = v[0] > v[1] ? v[0] : v[1], b = v[2] > v[3] ? v[2] : v[3], m = a > b ? a : b;
#pragma unroll
        for (int bit = BITS - 1; bit >= LOW; --bit)
            if (count(m, t | (1u << bit)) >= k) t |= 1u << bit;
    } else {
#pragma unroll 1
        for (int bit = BITS - 1; bit >= LOW; --bit)
            if (count(v[0], t | (1u << bit)) + count(v[1], t | (1u << bit)) + count(v[2], t | (1u << bit)) + count(v[3], t | (1u << bit)) >= k) t |= 1u << bit;
    }
    return t;
}

template <int VEC>   // 16-byte loads of a thread
__global__ __launch_bounds__(256) void beam_select_kernel(const BeamArgs a) {
    constexpr uint32_t PIECE = 2048u * VEC;
    typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));   // (rows of an odd length start anywhere)
    __shared__ uint32_t all[256];
    __shared__ uint4 list4[kBeamList / 4];
    uint32_t* const list = reinterpret_cast<uint32_t*>(list4);
    __shared__ double values[kBeamList], part[4], base[kBeamMax];
    __shared__ uint64_t flats[kBeamList];
    __shared__ uint32_t counts[4], flag, ended[kBeamMax];
    __shared__ float near[kBeamMax], peak[kBeamMax];
    constexpr uint32_t AHEAD = 6;
    __shared__ uint32_t keys[AHEAD * 256u];
    __shared__ float top[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t piece = blockIdx.x, row = blockIdx.y, g = row / a.beams, k = a.k;
    const uint32_t from = piece * PIECE, left = a.vocab - from;
    const bool over = a.finished && a.finished[row];   // (the same for the block)
    if (!over) {
        const uint16_t* x = a.logits + (size_t)row * a.row_stride + from;
        uint32_t w[VEC * 4];
        if (__builtin_expect(left >= PIECE, 1)) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const loose v = *reinterpret_cast<const loose*>(x + ((uint32_t)i * 256u + tid) * 8u);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[i * 4 + e] = v[e];
            }
        } else {   // the row's last piece: -inf behind its end
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint32_t at = ((uint32_t)i * 256u + tid) * 8u;
                loose v = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
                if (at + 8u <= left) {
                    v = *reinterpret_cast<const loose*>(x + at);
                } else if (at < left) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lo = at + 2u * e < left ? x[at + 2u * e] : 0xff80u, hi = at + 2u * e + 1u < left ? x[at + 2u * e + 1u] : 0xff80u;
                        v[e] = lo | hi << 16;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) w[i * 4 + e] = v[e];
            }
        }
        int most;
        float mw;
        double sum;
#pragma unroll 1
        for (int pass = 0;; ++pass) {
            i16x2_t m2 = beam_order(w[0]);
#pragma unroll
            for (int i = 1; i < VEC * 4; ++i) m2 = __builtin_elementwise_max(m2, beam_order(w[i]));
            most = m2[0] > m2[1] ? m2[0] : m2[1];
            mw = wave_max(beam_value(most));
            // exp(x - m) as 2^((x - m) L): the difference first, which is exact or far from 0 whatever the logits' size (x L - m L leaves
            // fp32 from 2.4e38 on, and is off by 2^-24 of m L before)
            const float ref = mw == -INFINITY ? 0.f : mw;
            sum = 0.0;
#pragma unroll
            for (int i = 0; i < VEC * 2; ++i) {
                const float e0 = __builtin_amdgcn_exp2f((bf16_lo(w[2 * i]) - ref) * kBeamLog2E), e1 = __builtin_amdgcn_exp2f((bf16_hi(w[2 * i]) - ref) * kBeamLog2E);
                const float e2 = __builtin_amdgcn_exp2f((bf16_lo(w[2 * i + 1]) - ref) * kBeamLog2E), e3 = __builtin_amdgcn_exp2f((bf16_hi(w[2 * i + 1]) - ref) * kBeamLog2E);
                sum += (double)((e0 + e1) + (e2 + e3));
            }
            sum = wave_sum_wide(sum);
            if (__builtin_expect(pass != 0 || sum == sum, 1)) break;
            // a NaN among them: it counts as -inf (and an infinity's sum stays what it is)
#pragma unroll
            for (int i = 0; i < VEC * 4; ++i) {
                if ((w[i] & 0x7fffu) > 0x7f80u) w[i] = (w[i] & 0xffff0000u) | 0xff80u;
                if ((w[i] & 0x7fff0000u) > 0x7f800000u) w[i] = (w[i] & 0xffffu) | 0xff800000u;
            }
        }
        if (lane == 0) {
            top[wave] = mw;
            part[wave] = sum;
        }
        const uint32_t found = bound_of_best<16, 0>(most >= kBeamLeast ? (uint32_t)(most + 0x8000) : 0u, k, all);
        int bound = (int)found - 0x8000;
        bound = bound < kBeamLeast ? kBeamLeast : bound;
        auto entry = [&](int order, int i, int h) { return (uint32_t)(order + 0x8000) << 16 | (0xffffu - (((uint32_t)(i / 4) * 256u + tid) * 8u + (uint32_t)((i % 4) * 2 + h))); };
        auto again = [&] {   // (the orders are formed anew, not kept: two registers a word are what lets fewer blocks stand on a CU)
#pragma unroll
            for (int i = 0; i < VEC * 4; ++i) asm volatile("" : "+v"(w[i]));
        };
        again();
        // a wave's part of the list, without a counter to wait for
        uint32_t mine = 0;   // entries of this wave so far
        {
            const i16x2_t below = {(short)(bound - 1), (short)(bound - 1)};
#pragma unroll
            for (int i = 0; i < VEC * 4; ++i) {
                const i16x2_t o = beam_order(w[i]), reached = __builtin_elementwise_max(o, below);
                if (__builtin_amdgcn_ballot_w64(__builtin_bit_cast(uint32_t, reached) != __builtin_bit_cast(uint32_t, below)) == 0) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned long long in = __builtin_amdgcn_ballot_w64(o[h] >= bound);
                    const uint32_t at = mine + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0u));
                    if (o[h] >= bound && at < kBeamPart) list[wave * kBeamPart + at] = entry(o[h], i, h);
                    mine += (uint32_t)__builtin_popcountll(in);
                }
            }
        }
        if (lane == 0) counts[wave] = mine;
        if (lane < 4u && mine + lane < kBeamPart) list[wave * kBeamPart + mine + lane] = 0u;   // (read four at a time below)
        __syncthreads();
        const uint32_t n = counts[0] + counts[1] + counts[2] + counts[3];
        const bool fits = counts[0] <= kBeamPart && counts[1] <= kBeamPart && counts[2] <= kBeamPart && counts[3] <= kBeamPart;
        uint32_t* const out = a.best + ((size_t)row * a.pieces + piece) * k;
        if (__builtin_expect(fits && n <= 64u, 1)) {   // one wave, an entry a lane
            if (wave == 0) {
                const uint32_t c0 = counts[0], c1 = c0 + counts[1], c2 = c1 + counts[2];
                const uint32_t at = lane < c0 ? lane : lane < c1 ? kBeamPart + lane - c0 : lane < c2 ? 2u * kBeamPart + lane - c1 : 3u * kBeamPart + lane - c2;
                const uint32_t key = lane < n ? list[at] : 0u, all_n = __builtin_amdgcn_readfirstlane(n);
                uint32_t rank = 0;
                for (uint32_t o = 0; o < all_n; ++o) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, (int)o) > key ? 1u : 0u;
                if (lane < n && rank < k) __hip_atomic_store(&out[rank], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (lane >= n && lane < k) __hip_atomic_store(&out[lane], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        } else if (__builtin_expect(fits, 1)) {
            for (uint32_t c = lane; c < mine; c += 64u) {
                const uint32_t key = list[wave * kBeamPart + c];
                uint32_t rank = 0;
                for (uint32_t p = 0; p < 4u; ++p)
                    for (uint32_t o = 0; o < counts[p]; o += 4u) {
                        const uint4 v = *reinterpret_cast<const uint4*>(&list[p * kBeamPart + o]);
                        rank += (v.x > key ? 1u : 0u) + (v.y > key ? 1u : 0u) + (v.z > key ? 1u : 0u) + (v.w > key ? 1u : 0u);
                    }
                if (rank < k) __hip_atomic_store(&out[rank], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            for (uint32_t c = n + tid; c < k; c += 256u) __hip_atomic_store(&out[c], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else {
            uint32_t last = ~0u;
#pragma unroll 1
            for (uint32_t c = 0; c < k; ++c) {
                uint32_t best = 0;
                again();
#pragma unroll
                for (int i = 0; i < VEC * 4; ++i) {
                    const i16x2_t o = beam_order(w[i]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t key = o[h] >= kBeamLeast ? entry(o[h], i, h) : 0u;
                        best = key < last && key > best ? key : best;
                    }
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
            for (int i = 0; i < 4; ++i) s += part[i] * (double)__builtin_amdgcn_exp2f((top[i] - rt) * kBeamLog2E);
            const size_t at = (size_t)row * a.pieces + piece;
            __hip_atomic_store(&a.tops[at], mt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(reinterpret_cast<unsigned long long*>(&a.sums[at]), (unsigned long long)__double_as_longlong(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }

    // ---- the group's last block ----
    wait_memory_ops_done();
    __syncthreads();
    if (tid == 0) flag = atomicAdd(&a.arrived[g * kBeamCounterStep], 1u) == a.beams * a.pieces - 1u ? 1u : 0u;
    __syncthreads();
    if (__builtin_expect(!flag, 1)) return;
    if (tid == 0) __hip_atomic_store(&a.arrived[g * kBeamCounterStep], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t total = a.beams * a.pieces * k;
    const uint32_t* const group_best = a.best + (size_t)g * total;
    auto load = [&](uint32_t i) { return i < total ? __hip_atomic_load(&group_best[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u; };
    // (of a finished row nothing was written: its keys are not looked at, whatever they are)
    // The first entries of all lists go into LDS with one request, as many of each as fit.
    const uint32_t lists = a.beams * a.pieces, deep = lists * k <= AHEAD * 256u ? k : AHEAD * 256u / lists;
    if (deep) {
        const uint32_t whole = lists * deep;
        uint32_t key[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t i = u * 256u + tid, l = i / deep;
            key[u] = i < whole ? load(l * k + (i - l * deep)) : 0u;
        }
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) keys[u * 256u + tid] = key[u];
    }
    auto key_of = [&](uint32_t l, uint32_t j) { return j < deep ? keys[l * deep + j] : load(l * k + j); };
    const uint32_t of_beam = g * a.beams + (tid < a.beams ? tid : 0u), is_over = a.finished ? a.finished[of_beam] : 0u;
    const float score = a.scores[of_beam];
    for (uint32_t b0 = wave; b0 < a.beams; b0 += 16u) {   // four beams of a wave with one request
        float m4[4];
        double s4[4];
        auto sums_of = [&](uint32_t b, uint32_t p, float& mp, double& sp) {
            const size_t at = (size_t)(g * a.beams + (b < a.beams ? b : b0)) * a.pieces + (p < a.pieces ? p : a.pieces - 1u);
            mp = __hip_atomic_load(&a.tops[at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sp = __longlong_as_double((long long)__hip_atomic_load(reinterpret_cast<unsigned long long*>(&a.sums[at]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) sums_of(b0 + 4u * u, lane, m4[u], s4[u]);
#pragma unroll 1
        for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t b = b0 + 4u * u;
            if (b >= a.beams) break;
            float m = wave_max(m4[0]), ref = m == -INFINITY ? 0.f : m;   // the sum is relative to m, which is the wave's
            double s = lane < a.pieces ? s4[0] * (double)__builtin_amdgcn_exp2f((m4[0] - ref) * kBeamLog2E) : 0.0;
            for (uint32_t p0 = 64u; __builtin_expect(p0 < a.pieces, 0); p0 += 64u) {
                float mp;
                double sp;
                sums_of(b, p0 + lane, mp, sp);
                const float mn = fmaxf(m, wave_max(mp));
                ref = mn == -INFINITY ? 0.f : mn;
                s = s * (double)__builtin_amdgcn_exp2f((m - ref) * kBeamLog2E) +
                    (p0 + lane < a.pieces ? sp * (double)__builtin_amdgcn_exp2f((mp - ref) * kBeamLog2E) : 0.0);
                m = mn;
            }
            s = wave_sum_wide(s);
            if (lane == 0) {
                peak[b] = m;
                values[b] = s;
            }
            m4[0] = m4[1], m4[1] = m4[2], m4[2] = m4[3];
            s4[0] = s4[1], s4[1] = s4[2], s4[2] = s4[3];
        }
    }
    __syncthreads();
    if (tid < a.beams) {
        ended[tid] = is_over;
        base[tid] = is_over ? (double)score : (double)score - log(values[tid]);   // and a continuation's total: base + (logit - peak)
        near[tid] = (float)base[tid];
    }
    __syncthreads();
    // Entry j of list l (a piece's, in order): bounds of its score's order in fp32, or nothing; and the score in 64 bits, with its place as
    // beam, how far the logit's order is below the highest, token: ties go to the lower beam, inside it by the logits and then to the lower
    // token, also where a score is so large that 64 bits do not tell logits apart.  A finished row's one candidate is the first entry of its first piece.
    auto rough = [&](uint32_t b, uint32_t p, uint32_t j, uint32_t key, uint32_t& least, uint32_t& most) {
        // (a sum that leaves fp32 although neither part does is still a candidate: its least order is that of -inf)
        const float c = near[b], x = ended[b] ? 0.f : fmaxf(beam_value((int)(key >> 16) - 0x8000) - peak[b], -FLT_MAX), v = c + x;
        const float margin = fminf(fmaxf(__builtin_fabsf(c), __builtin_fabsf(x)) * 0x1p-21f, 0x1p108f);
        least = order_key(v - margin);
        most = order_key(fmaxf(v, -FLT_MAX) + margin);
        return (ended[b] ? (p | j) == 0u : key != 0u) && c > -INFINITY;
    };
    auto exactly = [&](uint32_t b, uint32_t p, uint32_t j, uint32_t key, uint64_t& at) {
        at = (uint64_t)b << 48 | a.pad;
        if (ended[b]) return (p | j) == 0u ? base[b] : (double)-INFINITY;
        at = (uint64_t)b << 48 | (uint64_t)(0xffffu - (key >> 16)) << 32 | (p * PIECE + (0xffffu - (key & 0xffffu)));
        const double v = base[b] + ((double)beam_value((int)(key >> 16) - 0x8000) - (double)peak[b]);
        return key && v > -INFINITY ? v : (double)-INFINITY;
    };
    // The bound: of up to 256 lists from the first 256 / lists entries of each, of more from their first.  k fp32 scores less their margins reach it,
    // so that k scores do.
    uint32_t mine = 0;
#pragma unroll 1
    for (uint32_t l0 = tid; l0 < (lists < 256u ? 256u : lists); l0 += 256u) {
        const uint32_t j = lists < 256u ? l0 / lists : 0u, l = lists < 256u ? l0 - j * lists : l0;
        if (j >= k) break;
        const uint32_t b = l / a.pieces;
        uint32_t least, most;
        if (rough(b, l - b * a.pieces, j, key_of(l, j), least, most)) mine = least > mine ? least : mine;
    }
    const uint32_t bound = bound_of_best<32, 12>(mine, k, all);
    // Who reaches it: a thread goes down a list as far as fp32 scores with their margins do, and looks at those in 64 bits.
    uint32_t found_here = 0;   // of this wave
    __syncthreads();           // (the sums that lay in `values` have been read)
#pragma unroll 1
    for (uint32_t l0 = 0; l0 < lists; l0 += 256u) {
        const uint32_t l = l0 + tid < lists ? l0 + tid : 0u, b = l / a.pieces, p = l - b * a.pieces;
        bool on = l0 + tid < lists;
#pragma unroll 1
        for (uint32_t j = 0; j < k; ++j) {
            const uint32_t key = on ? key_of(l, j) : 0u;
            uint32_t least, most;
            on = rough(b, p, j, key, least, most) && on && most >= bound;
            if (__builtin_amdgcn_ballot_w64(on) == 0) break;
            uint64_t flat;
            const double v = exactly(b, p, j, key, flat);
            const bool is = on && v > -INFINITY && order_key((float)v) >= bound;
            const unsigned long long in = __builtin_amdgcn_ballot_w64(is);
            const uint32_t at = found_here + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0u));
            if (is && at < kBeamPart) {
                values[wave * kBeamPart + at] = v;
                flats[wave * kBeamPart + at] = flat;
            }
            found_here += (uint32_t)__builtin_popcountll(in);
        }
    }
    if (lane == 0) counts[wave] = found_here;
    __syncthreads();
    const uint32_t n = counts[0] + counts[1] + counts[2] + counts[3];
    const bool fits = counts[0] <= kBeamPart && counts[1] <= kBeamPart && counts[2] <= kBeamPart && counts[3] <= kBeamPart;
    auto put = [&](uint32_t at, double v, uint64_t flat) {
        a.out_scores[(size_t)g * k + at] = (float)v;
        a.out_beams[(size_t)g * k + at] = (uint32_t)(flat >> 48);
        a.out_tokens[(size_t)g * k + at] = (uint32_t)flat;
    };
    if (__builtin_expect(fits, 1)) {
        for (uint32_t c = lane; c < found_here; c += 64u) {
            const double v = values[wave * kBeamPart + c];
            const uint64_t flat = flats[wave * kBeamPart + c];
            uint32_t rank = 0;
            for (uint32_t p = 0; p < 4u; ++p)
#pragma unroll 2
                for (uint32_t o = p * kBeamPart; o < p * kBeamPart + counts[p]; ++o) {
                    const double other = values[o];
                    const uint64_t place = flats[o];
                    rank += (uint32_t)(other > v) | ((uint32_t)(other == v) & (uint32_t)(place < flat));
                }
            if (rank < k) put(rank, v, flat);
        }
        if (__builtin_expect(n >= k || tid != 0, 1)) return;
        // fewer than k above -inf: the lowest places that are not among them
        uint64_t at = 0;
        auto next = [&] { at = (uint32_t)at + 1u < a.vocab ? at + 1u : ((at >> 48) + 1u) << 48; };
        for (uint32_t i = n; i < k; ++i, next()) {
            for (bool again = true; again;) {
                again = false;
                for (uint32_t c = 0; c < kBeamList; ++c)
                    if (c % kBeamPart < counts[c / kBeamPart] && (flats[c] >> 48 << 48 | (uint32_t)flats[c]) == at) {
                        next();
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
            const uint32_t l = i / k, b = l / a.pieces;
            uint64_t flat;
            const double v = exactly(b, l - b * a.pieces, i - l * k, load(i), flat);
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
            flats[wave] = at;
        }
        __syncthreads();
        for (int i = 0; i < 4; ++i) {
            if (values[i] > best || (values[i] == best && flats[i] < at)) {
                best = values[i];
                at = flats[i];
            }
        }
        last = best;
        last_at = at;
        if (tid == 0) put(c, best, at);   // (more than fit into the list: k of them exist)
    }
}

// Pieces of 8192 tokens where that makes two blocks a CU, else of 2048 (measured above).
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
// A thread takes one column of a group and N of its output rows: it requests them all before it writes one.  In place N covers all rows (of 16-byte
// columns up to 16: more would not stay in registers, and go by words); apart, eight rows a thread and a part of the grid for each eight.
// Bound by the bytes; the two columns that a wave's rows share a line in cost nothing that shows.  64 rows of 2.4 MB in 49 us, 6.3 TB/s read and written (what
// the last-level cache holds of them counts); 4 rows of 8 KB in 2.6.
struct ReorderArgs {
    const void* src;
    void* dst;
    size_t src_stride, dst_stride, columns;   // in values of T
    const uint32_t* parents;
    uint32_t beams, n_out;
};
template <typename T, uint32_t N>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const ReorderArgs a) {
    const size_t c = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.columns) return;
    const uint32_t g = blockIdx.y, first = blockIdx.z * N;
    const T* src = static_cast<const T*>(a.src) + (size_t)g * a.beams * a.src_stride + c;
    T* dst = static_cast<T*>(a.dst) + ((size_t)g * a.n_out + first) * a.dst_stride + c;
    const uint32_t* parents = a.parents + (size_t)g * a.n_out + first;
    const uint32_t rows = a.n_out - first;
    T v[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        const uint32_t p = parents[i < rows ? i : rows - 1u];
        v[i] = src[(size_t)(p < a.beams ? p : a.beams - 1u) * a.src_stride];
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
        if (i < rows) dst[(size_t)i * a.dst_stride] = v[i];
}

namespace {
// the smallest form whose threads hold N rows or more, or null
template <typename T, uint32_t... N>
const void* reorder_form(uint32_t rows, uint32_t* held) {
    const void* f = nullptr;
    ((f == nullptr && rows <= N ? (f = reinterpret_cast<const void*>(&beam_reorder_kernel<T, N>), *held = N) : 0u), ...);
    return f;
}
}  // namespace

fk_status plan_beam_reorder(const void* src, size_t src_stride, void* dst, size_t dst_stride, size_t row_bytes, const uint32_t* parents, uint32_t groups,
                            uint32_t beams, uint32_t n_out, Launch* l) {
    if (!src || !dst || !parents) return set_error(FK_ERR_INVALID, "beam_reorder: null pointer");
    if (row_bytes == 0 || groups == 0 || beams == 0 || n_out == 0) return set_error(FK_ERR_INVALID, "beam_reorder: empty shape");
    if (beams > kBeamMax || n_out > kBeamMax) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: beams up to 64");
    if (groups > 65535) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: more than 65535 groups");
    if (src_stride < row_bytes || dst_stride < row_bytes) return set_error(FK_ERR_INVALID, "beam_reorder: a row stride is shorter than the row");
    if ((uintptr_t)parents & 3u) return set_error(FK_ERR_INVALID, "beam_reorder: parents must be 4-byte aligned");
    if (std::max(src_stride, dst_stride) > (SIZE_MAX >> 1) / ((size_t)groups * kBeamMax)) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: state too large");
    const uintptr_t s0 = (uintptr_t)src, d0 = (uintptr_t)dst;
    const size_t sn = ((size_t)groups * beams - 1) * src_stride + row_bytes, dn = ((size_t)groups * n_out - 1) * dst_stride + row_bytes;
    const bool in_place = s0 == d0;
    if (in_place ? n_out != beams || src_stride != dst_stride : (s0 < d0 + dn && d0 < s0 + sn))
        return set_error(FK_ERR_INVALID, "beam_reorder: src and dst must be the same rows, n_out then being beams, or not overlap");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    const uint32_t rows = in_place ? n_out : std::min(n_out, 8u);
    const uintptr_t all = s0 | d0 | row_bytes | src_stride | dst_stride;
    const uint32_t width = all % 16 == 0 && rows <= 16 ? 16 : all % 4 == 0 ? 4 : 1;
    ReorderArgs a{src, dst, src_stride / width, dst_stride / width, row_bytes / width, parents, beams, n_out};
    if ((a.columns + 255) / 256 > 0x7fffffffu) return set_error(FK_ERR_UNSUPPORTED, "beam_reorder: rows too long");
    uint32_t held = 1;
    l->func = width == 16 ? reorder_form<fk_u32x4_t, 2, 4, 8, 16>(rows, &held)
              : width == 4 ? reorder_form<uint32_t, 2, 4, 8, 16, 32, kBeamMax>(rows, &held) : reorder_form<uint8_t, 4, 16, kBeamMax>(rows, &held);
    l->grid = dim3((uint32_t)((a.columns + 255) / 256), groups, (n_out + held - 1) / held);
    l->block = dim3(256, 1, 1);
    l->set_args(a);
    return FK_OK;
}

}  // namespace fk
