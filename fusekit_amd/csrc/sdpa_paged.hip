// Attention of new rows -- chunks of prompts, single tokens, both in one batch -- over a paged cache.
//
//     out[r, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(x_j - max x),   x_j = c(q[r, h] . K[j] * scale),   max(0, p - window + 1) <= j <= p
//
// with p the row's position and c(x) = x, or softcap * tanh(x / softcap); with `sinks` also the positions j < sinks (j <= p) before the window.
#include <math.h>

#include <algorithm>

#include "fk_host.hpp"
#include "mma32_device.hpp"
#include "paged_device.hpp"

namespace fk {

// Probabilities carry the factor 2^-8, which cancels, since a step's maximum may lie 2^8 above the softmax reference: values down to the type's smallest
// keep their products in fp32's range, and sums of its largest that leave it are done again by paged_row, in 64 bits.
constexpr float kPagedLag = 8.0f;
constexpr float kLog2E = 1.44269504088896341f;

struct SdpaPagedArgs {
    PagedArgs b;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    uint32_t q_stride, out_stride, group;
    uint32_t window, sinks;
    float scale, softcap;
    float* partials;       // [slots][columns of a tile][D], then (m, l) [slots][columns of a tile]
    uint32_t* counters;    // [slots], zero before the first launch, left zero
    uint32_t slots, slot_bytes;
    uint32_t target, min_steps;   // items that a launch is cut into where its tiles are fewer; the least steps of an item
    uint32_t compact;             // tiles may be more than slots: only those that are cut have some
    uint32_t blocks;              // of the launch
    uint32_t only_few;            // of chunks among single tokens: whole chunks, cut tokens (compact)
};

// Positions up to that of a sequence's new row `place`; 0: the row sees nothing.
__device__ __forceinline__ uint32_t paged_limit(const PagedSeq& s, uint32_t place) { return s.len + place + 1u > s.rows ? s.len + place + 1u - s.rows : 0u; }

// What sums of probabilities are multiplied with, l their total: 0 for a row that sees nothing, and not a number, which has the column done again by
// paged_row, where l is not between bounds that it does not leave unless scores are beyond some 1e9: the reference, a rounded product, and the exponents,
// each one rounding of product and reference, are then apart by more than fp32's exponents hold.
__device__ __forceinline__ float paged_inverse(float l, uint32_t limit) {
    const float f = 1.0f / l;
    return __builtin_expect(f > 0x1p-60f && f < 0x1p60f, 1) ? f : limit ? __builtin_nanf("") : 0.f;
}

// Sinks are a matter of the kernel's type: kept at run time, none of them cost a chunk of 512 rows behind 2500 positions with a window of 2000 41.8 us for
// 38.5 (the registers that hold addresses go to them).
template <bool SINKS>
__device__ __forceinline__ uint32_t paged_sinks(const SdpaPagedArgs& a) {
    return SINKS ? a.sinks : 0u;
}

// ---- one row of one head by a wave: positions in the order they lie, what the row does not see is not touched ----
// The statement of the operator as it stands; the tiles below come here for a column whose sums are not finite, since a zero
// probability times an infinity that other rows of the tile see is no number.
template <int D, bool SINKS>
__device__ __forceinline__ void paged_row(const SdpaPagedArgs& a, uint32_t seq, const PagedSeq& s, uint32_t place, uint32_t head, uint32_t lane) {
    const uint32_t kvh = head / a.group, row = s.row0 + place, page_rows = 1u << a.b.page_shift;
    const uint32_t end = paged_limit(s, place);
    const uint32_t first = a.window && end > a.window ? end - a.window : 0u;
    const uint32_t sinks = paged_sinks<SINKS>(a) < first ? paged_sinks<SINKS>(a) : first, gap = first - sinks, seen = end - gap;   // the positions seen: sinks, then from `first` on
    const uint16_t* qr = a.q + (size_t)row * a.q_stride + (size_t)head * D;
    constexpr int DL = D / 64;
    uint32_t bad = 0;
    float m = -INFINITY;
    double l = 0.0, o[DL];   // (values of the type's whole range, and 2^31 of the largest)
#pragma unroll
    for (int i = 0; i < DL; ++i) o[i] = 0.0;
    for (uint32_t at = 0; at < seen; at += 64u) {
        const uint32_t place_seen = at + lane < seen ? at + lane : seen - 1u, pos = place_seen < sinks ? place_seen : place_seen + gap;
        const uint32_t page = paged_page(a.b, seq, pos >> a.b.page_shift, bad);
        const size_t base = (((size_t)page * a.b.n_kv + kvh) * page_rows + (pos & (page_rows - 1u))) * D;
        const uint4* kr = reinterpret_cast<const uint4*>(a.k + base);
        float x = 0.f;
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) {
            const uint4 kk = kr[i], qq = reinterpret_cast<const uint4*>(qr)[i];
            const uint32_t kw[4] = {kk.x, kk.y, kk.z, kk.w}, qw[4] = {qq.x, qq.y, qq.z, qq.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) x = fmaf(bf16_hi(kw[e]), bf16_hi(qw[e]), fmaf(bf16_lo(kw[e]), bf16_lo(qw[e]), x));
        }
        x *= a.scale;
        if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
        if (at + lane >= seen) x = -INFINITY;
        const float m_new = fmaxf(m, wave_max(x)), ref = m_new == -INFINITY ? 0.f : m_new, alpha = expf(m - ref), p = expf(x - ref);
        l = l * alpha + (double)wave_sum(p);
        m = m_new;
#pragma unroll
        for (int i = 0; i < DL; ++i) o[i] *= alpha;
        const uint32_t n = seen - at < 64u ? seen - at : 64u;
#pragma unroll 1
        for (uint32_t j = 0; j < n; ++j) {
            const float pj = __shfl(p, (int)j, 64);
            const size_t vb = __shfl((unsigned long long)base, (int)j, 64);
#pragma unroll
            for (int i = 0; i < DL; ++i) o[i] = fma((double)pj, (double)bf16_bits_to_f32(a.v[vb + lane + 64u * i]), o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < DL; ++i)
        a.out[(size_t)row * a.out_stride + (size_t)head * D + lane + 64u * i] = (uint16_t)f32_to_bf16_bits(seen ? (float)(o[i] / l) : 0.f);
}

// ---- which piece of the work a block does ----
// The columns of a sequence and KV head are its new rows times the query heads of a group, place * group + head; 128 of them are a tile, of a
// sequence of up to kFewMost 16.  A tile walks its positions in steps of 64 (single tokens in rounds of 128); where all tiles of the
// launch are fewer than `target` the steps are cut over several items.  Every wave finds its block's item by itself from the batch's arrays,
// 64 sequences with one request: lengths stay on the device.
constexpr uint32_t kTileCols = 128, kTileStep = 64;
constexpr uint32_t kFewCols = 16, kFewMost = 32, kFewStep = 32, kFewRound = 4 * kFewStep;
constexpr uint32_t kMostSplits = 64;   // items of a tile
struct PagedItem {
    uint32_t seq, kvh, tile, split, n_splits;
    uint32_t base;   // the slot of the tile's first item, whose others follow n_kv apart
    uint32_t slot;   // the item's own
    PagedSeq s;
    bool any;
};
// FEW: a launch of single tokens only.  TILES: `index` counts tiles, not items.
template <bool FEW, uint32_t COLS, bool SINKS, bool TILES = false>
__device__ __forceinline__ PagedItem paged_item(const SdpaPagedArgs& a, uint32_t index, uint32_t lane) {
    constexpr uint32_t STEP = FEW ? kFewRound : kTileStep;
    const uint32_t n_kv = a.b.n_kv;
    auto tiles_of = [&](const PagedSeq& s) {   // (rows times heads of a group: below 2^31, the host has checked)
        const uint32_t columns = s.rows * a.group, width = columns <= kFewMost ? kFewCols : COLS;
        return (columns + width - 1u) / width;
    };
    auto steps_of = [&](const PagedSeq& s) {   // of a tile of the sequence, at most
        uint32_t seen = s.len;
        if (a.window) {
            const uint32_t span = COLS / a.group + 2u;   // rows of a tile, at most
            const uint64_t w = (uint64_t)a.window + paged_sinks<SINKS>(a) + (s.rows < span ? s.rows : span) + (SINKS ? 2u * STEP : STEP) - 1u;
            seen = w < seen ? (uint32_t)w : seen;
        }
        return (seen + STEP - 1u) / STEP;
    };
    auto read = [&](uint32_t at) {
        const uint32_t i = at + lane;
        PagedSeq s = paged_seq(a.b, i < a.b.n_seqs ? i : a.b.n_seqs - 1u);
        if (i >= a.b.n_seqs) s.rows = 0;
        if (s.bad && i < a.b.n_seqs && index == 0) paged_fault(a.b, s.bad);
        return s;
    };
    bool only_few = !FEW && !TILES && a.only_few != 0;   // (whole tiles have no slots)
    auto whole = [&](const PagedSeq& s) { return only_few && s.rows * a.group > kFewMost; };
    float work = 0.f, pairs = 0.f, wholes = 0.f, longest_whole = 0.f, longest_cut = 0.f;   // pairs: of tiles that may be cut
    // (64 sequences at a time, three requests ahead, and once where nothing is cut: 1000 of them were 32 trips to memory one after another)
    const bool many = a.b.n_seqs > 64u;
    PagedSeq mine, ahead[3];
    auto from_the_first = [&] {
        mine = read(0);
        if (many)
#pragma unroll
            for (uint32_t u = 0; u < 3; ++u) ahead[u] = read(64u * (u + 1u));
    };
    auto next = [&](uint32_t at) {   // (past the last sequence: ones without rows)
        mine = ahead[0], ahead[0] = ahead[1], ahead[1] = ahead[2];
        ahead[2] = read(at + 192u);
    };
    from_the_first();
    const bool once = a.slots == 0 && index != 0;   // (nothing to cut: the sums are for the faults alone)
    for (uint32_t at = 0; !once;) {
        const float t = (float)tiles_of(mine) * (float)n_kv;
        work = fmaf(t, (float)steps_of(mine), work);   // (the merge forms the same value)
        pairs += whole(mine) ? 0.f : t;
        if (only_few) {
            const float steps = mine.rows ? (float)steps_of(mine) : 0.f;
            if (whole(mine)) {
                wholes += t;
                longest_whole = fmaxf(longest_whole, steps);
            } else {
                longest_cut = fmaxf(longest_cut, steps);
            }
        }
        if ((at += 64u) >= a.b.n_seqs) break;
        next(at);
    }
    work = wave_sum(work);
    pairs = wave_sum(pairs);
    // (compact: a tile that is cut has more than one share, and fewer than twice as many items as shares: 2 target of them have slots)
    const bool compact = only_few || (!TILES && a.compact != 0 && !(pairs + (float)a.target <= (float)a.slots));
    // (a batch whose row_start falls can have more tiles than the host has counted: cut, the last items of a tile would be behind the launch's end,
    // and its counter would never be left ready)
    bool cut = pairs + (float)a.target <= (float)(compact ? a.blocks : a.slots);
    // (of at least work / target steps: all items together are at most target + pairs)
    const float share = work / (float)a.target;
    uint32_t unit = share < 0x1p30f ? (uint32_t)ceilf(share) : 1u << 30;
    unit = unit < a.min_steps ? a.min_steps : unit;
    const float of_steps = 1.0f / fmaxf(share, (float)a.min_steps);
    PagedItem it;
    it.any = false;
    uint32_t left = index, before = 0;   // slots of the sequences before
    // Single tokens among whole tiles are cut where one of them is twice as long as the tiles; in a launch of more than the card takes at once they come
    // first, in a way through the sequences of their own, else last, so that each tile has a CU first.  Two chunks of 2048 rows and a token over 100 000
    // positions, us: not cut 1092, cut and in the sequences' order 215, tokens first 140; a chunk of 2048 and 16 tokens over 8000: 144, 152, 119; a
    // chunk of 509 rows among 24 tokens over up to 2000: 39, 39, 42.
    bool tokens = true;
    if (only_few) {
        longest_whole = wave_max(longest_whole);
        longest_cut = wave_max(longest_cut);
        const float tiles = wave_sum(wholes) + pairs;
        only_few = cut = longest_cut > 2.0f * longest_whole && tiles + (float)a.target <= (float)a.blocks;
        tokens = !only_few || tiles > (float)a.target;
    }
    bool second = !only_few;
    if (many && !once) from_the_first();
    for (uint32_t at = 0;;) {
        const uint32_t tiles = tiles_of(mine);
        // (tiles: as many as fit; an integer share gave a chunk of 512 rows behind 3000 384 items instead of 512)
        uint32_t splits = !cut || whole(mine) ? 1u : FEW || only_few ? (steps_of(mine) + unit - 1u) / unit : (uint32_t)fmaf((float)steps_of(mine), of_steps, 0x1p-10f);
        splits = splits < 1u ? 1u : splits > kMostSplits ? kMostSplits : splits;
        const uint32_t items = tiles * splits * n_kv;
        auto with_those_before = [&](uint32_t upto) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(upto, o, 64);
                upto += lane >= (uint32_t)o ? v : 0u;
            }
            return upto;
        };
        const uint32_t count = TILES ? tiles * n_kv : only_few && whole(mine) == tokens ? 0u : items;
        const uint32_t slots = compact && splits == 1u ? 0u : TILES ? items : count;
        const uint32_t counted = with_those_before(count), upto = TILES || compact ? with_those_before(slots) : counted;
        const unsigned long long past = __builtin_amdgcn_ballot_w64(counted > left);
        if (!past) {
            left -= (uint32_t)__builtin_amdgcn_readlane((int)counted, 63);
            before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
            at += 64u;
            if (at < a.b.n_seqs) {
                next(at);
                continue;
            }
            if (second) break;
            second = true;
            tokens = !tokens;
            at = 0;
            if (many) from_the_first();
            continue;
        }
        const int who = (int)__builtin_ctzll(past);
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, who); };
        left -= of(counted) - of(count);
        before += of(upto) - of(slots);
        it.seq = at + (uint32_t)who;
        it.s = PagedSeq{of(mine.row0), of(mine.rows), of(mine.len), of(mine.bad)};
        it.n_splits = of(splits);
        it.kvh = left % n_kv;
        left /= n_kv;
        it.split = TILES ? 0u : left % it.n_splits;
        left = TILES ? left : left / it.n_splits;
        it.tile = of(tiles) - 1u - left;   // the longest first
        it.base = before + left * it.n_splits * n_kv + it.kvh;
        it.slot = it.base + it.split * n_kv;
        it.any = true;
        break;
    }
    return it;
}
constexpr int kPastCaches = 16;   // (sc1: what another block wrote, or is to read)

// What a tile's columns e_tile .. e_last see, in steps of STEP positions, and how its items share them: item i takes `per` of the `steps` from i * per on.
// The steps are counted without those that lie between the sinks and the window: step number n is n, from `near` on n + gap.
// (Sinks cost their own steps: 64 tokens of up to 20000 positions, 32 / 8 heads x 128, with a window of 4096 and 100 of them 118 us, 115 without; two chunks of
// 2048 rows with as wide a window and 128 of them 302, 289 without.)
struct PagedRange {
    uint32_t kv_end, steps, per, n_active;   // n_active: items that have steps, one at least
    uint32_t near, gap;
    __device__ __forceinline__ uint32_t step(uint32_t n) const { return n < near ? n : n + gap; }
};
template <uint32_t STEP, bool SINKS>
__device__ __forceinline__ PagedRange paged_range(const SdpaPagedArgs& a, const PagedItem& it, uint32_t e_tile, uint32_t e_last) {
    auto limit_of = [&](uint32_t place) { return paged_limit(it.s, place); };
    PagedRange r;
    r.kv_end = __builtin_amdgcn_readfirstlane(limit_of(e_last / a.group));
    const uint32_t first = limit_of(e_tile / a.group);
    const uint32_t step0 = __builtin_amdgcn_readfirstlane((a.window && first > a.window ? first - a.window : 0u) / STEP);
    const uint32_t sinks = paged_sinks<SINKS>(a), sink_steps = sinks / STEP + (sinks % STEP ? 1u : 0u);
    r.near = sink_steps < step0 ? sink_steps : step0;
    r.gap = step0 - r.near;
    r.steps = (r.kv_end + STEP - 1u) / STEP - (r.kv_end ? r.gap : 0u);
    r.per = (r.steps + it.n_splits - 1u) / it.n_splits;
    r.n_active = r.per ? (r.steps + r.per - 1u) / r.per : 1u;
    return r;
}

// What a wave hands on of up to 32 columns, `live` of them, et the first, from ob, [32][D + 4] in LDS.  Where the tile is cut: the sums as they are, the reference and
// the sum of the probabilities into this item's slot (`c0`: the first column's place there).
template <int D>
__device__ __forceinline__ void paged_store_part(const SdpaPagedArgs& a, const PagedItem& it, const float* ob, uint32_t c0, uint32_t live, float m, float l, uint32_t lane) {
    constexpr uint32_t OS = D + 4;
    const __amdgpu_buffer_rsrc_t mem = __builtin_amdgcn_make_buffer_rsrc(a.partials + (size_t)it.slot * (kTileCols * (D + 2u)), 0, (int)(kTileCols * (D + 2u) * 4u), 0x27000);
    for (uint32_t idx = lane; idx < live * (uint32_t)(D / 4); idx += 64u) {
        const uint32_t col = idx / (uint32_t)(D / 4), pc = idx % (uint32_t)(D / 4);
        const pf_u32x4_t v = *reinterpret_cast<const pf_u32x4_t*>(ob + col * OS + pc * 4u);
        __builtin_amdgcn_raw_buffer_store_b128(v, mem, (int)(((c0 + col) * D + pc * 4u) * 4u), 0, 0);
    }
    if (lane < live) {   // (the lanes below 32 hold all of a column's l)
        const pf_u32x2_t ml = {__float_as_uint(m), __float_as_uint(l)};
        __builtin_amdgcn_raw_buffer_store_b64(ml, mem, (int)((kTileCols * D + (c0 + lane) * 2u) * 4u), 0, 0);
    }
}
// Where it is whole: outputs.
template <int D, bool SINKS>
__device__ __forceinline__ void paged_store_columns(const SdpaPagedArgs& a, const PagedItem& it, const float* ob, uint32_t et, uint32_t live, uint32_t lane) {
    constexpr uint32_t OS = D + 4, VP = D / 8;
    const uint32_t G = a.group;
    uint32_t again = 0;   // columns whose sums are not finite, done again one by one
    for (uint32_t base = 0; base < live * VP; base += 64u) {
        const uint32_t idx = base + lane, col = idx / VP, pc = idx % VP;
        const bool in = col < live;
        const float4 lo = *reinterpret_cast<const float4*>(ob + (in ? col : 0u) * OS + pc * 8u);
        const float4 hi = *reinterpret_cast<const float4*>(ob + (in ? col : 0u) * OS + pc * 8u + 4u);
        const uint32_t ec = et + col, pl = ec / G;
        if (in)
            *reinterpret_cast<uint4*>(a.out + (size_t)(it.s.row0 + pl) * a.out_stride + (size_t)(it.kvh * G + (ec - pl * G)) * D + pc * 8u) =
                make_uint4(pack_bf16(lo.x, lo.y), pack_bf16(lo.z, lo.w), pack_bf16(hi.x, hi.y), pack_bf16(hi.z, hi.w));
        const float t = (__builtin_fabsf(lo.x) + __builtin_fabsf(lo.y)) + (__builtin_fabsf(lo.z) + __builtin_fabsf(lo.w)) +
                        (__builtin_fabsf(hi.x) + __builtin_fabsf(hi.y)) + (__builtin_fabsf(hi.z) + __builtin_fabsf(hi.w));
        unsigned long long odd = __builtin_amdgcn_ballot_w64(in && !(t < INFINITY));
        for (; odd; odd &= odd - 1u) again |= 1u << ((base + (uint32_t)__builtin_ctzll(odd)) / VP);
    }
    for (; again; again &= again - 1u) {
        const uint32_t ec = et + (uint32_t)__builtin_ctz(again), pl = ec / G;
        paged_row<D, SINKS>(a, it.seq, it.s, pl, it.kvh * G + (ec - pl * G), lane);
    }
}

// ---- tiles of 128 columns ----
// A block is four waves of 32 columns on the same 64 positions a step (SPLIT 1).  The products and the softmax are those of the causal attention of one
// sequence over a contiguous cache (sdpa_prefill.hip: S^T = K Q^T, a lane owns one query; O^T += V^T P^T with the score registers as they lie; V^T
// through ds_read_b64_tr_b16; probabilities formed between the matrix instructions).  A wave requests 16 rows of K and of V a step (SPLIT
// times), which lie in one page: one page id, loaded two steps ahead into a scalar register.
// Two chunks of 2048 rows behind some 3000 positions, 32 / 8 heads x 128: 430 us, 1000 TFLOP/s (a large bf16 product of the vendor's library reaches 1150 to 1380
// on the same card).  The matrix unit works in half of the cycles, the vector unit as long.  What holds the rate is the card's power as much as that:
// tiles of 256 columns with the softmax of one step between the products of another took a fifth fewer cycles at a clock a fifth lower (1.94 -> 1.54 GHz),
// 428 us for 439, and lost a third where tiles are few.
// A probability enters the second product as bf16, off by 2^-8 of itself at most, the sum it is divided by as fp32: outputs are off by 2.1e-3 of their norm where
// their own rounding is 1.7e-3.  A second half, as single tokens have, would be half as many matrix instructions again.
// SPLIT 2: tiles of 64 columns and 128 positions a step, for launches that leave CUs to themselves; two waves share 32 columns, 64 positions a step each,
// and join at the end (the planner has the rule and its figures).
constexpr uint32_t tile_lds_bytes(uint32_t d, uint32_t split) {
    const uint32_t stage = split * 2u * 2u * kTileStep * d * 2u, outb = 4u * 32u * (d + 4u + 2u) * 4u;
    return stage > outb ? stage : outb;
}

template <int D, bool CAP, uint32_t SPLIT, bool SINKS>
__device__ __forceinline__ void paged_tile(const SdpaPagedArgs& a, const PagedItem& it, uint32_t lane) {
    constexpr int KB = D / 16, DT = D / 32, VP = D / 8;
    constexpr uint32_t COLS = kTileCols / SPLIT, STEP = kTileStep * SPLIT;           // of a block: columns, positions a step
    constexpr uint32_t ROW = D * 2u, TILE = STEP * ROW, STAGE = 2u * TILE;           // bytes: a row, K (or V) of a step, both
    constexpr uint32_t RPI = 1024u / ROW;                                            // rows of one wave's request
    constexpr int REQ = 16 / (int)RPI;                                               // requests of 16 rows of a matrix
    extern __shared__ uint4 lds_raw[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_raw);

    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kb = lane >> 5, nl = lane & 31u;
    const uint32_t G = a.group, columns = it.s.rows * G;   // (below 2^31: the host has checked)
    const uint32_t column_tile = SPLIT == 1 ? wave : wave & 1u, my_half = SPLIT == 1 ? 0u : wave >> 1;
    auto limit_of = [&](uint32_t place) { return paged_limit(it.s, place); };                              // positions a row may see end here
    auto low_of = [&](uint32_t limit) { return a.window && limit > a.window ? limit - a.window : 0u; };                           // and begin here
    const uint32_t e_tile = it.tile * COLS, e_last = columns - e_tile < COLS ? columns - 1u : e_tile + COLS - 1u;
    const uint32_t sinks = paged_sinks<SINKS>(a);
    const PagedRange range = paged_range<STEP, SINKS>(a, it, e_tile, e_last);
    const uint32_t kv_end = range.kv_end, n_active = range.n_active;
    if (it.split >= n_active) return;
    const uint32_t begin = __builtin_amdgcn_readfirstlane(it.split * range.per);
    const uint32_t stop = __builtin_amdgcn_readfirstlane(it.split + 1u == n_active ? range.steps : begin + range.per);

    // this lane's column; a wave's columns past the last repeat it, and a wave without columns does the last one's loads and nothing else
    const uint32_t e0 = e_tile + column_tile * 32u;
    const uint32_t live = e0 <= e_last ? (e_last - e0 < 31u ? e_last - e0 + 1u : 32u) : 0u;
    const uint32_t e = live ? e0 + (nl < live ? nl : live - 1u) : e_last;
    const uint32_t place = e / G, head = it.kvh * G + (e - place * G);
    const uint32_t q_limit = limit_of(place), q_low = low_of(q_limit);
    const uint32_t first_limit = live ? __builtin_amdgcn_readfirstlane(limit_of(e0 / G)) : 0u, first_low = __builtin_amdgcn_readfirstlane(low_of(first_limit));
    const uint32_t last_limit = live ? __builtin_amdgcn_readfirstlane(limit_of((e0 + live - 1u) / G)) : 0u, last_low = __builtin_amdgcn_readfirstlane(low_of(last_limit));
    pf_u32x4_t qreg[KB];
    {
        const pf_u32x4_t* qp = reinterpret_cast<const pf_u32x4_t*>(a.q + (size_t)(it.s.row0 + place) * a.q_stride + (size_t)head * D + kb * 8u);
#pragma unroll
        for (int j = 0; j < KB; ++j) qreg[j] = qp[2 * j];
    }

    // the 16-byte piece of a row that lies at place `at`: K reads 16 rows of one piece at a time, V 8 rows of 64 bytes
    auto k_swizzle = [](uint32_t row) { return D == 128 ? row & 15u : (row >> 1) & 7u; };
    auto v_swizzle = [](uint32_t row) { return D == 128 ? (row & 3u) << 2 : ((row >> 1) & 1u) << 2; };
    const uint32_t irow = lane / (uint32_t)VP, at_piece = lane % (uint32_t)VP;
    const uint32_t shift = a.b.page_shift, in_page = (1u << shift) - 1u;
    typedef const uint32_t __attribute__((address_space(4)))* scalar_ptr;
    const uintptr_t table = (uintptr_t)(a.b.table + (size_t)__builtin_amdgcn_readfirstlane(it.seq) * a.b.table_stride);
    uint32_t bad = 0;
    struct Pages {
        uint32_t id[SPLIT];
    };
    auto span_of = [&](uint32_t step, uint32_t g) { return range.step(step) * STEP + (wave * SPLIT + g) * 16u; };   // the first of 16 rows of a step that this wave requests
    auto pages_of = [&](uint32_t step) {                                                                 // (past the range: the last position's)
        Pages p;
#pragma unroll
        for (uint32_t g = 0; g < SPLIT; ++g) {
            const uint32_t span = span_of(step, g), at = span < kv_end ? span : kv_end - 1u;
            p.id[g] = *(scalar_ptr)(table + (size_t)(at >> shift) * 4u);
        }
        return p;
    };
    auto issue = [&](uint32_t step, const Pages& pages, uint32_t stage) {
#pragma unroll
        for (uint32_t g = 0; g < SPLIT; ++g) {
            uint32_t page = pages.id[g];
            if (page >= a.b.n_pages) {
                page = 0;
                bad = FK_PAGED_BAD_PAGE;
            }
            const uint32_t span = span_of(step, g), at = span < kv_end ? span : kv_end - 1u, left = kv_end - 1u - at;
            const size_t off = (((size_t)page * a.b.n_kv + it.kvh) * (in_page + 1u) + (at & in_page)) * ROW;
            const unsigned char *ks = reinterpret_cast<const unsigned char*>(a.k) + off, *vs = reinterpret_cast<const unsigned char*>(a.v) + off;
#pragma unroll
            for (int i = 0; i < REQ; ++i) {
                const uint32_t r = (uint32_t)i * RPI + irow, from = r < left ? r : left;   // (past the range: masked scores, zero probabilities; a swizzle repeats every 16 rows)
                const uint32_t to = stage * STAGE + ((wave * SPLIT + g) * (uint32_t)REQ + (uint32_t)i) * 1024u;
                dma16(to, from * ROW + ((at_piece ^ k_swizzle(r)) * 16u), ks);
                dma16(to + TILE, from * ROW + ((at_piece ^ v_swizzle(r)) * 16u), vs);
            }
        }
    };

    float m_run = -INFINITY, l_run = 0.f;
    pf_f32x16_t oacc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[i][r] = 0.f;

    // fragments: K row nl (+ 32), piece 2 j + kb; V rows 4 kb + (0..3) (+ 8) of 16, columns 32 i + nl
    const uint32_t vrow = 4u * kb + ((lane & 15u) >> 2), vcol = ((lane >> 4) & 1u) * 2u + ((lane & 3u) >> 1), vlow = (lane & 1u) * 8u;
    auto barrier = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const float scale2 = CAP ? 1.0f : a.scale * kLog2E;                              // scores to exponents of two
    const float cap2 = a.softcap * kLog2E, turn2 = CAP ? 2.0f * a.scale * kLog2E / a.softcap : 0.f;

    Pages next = {};
    if (begin < stop) {
        const Pages first = pages_of(begin);
        if (begin + 1u < stop) next = pages_of(begin + 1u);
        issue(begin, first, 0);
    }
    uint32_t stage = 0;
#pragma unroll 1
    for (uint32_t step = begin; step < stop; ++step, stage ^= 1u) {
        wait_loads<0>();
        barrier();   // this step's rows are everybody's; the other stage has been read
        if (step + 1u < stop) {
            issue(step + 1u, next, stage ^ 1u);
            if (step + 2u < stop) next = pages_of(step + 2u);
        }
        const uint32_t kv0 = range.step(step) * STEP + my_half * kTileStep;                   // this wave's 64 positions
        if (kv0 >= last_limit || (kv0 + kTileStep <= first_low && kv0 >= sinks)) continue;   // nothing that a row of this wave sees
        const unsigned char *ks = lds + stage * STAGE + my_half * kTileStep * ROW, *vs = ks + TILE;
        // (two of the eight pairs of fragments ahead of their matrix instructions; all of them first took 1 % longer of two chunks of 2048 rows, 2 % with a window)
        pf_u32x4_t kf[3][2];
        auto read_k = [&](auto j) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t row = (uint32_t)t * 32u + nl;
                kf[j() % 3][t] = *reinterpret_cast<const pf_u32x4_t*>(ks + row * ROW + (((uint32_t)(2 * j()) + kb) ^ k_swizzle(row)) * 16u);
            }
        };
        read_k(std::integral_constant<int, 0>{});
        read_k(std::integral_constant<int, 1>{});
        __builtin_amdgcn_sched_barrier(0);
        pf_f32x16_t s[2];
        static_for<KB>([&](auto j) __attribute__((always_inline)) {
            if constexpr (j() + 2 < KB) read_k(std::integral_constant<int, j() + 2>{});
            __builtin_amdgcn_sched_barrier(0);
            mfma32_scores<j() == 0>(s[0], kf[j() % 3][0], qreg[j()]);
            mfma32_scores<j() == 0>(s[1], kf[j() % 3][1], qreg[j()]);
        });
        __builtin_amdgcn_sched_barrier(0);
        pf_s16x4_t vf[4][DT][2];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t row = (uint32_t)(c * 16 + h * 8) + vrow;
                    const unsigned char* at = vs + row * ROW + (((uint32_t)(4 * i) + vcol) ^ v_swizzle(row)) * 16u + vlow;
                    typedef __attribute__((address_space(3))) pf_s16x4_t* lds_ptr;
                    vf[c][i][h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(pf_s16x4_t*)at);
                }
        __builtin_amdgcn_sched_barrier(0);
        settle_matrix_ops();
        asm volatile("" : "+v"(s[0]), "+v"(s[1]));
        if constexpr (CAP) {   // softcap * tanh(x / softcap) * log2 e, tanh(y) = 1 - 2 / (1 + 2^(2 y log2 e)): off by some 2^-22 of the cap
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[t][r] = fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[t][r] * turn2)), cap2);
        }
        if constexpr (SINKS) {
            // A step seldom has both the end of what a row sees and the gap behind the sinks, and a register's position counted from the lane's first is a
            // constant of its comparison: 509 rows of 32 / 8 heads x 128 with a window of 1500 and one sink 41.4 us with all three bounds on every such
            // step, 37.9 so (34.5 without the sink; two chunks of 2048 rows without sinks take 1 % longer this way).
            if (kv0 + kTileStep > first_limit) {
                const int seen = (int)(q_limit - kv0 - 4u * kb);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (t * 32 + r % 4 + 8 * (r / 4) >= seen) s[t][r] = -INFINITY;
            }
            if (kv0 < last_low && kv0 + kTileStep > sinks) {
                const uint32_t at = kv0 + 4u * kb - sinks, hidden = q_low > sinks ? q_low - sinks : 0u;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (at + (uint32_t)(t * 32 + r % 4 + 8 * (r / 4)) < hidden) s[t][r] = -INFINITY;
            }
        } else if (kv0 + kTileStep > first_limit || kv0 < last_low) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t kv = kv0 + (uint32_t)(t * 32 + r % 4 + 8 * (r / 4)) + 4u * kb;
                    if (kv >= q_limit || kv < q_low) s[t][r] = -INFINITY;
                }
        }
        // the softmax reference moves only when a step's maximum outgrows it by 2^8
        float mt = s[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) mt = fmaxf(mt, s[i / 16][i % 16]);
        mt = other_half_max(mt) * scale2;
        const bool grow = mt > m_run + kPagedLag;
        const float m_new = grow ? mt : m_run, m_ref = m_new == -INFINITY ? 0.f : m_new, m_sub = m_ref + kPagedLag;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_ref) : 1.0f;
        m_run = m_new;
        l_run *= alpha;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
            settle_matrix_ops();
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                asm volatile("" : "+v"(oacc[i]));
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[i][r] *= alpha;
            }
        }
        // the second product of 16 positions, and between its matrix instructions the probabilities of the next 16
        pf_u32x4_t pb[4];
        auto probabilities = [&](auto c, auto w) __attribute__((always_inline)) {
            constexpr int at = c() * 8 + w() * 2;
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[at / 16][at % 16], scale2, -m_sub));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[at / 16][at % 16 + 1], scale2, -m_sub));
            l_run += p0 + p1;
            pb[c()][w()] = pack_bf16(p0, p1);
        };
        static_for<4>([&](auto w) __attribute__((always_inline)) { probabilities(std::integral_constant<int, 0>{}, w); });
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1");
        __builtin_amdgcn_s_setprio(1);   // (ahead of the other block's wave, whose softmax fits between: 446 -> 429 us of two chunks of 2048 rows)
        static_for<4>([&](auto c) __attribute__((always_inline)) {
            static_for<DT>([&](auto i) __attribute__((always_inline)) {
                const pf_u32x2_t lo = __builtin_bit_cast(pf_u32x2_t, vf[c()][i()][0]), hi = __builtin_bit_cast(pf_u32x2_t, vf[c()][i()][1]);
                mfma32_acc(oacc[i()], pf_u32x4_t{lo[0], lo[1], hi[0], hi[1]}, pb[c()]);
                if constexpr (c() < 3)
                    static_for<4 / DT>([&](auto w) __attribute__((always_inline)) {
                        probabilities(std::integral_constant<int, c() + 1>{}, std::integral_constant<int, i() * (4 / DT) + w()>{});
                    });
                __builtin_amdgcn_sched_barrier(0);
            });
            asm volatile("s_nop 1");
        });
        __builtin_amdgcn_s_setprio(0);
    }
    settle_matrix_ops();
#pragma unroll
    for (int i = 0; i < DT; ++i) asm volatile("" : "+v"(oacc[i]));
    barrier();
    if (bad && lane == 0) paged_fault(a.b, bad);

    // ---- what the tile hands on: through this wave's own LDS rows, so that the stores are whole 16-byte pieces ----
    l_run = both_halves_sum(l_run);
    constexpr uint32_t OS = D + 4;
    float* const all = reinterpret_cast<float*>(lds_raw);
    float* const ob = all + wave * 32u * OS;
    const bool whole = n_active == 1u;   // (tiles of 64 columns are never cut)
    const float f = whole && SPLIT == 1 ? paged_inverse(l_run, q_limit) : 1.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(ob + nl * OS + (uint32_t)(i * 32 + 8 * g) + 4u * kb) =
                make_float4(oacc[i][4 * g + 0] * f, oacc[i][4 * g + 1] * f, oacc[i][4 * g + 2] * f, oacc[i][4 * g + 3] * f);
    if constexpr (SPLIT == 1) {
        wave_lds_order();
        if (whole) paged_store_columns<D, SINKS>(a, it, ob, e0, live, lane);
        else paged_store_part<D>(a, it, ob, wave * 32u, live, m_run, l_run, lane);
    } else {   // the two waves of a column tile join their halves, 16 columns each
        float* const ml = all + 4u * 32u * OS;   // [wave][column] reference, sum
        if (kb == 0) *reinterpret_cast<float2*>(ml + (wave * 32u + nl) * 2u) = make_float2(m_run, l_run);
        __syncthreads();
        const uint32_t c0 = my_half * 16u, mine = live > c0 ? (live - c0 < 16u ? live - c0 : 16u) : 0u;
        const float* const other = all + (wave ^ 2u) * 32u * OS;
        for (uint32_t idx = lane; idx < 16u * (D / 4u); idx += 64u) {
            const uint32_t c = c0 + idx / (D / 4u), d = idx % (D / 4u) * 4u;
            const float2 x = *reinterpret_cast<const float2*>(ml + (wave * 32u + c) * 2u), y = *reinterpret_cast<const float2*>(ml + ((wave ^ 2u) * 32u + c) * 2u);
            const float m = fmaxf(x.x, y.x), ref = m == -INFINITY ? 0.f : m;
            float w0 = __builtin_amdgcn_exp2f(x.x - ref), w1 = __builtin_amdgcn_exp2f(y.x - ref);
            const float r = paged_inverse(fmaf(x.y, w0, y.y * w1), limit_of((e0 + c) / G));
            w0 *= r;
            w1 *= r;
            const float4 u = *reinterpret_cast<const float4*>(ob + c * OS + d), v = *reinterpret_cast<const float4*>(other + c * OS + d);
            *reinterpret_cast<float4*>(ob + c * OS + d) = make_float4(fmaf(u.x, w0, v.x * w1), fmaf(u.y, w0, v.y * w1), fmaf(u.z, w0, v.z * w1), fmaf(u.w, w0, v.w * w1));
        }
        wave_lds_order();
        paged_store_columns<D, SINKS>(a, it, ob + c0 * OS, e0 + c0, mine, lane);
    }
}

// A wave's merge of the columns c0, c0 + step, ... below `end` from the parts of n items (64 at most) that lie `stride` slots apart: GROUP parts of each of
// T columns are requested together.  put(c, d, four sums, the sum of the probabilities) by the lanes that hold them; done(c) by all lanes.
template <int D, int CACHE, uint32_t GROUP, uint32_t T, typename Put, typename Done>
__device__ __forceinline__ void paged_merge_columns(const __amdgpu_buffer_rsrc_t& mem, uint32_t base, uint32_t stride, uint32_t slot_bytes, uint32_t ml_at, uint32_t c0,
                                                    uint32_t end, uint32_t step, uint32_t n, uint32_t lane, Put&& put, Done&& done) {
    constexpr uint32_t LP = D / 4u, SPR = 64u / LP, N = GROUP / SPR;   // lanes of a part, parts of a request, requests of a column
    for (uint32_t c = c0; c < end; c += T * step) {
        pf_u32x2_t ml[T];
        pf_u32x4_t u[T][N];
        auto request = [&](uint32_t from) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t t = 0; t < T; ++t) {
                const uint32_t ct = c + t * step < end ? c + t * step : c;
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    const uint32_t k = from + i * SPR + lane / LP;
                    u[t][i] = __builtin_bit_cast(pf_u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(mem, (int)((base + (k < n ? k : 0u) * stride) * slot_bytes + (ct * D + (lane % LP) * 4u) * 4u), 0, CACHE));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (uint32_t t = 0; t < T; ++t) {
            const uint32_t ct = c + t * step < end ? c + t * step : c;
            ml[t] = __builtin_bit_cast(pf_u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(mem, (int)((base + (lane < n ? lane : 0u) * stride) * slot_bytes + ml_at + ct * 8u), 0, CACHE));
        }
        request(0);
        float w_mine[T], l[T], o[T][4];
#pragma unroll
        for (uint32_t t = 0; t < T; ++t) {
            const float m = lane < n ? __uint_as_float(ml[t][0]) : -INFINITY, M = wave_max(m);
            w_mine[t] = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
            l[t] = wave_sum(lane < n ? __uint_as_float(ml[t][1]) * w_mine[t] : 0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][r] = 0.f;
        }
        for (uint32_t from = 0;;) {
#pragma unroll
            for (uint32_t t = 0; t < T; ++t)
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    const uint32_t k = from + i * SPR + lane / LP;
                    const float w = __int_as_float(__builtin_amdgcn_ds_bpermute((int)(k * 4u), __float_as_int(w_mine[t])));
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[t][r] = k < n ? fmaf(__uint_as_float(u[t][i][r]), w, o[t][r]) : o[t][r];
                }
            if ((from += GROUP) >= n) break;
            request(from);
        }
#pragma unroll
        for (uint32_t t = 0; t < T; ++t) {
            if (c + t * step >= end) break;
#pragma unroll
            for (int r = 0; r < 4; ++r) {   // the parts that a request brought side by side
                const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[t][r]), __float_as_uint(o[t][r]), false, false);
                o[t][r] = __uint_as_float(h[0]) + __uint_as_float(h[1]);
                if constexpr (SPR == 4) {
                    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(o[t][r]), __float_as_uint(o[t][r]), false, false);
                    o[t][r] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
                }
            }
            if (lane < LP) put(c + t * step, lane * 4u, make_float4(o[t][0], o[t][1], o[t][2], o[t][3]), l[t]);
            done(c + t * step);
        }
    }
}

// The parts of cut tiles of 128 columns joined, in a launch of its own: a block takes 16 columns of a tile, a wave one at a time.  (By the tile's last
// item, as single tokens are, one CU reads all parts, 66 KB each: a chunk of 64 rows behind 8000 positions, 16 parts a tile, 45 us.)
constexpr uint32_t kMergeCols = 16;
template <int D, bool SINKS>
__global__ __launch_bounds__(256) void sdpa_paged_merge_kernel(const SdpaPagedArgs a) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedItem it = paged_item<false, kTileCols, SINKS, true>(a, blockIdx.x / (kTileCols / kMergeCols), lane);
    if (!it.any) return;
    const uint32_t G = a.group, columns = it.s.rows * G, e_tile = it.tile * kTileCols, c0 = blockIdx.x % (kTileCols / kMergeCols) * kMergeCols;
    if (columns <= kFewMost || e_tile + c0 >= columns) return;
    const PagedRange range = paged_range<kTileStep, SINKS>(a, it, e_tile, columns - e_tile < kTileCols ? columns - 1u : e_tile + kTileCols - 1u);
    if (range.n_active == 1u) return;
    constexpr uint32_t SLOT = kTileCols * (D + 2u) * 4u;
    const __amdgpu_buffer_rsrc_t mem = __builtin_amdgcn_make_buffer_rsrc(a.partials, 0, (int)(a.slots * SLOT), 0x27000);
    const uint32_t left = columns - e_tile, end = left < c0 + kMergeCols ? left : c0 + kMergeCols;
    bool odd = false;
    auto put = [&](uint32_t c, uint32_t d, const float4& o, float l) {
        const float t = (__builtin_fabsf(o.x) + __builtin_fabsf(o.y)) + (__builtin_fabsf(o.z) + __builtin_fabsf(o.w));
        const uint32_t e = e_tile + c, place = e / G;
        const float f = paged_inverse(l, paged_limit(it.s, place));
        *reinterpret_cast<uint2*>(a.out + (size_t)(it.s.row0 + place) * a.out_stride + (size_t)(it.kvh * G + (e - place * G)) * D + d) =
            make_uint2(pack_bf16(o.x * f, o.y * f), pack_bf16(o.z * f, o.w * f));
        odd = !(t * f < INFINITY);
    };
    auto done = [&](uint32_t c) {
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0)) {
            const uint32_t e = e_tile + c, place = e / G;
            paged_row<D, SINKS>(a, it.seq, it.s, place, it.kvh * G + (e - place * G), lane);
            odd = false;
        }
    };
    if (range.n_active <= 8u) paged_merge_columns<D, 0, 8, 2>(mem, it.base, a.b.n_kv, SLOT, kTileCols * D * 4u, c0 + wave, end, 4u, range.n_active, lane, put, done);
    else paged_merge_columns<D, 0, 16, 1>(mem, it.base, a.b.n_kv, SLOT, kTileCols * D * 4u, c0 + wave, end, 4u, range.n_active, lane, put, done);
}

// ---- single tokens: at most 16 columns of a sequence and KV head ----
// The products are those of the decode attention over a contiguous cache (sdpa_mma.hip: 16x16x32, K rows and V^T as the first operand, the queries as
// columns), a probability as the sum of two bf16 values, hi + lo, which leaves 2^-17 of it: of up to 8 columns in the columns 8 on, of more in an
// instruction of its own.  A wave owns its steps of 32 positions and their place in LDS: it waits for no other wave until the block's waves
// meet, its keys are requested again as soon as they are in registers, its values behind the second product.  Two blocks a CU keep 128 KB in
// flight.  Bound by the bytes: 64 tokens over 620 MB of keys and values 119 us, 5.2 TB/s (a copy on the card reaches 4.75 read and written).  One token
// over 613 positions, 14 / 2 heads x 64: 7 us, which is what finding the item, one round and the merge take after one another.
constexpr uint32_t few_lds_bytes(uint32_t d) {
    const uint32_t stages = 4u * kFewStep * d * 4u, meet = 4u * kFewCols * (d + 4u) * 4u + 2u * 4u * kFewCols * 4u;
    return (stages > meet ? stages : meet) + 16u;   // and two words for the block
}

template <int D, bool CAP, bool WIDE, bool SINKS>
__device__ __forceinline__ void paged_few(const SdpaPagedArgs& a, const PagedItem& it, uint32_t lane) {
    constexpr uint32_t ROW = D * 2u, P = D / 8u, KT = kFewStep * ROW, STAGE = 2u * KT, RPI = 1024u / ROW;   // pieces of a row; rows of a request
    constexpr int REQ = (int)(KT / 1024u), KS = D / 32, DT = D / 16, PARTS = WIDE ? 2 : 1;
    constexpr uint32_t QT = WIDE ? 16u : 8u;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    extern __shared__ uint4 lds_raw[];
    unsigned char* const lds = reinterpret_cast<unsigned char*>(lds_raw);

    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t G = a.group, e0 = it.tile * kFewCols, left_cols = it.s.rows * G - e0, columns = left_cols < kFewCols ? left_cols : kFewCols;   // of this tile
    auto limit_of = [&](uint32_t place) { return paged_limit(it.s, place); };
    auto low_of = [&](uint32_t limit) { return a.window && limit > a.window ? limit - a.window : 0u; };
    const PagedRange range = paged_range<kFewRound, SINKS>(a, it, e0, e0 + columns - 1u);
    const uint32_t kv_end = range.kv_end, n_active = range.n_active, lim_lo = __builtin_amdgcn_readfirstlane(limit_of(e0 / G));
    const uint32_t low_hi = __builtin_amdgcn_readfirstlane(low_of(kv_end));
    if (it.split >= n_active) return;
    const uint32_t round0 = it.split * range.per;
    uint32_t rounds = range.steps < round0 + range.per ? range.steps - round0 : range.per;   // of this item
    // (of the sinks' last round a wave whose positions lie behind them sees nothing, and leaves it out)
    const uint32_t sinks = paged_sinks<SINKS>(a), near_wave = sinks > wave * kFewStep ? (sinks - wave * kFewStep + kFewRound - 1u) / kFewRound : 0u;
    const bool leaves = near_wave < range.near && near_wave >= round0 && near_wave - round0 < rounds;
    rounds -= leaves ? 1u : 0u;
    auto at_round = [&](uint32_t j) {
        const uint32_t n = round0 + j;
        return range.step(n + (leaves && n >= near_wave ? 1u : 0u)) * kFewRound + wave * kFewStep;
    };
    // (a wave's place in the last round may lie behind the context)
    const uint32_t n_steps = __builtin_amdgcn_readfirstlane(rounds ? rounds - (at_round(rounds - 1u) >= kv_end ? 1u : 0u) : 0u);

    const uint32_t mine = n % QT < columns ? n % QT : columns - 1u;   // (columns past the last repeat it and store nothing)
    const uint32_t place = (e0 + mine) / G, q_limit = limit_of(place), q_low = low_of(q_limit);
    pf_bf16x8_t qf[KS];
    {
        const uint16_t* qr = a.q + (size_t)(it.s.row0 + place) * a.q_stride + (size_t)(it.kvh * G + (e0 + mine - place * G)) * D + g * 8u;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const pf_bf16x8_t*>(qr + s * 32);
    }

    auto k_swizzle = [](uint32_t row) { return P == 16u ? row & 15u : (row >> 1) & 7u; };
    auto v_swizzle = [](uint32_t row) { return P == 16u ? (row & 7u) << 1 : ((row >> 1) & 3u) << 1; };
    const uint32_t irow = lane / P, at_piece = lane % P, my_stage = wave * STAGE;
    const uint32_t shift = a.b.page_shift, in_page = (1u << shift) - 1u;
    typedef const uint32_t __attribute__((address_space(4)))* scalar_ptr;
    const uintptr_t table = (uintptr_t)(a.b.table + (size_t)__builtin_amdgcn_readfirstlane(it.seq) * a.b.table_stride);
    uint32_t bad = 0;
    // a step's 32 positions lie in one page or two: 16 rows of each half in one
    auto page_of = [&](uint32_t pos) {
        const uint32_t at = pos < kv_end ? pos : kv_end - 1u;
        return *(scalar_ptr)(table + (size_t)(at >> shift) * 4u);
    };
    auto issue = [&](const uint16_t* pages, uint32_t to, uint32_t kv0, const uint32_t (&page)[2], auto swizzle) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t id = page[h];
            if (id >= a.b.n_pages) {
                id = 0;
                bad = FK_PAGED_BAD_PAGE;
            }
            const uint32_t span = kv0 + 16u * h, at = span < kv_end ? span : kv_end - 1u, left = kv_end - 1u - at;
            const unsigned char* base = reinterpret_cast<const unsigned char*>(pages) +
                                        (((size_t)id * a.b.n_kv + it.kvh) * (in_page + 1u) + (at & in_page)) * ROW;
#pragma unroll
            for (int i = 0; i < REQ / 2; ++i) {
                const uint32_t r = (uint32_t)i * RPI + irow, from = r < left ? r : left;   // (past the context: its last row, masked)
                dma16(to + (uint32_t)(h * (REQ / 2) + i) * 1024u, from * ROW + ((at_piece ^ swizzle(16u * h + r)) * 16u), base);
            }
        }
    };
    auto issue_k = [&](uint32_t kv0, const uint32_t (&page)[2]) { issue(a.k, my_stage, kv0, page, k_swizzle); };
    auto issue_v = [&](uint32_t kv0, const uint32_t (&page)[2]) { issue(a.v, my_stage + KT, kv0, page, v_swizzle); };

    f32x4_t acc[PARTS][DT];
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[p][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    const float scale2 = CAP ? 1.0f : a.scale * kLog2E;
    const float cap2 = a.softcap * kLog2E, turn2 = CAP ? 2.0f * a.scale * kLog2E / a.softcap : 0.f;

    uint32_t page[2] = {0, 0};
    if (n_steps) {
        const uint32_t first = at_round(0), second = at_round(1);
        page[0] = page_of(first);
        page[1] = page_of(first + 16u);
        issue_k(first, page);
        issue_v(first, page);
        if (n_steps > 1u) {
            page[0] = page_of(second);
            page[1] = page_of(second + 16u);
        }
    }
#pragma unroll 1
    for (uint32_t j = 0; j < n_steps; ++j) {
        const uint32_t kv0 = at_round(j), kv1 = at_round(j + 1u);
        unsigned char* const ks = lds + my_stage;
        unsigned char* const vs = ks + KT;
        const bool more = j + 1u < n_steps;
        wait_loads<REQ>();   // the keys; the values may be on their way
        pf_bf16x8_t kf[2][KS];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint32_t row = (uint32_t)t * 16u + n;
                kf[t][s] = *reinterpret_cast<const pf_bf16x8_t*>(ks + row * ROW + ((((uint32_t)s * 4u + g) ^ k_swizzle(row)) * 16u));
            }
        // (two chains a score beyond 64 dims: in one, each instruction's rounding is that of the whole sum so far)
        float x[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            constexpr int HALF = KS >= 4 ? KS / 2 : KS;
            f32x4_t s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < HALF; ++s) s4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][s], qf[s], s4, 0, 0, 0);
            if constexpr (HALF < KS) {
                f32x4_t s5 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = HALF; s < KS; ++s) s5 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][s], qf[s], s5, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s4[i] += s5[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t * 4 + i] = s4[i];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) issue_k(kv1, page);   // the keys are in registers: their place takes the next step's
        if constexpr (CAP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i] * turn2)), cap2);
        }
        if (kv0 + kFewStep > lim_lo || (kv0 < low_hi && kv0 + kFewStep > sinks)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t kv = kv0 + (uint32_t)(i / 4) * 16u + 4u * g + (uint32_t)(i % 4);
                if (kv >= q_limit || (kv < q_low && kv >= sinks)) x[i] = -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
        mx *= scale2;
        if (__builtin_amdgcn_ballot_w64(mx > m_run + kPagedLag) != 0) {   // rare after the first steps
            mx = rows_max(mx);
            const bool grow = mx > m_run + kPagedLag;
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - mx) : 1.0f;
            m_run = grow ? mx : m_run;
            l_run *= alpha;
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int i = 0; i < DT; ++i) acc[p][i] *= alpha;
        }
        const float m_sub = (m_run == -INFINITY ? 0.f : m_run) + kPagedLag;
        pf_u32x4_t pb[PARTS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p0 = __builtin_amdgcn_exp2f(fmaf(x[2 * i], scale2, -m_sub)), p1 = __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], scale2, -m_sub));
            l_run += p0 + p1;
            const uint32_t hi = pack_bf16(p0, p1), lo = pack_bf16(p0 - bf16_lo(hi), p1 - bf16_hi(hi));
            if constexpr (WIDE) {
                pb[0][i] = hi;
                pb[PARTS - 1][i] = lo;
            } else {
                pb[0][i] = n < 8u ? hi : lo;
            }
        }
        if (more) wait_loads<REQ>();   // the values; the next keys may be on their way
        else wait_loads<0>();
        pf_bf16x8_t vf[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            s16x4 v4[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t row = (uint32_t)h * 16u + 4u * g + (n >> 2), piece = (uint32_t)(2 * i) + ((n & 3u) >> 1);
                unsigned char* at = vs + row * ROW + ((piece ^ v_swizzle(row)) * 16u) + (n & 1u) * 8u;
                typedef __attribute__((address_space(3))) s16x4* lds_ptr;
                v4[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(s16x4*)at);
            }
            vf[i] = __builtin_bit_cast(pf_bf16x8_t, __builtin_shufflevector(v4[0], v4[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[p][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], __builtin_bit_cast(pf_bf16x8_t, pb[p]), acc[p][i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            issue_v(kv1, page);
            if (j + 2u < n_steps) {
                const uint32_t kv2 = at_round(j + 2u);
                page[0] = page_of(kv2);
                page[1] = page_of(kv2 + 16u);
            }
        }
    }
    if (bad && lane == 0) paged_fault(a.b, bad);

    // ---- the waves meet ----
    const float l_all = [&] {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
        const float v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
        const auto f = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(f[0]) + __uint_as_float(f[1]);
    }();
    __syncthreads();
    constexpr uint32_t OS = D + 4u;
    float* const red = reinterpret_cast<float*>(lds);                   // [wave][column][OS]
    float* const wm = red + 4u * kFewCols * OS;                         // [wave][column] references, sums
    float* const wl = wm + 4u * kFewCols;
    volatile uint32_t* const word = reinterpret_cast<volatile uint32_t*>(lds + few_lds_bytes(D) - 16u);
    if (tid == 0) word[1] = 0;
    if (g == 0) {
        wm[wave * kFewCols + n] = m_run;
        wl[wave * kFewCols + n] = l_all;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        f32x4_t o;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            o[r] = WIDE ? acc[0][i][r] + acc[PARTS - 1][i][r]
                        : acc[0][i][r] + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(acc[0][i][r]), 0x108, 0xF, 0xF, true));   // the columns 8 on
        if (n < QT) *reinterpret_cast<float4*>(red + (wave * kFewCols + n) * OS + (uint32_t)i * 16u + 4u * g) = make_float4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
    const bool whole = n_active == 1u;
    const __amdgpu_buffer_rsrc_t mem = __builtin_amdgcn_make_buffer_rsrc(a.partials, 0, (int)(a.slots * a.slot_bytes), 0x27000);
    auto store = [&](uint32_t c, uint32_t d, const float4& o, float l) {
        const float t = (__builtin_fabsf(o.x) + __builtin_fabsf(o.y)) + (__builtin_fabsf(o.z) + __builtin_fabsf(o.w));
        const uint32_t pl = (e0 + c) / G;
        const float f = paged_inverse(l, limit_of(pl));
        *reinterpret_cast<uint2*>(a.out + (size_t)(it.s.row0 + pl) * a.out_stride + (size_t)(it.kvh * G + (e0 + c - pl * G)) * D + d) =
            make_uint2(pack_bf16(o.x * f, o.y * f), pack_bf16(o.z * f, o.w * f));
        if (!(t * f < INFINITY)) atomicOr(const_cast<uint32_t*>(&word[1]), 1u << c);
    };
    for (uint32_t i = tid; i < columns * (D / 4u); i += 256u) {
        const uint32_t c = i / (D / 4u), d = (i % (D / 4u)) * 4u;
        float M = wm[c];
#pragma unroll
        for (uint32_t w = 1; w < 4; ++w) M = fmaxf(M, wm[w * kFewCols + c]);
        const float ref = M == -INFINITY ? 0.f : M;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(wm[w * kFewCols + c] - ref);
            const float4 p = *reinterpret_cast<const float4*>(red + (w * kFewCols + c) * OS + d);
            l = fmaf(wl[w * kFewCols + c], f, l);
            o = make_float4(fmaf(p.x, f, o.x), fmaf(p.y, f, o.y), fmaf(p.z, f, o.z), fmaf(p.w, f, o.w));
        }
        if (whole) {
            store(c, d, o, l);
        } else {
            const uint32_t at = it.slot * a.slot_bytes;
            const pf_u32x4_t v = {__float_as_uint(o.x), __float_as_uint(o.y), __float_as_uint(o.z), __float_as_uint(o.w)};
            __builtin_amdgcn_raw_buffer_store_b128(v, mem, (int)(at + (c * D + d) * 4u), 0, kPastCaches);
            if (d == 0) {
                const pf_u32x2_t ml = {__float_as_uint(M), __float_as_uint(l)};
                __builtin_amdgcn_raw_buffer_store_b64(ml, mem, (int)(at + (kFewCols * D + c * 2u) * 4u), 0, kPastCaches);
            }
        }
    }
    if (!whole) {   // the item that arrives last merges the sequence's, in their order
        const uint32_t stride = a.b.n_kv, base = it.base;
        wait_memory_ops_done();
        __syncthreads();
        if (tid == 0) word[0] = atomicAdd(&a.counters[base], 1u) == n_active - 1u ? 1u : 0u;
        __syncthreads();
        if (!word[0]) return;
        if (tid == 0) __hip_atomic_store(&a.counters[base], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        auto none = [](uint32_t) {};
        if (n_active <= 8u) paged_merge_columns<D, kPastCaches, 8, 4>(mem, base, stride, a.slot_bytes, kFewCols * D * 4u, wave, columns, 4u, n_active, lane, store, none);
        else paged_merge_columns<D, kPastCaches, 32, 1>(mem, base, stride, a.slot_bytes, kFewCols * D * 4u, wave, columns, 4u, n_active, lane, store, none);
    }
    __syncthreads();
    for (uint32_t again = word[1], c = 0; again; again >>= 1, ++c)
        if ((again & 1u) && c % 4u == wave) paged_row<D, SINKS>(a, it.seq, it.s, (e0 + c) / G, it.kvh * G + (e0 + c) % G, lane);
}

// Chunks and single tokens together: each sequence by its kind, in one launch, so that what is bound by the matrix units runs beside what is bound by the
// bytes.
template <int D, bool CAP, uint32_t SPLIT, bool SINKS>
__global__ __launch_bounds__(256, 2) void sdpa_paged_kernel(const SdpaPagedArgs a) {
    const uint32_t lane = threadIdx.x & 63u;
    const PagedItem it = paged_item<false, kTileCols / SPLIT, SINKS>(a, blockIdx.x, lane);
    if (!it.any) return;
    if (it.s.rows * a.group <= kFewMost) paged_few<D, CAP, true, SINKS>(a, it, lane);
    else paged_tile<D, CAP, SPLIT, SINKS>(a, it, lane);
}
template <int D, bool CAP, bool WIDE, bool SINKS>
__global__ __launch_bounds__(256, 2) void sdpa_paged_few_kernel(const SdpaPagedArgs a) {
    const uint32_t lane = threadIdx.x & 63u;
    const PagedItem it = paged_item<true, kFewCols, SINKS>(a, blockIdx.x, lane);
    if (it.any) paged_few<D, CAP, WIDE, SINKS>(a, it, lane);
}

namespace {

static_assert(16384u + 896u * kTileCols * (128u + 2u) * 4u <= FK_SDPA_PAGED_WORKSPACE_MOST && 16384u + 2048u * kFewCols * (128u + 2u) * 4u <= FK_SDPA_PAGED_WORKSPACE_MOST);

// How a launch is cut: fewer tiles than `target` are cut along their positions, into items of `min_steps` steps at least.
struct PagedPlan {
    bool few;          // single tokens: 16 columns a sequence and KV head at most
    bool compact;      // more tiles than slots
    uint32_t target, min_steps, slots, few_slots;
    uint64_t tiles;    // of all sequences and KV heads, at most
    size_t slot_bytes, bytes;
};
constexpr uint32_t kFewLeast = 16, kFewTarget = 512;   // steps of 64 positions of a token's item among whole chunks; items
constexpr size_t kPagedCounterBytes = 16384;   // a word for a slot
PagedPlan paged_plan(bool few, uint32_t n_heads, uint32_t n_kv, uint32_t head_dim, uint32_t n_seqs, uint32_t rows) {
    PagedPlan p;
    const uint32_t cols = few ? kFewCols : kTileCols;
    p.few = few;
    // (tiles: as many as stand on the card at once, two of 128 dims a CU, three of 64.  Of 64 dims, 32 / 4 heads, 1170 rows behind some 9000 positions 156 us with 768,
    // 205 with 512, 171 with 1024.)
    p.target = few || head_dim == 64 ? 768 : 512;
    p.min_steps = few ? 1 : 4;
    // (a sequence of up to kFewMost columns has tiles of 16 also among chunks)
    const uint64_t columns = (uint64_t)rows * (n_heads / n_kv);
    p.tiles = few ? (columns / kFewCols + n_seqs) * n_kv : (columns / kTileCols + (uint64_t)n_seqs * (kFewMost / kFewCols)) * n_kv;
    p.slot_bytes = (size_t)cols * (head_dim + 2) * 4;
    // (more tiles are not cut: of 64 dims 600 of 2400 rows behind few positions 90 us, cut 99)
    const uint32_t most_tiles = few ? 1024 : 448, most = few ? 2048 : head_dim == 64 ? 1216 : 896;   // slots: FK_SDPA_PAGED_WORKSPACE_MOST at the most
    p.compact = p.tiles > most_tiles;
    p.slots = !p.compact ? std::min((uint32_t)p.tiles + p.target, most) : few ? 2 * p.target + 64 : 0;   // (rounding leaves an item more for every tile)
    p.target = p.compact ? p.target : p.slots - (uint32_t)p.tiles;
    p.few_slots = !few && p.compact ? 2 * kFewTarget + 64 : 0;   // tiles of 128 that are too many to cut: the single tokens among them, which need not be short
    p.bytes = kPagedCounterBytes + (p.few_slots ? p.few_slots * (size_t)kFewCols * (head_dim + 2) * 4 : p.slots * p.slot_bytes);
    return p;
}

}  // namespace

fk_status sdpa_paged_workspace_bytes(uint32_t n_heads, uint32_t n_kv, uint32_t head_dim, uint32_t n_seqs, uint32_t rows, uint32_t max_len,
                                     size_t* bytes) {
    if (!bytes) return set_error(FK_ERR_INVALID, "sdpa_paged workspace: null pointer");
    if (n_heads == 0 || n_kv == 0 || n_heads % n_kv || n_seqs == 0 || rows == 0 || max_len == 0)
        return set_error(FK_ERR_INVALID, "sdpa_paged workspace: empty shape, or n_heads not a multiple of n_kv");
    if (head_dim != 64 && head_dim != 128) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged workspace: head dimension 64 or 128");
    const size_t few = paged_plan(true, n_heads, n_kv, head_dim, n_seqs, rows).bytes, tiles = paged_plan(false, n_heads, n_kv, head_dim, n_seqs, rows).bytes;
    *bytes = few > tiles ? few : tiles;
    return FK_OK;
}

fk_status plan_sdpa_paged(const uint16_t* q, uint32_t q_stride, uint16_t* out, uint32_t out_stride, uint32_t n_heads, float scale, float softcap,
                          uint32_t window, uint32_t sinks, const fk_paged_batch* batch, const fk_page_pool* pool, void* workspace, size_t workspace_bytes,
                          Launch* l) {
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
    if (!(scale * kLog2E < 3e38f)) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: scale too large");
    if (!(softcap >= 0.f) || !std::isfinite(softcap)) return set_error(FK_ERR_INVALID, "sdpa_paged: softcap must not be negative");
    // (the kernels' tanh is off by 2^-23 of the cap, which is what a probability's exponent is then off by)
    if (softcap > 1024.f || (softcap > 0.f && !std::isfinite(2.0f * scale * kLog2E / softcap)))
        return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: softcap up to 1024, and not so small that scale / softcap overflows (0: none)");
    if (rows_overlap(q, q_stride, (size_t)n_heads * D, out, out_stride, (size_t)n_heads * D, batch->rows))
        return set_error(FK_ERR_INVALID, "sdpa_paged: out overlaps q");
    if ((uint64_t)batch->max_rows * (n_heads / n_kv) > 0x7fffffffull) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: too many rows of a sequence");
    size_t need = 0;
    FK_TRY(sdpa_paged_workspace_bytes(n_heads, n_kv, D, batch->n_seqs, batch->rows, batch->max_len, &need));
    if (workspace_bytes < need) return set_error(FK_ERR_INVALID, "sdpa_paged: workspace too small");
    const PagedPlan p = paged_plan(batch->max_rows * (n_heads / n_kv) <= kFewMost, n_heads, n_kv, D, batch->n_seqs, batch->rows);
    if (p.tiles + p.target > 0x7fffffffull) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: too many rows");
    const DeviceFacts* dev;
    FK_TRY(device_facts(&dev));
    a.q = q; a.k = pool->k; a.v = pool->v; a.out = out;
    a.q_stride = q_stride; a.out_stride = out_stride; a.group = n_heads / n_kv;
    // (without a window everything is seen, and sinks beyond the longest sequence are as many)
    a.sinks = window ? std::min(sinks, batch->max_len) : 0;
    a.window = window; a.scale = scale; a.softcap = softcap;
    a.counters = static_cast<uint32_t*>(workspace);
    a.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kPagedCounterBytes);
    a.slots = p.slots; a.target = p.target; a.min_steps = p.min_steps;
    // [sinks][D == 128][softcap][split or wide]
    const void* tile[2][2][2][2] = {
        {{{reinterpret_cast<const void*>(&sdpa_paged_kernel<64, false, 1, false>), reinterpret_cast<const void*>(&sdpa_paged_kernel<64, false, 2, false>)},
          {reinterpret_cast<const void*>(&sdpa_paged_kernel<64, true, 1, false>), reinterpret_cast<const void*>(&sdpa_paged_kernel<64, true, 2, false>)}},
         {{reinterpret_cast<const void*>(&sdpa_paged_kernel<128, false, 1, false>), reinterpret_cast<const void*>(&sdpa_paged_kernel<128, false, 2, false>)},
          {reinterpret_cast<const void*>(&sdpa_paged_kernel<128, true, 1, false>), reinterpret_cast<const void*>(&sdpa_paged_kernel<128, true, 2, false>)}}},
        {{{reinterpret_cast<const void*>(&sdpa_paged_kernel<64, false, 1, true>), reinterpret_cast<const void*>(&sdpa_paged_kernel<64, false, 2, true>)},
          {reinterpret_cast<const void*>(&sdpa_paged_kernel<64, true, 1, true>), reinterpret_cast<const void*>(&sdpa_paged_kernel<64, true, 2, true>)}},
         {{reinterpret_cast<const void*>(&sdpa_paged_kernel<128, false, 1, true>), reinterpret_cast<const void*>(&sdpa_paged_kernel<128, false, 2, true>)},
          {reinterpret_cast<const void*>(&sdpa_paged_kernel<128, true, 1, true>), reinterpret_cast<const void*>(&sdpa_paged_kernel<128, true, 2, true>)}}}};
    const void* few[2][2][2][2] = {
        {{{reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, false, false, false>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, false, true, false>)},
          {reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, true, false, false>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, true, true, false>)}},
         {{reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, false, false, false>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, false, true, false>)},
          {reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, true, false, false>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, true, true, false>)}}},
        {{{reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, false, false, true>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, false, true, true>)},
          {reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, true, false, true>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<64, true, true, true>)}},
         {{reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, false, false, true>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, false, true, true>)},
          {reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, true, false, true>), reinterpret_cast<const void*>(&sdpa_paged_few_kernel<128, true, true, true>)}}}};
    // Positions that a tile can see, in steps.  Chunks of up to 8 steps are not cut: the merge costs what it saves (a prompt of 512 rows, 32 / 8 heads x
    // 128: 18 us whole, 24 in halves).
    const uint32_t step = p.few ? kFewRound : kTileStep, span = (p.few ? kFewCols : kTileCols) / a.group + 2u;
    const uint64_t seen = window ? std::min<uint64_t>(batch->max_len, (uint64_t)window + a.sinks + std::min(batch->max_rows, span) + (a.sinks ? 2u : 1u) * step) : batch->max_len;
    const uint32_t most = (uint32_t)((seen + step - 1u) / step), splits = (most + p.min_steps - 1u) / p.min_steps;
    // Tiles of 64 columns and twice the positions a step where each has a CU to itself: a lone block's step takes 1.3 to 1.5 us, most of it waits that do not
    // depend on what it holds, and half as many are left.  32 / 8 heads x 128, us in whole or cut tiles of 128 and in these: a fresh prompt of 512 rows 17.2,
    // 14.5; of 256 11.6, 11.0; of 200 10.7, 11.0; 512 rows behind 1000 positions 31.8, 28.2; behind 1300 33.7, 32.1; behind 3000 45.8, 54; 384 behind 1100 27.7,
    // 26.3; 256 behind 1000 24.0, 23.7; 128 behind 512 19.8, 15.7; behind 1000 21.2, 21.4; 64 behind 512 18.0, 15.4; behind 1000 19.1, 21.4.
    // (at most so many tiles: a sequence of few columns has two, of more one beyond what all together fill)
    const uint64_t filled = ((uint64_t)batch->rows * a.group + kTileCols / 2 - 1) / (kTileCols / 2), halves = (std::max<uint64_t>(filled, 2) + 2 * (uint64_t)(batch->n_seqs - 1)) * n_kv;
    const bool split = !p.few && halves <= (uint64_t)dev->cus && most > 4u && most <= 12u + halves / 12u;
    // (more single tokens than have slots: a block for each that may be cut off takes what it takes to find none, up to a tenth of 256 tokens over 500
    // positions; over more than 8 rounds nothing that shows, and of 255 over 500 and one over 60 000 156 us for 688)
    const bool cut = !split && p.slots && (p.few && !p.compact ? splits > 1u : most > 8u);
    a.slot_bytes = (uint32_t)p.slot_bytes;
    a.compact = cut && p.few && p.compact;
    a.only_few = !cut && !split && p.few_slots && most > 2u * kFewLeast;
    if (!cut) a.slots = 0;
    if (a.only_few) {
        a.slots = p.few_slots;
        a.slot_bytes = kFewCols * (D + 2u) * 4u;
        a.target = kFewTarget;
        a.min_steps = kFewLeast;
    }
    l->func = p.few ? few[a.sinks > 0][D == 128][softcap > 0.f][batch->max_rows * (n_heads / n_kv) > 8u] : tile[a.sinks > 0][D == 128][softcap > 0.f][split];
    // (no more blocks than there can be items: one that finds none costs what it takes to look)
    a.blocks = (uint32_t)(cut && !a.compact ? std::min<uint64_t>(p.slots, p.tiles * splits) : split ? halves : p.tiles + (cut || a.only_few ? a.target : 0u));
    l->grid = dim3(a.blocks, 1, 1);
    l->block = dim3(256, 1, 1);
    l->shmem = p.few ? few_lds_bytes(D) : std::max(tile_lds_bytes(D, split ? 2u : 1u), few_lds_bytes(D));
    if ((int)l->shmem > dev->max_dyn_lds) return set_error(FK_ERR_UNSUPPORTED, "sdpa_paged: LDS tile does not fit");
    FK_TRY(raise_dynamic_lds(l->func, l->shmem));
    l->set_args(a);
    if (!p.few && cut) {
        Launch m;
        if (a.sinks) m.func = D == 64 ? reinterpret_cast<const void*>(&sdpa_paged_merge_kernel<64, true>) : reinterpret_cast<const void*>(&sdpa_paged_merge_kernel<128, true>);
        else m.func = D == 64 ? reinterpret_cast<const void*>(&sdpa_paged_merge_kernel<64, false>) : reinterpret_cast<const void*>(&sdpa_paged_merge_kernel<128, false>);
        m.grid = dim3((uint32_t)p.tiles * (kTileCols / kMergeCols), 1, 1);
        m.block = dim3(256, 1, 1);
        m.set_args(a);
        l->then.push_back(m);
    }
    return FK_OK;
}

}  // namespace fk
