// Beam search: the selection of hypotheses and the reordering of their states.
#include <algorithm>
#include <cmath>
#include <numeric>
#include <vector>

#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kMostBeams = 64;

// A symbol of a row as one number: the larger logit first, of equals the lower
// symbol. 0 is none.
__device__ __forceinline__ uint64_t candidate(float z, uint32_t at) {
    return static_cast<uint64_t>(order_key(z + 0.0f)) << 32 | (0xffffffffu - at);
}
__device__ __forceinline__ float logit_of(uint64_t c) { return from_order_key(static_cast<uint32_t>(c >> 32)); }
__device__ __forceinline__ uint32_t symbol_of(uint64_t c) { return 0xffffffffu - static_cast<uint32_t>(c); }

__device__ __forceinline__ double wave_sum(double v) {
    const auto step = [&](auto ctrl, auto rows) {
        const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v));
        const auto moved = [&](uint32_t half) {
            return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(half), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
        };
        const uint64_t other = static_cast<uint64_t>(moved(static_cast<uint32_t>(bits >> 32))) << 32 | moved(static_cast<uint32_t>(bits));
        v += __longlong_as_double(static_cast<long long>(other));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // as wave_reduce does
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v));
    const auto last = [](uint32_t half) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(half), 63)); };
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(last(static_cast<uint32_t>(bits >> 32))) << 32 | last(static_cast<uint32_t>(bits))));
}

// The largest of v in each group of `lanes` neighbouring lanes (a power of two up to 16).
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t lanes) {
    const auto step = [&](auto ctrl) {
        v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, true)));
    };
    if (lanes >= 2) step(std::integral_constant<int, 0xb1>{});    // the neighbour in a pair
    if (lanes >= 4) step(std::integral_constant<int, 0x4e>{});    // the other pair of four
    if (lanes >= 8) step(std::integral_constant<int, 0x141>{});   // mirrored in eight
    if (lanes >= 16) step(std::integral_constant<int, 0x140>{});  // mirrored in sixteen
    return v;
}

// A value that is not above the kept-th largest of a wave's 64, and equals it in its
// upper 20 bits; 0 where fewer than `kept` are above 0.
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t v, uint32_t kept) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t higher = t | 1u << bit;
        if (__popcll(__ballot(v >= higher)) >= static_cast<int>(kept)) t = higher;
    }
    return t;
}

// The same over a workgroup of 1, 2, 4, 8 or 16 waves, whose lanes make 64 groups: so
// many different groups hold something as large that the value bounds the kept-th
// largest of all. Where much is kept, every thread is a group: the least of 64 groups'
// largest lets through five times what is kept, and 32 x 8 beams of 131,075 to 64 took
// 1.2 ms. `maxima`: a word of LDS for each thread, none where kWave.
constexpr uint32_t kFewKept = 16, kMostWaves = 16;
template <bool kWave>
__device__ __forceinline__ uint32_t bar_of(uint32_t largest, uint32_t kept, uint32_t* maxima) {
    const uint32_t lane = threadIdx.x % 64, waves = kWave ? 1 : blockDim.x / 64;
    if (waves == 1) return kth_of_wave(largest, kept);
    if (kept <= kFewKept) {
        const uint32_t m = group_max(largest, waves);
        if (lane % waves == 0) maxima[(threadIdx.x / 64 * 64 + lane) / waves] = m;
        __syncthreads();
        return kth_of_wave(maxima[lane], kept);
    }
    maxima[threadIdx.x] = largest;
    __syncthreads();
    uint32_t all[kMostWaves], t = 0;
#pragma unroll
    for (uint32_t w = 0; w < kMostWaves; ++w) all[w] = w < waves ? maxima[w * 64 + lane] : 0;
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t higher = t | 1u << bit;
        uint32_t count = 0;
#pragma unroll
        for (uint32_t w = 0; w < kMostWaves; ++w)
            if (w < waves) count += static_cast<uint32_t>(__popcll(__ballot(all[w] >= higher)));
        if (count >= kept) t = higher;
    }
    return t;
}

// Orders what one wave (kWave) or a workgroup wrote to LDS.
template <bool kWave>
__device__ __forceinline__ void settle_lds() {
    if constexpr (kWave) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else __syncthreads();
}

// The bits of a mask below this lane's.
__device__ __forceinline__ uint32_t below_in(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// A place behind what the wave's other lanes and the other waves take.
__device__ __forceinline__ uint32_t place_for(bool taken, uint32_t* count) {
    const uint64_t mask = __ballot(taken);
    uint32_t base = 0;
    if (threadIdx.x % 64 == 0) base = atomicAdd(count, static_cast<uint32_t>(__popcll(mask)));
    return __builtin_amdgcn_readfirstlane(base) + below_in(mask);
}

// 1,024 neighbouring symbols of a row in the registers of a wave, 16 a lane in
// rising order; -inf for NaN and beyond the row's end.
constexpr uint32_t kSpan = 1024, kEach = 16;

template <class T>
struct Span {
    static constexpr uint32_t kWide = 16 / sizeof(typename T::type);  // elements of a 16-byte load
    float z[kEach];

    static __device__ __forceinline__ uint32_t index(uint32_t base, uint32_t i) {
        return base + i / kWide * (64 * kWide) + threadIdx.x % 64 * kWide + i % kWide;
    }
    __device__ __forceinline__ void load(const LeoBeams& a, uint64_t row, uint32_t base) {
        const uint32_t n = static_cast<uint32_t>(a.symbols);
        const auto* logits = static_cast<const typename T::type*>(a.logits) + row * a.logits_stride;
        uint4v raw[kEach / kWide];
#pragma unroll
        for (uint32_t v = 0; v < kEach / kWide; ++v) raw[v] = load_row<T>(logits, index(base, v * kWide), n);
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) z[i] = fmaxf(T::at(raw[i / kWide], i % kWide), negative_infinity());
    }
    __device__ __forceinline__ float top() const {
        float m = z[0];
#pragma unroll
        for (uint32_t i = 1; i < kEach; ++i) m = fmaxf(m, z[i]);
        return m;
    }
    __device__ __forceinline__ uint64_t key(uint32_t base, uint32_t i) const {
        return z[i] > negative_infinity() ? candidate(z[i], index(base, i)) : 0;
    }
};

// What symbols, a span or a run of spans leave for their row: the largest logit, and the sum
// of exponentials as mass * 2^power_of(top) * e^base_of(top). A power of two in place of the
// largest itself, so that no difference of two logits is rounded, and sums meet exactly. From
// 2^10 on the largest comes off first, which is exact for all that counts beside it.
constexpr float kLog2E = 1.44269504f;
constexpr double kLog2ERest = 1.92596299e-8, kLn2 = 0.69314718055994531;  // log2(e) is kLog2E + kLog2ERest
__device__ __forceinline__ float base_of(float top) { return fabsf(top) < 0x1p10f ? 0.0f : top; }
__device__ __forceinline__ float power_of(float top) { return fabsf(top) < 0x1p10f ? ceilf(top * kLog2E) : 0.0f; }

struct SpanRecord {
    float top;
    uint32_t pad0;
    double mass;
};
__device__ __forceinline__ double against(const SpanRecord& r, float top) {
    if (r.top == top) return r.mass;
    if (!(r.top > top - 800.0f)) return 0.0;
    const float base = base_of(r.top), to = base_of(top), power = power_of(r.top) - power_of(top);
    if (base == to) return ldexp(r.mass, static_cast<int>(power));
    return r.mass * exp(static_cast<double>(base) - to + power * kLn2);
}
// A lane takes its sixteen against a power of two near their own largest, in floats: the fused
// product rounds an exponent by half a step, which is 2^-25 for one near that power and grows as
// the exponential gets smaller: for fifteen beside the largest 1.1e-7 of the sum at most, when
// they lie four powers of two below. Exponentials are off by a step, 1.2e-7, three additions by
// 2^-24 each, 1.8e-7, what is left of log2(e) by 0.3e-7 once the lane's largest has it: together
// 4.4e-7, less than 2^-21, however alike the terms are. All else has 64 bits.
template <class T>
__device__ __forceinline__ SpanRecord weigh(const Span<T>& s, float lane_top) {
    const float top = wave_max(lane_top);
    if (top == negative_infinity()) return {top, 0, 0.0};
    float e[kEach];
    const float base = base_of(top), mine = fmaxf(lane_top - base, -2000.0f), power = ceilf(mine * kLog2E);  // much lower ones come to 0
    if (top < __builtin_inff()) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s.z[i] - base, kLog2E, -power));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) e[i] = s.z[i] == top ? 1.0f : 0.0f;
    }
#pragma unroll
    for (uint32_t half = kEach / 2; half > 1; half /= 2)
#pragma unroll
        for (uint32_t i = 0; i < half; ++i) e[i] += e[i + half];
    const double sum = static_cast<double>(e[0]) + e[1], rest = mine * static_cast<float>(kLog2ERest * kLn2);
    if (top == __builtin_inff()) return {top, 0, wave_sum(sum)};
    return {top, 0, wave_sum(ldexp(__builtin_fma(sum, rest, sum), static_cast<int>(power - power_of(top))))};
}

// The `kept` best of the spans of a workgroup (or of one wave's span, kWave), in
// falling order, 0 behind the last. All that is not below a bar is gathered in `pool`
// and finds its place by counting. Where more lies there than the pool holds, as ties
// may, the kept-th best is found bit by bit, which no other symbol equals.
template <class T, bool kWave>
__device__ __forceinline__ void pick(const Span<T>& s, uint32_t base, float lane_top, uint32_t kept, uint64_t* pool, uint32_t capacity,
                                     uint32_t* counters, uint32_t* maxima, uint64_t* to) {
    const uint32_t thread = kWave ? threadIdx.x % 64 : threadIdx.x, threads = kWave ? 64 : blockDim.x;
    if (thread == 0) counters[0] = counters[1] = 0;
    const uint32_t largest = lane_top > negative_infinity() ? order_key(lane_top + 0.0f) : 0;
    uint32_t key = 0;
    if ((kWave || blockDim.x == 64) && kept > kFewKept) {  // the kept-th largest of the wave's symbols themselves
        for (int bit = 31; bit >= 12; --bit) {
            const float higher = from_order_key(key | 1u << bit);
            uint32_t above = 0;
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) above += static_cast<uint32_t>(__popcll(__ballot(s.z[i] >= higher)));
            if (above >= kept) key |= 1u << bit;
        }
    } else {
        key = bar_of<kWave>(largest, kept, maxima);
    }
    const float bar = from_order_key(max(key, 0x00800000u));  // the lowest finite value or more
    settle_lds<kWave>();
    const auto gather = [&](auto&& stays) {
        if (!__any(lane_top >= bar)) return;
        uint64_t masks[kEach];
        uint32_t total = 0, at = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            masks[i] = __ballot(stays(i));
            total += static_cast<uint32_t>(__popcll(masks[i]));
        }
        if (threadIdx.x % 64 == 0) at = atomicAdd(&counters[0], total);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if (!masks[i]) continue;
            const uint32_t mine = at + below_in(masks[i]);
            if (stays(i) && mine < capacity) pool[mine] = s.key(base, i);
            at += static_cast<uint32_t>(__popcll(masks[i]));
        }
    };
    gather([&](uint32_t i) { return s.z[i] >= bar; });
    settle_lds<kWave>();
    uint32_t count = counters[0];
    if (count > capacity) {
        uint64_t least = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t higher = least | 1ull << bit;
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) mine += s.key(base, i) >= higher;
            mine = wave_sum(mine);
            if constexpr (!kWave) {
                __syncthreads();
                if (threadIdx.x == 0) counters[1] = 0;
                __syncthreads();
                if (threadIdx.x % 64 == 0) atomicAdd(&counters[1], mine);
                __syncthreads();
                mine = counters[1];
            }
            if (mine >= kept) least = higher;
        }
        settle_lds<kWave>();
        if (thread == 0) counters[0] = 0;
        settle_lds<kWave>();
        gather([&](uint32_t i) { return s.key(base, i) >= least; });
        settle_lds<kWave>();
        count = counters[0];
    }
    for (uint32_t i = thread; i < count; i += threads) {
        const uint64_t mine = pool[i];
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < count; ++j) rank += pool[j] > mine;
        if (rank < kept) to[rank] = mine;
    }
    for (uint32_t i = count + thread; i < kept; i += threads) to[i] = 0;
}

__device__ __forceinline__ bool is_finished(const LeoBeams& a, uint64_t row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ bool is_open(const LeoBeams& a, uint64_t row) { return !is_finished(a, row) && a.scores[row] > negative_infinity(); }

// n^p for p >= 0. Whole and half powers by products and a root, which round nothing where
// the result is a whole number below 2^53, so that ranks that are equal as quotients tie;
// pow may be off by a step there, as it is for a p of 1.
__device__ __forceinline__ double power_of_length(double n, double p) {
    const double whole = floor(p);
    if (whole > 64.0 || (p != whole && p != whole + 0.5)) return pow(n, p);
    double r = p == whole ? 1.0 : sqrt(n), square = n;
    for (uint32_t left = static_cast<uint32_t>(whole); left; left /= 2, square *= square)
        if (left % 2) r *= square;
    return r;
}

// What makes a hypothesis' logits comparable with another's.
struct Hypothesis {
    double score, log_mass;  // log_mass against the top
    double factor, power;    // what makes a score a rank; the length's power that it is the inverse of
    float top;
    uint32_t kind;  // 0: none, 1: finished, 2: open
};

// A candidate on its way to its place: larger ranks first, of equals the lower
// hypothesis, then the better candidate.
struct Ranked {
    uint64_t rank, second;
    // 6 bits for the hypothesis, 32 for the logit, 26 for the symbol
    static __device__ __forceinline__ uint64_t second_of(uint32_t beam, uint64_t key) {
        return static_cast<uint64_t>(63 - beam) << 58 | (key >> 32) << 26 | (key & 0x3ffffffu);
    }
    __device__ __forceinline__ uint32_t beam() const { return 63 - static_cast<uint32_t>(second >> 58); }
    __device__ __forceinline__ uint64_t key() const { return (second >> 26 & 0xffffffffu) << 32 | 0xfc000000u | (second & 0x3ffffffu); }
};
__device__ __forceinline__ bool before(const Ranked& p, const Ranked& q) {
    return (p.rank > q.rank) | ((p.rank == q.rank) & (p.second > q.second));
}

constexpr uint32_t kPool = 1024;  // of a search's candidates
struct MergeShared {
    Hypothesis hypotheses[kMostBeams];
    Ranked pool[kPool];
    Ranked best[16];
    uint32_t maxima[kMostWaves * 64];
    uint32_t count;
};

// Where lists are four times as many as what is kept, the best of each say enough. With 16
// of 16 the least of them would be the bar, and a step of 16 beams of 1,000 took 18.5 us.
__host__ __device__ inline bool follows_lists(uint32_t all, uint32_t kept) { return all >= 4 * kept; }

// A search's answer from its hypotheses' records and candidates, [beams][lists] and
// [beams][lists][kept], by a whole workgroup of 2^n waves. What it reads is on
// its way before anything is needed; the lists of finished hypotheses and of those with no
// score hold anything, and count for nothing.
constexpr uint32_t kAhead = 2;
struct Given {
    float score;
    bool finished;
    int32_t length;
};
__device__ __forceinline__ Given given_of(const LeoBeams& a, uint64_t row) {
    return {a.scores[row], is_finished(a, row), a.lengths ? a.lengths[row] : 0};
}
// `mine_given` is what is given for the hypothesis of this thread's wave.
__device__ __forceinline__ void merge(const LeoBeams& a, uint64_t group, const Given& mine_given, const SpanRecord* records,
                                      const uint64_t* candidates, uint32_t lists, MergeShared& shared) {
    const uint64_t first = group * a.beams;
    const uint32_t thread = threadIdx.x, threads = blockDim.x, lane = thread % 64, wave = thread / 64, waves = threads / 64,
                   beams = static_cast<uint32_t>(a.beams), kept = static_cast<uint32_t>(a.kept), all = beams * lists;
    // A thread's first list, so that neighbouring lists fall to different groups of the bar's: where a search begins, one
    // hypothesis has all that counts.
    const uint32_t own = thread % waves * 64 + thread / waves;
    uint64_t ahead[kAhead];
#pragma unroll
    for (uint32_t p = 0; p < kAhead; ++p) ahead[p] = own < all && p < kept ? candidates[static_cast<uint64_t>(own) * kept + p] : 0;
    for (uint32_t b = wave; b < beams; b += waves) {
        const uint64_t row = first + b;
        const SpanRecord none = {negative_infinity(), 0, 0.0};
        const SpanRecord mine = lane < lists ? records[b * lists + lane] : none, next = lane + 64 < lists ? records[b * lists + lane + 64] : none;
        const Given given = b == wave ? mine_given : given_of(a, row);
        Hypothesis h{};
        h.score = given.score;
        h.kind = !(given.score > negative_infinity()) ? 0 : given.finished ? 1 : 2;
        h.factor = 1.0;
        if (a.length_penalty != 0.0) {  // while the records are on their way
            const int64_t grown = static_cast<int64_t>(given.length) + (h.kind == 1 ? 0 : 1);
            const double power = power_of_length(static_cast<double>(grown < 1 ? 1 : grown), fabs(a.length_penalty));
            h.factor = a.length_penalty < 0.0 ? power : 1.0 / power;
            h.power = power < __builtin_inf() ? power : 0.0;
        }
        if (h.kind == 2) {
            float top = fmaxf(mine.top, next.top);
#pragma unroll 4
            for (uint32_t i = lane + 128; i < lists; i += 64) top = fmaxf(top, records[b * lists + i].top);
            top = wave_max(top);
            double mass = against(mine, top) + against(next, top);
#pragma unroll 4
            for (uint32_t i = lane + 128; i < lists; i += 64) mass += against(records[b * lists + i], top);
            h.log_mass = log(wave_sum(mass)) + (base_of(top) == top ? 0.0 : power_of(top) * kLn2 - top);
            h.top = top;
        }
        if (lane == 0) shared.hypotheses[b] = h;
    }
    if (thread == 0) shared.count = 0;
    __syncthreads();
    const auto score_of = [&](const Hypothesis& h, uint64_t key) {
        const float z = logit_of(key);
        const double below = static_cast<double>(z) - h.top, grown = h.score + ((z == h.top ? 0.0 : below) - h.log_mass);
        return h.kind == 1 ? h.score : grown;
    };
    // rank 0 is none
    const auto ranked = [&](uint32_t list, uint32_t place, uint64_t key) -> Ranked {
        const uint32_t beam = list / lists;
        const Hypothesis& h = shared.hypotheses[beam];
        key = h.kind != 1 ? key : place == 0 && list == beam * lists ? 1 : 0;
        const double score = score_of(h, key);
        // The remainder of the product with the inverse makes it the quotient, rounded once: -49 over 49 and -3 over 3 are
        // one rank. A division here took 590 us of a step of 32 x 8 beams of 131,075 to 64 whose pool runs over, this 555, the product alone 520.
        double value = score * h.factor;
        if (a.length_penalty > 0.0) value = __builtin_fma(__builtin_fma(-value, h.power, score), h.factor, value);
        const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(value + 0.0));
        const bool none = h.kind == 0 || key == 0 || !(score > -__builtin_inf());
        return {none ? 0 : bits >> 63 ? ~bits : bits | 1ull << 63, Ranked::second_of(beam, key)};
    };
    const Ranked nothing = {0, 0};
    const auto load_ranked = [&](uint32_t list, uint32_t place) {
        if (shared.hypotheses[list / lists].kind == 0) return nothing;
        return ranked(list, place, candidates[static_cast<uint64_t>(list) * kept + place]);
    };
    const uint32_t items = all * kept;
    const auto item = [&](uint32_t i) { return i < items ? load_ranked(i % all, i / all) : nothing; };
    const auto answer = [&](uint32_t k, const Ranked& r) {
        const bool found = r.rank != 0;
        const uint32_t beam = found ? r.beam() : 0;
        const uint64_t to = group * kept + k, row = first + beam;
        const Hypothesis& h = shared.hypotheses[beam];
        const bool grows = found && h.kind == 2;
        const int32_t symbol = grows ? static_cast<int32_t>(symbol_of(r.key())) : -1;
        a.out_symbols[to] = symbol;
        a.out_parents[to] = static_cast<int32_t>(beam);
        a.out_scores[to] = found ? static_cast<float>(score_of(h, r.key())) : negative_infinity();
        if (a.out_finished) a.out_finished[to] = found && (!grows || symbol == a.end);
        if (a.out_lengths) a.out_lengths[to] = a.lengths[row] + (grows ? 1 : 0);
    };
    const auto gather = [&](const Ranked& r, uint32_t bar) {  // whether any of the wave's was taken
        const bool taken = r.rank >> 32 >= bar;
        if (!__any(taken)) return false;
        const uint32_t at = place_for(taken, &shared.count);
        if (taken && at < kPool) shared.pool[at] = r;
        return true;
    };
    const uint32_t kind = lane < beams ? shared.hypotheses[lane].kind : 0;
    const uint32_t live = static_cast<uint32_t>(__popcll(__ballot(kind == 2))) * lists + static_cast<uint32_t>(__popcll(__ballot(kind == 1)));
    uint32_t largest = 0;
    if (follows_lists(live, kept)) {
        // the lists' best bound what can be kept, and each list is followed down to the bar
        for (uint32_t list = own; list < all; list += threads)
            largest = max(largest, static_cast<uint32_t>((list == own ? ranked(list, 0, ahead[0]) : load_ranked(list, 0)).rank >> 32));
        const uint32_t bar = max(bar_of<false>(largest, kept, shared.maxima), 1u);
        for (uint32_t from = 0; from < all; from += threads) {
            if (!__any(largest >= bar)) break;
            const uint32_t list = from + own;
            bool more = true;
            if (from == 0) {  // one addition for what the lists' first places hold, which is mostly all
                Ranked r[kAhead];
                uint64_t masks[kAhead];
                uint32_t total = 0, at = 0;
#pragma unroll
                for (uint32_t p = 0; p < kAhead; ++p) {
                    r[p] = list < all && p < kept ? ranked(list, p, ahead[p]) : nothing;
                    masks[p] = __ballot(r[p].rank >> 32 >= bar);
                    total += static_cast<uint32_t>(__popcll(masks[p]));
                }
                if (lane == 0) at = atomicAdd(&shared.count, total);
                at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
                for (uint32_t p = 0; p < kAhead; ++p) {
                    const uint32_t mine = at + below_in(masks[p]);
                    if (masks[p] >> lane & 1 && mine < kPool) shared.pool[mine] = r[p];
                    at += static_cast<uint32_t>(__popcll(masks[p]));
                }
                more = masks[kAhead - 1] != 0;
            }
            for (uint32_t p = from == 0 ? kAhead : 0; more && p < kept; ++p) more = gather(list < all ? load_ranked(list, p) : nothing, bar);
        }
    } else {
        // few lists: all their candidates
        const Ranked one = item(own);
        largest = static_cast<uint32_t>(one.rank >> 32);
#pragma unroll 4
        for (uint32_t i = own + threads; i < items; i += threads) largest = max(largest, static_cast<uint32_t>(item(i).rank >> 32));
        const uint32_t bar = max(bar_of<false>(largest, kept, shared.maxima), 1u);
        for (uint32_t from = 0; from < items; from += threads) {
            if (!__any(largest >= bar)) break;
            gather(from == 0 ? one : item(from + own), bar);
        }
    }
    __syncthreads();
    uint32_t count = shared.count;
    if (count > kPool) {
        // the bar let through too much, as with rows in falling order: the kept-th rank's upper half, bit by bit
        uint32_t bar = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t higher = bar | 1u << bit;
            uint32_t mine = 0;
#pragma unroll 4
            for (uint32_t i = thread; i < items; i += threads) mine += item(i).rank >> 32 >= higher;
            mine = wave_sum(mine);
            __syncthreads();
            if (thread == 0) shared.count = 0;
            __syncthreads();
            if (lane == 0) atomicAdd(&shared.count, mine);
            __syncthreads();
            if (shared.count >= kept) bar = higher;
        }
        __syncthreads();
        if (thread == 0) shared.count = 0;
        __syncthreads();
        for (uint32_t from = 0; from < items; from += threads) gather(item(from + thread), max(bar, 1u));
        __syncthreads();
        count = shared.count;
    }
    if (count <= kPool) {
        for (uint32_t i = thread; i < count; i += threads) {
            const Ranked mine = shared.pool[i];
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t j = 0; j < count; ++j) rank += before(shared.pool[j], mine);
            if (rank < kept) answer(rank, mine);
        }
        for (uint32_t k = count + thread; k < kept; k += threads) answer(k, nothing);
        return;
    }
    // more ties than the pool holds: one after the other
    Ranked last = {~0ull, ~0ull};
    for (uint32_t k = 0; k < kept; ++k) {
        Ranked best = nothing;
#pragma unroll 4
        for (uint32_t i = thread; i < items; i += threads) {
            const Ranked r = item(i);
            if (r.rank && before(last, r) && (!best.rank || before(r, best))) best = r;
        }
        const auto meet = [&](const Ranked& other) {
            if (other.rank && (!best.rank || before(other, best))) best = other;
        };
#pragma unroll
        for (int step = 32; step; step /= 2)
            meet({__shfl_xor(static_cast<unsigned long long>(best.rank), step), __shfl_xor(static_cast<unsigned long long>(best.second), step)});
        if (lane == 0) shared.best[wave] = best;
        __syncthreads();
        for (uint32_t w = 0; w < waves; ++w) meet(shared.best[w]);
        __syncthreads();
        if (thread == 0) answer(k, best);
        if (!best.rank) {
            for (uint32_t j = k + 1 + thread; j < kept; j += threads) answer(j, nothing);
            return;
        }
        last = best;
    }
}

// Searches whose rows make up to 16 spans take one workgroup each: a wave a span,
// which picks from its registers, then the search's answer. A chain of reductions bounds
// it: 7.4 us for 4 beams of 257.
constexpr uint32_t kWavePool = 320;
template <class T>
__global__ __launch_bounds__(kMostWaves * 64) void leo_beam_whole(LeoBeams a, uint32_t spans) {
    union Shared {
        uint64_t pools[kMostWaves][kWavePool];
        MergeShared merge;
    };
    __shared__ Shared shared;
    __shared__ uint64_t candidates[kMostWaves][kMostBeams];
    __shared__ SpanRecord records[kMostWaves];
    __shared__ uint32_t counters[kMostWaves][2];
    const uint32_t wave = threadIdx.x / 64, beam = wave / spans, base = wave % spans * kSpan, kept = static_cast<uint32_t>(a.kept);
    const uint64_t row = blockIdx.x * a.beams + beam;
    const Given given = given_of(a, blockIdx.x * a.beams + min(static_cast<uint64_t>(wave), a.beams - 1));
    if (beam < a.beams) {
        Span<T> s;
        s.load(a, row, base);  // also where nothing comes of it: sooner than after asking
        const float lane_top = s.top();
        const SpanRecord r = weigh(s, lane_top);
        if (threadIdx.x % 64 == 0) records[wave] = r;
        pick<T, true>(s, base, lane_top, kept, shared.pools[wave], kWavePool, counters[wave], nullptr, &candidates[0][0] + wave * kept);
    }
    __syncthreads();
    merge(a, blockIdx.x, given, records, &candidates[0][0], spans, shared.merge);
}

// Longer rows: a workgroup a run of spans, a wave each, which leaves its record and its
// best candidates; then a workgroup a search. 32 x 8 beams of 131,075, of which 94 MB count,
// take the first 21.3 us (4.4 TB/s) and 23.1 where no input is left in the cache beside memory,
// four fifths of its rate (with 16 waves a workgroup, which wait for each other longer, a fifth
// more). Latency bounds the second: 7.4 to 8.0 us.
constexpr uint32_t kRowPool = 1024;
template <class T>
__global__ __launch_bounds__(256) void leo_beam_rows(LeoBeams a, uint32_t lists, SpanRecord* records, uint64_t* candidates) {
    __shared__ uint64_t pool[kRowPool];
    __shared__ uint32_t maxima[256], counters[2];
    __shared__ SpanRecord parts[4];
    const uint64_t row = blockIdx.y;
    if (!is_open(a, row)) return;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64, span = blockIdx.x * waves + wave;
    Span<T> s;
    s.load(a, row, span * kSpan);
    const float lane_top = s.top();
    const SpanRecord r = weigh(s, lane_top);
    if (lane == 0) parts[wave] = r;
    pick<T, false>(s, span * kSpan, lane_top, static_cast<uint32_t>(a.kept), pool, kRowPool, counters, maxima,
                   candidates + (row * lists + blockIdx.x) * a.kept);
    if (wave != 0) return;
    const SpanRecord mine = lane < waves ? parts[lane] : SpanRecord{negative_infinity(), 0, 0.0};
    const float top = wave_max(mine.top);
    const double mass = wave_sum(against(mine, top));
    if (lane == 0) records[row * lists + blockIdx.x] = {top, 0, top > negative_infinity() ? mass : 0.0};
}

__global__ __launch_bounds__(kMostWaves * 64) void leo_beam_groups(LeoBeams a, uint32_t lists, const SpanRecord* records,
                                                                  const uint64_t* candidates) {
    __shared__ MergeShared shared;
    const uint64_t first = blockIdx.x * a.beams;
    const Given given = given_of(a, first + min(static_cast<uint64_t>(threadIdx.x / 64), a.beams - 1));
    merge(a, blockIdx.x, given, records + first * lists, candidates + first * lists * a.kept, lists, shared);
}

struct BeamPlan {
    uint32_t spans, lists;         // of a row
    uint32_t waves, merge_waves;   // of a workgroup
    bool whole;
    uint64_t candidates, workspace;  // the candidates' offset, and the whole
};
BeamPlan beam_plan(uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols) {
    const uint64_t rows = groups * beams;
    BeamPlan p{};
    const auto power = [](uint64_t most) {  // the least power of two that is no less
        uint32_t v = 1;
        while (v < most && v < kMostWaves) v *= 2;
        return v;
    };
    p.spans = static_cast<uint32_t>((symbols + kSpan - 1) / kSpan);
    // One launch took 6.4 us for the two's 8.1 for 4 beams of 257, 9.7 for 11.4 for 256 searches of 8 beams of 2,000, but
    // 8.7 for 8.1 for 4 beams of 4,000, whose rows one workgroup each answers with fewer lists.
    p.whole = beams * p.spans <= kMostWaves && p.spans <= 2;
    if (p.whole) {
        p.waves = power(beams * p.spans);
        return p;
    }
    p.waves = std::min(power(p.spans), 4u);
    p.lists = (p.spans + p.waves - 1) / p.waves;
    const uint64_t all = beams * p.lists;
    p.merge_waves = power(std::max(beams, ((follows_lists(static_cast<uint32_t>(all), static_cast<uint32_t>(kept)) ? all : all * kept) + 63) / 64));
    p.candidates = (rows * p.lists * sizeof(SpanRecord) + 255) / 256 * 256;
    p.workspace = p.candidates + rows * p.lists * kept * sizeof(uint64_t);
    return p;
}

void check_beams(const char* who, uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols) {
    const auto need = [&](bool ok, const char* what) {
        if (!ok) throw Error(LEO_ERR_INVALID_ARGUMENT, std::string(who) + ": " + what);
    };
    need(beams >= 1 && beams <= kMostBeams, "beams must be 1 .. 64");
    need(kept >= 1 && kept <= kMostBeams, "kept must be 1 .. 64");
    need(groups <= 65535 / beams, "too many hypotheses");  // a product could wrap
    need(symbols >= 1 && symbols <= 1u << 26, "symbols must be 1 .. 2^26");
}

template <class T>
void launch_beams(const BeamPlan& p, const LeoBeams& b, hipStream_t stream) {
    const dim3 groups(static_cast<uint32_t>(b.groups));
    if (p.whole) return launch(leo_beam_whole<T>, groups, dim3(p.waves * 64), 0, stream, b, p.spans);
    auto* records = static_cast<SpanRecord*>(b.workspace);
    auto* candidates = reinterpret_cast<uint64_t*>(static_cast<char*>(b.workspace) + p.candidates);
    launch(leo_beam_rows<T>, dim3(p.lists, static_cast<uint32_t>(b.groups * b.beams)), dim3(p.waves * 64), 0, stream, b, p.lists, records,
           candidates);
    launch(leo_beam_groups, groups, dim3(p.merge_waves * 64), 0, stream, b, p.lists, static_cast<const SpanRecord*>(records),
           static_cast<const uint64_t*>(candidates));
}

// --- reordering ------------------------------------------------------------------------------------------------------

// A thread takes 16 bytes of a place of its search's rows, for all of their targets, so a
// row that several hypotheses continue comes from memory once. Memory bounds it. Stores
// start at multiples of 16, loads at multiples of 4: the bytes that a row's place lies off
// those are shifted in registers. In place a thread writes nothing but the columns that it
// alone reads, the same in every row, and holds what it moves in LDS that is its own. 8
// planes of 8 rows of 4 MB take 75 to 89 us (5.0 to 5.9 TB/s of memory and the cache beside
// it), 8-bit caches with rows off all boundaries, 266 MB, 57, and 66 from memory alone.
constexpr uint32_t kArrays = 32;

struct ReorderArgs {
    LeoStateArray arrays[kArrays];
    uint32_t columns[kArrays];  // of 16 bytes, of a place
    uint32_t units[kArrays];    // workgroups of a search
    uint32_t before[kArrays];   // workgroups of the arrays before
    uint32_t all;               // workgroups
    uint32_t count;
    uint32_t groups, beams, kept;
    const int32_t* parents;
};

// 16 bytes from any address, by way of the five words that hold them.
__device__ __forceinline__ uint4v load_shifted(const char* p) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 3u;
    const char* words = p - off;
    uint4v v = load_16(__builtin_assume_aligned(words, 4));
    if (__any(off != 0)) {
        // where off is 0, the last word again: the next one may be another's
        const uint32_t next = *reinterpret_cast<const uint32_t*>(words + (off ? 16 : 12));
        v = uint4v{__builtin_amdgcn_alignbyte(v[1], v[0], off), __builtin_amdgcn_alignbyte(v[2], v[1], off),
                   __builtin_amdgcn_alignbyte(v[3], v[2], off), __builtin_amdgcn_alignbyte(next, v[3], off)};
    }
    return v;
}

template <bool kInPlace>
__global__ __launch_bounds__(256) void leo_reorder(ReorderArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint4v held[];
    const uint32_t block = block_of_grid();
    if (block >= a.all) return;
    uint32_t which = 0;
    while (which + 1 < a.count && block >= a.before[which + 1]) ++which;
    const LeoStateArray& s = a.arrays[which];
    const uint32_t columns = a.columns[which], units = a.units[which], unit = block - a.before[which];
    const uint64_t group = unit / units, all = columns * s.outer, column = static_cast<uint64_t>(unit % units) * blockDim.x + threadIdx.x;
    if (column >= all) return;
    uint64_t outer = 0;
    if (s.outer > 1) outer = all >> 32 ? column / columns : static_cast<uint32_t>(column) / columns;
    const int64_t place = static_cast<int64_t>(column - outer * columns) * 16, width = static_cast<int64_t>(s.width);
    const char* source = static_cast<const char*>(s.source) + outer * s.source_outer;
    char* target = static_cast<char*>(s.target) + outer * s.target_outer;
    const int32_t* parents = a.parents + group * a.kept;
    const auto row_of = [&](uint32_t k) { return target + static_cast<int64_t>(group * a.kept + k) * s.target_row; };
    const auto start = [&](uint32_t k) {
        return kInPlace ? place : place - static_cast<int64_t>(reinterpret_cast<uintptr_t>(row_of(k)) & 15u);
    };
    const auto read = [&](uint32_t k) {
        const int32_t parent = parents[k];
        const int64_t at = start(k);
        uint4v v = {0, 0, 0, 0};
        if (parent < 0 || parent >= static_cast<int32_t>(a.beams)) return v;
        const char* from = source + static_cast<int64_t>(group * a.beams + parent) * s.source_row;
        if (at >= 0 && at + 16 <= width) {
            v = load_shifted(from + at);
        } else {
            // the bytes beyond an end are its own again, so that all are on their way at once
            uint8_t bytes[16];
#pragma unroll
            for (int32_t i = 0; i < 16; ++i) bytes[i] = static_cast<uint8_t>(from[at + i < 0 ? 0 : at + i < width ? at + i : width - 1]);
#pragma unroll
            for (int32_t i = 0; i < 16; ++i) v[i / 4] |= static_cast<uint32_t>(bytes[i]) << (8 * (i % 4));
        }
        return v;
    };
    const auto write = [&](uint32_t k, const uint4v& v) {
        const int64_t at = start(k);
        char* to = row_of(k);
        if (at >= 0 && at + 16 <= width) {
            // past the caches, which keep what is read: 64 rows of 8 x 511 x 64 16-bit values took 107 us without and 66 so
            if constexpr (kInPlace) __builtin_memcpy(to + at, &v, 16);
            else __builtin_nontemporal_store(v, reinterpret_cast<uint4v*>(to + at));
        } else {
#pragma unroll
            for (int32_t i = 0; i < 16; ++i)
                if (at + i >= 0 && at + i < width) to[at + i] = static_cast<char>(v[i / 4] >> (8 * (i % 4)));
        }
    };
    const auto moves = [&](uint32_t k) { return k < a.kept && (!kInPlace || parents[k] != static_cast<int32_t>(k)); };
    constexpr uint32_t kTogether = 4;  // loads on their way; eight took registers, and 89 us for 80 of 8 planes of 8 rows of 4 MB
    for (uint32_t k = 0; k < a.kept; k += kTogether) {
        uint4v v[kTogether];
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j)
            if (moves(k + j)) v[j] = read(k + j);
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j) {
            if (!moves(k + j)) continue;
            if (kInPlace) held[(k + j) * blockDim.x + threadIdx.x] = v[j];
            else write(k + j, v[j]);
        }
    }
    if constexpr (kInPlace) {
        for (uint32_t k = 0; k < a.kept; ++k)
            if (moves(k)) write(k, held[k * blockDim.x + threadIdx.x]);
    }
}

// The bytes from an array's first to its last.
struct Extent {
    uint64_t begin, end;
    uint32_t array;
    bool target;
};

// Whether a target shares a byte with another of them; sorts them.
bool any_meet(std::vector<Extent>& extents) {
    std::sort(extents.begin(), extents.end(), [](const Extent& p, const Extent& q) { return p.begin < q.begin; });
    uint64_t all = 0, targets = 0;  // the ends of what came before
    for (const Extent& e : extents) {
        if (e.begin < targets || (e.target && e.begin < all)) return true;
        all = std::max(all, e.end);
        if (e.target) targets = std::max(targets, e.end);
    }
    return false;
}

// The same for arrays whose ranges meet, as the columns of one buffer do: where the
// starts of all their rows (or of all pieces of them) lie apart modulo a common
// divisor of the strides, no two meet.
bool may_meet(const LeoReorder& r, const std::vector<Extent>& extents) {
    for (const bool pieces : {false, true}) {
        uint64_t modulus = 0;
        const auto strides_of = [&](const Extent& e, uint64_t& row, uint64_t& outer) {
            const LeoStateArray& s = r.arrays[e.array];
            const uint64_t rows = r.groups * (e.target ? r.kept : r.beams);
            row = rows == 1 ? 0 : static_cast<uint64_t>(e.target ? s.target_row : s.source_row);
            outer = s.outer == 1 ? 0 : static_cast<uint64_t>(e.target ? s.target_outer : s.source_outer);
        };
        uint64_t row, outer;
        for (const Extent& e : extents) {
            strides_of(e, row, outer);
            modulus = std::gcd(modulus, row);
            if (pieces) modulus = std::gcd(modulus, outer);
        }
        if (modulus == 0) continue;  // single rows, whose pieces may still lie apart
        std::vector<Extent> folded;
        bool fits = true;
        for (const Extent& e : extents) {
            strides_of(e, row, outer);
            const LeoStateArray& s = r.arrays[e.array];
            const uint64_t length = s.width + (pieces ? 0 : (s.outer - 1) * outer), begin = e.begin % modulus;
            fits = fits && length <= modulus;
            folded.push_back({begin, std::min(begin + length, modulus), e.array, e.target});
            if (begin + length > modulus) folded.push_back({0, begin + length - modulus, e.array, e.target});
        }
        if (fits && !any_meet(folded)) return false;
    }
    return true;
}

// Refuses targets that share memory with anything else.
void check_apart(const LeoReorder& r, std::vector<Extent>& extents) {
    if (!any_meet(extents)) return;
    for (size_t from = 0; from < extents.size();) {
        std::vector<Extent> cluster;
        uint64_t end = 0;
        for (; from < extents.size() && (cluster.empty() || extents[from].begin < end); ++from) {
            end = std::max(end, extents[from].end);
            cluster.push_back(extents[from]);
        }
        std::vector<Extent> copy = cluster;
        require(!any_meet(copy) || !may_meet(r, cluster), "leo_reorder_states: a target overlaps another array");
    }
}

}  // namespace
}  // namespace leo

using namespace leo;

extern "C" {

int32_t leo_beam_workspace_bytes(uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols, uint64_t* bytes) {
    return guarded([&] {
        require(bytes, "leo_beam_workspace_bytes: null argument");
        check_beams("leo_beam_workspace_bytes", groups, beams, kept, symbols);
        *bytes = groups ? beam_plan(groups, beams, kept, symbols).workspace : 0;
    });
}

int32_t leo_beam_select(const LeoBeams* beams, void* stream) {
    return guarded([&] {
        require(beams, "leo_beam_select: null argument");
        const LeoBeams& b = *beams;
        check_beams("leo_beam_select", b.groups, b.beams, b.kept, b.symbols);
        require(valid_type(b.type), "leo_beam_select: unknown type");
        if (b.groups == 0) return;
        require(b.logits && b.scores && b.out_symbols && b.out_parents && b.out_scores, "leo_beam_select: null argument");
        require(b.logits_stride >= 0, "leo_beam_select: logits_stride must not be negative");
        require(std::isfinite(b.length_penalty), "leo_beam_select: length_penalty must be finite");
        require(b.lengths || (b.length_penalty == 0.0 && !b.out_lengths), "leo_beam_select: length_penalty or out_lengths without lengths");
        require(b.end >= -1 && b.end < static_cast<int64_t>(b.symbols), "leo_beam_select: end must be a symbol, or -1");
        struct Range {
            uintptr_t begin, end;
        };
        const auto range = [](const void* at, uint64_t bytes) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(at);
            return Range{begin, at ? begin + bytes : begin};
        };
        const uint64_t rows = b.groups * b.beams, places = b.groups * b.kept;
        const Range logits = range(b.logits, ((rows - 1) * static_cast<uint64_t>(b.logits_stride) + b.symbols) * type_bytes(b.type));
        const Range all[] = {range(b.out_symbols, places * 4), range(b.out_parents, places * 4), range(b.out_scores, places * 4),
                             range(b.out_finished, places), range(b.out_lengths, places * 4), logits, range(b.scores, rows * 4),
                             range(b.finished, rows), range(b.lengths, rows * 4)};
        for (int out = 0; out < 5; ++out)
            for (int other = out + 1; other < 9; ++other)
                require(all[out].end <= all[other].begin || all[other].end <= all[out].begin, "leo_beam_select: outputs overlap inputs or each other");
        const BeamPlan p = beam_plan(b.groups, b.beams, b.kept, b.symbols);
        require(p.workspace == 0 || (b.workspace && reinterpret_cast<uintptr_t>(b.workspace) % 256 == 0 && b.workspace_bytes >= p.workspace),
                "leo_beam_select: workspace is missing, too small or not 256-byte aligned");
        const auto at = static_cast<hipStream_t>(stream);
        if (b.type == LEO_TYPE_F32) launch_beams<F32>(p, b, at);
        else if (b.type == LEO_TYPE_F16) launch_beams<F16>(p, b, at);
        else launch_beams<BF16>(p, b, at);
    });
}

int32_t leo_reorder_states(const LeoReorder* reorder, void* stream) {
    return guarded([&] {
        require(reorder, "leo_reorder_states: null argument");
        const LeoReorder& r = *reorder;
        require(r.beams >= 1 && r.beams <= kMostBeams, "leo_reorder_states: beams must be 1 .. 64");
        require(r.kept >= 1 && r.kept <= kMostBeams, "leo_reorder_states: kept must be 1 .. 64");
        require(r.groups <= 65535, "leo_reorder_states: too many groups");
        if (r.count == 0 || r.groups == 0) return;
        require(r.arrays && r.parents, "leo_reorder_states: null argument");
        require(r.count <= 65535, "leo_reorder_states: too many arrays");
        const uint64_t from_rows = r.groups * r.beams, to_rows = r.groups * r.kept;
        constexpr uint64_t kMost = 1ull << 46;  // of sizes and strides, so that their products stay inside 64 bits
        std::vector<Extent> extents;
        std::vector<uint32_t> order[2];  // arrays out of place, in place
        for (uint32_t i = 0; i < r.count; ++i) {
            const LeoStateArray& s = r.arrays[i];
            if (s.outer == 0 || s.width == 0) continue;
            require(s.source && s.target, "leo_reorder_states: null array");
            require(s.outer <= 0x7fffffffu && s.width <= 1ull << 32, "leo_reorder_states: an array is too large");
            for (int64_t stride : {s.source_row, s.source_outer, s.target_row, s.target_outer})
                require(stride >= 0 && static_cast<uint64_t>(stride) <= kMost, "leo_reorder_states: strides must be 0 .. 2^46");
            const auto span = [&](uint64_t rows, int64_t row, int64_t outer) {
                return static_cast<uint64_t>(static_cast<unsigned __int128>(rows - 1) * row + static_cast<unsigned __int128>(s.outer - 1) * outer) + s.width;
            };
            // each of a target's pieces has bytes of its own: rows of pieces, or pieces of rows
            const uint64_t row = static_cast<uint64_t>(s.target_row), outer = static_cast<uint64_t>(s.target_outer);
            const bool by_row = (s.outer == 1 || outer >= s.width) && (to_rows == 1 || row >= (s.outer - 1) * outer + s.width);
            const bool by_outer = (to_rows == 1 || row >= s.width) && (s.outer == 1 || outer >= (to_rows - 1) * row + s.width);
            require(by_row || by_outer, "leo_reorder_states: a target's rows overlap");
            const bool same = s.source == s.target;
            if (same)
                require(r.beams == r.kept && s.source_row == s.target_row && (s.outer == 1 || s.source_outer == s.target_outer),
                        "leo_reorder_states: an array that is its own target needs the same strides and as many kept as beams");
            order[same].push_back(i);
            const uintptr_t from = reinterpret_cast<uintptr_t>(s.source), to = reinterpret_cast<uintptr_t>(s.target);
            const uintptr_t listed = reinterpret_cast<uintptr_t>(r.parents);
            require(listed >= to + span(to_rows, s.target_row, s.target_outer) || listed + to_rows * sizeof(int32_t) <= to,
                    "leo_reorder_states: a target overlaps the parents");
            if (!same) extents.push_back({from, from + span(from_rows, s.source_row, s.source_outer), i, false});
            extents.push_back({to, to + span(to_rows, s.target_row, s.target_outer), i, true});
        }
        check_apart(r, extents);
        // in place, the rows of a column are held in LDS: 64 KB
        const uint32_t threads = r.kept <= 16 ? 256 : r.kept <= 32 ? 128 : 64;
        ReorderArgs a{};
        a.groups = static_cast<uint32_t>(r.groups);
        a.beams = static_cast<uint32_t>(r.beams);
        a.kept = static_cast<uint32_t>(r.kept);
        a.parents = r.parents;
        for (int in_place = 0; in_place < 2; ++in_place) {
            for (size_t from = 0; from < order[in_place].size();) {
                uint64_t units = 0;
                a.count = 0;
                for (; from < order[in_place].size() && a.count < kArrays; ++from) {
                    const LeoStateArray& s = r.arrays[order[in_place][from]];
                    // a place that starts anywhere may touch one column more
                    const bool aligned = (reinterpret_cast<uintptr_t>(s.target) | s.target_row | s.target_outer) % 16 == 0;
                    const uint64_t columns = (s.width + (in_place || aligned ? 15 : 30)) / 16, mine = (columns * s.outer + threads - 1) / threads;
                    require(mine <= 0x7fffffffu / r.groups, "leo_reorder_states: an array is too large");
                    if (units + mine * r.groups > 0x7fffffffu) break;
                    a.arrays[a.count] = s;
                    a.columns[a.count] = static_cast<uint32_t>(columns);
                    a.units[a.count] = static_cast<uint32_t>(mine);
                    a.before[a.count++] = static_cast<uint32_t>(units);
                    units += mine * r.groups;
                }
                const auto at = static_cast<hipStream_t>(stream);
                a.all = static_cast<uint32_t>(units);
                const dim3 grid = grid_of(a.all), block(threads);
                if (in_place) launch(leo_reorder<true>, grid, block, a.kept * threads * 16, at, a);
                else launch(leo_reorder<false>, grid, block, 0, at, a);
            }
        }
    });
}

}  // extern "C"
