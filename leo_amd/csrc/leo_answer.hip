// Control of a row's logits and the draw of its next symbol.
#include <algorithm>

#include "decode_common.h"

namespace leo {
namespace {

__device__ __forceinline__ float negative_infinity() { return -__builtin_inff(); }

// Entries [begin, end) of a ragged list's row, held inside the list whatever
// the offsets say.
struct Run {
    int64_t begin, end;
};
__device__ __forceinline__ Run row_run(const int64_t* offsets, uint64_t row, uint64_t count) {
    if (!offsets) return {0, 0};
    const int64_t most = static_cast<int64_t>(count);
    const auto inside = [most](int64_t v) { return v < 0 ? 0 : v > most ? most : v; };
    return {inside(offsets[row]), inside(offsets[row + 1])};
}

// One workgroup a row and chunk of symbols. It notes in LDS, for each symbol of
// its chunk, the row's last bias entry and how often the history holds it
// (whole-number operations, whose order does not matter), and passes once over
// the logits, 16 bytes a lane. A word holds both, 16 bits each; a row with more
// entries than that takes its chunk by halves, with a word for each. Memory bounds
// the large calls: 128 rows of 131,075 float32 symbols with 8,192 symbols of history
// and 300 biases a row, 138 MB, take 33 to 40 us (3.5 to 4.2 TB/s), of which the lists,
// read once a chunk, are some 9 (31 us without them); hence the widest chunk that the
// LDS of two workgroups a CU holds: 64 KB. A launch bounds the small: 3.4 to 5 us for 257.
constexpr uint32_t kTable = 16384, kControlThreads = 1024;

template <class T>
__global__ __launch_bounds__(kControlThreads, 8) void leo_control_rows(LeoLogitControl a, uint32_t chunk) {
    extern __shared__ __attribute__((aligned(16))) uint32_t table[];
    constexpr uint32_t kWide = 16 / sizeof(typename T::type), kHeld = kTable / kControlThreads / kWide;
    const uint64_t row = blockIdx.y;
    const uint32_t n = static_cast<uint32_t>(a.symbols), threads = blockDim.x;
    const uint32_t begin = blockIdx.x * chunk, end = min(begin + chunk, n);
    const Run history = row_run(a.history_offsets, row, a.history_count);
    const Run bias = row_run(a.bias_offsets, row, a.bias_count);
    const bool listed = history.end > history.begin || bias.end > bias.begin;
    const bool wide = max(history.end - history.begin, bias.end - bias.begin) >= 0xffff;
    const uint32_t step = wide ? chunk / 2 : chunk;
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f;
    const float frequency = a.frequency ? a.frequency[row] : 0.0f;
    const int32_t* mask = nullptr;
    bool shut = false;
    if (a.masks) {
        const int64_t which = a.mask_rows ? a.mask_rows[row] : a.mask_count == 1 ? 0 : static_cast<int64_t>(row);
        shut = which < -1 || which >= static_cast<int64_t>(a.mask_count);
        if (!shut && which >= 0) mask = a.masks + which * a.masks_stride;
    }
    const auto* logits = static_cast<const typename T::type*>(a.logits) + row * a.logits_stride;
    auto* out = static_cast<typename T::type*>(a.out) + row * a.out_stride;
    const auto bits_of = [&](uint32_t v) {  // from symbol v's bit on
        return shut ? 0u : mask ? static_cast<uint32_t>(mask[v / 32]) >> (v % 32) : ~0u;
    };
    const auto adjusted = [&](float z, uint32_t count, uint32_t entry) {
        if (count) {
            z = z > 0.0f ? z / repetition : z * repetition;
            z = z - (presence + frequency * static_cast<float>(count));
        }
        if (entry) z = z + a.bias_values[bias.begin + entry - 1];
        return z;
    };
    for (uint32_t from = begin; from < end; from += step) {
        const uint32_t width = min(step, end - from), whole = wide ? 0 : width / kWide * kWide;  // wide rows go one by one
        // Chunks and halves begin at multiples of 32: the symbols of 16 bytes share a mask word. Logits and mask words
        // are on their way while the lists are read.
        uint4v raw[kHeld];
        uint32_t allowed[kHeld];
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h)
            if (const uint32_t i = (threadIdx.x + h * threads) * kWide; i < whole) {
                raw[h] = load_16(logits + from + i);
                allowed[h] = bits_of(from + i);
            }
        if (listed) {
            if (from != begin) __syncthreads();
            for (uint32_t i = threadIdx.x * 4; i < chunk; i += threads * 4)
                *reinterpret_cast<uint4v*>(table + i) = uint4v{0, 0, 0, 0};
            __syncthreads();
            // an entry counts from the row's first, 0 is none
            for (int64_t i = bias.begin + threadIdx.x; i < bias.end; i += threads) {
                const uint32_t at = static_cast<uint32_t>(a.bias_ids[i]) - from, entry = static_cast<uint32_t>(i - bias.begin) + 1;
                if (at < width) atomicMax(&table[wide ? chunk / 2 + at : at], wide ? entry : entry << 16);
            }
            if (!wide && bias.end > bias.begin) __syncthreads();
            const auto note = [&](uint32_t symbol) {
                if (symbol - from < width) atomicAdd(&table[symbol - from], 1u);
            };
            const int64_t fours = history.begin + (history.end - history.begin) / 4 * 4;
            for (int64_t first = history.begin + threadIdx.x * 4; first < fours; first += threads * 8) {
                const int64_t second = first + threads * 4;
                const uint4v four = load_16(a.history + first);
                uint4v more = {~0u, ~0u, ~0u, ~0u};
                if (second < fours) more = load_16(a.history + second);
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) note(four[e]);
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) note(more[e]);
            }
            if (fours + threadIdx.x < history.end) note(static_cast<uint32_t>(a.history[fours + threadIdx.x]));
            __syncthreads();
        }
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h) {
            const uint32_t i = (threadIdx.x + h * threads) * kWide;
            if (i >= whole) break;
            uint32_t word[kWide] = {}, any = 0;
            if (listed) {
#pragma unroll
                for (uint32_t e = 0; e < kWide; e += 4) {
                    const uint4v w = *reinterpret_cast<const uint4v*>(table + i + e);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) any |= word[e + k] = w[k];
                }
            }
            float z[kWide];
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e) z[e] = T::at(raw[h], e);
            if (any) {
#pragma unroll
                for (uint32_t e = 0; e < kWide; ++e) z[e] = adjusted(z[e], word[e] & 0xffffu, word[e] >> 16);
            }
            uint4v to;
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e) T::put(to, e, allowed[h] >> e & 1u ? z[e] : negative_infinity());
            __builtin_memcpy(out + from + i, &to, 16);
        }
        for (uint32_t i = whole + threadIdx.x; i < width; i += threads) {
            float z = T::load(logits, from + i);
            if (listed) z = wide ? adjusted(z, table[i], table[chunk / 2 + i]) : adjusted(z, table[i] & 0xffffu, table[i] >> 16);
            T::store(out, from + i, bits_of(from + i) & 1u ? z : negative_infinity());
        }
    }
}

// A float's bits in the order of its value.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// --- the draw ---------------------------------------------------------------
// The race: the symbol with the largest key z + noise, the lowest of equals.
struct Racer {
    float key;
    uint32_t at;
    float z;
    // A symbol whose noise makes no number races last, but it races: a race
    // over any symbols has a winner.
    __device__ __forceinline__ void meet(float k, uint32_t i, float value) {
        k = k == k ? k : negative_infinity();
        if (k > key || (k == key && i < at)) {
            key = k;
            at = i;
            z = value;
        }
    }
};
__device__ __forceinline__ Racer nobody() { return {negative_infinity(), 0xffffffffu, negative_infinity()}; }

__device__ __forceinline__ Racer wave_race(Racer r) {
    const float key = wave_max(r.key);
    const uint32_t at = wave_min(r.key == key ? r.at : 0xffffffffu);
    const uint64_t here = __ballot(r.key == key && r.at == at);
    const int lane = __ffsll(static_cast<unsigned long long>(here)) - 1;
    return {key, at, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(r.z), lane))};
}

// exp of a difference that is not above 0, 1 for a difference of infinities;
// its error grows with the size of the difference, as its share of a sum falls.
__device__ __forceinline__ float mass_of(float z, float top) {
    return z == top ? 1.0f : __builtin_amdgcn_exp2f((z - top) * 1.44269504f);
}

constexpr float kMost = 0x1.fffffep127f;

// A row's parameters.
struct Rules {
    float t, inverse, top_p, min_p;
    uint32_t top_k;
    bool greedy, ordinary, filtered;

    // logit / t, -inf for NaN. A finite logit's quotient does not fall to -inf: a row
    // that a mask left at its type's lowest value is not an empty one. A product with
    // the reciprocal and one correction by its remainder rounds as the division does
    // (3e8 random pairs, none apart) from logits of 2^-90 on; below, where the remainder
    // leaves float's range, it may be a unit in the last place off, and is still in the
    // logits' order.
    __device__ __forceinline__ float divided(float logit) const {
        float q = logit * inverse;
        if (ordinary) {
            const float exact = __builtin_fmaf(__builtin_fmaf(-q, t, logit), inverse, q);
            q = fabsf(q) < __builtin_inff() ? exact : q;
        } else {
            q = logit / t;
        }
        return logit > negative_infinity() ? fmaxf(q, -kMost) : negative_infinity();
    }
};
__device__ __forceinline__ Rules rules_of(const LeoSample& a, uint64_t row) {
    Rules r;
    r.t = a.noise ? (a.temperature ? a.temperature[row] : 1.0f) : 0.0f;
    r.greedy = !(r.t > 0.0f);
    if (r.greedy) r.t = 1.0f;
    r.inverse = 1.0f / r.t;
    r.ordinary = r.t > 0x1p-100f && r.t < 0x1p100f;
    r.top_k = a.top_k ? static_cast<uint32_t>(max(a.top_k[row], 1)) : 0x7fffffffu;
    r.top_p = a.top_p ? a.top_p[row] : 1.0f;
    r.min_p = a.min_p ? a.min_p[row] : 0.0f;
    r.filtered = !r.greedy && !(r.top_k >= a.symbols && r.top_p >= 1.0f && r.min_p <= 0.0f);
    return r;
}

// 1,024 neighbouring symbols of a row in the registers of a wave, 16 a lane in
// rising order: z, -inf for NaN and beyond the row's end, and the noise.
constexpr uint32_t kSpan = 1024, kEach = 16;

template <class T>
struct Span {
    static constexpr uint32_t kWide = 16 / sizeof(typename T::type);  // elements of a 16-byte load
    float z[kEach], noise[kEach];

    static __device__ __forceinline__ uint32_t index(uint32_t base, uint32_t i) {
        return base + i / kWide * (64 * kWide) + threadIdx.x % 64 * kWide + i % kWide;
    }
    __device__ __forceinline__ void load(const LeoSample& a, const Rules& r, uint64_t row, uint32_t base) {
        const uint32_t n = static_cast<uint32_t>(a.symbols);
        const auto* logits = static_cast<const typename T::type*>(a.logits) + row * a.logits_stride;
        const float* from = a.noise + row * a.noise_stride;
#pragma unroll
        for (uint32_t v = 0; v < kEach; v += kWide) {
            const uint32_t at = index(base, v);
            const uint4v raw = load_row<T>(logits, at, n);
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e) z[v + e] = T::at(raw, e);
        }
#pragma unroll
        for (uint32_t v = 0; v < kEach; v += 4) {
            const uint32_t at = index(base, v);
            if (r.greedy) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) noise[v + e] = 0.0f;
            } else {
                const uint4v raw = load_row<F32>(from, at, n);
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) noise[v + e] = __uint_as_float(raw[e]);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) z[i] = r.divided(z[i]);
    }
    __device__ __forceinline__ float key(const Rules& r, uint32_t i) const { return r.greedy ? z[i] : z[i] + noise[i]; }

    __device__ __forceinline__ float top() const {
        float m = z[0];
#pragma unroll
        for (uint32_t i = 1; i < kEach; ++i) m = fmaxf(m, z[i]);
        return wave_max(m);
    }
    // The lane's mass, against `top`, which is not -inf.
    __device__ __forceinline__ float mass(float top) const {
        float sum = 0.0f;
        if (top < __builtin_inff()) {
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) sum += __builtin_amdgcn_exp2f((z[i] - top) * 1.44269504f);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) sum += z[i] == top ? 1.0f : 0.0f;
        }
        return sum;
    }
    // The wave's winner. In rising order a larger key is enough; symbols whose
    // key is no number or -inf race only where a lane holds no others.
    __device__ __forceinline__ Racer race(const Rules& r, uint32_t base) const {
        Racer best = nobody();
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const float k = key(r, i);
            if (k > best.key) best = {k, index(base, i), z[i]};
        }
        if (__any(best.at == 0xffffffffu)) {
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i)
                if (best.at == 0xffffffffu && z[i] > negative_infinity()) best = {negative_infinity(), index(base, i), z[i]};
        }
        return wave_race(best);
    }
};

// What lies above a value: how many, their mass, the race among them.
struct Above {
    uint32_t count;
    float mass;
    Racer best;
    __device__ __forceinline__ void add(float w, float key, uint32_t at, float z) {
        count += 1;
        mass += w;
        best.meet(key, at, z);
    }
};

__device__ __forceinline__ Above wave_above(const Above& v) {
    return {wave_sum(v.count), wave_sum(v.mass), wave_race(v.best)};
}

constexpr uint32_t kMostWaves = 16;
struct SampleShared {
    Racer best[kMostWaves];
    float top[kMostWaves], mass[kMostWaves];
    Above above[2][2][kMostWaves];  // two pivots, alternating between sweeps
};

// What stays is a prefix of the values in falling order, so one value decides:
// the race's winner over the whole row is the answer if it stays; if not, no
// value up to its own stays, and the race is held again above.
struct Search {
    float top, whole;  // the row's largest value and its mass
    float lowest;      // of the values known to stay
    Racer best;        // the winner among what is not known not to stay

    __device__ __forceinline__ bool open(const Rules& r) const { return r.filtered && best.z < lowest; }
    // Halfway, in the order of floats, to the lowest value known to stay.
    __device__ __forceinline__ float halfway(float low) const {
        const uint32_t key = order_key(low);
        return from_order_key(key + (order_key(lowest) - key) / 2);
    }
    // Whether a value stays that has this above it.
    __device__ __forceinline__ bool stays(const Rules& r, float z, const Above& v) const {
        return v.count < r.top_k && (r.top_p >= 1.0f || v.mass < r.top_p * whole) && mass_of(z, top) >= r.min_p;
    }
    // Takes what lies above a value that is not below the winner's, and above a
    // higher one, if that was tried.
    __device__ __forceinline__ void narrow(const Rules& r, float low, float high, const Above (&above)[2], bool both) {
        if (stays(r, low, above[0])) {
            lowest = low;
        } else if (!both) {
            best = above[0].best;
        } else if (stays(r, high, above[1])) {
            lowest = high;
            best = above[0].best;
        } else {
            best = above[1].best;
        }
    }
};

// Narrows a search until it is decided, and stores its answer. `probe`, where it
// lies above the winner, is tried before: a value that is likely not to stay and
// has little above it. Few turns are enough where the noise is what it should
// be; from the fifth on a second value is tried with each, halfway to the lowest
// one known to stay, which bounds the turns by the 32 bits of a float. sweep(low,
// high, above) adds what a thread holds above either; all threads take part.
template <class Sweep>
__device__ __forceinline__ void settle(const LeoSample& a, const Rules& r, uint64_t row, Search s, float probe, SampleShared& shared,
                                       Sweep&& sweep) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    for (uint32_t turn = 0; s.open(r); ++turn) {
        const bool probing = probe > s.best.z && probe < s.lowest, both = turn >= 4;
        const float low = probing ? probe : s.best.z, high = both ? s.halfway(low) : __builtin_inff();
        Above above[2] = {{0, 0.0f, nobody()}, {0, 0.0f, nobody()}};
        sweep(low, high, above);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h == 1 && !both) break;
            above[h] = wave_above(above[h]);
            if (waves > 1 && lane == 0) shared.above[turn % 2][h][wave] = above[h];
        }
        if (waves > 1) {
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && !both) break;
                above[h] = wave_above(lane < waves ? shared.above[turn % 2][h][lane] : Above{0, 0.0f, nobody()});
            }
        }
        s.narrow(r, low, high, above, both);
        probe = negative_infinity();
    }
    if (threadIdx.x == 0) {
        const bool empty = s.top == negative_infinity();
        a.out_symbols[row] = empty ? -1 : static_cast<int32_t>(s.best.at);
        a.out_logprobs[row] = empty ? negative_infinity() : (s.best.z == s.top ? 0.0f : s.best.z - s.top) - logf(s.whole);
    }
}

__device__ __forceinline__ void add_above(float low, float high, float top, float z, float key, uint32_t at, Above (&above)[2]) {
    if (z > low) {
        const float w = mass_of(z, top);
        above[0].add(w, key, at, z);
        if (z > high) above[1].add(w, key, at, z);
    }
}

// A short row, in the registers of one workgroup: one span a wave, so that logits
// and noise are read once and every turn works on registers. A launch bounds it
// (257 symbols: 4.6 us), then one workgroup's turns.
// Up to 16 spans: 128 rows of 12,000 symbols took 23.0 us in the two launches below
// and 19.5 so, of 16,000 32.1 and 20.4, one row of 12,000 9.8 and 6.8.
template <class T>
__global__ __launch_bounds__(kMostWaves * 64) void leo_sample_row(LeoSample a) {
    __shared__ SampleShared shared;
    const uint64_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const Rules r = rules_of(a, row);
    Span<T> span;
    span.load(a, r, row, wave * kSpan);
    float top = span.top();
    Racer best = span.race(r, wave * kSpan);
    float mass = top > negative_infinity() ? wave_sum(span.mass(top)) : 0.0f;
    if (waves > 1) {
        if (lane == 0) {
            shared.best[wave] = best;
            shared.top[wave] = top;
            shared.mass[wave] = mass;
        }
        __syncthreads();
        const float theirs = lane < waves ? shared.top[lane] : negative_infinity();
        top = wave_max(theirs);
        mass = wave_sum(theirs > negative_infinity() ? shared.mass[lane] * mass_of(theirs, top) : 0.0f);
        best = wave_race(lane < waves ? shared.best[lane] : nobody());
    }
    settle(a, r, row, {top, mass, top, best}, negative_infinity(), shared, [&](float low, float high, Above (&above)[2]) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            add_above(low, high, top, span.z[i], span.key(r, i), Span<T>::index(wave * kSpan, i), above);
    });
}

// Longer rows take two launches: one wave a span weighs it and holds its race,
// and one workgroup a row settles the rest from the spans' records. This one reads
// everything once and is bound by memory: 128 rows of 131,075 float32 logits with
// noise, 134 MB, take 22.4 us (6.0 TB/s).
struct SpanRecord {
    Racer best;
    float top, mass;
};

template <class T>
__global__ __launch_bounds__(256) void leo_sample_spans(LeoSample a, uint32_t spans, SpanRecord* records) {
    const uint64_t row = blockIdx.y;
    const uint32_t which = blockIdx.x * 4 + threadIdx.x / 64;
    if (which >= spans) return;
    const Rules r = rules_of(a, row);
    Span<T> span;
    span.load(a, r, row, which * kSpan);
    SpanRecord rec;
    rec.top = span.top();
    rec.best = span.race(r, which * kSpan);
    rec.mass = rec.top > negative_infinity() ? wave_sum(span.mass(rec.top)) : 0.0f;
    if (threadIdx.x % 64 == 0) records[row * spans + which] = rec;
}

// What lies above a value is first gathered in LDS, by each lane in its own
// column, and counted and weighed from there: one compare a logit passes over
// the others. If no column runs over, later values, which are higher, need the
// columns alone. One CU's loads bound it: it reads again the spans that reach above
// the value, a megabyte for 262,147 symbols, and 128 rows of 131,075 take 24.3 us, 16
// rows of 32,001 11.1 and two of 262,147 10 to 146 as the values fall (24 states: half
// of them below 22). A third launch that gathered over all CUs gave back in latency what
// it saved (32,001: 5 + 7 + 10 us for 5 + 11, 131,075: 23 + 22 + 21 for 23 + 25). Two
// launches that take the first two turns with a wave a span: calls of 1, 2, 4 and 8 rows
// of 262,147 under min_p took 28.0, 28.2, 29.3 and 31.8 us against 24.3, 27.4, 30.4 and
// 60.9 so, the mean of 4 states, and of a million symbols 46 to 134 against 26 to 225;
// with top_k they cost 3 to 63 us below a million symbols. Not taken: the sizes do not
// tell the two apart, and which filters a call has was not made part of the rule. kProbe:
// 1.5, 2 and 2.5 deviations took 48.2, 50.6 and 58 us for both kernels at 128 rows of
// 131,075 normal logits; other sizes and distributions were not tried.
constexpr uint32_t kColumn = 12, kTogether = 2;
constexpr float kProbe = 1.5f;
struct Column {
    float z[kColumn][64], key[kColumn][64];
    uint32_t at[kColumn][64];
};

template <class T>
__global__ __launch_bounds__(kMostWaves * 64) void leo_sample_settle(LeoSample a, uint32_t spans, const SpanRecord* records) {
    __shared__ SampleShared shared;
    __shared__ Column columns[kMostWaves];
    constexpr uint32_t kWide = Span<T>::kWide, kLoads = kEach / kWide;
    const uint64_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t n = static_cast<uint32_t>(a.symbols);
    const Rules r = rules_of(a, row);
    records += row * spans;
    const auto* logits = static_cast<const typename T::type*>(a.logits) + row * a.logits_stride;
    const float* noise = a.noise + row * a.noise_stride;
    // every wave takes all records: no wave waits for another
    float top = negative_infinity(), mass = 0.0f, sum = 0.0f, squares = 0.0f;
    uint32_t counted = 0;
    Racer best = nobody();
#pragma unroll 2
    for (uint32_t i = lane; i < spans; i += 64) {
        const SpanRecord rec = records[i];
        if (rec.top == negative_infinity()) continue;
        const float higher = fmaxf(top, rec.top);
        mass = (top > negative_infinity() ? mass * mass_of(top, higher) : 0.0f) + rec.mass * mass_of(rec.top, higher);
        top = higher;
        best.meet(rec.best.key, rec.best.at, rec.best.z);
        counted += 1;
        sum += rec.top;
        squares += rec.top * rec.top;
    }
    const float mine = top;
    top = wave_max(top);
    mass = wave_sum(mine > negative_infinity() ? mass * mass_of(mine, top) : 0.0f);
    const Search s = {top, mass, top, wave_race(best)};
    // The value that is tried first, with a few of each span's above it: kProbe
    // standard deviations below the mean of the spans' largest, or where min_p
    // cuts.
    float probe = negative_infinity();
    if (s.open(r)) {
        const float count = static_cast<float>(wave_sum(counted)), mean = wave_sum(sum) / count;
        probe = mean - kProbe * sqrtf(fmaxf(wave_sum(squares) / count - mean * mean, 0.0f));
        if (r.min_p > 0.0f) probe = fmaxf(probe, top + logf(r.min_p) * 1.0001f - 0.0001f);
    }

    Column& column = columns[wave];
    uint32_t filled = 0;            // of this lane's column
    float held = __builtin_inff();  // the wave's columns hold all there is above this
    settle(a, r, row, s, probe, shared, [&](float low, float high, Above (&above)[2]) {
        const auto weigh = [&] {
            for (uint32_t c = 0; __any(c < filled); ++c)
                if (c < filled) add_above(low, high, top, column.z[c][lane], column.key[c][lane], column.at[c][lane], above);
        };
        if (low >= held) return weigh();
        const auto weigh_logits = [&] {  // their noise comes all at once
            float race[kColumn];
#pragma unroll
            for (uint32_t c = 0; c < kColumn; ++c)
                if (c < filled) race[c] = noise[column.at[c][lane]];
#pragma unroll
            for (uint32_t c = 0; c < kColumn; ++c)
                if (c < filled) {
                    const float z = r.divided(column.z[c][lane]);
                    column.z[c][lane] = z;
                    column.key[c][lane] = z + race[c];
                }
            weigh();
        };
        // z above low needs a logit above this, whatever the division rounds
        const float cut = __builtin_amdgcn_fmed3f(low * r.t, -kMost, kMost), least = cut - (fabsf(cut) * 0x1p-20f + 0x1p-120f);
        held = low;
        filled = 0;
        for (uint32_t from = wave; from < spans; from += kMostWaves * 64) {
            const uint32_t mine = from + lane * kMostWaves;
            uint64_t left = __ballot(mine < spans && records[min(mine, spans - 1)].top > low);
            while (left) {
                uint32_t base[kTogether];
                bool some[kTogether];
                uint4v raw[kTogether][kLoads];
#pragma unroll
                for (uint32_t u = 0; u < kTogether; ++u) {  // in flight together
                    some[u] = left != 0;
                    if (!some[u]) continue;
                    base[u] = (from + static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(left)) - 1) * kMostWaves) * kSpan;
                    left &= left - 1;
#pragma unroll
                    for (uint32_t v = 0; v < kLoads; ++v) raw[u][v] = load_row<T>(logits, Span<T>::index(base[u], v * kWide), n);
                }
#pragma unroll
                for (uint32_t u = 0; u < kTogether; ++u) {
                    if (!some[u]) continue;
#pragma unroll
                    for (uint32_t i = 0; i < kEach; ++i) {
                        if (i % 4 == 0 && __any(filled > kColumn - 4)) {
                            weigh_logits();
                            filled = 0;
                            held = __builtin_inff();
                        }
                        const float logit = T::at(raw[u][i / kWide], i % kWide);
                        if (logit > least) {
                            column.z[filled][lane] = logit;
                            column.at[filled][lane] = Span<T>::index(base[u], i);
                            filled += 1;
                        }
                    }
                }
            }
        }
        weigh_logits();
    });
}

struct SamplePlan {
    uint32_t spans;
    bool whole;  // leo_sample_row takes a row at once
    uint64_t workspace;
};
SamplePlan sample_plan(uint64_t rows, uint64_t symbols) {
    SamplePlan p{};
    p.spans = static_cast<uint32_t>((symbols + kSpan - 1) / kSpan);
    p.whole = p.spans <= kMostWaves;
    p.workspace = p.whole ? 0 : rows * p.spans * sizeof(SpanRecord);
    return p;
}

template <class T>
void launch_sample(const SamplePlan& p, const LeoSample& s, hipStream_t stream) {
    const uint32_t rows = static_cast<uint32_t>(s.rows);
    if (p.whole) return launch(leo_sample_row<T>, dim3(rows), dim3(p.spans * 64), 0, stream, s);
    auto* records = static_cast<SpanRecord*>(s.workspace);
    launch(leo_sample_spans<T>, dim3((p.spans + 3) / 4, rows), dim3(256), 0, stream, s, p.spans, records);
    launch(leo_sample_settle<T>, dim3(rows), dim3(kMostWaves * 64), 0, stream, s, p.spans, static_cast<const SpanRecord*>(records));
}

}  // namespace
}  // namespace leo

using namespace leo;

extern "C" {

int32_t leo_control_logits(const LeoLogitControl* control, void* stream) {
    return guarded([&] {
        require(control, "leo_control_logits: null argument");
        const LeoLogitControl& c = *control;
        require(valid_type(c.type), "leo_control_logits: unknown type");
        require(c.rows <= 65535, "leo_control_logits: too many rows");
        require(c.symbols <= 0x7fffffffu, "leo_control_logits: too many symbols");
        if (c.rows == 0 || c.symbols == 0) return;
        require(c.logits && c.out, "leo_control_logits: null argument");
        require(c.logits_stride >= 0, "leo_control_logits: logits_stride must not be negative");
        require(c.rows == 1 || c.out_stride >= static_cast<int64_t>(c.symbols), "leo_control_logits: out_stride is too small");
        require((c.out == c.logits && (c.rows == 1 || c.out_stride == c.logits_stride)) ||
                    !overlap(rows_of(c.logits, c.rows, c.symbols, c.logits_stride, c.type),
                             rows_of(c.out, c.rows, c.symbols, c.out_stride, c.type)),
                "leo_control_logits: out overlaps the logits without being them");
        require(!c.history_offsets || c.history || c.history_count == 0, "leo_control_logits: offsets without a history");
        require(!c.bias_offsets || (c.bias_ids && c.bias_values) || c.bias_count == 0,
                "leo_control_logits: offsets without biases");
        require(c.bias_count < 0xffffffffu, "leo_control_logits: too many biases");
        if (c.masks) {
            require(c.mask_count >= 1, "leo_control_logits: masks without rows");
            require(c.masks_stride >= 0, "leo_control_logits: masks_stride must not be negative");
            require(c.mask_rows || c.mask_count == 1 || c.mask_count == c.rows,
                    "leo_control_logits: masks need one row, a row for each of the logits, or mask_rows");
        } else {  // an empty table has no memory: it must not open what its rows' numbers shut
            require(c.mask_count == 0 && !c.mask_rows, "leo_control_logits: mask_count or mask_rows without masks");
        }
        // Chunks small enough for some 512 workgroups, but of 2,048 symbols at least (each reads the row's lists
        // again) and of a table's size at most: 16 symbols a thread.
        const uint64_t least = (c.symbols + kTable - 1) / kTable, most = (c.symbols + 2047) / 2048;
        const uint64_t chunks = std::max(least, std::min(most, (512 + c.rows - 1) / c.rows));
        const uint32_t chunk = static_cast<uint32_t>(((c.symbols + chunks - 1) / chunks + 63) / 64 * 64);
        const dim3 grid(static_cast<uint32_t>((c.symbols + chunk - 1) / chunk), static_cast<uint32_t>(c.rows));
        const auto kernel = c.type == LEO_TYPE_F32   ? leo_control_rows<F32>
                            : c.type == LEO_TYPE_F16 ? leo_control_rows<F16>
                                                     : leo_control_rows<BF16>;
        launch(kernel, grid, dim3(chunk > 8192 ? kControlThreads : chunk > 4096 ? kControlThreads / 2 : kControlThreads / 4), chunk * 4, static_cast<hipStream_t>(stream), c, chunk);
    });
}

int32_t leo_sample_workspace_bytes(uint64_t rows, uint64_t symbols, uint64_t* bytes) {
    return guarded([&] {
        require(bytes, "leo_sample_workspace_bytes: null argument");
        require(rows <= 65535 && symbols <= 0x7fffffffu, "leo_sample_workspace_bytes: too many rows or symbols");
        *bytes = sample_plan(rows, symbols).workspace;
    });
}

int32_t leo_sample(const LeoSample* sample, void* stream) {
    return guarded([&] {
        require(sample, "leo_sample: null argument");
        const LeoSample& s = *sample;
        require(valid_type(s.type), "leo_sample: unknown type");
        require(s.rows <= 65535, "leo_sample: too many rows");
        require(s.symbols <= 0x7fffffffu, "leo_sample: too many symbols");
        if (s.rows == 0) return;
        require(s.symbols >= 1, "leo_sample: no symbols to draw from");
        require(s.logits && s.out_symbols && s.out_logprobs, "leo_sample: null argument");
        require(s.logits_stride >= 0 && s.noise_stride >= 0, "leo_sample: strides must not be negative");
        const SamplePlan p = sample_plan(s.rows, s.symbols);
        require(p.workspace == 0 || (s.workspace && reinterpret_cast<uintptr_t>(s.workspace) % 256 == 0 &&
                                     s.workspace_bytes >= p.workspace),
                "leo_sample: workspace is missing, too small or not 256-byte aligned");
        const auto at = static_cast<hipStream_t>(stream);
        if (s.type == LEO_TYPE_F32) launch_sample<F32>(p, s, at);
        else if (s.type == LEO_TYPE_F16) launch_sample<F16>(p, s, at);
        else launch_sample<BF16>(p, s, at);
    });
}

}  // extern "C"
