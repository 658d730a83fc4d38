// Control of a row's logits and the draw of its next symbol.
#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kChunk = 4096;  // logits of one workgroup of the control

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

// One workgroup a row and chunk of symbols: it counts the row's history over
// its chunk in LDS (whole-number adds, whose order does not matter), notes the
// last bias entry of each symbol, and passes once over the logits.
template <class T>
__global__ __launch_bounds__(256) void leo_control_rows(LeoLogitControl a) {
    __shared__ uint32_t count[kChunk];
    __shared__ uint32_t bias_at[kChunk];  // last entry + 1, counted from the row's first
    const uint64_t row = blockIdx.y;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kChunk;
    const int64_t width = min(static_cast<int64_t>(kChunk), static_cast<int64_t>(a.symbols) - base);
    for (uint32_t i = threadIdx.x; i < kChunk; i += 256) count[i] = bias_at[i] = 0;
    __syncthreads();
    const Run history = row_run(a.history_offsets, row, a.history_count);
    for (int64_t i = history.begin + threadIdx.x; i < history.end; i += 256) {
        const int64_t at = a.history[i] - base;
        if (at >= 0 && at < width) atomicAdd(&count[at], 1u);
    }
    const Run bias = row_run(a.bias_offsets, row, a.bias_count);
    for (int64_t i = bias.begin + threadIdx.x; i < bias.end; i += 256) {
        const int64_t at = a.bias_ids[i] - base;
        if (at >= 0 && at < width) atomicMax(&bias_at[at], static_cast<uint32_t>(i - bias.begin) + 1);
    }
    __syncthreads();
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
    for (int64_t i = threadIdx.x; i < width; i += 256) {
        const int64_t v = base + i;
        float z = T::load(a.logits, row * a.logits_stride + v);
        if (const uint32_t c = count[i]) {
            z = z > 0.0f ? z / repetition : z * repetition;
            z = z - (presence + frequency * static_cast<float>(c));
        }
        if (const uint32_t b = bias_at[i]) z = z + a.bias_values[bias.begin + b - 1];
        if (shut || (mask && !(static_cast<uint32_t>(mask[v / 32]) >> (v % 32) & 1u))) z = negative_infinity();
        T::store(a.out, row * a.out_stride + v, z);
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

constexpr uint32_t kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;

struct SampleShared {
    Racer racer[kSampleWaves];
    float value[kSampleWaves];
    uint32_t count[kSampleWaves];
};

__device__ Racer block_racer(Racer r, SampleShared& s) {
    for (uint32_t d = 32; d; d /= 2) r.meet(__shfl_xor(r.key, d), __shfl_xor(r.at, d), __shfl_xor(r.z, d));
    __syncthreads();
    if (threadIdx.x % 64 == 0) s.racer[threadIdx.x / 64] = r;
    __syncthreads();
    for (uint32_t w = 0; w < kSampleWaves; ++w) r.meet(s.racer[w].key, s.racer[w].at, s.racer[w].z);
    return r;
}
__device__ float block_max(float v, SampleShared& s) {
    for (uint32_t d = 32; d; d /= 2) v = fmaxf(v, __shfl_xor(v, d));
    __syncthreads();
    if (threadIdx.x % 64 == 0) s.value[threadIdx.x / 64] = v;
    __syncthreads();
    for (uint32_t w = 0; w < kSampleWaves; ++w) v = fmaxf(v, s.value[w]);
    return v;
}
__device__ float block_sum(float v, SampleShared& s) {
    for (uint32_t d = 32; d; d /= 2) v += __shfl_xor(v, d);
    __syncthreads();
    if (threadIdx.x % 64 == 0) s.value[threadIdx.x / 64] = v;
    __syncthreads();
    float sum = 0.0f;
    for (uint32_t w = 0; w < kSampleWaves; ++w) sum += s.value[w];
    return sum;
}
__device__ uint32_t block_count(uint32_t v, SampleShared& s) {
    for (uint32_t d = 32; d; d /= 2) v += __shfl_xor(v, d);
    __syncthreads();
    if (threadIdx.x % 64 == 0) s.count[threadIdx.x / 64] = v;
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t w = 0; w < kSampleWaves; ++w) sum += s.count[w];
    return sum;
}

// One workgroup a row. What stays is a prefix of the values in falling order,
// so one value decides: the race's winner over the whole row is the answer if
// it stays; if not, no value up to its own stays, and the race is held again
// above. A second value halfway (in the order of floats) to the lowest one known to stay is tried in
// the same pass, which bounds the passes by the 32 bits of a float.
template <class T>
__global__ __launch_bounds__(kSampleThreads) void leo_sample_rows(LeoSample a) {
    __shared__ SampleShared shared;
    const uint64_t row = blockIdx.x;
    const uint32_t n = static_cast<uint32_t>(a.symbols);
    const float t = a.noise ? (a.temperature ? a.temperature[row] : 1.0f) : 0.0f;
    const bool greedy = !(t > 0.0f);
    const float divide = greedy ? 1.0f : t;
    const auto value = [&](uint32_t i) {
        const float z = T::load(a.logits, row * a.logits_stride + i) / divide;
        return z == z ? z : negative_infinity();
    };
    const float* noise = a.noise ? a.noise + row * a.noise_stride : nullptr;
    Racer best = nobody();
    float top = negative_infinity();
    for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads) {
        const float z = value(i);
        top = fmaxf(top, z);
        if (z > negative_infinity()) best.meet(greedy ? z : z + noise[i], i, z);
    }
    top = block_max(top, shared);
    best = block_racer(best, shared);
    const auto mass_of = [&](float z) { return z == top ? 1.0f : expf(z - top); };
    float whole = 0.0f;
    if (top > negative_infinity())
        for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads) whole += mass_of(value(i));
    whole = block_sum(whole, shared);
    if (top == negative_infinity()) {
        if (threadIdx.x == 0) {
            a.out_symbols[row] = -1;
            a.out_logprobs[row] = negative_infinity();
        }
        return;
    }
    if (!greedy) {
        const uint32_t k = a.top_k ? static_cast<uint32_t>(max(a.top_k[row], 1)) : n;
        const float p = a.top_p ? a.top_p[row] : 1.0f;
        const float floor_p = a.min_p ? a.min_p[row] : 0.0f;
        float lowest = top;  // of the values known to stay
        while (best.z < lowest) {
            const float low = best.z;
            const uint32_t key = order_key(low);
            const float high = from_order_key(key + (order_key(lowest) - key) / 2);
            uint32_t larger[2] = {0, 0};
            float mass[2] = {0.0f, 0.0f};
            Racer next[2] = {nobody(), nobody()};
            for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads) {
                const float z = value(i);
                if (!(z > low)) continue;
                const float w = mass_of(z), race = z + noise[i];
                larger[0] += 1;
                mass[0] += w;
                next[0].meet(race, i, z);
                if (!(z > high)) continue;
                larger[1] += 1;
                mass[1] += w;
                next[1].meet(race, i, z);
            }
            const auto stays = [&](float z, uint32_t above, float before) {
                return above < k && (p >= 1.0f || before < p * whole) && mass_of(z) >= floor_p;
            };
            for (int h = 0; h < 2; ++h) {
                larger[h] = block_count(larger[h], shared);
                mass[h] = block_sum(mass[h], shared);
                next[h] = block_racer(next[h], shared);
            }
            if (stays(low, larger[0], mass[0])) break;
            if (stays(high, larger[1], mass[1])) {
                lowest = high;
                best = next[0];
            } else {
                best = next[1];
            }
        }
    }
    if (threadIdx.x == 0) {
        a.out_symbols[row] = static_cast<int32_t>(best.at);
        a.out_logprobs[row] = (best.z == top ? 0.0f : best.z - top) - logf(whole);
    }
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
        require(!c.history_offsets || c.history || c.history_count == 0, "leo_control_logits: offsets without a history");
        require(!c.bias_offsets || (c.bias_ids && c.bias_values) || c.bias_count == 0,
                "leo_control_logits: offsets without biases");
        require(c.bias_count < 0xffffffffu, "leo_control_logits: too many biases");
        if (c.masks) {
            require(c.mask_count >= 1, "leo_control_logits: masks without rows");
            require(c.masks_stride >= 0, "leo_control_logits: masks_stride must not be negative");
            require(c.mask_rows || c.mask_count == 1 || c.mask_count == c.rows,
                    "leo_control_logits: masks need one row, a row for each of the logits, or mask_rows");
        }
        const dim3 grid(static_cast<uint32_t>((c.symbols + kChunk - 1) / kChunk), static_cast<uint32_t>(c.rows));
        const auto kernel = c.type == LEO_TYPE_F32   ? leo_control_rows<F32>
                            : c.type == LEO_TYPE_F16 ? leo_control_rows<F16>
                                                     : leo_control_rows<BF16>;
        launch(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), c);
    });
}

int32_t leo_sample_workspace_bytes(uint64_t rows, uint64_t symbols, uint64_t* bytes) {
    return guarded([&] {
        require(bytes, "leo_sample_workspace_bytes: null argument");
        require(rows <= 65535 && symbols <= 0x7fffffffu, "leo_sample_workspace_bytes: too many rows or symbols");
        *bytes = 0;
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
        const auto kernel = s.type == LEO_TYPE_F32   ? leo_sample_rows<F32>
                            : s.type == LEO_TYPE_F16 ? leo_sample_rows<F16>
                                                     : leo_sample_rows<BF16>;
        launch(kernel, dim3(static_cast<uint32_t>(s.rows)), dim3(kSampleThreads), 0, static_cast<hipStream_t>(stream), s);
    });
}

}  // extern "C"
