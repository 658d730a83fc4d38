// Matrix-vector products with 4-bit weights and group scales, and the layout
// they read.
//
//     y[m, n] = bias[n] + sum_k x[m, k] s[n, k/G] (u[n, k] - z[n, k/G])
//
// Layout. Outputs go in tiles of 16, inputs in blocks of 128; the codes of one
// tile and block are 1,024 bytes, 16 for each lane of a wave: lane l holds
// output l % 16 and, in dword j, the eight inputs 32 j + 8 (l / 16) + 0..7 of
// the block, so that dword j of a wave is the 32 x 16 operand of one matrix
// instruction. Half byte p of a dword is input 2p, half byte 4 + p input 2p+1:
// one AND leaves two neighbours in the two halves of a register. Blocks of one
// tile follow each other, so a wave that walks a tile reads one stream. Scales
// (and zeros) have the same order: [tile][block][output % 16][group of the
// block]. Outputs and inputs beyond the matrix have scale 0 and the zero's code.
#include <algorithm>

#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kTile = 16, kBlock = 128, kBlockBytes = 1024;
constexpr uint64_t kMostRows = 1 << 20;

struct Q4Layout {
    uint64_t tiles, blocks;
    uint32_t groups;      // of a block
    uint32_t zero_bytes;  // of an output's block: half bytes, one a group
    uint64_t scales, zeros, bytes;  // offsets of the parts, and the whole
};

void check_shape(const LeoQ4Shape& s) {
    require(s.outputs >= 1 && s.outputs <= (1ull << 31), "q4: outputs must be 1 .. 2^31");
    require(s.inputs >= 1 && s.inputs <= (1ull << 31), "q4: inputs must be 1 .. 2^31");
    require(s.group == 32 || s.group == 64 || s.group == 128, "q4: group must be 32, 64 or 128");
    require(valid_type(s.scale_type), "q4: unknown scale type");
}

Q4Layout layout_of(const LeoQ4Shape& s) {
    const auto up = [](uint64_t v) { return (v + 255) / 256 * 256; };
    Q4Layout l;
    l.tiles = (s.outputs + kTile - 1) / kTile;
    l.blocks = (s.inputs + kBlock - 1) / kBlock;
    l.groups = kBlock / s.group;
    l.zero_bytes = s.has_zeros ? (l.groups + 1) / 2 : 0;
    l.scales = l.tiles * l.blocks * kBlockBytes;
    l.zeros = l.scales + up(l.tiles * l.blocks * kTile * l.groups * type_bytes(s.scale_type));
    l.bytes = l.zeros + up(l.tiles * l.blocks * kTile * l.zero_bytes);
    return l;
}

struct LayoutArgs {
    LeoQ4Source src;
    Q4Layout l;
};

__device__ __forceinline__ uint32_t source_zero(const LeoQ4Source& s, uint64_t n, uint64_t group) {
    return s.zeros ? static_cast<const uint8_t*>(s.zeros)[n * s.zeros_stride + group] & 15u : 8u;
}

// One workgroup a tile and block, one lane a dword quadruple.
__global__ __launch_bounds__(64) void leo_q4_lay_out(LayoutArgs a) {
    const LeoQ4Source& s = a.src;
    const uint64_t at = blockIdx.x + static_cast<uint64_t>(blockIdx.y) * gridDim.x;
    if (at >= a.l.tiles * a.l.blocks) return;
    const uint64_t tile = at / a.l.blocks, block = at % a.l.blocks;
    const uint32_t lane = threadIdx.x;
    const uint64_t n = tile * kTile + lane % kTile;
    const bool output = n < s.shape.outputs;
    uint32_t words[4];
    for (uint32_t j = 0; j < 4; ++j) {
        uint32_t word = 0;
        for (uint32_t i = 0; i < 8; ++i) {
            const uint64_t k = block * kBlock + 32 * j + 8 * (lane / kTile) + i;
            uint32_t code = 0;
            if (output && k < s.shape.inputs) {
                code = static_cast<const uint8_t*>(s.codes)[n * s.codes_stride + k / 2] >> (4 * (k % 2)) & 15u;
            } else if (output && k / s.shape.group * s.shape.group < s.shape.inputs) {
                code = source_zero(s, n, k / s.shape.group);
            }
            word |= code << (4 * (i / 2 + 4 * (i % 2)));
        }
        words[j] = word;
    }
    uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(s.layout) + at * kBlockBytes);
    to[lane] = make_uint4(words[0], words[1], words[2], words[3]);
    if (lane >= kTile) return;
    uint32_t zeros = 0;
    for (uint32_t g = 0; g < a.l.groups; ++g) {
        const uint64_t group = (block * kBlock) / s.shape.group + g;
        const bool inside = output && group * s.shape.group < s.shape.inputs;
        const uint64_t to_scale = (at * kTile + lane) * a.l.groups + g;
        char* scales = static_cast<char*>(s.layout) + a.l.scales;
        if (s.shape.scale_type == LEO_TYPE_F32) {
            reinterpret_cast<float*>(scales)[to_scale] =
                inside ? static_cast<const float*>(s.scales)[n * s.scales_stride + group] : 0.0f;
        } else {
            reinterpret_cast<uint16_t*>(scales)[to_scale] =
                inside ? static_cast<const uint16_t*>(s.scales)[n * s.scales_stride + group] : uint16_t{0};
        }
        zeros |= (inside ? source_zero(s, n, group) : 0u) << (4 * g);
    }
    char* to_zero = static_cast<char*>(s.layout) + a.l.zeros + (at * kTile + lane) * a.l.zero_bytes;
    if (a.l.zero_bytes == 1) *reinterpret_cast<uint8_t*>(to_zero) = static_cast<uint8_t>(zeros);
    if (a.l.zero_bytes == 2) *reinterpret_cast<uint16_t*>(to_zero) = static_cast<uint16_t>(zeros);
}

__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int32_t type) {
    if (type == LEO_TYPE_F32) F32::store(p, i, v);
    else if (type == LEO_TYPE_F16) F16::store(p, i, v);
    else BF16::store(p, i, v);
}

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

struct TileArgs {
    const char* codes;
    const char* scales;
    const char* zeros;
    const void* x;
    int64_t x_stride;
    const float* bias;
    void* y;
    int64_t y_stride;
    int32_t y_type;
    uint32_t scale_bf16;
    uint32_t rows, inputs, outputs, tiles, blocks;
    uint32_t slices, slice_blocks;
    uint32_t row_bits, stage_blocks;  // of leo_q4_few: its rows rounded up to a power of two, blocks of x in LDS at a time
    float* partials;  // [slice][row][16 tiles], where there are several slices
    const half8* ready;
    const float* factors;
    uint32_t row_tiles;
};

// Eight neighbouring inputs of a row, as the type has them in memory.
template <class X>
struct Eight {
    uint4v w[sizeof(typename X::type) / 2];
};

template <class X>
__device__ __forceinline__ Eight<X> load_eight(const void* x, int64_t at) {
    Eight<X> v;
    __builtin_memcpy(&v, static_cast<const typename X::type*>(x) + at, sizeof(v));  // rows need no alignment
    return v;
}

// The first `inside` of them (a row's end); the others are 0.
template <class X>
__device__ __forceinline__ Eight<X> load_some(const void* x, int64_t at, int32_t inside) {
    union {
        Eight<X> v;
        typename X::type e[8];
    } u;
#pragma unroll
    for (int32_t i = 0; i < 8; ++i)
        u.e[i] = i < inside ? static_cast<const typename X::type*>(x)[at + i] : typename X::type(0.0f);
    return u.v;
}

__device__ __forceinline__ void widen(const Eight<F32>& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v.w[i / 4][i % 4]);
}
__device__ __forceinline__ void widen(const Eight<BF16>& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(v.w[0][i] << 16);
        f[2 * i + 1] = __uint_as_float(v.w[0][i] & 0xffff0000u);
    }
}

// The largest exponent field of a row's finite values among a block's 128.
template <class X>
__device__ __forceinline__ uint32_t top_exponent(const Eight<X> (&v)[4]) {
    uint32_t most = 0, finite = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float f[8];
        widen(v[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);
    }
    if (__any(most >= 0x7f800000u)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[8];
            widen(v[j], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
                finite = max(finite, b < 0x7f800000u ? b : 0u);
            }
        }
        most = finite;
    }
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
    return max(most >> 23, 15u);
}

// Half precision halves of x * factor: the value to 11 bits and, of a 32-bit x,
// the 11 below them. With the block's largest at 2^14 .. 2^15 and half precision's
// smallest at 2^-24, a bfloat16 x is exact down to 2^-31 of the largest, and nothing
// is further off than its last bit or 2^-39 of the largest: a third half would add
// half as many matrix instructions for bits that a float sum of a block drops too,
// unless the largest meet weights of 0.
template <class X, int kParts>
__device__ __forceinline__ void halves(const Eight<X>& v, float factor, half8 (&a)[kParts]) {
    float f[8];
    widen(v, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = f[i] * factor;
        const _Float16 high = static_cast<_Float16>(s);
        a[0][i] = high;
        if constexpr (kParts == 2) {
            const float low = s - static_cast<float>(high);
            a[1][i] = static_cast<_Float16>(low == low ? low : 0.0f);  // infinity - infinity
        }
    }
}

// word & mask | high in one instruction: two constants in one need a register,
// which the compiler does not spend by itself.
__device__ __forceinline__ uint32_t and_or(uint32_t word, uint32_t mask, uint32_t high) {
    uint32_t v;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(v) : "v"(word), "s"(mask), "v"(high));
    return v;
}

// Four pairs of codes less their zero, exactly, by the known way of placing a whole
// number in a float's last bits: in half precision 1024 + u is the bits 0x6400 | u
// and 1024 + 16 u the bits 0x6400 | u << 4.
__device__ __forceinline__ half8 weights_of(uint32_t word, half2 minus, half2 minus_high) {
    const half2 sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    union {
        uint32_t w[4];
        half2 h[4];
        half8 v;
    } u;
    const uint32_t next = word >> 8;
    u.w[0] = and_or(word, 0x000f000fu, 0x64006400u);
    u.w[1] = and_or(word, 0x00f000f0u, 0x64006400u);
    u.w[2] = and_or(next, 0x000f000fu, 0x64006400u);
    u.w[3] = and_or(next, 0x00f000f0u, 0x64006400u);
    u.h[0] = u.h[0] + minus;
    u.h[1] = __builtin_elementwise_fma(u.h[1], sixteenth, minus_high);
    u.h[2] = u.h[2] + minus;
    u.h[3] = __builtin_elementwise_fma(u.h[3], sixteenth, minus_high);
    return u.v;
}

// The scales and zeros of one tile's block as bits, and its codes.
template <int kGroups, bool kZero, bool kWide>
struct WeightBlock {
    static constexpr int kScaleWords = kWide ? kGroups : (kGroups + 1) / 2;
    uint4v code;
    uint32_t scale[kScaleWords];
    uint32_t zero;

    // `at` is the same for the whole wave: its addresses are a scalar and an
    // offset that stays.
    __device__ __forceinline__ void load(const TileArgs& a, uint64_t at, uint32_t lane) {
        const uint32_t column = lane % kTile;
        code = reinterpret_cast<const uint4v*>(a.codes + at * kBlockBytes)[lane];
        const char* of_block = a.scales + at * (kTile * kGroups * (kWide ? 4 : 2));
        if constexpr (!kWide && kGroups == 1) {
            scale[0] = reinterpret_cast<const uint16_t*>(of_block)[column];
        } else {
            __builtin_memcpy(scale, __builtin_assume_aligned(of_block + column * (kGroups * (kWide ? 4 : 2)), sizeof(scale)),
                             sizeof(scale));
        }
        if constexpr (kZero) {
            if constexpr (kGroups == 4) zero = reinterpret_cast<const uint16_t*>(a.zeros + at * (kTile * 2))[column];
            else zero = reinterpret_cast<const uint8_t*>(a.zeros + at * kTile)[column];
        }
    }
    // `bf16` has every bit set where the scales are bf16; a branch here would
    // part the matrix instructions of one group from the next's.
    __device__ __forceinline__ float scale_of(int g, uint32_t bf16) const {
        if constexpr (kWide) {
            return __uint_as_float(scale[g]);
        } else {
            const uint32_t bits = scale[g / 2] >> (16 * (g % 2));
            const uint32_t half = __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits))));
            return __uint_as_float((bits << 16 & bf16) | (half & ~bf16));
        }
    }
    // The 8 weights of a lane in matrix instruction j of the block.
    __device__ __forceinline__ half8 weights(int j) const {
        half2 minus = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
        half2 minus_high = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
        if constexpr (kZero) {
            // -(1024 + z) and -(64 + z) are the bits 0xe400 | z and 0xd400 | z << 4
            const uint32_t z = zero >> (j * kGroups / 4 * 4) & 15u, both = z | z << 16;
            minus = __builtin_bit_cast(half2, both | 0xe400e400u);
            minus_high = __builtin_bit_cast(half2, both << 4 | 0xd400d400u);
        }
        return weights_of(code[j], minus, minus_high);
    }
};

// A lane's share of 16 rows (or rows times blocks) and 128 inputs of x on its
// way to LDS: inputs 32 j + 8 (lane / 16) + 0..7.
template <class X>
struct XBlock {
    static constexpr bool kScaled = !__is_same(X, F16);  // x goes to half precision by a power of two a row and block
    static constexpr int kParts = __is_same(X, F32) ? 2 : 1;
    static constexpr bool kWhole = false;
    Eight<X> v[4];

    static __device__ __forceinline__ int64_t place(const TileArgs& a, uint32_t row, uint32_t block, uint32_t quad) {
        return min(row, a.rows - 1) * a.x_stride + static_cast<int64_t>(block) * kBlock + quad * 8;
    }
    // A block inside the row.
    __device__ __forceinline__ void load(const TileArgs& a, uint32_t row, uint32_t block, uint32_t quad) {
        const int64_t at = place(a, row, block, quad);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load_eight<X>(a.x, at + 32 * j);
    }
    // The block in which it ends.
    __device__ __forceinline__ void load_last(const TileArgs& a, uint32_t row, uint32_t block, uint32_t quad) {
        const int64_t at = place(a, row, block, quad);
        const int32_t inside = static_cast<int32_t>(a.inputs - block * kBlock) - 8 * static_cast<int32_t>(quad);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load_some<X>(a.x, at + 32 * j, inside - 32 * j);
    }
    // Writes part p of instruction j to at(p, j); returns the factor that takes
    // sums over the block back to x's values. Lanes of one row take part together.
    template <class At>
    __device__ __forceinline__ float store(At&& at) const {
        if constexpr (kScaled) {
            // the largest value of the row's block goes to 2^14 .. 2^15, below half precision's end
            const uint32_t e = top_exponent<X>(v);
            const float factor = __uint_as_float((268u - e) << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                half8 h[kParts];
                halves<X, kParts>(v[j], factor, h);
#pragma unroll
                for (int p = 0; p < kParts; ++p) *at(p, j) = h[p];
            }
            return __uint_as_float((e - 14u) << 23);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) *at(0, j) = __builtin_bit_cast(half8, v[j].w[0]);
            return 1.0f;
        }
    }
};

// x as leo_q4_prepare leaves it: [block][16 rows][part][instruction][lane], then
// the factors [block][row].
template <int kPartsOf, bool kScaledOf>
struct Ready {};

template <int kPartsOf, bool kScaledOf>
struct XBlock<Ready<kPartsOf, kScaledOf>> {
    static constexpr bool kScaled = kScaledOf;
    static constexpr int kParts = kPartsOf;
    static constexpr bool kWhole = true;  // a row's end is filled up
    half8 v[kParts][4];
    float factor;

    static __device__ __forceinline__ uint64_t place(const TileArgs& a, uint32_t row, uint32_t block) {
        return static_cast<uint64_t>(block) * a.row_tiles + row / 16;
    }
    __device__ __forceinline__ void load(const TileArgs& a, uint32_t row, uint32_t block, uint32_t) {
        const half8* from = a.ready + place(a, row, block) * (kParts * 256) + threadIdx.x % 64;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[p][j] = from[(p * 4 + j) * 64];
        if constexpr (kScaled) factor = a.factors[place(a, row, block) * 16 + row % 16];
    }
    template <class At>
    __device__ __forceinline__ float store(At&& at) const {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int p = 0; p < kParts; ++p) *at(p, j) = v[p][j];
        return kScaled ? factor : 1.0f;
    }
};

// Brings x into that form once for all workgroups of a product: one wave 16 rows
// of a block. A launch bounds it: 3 to 4.2 us for 64 rows of 5,001.
template <class X>
__global__ __launch_bounds__(256) void leo_q4_prepare(TileArgs a, half8* ready, float* factors) {
    const uint32_t lane = threadIdx.x % 64, block = blockIdx.x, tile = blockIdx.y * 4 + threadIdx.x / 64;
    if (tile >= a.row_tiles) return;
    const uint32_t row = tile * 16 + lane % 16, quad = lane / 16;
    XBlock<X> x;
    if ((block + 1) * kBlock <= a.inputs) x.load(a, row, block, quad);
    else x.load_last(a, row, block, quad);
    const uint64_t place = static_cast<uint64_t>(block) * a.row_tiles + tile;
    half8* to = ready + place * (XBlock<X>::kParts * 256) + lane;
    const float factor = x.store([&](uint32_t p, uint32_t j) { return to + (p * 4 + j) * 64; });
    if (XBlock<X>::kScaled && quad == 0) factors[place * 16 + lane] = factor;
}

// Few rows: one workgroup takes kFewTiles tiles of 16 outputs and a slice of
// the inputs, its eight waves the slice's blocks in turn. x goes through LDS
// once a workgroup, in the order in which matrix instructions take it; the 16
// row lanes of a staging wave cover several blocks, so that no lane converts a
// row that is not there. Instructions bound it, not memory: a tile and block of
// 1,024 bytes of codes takes 60 to 90 of them to widen the codes and apply the
// scales, while the matrix instructions have 15 of 16 rows idle. One row of 1,048,576
// float32 inputs to 257 outputs (147 MB) takes 35.7 us, 4.1 TB/s; 8,192 to 8,192 in
// bfloat16 (35 MB) 9.6 us, 3.6 TB/s; 1,024 to 257 a launch, 4.7 us. Two tiles a
// workgroup: x is brought into LDS half as often.
constexpr uint32_t kFewWaves = 8, kAhead = 2, kFewTiles = 2;

template <class X, int kGroups, bool kZero, bool kWide>
__global__ __launch_bounds__(kFewWaves * 64) void leo_q4_few(TileArgs a) {
    constexpr bool kScaled = XBlock<X>::kScaled;
    constexpr int kParts = XBlock<X>::kParts;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x % 64, wave = wave_of_workgroup();
    const uint32_t column = lane % 16, quad = lane / 16;
    const uint32_t bits = a.row_bits;
    const uint32_t begin = blockIdx.y * a.slice_blocks, end = min(begin + a.slice_blocks, a.blocks);
    const uint32_t back_rows = max(1u << bits, 4u);
    half8* parts = reinterpret_cast<half8*>(lds);
    float* back = reinterpret_cast<float*>(lds + a.stage_blocks * (kParts * 16u << bits) * sizeof(half8));
    const auto part_at = [&](uint32_t block, uint32_t part, uint32_t j, uint32_t q) {
        return (((block * kParts + part) * 4 + j) * 4 + q) << bits;
    };
    uint64_t tile_at[kFewTiles];
#pragma unroll
    for (uint32_t t = 0; t < kFewTiles; ++t)
        tile_at[t] = static_cast<uint64_t>(min(blockIdx.x * kFewTiles + t, a.tiles - 1)) * a.blocks;
    float4v sum[kFewTiles] = {};
    for (uint32_t from = begin; from < end; from += a.stage_blocks) {
        const uint32_t to = min(from + a.stage_blocks, end);
        WeightBlock<kGroups, kZero, kWide> ring[kAhead][kFewTiles];
        // Loads run on past the stage's end, to its last block again: a load under a condition would make every wait one
        // for all of them.
        const auto load_weights = [&](uint32_t u, uint32_t block) {
#pragma unroll
            for (uint32_t t = 0; t < kFewTiles; ++t) ring[u][t].load(a, tile_at[t] + min(block, to - 1), lane);
        };
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) load_weights(u, from + wave + u * kFewWaves);
        if (from != begin) __syncthreads();
        const uint32_t row = column & ((1u << bits) - 1), ahead = column >> bits, step = 16u >> bits;
        for (uint32_t first = from + wave * step; first < to; first += kFewWaves * step) {
            const uint32_t block = first + ahead, in_stage = block - from;
            if (block < to) {
                XBlock<X> x;
                if ((block + 1) * kBlock <= a.inputs) x.load(a, row, block, quad);
                else x.load_last(a, row, block, quad);
                const float factor = x.store([&](uint32_t p, uint32_t j) { return parts + part_at(in_stage, p, j, quad) + row; });
                if (kScaled && quad == 0) back[in_stage * back_rows + row] = factor;
            }
        }
        __syncthreads();
        const uint32_t read_row = min(column, (1u << bits) - 1);
        for (uint32_t first = from + wave; first < to; first += kAhead * kFewWaves) {
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                const uint32_t block = first + u * kFewWaves;
                if (block < to) {
                    const uint32_t in_stage = block - from;
                    float4v whole[kFewTiles] = {};
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        float4v d[kFewTiles] = {};
#pragma unroll
                        for (int j = g * 4 / kGroups; j < (g + 1) * 4 / kGroups; ++j) {
                            half8 w[kFewTiles];
#pragma unroll
                            for (uint32_t t = 0; t < kFewTiles; ++t) w[t] = ring[u][t].weights(j);
#pragma unroll
                            for (int p = 0; p < kParts; ++p) {
                                const half8 v = parts[part_at(in_stage, p, j, quad) + read_row];
#pragma unroll
                                for (uint32_t t = 0; t < kFewTiles; ++t)
                                    d[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[t], d[t], 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (uint32_t t = 0; t < kFewTiles; ++t) {
                            const float scale = ring[u][t].scale_of(g, a.scale_bf16);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if constexpr (kScaled) whole[t][i] = __builtin_fmaf(scale, d[t][i], whole[t][i]);
                                else sum[t][i] = __builtin_fmaf(scale, d[t][i], sum[t][i]);
                            }
                        }
                    }
                    if constexpr (kScaled) {
                        const float4v f = *reinterpret_cast<const float4v*>(back + in_stage * back_rows + 4 * min(quad, back_rows / 4 - 1));
#pragma unroll
                        for (uint32_t t = 0; t < kFewTiles; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[t][i] = __builtin_fmaf(f[i], whole[t][i], sum[t][i]);
                    }
                }
                load_weights(u, block + kAhead * kFewWaves);
            }
        }
    }

    // register i of a lane is output 16 tile + column and row 4 quad + i; wave t ends up with tile t's sums
    float4v* joined = reinterpret_cast<float4v*>(lds);
    const uint32_t tile = blockIdx.x * kFewTiles + wave, output = tile * kTile + column;
    const bool mine = wave < kFewTiles && output < a.outputs;
    __syncthreads();
#pragma unroll
    for (uint32_t t = 0; t < kFewTiles; ++t) joined[(t * kFewWaves + wave) * 64 + lane] = sum[t];
    __syncthreads();
    if (!mine) return;
    float4v v = {};
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w) v += joined[(wave * kFewWaves + w) * 64 + lane];
    const float bias = a.bias && a.slices == 1 ? a.bias[output] : 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = quad * 4 + i;
        if (row >= a.rows) continue;
        if (a.slices == 1) store_any(a.y, row * a.y_stride + output, v[i] + bias, a.y_type);
        else a.partials[(static_cast<uint64_t>(blockIdx.y) * a.rows + row) * (a.tiles * kTile) + output] = v[i];
    }
}

// More rows: one workgroup takes 16 kRows rows, eight tiles of outputs (two a
// wave) and a slice of the inputs. x goes through two buffers in LDS that the
// four waves share, each wave bringing 16 rows of one block a step, so a step is
// 4 / kRows blocks; codes go straight to registers, some blocks ahead. A weight is
// widened once for all 16 kRows rows. 8 rows of 131,072 bfloat16 inputs to 257 outputs
// (20 MB) take 12.5 us: the way in and out of 441 short workgroups, and 257 outputs are
// 17 tiles in 24 places, of which 7 read and multiply the last tile again. 64 rows
// of 5,001 to 11,007 (7 GFLOP) 21.4 us, 330 TFLOP/s, bound by the some 420 vector
// instructions of a step at two waves a SIMD, which the registers allow; its 430
// workgroups leave 82 of the 256 CUs with one where the others have two.
constexpr uint32_t kManyWaves = 4, kManyTiles = 2;

template <class X, int kGroups, bool kZero, bool kWide, int kRows>
__global__ __launch_bounds__(kManyWaves * 64, 2) void leo_q4_many(TileArgs a) {
    constexpr bool kScaled = XBlock<X>::kScaled;
    constexpr int kParts = XBlock<X>::kParts;
    constexpr uint32_t kRing = kRows == 4 ? 2 : 4;  // blocks ahead, as the registers allow
    constexpr uint32_t kStep = kManyWaves / kRows, kSteps = kRing / kStep;
    constexpr uint32_t kSets = kSteps == 1 ? 1 : 2;  // steps of x on their way; one is enough where a step is long
    __shared__ half8 parts[2][kStep][kRows][kParts][4][64];
    __shared__ __attribute__((aligned(16))) float back[2][kStep][kRows * 16];
    const uint32_t lane = threadIdx.x % 64, wave = wave_of_workgroup();
    const uint32_t column = lane % 16, quad = lane / 16;
    const uint32_t tile0 = (blockIdx.x * kManyWaves + wave) * kManyTiles, row0 = blockIdx.z * kRows * 16;
    const uint32_t begin = blockIdx.y * a.slice_blocks, end = min(begin + a.slice_blocks, a.blocks);
    const uint32_t my_block = wave / kRows, my_rows = wave % kRows;  // of a step
    uint64_t tile_at[kManyTiles];
#pragma unroll
    for (uint32_t t = 0; t < kManyTiles; ++t) tile_at[t] = static_cast<uint64_t>(min(tile0 + t, a.tiles - 1)) * a.blocks;

    // Blocks inside the row go through the pipeline, the one in which it ends after it. Loads run on past the last
    // block, to that one again: a load under a condition would make every wait one for all of them.
    const uint32_t full = XBlock<X>::kWhole ? end : min(end, a.inputs / kBlock);
    XBlock<X> x[kSets];
    const auto load_x = [&](XBlock<X>& v, uint32_t block) {
        v.load(a, row0 + my_rows * 16 + column, min(block + my_block, full - 1), quad);
    };
    const auto stage = [&](const XBlock<X>& v, uint32_t buffer) {
        const float factor = v.store([&](uint32_t p, uint32_t j) { return &parts[buffer][my_block][my_rows][p][j][lane]; });
        if (kScaled && quad == 0) back[buffer][my_block][my_rows * 16 + column] = factor;
    };
    float4v sum[kManyTiles][kRows] = {};
    WeightBlock<kGroups, kZero, kWide> ring[kRing][kManyTiles];
    const auto load_weights = [&](uint32_t u, uint32_t block) {
#pragma unroll
        for (uint32_t t = 0; t < kManyTiles; ++t) ring[u][t].load(a, tile_at[t] + block, lane);
    };
    const auto multiply = [&](uint32_t u, uint32_t buffer, uint32_t b) {
        float4v whole[kManyTiles][kRows] = {};
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            float4v d[kManyTiles][kRows] = {};
#pragma unroll
            for (int j = g * 4 / kGroups; j < (g + 1) * 4 / kGroups; ++j) {
                half8 w[kManyTiles];
#pragma unroll
                for (uint32_t t = 0; t < kManyTiles; ++t) w[t] = ring[u][t].weights(j);
#pragma unroll
                for (int m = 0; m < kRows; ++m)
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        const half8 v = parts[buffer][b][m][p][j][lane];
#pragma unroll
                        for (uint32_t t = 0; t < kManyTiles; ++t)
                            d[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[t], d[t][m], 0, 0, 0);
                    }
            }
#pragma unroll
            for (uint32_t t = 0; t < kManyTiles; ++t) {
                const float scale = ring[u][t].scale_of(g, a.scale_bf16);
#pragma unroll
                for (int m = 0; m < kRows; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (kScaled) whole[t][m][i] = __builtin_fmaf(scale, d[t][m][i], whole[t][m][i]);
                        else sum[t][m][i] = __builtin_fmaf(scale, d[t][m][i], sum[t][m][i]);
                    }
            }
        }
        if constexpr (kScaled) {
#pragma unroll
            for (int m = 0; m < kRows; ++m) {
                const float4v f = *reinterpret_cast<const float4v*>(&back[buffer][b][m * 16 + quad * 4]);
#pragma unroll
                for (uint32_t t = 0; t < kManyTiles; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[t][m][i] = __builtin_fmaf(f[i], whole[t][m][i], sum[t][m][i]);
            }
        }
    };
    if (begin < full) {
        load_x(x[0], begin);
        if constexpr (kSets == 2) load_x(x[1], begin + kStep);
#pragma unroll
        for (uint32_t u = 0; u < kRing; ++u) load_weights(u, min(begin + u, full - 1));
        stage(x[0], 0);
        __syncthreads();
        uint32_t odd = 0;  // the buffer of a round of one step
        for (uint32_t block = begin; block < full; block += kRing, odd ^= 1) {
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                const uint32_t at = block + s * kStep, buffer = kSets == 2 ? s % 2 : odd;
                if (at >= full) break;
                load_x(x[s % kSets], at + kSets * kStep);
#pragma unroll
                for (uint32_t b = 0; b < kStep; ++b) {
                    if (at + b < full) multiply(s * kStep + b, buffer, b);
                    load_weights(s * kStep + b, min(at + b + kRing, full - 1));
                }
                stage(x[(s + 1) % kSets], 1 - buffer);
                __syncthreads();
            }
        }
    }
    if constexpr (!XBlock<X>::kWhole) {
        if (full < end && begin <= full) {
            load_weights(0, full);
            if (my_block == 0) {
                x[0].load_last(a, row0 + my_rows * 16 + column, full, quad);
                stage(x[0], 0);
            }
            __syncthreads();
            multiply(0, 0, 0);
        }
    }

    // register (t, m, i) of a lane is output 16 (tile0 + t) + column and row 16 m + 4 quad + i
#pragma unroll
    for (uint32_t t = 0; t < kManyTiles; ++t) {
        const uint32_t output = (tile0 + t) * kTile + column;
        if (output >= a.outputs) continue;
        const float bias = a.bias && a.slices == 1 ? a.bias[output] : 0.0f;
#pragma unroll
        for (uint32_t m = 0; m < kRows; ++m)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t row = row0 + m * 16 + quad * 4 + i;
                if (row >= a.rows) continue;
                if (a.slices == 1) store_any(a.y, row * a.y_stride + output, sum[t][m][i] + bias, a.y_type);
                else a.partials[(static_cast<uint64_t>(blockIdx.y) * a.rows + row) * (a.tiles * kTile) + output] = sum[t][m][i];
            }
    }
}

// Adds the slices of 256 / kLanes outputs of one row, kLanes threads an output,
// always in the same order, so that results do not depend on which workgroup ends
// first. A launch bounds it (3.8 to 4.8 us); joining in the last workgroup to arrive
// cost 4 to 7 us, and up to 40 with 64 slices, for its waits on stores and its atomics.
template <uint32_t kLanes>
__global__ __launch_bounds__(256) void leo_q4_join(TileArgs a) {
    constexpr uint32_t kOutputs = 256 / kLanes;
    __shared__ float joined[kLanes][kOutputs];
    const uint32_t output = blockIdx.x * kOutputs + threadIdx.x % kOutputs, part = threadIdx.x / kOutputs;
    const uint32_t row = blockIdx.y;
    const uint32_t width = a.tiles * kTile;
    float sum = 0.0f;
    if (output < a.outputs) {
        const float* at = a.partials + static_cast<uint64_t>(row) * width + output;
        const uint64_t step = static_cast<uint64_t>(a.rows) * width;
        for (uint32_t s = part; s < a.slices; s += kLanes * 8) {
            float v[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u)  // in flight together
                v[u] = at[min(s + u * kLanes, a.slices - 1) * step];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) sum += s + u * kLanes < a.slices ? v[u] : 0.0f;
        }
    }
    if constexpr (kLanes > 1) {
        joined[part][threadIdx.x % kOutputs] = sum;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (uint32_t p = 1; p < kLanes; ++p) sum += joined[p][threadIdx.x];
    }
    if (output < a.outputs)
        store_any(a.y, row * a.y_stride + output, sum + (a.bias ? a.bias[output] : 0.0f), a.y_type);
}

// Both sides of these rules, in us, codes in groups of 64:
// kFewRows   2 rows of 131,072 inputs to 257 outputs: few 11.2 (float32) and 9.8 (bfloat16), many 15.3 and 13.1; 4 rows
//            12.6 and 10.7 against 15.9 and 13.5; 8 rows 17.0 and 12.1 against 15.6 and 13.4. 8,192 to 8,192: 2 rows
//            13.2 and 9.8 against 15.3 and 12.9, 4 rows 17.4 and 12.2 against 15.9 and 13.4, 8 rows 28.2 and 15.7
//            against 16.6 and 13.7.
// k..Groups  256, 512 and 1,024 workgroups aimed at: one row of 1,048,576 to 257 46.2, 41.6 and 42.5, 8 rows 72.8, 63.4
//            and 69.8; 64 rows of 5,000 to 11,007 31.1, 26.2 and 31.7; one row of 131,072 to 257 10.9, 11.2 and 12.5.
//            512 are what two workgroups a CU take at once: 516 need a second turn.
constexpr uint32_t kStageBytes = 64 << 10, kFewGroups = 512, kManyGroups = 512, kFewRows = 4;

struct Plan {
    bool few;         // leo_q4_few, else leo_q4_many
    uint32_t rows;    // of 16, of one workgroup
    uint32_t groups, slabs, slices, slice_blocks;
    uint32_t row_bits, stage_blocks, lds;
    uint64_t ready, factors, workspace;  // places in the workspace, after the slices' sums
};

Plan plan_of(const LeoQ4Shape& s, uint64_t rows, int32_t x_type) {
    const Q4Layout l = layout_of(s);
    const uint32_t blocks = static_cast<uint32_t>(l.blocks);
    const auto over = [](uint64_t n, uint64_t d) { return static_cast<uint32_t>((n + d - 1) / d); };
    Plan p{};
    p.few = rows <= kFewRows;
    if (p.few) {
        const uint32_t parts = x_type == LEO_TYPE_F32 ? 2 : 1;
        p.rows = 1;
        p.slabs = 1;
        p.groups = over(l.tiles, kFewTiles);
        while ((1u << p.row_bits) < rows) ++p.row_bits;
        const uint32_t block_bytes = (parts * 256 << p.row_bits) + 4 * std::max(1u << p.row_bits, 4u);
        const uint32_t most = std::max(kFewWaves, (kStageBytes / block_bytes) / kFewWaves * kFewWaves);
        p.slices = p.groups >= kFewGroups / 4 ? 1 : std::min(kFewGroups / p.groups, std::max(1u, blocks / (kFewWaves * 2)));
        p.slice_blocks = over(blocks, p.slices);
        p.stage_blocks = std::min(p.slice_blocks, most);
        p.lds = std::max(p.stage_blocks * block_bytes, kFewTiles * kFewWaves * 64 * 16);
    } else {
        p.rows = rows <= 16 ? 1 : rows <= 32 || x_type == LEO_TYPE_F32 ? 2 : 4;
        p.slabs = over(rows, 16 * p.rows);
        p.groups = over(l.tiles, kManyWaves * kManyTiles);
        p.slices = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(kManyGroups / (static_cast<uint64_t>(p.groups) * p.slabs), blocks / 4)));
    }
    p.slice_blocks = over(blocks, p.slices);
    p.slices = over(blocks, p.slice_blocks);
    const auto up = [](uint64_t v) { return (v + 255) / 256 * 256; };
    p.ready = p.factors = p.workspace = p.slices == 1 ? 0 : up(4ull * p.slices * rows * l.tiles * kTile);
    if (p.rows > 1 && x_type != LEO_TYPE_F32) {  // where its rows turn out not to be aligned
        const uint64_t places = static_cast<uint64_t>(blocks) * p.slabs * p.rows;
        p.factors = p.ready + places * 4096;
        p.workspace = p.factors + (x_type == LEO_TYPE_F16 ? 0 : places * 64);
    }
    return p;
}

template <class X, int kGroups, bool kZero, bool kWide>
void launch_tiles(const Plan& p, const TileArgs& a, hipStream_t stream) {
    using Prepared = Ready<XBlock<X>::kParts, XBlock<X>::kScaled>;
    const dim3 grid(p.groups, p.slices, p.slabs), block(kManyWaves * 64);
    if (p.few) return launch(leo_q4_few<X, kGroups, kZero, kWide>, grid, dim3(kFewWaves * 64), p.lds, stream, a);
    if (p.rows == 1) return launch(leo_q4_many<X, kGroups, kZero, kWide, 1>, grid, block, 0, stream, a);
    if constexpr (!__is_same(X, F32)) {
        if (a.ready && p.rows == 2) return launch(leo_q4_many<Prepared, kGroups, kZero, kWide, 2>, grid, block, 0, stream, a);
        if (a.ready) return launch(leo_q4_many<Prepared, kGroups, kZero, kWide, 4>, grid, block, 0, stream, a);
        if (p.rows == 4) return launch(leo_q4_many<X, kGroups, kZero, kWide, 4>, grid, block, 0, stream, a);
    }
    launch(leo_q4_many<X, kGroups, kZero, kWide, 2>, grid, block, 0, stream, a);
}

template <class X, int kGroups>
void launch_groups(const LeoQ4Shape& s, const Plan& p, const TileArgs& a, hipStream_t stream) {
    const bool wide = s.scale_type == LEO_TYPE_F32;
    if (s.has_zeros && wide) launch_tiles<X, kGroups, true, true>(p, a, stream);
    else if (s.has_zeros) launch_tiles<X, kGroups, true, false>(p, a, stream);
    else if (wide) launch_tiles<X, kGroups, false, true>(p, a, stream);
    else launch_tiles<X, kGroups, false, false>(p, a, stream);
}

template <class X>
void launch_products(const LeoQ4Shape& s, const Plan& p, const TileArgs& a, hipStream_t stream) {
    if constexpr (!__is_same(X, F32))
        if (a.ready) launch(leo_q4_prepare<X>, dim3(a.blocks, (a.row_tiles + 3) / 4), dim3(256), 0, stream, a,
                            const_cast<half8*>(a.ready), const_cast<float*>(a.factors));
    if (s.group == 32) launch_groups<X, 4>(s, p, a, stream);
    else if (s.group == 64) launch_groups<X, 2>(s, p, a, stream);
    else launch_groups<X, 1>(s, p, a, stream);
}

}  // namespace
}  // namespace leo

using namespace leo;

extern "C" {

int32_t leo_q4_layout_bytes(const LeoQ4Shape* shape, uint64_t* bytes) {
    return guarded([&] {
        require(shape && bytes, "leo_q4_layout_bytes: null argument");
        check_shape(*shape);
        *bytes = layout_of(*shape).bytes;
    });
}

int32_t leo_q4_layout(const LeoQ4Source* source, void* stream) {
    return guarded([&] {
        require(source, "leo_q4_layout: null argument");
        const LeoQ4Source& s = *source;
        check_shape(s.shape);
        LayoutArgs a{s, layout_of(s.shape)};
        require(s.codes && s.scales && s.layout, "leo_q4_layout: null argument");
        require(!s.shape.has_zeros == !s.zeros, "leo_q4_layout: has_zeros and zeros disagree");
        require(s.codes_stride >= static_cast<int64_t>((s.shape.inputs + 1) / 2), "leo_q4_layout: codes_stride is too small");
        const int64_t groups = static_cast<int64_t>((s.shape.inputs + s.shape.group - 1) / s.shape.group);
        require(s.scales_stride >= groups && (!s.zeros || s.zeros_stride >= groups),
                "leo_q4_layout: scales_stride or zeros_stride is too small");
        require(reinterpret_cast<uintptr_t>(s.layout) % 256 == 0, "leo_q4_layout: layout must be 256-byte aligned");
        require(s.layout_bytes >= a.l.bytes, "leo_q4_layout: layout is too small");
        const uint64_t count = a.l.tiles * a.l.blocks;
        const uint32_t wide = static_cast<uint32_t>(count < 65536 ? count : 65536);
        launch(leo_q4_lay_out, dim3(wide, static_cast<uint32_t>((count + wide - 1) / wide)), dim3(64),
               0, static_cast<hipStream_t>(stream), a);
    });
}

int32_t leo_q4_workspace_bytes(const LeoQ4Shape* shape, uint64_t rows, int32_t x_type, uint64_t* bytes) {
    return guarded([&] {
        require(shape && bytes, "leo_q4_workspace_bytes: null argument");
        check_shape(*shape);
        require(rows <= kMostRows, "leo_q4_workspace_bytes: too many rows");
        require(valid_type(x_type), "leo_q4_workspace_bytes: unknown type");
        *bytes = rows ? plan_of(*shape, rows, x_type).workspace : 0;
    });
}

int32_t leo_q4_matvec(const LeoQ4Product* product, void* stream) {
    return guarded([&] {
        require(product, "leo_q4_matvec: null argument");
        const LeoQ4Product& p = *product;
        check_shape(p.shape);
        if (p.rows == 0) return;
        require(p.rows <= kMostRows, "leo_q4_matvec: too many rows");
        require(valid_type(p.x_type) && valid_type(p.y_type), "leo_q4_matvec: unknown type");
        require(p.layout && p.x && p.y, "leo_q4_matvec: null argument");
        require(p.x_stride >= 0, "leo_q4_matvec: x_stride must not be negative");
        require(p.y_stride >= static_cast<int64_t>(p.shape.outputs) || p.rows == 1, "leo_q4_matvec: y_stride is too small");
        const Rows y = rows_of(p.y, p.rows, p.shape.outputs, p.y_stride, p.y_type);
        require(!overlap(rows_of(p.x, p.rows, p.shape.inputs, p.x_stride, p.x_type), y), "leo_q4_matvec: y overlaps x");
        require(!meets_bias(p.bias, y, p.shape.outputs, p.y_type), "leo_q4_matvec: y overlaps the bias");
        require(reinterpret_cast<uintptr_t>(p.layout) % 256 == 0, "leo_q4_matvec: layout must be 256-byte aligned");
        const Q4Layout l = layout_of(p.shape);
        require(p.layout_bytes >= l.bytes, "leo_q4_matvec: layout is too small for its shape");
        const Plan plan = plan_of(p.shape, p.rows, p.x_type);
        require(plan.workspace == 0 || (p.workspace && reinterpret_cast<uintptr_t>(p.workspace) % 256 == 0 &&
                                        p.workspace_bytes >= plan.workspace),
                "leo_q4_matvec: workspace is missing, too small or not 256-byte aligned");
        const char* layout = static_cast<const char*>(p.layout);
        TileArgs a{};
        a.codes = layout;
        a.scales = layout + l.scales;
        a.zeros = layout + l.zeros;
        a.x = p.x;
        a.x_stride = p.x_stride;
        a.bias = p.bias;
        a.y = p.y;
        a.y_stride = p.y_stride;
        a.y_type = p.y_type;
        a.scale_bf16 = p.shape.scale_type == LEO_TYPE_BF16 ? ~0u : 0u;
        a.rows = static_cast<uint32_t>(p.rows);
        a.inputs = static_cast<uint32_t>(p.shape.inputs);
        a.outputs = static_cast<uint32_t>(p.shape.outputs);
        a.tiles = static_cast<uint32_t>(l.tiles);
        a.blocks = static_cast<uint32_t>(l.blocks);
        a.slices = plan.slices;
        a.slice_blocks = plan.slice_blocks;
        a.row_bits = plan.row_bits;
        a.stage_blocks = plan.stage_blocks;
        char* space = static_cast<char*>(p.workspace);
        a.partials = reinterpret_cast<float*>(space);
        // Loads of 16 bytes are fast at multiples of 4 only, and eight tiles a workgroup read x again for each: 64 rows of
        // 5,001 16-bit inputs against 11,007 outputs took 43 us, and 30 with x brought into place first, 5,000 inputs 28
        // and 29.
        if (plan.rows > 1 && p.x_type != LEO_TYPE_F32 && (reinterpret_cast<uintptr_t>(p.x) % 4 || p.x_stride % 2)) {
            a.ready = reinterpret_cast<const half8*>(space + plan.ready);
            a.factors = reinterpret_cast<const float*>(space + plan.factors);
        }
        a.row_tiles = plan.slabs * plan.rows;
        const auto at = static_cast<hipStream_t>(stream);
        if (p.x_type == LEO_TYPE_F32) launch_products<F32>(p.shape, plan, a, at);
        else if (p.x_type == LEO_TYPE_F16) launch_products<F16>(p.shape, plan, a, at);
        else launch_products<BF16>(p.shape, plan, a, at);
        if (plan.slices == 1) return;
        const bool many = plan.slices >= 16;  // slices enough to share among threads
        // slices are several only where groups times slabs are half of kManyGroups at most: 16,384 rows
        const uint32_t outputs = many ? 32 : 256;
        const dim3 grid((a.outputs + outputs - 1) / outputs, a.rows);
        launch(many ? leo_q4_join<8> : leo_q4_join<1>, grid, dim3(256), 0, at, a);
    });
}

}  // extern "C"
