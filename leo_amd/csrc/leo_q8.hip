// Products with 8-bit weights and 8-bit activations, and the layout they read.
//
//     y[m, n] = bias[n] + s[m] c[n] sum_k q[m, k] w[n, k]
//     s[m] = max(max_k |x[m, k]| * float(1 / 127), 2^-126),  q[m, k] = round(x[m, k] / s[m])
//
// Layout. Rows (outputs of the weights, rows of x) go in tiles of 16, inputs in
// blocks of 64; the codes of one tile and block are 1,024 bytes, 16 for each lane
// of a wave: lane l holds row l % 16, inputs 16 (l / 16) + 0..15 of the block, which
// is its operand of one matrix instruction (16x16x64). Blocks of one tile follow
// each other. Behind the weights' codes stand their scales as floats, 16 a tile.
// Rows and inputs beyond the matrix are 0.
#include <algorithm>

#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kTile = 16, kBlock = 64, kBlockBytes = 1024;
constexpr uint64_t kMostRows = 1 << 20;
// Products are 128 * 127 at most: sums over so many blocks stay inside 32 bits.
constexpr uint32_t kMostSliceBlocks = 131072 / kBlock;

typedef int32_t int4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

struct Q8Layout {
    uint64_t tiles, blocks;
    uint64_t scales, bytes;  // the scales' offset, and the whole
};

void check_shape(const LeoQ8Shape& s) {
    require(s.outputs >= 1 && s.outputs <= (1ull << 31), "q8: outputs must be 1 .. 2^31");
    require(s.inputs >= 1 && s.inputs <= (1ull << 27), "q8: inputs must be 1 .. 2^27");
}

uint64_t up(uint64_t v) { return (v + 255) / 256 * 256; }

Q8Layout layout_of(const LeoQ8Shape& s) {
    Q8Layout l;
    l.tiles = (s.outputs + kTile - 1) / kTile;
    l.blocks = (s.inputs + kBlock - 1) / kBlock;
    l.scales = l.tiles * l.blocks * kBlockBytes;
    l.bytes = l.scales + up(l.tiles * kTile * sizeof(float));
    return l;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int32_t type) {
    return type == LEO_TYPE_F32 ? F32::load(p, i) : type == LEO_TYPE_F16 ? F16::load(p, i) : BF16::load(p, i);
}

// One wave a tile and block, one lane its 16 bytes.
__global__ __launch_bounds__(64) void leo_q8_lay_out(LeoQ8Source s, Q8Layout l) {
    const uint64_t at = blockIdx.x + static_cast<uint64_t>(blockIdx.y) * gridDim.x;
    if (at >= l.tiles * l.blocks) return;
    const uint64_t tile = at / l.blocks, block = at % l.blocks;
    const uint32_t lane = threadIdx.x;
    const uint64_t n = tile * kTile + lane % kTile, k = block * kBlock + lane / kTile * 16;
    union {
        uint4v words;
        int8_t codes[16];
    } u;
    u.words = uint4v{0, 0, 0, 0};
    if (n < s.shape.outputs) {
        const int8_t* row = static_cast<const int8_t*>(s.codes) + n * s.codes_stride;
        if (k + 16 <= s.shape.inputs) u.words = load_16(row + k);
        else for (uint32_t i = 0; i < 16; ++i)
            if (k + i < s.shape.inputs) u.codes[i] = row[k + i];
    }
    reinterpret_cast<uint4v*>(static_cast<char*>(s.layout) + at * kBlockBytes)[lane] = u.words;
    if (block == 0 && lane < kTile)
        reinterpret_cast<float*>(static_cast<char*>(s.layout) + l.scales)[n] =
            n < s.shape.outputs ? load_any(s.scales, static_cast<int64_t>(n), s.scale_type) : 0.0f;
}

struct ProductArgs {
    const char* codes;
    const float* scales;
    const void* x;
    int64_t x_stride;
    const float* bias;
    void* y;
    int64_t y_stride;
    int32_t y_type;
    uint32_t rows, inputs, outputs, tiles, blocks, row_tiles;
    uint32_t slices, slice_blocks;
    uint32_t parts, part_inputs;  // of a row, whose largest magnitudes were taken before; 0: none were
    const uint32_t* largest;      // [row][part], bits of magnitudes
    char* x_codes;                // x as a layout; what is beyond its rows and inputs holds anything: those
                                  // rows' sums are not used, and the weights of those inputs are 0
    float* x_scales;              // one a row
    int32_t* partials;            // [slice][row][16 tiles]
};

__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
    return wave_reduce(v, 0u, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
}

// 16 neighbouring inputs of a row from k on; 0 beyond its end.
struct Sixteen {
    float f[16];
};
template <class X>
__device__ __forceinline__ Sixteen load_sixteen(const ProductArgs& a, uint32_t row, uint32_t k) {
    constexpr uint32_t kWide = 16 / sizeof(typename X::type);
    const auto* p = static_cast<const typename X::type*>(a.x) + static_cast<int64_t>(row) * a.x_stride + k;
    Sixteen s;
    if (k + 16 <= a.inputs) {
        uint4v raw[16 / kWide];
#pragma unroll
        for (uint32_t v = 0; v < 16 / kWide; ++v) raw[v] = load_16(p + v * kWide);
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) s.f[i] = X::at(raw[i / kWide], i % kWide);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) s.f[i] = k + i < a.inputs ? X::load(p, i) : 0.0f;
    }
    return s;
}
__device__ __forceinline__ uint32_t largest_of(const Sixteen& s) {
    uint32_t most = 0;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) most = max(most, __float_as_uint(s.f[i]) & 0x7fffffffu);
    return most;
}

// The scale of a row from the largest magnitude of its values, as bits; NaN where that is no finite number.
__device__ __forceinline__ float scale_of(uint32_t largest) {
    return largest < 0x7f800000u ? fmaxf(__uint_as_float(largest) * (1.0f / 127.0f), 0x1p-126f) : __builtin_nanf("");
}

// The whole numbers nearest to the exact quotients x / s, of two the even one. The sum
// with 1.5 * 2^23 of x and the rounded inverse rounds to a whole number once and has it in
// its last byte. The inverse is off by 2^-24 of itself, so a quotient of 127 at most by
// less than 2^-16: only where one lies as near to a half, as in some 3% of waves, twice the
// remainder x - n s tells, held against s: near s / 2 neither it nor its double needs rounding,
// whereas half of a scale below 2^-125 may.
__device__ __forceinline__ uint4v codes_of(const Sixteen& s, float scale) {
    constexpr float kMagic = 12582912.0f;
    const float inverse = 1.0f / scale;
    float number[16], off = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
        number[i] = __builtin_fmaf(s.f[i], inverse, kMagic);
        off = fmaxf(off, fabsf(__builtin_fmaf(s.f[i], inverse, kMagic - number[i])));
    }
    if (__any(off > 0.5f - 0x1p-16f)) {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
            const float n = number[i] - kMagic, rest = __builtin_fmaf(-n, scale, s.f[i]), twice = rest + rest;
            const bool odd = __float_as_uint(number[i]) & 1u;
            if (twice > scale || (twice == scale && odd)) number[i] += 1.0f;
            if (twice < -scale || (twice == -scale && odd)) number[i] -= 1.0f;
        }
    }
    uint4v words;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        const uint32_t low = __builtin_amdgcn_perm(__float_as_uint(number[4 * w + 1]), __float_as_uint(number[4 * w]), 0x0c0c0400);
        const uint32_t high = __builtin_amdgcn_perm(__float_as_uint(number[4 * w + 3]), __float_as_uint(number[4 * w + 2]), 0x04000c0c);
        words[w] = low | high;
    }
    return scale == scale ? words : uint4v{0, 0, 0, 0};
}

// A whole sum as a value: three roundings of 2^-24, of which the second may be of a value
// past the result's, then the one to y's type. 64 bits here took 11 us of a 256 x 256
// tile's time, for bits that the 8-bit x does not have. The row's scale, which alone may be
// next to the smallest float, comes last.
__device__ __forceinline__ float value_of(float sum, float scale, float row_scale, float bias) {
    return __builtin_fmaf(sum * scale, row_scale, bias);
}

__device__ __forceinline__ void store_y(const ProductArgs& a, uint32_t row, uint32_t n, int64_t sum, float scale) {
    const float v = value_of(static_cast<float>(static_cast<double>(sum)), a.scales[n], scale, a.bias ? a.bias[n] : 0.0f);
    const int64_t at = static_cast<int64_t>(row) * a.y_stride + n;
    if (a.y_type == LEO_TYPE_F32) static_cast<float*>(a.y)[at] = static_cast<float>(v);
    else if (a.y_type == LEO_TYPE_F16) static_cast<_Float16*>(a.y)[at] = static_cast<_Float16>(v);
    else static_cast<__bf16*>(a.y)[at] = static_cast<__bf16>(v);
}

// The largest magnitude of each part of a row.
template <class X>
__global__ __launch_bounds__(256) void leo_q8_largest(ProductArgs a, uint32_t* to) {
    __shared__ uint32_t most[4];
    const uint32_t row = blockIdx.x, begin = blockIdx.y * a.part_inputs, end = min(begin + a.part_inputs, a.inputs);
    uint32_t largest = 0;
    for (uint32_t k = begin + threadIdx.x * 16; k < end; k += 256 * 16) largest = max(largest, largest_of(load_sixteen<X>(a, row, k)));
    largest = wave_largest(largest);
    if (threadIdx.x % 64 == 0) most[threadIdx.x / 64] = largest;
    __syncthreads();
    if (threadIdx.x == 0) to[row * a.parts + blockIdx.y] = max(max(most[0], most[1]), max(most[2], most[3]));
}

constexpr uint32_t kMostParts = 256;
__device__ __forceinline__ float scale_of_parts(const ProductArgs& a, uint32_t row) {  // by a whole wave
    const uint32_t lane = threadIdx.x % 64;
    uint32_t largest = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMostParts; i += 64)
        if (i + lane < a.parts) largest = max(largest, a.largest[row * a.parts + i + lane]);
    return scale_of(wave_largest(largest));
}

__device__ __forceinline__ uint4v* place_of(const ProductArgs& a, uint32_t row, uint32_t sixteen) {
    char* to = a.x_codes + (static_cast<uint64_t>(row / kTile) * a.blocks + sixteen / 4) * kBlockBytes;
    return reinterpret_cast<uint4v*>(to) + (sixteen % 4 * kTile + row % kTile);
}

// x in 8 bits in the weights' layout, for the products of many rows: one workgroup a
// row of up to 16,384 inputs, which its threads hold in registers, or a part of a longer one.
// 2,048 rows of 8,192 bfloat16, 50 MB in and out, take 12.5 to 14.2 us.
constexpr uint32_t kHeldInputs = 16384;
template <class X>
__global__ __launch_bounds__(1024) void leo_q8_quantize_row(ProductArgs a) {
    __shared__ uint32_t most[16];
    // Workgroups go to the XCDs in turn: the rows of a tile, which share lines, to one of them.
    const uint32_t turn = blockIdx.x / 8, row = (turn / kTile * 8 + blockIdx.x % 8) * kTile + turn % kTile;
    if (row >= a.rows) return;
    const uint32_t lane = threadIdx.x % 64, k = threadIdx.x * 16;
    const Sixteen s = load_sixteen<X>(a, row, k);
    const uint32_t largest = wave_largest(largest_of(s));
    if (lane == 0) most[threadIdx.x / 64] = largest;
    __syncthreads();
    const float scale = scale_of(wave_largest(lane < blockDim.x / 64 ? most[lane] : 0u));
    if (threadIdx.x == 0) a.x_scales[row] = scale;
    if (k < a.inputs) *place_of(a, row, threadIdx.x) = codes_of(s, scale);
}
template <class X>
__global__ __launch_bounds__(256) void leo_q8_quantize_part(ProductArgs a) {
    const uint32_t row = blockIdx.x, begin = blockIdx.y * a.part_inputs, end = min(begin + a.part_inputs, a.inputs);
    const float scale = scale_of_parts(a, row);
    if (begin == 0 && threadIdx.x == 0) a.x_scales[row] = scale;
    for (uint32_t k = begin + threadIdx.x * 16; k < end; k += 256 * 16) *place_of(a, row, k / 16) = codes_of(load_sixteen<X>(a, row, k), scale);
}

// Up to 16 rows. A workgroup takes kTiles output tiles and a slice of the inputs,
// and brings the slice of x to LDS in 8 bits itself; its eight waves share the
// slice's blocks, each block's weights a run of 1,024 bytes a tile. x is the A
// operand, so lane l gets output l % 16 of rows 4 (l / 16) + 0..3; rows beyond the
// last read it again and are not stored. Whole sums go to LDS by whole-number
// additions, whose order does not matter. The slice of x is asked for before the weights,
// which would stand before it in memory's queue: 13.9 us for 14.7 with 8 rows of 131,072
// -> 257. Memory bounds a long product, 1 row of 1,048,576 -> 257 in 51.5 to 51.9 us for 298 MB (5.7
// TB/s, also where no input is left in the cache beside memory), a launch a short one, 1,024 -> 257 in 4.0.
constexpr uint32_t kFewThreads = 512, kFewWaves = kFewThreads / 64;
constexpr uint32_t kFewStage = 48 << 10;  // bytes of x in LDS

template <class X, int kTiles>
__global__ __launch_bounds__(kFewThreads, 4) void leo_q8_few(ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint4v staged[];
    __shared__ int32_t sums[kTiles * 256];
    __shared__ uint32_t most[16][kFewWaves];
    __shared__ float scales[16];
    constexpr uint32_t kAhead = kTiles >= 5 ? 1 : kTiles >= 3 ? 2 : kTiles == 2 ? 4 : 8;
    const uint32_t lane = threadIdx.x % 64, wave = wave_of_workgroup();
    const uint32_t first = blockIdx.y * a.slice_blocks, count = min(a.slice_blocks, a.blocks - first);
    const uint32_t each = (count + kFewWaves - 1) / kFewWaves;
    const uint32_t begin = min(first + wave * each, first + count), end = min(begin + each, first + count);
    const char* weights[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
        weights[t] = a.codes + static_cast<uint64_t>(min(blockIdx.x * kTiles + t, a.tiles - 1)) * a.blocks * kBlockBytes;
    const auto fetch = [&](int4v (&to)[kAhead][kTiles], uint32_t block) {
        if (block >= end) return;
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                to[u][t] = reinterpret_cast<const int4v*>(weights[t] + static_cast<uint64_t>(min(block + u, end - 1)) * kBlockBytes)[lane];
    };
    int4v even[kAhead][kTiles], odd[kAhead][kTiles];
    const uint32_t each_row = count * 4, sixteens = a.rows * each_row;
    const auto load_staged = [&](uint32_t i) { return load_sixteen<X>(a, i / each_row, (first * 4 + i % each_row) * 16); };
    Sixteen ahead;
    if (threadIdx.x < sixteens) ahead = load_staged(threadIdx.x);
    fetch(even, begin);  // on their way while x is prepared, and behind it
    for (uint32_t i = threadIdx.x; i < kTiles * 256; i += kFewThreads) sums[i] = 0;

    if (a.parts) {
        for (uint32_t row = wave; row < a.rows; row += kFewWaves) {
            const float scale = scale_of_parts(a, row);
            if (lane == 0) scales[row] = scale;
        }
    } else {
        for (uint32_t row = 0; row < a.rows; ++row) {
            uint32_t largest = 0;
            for (uint32_t k = threadIdx.x * 16; k < a.inputs; k += kFewThreads * 16)
                largest = max(largest, largest_of(load_sixteen<X>(a, row, k)));
            largest = wave_largest(largest);
            if (lane == 0) most[row][wave] = largest;
        }
        __syncthreads();
        for (uint32_t row = wave; row < a.rows; row += kFewWaves) {
            const float scale = scale_of(wave_largest(lane < kFewWaves ? most[row][lane] : 0u));
            if (lane == 0) scales[row] = scale;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < sixteens; i += kFewThreads) {
        const uint32_t row = i / each_row, sixteen = i % each_row;
        staged[sixteen * a.rows + row] = codes_of(i == threadIdx.x ? ahead : load_staged(i), scales[row]);
    }
    if (a.slices > 1 && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < a.rows) a.x_scales[threadIdx.x] = scales[threadIdx.x];
    __syncthreads();

    int4v sum[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sum[t] = int4v{0, 0, 0, 0};
    const uint32_t mine = lane / kTile * a.rows + min(lane % kTile, a.rows - 1);
    const auto multiply = [&](const int4v (&w)[kAhead][kTiles], uint32_t block) {
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
            if (block + u >= end) break;
            const int4v x = __builtin_bit_cast(int4v, staged[(block + u - first) * 4 * a.rows + mine]);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, w[u][t], sum[t], 0, 0, 0);
        }
    };
    for (uint32_t block = begin; block < end; block += 2 * kAhead) {
        fetch(odd, block + kAhead);
        multiply(even, block);
        fetch(even, block + 2 * kAhead);
        multiply(odd, block + kAhead);
    }
    if (begin < end) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = lane / kTile * 4 + i;
            if (row >= a.rows) break;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) atomicAdd(&sums[row * (kTiles * kTile) + t * kTile + lane % kTile], sum[t][i]);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.rows * (kTiles * kTile); i += kFewThreads) {
        const uint32_t row = i / (kTiles * kTile), n = blockIdx.x * (kTiles * kTile) + i % (kTiles * kTile);
        if (a.slices > 1) {
            if (n < a.tiles * kTile) a.partials[(static_cast<uint64_t>(blockIdx.y) * a.rows + row) * a.tiles * kTile + n] = sums[i];
        } else if (n < a.outputs) {
            store_y(a, row, n, sums[i], scales[row]);
        }
    }
}

// More rows: 16 kRows rows and 16 kTiles outputs a workgroup, x and the weights
// straight from their layouts to registers, the blocks of a slice shared by eight waves, one
// block ahead (two ahead, or 4 or 16 waves, took as long or longer). 64 rows of 5,001 -> 11,007, 55 MB, take 15.1 us
// with the weights in the cache beside memory and 23 without: 344 workgroups on 256 CUs, and 323 KB of x for each of
// them from L2.
template <int kManyRows, int kManyTiles>
__global__ __launch_bounds__(kFewThreads) void leo_q8_many(ProductArgs a) {
    __shared__ int32_t sums[kManyRows * kManyTiles * 256];
    constexpr uint32_t kOperands = kManyRows + kManyTiles, kWide = kManyTiles * kTile;
    const uint32_t lane = threadIdx.x % 64, wave = wave_of_workgroup();
    const uint32_t first = blockIdx.z * a.slice_blocks, count = min(a.slice_blocks, a.blocks - first);
    const uint32_t each = (count + kFewWaves - 1) / kFewWaves;
    const uint32_t begin = min(first + wave * each, first + count), end = min(begin + each, first + count);
    const char* from[kOperands];
#pragma unroll
    for (uint32_t r = 0; r < kManyRows; ++r)
        from[r] = a.x_codes + static_cast<uint64_t>(min(blockIdx.y * kManyRows + r, a.row_tiles - 1)) * a.blocks * kBlockBytes;
#pragma unroll
    for (uint32_t t = 0; t < kManyTiles; ++t)
        from[kManyRows + t] = a.codes + static_cast<uint64_t>(min(blockIdx.x * kManyTiles + t, a.tiles - 1)) * a.blocks * kBlockBytes;
    const auto fetch = [&](int4v (&to)[kOperands], uint32_t block) {
        if (block >= end) return;
#pragma unroll
        for (uint32_t o = 0; o < kOperands; ++o) to[o] = reinterpret_cast<const int4v*>(from[o] + static_cast<uint64_t>(block) * kBlockBytes)[lane];
    };
    int4v sum[kManyRows][kManyTiles];
#pragma unroll
    for (int r = 0; r < kManyRows; ++r)
#pragma unroll
        for (int t = 0; t < kManyTiles; ++t) sum[r][t] = int4v{0, 0, 0, 0};
    const auto multiply = [&](const int4v (&v)[kOperands], uint32_t block) {
        if (block >= end) return;
#pragma unroll
        for (int r = 0; r < kManyRows; ++r)
#pragma unroll
            for (int t = 0; t < kManyTiles; ++t) sum[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[r], v[kManyRows + t], sum[r][t], 0, 0, 0);
    };
    int4v one[kOperands], two[kOperands];
    fetch(one, begin);
    for (uint32_t i = threadIdx.x; i < kManyRows * kManyTiles * 256; i += kFewThreads) sums[i] = 0;
    __syncthreads();
    for (uint32_t block = begin; block < end; block += 2) {
        fetch(two, block + 1);
        multiply(one, block);
        fetch(one, block + 2);
        multiply(two, block + 1);
    }
    if (begin < end) {
#pragma unroll
        for (int r = 0; r < kManyRows; ++r)
#pragma unroll
            for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    atomicAdd(&sums[(r * kTile + lane / kTile * 4 + i) * kWide + t * kTile + lane % kTile], sum[r][t][i]);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kManyRows * kManyTiles * 256; i += kFewThreads) {
        const uint32_t row = blockIdx.y * (kManyRows * kTile) + i / kWide, n = blockIdx.x * kWide + i % kWide;
        if (row >= a.rows) break;
        if (a.slices > 1) {
            if (n < a.tiles * kTile) a.partials[(static_cast<uint64_t>(blockIdx.z) * a.rows + row) * a.tiles * kTile + n] = sums[i];
        } else if (n < a.outputs) {
            store_y(a, row, n, sums[i], a.x_scales[row]);
        }
    }
}

// Many rows: tiles of both operands go to LDS, in the order of their layouts, some
// steps of 64 inputs ahead, and from there to registers one step ahead. The weights
// are the A operand, so a lane gets four neighbouring outputs of one row. 2,048 rows of
// 8,192 -> 8,192 take 104 to 118 us as the clock goes (2.6 to 2.3 PFLOP/s; the matrix units
// are busy 63% of the cycles): a barrier a step, and 96 KB that eight waves of 64 x 128 sums
// read from LDS in the time of 1,024 cycles of products. Four waves of 128 x 128 sums read 64,
// but one wave a SIMD has nothing to run while it waits: 141 us.
constexpr uint32_t kSlots = 4;  // steps in LDS

// 16 bytes a lane from `from` + `offset` to 1,024 bytes of LDS. The instruction writes
// no register, so nothing can be read before it has come but LDS, whose waits a step
// makes itself. M0 holds the place in LDS.
__device__ __forceinline__ void load_to_lds(uint32_t lds, const char* from, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(from) : "memory", "m0");
}

template <int kN, int kM, int kWavesN, int kWavesM>
struct TileShape {
    static constexpr int kWaves = kWavesN * kWavesM, kOutputs = kN * kWavesN, kRows = kM * kWavesM;  // in tiles of 16
    static constexpr int kLoads = (kOutputs + kRows) / kWaves;  // of a wave and step
    static constexpr uint32_t kSlotBytes = (kOutputs + kRows) * kBlockBytes;
};

template <int kN, int kM, int kWavesN, int kWavesM>
__global__ __launch_bounds__(64 * kWavesN * kWavesM) void leo_q8_tiles(ProductArgs a, uint32_t across) {
    using Shape = TileShape<kN, kM, kWavesN, kWavesM>;
    extern __shared__ __attribute__((aligned(16))) char slots[];
    __shared__ float row_scales[Shape::kRows * kTile];
    const uint32_t lane = threadIdx.x % 64, wave = wave_of_workgroup();
    const uint32_t place = blockIdx.x;
    const uint32_t tile_n = place % across * Shape::kOutputs, tile_m = place / across * Shape::kRows;
    const uint32_t first = blockIdx.y * a.slice_blocks, last = min(first + a.slice_blocks, a.blocks) - 1;
    const float scale_of_row = a.x_scales[min(tile_m * kTile + threadIdx.x, a.rows - 1)];
    const char* from[Shape::kLoads];
#pragma unroll
    for (int j = 0; j < Shape::kLoads; ++j) {
        const uint32_t f = wave * Shape::kLoads + j;
        from[j] = f < Shape::kOutputs ? a.codes + static_cast<uint64_t>(min(tile_n + f, a.tiles - 1)) * a.blocks * kBlockBytes
                                      : a.x_codes + static_cast<uint64_t>(min(tile_m + f - Shape::kOutputs, a.row_tiles - 1)) * a.blocks * kBlockBytes;
    }
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)slots));
    const auto send = [&](uint32_t block, uint32_t slot) {
        const uint32_t offset = min(block, last) * kBlockBytes + lane * 16;
#pragma unroll
        for (int j = 0; j < Shape::kLoads; ++j)
            load_to_lds(base + slot * Shape::kSlotBytes + (wave * Shape::kLoads + j) * kBlockBytes, from[j], offset);
    };
    const uint32_t wave_n = wave % kWavesN * kN, wave_m = Shape::kOutputs + wave / kWavesN * kM;
    const auto read = [&](int4v (&n)[kN], int4v (&m)[kM], uint32_t slot) {
        const char* at = slots + slot * Shape::kSlotBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < kN; ++i) n[i] = *reinterpret_cast<const int4v*>(at + (wave_n + i) * kBlockBytes);
#pragma unroll
        for (int i = 0; i < kM; ++i) m[i] = *reinterpret_cast<const int4v*>(at + (wave_m + i) * kBlockBytes);
    };
    int4v sum[kN][kM];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int m = 0; m < kM; ++m) sum[n][m] = int4v{0, 0, 0, 0};
    const auto multiply = [&](const int4v (&n)[kN], const int4v (&m)[kM]) {
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < kM; ++j) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(n[i], m[j], sum[i][j], 0, 0, 0);
    };
    // This wave's loads of all but the newest `kLeft` steps are done and its reads of
    // LDS too; then those of all waves.
    const auto arrive = [&](auto left) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(left)::value * Shape::kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const auto step = [&](const int4v (&n)[kN], const int4v (&m)[kM], int4v (&next_n)[kN], int4v (&next_m)[kM], uint32_t block) {
        const uint32_t slot = (block - first) % kSlots;
        arrive(std::integral_constant<int, kSlots - 2>{});  // the next step has come, and nobody reads this one's slot any more
        send(block + kSlots, slot);
        __builtin_amdgcn_sched_barrier(0);
        read(next_n, next_m, (slot + 1) % kSlots);
        multiply(n, m);
        // a read of LDS between the matrix instructions until all are on their way
#pragma unroll
        for (int i = 0; i < kN + kM; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, kN * kM / (kN + kM), 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (uint32_t s = 0; s < kSlots; ++s) send(first + s, s);
    arrive(std::integral_constant<int, kSlots - 1>{});
    int4v n0[kN], m0[kM], n1[kN], m1[kM];
    read(n0, m0, 0);
    uint32_t block = first;
    for (; block + 1 <= last; block += 2) {
        step(n0, m0, n1, m1, block);
        step(n1, m1, n0, m0, block + 1);
    }
    if (block <= last) multiply(n0, m0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // LDS is another workgroup's after the end

    if (threadIdx.x < Shape::kRows * kTile) row_scales[threadIdx.x] = scale_of_row;
    const uint32_t n_of = (tile_n + wave_n) * kTile + lane / kTile * 4, m_of = (tile_m + wave_m - Shape::kOutputs) * kTile + lane % kTile;
    if (a.slices > 1) {
#pragma unroll
        for (int j = 0; j < kM; ++j)
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const uint32_t row = m_of + j * kTile, n = n_of + i * kTile;
                if (row < a.rows && n < a.tiles * kTile)
                    *reinterpret_cast<int4v*>(a.partials + (static_cast<uint64_t>(blockIdx.y) * a.rows + row) * a.tiles * kTile + n) = sum[i][j];
            }
        return;
    }
    // By way of LDS, each wave in a part of its own, so that rows leave in whole runs and the
    // rounding stands in a loop: written out for all sums it was 100 KB of code, and most of
    // a short product's time was spent fetching it.
    __syncthreads();
    constexpr uint32_t kQuads = kN * 4, kHalf = kM / 2 * kTile;  // fours of a row's outputs, rows at a time
    int4v* held = reinterpret_cast<int4v*>(slots) + wave * (kQuads * kHalf);
    const uint32_t quad = lane % kQuads, n = (tile_n + wave_n) * kTile + quad * 4;
    float4v scales, bias;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        scales[e] = a.scales[min(n + e, a.outputs - 1)];
        bias[e] = a.bias ? a.bias[min(n + e, a.outputs - 1)] : 0.0f;
    }
    const auto store = [&](auto type, uint32_t from) {
        using Y = decltype(type);
#pragma unroll 2
        for (uint32_t r = lane / kQuads; r < kHalf; r += 64 / kQuads) {
            const uint32_t of_tile = (wave_m - Shape::kOutputs) * kTile + from + r, row = tile_m * kTile + of_tile;
            if (row >= a.rows) break;
            const float scale = row_scales[of_tile];
            const int4v whole = held[r * kQuads + (quad ^ (r % kQuads))];
            typename Y::type four[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                four[e] = static_cast<typename Y::type>(value_of(static_cast<float>(whole[e]), scales[e], scale, bias[e]));
            auto* to = static_cast<typename Y::type*>(a.y) + static_cast<int64_t>(row) * a.y_stride + n;
            if (n + 4 <= a.outputs) {
                __builtin_memcpy(to, four, sizeof(four));  // rows need no alignment
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (n + e < a.outputs) to[e] = four[e];
            }
        }
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < kM / 2; ++j)
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const uint32_t r = j * kTile + lane % kTile;
                held[r * kQuads + ((i * 4 + lane / kTile) ^ (r % kQuads))] = sum[i][half * (kM / 2) + j];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (a.y_type == LEO_TYPE_F32) store(F32{}, half * kHalf);
        else if (a.y_type == LEO_TYPE_F16) store(F16{}, half * kHalf);
        else store(BF16{}, half * kHalf);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// The slices of one output by kShare threads.
template <uint32_t kShare>
__global__ __launch_bounds__(256) void leo_q8_join(ProductArgs a) {
    constexpr uint32_t kOutputs = 256 / kShare;
    __shared__ int64_t parts[kShare][kOutputs];
    const uint32_t wide = (a.outputs + kOutputs - 1) / kOutputs, block = block_of_grid(), row = block / wide;
    if (row >= a.rows) return;
    const uint32_t n = block % wide * kOutputs + threadIdx.x % kOutputs, share = threadIdx.x / kOutputs;
    int64_t sum = 0;
    if (n < a.outputs) {
#pragma unroll 8
        for (uint32_t s = share; s < a.slices; s += kShare) sum += a.partials[(static_cast<uint64_t>(s) * a.rows + row) * a.tiles * kTile + n];
    }
    if constexpr (kShare > 1) {
        parts[share][threadIdx.x % kOutputs] = sum;
        __syncthreads();
        if (share) return;
#pragma unroll
        for (uint32_t s = 1; s < kShare; ++s) sum += parts[s][threadIdx.x];
    }
    if (n < a.outputs) store_y(a, row, n, sum, a.x_scales[row]);
}

struct Plan {
    bool few;
    uint32_t tiles;        // both sides of a workgroup of leo_q8_tiles, 0: none
    uint32_t group_tiles;  // of a workgroup of leo_q8_few or leo_q8_many
    uint32_t group_rows;   // in tiles, of a workgroup of leo_q8_many
    uint32_t slices, slice_blocks;
    uint32_t parts, part_inputs;
    uint64_t x_scales, largest, partials, workspace;  // offsets behind x's codes, and the whole
};
Plan plan_of(const LeoQ8Shape& s, uint64_t rows) {
    const Q8Layout l = layout_of(s);
    const uint64_t row_tiles = (rows + kTile - 1) / kTile;
    Plan p{};
    const bool whole = l.tiles >= 128 || l.blocks <= 32;
    // Where every workgroup would bring whole rows to 8 bits by itself, only as long as those are short: 2, 4 and 8 rows of
    // 8,192 -> 8,192 took 15.4, 20.2 and 30.7 us so and 16.2 to 16.3 with rows brought to 8 bits before, 4 and 8 rows of
    // 4,096 -> 2,048 7.7 and 11.3 against 9.0 and 9.1.
    p.few = rows <= kTile && (!whole || rows * s.inputs <= 24576);
    uint64_t slices = 1;
    const auto over = [](uint64_t v, uint64_t by) { return (v + by - 1) / by; };
    if (p.few) {
        // A workgroup a tile (or up to eight) over whole rows where that makes enough workgroups, or where rows are
        // short: 8,192 -> 8,192 took 12.9 us with a tile each and 15.0 to 16.7 with more or in slices, 1,024 -> 257 3.3
        // and 5.3. Else slices of 16 blocks, two a wave, and more where they would be over 512, for all tiles in groups
        // that differ little: 8 rows of 131,072 -> 257 in 128 slices took 14.9 us, in 170 16.0, in 85 16.6.
        p.group_tiles = static_cast<uint32_t>(whole ? std::min<uint64_t>(8, over(l.tiles, 512)) : over(l.tiles, over(l.tiles, 8)));
        if (!whole) {
            const uint64_t most = std::max<uint64_t>(1, 1024 / over(l.tiles, p.group_tiles));
            slices = over(l.blocks, over(std::max<uint64_t>(16, over(l.blocks, most)), 8) * 8);
        }
        slices = std::max(slices, over(l.blocks * rows * kBlock, kFewStage));
    } else if (row_tiles <= 8 || l.tiles < 8) {
        // 64 rows of 8,192 -> 8,192 took 20.6 us with 512 workgroups of one tile and 23.0 with 256 of two, of 5,001 ->
        // 11,007 20.3 with 688 and 18.9 with 344; 128 rows, each tile read twice, 24 with four tiles and 29 with two.
        p.group_rows = row_tiles <= 2 ? static_cast<uint32_t>(row_tiles) : 4;
        p.group_tiles = row_tiles > 4 ? (l.tiles > 2 ? 4 : static_cast<uint32_t>(l.tiles)) : l.tiles > 600 ? 2 : 1;
        const uint64_t groups = over(l.tiles, p.group_tiles) * over(row_tiles, p.group_rows);
        slices = l.blocks <= 64 ? 1 : std::max<uint64_t>(1, std::min<uint64_t>(512 / groups, over(l.blocks, 16)));
    } else {
        // A CU has one workgroup of the larger tile, or two of the smaller, and those two together do half as much: the
        // larger where it takes fewer rounds. 1,536 rows of 4,096 -> 4,096 took 52 us with the larger and 46 with the
        // smaller, 1,024 of 8,192 -> 8,192 89 and 87, 2,048 117 with the larger. A few of them share the inputs: 256
        // rows of 8,192 -> 8,192 took 48 us in one slice, 41 in two, 45 in four.
        const uint64_t large = over(l.tiles, 16) * over(row_tiles, 16), small = over(l.tiles, 8) * over(row_tiles, 8);
        p.tiles = over(small, 512) > over(large, 256) ? 16 : 8;
        slices = p.tiles == 16 ? 1 : std::max<uint64_t>(1, std::min<uint64_t>(256 / small, l.blocks / 16));
    }
    slices = std::max<uint64_t>(slices, over(l.blocks, kMostSliceBlocks));
    p.slice_blocks = static_cast<uint32_t>(over(l.blocks, slices));
    p.slices = static_cast<uint32_t>(over(l.blocks, p.slice_blocks));
    // Each workgroup of leo_q8_few looks through short rows itself: 1 row of 16,384 -> 257 took 6.8 us so and 8.1 with a
    // launch for it, 8 rows of 8,192 10.6 and 9.1, 1 row of 40,000 9.9 both ways. Rows that the threads of a workgroup hold
    // are read once: 2,000 rows of 16,384 -> 1,000 took 87 us so and 130 in parts.
    if (p.few ? rows * s.inputs > 32768 : s.inputs > kHeldInputs) {
        const uint64_t want = std::max<uint64_t>(4096, (s.inputs + kMostParts - 1) / kMostParts);
        p.part_inputs = static_cast<uint32_t>((want + 15) / 16 * 16);
        p.parts = static_cast<uint32_t>((s.inputs + p.part_inputs - 1) / p.part_inputs);
    }
    p.x_scales = p.few ? 0 : row_tiles * l.blocks * kBlockBytes;
    p.largest = p.x_scales + (p.few && p.slices == 1 ? 0 : up(rows * sizeof(float)));
    p.partials = p.largest + up(rows * p.parts * sizeof(uint32_t));
    p.workspace = p.partials + (p.slices > 1 ? up(p.slices * rows * l.tiles * kTile * sizeof(int32_t)) : 0);
    return p;
}

template <class X>
void launch_few(const Plan& p, const ProductArgs& a, hipStream_t stream) {
    const dim3 grid((a.tiles + p.group_tiles - 1) / p.group_tiles, a.slices);
    const uint32_t lds = a.rows * a.slice_blocks * kBlock;
    static constexpr void (*kKernels[])(ProductArgs) = {leo_q8_few<X, 1>, leo_q8_few<X, 2>, leo_q8_few<X, 3>, leo_q8_few<X, 4>,
                                                        leo_q8_few<X, 5>, leo_q8_few<X, 6>, leo_q8_few<X, 7>, leo_q8_few<X, 8>};
    launch(kKernels[p.group_tiles - 1], grid, dim3(kFewThreads), lds, stream, a);
}

template <int kN, int kM, int kWavesN, int kWavesM>
void launch_tiles(const ProductArgs& a, hipStream_t stream) {
    using Shape = TileShape<kN, kM, kWavesN, kWavesM>;
    const uint32_t across = (a.tiles + Shape::kOutputs - 1) / Shape::kOutputs, down = (a.row_tiles + Shape::kRows - 1) / Shape::kRows;
    launch(leo_q8_tiles<kN, kM, kWavesN, kWavesM>, dim3(across * down, a.slices), dim3(64 * Shape::kWaves), kSlots * Shape::kSlotBytes, stream, a, across);
}

template <class X>
void launch_product(const Plan& p, const ProductArgs& a, uint32_t* largest, hipStream_t stream) {
    if (a.parts) launch(leo_q8_largest<X>, dim3(a.rows, a.parts), dim3(256), 0, stream, a, largest);
    if (p.few) return launch_few<X>(p, a, stream);
    if (a.parts) launch(leo_q8_quantize_part<X>, dim3(a.rows, a.parts), dim3(256), 0, stream, a);
    else launch(leo_q8_quantize_row<X>, dim3((a.row_tiles + 7) / 8 * 8 * kTile), dim3((a.inputs + 1023) / 1024 * 64), 0, stream, a);
    if (p.tiles == 16) return launch_tiles<4, 8, 4, 2>(a, stream);
    if (p.tiles == 8) return launch_tiles<4, 4, 2, 2>(a, stream);
    const bool one = p.group_tiles == 1;
    const auto many = p.group_rows == 1 ? (one ? leo_q8_many<1, 1> : leo_q8_many<1, 2>)
                      : p.group_rows == 2 ? (one ? leo_q8_many<2, 1> : leo_q8_many<2, 2>)
                      : p.group_tiles == 4 ? leo_q8_many<4, 4> : one ? leo_q8_many<4, 1> : leo_q8_many<4, 2>;
    launch(many, dim3((a.tiles + p.group_tiles - 1) / p.group_tiles, (a.row_tiles + p.group_rows - 1) / p.group_rows, a.slices), dim3(kFewThreads), 0, stream, a);
}

}  // namespace
}  // namespace leo

using namespace leo;

extern "C" {

int32_t leo_q8_layout_bytes(const LeoQ8Shape* shape, uint64_t* bytes) {
    return guarded([&] {
        require(shape && bytes, "leo_q8_layout_bytes: null argument");
        check_shape(*shape);
        *bytes = layout_of(*shape).bytes;
    });
}

int32_t leo_q8_layout(const LeoQ8Source* source, void* stream) {
    return guarded([&] {
        require(source, "leo_q8_layout: null argument");
        const LeoQ8Source& s = *source;
        check_shape(s.shape);
        require(valid_type(s.scale_type), "leo_q8_layout: unknown scale type");
        require(s.codes && s.scales && s.layout, "leo_q8_layout: null argument");
        require(s.codes_stride >= static_cast<int64_t>(s.shape.inputs) || s.shape.outputs == 1,
                "leo_q8_layout: codes_stride is too small");
        require(reinterpret_cast<uintptr_t>(s.layout) % 256 == 0, "leo_q8_layout: layout must be 256-byte aligned");
        const Q8Layout l = layout_of(s.shape);
        require(s.layout_bytes >= l.bytes, "leo_q8_layout: layout is too small");
        const uint64_t count = l.tiles * l.blocks;
        const uint32_t wide = static_cast<uint32_t>(std::min<uint64_t>(count, 65536));
        const uint64_t high = (count + wide - 1) / wide;
        require(high <= 65535, "leo_q8_layout: too many codes");
        launch(leo_q8_lay_out, dim3(wide, static_cast<uint32_t>(high)), dim3(64), 0, static_cast<hipStream_t>(stream), s, l);
    });
}

int32_t leo_q8_workspace_bytes(const LeoQ8Shape* shape, uint64_t rows, int32_t x_type, uint64_t* bytes) {
    return guarded([&] {
        require(shape && bytes, "leo_q8_workspace_bytes: null argument");
        check_shape(*shape);
        require(rows <= kMostRows, "leo_q8_workspace_bytes: too many rows");
        require(valid_type(x_type), "leo_q8_workspace_bytes: unknown type");
        *bytes = rows ? plan_of(*shape, rows).workspace : 0;
    });
}

int32_t leo_q8_matmul(const LeoQ8Product* product, void* stream) {
    return guarded([&] {
        require(product, "leo_q8_matmul: null argument");
        const LeoQ8Product& p = *product;
        check_shape(p.shape);
        if (p.rows == 0) return;
        require(p.rows <= kMostRows, "leo_q8_matmul: too many rows");
        require(valid_type(p.x_type) && valid_type(p.y_type), "leo_q8_matmul: unknown type");
        require(p.layout && p.x && p.y, "leo_q8_matmul: null argument");
        require(p.x_stride >= 0, "leo_q8_matmul: x_stride must not be negative");
        require(p.y_stride >= static_cast<int64_t>(p.shape.outputs) || p.rows == 1, "leo_q8_matmul: y_stride is too small");
        const Rows y = rows_of(p.y, p.rows, p.shape.outputs, p.y_stride, p.y_type);
        require(!overlap(rows_of(p.x, p.rows, p.shape.inputs, p.x_stride, p.x_type), y), "leo_q8_matmul: y overlaps x");
        require(!meets_bias(p.bias, y, p.shape.outputs, p.y_type), "leo_q8_matmul: y overlaps the bias");
        require(reinterpret_cast<uintptr_t>(p.layout) % 256 == 0, "leo_q8_matmul: layout must be 256-byte aligned");
        const Q8Layout l = layout_of(p.shape);
        require(p.layout_bytes >= l.bytes, "leo_q8_matmul: layout is too small for its shape");
        const Plan plan = plan_of(p.shape, p.rows);
        const uint64_t wide = plan.tiles ? plan.tiles : plan.group_tiles, high = plan.tiles ? plan.tiles * uint64_t{kTile} : p.rows;
        const uint64_t groups = (l.tiles + wide - 1) / wide * ((p.rows + high - 1) / high);  // on the grid's first axis
        require((p.shape.outputs + 7) / 8 * p.rows <= 0x7fffffffu && groups * kFewThreads < 1ull << 32, "leo_q8_matmul: the result is too large");
        require(plan.workspace == 0 || (p.workspace && reinterpret_cast<uintptr_t>(p.workspace) % 256 == 0 &&
                                        p.workspace_bytes >= plan.workspace),
                "leo_q8_matmul: workspace is missing, too small or not 256-byte aligned");
        ProductArgs a{};
        a.codes = static_cast<const char*>(p.layout);
        a.scales = reinterpret_cast<const float*>(a.codes + l.scales);
        a.x = p.x;
        a.x_stride = p.x_stride;
        a.bias = p.bias;
        a.y = p.y;
        a.y_stride = p.y_stride;
        a.y_type = p.y_type;
        a.rows = static_cast<uint32_t>(p.rows);
        a.inputs = static_cast<uint32_t>(p.shape.inputs);
        a.outputs = static_cast<uint32_t>(p.shape.outputs);
        a.tiles = static_cast<uint32_t>(l.tiles);
        a.blocks = static_cast<uint32_t>(l.blocks);
        a.row_tiles = (a.rows + kTile - 1) / kTile;
        a.slices = plan.slices;
        a.slice_blocks = plan.slice_blocks;
        a.parts = plan.parts;
        a.part_inputs = plan.part_inputs;
        a.x_codes = static_cast<char*>(p.workspace);
        a.x_scales = reinterpret_cast<float*>(a.x_codes + plan.x_scales);
        auto* largest = reinterpret_cast<uint32_t*>(a.x_codes + plan.largest);
        a.largest = largest;
        a.partials = reinterpret_cast<int32_t*>(a.x_codes + plan.partials);
        const auto at = static_cast<hipStream_t>(stream);
        if (p.x_type == LEO_TYPE_F32) launch_product<F32>(plan, a, largest, at);
        else if (p.x_type == LEO_TYPE_F16) launch_product<F16>(plan, a, largest, at);
        else launch_product<BF16>(plan, a, largest, at);
        if (plan.slices == 1) return;
        // 340 slices took 1.5 us less with 32 threads an output than with 8, 128 0.4 less with 16
        const uint32_t share = plan.slices >= 256 ? 32 : plan.slices >= 16 ? 16 : 1;
        const uint64_t count = (p.shape.outputs + 256 / share - 1) / (256 / share) * p.rows;
        launch(share == 32 ? leo_q8_join<32> : share == 16 ? leo_q8_join<16> : leo_q8_join<1>, grid_of(static_cast<uint32_t>(count)), dim3(256), 0, at, a);
    });
}

}  // extern "C"
