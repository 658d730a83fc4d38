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
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

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
    uint32_t* counters;
    float* partials;
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
// the 11 below them.
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

// Four pairs of codes less their zero, exactly: in half precision 1024 + u is
// the bits 0x6400 | u and 1024 + 16 u the bits 0x6400 | u << 4.
__device__ __forceinline__ half8 weights_of(uint32_t word, half2 minus, half2 minus_high) {
    const half2 sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    union {
        uint32_t w[4];
        half2 h[4];
        half8 v;
    } u;
    const uint32_t next = word >> 8;
    u.w[0] = (word & 0x000f000fu) | 0x64006400u;
    u.w[1] = (word & 0x00f000f0u) | 0x64006400u;
    u.w[2] = (next & 0x000f000fu) | 0x64006400u;
    u.w[3] = (next & 0x00f000f0u) | 0x64006400u;
    u.h[0] = u.h[0] + minus;
    u.h[1] = __builtin_elementwise_fma(u.h[1], sixteenth, minus_high);
    u.h[2] = u.h[2] + minus;
    u.h[3] = __builtin_elementwise_fma(u.h[3], sixteenth, minus_high);
    return u.v;
}

template <int kGroups, bool kZero, bool kWide, int kTiles>
struct WeightStage {
    static constexpr int kScaleWords = kWide ? kGroups : (kGroups + 1) / 2;
    uint4v code[kTiles];
    uint32_t scale[kTiles][kScaleWords];
    uint32_t zero[kTiles];
};

// One workgroup: kTiles tiles of 16 outputs, 16 kRows rows of x and one slice of
// the inputs, whose blocks its waves take in turn.
template <class X, int kGroups, bool kZero, bool kWide, int kRows, int kTiles>
__global__ __launch_bounds__(kRows == 1 ? 512 : 256) void leo_q4_tiles(TileArgs a) {
    constexpr bool kScaled = !__is_same(X, F16);  // x goes to half precision by a power of two a row and block
    constexpr int kParts = __is_same(X, F32) ? 2 : 1;
    constexpr int kRegs = kTiles * kRows * 4;
    constexpr int kWaves = kRows == 1 ? 8 : 4;
    using Stage = WeightStage<kGroups, kZero, kWide, kTiles>;
    __shared__ float joined[kWaves][kRegs][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const uint32_t column = lane % 16, quad = lane / 16;
    const uint32_t tile0 = blockIdx.x * kTiles, row0 = blockIdx.z * kRows * 16;
    const uint32_t begin = blockIdx.y * a.slice_blocks, end = min(begin + a.slice_blocks, a.blocks);

    int64_t row_at[kRows];
#pragma unroll
    for (int m = 0; m < kRows; ++m) row_at[m] = min(row0 + m * 16 + column, a.rows - 1) * a.x_stride + quad * 8;
    uint64_t tile_at[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) tile_at[t] = static_cast<uint64_t>(min(tile0 + t, a.tiles - 1)) * a.blocks;

    const auto load_weights = [&](uint32_t block, Stage& s) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const uint64_t at = tile_at[t] + block;
            s.code[t] = reinterpret_cast<const uint4v*>(a.codes)[at * 64 + lane];
            const uint64_t group = (at * kTile + column) * kGroups;
            if constexpr (!kWide && kGroups == 1) {
                s.scale[t][0] = reinterpret_cast<const uint16_t*>(a.scales)[group];
            } else {
                __builtin_memcpy(s.scale[t], __builtin_assume_aligned(a.scales + group * (kWide ? 4 : 2), sizeof(s.scale[t])),
                                 sizeof(s.scale[t]));
            }
            if constexpr (kZero) {
                if constexpr (kGroups == 4) s.zero[t] = reinterpret_cast<const uint16_t*>(a.zeros)[at * kTile + column];
                else s.zero[t] = reinterpret_cast<const uint8_t*>(a.zeros)[at * kTile + column];
            }
        }
    };
    const auto load_x = [&](uint32_t block, Eight<X> (&v)[kRows][4]) {
        if ((block + 1) * kBlock <= a.inputs) {
#pragma unroll
            for (int m = 0; m < kRows; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[m][j] = load_eight<X>(a.x, row_at[m] + block * kBlock + 32 * j);
        } else {
#pragma unroll
            for (int m = 0; m < kRows; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[m][j] = load_some<X>(a.x, row_at[m] + block * kBlock + 32 * j,
                                           static_cast<int32_t>(a.inputs - block * kBlock) - 32 * j - 8 * static_cast<int32_t>(quad));
        }
    };

    float4v sum[kTiles][kRows] = {};
    Stage now, next;
    Eight<X> x_now[kRows][4], x_next[kRows][4];
    uint32_t block = begin + wave;
    if (block < end) {
        load_weights(block, now);
        load_x(block, x_now);
    }
    for (; block < end; block += waves) {
        if (block + waves < end) {
            load_weights(block + waves, next);
            load_x(block + waves, x_next);
        }
        half8 part[kRows][4][kParts];
        float4v back[kRows];
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            if constexpr (kScaled) {
                // the largest value of the block goes to 2^14 .. 2^15, below half precision's end
                const uint32_t e = top_exponent<X>(x_now[m]);
                const float factor = __uint_as_float((268u - e) << 23), inverse = __uint_as_float((e - 14u) << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) back[m][i] = __shfl(inverse, static_cast<int>(quad * 4 + i));
#pragma unroll
                for (int j = 0; j < 4; ++j) halves<X, kParts>(x_now[m][j], factor, part[m][j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) part[m][j][0] = __builtin_bit_cast(half8, x_now[m][j].w[0]);
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            float4v whole[kRows] = {};
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                half2 minus = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
                half2 minus_high = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
                if constexpr (kZero) {
                    // -(1024 + z) and -(64 + z) are the bits 0xe400 | z and 0xd400 | z << 4
                    const uint32_t z = now.zero[t] >> (4 * g) & 15u, both = z | z << 16;
                    minus = __builtin_bit_cast(half2, both | 0xe400e400u);
                    minus_high = __builtin_bit_cast(half2, both << 4 | 0xd400d400u);
                }
                float4v d[kRows] = {};
#pragma unroll
                for (int j = g * 4 / kGroups; j < (g + 1) * 4 / kGroups; ++j) {
                    const half8 w = weights_of(now.code[t][j], minus, minus_high);
#pragma unroll
                    for (int m = 0; m < kRows; ++m)
#pragma unroll
                        for (int s = 0; s < kParts; ++s)
                            d[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[m][j][s], w, d[m], 0, 0, 0);
                }
                float scale;
                if constexpr (kWide) {
                    scale = __uint_as_float(now.scale[t][g]);
                } else {
                    const uint32_t bits = now.scale[t][g / 2] >> (16 * (g % 2)) & 0xffffu;
                    scale = a.scale_bf16 ? __uint_as_float(bits << 16)
                                         : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
                }
#pragma unroll
                for (int m = 0; m < kRows; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (kScaled) whole[m][i] = __builtin_fmaf(scale, d[m][i], whole[m][i]);
                        else sum[t][m][i] = __builtin_fmaf(scale, d[m][i], sum[t][m][i]);
                    }
            }
            if constexpr (kScaled) {
#pragma unroll
                for (int m = 0; m < kRows; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[t][m][i] = __builtin_fmaf(back[m][i], whole[m][i], sum[t][m][i]);
            }
        }
        now = next;
#pragma unroll
        for (int m = 0; m < kRows; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) x_now[m][j] = x_next[m][j];
    }

    // a register of a lane is the sum of output 16 tile + column and row 16 m + 4 quad + i
    const auto row_of = [&](uint32_t reg, uint32_t of) { return row0 + reg / 4 % kRows * 16 + of / 16 * 4 + reg % 4; };
    const auto each = [&](auto&& f) {
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < kRegs * 64; at += blockDim.x) {
            const uint32_t reg = at / 64, of = at % 64, row = row_of(reg, of);
            const uint32_t output = (tile0 + reg / (4 * kRows)) * kTile + of % 16;
            if (row >= a.rows || output >= a.outputs) continue;
            float v = joined[0][reg][of];
            for (uint32_t w = 1; w < waves; ++w) v += joined[w][reg][of];
            f(at, row, output, v);
        }
    };
    const auto store = [&](uint32_t, uint32_t row, uint32_t output, float v) {
        store_any(a.y, row * a.y_stride + output, v + (a.bias ? a.bias[output] : 0.0f), a.y_type);
    };
#pragma unroll
    for (int r = 0; r < kRegs; ++r) joined[wave][r][lane] = sum[r / (4 * kRows)][r / 4 % kRows][r % 4];
    if (a.slices == 1) {
        each(store);
        return;
    }
    // every slice's sums go to memory; the workgroup that comes last adds them, in the slices' order
    const uint64_t group = blockIdx.z * gridDim.x + blockIdx.x;
    float* mine = a.partials + group * a.slices * (kRegs * 64);
    each([&](uint32_t at, uint32_t, uint32_t, float v) { hand_over(mine + blockIdx.y * (kRegs * 64) + at, v); });
    if (!last_to_arrive(a.counters + group, a.slices)) return;
    float total[kRegs] = {};
    for (uint32_t s = wave; s < a.slices; s += waves)
#pragma unroll
        for (int r = 0; r < kRegs; ++r)
            if (row_of(r, lane) < a.rows && (tile0 + r / (4 * kRows)) * kTile + column < a.outputs)
                total[r] += take_over(mine + s * (kRegs * 64) + r * 64 + lane);
#pragma unroll
    for (int r = 0; r < kRegs; ++r) joined[wave][r][lane] = total[r];
    each(store);
}

struct Plan {
    uint32_t rows, tiles, waves;  // rows (of 16) and tiles of a workgroup, waves that share its blocks
    uint32_t groups, slabs, slices, slice_blocks;
    uint64_t workspace;
};

Plan plan_of(const LeoQ4Shape& s, uint64_t rows, int32_t x_type) {
    const Q4Layout l = layout_of(s);
    Plan p;
    p.rows = rows <= 16 ? 1 : x_type == LEO_TYPE_F32 ? 2 : 4;
    p.slabs = static_cast<uint32_t>((rows + 16 * p.rows - 1) / (16 * p.rows));
    const uint64_t work = l.tiles * l.blocks * p.slabs;
    p.tiles = p.rows > 1 ? 2 : work < 4096 ? 1 : 4;
    p.groups = static_cast<uint32_t>((l.tiles + p.tiles - 1) / p.tiles);
    const uint32_t most = p.rows == 1 ? 8 : 4;
    p.waves = static_cast<uint32_t>(l.blocks < most ? l.blocks : most);
    const uint64_t wanted = p.rows == 1 ? 512 : 768;
    uint64_t slices = (wanted + p.groups * p.slabs - 1) / (static_cast<uint64_t>(p.groups) * p.slabs);
    slices = std::min<uint64_t>(slices, std::max<uint64_t>(1, l.blocks / (2 * p.waves)));
    if (static_cast<uint64_t>(p.groups) * p.slabs > kCounters) slices = 1;
    p.slice_blocks = static_cast<uint32_t>((l.blocks + slices - 1) / slices);
    p.slices = static_cast<uint32_t>((l.blocks + p.slice_blocks - 1) / p.slice_blocks);
    p.workspace = p.slices == 1 ? 0 : kCounterBytes + static_cast<uint64_t>(p.groups) * p.slabs * p.slices * p.tiles * p.rows * 1024;
    return p;
}

template <class X, int kGroups, bool kZero, bool kWide>
void launch_tiles(const Plan& p, const TileArgs& a, hipStream_t stream) {
    const dim3 grid(p.groups, p.slices, p.slabs), block(p.waves * 64);
    if (p.rows == 1 && p.tiles == 1) launch(leo_q4_tiles<X, kGroups, kZero, kWide, 1, 1>, grid, block, stream, a);
    else if (p.rows == 1) launch(leo_q4_tiles<X, kGroups, kZero, kWide, 1, 4>, grid, block, stream, a);
    else if constexpr (__is_same(X, F32)) launch(leo_q4_tiles<X, kGroups, kZero, kWide, 2, 2>, grid, block, stream, a);
    else launch(leo_q4_tiles<X, kGroups, kZero, kWide, 4, 2>, grid, block, stream, a);
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
               static_cast<hipStream_t>(stream), a);
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
        a.scale_bf16 = p.shape.scale_type == LEO_TYPE_BF16;
        a.rows = static_cast<uint32_t>(p.rows);
        a.inputs = static_cast<uint32_t>(p.shape.inputs);
        a.outputs = static_cast<uint32_t>(p.shape.outputs);
        a.tiles = static_cast<uint32_t>(l.tiles);
        a.blocks = static_cast<uint32_t>(l.blocks);
        a.slices = plan.slices;
        a.slice_blocks = plan.slice_blocks;
        a.counters = static_cast<uint32_t*>(p.workspace);
        a.partials = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + (plan.workspace ? kCounterBytes : 0));
        const auto at = static_cast<hipStream_t>(stream);
        if (p.x_type == LEO_TYPE_F32) launch_products<F32>(p.shape, plan, a, at);
        else if (p.x_type == LEO_TYPE_F16) launch_products<F16>(p.shape, plan, a, at);
        else launch_products<BF16>(p.shape, plan, a, at);
    });
}

}  // extern "C"
