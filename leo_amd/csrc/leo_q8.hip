// Products with 8-bit weights and 8-bit activations, and the layout they read.
//
//     y[m, n] = bias[n] + s[m] c[n] sum_k q[m, k] w[n, k]
//     s[m] = max(max_k |x[m, k]| / 127, 2^-126),  q[m, k] = round(x[m, k] / s[m])
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

struct Q8Layout {
    uint64_t tiles, blocks;
    uint64_t scales, bytes;  // the scales' offset, and the whole
};

void check_shape(const LeoQ8Shape& s) {
    require(s.outputs >= 1 && s.outputs <= (1ull << 31), "q8: outputs must be 1 .. 2^31");
    require(s.inputs >= 1 && s.inputs <= (1ull << 31), "q8: inputs must be 1 .. 2^31");
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
        for (uint32_t i = 0; i < 16; ++i)
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
    char* x_codes;    // x as a layout
    float* x_scales;  // 16 a tile
    int32_t* partials;  // [slice][row][16 tiles]
};

// The whole number nearest to the exact quotient x / s, of two the even one: the
// product with the rounded inverse is off by less than one half, and the remainder
// x - n s, which needs no rounding where it is near s / 2, tells where it matters.
__device__ __forceinline__ int32_t code_of(float x, float s, float inverse) {
    const float n = __builtin_rintf(x * inverse), rest = __builtin_fmaf(-n, s, x), half = 0.5f * s;
    const int32_t code = static_cast<int32_t>(n);
    if (rest > half || (rest == half && (code & 1))) return code + 1;
    if (rest < -half || (rest == -half && (code & 1))) return code - 1;
    return code;
}

// The scale of a row from the largest magnitude of its values, as bits; NaN where that is no finite number.
__device__ __forceinline__ float scale_of(uint32_t largest) {
    return largest < 0x7f800000u ? fmaxf(__uint_as_float(largest) / 127.0f, 0x1p-126f) : __builtin_nanf("");
}

// One workgroup a row of a tile.
template <class T>
__global__ __launch_bounds__(256) void leo_q8_quantize(ProductArgs a) {
    __shared__ uint32_t most[4];
    const uint32_t row = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const bool inside = row < a.rows;
    const auto* x = static_cast<const typename T::type*>(a.x) + static_cast<int64_t>(row) * a.x_stride;
    uint32_t largest = 0;
    if (inside)
        for (uint32_t k = threadIdx.x; k < a.inputs; k += 256)
            largest = max(largest, __float_as_uint(T::load(x, k)) & 0x7fffffffu);
    largest = wave_reduce(largest, 0u, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
    if (lane == 0) most[wave] = largest;
    __syncthreads();
    const float scale = scale_of(max(max(most[0], most[1]), max(most[2], most[3]))), inverse = 1.0f / scale;
    if (threadIdx.x == 0) a.x_scales[row] = inside ? scale : 0.0f;
    const bool counts = inside && scale == scale;
    for (uint32_t part = threadIdx.x; part < a.blocks * 4; part += 256) {
        union {
            uint4v words;
            int8_t codes[16];
        } u;
        for (uint32_t i = 0; i < 16; ++i) {
            const uint32_t k = part * 16 + i;
            u.codes[i] = counts && k < a.inputs ? static_cast<int8_t>(code_of(T::load(x, k), scale, inverse)) : int8_t{0};
        }
        char* to = a.x_codes + (static_cast<uint64_t>(row / kTile) * a.blocks + part / 4) * kBlockBytes;
        reinterpret_cast<uint4v*>(to)[part % 4 * kTile + row % kTile] = u.words;
    }
}

__device__ __forceinline__ void store_y(const ProductArgs& a, uint32_t row, uint32_t n, int64_t sum) {
    const double v = static_cast<double>(sum) * a.x_scales[row] * a.scales[n] + (a.bias ? a.bias[n] : 0.0f);
    const int64_t at = static_cast<int64_t>(row) * a.y_stride + n;
    if (a.y_type == LEO_TYPE_F32) static_cast<float*>(a.y)[at] = static_cast<float>(v);
    else if (a.y_type == LEO_TYPE_F16) static_cast<_Float16*>(a.y)[at] = static_cast<_Float16>(v);
    else static_cast<__bf16*>(a.y)[at] = static_cast<__bf16>(v);
}

// One wave 16 rows, 16 outputs and a slice of the inputs. x is the A operand, so lane
// l gets output l % 16 of rows 4 (l / 16) + 0..3.
__global__ __launch_bounds__(64) void leo_q8_multiply(ProductArgs a) {
    const uint32_t tile = blockIdx.x, row_tile = blockIdx.y, slice = blockIdx.z, lane = threadIdx.x;
    const uint32_t begin = slice * a.slice_blocks, end = min(begin + a.slice_blocks, a.blocks);
    const char* w = a.codes + static_cast<uint64_t>(tile) * a.blocks * kBlockBytes;
    const char* x = a.x_codes + static_cast<uint64_t>(row_tile) * a.blocks * kBlockBytes;
    int4v sum = {0, 0, 0, 0};
    for (uint32_t block = begin; block < end; ++block) {
        const int4v p = reinterpret_cast<const int4v*>(x + static_cast<uint64_t>(block) * kBlockBytes)[lane];
        const int4v q = reinterpret_cast<const int4v*>(w + static_cast<uint64_t>(block) * kBlockBytes)[lane];
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(p, q, sum, 0, 0, 0);
    }
    const uint32_t n = tile * kTile + lane % kTile;
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = row_tile * kTile + lane / kTile * 4 + i;
        if (row >= a.rows) break;
        if (a.slices == 1) {
            if (n < a.outputs) store_y(a, row, n, sum[i]);
        } else {
            a.partials[(static_cast<uint64_t>(slice) * a.rows + row) * a.tiles * kTile + n] = sum[i];
        }
    }
}

__global__ __launch_bounds__(256) void leo_q8_join(ProductArgs a) {
    const uint32_t n = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y;
    if (n >= a.outputs) return;
    int64_t sum = 0;
    for (uint32_t s = 0; s < a.slices; ++s) sum += a.partials[(static_cast<uint64_t>(s) * a.rows + row) * a.tiles * kTile + n];
    store_y(a, row, n, sum);
}

struct Plan {
    uint32_t slices, slice_blocks;
    uint64_t x_scales, partials, workspace;  // offsets behind x's codes, and the whole
};
Plan plan_of(const LeoQ8Shape& s, uint64_t rows) {
    const Q8Layout l = layout_of(s);
    const uint64_t row_tiles = (rows + kTile - 1) / kTile;
    Plan p{};
    const uint64_t want = std::max<uint64_t>(1, 1024 / (l.tiles * row_tiles));
    const uint64_t slices = std::max((l.blocks + kMostSliceBlocks - 1) / kMostSliceBlocks, std::min(want, (l.blocks + 15) / 16));
    p.slice_blocks = static_cast<uint32_t>((l.blocks + slices - 1) / slices);
    p.slices = static_cast<uint32_t>((l.blocks + p.slice_blocks - 1) / p.slice_blocks);
    p.x_scales = row_tiles * l.blocks * kBlockBytes;
    p.partials = p.x_scales + up(row_tiles * kTile * sizeof(float));
    p.workspace = p.partials + (p.slices > 1 ? up(p.slices * rows * l.tiles * kTile * sizeof(int32_t)) : 0);
    return p;
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
        require(!overlap(rows_of(p.x, p.rows, p.shape.inputs, p.x_stride, p.x_type),
                         rows_of(p.y, p.rows, p.shape.outputs, p.y_stride, p.y_type)), "leo_q8_matmul: y overlaps x");
        require(reinterpret_cast<uintptr_t>(p.layout) % 256 == 0, "leo_q8_matmul: layout must be 256-byte aligned");
        const Q8Layout l = layout_of(p.shape);
        require(p.layout_bytes >= l.bytes, "leo_q8_matmul: layout is too small for its shape");
        const Plan plan = plan_of(p.shape, p.rows);
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
        a.x_codes = static_cast<char*>(p.workspace);
        a.x_scales = reinterpret_cast<float*>(a.x_codes + plan.x_scales);
        a.partials = reinterpret_cast<int32_t*>(a.x_codes + plan.partials);
        const auto at = static_cast<hipStream_t>(stream);
        launch(p.x_type == LEO_TYPE_F32 ? leo_q8_quantize<F32> : p.x_type == LEO_TYPE_F16 ? leo_q8_quantize<F16> : leo_q8_quantize<BF16>,
               dim3(a.row_tiles * kTile), dim3(256), 0, at, a);
        launch(leo_q8_multiply, dim3(a.tiles, a.row_tiles, a.slices), dim3(64), 0, at, a);
        if (a.slices > 1) launch(leo_q8_join, dim3((a.outputs + 255) / 256, a.rows), dim3(256), 0, at, a);
    });
}

}  // extern "C"
