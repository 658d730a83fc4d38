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
#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kTile = 16, kBlock = 128, kBlockBytes = 1024;

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

struct MatvecArgs {
    LeoQ4Product p;
    Q4Layout l;
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int32_t type) {
    return type == LEO_TYPE_F32 ? F32::load(p, i) : type == LEO_TYPE_F16 ? F16::load(p, i) : BF16::load(p, i);
}

__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int32_t type) {
    if (type == LEO_TYPE_F32) F32::store(p, i, v);
    else if (type == LEO_TYPE_F16) F16::store(p, i, v);
    else BF16::store(p, i, v);
}

// One wave an output and row; each lane takes every 64th run of eight inputs.
__global__ __launch_bounds__(256) void leo_q4_products(MatvecArgs a) {
    const LeoQ4Product& p = a.p;
    const uint32_t lane = threadIdx.x % 64;
    const uint64_t n = blockIdx.x * 4ull + threadIdx.x / 64;
    const uint64_t m = blockIdx.y;
    if (n >= p.shape.outputs) return;
    const uint64_t tile = n / kTile, r = n % kTile;
    const char* layout = static_cast<const char*>(p.layout);
    float sum = 0.0f;
    for (uint64_t run = lane; run < a.l.blocks * 16; run += 64) {
        const uint64_t at = tile * a.l.blocks + run / 16;
        const uint32_t j = run / 4 % 4, q = run % 4;
        const uint32_t word = reinterpret_cast<const uint32_t*>(layout)[at * 256 + (q * kTile + r) * 4 + j];
        const uint32_t g = 32 * j / p.shape.group;
        const float scale = load_any(layout + a.l.scales, (at * kTile + r) * a.l.groups + g, p.shape.scale_type);
        uint32_t zero = 8;
        if (a.l.zero_bytes) {
            const uint8_t* z = reinterpret_cast<const uint8_t*>(layout) + a.l.zeros + (at * kTile + r) * a.l.zero_bytes;
            zero = z[g / 2] >> (4 * (g % 2)) & 15u;
        }
        float part = 0.0f;
        for (uint32_t i = 0; i < 8; ++i) {
            const uint64_t k = (run / 16) * kBlock + 32 * j + 8 * q + i;
            if (k >= p.shape.inputs) break;
            const int32_t code = static_cast<int32_t>(word >> (4 * (i / 2 + 4 * (i % 2))) & 15u);
            part += load_any(p.x, m * p.x_stride + k, p.x_type) * static_cast<float>(code - static_cast<int32_t>(zero));
        }
        sum += scale * part;
    }
    for (uint32_t d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) store_any(p.y, m * p.y_stride + n, sum + (p.bias ? p.bias[n] : 0.0f), p.y_type);
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

int32_t leo_q4_workspace_bytes(const LeoQ4Shape* shape, uint64_t rows, uint64_t* bytes) {
    return guarded([&] {
        require(shape && bytes, "leo_q4_workspace_bytes: null argument");
        check_shape(*shape);
        require(rows <= (1ull << 31), "leo_q4_workspace_bytes: too many rows");
        *bytes = 0;
    });
}

int32_t leo_q4_matvec(const LeoQ4Product* product, void* stream) {
    return guarded([&] {
        require(product, "leo_q4_matvec: null argument");
        const LeoQ4Product& p = *product;
        check_shape(p.shape);
        MatvecArgs a{p, layout_of(p.shape)};
        if (p.rows == 0) return;
        require(p.layout && p.x && p.y, "leo_q4_matvec: null argument");
        require(p.rows <= 65535, "leo_q4_matvec: too many rows");
        require(valid_type(p.x_type) && valid_type(p.y_type), "leo_q4_matvec: unknown type");
        require(p.x_stride >= 0, "leo_q4_matvec: x_stride must not be negative");
        require(p.y_stride >= static_cast<int64_t>(p.shape.outputs) || p.rows == 1, "leo_q4_matvec: y_stride is too small");
        require(reinterpret_cast<uintptr_t>(p.layout) % 256 == 0, "leo_q4_matvec: layout must be 256-byte aligned");
        require(p.layout_bytes >= a.l.bytes, "leo_q4_matvec: layout is too small for its shape");
        launch(leo_q4_products, dim3(static_cast<uint32_t>((p.shape.outputs + 3) / 4), static_cast<uint32_t>(p.rows)),
               dim3(256), static_cast<hipStream_t>(stream), a);
    });
}

}  // extern "C"
