// What the decoding operators' translation units share: element loads and
// stores in 32 bits, wave reductions and checked launches.
#ifndef LEO_DECODE_COMMON_H
#define LEO_DECODE_COMMON_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <type_traits>

#include "leo_decode.h"
#include "leo_host.h"

namespace leo {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// Element e of 16 bytes of a type is at(words, e); put rounds into it.
struct F32 {
    using type = float;
    using bits = uint32_t;
    static constexpr uint32_t kNegativeInfinity = 0xff800000u;
    static __device__ __forceinline__ float at(const uint4v& w, uint32_t e) { return __uint_as_float(w[e]); }
    static __device__ __forceinline__ void put(uint4v& w, uint32_t e, float v) { w[e] = __float_as_uint(v); }
    static __device__ __forceinline__ float load(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};
struct F16 {
    using type = _Float16;
    using bits = uint16_t;
    static constexpr uint32_t kNegativeInfinity = 0xfc00u;
    static __device__ __forceinline__ float at(const uint4v& w, uint32_t e) {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2)))));
    }
    static __device__ __forceinline__ void put(uint4v& w, uint32_t e, float v) {
        const uint32_t half = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
        w[e / 2] = e % 2 ? w[e / 2] | half << 16 : half;
    }
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return static_cast<float>(static_cast<const _Float16*>(p)[i]);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    }
};
struct BF16 {
    using type = __bf16;
    using bits = uint16_t;
    static constexpr uint32_t kNegativeInfinity = 0xff80u;
    static __device__ __forceinline__ float at(const uint4v& w, uint32_t e) {
        return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
    static __device__ __forceinline__ void put(uint4v& w, uint32_t e, float v) {
        const uint32_t half = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
        w[e / 2] = e % 2 ? w[e / 2] | half << 16 : half;
    }
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
    }
};

// Reductions over the 64 lanes of a wave in the register file (six DPP steps);
// every lane gets the result.
template <class F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, uint32_t identity, F&& f) {
    const auto step = [&](auto ctrl, auto rows) {
        v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(identity), static_cast<int>(v),
                                                                  decltype(ctrl)::value, decltype(rows)::value, 0xf, false)));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // within rows of 16, by 1, 2, 4 and 8
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // rows 0 and 2 into 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // the lower half into the upper
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), 0xff800000u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
    return wave_reduce(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
    return wave_reduce(v, 0xffffffffu, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// The same for all of a wave's lanes, so what follows from it is scalar.
__device__ __forceinline__ uint32_t wave_of_workgroup() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }

__device__ __forceinline__ float negative_infinity() { return -__builtin_inff(); }

// A float's bits in the order of its value.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 16 bytes from any address: rows need no alignment.
__device__ __forceinline__ uint4v load_16(const void* p) {
    uint4v v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// 16 bytes of a row of n elements from element i on; -inf beyond its end.
template <class T>
__device__ __forceinline__ uint4v load_row(const void* row, uint32_t i, uint32_t n) {
    constexpr uint32_t kWide = 16 / sizeof(typename T::bits), kInWord = 4 / sizeof(typename T::bits);
    const auto* p = static_cast<const typename T::bits*>(row);
    if (i + kWide <= n) return load_16(p + i);
    uint4v v;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        v[w] = 0;
#pragma unroll
        for (uint32_t e = 0; e < kInWord; ++e) {
            const uint32_t at = i + w * kInWord + e;
            v[w] |= (at < n ? static_cast<uint32_t>(p[at]) : T::kNegativeInfinity) << (32 / kInWord * e);
        }
    }
    return v;
}

inline bool valid_type(int32_t type) { return type == LEO_TYPE_F32 || type == LEO_TYPE_F16 || type == LEO_TYPE_BF16; }
inline uint64_t type_bytes(int32_t type) { return type == LEO_TYPE_F32 ? 4 : 2; }

inline void require(bool ok, const char* what) {
    if (!ok) throw Error(LEO_ERR_INVALID_ARGUMENT, what);
}

// The bytes of a matrix with dense rows.
struct Rows {
    uintptr_t at;
    uint64_t count, width, stride;
};
inline Rows rows_of(const void* p, uint64_t count, uint64_t width, int64_t stride, int32_t type) {
    const uint64_t e = type_bytes(type);
    return {reinterpret_cast<uintptr_t>(p), count, width * e, count > 1 ? static_cast<uint64_t>(stride) * e : 0};
}
// Whether two of them share a byte. Columns of one buffer do not, though their
// ranges do: only then are the rows gone through, in the order of both.
inline bool overlap(const Rows& a, const Rows& b) {
    const auto end = [](const Rows& r) { return r.at + (r.count - 1) * r.stride + r.width; };
    if (end(a) <= b.at || end(b) <= a.at) return false;
    for (uint64_t i = 0, j = 0; i < a.count && j < b.count;) {
        const uintptr_t in_a = a.at + i * a.stride, in_b = b.at + j * b.stride;
        if (in_a + a.width <= in_b) ++i;
        else if (in_b + b.width <= in_a) ++j;
        else return true;
    }
    return false;
}

// Whether a product's result shares memory with its float bias. One row of floats may be the bias itself: each of its
// values is read by the thread that writes it, and before.
inline bool meets_bias(const float* bias, const Rows& y, uint64_t outputs, int32_t y_type) {
    if (!bias || (y.count == 1 && y_type == LEO_TYPE_F32 && y.at == reinterpret_cast<uintptr_t>(bias))) return false;
    return overlap(rows_of(bias, 1, outputs, 0, LEO_TYPE_F32), y);
}

// An axis of a grid has to have fewer than 2^32 threads: workgroups past the first 2^22 go on
// along the second axis, whose last row may hold some too many.
constexpr uint32_t kAcross = 1u << 22;
inline dim3 grid_of(uint32_t count) { return dim3(count < kAcross ? count : kAcross, (count + kAcross - 1) / kAcross); }
__device__ __forceinline__ uint32_t block_of_grid() { return blockIdx.y * kAcross + blockIdx.x; }

// Launches through the returned status, not the thread's last error, which an
// earlier call of the program may have left.
template <class... Args>
void launch(void (*kernel)(Args...), dim3 grid, dim3 block, uint32_t lds, hipStream_t stream, Args... args) {
    void* list[] = {&args...};
    const hipError_t status = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, lds, stream);
    if (status != hipSuccess)
        throw Error(LEO_ERR_DEVICE, std::string("kernel launch: ") + hipGetErrorString(status));
}

}  // namespace leo

#endif
