// What the decoding operators' translation units share: element loads and
// stores in 32 bits, wave reductions and checked launches.
#ifndef LEO_DECODE_COMMON_H
#define LEO_DECODE_COMMON_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "leo_decode.h"
#include "leo_host.h"

namespace leo {

struct F32 {
    using type = float;
    static __device__ __forceinline__ float load(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};
struct F16 {
    using type = _Float16;
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return static_cast<float>(static_cast<const _Float16*>(p)[i]);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    }
};
struct BF16 {
    using type = __bf16;
    static __device__ __forceinline__ float load(const void* p, int64_t i) {
        return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
        static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
    }
};

inline bool valid_type(int32_t type) { return type == LEO_TYPE_F32 || type == LEO_TYPE_F16 || type == LEO_TYPE_BF16; }
inline uint64_t type_bytes(int32_t type) { return type == LEO_TYPE_F32 ? 4 : 2; }

inline void require(bool ok, const char* what) {
    if (!ok) throw Error(LEO_ERR_INVALID_ARGUMENT, what);
}

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
