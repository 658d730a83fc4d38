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

// Workspaces begin with counters that are zero between calls.
constexpr uint64_t kCounterBytes = 64 << 10, kCounters = kCounterBytes / 4;

// Values that workgroups of one launch hand each other go past the caches of
// one XCD: stores and loads of agent scope, and the writer waits for its stores
// before it says so.
__device__ __forceinline__ void hand_over(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float take_over(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whether this workgroup is the last of `count` to arrive, after every wave's
// handed-over values are in memory. The last one leaves the counter at zero.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t count) {
    __shared__ uint32_t last;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

}  // namespace leo

#endif
