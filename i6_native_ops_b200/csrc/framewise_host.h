// framewise_host.h -- what the host sides of the operators of framewise training share: status macros, the count of
// launches, a buffer's parts, the device's number of SMs, shared memory past 48 KB, tensor maps.
#pragma once

#include "framewise_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

namespace framewise_host {

inline std::atomic<int64_t> g_launches{0};

#define FW_TRY(call)                                     \
    do {                                                 \
        if ((call) != cudaSuccess) return FRAMEWISE_B200_CUDA_ERROR; \
    } while (0)
#define FW_LAUNCHED()                                    \
    do {                                                 \
        framewise_host::g_launches.fetch_add(1, std::memory_order_relaxed); \
        FW_TRY(cudaGetLastError());                      \
    } while (0)

#define FW_DO(...)                                       \
    do {                                                 \
        const int status_ = (__VA_ARGS__);                     \
        if (status_ != FRAMEWISE_B200_OK) return status_; \
    } while (0)

constexpr size_t kAlign = 256;
inline size_t aligned(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }
inline bool   misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & (kAlign - 1)) != 0; }
inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// A buffer's parts one after another, each aligned.
struct Parts {
    char*  base;
    size_t used = 0;
    explicit Parts(void* p) : base(static_cast<char*>(p)) {}
    template <typename X>
    X* take(int64_t n) {
        X* at = base ? reinterpret_cast<X*>(base + used) : nullptr;
        used += aligned((size_t)n * sizeof(X));
        return at;
    }
};

constexpr int kMostDevices = 64;

// The current device's number of SMs.
inline int sm_count() {
    static std::atomic<int> known[kMostDevices];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < kMostDevices && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < kMostDevices) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// The current device's context is current afterwards: a thread that has made no CUDA call yet, such as torch's for
// backward passes, has none, and tensor maps need one.
inline int bind_device() {
    static thread_local int bound = -1;
    int dev = 0;
    FW_TRY(cudaGetDevice(&dev));
    if (dev != bound) FW_TRY(cudaSetDevice(dev));
    bound = dev;
    return FRAMEWISE_B200_OK;
}

// Dynamic shared memory past 48 KB has to be asked for, once per kernel (each has a `done` of its own) and device.
template <typename K>
int allow_shared(K* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    FW_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < kMostDevices ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return FRAMEWISE_B200_OK;
    FW_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return FRAMEWISE_B200_OK;
}

// ---- tensor maps

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
    static std::atomic<EncodeTiled> cached{nullptr};
    EncodeTiled f = cached.load(std::memory_order_acquire);
    if (f) return f;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
        return nullptr;
    f = reinterpret_cast<EncodeTiled>(p);
    cached.store(f, std::memory_order_release);
    return f;
}

// planes x rows x cols, rows `pitch` elements apart, read or written in boxes of box_cols x box_rows (of box_planes planes)
inline bool map_of(CUtensorMap* map, const void* base, bool f32, int64_t cols, int64_t rows, int64_t planes, int64_t pitch, int64_t plane,
                   int box_cols, int box_rows, int box_planes = 1) {
    const EncodeTiled f = encode_tiled();
    if (!f) return false;
    const int64_t    size = f32 ? 4 : 2;
    const cuuint64_t dims[3]    = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)(pitch * size), (cuuint64_t)(plane * size)};
    const cuuint32_t box[3]     = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, (cuuint32_t)box_planes};
    const cuuint32_t step[3]    = {1, 1, 1};
    const int row_bytes = box_cols * (int)size;
    return f(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
             strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace framewise_host
