// Copies of cache pages and state slots: unit `source` of every array becomes unit `target`, for a list of pairs on
// the device.  A page of a sequence's cache is the same unit of K and V of every attention layer, and a state slot the
// same unit of codes, scales and convolution history of every DeltaNet layer, so one launch does what is one small
// memcpy per array and pair otherwise (crates/qwc-engine/src/executor.rs:825-835, copy_kv_block).
//
// Nothing is computed: every byte is read and written once, 16 at a time.  A CTA copies up to 16 KiB of one unit, all
// of a thread's loads in flight before its first store.

#include "common.cuh"

#include "../../../include/qwc_abi.h"

namespace qwc {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyDepth = 4;                                   // 16-byte loads of a thread in flight
constexpr int kCopyTile = kCopyThreads * kCopyDepth * 16;       // bytes of a unit that a CTA copies
constexpr int kArraysPerLaunch = 128;                           // what fits the kernel's parameters

struct CopyArrays {
    qwc_copy_array array[kArraysPerLaunch];
};

__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const __grid_constant__ CopyArrays arrays,
                                                                 const uint2* __restrict__ pairs, int* status) {
    pdl_launch_dependents();
    const qwc_copy_array array = arrays.array[blockIdx.z];
    const size_t begin = static_cast<size_t>(blockIdx.y) * kCopyTile;
    if (begin >= array.unit_bytes) {
        return;
    }
    pdl_wait();
    const uint2 pair = __ldcg(pairs + blockIdx.x);
    if (pair.x == pair.y) {
        return;  // nothing to do (and how a list is padded)
    }
    if (pair.x >= array.units || pair.y >= array.units) {
        if (threadIdx.x == 0) {
            atomicCAS(status, 0, kStatusCopyRange);
        }
        return;
    }
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(array.base) + pair.x * array.unit_bytes + begin);
    uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(array.base) + pair.y * array.unit_bytes + begin);
    const size_t left = (array.unit_bytes - begin) / 16;
    uint4 held[kCopyDepth];
#pragma unroll
    for (int i = 0; i < kCopyDepth; ++i) {
        const int at = threadIdx.x + i * kCopyThreads;
        if (at < left) {
            held[i] = __ldcs(from + at);
        }
    }
#pragma unroll
    for (int i = 0; i < kCopyDepth; ++i) {
        const int at = threadIdx.x + i * kCopyThreads;
        if (at < left) {
            to[at] = held[i];
        }
    }
}

}  // namespace
}  // namespace qwc

extern "C" int qwc_cache_copy(const qwc_copy_array* arrays, int array_count, const uint32_t* pairs, int count,
                              qwc_stream stream) {
    using namespace qwc;
    if (arrays == nullptr || array_count <= 0 || array_count > 4096 || count < 0 || (count > 0 && pairs == nullptr) ||
        (reinterpret_cast<uintptr_t>(pairs) & 7) != 0) {
        return cudaErrorInvalidValue;
    }
    for (int i = 0; i < array_count; ++i) {
        const qwc_copy_array& array = arrays[i];
        if (array.base == nullptr || (reinterpret_cast<uintptr_t>(array.base) & 15) != 0 || array.unit_bytes == 0 ||
            array.unit_bytes % 16 != 0 || array.unit_bytes > 65535ull * kCopyTile || array.units == 0 ||
            array.units > 0xffffffffull || array.units > (1ull << 48) / array.unit_bytes) {
            return cudaErrorInvalidValue;
        }
    }
    if (count == 0) {
        return cudaSuccess;
    }
    int* status = status_ptr();
    if (status == nullptr) {
        return cudaErrorInvalidValue;
    }
    for (int first = 0; first < array_count; first += kArraysPerLaunch) {
        const int here = array_count - first < kArraysPerLaunch ? array_count - first : kArraysPerLaunch;
        CopyArrays table = {};
        uint64_t longest = 0;
        for (int i = 0; i < here; ++i) {
            table.array[i] = arrays[first + i];
            longest = longest < table.array[i].unit_bytes ? table.array[i].unit_bytes : longest;
        }
        const dim3 grid(count, static_cast<unsigned>((longest + kCopyTile - 1) / kCopyTile), here);
        const cudaError_t launched = launch_chained(cache_copy_kernel, grid, dim3(kCopyThreads), 0,
                                                    static_cast<cudaStream_t>(stream), table,
                                                    reinterpret_cast<const uint2*>(pairs), status);
        if (launched != cudaSuccess) {
            return launched;
        }
    }
    return cudaSuccess;
}
