// Pages of a cache, copied.
//
// copy_pages_kernel: a workgroup moves up to 16 KiB of one page of one tensor, four 16-byte pieces a lane on their way at once.  Bound by HBM:
// a read and a write of each page (552 MB read and written: 111 us, 4.97 TB/s, what a large copy reaches); in small calls by the launch (3.1 us, the call 5.7),
// which is why keys, values and scales of several layers go in one.
#include <hip/hip_runtime.h>

#include "cq_attention_internal.hpp"
#include "cq_device.hpp"

namespace cq {
namespace {

constexpr uint32_t kPieces = 4, kChunk = kCopyAccesses;  // accesses of a lane and of a workgroup
static_assert(kChunk == 256 * kPieces);

template <class T>
__device__ __forceinline__ void copy_chunk(const char* from, char* to, uint64_t bytes, uint64_t chunk) {
    const uint64_t n = bytes / sizeof(T), first = chunk * kChunk + threadIdx.x;
    T v[kPieces];
#pragma unroll
    for (uint32_t i = 0; i < kPieces; i++)
        if (first + i * 256u < n) v[i] = reinterpret_cast<const T*>(from)[first + i * 256u];
#pragma unroll
    for (uint32_t i = 0; i < kPieces; i++)
        if (first + i * 256u < n) reinterpret_cast<T*>(to)[first + i * 256u] = v[i];
}

__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a, uint32_t pair0) {
    const CopyArgs::Pool& pool = a.pools[blockIdx.y];
    const uint32_t pair = pair0 + blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    if (static_cast<uint64_t>(chunk) * kChunk * pool.unit >= pool.bytes) return;
    const int32_t from = a.pairs[2ull * pair], to = a.pairs[2ull * pair + 1ull];
    const auto inside = [&](int32_t page) { return page >= 0 && static_cast<uint32_t>(page) < pool.pages; };
    if (!inside(from) || !inside(to) || from == to) return;
    const char* const source = pool.base + static_cast<uint64_t>(from) * pool.stride;
    char* const target = pool.base + static_cast<uint64_t>(to) * pool.stride;
    if (pool.unit == 16)
        copy_chunk<u32x4>(source, target, pool.bytes, chunk);
    else if (pool.unit == 4)
        copy_chunk<uint32_t>(source, target, pool.bytes, chunk);
    else
        copy_chunk<char>(source, target, pool.bytes, chunk);
}

}  // namespace

hipError_t launch_copy(hipStream_t s, const CopyArgs& args, uint32_t tensors) {
    CopyArgs a = args;
    uint64_t chunks = 1;
    for (uint32_t t = 0; t < tensors; t++) {
        const uint64_t n = copy_groups(a.pools[t]);  // kMostCopyGroups at most, as cq_cache_copy has seen to
        chunks = n > chunks ? n : chunks;
    }
    a.chunks = static_cast<uint32_t>(chunks);
    const uint32_t piece = static_cast<uint32_t>(kMostCopyGroups / chunks);
    for (uint64_t pair = 0; pair < a.count; pair += piece) {
        const uint32_t n = a.count - pair < piece ? static_cast<uint32_t>(a.count - pair) : piece;
        hipLaunchKernelGGL(copy_pages_kernel, dim3(n * a.chunks, tensors), dim3(256), 0, s, a, static_cast<uint32_t>(pair));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cq
