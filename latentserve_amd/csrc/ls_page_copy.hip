// Pages copied to other pages of the same pools: t[dst[i]] = t[src[i]] for every
// tensor t (all layers' K and V pools, scales, bounds) in one launch.
//
// Bound by HBM (160 pages of 56 pools, 147 MB read and written: 26.4 us, 5.6 TB/s), and
// for a few pages by the launch itself (8 pages: 2.6 us): the pointers, strides and page
// numbers travel in the kernel's arguments, so a branch of a sequence costs one launch
// and no transfer.

#include "ls_common.h"
#include "ls_serving.h"

namespace ls {

constexpr int COPY_THREADS = 256;

// (blockIdx.x: pair, blockIdx.y: tensor)
template <class T>
__global__ __launch_bounds__(COPY_THREADS) void page_copy_kernel(const PageCopyParams a) {
    const int i = blockIdx.x, k = blockIdx.y;
    const int64_t stride = a.stride[k];
    const T* src = (const T*)(a.base[k] + a.src[i] * stride);
    T* dst = (T*)(a.base[k] + a.dst[i] * stride);
    const int n = a.bytes[k] / (int)sizeof(T);
    // Two pieces a thread at a time; the source past the caches (read once, unless it
    // goes to several pages, then the lines are there for a while all the same), the
    // copy through them: the next step's attention reads it.  (One piece, through the
    // caches: 160 pages of 8 KB by 56 tensors take 5 us more.)
    for (int e = threadIdx.x; e < n; e += 2 * COPY_THREADS) {
        const int e2 = e + COPY_THREADS;
        const T v = stream_load(src + e), v2 = stream_load(src + (e2 < n ? e2 : e));
        dst[e] = v;
        if (e2 < n) dst[e2] = v2;
    }
}

hipError_t launch_page_copy(const PageCopyParams& a, int tensors, int pairs, int vec,
                            hipStream_t stream) {
    const dim3 grid(pairs, tensors), block(COPY_THREADS);
    if (vec == 16) hipLaunchKernelGGL(page_copy_kernel<u4>, grid, block, 0, stream, a);
    else if (vec == 8) hipLaunchKernelGGL(page_copy_kernel<u2>, grid, block, 0, stream, a);
    else if (vec == 4) hipLaunchKernelGGL(page_copy_kernel<uint32_t>, grid, block, 0, stream, a);
    else if (vec == 2) hipLaunchKernelGGL(page_copy_kernel<uint16_t>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(page_copy_kernel<uint8_t>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace ls
