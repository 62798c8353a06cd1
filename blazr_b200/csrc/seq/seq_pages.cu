// seq_pages.cu -- pages copied inside every pool of a model in one launch (a forked request's last page, a compaction of the cache).
//
// A step between two steps of a serving loop: few bytes in many places.  The (from, to) pairs and the pools travel in the launch's own parameters, so a
// copy is one launch with no upload before it; nothing of it is kept.  Bounded by the memory, 2 bytes a byte copied (700 pages of 32 KB in 8 pools: 57.5 us, 6.4 TB/s), or by
// the launch (4 pages in 16 pools: 1.9 us).
#include <cstring>
#include <vector>

#include "seq_common.cuh"

namespace b200seq {

namespace {

constexpr int POOLS = 32, FEW = 56, MANY = 1400;
constexpr int THREADS = 256, CHUNK = THREADS * 16 * 4;   // bytes of a block's share of a page

template <int N>
struct PageCopy {
    uint8_t* pool[POOLS];
    int64_t bytes[POOLS];   // of one page
    int2 pair[N];           // from, to
};

template <class V>
__device__ __forceinline__ void copy_run(const V* src, V* dst, int64_t n) {
    int64_t i = threadIdx.x;
    for (; i + 3 * THREADS < n; i += 4 * THREADS) {
        V x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = src[i + j * THREADS];
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[i + j * THREADS] = x[j];
    }
    for (; i < n; i += THREADS) dst[i] = src[i];
}

// grid (pairs, pools, parts of a page)
template <int N>
__global__ void __launch_bounds__(THREADS) copy_pages_kernel(const __grid_constant__ PageCopy<N> c) {
    chain_enter();
    uint8_t* pool = c.pool[blockIdx.y];
    const int64_t bytes = c.bytes[blockIdx.y];
    const int2 pair = c.pair[blockIdx.x];
    const uint8_t* src = pool + pair.x * bytes;
    uint8_t* dst = pool + pair.y * bytes;
    const bool wide = ((reinterpret_cast<uintptr_t>(pool) | (uintptr_t)bytes) & 15) == 0;
    for (int64_t at = (int64_t)blockIdx.z * CHUNK; at < bytes; at += (int64_t)gridDim.z * CHUNK) {
        const int64_t n = min((int64_t)CHUNK, bytes - at);
        if (wide) copy_run(reinterpret_cast<const uint4*>(src + at), reinterpret_cast<uint4*>(dst + at), n / 16);
        else copy_run(src + at, dst + at, n);
    }
}

template <int N>
int run(void* const* pools, const int64_t* bytes, int npools, const int32_t* pairs, int n, cudaStream_t cs) {
    for (int p0 = 0; p0 < npools; p0 += POOLS) {
        PageCopy<N> c;
        const int np = npools - p0 < POOLS ? npools - p0 : POOLS;
        int64_t most = 0;
        for (int i = 0; i < POOLS; ++i) {
            c.pool[i] = i < np ? (uint8_t*)pools[p0 + i] : nullptr, c.bytes[i] = i < np ? bytes[p0 + i] : 0;
            most = c.bytes[i] > most ? c.bytes[i] : most;
        }
        if (most == 0) continue;
        for (int q0 = 0; q0 < n; q0 += N) {
            const int nq = n - q0 < N ? n - q0 : N;
            std::memcpy(c.pair, pairs + 2 * q0, (size_t)nq * 8);
            const int64_t parts = (most + CHUNK - 1) / CHUNK;
            launch_chained(copy_pages_kernel<N>, dim3(nq, np, (unsigned)(parts < 65535 ? parts : 65535)), THREADS, 0, cs, c);
            SEQ_LAUNCH_CHECK("copy_pages");
        }
    }
    return 0;
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" int b200seq_copy_pages(void* const* pools, const int64_t* page_bytes, int npools, int pages, const int32_t* pairs, int n, void* stream) {
    if (npools < 0 || pages < 0 || n < 0 || (npools > 0 && (!pools || !page_bytes)) || (n > 0 && !pairs)) return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: bad arguments");
    for (int i = 0; i < npools; ++i)
        if (!pools[i] || page_bytes[i] < 0) return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: pool %d is null or its pages have no size", i);
    // A copy's result does not depend on the order of its pairs: no page is written twice, none is both read and written.
    for (int i = 0; i < 2 * n; ++i)
        if (pairs[i] < 0 || pairs[i] >= pages)
            return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: pair %d names a page outside the pool's %d (%d -> %d)", i / 2, pages, pairs[i & ~1], pairs[i | 1]);
    try {
        std::vector<bool> written((size_t)pages, false);
        for (int i = 0; i < n; ++i) {
            if (written[pairs[2 * i + 1]]) return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: page %d is written twice by one call", pairs[2 * i + 1]);
            written[pairs[2 * i + 1]] = true;
        }
        for (int i = 0; i < n; ++i)
            if (written[pairs[2 * i]]) return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: page %d is both read and written by one call", pairs[2 * i]);
    } catch (const std::exception&) {
        return fail(B200SEQ_ERR_INVALID_ARG, "copy_pages: no memory for the check of %d pages", pages);
    }
    if (n == 0 || npools == 0) return 0;
    return n <= FEW ? run<FEW>(pools, page_bytes, npools, pairs, n, (cudaStream_t)stream) : run<MANY>(pools, page_bytes, npools, pairs, n, (cudaStream_t)stream);
}
