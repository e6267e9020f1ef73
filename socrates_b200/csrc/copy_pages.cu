// Copies of cache pages inside the pools of one cache group: pool[r, dst_i] = pool[r, src_i] for every layer run r, keys
// and values, in one launch.  What a fork of a row takes: whole pages are shared, the page that both rows will go on
// writing is copied.
//
// What bounds it: bytes, each read once and written once (63 pages of 64 KB through 64 layer runs: 80 us, 6.55 TB/s; one page
// through 36: 8.5 us a call, the host's).  The pairs come from the host as a launch argument, so nothing is copied to the
// device first and the host has checked every number before the kernel sees it.
#include <memory>
#include <new>

#include "common.cuh"

namespace {

template <int N> struct Pairs { int src[N], dst[N]; };
constexpr int FEW = 32, SOME = 512, MANY = 2000;      // pairs of one launch (its arguments are 256 bytes, 4 or 16 KB)
constexpr int THREADS = 256, UNROLL = 4;     // a block copies 256 x 4 vectors: 16 KB with 16-byte vectors

// grid.x = pieces x 2 (keys, values) x pairs x runs, in that order from the fastest; V: the vector that divides a page
template <typename V, int N>
__global__ void __launch_bounds__(THREADS)
copy_pages_kernel(V* k, V* v, const __grid_constant__ Pairs<N> pairs, int n, long long k_run, long long v_run, int k_page,
                  int v_page, int pieces) {
    // No launch_dependents, and a fence at the end: kernels that read pages before their own wait must find the copies done.
    sb::pdl_wait();
    long long b = blockIdx.x;
    const int piece = (int)(b % pieces);
    b /= pieces;
    const bool values = b & 1;
    b >>= 1;
    const int pair = (int)(b % n);
    const long long run = b / n;
    const int page = values ? v_page : k_page;
    V* pool = values ? v + run * v_run : k + run * k_run;
    const V* from = pool + (long long)pairs.src[pair] * page;
    V* to = pool + (long long)pairs.dst[pair] * page;
    const int at = piece * THREADS * UNROLL + threadIdx.x;
    V x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
        if (at + u * THREADS < page) x[u] = from[at + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
        if (at + u * THREADS < page) to[at + u * THREADS] = x[u];
    __threadfence();
}

template <typename V, int N>
int launch_pairs(void* k, void* v, const int* src, const int* dst, int n, int runs, long long pages, long long k_bytes,
                 long long v_bytes, cudaStream_t stream) {
    Pairs<N> p;
    for (int i = 0; i < n; ++i) {
        p.src[i] = src[i];
        p.dst[i] = dst[i];
    }
    const int kp = (int)(k_bytes / (long long)sizeof(V)), vp = (int)(v_bytes / (long long)sizeof(V));
    const int per = THREADS * UNROLL;
    const int pieces = ((kp > vp ? kp : vp) + per - 1) / per;
    const long long blocks = 2ll * pieces * n * runs;
    SB_REQUIRE(blocks <= 0x7fffffffll, "copy_pages: %lld blocks are too many for one launch", blocks);
    sb::launch(copy_pages_kernel<V, N>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, (V*)k, (V*)v, p, n, pages * kp,
               pages * vp, kp, vp, pieces);
    return 0;
}

template <typename V>
int launch_vec(void* k, void* v, const int* src, const int* dst, int n, int runs, long long pages, long long k_bytes,
               long long v_bytes, cudaStream_t stream) {
    for (int i = 0; i < n; i += MANY) {
        const int m = n - i < MANY ? n - i : MANY;
        const int rc = m <= FEW ? launch_pairs<V, FEW>(k, v, src + i, dst + i, m, runs, pages, k_bytes, v_bytes, stream)
                      : m <= SOME ? launch_pairs<V, SOME>(k, v, src + i, dst + i, m, runs, pages, k_bytes, v_bytes, stream)
                                  : launch_pairs<V, MANY>(k, v, src + i, dst + i, m, runs, pages, k_bytes, v_bytes, stream);
        if (rc != 0) return rc;
    }
    SB_LAUNCH_CHECK();
}

}  // namespace

// How many kernels a copy of n pairs launches.
extern "C" int sb_copy_pages_kernels(int n) { return n <= 0 ? 0 : (n + MANY - 1) / MANY; }

// k, v: pools [runs, pages, page bytes]; src, dst: n page numbers each, on the HOST (read before the call returns).  A page
// may be copied to several places; nothing is written twice, and no page is both read and written.
extern "C" int sb_copy_pages(void* k, void* v, const int* src, const int* dst, int n, int runs, int pages,
                             long long k_bytes, long long v_bytes, cudaStream_t stream) {
    SB_REQUIRE(n >= 0 && runs > 0 && pages > 0 && k_bytes > 0 && v_bytes > 0 && k_bytes < (1ll << 30) && v_bytes < (1ll << 30),
               "copy_pages: bad sizes (%d pairs, %d runs, %d pages of %lld and %lld bytes)", n, runs, pages, k_bytes, v_bytes);
    if (n == 0) return 0;
    SB_REQUIRE(n < pages, "copy_pages: %d copies into a pool of %d pages", n, pages);
    SB_REQUIRE(k != nullptr && v != nullptr && src != nullptr && dst != nullptr, "copy_pages: a pointer is missing");
    for (int i = 0; i < n; ++i)
        SB_REQUIRE(src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages,
                   "copy_pages: page %d to %d of a pool of %d", src[i], dst[i], pages);
    if (n <= FEW) {                                          // pair by pair; a map of the pool costs more than it saves
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < n; ++j) {
                SB_REQUIRE(i == j || dst[i] != dst[j], "copy_pages: page %d is written twice", dst[i]);
                SB_REQUIRE(dst[i] != src[j], "copy_pages: page %d is read and written", dst[i]);
            }
    } else {
        std::unique_ptr<char[]> written(new (std::nothrow) char[pages]());
        SB_REQUIRE(written != nullptr, "copy_pages: no host memory for a map of %d pages", pages);
        for (int i = 0; i < n; ++i) {
            SB_REQUIRE(!written[dst[i]], "copy_pages: page %d is written twice", dst[i]);
            written[dst[i]] = 1;
        }
        for (int i = 0; i < n; ++i)
            SB_REQUIRE(!written[src[i]], "copy_pages: page %d is read and written", src[i]);
    }
    const uintptr_t all = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (uintptr_t)k_bytes | (uintptr_t)v_bytes;
    if (all % 16 == 0) return launch_vec<uint4>(k, v, src, dst, n, runs, pages, k_bytes, v_bytes, stream);
    if (all % 4 == 0) return launch_vec<uint32_t>(k, v, src, dst, n, runs, pages, k_bytes, v_bytes, stream);
    SB_REQUIRE(all % 2 == 0, "copy_pages: elements of one byte are not supported");
    return launch_vec<uint16_t>(k, v, src, dst, n, runs, pages, k_bytes, v_bytes, stream);
}
