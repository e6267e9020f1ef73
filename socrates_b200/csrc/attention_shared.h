// The parts of the attention over a shared prefix: the lists of a call, the walk of small units and own keys
// (attention_shared_mma.cu) and the large families' shared keys (attention_shared_tc.cu).  The entry point is in
// attention_shared.cu.
#pragma once

#include <cuda_runtime.h>

namespace sb {

struct SharedLists {
    const int *block_table, *token_rows, *positions, *members, *group_starts, *shared_lens;
    int table_width, M, R;
};

constexpr int TC_ROWS = 128;                     // query rows of a large family's unit
constexpr int TC_SMEM_MOST = 112 * 1024;         // two blocks an SM
constexpr long long TC_PRODUCTS = 1 << 18;

// Whether a family of n tokens goes to the kernel for large ones: by its products, rows x keys.  Measured (us a call in a graph,
// keys in no cache, 8 KV heads of 128, a hundred keys of its own a token; that kernel / units of 16 rows): 64 rows behind 1,024
// keys 25 / 18, 4,096 28 / 29, 8,192 30 / 47; 128 rows behind 1,024 30 / 25, 4,096 34 / 49; 256 rows behind 256 33 / 28, 1,024
// 37 / 37, 4,096 44 / 86, 8,192 53 / 150.
__host__ __device__ inline bool tc_family(int n, int G, int shared) {
    return n * G > 32 && (long long)n * G * shared >= TC_PRODUCTS;
}
// Units that the large families of M members in R groups can have: each has more than 32 rows.
__host__ __device__ inline int tc_units(int M, int R, int G) {
    const int families = M * G / 33;
    return M * G / TC_ROWS + (families < R ? families : R);
}

// T tiles in `pieces` pieces of equal length.
struct Cut {
    int T, pieces;
    __device__ __forceinline__ int begin(int c) const { return (int)((long long)c * T / pieces); }
    // the piece that tile x lies in
    __device__ __forceinline__ int of(int x) const { return (int)(((long long)(x + 1) * pieces + T - 1) / T) - 1; }
    // Where the partial results of an item with tiles [from, end) lie: its first piece (bit 31: that piece's second result, as
    // the end of another item is its first) and the end of its pieces.
    __device__ __forceinline__ int2 parts(int from, int end) const {
        if (end <= from) return make_int2(0, 0);
        const int s = of(from);
        return make_int2(from <= begin(s) ? s : s | (int)0x80000000u, of(end - 1) + 1);
    }
};

// Partial results of the large families' units, and what the joining kernel needs to find them.
struct TcPart {
    float *whole_o, *whole_ml;                   // [Hkv][units][128][D] and [..][2]
    float *piece_o, *piece_ml;                   // [Hkv][W][2][128][D] and [..][2]
    // Per call, eight entries a member: the flat row of its first head among the rows of the units (-1: none), the parts of that
    // row's unit and of the next one (Cut::parts), those of the walk's own item, the token.  Null: not used.
    int* items;
    int W;                                       // shares of a KV head
};

bool shared_tc_supports(int M, int R, int Hq, int Hkv, int D, int page_size, long long num_pages);
int shared_tc(const TcPart& part, const void* q, const void* k_pool, const void* v_pool, const SharedLists& l, int Hq, int Hkv,
              int D, int page_size, long long num_pages, int window, float scale, int* status, cudaStream_t stream);

bool shared_stream_supports(int M, int R, int Hq, int Hkv, int D, int page_size);
void shared_stream_scratch(int M, int R, int Hq, int Hkv, int D, int page_size, int num_sms, long long* floats, long long* ints);
int shared_stream(void* out, float* part, int* items, const void* q, const void* k_pool, const void* v_pool,
                  const SharedLists& l, int Hq, int Hkv, int D, int page_size, long long num_pages, int window, float scale,
                  int num_sms, int* status, cudaStream_t stream);

}  // namespace sb
