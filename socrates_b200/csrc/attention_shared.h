// The parts of the attention over a shared prefix: the lists of a call, and the tensor-core form (attention_shared_mma.cu) that
// the entry point in attention_shared.cu chooses where it serves.
#pragma once

#include <cuda_runtime.h>

namespace sb {

struct SharedLists {
    const int *block_table, *token_rows, *positions, *members, *group_starts, *shared_lens;
    int table_width, M, R;
};

bool shared_stream_supports(int M, int R, int Hq, int Hkv, int D, int page_size);
void shared_stream_scratch(int M, int R, int Hq, int Hkv, int D, int num_sms, long long* floats, long long* ints);
int shared_stream(void* out, float* part, int* items, const void* q, const void* k_pool, const void* v_pool,
                  const SharedLists& l, int Hq, int Hkv, int D, int page_size, int window, float scale, int num_sms,
                  cudaStream_t stream);

}  // namespace sb
