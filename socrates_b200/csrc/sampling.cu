// Sampling over float32 logits: greedy argmax and temperature (Gumbel-max) with a
// counter-based generator, one block per row.  The generator is a function of
// (seed, counter, vocabulary index) alone, so a request's draws do not depend on
// what else is in the batch.
#include "common.cuh"

namespace {

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    x ^= x >> 16;
    return x;
}

// Uniform in (0,1) with 23 random bits, centred in its cell: (k + 0.5) / 2^23 is
// exact in float32 and never 0 or 1.
__device__ __forceinline__ float uniform_for(uint32_t key, uint32_t index) {
    const uint32_t x = mix32((index + 0x165667B1u) ^ key);
    return ((float)(x >> 9) + 0.5f) * (1.0f / 8388608.0f);
}

__device__ __forceinline__ bool better(float v, int i, float best, int best_i) {
    return v > best || (v == best && i < best_i);
}

// The end of a block that looked through a slice of row m: its warps' best (in s_val, s_idx, behind a barrier) become the
// slice's, and the row's last block to come merges the slices (see sample_kernel).
__device__ __forceinline__ void merge_slices(int* __restrict__ out, int* __restrict__ scratch, int m, int C, float best,
                                             int best_i, const float* s_val, const int* s_idx, int* s_last) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* mine = scratch + (size_t)m * (2 * C + 1);
    if (warp == 0) {
        const int nw = (blockDim.x + 31) >> 5;
        best = lane < nw ? s_val[lane] : -INFINITY;
        best_i = lane < nw ? s_idx[lane] : 0x7fffffff;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, best, o);
            const int oi = __shfl_xor_sync(0xffffffffu, best_i, o);
            if (better(ov, oi, best, best_i)) { best = ov; best_i = oi; }
        }
        if (lane == 0) {
            mine[2 * blockIdx.y] = __float_as_int(best);
            mine[2 * blockIdx.y + 1] = best_i;
            __threadfence();
            *s_last = atomicAdd(&mine[2 * C], 1) == C - 1;
        }
    }
    __syncthreads();
    if (!*s_last) return;
    __threadfence();
    if (warp == 0) {
        best = -INFINITY;
        best_i = 0x7fffffff;
        for (int c = lane; c < C; c += 32) {
            const float v = __int_as_float(((volatile int*)mine)[2 * c]);
            const int i = ((volatile int*)mine)[2 * c + 1];
            if (better(v, i, best, best_i)) { best = v; best_i = i; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, best, o);
            const int oi = __shfl_xor_sync(0xffffffffu, best_i, o);
            if (better(ov, oi, best, best_i)) { best = ov; best_i = oi; }
        }
        if (lane == 0) {
            // A row of NaNs or -inf leaves best_i untouched; report index 0 rather than garbage.
            out[m] = best_i == 0x7fffffff ? 0 : best_i;
            mine[2 * C] = 0;
        }
    }
}

// temperature[m] == 0: argmax, ties to the lowest index.
// temperature[m] > 0 : argmax_i (logit_i / T - log(-log u_i)).
// grid (M, C): block c of row m scans one slice of the vocabulary and leaves its best
// (score, index) in `scratch`; the block of a row that finishes last (a counter in
// `scratch`) merges the C candidates and writes out[m].  The merge is an argmax over
// exact values with the index as tie-break, so its order does not matter.
//   scratch: int32 [M, 2*C + 1]; the counters (last entry of each row) are zero before
//   the first call and are reset by the merging block.
__global__ void sample_kernel(int* __restrict__ out, const float* __restrict__ logits,
                              const float* __restrict__ temperature, const uint32_t* __restrict__ seeds,
                              const uint32_t* __restrict__ counters, int V, int* __restrict__ scratch) {
    sb::pdl_launch_dependents();     // the next kernel may begin its prologue
    sb::pdl_wait();                  // everything before this kernel is complete and visible
    __shared__ float s_val[32];
    __shared__ int s_idx[32];
    __shared__ int s_last;
    const int m = blockIdx.x, C = gridDim.y;
    const float* row = logits + (size_t)m * V;
    const float T = temperature ? temperature[m] : 0.f;
    uint32_t key = 0;
    if (T > 0.f) {
        key = mix32(seeds[m] ^ 0x9E3779B9u);
        key = mix32(key ^ mix32(counters[m] + 0x85EBCA6Bu));
    }
    const float inv_t = T > 0.f ? 1.0f / T : 1.0f;
    const int per = ((V + C - 1) / C + 3) & ~3;
    const int begin = min(V, (int)blockIdx.y * per), end = min(V, begin + per);
    float best = -INFINITY;
    int best_i = 0x7fffffff;
    auto look = [&](float v, int i) {
        if (T > 0.f) {
            const float u = uniform_for(key, (uint32_t)i);
            v = v * inv_t - logf(-logf(u));
        }
        if (better(v, i, best, best_i)) { best = v; best_i = i; }
    };
    if (V % 4 == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
        // a slice of 8,192 is four 16-byte loads a thread, all in flight: one round trip where a value at a time took
        // several.  Decode steps of one request 1,111 -> 1,104 us (4B shape), of eight 1,053.1 -> 1,051.2 (32B).
        constexpr int U = 4;
        for (int i0 = begin + 4 * threadIdx.x; i0 < end; i0 += 4 * U * blockDim.x) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 4 * u * blockDim.x;
                if (i < end) v[u] = *reinterpret_cast<const float4*>(row + i);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 4 * u * blockDim.x;
                if (i >= end) break;
                look(v[u].x, i);
                look(v[u].y, i + 1);
                look(v[u].z, i + 2);
                look(v[u].w, i + 3);
            }
        }
    } else {
        for (int i = begin + threadIdx.x; i < end; i += blockDim.x) look(row[i], i);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, best, o);
        const int oi = __shfl_xor_sync(0xffffffffu, best_i, o);
        if (better(ov, oi, best, best_i)) { best = ov; best_i = oi; }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) { s_val[warp] = best; s_idx[warp] = best_i; }
    __syncthreads();
    merge_slices(out, scratch, m, C, best, best_i, s_val, s_idx, &s_last);
}

// What a row's logits go through before they are compared: with c the number of times a token stands in the row's output
// and "met" whether it stands in its prompt or output,
//   l1 = met ? (l > 0 ? l / repetition : l * repetition) : l
//   l2 = l1 - frequency * c - presence * (c > 0),   l3 = l2 + bias,   l4 = allowed ? l3 : -inf.
struct Adjust {
    const int *history, *history_rows, *prompt_lens, *lengths;      // tokens [rows, width]; null: no penalties
    const float* penalties;                                         // [M, 3]: repetition, presence, frequency
    const int *bias_starts, *bias_ids;                              // null: no biases
    const float* bias_values;
    const uint32_t* mask;                                           // [rows, words]; null: no masks
    const int* mask_rows;                                           // [M], -1: none
    float* adjusted;                                                // [M, V], or null
    int history_width, mask_words;
};

constexpr int SLICE = 8192;          // logits of a block, whose counts and biases are held in shared memory

// sample_kernel with adjusted logits.  A block counts the row's tokens that fall into its slice (integer atomics in shared
// memory: the order does not matter), so no table as wide as the vocabulary is kept from step to step.
__global__ void __launch_bounds__(512)
sample_adjusted_kernel(int* __restrict__ out, const float* __restrict__ logits, const float* __restrict__ temperature,
                       const uint32_t* __restrict__ seeds, const uint32_t* __restrict__ counters, int V, int per,
                       int* __restrict__ scratch, const Adjust a) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    int* count = reinterpret_cast<int*>(smem);              // [per]: bit 31 "stands in the prompt", below it c
    float* bias = reinterpret_cast<float*>(smem) + (a.history != nullptr ? per : 0);      // [per]
    __shared__ float s_val[32];
    __shared__ int s_idx[32];
    __shared__ int s_last;
    const int m = blockIdx.x, C = gridDim.y, tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    const float* row = logits + (size_t)m * V;
    const float T = temperature ? temperature[m] : 0.f;
    uint32_t key = 0;
    if (T > 0.f) {
        key = mix32(seeds[m] ^ 0x9E3779B9u);
        key = mix32(key ^ mix32(counters[m] + 0x85EBCA6Bu));
    }
    const float inv_t = T > 0.f ? 1.0f / T : 1.0f;
    const int begin = min(V, (int)blockIdx.y * per), end = min(V, begin + per), n = end - begin;

    const bool penal = a.history != nullptr, biased = a.bias_starts != nullptr;
    float rep = 1.f, presence = 0.f, frequency = 0.f;
    if (penal)
        for (int i = tid; i < n; i += blockDim.x) count[i] = 0;
    if (biased)
        for (int i = tid; i < n; i += blockDim.x) bias[i] = 0.f;
    __syncthreads();
    if (penal) {
        rep = a.penalties[3 * m];
        presence = a.penalties[3 * m + 1];
        frequency = a.penalties[3 * m + 2];
        const int* told = a.history + (size_t)a.history_rows[m] * a.history_width;
        const int len = min(a.lengths[m], a.history_width), prompt = a.prompt_lens[m];
        for (int i = tid; i < len; i += blockDim.x) {
            const int t = told[i] - begin;
            if (t < 0 || t >= n) continue;
            if (i < prompt) atomicOr(&count[t], (int)0x80000000u);
            else atomicAdd(&count[t], 1);
        }
    }
    if (biased && warp == 0) {
        // in the order of the list, so that a token named twice gets both in that order
        const int e1 = a.bias_starts[m + 1];
        for (int e0 = a.bias_starts[m]; e0 < e1; e0 += 32) {
            const int t = e0 + lane < e1 ? a.bias_ids[e0 + lane] - begin : -1;
            const bool mine = t >= 0 && t < n;
            const uint32_t same = __match_any_sync(0xffffffffu, mine ? t : -1 - lane);
            const int rank = __popc(same & ((1u << lane) - 1u));
            const int rounds = __reduce_max_sync(0xffffffffu, rank);
            for (int r = 0; r <= rounds; ++r) {
                if (mine && rank == r) bias[t] += a.bias_values[e0 + lane];
                __syncwarp();
            }
        }
    }
    __syncthreads();

    const int mask_row = a.mask != nullptr ? a.mask_rows[m] : -1;
    const uint32_t* allowed = mask_row >= 0 ? a.mask + (size_t)mask_row * a.mask_words : nullptr;
    float best = -INFINITY;
    int best_i = 0x7fffffff;
    auto adjust = [&](float v, int i) {
        if (penal) {
            const int c = count[i - begin];
            if (c != 0) {
                v = v > 0.f ? v / rep : v * rep;
                const int made = c & 0x7fffffff;
                if (made > 0) v = v - frequency * (float)made - presence;
            }
        }
        if (biased) v += bias[i - begin];
        return v;
    };
    auto look = [&](float v, int i) {
        if (T > 0.f) {
            const float u = uniform_for(key, (uint32_t)i);
            v = v * inv_t - logf(-logf(u));
        }
        if (better(v, i, best, best_i)) { best = v; best_i = i; }
    };
    for (int i = begin + tid; i < end; i += blockDim.x) {
        const bool may = allowed == nullptr || (allowed[i >> 5] >> (i & 31)) & 1u;
        float v = -INFINITY;
        if (may) {
            v = adjust(row[i], i);
            look(v, i);
        }
        if (a.adjusted != nullptr) a.adjusted[(size_t)m * V + i] = v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, best, o);
        const int oi = __shfl_xor_sync(0xffffffffu, best_i, o);
        if (better(ov, oi, best, best_i)) { best = ov; best_i = oi; }
    }
    if (lane == 0) { s_val[warp] = best; s_idx[warp] = best_i; }
    __syncthreads();
    merge_slices(out, scratch, m, C, best, best_i, s_val, s_idx, &s_last);
}


}  // namespace

// How many slices a row of V logits is cut into (so callers can size `scratch`).
extern "C" int sb_sample_slices(int V) {
    int c = (V + 8191) / 8192;
    return c < 1 ? 1 : (c > 32 ? 32 : c);
}

// scratch: int32, at least M * (2 * sb_sample_slices(V) + 1) entries, zero before the first use.
extern "C" int sb_sample(int* out, const float* logits, const float* temperature, const uint32_t* seeds,
                         const uint32_t* counters, int M, int V, int* scratch, cudaStream_t stream) {
    SB_REQUIRE(M >= 0 && V > 0, "sample: bad sizes M=%d V=%d", M, V);
    SB_REQUIRE(temperature == nullptr || (seeds != nullptr && counters != nullptr),
               "sample: temperature sampling needs seeds and counters");
    SB_REQUIRE(scratch != nullptr, "sample: scratch is required");
    SB_REQUIRE(M <= 65535 * 32, "sample: too many rows");
    if (M == 0) return 0;
    dim3 grid(M, sb_sample_slices(V));
    sb::launch(sample_kernel, dim3(grid), dim3(512), 0, stream, out, logits, temperature, seeds, counters, V, scratch);
    SB_LAUNCH_CHECK();
}

// sb_sample with adjusted logits.  history [rows, history_width]: row history_rows[m] holds lengths[m] tokens of which the first
// prompt_lens[m] are the prompt; tokens outside the vocabulary are passed over.  penalties [M, 3].  Biases of row m: entries
// bias_starts[m] .. bias_starts[m + 1] - 1.  mask: bit t % 32 of word t / 32 of row mask_rows[m] allows token t.  `adjusted`
// may be `logits`.  Any of the three parts may be absent (null).
extern "C" int sb_sample_adjusted(int* out, const float* logits, const float* temperature, const uint32_t* seeds,
                                  const uint32_t* counters, int M, int V, int* scratch, const int* history, int history_width,
                                  const int* history_rows, const int* prompt_lens, const int* lengths, const float* penalties,
                                  const int* bias_starts, const int* bias_ids, const float* bias_values, const void* mask,
                                  int mask_words, const int* mask_rows, float* adjusted, cudaStream_t stream) {
    SB_REQUIRE(M >= 0 && V > 0, "sample_adjusted: bad sizes M=%d V=%d", M, V);
    SB_REQUIRE(temperature == nullptr || (seeds != nullptr && counters != nullptr),
               "sample_adjusted: temperature sampling needs seeds and counters");
    SB_REQUIRE(scratch != nullptr, "sample_adjusted: scratch is required");
    SB_REQUIRE(V <= 32 * SLICE, "sample_adjusted: a vocabulary of %d (at most %d)", V, 32 * SLICE);
    SB_REQUIRE(history == nullptr || (history_width > 0 && history_rows != nullptr && prompt_lens != nullptr &&
                                      lengths != nullptr && penalties != nullptr),
               "sample_adjusted: penalties need the rows' tokens, their lengths and the three numbers of each row");
    SB_REQUIRE(bias_starts == nullptr || (bias_ids != nullptr && bias_values != nullptr), "sample_adjusted: biases need ids and values");
    SB_REQUIRE(mask == nullptr || (mask_rows != nullptr && mask_words == (V + 31) / 32), "sample_adjusted: masks of %d words for %d tokens", mask_words, V);
    if (M == 0) return 0;
    const int C = sb_sample_slices(V);
    const int per = ((V + C - 1) / C + 3) & ~3;
    const Adjust a{history, history_rows, prompt_lens, lengths, penalties, bias_starts, bias_ids, bias_values, (const uint32_t*)mask,
                   mask_rows, adjusted, history_width, mask_words};
    const int smem = per * 4 * ((history != nullptr) + (bias_starts != nullptr));
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(sample_adjusted_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * SLICE * 4);
        if (e != cudaSuccess) { sb_set_error("sample_adjusted: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    sb::launch(sample_adjusted_kernel, dim3(M, C), dim3(512), smem, stream, out, logits, temperature, seeds, counters, V, per,
               scratch, a);
    SB_LAUNCH_CHECK();
}
