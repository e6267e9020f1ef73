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
// memory: the order does not matter), so no table as wide as the vocabulary is kept from step to step.  What bounds it: the
// logits' bytes and, for rows that draw, two logarithms a logit.  A thread holds its 16 logits in registers, loaded (16 bytes
// each where rows allow it) before the counts are made; logits of tokens that a mask forbids are not read.
//
// A row that draws needs the noise of few logits: with N = 2^23 - (hash >> 9) in [1, 2^23] the noise -log(-log(u)) is at most
// -log(1 - u) = log(2^23 / (N - 1/2)).  A block first takes the largest of the scores of its threads' largest logits; a logit l
// can exceed that, F, only where N - 1/2 <= 2^23 e^(l / T - F), and the others are not looked at.
// 64 rows of 151,936 logits, half of them drawn, tokens of up to 4,096 and 40 biases a row: 60 us a logit at a time, 42 so.
__global__ void __launch_bounds__(512, 2)
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
    constexpr int THREADS = 512, J = SLICE / (4 * THREADS);  // four times four logits a thread
    const int m = blockIdx.x, C = gridDim.y, tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    const float* row = logits + (size_t)m * V;
    const int begin = min(V, (int)blockIdx.y * per), end = min(V, begin + per);
    // logit (j, e) of a thread is `at + 2048 j + step e`: neighbours where 16-byte loads are possible
    const bool wide = V % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(a.adjusted)) & 15) == 0;
    const int at = begin + (wide ? 4 * tid : tid), step = wide ? 1 : THREADS;

    const int mask_row = a.mask != nullptr ? a.mask_rows[m] : -1;
    uint32_t may = 0xffffu;                                 // bit 4 j + e: the token is allowed
    if (mask_row >= 0) {
        const uint32_t* allowed = a.mask + (size_t)mask_row * a.mask_words;
        may = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = at + 4 * THREADS * j;
            if (wide) {
                if (i < end) may |= (allowed[i >> 5] >> (i & 31) & 15u) << (4 * j);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + step * e < end) may |= (allowed[(i + step * e) >> 5] >> ((i + step * e) & 31) & 1u) << (4 * j + e);
            }
        }
    }
    // a place behind the slice holds NaN, which is never the best, one that is not allowed -inf
    float v[4 * J];
    const float none = __int_as_float(0x7fffffff);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = at + 4 * THREADS * j;
        float4 x = make_float4(none, none, none, none);
        if (wide) {
            if (i < end) x = may >> (4 * j) & 15u ? *reinterpret_cast<const float4*>(row + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
            if (i < end) x.x = row[i];
            if (i + step < end) x.y = row[i + step];
            if (i + 2 * step < end) x.z = row[i + 2 * step];
            if (i + 3 * step < end) x.w = row[i + 3 * step];
        }
        v[4 * j] = x.x; v[4 * j + 1] = x.y; v[4 * j + 2] = x.z; v[4 * j + 3] = x.w;
    }
    const float T = temperature ? temperature[m] : 0.f;
    uint32_t key = 0;
    if (T > 0.f) {
        key = mix32(seeds[m] ^ 0x9E3779B9u);
        key = mix32(key ^ mix32(counters[m] + 0x85EBCA6Bu));
    }
    const float inv_t = T > 0.f ? 1.0f / T : 1.0f;

    // ---- counts and biases of the slice's tokens
    const bool penal = a.history != nullptr, biased = a.bias_starts != nullptr;
    if (penal || biased) {
        const int4 zero = make_int4(0, 0, 0, 0);
        for (int i = 4 * tid; i < per * (penal + biased); i += 4 * THREADS) *reinterpret_cast<int4*>(count + i) = zero;
        __syncthreads();
    }
    float rep = 1.f, presence = 0.f, frequency = 0.f;
    const int n = end - begin;
    if (penal) {
        rep = a.penalties[3 * m];
        presence = a.penalties[3 * m + 1];
        frequency = a.penalties[3 * m + 2];
        const int* told = a.history + (size_t)a.history_rows[m] * a.history_width;
        const int len = min(a.lengths[m], a.history_width), prompt = a.prompt_lens[m];
        constexpr int AT = 8;                               // loads in flight
        for (int i0 = tid; i0 < len; i0 += AT * THREADS) {
            int t[AT];
#pragma unroll
            for (int u = 0; u < AT; ++u) t[u] = i0 + u * THREADS < len ? told[i0 + u * THREADS] - begin : -1;
#pragma unroll
            for (int u = 0; u < AT; ++u)
                if (t[u] >= 0 && t[u] < n) {
                    if (i0 + u * THREADS < prompt) atomicOr(&count[t[u]], (int)0x80000000u);
                    else atomicAdd(&count[t[u]], 1);
                }
        }
    }
    if (biased && warp == THREADS / 32 - 1) {
        // in the order of the list, so that a token named twice gets both in that order
        const int e1 = a.bias_starts[m + 1];
        for (int e0 = a.bias_starts[m]; e0 < e1; e0 += 32) {
            const int t = e0 + lane < e1 ? a.bias_ids[e0 + lane] - begin : -1;
            const float x = e0 + lane < e1 ? a.bias_values[e0 + lane] : 0.f;
            const bool mine = t >= 0 && t < n;
            const uint32_t same = __match_any_sync(0xffffffffu, mine ? t : -1 - lane);
            const int rank = __popc(same & ((1u << lane) - 1u));
            const int rounds = __reduce_max_sync(0xffffffffu, rank);
            for (int r = 0; r <= rounds; ++r) {
                if (mine && rank == r) bias[t] += x;
                __syncwarp();
            }
        }
    }
    if (penal || biased) __syncthreads();

    // ---- the adjusted logits
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = at + 4 * THREADS * j;
        if (penal && i < end) {
            int c[4] = {0, 0, 0, 0};
            if (wide) {
                const int4 x = *reinterpret_cast<const int4*>(count + i - begin);
                c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + step * e < end) c[e] = count[i + step * e - begin];
            }
            if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c[e] != 0) {
                        float x = v[4 * j + e];
                        x = x > 0.f ? x / rep : x * rep;
                        const int made = c[e] & 0x7fffffff;
                        v[4 * j + e] = made > 0 ? x - frequency * (float)made - presence : x;
                    }
            }
        }
        if (biased && i < end) {
            if (wide) {
                const float4 x = *reinterpret_cast<const float4*>(bias + i - begin);
                v[4 * j] += x.x; v[4 * j + 1] += x.y; v[4 * j + 2] += x.z; v[4 * j + 3] += x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + step * e < end) v[4 * j + e] += bias[i + step * e - begin];
            }
        }
    }
    if (mask_row >= 0) {
#pragma unroll
        for (int k = 0; k < 4 * J; ++k)
            if (!(may >> k & 1u) && at + 4 * THREADS * (k / 4) + step * (k % 4) < end) v[k] = -INFINITY;
    }
    if (a.adjusted != nullptr) {
        float* to = a.adjusted + (size_t)m * V;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = at + 4 * THREADS * j;
            if (wide) {
                if (i < end) *reinterpret_cast<float4*>(to + i) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + step * e < end) to[i + step * e] = v[4 * j + e];
            }
        }
    }

    // ---- the best of them.  A thread's places come in the order of their indices, so the first of equal ones stays.
    float best = -INFINITY;
    int best_k = -1;
    if (T > 0.f) {
        auto score = [&](float x, int k) {                  // as sample_kernel's, operation by operation
            const float u = uniform_for(key, (uint32_t)(at + 4 * THREADS * (k / 4) + step * (k % 4)));
            return x * inv_t - logf(-logf(u));
        };
        float top = -INFINITY;
        int top_k = -1;
#pragma unroll
        for (int k = 0; k < 4 * J; ++k)
            if (v[k] > top) { top = v[k]; top_k = k; }
        float least = top_k >= 0 ? score(top, top_k) : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) least = fmaxf(least, __shfl_xor_sync(0xffffffffu, least, o));
        if (lane == 0) s_val[warp] = least;
        __syncthreads();
        least = s_val[lane & (THREADS / 32 - 1)];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) least = fmaxf(least, __shfl_xor_sync(0xffffffffu, least, o));
        // l / T in units of log2, less F, and 23: the exponent of the largest N.  2e-3 and 2e-6 of a score are far more than the
        // roundings on both sides.
        constexpr float LOG2E = 1.4426950408889634f;
        const float slope = inv_t * LOG2E, offset = 23.0f + 2e-3f + 2e-6f * fabsf(least) - least * LOG2E;
        uint32_t look = 0;
#pragma unroll
        for (int k = 0; k < 4 * J; ++k) {
            const uint32_t i = (uint32_t)(at + 4 * THREADS * (k / 4) + step * (k % 4));
            const float N = (float)(8388608u - (mix32((i + 0x165667B1u) ^ key) >> 9));
            const float exponent = fmaf(v[k], slope, offset);
            float most;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(most) : "f"(fmaf(fabsf(exponent), 2e-6f, exponent)));
            if (!(N - 0.5f > most)) look |= 1u << k;        // NaN and infinities are looked at
        }
        while (__any_sync(0xffffffffu, look != 0)) {         // in the order of the places
            const int k = __ffs(look) - 1;
            if (k >= 0) {
                float x = v[0];
#pragma unroll
                for (int y = 1; y < 4 * J; ++y) x = k == y ? v[y] : x;
                x = score(x, k);
                if (x > best) { best = x; best_k = k; }
                look &= look - 1;
            }
        }
        __syncthreads();                                    // s_val is written again below
    } else {
#pragma unroll
        for (int k = 0; k < 4 * J; ++k)
            if (v[k] > best) { best = v[k]; best_k = k; }
    }
    int best_i = best_k < 0 ? 0x7fffffff : at + 4 * THREADS * (best_k >> 2) + step * (best_k & 3);
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
                                  const uint32_t* counters, int M, int V, int* scratch, long long scratch_ints,
                                  const int* history, int history_width,
                                  const int* history_rows, const int* prompt_lens, const int* lengths, const float* penalties,
                                  const int* bias_starts, const int* bias_ids, const float* bias_values, const void* mask,
                                  int mask_words, const int* mask_rows, float* adjusted, cudaStream_t stream) {
    SB_REQUIRE(M >= 0 && V > 0, "sample_adjusted: bad sizes M=%d V=%d", M, V);
    SB_REQUIRE(temperature == nullptr || (seeds != nullptr && counters != nullptr),
               "sample_adjusted: temperature sampling needs seeds and counters");
    SB_REQUIRE(scratch != nullptr && scratch_ints >= (long long)M * (2 * sb_sample_slices(V) + 1),
               "sample_adjusted: scratch has %lld entries, %lld are needed", scratch_ints, (long long)M * (2 * sb_sample_slices(V) + 1));
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
