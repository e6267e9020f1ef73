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

// The end of a block that looked through a part of row m: its warps' best (in s_val, s_idx, behind a barrier) become the
// part's, and the last of the row's C blocks to come merges the parts (see sample_kernel).  `mine`: 2 C entries, `counter`: zero
// before and after.
__device__ __forceinline__ void merge_slices(int* __restrict__ out, int* __restrict__ mine, int* __restrict__ counter, int m, int C,
                                             float best, int best_i, const float* s_val, const int* s_idx, int* s_last) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
            *s_last = atomicAdd(counter, 1) == C - 1;
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
            *counter = 0;
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
    int* mine = scratch + (size_t)m * (2 * C + 1);
    merge_slices(out, mine, mine + 2 * C, m, C, best, best_i, s_val, s_idx, &s_last);
}

// What a row's logits go through before they are compared: with c the number of times a token stands in the row's output
// and "met" whether it stands in its prompt or output,
//   l1 = met ? (l > 0 ? l / repetition : l * repetition) : l
//   l2 = l1 - frequency * c - presence * (c > 0),   l3 = l2 + bias,   l4 = allowed ? l3 : -inf.
struct Adjust {
    const int *history, *history_rows, *prompt_lens, *lengths;      // tokens [rows, width]
    const float* penalties;                                         // [M, 3]: repetition, presence, frequency; null: none
    const int *bias_starts, *bias_ids;                              // null: no biases
    const float* bias_values;
    const uint32_t* mask;                                           // [rows, words]; null: no masks
    const int* mask_rows;                                           // [M], -1: none
    float* adjusted;                                                // [M, V], or null
    int history_width, mask_words;
};

constexpr int SLICE = 8192;          // logits of a block at most, held in shared memory with their tokens' counts

// sample_kernel with adjusted logits.  What bounds it: the logits' bytes, and instructions.  A block brings a slice of a row to
// shared memory and marks in a table beside it which of the slice's tokens the row's tokens and biases name, and how often
// (integer atomics in shared memory: the order does not matter, and no table as wide as the vocabulary is kept from step to step).
// Then whoever named a token takes its mark out of the table, which one thread gets, and adjusts its logit: few logits are met,
// and the scan that follows is a plain one.  Logits of tokens that a mask forbids are not read, four at a time.  Blocks are
// small (three an SM), so that the phases of one, which wait for one another, run beside those of others.
//
// A row that draws needs the noise of few logits: with N = 2^23 - (hash >> 9) in [1, 2^23] the noise -log(-log(u)) is at most
// -log(1 - u) = log(2^23 / (N - 1/2)).  A block first takes the largest of the scores of its threads' largest logits, F; a logit that is at
// most l can exceed it only where N - 1/2 <= 2^23 e^(l / T - F), a bound on the hash that a thread takes once, with its
// largest logit.  The others are not looked at.
// 64 rows of 151,936 logits, half of them drawn, tokens of up to 4,096 and 40 biases a row: 60 us a logit at a time with tables for
// counts and biases, 42 with 16 logits a thread in registers, 30 so (22 if none is drawn, 14 if nothing is adjusted either).
__global__ void __launch_bounds__(512, 3)
sample_adjusted_kernel(int* __restrict__ out, const float* __restrict__ logits, const float* __restrict__ temperature,
                       const uint32_t* __restrict__ seeds, const uint32_t* __restrict__ counters, int V, int per,
                       int* __restrict__ scratch_end, const Adjust a) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    constexpr int THREADS = 512, J = SLICE / (4 * THREADS), AT = 2;
    constexpr int PROMPT = (int)0x80000000u, BIASED = 0x40000000, TWICE = 0x20000000, MADE = TWICE - 1;
    extern __shared__ __align__(16) uint8_t smem[];
    float* lg = reinterpret_cast<float*>(smem);             // [per] the slice's logits
    int* marks = reinterpret_cast<int*>(lg + per);          // [per]: PROMPT, BIASED, TWICE (so), times in the output
    __shared__ float s_val[32];
    __shared__ int s_idx[32];
    __shared__ int s_last;
    const int m = blockIdx.x, slices = gridDim.y, tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    const float* row = logits + (size_t)m * V;
    const int begin = min(V, (int)blockIdx.y * per), n = min(V, begin + per) - begin;
    const bool wide = V % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(a.adjusted)) & 15) == 0;

    const bool penal = a.penalties != nullptr, biased = a.bias_starts != nullptr;
    const int* told = nullptr;
    int len = 0, prompt = 0, bias0 = 0, bias1 = 0;
    float rep = 1.f, presence = 0.f, frequency = 0.f;
    if (penal) {
        told = a.history + (size_t)a.history_rows[m] * a.history_width;
        len = min(a.lengths[m], a.history_width);
        prompt = a.prompt_lens[m];
        rep = a.penalties[3 * m];
        presence = a.penalties[3 * m + 1];
        frequency = a.penalties[3 * m + 2];
    }
    if (biased) {
        bias0 = a.bias_starts[m];
        bias1 = a.bias_starts[m + 1];
    }
    const float T = temperature ? temperature[m] : 0.f;
    uint32_t key = 0;
    if (T > 0.f) {
        key = mix32(seeds[m] ^ 0x9E3779B9u);
        key = mix32(key ^ mix32(counters[m] + 0x85EBCA6Bu));
    }

    // four logits a thread and round: 4 (tid + 512 j) .. + 3 of the slice.  `begin` is a multiple of 4: the four lie in one word of
    // the mask.
    const int mask_row = a.mask != nullptr ? a.mask_rows[m] : -1;
    uint32_t may = 0xffffu;                                 // bit 4 j + e: the token is allowed
    if (mask_row >= 0) {
        const uint32_t* allowed = a.mask + (size_t)mask_row * a.mask_words;
        may = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = 4 * (tid + THREADS * j);
            if (i < n) may |= (allowed[(begin + i) >> 5] >> ((begin + i) & 31) & 15u) << (4 * j);
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = 4 * (tid + THREADS * j);
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(lg + i));
        if (i < n && (may >> (4 * j) & 15u)) {
            if (wide) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(row + begin + i) : "memory");
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < n)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * e), "l"(row + begin + i + e) : "memory");
            }
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");

    if (penal || biased) {
        const bool wide_told = (reinterpret_cast<uintptr_t>(told) & 15) == 0;
        auto tokens = [&](int i) {                          // four from i on, less `begin`; behind the row's last one: none
            int4 x = make_int4(-1, -1, -1, -1);
            if (wide_told && i + 3 < len) {
                x = *reinterpret_cast<const int4*>(told + i);
            } else {
                if (i < len) x.x = told[i];
                if (i + 1 < len) x.y = told[i + 1];
                if (i + 2 < len) x.z = told[i + 2];
                if (i + 3 < len) x.w = told[i + 3];
            }
            x.x -= begin; x.y -= begin; x.z -= begin; x.w -= begin;
            return x;
        };
        int4 t[AT];                                         // the first 4,096 tokens
#pragma unroll
        for (int u = 0; u < AT; ++u) t[u] = tokens(4 * (tid + u * THREADS));
        // the first 512 biases, one a thread
        int named = -1;
        float bias = 0.f;
        if (bias0 + tid < bias1) {
            named = a.bias_ids[bias0 + tid] - begin;
            bias = a.bias_values[bias0 + tid];
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (4 * (tid + THREADS * j) < per) reinterpret_cast<int4*>(marks)[tid + THREADS * j] = make_int4(0, 0, 0, 0);
        __syncthreads();
        // f(token - begin, place in the list) for the row's tokens that lie in the slice, f(token - begin, bias) for its biases.
        // (A token outside the vocabulary lies in no slice: what it is less `begin` is negative or, wrapped round, far too large.)
        auto each = [&](auto f) {
            auto one = [&](int x, int i) {
                if ((unsigned)x < (unsigned)n) f(x, i);
            };
            auto four = [&](const int4& x, int i) { one(x.x, i); one(x.y, i + 1); one(x.z, i + 2); one(x.w, i + 3); };
#pragma unroll
            for (int u = 0; u < AT; ++u) four(t[u], 4 * (tid + u * THREADS));
            for (int i0 = AT * THREADS; 4 * i0 < len; i0 += AT * THREADS) {
                int4 x[AT];
#pragma unroll
                for (int u = 0; u < AT; ++u) x[u] = tokens(4 * (i0 + tid + u * THREADS));
#pragma unroll
                for (int u = 0; u < AT; ++u) four(x[u], 4 * (i0 + tid + u * THREADS));
            }
        };
        auto each_bias = [&](auto f) {
            if ((unsigned)named < (unsigned)n) f(named, bias);
            for (int e = bias0 + THREADS + tid; e < bias1; e += THREADS) {
                const int x = a.bias_ids[e] - begin;
                if ((unsigned)x < (unsigned)n) f(x, a.bias_values[e]);
            }
        };
        each([&](int x, int i) {
            if (i < prompt) atomicOr(&marks[x], PROMPT);
            else atomicAdd(&marks[x], 1);
        });
        each_bias([&](int x, float) {
            if (atomicOr(&marks[x], BIASED) & BIASED) atomicOr(&marks[x], TWICE);
        });
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        auto adjust = [&](int x, bool knows, float value) {
            const int c = atomicExch(&marks[x], 0);          // whoever else names this token gets 0
            if (c == 0) return;
            float l = lg[x];
            const int made = c & MADE;
            if (c & (PROMPT | MADE)) l = l > 0.f ? l / rep : l * rep;       // one rounding, as the formula has it
            if (made > 0) l = l - frequency * (float)made - presence;
            if (c & BIASED) {
                if (knows && !(c & TWICE)) l += value;
                else                                        // in the order of the list: a token named twice gets both so
                    for (int e = bias0; e < bias1; ++e)
                        if (a.bias_ids[e] == begin + x) l += a.bias_values[e];
            }
            lg[x] = l;
        };
        each_bias([&](int x, float value) { adjust(x, true, value); });
        each([&](int x, int) { adjust(x, false, 0.f); });
    } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();

    // ---- the scan.  A place behind the slice holds NaN, which is never the best, one that is not allowed -inf.  A thread's places
    // come in the order of their indices: the first of equal ones stays.
    const float none = __int_as_float(0x7fffffff);
    auto four = [&](int j) {
        const int i = 4 * (tid + THREADS * j);
        float4 x = make_float4(none, none, none, none);
        if (i < n) x = *reinterpret_cast<const float4*>(lg + i);
        if (mask_row >= 0) {
            if (!(may >> (4 * j) & 1u)) x.x = -INFINITY;
            if (!(may >> (4 * j) & 2u)) x.y = -INFINITY;
            if (!(may >> (4 * j) & 4u)) x.z = -INFINITY;
            if (!(may >> (4 * j) & 8u)) x.w = -INFINITY;
        }
        if (i + 3 >= n) {
            if (i >= n) x.x = none;
            if (i + 1 >= n) x.y = none;
            if (i + 2 >= n) x.z = none;
            x.w = none;
        }
        return x;
    };
    float best = -INFINITY;
    int best_k = -1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float4 x = four(j);
        if (x.x > best) { best = x.x; best_k = 4 * j; }
        if (x.y > best) { best = x.y; best_k = 4 * j + 1; }
        if (x.z > best) { best = x.z; best_k = 4 * j + 2; }
        if (x.w > best) { best = x.w; best_k = 4 * j + 3; }
        if (a.adjusted != nullptr) {
            const int i = 4 * (tid + THREADS * j);
            float* to = a.adjusted + (size_t)m * V + begin + i;
            if (wide) {
                if (i < n) *reinterpret_cast<float4*>(to) = x;
            } else {
                if (i < n) to[0] = x.x;
                if (i + 1 < n) to[1] = x.y;
                if (i + 2 < n) to[2] = x.z;
                if (i + 3 < n) to[3] = x.w;
            }
        }
    }
    const int first = begin + 4 * tid;
    auto place = [&](int k) { return first + 4 * THREADS * (k >> 2) + (k & 3); };
    if (T > 0.f) {
        const float inv_t = 1.0f / T;
        auto score = [&](float x, int k) {                  // as sample_kernel's, operation by operation
            const float u = uniform_for(key, (uint32_t)place(k));
            return x * inv_t - logf(-logf(u));
        };
        float least = best_k >= 0 ? score(best, best_k) : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) least = fmaxf(least, __shfl_xor_sync(0xffffffffu, least, o));
        if (lane == 0) s_val[warp] = least;
        __syncthreads();
        least = s_val[lane & (THREADS / 32 - 1)];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) least = fmaxf(least, __shfl_xor_sync(0xffffffffu, least, o));
        // The bound on N and from it the one on the hash.  The exponent is enlarged by 2e-3 and 4e-6 of its terms, far more than the
        // roundings on both sides; whatever is not finite looks at everything.
        constexpr float LOG2E = 1.4426950408889634f;
        auto bound = [&](float x) {
            const float l = x * inv_t, exponent = (l - least) * LOG2E + 2e-3f + 4e-6f * (fabsf(l) + fabsf(least));
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(23.0f + exponent));
            return exponent < 0.f ? e + 1.0f : 8388608.0f;
        };
        const uint32_t hash = (8388608u - (uint32_t)fminf(bound(best), 8388608.0f)) << 9;
        uint32_t look = 0;
        if (best_k >= 0) {                                  // else nothing of this thread's can win
#pragma unroll
            for (int k = 0; k < 4 * J; ++k)
                if (mix32(((uint32_t)place(k) + 0x165667B1u) ^ key) >= hash) look |= 1u << k;
        }
        best = -INFINITY;
        best_k = -1;
        while (look != 0) {                                 // in the order of the places
            const int k = __ffs(look) - 1;
            look &= look - 1;
            const float4 four_of = four(k >> 2);
            const float x = (k & 3) == 0 ? four_of.x : (k & 3) == 1 ? four_of.y : (k & 3) == 2 ? four_of.z : four_of.w;
            // the bound of this logit itself, which few pass: two logarithms are paid by the whole warp
            if ((float)(8388608u - (mix32(((uint32_t)place(k) + 0x165667B1u) ^ key) >> 9)) > bound(x)) continue;
            const float y = score(x, k);
            if (y > best) { best = y; best_k = k; }
        }
        __syncthreads();                                    // s_val is written again below
    }
    int best_i = best_k < 0 ? 0x7fffffff : place(best_k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, best, o);
        const int oi = __shfl_xor_sync(0xffffffffu, best_i, o);
        if (better(ov, oi, best, best_i)) { best = ov; best_i = oi; }
    }
    if (lane == 0) { s_val[warp] = best; s_idx[warp] = best_i; }
    __syncthreads();
    // rows from the end of the scratch: what sample_kernel left at its beginning is not met
    int* mine = scratch_end - (size_t)(m + 1) * (2 * slices + 1);
    merge_slices(out, mine, mine + 2 * slices, m, slices, best, best_i, s_val, s_idx, &s_last);
}

__global__ void note_tokens_kernel(int* __restrict__ history, int rows, int width, const int* __restrict__ ids,
                                   const int* __restrict__ token_rows, const int* __restrict__ positions, int N,
                                   const int* __restrict__ feedback, int samples) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    const int n = blockIdx.x * blockDim.x + threadIdx.x;
    if (n >= N) return;
    const int r = token_rows[n], p = positions[n];
    int id = ids[n];
    if (id < 0 && -1 - id < samples) id = feedback[-1 - id];
    if (r >= 0 && r < rows && p >= 0 && p < width) history[(size_t)r * width + p] = id;
}

}  // namespace

// How many slices a row of V logits is cut into (so callers can size `scratch`).
extern "C" int sb_sample_slices(int V) {
    int c = (V + 8191) / 8192;
    return c < 1 ? 1 : (c > 32 ? 32 : c);
}

// The same for sb_sample_adjusted.
extern "C" int sb_sample_adjusted_slices(int V) {
    int c = (V + SLICE - 1) / SLICE;
    return c < 1 ? 1 : c;
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
    SB_REQUIRE(V <= 32 * SLICE, "sample_adjusted: a vocabulary of %d (at most %d)", V, 32 * SLICE);
    SB_REQUIRE(M <= 65535 * 32, "sample_adjusted: too many rows");
    const int slices = sb_sample_adjusted_slices(V);
    SB_REQUIRE(scratch != nullptr && scratch_ints >= (long long)M * (2 * sb_sample_slices(V) + 1 + 2 * slices + 1),
               "sample_adjusted: scratch has %lld entries, %lld are needed", scratch_ints,
               (long long)M * (2 * sb_sample_slices(V) + 1 + 2 * slices + 1));
    SB_REQUIRE(penalties == nullptr || (history != nullptr && history_width > 0 && history_rows != nullptr && prompt_lens != nullptr &&
                                      lengths != nullptr),
               "sample_adjusted: penalties need the rows' tokens, their lengths and the three numbers of each row");
    SB_REQUIRE(bias_starts == nullptr || (bias_ids != nullptr && bias_values != nullptr), "sample_adjusted: biases need ids and values");
    SB_REQUIRE(mask == nullptr || (mask_rows != nullptr && mask_words == (V + 31) / 32), "sample_adjusted: masks of %d words for %d tokens", mask_words, V);
    if (M == 0) return 0;
    const int per = ((V + slices - 1) / slices + 3) & ~3;
    const Adjust a{history, history_rows, prompt_lens, lengths, penalties, bias_starts, bias_ids, bias_values, (const uint32_t*)mask,
                   mask_rows, adjusted, history_width, mask_words};
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(sample_adjusted_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * SLICE * 4);
        if (e != cudaSuccess) { sb_set_error("sample_adjusted: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    const int smem = per * 4 * (1 + (penalties != nullptr || bias_starts != nullptr));
    sb::launch(sample_adjusted_kernel, dim3(M, slices), dim3(512), smem, stream, out, logits, temperature, seeds, counters, V, per,
               scratch + scratch_ints, a);
    SB_LAUNCH_CHECK();
}

// history [rows, width]: token n to place positions[n] of row token_rows[n]; an id -1 - j stands for feedback[j] (null: for nothing).
extern "C" int sb_note_tokens(int* history, int rows, int width, const int* ids, const int* token_rows, const int* positions, int N,
                              const int* feedback, int samples, cudaStream_t stream) {
    SB_REQUIRE(N >= 0 && rows > 0 && width > 0 && samples >= 0, "note_tokens: bad sizes (%d tokens, history of %d x %d)", N, rows, width);
    if (N == 0) return 0;
    sb::launch(note_tokens_kernel, dim3((N + 255) / 256), dim3(256), 0, stream, history, rows, width, ids, token_rows, positions, N,
               feedback, feedback != nullptr ? samples : 0);
    SB_LAUNCH_CHECK();
}
