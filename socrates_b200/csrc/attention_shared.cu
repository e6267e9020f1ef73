// Paged GQA attention of decode tokens whose rows share a prefix (answers of one prompt, requests behind one system
// prompt): the shared keys are read once for all tokens of a family, not once a token.
//
// With S the keys [0, shared) of a family and T_n the keys [shared, pos_n] of token n, softmax over S and T_n is joined
// from what each set gives alone,
//   m = max(m_S, m_T),  l = e^{m_S - m} l_S + e^{m_T - m} l_T,  o = (e^{m_S - m} o_S + e^{m_T - m} o_T) / l,
// so the family's query heads (tokens x G rows) meet S as the rows of one tile and every token meets its own T_n as G rows.
//
// This file's kernel runs on the CUDA cores in float32: calls in float32 (the 32-bit engine makes none, as its numbers do not
// depend on the batch), and in bfloat16 the shapes that the tensor-core kernels do not take.  A block serves 16 rows of one KV head (of a family: any 16 of its tokens x G rows; of one token: its
// G rows) and one part of their keys; parts are joined by a second kernel.
#include <math.h>

#include "attention_shared.h"
#include "common.cuh"

using namespace sb;

namespace {

constexpr int THREADS = 128;
constexpr int RT = 16;               // rows of a block: eight threads a row
constexpr int KT = 32;               // keys of a tile
constexpr int PER = THREADS / RT;    // threads of a row

struct Shared {
    const int *block_table, *token_rows, *positions, *members, *group_starts, *shared_lens;
    int table_width, M, R, Hq, Hkv, D, BS, window;
};

__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 && pos + 1 > window ? pos + 1 - window : 0; }

// grid: KV heads x (prefix units x parts, then own-key units x parts).  Partial results [member][head][NP + NS].
template <typename T>
__global__ void __launch_bounds__(THREADS)
shared_rows_kernel(float* __restrict__ part_o, float* __restrict__ part_ml, const T* __restrict__ q,
                   const T* __restrict__ k_pool, const T* __restrict__ v_pool, const Shared a, float scale, int NP, int NS,
                   int prefix_units, int own_units) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    extern __shared__ float smem[];
    const int D = a.D, pitch = D + 4, G = a.Hq / a.Hkv;
    float* qs = smem;                                        // [RT][D]
    float* ks = qs + RT * D;                                 // [KT][D + 4]
    float* vs = ks + KT * pitch;                             // [KT][D]
    float* ps = vs + KT * D;                                 // [RT][KT + 1]
    __shared__ int r_mem[RT], r_tok[RT], r_head[RT], r_pos[RT];

    const int tid = threadIdx.x;
    const int kh = blockIdx.x % a.Hkv;
    int u = blockIdx.x / a.Hkv;
    const bool own = u >= prefix_units * NP;
    if (own) u -= prefix_units * NP;
    const int parts = own ? NS : NP, part = u % parts;
    u /= parts;

    // ---- the unit's rows and keys
    int n_rows = 0, lo = 0, hi = 0;
    if (own) {
        const int per_tok = (G + RT - 1) / RT, i = u / per_tok, g0 = (u % per_tok) * RT;
        if (i >= a.group_starts[a.R]) return;
        int r = 0, top = a.R - 1;                            // the family whose members hold place i
        while (r < top) {
            const int mid = (r + top + 1) / 2;
            if (a.group_starts[mid] <= i) r = mid;
            else top = mid - 1;
        }
        const int n = a.members[i], pos = a.positions[n];
        n_rows = min(RT, G - g0);
        lo = max(first_seen(pos, a.window), a.shared_lens[r]);
        hi = pos + 1;
        if (tid < RT) { r_mem[tid] = i; r_tok[tid] = n; r_head[tid] = kh * G + g0 + tid; r_pos[tid] = tid < n_rows ? pos : -1; }
    } else {
        // the family that unit u belongs to: its thread finds it, THREADS families at a time
        __shared__ int s_warp[THREADS / 32], s_found[3];
        const int lane = tid & 31;
        bool found = false;
        for (int base = 0; base < a.R && !found; base += THREADS) {
            const int r = base + tid, start = r < a.R ? a.group_starts[r] : 0;
            const int rows = r < a.R ? (a.group_starts[r + 1] - start) * G : 0, units = (rows + RT - 1) / RT;
            int to = units;                                  // units up to this family's end, of this round's
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, to, o);
                if (lane >= o) to += up;
            }
            if (lane == 31) s_warp[tid >> 5] = to;
            __syncthreads();
            int total = 0;
            for (int w = 0; w < THREADS / 32; ++w) {
                if (w < tid >> 5) to += s_warp[w];
                total += s_warp[w];
            }
            if (u < to && u >= to - units) {
                s_found[0] = r;
                s_found[1] = rows;
                s_found[2] = u - (to - units);
            }
            found = u < total;
            __syncthreads();
            if (!found) u -= total;
        }
        if (!found) return;
        const int r = s_found[0], rows = s_found[1], start = a.group_starts[r];
        u = s_found[2];
        n_rows = min(RT, rows - u * RT);
        hi = a.shared_lens[r];
        if (tid < RT) {
            const int row = u * RT + min(tid, n_rows - 1), i = start + row / G, n = a.members[i];
            r_mem[tid] = i;
            r_tok[tid] = n;
            r_head[tid] = kh * G + row % G;
            r_pos[tid] = tid < n_rows ? a.positions[n] : -1;
        }
        __syncthreads();
        lo = hi;
        int last = -1;
        for (int i = 0; i < n_rows; ++i) {
            lo = min(lo, first_seen(r_pos[i], a.window));
            last = max(last, r_pos[i]);
        }
        hi = min(hi, last + 1);
    }
    __syncthreads();
    const int t0 = lo / KT, tiles = hi > lo ? (hi + KT - 1) / KT - t0 : 0;
    const int begin = (int)((long long)part * tiles / parts), end = (int)((long long)(part + 1) * tiles / parts);

    const int row = tid / PER, sub = tid % PER;
    const int pos = r_pos[row], qlo = max(first_seen(pos, a.window), lo);
    for (int i = tid; i < RT * D; i += THREADS) {
        const int x = i / D;
        qs[i] = x < n_rows ? to_float(q[((size_t)r_tok[x] * a.Hq + r_head[x]) * D + i % D]) * scale : 0.f;
    }
    // every row of a unit reads the prefix through the first one's table: they hold the same pages there
    const int* table = a.block_table + (size_t)a.token_rows[r_tok[0]] * a.table_width;
    float m = -INFINITY, l = 0.f, acc[32];                   // thread `sub` of a row: dims 4 sub .. + 3, + 32, ...
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
    constexpr int VEC = Vec16<T>::N;
    for (int t = begin; t < end; ++t) {
        const int k0 = (t0 + t) * KT;
        __syncthreads();
        for (int i = tid; i < KT * D / VEC; i += THREADS) {
            const int key = i / (D / VEC), c = (i % (D / VEC)) * VEC, kpos = k0 + key;
            Vec16<T> kv, vv;
            const bool in = kpos >= lo && kpos < hi;
            if (in) {
                const size_t at = (((size_t)table[kpos / a.BS] * a.Hkv + kh) * a.BS + kpos % a.BS) * D + c;
                kv.load(k_pool + at);
                vv.load(v_pool + at);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                ks[key * pitch + c + e] = in ? kv.get(e) : 0.f;
                vs[key * D + c + e] = in ? vv.get(e) : 0.f;
            }
        }
        __syncthreads();
        // ---- scores of keys sub, sub + 8, ... of the tile
        float s[KT / PER];
#pragma unroll
        for (int j = 0; j < KT / PER; ++j) s[j] = 0.f;
        for (int d = 0; d < D; d += 4) {
            const float4 x = *reinterpret_cast<const float4*>(qs + row * D + d);
#pragma unroll
            for (int j = 0; j < KT / PER; ++j) {
                const float4 y = *reinterpret_cast<const float4*>(ks + (sub + j * PER) * pitch + d);
                s[j] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[j]))));
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT / PER; ++j) {
            const int kpos = k0 + sub + j * PER;
            if (!(kpos <= pos && kpos >= qlo && kpos < hi)) s[j] = -INFINITY;
            top = fmaxf(top, s[j]);
        }
#pragma unroll
        for (int o = 1; o < PER; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float next = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.f : expf(m - next);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[i] *= alpha;
        m = next;
#pragma unroll
        for (int j = 0; j < KT / PER; ++j) {
            const float p = s[j] == -INFINITY ? 0.f : expf(s[j] - m);
            l += p;
            ps[row * (KT + 1) + sub + j * PER] = p;
        }
        __syncwarp();                                        // a row's eight threads are neighbours in a warp
        for (int key = 0; key < KT; ++key) {
            const float p = ps[row * (KT + 1) + key];
            if (p == 0.f) continue;                          // a masked key's value is not met, whatever it is
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = 4 * sub + 32 * i;
                if (d < D) {
                    const float4 y = *reinterpret_cast<const float4*>(vs + key * D + d);
                    acc[4 * i] = fmaf(p, y.x, acc[4 * i]);
                    acc[4 * i + 1] = fmaf(p, y.y, acc[4 * i + 1]);
                    acc[4 * i + 2] = fmaf(p, y.z, acc[4 * i + 2]);
                    acc[4 * i + 3] = fmaf(p, y.w, acc[4 * i + 3]);
                }
            }
        }
    }
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (row >= n_rows) return;
    const size_t p = ((size_t)r_mem[row] * a.Hq + r_head[row]) * (NP + NS) + (own ? NP : 0) + part;
    if (sub == 0) *reinterpret_cast<float2*>(part_ml + 2 * p) = make_float2(m, l);
    if (l != 0.f) {                                          // NaN goes on to the result
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = 4 * sub + 32 * i;
            if (d < D) *reinterpret_cast<float4*>(part_o + p * D + d) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
    }
}

// out[n, h] from the parts of token n = members[blockIdx.y], in their order; a part without a key is not read.
template <typename T>
__global__ void shared_join_kernel(T* __restrict__ out, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                   const int* __restrict__ members, const int* __restrict__ group_starts, int R, int Hq,
                                   int D, int parts) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    if ((int)blockIdx.y >= group_starts[R]) return;
    const int n = members[blockIdx.y], h = blockIdx.x;
    const size_t base = ((size_t)blockIdx.y * Hq + h) * parts;
    const float2* ml = reinterpret_cast<const float2*>(part_ml) + base;
    float M = -INFINITY;
    for (int p = 0; p < parts; ++p)
        if (ml[p].y != 0.f) M = fmaxf(M, ml[p].x);
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float L = 0.f, o = 0.f;
        for (int p = 0; p < parts; ++p) {
            const float2 v = ml[p];
            if (v.y != 0.f) {
                const float w = expf(v.x - M);
                L += w * v.y;
                o += w * part_o[(base + p) * D + d];
            }
        }
        out[((size_t)n * Hq + h) * D + d] = from_float<T>(o / L);
    }
}

template <typename T>
int launch_rows(void* out, float* part, const void* q, const void* k_pool, const void* v_pool, const Shared& a,
                float scale, int NP, int NS, cudaStream_t stream) {
    auto kernel = shared_rows_kernel<T>;
    const int smem = (RT * a.D + KT * (a.D + 4) + KT * a.D + RT * (KT + 1)) * 4;
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        const int most = (RT * 256 + KT * 260 + KT * 256 + RT * (KT + 1)) * 4;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) { sb_set_error("attention_shared: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    const int G = a.Hq / a.Hkv;
    const int prefix_units = a.M * G / RT + a.R, own_units = a.M * ((G + RT - 1) / RT);
    float* part_o = part;
    float* part_ml = part + (size_t)a.M * a.Hq * (NP + NS) * a.D;
    const long long blocks = (long long)a.Hkv * ((long long)prefix_units * NP + (long long)own_units * NS);
    SB_REQUIRE(blocks <= 0x7fffffffll, "attention_shared: %lld blocks are too many", blocks);
    sb::launch(kernel, dim3((unsigned)blocks), dim3(THREADS), smem, stream, part_o, part_ml, (const T*)q, (const T*)k_pool,
               (const T*)v_pool, a, scale, NP, NS, prefix_units, own_units);
    sb::launch(shared_join_kernel<T>, dim3(a.Hq, a.M), dim3(a.D < 128 ? 64 : 128), 0, stream, (T*)out, part_o, part_ml, a.members,
               a.group_starts, a.R, a.Hq, a.D, NP + NS);
    SB_LAUNCH_CHECK();
}

// Parts of the shared and of the own keys: enough blocks for two rounds of the GPU, at most 16 and 8.
void rows_parts(int M, int Hq, int Hkv, int num_sms, int* NP, int* NS) {
    const int G = Hq / Hkv;
    const int up = Hkv * ((M * G + RT - 1) / RT), us = Hkv * M * ((G + RT - 1) / RT);
    *NP = 4 * num_sms / up;
    *NP = *NP < 1 ? 1 : *NP > 16 ? 16 : *NP;
    *NS = 4 * num_sms / us;
    *NS = *NS < 1 ? 1 : *NS > 8 ? 8 : *NS;
}

}  // namespace

// Scratch of a call with up to M members in up to R families (more than M where some are empty), in entries: float32, and int32.
extern "C" int sb_attention_shared_scratch(int M, int R, int Hq, int Hkv, int D, int page_size, int dtype, long long* floats,
                                           long long* ints) {
    SB_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D > 0 && M > 0 && R > 0,
               "attention_shared: %d members in %d groups, %d query heads on %d KV heads of %d", M, R, Hq, Hkv, D);
    long long most = 0, whole = 1;
    for (int m = 1; m <= M; ++m) {                           // fewer members are cut into more parts
        int NP, NS;
        rows_parts(m, Hq, Hkv, sm_count(), &NP, &NS);
        const long long need = (long long)m * Hq * (NP + NS) * (D + 2);
        most = need > most ? need : most;
    }
    if (dtype == SB_BF16) {
        for (int m = 1; m <= M && sb::shared_stream_supports(m, 1, Hq, Hkv, D, page_size); ++m) {
            long long f, i;
            sb::shared_stream_scratch(m, R, Hq, Hkv, D, page_size, sm_count(), &f, &i);
            most = f > most ? f : most;
            whole = i > whole ? i : whole;
        }
    }
    *floats = most;
    *ints = whole;
    return 0;
}

// 1 if a family of n tokens of G query heads a KV head with so many shared keys is a large one, else 0.
extern "C" int sb_attention_shared_large(int n, int G, int shared) { return n > 0 && G > 0 && sb::tc_family(n, G, shared); }

// 1 if the tensor-core kernels serve bfloat16 calls of so many members, 0 if the one on the CUDA cores does (or none).
extern "C" int sb_attention_shared_supports(int M, int Hq, int Hkv, int D, int page_size) {
    return sb::shared_stream_supports(M, M, Hq, Hkv, D, page_size);
}

// Whether a bfloat16 call launches the kernel for large families too (three kernels instead of two).
extern "C" int sb_attention_shared_kernels(int M, int R, int Hq, int Hkv, int D, int page_size, int num_pages, int with_status) {
    return Hkv > 0 && with_status && sb::shared_stream_supports(M, R, Hq, Hkv, D, page_size) &&
                   sb::shared_tc_supports(M, R, Hq, Hkv, D, page_size, num_pages)
               ? 3 : 2;
}

extern "C" int sb_attention_shared(void* out, float* part, long long part_floats, int* lists, long long lists_ints, const void* q,
                                   const void* k_pool, const void* v_pool, int num_pages, const int* block_table,
                                   int table_width, const int* token_rows, const int* positions, const int* members, int M,
                                   const int* group_starts, const int* shared_lens, int R, int N, int Hq, int Hkv, int D,
                                   int page_size, int window, float scale, int dtype, int* status,
                                   cudaStream_t stream) {
    SB_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "attention_shared: %d query heads on %d KV heads", Hq, Hkv);
    SB_REQUIRE(D % 16 == 0 && D >= 16 && D <= 256, "attention_shared: head_dim %d", D);
    SB_REQUIRE(page_size > 0 && table_width > 0 && window >= 0, "attention_shared: pages of %d, table of %d, window of %d",
               page_size, table_width, window);
    SB_REQUIRE(N > 0 && M > 0 && M <= N && R > 0 && R <= N && M <= 65535, "attention_shared: %d members of %d tokens in %d groups", M, N, R);
    SB_REQUIRE(dtype == SB_F32 || dtype == SB_BF16, "attention_shared: element type %d", dtype);
    SB_REQUIRE(scale > 0.f && scale < INFINITY, "attention_shared: a scale of %g", (double)scale);
    const uintptr_t all = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) |
                          reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(part) | reinterpret_cast<uintptr_t>(lists);
    SB_REQUIRE(all % 16 == 0, "attention_shared: out, q, the pools and the scratch must start on 16 bytes");
    if (dtype == SB_BF16 && sb::shared_stream_supports(M, R, Hq, Hkv, D, page_size)) {
        long long floats, ints;
        sb::shared_stream_scratch(M, R, Hq, Hkv, D, page_size, sm_count(), &floats, &ints);
        SB_REQUIRE(part != nullptr && part_floats >= floats && lists != nullptr && lists_ints >= ints, "attention_shared: scratch is too small");
        const sb::SharedLists l{block_table, token_rows, positions, members, group_starts, shared_lens, table_width, M, R};
        const int rc = sb::shared_stream(out, part, lists, q, k_pool, v_pool, l, Hq, Hkv, D, page_size, num_pages,
                                         window, scale, sm_count(), status, stream);
        if (rc != 0) return rc;
        SB_LAUNCH_CHECK();
    }
    const Shared a{block_table, token_rows, positions, members, group_starts, shared_lens, table_width, M, R, Hq, Hkv, D,
                   page_size, window};
    int NP, NS;
    rows_parts(M, Hq, Hkv, sm_count(), &NP, &NS);
    SB_REQUIRE(part != nullptr && part_floats >= (long long)M * Hq * (NP + NS) * (D + 2), "attention_shared: scratch is too small");
    return dtype == SB_F32 ? launch_rows<float>(out, part, q, k_pool, v_pool, a, scale, NP, NS, stream)
                           : launch_rows<__nv_bfloat16>(out, part, q, k_pool, v_pool, a, scale, NP, NS, stream);
}
