// attention_shared.cu's operator on the tensor cores (bfloat16, mma.sync m16n8k16, float32 accumulation).
//
// What bounds it: the bytes of the cached keys and values, the shared ones once for up to 16 query rows of a family.  A key
// tile of 64 meets its rows as COLUMNS (warp_tile_decode: S^T = K Q^T, O^T += V^T P^T): a token's own keys its G query heads,
// a family's shared keys 16 of its tokens x G rows at a time, so both kinds of work are the same walk.
//
// An item is one set of rows with the keys that all of them meet: first the families' units of 16 rows, then the tokens.
// The 64-key tiles of all items are laid end to end (per KV head) and dealt to the GPU's blocks in equal shares, as in
// attention_balanced.cu; the cut is made on the device, so a recorded graph follows the lists.  Every item leaves partial
// results (max, sum, O): one if it lies in one share, one per share otherwise.  A second kernel joins a token's own
// and its unit's partial results in key order: no atomics, the same bits every time.
#include <math.h>

#include "attention_mma.cuh"
#include "attention_shared.h"

namespace {

constexpr int NW = 4;                    // warps of a block; a tile holds 16 keys for each
constexpr int STAGES = 3;
constexpr int AHEAD = 7;                 // tiles that page numbers are read ahead (their copies go out STAGES - 1 ahead)
constexpr int PAGE_SLOTS = 8;            // tiles whose page numbers are held: more than AHEAD, a power of two
constexpr int TILE_PAGES = 4;            // pages of 16 keys and more
constexpr int RQ = 16;                   // rows of an item: two column blocks
constexpr int SMEM_MOST = 220 * 1024, TWO_AN_SM = 112 * 1024;      // dynamic shared memory of a block
constexpr int MAX_MEMBERS = 512;         // (their lists live in shared memory)

// Units of 16 rows that the families of M members can have.
__host__ __device__ inline int most_units(int M, int R, int G) { return M * G / RQ + R; }

struct StreamArgs {
    float *whole_o, *whole_ml;           // [Hkv][items][16][D] and [Hkv][items][16][2]
    float *piece_o, *piece_ml;           // [Hkv][W][2][16][D] and [Hkv][W][2][16][2]
    int* items;                          // for the joining kernel: tiles, units, [items + 1] tiles before each, [M] places
    const bf16 *q, *k_pool, *v_pool;
    const int *block_table, *token_rows, *positions, *members, *group_starts, *shared_lens;
    int table_width, M, R, Hq, Hkv, BS, window, W;
    float scale_log2;
};

__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 && pos + 1 > window ? pos + 1 - window : 0; }

// The lists of a call in shared memory.  Item i < U is a unit, item U + x is member x.
struct Lists {
    int *token, *pos, *row, *own_lo;     // [M]: a member's token, position, cache row, and where its own keys begin
    int *starts, *uoff;                  // [R + 1]: members and units before each family
    int *unit, *unit_lo, *unit_hi;       // [units]: first flat row x 32 + rows; keys
    int* pre;                            // [items + 1]: tiles before each item
    int U, G, window;
    __device__ __forceinline__ int row0(int i) const { return i < U ? unit[i] >> 5 : (i - U) * G; }
    __device__ __forceinline__ int rows(int i) const { return i < U ? unit[i] & 31 : G; }
    __device__ __forceinline__ int lo(int i) const { return i < U ? unit_lo[i] : own_lo[i - U]; }
    __device__ __forceinline__ int hi(int i) const { return i < U ? unit_hi[i] : pos[i - U] + 1; }
    __device__ __forceinline__ int tiles(int i) const { return hi(i) > lo(i) ? (hi(i) + KT - 1) / KT - lo(i) / KT : 0; }
};

__host__ __device__ inline int list_ints(int M, int R, int units) { return 4 * M + 2 * (R + 1) + 3 * units + units + M + 1; }

struct Cursor {
    int i, begin, end, lo, hi, first;    // first: the tile index inside the row of flat tile 0
    const int* table;
    __device__ __forceinline__ void seek(int x, const Lists& it, const StreamArgs& a) {
        while (x >= it.pre[i + 1]) ++i;
        begin = it.pre[i];
        end = it.pre[i + 1];
        lo = it.lo(i);
        hi = it.hi(i);
        first = lo / KT - begin;
        table = a.block_table + (size_t)it.row[it.row0(i) / it.G] * a.table_width;
    }
    __device__ __forceinline__ int tile_start(int x) const { return (first + x) * KT; }
};

// Running sum over `n` values in shared memory, v[0] = 0 .. v[n]: v[i + 1] holds the i-th value when it is called.
__device__ __forceinline__ void running_sum(int* v, int n, int* scan) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int total = 0;
    for (int base = 0; base < n; base += 32 * NW) {
        const int i = base + tid;
        int t = i < n ? v[i + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += up;
        }
        if (lane == 31) scan[warp] = t;
        __syncthreads();
        int before = total;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += scan[w];
            total += scan[w];
        }
        if (i < n) v[i + 1] = before + t;
        __syncthreads();
    }
    if (tid == 0) v[0] = 0;
    __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(32 * NW, 2) shared_stream_kernel(const StreamArgs a) {
    sb::pdl_launch_dependents();
    // Before pdl_wait(): the lists, positions, block table (host copies) and keys and values below a row's newest position
    // (earlier steps).
    constexpr int NTHR = 32 * NW;
    constexpr int STAGE = 2 * KT * D;                       // elements of a stage: keys, then values
    extern __shared__ __align__(128) uint8_t smem[];
    bf16* ring = reinterpret_cast<bf16*>(smem);
    bf16* qring = ring + STAGES * STAGE;                    // the rows of the item that begins with the stage's tile
    int* pages = reinterpret_cast<int*>(qring + STAGES * RQ * D);        // [PAGE_SLOTS][TILE_PAGES] physical pages of a tile
    const int G = a.Hq / a.Hkv, units = most_units(a.M, a.R, G), most = units + a.M;
    Lists it;
    it.G = G;
    it.window = a.window;
    it.token = pages + PAGE_SLOTS * TILE_PAGES;
    it.pos = it.token + a.M;
    it.row = it.pos + a.M;
    it.own_lo = it.row + a.M;
    it.starts = it.own_lo + a.M;
    it.uoff = it.starts + a.R + 1;
    it.unit = it.uoff + a.R + 1;
    it.unit_lo = it.unit + units;
    it.unit_hi = it.unit_lo + units;
    it.pre = it.unit_hi + units;
    __shared__ float w_m[NW][16], w_l[NW][16];
    __shared__ int s_scan[NW], s_item0;

    const int bs_log2 = 31 - __clz(a.BS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kh = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;

    // ---- the lists, then the items and their tiles
    for (int i = tid; i < a.R; i += NTHR) {
        const int s0 = a.group_starts[i], n = a.group_starts[i + 1] - s0;
        it.starts[i] = s0;
        it.uoff[i + 1] = a.shared_lens[i] > 0 ? (n * G + RQ - 1) / RQ : 0;
    }
    if (tid == 0) it.starts[a.R] = a.group_starts[a.R];
    for (int i = tid; i < a.M; i += NTHR) {
        const int n = a.members[i];
        it.token[i] = n;
        it.pos[i] = a.positions[n];
        it.row[i] = a.token_rows[n];
    }
    __syncthreads();
    running_sum(it.uoff, a.R, s_scan);
    const int U = it.U = it.uoff[a.R], served = min(a.M, it.starts[a.R]), I = U + served;
    auto family_of = [&](const int* begin, int x) {         // the last one that begins at x or before
        int r = 0, top = a.R - 1;
        while (r < top) {
            const int mid = (r + top + 1) / 2;
            if (begin[mid] <= x) r = mid;
            else top = mid - 1;
        }
        return r;
    };
    for (int i = tid; i < I; i += NTHR) {
        if (i < U) {
            const int r = family_of(it.uoff, i), u = i - it.uoff[r], rows = (it.starts[r + 1] - it.starts[r]) * G;
            const int row0 = it.starts[r] * G + u * RQ, nr = min(RQ, rows - u * RQ);
            int lo = 0x7fffffff, last = -1;
            for (int x = row0 / G; x <= (row0 + nr - 1) / G; ++x) {
                lo = min(lo, first_seen(it.pos[x], a.window));
                last = max(last, it.pos[x]);
            }
            it.unit[i] = row0 * 32 + nr;
            it.unit_lo[i] = lo;
            it.unit_hi[i] = min(a.shared_lens[r], last + 1);
        } else {
            const int x = i - U;
            it.own_lo[x] = max(first_seen(it.pos[x], a.window), a.shared_lens[family_of(it.starts, x)]);
        }
        it.pre[i + 1] = it.tiles(i);
    }
    __syncthreads();
    running_sum(it.pre, I, s_scan);
    const int T = it.pre[I];
    const int W = max(1, min(a.W, T));
    if (blockIdx.x == 0) {
        // the previous call's joining kernel may still read this
        sb::pdl_wait();
        int* pre = a.items + 2;
        int* place = pre + most + 1;
        if (tid == 0) { a.items[0] = T; a.items[1] = U; }
        for (int i = tid; i <= I; i += NTHR) pre[i] = it.pre[i];
        for (int i = tid; i < a.M; i += NTHR) {             // the flat row of a member's first head among the units' rows
            int p = -2;
            if (i < served) {
                const int r = family_of(it.starts, i);
                p = it.uoff[r + 1] > it.uoff[r] ? it.uoff[r] * RQ + (i - it.starts[r]) * G : -1;
            }
            place[i] = p;
        }
    }
    if (slot >= W || T == 0) {
        sb::pdl_wait();
        return;
    }
    const int x0 = (int)((long long)slot * T / W), x1 = (int)((long long)(slot + 1) * T / W);
    for (int i = tid; i < I; i += NTHR)
        if (it.pre[i] <= x0 && x0 < it.pre[i + 1]) s_item0 = i;
    __syncthreads();

    const int n_pages = max(1, KT >> bs_log2);              // logical pages a tile touches
    // Bring the physical page of entry e of tile x to its slot (0 where the item does not reach: such keys are never
    // read, see load_kv_tile).  Asynchronous: part of the commit group that is open.
    auto fetch_page = [&](const Cursor& c, int x, int e) {
        const int logical = (c.tile_start(x) >> bs_log2) + e;
        const bool valid = logical <= ((c.hi - 1) >> bs_log2);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                     ::"r"(smem_u32(pages + ((x - x0) % PAGE_SLOTS) * TILE_PAGES + e)),
                       "l"(c.table + (valid ? logical : 0)), "r"(valid ? 4 : 0)
                     : "memory");
    };
    for (int i = tid; i < AHEAD * n_pages; i += NTHR) {
        const int x = x0 + i / n_pages;
        if (x < x1) {
            Cursor c;
            c.i = s_item0;
            c.seek(x, it, a);
            fetch_page(c, x, i % n_pages);
        }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    // flat row f of the members' rows: token f / G of the members, head kh G + f % G
    auto load_query = [&](const Cursor& c, int stage) {
        constexpr int CH = D / 8;
        bf16* qs = qring + stage * RQ * D;
        const int row0 = it.row0(c.i), nr = it.rows(c.i);
        for (int idx = tid; idx < RQ * CH; idx += NTHR) {
            const int row = idx / CH, ch = idx - row * CH;
            const bool valid = row < nr;
            const int f = row0 + (valid ? row : 0);
            cp_async16(smem_u32(qs + tile_off<D>(row, ch)), a.q + ((size_t)it.token[f / G] * a.Hq + kh * G + f % G) * D + ch * 8,
                       valid ? 16 : 0);
        }
    };

    // ---- the first tiles: those of shared keys and those below their token's newest key before the wait, the others after it
    Cursor cl;                                              // of the tile whose copies go out
    cl.i = s_item0;
    cl.seek(x0, it, a);
    const Cursor c0 = cl;
#pragma unroll
    for (int late = 0; late < 2; ++late) {
        if (late) sb::pdl_wait();
        cl = c0;
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            const int x = x0 + s;
            if (x >= x1) break;
            if (x >= cl.end) cl.seek(x, it, a);
            const int ts = cl.tile_start(x);
            if ((ts + KT >= cl.hi) == (late != 0))
                load_kv_tile<D, KT, NTHR>(ring + s * STAGE, ring + s * STAGE + KT * D, a.k_pool, a.v_pool, pages + s * TILE_PAGES,
                                          ts >> bs_log2, bs_log2, a.Hkv, kh, ts, cl.lo, cl.hi);
            if (late && (s == 0 || x == cl.begin)) load_query(cl, s);
        }
    }
    cp_async_commit();
#pragma unroll
    for (int s = 1; s < STAGES - 1; ++s) cp_async_commit();

    const WholeTileCopy<D, KT, NTHR> copy(ring, ring + KT * D, STAGE, a.k_pool, a.v_pool, bs_log2, a.Hkv, kh);
    ColState<D, 2> st;
    st.init();
    uint32_t qf[D / 16][4];
    int cpos[4], clo[4];                                    // the keys that this thread's columns see
    Cursor cc = c0, ct = c0;                                // of the tile that is computed, and of the page read-ahead
    int stage = STAGES - 1;                                 // of tile x: (x - x0) % STAGES
    for (int x = x0; x < x1; ++x) {
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        cp_async_wait<STAGES - 2>();
        __syncthreads();                                    // tile x is there; everybody is done with tile x - 1
        const int xt = x + AHEAD, xl = x + STAGES - 1;
        if (xl < x1 && xl >= cl.end) cl.seek(xl, it, a);
        if (xt < x1) {
            if (xt >= ct.end) ct.seek(xt, it, a);
            if (tid < n_pages) fetch_page(ct, xt, tid);
        }
        if (x >= cc.end) cc.seek(x, it, a);
        const int nr = it.rows(cc.i);
        if (x == x0 || x == cc.begin) {
            const bf16* qs = qring + stage * RQ * D;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
                ldmatrix_x4(qf[kk], smem_u32(qs + tile_off<D>(lane & 15, kk * 2 + (lane >> 4))));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int col = 8 * (c >> 1) + 2 * (lane & 3) + (c & 1);
                const int pos = col < nr ? it.pos[(it.row0(cc.i) + col) / G] : -1;
                cpos[c] = min(pos, cc.hi - 1);
                clo[c] = max(first_seen(pos, a.window), cc.lo);
            }
        }
        // the copies of tile xl: in doses between the phases of tile x, or (a tile at an item's edge) at once
        const int stage_l = stage == 0 ? STAGES - 1 : stage - 1;
        const int* pg_l = pages + ((xl - x0) % PAGE_SLOTS) * TILE_PAGES;
        const int tl = cl.tile_start(xl);
        bool doses = false;
        if (xl < x1) {
            doses = tl >= cl.lo && tl + KT <= cl.hi;
            if (!doses) {
                bf16* ks = ring + stage_l * STAGE;
                load_kv_tile<D, KT, NTHR>(ks, ks + KT * D, a.k_pool, a.v_pool, pg_l, tl >> bs_log2, bs_log2, a.Hkv, kh, tl,
                                          cl.lo, cl.hi);
            }
            if (xl == cl.begin) load_query(cl, stage_l);
        }
        auto between = [&](int part) {
            if (doses) copy.dose(part, stage_l, pg_l - (tl >> bs_log2), tl);
        };
        // scores in units of log2, -inf where a column does not see a key
        auto seen = [&](float s, int kpos, int nb, int e) {
            const int c = 2 * nb + e;
            return kpos <= cpos[c] && kpos >= clo[c] ? s * a.scale_log2 : -INFINITY;
        };
        const int ts = cc.tile_start(x);
        const bf16* ks = ring + stage * STAGE;
        if (nr <= 8) warp_tile_decode<D, 1>(st, qf, ks, ks + KT * D, warp * 16, ts, 0, 0, 0, 1.0f, false, between, seen);
        else warp_tile_decode<D, 2>(st, qf, ks, ks + KT * D, warp * 16, ts, 0, 0, 0, 1.0f, false, between, seen);
        cp_async_commit();
        if (x + 1 != x1 && x + 1 != cc.end) continue;

        // ---- the item, or this share of it, ends: merge the warps through the stage that was just read
        __syncthreads();
        float* wo = reinterpret_cast<float*>(ring + stage * STAGE);        // [NW][16][D]: exactly a stage
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            if (nb == 1 && nr <= 8) break;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = 2 * nb + e;
                float l = st.l[c];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                const int row = 8 * nb + 2 * (lane & 3) + e;
                if (lane < 4) { w_m[warp][row] = st.m[c]; w_l[warp][row] = l; }
#pragma unroll
                for (int mb = 0; mb < D / 16; ++mb) {
                    float* dst = wo + ((size_t)(warp * 16 + row)) * D + mb * 16 + (lane >> 2);
                    dst[0] = st.o[mb][nb][e];
                    dst[8] = st.o[mb][nb][e + 2];
                }
            }
        }
        __syncthreads();
        st.init();
        const bool whole = cc.begin >= x0 && cc.end <= x1;  // the item lies in this share
        const size_t p = whole ? (size_t)kh * most + cc.i : ((size_t)kh * a.W + slot) * 2 + (cc.begin <= x0 ? 0 : 1);
        float* to_o = (whole ? a.whole_o : a.piece_o) + p * RQ * D;
        float* to_ml = (whole ? a.whole_ml : a.piece_ml) + p * RQ * 2;
        for (int idx = tid * 4; idx < nr * D; idx += NTHR * 4) {
            const int row = idx / D;
            float m = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w) m = w_l[w][row] != 0.f ? fmaxf(m, w_m[w][row]) : m;
#pragma unroll
            for (int w = 0; w < NW; ++w) {                  // a warp without a visible key has weight 0
                if (w_l[w][row] != 0.f) {
                    const float f = ex2_approx(w_m[w][row] - m);
                    const float4 v = *reinterpret_cast<const float4*>(wo + (size_t)w * 16 * D + idx);
                    l += f * w_l[w][row];
                    o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
                }
            }
            *reinterpret_cast<float4*>(to_o + idx) = o;
            if (idx == row * D) *reinterpret_cast<float2*>(to_ml + 2 * row) = make_float2(m, l);
        }
    }
    cp_async_wait<0>();
}

// grid (M, Hkv): the G rows of a token of one KV head from its unit's partial results, then its own, in key order.
template <int D>
__global__ void __launch_bounds__(128) shared_stream_join_kernel(bf16* __restrict__ out, const StreamArgs a) {
    sb::pdl_launch_dependents();
    sb::pdl_wait();
    const int i = blockIdx.x, kh = blockIdx.y, G = a.Hq / a.Hkv, most = most_units(a.M, a.R, G) + a.M;
    const int T = a.items[0], U = a.items[1], W = max(1, min(a.W, T));
    const int* pre = a.items + 2;
    const int place = pre[most + 1 + i];
    if (place == -2) return;
    const int n = a.members[i];
    for (int idx = threadIdx.x * 4; idx < G * D; idx += blockDim.x * 4) {
        const int g = idx / D, d = idx - g * D;
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](int item, int row) {
            const int begin = pre[item], end = pre[item + 1];
            if (end == begin) return;
            const int s0 = (int)(((long long)(begin + 1) * W + T - 1) / T) - 1, s1 = (int)(((long long)end * W + T - 1) / T);
            const bool whole = s1 == s0 + 1;
            constexpr int AT = 8;                           // partial results in flight
            for (int s = s0; s < s1; s += AT) {
                float2 ml[AT];
                float4 v[AT];
#pragma unroll
                for (int u = 0; u < AT; ++u) {
                    ml[u] = make_float2(-INFINITY, 0.f);
                    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (s + u < s1) {
                        const size_t p = whole ? (size_t)kh * most + item
                                               : ((size_t)kh * a.W + s + u) * 2 + (begin <= (int)((long long)(s + u) * T / W) ? 0 : 1);
                        ml[u] = __ldcg(reinterpret_cast<const float2*>((whole ? a.whole_ml : a.piece_ml) + (p * RQ + row) * 2));
                        v[u] = __ldcg(reinterpret_cast<const float4*>((whole ? a.whole_o : a.piece_o) + (p * RQ + row) * D + d));
                    }
                }
                float top = M;
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    if (ml[u].y != 0.f) top = fmaxf(top, ml[u].x);
                const float keep = L != 0.f ? exp2f(M - top) : 0.f;
                L *= keep;
                o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
                for (int u = 0; u < AT; ++u)
                    if (ml[u].y != 0.f) {
                        const float f = exp2f(ml[u].x - top);
                        L += f * ml[u].y;
                        o.x += f * v[u].x; o.y += f * v[u].y; o.z += f * v[u].z; o.w += f * v[u].w;
                    }
                M = top;
            }
        };
        if (place >= 0) add((place + g) / RQ, (place + g) % RQ);
        add(U + i, g);
        __nv_bfloat162* to = reinterpret_cast<__nv_bfloat162*>(out + ((size_t)n * a.Hq + kh * G) * D + idx);
        to[0] = __floats2bfloat162_rn(o.x / L, o.y / L);
        to[1] = __floats2bfloat162_rn(o.z / L, o.w / L);
    }
}

int stream_smem(int M, int R, int G, int D) {
    return (STAGES * 2 * KT * D + STAGES * RQ * D) * 2 + PAGE_SLOTS * TILE_PAGES * 4 + list_ints(M, R, most_units(M, R, G)) * 4;
}

// Shares a KV head's tiles are cut into: as many blocks as the GPU holds at once (two an SM, or one beside long lists).
int shares_of(int M, int R, int Hq, int Hkv, int D, int num_sms) {
    const int w = num_sms * (stream_smem(M, R, Hq / Hkv, D) <= TWO_AN_SM ? 2 : 1) / Hkv;
    return w < 1 ? 1 : w;
}

template <int D>
int launch_stream(void* out, StreamArgs a, cudaStream_t stream) {
    auto kernel = shared_stream_kernel<D>;
    const int G = a.Hq / a.Hkv, smem = stream_smem(a.M, a.R, G, D);
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST);
        if (e != cudaSuccess) { sb_set_error("attention_shared: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    sb::launch(kernel, dim3(a.W * a.Hkv), dim3(32 * NW), smem, stream, a);
    sb::launch(shared_stream_join_kernel<D>, dim3(a.M, a.Hkv), dim3(G * D >= 512 ? 128 : 64), 0, stream, (bf16*)out, a);
    return 0;
}

}  // namespace

namespace sb {

bool shared_stream_supports(int M, int R, int Hq, int Hkv, int D, int page_size) {
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > RQ || M <= 0 || M > MAX_MEMBERS || R <= 0) return false;
    if (!(D == 16 || D == 32 || D == 64 || D == 128)) return false;
    if (page_size < KT / TILE_PAGES || (page_size & (page_size - 1)) != 0) return false;
    return stream_smem(M, R, Hq / Hkv, D) <= SMEM_MOST;
}

void shared_stream_scratch(int M, int R, int Hq, int Hkv, int D, int num_sms, long long* floats, long long* ints) {
    const int items = most_units(M, R, Hq / Hkv) + M;
    // (as many shares as two blocks an SM make, whatever this call's lists leave room for: no less for more members)
    *floats = ((long long)Hkv * items + 2ll * (2 * num_sms > Hkv ? 2 * num_sms : Hkv)) * RQ * (D + 2);
    *ints = 2 + items + 1 + M;
}

int shared_stream(void* out, float* part, int* items, const void* q, const void* k_pool, const void* v_pool,
                  const SharedLists& l, int Hq, int Hkv, int D, int page_size, int window, float scale, int num_sms,
                  cudaStream_t stream) {
    StreamArgs a{};
    const int W = shares_of(l.M, l.R, Hq, Hkv, D, num_sms);
    const long long most = most_units(l.M, l.R, Hq / Hkv) + l.M;
    a.whole_o = part;
    a.whole_ml = a.whole_o + Hkv * most * RQ * D;
    a.piece_o = a.whole_ml + Hkv * most * RQ * 2;
    a.piece_ml = a.piece_o + 2ll * Hkv * W * RQ * D;
    a.items = items;
    a.q = (const bf16*)q; a.k_pool = (const bf16*)k_pool; a.v_pool = (const bf16*)v_pool;
    a.block_table = l.block_table; a.token_rows = l.token_rows; a.positions = l.positions;
    a.members = l.members; a.group_starts = l.group_starts; a.shared_lens = l.shared_lens;
    a.table_width = l.table_width; a.M = l.M; a.R = l.R; a.Hq = Hq; a.Hkv = Hkv; a.BS = page_size; a.window = window; a.W = W;
    a.scale_log2 = scale * LOG2E;
    switch (D) {
        case 16: return launch_stream<16>(out, a, stream);
        case 32: return launch_stream<32>(out, a, stream);
        case 64: return launch_stream<64>(out, a, stream);
        default: return launch_stream<128>(out, a, stream);
    }
}

}  // namespace sb
