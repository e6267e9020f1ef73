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
//
// (Chunks of tiles that blocks claim, beside one block an SM of the kernel for large families instead of behind two: 106 us for
// 64 rows behind 6,144 keys with up to 2,048 of their own, 91 so.  What the claims add to the loop over tiles costs it a tenth,
// and a block of either kernel is slower beside one of the other.)
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
    int* items;                          // for the joining kernel: eight entries a member (see sb::TcPart), -2 first: not served
    const bf16 *q, *k_pool, *v_pool;
    const int *block_table, *token_rows, *positions, *members, *group_starts, *shared_lens;
    int table_width, M, R, Hq, Hkv, BS, window, W, num_sms;
    float scale_log2;
    sb::TcPart tc;                       // items: the large families' shared keys are the kernel's before this one, else null
};

__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 && pos + 1 > window ? pos + 1 - window : 0; }

// The lists of a call in shared memory.  Item i < U is a unit, item U + x is member x.
struct Lists {
    int *token, *pos, *row, *own_lo;     // [M]: a member's token, position, cache row, and where its own keys begin
    int *starts, *uoff;                  // [R + 1]: members and units before each family
    int *unit, *unit_lo, *unit_hi;       // [units]: first flat row x 32 + rows; keys
    int* pre;                            // [items + 1]: tiles before each item
    int U, I, G, window;
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
    // (item by item: the loop over tiles holds this code three times)
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

// `large`: the large families' shared keys are the kernel's before this one.
template <int D, bool large>
__global__ void __launch_bounds__(32 * NW, 2) shared_stream_kernel(const StreamArgs a) {
    sb::pdl_launch_dependents();
    // Before pdl_wait(): the lists, positions, block table (host copies) and keys and values below a row's newest position
    // (earlier steps).  Behind the kernel for large families, which lets this one in when its own wait has returned (if there is a
    // large family), queries and newest keys are complete too, and the partial results of an earlier call are read: this
    // one then waits for it only at its end, for the joining kernel's sake.
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
    __shared__ int s_scan[NW], s_large;

    const int bs_log2 = 31 - __clz(a.BS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kh = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;

    // ---- the lists, then the items and their tiles
    if constexpr (large) {
        if (tid == 0) s_large = 0;
        __syncthreads();
    }
    for (int i = tid; i < a.R; i += NTHR) {
        const int s0 = a.group_starts[i], n = a.group_starts[i + 1] - s0;
        it.starts[i] = s0;
        const int shared = a.shared_lens[i];
        const bool elsewhere = large && sb::tc_family(n, G, shared);
        if (elsewhere) s_large = 1;
        it.uoff[i + 1] = shared > 0 && !elsewhere ? (n * G + RQ - 1) / RQ : 0;
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
    const bool behind = large && s_large != 0;
    const int U = it.U = it.uoff[a.R], served = min(a.M, it.starts[a.R]), I = it.I = U + served;
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
    const sb::Cut cut{T, max(1, min(a.W, T))};
    if (blockIdx.x == 0) {
        if (!behind) sb::pdl_wait();                        // the previous call's joining kernel may still read this
        int4* where = reinterpret_cast<int4*>(a.items);
        for (int i = tid; i < a.M; i += NTHR) {
            int4 w = make_int4(i < served ? -1 : -2, 0, 0, 0), v = make_int4(0, 0, 0, it.token[i]);
            if (i < served) {
                const int r = family_of(it.starts, i);
                if (it.uoff[r + 1] > it.uoff[r]) {
                    w.x = it.uoff[r] * RQ + (i - it.starts[r]) * G;
                    const int u = w.x / RQ;
                    const int2 first = cut.parts(it.pre[u], it.pre[u + 1]), second = cut.parts(it.pre[u + 1], it.pre[u + 2]);
                    w.y = first.x; w.z = first.y; w.w = second.x; v.x = second.y;
                }
                const int2 own = cut.parts(it.pre[U + i], it.pre[U + i + 1]);
                v.y = own.x; v.z = own.y;
            }
            where[2 * i] = w;
            where[2 * i + 1] = v;
        }
    }
    if (slot >= cut.pieces || T == 0) {
        sb::pdl_wait();
        return;
    }
    const int x0 = cut.begin(slot), x1 = cut.begin(slot + 1);
    const int n_pages = max(1, KT >> bs_log2);              // logical pages a tile touches
    // Bring the physical page of entry e of tile x, the share's at-th, to its slot (0 where the item does not reach: such keys are never
    // read, see load_kv_tile).  Asynchronous: part of the commit group that is open.
    auto fetch_page = [&](const Cursor& c, int x, int at, int e) {
        const int logical = (c.tile_start(x) >> bs_log2) + e;
        const bool valid = logical <= ((c.hi - 1) >> bs_log2);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                     ::"r"(smem_u32(pages + (at % PAGE_SLOTS) * TILE_PAGES + e)),
                       "l"(c.table + (valid ? logical : 0)), "r"(valid ? 4 : 0)
                     : "memory");
    };
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

    const WholeTileCopy<D, KT, NTHR> copy(ring, ring + KT * D, STAGE, a.k_pool, a.v_pool, bs_log2, a.Hkv, kh);
    ColState<D, 2> st;
    st.init();
    uint32_t qf[D / 16][4];
    int cpos[4], clo[4];                                    // the keys that this thread's columns see
    Cursor c0;                                              // of the share's first tile
    c0.i = 0;
    for (int top = I - 1; c0.i < top;) {
        const int mid = (c0.i + top) / 2;
        if (x0 >= it.pre[mid + 1]) c0.i = mid + 1;
        else top = mid;
    }
    c0.seek(x0, it, a);
    for (int i = tid; i < AHEAD * n_pages; i += NTHR) {
        const int x = x0 + i / n_pages;
        if (x < x1) {
            Cursor c = c0;
            if (x >= c.end) c.seek(x, it, a);
            fetch_page(c, x, i / n_pages, i % n_pages);
        }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    // ---- the first tiles: those of shared keys and those below their token's newest key before the wait, the others after it
    Cursor cl = c0;                                         // of the tile whose copies go out
#pragma unroll
    for (int late = 0; late < 2; ++late) {
        if (late && !behind) sb::pdl_wait();
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

    Cursor cc = c0, ct = c0;                                // of the tile that is computed, and of the page read-ahead
    int stage = STAGES - 1;                                 // of tile x: (x - x0) % STAGES
    for (int x = x0; x < x1; ++x) {
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        cp_async_wait<STAGES - 2>();
        __syncthreads();                                    // tile x is there; everybody is done with the tile before
        const int xt = x + AHEAD, xl = x + STAGES - 1;
        if (xl < x1 && xl >= cl.end) cl.seek(xl, it, a);
        if (xt < x1) {
            if (xt >= ct.end) ct.seek(xt, it, a);
            if (tid < n_pages) fetch_page(ct, xt, xt - x0, tid);
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
        const size_t p = whole ? (size_t)kh * most + (cc.i < U ? cc.i : units + cc.i - U) : ((size_t)kh * a.W + slot) * 2 + (cc.begin <= x0 ? 0 : 1);
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
    if (behind) sb::pdl_wait();
}

// grid (M, Hkv): the G rows of a token of one KV head from its unit's partial results, then its own, in key order.  The
// threads of a block are two to JOIN groups, each of which takes every so many-th partial result, so that many loads of a token
// are in flight; the groups' sums are added in the groups' order.
constexpr int JOIN = 4;

template <int D>
__global__ void __launch_bounds__(128 * JOIN, 2)
shared_stream_join_kernel(bf16* __restrict__ out, const StreamArgs a, int groups) {
    sb::pdl_launch_dependents();
    __shared__ float4 s_o[JOIN - 1][128];
    __shared__ float2 s_ml[JOIN - 1][128];
    sb::pdl_wait();
    const int i = blockIdx.x, kh = blockIdx.y, G = a.Hq / a.Hkv;
    const int4 w = reinterpret_cast<const int4*>(a.items)[2 * i], v = reinterpret_cast<const int4*>(a.items)[2 * i + 1];
    if (w.x == -2) return;
    int4 tw = make_int4(-1, 0, 0, 0);
    int tv = 0;
    if (a.tc.items != nullptr) {
        tw = reinterpret_cast<const int4*>(a.tc.items)[2 * i];
        tv = a.tc.items[8 * i + 4];
    }
    const int threads = blockDim.x / groups, group = threadIdx.x / threads, t = threadIdx.x - group * threads;
    for (int base = 0; base < G * D; base += threads * 4) {
        const int idx = base + t * 4;
        const bool mine = idx < G * D;
        const int g = idx / D, d = idx - g * D;
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto take = [&](const float2 ml, const float4 x) {
            if (ml.y == 0.f) return;
            const float top = fmaxf(M, ml.x), keep = L != 0.f ? exp2f(M - top) : 0.f, f = exp2f(ml.x - top);
            M = top;
            L = L * keep + f * ml.y;
            o.x = o.x * keep + f * x.x; o.y = o.y * keep + f * x.y; o.z = o.z * keep + f * x.z; o.w = o.w * keep + f * x.w;
        };
        if (mine) {
            // The partial results of this row's unit, then those of the token's own keys.  Of an item that lies in one share
            // there is one in whole_*, of another one in piece_* for each share (its first share's second one, if bit 31 says so).
            const int units = most_units(a.M, a.R, G), items = units + a.M;
            const bool tc = tw.x >= 0;
            const int rows = tc ? sb::TC_ROWS : RQ, place = tc ? tw.x : w.x, row = place + g, unit = row / rows;
            const bool next = place >= 0 && unit > place / rows;
            const int from = place < 0 ? 0 : tc ? (next ? tw.w : tw.y) : next ? w.w : w.y;
            const int end = place < 0 ? 0 : tc ? (next ? tv : tw.z) : next ? v.x : w.z;
            const int n_unit = end - (from & 0x7fffffff), n_own = v.z - (v.y & 0x7fffffff);
            // result x of one of the two lists: its row's place among whole_* (n = 1) or piece_*
            auto at = [&](int x, int n, int first, size_t whole, size_t pieces, int per, int r) {
                return (n == 1 ? whole : pieces + 2 * ((first & 0x7fffffff) + x) + (x == 0 && first < 0 ? 1 : 0)) * per + r;
            };
            constexpr int AT = 6;                           // partial results in flight a thread
            for (int s = group; s < n_unit + n_own; s += AT * groups) {
                float2 ml[AT];
                float4 x[AT];
#pragma unroll
                for (int u = 0; u < AT; ++u) {
                    const int y = s + u * groups;
                    ml[u] = make_float2(-INFINITY, 0.f);
                    x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (y >= n_unit + n_own) continue;
                    const float *po, *pml;
                    size_t p;
                    if (y < n_unit && tc) {
                        p = at(y, n_unit, from, (size_t)kh * sb::tc_units(a.M, a.R, G) + unit, (size_t)kh * 2 * a.tc.W, rows, row % rows);
                        po = n_unit == 1 ? a.tc.whole_o : a.tc.piece_o;
                        pml = n_unit == 1 ? a.tc.whole_ml : a.tc.piece_ml;
                    } else {
                        const bool own = y >= n_unit;
                        const int n = own ? n_own : n_unit;
                        p = at(own ? y - n_unit : y, n, own ? v.y : from, (size_t)kh * items + (own ? units + i : unit),
                               (size_t)kh * 2 * a.W, RQ, own ? g : row % RQ);
                        po = n == 1 ? a.whole_o : a.piece_o;
                        pml = n == 1 ? a.whole_ml : a.piece_ml;
                    }
                    ml[u] = __ldcg(reinterpret_cast<const float2*>(pml + p * 2));
                    x[u] = __ldcg(reinterpret_cast<const float4*>(po + p * D + d));
                }
#pragma unroll
                for (int u = 0; u < AT; ++u) take(ml[u], x[u]);
            }
        }
        if (group > 0) {
            s_ml[group - 1][t] = make_float2(M, L);
            s_o[group - 1][t] = o;
        }
        __syncthreads();
        if (group == 0 && mine) {
            for (int j = 0; j < groups - 1; ++j) take(s_ml[j][t], s_o[j][t]);
            __nv_bfloat162* to = reinterpret_cast<__nv_bfloat162*>(out + ((size_t)v.w * a.Hq + kh * G) * D + idx);
            to[0] = __floats2bfloat162_rn(o.x / L, o.y / L);
            to[1] = __floats2bfloat162_rn(o.z / L, o.w / L);
        }
        __syncthreads();
    }
}

int stream_smem(int M, int R, int G, int D) {
    return (STAGES * 2 * KT * D + STAGES * RQ * D) * 2 + PAGE_SLOTS * TILE_PAGES * 4 + list_ints(M, R, most_units(M, R, G)) * 4;
}

// Blocks of a KV head: as many as the GPU holds at once (two an SM, or one beside long lists: from 83 members in as many groups on
// at 4 query heads a KV head of 128, from 77 at 8.  One family behind 4,096 keys with up to 1,024 of their own, us a call in a
// graph: 32 query heads, 82 members 82, 84 members 110; 64 query heads, 76 members 85, 78 members 120).
int blocks_of(int M, int R, int Hq, int Hkv, int D, int num_sms) {
    const int w = num_sms * (stream_smem(M, R, Hq / Hkv, D) <= TWO_AN_SM ? 2 : 1) / Hkv;
    return w < 1 ? 1 : w;
}

template <int D, bool large>
int launch_stream(void* out, StreamArgs a, cudaStream_t stream) {
    auto kernel = shared_stream_kernel<D, large>;
    const int G = a.Hq / a.Hkv, smem = stream_smem(a.M, a.R, G, D);
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST);
        if (e != cudaSuccess) { sb_set_error("attention_shared: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    sb::launch(kernel, dim3(a.W * a.Hkv), dim3(32 * NW), smem, stream, a);
    // (four groups where all blocks of four fit the GPU at once)
    const int groups = a.M * a.Hkv <= 2 * a.num_sms ? JOIN : 2;
    sb::launch(shared_stream_join_kernel<D>, dim3(a.M, a.Hkv), dim3(groups * (G * D >= 512 ? 128 : G * D >= 256 ? 64 : 32)), 0, stream,
               (bf16*)out, a, groups);
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

// Entries for at most M members in at most R families; calls with fewer need no more.
void shared_stream_scratch(int M, int R, int Hq, int Hkv, int D, int page_size, int num_sms, long long* floats, long long* ints) {
    const int G = Hq / Hkv, items = most_units(M, R, G) + M;
    const long long blocks = 2ll * num_sms > Hkv ? 2ll * num_sms : Hkv;          // of all KV heads, two an SM
    *floats = ((long long)Hkv * items + 2 * blocks) * RQ * (D + 2);
    *ints = 8ll * M;
    if (shared_tc_supports(M, 1, Hq, Hkv, D, page_size, 1)) {        // (lists of fewer families may fit where these do not)
        *floats += ((long long)Hkv * tc_units(M, R, G) + 2 * blocks) * TC_ROWS * (D + 2);
        *ints += 8ll * M;
    }
}

int shared_stream(void* out, float* part, int* items, const void* q, const void* k_pool, const void* v_pool,
                  const SharedLists& l, int Hq, int Hkv, int D, int page_size, long long num_pages, int window, float scale,
                  int num_sms, int* status, cudaStream_t stream) {
    StreamArgs a{};
    const int G = Hq / Hkv, W = blocks_of(l.M, l.R, Hq, Hkv, D, num_sms);
    const long long most = most_units(l.M, l.R, G) + l.M;
    a.whole_o = part;
    a.whole_ml = a.whole_o + Hkv * most * RQ * D;
    a.piece_o = a.whole_ml + Hkv * most * RQ * 2;
    a.piece_ml = a.piece_o + 2ll * Hkv * W * RQ * D;
    a.items = items;
    a.q = (const bf16*)q; a.k_pool = (const bf16*)k_pool; a.v_pool = (const bf16*)v_pool;
    a.block_table = l.block_table; a.token_rows = l.token_rows; a.positions = l.positions;
    a.members = l.members; a.group_starts = l.group_starts; a.shared_lens = l.shared_lens;
    a.table_width = l.table_width; a.M = l.M; a.R = l.R; a.Hq = Hq; a.Hkv = Hkv; a.BS = page_size; a.window = window; a.W = W;
    a.num_sms = num_sms;
    a.scale_log2 = scale * LOG2E;
    if (status != nullptr && shared_tc_supports(l.M, l.R, Hq, Hkv, D, page_size, num_pages)) {
        const long long units = tc_units(l.M, l.R, G);
        a.tc.W = 2 * num_sms > Hkv ? 2 * num_sms / Hkv : 1;
        a.tc.whole_o = a.piece_ml + 2ll * Hkv * W * RQ * 2;
        a.tc.whole_ml = a.tc.whole_o + Hkv * units * TC_ROWS * D;
        a.tc.piece_o = a.tc.whole_ml + Hkv * units * TC_ROWS * 2;
        a.tc.piece_ml = a.tc.piece_o + 2ll * Hkv * a.tc.W * TC_ROWS * D;
        a.tc.items = a.items + 8ll * l.M;
        const int rc = shared_tc(a.tc, q, k_pool, v_pool, l, Hq, Hkv, D, page_size, num_pages, window, scale, status, stream);
        if (rc != 0) return rc;
        return D == 64 ? launch_stream<64, true>(out, a, stream) : launch_stream<128, true>(out, a, stream);
    }
    switch (D) {
        case 16: return launch_stream<16, false>(out, a, stream);
        case 32: return launch_stream<32, false>(out, a, stream);
        case 64: return launch_stream<64, false>(out, a, stream);
        default: return launch_stream<128, false>(out, a, stream);
    }
}

}  // namespace sb
