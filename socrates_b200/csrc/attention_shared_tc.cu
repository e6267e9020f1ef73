// The shared keys of large families on the 5th-generation tensor cores: the part of attention_shared_mma.cu's operator that
// is bound by products, not by bytes.
//
// A family of n tokens brings n x G query rows per KV head to its shared keys.  Units of 16 rows (attention_shared_mma.cu)
// read each key tile once per unit; from a few units on that traffic and the products of mma.sync take longer than the keys'
// bytes from memory.  Here a unit is 128 rows: TMEM lanes, one softmax thread each.  Per tile of 64 keys
//   S = Q K^T          tcgen05.mma kind::f16, both operands in shared memory, S in TMEM (two buffers)
//   softmax            running maximum and sum in float32; the weights go back over the scores as TWO bfloat16 terms, so that
//                      they are not cut to 8 bits before the product
//   O += P V           P from TMEM, V from shared memory (MN-major), O in TMEM, rescaled only when a row's maximum grew by 2^8
// with a warp that issues the copies (TMA, one box per page and 64-dim panel), one the score products, one the P.V
// products, four the softmax, as in attention_tcgen05.cu.
//
// The key tiles of all units are laid end to end (per KV head) and dealt to the blocks in equal shares.  A share may hold the end
// of one unit and the beginning of another (segments): the copies run on across them, and each segment leaves a
// partial result (max, sum, O) for the joining kernel.
//
// 64 tokens (256 rows) behind 8,192 keys, 8 KV heads of 128: 1.2 us a tile and block, two blocks an SM, 1,024 tiles of 128 rows a
// round in 8.5 us; about 10 us more until the first weights are there and 2 for the last results.  The whole call 53 us, 150 with units
// of 16 rows alone, 298 where every row reads its own way (floor 5.4 us of bytes, 5.3 of products).
//
// Every wait on an mbarrier is bounded; a give-up sets *status, and the block still frees its TMEM.
#include <cuda.h>
#include <math.h>

#include "attention_shared.h"
#include "tcgen05_gemm.cuh"
#include "tma_maps.cuh"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int ROWS = sb::TC_ROWS;    // rows of a unit = TMEM lanes = softmax threads
constexpr int KTILE = 64;
constexpr int THREADS = ROWS + 96;   // four softmax warps, the warps that issue score products, copies and P.V products
constexpr int COL_O = 128;           // TMEM columns: S/P buffers of 64 at 0 and 64, then O
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_LOG2 = 8.0f;

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    tcgen05_mma_bf16(d, da, db, idesc, acc);
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// An operand whose contraction dim runs over the rows of 128 bytes: `lbo16` (in 16 bytes) between its 64-dim panels.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr, uint32_t lbo16) {
    const uint32_t lo = ((addr & 0x3FFFFu) >> 4) | (lbo16 << 16);
    const uint32_t hi = 64u | (1u << 14) | (2u << 29);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
// D float32, A and B bfloat16, A K-major, M = 128.
__host__ __device__ constexpr uint32_t make_idesc(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(ROWS >> 4) << 24);
}
__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 && pos + 1 > window ? pos + 1 - window : 0; }

template <int D> constexpr int q_bytes() { return ROWS * D * 2; }
template <int D> constexpr int kv_bytes() { return KTILE * D * 2; }          // one of K or V, one buffer

struct TcArgs {
    sb::TcPart part;
    const bf16* q;
    sb::SharedLists l;
    int Hq, Hkv, BS, window;
    float scale_log2;
    int* status;
};

// A piece of one unit's keys that lies in one share.
struct Segment {
    int unit, begin, end;                // flat tiles of the whole unit
    int x0, x1;                          // flat tiles of the segment
    int row0, nr, lo, hi, tile0;         // rows, keys, and the key tile of flat tile 0
};

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
shared_tc_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const TcArgs a) {
    constexpr int PANELS = D / 64;
    constexpr int PANEL_Q = ROWS * 128, PANEL_KV = KTILE * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], s_full[2], p_ready[2], v_free[2], pv_full, q_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const bool issuer = warp == 4, copier = warp == 5, pv_issuer = warp == 6;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, k_s = q_s + q_bytes<D>(), v_s = k_s + 2 * kv_bytes<D>();
    uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
    const int M = a.l.M, R = a.l.R, G = a.Hq / a.Hkv, units = sb::tc_units(M, R, G);
    int* pre = reinterpret_cast<int*>(gen_base + q_bytes<D>() + 4 * kv_bytes<D>());     // [units + 1] tiles before each unit
    int* uoff = pre + units + 1;                            // [R + 1] units before each family
    int* unit_row0 = uoff + R + 1;                          // [units] first flat row
    int* unit_nr = unit_row0 + units;
    int* unit_lo = unit_nr + units;
    int* unit_hi = unit_lo + units;
    int* unit_table = unit_hi + units;                      // cache row whose table is read
    int* starts = unit_table + units;                       // [R + 1] members before each family
    int* token = starts + R + 1;                            // [M] a member's token and its position
    int* mpos = token + M;
    const int bs_log2 = 31 - __clz(a.BS);
    const int kh = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;

    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&k_full[b]), 1);
            mbar_init(smem_u32(&v_full[b]), 1);
            mbar_init(smem_u32(&s_full[b]), 1);
            mbar_init(smem_u32(&p_ready[b]), ROWS);
            mbar_init(smem_u32(&v_free[b]), 1);
        }
        mbar_init(smem_u32(&pv_full), 1);
        mbar_init(smem_u32(&q_full), ROWS);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (issuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (copier && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tma_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tma_v) : "memory");
    }
    // ---- before pdl_wait(): the lists, positions and the block table (host copies); which families are large, their units
    for (int r = tid; r < R; r += THREADS) {
        const int s0 = a.l.group_starts[r], n = a.l.group_starts[r + 1] - s0;
        starts[r] = s0;
        uoff[r + 1] = sb::tc_family(n, G, a.l.shared_lens[r]) ? (n * G + ROWS - 1) / ROWS : 0;
    }
    if (tid == 0) starts[R] = a.l.group_starts[R];
    for (int i = tid; i < M; i += THREADS) {
        token[i] = a.l.members[i];
        mpos[i] = a.l.positions[token[i]];
    }
    __syncthreads();
    if (warp == 0) {                                        // running sums by one warp: families are few
        if (lane == 0) uoff[0] = 0;
        int before = 0;
        for (int r0 = 0; r0 < R; r0 += 32) {
            int t = r0 + lane < R ? uoff[r0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += up;
            }
            t += before;
            if (r0 + lane < R) uoff[r0 + lane + 1] = t;
            before = __shfl_sync(0xffffffffu, t, 31);
        }
    }
    __syncthreads();
    const int U = uoff[R];
    for (int u = warp; u < U; u += THREADS / 32) {          // a warp per unit, its lanes over the unit's members
        int r = 0, top = R - 1;
        while (r < top) {
            const int mid = (r + top + 1) / 2;
            if (uoff[mid] <= u) r = mid;
            else top = mid - 1;
        }
        const int rows = (starts[r + 1] - starts[r]) * G, v = u - uoff[r];
        const int row0 = starts[r] * G + v * ROWS, nr = min(ROWS, rows - v * ROWS);
        int lo = 0x7fffffff, last = -1;
        for (int x = row0 / G + lane; x <= (row0 + nr - 1) / G; x += 32) {
            lo = min(lo, first_seen(mpos[x], a.window));
            last = max(last, mpos[x]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) {
            const int hi = min(a.l.shared_lens[r], last + 1);
            unit_row0[u] = row0;
            unit_nr[u] = nr;
            unit_lo[u] = lo;
            unit_hi[u] = hi;
            unit_table[u] = a.l.token_rows[token[row0 / G]];
            pre[u + 1] = hi > lo ? (hi + KTILE - 1) / KTILE - lo / KTILE : 0;
        }
    }
    __syncthreads();
    if (warp == 0) {
        if (lane == 0) pre[0] = 0;
        int before = 0;
        for (int u0 = 0; u0 < U; u0 += 32) {
            int t = u0 + lane < U ? pre[u0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += up;
            }
            t += before;
            if (u0 + lane < U) pre[u0 + lane + 1] = t;
            before = __shfl_sync(0xffffffffu, t, 31);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = tmem_slot;
    const int T = U > 0 ? pre[U] : 0, W = max(1, min(a.part.W, T));
    const sb::Cut cut{T, W};
    const bool active = slot < W && T > 0;
    const int x0 = active ? cut.begin(slot) : 0, x1 = active ? cut.begin(slot + 1) : 0;
    auto segment_at = [&](int x, int from) {                // the segment that begins with flat tile x; units before `from` end earlier
        Segment s;
        int u = from;
        while (x >= pre[u + 1]) ++u;
        s.unit = u;
        s.begin = pre[u];
        s.end = pre[u + 1];
        s.x0 = x;
        s.x1 = min(x1, s.end);
        s.row0 = unit_row0[u];
        s.nr = unit_nr[u];
        s.lo = unit_lo[u];
        s.hi = unit_hi[u];
        s.tile0 = s.lo / KTILE - s.begin;
        return s;
    };
    auto give_up = [&](int code) {
        atomicExch(a.status, code);
        atomicExch(&abort_flag, 1);
    };

    // (a softmax thread's query row)
    auto query_row = [&](const Segment& s) {
        const int f = s.row0 + min(tid, s.nr - 1), i = f / G;
        return reinterpret_cast<const uint4*>(a.q + ((size_t)token[i] * a.Hq + kh * G + f - i * G) * D);
    };
    Segment seg0{};
    const uint4* src0 = nullptr;
    if (active && warp < 4) {
        seg0 = segment_at(x0, 0);
        src0 = query_row(seg0);
    }
    // The kernel behind this one goes on from what was complete before this one's wait returned (queries, pages): it is let in
    // only then, and its blocks start where blocks of this one end.  Without a large family it does its own waiting, for
    // this kernel, which ends when its first block has waited: the other blocks make room at once.
    if (U == 0) sb::pdl_launch_dependents();
    if (U > 0 || blockIdx.x == 0) sb::pdl_wait();
    if (U > 0) sb::pdl_launch_dependents();
    if (blockIdx.x == 0) {                                  // for the joining kernel
        int4* where = reinterpret_cast<int4*>(a.part.items);
        for (int i = tid; i < M; i += THREADS) {
            int r = 0, top = R - 1;
            while (r < top) {
                const int mid = (r + top + 1) / 2;
                if (starts[mid] <= i) r = mid;
                else top = mid - 1;
            }
            int4 w = make_int4(-1, 0, 0, 0);
            int rest = 0;
            if (uoff[r + 1] > uoff[r]) {
                w.x = uoff[r] * ROWS + (i - starts[r]) * G;
                const int u = w.x / ROWS;
                const int2 first = cut.parts(pre[u], pre[u + 1]), second = cut.parts(pre[u + 1], pre[min(u + 2, U)]);
                w.y = first.x; w.z = first.y; w.w = second.x;
                rest = second.y;
            }
            where[2 * i] = w;
            a.part.items[8 * i + 4] = rest;
        }
    }
    if (!active) {
    } else if (copier) {
        // Tile t's keys go to K buffer t&1 once QK(t-2) has read it, its values to V buffer t&1 once PV(t-2) has.  Each lane
        // issues one box (page, panel); page numbers are read a tile ahead.
        const int pages = KTILE >> bs_log2, n_ops = pages * PANELS;          // at most 8
        const int pg = lane / PANELS, p = lane - pg * PANELS;
        Segment s = segment_at(x0, 0);
        auto page_of = [&](int x) {
            const int logical = (((s.tile0 + x) * KTILE) >> bs_log2) + pg;
            return logical <= ((s.hi - 1) >> bs_log2) ? a.l.block_table[(size_t)unit_table[s.unit] * a.l.table_width + logical] : 0;
        };
        int next = lane < n_ops ? page_of(x0) : 0;
        int keys = 0, values = 0;                           // tiles whose keys and values were asked for
        for (int t = 0; t < x1 - x0; ++t) {
            const int b = t & 1, y = (next * a.Hkv + kh) * a.BS;
            if (x0 + t + 1 < x1) {
                if (x0 + t + 1 == s.end) s = segment_at(x0 + t + 1, s.unit + 1);
                if (lane < n_ops) next = page_of(x0 + t + 1);
            }
            const uint32_t off = b * kv_bytes<D>() + p * PANEL_KV + pg * a.BS * 128;
            if (t >= 2 && !mbar_wait_warp(smem_u32(&s_full[b]), ((t - 2) >> 1) & 1)) { if (lane == 0) give_up(27); break; }
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&k_full[b]), kv_bytes<D>());
            keys = t + 1;
            __syncwarp();
            if (lane < n_ops) tma_load_2d(k_s + off, &tma_k, smem_u32(&k_full[b]), p * 64, y);
            if (t >= 2 && !mbar_wait_warp(smem_u32(&v_free[b]), ((t - 2) >> 1) & 1)) { if (lane == 0) give_up(28); break; }
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&v_full[b]), kv_bytes<D>());
            values = t + 1;
            __syncwarp();
            if (lane < n_ops) tma_load_2d(v_s + off, &tma_v, smem_u32(&v_full[b]), p * 64, y);
        }
        // the block outlives its copies, also when a wait gave up (bounded; both buffers' last ones)
        for (int t = max(0, keys - 2); t < keys; ++t) mbar_wait_warp(smem_u32(&k_full[t & 1]), (t >> 1) & 1);
        for (int t = max(0, values - 2); t < values; ++t) mbar_wait_warp(smem_u32(&v_full[t & 1]), (t >> 1) & 1);
    } else if (issuer) {
        constexpr uint32_t idesc_qk = make_idesc(KTILE, false);
        const uint64_t dq = make_smem_desc(q_s), dk = make_smem_desc(k_s);
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const int n = __shfl_sync(0xffffffffu, x1 - x0, 0);
        int segments = 0, seg_end = 0, u = 0;                // tile at which the next segment begins
        for (int i = 0; i < n; ++i) {
            const int b = i & 1;
            if (i == seg_end) {                             // the segment's queries
                while (x0 + i >= pre[u + 1]) ++u;
                seg_end = __shfl_sync(0xffffffffu, min(x1, pre[u + 1]) - x0, 0);
                if (!mbar_wait_warp(smem_u32(&q_full), segments & 1)) { give_up(29); break; }
                ++segments;
            }
            if (!mbar_wait_warp(smem_u32(&k_full[b]), (i >> 1) & 1)) { give_up(21); break; }
            // S[b] still holds P(i-2), the A operand of PV(i-2), which must have completed before it is overwritten
            if (i >= 2 && !mbar_wait_warp(smem_u32(&v_free[b]), ((i - 2) >> 1) & 1)) { give_up(23); break; }
            if (__any_sync(0xffffffffu, *((volatile int*)&abort_flag))) break;
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t pq = ((kk >> 2) * PANEL_Q + (kk & 3) * 32) >> 4;
                    const uint32_t pk = (b * kv_bytes<D>() + (kk >> 2) * PANEL_KV + (kk & 3) * 32) >> 4;
                    mma_ss(tmem_u + 64 * b, dq + pq, dk + pk, idesc_qk, kk > 0 ? 1u : 0u);
                }
                tcgen05_commit(smem_u32(&s_full[b]));
            }
        }
    } else if (pv_issuer) {
        constexpr uint32_t idesc_pv = make_idesc(D, true);
        const uint64_t dv = desc_mnmajor(v_s, PANEL_KV >> 4);
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const int n = __shfl_sync(0xffffffffu, x1 - x0, 0);
        int seg_end = 0, u = 0;
        for (int i = 0; i < n; ++i) {
            const int b = i & 1;
            const bool first = i == seg_end;                // O starts anew
            if (first) {
                while (x0 + i >= pre[u + 1]) ++u;
                seg_end = __shfl_sync(0xffffffffu, min(x1, pre[u + 1]) - x0, 0);
            }
            if (!mbar_wait_warp(smem_u32(&p_ready[b]), (i >> 1) & 1)) { give_up(26); break; }
            if (!mbar_wait_warp(smem_u32(&v_full[b]), (i >> 1) & 1)) { give_up(24); break; }
            if (__any_sync(0xffffffffu, *((volatile int*)&abort_flag))) break;
            tcgen05_fence_after();
            if (elect_one()) {
                const uint32_t pbase = tmem_u + 64 * b;
#pragma unroll
                for (int j = 0; j < KTILE / 16; ++j)
                    mma_ts(tmem_u + COL_O, pbase + j * 8, dv + ((b * kv_bytes<D>() + j * 2048) >> 4), idesc_pv, !first || j > 0 ? 1u : 0u);
#pragma unroll
                for (int j = 0; j < KTILE / 16; ++j)
                    mma_ts(tmem_u + COL_O, pbase + 32 + j * 8, dv + ((b * kv_bytes<D>() + j * 2048) >> 4), idesc_pv, 1u);
                tcgen05_commit(smem_u32(&pv_full));
                tcgen05_commit(smem_u32(&v_free[b]));
            }
        }
    } else {
        // =============================================================== the softmax warps
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        bool ok = true;
        int i = 0, u = 0;
        while (ok && x0 + i < x1) {
            const Segment s = i == 0 ? seg0 : segment_at(x0 + i, u);
            u = s.unit;
            // ---- Q: flat row row0 + r is head r % G of a member, into the swizzled panels, a row by D / 8 neighbouring threads.
            // The score products of the segment before have read theirs: their last scores were met here.
            {
                // A thread brings its own row: lanes read 16 bytes of 32 rows at a time, which costs little of 32 KB and few
                // instructions.  (Straight code is paid for when it is met the first time: about 3 ns an instruction.)
                constexpr int CH = D / 8;
                uint4 v[CH];
                const bool mine = tid < s.nr;
                const uint4* src = i == 0 ? src0 : query_row(s);
#pragma unroll
                for (int c = 0; c < CH; ++c) v[c] = mine ? __ldcg(src + c) : make_uint4(0, 0, 0, 0);
                uint8_t* to = gen_base + tid * 128;
                const int swizzle = (tid & 7) << 4;
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    *reinterpret_cast<uint4*>(to + (c >> 3) * PANEL_Q + (((c & 7) << 4) ^ swizzle)) = v[c];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(smem_u32(&q_full));
            }
            // what row `tid` sees, and what every row of the unit sees
            const int pos = tid < s.nr ? mpos[(s.row0 + tid) / G] : -1;
            const int khi = min(pos, s.hi - 1), klo = max(first_seen(pos, a.window), s.lo);
            const bool busy = warp * 32 < s.nr;              // a warp without rows only keeps the pace
            float m_ref = -INFINITY, l_run = 0.f;
            const int first = i;
            for (; x0 + i < s.x1; ++i) {
                const int b = i & 1;
                const int tile_start = (s.tile0 + x0 + i) * KTILE;
                bool got = mbar_wait(smem_u32(&s_full[b]), (i >> 1) & 1);
                if (*((volatile int*)&abort_flag)) got = false;
                if (!__all_sync(0xffffffffu, got)) { ok = false; if (lane == 0) give_up(22); break; }
                tcgen05_fence_after();
                if (busy) {
                    float sc[64];
                    {
                        uint32_t raw[32];
                        tmem_ld32(lane_base + 64 * b, raw);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) sc[j] = __uint_as_float(raw[j]);
                        tmem_ld32(lane_base + 64 * b + 32, raw);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) sc[32 + j] = __uint_as_float(raw[j]);
                    }
                    const int see0 = klo - tile_start, see1 = khi - tile_start;      // keys see0 .. see1 of the tile
                    if (!__all_sync(0xffffffffu, see0 <= 0 && see1 >= KTILE - 1)) {
                        auto bits = [&](int n) {             // the lowest n of 32
                            return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
                        };
                        const uint32_t m0 = bits(see1 + 1) & ~bits(see0), m1 = bits(see1 - 31) & ~bits(see0 - 32);
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            sc[j] = m0 >> j & 1u ? sc[j] : -INFINITY;
                            sc[32 + j] = m1 >> j & 1u ? sc[32 + j] : -INFINITY;
                        }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        mx4[0] = fmaxf(mx4[0], sc[j]);
                        mx4[1] = fmaxf(mx4[1], sc[j + 1]);
                        mx4[2] = fmaxf(mx4[2], sc[j + 2]);
                        mx4[3] = fmaxf(mx4[3], sc[j + 3]);
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    const bool grow = mx > -INFINITY && (m_ref == -INFINITY || (mx - m_ref) * a.scale_log2 > RESCALE_LOG2);
                    if (__any_sync(0xffffffffu, grow)) {
                        float alpha = 1.0f;
                        if (grow) {
                            alpha = m_ref == -INFINITY ? 0.f : exp2f((m_ref - mx) * a.scale_log2);
                            m_ref = mx;
                            l_run *= alpha;
                        }
                        if (i > first) {                    // O of the tiles before this one is complete once PV(i-1) is
                            if (!mbar_wait_warp(smem_u32(&pv_full), (i - 1) & 1)) { ok = false; if (lane == 0) give_up(23); break; }
                            tcgen05_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t ov[32];
                                tmem_ld32(lane_base + COL_O + c, ov);
                                tmem_ld_wait();
                                uint32_t w0[16], w1[16];
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    w0[j] = __float_as_uint(__uint_as_float(ov[j]) * alpha);
                                    w1[j] = __float_as_uint(__uint_as_float(ov[16 + j]) * alpha);
                                }
                                tmem_st16(lane_base + COL_O + c, w0);
                                tmem_st16(lane_base + COL_O + c + 16, w1);
                            }
                        }
                    }
                    const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref * a.scale_log2;
                    float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KTILE; c += 32) {
                        uint32_t ph[16], pl[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float p0 = ex2_approx(fmaf(sc[c + 2 * j], a.scale_log2, neg_m));
                            const float p1 = ex2_approx(fmaf(sc[c + 2 * j + 1], a.scale_log2, neg_m));
                            l4[j & 3] += p0 + p1;
                            const uint32_t h = pack_bf16(p0, p1);
                            ph[j] = h;
                            pl[j] = pack_bf16(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
                        }
                        tmem_st16(lane_base + 64 * b + (c >> 1), ph);
                        tmem_st16(lane_base + 64 * b + 32 + (c >> 1), pl);
                    }
                    l_run += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                    tmem_st_wait();
                }
                // slots of this tile outside [lo, hi): zero their V rows (thread j < 64 owns key j), whatever stands there
                if (tile_start < s.lo || tile_start + KTILE > s.hi) {
                    if (!mbar_wait_warp(smem_u32(&v_full[b]), (i >> 1) & 1)) { ok = false; if (lane == 0) give_up(24); break; }
                    if (tid < KTILE && (tile_start + tid < s.lo || tile_start + tid >= s.hi)) {
#pragma unroll
                        for (int p = 0; p < PANELS; ++p) {
                            uint4* row = reinterpret_cast<uint4*>(gen_base + (v_s - base) + b * kv_bytes<D>() + p * PANEL_KV + tid * 128);
#pragma unroll
                            for (int c = 0; c < 8; ++c) row[c] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                // follow the product barrier phase by phase: a parity wait cannot tell a phase from the one two before it
                if (i > 0 && !mbar_wait_warp(smem_u32(&pv_full), (i - 1) & 1)) { ok = false; if (lane == 0) give_up(23); break; }
                tcgen05_fence_before();
                mbar_arrive(smem_u32(&p_ready[b]));
            }
            if (!ok) break;
            // ---- the segment's partial result: row `tid`
            bool done = mbar_wait(smem_u32(&pv_full), (i - 1) & 1);
            if (*((volatile int*)&abort_flag)) done = false;
            if (!__all_sync(0xffffffffu, done)) { if (lane == 0) give_up(25); break; }
            tcgen05_fence_after();
            if (busy) {
                const bool whole = s.begin >= x0 && s.end <= x1;
                const size_t p = whole ? (size_t)kh * units + s.unit : ((size_t)kh * a.part.W + slot) * 2 + (s.begin <= x0 ? 0 : 1);
                float* to_o = (whole ? a.part.whole_o : a.part.piece_o) + (p * ROWS + tid) * D;
                float* to_ml = (whole ? a.part.whole_ml : a.part.piece_ml) + (p * ROWS + tid) * 2;
                if (tid < s.nr) *reinterpret_cast<float2*>(to_ml) = make_float2(m_ref * a.scale_log2, l_run);
                // 32 columns at a time through shared memory, where the queries were (the segment's products are done): a warp's
                // rows of 32 floats, 16-byte pieces swizzled by the row, are read back so that eight lanes store 128 bytes of a row.
                float4* stage = reinterpret_cast<float4*>(gen_base + warp * 4096);
                float* warp_o = to_o - (size_t)lane * D;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t ov[32];
                    tmem_ld32(lane_base + COL_O + c, ov);
                    tmem_ld_wait();
                    const float* f = reinterpret_cast<const float*>(ov);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        stage[lane * 8 + (j ^ (lane & 7))] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int row = 4 * j + (lane >> 3), x = lane & 7;
                        const float4 v = stage[row * 8 + (x ^ (row & 7))];
                        if (warp * 32 + row < s.nr) *reinterpret_cast<float4*>(warp_o + (size_t)row * D + c + 4 * x) = v;
                    }
                }
                __syncwarp();
                tcgen05_fence_before();                     // before the next segment's first product writes O
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (issuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
}

template <int D> int tc_smem(int M, int R, int G) {
    const int units = sb::tc_units(M, R, G);
    return q_bytes<D>() + 4 * kv_bytes<D>() + 1024 + (units + 1 + 2 * (R + 1) + 5 * units + 2 * M) * 4;
}

template <int D> int launch_tc(const CUtensorMap& mk, const CUtensorMap& mv, const TcArgs& a, cudaStream_t stream) {
    auto kernel = shared_tc_kernel<D>;
    static sb::OncePerDevice once_per_device;
    bool& configured = once_per_device.flag();
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sb::TC_SMEM_MOST);
        if (e != cudaSuccess) { sb_set_error("attention_shared: %s", cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    sb::launch(kernel, dim3(a.part.W * a.Hkv), dim3(THREADS), tc_smem<D>(a.l.M, a.l.R, a.Hq / a.Hkv), stream, mk, mv, a);
    return 0;
}

}  // namespace

namespace sb {

bool shared_tc_supports(int M, int R, int Hq, int Hkv, int D, int page_size, long long num_pages) {
    if (!(D == 64 || D == 128) || !(page_size == 16 || page_size == 32 || page_size == 64)) return false;
    if (M * (Hq / Hkv) <= 32) return false;                 // no family can be large
    if (num_pages <= 0 || num_pages * Hkv * page_size >= (1ll << 31)) return false;
    return tc_smem<128>(M, R, Hq / Hkv) <= TC_SMEM_MOST;
}

int shared_tc(const TcPart& part, const void* q, const void* k_pool, const void* v_pool, const SharedLists& l, int Hq, int Hkv,
              int D, int page_size, long long num_pages, int window, float scale, int* status, cudaStream_t stream) {
    CUtensorMap mk, mv;
    const int rows = (int)(num_pages * Hkv * page_size);
    if (!get_map(&mk, k_pool, rows, D, page_size) || !get_map(&mv, v_pool, rows, D, page_size)) {
        sb_set_error("attention_shared: cuTensorMapEncodeTiled failed");
        return SB_ERR_ARG;
    }
    const TcArgs a{part, (const bf16*)q, l, Hq, Hkv, page_size, window, scale * LOG2E, status};
    return D == 64 ? launch_tc<64>(mk, mv, a, stream) : launch_tc<128>(mk, mv, a, stream);
}

}  // namespace sb
