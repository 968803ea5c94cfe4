// Paged attention for many packed rows a key head (a batch behind a shared prefix, parts of prompts), f16, on
// the fifth-generation tensor cores.
//
// Bound: the tensor cores, and nearly as much the exponentials: a tile of 128 rows x 128 keys of 128 elements is 512
// cycles of scores and 2 * 512 of values (P has two parts) and, at 16 exponentials a cycle, 1024 of softmax.  (Measured:
// 2240 from the scores to P and 1990 from P to the next scores, a chain of 4230 in which the other tile of the pair has
// its turn, 2 x 1536 of them products; 256 rows a key head behind 16000 shared tokens 38 us, a prompt of 4096 tokens with 32
// heads 137 GF in 208 us = 0.66 PFLOP/s.  A block's start -- counting the work, its first tile -- is 23000 cycles behind
// a prefix and 41000 with row offsets, much of it waiting for instructions; an item's result 4000.)  So an item is two
// tiles of 128 packed rows that share the keys in shared memory and take turns: while one tile's scores are on the tensor
// cores, the other's are exponentials.  One persistent block an SM, 20 warps:
//   warps 0-7, 8-15  softmax of tile 0 / 1, two threads a row (= TMEM lane), 64 keys each -- half the
//                    chain of one thread a row, and half the time results take to leave: the maximum of the scores, the
//                    accumulator rescaled when it has moved by more than 2^4, then the exponentials (f32) against it,
//                    written as the sum of two f16 over the scores they came from (one f16 rounds by as much as the
//                    result's type does, and the row's error was 2.9e-4 of the result instead of 2.1e-4); and the copies
//                    of the tile's queries, those of the next item as soon as the last scores are there
//   warp 16          issues the products: S_t = Q_t K^T into TMEM, O_t += P_t V with P_t's two parts read from TMEM
//   warps 17-19      copy the pages into the 128-byte-swizzled tiles the tensor cores read, 16 keys of one page at a
//                    time (a warp every third 16; one by one where pages are no multiple of 16 tokens, and in the
//                    sequence's last tile); page numbers are fetched a tile ahead; two stages each for keys and
//                    values.  (With every row's address sent through a shuffle a tile's 64 KB took 8700 cycles.)
// TMEM: scores 2 x 128 columns, accumulators 2 x 128.  Products of one thread are done in order, so S_t of the
// next tile may be issued over P_t as soon as P_t V is, and whoever sees S_t complete knows P_t V to be.
// Tried and dropped, with P in one part: a third of the exponentials as polynomials on the fused multiply-add units (a
// 4096-token prompt 171 -> 186 us), P handed over in halves (the same), a first pass over an empty tile to warm the
// instruction cache (64 sequences behind 16000 tokens 60 -> 66 us).  With two: half of the scores kept in registers
// between the two passes (the prompt 210 -> 222), all 64 loaded at once for the maximum (208 -> 215).
// Every wait is bounded; on expiry the kernel records 0x31-0x39, lets its copies land, frees TMEM and returns.
#pragma once
#include "paged_mma.h"

namespace es {
namespace {

constexpr int      WIDE_TR = 256, WIDE_BK = 128, WIDE_OVH = 4, WIDE_SOFTMAX_WARPS = 16, WIDE_COPY_WARPS = 3,
                   WIDE_THREADS = (WIDE_SOFTMAX_WARPS + 1 + WIDE_COPY_WARPS) * 32;
constexpr uint64_t WIDE_WAIT_LIMIT_CYCLES = 4000000000ull; // ~2 s at 2 GHz

struct wide_ctrl_t {
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_done[2], o_free[2], pair[8];
    uint32_t tmem_base;
    uint32_t abort_flag;
};

__device__ __forceinline__ bool wide_wait(paged_params_t const& p, uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t code)
{
    if (mbar_try_wait(bar, parity)) return true;
    long long t0 = clock64();
    uint32_t  spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++spins & 0x3ff) == 0) {
            if (*abort_flag) return false;
            if ((uint64_t)(clock64() - t0) > WIDE_WAIT_LIMIT_CYCLES) {
                *abort_flag = code;
                report(p, code);
                return false;
            }
        }
    }
    return true;
}

// D (TMEM) += A (TMEM, f16 pairs) x B (shared memory)
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, uint32_t const (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// two f32 at a time
__device__ __forceinline__ uint64_t pack2(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& lo, float& hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

constexpr uint32_t WIDE_STAGE_BYTES = WIDE_SOFTMAX_WARPS * 1024; // results on their way out: 32 rows of 16 f16 a warp
template <int DPAD> constexpr uint32_t wide_smem_bytes()
{
    return 6 * (DPAD / 64) * 16384 + WIDE_STAGE_BYTES + (uint32_t)sizeof(wide_ctrl_t) + 1024;
}

template <int DPAD, bool PAGE16> // PAGE16: pages are a multiple of 16 tokens
__global__ void __launch_bounds__(WIDE_THREADS, 1) paged_wide_kernel(const __grid_constant__ paged_params_t p)
{
    constexpr int      TR = WIDE_TR, BK = WIDE_BK, OVH = WIDE_OVH;
    constexpr uint32_t KB = DPAD / 64, BLOCK = 16384, TILE = KB * BLOCK; // 64-element blocks: 128 rows of 128 bytes
    __shared__ sched_smem_t<WIDE_THREADS, 1> sched;
    __shared__ float                         row_value[2][2][2][128]; // what a row's two threads tell one another: [turn][tile][half][row]
    extern __shared__ uint8_t                smem_wide[];
    uint8_t* const     smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_wide) + 1023) & ~uintptr_t(1023));
    wide_ctrl_t* const ctrl = reinterpret_cast<wide_ctrl_t*>(smem + 6 * TILE + WIDE_STAGE_BYTES);
    volatile uint32_t* abort_flag = &ctrl->abort_flag;
    uint32_t const     sQ = smem_u32(smem), sK = sQ + 2 * TILE, sV = sK + 2 * TILE; // two tiles each
    uint32_t const     bars = smem_u32(ctrl);
    // in the order of wide_ctrl_t
    uint32_t const     q_full = bars, k_full = q_full + 16, k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 16, s_full = v_empty + 16,
                   p_ready = s_full + 16, o_done = p_ready + 16, o_free = o_done + 16,
                   pair = o_free + 16;
    int const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 256);
            mbar_init(k_full + 8 * i, WIDE_COPY_WARPS * 32);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, WIDE_COPY_WARPS * 32);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_ready + 8 * i, 256);
            mbar_init(o_done + 8 * i, 1);
            mbar_init(o_free + 8 * i, 256);
        }
        for (int i = 0; i < 8; ++i) mbar_init(pair + 8 * i, 64);
        ctrl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (p.d != DPAD) // columns that no copy fills: zeros
        for (uint32_t i = threadIdx.x * 16; i < 6 * TILE; i += WIDE_THREADS * 16)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sQ + i), "r"(0) : "memory");
    // TMEM is taken when the kernel before is done (ORDER_LATE: that one belongs to this call, and holds what it needs), and
    // the next one may start when it is taken: a kernel that waits for another never holds what that one still has to take.
    if (p.order != ORDER_LATE) ES_PDL_WAIT();
    if (warp == WIDE_SOFTMAX_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t const tmem = ctrl->tmem_base; // scores: + 128 t; accumulators: + 256 + 128 t
    asm volatile("griddepcontrol.launch_dependents;");
    work_t w;
    find_work<TR, BK, OVH, WIDE_THREADS, 1>(p, w, sched);

    if (warp > WIDE_SOFTMAX_WARPS) {
        // ------------------------------------------------------------ copies of keys and values
        constexpr int  CH = DPAD / 8, ROWS_AT = 32 / CH, STEPS = 16 / ROWS_AT;
        int const      lw = warp - WIDE_SOFTMAX_WARPS - 1, c_row = lane / CH, c_chunk = lane % CH;
        bool const     c_on = (uint32_t)c_chunk * 8 < p.d;
        // chunk c of row r lies in block c / 8 at chunk (c % 8) ^ (r % 8)
        uint32_t const c_dst = (uint32_t)(c_chunk >> 3) * BLOCK + c_row * 128 + (((c_chunk & 7) ^ c_row) << 4);
        uint32_t const k_step = (uint32_t)p.k_stride[1] * ROWS_AT, v_step = (uint32_t)p.v_stride[1] * ROWS_AT;
        // the barrier is arrived at when this thread's copies so far have landed; nobody waits here for them
        // (whoever waits for the barrier orders what they wrote before the tensor cores' reads)
        auto commit = [&](uint32_t b) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(b) : "memory"); };
        auto acquire = [&](uint32_t b, uint32_t parity) { // a tile that the products no longer read
            return __all_sync(0xffffffffu, wide_wait(p, b, parity, abort_flag, 0x37)) != 0;
        };
        uint32_t tiles = 0;
        bool     ok = true;
        while (w.left && ok) {
            uint32_t const n = min(w.kt - w.j, w.left), f0 = first_tile_of<OVH>(w.j), f1 = first_tile_of<OVH>(w.j + n);
            // lane g: the page of this tile's keys 16 g ..
            auto page_of = [&](uint32_t j) {
                uint32_t const key = j * BK + lane * 16;
                return PAGE16 && lane < BK / 16 && key < (uint32_t)w.s.len ? (uint32_t)w.s.table[fdivide(key, p.page)] : 0u;
            };
            uint32_t next_page = f1 > f0 ? page_of(f0) : 0u;
            for (uint32_t j = f0; j < f1 && ok; ++j, ++tiles) {
                uint32_t page = next_page;
                if (j + 1 < f1) next_page = page_of(j + 1);
                uint32_t const st = tiles & 1, par = ((tiles >> 1) & 1) ^ 1;
                uint32_t const to_k = sK + st * TILE, to_v = sV + st * TILE;
                if (PAGE16 && (j + 1) * BK <= (uint32_t)w.s.len) {
                    if (page >= p.n_pages) {
                        report(p, PAGED_BAD_PAGE); // (reads page 0, which is there)
                        page = 0;
                    }
                    uint32_t const key = j * BK + lane * 16;
                    uint32_t const slot = lane < BK / 16 ? key - fdivide(key, p.page) * p.page.d : 0u;
                    auto copy_tile = [&](uint32_t to, void const* base, int64_t const (&stride)[3], uint32_t step) {
#pragma unroll
                        for (int x = 0; x < 3; ++x) {
                            uint32_t const g = lw + WIDE_COPY_WARPS * x;
                            if (g < BK / 16) {
                                uint32_t const pg = __shfl_sync(0xffffffffu, page, g), sl = __shfl_sync(0xffffffffu, slot, g);
                                __half const*  src = static_cast<__half const*>(base) + (int64_t)pg * stride[0] +
                                                    (int64_t)(sl + c_row) * stride[1] + (int64_t)w.head * stride[2] + c_chunk * 8;
                                uint32_t const dst = to + g * 2048;
                                if (c_on) {
#pragma unroll
                                    for (int i = 0; i < STEPS; ++i)
                                        copy16(dst + (c_dst ^ (((i * ROWS_AT) & 7) << 4)) + i * ROWS_AT * 128, src + (uint64_t)step * i, true);
                                }
                            }
                        }
                    };
                    if (!(ok = acquire(k_empty + 8 * st, par))) break;
                    copy_tile(to_k, p.k, p.k_stride, k_step);
                    commit(k_full + 8 * st);
                    if (!(ok = acquire(v_empty + 8 * st, par))) break;
                    copy_tile(to_v, p.v, p.v_stride, v_step);
                    commit(v_full + 8 * st);
                } else {
                    if (!(ok = acquire(k_empty + 8 * st, par))) break;
                    if (!(ok = acquire(v_empty + 8 * st, par))) break;
#pragma unroll 1
                    for (uint32_t g = lw; g < BK / 16; g += WIDE_COPY_WARPS) { // lane r < 16 finds key r of 16
                        uint32_t const key = j * BK + g * 16 + lane;
                        int64_t        ko = 0, vo = 0;
                        bool           on = lane < 16 && key < (uint32_t)w.s.len;
                        if (on) {
                            uint32_t const pi = fdivide(key, p.page), slot = key - pi * p.page.d;
                            uint32_t const pg = (uint32_t)w.s.table[pi];
                            on = pg < p.n_pages;
                            if (!on) report(p, PAGED_BAD_PAGE);
                            ko = (int64_t)pg * p.k_stride[0] + (int64_t)slot * p.k_stride[1] + (int64_t)w.head * p.k_stride[2];
                            vo = (int64_t)pg * p.v_stride[0] + (int64_t)slot * p.v_stride[1] + (int64_t)w.head * p.v_stride[2];
                        }
                        unsigned const ons = __ballot_sync(0xffffffffu, on);
#pragma unroll 2
                        for (int i = 0; i < STEPS; ++i) {
                            uint32_t const r = c_row + i * ROWS_AT;
                            int64_t const  k_at = __shfl_sync(0xffffffffu, ko, r), v_at = __shfl_sync(0xffffffffu, vo, r);
                            bool const     live = (ons >> r) & 1;
                            uint32_t const dst = (c_dst ^ (((i * ROWS_AT) & 7) << 4)) + i * ROWS_AT * 128 + g * 2048;
                            if (c_on) {
                                copy16(to_k + dst, live ? (void const*)(static_cast<__half const*>(p.k) + k_at + c_chunk * 8) : p.k, live);
                                copy16(to_v + dst, live ? (void const*)(static_cast<__half const*>(p.v) + v_at + c_chunk * 8) : p.v, live);
                            }
                        }
                    }
                    commit(k_full + 8 * st);
                    commit(v_full + 8 * st);
                }
            }
            next_item<TR, BK, OVH>(p, w, n);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == WIDE_SOFTMAX_WARPS) {
        // ------------------------------------------------------------ products (the whole warp; one lane issues)
        bool leader;
        {
            uint32_t pred;
            asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(pred));
            leader = pred != 0;
        }
        uint64_t const desc_hi = (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32; // 128B swizzle, 1024 bytes between 8-row groups
        uint64_t const desc_v = desc_hi | ((uint64_t)(BLOCK >> 4) << 16);                  // + distance between column blocks
        // D = f32, A / B = f16, N >> 3, M >> 4; P V reads V with the head dim (its N) contiguous
        uint32_t const idesc_s = (1u << 4) | ((uint32_t)(BK >> 3) << 17) | ((128u >> 4) << 24);
        uint32_t const idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DPAD >> 3) << 17) | ((128u >> 4) << 24);
        // (every descriptor is formed by the whole warp, outside the one-lane region: formed inside it a product of
        // K took 59 cycles to issue instead of 35)
        auto issue_s = [&](uint32_t t, uint32_t st) {
            uint64_t const a0 = desc_hi | (uint64_t)((sQ + t * TILE) >> 4), b0 = desc_hi | (uint64_t)((sK + st * TILE) >> 4);
            uint32_t const d = tmem + t * 128, bar = s_full + 8 * t;
            uint64_t       a[KB * 4], b[KB * 4];
#pragma unroll
            for (uint32_t i = 0; i < KB * 4; ++i) {
                uint64_t const o = (uint64_t)(((i >> 2) * BLOCK + (i & 3) * 32) >> 4);
                a[i] = a0 + o;
                b[i] = b0 + o;
            }
            if (leader) {
#pragma unroll
                for (uint32_t i = 0; i < KB * 4; ++i) umma<0>(d, a[i], b[i], idesc_s, i ? 1u : 0u);
                umma_commit(bar);
            }
        };
        auto issue_o = [&](uint32_t t, uint32_t st, bool keep) {
            uint64_t const b0 = desc_v | (uint64_t)((sV + st * TILE) >> 4);
            uint32_t const d = tmem + 256 + t * 128, a0 = tmem + t * 128;
            uint64_t       b[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) b[i] = b0 + (uint64_t)((i * 2048) >> 4);
            if (leader) {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) { // 16 keys a product: 8 TMEM columns of P's larger, 8 of its smaller parts, 16 rows of V
                    uint32_t const a = a0 + (i >> 1) * 32 + (i & 1) * 8;
                    umma_ts(d, a, b[i], idesc_o, (keep || i) ? 1u : 0u);
                    umma_ts(d, a + 16, b[i], idesc_o, 1u);
                }
            }
        };
        auto commit = [&](uint32_t b) {
            if (leader) umma_commit(b);
        };
        auto wait = [&](uint32_t b, uint32_t parity, uint32_t code) {
            bool const got = __all_sync(0xffffffffu, wide_wait(p, b, parity, abort_flag, code)) != 0;
            // keys and values: the copies are ordinary writes, the products' reads are not
            if (code == 0x32 || code == 0x33) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_after();
            return got;
        };
        uint32_t tiles = 0, n_p[2] = {0, 0}, n_o[2] = {0, 0}; // tiles and items of each row tile so far
        bool     ok = true;
        while (w.left && ok) {
            uint32_t const n = min(w.kt - w.j, w.left), f0 = first_tile_of<OVH>(w.j), f1 = first_tile_of<OVH>(w.j + n);
            if (f1 > f0) {
                uint32_t const start = w.t * TR, count = min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
                uint32_t const both = count > 128 ? 2 : 1, n_tiles = f1 - f0;
                ok = wait(k_full + 8 * (tiles & 1), (tiles >> 1) & 1, 0x32);
                for (uint32_t t = 0; t < both && ok; ++t)
                    if ((ok = wait(q_full + 8 * t, n_o[t] & 1, 0x31))) issue_s(t, tiles & 1);
                if (!ok) break;
                commit(k_empty + 8 * (tiles & 1));
                for (uint32_t j = 0; j < n_tiles && ok; ++j) {
                    uint32_t const at = tiles + j;
                    for (uint32_t t = 0; t < both; ++t) {
                        if (j == 0 && !(ok = wait(o_free + 8 * t, (n_o[t] & 1) ^ 1, 0x38))) break;
                        if (t == 0) { // this tile's values and the next one's keys, while the exponentials are under way
                            if (!(ok = wait(v_full + 8 * (at & 1), (at >> 1) & 1, 0x33))) break;
                            if (j + 1 < n_tiles && !(ok = wait(k_full + 8 * ((at + 1) & 1), ((at + 1) >> 1) & 1, 0x32))) break;
                        }
                        if (!(ok = wait(p_ready + 8 * t, n_p[t] & 1, 0x34))) break;
                        ++n_p[t];
                        issue_o(t, at & 1, j != 0);
                        if (t + 1 == both) commit(v_empty + 8 * (at & 1));
                        if (j + 1 == n_tiles) {
                            commit(o_done + 8 * t);
                            ++n_o[t];
                        } else {
                            issue_s(t, (at + 1) & 1);
                            if (t + 1 == both) commit(k_empty + 8 * ((at + 1) & 1));
                        }
                    }
                }
                tiles += n_tiles;
            }
            next_item<TR, BK, OVH>(p, w, n);
        }
    } else {
        // ------------------------------------------------------------ softmax: two threads a row
        constexpr int  OH = DPAD / 2; // columns of the accumulator that a thread looks after
        uint32_t const t = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, r_tile = quarter * 32 + lane;
        uint32_t const lanes = (uint32_t)(quarter * 32) << 16;
        uint32_t const row_s = tmem + t * 128 + half * 64 + lanes, row_o = tmem + 256 + t * 128 + half * OH + lanes;
        uint32_t       n_s = 0, n_o = 0, turn = 0;
        bool           ok = true, split = false;
        // (after a wait has given up nothing is waited for any more, and what is computed means nothing)
        auto wait = [&](uint32_t b, uint32_t parity, uint32_t code) {
            if (ok) ok = __all_sync(0xffffffffu, wide_wait(p, b, parity, abort_flag, code)) != 0;
            tc_fence_after();
        };
        // the other thread's value (the two warps of a quarter meet)
        auto exchange = [&](float x) {
            uint32_t const meet = pair + 8 * (t * 4 + quarter);
            row_value[turn][t][half][r_tile] = x;
            mbar_arrive(meet);
            wait(meet, turn, 0x39);
            float const y = row_value[turn][t][half ^ 1][r_tile];
            turn ^= 1; // (a value is overwritten two meetings later)
            return y;
        };
        // this warp's 16 query rows of an item's tile t (none if the item has no key tile here); tell_q follows
        auto load_q = [&](work_t const& x) -> bool {
            if (x.left == 0) return false;
            uint32_t const n = min(x.kt - x.j, x.left), start = x.t * TR, count = min((uint32_t)TR, (uint32_t)x.s.n * p.group - start);
            if (first_tile_of<OVH>(x.j + n) == first_tile_of<OVH>(x.j) || t * 128 >= count) return false;
            constexpr int  CH = DPAD / 8, ROWS_AT = 32 / CH;
            uint32_t const first = t * 128 + quarter * 32 + half * 16;
            uint32_t const pr = start + min(first + (lane & 15), count - 1), tok = fdivide(pr, p.grp);
            int64_t const  mine = (int64_t)(x.s.row0 + (int)tok) * p.q_stride[0] + (int64_t)(x.head * p.group + (pr - tok * p.group)) * p.q_stride[1];
            uint32_t const c_row = lane / CH, c = lane % CH;
            __half const*  q = static_cast<__half const*>(p.q) + c * 8;
#pragma unroll 4
            for (int i = 0; i < 16 / ROWS_AT; ++i) {
                uint32_t const r = c_row + i * ROWS_AT, row = (first & 127) + r;
                int64_t const  at = __shfl_sync(0xffffffffu, mine, r);
                if (c * 8 < p.d) copy16(sQ + t * TILE + (c >> 3) * BLOCK + row * 128 + (((c & 7) ^ (row & 7)) << 4), q + at, first + r < count);
            }
            return true;
        };
        auto tell_q = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(q_full + 8 * t);
        };
        if (load_q(w)) tell_q();
        while (w.left) {
            uint32_t const n = min(w.kt - w.j, w.left), f0 = first_tile_of<OVH>(w.j), f1 = first_tile_of<OVH>(w.j + n);
            uint32_t const start = w.t * TR, count = min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
            uint32_t const r = t * 128 + r_tile;
            int const      to = segment_slot(w, n);
            auto load_next_q = [&]() { // (not kept: registers)
                work_t wn = w;
                next_item<TR, BK, OVH>(p, wn, n);
                return load_q(wn);
            };
            bool const here = t * 128 < count && f1 > f0; // this warp has rows and keys in the item
            if (!here && load_next_q()) tell_q();
            if (t * 128 < count) {
                float          m = MMA_NO_KEY, l = 0.f; // l: of this thread's keys
                uint32_t const pr = start + min(r, count - 1), tok = fdivide(pr, p.grp);
                int const      vis = visible(p, w.s, (int)tok);
                for (uint32_t j = f0; j < f1; ++j) {
                    wait(s_full + 8 * t, n_s & 1, 0x35);
                    ++n_s;
                    // every product with this item's queries is done: the next item's may come
                    bool const more = j + 1 == f1 && load_next_q();
                    int const  allow = vis - (int)(j * BK + half * 64); // this row sees the first `allow` of the thread's keys
                    bool const mask = __any_sync(0xffffffffu, allow < 64);
                    auto       mask_from = [&](uint32_t (&x)[32], int c) { // scores of keys that the row does not see: -inf
                        if (mask) {
                            int const here = allow - c * 32;
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i >= here) x[i] = 0xff800000u;
                        }
                    };
                    // The tile's maximum first, from one pass over the scores; they are read again for the exponentials, as
                    // there are no registers for 64 of them.
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t x[32];
                        tmem_ld32(row_s + c * 32, x);
                        mask_from(x, c);
#pragma unroll
                        for (int i = 0; i < 16; ++i) mx[i & 1] = max3(mx[i & 1], __uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
                    }
                    float top = fmaxf(mx[0], mx[1]);
                    top = fmaxf(top, exchange(top));
                    if (__any_sync(0xffffffffu, (top - m) * p.scale_log2 > MMA_RESCALE)) { // (the same in both warps)
                        float const mn = fmaxf(m, top), a = ex2((m - mn) * p.scale_log2);
                        m = mn;
                        l *= a;
                        if (j != f0) {
#pragma unroll 1
                            for (int c = 0; c < OH / 16; ++c) {
                                uint32_t o[16];
                                tmem_ld16(row_o + c * 16, o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                                tmem_st16(row_o + c * 16, o);
                            }
                        }
                    }
                    // P as the sum of two f16: 16 columns of the larger and 16 of the smaller parts, over the 32 scores they
                    // came from
                    uint64_t const scale2 = pack2(p.scale_log2, p.scale_log2), lift2 = pack2(MMA_LIFT, MMA_LIFT), m2 = pack2(-m, -m), minus2 = pack2(-1.f, -1.f);
                    uint64_t       sum[2] = {0, 0};
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        uint32_t x[32], y[32];
                        tmem_ld32(row_s + c * 32, x);
                        mask_from(x, c);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float s0, s1;
                            unpack2(fma2(add2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), m2), scale2, lift2), s0, s1);
                            s0 = ex2(s0);
                            s1 = ex2(s1);
                            uint64_t const e = pack2(s0, s1);
                            sum[i & 1] = add2(sum[i & 1], e);
                            y[i] = pack_h2(s0, s1);
                            float2 const f = __half22float2(*reinterpret_cast<__half2 const*>(&y[i]));
                            unpack2(fma2(pack2(f.x, f.y), minus2, e), s0, s1);
                            y[16 + i] = pack_h2(s0, s1);
                        }
                        tmem_st32(row_s + c * 32, y); // (waits for the stores to be done)
                    }
                    tc_fence_before();
                    mbar_arrive(p_ready + 8 * t);
                    float s0, s1;
                    unpack2(add2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                    if (more) tell_q();
                }
                m = fmaf(m, p.scale_log2, -MMA_LIFT); // what the sums are relative to, in log2 units
                float const others = exchange(l);
                l = half ? others + l : l + others; // (the same sum in both)
                if (f1 > f0) {
                    wait(o_done + 8 * t, n_o & 1, 0x36);
                    ++n_o;
                }
                int const      row = w.s.row0 + (int)tok;
                uint32_t const head = w.head * p.group + (pr - tok * p.group);
                uint64_t const at = (uint64_t)row * p.heads + head, part = (uint64_t)(2 * w.worker + max(to, 0)) * TR + r;
                finish_t       f = {0.f, 0.f, 0.f};
                if (to < 0 && p.base_out) wait_for_base(p);
                if (to < 0 && r < count) {
                    f = finish(m, l, p.base_lse != nullptr, p.base_lse ? p.base_lse[at] : 0.f);
                    if (p.lse && half == 0) p.lse[at] = f.lse;
                }
                if (to >= 0 && r < count && half == 0) p.part_ml[part] = make_float2(m, l);
                bool const staged = to < 0 && !p.out_f32; // f16 rows go out through shared memory
                __half*    dst[2] = {};                   // row lane / 2 + 16 i of the warp's 32, elements 8 (lane % 2) ..
                if (staged) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t const rw = t * 128 + quarter * 32 + (lane >> 1) + 16 * i;
                        uint32_t const q = start + min(rw, count - 1), qt = fdivide(q, p.grp);
                        if (rw < count)
                            dst[i] = static_cast<__half*>(p.out) + (int64_t)(w.s.row0 + (int)qt) * p.out_stride[0] +
                                     (int64_t)(w.head * p.group + (q - qt * p.group)) * p.out_stride[1] + half * OH + (lane & 1) * 8;
                    }
                }
                uint32_t const stage = sQ + 6 * TILE + warp * 1024;
#pragma unroll 1
                for (int c = 0; c < OH / 16; ++c) {
                    uint32_t const e = half * OH + c * 16; // of the head dim (a multiple of 8)
                    uint32_t       x[16];
                    if (f1 > f0) {
                        tmem_ld16(row_o + c * 16, x);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = 0;
                    }
                    if (staged) {
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = f.wa == 0.f ? 0.f : __uint_as_float(x[i]) * f.wa; // a weight of 0: the sum may be anything
                        if (p.base_out && f.wb != 0.f) {
                            float const* base = p.base_out + at * p.d + e;
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                if (e + i < p.d) {
                                    float4 const b = *reinterpret_cast<float4 const*>(base + i);
                                    v[i] = fmaf(b.x, f.wb, v[i]);
                                    v[i + 1] = fmaf(b.y, f.wb, v[i + 1]);
                                    v[i + 2] = fmaf(b.z, f.wb, v[i + 2]);
                                    v[i + 3] = fmaf(b.w, f.wb, v[i + 3]);
                                }
                            }
                        }
                        __syncwarp(); // the chunk before has been read
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 32 + ((i ^ ((lane >> 2) & 1)) << 4)),
                                         "r"(pack_h2(v[8 * i], v[8 * i + 1])), "r"(pack_h2(v[8 * i + 2], v[8 * i + 3])),
                                         "r"(pack_h2(v[8 * i + 4], v[8 * i + 5])), "r"(pack_h2(v[8 * i + 6], v[8 * i + 7])) : "memory");
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t const rw = (lane >> 1) + 16 * i;
                            uint4          y;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                                         : "r"(stage + rw * 32 + (((lane & 1) ^ ((rw >> 2) & 1)) << 4)) : "memory");
                            if (dst[i] && e + (lane & 1) * 8 < p.d) *reinterpret_cast<uint4*>(dst[i] + c * 16) = y;
                        }
                    } else if (r < count) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float const v4[4] = {__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])};
                            if (to < 0) {
                                if (e + i < p.d) write_out<__half, 4>(p, row, head, e + i, v4, f, true);
                            } else {
                                // four elements of 256 rows, then the next four: a warp's store is one run of 512 bytes
                                *reinterpret_cast<float4*>(p.part_out + (uint64_t)(2 * w.worker + to) * TR * DPAD + (((e + i) / 4) * TR + r) * 4) =
                                    make_float4(v4[0], v4[1], v4[2], v4[3]);
                            }
                        }
                    }
                }
                if (f1 > f0) {
                    tc_fence_before();
                    mbar_arrive(o_free + 8 * t);
                }
            }
            if (to == 1) {
                split = true;
                if (threadIdx.x == 0) write_meta<TR>(p, w, true);
            }
            next_item<TR, BK, OVH>(p, w, n);
        }
        if (!split && threadIdx.x == 0) write_meta<TR>(p, w, false);
    }
    wait_for_base(p);
    // ------------------------------------------------------------------ teardown
    tc_fence_before();
    __syncthreads();
    if (ctrl->abort_flag) { // a bounded wait expired: products in flight still read shared memory (bounded: ~1 ms)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == WIDE_SOFTMAX_WARPS) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Joins the partial results of the items that crossed shares (see paged_join_kernel): block x the item that
// starts last in share x, block y 16 of its rows; thread (row, 4 elements), a half warp reads 16 rows' runs.  The
// rows leave through shared memory in 16-byte pieces.
template <int DPAD> __global__ void __launch_bounds__(256) paged_wide_join_kernel(const __grid_constant__ paged_params_t p)
{
    constexpr int    TR = WIDE_TR, CH = DPAD / 64; // chunks of 64 elements, 4 a thread
    __shared__ float so[16][DPAD + 4];
    ES_PDL_PROLOGUE();
    int4 const     m0 = p.meta[2 * blockIdx.x], m1 = p.meta[2 * blockIdx.x + 1]; // (m1 means something if m0.x > 0)
    uint32_t const r0 = blockIdx.y * 16;
    if (r0 >= (uint32_t)m0.x) return;
    int const      first = (int)blockIdx.x, n = m1.x - first + 1;
    uint32_t const rows = min((uint32_t)m0.x - r0, 16u), rr = threadIdx.x & 15, c4 = threadIdx.x >> 4;
    uint32_t const r = r0 + min(rr, rows - 1);
    auto  slot = [&](int i) { return (uint64_t)(2 * (first + i) + (i == 0 ? 1 : 0)) * TR; };
    float top = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        float2 const ml = p.part_ml[slot(i) + r];
        top = fmaxf(top, ml.y == 0.f ? -INFINITY : ml.x);
    }
    float o[CH][4] = {}, l = 0.f;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        float2 const ml = p.part_ml[slot(i) + r];
        float const  wgt = ml.y == 0.f ? 0.f : ex2(ml.x - top);
        l = fmaf(ml.y, wgt, l);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float4 const x = *reinterpret_cast<float4 const*>(p.part_out + slot(i) * DPAD + ((c * 16 + c4) * TR + r) * 4);
            o[c][0] = fmaf(x.x, wgt, o[c][0]);
            o[c][1] = fmaf(x.y, wgt, o[c][1]);
            o[c][2] = fmaf(x.z, wgt, o[c][2]);
            o[c][3] = fmaf(x.w, wgt, o[c][3]);
        }
    }
    auto place = [&](uint32_t at_row, int& row, uint32_t& head) {
        uint32_t const pr = (uint32_t)m0.z + at_row, tok = fdivide(pr, p.grp);
        row = m0.y + (int)tok;
        head = (uint32_t)m0.w * p.group + (pr - tok * p.group);
    };
    int      row;
    uint32_t head;
    place(r, row, head);
    uint64_t const at = (uint64_t)row * p.heads + head;
    finish_t const f = finish(top, l, p.base_lse != nullptr, p.base_lse ? p.base_lse[at] : 0.f);
    if (p.lse && c4 == 0 && rr < rows) p.lse[at] = f.lse;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        uint32_t const e = (c * 16 + c4) * 4;
        float          v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = f.wa == 0.f ? 0.f : o[c][k] * f.wa;
            if (p.base_out && f.wb != 0.f && e + k < p.d) v[k] = fmaf(p.base_out[at * p.d + e + k], f.wb, v[k]);
        }
        *reinterpret_cast<float4*>(&so[rr][e]) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    uint32_t const wr = threadIdx.x >> 4;
    if (wr >= rows) return;
    place(r0 + wr, row, head);
    for (uint32_t e = (threadIdx.x & 15) * 8; e < p.d; e += 128) { // (the head dim is a multiple of 8)
        float4 const a = *reinterpret_cast<float4 const*>(&so[wr][e]), b = *reinterpret_cast<float4 const*>(&so[wr][e + 4]);
        if (p.out_f32) {
            float* d = static_cast<float*>(p.out) + ((uint64_t)row * p.heads + head) * p.d + e;
            *reinterpret_cast<float4*>(d) = a;
            *reinterpret_cast<float4*>(d + 4) = b;
        } else {
            __half* d = static_cast<__half*>(p.out) + (int64_t)row * p.out_stride[0] + (int64_t)head * p.out_stride[1] + e;
            *reinterpret_cast<uint4*>(d) = make_uint4(pack_h2(a.x, a.y), pack_h2(a.z, a.w), pack_h2(b.x, b.y), pack_h2(b.z, b.w));
        }
    }
}

} // namespace
} // namespace es
