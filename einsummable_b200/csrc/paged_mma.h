// Paged attention for few packed rows a key head (single tokens), f16, on the warp-level matrix units.
//
// Bound: memory -- a key and value of 128 are 512 bytes for 4 * 128 flops a row.  So everything serves a steady
// stream of loads: a warp is a worker of its own.  It owns a ring of tiles of 16 keys and their values in
// shared memory, filled by 16-byte asynchronous copies that run MMA_STAGES - 1 tiles ahead, also across the
// end of one item and the start of the next (the queries of an item travel with its first tile), and meets no
// other warp after the work has been shared out.  What a warp does for a tile is one chain of dependent
// instructions with one other warp on its scheduler, so their number counts: the products are taken transposed,
//   S^T = K Q^T  (16 keys x 8 rows),   O^T += V^T P^T  (head dim x 8 rows),
// keys and head dim as the 16 of m16n8k16 and 8 packed rows as its N -- half the matrix instructions, half the
// accumulators and half the exponentials of 16-row tiles when a key head has up to 8 query heads.  P^T goes from
// accumulators to the second product through a register transpose.  The running maximum is moved, and the
// accumulators rescaled, only when a score passes it by more than 2^4: one vote a tile, no reduction.
// (With 16-row tiles, per-tile maxima and copy addresses formed anew for every copy a tile took 570
// instructions and 1.6 us a warp, and 64 ragged sequences 117 us.)
// Measured, 32 query heads on 8 key heads of 128: 2 x 131070 keys (1.07 GB) 175 us = 6.1 TB/s, 64 sequences of
// 1 to 8192 tokens (252 MB) 51 us = 4.9 TB/s; 8 warps of 3 stages an SM (2 stages: 66 us for the ragged batch where
// 3 took 62).
#pragma once
#include "paged_work.h"
#include "tc_ptx.h"

namespace es {
namespace {

constexpr int MMA_BK = 16, MMA_OVH = 6, MMA_WARPS = 4, MMA_STAGES = 3;
// Exponentials are taken 2^11 times as large: f16 has steps of 2^-24 below 2^-14, and what is lost of a weight there
// is then 2^-36 of the largest instead of 2^-25, which put 30000 small weights behind a large one of value 0
// off by 0.6 %.  2^11 x 2^4, what the maximum may be passed by, stays within f16.
constexpr float MMA_LIFT = 11.f, MMA_RESCALE = 4.f;
// The maximum is kept in units of the scores and subtracted before they are scaled: the difference of near scores is
// exact, and that of the largest from itself 0, however large they are (against a scaled and rounded maximum the
// exponentials of scores beyond 2^28 were infinite).
constexpr float MMA_NO_KEY = -1e37f; // the maximum before the first key: below all f16 scores, and finite: no inf - inf

template <int OFF> __device__ __forceinline__ void copy16_at(uint32_t dst, void const* src)
{
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
// 16 bytes into shared memory, zeros when !on
__device__ __forceinline__ void copy16(uint32_t dst, void const* src, bool on)
{
    int const n = on ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int OFF> __device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFF) : "memory");
}
template <int OFF> __device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFF) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t const (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) // of f16 pairs
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// copies i = 0 .. N - 1: row i of `src`, `step` elements apart, to place i % PLACES, i * PITCH + OFF behind it
template <int OFF, int N, int PLACES, int PITCH, int I = 0>
__device__ __forceinline__ void copy_rows(uint32_t const (&to)[PLACES], __half const* src, uint32_t step)
{
    if constexpr (I < N) {
        copy16_at<OFF + I * PITCH>(to[I % PLACES], src + (uint64_t)step * I);
        copy_rows<OFF, N, PLACES, PITCH, I + 1>(to, src, step);
    }
}

// bytes of shared memory a warp; q_rows: rows of a query tile that can exist
template <int DPAD> constexpr uint32_t mma_warp_bytes(uint32_t q_rows)
{
    return MMA_STAGES * (2 * MMA_BK * DPAD * 2 + q_rows * DPAD * 2);
}

// NT: tiles of 8 packed rows an item; PAGE16: pages are a multiple of 16 tokens, so that a tile lies in one; BASE: a
// prefix's result is merged in (a kernel of its own, for the registers that takes)
template <int DPAD, int NT, bool PAGE16, bool BASE>
__global__ void __launch_bounds__(MMA_WARPS * 32, 2) paged_mma_kernel(const __grid_constant__ paged_params_t p, uint32_t q_rows)
{
    constexpr int TR = 8 * NT, BK = MMA_BK, OVH = MMA_OVH, THREADS = MMA_WARPS * 32, CH = DPAD / 8; // CH: 16-byte chunks a row
    constexpr int ROW = DPAD * 2, TILE = BK * ROW, KS = DPAD / 16;
    __shared__ sched_smem_t<THREADS, MMA_WARPS> sched;
    extern __shared__ __align__(128) uint8_t smem_mma[];
    int const      lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t const stage_bytes = 2 * TILE + q_rows * ROW;
    uint32_t const ring = smem_u32(smem_mma) + warp * MMA_STAGES * stage_bytes, ring_end = ring + MMA_STAGES * stage_bytes;
    if (p.d != DPAD) { // columns that no copy fills: zeros (0 * what lies there would not do)
        for (uint32_t i = ring + lane * 16; i < ring_end; i += 512)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(i), "r"(0) : "memory");
        __syncwarp();
    }
    begin_order(p);
    work_t w;
    find_work<TR, BK, OVH, THREADS, MMA_WARPS>(p, w, sched);
    bool split = false;
    if (w.left) {
        // a copy: CH lanes a row, ROWS_AT rows at a time; 16-byte chunk c of row r lies at chunk c ^ (r & 7)
        constexpr int  ROWS_AT = 32 / CH, COPIES = BK / ROWS_AT;
        uint32_t const c_row = lane / CH, c_chunk = lane % CH;
        bool const     c_on = c_chunk * 8 < p.d;
        uint32_t const c_dst = c_row * ROW + ((c_chunk ^ c_row) << 4);
        uint32_t const k_step = (uint32_t)p.k_stride[1] * ROWS_AT, v_step = (uint32_t)p.v_stride[1] * ROWS_AT; // elements
        // chunks' places in the rows r + ROWS_AT * i repeat after 4 (128 elements) or 2 (64) steps
        constexpr int PLACES = 8 / ROWS_AT;
        work_t         wl = w; // the copies' place in the work
        uint32_t       fill = ring;
        bool           first_tile = true; // of an item
        __half const  *ks = nullptr, *vs = nullptr; // this lane's part of the next tile's first rows
        uint32_t       slot = 0, page_no = 0, page_next = 0;
        uint32_t const fronts = (p.front + BK - 1) / BK; // key tiles in front of a sequence's own
        int32_t const* table = nullptr;                  // the pages being read and the tokens in them
        int            len = 0;
        // next tile of the item in a new page: its number was fetched a page ahead
        auto enter_page = [&](uint32_t page) {
            if (page >= p.n_pages) { // reported where it was found; reads page 0, which is there
                report(p, PAGED_BAD_PAGE);
                page = 0;
            }
            ks = static_cast<__half const*>(p.k) + (int64_t)page * p.k_stride[0] + (int64_t)(slot + c_row) * p.k_stride[1] +
                 (int64_t)wl.head * p.k_stride[2] + c_chunk * 8;
            vs = static_cast<__half const*>(p.v) + (int64_t)page * p.v_stride[0] + (int64_t)(slot + c_row) * p.v_stride[1] +
                 (int64_t)wl.head * p.v_stride[2] + c_chunk * 8;
            ++page_no;
            if ((uint64_t)page_no * p.page.d < (uint32_t)len) page_next = (uint32_t)table[page_no];
        };
        auto issue = [&]() { // one tile's copies (or none) and their group
            if (wl.left && to_next_tile<OVH>(wl)) {
                uint32_t const tile = wl.j - OVH;
                bool const     front = tile < fronts, enter = first_tile || tile == fronts;
                int const      key0 = (int)((front ? tile : tile - fronts) * BK);
                if (enter) {
                    table = front ? p.front_pages : wl.s.table;
                    len = front ? (int)p.front : wl.s.len;
                }
                if (first_tile) {
                    first_tile = false;
                    uint32_t const start = wl.t * TR;
                    uint32_t const count = min((uint32_t)TR, (uint32_t)wl.s.n * p.group - start);
                    for (uint32_t r = c_row; r < count; r += ROWS_AT) {
                        uint32_t const pr = start + r, tok = fdivide(pr, p.grp);
                        __half const*  src = static_cast<__half const*>(p.q) + (int64_t)(wl.s.row0 + (int)tok) * p.q_stride[0] +
                                            (int64_t)(wl.head * p.group + (pr - tok * p.group)) * p.q_stride[1] + c_chunk * 8;
                        if (c_on) copy16(fill + 2 * TILE + r * ROW + ((c_chunk ^ (r & 7)) << 4), src, true);
                    }
                }
                if (PAGE16 && enter && key0 < len) {
                    page_no = fdivide((uint32_t)key0, p.page);
                    slot = (uint32_t)key0 - page_no * p.page.d;
                    enter_page((uint32_t)table[page_no]);
                }
                if (PAGE16 && key0 + BK <= len) {
                    if (slot == p.page.d) {
                        slot = 0;
                        enter_page(page_next);
                    }
                    slot += BK;
                    if (c_on) {
                        uint32_t to[PLACES];
#pragma unroll
                        for (int i = 0; i < PLACES; ++i) to[i] = fill + (c_dst ^ ((i * ROWS_AT) << 4));
                        copy_rows<0, COPIES, PLACES, ROWS_AT * ROW>(to, ks, k_step);
                        copy_rows<TILE, COPIES, PLACES, ROWS_AT * ROW>(to, vs, v_step);
                    }
                    ks += k_step * (uint32_t)COPIES;
                    vs += v_step * (uint32_t)COPIES;
                } else {
                    // the sequence's last, incomplete tile, or pages that end inside tiles: lane r < 16 finds key r
                    int64_t ko = 0, vo = 0;
                    bool    ok = false;
                    if (lane < BK && key0 + lane < len) {
                        uint32_t const key = (uint32_t)(key0 + lane), pi = fdivide(key, p.page);
                        uint32_t const page = (uint32_t)table[pi], at = key - pi * p.page.d;
                        ok = page < p.n_pages;
                        if (!ok) report(p, PAGED_BAD_PAGE);
                        ko = (int64_t)page * p.k_stride[0] + (int64_t)at * p.k_stride[1] + (int64_t)wl.head * p.k_stride[2];
                        vo = (int64_t)page * p.v_stride[0] + (int64_t)at * p.v_stride[1] + (int64_t)wl.head * p.v_stride[2];
                    }
                    unsigned const oks = __ballot_sync(0xffffffffu, ok);
#pragma unroll 2
                    for (int i = 0; i < COPIES; ++i) {
                        uint32_t const r = c_row + i * ROWS_AT;
                        uint32_t const d = fill + (c_dst ^ (((i * ROWS_AT) & 7) << 4)) + i * ROWS_AT * ROW;
                        int64_t const  k_at = __shfl_sync(0xffffffffu, ko, r), v_at = __shfl_sync(0xffffffffu, vo, r);
                        bool const     on = (oks >> r) & 1;
                        if (c_on) { // (a copy that is off reads nothing and writes zeros)
                            copy16(d, on ? (void const*)(static_cast<__half const*>(p.k) + k_at + c_chunk * 8) : p.k, on);
                            copy16(d + TILE, on ? (void const*)(static_cast<__half const*>(p.v) + v_at + c_chunk * 8) : p.v, on);
                        }
                    }
                }
                fill = fill + stage_bytes == ring_end ? ring : fill + stage_bytes;
                if (++wl.j == wl.kt || wl.left == 1) {
                    first_tile = true;
                    next_item<TR, BK, OVH>(p, wl, 1);
                } else {
                    --wl.left;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll 1
        for (int i = 0; i < MMA_STAGES - 1; ++i) issue();
        uint32_t  st = ring;
        int const g = lane >> 2, t4 = lane & 3, mi = lane >> 3, l7 = lane & 7;
        // ldmatrix: where this lane's 8 elements lie, for the even and odd step pairs of the head dim
        uint32_t kx[4], vx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kx[i] = (((mi & 1) * 8 + l7) * ROW + (((mi >> 1) ^ l7) << 4)) ^ (i << 5);
            vx[i] = ((((mi >> 1) * 8 + l7) * ROW + (((mi & 1) ^ l7) << 4)) ^ (i << 5)) + TILE;
        }
        while (w.left) {
            uint32_t const n_units = min(w.kt - w.j, w.left);
            uint32_t const start = w.t * TR;
            uint32_t const count = min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
            // thread: rows 8 nt + 2 t4 + x; in S^T keys g and g + 8, in O^T elements 16 dt + g and + 8
            float    o[NT][KS][4], l[NT][2], m[NT][2];
            int      vis[NT][2];
            uint32_t q[NT][KS][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < KS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    l[nt][x] = 0.f;
                    m[nt][x] = MMA_NO_KEY;
                    uint32_t const pr = min(start + nt * 8 + t4 * 2 + x, start + count - 1);
                    vis[nt][x] = visible(p, w.s, (int)fdivide(pr, p.grp));
                }
            }
            int const vis_all = visible(p, w.s, (int)fdivide(start, p.grp)); // keys that every row of the tile sees
            uint32_t const n_tiles = first_tile_of<OVH>(w.j + n_units) - first_tile_of<OVH>(w.j);
            // number of the tile's first key among the sequence's own; of a key in front: negative
            int const fronts = (int)((p.front + BK - 1) / BK * BK);
            int       key0 = (int)(first_tile_of<OVH>(w.j) * BK) - fronts;
#pragma unroll 1
            for (uint32_t u = 0; u < n_tiles; ++u) {
                asm volatile("cp.async.wait_group %0;" ::"n"(MMA_STAGES - 2) : "memory");
                __syncwarp(); // the other lanes' copies too; and the stage that issue() fills next has been read
                if (u == 0) {
                    // B operand of K Q^T: 8 rows x 32 elements a load.  Rows that the item lacks are its last one once more: what
                    // lies in their place is left from other kernels, and would take part in the vote on the maximum
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t const r = min((uint32_t)(nt * 8 + l7), count - 1);
#pragma unroll
                        for (int i = 0; i < KS / 2; ++i) {
                            uint32_t t[4];
                            ldm4<0>(st + 2 * TILE + r * ROW + (((i * 4 + mi) ^ (r & 7)) << 4), t);
                            q[nt][2 * i][0] = t[0];
                            q[nt][2 * i][1] = t[1];
                            q[nt][2 * i + 1][0] = t[2];
                            q[nt][2 * i + 1][1] = t[3];
                        }
                    }
                }
                issue();
                // (elements between the head dim and DPAD are zeros in shared memory)
                float s[NT][2][4] = {}; // two chains of products
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t a[4];
                    if (i < 4) ldm4<0>(st + kx[i & 3], a);
                    else ldm4<128>(st + kx[i & 3], a);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][i & 1], a, q[nt][i][0], q[nt][i][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][0][i] += s[nt][1][i];
                int const limit = (int)p.front - fronts; // keys in front end here
                if (key0 < 0 ? key0 + BK > limit : key0 + BK > vis_all) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (key0 + g + 8 * (i >> 1) >= (key0 < 0 ? limit : vis[nt][i & 1])) s[nt][0][i] = -INFINITY; // (the scale is positive)
                }
                key0 += BK;
                bool over = false; // a score beyond the running maximum
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[nt][1][i] = fmaf(s[nt][0][i] - m[nt][i & 1], p.scale_log2, MMA_LIFT);
                        over |= s[nt][1][i] > MMA_LIFT + MMA_RESCALE;
                    }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float mx = fmaxf(s[nt][0][x], s[nt][0][2 + x]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                            float const mn = fmaxf(m[nt][x], mx);
                            float const a = ex2((m[nt][x] - mn) * p.scale_log2);
                            m[nt][x] = mn;
                            l[nt][x] *= a;
#pragma unroll
                            for (int i = 0; i < KS; ++i) {
                                o[nt][i][x] *= a;
                                o[nt][i][2 + x] *= a;
                            }
                            s[nt][1][x] = fmaf(s[nt][0][x] - mn, p.scale_log2, MMA_LIFT);
                            s[nt][1][2 + x] = fmaf(s[nt][0][2 + x] - mn, p.scale_log2, MMA_LIFT);
                        }
                }
                uint32_t b[NT][2], low[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = ex2(s[nt][1][i]);
                    l[nt][0] += e[0] + e[2]; // (the sum of the unrounded ones)
                    l[nt][1] += e[1] + e[3];
                    // P as the sum of two f16: its rounding alone would cost as much as that of the result, and the matrix
                    // units have time
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        uint32_t const hi = pack_h2(e[2 * x], e[2 * x + 1]);
                        float2 const   f = __half22float2(*reinterpret_cast<__half2 const*>(&hi));
                        b[nt][x] = transpose8x8(hi);
                        low[nt][x] = transpose8x8(pack_h2(e[2 * x] - f.x, e[2 * x + 1] - f.y));
                    }
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t a[4];
                    if (i < 4) ldm4t<0>(st + vx[i & 3], a);
                    else ldm4t<128>(st + vx[i & 3], a);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(o[nt][i], a, b[nt][0], b[nt][1]);
                        mma16816(o[nt][i], a, low[nt][0], low[nt][1]);
                    }
                }
                st = st + stage_bytes == ring_end ? ring : st + stage_bytes;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) // what the sums are relative to, in log2 units
#pragma unroll
                for (int x = 0; x < 2; ++x) m[nt][x] = fmaf(m[nt][x], p.scale_log2, -MMA_LIFT);
            if (p.direct == DIRECT_BLOCK) { // into this warp's ring, which is done with: maxima and sums, then the rows
                __syncwarp();
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], d);
                        uint32_t const r = nt * 8 + t4 * 2 + x;
                        float* const   mine = reinterpret_cast<float*>(smem_mma + warp * MMA_STAGES * stage_bytes);
                        if (g == 0) {
                            mine[2 * r] = m[nt][x];
                            mine[2 * r + 1] = l[nt][x];
                        }
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            mine[2 * TR + r * DPAD + i * 16 + g] = o[nt][i][x];
                            mine[2 * TR + r * DPAD + i * 16 + g + 8] = o[nt][i][2 + x];
                        }
                    }
                break;
            }
            int const to = segment_slot(w, n_units);
            if (BASE && to < 0) wait_for_base(p);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], d);
                    uint32_t const r = nt * 8 + t4 * 2 + x;
                    if (r >= count) continue;
                    if (to < 0) {
                        uint32_t const pr = start + r, tok = fdivide(pr, p.grp);
                        uint64_t const at = (uint64_t)(w.s.row0 + (int)tok) * p.heads + w.head * p.group + (pr - tok * p.group);
                        // the prefix's row comes beside its weight, not behind it (250 sequences x 32 heads, 8000 items of 4 tiles:
                        // 71 -> 65 us; fetched a tile earlier: 66, and a batch of 64 then took 19 instead of 15); with 16 rows a
                        // tile there is no room for it
                        float bases[2 * KS];
                        if (BASE && NT == 1) {
                            float const* base = p.base_out + at * p.d + g;
#pragma unroll
                            for (int i = 0; i < 2 * KS; ++i) bases[i] = i * 8 < p.d - g ? base[i * 8] : 0.f;
                        }
                        finish_t const f = finish(m[nt][x], l[nt][x], BASE, BASE ? p.base_lse[at] : 0.f);
                        if (p.lse && g == 0) p.lse[at] = f.lse;
                        if (f.wa == 0.f) { // the sum may be anything
#pragma unroll
                            for (int i = 0; i < KS; ++i) o[nt][i][x] = o[nt][i][2 + x] = 0.f;
                        }
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            o[nt][i][x] *= f.wa;
                            o[nt][i][2 + x] *= f.wa;
                        }
                        if (BASE && NT == 1 && f.wb != 0.f) {
#pragma unroll
                            for (int i = 0; i < KS; ++i) {
                                o[nt][i][x] = fmaf(bases[2 * i], f.wb, o[nt][i][x]);
                                o[nt][i][2 + x] = fmaf(bases[2 * i + 1], f.wb, o[nt][i][2 + x]);
                            }
                        }
                        if (BASE && NT > 1 && f.wb != 0.f) {
                            float const* base = p.base_out + at * p.d + g;
#pragma unroll
                            for (int i = 0; i < KS; ++i) {
                                if (i * 16 < p.d - g) o[nt][i][x] = fmaf(base[i * 16], f.wb, o[nt][i][x]);
                                if (i * 16 + 8 < p.d - g) o[nt][i][2 + x] = fmaf(base[i * 16 + 8], f.wb, o[nt][i][2 + x]);
                            }
                        }
                        if (p.out_f32) {
                            float* dst = static_cast<float*>(p.out) + at * p.d + g;
#pragma unroll
                            for (int i = 0; i < KS; ++i) {
                                if (i * 16 < p.d - g) dst[i * 16] = o[nt][i][x];
                                if (i * 16 + 8 < p.d - g) dst[i * 16 + 8] = o[nt][i][2 + x];
                            }
                        }
                    } else {
                        uint64_t const at = (uint64_t)(2 * w.worker + to) * TR + r;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            p.part_out[at * p.part_d + i * 16 + g] = o[nt][i][x];
                            p.part_out[at * p.part_d + i * 16 + g + 8] = o[nt][i][2 + x];
                        }
                        if (g == 0) p.part_ml[at] = make_float2(m[nt][x], l[nt][x]);
                    }
                }
                if (to < 0 && !p.out_f32) { // transposed back: row g, elements 2 t4 and 2 t4 + 1 of each 8
                    uint32_t const r = nt * 8 + g, pr = start + min(r, count - 1), tok = fdivide(pr, p.grp);
                    __half* const  dst = static_cast<__half*>(p.out) + (int64_t)(w.s.row0 + (int)tok) * p.out_stride[0] +
                                        (int64_t)(w.head * p.group + (pr - tok * p.group)) * p.out_stride[1] + t4 * 2;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        uint32_t const y0 = transpose8x8(pack_h2(o[nt][i][0], o[nt][i][1]));
                        uint32_t const y1 = transpose8x8(pack_h2(o[nt][i][2], o[nt][i][3]));
                        if (r < count && (uint32_t)i * 16 < p.d) *reinterpret_cast<uint32_t*>(dst + i * 16) = y0;
                        if (r < count && (uint32_t)i * 16 + 8 < p.d) *reinterpret_cast<uint32_t*>(dst + i * 16 + 8) = y1;
                    }
                }
            }
            if (to == 1) {
                split = true;
                if (lane == 0) write_meta<TR>(p, w, true);
            }
            next_item<TR, BK, OVH>(p, w, n_units);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (p.direct == DIRECT_BLOCK && w.s.n > 0) { // (the same in the whole block)
        if (w.left == 0 && lane < TR) { // no tile for this warp: nothing to add (its rows stay unread)
            float* const mine = reinterpret_cast<float*>(smem_mma + warp * MMA_STAGES * stage_bytes);
            mine[2 * lane] = MMA_NO_KEY;
            mine[2 * lane + 1] = 0.f;
        }
        if (BASE) wait_for_base(p);
        __syncthreads();
        uint32_t const start = w.t * TR, count = min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
        for (uint32_t i = threadIdx.x; i < count * (DPAD / 2); i += THREADS) { // two elements of a row
            uint32_t const r = i / (DPAD / 2), e = i % (DPAD / 2) * 2;
            auto           of = [&](int x) { return reinterpret_cast<float const*>(smem_mma + x * MMA_STAGES * stage_bytes); };
            float          top = -INFINITY, l = 0.f, v[2] = {0.f, 0.f};
#pragma unroll
            for (int x = 0; x < MMA_WARPS; ++x)
                if (of(x)[2 * r + 1] != 0.f) top = fmaxf(top, of(x)[2 * r]);
#pragma unroll
            for (int x = 0; x < MMA_WARPS; ++x) {
                float const lx = of(x)[2 * r + 1];
                if (lx == 0.f) continue;
                float const  wgt = ex2(of(x)[2 * r] - (top == -INFINITY ? 0.f : top));
                float2 const y = *reinterpret_cast<float2 const*>(of(x) + 2 * TR + r * DPAD + e);
                l = fmaf(lx, wgt, l);
                v[0] = fmaf(y.x, wgt, v[0]);
                v[1] = fmaf(y.y, wgt, v[1]);
            }
            uint32_t const pr = start + r, tok = fdivide(pr, p.grp);
            int const      row = w.s.row0 + (int)tok;
            uint32_t const head = w.head * p.group + (pr - tok * p.group);
            uint64_t const at = (uint64_t)row * p.heads + head;
            finish_t const f = finish(top, l, BASE, BASE ? p.base_lse[at] : 0.f);
            if (e < p.d) write_out<__half, 2>(p, row, head, e, v, f, true);
            if (e == 0 && p.lse) p.lse[at] = f.lse;
        }
    }
    if (!split && !p.direct && lane == 0) write_meta<TR>(p, w, false);
    wait_for_base(p);
}

} // namespace
} // namespace es
