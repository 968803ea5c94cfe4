// Paged attention without the tensor cores: f32, and f16 whose strides or head dim the other kernels do not
// take.
//
// 8 lanes hold one key's head dim (4 elements at a time, 32 elements apart); a block's 16 such groups each
// take every 16th key and keep running maxima, sums and results of their own for TR rows, so that nothing is
// exchanged between groups until the segment ends.  The query rows stay in registers, multiplied by
// scale * log2 e.  The next KEYS keys and values are loaded before the current ones are used.  Bound: the latency
// of those loads for short sequences, memory for long ones with up to TR packed rows a key head; beyond that a key
// is read once per TR rows, and the multiply-adds with their shuffles are what it waits for.  TR follows the rows
// there are: 12 sequences of up to 2900 tokens, 4 query heads of 64 a key head, 14.5 MB: 17 us with 8 rows and one
// key at a time, 13 with 4 rows and two keys, 15.6 with the join -- launch, counting and the first loads are most of it.
#pragma once
#include "paged_work.h"

namespace es {
namespace {

constexpr int SIMT_BK = 64, SIMT_OVH = 2;

// 4 elements of type T as f32; vec: one load, else the first n of them one by one
template <typename T> __device__ __forceinline__ void load4(T const* p, float (&x)[4], bool vec, int n)
{
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            float4 const t = *reinterpret_cast<float4 const*>(p);
            x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
        } else {
            uint2 const  t = *reinterpret_cast<uint2 const*>(p);
            float2 const a = __half22float2(*reinterpret_cast<__half2 const*>(&t.x));
            float2 const b = __half22float2(*reinterpret_cast<__half2 const*>(&t.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}

template <typename T, int NCH, int TR, bool VEC> // NCH: chunks of 32 elements of the head dim
__global__ void __launch_bounds__(128) paged_simt_kernel(const __grid_constant__ paged_params_t p)
{
    constexpr int KEYS = NCH * TR <= 8 && NCH <= 4 ? 2 : 1, BK = SIMT_BK, OVH = SIMT_OVH, NT = 128;
    constexpr bool AHEAD = NCH <= 4; // (head dims above 128: no registers for it)
    __shared__ sched_smem_t<NT, 1> sched;
    __shared__ float            so[4][TR][NCH * 32];
    __shared__ float2           sml[4][TR];
    begin_order(p);
    int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, stream = threadIdx.x >> 3;
    work_t    w;
    find_work<TR, BK, OVH, NT, 1>(p, w, sched);
    bool split = false;
    while (w.left) {
        uint32_t const n_units = min(w.kt - w.j, w.left);
        uint32_t const start = w.t * TR;
        int const      count = (int)min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
        float          q[TR][NCH][4], o[TR][NCH][4], m[TR], l[TR];
        int            vis[TR], vis_max = 0;
#pragma unroll
        for (int r = 0; r < TR; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            vis[r] = 0;
            uint32_t const pr = start + r, tok = fdivide(pr, p.grp);
            if (r < count) vis[r] = visible(p, w.s, (int)tok);
            vis_max = max(vis_max, vis[r]);
            T const* src = static_cast<T const*>(p.q) + (int64_t)(w.s.row0 + (int)tok) * p.q_stride[0] +
                           (int64_t)(w.head * p.group + (pr - tok * p.group)) * p.q_stride[1];
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                uint32_t const e = c * 32 + l8 * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) q[r][c][i] = o[r][c][i] = 0.f;
                if (r < count && e < p.d) load4<T>(src + e, q[r][c], VEC, (int)(p.d - e));
#pragma unroll
                for (int i = 0; i < 4; ++i) q[r][c][i] *= p.scale_log2;
            }
        }
        // keys are numbered from the first of those in front on, the sequence's own from `own` on
        int const own = (int)((p.front + BK - 1) / BK * BK);
        int const key_begin = (int)(first_tile_of<OVH>(w.j) * BK);
        int const key_end = (int)min((uint64_t)first_tile_of<OVH>(w.j + n_units) * BK, (uint64_t)own + (uint64_t)vis_max);
        T const*  kb = static_cast<T const*>(p.k) + (int64_t)w.head * p.k_stride[2];
        T const*  vb = static_cast<T const*>(p.v) + (int64_t)w.head * p.v_stride[2];
        auto      load = [&](int key, float (&k)[NCH][4], float (&v)[NCH][4]) -> bool {
            if (key >= key_end || (key < own && key >= (int)p.front)) return false;
            int32_t const* table = key < own ? p.front_pages : w.s.table;
            if (key >= own) key -= own;
            uint32_t const pi = fdivide((uint32_t)key, p.page);
            uint32_t const page = (uint32_t)table[pi];
            if (page >= p.n_pages) {
                report(p, PAGED_BAD_PAGE);
                return false;
            }
            uint32_t const slot = (uint32_t)key - pi * p.page.d;
            T const* const ks = kb + (int64_t)page * p.k_stride[0] + (int64_t)slot * p.k_stride[1];
            T const* const vs = vb + (int64_t)page * p.v_stride[0] + (int64_t)slot * p.v_stride[1];
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                uint32_t const e = c * 32 + l8 * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) k[c][i] = v[c][i] = 0.f;
                if (e < p.d) {
                    load4<T>(ks + e, k[c], VEC, (int)(p.d - e));
                    load4<T>(vs + e, v[c], VEC, (int)(p.d - e));
                }
            }
            return true;
        };
        float     k[KEYS][NCH][4], v[KEYS][NCH][4];
        bool      have[KEYS];
        int const key0 = key_begin + stream;
#pragma unroll
        for (int x = 0; x < KEYS; ++x) have[x] = load(key0 + x * 16, k[x], v[x]);
        // (every group of the warp makes the same number of rounds: the shuffles are the warp's)
        int const rounds = key_end > key_begin ? (key_end - key_begin + 16 * KEYS - 1) / (16 * KEYS) : 0;
        for (int i = 0; i < rounds; ++i) {
            int const key = key0 + i * 16 * KEYS;
            float     kn[KEYS][NCH][4], vn[KEYS][NCH][4];
            bool      next[KEYS];
#pragma unroll
            for (int x = 0; x < KEYS; ++x) next[x] = AHEAD && i + 1 < rounds && load(key + (KEYS + x) * 16, kn[x], vn[x]);
#pragma unroll
            for (int r = 0; r < TR; ++r) {
                float s[KEYS];
#pragma unroll
                for (int x = 0; x < KEYS; ++x) {
                    s[x] = 0.f;
#pragma unroll
                    for (int c = 0; c < NCH; ++c)
#pragma unroll
                        for (int y = 0; y < 4; ++y) s[x] = fmaf(q[r][c][y], k[x][c][y], s[x]);
                }
#pragma unroll
                for (int d = 4; d; d >>= 1)
#pragma unroll
                    for (int x = 0; x < KEYS; ++x) s[x] += __shfl_xor_sync(0xffffffffu, s[x], d);
#pragma unroll
                for (int x = 0; x < KEYS; ++x) {
                    if (have[x] && key + x * 16 - own < vis[r]) {
                        if (s[x] > m[r]) {
                            float const a = ex2(m[r] - s[x]); // m = -inf: 0
                            m[r] = s[x];
                            l[r] *= a;
#pragma unroll
                            for (int c = 0; c < NCH; ++c)
#pragma unroll
                                for (int y = 0; y < 4; ++y) o[r][c][y] *= a;
                        }
                        float const e = ex2(s[x] - (m[r] == -INFINITY ? 0.f : m[r]));
                        l[r] += e;
#pragma unroll
                        for (int c = 0; c < NCH; ++c)
#pragma unroll
                            for (int y = 0; y < 4; ++y) o[r][c][y] = fmaf(e, v[x][c][y], o[r][c][y]);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < KEYS; ++x) {
                if constexpr (AHEAD) {
                    have[x] = next[x];
#pragma unroll
                    for (int c = 0; c < NCH; ++c)
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            k[x][c][y] = kn[x][c][y];
                            v[x][c][y] = vn[x][c][y];
                        }
                } else {
                    have[x] = i + 1 < rounds && load(key + (KEYS + x) * 16, k[x], v[x]);
                }
            }
        }
        // the warp's four groups
#pragma unroll
        for (int r = 0; r < TR; ++r) {
#pragma unroll
            for (int x = 8; x <= 16; x <<= 1) {
                float const mo = __shfl_xor_sync(0xffffffffu, m[r], x), lo = __shfl_xor_sync(0xffffffffu, l[r], x);
                float const mn = fmaxf(m[r], mo);
                float const a = m[r] == -INFINITY ? (l[r] == 0.f ? 0.f : 1.f) : ex2(m[r] - mn);
                float const b = mo == -INFINITY ? (lo == 0.f ? 0.f : 1.f) : ex2(mo - mn);
                l[r] = l[r] * a + lo * b;
#pragma unroll
                for (int c = 0; c < NCH; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float const oo = __shfl_xor_sync(0xffffffffu, o[r][c][i], x);
                        o[r][c][i] = o[r][c][i] * a + oo * b;
                    }
                m[r] = mn;
            }
            if (lane < 8) {
#pragma unroll
                for (int c = 0; c < NCH; ++c)
                    *reinterpret_cast<float4*>(&so[warp][r][c * 32 + l8 * 4]) = make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]);
                if (l8 == 0) sml[warp][r] = make_float2(m[r], l[r]);
            }
        }
        __syncthreads();
        int const slot = segment_slot(w, n_units);
        if (slot < 0 && p.base_out) wait_for_base(p);
        // the four warps' results; a thread 4 elements of a row
        for (int x = threadIdx.x; x < count * NCH * 8; x += NT) {
            int const      r = x / (NCH * 8);
            uint32_t const e = (uint32_t)(x % (NCH * 8)) * 4;
            float          top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sml[i][r].y != 0.f) top = fmaxf(top, sml[i][r].x);
            float sum[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 const ml = sml[i][r];
                if (ml.y == 0.f) continue;
                float const wgt = ex2(ml.x - (top == -INFINITY ? 0.f : top));
                float4 const a = *reinterpret_cast<float4 const*>(&so[i][r][e]);
                ls = fmaf(ml.y, wgt, ls);
                sum[0] = fmaf(a.x, wgt, sum[0]);
                sum[1] = fmaf(a.y, wgt, sum[1]);
                sum[2] = fmaf(a.z, wgt, sum[2]);
                sum[3] = fmaf(a.w, wgt, sum[3]);
            }
            if (slot < 0) {
                uint32_t const pr = start + r, tok = fdivide(pr, p.grp);
                int const      row = w.s.row0 + (int)tok;
                uint32_t const head = w.head * p.group + (pr - tok * p.group);
                uint64_t const at = (uint64_t)row * p.heads + head;
                finish_t const f = finish(top, ls, p.base_lse != nullptr, p.base_lse ? p.base_lse[at] : 0.f);
                if (e < p.d) write_out<T, 4>(p, row, head, e, sum, f, VEC);
                if (e == 0 && p.lse) p.lse[at] = f.lse;
            } else {
                uint64_t const at = (uint64_t)(2 * blockIdx.x + slot) * TR + r;
                *reinterpret_cast<float4*>(p.part_out + at * p.part_d + e) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                if (e == 0) p.part_ml[at] = make_float2(top, ls);
            }
        }
        __syncthreads();
        if (slot == 1) {
            split = true;
            if (threadIdx.x == 0) write_meta<TR>(p, w, true);
        }
        next_item<TR, BK, OVH>(p, w, n_units);
    }
    if (!split && !p.direct && threadIdx.x == 0) write_meta<TR>(p, w, false);
    wait_for_base(p);
}

} // namespace
} // namespace es
