// New tokens into a paged cache: keys rotated by their positions, values copied, queries rotated.
//
//   p = L_i - n_i + r,   (x, y)_j <- (x cos - y sin, x sin + y cos)_j with angle table entry f[p + offset, j]
//   K[table_i[p / page], p % page] <- rotated k_r,   V[...] <- v_r,   q_out_r <- rotated q_r
//
// Bound: memory (each element is read and written once; 3 flops an element).  One thread moves 8
// elements of a head (16 bytes of f16), or 2 + 2 runs of 4 that belong together when a pair's members are
// half a head apart; neighbouring threads on neighbouring elements.  A block takes a token's whole row of
// heads at a time, so that the token's sequence, page and angles are found once a block: the sequence by
// counting, with all threads at once, how many sequences end at or before the row (one round of loads, not a
// chain of log2(batch) dependent ones).
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "paged.h"
#include "paged_device.h"
#include "pdl.h"

namespace es {

namespace {

__device__ unsigned int g_append_error;

struct append_params_t {
    void const*    q;
    void const*    k;
    void const*    v;
    float const*   freqs;
    void*          q_out;
    void*          k_cache;
    void*          v_cache;
    int32_t const* row_offsets;
    int32_t const* lengths;
    int32_t const* tables;
    int64_t        q_stride[2], k_stride[2], v_stride[2], q_out_stride[2], kc_stride[3], vc_stride[3];
    int64_t        pos_offset;
    uint64_t       n_positions;
    uint32_t       batch, rows, heads, kv_heads, d, rot, n_pages, table_stride, capacity;
    uint32_t       units_per_head; // threads a head
    fastdiv_t      page, upd; // page_size; units per head
};

template <typename T, int N> struct vec_t;
template <> struct alignas(16) vec_t<__half, 8> { __half v[8]; };
template <> struct alignas(8) vec_t<__half, 4> { __half v[4]; };
template <> struct alignas(16) vec_t<float, 4> { float v[4]; };

// N consecutive elements as f32; N = 8 or 4 with VEC (16-byte aligned rows), else one by one up to `n`
template <int N, bool VEC, typename T> __device__ __forceinline__ void load_n(T const* p, float (&x)[N], int n)
{
    if constexpr (VEC && sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            vec_t<float, 4> t = *reinterpret_cast<vec_t<float, 4> const*>(p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i + j] = t.v[j];
        }
    } else if constexpr (VEC) {
        vec_t<__half, N> t = *reinterpret_cast<vec_t<__half, N> const*>(p);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = __half2float(t.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = j < n ? to_f32(p[j]) : 0.f;
    }
}

template <int N, bool VEC, typename T> __device__ __forceinline__ void store_n(T* p, float const (&x)[N], int n)
{
    if constexpr (VEC && sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            vec_t<float, 4> t;
#pragma unroll
            for (int j = 0; j < 4; ++j) t.v[j] = x[i + j];
            *reinterpret_cast<vec_t<float, 4>*>(p + i) = t;
        }
    } else if constexpr (VEC) {
        vec_t<__half, N> t;
#pragma unroll
        for (int j = 0; j < N; ++j) t.v[j] = __float2half_rn(x[j]);
        *reinterpret_cast<vec_t<__half, N>*>(p) = t;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) from_f32(p[j], x[j]);
    }
}

// One unit of a head: adjacent pairs: 8 elements from 8u on.  Halves: unit u of the first rot / 8 ones holds
// elements 4u.. and rot/2 + 4u.., the units behind them 8 elements each from `rot` on.
template <typename TI, typename TC, bool HALVES, bool VEC>
__device__ __forceinline__ void move_unit(TI const* src, TC* dst, uint32_t u, uint32_t d, uint32_t rot, float const* f)
{
    if constexpr (HALVES) {
        uint32_t const half = rot / 2, n_rot = (half + 3) / 4;
        if (u < n_rot) {
            uint32_t const e = 4 * u;
            int const      n = min(4, (int)(half - e));
            float          a[4], b[4], c[8];
            load_n<4, VEC>(src + e, a, n);
            load_n<4, VEC>(src + half + e, b, n);
            load_n<8, VEC>(f + 2 * e, c, 2 * n);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float const x = a[j], y = b[j];
                a[j] = x * c[2 * j] - y * c[2 * j + 1];
                b[j] = x * c[2 * j + 1] + y * c[2 * j];
            }
            store_n<4, VEC>(dst + e, a, n);
            store_n<4, VEC>(dst + half + e, b, n);
        } else {
            uint32_t const e = rot + 8 * (u - n_rot);
            int const      n = min(8, (int)(d - e));
            float          x[8];
            load_n<8, VEC>(src + e, x, n);
            store_n<8, VEC>(dst + e, x, n);
        }
    } else {
        uint32_t const e = 8 * u;
        int const      n = min(8, (int)(d - e));
        float          x[8], c[8];
        load_n<8, VEC>(src + e, x, n);
        if (e < rot) {
            int const nr = min(n, (int)(rot - e)); // even
            if (VEC && nr == 8) {
                load_n<8, true>(f + e, c, 8);
            } else {
                load_n<8, false>(f + e, c, nr);
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                if (j < nr) {
                    float const a = x[j], b = x[j + 1];
                    x[j] = a * c[j] - b * c[j + 1];
                    x[j + 1] = a * c[j + 1] + b * c[j];
                }
            }
        }
        store_n<8, VEC>(dst + e, x, n);
    }
}

template <typename TI, typename TC, bool HALVES, bool VEC>
__global__ void __launch_bounds__(256) cache_append_kernel(const __grid_constant__ append_params_t p)
{
    ES_PDL_PROLOGUE();
    uint32_t const n_heads = p.heads + 2 * p.kv_heads;
    uint32_t const units = n_heads * p.units_per_head;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        // the row's sequence and position
        int  seq = (int)row;
        int  back = 1; // rows from this one to the end of its sequence
        bool used = true;
        if (p.row_offsets) {
            int below = 0; // sequences that end at or before this row
            for (uint32_t i0 = 0; i0 < p.batch; i0 += blockDim.x) {
                uint32_t const i = i0 + threadIdx.x;
                below += __syncthreads_count(i < p.batch && p.row_offsets[i + 1] <= (int)row);
            }
            seq = below;
            used = seq < (int)p.batch;
            if (used) {
                int const a = p.row_offsets[seq], b = p.row_offsets[seq + 1];
                back = b - (int)row;
                if (a < 0 || a > (int)row || back <= 0 || b > (int)p.rows) { // offsets that fall, or pass the rows
                    if (threadIdx.x == 0) atomicCAS(&g_append_error, 0u, (unsigned)PAGED_BAD_ROWS);
                    used = false;
                }
            }
        }
        if (!used) continue; // (uniform in the block, as is every branch up to the units)
        int const length = p.lengths[seq];
        if (length < 0 || (uint32_t)length > p.capacity) {
            if (threadIdx.x == 0) atomicCAS(&g_append_error, 0u, (unsigned)PAGED_BAD_LENGTH);
            continue;
        }
        int const pos = length - back;
        if (pos < 0) continue; // no place in the cache
        uint32_t const pi = fdivide((uint32_t)pos, p.page);
        uint32_t const slot = (uint32_t)pos - pi * p.page.d;
        uint32_t const page = (uint32_t)p.tables[(uint64_t)seq * p.table_stride + pi];
        uint64_t const angle = (uint64_t)(pos + p.pos_offset);
        bool const     page_ok = page < p.n_pages, angle_ok = p.rot == 0 || angle < p.n_positions;
        if (threadIdx.x == 0 && !page_ok) atomicCAS(&g_append_error, 0u, (unsigned)PAGED_BAD_PAGE);
        if (threadIdx.x == 0 && !angle_ok) atomicCAS(&g_append_error, 0u, (unsigned)PAGED_BAD_POSITION);
        if (!angle_ok) continue;
        float const* f = p.freqs + angle * p.rot; // rot / 2 pairs of floats
        TC* const    kc = static_cast<TC*>(p.k_cache) + (int64_t)page * p.kc_stride[0] + (int64_t)slot * p.kc_stride[1];
        TC* const    vc = static_cast<TC*>(p.v_cache) + (int64_t)page * p.vc_stride[0] + (int64_t)slot * p.vc_stride[1];
        // blockIdx.y shares out a row's units when there are few rows
        for (uint32_t w = blockIdx.y * blockDim.x + threadIdx.x; w < units; w += gridDim.y * blockDim.x) {
            uint32_t const head = fdivide(w, p.upd);
            uint32_t const u = w - head * p.units_per_head;
            if (head < p.heads) {
                move_unit<TI, TC, HALVES, VEC>(
                    static_cast<TI const*>(p.q) + (int64_t)row * p.q_stride[0] + (int64_t)head * p.q_stride[1],
                    static_cast<TC*>(p.q_out) + (int64_t)row * p.q_out_stride[0] + (int64_t)head * p.q_out_stride[1], u, p.d,
                    p.rot, f);
            } else if (page_ok) {
                uint32_t const hk = head - p.heads;
                if (hk < p.kv_heads) {
                    move_unit<TI, TC, HALVES, VEC>(
                        static_cast<TI const*>(p.k) + (int64_t)row * p.k_stride[0] + (int64_t)hk * p.k_stride[1],
                        kc + (int64_t)hk * p.kc_stride[2], u, p.d, p.rot, f);
                } else {
                    uint32_t const hv = hk - p.kv_heads;
                    // values are not rotated: with halves the unit's two runs are moved as they are
                    TI const* src = static_cast<TI const*>(p.v) + (int64_t)row * p.v_stride[0] + (int64_t)hv * p.v_stride[1];
                    TC*       dst = vc + (int64_t)hv * p.vc_stride[2];
                    uint32_t const e = 8 * u;
                    if (e < p.d) {
                        float     x[8];
                        int const n = min(8, (int)(p.d - e));
                        load_n<8, VEC>(src + e, x, n);
                        store_n<8, VEC>(dst + e, x, n);
                    }
                }
            }
        }
    }
}

} // namespace

void check_cache_append(es_cache_append_t const& a, es_cache_append_args_t const& x)
{
    check_paged_cache(a.cache, "cache append");
    if (a.in_dtype != ES_F16 && a.in_dtype != ES_F32) fail(ES_NOT_SUPPORTED, "cache append: rows must be f16 or f32");
    if (!x.k || !x.v || !x.k_cache || !x.v_cache || !x.lengths || !x.tables) fail(ES_BAD_ARGUMENT, "cache append: null pointer");
    if (a.heads && (!x.q || !x.q_out)) fail(ES_BAD_ARGUMENT, "cache append: null query pointer");
    if (a.heads > 65535) fail(ES_NOT_SUPPORTED, "cache append: more than 65535 heads");
    if (a.rotary_dim % 2 || a.rotary_dim > a.cache.head_dim)
        fail(ES_BAD_DESCRIPTOR, "cache append: the rotated part of a head must be even and at most the head dim");
    if (a.rotary_dim && (!x.freqs || a.n_positions == 0)) fail(ES_BAD_ARGUMENT, "cache append: no table of angles");
    if (a.pairing != ES_ROPE_ADJACENT && a.pairing != ES_ROPE_HALVES) fail(ES_BAD_DESCRIPTOR, "cache append: unknown pairing");
    if (a.pos_offset < 0) fail(ES_BAD_DESCRIPTOR, "cache append: negative position offset");
    if (!x.row_offsets && a.cache.rows != a.cache.batch)
        fail(ES_BAD_DESCRIPTOR, "cache append: without row offsets there is one row a sequence");
    for (int i = 0; i != 2; ++i)
        if (a.k_stride[i] < 0 || a.v_stride[i] < 0 || (a.heads && (a.q_stride[i] < 0 || a.q_out_stride[i] < 0)))
            fail(ES_BAD_DESCRIPTOR, "cache append: negative stride");
    uintptr_t const ie = dtype_size(a.in_dtype) - 1, ce = dtype_size(a.cache.dtype) - 1;
    if (((reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.k) | reinterpret_cast<uintptr_t>(x.v)) & ie) ||
        ((reinterpret_cast<uintptr_t>(x.q_out) | reinterpret_cast<uintptr_t>(x.k_cache) | reinterpret_cast<uintptr_t>(x.v_cache)) & ce) ||
        ((reinterpret_cast<uintptr_t>(x.freqs) | reinterpret_cast<uintptr_t>(x.row_offsets) | reinterpret_cast<uintptr_t>(x.lengths) |
          reinterpret_cast<uintptr_t>(x.tables)) & 3))
        fail(ES_BAD_ARGUMENT, "cache append: a pointer is not aligned to its elements");
}

int launch_cache_append(es_cache_append_t const& a, es_cache_append_args_t const& x, cudaStream_t stream)
{
    check_cache_append(a, x);
    es_paged_cache_t const& c = a.cache;
    if (c.rows == 0) return 0;
    append_params_t p = {};
    p.q = x.q;
    p.k = x.k;
    p.v = x.v;
    p.freqs = x.freqs;
    p.q_out = x.q_out;
    p.k_cache = x.k_cache;
    p.v_cache = x.v_cache;
    p.row_offsets = x.row_offsets;
    p.lengths = x.lengths;
    p.tables = x.tables;
    for (int i = 0; i != 2; ++i) {
        p.q_stride[i] = a.q_stride[i];
        p.k_stride[i] = a.k_stride[i];
        p.v_stride[i] = a.v_stride[i];
        p.q_out_stride[i] = a.q_out_stride[i];
    }
    for (int i = 0; i != 3; ++i) {
        p.kc_stride[i] = c.k_stride[i];
        p.vc_stride[i] = c.v_stride[i];
    }
    p.pos_offset = a.pos_offset;
    p.n_positions = a.n_positions;
    p.batch = c.batch;
    p.rows = c.rows;
    p.heads = a.heads;
    p.kv_heads = c.kv_heads;
    p.d = c.head_dim;
    p.rot = a.rotary_dim;
    p.n_pages = c.n_pages;
    p.table_stride = c.table_stride;
    p.capacity = paged_capacity(c);
    p.page = make_fastdivide(c.page_size);
    bool const     halves = a.pairing == ES_ROPE_HALVES && a.rotary_dim > 0;
    uint32_t const half = a.rotary_dim / 2;
    // threads a head: adjacent pairs ceil(d / 8); halves: runs of 4 of either half, then 8 of the rest (and at
    // least ceil(d / 8) for the values)
    p.units_per_head = halves ? std::max((half + 3) / 4 + (c.head_dim - a.rotary_dim + 7) / 8, (c.head_dim + 7) / 8) : (c.head_dim + 7) / 8;
    p.upd = make_fastdivide(p.units_per_head);
    // 16-byte accesses when every run of 8 (with halves: 4) elements of every head starts on its own size
    uint64_t  bits = reinterpret_cast<uintptr_t>(x.k) | reinterpret_cast<uintptr_t>(x.v) | reinterpret_cast<uintptr_t>(x.k_cache) |
                     reinterpret_cast<uintptr_t>(x.v_cache) | reinterpret_cast<uintptr_t>(x.freqs);
    uint64_t  el = c.head_dim;
    for (int i = 0; i != 2; ++i) el |= (uint64_t)a.k_stride[i] | (uint64_t)a.v_stride[i];
    for (int i = 0; i != 3; ++i) el |= (uint64_t)c.k_stride[i] | (uint64_t)c.v_stride[i];
    if (a.heads) {
        bits |= reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.q_out);
        for (int i = 0; i != 2; ++i) el |= (uint64_t)a.q_stride[i] | (uint64_t)a.q_out_stride[i];
    }
    el |= a.rotary_dim; // a multiple of 8: a row of angles is a multiple of 32 bytes, a half of 4 elements
    bool const vec = (bits & 15) == 0 && (el & 7) == 0;
    // A block a row; when the rows alone would leave SMs empty (under 2 blocks an SM) a row's heads are shared
    // out to up to 16 blocks of fewer threads.
    uint32_t const units = (a.heads + 2 * c.kv_heads) * p.units_per_head;
    uint32_t const want = std::max<uint32_t>(1, (2 * SM_COUNT + c.rows - 1) / c.rows);
    uint32_t       threads = 256;
    while (threads > 64 && (units + threads - 1) / threads < want) threads /= 2;
    uint32_t const gy = std::min<uint32_t>(std::min<uint32_t>(want, 16), (units + threads - 1) / threads);
    dim3 const     grid(std::min<uint32_t>(c.rows, 1u << 20), gy);
    auto           go = [&](auto kernel) { launch_k(kernel, grid, dim3(threads), 0, stream, p); };
    auto           pick = [&](auto ti, auto tc) {
        using TI = decltype(ti);
        using TC = decltype(tc);
        if (vec) {
            if (halves) go(cache_append_kernel<TI, TC, true, true>);
            else go(cache_append_kernel<TI, TC, false, true>);
        } else {
            if (halves) go(cache_append_kernel<TI, TC, true, false>);
            else go(cache_append_kernel<TI, TC, false, false>);
        }
    };
    if (a.in_dtype == ES_F16 && c.dtype == ES_F16) pick(__half(), __half());
    else if (a.in_dtype == ES_F16) pick(__half(), float());
    else if (c.dtype == ES_F16) pick(float(), __half());
    else pick(float(), float());
    return 1;
}

unsigned int read_and_clear_append_error()
{
    unsigned int v = 0, zero = 0;
    ES_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_append_error, sizeof v));
    if (v) ES_CUDA_CHECK(cudaMemcpyToSymbol(g_append_error, &zero, sizeof zero));
    return v;
}

} // namespace es
