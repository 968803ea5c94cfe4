// New tokens into a paged cache: keys rotated by their positions, values copied, queries rotated.
//
//   p = L_i - n_i + r,   (x, y)_j <- (x cos - y sin, x sin + y cos)_j with angle table entry f[p + offset, j]
//   K[table_i[p / page], p % page] <- rotated k_r,   V[...] <- v_r,   q_out_r <- rotated q_r
//
// Bound: memory (each element is read and written once; 3 flops an element), and close behind it the number of
// instructions a move takes.  A thread moves 8 elements of a head -- 16 bytes of f16, or 2 runs of 4 when a pair's
// members are half a head apart.  A block moves one of the three tensors, so that nothing about a move is decided by
// thread, for several rows: what a row needs to know first is a chain of loads -- its sequence (found by counting, a
// lane a sequence, how many end at or before the row), the sequence's length, the page -- and a block's warps find
// the places of all its rows before it moves them.  Moves are short chains of loads, so warps count: 40 an SM.  The
// blocks make one wave.  Measured: 7311 rows of 32 + 64 heads of 128, f16 (361 MB) 70 us = 5.1 TB/s (a row a block, its
// places found by every block for itself: 75 us; six heads of a thread at once: 97, with half the warps); a row of
// one sequence 3 us.
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
    fastdiv_t      page, upd, by_heads[2]; // page_size; units a head; heads of the queries, of keys and values
    uint32_t       first_block[2], rows_a_block[2];
};

template <typename T, int N> struct vec_t;
template <> struct alignas(16) vec_t<__half, 8> { __half v[8]; };
template <> struct alignas(8) vec_t<__half, 4> { __half v[4]; };
template <> struct alignas(16) vec_t<float, 4> { float v[4]; };

// 8 consecutive floats, 16-byte aligned
__device__ __forceinline__ void load_8(float const* p, float (&x)[8])
{
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        vec_t<float, 4> const t = *reinterpret_cast<vec_t<float, 4> const*>(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i + j] = t.v[j];
    }
}

// N consecutive elements from f32; N = 8 or 4 with VEC (aligned to their size, at most 16 bytes), else one by one up to `n`
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

// The 8 elements of unit u of a head.  Adjacent pairs: from 8u on.  Halves: unit u of the first ceil(rot / 8)
// holds 4u.. and rot / 2 + 4u.., the units behind them 8 elements each from `rot` on.
struct unit_t {
    uint32_t e0, e1; // where its two runs of 4 begin (one run of 8: e1 = e0 + 4)
    int      n0, n1; // elements of each that exist
    bool     rotated;
};
template <bool HALVES> __device__ __forceinline__ unit_t unit_of(uint32_t u, uint32_t d, uint32_t rot)
{
    unit_t         t;
    uint32_t const half = rot / 2, n_rot = (half + 3) / 4;
    if (HALVES && u < n_rot) {
        t.e0 = 4 * u;
        t.e1 = half + 4 * u;
        t.n0 = t.n1 = min(4, (int)(half - t.e0));
        t.rotated = true;
    } else {
        t.e0 = HALVES ? rot + 8 * (u - n_rot) : 8 * u;
        t.e1 = t.e0 + 4;
        t.n0 = min(4, (int)d - (int)t.e0);
        t.n1 = min(4, (int)d - (int)t.e1);
        t.rotated = !HALVES && t.e0 < rot;
    }
    return t;
}

// (as they lie in memory: converted when their turn comes)
template <typename T> struct alignas(16) raw_t {
    T v[8];
};
template <bool HALVES, bool VEC, typename T> __device__ __forceinline__ void load_unit(T const* p, unit_t const& t, raw_t<T>& x)
{
    if constexpr (VEC && !HALVES) {
        x = *reinterpret_cast<raw_t<T> const*>(p + t.e0);
    } else if constexpr (VEC) {
        *reinterpret_cast<vec_t<T, 4>*>(&x.v[0]) = *reinterpret_cast<vec_t<T, 4> const*>(p + t.e0);
        *reinterpret_cast<vec_t<T, 4>*>(&x.v[4]) = *reinterpret_cast<vec_t<T, 4> const*>(p + t.e1);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < t.n0) x.v[j] = p[t.e0 + j];
            if (j < t.n1) x.v[4 + j] = p[t.e1 + j];
        }
    }
}
template <bool HALVES, bool VEC, typename T> __device__ __forceinline__ void store_unit(T* p, unit_t const& t, float const (&x)[8])
{
    if constexpr (VEC && !HALVES) {
        store_n<8, true>(p + t.e0, x, 8);
    } else {
        float const a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
        store_n<4, VEC>(p + t.e0, a, t.n0);
        store_n<4, VEC>(p + t.e1, b, t.n1);
    }
}
// c: cosine and sine of the unit's four pairs, of which the first n are rotated
template <bool HALVES> __device__ __forceinline__ void rotate(float (&x)[8], float const (&c)[8], int n)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j >= n) break; // (by a factor of 1 + 0 i an infinity would become its neighbour's NaN)
        int const   i0 = HALVES ? j : 2 * j, i1 = HALVES ? 4 + j : 2 * j + 1;
        float const a = x[i0], b = x[i1];
        x[i0] = a * c[2 * j] - b * c[2 * j + 1];
        x[i1] = a * c[2 * j + 1] + b * c[2 * j];
    }
}

constexpr uint32_t ROWS_MAX = 64, APPEND_THREADS = 256;
constexpr uint32_t blocks_an_sm(bool f16_rows) { return f16_rows ? 5 : 3; } // (what their registers leave room for)

struct place_t { // of a row, in one tensor
    int64_t to;    // element of the tensor written to, without the head; < 0: the row is not moved
    int64_t angle; // element of the table of angles
};

// (what: 0 queries, 1 keys, 2 values; all lanes of a warp call)
__device__ __forceinline__ place_t find_place(append_params_t const& p, uint32_t row, int what)
{
    place_t   t = {-1, 0};
    int const lane = threadIdx.x & 31;
    auto      report = [&](unsigned code) {
        if (lane == 0) atomicCAS(&g_append_error, 0u, code);
        return t;
    };
    int seq = (int)row, back = 1; // rows from this one to the end of its sequence
    if (p.row_offsets) {
        seq = 0; // sequences that end at or before this row
        for (uint32_t i0 = 0; i0 < p.batch; i0 += 32)
            seq += __popc(__ballot_sync(0xffffffffu, i0 + lane < p.batch && p.row_offsets[i0 + lane + 1] <= (int)row));
        if (seq >= (int)p.batch) return t; // padding
        int  a = p.row_offsets[seq], b = p.row_offsets[seq + 1];
        auto holds = [&] { return a >= 0 && a <= (int)row && b > (int)row && b <= (int)p.rows; };
        if (!holds()) { // offsets that fall, or pass the rows: the first sequence that holds the row nonetheless
            report(PAGED_BAD_ROWS);
            seq = -1;
            for (uint32_t i0 = 0; i0 < p.batch && seq < 0; i0 += 32) {
                if (i0 + lane < p.batch) a = p.row_offsets[i0 + lane], b = p.row_offsets[i0 + lane + 1];
                seq = __ffs(__ballot_sync(0xffffffffu, i0 + lane < p.batch && holds())) - 1;
                if (seq >= 0) seq += (int)i0;
            }
            if (seq < 0) return t;
            b = p.row_offsets[seq + 1];
        }
        back = b - (int)row;
    }
    int const length = p.lengths[seq];
    if (length < 0 || (uint32_t)length > p.capacity) return report(PAGED_BAD_LENGTH);
    int const pos = length - back;
    if (pos < 0) return t; // no place in the cache
    uint64_t const angle = (uint64_t)(pos + p.pos_offset);
    if (p.rot && angle >= p.n_positions) return report(PAGED_BAD_POSITION);
    t.angle = (int64_t)(angle * p.rot);
    if (what == 0) {
        t.to = (int64_t)row * p.q_out_stride[0];
        return t;
    }
    uint32_t const pi = fdivide((uint32_t)pos, p.page);
    uint32_t const slot = (uint32_t)pos - pi * p.page.d;
    uint32_t const page = (uint32_t)p.tables[(uint64_t)seq * p.table_stride + pi];
    if (page >= p.n_pages) return report(PAGED_BAD_PAGE);
    int64_t const* so = what == 1 ? p.kc_stride : p.vc_stride;
    t.to = (int64_t)page * so[0] + (int64_t)slot * so[1];
    return t;
}

// Blocks [0, first_block[0]) move queries, [.., first_block[1]) keys, the others values, rows_a_block[.] rows each.
// A thread keeps its unit and steps through heads and rows by adding strides.
template <typename TI, typename TC, bool HALVES, bool VEC>
__global__ void __launch_bounds__(APPEND_THREADS, blocks_an_sm(sizeof(TI) == 2 && VEC)) cache_append_kernel(const __grid_constant__ append_params_t p)
{
    __shared__ place_t places[ROWS_MAX];
    ES_PDL_PROLOGUE();
    int const      what = blockIdx.x < p.first_block[0] ? 0 : blockIdx.x < p.first_block[1] ? 1 : 2;
    uint32_t const block = blockIdx.x - (what ? p.first_block[what - 1] : 0), per = p.rows_a_block[what != 0];
    uint32_t const row0 = block * per, rows = min(per, p.rows - row0);
    for (uint32_t r = threadIdx.x >> 5; r < rows; r += APPEND_THREADS / 32) {
        place_t const w = find_place(p, row0 + r, what);
        if ((threadIdx.x & 31) == 0) places[r] = w;
    }
    if (blockIdx.x == 0 && p.row_offsets) // wrong offsets that no row meets are reported too
        for (uint32_t i = threadIdx.x; i < p.batch; i += APPEND_THREADS) {
            int const a = p.row_offsets[i], b = p.row_offsets[i + 1];
            if (a < 0 || b < a || b > (int)p.rows) atomicCAS(&g_append_error, 0u, (unsigned)PAGED_BAD_ROWS);
        }
    uint32_t const heads = what ? p.kv_heads : p.heads;
    uint32_t const at_once = APPEND_THREADS / p.upd.d; // heads that the block moves at once: of one row, or of several rows
    uint32_t const mine = fdivide(threadIdx.x, p.upd), u = threadIdx.x - mine * p.upd.d;
    uint32_t const rows_at_once = max(at_once / heads, 1u), row_off = heads < at_once ? fdivide(mine, p.by_heads[what != 0]) : 0;
    uint32_t const h0 = mine - row_off * heads;
    bool const     on = mine < at_once && row_off < rows_at_once && h0 < heads;
    unit_t const   t = unit_of<HALVES>(u, p.d, p.rot);
    bool const     turn = what != 2 && t.rotated;
    int64_t const  si0 = (what == 0 ? p.q_stride : what == 1 ? p.k_stride : p.v_stride)[0];
    int64_t const  si1 = (what == 0 ? p.q_stride : what == 1 ? p.k_stride : p.v_stride)[1];
    int64_t const  so1 = what == 0 ? p.q_out_stride[1] : what == 1 ? p.kc_stride[2] : p.vc_stride[2];
    TI const*      src = static_cast<TI const*>(what == 0 ? p.q : what == 1 ? p.k : p.v) + (int64_t)(row0 + row_off) * si0 + (int64_t)h0 * si1;
    TC*            dst = static_cast<TC*>(what == 0 ? p.q_out : what == 1 ? p.k_cache : p.v_cache) + (int64_t)h0 * so1;
    float const*   angles = p.freqs + (HALVES ? 2 * t.e0 : t.e0); // rot / 2 pairs of floats a position
    __syncthreads();
    if (!on) return;
    for (uint32_t r = row_off; r < rows; r += rows_at_once, src += rows_at_once * si0) {
        place_t const at = places[r];
        if (at.to < 0) continue;
        float     c[8];
        int const pairs = VEC ? 4 : HALVES ? t.n0 : min(4, (int)(p.rot - t.e0) / 2); // of the unit that are rotated (turn)
        if (turn) {
            float const* f = angles + at.angle;
            if (VEC) {
                load_8(f, c);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < pairs) c[2 * j] = f[2 * j], c[2 * j + 1] = f[2 * j + 1];
            }
        }
        TI const* s = src;
        TC*       d = dst + at.to;
        for (uint32_t h = h0; h < heads; h += 2 * at_once) { // two heads' loads in flight, beside the angles'
            bool const two = h + at_once < heads;
            raw_t<TI>  in[2];
            load_unit<HALVES, VEC>(s, t, in[0]);
            if (two) load_unit<HALVES, VEC>(s + at_once * si1, t, in[1]);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (x && !two) break;
                TC* const to = d + (x ? at_once * so1 : 0);
                float     y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = to_f32(in[x].v[j]);
                if (turn) rotate<HALVES>(y, c, pairs);
                store_unit<HALVES, VEC>(to, t, y);
            }
            s += 2 * at_once * si1;
            d += 2 * at_once * so1;
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
    // units a head: adjacent pairs ceil(d / 8); halves: runs of 4 of either half, then 8 of the rest
    uint32_t const units = halves ? (half + 3) / 4 + (c.head_dim - a.rotary_dim + 7) / 8 : (c.head_dim + 7) / 8;
    p.upd = make_fastdivide(units);
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
    // one wave of blocks, the same number of units each
    p.by_heads[0] = make_fastdivide(std::max(a.heads, 1u));
    p.by_heads[1] = make_fastdivide(c.kv_heads);
    uint64_t const wave = blocks_an_sm(a.in_dtype == ES_F16 && vec) * SM_COUNT;
    uint64_t const all = (uint64_t)c.rows * (a.heads + 2ull * c.kv_heads) * units;
    uint64_t const share = std::max<uint64_t>(APPEND_THREADS, (all + wave - 1) / wave);
    auto           rows_for = [&](uint64_t a_row) { return (uint32_t)std::min<uint64_t>(ROWS_MAX, std::max<uint64_t>(1, (share + a_row - 1) / a_row)); };
    p.rows_a_block[0] = rows_for((uint64_t)std::max(a.heads, 1u) * units);
    p.rows_a_block[1] = rows_for((uint64_t)c.kv_heads * units);
    uint64_t const bq = a.heads ? (c.rows + (uint64_t)p.rows_a_block[0] - 1) / p.rows_a_block[0] : 0;
    uint64_t const bk = (c.rows + (uint64_t)p.rows_a_block[1] - 1) / p.rows_a_block[1];
    if (bq + 2 * bk > 0x7fffffffull) fail(ES_NOT_SUPPORTED, "cache append: too many rows");
    p.first_block[0] = (uint32_t)bq;
    p.first_block[1] = (uint32_t)(bq + bk);
    dim3 const  grid((uint32_t)(bq + 2 * bk));
    pdl_scope_t scope(pdl_allowed()); // (the kernel waits for those before it itself)
    auto        go = [&](auto kernel) { launch_k(kernel, grid, dim3(APPEND_THREADS), 0, stream, p); };
    auto        pick = [&](auto ti, auto tc) {
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
