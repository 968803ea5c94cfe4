// Attention over a paged cache, with or without a shared prefix: checks, choice of kernel, launches.
//
//   s_j = scale q . k_j,   out = sum_j exp(s_j - lse) v_j,   lse = log sum_j exp(s_j)
//
// in one pass over the keys with the running maximum and sum of a softmax.  A shared prefix is attended first,
// as one sequence whose rows are the rows of the whole batch -- its keys are read once for a tile of them, which is
// 8, 16 or 256 rows a key head on the tensor cores and 1 to 8 without --
// into an f32 result and its lse; the sequences' own keys follow, and the two are weighed by exp(lse) where a
// row is finished.
#include <algorithm>
#include <cstring>
#include <string>

#include "paged.h"
#include "paged_mma.h"
#include "paged_simt.h"
#include "paged_wide.h"
#include "paged_work.h"

namespace es {

namespace {

__device__ unsigned int g_paged_error;

constexpr uint32_t SIMT_BLOCKS = 2 * SM_COUNT;
constexpr uint32_t MMA_BLOCKS = 2 * SM_COUNT, MMA_WORKERS = MMA_BLOCKS * MMA_WARPS, MMA_MAX_TR = 16;
constexpr uint32_t WIDE_BLOCKS = SM_COUNT;

uint64_t align256(uint64_t x)
{
    return (x + 255) / 256 * 256;
}

// Partial results of the two kernels that a call may have in flight at once, and a prefix's result
struct layout_t {
    struct region_t {
        uint64_t out, ml, meta;
    } region[2];
    uint64_t base_out, base_lse, total;
};

layout_t layout(es_paged_attention_t const& a)
{
    es_paged_cache_t const& c = a.cache;
    layout_t                l;
    // of every kernel that the pointers may make the call choose: workers x 2 slots x rows (x head dim)
    uint64_t part = 2ull * SIMT_BLOCKS * 16 * 32, ml = 2ull * SIMT_BLOCKS * 8, meta = SIMT_BLOCKS;
    if (c.dtype == ES_F16 && c.head_dim <= 128) {
        uint64_t const d = c.head_dim <= 64 ? 64 : 128;
        part = std::max<uint64_t>(part, 2ull * MMA_WORKERS * MMA_MAX_TR * d);
        part = std::max<uint64_t>(part, 2ull * WIDE_BLOCKS * WIDE_TR * d);
        ml = std::max<uint64_t>(ml, 2ull * MMA_WORKERS * MMA_MAX_TR);
        ml = std::max<uint64_t>(ml, 2ull * WIDE_BLOCKS * WIDE_TR);
        meta = std::max<uint64_t>(meta, MMA_WORKERS);
    }
    uint64_t at = 0;
    for (auto& r : l.region) {
        r.out = at;
        at += align256(part * 4);
        r.ml = at;
        at += align256(ml * 8);
        r.meta = at;
        at += align256(meta * 2 * 16);
    }
    l.base_out = at;
    if (a.prefix_len) at += align256((uint64_t)c.rows * a.heads * c.head_dim * 4);
    l.base_lse = at;
    if (a.prefix_len) at += align256((uint64_t)c.rows * a.heads * 4);
    l.total = at;
    return l;
}

void use_region(paged_params_t& p, char* ws, layout_t::region_t const& r)
{
    p.part_out = reinterpret_cast<float*>(ws + r.out);
    p.part_ml = reinterpret_cast<float2*>(ws + r.ml);
    p.meta = reinterpret_cast<int4*>(ws + r.meta);
}

unsigned int* error_address()
{
    static unsigned int* addr[64] = {};
    int                  dev = 0;
    ES_CUDA_CHECK(cudaGetDevice(&dev));
    if (!addr[dev & 63]) ES_CUDA_CHECK(cudaGetSymbolAddress(reinterpret_cast<void**>(&addr[dev & 63]), g_paged_error));
    return addr[dev & 63];
}

// Whether 16-byte accesses may be used on every row of every operand
bool aligned16(es_paged_attention_t const& a, es_paged_attention_args_t const& x)
{
    es_paged_cache_t const& c = a.cache;
    uint64_t const per = 16 / dtype_size(c.dtype);
    uint64_t       el = c.head_dim;
    for (int i = 0; i != 2; ++i) el |= (uint64_t)a.q_stride[i] | (uint64_t)a.out_stride[i];
    for (int i = 0; i != 3; ++i) el |= (uint64_t)c.k_stride[i] | (uint64_t)c.v_stride[i];
    uintptr_t const bits = reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.out) |
                           reinterpret_cast<uintptr_t>(x.k_cache) | reinterpret_cast<uintptr_t>(x.v_cache);
    // (the tensor-core kernels step through a page in 32 bits of bytes)
    return (el % per) == 0 && (bits & 15) == 0 && c.k_stride[1] < (1 << 26) && c.v_stride[1] < (1 << 26);
}

// One kernel's part of a call: `main` cuts the work into shares, `join` (null: nothing can be split) puts items
// that crossed shares together.
struct part_t {
    paged_params_t p;
    void (*main)(paged_params_t const&, cudaStream_t);
    void (*join)(paged_params_t const&, cudaStream_t);
};

// Tokens an item can have to visit (an upper bound from the descriptor; what there is only the device knows)
uint64_t most_keys(paged_params_t const& p)
{
    return p.prefix_len >= 0 ? (uint64_t)p.prefix_len : (uint64_t)p.capacity + p.front;
}

template <typename T, int NCH, int TR, bool VEC> part_t simt_as(paged_params_t p)
{
    part_t c;
    p.part_d = NCH * 32;
    // Direct: with at most 8 key tiles an item, one block an item and no join -- a join costs as much as
    // about 8 tiles take
    p.direct = !p.row_offsets && p.prefix_len < 0 && most_keys(p) <= 8 * SIMT_BK && p.batch <= 65535;
    c.p = p;
    c.main = [](paged_params_t const& p, cudaStream_t s) {
        dim3 const grid(p.direct ? p.kv_heads * ((p.group + TR - 1) / TR) : SIMT_BLOCKS, p.direct ? p.batch : 1);
        launch_k(paged_simt_kernel<T, NCH, TR, VEC>, grid, dim3(128), 0, s, p);
    };
    c.join = nullptr;
    if (!p.direct)
        c.join = [](paged_params_t const& p, cudaStream_t s) {
            launch_k(paged_join_kernel<T, TR, (NCH * 32 + 127) / 128>, dim3(SIMT_BLOCKS), dim3(256), 0, s, p, VEC ? 1 : 0);
        };
    return c;
}
// TR: rows that read a key together: as many as there are for one token, up to what fits the registers
template <typename T, bool VEC> part_t simt_part(paged_params_t const& p)
{
    bool const one = sizeof(T) == 4 && p.group == 1 && !p.row_offsets && p.prefix_len < 0;
    if (p.d <= 64) {
        if constexpr (sizeof(T) == 4) {
            if (one) return simt_as<T, 2, 1, VEC>(p);
            if (p.group > 4 || p.prefix_len >= 0) return simt_as<T, 2, 8, VEC>(p);
        }
        return simt_as<T, 2, 4, VEC>(p);
    }
    if (p.d <= 128) {
        if constexpr (sizeof(T) == 4)
            if (one) return simt_as<T, 4, 1, VEC>(p);
        return simt_as<T, 4, 4, VEC>(p);
    }
    if constexpr (sizeof(T) == 4)
        if (one) return simt_as<T, 8, 1, VEC>(p);
    return simt_as<T, 8, 2, VEC>(p);
}
template <typename T> part_t simt_part(paged_params_t const& p, bool vec)
{
    return vec ? simt_part<T, true>(p) : simt_part<T, false>(p);
}

// Kernels with more shared memory than 48 KB say so once per device
template <typename K> void allow_smem(K kernel, uint32_t bytes, bool (&done)[64])
{
    int dev = 0;
    ES_CUDA_CHECK(cudaGetDevice(&dev));
    if (done[dev & 63]) return;
    ES_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done[dev & 63] = true;
}

template <int DPAD, int NT, bool PAGE16> part_t mma_as(paged_params_t p)
{
    constexpr uint32_t TR = 8 * NT;
    part_t             c;
    p.part_d = DPAD;
    // Direct: nothing is counted, and there is no join kernel.  While no block takes a second item: a block each, if a
    // warp's part is at most 16 tiles (32 heads on 8, cut / a block each: 1 x 500 keys 17.3 / 14.3 us, 4 x 500 19.4 /
    // 14.3, 36 x 1000 46 / 39, and 1 x 1000 19.4 / 19.5); more of them: a warp each, if its 16 tiles are the whole item
    // (1 x 250 keys 19.5 us that way, 11.2 a block each; 16 x 250 20.4 and 13.2).
    uint32_t const items = p.kv_heads * ((p.group + TR - 1) / TR); // of a sequence
    uint64_t const all = (uint64_t)p.batch * items, keys = most_keys(p);
    p.direct = DIRECT_NO;
    if (!p.row_offsets && p.prefix_len < 0 && p.batch <= 65535) {
        if (all <= MMA_BLOCKS && keys <= 16 * MMA_BK * MMA_WARPS) p.direct = DIRECT_BLOCK;
        else if (keys <= 16 * MMA_BK) p.direct = DIRECT_WORKER;
    }
    p.min_units = 4;
    c.p = p;
    c.main = [](paged_params_t const& p, cudaStream_t s) {
        static bool done[2][64] = {};
        auto* const kernel = p.base_out ? paged_mma_kernel<DPAD, NT, PAGE16, true> : paged_mma_kernel<DPAD, NT, PAGE16, false>;
        allow_smem(kernel, MMA_WARPS * mma_warp_bytes<DPAD>(TR), done[p.base_out ? 1 : 0]);
        uint32_t const items = p.kv_heads * ((p.group + TR - 1) / TR); // of a sequence
        dim3 const     grid(p.direct == DIRECT_BLOCK ? items : p.direct ? (items + MMA_WARPS - 1) / MMA_WARPS : MMA_BLOCKS,
                            p.direct ? p.batch : 1);
        // rows of a query tile: the packed rows of one token, or of all there are
        uint32_t const q_rows = std::min(uint32_t(TR), !p.row_offsets && p.prefix_len < 0 ? p.group : p.rows * p.group);
        launch_k(kernel, grid, dim3(MMA_WARPS * 32), MMA_WARPS * mma_warp_bytes<DPAD>(q_rows), s, p, q_rows);
    };
    c.join = nullptr;
    if (!p.direct)
        c.join = [](paged_params_t const& p, cudaStream_t s) {
            launch_k(paged_join_kernel<__half, TR, 1>, dim3(MMA_WORKERS, (TR + 15) / 16), dim3(256), 0, s, p, 1);
        };
    return c;
}
template <int NT> part_t mma_part(paged_params_t const& p)
{
    bool const page16 = p.page.d % MMA_BK == 0;
    if (p.d <= 64) return page16 ? mma_as<64, NT, true>(p) : mma_as<64, NT, false>(p);
    return page16 ? mma_as<128, NT, true>(p) : mma_as<128, NT, false>(p);
}

template <int DPAD, bool PAGE16> part_t wide_as(paged_params_t p)
{
    part_t c;
    p.part_d = DPAD;
    p.direct = 0;
    p.min_units = 4;
    c.p = p;
    c.main = [](paged_params_t const& p, cudaStream_t s) {
        static bool done[64] = {};
        allow_smem(paged_wide_kernel<DPAD, PAGE16>, wide_smem_bytes<DPAD>(), done);
        launch_k(paged_wide_kernel<DPAD, PAGE16>, dim3(WIDE_BLOCKS), dim3(WIDE_THREADS), wide_smem_bytes<DPAD>(), s, p);
    };
    c.join = [](paged_params_t const& p, cudaStream_t s) {
        launch_k(paged_wide_join_kernel<DPAD>, dim3(WIDE_BLOCKS, WIDE_TR / 16), dim3(256), 0, s, p);
    };
    return c;
}
part_t wide_part(paged_params_t const& p)
{
    bool const page16 = p.page.d % 16 == 0;
    if (p.d <= 64) return page16 ? wide_as<64, true>(p) : wide_as<64, false>(p);
    return page16 ? wide_as<128, true>(p) : wide_as<128, false>(p);
}

// The kernels of one phase (a prefix, or the sequences' own keys), at most two.  f16 on the tensor cores:
// sequences (or the prefix) with up to MMA_MAX_TR packed rows a key head are bound by memory and go to the
// warp-level units, those with more to tcgen05.  How many rows a sequence has is known on the device when there
// are row offsets: then both kernels run and each takes its own.
int choose(paged_params_t const& q, int dtype, bool vec, part_t (&c)[2])
{
    paged_params_t p = q;
    p.packed_min = 0;
    p.packed_max = 0x7fffffff;
    if (dtype != ES_F16) {
        c[0] = simt_part<float>(p, vec);
        return 1;
    }
    if (!vec || p.d > 128) {
        c[0] = simt_part<__half>(p, vec);
        return 1;
    }
    // packed rows of an item: one token's, those of all rows there are, or (row offsets) something in between
    uint32_t const most = p.prefix_len < 0 && !p.row_offsets ? p.group : p.rows * p.group;
    uint32_t const fewest = p.row_offsets ? 1 : most;
    int            n = 0;
    if (fewest <= MMA_MAX_TR) {
        p.packed_max = MMA_MAX_TR;
        uint32_t const rows = p.prefix_len >= 0 ? most : p.group; // of an item, where tokens come singly
        // (tiles of 32 rows spill: 8 sequences of 4 query heads a key head behind 8000 tokens took 76 us, 45 with tcgen05)
        c[n++] = rows <= 8 ? mma_part<1>(p) : mma_part<2>(p);
    }
    if (most > MMA_MAX_TR) {
        p.packed_min = MMA_MAX_TR;
        p.packed_max = 0x7fffffff;
        c[n++] = wide_part(p);
    }
    return n;
}

} // namespace

void check_paged_attention(es_paged_attention_t const& a, es_paged_attention_args_t const& x, bool prefix)
{
    es_paged_cache_t const& c = a.cache;
    check_paged_cache(c, "paged attention");
    if (!a.heads || a.heads % c.kv_heads) fail(ES_BAD_DESCRIPTOR, "paged attention: query heads must be a multiple of the key heads");
    if (a.heads > 65535) fail(ES_NOT_SUPPORTED, "paged attention: more than 65535 heads");
    if ((uint64_t)c.rows * (a.heads / c.kv_heads) > 0x7fffffffull) fail(ES_NOT_SUPPORTED, "paged attention: too many rows");
    // (f16: 256 * 65504^2 * 1e26 * log2 e, so that every score and lse is finite)
    if (!(a.scale >= 1e-30f && a.scale <= (c.dtype == ES_F16 ? 1e26f : 1e30f)))
        fail(ES_BAD_DESCRIPTOR, "paged attention: the scale must lie in 1e-30 .. 1e30 (f16: 1e26)");
    if (!x.q || !x.k_cache || !x.v_cache || !x.out || !x.lengths || !x.tables) fail(ES_BAD_ARGUMENT, "paged attention: null pointer");
    if (!prefix && a.prefix_len) fail(ES_BAD_ARGUMENT, "paged attention: a prefix needs es_b200_launch_prefix_attention");
    if (a.prefix_len > MAX_TOKENS) fail(ES_NOT_SUPPORTED, "paged attention: prefix beyond 2^30 tokens");
    if (a.prefix_len && !x.prefix_pages) fail(ES_BAD_ARGUMENT, "paged attention: null list of the prefix's pages");
    if (!x.row_offsets && c.rows != c.batch) fail(ES_BAD_DESCRIPTOR, "paged attention: without row offsets there is one row a sequence");
    for (int i = 0; i != 2; ++i)
        if (a.q_stride[i] < 0 || a.out_stride[i] < 0) fail(ES_BAD_DESCRIPTOR, "paged attention: negative stride");
    uintptr_t const e = dtype_size(c.dtype) - 1;
    if (((reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.out) | reinterpret_cast<uintptr_t>(x.k_cache) |
          reinterpret_cast<uintptr_t>(x.v_cache)) & e) ||
        ((reinterpret_cast<uintptr_t>(x.lse) | reinterpret_cast<uintptr_t>(x.row_offsets) | reinterpret_cast<uintptr_t>(x.lengths) |
          reinterpret_cast<uintptr_t>(x.tables) | reinterpret_cast<uintptr_t>(x.prefix_pages)) & 3))
        fail(ES_BAD_ARGUMENT, "paged attention: a pointer is not aligned to its elements");
}

uint64_t paged_attention_workspace(es_paged_attention_t const& a)
{
    check_paged_cache(a.cache, "paged attention");
    return layout(a).total;
}

int launch_paged_attention(es_paged_attention_t const& a, es_paged_attention_args_t const& x, void* workspace,
                           uint64_t workspace_bytes, cudaStream_t stream)
{
    es_paged_cache_t const& c = a.cache;
    if (c.rows == 0) return 0;
    layout_t const l = layout(a);
    if (!workspace || workspace_bytes < l.total)
        fail(ES_WORKSPACE_TOO_SMALL, "paged attention: workspace of " + std::to_string(l.total) + " bytes required");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) fail(ES_BAD_ARGUMENT, "paged attention: workspace must be 16-byte aligned");
    char* const    ws = static_cast<char*>(workspace);
    paged_params_t p = {};
    p.q = x.q;
    p.k = x.k_cache;
    p.v = x.v_cache;
    p.out = x.out;
    p.lse = x.lse;
    p.row_offsets = x.row_offsets;
    p.lengths = x.lengths;
    p.tables = x.tables;
    for (int i = 0; i != 2; ++i) {
        p.q_stride[i] = a.q_stride[i];
        p.out_stride[i] = a.out_stride[i];
    }
    for (int i = 0; i != 3; ++i) {
        p.k_stride[i] = c.k_stride[i];
        p.v_stride[i] = c.v_stride[i];
    }
    p.batch = c.batch;
    p.rows = c.rows;
    p.heads = a.heads;
    p.kv_heads = c.kv_heads;
    p.group = a.heads / c.kv_heads;
    p.d = c.head_dim;
    p.n_pages = c.n_pages;
    p.table_stride = c.table_stride;
    p.capacity = paged_capacity(c);
    p.page = make_fastdivide(c.page_size);
    p.grp = make_fastdivide(p.group);
    p.causal = a.causal != 0;
    p.prefix_len = -1;
    p.min_units = 1;
    p.scale_log2 = a.scale * LOG2_E;
    p.error = error_address();
    bool const vec = aligned16(a, x);
    // A short prefix is read by every sequence for itself, in front of its own keys and out of the L2 cache: one
    // kernel and a join.  Reading it once adds two kernels -- few rows: the same kind again (8 sequences of 32 key
    // heads behind 500 / 1000 / 2000 tokens, 62 / 125 / 250 MB read in all: 24 / 26 / 36 us shared, 18 / 32 / 42 in
    // front; 3 sequences of 8 behind 4000, 47 MB: 36 and 26), more: tcgen05's, whose start alone is worth some 20 us
    // (16 sequences of 8 key heads behind 1000 / 2000 / 4000 tokens, 62 / 125 / 250 MB: 38 / 38 / 40 us shared,
    // 26 / 30 / 40 in front; 64 sequences behind 500 / 1000 / 2000, 125 / 250 / 500 MB: 46 / 46 / 46 and 34 / 44 /
    // 63; 16 of 4 key heads of 64 behind 8000, 125 MB: 36 and 36).  f32, 4 key heads of 64: 8 sequences behind 4000,
    // 62 MB, 42 and 38; 64 behind 2000, 250 MB, 99 and 95.  Single tokens only: parts of prompts have rows enough to
    // share.
    bool const     tc = c.dtype == ES_F16 && vec && c.head_dim <= 128;
    uint64_t const all = (uint64_t)c.batch * a.prefix_len * c.kv_heads * c.head_dim * 2 * dtype_size(c.dtype);
    uint64_t const most = (tc && c.rows * p.group > MMA_MAX_TR ? 224ull : 64ull) << 20;
    bool const     front = a.prefix_len && !x.row_offsets && (!tc || p.group <= MMA_MAX_TR) && all <= most;
    int            launches = 0;
    pdl_scope_t    scope(pdl_allowed()); // (every kernel waits for those before it itself)
    if (front) {
        p.front = a.prefix_len;
        p.front_pages = x.prefix_pages;
    } else if (a.prefix_len) {
        paged_params_t f = p;
        f.prefix_len = (int32_t)a.prefix_len;
        f.tables = x.prefix_pages;
        f.causal = 0;
        f.out = ws + l.base_out;
        f.out_f32 = 1;
        f.lse = reinterpret_cast<float*>(ws + l.base_lse);
        part_t    k[2];
        int const n = choose(f, c.dtype, vec, k);
        for (int i = 0; i != n; ++i) {
            use_region(k[i].p, ws, l.region[0]);
            k[i].p.order = i == 0 && n == 1 ? ORDER_FIRST : ORDER_PLAIN;
            k[i].main(k[i].p, stream);
            if (k[i].join) k[i].join(k[i].p, stream);
            launches += k[i].join ? 2 : 1;
        }
        // the sequences' own keys need the prefix's result only where a row is finished
        p.order = n == 1 ? ORDER_LATE : ORDER_PLAIN;
        p.base_out = reinterpret_cast<float const*>(ws + l.base_out);
        p.base_lse = reinterpret_cast<float const*>(ws + l.base_lse);
    }
    part_t    k[2];
    int const n = choose(p, c.dtype, vec, k);
    if (n == 2 && p.order == ORDER_PLAIN) { // independent of one another
        k[0].p.order = ORDER_FIRST;
        k[1].p.order = ORDER_LATE;
    } else if (n == 2) {
        k[0].p.order = k[1].p.order = ORDER_PLAIN;
    }
    for (int i = 0; i != n; ++i) {
        use_region(k[i].p, ws, l.region[n == 2 ? i : 1]);
        k[i].main(k[i].p, stream);
        launches += k[i].join ? 2 : 1;
    }
    for (int i = 0; i != n; ++i)
        if (k[i].join) k[i].join(k[i].p, stream);
    return launches;
}

unsigned int read_and_clear_paged_error()
{
    unsigned int v = 0, zero = 0;
    ES_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_paged_error, sizeof v));
    if (v) ES_CUDA_CHECK(cudaMemcpyToSymbol(g_paged_error, &zero, sizeof zero));
    return v;
}

} // namespace es
