// Attention over a paged cache, with or without a shared prefix: checks, choice of kernel, launches.
//
//   s_j = scale q . k_j,   out = sum_j exp(s_j - lse) v_j,   lse = log sum_j exp(s_j)
//
// in one pass over the keys with the running maximum and sum of a softmax.  A shared prefix is attended first,
// as one sequence whose rows are the rows of the whole batch -- its keys are read once for all of them --
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
constexpr uint32_t MMA_BLOCKS = 2 * SM_COUNT, MMA_WORKERS = MMA_BLOCKS * MMA_WARPS, MMA_MAX_TR = 32;
constexpr uint32_t WIDE_BLOCKS = SM_COUNT;

uint64_t align256(uint64_t x)
{
    return (x + 255) / 256 * 256;
}

struct layout_t {
    uint64_t part_out, part_ml, meta, base_out, base_lse, total;
};

layout_t layout(es_paged_attention_t const& a)
{
    es_paged_cache_t const& c = a.cache;
    layout_t                l;
    // of every kernel that the pointers may make the call choose: workers x 2 slots x rows (x head dim)
    uint64_t part = 2ull * SIMT_BLOCKS * 16 * 32, ml = 2ull * SIMT_BLOCKS * 8, meta = SIMT_BLOCKS;
    if (c.dtype == ES_F16 && c.head_dim <= 128) {
        part = std::max<uint64_t>(part, 2ull * MMA_WORKERS * MMA_MAX_TR * (c.head_dim <= 64 ? 64 : 128));
        ml = std::max<uint64_t>(ml, 2ull * MMA_WORKERS * MMA_MAX_TR);
        meta = std::max<uint64_t>(meta, MMA_WORKERS);
        part = std::max<uint64_t>(part, 2ull * WIDE_BLOCKS * WIDE_TR * (c.head_dim <= 64 ? 64 : 128));
        ml = std::max<uint64_t>(ml, 2ull * WIDE_BLOCKS * WIDE_TR);
    }
    uint64_t at = 0;
    l.part_out = at;
    at += align256(part * 4);
    l.part_ml = at;
    at += align256(ml * 8);
    l.meta = at;
    at += align256(meta * 2 * 16);
    l.base_out = at;
    if (a.prefix_len) at += align256((uint64_t)c.rows * a.heads * c.head_dim * 4);
    l.base_lse = at;
    if (a.prefix_len) at += align256((uint64_t)c.rows * a.heads * 4);
    l.total = at;
    return l;
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

template <typename T> int launch_simt(paged_params_t& p, bool vec, cudaStream_t stream)
{
    uint32_t const nch = p.d <= 64 ? 2 : p.d <= 128 ? 4 : 8;
    uint32_t const tr = 16 / nch;
    p.part_d = nch * 32;
    // Direct: with at most 8 key tiles an item, one block an item and no join -- a join costs as much as
    // about 8 tiles take
    p.direct = !p.row_offsets && p.prefix_len < 0 && p.capacity <= 8 * SIMT_BK;
    if (p.batch > 65535) p.direct = 0;
    uint32_t const grid = p.direct ? p.kv_heads * ((p.group + tr - 1) / tr) : SIMT_BLOCKS;
    auto           go = [&](auto kernel) { launch_k(kernel, dim3(grid, p.direct ? p.batch : 1), dim3(128), 0, stream, p); };
    if (nch == 2) vec ? go(paged_simt_kernel<T, 2, true>) : go(paged_simt_kernel<T, 2, false>);
    else if (nch == 4) vec ? go(paged_simt_kernel<T, 4, true>) : go(paged_simt_kernel<T, 4, false>);
    else vec ? go(paged_simt_kernel<T, 8, true>) : go(paged_simt_kernel<T, 8, false>);
    if (p.direct) return 1;
    pdl_scope_t scope(true);
    auto        join = [&](auto kernel) { launch_k(kernel, dim3(grid), dim3(256), 0, stream, p, vec ? 1 : 0); };
    if (nch == 2) join(paged_join_kernel<T, 8, 1>);
    else if (nch == 4) join(paged_join_kernel<T, 4, 1>);
    else join(paged_join_kernel<T, 2, 2>);
    return 2;
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

template <int DPAD, int NT, bool PAGE16> void launch_mma_as(paged_params_t const& p, dim3 grid, uint32_t q_rows, cudaStream_t stream)
{
    static bool done[64] = {};
    allow_smem(paged_mma_kernel<DPAD, NT, PAGE16>, MMA_WARPS * mma_warp_bytes<DPAD>(8 * NT), done);
    launch_k(paged_mma_kernel<DPAD, NT, PAGE16>, grid, dim3(MMA_WARPS * 32), MMA_WARPS * mma_warp_bytes<DPAD>(q_rows), stream, p, q_rows);
}

template <int NT> int launch_mma(paged_params_t& p, cudaStream_t stream)
{
    constexpr uint32_t TR = 8 * NT;
    bool const         page16 = p.page.d % MMA_BK == 0;
    p.part_d = p.d <= 64 ? 64 : 128;
    // Direct: with at most 16 key tiles an item, one warp an item and no join
    p.direct = !p.row_offsets && p.prefix_len < 0 && p.capacity <= 16 * MMA_BK;
    p.min_units = 4;
    if (p.batch > 65535) p.direct = 0;
    uint32_t const items = p.kv_heads * ((p.group + TR - 1) / TR); // of a sequence
    dim3 const     grid(p.direct ? (items + MMA_WARPS - 1) / MMA_WARPS : MMA_BLOCKS, p.direct ? p.batch : 1);
    // rows of a query tile: the packed rows of one token, or of all there are
    uint32_t const q_rows = std::min<uint32_t>(TR, !p.row_offsets && p.prefix_len < 0 ? p.group : p.rows * p.group);
    if (p.part_d == 64) page16 ? launch_mma_as<64, NT, true>(p, grid, q_rows, stream) : launch_mma_as<64, NT, false>(p, grid, q_rows, stream);
    else page16 ? launch_mma_as<128, NT, true>(p, grid, q_rows, stream) : launch_mma_as<128, NT, false>(p, grid, q_rows, stream);
    if (p.direct) return 1;
    pdl_scope_t scope(true);
    launch_k(paged_join_kernel<__half, TR, 1>, dim3(MMA_WORKERS, (TR + 15) / 16), dim3(256), 0, stream, p, 1);
    return 2;
}

template <int DPAD, bool PAGE16> void launch_wide_as(paged_params_t const& p, cudaStream_t stream)
{
    static bool done[64] = {};
    allow_smem(paged_wide_kernel<DPAD, PAGE16>, wide_smem_bytes<DPAD>(), done);
    launch_k(paged_wide_kernel<DPAD, PAGE16>, dim3(WIDE_BLOCKS), dim3(WIDE_THREADS), wide_smem_bytes<DPAD>(), stream, p);
}

int launch_wide(paged_params_t& p, cudaStream_t stream)
{
    bool const page16 = p.page.d % 16 == 0;
    p.part_d = p.d <= 64 ? 64 : 128;
    p.direct = 0;
    p.min_units = 4;
    if (p.part_d == 64) page16 ? launch_wide_as<64, true>(p, stream) : launch_wide_as<64, false>(p, stream);
    else page16 ? launch_wide_as<128, true>(p, stream) : launch_wide_as<128, false>(p, stream);
    pdl_scope_t scope(true);
    if (p.part_d == 64) launch_k(paged_wide_join_kernel<64>, dim3(WIDE_BLOCKS, WIDE_TR / 16), dim3(256), 0, stream, p);
    else launch_k(paged_wide_join_kernel<128>, dim3(WIDE_BLOCKS, WIDE_TR / 16), dim3(256), 0, stream, p);
    return 2;
}

// f16 on the tensor cores: sequences (or the prefix) with up to MMA_MAX_TR packed rows a key head are bound by
// memory and go to the warp-level units, those with more to tcgen05.  How many rows a sequence has is known on
// the device when there are row offsets: then both kernels run and each takes its own.
int launch_phase(paged_params_t& p, int dtype, bool vec, cudaStream_t stream)
{
    p.packed_min = 0;
    p.packed_max = 0x7fffffff;
    if (dtype != ES_F16) return launch_simt<float>(p, vec, stream);
    if (!vec || p.d > 128) return launch_simt<__half>(p, vec, stream);
    // packed rows of an item: one token's, those of all rows there are, or (row offsets) something in between
    uint32_t const most = p.prefix_len < 0 && !p.row_offsets ? p.group : p.rows * p.group;
    uint32_t const fewest = p.row_offsets ? 1 : most;
    int            launches = 0;
    if (fewest <= MMA_MAX_TR) {
        p.packed_max = MMA_MAX_TR;
        uint32_t const rows = p.prefix_len >= 0 ? most : p.group; // of an item, where tokens come singly
        launches += rows <= 8 ? launch_mma<1>(p, stream) : rows <= 16 ? launch_mma<2>(p, stream) : launch_mma<4>(p, stream);
    }
    if (most > MMA_MAX_TR) {
        pdl_scope_t scope(launches > 0 || pdl_launch_flag());
        p.packed_min = MMA_MAX_TR;
        p.packed_max = 0x7fffffff;
        launches += launch_wide(p, stream);
    }
    return launches;
}

} // namespace

void check_paged_attention(es_paged_attention_t const& a, es_paged_attention_args_t const& x, bool prefix)
{
    es_paged_cache_t const& c = a.cache;
    check_paged_cache(c, "paged attention");
    if (!a.heads || a.heads % c.kv_heads) fail(ES_BAD_DESCRIPTOR, "paged attention: query heads must be a multiple of the key heads");
    if (a.heads > 65535) fail(ES_NOT_SUPPORTED, "paged attention: more than 65535 heads");
    if ((uint64_t)c.rows * (a.heads / c.kv_heads) > 0x7fffffffull) fail(ES_NOT_SUPPORTED, "paged attention: too many rows");
    if (!(a.scale >= 1e-30f && a.scale <= 1e30f)) fail(ES_BAD_DESCRIPTOR, "paged attention: the scale must lie in 1e-30 .. 1e30");
    if (!x.q || !x.k_cache || !x.v_cache || !x.out || !x.lengths || !x.tables) fail(ES_BAD_ARGUMENT, "paged attention: null pointer");
    if (!prefix && a.prefix_len) fail(ES_BAD_ARGUMENT, "paged attention: a prefix needs es_b200_launch_prefix_attention");
    if (a.prefix_len > 0x7fffffffu) fail(ES_NOT_SUPPORTED, "paged attention: prefix beyond 31 bits");
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
    p.part_out = reinterpret_cast<float*>(ws + l.part_out);
    p.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
    p.meta = reinterpret_cast<int4*>(ws + l.meta);
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
    int        launches = 0;
    if (a.prefix_len) {
        paged_params_t f = p;
        f.prefix_len = (int32_t)a.prefix_len;
        f.tables = x.prefix_pages;
        f.causal = 0;
        f.out = ws + l.base_out;
        f.out_f32 = 1;
        f.lse = reinterpret_cast<float*>(ws + l.base_lse);
        launches += launch_phase(f, c.dtype, vec, stream);
        p.base_out = reinterpret_cast<float const*>(ws + l.base_out);
        p.base_lse = reinterpret_cast<float const*>(ws + l.base_lse);
    }
    pdl_scope_t scope(launches > 0 || pdl_launch_flag());
    launches += launch_phase(p, c.dtype, vec, stream);
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
