// Shared by the kernels of the paged cache: how positions become addresses, what a sequence of the batch
// is, and how the attention's work is cut into equal shares.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "common.h"
#include "kernels.h"

namespace es {
namespace {

constexpr uint32_t SM_COUNT = 148;

// codes of es_b200_device_status
enum : unsigned { PAGED_BAD_PAGE = 0x21, PAGED_BAD_LENGTH = 0x22, PAGED_BAD_ROWS = 0x23, PAGED_BAD_POSITION = 0x24 };

// Exact division of numerators below 2^31 (see fastdiv_t).
inline fastdiv_t make_fastdivide(uint32_t d)
{
    fastdiv_t f = {0, 0, d, 0};
    if (d > 1) {
        uint32_t l = 0;
        while ((1ull << l) < d) ++l;
        f.m = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
        f.s = l - 1;
    }
    return f;
}
__device__ __forceinline__ uint32_t fdivide(uint32_t n, fastdiv_t const& f)
{
    return f.d == 1 ? n : __umulhi(n, f.m) >> f.s;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void  from_f32(float& y, float x) { y = x; }
__device__ __forceinline__ void  from_f32(__half& y, float x) { y = __float2half_rn(x); }

// Tokens a sequence's row of pages can hold; at most 2^30, so that a position and a few tiles fit 32 bits.
constexpr uint32_t MAX_TOKENS = 1u << 30;
inline uint32_t    paged_capacity(es_paged_cache_t const& c)
{
    uint64_t const n = (uint64_t)c.table_stride * c.page_size;
    return (uint32_t)(n < MAX_TOKENS ? n : MAX_TOKENS);
}

inline void check_paged_cache(es_paged_cache_t const& c, char const* who)
{
    std::string const w(who);
    if (c.dtype != ES_F16 && c.dtype != ES_F32) fail(ES_NOT_SUPPORTED, w + ": the cache must be f16 or f32");
    if (!c.batch || !c.kv_heads || !c.head_dim || !c.page_size || !c.n_pages || !c.table_stride)
        fail(ES_BAD_DESCRIPTOR, w + ": empty extent");
    if (c.head_dim > 256) fail(ES_NOT_SUPPORTED, w + ": head dim above 256");
    if (c.kv_heads > 65535) fail(ES_NOT_SUPPORTED, w + ": more than 65535 heads");
    if (c.batch > (1u << 24) || c.rows > 0x7fffffffu || c.page_size > 0x7fffffffu || c.n_pages > 0x7fffffffu)
        fail(ES_NOT_SUPPORTED, w + ": an extent beyond 31 bits (sequences: 24)");
    for (int i = 0; i != 3; ++i)
        if (c.k_stride[i] < 0 || c.v_stride[i] < 0) fail(ES_BAD_DESCRIPTOR, w + ": negative stride");
}

} // namespace
} // namespace es
