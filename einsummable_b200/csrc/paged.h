// Paged key / value cache: appending rotated keys and values (cache_append.cu) and the attention that
// reads the cache (paged_attention.cu).
#pragma once
#include <cuda_runtime.h>

#include "common.h"

namespace es {

// Throw es_error when the descriptor or the pointers cannot be served.
void check_cache_append(es_cache_append_t const& a, es_cache_append_args_t const& x);
void check_paged_attention(es_paged_attention_t const& a, es_paged_attention_args_t const& x, bool prefix);

uint64_t paged_attention_workspace(es_paged_attention_t const& a);

// The number of kernels launched is returned.
int launch_cache_append(es_cache_append_t const& a, es_cache_append_args_t const& x, cudaStream_t stream);
int launch_paged_attention(es_paged_attention_t const& a, es_paged_attention_args_t const& x, void* workspace,
                           uint64_t workspace_bytes, cudaStream_t stream);

// Algorithmic work of one launch.  What the sequences hold is known on the device only: an attention
// counts its queries, results and the shared prefix, not the sequences' own keys.
inline uint64_t cache_append_bytes(es_cache_append_t const& a)
{
    uint64_t const in = dtype_size(a.in_dtype), out = dtype_size(a.cache.dtype);
    return (uint64_t)a.cache.rows * a.cache.head_dim * (a.heads + 2ull * a.cache.kv_heads) * (in + out);
}
inline uint64_t paged_attention_bytes(es_paged_attention_t const& a)
{
    uint64_t const e = dtype_size(a.cache.dtype);
    return e * a.cache.head_dim * (2ull * a.cache.rows * a.heads + 2ull * a.prefix_len * a.cache.kv_heads);
}

// 0 = fine; 0x21.. = what the kernels found in the arrays on the device (es_b200_device_status)
unsigned int read_and_clear_append_error();
unsigned int read_and_clear_paged_error();

} // namespace es
