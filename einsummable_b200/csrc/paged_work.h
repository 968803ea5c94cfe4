// The work of a paged attention call, how it is cut into equal shares, and how partial results are joined.
//
// An item is one (sequence, key / value head, tile of TR packed rows): packed row r of a sequence stands for
// query head r % group of its token r / group, so that all heads that read the same keys share them.  An
// item's keys are visited in tiles of BK; one (item, key tile) is a unit, and OVH more stand for what an item
// costs beside its tiles (queries, page list, result): units that nothing is done for.  Without them a share of
// many short items took several times as long as one of few long ones (64 sequences of 1 to 8192 tokens: 87 us, 55
// with them).  Lengths are known on the device only, and differ: so every block counts all units (a scan over the
// batch), and every worker -- the block, or each of its warps -- takes the same number of consecutive units and
// finds its first one.  An item inside one worker's share is finished there; one that crosses shares leaves an
// unnormalised partial result per share, at most two a worker (its first and its last item), which a second small
// kernel joins in order of the keys (about 5 us behind the first).  Nothing depends on the order in which blocks
// run: the same call gives the same bits.
#pragma once
#include "paged_device.h"
#include "pdl.h"

namespace es {
namespace {

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float LOG2_E = 1.4426950408889634f;
constexpr float LN_2 = 0.6931471805599453f;

struct paged_params_t {
    void const*    q;
    void const*    k;
    void const*    v;
    void*          out;         // rows of the cache's type, or (out_f32) the joined prefix in f32, dense
    float*         lse;         // natural log; may be null
    int32_t const* row_offsets; // may be null
    int32_t const* lengths;
    int32_t const* tables;
    float const*   base_out;    // result over a prefix [rows, heads, d], merged in; may be null
    float const*   base_lse;
    float*         part_out;    // [workers][2][TR][part_d]
    float2*        part_ml;     // [workers][2][TR]: what the sum is relative to (log2 units), sum
    int4*          meta;        // [workers][2]
    int64_t        q_stride[2], out_stride[2], k_stride[3], v_stride[3];
    uint32_t       batch, rows, heads, kv_heads, group, d, part_d, n_pages, table_stride, capacity;
    fastdiv_t      page, grp;
    int32_t        causal;
    int32_t        prefix_len;  // >= 0: all rows attend the one list of pages `tables`, of this many tokens
    int32_t const* front_pages; // front > 0: so many tokens, listed here, lie in front of every sequence's own (each
    uint32_t       front;       // sequence reads them for itself); their last key tile is not shared with its own
    int32_t        direct;      // nothing is split among workers (one row a sequence): DIRECT_*
    uint32_t       packed_min, packed_max; // sequences with more than / at most so many packed rows
    uint32_t       min_units;   // a worker's share is at least this
    float          scale_log2;  // scale * log2 e
    int32_t        out_f32;
    int32_t        order;       // ORDER_*: when the kernel waits for the kernels before it
    unsigned int*  error;
};

// DIRECT_WORKER: one worker an item.  DIRECT_BLOCK: the warps of a block share an item's key tiles out among
// themselves and join what they have in shared memory.
enum { DIRECT_NO = 0, DIRECT_WORKER = 1, DIRECT_BLOCK = 2 };

// Programmatic dependent launch between the kernels of one call (pdl.h).  A kernel starts when the one before it
// has let it; what it may touch then is another matter:
//   ORDER_PLAIN  lets the next one start at once and waits for the kernels before it
//   ORDER_FIRST  waits, then lets the next one start: whoever starts after it finds the call's inputs ready
//   ORDER_LATE   needs nothing of the kernel before it but a prefix's result, if that: it waits before it reads
//                that, and before it ends (the kernel behind it waits for this one alone)
enum { ORDER_PLAIN = 0, ORDER_FIRST = 1, ORDER_LATE = 2 };
__device__ __forceinline__ void begin_order(paged_params_t const& p)
{
    if (p.order != ORDER_FIRST) asm volatile("griddepcontrol.launch_dependents;");
    if (p.order != ORDER_LATE) ES_PDL_WAIT();
    if (p.order == ORDER_FIRST) asm volatile("griddepcontrol.launch_dependents;");
}
__device__ __forceinline__ void wait_for_base(paged_params_t const& p)
{
    if (p.order == ORDER_LATE) ES_PDL_WAIT();
}

__device__ __forceinline__ void report(paged_params_t const& p, unsigned code)
{
    atomicMax(p.error, code); // a wait that expired (0x31..) passes what the arrays hold (0x21..)
}

struct sequence_t {
    int32_t        n;    // rows in this call (0: not this kernel's)
    int32_t        len;  // tokens in the cache
    int32_t        row0; // its first row
    int32_t const* table;
};

// Rows that attend a prefix: up to where the last sequence ends.  When the offsets are wrong (some sequence ends behind
// that, or it lies outside the tensors) all rows there are, as the good sequences may lie anywhere among them.  All
// threads of the block call.
__device__ __forceinline__ uint32_t prefix_rows(paged_params_t const& p)
{
    if (!p.row_offsets) return p.rows;
    int const end = p.row_offsets[p.batch];
    bool      ok = end >= 0 && end <= (int)p.rows;
    for (uint32_t i = threadIdx.x; i < p.batch; i += blockDim.x) ok = ok && p.row_offsets[i] <= end;
    if (__syncthreads_and(ok)) return (uint32_t)end;
    if (threadIdx.x == 0) report(p, PAGED_BAD_ROWS);
    return p.rows;
}

// rows: of a prefix (prefix_rows)
__device__ __forceinline__ sequence_t get_sequence(paged_params_t const& p, uint32_t i, uint32_t rows = 0)
{
    sequence_t s;
    if (p.prefix_len >= 0) {
        s.n = (int)rows;
        s.len = p.prefix_len;
        s.row0 = 0;
        s.table = p.tables;
    } else {
        s.len = p.lengths[i];
        if (s.len < 0 || (uint32_t)s.len > p.capacity) {
            report(p, PAGED_BAD_LENGTH);
            s.len = 0;
        }
        s.row0 = (int)i;
        s.n = 1;
        if (p.row_offsets) {
            int const a = p.row_offsets[i], b = p.row_offsets[i + 1];
            s.row0 = a;
            s.n = b - a;
            if (a < 0 || b < a || b > (int)p.rows) {
                report(p, PAGED_BAD_ROWS);
                s.n = 0;
            }
        }
        s.table = p.tables + (uint64_t)i * p.table_stride;
    }
    uint32_t const packed = (uint32_t)s.n * p.group; // < 2^31 (checked by the host)
    if (packed <= p.packed_min || packed > p.packed_max) s.n = 0;
    return s;
}

// keys that token `tok` of the sequence's rows may see
__device__ __forceinline__ int visible(paged_params_t const& p, sequence_t const& s, int tok)
{
    return p.causal ? max(0, min(s.len, s.len - s.n + tok + 1)) : s.len;
}

// units of the sequence's row tile t: the key tiles that its last token sees, one at least, and OVH in front
template <int TR, int BK, int OVH> __device__ __forceinline__ uint32_t tile_units(paged_params_t const& p, sequence_t const& s, uint32_t t)
{
    uint32_t const last = min((t + 1) * TR, (uint32_t)s.n * p.group) - 1;
    uint32_t const keys = (uint32_t)visible(p, s, (int)fdivide(last, p.grp));
    return max(1u, (keys + BK - 1) / BK + (p.front + BK - 1) / BK) + OVH;
}
template <int TR> __device__ __forceinline__ uint32_t row_tiles(paged_params_t const& p, sequence_t const& s)
{
    return ((uint32_t)s.n * p.group + TR - 1) / TR;
}

// Units of one head of the lane's sequence.  Causal parts of several tokens have row tiles of different
// length: those are summed by the whole warp, one lane's sequence after the other.  All 32 lanes call.
template <int TR, int BK, int OVH> __device__ __forceinline__ uint64_t head_units(paged_params_t const& p, sequence_t const& s)
{
    uint64_t   u = 0;
    bool const even = s.n <= 1 || !p.causal;
    if (s.n > 0 && even) u = (uint64_t)row_tiles<TR>(p, s) * tile_units<TR, BK, OVH>(p, s, 0);
    unsigned todo = __ballot_sync(0xffffffffu, s.n > 0 && !even);
    int const lane = threadIdx.x & 31;
    while (todo) {
        int const  src = __ffs(todo) - 1;
        sequence_t o;
        o.n = __shfl_sync(0xffffffffu, s.n, src);
        o.len = __shfl_sync(0xffffffffu, s.len, src);
        uint32_t const rt = row_tiles<TR>(p, o);
        uint64_t       sum = 0;
        for (uint32_t t = lane; t < rt; t += 32) sum += tile_units<TR, BK, OVH>(p, o, t);
#pragma unroll
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == src) u = sum;
        todo &= todo - 1;
    }
    return u;
}

// A worker's place in the work
struct work_t {
    uint32_t   seq, head, t, rt;
    uint32_t   j, kt;   // next unit of the item, number of its units
    uint32_t   left;    // units of this worker's share still to do
    uint64_t   unit;    // number of the next unit
    uint32_t   chunk;   // units a share
    uint32_t   worker;
    sequence_t s;
};

template <int NT, int WPB> struct sched_smem_t {
    uint64_t warp_sum[NT / 32];
    uint64_t found_off[WPB];
    uint32_t found_seq[WPB];
};

// All NT threads call.  WPB workers a block: 1, or its NT / 32 warps.
template <int TR, int BK, int OVH, int NT, int WPB>
__device__ __forceinline__ void find_work(paged_params_t const& p, work_t& w, sched_smem_t<NT, WPB>& sm)
{
    static_assert(WPB == 1 || WPB == NT / 32, "a worker is a block or a warp");
    int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int const mine_in_block = WPB == 1 ? 0 : warp;
    w.worker = blockIdx.x * WPB + mine_in_block;
    uint32_t const n_seq = p.prefix_len >= 0 ? 1u : p.batch;
    w.left = 0;
    w.j = 0;
    w.unit = 0;
    w.chunk = 0xffffffffu;
    if (p.direct) {
        // one row a sequence: blocks (items of a sequence, sequences); nothing to count
        w.rt = (p.group + TR - 1) / TR;
        w.head = p.direct == DIRECT_BLOCK ? blockIdx.x : w.worker;
        w.t = 0;
        if (w.rt > 1) {
            uint32_t const item = w.head;
            w.head = item / w.rt;
            w.t = item - w.head * w.rt;
        }
        w.seq = blockIdx.y;
        w.s.n = 0;
        if (w.head >= p.kv_heads) return;
        w.s = get_sequence(p, w.seq);
        if (w.s.n == 0) return;
        w.kt = tile_units<TR, BK, OVH>(p, w.s, w.t);
        w.left = w.kt;
        if (p.direct == DIRECT_BLOCK) { // this warp's part of the tiles
            uint32_t const tiles = w.kt - OVH, from = tiles * warp / (NT / 32);
            w.j = OVH + from;
            w.left = tiles * (warp + 1) / (NT / 32) - from;
        }
        return;
    }
    uint32_t const rows = p.prefix_len >= 0 ? prefix_rows(p) : 0;
    uint64_t       mine = 0, u0 = 0;
    for (uint32_t i0 = 0; i0 < n_seq; i0 += NT) {
        sequence_t s;
        s.n = 0;
        s.len = 0;
        if (i0 + threadIdx.x < n_seq) s = get_sequence(p, i0 + threadIdx.x, rows);
        u0 = head_units<TR, BK, OVH>(p, s) * p.kv_heads;
        mine += u0;
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, x);
    if (lane == 0) sm.warp_sum[warp] = mine;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) total += sm.warp_sum[i];
    __syncthreads();
    uint64_t const share = max((total + gridDim.x * WPB - 1) / (gridDim.x * WPB), (uint64_t)p.min_units);
    w.chunk = (uint32_t)min(share, (uint64_t)0xffffffffu);
    uint64_t const lo0 = (uint64_t)blockIdx.x * WPB * w.chunk; // the block's first worker's first unit
    if (lo0 >= total) return;                                  // (the block has no work)
    uint64_t const lo = lo0 + (uint64_t)mine_in_block * w.chunk;
    uint64_t const lo_last = min(lo0 + (uint64_t)(WPB - 1) * w.chunk, total - 1);
    // the sequences that hold the workers' first units
    uint64_t base = 0;
    for (uint32_t i0 = 0; i0 < n_seq; i0 += NT) {
        uint64_t u = u0;
        if (n_seq > NT) {
            sequence_t s;
            s.n = 0;
            s.len = 0;
            if (i0 + threadIdx.x < n_seq) s = get_sequence(p, i0 + threadIdx.x, rows);
            u = head_units<TR, BK, OVH>(p, s) * p.kv_heads;
        }
        uint64_t incl = u;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            uint64_t const o = __shfl_up_sync(0xffffffffu, incl, x);
            if (lane >= x) incl += o;
        }
        if (lane == 31) sm.warp_sum[warp] = incl;
        __syncthreads();
        uint64_t before = base, all = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) {
            if (i < warp) before += sm.warp_sum[i];
            all += sm.warp_sum[i];
        }
        incl += before;
#pragma unroll
        for (int x = 0; x < WPB; ++x) {
            uint64_t const first = lo0 + (uint64_t)x * w.chunk;
            if (first < incl && first >= incl - u) {
                sm.found_seq[x] = i0 + threadIdx.x;
                sm.found_off[x] = first - (incl - u);
            }
        }
        base += all;
        __syncthreads();
        if (lo_last < base) break; // (the same in the whole block)
    }
    if (lo >= total) return; // this warp has no work
    w.unit = lo;
    w.left = (uint32_t)min((uint64_t)w.chunk, total - lo);
    w.seq = sm.found_seq[mine_in_block];
    uint64_t off = sm.found_off[mine_in_block];
    w.s = get_sequence(p, w.seq, rows);
    uint64_t const per_head = head_units<TR, BK, OVH>(p, w.s); // every lane of every warp has the same sequence
    w.head = (uint32_t)(off / per_head);
    off -= w.head * per_head;
    w.rt = row_tiles<TR>(p, w.s);
    if (w.s.n <= 1 || !p.causal) {
        w.kt = tile_units<TR, BK, OVH>(p, w.s, 0);
        w.t = (uint32_t)(off / w.kt);
        w.j = (uint32_t)(off - (uint64_t)w.t * w.kt);
        return;
    }
    for (uint32_t t0 = 0;; t0 += 32) {
        uint32_t const t = t0 + lane;
        uint64_t const u = t < w.rt ? tile_units<TR, BK, OVH>(p, w.s, t) : 0;
        uint64_t       incl = u;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            uint64_t const o = __shfl_up_sync(0xffffffffu, incl, x);
            if (lane >= x) incl += o;
        }
        unsigned const hit = __ballot_sync(0xffffffffu, off < incl);
        if (hit) {
            int const src = __ffs(hit) - 1;
            w.t = t0 + src;
            w.kt = (uint32_t)__shfl_sync(0xffffffffu, u, src);
            w.j = (uint32_t)(off - __shfl_sync(0xffffffffu, incl - u, src));
            return;
        }
        off -= __shfl_sync(0xffffffffu, incl, 31);
    }
}

// The next item, after `done` units of this one
template <int TR, int BK, int OVH> __device__ __forceinline__ void next_item(paged_params_t const& p, work_t& w, uint32_t done)
{
    w.left -= done;
    w.unit += done;
    w.j = 0;
    if (w.left == 0) return;
    if (++w.t == w.rt) {
        w.t = 0;
        if (++w.head == p.kv_heads) {
            w.head = 0;
            do { // (units are left, so a sequence with some follows -- unless the arrays changed meanwhile)
                if (++w.seq >= p.batch || p.prefix_len >= 0) {
                    w.left = 0;
                    return;
                }
                w.s = get_sequence(p, w.seq);
            } while (w.s.n == 0);
            w.rt = row_tiles<TR>(p, w.s);
        }
    }
    w.kt = tile_units<TR, BK, OVH>(p, w.s, w.t);
}

// Key tiles [first, end) among the item's units [j, j + n)
template <int OVH> __device__ __forceinline__ uint32_t first_tile_of(uint32_t j)
{
    return j > OVH ? j - OVH : 0u;
}
// Moves over units that stand for no tile; false: the share ends among them
template <int OVH> __device__ __forceinline__ bool to_next_tile(work_t& w)
{
    if (w.j < OVH) {
        uint32_t const n = min(OVH - w.j, w.left);
        w.j += n;
        w.left -= n;
    }
    return w.left != 0;
}

// Where a segment's result goes: -1 finished here, 0 / 1 the worker's first / last partial result
__device__ __forceinline__ int segment_slot(work_t const& w, uint32_t n)
{
    if (w.j == 0 && n == w.kt) return -1;
    return w.j == 0 ? 1 : 0;
}

// Every worker says whether its last item goes on in the following shares (one thread)
template <int TR>
__device__ __forceinline__ void write_meta(paged_params_t const& p, work_t const& w, bool split)
{
    int4* m = p.meta + 2 * (uint64_t)w.worker;
    if (!split) {
        m[0] = make_int4(0, 0, 0, 0);
        return;
    }
    uint32_t const start = w.t * TR;
    uint32_t const count = min((uint32_t)TR, (uint32_t)w.s.n * p.group - start);
    uint64_t const last = w.unit + w.kt - 1; // unit numbers: w.unit is the item's first
    m[0] = make_int4((int)count, w.s.row0, (int)start, (int)w.head);
    m[1] = make_int4((int)(last / w.chunk), 0, 0, 0);
}

// The weights that turn an unnormalised sum (reference point m in log2 units, sum of exponentials l) and,
// where there is one, the prefix's normalised result (natural log lse) into the result:
// out = wa * sum + wb * prefix.  No key at all: both weights 0, lse -inf.  Without a prefix wb is 0 whatever the
// scores were: a weight that is not 0 is what lets the prefix's result be read.
struct finish_t {
    float wa, wb, lse;
};
__device__ __forceinline__ finish_t finish(float m, float l, bool has_base, float base_lse)
{
    finish_t    f;
    float const b2 = has_base ? base_lse * LOG2_E : -INFINITY;
    float const top = fmaxf(l == 0.f ? -INFINITY : m, b2);
    if (l == 0.f && b2 == -INFINITY) {
        f.wa = f.wb = 0.f;
        f.lse = -INFINITY;
        return f;
    }
    // (the hardware's 2^x, log2 and reciprocal: a few steps of 2^-23)
    float const a = l == 0.f ? 0.f : ex2(m - top);
    float const b = b2 == -INFINITY ? 0.f : ex2(b2 - top);
    float const total = fmaf(l, a, b), inv = __fdividef(1.f, total);
    f.wa = a * inv;
    f.wb = has_base ? b * inv : 0.f; // (0 * inv may be NaN, and there is nothing to read)
    f.lse = (top + __log2f(total)) * LN_2;
    return f;
}

// W consecutive elements (4; of f16 also 2) of a finished row
template <typename T, int W>
__device__ __forceinline__ void write_out(paged_params_t const& p, int row, uint32_t head, uint32_t e, float const (&o)[W],
                                          finish_t const& f, bool aligned)
{
    float r[W];
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = f.wa == 0.f ? 0.f : o[i] * f.wa; // a weight of 0: the sum may be anything
    if (p.base_out && f.wb != 0.f) {
        float const* b = p.base_out + ((uint64_t)row * p.heads + head) * p.d + e;
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (e + i < p.d) r[i] = fmaf(b[i], f.wb, r[i]);
    }
    if (p.out_f32) {
        float* d = static_cast<float*>(p.out) + ((uint64_t)row * p.heads + head) * p.d + e;
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (e + i < p.d) d[i] = r[i];
        return;
    }
    T* d = static_cast<T*>(p.out) + (int64_t)row * p.out_stride[0] + (int64_t)head * p.out_stride[1] + e;
    if (aligned && e + W <= p.d) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(d) = make_float4(r[0], r[1], r[2], r[3]);
        } else {
            if constexpr (W == 4) {
                __half2 const a = __floats2half2_rn(r[0], r[1]), b = __floats2half2_rn(r[2], r[3]);
                *reinterpret_cast<uint2*>(d) = make_uint2(*reinterpret_cast<uint32_t const*>(&a), *reinterpret_cast<uint32_t const*>(&b));
            } else {
                *reinterpret_cast<__half2*>(d) = __floats2half2_rn(r[0], r[1]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (e + i < p.d) from_f32(d[i], r[i]);
}

// Joins the partial results of the items that crossed shares.  Block x: the item that starts last in share x
// (if it goes on behind it); block y: 16 rows of it.  A warp takes a row, or with fewer rows than warps every
// SLICES-th part of one; lanes over the head dim.  The parts' weights are found 32 at a time, a lane a part, so
// that the loads of the parts' sums wait for nothing but each other.
template <typename T, int TR, int CHUNKS> // CHUNKS: of 128 elements of the head dim
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ paged_params_t p, int aligned)
{
    constexpr uint32_t WARPS = 8;
    constexpr int      BATCH = 8 / CHUNKS;
    __shared__ float   so[WARPS][CHUNKS * 128];
    __shared__ float2  sml[WARPS];
    ES_PDL_PROLOGUE();
    int4 const     m0 = p.meta[2 * blockIdx.x], m1 = p.meta[2 * blockIdx.x + 1]; // (m1 means something if m0.x > 0)
    uint32_t const r0 = blockIdx.y * 16;
    if (r0 >= (uint32_t)m0.x) return;
    int const      first = (int)blockIdx.x, n = m1.x - first + 1;
    uint32_t const rows = min((uint32_t)m0.x - r0, 16u), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t const at_once = min(rows, WARPS), slices = WARPS / at_once, slice = warp / at_once;
    for (uint32_t rr = 0; rr < rows; rr += at_once) {
        uint32_t const r = r0 + rr + warp % at_once;
        bool const     on = slice < slices && r < r0 + rows;
        // part i lies in share first + i: its last slot for i = 0, the first slot of the others
        auto  slot = [&](int i) { return (uint64_t)(2 * (first + i) + (i == 0 ? 1 : 0)) * TR + r; };
        float top = -INFINITY, l = 0.f, o[CHUNKS][4] = {};
        if (on) {
            for (int i0 = (int)slice * 32; i0 < n; i0 += (int)slices * 32) {
                int const    i = i0 + (int)lane, here = min(32, n - i0);
                float4       x[BATCH][CHUNKS];
                auto         fetch = [&](int k0) { // (parts beyond the last: weight 0)
#pragma unroll
                    for (int k = 0; k < BATCH; ++k) {
                        float const* src = p.part_out + slot(i0 + min(k0 + k, here - 1)) * p.part_d;
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c)
                            if (c * 128 + lane * 4 < p.part_d) x[k][c] = *reinterpret_cast<float4 const*>(src + c * 128 + lane * 4);
                    }
                };
                fetch(0);
                float2 const ml = i < n ? p.part_ml[slot(i)] : make_float2(-INFINITY, 0.f);
                float        tm = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
                for (int x = 16; x; x >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, x));
                if (tm > top) {
                    float const a = ex2(top - tm); // top = -inf: 0
                    l *= a;
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[c][k] *= a;
                    top = tm;
                }
                float const wgt = ml.y == 0.f ? 0.f : ex2(ml.x - (top == -INFINITY ? 0.f : top));
                float       ls = ml.y * wgt;
#pragma unroll
                for (int x = 16; x; x >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, x);
                l += ls;
                for (int k0 = 0; k0 < here; k0 += BATCH) {
                    if (k0) fetch(k0);
#pragma unroll
                    for (int k = 0; k < BATCH; ++k) {
                        float const wk = __shfl_sync(0xffffffffu, wgt, k0 + k);
                        if (k0 + k < here) {
#pragma unroll
                            for (int c = 0; c < CHUNKS; ++c) {
                                o[c][0] = fmaf(x[k][c].x, wk, o[c][0]);
                                o[c][1] = fmaf(x[k][c].y, wk, o[c][1]);
                                o[c][2] = fmaf(x[k][c].z, wk, o[c][2]);
                                o[c][3] = fmaf(x[k][c].w, wk, o[c][3]);
                            }
                        }
                    }
                }
            }
        }
        if (slices > 1) { // (the same in the whole block; then all rows are done in this one round)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) *reinterpret_cast<float4*>(&so[warp][c * 128 + lane * 4]) = make_float4(o[c][0], o[c][1], o[c][2], o[c][3]);
            if (lane == 0) sml[warp] = make_float2(top, l);
            __syncthreads();
            if (warp >= at_once) return;
            float all = -INFINITY;
            for (uint32_t x = 0; x < slices; ++x)
                if (sml[warp + x * at_once].y != 0.f) all = fmaxf(all, sml[warp + x * at_once].x);
            float sum[CHUNKS][4] = {};
            l = 0.f;
            for (uint32_t x = 0; x < slices; ++x) {
                float2 const ml = sml[warp + x * at_once];
                if (ml.y == 0.f) continue;
                float const wgt = ex2(ml.x - (all == -INFINITY ? 0.f : all));
                l = fmaf(ml.y, wgt, l);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k) sum[c][k] = fmaf(so[warp + x * at_once][c * 128 + lane * 4 + k], wgt, sum[c][k]);
            }
            top = all;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[c][k] = sum[c][k];
        }
        if (!on) continue;
        uint32_t const pr = (uint32_t)m0.z + r;
        uint32_t const tok = fdivide(pr, p.grp);
        int const      row = m0.y + (int)tok;
        uint32_t const head = (uint32_t)m0.w * p.group + (pr - tok * p.group);
        uint64_t const at = (uint64_t)row * p.heads + head;
        finish_t const f = finish(top, l, p.base_lse != nullptr, p.base_lse ? p.base_lse[at] : 0.f);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            uint32_t const e = c * 128 + lane * 4;
            if (e < p.d) write_out<T, 4>(p, row, head, e, o[c], f, aligned != 0);
        }
        if (p.lse && lane == 0) p.lse[at] = f.lse;
    }
}

} // namespace
} // namespace es
