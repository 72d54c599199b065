// What the kernels of the paged attention share: how the work is cut up, and how partial results are kept and added up.
//
// The work is all blocks of 128 keys of all tiles of all (sequence, kv head)s, laid out behind one another; every CTA gets an
// equal, contiguous share of it, cut anywhere.  Each finds its share from starts and lens (pg_find_share), so that lengths live
// on the device and a captured call serves others.  A tile that is cut leaves partial sums (O, maximum, sum) in the scratch, and
// a second launch adds them up in a fixed order: the same bits every time.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "kernels.h"

namespace eet {

namespace {

constexpr int kPgRows = 128;            // rows of a tile (paged_tc.cu)
constexpr int kPgKeys = 128;            // keys of a block

// Powers are taken under a reference that may stay behind a row's maximum by kPgLag (in powers of two).  The probabilities enter the product
// as T: in fp16 they are held 2^kUp higher, so that they end at 2^15 and what lies down to 2^-21 of the largest is a normal value, to 2^-32
// counts at all (without it 2^-14 and 2^-25: 20000 keys at 2^-26 of one other were lost, 3e-4 of the result).  The sums are of the same
// powers, so nothing else knows.
constexpr float kPgLag = 8.0f;
constexpr float kPgNone = -3.402823466e38f;   // maximum and reference of a row that has seen nothing: no finite score lies below

template<typename T>
struct PgType;
template<>
struct PgType<__half> {
    static constexpr float kUp = 7.0f;
    static constexpr uint32_t idesc = 0;
    static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template<>
struct PgType<__nv_bfloat16> {
    static constexpr float kUp = 0.0f;
    static constexpr uint32_t idesc = (1u << 7) | (1u << 10);
    static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

// ------------------------------------------------------------------------------------------------ the shares of the work

struct PgSeq {
    int row0, tokens;   // rows of q
    int p0;             // position of the first of them
    int first;          // first position that counts
};

// What a kernel works on: sequences with `least` to `most` new tokens, `tokens` of them to a tile (both tiles of a pair counted).
// A tile counts as `extra` blocks more than it has: what its beginning and end cost.  These stand before its first block; a share
// that ends within them leaves the tile to the next.
struct PgTiling {
    int tokens, least, most, extra;
    __device__ __forceinline__ int tiles(const PgSeq& s) const { return (s.tokens + tokens - 1) / tokens; }
};

// Rows [row0, end) of q as far as they exist (`tokens` of them do), whatever starts holds: no difference is taken that could overflow.
constexpr __host__ __device__ int pg_rows_of(int row0, int end, int tokens)
{
    const int to = end < tokens ? end : tokens;
    return row0 >= 0 && to > row0 ? to - row0 : 0;
}

__device__ __forceinline__ PgSeq pg_seq(const PagedMhaArgs& a, const PgTiling& g, int b)
{
    PgSeq s;
    s.row0 = a.starts[b];
    const int end = a.starts[b + 1];
    s.tokens = pg_rows_of(s.row0, end, a.tokens);
    s.p0 = max(a.lens[b], 0) - (s.tokens > 0 ? end - s.row0 : 0);
    if (s.tokens < g.least || s.tokens > g.most) s.tokens = 0;
    s.first = a.first_key != nullptr ? max(0, a.first_key[b]) : 0;
    return s;
}

// The key blocks of tile t: keys [lo, hi) are seen by some row of it.
struct PgSpan {
    int lo, hi;
    __device__ __forceinline__ int first_block() const { return lo / kPgKeys; }
    __device__ __forceinline__ int blocks() const { return hi > lo ? (hi + kPgKeys - 1) / kPgKeys - lo / kPgKeys : 0; }
};

__device__ __forceinline__ PgSpan pg_span(const PagedMhaArgs& a, const PgSeq& s, int token0, int token1)
{
    PgSpan r;
    const long long cap = (long long)a.max_pages << a.page_shift;
    r.hi = (int)min((long long)s.p0 + min(token1, s.tokens), cap);
    r.lo = s.first;
    if (a.window > 0) r.lo = (int)max((long long)r.lo, (long long)s.p0 + token0 - a.window + 1);
    return r;
}

// (The newest keys first: with ALiBi, and mostly without, the largest scores are there, and the reference of the powers stays
// where the first block puts it.  Oldest first it moved with every block of a head with a steep slope.)
struct PgPiece {
    PgSeq s;
    int seq, head, tile;
    int top, blocks;      // key blocks top, top - 1, .. of it to be worked on; 0: its rows see nothing
    bool starts, ends;    // whether those begin with its first, end with its last
};

// Walks the share of a CTA tile by tile.  All threads of a warp hold the same.
struct PgShare {
    long long left;       // of the share still to come, in blocks
    int seq, head, tile, at;
    PgSeq s;
    bool whole;           // tiles are not cut: the share has those that begin in it

    __device__ __forceinline__ void step(const PagedMhaArgs& a, const PgTiling& g)
    {
        at = 0;
        if (++tile < g.tiles(s)) return;
        tile = 0;
        if (++head < a.kv_heads) return;
        head = 0;
        for (;;) {
            if (++seq >= a.seqs) {
                left = 0;
                return;
            }
            s = pg_seq(a, g, seq);
            if (s.tokens > 0) return;
            // Not one for this kernel; there may be many of them (slots without a sequence, single tokens around a chunk), so eight
            // are looked at with one trip to memory (single tokens in the first and last of 300 slots: 31 us one by one, 21 so).
            bool none = true;
            while (none && seq + 1 < a.seqs) {
                int found = 8;
#pragma unroll
                for (int i = 7; i >= 0; --i) {
                    if (pg_seq(a, g, min(seq + 1 + i, a.seqs - 1)).tokens > 0) found = i;
                }
                none = found == 8;
                seq += found;
            }
        }
    }
    __device__ __forceinline__ bool next(const PagedMhaArgs& a, const PgTiling& g, PgPiece& p)
    {
        while (left > 0) {
            const PgSpan span = pg_span(a, s, tile * g.tokens, (tile + 1) * g.tokens);
            const int n = span.blocks(), cost = n + g.extra;
            if (whole && at > 0) {   // it began in the share before
                left -= cost - at;
                step(a, g);
                continue;
            }
            const int take = whole ? cost : (int)min(left, (long long)(cost - at));
            const int from = max(0, at - g.extra), to = max(0, at + take - g.extra);
            p.s = s;
            p.seq = seq;
            p.head = head;
            p.tile = tile;
            p.top = span.first_block() + to - 1;
            p.blocks = to - from;
            p.starts = from == 0;
            p.ends = at + take == cost;
            left -= take;
            at += take;
            if (p.ends && left > 0) step(a, g);
            if (p.blocks > 0 || n == 0 && p.ends) return true;
        }
        return false;
    }
};

__device__ __forceinline__ long long pg_warp_scan(long long v)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// Blocks of all tiles of a kv head of the sequences that the lanes of a warp hold.  One with many tiles is added up by the warp.
__device__ __forceinline__ long long pg_seq_blocks(const PagedMhaArgs& a, const PgTiling& g, const PgSeq& mine)
{
    const int tiles = g.tiles(mine);
    long long sum = 0;
    if (tiles <= 4) {
        for (int t = 0; t < tiles; ++t) sum += pg_span(a, mine, t * g.tokens, (t + 1) * g.tokens).blocks() + g.extra;
    }
    uint32_t many = __ballot_sync(0xffffffffu, tiles > 4);
    while (many) {
        const int src = __ffs(many) - 1;
        many &= many - 1;
        PgSeq s;
        s.row0 = 0;
        s.tokens = __shfl_sync(0xffffffffu, mine.tokens, src);
        s.p0 = __shfl_sync(0xffffffffu, mine.p0, src);
        s.first = __shfl_sync(0xffffffffu, mine.first, src);
        const int n = g.tiles(s);
        long long part = 0;
        for (int t = threadIdx.x & 31; t < n; t += 32) part += pg_span(a, s, t * g.tokens, (t + 1) * g.tokens).blocks() + g.extra;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if ((int)(threadIdx.x & 31) == src) sum = part;
    }
    return sum;
}

// Kernels this short spend much of their time on what runs once - the first fetch of every instruction among it - so what follows
// is kept small: no 64-bit divisions, no barrier where a warp has a lane for each sequence.
constexpr int kPgMostWarps = 16;   // of a block of any of the kernels

struct PgFound {           // by the block together, where it takes more
    long long warp_sum[kPgMostWarps];
    long long rest, per_head;
    PgSeq s;
    int seq;
};

// What the header of a share goes by: blocks in all, and where the share begins.
struct PgPlace {
    long long total, begin;
};

// CTA c's share of `total` blocks begins at q c + min(c, r), with total = q ctas + r.
struct PgCut {
    long long q;
    int r;
    __device__ __forceinline__ PgCut(long long total, int ctas)
    {
        q = total >> 32 ? total / ctas : (long long)((uint32_t)total / (uint32_t)ctas);
        r = (int)(total - q * ctas);
    }
    __device__ __forceinline__ long long begin(int cta) const { return q * cta + min(cta, r); }
    // the CTA whose share holds block x
    __device__ __forceinline__ int of(long long x) const
    {
        const long long large = (q + 1) * r;
        const long long y = x < large ? x : x - large, d = x < large ? q + 1 : q;
        return (x < large ? 0 : r) + (int)(y >> 32 ? y / d : (long long)((uint32_t)y / (uint32_t)d));
    }
};

// Blocks in all, by every warp.
__device__ __forceinline__ long long pg_total(const PagedMhaArgs& a, const PgTiling& g)
{
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    for (int base = 0; base < a.seqs; base += 32) {
        PgSeq s = {0, 0, 0, 0};
        if (base + lane < a.seqs) s = pg_seq(a, g, base + lane);
        sum += pg_seq_blocks(a, g, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return a.kv_heads * sum;
}

__device__ __forceinline__ int pg_div(long long x, long long d)
{
    return (x | d) >> 32 ? (int)(x / d) : (int)((uint32_t)x / (uint32_t)d);
}

// The share of CTA `cta` of `ctas`, found by every warp of the block; false: it has none.
__device__ __forceinline__ bool pg_find_share(const PagedMhaArgs& a, const PgTiling& g, int cta, int ctas, bool whole, PgFound& f,
                                              PgShare& share, PgPlace& place)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5, threads = blockDim.x;
    long long rest, per_head;    // from the begin of the share's first sequence to the share's; blocks of a kv head of that sequence
    if (a.seqs <= 32) {
        PgSeq s = {0, 0, 0, 0};
        if (lane < a.seqs) s = pg_seq(a, g, lane);
        per_head = pg_seq_blocks(a, g, s);
        const long long cost = a.kv_heads * per_head, upto = pg_warp_scan(cost);
        place.total = __shfl_sync(0xffffffffu, upto, 31);
        const PgCut cut(place.total, ctas);
        place.begin = cut.begin(cta);
        share.left = cut.begin(cta + 1) - place.begin;
        if (share.left == 0) return false;
        share.seq = __ffs(__ballot_sync(0xffffffffu, upto - cost <= place.begin && place.begin < upto)) - 1;
        rest = place.begin - __shfl_sync(0xffffffffu, upto - cost, share.seq);
        per_head = __shfl_sync(0xffffffffu, per_head, share.seq);
        share.s.row0 = __shfl_sync(0xffffffffu, s.row0, share.seq);
        share.s.tokens = __shfl_sync(0xffffffffu, s.tokens, share.seq);
        share.s.p0 = __shfl_sync(0xffffffffu, s.p0, share.seq);
        share.s.first = __shfl_sync(0xffffffffu, s.first, share.seq);
    }
    else {
        const bool once = a.seqs <= threads;
        place.total = place.begin = 0;
        for (int pass = once; pass < 2; ++pass) {   // the first pass adds up, the second (or only) one looks for the share's begin
            long long before = 0;                   // of the sequences of earlier rounds
            for (int base = 0; base < a.seqs; base += threads) {
                PgSeq s = {0, 0, 0, 0};
                if (base + tid < a.seqs) s = pg_seq(a, g, base + tid);
                per_head = pg_seq_blocks(a, g, s);
                const long long cost = a.kv_heads * per_head, upto = pg_warp_scan(cost);
                if (lane == 31) f.warp_sum[warp] = upto;
                __syncthreads();
                long long end = before + upto;
                for (int w = 0; w < warps; ++w) {
                    if (w < warp) end += f.warp_sum[w];
                    before += f.warp_sum[w];
                }
                if (once) place.total = before;
                if (pass == 1) {
                    place.begin = PgCut(place.total, ctas).begin(cta);
                    if (end - cost <= place.begin && place.begin < end) {
                        f.rest = place.begin - (end - cost);
                        f.per_head = per_head;
                        f.s = s;
                        f.seq = base + tid;
                    }
                }
                __syncthreads();
            }
            place.total = before;
        }
        share.left = PgCut(place.total, ctas).begin(cta + 1) - place.begin;
        if (share.left == 0) return false;
        rest = f.rest;
        per_head = f.per_head;
        share.s = f.s;
        share.seq = f.seq;
    }
    share.whole = whole;
    share.head = pg_div(rest, per_head);
    rest -= share.head * per_head;
    share.tile = 0;
    const int tiles = g.tiles(share.s);
    if (tiles > 1) {
        for (int t0 = 0;; t0 += 32) {
            const int t = t0 + lane;
            const long long cost = t < tiles ? pg_span(a, share.s, t * g.tokens, (t + 1) * g.tokens).blocks() + g.extra : 0;
            const long long upto = pg_warp_scan(cost), all = __shfl_sync(0xffffffffu, upto, 31);
            if (rest < all || t0 + 32 >= tiles) {
                const int src = __ffs(__ballot_sync(0xffffffffu, upto - cost <= rest && rest < upto)) - 1;
                share.tile = t0 + src;
                rest -= __shfl_sync(0xffffffffu, upto - cost, src);
                break;
            }
            rest -= all;
        }
    }
    share.at = (int)rest;
    return true;
}

// ------------------------------------------------------------------------------------------------ scratch
// Per CTA a header of the piece that it begins with, and two partial results: of that piece where it continues a tile (0), and
// of the piece that it ends with where that begins a tile and does not end it (1).  A partial result of R rows: the maximum (as a
// power of two) and the sum of each, and O as float4 [R][D / 4], or for the 256 rows of a pair of tiles as [D / 4][R].
struct PgHeader {
    int kind;              // 0: nothing to add up; 1: the piece ends a tile that began in CTA `from`; 2: it neither begins nor ends one
    int from;
    int head;              // kv head
    int row0, tokens;      // of q: of the tile
    int pad[3];
};

__host__ __device__ constexpr size_t pg_partial_bytes(int rows, int head_dim)
{
    return (size_t)rows * (2 + head_dim) * sizeof(float);
}

__host__ __device__ constexpr size_t pg_scratch_bytes(int ctas, int rows, int head_dim)
{
    return ctas * (sizeof(PgHeader) + 2 * pg_partial_bytes(rows, head_dim));
}

struct PgPartial {
    float *max2, *sum;
    float4* o;
};

__device__ __forceinline__ PgPartial pg_partial(void* ws, int ctas, int cta, int which, int rows, int head_dim)
{
    float* at = reinterpret_cast<float*>((char*)ws + ctas * sizeof(PgHeader) + (2 * (size_t)cta + which) * pg_partial_bytes(rows, head_dim));
    return {at, at + rows, reinterpret_cast<float4*>(at + 2 * rows)};
}

// The header of a CTA's share (as pg_find_share left it), written by one thread that has time for the divisions.
__device__ __forceinline__ void pg_write_header(const PagedMhaArgs& a, const PgTiling& g, void* ws, int cta, int ctas, bool work,
                                                const PgShare& share, const PgPlace& place)
{
    PgHeader h = {};
    if (work && share.at > g.extra) {
        const PgSpan span = pg_span(a, share.s, share.tile * g.tokens, (share.tile + 1) * g.tokens);
        h.kind = share.at + share.left >= span.blocks() + g.extra ? 1 : 2;
        h.from = PgCut(place.total, ctas).of(place.begin - share.at + g.extra);   // where its first block is
        h.head = share.head;
        h.row0 = share.s.row0 + share.tile * g.tokens;
        h.tokens = min(g.tokens, share.s.tokens - share.tile * g.tokens);
    }
    reinterpret_cast<PgHeader*>(ws)[cta] = h;
}

struct PgScratch {
    void* ws;
    int rows;              // of a partial result; 0: none
    int by_dim;            // O is [D / 4][rows], and a tile of 128 rows holds whole tokens only
    int ctas;              // that it is laid out for
};

// Adds up the partial results of the tiles that end in CTA blockIdx.x of one of the kernels (blockIdx.z), 8 dims of a row a
// thread and turn.  Bound: latency.  Two trips to L2, four parts on their way at once, and CTAs small enough (128 threads of 80
// registers) to be resident beside the first kernel's, so that they wait for its end in place.  With CTAs of 256 threads of 64 registers,
// which the 53760 of the 128-row kernel left no room for, and two passes over the parts: 16 x 5 tokens 39 us and not 36, the window
// 24.7 and not 22.4, 64 single tokens 93.7 and not 91.6.
constexpr int kPgJoinThreads = 128;

template<typename T, int D>
__global__ void __launch_bounds__(kPgJoinThreads, 6) paged_mha_join_kernel(const __grid_constant__ PagedMhaArgs a, PgScratch s0, PgScratch s1)
{
    constexpr int kAhead = 4;   // parts on their way
    pdl_wait();
    const PgScratch s = blockIdx.z ? s1 : s0;
    if ((int)blockIdx.x >= s.ctas) return;
    const PgHeader h = reinterpret_cast<const PgHeader*>(s.ws)[blockIdx.x];
    if (h.kind != 1) return;
    const int cta = blockIdx.x, ctas = s.ctas;
    const int group = a.heads / a.kv_heads;
    const int rows = h.tokens * group;
    const int per_tile = s.by_dim ? kPgRows / group * group : s.rows;   // rows of a tile in use
    for (int i = (int)(blockIdx.y * blockDim.x + threadIdx.x); i < rows * (D / 8); i += (int)(gridDim.y * blockDim.x)) {
        const int row = s.by_dim ? i % rows : i / (D / 8), d8 = s.by_dim ? i / rows : i % (D / 8);
        const int at = s.by_dim ? row / per_tile * kPgRows + row % per_tile : row;
        const size_t o_at = s.by_dim ? (size_t)(2 * d8) * s.rows + at : (size_t)at * (D / 4) + 2 * d8;
        const int o_step = s.by_dim ? s.rows : 1;
        float top = -INFINITY, sum = 0.f;
        float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int c0 = h.from; c0 <= cta; c0 += kAhead) {
            float l[kAhead], m[kAhead], next = top;
            float4 o[kAhead][2];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                l[k] = 0.f;
                if (c0 + k > cta) continue;
                const PgPartial p = pg_partial(s.ws, ctas, c0 + k, c0 + k == h.from ? 1 : 0, s.rows, D);
                l[k] = p.sum[at], m[k] = p.max2[at];
                o[k][0] = p.o[o_at], o[k][1] = p.o[o_at + o_step];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (l[k] != 0.f) next = fmaxf(next, m[k]);
            }
            const float keep = sum != 0.f ? ex2_approx(top - next) : 0.f;
            top = next;
            sum *= keep;
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[e] = make_float4(acc[e].x * keep, acc[e].y * keep, acc[e].z * keep, acc[e].w * keep);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (l[k] == 0.f) continue;   // (a piece that sees nothing has left no O)
                const float w = ex2_approx(m[k] - top);
                sum += l[k] * w;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    acc[e].x += o[k][e].x * w;
                    acc[e].y += o[k][e].y * w;
                    acc[e].z += o[k][e].z * w;
                    acc[e].w += o[k][e].w * w;
                }
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* dst = (T*)a.out + (size_t)(h.row0 + row / group) * a.o_tok + (size_t)(h.head * group + row % group) * a.o_head + 8 * d8;
        uint4 w;
        w.x = PgType<T>::pack(acc[0].x * inv, acc[0].y * inv);
        w.y = PgType<T>::pack(acc[0].z * inv, acc[0].w * inv);
        w.z = PgType<T>::pack(acc[1].x * inv, acc[1].y * inv);
        w.w = PgType<T>::pack(acc[1].z * inv, acc[1].w * inv);
        *reinterpret_cast<uint4*>(dst) = w;
    }
}

// ------------------------------------------------------------------------------------------------ tensor memory

// Takes `columns` of tensor memory, by warp 9, and waits for the kernel in front.  The columns are taken, by all CTAs, before a dependent may
// begin: the kernels that allocate before they wait (the projections do) rest on that no CTA of an earlier kernel waits for a later one, and
// a dependent beside a CTA of this one could otherwise hold the columns that this one is still to take while it waits for its end.
__device__ __forceinline__ void pg_begin(uint32_t* tmem_base, uint32_t columns)
{
    if ((threadIdx.x >> 5) == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    pdl_launch_dependents();
    pdl_wait();
}

__device__ __forceinline__ void pg_end(const uint32_t* tmem_base, uint32_t columns)
{
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if ((threadIdx.x >> 5) == 9) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_base), "r"(columns) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------ keys and values

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_u32(smem_dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

// The blocks of a piece on their way into the ring, by a whole warp: a lane per page and 64 dims.  Pages that hold none of the keys
// that the tile sees are not asked for.
template<int D>
struct PgLoader {
    static constexpr int kHalves = D / 64;
    const PagedMhaArgs& a;
    const int* row;      // the sequence's row of the page table
    int head;
    PgSpan span;

    __device__ __forceinline__ int lane_key() const { return (int)(threadIdx.x & 31) / kHalves * min(1 << a.page_shift, kPgKeys); }
    __device__ __forceinline__ bool mine(int key0) const
    {
        const int at = lane_key();
        return at < kPgKeys && key0 + at < span.hi && key0 + at + min(1 << a.page_shift, kPgKeys) > span.lo;
    }
    // the page of this lane's keys of the block at key0
    __device__ __forceinline__ int page(int key0) const { return mine(key0) ? row[(key0 + lane_key()) >> a.page_shift] : 0; }
    __device__ __forceinline__ void load(const CUtensorMap* map, int key0, int page, uint8_t* stage, uint64_t* full) const
    {
        const int lane = threadIdx.x & 31, rows = min(1 << a.page_shift, kPgKeys), at = lane_key(), h = lane % kHalves;
        const bool m = mine(key0);
        const int count = __popc(__ballot_sync(0xffffffffu, m));
        if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(count * rows * 128));
        __syncwarp();
        if (m) {
            if (page < 0 || page >= a.num_pages) {
                g_device_status = 6;
                page = a.num_pages;   // behind the last: reads as zeros
            }
            tma_load_4d(stage + h * (kPgKeys * 128) + at * 128, map, 64 * h, (key0 + at) & ((1 << a.page_shift) - 1), head, page, full);
        }
    }
};

// Where K and V of block j of a piece of n blocks stand in its order of loads: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1).
__device__ __forceinline__ int pg_k_entry(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int pg_v_entry(int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; }

// [..][rows][values] of 16-bit values as boxes of 64 values (128 bytes, swizzled); dims and strides from the innermost.
int pg_encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank, const long long* dims, const long long* strides,
              const int* box)
{
    EncodeTiledFn encode = encode_tiled_fn();
    EET_CHECK(encode != nullptr, "paged attention: cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t d[4], st[3];
    cuuint32_t bx[4], elem[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) {
        d[i] = (cuuint64_t)dims[i];
        bx[i] = (cuuint32_t)box[i];
        if (i > 0) st[i - 1] = (cuuint64_t)strides[i] * 2;
    }
    const CUresult rc = encode(map, type, (cuuint32_t)rank, const_cast<void*>(base), d, st, bx, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    EET_CHECK(rc == CUDA_SUCCESS, "paged attention: cuTensorMapEncodeTiled failed with code %d (strides too large or negative)", (int)rc);
    return 0;
}

// Q as [token][head][dim] with boxes of `tokens` x the heads of a group, K and V as [page][head][slot][dim] with boxes of a page
// (of 128 slots of a larger one).
template<typename T, int D>
int pg_encode_maps(const PagedMhaArgs& a, int tokens, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v)
{
    const long long q_dims[3] = {D, a.heads, a.tokens}, q_str[3] = {1, a.q_head, a.q_tok};
    const int q_box[3] = {64, a.heads / a.kv_heads, tokens};
    if (int rc = pg_encode(q, PgType<T>::tma, a.q, 3, q_dims, q_str, q_box)) return rc;
    const int page = 1 << a.page_shift;
    const long long dims[4] = {D, page, a.kv_heads, a.num_pages};
    const int box[4] = {64, page < kPgKeys ? page : kPgKeys, 1, 1};
    const long long ks[4] = {1, a.kc_slot, a.kc_head, a.kc_page}, vs[4] = {1, a.vc_slot, a.vc_head, a.vc_page};
    if (int rc = pg_encode(k, PgType<T>::tma, a.k_cache, 4, dims, ks, box)) return rc;
    return pg_encode(v, PgType<T>::tma, a.v_cache, 4, dims, vs, box);
}

}  // namespace

}  // namespace eet
