// Rotary positions and the append of new keys and values to a paged cache.
//
// One CTA takes a token (or, when the tokens are few, a share of its heads).  The angles of a token are the same for all of its
// heads: they are computed once, into shared memory.  An angle is position * freqs[i] in 64 bits, reduced to a part of one turn
// there and only then rounded to 32 bits: at position 10^6 a 32-bit product would be off by 0.06 radians.  sincospif of the
// rest is good to 2 ulp.
//
// Bound: HBM for prompts, launch latency for decode steps.
#include "common.cuh"
#include "kernels.h"

namespace eet {

namespace {

constexpr int kRotThreads = 128;
constexpr int kRotMaxPairs = 128;   // head sizes up to 256

template<typename T>
struct Pair2;
template<>
struct Pair2<__half> {
    using type = __half2;
    static __device__ __forceinline__ float2 up(__half2 v) { return __half22float2(v); }
    static __device__ __forceinline__ __half2 down(float a, float b) { return __floats2half2_rn(a, b); }
};
template<>
struct Pair2<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ float2 up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
    static __device__ __forceinline__ __nv_bfloat162 down(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

// kStore: the keys go to their pages and the values with them, the position follows from the lengths unless it is given.
// An item is 16 dims of a head: with the half layout dims 8c .. 8c+7 and the partners half the rotated part further, with the
// interleaved layout and in the part that is not rotated dims 16c .. 16c+15.
template<typename T, bool kStore>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a)
{
    using P2 = Pair2<T>;
    using V2 = typename P2::type;
    constexpr int kAhead = 3;   // items a thread has in flight
    __shared__ __align__(16) float2 cs[kRotMaxPairs];
    const int token = blockIdx.x;
    const int tid = threadIdx.x;
    const int pairs = a.rotary_dim >> 1;
    long long pos = 0;
    T* kdst = nullptr;
    T* vdst = nullptr;
    pdl_launch_dependents();
    pdl_wait();

    const int per_row = a.head_dim >> 4;
    const int at_once = kRotThreads / per_row;
    const int rows = a.heads + a.kv_heads + (kStore ? a.kv_heads : 0);
    const int step = (int)gridDim.y * at_once;
    const int c = tid % per_row;
    const bool turned = c < (a.rotary_dim >> 4);
    const int d0 = (turned && !a.interleaved) ? 8 * c : 16 * c;
    const int d1 = (turned && !a.interleaved) ? 8 * c + pairs : 16 * c + 8;
    const int row0 = tid / per_row < at_once ? (int)blockIdx.y * at_once + tid / per_row : rows;
    uint4 x[kAhead], y[kAhead];
    auto load = [&](int row, uint4& u, uint4& w) {
        const T* src;
        if (row < a.heads) src = (const T*)a.q + (size_t)token * a.q_tok + (size_t)row * a.q_head;
        else if (row < a.heads + a.kv_heads) src = (const T*)a.k + (size_t)token * a.k_tok + (size_t)(row - a.heads) * a.k_head;
        else src = (const T*)a.v + (size_t)token * a.v_tok + (size_t)(row - a.heads - a.kv_heads) * a.v_head;
        u = *reinterpret_cast<const uint4*>(src + d0);
        w = *reinterpret_cast<const uint4*>(src + d1);
    };
    // (on their way while the angles are computed)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        if (row0 + i * step < rows) load(row0 + i * step, x[i], y[i]);
    }

    if (kStore) {
        // the sequence of the token: how many of them end at or before it
        int seq = 0;
        for (int i = 0; i < a.seqs; i += kRotThreads) {
            seq += __syncthreads_count(i + tid < a.seqs && a.starts[i + tid + 1] <= token);
        }
        if (seq >= a.seqs || a.starts[seq] > token) return;   // a row that belongs to no sequence
        pos = (long long)a.lens[seq] - a.starts[seq + 1] + token;
        if (pos >= 0) {
            const long long column = pos >> a.page_shift;
            const int page = column < a.max_pages ? a.pages[seq * a.pages_stride + column] : -1;
            if (page >= 0 && page < a.num_pages) {
                const long long slot = pos & ((1 << a.page_shift) - 1);
                kdst = (T*)a.k_cache + page * a.kc_page + slot * a.kc_slot;
                vdst = (T*)a.v_cache + page * a.vc_page + slot * a.vc_slot;
            }
            else if (tid == 0) {
                g_device_status = 6;
            }
        }
    }
    if (a.positions != nullptr) pos = a.positions[token];
    for (int i = tid; i < pairs; i += kRotThreads) {
        const double turns = (double)pos * (a.freqs[i] * 0.15915494309189533577);   // 1 / (2 pi)
        float s, co;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
        cs[i] = make_float2(co * a.magnitude, s * a.magnitude);
    }
    __syncthreads();

    auto store = [&](int row, uint4 u, uint4 w) {
        T* dst;
        if (row < a.heads) {
            dst = (T*)a.q_out + (size_t)token * a.qo_tok + (size_t)row * a.qo_head;
        }
        else if (row < a.heads + a.kv_heads) {
            dst = kStore ? kdst : (T*)a.k_out + (size_t)token * a.ko_tok;
            if (dst != nullptr) dst += (size_t)(row - a.heads) * (kStore ? a.kc_head : a.ko_head);
        }
        else {
            dst = vdst;
            if (dst != nullptr) dst += (size_t)(row - a.heads - a.kv_heads) * a.vc_head;
        }
        if (dst == nullptr) return;
        if (turned && row < a.heads + a.kv_heads) {
            V2* xh = reinterpret_cast<V2*>(&u);
            V2* yh = reinterpret_cast<V2*>(&w);
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 t0 = cs[8 * c + e], t1 = cs[8 * c + 4 + e];
                    const float2 f = P2::up(xh[e]), g = P2::up(yh[e]);
                    xh[e] = P2::down(f.x * t0.x - f.y * t0.y, f.y * t0.x + f.x * t0.y);
                    yh[e] = P2::down(g.x * t1.x - g.y * t1.y, g.y * t1.x + g.x * t1.y);
                }
            }
            else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 t0 = cs[8 * c + 2 * e], t1 = cs[8 * c + 2 * e + 1];
                    const float2 f = P2::up(xh[e]), g = P2::up(yh[e]);
                    xh[e] = P2::down(f.x * t0.x - g.x * t0.y, f.y * t1.x - g.y * t1.y);
                    yh[e] = P2::down(g.x * t0.x + f.x * t0.y, g.y * t1.x + f.y * t1.y);
                }
            }
        }
        *reinterpret_cast<uint4*>(dst + d0) = u;
        *reinterpret_cast<uint4*>(dst + d1) = w;
    };
    for (int row = row0; row < rows; row += kAhead * step) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (row + i * step < rows) store(row + i * step, x[i], y[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int next = row + (kAhead + i) * step;
            if (next < rows) load(next, x[i], y[i]);
        }
    }
}

}  // namespace

template<typename T, bool kStore>
static int launch_rotary_t(const RotaryArgs& a, cudaStream_t stream)
{
    // few tokens: their heads are shared out, so that some 600 CTAs exist
    const int rows_at_once = kRotThreads / (a.head_dim / 16);
    const int rows = a.heads + a.kv_heads + (kStore ? a.kv_heads : 0);
    int shares = (rows + rows_at_once - 1) / rows_at_once;
    const int wanted = (4 * sm_count() + a.tokens - 1) / a.tokens;
    if (shares > wanted) shares = wanted;
    if (shares < 1) shares = 1;
    EET_CUDA(launch_pdl(rotary_kernel<T, kStore>, dim3((unsigned)a.tokens, (unsigned)shares), dim3(kRotThreads), 0, stream, a));
    return 0;
}

int launch_rotary(const RotaryArgs& a, bool store, cudaStream_t stream)
{
    if (a.tokens == 0 || (store && a.seqs == 0)) return 0;
    if (a.bf16) return store ? launch_rotary_t<__nv_bfloat16, true>(a, stream) : launch_rotary_t<__nv_bfloat16, false>(a, stream);
    return store ? launch_rotary_t<__half, true>(a, stream) : launch_rotary_t<__half, false>(a, stream);
}

// Which kernels serve a call.  Sequences whose new tokens make at most 16 rows with the heads that share a kv head are for the kernel
// of few rows (paged_rows.cu), the others for that of 128-row tiles (paged_tc.cu); each takes any number of tokens where it is alone.
// Measured with 16 sequences of 1000 to 3000 positions, 32 / 8 heads: 20 rows (5 tokens) 39 us on the first kernel with 32 columns, 40 on the
// second; 48 rows 95 with 64 columns and 47; 4 rows (64 sequences) 93 and 140.
struct PagedPlan {
    bool rows, tiles;    // which of them run
    int few;             // sequences of up to so many tokens go to the first
    bool whole[2];       // their tiles are not cut (no scratch, no second launch)
    size_t bytes[2];     // scratch
};

static PagedPlan paged_plan(const PagedMhaArgs& a)
{
    PagedPlan p = {};
    const int group = a.heads / a.kv_heads;
    auto is_few = [&](long long tokens) { return (tokens > 0 ? tokens : 1) * group <= kPwRows; };
    p.rows = is_few(a.max_tokens);
    p.tiles = !p.rows;
    p.few = 0x7fffffff;
    if (p.tiles) {
        // Few tokens each beside the longest, and something to read for them?  One chunk of 200 and 31 single tokens behind up to 1000
        // positions take, with both kinds of CTAs and with tiles alone: 32 heads 67 and 82 us, 32 / 8 heads 32 and 36; with 7 single
        // tokens 34 and 41, 28 and 26.
        const long long others = a.seqs - 1, rest = a.tokens - a.max_tokens;
        p.rows = others > 0 && is_few((rest + others - 1) / others) && others * a.kv_heads * (a.max_len / kPgKeys + 1) >= 1024;
        p.few = p.rows ? kPwRows / group : 0;
    }
    // Cutting tiles evens out the shares and costs a second launch and parts to write, 4 to 6 us; a block takes 0.8 us in the first kernel
    // and 1.4 (heads of 64) or 1.9 us in the second.  Not where whole tiles make the longest share no more than that longer, taking tiles
    // to be three quarters as long as the longest on average.  (One block less for either, or two: 180 calls of the smaller kind 1.5 % and
    // 2.3 % slower.)
    auto whole = [&](long long tokens, int most) {
        const long long sms = sm_count();
        const long long keys = a.window > 0 && a.window + tokens < a.max_len ? a.window + tokens : a.max_len;
        const long long blocks = keys / kPgKeys + 1;
        const long long tiles = (a.seqs + (a.max_tokens > tokens ? a.tokens / tokens : 0)) * a.kv_heads;
        return blocks - (tiles < sms ? 3 * blocks * tiles / (4 * sms) : 0) <= most;
    };
    if (p.rows) p.whole[0] = whole(kPwRows / group, 5);
    if (p.tiles) p.whole[1] = whole(2 * (kPgRows / group), 4);
    if (p.rows && !p.whole[0]) p.bytes[0] = pg_scratch_bytes(sm_count(), kPwRows, a.head_dim);
    if (p.tiles && !p.whole[1]) p.bytes[1] = pg_scratch_bytes(sm_count(), 2 * kPgRows, a.head_dim);
    return p;
}

size_t paged_mha_workspace_bytes(const PagedMhaArgs& a)
{
    const PagedPlan p = paged_plan(a);
    return p.bytes[0] + p.bytes[1];
}

template<typename T, int D>
static int launch_paged_mha_t(const PagedMhaArgs& a, const PagedPlan& p, cudaStream_t stream)
{
    void* ws[2] = {a.ws, (char*)a.ws + p.bytes[0]};
    // (the tiles without a bias take the maximum of the scores before the scale, which a negative one would turn round)
    const bool bias = a.slopes != nullptr || !(a.scale > 0.f);
    int rc;
    if (!p.tiles) rc = pg_launch_rows<T, D>(a, ws[0], p.whole[0], stream);
    else if (!p.rows && bias) rc = pg_launch_tc<T, D, true>(a, ws[1], p.whole[1], stream);
    else if (!p.rows) rc = pg_launch_tc<T, D, false>(a, ws[1], p.whole[1], stream);
    else if (bias) rc = pg_launch_both<T, D, true>(a, ws[0], ws[1], p.few, p.whole[0], p.whole[1], stream);
    else rc = pg_launch_both<T, D, false>(a, ws[0], ws[1], p.few, p.whole[0], p.whole[1], stream);
    if (rc) return rc;
    PgScratch s[2] = {};
    int n = 0;
    if (p.bytes[0]) s[n++] = {ws[0], kPwRows, 0};
    if (p.bytes[1]) s[n++] = {ws[1], 2 * kPgRows, 1};
    if (n > 0) {
        const long long rows = (long long)a.max_tokens * (a.heads / a.kv_heads), most = p.bytes[1] ? 2 * kPgRows : kPwRows;
        const int y = (int)((rows < most ? rows : most) * (D / 8) + kPgJoinThreads - 1) / kPgJoinThreads;   // 8 dims a thread
        EET_CUDA(launch_pdl(paged_mha_join_kernel<T, D>, dim3(sm_count(), y, n), dim3(kPgJoinThreads), 0, stream, a, s[0], s[1]));
    }
    return 0;
}

int launch_paged_mha(const PagedMhaArgs& a, cudaStream_t stream)
{
    const PagedPlan p = paged_plan(a);
    if (a.bf16) {
        return a.head_dim == 128 ? launch_paged_mha_t<__nv_bfloat16, 128>(a, p, stream) : launch_paged_mha_t<__nv_bfloat16, 64>(a, p, stream);
    }
    return a.head_dim == 128 ? launch_paged_mha_t<__half, 128>(a, p, stream) : launch_paged_mha_t<__half, 64>(a, p, stream);
}

}  // namespace eet
