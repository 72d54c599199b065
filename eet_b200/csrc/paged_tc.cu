// Attention of new tokens over a paged cache on the tensor cores (tcgen05 / TMEM).
//
//   out = softmax(scale Q.K^T + slope (j - p), keys max(first, p - window + 1) .. p).V
//
// Rows of a tile are (token, query head) pairs that share a kv head: 128 / group tokens of the `group` heads, so that K and V
// of a head are read once for all of them.  A CTA (one per SM, all 512 columns of tensor memory) works on two tiles a and b of
// 128 rows at a time against blocks of 128 keys: while the softmax of one tile runs, the tensor core works for the other.
//   paired   a and b are neighbouring tiles of a long chunk and use the same key blocks
//   split    there is only one tile (few new tokens): a takes its even key blocks, b its odd ones, merged at the end
//
// The work is cut up as paged_share.cuh says.
//
// Bound: the softmax.  A block of both tiles takes 3200 cycles where the tensor core and the exponential unit need 2048 each: P lies over S
// and tensor memory is full, so the next Q.K^T follows P.V, and a warp waits 1300 cycles for it after 1900 of its own.  P.V begins with the
// first half of P, the reference under which O is accumulated moves in steps of 2^8 only, and code that runs with few registers beat
// everything that did not (1024 tokens behind 24000, 64 / 8 heads, bf16: 788 us = 1.04 PF/s among other calls at the power cap, 711 alone;
// 512 behind 8192, 32 / 8 heads: 87 us).  168 registers; 8 bytes of spills with a bias, in the kernel of both kinds of CTAs 8 without and 24
// with it.
//
//   warps 0-3, 4-7  softmax of tile a / b: one thread per row = TMEM lane
//   warp 8          producer: Q, then K and V blocks through a ring of five 32 KiB stages (order K0 K1 V0 K2 V1 ...), a lane
//                   per page and 64 dims: 4-D tensor maps over [page][head][slot][dim], 128-byte swizzle
//   warp 9          one thread issues S = Q.K^T and O += P.V (P from tensor memory, V as MN-major operand)
// Keys outside of what any row of the pair sees may be anything, even NaN (slots behind the end of a sequence): their scores are
// masked by selection and their rows of V are set to zero in shared memory before the product reads them.
//
// Over a cache of 8-bit codes the products take the codes, which are exact in q's type, and the scales stay outside: that of a key on its
// scores, that of a value on its weight, before that is rounded.  (With code times scale rounded to 16 bits in front of the products
// the result was off by 2.9 times as much as the exact one rounded once, and by 1.4 times so: scores are sums of 128 rounded keys.)
// In fp16 O and the weights are held under a power of two that follows the largest scale of the values so far.  Warp 8 brings codes to three places in shared
// memory, half an entry each, and the scales of a block to a ring of six; four more warps (12-15, a warpgroup of their own) turn the
// codes into 16-bit values where the copy engine would have put K and V.  What these warps and the softmax do has to be little code as well
// as few instructions: five kinds of warps share an instruction cache.  512 tokens behind 8192, 32 / 8 heads, bf16: conversions written
// out 187 us, in a loop 130, with the copies taken from them 101; that was with rounded keys.  With exact codes, and the softmax written
// out as it is for 16 bits, 143; its scores put back after their scales instead of scaled twice 129, in loops of 32 keys 123.  (The 16-bit cache: 87.)
// 512 threads of 128 registers, 12 to 28 bytes of spills.  (Shares of 136 for the softmax and 120 for the others, by setmaxnreg: 24 to 48 bytes, the chunk
// 122 us and not 123, 333 tokens with a bias beside 23 single ones 115 and not 113; 144 and 112: 124.5 and 113.)
#include <type_traits>

#include "codes.cuh"
#include "paged_share.cuh"

namespace eet {

namespace {

constexpr int kPgThreads = 320;
constexpr int kPgCodesThreads = 512;    // with the warps that convert codes
static_assert(kPgThreads <= 32 * kPgMostWarps && kPgCodesThreads <= 32 * kPgMostWarps, "a sum for each warp in PgFound");
constexpr int kPgStages = 5;
// (the codes' own places take room)
constexpr __host__ __device__ int pg_ring(int head_dim, int codes) { return codes && head_dim == 128 ? 4 : kPgStages; }
constexpr int kPgExtra = 3;             // a tile's beginning and end cost as much as three blocks
constexpr uint32_t kPgTmemCols = 512;   // S of a, S of b (their probabilities over them), O of a, O of b: 128 each

// ------------------------------------------------------------------------------------------------ the kernel

struct PgSmem {
    uint64_t q_full, q_empty;
    uint64_t full[kPgStages], empty[kPgStages];
    uint64_t s_full[2];      // Q.K^T of a block has completed, and the P.V before it
    uint64_t p_half[2];      // the probabilities of the block's first 64 keys are there, O is rescaled (four warps)
    uint64_t p_ready[2];     // those of the others, too
    uint64_t o_full[2];      // the last P.V of a piece has completed
    uint64_t o_free[2];      // O has been read (four warps)
    uint64_t b_ready;        // split: b's maximum and sum are in b_max, b_sum, its O is complete (four warps)
    uint64_t staged_full[3], staged_empty[3];   // codes: the places they come to (the bytes; four warps)
    uint64_t scales_full[6];                    // the scales of a block (32 threads' copies)
    float b_unit;            // split: what b's O is to be multiplied with
    volatile int abort;
    __align__(8) float b_max[kPgRows], b_sum[kPgRows];
    // what a softmax warp needs between its pieces, out of its registers while it works on one
    PgShare share[8];
    PgPiece piece[8];
};

struct PgSmemFound : PgSmem {
    PgFound found;
};

__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// The reference of a row: the power of a score s is 2^(s factor + off).  factor is log2(e) (and the scale, where scores are taken before it)
// and off the reference times that, rounded to 24 bits: what of it is lost is a factor of all of the row's powers, and would be 2^512 at
// scores of 10^10.  So from 2^24 on, where a unit in the last place of a score is a factor of 4 and more and a sum of products does not
// hold so much, factor is the power of two below and off exact: equal scores weigh the same, one that leads by more than that hides the
// others.  (Subtracting the reference from the scores first takes 2.5 % of a chunk, 4.5 with a bias.)
struct PgReference {
    float factor, off;
    // what the sums under it are to be multiplied with, as a power of two
    __device__ __forceinline__ float log2_of(float to_log2) const
    {
        const float inverse = __uint_as_float(0x7f000000u - __float_as_uint(factor));   // where it is a power of two
        return factor == to_log2 ? -off : -off * inverse * to_log2;
    }
};

template<typename T>
__device__ __forceinline__ PgReference pg_reference(float maximum, float to_log2)
{
    if (!(fabsf(maximum * to_log2) >= 16777216.0f)) return {to_log2, fmaf(-maximum, to_log2, PgType<T>::kUp)};
    const float below = __uint_as_float(__float_as_uint(to_log2) & 0xff800000u);
    return {below, -maximum * below};
}

// The blocks of a piece that tile x (0: a, 1: b) works on: first, first + stride, ... below end (block numbers of the piece).
struct PgTurns {
    int first, end, stride;
    __device__ __forceinline__ bool any() const { return first < end; }
};

__device__ __forceinline__ PgTurns pg_turns(const PagedMhaArgs& a, const PgPiece& p, int tile_tokens, int x)
{
    const int token0 = 2 * p.tile * tile_tokens;
    PgTurns r;
    if (p.s.tokens - token0 <= tile_tokens) {   // split
        r.first = x;
        r.end = p.blocks;
        r.stride = 2;
        return r;
    }
    const PgSpan span = pg_span(a, p.s, token0 + x * tile_tokens, token0 + (x + 1) * tile_tokens);
    const int n = span.blocks();
    r.first = max(0, p.top - (span.first_block() + n - 1));
    r.end = n > 0 ? min(p.blocks, p.top - span.first_block() + 1) : 0;
    r.stride = 1;
    return r;
}

// By one thread, in front of a barrier.  `writers`: arrivals that fill a stage.
__device__ __forceinline__ void pg_init(PgSmem& sm, uint32_t writers = 1)
{
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < kPgStages; ++i) {
        mbar_init(&sm.full[i], writers);
        mbar_init(&sm.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
        mbar_init(&sm.s_full[x], 1);
        mbar_init(&sm.p_half[x], 4);
        mbar_init(&sm.p_ready[x], 4);
        mbar_init(&sm.o_full[x], 1);
        mbar_init(&sm.o_free[x], 4);
    }
    mbar_init(&sm.b_ready, 4);
    for (int i = 0; i < 3; ++i) {
        mbar_init(&sm.staged_full[i], 1);
        mbar_init(&sm.staged_empty[i], 4);
    }
    for (int i = 0; i < 6; ++i) mbar_init(&sm.scales_full[i], 32);
    sm.abort = 0;
    mbar_fence_init();
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Four codes as two words of T.  int8 as bf16: a byte under the exponent of 128, where the low seven bits are units, less 128, or 256 where
// its top bit says that it is negative.
template<typename T, int kCodes>
__device__ __forceinline__ void pg_values4(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    if (std::is_same<T, __half>::value) {
        codes_to_half<kCodes>(w, lo, hi);
    }
    else if (kCodes == kCodesInt8) {
        const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
        const uint32_t more[2] = {a & 0xff7fff7fu, b & 0xff7fff7fu}, less[2] = {a & 0xff80ff80u, b & 0xff80ff80u};
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(more[0]), "r"(less[0]));
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(more[1]), "r"(less[1]));
    }
    else {
        uint32_t h[2];
        codes_to_half<kCodes>(w, h[0], h[1]);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[0])), g = __half22float2(*reinterpret_cast<const __half2*>(&h[1]));
        lo = PgType<T>::pack(f.x, f.y);
        hi = PgType<T>::pack(g.x, g.y);
    }
}

__device__ __forceinline__ void tmem_ld_wait32(uint32_t* v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 32; ++c) asm volatile("" : "+r"(v[c]));
}
__device__ __forceinline__ void tmem_st32_async(uint32_t taddr, uint32_t* v)
{
    tmem_st16_async(taddr, *reinterpret_cast<uint32_t(*)[16]>(v));
    tmem_st16_async(taddr + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
}

// Codes and scales on their way to their places, by a whole warp.  Scales of keys that the tile does not see, and of pages outside the cache, become
// zero.
template<int D>
struct PgCodesLoader {
    static constexpr int kPlaces = 3, kScales = 6;
    static constexpr int kPlace = kPgKeys / 2 * D;                         // bytes: half an entry
    static constexpr int kBytes = kPlaces * kPlace + kScales * 2 * kPgKeys * 4;
    const PagedMhaArgs& a;
    const int* row;      // the sequence's row of the page table
    int head;
    PgSpan span;

    // the page of the run of 16 keys lane .. of the block at key0, in the first eight lanes, as the table has it; -1: nobody sees them
    __device__ __forceinline__ int page(int key0) const
    {
        const int lane = threadIdx.x & 31, key = key0 + 16 * lane;
        return lane < kPgKeys / 16 && key < span.hi && key + 16 > span.lo ? row[key >> a.page_shift] : -1;
    }
    // half `half` of an entry: a lane a page
    __device__ __forceinline__ void load(const CUtensorMap* map, int key0, int half, int page, uint8_t* place, uint64_t* full) const
    {
        constexpr int kKeys = kPgKeys / 2;
        const int lane = threadIdx.x & 31, n = min(1 << a.page_shift, kKeys), at = lane * n, key = key0 + half * kKeys + at;
        // (the first run of a page may be one that nobody sees: any of its runs knows the page)
        int of = -1;
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
            const int other = __shfl_sync(0xffffffffu, page, half * (kKeys / 16) + min(at / 16 + i, kKeys / 16 - 1));
            if (16 * i < n) of = max(of, other);
        }
        const bool mine = at < kKeys && key < span.hi && key + n > span.lo;
        const int count = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(count * n * D));
        __syncwarp();
        if (mine) {
            if (of < 0 || of >= a.num_pages) {
                g_device_status = 6;
                of = a.num_pages;   // behind the last: reads as zeros
            }
            tma_load_4d(place + at * D, map, 0, key & ((1 << a.page_shift) - 1), head, of, full);
        }
    }
    // the scales of a block: four keys a lane, k in front of v
    __device__ __forceinline__ void load_scales(int key0, int page, float* place, uint64_t* full) const
    {
        const int lane = threadIdx.x & 31;
        const float *k = a.k_scale + head * a.ks_head, *v = a.v_scale + head * a.vs_head;
        const uint32_t to = smem_u32(place + lane);
#pragma unroll
        for (int i = 0; i < kPgKeys / 32; ++i) {
            const int of = __shfl_sync(0xffffffffu, page, 2 * i + (lane >> 4)), key = key0 + 32 * i + lane, slot = key & ((1 << a.page_shift) - 1);
            const uint32_t bytes = key >= span.lo && key < span.hi && of >= 0 && of < a.num_pages ? 4 : 0;
            copy4_async(to + 128 * i, k + (bytes ? of : 0) * a.ks_page + slot, bytes);
            copy4_async(to + 128 * i + kPgKeys * 4, v + (bytes ? of : 0) * a.vs_page + slot, bytes);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
    }
};

// 16 keys of half an entry into the ring, from key0 of it, eight at a time.  Lane (r, c) = (lane / 4, lane % 4) has 16 codes of key r in
// either half of a row, odd keys the halves in the other order: eight lanes then meet no bank twice, reading or writing.  scales: of the
// block's values, where rows are to be zero that nobody sees, and those whose scale is not finite: what is there may be NaN, and nothing
// times that is NaN.
template<typename T, int D, int kCodes>
__device__ __forceinline__ void pg_convert(const uint8_t* place, int key0, const float* scales, uint8_t* stage, int stage_key)
{
    constexpr int kHalves = D / 64, kHalf = kPgRows * 128;
    const int lane = threadIdx.x & 31, c = 2 * (lane & 3);
    const uint32_t codes = smem_u32(place) + 16 * (lane & 3);
#pragma unroll 1
    for (int i = 0; i < 16; i += 8) {
        const int from = key0 + i + (lane >> 2), key = stage_key + i + (lane >> 2);
        uint4 x[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) x[h] = lds128(codes + (uint32_t)(from * D + 64 * (kHalves == 2 ? h ^ (key & 1) : 0)));
        if (kCodes == kCodesE4M3 && scales != nullptr) {
            const bool none = (__float_as_uint(scales[key]) & 0x7fffffffu) - 1u >= 0x7f7fffffu;
#pragma unroll
            for (int h = 0; h < kHalves; ++h) x[h] = none ? make_uint4(0u, 0u, 0u, 0u) : x[h];
        }
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            uint4 y[2];
            pg_values4<T, kCodes>(x[h].x, y[0].x, y[0].y);
            pg_values4<T, kCodes>(x[h].y, y[0].z, y[0].w);
            pg_values4<T, kCodes>(x[h].z, y[1].x, y[1].y);
            pg_values4<T, kCodes>(x[h].w, y[1].z, y[1].w);
            uint8_t* dst = stage + (kHalves == 2 ? h ^ (key & 1) : 0) * kHalf + key * 128;
            *reinterpret_cast<uint4*>(dst + ((c ^ (key & 7)) << 4)) = y[0];
            *reinterpret_cast<uint4*>(dst + (((c + 1) ^ (key & 7)) << 4)) = y[1];
        }
    }
}

// The work of CTA `cta` of `ctas`; the scratch is laid out for `region` of them.  kCodes: the cache holds codes, which warps 12-15
// convert, and map_k and map_v are of those.
template<typename T, int D, bool kBias, int kCodes = 0>
__device__ __forceinline__ void pg_tiles(const CUtensorMap* map_q, const CUtensorMap* map_k, const CUtensorMap* map_v, const PagedMhaArgs& a,
                                         void* ws, int least, int whole, int cta, int ctas, int region, PgSmem& sm,
                                         PgFound& found, const uint32_t& tmem_base, uint8_t* dyn)
{
    constexpr int kHalves = D / 64;
    constexpr int kHalf = kPgRows * 128;         // bytes of [128 rows][64 values], swizzled
    constexpr int kTile = kHalves * kHalf;       // a Q tile, a K or a V block
    constexpr int kRing = pg_ring(D, kCodes);
    uint8_t* q_tiles = dyn;
    uint8_t* ring = q_tiles + 2 * kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    const int tile_tokens = kPgRows / group, pair_tokens = 2 * tile_tokens;
    const PgTiling tiling = {pair_tokens, least, 0x7fffffff, kPgExtra};

    PgShare share;
    PgPlace place;
    const bool work = pg_find_share(a, tiling, cta, ctas, whole != 0, found, share, place);
    if (kCodes) __syncthreads();   // (what it was found with lies in b_max, b_sum)
    const uint32_t tmem = tmem_base;
    PgPiece p;

    if (!work) {
        if (!whole && threadIdx.x == 0) pg_write_header(a, tiling, ws, cta, ctas, false, share, place);
    }
    else if (warp == 8) {
        // ------------------------------------------------------------------ producer
        const long long cap = (long long)a.max_pages << a.page_shift;
        int stage = 0, issued = 0, pieces = 0, scaled = 0;
        uint32_t phase = 1;                                       // of `empty`: the first round finds the stages free
        bool ok = true;
        const PgShare all = share;
        while (ok && share.next(a, tiling, p)) {
            if (p.blocks == 0) continue;
            const PgSpan span = pg_span(a, p.s, p.tile * pair_tokens, (p.tile + 1) * pair_tokens);
            if (pieces > 0 && !tc_wait_warp(&sm.q_empty, (uint32_t)((pieces - 1) & 1), &sm.abort)) break;
            ++pieces;
            const int token0 = p.tile * pair_tokens;
            const bool pair = p.s.tokens - token0 > tile_tokens;
            const uint32_t q_bytes = (uint32_t)(tile_tokens * group * 128 * kHalves);
            if (lane == 0) mbar_arrive_expect_tx(&sm.q_full, pair ? 2 * q_bytes : q_bytes);
            __syncwarp();
            if (lane < (pair ? 2 : 1) * kHalves) {
                const int x = lane / kHalves, h = lane % kHalves;
                tma_load_3d(q_tiles + x * kTile + h * kHalf, map_q, 64 * h, p.head * group, p.s.row0 + token0 + x * tile_tokens,
                            &sm.q_full);
            }
            if (p.s.p0 + p.s.tokens > cap && lane == 0) g_device_status = 6;
            if (kCodes) {
                using Loader = PgCodesLoader<D>;
                const Loader loader = {a, a.pages + p.seq * a.pages_stride, p.head, span};
                uint8_t* places = ring + kRing * kTile;
                float* scales = reinterpret_cast<float*>(places + Loader::kPlaces * Loader::kPlace);
                const int n = p.blocks, key_top = p.top * kPgKeys;
                int next = loader.page(key_top), last = -1, older = -1;   // pages of the next K, of the last one and of that before
                for (int e = 0; e < 2 * n && ok; ++e) {                   // K0 K1 V0 K2 V1 ..
                    const bool end = e == 2 * n - 1, v = end || (e > 0 && e % 2 == 0);
                    const int j = end ? n - 1 : v ? e / 2 - 1 : (e + 1) / 2, page = !v ? next : end ? last : older;
                    for (int half = 0; half < 2 && ok; ++half) {
                        const int x = issued % Loader::kPlaces;
                        ok = tc_wait_warp(&sm.staged_empty[x], (uint32_t)((issued / Loader::kPlaces + 1) & 1), &sm.abort);
                        if (!ok) break;
                        // (the softmax has done with the scales of six blocks before: their K has left the ring three blocks ago, behind
                        // products that wait for its weights)
                        if (!v && half == 0) {
                            const int slot = scaled++ % Loader::kScales;
                            loader.load_scales(key_top - j * kPgKeys, page, scales + slot * 2 * kPgKeys, &sm.scales_full[slot]);
                        }
                        loader.load(v ? map_v : map_k, key_top - j * kPgKeys, half, page, places + x * Loader::kPlace, &sm.staged_full[x]);
                        ++issued;
                    }
                    if (!v) {
                        older = last;
                        last = next;
                        if (j + 1 < n) next = loader.page(key_top - (j + 1) * kPgKeys);
                    }
                }
                continue;
            }
            const PgLoader<D> loader = {a, a.pages + p.seq * a.pages_stride, p.head, span};
            auto put = [&](const CUtensorMap* map, int j, int page) -> bool {
                if (!tc_wait_warp(&sm.empty[stage], phase, &sm.abort)) return false;
                loader.load(map, (p.top - j) * kPgKeys, page, ring + stage * kTile, &sm.full[stage]);
                ++issued;
                if (++stage == kRing) {
                    stage = 0;
                    phase ^= 1;
                }
                return true;
            };
            int page = loader.page(p.top * kPgKeys), before = 0;
            for (int j = 0; j <= p.blocks && ok; ++j) {
                const int next = j + 1 < p.blocks ? loader.page((p.top - j - 1) * kPgKeys) : 0;
                if (j < p.blocks) ok = put(map_k, j, page);
                if (j > 0 && ok) ok = put(map_v, j - 1, before);
                before = page;
                page = next;
            }
        }
        if (!whole && lane == 0) pg_write_header(a, tiling, ws, cta, ctas, true, all, place);
        if (kCodes) {
            // (nor may copies by this warp's threads be on their way)
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (sm.abort) {
                for (int e = max(0, issued - 3); e < issued; ++e) mbar_wait_bounded(&sm.staged_full[e % 3], (uint32_t)((e / 3) & 1));
                if (pieces > 0) mbar_wait_bounded(&sm.q_full, (uint32_t)((pieces - 1) & 1));
            }
        }
        else if (sm.abort) {
            // nothing of this CTA may still be on its way when it ends
            for (int e = max(0, issued - kRing); e < issued; ++e) {
                mbar_wait_bounded(&sm.full[e % kRing], (uint32_t)((e / kRing) & 1));
            }
            if (pieces > 0) mbar_wait_bounded(&sm.q_full, (uint32_t)((pieces - 1) & 1));
        }
    }
    else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issuer
        if (elect_one()) {
            constexpr uint32_t idesc_qk = umma_idesc_f16(kPgRows, kPgKeys) | PgType<T>::idesc;
            constexpr uint32_t idesc_pv = umma_idesc_f16(kPgRows, D) | PgType<T>::idesc | (1u << 16);   // V MN-major
            const uint64_t q_desc = umma_desc_sw128(smem_u32(q_tiles));
            const uint64_t k_desc = umma_desc_sw128(smem_u32(ring));
            const uint64_t v_desc = umma_desc_mn_sw128(smem_u32(ring), (uint32_t)kHalf);
            int entry0 = 0;                      // ring entries of the pieces before
            int pieces = 0;
            int used[2] = {0, 0};                // p_ready phases taken
            int outs[2] = {0, 0};                // pieces that wrote O
            bool ok = true;
            auto landed = [&](int entry) -> bool {
                // (entries are waited for in any order within the ring's length)
                return tc_wait(&sm.full[entry % kRing], (uint32_t)((entry / kRing) & 1), &sm.abort);
            };
            while (ok && share.next(a, tiling, p)) {
                if (p.blocks == 0) continue;
                const bool split = p.s.tokens - p.tile * pair_tokens <= tile_tokens;
                const PgTurns turns[2] = {pg_turns(a, p, tile_tokens, 0), pg_turns(a, p, tile_tokens, 1)};
                const int n = p.blocks;
                ok = tc_wait(&sm.q_full, (uint32_t)(pieces & 1), &sm.abort);
                ++pieces;
                if (!ok) break;
                auto k_entry = [&](int j) { return entry0 + pg_k_entry(j); };
                auto v_entry = [&](int j) { return entry0 + pg_v_entry(j, n); };
                auto active = [&](int x, int j) { return j >= turns[x].first && j < turns[x].end; };
                auto issue_qk = [&](int x, int j) -> bool {
                    if (!landed(k_entry(j))) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t qd = q_desc + (uint64_t)((split ? 0 : x) * (kTile >> 4));
                    const uint64_t kd = k_desc + (uint64_t)((k_entry(j) % kRing) * (kTile >> 4));
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint64_t off = (uint64_t)((kk >> 2) * (kHalf >> 4) + (kk & 3) * 2);
                        umma_f16(tmem + x * kPgKeys, qd + off, kd + off, idesc_qk, kk != 0);
                    }
                    umma_commit(&sm.s_full[x]);
                    return true;
                };
                auto issue_pv = [&](int x, int j) -> bool {
                    const bool first = j == turns[x].first;
                    if (first && outs[x] > 0 && !tc_wait(&sm.o_free[x], (uint32_t)((outs[x] - 1) & 1), &sm.abort)) return false;
                    if (!landed(v_entry(j))) return false;
                    const uint64_t vd = v_desc + (uint64_t)((v_entry(j) % kRing) * (kTile >> 4));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!tc_wait(half ? &sm.p_ready[x] : &sm.p_half[x], (uint32_t)(used[x] & 1), &sm.abort)) return false;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                        for (int kk = half * 4; kk < half * 4 + 4; ++kk) {
                            umma_f16_ts(tmem + 256 + x * 128, tmem + x * kPgKeys + kk * 8, vd + (uint64_t)(kk * (2048 >> 4)), idesc_pv,
                                        !first || kk != 0);
                        }
                    }
                    ++used[x];
                    return true;
                };
                // The last Q.K^T of the piece lets go of Q, whoever issues it; a K or V stage is free behind its last user.
                const int last_qk = n - 1;
                const int rounds = split ? (n + 1) / 2 : n;
                // block of tile x in round r
                auto block_of = [&](int x, int r) { return split ? 2 * r + x : r; };
                auto do_qk = [&](int x, int r) -> bool {
                    const int j = block_of(x, r);
                    if (j >= n) return true;
                    if (active(x, j) && !issue_qk(x, j)) return false;
                    if (split || x == 1) {
                        if (!split && !active(0, j) && !active(1, j) && !landed(k_entry(j))) return false;
                        umma_commit(&sm.empty[k_entry(j) % kRing]);
                        if (j == last_qk) umma_commit(&sm.q_empty);
                    }
                    return true;
                };
                auto do_pv = [&](int x, int r) -> bool {
                    const int j = block_of(x, r);
                    if (j >= n) return true;
                    const bool act = active(x, j);
                    if (act && !issue_pv(x, j)) return false;
                    if (split || x == 1) {
                        if (!split && !active(0, j) && !active(1, j) && !landed(v_entry(j))) return false;
                        umma_commit(&sm.empty[v_entry(j) % kRing]);
                    }
                    if (act && j + turns[x].stride >= turns[x].end) {
                        ++outs[x];
                        umma_commit(&sm.o_full[x]);
                    }
                    return true;
                };
                ok = do_qk(0, 0) && do_qk(1, 0);
                for (int r = 0; r < rounds && ok; ++r) {
                    ok = do_pv(0, r) && do_qk(0, r + 1) && do_pv(1, r) && do_qk(1, r + 1);
                }
                entry0 += 2 * n;
            }
        }
    }
    else if (kCodes && warp >= 12) {
        // ------------------------------------------------------------------ codes into the ring
        using Loader = PgCodesLoader<D>;
        const uint8_t* places = ring + kRing * kTile;
        const float* scales = reinterpret_cast<const float*>(places + Loader::kPlaces * Loader::kPlace);
        int stage = 0, done = 0, before = 0;                      // before: blocks of the pieces before
        uint32_t phase = 1;                                       // of `empty`: the first round finds the stages free
        bool ok = true;
        while (ok && share.next(a, tiling, p)) {
            const int n = p.blocks;
            for (int e = 0; e < 2 * n && ok; ++e) {
                ok = tc_wait_warp(&sm.empty[stage], phase, &sm.abort);
                const bool end = e == 2 * n - 1, v = end || (e > 0 && e % 2 == 0);
                const int block = before + (end ? n - 1 : e / 2 - 1);   // (of V)
                // (rows that nobody sees: at the ends of what the tile reads, and of pages outside the cache; K's scores are masked)
                const float* of = kCodes == kCodesE4M3 && v ? scales + (block % Loader::kScales * 2 + 1) * kPgKeys : nullptr;
                if (of != nullptr && ok) {
                    ok = tc_wait_warp(&sm.scales_full[block % Loader::kScales], (uint32_t)((block / Loader::kScales) & 1), &sm.abort);
                }
#pragma unroll 1
                for (int half = 0; half < 2 && ok; ++half, ++done) {
                    const int x = done % Loader::kPlaces, at = 16 * (warp - 12);
                    ok = tc_wait_warp(&sm.staged_full[x], (uint32_t)((done / Loader::kPlaces) & 1), &sm.abort);
                    if (!ok) break;
                    pg_convert<T, D, kCodes ? kCodes : kCodesInt8>(places + x * Loader::kPlace, at, of, ring + stage * kTile,
                                                                   kPgKeys / 2 * half + at);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.staged_empty[x]);
                }
                if (!ok) break;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.full[stage]);
                if (++stage == kRing) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            before += n;
        }
    }
    else if (warp < 8) {
        // ------------------------------------------------------------------ softmax, epilogue
        const int x = warp >> 2;
        const int r = (warp & 3) * 32 + lane;                 // row of the tile = lane of tensor memory
        const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + t_lane + (uint32_t)(x * kPgKeys), t_o = tmem + t_lane + 256u + (uint32_t)(x * 128);
        const int tok = r / group, g = r - tok * group;
        const float log2e = 1.4426950408889634f;
        const float to_log2 = kBias ? log2e : a.scale * log2e;
        const int cap = (int)min((long long)a.max_pages << a.page_shift, 0x7fffffffLL);
        int entry0 = 0, used = 0, outs = 0, merges = 0;
        bool ok = true;
        if (lane == 0) sm.share[warp] = share;
        __syncwarp();
        while (ok) {
            PgTurns turns;
            PgSpan span;
            int top, blocks, low, high, pos;
            float slope = 0.f;
            {
                PgShare walk = sm.share[warp];
                if (!walk.next(a, tiling, p)) break;
                __syncwarp();
                if (lane == 0) {
                    sm.share[warp] = walk;
                    sm.piece[warp] = p;
                }
                __syncwarp();
                const int token0 = p.tile * pair_tokens;
                const bool split = p.s.tokens - token0 <= tile_tokens;
                const int token = token0 + (split ? 0 : x * tile_tokens) + tok;      // of the sequence
                const bool valid = tok < tile_tokens && token < p.s.tokens;
                pos = p.s.p0 + token;
                top = p.top;
                blocks = p.blocks;
                turns = pg_turns(a, p, tile_tokens, x);
                span = pg_span(a, p.s, token0, token0 + pair_tokens);
                // the keys that this row sees; a row that stands for no token takes whatever comes
                low = valid ? p.s.first : 0;
                high = valid ? min(pos, cap - 1) : 0x7ffffffe;
                if (valid && a.window > 0) low = (int)max((long long)low, (long long)pos - a.window + 1);
                if (kBias && valid && a.slopes != nullptr) slope = a.slopes[p.head * group + g];
            }
            const uint64_t rise[2] = {pair2(0.f, slope), pair2(2.f * slope, 3.f * slope)};   // of the bias over four keys
            float m_run = kPgNone, l_run = 0.f;
            PgReference ref = {1.0f, -kPgNone};   // (-inf stays -inf, and any score moves it)
            // Codes in fp16: O is held under 2^unit, above the largest scale of the values so far, so that weights times scales stay below 2^15.
            constexpr bool kUnit = kCodes != 0 && std::is_same<T, __half>::value;
            constexpr int kLeastUnit = -110;   // 2^15 over it is still a number
            int unit = kLeastUnit - 1;         // (none yet)
            // A wait for scales by parity is only good less than a turn of their ring ahead of the copies.  Tile b, which has no turn in a split
            // piece of one block, comes from any number of those to its next first block: the parity would be that of the turn before, and the
            // wait would end before the scales are there.  So the scores of a piece's first block are waited for in front of its scales: the
            // copies of those were asked for in front of their keys'.
            if (kCodes && turns.any()) ok = tc_wait_warp(&sm.s_full[x], (uint32_t)(used & 1), &sm.abort);
            for (int j = turns.first; j < turns.end && ok; j += turns.stride) {
                const int key0 = (top - j) * kPgKeys;
                const float *k_scales = nullptr, *v_scales = nullptr;
                float less = 1.0f;             // a power of two: of O under the unit before
                if (kCodes) {
                    const int block = entry0 / 2 + j, slot = block % PgCodesLoader<D>::kScales;
                    const uint8_t* ring_end = ring + kRing * kTile + PgCodesLoader<D>::kPlaces * PgCodesLoader<D>::kPlace;
                    k_scales = reinterpret_cast<const float*>(ring_end) + slot * 2 * kPgKeys;
                    v_scales = k_scales + kPgKeys;
                    if (!tc_wait_warp(&sm.scales_full[slot], (uint32_t)((block / PgCodesLoader<D>::kScales) & 1), &sm.abort)) {
                        ok = false;
                        break;
                    }
                    if (kUnit) {
                        const float4 v = reinterpret_cast<const float4*>(v_scales)[lane];
                        auto finite = [](float f) { return fabsf(f) < __uint_as_float(0x7f800000u) ? fabsf(f) : 0.f; };
                        const uint32_t bits = __float_as_uint(warp_max(fmaxf(fmaxf(finite(v.x), finite(v.y)), fmaxf(finite(v.z), finite(v.w)))));
                        const int needed = max(kLeastUnit, min((int)(bits >> 23) - 126, 126));
                        if (needed > unit) {
                            less = unit < kLeastUnit ? 1.0f : ex2_approx((float)(unit - needed));
                            unit = needed;
                        }
                    }
                }
                if (!tc_wait_warp(&sm.s_full[x], (uint32_t)(used & 1), &sm.abort)) {
                    ok = false;
                    break;
                }
                ++used;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                // scores of keys c0 .. c0 + 31 of the block: bias, masks
                float base0 = kBias ? slope * (float)(key0 - pos) : 0.f;
                const bool masked = !__all_sync(0xffffffffu, low <= key0 && high >= key0 + kPgKeys - 1);
                auto finish = [&](uint32_t* v, int c0, const float4* k) {
                    if (kCodes) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const float4 f = k[c / 4];
                            const float2 t = split2(mul2(pair2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), pair2(f.x, f.y)));
                            const float2 u = split2(mul2(pair2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), pair2(f.z, f.w)));
                            v[c] = __float_as_uint(t.x), v[c + 1] = __float_as_uint(t.y);
                            v[c + 2] = __float_as_uint(u.x), v[c + 3] = __float_as_uint(u.y);
                        }
                    }
                    if (kBias) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const float base = fmaf(slope, (float)(c0 + c), base0);
                            const uint64_t base2 = pair2(base, base);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float2 t = split2(fma2(pair2(__uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1])),
                                                             pair2(a.scale, a.scale), add2(base2, rise[e])));
                                v[c + 2 * e] = __float_as_uint(t.x);
                                v[c + 2 * e + 1] = __float_as_uint(t.y);
                            }
                        }
                    }
                    if (masked) {
                        const int from = min(max(low - key0 - c0, 0), 32), to = min(max(high + 1 - key0 - c0, 0), 32);
                        const uint32_t seen = (to < 32 ? (1u << to) - 1 : 0xffffffffu) & ~(from < 32 ? (1u << from) - 1 : 0xffffffffu);
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!(seen & (1u << c))) v[c] = 0xff800000u;   // -inf
                        }
                    }
                };
                float mx[4] = {kPgNone, kPgNone, kPgNone, kPgNone};
                auto maxima = [&](const uint32_t* v) {
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
                    }
                };
                // The upper half of the row for its maximum, then the lower half, which stays; the upper one is read again for
                // its exponentials (all 128 at once did not fit the registers).  The probabilities go over the scores of keys
                // 0 .. 63, so the lower half comes first.
                uint32_t v[64];
                if (kCodes) {
                    // (in loops of 32 keys, with the scores back where they were as they are now: cheaper than scales, bias and masks a second
                    // time, and without spills)
                    float4 k[8];
#pragma unroll 1
                    for (int c0 = 96; c0 >= 0; c0 -= 32) {
                        tmem_ld32_async(t_s + c0, v);
#pragma unroll
                        for (int c = 0; c < 8; ++c) k[c] = reinterpret_cast<const float4*>(k_scales + c0)[c];
                        tmem_ld_wait32(v);
                        finish(v, c0, k);
                        maxima(v);
                        if (c0) tmem_st32_async(t_s + c0, v);
                    }
                }
                else {
                    tmem_ld32_async(t_s + 64, v);
                    tmem_ld32_async(t_s + 96, v + 32);
                    tmem_ld_wait(v);
                    finish(v, 64, nullptr);
                    finish(v + 32, 96, nullptr);
                    maxima(v);
                    maxima(v + 32);
                    tmem_ld32_async(t_s, v);
                    tmem_ld32_async(t_s + 32, v + 32);
                    tmem_ld_wait(v);
                    finish(v, 0, nullptr);
                    finish(v + 32, 32, nullptr);
                    maxima(v);
                    maxima(v + 32);
                }
                m_run = fmaxf(m_run, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                float corr = 1.0f;
                const bool first = j == turns.first;
                const bool moves = fmaf(m_run, ref.factor, ref.off) > kPgLag + PgType<T>::kUp;
                if (moves) {
                    const float old = ref.log2_of(to_log2);
                    ref = pg_reference<T>(m_run, to_log2);
                    corr = ex2_approx(old - ref.log2_of(to_log2));
                }
                // O under the new reference.  The P.V of the block before has completed: s_full was committed behind it.
                if (!first && __any_sync(0xffffffffu, moves || less != 1.0f)) {
                    const float times = kUnit ? corr * less : corr;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(t_o + (uint32_t)c0, o);
#pragma unroll
                        for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * times);
                        tmem_st16_async(t_o + (uint32_t)c0, o);
                    }
                }
                const uint64_t scale2 = pair2(ref.factor, ref.factor), off2 = pair2(ref.off, ref.off);
                uint64_t psum[2] = {0ull, 0ull};
                const float per_unit = kUnit ? __uint_as_float((uint32_t)(127 - unit) << 23) : 1.0f;
                const uint64_t per_unit2 = pair2(per_unit, per_unit);
                auto exponents = [&](const uint32_t* v, uint32_t* pk, const float4* k) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float2 e = split2(fma2(pair2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), scale2, off2));
                        const float p0 = ex2_approx(e.x), p1 = ex2_approx(e.y);
                        psum[c & 1] = add2(psum[c & 1], pair2(p0, p1));
                        if (kCodes) {
                            const float4 of = k[c / 2];
                            uint64_t w = pair2(p0, p1);
                            if (kUnit) w = mul2(w, per_unit2);
                            const float2 q = split2(mul2(w, c % 2 ? pair2(of.z, of.w) : pair2(of.x, of.y)));
                            pk[c] = PgType<T>::pack(q.x, q.y);
                        }
                        else {
                            pk[c] = PgType<T>::pack(p0, p1);
                        }
                    }
                };
                uint32_t pk[16];
                if (kCodes) {
                    float4 k[8];
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) k[c] = reinterpret_cast<const float4*>(v_scales + 32 * i)[c];
                        if (i > 0) tmem_ld_wait32(v);
                        exponents(v, pk, k);
                        if (masked) {
                            // (a scale that is not finite, of a value that this row does not see)
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                pk[c] &= (v[2 * c] == 0xff800000u ? 0u : 0xffffu) | (v[2 * c + 1] == 0xff800000u ? 0u : 0xffff0000u);
                            }
                        }
                        tmem_st16_async(t_s + 16 * i, pk);
                        if (i < 3) tmem_ld32_async(t_s + 32 * i + 32, v);
                        if (i & 1) {
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) mbar_arrive(i == 1 ? &sm.p_half[x] : &sm.p_ready[x]);
                        }
                    }
                }
                else {
                    exponents(v, pk, nullptr);
                    tmem_st16_async(t_s, pk);
                    exponents(v + 32, pk, nullptr);
                    tmem_st16_async(t_s + 16, pk);
                    tmem_ld32_async(t_s + 64, v);
                    tmem_ld32_async(t_s + 96, v + 32);
                    if (key0 < span.lo || key0 + kPgKeys > span.hi) {
                        // rows of V that nobody sees
                        const int entry = entry0 + pg_v_entry(j, blocks), stage = entry % kRing;
                        if (!tc_wait_warp(&sm.full[stage], (uint32_t)((entry / kRing) & 1), &sm.abort)) {
                            ok = false;
                            break;
                        }
                        if (key0 + r < span.lo || key0 + r >= span.hi) {
                            uint4* dst = reinterpret_cast<uint4*>(ring + stage * kTile + r * 128);
#pragma unroll
                            for (int h = 0; h < kHalves; ++h) {
#pragma unroll
                                for (int c = 0; c < 8; ++c) dst[h * (kHalf / 16) + c] = make_uint4(0u, 0u, 0u, 0u);
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.p_half[x]);
                    tmem_ld_wait(v);
                    if (kBias) asm volatile("" : "+f"(base0), "+f"(slope));   // (or the bias would be kept from the first time, in 64 registers)
                    finish(v, 64, nullptr);
                    finish(v + 32, 96, nullptr);
                    exponents(v, pk, nullptr);
                    tmem_st16_async(t_s + 32, pk);
                    exponents(v + 32, pk, nullptr);
                    tmem_st16_async(t_s + 48, pk);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.p_ready[x]);
                }
                const float2 ps = split2(add2(psum[0], psum[1]));
                l_run = l_run * corr + (ps.x + ps.y);
            }
            entry0 += 2 * blocks;
            if (!ok) break;
            p = sm.piece[warp];
            const int token0 = p.tile * pair_tokens;
            const bool split = p.s.tokens - token0 <= tile_tokens;
            const int token = token0 + (split ? 0 : x * tile_tokens) + tok;
            const bool valid = tok < tile_tokens && token < p.s.tokens;
            const int head = p.head * group + g;
            const bool mine = turns.any();
            if (mine) {
                if (!tc_wait_warp(&sm.o_full[x], (uint32_t)(outs & 1), &sm.abort)) {
                    ok = false;
                    break;
                }
                ++outs;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            float max2 = fmaxf(ref.log2_of(to_log2), kPgNone);
            float scale_a = kUnit ? __uint_as_float((uint32_t)(127 + unit) << 23) : 1.f, scale_b = 0.f;
            bool other = false;              // b's sums are to be added
            if (split && x == 1) {
                if (mine) {
                    sm.b_max[r] = max2;
                    sm.b_sum[r] = l_run;
                    if (kUnit) sm.b_unit = scale_a;   // (all threads the same)
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.b_ready);
                }
                continue;
            }
            if (split && p.blocks > 1) {
                if (!tc_wait_warp(&sm.b_ready, (uint32_t)(merges & 1), &sm.abort)) {
                    ok = false;
                    break;
                }
                ++merges;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                other = true;
                const float bm = sm.b_max[r], top = fmaxf(max2, bm);
                const float unit_a = scale_a;
                scale_a = ex2_approx(max2 - top);
                scale_b = ex2_approx(bm - top);
                max2 = top;
                l_run = l_run * scale_a + sm.b_sum[r] * scale_b;
                if (kUnit) scale_a *= unit_a, scale_b *= sm.b_unit;
            }
            const bool complete = p.starts && p.ends;
            const PgPartial part = pg_partial(ws, region, cta, p.starts ? 1 : 0, 2 * kPgRows, D);
            if (complete) {
                const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
                scale_a *= inv;
                scale_b *= inv;
            }
            else if (valid) {
                part.max2[x * kPgRows + r] = max2;
                part.sum[x * kPgRows + r] = l_run;
            }
            T* dst = (T*)a.out + (size_t)(p.s.row0 + token) * a.o_tok + (size_t)head * a.o_head;
            if (!mine && complete && valid) {
#pragma unroll
                for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (mine) {
                const bool nothing = complete && l_run == 0.f;
                const int dims = __any_sync(0xffffffffu, valid) ? D : 0;   // (few rows: some warps have none)
#pragma unroll 1
                for (int c0 = 0; c0 < dims; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(t_o + (uint32_t)c0, o);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * scale_a);
                    if (other) {
                        uint32_t u[32];
                        tmem_ld32(t_o + 128u + (uint32_t)c0, u);
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(fmaf(__uint_as_float(u[c]), scale_b, __uint_as_float(o[c])));
                    }
                    if (!complete) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            part.o[(c0 + c) / 4 * 2 * kPgRows + x * kPgRows + r] = make_float4(
                                __uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
                        }
                    }
                    else if (valid) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8) {
                            uint4 w;
                            w.x = PgType<T>::pack(__uint_as_float(o[c]), __uint_as_float(o[c + 1]));
                            w.y = PgType<T>::pack(__uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
                            w.z = PgType<T>::pack(__uint_as_float(o[c + 4]), __uint_as_float(o[c + 5]));
                            w.w = PgType<T>::pack(__uint_as_float(o[c + 6]), __uint_as_float(o[c + 7]));
                            if (nothing) w = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint4*>(dst + c0 + c) = w;
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.o_free[0 + x]);
                    if (other) mbar_arrive(&sm.o_free[1]);
                }
            }
        }
    }
}

constexpr int pg_tiles_smem(int head_dim, int codes = 0)
{
    return (2 + pg_ring(head_dim, codes)) * (head_dim / 64) * kPgRows * 128 + (codes ? 3 * (kPgKeys / 2) * head_dim + 6 * 2 * kPgKeys * 4 : 0);
}

template<typename T, int D, bool kBias>
__global__ void __launch_bounds__(kPgThreads, 1)
paged_mha_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedMhaArgs a, void* ws, int whole)
{
    extern __shared__ __align__(1024) uint8_t pg_dyn[];
    __shared__ PgSmemFound sm;
    __shared__ uint32_t tmem_base;
    if (smem_u32(pg_dyn) & 1023) {   // the swizzle goes by addresses; the alignment above is there, so this does not happen
        g_device_status = 2;
        return;
    }
    if (threadIdx.x == 0) pg_init(sm);
    pg_begin(&tmem_base, kPgTmemCols);
    pg_tiles<T, D, kBias>(&map_q, &map_k, &map_v, a, ws, 1, whole, (int)blockIdx.x, (int)gridDim.x, (int)gridDim.x, sm, sm.found, tmem_base,
                          pg_dyn);
    pg_end(&tmem_base, kPgTmemCols);
}

template<typename T, int D, bool kBias>
int pg_launch_tc(const PagedMhaArgs& a, void* ws, int whole, cudaStream_t stream)
{
    constexpr int kSmem = pg_tiles_smem(D);
    CUtensorMap map_q, map_k, map_v;
    if (int rc = pg_encode_maps<T, D>(a, kPgRows / (a.heads / a.kv_heads), &map_q, &map_k, &map_v)) return rc;
    auto kern = paged_mha_tc_kernel<T, D, kBias>;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        attr_set[dev] = true;
    }
    EET_CUDA(launch_pdl(kern, dim3(sm_count()), dim3(kPgThreads), kSmem, stream, map_q, map_k, map_v, a, ws, whole));
    return 0;
}

}  // namespace

}  // namespace eet
