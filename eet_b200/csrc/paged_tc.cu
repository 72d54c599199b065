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
#include "paged_share.cuh"

namespace eet {

namespace {

constexpr int kPgThreads = 320;
constexpr int kPgStages = 5;
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
    volatile int abort;
    float b_max[kPgRows], b_sum[kPgRows];
    // what a softmax warp needs between its pieces, out of its registers while it works on one
    PgShare share[8];
    PgPiece piece[8];
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

// By one thread, in front of a barrier.
__device__ __forceinline__ void pg_init(PgSmem& sm)
{
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < kPgStages; ++i) {
        mbar_init(&sm.full[i], 1);
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
    sm.abort = 0;
    mbar_fence_init();
}

// The work of CTA `cta` of `ctas`; the scratch is laid out for `region` of them.
template<typename T, int D, bool kBias>
__device__ __forceinline__ void pg_tiles(const CUtensorMap* map_q, const CUtensorMap* map_k, const CUtensorMap* map_v, const PagedMhaArgs& a,
                                         void* ws, int least, int whole, int cta, int ctas, int region, PgSmem& sm,
                                         const uint32_t& tmem_base, uint8_t* dyn)
{
    constexpr int kHalves = D / 64;
    constexpr int kHalf = kPgRows * 128;         // bytes of [128 rows][64 values], swizzled
    constexpr int kTile = kHalves * kHalf;       // a Q tile, a K or a V block
    uint8_t* q_tiles = dyn;
    uint8_t* ring = q_tiles + 2 * kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    const int tile_tokens = kPgRows / group, pair_tokens = 2 * tile_tokens;
    const PgTiling tiling = {pair_tokens, least, 0x7fffffff, kPgExtra};

    PgShare share;
    PgPlace place;
    const bool work = pg_find_share(a, tiling, cta, ctas, whole != 0, sm.found, share, place);
    const uint32_t tmem = tmem_base;
    PgPiece p;

    if (!work) {
        if (!whole && threadIdx.x == 0) pg_write_header(a, tiling, ws, cta, ctas, false, share, place);
    }
    else if (warp == 8) {
        // ------------------------------------------------------------------ producer
        const long long cap = (long long)a.max_pages << a.page_shift;
        int stage = 0, issued = 0, pieces = 0;
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
            const PgLoader<D> loader = {a, a.pages + p.seq * a.pages_stride, p.head, span};
            auto put = [&](const CUtensorMap* map, int j, int page) -> bool {
                if (!tc_wait_warp(&sm.empty[stage], phase, &sm.abort)) return false;
                loader.load(map, (p.top - j) * kPgKeys, page, ring + stage * kTile, &sm.full[stage]);
                ++issued;
                if (++stage == kPgStages) {
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
        if (sm.abort) {
            // nothing of this CTA may still be on its way when it ends
            for (int e = max(0, issued - kPgStages); e < issued; ++e) {
                mbar_wait_bounded(&sm.full[e % kPgStages], (uint32_t)((e / kPgStages) & 1));
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
                return tc_wait(&sm.full[entry % kPgStages], (uint32_t)((entry / kPgStages) & 1), &sm.abort);
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
                    const uint64_t kd = k_desc + (uint64_t)((k_entry(j) % kPgStages) * (kTile >> 4));
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
                    const uint64_t vd = v_desc + (uint64_t)((v_entry(j) % kPgStages) * (kTile >> 4));
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
                        umma_commit(&sm.empty[k_entry(j) % kPgStages]);
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
                        umma_commit(&sm.empty[v_entry(j) % kPgStages]);
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
    else {
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
            for (int j = turns.first; j < turns.end && ok; j += turns.stride) {
                const int key0 = (top - j) * kPgKeys;
                if (!tc_wait_warp(&sm.s_full[x], (uint32_t)(used & 1), &sm.abort)) {
                    ok = false;
                    break;
                }
                ++used;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                // scores of keys c0 .. c0 + 31 of the block: bias, masks
                float base0 = kBias ? slope * (float)(key0 - pos) : 0.f;
                const bool masked = !__all_sync(0xffffffffu, low <= key0 && high >= key0 + kPgKeys - 1);
                auto finish = [&](uint32_t* v, int c0) {
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
                tmem_ld32_async(t_s + 64, v);
                tmem_ld32_async(t_s + 96, v + 32);
                tmem_ld_wait(v);
                finish(v, 64);
                finish(v + 32, 96);
                maxima(v);
                maxima(v + 32);
                tmem_ld32_async(t_s, v);
                tmem_ld32_async(t_s + 32, v + 32);
                tmem_ld_wait(v);
                finish(v, 0);
                finish(v + 32, 32);
                maxima(v);
                maxima(v + 32);
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
                if (!first && __any_sync(0xffffffffu, moves)) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(t_o + (uint32_t)c0, o);
#pragma unroll
                        for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
                        tmem_st16_async(t_o + (uint32_t)c0, o);
                    }
                }
                const uint64_t scale2 = pair2(ref.factor, ref.factor), off2 = pair2(ref.off, ref.off);
                uint64_t psum[2] = {0ull, 0ull};
                auto exponents = [&](const uint32_t* v, uint32_t* pk) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float2 e = split2(fma2(pair2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), scale2, off2));
                        const float p0 = ex2_approx(e.x), p1 = ex2_approx(e.y);
                        psum[c & 1] = add2(psum[c & 1], pair2(p0, p1));
                        pk[c] = PgType<T>::pack(p0, p1);
                    }
                };
                uint32_t pk[16];
                exponents(v, pk);
                tmem_st16_async(t_s, pk);
                exponents(v + 32, pk);
                tmem_st16_async(t_s + 16, pk);
                tmem_ld32_async(t_s + 64, v);
                tmem_ld32_async(t_s + 96, v + 32);
                if (key0 < span.lo || key0 + kPgKeys > span.hi) {
                    // rows of V that nobody sees
                    const int entry = entry0 + pg_v_entry(j, blocks), stage = entry % kPgStages;
                    if (!tc_wait_warp(&sm.full[stage], (uint32_t)((entry / kPgStages) & 1), &sm.abort)) {
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
                finish(v, 64);
                finish(v + 32, 96);
                exponents(v, pk);
                tmem_st16_async(t_s + 32, pk);
                exponents(v + 32, pk);
                tmem_st16_async(t_s + 48, pk);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[x]);
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
            float scale_a = 1.f, scale_b = 0.f;
            bool other = false;              // b's sums are to be added
            if (split && x == 1) {
                if (mine) {
                    sm.b_max[r] = max2;
                    sm.b_sum[r] = l_run;
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
                scale_a = ex2_approx(max2 - top);
                scale_b = ex2_approx(bm - top);
                max2 = top;
                l_run = l_run * scale_a + sm.b_sum[r] * scale_b;
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

constexpr int pg_tiles_smem(int head_dim)
{
    return (2 + kPgStages) * (head_dim / 64) * kPgRows * 128;
}

template<typename T, int D, bool kBias>
__global__ void __launch_bounds__(kPgThreads, 1)
paged_mha_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedMhaArgs a, void* ws, int whole)
{
    extern __shared__ __align__(1024) uint8_t pg_dyn[];
    __shared__ PgSmem sm;
    __shared__ uint32_t tmem_base;
    if (smem_u32(pg_dyn) & 1023) {   // the swizzle goes by addresses; the alignment above is there, so this does not happen
        g_device_status = 2;
        return;
    }
    if (threadIdx.x == 0) pg_init(sm);
    pg_begin(&tmem_base, kPgTmemCols);
    pg_tiles<T, D, kBias>(&map_q, &map_k, &map_v, a, ws, 1, whole, (int)blockIdx.x, (int)gridDim.x, (int)gridDim.x, sm, tmem_base, pg_dyn);
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
