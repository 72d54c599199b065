// Attention of few new tokens over a paged cache (decode steps, guessed tokens): up to 16 rows a kv head, a row being a (token,
// query head) pair that shares it.
//
// Bound: HBM, the keys and values of every sequence once.  So that everything else fits behind that, the products are turned
// round - keys and dims are the 128 rows of the tensor core's tile, the few query rows its columns:
//   S^T [128 keys][16] = K.Q^T       both K-major from shared memory
//   O^T [dims][16] += V^T.P^T        V as an MN-major A operand straight from its [key][dim] tile, P K-major from shared memory
// (queries as the 128 rows, as in paged_tc.cu, spend an exponential on every one of 128 x 128 scores of which 1 to 16 rows count:
// 64 sequences of 200 to 8000 tokens, 32 / 8 heads: 140 us, of which the transfer needs 81).
//
// One CTA per SM, its share of the work as paged_share.cuh says:
//   warps 0-3, 4-7  softmax, two groups that take the pieces of the share in turn, so that the beginning of one runs beside the end
//              of the one before (2.7 us a piece when there was one group): a thread per key = TMEM lane.  The powers are taken
//              under a reference per row that all threads share; it moves only when a score has outgrown it by 2^8 (one vote of the
//              128 threads a block tells), so that no maximum crosses the threads in the usual block.  Sums stay with the threads
//              until the end.
//   warp 8     producer: Q, then K and V blocks of 128 keys through two rings of 32 KiB stages
//   warp 9     one thread issues the products; scores and probabilities have two buffers, so that S of the next block - of the next
//              piece, too - is there when the softmax of this one ends
//
// Measured: 64 sequences of 200 to 8000 tokens, 32 / 8 heads, bf16 92 us = 5.7 TB/s with everything around it; two of 60000 to 100000, 64 / 8
// heads 114 us, 2760 cycles a block and SM in the loop = 6.5 TB/s.
// Keys that no row sees may be anything, even NaN: masked by selection, their rows of V set to zero before the product.
#include "paged_share.cuh"

namespace eet {

namespace {

constexpr int kPwRows = 16;          // rows of a tile: the fewest columns that a product with 128 rows has
constexpr int kPwThreads = 320;
constexpr int kPwExtra = 2;         // a piece's beginning and end cost as much as two blocks

template<int D>
struct PwShape {
    static constexpr int kHalves = D / 64;
    static constexpr int kTile = kHalves * kPgKeys * 128;                    // a K or V block
    static constexpr int kStages = D == 64 ? 4 : 3;                          // blocks in flight, K and V each
    static constexpr int kQ = kHalves * kPwRows * 128;                       // rows of Q; two of them
    static constexpr int kP = 2 * kPwRows * 128;                             // probabilities [2 x 64 keys][16]; two of them a group
    static constexpr int kSmem = 2 * kStages * kTile + 2 * kQ + 4 * kP;
    static constexpr uint32_t kTmemCols = 128;                               // two S, one O of either group: 96
};

// What the four warps of a softmax group know of their piece, by row.
struct PwRows {
    int low[kPwRows], high[kPwRows];   // keys that a row sees
    float slope[kPwRows];         // of the bias, to the power of two
    int pos[kPwRows];             // its position
    long long out_at[kPwRows];    // where its result goes
    float ref[kPwRows];           // the reference of its powers, as a power of two, less kUp
    float corr[kPwRows];          // what a moved reference takes from the sums so far; at the end 1 / sum
};

struct PwSmem {
    uint64_t q_full[2], q_empty[2];
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];   // block i of the CTA is in stage i % kStages
    uint64_t s_full[2][2];      // [group][buffer]: S^T of a block has been computed
    uint64_t p_ready[2][2];     // its probabilities are there (four warps)
    uint64_t pv_done[2][2];     // its V^T.P^T has completed
    uint64_t o_free[2];         // O of a piece has been read (four warps)
    volatile int abort;
    PwRows rows[2];
    PgFound found;
};

// Barrier of the four warps of a softmax group: whether any thread says so.
__device__ __forceinline__ bool pw_any(int group, bool p)
{
    uint32_t r;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}\n"
        : "=r"(r)
        : "r"((uint32_t)p), "r"(1 + group)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ void tmem_st8_async(uint32_t taddr, const uint32_t (&v)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// By one thread, in front of a barrier.
template<int D>
__device__ __forceinline__ void pw_init(PwSmem& sm)
{
    for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.q_full[i], 1);
        mbar_init(&sm.q_empty[i], 1);
        for (int buf = 0; buf < 2; ++buf) {
            mbar_init(&sm.s_full[i][buf], 1);
            mbar_init(&sm.p_ready[i][buf], 4);
            mbar_init(&sm.pv_done[i][buf], 1);
        }
        mbar_init(&sm.o_free[i], 4);
    }
    for (int i = 0; i < PwShape<D>::kStages; ++i) {
        mbar_init(&sm.k_full[i], 1);
        mbar_init(&sm.k_empty[i], 1);
        mbar_init(&sm.v_full[i], 1);
        mbar_init(&sm.v_empty[i], 1);
    }
    sm.abort = 0;
    mbar_fence_init();
}

// The work of CTA `cta` of `ctas`; the scratch is laid out for `region` of them.
template<typename T, int D>
__device__ __forceinline__ void pw_rows(const CUtensorMap* map_q, const CUtensorMap* map_k, const CUtensorMap* map_v, const PagedMhaArgs& a,
                                        void* ws, int most, int whole, int cta, int ctas, int region, PwSmem& sm, const uint32_t& tmem_base,
                                        uint8_t* dyn)
{
    using Shape = PwShape<D>;
    constexpr int kHalves = Shape::kHalves, kTile = Shape::kTile, kStages = Shape::kStages, kHalf = kPgKeys * 128;
    uint8_t* k_ring = dyn;
    uint8_t* v_ring = k_ring + kStages * kTile;
    uint8_t* q_rows = v_ring + kStages * kTile;
    uint8_t* p_rows = q_rows + 2 * Shape::kQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    const int tile_tokens = kPwRows / group;
    const PgTiling tiling = {tile_tokens, 1, most, kPwExtra};

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
        int k_loads = 0, v_loads = 0, pieces = 0;
        bool ok = true;
        // K of a block goes out before V of the one in front, in the order of their use.
        const int* v_row = nullptr;
        int v_head = 0, v_key0 = 0, v_page = 0;
        PgSpan v_span = {0, 0};
        auto load_v = [&]() -> bool {
            const int stage = v_loads % kStages;
            if (!tc_wait_warp(&sm.v_empty[stage], (uint32_t)((v_loads / kStages + 1) & 1), &sm.abort)) return false;
            PgLoader<D>{a, v_row, v_head, v_span}.load(map_v, v_key0, v_page, v_ring + stage * kTile, &sm.v_full[stage]);
            ++v_loads;
            return true;
        };
        const PgShare all = share;
        while (ok && share.next(a, tiling, p)) {
            if (p.blocks == 0) continue;
            const PgSpan span = pg_span(a, p.s, p.tile * tile_tokens, (p.tile + 1) * tile_tokens);
            const PgLoader<D> loader = {a, a.pages + p.seq * a.pages_stride, p.head, span};
            int page = loader.page(p.top * kPgKeys);
            const int qb = pieces & 1;
            if (pieces > 1 && !tc_wait_warp(&sm.q_empty[qb], (uint32_t)((pieces / 2 - 1) & 1), &sm.abort)) break;
            ++pieces;
            if (lane == 0) mbar_arrive_expect_tx(&sm.q_full[qb], (uint32_t)(tile_tokens * group * 128 * kHalves));
            __syncwarp();
            if (lane < kHalves) {
                tma_load_3d(q_rows + qb * Shape::kQ + lane * kPwRows * 128, map_q, 64 * lane, p.head * group, p.s.row0 + p.tile * tile_tokens,
                            &sm.q_full[qb]);
            }
            if (p.s.p0 + p.s.tokens > cap && lane == 0) g_device_status = 6;
            for (int j = 0; j < p.blocks && ok; ++j) {
                const int key0 = (p.top - j) * kPgKeys;
                const int next = j + 1 < p.blocks ? loader.page(key0 - kPgKeys) : 0;
                const int stage = k_loads % kStages;
                ok = tc_wait_warp(&sm.k_empty[stage], (uint32_t)((k_loads / kStages + 1) & 1), &sm.abort);
                if (!ok) break;
                loader.load(map_k, key0, page, k_ring + stage * kTile, &sm.k_full[stage]);
                if (k_loads++ > 0) ok = load_v();
                v_row = loader.row;
                v_head = p.head;
                v_span = span;
                v_key0 = key0;
                v_page = page;
                page = next;
            }
        }
        if (ok && k_loads > 0) load_v();
        if (!whole && lane == 0) pg_write_header(a, tiling, ws, cta, ctas, true, all, place);
        if (sm.abort) {
            // nothing of this CTA may still be on its way when it ends
            for (int i = max(0, k_loads - kStages); i < k_loads; ++i) {
                mbar_wait_bounded(&sm.k_full[i % kStages], (uint32_t)((i / kStages) & 1));
            }
            for (int i = max(0, v_loads - kStages); i < v_loads; ++i) {
                mbar_wait_bounded(&sm.v_full[i % kStages], (uint32_t)((i / kStages) & 1));
            }
            for (int i = max(0, pieces - 2); i < pieces; ++i) mbar_wait_bounded(&sm.q_full[i & 1], (uint32_t)((i / 2) & 1));
        }
    }
    else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issuer
        if (elect_one()) {
            constexpr uint32_t idesc_qk = umma_idesc_f16(kPgKeys, kPwRows) | PgType<T>::idesc;
            constexpr uint32_t idesc_pv = umma_idesc_f16(128, kPwRows) | PgType<T>::idesc | (1u << 15);   // A (V^T) MN-major
            const uint64_t q_desc = umma_desc_sw128(smem_u32(q_rows));
            const uint64_t p_desc = umma_desc_sw128(smem_u32(p_rows));
            const uint64_t k_desc = umma_desc_sw128(smem_u32(k_ring));
            // (heads of 64: the tile's upper 64 rows read the same dims once more, nobody reads their sums)
            const uint64_t v_desc = umma_desc_mn_sw128(smem_u32(v_ring), D == 128 ? (uint32_t)kHalf : 0u);
            int k_stage = 0, v_stage = 0;
            uint32_t k_phase = 0, v_phase = 0;
            int done[2] = {0, 0};           // blocks of either group whose scores have been asked for
            // S^T of block j of piece number i (of n blocks), which is the next that has been loaded
            auto issue_qk = [&](int i, int j, int n) -> bool {
                const int x = i & 1;
                if (j == 0 && !tc_wait(&sm.q_full[x], (uint32_t)((i / 2) & 1), &sm.abort)) return false;
                if (!tc_wait(&sm.k_full[k_stage], k_phase, &sm.abort)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int buf = (x ? done[1] : done[0]) & 1;
                const uint64_t kd = k_desc + (uint64_t)(k_stage * (kTile >> 4)), qd = q_desc + (uint64_t)(x * (Shape::kQ >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    umma_f16(tmem + (uint32_t)(x * 3 * kPwRows + buf * kPwRows), kd + (uint64_t)((kk >> 2) * (kHalf >> 4) + (kk & 3) * 2),
                             qd + (uint64_t)((kk >> 2) * (kPwRows * 128 >> 4) + (kk & 3) * 2), idesc_qk, kk != 0);
                }
                umma_commit(&sm.s_full[x][buf]);
                umma_commit(&sm.k_empty[k_stage]);
                if (j == n - 1) umma_commit(&sm.q_empty[x]);
                if (x) ++done[1];
                else ++done[0];
                if (++k_stage == kStages) {
                    k_stage = 0;
                    k_phase ^= 1;
                }
                return true;
            };
            auto next_piece = [&](int& n) -> bool {   // that has keys to read
                while (share.next(a, tiling, p)) {
                    n = p.blocks;
                    if (n > 0) return true;
                }
                return false;
            };
            // Scores are asked for one block ahead of the probabilities, across the pieces: those of a piece's first block are there
            // when the other group begins it.  They go where those of two blocks before were, which have been read then.
            int n = 0, next_n = 0;
            bool ok = next_piece(n) && issue_qk(0, 0, n);
            for (int i = 0; ok; ++i) {
                const int x = i & 1;
                const uint32_t tmem_o = tmem + (uint32_t)(x * 3 * kPwRows + 2 * kPwRows);
                int block = (x ? done[1] : done[0]) - 1;      // of this group
                bool more = true;
                for (int j = 0; j < n && ok; ++j, ++block) {
                    if (j + 1 < n) ok = issue_qk(i, j + 1, n);
                    else if ((more = next_piece(next_n))) ok = issue_qk(i + 1, 0, next_n);
                    if (ok && j == 0 && i > 1) ok = tc_wait(&sm.o_free[x], (uint32_t)((i / 2 - 1) & 1), &sm.abort);
                    ok = ok && tc_wait(&sm.v_full[v_stage], v_phase, &sm.abort) &&
                         tc_wait(&sm.p_ready[x][block & 1], (uint32_t)((block >> 1) & 1), &sm.abort);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t vd = v_desc + (uint64_t)(v_stage * (kTile >> 4)),
                                   pd = p_desc + (uint64_t)((2 * x + (block & 1)) * (Shape::kP >> 4));
#pragma unroll
                    for (int kk = 0; kk < kPgKeys / 16; ++kk) {
                        umma_f16(tmem_o, vd + (uint64_t)(kk * (2048 >> 4)), pd + (uint64_t)((kk >> 2) * (kPwRows * 128 >> 4) + (kk & 3) * 2),
                                 idesc_pv, j != 0 || kk != 0);
                    }
                    umma_commit(&sm.pv_done[x][block & 1]);
                    umma_commit(&sm.v_empty[v_stage]);
                    if (++v_stage == kStages) {
                        v_stage = 0;
                        v_phase ^= 1;
                    }
                }
                if (!more) break;
                n = next_n;
            }
        }
    }
    else {
        // ------------------------------------------------------------------ softmax, epilogue
        const int x = warp >> 2;                              // pieces go to the two groups in turn
        const int r = (warp & 3) * 32 + lane;                 // key of the block, and dim of O
        const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + t_lane + (uint32_t)(x * 3 * kPwRows), tmem_o = tmem_s + 2 * kPwRows;
        constexpr float kUp = PgType<T>::kUp;
        const float log2e = 1.4426950408889634f;
        const float to_log2 = a.scale * log2e;
        const int cap = (int)min((long long)a.max_pages << a.page_shift, 0x7fffffffLL);
        PwRows& row = sm.rows[x];
        uint8_t* p_mine = p_rows + x * 2 * Shape::kP;
        float* cross = reinterpret_cast<float*>(p_mine);      // [kPwRows][128], for what crosses the threads while no product reads P
        int before = 0;                                       // blocks of the share in front of the piece
        int block = 0;                                        // blocks that this group has done
        int pieces = 0;
        bool ok = true, failed = false;                       // this thread's waits; what the group has agreed on: all leave together
        while (share.next(a, tiling, p)) {
            const bool mine = p.blocks > 0 ? (pieces & 1) == x : x == 0;
            pieces += p.blocks > 0;
            const int first_block = before;
            before += p.blocks;
            if (!mine) continue;
            const int token0 = p.tile * tile_tokens;
            const int rows = min(tile_tokens, p.s.tokens - token0) * group;
            const PgSpan span = pg_span(a, p.s, token0, token0 + tile_tokens);
            // (everybody has left the piece before: its last barrier stands behind the last use of these)
            if (r < kPwRows) {
                const int pos = p.s.p0 + token0 + r / group;
                row.pos[r] = pos;
                row.low[r] = a.window > 0 ? (int)max((long long)p.s.first, (long long)pos - a.window + 1) : p.s.first;
                row.high[r] = r < rows ? min(pos, cap - 1) : -1;
                row.slope[r] = a.slopes != nullptr && r < rows ? a.slopes[p.head * group + r % group] * log2e : 0.f;
                row.out_at[r] = (long long)(p.s.row0 + token0 + r / group) * a.o_tok + (long long)(p.head * group + r % group) * a.o_head;
                row.ref[r] = kPgNone;
            }
            pw_any(x, false);
            // blocks all of whose keys every row sees
            const int all_low = row.low[rows - 1], all_high = row.high[0];
            float l[kPwRows];
#pragma unroll
            for (int n = 0; n < kPwRows; ++n) l[n] = 0.f;
            for (int j = 0; j < p.blocks; ++j, ++block) {
                const int key0 = (p.top - j) * kPgKeys, key = key0 + r;
                const int buf = block & 1;
                ok = tc_wait_warp(&sm.s_full[x][buf], (uint32_t)((block >> 1) & 1), &sm.abort) && ok;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float t[kPwRows];
                {
                    uint32_t u[kPwRows];
                    tmem_ld16(tmem_s + (uint32_t)(buf * kPwRows), u);
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) t[n] = __uint_as_float(u[n]);
                }
                if (a.slopes != nullptr) {
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) t[n] = fmaf(t[n], to_log2, row.slope[n] * (float)(key - row.pos[n]));
                }
                else {
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) t[n] *= to_log2;
                }
                if (all_low <= key0 && all_high >= key0 + kPgKeys - 1) {
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) t[n] = n < rows ? t[n] : -INFINITY;
                }
                else {
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) t[n] = key >= row.low[n] && key <= row.high[n] ? t[n] : -INFINITY;
                }
                bool over = j == 0;
#pragma unroll
                for (int n = 0; n < kPwRows; ++n) over |= t[n] - row.ref[n] > kPgLag + kUp;
                // the buffer that the probabilities go to has been read by the product of two blocks before
                if (block > 1) ok = tc_wait_warp(&sm.pv_done[x][buf], (uint32_t)(((block >> 1) - 1) & 1), &sm.abort) && ok;
                if (pw_any(x, over || !ok)) {
                    // Some row's reference moves (or a wait has run out: all leave together).
                    if (j > 0) ok = tc_wait_warp(&sm.pv_done[x][buf ^ 1], (uint32_t)(((block - 1) >> 1) & 1), &sm.abort) && ok;
                    // (no product reads the probabilities now: their place holds the scores for a moment, row by row)
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) cross[n * kPgKeys + r] = t[n];
                    failed = pw_any(x, !ok);
                    if (failed) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    // (eight lanes a row: four rows of a warp at once)
                    {
                        const int n = (warp & 3) * 4 + (lane >> 3);
                        const float4* v = reinterpret_cast<const float4*>(cross + n * kPgKeys) + (lane & 7);
                        float m = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fmaxf(v[8 * i].x, v[8 * i].y), fmaxf(v[8 * i].z, v[8 * i].w)));
#pragma unroll
                        for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        if ((lane & 7) == 0) {
                            const float old = row.ref[n];
                            const bool moves = m - old > kPgLag + kUp;
                            row.corr[n] = moves ? ex2_approx(old - (m - kUp)) : 1.0f;
                            row.ref[n] = moves ? m - kUp : old;
                        }
                    }
                    pw_any(x, false);
#pragma unroll
                    for (int n = 0; n < kPwRows; ++n) l[n] *= row.corr[n];
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < kPwRows; c += 8) {
                            uint32_t o[8];
                            tmem_ld8(tmem_o + (uint32_t)c, o);
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * row.corr[c + i]);
                            tmem_st8_async(tmem_o + (uint32_t)c, o);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                }
                // probabilities: row n of P holds 64 keys in 128 bytes, 16-byte pieces swizzled by n
                uint8_t* dst = p_mine + buf * Shape::kP + (r >> 6) * (kPwRows * 128) + (r & 7) * 2;
                const int piece = (r & 63) >> 3;
#pragma unroll
                for (int n = 0; n < kPwRows; ++n) {
                    // (the sum is of the rounded ones: where one key has most of the weight, its rounding then cancels)
                    const T e = (T)ex2_approx(t[n] - row.ref[n]);
                    l[n] += (float)e;
                    *reinterpret_cast<T*>(dst + n * 128 + ((piece ^ (n & 7)) << 4)) = e;
                }
                if (key0 < span.lo || key0 + kPgKeys > span.hi) {
                    // rows of V that nobody sees (late: V lands behind K, and this is the first block of most pieces)
                    const int v_stage = (first_block + j) % kStages;
                    const uint32_t parity = (uint32_t)(((first_block + j) / kStages) & 1);
                    ok = tc_wait_warp(&sm.v_full[v_stage], parity, &sm.abort) && ok;   // (told at the next barrier)
                    if (key < span.lo || key >= span.hi) {
                        uint4* zero = reinterpret_cast<uint4*>(v_ring + v_stage * kTile + r * 128);
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) zero[h * (kHalf / 16) + c] = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[x][buf]);
            }
            if (failed) break;

            // ---- epilogue: the sums of the threads, then O, a dim a thread
            if (p.blocks > 0) ok = tc_wait_warp(&sm.pv_done[x][(block - 1) & 1], (uint32_t)(((block - 1) >> 1) & 1), &sm.abort) && ok;
#pragma unroll
            for (int n = 0; n < kPwRows; ++n) cross[n * kPgKeys + r] = l[n];
            if (pw_any(x, !ok)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool complete = p.starts && p.ends;
            const PgPartial part = pg_partial(ws, region, cta, p.starts ? 1 : 0, kPwRows, D);
            {
                const int n = (warp & 3) * 4 + (lane >> 3);
                const float4* v = reinterpret_cast<const float4*>(cross + n * kPgKeys) + (lane & 7);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += (v[8 * i].x + v[8 * i].y) + (v[8 * i].z + v[8 * i].w);
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if ((lane & 7) == 0) {
                    row.corr[n] = sum == 0.f ? 0.f : 1.0f / sum;
                    if (!complete) {
                        part.max2[n] = row.ref[n];
                        part.sum[n] = sum;
                    }
                }
            }
            pw_any(x, false);
#pragma unroll 1
            for (int c = 0; c < rows; c += 8) {
                uint32_t o[8] = {};
                if (p.blocks > 0) tmem_ld8(tmem_o + (uint32_t)c, o);
                if (r < D) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (c + i < rows) {
                            const float v = __uint_as_float(o[i]), inv = row.corr[c + i];
                            if (!complete) reinterpret_cast<float*>(part.o)[(c + i) * D + r] = v;
                            else ((T*)a.out)[row.out_at[c + i] + r] = (T)(inv == 0.f ? 0.f : v * inv);
                        }
                    }
                }
            }
            if (p.blocks > 0) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.o_free[x]);
            }
            pw_any(x, false);   // the row's values have been read
        }
    }
}

template<typename T, int D>
__global__ void __launch_bounds__(kPwThreads, 1)
paged_mha_rows_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedMhaArgs a, void* ws, int whole)
{
    extern __shared__ __align__(1024) uint8_t pw_dyn[];
    __shared__ PwSmem sm;
    __shared__ uint32_t tmem_base;
    if (smem_u32(pw_dyn) & 1023) {   // the swizzle goes by addresses; the alignment above is there, so this does not happen
        g_device_status = 2;
        return;
    }
    if (threadIdx.x == 0) pw_init<D>(sm);
    pg_begin(&tmem_base, PwShape<D>::kTmemCols);
    pw_rows<T, D>(&map_q, &map_k, &map_v, a, ws, 0x7fffffff, whole, (int)blockIdx.x, (int)gridDim.x, (int)gridDim.x, sm, tmem_base, pw_dyn);
    pg_end(&tmem_base, PwShape<D>::kTmemCols);
}

// Both kinds of work in one launch: sequences of up to `few` new tokens for the first CTAs, the others for the rest, as many as their blocks
// take of the time.  Measured, a block on one CTA (heads of 128): few rows 1.46 us with pages of 16 (32 copies of 2 KB), 0.85 with pages of
// 64 and more; tiles 1.9 us, with a bias and masks 3 to 3.5.  All CTAs together get a block of the first kind every 0.0106 us from HBM: more
// of them than use that up are better spent on the tiles.  The other constants below are estimates, and close: measured afterwards, 148
// histories in the same pages (so from L2), us a block and CTA
//   few rows, pages of 16 / 32 / 64 and more   heads of 128: 1.50 / 1.01 / 0.86     heads of 64: 1.00 / 0.83 / 0.84
//   tiles that need no masks, without / with a bias   heads of 128: 1.76 / 2.44     heads of 64: 1.68 / 2.43
// and with pages of their own, from HBM, 1.43 for heads of 128 (one every 0.0097 us) and 0.84, not bound by HBM, for heads of 64.
// (As two launches one chunk of 777 tokens beside 23 single ones, 40 heads, took 65 + 49 us, with HBM idle in the second.)
template<int D>
__device__ __forceinline__ int pg_divide(int ctas, float in_rows, float in_tiles, int page_shift, bool bias)
{
    if (!(in_rows > 0.f)) return 0;
    if (!(in_tiles > 0.f)) return ctas;
    const float per_row = (page_shift == 4 ? 1.46f : page_shift == 5 ? 1.1f : 0.85f) * (D == 64 ? 0.7f : 1.0f);
    const float per_tile = (bias ? 3.5f : 1.9f) * (D == 64 ? 0.7f : 1.0f);
    const float all_of_hbm = per_row / (D == 64 ? 0.0053f : 0.0106f);
    const float n = fminf((float)ctas * in_rows * per_row / (in_rows * per_row + in_tiles * per_tile), all_of_hbm);
    // An even number: two neighbouring CTAs share more of an instruction cache than they should with different code (as the two at an
    // odd border they took 126 and 131 us where the others had ended after 110).
    const int even = 2 * (int)(0.5f * n + 0.5f);
    return min(max(even, min(2, ctas - 1)), ctas - 1);
}

template<typename T, int D, bool kBias>
__global__ void __launch_bounds__(kPwThreads, 1)
paged_mha_both_kernel(const __grid_constant__ CUtensorMap map_q_rows, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ PagedMhaArgs a, void* ws_rows, void* ws, int few, int whole_rows, int whole)
{
    static_assert(kPwThreads == kPgThreads, "one launch serves both");
    extern __shared__ __align__(1024) uint8_t pb_dyn[];
    __shared__ __align__(16) uint8_t sm[sizeof(PgSmem) > sizeof(PwSmem) ? sizeof(PgSmem) : sizeof(PwSmem)];
    __shared__ uint32_t tmem_base;
    if (smem_u32(pb_dyn) & 1023) {
        g_device_status = 2;
        return;
    }
    pg_begin(&tmem_base, kPgTmemCols);   // for either kind: which one follows from what the kernel in front leaves
    const int group = a.heads / a.kv_heads, n = gridDim.x, cta = blockIdx.x;
    const PgTiling few_rows = {kPwRows / group, 1, few, kPwExtra}, tiles = {2 * (kPgRows / group), few + 1, 0x7fffffff, kPgExtra};
    const int n_rows = pg_divide<D>(n, (float)pg_total(a, few_rows), (float)pg_total(a, tiles), a.page_shift, kBias);
    // every header is written: those behind the CTAs of one kind by those of the other
    if (threadIdx.x == 0) {
        const PgHeader none = {};
        if (cta < n_rows && !whole) reinterpret_cast<PgHeader*>(ws)[n - n_rows + cta] = none;
        if (cta >= n_rows && !whole_rows) reinterpret_cast<PgHeader*>(ws_rows)[cta] = none;
    }
    if (threadIdx.x == 0) {
        if (cta < n_rows) pw_init<D>(*reinterpret_cast<PwSmem*>(sm));
        else pg_init(*reinterpret_cast<PgSmem*>(sm));
    }
    __syncthreads();
    if (cta < n_rows) {
        pw_rows<T, D>(&map_q_rows, &map_k, &map_v, a, ws_rows, few, whole_rows, cta, n_rows, n, *reinterpret_cast<PwSmem*>(sm), tmem_base,
                      pb_dyn);
    }
    else {
        pg_tiles<T, D, kBias>(&map_q, &map_k, &map_v, a, ws, few + 1, whole, cta - n_rows, n - n_rows, n, *reinterpret_cast<PgSmem*>(sm),
                              tmem_base, pb_dyn);
    }
    pg_end(&tmem_base, kPgTmemCols);
}

template<typename T, int D>
int pg_launch_rows(const PagedMhaArgs& a, void* ws, int whole, cudaStream_t stream)
{
    CUtensorMap map_q, map_k, map_v;
    if (int rc = pg_encode_maps<T, D>(a, kPwRows / (a.heads / a.kv_heads), &map_q, &map_k, &map_v)) return rc;
    auto kern = paged_mha_rows_kernel<T, D>;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    constexpr int kSmem = PwShape<D>::kSmem;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        attr_set[dev] = true;
    }
    EET_CUDA(launch_pdl(kern, dim3(sm_count()), dim3(kPwThreads), kSmem, stream, map_q, map_k, map_v, a, ws, whole));
    return 0;
}

template<typename T, int D, bool kBias>
int pg_launch_both(const PagedMhaArgs& a, void* ws_rows, void* ws, int few, int whole_rows, int whole, cudaStream_t stream)
{
    const int group = a.heads / a.kv_heads;
    CUtensorMap map_q_rows, map_q, map_k, map_v;
    if (int rc = pg_encode_maps<T, D>(a, kPwRows / group, &map_q_rows, &map_k, &map_v)) return rc;
    if (int rc = pg_encode_maps<T, D>(a, kPgRows / group, &map_q, &map_k, &map_v)) return rc;
    auto kern = paged_mha_both_kernel<T, D, kBias>;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    constexpr int kSmem = pg_tiles_smem(D) > PwShape<D>::kSmem ? pg_tiles_smem(D) : PwShape<D>::kSmem;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        attr_set[dev] = true;
    }
    EET_CUDA(launch_pdl(kern, dim3(sm_count()), dim3(kPwThreads), kSmem, stream, map_q_rows, map_q, map_k, map_v, a, ws_rows, ws,
                        few, whole_rows, whole));
    return 0;
}

}  // namespace

}  // namespace eet
