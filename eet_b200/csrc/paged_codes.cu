// Attention of few new tokens over a paged cache of 8-bit codes: up to kRows (8 or 16) rows a kv head, a row being a (token, query
// head) pair that shares it.
//
//   out = sum_j w_j c^v_j / sum_j w_j / s^v_j,   w_j = s^v_j 2^(s^k_j (q . c^k_j) scale log2(e) + slope (j - p) log2(e) - ref)
//
// The codes enter the products as fp16, where they are exact, and the scales stay outside: that of a key on its score, that of its
// value on its weight, before that is rounded to fp16 (the sum that divides is of the powers, which are not).  So that the weights fit
// fp16 whatever the scales are, the reference ref of a row follows the largest score + log2(s^v), not the largest score.  q of bf16 is
// multiplied by a power of two that brings its largest value to 2^14 and enters as fp16 too: eight bits of every value down to 2^-28 of
// the largest are kept.
//
// Bound: HBM, the codes and scales of every sequence once.  A block of 128 keys is half the bytes of a 16-bit one, and everything on
// the way has to keep up: pages of 16 slots are eight copies of 2 KiB a block, which the copy engine takes 85 cycles each for, so the
// warps copy themselves (cp.async), each into a ring of its own that nobody else waits for; and a code becomes a value in registers, in
// the layout in which mma.sync takes its 16-row operand, so that nothing is written back to shared memory:
//   S^T [16 keys][8] = K.Q^T       lane (g, t) = (lane / 4, lane % 4) holds dims 32 t .. 32 t + 31 of keys g and g + 8: which dims stand
//                                  for which index of the sum is free as long as Q's do the same
//   O^T [16 dims][8] += V^T.P^T    lane (g, t) holds dims 16 g .. 16 g + 15 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9; two keys' bytes are
//                                  interleaved to pairs, dims 16 g + 2 i and 16 g + 2 i + 1 are rows g and g + 8 of tile i
// P^T leaves S^T's layout by a transposition of 8 x 8 in the warp (movmatrix).  (Tensor memory and tcgen05 would need the values in shared
// memory: 64 KiB written and read again for every 32 KiB that arrive.)
//
// A CTA is four warps, 32 keys of a block each; three CTAs share an SM, two where there are 16 rows, so that the beginning and the end of a
// piece of one run beside the others' blocks.  The warps' sums meet in shared memory at the end of a piece.  The work is cut up as
// paged_share.cuh says.  Measured: 64 sequences of 200 to 8000 tokens, 32 / 8 heads, bf16 over int8, 66 us (75 with two CTAs), which is 4.1 TB/s;
// two of 60 and 100 thousand tokens, 64 / 8 heads, fp16 over e4m3, 71 us (4.6 TB/s).  What bounds it then is how fast three warps a scheduler
// go through their instructions: one in six cycles each (issue slots 46 % taken, 41 in the second case).  Of the six, 1.2 are fixed
// latencies, 1.1 instructions that are not there yet, 0.6 another warp's turn, 0.6 shared memory, 0.5 the pipe of conversions' and bytes'
// selections, the fullest one at 40 %, and 0.4 the copies (1.2 in the second case).
//
// Longer chunks go to tiles of 128 rows (paged_tc.cu has what a CTA does), in a kernel of their own behind the same plan.  Where a call has both kinds of
// sequences, the kernels run side by side on parts of the SMs, divided by what a block takes on either, and one launch adds up the parts of both.
#include <type_traits>

#include "codes.cuh"
#include "paged_share.cuh"

namespace eet {

namespace {

constexpr int kPcExtra = 2;                     // a piece's beginning and end cost as much as two blocks

// Scales of values below 2^-90 count as that where a reference is chosen.  The powers, of which the sum that divides is, then end at 2^(90 + 15),
// and 2^22 of them are still a number in fp32; weights are good to 11 bits down to scales of 2^-111, to fewer below that (bf16 values of 10^-31).
// With 2^-60 bf16 values below 10^-16 came out as zeros.
constexpr float kPcLeastScale = 8.07793567e-28f;

template<int D, int kRows>
struct PcShape {
    static constexpr int kWarps = 4;
    static constexpr int kKeys = kPgKeys / kWarps;                      // of a block, for a warp: one or two runs of 16
    static constexpr int kAtOnce = kRows == 8 ? 2 : 1;                  // runs that are worked on together
    static constexpr int kPerSm = kRows == 8 ? 3 : 2;                   // CTAs
    static constexpr int kStages = kRows == 8 && D == 128 ? 2 : 3;
    static constexpr int kTile = kKeys * D;                             // bytes: a warp's codes of K or V of a block
    static constexpr int kStage = 2 * kTile + 2 * kKeys * 4;            // and the scales
    static constexpr int kSmem = kWarps * kStages * kStage;
    static_assert(kStage >= kRows * D * 4, "the sums of a warp fit where its codes were");
};

constexpr int pc_per_sm(int rows) { return rows == 8 ? PcShape<128, 8>::kPerSm : PcShape<128, 16>::kPerSm; }

// What a warp knows of the rows of its piece, out of its registers: few blocks ask for it.
struct PcRows {
    int low[16], high[16];        // keys that a row sees
    int pos[16];
    float slope[16];              // of the bias, to the power of two
};

struct PcSmem {
    PcRows rows[8];
    PgShare share[8];
    PgPiece piece[8][2];          // of a warp: the one at work and the one behind it
    float ref[8][16], sum[8][16];
    PgFound found;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint2 lds64(uint32_t at)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}

// Where 16 bytes of a row lie in a tile: swizzled, so that neither of the two ways of reading meets a bank twice.
template<int D>
__device__ __forceinline__ uint32_t pc_place(int row, int chunk)
{
    if (D == 128) return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
    return (uint32_t)((row >> 1) * 128 + ((((row & 1) * 4 + chunk) ^ (row & 6)) << 4));
}

// What a warp copies: its keys of a block of a piece.
template<int D, int kRows>
struct PcCopies {
    using Shape = PcShape<D, kRows>;
    static constexpr int kRuns = Shape::kKeys / 16;
    const PagedMhaArgs& a;
    uint32_t ring;                // of this warp
    int offset;                   // of its keys in a block

    // The pages of its runs of 16 keys, of the block at key0, in the lanes 0 .. 15 and 16 .. 31, as the table has them; -1: nobody sees them.
    // (Nothing looks at them before the copies: a trip to L2 that they would wait for with every block.)
    __device__ __forceinline__ int page(const int* row, int lo, int hi, int key0) const
    {
        const int key = key0 + offset + (kRuns == 2 ? (int)(threadIdx.x & 16) : 0);
        return key < hi && key + 16 > lo ? row[key >> a.page_shift] : -1;
    }
    // Keys that the tile does not see, and pages outside the cache, become zeros: codes and scales there may be anything.
    __device__ __forceinline__ void issue(int head, int lo, int hi, int key0, int page, int stage) const
    {
        constexpr int kChunks = D / 16, kRowsAtOnce = 32 / kChunks, kTimes = 16 / kRowsAtOnce;
        const int lane = threadIdx.x & 31, row0 = lane / kChunks, c = lane % kChunks;
        const uint32_t at = ring + (uint32_t)(stage * Shape::kStage);
#pragma unroll 1
        for (int run = 0; run < kRuns; ++run) {
            int n = kRuns == 2 ? __shfl_sync(0xffffffffu, page, 16 * run) : page;
            const int key = key0 + offset + 16 * run, slot = key & ((1 << a.page_shift) - 1);
            if (n < 0 || n >= a.num_pages) {
                if (key < hi && key + 16 > lo) g_device_status = 6;
                n = -1;
            }
            const long long page_at = max(n, 0);
            const uint8_t* k = (const uint8_t*)a.k_cache + page_at * a.kc_page + head * a.kc_head + (slot + row0) * a.kc_slot + 16 * c;
            const uint8_t* v = (const uint8_t*)a.v_cache + page_at * a.vc_page + head * a.vc_head + (slot + row0) * a.vc_slot + 16 * c;
            // a half of the warp for the scales of either
            const float* scale = (lane < 16 ? a.k_scale + page_at * a.ks_page + head * a.ks_head
                                            : a.v_scale + page_at * a.vs_page + head * a.vs_head) + slot + (lane & 15);
            const uint32_t to = at + (uint32_t)(16 * run * D) + pc_place<D>(row0, c);
            // (nothing is read where a size is zero; the addresses stay inside the cache)
            const int from = n < 0 ? 16 : lo - key, upto = hi - key;
            const long long k_step = kRowsAtOnce * a.kc_slot, v_step = kRowsAtOnce * a.vc_slot;
#pragma unroll
            for (int i = 0; i < kTimes; ++i) {
                const int r = row0 + kRowsAtOnce * i;
                const uint32_t bytes = r >= from && r < upto ? 16 : 0;
                const uint32_t to_i = (D == 128 ? to ^ (uint32_t)((kRowsAtOnce * i & 7) << 4) : to) + kRowsAtOnce * i * D;   // (a row's swizzle)
                copy16_async(to_i, k, bytes);
                copy16_async(to_i + Shape::kTile, v, bytes);
                k += k_step;
                v += v_step;
            }
            const int r = lane & 15;
            copy4_async(at + 2 * Shape::kTile + (uint32_t)(((lane < 16 ? 0 : Shape::kKeys) + 16 * run + r) * 4), scale,
                        r >= from && r < upto ? 4 : 0);
        }
    }
};

// Both kinds of work at once: sequences of up to `few` new tokens for the kernel of few rows, the others for tiles of 128, each on a part of the
// SMs that goes by what their blocks take (measured with heads of 128: 1.0 us a block with an SM's three CTAs, 2.7 as a pair of tiles, 3.5
// with a bias).  The kernel of tiles is launched first: a CTA of it fills an SM, those without work leave theirs, and the three of the
// other kernel go where there is room - which they find by themselves, since that one does not wait for this one before its end.  So
// this one lets it begin only when the kernels in front have ended for sure.
struct PcSplit {
    int sms_rows, sms_tiles;
};

__device__ __forceinline__ PcSplit pc_split(const PagedMhaArgs& a, int rows_tokens, int few, int sms, bool bias)
{
    const PgTiling rows = {rows_tokens, 1, few, kPcExtra}, tiles = {2 * (kPgRows / (a.heads / a.kv_heads)), few + 1, 0x7fffffff, kPgExtra};
    const float in_rows = (float)pg_total(a, rows), in_tiles = (float)pg_total(a, tiles) * (bias ? 3.5f : 2.7f);
    if (!(in_rows > 0.f)) return {0, sms};
    if (!(in_tiles > 0.f)) return {sms, 0};
    const int n = min(max((int)(sms * in_rows / (in_rows + in_tiles) + 0.5f), 1), sms - 1);
    return {n, sms - n};
}

template<int kCodes, int D, int kRows>
__global__ void __launch_bounds__(32 * PcShape<D, kRows>::kWarps, PcShape<D, kRows>::kPerSm)
paged_mha_codes_kernel(const __grid_constant__ PagedMhaArgs a, void* ws, int few, int beside, int whole)
{
    using Shape = PcShape<D, kRows>;
    constexpr int kN = kRows / 8;                // tiles of 8 rows
    constexpr int kSteps = D / 16;               // of the sum over dims; tiles of 16 dims
    constexpr float kUp = PgType<__half>::kUp;
    constexpr float kLog2e = 1.4426950408889634f;
    extern __shared__ __align__(1024) uint8_t pc_dyn[];
    __shared__ PcSmem sm;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads, tile_tokens = kRows / group;
    const int cta = blockIdx.x, region = gridDim.x;
    const PgTiling tiling = {tile_tokens, 1, few, kPcExtra};
    pdl_launch_dependents();
    // (beside the kernel of tiles: that one has waited already, and its end is waited for at the end)
    if (!beside) pdl_wait();
    const int ctas = beside ? Shape::kPerSm * pc_split(a, tile_tokens, few, region / Shape::kPerSm, beside > 1).sms_rows : region;
    if (cta >= ctas) {
        if (!whole && threadIdx.x == 0) reinterpret_cast<PgHeader*>(ws)[cta] = {};
        pdl_wait();
        return;
    }
    {
        PgShare share;
        PgPlace place;
        const bool work = pg_find_share(a, tiling, cta, ctas, whole != 0, sm.found, share, place);
        if (!whole && threadIdx.x == 0) pg_write_header(a, tiling, ws, cta, ctas, work, share, place);
        if (!work) {
            pdl_wait();
            return;
        }
        if (lane == 0) sm.share[warp] = share;
        __syncwarp();
    }
    PcRows& row_of = sm.rows[warp];
    auto span_of = [&](const PgPiece& p) { return pg_span(a, p.s, p.tile * tile_tokens, (p.tile + 1) * tile_tokens); };
    // walks on: the piece into place `which`; false: there is none
    auto walk = [&](int which) -> bool {
        PgShare share = sm.share[warp];
        PgPiece p;
        const bool any = share.next(a, tiling, p);
        __syncwarp();
        if (lane == 0) {
            sm.share[warp] = share;
            if (any) sm.piece[warp][which] = p;
        }
        __syncwarp();
        return any;
    };
    const PcCopies<D, kRows> copies = {a, smem_u32(pc_dyn) + (uint32_t)(warp * Shape::kStages * Shape::kStage), warp * Shape::kKeys};

    // The copies run some blocks ahead of the work, into the piece behind the one at work but not beyond.
    int now = 0;                   // place of the piece at work
    bool have_next = false;
    int copy_key0 = 0, copy_left = 0, copy_lo = 0, copy_hi = 0, copy_head = 0, page = -1;   // what is copied next; copy_left blocks of it
    const int* copy_row = nullptr;
    bool copy_next = false;        // it is the piece behind
    int ahead = 0, into = 0;       // blocks copied and not worked on; the next one's stage
    int stage = 0;                 // of the next block to work on
    auto copy_from = [&](int which) {
        const PgPiece& p = sm.piece[warp][which];
        const PgSpan span = span_of(p);
        copy_key0 = p.top * kPgKeys, copy_left = p.blocks, copy_lo = span.lo, copy_hi = span.hi, copy_head = p.head;
        copy_row = a.pages + p.seq * a.pages_stride;
        copy_next = which != now;
        if (copy_left > 0) page = copies.page(copy_row, copy_lo, copy_hi, copy_key0);
    };
    bool more = walk(0);
    if (more) {
        have_next = walk(1);
        copy_from(0);
        if (copy_left == 0 && have_next) copy_from(1);
    }

    while (more) {
        const PgPiece& p = sm.piece[warp][now];
        const int token0 = p.tile * tile_tokens, blocks = p.blocks;
        const int rows = min(tile_tokens, p.s.tokens - token0) * group;
        const PgSpan span = span_of(p);
        int all_low, all_high;     // keys that every row sees
        {
            const long long cap = (long long)a.max_pages << a.page_shift;
            const int last = (int)min(cap, 0x7fffffffLL) - 1;      // position that has a place in the table
            if (p.s.p0 + p.s.tokens > cap && threadIdx.x == 0) g_device_status = 6;
            __syncwarp();
            if (lane < kRows) {
                const bool valid = lane < rows;
                const int pos = p.s.p0 + token0 + lane / group;
                row_of.pos[lane] = pos;
                row_of.low[lane] = !valid ? 0 : a.window > 0 ? (int)max((long long)p.s.first, (long long)pos - a.window + 1) : p.s.first;
                row_of.high[lane] = valid ? min(pos, last) : 0x7fffffff;   // (a row that stands for no token takes what comes)
                row_of.slope[lane] = a.slopes != nullptr && valid ? a.slopes[p.head * group + lane % group] * kLog2e : 0.f;
            }
            __syncwarp();
            all_low = row_of.low[rows - 1], all_high = row_of.high[0];
        }
        // Q: lane (g, t) holds dims D / 4 t .. of rows g, and what of rows 2 t and 2 t + 1 the scores need
        uint32_t q[kN][kSteps][2];
        float factor[kN][2], ref[kN][2], l[kN][2];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            const int r = 8 * n + g;
            uint32_t* w = &q[n][0][0];
#pragma unroll
            for (int i = 0; i < 2 * kSteps; ++i) w[i] = 0u;
            if (r < rows) {
                const uint16_t* src = (const uint16_t*)a.q + (size_t)(p.s.row0 + token0 + r / group) * a.q_tok +
                                      (size_t)(p.head * group + r % group) * a.q_head + t * (D / 4);
#pragma unroll
                for (int i = 0; i < kSteps / 2; ++i) {
                    const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * i);
                    w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
                }
            }
            int e = 0;             // what the row was multiplied with, as a power of two
            if (a.bf16) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 2 * kSteps; ++i) top = max(top, max(w[i] << 16 & 0x7fffffffu, w[i] & 0x7fff0000u));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // (in two factors, since 2^(14 - exponent) may lie outside fp32's range)
                e = top >= 0x00800000u ? 141 - (int)(top >> 23) : 140;
                const float f0 = __uint_as_float((uint32_t)(127 + e / 2) << 23), f1 = __uint_as_float((uint32_t)(127 + e - e / 2) << 23);
#pragma unroll
                for (int i = 0; i < 2 * kSteps; ++i) {
                    const __half2 h = __floats2half2_rn(__uint_as_float(w[i] << 16) * f0 * f1, __uint_as_float(w[i] & 0xffff0000u) * f0 * f1);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int down = __shfl_sync(0xffffffffu, e, 4 * (2 * t + i));
                factor[n][i] = a.scale * kLog2e * __uint_as_float((uint32_t)(127 - down / 2) << 23) *
                               __uint_as_float((uint32_t)(127 - (down - down / 2)) << 23);
                ref[n][i] = kPgNone;
                l[n][i] = 0.f;
            }
        }
        float o[kN][kSteps][4];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
            }
        }
        bool huge = false;
        int used = stage;          // stage of the piece's last block
        int key0 = p.top * kPgKeys + copies.offset;
        for (int j = 0; j < blocks; ++j, key0 -= kPgKeys) {
            __syncwarp();          // all lanes have read the block before, whose stage is the next to be copied to
            while (ahead < Shape::kStages && copy_left > 0) {
                copies.issue(copy_head, copy_lo, copy_hi, copy_key0, page, into);
                asm volatile("cp.async.commit_group;" ::: "memory");
                ++ahead;
                into = into == Shape::kStages - 1 ? 0 : into + 1;
                copy_key0 -= kPgKeys;
                if (--copy_left > 0) page = copies.page(copy_row, copy_lo, copy_hi, copy_key0);
                else if (!copy_next && have_next) copy_from(now ^ 1);
            }
            if (ahead >= Shape::kStages) asm volatile("cp.async.wait_group %0;" ::"n"(Shape::kStages - 1) : "memory");
            else if (ahead == Shape::kStages - 1) asm volatile("cp.async.wait_group %0;" ::"n"(Shape::kStages - 2) : "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            --ahead;
            used = stage;
            const uint32_t at = copies.ring + (uint32_t)(stage * Shape::kStage);
            stage = stage == Shape::kStages - 1 ? 0 : stage + 1;
            if (key0 >= span.hi || key0 + Shape::kKeys <= span.lo) continue;
            const bool masked = key0 < all_low || key0 + Shape::kKeys - 1 > all_high;
#pragma unroll 1
            for (int m0 = 0; m0 < Shape::kKeys / 16; m0 += Shape::kAtOnce) {
                constexpr int kM = Shape::kAtOnce;
                const uint32_t at_m = at + (uint32_t)(m0 * 16 * D);
                const int key_m = key0 + 16 * m0 + g;
                // ---- scores
                float s[kM][kN][4];
#pragma unroll
                for (int m = 0; m < kM; ++m) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[m][n][e] = 0.f;
                    }
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) {
                        const int c = D / 64 * t + h;
                        const uint4 x = lds128(at_m + 16 * m * D + pc_place<D>(g, c)), y = lds128(at_m + 16 * m * D + pc_place<D>(8 + g, c));
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t a0, a1, a2, a3;
                            codes_to_half<kCodes>(xs[i], a0, a2);
                            codes_to_half<kCodes>(ys[i], a1, a3);
#pragma unroll
                            for (int n = 0; n < kN; ++n) mma_m16n8k16(s[m][n], a0, a1, a2, a3, q[n][4 * h + i][0], q[n][4 * h + i][1]);
                        }
                    }
                }
                // ---- weights
                float vs[kM][2], top_scale = kPcLeastScale;   // (a scale of zero weighs nothing)
#pragma unroll
                for (int m = 0; m < kM; ++m) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t place = at + 2 * Shape::kTile + (uint32_t)((16 * (m0 + m) + 8 * i + g) * 4);
                        float ks;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks) : "r"(place));
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs[m][i]) : "r"(place + Shape::kKeys * 4));
                        top_scale = fmaxf(top_scale, vs[m][i]);
#pragma unroll
                        for (int n = 0; n < kN; ++n) {
#pragma unroll
                            for (int r = 0; r < 2; ++r) s[m][n][2 * i + r] *= ks * factor[n][r];
                        }
                    }
                }
                if (a.slopes != nullptr) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = 8 * n + 2 * t + r;
                            const float slope = row_of.slope[row], from = (float)(key_m - row_of.pos[row]);
#pragma unroll
                            for (int k = 0; k < 2 * kM; ++k) {
                                float& x = s[k >> 1][n][2 * (k & 1) + r];
                                x = fmaf(slope, from + 8.0f * k, x);
                            }
                        }
                    }
                }
                if (masked) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = 8 * n + 2 * t + r, low = row_of.low[row] - key_m, high = row_of.high[row] - key_m;
#pragma unroll
                            for (int k = 0; k < 2 * kM; ++k) {
                                if (8 * k < low || 8 * k > high) s[k >> 1][n][2 * (k & 1) + r] = -INFINITY;
                            }
                        }
                    }
                }
                // (with the largest scale of the lane's keys: never too small, and looked at closely where it says so)
                bool over = false;
                const float most = __log2f(top_scale) - kPgLag - kUp;
#pragma unroll
                for (int n = 0; n < kN; ++n) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float top = fmaxf(s[0][n][r], s[0][n][2 + r]);
                        if (kM == 2) top = fmaxf(top, fmaxf(s[kM - 1][n][r], s[kM - 1][n][2 + r]));
                        over |= top + most > ref[n][r];
                    }
                }
                if (__any_sync(0xffffffffu, over)) {
                    // some row's reference moves
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            float top = -INFINITY;
#pragma unroll
                            for (int k = 0; k < 2 * kM; ++k) {
                                top = fmaxf(top, s[k >> 1][n][2 * (k & 1) + r] + __log2f(fmaxf(vs[k >> 1][k & 1], kPcLeastScale)));
                            }
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            const bool moves = top - ref[n][r] > kPgLag + kUp;
                            const float to = moves ? top - kUp : ref[n][r], corr = moves ? ex2_approx(ref[n][r] - to) : 1.0f;
                            ref[n][r] = to;
                            huge |= fabsf(to) >= 1048576.0f && moves;
                            l[n][r] *= corr;
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) {
                                o[n][i][r] *= corr;
                                o[n][i][2 + r] *= corr;
                            }
                        }
                    }
                }
                uint32_t w[kM][kN][2];
#pragma unroll
                for (int m = 0; m < kM; ++m) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float e[2];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float power = ex2_approx(s[m][n][2 * i + r] - ref[n][r]);
                                l[n][r] += power;
                                e[r] = power * vs[m][i];
                            }
                            if (huge) {   // (beyond 2^20 a score knows little of log2 s^v, and a weight could leave fp16)
#pragma unroll
                                for (int r = 0; r < 2; ++r) asm("min.NaN.f32 %0, %0, %1;" : "+f"(e[r]) : "f"(65504.0f));
                            }
                            if (masked) {   // (a scale that is not finite, of a value that the row does not see)
#pragma unroll
                                for (int r = 0; r < 2; ++r) e[r] = s[m][n][2 * i + r] == -INFINITY ? 0.f : e[r];
                            }
                            const __half2 h = __floats2half2_rn(e[0], e[1]);
                            w[m][n][i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
                        }
                    }
                }
                // ---- sums
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    constexpr int kWords = D / 32;     // of the D / 8 bytes of a key that a lane has
                    uint32_t v[4][kWords];             // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t tile = at_m + 16 * m * D + Shape::kTile;
                        const int row = 2 * t + (k & 1) + 8 * (k >> 1);
                        if (D == 128) {
                            const uint4 x = lds128(tile + pc_place<D>(row, g));
                            v[k][0] = x.x, v[k][1] = x.y, v[k][2 % kWords] = x.z, v[k][3 % kWords] = x.w;
                        }
                        else {
                            const uint2 x = lds64(tile + pc_place<D>(row, g >> 1) + (uint32_t)((g & 1) * 8));
                            v[k][0] = x.x, v[k][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        // dims 4 i .. 4 i + 3 of the lane's, pairs of keys
                        uint32_t lo[4], hi[4];
                        codes_to_half<kCodes>(__byte_perm(v[0][i], v[1][i], 0x5140), lo[0], lo[1]);
                        codes_to_half<kCodes>(__byte_perm(v[0][i], v[1][i], 0x7362), lo[2], lo[3]);
                        codes_to_half<kCodes>(__byte_perm(v[2][i], v[3][i], 0x5140), hi[0], hi[1]);
                        codes_to_half<kCodes>(__byte_perm(v[2][i], v[3][i], 0x7362), hi[2], hi[3]);
#pragma unroll
                        for (int n = 0; n < kN; ++n) {
                            mma_m16n8k16(o[n][2 * i], lo[0], lo[1], hi[0], hi[1], w[m][n][0], w[m][n][1]);
                            mma_m16n8k16(o[n][2 * i + 1], lo[2], lo[3], hi[2], hi[3], w[m][n][0], w[m][n][1]);
                        }
                    }
                }
            }
        }

        // ---- the end of a piece: the sums of the lanes, then of the warps
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], x);
                if (g == 0) {
                    sm.ref[warp][8 * n + 2 * t + r] = ref[n][r];
                    sm.sum[warp][8 * n + 2 * t + r] = l[n][r];
                }
            }
        }
        // O goes where the codes of the piece's last block were, [row][dim], rows D floats apart and rotated against the banks.  (Nothing
        // is on its way there: the copies that follow go to that stage with the next block.)
        float* mine = reinterpret_cast<float*>(pc_dyn + (warp * Shape::kStages + used) * Shape::kStage);
        __syncwarp();
        if (blocks > 0) {
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 8 * n + 2 * t + (e & 1), d = D / 8 * g + 2 * i + (e >> 1);
                        mine[row * D + ((d + 8 * row) & (D - 1))] = o[n][i][e];
                    }
                }
            }
        }
        __syncthreads();
        const bool complete = p.starts && p.ends;
        const PgPartial part = pg_partial(ws, region, cta, p.starts ? 1 : 0, kRows, D);
        for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * Shape::kWarps) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float top = kPgNone, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < Shape::kWarps; ++w) {
                if (sm.sum[w][row] != 0.f) top = fmaxf(top, sm.ref[w][row]);
            }
#pragma unroll
            for (int w = 0; w < Shape::kWarps; ++w) {
                const float part_sum = sm.sum[w][row];
                if (part_sum == 0.f) continue;      // (it has seen nothing)
                const float f = ex2_approx(sm.ref[w][row] - top);
                sum += part_sum * f;
                const float4 x = *reinterpret_cast<const float4*>(
                    reinterpret_cast<const float*>(pc_dyn + (w * Shape::kStages + used) * Shape::kStage) + row * D + ((d + 8 * row) & (D - 1)));
                v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
            }
            const float f = complete ? (sum == 0.f ? 0.f : 1.0f / sum) : 1.0f;
            v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
            if (!complete) {
                part.o[row * (D / 4) + d / 4] = v;
                if (d == 0) {
                    part.max2[row] = top;
                    part.sum[row] = sum;
                }
            }
            else {
                uint16_t* dst = (uint16_t*)a.out + (size_t)(p.s.row0 + token0 + row / group) * a.o_tok +
                                (size_t)(p.head * group + row % group) * a.o_head + d;
                uint2 w;
                if (a.bf16) w = make_uint2(PgType<__nv_bfloat16>::pack(v.x, v.y), PgType<__nv_bfloat16>::pack(v.z, v.w));
                else w = make_uint2(PgType<__half>::pack(v.x, v.y), PgType<__half>::pack(v.z, v.w));
                *reinterpret_cast<uint2*>(dst) = w;
            }
        }
        __syncthreads();   // the stage is free again
        more = have_next;
        if (!more) break;
        have_next = walk(now);
        now ^= 1;
        if (copy_next && copy_left > 0) copy_next = false;   // in the piece at work now
        else if (have_next) copy_from(now ^ 1);              // that one is copied, or has nothing to copy
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    pdl_wait();
}

// As pg_begin, but a dependent may begin only when the kernels in front have ended.
__device__ __forceinline__ void pc_begin(uint32_t* tmem_base, uint32_t columns)
{
    if ((threadIdx.x >> 5) == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    pdl_wait();
    pdl_launch_dependents();
}

// Sequences of more than `few` new tokens; rows_tokens: those of a tile of the other kernel, where that one runs beside this (else 0).
template<typename T, int D, bool kBias, int kCodes>
__global__ void __launch_bounds__(kPgCodesThreads, 1)
paged_mha_tc_codes_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedMhaArgs a, void* ws, int few, int rows_tokens,
                          int whole)
{
    extern __shared__ __align__(1024) uint8_t pg_dyn[];
    __shared__ PgSmem sm;
    __shared__ uint32_t tmem_base;
    if (smem_u32(pg_dyn) & 1023) {   // the swizzle goes by addresses; the alignment above is there, so this does not happen
        g_device_status = 2;
        return;
    }
    if (threadIdx.x == 0) pg_init(sm, 4);
    pc_begin(&tmem_base, kPgTmemCols);
    const int n = gridDim.x, cta = blockIdx.x, ctas = rows_tokens ? pc_split(a, rows_tokens, few, n, kBias).sms_tiles : n;
    static_assert(sizeof(PgFound) <= sizeof(sm.b_max) + sizeof(sm.b_sum) && alignof(PgFound) <= 8, "lies there for a while");
    if (cta < ctas) {
        pg_tiles<T, D, kBias, kCodes>(&map_q, &map_k, &map_v, a, ws, few + 1, whole, cta, ctas, n, sm, *reinterpret_cast<PgFound*>(sm.b_max), tmem_base,
                                      pg_dyn);
    }
    else if (!whole && threadIdx.x == 0) {
        reinterpret_cast<PgHeader*>(ws)[cta] = {};
    }
    pg_end(&tmem_base, kPgTmemCols);
}

// Codes as [page][head][slot][dim] bytes, boxes of a page (of 64 slots of a larger one) and a head.
template<int D>
int pg_encode_codes(CUtensorMap* map, const void* base, const PagedMhaArgs& a, long long page_step, long long head_step, long long slot_step)
{
    EncodeTiledFn encode = encode_tiled_fn();
    EET_CHECK(encode != nullptr, "paged attention: cuTensorMapEncodeTiled is not available from the driver");
    const int page = 1 << a.page_shift;
    const cuuint64_t dims[4] = {D, (cuuint64_t)page, (cuuint64_t)a.kv_heads, (cuuint64_t)a.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)slot_step, (cuuint64_t)head_step, (cuuint64_t)page_step};
    const cuuint32_t box[4] = {D, (cuuint32_t)(page < kPgKeys / 2 ? page : kPgKeys / 2), 1, 1}, elem[4] = {1, 1, 1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, elem,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    EET_CHECK(rc == CUDA_SUCCESS, "paged attention: cuTensorMapEncodeTiled failed with code %d (strides too large or negative)", (int)rc);
    return 0;
}

template<typename T, int D, bool kBias, int kCodes>
int pc_launch_tiles(const PagedMhaArgs& a, void* ws, int few, int rows_tokens, int whole, cudaStream_t stream)
{
    constexpr int kSmem = pg_tiles_smem(D, kCodes);
    CUtensorMap map_q, map_k, map_v;
    const long long q_dims[3] = {D, a.heads, a.tokens}, q_str[3] = {1, a.q_head, a.q_tok};
    const int group = a.heads / a.kv_heads, q_box[3] = {64, group, kPgRows / group};
    if (int rc = pg_encode(&map_q, PgType<T>::tma, a.q, 3, q_dims, q_str, q_box)) return rc;
    if (int rc = pg_encode_codes<D>(&map_k, a.k_cache, a, a.kc_page, a.kc_head, a.kc_slot)) return rc;
    if (int rc = pg_encode_codes<D>(&map_v, a.v_cache, a, a.vc_page, a.vc_head, a.vc_slot)) return rc;
    auto kern = paged_mha_tc_codes_kernel<T, D, kBias, kCodes>;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        attr_set[dev] = true;
    }
    EET_CUDA(launch_pdl(kern, dim3(sm_count()), dim3(kPgCodesThreads), kSmem, stream, map_q, map_k, map_v, a, ws, few, rows_tokens, whole));
    return 0;
}

template<int kCodes, int D, int kRows>
int pc_launch(const PagedMhaArgs& a, void* ws, int few, int beside, int whole, cudaStream_t stream)
{
    auto kern = paged_mha_codes_kernel<kCodes, D, kRows>;
    constexpr int kSmem = PcShape<D, kRows>::kSmem;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        attr_set[dev] = true;
    }
    EET_CUDA(launch_pdl(kern, dim3(PcShape<D, kRows>::kPerSm * sm_count()), dim3(32 * PcShape<D, kRows>::kWarps), kSmem, stream, a, ws, few, beside, whole));
    return 0;
}

}  // namespace

// Which kernels serve a call, as in paged_plan: sequences of up to `few` tokens go to the tiles of 8 or 16 rows, the others to those of 128.
struct PagedCodesPlan {
    int rows;            // of a tile of the first kind: 8 or 16; 0: none
    bool tiles;
    int few;
    bool whole[2];       // their tiles are not cut (no scratch, no second launch)
    size_t bytes[2];     // scratch
};

static PagedCodesPlan paged_codes_plan(const PagedMhaArgs& a)
{
    PagedCodesPlan p = {};
    const int group = a.heads / a.kv_heads;
    auto is_few = [&](long long tokens) { return (tokens > 0 ? tokens : 1) * group <= 16; };
    p.tiles = !is_few(a.max_tokens);
    p.few = 0x7fffffff;
    if (!p.tiles) {
        p.rows = (long long)a.max_tokens * group <= 8 ? 8 : 16;
    }
    else if (group <= 16) {
        // few tokens each beside the longest, and something to read for them?
        const long long others = a.seqs - 1, rest = a.tokens - a.max_tokens, each = others > 0 && rest > others ? (rest + others - 1) / others : 1;
        if (others > 0 && is_few(each) && others * a.kv_heads * (a.max_len / kPgKeys + 1) >= 1024) {
            p.rows = each * group <= 8 ? 8 : 16;
            p.few = p.rows / group;
        }
    }
    // Cutting tiles evens out the shares and costs a second launch and parts to write, 4 to 10 us.  Not where the longest share of whole tiles is
    // a few blocks longer, taking tiles to be three quarters as long as the longest on average, as in paged_plan; a block takes 0.7 us with few
    // rows and an SM for itself, 1.5 us as a tile.
    auto whole = [&](long long tokens, long long ctas, int most) {
        const long long keys = a.window > 0 && a.window + tokens < a.max_len ? a.window + tokens : a.max_len;
        const long long blocks = keys / kPgKeys + 1;
        const long long tiles = (a.seqs + (a.max_tokens > tokens ? a.tokens / tokens : 0)) * a.kv_heads;
        return blocks - (tiles < ctas ? 3 * blocks * tiles / (4 * ctas) : 0) <= most;
    };
    if (p.rows) p.whole[0] = whole(p.rows / group, pc_per_sm(p.rows) * sm_count(), 5);
    if (p.tiles) p.whole[1] = whole(2 * (kPgRows / group), sm_count(), 4);
    if (p.rows && !p.whole[0]) p.bytes[0] = pg_scratch_bytes(pc_per_sm(p.rows) * sm_count(), p.rows, a.head_dim);
    if (p.tiles && !p.whole[1]) p.bytes[1] = pg_scratch_bytes(sm_count(), 2 * kPgRows, a.head_dim);
    return p;
}

size_t paged_mha_codes_workspace_bytes(const PagedMhaArgs& a)
{
    const PagedCodesPlan p = paged_codes_plan(a);
    return p.bytes[0] + p.bytes[1];
}

template<typename T, int D, int kCodes>
static int launch_paged_mha_codes_t(const PagedMhaArgs& a, const PagedCodesPlan& p, cudaStream_t stream)
{
    void* ws[2] = {a.ws, (char*)a.ws + p.bytes[0]};
    const bool both = p.rows && p.tiles;
    // (the tiles without a bias take the maximum of the scores before the scale, which a negative one would turn round)
    const bool bias = a.slopes != nullptr || !(a.scale > 0.f);
    if (p.tiles) {
        const int few = both ? p.few : 0, rows_tokens = both ? p.few : 0;
        if (int rc = bias ? pc_launch_tiles<T, D, true, kCodes>(a, ws[1], few, rows_tokens, p.whole[1], stream)
                          : pc_launch_tiles<T, D, false, kCodes>(a, ws[1], few, rows_tokens, p.whole[1], stream)) return rc;
    }
    if (p.rows) {
        const int few = both ? p.few : 0x7fffffff, beside = !both ? 0 : bias ? 2 : 1;
        if (int rc = p.rows == 8 ? pc_launch<kCodes, D, 8>(a, ws[0], few, beside, p.whole[0], stream)
                                 : pc_launch<kCodes, D, 16>(a, ws[0], few, beside, p.whole[0], stream)) return rc;
    }
    // One launch adds up the parts of either kind.  (Its grid is that of the larger number of CTAs; the scratch of each kind knows its own.)
    PgScratch s[2] = {};
    int n = 0;
    if (p.bytes[0]) s[n++] = {ws[0], p.rows, 0, pc_per_sm(p.rows) * sm_count()};
    if (p.bytes[1]) s[n++] = {ws[1], 2 * kPgRows, 1, sm_count()};
    if (n == 0) return 0;
    const long long rows = (long long)a.max_tokens * (a.heads / a.kv_heads), most = p.bytes[1] ? 2 * kPgRows : p.rows;
    const int y = (int)((rows < most ? rows : most) * (D / 8) + kPgJoinThreads - 1) / kPgJoinThreads;   // 8 dims a thread
    const int ctas = s[0].ctas > s[1].ctas ? s[0].ctas : s[1].ctas;
    EET_CUDA(launch_pdl(paged_mha_join_kernel<T, D>, dim3(ctas, y, n), dim3(kPgJoinThreads), 0, stream, a, s[0], s[1]));
    return 0;
}

int launch_paged_mha_codes(const PagedMhaArgs& a, cudaStream_t stream)
{
    const PagedCodesPlan p = paged_codes_plan(a);
    auto launch = [&](auto codes) -> int {
        constexpr int kCodes = decltype(codes)::value;
        if (a.bf16) {
            return a.head_dim == 128 ? launch_paged_mha_codes_t<__nv_bfloat16, 128, kCodes>(a, p, stream)
                                     : launch_paged_mha_codes_t<__nv_bfloat16, 64, kCodes>(a, p, stream);
        }
        return a.head_dim == 128 ? launch_paged_mha_codes_t<__half, 128, kCodes>(a, p, stream)
                                 : launch_paged_mha_codes_t<__half, 64, kCodes>(a, p, stream);
    };
    return a.codes == kCodesInt8 ? launch(std::integral_constant<int, kCodesInt8>()) : launch(std::integral_constant<int, kCodesE4M3>());
}

}  // namespace eet
