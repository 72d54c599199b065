// The next token of each row of logits, drawn with temperature, top-k, top-p and min-p from a given random number.
//
//   w_i = exp((x_i - max x) / T).  In the order of x, the lowest index first among equals: top-k leaves the first k; top-p those of them in
//   front of which stands less than top_p of the w of the k; min-p those with w >= min_p; the first always stays.  Of what is left, in the
//   order of the indices, the first token whose running sum of w exceeds u times the sum of all is drawn.
//
// All of these leave a beginning of one order, so they come down to a cut: a value x*, and how many of its equals stay.  Nothing is sorted but
// a few candidates around it.
//   1  the row into shared memory, its maximum
//   2  a histogram over (max - x) / T, 64 bins to a factor of e in w (fewer where top-k may reach further down than 32 such factors): counts in
//      front of a bin are exact, sums of w known to 1.6 %, and mostly to 1e-4
//   3  the bins in which the cut must lie - by mass first those where it very likely lies, which the sums in step 4 confirm or not; where they
//      hold too many values for a list, a second histogram over them alone
//   4  those values in a list, and the exact sums of w of all and of what stands in front of them; the list sorted: the cut.  (Where one bin
//      of the second histogram holds more than the list can, as with very many equal values: bisection on x.)
//   5  what is left, summed by threads in the order of the indices; the thread whose part of the sum the random number falls into draws
// Sums are of w as whole multiples of 2^-44, from powers in 64 bits: whatever the number of CTAs and their order, they are the same, and a cut
// or a draw lies where the definition puts it but for one chance in about 2^-44 times the vocabulary.  (In 32 bits a draw from 64000 tokens would
// miss the border of some token once in some hundred rows.)
//
// A row is worked on by a cluster of 1 to 8 CTAs, which hold it in shared memory and exchange counts and candidates there.  Bound: latency,
// six barriers of the cluster and four trips through a slice of the row; with many rows the issue of instructions, the powers of all
// tokens first (11 instructions in 64 bits each, with a table of 128; exp() took three times as long): 58 % of the slots taken, the pipe
// of whole numbers 46 % full, that of 64 bits 12 %.  Measured: one row of 32000 fp32 logits 18 us, 64 rows of 64000 fp16 41, 256 of 64000
// bf16 139 (22, 119 and 287 with exp() and lists gathered by atomics on one counter).
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace eet {

namespace {

namespace cg = cooperative_groups;

constexpr int kSaThreads = 512;
constexpr int kSaWarps = kSaThreads / 32;
constexpr int kSaBins = 2048;
constexpr int kSaPerThread = kSaBins / kSaThreads;
constexpr float kSaBinsPerE = 64.0f;
constexpr int kSaList = 4096;
constexpr int kSaMaxCluster = 8;
constexpr int kSaMaxVocab = 1 << 18;         // their sum of w stays below 2^62
constexpr int kSaMaxSlice = 128 * 1024;      // bytes of a row in a CTA at the most,
constexpr int kSaSlice = 68 * 1024;          // and where there are CTAs for more of them: two share an SM
constexpr double kSaUnit = 17592186044416.0; // 2^44
constexpr uint32_t kSaNothing = 0x007fffffu; // the key of -inf

constexpr uint32_t kSaUnlisted = 0xffffffffu, kSaMissed = 0xfffffffeu;
constexpr int kSaTable = 128;                // powers of 2^(1 / 128)
constexpr int kSaCounted = 256;              // lists up to here are sorted by counting

typedef unsigned long long u64;

struct SaCut {
    uint32_t key;      // values above it stay,
    uint32_t equals;   // and the first so many of its equals
    uint32_t listed;   // the largest value of the list that it was found in: what lies above stood in front (kSaMissed: it is not in the list)
};

struct SaBracket {
    int b0, b1;        // bins that hold the cut
    uint32_t count;    // values in them
    uint32_t before;   // values in front of them
};

struct SaSmem {
    double table[kSaTable];
    uint32_t hist[kSaBins], fine[kSaBins];
    uint32_t list[kSaList];
    uint32_t listed;
    // from every CTA of the cluster, two buffers each
    float maxima[kSaMaxCluster], minima[kSaMaxCluster];
    u64 sums[2][kSaMaxCluster], fronts[2][kSaMaxCluster];
    uint32_t counts[2][kSaMaxCluster];
    // from the first CTA
    SaBracket bracket;
    SaCut cut;
    // of this CTA
    u64 warp_sum[kSaWarps], warp_front[kSaWarps];
    uint32_t warp_count[kSaWarps];
    double warp_low[kSaWarps], warp_high[kSaWarps];
    float warp_max[kSaWarps], warp_min[kSaWarps];
    uint32_t front, upto;
};

// Values in an order of whole numbers; -0 has become 0 and NaN -inf before.
__device__ __forceinline__ uint32_t sa_key(float x)
{
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float sa_value(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The words of a row in shared memory: one or two values each.
template<typename T>
struct SaWord;
template<>
struct SaWord<float> {
    static constexpr int kValues = 1;
    static constexpr uint32_t kNothing = 0xff800000u;
    static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
    // NaN to -inf, -0 to 0
    static __device__ __forceinline__ uint32_t clean(uint32_t w)
    {
        const float x = __uint_as_float(w);
        return x == x ? __float_as_uint(x + 0.0f) : kNothing;
    }
};
template<>
struct SaWord<__half> {
    static constexpr int kValues = 2;
    static constexpr uint32_t kNothing = 0xfc00fc00u;
    static __device__ __forceinline__ float get(uint32_t w, int i) { return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffffu))); }
    static __device__ __forceinline__ uint32_t clean(uint32_t w)
    {
        const __half2 x = *reinterpret_cast<const __half2*>(&w), y = __hadd2(x, __floats2half2_rn(0.f, 0.f));
        const uint32_t is = __heq2_mask(x, x);
        return (*reinterpret_cast<const uint32_t*>(&y) & is) | (kNothing & ~is);
    }
};
template<>
struct SaWord<__nv_bfloat16> {
    static constexpr int kValues = 2;
    static constexpr uint32_t kNothing = 0xff80ff80u;
    static __device__ __forceinline__ float get(uint32_t w, int i) { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }
    static __device__ __forceinline__ uint32_t clean(uint32_t w)
    {
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w), y = __hadd2(x, __floats2bfloat162_rn(0.f, 0.f));
        const uint32_t is = __heq2_mask(x, x);
        return (*reinterpret_cast<const uint32_t*>(&y) & is) | (kNothing & ~is);
    }
};

struct SaRow {
    float top;            // finite
    float scale;          // bins a unit of x,
    float per_bin;        // and units of (max - x) / T a bin
    float least;          // below it exp(-745) is passed, where a number in 64 bits ends: w is 0
    double over_t;        // 1 / T
    double step;          // kSaTable log2(e) / T
    const double* table;

    // (x - max) / T
    __device__ __forceinline__ double power(float x) const { return ((double)x - (double)top) * over_t; }
    // w in multiples of 2^-44, without a branch.  2^(t / 128) is 2^(k >> 7) times the table's entry k & 127 times a polynomial in what is left of
    // t, at most half a step: the fourth power's rest is below 2^-49.  What can be drawn stays so, with one unit at least.
    __device__ __forceinline__ u64 weight(float x) const
    {
        const double t = fmax(((double)x - (double)top) * step, -5760.0);   // (2^-45: rounds to nothing)
        constexpr double kShift = 6755399441055744.0;        // 1.5 2^52: whole numbers in the low bits
        const double shifted = t + kShift;
        const int k = __double2loint(shifted);
        const double f = t - (shifted - kShift);
        double p = 3.583032305400251e-11;                    // (ln 2 / 128)^4 / 24
        p = fma(p, f, 2.6466421444330967e-8);                // ^3 / 6
        p = fma(p, f, 1.4662262387640423e-5);                // ^2 / 2
        p = fma(p, f, 5.4152123481245725e-3);                // ln 2 / 128
        p = fma(p, f, 1.0);
        const double e = table[k & (kSaTable - 1)] * p;
        // times 2^(44 + (k >> 7)), then rounded by adding 2^52
        const double w = __hiloint2double(__double2hiint(e) + ((44 + (k >> 7)) << 20), __double2loint(e)) + 4503599627370496.0;
        const u64 units = (u64)__double_as_longlong(w) & 0xfffffffffffffull;
        return units | (units == 0 && x > least ? 1u : 0u);
    }
    __device__ __forceinline__ float place(float x) const { return fmaxf((top - x) * scale, 0.f); }
    // (to the nearest whole number: the low bits of a sum with 2^23)
    __device__ __forceinline__ int bin(float x) const
    {
        return __float_as_int(fminf(place(x), (float)(kSaBins - 1)) + 8388608.0f) - 0x4b000000;
    }
    // bins of the second histogram: those of [b0, b1] cut into kSaBins
    __device__ __forceinline__ int sub_bin(float x, int b0, float per_bin) const
    {
        return max(0, min(kSaBins - 1, (int)((place(x) - (b0 - 0.5f)) * per_bin)));
    }
};

template<typename T>
struct SaKernel {
    using Word = SaWord<T>;
    SaSmem& sm;
    const uint32_t* x;     // the slice's words, in shared memory
    int begin, end;        // this thread's: consecutive, an odd number to a thread, so that a warp's reads meet no bank twice
    int ranks, rank;
    SaRow row;
    int turn = 0;          // buffer of the next exchange

    // f(value) for this thread's values, in the order of the indices; -inf among them, but neither NaN nor -0
    template<typename F>
    __device__ __forceinline__ void each(F f) const
    {
        for (int i0 = begin; i0 < end; i0 += 4) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = i0 + k < end ? x[i0 + k] : Word::kNothing;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int h = 0; h < Word::kValues; ++h) f(Word::get(w[k], h));
            }
        }
    }
    __device__ __forceinline__ void barrier() const
    {
        if (ranks > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    template<typename V>
    __device__ __forceinline__ V* of(V* p, int r) const
    {
        return ranks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
    }

    // Sums over the threads of the CTA in front of this one, and over all of them.
    struct Sums {
        u64 sum, sum_before, front;
        uint32_t count, count_before;
    };
    __device__ __forceinline__ Sums scan(u64 sum, uint32_t count, u64 front = 0) const
    {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        u64 s = sum;
        uint32_t c = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 u = __shfl_up_sync(0xffffffffu, s, o);
            const uint32_t d = __shfl_up_sync(0xffffffffu, c, o);
            front += __shfl_xor_sync(0xffffffffu, front, o);
            if (lane >= o) s += u, c += d;
        }
        __syncthreads();   // the last scan's may still be read
        if (lane == 31) sm.warp_sum[warp] = s, sm.warp_count[warp] = c, sm.warp_front[warp] = front;
        __syncthreads();
        Sums r = {0, s - sum, 0, 0, c - count};
#pragma unroll
        for (int w = 0; w < kSaWarps; ++w) {
            const u64 u = sm.warp_sum[w];
            const uint32_t d = sm.warp_count[w];
            if (w < warp) r.sum_before += u, r.count_before += d;
            r.sum += u, r.count += d, r.front += sm.warp_front[w];
        }
        return r;
    }
    // Leaves a CTA's sums with all of the cluster, to be read with collect() behind a barrier.  (Whoever writes a buffer again has passed the
    // barrier of the other one, behind everybody's reads.)
    __device__ __forceinline__ void publish(const Sums& s)
    {
        if ((int)threadIdx.x < ranks) {
            *of(&sm.sums[turn][rank], threadIdx.x) = s.sum;
            *of(&sm.counts[turn][rank], threadIdx.x) = s.count;
            *of(&sm.fronts[turn][rank], threadIdx.x) = s.front;
        }
    }
    __device__ __forceinline__ Sums collect(Sums s)
    {
        s.sum = 0, s.count = 0, s.front = 0;
        for (int r = 0; r < ranks; ++r) {
            const u64 u = sm.sums[turn][r];
            const uint32_t d = sm.counts[turn][r];
            if (r < rank) s.sum_before += u, s.count_before += d;
            s.sum += u, s.count += d, s.front += sm.fronts[turn][r];
        }
        turn ^= 1;
        return s;
    }
    __device__ __forceinline__ Sums exchange(u64 sum, uint32_t count, u64 front = 0)
    {
        const Sums s = scan(sum, count, front);
        publish(s);
        barrier();
        return collect(s);
    }

    // This CTA's counts to those of the first.  (Its own are complete behind the barriers of a scan.)
    __device__ __forceinline__ void merge(uint32_t* bins) const
    {
        if (rank == 0) return;
        uint32_t* first = of(bins, 0);
        for (int i = threadIdx.x; i < kSaBins; i += kSaThreads) {
            if (bins[i] != 0) atomicAdd(&first[i], bins[i]);
        }
    }

    // The bins of the first CTA's histogram that hold the cut, by that CTA; to all.
    //   by count   the one in which the count passes `k`, `counted` values standing in front of all of them
    //   by mass    those in which the sum of w may pass `goal`, or where that is 0 `part` of the sum of all; `mass` stands in front, and bin b's w
    //              are between e^(-low(b + 1)) and e^(-low(b)), or with slack > 0 taken to be those at its middle but for that part
    // `total` values are in the bins; what they do not say is in the last one.  open_end: it holds all that lie behind.
    template<typename F>
    __device__ __forceinline__ SaBracket narrow(const uint32_t* bins, uint32_t total, bool by_mass, uint32_t k, uint32_t counted, double goal,
                                                float part, double mass, float slack, F low, bool open_end)
    {
        if (rank == 0) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = threadIdx.x * kSaPerThread;
            uint32_t c[kSaPerThread], count = 0;
            double lo[kSaPerThread], hi[kSaPerThread], low_sum = 0, high_sum = 0;
#pragma unroll
            for (int i = 0; i < kSaPerThread; ++i) {
                const int b = first + i;
                c[i] = bins[b];
                count += c[i];
                lo[i] = hi[i] = 0;
                if (by_mass && c[i] > 0) {
                    // (2e-5: what single precision may do to a value's place, and expf)
                    const float most = expf(-low(b)), fewest = expf(-low(b + 1)), middle = 0.5f * (most + fewest);
                    hi[i] = c[i] * kSaUnit * (double)(slack > 0.f ? middle * (1.0f + slack) : most * 1.00002f);
                    lo[i] = c[i] * kSaUnit * (double)(slack > 0.f ? middle * (1.0f - slack) : open_end && b == kSaBins - 1 ? 0.f : fewest * 0.99998f);
                }
                low_sum += lo[i];
                high_sum += hi[i];
            }
            if (threadIdx.x == 0) {
                sm.bracket.b0 = sm.bracket.b1 = kSaBins - 1;
                sm.front = sm.upto = 0xffffffffu;
            }
            uint32_t cs = count;
            double ls = low_sum, hs = high_sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t cu = __shfl_up_sync(0xffffffffu, cs, o);
                const double lu = __shfl_up_sync(0xffffffffu, ls, o), hu = __shfl_up_sync(0xffffffffu, hs, o);
                if (lane >= o) cs += cu, ls += lu, hs += hu;
            }
            __syncthreads();
            if (lane == 31) sm.warp_count[warp] = cs, sm.warp_low[warp] = ls, sm.warp_high[warp] = hs;
            __syncthreads();
            uint32_t at = cs - count, all = 0;
            double low_at = mass + (ls - low_sum), high_at = mass + (hs - high_sum), low_all = mass, high_all = mass;
#pragma unroll
            for (int w = 0; w < kSaWarps; ++w) {
                if (w < warp) at += sm.warp_count[w], low_at += sm.warp_low[w], high_at += sm.warp_high[w];
                all += sm.warp_count[w], low_all += sm.warp_low[w], high_all += sm.warp_high[w];
            }
            const double rest = by_mass ? (total - all) * kSaUnit * (double)(expf(-low(kSaBins - 1)) * 1.00002f) : 0.0;
            high_all += rest;
            if (threadIdx.x == kSaThreads - 1) c[kSaPerThread - 1] += total - all, hi[kSaPerThread - 1] += rest;
            // (the rounding of these sums is far below what the bins leave open)
            const double goal_low = goal > 0.0 ? goal : fmax(0.999999 * part * low_all, 0.5), goal_high = goal > 0.0 ? goal : fmax(1.000001 * part * high_all, 0.5);
#pragma unroll
            for (int i = 0; i < kSaPerThread; ++i) {
                if (by_mass) {
                    if (high_at < goal_low && high_at + hi[i] >= goal_low) sm.bracket.b0 = first + i, sm.front = at;
                    if (low_at < goal_high && low_at + lo[i] >= goal_high) sm.bracket.b1 = first + i, sm.upto = at + c[i];
                    high_at += hi[i];
                    low_at += lo[i];
                }
                else if (counted + at < k && counted + at + c[i] >= k) {
                    sm.bracket.b0 = sm.bracket.b1 = first + i;
                    sm.front = at;
                    sm.upto = at + c[i];
                }
                at += c[i];
            }
            __syncthreads();
            // (sums of doubles over the warps are rounded: a border between two threads may be nobody's, and then all bins are looked at)
            const bool none = sm.front == 0xffffffffu;
            const uint32_t upto = sm.upto == 0xffffffffu ? total : sm.upto, front = none ? 0 : min(sm.front, upto);
            const SaBracket found = {none ? 0 : min(sm.bracket.b0, sm.bracket.b1), sm.bracket.b1, upto - front, counted + front};
            __syncthreads();
            if ((int)threadIdx.x < ranks) *of(&sm.bracket, threadIdx.x) = found;
        }
        barrier();
        return sm.bracket;
    }

    // The values between the cut's bins into the first CTA's list, and with `sums` those of w: of all, and of what stands in front (`mine`: this
    // thread's of that).  f(v): 0 in front, 1 in the bins, 2 behind.
    template<typename F>
    __device__ __forceinline__ Sums gather(bool sums, u64& mine, F f)
    {
        u64 all = 0;
        mine = 0;
        // (first into this CTA's own: a counter that all of the cluster adds to, value by value, took 40 us for 4000)
        auto put = [&](float v) {
            const uint32_t i = atomicAdd(&sm.listed, 1u);
            if (i < kSaList) sm.list[i] = sa_key(v);
        };
        if (sums) {
            each([&](float v) {
                const int where = f(v);
                const u64 w = row.weight(v);
                all += w;
                mine += where == 0 ? w : 0;
                if (where == 1 && v > -INFINITY) put(v);
            });
        }
        else {
            each([&](float v) {
                if (f(v) == 1 && v > -INFINITY) put(v);
            });
        }
        if (rank > 0) {
            __syncthreads();
            const uint32_t n = min(sm.listed, (uint32_t)kSaList);
            if (threadIdx.x == 0) sm.front = atomicAdd(of(&sm.listed, 0), n);
            __syncthreads();
            const uint32_t at = sm.front;
            uint32_t* list = of(sm.list, 0);
            for (uint32_t i = threadIdx.x; i < n && at + i < kSaList; i += kSaThreads) list[at + i] = sm.list[i];
            if (threadIdx.x == 0) sm.listed = 0;   // (for the next list)
        }
        return exchange(all, 0, mine);
    }

    // By the first CTA: the list, from the largest.
    __device__ __forceinline__ const uint32_t* sorted(int count)
    {
        if (count <= kSaCounted) {
            // (a value's place is the number of those in front of it)
            if ((int)threadIdx.x < count) {
                const uint32_t mine = sm.list[threadIdx.x];
                int place = 0;
#pragma unroll 8
                for (int i = 0; i < count; ++i) {
                    const uint32_t other = sm.list[i];
                    place += other > mine || (other == mine && i < (int)threadIdx.x);
                }
                sm.fine[place] = mine;
            }
            __syncthreads();
            return sm.fine;
        }
        // Bitonic: what lies 32 and more apart is compared through shared memory, the rest of a round within warps.
        int size = 2 * kSaCounted;
        while (size < count) size <<= 1;
        for (int i = count + threadIdx.x; i < size; i += kSaThreads) sm.list[i] = 0;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        for (int k = 32; k <= size; k <<= 1) {
            for (int j = k >> 1; j >= 32; j >>= 1) {
                __syncthreads();
                for (int i = threadIdx.x; i < size / 2; i += kSaThreads) {
                    const int a = 2 * i - (i & (j - 1)), b = a + j;
                    const uint32_t u = sm.list[a], v = sm.list[b];
                    if ((u < v) == ((a & k) == 0)) {
                        sm.list[a] = v;
                        sm.list[b] = u;
                    }
                }
            }
            __syncthreads();
            for (int g = warp; g < size / 32; g += kSaWarps) {
                uint32_t u = sm.list[32 * g + lane];
                for (int kk = k == 32 ? 2 : k; kk <= k; kk <<= 1) {
                    const bool falls = ((32 * g + lane) & kk) == 0;
                    for (int j = min(kk >> 1, 16); j > 0; j >>= 1) {
                        const uint32_t v = __shfl_xor_sync(0xffffffffu, u, j);
                        u = falls == ((lane & j) == 0) ? max(u, v) : min(u, v);
                    }
                }
                sm.list[32 * g + lane] = u;
            }
        }
        __syncthreads();
        return sm.list;
    }

    // By the first CTA, the cut in the list of `count` values, in front of which stand `before` with the sum `front`; to all, behind a barrier.  The
    // first `k` stay (0: it is not cut by count), of those the ones in front of which stands less than `goal`, or where that is 0 and part
    // above it less than that part of the sum of the k.
    __device__ __forceinline__ SaCut cut_list(uint32_t count, uint32_t before, u64 front, uint32_t k, double goal, float part)
    {
        if (rank == 0) {
            constexpr int kEach = kSaList / kSaThreads;
            const uint32_t* list = sorted((int)count);
            bool missed = count == 0;
            uint32_t keep = k > 0 ? min(count, k - before) : count;
            if (part > 0.f || goal > 0.0) {
                u64 w[kEach], sum = 0;
                const int per = ((int)count + kSaThreads - 1) / kSaThreads, at = threadIdx.x * per;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    w[i] = i < per && at + i < (int)keep ? row.weight(sa_value(list[at + i])) : 0;
                    sum += w[i];
                }
                const Sums s = scan(sum, 0);
                u64 run = front + s.sum_before;
                if (!(goal > 0.0)) goal = fmax((double)part * (double)(front + s.sum), 0.5);
                missed = k == 0 && ((double)front >= goal || (double)(front + s.sum) < goal);
                uint32_t stay = 0;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    if (i < per && at + i < (int)keep && (double)run < goal) ++stay;
                    run += w[i];
                }
                keep = max(scan(0, stay).count, 1u);
            }
            const uint32_t key = missed ? 0 : list[keep - 1];
            uint32_t equals = 0;
            for (int i = threadIdx.x; i < (int)keep; i += kSaThreads) equals += list[i] == key;
            const SaCut cut = {key, scan(0, equals).count, missed ? kSaMissed : list[0]};
            if ((int)threadIdx.x < ranks) *of(&sm.cut, threadIdx.x) = cut;
            if (threadIdx.x == 0) sm.listed = 0;   // (for the next list)
        }
        barrier();
        return sm.cut;
    }

    // The cut by bisection: the largest key with `k` values, or a sum of w of `goal`, from it on.
    __device__ __forceinline__ SaCut bisect(bool by_mass, uint32_t k, double goal)
    {
        uint32_t lo = kSaNothing + 1, hi = sa_key(row.top);
        auto from = [&](uint32_t key) {
            u64 m = 0;
            uint32_t c = 0;
            each([&](float v) {
                if (sa_key(v) < key) return;
                ++c;
                if (by_mass) m += row.weight(v);
            });
            return exchange(m, c);
        };
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            const Sums s = from(mid);
            if (by_mass ? (double)s.sum >= goal : s.count >= k) lo = mid;
            else hi = mid - 1;
        }
        Sums above = {};
        if (lo < 0xffffffffu) above = from(lo + 1);
        if (!by_mass) return {lo, k - above.count, kSaUnlisted};
        // the first sum of equals that reaches the goal
        const u64 w = row.weight(sa_value(lo));
        uint32_t a = 1, b = kSaMaxVocab;
        while (a < b) {
            const uint32_t m = a + (b - a) / 2;
            if ((double)(above.sum + (u64)m * w) >= goal) b = m;
            else a = m + 1;
        }
        return {lo, a, kSaUnlisted};
    }

    // The cut by count, or by mass: where the sum of w passes `goal`, or where that is 0 `part` of the sum of all.  By count with part > 0 both
    // where one list does (`both` says so).  The first histogram, of `total` values, is there.  mine: as in gather().
    __device__ __forceinline__ SaCut find(uint32_t total, bool by_mass, uint32_t k, double goal, float part, bool& both, u64& mine)
    {
        const float per_e = row.per_bin;
        const auto low = [&](int b) { return fmaxf(b - 0.5f, 0.f) * per_e; };
        both = false;
        const auto goal_of = [&](const Sums& s) { return goal > 0.0 || !by_mass ? goal : fmax((double)part * (double)s.sum, 0.5); };
        if (by_mass) {
            const SaBracket b = narrow(sm.hist, total, true, 0, 0, goal, part, 0.0, 1e-3f, low, true);
            if (b.count <= kSaList) {
                const Sums s = gather(true, mine, [&](float v) {
                    const int i = row.bin(v);
                    return i < b.b0 ? 0 : i <= b.b1 ? 1 : 2;
                });
                const SaCut cut = cut_list(b.count, b.before, s.front, 0, goal_of(s), 0.f);
                if (cut.listed != kSaMissed) return cut;
                goal = goal_of(s);
            }
            else {
                barrier();     // all have read the bracket that narrow() writes again
            }
        }
        SaBracket br = narrow(sm.hist, total, by_mass, k, 0, goal, part, 0.0, 0.f, low, true);
        if (!by_mass && part > 0.f && br.before + br.count <= kSaList) {
            both = true;       // everything up to the cut
            br = {0, br.b1, br.before + br.count, 0};
        }
        if (br.count <= kSaList) {
            const SaBracket b = br;
            const Sums s = gather(by_mass, mine, [&](float v) {
                const int i = row.bin(v);
                return i < b.b0 ? 0 : i <= b.b1 ? 1 : 2;
            });
            return cut_list(b.count, b.before, s.front, by_mass ? 0 : k, goal_of(s), both ? part : 0.f);
        }
        // the second histogram, and what stands in front of it
        const int c0 = br.b0, c1 = br.b1;
        const float per_bin = (float)kSaBins / (float)(c1 - c0 + 1);
        for (int i = threadIdx.x; i < kSaBins; i += kSaThreads) sm.fine[i] = 0;
        barrier();
        u64 all = 0, ahead = 0;
        each([&](float v) {
            if (v == -INFINITY) return;
            const int i = row.bin(v);
            if (by_mass) {
                const u64 w = row.weight(v);
                all += w;
                ahead += i < c0 ? w : 0;
            }
            if (i >= c0 && i <= c1) atomicAdd(&sm.fine[row.sub_bin(v, c0, per_bin)], 1u);
        });
        const Sums own = scan(all, 0, ahead);
        publish(own);
        merge(sm.fine);
        barrier();
        const Sums sums = collect(own);
        goal = goal_of(sums);
        br = narrow(sm.fine, br.count, by_mass, k, br.before, goal, 0.f, (double)sums.front, 0.f,
                    [&](int b) { return fmaxf(c0 - 0.5f + b / per_bin, 0.f) * per_e; }, c1 == kSaBins - 1);
        if (br.count > kSaList) return bisect(by_mass, k, goal);
        const SaBracket b = br;
        const Sums s = gather(by_mass, mine, [&](float v) {
            const int i = row.bin(v);
            if (i < c0 || i > c1) return i < c0 ? 0 : 2;
            const int j = row.sub_bin(v, c0, per_bin);
            return j < b.b0 ? 0 : j <= b.b1 ? 1 : 2;
        });
        return cut_list(b.count, b.before, s.front, by_mass ? 0 : k, goal, 0.f);
    }
};

template<typename T>
__global__ void __launch_bounds__(kSaThreads, 2) sample_rows_kernel(const SampleArgs a, int ranks, int slice)
{
    extern __shared__ __align__(16) uint8_t sa_dyn[];
    __shared__ SaSmem sm;
    const int tid = threadIdx.x;
    const int rank = ranks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const long long r = blockIdx.x / ranks;
    if (ranks > 1) cluster_arrive();             // waited for before the first remote access
    for (int i = tid; i < kSaBins; i += kSaThreads) sm.hist[i] = 0;
    if (tid < kSaTable) sm.table[tid] = exp2(tid * (1.0 / kSaTable));
    if (tid == 0) sm.listed = 0;
    pdl_launch_dependents();
    pdl_wait();
    const T* src = (const T*)a.logits + r * a.row_stride + (long long)rank * slice;
    const int n = max(0, min(slice, a.vocab - rank * slice));
    // ---- 1  the slice, whole 16 bytes at a time, as it lies in global memory: what is not of it at its ends becomes -inf
    constexpr int kPer = 16 / sizeof(T);
    const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    const int loads = n > 0 ? (skew + n + kPer - 1) / kPer : 0;
    float temperature = a.temperatures != nullptr ? a.temperatures[r] : a.temperature;
    const float part = a.top_ps != nullptr ? a.top_ps[r] : a.top_p;
    float least = a.min_ps != nullptr ? a.min_ps[r] : a.min_p;
    const int wanted = a.top_ks != nullptr ? a.top_ks[r] : a.top_k;
    const bool greedy = !(temperature > 0.f);
    if (greedy) temperature = 1.0f;
    if (temperature == INFINITY) least = 0.f;   // every w is 1, the largest min-p
    const bool by_count = wanted > 0 && wanted < a.vocab, by_mass = part < 1.0f;
    float top = -INFINITY, bottom = INFINITY;   // of the finite and infinite values above -inf
    {
        const uint4* from = reinterpret_cast<const uint4*>(src - skew);
        constexpr int kAhead = 4;
        for (int i0 = tid; i0 < loads; i0 += kAhead * kSaThreads) {
            uint4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kSaThreads;
                if (i >= loads) continue;
                if (i * kPer >= skew && (i + 1) * kPer <= skew + n) {
                    v[k] = from[i];
                }
                else {
                    T* e = reinterpret_cast<T*>(&v[k]);
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        const int at = i * kPer + j - skew;
                        e[j] = at >= 0 && at < n ? src[at] : T(-INFINITY);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kSaThreads;
                if (i >= loads) continue;
                uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = SaWord<T>::clean(w[j]);
#pragma unroll
                    for (int h = 0; h < SaWord<T>::kValues; ++h) {
                        const float value = SaWord<T>::get(w[j], h);
                        top = fmaxf(top, value);
                        if (by_count && value > -INFINITY) bottom = fminf(bottom, value);
                    }
                }
                reinterpret_cast<uint4*>(sa_dyn)[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    const int words = 4 * loads, run = ((words + kSaThreads - 1) / kSaThreads) | 1, begin = min(words, tid * run);
    SaKernel<T> s = {sm, reinterpret_cast<const uint32_t*>(sa_dyn), begin, min(words, begin + run), ranks, rank, {}};
    top = warp_max(top);
    bottom = -warp_max(-bottom);
    if ((tid & 31) == 0) sm.warp_max[tid >> 5] = top, sm.warp_min[tid >> 5] = bottom;
    __syncthreads();
    if (ranks > 1) cluster_wait();
#pragma unroll
    for (int w = 0; w < kSaWarps; ++w) top = fmaxf(top, sm.warp_max[w]), bottom = fminf(bottom, sm.warp_min[w]);
    if (tid < ranks) *s.of(&sm.maxima[rank], tid) = top, *s.of(&sm.minima[rank], tid) = bottom;
    s.barrier();
    for (int i = 0; i < ranks; ++i) top = fmaxf(top, sm.maxima[i]), bottom = fminf(bottom, sm.minima[i]);
    if (top == -INFINITY) {        // nothing can be drawn
        if (rank == 0 && tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = -INFINITY;
        }
        return;                    // (all of the cluster, and the last word to another CTA lies in front of a barrier)
    }
    // (a finite scale: nothing times infinity is no place; and above zero, also where the temperature is infinite and all weigh the same: -inf would
    // stand in the first bin)
    float scale = fmaxf(fminf(kSaBinsPerE / temperature, 1e30f), 1e-37f);
    if (by_count && (top - bottom) * scale > kSaBins - 2) scale = fmaxf((kSaBins - 2) / (top - bottom), scale / 32);
    s.row = {top, scale, 1.0f / (scale * temperature), (float)((double)top - 745.0 * (double)temperature), 1.0 / (double)temperature,
             kSaTable * 1.4426950408889634 / (double)temperature, sm.table};

    SaCut cut = {kSaNothing, 0u, kSaUnlisted};   // everything above -inf
    float floor = -INFINITY;        // of min-p
    u64 ahead = 0;                  // this thread's part of the sum of what lies above the list of the cut, where known
    bool know_ahead = false;
    if (greedy) {
        cut.key = sa_key(top);
        cut.equals = 1u;
    }
    else if (top == INFINITY) {     // those of infinity share everything
        uint32_t count = 0;
        s.each([&](float v) { count += v == INFINITY; });
        count = s.exchange(0, count).count;
        if (by_count) count = min(count, (uint32_t)wanted);
        if (by_mass) count = max(1u, (uint32_t)ceil((double)part * count));
        cut.key = sa_key(top);
        cut.equals = count;
    }
    else {
        if (least > 0.f) floor = __double2float_ru((double)top + (double)temperature * log(fmin((double)least, 1.0)));
        if (by_count || by_mass) {
            // ---- 2  (the last bin, which may hold most of the row, is not counted but follows from the others)
            uint32_t count = 0;
            s.each([&](float v) {
                const int b = s.row.bin(v);
                count += v > -INFINITY;
                if (b < kSaBins - 1) atomicAdd(&sm.hist[b], 1u);
            });
            const auto mine = s.scan(0, count);
            s.publish(mine);
            s.merge(sm.hist);
            s.barrier();
            count = s.collect(mine).count;
            // ---- 3, 4
            bool both = false;
            const bool cut_count = by_count && (uint32_t)wanted < count;
            const float share = by_mass ? fmaxf(part, 1e-30f) : 0.f;
            if (cut_count) cut = s.find(count, false, wanted, 0.0, share, both, ahead);
            if (by_mass && !both) {
                double goal = 0.0;
                if (cut_count) {   // a part of the sum of what top-k leaves
                    u64 w = 0;
                    s.each([&](float v) {
                        if (sa_key(v) > cut.key) w += s.row.weight(v);
                    });
                    goal = fmax((double)part * (double)(s.exchange(w, 0).sum + cut.equals * s.row.weight(sa_value(cut.key))), 0.5);
                }
                const SaCut by_k = cut;
                cut = s.find(count, true, 0, goal, share, both, ahead);
                if (cut_count && cut.key == by_k.key) cut.equals = min(cut.equals, by_k.equals);
                know_ahead = cut.listed != kSaUnlisted;
            }
        }
    }
    // ---- 5  sums of what lies above the cut, and its equals, in the order of the indices: how many of a thread's equals stay follows from those
    // in front
    const float edge = sa_value(cut.key);
    const bool some = cut.equals > 0 && edge >= floor;
    const float listed = know_ahead ? sa_value(cut.listed) : INFINITY;
    const bool skip = know_ahead && floor <= listed;
    u64 mine = skip ? ahead : 0;
    uint32_t equals = 0;
    s.each([&](float v) {
        if (v > edge && v >= floor && !(skip && v > listed)) mine += s.row.weight(v);
        equals += some && v == edge;
    });
    const auto at = s.exchange(mine, equals);
    const u64 edge_weight = !some ? 0 : edge == top ? 1ull << 44 : s.row.weight(edge);
    const uint32_t stay = at.count_before < cut.equals ? min(equals, cut.equals - at.count_before) : 0;
    const u64 before = at.sum_before + min(at.count_before, cut.equals) * edge_weight, all = at.sum + min(at.count, cut.equals) * edge_weight;
    mine += stay * edge_weight;
    double goal = (double)a.uniform[r] * (double)all;
    if (!(goal >= 0.0)) goal = 0.0;
    if (goal >= (double)all) goal = __longlong_as_double(__double_as_longlong((double)all) - 1);   // (the number below)
    if ((double)before <= goal && (double)(before + mine) > goal && mine > 0) {
        uint32_t seen = 0;
        u64 run_sum = before;
        constexpr int kValues = SaWord<T>::kValues;
        for (int i = s.begin * kValues; i < s.end * kValues; ++i) {
            const float v = SaWord<T>::get(s.x[i / kValues], i % kValues);
            u64 w = 0;
            if (v > edge && v >= floor) w = s.row.weight(v);
            else if (some && v == edge && seen < stay) w = edge_weight, ++seen;
            run_sum += w;
            if (w > 0 && (double)run_sum > goal) {
                a.tokens[r] = (long long)rank * slice + i - skew;
                a.logprobs[r] = (float)((v == top ? 0.0 : s.row.power(v)) - log((double)all / kSaUnit));
                break;
            }
        }
    }
    // (the last word to another CTA lies in front of the barrier in exchange)
}

template<typename T>
int launch_sample_t(const SampleArgs& a, int ranks, cudaStream_t stream)
{
    constexpr int kPer = 16 / sizeof(T);
    const int slice = ((a.vocab + ranks - 1) / ranks + kPer - 1) / kPer * kPer;
    const size_t smem = ((size_t)slice + 2 * kPer) * sizeof(T);
    auto kern = sample_rows_kernel<T>;
    static bool attr_set[64] = {};
    int dev = 0;
    EET_CUDA(cudaGetDevice(&dev));
    dev &= 63;
    if (!attr_set[dev]) {
        EET_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSaMaxSlice + 64));
        attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * ranks));
    cfg.blockDim = dim3(kSaThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    EET_CUDA(cudaLaunchKernelEx(&cfg, kern, a, ranks, slice));
    return 0;
}

}  // namespace

int launch_sample(const SampleArgs& a, cudaStream_t stream)
{
    const int bytes = a.type == 2 ? 4 : 2;
    // As many CTAs a row as its slices need, and as fit the GPU at once; a slice of some thousand values at least.
    int ranks = 1;
    while (ranks < kSaMaxCluster && (long long)a.vocab * bytes > (long long)ranks * kSaSlice) ranks *= 2;
    while (ranks < kSaMaxCluster && (long long)a.rows * ranks <= sm_count() && a.vocab / ranks >= 4096) ranks *= 2;
    if (a.type == 0) return launch_sample_t<__half>(a, ranks, stream);
    if (a.type == 1) return launch_sample_t<__nv_bfloat16>(a, ranks, stream);
    return launch_sample_t<float>(a, ranks, stream);
}

}  // namespace eet
