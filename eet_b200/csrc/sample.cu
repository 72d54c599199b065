// The next token of each row of logits, drawn with temperature, top-k, top-p and min-p from a given random number.
//
//   w_i = exp((x_i - max x) / T).  In the order of x, the lowest index first among equals: top-k leaves the first k; top-p those of them in
//   front of which stands less than top_p of the w of the k; min-p those with w >= min_p; the first always stays.  Of what is left, in the
//   order of the indices, the first token whose running sum of w exceeds u times the sum of all is drawn.
//
// All of these leave a beginning of one order, so they come down to a cut: a value x*, and how many of its equals stay.  Nothing is sorted but
// a few candidates around it.
//   1  the row into shared memory, its maximum
//   2  a histogram over (max - x) / T, 64 bins to a factor of e in w: counts in front of a bin are exact, sums of w known to 1.6 %
//   3  the bins in which the cut must lie; where they hold too many values for a list, a second histogram over them alone
//   4  those values, sorted, with exact sums in front of each: the cut.  (Where one bin of the second histogram holds more than the list can,
//      as with very many equal values: bisection on x.)
//   5  what is left, summed by threads in the order of the indices; the thread whose part of the sum the random number falls into draws
// Sums are of w as whole multiples of 2^-44, from exp in 64 bits: whatever the number of CTAs and their order, they are the same, and a cut or
// a draw lies where the definition puts it but for one chance in about 2^-44 times the vocabulary.  (In 32 bits a draw from 64000 tokens would
// miss the border of some token once in some hundred rows.)
//
// A row is worked on by a cluster of 1 to 8 CTAs, which hold it in shared memory and exchange counts and candidates there.  Bound: latency,
// seven barriers of the cluster and as many trips through a slice of the row.
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
constexpr int kSaMaxSlice = 160 * 1024;      // bytes of a row in a CTA
constexpr double kSaUnit = 17592186044416.0; // 2^44
constexpr uint32_t kSaNothing = 0x007fffffu; // the key of -inf

typedef unsigned long long u64;

struct SaCut {
    uint32_t key;      // values above it stay,
    uint32_t equals;   // and the first so many of its equals
};

struct SaBracket {
    int b0, b1;        // bins that hold the cut
    uint32_t count;    // values in them
    uint32_t before;   // values in front of them
};

struct SaSmem {
    uint32_t hist[kSaBins], fine[kSaBins];
    uint32_t list[kSaList];
    uint32_t listed;
    // from every CTA of the cluster, two buffers each
    float maxima[kSaMaxCluster];
    u64 sums[2][kSaMaxCluster];
    uint32_t counts[2][kSaMaxCluster];
    // from the first CTA
    SaBracket bracket;
    SaCut cut;
    // of this CTA
    u64 warp_sum[kSaWarps];
    double warp_low[kSaWarps], warp_high[kSaWarps];
    uint32_t warp_count[kSaWarps];
    float warp_max[kSaWarps];
    uint32_t total;
    u64 mass;
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

__device__ __forceinline__ float sa_clean(float x)
{
    return x == x ? x + 0.0f : -INFINITY;
}

__device__ __forceinline__ float sa_float(float x) { return x; }
__device__ __forceinline__ float sa_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float sa_float(__nv_bfloat16 x) { return __bfloat162float(x); }

struct SaRow {
    float top;
    double over_t;       // 1 / T
    float scale;         // bins a unit of x
    // (max - x) / T, negative
    __device__ __forceinline__ double power(float x) const { return x == top ? 0.0 : ((double)x - (double)top) * over_t; }
    __device__ __forceinline__ u64 weight(float x) const
    {
        if (x == -INFINITY) return 0;
        const double e = exp(power(x));
        const u64 w = __double2ull_rn(e * kSaUnit);
        return w == 0 && e > 0.0 ? 1 : w;   // (what can be drawn stays so)
    }
    __device__ __forceinline__ float place(float x) const { return (top - x) * scale; }
    __device__ __forceinline__ int bin(float x) const { return min(kSaBins - 1, (int)place(x)); }
    // bins of the second histogram: those of [b0, b1] cut into kSaBins
    __device__ __forceinline__ int fine(float x, int b0, float per_bin) const
    {
        return max(0, min(kSaBins - 1, (int)((place(x) - (float)b0) * per_bin)));
    }
};

// Sums over the threads in front of this one, and over all (to be read behind the barrier it ends with).
template<typename V>
__device__ __forceinline__ V sa_scan(V v, V* per_warp, V& all)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();   // per_warp may still be read
    if (lane == 31) per_warp[warp] = s;
    __syncthreads();
    V before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kSaWarps; ++w) {
        if (w < warp) before += per_warp[w];
        all += per_warp[w];
    }
    return before + s - v;
}

template<typename T>
struct SaKernel {
    SaSmem& sm;
    const T* x;            // the slice, in shared memory
    int n, run;            // its values; those of a thread, consecutive and an odd number
    int ranks, rank;
    SaRow row;
    int turn = 0;          // buffer of the next exchange

    __device__ __forceinline__ float at(int i) const { return sa_clean(sa_float(x[i])); }
    template<typename F>
    __device__ __forceinline__ void each(F f) const
    {
        const int begin = (int)threadIdx.x * run, end = min(n, begin + run);
        for (int i = begin; i < end; ++i) f(at(i));
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

    // Sum and count of all CTAs' threads, to all; `before`, where asked for, those of the threads in front of this one.
    __device__ __forceinline__ void exchange(u64 sum, uint32_t count, u64& all_sum, uint32_t& all_count, u64* sum_before = nullptr,
                                             uint32_t* count_before = nullptr)
    {
        u64 cta_sum;
        uint32_t cta_count;
        u64 s = sa_scan(sum, sm.warp_sum, cta_sum);
        uint32_t c = sa_scan(count, sm.warp_count, cta_count);
        if ((int)threadIdx.x < ranks) {
            *of(&sm.sums[turn][rank], threadIdx.x) = cta_sum;
            *of(&sm.counts[turn][rank], threadIdx.x) = cta_count;
        }
        barrier();
        all_sum = 0;
        all_count = 0;
        for (int r = 0; r < ranks; ++r) {
            if (r < rank) {
                s += sm.sums[turn][r];
                c += sm.counts[turn][r];
            }
            all_sum += sm.sums[turn][r];
            all_count += sm.counts[turn][r];
        }
        if (sum_before != nullptr) *sum_before = s;
        if (count_before != nullptr) *count_before = c;
        turn ^= 1;         // (whoever writes this buffer again has passed the barrier of the other one, behind everybody's reads)
    }

    // Counts into `bins` of the first CTA; `f` is handed a value and answers its bin, or -1.
    template<typename F>
    __device__ __forceinline__ void histogram(uint32_t* bins, F f)
    {
        for (int i = threadIdx.x; i < kSaBins; i += kSaThreads) bins[i] = 0;
        barrier();         // (the first CTA's are empty, too)
        each([&](float v) {
            const int b = f(v);
            if (b >= 0) atomicAdd(&bins[b], 1u);
        });
        if (rank > 0) {
            __syncthreads();
            uint32_t* first = of(bins, 0);
            for (int i = threadIdx.x; i < kSaBins; i += kSaThreads) {
                if (bins[i] != 0) atomicAdd(&first[i], bins[i]);
            }
        }
        barrier();
    }

    // The bins of the first CTA's histogram that hold the cut, by that CTA; to all.
    //   by count   the one in which the count passes `k`, `counted` values standing in front of all of them
    //   by mass    those in which the sum of w may pass `goal`, `mass` standing in front; bin b's are between e^(-low(b + 1)) and e^(-low(b))
    template<typename F>
    __device__ __forceinline__ SaBracket narrow(const uint32_t* bins, bool by_mass, uint32_t k, uint32_t counted, double goal, double mass,
                                                F low, bool open_end)
    {
        if (rank == 0) {
            uint32_t c[kSaPerThread], sum = 0, all;
#pragma unroll
            for (int i = 0; i < kSaPerThread; ++i) {
                c[i] = bins[threadIdx.x * kSaPerThread + i];
                sum += c[i];
            }
            if (threadIdx.x == 0) sm.bracket = {kSaBins - 1, kSaBins - 1, 0, 0};   // (there behind the barriers of the sum)
            const uint32_t before = sa_scan(sum, sm.warp_count, all);
            if (by_mass) {
                double lo[kSaPerThread], hi[kSaPerThread], lo_sum = 0, hi_sum = 0, rest;
#pragma unroll
                for (int i = 0; i < kSaPerThread; ++i) {
                    const int b = threadIdx.x * kSaPerThread + i;
                    // (2e-5: what single precision may do to a value's place, and expf)
                    hi[i] = c[i] * kSaUnit * (double)(expf(-low(b)) * 1.00002f);
                    lo[i] = open_end && b == kSaBins - 1 ? 0.0 : c[i] * kSaUnit * (double)(expf(-low(b + 1)) * 0.99998f);
                    lo_sum += lo[i];
                    hi_sum += hi[i];
                }
                double lo_before = mass + sa_scan(lo_sum, sm.warp_low, rest), hi_before = mass + sa_scan(hi_sum, sm.warp_high, rest);
#pragma unroll
                for (int i = 0; i < kSaPerThread; ++i) {
                    const int b = threadIdx.x * kSaPerThread + i;
                    if (hi_before < goal && hi_before + hi[i] >= goal) sm.bracket.b0 = b;
                    if (lo_before < goal && lo_before + lo[i] >= goal) sm.bracket.b1 = b;
                    hi_before += hi[i];
                    lo_before += lo[i];
                }
            }
            else {
                uint32_t at = counted + before;
#pragma unroll
                for (int i = 0; i < kSaPerThread; ++i) {
                    if (at < k && at + c[i] >= k) sm.bracket.b0 = sm.bracket.b1 = threadIdx.x * kSaPerThread + i;
                    at += c[i];
                }
            }
            __syncthreads();
            const int b0 = sm.bracket.b0, b1 = sm.bracket.b1;
            uint32_t in = 0, front = 0;
#pragma unroll
            for (int i = 0; i < kSaPerThread; ++i) {
                const int b = threadIdx.x * kSaPerThread + i;
                front += b < b0 ? c[i] : 0;
                in += b >= b0 && b <= b1 ? c[i] : 0;
            }
            uint32_t all_in, all_front;
            sa_scan(in, sm.warp_count, all_in);
            sa_scan(front, sm.warp_count, all_front);
            if ((int)threadIdx.x < ranks) *of(&sm.bracket, threadIdx.x) = {b0, b1, all_in, counted + all_front};
        }
        barrier();
        return sm.bracket;
    }

    // The list of values between the cut's bins into the first CTA, sorted from the largest; returns the sum of w of those in front.
    // f(v): 0 in front, 1 in the bins, 2 behind.
    template<typename F>
    __device__ __forceinline__ u64 gather(uint32_t count, bool sums, F f)
    {
        if (rank == 0 && threadIdx.x == 0) sm.listed = 0;
        barrier();
        u64 front = 0;
        uint32_t* listed = of(&sm.listed, 0);
        uint32_t* list = of(sm.list, 0);
        each([&](float v) {
            const int where = f(v);
            if (where == 0 && sums) front += row.weight(v);
            if (where == 1) {
                const uint32_t i = atomicAdd(listed, 1u);
                if (i < kSaList) list[i] = sa_key(v);
            }
        });
        u64 all_front;
        uint32_t none;
        exchange(front, 0, all_front, none);
        if (rank == 0) {
            int size = 32;
            while (size < (int)count) size <<= 1;
            for (int i = count + threadIdx.x; i < size; i += kSaThreads) sm.list[i] = 0;
            __syncthreads();
            for (int k = 2; k <= size; k <<= 1) {
                for (int j = k >> 1; j > 0; j >>= 1) {
                    for (int i = threadIdx.x; i < size / 2; i += kSaThreads) {
                        const int a = 2 * i - (i & (j - 1)), b = a + j;
                        const uint32_t u = sm.list[a], v = sm.list[b];
                        if ((u < v) == ((a & k) == 0)) {
                            sm.list[a] = v;
                            sm.list[b] = u;
                        }
                    }
                    __syncthreads();
                }
            }
        }
        return all_front;
    }

    // By the first CTA, the cut in the sorted list: of `count` values, in front of which stand `before` with the sum `front`.  Leaves the first
    // `k` (none of them at all: the list is not cut by count), of those the ones in front of which stands less than `goal`, or with part > 0
    // less than that part of the sum of the k.
    __device__ __forceinline__ void cut_list(uint32_t count, uint32_t before, u64 front, uint32_t k, double goal, float part)
    {
        constexpr int kEach = kSaList / kSaThreads;
        uint32_t keep = count;
        if (k > 0) keep = min(count, k - before);
        if (part > 0.f || goal > 0.0) {
            u64 w[kEach], sum = 0, all;
            const int per = ((int)count + kSaThreads - 1) / kSaThreads, at = threadIdx.x * per;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                w[i] = i < per && at + i < (int)keep ? row.weight(sa_value(sm.list[at + i])) : 0;
                sum += w[i];
            }
            u64 run_sum = front + sa_scan(sum, sm.warp_sum, all);
            if (part > 0.f) goal = fmax((double)part * (double)(front + all), 0.5);
            uint32_t stay = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (i < per && at + i < (int)keep && (double)run_sum < goal) ++stay;
                run_sum += w[i];
            }
            sa_scan(stay, sm.warp_count, keep);
            keep = max(keep, 1u);
        }
        const uint32_t key = sm.list[keep - 1];
        uint32_t equals = 0, all_equals;
        for (int i = threadIdx.x; i < (int)keep; i += kSaThreads) equals += sm.list[i] == key;
        sa_scan(equals, sm.warp_count, all_equals);
        if ((int)threadIdx.x < ranks) *of(&sm.cut, threadIdx.x) = {key, all_equals};
    }

    // The cut by bisection: the largest key with `k` values, or a sum of w of `goal`, from it on.
    __device__ __forceinline__ SaCut bisect(bool by_mass, uint32_t k, double goal)
    {
        uint32_t lo = kSaNothing + 1, hi = sa_key(row.top);
        auto from = [&](uint32_t key, u64& mass, uint32_t& count) {
            u64 m = 0;
            uint32_t c = 0;
            each([&](float v) {
                if (sa_key(v) < key) return;
                ++c;
                if (by_mass) m += row.weight(v);
            });
            exchange(m, c, mass, count);
        };
        u64 mass;
        uint32_t count;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            from(mid, mass, count);
            if (by_mass ? (double)mass >= goal : count >= k) lo = mid;
            else hi = mid - 1;
        }
        mass = 0, count = 0;
        if (lo < 0xffffffffu) from(lo + 1, mass, count);
        uint32_t equals = by_mass ? 0 : k - count;
        if (by_mass) {
            // the first sum of equals that reaches the goal
            const u64 w = row.weight(sa_value(lo));
            uint32_t a = 1, b = kSaMaxVocab;
            while (a < b) {
                const uint32_t m = a + (b - a) / 2;
                if ((double)(mass + (u64)m * w) >= goal) b = m;
                else a = m + 1;
            }
            equals = a;
        }
        return {lo, equals};
    }

    // The cut by count, or by mass; with part > 0 both where one list does (`both` says so).  The first histogram is there.
    __device__ __forceinline__ SaCut find(bool by_mass, uint32_t k, double goal, float part, bool& both, u64& front)
    {
        const float per_e = 1.0f / kSaBinsPerE;
        SaBracket br = narrow(sm.hist, by_mass, k, 0, goal, 0.0, [&](int b) { return b * per_e; }, true);
        both = false;
        if (!by_mass && part > 0.f && br.before + br.count <= kSaList) {
            both = true;       // everything up to the cut
            br = {0, br.b1, br.before + br.count, 0};
        }
        if (br.count <= kSaList) {
            const SaBracket b = br;
            front = gather(b.count, by_mass, [&](float v) {
                if (v == -INFINITY) return 2;
                const int i = row.bin(v);
                return i < b.b0 ? 0 : i <= b.b1 ? 1 : 2;
            });
            if (rank == 0) cut_list(b.count, b.before, front, by_mass ? 0 : k, by_mass ? goal : 0.0, both ? part : 0.f);
            barrier();
            return sm.cut;
        }
        // the second histogram, and what stands in front of it
        const int c0 = br.b0, c1 = br.b1;
        const float per_bin = (float)kSaBins / (float)(c1 - c0 + 1);
        u64 ahead = 0;
        histogram(sm.fine, [&](float v) {
            if (v == -INFINITY) return -1;
            const int i = row.bin(v);
            if (i < c0 && by_mass) ahead += row.weight(v);
            return i < c0 || i > c1 ? -1 : row.fine(v, c0, per_bin);
        });
        u64 mass;
        uint32_t none;
        exchange(ahead, 0, mass, none);
        br = narrow(sm.fine, by_mass, k, br.before, goal, (double)mass, [&](int b) { return (c0 + b / per_bin) * per_e; }, c1 == kSaBins - 1);
        if (br.count <= kSaList) {
            const SaBracket b = br;
            front = gather(b.count, by_mass, [&](float v) {
                if (v == -INFINITY) return 2;
                const int i = row.bin(v);
                if (i < c0 || i > c1) return i < c0 ? 0 : 2;
                const int j = row.fine(v, c0, per_bin);
                return j < b.b0 ? 0 : j <= b.b1 ? 1 : 2;
            });
            if (rank == 0) cut_list(b.count, b.before, front, by_mass ? 0 : k, by_mass ? goal : 0.0, 0.f);
            barrier();
            return sm.cut;
        }
        front = 0;
        return bisect(by_mass, k, goal);
    }
};

template<typename T>
__global__ void __launch_bounds__(kSaThreads) sample_rows_kernel(const SampleArgs a, int ranks, int slice)
{
    extern __shared__ __align__(16) uint8_t sa_dyn[];
    __shared__ SaSmem sm;
    const int tid = threadIdx.x;
    const int rank = ranks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const long long r = blockIdx.x / ranks;
    pdl_launch_dependents();
    pdl_wait();
    const T* src = (const T*)a.logits + r * a.row_stride + (long long)rank * slice;
    const int n = max(0, min(slice, a.vocab - rank * slice));
    // ---- 1  the slice, whole 16 bytes at a time; it begins in shared memory where its first byte lies in 16 of global memory
    constexpr int kPer = 16 / sizeof(T);
    const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T* x = reinterpret_cast<T*>(sa_dyn) + skew;
    float top = -INFINITY;
    {
        const uint4* from = reinterpret_cast<const uint4*>(src - skew);
        const int words = (skew + n + kPer - 1) / kPer;
        constexpr int kAhead = 4;
        for (int i0 = tid; i0 < words; i0 += kAhead * kSaThreads) {
            uint4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kSaThreads;
                if (i >= words) continue;
                if (i * kPer >= skew && (i + 1) * kPer <= skew + n) {
                    v[k] = from[i];
                }
                else {             // the ends
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
                if (i >= words) continue;
                reinterpret_cast<uint4*>(sa_dyn)[i] = v[k];
                const T* e = reinterpret_cast<const T*>(&v[k]);
#pragma unroll
                for (int j = 0; j < kPer; ++j) top = fmaxf(top, sa_clean(sa_float(e[j])));
            }
        }
    }
    SaKernel<T> s = {sm, x, n, ((n + kSaThreads - 1) / kSaThreads) | 1, ranks, rank, {}};
    top = warp_max(top);
    if ((tid & 31) == 0) sm.warp_max[tid >> 5] = top;
    s.barrier();                   // (every CTA of the cluster has begun)
    for (int w = 0; w < kSaWarps; ++w) top = fmaxf(top, sm.warp_max[w]);
    if (tid < ranks) *s.of(&sm.maxima[rank], tid) = top;
    s.barrier();
    for (int i = 0; i < ranks; ++i) top = fmaxf(top, sm.maxima[i]);
    if (top == -INFINITY) {        // nothing can be drawn
        if (rank == 0 && tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = -INFINITY;
        }
        return;                    // (all of the cluster, and the last word to another CTA lies in front of a barrier)
    }
    float temperature = a.temperatures != nullptr ? a.temperatures[r] : a.temperature;
    const float part = a.top_ps != nullptr ? a.top_ps[r] : a.top_p;
    const float least = a.min_ps != nullptr ? a.min_ps[r] : a.min_p;
    const int wanted = a.top_ks != nullptr ? a.top_ks[r] : a.top_k;
    const bool greedy = !(temperature > 0.f);
    if (greedy) temperature = 1.0f;
    s.row = {top, 1.0 / (double)temperature, kSaBinsPerE / temperature};

    SaCut cut = {kSaNothing, 0u};   // everything above -inf
    float floor = -INFINITY;        // of min-p
    if (greedy) {
        cut = {sa_key(top), 1u};
    }
    else {
        if (least > 0.f) floor = __double2float_ru((double)top + (double)temperature * log(fmin((double)least, 1.0)));
        const bool by_count = wanted > 0 && wanted < a.vocab, by_mass = part < 1.0f;
        if (by_count || by_mass) {
            // ---- 2
            u64 sum = 0;
            uint32_t count = 0;
            s.histogram(sm.hist, [&](float v) {
                if (v == -INFINITY) return -1;
                ++count;
                if (!by_count) sum += s.row.weight(v);
                return s.row.bin(v);
            });
            s.exchange(sum, count, sum, count);
            // ---- 3, 4
            bool both = false;
            u64 front = 0;
            const bool cut_count = by_count && (uint32_t)wanted < count;
            if (cut_count) cut = s.find(false, wanted, 0.0, by_mass ? fmaxf(part, 1e-30f) : 0.f, both, front);
            if (by_mass && !both) {
                if (by_count) {    // the sum of what top-k leaves
                    u64 w = 0;
                    s.each([&](float v) {
                        if (sa_key(v) > cut.key) w += s.row.weight(v);
                    });
                    uint32_t none;
                    s.exchange(w, 0, sum, none);
                    sum += cut.equals * s.row.weight(sa_value(cut.key));
                }
                const SaCut by_k = cut;
                cut = s.find(true, 0, fmax((double)part * (double)sum, 0.5), 0.f, both, front);
                if (cut.key == by_k.key) cut.equals = min(cut.equals, by_k.equals);
            }
        }
    }
    // ---- 5
    u64 mine = 0, all, before;
    uint32_t equals = 0, all_equals, equals_before;
    const int begin = tid * s.run, end = min(n, begin + s.run);
    const float edge = sa_value(cut.key);
    const bool some = cut.equals > 0 && edge >= floor;
    for (int i = begin; i < end; ++i) {
        const float v = s.at(i);
        if (v > edge && v >= floor) mine += s.row.weight(v);
        equals += v == edge;
    }
    // (equals first: how many of this thread's stay follows from those in front)
    u64 none;
    s.exchange(0, some ? equals : 0, none, all_equals, nullptr, &equals_before);
    const u64 edge_weight = some ? s.row.weight(edge) : 0;
    const uint32_t stay = some && equals_before < cut.equals ? min(equals, cut.equals - equals_before) : 0;
    mine += stay * edge_weight;
    uint32_t one;
    s.exchange(mine, 0, all, one, &before, nullptr);
    double goal = (double)a.uniform[r] * (double)all;
    if (!(goal >= 0.0)) goal = 0.0;
    if (goal >= (double)all) goal = __longlong_as_double(__double_as_longlong((double)all) - 1);   // (the number below)
    if ((double)before <= goal && (double)(before + mine) > goal && mine > 0) {
        uint32_t seen = 0;
        u64 sum = before;
        for (int i = begin; i < end; ++i) {
            const float v = s.at(i);
            u64 w = 0;
            if (v > edge && v >= floor) w = s.row.weight(v);
            else if (v == edge && seen < stay) w = edge_weight, ++seen;
            sum += w;
            if (w > 0 && (double)sum > goal) {
                a.tokens[r] = (long long)rank * slice + i;
                a.logprobs[r] = (float)(s.row.power(v) - log((double)all / kSaUnit));
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
    while (ranks < kSaMaxCluster && (long long)a.vocab * bytes > (long long)ranks * (kSaMaxSlice - 64)) ranks *= 2;
    while (ranks < kSaMaxCluster && (long long)a.rows * 2 * ranks <= sm_count() && a.vocab / ranks >= 4096) ranks *= 2;
    if (a.type == 0) return launch_sample_t<__half>(a, ranks, stream);
    if (a.type == 1) return launch_sample_t<__nv_bfloat16>(a, ranks, stream);
    return launch_sample_t<float>(a, ranks, stream);
}

}  // namespace eet
