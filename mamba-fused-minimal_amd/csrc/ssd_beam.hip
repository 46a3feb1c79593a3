// Beam search's selection: the k best of beams x vocab candidates of a row,
//
//   c[i, v] = scores[i] + (logits[i, v] - log(sum_u exp(logits[i, u])))
//
// best first, equals by the lowest i * vocab + v.  A beam that has finished has one candidate, `pad` at scores[i].  What is not a number
// (a NaN or +inf among a beam's logits, in its score) counts as -inf.
//
// Order within a beam is that of its logits, so one pass over them does: rows_kernel takes a part of one beam's row into registers,
// leaves its largest, the sum of its exponentials and its k best; merge_kernel puts the parts' sums together and selects among what the parts
// left.  The scores that decide between beams are made in 64 bits from sums whose terms have the error of one fp32 exponential; the sums
// of a part are fp32 over a thread's 32 terms and 64 bits beyond.
//
// The k best of n values: k lanes of a wave whose largest reach T are k values that do, so whatever is below T is out; a T is found
// from the lanes' largest with 16 ballots.  What reaches the largest T of the waves goes into a list, a little more than k as a rule, and a
// value's rank in it is the number of those before it.  Lists of many equals are cut by a search for the k-th, bit by bit.
//
// Bound by vector instructions where rows are many (16 for a logit, one of them an exponential of four times the others' time) and by latency where
// they are few.  A part is 8192 logits: 32 to a thread, eight waves to a SIMD.  Measured: 64 rows of 8 beams x 50000 bf16, 16 best, in 25.3 us (rows 20.0 on
// 51 MB, merge 6.5), one row of 4 x 32000 in 10.6 (5.4 + 4.1), 3 rows of 5 x 128001 fp32 in 11.2 (6.7 + 5.0).  Slower: two parts to a workgroup with the
// second one's logits on the way (rows 30), values found by way of LDS in the few lanes that have one (rows 22.4).
#include "ssd_decode.h"

namespace ssd {
namespace {

using namespace layer;

constexpr int kThreads = 256, kPer = kBeamPart / kThreads;      // logits of a thread
constexpr int kList = 2048, kShort = 128;                        // what is listed; lists that are ranked as they are

// fp32 as integers of the same order; -0 as +0
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ uint64_t ordered(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(uint64_t o) { return __builtin_bit_cast(double, o >> 63 ? o ^ 0x8000000000000000ull : ~o); }

constexpr uint32_t kNone = 0x007fffffu;      // ordered(-inf)

// A bound that the keys of at least k lanes reach: the largest one in the upper bits down to LOWEST
template <int LOWEST> __device__ __forceinline__ uint32_t reached(uint32_t key, int k)
{
    uint32_t t = 0;
#pragma unroll 4
    for (uint32_t bit = 1u << 31; bit >= 1u << LOWEST; bit >>= 1)
        if (__popcll(__ballot(key >= (t | bit))) >= k) t |= bit;
    return t;
}

// The sum over the workgroup of what its threads count; `step` alternates between calls
struct Counter {
    float *part;      // [2][waves]
    int waves, step;
    __device__ __forceinline__ int operator()(int mine)
    {
        const float sum = group_sum<64>((float)mine);
        float *at = part + (step & 1) * waves;
        ++step;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = sum;
        __syncthreads();
        float all = 0.f;
        for (int w = 0; w < waves; ++w) all += at[w];
        return (int)all;
    }
};

// Sum and largest over a wave, in every lane: moves between lanes of sixteen, then between sixteens and halves
template <class T, class F> __device__ __forceinline__ T over_wave(T v, F &&join)
{
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int WORDS = sizeof(T) / 4;
    struct Words { uint32_t w[WORDS]; };
    auto each = [&](auto &&f) {
        Words x = __builtin_bit_cast(Words, v);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) x.w[i] = f(x.w[i]);
        return __builtin_bit_cast(T, x);
    };
    v = join(v, each([](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true); }));      // lane ^ 1
    v = join(v, each([](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true); }));      // lane ^ 2
    v = join(v, each([](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true); }));     // the other quad of eight
    v = join(v, each([](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true); }));     // the other half of sixteen
    auto both = [&](auto &&swap) {
        const Words x = __builtin_bit_cast(Words, v);
        Words l, r;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            const auto t = swap(x.w[i]);
            l.w[i] = t[0];
            r.w[i] = t[1];
        }
        v = join(__builtin_bit_cast(T, l), __builtin_bit_cast(T, r));
    };
    both([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    both([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
#endif
    return v;
}

// Sum over four lanes, in each of them
__device__ __forceinline__ int quad_sum(int v)
{
#if defined(__HIP_DEVICE_COMPILE__)
    v += __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true);
#endif
    return v;
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads, TYPE == DT_F32 ? 5 : 8) rows_kernel(const BeamParams p)
{
    typedef Wide<TYPE> W;
    typedef element<TYPE> E;
    constexpr int SETS = kPer / W::n;
    __shared__ uint64_t list[kList];
    __shared__ uint32_t bounds[4], largest[4];
    __shared__ double sums[4];
    __shared__ float counts[8];
    __shared__ int listed[4], chosen;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x;
    const int64_t row = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    if (row >= (int64_t)p.batch * p.beams) return;
    const int b = (int)((uint32_t)row / (uint32_t)p.beams), i = (int)((uint32_t)row % (uint32_t)p.beams);
    if (p.finished && p.finished[b * p.sf_b + i * p.sf_i]) return;      // nothing of it is asked for
    const E *const at = (const E *)p.logits + b * p.sl_b + i * p.sl_i;
    const int first = part * kBeamPart;
    // (as they are in memory: taken apart again where they are used, for more waves on a compute unit)
    typename W::Pack raw[SETS];
    const float none = -__builtin_inff();
    const int sets = (min(p.vocab - first, kBeamPart) + kThreads * W::n - 1) / (kThreads * W::n);      // (the last part may have fewer)
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        if (s > 0 && s >= sets) break;
        const int t = first + (s * kThreads + tid) * W::n;
        if (t + W::n <= p.vocab) raw[s] = W::load_once(at + t);
        else
#pragma unroll
            for (int j = 0; j < W::n; ++j) raw[s].e[j] = t + j < p.vocab ? at[t + j] : from_f32<TYPE>(none);
    }
    // (the 32 numbers are not to be kept between their uses)
    auto forget = [&] {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (sizeof(E) == 2)
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
                u32x4 x = __builtin_bit_cast(u32x4, raw[s]);
                asm volatile("" : "+v"(x));
                raw[s] = __builtin_bit_cast(typename W::Pack, x);
            }
#endif
    };
    auto value = [&](int e) { return to_f32<TYPE>(raw[e / W::n].e[e % W::n]); };
    auto token = [&](int e) { return first + (e / W::n * kThreads + tid) * W::n + e % W::n; };
    // (a NaN is passed over here and makes the sum one)
    float most = none;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        if (s > 0 && s >= sets) break;
#pragma unroll
        for (int e = s * W::n; e < (s + 1) * W::n; ++e) most = fmaxf(most, value(e));
    }
    const uint32_t bound = reached<16>(ordered(most), p.k), top = ordered(over_wave(most, [](float x, float y) { return fmaxf(x, y); }));
    if (lane == 0) {
        bounds[wave] = bound;
        largest[wave] = top;
    }
    __syncthreads();
    // (-inf is not listed: a part with fewer than k others is filled up with its first ones below)
    const uint32_t T = max(max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3])), kNone + 1);
    const float m = value_of(max(max(largest[0], largest[1]), max(largest[2], largest[3])));
    forget();
    // 2^(v log2(e) - shift), one rounding to an exponent: `shift` is a rounded product, and log2(e) in fp32 is off by a factor of 1 + kOff.  What the
    // sum is relative to takes both in (the second at the largest logit, around which the sum is).  The exponent of the largest logit is what `shift`
    // is rounded off by: 1/16 at most up to kFar, more than fp32 has exponents for from 3e9 on, where logits that forbid a token lie (-1e10, the
    // lowest number).  A part whose largest is farther out than kFar is summed as 2^((v - m) log2(e)), relative to m: v - m is exact, or so far down
    // that nothing is left of it.
    constexpr float kLog = 1.44269504088896341f, kFar = 1048576.f;
    constexpr double kOff = (double)kLog / 1.44269504088896340736 - 1;
    // (fp16 does not reach it)
    const bool far = TYPE != DT_F16 && __builtin_amdgcn_readfirstlane(fabsf(m) > kFar && m != none);
    const float shift = m == none ? 0.f : m * kLog, least_value = value_of(T);
    float far_sum = 0.f;
    if (far) {
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            if (s > 0 && s >= sets) break;
#pragma unroll
            for (int e = s * W::n; e < (s + 1) * W::n; ++e) far_sum += __builtin_amdgcn_exp2f((value(e) - m) * kLog);
        }
        forget();
    }
    // (a wave lists by itself: a count in common would be a round trip through LDS for each value found)
    float sum = 0.f;
    int found = 0;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        if (s > 0 && s >= sets) break;
#pragma unroll
        for (int e = s * W::n; e < (s + 1) * W::n; ++e) {
            const float v = value(e);
            sum += __builtin_amdgcn_exp2f(fmaf(v, kLog, -shift));
            const uint64_t who = __ballot(v >= least_value);
            if (!who) continue;
            const int place = found + __popcll(who & ((1ull << lane) - 1));
            if (v >= least_value && place < kList / 4) list[wave * (kList / 4) + place] = (uint64_t)ordered(v) << 32 | (uint32_t)~token(e);
            found += __popcll(who);
        }
    }
    const double all = over_wave((double)(far ? far_sum : sum), [](double x, double y) { return x + y; });
    if (lane == 0) {
        sums[wave] = all;
        listed[wave] = found;
    }
    __syncthreads();
    int n = 0, most_listed = 0, start[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        start[w] = n;
        n += listed[w];
        most_listed = max(most_listed, listed[w]);
    }
    // the j-th of what is listed (n of them, none left out)
    auto at_list = [&](int j) {
        const int w = (j >= start[1]) + (j >= start[2]) + (j >= start[3]);
        return list[w * (kList / 4) + j - (w == 0 ? 0 : w == 1 ? start[1] : w == 2 ? start[2] : start[3])];
    };
    if (tid == 0) {
        double *const to = p.ws_sums + (row * p.parts + part) * 2;
        to[0] = m == none || far ? (double)m : 0.69314718055994530942 * shift - kOff * m;
        to[1] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    uint64_t *const best = p.ws_best + (row * p.parts + part) * p.k;
    if (n <= kShort && most_listed <= kList / 4) {
        // four lanes to a value, each a quarter of those it is compared with
        for (int first = 0; first < n; first += kThreads / 4) {
            const int e = first + tid / 4;
            const uint64_t mine = e < n ? at_list(e) : 0;
            int rank = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll 4
                for (int j = tid & 3; j < listed[w]; j += 4) rank += list[w * (kList / 4) + j] > mine;
            rank = quad_sum(rank);
            if (e < n && (tid & 3) == 0 && rank < p.k) best[rank] = mine;
        }
        if (n < p.k && wave == 0) {
            // fewer than k of the first 128 are not -inf
            int place = n;
            for (int h = 0; h < 2; ++h) {
                const int t = first + 64 * h + lane;
                const bool none = t < p.vocab && ordered(to_f32<TYPE>(at[t])) == kNone;
                const uint64_t who = __ballot(none);
                const int to = place + __popcll(who & ((1ull << lane) - 1));
                if (none && to < p.k) best[to] = (uint64_t)kNone << 32 | (uint32_t)~t;
                place += __popcll(who);
            }
            if (place + lane < p.k) best[place + lane] = 0;
        }
        return;
    }
    // the k-th of them, bit by bit from the first in which they differ: entries are all different
    Counter count{counts, 4, 0};
    const uint64_t differ = (uint64_t)T << 32 ^ ((uint64_t)ordered(m) << 32 | 0xffffffffu), high = 1ull << (63 - __builtin_clzll(differ));
    uint64_t least = ((uint64_t)T << 32) & ~(2 * high - 1);
    auto search = [&](auto &&each) {
        for (uint64_t bit = high; bit; bit >>= 1) {
            const uint64_t t = least | bit;
            int mine = 0;
            each([&](uint64_t entry) { mine += entry >= t; });
            const int reach = count(mine);
            if (reach >= p.k) least = t;
            if (reach == p.k) break;
        }
        if (tid == 0) chosen = 0;
        __syncthreads();
        each([&](uint64_t entry) {
            if (entry < least) return;
            const int place = atomicAdd(&chosen, 1);
            if (place < p.k) best[place] = entry;
        });
    };
    if (most_listed <= kList / 4)
        search([&](auto &&f) {
#pragma unroll 1
            for (int e = tid; e < n; e += kThreads) f(at_list(e));
        });
    else
        search([&](auto &&f) {      // (read again: what few calls need is not worth registers in all of them)
#pragma unroll 1
            for (int s = 0; s < SETS; ++s) {
                const int t = first + (s * kThreads + tid) * W::n;
#pragma unroll 1
                for (int j = 0; j < W::n; ++j) {
                    const float v = t + j < p.vocab ? to_f32<TYPE>(at[t + j]) : none;
                    const uint32_t key = v == v ? ordered(v) : 0;
                    f(key > kNone ? (uint64_t)key << 32 | (uint32_t)~(t + j) : 0);
                }
            }
        });
}

constexpr int kMerged = 1 << 22;      // rows of a launch, which has below 2^32 threads

// ENTRIES: candidates of a thread, kept in registers; 0: of any number, made again where they are looked at
template <int THREADS, int ENTRIES>
__global__ void __launch_bounds__(THREADS) merge_kernel(const BeamParams p)
{
    constexpr int WAVES = THREADS / 64, kKeep = 1024;
    __shared__ double score[kBeamMost], top_of[kBeamMost], log_of[kBeamMost];      // a beam's sum: e^(top_of + log_of)
    __shared__ int kind[kBeamMost];                  // 0: its candidates are what the parts left; 1: all -inf; 2: pad alone is not
    __shared__ uint64_t keys[kKeep];
    __shared__ uint32_t flats[kKeep];
    __shared__ uint32_t bounds[WAVES];
    __shared__ float counts[2 * WAVES];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = p.first + (int)blockIdx.x;
    const int left = p.parts * p.k, per = max(left, p.k + 1), total = p.beams * per;
    const uint64_t *const best = p.ws_best + (int64_t)b * p.beams * left;
    // what the parts left, asked for in front of everything else
    uint64_t found[ENTRIES > 0 ? ENTRIES : 1], key[ENTRIES > 0 ? ENTRIES : 1];
    int beam[ENTRIES > 0 ? ENTRIES : 1];
    auto split = [&](int e, int &i) {                // an entry's beam, and its place there
        i = e / per;
        return e - i * per;
    };
#pragma unroll
    for (int j = 0; j < ENTRIES; ++j) {
        const int e = j * THREADS + tid;
        found[j] = 0;
        beam[j] = 0;
        if (e < total) {
            const int r = split(e, beam[j]);
            if (r < left) found[j] = best[beam[j] * left + r];
        }
    }
    // sums of the beams: as many lanes to one as it has parts, up to a wave
    int lanes = 1;
    while (lanes < p.parts && lanes < 64) lanes *= 2;
    for (int first = 0; first < p.beams; first += THREADS / lanes) {
        const int i = first + tid / lanes, at = tid & (lanes - 1);
        const bool there = i < p.beams;
        double own = 0, sum = 0, top = -(double)__builtin_inff();
        bool ended = false;
        if (there) {
            own = p.scores[b * p.ss_b + i * p.ss_i];
            ended = p.finished && p.finished[b * p.sf_b + i * p.sf_i];
        }
        const double *const of = p.ws_sums + ((int64_t)b * p.beams + i) * p.parts * 2;
        const bool look = there && !ended;
        if (look)
            for (int t = at; t < p.parts; t += lanes) top = fmax(top, of[2 * t]);
        for (int d = 1; d < lanes; d *= 2) top = fmax(top, __shfl_xor(top, d));
        // (a part of -inf has a sum of zero; a NaN or +inf anywhere makes its part's sum a NaN)
        if (look)
            for (int t = at; t < p.parts; t += lanes) sum += of[2 * t + 1] == 0 ? 0 : of[2 * t + 1] * exp(of[2 * t] - top);
        for (int d = 1; d < lanes; d *= 2) sum += __shfl_xor(sum, d);
        if (there && at == 0) {
            const bool fine = own < (double)__builtin_inff() && own > -(double)__builtin_inff();
            kind[i] = !fine ? 1 : ended ? 2 : sum > 0 && sum < (double)__builtin_inff() ? 0 : 1;
            score[i] = own;
            top_of[i] = top;
            log_of[i] = kind[i] == 0 ? log(sum) : 0;
        }
    }
    if (tid == 0) listed = 0;
    __syncthreads();
    // an entry's key (0: there is none) and flat index
    auto entry = [&](int i, int r, uint64_t found, uint32_t &flat) -> uint64_t {
        int t = r;
        double c = -(double)__builtin_inff();
        const int what = kind[i];
        if (what == 0) {
            if (!found) return 0;
            t = (int)~(uint32_t)found;
            // (not less the sum of both: beside a large logit 64 bits do not hold the second)
            c = score[i] + (((double)value_of((uint32_t)(found >> 32)) - top_of[i]) - log_of[i]);
        } else {
            if (r > p.k) return 0;
            if (what == 2) {
                c = r == 0 ? score[i] : c;
                t = r == 0 ? p.pad : r - 1 < p.pad ? r - 1 : r;
            }
            if (t >= p.vocab) return 0;
        }
        flat = (uint32_t)i * (uint32_t)p.vocab + (uint32_t)t;
        return ordered(c);
    };
    if constexpr (ENTRIES > 0) {
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j) {
            const int e = j * THREADS + tid;
            uint32_t flat;
            key[j] = e < total ? entry(beam[j], e - beam[j] * per, found[j], flat) : 0;
        }
    }
    auto each = [&](auto &&f) {                      // f(key, flat index, as a function: it is seldom asked for)
        if constexpr (ENTRIES > 0) {
#pragma unroll
            for (int j = 0; j < ENTRIES; ++j)
                if (key[j]) f(key[j], [&] {
                    uint32_t flat;
                    entry(beam[j], j * THREADS + tid - beam[j] * per, found[j], flat);
                    return flat;
                });
        } else {
            for (int e = tid; e < total; e += THREADS) {
                int i;
                const int r = split(e, i);
                uint32_t flat;
                const uint64_t k = entry(i, r, r < left ? best[i * left + r] : 0, flat);
                if (k) f(k, [&] { return flat; });
            }
        }
    };
    uint32_t most = 0;
    each([&](uint64_t k, auto &&) { most = max(most, (uint32_t)(k >> 32)); });
    const uint32_t bound = reached<4>(most, p.k);      // (of scores 1e-4 apart)
    if (lane == 0) bounds[wave] = bound;
    __syncthreads();
    uint32_t high = 0;
    for (int w = 0; w < WAVES; ++w) high = max(high, bounds[w]);
    const uint64_t T = (uint64_t)high << 32;
    auto keep = [&](uint64_t k, uint32_t flat) {
        const int place = atomicAdd(&listed, 1);
        if (place < kKeep) {
            keys[place] = k;
            flats[place] = flat;
        }
    };
    each([&](uint64_t k, auto &&flat) {
        if (k >= T) keep(k, flat());
    });
    __syncthreads();
    int n = listed;
    if (n > kShort) {
        // the k-th key, then, among its equals, the index up to which they are in
        Counter count{counts, WAVES, 0};
        uint64_t least = 0;
        uint32_t last = 0xffffffffu;
        int reach = n;
        for (uint64_t bit = 1ull << 63; bit && reach != p.k; bit >>= 1) {
            const uint64_t t = least | bit;
            int mine = 0;
            each([&](uint64_t k, auto &&) { mine += k >= t; });
            const int c = count(mine);
            if (c >= p.k) {
                least = t;
                reach = c;
            }
        }
        if (reach != p.k) {
            last = 0;
            for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
                // whether fewer than k are in with indices below last + bit
                const uint32_t t = last | bit;
                int mine = 0;
                each([&](uint64_t k, auto &&flat) { mine += k > least || (k == least && flat() < t); });
                if (count(mine) < p.k) last = t;
            }
        }
        if (tid == 0) listed = 0;
        __syncthreads();
        each([&](uint64_t k, auto &&flat) {
            if (k < least) return;
            const uint32_t f = flat();
            if (k > least || f <= last) keep(k, f);
        });
        __syncthreads();
        n = min(listed, kKeep);
    }
    for (int first = 0; first < n; first += THREADS / 4) {
        const int e = first + tid / 4;
        const uint64_t mine = e < n ? keys[e] : 0;
        const uint32_t flat = e < n ? flats[e] : 0;
        int rank = 0;
#pragma unroll 4
        for (int j = tid & 3; j < n; j += 4) rank += keys[j] > mine || (keys[j] == mine && flats[j] < flat);
        rank = quad_sum(rank);
        if (e < n && (tid & 3) == 0 && rank < p.k) {
            p.out_scores[b * p.so_b + rank] = (float)value_of(mine);
            p.parents[b * p.sp_b + rank] = (int32_t)(flat / (uint32_t)p.vocab);
            p.tokens[b * p.st_b + rank] = (int32_t)(flat % (uint32_t)p.vocab);
        }
    }
}

}  // namespace

hipError_t launch_beam_select(const BeamParams &p, hipStream_t s)
{
    if (p.batch == 0 || p.k == 0) return hipSuccess;
    const int64_t rows = (int64_t)p.batch * p.beams;
    const uint32_t gy = (uint32_t)(rows < 32768 ? rows : 32768), gz = (uint32_t)((rows + gy - 1) / gy);
    const dim3 grid((uint32_t)p.parts, gy, gz);
    if (p.type == DT_F32) hipLaunchKernelGGL(rows_kernel<DT_F32>, grid, dim3(kThreads), 0, s, p);
    else if (p.type == DT_BF16) hipLaunchKernelGGL(rows_kernel<DT_BF16>, grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL(rows_kernel<DT_F16>, grid, dim3(kThreads), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t total = (int64_t)p.beams * (p.parts * p.k > p.k ? p.parts * p.k : p.k + 1);
    // (entries in registers, as few to a thread as threads allow: 64 rows of 896, 512 threads 6.3 us, 256 8.1, 1024 6.5; one of 64, 4.2 against 4.6)
    BeamParams some = p;
    for (int64_t first = 0; first < p.batch; first += kMerged) {
        some.first = (int)first;
        const dim3 rows_of((uint32_t)(p.batch - first < kMerged ? p.batch - first : kMerged));
        if (total <= 256) hipLaunchKernelGGL((merge_kernel<256, 1>), rows_of, dim3(256), 0, s, some);
        else if (total <= 512 * 2) hipLaunchKernelGGL((merge_kernel<512, 2>), rows_of, dim3(512), 0, s, some);
        else if (total <= 512 * 16) hipLaunchKernelGGL((merge_kernel<512, 16>), rows_of, dim3(512), 0, s, some);
        else hipLaunchKernelGGL((merge_kernel<512, 0>), rows_of, dim3(512), 0, s, some);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ssd
