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

// A bound, in its upper half, that the keys of at least k lanes reach
__device__ __forceinline__ uint32_t reached(uint32_t key, int k)
{
    uint32_t t = 0;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
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

__device__ __forceinline__ double wave_sum(double v)
{
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) rows_kernel(const BeamParams p)
{
    typedef Wide<TYPE> W;
    typedef element<TYPE> E;
    constexpr int SETS = kPer / W::n;
    __shared__ uint64_t list[kList];
    __shared__ uint32_t bounds[4], largest[4];
    __shared__ double sums[4];
    __shared__ float counts[8];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x;
    const int64_t row = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    const int b = (int)(row / p.beams), i = (int)(row % p.beams);
    if (row >= (int64_t)p.batch * p.beams) return;
    if (p.finished && p.finished[b * p.sf_b + i * p.sf_i]) return;      // nothing of it is asked for
    const E *const at = (const E *)p.logits + b * p.sl_b + i * p.sl_i;
    const int first = part * kBeamPart;
    if (tid == 0) listed = 0;

    float v[kPer];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        const int t = first + (s * kThreads + tid) * W::n;
        if (t + W::n <= p.vocab) {
            const auto raw = W::load(at + t);
#pragma unroll
            for (int j = 0; j < W::n; ++j) v[s * W::n + j] = to_f32<TYPE>(raw.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < W::n; ++j) v[s * W::n + j] = t + j < p.vocab ? to_f32<TYPE>(at[t + j]) : -__builtin_inff();
        }
    }
    auto token = [&](int e) { return first + (e / W::n * kThreads + tid) * W::n + e % W::n; };
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) most = max(most, ordered(v[e]));
    const uint32_t bound = reached(most, p.k), top = group_max<64>(most);
    if (lane == 0) {
        bounds[wave] = bound;
        largest[wave] = top;
    }
    __syncthreads();
    // (-inf is not listed: a part with fewer than k others is filled up with its first ones below)
    const uint32_t T = max(max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3])), kNone + 1);
    const float m = value_of(max(max(largest[0], largest[1]), max(largest[2], largest[3])));
    const float from = m == -__builtin_inff() ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        sum += __builtin_amdgcn_exp2f((v[e] - from) * 1.44269504088896341f);
        const uint32_t key = ordered(v[e]);
        if (key >= T) {
            const int place = atomicAdd(&listed, 1);
            if (place < kList) list[place] = (uint64_t)key << 32 | (uint32_t)~token(e);
        }
    }
    const double all = wave_sum((double)sum);
    if (lane == 0) sums[wave] = all;
    __syncthreads();
    const int n = listed;
    if (tid == 0) {
        double *const to = p.ws_sums + (row * p.parts + part) * 2;
        to[0] = m;
        to[1] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    uint64_t *const best = p.ws_best + (row * p.parts + part) * p.k;
    if (n <= kShort) {
        if (tid < n) {
            const uint64_t mine = list[tid];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > mine;
            if (rank < p.k) best[rank] = mine;
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
        if (tid == 0) listed = 0;
        __syncthreads();
        each([&](uint64_t entry) {
            if (entry < least) return;
            const int place = atomicAdd(&listed, 1);
            if (place < p.k) best[place] = entry;
        });
    };
    if (n <= kList) {
        uint64_t mine[kList / kThreads];
#pragma unroll
        for (int e = 0; e < kList / kThreads; ++e) mine[e] = e * kThreads + tid < n ? list[e * kThreads + tid] : 0;
        search([&](auto &&f) {
#pragma unroll
            for (int e = 0; e < kList / kThreads; ++e) f(mine[e]);
        });
    } else {
        search([&](auto &&f) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const uint32_t key = ordered(v[e]);
                f(key > kNone ? (uint64_t)key << 32 | (uint32_t)~token(e) : 0);
            }
        });
    }
}

__global__ void __launch_bounds__(kThreads) merge_kernel(const BeamParams p)
{
    constexpr int kKeep = 1024;
    __shared__ double score[kBeamMost], lse[kBeamMost];
    __shared__ int kind[kBeamMost];                  // 0: its candidates are what the parts left; 1: all -inf; 2: pad alone is not
    __shared__ uint64_t keys[kKeep];
    __shared__ uint32_t flats[kKeep];
    __shared__ uint32_t bounds[4];
    __shared__ float counts[8];
    __shared__ int listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x;
    for (int i = wave; i < p.beams; i += 4) {
        const int64_t row = (int64_t)b * p.beams + i;
        const double own = p.scores[b * p.ss_b + i * p.ss_i];
        const bool fine = own < (double)__builtin_inff() && own > -(double)__builtin_inff();
        int what = 0;
        double sum = 0, top = -(double)__builtin_inff();
        if (p.finished && p.finished[b * p.sf_b + i * p.sf_i]) what = 2;
        else {
            const double *const of = p.ws_sums + row * p.parts * 2;
            for (int t = lane; t < p.parts; t += 64) top = fmax(top, of[2 * t]);
            for (int d = 1; d < 64; d *= 2) top = fmax(top, __shfl_xor(top, d));
            // (a part of -inf has a sum of zero; a NaN or +inf anywhere makes its part's sum a NaN)
            for (int t = lane; t < p.parts; t += 64) sum += of[2 * t + 1] == 0 ? 0 : of[2 * t + 1] * exp(of[2 * t] - top);
            sum = wave_sum(sum);
            if (!(sum > 0 && sum < (double)__builtin_inff())) what = 1;
        }
        if (!fine) what = 1;
        if (lane == 0) {
            kind[i] = what;
            score[i] = own;
            lse[i] = what == 0 ? top + log(sum) : 0;
        }
    }
    if (tid == 0) listed = 0;
    __syncthreads();
    const int per = max(p.parts * p.k, p.k + 1), total = p.beams * per;
    // entry e of all: its key (0: there is none) and flat index
    auto entry = [&](int e, uint32_t &flat) -> uint64_t {
        const int i = e / per, r = e - i * per;
        int t = r;
        double c = -(double)__builtin_inff();
        if (kind[i] == 0) {
            if (r >= p.parts * p.k) return 0;
            const uint64_t found = p.ws_best[((int64_t)b * p.beams + i) * p.parts * p.k + r];
            if (!found) return 0;
            t = (int)~(uint32_t)found;
            c = score[i] + ((double)value_of((uint32_t)(found >> 32)) - lse[i]);
        } else {
            if (r > p.k) return 0;
            if (kind[i] == 2) {
                c = r == 0 ? score[i] : c;
                t = r == 0 ? p.pad : r - 1 < p.pad ? r - 1 : r;
            }
            if (t >= p.vocab) return 0;
        }
        flat = (uint32_t)i * (uint32_t)p.vocab + (uint32_t)t;
        return ordered(c);
    };
    uint32_t most = 0;
    for (int e = tid; e < total; e += kThreads) {
        uint32_t flat;
        most = max(most, (uint32_t)(entry(e, flat) >> 32));
    }
    const uint32_t bound = reached(most, p.k);
    if (lane == 0) bounds[wave] = bound;
    __syncthreads();
    const uint64_t T = (uint64_t)max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3])) << 32;
    for (int e = tid; e < total; e += kThreads) {
        uint32_t flat;
        const uint64_t key = entry(e, flat);
        if (key && key >= T) {
            const int place = atomicAdd(&listed, 1);
            if (place < kKeep) {
                keys[place] = key;
                flats[place] = flat;
            }
        }
    }
    __syncthreads();
    int n = listed;
    if (n > kShort) {
        // the k-th key, then, among its equals, the index up to which they are in
        Counter count{counts, 4, 0};
        uint64_t least = 0;
        uint32_t last = 0xffffffffu;
        auto search = [&](auto &&each) {
            int reach = n;
            for (uint64_t bit = 1ull << 63; bit && reach != p.k; bit >>= 1) {
                const uint64_t t = least | bit;
                int mine = 0;
                each([&](uint64_t key, uint32_t) { mine += key >= t; });
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
                    each([&](uint64_t key, uint32_t flat) { mine += key > least || (key == least && flat < t); });
                    if (count(mine) < p.k) last = t;
                }
            }
        };
        auto in = [&](uint64_t key, uint32_t flat) { return key > least || (key == least && flat <= last); };
        if (n <= kKeep) {
            uint64_t key[kKeep / kThreads];
            uint32_t flat[kKeep / kThreads];
#pragma unroll
            for (int e = 0; e < kKeep / kThreads; ++e) {
                const int at = e * kThreads + tid;
                key[e] = at < n ? keys[at] : 0;
                flat[e] = at < n ? flats[at] : 0;
            }
            search([&](auto &&f) {
#pragma unroll
                for (int e = 0; e < kKeep / kThreads; ++e)
                    if (key[e]) f(key[e], flat[e]);
            });
            if (tid == 0) listed = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kKeep / kThreads; ++e)
                if (key[e] && in(key[e], flat[e])) {
                    const int place = atomicAdd(&listed, 1);
                    if (place < kKeep) {
                        keys[place] = key[e];
                        flats[place] = flat[e];
                    }
                }
        } else {
            auto each = [&](auto &&f) {
                for (int e = tid; e < total; e += kThreads) {
                    uint32_t flat;
                    const uint64_t key = entry(e, flat);
                    if (key) f(key, flat);
                }
            };
            search(each);
            if (tid == 0) listed = 0;
            __syncthreads();
            each([&](uint64_t key, uint32_t flat) {
                if (!in(key, flat)) return;
                const int place = atomicAdd(&listed, 1);
                if (place < kKeep) {
                    keys[place] = key;
                    flats[place] = flat;
                }
            });
        }
        __syncthreads();
        n = min(listed, kKeep);
    }
    if (tid < n) {
        const uint64_t key = keys[tid];
        const uint32_t flat = flats[tid];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += keys[j] > key || (keys[j] == key && flats[j] < flat);
        if (rank < p.k) {
            p.out_scores[b * p.so_b + rank] = (float)value_of(key);
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
    hipLaunchKernelGGL(merge_kernel, dim3((uint32_t)p.batch), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace ssd
