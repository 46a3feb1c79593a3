// What stands between two blocks: the norm behind a block, its gate, the residual with its scale, and the next block's norm.
//
//   n = x w / sqrt(mean(x^2) + eps)   (n = x without w);   t = factor residual + gate n;   r = 1 / sqrt(mean(t^2) + eps);   u = t next_w
//   out = u r,   or in 8 bits  q = rint(u (127 (1 / max|u|))), scale = max|u| r / 127;   residual_out = t, rounded
//
// The second norm is that of t in 32 bits, and so are its 8 bits: r is common to a row and cancels in them.  A row of zeros has q = 0
// and scale = 0, a row with a NaN or an infinity in u a scale of NaN.
//
// HBM bound: x and the residual are read once and t and out written once, with the row in registers between its two sums, the second of which
// depends on the first.  Four waves share a row, or as many as hold a long one; many short ones have a wave each (lane-to-lane moves
// only).  Rows of some thousand 16-bit elements are worked on one after the other by workgroups that stay: the weights in registers, the next row
// on its way.  Large results go past the caches.  Rows too long for the registers are read three times, from the caches as a rule.
// Measured: 32768 x 2560 bf16 in 128 us, 5.2 TB/s, a copy's rate (8-bit results 113 us); 5703 x 1537 fp32 in 32 us, 4.4 TB/s; 64 x 2560 in 3.9 us,
// most of it the wait for two loads, two sums and a store in turn.
#include "ssd_decode.h"

namespace ssd {
namespace {

using namespace layer;

constexpr float kSmallest = 1e-36f;      // 127 / max|u| stays finite above it; rows of nothing larger are zeros

template <int TYPE, int N> struct Set {
    typedef Wide<TYPE> W;
    typedef element<TYPE> E;
    typename W::Pack v[N == 8 ? 8 / W::n : 1];
    __device__ __forceinline__ void load(const E *p)
    {
        if constexpr (N == 8) {
#pragma unroll
            for (int h = 0; h < 8 / W::n; ++h) v[h] = W::load(p + h * W::n);
        } else v[0].e[0] = *p;
    }
    __device__ __forceinline__ void load_once(const E *p)
    {
        if constexpr (N == 8) {
#pragma unroll
            for (int h = 0; h < 8 / W::n; ++h) v[h] = W::load_once(p + h * W::n);
        } else v[0].e[0] = *p;
    }
    __device__ __forceinline__ float operator[](int j) const { return to_f32<TYPE>(v[j / W::n].e[j % W::n]); }
    // past: results go past the caches
    __device__ __forceinline__ static void store(E *p, const float (&f)[N], bool past)
    {
        if constexpr (N == 8) {
#pragma unroll
            for (int h = 0; h < 8 / W::n; ++h) {
                typename W::Pack q;
#pragma unroll
                for (int j = 0; j < W::n; ++j) q.e[j] = from_f32<TYPE>(f[h * W::n + j]);
                if (past) W::store_past(p + h * W::n, q);
                else W::store(p + h * W::n, q);
            }
        } else *p = from_f32<TYPE>(f[0]);
    }
};

// N of a row of weights or gates, in the type of x or in fp32
template <int TYPE, int N> __device__ __forceinline__ void factors(const void *base, int64_t at, int wide, float (&f)[N])
{
    if (TYPE == DT_F32 || wide) {
        Set<DT_F32, N> s;
        s.load((const float *)base + at);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = s[j];
    } else {
        Set<TYPE, N> s;
        s.load((const element<TYPE> *)base + at);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = s[j];
    }
}

// The largest over a wave, in every lane
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#if defined(__HIP_DEVICE_COMPILE__)
    auto moved = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true); };
    using std::integral_constant;
    v = max(v, moved(v, integral_constant<int, 0xb1>{}));       // lane ^ 1
    v = max(v, moved(v, integral_constant<int, 0x4e>{}));       // lane ^ 2
    v = max(v, moved(v, integral_constant<int, 0x141>{}));      // the other quad of eight lanes
    v = max(v, moved(v, integral_constant<int, 0x140>{}));      // the other half of sixteen
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(h[0], h[1]);
#endif
    return v;
}

template <int N> __device__ __forceinline__ void store_i8(int8_t *p, const float (&u)[N], float inverse)
{
    if constexpr (N == 8) {
        typedef __attribute__((ext_vector_type(2), aligned(1))) uint32_t raw;
        uint32_t q[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j / 4] |= (uint32_t)((int)rintf(u[j] * inverse) & 255) << (8 * (j % 4));
        *(raw *)p = raw{q[0], q[1]};
    } else *p = (int8_t)(int)rintf(u[0] * inverse);
}

// WAVES waves per row, V sets of N elements per lane: rows of up to 64 N V WAVES elements.  V = 0: rows of any length, read three times.
// A row that is no multiple of N ends in a set that reaches back; its first elements count once.
// KEEP: weights, and a gate that all rows share, are of the type of x and stay in registers from row to row, and a row's loads are
// requested while the one in front of it is worked on.
template <int TYPE, bool INT8, int WAVES, int V, int N, bool KEEP>
__global__ void __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) norm_block_kernel(const NormBlockParams p)
{
    typedef element<TYPE> E;
    constexpr int ROWS = WAVES == 1 ? 4 : 1, LANES = 64 * WAVES, SETS = V > 0 ? V : 1, KEPT = KEEP ? SETS : 1;
    __shared__ float part[2][WAVES];
    __shared__ uint32_t part_most[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = WAVES == 1 ? lane : (int)threadIdx.x;                // this thread's place among those of the row
    auto each = [&](auto &&f) {                                         // f(set, first element, elements of it that count already)
        if constexpr (V > 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int first = N * (at + LANES * v), d = min(first, p.dim - N);
                if (first < p.dim) f(v, d, first - d);
            }
        } else {
            for (int first = N * at; first < p.dim; first += N * LANES) {
                const int d = min(first, p.dim - N);
                f(0, d, first - d);
            }
        }
    };
    auto whole = [&](float v, int which) {
        v = group_sum<64>(v);
        if constexpr (WAVES > 1) {
            if (lane == 0) part[which][wave] = v;
            __syncthreads();
            v = part[which][0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) v += part[which][i];
        }
        return v;
    };
    const bool one_gate = p.gate && p.gate_every >= p.rows;
    Set<TYPE, N> kept_w[KEPT], kept_next[KEPT], kept_gate[KEPT];
    if constexpr (KEEP)
        each([&](int v, int d, int) {
            if (p.w) kept_w[v].load((const E *)p.w + d);
            kept_next[v].load((const E *)p.next_w + d);
            if (one_gate) kept_gate[v].load((const E *)p.gate + d);
        });
    Set<TYPE, N> xs[SETS], rs[SETS], next_x[KEPT], next_r[KEPT];
    auto request = [&](int64_t row, Set<TYPE, N> (&x)[KEPT], Set<TYPE, N> (&r)[KEPT]) {
        each([&](int v, int d, int) {
            x[v].load_once((const E *)p.x + row * p.sx + d);
            r[v].load_once((const E *)p.residual + row * p.sr + d);
        });
    };
    const int64_t step = (int64_t)gridDim.x * ROWS, mine = WAVES == 1 ? wave : 0;
    if constexpr (KEEP)
        if ((int64_t)blockIdx.x * ROWS + mine < p.rows) request((int64_t)blockIdx.x * ROWS + mine, next_x, next_r);
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < p.rows; base += step) {
        const int64_t row = base + mine;
        const bool live = row < p.rows;
        const E *const x = (const E *)p.x + row * p.sx, *const residual = (const E *)p.residual + row * p.sr;
        const int64_t gate_at = p.gate ? row / p.gate_every * p.sg : 0;
        if constexpr (KEEP) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                xs[v] = next_x[v];
                rs[v] = next_r[v];
            }
            if (row + step < p.rows) request(row + step, next_x, next_r);
        } else if (V > 0 && live)
            each([&](int v, int d, int) {
                xs[v].load_once(x + d);
                rs[v].load_once(residual + d);
            });
        float u[SETS][N];
        float first_r = 1.f, sum = 0.f;
        if (p.w) {
            if (live)
                each([&](int v, int d, int skip) {
                    if constexpr (V == 0) xs[v].load(x + d);
#pragma unroll
                    for (int j = 0; j < N; ++j) sum = j >= skip ? fmaf(xs[v][j], xs[v][j], sum) : sum;
                });
            first_r = rsqrtf(whole(sum, 0) / (float)p.dim + p.eps);
        }
        auto weigh = [&](const void *base, int64_t at, int wide, const Set<TYPE, N> (&kept)[KEPT], bool keeps, int v, float (&w)[N]) {
            if (KEEP && keeps)
#pragma unroll
                for (int j = 0; j < N; ++j) w[j] = kept[KEEP ? v : 0][j];
            else factors<TYPE, N>(base, at, wide, w);
        };
        auto total = [&](int v, int d, float (&t)[N]) {                 // t of a set
            if constexpr (V == 0) {
                xs[v].load(x + d);
                rs[v].load(residual + d);
            }
            float w[N];
#pragma unroll
            for (int j = 0; j < N; ++j) t[j] = xs[v][j];
            if (p.w) {
                weigh(p.w, d, p.w_wide, kept_w, true, v, w);
#pragma unroll
                for (int j = 0; j < N; ++j) t[j] = t[j] * first_r * w[j];
            }
            if (p.gate) {
                weigh(p.gate, gate_at + d, p.gate_wide, kept_gate, one_gate, v, w);
#pragma unroll
                for (int j = 0; j < N; ++j) t[j] *= w[j];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) t[j] = p.factor * rs[v][j] + t[j];
        };
        uint32_t most_bits = 0;      // of |u|, largest as integers: a NaN is larger than any value
        sum = 0.f;
        if (live)
            each([&](int v, int d, int skip) {
                float t[N], w[N];
                total(v, d, t);
                Set<TYPE, N>::store((E *)p.residual_out + row * p.sro + d, t, p.past);
#pragma unroll
                for (int j = 0; j < N; ++j) sum = j >= skip ? fmaf(t[j], t[j], sum) : sum;
                weigh(p.next_w, d, p.next_wide, kept_next, true, v, w);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    u[v][j] = t[j] * w[j];
                    if (INT8) most_bits = max(most_bits, __builtin_bit_cast(uint32_t, u[v][j]) & 0x7fffffffu);
                }
            });
        if constexpr (INT8) {
            most_bits = wave_max(most_bits);
            if constexpr (WAVES > 1)
                if (lane == 0) part_most[wave] = most_bits;
        }
        const float r = rsqrtf(whole(sum, 1) / (float)p.dim + p.eps);
        float inverse = 0.f;
        if constexpr (INT8) {
            if constexpr (WAVES > 1)
#pragma unroll
                for (int i = 0; i < WAVES; ++i) most_bits = max(most_bits, part_most[i]);
            const float most = __builtin_bit_cast(float, most_bits);
            inverse = most > kSmallest ? 127.f * (1.f / most) : 0.f;
            if (live && at == 0)
                p.scale[row * p.sscale] = most <= kSmallest ? 0.f : most < __builtin_inff() ? most * r / 127.f : __builtin_nanf("");
        }
        if (live)
            each([&](int v, int d, int) {
                if constexpr (V == 0) {
                    float t[N], w[N];
                    total(v, d, t);
                    factors<TYPE, N>(p.next_w, d, p.next_wide, w);
#pragma unroll
                    for (int j = 0; j < N; ++j) u[v][j] = t[j] * w[j];
                }
                if constexpr (INT8) store_i8<N>((int8_t *)p.out + row * p.so + d, u[v], inverse);
                else {
#pragma unroll
                    for (int j = 0; j < N; ++j) u[v][j] *= r;
                    Set<TYPE, N>::store((E *)p.out + row * p.so + d, u[v], p.past);
                }
            });
        if constexpr (WAVES > 1) __syncthreads();                        // part is written again
    }
}

template <int TYPE, bool INT8>
hipError_t run(const NormBlockParams &p, hipStream_t s)
{
    auto go = [&](auto waves, auto vectors, auto elements, auto keep) {
        constexpr int W = decltype(waves)::value, V = decltype(vectors)::value, N = decltype(elements)::value;
        constexpr bool KEEP = decltype(keep)::value;
        // (KEEP: as many workgroups as are on the card together, so that weights are read once for several rows)
        constexpr int64_t threads = W > 4 ? 64 * W : 256, most = KEEP ? 1024 : 1 << 21;
        static_assert(most * threads < (int64_t)1 << 32, "a launch has below 2^32 threads");
        const int64_t blocks = W == 1 ? (p.rows + 3) / 4 : p.rows;
        const uint32_t grid = (uint32_t)(blocks < most ? blocks : most);
        hipLaunchKernelGGL((norm_block_kernel<TYPE, INT8, W, V, N, KEEP>), dim3(grid), dim3(threads), 0, s, p);
        return hipGetLastError();
    };
    using std::integral_constant;
    typedef integral_constant<int, 0> zero;
    typedef integral_constant<int, 1> one;
    typedef integral_constant<int, 4> four;
    typedef integral_constant<int, 8> eight;
    typedef integral_constant<bool, false> no;
    typedef integral_constant<bool, true> yes;
    if (p.dim < 8) return go(four{}, zero{}, one{}, no{});
    // Four waves to a row but for many short ones and long ones.  Measured (us, 16 bits, a gate per channel; the other way in brackets):
    //   weights kept     32768 x 2560: 128 (173);  4096 x 2560: 19.0 (25.3);  64 x 2560: 3.9 (4.6);  8192 x 5120: 70 (77)
    //   a wave per row, nothing kept    4096 x 1024: 9.7 (11.0);  16384 x 300: 15.5 (18.9);  32768 x 1024: 56 (62)
    //   fp32, nothing kept               5703 x 1537: 32.1 (35.1)
    //   8 waves, nothing kept    8192 x 8192, a gate per token: 121 (4 waves 156, 16 waves 145);  4096 x 10000: 79 (81, 86)
    //   16 waves    5967 x 13906: 146 (8 waves 178, read three times 187);  64 x 16384: 6.1 (7.4, 15.8);  2048 x 20000: 80 (94, 109)
    if (p.dim <= 1024 && p.rows >= 1024) return go(one{}, integral_constant<int, 2>{}, eight{}, no{});
    if constexpr (TYPE != DT_F32)
        if (p.dim > 1024 && p.dim <= 6144 && !p.w_wide && !p.next_wide && !(p.gate && p.gate_every >= p.rows && p.gate_wide)) {
            if (p.dim <= 2048) return go(four{}, one{}, eight{}, yes{});
            if (p.dim <= 4096) return go(four{}, integral_constant<int, 2>{}, eight{}, yes{});
            return go(four{}, integral_constant<int, 3>{}, eight{}, yes{});
        }
    if (p.dim <= 2048) return go(four{}, one{}, eight{}, no{});
    if (p.dim <= 4096) return go(four{}, integral_constant<int, 2>{}, eight{}, no{});
    if (p.dim <= 6144) return go(four{}, integral_constant<int, 3>{}, eight{}, no{});
    if (p.dim <= 8192) return go(eight{}, integral_constant<int, 2>{}, eight{}, no{});
    if (p.dim <= 12288) return go(eight{}, integral_constant<int, 3>{}, eight{}, no{});
    if (p.dim <= 16384) return go(integral_constant<int, 16>{}, integral_constant<int, 2>{}, eight{}, no{});
    if constexpr (TYPE != DT_F32)                        // (no registers for it)
        if (p.dim <= 24576) return go(integral_constant<int, 16>{}, integral_constant<int, 3>{}, eight{}, no{});
    return go(four{}, zero{}, eight{}, no{});
}

template <int TYPE> hipError_t of_type(const NormBlockParams &p, hipStream_t s) { return p.int8 ? run<TYPE, true>(p, s) : run<TYPE, false>(p, s); }

}  // namespace

hipError_t launch_norm_block(const NormBlockParams &p, hipStream_t s)
{
    if (p.rows == 0) return hipSuccess;
    if (p.type == DT_F32) return of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? of_type<DT_BF16>(p, s) : of_type<DT_F16>(p, s);
}

}  // namespace ssd
