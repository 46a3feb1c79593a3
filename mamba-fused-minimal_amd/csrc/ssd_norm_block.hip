// What stands between two blocks: the norm behind a block, its gate, the residual with its scale, and the next block's norm.
//
//   n = x w / sqrt(mean(x^2) + eps)   (n = x without w);   t = factor residual + gate n;   r = 1 / sqrt(mean(t^2) + eps);   u = t next_w
//   out = u r,   or in 8 bits  q = rint(u (127 (1 / max|u|))), scale = max|u| r / 127;   residual_out = t, rounded
//
// The second norm is that of t in 32 bits, and so are its 8 bits: r is common to a row and cancels in them.  A row of zeros has q = 0
// and scale = 0, a row with a NaN or an infinity in u a scale of NaN.
//
// HBM bound: x and the residual are read once and t and out written once, with the row in registers between its two sums, the second of which
// depends on the first.  Where there are rows enough to fill the card a wave owns a row (lane-to-lane moves only), otherwise four waves
// share one.  Rows too long for the registers are read three times, from the caches as a rule.
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
    __device__ __forceinline__ static void store(E *p, const float (&f)[N])
    {
        if constexpr (N == 8) {
#pragma unroll
            for (int h = 0; h < 8 / W::n; ++h) {
                typename W::Pack q;
#pragma unroll
                for (int j = 0; j < W::n; ++j) q.e[j] = from_f32<TYPE>(f[h * W::n + j]);
                W::store(p + h * W::n, q);
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
template <int TYPE, bool INT8, int WAVES, int V, int N>
__global__ void __launch_bounds__(256) norm_block_kernel(const NormBlockParams p)
{
    typedef element<TYPE> E;
    constexpr int ROWS = 4 / WAVES, LANES = 64 * WAVES;
    __shared__ float part[2][4];
    __shared__ uint32_t part_most[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = WAVES == 1 ? lane : (int)threadIdx.x;                // this thread's place among those of the row
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < p.rows; base += (int64_t)gridDim.x * ROWS) {
        const int64_t row = base + (WAVES == 1 ? wave : 0);
        const bool live = row < p.rows;
        const E *const x = (const E *)p.x + row * p.sx, *const residual = (const E *)p.residual + row * p.sr;
        const int64_t gate_at = p.gate ? row / p.gate_every * p.sg : 0;
        auto whole = [&](float v, int which) {
            v = group_sum<64>(v);
            if constexpr (WAVES > 1) {
                if (lane == 0) part[which][wave] = v;
                __syncthreads();
                v = (part[which][0] + part[which][1]) + (part[which][2] + part[which][3]);
            }
            return v;
        };
        auto each = [&](auto &&f) {                                     // f(set, first element, elements of it that count already)
            if (!live) return;
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
        Set<TYPE, N> xs[V > 0 ? V : 1], rs[V > 0 ? V : 1];
        float u[V > 0 ? V : 1][N];
        float first_r = 1.f, sum = 0.f;
        each([&](int v, int d, int) {
            if constexpr (V > 0) {
                xs[v].load_once(x + d);
                rs[v].load_once(residual + d);
            }
        });
        if (p.w) {
            each([&](int v, int d, int skip) {
                if constexpr (V == 0) xs[v].load(x + d);
#pragma unroll
                for (int j = 0; j < N; ++j) sum = j >= skip ? fmaf(xs[v][j], xs[v][j], sum) : sum;
            });
            first_r = rsqrtf(whole(sum, 0) / (float)p.dim + p.eps);
        }
        auto total = [&](int v, int d, float (&t)[N]) {                 // t of a set
            if constexpr (V == 0) {
                xs[v].load(x + d);
                rs[v].load(residual + d);
            }
            float w[N], g[N];
            if (p.w) factors<TYPE, N>(p.w, d, p.w_wide, w);
            if (p.gate) factors<TYPE, N>(p.gate, gate_at + d, p.gate_wide, g);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float n = xs[v][j];
                if (p.w) n = n * first_r * w[j];
                if (p.gate) n *= g[j];
                t[j] = p.factor * rs[v][j] + n;
            }
        };
        uint32_t most_bits = 0;      // of |u|, largest as integers: a NaN is larger than any value
        sum = 0.f;
        each([&](int v, int d, int skip) {
            float t[N], w[N];
            total(v, d, t);
            Set<TYPE, N>::store((E *)p.residual_out + row * p.sro + d, t);
#pragma unroll
            for (int j = 0; j < N; ++j) sum = j >= skip ? fmaf(t[j], t[j], sum) : sum;
            factors<TYPE, N>(p.next_w, d, p.next_wide, w);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                u[v][j] = t[j] * w[j];
                if (INT8) most_bits = max(most_bits, __builtin_bit_cast(uint32_t, u[v][j]) & 0x7fffffffu);
            }
        });
        if constexpr (INT8) {
            most_bits = group_max<64>(most_bits);
            if constexpr (WAVES > 1)
                if (lane == 0) part_most[wave] = most_bits;
        }
        const float r = rsqrtf(whole(sum, 1) / (float)p.dim + p.eps);
        float inverse = 0.f;
        if constexpr (INT8) {
            if constexpr (WAVES > 1) most_bits = max(max(part_most[0], part_most[1]), max(part_most[2], part_most[3]));
            const float most = __builtin_bit_cast(float, most_bits);
            inverse = most > kSmallest ? 127.f * (1.f / most) : 0.f;
            if (live && at == 0)
                p.scale[row * p.sscale] = most <= kSmallest ? 0.f : most < __builtin_inff() ? most * r / 127.f : __builtin_nanf("");
        }
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
                Set<TYPE, N>::store((E *)p.out + row * p.so + d, u[v]);
            }
        });
        if constexpr (WAVES > 1) __syncthreads();                        // part is written again
    }
}

template <int TYPE, bool INT8>
hipError_t run(const NormBlockParams &p, hipStream_t s)
{
    auto go = [&](auto waves, auto vectors, auto elements) {
        constexpr int W = decltype(waves)::value, V = decltype(vectors)::value, N = decltype(elements)::value;
        const int64_t blocks = (p.rows + 4 / W - 1) / (4 / W);
        const uint32_t grid = (uint32_t)(blocks < (1 << 22) ? blocks : 1 << 22);
        hipLaunchKernelGGL((norm_block_kernel<TYPE, INT8, W, V, N>), dim3(grid), dim3(256), 0, s, p);
        return hipGetLastError();
    };
    using std::integral_constant;
    typedef integral_constant<int, 1> one;
    typedef integral_constant<int, 4> four;
    typedef integral_constant<int, 8> eight;
    if (p.dim < 8) return go(four{}, integral_constant<int, 0>{}, one{});
    if (p.rows >= 1024) {
        if (p.dim <= 1024) return go(one{}, integral_constant<int, 2>{}, eight{});
        if (p.dim <= 2560) return go(one{}, integral_constant<int, 5>{}, eight{});
    }
    if (p.dim <= 2048) return go(four{}, one{}, eight{});
    if (p.dim <= 6144) return go(four{}, integral_constant<int, 3>{}, eight{});
    if (p.dim <= 10240) return go(four{}, integral_constant<int, 5>{}, eight{});
    return go(four{}, integral_constant<int, 0>{}, eight{});
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
