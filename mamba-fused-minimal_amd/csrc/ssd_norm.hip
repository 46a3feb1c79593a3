// Root-mean-square norm of rows, behind the addition of the residual or behind a gate, with an output in the type of x or in 8
// bits with a scale per row.
//
//   t = x + residual   or   t = x silu(z);   r = 1 / sqrt(mean(t^2) + eps);   u = t w
//   out = u r          or   q = rint(u (127 (1 / max|u|))), scale = max|u| r / 127
//
// r is common to a row, so it cancels in q: the row's largest and its sum of squares come from one pass, with the row in
// registers, and what is rounded to 8 bits does not depend on the rounding of r.  residual_out = t, rounded; the norm itself is
// that of the sum in 32 bits.  Everything in front of the rounding to 8 bits is rounded as the formulas in fp32 are, an operation at a
// time (a division by its definition, the exponential of the gate in full), so that q is theirs and not a neighbour's.  A row of zeros has
// q = 0 and scale = 0; a row with a NaN or an infinity, from t or from w, has a scale of NaN.
//
// HBM bound: one read, one write, two reductions over the row.  Where there are rows enough to fill the card a wave owns a row
// (no LDS, no barrier: only lane-to-lane moves), otherwise four waves share one.  In bf16 to 8 bits: 32768 rows of 2560 with a residual 95 to
// 101 us, 5.8 to 6.2 TB/s; 32768 gated rows of 5120 198 us, 4.2 TB/s (a division and a full exponential per element, two barriers a row);
// 64 gated rows of 5120 5.4 us, latency.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

constexpr float kSmallest = 1e-36f;      // 127 / max|u| stays finite above it; rows of nothing larger are zeros

__device__ __forceinline__ int quantized(float u, float inverse) { return (int)rintf(u * inverse); }

// N consecutive elements as fp32: 8, or 1 where rows are shorter than that
template <int TYPE, int N, bool ONCE = false> __device__ __forceinline__ void load(const element<TYPE> *p, float (&f)[N])
{
    typedef Wide<TYPE> W;
    if constexpr (N == 8) {
#pragma unroll
        for (int h = 0; h < 8 / W::n; ++h) {
            const auto v = ONCE ? W::load_once(p + h * W::n) : W::load(p + h * W::n);
#pragma unroll
            for (int j = 0; j < W::n; ++j) f[h * W::n + j] = to_f32<TYPE>(v.e[j]);
        }
    } else f[0] = to_f32<TYPE>(*p);
}
template <int TYPE, int N> __device__ __forceinline__ void store(element<TYPE> *p, const float (&f)[N])
{
    typedef Wide<TYPE> W;
    if constexpr (N == 8) {
#pragma unroll
        for (int h = 0; h < 8 / W::n; ++h) {
            typename W::Pack v;
#pragma unroll
            for (int j = 0; j < W::n; ++j) v.e[j] = from_f32<TYPE>(f[h * W::n + j]);
            W::store(p + h * W::n, v);
        }
    } else *p = from_f32<TYPE>(f[0]);
}
template <int N> __device__ __forceinline__ void store_i8(int8_t *p, const float (&u)[N], float inverse)
{
    if constexpr (N == 8) {
        typedef __attribute__((ext_vector_type(2), aligned(1))) uint32_t raw;
        uint32_t q[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j / 4] |= (uint32_t)(quantized(u[j], inverse) & 255) << (8 * (j % 4));
        *(raw *)p = raw{q[0], q[1]};
    } else *p = (int8_t)quantized(u[0], inverse);
}

// t of N elements.  ONCE: they are not read again, here or, as rows of activations, by what follows (32768 rows of 2560 with a
// residual: 101 us, 118 without the hint)
template <int TYPE, int MODE, bool INT8, int N, bool ONCE> __device__ __forceinline__ void inputs(const NormParams &p, int64_t row, int d, float (&t)[N])
{
    typedef element<TYPE> E;
    load<TYPE, N, ONCE>((const E *)p.x + row * p.sx + d, t);
    float o[N];
    if constexpr (MODE == 1) {
        load<TYPE, N, ONCE>((const E *)p.residual + row * p.sr + d, o);
#pragma unroll
        for (int j = 0; j < N; ++j) t[j] += o[j];
    }
    if constexpr (MODE == 2) {
        load<TYPE, N, ONCE>((const E *)p.z + row * p.sz + d, o);
#pragma unroll
        for (int j = 0; j < N; ++j) t[j] *= INT8 ? o[j] / (1.f + expf(-o[j])) : silu(o[j]);
    }
}

// WAVES waves per row, V sets of N elements per lane: rows of up to 64 N V WAVES elements, whose weights have the type WTYPE and a
// stride of one.  V = 0: rows of any length and weights of any kind, read twice.  MODE: 0 x alone, 1 with a residual, 2 with a gate.
// A row that is no multiple of N ends in a set that reaches back; its first elements count once.
template <int TYPE, int MODE, bool INT8, int WAVES, int V, int N, int WTYPE>
__global__ void __launch_bounds__(256) norm_kernel(const NormParams p)
{
    typedef element<TYPE> E;
    constexpr int ROWS = 4 / WAVES, LANES = 64 * WAVES;
    __shared__ float part[4];
    __shared__ uint32_t part_most[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = WAVES == 1 ? lane : (int)threadIdx.x;                // this thread's place among those of the row
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < p.rows; base += (int64_t)gridDim.x * ROWS) {
        const int64_t row = base + (WAVES == 1 ? wave : 0);
        const bool live = row < p.rows;
        float u[V > 0 ? V : 1][N];
        float sum = 0.f;
        uint32_t most_bits = 0;      // of |u|, largest as integers: a NaN is larger than any value
        auto weigh = [&](int d, float (&t)[N]) {
            float w[N];
            if constexpr (V > 0) load<WTYPE, N>((const element<WTYPE> *)p.w + d, w);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) w[j] = load_as_f32(p.w, (d + j) * p.sw, p.w_type);
#pragma unroll
            for (int j = 0; j < N; ++j) t[j] *= w[j];
        };
        auto take = [&](int first, float (&t)[N]) {
            const int d = min(first, p.dim - N), skip = first - d;
            inputs<TYPE, MODE, INT8, N, (V > 0)>(p, row, d, t);
            if constexpr (MODE == 1) store<TYPE, N>((E *)p.residual_out + row * p.sro + d, t);
#pragma unroll
            for (int j = 0; j < N; ++j) sum = j >= skip ? fmaf(t[j], t[j], sum) : sum;
            weigh(d, t);
#pragma unroll
            for (int j = 0; j < N; ++j) most_bits = max(most_bits, __builtin_bit_cast(uint32_t, t[j]) & 0x7fffffffu);
        };
        if constexpr (V > 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int first = N * (at + LANES * v);
                if (live && first < p.dim) take(first, u[v]);
            }
        } else if (live) {
            for (int first = N * at; first < p.dim; first += N * LANES) take(first, u[0]);
        }
        sum = group_sum<64>(sum);
        most_bits = group_max<64>(most_bits);
        if constexpr (WAVES > 1) {
            if (lane == 0) {
                part[wave] = sum;
                part_most[wave] = most_bits;
            }
            __syncthreads();
            sum = part[0] + part[1] + part[2] + part[3];
            most_bits = max(max(part_most[0], part_most[1]), max(part_most[2], part_most[3]));
            __syncthreads();
        }
        const float most = __builtin_bit_cast(float, most_bits);
        const float r = rsqrtf(sum / (float)p.dim + p.eps);
        const float inverse = most > kSmallest ? 127.f * (1.f / most) : 0.f;
        // (zeros whatever eps is: with none of it r is infinite)
        if (INT8 && live && at == 0)
            p.scale[row * p.sscale] = most <= kSmallest ? 0.f : most < __builtin_inff() ? most * r / 127.f : __builtin_nanf("");
        auto give = [&](int first, float (&t)[N]) {
            const int d = min(first, p.dim - N);
            if constexpr (INT8) store_i8<N>((int8_t *)p.out + row * p.so + d, t, inverse);
            else {
#pragma unroll
                for (int j = 0; j < N; ++j) t[j] *= r;
                store<TYPE, N>((E *)p.out + row * p.so + d, t);
            }
        };
        if constexpr (V > 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int first = N * (at + LANES * v);
                if (live && first < p.dim) give(first, u[v]);
            }
        } else if (live) {
            for (int first = N * at; first < p.dim; first += N * LANES) {
                inputs<TYPE, MODE, INT8, N, true>(p, row, min(first, p.dim - N), u[0]);
                weigh(min(first, p.dim - N), u[0]);
                give(first, u[0]);
            }
        }
    }
}

template <int TYPE, int MODE, bool INT8>
hipError_t run(const NormParams &p, hipStream_t s)
{
    auto go = [&](auto waves, auto vectors, auto elements, auto wtype) {
        constexpr int W = decltype(waves)::value, V = decltype(vectors)::value, N = decltype(elements)::value, T = decltype(wtype)::value;
        const int64_t blocks = (p.rows + 4 / W - 1) / (4 / W);
        const uint32_t grid = (uint32_t)(blocks < (1 << 22) ? blocks : 1 << 22);
        hipLaunchKernelGGL((norm_kernel<TYPE, MODE, INT8, W, V, N, T>), dim3(grid), dim3(256), 0, s, p);
        return hipGetLastError();
    };
    using std::integral_constant;
    typedef integral_constant<int, 0> zero;
    typedef integral_constant<int, 1> one;
    typedef integral_constant<int, 4> four;
    typedef integral_constant<int, 8> eight;
    if (p.dim < 8) return go(four{}, zero{}, one{}, zero{});
    auto of_weights = [&](auto wtype) {
        // A wave per row from 1024 rows on, a wave for each of the card's 1024 SIMDs, and as few registers as hold a row.  Measured (us, to 8
        // bits, with a residual / gated; the neighbour in brackets):
        //   a wave per row      512 x 1024: 6.8 / 5.7 (four waves 7.4 / 6.2);  2048 x 2560: 11.0 / 11.2 (11.5 / 11.3);  32768 x 2560: 95 / 106 (111 / 124)
        //   four waves         1024 x 2560: 7.5 / 7.0 (one 8.4 / 8.5);  512 x 2560: 7.1 / 6.3 (7.8 / 8.0)
        //   two sets to 1024  32768 x 1024: 42 / 47 (five 49 / 55)
        //   one to 2048        4096 x 2048, four waves: 13.7 / 13.4 (three sets 15.4 / 14.8)
        //   three to 6144     32768 x 5120: 211 / 201 (five 212 / 225)
        //   five to 10240      8192 x 10240: 95 / 100 (rows read twice 223 / 220)
        if (p.rows >= 1024) {
            if (p.dim <= 1024) return go(one{}, integral_constant<int, 2>{}, eight{}, wtype);
            if (p.dim <= 2560) return go(one{}, integral_constant<int, 5>{}, eight{}, wtype);
        }
        if (p.dim <= 2048) return go(four{}, one{}, eight{}, wtype);
        if (p.dim <= 6144) return go(four{}, integral_constant<int, 3>{}, eight{}, wtype);
        if (p.dim <= 10240) return go(four{}, integral_constant<int, 5>{}, eight{}, wtype);
        return go(four{}, zero{}, eight{}, wtype);
    };
    if (p.sw != 1 || (p.w_type != TYPE && p.w_type != DT_F32)) return go(four{}, zero{}, eight{}, zero{});
    if (p.w_type == DT_F32) return of_weights(integral_constant<int, DT_F32>{});
    return of_weights(integral_constant<int, TYPE>{});
}

template <int TYPE>
hipError_t of_type(const NormParams &p, hipStream_t s)
{
    if (p.residual) return p.int8 ? run<TYPE, 1, true>(p, s) : run<TYPE, 1, false>(p, s);
    if (p.z) return p.int8 ? run<TYPE, 2, true>(p, s) : run<TYPE, 2, false>(p, s);
    return p.int8 ? run<TYPE, 0, true>(p, s) : run<TYPE, 0, false>(p, s);
}

}  // namespace

hipError_t launch_norm(const NormParams &p, hipStream_t s)
{
    if (p.rows == 0) return hipSuccess;
    if (p.type == DT_F32) return of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? of_type<DT_BF16>(p, s) : of_type<DT_F16>(p, s);
}

}  // namespace ssd
