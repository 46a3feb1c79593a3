// Matrix product with weights in 4 bits and a scale (and a zero point) per group of weights of a channel:
//
//   out[m, n] = sum_g scale[n, g] sum_{k in g} a[m, k] (q[n, k] - zero[n, g])  (+ bias[n])
//
// Whole numbers q - zero of up to 8 bits are exact in bf16 and fp16, so products and a group's sums are those of the matrix
// instructions, in fp32; a group's sum is scaled in fp32, and the result is rounded once.  fp32 activations enter as three bf16 parts, which
// hold their 24 bits.  Two weights share a byte, the even one in its lower half.
//
// direct_kernel: any size and alignment: the waves of a workgroup share a (16 MT) x 16 tile by K and add their sums through LDS.
#include "ssd_decode.h"

namespace ssd {
namespace {

using namespace layer;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((aligned(1))) uint32_t any_u32;

// What a product's operands look like by the type of the activations
template <int TYPE> struct Operand {
    static constexpr int parts = 1;
    typedef bf16x8 Vec;
};
template <> struct Operand<DT_F16> {
    static constexpr int parts = 1;
    typedef f16x8 Vec;
};
template <> struct Operand<DT_F32> {
    static constexpr int parts = 3;
    typedef bf16x8 Vec;
};

__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}
__device__ __forceinline__ f32x4 product(f16x8 a, f16x8 b, f32x4 c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

// Eight weights less their zero point, in the order of their places
template <int TYPE> __device__ __forceinline__ typename Operand<TYPE>::Vec weights(uint32_t w, float zero)
{
    float f[8];
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = (float)((even >> (8 * j)) & 255u) - zero;
        f[2 * j + 1] = (float)((odd >> (8 * j)) & 255u) - zero;
    }
    if constexpr (TYPE == DT_F16) {
        f16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (_Float16)f[j];
        return v;
    } else {
        // (of at most 8 bits: the upper half of an fp32 holds all of them)
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = (__builtin_bit_cast(uint32_t, f[2 * j]) >> 16) | (__builtin_bit_cast(uint32_t, f[2 * j + 1]) & 0xffff0000u);
        return __builtin_bit_cast(bf16x8, v);
    }
}

// Eight activations as operands
template <int TYPE> struct Activations {
    typename Operand<TYPE>::Vec v[Operand<TYPE>::parts];
    // n of them are there, the others are zero
    __device__ __forceinline__ void load(const element<TYPE> *p, int n)
    {
        typedef element<TYPE> E;
        typedef Wide<TYPE> W;
        struct { E e[8]; } raw;
        if (n >= 8) {
#pragma unroll
            for (int h = 0; h < 8 / W::n; ++h) {
                const auto q = W::load(p + h * W::n);
#pragma unroll
                for (int j = 0; j < W::n; ++j) raw.e[h * W::n + j] = q.e[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) raw.e[j] = j < n ? p[j] : (E)0;
        }
        if constexpr (TYPE == DT_F32) {
            // three parts of 8 bits, cut off and so exact; an infinity stands in the first alone, a NaN in all
            u32x4 part[3];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int t = 0; t < 3; ++t) part[t][j] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float rest = raw.e[j];
                if (rest != rest) rest = __builtin_nanf("");
#pragma unroll
                for (int t = 0; t < 3; ++t) {
                    const uint32_t top = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
                    part[t][j / 2] |= j & 1 ? top : top >> 16;
                    const float less = rest - __builtin_bit_cast(float, top);
                    rest = __builtin_isinf(rest) ? 0.f : less;
                }
            }
#pragma unroll
            for (int t = 0; t < 3; ++t) v[t] = __builtin_bit_cast(bf16x8, part[t]);
        } else v[0] = __builtin_bit_cast(typename Operand<TYPE>::Vec, raw);
    }
};

template <int TYPE, int MT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) direct_kernel(const PackedParams p, int tiles_m)
{
    typedef element<TYPE> E;
    constexpr int PARTS = Operand<TYPE>::parts;
    __shared__ f32x4 sums[MT * WAVES * 64];
    // (known to be the same in all lanes: matrix instructions run whatever the execution mask)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int m0 = (int)(blockIdx.x % (uint32_t)tiles_m) * 16 * MT, n0 = (int)(blockIdx.x / (uint32_t)tiles_m) * 16;
    const int n = min(n0 + i, p.N - 1);
    const uint8_t *const w = p.w + (int64_t)n * p.sw_n;
    const E *a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = (const E *)p.a + (int64_t)min(m0 + 16 * t + i, p.M - 1) * p.sa_m;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int blocks = (p.K + 31) / 32, bytes = (p.K + 1) / 2;
    for (int c = wave; c < blocks; c += WAVES) {
        const int k = 32 * c + 8 * g, of = 32 * c / p.group;
        uint32_t q = 0;
        if (k / 2 + 4 <= bytes) q = *(const any_u32 *)(w + k / 2);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k / 2 + j < bytes) q |= (uint32_t)w[k / 2 + j] << (8 * j);
        const float scale = load_as_f32(p.scale, n * p.ss_n + of * p.ss_g, p.scale_type);
        const float zero = p.zero ? (float)p.zero[n * p.sz_n + of * p.sz_g] : 8.f;
        Activations<TYPE> av[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) av[t].load(a[t] + k, p.K - k);
        const auto wv = weights<TYPE>(q, zero);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = PARTS - 1; h >= 0; --h) sum = product(av[t].v[h], wv, sum);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][j] = fmaf(scale, sum[j], acc[t][j]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[(t * WAVES + wave) * 64 + lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += WAVES) {
        f32x4 sum = sums[t * WAVES * 64 + lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) sum += sums[(t * WAVES + k) * 64 + lane];
        const float bias = p.bias ? load_as_f32(p.bias, n * p.sbias, p.bias_type) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + 16 * t + 4 * g + j;
            if (m < p.M && n0 + i < p.N) store_from_f32(p.out, m * p.so_m + n, p.out_type, sum[j] + bias);
        }
    }
}

template <int TYPE, int MT, int WAVES> hipError_t run_direct(const PackedParams &p, hipStream_t s)
{
    const int64_t tm = (p.M + 16 * MT - 1) / (16 * MT), tn = (p.N + 15) / 16;
    if (tm * tn * 64 * WAVES > 0xffffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((direct_kernel<TYPE, MT, WAVES>), dim3((uint32_t)(tm * tn)), dim3(64 * WAVES), 0, s, p, (int)tm);
    return hipGetLastError();
}

template <int TYPE> hipError_t of_type(const PackedParams &p, int, hipStream_t s)
{
    return p.M <= 16 ? run_direct<TYPE, 1, 8>(p, s) : run_direct<TYPE, 4, 8>(p, s);
}

}  // namespace

hipError_t launch_matmul_packed(const PackedParams &p, int n_cu, hipStream_t s)
{
    if (p.M == 0 || p.N == 0) return hipSuccess;
    if (p.type == DT_F32) return of_type<DT_F32>(p, n_cu, s);
    return p.type == DT_BF16 ? of_type<DT_BF16>(p, n_cu, s) : of_type<DT_F16>(p, n_cu, s);
}

}  // namespace ssd
