// Matrix product with weights in 4 bits and a scale (and a zero point) per group of weights of a channel:
//
//   out[m, n] = sum_g scale[n, g] sum_{k in g} a[m, k] (q[n, k] - zero[n, g])  (+ bias[n])
//
// Whole numbers q - zero of up to 8 bits are exact in bf16 and fp16, so products and a group's sums are those of the matrix
// instructions, in fp32; a group's sum is scaled in fp32, and the result is rounded once.  fp32 activations enter as three bf16 parts, which
// hold their 24 bits.  Two weights share a byte, the even one in its lower half.
//
// Few tokens are HBM bound (the weights, half a byte each), many are bound by the matrix instructions, and what lies between by the wait for the first
// bytes and by the instructions of one wave.
//
// direct_kernel: any size and alignment, up to 16 tokens always.  The waves of a workgroup share a (16 MT) x (16 NT) tile by K, each with wide requests for its
// own weights and activations, and add their sums through LDS.  Measured: 1 x 2560 x 10576 bf16 (13.5 MB) in 7.3 us; 7 x 1543 x 777 fp16 in 6.0 us,
// both of which wait for memory two or three times over and need 2.5 us for being launched.
// tile_kernel: packed weights go straight into LDS several steps ahead and are unpacked there once for all tokens of a tile; the products of a group
// are scaled in registers.  Tiles of 64 x 64 for few tokens, activations by way of LDS too, K shared out where tiles are few.  Tiles of 256 x 128 and 256 x 64
// for many: LDS would have to give each wave activations and weights, which takes longer than the products (139 us for the size below), so activations are
// laid out as operands by a launch in front and come straight into the registers of the one wave that multiplies them, a step ahead.
// Measured: 2048 x 2560 x 10576 bf16 in 130 to 140 us, 790 to 850 TFLOP/s (6 to 7 of them that launch; 664 tiles are three rounds of 256, of which the last is
// 60 % full; a fifth of the time goes for LDS, which gives eight waves the same weights, a seventh for the unpacking); 512 x 8192 x 8192 in 82 us,
// 840 TFLOP/s; 64 x 5120 x 2560 with groups of 64 and zero points in 16.4 us (3 until the first step, 8 steps of 0.57, the joining launch 4).
#include "ssd_decode.h"

#include <cmath>

namespace ssd {
namespace {

using namespace layer;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((aligned(1))) uint32_t any_u32;
typedef __attribute__((ext_vector_type(4), aligned(1))) uint32_t any_u32x4;

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
    uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
#if defined(__HIP_DEVICE_COMPILE__)
    // (bytes are converted as they lie; taken apart again into fields of four bits they would cost an instruction each)
    asm("" : "+v"(even), "+v"(odd));
#endif
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
            v[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[2 * j + 1]), __builtin_bit_cast(uint32_t, f[2 * j]), 0x07060302u);
        return __builtin_bit_cast(bf16x8, v);
    }
}

// Eight activations, and as operands
template <int TYPE> struct Activations {
    typedef typename Operand<TYPE>::Vec Vec;
    struct { element<TYPE> e[8]; } raw;
    __device__ __forceinline__ void load(const element<TYPE> *p)
    {
        typedef Wide<TYPE> W;
#pragma unroll
        for (int h = 0; h < 8 / W::n; ++h) {
            const auto q = W::load(p + h * W::n);
#pragma unroll
            for (int j = 0; j < W::n; ++j) raw.e[h * W::n + j] = q.e[j];
        }
    }
    // n of them are there, the others are zero
    __device__ __forceinline__ void load(const element<TYPE> *p, int n)
    {
        if (n >= 8) load(p);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) raw.e[j] = j < n ? p[j] : (element<TYPE>)0;
    }
    __device__ __forceinline__ void operands(Vec (&v)[Operand<TYPE>::parts]) const
    {
        if constexpr (TYPE == DT_F32) {
            // three parts of 8 bits, cut off and so exact; an infinity stands in the first alone, a NaN in all
            u32x4 part[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t top[3][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float rest = raw.e[2 * j + h];
                    rest = rest == rest ? rest : __builtin_nanf("");
#pragma unroll
                    for (int t = 0; t < 3; ++t) {
                        top[t][h] = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
                        const float less = rest - __builtin_bit_cast(float, top[t][h]);
                        rest = __builtin_isinf(rest) ? 0.f : less;
                    }
                }
#pragma unroll
                for (int t = 0; t < 3; ++t) part[t][j] = __builtin_amdgcn_perm(top[t][1], top[t][0], 0x07060302u);
            }
#pragma unroll
            for (int t = 0; t < 3; ++t) v[t] = __builtin_bit_cast(Vec, part[t]);
        } else v[0] = __builtin_bit_cast(Vec, raw);
    }
};

// Scales of any of the three types without a branch, which would end what the compiler can arrange: the lower and the upper half of one
// (the same half twice where there are only 16 bits), and the number that they are
struct ScaleType {
    int size, upper;
    uint32_t as_f32, as_bf16, as_f16;      // masks
    __device__ __forceinline__ explicit ScaleType(int type)
        : size(type == DT_F32 ? 4 : 2), upper(type == DT_F32 ? 2 : 0), as_f32(type == DT_F32 ? ~0u : 0u), as_bf16(type == DT_BF16 ? ~0u : 0u),
          as_f16(type == DT_F16 ? ~0u : 0u) {}
    struct Raw { uint32_t lo, hi; };
    __device__ __forceinline__ Raw load(const void *base, int64_t at) const
    {
        const char *const p = (const char *)base + at * size;
        return Raw{*(const uint16_t *)p, *(const uint16_t *)(p + upper)};
    }
    __device__ __forceinline__ float value(Raw r) const
    {
        const float h = (float)__builtin_bit_cast(_Float16, (uint16_t)r.lo);
        return __builtin_bit_cast(float, ((r.lo | r.hi << 16) & as_f32) | (r.lo << 16 & as_bf16) | (__builtin_bit_cast(uint32_t, h) & as_f16));
    }
};

// d[i] of lane group g <-> d[g] of lane group i (groups of 16 lanes)
__device__ __forceinline__ void turn(uint32_t (&d)[4])
{
#if defined(__HIP_DEVICE_COMPILE__)
    auto halves = [&](int i, int j) {
        const auto v = __builtin_amdgcn_permlane32_swap(d[i], d[j], false, false);
        d[i] = v[0];
        d[j] = v[1];
    };
    auto rows = [&](int i, int j) {
        const auto v = __builtin_amdgcn_permlane16_swap(d[i], d[j], false, false);
        d[i] = v[0];
        d[j] = v[1];
    };
    halves(0, 2);
    halves(1, 3);
    rows(0, 1);
    rows(2, 3);
#endif
}

// 128 weights of a channel are a step: a lane group has 32 of them, one request of 16 bytes, and takes from the other groups what belongs to the
// blocks of 32 that the products go through.  A wave has steps that follow each other, U of them requested together.  A workgroup has 16 NT channels.
// FLUSH: blocks that make a sum in front of its scale.  WIDE: scales of 32 bits.
template <int TYPE, int MT, int NT, int WAVES, int U, int FLUSH, bool WIDE>
__global__ void __launch_bounds__(64 * WAVES) direct_kernel(const PackedParams p, int tiles_m, uint32_t first_tile)
{
    typedef element<TYPE> E;
    typedef typename Operand<TYPE>::Vec Vec;
    constexpr int PARTS = Operand<TYPE>::parts, SUMS = 4 / FLUSH;
    __shared__ f32x4 sums[MT * NT * WAVES * 64];
    // (known to be the same in all lanes: matrix instructions run whatever the execution mask)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const uint32_t tile = first_tile + blockIdx.x;
    const int m0 = (int)(tile % (uint32_t)tiles_m) * 16 * MT, n0 = (int)(tile / (uint32_t)tiles_m) * 16 * NT;
    typedef std::conditional_t<WIDE, float, uint16_t> S;
    const bool zeros = p.zero != nullptr;
    const uint8_t *w[NT], *zero_at[NT];
    const S *scale_at[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const int n = min(n0 + 16 * c + i, p.N - 1);
        w[c] = p.w + (int64_t)n * p.sw_n;
        scale_at[c] = (const S *)p.scale + n * p.ss_n;
        zero_at[c] = zeros ? p.zero + n * p.sz_n : nullptr;
    }
    const E *a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = (const E *)p.a + (int64_t)min(m0 + 16 * t + i, p.M - 1) * p.sa_m;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int c = 0; c < NT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto scale_of = [&](S raw) {
        if constexpr (WIDE) return raw;
        else return p.scale_type == DT_BF16 ? bf16_bits_to_f32(raw) : (float)__builtin_bit_cast(_Float16, raw);
    };
    // a step's scales lie beside each other, and so do its zero points: a request for all of them
    const bool beside = p.group == 32 * FLUSH && p.ss_g == 1 && (!zeros || p.sz_g == 1);
    typedef __attribute__((ext_vector_type(SUMS), aligned(sizeof(S)))) S any_scales;
    typedef __attribute__((ext_vector_type(SUMS), aligned(1))) uint8_t any_zeros;
    const int whole = p.K / 128, per = (whole + WAVES - 1) / WAVES, last = min(whole, (wave + 1) * per);
    for (int first = wave * per; first < last; first += U) {
        uint32_t wv[U][NT][4], zv[U][NT][SUMS];
        S sv[U][NT][SUMS];
        Activations<TYPE> av[U][4][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u > 0 && first + u >= last) break;
            const int k = (first + u) * 128;
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const any_u32x4 v = *(const any_u32x4 *)(w[c] + k / 2 + g * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) wv[u][c][j] = v[j];
            }
            if (SUMS > 1 && beside) {
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    const any_scales v = *(const any_scales *)(scale_at[c] + k / (32 * FLUSH));
                    any_zeros z = {};
                    if (zeros) z = *(const any_zeros *)(zero_at[c] + k / (32 * FLUSH));
#pragma unroll
                    for (int t = 0; t < SUMS; ++t) {
                        sv[u][c][t] = v[t];
                        zv[u][c][t] = z[t];
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < SUMS; ++t) {
                    const int of = (k + 32 * FLUSH * t) / p.group;
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        sv[u][c][t] = scale_at[c][of * p.ss_g];
                        if (zeros) zv[u][c][t] = zero_at[c][of * p.sz_g];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
                // (rows that are not there need not be asked for: their results are left out)
                if (m0 + 16 * t + i < p.M)
#pragma unroll
                    for (int j = 0; j < 4; ++j) av[u][j][t].load(a[t] + k + 32 * j + 8 * g);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u == 0 || first + u < last) {
#pragma unroll
                for (int c = 0; c < NT; ++c) turn(wv[u][c]);
                f32x4 sum[MT][NT];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    Vec x[MT][PARTS];
#pragma unroll
                    for (int t = 0; t < MT; ++t) av[u][j][t].operands(x[t]);
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        const Vec q = weights<TYPE>(wv[u][c][j], zeros ? (float)zv[u][c][j / FLUSH] : 8.f);
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            if (j % FLUSH == 0) sum[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int h = PARTS - 1; h >= 0; --h) sum[t][c] = product(x[t][h], q, sum[t][c]);
                        }
                        if (j % FLUSH == FLUSH - 1) {
                            const float scale = scale_of(sv[u][c][j / FLUSH]);
#pragma unroll
                            for (int t = 0; t < MT; ++t)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[t][c][e] = fmaf(scale, sum[t][c][e], acc[t][c][e]);
                        }
                    }
                }
            }
    }
    // what is left of K, block by block
    const int blocks = (p.K + 31) / 32, bytes = (p.K + 1) / 2;
    for (int b = whole * 4 + wave; b < blocks; b += WAVES) {
        const int k = 32 * b + 8 * g, of = 32 * b / p.group;
        Vec x[MT][PARTS];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            Activations<TYPE> av;
            av.load(a[t] + k, p.K - k);
            av.operands(x[t]);
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            uint32_t q = 0;
            if (k / 2 + 4 <= bytes) q = *(const any_u32 *)(w[c] + k / 2);
            else
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k / 2 + j < bytes) q |= (uint32_t)w[c][k / 2 + j] << (8 * j);
            const float scale = scale_of(scale_at[c][of * p.ss_g]), zero = zeros ? (float)zero_at[c][of * p.sz_g] : 8.f;
            const Vec wv = weights<TYPE>(q, zero);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = PARTS - 1; h >= 0; --h) sum = product(x[t][h], wv, sum);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][c][j] = fmaf(scale, sum[j], acc[t][c][j]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int c = 0; c < NT; ++c) sums[((t * NT + c) * WAVES + wave) * 64 + lane] = acc[t][c];
    __syncthreads();
    for (int f = wave; f < MT * NT; f += WAVES) {
        const int t = f / NT, n = n0 + 16 * (f % NT) + i;
        f32x4 sum = sums[f * WAVES * 64 + lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) sum += sums[(f * WAVES + k) * 64 + lane];
        if (n >= p.N) continue;
        const float bias = p.bias ? load_as_f32(p.bias, n * p.sbias, p.bias_type) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + 16 * t + 4 * g + j;
            if (m < p.M) store_from_f32(p.out, m * p.so_m + n, p.out_type, sum[j] + bias);
        }
    }
}

// eight consecutive results of a row, `left` of them in it
template <int TYPE> __device__ __forceinline__ void store8(char *at, int left, const float (&v)[8])
{
    typedef Wide<TYPE> W;
    typedef element<TYPE> E;
    E *const o = (E *)at;
    if (left >= 8) {
#pragma unroll
        for (int k = 0; k < 8 / W::n; ++k) {
            typename W::Pack q;
#pragma unroll
            for (int e = 0; e < W::n; ++e) q.e[e] = from_f32<TYPE>(v[k * W::n + e]);
            W::store(o + k * W::n, q);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) o[e] = from_f32<TYPE>(v[e]);
    }
}

// ---- many tokens ---------------------------------------------------------------------------------------------------

typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int kStep = 64;                 // weights of a channel per step
constexpr int kTable = 24;                // groups whose scales and zero points are in LDS
constexpr int kNowhere = 0x7ffffff0;      // an offset behind every descriptor's end: reads as zero
constexpr int kLongest = 1 << 20;         // K of the tile kernel: offsets inside a tile in 31 bits, with three parts too

__device__ __forceinline__ f32x16 product(bf16x8 a, bf16x8 b, f32x16 c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}
__device__ __forceinline__ f32x16 product(f16x8 a, f16x8 b, f32x16 c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

// s_waitcnt: at most n vector-memory operations outstanding
__device__ __forceinline__ constexpr int vm_only(int n) { return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14); }

// 1 KB (64 lanes x 16 bytes) from memory into LDS at `to`, without a register between: the compiler does not know of the write, so
// the kernel waits by count
__device__ __forceinline__ void into_lds(__amdgpu_buffer_rsrc_t from, int offset, int more, uint32_t to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    // (the same in all lanes, which the compiler does not always see)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(from),
                 "s"(__builtin_amdgcn_readfirstlane(more)) : "memory");
#endif
}

// What of a product a launch does: operands as the tile kernel walks them
struct Walk {
    const void *a;        // rows of parts x padded columns, at multiples of 16 bytes; or blocks of 32 of them, as lay_blocks_kernel leaves them
    const uint8_t *w;     // rows of w_bytes, at multiples of four
    int64_t sa_m, sw_n;   // elements, bytes
    int parts, padded;    // fp32 activations as three parts beside each other, of `padded` columns each
    int w_bytes;
    int steps;            // of kStep columns, per part
    int splits, per;      // workgroups that share a tile by steps, and the steps of each
    float *sums;          // [splits][M][N], or null: the result is written
};

// Where a step stands, kept up from step to step with little scalar arithmetic, of which a wave's instructions would otherwise mostly be: its
// weights begin at k, in group `of`, which has `left` more from there on
template <int PARTS> struct Cursor {
    int k, of, left, until;      // until: steps to the end of the part
    __device__ __forceinline__ Cursor(const PackedParams &p, const Walk &w, int step)
    {
        const int part = step / w.steps;
        k = (step - part * w.steps) * kStep;
        until = (part + 1) * w.steps - step;
        of = k / p.group;
        left = (of + 1) * p.group - k;
    }
    // the group of a weight 0 .. 63 behind k
    __device__ __forceinline__ int group_of(const PackedParams &p, int more) const
    {
        return min(of + (more >= left) + (more >= left + p.group), p.groups - 1);
    }
    template <int FLUSH> __device__ __forceinline__ void next(const PackedParams &p, const Walk &w)
    {
        k += kStep;
        left -= kStep;
#pragma unroll
        for (int i = 0; i < (FLUSH == 1 ? 2 : 1); ++i) {      // (groups of 32 end twice)
            const bool over = left <= 0;
            of += over;
            left += over ? p.group : 0;
        }
        if (PARTS > 1 && --until == 0) {
            until = w.steps;
            k = of = 0;
            left = p.group;
        }
    }
    // steps from this one on whose groups are below `end`
    __device__ __forceinline__ int steps_below(const PackedParams &p, int end) const
    {
        const int64_t all = ((int64_t)end * p.group - k) / kStep;
        const int n = end >= p.groups ? 0x7fffffff : (int)(all < 0x7fffffff ? all : 0x7fffffff);
        return PARTS > 1 ? min(n, until) : n;
    }
};

// whether two workgroups of eight waves find registers on a compute unit: one then loads, unpacks and stores while the other one multiplies (164 -> 137 us
// for 2048 x 10576 x 2560 in tiles of 256 x 64)
constexpr bool two_to_a_unit(int type, int tn, int flush) { return type != DT_F32 && tn == 2 && flush > 1; }

// TM x TN products of 32 x 32 to a wave, WM x WN waves, RING steps of operands in LDS.  DIRECT: activations are laid out as operands and do not go through
// LDS.  FLUSH: of 32 weights, how many such blocks make a sum in front of its scale: 4 where groups are of whole pairs of steps, 2 of whole steps, 1 otherwise.
// HALVES: twice as many waves, each half of them with its half of the steps.
template <int TYPE, int WM, int WN, int TM, int TN, int RING, int FLUSH, int HALVES, bool DIRECT>
__global__ void __launch_bounds__(64 * WM * WN * HALVES, DIRECT && two_to_a_unit(TYPE, TN, FLUSH) ? 4 : 2)
tile_kernel(const PackedParams p, const Walk walk, int tiles_m, int tiles_n)
{
    typedef typename Operand<TYPE>::Vec Vec;
    constexpr int PARTS = Operand<TYPE>::parts, THREADS = 64 * WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN, A_STAGE = DIRECT ? 0 : BM * 128, W_STAGE = BN * 128;
    constexpr int AHEAD = TM * TN == 4 || DIRECT ? 1 : 3;                             // quarters of a step whose operands are read from LDS in front of their products
    constexpr int LOADS = DIRECT ? 4 * TM : BM / 8 / (WM * WN), WORDS = BN * 8 / THREADS;      // of 1 KB of activations in a step, per wave; of eight weights, per thread
    static_assert(LOADS % 2 == 0, "a wave's rows begin at multiples of 16");
    constexpr int RAW_STAGE = BN * 32, RAW_LOADS = RAW_STAGE / 1024;
    // in LDS: RING steps of activations, two of weights, RING of weights as they come, scales and zero points of kTable groups
    constexpr int W_AT = RING * A_STAGE, RAW_AT = W_AT + 2 * W_STAGE, SCALE_AT = RAW_AT + RING * RAW_STAGE, ZERO_AT = SCALE_AT + kTable * BN * 4, HALF = ZERO_AT + kTable * BN;
    static_assert(HALVES == 1 || (PARTS == 1 && TM == 1), "halves are of one part, and their sums meet once");
    extern __shared__ __attribute__((aligned(16))) char all_lds[];
    const int lane = threadIdx.x & 63, half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    const int tid = (int)threadIdx.x - half * THREADS, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char *const lds = all_lds + half * HALF;
    const int wm = wave % WM, wn = wave / WM;
    // XCDs get workgroups in turn: each gets a contiguous part of the tiles, columns of eight tiles of tokens
    const int tiles = tiles_m * tiles_n, id = (int)blockIdx.x % tiles, split = (int)blockIdx.x / tiles, share = tiles / 8;
    const int t = id < share * 8 ? id % 8 * share + id / 8 : id;
    const int band = t / (8 * tiles_n), high = min(8, tiles_m - 8 * band), in = t - band * 8 * tiles_n;
    const int m0 = (8 * band + in % high) * BM, n0 = in / high * BN;

    const int64_t row_bytes = walk.sa_m * 2;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
        (void *)((const char *)walk.a + m0 * row_bytes), 0,
        (int)(DIRECT ? (min(BM, p.M - m0) + 31) / 32 * 32 * row_bytes : (min(BM, p.M - m0) - 1) * row_bytes + (int64_t)walk.parts * walk.padded * 2), 0x00020000);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(walk.w + n0 * walk.sw_n), 0, (int)((min(BN, p.N - n0) - 1) * walk.sw_n + walk.w_bytes), 0x00020000);
    // Rows of 128 bytes: 16-byte unit u of row r lies at place u ^ (r / 2 % 8), so 16 lanes that read the same unit of 16 rows touch all 64
    // banks once.  A load fills 8 rows.
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    int off[LOADS];
    if constexpr (!DIRECT)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int r = (wave * LOADS + j) * 8 + (lane >> 3);
            off[j] = m0 + r < p.M ? (int)(r * row_bytes) + (((lane & 7) ^ (lane >> 4) ^ (j % 2 * 4)) * 16) : kNowhere;
        }
    // steps of this workgroup, or of a half of it: the second half's, where they end early, go on with activations of zero
    const int begin = split * walk.per, first = begin + half * (walk.per / 2), steps = min(HALVES == 1 ? walk.per : walk.per / 2, walk.parts * walk.steps - begin);
    // A step's activations, LOADS requests a wave, and its weights as they come, one (of more waves than pieces two ask for the same).  What lies
    // behind a row's last column is zero; the number of requests is the same in every step, behind the last one too.
    int a_at = first * (kStep * 2), a_rest = walk.padded - first * kStep, a_until = 0;      // bytes into a row; columns of the part from there on
    if (PARTS > 1) {
        const int part = first / walk.steps, k = (first - part * walk.steps) * kStep;
        a_at = (part * walk.padded + k) * 2;
        a_rest = walk.padded - k;
        a_until = (part + 1) * walk.steps - first;
    }
    auto request = [&](uint32_t to) {
        if constexpr (DIRECT) return;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int u = (lane & 7) ^ (lane >> 4) ^ (j % 2 * 4);
            into_lds(ra, 8 * u < a_rest ? off[j] : kNowhere, a_at, base + to + (wave * LOADS + j) * 1024);
        }
        a_at += kStep * 2;
        a_rest -= kStep;
        if (PARTS > 1 && --a_until == 0) {
            a_until = walk.steps;
            a_at += (walk.padded - walk.steps * kStep) * 2;
            a_rest = walk.padded;
        }
    };
    // (behind a row's last byte lie the next row's: weights that meet activations of zero)
    const int raw_row = wave % RAW_LOADS * 32 + (lane >> 1), raw_off = n0 + raw_row < p.N ? (int)(raw_row * walk.sw_n) + (lane & 1) * 16 : kNowhere;
    int raw_at = (first % walk.steps) * (kStep / 2), raw_until = walk.steps - first % walk.steps;
    auto request_raw = [&](uint32_t to) {
        into_lds(rw, raw_off, raw_at, base + to + wave % RAW_LOADS * 1024);
        raw_at += kStep / 2;
        if (PARTS > 1 && --raw_until == 0) {
            raw_until = walk.steps;
            raw_at = 0;
        }
    };
    // scales and zero points of the groups from `of` on, BATCH of a thread's requested together; called between barriers
    constexpr int ENTRIES = kTable * BN / THREADS;
    static_assert(kTable * BN % THREADS == 0, "every thread has as many entries");
    const ScaleType scale_type(p.scale_type);
    auto tables = [&](int of, bool scales, bool zeros, auto batch) {
        constexpr int BATCH = decltype(batch)::value;
#pragma unroll 1
        for (int first = 0; first < ENTRIES; first += BATCH) {
            ScaleType::Raw raw[BATCH];
            uint8_t zero[BATCH];
            int to[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int i = (first + e) * THREADS + tid, n = i / kTable, g = i - n * kTable, at = min(of + g, p.groups - 1);
                const int64_t row = min(n0 + n, p.N - 1);
                to[e] = g * BN + n;
                if (scales) raw[e] = scale_type.load(p.scale, row * p.ss_n + at * p.ss_g);
                if (zeros) zero[e] = p.zero[row * p.sz_n + at * p.sz_g];
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                if (scales) ((float *)(lds + SCALE_AT))[to[e]] = scale_type.value(raw[e]);
                if (zeros) ((uint8_t *)(lds + ZERO_AT))[to[e]] = zero[e];
            }
        }
    };
    // weights: a thread's 8 WORDS of a row
    const int wr = tid / (8 / WORDS), wk = tid % (8 / WORDS) * 8 * WORDS;
    const bool zeros = p.zero != nullptr;
    int scale_base, zero_base;                                           // first groups of the tables
    struct Raw { uint32_t w[WORDS]; float zero; };
    auto fetch = [&](const Cursor<PARTS> &c, uint32_t raw_slot, Raw &raw) {
        typedef __attribute__((ext_vector_type(WORDS))) uint32_t words;
        const words v = *(const words *)(lds + raw_slot + wr * 32 + wk / 2);
#pragma unroll
        for (int j = 0; j < WORDS; ++j) raw.w[j] = v[j];
        const int of = c.group_of(p, FLUSH == 1 ? wk : 0) - zero_base;
        raw.zero = zeros ? (float)((const uint8_t *)(lds + ZERO_AT))[of * BN + wr] : 8.f;
    };
    auto put = [&](int slot, const Raw &raw, int j) {
        const int u = wk / 8 + j;
        *(Vec *)(lds + W_AT + slot * W_STAGE + wr * 128 + (u ^ ((wr >> 1) & 7)) * 16) = weights<TYPE>(raw.w[j], raw.zero);
    };

    // LATE: a sum is scaled while the products of the next one are under way
    constexpr bool LATE = TM * TN == 1 && FLUSH == 1 && PARTS == 1;
    f32x16 acc[TM][TN], sum[LATE ? 2 : 1][TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[i][j][e] = 0.f;
                if (LATE) sum[LATE][i][j][e] = 0.f;
            }
    float scale[LATE ? 2 : 1][TN];
    if (LATE) scale[LATE][0] = 0.f;
    const int hi = lane >> 5, sw = (lane >> 1) & 7;
    const char *const fa_at = lds + (wm * TM * 32 + (lane & 31)) * 128, *const fw_at = lds + W_AT + (wn * TN * 32 + (lane & 31)) * 128;
    auto scales = [&](int of, int at) {
#pragma unroll
        for (int j = 0; j < TN; ++j) scale[at][j] = ((const float *)(lds + SCALE_AT))[(of - scale_base) * BN + (wn * TN + j) * 32 + (lane & 31)];
    };
    auto flush = [&](int at) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(scale[at][j], sum[at][i][j][e], acc[i][j][e]);
    };
    struct Operands { Vec a[TM], w[TN]; };
    // activations that come straight into registers, a quarter's a step ahead
    typedef __attribute__((ext_vector_type(4))) int words4;
    words4 now_a[4][TM];
    const int a_lane = lane * 16 + wm * TM * 32 * (int)row_bytes;
    int a_step = first * 4096;
    auto ask = [&](int kk, int from) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            now_a[kk][i] = __builtin_amdgcn_raw_buffer_load_b128(ra, a_lane + i * 32 * (int)row_bytes, __builtin_amdgcn_readfirstlane(from + kk * 1024), 0);
    };
    auto take = [&](const char *fa_step, const char *fw_step, int kk, Operands &f) {
        const int at = ((2 * kk + hi) ^ sw) * 16;
        if constexpr (!DIRECT)
#pragma unroll
            for (int i = 0; i < TM; ++i) f.a[i] = *(const Vec *)(fa_step + i * 32 * 128 + at);
#pragma unroll
        for (int j = 0; j < TN; ++j) f.w[j] = *(const Vec *)(fw_step + j * 32 * 128 + at);
    };
    // a quarter of a step's products; fresh: the first of a sum
    auto multiply = [&](const Operands &f, bool fresh, int at) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                f32x16 none;
#pragma unroll
                for (int e = 0; e < 16; ++e) none[e] = 0.f;
                sum[at][i][j] = product(f.a[i], f.w[j], fresh ? none : sum[at][i][j]);
            }
    };

    // Step s multiplies its own operands, makes the weights of step s + 1, and asks for the activations of step s + RING - 1 and the weights of
    // step s + RING: into the places that step s - 1 has left.  (DIRECT: for the activations of step s + 1, a quarter as soon as its own are multiplied.)
    Cursor<PARTS> c0(p, walk, first), c1 = c0;
    c1.template next<FLUSH>(p, walk);
    scale_base = zero_base = c0.of;
    request_raw(RAW_AT);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) {
        request(i * A_STAGE);
        request_raw(RAW_AT + (i + 1) * RAW_STAGE);
    }
    if constexpr (DIRECT)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) ask(kk, a_step);
    tables(c0.of, true, zeros, std::integral_constant<int, ENTRIES>{});
    // (halves ask for tables in the same steps, for they meet at barriers: in those that the tables last for wherever they begin)
    const int64_t sure = (int64_t)(kTable - 1) * p.group / kStep;
    auto lasts = [&](const Cursor<PARTS> &c, int end) {
        if constexpr (HALVES == 1) return c.steps_below(p, end);
        else return (int)(sure < 0x7fffffff ? sure : 0x7fffffff);
    };
    int scales_until = lasts(c0, scale_base + kTable), zeros_until = zeros ? scales_until - 1 : 0x7fffffff;
    __builtin_amdgcn_s_waitcnt(vm_only(0));
    __syncthreads();
    {
        Raw raw;
        fetch(c0, RAW_AT, raw);
#pragma unroll
        for (int j = 0; j < WORDS; ++j) put(0, raw, j);
    }
    __syncthreads();
    // LDS places of this step's activations, of those asked for now, of the next step's weights as they come, of those asked for now
    uint32_t a_now = 0, a_ask = (RING - 1) * A_STAGE, raw_next = RAW_AT + RAW_STAGE, raw_ask = RAW_AT;
    auto one = [&](int parity) {
        request(a_ask);
        request_raw(raw_ask);
        a_ask = a_now;
        raw_ask = raw_next;
        // (seldom: a table lasts for hundreds of columns)
        if (scales_until <= 0 || zeros_until <= 0) {
            if (scales_until <= 0) {
                tables(scale_base = min(c0.of, p.groups - 1), true, false, std::integral_constant<int, 1>{});
                scales_until = lasts(c0, scale_base + kTable);
            }
            if (zeros_until <= 0) {
                tables(zero_base = min(c1.of, p.groups - 1), false, true, std::integral_constant<int, 1>{});
                zeros_until = lasts(c1, zero_base + kTable);
            }
            __syncthreads();
        }
        --scales_until;
        --zeros_until;
        const char *const fa_step = fa_at + a_now, *const fw_step = fw_at + parity * W_STAGE;
        Operands f[AHEAD + 1];
        Raw raw;
#pragma unroll
        for (int kk = 0; kk < AHEAD; ++kk) take(fa_step, fw_step, kk, f[kk]);
        fetch(c1, raw_next, raw);
        if (FLUSH < 4 || parity == 0) scales(c0.group_of(p, 0), 0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            if (kk + AHEAD < 4) take(fa_step, fw_step, kk + AHEAD, f[(kk + AHEAD) % (AHEAD + 1)]);
            const bool second = FLUSH == 1 && kk >= 2;
            if (second && kk == 2) {
                if (!LATE) flush(0);
                scales(c0.group_of(p, 32), LATE);
            }
            if constexpr (DIRECT)
#pragma unroll
                for (int i = 0; i < TM; ++i) f[kk % (AHEAD + 1)].a[i] = __builtin_bit_cast(Vec, now_a[kk][i]);
            multiply(f[kk % (AHEAD + 1)], kk == 0 ? FLUSH < 4 || parity == 0 : FLUSH == 1 && kk == 2, second ? LATE : 0);
            if (LATE && kk == 0) flush(LATE);
            if (LATE && kk == 2) flush(0);
            if constexpr (DIRECT) ask(kk, a_step + 4096);
            if (kk < WORDS) put(parity ^ 1, raw, kk < WORDS ? kk : 0);
        }
        if constexpr (DIRECT) a_step += 4096;
        if (!LATE && (FLUSH < 4 || parity == 1)) flush(0);
        c0 = c1;
        c1.template next<FLUSH>(p, walk);
        a_now = a_now == (RING - 1) * A_STAGE ? 0 : a_now + A_STAGE;
        raw_next = raw_next == RAW_AT + (RING - 1) * RAW_STAGE ? RAW_AT : raw_next + RAW_STAGE;
        // what the next step reads has been asked for RING - 2 steps ago
        __builtin_amdgcn_s_waitcnt(vm_only((RING - 2) * (LOADS + 1) + (DIRECT ? LOADS : 0)));
        __syncthreads();
    };
    // (an odd number of steps ends in one of zeros)
    for (int step = 0; step < steps; step += 2) {
        one(0);
        one(1);
    }
    if (LATE) flush(LATE);
    __builtin_amdgcn_s_waitcnt(vm_only(0));
    __syncthreads();

    // 32 tokens of a wave at a time through its own part of LDS, from where rows leave in wide pieces; of halves, half the rows each, both sums put together
    constexpr int PITCH = 32 * TN + 4, LPR = 4 * TN, RPI = 64 / LPR;
    float *const mine = (float *)all_lds + (half * WM * WN + wave) * 32 * PITCH;
    const float *const parts = (const float *)all_lds + wave * 32 * PITCH;
    const int n = n0 + wn * TN * 32 + lane % LPR * 8;
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = p.bias && !walk.sums ? load_as_f32(p.bias, min(n + e, p.N - 1) * p.sbias, p.bias_type) : 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[(8 * (e / 4) + 4 * hi + e % 4) * PITCH + 32 * j + (lane & 31)] = acc[i][j][e];
        if constexpr (HALVES > 1) __syncthreads();
        else __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 32 / HALVES; r += RPI) {
            const int row = half * (32 / HALVES) + r + lane / LPR, m = m0 + (wm * TM + i) * 32 + row;
            const float *const at = &parts[row * PITCH + lane % LPR * 8];
            f32x4 lo = *(const f32x4 *)at, up = *(const f32x4 *)(at + 4);
            if constexpr (HALVES > 1) {
                lo += *(const f32x4 *)(at + WM * WN * 32 * PITCH);
                up += *(const f32x4 *)(at + WM * WN * 32 * PITCH + 4);
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (e < 4 ? lo[e] : up[e - 4]) + bias[e];
            if (m < p.M && n < p.N) {
                if (walk.sums) store8<DT_F32>((char *)(walk.sums + ((int64_t)split * p.M + m) * p.N + n), p.N - n, v);
                else if (p.out_type == DT_BF16) store8<DT_BF16>((char *)p.out + (m * p.so_m + n) * 2, p.N - n, v);
                else if (p.out_type == DT_F16) store8<DT_F16>((char *)p.out + (m * p.so_m + n) * 2, p.N - n, v);
                else store8<DT_F32>((char *)p.out + (m * p.so_m + n) * 4, p.N - n, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The sums of workgroups that shared tiles by K
__global__ void __launch_bounds__(256) join_kernel(const PackedParams p, const float *sums, int splits)
{
    const int64_t total = (int64_t)p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / p.N, n = i - m * p.N;
        float v = sums[i];
        for (int t = 1; t < splits; ++t) v += sums[t * total + i];
        if (p.bias) v += load_as_f32(p.bias, n * p.sbias, p.bias_type);
        store_from_f32(p.out, m * p.so_m + n, p.out_type, v);
    }
}

// Activations as the small tiles take them: 16-bit rows of `padded` columns, zeros behind the last; fp32 as three parts beside each other
template <int TYPE>
__global__ void __launch_bounds__(256) lay_kernel(const PackedParams p, uint16_t *to, int padded)
{
    const int sets = padded / 8;
    const int64_t total = (int64_t)p.M * sets;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / sets;
        const int k = (int)(i - m * sets) * 8;
        Activations<TYPE> v;
        v.load((const element<TYPE> *)p.a + m * p.sa_m + k, p.K - k);
        typename Operand<TYPE>::Vec x[Operand<TYPE>::parts];
        v.operands(x);
#pragma unroll
        for (int t = 0; t < Operand<TYPE>::parts; ++t) *(u32x4 *)(to + (m * Operand<TYPE>::parts + t) * padded + k) = __builtin_bit_cast(u32x4, x[t]);
    }
}

// Activations as operands of the matrix instructions: 32 rows x 16 columns are 1 KB, lane by lane, those of a row of such blocks one behind another;
// `columns` of each part, zeros behind the last row and column
template <int TYPE>
__global__ void __launch_bounds__(256) lay_blocks_kernel(const PackedParams p, uint16_t *to, int columns)
{
    constexpr int PARTS = Operand<TYPE>::parts;
    const int row = (int)(blockIdx.x * 32 + threadIdx.x / 8), k = (int)(blockIdx.y * 64 + threadIdx.x % 8 * 8);
    Activations<TYPE> v;
    v.load((const element<TYPE> *)p.a + (int64_t)min(row, p.M - 1) * p.sa_m + k, row < p.M ? p.K - k : 0);
    typename Operand<TYPE>::Vec x[PARTS];
    v.operands(x);
#pragma unroll
    for (int t = 0; t < PARTS; ++t)
        *(u32x4 *)(to + ((int64_t)(row / 32) * (PARTS * columns) + (t * columns + k) / 16 * 16) * 32 + (k / 8 % 2 * 32 + row % 32) * 8) = __builtin_bit_cast(u32x4, x[t]);
}

// blocks of 32 weights that make a sum in front of its scale
int flush_of(const PackedParams &p) { return p.groups <= 1 || p.group % 128 == 0 ? 4 : p.group % 64 == 0 ? 2 : 1; }

template <int TYPE, int MT, int NT, int WAVES, int U> hipError_t run_direct(const PackedParams &p, hipStream_t s)
{
    const int64_t tm = (p.M + 16 * MT - 1) / (16 * MT), tn = (p.N + 16 * NT - 1) / (16 * NT);
    if (tm * tn > 0xffffffffLL) return hipErrorInvalidConfiguration;      // (of 2^39 results and more)
    const int flush = flush_of(p);
    auto of = [&](auto wide) {
        constexpr bool W = decltype(wide)::value;
        return flush == 4 ? direct_kernel<TYPE, MT, NT, WAVES, U, 4, W> : flush == 2 ? direct_kernel<TYPE, MT, NT, WAVES, U, 2, W> : direct_kernel<TYPE, MT, NT, WAVES, U, 1, W>;
    };
    auto *const kernel = p.scale_type == DT_F32 ? of(std::integral_constant<bool, true>{}) : of(std::integral_constant<bool, false>{});
    // (tiles from 2^22 on in several launches: one has below 2^32 threads)
    for (int64_t first = 0; first < tm * tn; first += 1 << 22) {
        const int64_t left = tm * tn - first;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)(left < 1 << 22 ? left : 1 << 22)), dim3(64 * WAVES), 0, s, p, (int)tm, (uint32_t)first);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Rows of weights at multiples of four bytes
__global__ void __launch_bounds__(256) lay_weights_kernel(const PackedParams p, uint8_t *to, int bytes, int stride)
{
    const int64_t total = (int64_t)p.N * bytes;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t n = i / bytes;
        to[n * stride + (i - n * bytes)] = p.w[n * p.sw_n + (i - n * bytes)];
    }
}

// The kernel of a call: what an estimate of each, in microseconds, finds fastest.  tm: 0 the direct kernel, 1 tiles of 64 x 64, 2 the same with two
// halves of waves that share a tile by K (16-bit activations), 3 and 4 tiles of 256 x 64 and 256 x 128; splits: workgroups that share a tile by K.
//
// Tiles: workgroups in rounds of one (256 x 128, halves) or two (small, 256 x 64) to a compute unit; a round takes 5 to 8 and a step of 64 weights what is measured
// below; sums of parts go through memory, 3 for the launch that joins them and 4.5 TB/s; activations that are laid out, 2.5 for a launch and 5 TB/s. Direct: 2.5,
// and for each 1024 of K, in a workgroup's eight waves, 0.45, 0.35 per 16 channels and 0.65 per 16 tokens, over again as often as workgroups fill the
// card.  fp32: three parts are three times the steps.  Measured (us, groups of 128, direct / 64 x 64 with splits / halves / 256 x 64 / 256 x 128):
//   64 x 2560 x 5120: 15.5 / 14.7 (6) / 14.2 (5), 21.3 (8) / - / -     32 x 2560 x 5120: 13.1 / 14.1 (6) / 13.3 (5) / - / -
//   200 x 4096 x 1024: 16.4 / 11.0 (1) / 9.9 (1) / - / -     64 x 10576 x 2560: 21.7 / 19.4 (3), 22.4 (1) / 17.2 (1) / - / -
//   64 x 20000 x 2560: 33.7 / 28.1 (1) / 32.8 (1) / - / -     32 x 50000 x 2560: 44.7 / 53.2 (1) / 62.7 (1) / - / -
//   128 x 10576 x 2560: 39 / 27.9 (1) / 32.5 (1) / 27.3 (1) / 30.0 (2)     1024 x 800 x 704: 10.7 / 9.6 (1) / 8.7 (1) / 13.9 (1) / 18.7 (4)
//   512 x 2560 x 5120: 64 / 51 (1) / 56 (1) / 31.4 (3), 34.7 (2) / 35.8 (4)     700 x 4000 x 1000: 27.9 / 24.8 (1) / - / 16.8 (1) / 22.7 (1)
//   1024 x 4096 x 4096: - / 83 (1) / 93 (1) / 46 (1), 67 (2) / 62 (1), 57 (2)     300 x 10576 x 2560: 81 / 53 (1) / - / 50 (1) / 39.8 (1)
//   2048 x 5120 x 2560: 240 / 130 (1) / - / 71 (1) / 83.3 (1)     1490 x 3312 x 256: 32 / 18.8 (1) / - / 16.9 (1) / 14.5 (1)
int direct_rows(int M) { return M <= 16 ? 16 : 32; }
// 16s of channels of a workgroup of the direct kernel: activations are read once for all of them.  Enough that the workgroups run at once, two where that
// cannot be; one where activations are few and the time is that of the first weights to come.  Measured (us, one / two / four, bf16, groups of 128):
//   16 x 2560 x 5120: 8.8 / 10.6 / 14.5     16 x 5000 x 5000: 12.3 / 9.5 / 14.2     16 x 10576 x 2560: 12.0 / 11.4 / 10.2
//   32 x 10576 x 2560: 18.9 / 15.4 / 11.9     16 x 20000 x 2560: 18.2 / 15.1 / 16.2     32 x 20000 x 2560: 34.6 / 21.4 / 22.0
//   1 x 10576 x 2560: 7.3 / 8.1 / 9.0     1 x 20000 x 2560: 10.4 / 11.2 / 13.8     1 x 50000 x 2560: 22.4 / 19.8 / 24.0
int direct_width(int M, int N, int n_cu)
{
    const int64_t tiles_m = (M + direct_rows(M) - 1) / direct_rows(M), units = n_cu > 0 ? n_cu : 256;
    if (M <= 4) return N < 128 * units ? 1 : 2;
    for (int wide = 1; wide <= 4; wide *= 2)
        if ((N + 16 * wide - 1) / (16 * wide) * tiles_m <= units) return wide;
    return 2;
}
struct Plan {
    int tm, splits;
};
Plan plan_of(int M, int N, int K, int group, int type, int n_cu)
{
    if (M <= 16 || K > kLongest || K == 0) return {0, 1};
    const double units = n_cu > 0 ? n_cu : 256;
    const int flush = group >= K || group % 128 == 0 ? 4 : group % 64 == 0 ? 2 : 1, parts = type == DT_F32 ? 3 : 1;
    const int pairs = (K + 2 * kStep - 1) / (2 * kStep) * parts;
    const double blocks = 2.5 + (type == DT_F32 ? 10. : 4.) * M * K / 5e6, lay = type == DT_F32 ? blocks : 0;
    const int wide = direct_width(M, N, n_cu);
    const double filled = (double)((N + 16 * wide - 1) / (16 * wide)) * ((M + 31) / 32) / units, step = 0.45 + 0.35 * wide + 0.65 * parts * (M < 32 ? M : 32) / 16;
    Plan best{0, 1};
    double least = 2.5 + (filled <= 1 ? (K / 128 + 7) / 8 * step : ((K / 128 + 7) / 8 * step + 0.6) * (0.85 * filled + 0.5));
    auto tiles = [&](int tm, int bm, int bn, int halves, double slots, double lay, double begin, double step) {
        const double n = (double)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
        // (launches of below 2^32 threads: of tiles, and of the activations' layout)
        const double threads = tm == 1 ? 256 : 512, most = 4294967295.;
        if (tm >= 3 && (M + 31.) / 32 * 256 > most) return;
        for (int splits = 1; splits <= 16 && splits * halves * 2 <= pairs + 1 && n * splits * threads <= most; ++splits) {
            const double rounds = n * splits / slots;
            double whole = tm != 1 ? ceil(rounds) : rounds < 1 ? 1 : (rounds + 2 * ceil(rounds)) / 3;
            if (tm == 3 && two_to_a_unit(type, 2, flush))           // two take 1.53 times as long as one
                whole = 1.53 * floor(rounds / 2) + (rounds <= 2 * floor(rounds / 2) ? 0 : rounds <= 2 * floor(rounds / 2) + 1 ? 1 : 1.53);
            const double join = splits > 1 ? 3 + 8. * splits * M * N / 4.5e6 : 0;
            const double t = lay + join + whole * (begin + 2 * step * ((pairs + splits * halves - 1) / (splits * halves)));
            if (t < least) {
                least = t;
                best = {tm, splits};
            }
        }
    };
    tiles(1, 64, 64, 1, 2 * units, lay, 5, flush == 4 ? 0.55 : flush == 2 ? 0.6 : 0.72);
    if (parts == 1) tiles(2, 64, 64, 2, units, lay, 5, flush == 4 ? 0.57 : flush == 2 ? 0.59 : 0.64);
    if (M > 64) {
        tiles(3, 256, 64, 1, units, blocks, 6.6, flush == 4 ? 0.55 : flush == 2 ? 0.58 : 0.7);
        if (parts == 1 || flush > 1) tiles(4, 256, 128, 1, units, blocks, 8, flush == 4 ? 0.82 : flush == 2 ? 0.88 : 1.15);
    }
    return best;
}

bool laid(const PackedParams &p)       // rows as the tile kernel takes them already
{
    return p.type != DT_F32 && p.K % 8 == 0 && p.sa_m % 8 == 0 && p.sa_m >= 0 && p.sa_m < (1 << 22) && ((uintptr_t)p.a & 15) == 0;
}
bool weights_laid(const PackedParams &p)
{
    return p.K % 8 == 0 && p.sw_n % 4 == 0 && p.sw_n >= 0 && p.sw_n < (1 << 22) && ((uintptr_t)p.w & 3) == 0;
}
uint64_t weights_bytes(int N, int K) { return (uint64_t)N * ((K + 7) / 8 * 4); }
uint64_t laid_bytes(int M, int K, int type, int tm)
{
    const uint64_t rows = tm >= 3 ? ((uint64_t)M + 31) / 32 * 32 : M, columns = tm >= 3 ? (K + 2 * kStep - 1) / (2 * kStep) * (2 * kStep) : (K + 7) / 8 * 8;
    return rows * columns * 2 * (type == DT_F32 ? 3 : 1);
}

template <int TYPE, int WM, int WN, int TM, int TN, int RING, int FLUSH, int HALVES, bool DIRECT> hipError_t run_tile(const PackedParams &p, const Walk &walk, hipStream_t s)
{
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    constexpr int ring = (RING * ((DIRECT ? 0 : BM * 128) + BN * 32) + 2 * BN * 128 + kTable * BN * 5) * HALVES, out = WM * WN * HALVES * 32 * (32 * TN + 4) * 4, lds = ring > out ? ring : out;
    static std::atomic<uint64_t> done;
    auto *const kernel = tile_kernel<TYPE, WM, WN, TM, TN, RING, FLUSH, HALVES, DIRECT>;
    const hipError_t e = ensure_dynamic_lds((const void *)kernel, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tm * tn * walk.splits)), dim3(64 * WM * WN * HALVES), lds, s, p, walk, (int)tm, (int)tn);
    return hipGetLastError();
}

template <int TYPE> hipError_t run_tiles(const PackedParams &p, const Plan &plan, hipStream_t s)
{
    constexpr int T = TYPE;
    Walk walk{p.a, p.w, p.sa_m, p.sw_n, 1, p.K, (p.K + 1) / 2, (p.K + kStep - 1) / kStep, plan.splits, 0, nullptr};
    char *room = (char *)p.room;
    if (!weights_laid(p)) {
        walk.sw_n = walk.w_bytes = (p.K + 7) / 8 * 4;
        walk.w = (const uint8_t *)room;
        room += (weights_bytes(p.N, p.K) + 255) / 256 * 256;
        const int64_t blocks = ((int64_t)p.N * ((p.K + 1) / 2) + 255) / 256;
        hipLaunchKernelGGL(lay_weights_kernel, dim3((uint32_t)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, p, (uint8_t *)walk.w, (p.K + 1) / 2, walk.w_bytes);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (plan.tm >= 3) {
        walk.parts = Operand<TYPE>::parts;
        walk.padded = (walk.steps + 1) / 2 * 2 * kStep;
        walk.sa_m = (int64_t)walk.parts * walk.padded;
        walk.a = room;
        room += (laid_bytes(p.M, p.K, p.type, plan.tm) + 255) / 256 * 256;
        hipLaunchKernelGGL(lay_blocks_kernel<TYPE>, dim3((uint32_t)((p.M + 31) / 32), (uint32_t)(walk.padded / 64)), dim3(256), 0, s, p, (uint16_t *)walk.a, walk.padded);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    } else if (!laid(p)) {
        walk.parts = Operand<TYPE>::parts;
        walk.padded = (p.K + 7) / 8 * 8;
        walk.sa_m = (int64_t)walk.parts * walk.padded;
        walk.a = room;
        room += (laid_bytes(p.M, p.K, p.type, plan.tm) + 255) / 256 * 256;
        const int64_t blocks = ((int64_t)p.M * (walk.padded / 8) + 255) / 256;
        hipLaunchKernelGGL(lay_kernel<TYPE>, dim3((uint32_t)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, p, (uint16_t *)walk.a, walk.padded);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    walk.steps = (walk.steps + 1) / 2 * 2;                   // pairs of steps stay in a part, and in a workgroup
    const int steps = walk.parts * walk.steps;
    const int units = plan.tm == 2 ? 4 : 2;                  // (pairs of steps, for two halves)
    walk.per = (steps + units * walk.splits - 1) / (units * walk.splits) * units;
    walk.splits = (steps + walk.per - 1) / walk.per;
    if (walk.splits > 1) walk.sums = (float *)room;
    const int flush = flush_of(p);
    hipError_t e;
    auto small = [&](auto halves) {
        constexpr int H = decltype(halves)::value;
        if (flush == 4) return run_tile<T, 2, 2, 1, 1, 5, 4, H, false>(p, walk, s);
        return flush == 2 ? run_tile<T, 2, 2, 1, 1, 5, 2, H, false>(p, walk, s) : run_tile<T, 2, 2, 1, 1, 5, 1, H, false>(p, walk, s);
    };
    auto wide = [&](auto tn) {
        constexpr int TN = decltype(tn)::value;
        if (flush == 4) return run_tile<T, 8, 1, 1, TN, 4, 4, 1, true>(p, walk, s);
        if (flush == 2) return run_tile<T, 8, 1, 1, TN, 4, 2, 1, true>(p, walk, s);
        if constexpr (TN == 2 || Operand<T>::parts == 1) return run_tile<T, 8, 1, 1, TN, 4, 1, 1, true>(p, walk, s);
        else return hipErrorInvalidConfiguration;
    };
    if (plan.tm == 4) e = wide(std::integral_constant<int, 4>{});
    else if (plan.tm == 3) e = wide(std::integral_constant<int, 2>{});
    else if (plan.tm == 1) e = small(std::integral_constant<int, 1>{});
    else if constexpr (Operand<T>::parts == 1) e = small(std::integral_constant<int, 2>{});
    else e = hipErrorInvalidConfiguration;
    if (e != hipSuccess || !walk.sums) return e;
    const int64_t blocks = ((int64_t)p.M * p.N + 255) / 256;
    hipLaunchKernelGGL(join_kernel, dim3((uint32_t)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, p, walk.sums, walk.splits);
    return hipGetLastError();
}

template <int TYPE> hipError_t of_type(const PackedParams &p, int n_cu, hipStream_t s)
{
    const Plan plan = plan_of(p.M, p.N, p.K, p.group, p.type, n_cu);
    if (plan.tm && p.K > 0 && p.room_bytes >= matmul_packed_room(p.M, p.N, p.K, p.group, p.type, n_cu)) return run_tiles<TYPE>(p, plan, s);
    const int wide = direct_width(p.M, p.N, n_cu);
    if (p.M <= 16) return wide == 1 ? run_direct<TYPE, 1, 1, 8, 2>(p, s) : wide == 2 ? run_direct<TYPE, 1, 2, 8, 1>(p, s) : run_direct<TYPE, 1, 4, 8, 1>(p, s);
    return wide == 1 ? run_direct<TYPE, 2, 1, 8, 1>(p, s) : wide == 2 ? run_direct<TYPE, 2, 2, 8, 1>(p, s) : run_direct<TYPE, 2, 4, 8, 1>(p, s);
}

}  // namespace

uint64_t matmul_packed_room(int M, int N, int K, int group, int type, int n_cu)
{
    const Plan plan = plan_of(M, N, K, group, type, n_cu);
    if (!plan.tm || K == 0) return 0;
    return (laid_bytes(M, K, type, plan.tm) + 255) / 256 * 256 + (weights_bytes(N, K) + 255) / 256 * 256 + (plan.splits > 1 ? (uint64_t)plan.splits * M * N * 4 : 0);
}

hipError_t launch_matmul_packed(const PackedParams &p, int n_cu, hipStream_t s)
{
    if (p.M == 0 || p.N == 0) return hipSuccess;
    if (p.type == DT_F32) return of_type<DT_F32>(p, n_cu, s);
    return p.type == DT_BF16 ? of_type<DT_BF16>(p, n_cu, s) : of_type<DT_F16>(p, n_cu, s);
}

}  // namespace ssd
