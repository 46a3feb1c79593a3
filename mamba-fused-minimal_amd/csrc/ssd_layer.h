// Argument blocks and small device helpers of the operators around the state path: the short convolution, the whole selective
// scan, the norm and the 8-bit matrix product (ssd_conv.hip, ssd_scan*.hip, ssd_norm.hip, ssd_matmul.hip).
#pragma once
#include "ssd_params.h"

namespace ssd {

enum : int { DT_I8 = 3 };

// Short causal convolution over tokens, one filter per channel.  All strides in elements.
struct ConvParams {
    const void *x;          // (b, L, D)
    const void *w;          // (D, K)
    const void *bias;       // (D) or null
    const void *init;       // (b, D, K-1) or null; the type of x
    const int32_t *seq;     // (b, L) or null
    const int32_t *len;     // (b) or null
    void *y;                // (b, L, D)
    void *fin;              // (b, D, K-1), the type of x
    int batch, seqlen, dim, width;
    int64_t sx_b, sx_l, sw_d, sw_k, sbias, si_b, si_d, si_k, sq_b, sq_l, slen, sy_b, sy_l, sf_b, sf_d, sf_k;
    int type, w_type, bias_type, silu;
};

// One token of it; the states of row b are slot slots[b] of a pool.
struct ConvStepParams {
    const void *x;          // (b, D)
    void *states;           // (slots, D, K-1), the type of x; updated
    const void *w, *bias;
    const int32_t *slots;   // (b) or null: row b is slot b
    void *y;                // (b, D)
    int batch, dim, width, n_slots;
    int64_t sx_b, ss_s, ss_d, ss_k, sw_d, sw_k, sbias, sslots, sy_b;
    int type, w_type, bias_type, silu;
};

// What turns the raw dt into a step: bias, softplus, limits.
struct DeltaParams {
    const void *bias;       // (H) or null
    int64_t sbias;
    int bias_type, softplus;
    float lo, hi;
};

// The selective scan over prompts.
struct SelScanParams {
    const void *x, *z;      // (b, L, H, P); z null: no gate
    const void *dt;         // (b, L, H)
    const void *A;          // (H)
    const void *B, *C;      // (b, L, G, N), the type of x
    const void *D;          // (H) or (H, P), or null
    const void *init;       // (b, H, P, N) or null
    const int32_t *seq;     // (b, L) or null
    const int32_t *len;     // (b) or null
    void *y;                // (b, L, H, P), the type of x
    float *fin;             // (b, H, P, N)
    float *ws_states;       // (b, H, segments, P, N), contiguous: the state each segment adds, then the one that enters it
    float *ws_decay;        // (b, H, segments): the factor on what enters (negative: nothing passes)
    float *ws_steps;        // on the matrix instructions: (b, H, chunks) records of steps and decays
    int chunks;             // of 64 tokens
    int batch, seqlen, nheads, headdim, dstate, ngroups;
    int segments, segment_tokens;
    int head_tokens, head;  // on the matrix instructions of bf16: of the first segment; it is done in front of the others, y and all
    int joined;             // ws_states holds what enters the segments (launch_scan_join has run)
    int64_t sx_b, sx_l, sx_h, sz_b, sz_l, sz_h, sdt_b, sdt_l, sdt_h, sA, sB_b, sB_l, sB_g, sC_b, sC_l, sC_g, sD_h, sD_p;
    int64_t si_b, si_h, si_p, sq_b, sq_l, slen, sy_b, sy_l, sy_h, sf_b, sf_h, sf_p;
    int type, z_type, dt_type, A_type, D_type, init_type;
    DeltaParams delta;
};

// One token of it, the states in a pool.
struct SelStepParams {
    const void *x, *z;      // (b, H, P)
    const void *dt;         // (b, H)
    const void *A;          // (H)
    const void *B, *C;      // (b, G, N)
    const void *D;          // (H) or (H, P), or null
    float *states;          // (slots, H, P, N); updated
    const int32_t *slots;   // (b) or null
    void *y;                // (b, H, P)
    int batch, nheads, headdim, dstate, ngroups, n_slots;
    int64_t sx_b, sx_h, sz_b, sz_h, sdt_b, sdt_h, sA, sB_b, sB_g, sC_b, sC_g, sD_h, sD_p, ss_s, ss_h, ss_p, sslots, sy_b, sy_h;
    int type, z_type, dt_type, A_type, D_type;
    DeltaParams delta;
};

struct NormParams {
    const void *x, *residual, *z;      // (rows, D); residual and z null where there is none
    const void *w;                     // (D)
    void *out;                         // (rows, D): the type of x, or 8 bits
    float *scale;                      // (rows), with 8 bits
    void *residual_out;                // (rows, D), with a residual
    int64_t rows;
    int dim;
    int64_t sx, sr, sz, sw, so, sro, sscale;
    int type, r_type, z_type, w_type, int8;
    float eps;
};

struct MatmulParams {
    const int8_t *a;                   // (M, K)
    const int8_t *w;                   // (N, K)
    const float *sa, *sw;              // (M), (N)
    const void *bias;                  // (N) or null
    void *out;                         // (M, N)
    int M, N, K;
    int64_t sa_m, sw_n, ssa, ssw, sbias, so_m;
    int out_type, bias_type;
};

hipError_t launch_short_conv(const ConvParams &p, hipStream_t s);
hipError_t launch_short_conv_step(const ConvStepParams &p, hipStream_t s);
hipError_t launch_scan_step(const SelStepParams &p, hipStream_t s);
// the scan for any type and size up to kScanMaxState state columns; and on the bf16 matrix instructions
constexpr int kScanMaxState = 256;
hipError_t launch_scan_any(const SelScanParams &p, hipStream_t s);
constexpr int kScanRecord = 5 * 64;      // words of ws_steps per (row, head, chunk)
bool scan_mfma_supported(const SelScanParams &p);
hipError_t launch_scan_mfma(const SelScanParams &p, hipStream_t s);
// ws_states: what every segment adds -> what enters it
hipError_t launch_scan_join(const SelScanParams &p, hipStream_t s);
hipError_t launch_norm(const NormParams &p, hipStream_t s);
hipError_t launch_matmul(const MatmulParams &p, int n_cu, hipStream_t s);

namespace layer {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

template <int TYPE> struct Element;
template <> struct Element<DT_F32> { typedef float type; };
template <> struct Element<DT_BF16> { typedef uint16_t type; };
template <> struct Element<DT_F16> { typedef _Float16 type; };
template <int TYPE> using element = typename Element<TYPE>::type;

template <int TYPE> __device__ __forceinline__ float to_f32(element<TYPE> v)
{
    if constexpr (TYPE == DT_BF16) return bf16_bits_to_f32(v);
    else return (float)v;
}
template <int TYPE> __device__ __forceinline__ element<TYPE> from_f32(float v)
{
    if constexpr (TYPE == DT_BF16) return f32_to_bf16_bits(v);
    else return (element<TYPE>)v;
}

// 16 bytes at any address that an element may have: gfx950 loads and stores them in one instruction whatever their alignment
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t wide2;
typedef __attribute__((ext_vector_type(4), aligned(4))) uint32_t wide4;
template <int TYPE> struct Wide {
    typedef element<TYPE> E;
    static constexpr int n = 16 / sizeof(E);
    typedef std::conditional_t<sizeof(E) == 4, wide4, wide2> raw;
    struct Pack { E e[n]; };
    __device__ static __forceinline__ Pack load(const E *p) { return __builtin_bit_cast(Pack, *(const raw *)p); }
    __device__ static __forceinline__ void store(E *p, const Pack &v) { *(raw *)p = __builtin_bit_cast(raw, v); }
    // the same for what no later access is near to: the lines are the first to leave the caches
    __device__ static __forceinline__ Pack load_once(const E *p) { return __builtin_bit_cast(Pack, __builtin_nontemporal_load((const raw *)p)); }
    __device__ static __forceinline__ void store_past(E *p, const Pack &v) { __builtin_nontemporal_store(__builtin_bit_cast(raw, v), (raw *)p); }
};

__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// dt as the scan uses it.  log1p(t) = log(u) t / (u - 1) with u = fl(1 + t): the quotient compensates the rounding of u.
__device__ __forceinline__ float delta_of(const DeltaParams &p, float d)
{
    if (p.softplus && d <= 20.f) {
        const float t = __expf(d), u = 1.f + t;
        d = u == 1.f ? t : __logf(u) * __fdividef(t, u - 1.f);
    }
    // not fminf(fmaxf()): those drop a NaN
    d = d < p.lo ? p.lo : d;
    return d > p.hi ? p.hi : d;
}

// A decay over many tokens.  Never zero: an infinity that it is applied to stays one, as it does token by token; to a finite value the
// smallest normal number is as little as zero.
__device__ __forceinline__ float not_zero(float decay) { return decay < 1.17549435e-38f ? 1.17549435e-38f : decay; }

// A row's tokens: its length, never beyond the tensor
__device__ __forceinline__ int row_tokens(const int32_t *len, int64_t stride, int b, int L)
{
    if (!len) return L;
    const int n = len[b * stride];
    return n < 0 ? 0 : n > L ? L : n;
}

// Sum over the lanes of aligned groups of `N` lanes (a power of two), in every lane of the group
template <int N> __device__ __forceinline__ float group_sum(float v)
{
#if defined(__HIP_DEVICE_COMPILE__)
    auto moved = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    using std::integral_constant;
    if constexpr (N >= 2) v += moved(v, integral_constant<int, 0xb1>{});      // quad_perm: lane ^ 1
    if constexpr (N >= 4) v += moved(v, integral_constant<int, 0x4e>{});      // quad_perm: lane ^ 2
    if constexpr (N >= 8) v += moved(v, integral_constant<int, 0x141>{});     // row_half_mirror: the other quad of eight lanes
    if constexpr (N >= 16) v += moved(v, integral_constant<int, 0x140>{});    // row_mirror: the other half of sixteen
    if constexpr (N >= 32) v += __shfl_xor(v, 16);
    if constexpr (N >= 64) v += __shfl_xor(v, 32);
#endif
    return v;
}
template <int N> __device__ __forceinline__ uint32_t group_max(uint32_t v)
{
    for (int d = 1; d < N; d *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

}  // namespace layer
}  // namespace ssd
