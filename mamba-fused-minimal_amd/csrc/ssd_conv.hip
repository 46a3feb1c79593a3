// Short causal convolution over tokens with one filter of up to four taps per channel, bias and silu: for prompts and for
// single tokens.
//
//   y[t, d] = act(bias[d] + sum_k w[d, k] x[t - (K-1) + k, d])
//
// in 32 bits, rounded once.  Tokens in front of the row come from initial_states (they belong to sequence 0) or are zero; a
// tap that lies in another sequence than its token counts as zero, whatever it holds; behind a row's length y is zero.
// final_states: the K-1 inputs in front of the row's end, zero where another sequence's.
//
// HBM bound: every input element is read and every output element written once, K + a silu's operations between.  A thread
// owns 16 bytes of channels and walks a run of tokens with the last K-1 inputs in registers, so what is read twice is K-1 of
// every run + K-1 rows, and those are in the L2 of the neighbour.  4 x 8192 tokens of 5376 channels in bf16: 139 us, 5.07 TB/s of the 5.2
// that a copy reaches; 64 single tokens: 5.1 us, the latency of a launch and three loads.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

// N channels at a time: 16 bytes of them, or one where a row has fewer than that.  A row whose channels are no multiple of N ends in
// a set that reaches back: its first channels are computed twice, to the same values.
template <int TYPE, int N> struct Row {
    typedef element<TYPE> E;
    E e[N];
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = (E)0;
    }
    __device__ __forceinline__ void load(const E *p)
    {
        if constexpr (N == Wide<TYPE>::n) {
            const auto v = Wide<TYPE>::load(p);
#pragma unroll
            for (int i = 0; i < N; ++i) e[i] = v.e[i];
        } else e[0] = *p;
    }
    __device__ __forceinline__ void load(const E *p, int64_t stride)
    {
        if (stride == 1) load(p);
        else
#pragma unroll
            for (int i = 0; i < N; ++i) e[i] = p[i * stride];
    }
    // PAST: what is written leaves the caches first
    template <bool PAST = false> __device__ __forceinline__ void store(E *p) const
    {
        if constexpr (N == Wide<TYPE>::n) {
            typename Wide<TYPE>::Pack v;
#pragma unroll
            for (int i = 0; i < N; ++i) v.e[i] = e[i];
            if constexpr (PAST) Wide<TYPE>::store_past(p, v);
            else Wide<TYPE>::store(p, v);
        } else *p = e[0];
    }
    // all but the first `skip`
    __device__ __forceinline__ void store(E *p, int64_t stride, int skip) const
    {
        if (stride == 1 && skip == 0) store(p);
        else
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i >= skip) p[i * stride] = e[i];
    }
};

// The taps and the bias of N channels from d0 on.  A filter stored densely in the type of x comes in wide
// loads: element by element the 40 loads took longer than the inputs of a short run.
template <int TYPE, int K, int N, class P>
__device__ __forceinline__ void load_filter(const P &p, int d0, float (&w)[K][N], float (&bias)[N])
{
    typedef element<TYPE> E;
    if (p.w_type == TYPE && p.sw_k == 1 && p.sw_d == K) {
        Row<TYPE, N> q[K];
#pragma unroll
        for (int k = 0; k < K; ++k) q[k].load((const E *)p.w + (int64_t)d0 * K + k * N);
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][j] = to_f32<TYPE>(q[(j * K + k) / N].e[(j * K + k) % N]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][j] = load_as_f32(p.w, (d0 + j) * p.sw_d + k * p.sw_k, p.w_type);
    }
    if (p.bias && p.bias_type == TYPE && p.sbias == 1) {
        Row<TYPE, N> q;
        q.load((const E *)p.bias + d0);
#pragma unroll
        for (int j = 0; j < N; ++j) bias[j] = to_f32<TYPE>(q.e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) bias[j] = p.bias ? load_as_f32(p.bias, (d0 + j) * p.sbias, p.bias_type) : 0.f;
    }
}

// RUN tokens per thread; SEQ: seq_idx may be given
template <int TYPE, int K, int RUN, bool SEQ, int N>
__global__ void __launch_bounds__(256) conv_kernel(const ConvParams p, int vectors, int runs)
{
    typedef element<TYPE> E;
    constexpr int H = K - 1;
    // workgroups are dealt to the 8 XCDs in turn: each XCD gets a contiguous part of the runs, whose shared rows its L2 then holds
    const uint32_t per = gridDim.x / 8, wg = blockIdx.x < per * 8 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
    const uint32_t i = wg * 256u + threadIdx.x;
    const uint32_t v = i % (uint32_t)vectors, rb = i / (uint32_t)vectors;
    const int r = (int)(rb % (uint32_t)(runs + 1)), b = (int)(rb / (uint32_t)(runs + 1));
    if (b >= p.batch) return;
    const int d0 = min((int)v * N, p.dim - N);
    const int len = row_tokens(p.len, p.slen, b, p.seqlen);
    const E *x = (const E *)p.x + b * p.sx_b + d0;
    const int32_t *seq = SEQ && p.seq ? p.seq + b * p.sq_b : nullptr;
    auto id = [&](int t) { return t < 0 || !seq ? 0 : seq[t * p.sq_l]; };
    // the input of token t (t < len), in front of the row the initial state
    auto input = [&](int t, Row<TYPE, N> &to) {
        if (t >= 0) to.load(x + t * p.sx_l);
        else if (p.init) to.load((const E *)p.init + b * p.si_b + (H + t) * p.si_k + d0 * p.si_d, p.si_d);
        else to.zero();
    };

    if (r == runs) {
        // the state behind the row
        E *f = (E *)p.fin + b * p.sf_b + d0 * p.sf_d;
        bool same = true;
#pragma unroll
        for (int k = H - 1; k >= 0; --k) {
            const int t = len - H + k;
            if constexpr (SEQ) {
                if (k < H - 1 && len > 0 && t + 1 >= 0) same = same && id(t) == id(t + 1);
            }
            Row<TYPE, N> row;
            if (same) input(t, row);
            else row.zero();
            row.store(f + k * p.sf_k, p.sf_d, 0);
        }
        return;
    }

    float w[K][N], bias[N];
    load_filter<TYPE, K, N>(p, d0, w, bias);
    const int t0 = r * RUN, t1 = min(t0 + RUN, p.seqlen), tv = min(t1, len);
    E *y = (E *)p.y + b * p.sy_b + d0;
    Row<TYPE, N> past[H > 0 ? H : 1];      // inputs of t-H .. t-1
    int fresh = H;                         // tokens in front of t that belong to its sequence, H at most
    if (t0 < tv) {
#pragma unroll
        for (int k = 0; k < H; ++k) input(t0 - H + k, past[k]);
        if constexpr (SEQ) {
            fresh = 0;
            bool same = true;
#pragma unroll
            for (int k = 1; k < H; ++k) {
                same = same && (t0 - k < 0 || id(t0 - k) == id(t0 - k - 1));
                fresh += same ? 1 : 0;
            }
            fresh = H > 0 ? min(fresh + 1, H) : 0;      // of token t0 - 1's sequence: itself and those before it
        }
    }
    constexpr int U = RUN < 8 ? RUN : 8;      // rows requested together
    // Long runs write 256 MB or more, the size of the caches: it would be gone from them when it is read, but push out the input's rows
    // that the next run starts with (4 x 8192 tokens of 5376 channels: 139 us, 146 without the hint).
    constexpr bool PAST = RUN == 32;
    for (int t = t0; t < tv; t += U) {
        Row<TYPE, N> in[U];
        int start[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            start[u] = 0;
            if (t + u < tv) {
                in[u].load(x + (t + u) * p.sx_l);
                if constexpr (SEQ) start[u] = id(t + u) != id(t + u - 1);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= tv) break;
            if constexpr (SEQ) fresh = start[u] ? 0 : fresh;
            Row<TYPE, N> out;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float acc = bias[j] + w[H][j] * to_f32<TYPE>(in[u].e[j]);
#pragma unroll
                for (int k = 0; k < H; ++k) {
                    float a = to_f32<TYPE>(past[k].e[j]);
                    if constexpr (SEQ) a = fresh >= H - k ? a : 0.f;
                    acc = fmaf(w[k][j], a, acc);
                }
                out.e[j] = from_f32<TYPE>(p.silu ? silu(acc) : acc);
            }
            out.template store<PAST>(y + (t + u) * p.sy_l);
#pragma unroll
            for (int k = 0; k + 1 < H; ++k) past[k] = past[k + 1];
            if constexpr (H > 0) past[H - 1] = in[u];
            if constexpr (SEQ) fresh = min(fresh + 1, H);
        }
    }
    Row<TYPE, N> none;
    none.zero();
    for (int t = max(t0, tv); t < t1; ++t) none.store(y + t * p.sy_l);
}

// One token: a thread per 16 bytes of channels of a row.  A set that reaches back leaves the states (and y) of its first channels to
// the set that owns them: it may read them before or after their update.
template <int TYPE, int K, int N>
__global__ void __launch_bounds__(64) conv_step_kernel(const ConvStepParams p, int vectors)
{
    typedef element<TYPE> E;
    constexpr int H = K - 1;
    const uint32_t i = blockIdx.x * 64u + threadIdx.x;
    const int v = (int)(i % (uint32_t)vectors), b = (int)(i / (uint32_t)vectors);
    if (b >= p.batch) return;
    const int d0 = min(v * N, p.dim - N), skip = v * N - d0;
    const int slot = p.slots ? p.slots[b * p.sslots] : b;
    E *y = (E *)p.y + b * p.sy_b + d0;
    Row<TYPE, N> row[K], out;
    if (slot < 0 || slot >= p.n_slots) {
        out.zero();
        out.store(y, 1, skip);
        return;
    }
    E *s = (E *)p.states + slot * p.ss_s + d0 * p.ss_d;
#pragma unroll
    for (int k = 0; k < H; ++k) row[k].load(s + k * p.ss_k, p.ss_d);
    row[H].load((const E *)p.x + b * p.sx_b + d0);
    float w[K][N], bias[N];
    load_filter<TYPE, K, N>(p, d0, w, bias);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float acc = bias[j];
#pragma unroll
        for (int k = 0; k < K; ++k) acc = fmaf(w[k][j], to_f32<TYPE>(row[k].e[j]), acc);
        out.e[j] = from_f32<TYPE>(p.silu ? silu(acc) : acc);
    }
    out.store(y, 1, skip);
#pragma unroll
    for (int k = 0; k < H; ++k) row[k + 1].store(s + k * p.ss_k, p.ss_d, skip);
}

template <int TYPE, int K, bool SEQ, int N>
hipError_t run_conv(const ConvParams &p, hipStream_t s)
{
    const int64_t vectors = (p.dim + N - 1) / N;
    // runs long enough to make little of the rows read twice, short enough for 2048 workgroups (8 per compute unit) to have one
    const bool large = vectors * ((p.seqlen + 31) / 32) * p.batch >= 2048 * 256;
    const int64_t runs = large ? (p.seqlen + 31) / 32 : (p.seqlen + 3) / 4;
    const int64_t blocks = (vectors * (runs + 1) * p.batch + 255) / 256;
    if (blocks * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    if (large) hipLaunchKernelGGL((conv_kernel<TYPE, K, 32, SEQ, N>), dim3((uint32_t)blocks), dim3(256), 0, s, p, (int)vectors, (int)runs);
    else hipLaunchKernelGGL((conv_kernel<TYPE, K, 4, SEQ, N>), dim3((uint32_t)blocks), dim3(256), 0, s, p, (int)vectors, (int)runs);
    return hipGetLastError();
}

template <int TYPE, int K, int N>
hipError_t run_conv_step(const ConvStepParams &p, hipStream_t s)
{
    const int64_t vectors = (p.dim + N - 1) / N, blocks = (vectors * p.batch + 63) / 64;
    if (blocks * 64 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((conv_step_kernel<TYPE, K, N>), dim3((uint32_t)blocks), dim3(64), 0, s, p, (int)vectors);
    return hipGetLastError();
}

template <int K> using taps = std::integral_constant<int, K>;
template <class F> hipError_t of_width(int width, F &&go)
{
    return width == 1 ? go(taps<1>{}) : width == 2 ? go(taps<2>{}) : width == 3 ? go(taps<3>{}) : go(taps<4>{});
}

template <int TYPE>
hipError_t conv_of_type(const ConvParams &p, hipStream_t s)
{
    return of_width(p.width, [&](auto k) {
        constexpr int K = decltype(k)::value, N = Wide<TYPE>::n;
        if (p.dim < N) return run_conv<TYPE, K, true, 1>(p, s);
        return p.seq ? run_conv<TYPE, K, true, N>(p, s) : run_conv<TYPE, K, false, N>(p, s);
    });
}

template <int TYPE>
hipError_t step_of_type(const ConvStepParams &p, hipStream_t s)
{
    return of_width(p.width, [&](auto k) {
        constexpr int K = decltype(k)::value, N = Wide<TYPE>::n;
        return p.dim < N ? run_conv_step<TYPE, K, 1>(p, s) : run_conv_step<TYPE, K, N>(p, s);
    });
}

}  // namespace

hipError_t launch_short_conv(const ConvParams &p, hipStream_t s)
{
    if (p.batch == 0) return hipSuccess;
    if (p.type == DT_F32) return conv_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? conv_of_type<DT_BF16>(p, s) : conv_of_type<DT_F16>(p, s);
}

hipError_t launch_short_conv_step(const ConvStepParams &p, hipStream_t s)
{
    if (p.batch == 0) return hipSuccess;
    if (p.type == DT_F32) return step_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? step_of_type<DT_BF16>(p, s) : step_of_type<DT_F16>(p, s);
}

}  // namespace ssd
