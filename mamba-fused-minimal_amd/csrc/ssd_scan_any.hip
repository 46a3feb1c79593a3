// The selective scan for every type and size, and its single-token form.
//
//   d = limit(softplus(dt + bias));   h = [same sequence] exp(d A) h + d x (x) B;   y = h C + D x;   y *= silu(z)
//
// everything in 32 bits, y rounded once.
//
// Prompts (walk_kernel): 32 tokens at a time.  With cs the running sum of d A inside such a chunk and h the state entering it,
//
//   y_t = e^(cs_t) h C_t + sum_{j <= t} e^(cs_t - cs_j) d_j (C_t . B_j) x_j + D x_t,     y_t *= silu(z_t)
//   h'  = e^(cs_31) h + sum_j e^(cs_31 - cs_j) d_j x_j (x) B_j
//
// all four products on v_mfma_f32_16x16x4_f32, which multiplies fp32 as it is.  A workgroup of four waves takes 64 rows of a head, a
// wave 16 of them with all state columns in its accumulators: their layout is that of a right operand too, so the state is
// multiplied from where it is.  x, B and C of a chunk come through LDS in 32 bits; the scores are made once per workgroup.  Where
// batch x heads are too few for the card, the row is cut into segments: a first launch computes what each segment but the last adds to a
// state of zero, and a second one starts each from the state that enters it: few segments read what those in front of them add, for
// more launch_scan_join puts them together in between.
// fp32, 2 x 1900 tokens of 15 heads of 48 x 96 with gate and states: 41 us, and 19 and 6 for the launches in front (token by token on the
// vector ALU 480 in all).  The matrix instructions are 9 us of the 41: four chunks to a segment, and in each a workgroup waits for its
// loads, its barriers and its exponentials in turn, with one other beside it.  Where there are heads enough the matrix instructions
// take two thirds of the time: 4 x 3001 tokens of 64 heads of 64 x 128 in fp16, one segment, 518 us.
//
// A decay across tokens is the exponential of a difference of sums, so the sums are made in 64 bits and kept as two floats; a token
// that lets nothing pass (below e^-120 = 0) counts as e^-120, or the sums behind it would lose what their differences need.  A product with
// what a mask leaves out would be 0 x NaN: chunks that hold values of no use to a sum (infinities, NaN, more than 1e15) or a growing
// state (d A > 1) are walked token by token.
//
// Single tokens (step_kernel): the states are read and written once, 8 bytes per element for 5 operations: HBM bound (61 rows of 80 heads
// of 64 x 128: 66 us, 4.9 TB/s of the 5.2 that a copy reaches).  Lanes share a row's columns, 16 bytes each, and every load of a workgroup is
// in flight before the first is used.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

constexpr int T = 32;                    // tokens of a chunk
constexpr int ROWS = 64, PX = ROWS + 4;  // rows of a workgroup; floats between tokens of x in LDS
constexpr int PS = T + 4;                // and between rows of the scores.  Pitches are 4 x odd: 16 rows of 16 bytes then cover all 64 banks
constexpr float kLarge = 1e15f;

// Four consecutive elements as they are in memory, from a row of `count`: the ones at n, or the row's last four where those would pass
// its end (of rows shorter than four the last one repeated).
template <int TYPE> struct Quad {
    typedef element<TYPE> E;
    typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t half4;
    typedef std::conditional_t<sizeof(E) == 4, wide4, half4> raw;
    struct Pack { E e[4]; } q;
    __device__ __forceinline__ void load(const E *row, int n, int count)
    {
        if (count >= 4) q = __builtin_bit_cast(Pack, *(const raw *)(row + min(n, count - 4)));
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) q.e[j] = row[min(n + j, count - 1)];
    }
    __device__ __forceinline__ f32x4 values() const
    {
        f32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = to_f32<TYPE>(q.e[j]);
        return f;
    }
    // largest magnitudes so far, as bits: those of an infinity or a NaN are larger still
    typedef __attribute__((ext_vector_type(sizeof(E) == 4 ? 4 : 2))) uint32_t words;
    typedef __attribute__((ext_vector_type(4))) uint16_t u16x4;
    typedef std::conditional_t<sizeof(E) == 4, u32x4, u16x4> Most;
    __device__ __forceinline__ void most(Most &m) const
    {
        const words w = __builtin_bit_cast(words, q) & (sizeof(E) == 4 ? 0x7fffffffu : 0x7fff7fffu);
        m = __builtin_elementwise_max(m, __builtin_bit_cast(Most, w));
    }
    static __device__ __forceinline__ bool large(const Most &m)
    {
        constexpr uint32_t limit = TYPE == DT_F32 ? 0x58635fa9u : TYPE == DT_BF16 ? 0x5863u : 0x7c00u;      // 1e15; infinity
        return m[0] >= limit || m[1] >= limit || m[2] >= limit || m[3] >= limit;
    }
    // the elements at n, zeros behind the row
    __device__ __forceinline__ f32x4 at(int n, int count) const
    {
        asm volatile("" : "+v"(n));      // or the masks of all elements are made once and kept in scalar registers
        f32x4 f = values();
        if (count >= 4 && count % 4) {
            const int skip = n - min(n, count - 4);
            f = skip & 1 ? f32x4{f[1], f[2], f[3], 0.f} : f;
            f = skip & 2 ? f32x4{f[2], f[3], 0.f, 0.f} : f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = n + j < count ? f[j] : 0.f;
        return f;
    }
};

__device__ __forceinline__ f32x4 product(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// the same address in global memory, in vector registers
template <class E> __device__ __forceinline__ E *in_vector(E *p)
{
    uint64_t at = (uint64_t)p;
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(at));
#endif
    return (E *)(__attribute__((address_space(1))) E *)at;
}

// floats of LDS
constexpr int walk_words(int NT, bool out) { return (out ? 2 : 1) * T * (16 * NT + 4) + T * PX + (out ? T * PS : 0) + 2 * 6 * T + 4; }

// NT: tiles of 16 state columns.  OUT: write y (otherwise only what the segment adds and the factor on what enters it).
template <int TYPE, int NT, bool OUT>
__global__ void __launch_bounds__(256, NT == 16 ? 1 : 2) walk_kernel(const SelScanParams p, int row_blocks)
{
    typedef element<TYPE> E;
    constexpr int NP = 16 * NT, PB = NP + 4;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *const Bt = lds, *const Ct = Bt + T * PB, *const xt = Ct + (OUT ? T * PB : 0), *const St = xt + T * PX;
    float *const records = St + (OUT ? T * PS : 0);      // of the steps of two chunks
    int *const bad = (int *)(records + 2 * 6 * T);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
    uint32_t id = blockIdx.x;
    const int rb = (int)(id % (uint32_t)row_blocks); id /= (uint32_t)row_blocks;
    const int h = (int)(id % (uint32_t)p.nheads); id /= (uint32_t)p.nheads;
    const int seg = (int)(id % (uint32_t)p.segments), b = (int)(id / (uint32_t)p.segments);
    if (!OUT && seg == p.segments - 1) return;                                 // nothing enters a segment behind the last
    const int P = p.headdim - rb * ROWS, N = p.dstate, r = 16 * wave + i;      // rows left; this lane's
    const bool wave_live = 16 * wave < P, live = r < P;
    const int len = row_tokens(p.len, p.slen, b, p.seqlen);
    const int t0 = seg * p.segment_tokens, t_end = min(t0 + p.segment_tokens, p.seqlen), t1 = min(t_end, len);
    const E *x = (const E *)p.x + b * p.sx_b + h * p.sx_h + rb * ROWS, *z = p.z ? (const E *)p.z + b * p.sz_b + h * p.sz_h + rb * ROWS : nullptr;
    const int group = h / (p.nheads / p.ngroups);
    const E *Bg = (const E *)p.B + b * p.sB_b + group * p.sB_g, *Cg = (const E *)p.C + b * p.sC_b + group * p.sC_g;
    E *y = (E *)p.y + b * p.sy_b + h * p.sy_h + rb * ROWS;
    // in vector registers: there are not enough scalar ones for all that is the same in a workgroup
    x = in_vector(x), z = in_vector(z), Bg = in_vector(Bg), Cg = in_vector(Cg), y = in_vector(y);
    // The steps of a chunk, by the last wave: it has no scores to make
    struct Steps { float *d, *hi, *lo, *weight, *keep; int *start; };
    auto record = [&](int parity) {
        float *at = records + parity * 6 * T;
        return Steps{at, at + T, at + 2 * T, at + 3 * T, at + 4 * T, (int *)(at + 5 * T)};
    };
    uint32_t dt_bits = 0;
    int ids[2] = {0, 0};
    auto request_steps = [&](int t) {
        const int tok = min(t + (lane & 31), t1 - 1);
        const int64_t at = b * p.sdt_b + tok * p.sdt_l + h * p.sdt_h;
        if (p.dt_type == DT_F32) dt_bits = ((const uint32_t *)p.dt)[at];
        else dt_bits = ((const uint16_t *)p.dt)[at];
        if (p.seq) {
            ids[0] = p.seq[b * p.sq_b + tok * p.sq_l];
            ids[1] = tok > 0 ? p.seq[b * p.sq_b + (tok - 1) * p.sq_l] : 0;
        }
    };
    // A chunk's inputs, requested while the one in front of it is computed with
    // (eight threads to a token, 16 bytes of every 32 elements each)
    constexpr int BQ = (NP + 31) / 32, XQ = ROWS / 32;
    const int token = tid >> 3;
    Quad<TYPE> qB[BQ], qC[BQ], qx[XQ];
    E qz[2][4];
    auto request = [&](int t) {
        const int last = min(T, t1 - t) - 1, tok = t + min(token, last);
        // (opaque, here and below: what is the same for all chunks would be kept in registers, of which there are too few)
        int column = 4 * (tid & 7);
        int64_t pitch = p.sz_l;
        asm volatile("" : "+v"(column), "+s"(pitch));
        const E *const rB = Bg + tok * p.sB_l, *const rC = Cg + tok * p.sC_l, *const rx = x + tok * p.sx_l;
#pragma unroll
        for (int k = 0; k < BQ; ++k) {
            qB[k].load(rB, column + 32 * k, N);
            if constexpr (OUT) qC[k].load(rC, column + 32 * k, N);
        }
#pragma unroll
        for (int k = 0; k < XQ; ++k) qx[k].load(rx, column + 32 * k, P);
        if (OUT && p.z) {
            const E *const rz = z + min(r, P - 1);
            if (last == T - 1) {
                const E *at = rz + (t + 4 * g) * pitch;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) qz[u][j] = at[(16 * u + j) * pitch];
            } else
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) qz[u][j] = rz[(t + min(16 * u + 4 * g + j, last)) * p.sz_l];
        }
    };
    // all that the first chunk needs is on its way before the first of it is waited for
    if (wave == 3 && t0 < t1) request_steps(t0);
    if (t0 < t1) request(t0);

    // s[v][j] = h[row r][column 16 v + 4 g + j]
    f32x4 s[NT];
    const int64_t plane = ((int64_t)b * p.nheads + h) * p.segments + seg;
    float *ws = p.ws_states + plane * p.headdim * N + (int64_t)rb * ROWS * N;
    auto from = [&](auto type, const void *state, int64_t first) {
        typedef Quad<decltype(type)::value> Q;
#pragma unroll
        for (int v = 0; v < NT; ++v) {
            Q q;
            q.load((const typename Q::E *)state + (live ? first : 0), 16 * v + 4 * g, N);
            s[v] = q.at(16 * v + 4 * g, live ? N : 0);
        }
    };
    if (OUT && p.joined) from(std::integral_constant<int, DT_F32>{}, ws, (int64_t)r * N);
    else if (OUT && p.init) {
        const int64_t first = b * p.si_b + h * p.si_h + (rb * ROWS + r) * p.si_p;
        if (p.init_type == DT_F32) from(std::integral_constant<int, DT_F32>{}, p.init, first);
        else if (p.init_type == DT_BF16) from(std::integral_constant<int, DT_BF16>{}, p.init, first);
        else from(std::integral_constant<int, DT_F16>{}, p.init, first);
    } else
#pragma unroll
        for (int v = 0; v < NT; ++v) s[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (OUT && !p.joined)
        // few segments: what enters this one from what those in front of it add
        for (int k = 0; k < seg; ++k) {
            const float f = p.ws_decay[plane - seg + k];
            const float *const add = ws + (k - seg) * (int64_t)p.headdim * N + (live ? (int64_t)r * N : 0);
#pragma unroll
            for (int v = 0; v < NT; ++v) {
                Quad<DT_F32> q;
                q.load(add, 16 * v + 4 * g, N);
                const f32x4 more = q.at(16 * v + 4 * g, live ? N : 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[v][j] = f < 0.f ? more[j] : fmaf(f, s[v][j], more[j]);
            }
        }
    const float D = OUT && p.D && live ? load_as_f32(p.D, h * p.sD_h + (rb * ROWS + r) * p.sD_p, p.D_type) : 0.f;
    float through = 1.f;

    const float A = load_as_f32(p.A, h * p.sA, p.A_type);
    const float bias = p.delta.bias ? load_as_f32(p.delta.bias, h * p.delta.sbias, p.delta.bias_type) : 0.f;

    // (from the requests in front of it, into a record; what it finds is out of the ordinary goes to `bad`)
    auto make_steps = [&](int t, int parity) {
        // (the second half of the wave repeats the first)
        const int at = lane & 31, n_t = min(T, t1 - t);
        const Steps to = record(parity);
        const float raw = p.dt_type == DT_F32 ? __builtin_bit_cast(float, dt_bits) : p.dt_type == DT_BF16 ? bf16_bits_to_f32((uint16_t)dt_bits)
                                              : (float)__builtin_bit_cast(_Float16, (uint16_t)dt_bits);
        const bool starts = at < n_t && ids[0] != ids[1];
        const float d = at < n_t ? delta_of(p.delta, raw + bias) : 0.f, a = d * A;
        double sum = a < -120.f ? -120. : (double)d * (double)A;
#pragma unroll
        for (int k = 1; k < T; k *= 2) {
            const double other = __shfl_up(sum, k, 32);
            sum += at >= k ? other : 0.;
        }
        const uint32_t from = (uint32_t)__ballot(starts), upto = from & (0xffffffffu >> (31 - at));
        const double end = __shfl(sum, 31, 32);
        const bool off = __any(!(fabsf(d) < kLarge) || !(a <= 1.f));
        if (lane < 32) {
            const float hi = (float)sum;
            to.d[at] = d;
            to.hi[at] = hi;
            to.lo[at] = (float)(sum - (double)hi);
            to.weight[at] = at >= (from ? 31 - __builtin_clz(from) : 0) ? d * __expf((float)(end - sum)) : 0.f;
            to.keep[at] = upto ? -1.f : not_zero(__expf(hi));      // of the state in front of the chunk; negative: another sequence's
            to.start[at] = upto ? 31 - __builtin_clz(upto) : -1;
        }
        if (lane == 0) bad[parity] = off;
    };
    if (wave == 3 && t0 < t1) {
        make_steps(t0, 0);
        request_steps(t0 + T);
    }

    int parity = 0;
    for (int t = t0; t < t1; t += T, parity ^= 1) {
        const int n_t = min(T, t1 - t);
        __syncthreads();
        // whole chunks of whole tiles are what they are; others have zeros for tokens and columns that are not there
        const bool whole = n_t == T, whole_N = whole && N == NP, whole_P = whole && P >= ROWS;
        typename Quad<TYPE>::Most most = {0, 0, 0, 0};
        int column = 4 * (tid & 7);
        asm volatile("" : "+v"(column));
        auto place = [&](float *to, const Quad<TYPE> &q, int n, int count, bool as_is) {
            f32x4 f = q.values();
            if (!as_is) {
                f = q.at(n, count);
                f = token < n_t ? f : f32x4{0.f, 0.f, 0.f, 0.f};
            }
            q.most(most);
            *(f32x4 *)to = f;
        };
        if (NP >= 32 || column < NP)
#pragma unroll
            for (int k = 0; k < BQ; ++k) {
                place(&Bt[token * PB + column + 32 * k], qB[k], column + 32 * k, N, whole_N);
                if constexpr (OUT) place(&Ct[token * PB + column + 32 * k], qC[k], column + 32 * k, N, whole_N);
            }
#pragma unroll
        for (int k = 0; k < XQ; ++k) place(&xt[token * PX + column + 32 * k], qx[k], column + 32 * k, P, whole_P);
        float gate[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) gate[u][j] = OUT && p.z ? to_f32<TYPE>(qz[u][j]) : 0.f;
        if (t + T < t1) request(t + T);
        if (Quad<TYPE>::large(most)) bad[parity] = 1;
        __syncthreads();
        const bool slow = __builtin_amdgcn_readfirstlane(bad[parity]) != 0;
        const Steps rec = record(parity);
        // behind what the other waves meanwhile do with this chunk, or in front of it
        auto next_steps = [&] {
            if (wave == 3 && t + T < t1) {
                make_steps(t + T, parity ^ 1);
                request_steps(t + 2 * T);
            }
        };
        auto give = [&](int tt, float v, float gated) {
            asm volatile("" : "+v"(tt));      // (masks again)
            if (!live || tt >= n_t) return;
            v *= p.z ? silu(gated) : 1.f;
            y[(t + tt) * p.sy_l + r] = from_f32<TYPE>(v);
        };
        if (slow) {
            next_steps();
            for (int tt = 0; tt < n_t; ++tt) {
                const bool starts = rec.start[tt] == tt;
                const float d = rec.d[tt], e = __expf(d * A), xv = xt[tt * PX + r], dx = d * xv;
                through = starts || through < 0.f ? -1.f : through * e;
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < NT; ++v) {
                    const f32x4 Bv = *(const f32x4 *)&Bt[tt * PB + 16 * v + 4 * g];
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[v][j] = fmaf(starts ? 0.f : s[v][j], starts ? 0.f : e, dx * Bv[j]);
                    if constexpr (OUT) {
                        const f32x4 Cv = *(const f32x4 *)&Ct[tt * PB + 16 * v + 4 * g];
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum = fmaf(s[v][j], Cv[j], sum);
                    }
                }
                if constexpr (OUT) {
                    sum += __shfl_xor(sum, 16);
                    sum += __shfl_xor(sum, 32);
                    if (g == 0) give(tt, p.D ? fmaf(D, xv, sum) : sum, p.z && live ? to_f32<TYPE>(z[(t + tt) * p.sz_l + r]) : 0.f);
                }
            }
            if constexpr (OUT) __syncthreads();      // as on the other way
            continue;
        }
        f32x4 out[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        next_steps();
        if constexpr (OUT) {
            // scores: tiles of 16 x 16 tokens (0, 0), (1, 0), (1, 1), one to a wave
            if (wave < 3) {
                const int tt = wave > 0 ? 16 : 0, jt = wave > 1 ? 16 : 0;
                f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int v = 0; v < NT; ++v) {
                    const f32x4 c = *(const f32x4 *)&Ct[(tt + i) * PB + 16 * v + 4 * g], f = *(const f32x4 *)&Bt[(jt + i) * PB + 16 * v + 4 * g];
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[j & 1] = product(c[j], f[j], sc[j & 1]);
                }
                const int at = jt + i;
                const float hi = rec.hi[at], lo = rec.lo[at], d = rec.d[at];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int to = tt + 4 * g + j;
                    const float f = (sc[0][j] + sc[1][j]) * (__expf((rec.hi[to] - hi) + (rec.lo[to] - lo)) * d);
                    St[to * PS + at] = at <= to && at >= rec.start[to] ? f : 0.f;
                }
            }
            if (wave_live) {
#pragma unroll
                for (int v = 0; v < NT; ++v) {
                    const f32x4 c0 = *(const f32x4 *)&Ct[i * PB + 16 * v + 4 * g], c1 = *(const f32x4 *)&Ct[(16 + i) * PB + 16 * v + 4 * g];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        out[0] = product(c0[j], s[v][j], out[0]);
                        out[1] = product(c1[j], s[v][j], out[1]);
                    }
                }
            }
            __syncthreads();
        }
        const float end = rec.keep[T - 1];
        through = end < 0.f || through < 0.f ? -1.f : through * end;
        if (!wave_live) continue;
        f32x4 xv[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) xv[u][j] = xt[(16 * u + 4 * g + j) * PX + r];
        if constexpr (OUT) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f32x4 k = *(const f32x4 *)&rec.keep[16 * u + 4 * g];
#pragma unroll
                for (int j = 0; j < 4; ++j) out[u][j] = k[j] < 0.f ? 0.f : out[u][j] * k[j];
            }
            const f32x4 s00 = *(const f32x4 *)&St[i * PS + 4 * g], s10 = *(const f32x4 *)&St[(16 + i) * PS + 4 * g],
                        s11 = *(const f32x4 *)&St[(16 + i) * PS + 16 + 4 * g];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                out[0] = product(s00[j], xv[0][j], out[0]);
                out[1] = product(s10[j], xv[0][j], out[1]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) out[1] = product(s11[j], xv[1][j], out[1]);
        }
        f32x4 xw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const f32x4 w = *(const f32x4 *)&rec.weight[16 * u + 4 * g];
#pragma unroll
            for (int j = 0; j < 4; ++j) xw[u][j] = xv[u][j] * w[j];
        }
#pragma unroll
        for (int v = 0; v < NT; ++v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[v][j] = end < 0.f ? 0.f : s[v][j] * end;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[v] = product(Bt[(16 * u + 4 * g + j) * PB + 16 * v + i], xw[u][j], s[v]);
        }
        if (OUT && whole) {
            if (live) {
                int64_t pitch = p.sy_l;
                asm volatile("" : "+s"(pitch));
                E *const at = y + (t + 4 * g) * pitch + r;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v = p.D ? fmaf(D, xv[u][j], out[u][j]) : out[u][j];
                        v *= p.z ? silu(gate[u][j]) : 1.f;
                        at[(16 * u + j) * pitch] = from_f32<TYPE>(v);
                    }
            }
        } else if constexpr (OUT)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) give(16 * u + 4 * g + j, p.D ? fmaf(D, xv[u][j], out[u][j]) : out[u][j], gate[u][j]);
    }
    if constexpr (OUT) {
        for (int t = max(t0, t1) + tid / ROWS; t < t_end; t += 256 / ROWS)
            if (tid % ROWS < P) y[t * p.sy_l + tid % ROWS] = from_f32<TYPE>(0.f);
    }
    if (!OUT || seg == p.segments - 1) {
        float *to = OUT ? p.fin + b * p.sf_b + h * p.sf_h + (rb * ROWS + r) * p.sf_p : ws + (int64_t)r * N;
        int q = 4 * g;
        asm volatile("" : "+v"(q));      // or the compiler keeps every element's mask from the loads above
        if (live && N % 4 == 0) {
#pragma unroll
            for (int v = 0; v < NT; ++v)
                if (16 * v + q < N) *(wide4 *)(to + 16 * v + q) = __builtin_bit_cast(wide4, s[v]);
        } else if (live) {
#pragma unroll
        for (int v = 0; v < NT; ++v)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (16 * v + q + j < N) to[16 * v + q + j] = s[v][j];
        }
    }
    if (!OUT && tid == 0 && rb == 0) p.ws_decay[plane] = through < 0.f ? through : not_zero(through);
}

// ws_states of a (row, head): what each segment adds -> what enters it.  A thread per state element walks the segments; the
// loads of sixteen are in flight together.
__global__ void __launch_bounds__(256) join_kernel(const SelScanParams p, int plane_blocks)
{
    const int plane = p.headdim * p.dstate, S = p.segments;
    const uint32_t bh = blockIdx.x / (uint32_t)plane_blocks;
    const int i = (int)(blockIdx.x % (uint32_t)plane_blocks) * 256 + threadIdx.x;
    if (i >= plane) return;
    const int b = (int)(bh / (uint32_t)p.nheads), h = (int)(bh % (uint32_t)p.nheads);
    float *ws = p.ws_states + (int64_t)bh * S * plane + i;
    const float *decay = p.ws_decay + (int64_t)bh * S;
    float in = 0.f;
    if (p.init) in = load_as_f32(p.init, b * p.si_b + h * p.si_h + (i / p.dstate) * p.si_p + i % p.dstate, p.init_type);
    for (int s0 = 0; s0 < S; s0 += 16) {
        float add[16], f[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const int k = min(s0 + u, S - 2);      // (the last adds to nothing)
            add[u] = ws[(int64_t)k * plane];
            f[u] = decay[k];
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            if (s0 + u >= S) break;
            ws[(int64_t)(s0 + u) * plane] = in;
            in = f[u] < 0.f ? add[u] : fmaf(f[u], in, add[u]);
        }
    }
}

// A workgroup of four waves takes 4 * RPW rows of a head.  LANES lanes share a row, COLS columns each (4: 16 bytes at a time).
template <int TYPE, int LANES, int COLS, int ROUNDS, bool PAST>
__global__ void __launch_bounds__(256) step_kernel(const SelStepParams p, int row_blocks)
{
    typedef element<TYPE> E;
    constexpr int RW = 64 / LANES;                      // rows of a wave at a time
    constexpr int ROWS = 4 * RW * ROUNDS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % LANES * COLS;
    uint32_t i = blockIdx.x;
    const int rb = (int)(i % (uint32_t)row_blocks); i /= (uint32_t)row_blocks;
    const int h = (int)(i % (uint32_t)p.nheads), b = (int)(i / (uint32_t)p.nheads);
    const int P = p.headdim, N = p.dstate, g = h / (p.nheads / p.ngroups);
    const int slot = p.slots ? p.slots[b * p.sslots] : b;
    E *y = (E *)p.y + b * p.sy_b + h * p.sy_h;
    if (slot < 0 || slot >= p.n_slots) {
        for (int r = threadIdx.x; r < ROWS; r += 256)
            if (rb * ROWS + r < P) y[rb * ROWS + r] = from_f32<TYPE>(0.f);
        return;
    }
    float *state = p.states + slot * p.ss_s + h * p.ss_h;
    const int r0 = rb * ROWS + wave * (RW * ROUNDS) + lane / LANES;
    const E *x = (const E *)p.x + b * p.sx_b + h * p.sx_h, *z = p.z ? (const E *)p.z + b * p.sz_b + h * p.sz_h : nullptr;
    const E *B = (const E *)p.B + b * p.sB_b + g * p.sB_g, *C = (const E *)p.C + b * p.sC_b + g * p.sC_g;
    const float A = load_as_f32(p.A, h * p.sA, p.A_type);
    float d = load_as_f32(p.dt, b * p.sdt_b + h * p.sdt_h, p.dt_type);
    if (p.delta.bias) d += load_as_f32(p.delta.bias, h * p.delta.sbias, p.delta.bias_type);

    float acc[ROUNDS], xv[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        acc[r] = 0.f;
        const int row = r0 + r * RW;
        xv[r] = row < P ? to_f32<TYPE>(x[row]) : 0.f;
    }
    // COLS = 4: one pass, dstate = 4 LANES at most and a multiple of 4, rows at 16 bytes.  COLS = 1: any dstate, 64 columns at a time.
    for (int n0 = 0; n0 < (COLS == 4 ? 1 : N); n0 += LANES) {
        const int n = COLS == 4 ? col : n0 + col;
        const bool there = n < N;
        float s[ROUNDS][COLS], Bv[COLS], Cv[COLS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int row = r0 + r * RW;
            if (there && row < P) {
                if constexpr (COLS == 4) {
                    const f32x4 *const from = (const f32x4 *)&state[row * p.ss_p + n];
                    const f32x4 q = PAST ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[r][j] = q[j];
                } else s[r][0] = state[row * p.ss_p + n];
            }
        }
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
            Bv[j] = there ? to_f32<TYPE>(B[n + j]) : 0.f;
            Cv[j] = there ? to_f32<TYPE>(C[n + j]) : 0.f;
        }
        const float delta = delta_of(p.delta, d), keep = __expf(delta * A);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int row = r0 + r * RW;
            if (there && row < P) {
                const float dx = delta * xv[r];
#pragma unroll
                for (int j = 0; j < COLS; ++j) {
                    s[r][j] = fmaf(s[r][j], keep, dx * Bv[j]);
                    acc[r] = fmaf(s[r][j], Cv[j], acc[r]);
                }
                if constexpr (COLS == 4) {
                    const f32x4 q = {s[r][0], s[r][1], s[r][2], s[r][3]};
                    f32x4 *const to = (f32x4 *)&state[row * p.ss_p + n];
                    if constexpr (PAST) __builtin_nontemporal_store(q, to);
                    else *to = q;
                }
                else state[row * p.ss_p + n] = s[r][0];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int row = r0 + r * RW;
        float v = group_sum<LANES>(acc[r]);
        if (lane % LANES == 0 && row < P) {
            if (p.D) v = fmaf(load_as_f32(p.D, h * p.sD_h + row * p.sD_p, p.D_type), xv[r], v);
            if (z) v *= silu(to_f32<TYPE>(z[row]));
            y[row] = from_f32<TYPE>(v);
        }
    }
}

template <int TYPE, int NT>
hipError_t run_walk(SelScanParams p, hipStream_t s)
{
    const int row_blocks = (p.headdim + ROWS - 1) / ROWS;
    const int64_t blocks = (int64_t)row_blocks * p.nheads * p.segments * p.batch;
    if (blocks * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    constexpr int lds_add = 4 * walk_words(NT, false), lds_out = 4 * walk_words(NT, true);
    static std::atomic<uint64_t> done[2];
    hipError_t e = ensure_dynamic_lds((const void *)walk_kernel<TYPE, NT, true>, lds_out, done[0]);
    if (e == hipSuccess) e = ensure_dynamic_lds((const void *)walk_kernel<TYPE, NT, false>, lds_add, done[1]);
    if (e != hipSuccess) return e;
    if (p.segments > 1) {
        hipLaunchKernelGGL((walk_kernel<TYPE, NT, false>), dim3((uint32_t)blocks), dim3(256), lds_add, s, p, row_blocks);
        e = hipGetLastError();
        // few segments: who enters one reads what those in front of it add, in less time than a launch in between takes
        p.joined = p.segments > 4;
        if (e == hipSuccess && p.joined) e = launch_scan_join(p, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((walk_kernel<TYPE, NT, true>), dim3((uint32_t)blocks), dim3(256), lds_out, s, p, row_blocks);
    return hipGetLastError();
}

template <int TYPE>
hipError_t walk_of_type(const SelScanParams &p, hipStream_t s)
{
    if (p.dstate <= 16) return run_walk<TYPE, 1>(p, s);
    if (p.dstate <= 32) return run_walk<TYPE, 2>(p, s);
    if (p.dstate <= 64) return run_walk<TYPE, 4>(p, s);
    if (p.dstate <= 96) return run_walk<TYPE, 6>(p, s);
    return p.dstate <= 128 ? run_walk<TYPE, 8>(p, s) : run_walk<TYPE, 16>(p, s);
}

template <int TYPE, int LANES, int COLS, int ROUNDS, bool PAST = false>
hipError_t run_step(const SelStepParams &p, hipStream_t s)
{
    constexpr int ROWS = 4 * (64 / LANES) * ROUNDS;
    const int row_blocks = (p.headdim + ROWS - 1) / ROWS;
    const int64_t blocks = (int64_t)row_blocks * p.nheads * p.batch;
    if (blocks * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((step_kernel<TYPE, LANES, COLS, ROUNDS, PAST>), dim3((uint32_t)blocks), dim3(256), 0, s, p, row_blocks);
    return hipGetLastError();
}

template <int TYPE>
hipError_t step_of_type(const SelStepParams &p, hipStream_t s)
{
    const bool wide = p.dstate % 4 == 0 && p.dstate <= 256 && (p.ss_s | p.ss_h | p.ss_p) % 4 == 0 && ((uintptr_t)p.states & 15) == 0;
    if (!wide) return run_step<TYPE, 64, 1, 4>(p, s);
    // Few rows in all (16 MB of states): smaller workgroups, so that more compute units have one.  More: the states go past the caches,
    // as nothing reads them before the next token (61 rows of 80 heads of 64 x 128, 320 MB of traffic: 65.7 us, 4.9 TB/s; 87 without the
    // hint; with half or twice the rows per workgroup 87 and 67).
    const bool few = (int64_t)p.batch * p.nheads * p.headdim * p.dstate <= 1 << 22;
    if (p.dstate <= 16) return run_step<TYPE, 4, 4, 1>(p, s);
    if (p.dstate <= 64) return few ? run_step<TYPE, 16, 4, 1>(p, s) : run_step<TYPE, 16, 4, 4, true>(p, s);
    if (p.dstate <= 128) return few ? run_step<TYPE, 32, 4, 2>(p, s) : run_step<TYPE, 32, 4, 4, true>(p, s);
    return few ? run_step<TYPE, 64, 4, 4>(p, s) : run_step<TYPE, 64, 4, 4, true>(p, s);
}

}  // namespace

hipError_t launch_scan_join(const SelScanParams &p, hipStream_t s)
{
    const int64_t plane_blocks = ((int64_t)p.headdim * p.dstate + 255) / 256, blocks = plane_blocks * p.nheads * p.batch;
    if (blocks * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(join_kernel, dim3((uint32_t)blocks), dim3(256), 0, s, p, (int)plane_blocks);
    return hipGetLastError();
}

hipError_t launch_scan_any(const SelScanParams &p, hipStream_t s)
{
    if (p.type == DT_F32) return walk_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? walk_of_type<DT_BF16>(p, s) : walk_of_type<DT_F16>(p, s);
}

hipError_t launch_scan_step(const SelStepParams &p, hipStream_t s)
{
    if (p.batch == 0) return hipSuccess;
    if (p.type == DT_F32) return step_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? step_of_type<DT_BF16>(p, s) : step_of_type<DT_F16>(p, s);
}

}  // namespace ssd
