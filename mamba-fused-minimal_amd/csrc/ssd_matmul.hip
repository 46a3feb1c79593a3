// Matrix product in 8-bit integers with a scale per token and per channel:
//
//   out[m, n] = sa[m] sw[n] sum_k a[m, k] w[n, k]  (+ bias[n])
//
// Sums are 32-bit integers and exact (|sum| < 2^31 for K <= 131071), so the order in which parts are added does not matter.  What follows
// is fp32, each step rounded: the conversion (of sums beyond 2^24, possible from K = 1025 on), both scales, the bias; then one rounding to the
// type of out.  Weights are rows of K, as the matrix instructions take both operands.
//
// tile_kernel: workgroups of four waves take (64 TM) tokens x (64 TN) channels, each wave (32 TM) x (32 TN) of them on
// v_mfma_i32_32x32x32_i8.  Operands go straight from memory into an LDS ring of four steps of 64 bytes of K; a step's second half is
// read into registers while the first half's products run, and the next step's first half while the second's run.
// The requests of a step and the reads of the next half stand between the products, one or two to a product, so that the matrix
// unit runs on while they are issued.  Bound by the matrix instructions, whose clock falls under this load: 8192 x 10576 x 2560 to
// bf16 takes 267 us, 1.66e15 integer operations a second (a product of 8192^3 on this card: 2.3e15); 40 steps of 1540 cycles to a
// tile of 256 x 256, 1024 of them the instructions', and 22000 around the loop.
// odd_tile_kernel: the same tiles for rows of any alignment, whose operands come through registers (4096 x 10576 x 2561 to bf16 245 us, with
// K = 2560 in tile_kernel 130: a load that begins at an odd byte is several).
// direct_kernel: any size and alignment, few tokens: the waves of a workgroup share a (16 MT) x (16 NT) tile by K, load their
// operands from memory into registers and add their sums through LDS.  Few tokens are bound by the weights' bytes and the launch:
// 1 x 10576 x 2560 takes 6.9 us, 27 MB of weights at 4.0 TB/s.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;
typedef __attribute__((ext_vector_type(4), aligned(1))) int any4;

// four consecutive results of a row, the first at channel n
template <int TYPE> __device__ __forceinline__ void store4(const MatmulParams &p, int64_t m, int n, const float (&v)[4])
{
    typedef element<TYPE> E;
    E *o = (E *)p.out + m * p.so_m + n;
    if (n + 4 <= p.N) {
        if constexpr (sizeof(E) == 4) *(wide4 *)o = __builtin_bit_cast(wide4, f32x4{v[0], v[1], v[2], v[3]});
        else {
            typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t raw;
            struct { E e[4]; } q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q.e[j] = from_f32<TYPE>(v[j]);
            *(raw *)o = __builtin_bit_cast(raw, q);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) o[j] = from_f32<TYPE>(v[j]);
    }
}

// ---- few tokens, odd sizes -----------------------------------------------------------------------------------------

// 16 bytes of a row of K at byte k; what lies behind the row's end is zero
__device__ __forceinline__ i32x4 row_tail(const int8_t *row, int k, int K)
{
    if (k + 16 <= K) return __builtin_bit_cast(i32x4, *(const any4 *)(row + k));
    i32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (k + j < K) v[j / 4] |= (int)((uint32_t)(uint8_t)row[k + j] << (8 * (j % 4)));
    return v;
}

// A lane's operands of 128 bytes of K are 32 consecutive bytes of its row: the four lanes of a row read a whole cache line, and the
// order of K inside a product is the same for both operands.
template <int TYPE, int MT, int NT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) direct_kernel(const MatmulParams p, int tiles_m)
{
    extern __shared__ __attribute__((aligned(16))) i32x4 sums[];      // [tile][wave][lane]
    // (known to be the same in all lanes: matrix instructions run whatever the execution mask, so they stand behind branches only)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int m0 = (int)(blockIdx.x % (uint32_t)tiles_m) * 16 * MT, n0 = (int)(blockIdx.x / (uint32_t)tiles_m) * 16 * NT;
    const int8_t *a[MT], *w[NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = p.a + (int64_t)min(m0 + 16 * t + i, p.M - 1) * p.sa_m;
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = p.w + (int64_t)min(n0 + 16 * t + i, p.N - 1) * p.sw_n;
    i32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = i32x4{0, 0, 0, 0};

    auto products = [&](const i32x4 (&av)[MT][2], const i32x4 (&wv)[NT][2]) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < MT; ++u)
                    acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[t][half], av[u][half], acc[t][u], 0, 0, 0);
    };
    const int whole = p.K / 128, steps = (p.K + 127) / 128;
    constexpr int U = MT * NT >= 4 ? 1 : 4;      // steps requested together
    int c = wave;
    for (; c + (U - 1) * WAVES < whole; c += U * WAVES) {
        i32x4 av[U][MT][2], wv[U][NT][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int k = (c + u * WAVES) * 128 + g * 32 + half * 16;
#pragma unroll
                for (int t = 0; t < NT; ++t) wv[u][t][half] = __builtin_bit_cast(i32x4, *(const any4 *)(w[t] + k));
#pragma unroll
                for (int t = 0; t < MT; ++t) av[u][t][half] = __builtin_bit_cast(i32x4, *(const any4 *)(a[t] + k));
            }
#pragma unroll
        for (int u = 0; u < U; ++u) products(av[u], wv[u]);
    }
    if (U > 1 && c < whole) {                    // fewer than U are left: those, together too
        i32x4 av[U][MT][2], wv[U][NT][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int k = (c + u * WAVES) * 128 + g * 32 + half * 16;
                if (u == 0 || c + u * WAVES < whole) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) wv[u][t][half] = __builtin_bit_cast(i32x4, *(const any4 *)(w[t] + k));
#pragma unroll
                    for (int t = 0; t < MT; ++t) av[u][t][half] = __builtin_bit_cast(i32x4, *(const any4 *)(a[t] + k));
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u == 0 || c + u * WAVES < whole) products(av[u], wv[u]);
    }
    if (whole < steps && whole % WAVES == wave) {
        i32x4 av[MT][2], wv[NT][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = whole * 128 + g * 32 + half * 16;
#pragma unroll
            for (int t = 0; t < NT; ++t) wv[t][half] = row_tail(w[t], k, p.K);
#pragma unroll
            for (int t = 0; t < MT; ++t) av[t][half] = row_tail(a[t], k, p.K);
        }
        products(av, wv);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) sums[((t * MT + u) * WAVES + wave) * 64 + lane] = acc[t][u];
    __syncthreads();
    for (int tile = wave; tile < MT * NT; tile += WAVES) {
        i32x4 sum = sums[tile * WAVES * 64 + lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) sum += sums[(tile * WAVES + k) * 64 + lane];
        const int m = m0 + tile % MT * 16 + i, n = n0 + tile / MT * 16 + 4 * g;
        if (m < p.M && n < p.N) {
            const float sa = p.sa[m * p.ssa];
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int nc = min(n + j, p.N - 1);
                v[j] = (float)sum[j] * sa * p.sw[nc * p.ssw];
                if (p.bias) v[j] += load_as_f32(p.bias, nc * p.sbias, p.bias_type);
            }
            store4<TYPE>(p, m, n, v);
        }
    }
}

// ---- many tokens ---------------------------------------------------------------------------------------------------

constexpr int kStep = 64;       // bytes of K per step
constexpr int kRing = 4;        // steps in LDS
constexpr int kNowhere = 0x7ffffff0;      // an offset behind every descriptor's end: reads as zero

// s_waitcnt: at most n vector-memory operations outstanding; the LDS counter to zero
__device__ __forceinline__ constexpr int vm_only(int n) { return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14); }
constexpr int kLgkmZero = 15 | (7 << 4) | (0 << 8) | (3 << 14);

// 1 KB (64 lanes x 16 bytes) from memory into LDS at `to`, without a register between: the compiler does not know of the write, so
// it puts no wait of its own in front of the LDS reads; the kernel waits by count.  (m0 is the compiler's to set right in front of
// each of its own uses.)
__device__ __forceinline__ void into_lds(__amdgpu_buffer_rsrc_t from, int offset, int more, uint32_t to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(offset), "s"(from), "s"(more) : "memory");
#endif
}

// The workgroup's tile.  XCDs get workgroups in turn: each gets a contiguous part of the tiles; within it GROUP rows of tiles column
// by column, for the operands' reuse in L2.
struct Place {
    int m, n;
    __device__ __forceinline__ Place(int tiles_m, int tiles_n)
    {
        constexpr int GROUP = 8;
        const int total = tiles_m * tiles_n, per = total / 8, id = (int)blockIdx.x;
        const int t = id < per * 8 ? (id % 8) * per + id / 8 : id;
        const int group = t / (GROUP * tiles_n), rows = min(GROUP, tiles_m - group * GROUP), in = t - group * GROUP * tiles_n;
        m = group * GROUP + in % rows;
        n = in / rows;
    }
};

// What a wave's (32 TM) tokens x (32 TN) channels are scaled by: a lane's tokens as the products leave them, its 8 channels as they
// are written
template <int TM, int TN> struct Scales {
    static constexpr int LPR = 4 * TN;                  // lanes per row of 32 TN channels, 8 each
    int n;
    float sa[TM], sw[8], bias[8];
    __device__ __forceinline__ void load(const MatmulParams &p, int m0, int n0, int lane)
    {
        n = n0 + lane % LPR * 8;
#pragma unroll
        for (int u = 0; u < TM; ++u) sa[u] = p.sa[min(m0 + u * 32 + (lane & 31), p.M - 1) * p.ssa];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int nc = min(n + j, p.N - 1);
            sw[j] = p.sw[nc * p.ssw];
            bias[j] = p.bias ? load_as_f32(p.bias, nc * p.sbias, p.bias_type) : 0.f;
        }
    }
    __device__ __forceinline__ void arrived()
    {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(sw[j]), "+v"(bias[j]));
#pragma unroll
        for (int u = 0; u < TM; ++u) asm volatile("" : "+v"(sa[u]));
#endif
    }
};

// 32 tokens x (32 TN) channels of a wave at a time through its own part of LDS, from where rows leave in 16-byte pieces
template <int TYPE, int TM, int TN>
__device__ __forceinline__ void write(const MatmulParams &p, const i32x16 (&acc)[TN][TM], const Scales<TM, TN> &by, char *lds, int m0, int wave, int lane)
{
    typedef element<TYPE> E;
    constexpr int LPR = 4 * TN, RPI = 64 / LPR;         // lanes per row; rows that a wave writes at a time
    constexpr int PITCH = 32 * TN + 4;                  // floats
    const int hi = lane >> 5, n = by.n;
    float *mine = (float *)lds + wave * 32 * PITCH;
#pragma unroll
    for (int u = 0; u < TM; ++u) {
        const int mb = m0 + u * 32;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)acc[j][u][4 * q + e] * by.sa[u];
                *(f32x4 *)&mine[(lane & 31) * PITCH + 32 * j + 8 * q + 4 * hi] = v;
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 32; r += RPI) {
            const int row = r + lane / LPR;
            const f32x4 lo = *(const f32x4 *)&mine[row * PITCH + lane % LPR * 8], hi4 = *(const f32x4 *)&mine[row * PITCH + lane % LPR * 8 + 4];
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (e < 4 ? lo[e] : hi4[e - 4]) * by.sw[e] + by.bias[e];
            if (mb + row < p.M) {
                E *o = (E *)p.out + (int64_t)(mb + row) * p.so_m + n;
                if (n + 8 <= p.N) {
                    typedef Wide<TYPE> W;
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
                        if (n + e < p.N) o[e] = from_f32<TYPE>(v[e]);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TYPE, int TM, int TN>
__global__ void __launch_bounds__(256, TM * TN == 16 ? 1 : 2) tile_kernel(const MatmulParams p, int tiles_m, int tiles_n)
{
    constexpr int BM = 64 * TM, BN = 64 * TN;
    constexpr int STAGE = (BM + BN) * kStep;            // bytes
    constexpr int LOADS = TM + TN;                      // per wave and step
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    const Place at_tile(tiles_m, tiles_n);
    const int m0 = at_tile.m * BM, n0 = at_tile.n * BN;

    auto descriptor = [](const int8_t *base, int64_t stride, int n, int K) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)((n - 1) * stride + K), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t ra = descriptor(p.a + (int64_t)m0 * p.sa_m, p.sa_m, min(BM, p.M - m0), p.K),
                                 rw = descriptor(p.w + (int64_t)n0 * p.sw_n, p.sw_n, min(BN, p.N - n0), p.K);
    // A load fills 16 rows of 64 bytes.  16-byte unit u of row r lies at place u ^ (r / 4 % 4): 8 lanes that read the same unit of 8
    // rows then touch all 64 banks once.
    const int lr = lane >> 2, lu = ((lane & 3) ^ ((lr >> 2) & 3)) * 16;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    int off[TM + TN];                                    // this lane's 16 bytes of the wave's loads, at k = 0
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int r = (wave * TM + j) * 16 + lr;
        off[j] = m0 + r < p.M ? (int)(r * p.sa_m) + lu : kNowhere;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int r = (wave * TN + j) * 16 + lr;
        off[TM + j] = n0 + r < p.N ? (int)(r * p.sw_n) + lu : kNowhere;
    }
    auto request = [&](int step, int j) {
        const int k = step * kStep;
        const uint32_t slot = base + (step % kRing) * STAGE;
        const int at = k + lu < p.K ? off[j] : kNowhere;
        if (j < TM) into_lds(ra, at, k, slot + (wave * TM + j) * 1024);
        else into_lds(rw, at, k, slot + BM * kStep + (wave * TN + j - TM) * 1024);
    };
    const int f = (lane >> 2) & 3, hi = lane >> 5;
    int at[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) at[kk] = (lane & 31) * kStep + (((kk * 2 + hi) ^ f) * 16);
    i32x4 fa[2][TM], fw[2][TN];
    auto fetch = [&](int step, auto half, int j) {
        constexpr int kk = decltype(half)::value;
        const char *s = lds + (step % kRing) * STAGE + at[kk];
        if (j < TM) fa[kk][j] = *(const i32x4 *)(s + (wm * TM + j) * 32 * kStep);
        else fw[kk][j - TM] = *(const i32x4 *)(s + BM * kStep + (wn * TN + j - TM) * 32 * kStep);
    };
    i32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int u = 0; u < TM; ++u) acc[j][u] = i32x16{};
    // TM TN products, and beside each what `beside` issues: a wave that waits for room to issue a load waits while a product runs
    auto products = [&](auto half, auto &&beside) {
        constexpr int kk = decltype(half)::value;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int u = 0; u < TM; ++u) {
                beside(j * TM + u);
                __builtin_amdgcn_sched_barrier(0);
                acc[j][u] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[kk][j], fa[kk][u], acc[j][u], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    Scales<TM, TN> by;                                   // asked for in front of the loop
    by.load(p, m0 + wm * 32 * TM, n0 + wn * 32 * TN, lane);
    typedef std::integral_constant<int, 0> first;
    typedef std::integral_constant<int, 1> second;
    // what goes beside product n of TM TN: one of k things each, evenly from the first product on
    auto spread = [](int n, int k, auto &&f) {
#pragma unroll
        for (int j = 0; j < k; ++j)
            if (j * (TM * TN) / k == n) f(j);
    };
    constexpr int EARLY = LOADS / 2;                     // a step's requests: these behind one barrier, the others up to the next

    const int steps = (p.K + kStep - 1) / kStep;
#pragma unroll
    for (int j = 0; j < (kRing - 1) * LOADS + EARLY; ++j) request(j / LOADS, j % LOADS);
    by.arrived();      // here, not behind the loop
    __builtin_amdgcn_s_waitcnt(vm_only((kRing - 2) * LOADS + EARLY));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < LOADS; ++j) fetch(0, first{}, j);
    for (int s = 0; s < steps; ++s) {
        products(first{}, [&](int n) {
            spread(n, LOADS, [&](int j) { fetch(s, second{}, j); });
            spread(n, LOADS - EARLY, [&](int j) { request(s + kRing - 1, EARLY + j); });
        });
        // this step's operands are in registers, the next step's in LDS (two steps' requests behind it)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(kLgkmZero);
        __builtin_amdgcn_s_waitcnt(vm_only((kRing - 2) * LOADS));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        products(second{}, [&](int n) {
            spread(n, LOADS, [&](int j) { fetch(s + 1, first{}, j); });
            spread(n, EARLY, [&](int j) { request(s + kRing, j); });
        });
    }
    __builtin_amdgcn_s_waitcnt(vm_only(0));
    asm volatile("" ::: "memory");
    __syncthreads();

    write<TYPE, TM, TN>(p, acc, by, lds, m0 + wm * 32 * TM, wave, lane);
}

// The same for rows that begin at any byte or end at any: operands come through registers, two steps ahead, into a ring of two steps.
template <int TYPE, int TM, int TN>
__global__ void __launch_bounds__(256, 2) odd_tile_kernel(const MatmulParams p, int tiles_m, int tiles_n)
{
    constexpr int BM = 64 * TM, BN = 64 * TN, STAGE = (BM + BN) * kStep, LOADS = TM + TN;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    const Place at_tile(tiles_m, tiles_n);
    const int m0 = at_tile.m * BM, n0 = at_tile.n * BN;
    // places in LDS as above
    const int lr = lane >> 2, unit = (lane & 3) * 16, lu = ((lane & 3) ^ ((lr >> 2) & 3)) * 16;
    const int8_t *from[LOADS];
#pragma unroll
    for (int j = 0; j < TM; ++j) from[j] = p.a + min(m0 + (wave * TM + j) * 16 + lr, p.M - 1) * p.sa_m;
#pragma unroll
    for (int j = 0; j < TN; ++j) from[TM + j] = p.w + min(n0 + (wave * TN + j) * 16 + lr, p.N - 1) * p.sw_n;
    const int steps = (p.K + kStep - 1) / kStep;
    auto request = [&](int step, i32x4 (&q)[LOADS]) {
        const int k = step * kStep + unit;
        if ((step + 1) * kStep <= p.K) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) q[j] = __builtin_bit_cast(i32x4, *(const any4 *)(from[j] + k));
        } else if (step < steps) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) q[j] = row_tail(from[j], k, p.K);
        }
    };
    auto place = [&](int step, const i32x4 (&q)[LOADS]) {
        char *s = lds + (step & 1) * STAGE + lr * kStep + lu;
#pragma unroll
        for (int j = 0; j < TM; ++j) *(i32x4 *)(s + (wave * TM + j) * 1024) = q[j];
#pragma unroll
        for (int j = 0; j < TN; ++j) *(i32x4 *)(s + BM * kStep + (wave * TN + j) * 1024) = q[TM + j];
    };
    i32x16 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int u = 0; u < TM; ++u) acc[j][u] = i32x16{};
    const int f = (lane >> 2) & 3, hi = lane >> 5;
    auto products = [&](int step) {
        const char *s = lds + (step & 1) * STAGE;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const char *at = s + (lane & 31) * kStep + (((kk * 2 + hi) ^ f) * 16);
            i32x4 fa[TM], fw[TN];
#pragma unroll
            for (int j = 0; j < TM; ++j) fa[j] = *(const i32x4 *)(at + (wm * TM + j) * 32 * kStep);
#pragma unroll
            for (int j = 0; j < TN; ++j) fw[j] = *(const i32x4 *)(at + BM * kStep + (wn * TN + j) * 32 * kStep);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int u = 0; u < TM; ++u) acc[j][u] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fa[u], acc[j][u], 0, 0, 0);
        }
    };
    Scales<TM, TN> by;
    by.load(p, m0 + wm * 32 * TM, n0 + wn * 32 * TN, lane);
    i32x4 q[2][LOADS];
    request(0, q[0]);
    request(1, q[1]);
    // one barrier a step: what a step overwrites was read in front of the barrier of the step before it
    for (int s = 0; s < steps; s += 2) {
        place(s, q[0]);
        request(s + 2, q[0]);
        __syncthreads();
        products(s);
        if (s + 1 < steps) {
            place(s + 1, q[1]);
            request(s + 3, q[1]);
            __syncthreads();
            products(s + 1);
        }
    }
    __syncthreads();
    write<TYPE, TM, TN>(p, acc, by, lds, m0 + wm * 32 * TM, wave, lane);
}

template <int TYPE, int MT, int NT, int WAVES>
hipError_t run_direct(const MatmulParams &p, hipStream_t s)
{
    const int64_t tm = (p.M + 16 * MT - 1) / (16 * MT), tn = (p.N + 16 * NT - 1) / (16 * NT);
    if (tm * tn * 64 * WAVES > 0xffffffffLL) return hipErrorInvalidConfiguration;
    constexpr int lds = MT * NT * WAVES * 1024;
    static std::atomic<uint64_t> done;
    const hipError_t e = ensure_dynamic_lds((const void *)direct_kernel<TYPE, MT, NT, WAVES>, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((direct_kernel<TYPE, MT, NT, WAVES>), dim3((uint32_t)(tm * tn)), dim3(64 * WAVES), lds, s, p, (int)tm);
    return hipGetLastError();
}

// ALIGNED: tile_kernel, otherwise odd_tile_kernel
template <int TYPE, int TM, int TN, bool ALIGNED = true>
hipError_t run_tile(const MatmulParams &p, hipStream_t s)
{
    const int64_t tm = (p.M + 64 * TM - 1) / (64 * TM), tn = (p.N + 64 * TN - 1) / (64 * TN);
    if (tm * tn * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    constexpr int ring = (ALIGNED ? kRing : 2) * 64 * (TM + TN) * kStep, out = 4 * 32 * (32 * TN + 4) * 4, lds = ring > out ? ring : out;
    static std::atomic<uint64_t> done;
    auto *const kernel = [] {
        if constexpr (ALIGNED) return tile_kernel<TYPE, TM, TN>;
        else return odd_tile_kernel<TYPE, TM, TN>;
    }();
    const hipError_t e = ensure_dynamic_lds((const void *)kernel, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tm * tn)), dim3(256), lds, s, p, (int)tm, (int)tn);
    return hipGetLastError();
}

template <int TYPE>
hipError_t of_type(const MatmulParams &p, int n_cu, hipStream_t s)
{
    // what the tile kernel asks for: 16-byte pieces of K, offsets inside a tile in 31 bits
    const bool aligned = p.K % 16 == 0 && (p.sa_m | p.sw_n) % 16 == 0 && (((uintptr_t)p.a | (uintptr_t)p.w) & 15) == 0 &&
                         p.sa_m >= 0 && p.sw_n >= 0 && p.sa_m < (1 << 22) && p.sw_n < (1 << 22);
    // Large tiles read the operands less often, small ones reach more compute units: the largest whose tiles occupy about half of the
    // units.  Measured (us, the neighbours of each bound; tokens x channels x K):
    //   256x256 from half of the units on   1024 x 10576 x 2560 (0.66): 42.7, 128x128 47.0;  2048 x 2560 x 5120 (0.31): 58.2 and 47.6
    //   128x128 from half                    777 x  2560 x 5120 (0.55): 25.2, 128x64  27.5;   512 x 2560 x 5120 (0.31): 28.2 and 20.7
    //   128x64 from 0.6                      128 x 10576 x 2560 (0.65): 12.4, 64x64   14.6;   256 x 2560 x 5120 (0.31): 19.0 and 16.1
    //   64x64 from a quarter                 256 x  3352 x  768 (0.83): 5.4, direct    9.6;    64 x 2560 x 5120 (0.16): 15.7 and 13.0
    //   direct 32x32 from 0.35                64 x  2560 x 5120 (0.63): 13.0, 16x16   17.0;    64 x  768 x 1536 (0.19): 5.5 and 4.3
    const double units = n_cu > 0 ? n_cu : 256;
    const auto reach = [&](int64_t m, int64_t n) { return (double)(((p.M + m - 1) / m) * ((p.N + n - 1) / n)) / units; };
    if (aligned && p.M > 64) {
        if (reach(256, 256) >= 0.5) return run_tile<TYPE, 4, 4>(p, s);
        if (reach(128, 128) >= 0.5) return run_tile<TYPE, 2, 2>(p, s);
        if (reach(128, 64) >= 0.6) return run_tile<TYPE, 2, 1>(p, s);
    }
    if (aligned && p.M > 16 && reach(64, 64) >= 0.25) return run_tile<TYPE, 1, 1>(p, s);
    // Rows of other alignments: 128x128 from one tile per unit on (1024 x 10576 x 2561 (2.6): 68, 64x64 114;  4096 x 768 x 1530 (0.75): 25.3 and
    // 20.3), 64x64 from a quarter (128 x 3352 x 770 (0.41): 9.0, direct 14.1;  256 x 768 x 1530 (0.19): 13.4 and 12.0)
    if (!aligned && p.M > 64 && reach(128, 128) >= 1) return run_tile<TYPE, 2, 2, false>(p, s);
    if (!aligned && p.M > 4 && reach(64, 64) >= 0.25) return run_tile<TYPE, 1, 1, false>(p, s);
    if (p.M > 16 && reach(32, 32) >= 0.35) return run_direct<TYPE, 2, 2, 4>(p, s);
    // 16 x 16: eight waves share a tile by K where the tiles leave units idle (1 x 2560 x 5120: 6.0, four waves 7.0), four where there
    // are tiles enough (1 x 10576 x 2560: 7.8 and 8.0)
    return reach(16, 16) >= 2 ? run_direct<TYPE, 1, 1, 4>(p, s) : run_direct<TYPE, 1, 1, 8>(p, s);
}

}  // namespace

hipError_t launch_matmul(const MatmulParams &p, int n_cu, hipStream_t s)
{
    if (p.M == 0 || p.N == 0) return hipSuccess;
    if (p.out_type == DT_F32) return of_type<DT_F32>(p, n_cu, s);
    return p.out_type == DT_BF16 ? of_type<DT_BF16>(p, n_cu, s) : of_type<DT_F16>(p, n_cu, s);
}

}  // namespace ssd
