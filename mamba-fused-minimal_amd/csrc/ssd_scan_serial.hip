// The selective scan token by token, for every type and size, and its single-token form.
//
//   d = limit(softplus(dt + bias));   h = [same sequence] exp(d A) h + d x (x) B;   y = h C + D x;   y *= silu(z)
//
// everything in 32 bits, y rounded once.
//
// Prompts (serial_kernel): the state h (headdim rows x dstate columns of a head) stays in registers -- four lanes share a row, a lane
// holds two rows' quarter -- and a workgroup walks its tokens; B, C, x and the steps of 32 tokens at a time come through LDS in 32
// bits.  Three multiply-adds per state element and token and no matrix instruction: the vector ALU bounds it.  Where batch x heads
// are too few for the card, the row is cut into segments: a first launch computes what each segment adds to a state of zero,
// launch_scan_join turns that into the state entering each segment, and a second launch starts from there.
//
// Single tokens (step_kernel): the states are read and written once, 8 bytes per element for 5 operations: HBM bound.  Lanes share a
// row's columns, 16 bytes each, and every load of a workgroup is in flight before the first is used.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

constexpr int kTile = 32;      // tokens staged at a time

// NV: float4 per lane, row and operand (dstate <= 16 NV).  WAVES x 32 rows per workgroup.  OUT: write y (otherwise only what the
// segment adds and the factor on what enters it).
template <int TYPE, int NV, int WAVES, bool OUT>
__global__ void __launch_bounds__(64 * WAVES) serial_kernel(const SelScanParams p, int row_blocks)
{
    typedef element<TYPE> E;
    constexpr int NP = 16 * NV, ROWS = 32 * WAVES, THREADS = 64 * WAVES;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *Bt = lds, *Ct = Bt + kTile * NP, *xt = Ct + (OUT ? kTile * NP : 0), *dt = xt + kTile * ROWS, *et = dt + kTile;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quarter = lane & 3;
    uint32_t i = blockIdx.x;
    const int rb = (int)(i % (uint32_t)row_blocks); i /= (uint32_t)row_blocks;
    const int h = (int)(i % (uint32_t)p.nheads); i /= (uint32_t)p.nheads;
    const int seg = (int)(i % (uint32_t)p.segments), b = (int)(i / (uint32_t)p.segments);
    const int g = h / (p.nheads / p.ngroups), P = p.headdim, N = p.dstate, p0 = rb * ROWS;
    const int len = row_tokens(p.len, p.slen, b, p.seqlen);
    const int t0 = seg * p.segment_tokens, t_end = min(t0 + p.segment_tokens, p.seqlen), t1 = min(t_end, len);
    const E *x = (const E *)p.x + b * p.sx_b + h * p.sx_h + p0, *z = p.z ? (const E *)p.z + b * p.sz_b + h * p.sz_h + p0 : nullptr;
    const E *Bg = (const E *)p.B + b * p.sB_b + g * p.sB_g, *Cg = (const E *)p.C + b * p.sC_b + g * p.sC_g;
    E *y = (E *)p.y + b * p.sy_b + h * p.sy_h + p0;
    const float A = load_as_f32(p.A, h * p.sA, p.A_type);
    const float bias = p.delta.bias ? load_as_f32(p.delta.bias, h * p.delta.sbias, p.delta.bias_type) : 0.f;
    const int row[2] = {wave * 32 + (lane >> 2), wave * 32 + 16 + (lane >> 2)};

    f32x4 s[2][NV];
    float *ws = p.ws_states + ((((int64_t)b * p.nheads + h) * p.segments + seg) * P) * N;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // clamped loads and a select: a branch per element would keep its mask in scalar registers
                const int n = 16 * v + 4 * quarter + j, pr = p0 + row[r], nc = min(n, N - 1), pc = min(pr, P - 1);
                float f = 0.f;
                if (OUT && p.segments > 1) f = ws[(int64_t)pc * N + nc];
                else if (OUT && p.init) f = load_as_f32(p.init, b * p.si_b + h * p.si_h + pc * p.si_p + nc, p.init_type);
                s[r][v][j] = n < N && pr < P ? f : 0.f;
            }
    float D[2] = {0.f, 0.f};
    if (OUT && p.D)
#pragma unroll
        for (int r = 0; r < 2; ++r)
            if (p0 + row[r] < P) D[r] = load_as_f32(p.D, h * p.sD_h + (p0 + row[r]) * p.sD_p, p.D_type);
    float through = 1.f;

    for (int t = t0; t < t1; t += kTile) {
        const int n_t = min(kTile, t1 - t);
        __syncthreads();
        for (int k = tid; k < kTile * NP; k += THREADS) {
            const int tt = k / NP, n = k % NP;
            const bool there = tt < n_t && n < N;
            Bt[k] = there ? to_f32<TYPE>(Bg[(t + tt) * p.sB_l + n]) : 0.f;
            if constexpr (OUT) Ct[k] = there ? to_f32<TYPE>(Cg[(t + tt) * p.sC_l + n]) : 0.f;
        }
        for (int k = tid; k < kTile * ROWS; k += THREADS) {
            const int tt = k / ROWS, r = k % ROWS;
            xt[k] = tt < n_t && p0 + r < P ? to_f32<TYPE>(x[(t + tt) * p.sx_l + r]) : 0.f;
        }
        if (tid < n_t) {
            const int tok = t + tid;
            const float d = delta_of(p.delta, load_as_f32(p.dt, b * p.sdt_b + tok * p.sdt_l + h * p.sdt_h, p.dt_type) + bias);
            bool starts = false;
            if (p.seq) starts = p.seq[b * p.sq_b + tok * p.sq_l] != (tok > 0 ? p.seq[b * p.sq_b + (tok - 1) * p.sq_l] : 0);
            dt[tid] = d;
            et[tid] = starts ? -1.f : __expf(d * A);      // negative: a sequence starts, nothing of the state passes
        }
        __syncthreads();
        for (int tt = 0; tt < n_t; ++tt) {
            const float d = dt[tt], e = et[tt];
            through = e < 0.f || through < 0.f ? -1.f : through * e;
            const float keep = e < 0.f ? 0.f : e;
            if (e < 0.f) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int v = 0; v < NV; ++v) s[r][v] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            const float xv[2] = {xt[tt * ROWS + row[0]], xt[tt * ROWS + row[1]]};
            const float dx[2] = {d * xv[0], d * xv[1]};
            float acc[2] = {0.f, 0.f};
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const f32x4 Bv = *(const f32x4 *)&Bt[tt * NP + 16 * v + 4 * quarter];
                f32x4 Cv = {0.f, 0.f, 0.f, 0.f};
                if constexpr (OUT) Cv = *(const f32x4 *)&Ct[tt * NP + 16 * v + 4 * quarter];
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[r][v][j] = fmaf(s[r][v][j], keep, dx[r] * Bv[j]);
                        if constexpr (OUT) acc[r] = fmaf(s[r][v][j], Cv[j], acc[r]);
                    }
            }
            if constexpr (OUT) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float sum = group_sum<4>(acc[r]);
                    // in the place of x, which only these four lanes read
                    if (quarter == 0) xt[tt * ROWS + row[r]] = p.D ? fmaf(D[r], xv[r], sum) : sum;
                }
            }
        }
        if constexpr (OUT) {
            __syncthreads();
            for (int k = tid; k < n_t * ROWS; k += THREADS) {
                const int tt = k / ROWS, r = k % ROWS;
                if (p0 + r < P) {
                    float v = xt[k];
                    if (z) v *= silu(to_f32<TYPE>(z[(t + tt) * p.sz_l + r]));
                    y[(t + tt) * p.sy_l + r] = from_f32<TYPE>(v);
                }
            }
        }
    }
    if constexpr (OUT) {
        for (int t = max(t0, t1); t < t_end; ++t)
            for (int r = tid; r < ROWS; r += THREADS)
                if (p0 + r < P) y[t * p.sy_l + r] = from_f32<TYPE>(0.f);
    }
    const bool last = OUT && seg == p.segments - 1;
    if (!OUT || last) {
        float *to = OUT ? p.fin + b * p.sf_b + h * p.sf_h : ws;
        const int64_t pitch = OUT ? p.sf_p : N;
        int q = quarter;
        asm volatile("" : "+v"(q));      // or the compiler keeps every element's mask from the loads above
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = 16 * v + 4 * q + j, pr = p0 + row[r];
                    if (n < N && pr < P) to[pr * pitch + n] = s[r][v][j];
                }
    }
    if (!OUT && tid == 0 && rb == 0) p.ws_decay[((int64_t)b * p.nheads + h) * p.segments + seg] = through;
}

// ws_states of a (row, head): what each segment adds -> what enters it.  A thread per state element walks the segments; the
// loads of eight are in flight together.
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
    for (int s0 = 0; s0 < S; s0 += 8) {
        float add[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) add[u] = s0 + u < S ? ws[(int64_t)(s0 + u) * plane] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (s0 + u >= S) break;
            const float f = decay[s0 + u];
            ws[(int64_t)(s0 + u) * plane] = in;
            in = f < 0.f ? add[u] : fmaf(f, in, add[u]);
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

template <int TYPE, int NV, int WAVES>
hipError_t run_serial(const SelScanParams &p, hipStream_t s)
{
    constexpr int NP = 16 * NV, ROWS = 32 * WAVES;
    const int row_blocks = (p.headdim + ROWS - 1) / ROWS;
    const int64_t blocks = (int64_t)row_blocks * p.nheads * p.segments * p.batch;
    if (blocks * 64 * WAVES > 0xffffffffLL) return hipErrorInvalidConfiguration;
    const int lds_add = 4 * kTile * (NP + ROWS + 2), lds_out = lds_add + 4 * kTile * NP;
    static std::atomic<uint64_t> done[2];
    hipError_t e = ensure_dynamic_lds((const void *)serial_kernel<TYPE, NV, WAVES, true>, lds_out, done[0]);
    if (e == hipSuccess) e = ensure_dynamic_lds((const void *)serial_kernel<TYPE, NV, WAVES, false>, lds_add, done[1]);
    if (e != hipSuccess) return e;
    if (p.segments > 1) {
        hipLaunchKernelGGL((serial_kernel<TYPE, NV, WAVES, false>), dim3((uint32_t)blocks), dim3(64 * WAVES), lds_add, s, p, row_blocks);
        e = hipGetLastError();
        if (e == hipSuccess) e = launch_scan_join(p, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((serial_kernel<TYPE, NV, WAVES, true>), dim3((uint32_t)blocks), dim3(64 * WAVES), lds_out, s, p, row_blocks);
    return hipGetLastError();
}

template <int TYPE>
hipError_t serial_of_type(const SelScanParams &p, hipStream_t s)
{
    auto waves = [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        if (p.headdim <= 32) return run_serial<TYPE, NV, 1>(p, s);
        return p.headdim <= 64 ? run_serial<TYPE, NV, 2>(p, s) : run_serial<TYPE, NV, 4>(p, s);
    };
    if (p.dstate <= 16) return waves(std::integral_constant<int, 1>{});
    if (p.dstate <= 64) return waves(std::integral_constant<int, 4>{});
    if (p.dstate <= 128) return waves(std::integral_constant<int, 8>{});
    return waves(std::integral_constant<int, 16>{});
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

hipError_t launch_scan_serial(const SelScanParams &p, hipStream_t s)
{
    if (p.type == DT_F32) return serial_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? serial_of_type<DT_BF16>(p, s) : serial_of_type<DT_F16>(p, s);
}

hipError_t launch_scan_step(const SelStepParams &p, hipStream_t s)
{
    if (p.batch == 0) return hipSuccess;
    if (p.type == DT_F32) return step_of_type<DT_F32>(p, s);
    return p.type == DT_BF16 ? step_of_type<DT_BF16>(p, s) : step_of_type<DT_F16>(p, s);
}

}  // namespace ssd
