// The selective scan of prompts on the bf16 matrix instructions (bf16 x, B, C, z; dstate <= 128; any other size).
//
// Tokens are taken 64 at a time.  With cs the running sum of d A inside such a chunk and h the state entering it,
//
//   y_t = e^(cs_t) h C_t + sum_{j <= t} e^(cs_t - cs_j) d_j (C_t . B_j) x_j + D x_t,     y_t *= silu(z_t)
//   h'  = e^(cs_63) h + sum_j e^(cs_63 - cs_j) d_j x_j (x) B_j
//
// where terms of another sequence are left out: four products of matrices per chunk.  A wave owns 32 rows of a head's state (32 headdim x
// dstate, in registers as accumulators) and walks the tokens of its segment; the eight waves of a workgroup share a chunk's B and C.
// The next chunk's x, B and C go from memory into the other half of LDS meanwhile, without a register between.
//
// Every operand that is made here goes from accumulators to operands inside registers.  The matrix instructions take k in any
// order that both operands agree on, and a tile's rows may stand for any rows: tile `half` of a pair stands for rows
// 8 (i / 4) + 4 half + i % 4 of 32 (i = the tile's row), so that a lane, which gets rows 4 g .. 4 g + 3 of a tile (g = lane / 16), holds 8
// consecutive ones of the pair -- the 8 k that it has to deliver as an operand of the next product.  The same order makes a
// lane's outputs 16 contiguous bytes.
//
// Rounding: x, B and C are bf16 already.  The state, the weighted x and the scores enter products as the sum of two bf16 parts (16 bits:
// one part alone would add as much error as the rounding of y, and the final states are fp32).  Sums, states and decays are fp32.
//
// Values that are not finite: a masked factor is selected away, not multiplied by zero, but a matrix product would still carry a
// NaN of x_j to the tokens in front of j.  A chunk whose x, B or d is not finite is therefore taken token by token (slow path).
//
// What bounds it: 1050 MB of x, z, y and states (4 x 8192 tokens, 80 heads of 64 x 128) against about 1400 vector and 200 matrix
// instructions per wave and chunk; both are near 190 us.
#include "ssd_layer.h"

namespace ssd {
namespace {

using namespace layer;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int T = 64;                 // tokens per chunk
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeast = -160.f;      // of log2(decay): 2^-160 is zero in fp32 already, and sums of 64 such stay exact enough to subtract

__device__ __forceinline__ float pow2(float v) { return __builtin_amdgcn_exp2f(v); }

// eight values -> two bf16 parts each
struct Parts { bf16x8 hi, lo; };
__device__ __forceinline__ Parts split(const float (&v)[8])
{
    Parts r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const bf16x2 h = {(__bf16)v[j], (__bf16)v[j + 1]};
        const uint32_t b = __builtin_bit_cast(uint32_t, h);
        const bf16x2 l = {(__bf16)(v[j] - __builtin_bit_cast(float, b << 16)), (__bf16)(v[j + 1] - __builtin_bit_cast(float, b & 0xffff0000u))};
        r.hi[j] = h[0]; r.hi[j + 1] = h[1];
        r.lo[j] = l[0]; r.lo[j + 1] = l[1];
    }
    return r;
}
__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

// 16 bytes of LDS; and four tokens' values of one column: lane i of 16 addresses 8 bytes of token i / 4, columns 4 (i % 4) .. + 3, and gets
// column i of the four tokens
__device__ __forceinline__ bf16x8 row8(const char *p) { return *(const bf16x8 *)p; }
__device__ __forceinline__ s16x4 column4(const char *p)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
#else
    return s16x4{};
#endif
}
__device__ __forceinline__ bf16x8 column8(const char *lo, const char *hi)
{
    struct { s16x4 a, b; } v = {column4(lo), column4(hi)};
    return __builtin_bit_cast(bf16x8, v);
}

constexpr int kNowhere = 0x7ffffff0;      // an offset behind every descriptor's end: reads as zero, is not written

// 64 lanes x 16 bytes from memory into LDS at `to`.  The compiler does not know of the write, so it puts no wait of its own in front of
// the LDS reads; the kernel waits by count.  (m0 is the compiler's to set right in front of each of its own uses.)
__device__ __forceinline__ void into_lds(__amdgpu_buffer_rsrc_t from, int offset, int more, uint32_t to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(offset), "s"(from), "s"(more) : "memory");
#endif
}
__device__ __forceinline__ constexpr int vm_only(int n) { return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14); }

// a bit set where one of the values so far is not finite (all exponent bits set: + 1 carries into the sign)
__device__ __forceinline__ uint32_t infinite(u32x4 v)
{
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= (v[j] & 0x7f807f80u) + 0x00800080u;
    return bad & 0x80008000u;
}

// a token's 8 values of 16-bit type as fp32
__device__ __forceinline__ float half_of(const u32x4 &v, int e) { return __builtin_bit_cast(float, e % 2 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16); }

constexpr int kWaves = 8;
constexpr int META = 5 * T + 32;                                 // floats per wave: cs, d, weights, starts, decays in the first half, D

// NK: 32-column steps of dstate; OUT: write y (otherwise only what the segment adds and the factor on what enters it); SEQ: seq_idx
template <int NK, bool OUT, bool SEQ>
__global__ void __launch_bounds__(64 * kWaves, 2) chunk_kernel(const SelScanParams p, int blocks_per_head, int sets)
{
    constexpr int UNITS = 4 * NK, ROW = 16 * UNITS, TILE = T * ROW;     // 16-byte units and bytes of a token's B or C; bytes of a chunk's
    constexpr int HALF = (OUT ? 2 : 1) * TILE, XTILE = T * 64;          // bytes of B (and C), and of a wave's x, per half of LDS
    constexpr int LOADS = TILE / 1024 / kWaves;                         // of B per wave and chunk, and of C
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int i = lane & 15, g = lane >> 4;
    const int xat = 2 * HALF + wave * 2 * XTILE;
    float *const meta = (float *)(lds + 2 * HALF + kWaves * 2 * XTILE) + wave * META;
    float *const cs_l = meta, *const d_l = meta + T, *const w_l = meta + 2 * T, *const mid_l = meta + 4 * T, *const D_l = meta + 5 * T;
    int *const start_l = (int *)(meta + 3 * T);

    // XCDs get workgroups in turn: each gets a contiguous part, whose workgroups share B and C
    const int total = (int)gridDim.x, per = total / 8, id = (int)blockIdx.x;
    int at = id < per * 8 ? (id % 8) * per + id / 8 : id;
    const int set = at % sets; at /= sets;
    const int gr = at % p.ngroups; at /= p.ngroups;
    const int seg = at % p.segments, b = at / p.segments;
    const int heads = p.nheads / p.ngroups, unit = set * kWaves + wave;
    const bool live = unit < heads * blocks_per_head;
    const int h = gr * heads + (live ? unit / blocks_per_head : 0), p0 = live ? unit % blocks_per_head * 32 : 0;
    const int P = p.headdim, N = p.dstate, np = live ? P - p0 : 0;      // rows from p0 on
    const int len = row_tokens(p.len, p.slen, b, p.seqlen);
    const int t0 = seg * p.segment_tokens, t_end = min(t0 + p.segment_tokens, p.seqlen), t1 = min(t_end, len);
    const uint16_t *const x = (const uint16_t *)p.x + b * p.sx_b + h * p.sx_h + p0;
    const uint16_t *const z = OUT && p.z ? (const uint16_t *)p.z + b * p.sz_b + h * p.sz_h + p0 : nullptr;
    const uint16_t *const Bg = (const uint16_t *)p.B + b * p.sB_b + gr * p.sB_g, *const Cg = (const uint16_t *)p.C + b * p.sC_b + gr * p.sC_g;
    uint16_t *const y = OUT ? (uint16_t *)p.y + b * p.sy_b + h * p.sy_h + p0 : nullptr;
    const float A2 = load_as_f32(p.A, h * p.sA, p.A_type) * kLog2e;
    const float bias = p.delta.bias ? load_as_f32(p.delta.bias, h * p.delta.sbias, p.delta.bias_type) : 0.f;
    if (OUT && lane < 32) D_l[lane] = p.D && lane < np ? load_as_f32(p.D, h * p.sD_h + (p0 + lane) * p.sD_p, p.D_type) : 0.f;

    // a chunk's rows of a tensor: what lies behind its last token reads as zero and is not written
    auto rows_of = [&](const uint16_t *base, int64_t stride, int t, int columns) {
        const int n = min(T, t1 - t);
        return __builtin_amdgcn_make_buffer_rsrc((void *)(base + t * stride), 0, n > 0 ? (int)((n - 1) * stride + columns) * 2 : 0, 0x00020000);
    };
    // Unit u of a row of B or C lies at place u ^ swizzle(row): neither eight rows' same unit nor four rows' four units share a bank.
    // (The rows that a lane reads differ by multiples of 16 in what it does not know at compile time, which leaves swizzle alone.)
    auto swizzle = [](int row) { return NK == 4 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3); };
    auto place = [&](int row, int u) { return row * ROW + (u ^ swizzle(row)) * 16; };
    auto xplace = [](int row, int u) { return row * 64 + (u ^ (row >> 2 & 3)) * 16; };
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    int offB[LOADS], offC[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const int slot = (wave * LOADS + k) * 64 + lane, row = slot / UNITS, u = slot % UNITS ^ swizzle(row);
        offB[k] = 8 * u < N ? (int)(row * p.sB_l + 8 * u) * 2 : kNowhere;
        offC[k] = 8 * u < N ? (int)(row * p.sC_l + 8 * u) * 2 : kNowhere;
    }
    const int xu = (lane & 3) ^ (lane >> 4), offX = 8 * xu < np ? (int)((lane >> 2) * p.sx_l + 8 * xu) * 2 : kNowhere;
    float dn = 0.f;
    int sn = 0;
    auto request = [&](int t, int half) {
        const __amdgpu_buffer_rsrc_t rB = rows_of(Bg, p.sB_l, t, N), rX = rows_of(x, p.sx_l, t, np);
#pragma unroll
        for (int k = 0; k < LOADS; ++k) into_lds(rB, offB[k], 0, base + half * HALF + (wave * LOADS + k) * 1024);
        if constexpr (OUT) {
            const __amdgpu_buffer_rsrc_t rC = rows_of(Cg, p.sC_l, t, N);
#pragma unroll
            for (int k = 0; k < LOADS; ++k) into_lds(rC, offC[k], 0, base + half * HALF + TILE + (wave * LOADS + k) * 1024);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) into_lds(rX, offX, (int)(16 * k * p.sx_l) * 2, base + xat + half * XTILE + k * 1024);
        const int tok = t + lane;
        dn = tok < t1 ? load_as_f32(p.dt, b * p.sdt_b + tok * p.sdt_l + h * p.sdt_h, p.dt_type) : 0.f;
        if constexpr (SEQ) {
            const int32_t *q = p.seq + b * p.sq_b;
            sn = tok < t1 && q[tok * p.sq_l] != (tok > 0 ? q[(tok - 1) * p.sq_l] : 0);
        }
    };

    // the state: S[ks][half][a][r] is column 32 ks + 8 g + 4 half + r of row 8 (i / 4) + 4 a + i % 4
    f32x4 S[NK][2][2];
    float *const ws = p.ws_states + ((((int64_t)b * p.nheads + h) * p.segments + seg) * P + p0) * N;
    auto row_of = [&](int a) { return 8 * (i >> 2) + 4 * a + (i & 3); };
    const float *const in = !OUT ? nullptr : p.segments > 1 ? ws : p.init ? (const float *)p.init + b * p.si_b + h * p.si_h + p0 * p.si_p : nullptr;
    const int64_t in_pitch = p.segments > 1 ? N : p.si_p;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                S[ks][half][a] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (in && 32 * ks + 8 * g < N && row_of(a) < np) S[ks][half][a] = *(const f32x4 *)&in[row_of(a) * in_pitch + 32 * ks + 8 * g + 4 * half];
            }
    float through = 0.f;        // log2 of the factor on what enters the segment
    bool passes = true;

    if (t0 < t1) {
        request(t0, 0);
        __builtin_amdgcn_s_waitcnt(vm_only(0));
    }
    int half_now = 0;
    for (int t = t0; t < t1; t += T, half_now ^= 1) {
        // steps and decays: lane = token
        const bool there = t + lane < t1;
        const float d = there ? delta_of(p.delta, dn + bias) : 0.f;
        const float a2 = d * A2, la = a2 < kLeast ? kLeast : a2;
        const bool dbad = !(fabsf(d) < __builtin_inff()) || !(fabsf(la) < __builtin_inff());
        const float cs = wave_inclusive_sum(la);
        const float cs_end = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, cs), 63));
        const float cs_mid = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, cs), 31));
        uint64_t starts = 0;
        if constexpr (SEQ) {
            starts = __ballot(sn);
            const uint64_t upto = starts & (~0ull >> (63 - lane));
            start_l[lane] = upto ? 63 - __builtin_clzll(upto) : -1;      // the lane's sequence from this token on; -1: it entered the chunk
        }
        const int from_end = SEQ && starts ? 63 - __builtin_clzll(starts) : 0;
        cs_l[lane] = cs;
        d_l[lane] = d;
        w_l[lane] = lane >= from_end ? pow2(cs_end - cs) * d : 0.f;
        if (OUT) mid_l[lane] = pow2(cs_mid - cs) * d;            // of the first 32 tokens, towards the others
        const bool whole = !SEQ || starts == 0;                  // the entering state reaches the chunk's end
        through += cs_end;
        passes = passes && whole;
        // every wave's part of this chunk is in LDS, and every wave is done with the chunk before
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        request(t + T, half_now ^ 1);
        asm volatile("" : "+v"(i), "+v"(g));       // addresses are made where they are used: kept over the loop they would not fit the registers
        const char *const Bl = lds + half_now * HALF, *const Cl = Bl + TILE, *const Xl = lds + xat + half_now * XTILE;

        bf16x8 xo[2][2];                                         // [32 tokens][a]: tokens 8 g .. of row row_of(a)
        uint32_t bad = 0;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int tok = 32 * kt + 8 * g + (i >> 2);
                xo[kt][a] = column8(Xl + xplace(tok, i & 3) + 8 * a, Xl + xplace(tok + 4, i & 3) + 8 * a);
                bad |= infinite(__builtin_bit_cast(u32x4, xo[kt][a]));
            }
        if (SEQ && starts) {
            // a weight of zero would not keep another sequence's NaN out of the state
            for (int k = lane; k < T * UNITS; k += 64) bad |= infinite(*(const u32x4 *)(Bl + 16 * k));
        }
        const bool slow = __any((OUT || starts ? bad : 0) != 0 || dbad);

        if (!slow && live) {
            if constexpr (OUT) {
                // y's transposed tiles: Y[tt][a][r] is row 8 g + 4 a + r of token 16 tt + i
                f32x4 Y[4][2];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) Y[tt][0] = Y[tt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    Parts s[2];
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = S[ks][e / 4][a][e % 4];
                        s[a] = split(v);
                    }
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) {
                        const bf16x8 c = row8(Cl + place(i, 4 * ks + g) + 16 * tt * ROW);
#pragma unroll
                        for (int a = 0; a < 2; ++a) Y[tt][a] = product(s[a].lo, c, product(s[a].hi, c, Y[tt][a]));
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                const __amdgpu_buffer_rsrc_t rZ = rows_of(z ? z : y, z ? p.sz_l : p.sy_l, t, z ? np : 0), rY = rows_of(y, p.sy_l, t, np);
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                    const float cst = cs_l[16 * tt + i], e = pow2(cst);
                    const int tok = 16 * tt + i;
                    const u32x4 zv = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rZ, 8 * g < np ? (int)(tok * p.sz_l + 8 * g) * 2 : kNowhere, 0, 0));
                    int first = 0;
                    bool entered = true;
                    if constexpr (SEQ) {
                        first = start_l[tok];
                        entered = first < 0;
                    }
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int r = 0; r < 4; ++r) Y[tt][a][r] = entered ? Y[tt][a][r] * e : 0.f;
                    bf16x8 c[NK];
#pragma unroll
                    for (int ks = 0; ks < NK; ++ks) c[ks] = row8(Cl + place(i, 4 * ks + g) + 16 * tt * ROW);
#pragma unroll
                    for (int kt = 0; kt <= tt / 2; ++kt) {
                        f32x4 G[2];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            G[half] = f32x4{0.f, 0.f, 0.f, 0.f};
                            const int j = 8 * (i >> 2) + 4 * half + (i & 3);
#pragma unroll
                            for (int ks = 0; ks < NK; ++ks) G[half] = product(row8(Bl + place(j, 4 * ks + g) + 32 * kt * ROW), c[ks], G[half]);
                        }
                        float m[8];
                        const float reach = pow2(cst - cs_mid);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int j0 = 32 * kt + 8 * g + 4 * half;
                            if (kt < tt / 2) {
                                // all of these tokens are behind the first 32: their decay in two factors, one per token of each side
                                const f32x4 mj = *(const f32x4 *)&mid_l[j0];
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const float v = G[half][r] * (reach * mj[r]);
                                    m[4 * half + r] = !SEQ || j0 + r >= first ? v : 0.f;
                                }
                            } else {
                                const f32x4 dj = *(const f32x4 *)&d_l[j0], cj = *(const f32x4 *)&cs_l[j0];
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const float v = G[half][r] * (pow2(cst - cj[r]) * dj[r]);
                                    m[4 * half + r] = j0 + r <= tok && (!SEQ || j0 + r >= first) ? v : 0.f;
                                }
                            }
                        }
                        const Parts mp = split(m);
#pragma unroll
                        for (int a = 0; a < 2; ++a) Y[tt][a] = product(xo[kt][a], mp.lo, product(xo[kt][a], mp.hi, Y[tt][a]));
                    }
                    // skip, gate, 16 bytes per lane
                    const f32x4 D0 = *(const f32x4 *)&D_l[8 * g], D1 = *(const f32x4 *)&D_l[8 * g + 4];
                    const u32x4 xv = *(const u32x4 *)(Xl + xplace(tok, g));
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = fmaf(e < 4 ? D0[e % 4] : D1[e % 4], half_of(xv, e), Y[tt][e / 4][e % 4]);
                    if (z)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] *= silu(half_of(zv, e));
                    u32x4 out;
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[e] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * e], (__bf16)v[2 * e + 1]});
                    __builtin_amdgcn_raw_buffer_store_b128(out, rY, 8 * g < np ? (int)(tok * p.sy_l + 8 * g) * 2 : kNowhere, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // the state behind the chunk
            const float keep = pow2(cs_end);
#pragma unroll
            for (int ks = 0; ks < NK; ++ks)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[ks][half][a][r] = whole ? S[ks][half][a][r] * keep : 0.f;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const f32x4 w0 = *(const f32x4 *)&w_l[32 * kt + 8 * g], w1 = *(const f32x4 *)&w_l[32 * kt + 8 * g + 4];
                Parts xw[2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const u32x4 raw = __builtin_bit_cast(u32x4, xo[kt][a]);
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = half_of(raw, e) * (e < 4 ? w0[e % 4] : w1[e % 4]);
                    xw[a] = split(v);
                }
                const int tok = 8 * g + (i >> 2);
#pragma unroll
                for (int ks = 0; ks < NK; ++ks)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const bf16x8 bt = column8(Bl + place(tok, 4 * ks + (i & 3)) + 32 * kt * ROW + 8 * half,
                                                  Bl + place(tok + 4, 4 * ks + (i & 3)) + 32 * kt * ROW + 8 * half);
#pragma unroll
                        for (int a = 0; a < 2; ++a) S[ks][half][a] = product(bt, xw[a].lo, product(bt, xw[a].hi, S[ks][half][a]));
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            // the requests for the next chunk are older than this chunk's four stores
            if constexpr (OUT) __builtin_amdgcn_s_waitcnt(vm_only(4));
            else __builtin_amdgcn_s_waitcnt(vm_only(0));
        } else if (live) {
            // token by token: lanes of the same i share a row's columns
            w_l[lane] = la;
            for (int k = 0; k < T && t + k < t1; ++k) {
                const bool fresh = SEQ && (starts >> k & 1);
                const float keep = pow2(w_l[k]), dk = d_l[k];
                float xv[2], sum[2] = {0.f, 0.f};
#pragma unroll
                for (int a = 0; a < 2; ++a) xv[a] = bf16_bits_to_f32(*(const uint16_t *)(Xl + xplace(k, i >> 2) + 8 * a + 2 * (i & 3)));
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    const u32x4 bv = *(const u32x4 *)(Bl + place(k, 4 * ks + g));
                    u32x4 cv = {0, 0, 0, 0};
                    if constexpr (OUT) cv = *(const u32x4 *)(Cl + place(k, 4 * ks + g));
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
#pragma unroll
                        for (int a = 0; a < 2; ++a) {
                            const float s = fresh ? 0.f : S[ks][e / 4][a][e % 4] * keep;
                            // columns behind dstate hold zeros and stay so
                            S[ks][e / 4][a][e % 4] = 32 * ks + 8 * g < N ? fmaf(dk * xv[a], half_of(bv, e), s) : 0.f;
                            sum[a] = fmaf(S[ks][e / 4][a][e % 4], half_of(cv, e), sum[a]);
                        }
                    }
                }
                if constexpr (OUT) {
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        float v = sum[a] + __shfl_xor(sum[a], 16);
                        v += __shfl_xor(v, 32);
                        const int row = row_of(a);
                        if (g == a && row < np) {
                            v = p.D ? fmaf(D_l[row], xv[a], v) : v;
                            if (z) v *= silu(bf16_bits_to_f32(z[(t + k) * p.sz_l + row]));
                            y[(t + k) * p.sy_l + row] = f32_to_bf16_bits(v);
                        }
                    }
                }
            }
            __builtin_amdgcn_s_waitcnt(vm_only(0));
        } else __builtin_amdgcn_s_waitcnt(vm_only(0));
        asm volatile("" ::: "memory");
    }
    if constexpr (OUT) {
        for (int t = max(t0, t1); t < t_end; ++t)
            if (lane < 32 && lane < np) y[t * p.sy_l + lane] = 0;
    }
    if (!OUT || seg == p.segments - 1) {
        float *to = OUT ? p.fin + b * p.sf_b + h * p.sf_h + p0 * p.sf_p : ws;
        const int64_t pitch = OUT ? p.sf_p : N;
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int a = 0; a < 2; ++a)
                    if (32 * ks + 8 * g < N && row_of(a) < np) *(f32x4 *)&to[row_of(a) * pitch + 32 * ks + 8 * g + 4 * half] = S[ks][half][a];
    }
    if (!OUT && live && lane == 0 && p0 == 0) p.ws_decay[((int64_t)b * p.nheads + h) * p.segments + seg] = passes ? pow2(through) : -1.f;
}

template <int NK, bool SEQ>
hipError_t run(const SelScanParams &p, hipStream_t s)
{
    const int blocks_per_head = (p.headdim + 31) / 32;
    const int64_t units = (int64_t)(p.nheads / p.ngroups) * blocks_per_head, sets = (units + kWaves - 1) / kWaves;
    const int64_t blocks = sets * p.ngroups * p.segments * p.batch;
    if (blocks * 64 * kWaves > 0xffffffffLL || units > 0x7fffffffLL) return hipErrorInvalidConfiguration;
    constexpr int common = kWaves * (2 * T * 64 + META * 4), tile = 2 * T * 64 * NK;
    static std::atomic<uint64_t> done[2];
    hipError_t e = ensure_dynamic_lds((const void *)chunk_kernel<NK, true, SEQ>, common + 2 * tile, done[0]);
    if (e == hipSuccess) e = ensure_dynamic_lds((const void *)chunk_kernel<NK, false, SEQ>, common + tile, done[1]);
    if (e != hipSuccess) return e;
    if (p.segments > 1) {
        hipLaunchKernelGGL((chunk_kernel<NK, false, SEQ>), dim3((uint32_t)blocks), dim3(64 * kWaves), common + tile, s, p, blocks_per_head, (int)sets);
        e = hipGetLastError();
        if (e == hipSuccess) e = launch_scan_join(p, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((chunk_kernel<NK, true, SEQ>), dim3((uint32_t)blocks), dim3(64 * kWaves), common + 2 * tile, s, p, blocks_per_head, (int)sets);
    return hipGetLastError();
}

}  // namespace

bool scan_mfma_supported(const SelScanParams &p)
{
    if (p.type != DT_BF16 || p.dstate > 128 || p.headdim % 8 || p.dstate % 8) return false;
    // 16-byte pieces of rows, offsets inside a chunk of 64 tokens in 31 bits
    auto rows = [](const void *base, int64_t s_b, int64_t s_l, int64_t s_h) {
        return ((uintptr_t)base & 15) == 0 && (s_b | s_l | s_h) % 8 == 0 && s_l >= 0 && s_l < (1 << 23);
    };
    auto states = [](const void *base, int64_t s_b, int64_t s_h, int64_t s_p) { return ((uintptr_t)base & 15) == 0 && (s_b | s_h | s_p) % 4 == 0; };
    return rows(p.x, p.sx_b, p.sx_l, p.sx_h) && rows(p.B, p.sB_b, p.sB_l, p.sB_g) && rows(p.C, p.sC_b, p.sC_l, p.sC_g) && rows(p.y, p.sy_b, p.sy_l, p.sy_h) &&
           (!p.z || rows(p.z, p.sz_b, p.sz_l, p.sz_h)) && states(p.fin, p.sf_b, p.sf_h, p.sf_p) &&
           (!p.init || (p.init_type == DT_F32 && states(p.init, p.si_b, p.si_h, p.si_p)));
}

hipError_t launch_scan_mfma(const SelScanParams &p, hipStream_t s)
{
    if (p.dstate <= 64) return p.seq ? run<2, true>(p, s) : run<2, false>(p, s);
    return p.seq ? run<4, true>(p, s) : run<4, false>(p, s);
}

}  // namespace ssd
