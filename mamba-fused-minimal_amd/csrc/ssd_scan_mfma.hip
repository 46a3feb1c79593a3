// The selective scan of prompts on the bf16 matrix instructions: bf16 x, B, C, z in rows at multiples of 16 bytes, initial states in fp32, dstate
// up to 128, dstate and headdim multiples of 8 (scan_mfma_supported).
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
// one part alone would add as much error as the rounding of y).  Sums, states and decays are fp32, sums of log-decays 64 bits.  The final
// states are within 2.2e-6 of their norm, behind strong decays as behind weak ones; a third part of the weighted x would make that 2e-7 and
// 4 x 8192 tokens x 80 heads 552 us instead of 498 (both without the first segment in front).
//
// Values that are not finite: a masked factor is selected away, not multiplied by zero, but a matrix product would still carry a
// NaN of x_j to the tokens in front of j, and an infinity split into two parts is an infinity and a NaN.  A chunk in which x, B, C or d is
// not finite, or which a state with an infinity enters, is therefore taken token by token (slow path): they reach what they reach in the
// recurrence.  A segment whose results are not finite is walked a second time to find out which chunks these are: a NaN in one of four
// rows of 8192 tokens makes the call twice, an infinity that stays in a state nine times as long.
//
// Rows are cut into segments where heads are too few for the card.  A first launch computes what each but the last adds to a state of
// zero (two fifths of the work, without C, z and y) -- or, where rows are long, the first segment in full and what the middle ones
// add beside it -- and a second one the segments with y, from the state that the segments in front leave.
//
// What bounds it: 4 x 8192 tokens of 80 heads of 64 x 128 with gate and states take 466 to 484 us, from card to card (profiled on its own,
// with clocks that have not settled: 23 + 131 + 418 for the steps, the launch in front and the one with y).  1050 MB of x, z, y and
// states are 202 us of that at a copy's rate.  A chunk takes the eight waves of a workgroup, two to a SIMD, 18.9 thousand cycles: each has
// 1400 vector instructions (splitting operands, scores) and 200 matrix instructions, the matrix unit is busy a quarter of the time, and
// 37 % of a wave's time is waits at the two barriers and for LDS and memory, which a third wave on the SIMD would fill; its registers (243
// of 256) leave no room for one.  A part of the waits is of this order of things, not of the registers: the last rows of x and z are asked
// for directly in front of the wait that ends a chunk, which also drains its stores.
#include "ssd_layer.h"
#include "ssd_tile.h"

namespace ssd {
namespace {

using namespace layer;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int T = 64;                 // tokens per chunk
constexpr double kLog2e = 1.4426950408889634;
constexpr double kLeast = -160.;      // of log2(decay): 2^-160 is zero in fp32 already, and 64 such in front of weaker ones leave those their bits

__device__ __forceinline__ float pow2(float v) { return __builtin_amdgcn_exp2f(v); }

// eight values -> two bf16 parts each
struct Parts { bf16x8 hi, lo; };
__device__ __forceinline__ Parts split(const float (&v)[8])
{
    Parts r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const bf16x2 h = {(__bf16)v[j], (__bf16)v[j + 1]};
        uint32_t b = __builtin_bit_cast(uint32_t, h);
#if defined(__HIP_DEVICE_COMPILE__)
        asm("" : "+v"(b));        // (or the compiler converts the first value a second time to get its high part)
#endif
        const bf16x2 l = {(__bf16)(v[j] - __builtin_bit_cast(float, b << 16)), (__bf16)(v[j + 1] - __builtin_bit_cast(float, b & 0xffff0000u))};
        r.hi[j] = __builtin_bit_cast(bf16x2, b)[0]; r.hi[j + 1] = __builtin_bit_cast(bf16x2, b)[1];
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
// 64 lanes x 4 bytes
__device__ __forceinline__ void words_into_lds(__amdgpu_buffer_rsrc_t from, int offset, int more, uint32_t to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(to), "v"(offset), "s"(from), "s"(more) : "memory");
#endif
}
__device__ __forceinline__ constexpr int vm_only(int n) { return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14); }
constexpr int kLgkmZero = 15 | (7 << 4) | (0 << 8) | (3 << 14);

// the larger of each 16-bit half: of values without their signs, which are not finite from 0x7f80 on
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
__device__ __forceinline__ u16x2 largest(u16x2 so_far, u32x4 v)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) so_far = __builtin_elementwise_max(so_far, __builtin_bit_cast(u16x2, v[j] & 0x7fff7fffu));
    return so_far;
}

// a token's 8 values of 16-bit type as fp32
__device__ __forceinline__ float half_of(const u32x4 &v, int e) { return __builtin_bit_cast(float, e % 2 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16); }

constexpr float kFar = 100.f;      // log2 of the largest factor that one side's decay is scaled by

// ---- steps and decays ------------------------------------------------------------------------------------------------

// A record of a (row, head, chunk): arrays over its 64 tokens, in this order.  cs: running sum of log2 of the decays, made in 64 bits: a
// decay between two tokens is the exponential of a difference of sums, and behind tokens that let nothing pass those are
// thousands (in fp32 alone the weights behind 40 such tokens were off by 7e-4).
//   weight   2^(cs_63 - cs) d: what a token adds to the state behind the chunk (0: another sequence's)
//   cs       rounded to fp32
//   score    2^(cs_e - cs) d with e = the last of the token's 32: its side of the decay towards a later token
//   mark     high half: what the rounding of cs left, as bf16 (|cs| <= 64 x 160: up to 2^-11, known to 2^-20); low byte: the token from which
//            on the chunk belongs to the token's sequence, -1 where that entered the chunk; bit 8 of the last one: some step is not
//            finite, go token by token
//   d        (not kept in LDS: for what is rare)
// score[0] is NaN where some 2^(cs_e - cs) would be out of range: the scores then take the exponential of the difference.
constexpr int RECORD = 5 * T;
enum : int { WEIGHT = 0, CS = T, SCORE = 2 * T, MARK = 3 * T, STEP = 4 * T };
constexpr int kHeadTile = 32;
__device__ __forceinline__ int start_of(uint32_t mark) { return (int8_t)mark; }
__device__ __forceinline__ bool serial(uint32_t last_mark) { return last_mark & 0x100; }
__device__ __forceinline__ float rest_of(uint32_t mark) { return __builtin_bit_cast(float, mark & 0xffff0000u); }

// wave_inclusive_sum in 64 bits
__device__ __forceinline__ double inclusive_sum(double x)
{
#if defined(__HIP_DEVICE_COMPILE__)
    auto shifted = [](double v, auto ctrl, auto rows) {
        const u32x2 w = __builtin_bit_cast(u32x2, v);
        u32x2 r;
#pragma unroll
        for (int k = 0; k < 2; ++k) r[k] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], decltype(ctrl)::value, decltype(rows)::value, 0xf, true);
        return __builtin_bit_cast(double, r);
    };
    using std::integral_constant;
    typedef integral_constant<int, 0xf> all;
    x += shifted(x, integral_constant<int, 0x111>{}, all{});     // row_shr:1
    x += shifted(x, integral_constant<int, 0x112>{}, all{});     // row_shr:2
    x += shifted(x, integral_constant<int, 0x114>{}, all{});     // row_shr:4
    x += shifted(x, integral_constant<int, 0x118>{}, all{});     // row_shr:8
    x += shifted(x, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});     // row_bcast:15 into rows 1, 3
    x += shifted(x, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});     // row_bcast:31 into rows 2, 3
#endif
    return x;
}
__device__ __forceinline__ double of_lane(double v, int lane)
{
    u32x2 w = __builtin_bit_cast(u32x2, v);
#pragma unroll
    for (int k = 0; k < 2; ++k) w[k] = (uint32_t)__builtin_amdgcn_readlane((int)w[k], lane);
    return __builtin_bit_cast(double, w);
}

// A workgroup takes 32 heads of a chunk, whose steps come as rows of heads, through LDS; a wave then has a head's tokens in its lanes.
template <bool SEQ>
__global__ void __launch_bounds__(256) steps_kernel(const SelScanParams p, int head_tiles)
{
    __shared__ float tile[kHeadTile][T + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h0 = (int)(blockIdx.x % (uint32_t)head_tiles) * kHeadTile, c = (int)(blockIdx.x / (uint32_t)head_tiles % (uint32_t)p.chunks),
              b = (int)(blockIdx.x / (uint32_t)head_tiles / (uint32_t)p.chunks);
    const int t0 = c * T, len = row_tokens(p.len, p.slen, b, p.seqlen), hh = tid % kHeadTile, h = h0 + hh;
    const float bias = h < p.nheads && p.delta.bias ? load_as_f32(p.delta.bias, h * p.delta.sbias, p.delta.bias_type) : 0.f;
    float raw[T / 8];
#pragma unroll
    for (int k = 0; k < T / 8; ++k) {
        const int tok = t0 + tid / kHeadTile + 8 * k;
        raw[k] = tok < len && h < p.nheads ? load_as_f32(p.dt, b * p.sdt_b + tok * p.sdt_l + h * p.sdt_h, p.dt_type) : 0.f;
    }
    int starts_here = 0;
    if constexpr (SEQ) {
        const int32_t *q = p.seq + b * p.sq_b;
        const int tok = t0 + lane;
        starts_here = tok < len && q[tok * p.sq_l] != (tok > 0 ? q[(tok - 1) * p.sq_l] : 0);
    }
#pragma unroll
    for (int k = 0; k < T / 8; ++k) {
        const int at = tid / kHeadTile + 8 * k;
        tile[hh][at] = t0 + at < len ? delta_of(p.delta, raw[k] + bias) : 0.f;
    }
    __syncthreads();
    const uint64_t starts = SEQ ? __ballot(starts_here) : 0;
    const uint64_t upto = starts & (~0ull >> (63 - lane));
    const int from_end = starts ? 63 - __builtin_clzll(starts) : 0;
#pragma unroll 2
    for (int k = 0; k < kHeadTile / 4; ++k) {
        const int hl = wave * (kHeadTile / 4) + k, hd = h0 + hl;
        if (hd >= p.nheads) break;
        const float d = tile[hl][lane];
        const double a2 = (double)d * (double)load_as_f32(p.A, hd * p.sA, p.A_type) * kLog2e, la = a2 < kLeast ? kLeast : a2;
        const double sum = inclusive_sum(la), end = of_lane(sum, 63), mid = of_lane(sum, 31);
        const bool bad = __any(!(fabsf(d) < __builtin_inff()) || !(fabsf((float)la) < __builtin_inff()));
        const float cs = (float)sum, back = (float)((lane < 32 ? mid : end) - sum);
        const bool far = __any(!(fabsf(back) < kFar));
        float *r = p.ws_steps + (((int64_t)b * p.nheads + hd) * p.chunks + c) * RECORD + lane;
        r[WEIGHT] = lane >= from_end ? pow2((float)(end - sum)) * d : 0.f;
        r[CS] = cs;
        r[SCORE] = far && lane == 0 ? __builtin_nanf("") : pow2(back) * d;
        r[STEP] = d;
        const int start = upto ? 63 - __builtin_clzll(upto) : -1;
        ((uint32_t *)r)[MARK] = (uint32_t)f32_to_bf16_bits((float)(sum - (double)cs)) << 16 | (bad ? 0x100u : 0u) | (uint8_t)start;
    }
}

// ---- the walk ----------------------------------------------------------------------------------------------------------

constexpr int WAVES = 8;

struct Place { int set, group, segment, row; };
// XCDs get workgroups in turn: each gets a contiguous part, whose workgroups share B and C.  `segments` of them from `first` on.
__device__ __forceinline__ Place place_of_workgroup(const SelScanParams &p, int sets, int first, int segments)
{
    const int total = (int)gridDim.x, per = total / 8, id = (int)blockIdx.x;
    int at = id < per * 8 ? (id % 8) * per + id / 8 : id;
    Place r;
    r.set = at % sets; at /= sets;
    r.group = at % p.ngroups; at /= p.ngroups;
    r.segment = first + at % segments;
    r.row = at / segments;
    return r;
}

// NK: 32-column steps of dstate; OUT: write y (otherwise only what the segment adds and the factor on what enters it); GATE: z;
// SEQ: seq_idx; LEAVE: write the state behind the segment, or what it adds, and the factor to the workspace.  Only a launch in front of
// the one that reads them may: workgroups of one launch start and end in no order.
// `careful`: look in every chunk for what is not finite in x, B and C and for infinities in the state.  Otherwise that would cost 2 to 5 %:
// results show it, scores and y or, without y, the state that is left, and the walk returns true to all of the workgroup in front of
// writing states, to be done again with care.
template <int NK, bool OUT, bool GATE, bool SEQ, bool LEAVE>
__device__ __forceinline__ bool walk_once(const SelScanParams &p, int blocks_per_head, const Place &place_of, bool careful)
{
    static_assert(OUT || LEAVE, "a walk without y is there for what it leaves");
    constexpr int UNITS = 4 * NK, ROW = 16 * UNITS, TILE = T * ROW;     // 16-byte units and bytes of a token's B or C; bytes of a chunk's
    constexpr int RING = OUT ? 2 : 3;                                   // chunks of B (and C) and of records in LDS
    constexpr int XRING = OUT ? 1 : 3;                                  // of x; with y (and z) a chunk's rows make room for the next one's when they are used
    constexpr int PART = (OUT ? 2 : 1) * TILE, XTILE = T * 64;          // bytes of B (and C), and of a wave's x (or z), per chunk
    // bytes of a record in LDS; without y the weights, and in front of 64 more words the chunk's last cs and mark
    constexpr int REC = OUT ? STEP * 4 : 2 * T * 4;
    constexpr int LOADS = TILE / 1024 / WAVES;                          // of B per wave and chunk, and of C
    constexpr int REQUESTS = LOADS + 4 + 2;                             // of a wave and chunk without y
    constexpr int SCORES = OUT ? 12 * 1024 : 0;                         // bytes of a chunk's scores
    constexpr int MINE = XRING * XTILE + (OUT ? XTILE + 128 : 0) + RING * REC;      // a wave's own LDS: x, z, D, records
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tid = threadIdx.x;
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(tid));
#endif
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int i = lane & 15, g = lane >> 4;
    const int xat = RING * PART + SCORES + wave * MINE, zat = xat + XRING * XTILE, rat = zat + (OUT ? XTILE + 128 : 0);
    float *const D_l = (float *)(lds + zat + XTILE);
    char *const Gl = lds + RING * PART;

    const int set = place_of.set, gr = place_of.group, seg = place_of.segment, b = place_of.row;
    const int heads = p.nheads / p.ngroups, unit = set * WAVES + wave;
    const bool live = unit < heads * blocks_per_head;
    const int h = gr * heads + (live ? unit / blocks_per_head : 0), p0 = live ? unit % blocks_per_head * 32 : 0;
    const int N = p.dstate, np = live ? p.headdim - p0 : 0;             // rows from p0 on
    const int len = row_tokens(p.len, p.slen, b, p.seqlen);
    const int t0 = seg == 0 ? 0 : p.head_tokens + (seg - 1) * p.segment_tokens, t_end = min(seg == 0 ? p.head_tokens : t0 + p.segment_tokens, p.seqlen),
              t1 = min(t_end, len);
    if (OUT && lane < 32) D_l[lane] = p.D && lane < np ? load_as_f32(p.D, h * p.sD_h + (p0 + lane) * p.sD_p, p.D_type) : 0.f;

    // the rows of the chunk to be requested next (x, z, B, C) or written now (y): a pointer that moves on, and the bytes of a row
    struct Rows {
        const char *at;
        int pitch, width;
        __device__ __forceinline__ Rows(const void *base, int64_t first, int64_t stride, int columns) : at((const char *)base + 2 * first), pitch((int)stride * 2), width(columns * 2) {}
        // n rows; what lies behind reads as zero and is not written
        __device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(int n) const
        {
            return __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, n > 0 ? (n - 1) * pitch + width : 0, 0x00020000);
        }
        __device__ __forceinline__ void next() { at += T * pitch; }
    };
    Rows xr(p.x, b * p.sx_b + t0 * p.sx_l + h * p.sx_h + p0, p.sx_l, np), Br(p.B, b * p.sB_b + t0 * p.sB_l + gr * p.sB_g, p.sB_l, N),
        Cr(p.C, b * p.sC_b + t0 * p.sC_l + gr * p.sC_g, p.sC_l, OUT ? N : 0), yr(p.y, b * p.sy_b + t0 * p.sy_l + h * p.sy_h + p0, p.sy_l, OUT ? np : 0),
        zr(p.z, b * p.sz_b + t0 * p.sz_l + h * p.sz_h + p0, p.sz_l, GATE ? np : 0);

    // Unit u of a row of B or C lies at place u ^ swizzle(row): neither eight rows' same unit nor four rows' four units share a bank.
    // (The rows that a lane reads differ by multiples of 16 in what it does not know at compile time, which leaves swizzle alone.)
    auto swizzle = [](int row) { return NK == 4 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3); };
    auto place = [&](int row, int u) { return row * ROW + (u ^ swizzle(row)) * 16; };
    auto xplace = [](int row, int u) { return row * 64 + (u ^ (row >> 2 & 3)) * 16; };
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    int offB[LOADS], offC[OUT ? LOADS : 1];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const int slot = (wave * LOADS + k) * 64 + lane, row = slot / UNITS, u = slot % UNITS ^ swizzle(row);
        offB[k] = 8 * u < N ? row * Br.pitch + 16 * u : kNowhere;
        if constexpr (OUT) offC[k] = 8 * u < N ? row * Cr.pitch + 16 * u : kNowhere;
    }
    const int xu = (lane & 3) ^ (lane >> 4), offX = 8 * xu < np ? (lane >> 2) * xr.pitch + 16 * xu : kNowhere,
              offZ = 8 * xu < np ? (lane >> 2) * zr.pitch + 16 * xu : kNowhere;
    const int offY = 8 * g < np ? i * yr.pitch + 16 * g : kNowhere;
    const int64_t record = ((int64_t)b * p.nheads + h) * p.chunks + t0 / T;
    const float *steps = p.ws_steps + record * RECORD;
    const int off_last = lane == 0 ? (CS + T - 1) * 4 : lane == 1 ? (MARK + T - 1) * 4 : kNowhere;
    // B, C and the records of the chunk at token t into slot `to` of LDS
    auto request = [&](int t, int to) {
        const int n = min(T, t1 - t);
        const __amdgpu_buffer_rsrc_t rB = Br.descriptor(n), rR = __builtin_amdgcn_make_buffer_rsrc((void *)steps, 0, n > 0 ? RECORD * 4 : 0, 0x00020000);
#pragma unroll
        for (int k = 0; k < LOADS; ++k) into_lds(rB, offB[k], 0, base + to * PART + (wave * LOADS + k) * 1024);
        if constexpr (OUT) {
            const __amdgpu_buffer_rsrc_t rC = Cr.descriptor(n);
#pragma unroll
            for (int k = 0; k < LOADS; ++k) into_lds(rC, offC[k], 0, base + to * PART + TILE + (wave * LOADS + k) * 1024);
            Cr.next();
            into_lds(rR, lane * 16, 0, base + rat + to * REC);
        } else {
            words_into_lds(rR, lane * 4, WEIGHT * 4, base + rat + to * REC);
            words_into_lds(rR, off_last, 0, base + rat + to * REC + T * 4);
        }
        Br.next();
        steps += RECORD;
    };
    // 16 rows of x (and z) of the chunk at token t into slot `to`
    auto request_rows = [&](int t, int tt, int to) {
        const int n = min(T, t1 - t);
        into_lds(xr.descriptor(n), offX, 16 * tt * xr.pitch, base + xat + to * XTILE + tt * 1024);
        if constexpr (GATE) into_lds(zr.descriptor(n), offZ, 16 * tt * zr.pitch, base + zat + tt * 1024);
    };

    // the state: S[ks][half][a][r] is column 32 ks + 8 g + 4 half + r of row 8 (i / 4) + 4 a + i % 4
    f32x4 S[NK][2][2];
    const int64_t plane = (int64_t)p.headdim * N;
    float *const ws = p.ws_states + (((int64_t)b * p.nheads + h) * p.segments + seg) * plane + (int64_t)p0 * N;
    auto row_of = [&](int a) { return 8 * (i >> 2) + 4 * a + (i & 3); };
    auto all_states = [&](auto &&f) {
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int a = 0; a < 2; ++a) f(S[ks][half][a], 32 * ks + 8 * g + 4 * half, row_of(a), 32 * ks + 8 * g < N && row_of(a) < np);
    };
    all_states([&](f32x4 &v, int n, int row, bool there) {
        v = f32x4{0.f, 0.f, 0.f, 0.f};
        const float *in = !OUT ? nullptr : p.joined ? ws + row * N : p.init ? (const float *)p.init + b * p.si_b + h * p.si_h + (p0 + row) * p.si_p : nullptr;
        if (in && there) v = *(const f32x4 *)&in[n];
    });
    if (OUT && !p.joined) {
        // few segments: the state entering this one from what those in front of it add
        const float *decay = p.ws_decay + ((int64_t)b * p.nheads + h) * p.segments;
        for (int k = 0; k < seg; ++k) {
            const float f = decay[k];
            const float *add = ws + (k - seg) * plane;
            all_states([&](f32x4 &v, int n, int row, bool there) {
                f32x4 more = {0.f, 0.f, 0.f, 0.f};
                if (there) more = *(const f32x4 *)&add[row * N + n];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = f < 0.f ? more[r] : fmaf(f, v[r], more[r]);
            });
        }
    }
    // The loads above are waited for here: the compiler would wait in the loop, for everything under way, at the states' first use.
    all_states([&](f32x4 &v, int, int, bool) { asm volatile("" : "+v"(v)); });
    float through = 0.f;        // log2 of the factor on what enters the segment
    bool passes = true;
    float probe = 0.f;          // a NaN where something was not finite

    if (t0 < t1) {
#pragma unroll
        for (int k = 0; k < RING - 1; ++k) {
            request(t0 + k * T, k);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) request_rows(t0 + k * T, tt, k);
            xr.next();
        }
        zr.next();
        __builtin_amdgcn_s_waitcnt(vm_only(OUT ? 0 : REQUESTS));
    }
    int slot = 0;
    for (int t = t0; t < t1; t += T) {
        // every wave's part of this chunk is in LDS, and every wave is done with the chunk before
        __builtin_amdgcn_s_barrier();
        asm volatile("" : "+v"(i), "+v"(g)::"memory");           // (addresses are made where they are used: kept over the loop they would not fit)
        const int ahead = t + (RING - 1) * T, free_slot = slot == 0 ? RING - 1 : slot - 1;
        request(ahead, free_slot);
        if constexpr (!OUT) {
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) request_rows(ahead, tt, free_slot);
            xr.next();
        }
        const char *const Bl = lds + slot * PART, *const Cl = Bl + TILE, *const Xl = lds + xat + (OUT ? 0 : slot) * XTILE, *const Zl = lds + zat;
        const float *const rec = (const float *)(lds + rat + slot * REC), *const w_l = rec + WEIGHT;
        const uint32_t *const mark_l = (const uint32_t *)rec + MARK;

        bool careful_slow = false;
        if (careful) {
            u16x2 most = {0, 0};
            bool infinite = false;
            for (int k = lane; k < XTILE / 16; k += 64) most = largest(most, *(const u32x4 *)(Xl + 16 * k));
            for (int k = lane; k < T * UNITS; k += 64) {
                most = largest(most, *(const u32x4 *)(Bl + 16 * k));
                if constexpr (OUT) most = largest(most, *(const u32x4 *)(Cl + 16 * k));
            }
            all_states([&](f32x4 &v, int, int, bool) {
#pragma unroll
                for (int r = 0; r < 4; ++r) infinite = infinite || fabsf(v[r]) == __builtin_inff();
            });
            careful_slow = __any(infinite || most[0] >= 0x7f80 || most[1] >= 0x7f80);
        }
        bf16x8 xo[2][2];                                         // [32 tokens][a]: tokens 8 g .. of row row_of(a)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int tok = 32 * kt + 8 * g + (i >> 2);
                xo[kt][a] = column8(Xl + xplace(tok, i & 3) + 8 * a, Xl + xplace(tok + 4, i & 3) + 8 * a);
            }
        auto C_row = [&](int tt, int ks) { return row8(Cl + place(i, 4 * ks + g) + 16 * tt * ROW); };
        auto B_column = [&](int kt, int ks, int half) {
            const int tok = 8 * g + (i >> 2);
            return column8(Bl + place(tok, 4 * ks + (i & 3)) + 32 * kt * ROW + 8 * half, Bl + place(tok + 4, 4 * ks + (i & 3)) + 32 * kt * ROW + 8 * half);
        };
        auto uniform = [](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); };
        const float cs_end = uniform(OUT ? rec[CS + T - 1] : rec[T]);
        const uint32_t last_mark = __builtin_amdgcn_readfirstlane(OUT ? mark_l[T - 1] : ((const uint32_t *)rec)[T + 1]);
        const bool starts = SEQ && start_of(last_mark) >= 0;
        const bool whole = !starts;                              // the entering state reaches the chunk's end
        through += cs_end;
        passes = passes && whole;
        const bool slow = careful_slow || serial(last_mark) || !(fabsf(cs_end) < __builtin_inff());

        if (slow && live) {
            // token by token: lanes of the same i share a row's columns
            const float *const now = steps - RING * RECORD;
            const double A2 = (double)load_as_f32(p.A, h * p.sA, p.A_type) * kLog2e;
            const uint16_t *const z = (const uint16_t *)(zr.at - T * zr.pitch);
            uint16_t *const y = (uint16_t *)yr.at;
            for (int k = 0; k < T && t + k < t1; ++k) {
                const bool fresh = SEQ && start_of(((const uint32_t *)now)[MARK + k]) == k;
                const double a2 = (double)now[STEP + k] * A2;
                const float dk = now[STEP + k], keep = pow2((float)(a2 < kLeast ? kLeast : a2));
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
                            if constexpr (GATE) v *= silu(bf16_bits_to_f32(z[k * (zr.pitch / 2) + row]));
                            y[k * (yr.pitch / 2) + row] = f32_to_bf16_bits(v);
                        }
                    }
                }
            }
        }
        if (OUT && (slow || !live)) {
            __builtin_amdgcn_s_waitcnt(kLgkmZero);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) request_rows(t + T, tt, 0);
        }
        // Products and vector instructions are interleaved all along: a wave can issue three or four of the latter while one of the former
        // runs, and the waves of a workgroup, which start a chunk together, are otherwise all at the one or all at the other.
        auto mixed = [](auto products, auto vectors) {
#pragma unroll
            for (int k = 0; k < decltype(products)::value; ++k) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, decltype(vectors)::value, 0);
            }
        };
        using std::integral_constant;
        // weighted x of 32 tokens, two parts
        auto weighted = [&](int kt, Parts (&xw)[2]) {
            const f32x4 w0 = *(const f32x4 *)&w_l[32 * kt + 8 * g], w1 = *(const f32x4 *)&w_l[32 * kt + 8 * g + 4];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const u32x4 raw = __builtin_bit_cast(u32x4, xo[kt][a]);
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = half_of(raw, e) * (e < 4 ? w0[e % 4] : w1[e % 4]);
                xw[a] = split(v);
            }
        };
        // two tiles of the state behind 32 tokens; in front of the first 32 they decay by the whole chunk
        const float keep = pow2(cs_end);
        auto update = [&](int kt, int ks, int half, const bf16x8 &bt, const Parts (&xw)[2]) {
            if (kt == 0)
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[ks][half][a][r] = whole ? S[ks][half][a][r] * keep : 0.f;
#pragma unroll
            for (int a = 0; a < 2; ++a) S[ks][half][a] = product(bt, xw[a].hi, S[ks][half][a]);
#pragma unroll
            for (int a = 0; a < 2; ++a) S[ks][half][a] = product(bt, xw[a].lo, S[ks][half][a]);
        };
        Parts xw[2];
        if constexpr (!OUT) {
            if (!slow && live) {
                bf16x8 bt[NK][2];
#pragma unroll
                for (int k = 0; k < 2 * NK; ++k) bt[k / 2][k % 2] = B_column(0, k / 2, k % 2);
                __builtin_amdgcn_sched_barrier(0);
                weighted(0, xw);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2 * NK; ++k) {
                    update(0, k / 2, k % 2, bt[k / 2][k % 2], xw);
                    bt[k / 2][k % 2] = B_column(1, k / 2, k % 2);
                }
                Parts more[2];
                weighted(1, more);
                mixed(integral_constant<int, 8 * NK>{}, integral_constant<int, 4>{});
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2 * NK; ++k) update(1, k / 2, k % 2, bt[k / 2][k % 2], more);
            }
        } else {
            // The chunk's scores C B^T, which all waves need, are computed once: two tiles each by four waves, one by the others.  Transposed:
            // tile `half` of unit u is 16 tokens 16 tt + i against 4 g + r of 32 kt + ..., u = 0 .. 5 for (tt, kt) = 00 10 20 21 30 31.
            auto tt_of = [](int u) { return u < 2 ? u : u < 4 ? 2 : 3; };
            auto kt_of = [](int u) { return u == 3 || u == 5 ? 1 : 0; };
            auto score_tile = [&](int n) {
                const int u = n >> 1, half = n & 1;
                bf16x8 c[NK], bb[NK];
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    c[ks] = C_row(tt_of(u), ks);
                    bb[ks] = row8(Bl + place(8 * (i >> 2) + 4 * half + (i & 3), 4 * ks + g) + 32 * kt_of(u) * ROW);
                }
                f32x4 G = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) G = product(bb[ks], c[ks], G);
                // an infinity or a NaN in a row of B or C is in all scores of its token
#pragma unroll
                for (int r = 0; r < 4; ++r) probe = fmaf(G[r], 0.f, probe);
                *(f32x4 *)(Gl + n * 1024 + lane * 16) = G;
            };
            score_tile(wave);
            if (wave < 4) score_tile(8 + wave);
            const bool fast = !slow && live;
            // y's transposed tiles: Y[tt][a][r] is row 8 g + 4 a + r of token 16 tt + i
            f32x4 Y[4][2];
            if (fast) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) Y[tt][0] = Y[tt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
                // LDS is read a step ahead of its use; sched_barrier keeps the compiler from moving the reads back in front of it
                bf16x8 c[2][4];
                Parts s[2][2];
                auto parts = [&](int ks, Parts (&to)[2]) {
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = S[ks][e / 4][a][e % 4];
                        to[a] = split(v);
                    }
                };
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) c[0][tt] = C_row(tt, 0);
                parts(0, s[0]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    if (ks + 1 < NK) {
#pragma unroll
                        for (int tt = 0; tt < 4; ++tt) c[(ks + 1) % 2][tt] = C_row(tt, ks + 1);
                        parts(ks + 1, s[(ks + 1) % 2]);
                    }
                    if (ks == NK - 1) weighted(0, xw);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int a = 0; a < 2; ++a)
#pragma unroll
                            for (int tt = 0; tt < 4; ++tt) Y[tt][a] = product(part ? s[ks % 2][a].lo : s[ks % 2][a].hi, c[ks % 2][tt], Y[tt][a]);
                    mixed(integral_constant<int, 16>{}, integral_constant<int, 6>{});
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_waitcnt(kLgkmZero);
            __builtin_amdgcn_s_barrier();                        // all scores are in LDS
            asm volatile("" ::: "memory");
            const int n = min(T, t1 - t);
            const __amdgpu_buffer_rsrc_t rY = yr.descriptor(n);
            const float cs_mid = uniform(rec[CS + 31]), rest_mid = uniform(rest_of(mark_l[31])), rest_end = uniform(rest_of(mark_l[T - 1])), score0 = uniform(rec[SCORE]);
            const bool far = score0 != score0;
            if (fast) {
                f32x4 G[2][2];
                auto fetch = [&](int u) {
                    G[u % 2][0] = *(const f32x4 *)(Gl + 2 * u * 1024 + lane * 16);
                    G[u % 2][1] = *(const f32x4 *)(Gl + (2 * u + 1) * 1024 + lane * 16);
                };
                float cst = 0.f, rest = 0.f;
                int first = 0;
                fetch(0);
                ssd::tile::static_for<6>([&](auto uc) {
                    constexpr int u = decltype(uc)::value, tt = u < 2 ? u : u < 4 ? 2 : 3, kt = u == 3 || u == 5 ? 1 : 0;
                    // this stage's part of the state's update
                    constexpr int from = u * 4 * NK / 6, to = (u + 1) * 4 * NK / 6;
                    bf16x8 bt[to - from];
#pragma unroll
                    for (int k = from; k < to; ++k) bt[k - from] = B_column(k / (2 * NK), k % (2 * NK) / 2, k % 2);
                    if constexpr (u < 5) fetch(u + 1);
                    if constexpr (kt == 0) {
                        // what the entering state gives to 16 tokens
                        cst = rec[CS + 16 * tt + i];
                        const float e = pow2(cst);
                        bool entered = true;
                        // ... and one in a row of the entering state in what that gives
                        if constexpr (u == 0)
#pragma unroll
                            for (int k = 0; k < 8; ++k) probe = fmaf(Y[tt][k / 4][k % 4], 0.f, probe);
                        const uint32_t mark = mark_l[16 * tt + i];
                        rest = rest_of(mark);
                        if constexpr (SEQ) {
                            first = start_of(mark);
                            entered = first < 0;
                        }
#pragma unroll
                        for (int a = 0; a < 2; ++a)
#pragma unroll
                            for (int r = 0; r < 4; ++r) Y[tt][a][r] = entered ? Y[tt][a][r] * e : 0.f;
                    }
                    // scores -> weights of 32 tokens' x
                    float m[8];
                    int seen = 16 * (tt - 2 * kt) + i - 8 * g, hidden = SEQ ? first - 32 * kt - 8 * g : 0;     // of the lane's 8 tokens: up to, from
                    asm volatile("" : "+v"(seen));               // (or the masks of all 16 tokens x 32 are kept in scalar registers)
                    if (!far) {
                        const float reach = pow2((cst - (kt == 0 ? cs_mid : cs_end)) + (rest - (kt == 0 ? rest_mid : rest_end)));
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const f32x4 bj = *(const f32x4 *)&rec[SCORE + 32 * kt + 8 * g + 4 * half];
#pragma unroll
                            for (int r = 0; r < 4; ++r) m[4 * half + r] = G[u % 2][half][r] * (reach * bj[r]);
                        }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const float *const dj = steps - RING * RECORD + STEP + 32 * kt + 8 * g + 4 * half;
                            const f32x4 cj = *(const f32x4 *)&rec[CS + 32 * kt + 8 * g + 4 * half];
                            const u32x4 mj = *(const u32x4 *)&mark_l[32 * kt + 8 * g + 4 * half];
#pragma unroll
                            for (int r = 0; r < 4; ++r) m[4 * half + r] = G[u % 2][half][r] * (pow2((cst - cj[r]) + (rest - rest_of(mj[r]))) * dj[r]);
                        }
                    }
                    if constexpr (SEQ)
#pragma unroll
                        for (int e = 0; e < 8; ++e) m[e] = e >= hidden ? m[e] : 0.f;
                    if constexpr (kt == tt / 2)
#pragma unroll
                        for (int e = 0; e < 8; ++e) m[e] = e <= seen ? m[e] : 0.f;
                    const Parts mp = split(m);
#pragma unroll
                    for (int k = from; k < to; ++k) update(k / (2 * NK), k % (2 * NK) / 2, k % 2, bt[k - from], xw);
                    if constexpr (to == 2 * NK) weighted(1, xw);
#pragma unroll
                    for (int a = 0; a < 2; ++a) Y[tt][a] = product(xo[kt][a], mp.hi, Y[tt][a]);
#pragma unroll
                    for (int a = 0; a < 2; ++a) Y[tt][a] = product(xo[kt][a], mp.lo, Y[tt][a]);
                    // an infinity or a NaN in a row of x is in all of that row in the last tile
                    if constexpr (u == 5)
#pragma unroll
                        for (int k = 0; k < 8; ++k) probe = fmaf(Y[tt][k / 4][k % 4], 0.f, probe);
                    // the tile that the stage before has finished: skip, gate, 16 bytes per lane; the rows of x and z that it took make room
                    auto give = [&](int tt) {
                        const f32x4 D0 = *(const f32x4 *)&D_l[8 * g], D1 = *(const f32x4 *)&D_l[8 * g + 4];
                        const u32x4 xv = *(const u32x4 *)(Xl + xplace(i, g) + 16 * tt * 64);
                        u32x4 zv = {0, 0, 0, 0};
                        if constexpr (GATE) zv = *(const u32x4 *)(Zl + xplace(i, g) + 16 * tt * 64);
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = fmaf(e < 4 ? D0[e % 4] : D1[e % 4], half_of(xv, e), Y[tt][e / 4][e % 4]);
                        if constexpr (GATE)
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] *= silu(half_of(zv, e));
                        u32x4 out;
#pragma unroll
                        for (int e = 0; e < 4; ++e) out[e] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * e], (__bf16)v[2 * e + 1]});
                        // (the whole offset in the lanes' register: 16 bytes stored with a scalar offset are still being read from their
                        // registers when the next instruction writes those, and the compiler waits only in the other form)
                        __builtin_amdgcn_raw_buffer_store_b128(out, rY, (int)((uint32_t)offY + 16u * tt * (uint32_t)yr.pitch), 0, 0);
                    };
                    if constexpr (u == 1) give(0);
                    if constexpr (u == 2) give(1);
                    if constexpr (u == 4) give(2);
                    mixed(integral_constant<int, 4 * (to - from) + 4>{}, integral_constant<int, 8>{});
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (u == 1) request_rows(t + T, 0, 0);
                    if constexpr (u == 2) request_rows(t + T, 1, 0);
                    if constexpr (u == 4) request_rows(t + T, 2, 0);
                    if constexpr (u == 5) {
                        give(3);
                        request_rows(t + T, 3, 0);
                    }
                });
            }
        }
        // with y: everything asked for is for the next chunk; without: the youngest are for the one behind it
        __builtin_amdgcn_s_waitcnt(vm_only(OUT ? 0 : REQUESTS));
        asm volatile("" ::: "memory");
        if constexpr (OUT) {
            xr.next();
            yr.next();
            zr.next();
        }
        slot = slot == RING - 1 ? 0 : slot + 1;
    }
    if (!careful) {
        if constexpr (!OUT)
            all_states([&](f32x4 &v, int, int, bool) {
#pragma unroll
                for (int r = 0; r < 4; ++r) probe = fmaf(v[r], 0.f, probe);
            });
        const bool odd = __any(!(probe == 0.f));
        int *const flags = (int *)(lds + RING * PART + SCORES + WAVES * MINE);
        if (lane == 0) flags[wave] = odd;
        __builtin_amdgcn_s_waitcnt(vm_only(0));        // (nor is anything on its way into LDS)
        __syncthreads();
        if (__any(flags[lane & (WAVES - 1)])) {
            __syncthreads();
            return true;
        }
    }
    if constexpr (OUT) {
        uint16_t *const y = (uint16_t *)p.y + b * p.sy_b + h * p.sy_h + p0;
        for (int t = max(t0, t1); t < t_end; ++t)
            if (lane < 32 && lane < np) y[t * p.sy_l + lane] = 0;
    }
    const bool last = OUT && !LEAVE && seg == p.segments - 1;
    if (last || LEAVE) {
        float *to = last ? p.fin + b * p.sf_b + h * p.sf_h + p0 * p.sf_p : ws;
        const int64_t pitch = last ? p.sf_p : N;
        all_states([&](f32x4 &v, int n, int row, bool there) {
            if (there) *(f32x4 *)&to[row * pitch + n] = v;
        });
    }
    // (what the first segment leaves is a state, whatever entered it)
    if (LEAVE && live && lane == 0 && p0 == 0) p.ws_decay[((int64_t)b * p.nheads + h) * p.segments + seg] = !OUT && passes ? not_zero(pow2(through)) : -1.f;
    if (!OUT) __builtin_amdgcn_s_waitcnt(vm_only(0));             // no request may be under way when the workgroup's LDS is given away
    return false;
}

// One copy of the code: the second walk is rare.  The parameters come from an address, and the lane from a register, that the compiler does
// not know: what both walks have in common would otherwise be kept in registers over the first one.
typedef const __attribute__((address_space(4))) SelScanParams *Arguments;
template <int NK, bool OUT, bool GATE, bool SEQ, bool LEAVE>
__device__ __forceinline__ void walk(Arguments from, int blocks_per_head, const Place &place_of)
{
#pragma clang loop unroll(disable)
    for (int careful = 0; careful < 2; ++careful) {
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("" : "+s"(from));
#endif
        if (!walk_once<NK, OUT, GATE, SEQ, LEAVE>(*(const SelScanParams *)from, blocks_per_head, place_of, careful != 0)) break;
    }
}
// the arguments of a kernel whose `n`th is this, of those that begin with such
__device__ __forceinline__ Arguments arguments(int n)
{
#if defined(__HIP_DEVICE_COMPILE__)
    return (Arguments)__builtin_amdgcn_kernarg_segment_ptr() + n;
#else
    return nullptr;
#endif
}

// The segments from `first` on, with y: what enters them is known
template <int NK, bool GATE, bool SEQ>
__global__ void __launch_bounds__(64 * WAVES, 2) chunk_kernel(const SelScanParams p, int blocks_per_head, int sets, int first)
{
    walk<NK, true, GATE, SEQ, false>(arguments(0), blocks_per_head, place_of_workgroup(p, sets, first, p.segments - first));
}
// In front of that: what each segment but the last adds to a state of zero
template <int NK, bool SEQ>
__global__ void __launch_bounds__(64 * WAVES, 2) add_kernel(const SelScanParams p, int blocks_per_head, int sets)
{
    walk<NK, false, false, SEQ, true>(arguments(0), blocks_per_head, place_of_workgroup(p, sets, 0, p.segments - 1));
}
// or, beside it, the first segment with y.  (The two ways have their parameters each: what both would load from the same place is loaded
// in front of the branch, more than there are scalar registers for.)
template <int NK, bool GATE, bool SEQ>
__global__ void __launch_bounds__(64 * WAVES, 2) front_kernel(const SelScanParams p, const SelScanParams q, int blocks_per_head, int sets)
{
    const Place at = place_of_workgroup(p, sets, 0, p.segments - 1);
    if (at.segment == 0) walk<NK, true, GATE, SEQ, true>(arguments(0), blocks_per_head, at);
    else walk<NK, false, false, SEQ, true>(arguments(1), blocks_per_head, at);
}

template <int NK, bool GATE, bool SEQ>
hipError_t run(SelScanParams p, hipStream_t s)
{
    const int blocks_per_head = (p.headdim + 31) / 32;
    const int64_t units = (int64_t)(p.nheads / p.ngroups) * blocks_per_head, sets = (units + WAVES - 1) / WAVES;
    const int64_t blocks = sets * p.ngroups * p.batch;      // of a segment
    const int S = p.segments, first = p.head ? 1 : 0;
    if (blocks * S * 64 * WAVES > 0xffffffffLL || units > 0x7fffffffLL) return hipErrorInvalidConfiguration;
    constexpr int tile = T * 64 * NK, x = T * 64, add = 3 * tile + WAVES * (3 * x + 3 * 2 * T * 4 + 4),
                  out = 2 * 2 * tile + 12 * 1024 + WAVES * (2 * x + 128 + 2 * STEP * 4 + 4);
    constexpr int front = add > out ? add : out;
    static std::atomic<uint64_t> done[3];
    hipError_t e = ensure_dynamic_lds((const void *)chunk_kernel<NK, GATE, SEQ>, out, done[0]);
    if (e == hipSuccess) e = ensure_dynamic_lds((const void *)front_kernel<NK, GATE, SEQ>, front, done[1]);
    if (e == hipSuccess) e = ensure_dynamic_lds((const void *)add_kernel<NK, SEQ>, add, done[2]);
    if (e != hipSuccess) return e;
    const int head_tiles = (p.nheads + kHeadTile - 1) / kHeadTile;
    const int64_t records = (int64_t)head_tiles * p.chunks * p.batch;
    if (records * 256 > 0xffffffffLL) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((steps_kernel<SEQ>), dim3((uint32_t)records), dim3(256), 0, s, p, head_tiles);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    p.joined = 0;
    if (S > 1) {
        const dim3 grid((uint32_t)(blocks * (S - 1)));
        if (p.head) hipLaunchKernelGGL((front_kernel<NK, GATE, SEQ>), grid, dim3(64 * WAVES), front, s, p, p, blocks_per_head, (int)sets);
        else hipLaunchKernelGGL((add_kernel<NK, SEQ>), grid, dim3(64 * WAVES), add, s, p, blocks_per_head, (int)sets);
        e = hipGetLastError();
        // few segments: who enters one reads what those in front of it left, in less time than a launch in between takes
        p.joined = S - first > 3;
        if (e == hipSuccess && p.joined) e = launch_scan_join(p, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((chunk_kernel<NK, GATE, SEQ>), dim3((uint32_t)(blocks * (S - first))), dim3(64 * WAVES), out, s, p, blocks_per_head, (int)sets, first);
    return hipGetLastError();
}

template <int NK>
hipError_t of_case(const SelScanParams &p, hipStream_t s)
{
    if (p.seq) return p.z ? run<NK, true, true>(p, s) : run<NK, false, true>(p, s);
    return p.z ? run<NK, true, false>(p, s) : run<NK, false, false>(p, s);
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
    return p.dstate <= 64 ? of_case<2>(p, s) : of_case<4>(p, s);
}

}  // namespace ssd
