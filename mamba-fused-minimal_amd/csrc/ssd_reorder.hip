// States follow their beams after a selection: child j of row b goes on from beam parents[b, j].
//
//   the first child of a beam takes its slot; every other one takes the slot of a beam without a child, in order, and
//   pool[its slot] = pool[its parent's slot]
//
// A slot that is read is some child's own and is never written; a slot that is written belonged to a beam without a child and is never
// read: the copies are in place, in any order, and only what goes on twice is moved.
//
// HBM bound: a copied slot is read once and written once.  Every workgroup works the assignment out for itself from the row's beams
// (scalar work on at most 64 of them, behind two loads) and then copies its piece of the slot for all copies of the row.
// Measured: 16 rows of 4 beams, a copy in each, 10.6 MB a slot, in 58 us (5.9 TB/s); one row of 3, 19 MB in 48 pools, in 8.5 us (4.5 TB/s).
// Pieces of 8 KB: 57.9 and 8.5 us, 16 KB: 60.8 and 10.2 us, 64 KB: 66.6 and 11.9 us, 4 KB: 78.8 and 11.8 us.  Where a slot of every row is 64 MB
// or more the copies go past the caches (57.9 us, 66.2 through them); fewer bytes go through them (8.5 us, 10.4 past them).
#include "ssd_decode.h"

namespace ssd {
namespace {

using namespace layer;

constexpr int kPiece = 8192;      // bytes of a slot per workgroup

// One row's beams, a lane each (the same in every wave)
struct Row {
    uint64_t there, own;           // beams with a slot, with one of their own
    int parent, slot;              // this lane's
    bool known;                    // its parent has a slot
    __device__ __forceinline__ Row(const ReorderParams &p, int b)
    {
        const int lane = threadIdx.x & 63;
        parent = -1;
        slot = -1;
        if (lane < p.beams) {
            parent = p.parents[b * p.sp_b + lane * p.sp_i];
            slot = p.slots[b * p.ss_b + lane * p.ss_i];
        }
        there = __ballot(slot >= 0 && slot < p.n_slots);
        known = parent >= 0 && parent < p.beams && ((there >> (parent & 63)) & 1);
        // beams that share a slot are one, the first of them
        int first = lane;
        for (int j = p.beams - 1; j >= 0; --j) first = slot == __builtin_amdgcn_readlane(slot, j) ? j : first;
        own = __ballot(first == lane);
        const int of = __shfl(first, parent & 63);      // (by all lanes: the ones that are asked have to take part)
        if (known) parent = of;
    }
    // f(child, slot it goes on from, slot it is given or -1, whether to copy) for every child, in order
    template <class F> __device__ __forceinline__ void children(const ReorderParams &p, F &&f) const
    {
        const uint64_t alive = __ballot(known);
        uint64_t parents = 0;
        for (int j = 0; j < p.beams; ++j)
            if ((alive >> j) & 1) parents |= 1ull << (__builtin_amdgcn_readlane(parent, j) & 63);
        uint64_t spare = there & own & ~parents, taken = 0;
        for (int j = 0; j < p.beams; ++j) {
            if (!((alive >> j) & 1)) {
                f(j, -1, -1, false);
                continue;
            }
            const int of = __builtin_amdgcn_readlane(parent, j) & 63, from = __builtin_amdgcn_readlane(slot, of);
            if (!((taken >> of) & 1)) {
                taken |= 1ull << of;
                f(j, from, from, false);
            } else if (spare) {
                const int to = __builtin_amdgcn_readlane(slot, __builtin_ctzll(spare));
                spare &= spare - 1;
                f(j, from, to, true);
            } else f(j, from, -1, false);
        }
    }
};

__device__ __forceinline__ void write_slots(const ReorderParams &p, const Row &row, int b)
{
    int mine = -1;
    row.children(p, [&](int j, int, int to, bool) { mine = (int)(threadIdx.x & 63) == j ? to : mine; });
    if ((int)threadIdx.x < p.beams) p.new_slots[b * p.sn_b + threadIdx.x * p.sn_i] = mine;
}

typedef __attribute__((ext_vector_type(4), aligned(1))) uint32_t piece16;      // (slots begin at any byte)

// PAST: past the caches
template <bool PAST> __device__ __forceinline__ void copy_run(const char *src, char *dst, int pieces)
{
    constexpr int U = kPiece / 4096;
    int i = threadIdx.x;
    for (; i + (U - 1) * 256 < pieces; i += U * 256) {
        piece16 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const piece16 *const at = (const piece16 *)src + i + u * 256;
            v[u] = PAST ? __builtin_nontemporal_load(at) : *at;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            piece16 *const at = (piece16 *)dst + i + u * 256;
            if (PAST) __builtin_nontemporal_store(v[u], at);
            else *at = v[u];
        }
    }
    for (; i < pieces; i += 256) ((piece16 *)dst)[i] = ((const piece16 *)src)[i];
}

__global__ void __launch_bounds__(256) reorder_kernel(const ReorderParams p)
{
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= p.batch) return;
    const Row row(p, b);
    if (p.new_slots && blockIdx.x == 0 && threadIdx.x < 64) write_slots(p, row, b);
    if (p.n_pools == 0) return;
    const int lane = threadIdx.x & 63;
    const int which = __builtin_popcountll(__ballot(lane < p.n_pools && (int)blockIdx.x >= p.pools[lane < p.n_pools ? lane : 0].first)) - 1;
    const PoolParams &pool = p.pools[which];
    const int64_t begin = (int64_t)((int)blockIdx.x - pool.first) * kPiece;
    const int64_t left = pool.bytes - begin;
    const int n = (int)(left < kPiece ? left : kPiece);
    row.children(p, [&](int, int from, int to, bool copy) {
        if (!copy) return;
        const char *src = pool.data + from * pool.slot_stride + begin;
        char *dst = pool.data + to * pool.slot_stride + begin;
        const int pieces = n / 16;
        if (p.past) copy_run<true>(src, dst, pieces);
        else copy_run<false>(src, dst, pieces);
        for (int t = pieces * 16 + threadIdx.x; t < n; t += 256) dst[t] = src[t];
    });
}

template <class E>
__global__ void __launch_bounds__(256) strided_kernel(const ReorderParams p, const StridedPool pool)
{
    const int b = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (b >= p.batch) return;
    const Row row(p, b);
    row.children(p, [&](int, int from, int to, bool copy) {
        if (!copy) return;
        E *const base = (E *)pool.data;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pool.count; i += (int64_t)gridDim.x * 256) {
            int64_t rest = i, at = 0;
#pragma unroll
            for (int d = 3; d >= 0; --d) {
                at += rest % pool.size[d] * pool.stride[d];
                rest /= pool.size[d];
            }
            base[to * pool.slot_stride + at] = base[from * pool.slot_stride + at];
        }
    });
}

struct Sixteen { uint32_t w[4]; };

dim3 grid_of(uint32_t pieces, int batch)
{
    const uint32_t y = batch < 32768 ? (uint32_t)batch : 32768;
    return dim3(pieces, y, ((uint32_t)batch + y - 1) / y);
}

}  // namespace

int reorder_pieces(int64_t bytes) { return (int)((bytes + kPiece - 1) / kPiece); }

hipError_t launch_reorder(const ReorderParams &p, int pieces, hipStream_t s)
{
    if (p.batch == 0 || p.beams == 0) return hipSuccess;
    hipLaunchKernelGGL(reorder_kernel, grid_of(pieces > 0 ? (uint32_t)pieces : 1, p.batch), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_reorder_strided(const ReorderParams &p, const StridedPool &pool, hipStream_t s)
{
    if (p.batch == 0 || p.beams == 0 || pool.count == 0) return hipSuccess;
    const int64_t blocks = (pool.count + 255) / 256;
    const dim3 grid = grid_of((uint32_t)(blocks < 4096 ? blocks : 4096), p.batch);
    switch (pool.element) {
        case 1: hipLaunchKernelGGL(strided_kernel<uint8_t>, grid, dim3(256), 0, s, p, pool); break;
        case 2: hipLaunchKernelGGL(strided_kernel<uint16_t>, grid, dim3(256), 0, s, p, pool); break;
        case 4: hipLaunchKernelGGL(strided_kernel<uint32_t>, grid, dim3(256), 0, s, p, pool); break;
        case 8: hipLaunchKernelGGL(strided_kernel<uint64_t>, grid, dim3(256), 0, s, p, pool); break;
        default: hipLaunchKernelGGL(strided_kernel<Sixteen>, grid, dim3(256), 0, s, p, pool); break;
    }
    return hipGetLastError();
}

}  // namespace ssd
