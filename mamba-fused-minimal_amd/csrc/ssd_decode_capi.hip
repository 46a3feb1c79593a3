// extern "C" entry points of the operators of a decoding step: argument checks, launch.
#include "../../include/ssd_gfx950.h"
#include "ssd_decode.h"

#include <string.h>

namespace ssd {
int device_status();        // SSD_OK on a gfx950 device (ssd_capi.hip)
int device_compute_units();
}

namespace {

using namespace ssd;

bool present(const ssd_tensor *t) { return t && t->data; }
bool real(const ssd_tensor *t) { return t->dtype == SSD_F32 || t->dtype == SSD_BF16 || t->dtype == SSD_F16; }
bool real_or_absent(const ssd_tensor *t) { return !present(t) || real(t); }
// A dimension of size one may carry any stride.
int64_t stride(const ssd_tensor *t, int i, int64_t size) { return size == 1 ? 0 : t->stride[i]; }
bool unit(const ssd_tensor *t, int i, int64_t size) { return size == 1 || t->stride[i] == 1; }
constexpr int32_t kLongest = 1 << 30;      // of a row, and rows: the ends of tiles behind the last one fit 32 bits
int launched(hipError_t e) { return e == hipSuccess ? SSD_OK : e == hipErrorInvalidConfiguration ? SSD_ERR_SHAPE : (int)e; }

int beam_parts(int32_t vocab) { return (int)(((int64_t)vocab + kBeamPart - 1) / kBeamPart); }
bool beam_sizes(int32_t batch, int32_t beams, int32_t vocab, int32_t k)
{
    if (batch < 0 || beams <= 0 || vocab <= 0 || k <= 0 || beams > kBeamMost || k > kBeamMost) return false;
    const int64_t candidates = (int64_t)beams * vocab;
    return vocab <= kLongest && candidates <= INT32_MAX && k <= candidates && (int64_t)batch * beams <= INT32_MAX;
}
uint64_t beam_rows(int32_t batch, int32_t beams, int32_t vocab) { return (uint64_t)batch * beams * beam_parts(vocab); }

constexpr int64_t kSlotMost = (int64_t)1 << 36;      // bytes of a slot: workgroups of a launch fit its grid
// The dimensions of a slot that say where its elements are: those of size one left out, the largest stride first, one behind another joined.
// false: more than four are left, or elements share a place.
bool slot_of(const ssd_pool &pool, StridedPool &to)
{
    if (pool.dims < 0 || pool.dims > 4 || pool.element_bytes <= 0) return false;
    int64_t size[4], step[4];
    int n = 0;
    to.count = 1;
    for (int i = 0; i < pool.dims; ++i) {
        if (pool.size[i] < 0 || __builtin_mul_overflow(to.count, pool.size[i], &to.count)) return false;
        if (pool.size[i] == 1) continue;
        if (pool.stride[i] <= 0 && pool.size[i] > 1) return false;
        int at = n++;
        for (; at > 0 && step[at - 1] < pool.stride[i]; --at) {
            size[at] = size[at - 1];
            step[at] = step[at - 1];
        }
        size[at] = pool.size[i];
        step[at] = pool.stride[i];
    }
    int m = 0;
    for (int i = 0; i < n; ++i) {
        if (m > 0 && to.stride[m - 1] == size[i] * step[i]) {
            to.size[m - 1] *= size[i];
            to.stride[m - 1] = step[i];
        } else {
            to.size[m] = size[i];
            to.stride[m++] = step[i];
        }
    }
    for (; m < 4; ++m) {
        to.size[m] = 1;
        to.stride[m] = 0;
    }
    to.data = (char *)pool.data;
    to.element = pool.element_bytes;
    to.slot_stride = pool.slot_stride;
    return true;
}
// Whether no two elements of any slots share a place, the slots being one more dimension: each stride is beyond what the smaller ones reach.
bool apart(const StridedPool &p, int32_t slots)
{
    int64_t reach = 0;                            // from the first to the last place of the dimensions so far, the smallest strides first
    bool seen = slots <= 1;
    for (int i = 3; i >= -1; --i) {
        if (!seen && (i < 0 || p.size[i] > 1) && (i < 0 || p.slot_stride < p.stride[i])) {
            if (p.slot_stride <= reach || __builtin_add_overflow(reach, (slots - 1) * (__int128)p.slot_stride, &reach)) return false;
            seen = true;
        }
        if (i < 0 || p.size[i] <= 1) continue;
        if (p.stride[i] <= reach || __builtin_add_overflow(reach, (p.size[i] - 1) * (__int128)p.stride[i], &reach)) return false;
    }
    return true;
}
// ... whether that is one run
bool is_run(const StridedPool &p) { return p.size[1] == 1 && (p.size[0] == 1 || p.stride[0] == 1); }

}  // namespace

extern "C" {

uint64_t ssd_matmul_packed_workspace_bytes(int32_t M, int32_t N, int32_t K, int32_t group, int type)
{
    if (M <= 0 || N <= 0 || K <= 0 || M > kLongest || N > kLongest || K > SSD_MATMUL_PACKED_MAX_K || group <= 0) return 0;
    return matmul_packed_room(M, N, K, group, type, device_compute_units());
}

int ssd_matmul_packed_fwd(const ssd_tensor *a, const ssd_tensor *w, const ssd_tensor *w_scale, const ssd_tensor *w_zero, const ssd_tensor *bias,
                          const ssd_tensor *out, int32_t M, int32_t N, int32_t K, int32_t group, void *workspace, uint64_t workspace_bytes,
                          void *stream)
{
    if (M < 0 || N < 0 || K < 0 || M > kLongest || N > kLongest || K > SSD_MATMUL_PACKED_MAX_K || group <= 0 || (group % 32 != 0 && group < K)) return SSD_ERR_SHAPE;
    if (M == 0 || N == 0) return SSD_OK;
    if (!present(out) || (K > 0 && (!present(a) || !present(w) || !present(w_scale)))) return SSD_ERR_NULL;
    if (!real(out) || !real_or_absent(bias) || (K > 0 && (!real(a) || w->dtype != SSD_U8 || !real(w_scale))) ||
        (K > 0 && present(w_zero) && w_zero->dtype != SSD_U8))
        return SSD_ERR_DTYPE;
    const int64_t bytes = ((int64_t)K + 1) / 2;
    if ((K > 0 && (!unit(a, 1, K) || !unit(w, 1, bytes))) || !unit(out, 1, N)) return SSD_ERR_STRIDE;
    PackedParams p;
    memset(&p, 0, sizeof(p));
    p.group = group < K ? group : K > 0 ? (K + 31) / 32 * 32 : 32;
    p.groups = K > 0 ? (K - 1) / p.group + 1 : 0;
    if (K > 0) {
        p.a = a->data; p.sa_m = stride(a, 0, M); p.type = a->dtype;
        p.w = (const uint8_t *)w->data; p.sw_n = stride(w, 0, N);
        p.scale = w_scale->data; p.scale_type = w_scale->dtype; p.ss_n = stride(w_scale, 0, N); p.ss_g = stride(w_scale, 1, p.groups);
        if (present(w_zero)) { p.zero = (const uint8_t *)w_zero->data; p.sz_n = stride(w_zero, 0, N); p.sz_g = stride(w_zero, 1, p.groups); }
    } else p.type = out->dtype;
    if (present(bias)) { p.bias = bias->data; p.bias_type = bias->dtype; p.sbias = stride(bias, 0, N); }
    p.out = out->data; p.out_type = out->dtype; p.so_m = stride(out, 0, M);
    p.M = M; p.N = N; p.K = K;
    if (workspace && !((uintptr_t)workspace & 15)) { p.room = workspace; p.room_bytes = workspace_bytes; }
    const int rc = device_status();
    return rc ? rc : launched(launch_matmul_packed(p, device_compute_units(), (hipStream_t)stream));
}

int ssd_norm_block_fwd(const ssd_tensor *x, const ssd_tensor *weight, const ssd_tensor *residual, const ssd_tensor *next_weight,
                       const ssd_tensor *gate, const ssd_tensor *out, const ssd_tensor *scale, const ssd_tensor *residual_out, int64_t rows,
                       int32_t dim, int64_t gate_every, float residual_scale, float eps, void *stream)
{
    if (rows < 0 || dim <= 0 || dim > kLongest || (present(gate) && gate_every <= 0)) return SSD_ERR_SHAPE;
    if (rows == 0) return SSD_OK;
    if (!present(x) || !present(residual) || !present(next_weight) || !present(out) || !present(residual_out)) return SSD_ERR_NULL;
    const bool int8 = out->dtype == SSD_I8;
    if (int8 && !present(scale)) return SSD_ERR_NULL;
    const auto narrow = [&](const ssd_tensor *t) { return !present(t) || t->dtype == x->dtype || t->dtype == SSD_F32; };
    if (!real(x) || residual->dtype != x->dtype || residual_out->dtype != x->dtype || (!int8 && out->dtype != x->dtype) ||
        (int8 && scale->dtype != SSD_F32) || !narrow(weight) || !narrow(next_weight) || !narrow(gate))
        return SSD_ERR_DTYPE;
    if (!unit(x, 1, dim) || !unit(residual, 1, dim) || !unit(out, 1, dim) || !unit(residual_out, 1, dim) || (present(weight) && !unit(weight, 0, dim)) ||
        !unit(next_weight, 0, dim) || (present(gate) && !unit(gate, 1, dim)))
        return SSD_ERR_STRIDE;
    NormBlockParams p;
    memset(&p, 0, sizeof(p));
    p.x = x->data; p.sx = stride(x, 0, rows); p.type = x->dtype;
    p.residual = residual->data; p.sr = stride(residual, 0, rows);
    if (present(weight)) { p.w = weight->data; p.w_wide = weight->dtype != x->dtype; }
    p.next_w = next_weight->data; p.next_wide = next_weight->dtype != x->dtype;
    p.gate_every = 1;
    if (present(gate)) {
        p.gate = gate->data; p.gate_wide = gate->dtype != x->dtype;
        p.gate_every = gate_every; p.sg = gate_every >= rows ? 0 : gate->stride[0];
    }
    p.out = out->data; p.so = stride(out, 0, rows); p.int8 = int8;
    if (int8) { p.scale = (float *)scale->data; p.sscale = stride(scale, 0, rows); }
    p.residual_out = residual_out->data; p.sro = stride(residual_out, 0, rows);
    p.rows = rows; p.dim = dim; p.factor = residual_scale; p.eps = eps;
    // (two results of 64 MB: what reads them finds little of them in the caches anyway)
    p.past = rows * (int64_t)dim * (x->dtype == SSD_F32 ? 4 : 2) >= (int64_t)64 << 20;
    const int rc = device_status();
    return rc ? rc : launched(launch_norm_block(p, (hipStream_t)stream));
}

uint64_t ssd_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t k)
{
    return beam_sizes(batch, beams, vocab, k) ? beam_rows(batch, beams, vocab) * (16 + 8 * (uint64_t)k) : 0;
}

int ssd_beam_select_fwd(const ssd_tensor *logits, const ssd_tensor *scores, const ssd_tensor *finished, const ssd_tensor *out_scores,
                        const ssd_tensor *parents, const ssd_tensor *tokens, int32_t batch, int32_t beams, int32_t vocab, int32_t k, int32_t pad,
                        void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (!beam_sizes(batch, beams, vocab, k) || (present(finished) && (pad < 0 || pad >= vocab))) return SSD_ERR_SHAPE;
    if (batch == 0) return SSD_OK;
    if (!present(logits) || !present(scores) || !present(out_scores) || !present(parents) || !present(tokens)) return SSD_ERR_NULL;
    if (!real(logits) || scores->dtype != SSD_F32 || out_scores->dtype != SSD_F32 || parents->dtype != 0 || tokens->dtype != 0 ||
        (present(finished) && finished->dtype != SSD_U8))
        return SSD_ERR_DTYPE;
    if (!unit(logits, 2, vocab) || !unit(out_scores, 1, k) || !unit(parents, 1, k) || !unit(tokens, 1, k)) return SSD_ERR_STRIDE;
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < ssd_beam_workspace_bytes(batch, beams, vocab, k)) return SSD_ERR_SCRATCH;
    BeamParams p;
    memset(&p, 0, sizeof(p));
    p.logits = logits->data; p.type = logits->dtype; p.sl_b = stride(logits, 0, batch); p.sl_i = stride(logits, 1, beams);
    p.scores = (const float *)scores->data; p.ss_b = stride(scores, 0, batch); p.ss_i = stride(scores, 1, beams);
    if (present(finished)) { p.finished = (const uint8_t *)finished->data; p.sf_b = stride(finished, 0, batch); p.sf_i = stride(finished, 1, beams); }
    p.out_scores = (float *)out_scores->data; p.so_b = stride(out_scores, 0, batch);
    p.parents = (int32_t *)parents->data; p.sp_b = stride(parents, 0, batch);
    p.tokens = (int32_t *)tokens->data; p.st_b = stride(tokens, 0, batch);
    p.batch = batch; p.beams = beams; p.vocab = vocab; p.k = k; p.pad = pad; p.parts = beam_parts(vocab);
    p.ws_sums = (double *)workspace;
    p.ws_best = (uint64_t *)workspace + 2 * beam_rows(batch, beams, vocab);
    const int rc = device_status();
    return rc ? rc : launched(launch_beam_select(p, (hipStream_t)stream));
}

int ssd_beam_reorder(const ssd_tensor *parents, const ssd_tensor *slots, const ssd_tensor *new_slots, const ssd_pool *pools, int32_t num_pools,
                     int32_t num_slots, int32_t batch, int32_t beams, void *stream)
{
    if (batch < 0 || beams <= 0 || beams > kBeamMost || num_pools < 0 || num_slots < 0) return SSD_ERR_SHAPE;
    if (batch == 0) return SSD_OK;
    if (!present(parents) || !present(slots) || !present(new_slots) || (num_pools > 0 && !pools)) return SSD_ERR_NULL;
    if (parents->dtype != 0 || slots->dtype != 0 || new_slots->dtype != 0) return SSD_ERR_DTYPE;
    for (int i = 0; i < num_pools; ++i) {
        StridedPool slot;
        const int e = pools[i].element_bytes;
        if (e != 1 && e != 2 && e != 4 && e != 8 && e != 16) return SSD_ERR_DTYPE;
        if (!slot_of(pools[i], slot)) return SSD_ERR_STRIDE;
        if (slot.count > 0 && !apart(slot, num_slots)) return SSD_ERR_STRIDE;
        if (num_slots > 0 && slot.count > 0 && !pools[i].data) return SSD_ERR_NULL;
        if (slot.count > kSlotMost / e) return SSD_ERR_SHAPE;
    }
    const int rc = device_status();
    if (rc) return rc;
    ReorderParams p;
    memset(&p, 0, sizeof(p));
    p.parents = (const int32_t *)parents->data; p.sp_b = stride(parents, 0, batch); p.sp_i = stride(parents, 1, beams);
    p.slots = (const int32_t *)slots->data; p.ss_b = stride(slots, 0, batch); p.ss_i = stride(slots, 1, beams);
    p.new_slots = (int32_t *)new_slots->data; p.sn_b = stride(new_slots, 0, batch); p.sn_i = stride(new_slots, 1, beams);
    p.batch = batch; p.beams = beams; p.n_slots = num_slots;
    int pieces = 0;
    int64_t bytes = 0;                                                  // of a slot, in all pools
    for (int i = 0; i < num_pools; ++i) {
        StridedPool slot;
        slot_of(pools[i], slot);
        bytes += slot.count * slot.element;
    }
    p.past = bytes > (64ll << 20) / batch;
    auto flush = [&](bool last) {
        if (p.n_pools == 0 && !(last && p.new_slots)) return hipSuccess;
        const hipError_t e = launch_reorder(p, pieces, (hipStream_t)stream);
        p.new_slots = nullptr;
        p.n_pools = pieces = 0;
        return e;
    };
    for (int i = 0; i < num_pools; ++i) {
        StridedPool slot;
        slot_of(pools[i], slot);
        if (slot.count == 0 || num_slots == 0) continue;
        if (!is_run(slot)) {
            const hipError_t e = launch_reorder_strided(p, slot, (hipStream_t)stream);
            if (e != hipSuccess) return launched(e);
            continue;
        }
        PoolParams &to = p.pools[p.n_pools];
        to.data = slot.data;
        to.bytes = slot.count * slot.element;
        to.slot_stride = slot.slot_stride * slot.element;
        to.first = pieces;
        pieces += reorder_pieces(to.bytes);
        if (++p.n_pools == kPoolsPerLaunch || pieces > 1 << 22) {
            const hipError_t e = flush(false);
            if (e != hipSuccess) return launched(e);
        }
    }
    return launched(flush(true));
}

}  // extern "C"
