// extern "C" entry points of the operators around the state path: argument checks, choice of kernel, launch.
#include "../../include/ssd_gfx950.h"
#include "ssd_layer.h"

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
bool ints_or_absent(const ssd_tensor *t) { return !present(t) || t->dtype == 0; }

// A dimension of size one may carry any stride.
int64_t stride(const ssd_tensor *t, int i, int64_t size) { return size == 1 ? 0 : t->stride[i]; }
// ... and an innermost one of size one counts as contiguous
bool unit(const ssd_tensor *t, int i, int64_t size) { return size == 1 || t->stride[i] == 1; }

int launched(hipError_t e) { return e == hipSuccess ? SSD_OK : e == hipErrorInvalidConfiguration ? SSD_ERR_SHAPE : (int)e; }

void fill_delta(DeltaParams &d, const ssd_tensor *bias, int softplus, float lo, float hi)
{
    memset(&d, 0, sizeof(d));
    if (present(bias)) {
        d.bias = bias->data;
        d.bias_type = bias->dtype;
        d.sbias = bias->stride[0];
    }
    d.softplus = softplus;
    d.lo = lo;
    d.hi = hi;
}

// What a scan's kernel on the matrix instructions takes by sizes and type; pointers and strides may still send it the other way.
bool scan_tiles(const ssd_dims *d, int type) { return type == SSD_BF16 && d->dstate <= 128 && d->dstate % 8 == 0 && d->headdim % 8 == 0; }

// The kernel of a scan call and the segments that it cuts its rows into: what the estimates below, in microseconds, find cheapest.
//
// On the matrix instructions of bf16 a compute unit has one workgroup (8 waves of 32 headdim rows) at a time: whole rounds of as many
// workgroups as there are units, each as long as a segment.  9 for the steps' kernel and its launch; a workgroup takes 8 to begin and 8
// per chunk of 64 tokens; with more than one segment a pass over x and B goes in front, 5 and 3 per chunk, and the segments' states are
// written and read at 4 TB/s, twice with a launch of 6 that joins them (more than three; fewer are joined by who enters them).  Beside
// that pass there is room for the first segment itself, y and all: 25 more for its way through the other half of a larger kernel.
// 24 heads of 64 x 128: 64 tokens 25, 128 tokens 32, 200 tokens in four segments 40 (joined by who enters them 46).
//
// The kernel for any size: 6 to begin; a chunk of 32 tokens takes a workgroup 5.6 alone on its compute unit, two of them 8 together (with
// 128 state columns; with fewer, less), the pass in front, over all segments but the last, 3.5 and 5.3, and four of its workgroups 6; 5 to
// begin with more than one segment, 12 with more than four (joined in a launch), and 4 for every round of workgroups behind the first.
// With more than 128 state columns a unit has room for one.  Measured (fp16, 64 x 128): 64 heads, 3001 tokens: 499 in one segment, 215
// in four, 168 in sixteen; 256 heads, 3001 tokens: 517 in one, 592 in two; 320 heads, 8192 tokens: 2127 in one, 1776 in four, 1832 in
// eight; 576 heads, 3000 tokens: 1230 in one, 1182 in four.  Few tokens of few heads in bf16 are its too: 24 heads, one token 12 (23 on
// the other), 200 tokens 28 in four segments of two chunks (40).
// chunks of the first segment and of each other one; whether the first is done in front of the others, y and all
struct ScanPlan { bool tiles; int segments, first, others; bool head; };
// That of the kernel for any size, and its cost.
ScanPlan any_plan(const ssd_dims *d, int n_cu, double &best)
{
    if (n_cu <= 0) n_cu = 256;
    ScanPlan plan = {false, 1, 0, 0, false};
    double least = 0;
    const int64_t walks = (int64_t)d->batch * d->nheads * ((d->headdim + 63) / 64);
    const int64_t plane = (int64_t)d->batch * d->nheads * d->headdim * d->dstate;
    const int64_t chunks = ((int64_t)d->seqlen + 31) / 32;
    const bool one = d->dstate > 128;      // workgroup to a unit
    const double size = one ? 1 : (d->dstate + 64) / 192.0;
    for (int64_t n = 1; n == 1 || (n <= ((int64_t)d->seqlen + 63) / 64 && d->seqlen >= 128 && (n - 1) * walks < 4LL * n_cu); n += 1 + n / 16) {
        const double length = (double)((chunks + n - 1) / n);
        const int64_t all = walks * n, front = all - walks, rest = all % (2 * n_cu);
        const double tail = rest == 0 ? 0 : rest <= n_cu ? 5.6 : 8.0;
        const double out = size * (one ? 5.6 * ((all + n_cu - 1) / n_cu) : 8.0 * (all / (2 * n_cu)) + tail);
        const double four = 6.0 * front / (4 * n_cu), add = size * (one ? 3.5 * ((front + n_cu - 1) / n_cu) : front <= n_cu ? 3.5 : four < 5.3 ? 5.3 : four);
        const double moved = (n > 4 ? 4.0 : 2.0) * n * plane * 4 / 4e6;
        const double begin = n == 1 ? 6 : 6 + 4.0 * ((all - 1) / ((one ? 1 : 2) * n_cu)) + (n > 4 ? 12 : 5);
        const double cost = begin + length * out + (n == 1 ? 0 : length * add + moved);
        if (n == 1 || cost < least) {
            least = cost;
            // (Beside the other kernel a call in one segment counts whole rounds of two workgroups to a unit: with less for a last round of
            // one each, 640 or 960 of them over 64 to 384 tokens came here, 5 to 15 % slower.)
            const double whole = one || all <= n_cu ? out : size * 8.0 * ((all + 2 * n_cu - 1) / (2 * n_cu));
            best = n == 1 ? begin + length * whole : cost;
            plan = {false, (int)n, (int)length, (int)length, false};
        }
    }
    return plan;
}

ScanPlan scan_plan(const ssd_dims *d, int type, int n_cu)
{
    if (n_cu <= 0) n_cu = 256;
    double best;
    ScanPlan plan = any_plan(d, n_cu, best);
    if (!scan_tiles(d, type)) return plan;
    const int64_t plane = (int64_t)d->batch * d->nheads * d->headdim * d->dstate;
    const int64_t blocks = (d->headdim + 31) / 32, workgroups = (int64_t)d->batch * d->ngroups * ((d->nheads / d->ngroups * blocks + 7) / 8);
    const int64_t chunks = ((int64_t)d->seqlen + 63) / 64;
    for (int64_t n = 1; n == 1 || (n <= 2 * n_cu && n <= chunks); n += 1 + n / 16) {
        const double rounds = (double)((workgroups * n + n_cu - 1) / n_cu), moved = (n > 3 ? 4.0 : 2.0) * n * plane * 4 / 4e6 + (n > 3 ? 6 : 0);
        const int64_t length = (chunks + n - 1) / n;
        const double cost = 9 + rounds * (8 + 8 * (double)length) + (n == 1 ? 0 : 5 + rounds * 3 * length + moved);
        if (cost < best) {
            best = cost;
            plan = {true, (int)n, (int)length, (int)length, false};
        }
        // The same number of workgroups with one segment more, the first, of a quarter of the others' length: about as long as what they add
        // takes (4 x 8192 tokens of 80 heads, three others: 471; an eighth 483, half 499; without 498)
        const int64_t first = chunks / (4 * n + 1), others = (chunks - first + n - 1) / n;
        if (n > 1 && first > 0) {
            const double with = 9 + rounds * (8 + 8 * (double)others) + 25 + rounds * 8 * first + moved;
            if (with < best) {
                best = with;
                plan = {true, (int)n + 1, (int)first, (int)others, true};
            }
        }
    }
    return plan;
}

// Words of a scan's workspace: the segments' states and factors; on the matrix instructions records of the steps.
struct ScanRoom {
    uint64_t states = 0, decay = 0, steps = 0;
    uint64_t bytes() const { return 4 * (states + decay + steps); }
};
uint64_t whole(uint64_t n) { return (n + 3) / 4 * 4; }
ScanRoom scan_room(const ssd_dims *d, const ScanPlan &plan)
{
    ScanRoom r;
    const uint64_t rows = (uint64_t)d->batch * d->nheads;
    if (plan.tiles) r.steps = rows * (((uint64_t)d->seqlen + 63) / 64) * kScanRecord;
    if (plan.segments > 1) {
        r.states = whole(rows * plan.segments * d->headdim * d->dstate);
        r.decay = whole(rows * plan.segments);
    }
    return r;
}

// A call whose strides or addresses are not those that its sizes' plan is for runs on the kernel for any size, by that one's own plan.
ScanPlan other_plan(const ssd_dims *d, int n_cu)
{
    double cost;
    return any_plan(d, n_cu, cost);
}

int scan_dims(const ssd_dims *d, bool tokens)
{
    if (!d) return SSD_ERR_NULL;
    if (d->batch < 0 || (tokens && d->seqlen < 0) || d->nheads <= 0 || d->headdim <= 0 || d->dstate <= 0 || d->ngroups <= 0 ||
        d->nheads % d->ngroups)
        return SSD_ERR_SHAPE;
    return SSD_OK;
}

}  // namespace

extern "C" {

int ssd_short_conv_fwd(const ssd_tensor *x, const ssd_tensor *weight, const ssd_tensor *bias, const ssd_tensor *initial_states,
                       const ssd_tensor *seq_idx, const ssd_tensor *lengths, const ssd_tensor *y, const ssd_tensor *final_states,
                       int32_t batch, int32_t seqlen, int32_t dim, int32_t width, int silu, void *stream)
{
    if (batch < 0 || seqlen < 0 || dim <= 0 || width < 1 || width > 4) return SSD_ERR_SHAPE;
    if (batch == 0) return SSD_OK;
    const bool rows = seqlen > 0, state = width > 1;
    if (!present(weight) || (rows && (!present(x) || !present(y))) || (state && !present(final_states))) return SSD_ERR_NULL;
    if (!rows && !state) return SSD_OK;
    // without tokens the states say what the type is
    const int type = rows ? x->dtype : final_states->dtype;
    if (type != SSD_F32 && type != SSD_BF16 && type != SSD_F16) return SSD_ERR_DTYPE;
    if (rows && y->dtype != type) return SSD_ERR_DTYPE;
    if (!real(weight) || !real_or_absent(bias) || !ints_or_absent(seq_idx) || !ints_or_absent(lengths)) return SSD_ERR_DTYPE;
    if ((state && final_states->dtype != type) || (state && present(initial_states) && initial_states->dtype != type)) return SSD_ERR_DTYPE;
    if (rows && (!unit(x, 2, dim) || !unit(y, 2, dim))) return SSD_ERR_STRIDE;
    ConvParams p;
    memset(&p, 0, sizeof(p));
    p.w = weight->data; p.w_type = weight->dtype; p.sw_d = stride(weight, 0, dim); p.sw_k = width == 1 ? 1 : weight->stride[1];
    if (present(bias)) { p.bias = bias->data; p.bias_type = bias->dtype; p.sbias = dim == 1 ? 1 : bias->stride[0]; }
    if (state && present(initial_states)) {
        p.init = initial_states->data;
        p.si_b = initial_states->stride[0]; p.si_d = dim == 1 ? 1 : initial_states->stride[1]; p.si_k = initial_states->stride[2];
    }
    if (present(seq_idx)) { p.seq = (const int32_t *)seq_idx->data; p.sq_b = seq_idx->stride[0]; p.sq_l = seq_idx->stride[1]; }
    if (present(lengths)) { p.len = (const int32_t *)lengths->data; p.slen = lengths->stride[0]; }
    if (rows) {
        p.x = x->data; p.sx_b = x->stride[0]; p.sx_l = x->stride[1];
        p.y = y->data; p.sy_b = y->stride[0]; p.sy_l = y->stride[1];
    }
    if (state) {
        p.fin = final_states->data;
        p.sf_b = final_states->stride[0]; p.sf_d = dim == 1 ? 1 : final_states->stride[1]; p.sf_k = final_states->stride[2];
    }
    p.batch = batch; p.seqlen = seqlen; p.dim = dim; p.width = width; p.type = type; p.silu = silu;
    const int rc = device_status();
    return rc ? rc : launched(launch_short_conv(p, (hipStream_t)stream));
}

int ssd_short_conv_step(const ssd_tensor *x, const ssd_tensor *states, const ssd_tensor *weight, const ssd_tensor *bias,
                        const ssd_tensor *slots, const ssd_tensor *y, int32_t batch, int32_t dim, int32_t width, int32_t num_slots,
                        int silu, void *stream)
{
    if (batch < 0 || dim <= 0 || width < 1 || width > 4 || num_slots < 0) return SSD_ERR_SHAPE;
    if (batch == 0) return SSD_OK;
    const bool state = width > 1 && num_slots > 0;
    if (!present(x) || !present(weight) || !present(y) || (state && !present(states))) return SSD_ERR_NULL;
    if (!real(x) || y->dtype != x->dtype || !real(weight) || !real_or_absent(bias) || !ints_or_absent(slots) || (state && states->dtype != x->dtype))
        return SSD_ERR_DTYPE;
    if (!unit(x, 1, dim) || !unit(y, 1, dim)) return SSD_ERR_STRIDE;
    ConvStepParams p;
    memset(&p, 0, sizeof(p));
    p.x = x->data; p.sx_b = x->stride[0];
    p.y = y->data; p.sy_b = y->stride[0];
    if (state) { p.states = states->data; p.ss_s = states->stride[0]; p.ss_d = dim == 1 ? 1 : states->stride[1]; p.ss_k = states->stride[2]; }
    p.w = weight->data; p.w_type = weight->dtype; p.sw_d = stride(weight, 0, dim); p.sw_k = width == 1 ? 1 : weight->stride[1];
    if (present(bias)) { p.bias = bias->data; p.bias_type = bias->dtype; p.sbias = dim == 1 ? 1 : bias->stride[0]; }
    if (present(slots)) { p.slots = (const int32_t *)slots->data; p.sslots = slots->stride[0]; }
    p.batch = batch; p.dim = dim; p.width = width; p.n_slots = num_slots; p.type = x->dtype; p.silu = silu;
    const int rc = device_status();
    return rc ? rc : launched(launch_short_conv_step(p, (hipStream_t)stream));
}

uint64_t ssd_scan_workspace_bytes(const ssd_dims *dims, int type)
{
    if (scan_dims(dims, true) || dims->batch == 0 || dims->dstate > kScanMaxState) return 0;
    const int n_cu = device_compute_units();
    const ScanPlan plan = scan_plan(dims, type, n_cu);
    const uint64_t bytes = scan_room(dims, plan).bytes();
    if (!plan.tiles) return bytes;
    // (which kernel it will be is not known here)
    const uint64_t other = scan_room(dims, other_plan(dims, n_cu)).bytes();
    return bytes > other ? bytes : other;
}

int ssd_scan_fwd(const ssd_tensor *x, const ssd_tensor *dt, const ssd_tensor *A, const ssd_tensor *B, const ssd_tensor *C,
                 const ssd_tensor *D, const ssd_tensor *z, const ssd_tensor *dt_bias, const ssd_tensor *initial_states,
                 const ssd_tensor *seq_idx, const ssd_tensor *lengths, const ssd_tensor *y, const ssd_tensor *final_states,
                 const ssd_dims *dims, int dt_softplus, float dt_min, float dt_max, void *workspace, uint64_t workspace_bytes,
                 void *stream)
{
    int rc = scan_dims(dims, true);
    if (rc) return rc;
    if (dims->dstate > kScanMaxState) return SSD_ERR_SHAPE;
    const int64_t H = dims->nheads, P = dims->headdim, N = dims->dstate, G = dims->ngroups;
    if (dims->batch == 0) return SSD_OK;
    const bool rows = dims->seqlen > 0;
    if (!present(A) || !present(final_states) || (rows && (!present(x) || !present(dt) || !present(B) || !present(C) || !present(y))))
        return SSD_ERR_NULL;
    if (!real(A) || !real_or_absent(D) || !real_or_absent(dt_bias) || !real_or_absent(initial_states) || !ints_or_absent(seq_idx) ||
        !ints_or_absent(lengths) || final_states->dtype != SSD_F32)
        return SSD_ERR_DTYPE;
    if (rows && (!real(x) || !real(dt) || B->dtype != x->dtype || C->dtype != x->dtype || y->dtype != x->dtype ||
                 (present(z) && z->dtype != x->dtype)))
        return SSD_ERR_DTYPE;
    if (!unit(final_states, 3, N) || (present(initial_states) && !unit(initial_states, 3, N))) return SSD_ERR_STRIDE;
    if (rows && (!unit(x, 3, P) || !unit(B, 3, N) || !unit(C, 3, N) || !unit(y, 3, P) || (present(z) && !unit(z, 3, P)))) return SSD_ERR_STRIDE;
    SelScanParams p;
    memset(&p, 0, sizeof(p));
    p.batch = dims->batch; p.seqlen = dims->seqlen; p.nheads = dims->nheads; p.headdim = dims->headdim; p.dstate = dims->dstate;
    p.ngroups = dims->ngroups;
    p.A = A->data; p.A_type = A->dtype; p.sA = A->stride[0];
    if (rows) {
        p.type = x->dtype;
        p.x = x->data; p.sx_b = stride(x, 0, p.batch); p.sx_l = stride(x, 1, p.seqlen); p.sx_h = stride(x, 2, H);
        p.dt = dt->data; p.dt_type = dt->dtype; p.sdt_b = dt->stride[0]; p.sdt_l = dt->stride[1]; p.sdt_h = dt->stride[2];
        p.B = B->data; p.sB_b = stride(B, 0, p.batch); p.sB_l = stride(B, 1, p.seqlen); p.sB_g = stride(B, 2, G);
        p.C = C->data; p.sC_b = stride(C, 0, p.batch); p.sC_l = stride(C, 1, p.seqlen); p.sC_g = stride(C, 2, G);
        p.y = y->data; p.sy_b = stride(y, 0, p.batch); p.sy_l = stride(y, 1, p.seqlen); p.sy_h = stride(y, 2, H);
        if (present(z)) { p.z = z->data; p.z_type = z->dtype; p.sz_b = stride(z, 0, p.batch); p.sz_l = stride(z, 1, p.seqlen); p.sz_h = stride(z, 2, H); }
    }
    if (present(D)) { p.D = D->data; p.D_type = D->dtype; p.sD_h = D->stride[0]; p.sD_p = D->stride[1]; }
    if (present(initial_states)) {
        p.init = initial_states->data; p.init_type = initial_states->dtype;
        p.si_b = initial_states->stride[0]; p.si_h = initial_states->stride[1]; p.si_p = initial_states->stride[2];
    }
    if (present(seq_idx)) { p.seq = (const int32_t *)seq_idx->data; p.sq_b = seq_idx->stride[0]; p.sq_l = seq_idx->stride[1]; }
    if (present(lengths)) { p.len = (const int32_t *)lengths->data; p.slen = lengths->stride[0]; }
    p.fin = (float *)final_states->data;
    p.sf_b = stride(final_states, 0, p.batch); p.sf_h = stride(final_states, 1, H); p.sf_p = stride(final_states, 2, P);
    fill_delta(p.delta, dt_bias, dt_softplus, dt_min, dt_max);
    rc = device_status();
    if (rc) return rc;
    ScanPlan plan = scan_plan(dims, p.type, device_compute_units());
    if (plan.tiles && !scan_mfma_supported(p)) plan = other_plan(dims, device_compute_units());
    p.segments = plan.segments;
    const ScanRoom room = scan_room(dims, plan);
    const bool roomy = workspace && workspace_bytes >= room.bytes() && !((uintptr_t)workspace & 15);
    if (roomy) {
        p.ws_states = (float *)workspace;
        p.ws_decay = p.ws_states + room.states;
        p.ws_steps = p.ws_decay + room.decay;
    } else p.segments = 1;
    p.chunks = (int)(((int64_t)p.seqlen + 63) / 64);
    // whole chunks; the last segment may be shorter, or empty
    const bool tiles = rows && roomy && plan.tiles;
    if (tiles) {
        p.head = plan.head;
        p.head_tokens = p.segments > 1 ? 64 * plan.first : p.seqlen;
        p.segment_tokens = 64 * plan.others;
    } else p.segment_tokens = (int)((((int64_t)p.seqlen + p.segments - 1) / p.segments + 31) / 32 * 32);
    return launched(tiles ? launch_scan_mfma(p, (hipStream_t)stream) : launch_scan_any(p, (hipStream_t)stream));
}

int ssd_scan_step(const ssd_tensor *x, const ssd_tensor *dt, const ssd_tensor *A, const ssd_tensor *B, const ssd_tensor *C,
                  const ssd_tensor *D, const ssd_tensor *z, const ssd_tensor *dt_bias, const ssd_tensor *states,
                  const ssd_tensor *slots, const ssd_tensor *y, const ssd_dims *dims, int32_t num_slots, int dt_softplus,
                  float dt_min, float dt_max, void *stream)
{
    int rc = scan_dims(dims, false);
    if (rc) return rc;
    if (num_slots < 0) return SSD_ERR_SHAPE;
    if (dims->batch == 0) return SSD_OK;
    if (!present(x) || !present(dt) || !present(A) || !present(B) || !present(C) || !present(y) || (num_slots > 0 && !present(states)))
        return SSD_ERR_NULL;
    if (!real(x) || !real(dt) || !real(A) || B->dtype != x->dtype || C->dtype != x->dtype || y->dtype != x->dtype ||
        (present(z) && z->dtype != x->dtype) || !real_or_absent(D) || !real_or_absent(dt_bias) || !ints_or_absent(slots) ||
        (num_slots > 0 && states->dtype != SSD_F32))
        return SSD_ERR_DTYPE;
    const int64_t H = dims->nheads, P = dims->headdim, N = dims->dstate, G = dims->ngroups;
    if (!unit(x, 2, P) || !unit(B, 2, N) || !unit(C, 2, N) || !unit(y, 2, P) || (present(z) && !unit(z, 2, P)) ||
        (num_slots > 0 && !unit(states, 3, N)))
        return SSD_ERR_STRIDE;
    SelStepParams p;
    memset(&p, 0, sizeof(p));
    p.batch = dims->batch; p.nheads = dims->nheads; p.headdim = dims->headdim; p.dstate = dims->dstate; p.ngroups = dims->ngroups;
    p.n_slots = num_slots; p.type = x->dtype;
    p.x = x->data; p.sx_b = x->stride[0]; p.sx_h = x->stride[1];
    p.dt = dt->data; p.dt_type = dt->dtype; p.sdt_b = dt->stride[0]; p.sdt_h = dt->stride[1];
    p.A = A->data; p.A_type = A->dtype; p.sA = A->stride[0];
    p.B = B->data; p.sB_b = B->stride[0]; p.sB_g = B->stride[1];
    p.C = C->data; p.sC_b = C->stride[0]; p.sC_g = C->stride[1];
    if (present(D)) { p.D = D->data; p.D_type = D->dtype; p.sD_h = D->stride[0]; p.sD_p = D->stride[1]; }
    if (present(z)) { p.z = z->data; p.z_type = z->dtype; p.sz_b = z->stride[0]; p.sz_h = z->stride[1]; }
    if (num_slots > 0) {
        p.states = (float *)states->data;
        p.ss_s = stride(states, 0, num_slots); p.ss_h = stride(states, 1, H); p.ss_p = stride(states, 2, P);
    }
    if (present(slots)) { p.slots = (const int32_t *)slots->data; p.sslots = slots->stride[0]; }
    p.y = y->data; p.sy_b = y->stride[0]; p.sy_h = y->stride[1];
    fill_delta(p.delta, dt_bias, dt_softplus, dt_min, dt_max);
    (void)G;
    rc = device_status();
    return rc ? rc : launched(launch_scan_step(p, (hipStream_t)stream));
}

int ssd_norm_fwd(const ssd_tensor *x, const ssd_tensor *weight, const ssd_tensor *residual, const ssd_tensor *z, const ssd_tensor *out,
                 const ssd_tensor *scale, const ssd_tensor *residual_out, int64_t rows, int32_t dim, float eps, void *stream)
{
    if (rows < 0 || dim <= 0) return SSD_ERR_SHAPE;
    if (present(residual) && present(z)) return SSD_ERR_SHAPE;
    if (rows == 0) return SSD_OK;
    if (!present(x) || !present(weight) || !present(out) || present(residual) != present(residual_out)) return SSD_ERR_NULL;
    const bool int8 = out->dtype == SSD_I8;
    if (int8 && !present(scale)) return SSD_ERR_NULL;
    if (!real(x) || !real(weight) || (!int8 && out->dtype != x->dtype) || (int8 && scale->dtype != SSD_F32) ||
        (present(residual) && (residual->dtype != x->dtype || residual_out->dtype != x->dtype)) || (present(z) && z->dtype != x->dtype))
        return SSD_ERR_DTYPE;
    if (!unit(x, 1, dim) || !unit(out, 1, dim) || (present(residual) && (!unit(residual, 1, dim) || !unit(residual_out, 1, dim))) ||
        (present(z) && !unit(z, 1, dim)))
        return SSD_ERR_STRIDE;
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x->data; p.sx = x->stride[0]; p.type = x->dtype;
    p.w = weight->data; p.w_type = weight->dtype; p.sw = dim == 1 ? 1 : weight->stride[0];
    if (present(residual)) { p.residual = residual->data; p.sr = residual->stride[0]; p.residual_out = residual_out->data; p.sro = residual_out->stride[0]; }
    if (present(z)) { p.z = z->data; p.sz = z->stride[0]; }
    p.out = out->data; p.so = out->stride[0]; p.int8 = int8;
    if (int8) { p.scale = (float *)scale->data; p.sscale = scale->stride[0]; }
    p.rows = rows; p.dim = dim; p.eps = eps;
    const int rc = device_status();
    return rc ? rc : launched(launch_norm(p, (hipStream_t)stream));
}

int ssd_matmul_fwd(const ssd_tensor *a, const ssd_tensor *a_scale, const ssd_tensor *w, const ssd_tensor *w_scale,
                   const ssd_tensor *bias, const ssd_tensor *out, int32_t M, int32_t N, int32_t K, void *stream)
{
    if (M < 0 || N < 0 || K < 0 || K > SSD_MATMUL_MAX_K) return SSD_ERR_SHAPE;
    if (M == 0 || N == 0) return SSD_OK;
    if ((K > 0 && (!present(a) || !present(w))) || !present(a_scale) || !present(w_scale) || !present(out)) return SSD_ERR_NULL;
    if ((K > 0 && (a->dtype != SSD_I8 || w->dtype != SSD_I8)) || a_scale->dtype != SSD_F32 || w_scale->dtype != SSD_F32 ||
        !real_or_absent(bias) || !real(out))
        return SSD_ERR_DTYPE;
    if ((K > 0 && (!unit(a, 1, K) || !unit(w, 1, K))) || !unit(out, 1, N)) return SSD_ERR_STRIDE;
    MatmulParams p;
    memset(&p, 0, sizeof(p));
    if (K > 0) {
        p.a = (const int8_t *)a->data; p.sa_m = stride(a, 0, M);
        p.w = (const int8_t *)w->data; p.sw_n = stride(w, 0, N);
    }
    p.sa = (const float *)a_scale->data; p.ssa = a_scale->stride[0];
    p.sw = (const float *)w_scale->data; p.ssw = w_scale->stride[0];
    if (present(bias)) { p.bias = bias->data; p.bias_type = bias->dtype; p.sbias = bias->stride[0]; }
    p.out = out->data; p.out_type = out->dtype; p.so_m = stride(out, 0, M);
    p.M = M; p.N = N; p.K = K;
    const int rc = device_status();
    return rc ? rc : launched(launch_matmul(p, device_compute_units(), (hipStream_t)stream));
}

}  // extern "C"
