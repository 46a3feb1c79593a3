// Argument blocks of the operators of a decoding step around a served model's layers: product with 4-bit weights, norms around a block, beam
// selection and the reordering of states (ssd_matmul_packed.hip, ssd_norm_block.hip, ssd_beam.hip, ssd_reorder.hip).
#pragma once
#include "ssd_layer.h"

namespace ssd {

enum : int { DT_U8 = 4 };

struct PackedParams {
    const void *a;                     // (M, K)
    const uint8_t *w;                  // (N, ceil(K / 2)): the weight of an even k in the low half of its byte
    const void *scale;                 // (N, groups)
    const uint8_t *zero;               // (N, groups) or null: 8
    const void *bias;                  // (N) or null
    void *out;                         // (M, N)
    int M, N, K, group, groups;
    int64_t sa_m, sw_n, ss_n, ss_g, sz_n, sz_g, sbias, so_m;
    int type, scale_type, bias_type, out_type;
    void *room;                        // workspace
    uint64_t room_bytes;
};

struct NormBlockParams {
    const void *x, *residual;          // (rows, D)
    const void *w;                     // (D) or null: x is not normed
    const void *next_w;                // (D)
    const void *gate;                  // (ceil(rows / gate_every), D) or null
    void *out;                         // (rows, D): the type of x, or 8 bits
    float *scale;                      // (rows), with 8 bits
    void *residual_out;                // (rows, D)
    int64_t rows, gate_every;
    int dim;
    int64_t sx, sr, sg, so, sro, sscale;
    int type, int8, w_wide, next_wide, gate_wide;      // wide: fp32 where the type of x is not
    int past;                          // results go past the caches
    float factor, eps;
};

struct BeamParams {
    const void *logits;                // (b, beams, V)
    const float *scores;               // (b, beams)
    const uint8_t *finished;           // (b, beams) or null
    float *out_scores;                 // (b, k)
    int32_t *parents, *tokens;         // (b, k)
    double *ws_sums;                   // (b, beams, parts, 2): what a part's sum of exponentials is relative to (about its largest logit), and the sum
    uint64_t *ws_best;                 // (b, beams, parts, k): its k best
    int batch, beams, vocab, k, pad, parts, type;
    int first;                         // row of a merging launch
    int64_t sl_b, sl_i, ss_b, ss_i, sf_b, sf_i, so_b, sp_b, st_b;
};
constexpr int kBeamPart = 8192;        // tokens of a row that a workgroup takes
constexpr int kBeamMost = 64;          // selected, and beams

// One pool's slots as runs of bytes
struct PoolParams {
    char *data;
    int64_t slot_stride;               // bytes
    int64_t bytes;                     // of a slot
    int32_t first;                     // first workgroup of this pool in a row of the grid
};
constexpr int kPoolsPerLaunch = 48;
struct ReorderParams {
    const int32_t *parents, *slots;    // (b, beams)
    int32_t *new_slots;                // (b, beams); null: written by another launch
    int batch, beams, n_slots, n_pools;
    int past;                          // copies past the caches
    int64_t sp_b, sp_i, ss_b, ss_i, sn_b, sn_i;
    PoolParams pools[kPoolsPerLaunch];
};
// A pool whose slots are not runs of bytes
struct StridedPool {
    char *data;
    int element;                       // bytes
    int64_t slot_stride, count;        // elements
    int64_t size[4], stride[4];
};

uint64_t matmul_packed_room(int M, int N, int K, int group, int type, int n_cu);
hipError_t launch_matmul_packed(const PackedParams &p, int n_cu, hipStream_t s);
hipError_t launch_norm_block(const NormBlockParams &p, hipStream_t s);
hipError_t launch_beam_select(const BeamParams &p, hipStream_t s);
// workgroups of a pool of so many bytes a slot
int reorder_pieces(int64_t bytes);
hipError_t launch_reorder(const ReorderParams &p, int pieces, hipStream_t s);
hipError_t launch_reorder_strided(const ReorderParams &p, const StridedPool &pool, hipStream_t s);

}  // namespace ssd
