"""The operators of a decoding step around a served model's layers: matrix product with weights in 4 bits, the norms behind and in front of a
block with its gate and the residual's scale, beam search's selection, and the states' way to the beams that it selects.

Like the wrappers of layer.py: they own allocation and argument checking, the arithmetic runs in the gfx950 HIP kernels behind the C ABI
(include/ssd_gfx950.h, which states the formulas), asynchronously on the current torch stream; there is no CPU path.  Forward only:
results carry no gradient."""
import ctypes

import torch

from . import _lib
from .layer import _REAL, _arg, _as, _call, _common, _int32, _same_device, _unit
from .ops import _ordinary

_MOST_BEAMS = 64


def _bytes_arg(t):
    """ssd_tensor of a tensor of bytes or truth values, or of None."""
    if t is None:
        return _lib.tensor_arg(None)
    s = _lib.SsdTensor()
    s.data, s.dtype = t.data_ptr(), _lib.SSD_U8
    for i, st in enumerate(t.stride()):
        s.stride[i] = st
    return s


def _matmul_int4_fwd(a, w, w_scale, w_zero=None, group=128, bias=None, out_dtype=None):
    """Matrix product with weights in 4 bits: out[..., n] = sum_g w_scale[n, g] sum_{k in g} a[..., k] (q[n, k] - w_zero[n, g]) (+ bias[n]).

    a (..., K) bf16, fp16 or fp32; w (N, ceil(K / 2)) uint8 with two weights to a byte, q[n, 2 j] in the lower half of byte j; w_scale
    (N, ceil(K / group)) of any of the three types; w_zero of the same shape, uint8 (8 without it: weights -8 .. 7); bias (N).  ``group``
    weights of a channel share a scale: a multiple of 32, or K and more for one scale a channel.  Products and a group's sums are fp32 (so
    sums over a (q - zero) have to fit it), the result is rounded once to ``out_dtype`` (a's type by default)."""
    out_dtype = a.dtype if out_dtype is None else out_dtype
    group = int(group)
    done = _ordinary(a, "matmul_packed_call", a, w, w_scale, w_zero, group, bias, out_dtype)
    if done is not None:
        return done
    K, N = a.shape[-1], w.shape[0]
    assert a.dtype in _REAL and out_dtype in _REAL and w_scale.dtype in _REAL
    assert w.dtype == torch.uint8 and w.shape == (N, (K + 1) // 2), "two weights to a byte"
    assert group > 0 and (group % 32 == 0 or group >= K), "groups of a multiple of 32 weights, or one of all"
    rows = a.shape[:-1].numel()
    assert max(rows, N, K) <= 1 << 30
    assert w_scale.shape == (N, -(-K // group))
    if w_zero is not None:
        assert w_zero.dtype == torch.uint8 and w_zero.shape == w_scale.shape
    if bias is not None:
        assert bias.shape == (N,) and bias.dtype in _REAL
    _lib.require_device(a, "_matmul_int4_fwd")
    _same_device(a, w, w_scale, w_zero, bias)
    flat, w = _unit(a.reshape(rows, K)), _unit(w)
    out = torch.empty((rows, N), device=a.device, dtype=out_dtype)
    with torch.cuda.device(a.device):
        nbytes = int(_lib.load().ssd_matmul_packed_workspace_bytes(rows, N, K, min(group, 1 << 30), _lib._DTYPES[a.dtype]))
    room = torch.empty((nbytes + 3) // 4, device=a.device, dtype=torch.float32) if nbytes else None
    _call(a, "ssd_matmul_packed_fwd", _arg(flat), _bytes_arg(w), _arg(w_scale), _bytes_arg(w_zero), _arg(bias), _arg(out), rows, N, K, min(group, 1 << 30),
          ctypes.c_void_p(room.data_ptr() if nbytes else None), nbytes)
    return out.view(*a.shape[:-1], N)


def _norm_block_fwd(x, weight, residual, next_weight, gate=None, residual_scale=1.0, eps=1e-5, int8=False):
    """What stands between two blocks, x being the first one's output, over the last dimension:
    t = residual_scale residual + gate x weight / sqrt(mean(x^2) + eps);  out = t next_weight / sqrt(mean(t^2) + eps).

    ``weight`` (dim) or None (no norm behind the block), ``next_weight`` (dim), ``gate`` None or (dim), or of x's dimensions with those in front
    either x's or, from some one on, 1: a gate per channel, per row of a batch, or per token.  Returns (out, scale, t): ``int8=False``: out of
    x's type, scale None; ``int8=True``: out int8 and scale (fp32, one per row) as ``_norm_fwd`` has them.  t is the residual of what follows.
    A residual or a gate per token (of x's own shape) of another type than x is taken as it is: t has the type that holds all of them (fastest with one
    type).  Gates of other shapes may be of any type and do not change t's."""
    done = _ordinary(x, "norm_block_call", x, weight, residual, next_weight, gate, float(residual_scale), float(eps), 1 if int8 else 0)
    if done is not None:
        return done
    dim = x.shape[-1]
    assert 0 < dim <= 1 << 30 and x.dtype in _REAL
    assert residual.shape == x.shape
    assert next_weight.shape == (dim,) and (weight is None or weight.shape == (dim,))
    rows, every = x.numel() // dim, 1
    if gate is not None:
        assert gate.shape[-1:] == (dim,) and gate.dim() <= x.dim(), "a gate of x's last dimension"
        lead = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1])
        own = 0                                  # leading dimensions of its own
        while own < len(lead) and lead[own] == x.shape[own]:
            own += 1
        assert all(n == 1 for n in lead[own:]), "a gate's leading dimensions are x's and then 1"
        every = x.shape[own:-1].numel()
    # (in a single row a gate of fewer dimensions has every == 1 too, and stays one per channel: what t's type is must not depend on how many rows there are)
    full = gate is not None and x.dim() > 1 and gate.shape == x.shape
    given, common = x.dtype, _common(x, residual, gate if full else None)
    assert all(t is None or t.dtype in _REAL for t in (weight, next_weight, gate))
    _lib.require_device(x, "_norm_block_fwd")
    _same_device(x, weight, residual, next_weight, gate)
    flat, residual = (_unit(_as(t, common).reshape(rows, dim)) for t in (x, residual))
    # weights and gates of another type than the rows: in fp32, which holds them
    small = lambda t: None if t is None else _unit(t if t.dtype in (common, torch.float32) else t.float())  # noqa: E731
    weight, next_weight = small(weight), small(next_weight)
    gate = None if gate is None else small(gate.reshape(-1, dim))
    out = torch.empty((rows, dim), device=x.device, dtype=torch.int8 if int8 else common)
    scale = torch.empty((rows,), device=x.device, dtype=torch.float32) if int8 else None
    total = torch.empty((rows, dim), device=x.device, dtype=common)
    _call(x, "ssd_norm_block_fwd", _arg(flat), _arg(weight), _arg(residual), _arg(next_weight), _arg(gate), _arg(out), _arg(scale), _arg(total), rows, dim,
          max(every, 1), float(residual_scale), float(eps))
    out = out if int8 else _as(out, given)
    return out.view(x.shape), scale.view(x.shape[:-1]) if int8 else None, total.view(x.shape)


def _beam_select_fwd(logits, scores, k=None, finished=None, pad=0):
    """Beam search's selection: of the candidates scores[b, i] + log_softmax(logits[b, i])[v] of each row the ``k`` best (as many as beams by
    default), best first, equals by the lowest i * vocab + v.

    logits (batch, beams, vocab) bf16, fp16 or fp32; scores (batch, beams) fp32, the log-probability of each beam so far (-inf: a beam that is
    not there).  ``finished`` (batch, beams) bool: such a beam has one candidate, the token ``pad`` at its score as it is.  A token with a
    logit of -inf is not allowed; finite ones, however large, have the scores of the formula.  What is not a number counts as -inf: all of a beam
    whose score is not finite, or with a NaN or +inf among its logits.  Returns (scores, parents, tokens), (batch, k) each: fp32 and twice int32.
    beams and k are at most 64, beams * vocab below 2^31, vocab at most 2^30."""
    batch, beams, vocab = logits.shape
    k = beams if k is None else int(k)
    pad = int(pad)
    done = _ordinary(logits, "beam_select_call", logits, scores, k, finished, pad)
    if done is not None:
        return done
    assert logits.dtype in _REAL and scores.is_floating_point() and scores.shape == (batch, beams)
    assert 0 < beams <= _MOST_BEAMS and 0 < k <= _MOST_BEAMS, "beams and k are at most 64"
    assert 0 < vocab <= 1 << 30 and beams * vocab < 1 << 31 and k <= beams * vocab
    if finished is not None:
        assert finished.shape == (batch, beams) and finished.dtype in (torch.bool, torch.uint8) and 0 <= pad < vocab
    _lib.require_device(logits, "_beam_select_fwd")
    _same_device(logits, scores, finished)
    logits, scores = _unit(logits), _as(scores, torch.float32)
    best = torch.empty((batch, k), device=logits.device, dtype=torch.float32)
    parents, tokens = (torch.empty((batch, k), device=logits.device, dtype=torch.int32) for _ in range(2))
    nbytes = int(_lib.load().ssd_beam_workspace_bytes(batch, beams, vocab, k))
    room = torch.empty((nbytes // 8,), device=logits.device, dtype=torch.float64)
    _call(logits, "ssd_beam_select_fwd", _arg(logits), _arg(scores), _bytes_arg(finished), _arg(best), _arg(parents), _arg(tokens), batch, beams, vocab, k, pad,
          ctypes.c_void_p(room.data_ptr() if nbytes else None), nbytes)
    return best, parents, tokens


def _beam_reorder(parents, slots, pools):
    """States follow their beams: child j of row b goes on from beam parents[b, j], whose states are in slot slots[b, parents[b, j]] of every
    pool.  A beam's first child takes its slot; each other one the slot of a beam without a child, which is overwritten with its parent's states.

    parents and slots (batch, beams) whole numbers, beams at most 64; ``pools``: a sequence of tensors (num_slots, ...) of up to five
    dimensions, any type and layout, updated in place.  Returns the children's slots (batch, beams) int32.  A child whose parent is no beam
    or has a slot outside the pools (padding), or for whom no slot is left, has slot -1.  Beams of a row that share a slot count as one beam; rows share
    none."""
    pools = list(pools)
    done = _ordinary(parents, "beam_reorder_call", parents, slots, pools)
    if done is not None:
        return done
    batch, beams = parents.shape
    assert 0 < beams <= _MOST_BEAMS, "at most 64 beams"
    assert slots.shape == (batch, beams)
    n_slots = pools[0].shape[0] if pools else 1 << 31
    for pool in pools:
        assert 1 <= pool.dim() <= 5 and pool.shape[0] == n_slots, "pools of as many slots each"
        assert not pool.is_quantized and pool.layout == torch.strided
        assert all(n <= 1 or st > 0 for n, st in zip(pool.shape, pool.stride())), "elements of a pool that share a place"
    parents, slots = _int32(parents, -1, beams), _int32(slots, -1, min(n_slots, (1 << 31) - 1))
    _lib.require_device(parents, "_beam_reorder")
    _same_device(parents, slots, *pools)
    new = torch.empty((batch, beams), device=parents.device, dtype=torch.int32)
    described = (_lib.SsdPool * max(len(pools), 1))()
    for to, pool in zip(described, pools):
        to.data, to.element_bytes, to.dims, to.slot_stride = pool.data_ptr(), pool.element_size(), pool.dim() - 1, pool.stride(0)
        for i in range(pool.dim() - 1):
            to.size[i], to.stride[i] = pool.shape[i + 1], pool.stride(i + 1)
    _call(parents, "ssd_beam_reorder", _arg(parents), _arg(slots), _arg(new), described, len(pools), min(n_slots, (1 << 31) - 1), batch, beams)
    return new
