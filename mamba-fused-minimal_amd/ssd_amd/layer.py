"""The operators of a served Mamba2 layer around the state path: short convolution and selective scan (for prompts and for single
tokens), root-mean-square norm with an output in 8 bits, matrix product in 8 bits.

Like the wrappers of ops.py: they own allocation and argument checking, the arithmetic runs in the gfx950 HIP kernels behind the C ABI
(include/ssd_gfx950.h, which states the formulas), asynchronously on the current torch stream; there is no CPU path.  Forward only:
results carry no gradient."""
import ctypes
import functools

import torch

from . import _lib
from .ops import _on_device, _ordinary

_REAL = (torch.float32, torch.bfloat16, torch.float16)
_INF = float("inf")


def _arg(t):
    """ssd_tensor of a tensor or None; 8-bit integers too."""
    if t is not None and t.dtype == torch.int8:
        s = _lib.SsdTensor()
        s.data, s.dtype = t.data_ptr(), _lib.SSD_I8
        for i, st in enumerate(t.stride()):
            s.stride[i] = st
        return s
    return _lib.tensor_arg(t)


def _call(t, name, *args):
    """The C entry point on t's device and its current stream."""
    rc = _on_device(t, lambda *a: getattr(_lib.load(), name)(*a[:-1], ctypes.c_void_p(a[-1])), *args)
    _lib.check(rc, name)


def _unit(t):
    return t if t is None or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _as(t, dtype):
    return t if t is None or t.dtype == dtype else t.to(dtype)


def _common(*tensors):
    """The type that holds what all of them hold."""
    types = [t.dtype for t in tensors if t is not None]
    assert all(dtype in _REAL for dtype in types)
    return functools.reduce(torch.promote_types, types)


def _same_device(t, *others):
    for o in others:
        assert o is None or o.device == t.device, "tensors on different devices"


def _int32(t, lo, hi):
    """Whole numbers of any width as int32, those outside lo .. hi as the nearer of the two."""
    if t is None or t.dtype == torch.int32:
        return t
    assert not t.is_floating_point() and not t.is_complex(), "whole numbers"
    return (t.clamp(lo, hi) if t.dtype == torch.int64 else t).to(torch.int32)


def _check_marks(batch, seqlen, seq_idx, lengths):
    if seq_idx is not None:
        assert seq_idx.shape == (batch, seqlen)
    if lengths is not None:
        assert lengths.shape == (batch,)
    return _as(seq_idx, torch.int32), _int32(lengths, 0, seqlen)


def _check_slots(batch, states, slots):
    if slots is None:
        assert states.shape[0] == batch, "without slots row b has states[b]"
    else:
        assert slots.shape == (batch,)
    # (a slot of 64 bits outside the pool must not become one inside it)
    return _int32(slots, -1, states.shape[0])


def _short_conv_fwd(x, weight, bias=None, silu=True, initial_states=None, seq_idx=None, lengths=None):
    """Short causal convolution of prompts, a filter per channel: x (batch, seqlen, dim), weight (dim, width) with 1 to 4 taps, bias (dim).
    y[b,t,d] = silu(bias[d] + sum_k weight[d,k] x[b,t-width+1+k,d]) (without silu where ``silu`` is false).

    ``initial_states`` (batch, dim, width-1): the inputs in front of the row (of sequence 0; zeros by default).  ``seq_idx`` (batch,
    seqlen): packed sequences, a tap never reaches into another one.  ``lengths`` (batch): tokens of each row; y is zero behind them.
    Returns (y, final_states): final_states (batch, dim, width-1), channels contiguous, are the states ``_short_conv_step`` goes on from.
    y has x's type; initial states of a wider type are taken as they are, and final_states have that type then."""
    done = _ordinary(x, "short_conv_call", x, weight, bias, 1 if silu else 0, initial_states, seq_idx, lengths)
    if done is not None:
        return done
    batch, seqlen, dim = x.shape
    width = weight.shape[1]
    assert weight.shape == (dim, width) and 1 <= width <= 4, "a filter has 1 to 4 taps"
    assert dim > 0 and x.dtype in _REAL
    if bias is not None:
        assert bias.shape == (dim,)
    if initial_states is not None:
        assert initial_states.shape == (batch, dim, width - 1)
    seq_idx, lengths = _check_marks(batch, seqlen, seq_idx, lengths)
    given, common = x.dtype, _common(x, initial_states)
    _lib.require_device(x, "_short_conv_fwd")
    _same_device(x, weight, bias, initial_states, seq_idx, lengths)
    x, initial_states = _unit(_as(x, common)), _as(initial_states, common)
    y = torch.empty((batch, seqlen, dim), device=x.device, dtype=x.dtype)
    final_states = torch.empty((batch, width - 1, dim), device=x.device, dtype=x.dtype).transpose(1, 2)
    _call(x, "ssd_short_conv_fwd", _arg(x), _arg(weight), _arg(bias), _arg(initial_states), _arg(seq_idx), _arg(lengths), _arg(y),
          _arg(final_states), batch, seqlen, dim, width, 1 if silu else 0)
    return _as(y, given), final_states


def _short_conv_step(x, states, weight, bias=None, silu=True, slots=None):
    """One token of ``_short_conv_fwd``: x (batch, dim) -> y (batch, dim); ``states`` (num_slots, dim, width-1), of the type of x, are updated
    in place (fastest with contiguous channels).  ``slots`` (batch) int32: row b has states[slots[b]], a slot outside the pool marks
    padding (y = 0, nothing updated); without it row b has states[b].  No two rows may share a slot."""
    done = _ordinary(x, "short_conv_step_call", x, states, weight, bias, 1 if silu else 0, slots)
    if done is not None:
        return done
    batch, dim = x.shape
    width = weight.shape[1]
    assert weight.shape == (dim, width) and 1 <= width <= 4, "a filter has 1 to 4 taps"
    assert dim > 0 and x.dtype in _REAL
    assert states.dim() == 3 and states.shape[1:] == (dim, width - 1) and states.dtype == x.dtype
    if bias is not None:
        assert bias.shape == (dim,)
    slots = _check_slots(batch, states, slots)
    _lib.require_device(x, "_short_conv_step")
    _same_device(x, states, weight, bias, slots)
    x = _unit(x)
    y = torch.empty((batch, dim), device=x.device, dtype=x.dtype)
    _call(x, "ssd_short_conv_step", _arg(x), _arg(states), _arg(weight), _arg(bias), _arg(slots), _arg(y), batch, dim, width,
          states.shape[0], 1 if silu else 0)
    return y


def _check_heads(A, D, dt_bias, nheads, headdim, ngroups):
    assert nheads > 0 and headdim > 0 and ngroups > 0 and nheads % ngroups == 0
    assert A.shape == (nheads,)
    if D is not None:
        assert D.shape in ((nheads,), (nheads, headdim))
    if dt_bias is not None:
        assert dt_bias.shape == (nheads,)


def _ssd_scan_fwd(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, _INF), initial_states=None, seq_idx=None,
                  lengths=None):
    """The whole selective scan of prompts in one call: dt preparation, decay, both halves of the output, skip and gate.

    x (batch, seqlen, nheads, headdim), dt (batch, seqlen, nheads) raw, A (nheads), B and C (batch, seqlen, ngroups, dstate <= 256),
    D (nheads) or (nheads, headdim), z like x.  With d = clamp(softplus(dt + dt_bias), *dt_limit):
    h = exp(d A) h + d x (outer) B;  y = (h C + D x) silu(z).
    ``initial_states`` (batch, nheads, headdim, dstate), ``seq_idx`` and ``lengths`` as for ``_short_conv_fwd``.
    Returns (y of x's type, final_states (batch, nheads, headdim, dstate) fp32).  Where x, B, C and z are of several types the call runs in the
    one that holds them all (fastest with one type).  Larger calls in bf16 multiply on the bf16 matrix instructions what is not bf16 already
    (states, weighted x, scores) in 16 bits: final_states are then within 2.2e-6 of their norm, with x, B and C given in fp32 within 3e-7."""
    lo, hi = float(dt_limit[0]), float(dt_limit[1])
    done = _ordinary(x, "scan_call", x, dt, A, B, C, D, z, dt_bias, 1 if dt_softplus else 0, lo, hi, initial_states, seq_idx, lengths)
    if done is not None:
        return done
    batch, seqlen, nheads, headdim = x.shape
    ngroups, dstate = B.shape[2:]
    _check_heads(A, D, dt_bias, nheads, headdim, ngroups)
    assert x.dtype in _REAL and 0 < dstate <= 256, "dstate is at most 256"
    assert dt.shape == (batch, seqlen, nheads)
    assert B.shape == (batch, seqlen, ngroups, dstate) and C.shape == B.shape
    if z is not None:
        assert z.shape == x.shape
    if initial_states is not None:
        assert initial_states.shape == (batch, nheads, headdim, dstate)
    seq_idx, lengths = _check_marks(batch, seqlen, seq_idx, lengths)
    given, common = x.dtype, _common(x, B, C, z)
    _lib.require_device(x, "_ssd_scan_fwd")
    _same_device(x, dt, A, B, C, D, z, dt_bias, initial_states, seq_idx, lengths)
    x, B, C, z = (_unit(_as(t, common)) for t in (x, B, C, z))
    initial_states = _unit(_as(initial_states, torch.float32))
    y = torch.empty((batch, seqlen, nheads, headdim), device=x.device, dtype=x.dtype)
    final_states = torch.empty((batch, nheads, headdim, dstate), device=x.device, dtype=torch.float32)
    dims = _lib.dims_arg(batch, seqlen, nheads, headdim, dstate, ngroups, 0, 0)
    with torch.cuda.device(x.device):
        nbytes = int(_lib.load().ssd_scan_workspace_bytes(dims, _lib._DTYPES[x.dtype]))
    room = torch.empty((nbytes + 3) // 4, device=x.device, dtype=torch.float32) if nbytes else None
    _call(x, "ssd_scan_fwd", _arg(x), _arg(dt), _arg(A), _arg(B), _arg(C), _arg(D), _arg(z), _arg(dt_bias), _arg(initial_states), _arg(seq_idx),
          _arg(lengths), _arg(y), _arg(final_states), dims, 1 if dt_softplus else 0, lo, hi,
          ctypes.c_void_p(room.data_ptr() if nbytes else None), nbytes)
    return _as(y, given), final_states


def _ssd_scan_step(x, dt, A, B, C, states, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, _INF), slots=None):
    """One token of ``_ssd_scan_fwd``: x, z (batch, nheads, headdim), dt (batch, nheads), B and C (batch, ngroups, dstate); ``states``
    (num_slots, nheads, headdim, dstate) fp32 are updated in place, ``slots`` as for ``_short_conv_step``.  Returns y like x; several types as
    for ``_ssd_scan_fwd``."""
    lo, hi = float(dt_limit[0]), float(dt_limit[1])
    done = _ordinary(x, "scan_step_call", x, dt, A, B, C, states, D, z, dt_bias, 1 if dt_softplus else 0, lo, hi, slots)
    if done is not None:
        return done
    batch, nheads, headdim = x.shape
    ngroups, dstate = B.shape[1:]
    _check_heads(A, D, dt_bias, nheads, headdim, ngroups)
    assert x.dtype in _REAL and dstate > 0
    assert dt.shape == (batch, nheads)
    assert B.shape == (batch, ngroups, dstate) and C.shape == B.shape
    assert states.dim() == 4 and states.shape[1:] == (nheads, headdim, dstate) and states.dtype == torch.float32
    assert dstate == 1 or states.stride(-1) == 1, "states are updated in place: their columns must be contiguous"
    if z is not None:
        assert z.shape == x.shape
    slots = _check_slots(batch, states, slots)
    given, common = x.dtype, _common(x, B, C, z)
    _lib.require_device(x, "_ssd_scan_step")
    _same_device(x, dt, A, B, C, states, D, z, dt_bias, slots)
    x, B, C, z = (_unit(_as(t, common)) for t in (x, B, C, z))
    y = torch.empty((batch, nheads, headdim), device=x.device, dtype=x.dtype)
    _call(x, "ssd_scan_step", _arg(x), _arg(dt), _arg(A), _arg(B), _arg(C), _arg(D), _arg(z), _arg(dt_bias), _arg(states), _arg(slots), _arg(y),
          _lib.dims_arg(batch, 1, nheads, headdim, dstate, ngroups, 0, 0), states.shape[0], 1 if dt_softplus else 0, lo, hi)
    return _as(y, given)


def _norm_fwd(x, weight, residual=None, z=None, eps=1e-5, int8=False):
    """Root-mean-square norm over the last dimension of t = x + residual, or t = x silu(z), or x: t weight / sqrt(mean(t^2) + eps).

    Returns (out, scale, residual_out).  ``int8=False``: out of x's type, scale None.  ``int8=True``: out int8 and scale (fp32, one per row)
    with out * scale the normed values; a row's largest becomes +-127.  residual_out is x + residual, rounded (None without a residual):
    the residual of the next layer.  A residual or a gate of another type than x is taken as it is: residual_out has the type that holds
    both (fp32 for a residual kept in fp32), out x's (fastest with one type)."""
    done = _ordinary(x, "norm_call", x, weight, residual, z, float(eps), 1 if int8 else 0)
    if done is not None:
        return done
    dim = x.shape[-1]
    assert dim > 0 and x.dtype in _REAL
    assert weight.shape == (dim,)
    assert residual is None or z is None, "a residual or a gate, not both"
    for t in (residual, z):
        assert t is None or t.shape == x.shape
    given, common = x.dtype, _common(x, residual, z)
    _lib.require_device(x, "_norm_fwd")
    _same_device(x, weight, residual, z)
    rows = lambda t: None if t is None else _unit(_as(t, common).reshape(-1, dim))  # noqa: E731
    flat, residual, z = rows(x), rows(residual), rows(z)
    out = torch.empty(flat.shape, device=x.device, dtype=torch.int8 if int8 else common)
    scale = torch.empty(flat.shape[:1], device=x.device, dtype=torch.float32) if int8 else None
    residual_out = torch.empty(flat.shape, device=x.device, dtype=common) if residual is not None else None
    _call(x, "ssd_norm_fwd", _arg(flat), _arg(weight), _arg(residual), _arg(z), _arg(out), _arg(scale), _arg(residual_out), flat.shape[0], dim,
          float(eps))
    out = out if int8 else _as(out, given)
    return (out.view(x.shape), scale.view(x.shape[:-1]) if int8 else None, None if residual is None else residual_out.view(x.shape))


def _matmul_int8_fwd(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16):
    """Matrix product in 8-bit integers: out[..., n] = a_scale[...] w_scale[n] sum_k a[..., k] w[n, k] (+ bias[n]).

    a (..., K) int8 with a_scale (...) fp32 per token, w (N, K) int8 with w_scale (N) fp32 per channel, bias (N).  Sums are exact 32-bit
    integers (K <= 131071); the scales and the bias are applied in fp32, the result is rounded to ``out_dtype`` (bf16, fp16 or fp32)."""
    done = _ordinary(a, "matmul_call", a, a_scale, w, w_scale, bias, out_dtype)
    if done is not None:
        return done
    K, N = a.shape[-1], w.shape[0]
    assert a.dtype == torch.int8 and w.dtype == torch.int8 and w.shape == (N, K)
    assert K <= 131071, "beyond this 32-bit sums could overflow"
    assert a_scale.shape == a.shape[:-1] and w_scale.shape == (N,)
    assert out_dtype in _REAL
    if bias is not None:
        assert bias.shape == (N,)
    _lib.require_device(a, "_matmul_int8_fwd")
    _same_device(a, a_scale, w, w_scale, bias)
    flat, w, scales = _unit(a.reshape(a_scale.numel(), K)), _unit(w), _as(a_scale, torch.float32).reshape(-1)
    w_scale = _as(w_scale, torch.float32)
    out = torch.empty((flat.shape[0], N), device=a.device, dtype=out_dtype)
    _call(a, "ssd_matmul_fwd", _arg(flat), _arg(scales), _arg(w), _arg(w_scale), _arg(bias), _arg(out), flat.shape[0], N, K)
    return out.view(*a.shape[:-1], N)
