"""The operators around the state path, restated token by token in 64 bits on the CPU (test infrastructure).

Each scan and convolution also returns, where asked, the same sums over absolute values: what a bound on rounding errors scales with."""
import torch

f64 = torch.float64


def silu(t):
    return t * torch.sigmoid(t)


def tokens_of(b, L, lengths):
    return [L] * b if lengths is None else [min(max(int(n), 0), L) for n in lengths]


def starts_of(b, L, seq_idx):
    """Whether a sequence starts at a token: its id differs from the one before (0 in front of the row)."""
    ids = torch.zeros(b, L, dtype=torch.int64) if seq_idx is None else seq_idx.long().cpu()
    return ids != torch.nn.functional.pad(ids, (1, 0))[:, :L]


def short_conv_ref(x, weight, bias=None, act=True, initial_states=None, seq_idx=None, lengths=None):
    """-> y, final_states, and the sums over absolute values in front of the activation"""
    b, L, D = x.shape
    K = weight.shape[1]
    x, w = x.double().cpu(), weight.double().cpu()
    n, starts = tokens_of(b, L, lengths), starts_of(b, L, seq_idx)
    y, size, final = torch.zeros(b, L, D, dtype=f64), torch.zeros(b, L, D, dtype=f64), torch.zeros(b, D, K - 1, dtype=f64)
    for i in range(b):
        window = torch.zeros(D, K - 1, dtype=f64) if initial_states is None else initial_states[i].double().cpu().clone()
        for t in range(n[i]):
            if starts[i, t]:
                window = torch.zeros(D, K - 1, dtype=f64)
            full = torch.cat([window, x[i, t][:, None]], dim=1)
            pre = (full * w).sum(1) + (0 if bias is None else bias.double().cpu())
            size[i, t] = (full * w).abs().sum(1) + (0 if bias is None else bias.double().cpu().abs())
            y[i, t] = silu(pre) if act else pre
            window = full[:, 1:]
        final[i] = window
    return y, final, size


def short_conv_step_ref(x, states, weight, bias=None, act=True, slots=None):
    """-> y, the pool of states behind it"""
    b, D = x.shape
    y, states = torch.zeros(b, D, dtype=f64), states.double().cpu().clone()
    for i in range(b):
        slot = i if slots is None else int(slots[i])
        if 0 <= slot < states.shape[0]:
            full = torch.cat([states[slot], x[i].double().cpu()[:, None]], dim=1)
            pre = (full * weight.double().cpu()).sum(1) + (0 if bias is None else bias.double().cpu())
            y[i] = silu(pre) if act else pre
            states[slot] = full[:, 1:]
    return y, states


def delta_ref(dt, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf"))):
    d = dt.double().cpu() + (0 if dt_bias is None else dt_bias.double().cpu())
    if dt_softplus:
        d = torch.where(d > 20, d, torch.log1p(torch.exp(d.clamp(max=20))))
    return d.clamp(*dt_limit)


def ssd_scan_ref(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")), initial_states=None,
                 seq_idx=None, lengths=None):
    """-> y, final_states, and both over absolute values"""
    b, L, H, P = x.shape
    G, N = B.shape[2:]
    x, B, C, A = (t.double().cpu() for t in (x, B, C, A))
    B, C = (t.repeat_interleave(H // G, dim=2) for t in (B, C))
    d = delta_ref(dt, dt_bias, dt_softplus, dt_limit)
    skip = torch.zeros(H, 1, dtype=f64) if D is None else D.double().cpu().view(H, -1)
    gate = torch.ones(b, L, H, P, dtype=f64) if z is None else silu(z.double().cpu())
    n, starts = tokens_of(b, L, lengths), starts_of(b, L, seq_idx)
    y, size = torch.zeros(b, L, H, P, dtype=f64), torch.zeros(b, L, H, P, dtype=f64)
    final, final_size = torch.zeros(b, H, P, N, dtype=f64), torch.zeros(b, H, P, N, dtype=f64)
    for i in range(b):
        h = torch.zeros(H, P, N, dtype=f64) if initial_states is None else initial_states[i].double().cpu().clone()
        m = h.abs()
        for t in range(n[i]):
            keep = torch.exp(d[i, t] * A)[:, None, None]
            h, m = (torch.zeros_like(h), torch.zeros_like(m)) if starts[i, t] else (h, m)
            push = (d[i, t][:, None] * x[i, t])[:, :, None] * B[i, t][:, None]
            h, m = keep * h + push, keep * m + push.abs()
            y[i, t] = ((h * C[i, t][:, None]).sum(-1) + skip * x[i, t]) * gate[i, t]
            size[i, t] = ((m * C[i, t][:, None].abs()).sum(-1) + (skip * x[i, t]).abs()) * gate[i, t].abs()
        final[i], final_size[i] = h, m
    return y, final, size, final_size


def ssd_scan_step_ref(x, dt, A, B, C, states, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")), slots=None):
    """-> y, the pool of states behind it, and y's sums over absolute values"""
    b, H, P = x.shape
    y, size, states = torch.zeros(b, H, P, dtype=f64), torch.zeros(b, H, P, dtype=f64), states.double().cpu().clone()
    one = lambda t, i: None if t is None else t[i:i + 1, None]  # noqa: E731
    for i in range(b):
        slot = i if slots is None else int(slots[i])
        if 0 <= slot < states.shape[0]:
            out, last, mag, _ = ssd_scan_ref(one(x, i), one(dt, i), A, one(B, i), one(C, i), D, one(z, i), dt_bias, dt_softplus, dt_limit,
                                             initial_states=states[slot][None])
            y[i], size[i], states[slot] = out[0, 0], mag[0, 0], last[0]
    return y, states, size


def norm_ref(x, weight, residual=None, z=None, eps=1e-5):
    """-> the normed values (not quantized), the sum with the residual"""
    t = x.double().cpu()
    total = None
    if residual is not None:
        t = total = t + residual.double().cpu()
    if z is not None:
        t = t * silu(z.double().cpu())
    return t * weight.double().cpu() / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps), total


def matmul_int8_ref(a, a_scale, w, w_scale, bias=None):
    out = (a.long().cpu() @ w.long().cpu().t()).double() * a_scale.double().cpu()[..., None] * w_scale.double().cpu()
    return out if bias is None else out + bias.double().cpu()
