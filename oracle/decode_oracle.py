"""The operators of a decoding step around a served model's layers, restated in 64 bits on the CPU (test infrastructure).

The products and norms also return what a bound on rounding errors scales with."""
import torch

f64 = torch.float64


def d(t):
    return None if t is None else t.double().cpu()


def unpacked(w, K):
    """Bytes (N, ceil(K / 2)) -> the 4-bit weights (N, K)"""
    w = w.cpu().long()
    q = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.int64)
    q[:, 0::2], q[:, 1::2] = w % 16, w // 16
    return q[:, :K]


def matmul_int4_ref(a, w, w_scale, w_zero=None, group=128, bias=None):
    """-> out, and its sum over absolute values"""
    K = a.shape[-1]
    of = torch.arange(K) // group
    zero = torch.full((w.shape[0], K), 8) if w_zero is None else w_zero.cpu().long()[:, of]
    values = (unpacked(w, K) - zero).double() * d(w_scale)[:, of]
    out, size = d(a) @ values.t(), d(a).abs() @ values.abs().t()
    return out if bias is None else out + d(bias), size


def norm_block_ref(x, weight, residual, next_weight, gate=None, residual_scale=1.0, eps=1e-5):
    """-> out (not in 8 bits), t, and the branch's part of t"""
    n = d(x)
    if weight is not None:
        n = n / torch.sqrt(n.pow(2).mean(-1, keepdim=True) + eps) * d(weight)
    if gate is not None:
        n = n * d(gate)
    # (the factor as the call has it, in 32 bits)
    t = float(torch.tensor(residual_scale, dtype=torch.float32)) * d(residual) + n
    return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps) * d(next_weight), t, n


def beam_candidates(logits, scores, finished=None, pad=0):
    """-> all candidates (batch, beams, vocab)"""
    x, s = d(logits), d(scores)
    batch, beams, vocab = x.shape
    c = torch.full((batch, beams, vocab), -float("inf"), dtype=f64)
    for b in range(batch):
        for i in range(beams):
            if not bool(torch.isfinite(s[b, i])):
                continue
            if finished is not None and bool(finished[b, i]):
                c[b, i, pad] = s[b, i]
            elif not bool((torch.isnan(x[b, i]) | (x[b, i] == float("inf"))).any()) and float(x[b, i].max()) > -float("inf"):
                less = x[b, i] - x[b, i].max()      # (64 bits do not hold a large logit and the logarithm of a sum together)
                c[b, i] = s[b, i] + (less - torch.log(torch.exp(less).sum()))
    return c


def beam_select_ref(logits, scores, k, finished=None, pad=0):
    """-> scores, parents, tokens, and the distance of the nearest two of the k + 1 best that are of different beams and not equal"""
    c = beam_candidates(logits, scores, finished, pad)
    batch, beams, vocab = c.shape
    v, at = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    near = float("inf")
    for b in range(batch):
        for j in range(min(k, v.shape[1] - 1)):
            gap = float(v[b, j] - v[b, j + 1]) if float(v[b, j + 1]) > -float("inf") else float("inf")
            if 0 < gap and int(at[b, j]) // vocab != int(at[b, j + 1]) // vocab:
                near = min(near, gap)
    return v[:, :k], (at[:, :k] // vocab), (at[:, :k] % vocab), near


def beam_reorder_ref(parents, slots, pools):
    """-> the children's slots, the pools behind it"""
    pools, old = [p.clone().cpu() for p in pools], [p.cpu() for p in pools]
    n = old[0].shape[0] if old else 1 << 31
    new = []
    for row, held in zip(parents.tolist(), slots.tolist()):
        there = lambda p: 0 <= p < len(held) and 0 <= held[p] < n  # noqa: E731
        row = [held.index(held[p]) if there(p) else p for p in row]      # beams that share a slot are one
        spare = [s for i, s in enumerate(held) if there(i) and held.index(s) == i and i not in row]
        used, given = set(), []
        for p in row:
            if not there(p):
                given.append(-1)
            elif p not in used:
                used.add(p)
                given.append(held[p])
            elif spare:
                given.append(spare.pop(0))
                for pool, before in zip(pools, old):
                    pool[given[-1]] = before[held[p]]
            else:
                given.append(-1)
        new.append(given)
    return torch.tensor(new, dtype=torch.int64).view(parents.shape), pools
