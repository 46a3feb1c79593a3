"""What the operators of a served Mamba2 layer are measured on: short convolution, selective scan, norm with 8-bit output and
8-bit matrix product, each in plain torch operations (own = False) or as the framework's calls (own = True).

A case is a dict of plain values; "op" says which operator:
  conv       _short_conv_fwd: b rows of L tokens, D channels, K taps; x is a view into a projection of before + D + after columns
  conv_step  _short_conv_step: one token of each of b rows, whose states lie in a pool of `slots`
  scan       _ssd_scan_fwd: b, L tokens, H heads of P, N state columns, G groups; x, B and C are views of one packed tensor
  scan_step  _ssd_scan_step: one token of each of b rows, states in a pool
  norm       _norm_fwd: rows x D; mode "residual" (x + residual) or "gate" (x * silu(z)); int8 = an output in 8 bits with scales
  matmul     _matmul_int8_fwd: (M, K) x (N, K) in 8 bits -> M x N of `dtype`
  dtype      of activations: bf16, fp16 or fp32;  init: initial states are given;  seqs: packed sequences per row (0: no seq_idx);
  ragged     rows end early (lengths), the last one has no token at all where there are several
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _framework():
    module = sys.modules.get("ssd_amd")
    if module is None:
        package = os.path.join(os.getcwd(), "mamba-fused-minimal_amd")
        if package not in sys.path:
            sys.path.insert(1, package)
        import ssd_amd as module
    return module


def _conv(name, b, L, D, before, after, K=4, dtype="bf16", init=False, seqs=0, ragged=False):
    return dict(name=name, op="conv", b=b, L=L, D=D, before=before, after=after, K=K, dtype=dtype, init=init, seqs=seqs, ragged=ragged)


def _scan(name, b, L, H, P=64, N=128, G=1, dtype="bf16", gate=True, init=False, seqs=0, ragged=False):
    return dict(name=name, op="scan", b=b, L=L, H=H, P=P, N=N, G=G, dtype=dtype, gate=gate, init=init, seqs=seqs, ragged=ragged)


def listed():
    return [
        # a batch of long prompts through the layer of the 2.7B model: x, B and C of 80 heads of 64 behind z in the projection
        _conv("conv_prompt_2p7b", 4, 8192, 5376, 5120, 80),
        # decoding 64 rows of the same layer out of a pool of states, some rows being padding
        dict(name="conv_step_2p7b", op="conv_step", b=64, D=5376, K=4, slots=80, padded=3, dtype="bf16"),
        # the scan of the long prompts, continued from earlier states
        _scan("scan_prompt_2p7b", 4, 8192, 80, init=True),
        # one short chat turn through the 130M model's layer: latency
        _scan("scan_short_130m", 1, 200, 24),
        # prompts of different length in one batch, the last row empty, B and C in 8 groups
        _scan("scan_ragged_grouped", 4, 3001, 128, G=8, ragged=True),
        # one row of packed sequences in single precision, sizes off every tiling
        _scan("scan_odd_fp32", 2, 1900, 15, P=48, N=96, G=3, dtype="fp32", init=True, seqs=4),
        # decoding 64 rows: the states are all the traffic
        dict(name="scan_step_2p7b", op="scan_step", b=64, H=80, P=64, N=128, G=1, slots=80, padded=3, gate=True, dtype="bf16"),
        # in front of the first projection, all tokens of the long prompts; in front of the second one, while decoding
        dict(name="norm_prompt_2p7b", op="norm", rows=32768, D=2560, mode="residual", int8=True, dtype="bf16"),
        dict(name="norm_gate_step_2p7b", op="norm", rows=64, D=5120, mode="gate", int8=True, dtype="bf16"),
        # the first projection of the 2.7B layer for 8192 tokens, and for a single one
        dict(name="matmul_prompt_2p7b", op="matmul", M=8192, K=2560, N=10576, bias=False, dtype="bf16"),
        dict(name="matmul_step_2p7b", op="matmul", M=1, K=2560, N=10576, bias=False, dtype="bf16"),
        # the second projection of the 130M layer for a ragged number of tokens
        dict(name="matmul_ragged_130m", op="matmul", M=777, K=1536, N=768, bias=True, dtype="fp16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _off(n):
    return n + 8 if n == 3072 else n


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan", "scan_step", "norm", "norm", "matmul", "matmul"])
    dtype = rng.choice(["bf16"] * 5 + ["fp16", "fp32"])
    if op in ("conv", "conv_step"):
        D = _off(_spread(rng, 64, 5376))
        if rng.random() < 0.7:
            D = _off(-(-D // 8) * 8)
        K = rng.choice([4, 4, 4, 3, 2])
        if op == "conv_step":
            b = _spread(rng, 1, 256)
            return dict(op=op, b=b, D=D, K=K, slots=b + rng.choice([0, 5, 40]), padded=rng.choice([0, 0, b // 8]), dtype=dtype)
        tokens = min(_spread(rng, 1, 65536), 170_000_000 // D // (2 if dtype == "fp32" else 1))
        b = min(rng.choice([1, 1, 2, 3, 8]), tokens)
        L = _off(max(1, tokens // b))
        before = rng.choice([0, 2 * D // 16 * 8, D + 3])
        return dict(op=op, b=b, L=L, D=D, before=before, after=rng.choice([0, 24, 80]), K=K, dtype=dtype, init=rng.random() < 0.4,
                    seqs=rng.choice([0, 0, 5]) if L >= 64 else 0, ragged=rng.random() < 0.3)
    if op in ("scan", "scan_step"):
        G = rng.choice([1, 1, 1, 2, 8])
        H = G * max(1, round(_spread(rng, 4, 128) / G))
        P, N = rng.choice([64, 64, 64, 64, 128, 32, 48, 40]), rng.choice([128, 128, 128, 64, 64, 16, 96, 256])
        if op == "scan_step":
            b = min(_spread(rng, 1, 256), max(1, 42_000_000 // (H * P * N)))
            return dict(op=op, b=b, H=H, P=P, N=N, G=G, slots=b + rng.choice([0, 5, 40]), padded=rng.choice([0, 0, b // 8]),
                        gate=rng.random() < 0.7, dtype=dtype)
        most = 160_000_000 if dtype == "bf16" and N <= 128 else 32_000_000
        tokens = max(1, min(_spread(rng, 1, 131072), most // (H * P)))
        b = min(rng.choice([1, 1, 2, 3, 4, 8]), tokens)
        L = _off(max(1, tokens // b))
        return dict(op=op, b=b, L=L, H=H, P=P, N=N, G=G, dtype=dtype, gate=rng.random() < 0.7, init=rng.random() < 0.4,
                    seqs=rng.choice([0, 0, 5]) if L >= 64 else 0, ragged=rng.random() < 0.3)
    if op == "norm":
        D = _spread(rng, 64, 8192)
        D = _off(-(-D // 8) * 8 if rng.random() < 0.8 else D)
        return dict(op=op, rows=min(_off(_spread(rng, 1, 32768)), 83_000_000 // D // (2 if dtype == "fp32" else 1)), D=D,
                    mode=rng.choice(["residual", "gate"]), int8=rng.random() < 0.8, dtype=dtype)
    K, N = _spread(rng, 256, 5120), _spread(rng, 64, 10576)
    K = -(-K // 16) * 16 if rng.random() < 0.8 else K
    return dict(op=op, M=_off(_spread(rng, 1, 8192)), K=_off(K), N=_off(N), bias=rng.random() < 0.3, dtype=dtype)


def _lengths(case):
    """Tokens of each row of a ragged batch."""
    b, L = case["b"], case["L"]
    return [L * 2 // 3] if b == 1 else [L * (b - 1 - i) // (b - 1) for i in range(b)]


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *size, dtype=dtype: torch.randn(size, generator=g, device=dev, dtype=dtype)  # noqa: E731
    uniform = lambda lo, hi, *size: torch.rand(size, generator=g, device=dev) * (hi - lo) + lo  # noqa: E731
    op = case["op"]
    s = dict(case=case, op=op)

    def rows(slots, b, padded):
        # the pool's slots in no order, the last rows without one
        index = torch.randperm(slots, generator=g, device=dev)[:b].to(torch.int32)
        if padded:
            index[b - padded:] = -1
        return index

    def marks():
        s["seq"] = s["lengths"] = None
        b, L = case["b"], case["L"]
        if case["seqs"]:
            starts = torch.zeros(b, L, device=dev, dtype=torch.int32)
            starts.scatter_(1, torch.randint(1, L, (b, case["seqs"] - 1), generator=g, device=dev), 1)
            s["seq"] = torch.cumsum(starts, dim=1, dtype=torch.int32)
        if case["ragged"]:
            s["lengths"] = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)

    if op in ("conv", "conv_step"):
        b, D, K = case["b"], case["D"], case["K"]
        s["w"], s["bias"] = normal(D, K) * K ** -0.5, 0.1 * normal(D)
        if op == "conv":
            s["x"] = normal(b, case["L"], case["before"] + D + case["after"])[..., case["before"]:case["before"] + D]
            s["init"] = normal(b, K - 1, D).transpose(1, 2) if case["init"] else None
            marks()
        else:
            s["x"], s["slots"] = normal(b, D), rows(case["slots"], b, case["padded"])
            s["states"] = normal(case["slots"], K - 1, D).transpose(1, 2)
    elif op in ("scan", "scan_step"):
        b, H, P, N, G = (case[k] for k in "bHPNG")
        L = case["L"] if op == "scan" else 1
        # what the convolution leaves: values around one, mostly positive after its activation
        packed = torch.nn.functional.silu(normal(b, L, H * P + 2 * G * N))
        x, B, C = packed.split([H * P, G * N, G * N], dim=-1)
        s["x"], s["B"], s["C"] = x.view(b, L, H, P), B.view(b, L, G, N), C.view(b, L, G, N)
        # z and the raw dt from both ends of the projection; dt log-uniform in 1e-3 .. 1e-1 behind bias and softplus, A in -16 .. -1
        dt = torch.exp(uniform(math.log(1e-3), math.log(1e-1), b, L, H))
        s["dt_bias"] = torch.full((H,), -4.6, device=dev)
        s["dt"] = (dt + torch.log(-torch.expm1(-dt)) - s["dt_bias"]).to(dtype)
        s["z"] = normal(b, L, H * P + 80)[..., :H * P].view(b, L, H, P) if case["gate"] else None
        s["A"], s["D"] = -torch.exp(uniform(0.0, math.log(16.0), H)), uniform(0.5, 1.5, H)
        if op == "scan":
            s["init"] = 0.1 * normal(b, H, P, N, dtype=torch.float32) if case["init"] else None
            marks()
        else:
            for k in ("x", "B", "C", "dt", "z"):
                s[k] = None if s[k] is None else s[k][:, 0]
            s["states"], s["slots"] = normal(case["slots"], H, P, N, dtype=torch.float32), rows(case["slots"], b, case["padded"])
    elif op == "norm":
        n, D = case["rows"], case["D"]
        s["x"], s["w"] = normal(n, D), uniform(0.5, 1.5, D).to(dtype)
        s["residual"] = 4 * normal(n, D) if case["mode"] == "residual" else None
        s["z"] = normal(n, D + 80)[:, :D] if case["mode"] == "gate" else None
    else:
        M, K, N = (case[k] for k in "MKN")
        eight = lambda *size: torch.clamp(torch.round(32 * normal(*size, dtype=torch.float32)), -127, 127).to(torch.int8)  # noqa: E731
        s["a"], s["w"] = eight(M, K), eight(N, K)
        s["sa"], s["sw"] = uniform(0.01, 0.05, M), uniform(0.5, 1.5, N) / (32 * K ** 0.5)
        s["bias"] = normal(N) if case["bias"] else None
        s["dtype"] = dtype
    return s


def run(s):
    return _own(s) if own else _PLAIN[s["op"]](s)


def _own(s):
    f, op = _framework(), s["op"]
    if op == "conv":
        return f._short_conv_fwd(s["x"], s["w"], s["bias"], initial_states=s["init"], seq_idx=s["seq"], lengths=s["lengths"])
    if op == "conv_step":
        return f._short_conv_step(s["x"], s["states"], s["w"], s["bias"], slots=s["slots"]), s["states"]
    if op == "scan":
        return f._ssd_scan_fwd(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True,
                               initial_states=s["init"], seq_idx=s["seq"], lengths=s["lengths"])
    if op == "scan_step":
        return f._ssd_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["states"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                dt_softplus=True, slots=s["slots"]), s["states"]
    if op == "norm":
        out, scale, residual = f._norm_fwd(s["x"], s["w"], residual=s["residual"], z=s["z"], eps=1e-5, int8=s["case"]["int8"])
        # 8 bits as the values they stand for
        return (out if scale is None else torch.mul(out, scale[:, None])), residual
    return f._matmul_int8_fwd(s["a"], s["sa"], s["w"], s["sw"], bias=s["bias"], out_dtype=s["dtype"])


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end

def _silu(t):
    return t / (1 + torch.exp(-t))


def _runs(s, b, L, dev):
    """For every token the number of sequence starts up to it (0 in front of the row): tokens of equal number belong together."""
    if s["seq"] is None:
        return torch.zeros(b, L, device=dev, dtype=torch.int64)
    before = torch.nn.functional.pad(s["seq"], (1, 0))[:, :-1]
    return torch.cumsum(s["seq"] != before, dim=1)


def _valid(s, b, L, dev):
    if s["lengths"] is None:
        return torch.ones(b, L, device=dev, dtype=torch.bool)
    return torch.arange(L, device=dev)[None] < s["lengths"][:, None]


def _plain_conv(s):
    x, w = s["x"], s["w"].float()
    b, L, D = x.shape
    K, dev = w.shape[1], x.device
    valid = _valid(s, b, L, dev)
    front = torch.zeros(b, K - 1, D, device=dev) if s["init"] is None else s["init"].float().transpose(1, 2)
    xs = torch.cat([front, torch.where(valid[..., None], x.float(), 0.0)], dim=1)
    runs = torch.nn.functional.pad(_runs(s, b, L, dev), (K - 1, 0))
    y = s["bias"].float().expand(b, L, D)
    for k in range(K):
        same = runs[:, k:k + L] == runs[:, K - 1:]
        y = y + torch.where(same[..., None], xs[:, k:k + L], 0.0) * w[:, k]
    y = torch.where(valid[..., None], _silu(y), 0.0).to(x.dtype)
    n = torch.full((b,), L, device=dev) if s["lengths"] is None else s["lengths"].long()
    at = n[:, None] + torch.arange(K - 1, device=dev)[None]
    final = torch.gather(xs, 1, at[..., None].expand(b, K - 1, D))
    last = torch.gather(runs, 1, (n + K - 2)[:, None])
    final = torch.where((torch.gather(runs, 1, at) == last)[..., None], final, 0.0)
    return y, final.transpose(1, 2).to(x.dtype)


def _plain_conv_step(s):
    x, states, w, slots = s["x"], s["states"], s["w"].float(), s["slots"].long()
    there = slots >= 0
    at = slots.clamp(min=0)
    window = torch.cat([states[at], x[..., None]], dim=2)
    y = _silu((window.float() * w).sum(-1) + s["bias"].float())
    y = torch.where(there[:, None], y, 0.0).to(x.dtype)
    states[at[there]] = window[there][..., 1:]
    return y, states


def _delta(s):
    dt = s["dt"].float() + s["dt_bias"]
    return torch.where(dt > 20, dt, torch.log1p(torch.exp(dt.clamp(max=20))))


def _plain_scan(s, T=64):
    x, A = s["x"], s["A"]
    b, L, H, P = x.shape
    G, N, dev = s["B"].shape[2], s["B"].shape[3], x.device
    c, pad = -(-L // T), -L % T
    valid, runs, delta = _valid(s, b, L, dev), _runs(s, b, L, dev), _delta(s)
    delta = torch.where(valid[..., None], delta, 0.0)
    xf = torch.where(valid[..., None, None], x.float(), 0.0)
    chunks = lambda t: torch.nn.functional.pad(t.transpose(1, -1), (0, pad)).transpose(1, -1).unflatten(1, (c, T))  # noqa: E731
    if pad:
        runs = torch.cat([runs, runs[:, -1:].expand(b, pad)], dim=1)
    runs = runs.unflatten(1, (c, T))                                            # (b, c, T)
    d = chunks(delta).permute(0, 1, 3, 2)                                       # (b, c, H, T)
    cs = torch.cumsum(d * A[:, None], dim=-1)
    xd = chunks(xf).permute(0, 1, 3, 2, 4) * d[..., None]                       # (b, c, H, T, P)
    Bc, Cc = (chunks(t.float()).permute(0, 1, 3, 2, 4) for t in (s["B"], s["C"]))
    grouped = lambda t: t.unflatten(2, (G, H // G))  # noqa: E731
    scores = torch.matmul(Cc, Bc.transpose(-1, -2))                             # (b, c, G, T, T)
    seen = (runs[..., :, None] == runs[..., None, :]) & torch.ones(T, T, device=dev, dtype=torch.bool).tril()
    decay = torch.exp(torch.where(seen[:, :, None], cs[..., :, None] - cs[..., None, :], float("-inf")))
    y = torch.matmul((grouped(decay) * scores[:, :, :, None]).flatten(2, 3), xd)
    keep = (runs == runs[..., -1:])[:, :, None]
    w = torch.where(keep, torch.exp(cs[..., -1:] - cs), 0.0)
    add = torch.matmul(grouped(xd * w[..., None]).transpose(-1, -2), Bc[:, :, :, None]).flatten(2, 3)   # (b, c, H, P, N)
    entering = torch.empty(b, c, H, P, N, device=dev)
    state = torch.zeros(b, H, P, N, device=dev) if s["init"] is None else s["init"].float()
    ends = torch.nn.functional.pad(runs[..., -1], (1, 0))
    through = torch.where((ends[:, 1:] == ends[:, :-1])[..., None], torch.exp(cs[..., -1]), 0.0)
    for i in range(c):
        entering[:, i] = state
        state = state * through[:, i][..., None, None] + add[:, i]
    reach = torch.where((runs == ends[:, :-1, None])[:, :, None], torch.exp(cs), 0.0)
    y = y + torch.matmul(Cc[:, :, :, None], grouped(entering).transpose(-1, -2)).flatten(2, 3) * reach[..., None]
    y = y.permute(0, 1, 3, 2, 4).reshape(b, c * T, H, P)[:, :L] + s["D"][:, None] * xf
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return torch.where(valid[..., None, None], y, 0.0).to(x.dtype), state


def _plain_scan_step(s):
    x, states, slots = s["x"], s["states"], s["slots"].long()
    H, G = x.shape[1], s["B"].shape[1]
    there, at = slots >= 0, slots.clamp(min=0)
    heads = lambda t: t.float().repeat_interleave(H // G, dim=1)  # noqa: E731
    d = _delta(s)
    new = states[at] * torch.exp(d * s["A"])[..., None, None] + (d[..., None] * x.float())[..., None] * heads(s["B"])[:, :, None]
    y = (new * heads(s["C"])[:, :, None]).sum(-1) + s["D"][:, None] * x.float()
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    states[at[there]] = new[there]
    return torch.where(there[:, None, None], y, 0.0).to(x.dtype), states


def _plain_norm(s):
    x, residual = s["x"], None
    t = x.float()
    if s["residual"] is not None:
        t = t + s["residual"].float()
        residual = t.to(x.dtype)
    if s["z"] is not None:
        t = t * _silu(s["z"].float())
    u, r = t * s["w"].float(), torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)
    if not s["case"]["int8"]:
        return (u * r).to(x.dtype), residual
    # the root mean square only scales a row: what is rounded to 8 bits is u over the row's largest
    most = u.abs().amax(-1, keepdim=True)
    q = torch.round(u * (127 / most)).to(torch.int8)
    return torch.mul(q, most * r / 127), residual


def _plain_matmul(s):
    out = torch.matmul(s["a"].float(), s["w"].float().t()) * s["sa"][:, None] * s["sw"]
    return (out if s["bias"] is None else out + s["bias"].float()).to(s["dtype"])


_PLAIN = {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
          "norm": _plain_norm, "matmul": _plain_matmul}


def work(case):
    e, op = (4 if case["dtype"] == "fp32" else 2), case["op"]
    if op == "conv":
        b, L, D, K = (case[k] for k in "bLDK")
        T = sum(_lengths(case)) if case["ragged"] else b * L
        n = T * D * e + b * L * D * e + (D * K + D) * e + b * D * (K - 1) * e * (2 if case["init"] else 1)
        return {"bytes": n + (b * L * 4 if case["seqs"] else 0), "flops": 2 * K * T * D}
    if op == "conv_step":
        b, D, K = (case[k] for k in "bDK")
        live = b - case["padded"]
        return {"bytes": (live * D * (2 * K - 1) + b * D + D * (K + 1)) * e, "flops": 2 * K * live * D}
    if op == "scan":
        b, L, H, P, N, G = (case[k] for k in "bLHPNG")
        T = sum(_lengths(case)) if case["ragged"] else b * L
        n = (T * H * P * (2 if case["gate"] else 1) + 2 * T * G * N + T * H + b * L * H * P) * e
        n += b * H * P * N * 4 * (2 if case["init"] else 1) + (b * L * 4 if case["seqs"] else 0)
        return {"bytes": n, "flops": 6 * T * H * P * N}
    if op == "scan_step":
        b, H, P, N, G = (case[k] for k in "bHPNG")
        live = b - case["padded"]
        n = live * (2 * H * P * N * 4 + (H * P * (2 if case["gate"] else 1) + 2 * G * N + H) * e) + b * H * P * e
        return {"bytes": n, "flops": 6 * live * H * P * N}
    if op == "norm":
        n, D = case["rows"], case["D"]
        moved = n * D * e * (3 if case["mode"] == "residual" else 2) + D * e
        return {"bytes": moved + n * D * (4 if case["int8"] else e), "flops": 8 * n * D}
    M, K, N = (case[k] for k in "MKN")
    return {"bytes": M * K + N * K + M * N * e + 4 * (M + N) + (N * e if case["bias"] else 0), "flops": 2 * M * K * N}


# ---- the definitions in 64 bits

def _exact_marks(s, b, L):
    """Per row: its tokens, and for each of them whether a sequence starts there (host values)."""
    n = [L] * b if s["lengths"] is None else s["lengths"].tolist()
    ids = torch.zeros(b, L, dtype=torch.int64) if s["seq"] is None else s["seq"].long().cpu()
    starts = torch.ones(b, L, dtype=torch.bool)
    starts[:, 1:] = ids[:, 1:] != ids[:, :-1]
    starts[:, 0] = ids[:, 0] != 0
    return n, starts


def _exact_conv(s):
    b, L, D = s["x"].shape
    w, bias = s["w"].double(), s["bias"].double()
    K = w.shape[1]
    n, starts = _exact_marks(s, b, L)
    y = torch.zeros(b, L, D, device=w.device, dtype=torch.float64)
    final = torch.zeros(b, D, K - 1, device=w.device, dtype=torch.float64)
    for i in range(b):
        row = torch.zeros(K - 1 + n[i], D, device=w.device, dtype=torch.float64)
        if s["init"] is not None:
            row[:K - 1] = s["init"][i].double().t()
        row[K - 1:] = s["x"][i, :n[i]].double()
        edges = torch.nonzero(starts[i, :n[i]]).flatten().tolist()
        edges = [0] + [t for t in edges if t > 0] + [n[i]] if n[i] else [0]
        fresh = bool(starts[i, 0]) and n[i] > 0
        tail = row[n[i]:].clone()
        for lo, hi in zip(edges[:-1], edges[1:]):
            piece = row[lo:K - 1 + hi].clone()
            if lo > 0 or fresh:
                piece[:K - 1] = 0
            acc = (piece.unfold(0, K, 1) * w).sum(-1) + bias
            y[i, lo:hi] = acc * torch.sigmoid(acc)
            tail = piece[hi - lo:]
        final[i] = tail.t()
    return y, final


def _exact_delta(s):
    v = s["dt"].double() + s["dt_bias"].double()
    return torch.logaddexp(v, torch.zeros_like(v))


def _exact_scan(s):
    b, L, H, P = s["x"].shape
    G, N = s["B"].shape[2:]
    R, dev = H // G, s["x"].device
    n, starts = _exact_marks(s, b, L)
    delta, A = _exact_delta(s), s["A"].double()
    live = torch.arange(L)[None] < torch.tensor(n)[:, None]
    keep = torch.exp(delta * A) * (~starts).to(dev)[..., None]
    keep = torch.where(live.to(dev)[..., None], keep, torch.ones((), device=dev, dtype=torch.float64)).view(b, L, G, R, 1, 1)
    push = (delta * live.to(dev)[..., None])[..., None] * s["x"].double()
    push = push.view(b, L, G, R, P, 1)
    h = torch.zeros(b, H, P, N, device=dev, dtype=torch.float64) if s["init"] is None else s["init"].double()
    h = h.reshape(b, G, R, P, N).clone()
    y = torch.empty(b, L, G, R, P, device=dev, dtype=torch.float64)
    B, C = s["B"].double()[:, :, :, None, None, :], s["C"].double()[:, :, :, None, None, :]
    for t in range(L):
        h.mul_(keep[:, t]).addcmul_(push[:, t], B[:, t])
        torch.sum(h * C[:, t], dim=-1, out=y[:, t])
    y = y.view(b, L, H, P) + s["D"].double()[:, None] * s["x"].double()
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    return y * live.to(dev)[..., None, None], h.view(b, H, P, N)


def exact(case, seed):
    op = case["op"]
    if op == "scan":
        # token by token: launches, or passes over the states where those take longer
        if case["L"] * max(60e-6, case["b"] * case["H"] * case["P"] * case["N"] * 8 * 8 / 3e12) > 15:
            return None
        return _exact_scan(prepare(case, seed))
    s = prepare(case, seed)
    if op == "conv":
        return _exact_conv(s)
    if op == "conv_step":
        y, states = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64), s["states"].double()
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                window = torch.cat([states[slot], s["x"][i].double()[:, None]], dim=1)
                acc = (window * s["w"].double()).sum(1) + s["bias"].double()
                y[i], states[slot] = acc * torch.sigmoid(acc), window[:, 1:]
        return y, states
    if op == "scan_step":
        y, states = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64), s["states"].double()
        R, delta, A = case["H"] // case["G"], _exact_delta(s), s["A"].double()
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                x = s["x"][i].double()
                B, C = (s[k][i].double().repeat_interleave(R, dim=0) for k in "BC")
                h = states[slot] * torch.exp(delta[i] * A)[:, None, None] + (x * delta[i][:, None])[..., None] * B[:, None]
                y[i] = (h * C[:, None]).sum(-1) + s["D"].double()[:, None] * x
                if s["z"] is not None:
                    y[i] *= s["z"][i].double() * torch.sigmoid(s["z"][i].double())
                states[slot] = h
        return y, states
    if op == "norm":
        t, w = s["x"].double(), s["w"].double()
        if s["residual"] is not None:
            t = t + s["residual"].double()
        residual = t.clone() if s["residual"] is not None else None
        if s["z"] is not None:
            t = t * s["z"].double() * torch.sigmoid(s["z"].double())
        normed = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) * w
        if case["int8"]:
            step = normed.abs().amax(-1, keepdim=True) / 127
            normed = torch.round(normed / step) * step
        return normed, residual
    out = s["a"].double() @ s["w"].double().t()
    out = out * s["sa"].double()[:, None] * s["sw"].double()[None]
    return out if s["bias"] is None else out + s["bias"].double()
