"""What the operators of a decoding step around a served model's layers are measured on: matrix product with 4-bit weights, norms before and
after a block with its gate and residual scale, beam search's selection and the reordering of states that follows it, each in plain
torch operations (own = False) or as the framework's calls (own = True).

A case is a dict of plain values; "op" says which operator:
  matmul4  _matmul_int4_fwd: (M, K) of `dtype` x (N, K) in 4 bits -> M x N; `group` weights share a scale (0: all of a row); zeros: and a zero
           point of their own (8 without); bias
  block    _norm_block_fwd: x, residual (b, L, D); weight: a norm behind the block; gate "none", "channel" (D), "row" (b, D) or "token"
           (like x); int8 = an output in 8 bits with scales
  select   _beam_select_fwd: the k best of `beams` x V candidates in each of b rows; finished: some beams have ended, masked: some tokens
           are not allowed
  reorder  _beam_reorder: b rows of `beams` beams whose states lie in `layers` pools each of H x P x N fp32 and D x 3 `dtype`; in each row
           `copies` beams are dropped and as many others go on twice; padded: that many rows are padding
  dtype    of activations, logits and filter states: bf16, fp16 or fp32
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


def _matmul4(name, M, K, N, group=128, zeros=False, bias=False, dtype="bf16"):
    return dict(name=name, op="matmul4", M=M, K=K, N=N, group=group, zeros=zeros, bias=bias, dtype=dtype)


def _block(name, b, L, D, weight=True, gate="channel", scale=1.0, int8=False, dtype="bf16"):
    return dict(name=name, op="block", b=b, L=L, D=D, weight=weight, gate=gate, scale=scale, int8=int8, dtype=dtype)


def _select(name, b, beams, V, k, finished=False, masked=False, dtype="bf16"):
    return dict(name=name, op="select", b=b, beams=beams, V=V, k=k, finished=finished, masked=masked, dtype=dtype)


def _reorder(name, b, beams, copies, layers, H, P, N, D, padded=0, dtype="bf16"):
    return dict(name=name, op="reorder", b=b, beams=beams, copies=copies, layers=layers, H=H, P=P, N=N, D=D, padded=padded, dtype=dtype)


def listed():
    return [
        # the first projection of the 2.7B layer for a single token
        _matmul4("matmul4_step_2p7b", 1, 2560, 10576),
        # its second one for a batch of 64 decoded tokens, weights with zero points in smaller groups
        _matmul4("matmul4_batch_2p7b", 64, 5120, 2560, group=64, zeros=True),
        # a short prompt through the first projection
        _matmul4("matmul4_prompt_2p7b", 2048, 2560, 10576),
        # seven beams of one row through a layer whose sizes no tile divides
        _matmul4("matmul4_odd_fp16", 7, 1543, 777, group=32, zeros=True, bias=True, dtype="fp16"),
        # between two layers, all tokens of long prompts: norm of the block's output, a gate per channel, the next layer's norm
        _block("block_prompt_2p7b", 4, 8192, 2560, scale=0.8),
        # the same for 64 decoded tokens, in front of a projection in 8 bits
        _block("block_step_2p7b", 64, 1, 2560, int8=True),
        # rows of several conditions in single precision, sizes off every vector
        _block("block_odd_fp32", 3, 1901, 1537, gate="row", scale=1.2, dtype="fp32"),
        # one conversation searched with four beams: latency
        _select("select_one_row", 1, 4, 32000, 4),
        # a batch of 64 rows with eight beams, twice as many candidates as beams so that ended ones can be put aside
        _select("select_batch", 64, 8, 50000, 16, finished=True),
        # a large vocabulary in fp32, parts of it not allowed
        _select("select_wide_fp32", 3, 5, 128001, 5, masked=True, dtype="fp32"),
        # behind such a selection: the states of four of the 2.7B model's layers, 16 rows of four beams, one dropped in each
        _reorder("reorder_2p7b", 16, 4, 1, 4, 80, 64, 128, 5376),
        # the 130M model's 24 layers for one row with three beams
        _reorder("reorder_130m", 1, 3, 1, 24, 24, 64, 128, 1792),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["matmul4", "matmul4", "matmul4", "block", "block", "select", "select", "reorder"])
    dtype = rng.choice(["bf16"] * 5 + ["fp16", "fp32"])
    if op == "matmul4":
        K, N = _spread(rng, 64, 8192), _spread(rng, 64, 10576)
        K = -(-K // 64) * 64 if rng.random() < 0.8 else K
        N = -(-N // 16) * 16 if rng.random() < 0.7 else N
        M = _spread(rng, 1, 2048) if rng.random() < 0.5 else _spread(rng, 1, 64)
        M = max(1, min(M, 2048 * 10576 * 2560 // (K * N)))
        return dict(op=op, M=M, K=K, N=N, group=rng.choice([32, 64, 128, 128, 128, 256, 0]), zeros=rng.random() < 0.4, bias=rng.random() < 0.3, dtype=dtype)
    if op == "block":
        D = _spread(rng, 64, 16384)
        D = -(-D // 8) * 8 if rng.random() < 0.8 else D
        rows = min(_spread(rng, 1, 32768), 83_000_000 // D // (2 if dtype == "fp32" else 1))
        b = min(rng.choice([1, 2, 3, 8, 64]), rows)
        gate = rng.choice(["none", "channel", "channel", "row", "token"])
        return dict(op=op, b=b, L=max(1, rows // b // (2 if gate == "token" else 1)), D=D, weight=rng.random() < 0.8, gate=gate,
                    scale=rng.choice([1.0, 1.0, 0.5, 1.3]), int8=rng.random() < 0.3, dtype=dtype)
    if op == "select":
        beams, V = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 16, 32]), _spread(rng, 300, 260000)
        b = max(1, min(_spread(rng, 1, 128), 25_600_000 // (beams * V * (2 if dtype == "fp32" else 1))))
        return dict(op=op, b=b, beams=beams, V=V, k=rng.choice([beams, beams, 2 * beams]), finished=rng.random() < 0.3, masked=rng.random() < 0.3, dtype=dtype)
    H, P, N = rng.choice([8, 15, 24, 48, 80]), rng.choice([64, 64, 64, 48, 33]), rng.choice([128, 128, 64, 16, 96])
    beams, D = rng.choice([2, 3, 4, 4, 5, 8, 16]), H * P + 2 * N
    # (no more copied, and no more held, than in the largest listed case)
    b, copies = _spread(rng, 1, 16), rng.randint(0, min(4, beams - 1))
    layers = max(1, min(rng.choice([1, 2, 4, 8, 24]), 64 * 80 * 64 * 128 // (b * max(copies, -(-beams // 4)) * H * P * N)))
    return dict(op=op, b=b, beams=beams, copies=copies, layers=layers, H=H, P=P, N=N, D=D, padded=rng.choice([0, 0, b // 3]), dtype=dtype)


def _groups(case):
    group = case["group"] or case["K"]
    return group, -(-case["K"] // group)


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *size, dtype=dtype: torch.randn(size, generator=g, device=dev, dtype=dtype)  # noqa: E731
    uniform = lambda lo, hi, *size: torch.rand(size, generator=g, device=dev) * (hi - lo) + lo  # noqa: E731
    whole = lambda lo, hi, *size, dtype=torch.int64: torch.randint(lo, hi, size, generator=g, device=dev, dtype=dtype)  # noqa: E731
    op = case["op"]
    s = dict(case=case, op=op)
    if op == "matmul4":
        M, K, N = (case[k] for k in "MKN")
        s["group"], groups = _groups(case)
        s["a"] = normal(M, K)
        # two weights to a byte, the even one low; a row of odd length ends in half a byte
        s["w"] = whole(0, 256, N, -(-K // 2), dtype=torch.uint8)
        s["w_scale"] = (uniform(0.5, 1.5, N, groups) / (4.6 * K ** 0.5)).to(dtype)
        s["w_zero"] = whole(5, 11, N, groups, dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = normal(N) if case["bias"] else None
    elif op == "block":
        b, L, D = (case[k] for k in "bLD")
        s["x"], s["residual"] = normal(b, L, D), 4 * normal(b, L, D)
        s["weight"] = uniform(0.5, 1.5, D).to(dtype) if case["weight"] else None
        s["next_weight"] = uniform(0.5, 1.5, D).to(dtype)
        s["gate"] = {"none": lambda: None, "channel": lambda: uniform(0.0, 1.0, D).to(dtype), "row": lambda: normal(b, 1, D),
                     "token": lambda: normal(b, L, D)}[case["gate"]]()
    elif op == "select":
        b, beams, V = case["b"], case["beams"], case["V"]
        logits = 2 * normal(b, beams, V, dtype=torch.float32)
        # the tokens that a model finds likely stand out
        logits.scatter_add_(2, whole(0, V, b, beams, 24), uniform(4.0, 12.0, b, beams, 24))
        if case["masked"]:
            logits.masked_fill_(uniform(0.0, 1.0, b, 1, V) < 0.3, float("-inf"))
        s["logits"] = logits.to(dtype)
        s["scores"] = -torch.sort(uniform(1.0, 30.0, b, beams), dim=1)[0]
        s["finished"] = uniform(0.0, 1.0, b, beams) < 0.15 if case["finished"] else None
        s["pad"] = whole(0, V, 1).item()
    else:
        b, beams, copies, padded = (case[k] for k in ("b", "beams", "copies", "padded"))
        slots = b * beams + 3
        s["slots"] = torch.randperm(slots, generator=g, device=dev)[:b * beams].view(b, beams).to(torch.int32)
        s["slots"][b - padded:] = -1
        # the beams that go on, in no order, the first of them twice or more often; their children in no order
        order = torch.rand(b, beams, generator=g, device=dev).argsort(1)
        which = torch.arange(beams, device=dev) % (beams - copies)
        shuffled = torch.rand(b, beams, generator=g, device=dev).argsort(1)
        s["parents"] = order[:, which].gather(1, shuffled).to(torch.int32)
        s["pools"] = []
        for _ in range(case["layers"]):
            s["pools"].append(normal(slots, case["H"], case["P"], case["N"], dtype=torch.float32))
            s["pools"].append(normal(slots, 3, case["D"]).transpose(1, 2))
    return s


def run(s):
    return _own(s) if own else _PLAIN[s["op"]](s)


def _own(s):
    f, op = _framework(), s["op"]
    if op == "matmul4":
        return f._matmul_int4_fwd(s["a"], s["w"], s["w_scale"], s["w_zero"], group=s["group"], bias=s["bias"])
    if op == "block":
        out, scale, residual = f._norm_block_fwd(s["x"], s["weight"], s["residual"], s["next_weight"], gate=s["gate"], residual_scale=s["case"]["scale"],
                                                 eps=1e-5, int8=s["case"]["int8"])
        # 8 bits as the values they stand for, in the type of activations
        return (out if scale is None else _valued(out, scale, s["x"].dtype)), residual
    if op == "select":
        return f._beam_select_fwd(s["logits"], s["scores"], s["case"]["k"], finished=s["finished"], pad=s["pad"])
    return f._beam_reorder(s["parents"], s["slots"], s["pools"]), s["pools"]


def _valued(q, scale, dtype):
    return torch.mul(q, scale[..., None]).to(dtype)


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end; the candidates' scores, which decide an order, in 64

def _plain_matmul4(s):
    a, w, K = s["a"], s["w"], s["a"].shape[1]
    q = torch.stack([w & 15, w >> 4], dim=-1).flatten(1)[:, :K].float()
    spread = lambda t: t.float().repeat_interleave(s["group"], dim=1)[:, :K]  # noqa: E731
    values = (q - (8.0 if s["w_zero"] is None else spread(s["w_zero"]))) * spread(s["w_scale"])
    out = torch.matmul(a.float(), values.t())
    return (out if s["bias"] is None else out + s["bias"].float()).to(a.dtype)


def _plain_block(s):
    x = s["x"]
    n = x.float()
    if s["weight"] is not None:
        n = n * torch.rsqrt((n * n).mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    if s["gate"] is not None:
        n = n * s["gate"].float()
    t = s["case"]["scale"] * s["residual"].float() + n
    u, r = t * s["next_weight"].float(), torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)
    if not s["case"]["int8"]:
        return (u * r).to(x.dtype), t.to(x.dtype)
    most = u.abs().amax(-1, keepdim=True)
    q = torch.round(u * (127 / most)).to(torch.int8)
    return _valued(q, (most * r / 127)[..., 0], x.dtype), t.to(x.dtype)


def _plain_select(s):
    b, beams, V = s["logits"].shape
    logits = s["logits"].double()
    most = logits.amax(-1, keepdim=True)
    c = s["scores"].double()[..., None] + (logits - (torch.log(torch.exp(logits - most).sum(-1, keepdim=True)) + most))
    c = torch.where(torch.isnan(c), float("-inf"), c)
    if s["finished"] is not None:
        ended = torch.where(torch.arange(V, device=c.device) == s["pad"], s["scores"].double()[..., None], float("-inf"))
        c = torch.where(s["finished"][..., None], ended, c)
    c, at = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    c, at = c[:, :s["case"]["k"]], at[:, :s["case"]["k"]]
    return c.float(), torch.div(at, V, rounding_mode="floor").int(), (at % V).int()


def _plain_reorder(s):
    parents, slots, pools = s["parents"].long(), s["slots"].long(), s["pools"]
    beams, n = parents.shape[1], pools[0].shape[0]
    there = (slots >= 0) & (slots < n)
    same = parents[:, :, None] == parents[:, None, :]
    earlier = torch.ones(beams, beams, device=slots.device, dtype=torch.bool).tril(-1)
    alive = torch.gather(there, 1, parents)
    first = alive & ~(same & earlier).any(2)
    again = alive & ~first
    # the slots of beams without a child, in their order, go to the children that are not their parent's first
    childless = there & ~(parents[:, :, None] == torch.arange(beams, device=slots.device)).any(1)
    free = torch.gather(slots, 1, torch.argsort(~childless, dim=1, stable=True, descending=False))
    place = (torch.cumsum(again, 1) - 1).clamp(min=0)
    taken = again & (place < childless.sum(1, keepdim=True))
    source = torch.gather(slots, 1, parents)
    new = torch.where(first, source, torch.where(taken, torch.gather(free, 1, place), -1))
    to, of = new[taken], source[taken]
    copied = [pool.index_copy_(0, to, pool[of]) for pool in pools]
    return new.int(), copied


_PLAIN = {"matmul4": _plain_matmul4, "block": _plain_block, "select": _plain_select, "reorder": _plain_reorder}


def work(case):
    e, op = (4 if case["dtype"] == "fp32" else 2), case["op"]
    if op == "matmul4":
        M, K, N = (case[k] for k in "MKN")
        groups = _groups(case)[1]
        moved = (M * K + M * N + (N if case["bias"] else 0)) * e + N * -(-K // 2) + N * groups * (e + (1 if case["zeros"] else 0))
        return {"bytes": moved, "flops": 2 * M * K * N}
    if op == "block":
        b, L, D = (case[k] for k in "bLD")
        n, small = b * L * D, {"none": 0, "channel": D, "row": b * D, "token": b * L * D}[case["gate"]]
        moved = (3 * n + small + D * (2 if case["weight"] else 1)) * e + n * e
        return {"bytes": moved, "flops": 10 * n}
    if op == "select":
        b, beams, V, k = (case[c] for c in ("b", "beams", "V", "k"))
        # (what finished beams would have said need not be read: they are few, and which is only known at the call)
        return {"bytes": b * beams * V * e + b * beams * 4 + b * k * 12, "flops": 5 * b * beams * V}
    b, beams, copies, padded, H, P, N = (case[c] for c in ("b", "beams", "copies", "padded", "H", "P", "N"))
    slot = case["layers"] * (H * P * N * 4 + case["D"] * 3 * e)
    return {"bytes": (b - padded) * (copies + min(copies, beams - copies)) * slot + b * beams * 12, "flops": b * beams * beams}


# ---- the definitions in 64 bits

def _exact_reorder(s):
    parents, slots = s["parents"].tolist(), s["slots"].tolist()
    pools = [p.clone() for p in s["pools"]]
    n, new = pools[0].shape[0], []
    for row, held in zip(parents, slots):
        free = [held[i] for i in range(len(held)) if 0 <= held[i] < n and i not in row]
        kept, given = set(), []
        for p in row:
            if not 0 <= held[p] < n:
                given.append(-1)
            elif p not in kept:
                kept.add(p)
                given.append(held[p])
            elif free:
                given.append(free.pop(0))
                for pool, old in zip(pools, s["pools"]):
                    pool[given[-1]] = old[held[p]]
            else:
                given.append(-1)
        new.append(given)
    return torch.tensor(new, dtype=torch.int32), pools


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "matmul4":
        K = case["K"]
        at = torch.arange(K, device="cuda")
        q = (s["w"][:, at // 2] >> (4 * (at % 2)).to(torch.uint8)) % 16
        group = at // s["group"]
        zero = torch.full_like(q, 8) if s["w_zero"] is None else s["w_zero"][:, group]
        out = s["a"].double() @ ((q.double() - zero.double()) * s["w_scale"].double()[:, group]).t()
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "block":
        d = lambda t: 1.0 if t is None else t.double()  # noqa: E731
        rms = lambda t: torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
        x = s["x"].double()
        t = case["scale"] * s["residual"].double() + (x / rms(x) * d(s["weight"]) if case["weight"] else x) * d(s["gate"])
        normed = t / rms(t) * d(s["next_weight"])
        if case["int8"]:
            step = normed.abs().amax(-1, keepdim=True) / 127
            normed = torch.round(normed / step) * step
        return normed, t
    if op == "select":
        V, found = case["V"], ([], [], [])
        for i in range(case["b"]):
            rows = s["scores"][i].double()[:, None] + torch.log_softmax(s["logits"][i].double(), dim=-1)
            if s["finished"] is not None:
                for j in torch.nonzero(s["finished"][i]).flatten().tolist():
                    rows[j] = float("-inf")
                    rows[j, s["pad"]] = s["scores"][i, j].double()
            rows = rows.flatten()
            # all that reach the k-th largest, then the order of indices among equals
            least = torch.topk(rows, case["k"])[0][-1]
            at = torch.nonzero(rows >= least).flatten()
            at = at[torch.argsort(rows[at], descending=True, stable=True)][:case["k"]]
            for to, v in zip(found, (rows[at], at // V, at % V)):
                to.append(v)
        score, parents, tokens = (torch.stack(v) for v in found)
        return score, parents.int(), tokens.int()
    new, pools = _exact_reorder(s)
    return new, [p.double() for p in pools]
