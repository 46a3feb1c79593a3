"""The operators of a served Mamba2 layer together (examples/served_layer.py) against the layer in 64 bits."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def example():
    path = os.path.join(HERE, "..", "mamba-fused-minimal_amd", "examples", "served_layer.py")
    spec = importlib.util.spec_from_file_location("served_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def layer64(m, hidden, residual):
    """One row (tokens, width) in 64 bits, with the weights of the 8-bit projections and no rounding between."""
    f = lambda t: t.double().cpu()  # noqa: E731
    weights = [f(q) * f(s)[:, None] for q, s in (m.in_proj, m.out_proj)]
    t = f(hidden) + f(residual)
    rms = lambda t, w: t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) * f(w)  # noqa: E731
    z, mixed, dt = (rms(t, m.norm_weight) @ weights[0].T).split([m.inner, m.conv_weight.shape[0], m.nheads], dim=-1)
    K, L = m.conv_weight.shape[1], t.shape[0]
    front = torch.cat([torch.zeros(K - 1, mixed.shape[1], dtype=torch.float64), mixed])
    mixed = torch.nn.functional.silu(sum(front[k:k + L] * f(m.conv_weight)[:, k] for k in range(K)) + f(m.conv_bias))
    x, B, C = mixed.split([m.inner] + 2 * [m.ngroups * m.dstate], dim=-1)
    x = x.unflatten(-1, (m.nheads, m.headdim))
    B, C = (v.unflatten(-1, (m.ngroups, m.dstate)).repeat_interleave(m.nheads // m.ngroups, dim=1) for v in (B, C))
    d = torch.nn.functional.softplus(dt + f(m.dt_bias))
    h, y = torch.zeros(m.nheads, m.headdim, m.dstate, dtype=torch.float64), []
    for i in range(L):
        h = h * torch.exp(d[i] * f(m.A))[:, None, None] + (d[i][:, None] * x[i])[..., None] * B[i][:, None]
        y.append((h * C[i][:, None]).sum(-1) + f(m.D)[:, None] * x[i])
    gated = torch.stack(y).flatten(1) * torch.nn.functional.silu(z)
    return rms(gated, m.gate_weight) @ weights[1].T, t, h


# What the roundings to 8 bits may do: a rounding moves a value by up to half of 1/127 of its row's largest, 1/(127 sqrt(12)) of that in the
# mean; with a largest of 4 (normed rows) and 8 (gated rows) root mean squares 0.9% and 1.8% of the row.  The first passes through the
# convolution into x, B, C and dt, whose product doubles or triples it; bf16 adds 0.2% per operator: 0.9 * 3 + 1.8 + 1 = 5.5% at most.
NEAR = 0.06


@pytest.mark.parametrize("shape", [(256, 8, 64, 128, 1), (96, 6, 32, 64, 2), (64, 4, 48, 16, 1)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prompts_then_single_tokens(example, shape, dtype):
    width, nheads, headdim, dstate, ngroups = shape
    m = example.random_layer(width, nheads, headdim, dstate, ngroups, slots=7, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    lengths, steps, L = [70, 1, 33], 4, 70
    hidden, residual = (torch.randn(3, L + steps, width, generator=g).to(dtype).cuda() for _ in range(2))
    slots = torch.tensor([5, 0, 3], dtype=torch.int32).cuda()
    y, total = m.prompt(hidden[:, :L], residual[:, :L], slots, torch.tensor(lengths, dtype=torch.int32).cuda())
    outs = []
    for i in range(steps):
        # row b's next token; the middle row pauses once, as padding
        at = torch.tensor([n + i for n in lengths]).cuda()
        rows = torch.arange(3).cuda()
        now = slots.clone()
        if i == 2:
            now[1] = -1
        outs.append(m.step(hidden[rows, at], residual[rows, at], now)[0])
    for b, n in enumerate(lengths):
        want, t, h = layer64(m, hidden[b, :n + steps], residual[b, :n + steps])
        close = lambda got, want: float((got.double().cpu() - want).norm()) <= NEAR * float(want.norm())  # noqa: E731
        assert close(y[b, :n], want[:n])
        unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
        assert float((total[b, :n].double().cpu() - t[:n]).abs().max()) <= unit * float(t.abs().max())
        if b != 1:
            assert close(torch.stack([o[b] for o in outs]), want[n:]) and close(m.states[slots[b]], h)
        else:
            assert close(torch.stack([o[b] for o in outs[:2]]), want[n:n + 2])
    untouched = [s for s in range(7) if s not in slots.tolist()]
    assert not bool(m.states[untouched].any()) and not bool(m.conv_states[untouched].any())


def test_a_prompt_in_two_parts_and_a_step_from_a_graph(example):
    m = example.random_layer(256, 8, 64, 128, slots=4)
    g = torch.Generator().manual_seed(2)
    hidden, residual = (torch.randn(2, 200, 256, generator=g).bfloat16().cuda() for _ in range(2))
    slots = torch.tensor([2, 1], dtype=torch.int32).cuda()
    whole, _ = m.prompt(hidden, residual, slots)
    states = m.states.clone()
    first, _ = m.prompt(hidden[:, :77], residual[:, :77], slots)
    second, _ = m.prompt(hidden[:, 77:], residual[:, 77:], slots, resume=True)
    got = torch.cat([first, second], 1).double()
    # the parts end in other chunks: sums in another order, seen through one rounding to bf16 and now and then a neighbour in 8 bits
    assert float((got - whole.double()).norm()) <= 0.01 * float(whole.double().norm())
    assert float((m.states - states).norm()) <= 1e-4 * float(states.norm())
    token, more = hidden[:, 0].contiguous(), residual[:, 0].contiguous()
    saved = m.states.clone(), m.conv_states.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        m.step(token, more, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = m.step(token, more, slots)
    for _ in range(3):
        m.states.copy_(saved[0])
        m.conv_states.copy_(saved[1])
        want, _ = m.step(token, more, slots)
        after = m.states.clone()
        m.states.copy_(saved[0])
        m.conv_states.copy_(saved[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(m.states, after)
