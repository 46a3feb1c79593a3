"""A Mamba2 layer as it is served: weights of both projections in 8 bits, prompts of different length in one batch, then single tokens of
the rows that are still running, their states in a pool.

    norm (with the residual's addition, 8 bits) -> product -> short convolution -> selective scan -> gated norm (8 bits) -> product

The gated norm is over all inner channels of a token, whatever the number of groups of B and C: a layer whose gated norm takes its mean over
the channels of each group is another one.

python3 mamba-fused-minimal_amd/examples/served_layer.py     times a layer of width 2560 on random weights."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import ssd_amd as ops  # noqa: E402


def eight_bits(w):
    """A projection (channels, K) as 8-bit integers and a scale per channel; done once, when the weights are loaded."""
    scale = w.float().abs().amax(1).clamp(min=1e-30) / 127
    return torch.round(w.float() / scale[:, None]).to(torch.int8), scale


class ServedLayer:
    """in_proj (2 d + 2 ngroups dstate + nheads, width) with rows z, x, B, C, dt (d = nheads headdim); conv_weight (d + 2 ngroups dstate,
    taps); A, dt_bias, D (nheads); norm_weight (width), gate_weight (d); out_proj (width, d)."""

    def __init__(self, in_proj, out_proj, conv_weight, conv_bias, A, dt_bias, D, norm_weight, gate_weight, headdim, dstate, ngroups=1, slots=64):
        self.nheads, self.headdim, self.dstate, self.ngroups = A.shape[0], headdim, dstate, ngroups
        self.inner = self.nheads * headdim
        self.in_proj, self.out_proj = eight_bits(in_proj), eight_bits(out_proj)
        self.conv_weight, self.conv_bias, self.A, self.dt_bias, self.D = conv_weight, conv_bias, A, dt_bias, D
        self.norm_weight, self.gate_weight, self.dtype = norm_weight, gate_weight, conv_weight.dtype
        mixed, taps = conv_weight.shape
        # the pool: a slot per running sequence
        self.conv_states = torch.zeros((slots, taps - 1, mixed), device=A.device, dtype=self.dtype).transpose(1, 2)
        self.states = torch.zeros((slots, self.nheads, headdim, dstate), device=A.device)

    def _enter(self, hidden, residual):
        normed, scale, residual = ops._norm_fwd(hidden, self.norm_weight, residual=residual, int8=True)
        z, mixed, dt = ops._matmul_int8_fwd(normed, scale, *self.in_proj, out_dtype=self.dtype).split(
            [self.inner, self.conv_weight.shape[0], self.nheads], dim=-1)
        return z, mixed, dt, residual

    def _parts(self, mixed):
        x, B, C = mixed.split([self.inner] + 2 * [self.ngroups * self.dstate], dim=-1)
        return x.unflatten(-1, (self.nheads, self.headdim)), B.unflatten(-1, (self.ngroups, -1)), C.unflatten(-1, (self.ngroups, -1))

    def _leave(self, y, z):
        gated, scale, _ = ops._norm_fwd(y.flatten(-2), self.gate_weight, z=z, int8=True)
        return ops._matmul_int8_fwd(gated, scale, *self.out_proj, out_dtype=self.dtype)

    def prompt(self, hidden, residual, slots, lengths=None, resume=False):
        """hidden and residual (batch, tokens, width) -> the same; row b's states go to slot slots[b] of the pool (and, to resume, come from it).
        lengths (batch): tokens of each row; what is behind them is of no meaning."""
        z, mixed, dt, residual = self._enter(hidden, residual)
        at = slots.long()
        mixed, conv_states = ops._short_conv_fwd(mixed, self.conv_weight, self.conv_bias, initial_states=self.conv_states[at] if resume else None,
                                                 lengths=lengths)
        x, B, C = self._parts(mixed)
        y, states = ops._ssd_scan_fwd(x, dt, self.A, B, C, D=self.D, dt_bias=self.dt_bias, dt_softplus=True,
                                      initial_states=self.states[at] if resume else None, lengths=lengths)
        self.conv_states[at], self.states[at] = conv_states, states
        return self._leave(y, z), residual

    def step(self, hidden, residual, slots):
        """One token of every row: hidden and residual (batch, width).  A slot outside the pool is padding."""
        z, mixed, dt, residual = self._enter(hidden, residual)
        mixed = ops._short_conv_step(mixed, self.conv_states, self.conv_weight, self.conv_bias, slots=slots)
        x, B, C = self._parts(mixed)
        y = ops._ssd_scan_step(x, dt, self.A, B, C, self.states, D=self.D, dt_bias=self.dt_bias, dt_softplus=True, slots=slots)
        return self._leave(y, z), residual


def random_layer(width, nheads, headdim, dstate, ngroups=1, taps=4, slots=64, dtype=torch.bfloat16, device="cuda", seed=0):
    g = torch.Generator().manual_seed(seed)
    inner = nheads * headdim
    mixed = inner + 2 * ngroups * dstate
    randn = lambda *size: torch.randn(*size, generator=g)  # noqa: E731
    w = dict(in_proj=randn(inner + mixed + nheads, width) * width ** -0.5, out_proj=randn(width, inner) * inner ** -0.5,
             conv_weight=(randn(mixed, taps) * taps ** -0.5).to(dtype), conv_bias=(0.1 * randn(mixed)).to(dtype),
             A=-1 - 15 * torch.rand(nheads, generator=g), dt_bias=torch.log(torch.expm1(torch.exp(-6.9 + 4.6 * torch.rand(nheads, generator=g)))),
             D=torch.ones(nheads), norm_weight=(1 + 0.1 * randn(width)).to(dtype), gate_weight=(1 + 0.1 * randn(inner)).to(dtype))
    return ServedLayer(**{k: v.to(device) for k, v in w.items()}, headdim=headdim, dstate=dstate, ngroups=ngroups, slots=slots)


def main():
    layer = random_layer(2560, 80, 64, 128)
    slots = torch.arange(8, device="cuda", dtype=torch.int32)
    lengths = torch.tensor([4096, 4000, 3500, 3000, 2048, 2000, 1000, 1], device="cuda", dtype=torch.int32)
    hidden = torch.randn(8, 4096, 2560, device="cuda").bfloat16()
    many = torch.arange(64, device="cuda", dtype=torch.int32)
    token = torch.randn(64, 2560, device="cuda").bfloat16()

    def timed(what, f, n):
        f()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(n):
            f()
        end.record()
        end.synchronize()
        print(f"{what}: {begin.elapsed_time(end) / n * 1e3:.0f} us")

    timed("8 prompts, 4096 tokens at most", lambda: layer.prompt(hidden, hidden, slots, lengths), 20)
    timed("a token of 64 rows", lambda: layer.step(token, token, many), 100)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(token, token, many)
    timed("the same from a graph", graph.replay, 100)


if __name__ == "__main__":
    main()
