"""Beam search over a model of Mamba2 layers as it is served: weights of all projections in 4 bits, the states of all beams in pools.

    norm -> [product -> short convolution -> selective scan -> gated norm -> product -> norms between the blocks] per layer -> product (logits)
    -> selection -> states follow their beams

python3 mamba-fused-minimal_amd/examples/beam_search.py     times a step of eight rows of four beams, four layers of width 2560 on random weights."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import ssd_amd as ops  # noqa: E402


def four_bits(w, group=128):
    """A projection (channels, K) as 4-bit weights, two to a byte, with a scale and a zero point per group; done once, when the weights are loaded."""
    channels, K = w.shape
    groups = torch.nn.functional.pad(w.float(), (0, -K % group)).unflatten(1, (-1, group))
    low, high = groups.amin(-1).clamp(max=0), groups.amax(-1).clamp(min=0)
    scale = ((high - low) / 15).clamp(min=1e-30)
    zero = torch.round(-low / scale)
    q = torch.clamp(torch.round(groups / scale[..., None]) + zero[..., None], 0, 15).to(torch.uint8).flatten(1)[:, :K]
    q = torch.nn.functional.pad(q, (0, K % 2))
    return q[:, 0::2] | q[:, 1::2] << 4, scale, zero.to(torch.uint8)


class Layer:
    """A block's weights, of the shapes that ServedLayer (served_layer.py) has them in, and its pools of states."""

    def __init__(self, in_proj, out_proj, conv_weight, conv_bias, A, dt_bias, D, gate_weight, headdim, dstate, slots, group):
        self.nheads, self.headdim, self.dstate, self.group = A.shape[0], headdim, dstate, group
        self.inner = self.nheads * headdim
        self.in_proj, self.out_proj = four_bits(in_proj, group), four_bits(out_proj, group)
        self.conv_weight, self.conv_bias, self.A, self.dt_bias, self.D, self.gate_weight = conv_weight, conv_bias, A, dt_bias, D, gate_weight
        mixed, taps = conv_weight.shape
        self.conv_states = torch.zeros((slots, taps - 1, mixed), device=A.device, dtype=conv_weight.dtype).transpose(1, 2)
        self.states = torch.zeros((slots, self.nheads, headdim, dstate), device=A.device)

    def _enter(self, u):
        return ops._matmul_int4_fwd(u, *self.in_proj, group=self.group).split([self.inner, self.conv_weight.shape[0], self.nheads], dim=-1)

    def _parts(self, mixed):
        x, B, C = mixed.split([self.inner, self.dstate, self.dstate], dim=-1)
        return x.unflatten(-1, (self.nheads, self.headdim)), B.unsqueeze(-2), C.unsqueeze(-2)

    def _leave(self, y, z):
        return ops._matmul_int4_fwd(ops._norm_fwd(y.flatten(-2), self.gate_weight, z=z)[0], *self.out_proj, group=self.group)

    def prompt(self, u, slots, lengths):
        z, mixed, dt = self._enter(u)
        mixed, conv_states = ops._short_conv_fwd(mixed, self.conv_weight, self.conv_bias, lengths=lengths)
        x, B, C = self._parts(mixed)
        y, states = ops._ssd_scan_fwd(x, dt, self.A, B, C, D=self.D, dt_bias=self.dt_bias, dt_softplus=True, lengths=lengths)
        self.conv_states[slots.long()], self.states[slots.long()] = conv_states, states
        return self._leave(y, z)

    def step(self, u, slots):
        z, mixed, dt = self._enter(u)
        mixed = ops._short_conv_step(mixed, self.conv_states, self.conv_weight, self.conv_bias, slots=slots)
        x, B, C = self._parts(mixed)
        return self._leave(ops._ssd_scan_step(x, dt, self.A, B, C, self.states, D=self.D, dt_bias=self.dt_bias, dt_softplus=True, slots=slots), z)


class Model:
    """embedding (vocab, width); layers; norms (layers + 1, width): in front of each block and of the head; behind and gates (layers, width): the
    norm behind a block and its gate; factor: the residual's scale; head (vocab, width)."""

    def __init__(self, embedding, layers, norms, behind, gates, factor, head, group=128):
        self.embedding, self.layers, self.norms, self.behind, self.gates, self.factor, self.group = embedding, layers, norms, behind, gates, factor, group
        self.head = four_bits(head, group)
        self.pools = [pool for layer in layers for pool in (layer.states, layer.conv_states)]

    def _run(self, tokens, blocks):
        t = self.embedding[tokens]
        u = ops._norm_fwd(t, self.norms[0])[0]
        for i, block in enumerate(blocks):
            u, _, t = ops._norm_block_fwd(block(u), self.behind[i], t, self.norms[i + 1], gate=self.gates[i], residual_scale=self.factor)
        return u

    def prompt(self, tokens, lengths, slots):
        """tokens (batch, longest), of which lengths (batch) are there -> logits of each row's last (batch, vocab); its states go to slots (batch)."""
        u = self._run(tokens, [lambda u, layer=layer: layer.prompt(u, slots, lengths) for layer in self.layers])
        last = u[torch.arange(len(tokens), device=u.device), lengths.long() - 1]
        return ops._matmul_int4_fwd(last, *self.head, group=self.group)

    def step(self, tokens, slots):
        """A token of every beam, (batch, beams) -> logits (batch, beams, vocab)."""
        u = self._run(tokens.flatten().long(), [lambda u, layer=layer: layer.step(u, slots.flatten()) for layer in self.layers])
        return ops._matmul_int4_fwd(u, *self.head, group=self.group).unflatten(0, tokens.shape)


class Search:
    """A running search: scores, slots, tokens and whether they have ended, (batch, beams) each, kept in place so that a step can be a graph."""

    def __init__(self, model, tokens, lengths, beams, end):
        self.model, self.beams, self.end = model, beams, end
        batch, device = len(tokens), tokens.device
        first = torch.arange(batch * beams, device=device, dtype=torch.int32).view(batch, beams)
        logits = model.prompt(tokens, lengths, first[:, 0])
        # one beam is there; the others' states are its own, copied
        scores = torch.full((batch, beams), -float("inf"), device=device)
        scores[:, 0] = 0
        self.scores, parents, self.tokens = ops._beam_select_fwd(logits[:, None].expand(-1, beams, -1), scores)
        self.slots = ops._beam_reorder(parents, first, model.pools)
        self.finished = self.tokens == end
        self.parents = parents
        self.history = [(parents.clone(), self.tokens.clone())]

    def advance(self):
        """One step, into the same tensors."""
        logits = self.model.step(self.tokens, self.slots)
        scores, parents, tokens = ops._beam_select_fwd(logits, self.scores, finished=self.finished, pad=self.end)
        slots = ops._beam_reorder(parents, self.slots, self.model.pools)
        self.finished.copy_(tokens == self.end)      # (a beam that has ended goes on with that token)
        for to, value in ((self.scores, scores), (self.parents, parents), (self.tokens, tokens), (self.slots, slots)):
            to.copy_(value)

    def run(self, steps, graph=False):
        advance = self.advance
        if graph:
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                self.advance()
            advance = captured.replay
        for _ in range(steps):
            advance()
            self.history.append((self.parents.clone(), self.tokens.clone()))
        return self.sequences(), self.scores

    def sequences(self):
        """(batch, beams, steps): what each beam has said, best first."""
        at = torch.arange(self.beams, device=self.tokens.device).expand_as(self.tokens)
        said = []
        for parents, tokens in reversed(self.history):
            said.append(tokens.gather(1, at))
            at = parents.gather(1, at).long()
        return torch.stack(said[::-1], -1)


def random_model(vocab, width, nheads, headdim, dstate, layers, slots, taps=4, group=128, dtype=torch.bfloat16, device="cuda", seed=0):
    g = torch.Generator().manual_seed(seed)
    inner = nheads * headdim
    mixed = inner + 2 * dstate
    randn = lambda *size: torch.randn(*size, generator=g)  # noqa: E731
    near_one = lambda *size: (1 + 0.1 * randn(*size)).to(dtype).to(device)  # noqa: E731

    def layer():
        w = dict(in_proj=randn(inner + mixed + nheads, width) * width ** -0.5, out_proj=randn(width, inner) * inner ** -0.5,
                 conv_weight=(randn(mixed, taps) * taps ** -0.5).to(dtype), conv_bias=(0.1 * randn(mixed)).to(dtype), A=-1 - 15 * torch.rand(nheads, generator=g),
                 dt_bias=torch.log(torch.expm1(torch.exp(-6.9 + 4.6 * torch.rand(nheads, generator=g)))), D=torch.ones(nheads))
        return Layer(**{k: v.to(device) for k, v in w.items()}, gate_weight=near_one(inner), headdim=headdim, dstate=dstate, slots=slots, group=group)

    return Model(randn(vocab, width).to(dtype).to(device), [layer() for _ in range(layers)], near_one(layers + 1, width), near_one(layers, width),
                 near_one(layers, width), 0.8, (2 * randn(vocab, width) * width ** -0.5).to(device), group)


def main():
    model = random_model(50000, 2560, 80, 64, 128, 4, slots=32)
    tokens = torch.randint(0, 50000, (8, 512), device="cuda")
    lengths = torch.tensor([512, 500, 400, 300, 200, 100, 10, 1], device="cuda", dtype=torch.int32)
    for graph in (False, True):
        search = Search(model, tokens, lengths, 4, end=2)
        search.run(2)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        advance = search.advance
        if graph:
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                search.advance()
            advance = captured.replay
        begin.record()
        for _ in range(50):
            advance()
        end.record()
        end.synchronize()
        print(f"a step of 8 x 4 beams{' from a graph' if graph else ''}: {begin.elapsed_time(end) / 50 * 1e3:.0f} us")


if __name__ == "__main__":
    main()
