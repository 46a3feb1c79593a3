"""Calls of the operators of a decoding step at the ends of what they take: tokens forbidden by large finite logits, sizes whose
launches need more than one dimension, gates of another type than the rows.  Against oracle/decode_oracle.py, or the formula itself.

Bounds are those of test_gpu_decode.py.  Sums relative to a far logit m have exponents (v - m) log2(e): v - m is exact where a term is not zero, log2(e) in fp32 and
the product are off by 2^-24 of d = m - v each, and 2 d e^-d < 1: 2^-22 + 2^-23 + 32 2^-24 < 2.5e-6, as for the others."""
import pytest
import torch

from test_gpu_decode import INF, LSE, block_bounds, ops, ref  # noqa: F401  (fixtures)
from test_gpu_layer import TYPES, close, gpu, randn, rounded

pytestmark = pytest.mark.gpu

V, PART = 20001, 8192
KINDS = ["a part", "the short last part", "all but a part", "a few left", "a beam", "a beam and a part of the others", "everything"]


def finite_masks(dtype):
    low = torch.finfo(dtype).min
    return [low, -1e4] if dtype == torch.float16 else [low, -1e4, -2e6, -1e9, -3e9, -1e10, -1e12, -1e20, -1e30, -1e38]


def masked_logits(dtype, value, kind):
    """(2, 3, V) logits with tokens forbidden by `value`"""
    g = torch.Generator().manual_seed(KINDS.index(kind))
    logits = 2 * torch.randn(2, 3, V, generator=g)
    at = torch.arange(V)
    if kind == "a part":
        where = (at >= PART) & (at < 2 * PART)
    elif kind == "the short last part":
        where = at >= V // PART * PART
    elif kind == "all but a part":
        where = (at < PART) | (at >= 2 * PART)
    elif kind == "a few left":
        where = (at < PART + 100) | (at >= PART + 107)
    else:
        where = at >= 0
    where = where.expand(2, 3, V).clone()
    if kind == "a beam":
        where[:, (0, 2)] = False
    elif kind == "a beam and a part of the others":
        where[:, (0, 2), :PART] = False
    return logits.masked_fill(where, value).to(dtype), -torch.tensor([[2.0, 7.5, 4.0], [9.0, 1.0, 4.5]]) - torch.rand(2, 3, generator=g)


def wanted(ref, logits, scores, k, finished, pad):
    """The oracle's, for inputs whose candidates of different beams are farther apart than the error of a score and of its 64 bits."""
    want, parents, tokens, _ = ref.beam_select_ref(logits, scores, k + 1, finished, pad)
    gap = want[:, :-1] - want[:, 1:]
    known = (gap > 0) & torch.isfinite(gap) & (parents[:, :-1] != parents[:, 1:])
    assert bool((gap > 2 * LSE + 2.0 ** -50 * want[:, 1:].abs())[known].all()), gap
    return want[:, :k], parents[:, :k], tokens[:, :k]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_beam_selection_with_tokens_forbidden_by_large_finite_logits(ops, ref, dtype, kind):  # noqa: F811
    # every logit is a number: a beam has the scores of its formula however small they are, and its other tokens theirs
    for value in finite_masks(dtype):
        logits, scores = masked_logits(dtype, value, kind)
        for k, finished, pad in ((3, None, 0), (40, None, 0), (6, torch.tensor([[False, False, True], [True, False, False]]), V - 1)):
            want, parents, tokens = wanted(ref, logits, scores, k, finished, pad)
            got = ops._beam_select_fwd(gpu(logits), gpu(scores), k, finished=gpu(finished), pad=pad)
            what = f"{value} {k}"
            assert torch.equal(got[1].cpu().long(), parents) and torch.equal(got[2].cpu().long(), tokens), what
            # (what fp32 does not hold is an infinity there)
            none = want.float() == -INF
            assert torch.equal(got[0].cpu() == -INF, none), what
            want = torch.where(none, 0.0, want)
            close(torch.where(none.cuda(), 0.0, got[0]), want, LSE + rounded(want, torch.float32), what)


@pytest.mark.parametrize("vocab", [5, 8192, 8193, 30000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_beam_selection_among_large_logits(ops, ref, dtype, vocab):  # noqa: F811
    # beams of one value, and one large logit among ordinary ones: log-probabilities of -log(vocab) and of 0
    g = torch.Generator().manual_seed(vocab)
    scores = -torch.tensor([[1.0, 3.0, 2.0]])
    for value in [-v for v in finite_masks(dtype)] + finite_masks(dtype):
        logits = torch.full((1, 3, vocab), value).to(dtype)
        want, parents, tokens = wanted(ref, logits, scores, 4, None, 0)
        assert abs(float(want[0, 0]) + 1 + float(torch.log(torch.tensor(float(vocab))))) < 1e-5
        got = ops._beam_select_fwd(gpu(logits), gpu(scores), 4)
        assert torch.equal(got[1].cpu().long(), parents) and torch.equal(got[2].cpu().long(), tokens), value
        close(got[0], want, LSE + rounded(want, torch.float32), str(value))
        if value > 0:
            logits = torch.randn(1, 3, vocab, generator=g)
            logits[:, :, vocab // 2] = value
            logits = logits.to(dtype)
            got = ops._beam_select_fwd(gpu(logits), gpu(scores), 3)
            assert got[1].tolist() == [[0, 2, 1]] and got[2].tolist() == [[vocab // 2] * 3], value
            close(got[0], torch.tensor([[-1.0, -2.0, -3.0]], dtype=torch.float64), torch.full((1, 3), LSE, dtype=torch.float64), str(value))


def test_beam_selection_of_more_rows_than_a_launch_has_in_one_dimension(ops):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(2)
    b = (1 << 24) + 5
    logits = torch.randint(-4, 5, (b, 1, 2), generator=g, dtype=torch.int8, device="cuda").bfloat16()
    scores = -torch.rand(b, 1, generator=g, device="cuda")
    best, parents, tokens = ops._beam_select_fwd(logits, scores)
    less = logits.amin(2) - logits.amax(2)
    want = scores.double() - torch.log1p(torch.exp(less.double()))
    assert not bool(parents.any()) and torch.equal(tokens[:, 0], (logits[:, 0, 1] > logits[:, 0, 0]).int())
    assert bool(((best.double() - want).abs() <= LSE + rounded(want, torch.float32)).all())


@pytest.mark.parametrize("int8", [False, True])
def test_a_gate_of_fp32_does_not_make_the_residual_fp32_in_a_single_row(ops, ref, int8):  # noqa: F811
    # a gate per channel or per row of a batch: t has the type of x and the residual, with one row as with several
    g = torch.Generator().manual_seed(7)
    for D in (7, 520, 2560):
        x, residual, weight = randn(g, 3, D, dtype=torch.bfloat16), randn(g, 3, D, dtype=torch.bfloat16), randn(g, D, dtype=torch.bfloat16)
        gate = randn(g, D)
        on, gated = [gpu(t) for t in (x, weight, residual)], gpu(gate)

        def call(rows, shape, gate):
            out, scale, total = ops._norm_block_fwd(on[0][:rows].reshape(shape), on[1], on[2][:rows].reshape(shape), on[1], gate=gate, int8=int8)
            assert total.dtype == torch.bfloat16 and out.dtype == (torch.int8 if int8 else torch.bfloat16) and out.shape == total.shape == torch.Size(shape)
            return [t for t in (out.reshape(rows, D), total.reshape(rows, D), None if scale is None else scale.reshape(rows)) if t is not None]

        many = call(3, (3, D), gated)
        want, t, n = ref.norm_block_ref(x, weight, residual, weight, gate)
        close(many[1], t, block_bounds(x, weight, residual, weight, gate, 1.0, want, t, n, torch.bfloat16)[0], "residual")
        for shape, of in (((D,), (D,)), ((1, D), (D,)), ((1, 1, D), (D,)), ((1, 1, D), (1, D))):
            assert all(torch.equal(one[0], some[0]) for one, some in zip(call(1, shape, gated.view(of)), many))
        # a gate of the rows' own shape is one per token, and part of what t has to hold
        total = ops._norm_block_fwd(on[0], on[1], on[2], on[1], gate=gated.expand(3, D).contiguous())[2]
        assert total.dtype == torch.float32


def test_product_of_more_channels_or_tokens_than_a_launch_has_in_one_dimension(ops):  # noqa: F811
    # whole numbers, of which every sum is exact in bf16
    g = torch.Generator(device="cuda").manual_seed(1)
    N, chunk = (1 << 28) + 37, 1 << 26
    w = torch.randint(0, 256, (N, 1), generator=g, dtype=torch.uint8, device="cuda")
    scale = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    got = ops._matmul_int4_fwd(torch.tensor([[3.0, -5.0]], device="cuda").bfloat16(), w, scale.expand(N, 1), group=32)
    for at in range(0, N, chunk):
        part = w[at:at + chunk, 0].int()
        assert torch.equal(got[0, at:at + chunk].int(), 3 * (part % 16 - 8) - 5 * (part // 16 - 8))
    del w, got
    M = (1 << 29) + 33
    w = torch.tensor([[0x2f], [0x80], [0xc1]], dtype=torch.uint8, device="cuda")
    a = torch.empty(M, 2, dtype=torch.bfloat16, device="cuda")
    for at in range(0, M, chunk):
        a[at:at + chunk] = torch.randint(-7, 8, a[at:at + chunk].shape, generator=g, dtype=torch.int8, device="cuda")
    got = ops._matmul_int4_fwd(a, w, scale.expand(3, 1), group=32)
    for at in range(0, M, chunk):
        part = a[at:at + chunk].int()
        for n, (even, odd) in enumerate(((7, -6), (-8, 0), (-7, 4))):
            assert torch.equal(got[at:at + chunk, n].int(), even * part[:, 0] + odd * part[:, 1])


def test_norms_of_more_long_rows_than_a_launch_has_workgroups(ops):  # noqa: F811
    # rows of sixteen waves: all read the same ones, and leave their results in one place but for their scales
    from ssd_amd import _lib
    from ssd_amd.layer import _arg
    g = torch.Generator().manual_seed(3)
    rows, D = (1 << 22) + 3, 12296
    x, residual, weight = (gpu(randn(g, n, D, dtype=torch.bfloat16)) for n in (1, 1, 1))
    want, scale, total = ops._norm_block_fwd(x, weight[0], residual, weight[0], int8=True)
    got, sums = torch.zeros_like(want), torch.zeros_like(total)
    scales = torch.full((rows,), -1.0, device="cuda")
    torch.cuda.synchronize()
    each = lambda t: _arg(t.expand(rows, D))  # noqa: E731
    _lib.check(_lib.load().ssd_norm_block_fwd(each(x), _arg(weight[0]), each(residual), _arg(weight[0]), _arg(None), each(got), _arg(scales), each(sums),
                                              rows, D, 1, 1.0, 1e-5, torch.cuda.current_stream().cuda_stream), "ssd_norm_block_fwd")
    assert bool((scales == scale).all()) and torch.equal(got, want) and torch.equal(sums, total)
