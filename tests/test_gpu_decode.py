"""The operators of a decoding step -- product with 4-bit weights, norms around a block, beam selection, reordering of states -- against
their restatement in 64 bits (oracle/decode_oracle.py).

Bounds.  A result is rounded once to its type: half a unit, 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32) of its size.  In front of that:
  product   its terms are exact; a matrix instruction adds 32 of them, every addition off by a unit (2^-23) of a sum that is at most the
            block's sum over absolute values, and the K / 32 blocks are added in chains, over at most 32 waves and parts:
            (64 + K / 32 + 32) 2^-23 of the sum over absolute values; a scale and a bias are one operation more.
  norms     a mean of squares of D elements, in chains of D / 64 and a tree: (D / 64 + 16) 2^-24 of itself, its root half of that, the
            reciprocal root 2^-22; every product and sum behind it 2^-24 of itself.
  scores    an exponential is off by 2^-22 and its argument's rounding (2^-24 of d, and d e^-d < 1/2), a thread adds 32 of them in fp32:
            the logarithm of the sum is off by at most 2^-22 + 2^-24 + 32 2^-24 < 2.5e-6, and so is a score in front of its rounding."""
import pytest
import torch

from test_gpu_layer import TYPES, U, close, gpu, randn, rounded

pytestmark = pytest.mark.gpu
INF = float("inf")
LSE = 2.5e-6


@pytest.fixture(scope="module")
def ops():
    import ssd_amd
    from ssd_amd import _lib
    _lib.load()
    return ssd_amd


@pytest.fixture(scope="module")
def ref():
    import importlib
    return importlib.import_module("oracle.decode_oracle")


# ---- product with 4-bit weights ----------------------------------------------------------------------------------------

def weights_of(g, N, K, group, dtype, zeros):
    groups = -(-K // group)
    w = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    scale = ((0.5 + torch.rand(N, groups, generator=g)) / (4.6 * K ** 0.5)).to(dtype)
    return w, scale, torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None


def product_bound(want, size, K, out_dtype, bias=None):
    inner = (64 + K / 32 + 32) * 2.0 ** -23 * size + 2.0 ** -23 * (want.abs() + (0 if bias is None else bias.double().abs()))
    return rounded(want, out_dtype) + inner * (1 + U[out_dtype])


SIZES = [(1, 16, 64, 32), (1, 1, 1, 32), (2, 3, 2, 64), (1, 130, 31, 128), (5, 17, 33, 32), (16, 64, 128, 128), (17, 33, 160, 32), (64, 48, 96, 96), (65, 100, 257, 64),
         (3, 40, 1000, 1000), (1, 64, 2560, 128), (9, 31, 1543, 64), (128, 256, 512, 128), (130, 200, 320, 64), (257, 300, 384, 32), (300, 130, 130, 32),
         (513, 256, 640, 160), (40, 512, 1024, 128), (100, 77, 129, 128),
         # tiles of 64 x 64 and 256 x 128, K whole and shared out: groups of whole steps, of half steps, one group, lengths off 8
         (2048, 2050, 192, 128), (2000, 2040, 160, 32), (4100, 2047, 136, 200), (4090, 2056, 256, 64), (4097, 2048, 203, 64), (1500, 1030, 1032, 128),
         (1100, 1500, 1024, 64), (1500, 1030, 1032, 32), (2100, 2100, 520, 128), (300, 1100, 2048, 128), (96, 700, 4100, 64), (96, 700, 4099, 32),
         (96, 700, 4104, 4104), (512, 2560, 2568, 128), (512, 2560, 2570, 64), (512, 2500, 2600, 32), (512, 2500, 2601, 2601),
         # halves of a workgroup, with tables that are asked for again, ends in the first half, and more tiles than halves have room for
         (64, 2560, 9000, 32), (60, 10400, 2568, 32), (200, 4090, 1021, 64), (200, 4090, 1032, 1032), (33, 2560, 5120, 128), (60, 16400, 1000, 32),
         (64, 16400, 1032, 128), (70, 10400, 2568, 32), (130, 10571, 1032, 64),
         # two and four times sixteen channels to a workgroup, scales beside each other and not
         (20, 9001, 300, 32), (16, 9000, 200, 64), (5, 4999, 333, 96), (40, 8001, 1501, 128), (2, 33000, 65, 32), (9, 6005, 1100, 64), (31, 8222, 1280, 32),
         # tiles of 256 x 64 and 256 x 128, K whole and shared out, tables that are asked for again
         (1490, 3310, 250, 32), (520, 5000, 4100, 64), (520, 5000, 4100, 32), (500, 5100, 2100, 2100), (1030, 2050, 4097, 32), (300, 4100, 8200, 128)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_product_with_4_bit_weights(ops, ref, size, dtype):
    M, N, K, group = size
    g = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    zeros = (M + N + K) % 2 == 0
    w, scale, zero = weights_of(g, N, K, group, dtype, zeros)
    a, bias = randn(g, M, K, dtype=dtype), randn(g, N, dtype=dtype) if N % 3 else None
    want, total = ref.matmul_int4_ref(a, w, scale, zero, group, bias)
    got = ops._matmul_int4_fwd(gpu(a), gpu(w), gpu(scale), gpu(zero), group=group, bias=gpu(bias))
    assert got.dtype == dtype
    close(got, want, product_bound(want, total, K, dtype, bias), "out")


@pytest.mark.parametrize("M", [1, 20, 70, 200, 600])
@pytest.mark.parametrize("out_dtype", TYPES, ids=str)
def test_product_of_views_and_types(ops, ref, M, out_dtype):
    # activations between other columns, at an odd distance; weights and scales likewise; scales, bias and result of other types; (2, M / 2) rows
    g = torch.Generator().manual_seed(M)
    N, K, group = 90, 256, 64
    w, scale, zero = weights_of(g, N, K, group, torch.float32, True)
    wide = torch.randint(0, 256, (N, K // 2 + 5), generator=g, dtype=torch.uint8)
    wide[:, 3:3 + K // 2] = w
    turned = gpu(scale).t().contiguous().t()
    a = randn(g, M, K, dtype=torch.bfloat16, lead=3, trail=2)
    bias = randn(g, 2 * N, dtype=torch.float16)[::2]
    want, total = ref.matmul_int4_ref(a, w, scale, zero, group, bias)
    got = ops._matmul_int4_fwd(gpu(a), gpu(wide)[:, 3:3 + K // 2], turned, gpu(zero).t().contiguous().t(), group=group, bias=gpu(bias), out_dtype=out_dtype)
    close(got, want, product_bound(want, total, K, out_dtype, bias), "out")
    if M % 2 == 0:
        again = ops._matmul_int4_fwd(gpu(a).unflatten(0, (2, -1)), gpu(w), gpu(scale), gpu(zero), group=group, bias=gpu(bias), out_dtype=out_dtype)
        assert again.shape == (2, M // 2, N)
        close(again.flatten(0, 1), want, product_bound(want, total, K, out_dtype, bias), "three dimensions")


def test_product_of_no_rows_columns_or_weights(ops):
    w, s = torch.zeros(8, 16, dtype=torch.uint8).cuda(), torch.ones(8, 1).cuda()
    assert ops._matmul_int4_fwd(torch.zeros(0, 32).cuda(), w, s, group=32).shape == (0, 8)
    assert ops._matmul_int4_fwd(torch.zeros(3, 32).cuda(), w[:0], s[:0], group=32).shape == (3, 0)
    bias = torch.arange(8.0).cuda()
    out = ops._matmul_int4_fwd(torch.zeros(3, 0).cuda(), w[:, :0], s[:, :0], group=32, bias=bias)
    assert torch.equal(out, bias.expand(3, 8))


@pytest.mark.parametrize("M", [1, 33, 140])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_product_with_values_that_are_not_finite(ops, dtype, M):
    # an infinity times q - zero is an infinity of its sign, or a NaN where they are equal; other rows are as ever
    g = torch.Generator().manual_seed(M)
    N, K = 48, 256
    w, scale, _ = weights_of(g, N, K, 128, dtype, False)
    a = randn(g, M, K, dtype=dtype)
    a[0, 37], a[M // 2, 200], a[M - 1, 5] = INF, -INF, float("nan")
    from oracle import decode_oracle
    values = (decode_oracle.unpacked(w, K) - 8).double()
    got = ops._matmul_int4_fwd(gpu(a), gpu(w), gpu(scale)).double().cpu()
    plain = ops._matmul_int4_fwd(gpu(torch.where(torch.isfinite(a), a, 0)), gpu(w), gpu(scale)).double().cpu()
    for m in range(M):
        bad = [(k, float(a[m, k])) for k in range(K) if not bool(torch.isfinite(a[m, k]))]
        if bad:
            want = sum(v * values[:, k] for k, v in bad)
            assert torch.equal(torch.isnan(got[m]), torch.isnan(want)) and torch.equal(got[m][~torch.isnan(want)], want[~torch.isnan(want)])
        else:
            assert torch.equal(got[m], plain[m])


# ---- norms around a block ------------------------------------------------------------------------------------------------

def block_bounds(x, weight, residual, next_weight, gate, factor, want, t, n, dtype):
    D, e = x.shape[-1], 2.0 ** -24
    c = (D / 64 + 16) / 2 + 4          # of a reciprocal root, in units
    e_t = e * (2 * (t - n).abs() + t.abs() + (c + 4) * n.abs())
    square = t.pow(2).sum(-1, keepdim=True)
    r = ((t.abs() * e_t).sum(-1, keepdim=True) / square.clamp(min=1e-300)).clamp(max=1.0) + c * e
    w = next_weight.double().abs()
    inverse = 1 / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5)
    e_out = w * inverse * e_t * 1.01 + want.abs() * (r * 1.01 + 3 * e)
    return rounded(t, dtype) + e_t * (1 + U[dtype]), rounded(want, dtype) + e_out * (1 + U[dtype]), e_out


def block_inputs(g, shape, dtype, gate):
    D = shape[-1]
    x, residual = randn(g, *shape, dtype=dtype), (4 * randn(g, *shape)).to(dtype)
    weight, next_weight = ((0.5 + torch.rand(D, generator=g)).to(dtype) for _ in range(2))
    of = {"none": None, "channel": (D,), "ones": (1,) * (len(shape) - 1) + (D,), "row": shape[:1] + (1,) * (len(shape) - 2) + (D,), "token": shape}[gate]
    return x, weight, residual, next_weight, None if of is None else randn(g, *of, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("shape,gate", [((1, 1), "channel"), ((3, 7), "none"), ((5, 8), "token"), ((2, 3, 65), "row"), ((64, 1, 2560), "channel"), ((1100, 1000), "none"),
                                        ((3, 400, 1537), "row"), ((1030, 2560), "channel"), ((2, 5, 4096), "token"), ((7, 6145), "ones"), ((4, 10240), "row"),
                                        ((3, 16391), "channel"), ((2, 2, 3, 520), "row"), ((5, 8192), "token"), ((3, 8199), "channel"), ((2, 12289), "none"),
                                        ((3, 16384), "row"), ((2, 24576), "token"), ((2, 24579), "channel"), ((1025, 5120), "row"), ((2, 1030, 1033), "row")], ids=str)
def test_norms_around_a_block(ops, ref, shape, gate, int8, dtype):
    g = torch.Generator().manual_seed(sum(shape) + int8)
    x, weight, residual, next_weight, gated = block_inputs(g, shape, dtype, gate)
    weight = None if sum(shape) % 4 == 1 else weight
    factor = [1.0, 0.7][sum(shape) % 2]
    want, t, n = ref.norm_block_ref(x, weight, residual, next_weight, gated, factor)
    out, scale, total = ops._norm_block_fwd(gpu(x), gpu(weight), gpu(residual), gpu(next_weight), gate=gpu(gated), residual_scale=factor, int8=int8)
    bound_t, bound_out, e_out = block_bounds(x, weight, residual, next_weight, gated, factor, want, t, n, dtype)
    close(total, t, bound_t, "residual")
    if not int8:
        assert scale is None and out.dtype == dtype
        return close(out, want, bound_out, "out")
    assert out.dtype == torch.int8 and scale.shape == out.shape[:-1]
    step = want.abs().amax(-1, keepdim=True) / 127
    close(scale[..., None], step, e_out.amax(-1, keepdim=True) / 127 + 4 * 2.0 ** -24 * step, "scale")
    # half a step from its value, which the errors in front of the rounding move
    close(out.double().cpu() * scale.double().cpu()[..., None], want, step * (0.5 + 2.0 ** -15) + 2 * e_out + want.abs() * 2.0 ** -22, "8 bits")
    assert bool((out.abs().amax(-1) == 127).all())


@pytest.mark.parametrize("int8", [False, True])
def test_norms_of_zeros_and_of_values_that_are_not_finite(ops, int8):
    D = 264
    x, residual = torch.randn(6, D).bfloat16(), torch.randn(6, D).bfloat16()
    x[1], residual[1] = 0, 0
    x[2, 5], residual[3, D - 1], x[4, 0] = float("nan"), INF, INF
    one = torch.ones(D).bfloat16().cuda()
    out, scale, total = ops._norm_block_fwd(gpu(x), one, gpu(residual), one, int8=int8)
    if int8:
        values = scale.cpu()
        assert bool(torch.isfinite(values[[0, 5]]).all()) and float(values[1]) == 0 and not bool(out[1].any()) and bool(torch.isnan(values[2:5]).all())
    else:
        finite = torch.isfinite(out.float()).all(-1).cpu()
        assert finite.tolist() == [True, True, False, False, False] + [True] and not bool(out[1].any())
    assert not bool(total[1].any()) and bool(torch.isnan(total[2]).all()) and float(total[3, D - 1]) == INF


def test_norms_of_several_types_and_views(ops, ref):
    # a residual kept in fp32, weights and a gate in fp32, rows between other columns
    g = torch.Generator().manual_seed(3)
    for D in (96, 250):
        x = randn(g, 4, 9, D, dtype=torch.bfloat16, lead=3, trail=1)
        residual, weight, next_weight = randn(g, 4, 9, D), torch.rand(2 * D, generator=g)[::2], torch.rand(D, generator=g).half()
        gate = randn(g, 4, 1, D)
        want, t, n = ref.norm_block_ref(x, weight, residual, next_weight, gate, 1.25)
        out, _, total = ops._norm_block_fwd(gpu(x), gpu(weight), gpu(residual), gpu(next_weight), gate=gpu(gate), residual_scale=1.25)
        assert out.dtype == torch.bfloat16 and total.dtype == torch.float32
        bound_t, bound_out, _ = block_bounds(x, weight, residual, next_weight, gate, 1.25, want, t, n, torch.float32)
        close(total, t, bound_t, "residual")
        close(out, want, bound_out + rounded(want, torch.bfloat16) * 1.01, "out")
        # bf16 rows, weights of three types
        out, _, total = ops._norm_block_fwd(gpu(x), gpu(weight), gpu(residual.bfloat16()), gpu(next_weight), gate=gpu(gate), residual_scale=1.25)
        want, t, n = ref.norm_block_ref(x, weight, residual.bfloat16(), next_weight, gate, 1.25)
        bound_t, bound_out, _ = block_bounds(x, weight, residual, next_weight, gate, 1.25, want, t, n, torch.bfloat16)
        close(total, t, bound_t, "residual")
        close(out, want, bound_out, "out")


def test_norms_of_no_rows(ops):
    x, w = torch.zeros(2, 0, 16).cuda(), torch.ones(16).cuda()
    out, scale, total = ops._norm_block_fwd(x, w, x, w, gate=torch.ones(2, 1, 16).cuda(), int8=True)
    assert out.shape == x.shape and scale.shape == (2, 0) and total.shape == x.shape


# ---- beam selection --------------------------------------------------------------------------------------------------------

def selected(ops, ref, logits, scores, k, finished=None, pad=0):
    want, parents, tokens, near = ref.beam_select_ref(logits, scores, k, finished, pad)
    # (candidates of two beams nearer than the error of their scores could change places)
    assert near > 2 * LSE, near
    got = ops._beam_select_fwd(gpu(logits), gpu(scores), k, finished=gpu(finished), pad=pad)
    assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.int32]
    assert torch.equal(got[1].cpu().long(), parents) and torch.equal(got[2].cpu().long(), tokens)
    none = want == -INF
    assert torch.equal(got[0].cpu() == -INF, none)
    close(torch.where(none.cuda(), 0.0, got[0]), torch.where(none, 0.0, want), LSE + rounded(torch.where(none, 0.0, want), torch.float32), "scores")
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 1, 5, 3), (2, 4, 3, 7), (1, 4, 1000, 4), (3, 5, 8191, 10), (2, 8, 8193, 16), (1, 3, 30001, 64), (2, 32, 700, 64),
                                  (2, 64, 129, 1), (1, 2, 100003, 2), (5, 2, 16384, 33), (1, 64, 9000, 64)], ids=str)
def test_beam_selection(ops, ref, size, dtype):
    b, beams, V, k = size
    g = torch.Generator().manual_seed(V + k)
    logits = (2 * torch.randn(b, beams, V, generator=g)).to(dtype)
    scores = -30 * torch.rand(b, beams, generator=g)
    selected(ops, ref, logits, scores, k)
    finished = torch.rand(b, beams, generator=g) < 0.4
    selected(ops, ref, logits, scores, k, finished, pad=V // 2)
    # many tokens that are not allowed, now and then all of a beam's
    masked = logits.masked_fill(torch.rand(b, beams, V, generator=g) < 0.9, -INF)
    masked[torch.rand(b, beams, generator=g) < 0.3] = -INF
    selected(ops, ref, masked, scores, k, finished, pad=V - 1)


@pytest.mark.parametrize("size", [(2, 3, 20000, 5), (1, 4, 60, 50), (2, 8, 9001, 64), (1, 2, 40000, 64)], ids=str)
def test_beam_selection_among_equals(ops, ref, size):
    # all logits equal; few values; beams that are the same: the lowest index first, however many there are
    b, beams, V, k = size
    g = torch.Generator().manual_seed(k)
    scores = torch.full((b, beams), -1.5)
    for logits in (torch.zeros(b, beams, V), torch.zeros(b, beams, V).masked_fill(torch.arange(V) % 2 == 0, -0.0), torch.randint(0, 3, (b, 1, V), generator=g).float().expand(b, beams, V).contiguous(),
                   torch.randint(0, 40, (b, 1, V), generator=g).float().repeat(1, beams, 1)):
        for dtype in (torch.float32, torch.bfloat16):
            got = ops._beam_select_fwd(gpu(logits.to(dtype)), gpu(scores), k)
            want, parents, tokens, _ = ref.beam_select_ref(logits, scores, k)
            # (the same beams have the same sums, bit for bit)
            same = torch.sort((scores.double()[..., None] + logits.double()).flatten(1), dim=1, descending=True, stable=True)[1][:, :k]
            assert torch.equal(got[1].cpu().long(), same // V) and torch.equal(got[2].cpu().long(), same % V)
            close(got[0], want, LSE + rounded(want, torch.float32), "scores")


def test_beam_selection_of_rows_at_odd_addresses_is_the_same(ops):
    # equal beams at different distances from an aligned address, and at large strides
    g = torch.Generator().manual_seed(1)
    V, k = 9001, 12
    row = torch.randn(V, generator=g).bfloat16()
    wide = torch.zeros(2, 3, V + 13).bfloat16()
    logits = wide[..., 5:5 + V]
    logits[:] = row
    scores = torch.full((2, 3), -2.0).cuda()
    best, parents, tokens = ops._beam_select_fwd(gpu(logits), scores, k)
    order = torch.sort(row.float().repeat(3), descending=True, stable=True)[1][:k]
    assert torch.equal(parents.cpu().long(), (order // V).expand(2, k)) and torch.equal(tokens.cpu().long(), (order % V).expand(2, k))
    whole = ops._beam_select_fwd(logits.contiguous().cuda(), scores, k)
    assert all(torch.equal(s, t) for s, t in zip((best, parents, tokens), whole))


def test_beam_selection_with_scores_and_logits_that_are_not_numbers(ops, ref):
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(3, 6, 500, generator=g)
    scores = -5 * torch.rand(3, 6, generator=g)
    scores[0, 0], scores[0, 1], scores[0, 2] = -INF, float("nan"), INF
    logits[0, 3, 77], logits[0, 4, 5], logits[1, :, 9] = float("nan"), INF, -INF
    scores[2] = -INF
    for k in (3, 6, 64):
        selected(ops, ref, logits, scores, k)
        selected(ops, ref, logits, scores, k, torch.tensor([[True, True, False, True, False, False]] * 3), pad=2)
    # nothing left at all: the first candidates, at -inf
    best, parents, tokens = ops._beam_select_fwd(gpu(logits[2:]), gpu(scores[2:]), 4)
    assert bool((best == -INF).all()) and parents.tolist() == [[0] * 4] and tokens.tolist() == [[0, 1, 2, 3]]
    # the first step: one beam there, the others not
    first = torch.tensor([[0.0, -INF, -INF, -INF]])
    _, parents, _ = selected(ops, ref, logits[1:2, :4], first, 4)
    assert not bool(parents.any())


def test_beam_selection_of_no_rows(ops):
    got = ops._beam_select_fwd(torch.zeros(0, 2, 9).cuda(), torch.zeros(0, 2).cuda(), 2)
    assert all(t.shape == (0, 2) for t in got)


# ---- reordering of states ----------------------------------------------------------------------------------------------------

def pools_of(g, n):
    conv = torch.randn(n, 3, 40, generator=g).bfloat16().transpose(1, 2)
    return [torch.randn(n, 4, 8, 16, generator=g), conv, torch.randint(-99, 99, (n,), generator=g, dtype=torch.int64), torch.randn(n, 1000, generator=g)[:, 100:777],
            torch.randn(7, 5, n, generator=g).permute(2, 0, 1), torch.rand(n, 3, generator=g) < 0.5, torch.randn(n, 3, 4, 5, 6, generator=g)[:, :, 1:3, :, ::2].double(),
            torch.randn(n, 40000, generator=g), torch.randn(n, 33, generator=g).half(), torch.zeros(n, 0)]


@pytest.mark.parametrize("size", [(1, 1), (1, 2), (3, 4), (2, 64), (5, 7), (40, 3)], ids=str)
def test_reordering_of_states(ops, ref, size):
    b, beams = size
    g = torch.Generator().manual_seed(beams)
    n = b * beams + 2
    for kind in range(4):
        pools = pools_of(g, n)
        slots = torch.randperm(n, generator=g)[:b * beams].view(b, beams)
        if kind == 0:
            parents = torch.randint(0, beams, (b, beams), generator=g)
        elif kind == 1:
            parents = torch.randint(0, beams, (b, 1), generator=g).repeat(1, beams)      # all from one
        elif kind == 2:
            parents = torch.stack([torch.randperm(beams, generator=g) for _ in range(b)])
        else:                                                                              # padding, no beams, not enough slots
            parents = torch.randint(-1, beams + 1, (b, beams), generator=g)
            slots[torch.rand(b, beams, generator=g) < 0.4] = -1
            slots[0, 0] = n
        want, after = ref.beam_reorder_ref(parents, slots, pools)
        on = [gpu(p) for p in pools]
        new = ops._beam_reorder(parents.cuda(), slots.int().cuda(), on)
        assert new.dtype == torch.int32 and torch.equal(new.cpu().long(), want)
        for got, p in zip(on, after):
            assert torch.equal(got.cpu(), p)


def test_reordering_of_many_pools_or_none(ops, ref):
    g = torch.Generator().manual_seed(5)
    parents, slots = torch.randint(0, 4, (6, 4), generator=g), torch.randperm(30, generator=g)[:24].view(6, 4)
    pools = [torch.randn(30, 5 + i, generator=g) for i in range(120)]
    want, after = ref.beam_reorder_ref(parents, slots, pools)
    on = [p.cuda() for p in pools]
    assert torch.equal(ops._beam_reorder(parents.int().cuda(), slots.cuda(), on).cpu().long(), want)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(on, after))
    assert torch.equal(ops._beam_reorder(parents.cuda(), slots.cuda(), []).cpu().long(), want)
    assert ops._beam_reorder(parents[:0].cuda(), slots[:0].cuda(), on).shape == (0, 4)
    strided = [torch.randn(9, 4, 30, generator=g).permute(2, 0, 1) for _ in range(2)]
    want, after = ref.beam_reorder_ref(parents, slots, strided)
    on = [gpu(p) for p in strided]
    assert torch.equal(ops._beam_reorder(parents.cuda(), slots.cuda(), on).cpu().long(), want)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(on, after))


def test_reordering_of_beams_that_share_a_slot(ops, ref):
    # they are one beam: its first child takes the slot, whoever of them is its parent, and none of them has one to give
    for slots, parents in (([[4, 4, 4, 1]], [[0, 1, 2, 0]]), ([[2, 2, 5]], [[1, 2, 2]]), ([[3, 0, 3, 0]], [[2, 0, 3, 1]]), ([[1, 1, 1, 1]], [[3, 3, 0, 1]]),
                           ([[5, -1, 5, 2, 0]], [[2, 2, 1, 0, 0]])):
        slots, parents = torch.tensor(slots), torch.tensor(parents)
        pools = [torch.randn(6, 40), torch.randn(7, 6).t()]
        want, after = ref.beam_reorder_ref(parents, slots, pools)
        on = [gpu(p) for p in pools]
        assert torch.equal(ops._beam_reorder(parents.cuda(), slots.int().cuda(), on).cpu().long(), want)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(on, after))


# ---- streams, graphs, large distances, calls at the C entry ------------------------------------------------------------

def step_of(ops, g, M):
    """Inputs of a step, and the step: every operator, one behind another, into results that are all returned."""
    K, N, V = 1032, 700, 9001
    w, scale, zero = (gpu(t) for t in weights_of(g, N, K, 32, torch.bfloat16, True))
    head, hs, hz = (gpu(t) for t in weights_of(g, V, N, 64, torch.bfloat16, True))
    one, two = (gpu(1 + 0.1 * torch.randn(N, generator=g)).bfloat16() for _ in range(2))
    pools = [torch.randn(M + 3, 50, 33, generator=g).cuda(), torch.randn(M + 3, 7, 3, generator=g).bfloat16().cuda()]
    keep = [p.clone() for p in pools]
    slots = torch.randperm(M, generator=g).view(-1, 2).int().cuda()
    inputs = dict(a=gpu(randn(g, M, K, dtype=torch.bfloat16)), residual=gpu(randn(g, M, N, dtype=torch.bfloat16)), scores=-torch.rand(M // 2, 2, generator=g).cuda())

    def run():
        for pool, before in zip(pools, keep):
            pool.copy_(before)
        x = ops._matmul_int4_fwd(inputs["a"], w, scale, zero, group=32)
        u, _, t = ops._norm_block_fwd(x, one, inputs["residual"], two, gate=one, residual_scale=0.7)
        q, s, _ = ops._norm_block_fwd(x, None, t, two, int8=True)
        logits = ops._matmul_int4_fwd(u, head, hs, hz, group=64)
        best, parents, tokens = ops._beam_select_fwd(logits.view(M // 2, 2, V), inputs["scores"])
        new = ops._beam_reorder(parents, slots, pools)
        return [x, u, t, q, s, best, parents, tokens, new, *pools]
    return inputs, run


def same(got, want):
    return all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_step_on_two_streams_at_once(ops):
    g = torch.Generator().manual_seed(11)
    steps = [step_of(ops, g, M) for M in (64, 300)]
    want = [[t.clone() for t in run()] for _, run in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        got = []
        for stream, (_, run) in zip(streams, steps):
            with torch.cuda.stream(stream):
                got.append([run(), run()][1])
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(got, want))


def test_steps_from_graphs_between_eager_ones(ops):
    # two graphs and eager calls of the same sizes: each has workspaces of its own, and a replay sees what its inputs hold by then
    g = torch.Generator().manual_seed(12)
    (inputs, run), (_, other) = step_of(ops, g, 64), step_of(ops, g, 300)
    want_other = [t.clone() for t in other()]
    run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (run, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(f())
        graphs.append(graph)
    for i in range(4):
        inputs["a"].copy_(gpu(randn(g, *inputs["a"].shape, dtype=torch.bfloat16)))
        inputs["scores"].copy_(-torch.rand(inputs["scores"].shape, generator=g))
        want = [t.clone() for t in run()]
        graphs[0].replay()
        graphs[1].replay()
        got, got_other = [t.clone() for t in outs[0]], [t.clone() for t in outs[1]]
        if i % 2:
            torch.cuda.synchronize()
        other()
        assert same(got, want) and same(got_other, want_other)


def test_rows_that_lie_far_apart(ops, ref):
    # rows, weights, logits and slots more than 2^31 elements and bytes from the first
    g = torch.Generator().manual_seed(13)
    far = 1 << 30
    room = torch.empty(3 * far + 4096, dtype=torch.bfloat16, device="cuda")
    small = randn(g, 4, 96, dtype=torch.bfloat16)
    x = room.as_strided((4, 96), (far, 1))
    x.copy_(small)
    w, scale, zero = weights_of(g, 20, 96, 32, torch.bfloat16, True)
    want, total = ref.matmul_int4_ref(small, w, scale, zero, 32)
    close(ops._matmul_int4_fwd(x, gpu(w), gpu(scale), gpu(zero), group=32), want, product_bound(want, total, 96, torch.bfloat16), "activations")
    near = [ops._norm_block_fwd(gpu(small), None, gpu(small), gpu(small[0]), gate=gpu(small)), ops._beam_select_fwd(gpu(small)[:, None], torch.zeros(4, 1).cuda(), k=7)]
    assert same(ops._norm_block_fwd(x, None, x, gpu(small[0]), gate=x)[::2], near[0][::2])
    assert same(ops._beam_select_fwd(x[:, None], torch.zeros(4, 1).cuda(), k=7), near[1])
    scores = torch.zeros(1, 4).cuda()
    assert same(ops._beam_select_fwd(x[None], scores), ops._beam_select_fwd(gpu(small)[None], scores))
    del x
    bytes_ = room.view(torch.uint8)
    wide = bytes_.as_strided((20, 48), ((1 << 28) + 3, 1))
    wide.copy_(w)
    close(ops._matmul_int4_fwd(gpu(small), wide, gpu(scale), gpu(zero), group=32), want, product_bound(want, total, 96, torch.bfloat16), "weights")
    many = randn(g, 300, 1032, dtype=torch.bfloat16)
    rows = room.as_strided((300, 1032), (10 << 20, 1))
    rows.copy_(many)
    w, scale, _ = weights_of(g, 512, 1032, 128, torch.bfloat16, False)
    assert torch.equal(ops._matmul_int4_fwd(rows, gpu(w), gpu(scale)), ops._matmul_int4_fwd(gpu(many), gpu(w), gpu(scale)))
    pool = bytes_.as_strided((5, 300), (1300000001, 1))
    before = torch.randint(0, 256, (5, 300), generator=g, dtype=torch.uint8)
    pool.copy_(before)
    new = ops._beam_reorder(torch.tensor([[4, 4, 0]]).cuda()[:, :3], torch.tensor([[4, 0, 2]]).int().cuda(), [pool])
    assert new.tolist() == [[-1, -1, 4]] and torch.equal(pool.cpu(), before)
    new = ops._beam_reorder(torch.tensor([[0, 0, 2]]).cuda(), torch.tensor([[4, 3, 1]]).int().cuda(), [pool])
    before[3] = before[4]
    assert new.tolist() == [[4, 3, 1]] and torch.equal(pool.cpu(), before)


@pytest.mark.parametrize("size", [(300, 1500, 1032, 64), (64, 2560, 5120, 128), (2048, 600, 300, 32)], ids=str)
def test_the_product_without_its_workspace(ops, ref, size):
    import ctypes
    from ssd_amd import _lib
    from ssd_amd.decode import _bytes_arg
    from ssd_amd.layer import _arg
    M, N, K, group = size
    g = torch.Generator().manual_seed(M)
    a = randn(g, M, K, dtype=torch.bfloat16)
    w, scale, zero = weights_of(g, N, K, group, torch.bfloat16, True)
    want, total = ref.matmul_int4_ref(a, w, scale, zero, group)
    lib, on = _lib.load(), [gpu(t) for t in (a, w, scale, zero)]
    need = lib.ssd_matmul_packed_workspace_bytes(M, N, K, group, _lib._DTYPES[a.dtype])
    for room in (0, max(need - 1, 0), need):
        space = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
        out = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        assert lib.ssd_matmul_packed_fwd(_arg(on[0]), _bytes_arg(on[1]), _arg(on[2]), _bytes_arg(on[3]), _arg(None), _arg(out), M, N, K, group,
                                         ctypes.c_void_p(space.data_ptr()) if room else None, room, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        close(out, want, product_bound(want, total, K, torch.bfloat16), "out")
        assert bool((space[room:] == 255).all())
