"""The operators around the state path -- short convolution, selective scan, norm, 8-bit matrix product, each for prompts and where it
has one for single tokens -- against their restatement in 64 bits (oracle/layer_oracle.py).

Bounds.  A result is rounded once to its type: half a unit of its last place, 2^-8 (bf16: 8 significant bits), 2^-11 (fp16) or
2^-24 of its size.  In front of that
stand sums in 32 bits, whose error is a multiple of 2^-24 of the same sum over absolute values (the oracle gives it), the hardware's
exponential, logarithm and reciprocal (errors of 2 units, 2^-22), and in the scan the decay: a product of L factors that each carry the
error of an exponential, or an exponential of a sum of L terms.  On the bf16 matrix instructions operands made here (weighted x,
decayed scores, states) are carried as two bf16 parts: 2^-16 of each term."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    import ssd_amd
    from ssd_amd import _lib
    _lib.load()
    return ssd_amd


@pytest.fixture(scope="module")
def ref():
    import importlib
    return importlib.import_module("oracle.layer_oracle")


def gpu(t):
    """To the GPU with the storage around it: the same strides, the same distance from an aligned address."""
    if t is None:
        return None
    n = t.untyped_storage().nbytes() // t.element_size()
    return torch.as_strided(t, (n,), (1,), 0).cuda().as_strided(t.shape, t.stride(), t.storage_offset())


def close(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: off by {float((off + bound).max()):.3e}, {float((off / bound.clamp(min=1e-300)).max() + 1):.2f} of the bound"


def rounded(want, dtype):
    # half a unit of the type; below its normal range half of its smallest step
    return U[dtype] * want.abs() + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]


def randn(g, *size, dtype=torch.float32, lead=0, trail=0):
    """Normal values; as a view with `lead` / `trail` columns around where asked."""
    t = torch.randn(*size[:-1], size[-1] + lead + trail, generator=g).to(dtype)
    return t[..., lead:lead + size[-1]]


def sequences(g, b, L, n, first=0):
    marks = torch.zeros(b, L, dtype=torch.int32)
    marks.scatter_(1, torch.randint(0, L, (b, n), generator=g), 1)
    return torch.cumsum(marks, 1, dtype=torch.int32) + first


# ---- short convolution ----------------------------------------------------------------------------------------------

def conv_bound(want, size, K, dtype):
    # K + 1 additions and products; the activation's slope is below 1.1, its own error 4 units of its argument
    return rounded(want, dtype) + (K + 8) * 2.0 ** -23 * size + 2.0 ** -126


CONVS = [  # b, L, D, K, init, seqs, lengths, lead
    (1, 1, 1, 4, True, 0, None, 0), (2, 3, 5, 4, True, 0, None, 0), (1, 2, 8, 2, False, 0, None, 0), (1, 5, 7, 1, False, 0, None, 0),
    (2, 33, 24, 4, False, 3, None, 3), (3, 40, 17, 3, True, 6, [40, 0, 7], 1), (2, 9, 64, 4, True, 4, [1, 2], 8), (3, 70, 1792, 4, True, 0, [70, 33, 0], 5),
    (1, 200, 100, 4, True, 30, None, 0), (2, 130, 256, 2, True, 5, None, 0), (2, 0, 24, 4, True, 0, None, 0), (4, 13, 24, 4, True, 13, [13, 3, 0, 12], 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CONVS, ids=str)
def test_short_conv(ops, ref, case, dtype):
    b, L, D, K, init, seqs, lengths, lead = case
    g = torch.Generator().manual_seed(L * 7 + D)
    x, w, bias = randn(g, b, L, D, dtype=dtype, lead=lead, trail=lead), randn(g, D, K, dtype=dtype), randn(g, D, dtype=dtype)
    state = randn(g, b, K - 1, D, dtype=dtype).transpose(1, 2) if init and K > 1 else None
    seq = sequences(g, b, L, seqs, first=L % 2) if seqs else None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    want, final, size = ref.short_conv_ref(x, w, bias, True, state, seq, n)
    y, last = ops._short_conv_fwd(gpu(x), gpu(w), gpu(bias), initial_states=gpu(state), seq_idx=gpu(seq), lengths=gpu(n))
    assert y.dtype == dtype and last.dtype == dtype
    close(y, want, conv_bound(want, size, K, dtype), "y")
    assert torch.equal(last.double().cpu(), final)
    # without bias and activation, other types of weight, states with contiguous taps
    w32 = w.float()
    want, final, size = ref.short_conv_ref(x, w32, None, False, state, seq, n)
    y, last = ops._short_conv_fwd(gpu(x), gpu(w32), None, silu=False, initial_states=None if state is None else gpu(state.contiguous()),
                                  seq_idx=gpu(seq), lengths=gpu(n))
    close(y, want, conv_bound(want, size, K, dtype), "plain y")
    assert torch.equal(last.double().cpu(), final)


def test_short_conv_long_runs(ops, ref):
    # large enough for the runs of 32 tokens; checked on a few channels
    g = torch.Generator().manual_seed(5)
    b, L, D = 2, 1100, 8200
    x, w, bias = randn(g, b, L, D, dtype=torch.bfloat16), randn(g, D, 4, dtype=torch.bfloat16), randn(g, D, dtype=torch.bfloat16)
    for seq in (None, sequences(g, b, L, 40)):
        n = torch.tensor([L, 555], dtype=torch.int32)
        y, last = ops._short_conv_fwd(gpu(x), gpu(w), gpu(bias), seq_idx=gpu(seq), lengths=gpu(n))
        some = torch.tensor([0, 1, 7, 8, 4095, 8191, 8192, 8199])
        want, final, size = ref.short_conv_ref(x[..., some], w[some], bias[some], True, None, seq, n)
        close(y[..., some.cuda()], want, conv_bound(want, size, 4, torch.bfloat16))
        assert torch.equal(last[:, some.cuda()].double().cpu(), final)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(1, 1, 4), (3, 5, 4), (5, 8, 2), (70, 24, 4), (4, 77, 3), (2, 1792, 4), (2, 100, 1)], ids=str)
def test_short_conv_step(ops, ref, case, dtype):
    b, D, K = case
    g = torch.Generator().manual_seed(b + D)
    x, w, bias = randn(g, b, D, dtype=dtype, lead=1), randn(g, D, K, dtype=dtype), randn(g, D, dtype=dtype)
    for pool, turned in ((b, True), (b + 3, False)):
        states = randn(g, pool, K - 1, D, dtype=dtype).transpose(1, 2)
        states = states if turned else states.contiguous()
        slots = None
        if pool > b:
            slots = torch.randperm(pool, generator=g)[:b].to(torch.int32)
            slots[b // 2] = -1 if b % 2 else pool
        want, after = ref.short_conv_step_ref(x, states, w, bias, True, slots)
        size = (torch.cat([states, torch.zeros(pool, D, 1)], 2).abs().amax() + x.double().abs().amax()) * w.double().abs().sum(1) + 4
        on_gpu = gpu(states)
        y = ops._short_conv_step(gpu(x), on_gpu, gpu(w), gpu(bias), slots=gpu(slots))
        close(y, want, conv_bound(want, size, K, dtype))
        assert torch.equal(on_gpu.double().cpu(), after)


def test_short_conv_prompt_then_steps(ops):
    # a prompt cut anywhere and continued, by a prompt or by single tokens, is the whole prompt
    g = torch.Generator().manual_seed(3)
    x, w, bias = (gpu(randn(g, *s, dtype=torch.bfloat16)) for s in ((2, 21, 40), (40, 4), (40,)))
    whole, final = ops._short_conv_fwd(x, w, bias)
    for cut in (1, 2, 3, 17):
        head, state = ops._short_conv_fwd(x[:, :cut], w, bias)
        tail, last = ops._short_conv_fwd(x[:, cut:], w, bias, initial_states=state)
        assert torch.equal(torch.cat([head, tail], 1), whole) and torch.equal(last, final)
        for t in range(cut, 21):
            assert torch.equal(ops._short_conv_step(x[:, t], state, w, bias), whole[:, t])
        assert torch.equal(state, final)


def test_short_conv_masked_places_may_hold_anything(ops):
    g = torch.Generator().manual_seed(4)
    x, w = randn(g, 2, 30, 24, dtype=torch.bfloat16), randn(g, 24, 4, dtype=torch.bfloat16)
    seq = torch.cat([torch.zeros(2, 11, dtype=torch.int32), torch.ones(2, 19, dtype=torch.int32)], 1)
    n = torch.tensor([25, 30], dtype=torch.int32)
    clean, last = ops._short_conv_fwd(gpu(x), gpu(w), seq_idx=gpu(seq), lengths=gpu(n))
    for junk in (float("nan"), float("inf")):
        dirty = x.clone()
        dirty[0, 25:] = junk            # behind the length
        dirty[1, :11] = junk            # another sequence
        y, fin = ops._short_conv_fwd(gpu(dirty), gpu(w), seq_idx=gpu(seq), lengths=gpu(n))
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1, 11:], clean[1, 11:]) and torch.equal(fin, last)


# ---- selective scan -------------------------------------------------------------------------------------------------

def scan_inputs(g, b, L, H, P, N, G, dtype, init=False, gate=True, packed=True):
    if packed:
        xbc = torch.nn.functional.silu(torch.randn(b, L, H * P + 2 * G * N, generator=g)).to(dtype)
        x, B, C = xbc.split([H * P, G * N, G * N], dim=-1)
    else:
        x, B, C = (torch.randn(b, L, n, generator=g).to(dtype) for n in (H * P, G * N, G * N))
    dt = torch.randn(b, L, H, generator=g) - 3
    return dict(x=x.reshape(b, L, H, P) if not packed else x.unflatten(-1, (H, P)), dt=dt.to(dtype), A=-torch.exp(torch.rand(H, generator=g) * 2.77),
                B=B.unflatten(-1, (G, N)), C=C.unflatten(-1, (G, N)), D=torch.randn(H, generator=g),
                z=randn(g, b, L, H * P, dtype=dtype, trail=8).unflatten(-1, (H, P)) if gate else None,
                dt_bias=torch.randn(H, generator=g) * 0.3, dt_softplus=True,
                initial_states=torch.randn(b, H, P, N, generator=g) if init else None)


def scan_bounds(want, size, L, dtype):
    # decay: L factors or terms of 2 units each, seen through a decaying state (64 of them at most matter: dt A is a few hundredths);
    # sums; and for bf16 the two parts of what is multiplied on the matrix instructions (three such products in a row)
    near = 3 * 2.0 ** -16 if dtype == torch.bfloat16 else 0.0
    return rounded(want, dtype) + (near + (128 + min(L, 512)) * 2.0 ** -23) * size + 2.0 ** -126


def check_scan(ops, ref, a, seq=None, n=None, dtype=None, **kw):
    want, final, size, final_size = ref.ssd_scan_ref(**a, seq_idx=seq, lengths=n, **kw)
    on = {k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}
    y, last = ops._ssd_scan_fwd(**on, seq_idx=gpu(seq), lengths=gpu(n), **kw)
    L = a["x"].shape[1]
    assert y.dtype == a["x"].dtype and last.dtype == torch.float32
    close(y, want, scan_bounds(want, size, L, a["x"].dtype), "y")
    close(last, final, scan_bounds(final, final_size, L, a["x"].dtype) - rounded(final, a["x"].dtype) + rounded(final, torch.float32), "final states")
    return y, last


SCANS = [  # b, L, H, P, N, G, init, seqs, lengths
    (1, 1, 1, 1, 1, 1, True, 0, None), (2, 3, 2, 5, 7, 1, True, 0, None), (1, 64, 2, 64, 128, 1, False, 0, None), (2, 65, 4, 64, 128, 2, True, 0, None),
    (1, 200, 3, 64, 128, 1, True, 0, None), (2, 130, 4, 64, 64, 4, True, 9, None), (3, 100, 2, 48, 96, 1, True, 0, [100, 0, 37]),
    (4, 150, 4, 64, 128, 2, True, 7, [150, 64, 0, 65]), (2, 63, 2, 128, 128, 1, False, 3, None), (1, 127, 2, 32, 16, 1, False, 60, None),
    (1, 90, 2, 40, 256, 1, True, 0, None), (1, 77, 5, 64, 40, 5, True, 2, None), (1, 700, 2, 64, 128, 1, True, 3, [600]), (2, 0, 2, 64, 128, 1, True, 0, None),
    (1, 64, 6, 64, 128, 2, False, 0, [0]), (1, 640, 1, 100, 128, 1, False, 0, None), (2, 320, 2, 16, 32, 1, True, 0, [257, 320]), (1, 33, 2, 80, 64, 1, True, 0, None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SCANS, ids=str)
def test_ssd_scan(ops, ref, case, dtype):
    b, L, H, P, N, G, init, seqs, lengths = case
    g = torch.Generator().manual_seed(L * 3 + P)
    a = scan_inputs(g, b, L, H, P, N, G, dtype, init=init)
    seq = sequences(g, b, L, seqs, first=P % 3 // 2) if seqs else None
    check_scan(ops, ref, a, seq, None if lengths is None else torch.tensor(lengths, dtype=torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_ssd_scan_arguments(ops, ref, dtype):
    # no gate, no skip, no bias, no softplus; D per channel; limits; steps of another type; heads and tokens in other orders
    g = torch.Generator().manual_seed(11)
    b, L, H, P, N, G = 2, 150, 4, 64, 128, 2
    a = scan_inputs(g, b, L, H, P, N, G, dtype, gate=False, packed=False)
    a.update(D=None, dt_bias=None, dt_softplus=False, dt=(torch.rand(b, L, H, generator=g) * 0.1).to(dtype))
    check_scan(ops, ref, a)
    a = scan_inputs(g, b, L, H, P, N, G, dtype, init=True)
    a.update(D=torch.randn(H, P, generator=g), dt=a["dt"].float())
    check_scan(ops, ref, a, dt_limit=(0.02, 0.06))
    a.update(x=a["x"].transpose(1, 2).contiguous().transpose(1, 2), z=a["z"].transpose(0, 1).contiguous().transpose(0, 1),
             B=a["B"].transpose(1, 2).contiguous().transpose(1, 2), initial_states=a["initial_states"].transpose(1, 2).contiguous().transpose(1, 2))
    check_scan(ops, ref, a)
    # nothing contiguous where the kernels want it, rows at odd addresses
    a.update(x=torch.randn(b, L, P, H, generator=g).to(dtype).transpose(2, 3), C=randn(g, b, L, G, N, dtype=dtype, lead=1, trail=2))
    check_scan(ops, ref, a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(8, 432, 22, 40, 16, 2, True), (2, 300, 8, 64, 128, 1, False), (1, 700, 6, 32, 64, 1, False), (3, 130, 10, 128, 96, 2, True)], ids=str)
def test_ssd_scan_without_gate(ops, ref, case, dtype):
    # chunks enough per workgroup for what one stores to be followed by the next one's work; the same again each time
    b, L, H, P, N, G, init = case
    g = torch.Generator().manual_seed(L + P)
    a = scan_inputs(g, b, L, H, P, N, G, dtype, init=init, gate=False)
    for seq in (None, sequences(g, b, L, 3)):
        y, last = check_scan(ops, ref, a, seq)
        for _ in range(3):
            again, states = ops._ssd_scan_fwd(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}, seq_idx=gpu(seq))
            assert torch.equal(again, y) and torch.equal(states, last)


def test_ssd_scan_of_strong_and_of_no_decay(ops, ref):
    g = torch.Generator().manual_seed(12)
    a = scan_inputs(g, 1, 200, 2, 64, 128, 1, torch.bfloat16, init=True)
    a.update(A=torch.tensor([-3e4, 0.0]), dt_softplus=False, dt_bias=None, dt=(torch.rand(1, 200, 2, generator=g) * 0.5).bfloat16())
    check_scan(ops, ref, a)
    a.update(A=torch.tensor([-1e38, -200.0]))
    check_scan(ops, ref, a)


def test_ssd_scan_in_segments(ops, ref):
    # rows long enough to be cut: with sequences, lengths that end in the first, inside and at the end of a segment, and states
    g = torch.Generator().manual_seed(13)
    for dtype in (torch.bfloat16, torch.float32):
        for L, lengths, seqs in ((1024, None, 0), (1100, [1100, 300], 5), (769, [0, 513], 0), (2000, [1024, 1999], 2)):
            a = scan_inputs(g, 2, L, 2, 64, 128, 1, dtype, init=True)
            check_scan(ops, ref, a, sequences(g, 2, L, seqs) if seqs else None, None if lengths is None else torch.tensor(lengths, dtype=torch.int32))


def on_bf16_instructions(b, L, H, P, N, G):
    """Whether such a call goes to the kernel on the bf16 matrix instructions: it keeps records of the steps."""
    from ssd_amd import _lib
    nbytes = int(_lib.load().ssd_scan_workspace_bytes(_lib.dims_arg(b, L, H, P, N, G, 0, 0), _lib.SSD_BF16))
    return nbytes >= b * H * ((L + 63) // 64) * 5 * 64 * 4


# sizes large enough for the bf16 matrix instructions: one segment, three (joined by who enters them) and many; rows of other lengths
@pytest.mark.parametrize("case", [(8, 190, 40, 64, 128, 4, True, 3, None), (4, 300, 128, 8, 64, 1, True, 0, [300, 0, 64, 65]),
                                  (2, 500, 80, 64, 128, 2, True, 5, [500, 77]), (3, 257, 96, 40, 72, 1, False, 2, [0, 257, 64]),
                                  (2, 1100, 40, 64, 128, 1, True, 3, [1100, 300]), (1, 1500, 24, 32, 128, 1, False, 0, None),
                                  (1, 2000, 16, 64, 128, 1, True, 9, [1999])], ids=str)
def test_ssd_scan_on_the_bf16_instructions(ops, ref, case):
    b, L, H, P, N, G, init, seqs, lengths = case
    assert on_bf16_instructions(b, L, H, P, N, G)
    g = torch.Generator().manual_seed(L + H)
    a = scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=init, gate=seqs != 9)
    a["A"][0], a["A"][1] = -3e4, 0.0
    check_scan(ops, ref, a, sequences(g, b, L, seqs) if seqs else None, None if lengths is None else torch.tensor(lengths, dtype=torch.int32))


@pytest.mark.parametrize("marks", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("case", [(8, 1500, 128, 32, 64, 8), (4, 2500, 128, 64, 128, 8), (2, 6000, 80, 64, 128, 1), (1, 16384, 80, 64, 96, 1)], ids=str)
def test_ssd_scan_of_long_rows_agrees_with_fp32(ops, case, gate, marks):
    # rows cut into segments of different length, the first beside what the others add: against the fp32 kernel on the same values, with a
    # bound of the magnitudes that are added (the fp32 kernel's, on absolute values)
    b, L, H, P, N, G = case
    assert on_bf16_instructions(*case)
    g = torch.Generator().manual_seed(L + N)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True, gate=gate).items()}
    kw = {}
    if marks:
        kw["seq_idx"] = gpu(sequences(g, b, L, 4))
        kw["lengths"] = gpu(torch.tensor([L, 700, L - 1, 64, 0, 1, 65, L // 2][:b], dtype=torch.int32))
    y, last = ops._ssd_scan_fwd(**a, **kw)
    wide = {k: v.float() if k in ("x", "B", "C", "z") and v is not None else v for k, v in a.items()}
    want, final = ops._ssd_scan_fwd(**wide, **kw)
    magnitudes = {k: v.abs() if k in ("x", "B", "C", "D", "initial_states") else v for k, v in wide.items()}
    size, final_size = ops._ssd_scan_fwd(**dict(magnitudes, z=None), **kw)
    if gate:
        size = size * torch.nn.functional.silu(wide["z"]).abs()
    near = 3 * 2.0 ** -16 + 2 * (128 + 512) * 2.0 ** -23      # as in scan_bounds, for either kernel
    assert bool(((y.float() - want).abs() <= 2.0 ** -8 * want.abs() + near * size + 1e-30).all())
    assert bool(((last - final).abs() <= near * final_size + 1e-30).all())


def test_ssd_scan_on_the_bf16_instructions_with_nan(ops):
    # a chunk that holds them goes token by token: what they may not reach is as without them
    g = torch.Generator().manual_seed(21)
    b, L, H, P, N, G = 2, 500, 80, 64, 128, 2
    assert on_bf16_instructions(b, L, H, P, N, G)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True).items()}
    seq, n = torch.zeros(b, L, dtype=torch.int32), torch.tensor([500, 333], dtype=torch.int32)
    seq[:, 101:] = 1
    y, last = ops._ssd_scan_fwd(**a, seq_idx=gpu(seq), lengths=gpu(n))
    for junk in (float("nan"), float("inf")):
        for key in ("x", "B", "C", "z", "dt"):
            t = a[key].clone()
            t[0, 97:101] = junk      # the end of a sequence
            t[1, 333:] = junk        # behind a row's length
            y2, last2 = ops._ssd_scan_fwd(**dict(a, **{key: t}), seq_idx=gpu(seq), lengths=gpu(n))
            # (in a chunk that goes token by token sums are in another order)
            assert torch.equal(y2[0, :64], y[0, :64]) and torch.equal(y2[1], y[1])
            torch.testing.assert_close(y2[0, 64:97].float(), y[0, 64:97].float(), rtol=2e-2, atol=2e-2)
            torch.testing.assert_close(y2[0, 101:].float(), y[0, 101:].float(), rtol=2e-2, atol=2e-2)
            torch.testing.assert_close(last2, last, rtol=1e-3, atol=1e-3)



@pytest.mark.parametrize("dtype", TYPES)
def test_ssd_scan_masked_places_may_hold_anything(ops, dtype):
    g = torch.Generator().manual_seed(14)
    a = scan_inputs(g, 2, 200, 2, 64, 128, 1, dtype, init=True)
    seq = torch.cat([torch.zeros(2, 70, dtype=torch.int32), torch.ones(2, 130, dtype=torch.int32)], 1)
    n = torch.tensor([150, 200], dtype=torch.int32)
    on = {k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}
    clean, last = ops._ssd_scan_fwd(**on, seq_idx=gpu(seq), lengths=gpu(n))
    for junk in (float("nan"), float("inf"), -float("inf")):
        for name in ("x", "B", "C", "dt", "z"):
            dirty = dict(on)
            dirty[name] = on[name].clone()
            dirty[name][0, 150:] = junk          # behind the length
            dirty[name][1, 30:60] = junk         # another sequence, in the chunk where the next one starts
            y, fin = ops._ssd_scan_fwd(**dirty, seq_idx=gpu(seq), lengths=gpu(n))
            assert torch.equal(fin, last), name
            assert torch.equal(y[0], clean[0]) and torch.equal(y[1, 70:], clean[1, 70:]), (name, junk)
            # ... and nothing reaches back to tokens in front of it
            close(y[1, :30], clean[1, :30].double().cpu(), 2 * U[dtype] * clean[1, :30].double().cpu().abs() + 1e-3, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 1), (2, 4, 64, 128, 2), (3, 2, 5, 7, 1), (5, 3, 64, 64, 1), (2, 8, 128, 16, 8), (1, 2, 33, 256, 1), (2, 2, 8, 300, 1),
                                  (70, 16, 64, 128, 1)], ids=str)
def test_ssd_scan_step(ops, ref, case, dtype):
    b, H, P, N, G = case
    g = torch.Generator().manual_seed(b * 5 + N)
    a = scan_inputs(g, b, 1, H, P, N, G, dtype)
    a.pop("initial_states")
    a = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    for pool, lead in ((b, 0), (b + 3, 1)):
        states = randn(g, pool, H, P, N, lead=lead)
        slots = None
        if pool > b:
            slots = torch.randperm(pool, generator=g)[:b].to(torch.int32)
            slots[b // 2] = -1 if b % 2 else pool
        want, after, size = ref.ssd_scan_step_ref(**a, states=states, slots=slots)
        on = {k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}
        on_gpu = gpu(states)
        y = ops._ssd_scan_step(**on, states=on_gpu, slots=gpu(slots))
        close(y, want, rounded(want, dtype) + 160 * 2.0 ** -23 * size + 2.0 ** -126)
        close(on_gpu, after, 8 * 2.0 ** -23 * (after.abs() + states.abs() + 1))
        untouched = torch.ones(pool, dtype=torch.bool) if slots is not None else torch.zeros(pool, dtype=torch.bool)
        if slots is not None:
            untouched[slots[(slots >= 0) & (slots < pool)].long()] = False
        assert torch.equal(on_gpu.cpu()[untouched], states[untouched])


@pytest.mark.parametrize("dtype", TYPES)
def test_ssd_scan_prompt_then_steps(ops, dtype):
    g = torch.Generator().manual_seed(15)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, 2, 90, 4, 64, 128, 2, dtype).items()}
    whole, final = ops._ssd_scan_fwd(**a)
    head = {k: v[:, :80] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    y, state = ops._ssd_scan_fwd(**head)
    assert torch.equal(y, whole[:, :80])
    a.pop("initial_states")
    for t in range(80, 90):
        out = ops._ssd_scan_step(**{k: v[:, t] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}, states=state)
        torch.testing.assert_close(out.float(), whole[:, t].float(), rtol=4 * U[dtype] + 1e-4, atol=2e-3)
    torch.testing.assert_close(state, final, rtol=1e-3, atol=1e-4)


# ---- norm -----------------------------------------------------------------------------------------------------------

NORMS = [(1, 1), (3, 5), (1, 8), (2, 9), (5, 100), (7, 768), (1030, 40), (1030, 1000), (1025, 2560), (64, 5120), (2, 9001), (3, 12001), (1024, 1024), (0, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mode", ["", "residual", "gate"])
@pytest.mark.parametrize("case", NORMS, ids=str)
def test_norm(ops, ref, case, mode, dtype):
    rows, D = case
    g = torch.Generator().manual_seed(rows + D)
    x, w = randn(g, rows, D, dtype=dtype, lead=1), (torch.rand(D, generator=g) + 0.5).to(dtype)
    residual = 4 * randn(g, rows, D, dtype=dtype) if mode == "residual" else None
    z = randn(g, rows, D, dtype=dtype, trail=3) if mode == "gate" else None
    want, total = ref.norm_ref(x, w, residual, z)
    # a sum of D squares (its error under a root), a gate's exponential and reciprocal
    near = (D / 2 / 64 + 32) * 2.0 ** -24
    out, scale, sum_out = ops._norm_fwd(gpu(x), gpu(w), gpu(residual), gpu(z))
    assert scale is None and out.dtype == dtype
    close(out, want, rounded(want, dtype) + near * want.abs() + 2.0 ** -120, "out")
    for weight in (w, w.float()):
        q, scale, sum8 = ops._norm_fwd(gpu(x), gpu(weight), gpu(residual), gpu(z), int8=True)
        assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == (rows,)
        if rows:
            assert int(q.abs().amax(-1).min()) == 127
            step = want.abs().amax(-1, keepdim=True) / 127
            close(scale[:, None], step, 2 * near * step, "scale")
            # half a step, and what rounding makes of a value that lies between two
            close(q.double().cpu() * scale.double().cpu()[:, None], want, (0.5 + 127 * near + 1e-4) * step, "8 bits")
    if residual is not None:
        close(sum_out, total, rounded(total, dtype) + 2.0 ** -24 * total.abs(), "residual")
        assert torch.equal(sum8, sum_out)
    else:
        assert sum_out is None


def test_norm_of_special_rows(ops):
    x = torch.zeros(6, 512)
    x[1, 3], x[2, 5], x[3], x[4, 0] = float("nan"), float("inf"), 1e-30, -2.0
    q, scale, _ = ops._norm_fwd(gpu(x), torch.ones(512, device="cuda"), int8=True)
    values = (q.float() * scale[:, None]).cpu()
    assert torch.equal(values[0], torch.zeros(512)) and torch.equal(values[5], torch.zeros(512))
    assert bool(values[1].isnan().all()) and bool(values[2].isnan().all())
    torch.testing.assert_close(values[3], torch.full((512,), 1e-30 / 1e-5 ** 0.5), rtol=1e-5, atol=0)
    assert int(q[4, 0]) == -127 and int(q[4, 1:].abs().max()) == 0
    y, _, _ = ops._norm_fwd(x.reshape(2, 3, 512).cuda(), torch.ones(512, device="cuda"))
    assert y.shape == (2, 3, 512) and bool(y[0, 1].isnan().all()) and bool(y[0, 0].eq(0).all())


# ---- matrix product -------------------------------------------------------------------------------------------------

MATMULS = [(1, 1, 1), (1, 16, 128), (1, 300, 2560), (3, 17, 100), (16, 64, 130), (17, 33, 1000), (33, 48, 64), (64, 768, 1536), (65, 100, 129), (130, 130, 256),
           (200, 520, 4000), (300, 1000, 48), (777, 768, 1536), (2049, 257, 336), (257, 2305, 80), (5, 9, 0), (0, 9, 16), (4100, 4100, 144), (8, 16, 131071)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", MATMULS, ids=str)
def test_matmul(ops, ref, case, dtype):
    M, N, K = case
    g = torch.Generator().manual_seed(M + N + K)
    a, w = (torch.randint(-128, 128, (n, K), generator=g, dtype=torch.int64).to(torch.int8) for n in (M, N))
    if K == 131071:
        a.fill_(-128)
        w.fill_(-128)
    sa, sw, bias = torch.rand(M, generator=g) * 1e-3, torch.rand(N, generator=g) * 1e-2, torch.randn(N, generator=g)
    want = ref.matmul_int8_ref(a, sa, w, sw)
    near = 3 * 2.0 ** -24 * want.abs() + 2.0 ** -120
    out = ops._matmul_int8_fwd(gpu(a), gpu(sa), gpu(w), gpu(sw), out_dtype=dtype)
    assert out.dtype == dtype
    close(out, want, rounded(want, dtype) * 1.01 + near)
    want = want + bias.to(dtype).double()
    out = ops._matmul_int8_fwd(gpu(a), gpu(sa), gpu(w), gpu(sw), bias=gpu(bias.to(dtype)), out_dtype=dtype)
    close(out, want, rounded(want, dtype) * 1.01 + near + 2.0 ** -23 * (want.abs() + bias.abs()))


# sizes on each side of the bounds between the kernels: tiles of 256 x 256 to 64 x 64, and without tiles
@pytest.mark.parametrize("case", [(1025, 6700, 208), (1000, 2100, 80), (100, 9900, 144), (65, 9900, 336), (64, 9900, 64), (17, 4200, 80), (40, 16400, 129), (50, 2500, 272),
                                  (20, 3000, 513), (2, 8200, 1100), (16, 100, 3500), (9, 40, 6000),
                                  (1030, 4100, 201), (2050, 2050, 63), (70, 2200, 1030), (300, 1000, 15), (129, 1100, 130)], ids=str)
def test_matmul_of_each_kernel(ops, ref, case):
    M, N, K = case
    g = torch.Generator().manual_seed(M + 3 * N + 5 * K)
    a = torch.randint(-128, 128, (M, K), dtype=torch.int8, generator=g)
    w = torch.randint(-128, 128, (N, K), dtype=torch.int8, generator=g)
    sa, sw = torch.rand(M, generator=g) * 1e-3, torch.rand(N, generator=g) * 1e-2
    want = ref.matmul_int8_ref(a, sa, w, sw)
    out = ops._matmul_int8_fwd(gpu(a), gpu(sa), gpu(w), gpu(sw), out_dtype=torch.float32)
    close(out, want, 4 * 2.0 ** -24 * want.abs() + 2.0 ** -120)


@pytest.mark.parametrize("lead", [0, 1, 16])
def test_matmul_of_views(ops, ref, lead):
    # rows inside wider ones, at aligned and at odd addresses; leading dimensions of any number
    g = torch.Generator().manual_seed(lead)
    for M, N, K in ((300, 1030, 256), (40, 70, 96), (2, 40, 512)):
        a, w = (torch.randint(-128, 128, (n, K + 32), generator=g, dtype=torch.int64).to(torch.int8)[:, lead:lead + K] for n in (M, N))
        sa, sw = torch.rand(M, generator=g), torch.rand(N, generator=g)
        want = ref.matmul_int8_ref(a, sa, w, sw)
        out = ops._matmul_int8_fwd(gpu(a), gpu(sa), gpu(w), gpu(sw), out_dtype=torch.float32)
        close(out, want, 4 * 2.0 ** -24 * want.abs() + 2.0 ** -120)
        if M % 2 == 0:
            out = ops._matmul_int8_fwd(gpu(a).unflatten(0, (2, M // 2)), gpu(sa).view(2, -1), gpu(w), gpu(sw), out_dtype=torch.float32)
            close(out.flatten(0, 1), want, 4 * 2.0 ** -24 * want.abs() + 2.0 ** -120)


# ---- common ---------------------------------------------------------------------------------------------------------

def all_calls(ops, g):
    """One call of each operator on small inputs, as functions without arguments."""
    s = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, 2, 600, 2, 64, 128, 1, torch.bfloat16).items()}
    one = {k: v[:, 0].contiguous() if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items() if k != "initial_states"}
    x, w = gpu(randn(g, 2, 50, 96, dtype=torch.bfloat16)), gpu(randn(g, 96, 4, dtype=torch.bfloat16))
    conv_state, scan_state = gpu(randn(g, 2, 3, 96, dtype=torch.bfloat16).transpose(1, 2)), gpu(randn(g, 2, 2, 64, 128))
    a = gpu(torch.randint(-128, 128, (300, 256), generator=g).to(torch.int8))
    sa = gpu(torch.rand(300, generator=g))
    rows, gain = gpu(randn(g, 300, 256, dtype=torch.bfloat16)), gpu(randn(g, 256))
    return {
        "short_conv": lambda: ops._short_conv_fwd(x, w), "scan": lambda: ops._ssd_scan_fwd(**s),
        "short_conv_step": lambda: (ops._short_conv_step(x[:, 0], conv_state, w), conv_state),
        "scan_step": lambda: (ops._ssd_scan_step(**one, states=scan_state), scan_state),
        "norm": lambda: ops._norm_fwd(rows, gain, int8=True)[:2], "matmul": lambda: (ops._matmul_int8_fwd(a, sa, a, sa),),
    }


def test_calls_on_another_stream_and_in_a_graph(ops):
    for name in all_calls(ops, torch.Generator().manual_seed(1)):
        fresh = lambda: all_calls(ops, torch.Generator().manual_seed(1))[name]  # noqa: E731
        call = fresh()
        eager = [[t.clone() for t in call()] for _ in range(4)]
        call = fresh()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            side = [[t.clone() for t in call()] for _ in range(4)]
        torch.cuda.current_stream().wait_stream(stream)
        for i in range(4):
            assert all(torch.equal(p, q) for p, q in zip(eager[i], side[i])), name
        call = fresh()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(eager[i], out)), (name, i)
            torch.ones(1000, device="cuda").mul_(2)
            torch.cuda.synchronize()


def test_results_do_not_depend_on_the_run(ops):
    for name, call in all_calls(ops, torch.Generator().manual_seed(2)).items():
        if name.endswith("step"):
            continue
        want = [t.clone() for t in call()]
        for _ in range(5):
            assert all(torch.equal(p, q) for p, q in zip(want, call())), name


# ---- offsets beyond 32 bits -------------------------------------------------------------------------------------------

FAR = (1 << 31) + 4096


def far(t, dim, stride=FAR):
    """The same values with this element stride along dim, in a buffer of that size"""
    buf = torch.empty((t.shape[dim] - 1) * stride + t.numel() + 16, device="cuda", dtype=t.dtype)
    strides = list(t.stride())
    strides[dim] = stride
    view = buf.as_strided(t.shape, strides)
    return view.copy_(t)


def test_rows_far_apart(ops):
    g = torch.Generator(device="cuda").manual_seed(31)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    i8 = lambda *s: torch.randint(-128, 128, s, device="cuda", dtype=torch.int8, generator=g)  # noqa: E731
    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)  # noqa: E731
    x, w, bias = rn(2, 40, 64).bfloat16(), rn(64, 4).bfloat16(), rn(64).bfloat16()
    assert same(ops._short_conv_fwd(x, w, bias), ops._short_conv_fwd(far(x, 0), w, bias))
    x, r, w = rn(2, 512).bfloat16(), rn(2, 512).bfloat16(), rn(512)
    assert same(ops._norm_fwd(x, w, residual=r, int8=True), ops._norm_fwd(far(x, 0), w, residual=far(r, 0), int8=True))
    for M, N in ((2, 40), (200, 2), (70, 3000)):
        a, w, sa, sw = i8(M, 256), i8(N, 256), rn(M).abs(), rn(N).abs()
        few, step = (a, w)[N < M], (FAR, (1 << 26) + 32)[M == 70]
        there = far(few, 0, step)
        assert torch.equal(ops._matmul_int8_fwd(a, sa, w, sw), ops._matmul_int8_fwd(*((a, sa, there, sw) if few is w else (there, sa, w, sw))))


@pytest.mark.parametrize("case", [(8, 100, torch.float32), (4, 33, torch.bfloat16), (96, 300, torch.bfloat16)], ids=str)
def test_ssd_scan_of_rows_far_apart(ops, case):
    H, L, dtype = case
    g = torch.Generator(device="cuda").manual_seed(32)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, z, B, C = rn(2, L, H, 64).to(dtype), rn(2, L, H, 64).to(dtype), 0.3 * rn(2, L, 1, 128), 0.3 * rn(2, L, 1, 128)
    B, C, dt, A = B.to(dtype), C.to(dtype), rn(2, L, H) - 3, -rn(H).abs()
    y, last = ops._ssd_scan_fwd(x, dt, A, B, C, z=z, dt_softplus=True)
    y2, last2 = ops._ssd_scan_fwd(far(x, 0), far(dt, 0), A, far(B, 0), far(C, 0), z=far(z, 0), dt_softplus=True)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    # tokens far apart, which only the kernel for any size takes
    y, last = ops._ssd_scan_fwd(x[:1, :33].float(), dt[:1, :33], A, B[:1, :33].float(), C[:1, :33].float(), dt_softplus=True)
    y2, last2 = ops._ssd_scan_fwd(far(x[:1, :33].float(), 1, (1 << 26) + 4096), dt[:1, :33], A, B[:1, :33].float(), C[:1, :33].float(), dt_softplus=True)
    assert torch.equal(y, y2) and torch.equal(last, last2)


def test_steps_in_a_large_pool(ops):
    # the last slots lie behind 2^31 elements
    g = torch.Generator(device="cuda").manual_seed(33)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    H, P, N, slots = 80, 64, 128, 3500
    pool = torch.zeros(slots, H, P, N, device="cuda")
    pool[-1] = rn(H, P, N)
    small = pool[-2:].clone()
    x, B, C, dt, A = rn(2, H, P).bfloat16(), rn(2, 1, N).bfloat16(), rn(2, 1, N).bfloat16(), rn(2, H) - 3, -rn(H).abs()
    at = torch.tensor([slots - 1, slots - 2], dtype=torch.int32, device="cuda")
    y = ops._ssd_scan_step(x, dt, A, B, C, pool, dt_softplus=True, slots=at)
    assert torch.equal(y, ops._ssd_scan_step(x, dt, A, B, C, small, dt_softplus=True, slots=at - (slots - 2)))
    assert torch.equal(pool[-2:], small) and not bool(pool[:4].any())
    del pool
    pool = torch.zeros(160000, 3, 5376, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    pool[-1] = rn(5376, 3).bfloat16()
    small = pool[-1:].contiguous()
    x, w = rn(1, 5376).bfloat16(), rn(5376, 4).bfloat16()
    y = ops._short_conv_step(x, pool, w, slots=torch.tensor([159999], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, ops._short_conv_step(x, small, w)) and torch.equal(pool[-1:], small)


def test_larger_calls_on_another_stream_and_in_a_graph(ops):
    # as above, for the kernels that small inputs do not reach
    assert on_bf16_instructions(2, 1500, 96, 64, 128, 1)
    g = torch.Generator().manual_seed(41)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, 2, 1500, 96, 64, 128, 1, torch.bfloat16, init=True).items()}
    conv = gpu(randn(g, 2, 700, 256, dtype=torch.bfloat16)), gpu(randn(g, 256, 4, dtype=torch.bfloat16))
    q, s = gpu(torch.randint(-128, 128, (1400, 256), dtype=torch.int8, generator=g)), gpu(torch.rand(1400, generator=g))
    norm = gpu(randn(g, 1400, 256, dtype=torch.bfloat16)), gpu(torch.rand(256, generator=g))

    def calls():
        out, scale, _ = ops._norm_fwd(*norm, int8=True)
        return [*ops._ssd_scan_fwd(**a), *ops._short_conv_fwd(*conv), out, scale, ops._matmul_int8_fwd(q, s, q[:300], s[:300])]

    want = calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert all(torch.equal(x, y) for x, y in zip(calls(), want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(calls(), want))
