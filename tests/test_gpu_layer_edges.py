"""The operators around the state path where they are easiest to get wrong: what the workgroups of one launch may share, decays of very
different strength, values that are not finite, tensors of several types.  Inputs and bounds as in test_gpu_layer.py."""
import ctypes

import pytest
import torch

from test_gpu_layer import close, gpu, ops, randn, ref, rounded, scan_bounds, scan_inputs  # noqa: F401

pytestmark = pytest.mark.gpu

RECORD = 5 * 64      # words of the steps of 64 tokens


def scan_through_c(a, lengths=None, fill=None, strided=None):
    """A bf16 scan through the C entry with a workspace of the caller's: y, final states, the workspace's words."""
    from ssd_amd import _lib
    from ssd_amd.layer import _arg as T
    b, L, H, P = a["x"].shape
    G, N = a["B"].shape[2:]
    dims = _lib.dims_arg(b, L, H, P, N, G, 0, 0)
    nbytes = int(_lib.load().ssd_scan_workspace_bytes(dims, _lib.SSD_BF16))
    room = torch.full((nbytes // 4,), 0.0 if fill is None else fill, device="cuda")
    y, fin = torch.empty(b, L, H, P, device="cuda", dtype=torch.bfloat16), torch.empty(b, H, P, N, device="cuda")
    rc = _lib.load().ssd_scan_fwd(T(a["x"]), T(a["dt"]), T(a["A"]), T(a["B"]), T(a["C"]), T(a["D"]), T(a["z"]), T(a["dt_bias"]), T(a["initial_states"]),
                                  T(None), T(lengths), T(y), T(fin), dims, 1, 0.0, float("inf"), ctypes.c_void_p(room.data_ptr()), nbytes,
                                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    torch.cuda.synchronize()
    return y, fin, room


# ---- segments of a row -----------------------------------------------------------------------------------------------

# rows cut into two and three segments, which read what those in front of them leave by themselves
FEW_SEGMENTS = [(1, 512, 80, 64, 128, 1, None, 3), (2, 500, 80, 64, 128, 2, [500, 0], 3), (8, 384, 24, 64, 128, 1, [0, 384, 1, 64, 100, 300, 383, 0], 3),
                (3, 1000, 128, 64, 128, 1, [1000, 40, 0], 2)]


@pytest.mark.parametrize("case", FEW_SEGMENTS, ids=str)
def test_a_launch_leaves_alone_what_its_segments_read(ops, ref, case):  # noqa: F811
    # what the first segment adds to a state of zero and the factor on what enters it stand in the workspace from the launch in front; the
    # launch with y reads them in its later segments, so its first one may not put anything in their place
    b, L, H, P, N, G, lengths, segments = case
    g = torch.Generator().manual_seed(L + H)
    a = scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    on = {k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}
    mark = -123.0
    y, fin, room = scan_through_c(on, gpu(n), fill=mark)
    rows, chunks = b * H, (L + 63) // 64
    states = room[:rows * segments * P * N].view(b, H, segments, P, N)[:, :, 0]
    factors = room[rows * segments * P * N:][:rows * segments].view(b, H, segments).double().cpu()
    # (that the workspace is laid out so: the last segment leaves nothing, the others do)
    assert bool((factors[:, :, -1] == mark).all()) and not bool((factors[:, :, :-1] == mark).any())
    factors = factors[:, :, 0]
    first = min(L, 64 * ((chunks + segments - 1) // segments))
    head = {k: v[:, :first] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    m = None if n is None else n.clamp(max=first)
    want, magnitudes = ref.ssd_scan_ref(**dict(head, initial_states=None), lengths=m)[1::2]
    close(states, want, scan_bounds(want, magnitudes, first, torch.bfloat16), "what the first segment adds")
    d = ref.delta_ref(head["dt"], a["dt_bias"], True)
    if m is not None:
        d = d * (torch.arange(first)[None] < m[:, None])[..., None]
    passed = torch.exp((d * a["A"].double()).sum(1))
    # a sum of up to 512 terms of 32 bits in front of an exponential
    close(factors, passed, passed * (1024 * 2.0 ** -24) * (1 - passed.log().clamp(min=-100)) + 2.0 ** -126, "factor")
    if lengths is not None:
        none = torch.tensor(lengths) == 0
        assert torch.equal(fin.cpu()[none], a["initial_states"][none])


@pytest.mark.parametrize("case", FEW_SEGMENTS, ids=str)
def test_a_scan_beside_other_work_is_the_same(ops, case):  # noqa: F811
    # another stream holds compute units for milliseconds: workgroups of the scan start when some of them become free
    b, L, H, P, N, G, lengths, _ = case
    g = torch.Generator().manual_seed(L)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True).items()}
    n = None if lengths is None else gpu(torch.tensor(lengths, dtype=torch.int32))
    y, last = ops._ssd_scan_fwd(**a, lengths=n)
    other = torch.randn(8192, 8192, device="cuda").bfloat16()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            product = other @ other
    again = [ops._ssd_scan_fwd(**a, lengths=n) for _ in range(20)]
    torch.cuda.synchronize()
    del product
    for y2, last2 in again:
        assert torch.equal(y2, y) and torch.equal(last2, last)


# ---- decays ----------------------------------------------------------------------------------------------------------

# which of a chunk's 64 tokens let (next to) nothing pass; the others decay by e^-0.001
STRONG = {"front": range(40), "middle": range(10, 50), "second half": range(32, 55), "every other": range(0, 64, 2), "last": range(60, 64), "first half": range(32)}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("strength", [30.0, 100.0])
@pytest.mark.parametrize("where", STRONG)
def test_weak_decays_behind_strong_ones(ops, ref, where, strength, dtype):  # noqa: F811
    # what passes between two tokens is an exponential of a difference of sums that the strong ones make large; x is smaller where the
    # step is larger, so that all tokens add alike
    b, L, H, P, N = 4, 300, 128, 8, 64
    g = torch.Generator().manual_seed(int(strength))
    a = scan_inputs(g, b, L, H, P, N, 1, dtype, init=True)
    marked = torch.zeros(64, dtype=torch.bool)
    marked[list(STRONG[where])] = True
    marked = marked.repeat(5)[:L]
    step = torch.where(marked, torch.full((L,), strength), torch.full((L,), 1e-3))
    a.update(dt=(step[None, :, None] * (1 + 0.1 * torch.rand(b, L, H, generator=g))), dt_bias=None, dt_softplus=False, A=-(0.5 + torch.rand(H, generator=g)),
             x=(a["x"].float() * torch.where(marked, 1e-3 / strength, 1.0)[None, :, None, None]).to(dtype))
    want, final, size, final_size = ref.ssd_scan_ref(**a)
    y, last = ops._ssd_scan_fwd(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()})
    close(y, want, scan_bounds(want, size, L, dtype), "y")
    close(last, final, scan_bounds(final, final_size, L, dtype) - rounded(final, dtype) + rounded(final, torch.float32), "final states")


# ---- a kernel and its plan -------------------------------------------------------------------------------------------

# sizes that the bf16 kernel cuts into segments and the other one, which calls of odd strides run on, does not (1), or into more of them (4)
@pytest.mark.parametrize("case", [(3, 1000, 128, 64, 128, 1, 1), (2, 1500, 128, 64, 128, 1, 1), (4, 500, 24, 64, 128, 1, 4)], ids=str)
def test_rows_at_odd_addresses_are_not_cut_by_the_other_kernels_plan(case):
    b, L, H, P, N, G, segments = case
    g = torch.Generator().manual_seed(L)
    a = scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True)
    odd = randn(g, b, L, H * P, dtype=torch.bfloat16, lead=1).unflatten(-1, (H, P))
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in dict(a, x=odd).items()}
    mark = -123.0
    y, last, room = scan_through_c(a, fill=mark)
    states = room[:b * H * segments * P * N].view(b, H, segments, P, N)
    if segments == 1:
        assert bool((room == mark).all())
    else:
        # all segments but the last were put there, and no more
        assert not bool((states[:, :, :-1] == mark).any()) and bool((states[:, :, -1] == mark).all())
    straight, last2, _ = scan_through_c(dict(a, x=odd.contiguous().cuda()))
    # the same values on the other kernel: its operands of two bf16 parts, seen through a rounding to bf16
    assert float((last - last2).norm()) <= 3 * 2.0 ** -16 * float(last.norm())
    assert float((y.float() - straight.float()).norm()) <= 2.0 ** -8 * float(straight.float().norm())


# ---- norm ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(3, 5), (4, 512), (1030, 1000), (1025, 2560), (3, 5120), (2, 12001)], ids=str)
def test_norm_to_8_bits_keeps_what_is_not_finite_in_the_weight(ops, shape, dtype):  # noqa: F811
    rows, D = shape
    g = torch.Generator().manual_seed(D)
    x = gpu(randn(g, rows, D, dtype=dtype))
    for junk in (float("nan"), float("inf"), -float("inf")):
        for weight_type in (dtype, torch.float32):
            w = torch.rand(D, generator=g).to(weight_type) + 0.5
            w[D // 2] = junk
            q, scale, _ = ops._norm_fwd(x, gpu(w), int8=True)
            assert bool(scale.isnan().all()), (junk, weight_type)
        y, _, _ = ops._norm_fwd(x, gpu(w))
        assert not bool(y[:, D // 2].isfinite().any()) and bool(y[:, :D // 2].isfinite().all())


@pytest.mark.parametrize("mode", ["", "residual", "gate"])
@pytest.mark.parametrize("shape", [(3, 5), (4, 512), (1030, 1000), (3, 5120), (2, 12001)], ids=str)
def test_norm_of_rows_of_zeros_without_eps(ops, ref, shape, mode):  # noqa: F811
    rows, D = shape
    g = torch.Generator().manual_seed(D)
    for dtype in (torch.float32, torch.bfloat16):
        x, other, w = randn(g, rows, D, dtype=dtype), randn(g, rows, D, dtype=dtype), torch.rand(D, generator=g) + 0.5
        x[1] = 0
        if mode == "residual":
            other[1] = 0
        kw = {"residual": other} if mode == "residual" else {"z": other} if mode == "gate" else {}
        q, scale, _ = ops._norm_fwd(gpu(x), gpu(w), int8=True, eps=0.0, **{k: gpu(v) for k, v in kw.items()})
        assert not bool(q[1].any()) and float(scale[1]) == 0.0
        want = ref.norm_ref(x, w, eps=0.0, **kw)[0]
        live = [i for i in range(rows) if i != 1]
        step = want[live].abs().amax(-1, keepdim=True) / 127
        # the bound of test_norm
        near = (D / 2 / 64 + 32) * 2.0 ** -24
        close(q.double()[live] * scale.double()[live][:, None], want[live], (0.5 + 127 * near + 1e-4) * step, "8 bits")


# ---- several types in one call ---------------------------------------------------------------------------------------

TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm_of_16_bits_with_a_residual_in_fp32(ops, ref, dtype, int8):  # noqa: F811
    # the residual stream of a model is often kept in fp32: it may not lose bits on its way through a layer
    g = torch.Generator().manual_seed(3)
    x, residual, w = randn(g, 40, 768, dtype=dtype, lead=1), 4 * randn(g, 40, 768), torch.rand(768, generator=g) + 0.5
    want, total = ref.norm_ref(x, w, residual)
    out, scale, after = ops._norm_fwd(gpu(x), gpu(w), residual=gpu(residual), int8=int8)
    assert after.dtype == torch.float32
    close(after, total, 2.0 ** -24 * total.abs(), "residual")
    near = (768 / 2 / 64 + 32) * 2.0 ** -24
    if int8:
        step = want.abs().amax(-1, keepdim=True) / 127
        close(out.double() * scale.double()[:, None], want, (0.5 + 127 * near + 1e-4) * step, "8 bits")
    else:
        assert out.dtype == dtype
        close(out, want, rounded(want, dtype) * 1.01 + near * want.abs(), "out")
    # a gate in fp32, and one of the other type of 16 bits
    for other in (torch.float32, TYPES[dtype == TYPES[0]]):
        z = randn(g, 40, 768).to(other)
        want, _ = ref.norm_ref(x, w, None, z)
        out, scale, _ = ops._norm_fwd(gpu(x), gpu(w), z=gpu(z), int8=int8)
        if int8:
            out = out.double() * scale.double()[:, None]
            step = want.abs().amax(-1, keepdim=True) / 127
            close(out, want, (0.5 + 127 * near + 1e-4) * step, "8 bits, gate")
        else:
            assert out.dtype == dtype
            close(out, want, rounded(want, dtype) * 1.01 + near * want.abs() + 2.0 ** -120, "gate")


@pytest.mark.parametrize("wide", ["x", "B", "C", "z", "BCz"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_of_several_types(ops, ref, dtype, wide):  # noqa: F811
    g = torch.Generator().manual_seed(5)
    b, L, H, P, N = 2, 130, 4, 64, 128
    a = scan_inputs(g, b, L, H, P, N, 2, torch.float32, init=True)
    for key in ("x", "B", "C", "z"):
        a[key] = a[key] if key in wide else a[key].to(dtype)
    want, final, size, final_size = ref.ssd_scan_ref(**a)
    y, last = ops._ssd_scan_fwd(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()})
    assert y.dtype == a["x"].dtype
    # the call runs in fp32; a single rounding to x's type at its end
    exact = scan_bounds(want, size, L, torch.float32)
    close(y, want, exact + rounded(want, y.dtype) * 1.01, "y")
    close(last, final, scan_bounds(final, final_size, L, torch.float32), "final states")
    one = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items() if k != "initial_states"}
    states = a["initial_states"].clone()
    want, after, size = ref.ssd_scan_step_ref(**one, states=states)
    there = gpu(states)
    y = ops._ssd_scan_step(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in one.items()}, states=there)
    assert y.dtype == a["x"].dtype
    close(y, want, rounded(want, y.dtype) * 1.01 + 160 * 2.0 ** -23 * size + 2.0 ** -126, "step")
    close(there, after, 8 * 2.0 ** -23 * (after.abs() + states.abs() + 1))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_conv_with_states_of_another_type(ops, ref, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(6)
    for L in (1, 2, 40):
        for given, kept in ((dtype, torch.float32), (torch.float32, dtype)):
            x, w, state = randn(g, 2, L, 24, dtype=given), randn(g, 24, 4), randn(g, 2, 3, 24, dtype=kept).transpose(1, 2)
            want, final, size = ref.short_conv_ref(x, w, None, True, state)
            y, last = ops._short_conv_fwd(gpu(x), gpu(w), initial_states=gpu(state))
            assert y.dtype == given and last.dtype == torch.float32
            close(y, want, rounded(want, given) * 1.01 + (4 + 8) * 2.0 ** -23 * size + 2.0 ** -126, "y")
            assert torch.equal(last.double().cpu(), final)


# ---- whole numbers of 64 bits ----------------------------------------------------------------------------------------

def test_slots_and_lengths_of_64_bits(ops):  # noqa: F811
    # a slot outside the pool is padding and a length beyond the row the row's, whatever their lower 32 bits say
    g = torch.Generator().manual_seed(8)
    a = {k: gpu(v) if torch.is_tensor(v) else v for k, v in scan_inputs(g, 3, 20, 2, 16, 32, 1, torch.bfloat16, init=True).items()}
    narrow, wide = (torch.tensor(v).cuda() for v in ([7, 20, 0], [7, (1 << 32) + 3, -(1 << 32) + 5]))
    x, w = gpu(randn(g, 3, 20, 24, dtype=torch.bfloat16)), gpu(randn(g, 24, 4))
    for call in (lambda n: ops._ssd_scan_fwd(**a, lengths=n), lambda n: ops._short_conv_fwd(x, w, lengths=n)):
        assert all(torch.equal(p, q) for p, q in zip(call(narrow.int()), call(wide)))
    narrow, wide = (torch.tensor(v).cuda() for v in ([1, -1, 4], [1, (1 << 32) + 2, -(1 << 33) + 3]))
    one = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items() if k != "initial_states"}
    pool, states = gpu(randn(g, 4, 2, 16, 32)), gpu(randn(g, 4, 3, 24, dtype=torch.bfloat16).transpose(1, 2))
    for call, s in ((lambda n, s: ops._ssd_scan_step(**one, states=s, slots=n), pool), (lambda n, s: ops._short_conv_step(x[:, 0], s, w, slots=n), states)):
        p, q = s.clone(), s.clone()
        assert torch.equal(call(narrow.int(), p), call(wide, q)) and torch.equal(p, q)
        assert torch.equal(q[[0, 2, 3]], s[[0, 2, 3]])


# ---- very long rows --------------------------------------------------------------------------------------------------

def test_tokens_behind_the_length_of_a_very_long_row(ops):  # noqa: F811
    # one segment (no workspace) of more than 2^25 tokens behind the row's last one: 2^31 places of 64 rows
    from ssd_amd import _lib
    from ssd_amd.layer import _arg as T
    L = (1 << 25) + 5
    x, B = (torch.ones(1, L, 1, 1, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    y, fin, dt, A = torch.ones_like(x), torch.empty(1, 1, 1, 1, device="cuda"), torch.ones(1, L, 1, device="cuda", dtype=torch.bfloat16), -torch.ones(1, device="cuda")
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    rc = _lib.load().ssd_scan_fwd(T(x), T(dt), T(A), T(B), T(B), T(None), T(None), T(None), T(None), T(None), T(n), T(y), T(fin),
                                  _lib.dims_arg(1, L, 1, 1, 1, 1, 0, 0), 0, 0.0, float("inf"), None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    assert bool(y[:, :3].ne(0).all()) and not bool(y[:, 3:].any())
    e = 2.718281828459045 ** -1
    assert abs(float(fin) - (1 + e + e * e)) < 1e-5


# ---- values that are not finite --------------------------------------------------------------------------------------

# one segment, three and many, with the first one in front of the others, and the kernel for any size
INFINITE = [(8, 190, 40, 64, 128, 4), (4, 300, 128, 8, 64, 1), (2, 500, 80, 16, 64, 2), (2, 1100, 80, 32, 128, 1), (4, 2500, 128, 8, 64, 8), (1, 150, 3, 20, 40, 1)]


@pytest.mark.parametrize("marks", [False, True])
@pytest.mark.parametrize("key", ["x", "B", "C", "initial_states"])
@pytest.mark.parametrize("case", INFINITE, ids=str)
def test_scan_of_infinities(ops, ref, case, key, marks):  # noqa: F811
    # they reach what they reach in the recurrence, with the sign that they have there
    b, L, H, P, N, G = case
    g = torch.Generator().manual_seed(L)
    a = scan_inputs(g, b, L, H, P, N, G, torch.bfloat16, init=True)
    a["x"], a["B"], a["C"] = (t + torch.where(t >= 0, 2.0 ** -6, -2.0 ** -6).to(t.dtype) for t in (a["x"], a["B"], a["C"]))      # no zeros
    a["A"] = a["A"] * 0.05      # what enters a row still counts at its end
    a["initial_states"] += torch.where(a["initial_states"] >= 0, 0.01, -0.01)
    t = a[key]
    for row, at, sign in ((0, 0, 1), (0, L // 2, -1), (b - 1, L - 1, 1)):
        if key == "initial_states":
            t[row, at % H, at % P, at % N] = sign * float("inf")
        else:
            t[row, at, at % t.shape[2], at % t.shape[3]] = sign * float("inf")
    seq, n = None, None
    if marks:
        # a sequence starts in the chunk where they are, behind them
        seq = torch.zeros(b, L, dtype=torch.int32)
        seq[0, 50:], seq[0, min(L - 1, L // 2 + 3):], n = 1, 2, torch.tensor([L - i for i in range(b)], dtype=torch.int32)
    want, final, size, final_size = ref.ssd_scan_ref(**a, seq_idx=seq, lengths=n)
    assert bool(want.isinf().any() or final.isinf().any() or want.isnan().any())
    y, last = ops._ssd_scan_fwd(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()}, seq_idx=gpu(seq), lengths=gpu(n))
    for got, exact, bound in ((y, want, scan_bounds(want, size, L, torch.bfloat16)), (last, final, scan_bounds(final, final_size, L, torch.bfloat16))):
        got = got.double().cpu()
        fine = exact.isfinite()
        assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), exact.isnan()) and torch.equal(got.isposinf(), exact.isposinf())
        close(got[fine], exact[fine], bound[fine])


# rows whose segments let less than the smallest number of fp32 pass, and one of a single segment
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("case", [(1, 2000, 16, 64, 128, 1), (4, 2500, 128, 8, 64, 8), (1, 1900, 4, 8, 16, 1), (1, 120, 4, 16, 32, 1)], ids=str)
def test_infinities_that_everything_else_has_decayed_around(ops, ref, case, dtype):  # noqa: F811
    b, L, H, P, N, G = case
    g = torch.Generator().manual_seed(L)
    a = scan_inputs(g, b, L, H, P, N, G, dtype, init=True)
    a["C"] = a["C"].abs() + 2.0 ** -6
    a["dt"], a["dt_softplus"], a["dt_bias"] = torch.full((b, L, H), 0.25).to(dtype), False, None
    a["A"] = -16 * torch.rand(H, generator=g) - 1      # up to e^-4.25 a token
    a["initial_states"][0, 0, 1, 2] = float("inf")
    a["initial_states"][0, H - 1, P - 1, 0] = -float("inf")
    want, final, size, final_size = ref.ssd_scan_ref(**a)
    assert int(final.isinf().sum()) == 2 and not bool(final.isnan().any()) and not bool(want.isnan().any())
    y, last = ops._ssd_scan_fwd(**{k: gpu(v) if torch.is_tensor(v) else v for k, v in a.items()})
    for got, exact, bound in ((y, want, scan_bounds(want, size, L, dtype)), (last, final, scan_bounds(final, final_size, L, dtype))):
        got = got.double().cpu()
        fine = exact.isfinite()
        assert torch.equal(got.isposinf(), exact.isposinf()) and torch.equal(got.isneginf(), exact.isneginf()) and not bool(got.isnan().any())
        close(got[fine], exact[fine], bound[fine])
