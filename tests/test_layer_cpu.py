"""The operators around the state path, without a GPU: what their wrappers and C entry points refuse, and that nothing is computed on
a CPU."""
import ctypes

import pytest
import torch

import ssd_amd as ops
from ssd_amd import _lib
from ssd_amd.layer import _arg as T

b16, i8 = torch.bfloat16, torch.int8


def scan_args(b=1, L=8, H=4, P=8, N=16, G=2):
    return dict(x=torch.zeros(b, L, H, P), dt=torch.zeros(b, L, H), A=torch.zeros(H), B=torch.zeros(b, L, G, N), C=torch.zeros(b, L, G, N))


def step_args(b=2, H=4, P=8, N=16, G=2):
    return dict(x=torch.zeros(b, H, P), dt=torch.zeros(b, H), A=torch.zeros(H), B=torch.zeros(b, G, N), C=torch.zeros(b, G, N),
                states=torch.zeros(b, H, P, N))


def test_nothing_is_computed_on_a_cpu():
    x, w = torch.zeros(1, 8, 16), torch.zeros(16, 4)
    for call in (lambda: ops._short_conv_fwd(x, w), lambda: ops._short_conv_step(x[0, :1], torch.zeros(1, 16, 3), w),
                 lambda: ops._ssd_scan_fwd(**scan_args()), lambda: ops._ssd_scan_step(**step_args()),
                 lambda: ops._norm_fwd(x, torch.zeros(16)), lambda: ops._norm_fwd(x, torch.zeros(16), int8=True),
                 lambda: ops._matmul_int8_fwd(x[0].to(i8), torch.zeros(8), x[0].to(i8), torch.zeros(8))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_wrappers_refuse_what_does_not_fit():
    x, w = torch.zeros(2, 8, 16), torch.zeros(16, 4)
    wrong = [
        lambda: ops._short_conv_fwd(x, torch.zeros(15, 4)), lambda: ops._short_conv_fwd(x, torch.zeros(16, 5)),
        lambda: ops._short_conv_fwd(x, w, torch.zeros(4)), lambda: ops._short_conv_fwd(x, w, initial_states=torch.zeros(2, 16, 4)),
        lambda: ops._short_conv_fwd(x, w, seq_idx=torch.zeros(2, 7, dtype=torch.int32)), lambda: ops._short_conv_fwd(x, w, lengths=torch.zeros(1, dtype=torch.int32)),
        lambda: ops._short_conv_fwd(x.double(), w),
        lambda: ops._short_conv_step(x[0], torch.zeros(8, 16, 2), w), lambda: ops._short_conv_step(x[0], torch.zeros(7, 16, 3), w),
        lambda: ops._short_conv_step(x[0], torch.zeros(8, 16, 3, dtype=b16), w), lambda: ops._short_conv_step(x[0], torch.zeros(8, 16, 3), w, slots=torch.zeros(7)),
        lambda: ops._norm_fwd(x, torch.zeros(15)), lambda: ops._norm_fwd(x, torch.zeros(16), residual=x, z=x), lambda: ops._norm_fwd(x, torch.zeros(16), z=x[0]),
        lambda: ops._norm_fwd(x.to(i8), torch.zeros(16)),
        lambda: ops._matmul_int8_fwd(x[0], torch.zeros(8), w.to(i8), torch.zeros(16)),
        lambda: ops._matmul_int8_fwd(x[0].to(i8), torch.zeros(8), w.to(i8), torch.zeros(16)),
        lambda: ops._matmul_int8_fwd(x[0].to(i8), torch.zeros(7), x[0].to(i8), torch.zeros(8)),
        lambda: ops._matmul_int8_fwd(x[0].to(i8), torch.zeros(8), x[0].to(i8), torch.zeros(8), out_dtype=torch.int32),
        lambda: ops._matmul_int8_fwd(torch.zeros(1, 131072, dtype=i8), torch.zeros(1), torch.zeros(1, 131072, dtype=i8), torch.zeros(1)),
    ]
    a, s = scan_args(), step_args()
    for key, value in dict(dt=torch.zeros(1, 8, 3), A=torch.zeros(5), B=torch.zeros(1, 8, 3, 16), C=torch.zeros(1, 8, 2, 15), D=torch.zeros(3), z=torch.zeros(1, 8, 4, 7),
                           dt_bias=torch.zeros(3), initial_states=torch.zeros(1, 4, 8, 15), seq_idx=torch.zeros(1, 7), lengths=torch.zeros(2)).items():
        wrong.append(lambda key=key, value=value: ops._ssd_scan_fwd(**{**a, key: value}))
    wrong.append(lambda: ops._ssd_scan_fwd(**scan_args(N=257)))
    for key, value in dict(dt=torch.zeros(2, 3), A=torch.zeros(5), B=torch.zeros(2, 3, 16), C=torch.zeros(2, 2, 15), states=torch.zeros(3, 4, 8, 16), D=torch.zeros(3),
                           z=torch.zeros(2, 4, 7), dt_bias=torch.zeros(3), slots=torch.zeros(3)).items():
        wrong.append(lambda key=key, value=value: ops._ssd_scan_step(**{**s, key: value}))
    wrong.append(lambda: ops._ssd_scan_step(**{**s, "states": torch.zeros(2, 4, 8, 16).half()}))
    wrong.append(lambda: ops._ssd_scan_step(**{**s, "states": torch.zeros(2, 4, 16, 8).transpose(2, 3)}))
    for i, call in enumerate(wrong):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")


def test_c_entry_points_refuse_in_front_of_any_device_work():
    lib = _lib.load()
    none = T(None)
    NULL, SHAPE, DTYPE, STRIDE = -1, -2, -3, -4
    x, w, bias, fin, y = torch.zeros(1, 8, 16), torch.zeros(16, 4), torch.zeros(16), torch.zeros(1, 16, 3), torch.zeros(1, 8, 16)
    conv = lambda x=x, w=w, bias=bias, y=y, fin=fin, b=1, L=8, D=16, K=4: lib.ssd_short_conv_fwd(  # noqa: E731
        T(x), T(w), T(bias), none, none, none, T(y), T(fin), b, L, D, K, 1, None)
    assert conv(K=5) == SHAPE and conv(K=0) == SHAPE and conv(D=0) == SHAPE and conv(L=-1) == SHAPE and conv(b=-1) == SHAPE
    assert conv(x=None) == NULL and conv(w=None) == NULL and conv(fin=None) == NULL and conv(y=None) == NULL and conv(b=0) == 0
    assert conv(y=y.to(b16)) == DTYPE and conv(fin=fin.to(b16)) == DTYPE and conv(w=w.to(i8)) == DTYPE
    assert conv(x=torch.zeros(1, 16, 8).transpose(1, 2)) == STRIDE
    step = lambda x=x[0], s=torch.zeros(8, 16, 3), y=y[0], n=8, K=4: lib.ssd_short_conv_step(T(x), T(s), T(w), none, none, T(y), 8, 16, K, n, 1, None)  # noqa: E731
    assert step(n=-1) == SHAPE and step(K=9) == SHAPE and step(s=None) == NULL and step(s=torch.zeros(8, 16, 3).half()) == DTYPE
    assert step(x=torch.zeros(16, 8).t()) == STRIDE

    a = scan_args()
    fin, y = torch.zeros(1, 4, 8, 16), torch.zeros(1, 8, 4, 8)
    dims = lambda b=1, L=8, H=4, P=8, N=16, G=2: _lib.dims_arg(b, L, H, P, N, G, 0, 0)  # noqa: E731

    def scan(d=dims(), fin=fin, y=y, **kw):
        t = {**a, **kw}
        return lib.ssd_scan_fwd(T(t["x"]), T(t["dt"]), T(t["A"]), T(t["B"]), T(t["C"]), none, T(t.get("z")), none, T(t.get("init")), none, none, T(y), T(fin), d,
                                1, 0.0, 1.0, None, 0, None)
    assert scan(d=dims(N=257)) == SHAPE and scan(d=dims(G=3)) == SHAPE and scan(d=dims(L=-1)) == SHAPE and scan(d=None) == NULL and scan(d=dims(b=0)) == 0
    assert scan(x=None) == NULL and scan(A=None) == NULL and scan(fin=None) == NULL and scan(y=None) == NULL
    assert scan(B=a["B"].to(b16)) == DTYPE and scan(y=y.half()) == DTYPE and scan(fin=fin.half()) == DTYPE and scan(z=y.half()) == DTYPE
    assert scan(init=torch.zeros(1, 4, 16, 8).transpose(2, 3)) == STRIDE and scan(C=torch.zeros(1, 8, 16, 2).transpose(2, 3)) == STRIDE
    s = step_args()

    def scan_step(d=dims(b=2), n=2, **kw):
        t = {**s, **kw}
        return lib.ssd_scan_step(T(t["x"]), T(t["dt"]), T(t["A"]), T(t["B"]), T(t["C"]), none, none, none, T(t["states"]), none, T(t["x"]), d, n, 1, 0.0, 1.0, None)
    assert scan_step(n=-1) == SHAPE and scan_step(d=dims(H=5)) == SHAPE and scan_step(states=None) == NULL and scan_step(dt=None) == NULL
    assert scan_step(states=s["states"].half()) == DTYPE and scan_step(C=s["C"].half()) == DTYPE
    assert scan_step(states=torch.zeros(2, 4, 16, 8).transpose(2, 3)) == STRIDE

    rows, gain, q, scale = torch.zeros(4, 16), torch.zeros(16), torch.zeros(4, 16, dtype=i8), torch.zeros(4)
    norm = lambda x=rows, w=gain, r=None, z=None, out=q, s=scale, ro=None, n=4, D=16: lib.ssd_norm_fwd(T(x), T(w), T(r), T(z), T(out), T(s), T(ro), n, D, 1e-5, None)  # noqa: E731
    assert norm(D=0) == SHAPE and norm(n=-1) == SHAPE and norm(r=rows, z=rows, ro=rows) == SHAPE and norm(n=0) == 0
    assert norm(r=rows) == NULL and norm(ro=rows) == NULL and norm(s=None) == NULL and norm(x=None) == NULL
    assert norm(x=rows.half(), out=rows) == DTYPE and norm(s=scale.half()) == DTYPE and norm(x=q) == DTYPE and norm(z=rows.half()) == DTYPE
    assert norm(z=torch.zeros(16, 4).t()) == STRIDE

    mm = lambda a=q, sa=scale, w=q, sw=scale, bias=None, out=torch.zeros(4, 4), M=4, N=4, K=16: lib.ssd_matmul_fwd(T(a), T(sa), T(w), T(sw), T(bias), T(out), M, N, K, None)  # noqa: E731
    assert mm(K=131072) == SHAPE and mm(M=-1) == SHAPE and mm(M=0) == 0 and mm(a=None) == NULL and mm(sw=None) == NULL and mm(out=None) == NULL
    assert mm(a=rows) == DTYPE and mm(sa=scale.half()) == DTYPE and mm(out=q) == DTYPE and mm(bias=q[0]) == DTYPE
    assert mm(w=torch.zeros(16, 4, dtype=i8).t()) == STRIDE
    # everything in order: only the device is missing here
    if not torch.cuda.is_available():
        assert conv() == step() == scan() == scan_step() == norm() == mm() == -5


def test_workspace_of_a_scan():
    lib = _lib.load()
    bytes_of = lambda *d, t=_lib.SSD_F32: int(lib.ssd_scan_workspace_bytes(_lib.dims_arg(*d, 0, 0), t))  # noqa: E731
    for t in (_lib.SSD_F32, _lib.SSD_BF16):
        assert bytes_of(0, 8, 4, 8, 16, 2, t=t) == 0 and bytes_of(1, 0, 4, 8, 16, 2, t=t) == 0
        assert bytes_of(1, 8, 4, 8, 16, 3, t=t) == 0 and bytes_of(1, 8192, 4, 8, 257, 2, t=t) == 0
    # the segments' states and factors: none for short rows, nor where there is work for every compute unit as it is
    assert bytes_of(1, 100, 4, 64, 128, 2) == 0 and bytes_of(64, 8192, 128, 64, 128, 1) == 0
    n = bytes_of(1, 8192, 4, 64, 128, 1)
    assert n % (4 * 4 * (64 * 128 + 1)) == 0 and 2 <= n // (4 * 4 * (64 * 128 + 1)) <= 8192 // 64
    # on the matrix instructions also a record of the steps per (row, head, 64 tokens)
    record = 4 * 64
    assert bytes_of(64, 8192, 128, 64, 128, 1, t=_lib.SSD_BF16) >= 64 * 128 * 128 * record * 4
    assert bytes_of(1, 200, 4, 64, 128, 2, t=_lib.SSD_BF16) >= 4 * 4 * record * 4


def test_struct_of_an_8_bit_tensor():
    t = T(torch.zeros(3, 5, dtype=i8))
    assert t.dtype == 3 and list(t.stride[:2]) == [5, 1]
    with pytest.raises(TypeError):
        T(torch.zeros(3, dtype=torch.float64))
    assert ctypes.sizeof(t) == 56


def test_the_check_of_stored_registers_finds_what_it_is_for():
    import os
    import sys
    sys.path.insert(0, os.path.dirname(os.path.abspath(_lib.__file__)) + "/..")
    import isa_check
    code = """
_Z6kernelv:                             ; @_Z6kernelv
	buffer_store_dwordx4 v[114:117], v169, s[12:15], s92 offen
	; a comment
	s_cbranch_vccnz .LBB0_1
	v_cndmask_b32_e64 v114, 0, 1, s[8:9]
	s_endpgm
"""
    found = isa_check.check_store_data(code)
    assert len(found) == 1 and found[0]["registers"] == [114] and found[0]["kernel"] == "_Z6kernelv"
    # the compiler's own wait, another register, an instruction between, a constant offset: nothing to find
    for old, new in (("s_cbranch_vccnz .LBB0_1", "s_nop 0"), ("v114, 0", "v118, 0"), ("s_cbranch_vccnz .LBB0_1", "v_mov_b32_e32 v1, v2"), (" s92 offen", " 0 offen")):
        assert isa_check.check_store_data(code.replace(old, new)) == []
