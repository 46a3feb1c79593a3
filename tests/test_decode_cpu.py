"""The operators of a decoding step, without a GPU: what their wrappers and C entry points refuse, and that nothing is computed on a CPU."""
import ctypes

import pytest
import torch

import ssd_amd as ops
from ssd_amd import _lib
from ssd_amd.decode import _bytes_arg as U
from ssd_amd.layer import _arg as T

b16, u8 = torch.bfloat16, torch.uint8
NULL, SHAPE, DTYPE, STRIDE, SCRATCH = -1, -2, -3, -4, -6


def mm(**kw):
    v = dict(a=torch.zeros(3, 64), w=torch.zeros(8, 32, dtype=u8), w_scale=torch.zeros(8, 2), w_zero=None, group=32, bias=None, out_dtype=None)
    return lambda: ops._matmul_int4_fwd(**{**v, **kw})


def block(**kw):
    v = dict(x=torch.zeros(2, 3, 16), weight=torch.zeros(16), residual=torch.zeros(2, 3, 16), next_weight=torch.zeros(16))
    return lambda: ops._norm_block_fwd(**{**v, **kw})


def select(**kw):
    v = dict(logits=torch.zeros(2, 3, 9), scores=torch.zeros(2, 3))
    return lambda: ops._beam_select_fwd(**{**v, **kw})


def reorder(**kw):
    v = dict(parents=torch.zeros(2, 3, dtype=torch.int32), slots=torch.zeros(2, 3, dtype=torch.int32), pools=[torch.zeros(6, 4)])
    return lambda: ops._beam_reorder(**{**v, **kw})


def test_nothing_is_computed_on_a_cpu():
    for call in (mm(), block(), block(int8=True, gate=torch.zeros(2, 1, 16)), select(), select(finished=torch.zeros(2, 3, dtype=torch.bool)), reorder(), reorder(pools=[])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


WRONG = [
    mm(w=torch.zeros(8, 31, dtype=u8)), mm(w=torch.zeros(8, 32, dtype=torch.int8)), mm(a=torch.zeros(3, 64).double()), mm(a=torch.zeros(3, 64, dtype=torch.int8)),
    mm(group=16), mm(group=0), mm(group=-32), mm(group=48), mm(w_scale=torch.zeros(8, 1)), mm(w_scale=torch.zeros(7, 2)), mm(w_scale=torch.zeros(8, 2, dtype=u8)),
    mm(w_zero=torch.zeros(8, 1, dtype=u8)), mm(w_zero=torch.zeros(8, 2)), mm(bias=torch.zeros(7)), mm(bias=torch.zeros(8, dtype=torch.int32)),
    mm(out_dtype=torch.int32), mm(out_dtype=torch.float64),
    block(weight=torch.zeros(15)), block(next_weight=torch.zeros(15)), block(residual=torch.zeros(2, 3, 15)), block(residual=torch.zeros(6, 16)),
    block(gate=torch.zeros(15)), block(gate=torch.zeros(1, 3, 16)), block(gate=torch.zeros(3, 16)), block(gate=torch.zeros(1, 2, 3, 16)), block(gate=torch.zeros(2, 2, 16)),
    block(x=torch.zeros(2, 3, 16).double()), block(weight=torch.zeros(16).double()), block(gate=torch.zeros(16, dtype=torch.int32)), block(x=torch.zeros(2, 3, 0)),
    select(scores=torch.zeros(2, 2)), select(scores=torch.zeros(2, 3, dtype=torch.int32)), select(k=0), select(k=28), select(k=-1), select(k=65, logits=torch.zeros(2, 3, 99)),
    select(logits=torch.zeros(1, 65, 4), scores=torch.zeros(1, 65)), select(logits=torch.zeros(2, 3, 9, dtype=torch.int64)), select(logits=torch.zeros(2, 3, 0)),
    select(finished=torch.zeros(2, 3)), select(finished=torch.zeros(2, 2, dtype=torch.bool)), select(finished=torch.zeros(2, 3, dtype=torch.bool), pad=9),
    select(finished=torch.zeros(2, 3, dtype=torch.bool), pad=-1),
    reorder(slots=torch.zeros(2, 2, dtype=torch.int32)), reorder(parents=torch.zeros(2, 3)), reorder(slots=torch.zeros(2, 3)),
    reorder(parents=torch.zeros(2, 65, dtype=torch.int32), slots=torch.zeros(2, 65, dtype=torch.int32)), reorder(pools=[torch.zeros(6, 4), torch.zeros(5, 4)]),
    reorder(pools=[torch.zeros(6, 1).expand(6, 4)]), reorder(pools=[torch.zeros(1, 4).expand(6, 4)]), reorder(pools=[torch.zeros(6, 1, 1, 1, 1, 1)]),
]


@pytest.mark.parametrize("i", range(len(WRONG)))
def test_wrappers_refuse_what_does_not_fit(i):
    with pytest.raises(AssertionError):
        WRONG[i]()


def test_c_entry_points_refuse_in_front_of_any_device_work():
    lib = _lib.load()
    none = T(None)
    a, w, s, out = torch.zeros(3, 64), torch.zeros(8, 32, dtype=u8), torch.zeros(8, 2), torch.zeros(3, 8)

    def product(a=a, w=U(w), s=T(s), z=none, bias=none, out=T(out), M=3, N=8, K=64, group=32):
        return lib.ssd_matmul_packed_fwd(T(a), w, s, z, bias, out, M, N, K, group, None, 0, None)
    assert product(group=16) == SHAPE and product(group=0) == SHAPE and product(M=-1) == SHAPE and product(K=(1 << 30) + 1, group=1 << 31 - 1) == SHAPE
    assert product(M=0) == 0 and product(N=0) == 0
    assert product(a=None) == NULL and product(w=none) == NULL and product(s=none) == NULL and product(out=none) == NULL
    assert product(w=T(a)) == DTYPE and product(a=a.to(torch.int8)) == DTYPE and product(z=T(s)) == DTYPE and product(out=T(out.to(torch.int8))) == DTYPE
    assert product(a=torch.zeros(64, 3).t()) == STRIDE and product(w=U(torch.zeros(32, 8, dtype=u8).t())) == STRIDE and product(out=T(torch.zeros(8, 3).t())) == STRIDE

    x, g = torch.zeros(4, 16), torch.zeros(16)
    q, sc = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)

    def norms(x=x, w=g, r=x, nw=g, gate=None, out=x, scale=None, total=x, rows=4, dim=16, every=1):
        return lib.ssd_norm_block_fwd(T(x), T(w), T(r), T(nw), T(gate), T(out), T(scale), T(total), rows, dim, every, 1.0, 1e-5, None)
    assert norms(dim=0) == SHAPE and norms(rows=-1) == SHAPE and norms(gate=x, every=0) == SHAPE and norms(rows=0) == 0
    assert norms(x=None) == NULL and norms(r=None) == NULL and norms(nw=None) == NULL and norms(out=None) == NULL and norms(total=None) == NULL and norms(out=q) == NULL
    assert norms(r=x.half()) == DTYPE and norms(out=x.half()) == DTYPE and norms(total=x.half()) == DTYPE and norms(w=g.half()) == DTYPE and norms(gate=x.to(b16)) == DTYPE
    assert norms(x=q, r=q, total=q, out=q, scale=sc) == DTYPE and norms(out=q, scale=sc.half()) == DTYPE
    assert norms(r=torch.zeros(16, 4).t()) == STRIDE and norms(w=torch.zeros(32)[::2]) == STRIDE and norms(gate=torch.zeros(16, 4).t()) == STRIDE

    lo, sco = torch.zeros(2, 3, 9), torch.zeros(2, 3)
    best, whole = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)
    room = torch.zeros(10000)
    address = room.data_ptr() + -room.data_ptr() % 16

    def choose(lo=lo, sc=T(sco), f=none, best=best, p=whole, t=whole, b=2, beams=3, V=9, k=4, pad=0, at=address, n=39000):
        return lib.ssd_beam_select_fwd(T(lo), sc, f, T(best), T(p), T(t), b, beams, V, k, pad, ctypes.c_void_p(at), n, None)
    assert choose(k=65) == SHAPE and choose(k=28) == SHAPE and choose(k=0) == SHAPE and choose(beams=65) == SHAPE and choose(beams=0) == SHAPE and choose(V=0) == SHAPE
    assert choose(b=-1) == SHAPE and choose(V=(1 << 31) - 1) == SHAPE and choose(f=U(torch.zeros(2, 3, dtype=u8)), pad=9) == SHAPE and choose(b=0) == 0
    assert choose(lo=None) == NULL and choose(sc=none) == NULL and choose(best=None) == NULL and choose(p=None) == NULL and choose(t=None) == NULL
    assert choose(lo=lo.to(torch.int8)) == DTYPE and choose(sc=T(sco.half())) == DTYPE and choose(p=best.half()) == DTYPE and choose(f=T(sco)) == DTYPE
    assert choose(lo=torch.zeros(2, 9, 3).transpose(1, 2)) == STRIDE and choose(best=torch.zeros(4, 2).t()) == STRIDE
    need = lib.ssd_beam_workspace_bytes(2, 3, 9, 4)
    assert need > 0 and lib.ssd_beam_workspace_bytes(2, 3, 9, 65) == 0
    assert choose(at=None) == SCRATCH and choose(n=need - 1) == SCRATCH and choose(at=address + 8) == SCRATCH

    index = torch.zeros(2, 3, dtype=torch.int32)
    pool = torch.zeros(6, 4, 5)

    def follow(p=index, s=index, n=index, b=2, beams=3, count=1, slots=6, element=4, dims=2, slot=20, size=(4, 5), stride=(5, 1), data=pool.data_ptr()):
        pools = (_lib.SsdPool * 1)()
        pools[0].data, pools[0].element_bytes, pools[0].dims, pools[0].slot_stride = data, element, dims, slot
        for i, (x, y) in enumerate(zip(size, stride)):
            pools[0].size[i], pools[0].stride[i] = x, y
        return lib.ssd_beam_reorder(T(p), T(s), T(n), pools, count, slots, b, beams, None)
    assert follow(b=-1) == SHAPE and follow(beams=65) == SHAPE and follow(beams=0) == SHAPE and follow(count=-1) == SHAPE and follow(slots=-1) == SHAPE and follow(b=0) == 0
    assert follow(p=None) == NULL and follow(s=None) == NULL and follow(n=None) == NULL and follow(data=None) == NULL
    assert follow(p=index.half()) == DTYPE and follow(element=3) == DTYPE and follow(element=0) == DTYPE
    assert follow(stride=(0, 1)) == STRIDE and follow(stride=(5, -1)) == STRIDE and follow(dims=5) == STRIDE and follow(slot=0) == STRIDE


def test_c_entry_points_refuse_sizes_whose_ends_do_not_fit_and_pools_that_overlap():
    # (nothing is read: every one of these is refused for its sizes)
    lib = _lib.load()
    none, x, w = T(None), torch.zeros(4, 16), torch.zeros(4, 8, dtype=u8)
    big = (1 << 30) + 1
    for M, N, K in ((big, 4, 16), ((1 << 31) - 1, 4, 1), (4, big, 16), (4, (1 << 31) - 1, 1)):
        assert lib.ssd_matmul_packed_fwd(T(x), U(w), T(x), none, none, T(x), M, N, K, 32, None, 0, None) == SHAPE
        assert lib.ssd_matmul_packed_workspace_bytes(M, N, K, 32, 0) == 0
    for dim in (big, (1 << 31) - 1):
        assert lib.ssd_norm_block_fwd(T(x), none, T(x), T(x[0]), none, T(x), none, T(x), 1, dim, 1, 1.0, 1e-5, None) == SHAPE
    assert lib.ssd_beam_workspace_bytes(1, 1, big, 1) == 0 and lib.ssd_beam_workspace_bytes(1, 1, big - 1, 1) > 0
    assert lib.ssd_beam_select_fwd(T(x[None]), T(x), none, T(x), T(x.int()), T(x.int()), 1, 1, (1 << 31) - 1, 1, 0, None, 0, None) == SHAPE
    index = torch.zeros(1, 2, dtype=torch.int32)

    def follow(slots, slot, size, stride, element=4, data=1 << 12):
        pools = (_lib.SsdPool * 1)()
        pools[0].data, pools[0].element_bytes, pools[0].dims, pools[0].slot_stride = data, element, len(size), slot
        for i, (a, b) in enumerate(zip(size, stride)):
            pools[0].size[i], pools[0].stride[i] = a, b
        return lib.ssd_beam_reorder(T(index), T(index), T(index.clone()), pools, 1, slots, 1, 2, None)
    assert follow(3, 19, (4, 5), (5, 1)) == STRIDE and follow(3, 1, (4, 5), (5, 1)) == STRIDE and follow(3, 20, (4, 2), (1, 2)) == STRIDE
    assert follow(3, -20, (4, 5), (5, 1)) == STRIDE and follow(3, 0, (), ()) == STRIDE and follow(3, 1, (7,), (2,)) == STRIDE
    assert follow(1, 0, (1 << 34, 4), (4, 1), 16) == SHAPE and follow(1, 0, (1 << 62, 4), (4, 1), 1) == STRIDE and follow(1, 0, (1 << 36, 2), (2, 1), 1) == SHAPE
    # dense ones in any order of their dimensions, and parts of them, are not refused for it, but for having no data
    for slots, slot, size, stride in ((3, 20, (4, 5), (5, 1)), (3, 1, (4, 5), (15, 3)), (3, 5, (4, 5), (15, 1)), (1, 0, (4, 5), (5, 1)), (3, 100, (4, 2), (7, 3)), (3, 1, (), ())):
        assert follow(slots, slot, size, stride, data=None) == NULL
