"""Refusals of the gated delta rule, layer norm and several-axes rotary, and
their tracing, without a GPU: meta tensors carry the shapes, and the C ABI
checks its arguments before any launch (stand-in addresses are never read)."""
import ctypes
import os

import pytest
import torch

from uttt_amd import _lib
from uttt_amd.delta import gated_delta_rule, gated_delta_step
from uttt_amd.norm import layer_norm
from uttt_amd.positions import axis_frequencies, rotary_axes

BF16 = torch.bfloat16
needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


def m(*shape, dtype=BF16, device="meta", grad=False):
    return torch.empty(*shape, dtype=dtype, device=device, requires_grad=grad)


def rule(B=2, T=10, Hk=1, Hv=2, Dk=64, Dv=32, dtype=BF16, gates=torch.float32, device="meta", **kw):
    x = dict(q=m(B, T, Hk, Dk, dtype=dtype, device=device), k=m(B, T, Hk, Dk, dtype=dtype, device=device),
             v=m(B, T, Hv, Dv, dtype=dtype, device=device), g=m(B, T, Hv, dtype=gates, device=device),
             beta=m(B, T, Hv, dtype=gates, device=device))
    x.update(kw)
    return x


@pytest.mark.parametrize("change,message", [
    (dict(dtype=torch.float16), "must be bf16"), (dict(dtype=torch.float32), "must be bf16"),
    (dict(Dk=264), "Dk = 264"), (dict(Dk=60), "Dk = 60"), (dict(Dv=12), "Dv = 12"), (dict(Dk=0), "Dk = 0"),
    (dict(Hk=2, Hv=3), "multiple of 2 key heads"), (dict(B=0), "empty batch"),
    (dict(gates=torch.float64), "g must be"), (dict(g=m(2, 10, 1, dtype=torch.float32)), "g and beta"),
    (dict(k=m(2, 10, 1, 32)), "must have q's shape"), (dict(v=m(2, 9, 2, 32)), "batch and tokens"),
    (dict(v=m(2, 10, 2, 32, dtype=torch.float16)), "one dtype"),
    (dict(initial_state=m(2, 2, 32, 64, dtype=torch.float32)), "initial_state must be"),
    (dict(initial_state=m(2, 2, 64, 32)), "states are fp32"),
    (dict(cu_seqlens=m(3, dtype=torch.int32)), "batch of 1"),
    (dict(B=1, cu_seqlens=m(1, dtype=torch.int32)), r"\[N \+ 1\]"),
    (dict(B=1, cu_seqlens=m(3, dtype=torch.float32)), "int32 or int64"),
    (dict(B=1, cu_seqlens=m(3, dtype=torch.int32), initial_state=m(1, 2, 64, 32, dtype=torch.float32)),
     "initial_state must be"),
])
def test_rule_refuses(change, message):
    x = rule(**change)
    kw = {n: x.pop(n) for n in ("initial_state", "cu_seqlens") if n in x}
    with pytest.raises(AssertionError, match=message):
        gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), **kw)


@pytest.mark.parametrize("change,kw,message", [
    ({}, dict(state=m(2, 2, 32, 64, dtype=torch.float32)), "state must be"),
    ({}, dict(state=m(2, 2, 64, 32)), "must be fp32"),
    ({}, dict(state=m(1, 2, 64, 32, dtype=torch.float32)), "2 rows, 1 states"),
    ({}, dict(state=m(4, 2, 32, 64, dtype=torch.float32).transpose(2, 3)), "contiguous"),
    ({}, dict(state=m(1, 2, 64, 32, dtype=torch.float32).expand(4, -1, -1, -1)), "apart"),
    ({}, dict(state_indices=m(3, dtype=torch.int32)), r"must be \[2\]"),
    ({}, dict(state_indices=m(2, dtype=torch.float32)), "int32 or int64"),
    (dict(Dv=6), dict(state=m(4, 2, 64, 6, dtype=torch.float32)), "Dv = 6"),
    (dict(Dk=300), dict(state=m(4, 2, 300, 32, dtype=torch.float32)), "Dk = 300"),
    (dict(dtype=torch.float64), {}, "dtype torch.float64"),
    ({}, dict(state=m(4, 2, 64, 32, dtype=torch.float32, grad=True)), "no gradient"),
])
def test_step_refuses(change, kw, message):
    x = rule(T=1, **change)
    kw = dict(kw)
    state = kw.pop("state", m(4, 2, 64, 32, dtype=torch.float32))
    with pytest.raises(AssertionError, match=message):
        gated_delta_step(*(x[n] for n in ("q", "k", "v", "g", "beta")), state, **kw)


@pytest.mark.parametrize("x,w,b,message", [
    (m(4, 8, dtype=torch.float64), None, None, "dtype"), (m(4, 8), m(7), None, r"weight must be \[8\]"),
    (m(4, 8), m(8), m(1, 8), r"bias must be \[8\]"), (m(4, 0), None, None, "N of 1 or more"),
    (m(4, 8), m(8, dtype=torch.float64), None, "weight has dtype"), (m(()), None, None, "must be"),
])
def test_layer_norm_refuses(x, w, b, message):
    with pytest.raises(AssertionError, match=message):
        layer_norm(x, w, b)


def rotary(D=64, sections=(16, 16), pos=None, freq=None, x=None):
    x = m(2, 5, 3, D) if x is None else x
    pos = m(2, 5, len(sections), dtype=torch.int32) if pos is None else pos
    freq = m(max(sum(sections), 0), dtype=torch.float32) if freq is None else freq
    return rotary_axes(x, pos, freq, sections)


@pytest.mark.parametrize("kw,message", [
    (dict(sections=(16, 17)), "do not fit"), (dict(sections=()), "sections"), (dict(sections=(1,) * 9), "sections"),
    (dict(sections=(-1, 4)), "sections"), (dict(sections=(0, 0)), "do not fit"),
    (dict(pos=m(2, 5, 3, dtype=torch.int32)), "positions must be"), (dict(pos=m(4, 2, dtype=torch.int32)), "positions"),
    (dict(pos=m(2, 5, 2, dtype=torch.float32)), "int32 or int64"), (dict(freq=m(31, dtype=torch.float32)), "inv_freq"),
    (dict(freq=m(32)), "inv_freq"), (dict(x=m(2, 5, 64)), "must be"), (dict(x=m(2, 5, 3, 64, dtype=torch.float64)), "dtype"),
])
def test_rotary_refuses(kw, message):
    with pytest.raises(AssertionError, match=message):
        rotary(**kw)


def test_cpu_tensors_are_refused():
    x = rule(device="cpu")
    args = [x[n] for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(RuntimeError, match="GPU only"):
        gated_delta_rule(*args)
    with pytest.raises(RuntimeError, match="GPU only"):
        gated_delta_step(*args, torch.zeros(2, 2, 64, 32))
    with pytest.raises(RuntimeError, match="GPU only"):
        layer_norm(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary_axes(torch.zeros(1, 1, 1, 4), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1), [1])


def test_frequencies():
    f = axis_frequencies([2, 2], base=16.0)
    assert torch.allclose(f, torch.tensor([1.0, 0.5, 0.25, 0.125]))
    assert torch.allclose(axis_frequencies([2, 4], base=16.0, per_axis=True),
                          torch.tensor([1.0, 0.25, 1.0, 0.5, 0.25, 0.125]))


def test_layer_traces_as_one_graph():
    """norm -> rotary -> rule forward and backward, and the step, without a graph break."""
    def layer(x, w, b, v, g, beta, pos, freq, h0):
        y = layer_norm(x, w, b).view(2, 70, 2, 64)
        q = rotary_axes(y, pos, freq, [16, 16])
        o, S = gated_delta_rule(q, q, v, g, beta, initial_state=h0, output_final_state=True)
        return o.float().sum() + S.sum()

    leaves = [m(2, 70, 128, grad=True), m(128, dtype=torch.float32, grad=True), m(128, grad=True),
              m(2, 70, 4, 32, grad=True), m(2, 70, 4, dtype=torch.float32, grad=True), m(2, 70, 4, grad=True)]
    h0 = m(2, 4, 64, 32, dtype=torch.float32, grad=True)
    rest = [m(2, 70, 2, dtype=torch.int32), m(32, dtype=torch.float32)]
    torch.compile(layer, fullgraph=True, backend="aot_eager")(*leaves, *rest, h0).backward()
    for t in leaves + [h0]:
        assert t.grad is not None and t.grad.shape == t.shape and t.grad.dtype == t.dtype
    x = rule(T=1)
    state, idx = m(4, 2, 64, 32, dtype=torch.float32), m(2, dtype=torch.int32)
    step = torch.compile(lambda *a: gated_delta_step(*a, state_indices=idx), fullgraph=True, backend="eager")
    assert step(*(x[n] for n in ("q", "k", "v", "g", "beta")), state).shape == (2, 1, 2, 32)


def strides(*s):
    return (ctypes.c_int64 * 3)(*s)


@needs_lib
def test_abi_rejects_bad_arguments_without_launch():
    lib, p = _lib.lib(), 1 << 20
    err = lambda: lib.uttt_last_error().decode()  # noqa: E731
    st = strides(640, 64, 64)

    def fwd(q=p, qs=st, gd=0, B=1, T=10, n=1, Hk=1, Hv=1, Dk=64, Dv=64, cu=None, out=p, u=None, s=None, ws=p, size=1 << 30):
        return lib.uttt_gated_delta_fwd(q, qs, p, st, p, st, p, gd, p, 0, cu, 0, B, T, n, Hk, Hv, Dk, Dv, 1.0, None,
                                        out, None, u, s, ws, size, None)

    for kw, text in ((dict(q=None), "null pointer"), (dict(qs=None), "null strides"), (dict(q=p + 2), "16-byte"),
                     (dict(qs=strides(640, 60, 64)), "multiple of 8"), (dict(gd=5), "dtype code 5"),
                     (dict(Dk=12), "Dk=12"), (dict(Dk=512), "Dk=512"), (dict(Dv=4), "Dv=4"), (dict(Hk=2, Hv=3), "Hv=3"),
                     (dict(n=2), "2 sequences in a batch of 1"), (dict(T=-1), "T=-1"), (dict(out=None), "null output"),
                     (dict(u=p), "both U and S"), (dict(size=100), "workspace of 100"), (dict(ws=None), "workspace"),
                     (dict(qs=strides(0, 1 << 23, 64)), "from token to token"),
                     (dict(B=2, n=2, cu=p), "batch of 2"), (dict(T=1 << 30, Hv=256, Hk=1, Dv=8, Dk=8), "too many")):
        assert fwd(**kw) == -1 and text in err(), (kw, err())
    size = lib.uttt_gated_delta_workspace_bytes
    assert size(1, 0, 1, 1, 1, 64, 64, 0, 0) == 0
    assert 0 < size(1, 64, 1, 1, 1, 64, 64, 0, 0) < size(1, 64, 1, 1, 1, 64, 64, 0, 1)
    assert lib.uttt_gated_delta_chunks(2, 65, 2, 0) == 4 and lib.uttt_gated_delta_chunks(1, 65, 3, 1) == 6
    rc = lib.uttt_gated_delta_bwd(p, st, p, st, p, st, p, 0, p, 0, None, 0, 1, 10, 1, 1, 1, 64, 64, 1.0, None, p, p, st,
                                  None, p, p, p, p, p, None, p, 1 << 30, None)
    assert rc == -1 and "null pointer" in err()

    def step(dtype=1, B=2, Dk=64, Dv=64, state=p, ss=4096, slots=4, idx=None, Hv=1):
        return lib.uttt_gated_delta_step(p, st, p, st, p, st, dtype, p, 0, p, 0, B, 1, 1, Hv, Dk, Dv, 1.0, state, ss, slots,
                                         idx, 0, p, None)

    for kw, text in ((dict(dtype=9), "dtype codes 9"), (dict(Dk=257), "Dk=257"), (dict(Dv=6), "Dv=6"),
                     (dict(B=5), "5 rows"), (dict(state=p + 4), "16-byte"), (dict(ss=64), "64 elements apart"),
                     (dict(state=None), "null pointer"), (dict(Hv=0), "Hv=0")):
        assert step(**kw) == -1 and text in err(), (kw, err())
    assert step(B=0) == 0

    assert lib.uttt_layer_norm_fwd(p, 1, 8, 4, 0, None, 0, None, 0, 1e-5, p, None, None) == -1 and "N=0" in err()
    assert lib.uttt_layer_norm_fwd(p, 4, 8, 4, 8, None, 0, None, 0, 1e-5, p, None, None) == -1 and "dtype" in err()
    assert lib.uttt_layer_norm_fwd(None, 1, 8, 4, 8, None, 0, None, 0, 1e-5, p, None, None) == -1 and "null" in err()
    assert lib.uttt_layer_norm_fwd(None, 1, 8, 0, 8, None, 0, None, 0, 1e-5, None, None, None) == 0
    rc = lib.uttt_layer_norm_bwd(p, 1, 8, p, 8, 4, 8, None, 0, p, p, p, None, 0, p, 8, None)
    assert rc == -1 and "workspace of 8 bytes" in err()
    assert lib.uttt_layer_norm_bwd(p, 1, 8, None, 8, 4, 8, None, 0, p, p, None, None, 0, None, 0, None) == -1

    sections = (ctypes.c_int * 2)(4, 4)

    def rot(x=p, dtype=1, D=16, axes=2, sec=sections, H=1):
        return lib.uttt_rotary_axes(x, dtype, strides(16, 16, 16), 1, 1, H, D, p, 0, strides(2, 2, 1), p, sec, axes, 0, 0,
                                    p, None)

    for kw, text in ((dict(x=None), "null"), (dict(dtype=3), "dtype code 3"), (dict(D=15), "8 pairs in 15"),
                     (dict(axes=0), "0 axes"), (dict(axes=9), "9 axes"), (dict(sec=None), "axes"),
                     (dict(sec=(ctypes.c_int * 2)(4, -4)), "section -4"), (dict(sec=(ctypes.c_int * 2)(0, 0)), "0 pairs"),
                     (dict(sec=(ctypes.c_int * 2)(2000, 2000), D=9000), "more than 2048")):
        assert rot(**kw) == -1 and text in err(), (kw, err())
    assert rot(H=0) == 0
