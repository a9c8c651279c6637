"""Refusals of the state space layer's operators and the block norms, what they
hand to the C ABI, and what autograd may do with them, without a GPU: meta
tensors carry the shapes, and the C ABI checks its arguments before any launch
(stand-in addresses are never read)."""
import ctypes
import os

import pytest
import torch
from torch.autograd import forward_ad

from uttt_amd import _lib, norm, state_space
from uttt_amd.norm import norm_after_block, norm_before_block
from uttt_amd.state_space import causal_conv, causal_conv_step, selective_scan, selective_scan_step

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


def m(*shape, dtype=BF16, device="meta", grad=False):
    shape = shape[0] if shape and isinstance(shape[0], tuple) else shape
    return torch.empty(shape, dtype=dtype, device=device, requires_grad=grad)


def scan_args(B=2, T=10, D=12, N=16, G=2, dtype=BF16, dt=F32, device="meta", grad=False, **kw):
    e = lambda *s, dtype=dtype: m(*s, dtype=dtype, device=device, grad=grad)  # noqa: E731
    a = dict(x=e(B, T, D), dt=e(B, T, D, dtype=dt), A=e(D, N, dtype=F32), B=e(B, T, G, N), C=e(B, T, G, N),
             D=e(D, dtype=F32), gate=e(B, T, D), dt_bias=e(D, dtype=F32))
    a.update(kw)
    return a


def scan(a, **kw):
    return selective_scan(*(a[n] for n in ("x", "dt", "A", "B", "C")), D=a["D"], gate=a["gate"], dt_bias=a["dt_bias"], **kw)


def scan_step(a, state, **kw):
    return selective_scan_step(*(a[n] for n in ("x", "dt", "A", "B", "C")), state, D=a["D"], gate=a["gate"],
                               dt_bias=a["dt_bias"], **kw)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=torch.float64), "dtype"), (dict(dt=torch.float64), "dt must be"), (dict(dt=F16), "dt must be"),
    (dict(dt=m(2, 9, 12, dtype=F32)), "x's shape"), (dict(A=m(12, 65, dtype=F32)), "N of 1 to 64"),
    (dict(A=m(11, 16, dtype=F32)), r"must be \[12, N\]"), (dict(A=m(12, 16)), "A must be fp32"),
    (dict(A=m(12, 0, dtype=F32), N=0), "N of 1 to 64"), (dict(B=m(2, 10, 2, 8)), "B must be"),
    (dict(C=m(2, 10, 1, 16)), "C .* B's shape"), (dict(G=5), "multiple of 5 groups"), (dict(G=0), "multiple of 0 groups"),
    (dict(B=m(2, 10, 2, 16, dtype=F32)), "B must have x's dtype"), (dict(gate=m(2, 10, 12, dtype=F32)), "gate must have"),
    (dict(gate=m(2, 10, 11)), "gate must have"), (dict(D=m(11, dtype=F32)), r"D must be \[12\]"),
    (dict(D=m(12)), "D must be fp32"), (dict(dt_bias=m(12)), "dt_bias must be fp32"),
    (dict(dt_bias=m(1, 12, dtype=F32)), "dt_bias must be"), (dict(x=m(2, 10)), "x must be"), (dict(B=m(0, 10, 2, 16)), "B must be"),
])
def test_scan_refuses(change, message):
    shape = {n: change[n] for n in ("dtype", "G", "N") if n in change}
    if isinstance(change.get("dt"), torch.dtype):
        shape["dt"] = change["dt"]
    a = scan_args(**shape)
    a.update({n: t for n, t in change.items() if isinstance(t, torch.Tensor)})
    for fn in (lambda: scan(a), lambda: scan_step(a, m(4, 12, 16, dtype=F32))):
        with pytest.raises(AssertionError, match=message):
            fn()


@pytest.mark.parametrize("kw,message", [
    (dict(initial_state=m(2, 16, 12, dtype=F32)), "initial_state must be"), (dict(initial_state=m(2, 12, 16)), "must be fp32"),
    (dict(cu_seqlens=m(3, dtype=torch.int32)), "batch of 1"),
])
def test_scan_refuses_states_and_offsets(kw, message):
    with pytest.raises(AssertionError, match=message):
        scan(scan_args(), **kw)


@pytest.mark.parametrize("cu,message", [(m(1, dtype=torch.int32), r"\[N \+ 1\]"), (m(3, dtype=F32), "int32 or int64"),
                                        (m(2, 3, dtype=torch.int32), r"\[N \+ 1\]")])
def test_offsets_are_refused(cu, message):
    with pytest.raises(AssertionError, match=message):
        scan(scan_args(B=1), cu_seqlens=cu)
    with pytest.raises(AssertionError, match=message):
        causal_conv(m(1, 10, 8), m(8, 4), cu_seqlens=cu)


def test_empty_batches_and_too_many_tokens_are_refused():
    with pytest.raises(AssertionError, match="empty batch"):
        scan(scan_args(B=0))
    with pytest.raises(AssertionError, match="empty batch"):
        causal_conv(m(0, 3, 8), m(8, 4))
    with pytest.raises(AssertionError, match="fewer than 2"):
        causal_conv(m(1 << 15, 1 << 15, 1), m(1, 4))


def test_too_many_channels_are_refused():
    wide = m(1, 1, (1 << 24) + 1)
    rates, one = m((1 << 24) + 1, 1, dtype=F32), m(1, 1, 1, 1)
    with pytest.raises(AssertionError, match="channels"):
        selective_scan(wide, wide, rates, one, one)
    with pytest.raises(AssertionError, match="channels"):
        selective_scan_step(wide, wide, rates, one, one, m(1, (1 << 24) + 1, 1, dtype=F32))


@pytest.mark.parametrize("kw,message", [
    (dict(state=m(4, 16, 12, dtype=F32)), "state must be"), (dict(state=m(4, 12, 16)), "state must be"),
    (dict(state=m(1, 12, 16, dtype=F32)), "2 rows, 1 states"), (dict(state=m(4, 16, 12, dtype=F32).transpose(1, 2)), "contiguous"),
    (dict(state=m(1, 12, 16, dtype=F32).expand(4, -1, -1)), "apart"), (dict(state=m(4, 12, 32, dtype=F32)[..., :16]), "contiguous"),
    (dict(state_indices=m(3, dtype=torch.int32)), r"must be \[2\]"), (dict(state_indices=m(2, dtype=F32)), "int32 or int64"),
    (dict(state=m(4, 12, 16, dtype=F32, grad=True)), "no gradient"),
])
def test_scan_step_refuses(kw, message):
    kw = dict(kw)
    with pytest.raises(AssertionError, match=message):
        scan_step(scan_args(T=1), kw.pop("state", m(4, 12, 16, dtype=F32)), **kw)


@pytest.mark.parametrize("x,w,b,kw,message", [
    (m(2, 3, 8, dtype=torch.float64), m(8, 4), None, {}, "dtype"), (m(2, 8), m(8, 4), None, {}, "x must be"),
    (m(2, 3, 8), m(8, 1), None, {}, "W of 2 to 8"), (m(2, 3, 8), m(8, 9), None, {}, "W of 2 to 8"),
    (m(2, 3, 8), m(7, 4), None, {}, "weight must be"), (m(2, 3, 8), m(8, 4), m(4), {}, "bias must be"),
    (m(2, 3, 8), m(8, 4, dtype=torch.float64), None, {}, "weight has dtype"), (m(2, 3, 8), m(8, 4), None, dict(activation="relu"), "activation"),
    (m(2, 3, 8), m(8, 1, 4), None, {}, "weight must be"),
])
def test_conv_refuses(x, w, b, kw, message):
    with pytest.raises(AssertionError, match=message):
        causal_conv(x, w, b, **kw)
    with pytest.raises(AssertionError, match=message):
        causal_conv_step(x, w, m(4, 3, 8), b, **kw)


@pytest.mark.parametrize("kw,message", [(dict(initial_state=m(2, 4, 8)), "initial_state must be"),
                                        (dict(initial_state=m(2, 3, 8, dtype=F32)), "must be torch.bfloat16")])
def test_conv_refuses_states(kw, message):
    with pytest.raises(AssertionError, match=message):
        causal_conv(m(2, 5, 8), m(8, 4), **kw)


@pytest.mark.parametrize("state,idx,message", [(m(4, 3, 8, dtype=F32), None, "state must be"), (m(4, 8, 3), None, "state must be"),
                                               (m(1, 3, 8), None, "2 rows, 1 states"), (m(4, 3, 8, grad=True), None, "no gradient"),
                                               (m(4, 3, 8), m(2, 1, dtype=torch.int32), r"must be \[2\]")])
def test_conv_step_refuses(state, idx, message):
    with pytest.raises(AssertionError, match=message):
        causal_conv_step(m(2, 1, 8), m(8, 4), state, state_indices=idx)


@pytest.mark.parametrize("x,kw,message", [
    (m(4, 8, dtype=torch.float64), {}, "dtype"), (m(4, 8), dict(weight=m(7)), r"weight must be \[8\]"),
    (m(4, 8193), {}, "N of 1 to 8192"), (m(4, 0), {}, "N of 1 to 8192"), (m(()), {}, "N of 1 to 8192"),
    (m(4, 8), dict(scale=m(1, 8)), r"scale must be \[8\]"), (m(4, 8), dict(weight=m(8, dtype=torch.float64)), "weight has dtype"),
    (m(4, 8), dict(residual=m(4, 7)), "x's shape"), (m(4, 8), dict(residual=m(4, 8, dtype=torch.float64)), "residual has dtype"),
])
def test_norms_refuse(x, kw, message):
    with pytest.raises(AssertionError, match=message):
        norm_after_block(x, **kw)
    kw = dict(kw)
    with pytest.raises(AssertionError, match=message):
        norm_before_block(x, kw.pop("residual", m(*x.shape)), **kw)


@pytest.mark.parametrize("gate,message", [(m(4, 8, dtype=F32), "x's dtype"), (m(8), "x's shape")])
def test_gates_are_refused(gate, message):
    with pytest.raises(AssertionError, match=message):
        norm_after_block(m(4, 8), gate=gate)


def test_cpu_tensors_are_refused():
    a = scan_args(device="cpu")
    c = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    for fn in (lambda: scan(a), lambda: scan_step(a, c(2, 12, 16, dtype=F32)), lambda: causal_conv(c(1, 2, 8), c(8, 4)),
               lambda: causal_conv_step(c(1, 2, 8), c(8, 4), c(1, 3, 8)), lambda: norm_after_block(c(2, 8)),
               lambda: norm_before_block(c(2, 8), c(2, 8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            fn()


# ----------------------------------------------------------- calls to the C ABI --
@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(state_space.L, "call_on", lambda t, name, *args: calls.append((name, args)))
    monkeypatch.setattr(state_space.L, "stream_of", lambda t: 0)
    return calls


@pytest.mark.parametrize("stride", [0, 1, 5, 191, 193, 2 ** 40 + 1])
def test_one_state_with_a_stride_of_no_use(launched, stride):
    state = m(200, dtype=F32).as_strided((1, 12, 16), (stride, 16, 1))
    scan_step(scan_args(B=1, T=1), state)
    conv = m(200).as_strided((1, 3, 8), (stride, 8, 1))
    causal_conv_step(m(1, 1, 8), m(8, 4), conv)
    assert launched[0][1][22] == 12 * 16 and launched[1][1][13] == 24
    pool = m(3, 5, 12, 16, dtype=F32)
    scan_step(scan_args(B=3, T=1), pool[:, 1])
    assert launched[2][1][22] == 5 * 12 * 16


def test_strides_along_an_axis_of_one_say_nothing(launched):
    x = m(1, 1, 8).as_strided((1, 1, 8), (3, 1 << 40, 1))
    causal_conv(x, m(8, 4))
    assert list(launched[0][1][1]) == [0, 0]


def test_the_steps_say_that_they_change_their_states(launched):
    """A state that another op has saved for its backward raises there."""
    for state, call in ((m(2, 12, 16, dtype=F32, grad=True), lambda s: scan_step(scan_args(T=1), s)),
                        (m(2, 3, 8, grad=True), lambda s: causal_conv_step(m(2, 1, 8), m(8, 4), s))):
        loss = state.square().sum()
        with torch.no_grad():
            call(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    pool = m(2, 4, 12, 16, dtype=F32)
    before = pool._version
    scan_step(scan_args(T=1), pool[:, 1])
    assert pool._version == before + 1
    with torch.inference_mode():
        scan_step(scan_args(T=1), m(2, 12, 16, dtype=F32))


@pytest.mark.parametrize("which", ["x", "dt", "A", "B", "C", "D", "gate", "dt_bias", "state"])
def test_the_steps_refuse_forward_gradients(launched, which):
    with forward_ad.dual_level():
        a = dict(scan_args(T=1), state=m(2, 12, 16, dtype=F32))
        a[which] = forward_ad.make_dual(a[which], torch.empty_like(a[which]))
        with pytest.raises(AssertionError, match="no gradient"):
            scan_step(a, a["state"])
        c = dict(x=m(2, 1, 8), w=m(8, 4), state=m(2, 3, 8))
        if which in ("x", "state"):
            c[which] = forward_ad.make_dual(c[which], torch.empty_like(c[which]))
            with pytest.raises(AssertionError, match="no gradient"):
                causal_conv_step(c["x"], c["w"], c["state"])
    assert not launched


def faked(monkeypatch):
    for mod, names in ((state_space, ("conv_fwd", "conv_bwd", "scan_fwd", "scan_bwd", "scan_infer")),
                       (norm, ("after_fwd", "after_bwd", "before_fwd", "before_bwd"))):
        for n in names:
            fake = {"after_fwd": "_after_fake", "before_fwd": "_before_fake"}.get(n, f"_{n}_fake")
            monkeypatch.setattr(mod, "_" + n, getattr(mod, fake))


def differentiable():
    """(leaves, outputs of them) of each operator."""
    e = lambda *s, dtype=BF16: m(*s, dtype=dtype)  # noqa: E731
    yield [e(2, 5, 8), e(8, 4, dtype=F32), e(8), e(2, 3, 8)], lambda x, w, b, h: causal_conv(
        x, w, b, activation="silu", initial_state=h, output_final_state=True)
    a = scan_args()
    names = list(a)
    yield list(a.values()) + [e(2, 12, 16, dtype=F32)], lambda *t: scan(
        dict(zip(names, t)), initial_state=t[-1], output_final_state=True)
    yield [e(4, 8), e(8, dtype=F32), e(4, 8), e(4, 8, dtype=F32), e(8)], lambda x, w, z, r, s: (
        norm_after_block(x, w, gate=z, residual=r, scale=s),)
    yield [e(4, 8), e(4, 8, dtype=F32), e(8), e(8)], lambda x, r, w, s: norm_before_block(x, r, w, scale=s)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("linear", [True, False])
def test_second_order_is_refused(monkeypatch, which, linear):
    """For any leaf alone, with gradients of the outputs that are constant and not."""
    faked(monkeypatch)
    tensors, fn = list(differentiable())[which]
    for one in [None, *range(len(tensors))]:
        leaves = [t.detach().requires_grad_(one is None or i == one) for i, t in enumerate(tensors)]
        loss = sum((y.float() if linear else y.float().square()).sum() for y in fn(*leaves))
        wanted = [t for t in leaves if t.requires_grad]
        once = torch.autograd.grad(loss, wanted, retain_graph=True)
        assert [g.shape for g in once] == [t.shape for t in wanted] and [g.dtype for g in once] == [t.dtype for t in wanted]
        assert not any(g.requires_grad for g in once)
        grads = torch.autograd.grad(loss, wanted, create_graph=True)
        for g in grads:
            if which == 2 and g.dtype == F32 and g.shape == (4, 8):
                continue   # the residual's gradient is the outputs' own, and torch's to differentiate
            for t in wanted:
                if which == 2 and linear and t.dtype == F32 and t.shape == (4, 8):
                    continue   # no other gradient depends on the residual
                with pytest.raises(RuntimeError, match="gradients of its gradients|does not require grad"):
                    torch.autograd.grad(loss + g.float().square().sum(), t, retain_graph=True)


def test_forward_mode_is_refused(monkeypatch):
    faked(monkeypatch)
    with forward_ad.dual_level():
        for tensors, fn in differentiable():
            duals = [forward_ad.make_dual(tensors[0], torch.empty_like(tensors[0])), *tensors[1:]]
            with pytest.raises((RuntimeError, NotImplementedError)):
                fn(*duals)


def test_without_gradients_nothing_is_kept(monkeypatch):
    faked(monkeypatch)
    for tensors, fn in differentiable():
        for y in fn(*tensors):
            assert not y.requires_grad
        with torch.no_grad():
            for y in fn(*(t.detach().requires_grad_() for t in tensors)):
                assert not y.requires_grad


def test_tracing():
    """The registered ops under fake tensors, forward and backward."""
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        dev = "cuda"
        a = {n: torch.empty(t.shape, dtype=t.dtype, device=dev) for n, t in scan_args(N=10).items()}
        y, h, tiles = torch.ops.uttt_hip.selective_scan_fwd(*a.values(), True, None, None, True)
        assert y.shape == (2, 10, 12) and h.shape == (2, 12, 10) and tiles.shape == (2, 16, 12)
        g = torch.ops.uttt_hip.selective_scan_bwd(*a.values(), True, None, tiles, y, h, True)
        assert [t.shape for t in g] == [*(t.shape for t in a.values()), h.shape]
        x, w = a["x"], torch.empty(12, 4, device=dev)
        y, s = torch.ops.uttt_hip.causal_conv_fwd(x, w, None, True, None, None, True)
        assert s.shape == (2, 3, 12) and torch.ops.uttt_hip.causal_conv_step(x, w, None, True, s, None).shape == x.shape
        y, t, r = torch.ops.uttt_hip.norm_before_fwd(x, x.float(), None, None, 1.0, 1e-5, True)
        assert y.dtype == BF16 and t.dtype == F32 and r.shape == (20,)


@needs_lib
def test_tile_count_is_the_librarys():
    lib = _lib.lib()
    for B, T in ((1, 0), (1, 1), (3, 15), (2, 16), (2, 17), (1, 100)):
        a = scan_args(B=B, T=T, N=5)
        fake = state_space._scan_fwd_fake(*a.values(), True, None, None, False)[2]
        assert fake.shape == (lib.uttt_selective_scan_tiles(B, T, B, 0), 8, 12)
        if B == 1:
            for n in (1, 4):
                fake = state_space._scan_fwd_fake(*a.values(), True, None, m(n + 1, dtype=torch.int32), False)[2]
                assert fake.shape[0] == lib.uttt_selective_scan_tiles(1, T, n, 1)


@needs_lib
def test_the_c_abi_refuses():
    """Argument checks, before anything is launched (the addresses are never read)."""
    lib, p = _lib.lib(), 1 << 20
    st = lambda *v: (ctypes.c_int64 * 3)(*v)  # noqa: E731
    err = lambda: lib.uttt_last_error().decode()  # noqa: E731
    big = 1 << 62

    def scan_fwd(B=1, T=10, n=None, D=8, N=4, G=1, dtype=1, dt=0, x=p, A=p, step=8, cu=None, ws=p, size=big):
        return lib.uttt_selective_scan_fwd(x, st(0, step, 0), dtype, p, st(0, 8, 0), dt, A, p, st(0, 8, 8), p, st(0, 8, 8), None,
                                           None, None, None, 0, None, cu, 0, B, T, B if n is None else n, D, N, G, p, None, None,
                                           ws, size, None)

    def scan_bwd(B=1, T=10, n=None, D=8, N=4, G=1, dtype=1, dt=0, x=p, A=p, step=8, cu=None, ws=p, size=big):
        return lib.uttt_selective_scan_bwd(x, st(0, step, 0), dtype, p, st(0, 8, 0), dt, A, p, st(0, 8, 8), p, st(0, 8, 8), None,
                                           None, None, None, 0, cu, 0, B, T, B if n is None else n, D, N, G, p, p, st(0, 8, 0),
                                           None, p, p, p, p, p, None, None, None, None, ws, size, None)

    for fn in (scan_fwd, scan_bwd):
        for kw, message in ((dict(N=65), "N=65"), (dict(N=0), "N=0"), (dict(D=7, G=2), "multiple"), (dict(D=(1 << 24) + 1), "2^24"),
                            (dict(dtype=7), "dtype"),
                            (dict(dtype=1, dt=2), "dtype"), (dict(dtype=0, dt=1), "dtype"), (dict(n=2), "bad sizes"),
                            (dict(B=2, n=2, cu=p), "bad sizes"), (dict(x=None), "null"), (dict(A=p + 4), "16-byte"),
                            (dict(step=1 << 24), "between tokens"), (dict(T=5000, size=16), "workspace"),
                            (dict(T=5000, ws=None), "workspace"), (dict(B=1 << 20, T=1, D=1 << 14), "too many"),
                            (dict(B=1 << 12, T=1, D=1 << 17, N=64), "too many")):
            assert fn(**kw) == -1 and message in err(), (fn.__name__, kw, err())

    def conv(B=1, T=10, n=None, D=8, W=4, dtype=1, x=p, cu=None):
        return lib.uttt_causal_conv_fwd(x, st(0, 8, 0), dtype, p, 0, None, 0, 1, None, cu, 0, B, T, B if n is None else n, D, W,
                                        p, None, None)

    for kw, message in ((dict(W=1), "W=1"), (dict(W=9), "W=9"), (dict(dtype=5), "dtype"), (dict(n=3), "bad sizes"), (dict(x=None), "null"),
                        (dict(B=1 << 16, T=1 << 10, D=1 << 12), "too many")):
        assert conv(**kw) == -1 and message in err(), (kw, err())
    assert lib.uttt_causal_conv_bwd(p, st(0, 8, 0), 1, p, 0, None, 0, 1, None, None, 0, 1, 10, 1, 8, 4, p, st(0, 8, 0), None, p,
                                    p, None, None, p, 4, None) == -1 and "workspace" in err()

    def conv_step(B=2, W=4, D=8, apart=24, slots=4, idx=None):
        return lib.uttt_causal_conv_step(p, st(8, 8, 0), 1, p, 0, None, 0, 1, B, 1, D, W, p, apart, slots, idx, 0, p, None)

    for kw, message in ((dict(slots=1), "slots"), (dict(apart=23), "apart"), (dict(W=9), "W=9"), (dict(B=1 << 24, slots=1 << 24), "too many")):
        assert conv_step(**kw) == -1 and message in err(), (kw, err())

    def step(B=2, D=8, N=4, apart=32, slots=4, state=p):
        return lib.uttt_selective_scan_step(p, st(8, 8, 0), 1, p, st(8, 8, 0), 0, p, p, st(8, 8, 8), p, st(8, 8, 8), None, None,
                                            None, None, 0, B, 1, D, N, 1, state, apart, slots, None, 0, p, None)

    for kw, message in ((dict(slots=1), "slots"), (dict(apart=31), "apart"), (dict(apart=33), "16-byte"), (dict(state=p + 4), "16-byte"),
                        (dict(N=65, apart=999), "N=65"), (dict(B=1 << 22, slots=1 << 22, D=1024, apart=1 << 12), "too many")):
        assert step(**kw) == -1 and message in err(), (kw, err())
    for N, rows, dtype, message in ((8193, 4, 1, "N=8193"), (0, 4, 1, "N=0"), (8, 1 << 31, 1, "rows"), (8, 4, 9, "dtype")):
        assert lib.uttt_norm_after_fwd(p, st(8, 8, 0), dtype, None, 0, None, None, None, None, 1, None, 0, 1.0, rows, 1, N, 1e-5, p,
                                       None, None) == -1 and message in err(), err()
    assert lib.uttt_norm_before_fwd(p, st(8, 8, 0), 1, None, None, 0, None, 0, None, 0, 1.0, 4, 1, 8, 1e-5, p, p, None,
                                    None) == -1 and "null" in err()
    assert lib.uttt_norm_before_bwd(p, st(8, 8, 0), 1, p, st(8, 8, 0), 0, p, 0, None, 0, 1.0, 4, 1, 8, p, None, None, None, None, p,
                                    p, p, None, p, 8, None) == -1 and "workspace" in err()
