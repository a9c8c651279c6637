"""What the memory layer's calls hand to the C ABI, without a GPU."""
import ctypes
import os

import pytest
import torch

from uttt_amd import _lib, delta

BF16, F32 = torch.bfloat16, torch.float32
E = dict(device="meta")


@pytest.fixture
def launched(monkeypatch):
    """The calls up to their launch, on meta tensors."""
    calls = []
    monkeypatch.setattr(delta.L, "call_on", lambda t, name, *args: calls.append((name, args)))
    monkeypatch.setattr(delta.L, "stream_of", lambda t: 0)
    return calls


def step_inputs(B=1):
    e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, **E)  # noqa: E731
    return e(B, 1, 1, 64), e(B, 1, 1, 64), e(B, 1, 2, 32), e(B, 1, 2, dtype=F32), e(B, 1, 2, dtype=F32)


@pytest.mark.parametrize("stride", [0, 1, 5, 64, 4095, 4097, 2 ** 40 + 1])
def test_one_state_with_a_stride_of_no_use(launched, stride):
    """The stride along a slot axis of one says nothing: the C ABI, which wants a
    multiple of 4, gets the state's own size."""
    state = torch.empty(2 * 64 * 32, dtype=F32, **E).as_strided((1, 2, 64, 32), (stride, 64 * 32, 32, 1))
    delta.gated_delta_step(*step_inputs(), state)
    (name, args), = launched
    assert name == "uttt_gated_delta_step" and args[19] == 2 * 64 * 32 and args[20] == 1


def test_the_stride_of_several_states(launched):
    pool = torch.empty(3, 5, 2, 64, 32, dtype=F32, **E)
    delta.gated_delta_step(*step_inputs(3), pool[:, 1])
    assert launched[0][1][19] == 5 * 2 * 64 * 32


needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


@needs_lib
def test_launches_of_too_many_threads_are_refused():
    """A launch has fewer than 2^32 threads: said by the argument check, before
    anything is launched (the addresses are never read)."""
    lib, p = _lib.lib(), 1 << 20
    st = (ctypes.c_int64 * 3)(8, 8, 8)
    err = lambda: lib.uttt_last_error().decode()  # noqa: E731

    def rule(B, T, H, Dk=8, Dv=8, bwd=False, cu=None, n=None):
        head = (p, st, p, st, p, st, p, 0, p, 0, cu, 0, B, T, B if n is None else n, H, H, Dk, Dv, 1.0)
        big = 1 << 62
        if bwd:
            return lib.uttt_gated_delta_bwd(*head, p, p, p, st, None, p, p, p, p, p, None, p, big, None)
        return lib.uttt_gated_delta_fwd(*head, None, p, None, None, None, p, big, None)

    for kw in (dict(B=1 << 20, T=1, H=16),                       # the scan: 512 threads a head
               dict(B=1, T=1 << 20, H=1 << 10),                  # the operands: 256 threads a chunk and head
               dict(B=1, T=1 << 18, H=1 << 10, Dk=256, bwd=True),   # the gradients: 1024
               dict(B=1, T=100, H=16, cu=p, n=1 << 20)):
        assert rule(**kw) == -1 and "too many" in err(), (kw, err())

    def step(B, Hv, Dv):
        return lib.uttt_gated_delta_step(p, st, p, st, p, st, 1, p, 0, p, 0, B, 1, 1, Hv, 8, Dv, 1.0, p, Hv * 8 * Dv, B, None,
                                         0, p, None)

    assert step(1 << 20, 16, 64) == -1 and "too many" in err()
    assert step(1 << 20, 4, 260) == -1 and "too many" in err()
    sections = (ctypes.c_int * 1)(1100)
    assert lib.uttt_rotary_axes(p, 1, st, 1, 1 << 24, 1, 2200, p, 0, st, p, sections, 1, 0, 0, p, None) == -1
    assert "too many" in err()
