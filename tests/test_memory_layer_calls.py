"""What the memory layer's calls hand to the C ABI, without a GPU."""
import pytest
import torch

from uttt_amd import delta

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
