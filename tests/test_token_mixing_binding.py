"""The Python side of the token-mixing calls, on the CPU: tensors of the wrong
place, type, shape or layout are refused before any address is passed on."""
import pytest
import torch

import mcv_b200


def half(*shape):
    return torch.zeros(*shape).half()


def delta(n=3, heads=2, dk=64, dv=32):
    return [half(n, heads, dk), half(n, heads, dk), half(n, heads, dv), torch.zeros(n, heads), torch.zeros(n, heads)]


def test_host_tensors_are_refused():
    """Calls whose tensors agree with each other but lie in host memory."""
    x, pos = half(3, 2, 64), torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="mrope: tensors must be on a CUDA device"):
        mcv_b200.mrope(x, pos, mcv_b200.MRope(64, [32]), half(3, 2, 64))
    with pytest.raises(RuntimeError, match="gated_delta_step: tensors must be on a CUDA device"):
        mcv_b200.gated_delta_step(*delta(), torch.zeros(3, 2, 64, 32), half(3, 2, 32))
    ws = torch.zeros(mcv_b200.lib().mcv_gated_delta_workspace_size(3, 1, 2, 64, 32), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="gated_delta_prefill: tensors must be on a CUDA device"):
        mcv_b200.gated_delta_prefill(*delta(), torch.tensor([0, 3], dtype=torch.int32), None, half(3, 2, 32), ws)


def test_workspace_layout():
    """A workspace whose elements share memory is refused whatever its size in bytes."""
    n = mcv_b200.lib().mcv_gated_delta_workspace_size(3, 1, 2, 64, 32)
    with pytest.raises(RuntimeError, match="workspace must be contiguous"):
        mcv_b200.gated_delta_prefill(*delta(), torch.tensor([0, 3], dtype=torch.int32), None, half(3, 2, 32),
                                     torch.zeros(1, dtype=torch.uint8).expand(n))


@pytest.mark.parametrize("which,bad,match", [
    (0, half(3, 2, 128)[:, :, ::2], "rows of q"), (0, torch.zeros(3, 2, 64), "q must be float16"),
    (1, half(3, 2, 32), "do not fit together"), (2, half(4, 2, 32), "do not fit together"),
    (3, torch.zeros(3, 2).double(), "g must be"), (3, torch.zeros(2, 3).t(), "g must be"), (4, torch.zeros(3, 1), "beta must be")])
def test_delta_tensors(which, bad, match):
    args = delta()
    args[which] = bad
    with pytest.raises(RuntimeError, match=match):
        mcv_b200.gated_delta_step(*args, torch.zeros(3, 2, 64, 32), half(3, 2, 32))


def test_delta_outputs_and_states():
    state, out = torch.zeros(3, 2, 64, 32), half(3, 2, 32)
    with pytest.raises(RuntimeError, match="state must be"):
        mcv_b200.gated_delta_step(*delta(), torch.zeros(3, 2, 32, 64).transpose(2, 3), out)
    with pytest.raises(RuntimeError, match="state_out must be"):
        mcv_b200.gated_delta_step(*delta(), state, out, state_out=torch.zeros(4, 2, 64, 32))
    with pytest.raises(RuntimeError, match="out must be"):
        mcv_b200.gated_delta_step(*delta(), state, half(3, 2, 16))
    with pytest.raises(RuntimeError, match="index must be"):
        mcv_b200.gated_delta_step(*delta(), state, out, index=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        mcv_b200.gated_delta_step(*delta()[:4], [0.0], state, out)
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        mcv_b200.gated_delta_prefill(*delta(), torch.zeros(1, dtype=torch.int32), None, out, torch.zeros(1, dtype=torch.uint8))


def test_output_over_its_input():
    """An output at the input's address is that input in place; one of another layout there is refused."""
    wide = half(3, 2, 128)
    x, dense = wide[:, :, :64], wide.view(-1)[:3 * 2 * 64].view(3, 2, 64)
    pos, rope = torch.zeros(1, 3, dtype=torch.int32), mcv_b200.MRope(64, [32])
    with pytest.raises(RuntimeError, match="out begins where its input does"):
        mcv_b200.mrope(x, pos, rope, dense)
    with pytest.raises(RuntimeError, match="CUDA device"):      # the input itself passes this check
        mcv_b200.mrope(x, pos, rope, x)


def test_strides_of_single_tokens_and_heads():
    """A dimension of size 1 may have any stride: a slice of one row of a wide projection, one head of many."""
    import mcv_b200 as mcv
    mcv._torch or mcv._setup()
    wide = half(1, 2049)
    assert wide.stride(0) == 2049
    assert mcv._f16_rows(wide[:, :2048].view(1, 8, 256), "q", -1)[1:] == (0, 256)
    assert mcv._f16_rows(half(3, 64).as_strided((3, 1, 64), (64, 5, 1)), "q", -1)[1:] == (64, 0)
    assert mcv._f16_rows(half(3, 2, 64), "q", -1)[1:] == (128, 64)
