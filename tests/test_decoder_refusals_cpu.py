"""Overlaps and sizes that the decoder-training entry points refuse, without a GPU (a refused call returns its own code before the device is
looked for; a sound one gets as far as the missing device)."""
import importlib

import pytest

from test_decoder_ops_cpu import A, B, C, D, E, F, G, H, I, J, K, SOUND, _call

capi = importlib.import_module("deep-learning-framework_b200").capi
BAD, LARGE = capi.E_INVALID_ARG, capi.E_TOO_LARGE


def _on_the_device(name, changes):
    """A sound call: it may only fail for want of a device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses of this test are not to be read")
    assert _call(name, changes) > 0


# gated layer: yvec 8, ndat 4, xvec 16; a weight is 512 bytes, a bias 32, an output 128
@pytest.mark.parametrize("name,changes", [
    ("kai_gated_linear_forward", {1: D}), ("kai_gated_linear_forward", {1: E + 508}), ("kai_gated_linear_forward", {2: D - 124}),
    ("kai_gated_linear_forward", {3: E}), ("kai_gated_linear_forward", {7: A + 64}), ("kai_gated_linear_forward", {8: B}),
    ("kai_gated_linear_forward", {8: C + 124}),
    ("kai_gated_linear_backward", {2: I}), ("kai_gated_linear_backward", {2: J}), ("kai_gated_linear_backward", {3: I - 4}),
    ("kai_gated_linear_backward", {3: J + 508}), ("kai_gated_linear_backward", {4: I}), ("kai_gated_linear_backward", {5: J + 400}),
])
def test_gated_outputs_over_weights_and_biases(name, changes):
    assert _call(name, changes) == BAD


def test_gated_neighbours_are_no_overlap():
    _on_the_device("kai_gated_linear_forward", {1: D + 512, 2: E - 128, 3: E + 512, 7: A - 32, 8: A + 128})
    _on_the_device("kai_gated_linear_backward", {2: I + 512, 3: J + 512, 4: I - 128, 5: J - 128})


def test_an_empty_operand_lies_nowhere():
    """Whatever its address: a call without rows is not refused for a pointer that falls into another buffer."""
    _on_the_device("kai_gated_linear_backward", {1: B + 64, 13: 0})
    _on_the_device("kai_gated_linear_forward", {1: D + 64, 10: 0})
    _on_the_device("kai_softmax_top_distill_step", {4: B + 4, 7: 0})
