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


# rotary: 2 x 3 tokens of 4 heads x 8 values; arguments 6 to 9 are nbat, ntimes, nhead, npiece, 13 and 14 the strides of output and input
@pytest.mark.parametrize("changes", [
    {2: A + 64, 13: 96, 14: 96},                  # rows of 128 bytes, half a row on
    {2: A + 96 * 4 - 64, 13: 96, 14: 96},         # half a row in front of the next one
    {2: A - 64, 13: 96, 14: 96},
    {2: A + 5 * 96 * 4 + 124, 13: 96, 14: 96},    # the last row's last value
    {2: A + 3 * 96 * 4, 13: 96, 14: 96},          # whole rows, three on
    {2: A + 2, 13: 96, 14: 96},
    {2: A + 128, 13: 96, 14: 64},                 # strides of 384 and 256 bytes
    {2: A + 300, 13: 64, 14: 32},
    {2: A + 4, 7: 1, 6: 1, 13: 96, 14: 40},       # one row: strides do not matter
])
@pytest.mark.parametrize("name", ["kai_rotary", "kai_rotary_backward"])
def test_rotary_rows_that_overlap(name, changes):
    assert _call(name, {10: 6, **changes}) == BAD


@pytest.mark.parametrize("changes", [
    {2: A, 13: 96, 14: 96}, {2: A + 128, 13: 96, 14: 96}, {2: A + 256, 13: 96, 14: 96}, {2: A - 128, 13: 96, 14: 96},
    {2: A + 6 * 96 * 4, 13: 96, 14: 96}, {2: A + 5 * 96 * 4 + 128, 13: 96, 14: 96},
    {2: A + 128, 13: 96, 14: 192}, {2: A + 128, 13: 128, 14: 64}, {2: A + 128, 6: 1, 7: 1, 13: 96, 14: 40},
])
def test_rotary_rows_that_do_not(changes):
    _on_the_device("kai_rotary", changes)


def test_rotary_rows_against_a_list_of_every_value():
    """The same answer as from the sets of addresses themselves, for many small strides, shifts and numbers of rows."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses of this test are not to be read")
    rng = __import__("random").Random(5)
    seen = set()
    for _ in range(3000):
        rows, w = rng.randint(1, 5), rng.randint(1, 4) * 2
        ldy, ldx = (w + rng.randint(0, 9) for _ in range(2))
        if rng.random() < 0.5:
            ldx = ldy
        shift = rng.randint(-60, 60)
        if shift == 0:
            continue
        y = {i * ldy + c for i in range(rows) for c in range(w)}
        x = {shift + i * ldx + c for i in range(rows) for c in range(w)}
        got = _call("kai_rotary", {2: A + 4 * shift, 6: 1, 7: rows, 8: 1, 9: w, 10: w, 13: ldy, 14: ldx})
        assert (got == BAD) == bool(x & y), (rows, w, ldy, ldx, shift)
        seen.add((got == BAD, ldx == ldy))
    assert len(seen) == 4


@pytest.mark.parametrize("name,changes", [
    # products that come to 0 or below modulo 2^64
    ("kai_rotary", {6: 1 << 30, 7: 1 << 30, 8: 1, 9: 16}), ("kai_rotary", {6: 1 << 30, 7: 1 << 30, 8: 1, 9: 8}),
    ("kai_rotary_backward", {6: 1 << 30, 7: 1 << 30, 8: 1, 9: 16, 10: 16}), ("kai_rotary", {6: 1 << 30, 7: 1 << 20, 13: 1 << 40}),
    ("kai_rotary", {14: 1 << 62}),
    ("kai_softmax_top_distill", {6: 1 << 62, 7: 4}), ("kai_softmax_top_distill_step", {7: 1 << 33, 8: (1 << 31) - 1}),
    ("kai_softmax_top_distill_backward_x", {7: 1 << 60, 8: 16}), ("kai_softmax_policy_loss", {9: 1 << 62, 10: 4}),
    ("kai_softmax_policy_loss_backward_x", {6: 1 << 60, 7: 16}), ("kai_softmax_policy_loss_step", {10: 1 << 62, 11: 1}),
    ("kai_softmax_top_distill", {6: 1 << 56, 7: 1, 8: 2048}),
])
def test_more_bytes_than_addresses(name, changes):
    assert _call(name, changes) == LARGE


# row losses: 4 rows of 100 columns (1600 bytes), 8 labels (128 bytes), per-row vectors of 16 bytes, statistics of 48
@pytest.mark.parametrize("name,changes", [
    ("kai_softmax_top_distill", {1: C + 1584}), ("kai_softmax_top_distill", {2: C}), ("kai_softmax_top_distill", {2: C - 44}),
    ("kai_softmax_top_distill", {1: B + 32}), ("kai_softmax_top_distill", {1: D}), ("kai_softmax_top_distill", {2: E + 124}),
    ("kai_softmax_top_distill_backward_x", {2: A + 16}), ("kai_softmax_top_distill_backward_x", {4: A + 1596}),
    ("kai_softmax_top_distill_backward_x", {5: A}), ("kai_softmax_top_distill_backward_x", {1: F - 1596}),
    ("kai_softmax_top_distill_step", {1: B}), ("kai_softmax_top_distill_step", {3: A}), ("kai_softmax_top_distill_step", {3: B + 800}),
    ("kai_softmax_top_distill_step", {1: D + 4}), ("kai_softmax_top_distill_step", {2: E}),
    ("kai_softmax_policy_loss", {1: D}), ("kai_softmax_policy_loss", {2: A}), ("kai_softmax_policy_loss", {3: A - 44}),
    ("kai_softmax_policy_loss", {2: E}), ("kai_softmax_policy_loss", {1: H + 12}), ("kai_softmax_policy_loss", {3: G}),
    ("kai_softmax_policy_loss_backward_x", {5: A + 4}), ("kai_softmax_policy_loss_backward_x", {2: A}),
    ("kai_softmax_policy_loss_backward_x", {4: A + 1552}),
    ("kai_softmax_policy_loss_step", {4: A}), ("kai_softmax_policy_loss_step", {2: A}), ("kai_softmax_policy_loss_step", {1: B + 1584}),
    ("kai_softmax_policy_loss_step", {2: D}), ("kai_softmax_policy_loss_step", {9: B + 1596}), ("kai_softmax_policy_loss_step", {7: B}),
    ("kai_softmax_policy_loss_step", {8: A}),
])
def test_row_loss_buffers_that_overlap(name, changes):
    assert _call(name, changes) == BAD
    assert b"overlap" in capi.load().kai_last_error_string()


def test_row_loss_neighbours_are_no_overlap():
    _on_the_device("kai_softmax_top_distill", {1: C + 1600, 2: C - 48})
    _on_the_device("kai_softmax_top_distill_step", {4: B, 1: B + 1600, 3: B - 16})
    _on_the_device("kai_softmax_policy_loss", {1: A, 2: A + 16, 3: A + 32, 4: A + 80})
    _on_the_device("kai_softmax_policy_loss_step", {2: A + 16, 5: B, 9: B + 1600, 7: B + 1616, 8: B + 1616})
    _on_the_device("kai_softmax_policy_loss_backward_x", {3: A, 2: A + 1600})
