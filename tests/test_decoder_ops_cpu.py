"""What the decoder-training entry points refuse, without a GPU: arguments are checked before the device is looked for, so
a refused call returns its own code here and a sound one gets as far as the missing device."""
import importlib

import numpy as np
import pytest

capi = importlib.import_module("deep-learning-framework_b200").capi
BAD, LARGE, NO_HOST = capi.E_INVALID_ARG, capi.E_TOO_LARGE, capi.E_NO_HOST_PATH
A, B, C, D, E, F, G, H, I, J, K = (0x1000000 * (i + 1) for i in range(11))   # addresses that nothing reads

# name -> a sound argument list
SOUND = {
    "kai_rotary": [0, A, B, C, D, 0, 2, 3, 4, 8, 6, 0, None, 32, 32, None],
    "kai_rotary_backward": [0, A, B, C, None, 5, 2, 3, 4, 8, 8, 1, E, 40, 36, None],
    "kai_rotary_frequencies": [0, A, 64, 10000.0, 3, 8.0, 1.0, 32.0, 4096, None],
    "kai_gated_linear_forward": [0, A, B, C, D, E, F, None, None, 8, 4, 16, 8, None, None],
    "kai_gated_linear_backward": [0, A, B, C, D, E, F, G, H, I, J, K, 8, 4, 16, 8, None, 0, 0, None],
    "kai_softmax_top_distill": [0, A, B, C, D, E, 4, 100, 8, None, None],
    "kai_softmax_top_distill_backward_x": [0, A, B, C, D, E, F, 4, 100, 8, None, None],
    "kai_softmax_top_distill_step": [0, A, B, None, D, E, F, 4, 100, 8, None, None],
    "kai_softmax_policy_loss": [0, A, None, C, D, E, F, G, H, 4, 100, None, None, None, None, None],
    "kai_softmax_policy_loss_backward_x": [0, A, B, C, D, E, 4, 100, None, None],
    "kai_softmax_policy_loss_step": [0, A, None, B, None, D, E, None, None, H, 4, 100, None, None, None, None, None],
}


def _call(name, changes):
    args = list(SOUND[name])
    for i, v in changes.items():
        args[i] = v
    return getattr(capi.load(), name)(*args)


@pytest.mark.parametrize("name", sorted(SOUND))
def test_sound_arguments_reach_the_device(name):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses of this test are not to be read")
    assert _call(name, {}) > 0                       # a cudaError_t: there is no device
    assert _call(name, {0: -1}) == NO_HOST


REFUSED = [
    ("kai_rotary", {1: None}, BAD), ("kai_rotary", {2: None}, BAD), ("kai_rotary", {3: None}, BAD),
    ("kai_rotary", {10: 5}, BAD), ("kai_rotary", {10: 10}, BAD), ("kai_rotary", {10: -2}, BAD),
    ("kai_rotary", {11: 2}, BAD), ("kai_rotary", {6: -1}, BAD), ("kai_rotary", {13: 31}, BAD), ("kai_rotary", {14: 31}, BAD),
    ("kai_rotary", {2: A, 14: 33}, BAD),                                   # in place with two strides
    ("kai_rotary", {2: A + 4}, BAD),                                       # shifted by one value
    ("kai_rotary", {8: 1 << 20, 9: 1 << 12, 13: 1 << 32, 14: 1 << 32}, LARGE),
    ("kai_rotary_backward", {1: None}, BAD), ("kai_rotary_backward", {11: -1}, BAD),
    ("kai_rotary_frequencies", {1: None}, BAD), ("kai_rotary_frequencies", {2: 63}, BAD),
    ("kai_rotary_frequencies", {3: 0.0}, BAD), ("kai_rotary_frequencies", {3: float("nan")}, BAD),
    ("kai_rotary_frequencies", {4: 4}, BAD), ("kai_rotary_frequencies", {5: 0.0}, BAD),
    ("kai_rotary_frequencies", {2: 2, 4: 2}, BAD), ("kai_rotary_frequencies", {6: 32.0}, BAD),
    ("kai_rotary_frequencies", {8: 0}, BAD), ("kai_rotary_frequencies", {6: -1.0}, BAD),
    ("kai_gated_linear_forward", {1: None}, BAD), ("kai_gated_linear_forward", {2: None}, BAD),
    ("kai_gated_linear_forward", {4: None}, BAD), ("kai_gated_linear_forward", {6: None}, BAD),
    ("kai_gated_linear_forward", {12: 9}, BAD), ("kai_gated_linear_forward", {9: -1}, BAD),
    ("kai_gated_linear_forward", {2: A}, BAD), ("kai_gated_linear_forward", {1: F + 16}, BAD),
    ("kai_gated_linear_forward", {11: 1 << 31}, LARGE),
    ("kai_gated_linear_backward", {2: None}, BAD), ("kai_gated_linear_backward", {4: None}, BAD),
    ("kai_gated_linear_backward", {6: None}, BAD), ("kai_gated_linear_backward", {9: None}, BAD),
    ("kai_gated_linear_backward", {11: None}, BAD), ("kai_gated_linear_backward", {15: 9}, BAD),
    ("kai_gated_linear_backward", {5: D}, BAD), ("kai_gated_linear_backward", {3: B}, BAD),
    ("kai_gated_linear_backward", {4: G + 4}, BAD), ("kai_gated_linear_backward", {1: K}, BAD),
    ("kai_gated_linear_backward", {1: J}, BAD), ("kai_gated_linear_backward", {13: 1 << 31}, LARGE),
] + [(n, ch, code) for n, first in (("kai_softmax_top_distill", 6), ("kai_softmax_top_distill_backward_x", 7),
                                    ("kai_softmax_top_distill_step", 7))
     for ch, code in (({first: -1}, BAD), ({first + 1: 0}, BAD), ({first + 2: -1}, BAD), ({first + 2: 2049}, LARGE),
                      ({first + 1: 1 << 31}, LARGE), ({1: None}, BAD), ({first - 1: None}, BAD), ({first - 2: None}, BAD))
] + [
    ("kai_softmax_top_distill", {2: None}, BAD), ("kai_softmax_top_distill_backward_x", {4: None}, BAD),
    ("kai_softmax_top_distill_backward_x", {3: A + 4}, BAD), ("kai_softmax_top_distill_step", {4: B + 400}, BAD),
    ("kai_softmax_policy_loss", {1: None}, BAD), ("kai_softmax_policy_loss", {3: None}, BAD),
    ("kai_softmax_policy_loss", {5: None}, BAD), ("kai_softmax_policy_loss", {8: None}, BAD),
    ("kai_softmax_policy_loss", {10: 0}, BAD), ("kai_softmax_policy_loss", {9: -3}, BAD),
    ("kai_softmax_policy_loss_backward_x", {5: None}, BAD), ("kai_softmax_policy_loss_backward_x", {3: A + 1196}, BAD),
    ("kai_softmax_policy_loss_step", {3: None}, BAD), ("kai_softmax_policy_loss_step", {9: None}, BAD),
    ("kai_softmax_policy_loss_step", {5: B + 4}, BAD), ("kai_softmax_policy_loss_step", {11: 1 << 31}, LARGE),
]


@pytest.mark.parametrize("name,changes,code", REFUSED)
def test_refusals(name, changes, code):
    assert _call(name, changes) == code
    assert capi.load().kai_last_error_string().startswith(name[4:].encode())


def test_allowed_aliases_reach_the_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses of this test are not to be read")
    assert _call("kai_rotary", {2: A}) > 0                                           # in place
    assert _call("kai_rotary", {2: A + 128, 13: 96, 14: 96}) > 0                     # two parts of a packed projection
    assert _call("kai_gated_linear_backward", {4: G, 5: H}) > 0                      # over the saved factors
    assert _call("kai_gated_linear_backward", {4: F}) > 0                            # over the incoming gradient
    assert _call("kai_gated_linear_backward", {1: None}) > 0                         # no gradient for the input
    assert _call("kai_gated_linear_backward", {2: None, 3: None}) > 0                # fixed weights
    assert _call("kai_softmax_top_distill_step", {4: B}) > 0                         # gradient over the logits
    assert _call("kai_softmax_policy_loss_backward_x", {3: A}) > 0


def test_tensors_of_another_type_are_refused(vm):
    import torch
    wrong = torch.zeros(4, dtype=torch.float32)
    with pytest.raises(TypeError):
        vm.rotary(0, A, B, wrong, None, 0, 1, 1, 1, 4, 4)
    with pytest.raises(TypeError):
        vm.rotary(0, A, B, C, torch.zeros(1, dtype=torch.int32), 0, 1, 1, 1, 4, 4)
    with pytest.raises(TypeError):
        vm.softmax_policy_loss(0, A, None, B, C, torch.zeros(4, dtype=torch.int64), None, None, D, 4, 10)
    with pytest.raises(TypeError):
        vm.softmax_top_distill(0, A, B, C, torch.zeros((4, 2), dtype=torch.int64), D, 4, 10, 2)
    with pytest.raises(KeyError):
        vm.rotary(0, A, B, C, None, 0, 1, 1, 1, 4, 4, layout="quarter")


def test_angle_in_turns_keeps_far_positions():
    """The reduction the rotary kernel uses, in numpy: position * frequency in turns in 64 bits, remainder to fp32."""
    rng = np.random.default_rng(0)
    for pos in (0, 1, 99_999, 2 ** 24 + 1, 2 ** 31 + 7, -5_000_000):
        f = 10000.0 ** -rng.uniform(0, 1, 200)
        turns = pos * (f * 0.15915494309189533577)
        rest = (turns - np.rint(turns)).astype(np.float32)
        # oracle: the angle's sine in extended precision
        t = np.longdouble(pos) * f.astype(np.longdouble)
        # 2^-26 turns of rounding of the remainder; 64-bit rounding of the product and of freq / 2 pi, in turns
        tol = 2 * np.pi * (2.0 ** -26 + 3 * 2.0 ** -53 * np.abs(turns)) + 2.0 ** -52
        assert np.all(np.abs(np.sin(2 * np.pi * rest.astype(np.float64)) - np.sin(t)) <= tol)
