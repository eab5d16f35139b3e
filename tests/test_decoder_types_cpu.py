"""Tensors of another type than the call reads are refused by the Python binding before any address is used: a 16-bit tensor would be read past
its end, a 64-bit one misread."""
import inspect

import pytest

A = 0x1000000
# call -> sound positional arguments behind the device, tensors as their type's first letter: f fp32, d fp64, l int64, i int32, p not a tensor
CALLS = {
    "rotary": "ffdl" + "p" * 6,
    "rotary_backward": "ffdl" + "p" * 6,
    "rotary_frequencies": "dp",
    "gated_linear_forward": "ffffffff" + "ppp",
    "gated_linear_backward": "fffffffffff" + "ppp",
    "softmax_top_distill": "fffif" + "ppp",
    "softmax_top_distill_backward_x": "ffffif" + "ppp",
    "softmax_top_distill_step": "ffffif" + "ppp",
    "softmax_policy_loss": "ffffifff" + "pp",
    "softmax_policy_loss_backward_x": "ffffi" + "pp",
    "softmax_policy_loss_step": "fffffifff" + "pp",
}
HYPERS = {"rotary": ["hScale"], "rotary_backward": ["hScale"], "gated_linear_forward": ["leaky_alpha"],
          "gated_linear_backward": ["leaky_alpha"], "softmax_top_distill": ["hTemp"], "softmax_top_distill_backward_x": ["hTemp"],
          "softmax_top_distill_step": ["hTemp"], "softmax_policy_loss": ["hClipLow", "hClipHigh", "hKlCoef", "hTemp"],
          "softmax_policy_loss_backward_x": ["hTemp"], "softmax_policy_loss_step": ["hClipLow", "hClipHigh", "hKlCoef", "hTemp"]}


def _sound(name):
    """Extents of 0, so that nothing would be launched."""
    return [0] + [0 if c == "p" else A * (i + 1) for i, c in enumerate(CALLS[name])]


@pytest.mark.parametrize("name", sorted(CALLS))
def test_every_tensor_of_another_type(vm, name):
    import torch
    right = {"f": torch.float32, "d": torch.float64, "l": torch.int64, "i": torch.int32}
    call = getattr(vm, name)
    for at, c in enumerate(CALLS[name]):
        if c == "p":
            continue
        for kind in (torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64):
            if kind is right[c]:
                continue
            args = _sound(name)
            args[1 + at] = torch.zeros(4, dtype=kind)
            with pytest.raises(TypeError):
                call(*args)
    for hyper in HYPERS.get(name, []):
        assert hyper in inspect.signature(call).parameters
        for kind in (torch.bfloat16, torch.float64):
            with pytest.raises(TypeError):
                call(*_sound(name), **{hyper: torch.zeros(1, dtype=kind)})


@pytest.mark.parametrize("name", sorted(CALLS))
def test_every_tensor_of_its_own_type(vm, pkg, monkeypatch, name):
    """The addresses arrive as they are, and the call is made once."""
    import torch
    right = {"f": torch.float32, "d": torch.float64, "l": torch.int64, "i": torch.int32}
    made = []
    monkeypatch.setattr(pkg.capi, "call", lambda *a: made.append(a))
    args = [0] + [0 if c == "p" else torch.zeros(4, dtype=right[c]) for c in CALLS[name]]
    getattr(vm, name)(*args)
    assert len(made) == 1 and made[0][0] == "kai_" + name
    assert list(made[0][2:2 + CALLS[name].index("p")]) == [a.data_ptr() for a in args[1:] if torch.is_tensor(a)]
