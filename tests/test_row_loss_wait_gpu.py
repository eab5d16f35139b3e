"""A bounded wait that ran out is not passed over by the row losses: until the status is cleared every call of theirs answers with it, as the
tensor-core calls do.  The wait is one on a barrier that nothing arrives at, with a limit of one millisecond."""
import pytest

pytestmark = pytest.mark.gpu


def _calls(torch, vm, n, c):
    x = torch.randn((n, c), device="cuda")
    gx, y, ps = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty((n, 3), device="cuda")
    idx, t = torch.zeros((n, 2), dtype=torch.int32, device="cuda"), torch.zeros((n, 2), device="cuda")
    idx[:, 1] = c - 1
    z, adv = idx[:, 0].contiguous(), torch.ones(n, device="cuda")
    return {
        "distill": lambda: vm.softmax_top_distill(0, y, ps, x, idx, t, n, c, 2),
        "distill gradient": lambda: vm.softmax_top_distill_backward_x(0, gx, None, x, ps, idx, t, n, c, 2),
        "distill step": lambda: vm.softmax_top_distill_step(0, y, gx, None, x, idx, t, n, c, 2),
        "policy": lambda: vm.softmax_policy_loss(0, y, None, ps, x, z, None, None, adv, n, c),
        "policy gradient": lambda: vm.softmax_policy_loss_backward_x(0, gx, None, x, ps, z, n, c),
        "policy step": lambda: vm.softmax_policy_loss_step(0, y, None, gx, None, x, z, None, None, adv, n, c),
    }


@pytest.mark.parametrize("ncol", [100, 9001, 40000, 450001])
def test_an_expired_wait_is_reported(torch_cuda, pkg, vm, ncol):
    torch = torch_cuda
    calls = _calls(torch, vm, 3, ncol)
    for call in calls.values():
        call()
    torch.cuda.synchronize()
    lib = pkg.load()
    assert lib.kai_device_status(0, None) == 0
    try:
        pkg.capi.call("kai_selftest_bounded_wait", 0, 1_000_000, None)
        assert lib.kai_device_status(0, None) == pkg.capi.E_DEVICE_WAIT
        for name, call in calls.items():
            with pytest.raises(pkg.KaiError) as e:
                call()
            assert e.value.code == pkg.capi.E_DEVICE_WAIT, name
    finally:
        pkg.capi.call("kai_device_status_clear", 0)
    for call in calls.values():
        call()
    torch.cuda.synchronize()
    assert lib.kai_device_status(0, None) == 0
