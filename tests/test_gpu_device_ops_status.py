"""fa_dev_status: a bounded device wait that gives up is reported by the backend whose call it was, and once."""
import pytest

pytestmark = pytest.mark.gpu


def test_each_backend_reports_its_own_waits(built_lib):
    import torch

    from funasrnet_b200._lib import FaError, check, lib
    from funasrnet_b200.backend import CudaFloatBackend
    from funasrnet_b200.device_ops import DeviceOps

    a, b = CudaFloatBackend(0), CudaFloatBackend(0)
    ops_a, ops_b = DeviceOps(a), DeviceOps(b)
    check(lib().fa_dev_fault_test(a.handle, None))  # a wait of two seconds that nothing ends
    ops_b.status()                                  # waits for the device; the failure is not b's
    with pytest.raises(FaError, match="timeout.*gave up"):
        ops_a.status()
    ops_a.status()
    ops_b.status()
    # Both still work, and a backend made after a failure starts without one.
    check(lib().fa_dev_fault_test(b.handle, None))
    b.dispose()
    c = CudaFloatBackend(0)
    torch.cuda.synchronize()
    DeviceOps(c).status()
    x = torch.randn(3, 100, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int32, device="cuda")
    for ops in (ops_a, DeviceOps(c)):
        assert ops.adjust_logits(x, torch.empty_like(x), tokens)
        ops.status()
        assert torch.equal(tokens.long(), x.argmax(-1))
    c.dispose()
    a.dispose()
