"""A device wait of the training operators that gives up reaches the caller, the
last call's too: the operators do not wait for their own work, so they report it
with the next call or when asked. The wait here is the operators' own, of 1 ms,
on a barrier that nothing arrives on; nothing else is in flight."""
import pytest


def test_nothing_to_report(vc):
    assert vc.lib().vrs_operators_status() == 0


def test_limits(vc):
    assert vc.lib().vrs_selftest_operator_wait(10, None) == 5
    assert vc.lib().vrs_selftest_operator_wait(5_000_000_000, None) == 5


@pytest.mark.gpu
def test_status_tells_once(gpu, vc):
    import torch
    from vector_cuda import ops
    L = vc.lib()
    stream = torch.cuda.current_stream().cuda_stream
    assert L.vrs_selftest_operator_wait(1_000_000, stream) == 0
    torch.cuda.synchronize()
    assert L.vrs_operators_status() == 7
    assert b"stage code 98" in L.vrs_last_error()
    assert L.vrs_operators_status() == 0
    assert L.vrs_selftest_operator_wait(1_000_000, stream) == 0
    with pytest.raises(vc.CudaError):
        ops.check()
    ops.check()


@pytest.mark.gpu
def test_next_call_tells_once(gpu, vc):
    import torch
    from vector_cuda import ops
    x = torch.randn(5, 64, device="cuda")
    want = ops.layer_norm_forward(x)[0]
    assert vc.lib().vrs_selftest_operator_wait(1_000_000, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    with pytest.raises(vc.CudaError):
        ops.layer_norm_forward(x)
    assert torch.equal(ops.layer_norm_forward(x)[0], want)
    ops.check()
