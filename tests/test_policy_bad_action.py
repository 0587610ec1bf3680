"""The flag of actions beyond the vocabulary: read per device, and never confused with a CUDA error."""
import pytest
import torch


@pytest.mark.skipif(torch.cuda.is_available(), reason="takes its CUDA error from a machine without a GPU")
def test_a_cuda_error_is_not_a_bad_action():
    import pufferlib_b200 as pb
    from pufferlib_b200 import cabi
    code = cabi.load().puff_policy_sm100_bad_action()
    assert code <= cabi.ERR_CUDA_BASE - 1
    assert cabi.strerror(code) != "unknown error code" and "CUDA" in cabi.strerror(code)
    with pytest.raises(RuntimeError, match="puff_policy_sm100_bad_action"):
        pb.bad_action()


def test_error_codes_of_cuda_calls_have_texts():
    from pufferlib_b200 import cabi
    # 2 is cudaErrorMemoryAllocation, 100 cudaErrorNoDevice; a positive code is a CUDA error as ever
    for code in (2, 100):
        assert cabi.strerror(code) in cabi.strerror(cabi.ERR_CUDA_BASE - code)


@pytest.mark.gpu
def test_bad_action_of_a_device():
    import pufferlib_b200 as pb
    logits = torch.zeros(2, 5, device="cuda")
    here = torch.cuda.current_device()
    pb.bad_action()
    for device in (None, here, torch.device("cuda", here), f"cuda:{here}"):
        assert pb.bad_action(device) is False
        pb.action_logprobs(logits, torch.tensor([0, 5], device="cuda"))
        assert pb.bad_action(device) is True
        assert pb.bad_action(device) is False
