"""The fault counters are those of every stream of the device: a call that still
waits in a stream of PyTorch's (which the CUDA runtime's symbol copies do not
wait for) is counted when the counter is read, and not after it was reset."""
import pytest
import torch

from sm120_rmsnorm import capi, fused_add_rms_norm_inplace, serving_capi
from test_gpu_attention import Prompt

pytestmark = pytest.mark.gpu
SLEEP = 200_000_000  # cycles: 0.1 s


def norm_call():
    x, r = (torch.randn(2048, 4096, device="cuda").to(torch.bfloat16) for _ in "xr")
    w = torch.ones(4096, device="cuda", dtype=torch.bfloat16)
    return lambda: fused_add_rms_norm_inplace(x, r, w)


def prompt_call():
    c = Prompt([300], seed=1)
    starts = torch.tensor(c.starts, dtype=torch.int32, device="cuda")
    from sm120_rmsnorm import serving
    return lambda: serving.prompt_attention(c.out, c.q, c.k, c.v, starts)


@pytest.mark.parametrize("library, call", [(capi, norm_call), (serving_capi, prompt_call)])
def test_counters_wait_for_all_streams(library, call):
    run = call()
    run()
    torch.cuda.synchronize()
    library.reset_device_faults()
    stream = torch.cuda.Stream()

    def late_fault():
        with torch.cuda.stream(stream):
            torch.cuda._sleep(SLEEP)
            run()

    capi.set_wait_limit(1)
    try:
        late_fault()
        assert library.device_faults() > 0
        late_fault()
        library.reset_device_faults()
        torch.cuda.synchronize()
        assert library.device_faults() == 0
    finally:
        torch.cuda.synchronize()
        capi.set_wait_limit(0)
        library.reset_device_faults()
