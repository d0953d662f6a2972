"""The gradient of a row without a number is none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gradient_of_rows_with_nan_and_infinity(ops, dtype):
    """A row whose scores are NaN has a gradient of NaN, one of nothing but -inf a gradient of 0."""
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(6, 5000, device="cuda", generator=g).to(dtype)
    z[0, 17] = float("nan")
    z[1] = float("nan")
    z[2, 4999] = float("inf")
    z[3] = -float("inf")
    z[3, 7] = float("nan")
    z[4] = -float("inf")
    t = torch.arange(6, dtype=torch.int32, device="cuda")
    s = ops.token_logprobs(z, t, top_k=2)
    ones = torch.ones(6, device="cuda")
    for args in (dict(grad_logp=ones), dict(grad_entropy=ones), dict(grad_logp=ones, grad_entropy=ones)):
        d = ops.token_logprobs_backward(z, t, s.stats, s.entropy, **args)
        assert d[:4].isnan().all()
        assert (d[4] == 0).all() and d[5].isfinite().all()
    ops.check_device()
