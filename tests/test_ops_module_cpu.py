"""The compiled half of ops (module raptor_ops) builds, loads without a GPU and is bound to the library that capi has loaded."""
import pytest
import torch

from raptor_t_b200 import build, capi, ops


def test_module_and_its_errors():
    mod = ops._native()
    assert mod is ops._native() and mod.__file__ == build.OPS_SHIM
    for name in ("kv_cache_write", "kv_cache_read", "cached_attention", "token_logprobs", "token_logprobs_backward", "Cache"):
        assert hasattr(mod, name)
    if torch.cuda.is_available():
        pytest.skip("CPU-only behaviour")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(10))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(10, 2).t())
    with pytest.raises(TypeError):
        ops.token_logprobs("logits")
    with pytest.raises(TypeError):
        ops.KvCache(*(torch.zeros(1, 1, 64, 64, dtype=torch.uint8) for _ in range(2)), torch.zeros(1, 1), torch.zeros(1, 1))
    assert issubclass(capi.RtError, RuntimeError)
