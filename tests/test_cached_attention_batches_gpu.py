"""Batches of many tiles: on both sides of the rules that order them and that look for their sequences."""
import random

import pytest
import torch

from test_cached_attention_gpu import _case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("n,heads", [(60, 3), (149, 1), (256, 1), (257, 1), (300, 4)])
@pytest.mark.parametrize("causal", [False, True])
def test_many_tiles(ops, n, heads, causal):
    """One tile or two a sequence, some without rows or keys, up to 256 of them ranked by length and more in order."""
    rng = random.Random(n)
    counts = [rng.choice([0, 65, 70, rng.randint(1, 130), rng.randint(66, 256)]) for _ in range(n)]
    context = [rng.choice([0, 1, 64, rng.randint(1, 300), rng.randint(1, 900)]) for _ in range(n)]
    _case(ops, torch.int8, torch.float16, heads, heads, counts, context, causal, spare_rows=3, max_q=256)
    counts[n // 2] = 300
    _case(ops, torch.float8_e4m3fn, torch.bfloat16, heads, heads, counts, context, causal, max_q=300)
