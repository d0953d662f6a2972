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


@pytest.mark.parametrize("group,kv_heads", [(1, 2), (3, 1)])
@pytest.mark.parametrize("seed", range(4))
def test_no_bound_for_the_rows_of_a_sequence(ops, group, kv_heads, seed):
    """Without max_q any sequence may have all rows: lengths around the tiles' ends, sequences without rows, rows behind the last one."""
    rng = random.Random(seed)
    n = [9, 40, 260, 800][seed]
    counts = [rng.choice([0, 1, 255, 256, 257, rng.randint(1, 600)]) if rng.random() < min(1, 30 / n) else rng.randint(0, 2) for _ in range(n)]
    context = [c + rng.choice([0, 1, 64, rng.randint(1, 300)]) for c in counts]
    for causal in (False, True):
        _case(ops, rng.choice([torch.int8, torch.float8_e4m3fn]), torch.float16, group * kv_heads, kv_heads, counts, context, causal, spare_rows=5)


def test_bad_first_rows_are_reported(ops):
    from raptor_t_b200.capi import RtError
    from test_kv_cache_gpu import _filled, _i32
    g = torch.Generator().manual_seed(2)
    n, cache = 40, _filled(g, ops, 40, 1, torch.int8)
    q = torch.randn(640, 1, 64, generator=g).half().cuda()
    table, context = _i32([[i] for i in range(n)]), _i32([50] * n)
    good = [16 * i for i in range(n + 1)]
    want = ops.cached_attention(q, cache, table, context, _i32(good), scale=0.125)
    assert torch.equal(want, ops.cached_attention(q, cache, table, context, _i32(good), max_q=200, scale=0.125))
    for first in (good[:-1] + [641], [-1] + good[1:], [-600, -500] + good[2:]):
        ops.cached_attention(q, cache, table, context, _i32(first), scale=0.125)
        with pytest.raises(RtError) as e:
            ops.check_device()
        assert e.value.code == 1 and "1003" in str(e.value)
    ops.check_device()


def test_many_sequences_with_many_rows_each(ops):
    """80,000 rows of 4,100 sequences: with all tiles for each sequence there would be 2^28 and more CTAs."""
    from test_kv_cache_gpu import _filled, _i32
    g = torch.Generator().manual_seed(3)
    n, heads, rows = 4100, 64, 80000
    cache = _filled(g, ops, 3, heads, torch.int8)
    first = torch.arange(n + 1, device="cuda").int()
    first[n // 2 + 1:] += rows - n
    q = torch.randn(64, heads, 64, generator=g).half().cuda().repeat(rows // 64, 1, 1)
    table = torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    table[:, 1] = 2
    context = torch.full((n,), 100, dtype=torch.int32, device="cuda")
    got = ops.cached_attention(q, cache, table, context, first, scale=0.125)
    want = ops.cached_attention(q[:64], cache, _i32([[0, 2]]), _i32([100]), _i32([0, 64]), scale=0.125)
    # the same rows in tiles of other shapes: two roundings to halves of probabilities, and of the output
    off = (got.view(rows // 64, 64, heads, 64).float() - want.float()[None]).abs().max()
    assert off <= 4 * 2.0 ** -11 * (cache.v.float().abs().amax() * cache.v_scale.max())
    ops.check_device()
