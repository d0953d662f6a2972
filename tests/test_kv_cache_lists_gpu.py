"""Calls that do not say how many tokens a sequence brings at most: the same codes, by a grid that grows with the tokens and not with
sequences times tokens."""
import random

import pytest
import torch

import kv_reference as ref
from test_kv_cache_gpu import FORMATS, _check, _expect, _filled, _first, _i32, _tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _clone(ops, cache):
    return ops.KvCache(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seed", range(6))
def test_ragged_batches(ops, fmt, seed):
    """Sequences of no token, of one, of several blocks, wherever they start; rows behind the last one stay."""
    rng = random.Random(seed)
    n, heads = rng.choice([5, 40, 127, 128, 129, 300]), rng.choice([1, 3])
    counts = [rng.choice([0, 1, 2, 63, 64, 65, 66, 127, 128, 129, rng.randint(1, 300)]) for _ in range(n)]
    start = [rng.choice([0, 1, 62, 63, 64, rng.randint(0, 200)]) for _ in range(n)]
    g = torch.Generator().manual_seed(seed)
    rows, blocks = _tables(g, start, counts)
    T, first = sum(counts), _first(counts)
    k, v = (torch.randn(T + 5, heads, 64, generator=g).half().cuda() for _ in range(2))
    a = _filled(g, ops, blocks, heads, fmt)
    b = _clone(ops, a)
    want = _expect(a, k, v, rows, start, first) if n <= 40 else None
    args = _i32(rows), _i32(start), _i32(first)
    ops.kv_cache_write(a, k, v, *args, max_tokens=max(counts))
    ops.kv_cache_write(b, k, v, *args)
    for s, t in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(s.view(torch.int8), t.view(torch.int8))
    assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
    if want:
        _check(b, want)
    outs = []
    for most in (max(counts), None):
        out = [torch.full((T + 5, heads, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        ops.kv_cache_read(b, *args, T + 5, torch.float16, max_tokens=most, out=out)
        assert all((t[T:] == 7.0).all() for t in out)
        outs.append(out)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    ops.check_device()


def test_places_behind_the_last_sequence(ops):
    """A batch with room for more sequences than there are: zeros behind the last one's first row."""
    g = torch.Generator().manual_seed(1)
    counts = [700, 0, 500, 129]
    rows, blocks = _tables(g, [0] * 4, counts)
    width = len(rows[0])
    first = _first(counts) + [0] * 60
    x = torch.randn(sum(counts), 1, 64, generator=g).half().cuda()
    a = _filled(g, ops, blocks, 1, torch.int8)
    b = _clone(ops, a)
    args = _i32(rows + [[-1] * width] * 60), _i32([0] * 64), _i32(first)
    ops.kv_cache_write(a, x, x, *args)
    ops.kv_cache_write(b, x, x, *(t[:n].contiguous() for t, n in zip(args, (4, 4, 5))), max_tokens=700)
    assert torch.equal(a.k, b.k) and torch.equal(a.k_scale, b.k_scale)
    ops.check_device()


def test_bad_first_rows_are_reported(ops):
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(2)
    x = torch.randn(640, 1, 64, generator=g).half().cuda()
    n = 40
    table, start = _i32([[i] for i in range(n)]), _i32([0] * n)
    good = [16 * i for i in range(n + 1)]
    for first in (good[:-1] + [641], [-1] + good[1:], [-600, -500] + good[2:], good[:20] + [0] + good[21:]):
        cache = _filled(g, ops, n, 1, torch.int8)
        ops.kv_cache_write(cache, x, x, table, start, _i32(first))
        with pytest.raises(RtError) as e:
            ops.check_device()
        assert e.value.code == 1 and "1001" in str(e.value)
        out = [torch.full((640, 1, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        ops.kv_cache_read(cache, table, start, _i32(first), 640, torch.float16, out=out)
        with pytest.raises(RtError):
            ops.check_device()
    ops.check_device()


def test_more_sequences_times_tokens_than_a_grid_has(ops):
    """33,000 sequences, of which one brings 66,000 tokens: with a place for each of them everywhere there would be 2^31 and more CTAs."""
    n, most, heads = 33000, 66000, 64
    width = -(-most // 64)
    counts = [1] * n
    counts[12345] = most
    first = torch.tensor(_first(counts), dtype=torch.int32, device="cuda")
    T = sum(counts)
    assert n * heads * (most // 64) > 2 ** 31
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(n, device="cuda")
    table[12345, 1:] = torch.arange(n, n + width - 1, device="cuda")
    cache = ops.KvCache.empty(n + width, heads, torch.int8)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, 1, 64, device="cuda", generator=g).half().expand(T, heads, 64).contiguous()
    start = torch.zeros(n, dtype=torch.int32, device="cuda")
    ops.kv_cache_write(cache, x, x, table, start, first)
    k, v = ops.kv_cache_read(cache, table, start, first, T, torch.float16)
    assert torch.equal(k, v) and torch.equal(k[:, 0], k[:, -1])
    # half a code, whose unit is at most amax / 127 * 129 / 128 of the block's values, and the rounding of the result
    assert ((k[:, 0].float() - x[:, 0].float()).abs().max() <= x.abs().max().float() * (0.5 / 127 * 129 / 128 + 2.0 ** -11))
    ops.check_device()
