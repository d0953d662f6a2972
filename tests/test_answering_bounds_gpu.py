"""Bounds that the caller states (max_tokens, max_q), and tensors whose strides say nothing because there is one row or one head."""
import pytest
import torch

from test_kv_cache_gpu import FORMATS, _filled, _first, _i32, _tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def test_a_bound_of_zero(ops):
    """A caller who says that no sequence has a token gets one token done all the same, and more than one reported."""
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 2, 64, generator=g).half().cuda()
    table, context = _i32([[0], [2], [1]]), _i32([5, 6, 7])
    one, three = _i32([0, 1, 1, 2]), _i32([0, 0, 3, 3])
    for first, fails in ((one, False), (three, True), (_i32([0, 0, 0, 0]), False)):
        a, b = _filled(g, ops, 3, 2, torch.int8), None
        b = ops.KvCache(*(t.clone() for t in (a.k, a.v, a.k_scale, a.v_scale)))
        ops.kv_cache_write(a, x, x, table, context, first, max_tokens=0)
        if fails:
            with pytest.raises(RtError):
                ops.check_device()
        else:
            ops.kv_cache_write(b, x, x, table, context, first)
        assert torch.equal(a.k, b.k) and torch.equal(a.v_scale, b.v_scale)
        outs = []
        for bound in (0, None):
            if fails and bound is None:
                continue
            back = [torch.full((3, 2, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
            ops.kv_cache_read(a, table, _i32([0, 0, 0]), first, 3, torch.float16, max_tokens=bound, out=back)
            if fails:
                with pytest.raises(RtError):
                    ops.check_device()
            got = torch.full((3, 2, 64), 7.0, dtype=torch.float16, device="cuda")
            ops.cached_attention(x, a, table, context, first, max_q=bound, scale=0.125, out=got)
            if fails:
                with pytest.raises(RtError):
                    ops.check_device()
            outs.append([*back, got])
        if fails:
            assert all((t == 7.0).all() for t in outs[0])
        else:
            assert all(torch.equal(s, t) for s, t in zip(*outs))
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
def test_strides_that_say_nothing(ops, fmt):
    """One token, or one head: the stride over it may be any number."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(5000, generator=g).half().cuda()
    table, first = _i32([[1, 0]]), _i32([0, 1])
    # one token
    x = base[:192].view(1, 3, 64)
    odd = torch.as_strided(base, (1, 3, 64), (7, 64, 1))
    zero = torch.as_strided(base, (1, 3, 64), (0, 64, 1))
    caches = [_filled(torch.Generator().manual_seed(4), ops, 2, 3, fmt) for _ in range(4)]
    for cache, k, v in zip(caches, (x, odd, zero, odd), (x, odd, zero, x)):
        ops.kv_cache_write(cache, k, v, table, _i32([70]), first)
    outs = [ops.cached_attention(q, cache, table, _i32([71]), first, scale=0.125) for cache, q in zip(caches, (x, odd, zero, x))]
    for cache, o in zip(caches[1:], outs[1:]):
        assert torch.equal(cache.k.view(torch.int8), caches[0].k.view(torch.int8)) and torch.equal(cache.v_scale, caches[0].v_scale)
        assert torch.equal(o, outs[0])
    # one head
    y = base[:640].view(10, 1, 64)
    odd = torch.as_strided(base, (10, 1, 64), (64, 3, 1))
    caches = [_filled(torch.Generator().manual_seed(4), ops, 2, 1, fmt) for _ in range(3)]
    first = _i32([0, 10])
    for cache, k, v in zip(caches, (y, odd, odd), (y, odd, y)):
        ops.kv_cache_write(cache, k, v, table, _i32([60]), first)
    outs = [ops.cached_attention(q, cache, table, _i32([70]), first, scale=0.125) for cache, q in zip(caches, (y, odd, y))]
    for cache, o in zip(caches[1:], outs[1:]):
        assert torch.equal(cache.k.view(torch.int8), caches[0].k.view(torch.int8)) and torch.equal(o, outs[0])
    ops.check_device()


def test_output_over_the_queries_is_refused(ops):
    """Every row's keys are read after other rows have been written."""
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(5)
    cache = _filled(g, ops, 2, 2, torch.int8)
    store = torch.randn(40, 2, 64, generator=g).half().cuda()
    args = cache, _i32([[0, 1]]), _i32([100]), _i32([0, 20])
    want = ops.cached_attention(store[:20], *args, scale=0.125)
    for out in (store[:20], store[19:39]):
        with pytest.raises(RtError) as e:
            ops.cached_attention(store[:20], *args, scale=0.125, out=out)
        assert e.value.code == 1
    assert torch.equal(ops.cached_attention(store[:20], *args, scale=0.125, out=store[20:]), want)
    # between the rows of wider ones: one row of output in the gap of the queries' buffer
    wide = torch.randn(20, 3 * 128, generator=g).half().cuda()
    q = wide[:1, :128].unflatten(1, (2, 64))
    one = cache, _i32([[0, 1]]), _i32([100]), _i32([0, 1])
    want = ops.cached_attention(q, *one, scale=0.125)
    assert torch.equal(ops.cached_attention(q, *one, scale=0.125, out=wide[:1, 128:256].view(1, 2, 64)), want)
    ops.check_device()
