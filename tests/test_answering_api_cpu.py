"""Refusals of the cache, attention and score entry points: no GPU is needed for what the arguments alone say."""
import ctypes as C

import pytest

from raptor_t_b200 import capi

lib = capi.lib
P = 1 << 20  # an aligned address that nobody reads


def _cache(**kw):
    f = dict(k_dev=P, v_dev=P, k_scale_dev=P, v_scale_dev=P, blocks=4, kv_heads=2, format=0, reserved=0)
    f.update(kw)
    return C.byref(capi.RtKvCache(**f))


def _write(cache=None, k=P, v=P, ts=128, hs=64, table=P, width=4, start=P, first=P, n=1, tokens=8, most=8, dtype=0):
    return lib.rt_kv_cache_write(cache or _cache(), k, v, ts, hs, table, width, start, first, n, tokens, most, dtype, None)


def _read(cache=None, k=P, v=P, table=P, width=4, start=P, first=P, n=1, tokens=8, most=8, dtype=0):
    return lib.rt_kv_cache_read(cache or _cache(), k, v, table, width, start, first, n, tokens, most, dtype, None)


def _attend(cache=None, out=P, q=P, qs=128, table=P, width=4, ctx=P, first=P, n=1, tokens=8, most=8, keys=0, heads=2, dtype=0):
    return lib.rt_cached_attention(out, q, qs, cache or _cache(), table, width, ctx, first, n, tokens, most, keys, heads, 0.125, 0,
                                   dtype, None)


def _score(z=P, pitch=100, t=P, rows=2, vocab=100, top=0, logp=P, h=P, stats=P, ids=P, best=P, dtype=0):
    return lib.rt_token_logprobs(z, pitch, t, rows, vocab, top, logp, h, stats, ids, best, dtype, None)


def _grad(out=P, op=100, z=2 * P, pitch=100, t=P, stats=P, h=P, rows=2, vocab=100, gl=P, gh=P, top=0, ids=P, gt=P, dtype=0):
    return lib.rt_token_logprobs_backward(out, op, z, pitch, t, stats, h, rows, vocab, gl, gh, top, ids, gt, dtype, None)


BAD_CACHES = [dict(k_dev=None), dict(v_scale_dev=None), dict(blocks=0), dict(kv_heads=0), dict(kv_heads=1025), dict(format=2),
              dict(k_dev=P + 8), dict(k_scale_dev=P + 2)]


@pytest.mark.parametrize("call", [_write, _read, _attend])
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_cache(call, bad):
    assert call(cache=_cache(**bad)) == capi_invalid()


def capi_invalid():
    return 1


@pytest.mark.parametrize("call,bad,code", [
    (_write, dict(k=None), 1), (_write, dict(table=None), 1), (_write, dict(first=None), 1), (_write, dict(start=None), 1),
    (_write, dict(k=P + 8), 1), (_write, dict(ts=124), 1), (_write, dict(hs=60), 1), (_write, dict(ts=-128), 1), (_write, dict(width=0), 1),
    (_write, dict(n=-1), 1), (_write, dict(dtype=2), 1), (_write, dict(most=-1), 1), (_write, dict(n=1 << 30, tokens=1 << 30, most=1 << 20), 2),
    (_read, dict(v=None), 1), (_read, dict(k=P + 4), 1), (_read, dict(dtype=7), 1), (_read, dict(tokens=-1), 1),
    (_attend, dict(q=None), 1), (_attend, dict(out=None), 1), (_attend, dict(out=P + 8), 1), (_attend, dict(qs=100), 1),
    (_attend, dict(heads=3), 2), (_attend, dict(heads=0), 1), (_attend, dict(heads=8192), 2), (_attend, dict(dtype=2), 1),
    (_attend, dict(ctx=None), 1), (_attend, dict(keys=-1), 1), (_attend, dict(n=1 << 30, tokens=1 << 30, most=1 << 26), 2),
    (_score, dict(z=None), 1), (_score, dict(pitch=99), 1), (_score, dict(vocab=0), 1), (_score, dict(top=33), 2), (_score, dict(top=-1), 2),
    (_score, dict(vocab=5, top=6), 2), (_score, dict(t=None), 1), (_score, dict(stats=None), 1), (_score, dict(stats=P + 4), 1),
    (_score, dict(top=2, ids=None), 1), (_score, dict(z=P + 1), 1), (_score, dict(z=P + 2, dtype=2), 1), (_score, dict(dtype=3), 1),
    (_score, dict(rows=-1), 1),
    (_grad, dict(out=None), 1), (_grad, dict(op=99), 1), (_grad, dict(t=None), 1), (_grad, dict(h=None), 1), (_grad, dict(stats=None), 1),
    (_grad, dict(top=1, gt=None), 1), (_grad, dict(top=33), 2), (_grad, dict(out=2 * P, op=108), 1), (_grad, dict(out=P + 1), 1),
])
def test_refusals(call, bad, code):
    assert call(**bad) == code
    assert lib.rt_last_error()


@pytest.mark.parametrize("call,none", [(_write, dict(tokens=0)), (_write, dict(n=0)), (_write, dict(most=0)), (_read, dict(tokens=0)),
                                       (_attend, dict(tokens=0)), (_attend, dict(n=0)), (_score, dict(rows=0)), (_grad, dict(rows=0))])
def test_nothing_to_do(call, none):
    """A batch without tokens is no error and needs no device."""
    before = lib.rt_kernel_launches()
    assert call(**none) == 0
    assert lib.rt_kernel_launches() == before


def test_python_refusals():
    import torch

    from raptor_t_b200 import ops
    z = torch.zeros(2, 64, 64)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(TypeError):
        ops.token_logprobs(torch.zeros(2, 10, dtype=torch.float64))
    with pytest.raises(TypeError):
        ops.KvCache(z, z, z, z)
    with pytest.raises(RuntimeError):
        ops.KvCache(*(torch.zeros(2, 1, 64, 64, dtype=torch.int8) for _ in range(2)), torch.zeros(2, 1), torch.zeros(2, 1))
    with pytest.raises(ValueError):
        ops.KvCache(torch.zeros(2, 1, 32, 64, dtype=torch.int8), z, z, z)
