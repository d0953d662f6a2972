"""Writing into blocks whose scales were made elsewhere: any positive number, not only what the writer itself chooses."""
import math

import pytest
import torch

import kv_reference as ref
from test_kv_cache_gpu import DTYPES, FORMATS, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _cache(ops, fmt, scale):
    """One block of one head whose first place is taken."""
    cache = ops.KvCache.empty(1, 1, fmt)
    for t in (cache.k, cache.v):
        t.view(torch.int8).zero_()
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(scale)
    return cache


def _write(ops, cache, x):
    """x [n, 64] into the places from 1 on; the codes there."""
    n = x.shape[0]
    y = x.unsqueeze(1).contiguous().cuda()
    ops.kv_cache_write(cache, y, y, _i32([[0]]), _i32([1]), _i32([0, n]))
    assert torch.equal(cache.k.view(torch.int8), cache.v.view(torch.int8))
    return cache.k[0, 0, 1:1 + n].cpu().double()


def _ties(fmt):
    """Values half-way between two neighbouring codes."""
    if fmt == torch.int8:
        return torch.arange(-126.5, 127, 1.0).double()
    codes = torch.arange(0, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    return torch.cat([mid, -mid])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("odd", [1, 3, 5, 7, 9, 11, 13, 15, 25, 31])
def test_ties_of_kept_scales(ops, fmt, odd):
    """x / scale on a border between two codes goes to the even one, also where 1 / scale has no end."""
    scale = odd * 2.0 ** -6
    x = _ties(fmt) * scale
    exact = x.half().double() == x
    x = x[exact & (x.abs() <= ref.MAX[fmt] * (scale if fmt == torch.int8 else 2.0 ** math.floor(math.log2(scale))))]  # the scale stays
    assert x.numel() > 40
    x = torch.cat([x, x.new_zeros(-x.numel() % 64)]).view(-1, 64)
    for part in x.split(63):
        cache = _cache(ops, fmt, scale)
        got = _write(ops, cache, part.half())
        assert cache.k_scale.item() == scale  # it fits all of them
        want = ref.codes(part / scale, fmt)
        assert torch.equal(got, want), (part[got != want][:4], got[got != want][:4])
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_kept_scale(ops, fmt, dtype):
    """Scales with all 24 bits: the code of the quotient as fp32 has it."""
    g = torch.Generator().manual_seed(7)
    for scale in (torch.rand(8, generator=g) + 0.5).tolist() + [0.3, 1e-3, 3e4, 2.0 ** -99 * 1.7]:
        scale = torch.tensor(scale, dtype=torch.float32)
        x = (torch.randn(63, 64, generator=g) * scale * ref.MAX[fmt] / 5).clamp(-6e4, 6e4).to(dtype)
        cache = _cache(ops, fmt, scale.item())
        if ref.needed_scale(x.double().abs().max().item(), fmt) > scale:
            x = (x.double() / 2).to(dtype)
        got = _write(ops, cache, x)
        assert cache.k_scale.item() == scale.item()
        assert torch.equal(got, ref.codes((x.float() / scale).double(), fmt))
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [2.0 ** -100, 0.75, 1e37, 2.0 ** 120])
def test_infinities_take_the_largest_code(ops, fmt, dtype, scale):
    """Also where the largest code times the scale is no fp32 number."""
    x = torch.zeros(2, 64)
    x[0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), scale if scale < 6e4 and scale > 1e-3 else 0.0])
    cache = _cache(ops, fmt, scale)
    got = _write(ops, cache, x.to(dtype))
    top = ref.MAX[fmt]
    assert got[0, :4].tolist() == [top, -top, 0.0, 1.0 if 1e-3 < scale < 6e4 else 0.0]
    assert (got[0, 4:] == 0).all() and (got[1] == 0).all()
    ops.check_device()
