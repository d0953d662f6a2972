"""Attention over blocks whose scales differ by many orders of magnitude, or are no numbers: a row depends on the keys that it
sees and on nothing else, whichever kernel its batch gets."""
import math

import pytest
import torch

from test_kv_cache_gpu import FORMATS, _filled, _i32

pytestmark = pytest.mark.gpu

ROWS = [1, 12, 40, 100, 300]  # tiles of 8 and 16 rows, one row tile and two
COPIES = [1, 160]  # of a sequence in a call: with one its blocks are spread over CTAs, with many a CTA takes all blocks of a tile


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _values(code, scale):
    return code.cpu().double() * scale.cpu().double()[:, :, None, None]


def _reference(q, cache, table, ctx, scale, causal):
    """Outputs of one sequence in 64 bits, and how far a kernel's may be from them: sums over the keys that the row sees.

    With p the probabilities before they are divided by their sum (the largest 1), a kernel rounds each to a half (2^-11 of it;
    what is below 2^-14 of its scaled reference is off by 2^-32 of that, or lost), its exponentials and scores are off by 2^-13
    together, twice because of the sum, and the offset that int8 codes carry leaves 2^-16 of a code's unit."""
    rows = q.shape[0]
    k, v = (_values(c, s)[table].transpose(0, 1).flatten(1, 2)[:, :ctx] for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    unit = cache.v_scale.cpu().double()[table].repeat_interleave(64, 0)[:ctx].t()  # [heads, keys]
    z = torch.einsum("thd,hkd->htk", q.cpu().double(), k) * scale
    if causal:
        seen = torch.arange(ctx)[None] <= ctx - rows + torch.arange(rows)[:, None]
        z = z.masked_fill(~seen, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m.isinf(), 0.0, m))
    total = p.sum(-1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    want = torch.einsum("htk,hkd->thd", p / total, v)
    there = (p > 0).double()
    tol = (2.0 ** -11 + 2.0 ** -12) * torch.einsum("htk,hkd->thd", p / total, v.abs())
    tol += torch.einsum("htk,hkd->thd", torch.minimum(p, 2.0 ** -31 * there), v.abs())
    tol += (2.0 ** -31 * 448 * ctx * (p * unit[:, None]).amax(-1) + 2.0 ** -15 * (p / total * unit[:, None]).sum(-1)).t()[:, :, None]
    return want, tol + torch.finfo(q.dtype).eps / 2 * want.abs()


def _attend(ops, q, cache, table, ctx, copies, causal):
    rows = q.shape[0]
    got = ops.cached_attention(q.repeat(copies, 1, 1), cache, _i32([table] * copies), _i32([ctx] * copies),
                               _i32([rows * i for i in range(copies + 1)]), max_q=rows, scale=0.125, causal=causal)
    got = got.unflatten(0, (copies, rows))
    assert (got == got[:1]).all() or got.isnan().any()
    return got[-1]


def _check(got, want, tol):
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), ((off / tol.clamp(min=1e-300)).nan_to_num(nan=math.inf).max().item(), got.isnan().sum().item())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("octaves", [10, 24, 40, 70])
def test_later_values_do_not_touch_earlier_rows(ops, fmt, rows, octaves):
    """The last tokens' values are far larger than all before: only the rows that see them may notice."""
    g = torch.Generator().manual_seed(rows + octaves)
    cache = _filled(g, ops, 9, 2, fmt)
    cache.k_scale.mul_(2.0 ** -2)
    table, ctx = [7, 2, 8, 0, 5, 3, 1, 6], 500
    cache.v_scale[table[-1]] *= 2.0 ** octaves  # tokens 448 to 499
    q = torch.randn(rows, 2, 64, generator=g).bfloat16().cuda()
    for causal in (True, False):
        want = _reference(q, cache, table, ctx, 0.125, causal)
        for copies in COPIES:
            _check(_attend(ops, q, cache, table, ctx, copies, causal), *want)
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("octaves", [24, 60, 100])
def test_rows_that_look_at_small_values(ops, fmt, rows, octaves):
    """Every row sees blocks with large values and blocks with small ones, and nearly all its weight lies on one of the two."""
    g = torch.Generator().manual_seed(rows + octaves)
    cache = _filled(g, ops, 9, 1, fmt)
    table, ctx = [7, 2, 8, 0, 5, 3], 384
    small = [7, 8, 3]
    cache.v_scale[small] *= 2.0 ** -octaves
    # keys: the first dimension tells small blocks (+) from large ones (-), queries look for one of the two
    one = 64 if fmt == torch.int8 else 64.0
    cache.k[:, :, :, 0] = -one
    cache.k[small, :, :, 0] = one
    cache.k_scale.fill_(2.0 ** -6)
    q = torch.randn(rows, 1, 64, generator=g)
    q[:, :, 0] = torch.where(torch.arange(rows)[:, None] % 3 < 2, 6000.0, -300.0)
    q = q.bfloat16().cuda()
    want = _reference(q, cache, table, ctx, 0.125, False)
    for copies in COPIES:
        _check(_attend(ops, q, cache, table, ctx, copies, False), *want)
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", ROWS)
def test_value_scales_at_the_ends_of_the_range(ops, fmt, rows):
    """Equal weights on values of 2^-95 and of 2^105 and on blocks of scale 0: the sum of the probabilities counts all of them."""
    g = torch.Generator().manual_seed(rows)
    cache = _filled(g, ops, 6, 2, fmt)
    cache.k_scale.mul_(2.0 ** -3)
    q = torch.randn(rows, 2, 64, generator=g).bfloat16().cuda()
    for exponents in ([-100, -100, 100, -100], [100, -100, -100, 100], [-100, -100, -100, -100], [0, -100, None, 3], [None] * 4):
        table = [4, 0, 5, 2]
        for b, e in zip(table, exponents):
            cache.v_scale[b] = 0.0 if e is None else 2.0 ** e
        for causal in (False, True):
            want, tol = _reference(q, cache, table, 250, 0.125, causal)
            for copies in COPIES:
                _check(_attend(ops, q, cache, table, 250, copies, causal), want, tol + 2.0 ** -120)  # below, bf16 runs out of places
    ops.check_device()


def test_a_large_value_far_behind(ops):
    """One CTA over more than 512 blocks, the largest scale in one of the last."""
    g = torch.Generator().manual_seed(12)
    cache = _filled(g, ops, 600, 1, torch.int8)
    cache.k_scale.mul_(2.0 ** -2)
    table = torch.randperm(600, generator=g).tolist()
    cache.v_scale[table[590]] *= 2.0 ** 30
    q = torch.randn(130, 1, 64, generator=g).bfloat16().cuda()
    for ctx in (590 * 64 + 100, 599 * 64):
        for causal in (False, True):
            _check(_attend(ops, q, cache, table, ctx, 160, causal), *_reference(q, cache, table[:-(-ctx // 64)], ctx, 0.125, causal))
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_scale_that_is_no_number(ops, fmt, rows, which):
    """NaN as a scale of a block in use: NaN for the rows that see one of its tokens, nothing for the others."""
    g = torch.Generator().manual_seed(rows)
    cache = _filled(g, ops, 9, 2, fmt)
    cache.k_scale.mul_(2.0 ** -2)
    table, ctx = [7, 2, 8, 0, 5, 3, 1, 6], min(500, 448 + (rows + 1) // 2)
    q = torch.randn(rows, 2, 64, generator=g).half().cuda()
    for causal in (True, False):
        want, tol = _reference(q, cache, table, ctx, 0.125, causal)
        for block in (7, 5):
            kept = getattr(cache, which + "_scale").clone()
            getattr(cache, which + "_scale")[table[block], 0] = float("nan")  # of one head
            first = max(0, 64 * block - (ctx - rows)) if causal else 0  # row that sees the block's first token
            for copies in COPIES:
                got = _attend(ops, q, cache, table, ctx, copies, causal)
                assert got[first:, 0].isnan().all()
                _check(got[:, 1], want[:, 1], tol[:, 1])
                _check(got[:first, 0], want[:first, 0], tol[:first, 0])
            getattr(cache, which + "_scale").copy_(kept)
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_negative_scale_is_reported(ops, fmt, rows, which):
    """Scales are at least 0: a block with a negative one is left out, as one that the cache does not have."""
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(rows)
    cache = _filled(g, ops, 9, 1, fmt)
    cache.k_scale.mul_(2.0 ** -2)
    q = torch.randn(rows, 1, 64, generator=g).half().cuda()
    want, tol = _reference(q, cache, [7, 8, 0], 172, 0.125, False)
    getattr(cache, which + "_scale")[2] *= -1
    if rows % 3 == 0:  # and the other one is NaN
        getattr(cache, "kv"[which == "k"] + "_scale")[2] = float("nan")
    for copies in COPIES:
        got = _attend(ops, q, cache, [7, 2, 8, 0], 236, copies, False)
        with pytest.raises(RtError) as e:
            ops.check_device()
        assert e.value.code == 1 and "1003" in str(e.value)
        _check(got, want, tol)
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", ROWS[1:])
def test_rows_that_see_nothing_hold_anything(ops, fmt, dtype, rows):
    """Query rows without a key give 0, be they NaN or infinite; the other rows do not notice."""
    g = torch.Generator().manual_seed(rows)
    cache = _filled(g, ops, 6, 2, fmt)
    cache.k_scale.mul_(2.0 ** -2)
    table, ctx = [4, 0, 5, 2], rows // 2
    q = torch.randn(rows, 2, 64, generator=g).to(dtype).cuda()
    want, tol = _reference(q, cache, table[:-(-ctx // 64)], ctx, 0.125, True)
    blind = rows - ctx
    q[:blind:2], q[1:blind:2] = float("nan"), float("inf")
    for copies in COPIES:
        got = _attend(ops, q, cache, table, ctx, copies, True)
        assert (got[:blind] == 0).all()
        _check(got[blind:], want[blind:], tol[blind:])
    ops.check_device()


@pytest.mark.parametrize("rows", ROWS)
def test_a_score_that_is_no_number(ops, rows):
    """An infinite query entry on keys of 0 there: the scores of these keys are NaN, whichever they are, and so is the row; the other
    scores are -inf."""
    g = torch.Generator().manual_seed(rows)
    cache = _filled(g, ops, 2, 1, torch.float8_e4m3fn)
    q = torch.randn(rows, 1, 64, generator=g).half().cuda()
    q[::2, :, 0] = float("inf")
    for keys in ([0], [13], [14], [15], [30, 31], [47], [63], [64 + 15], [79, 80]):
        cache.k[:, :, :, 0] = -2.0
        for key in keys:
            cache.k[key // 64, :, key % 64, 0] = 0.0
        for copies in COPIES:
            got = _attend(ops, q, cache, [0, 1], 81, copies, False)
            assert got[::2].isnan().all() and got[1::2].isfinite().all(), keys
    ops.check_device()
