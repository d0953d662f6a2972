"""The 8-bit key/value cache: every code and scale as defined, what is written is what is read, what holds no token stays."""
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

FORMATS = [torch.float8_e4m3fn, torch.int8]
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _first(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _tables(g, start, counts, spare=1):
    """A table of shuffled blocks, wide enough for every sequence, and the number of blocks."""
    need = [-(-(a + n) // 64) for a, n in zip(start, counts)]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    width = max(need) + 1
    at, rows = 0, []
    for n in need:
        rows.append(order[at:at + n] + [-7] * (width - n))  # behind the last token: not read
        at += n
    return rows, total


def _filled(g, ops, blocks, heads, fmt):
    """A cache with codes and scales in every place."""
    if fmt == torch.int8:
        k, v = (torch.randint(-127, 128, (blocks, heads, 64, 64), generator=g).to(fmt) for _ in range(2))
        ks, vs = (torch.ldexp(torch.randint(128, 256, (blocks, heads), generator=g).float(), torch.tensor(-14)) for _ in range(2))
    else:
        k, v = ((torch.randn(blocks, heads, 64, 64, generator=g) * 60).clamp(-448, 448).to(fmt) for _ in range(2))
        ks, vs = (torch.ldexp(torch.ones(blocks, heads), torch.randint(-9, -5, (blocks, heads), generator=g)) for _ in range(2))
    return ops.KvCache(*(t.cuda().contiguous() for t in (k, v, ks, vs)))


def _expect(cache, k, v, rows, start, first):
    out = []
    for code, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        c = {"dtype": code.dtype, "codes": code.cpu().double()}
        s = scale.cpu().double()
        ref.write(c, s, x.cpu(), rows, start, first)
        out += [c["codes"], s]
    return out


def _check(cache, want):
    for got, w, name in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), want, ("k", "k_scale", "v", "v_scale")):
        g = got.cpu().double()
        assert torch.equal(g, w), (name, (g != w).sum().item(), (g - w).abs().max().item())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,start,counts", [
    (1, [0], [1]),                                   # the first token of a sequence
    (3, [63, 64, 65, 0], [1, 1, 1, 1]),              # the last and the first place of a block
    (2, [5, 130, 0, 64], [59, 66, 0, 128]),          # a block filled up, a sequence without tokens, whole blocks
    (12, [0, 17, 200], [333, 64, 1]),
    (4, [1000, 7], [1, 700]),
])
def test_write(ops, fmt, dtype, heads, start, counts):
    g = torch.Generator().manual_seed(len(counts) + heads)
    rows, blocks = _tables(g, start, counts)
    cache = _filled(g, ops, blocks, heads, fmt)
    T, first = sum(counts), _first(counts)
    # magnitudes over many octaves: blocks whose scale grows and blocks whose scale stays
    size = torch.exp2(torch.randint(-6, 7, (T, heads, 1), generator=g).float())
    k, v = ((torch.randn(T, heads, 64, generator=g) * size).to(dtype).cuda() for _ in range(2))
    k[0, 0, :4] = torch.tensor([0.0, -0.0, 1.0, 0.5]).to(dtype)  # 0.5 of a maximum of 1 is on the border between two int8 codes
    want = _expect(cache, k, v, rows, start, first)
    ops.kv_cache_write(cache, k, v, _i32(rows), _i32(start), _i32(first), max_tokens=max(counts))
    _check(cache, want)
    # the same tokens once more: nothing changes
    ops.kv_cache_write(cache, k, v, _i32(rows), _i32(start), _i32(first))
    _check(cache, want)
    # and back
    for out_type in DTYPES:
        got = ops.kv_cache_read(cache, _i32(rows), _i32(start), _i32(first), T, out_type, max_tokens=max(counts))
        for c, s, o in ((want[0], want[1], got[0]), (want[2], want[3], got[1])):
            for i in range(len(counts)):
                for j in range(counts[i]):
                    p = start[i] + j
                    b = rows[i][p // 64]
                    x = (c[b, :, p % 64] * s[b][:, None]).float()  # at most 15 significant bits: exact
                    assert torch.equal(o[first[i] + j].cpu(), x.to(out_type))
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
def test_borders_between_codes(ops, fmt):
    """Values on and next to every border between two codes, for scales with all their bits."""
    g = torch.Generator().manual_seed(5)
    for most in (1.0, 127.0, 3.5, 448.0, 0.013671875, 60000.0):
        x = torch.zeros(64, 1, 64)
        s = ref.needed_scale(torch.tensor(most).half().double().item(), fmt)
        pick = torch.randint(0, 127, (64 * 64,), generator=g).double()
        border = (pick + 0.5) * s * torch.where(torch.rand(64 * 64, generator=g) < 0.5, -1.0, 1.0)
        x.view(-1)[:] = border.clamp(-most, most).float()
        x[0, 0, 0] = most
        x = x.half()
        cache = ops.KvCache.empty(1, 1, fmt)
        cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0), cache.k.view(torch.int8).zero_(), cache.v.view(torch.int8).zero_()
        want = _expect(cache, x, x, [[0]], [0], [0, 64])
        ops.kv_cache_write(cache, x.cuda(), x.cuda(), _i32([[0]]), _i32([0]), _i32([0, 64]))
        _check(cache, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers(ops, fmt, dtype):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(100, 2, 64, generator=g).to(dtype)
    x[3, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    x[70, 1] = float("nan")
    x[64:, 0] = 0  # nothing but zeros
    y = torch.full((100, 2, 64), float("inf")).to(dtype)  # no finite value
    cache = _filled(g, ops, 3, 2, fmt)
    want = _expect(cache, x, y, [[2, 0]], [0], [0, 100])
    ops.kv_cache_write(cache, x.cuda(), y.cuda(), _i32([[2, 0]]), _i32([0]), _i32([0, 100]))
    _check(cache, want)
    assert want[1][0, 0] == 2.0 ** -100 and cache.k.float().isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(ops, dtype):
    """Columns of a projection, and the head-major buffers of the encoder's projection."""
    g = torch.Generator().manual_seed(11)
    lens, heads = [128, 64, 192], 3
    T, first, rows = sum(lens), _first(lens), [[5, 0, -1], [1, -1, -1], [4, 2, 3]]
    qkv = torch.randn(T, 3 * heads * 64, generator=g).to(dtype).cuda()
    k, v = (qkv[:, i * heads * 64:(i + 1) * heads * 64].unflatten(1, (heads, 64)) for i in (1, 2))
    a, b = (ops.KvCache.empty(6, heads, torch.int8) for _ in range(2))
    ops.kv_cache_write(a, k, v, _i32(rows), _i32([0, 0, 0]), _i32(first))
    want = _expect(ops.KvCache(a.k, a.v, a.k_scale, a.v_scale), k, v, rows, [0, 0, 0], first)
    _check(a, want)
    zero = torch.zeros(3 * heads * 64, dtype=dtype, device="cuda")
    prefix = _i32([0, 2, 3, 6])
    _, hk, hv = ops.qkv_bias_transpose(qkv, zero, prefix, heads, 1.0)
    ops.kv_cache_write(b, hk, hv, _i32(rows), _i32([0, 0, 0]), _i32(first), head_major=True)
    _check(b, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_bad_indexes_are_skipped_and_reported(ops, fmt):
    """Entries outside the cache, tables that are too narrow, lengths outside the batch: only what is in range is written."""
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(13)
    x = torch.randn(192, 1, 64, generator=g).half().cuda()
    for table, start, first, good in (
        ([[0, 3, 1]], [0], [0, 192], [0, 1]),           # block 3 of 3
        ([[0, -1, 1]], [0], [0, 192], [0, 1]),
        ([[0, 1]], [0], [0, 192], [0, 1]),              # no third entry
        ([[0, 1, 2]], [-1], [0, 192], []),
        ([[0, 1, 2]], [0], [0, 193], []),               # a row that the batch does not have
        ([[0, 1, 2]], [2147483600], [0, 100], []),
    ):
        cache = _filled(g, ops, 3, 1, fmt)
        before = [t.clone() for t in (cache.k.view(torch.int8), cache.k_scale)]
        ops.kv_cache_write(cache, x, x, _i32(table), _i32(start), _i32(first))
        with pytest.raises(RtError) as e:
            ops.check_device()
        assert e.value.code == 1 and "1001" in str(e.value)
        for b in range(3):
            same = torch.equal(before[0][b], cache.k.view(torch.int8)[b]) and torch.equal(before[1][b], cache.k_scale[b])
            assert same == (b not in good), (table, b)
        out = [torch.full((192, 1, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        ops.kv_cache_read(cache, _i32(table), _i32(start), _i32(first), 192, torch.float16, out=out)
        with pytest.raises(RtError):
            ops.check_device()
    # more tokens than the caller said: nothing of that sequence
    cache = _filled(g, ops, 3, 1, fmt)
    before = cache.k.view(torch.int8).clone()
    ops.kv_cache_write(cache, x, x, _i32([[0, 1, 2]]), _i32([0]), _i32([0, 192]), max_tokens=191)
    with pytest.raises(RtError):
        ops.check_device()
    assert torch.equal(before, cache.k.view(torch.int8))
    ops.check_device()


def test_large_cache(ops):
    """Blocks behind the first 4 GB of codes."""
    blocks, heads = 90000, 16  # 5.9 GB each of keys and values
    cache = ops.KvCache.empty(blocks, heads, torch.int8)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(130, heads, 64, device="cuda", generator=g).half()
    rows = [[blocks - 1, 70000, 65536]]
    args = _i32(rows), _i32([0]), _i32([0, 130])
    ops.kv_cache_write(cache, x, x, *args)
    k, v = ops.kv_cache_read(cache, *args, 130, torch.float16)
    assert torch.equal(k, v)
    step = cache.k_scale[rows[0]].float()  # [3 blocks, heads]
    off = (k.float() - x.float()).abs().amax(2)
    for t in range(130):
        # half a code of the scale, and the value's own rounding to 16 bits
        assert (off[t] <= step[t // 64] * 0.5 + x[t].float().abs().amax(1) * 2.0 ** -11).all()
    q = torch.randn(1, heads, 64, device="cuda", generator=g).half()
    o = ops.cached_attention(q, cache, args[0], _i32([130]), _i32([0, 1]), scale=0.125)
    z = torch.einsum("hd,khd->hk", q[0].double(), k.double()) * 0.125
    want = torch.einsum("hk,khd->hd", torch.softmax(z, 1), v.double())
    # read-back values are rounded to 16 bits (2^-11), probabilities too, the output once more
    assert (o[0].double() - want).abs().max() <= 4 * 2.0 ** -11 * v.abs().max()
    ops.check_device()
