"""Attention over the 8-bit cache against the definition in 64 bits."""
import pytest
import torch

import kv_reference as ref
from test_kv_cache_gpu import FORMATS, DTYPES, _filled, _first, _i32, _tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _tolerance(want, vmax, keys, dtype):
    """Rounding of the output (half a step) + rounding of the probabilities to halves (2^-11 relative, 2^-25 absolute for each
    of the keys, against a sum of at least 1) + fp32 scores and exponentials (together under 2^-14 for the sizes here)."""
    return torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -14 + keys * 2.0 ** -25) * vmax + 1e-7


def _case(ops, fmt, dtype, heads, kv_heads, counts, context, causal, spare_rows=0, seed=0, stride=None, **more):
    g = torch.Generator().manual_seed(seed + sum(context) + heads)
    rows, blocks = _tables(g, [0] * len(context), context)
    cache = _filled(g, ops, max(1, blocks), kv_heads, fmt)
    cache.k_scale.mul_(2.0 ** -2)  # keys of about one
    T = sum(counts) + spare_rows
    first = _first(counts)
    width = stride or heads * 64
    store = torch.randn(T, width, generator=g).to(dtype).cuda()
    q = store[:, :heads * 64].unflatten(1, (heads, 64))
    out = torch.full((T, heads, 64), 7.0, dtype=dtype, device="cuda")
    got = ops.cached_attention(q, cache, _i32(rows), _i32(context), _i32(first), scale=0.125, causal=causal, out=out, **more)
    ops.check_device()
    k, v = ((c.cpu().double() * s.cpu().double()[:, :, None, None]) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, vmax = ref.attention(q.cpu().double(), k, v, rows, context, first, heads // kv_heads, 0.125, causal)
    used = slice(0, sum(counts))
    off = (got.cpu().double() - want).abs()[used]
    tol = _tolerance(want, vmax, max(context), dtype)[used]
    assert (off <= tol).all(), ((off / tol).max().item(), off.max().item())
    assert (got[sum(counts):] == 7.0).all()  # rows behind the last sequence
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (16, 4), (8, 1)])
def test_single_tokens(ops, fmt, dtype, causal, heads, kv_heads):
    _case(ops, fmt, dtype, heads, kv_heads, [1] * 7, [1, 63, 64, 65, 700, 0, 4097], causal, spare_rows=3)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 2)])
def test_ragged_questions(ops, fmt, dtype, causal, heads, kv_heads):
    _case(ops, fmt, dtype, heads, kv_heads, [5, 0, 64, 17, 1, 33], [5, 9, 64, 1000, 1, 130], causal, spare_rows=1)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("counts,context", [([128], [128]), ([129, 300], [129, 1500]), ([256, 1, 640], [2048, 300, 640]),
                                            ([127, 500], [4100, 499])])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1)])
def test_many_rows(ops, fmt, causal, counts, context, heads, kv_heads):
    for dtype in DTYPES:
        _case(ops, fmt, dtype, heads, kv_heads, counts, context, causal, spare_rows=2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("counts,context", [([32] + [3] * 40, [2000] + [64] * 40), ([64] * 33, [1100] * 33), ([256, 256, 65, 33, 32, 31, 1, 97], [4000] * 8),
                                            ([64] * 3, [64] * 3)])
def test_copies_of_rows_and_clusters(ops, fmt, causal, counts, context):
    """Tiles of 32, 64, 128 and 256 rows, with a CTA or a cluster for each; more clusters than fit at once."""
    _case(ops, fmt, torch.float16, 4, 4, counts, context, causal)


@pytest.mark.parametrize("causal", [False, True])
def test_rows_that_see_nothing(ops, causal):
    """More query rows than context: with the causal rule the first ones see no key."""
    got = _case(ops, torch.int8, torch.float16, 3, 3, [40, 200, 3], [10, 70, 0], causal)
    if causal:
        assert (got[:30] == 0).all() and (got[40:170] == 0).all()
    assert (got[240:] == 0).all()


def test_queries_with_a_stride(ops):
    _case(ops, torch.float8_e4m3fn, torch.bfloat16, 4, 2, [1, 20, 150], [100, 20, 400], True, stride=3 * 4 * 64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,most", [(2, 2, 1), (6, 2, 1), (8, 1, 4), (2, 1, 20)])
def test_many_sequences(ops, fmt, causal, heads, kv_heads, most):
    """Calls whose blocks are one list that all warps share: more than 128 sequences, some without rows, some without keys, lengths
    from one token to some that several warps work on."""
    import random
    rng = random.Random(heads + most)
    counts = [rng.choice([0, 1, 1, rng.randint(1, most)]) for _ in range(300)]
    context = [rng.choice([0, 1, 64, 65, rng.randint(1, 700), rng.randint(1, 2000)]) for _ in range(300)]
    counts[0], context[0], counts[-1], context[-1] = 0, 0, most, 3000
    for dtype in DTYPES:
        _case(ops, fmt, dtype, heads, kv_heads, counts, context, causal, spare_rows=2, max_q=most)


@pytest.mark.parametrize("counts,context", [([1] * 8, [6000, 1, 4096, 4097, 0, 63, 5000, 3333]), ([1], [60000]), ([3, 16], [17000, 16001])])
def test_long_contexts(ops, counts, context):
    _case(ops, torch.int8, torch.bfloat16, 12, 12, counts, context, True)


@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("max_context", [1, 64, 100000])
def test_max_context_only_guides(ops, rows, max_context):
    _case(ops, torch.int8, torch.bfloat16, 2, 2, [rows], [3000], False, max_context=max_context, max_q=rows)


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("fmt", FORMATS)
def test_places_without_tokens_do_not_count(ops, fmt, rows):
    """Every byte value and NaN scales where no token is; queries of many magnitudes; bf16 numbers outside a half's range."""
    g = torch.Generator().manual_seed(2)
    cache = _filled(g, ops, 8, 2, fmt)
    table = [[3, 6, 1, 0]]
    ctx = 150
    q = (torch.randn(rows, 2, 64, generator=g) * torch.exp2(torch.randint(-40, 30, (rows, 2, 1), generator=g).float())).bfloat16().cuda()
    args = _i32(table), _i32([ctx]), _i32([0, rows])
    a = ops.cached_attention(q, cache, *args, scale=2.0 ** -10)
    for garbage in (0x7f, 0xff, 0x80, 0x01):
        for c in (cache.k, cache.v):
            raw = c.view(torch.uint8)
            raw[1, :, ctx - 128:] = garbage
            for b in (0, 2, 4, 5, 7):
                raw[b] = garbage
        for s in (cache.k_scale, cache.v_scale):
            s[[0, 2, 4, 5, 7]] = float("nan")
        assert torch.equal(a, ops.cached_attention(q, cache, *args, scale=2.0 ** -10))
    k, v = ((c.cpu().double() * s.cpu().double()[:, :, None, None]) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    want, vmax = ref.attention(q.cpu().double(), k, v, table, [ctx], [0, rows], 1, 2.0 ** -10, False)
    # scores of up to 2^30 * 64 * 4 * 2^-10 in fp32: a softmax of one or a few keys; compare where the largest score leads by far
    z = torch.einsum("thd,khd->thk", q.cpu().double(), k[[3, 6, 1]].transpose(1, 2).flatten(0, 1)[:ctx]) * 2.0 ** -10
    top = z.topk(2, -1).values
    clear = (z.abs().amax(-1) < 64) | ((top[..., 0] - top[..., 1]) > 2.0 ** -16 * z.abs().amax(-1) + 20)
    tol = _tolerance(want, vmax, ctx, torch.bfloat16) + 2.0 ** -13 * vmax
    assert ((a.cpu().double() - want).abs() <= tol)[clear].all() and clear.float().mean() > 0.5
    ops.check_device()


def test_bad_indexes_are_reported(ops):
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(4)
    cache = _filled(g, ops, 4, 1, torch.int8)
    for rows in (1, 150):
        q = torch.randn(rows, 1, 64, generator=g).half().cuda()
        for table, ctx, first in (([[0, 4]], 100, rows), ([[0, -1]], 100, rows), ([[0, 1]], 129, rows), ([[0, 1]], -1, rows),
                                  ([[0, 1]], 100, rows + 1)):
            ops.cached_attention(q, cache, _i32(table), _i32([ctx]), _i32([0, first]))
            with pytest.raises(RtError) as e:
                ops.check_device()
            assert e.value.code == 1 and "1003" in str(e.value)
    ops.check_device()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 12, 40, 150, 300])
def test_a_bad_entry_leaves_out_its_keys(ops, fmt, rows):
    """Whatever the block holds that is read in its place."""
    from raptor_t_b200.capi import RtError
    g = torch.Generator().manual_seed(5)
    cache = _filled(g, ops, 6, 2, fmt)
    cache.k_scale.mul_(2.0 ** -2)
    k, v = ((c.cpu().double() * s.cpu().double()[:, :, None, None]) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    for c in (cache.k, cache.v):
        c.view(torch.uint8)[0] = 0x7f
    for s in (cache.k_scale, cache.v_scale):
        s[0] = float("nan")
    q = torch.randn(rows, 2, 64, generator=g).half().cuda()
    got = ops.cached_attention(q, cache, _i32([[4, -1, 2, 6, 1]]), _i32([300]), _i32([0, rows]), scale=0.125)
    with pytest.raises(RtError):
        ops.check_device()
    # keys of the entries 4, 2 and the 44 tokens of 1
    want, vmax = ref.attention(q.cpu().double(), k, v, [[4, 2, 1]], [172], [0, rows], 1, 0.125, False)
    assert ((got.cpu().double() - want).abs() <= _tolerance(want, vmax, 172, torch.float16)).all()


def test_two_streams_and_a_captured_graph(ops):
    """Calls on two streams at once, and replays with contexts that have grown, give what one call after the other gives."""
    g = torch.Generator().manual_seed(6)
    cache = _filled(g, ops, 70, 2, torch.int8)
    table = _i32([list(range(64))])
    for rows in (1, 300):
        q = torch.randn(rows, 2, 64, generator=g).half().cuda()
        ctx, first = _i32([1000]), _i32([0, rows])
        run = lambda out=None: ops.cached_attention(q, cache, table, ctx, first, scale=0.125, out=out)  # noqa: E731
        want = run()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for i in range(8):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        graph = torch.cuda.CUDAGraph()
        out = torch.empty_like(want)
        with torch.cuda.graph(graph):
            run(out)
        for n in (1000, 1, 4096, 777):
            ctx.fill_(n)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, run())
    ops.check_device()


def test_a_run_together(ops):
    """Documents are projected as the encoder does it and kept; tokens join them one by one, attend, and are scored."""
    from raptor_t_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(8)
    H, heads, lens, vocab = 128, 2, [128, 192], 500
    new = lambda *s: (torch.randn(*s, device="cuda", generator=g) / s[-1] ** 0.5).half()  # noqa: E731
    docs, w, b = torch.randn(sum(lens), H, device="cuda", generator=g).half(), new(3 * H, H), new(3 * H)
    emb = torch.zeros(512, H, dtype=torch.float16, device="cuda")
    emb[:vocab] = new(vocab, H)
    _, k, v = ops.gemm_qkv(docs, w, b, ops.block_seq_table(lens), heads)
    cache = ops.KvCache.empty(9, heads, torch.float8_e4m3fn)
    table = _i32([[8, 1, 3, -1], [0, 2, 7, 5]])
    ops.kv_cache_write(cache, k, v, table, _i32([0, 0]), _i32([0, 128, 320]), head_major=True)
    keys = [torch.nn.functional.linear(docs.double(), w.double(), b.double()).split(H, 1)]
    have, x = list(lens), torch.randn(2, H, device="cuda", generator=g).half()
    tail = [[], []]
    for step in range(3):
        qkv = ops.gemm(x, w, b, capi.RT_EPI_BIAS)
        q, kk, vv = (t.unflatten(1, (heads, 64)) for t in qkv.split(H, 1))
        ops.kv_cache_write(cache, kk, vv, table, _i32(have), _i32([0, 1, 2]), max_tokens=1)
        have = [n + 1 for n in have]
        o = ops.cached_attention(q, cache, table, _i32(have), _i32([0, 1, 2]), max_q=1, scale=0.125, causal=True)
        logits = ops.gemm(o.flatten(1), emb)[:, :vocab]
        got = ops.token_logprobs(logits, _i32([step, 7]), top_k=4)
        for s in range(2):
            tail[s].append(torch.stack([kk[s].double(), vv[s].double()]))
            lo = sum(lens[:s])
            dk, dv = (keys[0][i][lo:lo + lens[s]].unflatten(1, (heads, 64)) for i in (1, 2))
            more = torch.stack(tail[s])
            ak, av = torch.cat([dk, more[:, 0]]), torch.cat([dv, more[:, 1]])
            z = torch.einsum("hd,khd->hk", q[s].double(), ak) * 0.125
            want = torch.einsum("hk,khd->hd", torch.softmax(z, 1), av)
            # e4m3 is off by at most 2^-4 of a value: keys change a score by at most 2^-4 sum |q k| / 8 (under 0.25 here, a factor of
            # 1.28 on a probability), values an output by 2^-4 max |v|
            assert (o[s].double() - want).abs().max() <= (0.28 + 2.0 ** -4 + 2.0 ** -9) * av.abs().max()
        lp = torch.log_softmax(logits.double(), 1)
        assert (got.logp.double() - lp[[0, 1], [step, 7]]).abs().max() < 2.0 ** -16
        assert torch.equal(got.top_ids.long(), torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :4])
        x = emb[got.top_ids[:, 0].long()] * 4
    ops.check_device()


@pytest.mark.parametrize("seed", range(10))
def test_random_calls(ops, seed):
    """Heads in groups of any size, ragged rows and contexts on both sides of every rule that chooses a kernel or a split."""
    import random
    rng = random.Random(seed)
    for _ in range(6):
        group, kv_heads, n = rng.choice([1, 1, 2, 3, 5, 7, 13]), rng.choice([1, 2, 3]), rng.choice([1, 1, 2, 3, 9, 40])
        most = max(1, int(2 ** rng.uniform(0, 10 if n < 9 else 6)) // group)
        counts = [rng.choice([most, rng.randint(0, most), rng.randint(1, most)]) for _ in range(n)]
        context = [rng.choice([0, 1, rng.randint(1, 64), int(2 ** rng.uniform(5, 11))]) if rng.random() < 0.9 else c for c in counts]
        if sum(counts) == 0:
            continue
        _case(ops, rng.choice(FORMATS), rng.choice(DTYPES), group * kv_heads, kv_heads, counts, context, rng.random() < 0.5,
              spare_rows=rng.randint(0, 3), seed=seed)
