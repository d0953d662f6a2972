"""Log probabilities of given tokens, entropy and best alternatives, and their gradient, against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


def _rows(rows, vocab, dtype, pitch=None, seed=0, size=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + vocab)
    z = torch.randn(rows, pitch or vocab, device="cuda", generator=g) * size
    t = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda", generator=g)
    return z.to(dtype)[:, :vocab], t


def _check_forward(got, z, t, top):
    """|z - max| is under 64 here: fp32 differences, exponentials of 2^-22 and sums of up to 100 terms a thread are together
    under 2^-16 for the logarithm of the sum, and 16 times that for the weighted sum."""
    x = z.double()
    lp = torch.log_softmax(x, 1)
    rows = torch.arange(z.shape[0], device="cuda")
    want = torch.where(t < 0, 0.0, lp[rows, t.clamp(min=0).long()])
    assert ((got.logp.double() - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * want.abs()).all()
    h = -(lp.exp() * torch.where(lp.isinf(), 0.0, lp)).sum(1)
    assert ((got.entropy.double() - h).abs() <= 2.0 ** -12).all()
    assert ((got.stats.double().sum(1) - torch.logsumexp(x, 1)).abs() <= 2.0 ** -16 + 2.0 ** -23 * x.abs().amax(1)).all()
    assert torch.equal(got.stats[:, 0], z.float().amax(1))
    if top:
        ids = torch.sort(z.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids.long(), ids)
        want = lp.gather(1, ids)
        same = got.top_logp.double() == want  # -inf
        assert (same | ((got.top_logp.double() - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * want.abs())).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pitch,top", [
    (1, 1, 1, 1), (3, 2, 2, 2), (5, 7, 9, 0), (2, 33, 33, 32), (9, 1000, 1001, 20), (4, 4096, 4096, 5), (1, 50358, 50358, 8),
    (19, 50358, 50368, 5), (150, 30011, 30011, 1), (400, 5003, 5003, 32), (3, 130001, 130001, 32),
])
def test_scores(ops, dtype, rows, vocab, pitch, top):
    z, t = _rows(rows, vocab, dtype, pitch)
    t[::3] = -1
    _check_forward(ops.token_logprobs(z, t, top_k=top), z, t, top)
    none = ops.token_logprobs(z)
    assert none.logp is None and none.top_ids is None
    _check_forward(none._replace(logp=torch.zeros(rows, device="cuda")), z, torch.full_like(t, -1), 0)
    ops.check_device()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [592, 593, 741, 889])
def test_more_rows_than_an_sm_holds(ops, dtype, rows):
    z, t = _rows(rows, 5003, dtype)
    _check_forward(ops.token_logprobs(z, t, top_k=7), z, t, 7)
    ops.check_device()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 200])
def test_equal_logits(ops, dtype, rows):
    """Constant rows, two values, and the best ones in the last places: ties go to the lower id."""
    vocab = 20000
    z = torch.zeros(rows, vocab, dtype=dtype, device="cuda")
    z[1::3, ::2] = 1.0
    z[2::3, -3:] = 5.0
    z[0, 5] = -0.0
    t = torch.arange(rows, dtype=torch.int32, device="cuda")
    _check_forward(ops.token_logprobs(z, t, top_k=32), z, t, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 160])
def test_masked_vocabulary(ops, dtype, rows):
    """-inf and the type's lowest value in masked places, rows with one token left, rows with none."""
    vocab = 9000
    z, t = _rows(rows, vocab, dtype)
    z = z.clone()
    z[0] = -float("inf")
    z[1, :] = -float("inf")
    z[1, 4321] = 2.0
    t[1] = 4321
    z[2, 100:] = torch.finfo(dtype).min
    t[2] = 3
    z[3, ::2] = -float("inf")
    t[3] = 2  # a masked token
    got = ops.token_logprobs(z, t, top_k=6)
    assert got.logp[0] == -float("inf") and got.entropy[0] == 0
    assert got.top_ids[0].tolist() == [0, 1, 2, 3, 4, 5] and (got.top_logp[0] == -float("inf")).all()
    assert got.logp[1] == 0 and got.entropy[1] == 0 and got.top_ids[1].tolist() == [4321, 0, 1, 2, 3, 4]
    assert got.logp[3] == -float("inf")
    x = z.double()
    lp = torch.log_softmax(x[1:], 1)
    h = -(lp.exp() * torch.where(lp.exp() == 0, 0.0, lp)).sum(1)
    assert ((got.entropy[1:].double() - h).abs() <= 2.0 ** -12).all()
    ids = torch.sort(z.float(), dim=1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(got.top_ids.long(), ids)
    rest = torch.arange(4, rows, device="cuda")
    want = lp[rest - 1, t[rest].long()]
    assert ((got.logp[rest].double() - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * want.abs()).all()
    # the gradient: nothing where p is nothing
    d = ops.token_logprobs_backward(z, t, got.stats, got.entropy, grad_logp=torch.ones(rows, device="cuda"),
                                    grad_entropy=torch.ones(rows, device="cuda"))
    assert (d[0] == 0).all() and (d[1] == 0).all() and not d.isnan().any() and (d[3, 4::2] == 0).all() and d[3, 2] == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 160])
def test_rows_at_the_ends_of_the_type(ops, dtype, rows):
    """Rows of nothing but the lowest value, with -inf among them, with the largest value, with both; and a large common offset."""
    vocab, low, big = 6000, torch.finfo(dtype).min, torch.finfo(dtype).max
    z, t = _rows(rows, vocab, dtype)
    z = z.clone()
    z[0] = low
    z[1] = low
    z[1, 1::2] = -float("inf")
    t[1] = 2
    z[2] = 0
    z[2, 17] = big
    t[2] = 17
    z[3] = low
    z[3, 100] = low / 2
    z[3, 4000] = big
    t[3] = 4000
    z[4] = z[4] + (1000 if dtype != torch.float32 else 100000)
    got = ops.token_logprobs(z, t, top_k=3)
    lp = torch.log_softmax(z.double(), 1)
    want = lp[torch.arange(rows, device="cuda"), t.long()]
    assert ((got.logp.double() - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * want.abs()).all()
    h = -(lp.exp() * torch.where(lp.exp() == 0, 0.0, lp)).sum(1)
    assert ((got.entropy.double() - h).abs() <= 2.0 ** -12).all()
    assert torch.equal(got.top_ids.long(), torch.sort(z.float(), dim=1, descending=True, stable=True).indices[:, :3])
    assert got.top_ids[1].tolist() == [0, 2, 4] and got.logp[2] == 0
    d = ops.token_logprobs_backward(z, t, got.stats, got.entropy, grad_logp=torch.ones(rows, device="cuda"))
    assert not d.isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_nan_and_infinity(ops, dtype):
    z, t = _rows(6, 5000, dtype)
    z = z.clone()
    z[0, 17] = float("nan")
    z[1] = float("nan")
    z[2, 4999] = float("inf")
    z[3] = -float("inf")
    z[3, 7] = float("nan")
    got = ops.token_logprobs(z, t, top_k=3)
    for r in range(4):
        assert got.logp[r].isnan() and got.entropy[r].isnan() and got.top_logp[r].isnan().all()
    assert (got.top_ids[1] == -1).all() and got.top_ids[2, 0] == 4999
    want = torch.log_softmax(z[4:].double(), 1)[[0, 1], t[4:].long()]
    assert ((got.logp[4:].double() - want).abs() <= 2.0 ** -16 + 2.0 ** -22 * want.abs()).all()


def _grad(z, t, ids, gl, gh, gt):
    """The formula in 64 bits, and what its rounding is measured by."""
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    h = -(p * lp).sum(1, keepdim=True)
    g = torch.where(t < 0, 0.0, gl)
    pull = g + (gt.sum(1) if gt is not None else 0)
    d = -p * (pull[:, None] + gh[:, None] * (lp + h))
    rows = torch.arange(z.shape[0], device="cuda")
    d[rows, t.clamp(min=0).long()] += g
    size = p * (pull.abs()[:, None] + gh.abs()[:, None] * (lp.abs() + h)) * (1 + lp.abs())
    size[rows, t.clamp(min=0).long()] += g.abs()
    if gt is not None:
        for j in range(gt.shape[1]):
            d[rows, ids[:, j].long()] += gt[:, j]
            size[rows, ids[:, j].long()] += gt[:, j].abs()
    return d, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pitch,top", [(1, 1, 1, 1), (3, 7, 9, 2), (2, 1000, 1000, 0), (5, 8192, 8192, 8), (7, 30011, 30011, 4),
                                                  (6, 50358, 50368, 32)])
def test_gradient(ops, dtype, rows, vocab, pitch, top):
    z, t = _rows(rows, vocab, dtype, pitch)
    t[::3] = -1
    g = torch.Generator(device="cuda").manual_seed(1)
    gl, gh = (torch.randn(rows, device="cuda", generator=g) for _ in range(2))
    gt = torch.randn(rows, top, device="cuda", generator=g) if top else None
    got = ops.token_logprobs(z, t, top_k=top)
    ids = got.top_ids
    if top > 1:
        ids = ids.clone()
        ids[0, 1] = ids[0, 0]       # the same token twice
        ids[-1, 0] = t[-1].clamp(min=0)  # the given token
    want, size = _grad(z.double(), t, ids, gl.double(), gh.double(), None if gt is None else gt.double())
    # half a step of the output, halves below 2^-14 in steps of 2^-24; fp32: 2^-20 of the terms, (1 + |log p|) for the exponential
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20 * size + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
    args = dict(grad_logp=gl, grad_entropy=gh, top_ids=ids, grad_top=gt)
    d = ops.token_logprobs_backward(z, t, got.stats, got.entropy, **args)
    off = (d.double() - want).abs()
    assert (off <= tol).all(), (off / tol).max().item()
    # into a buffer whose rows begin elsewhere, and in place
    other = torch.full((rows, vocab + 3), 7.0, dtype=dtype, device="cuda")
    assert torch.equal(ops.token_logprobs_backward(z, t, got.stats, got.entropy, out=other[:, 1:1 + vocab], **args), d)
    assert (other[:, 0] == 7.0).all() and (other[:, 1 + vocab:] == 7.0).all()
    same = z.clone(memory_format=torch.preserve_format) if pitch == vocab else z
    assert torch.equal(ops.token_logprobs_backward(same, t, got.stats, got.entropy, out=same, **args), d)
    ops.check_device()


def test_gradient_against_differences(ops):
    rows, vocab, eps = 2, 11, 1e-4
    z, t = _rows(rows, vocab, torch.float32, size=1.0)
    gl, gh, gt = torch.tensor([0.3, -1.0], device="cuda"), torch.tensor([0.7, 0.2], device="cuda"), torch.tensor([[1.0, -0.5], [0.25, 2.0]], device="cuda")
    got = ops.token_logprobs(z, t, top_k=2)
    d = ops.token_logprobs_backward(z, t, got.stats, got.entropy, gl, gh, got.top_ids, gt)

    def value(x):
        lp = torch.log_softmax(x, 1)
        r = torch.arange(rows, device="cuda")
        return ((gl * lp[r, t.long()]).sum() - (gh * (lp.exp() * lp).sum(1)).sum() + (gt * lp.gather(1, got.top_ids.long())).sum()).item()

    for r in range(rows):
        for v in range(vocab):
            up, down = z.double(), z.double()
            up[r, v] += eps
            down[r, v] -= eps
            # differences of 64-bit values: error of eps^2; the kernel's fp32: 2^-20 of terms of at most 4
            assert abs((value(up) - value(down)) / (2 * eps) - d[r, v].item()) < 1e-5


def test_parts_of_the_gradient(ops):
    z, t = _rows(3, 700, torch.float32)
    got = ops.token_logprobs(z, t)
    gl = torch.ones(3, device="cuda")
    only = ops.token_logprobs_backward(z, t, got.stats, grad_logp=gl)
    zero = torch.zeros(3, device="cuda")
    assert torch.equal(only, ops.token_logprobs_backward(z, t, got.stats, got.entropy, grad_logp=gl, grad_entropy=zero))
    assert (ops.token_logprobs_backward(z, None, got.stats) == 0).all()


def test_bad_tokens_are_reported(ops):
    from raptor_t_b200.capi import RtError
    z, t = _rows(4, 100, torch.float16)
    t[2] = 100
    got = ops.token_logprobs(z, t)
    with pytest.raises(RtError) as e:
        ops.check_device()
    assert e.value.code == 1 and "1004" in str(e.value)
    assert got.logp[2].isnan() and not got.logp[[0, 1, 3]].isnan().any()
    ids = torch.tensor([[3, 100]] * 4, dtype=torch.int32, device="cuda")
    ops.token_logprobs_backward(z, None, got.stats, top_ids=ids, grad_top=torch.ones(4, 2, device="cuda"))
    with pytest.raises(RtError):
        ops.check_device()
    ops.check_device()


def test_two_graphs_and_streams(ops):
    z, t = _rows(5, 20011, torch.bfloat16)
    want = ops.token_logprobs(z, t, top_k=5)
    gl = torch.ones(5, device="cuda")
    d = ops.token_logprobs_backward(z, t, want.stats, grad_logp=gl)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = ops.token_logprobs(z, t, top_k=5)
            b = ops.token_logprobs_backward(z, t, r.stats, grad_logp=gl)
        graphs.append((graph, r, b))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, r, b in graphs:
        assert all(torch.equal(x, y) for x, y in zip(r, want)) and torch.equal(b, d)


def test_rows_far_apart(ops):
    """Row offsets past 32 bits, read and written."""
    vocab, pitch = 1000, 2300000001
    z = torch.as_strided(torch.empty(2 * pitch + vocab, dtype=torch.float16, device="cuda"), (3, vocab), (pitch, 1))
    x, t = _rows(3, vocab, torch.float16)
    z.copy_(x)
    got = ops.token_logprobs(z, t, top_k=4)
    _check_forward(got, z, t, 4)
    g = torch.ones(3, device="cuda")
    want = ops.token_logprobs_backward(x, t, got.stats, grad_logp=g)
    assert torch.equal(ops.token_logprobs_backward(z, t, got.stats, grad_logp=g, out=z), want)
    assert torch.equal(z, want)
    ops.check_device()
