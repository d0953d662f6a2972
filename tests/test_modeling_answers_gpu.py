"""The model layer on the cache, the attention over it and the token scores: a sub-layer over stored documents, the masked-token head."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H, HEADS = 128, 2


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import modeling_bert, ops
    return modeling_bert, ops


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _weights(g, *shape):
    return (torch.randn(*shape, device="cuda", generator=g) / math.sqrt(shape[0])).half()


def test_documents_are_remembered_and_continued(mods):
    modeling, ops = mods
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv_w, qkv_b, out_w, out_b = _weights(g, H, 3 * H), _weights(g, 3 * H) * 4, _weights(g, H, H), _weights(g, H)
    ln_w, ln_b = (1 + 0.1 * torch.randn(H, device="cuda", generator=g)).half(), _weights(g, H)
    layer = modeling.BertCachedAttention(qkv_w, qkv_b, out_w, out_b, ln_w, ln_b, HEADS)
    lens, more = [130, 64], [3, 5]
    docs, new = (torch.randn(sum(n), H, device="cuda", generator=g).half() for n in (lens, more))
    cache = ops.KvCache.empty(6, HEADS, torch.int8)
    table = _i32([[4, 1, 0], [2, 5, -1]])
    layer.remember(docs, cache, table, _i32([0, 0]), _i32([0, 130, 194]))
    got = layer(new, cache, table, _i32(lens), _i32([133, 69]), _i32([0, 3, 8]), max_tokens=5)
    ops.check_device()
    f = lambda x: torch.nn.functional.linear(x.double(), qkv_w.double().t(), qkv_b.double())  # noqa: E731
    ctx = torch.zeros(8, H, dtype=torch.float64, device="cuda")
    kmax = vmax = 0.0
    for s in range(2):
        a, b = (sum(lens[:s]), sum(more[:s]))
        kv = f(torch.cat([docs[a:a + lens[s]], new[b:b + more[s]]]))
        q = f(new[b:b + more[s]])[:, :H].unflatten(1, (HEADS, 64))
        k, v = (kv[:, i * H:(i + 1) * H].unflatten(1, (HEADS, 64)) for i in (1, 2))
        kmax, vmax = max(kmax, k.abs().max().item()), max(vmax, v.abs().max().item())
        z = torch.einsum("thd,khd->htk", q, k) / 8
        seen = torch.arange(kv.shape[0], device="cuda")[None] <= lens[s] + torch.arange(more[s], device="cuda")[:, None]
        ctx[b:b + more[s]] = torch.einsum("htk,khd->thd", torch.softmax(z.masked_fill(~seen, -math.inf), -1), v).flatten(1)
    pre = ctx @ out_w.double() + out_b.double() + new.double()
    want = torch.nn.functional.layer_norm(pre, (H,), ln_w.double(), ln_b.double(), 1e-12)
    # a code is off by half a step of at most amax / 127 * 129 / 128 (2^-7.9 amax) and the projections by 2^-11 of a value: scores by
    # 8 * max|q| * 2^-7.9 kmax / 8, here under 0.15 in the worst case; outputs by that share of the spread of the values and 2^-7.9 vmax; the dense layer
    # passes an error of e on as at most e * sum|w| (about 0.8 sqrt(H) e), the LayerNorm divides by a deviation of about 1
    q_max = f(new)[:, :H].abs().max().item()
    score = q_max * (2.0 ** -7.9 + 2.0 ** -10) * kmax
    bound = (2 * math.expm1(score) + 2.0 ** -7.9 + 2.0 ** -9) * vmax * out_w.double().abs().sum(0).max().item()
    dev = pre.std(1).min().item()
    off = (got.double() - want).abs().max().item()
    assert off <= 2 * bound / dev * ln_w.abs().max().item() + 2.0 ** -9
    # and far better than the worst case where the errors are independent
    assert (got.double() - want).pow(2).mean().sqrt() < 0.02


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_masked_token_head(mods, dtype):
    modeling, ops = mods
    g = torch.Generator(device="cuda").manual_seed(6)
    vocab, rows = 1003, 9
    w, b, e = (_weights(g, *s).to(dtype) for s in ((H, H), (H,), (vocab, H)))
    bias = _weights(g, vocab).to(dtype)
    ln_w, ln_b = torch.ones(H, device="cuda", dtype=dtype), torch.zeros(H, device="cuda", dtype=dtype)
    head = modeling.BertLMHead(w, b, ln_w, ln_b, e * 30, bias)
    x = torch.randn(rows, H, device="cuda", generator=g).to(dtype)
    t = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda", generator=g)
    t[2] = -1
    scores, z = head(x, t, top_k=4)
    assert z.shape == (rows, vocab) and z.stride(0) % 64 == 0
    h = torch.nn.functional.gelu(x.double() @ w.double() + b.double(), approximate="tanh")
    h = torch.nn.functional.layer_norm(h, (H,), None, None, 1e-12)
    want = h @ (e * 30).double().t() + bias.double()
    # GELU output, LayerNorm output and logits are rounded to 16 bits each: the first two reach a logit as sqrt(H) independent errors of
    # its terms, bounded here by 4 of them at their largest
    eps = torch.finfo(dtype).eps / 2
    tol = eps * want.abs() + 8 * eps * h.abs().max() * (e * 30).double().pow(2).sum(1).sqrt()
    assert ((z.double() - want).abs() <= tol + 0.02 * tol.max()).all()
    lp = torch.log_softmax(z.double(), 1)
    keep = t >= 0
    assert ((scores.logp.double() - lp.gather(1, t.clamp(min=0).long()[:, None])[:, 0]).abs()[keep] < 2.0 ** -15).all()
    assert scores.logp[2] == 0
    d = head.logits_gradient(z, t, scores, grad_logp=-torch.ones(rows, device="cuda"))
    ref = lp.exp()
    ref[torch.arange(rows, device="cuda"), t.clamp(min=0).long()] -= 1
    ref[2] = 0
    assert ((d.double() - ref).abs() <= eps * ref.abs() + 2.0 ** -16).all()
    ops.check_device()
