"""The operators that answer from encoded documents, as timed cases over their public entry points.

Kinds of a case:

* ``write``        keys and values of new tokens are quantised into a cache of 64-token blocks, 8 bits a value, with one
                   scale for each block and head (``ops.kv_cache_write``).
* ``read``         the values of a range of tokens are brought back in 16 bits (``ops.kv_cache_read``).
* ``attention``    query tokens attend over such a cache (``ops.cached_attention``).
* ``scores``       log probabilities of given tokens, entropy and the best alternatives of each row of logits
                   (``ops.token_logprobs``).
* ``scores_grad``  the gradient of those with respect to the logits (``ops.token_logprobs_backward``).

Heads are 64 wide.  Head counts, hidden sizes, document lengths and the vocabulary are those of the repository's
benchmark models (12 or 16 heads, documents of up to 4096, 8192 and 16384 tokens, 50358 tokens of vocabulary).
"""
import math
import random

import torch

own = False

BLOCK = 64
DIM = 64
VOCAB = 50358

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one step of 32 running answers: a token each joins its own document, most of them inside a block that has tokens
        dict(name="write_step", kind="write", format="e4m3", dtype="bf16", kv_heads=12, sequences=32, fewest=1, most=1,
             least_start=100, most_start=4095, lengths=1),
        # eight encoded documents go into the cache at once
        dict(name="write_documents", kind="write", format="int8", dtype="f16", kv_heads=12, sequences=8, fewest=1024,
             most=4096, least_start=0, most_start=0, lengths=2),
        # a paragraph is brought back
        dict(name="read_paragraph", kind="read", format="int8", dtype="bf16", kv_heads=12, sequences=1, fewest=301,
             most=301, least_start=77, most_start=77, lengths=3),
        # the documents of a batch of the large model are brought back, to be attended to in 16 bits
        dict(name="read_documents", kind="read", format="e4m3", dtype="f16", kv_heads=16, sequences=8, fewest=2000,
             most=8192, least_start=0, most_start=500, lengths=4),
        # one token of one answer over one document of the base model's maximum length: all latency
        dict(name="attention_one_token", kind="attention", format="e4m3", dtype="f16", heads=12, kv_heads=12,
             sequences=1, fewest=1, most=1, least_context=4096, most_context=4096, causal=True, lengths=5),
        # a step of 24 answers over ragged long documents, four query heads to a key head
        dict(name="attention_step", kind="attention", format="int8", dtype="bf16", heads=16, kv_heads=4, sequences=24,
             fewest=1, most=1, least_context=1000, most_context=16384, causal=True, lengths=6),
        # questions of some tokens, each over its document as a whole
        dict(name="attention_questions", kind="attention", format="int8", dtype="f16", heads=12, kv_heads=12,
             sequences=16, fewest=5, most=64, least_context=512, most_context=4096, causal=False, lengths=7),
        # long continuations that have just joined their documents: the largest call
        dict(name="attention_prompt", kind="attention", format="e4m3", dtype="bf16", heads=12, kv_heads=12, sequences=4,
             fewest=700, most=2048, least_context=2048, most_context=8192, causal=True, lengths=8),
        # the masked tokens of one text
        dict(name="scores_masked", kind="scores", dtype="bf16", rows=19, vocab=VOCAB, pitch=50368, top=5, ignored=0.0),
        # every token of a small batch, logits without padding columns (rows begin at odd addresses)
        dict(name="scores_batch", kind="scores", dtype="f16", rows=2048, vocab=VOCAB, pitch=VOCAB, top=8, ignored=0.1),
        # the loss gradient of the masked tokens of a small batch, logits in 32 bits
        dict(name="scores_grad_masked", kind="scores_grad", dtype="f32", rows=77, vocab=VOCAB, pitch=50368, top=0,
             ignored=0.1),
        # and of a training batch, with a reward on the entropy and on the alternatives
        dict(name="scores_grad_batch", kind="scores_grad", dtype="bf16", rows=4096, vocab=VOCAB, pitch=50368, top=4,
             ignored=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, without a name."""
    kind = rng.choice(["write", "read", "attention", "attention", "attention", "scores", "scores_grad"])
    lengths = rng.randrange(1, 1 << 20)
    if kind in ("scores", "scores_grad"):
        dtype = rng.choice(["f16", "bf16", "f32"])
        vocab = VOCAB if rng.random() < 0.5 else _log_int(rng, 1000, 130000)
        rows = _log_int(rng, 1, max(1, min(8192, 200_000_000 // (vocab * (2 if dtype == "f32" else 1)))))
        pitch = rng.choice([vocab, -(-vocab // 64) * 64, vocab + rng.randrange(1, 100)])
        return dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, pitch=pitch, top=rng.choice([0, 1, 5, 8, 20]),
                    ignored=rng.choice([0.0, 0.15]))
    fmt, dtype = rng.choice(["e4m3", "int8"]), rng.choice(["f16", "bf16"])
    if kind in ("write", "read"):
        kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
        most = 1 if kind == "write" and rng.random() < 0.3 else _log_int(rng, 1, 8192)
        sequences = _log_int(rng, 1, max(1, min(64, 65536 // most * 12 // kv_heads)))
        start = rng.choice([0, _log_int(rng, 1, 8192)])
        return dict(kind=kind, format=fmt, dtype=dtype, kv_heads=kv_heads, sequences=sequences,
                    fewest=max(1, int(most * rng.uniform(0.1, 1.0))), most=most, least_start=int(start * rng.random()),
                    most_start=start, lengths=lengths)
    heads, kv_heads = rng.choice([(12, 12), (16, 16), (16, 4), (12, 4), (8, 1), (12, 3)])
    most = rng.choice([1, 1, rng.randrange(2, 17), _log_int(rng, 2, 2048)])
    most_context = max(most, _log_int(rng, 16, 65536 if most == 1 else 16384))
    cost = heads * (most_context + 1) * max(most, 16 * kv_heads / heads)  # row-key pairs of a sequence
    sequences = max(1, min(48, int(270_000_000 / cost), 5_000_000 // (most_context * kv_heads)))
    sequences = _log_int(rng, 1, sequences)
    return dict(kind=kind, format=fmt, dtype=dtype, heads=heads, kv_heads=kv_heads, sequences=sequences,
                fewest=max(1, int(most * rng.uniform(0.1, 1.0))), most=most,
                least_context=max(most, int(most_context * rng.uniform(0.1, 1.0))), most_context=most_context,
                causal=rng.random() < 0.5, lengths=lengths)


def _batch(case):
    """Tokens of each sequence and what is in the cache before them (write, read) or with them (attention)."""
    rng = random.Random(case["lengths"])
    a, b = ("least_context", "most_context") if case["kind"] == "attention" else ("least_start", "most_start")
    n = [rng.randint(case["fewest"], case["most"]) for _ in range(case["sequences"])]
    before = [rng.randint(case[a], case[b]) for _ in range(case["sequences"])]
    n[rng.randrange(len(n))], before[rng.randrange(len(n))] = case["most"], case[b]
    return n, before


def work(case):
    if case["kind"] in ("scores", "scores_grad"):
        values = case["rows"] * case["vocab"]
        k = 1 if case["kind"] == "scores" else 2
        return {"bytes": values * _SIZE[case["dtype"]] * k + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * values}
    n, before = _batch(case)
    kvh = case["kv_heads"]
    if case["kind"] in ("write", "read"):
        return {"bytes": sum(n) * kvh * 2 * DIM * (2 + 1), "flops": sum(n) * kvh * 2 * DIM * 2}
    heads = case["heads"]
    pairs = sum(t * c - (t * (t - 1) // 2 if case["causal"] else 0) for t, c in zip(n, before))
    return {"bytes": sum(before) * kvh * 2 * DIM + sum(n) * heads * DIM * 4 + sum(-(-c // BLOCK) for c in before) * kvh * 8,
            "flops": 4 * DIM * heads * pairs}


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _first(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _keys(g, tokens, heads):
    """Projected keys or values: a spread of sizes over the channels and a few channels that stand out."""
    size = torch.exp(0.5 * torch.randn(1, heads, DIM, device="cuda", generator=g))
    size = size * (1 + 7 * (torch.rand(1, heads, DIM, device="cuda", generator=g) < 0.03))
    return torch.randn(tokens, heads, DIM, device="cuda", generator=g) * size


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TORCH[case["dtype"]]
    s = dict(case=case)
    if case["kind"] in ("scores", "scores_grad"):
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        store = torch.empty(rows, case["pitch"], dtype=dtype, device="cuda")
        sharp = 1 + 2 * torch.rand(rows, 1, device="cuda", generator=g)  # rows from unsure to nearly sure
        for i in range(0, rows, 1024):
            z = torch.randn(min(1024, rows - i), case["pitch"], device="cuda", generator=g)
            store[i:i + 1024] = z * sharp[i:i + 1024]
        logits = store[:, :vocab]
        targets = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda", generator=g)
        if case["ignored"]:
            targets[torch.rand(rows, device="cuda", generator=g) < case["ignored"]] = -1
        s.update(logits=logits, targets=targets)
        if case["kind"] == "scores_grad":
            z = logits.float()
            z -= z.max(1, keepdim=True).values
            total = z.exp().sum(1)
            s["stats"] = torch.stack([logits.float().max(1).values, total.log()], 1).contiguous()
            s["entropy"] = total.log() - (z.exp() * z).sum(1) / total
            s["grad_logp"] = torch.randn(rows, device="cuda", generator=g) / rows
            s["grad_entropy"] = torch.randn(rows, device="cuda", generator=g) / rows if top else None
            s["top_ids"] = s["grad_top"] = None
            if top:
                s["top_ids"] = torch.topk(z, top, 1).indices.int().contiguous()
                s["grad_top"] = torch.randn(rows, top, device="cuda", generator=g) / rows
        return s
    n, before = _batch(case)
    kvh = case["kv_heads"]
    attention = case["kind"] == "attention"
    held = before if attention else [b + t for b, t in zip(before, n)]  # tokens of each sequence in the cache
    blocks = [-(-c // BLOCK) for c in held]
    total = sum(blocks)
    order = torch.randperm(total, device="cuda", generator=g).int()
    table = torch.zeros(len(n), max(blocks), dtype=torch.int32, device="cuda")
    first = _first(blocks)
    for i, b in enumerate(blocks):
        table[i, :b] = order[first[i]:first[i + 1]]
    for name in ("k", "v"):
        x = _keys(g, total * BLOCK, kvh).view(total, BLOCK, kvh, DIM).permute(0, 2, 1, 3)
        scale = _scale_of(x.abs().amax((2, 3)), case["format"]) * 2.0 ** -(case["kind"] == "write")
        code = (x / scale[:, :, None, None])
        if case["format"] == "int8":
            s[name + "_cache"] = code.round().clamp(-127, 127).to(torch.int8).contiguous()
        else:
            s[name + "_cache"] = code.clamp(-448, 448).to(torch.float8_e4m3fn).contiguous()
        s[name + "_scale"] = scale.contiguous()
    s.update(table=table, first=_i32(_first(n)), before=_i32(before), tokens=sum(n), most=max(n))
    if case["kind"] == "write":
        qkv = torch.cat([_keys(g, sum(n), kvh).reshape(sum(n), -1) for _ in range(3)], 1).to(dtype)  # as projected: q | k | v
        s.update(k=qkv[:, kvh * DIM:2 * kvh * DIM].unflatten(1, (kvh, DIM)), v=qkv[:, 2 * kvh * DIM:].unflatten(1, (kvh, DIM)))
    if attention:
        s["q"] = torch.randn(sum(n), case["heads"], DIM, device="cuda", generator=g).to(dtype)
    if own:
        from raptor_t_b200 import ops
        s["cache"] = ops.KvCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from raptor_t_b200 import ops
    case = s["case"]
    if case["kind"] == "scores":
        r = ops.token_logprobs(s["logits"], s["targets"], top_k=case["top"])
        return [r.logp, r.entropy, r.stats] + ([r.top_ids, r.top_logp] if case["top"] else [])
    if case["kind"] == "scores_grad":
        return ops.token_logprobs_backward(s["logits"], s["targets"], s["stats"], s["entropy"], grad_logp=s["grad_logp"],
                                           grad_entropy=s["grad_entropy"], top_ids=s["top_ids"], grad_top=s["grad_top"])
    if case["kind"] == "write":
        ops.kv_cache_write(s["cache"], s["k"], s["v"], s["table"], s["before"], s["first"], max_tokens=s["most"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    if case["kind"] == "read":
        return ops.kv_cache_read(s["cache"], s["table"], s["before"], s["first"], s["tokens"], _TORCH[case["dtype"]],
                                 max_tokens=s["most"])
    return ops.cached_attention(s["q"], s["cache"], s["table"], s["before"], s["first"], max_q=s["most"], scale=0.125,
                                causal=case["causal"])


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _scale_of(most, fmt):
    """The scale of a block whose largest value is `most`: what brings it to the largest code, rounded up to a power of
    two (e4m3) or to eight significant bits (int8)."""
    low = 0x7FFFFF if fmt == "e4m3" else 0xFFFF
    bits = (most / (448 if fmt == "e4m3" else 127)).view(torch.int32)
    return ((bits + low) & ~low).view(torch.float32).clamp(min=2.0 ** -100)


def _run_plain(s):
    kind = s["case"]["kind"]
    return {"scores": _scores, "scores_grad": _scores_grad, "write": _write, "read": _read, "attention": _attention}[kind](s)


def _scores(s):
    z, top = s["logits"].float(), s["case"]["top"]
    m = z.max(1, keepdim=True).values
    e = (z - m).exp()
    total = e.sum(1)
    log_total = total.log()
    entropy = log_total - (e * (z - m)).sum(1) / total
    given = s["targets"] >= 0
    at = s["targets"].clamp(min=0).long()[:, None]
    logp = torch.where(given, z.gather(1, at)[:, 0] - m[:, 0] - log_total, 0.0)
    out = [logp, entropy, torch.stack([m[:, 0], log_total], 1)]
    if top:
        v, i = torch.sort(z, dim=1, descending=True, stable=True)
        out += [i[:, :top].int(), v[:, :top] - m - log_total[:, None]]
    return out


def _scores_grad(s):
    z = s["logits"].float()
    logp = z - s["stats"][:, :1] - s["stats"][:, 1:]
    given = s["targets"] >= 0
    g = torch.where(given, s["grad_logp"], 0.0)
    pull = g[:, None].clone()
    if s["case"]["top"]:
        pull = pull + s["grad_top"].sum(1, keepdim=True) + s["grad_entropy"][:, None] * (logp + s["entropy"][:, None])
    d = -logp.exp() * pull
    d.scatter_add_(1, s["targets"].clamp(min=0).long()[:, None], g[:, None])
    if s["case"]["top"]:
        d.scatter_add_(1, s["top_ids"].long(), s["grad_top"])
    return d.to(s["logits"].dtype)


def _positions(s, room):
    """For every sequence and each of `room` places: the row of the packed tokens there, and whether there is one."""
    n = s["first"][1:] - s["first"][:-1]
    at = torch.arange(room, dtype=torch.int32, device="cuda")[None]
    return s["first"][:-1, None] + at, at < n[:, None]


def _values(cache, scale):
    return cache.float() * scale[:, :, None, None]


def _write(s):
    case, start = s["case"], s["before"]
    n = s["first"][1:] - s["first"][:-1]
    room = s["most"] // BLOCK + 2  # blocks that a sequence's new tokens touch at most
    blk = start[:, None] // BLOCK + torch.arange(room, dtype=torch.int32, device="cuda")[None]
    pos = blk[:, :, None] * BLOCK + torch.arange(BLOCK, dtype=torch.int32, device="cuda")  # [sequences, room, 64]
    new = (pos >= start[:, None, None]) & (pos < (start + n)[:, None, None])
    row = (s["first"][:-1, None, None] + pos - start[:, None, None]).clamp(0, s["tokens"] - 1).long()
    touched = new.any(2)
    older = (pos[:, :, 0] < start[:, None])[:, :, None]
    page = s["table"].gather(1, blk.clamp(max=s["table"].shape[1] - 1).long()).long()
    pages = s["k_cache"].shape[0]
    # which touched block, if any, is the new content of each page
    owner = torch.full((pages + 1,), -1, dtype=torch.long, device="cuda")
    owner[torch.where(touched, page, pages).flatten()] = torch.arange(page.numel(), device="cuda")
    owner = owner[:pages]
    has, owner = owner >= 0, owner.clamp(min=0)
    out = []
    for x, code, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.float()[row]  # [sequences, room, 64, heads, 64]
        most = torch.where(new[..., None, None], x.abs(), 0.0).amax((2, 4))
        need, was = _scale_of(most, case["format"]), scale[page]
        now = torch.where(older & (need <= was), was, need)
        old = _values(code, scale)[page].permute(0, 1, 3, 2, 4)
        q = torch.where(new[..., None, None], x, old) / now[:, :, None, :, None]
        if case["format"] == "int8":
            q = q.round().clamp(-127, 127)
        kept = (~new & ~(older & (pos < start[:, None, None])))[..., None, None]  # rows that hold no token stay as they are
        now = now.flatten(0, 1)[owner]
        q = torch.where(kept, code.float()[page].permute(0, 1, 3, 2, 4), q).permute(0, 1, 3, 2, 4).flatten(0, 1)[owner]
        code.copy_(torch.where(has[:, None, None, None], q.to(code.dtype).float(), code.float()).to(code.dtype))
        scale.copy_(torch.where(has[:, None], now, scale))
        out.append((code, scale))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _read(s):
    case = s["case"]
    t = torch.arange(s["tokens"], dtype=torch.int32, device="cuda")
    seq = (t[:, None] >= s["first"][None, 1:]).sum(1)
    pos = t - s["first"][seq] + s["before"][seq]
    page, slot = s["table"][seq, pos // BLOCK].long(), (pos % BLOCK).long()
    return [(c[page, :, slot].float() * f[page][:, :, None]).to(_TORCH[case["dtype"]])
            for c, f in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]


def _attention(s):
    case = s["case"]
    heads, kvh = case["heads"], case["kv_heads"]
    row, there = _positions(s, s["most"])
    q = s["q"].float()[row.clamp(max=s["tokens"] - 1).long()]  # [sequences, most, heads, 64]
    q = q.unflatten(2, (kvh, heads // kvh)).permute(0, 2, 3, 1, 4)  # [sequences, kv heads, group, most, 64]
    k, v = (_values(c, f)[s["table"].long()].transpose(2, 3).flatten(1, 2).transpose(1, 2)[:, :, None]
            for c, f in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))  # [sequences, kv heads, 1, keys, 64]
    score = torch.matmul(q, k.transpose(3, 4)) * 0.125
    last = s["before"][:, None].expand(-1, s["most"])
    if case["causal"]:
        last = last - (s["first"][1:] - s["first"][:-1])[:, None] + torch.arange(1, s["most"] + 1, device="cuda")
    seen = torch.arange(score.shape[-1], device="cuda") < last[:, :, None]  # [sequences, most, keys]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    m = score.max(-1, keepdim=True).values
    p = (score - torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [sequences, most, heads, 64]
    out = torch.zeros(s["tokens"] + 1, heads, DIM, device="cuda")
    out[torch.where(there, row, s["tokens"]).long()] = o
    return out[:-1].to(_TORCH[case["dtype"]])


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attention": _exact_attention, "scores": _exact_scores,
            "scores_grad": _exact_scores_grad}[case["kind"]](s, case)


def _exact_scores(s, case):
    logp, entropy, stats, top = [], [], [], []
    for i in range(0, case["rows"], 256):
        z = s["logits"][i:i + 256].double()
        lse = torch.logsumexp(z, 1)
        lp = z - lse[:, None]
        t = s["targets"][i:i + 256].long()
        logp.append(torch.where(t < 0, 0.0, lp[torch.arange(len(t), device="cuda"), t.clamp(min=0)]))
        entropy.append(-(lp.exp() * lp).sum(1))
        m = z.amax(1)
        stats.append(torch.stack([m, lse - m], 1))
        if case["top"]:
            top.append(torch.topk(lp, case["top"], 1).values)
    out = [torch.cat(logp), torch.cat(entropy), torch.cat(stats)]
    return out + ([None, torch.cat(top)] if case["top"] else [])


def _exact_scores_grad(s, case):
    out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device="cuda")
    for i in range(0, case["rows"], 256):
        j = min(i + 256, case["rows"])
        z = s["logits"][i:j].double()
        lp = z - s["stats"][i:j].double().sum(1, keepdim=True)
        p = lp.exp()
        r, t = torch.arange(j - i, device="cuda"), s["targets"][i:j].long()
        g = s["grad_logp"][i:j].double() * (t >= 0)
        d = -p * g[:, None]
        d[r, t.clamp(min=0)] += g
        if case["top"]:
            h = s["entropy"][i:j].double()[:, None]
            d -= s["grad_entropy"][i:j].double()[:, None] * p * (lp + h)
            for c in range(case["top"]):
                gt = s["grad_top"][i:j, c].double()
                d -= p * gt[:, None]
                d[r, s["top_ids"][i:j, c].long()] += gt
        out[i:j] = d
    return out


def _e4m3(x):
    """The nearest value of four significant bits, exponents from -6, ties to even."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(x / step) * step, -448, 448)


def _exact_write(s, case):
    first, start, table = s["first"].tolist(), s["before"].tolist(), s["table"].tolist()
    out = []
    for x, code, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x, code, scale = x.double(), code.double(), scale.double()
        for i, b0 in enumerate(start):
            end = b0 + first[i + 1] - first[i]
            for b in range(b0 // BLOCK, -(-end // BLOCK)):
                lo, hi = max(b0, b * BLOCK), min(end, (b + 1) * BLOCK)
                page = table[i][b]
                new = x[first[i] + lo - b0:first[i] + hi - b0].transpose(0, 1)  # [heads, tokens, 64]
                a = new.abs().amax((1, 2))
                if case["format"] == "e4m3":
                    need = torch.exp2(torch.ceil(torch.log2(a / 448)))
                    need = torch.where(need / 2 * 448 >= a, need / 2, torch.where(need * 448 < a, need * 2, need))
                else:
                    unit = torch.exp2(torch.floor(torch.log2(a / 127)) - 7)
                    need = torch.ceil(a / 127 / unit) * unit
                need = need.clamp(min=2.0 ** -100)
                now = torch.where((need <= scale[page]) & (lo > b * BLOCK), scale[page], need)
                f = now[:, None, None]
                old = code[page, :, :lo - b * BLOCK] * (scale[page][:, None, None])
                both = torch.cat([old, new], 1) / f
                code[page, :, :hi - b * BLOCK] = _e4m3(both) if case["format"] == "e4m3" else torch.round(both)
                scale[page] = now
        out.append((code, scale))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _exact_read(s, case):
    first, start, table = s["first"].tolist(), s["before"].tolist(), s["table"].long()
    out = []
    for code, scale in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])):
        parts = []
        for i, b0 in enumerate(start):
            n = first[i + 1] - first[i]
            pages = table[i, :-(-(b0 + n) // BLOCK)]
            x = code[pages].double() * scale[pages].double()[:, :, None, None]
            parts.append(x.transpose(1, 2).flatten(0, 1)[b0:b0 + n])
        out.append(torch.cat(parts))
    return out


def _exact_attention(s, case):
    first, context, table = s["first"].tolist(), s["before"].tolist(), s["table"].long()
    group = case["heads"] // case["kv_heads"]
    out = []
    for i, c in enumerate(context):
        n = first[i + 1] - first[i]
        pages = table[i, :-(-c // BLOCK)]
        k, v = (x[pages].double().mul(f[pages].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :c]
                for x, f in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))  # [kv heads, keys, 64]
        o = torch.zeros(n, case["heads"], DIM, dtype=torch.float64, device="cuda")
        q = s["q"][first[i]:first[i + 1]].double()
        for h in range(case["heads"]):
            z = q[:, h] @ k[h // group].T / 8
            if case["causal"]:
                hidden = torch.arange(c, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + (c - n)
                z = z.masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(z, 1) @ v[h // group]
        out.append(o)
    return torch.cat(out)
