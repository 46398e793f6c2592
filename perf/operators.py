"""Cases of the prompt and beam-search operators that stand beside the decode-step attention.

Three operators over the token-major K/V pools ``[HK, T, D]``:

* ``chunk``: attention of ragged chunks of new tokens over each sequence's pages
  of the pools (prompt chunks, and single tokens as the decode form);
* ``rotary``: q/k RMSNorm, rotary positions and the append of K and V to the pools;
* ``beam``: the best continuations over beams x vocabulary, and the reordering of
  the beams' states.

``run`` computes an operator in elementary torch operations, or calls the
package's kernels where ``own`` is true; ``exact`` restates the definitions in
64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------
def _chunk(name, batch, chunk, context, hq, hk, dim, page, dtype, ragged, causal=True):
    return dict(name=name, op="chunk", batch=batch, chunk=chunk, context=context, hq=hq, hk=hk, dim=dim, page=page,
                dtype=dtype, ragged=ragged, causal=causal)


def _rotary(name, tokens, hq, hk, dim, rot, far, interleaved, norm, scaled, dtype):
    return dict(name=name, op="rotary", tokens=tokens, hq=hq, hk=hk, dim=dim, rot=rot, far=far,
                interleaved=interleaved, norm=norm, scaled=scaled, dtype=dtype)


def _beam(name, requests, beams, k, vocab, dtype, finished, masked, length):
    return dict(name=name, op="beam", requests=requests, beams=beams, k=k, vocab=vocab, dtype=dtype,
                finished=finished, masked=masked, length=length)


def listed():
    return [
        # one request's next token over its path of pool positions: the latency of a call
        _chunk("chunk one token", 1, 1, 1000, 32, 8, 128, 1, "bf16", False),
        # a decode batch with contexts of very different lengths, 16-token pages
        _chunk("chunk decode batch", 64, 1, 8192, 32, 8, 128, 16, "bf16", True),
        # the new parts of several prompts after cached prefixes, odd lengths, position by position
        _chunk("chunk ragged prompts", 6, 391, 3064, 32, 8, 128, 1, "f16", True),
        # small heads, chunks that are not a multiple of anything
        _chunk("chunk small heads", 5, 777, 2300, 16, 2, 64, 64, "bf16", True),
        # a whole document at once, as the shared root of a request tree
        _chunk("chunk document", 1, 8128, 8128, 32, 8, 128, 1, "bf16", False),
        # one decode step of a small batch: a call of every layer
        _rotary("rotary decode step", 16, 32, 8, 128, 128, 4096, False, True, False, "bf16"),
        # a long prompt
        _rotary("rotary prompt", 16384, 32, 8, 128, 128, 16384, False, True, False, "bf16"),
        # part of the head, interleaved pairs, far positions of a scaled context
        _rotary("rotary partial far", 1337, 16, 2, 64, 32, 1000000, True, False, True, "f16"),
        # one request, a small vocabulary, logits kept in 32 bits
        _beam("beam small", 1, 4, 8, 32000, "f32", False, False, 128),
        # a serving batch over a large vocabulary
        _beam("beam batch", 16, 4, 8, 151936, "bf16", False, False, 512),
        # many requests with wide beams, an odd vocabulary, finished beams, tokens ruled out
        _beam("beam wide", 32, 16, 32, 50257, "f16", True, True, 257),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("chunk", "chunk", "rotary", "beam"))
    if op == "chunk":
        dim, (hq, hk) = rng.choice((64, 128, 128)), rng.choice(((32, 8), (16, 2), (8, 8), (24, 8), (12, 4)))
        batch, chunk = _log_int(rng, 1, 48), rng.choice((1, 0))
        chunk = chunk or _log_int(rng, 2, 4096)
        # scores of the plain form: batch * hq * chunk * (context) values, bounded by the document's
        most = min(32768, 8128 * 8128 // (batch * chunk))
        context = max(chunk, _log_int(rng, 1, max(chunk, most, 64)))
        if batch * chunk * context > 8128 * 8128:
            batch = max(1, 8128 * 8128 // (chunk * context))
        return _chunk("", batch, chunk, context, hq, hk, dim, rng.choice((1, 1, 16, 32, 128)),
                      rng.choice(("bf16", "f16")), rng.random() < 0.7, rng.random() < 0.85)
    if op == "rotary":
        dim, (hq, hk) = rng.choice((64, 128, 128)), rng.choice(((32, 8), (16, 2), (8, 8), (24, 8), (12, 4)))
        return _rotary("", _log_int(rng, 1, 16384), hq, hk, dim, rng.choice((dim, dim, dim // 2)),
                       _log_int(rng, 64, 1000000), rng.random() < 0.4, rng.random() < 0.6, rng.random() < 0.4,
                       rng.choice(("bf16", "f16")))
    beams = rng.choice((1, 2, 3, 4, 5, 8, 16))
    vocab = _log_int(rng, 500, 152000)
    requests = _log_int(rng, 1, max(1, min(64, 25700000 // (beams * vocab))))
    return _beam("", requests, beams, rng.choice((beams, 2 * beams)), vocab, rng.choice(("f32", "bf16", "f16")),
                 rng.random() < 0.5, rng.random() < 0.5, _log_int(rng, 1, 2048))


def _case_lengths(case):
    """(new tokens, context length) of every sequence of a chunk case, on the host: the same for every seed."""
    batch, chunk, context = case["batch"], case["chunk"], case["context"]
    if not case["ragged"]:
        return [chunk] * batch, [context] * batch
    generator = torch.Generator().manual_seed(97)
    fresh, total = [], []
    for _ in range(batch):
        u = torch.rand(2, generator=generator).tolist()
        n = max(1, int(round(chunk * (0.25 + 0.75 * u[0]))))
        before = context - chunk
        fresh.append(n)
        total.append(n + int(round(before * u[1])))
    fresh[0], total[0] = chunk, context
    return fresh, total


# ---- inputs -----------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"chunk": _prepare_chunk, "rotary": _prepare_rotary, "beam": _prepare_beam}[case["op"]](case, seed, g)


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_chunk(case, seed, g):
    dtype, page, dim = _DTYPES[case["dtype"]], case["page"], case["dim"]
    fresh, total = _case_lengths(case)
    pages = [-(-t // page) for t in total]
    width = max(1, max(pages))
    # pages of a sequence lie anywhere in the pool, in any order; a quarter of the pool is other sequences'
    pool_pages = sum(pages) + max(1, sum(pages) // 4)
    order = torch.randperm(pool_pages, generator=g, device="cuda").to(torch.int32)
    row = torch.tensor(pages, device="cuda")
    first = torch.cumsum(row, 0) - row
    column = torch.arange(width, device="cuda")
    index = (first[:, None] + column).clamp(max=pool_pages - 1)
    table = torch.where(column < row[:, None], order[index], -1).to(torch.int32).contiguous()
    cu = torch.tensor([0] + fresh, device="cuda").cumsum(0).to(torch.int32)
    return dict(op="chunk", q=_normal(g, dtype, sum(fresh), case["hq"], dim) * 2,
                kp=_normal(g, dtype, case["hk"], pool_pages * page, dim),
                vp=_normal(g, dtype, case["hk"], pool_pages * page, dim),
                table=table, lens=torch.tensor(total, device="cuda", dtype=torch.int32), cu=cu, page=page,
                causal=case["causal"], most_new=max(fresh), most_keys=max(total))


def _prepare_rotary(case, seed, g):
    dtype, n, dim, hq, hk = _DTYPES[case["dtype"]], case["tokens"], case["dim"], case["hq"], case["hk"]
    # q, k and v are slices of one fused projection
    rows = _normal(g, dtype, n, (hq + 2 * hk) * dim) * 3
    parts = rows.split((hq * dim, hk * dim, hk * dim), dim=1)
    tokens = n + 64
    # a plain base, or frequencies stretched for a long context
    freq = 1.0 / 1000000.0 ** (torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float32) / case["rot"])
    if case["scaled"]:
        freq = torch.where(freq < 0.05, freq / 8, freq)
    start = torch.randint(0, max(1, case["far"]), (n,), generator=g, device="cuda")
    return dict(op="rotary", q=parts[0].view(n, hq, dim), k=parts[1].view(n, hk, dim), v=parts[2].view(n, hk, dim),
                positions=start, freq=freq.contiguous(),
                kp=_normal(g, dtype, hk, tokens, dim), vp=_normal(g, dtype, hk, tokens, dim),
                targets=torch.randperm(tokens, generator=g, device="cuda")[:n].contiguous(),
                interleaved=case["interleaved"], factor=1.2 if case["scaled"] else 1.0,
                qw=(1 + 0.2 * _normal(g, torch.float32, dim)).to(dtype) if case["norm"] else None,
                kw=(1 + 0.2 * _normal(g, torch.float32, dim)).to(dtype) if case["norm"] else None, eps=1e-6)


def _prepare_beam(case, seed, g):
    r, w, v, dtype = case["requests"], case["beams"], case["vocab"], _DTYPES[case["dtype"]]
    logits = torch.randn((r, w, v), generator=g, device="cuda").mul_(2.5)
    if case["masked"]:                                     # tokens a grammar rules out
        logits.masked_fill_(torch.rand((1, 1, v), generator=g, device="cuda") < 0.3, -math.inf)
    scores = -20 * torch.rand((r, w), generator=g, device="cuda")
    finished = (torch.rand((r, w), generator=g, device="cuda") < 0.25) if case["finished"] else None
    states = torch.randint(0, 1 << 30, (r, w, case["length"]), generator=g, device="cuda", dtype=torch.int32)
    return dict(op="beam", logits=logits.to(dtype), scores=scores.sort(1, descending=True)[0], finished=finished,
                end=v // 2, k=case["k"], states=states)


# ---- one pass ---------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"chunk": _plain_chunk, "rotary": _plain_rotary, "beam": _plain_beam}[state["op"]](state)


def _own(s):
    if s["op"] == "chunk":
        chunk_attention = _package("chunk").chunk_attention
        n, hq = s["q"].shape[:2]
        lse = torch.empty((n, hq), device=s["q"].device, dtype=torch.float32)
        out = chunk_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["cu"], page_size=s["page"],
                              causal=s["causal"], out_lse=lse)
        return out, lse
    if s["op"] == "rotary":
        q = _package("rotary").rotary_append(
            s["q"], s["k"], s["v"], s["positions"], s["freq"], s["kp"], s["vp"], s["targets"],
            interleaved=s["interleaved"], attention_factor=s["factor"], q_weight=s["qw"], k_weight=s["kw"],
            eps=s["eps"])
        return q, s["kp"], s["vp"]
    beam = _package("beam")
    scores, parents, tokens = beam.beam_select(s["logits"], s["scores"], s["k"], finished=s["finished"],
                                               end_token=s["end"])
    beams = s["states"].shape[1]
    return scores, parents, tokens, beam.beam_reorder(s["states"], parents[:, :beams])


_modules = {}


def _package(name):
    if name not in _modules:
        root = os.path.join(os.getcwd(), "tree-attention-scheduling_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        _modules[name] = __import__("tree_attention." + name, fromlist=[name])
    return _modules[name]


def _plain_chunk(s):
    q, lens, cu, page = s["q"], s["lens"], s["cu"], s["page"]
    n, hq, dim = q.shape
    hk = s["kp"].shape[0]
    fresh = cu[1:] - cu[:-1]
    i = torch.arange(s["most_new"], device=q.device)
    token = (cu[:-1, None] + i).clamp(max=n - 1).long()
    queries = q[token].float().view(len(lens), len(i), hk, hq // hk, dim)
    key = torch.arange(s["most_keys"], device=q.device)
    position = s["table"][:, key // page].clamp(min=0).long() * page + key % page
    keys, values = s["kp"][:, position].float(), s["vp"][:, position].float()
    scores = torch.einsum("bnhgd,hbkd->bhgnk", queries, keys) / math.sqrt(dim)
    limit = lens[:, None] - fresh[:, None] + i + 1 if s["causal"] else lens[:, None].expand(-1, len(i))
    hidden = key >= torch.minimum(limit, lens[:, None])[:, None, None, :, None]
    scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum("bhgnk,hbkd->bhgnd", weights, values) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    # back to the rows of the batch
    row = torch.arange(n, device=q.device, dtype=torch.int32)
    b = torch.searchsorted(cu[1:], row, right=True)
    j = (row - cu[b]).long()
    out = out.permute(0, 3, 1, 2, 4).reshape(len(lens), len(i), hq, dim)
    lse = lse.permute(0, 3, 1, 2).reshape(len(lens), len(i), hq)
    return out[b, j].to(q.dtype), lse[b, j]


def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["freq"].double()
    cos, sin = (f(angle).float()[:, None] * s["factor"] for f in (torch.cos, torch.sin))
    q, k = _rotate(s["q"], s["qw"], cos, sin, s), _rotate(s["k"], s["kw"], cos, sin, s)
    s["kp"][:, s["targets"]] = k.transpose(0, 1)
    s["vp"][:, s["targets"]] = s["v"].transpose(0, 1)
    return q, s["kp"], s["vp"]


def _rotate(x, weight, cos, sin, s):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * weight.float()
    rot = 2 * cos.shape[-1]
    if s["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_beam(s):
    # in 64 bits: candidates of different beams may lie closer than 32 bits tell apart
    x = s["logits"].double()
    r, w, v = x.shape
    top = x.amax(-1, keepdim=True)
    x = x - (top + (x - top).exp().sum(-1, keepdim=True).log()) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        token = torch.arange(v, device=x.device)
        ended = torch.where(token == s["end"], s["scores"].double()[..., None], -math.inf)
        x = torch.where(s["finished"][..., None], ended, x)
    best, index = x.view(r, w * v).sort(dim=1, descending=True, stable=True)
    best, index = best[:, :s["k"]], index[:, :s["k"]]
    parents, tokens = index // v, index % v
    states = s["states"].gather(1, parents[:, :w, None].expand(-1, -1, s["states"].shape[2]))
    return best.float(), parents, tokens, states


# ---- what a pass cannot do without ------------------------------------------
def work(case):
    if case["op"] == "chunk":
        fresh, total = _case_lengths(case)
        hq, hk, dim, page = case["hq"], case["hk"], case["dim"], case["page"]
        pairs = sum(_visible(n, t, case["causal"]) for n, t in zip(fresh, total))
        rows = sum(fresh)
        return {"bytes": rows * hq * (dim * 4 + 4) + sum(total) * hk * dim * 4 + sum(-(-t // page) for t in total) * 4,
                "flops": 4.0 * dim * hq * pairs}
    if case["op"] == "rotary":
        values = case["tokens"] * (case["hq"] + 2 * case["hk"]) * case["dim"]
        return {"bytes": values * 4 + case["tokens"] * 16, "flops": 6.0 * values}
    r, w, v = case["requests"], case["beams"], case["vocab"]
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": r * w * v * size + r * w * case["length"] * 8 + r * case["k"] * 20, "flops": 3.0 * r * w * v}


def _visible(n, t, causal):
    if not causal:
        return n * t
    low = max(0, t - n)                                    # keys before the chunk
    rows = min(n, t)                                       # rows that see at least one of the chunk's keys
    return rows * low + rows * (rows + 1) // 2


# ---- the definitions in 64 bits ---------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"chunk": _exact_chunk, "rotary": _exact_rotary, "beam": _exact_beam}[case["op"]](s)


def _exact_chunk(s):
    q, cu, lens, page = s["q"], s["cu"].tolist(), s["lens"].tolist(), s["page"]
    n, hq, dim = q.shape
    hk = s["kp"].shape[0]
    out = torch.zeros((n, hq, dim), dtype=torch.float64, device=q.device)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
    for b, total in enumerate(lens):
        rows = slice(cu[b], cu[b + 1])
        count = cu[b + 1] - cu[b]
        if not count or not total:
            continue
        places = [int(p) * page + o for p in s["table"][b].tolist() if p >= 0 for o in range(page)][:total]
        places = torch.tensor(places, device=q.device)
        for h in range(hq):
            k = s["kp"][h * hk // hq].double()[places]
            v = s["vp"][h * hk // hq].double()[places]
            scores = q[rows, h].double() @ k.T * dim ** -0.5
            if s["causal"]:
                later = torch.ones((count, total), dtype=torch.bool, device=q.device).triu(total - count + 1)
                scores = scores.masked_fill(later, -math.inf)
            lse[rows, h] = torch.logsumexp(scores, -1)
            out[rows, h] = torch.nan_to_num(torch.softmax(scores, -1)) @ v
    return out, lse


def _exact_rotary(s):
    rot = 2 * s["freq"].numel()
    unit = torch.polar(torch.full((1,), s["factor"], dtype=torch.float64, device=s["freq"].device),
                       s["positions"].double()[:, None] * s["freq"].double())

    def turn(x, weight):
        y = x.double()
        if weight is not None:
            y = y / (y.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * weight.double()
        part = y[..., :rot]
        pairs = part.unflatten(-1, (-1, 2)) if s["interleaved"] else part.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit[:, None])
        z = z if s["interleaved"] else z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), y[..., rot:]), -1)

    kp, vp = s["kp"].double(), s["vp"].double()
    kp[:, s["targets"]] = turn(s["k"], s["kw"]).transpose(0, 1)
    vp[:, s["targets"]] = s["v"].double().transpose(0, 1)
    return turn(s["q"], s["qw"]), kp, vp


def _exact_beam(s):
    logits = s["logits"].double()
    r, w, v = logits.shape
    best = torch.empty((r, s["k"]), dtype=torch.float64, device=logits.device)
    for i in range(r):
        table = torch.log_softmax(logits[i], -1) + s["scores"][i].double()[:, None]
        if s["finished"] is not None:
            for j in s["finished"][i].nonzero().flatten().tolist():
                table[j] = -math.inf
                table[j, s["end"]] = s["scores"][i, j].double()
        best[i] = table.flatten().topk(s["k"])[0]
    return best, None, None, None
