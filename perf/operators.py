"""Measured cases of the score-modified attention operators: the prompt form (tanh-capped scores, a distance bias, a
document mask or a prefix mask), its training step, its single-token form over a key/value cache, and the
single-token form for a batch whose requests share one long prefix.

``run`` computes a case either in plain elementary torch operations (``own = False``) or through this repository's
operators (``own = True``), from the same state that ``prepare`` makes.
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PACKAGE = "custom-tensorflow-compute-capability-sm-120_b200"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(op, dtype, batch, heads, kv_heads, seq_q, seq_k, head_dim, mask, softcap=0.0, alibi=False, documents=0, prefix=0, layout="bhsd",
          **more):
    return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, seq_q=seq_q, seq_k=seq_k, head_dim=head_dim, mask=mask,
                softcap=softcap, alibi=alibi, documents=documents, prefix=prefix, layout=layout, **more)


def listed():
    return [
        # one short prompt: the call's latency counts
        _case("prompt", "bf16", 1, 8, 8, 77, 77, 64, "causal", alibi=True, name="prompt_short"),
        # an ordinary batch of prompts, capped scores, shared key heads, activations as [batch, seq, heads, dim]
        _case("prompt", "bf16", 4, 16, 4, 2048, 2048, 128, "causal", softcap=30.0, layout="bshd", name="prompt_capped"),
        # prefix language model: bidirectional over the prefix, causal behind it; odd lengths
        _case("prompt", "fp16", 3, 16, 16, 1500, 1500, 64, "prefix", prefix=700, name="prompt_prefix_lm"),
        # one long row of packed documents with a distance bias
        _case("prompt", "bf16", 1, 16, 16, 8192, 8192, 128, "documents_causal", alibi=True, documents=6, name="prompt_packed_long"),
        # fine-tuning on short odd sequences
        _case("train", "fp16", 2, 8, 8, 257, 257, 64, "causal", alibi=True, name="train_short"),
        # an ordinary training step: capped scores, shared key heads
        _case("train", "bf16", 2, 16, 4, 2048, 2048, 128, "causal", softcap=30.0, layout="bshd", name="train_capped"),
        # a long packed training row, bidirectional documents, padding at the end
        _case("train", "bf16", 1, 16, 8, 8192, 8192, 128, "documents", documents=5, name="train_packed_long"),
        # one request's next token: latency counts
        _case("decode", "bf16", 1, 32, 8, 1, 700, 128, "lengths", name="decode_one"),
        # every query head with keys of its own, capped scores
        _case("decode", "fp16", 16, 16, 16, 1, 4096, 64, "lengths", softcap=30.0, name="decode_capped"),
        # a serving batch over long ragged caches kept as [batch, seq, heads, dim], with a distance bias
        _case("decode", "bf16", 64, 32, 8, 1, 8192, 128, "lengths", alibi=True, layout="bshd", name="decode_serving"),
        # few requests on a short common instruction
        _case("shared", "bf16", 4, 8, 8, 1, 96, 64, "lengths", prefix=1000, name="shared_few"),
        # a serving batch on a long common document
        _case("shared", "bf16", 128, 32, 8, 1, 640, 128, "lengths", prefix=16384, name="shared_serving"),
    ]


def _pairs(case):
    """Score entries of the case that the mask leaves, over the batch, for one head."""
    b, sq, sk = case["batch"], case["seq_q"], case["seq_k"]
    if case["op"] in ("decode", "shared"):
        return sum(_lengths(case)) + b * case["prefix"]
    first, kind = sk - sq, case["mask"]
    if kind == "full":
        return b * sq * sk
    if kind == "causal":
        return b * sum(max(0, i + first + 1) for i in range(sq))
    if kind == "prefix":
        return sum(sum(min(sk, max(i + first + 1, p)) for i in range(sq)) for p in _prefixes(case))
    n = 0
    for offsets in _offsets(case):
        for lo, hi in zip(offsets, offsets[1:]):
            rows = range(max(lo, first), max(hi, first))
            n += sum(i + 1 - lo for i in rows) if kind == "documents_causal" else len(rows) * (hi - lo)
    return n


def _cost(case):
    return _pairs(case) * case["heads"] * case["head_dim"] * (4 if case["op"] == "train" else 1)


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["prompt", "prompt", "train", "decode", "shared"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    head_dim = rng.choice([64, 128, 128, 80, 96])
    group = rng.choice([1, 1, 2, 4, 8]) if op in ("prompt", "train") else rng.choice([1, 4, 8, 7, 16])
    kv_heads = rng.choice([1, 2, 4, 8])
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    alibi = rng.random() < 0.4
    layout = rng.choice(["bhsd", "bshd"])
    while True:
        if op in ("prompt", "train"):
            mask = rng.choice(["full", "causal", "causal", "prefix", "documents", "documents_causal"])
            seq = spread(1, 8192)
            seq_k = seq if rng.random() < 0.7 else seq + spread(1, 2000)
            case = _case(op, dtype, spread(1, 8), kv_heads * group, kv_heads, seq, seq_k, head_dim, mask, softcap, alibi,
                         rng.randint(1, 12) if mask.startswith("documents") else 0, rng.randint(1, seq_k) if mask == "prefix" else 0, layout)
            fits = case["batch"] * case["heads"] * seq * seq_k <= 1.1e9
        elif op == "decode":
            case = _case(op, dtype, spread(1, 64), kv_heads * group, kv_heads, 1, spread(1, 16384), head_dim, "lengths", softcap, alibi, layout=layout)
            fits = True
        else:
            case = _case(op, dtype, spread(2, 128), kv_heads * group, kv_heads, 1, spread(1, 1000), head_dim, "lengths", softcap, alibi,
                         prefix=spread(100, 16384), layout=layout)
            fits = True
        # the listed cases' cost and, for a cache, their memory bound the drawn ones
        size = case["batch"] * case["kv_heads"] * case["seq_k"] * case["head_dim"]
        if fits and _cost(case) <= most and size <= 64 * 8 * 8192 * 128:
            return case


# ---------------------------------------------------------------------------
# inputs.  Where documents begin, how long prefixes and caches are follows from the case; the values from the seed.
# ---------------------------------------------------------------------------
def _offsets(case):
    """Per batch entry: where its documents begin, and where the last one ends (padding may follow)."""
    r, sk, rows = random.Random("documents %d %d" % (case["documents"], case["seq_k"])), case["seq_k"], []
    for _ in range(case["batch"]):
        end = sk - r.randint(0, sk // 16)
        rows.append([0] + sorted(r.randint(0, end) for _ in range(case["documents"] - 1)) + [end])
    return rows


def _prefixes(case):
    r = random.Random("prefix %d %d" % (case["prefix"], case["seq_k"]))
    return [case["prefix"]] + [r.randint(0, case["prefix"]) for _ in range(case["batch"] - 1)]


def _lengths(case):
    """Tokens in each request's cache: the longest fills it; behind a shared prefix a request may have none of its own yet."""
    r, low = random.Random("lengths %d %d" % (case["batch"], case["seq_k"])), 0 if case["op"] == "shared" else 1
    return [case["seq_k"]] + [r.randint(max(low, case["seq_k"] // 4) if r.random() < 0.9 else low, case["seq_k"]) for _ in range(case["batch"] - 1)]


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def prepare(case, seed):
    dev, dtype = _device(), TYPES[case["dtype"]]
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    b, h, hk, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))

    def normal(heads, seq, factor=1.0):
        shape = (b, heads, seq, d) if case["layout"] == "bhsd" else (b, seq, heads, d)
        t = (torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * factor).to(dtype)
        return t if case["layout"] == "bhsd" else t.transpose(1, 2)

    # a cap matters where scores get large: those models' queries are larger
    wide = 3.0 if case["softcap"] else 1.0
    state = {"case": dict(case), "scale": 1.0 / math.sqrt(d), "softcap": case["softcap"] or None, "slopes": None, "offsets": None, "prefixes": None}
    if case["alibi"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=torch.float32, device=dev)
    if case["op"] in ("decode", "shared"):
        state["q"] = (torch.randn((b, h, d), generator=gen, device=dev) * wide).to(dtype)
        state["k"], state["v"] = normal(hk, sk), normal(hk, sk)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        if case["op"] == "shared":
            state["pk"] = torch.randn((hk, case["prefix"], d), generator=gen, device=dev).to(dtype)
            state["pv"] = torch.randn((hk, case["prefix"], d), generator=gen, device=dev).to(dtype)
        return state
    state["q"], state["k"], state["v"] = normal(h, sq, wide), normal(hk, sk), normal(hk, sk)
    if case["op"] == "train":
        state["do"] = normal(h, sq)
    if case["documents"]:
        state["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device=dev)
    if case["mask"] == "prefix":
        state["prefixes"] = torch.tensor(_prefixes(case), dtype=torch.int32, device=dev)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    if state["case"]["op"] in ("decode", "shared"):
        return _plain_token(state)
    return _plain_sequence(state)


def _own(state):
    ops, op = importlib.import_module(PACKAGE).sm120_ops, state["case"]["op"]
    if op == "decode":
        return ops.score_attention_decode(state["q"], state["k"], state["v"], state["lengths"], scale=state["scale"], softcap=state["softcap"],
                                          alibi_slopes=state["slopes"])
    if op == "shared":
        return ops.shared_prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["lengths"], scale=state["scale"],
                                           softcap=state["softcap"], alibi_slopes=state["slopes"])
    options = dict(scale=state["scale"], causal_mask=state["case"]["mask"] in ("causal", "prefix", "documents_causal"), softcap=state["softcap"],
                   alibi_slopes=state["slopes"], document_offsets=state["offsets"], prefix_lengths=state["prefixes"])
    if op == "prompt":
        return ops.score_attention(state["q"], state["k"], state["v"], **options)
    out, lse = ops.score_attention(state["q"], state["k"], state["v"], return_lse=True, **options)
    dq, dk, dv = ops.score_attention_grad(state["do"], state["q"], state["k"], state["v"], out, lse, **options)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _allowed(state):
    """[batch or 1, seq_q, seq_k] truth values: which keys a query sees."""
    case = state["case"]
    sq, sk = case["seq_q"], case["seq_k"]
    j = torch.arange(sk, device=_device())
    i = torch.arange(sq, device=_device()) + (sk - sq)          # a query's position among the keys
    kind = case["mask"]
    seen = torch.ones((1, sq, sk), dtype=torch.bool, device=_device())
    if kind in ("causal", "documents_causal"):
        seen = (j[None, :] <= i[:, None])[None]
    if kind == "prefix":
        seen = (j[None, :] <= i[:, None])[None] | (j[None, None, :] < state["prefixes"][:, None, None])
    if state["offsets"] is not None:
        last = state["offsets"][:, -1]
        begun_j = (j[None, :, None] >= state["offsets"][:, None, :]).sum(-1)
        begun_i = (i[None, :, None] >= state["offsets"][:, None, :]).sum(-1)
        same = (begun_i[:, :, None] == begun_j[:, None, :]) & (begun_i[:, :, None] > 0) & (j[None, None, :] < last[:, None, None])
        seen = seen & same
    return seen


def _plain_sequence(state):
    case, cap, scale = state["case"], state["softcap"], state["scale"]
    b, h, hk, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))
    g = h // hk
    # heads that share keys side by side as rows of one product: [b, hk, g * sq, d]
    q, k, v = state["q"].float().reshape(b, hk, g * sq, d), state["k"].float(), state["v"].float()
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    t = None
    if cap:
        t = s.div_(cap).tanh_()
        s = t * cap
    s = s.view(b, h, sq, sk)
    if state["slopes"] is not None:
        j = torch.arange(sk, device=s.device)
        i = torch.arange(sq, device=s.device) + (sk - sq)
        s = s - state["slopes"].view(1, h, 1, 1) * (i[:, None] - j[None, :]).abs().float()
    s = s.masked_fill(~_allowed(state)[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p.view(b, hk, g * sq, sk), v).view(b, h, sq, d).to(TYPES[case["dtype"]])
    if case["op"] == "prompt":
        return out
    lse = (m + torch.log(total)).squeeze(-1)
    do = state["do"].float().reshape(b, hk, g * sq, d)
    p = p.view(b, hk, g * sq, sk)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    if cap:
        ds = ds * (1.0 - t * t)
    dq = torch.matmul(ds, k).mul_(scale).view(b, h, sq, d)
    dk = torch.matmul(ds.transpose(-1, -2), q).mul_(scale)
    dtype = TYPES[case["dtype"]]
    return {"out": out, "lse": lse, "dq": dq.to(dtype), "dk": dk.to(dtype), "dv": dv.to(dtype)}


def _plain_token(state):
    case, cap = state["case"], state["softcap"]
    b, h, hk, sk, d, n = (case[k] for k in ("batch", "heads", "kv_heads", "seq_k", "head_dim", "prefix"))
    q = state["q"].float().view(b, hk, h // hk, d)
    s = torch.matmul(q, state["k"].float().transpose(-1, -2)).view(b, h, sk)
    j = torch.arange(sk, device=q.device)
    s = s.masked_fill(j[None, None, :] >= state["lengths"][:, None, None], -math.inf)
    if n:
        rows = q.transpose(0, 1).reshape(hk, b * (h // hk), d)               # the batch's rows against the common keys
        common = torch.matmul(rows, state["pk"].float().transpose(-1, -2)).view(hk, b, h // hk, n).transpose(0, 1).reshape(b, h, n)
        s = torch.cat([common, s], -1)
    s = s * state["scale"]
    if cap:
        s = torch.where(s == -math.inf, s, cap * torch.tanh(s / cap))
    if state["slopes"] is not None:
        position = torch.arange(n + sk, device=q.device)
        away = (state["lengths"][:, None] + (n - 1) - position[None, :]).clamp(min=0).float()
        s = s - state["slopes"][None, :, None] * away[:, None, :]
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., n:].reshape(b, hk, h // hk, sk), state["v"].float()).view(b, h, d)
    if n:
        rows = p[..., :n].view(b, hk, h // hk, n).transpose(0, 1).reshape(hk, b * (h // hk), n)
        out = out + torch.matmul(rows, state["pv"].float()).view(hk, b, h // hk, d).transpose(0, 1).reshape(b, h, d)
    return out.to(TYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b, h, hk, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))
    pairs = _pairs(case)
    if case["op"] in ("decode", "shared"):
        keys = sum(_lengths(case)) + case["prefix"]                            # the common keys are read once
        return {"bytes": 2 * (2 * b * h * d + 2 * keys * hk * d), "flops": 4 * pairs * h * d}
    q, k = b * h * sq * d, b * hk * sk * d
    if case["op"] == "prompt":
        return {"bytes": 2 * (2 * q + 2 * k), "flops": 4 * pairs * h * d}
    # forward: q, k, v in, out and lse out; backward: q, k, v, out, its gradient and lse in, three gradients out
    return {"bytes": 2 * (2 * q + 2 * k) + 2 * (4 * q + 4 * k) + 8 * b * h * sq, "flops": 14 * pairs * h * d}


# ---------------------------------------------------------------------------
# the definition in 64 bits, one head of one batch entry at a time
# ---------------------------------------------------------------------------
def _sees(case, entry, i, j):
    """Does a query at position i (a column of them) see the key at position j (a row of them)?"""
    kind = case["mask"]
    if kind == "full":
        return (i >= -math.inf) & (j >= 0)
    if kind == "causal":
        return j <= i
    if kind == "prefix":
        return (j <= i) | (j < _prefixes(case)[entry])
    offsets = _offsets(case)[entry]
    seen = torch.zeros((i.numel(), j.numel()), dtype=torch.bool, device=i.device)
    for lo, hi in zip(offsets, offsets[1:]):
        seen |= (i >= lo) & (i < hi) & (j >= lo) & (j < hi)
    return seen & (j <= i) if kind == "documents_causal" else seen


def exact(case, seed):
    if _cost(case) > 4e12:
        return None
    state = prepare(case, seed)
    dev, f64 = _device(), torch.float64
    b, h, hk, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))
    cap, scale, g = case["softcap"], 1.0 / math.sqrt(d), h // hk
    slope = [2.0 ** (-8.0 * (x + 1) / h) if case["alibi"] else 0.0 for x in range(h)]
    if case["op"] in ("decode", "shared"):
        out = torch.zeros((b, h, d), dtype=f64, device=dev)
        for e, length in enumerate(_lengths(case)):
            for x in range(hk):
                keys, values = state["k"][e, x, :length].to(f64), state["v"][e, x, :length].to(f64)
                if case["op"] == "shared":
                    keys, values = torch.cat([state["pk"][x].to(f64), keys]), torch.cat([state["pv"][x].to(f64), values])
                score = state["q"][e, x * g:(x + 1) * g].to(f64) @ keys.T * scale
                if cap:
                    score = cap * torch.tanh(score / cap)
                away = torch.arange(keys.shape[0] - 1, -1, -1, device=dev, dtype=f64)
                score = score - torch.tensor(slope[x * g:(x + 1) * g], dtype=f64, device=dev)[:, None] * away[None, :]
                out[e, x * g:(x + 1) * g] = torch.softmax(score, -1) @ values
        return out
    i, j = (torch.arange(sq, device=dev) + (sk - sq))[:, None], torch.arange(sk, device=dev)[None, :]
    out = torch.zeros((b, h, sq, d), dtype=f64, device=dev)
    lse = torch.full((b, h, sq), -math.inf, dtype=f64, device=dev)
    dq, dk, dv = torch.zeros_like(out), torch.zeros((b, hk, sk, d), dtype=f64, device=dev), torch.zeros((b, hk, sk, d), dtype=f64, device=dev)
    for e in range(b):
        seen = _sees(case, e, i, j)
        some = seen.any(-1)
        for x in range(h):
            query, keys, values = state["q"][e, x].to(f64), state["k"][e, x // g].to(f64), state["v"][e, x // g].to(f64)
            curve = torch.tanh(query @ keys.T * (scale / cap)) if cap else None
            score = curve * cap if cap else query @ keys.T * scale
            score = torch.where(seen, score - slope[x] * (i - j).abs().to(f64), -math.inf)
            norm = torch.logsumexp(score, -1)
            weight = torch.where(some[:, None], torch.exp(score - torch.where(some, norm, 0.0)[:, None]), 0.0)
            del score
            out[e, x], lse[e, x] = weight @ values, norm
            if case["op"] == "train":
                grad = state["do"][e, x].to(f64)
                dv[e, x // g] += weight.T @ grad
                back = grad @ values.T
                back = weight * (back - (grad * out[e, x]).sum(-1, keepdim=True))
                if cap:
                    back = back * (1 - curve ** 2)
                dq[e, x] = back @ keys * scale
                dk[e, x // g] += back.T @ query * scale
    return out if case["op"] == "prompt" else {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
