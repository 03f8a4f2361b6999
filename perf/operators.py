"""Operators of the decoder's serving path, as cases that can be timed and compared: attention over packed prompts, the append of
finished q, k and v to a cache held in 4 bits (and the values that it stands for), single-token attention over such a cache, and log
probabilities of given tokens.

`own` chooses between the framework's kernels (`rptc_b200.ops`) and the same formulas in elementary torch operations.  Head layouts
are those of the Llama-2-7B and 70B shapes of this repository's benchmark; heads are 128 wide there, the prompt attention takes 64 too.

The 4-bit cache is four tensors: codes of k, uint8 [rows, kv_heads, max_pos, 64]; (scale, minimum) of its groups of 32 values,
fp16 [rows, kv_heads, max_pos, 4, 2]; the same for v.  A value is minimum + code * scale.  Value e of group g is nibble e % 4 of
the 16-bit word 4 * (e // 4) + g of its position's 64 bytes.
"""
import math
import os
import sys

import torch

own = False

D = 128
SEVEN, SEVENTY = dict(heads=32, kv_heads=32), dict(heads=64, kv_heads=8)


def listed():
    return [
        # a short question: the smallest prompt, where launches and latency count
        dict(name="prompt_24", kind="prompt", lengths="24", past="0", d=128, dtype="float16", **SEVEN),
        # the prompt of the benchmark's prefill
        dict(name="prompt_2048", kind="prompt", lengths="2048", past="0", d=128, dtype="float16", **SEVEN),
        # a server's batch: prompts of all lengths, some of which continue a conversation, grouped heads
        dict(name="prompt_ragged", kind="prompt", lengths="1021,1,333,64,517,7,129,255,40,777,18,2,450,91,200,65",
             past="0,300,0,0,1000,2047,0,0,513,0,60,0,0,129,0,999", d=128, dtype="bfloat16", **SEVENTY),
        # one long document
        dict(name="prompt_8192", kind="prompt", lengths="8192", past="0", d=128, dtype="float16", **SEVENTY),
        # a decode step's new token in each of sixteen sequences: accumulators of the fused qkv layer in, q out, k and v cached
        dict(name="append_16", kind="append", rows=16, tokens=1, past=130, source="float32", **SEVEN),
        # a prompt's tokens, finished and cached
        dict(name="append_2048", kind="append", rows=1, tokens=2048, past=0, source="float16", **SEVEN),
        # a token of one sequence at an ordinary context
        dict(name="decode_200", kind="decode", rows=1, shortest=200, longest=200, max_pos=512, **SEVEN),
        # one sequence over a whole book: the context is all there is to split
        dict(name="decode_131072", kind="decode", rows=1, shortest=131072, longest=131072, max_pos=131072, **SEVENTY),
        # a full batch of different contexts
        dict(name="decode_batch", kind="decode", rows=32, shortest=500, longest=32768, max_pos=32768, **SEVENTY),
        # the token just chosen and its alternatives
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=32000, top=5, dtype="float16", masked=0.0),
        # a scored prompt, with the alternatives that an interface shows
        dict(name="logprobs_2048", kind="logprobs", rows=2048, vocab=32000, top=20, dtype="float16", masked=0.0),
        # a perplexity run over a large vocabulary of odd size, part of it forbidden, in 32 bits
        dict(name="logprobs_128001", kind="logprobs", rows=1500, vocab=128001, top=0, dtype="float32", masked=0.3),
    ]


# ---- drawn cases ---------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _heads(rng):
    return rng.choice([SEVEN, SEVENTY, dict(heads=32, kv_heads=8), dict(heads=16, kv_heads=2), dict(heads=8, kv_heads=1), dict(heads=12, kv_heads=4)])


def draw(rng):
    kind = rng.choice(["prompt", "append", "decode", "logprobs"])
    heads = _heads(rng)
    if kind == "prompt":
        most = 8192 * 8192 * 64 // heads["heads"]
        while True:
            count, longest = _log(rng, 1, 48), _log(rng, 1, 8192)
            lengths = [rng.randint(max(1, longest // 8), longest) for _ in range(count)]
            past = [_log(rng, 1, 4000) if rng.random() < 0.5 else 0 for _ in range(count)] if rng.random() < 0.4 else [0] * count
            widest = max(lengths) * max(a + b for a, b in zip(lengths, past)) * count
            if sum(lengths) <= 16384 and widest <= most // 2:
                return dict(kind=kind, lengths=",".join(map(str, lengths)), past=",".join(map(str, past)), d=rng.choice([128, 128, 128, 64]),
                            dtype=rng.choice(["float16", "bfloat16"]), **heads)
    if kind == "append":
        rows = _log(rng, 1, 64)
        if rng.random() < 0.5:
            return dict(kind=kind, rows=rows, tokens=1, past=_log(rng, 1, 2048), source="float32", **heads)
        return dict(kind=kind, rows=rows, tokens=_log(rng, 1, max(1, 4096 // rows)), past=rng.choice([0, 0, _log(rng, 1, 500)]), source="float16", **heads)
    if kind == "decode":
        rows, longest = _log(rng, 1, 64), _log(rng, 1, 131072)
        longest = min(longest, 32 * 32768 * 8 // (rows * heads["kv_heads"]))
        return dict(kind=kind, rows=rows, shortest=rng.randint(1, longest), longest=longest, max_pos=longest + rng.randint(0, 100), **heads)
    dtype, vocab = rng.choice(["float16", "bfloat16", "float32"]), _log(rng, 1000, 160000)
    rows = _log(rng, 1, min(4096, 1500 * 128001 // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20]), dtype=dtype, masked=rng.choice([0.0, 0.0, 0.5]))


# ---- what a user's program has in hand -------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _numbers(text):
    return [int(t) for t in text.split(",")]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return _int32([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _angles(positions):
    """cosines and sines of the rotary angles, made in 64 bits"""
    inv = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack((a.cos(), a.sin()), dim=-1).float()


def _scales(g, *shape):
    """groups as a quantiser of values near N(0, 1) leaves them"""
    scale = 0.2 + 0.2 * torch.rand(shape, generator=g, device="cuda")
    low = -7.5 * scale + 0.3 * torch.randn(shape, generator=g, device="cuda")
    return torch.stack((scale, low), dim=-1).half()


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    s = {"case": case}
    if kind == "prompt":
        lengths, past, dtype = _numbers(case["lengths"]), _numbers(case["past"]), getattr(torch, case["dtype"])
        tokens, keys = sum(lengths), sum(lengths) + sum(past)
        s["q"] = torch.randn(tokens, case["heads"], case["d"], generator=g, device="cuda").to(dtype)
        s["k"] = torch.randn(keys, case["kv_heads"], case["d"], generator=g, device="cuda").to(dtype)
        s["v"] = torch.randn(keys, case["kv_heads"], case["d"], generator=g, device="cuda").to(dtype)
        s["starts"] = _starts(lengths)
        s["kv_len"] = _int32([a + b for a, b in zip(lengths, past)])
        s["kv_first"] = _starts([a + b for a, b in zip(lengths, past)])[:-1].contiguous()
        s["longest"], s["widest"] = max(lengths), max(a + b for a, b in zip(lengths, past))
    elif kind == "append":
        rows, tokens, past, hq, hkv = (case[n] for n in ("rows", "tokens", "past", "heads", "kv_heads"))
        s["x"] = (8 * torch.randn(rows * tokens, (hq + 2 * hkv) * D, generator=g, device="cuda")).to(getattr(torch, case["source"]))
        s["signs"] = (torch.randint(0, 2, ((hq + 2 * hkv) * D,), generator=g, device="cuda") * 2 - 1).half()
        s["scale"] = 0.125
        s["slots"] = torch.arange(rows, dtype=torch.int32, device="cuda").repeat_interleave(tokens)
        s["pos"] = torch.arange(past, past + tokens, dtype=torch.int32, device="cuda").repeat(rows)
        s["angles"] = _angles(past + tokens)
        shape = (rows, hkv, past + tokens)
        s["cache"] = tuple(torch.zeros(shape + t, dtype=dt, device="cuda") for t, dt in (((64,), torch.uint8), ((4, 2), torch.float16)) * 2)
        s["count"] = torch.full((rows,), past + tokens, dtype=torch.int32, device="cuda")
    elif kind == "decode":
        rows, hq, hkv, most = (case[n] for n in ("rows", "heads", "kv_heads", "max_pos"))
        s["q"] = torch.randn(rows, hq * D, generator=g, device="cuda").half()
        codes = [torch.randint(0, 256, (rows, hkv, most, 64), dtype=torch.uint8, generator=g, device="cuda") for _ in range(2)]
        scales = [_scales(g, rows, hkv, most, 4) for _ in range(2)]
        s["cache"] = (codes[0], scales[0], codes[1], scales[1])
        s["pos"] = _int32([_context(case, r) - 1 for r in range(rows)])
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
        s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        if case["masked"]:
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
            x.scatter_(1, s["targets"][:, None], 1.0)
        s["logits"] = x.to(getattr(torch, case["dtype"]))
    return s


def _context(case, row):
    """contexts spread evenly from the shortest to the longest"""
    return case["longest"] - (case["longest"] - case["shortest"]) * row // max(1, case["rows"] - 1)


# ---- one pass --------------------------------------------------------------------------------------------------------
_ops = None


def _load():
    """the framework's front end, from the package folder of the tree this runs in"""
    global _ops
    sys.path.insert(0, os.path.abspath("let-it-slide_b200"))
    from rptc_b200 import ops
    _ops = ops


def run(s):
    c = s["case"]
    if own and _ops is None:
        _load()
    if c["kind"] == "prompt":
        if own:
            if s["k"].shape[0] == s["q"].shape[0]:
                return _ops.attn_prompt(s["q"], s["k"], s["v"], s["starts"])
            return _ops.attn_prompt(s["q"], s["k"], s["v"], s["starts"], s["kv_first"], s["kv_len"])
        return _plain_prompt(s)
    if c["kind"] == "append":
        if own:
            out = _ops.qkv_append(s["x"], s["pos"], s["angles"], s["cache"], c["heads"], c["kv_heads"], slots=s["slots"],
                                    signs_out=s["signs"], scale=s["scale"], transform=True)
            k, v = _ops.kv4_values(s["cache"], s["count"])
            return {"qkv": out, "k": k, "v": v}
        return _plain_append(s)
    if c["kind"] == "decode":
        return _ops.attn_decode_kv4(s["q"], s["pos"], s["cache"], c["heads"]) if own else _plain_decode(s)
    if own:
        logprob, entropy, top, ids = _ops.token_logprobs(s["logits"], s["targets"], c["top"])
        return {"logprob": logprob, "entropy": entropy, "top": top, "ids": ids}
    return _plain_logprobs(s)


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plain_prompt(s):
    """Every prompt padded to the longest; a query sees the keys up to its own place behind the past."""
    q, k, v, starts, kv_len, L, W = s["q"], s["k"], s["v"], s["starts"].long(), s["kv_len"].long(), s["longest"], s["widest"]
    heads, kv_heads, d = q.shape[1], k.shape[1], q.shape[2]
    length = starts[1:] - starts[:-1]
    i, j = torch.arange(L, device="cuda"), torch.arange(W, device="cuda")
    qi = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    kj = (s["kv_first"].long()[:, None] + j).clamp(max=k.shape[0] - 1)
    qp = q.float()[qi].unflatten(2, (kv_heads, heads // kv_heads)).permute(0, 2, 3, 1, 4).flatten(2, 3)      # [n, kv, group * L, d]
    kp, vp = k.float()[kj].transpose(1, 2), v.float()[kj].transpose(1, 2)                                  # [n, kv, W, d]
    p = (qp @ kp.transpose(2, 3)).mul_(d ** -0.5).unflatten(2, (heads // kv_heads, L))
    seen = j <= (kv_len - length)[:, None, None] + i[:, None]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ vp).unflatten(2, (heads // kv_heads, L)).div_(total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                                             # [n, L, heads, d]
    return o[i < length[:, None]].to(q.dtype)


def _sums_and_differences(x, h):
    x = x.unflatten(-1, (D // (2 * h), 2, h))
    a, b = x[..., 0, :], x[..., 1, :]
    return torch.stack((a + b, a - b), dim=-2).flatten(-3)


def _hadamard(x):
    """unnormalised, in blocks of 128"""
    y = _sums_and_differences(x.unflatten(-1, (-1, D)), 1)
    y = _sums_and_differences(_sums_and_differences(_sums_and_differences(y, 2), 4), 8)
    return _sums_and_differences(_sums_and_differences(_sums_and_differences(y, 16), 32), 64)


def _quantised(x):
    """[tokens, heads, 128] -> codes [tokens, heads, 4, 32] and (scale, minimum), one rounding each"""
    g = x.unflatten(-1, (4, 32))
    low, high = g.amin(-1), g.amax(-1)
    scale = ((high - low) / 15).half()
    step = scale.float()[..., None]
    codes = torch.where(step > 0, torch.round((g - low[..., None]) / step), 0.0).clamp(0, 15)
    return codes.to(torch.int32), torch.stack((scale, low.half()), dim=-1)


def _packed(codes):
    """codes [..., 4, 32] -> bytes [..., 64]"""
    n = codes.unflatten(-1, (8, 2, 2)).movedim(-4, -3)              # [..., e // 4, group, pair, nibble]
    return (n[..., 0] + 16 * n[..., 1]).flatten(-3).to(torch.uint8)


def _values(codes, scales):
    """bytes [..., 64], fp16 [..., 4, 2] -> fp32 [..., 128]"""
    b = codes.unflatten(-1, (8, 4, 2))
    n = torch.stack((b & 15, b >> 4), dim=-1).movedim(-3, -4).flatten(-3)      # [..., group, 32]
    return (scales[..., 1:].float() + n.float() * scales[..., :1].float()).flatten(-2)


def _plain_append(s):
    hq, hkv, cache = s["case"]["heads"], s["case"]["kv_heads"], s["cache"]
    slots, pos = s["slots"].long(), s["pos"].long()
    y = _hadamard(s["x"].float()) * (s["scale"] * D ** -0.5)
    y = (y * s["signs"].float().unflatten(0, (-1, D))).half().float()
    cs, sn = s["angles"][pos][:, None].unbind(-1)
    a, b = y[:, : hq + hkv, : D // 2], y[:, : hq + hkv, D // 2:]
    y[:, : hq + hkv] = torch.cat((a * cs - b * sn, b * cs + a * sn), dim=-1)
    y = y.half()
    kc, ks = _quantised(y[:, hq: hq + hkv].float())
    vc, vs = _quantised(y[:, hq + hkv:].float())
    cache[0][slots, :, pos], cache[1][slots, :, pos] = _packed(kc), ks
    cache[2][slots, :, pos], cache[3][slots, :, pos] = _packed(vc), vs
    k, v = _values(cache[0], cache[1]), _values(cache[2], cache[3])
    return {"qkv": y.flatten(1), "k": k.transpose(1, 2).half().contiguous(), "v": v.transpose(1, 2).half().contiguous()}


def _plain_decode(s):
    hq, cache = s["case"]["heads"], s["cache"]
    rows, hkv, most = cache[0].shape[:3]
    q = s["q"].float().view(rows, hkv, hq // hkv, D)
    p = (q @ _values(cache[0], cache[1]).transpose(2, 3)).mul_(D ** -0.5)
    p.masked_fill_((torch.arange(most, device="cuda") > s["pos"][:, None])[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    return ((p @ _values(cache[2], cache[3])) / p.sum(-1, keepdim=True)).reshape(rows, hq * D).half()


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    vocab = x.shape[1]
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = y.exp()
    z = e.sum(-1, keepdim=True)
    log_z = z.log()
    entropy = (log_z - e.mul_(y.masked_fill(y == -math.inf, 0.0)).sum(-1, keepdim=True) / z)[:, 0]
    logprob = (y.gather(1, s["targets"][:, None]) - log_z)[:, 0]
    # the largest first, equal ones by their index: one whole number per entry (its bits in the order of the numbers, then the index)
    n = x.view(torch.int32).long()
    key = torch.where(n < 0, -(n & 0x7FFFFFFF), n) * 2 ** 20 + (vocab - 1 - torch.arange(vocab, device="cuda"))
    ids = vocab - 1 - (key.topk(top, dim=-1).values & (2 ** 20 - 1))
    return {"logprob": logprob, "entropy": entropy, "top": y.gather(1, ids) - log_z, "ids": ids}


# ---- bytes and operations that a pass cannot do without --------------------------------------------------------------
def work(case):
    kind, hq, hkv = case["kind"], case.get("heads"), case.get("kv_heads")
    if kind == "prompt":
        lengths, past, d = _numbers(case["lengths"]), _numbers(case["past"]), case["d"]
        seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(lengths, past))
        return {"bytes": 4 * d * (hq * sum(lengths) + hkv * (sum(lengths) + sum(past))), "flops": 4 * d * hq * seen}
    if kind == "append":
        tokens, whole = case["rows"] * case["tokens"], case["rows"] * (case["tokens"] + case["past"])
        size = 4 if case["source"] == "float32" else 2
        append = tokens * ((size + 2) * (hq + 2 * hkv) * D + 160 * hkv + 8) + (case["past"] + case["tokens"]) * 4 * D
        return {"bytes": append + whole * hkv * (160 + 4 * D), "flops": tokens * (hq + 2 * hkv) * D * 12}
    if kind == "decode":
        contexts = sum(_context(case, r) for r in range(case["rows"]))
        return {"bytes": contexts * hkv * 160 + 4 * case["rows"] * hq * D, "flops": 4 * contexts * hq * D}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "prompt":
        return _exact_prompt(s)
    if case["kind"] == "append":
        return _exact_append(s)
    return _exact_decode(s) if case["kind"] == "decode" else _exact_logprobs(s)


def _exact_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    starts, first, count = s["starts"].tolist(), s["kv_first"].tolist(), s["kv_len"].tolist()
    group = q.shape[1] // k.shape[1]
    for n in range(len(count)):
        a, b = starts[n], starts[n + 1]
        hidden = torch.ones(b - a, count[n], dtype=torch.bool, device="cuda").triu(count[n] - (b - a) + 1)
        for h in range(q.shape[1]):
            keys, values = (t[first[n]: first[n] + count[n], h // group].double() for t in (k, v))
            x = (q[a:b, h].double() @ keys.t()) / math.sqrt(q.shape[2])
            out[a:b, h] = x.masked_fill(hidden, -math.inf).softmax(-1) @ values
    return out


def _sylvester():
    h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for _ in range(7):
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h


def _exact_append(s):
    hq, hkv, past = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["past"]
    x = s["x"].double().view(len(s["pos"]), hq + 2 * hkv, D)
    y = (x @ _sylvester() * s["scale"] / math.sqrt(D) * s["signs"].double().view(hq + 2 * hkv, D)).half().double()
    cs, sn = (s["angles"][s["pos"].long()][:, None, :, n].double() for n in (0, 1))
    turned = y.clone()
    for h in range(hq + hkv):
        a, b = y[:, h: h + 1, :64], y[:, h: h + 1, 64:]
        turned[:, h: h + 1, :64], turned[:, h: h + 1, 64:] = a * cs - b * sn, a * sn + b * cs
    stored = turned.half().double()
    rows = s["case"]["rows"]
    found = {"qkv": turned.flatten(1)}
    for name, at in (("k", hq), ("v", hq + hkv)):
        g = stored[:, at: at + hkv].reshape(rows, -1, hkv, 4, 32)
        low = g.min(-1, keepdim=True).values
        step = ((g.max(-1, keepdim=True).values - low) / 15).half().double()
        n = torch.where(step > 0, ((g - low) / step).round(), 0.0).clamp(max=15.0)
        whole = torch.zeros(rows, past + g.shape[1], hkv, D, dtype=torch.float64, device="cuda")
        whole[:, past:] = (low + n * step).flatten(3)
        found[name] = whole
    return found


def _exact_decode(s):
    hq, (kc, ks, vc, vs) = s["case"]["heads"], s["cache"]
    rows, hkv = kc.shape[:2]
    out = torch.empty(rows, hq, D, dtype=torch.float64, device="cuda")
    # where value d of a position lies: byte and shift
    e, g = torch.arange(D, device="cuda") % 32, torch.arange(D, device="cuda") // 32
    byte, shift = 2 * (4 * (e // 4) + g) + (e % 4) // 2, 4 * (e % 2)

    def values(codes, scales):
        n = (codes[:, byte].long() >> shift) & 15
        return scales[:, g, 1].double() + n.double() * scales[:, g, 0].double()

    for r in range(rows):
        n = int(s["pos"][r]) + 1
        for h in range(hkv):
            k, v = values(kc[r, h, :n], ks[r, h, :n]), values(vc[r, h, :n], vs[r, h, :n])
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            out[r, heads] = ((s["q"][r].double().view(hq, D)[heads] @ k.t()) / math.sqrt(D)).softmax(-1) @ v
    return out.reshape(rows, hq * D)


def _exact_logprobs(s):
    found = {"logprob": [], "entropy": [], "top": []}
    top, vocab = s["case"]["top"], s["logits"].shape[1]
    for x, t in zip(s["logits"].split(64), s["targets"].split(64)):
        lp = x.double().log_softmax(-1)
        found["logprob"].append(lp.gather(1, t[:, None])[:, 0])
        found["entropy"].append(-(lp.exp() * lp.clamp(min=-1e300)).sum(-1))
        found["top"].append(lp.sort(dim=-1, descending=True).values[:, :top] if top else lp.new_empty(len(t), 0))
    return {**{n: torch.cat(v) for n, v in found.items()}, "ids": None}
