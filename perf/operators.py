"""Workloads of the sliding-window and quantised-cache operators, with their plain forms.

Five kinds of call, as a language-model trainer or server makes them:

``train``   forward and backward of causal attention with a sliding window and a few first tokens (sinks) that
            stay visible, grouped-query heads
``chunk``   the same forward without gradients for one chunk of each prompt of a batch against its key/value
            cache; every sequence stands at its own position
``decode``  one (or a few) new tokens per sequence against a 16-bit cache, sliding window and sinks
``write``   keys and values quantised into a 4-bit cache at each sequence's own position, and read back
``cache``   one (or a few) new tokens per sequence against the 4-bit cache, with or without a window

Visibility: the query row r of sequence b stands at position p = start[b] + r and sees key c of its sequence iff
c <= p and (c > p - window or c < sinks).  A row that sees nothing is zero.

4-bit cache: each token's channels in groups of 64; scale = round16((max - min) / 15), zero = min,
code = round_half_even((x - zero) / scale) in 0..15; a byte holds channels 2i (low half) and 2i + 1 (high half);
the value a code stands for is zero + scale * code.
"""

import math
import sys

import torch

own = False

GROUP = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a short fine-tuning batch of a small model: launch latency counts
        dict(name="train_small_d64", kind="train", B=1, Hq=4, Hkv=2, Sq=512, Sk=512, D=64, dtype="fp16", window=128, sinks=4),
        # an odd length and an odd window, heads of 96 channels
        dict(name="train_odd_d96", kind="train", B=2, Hq=8, Hkv=2, Sq=2047, Sk=2047, D=96, dtype="bf16", window=333, sinks=5),
        # the training step of a long-context layer
        dict(name="train_8k", kind="train", B=1, Hq=16, Hkv=4, Sq=8192, Sk=8192, D=128, dtype="bf16", window=1024, sinks=4),
        # prompts processed in chunks: 512 new tokens of each sequence against its cache
        dict(name="chunk_512", kind="chunk", B=4, Hq=32, Hkv=8, Sq=512, Sk=8192, D=128, dtype="bf16", window=4096, sinks=4),
        # one user's next token
        dict(name="decode_one", kind="decode", B=1, Hq=32, Hkv=8, Sq=1, Sk=4096, D=128, dtype="bf16", window=1024, sinks=4),
        # the next token of a full serving batch
        dict(name="decode_batch", kind="decode", B=48, Hq=32, Hkv=8, Sq=1, Sk=16384, D=128, dtype="bf16", window=4096, sinks=4),
        # the new token of every sequence of a batch appended to the cache and read back
        dict(name="write_token", kind="write", B=16, Hkv=8, Sq=1, Sk=4097, D=128, dtype="bf16"),
        # prompts of different lengths written at once and read back for the next chunk
        dict(name="write_prompts", kind="write", B=4, Hkv=8, Sq=8191, Sk=8192, D=128, dtype="bf16"),
        # one user of a small model, an odd cache
        dict(name="cache_one_d64", kind="cache", B=1, Hq=8, Hkv=8, Sq=1, Sk=777, D=64, dtype="fp16", window=0, sinks=0),
        # the next token of a serving batch over the whole cache
        dict(name="cache_8k", kind="cache", B=16, Hq=32, Hkv=8, Sq=1, Sk=8192, D=128, dtype="bf16", window=0, sinks=0),
        # four drafted tokens per sequence, eight query heads per cache head, window and sinks
        dict(name="cache_draft", kind="cache", B=8, Hq=64, Hkv=8, Sq=4, Sk=16384, D=128, dtype="bf16", window=4096, sinks=4),
        # long contexts
        dict(name="cache_32k", kind="cache", B=16, Hq=32, Hkv=8, Sq=1, Sk=32768, D=128, dtype="bf16", window=0, sinks=0),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        at = most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        at["bytes"], at["flops"] = max(at["bytes"], w["bytes"]), max(at["flops"], w["flops"])
    while True:
        kind = rng.choice(("train", "chunk", "decode", "write", "cache"))
        c = dict(kind=kind, dtype=rng.choice(("bf16", "fp16")), D=rng.choice((64, 128)), Hkv=rng.choice((1, 2, 4, 8)))
        if kind == "write":
            c["B"], c["Sq"] = _log(rng, 1, 32), _log(rng, 1, 8192)
            c["Sk"] = c["Sq"] + _log(rng, 1, 4096)
        else:
            c["Hq"] = c["Hkv"] * rng.choice((1, 2, 4, 8))
            c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice((0, 1, 4, 16, 130))
            if kind == "train":
                c["B"], c["Sq"], c["D"] = _log(rng, 1, 4), _log(rng, 64, 8192), rng.choice((64, 80, 96, 128))
                c["Sk"] = c["Sq"]
            elif kind == "chunk":
                c["B"], c["Sq"] = _log(rng, 1, 8), _log(rng, 33, 1024)
                c["Sk"] = c["Sq"] + _log(rng, 64, 8192)
            else:
                c["B"], c["Sq"] = _log(rng, 1, 64), rng.choice((1, 1, 1, 2, 4))
                c["Sk"] = _log(rng, 100, 32768)
                if kind == "cache" and rng.random() < 0.5:
                    c["window"], c["sinks"] = 0, 0
        w = work(c)
        if w["bytes"] <= most[kind]["bytes"] and w["flops"] <= most[kind]["flops"] and _scores(c) <= 1.1e9:
            return c


def _scores(case):
    """Query-key pairs that the plain form holds at once."""
    return 0 if case["kind"] == "write" else case["B"] * case["Hq"] * case["Sq"] * case["Sk"]


def _starts(case):
    """Each sequence's position of its first query (or written) row: the same for every seed, so that the work is known.
    A training sequence starts at 0; otherwise the last sequence fills its cache and the first is about half as long."""
    if case["kind"] == "train":
        return [0] * case["B"]
    last = case["Sk"] - case["Sq"]
    return [last - (last * (case["B"] - 1 - b)) // (2 * case["B"]) for b in range(case["B"])]


def _lengths(case):
    """Rows that each sequence writes: the first sequence all of them, the others fewer (a padded batch of prompts)."""
    return [case["Sq"] - (case["Sq"] * b) // (2 * case["B"]) for b in range(case["B"])]


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, and the keys that some query of a sequence sees."""
    window = case["window"] if case["window"] > 0 else 1 << 40
    pairs = keys = 0
    for start in _starts(case):
        for p in range(start, start + case["Sq"]):
            hi = min(p + 1, case["Sk"])
            lo = min(max(p + 1 - window, 0), hi)
            pairs += hi - lo + min(case["sinks"], lo)
        hi = min(start + case["Sq"], case["Sk"])
        lo = min(max(start + 1 - window, 0), hi)
        keys += hi - lo + min(case["sinks"], lo)
    return pairs, keys


def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    row4 = D // 2 + D // GROUP * 4  # bytes of a quantised row: codes, scales and zeros
    if case["kind"] == "write":
        written, read = sum(_lengths(case)) * Hkv, B * Hkv * case["Sq"]
        # new rows read and quantised, every row of the chunk read back
        return {"bytes": 2.0 * (written * (2 * D + row4) + read * (row4 + 2 * D)), "flops": 2.0 * (written + read) * D * 4}
    pairs, keys = _pairs(case)
    q = B * case["Hq"] * case["Sq"] * D * 2
    flops = 4.0 * D * pairs * case["Hq"]
    if case["kind"] == "train":
        kv = B * Hkv * case["Sk"] * D * 2
        return {"bytes": 5.0 * q + 4.0 * kv + 4.0 * B * case["Hq"] * case["Sq"] * 4, "flops": 3.5 * flops}
    row = row4 if case["kind"] == "cache" else 2 * D
    return {"bytes": 2.0 * q + 2.0 * keys * Hkv * row, "flops": flops}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """q, k, v (and dout) as a model makes them: keys with channels that carry an offset, a few outlier channels."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, Hkv, D = TYPES[case["dtype"]], case["B"], case["Hkv"], case["D"]
    got = {}
    if case["kind"] != "write":
        got["q"] = (1.5 * _randn(gen, B, case["Hq"], case["Sq"], D)).to(dtype)
    rows = case["Sq"] if case["kind"] == "write" else case["Sk"]
    offset = _randn(gen, 1, Hkv, 1, D) * (1 + 3 * (torch.rand((1, Hkv, 1, D), generator=gen, device="cuda") < 0.03))
    got["k"] = torch.cat([(_randn(gen, 1, Hkv, rows, D) + offset).to(dtype) for _ in range(B)])
    got["v"] = torch.cat([_randn(gen, 1, Hkv, rows, D).to(dtype) for _ in range(B)])
    if case["kind"] == "train":
        got["dout"] = _randn(gen, B, case["Hq"], case["Sq"], D).to(dtype)
    return got


def _quantise(x):
    """(codes as bytes, scale and zero pairs in x's type) of x [..., D]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(x.dtype)
    step = scale.float()
    code = torch.where(step > 0, torch.round((g - low) / torch.where(step > 0, step, 1.0)), 0.0).clamp(0, 15)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat((scale, low.to(x.dtype)), -1)


def _values(codes, params):
    """What the codes stand for, in float32."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    pair = params.float()
    return (pair[..., 1:2] + pair[..., 0:1] * code).flatten(-2)


def _cache(k, v):
    """The four tensors of a quantised cache that holds k and v, sequence by sequence."""
    rows = [_quantise(torch.stack((k[b], v[b]))) for b in range(k.shape[0])]
    codes, params = torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
    return codes[:, 0].contiguous(), params[:, 0].contiguous(), codes[:, 1].contiguous(), params[:, 1].contiguous()


def prepare(case, seed):
    state = dict(_inputs(case, seed), kind=case["kind"], window=case.get("window", 0), sinks=case.get("sinks", 0))
    state["start"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda")
    if case["kind"] == "train":
        for name in ("q", "k", "v"):
            state[name].requires_grad_(True)
    elif case["kind"] == "write":
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        # what the cache held before
        gen = torch.Generator(device="cuda").manual_seed(seed + 1)
        shape = (1, case["Hkv"], case["Sk"], case["D"])
        before = torch.cat([_randn(gen, *shape).to(TYPES[case["dtype"]]) for _ in range(case["B"])])
        state["cache"] = _cache(before, before.flip(2))
    elif case["kind"] == "cache":
        state["cache"] = _cache(state.pop("k"), state.pop("v"))
    return state


def _visible(start, sq, sk, window, sinks):
    at = start.long()[:, None, None] + torch.arange(sq, device=start.device)[None, :, None]
    key = torch.arange(sk, device=start.device)[None, None, :]
    seen = key <= at
    if window > 0:
        seen = seen & ((key > at - window) | (key < sinks))
    return seen[:, None, None]


def _plain_attention(q, k, v, start, window, sinks, dout=None):
    """q [B, Hq, Sq, D], k and v [B, Hkv, Sk, D] in any type: (out,) or (out, dq, dk, dv) in float32."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    group, scale = Hq // Hkv, D ** -0.5
    qf, kf, vf = q.float().reshape(B, Hkv, group * Sq, D), k.float(), v.float()  # a key head's query rows together
    seen = _visible(start, Sq, Sk, window, sinks)
    scores = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale)
    scores.view(B, Hkv, group, Sq, Sk).masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    out = torch.matmul(p, vf)
    if dout is None:
        return (out.view(B, Hq, Sq, D),)
    gf = dout.float().reshape(B, Hkv, group * Sq, D)
    dv = torch.matmul(p.transpose(-1, -2), gf)
    ds = torch.matmul(gf, vf.transpose(-1, -2)).sub_((gf * out).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, kf).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), qf).mul_(scale)
    return out.view(B, Hq, Sq, D), dq.view(B, Hq, Sq, D), dk, dv


def _run_plain(s):
    if s["kind"] == "write":
        k, v, start = s["k"], s["v"], s["start"].long()
        n = k.shape[2]
        row = torch.arange(n, device=k.device)
        at = start[:, None] + row[None]
        b, r = torch.nonzero(row[None] < s["lengths"][:, None], as_tuple=True)
        found = []
        for x, codes, params in ((k, s["cache"][0], s["cache"][1]), (v, s["cache"][2], s["cache"][3])):
            new_codes, new_params = _quantise(x)
            codes[b, :, at[b, r]] = new_codes[b, :, r]
            params[b, :, at[b, r]] = new_params[b, :, r]
            batch = torch.arange(k.shape[0], device=k.device)[:, None]
            held = _values(codes[batch, :, at], params[batch, :, at])  # [B, n, heads, D]
            found.append(held.transpose(1, 2).to(x.dtype).contiguous())
        return tuple(found)
    q = s["q"]
    if s["kind"] == "cache":
        kc, kp, vc, vp = s["cache"]
        k, v = _values(kc, kp), _values(vc, vp)
    else:
        k, v = s["k"], s["v"]
    with torch.no_grad():
        got = _plain_attention(q, k, v, s["start"], s["window"], s["sinks"], s.get("dout"))
    return tuple(t.to(q.dtype) for t in got)


def run(s):
    if not own:
        return _run_plain(s)
    if "kohakufa-cute_b200" not in sys.path:
        sys.path.insert(0, "kohakufa-cute_b200")
    import kohakufa_cute as kfa

    if s["kind"] == "write":
        cache = kfa.QuantizedCache(*s["cache"])
        kfa.quantized_cache_write(cache, s["k"], s["v"], start=s["start"], lengths=s["lengths"])
        return kfa.quantized_cache_read(cache, start=s["start"], length=s["k"].shape[2])
    if s["kind"] == "cache":
        return (kfa.quantized_cache_attention(s["q"], kfa.QuantizedCache(*s["cache"]), query_start=s["start"],
                                              window=s["window"] or None, sinks=s["sinks"]),)
    if s["kind"] == "train":
        out = kfa.sliding_window_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"])
        return (out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    with torch.no_grad():
        return (kfa.sliding_window_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"],
                                             query_start=s["start"]),)


def _stand_for(x):
    """In 64 bits: the values that x [rows, D] stands for once it is held in 4 bits."""
    groups = x.double().reshape(x.shape[0], -1, GROUP)
    low = groups.min(dim=2, keepdim=True).values
    step = ((groups.max(dim=2, keepdim=True).values - low) / 15.0).to(x.dtype).double()
    count = torch.where(step == 0, torch.zeros_like(groups), torch.round((groups - low) / step.masked_fill(step == 0, 1.0)))
    return (low + step * count.clamp(max=15.0)).reshape(x.shape)


def _exact_head(q, k, v, start, case, dout):
    """One sequence and one key/value head in 64 bits: q, dout [heads, Sq, D], k, v [Sk, D]."""
    scale = 1.0 / math.sqrt(case["D"])
    where = start + torch.arange(case["Sq"], device="cuda").view(-1, 1)
    col = torch.arange(case["Sk"], device="cuda").view(1, -1)
    hidden = col > where
    if case["window"] > 0:
        hidden = hidden | ((where - col >= case["window"]) & (col >= case["sinks"]))
    blind = hidden.all(dim=1, keepdim=True)
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for h in range(q.shape[0]):
        logits = (q[h] * scale) @ k.T
        logits[hidden] = -math.inf
        prob = torch.softmax(logits.masked_fill(blind, 0.0), dim=1).masked_fill(blind, 0.0)
        out[h] = prob @ v
        if dout is not None:
            dv += prob.T @ dout[h]
            grad = dout[h] @ v.T
            grad = prob * (grad - (grad * prob).sum(dim=1, keepdim=True))
            dq[h] = grad @ k * scale
            dk += grad.T @ q[h] * scale
    return out, dq, dk, dv


def exact(case, seed):
    s = _inputs(case, seed)
    B, Hkv, D, starts = case["B"], case["Hkv"], case["D"], _starts(case)
    if case["kind"] == "write":
        gen = torch.Generator(device="cuda").manual_seed(seed + 1)
        found = [torch.empty(B, Hkv, case["Sq"], D, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b in range(B):
            before = _randn(gen, 1, Hkv, case["Sk"], D).to(TYPES[case["dtype"]])[0]
            for out, new, old in zip(found, (s["k"][b], s["v"][b]), (before, before.flip(1))):
                n = _lengths(case)[b]
                rows = old[:, starts[b]: starts[b] + case["Sq"]].clone()
                rows[:, :n] = new[:, :n]
                out[b] = _stand_for(rows.reshape(-1, D)).reshape(Hkv, case["Sq"], D)
        return tuple(found)
    group = case["Hq"] // Hkv
    grads = case["kind"] == "train"
    out = torch.empty(B, case["Hq"], case["Sq"], D, dtype=torch.float64, device="cuda")
    dq = torch.empty_like(out) if grads else None
    dk = torch.empty(B, Hkv, case["Sk"], D, dtype=torch.float64, device="cuda") if grads else None
    dv = torch.empty_like(dk) if grads else None
    for b in range(B):
        for h in range(Hkv):
            heads = slice(h * group, (h + 1) * group)
            k, v = s["k"][b, h], s["v"][b, h]
            k, v = (_stand_for(k), _stand_for(v)) if case["kind"] == "cache" else (k.double(), v.double())
            o, q_, k_, v_ = _exact_head(s["q"][b, heads].double(), k, v, starts[b], case,
                                        s["dout"][b, heads].double() if grads else None)
            out[b, heads] = o
            if grads:
                dq[b, heads], dk[b, h], dv[b, h] = q_, k_, v_
    return (out, dq, dk, dv) if grads else (out,)
