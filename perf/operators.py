"""Cases for the packed-prompt operators: rotary positions with several axes, causal attention over
packed sequences, and log probabilities of given tokens with entropy and top alternatives.

``run`` computes a case in plain torch operations where ``own`` is false, and through the C ABI of
``libclef_b200.so`` where it is true.  Sizes come from the benchmark configurations (16 query / 8 key
heads of 256 and 32 / 16 heads of 128, hidden 3584, vocabulary 256000, prompts of up to 16384 tokens,
lognormal record lengths) and from the tests' small models.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 10000.0
EPS = 1e-6


def listed():
    return [
        # One short text prompt, one axis: nothing but latency.
        dict(name="rope-text-129", op="rope", dtype="bf16", tokens=129, hq=16, hkv=8, d=256, rot=64, axes=1, interleaved=False, far=0),
        # An odd number of image and video tokens with (time, height, width) positions behind a long
        # text, in the 32-bit parity mode: the angles of far positions.
        dict(name="rope-video-fp32", op="rope", dtype="fp32", tokens=4097, hq=16, hkv=8, d=256, rot=64, axes=3, interleaved=False,
             far=1000000),
        # The largest benchmark batch: 16 prompts of 8192 tokens, heads of 128, whole head rotated.
        dict(name="rope-131072", op="rope", dtype="bf16", tokens=131072, hq=32, hkv=16, d=128, rot=128, axes=3, interleaved=True,
             far=4096),
        # Three records of 1, 31 and 64 tokens: the smallest call.
        dict(name="attn-96", op="attention", dtype="bf16", lengths="mean", total=96, mean=32, lens_seed=3, pad=0, hq=16, hkv=8, d=256,
             gate=True, window=0, softcap=0.0, packed=True),
        # A serving batch: lognormal record lengths, median 600, the workspace a little longer than the records.
        dict(name="attn-serving", op="attention", dtype="bf16", lengths="lognormal", total=16384, mean=600, lens_seed=10, pad=100, hq=16,
             hkv=8, d=256, gate=True, window=0, softcap=0.0, packed=True),
        # Hundreds of short records, 1 to 64 tokens each.
        dict(name="attn-short", op="attention", dtype="bf16", lengths="mean", total=16001, mean=32, lens_seed=5, pad=0, hq=32, hkv=16,
             d=128, gate=True, window=0, softcap=0.0, packed=True),
        # The longest prompt the host admits.
        dict(name="attn-long", op="attention", dtype="bf16", lengths="one", total=16384, mean=16384, lens_seed=0, pad=0, hq=16, hkv=8,
             d=256, gate=True, window=0, softcap=0.0, packed=True),
        # 32-bit parity mode with a sliding window and capped scores, plain heads without a gate.
        dict(name="attn-window-fp32", op="attention", dtype="fp32", lengths="mean", total=2047, mean=512, lens_seed=7, pad=3, hq=16,
             hkv=8, d=128, gate=False, window=200, softcap=50.0, packed=False),
        # One row over the whole vocabulary: the next token's alternatives after one prompt.
        dict(name="logp-1-row", op="logprobs", dtype="bf16", rows=1, vocab=256000, dim=3584, targets=1, top=8, softcap=0.0),
        # Eight states with four questions each, four candidate tokens a question, capped logits.
        dict(name="logp-32-rows", op="logprobs", dtype="bf16", rows=32, vocab=256000, dim=3584, targets=4, top=4, softcap=30.0),
        # Every token of a 2048-token prompt scored.
        dict(name="logp-2048-rows", op="logprobs", dtype="bf16", rows=2048, vocab=256000, dim=3584, targets=1, top=8, softcap=0.0),
        # 32-bit parity mode, odd sizes.
        dict(name="logp-fp32", op="logprobs", dtype="fp32", rows=97, vocab=32003, dim=1024, targets=2, top=5, softcap=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attention", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "bf16", "fp32"])
    hq, hkv = rng.choice([(16, 8), (32, 16), (8, 1), (4, 4), (14, 2)])
    if op == "rope":
        d = rng.choice([64, 96, 128, 256])
        rot = rng.choice([d // 4, d // 2, d])
        cap = 131072 * 48 * 128 // (2 if dtype == "fp32" else 1)
        tokens = min(_log(rng, 1, 131072), cap // ((hq + hkv) * d))
        return dict(op=op, dtype=dtype, tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, axes=rng.choice([1, 2, 3]),
                    interleaved=rng.random() < 0.5, far=_log(rng, 1, 2000000))
    if op == "attention":
        total = _log(rng, 1, 16384 if dtype == "bf16" else 2048)
        kind = rng.choice(["mean", "lognormal", "one"])
        d = rng.choice([64, 96, 128, 256])
        if hq * total > 16 * 16384:
            total = 16 * 16384 // hq
        return dict(op=op, dtype=dtype, lengths=kind, total=total, mean=_log(rng, 1, total), lens_seed=rng.randrange(1 << 30),
                    pad=rng.choice([0, 0, 1, 37, 300]), hq=hq, hkv=hkv, d=d, gate=rng.random() < 0.6,
                    window=0 if rng.random() < 0.6 else _log(rng, 1, 4096), softcap=rng.choice([0.0, 0.0, 50.0]),
                    packed=rng.random() < 0.5)
    vocab = _log(rng, 50, 256000 if dtype == "bf16" else 65536)
    dim = 8 * _log(rng, 8, 576)
    rows = _log(rng, 1, 2048 if dtype == "bf16" else 256)
    rows = max(1, min(rows, 2048 * 256000 * 3584 // (vocab * dim)))
    return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, dim=dim, targets=rng.choice([1, 1, 2, 8]), top=rng.choice([0, 1, 4, 8, 20]),
                softcap=rng.choice([0.0, 0.0, 30.0]))


# --------------------------------------------------------------------------- shared by the forms


def sections_of(case):
    """Frequency pairs of each axis: the first axis takes what the others leave."""
    half, axes = case["rot"] // 2, case["axes"]
    rest = half // axes
    return [half - rest * (axes - 1)] + [rest] * (axes - 1)


def axis_of_pairs(case):
    half, axes, sec = case["rot"] // 2, case["axes"], sections_of(case)
    if not case["interleaved"]:
        return [a for a in range(axes) for _ in range(sec[a])]
    return [i % axes if i // axes < sec[i % axes] else 0 for i in range(half)]


def lengths_of(case):
    """The record lengths of a case (they are part of the case, not of its inputs)."""
    total, mean = case["total"], case["mean"]
    if case["lengths"] == "one":
        return [total]
    rng = random.Random(case["lens_seed"])
    got = []
    while sum(got) < total:
        if case["lengths"] == "lognormal":
            n = int(mean * math.exp(rng.gauss(0.0, 0.8)))
            n = max(min(32, mean), min(16384, n))
        else:
            n = rng.randint(0, 2 * mean)  # a record may be empty
        got.append(min(n, total - sum(got)))
    return got


def pairs_of(case):
    """Allowed (query, key) pairs of one head."""
    w, n = case["window"], 0
    for m in lengths_of(case):
        k = min(m, w) if w else m
        n += k * (k + 1) // 2 + (m - k) * k
    return n


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    ty = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).mul_(std).to(ty)

    st = {"case": case}
    if case["op"] == "rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        # the packed projection [q | gate per query head, k, v] a decoder layer makes
        st["proj"] = torch.empty(t, 2 * hq * d + 2 * hkv * d, device=DEVICE, dtype=ty)
        for i in range(0, t, 16384):
            st["proj"][i : i + 16384] = normal(min(16384, t - i), 2 * hq * d + 2 * hkv * d)
        st["q_norm"], st["k_norm"] = normal(d, std=0.1), normal(d, std=0.1)
        steps = torch.arange(t, device=DEVICE, dtype=torch.int32) + case["far"] + torch.randint(0, 64, (1,), generator=g, device=DEVICE,
                                                                                               dtype=torch.int32)
        rows = [steps]
        if case["axes"] > 1:  # frames of 32 x 32 patches: the time axis steps slowly, the others scan the frame
            rows = [steps // 1024 + case["far"], case["far"] + steps // 32 % 32, case["far"] + steps % 32][: case["axes"]]
        st["positions"] = torch.stack(rows).contiguous()
        st["sections"] = (ctypes.c_int32 * case["axes"])(*sections_of(case))
    elif case["op"] == "attention":
        lens = lengths_of(case)
        n, hq, hkv, d = sum(lens), case["hq"], case["hkv"], case["d"]
        t = n + case["pad"]
        if case["packed"]:
            proj = normal(t, 2 * hq * d + 2 * hkv * d)
            heads = proj[:, : 2 * hq * d].view(t, hq, 2 * d)
            st["q"], st["gate"] = heads[..., :d], heads[..., d:]
            st["k"] = proj[:, 2 * hq * d : 2 * hq * d + hkv * d].view(t, hkv, d)
            st["v"] = proj[:, 2 * hq * d + hkv * d :].view(t, hkv, d)
        else:
            proj = None
            st["q"], st["gate"], st["k"], st["v"] = normal(t, hq, d), normal(t, hq, d), normal(t, hkv, d), normal(t, hkv, d)
        for x in (st["q"], st["k"], st["v"], st["gate"]):
            x[n:] = math.nan  # rows behind the last record hold whatever the buffer held
        st["lens"] = lens
        st["cu"] = torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device=DEVICE)
        st["out"] = normal(t, hq, d)
    else:
        n, v, dim = case["rows"], case["vocab"], case["dim"]
        # Values on a grid (1/16 for the normed hidden states, 2^-11 for the head), so that every logit is
        # exact in 32 bits whatever the order of its sum, and equal logits are equal: ids have one answer.
        st["hidden"] = torch.randn(n, dim, generator=g, device=DEVICE).mul_(16).round_().clamp_(-127, 127).div_(16).to(ty)
        st["head"] = torch.empty(v, dim, device=DEVICE, dtype=ty)
        for i in range(0, v, 32768):
            w = torch.randn(min(32768, v - i), dim, generator=g, device=DEVICE)
            st["head"][i : i + 32768] = w.mul_(0.02 * 2048).round_().clamp_(-255, 255).div_(2048).to(ty)
        st["targets"] = torch.randint(0, v, (n, case["targets"]), generator=g, device=DEVICE, dtype=torch.int32)
    return st


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rope":
        values = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * values * size + 4 * case["axes"] * case["tokens"], "flops": 8 * values}
    if case["op"] == "attention":
        n = sum(lengths_of(case))
        heads = 2 * case["hq"] + 2 * case["hkv"] + (case["hq"] if case["gate"] else 0)
        return {"bytes": n * heads * case["d"] * size, "flops": 4 * case["d"] * case["hq"] * pairs_of(case)}
    n, v, d, k, c = case["rows"], case["vocab"], case["dim"], case["top"], case["targets"]
    return {"bytes": (n + v) * d * size + n * (8 * c + 4 + 8 * k), "flops": 2 * n * v * d}


# --------------------------------------------------------------------------- the calls


def run(st):
    case = st["case"]
    if own:
        return {"rope": _own_rope, "attention": _own_attention, "logprobs": _own_logprobs}[case["op"]](st, case)
    return {"rope": _rope, "attention": _attention, "logprobs": _logprobs}[case["op"]](st, case)


def _lib():
    from deciax_b200 import _lib as binding

    return binding, binding.load(), torch.cuda.current_stream().cuda_stream


def _code(binding, case):
    return binding.DTYPE_BF16 if case["dtype"] == "bf16" else binding.DTYPE_F32


def _own_rope(st, case):
    binding, lib, stream = _lib()
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    proj, pos = st["proj"], st["positions"]
    ld, at = proj.stride(0), proj.data_ptr()
    q = torch.empty(t, hq, d, device=DEVICE, dtype=proj.dtype)
    k = torch.empty(t, hkv, d, device=DEVICE, dtype=proj.dtype)
    binding.check(lib.clef_op_qk_norm_rope_axes(
        _code(binding, case), at, ld, 2 * d, at + 2 * hq * d * proj.element_size(), ld, d, q.data_ptr(), hq * d, d, k.data_ptr(), hkv * d,
        d, pos.data_ptr(), pos.stride(0), case["axes"], st["sections"], int(case["interleaved"]), t, hq, hkv, d, case["rot"], THETA,
        st["q_norm"].data_ptr(), st["k_norm"].data_ptr(), EPS, stream))
    return {"q": q, "k": k}


def _own_attention(st, case):
    binding, lib, stream = _lib()
    q, k, v, gate, out = st["q"], st["k"], st["v"], st["gate"], st["out"]
    gated = (gate.data_ptr(), gate.stride(0), gate.stride(1)) if case["gate"] else (None, 0, 0)
    binding.check(lib.clef_op_attention_packed(
        _code(binding, case), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), *gated, out.data_ptr(), out.stride(0), out.stride(1), st["cu"].data_ptr(), st["cu"].numel() - 1, q.shape[0],
        case["hq"], case["hkv"], case["d"], case["softcap"], case["window"], stream))
    return out


def _own_logprobs(st, case):
    binding, lib, stream = _lib()
    hidden, head, targets = st["hidden"], st["head"], st["targets"]
    n, c, k = case["rows"], case["targets"], case["top"]
    logp = torch.empty(n, c, device=DEVICE)
    entropy = torch.empty(n, device=DEVICE)
    ids = torch.empty(n, k, device=DEVICE, dtype=torch.int32)
    top = torch.empty(n, k, device=DEVICE)
    binding.check(lib.clef_op_token_logprobs(
        _code(binding, case), hidden.data_ptr(), hidden.stride(0), head.data_ptr(), head.stride(0), n, case["vocab"], case["dim"],
        case["softcap"], targets.data_ptr(), c, logp.data_ptr(), entropy.data_ptr(), k, ids.data_ptr() if k else None,
        top.data_ptr() if k else None, stream))
    return {"logprobs": logp, "entropy": entropy, "top_ids": ids, "top_logprobs": top}


# --------------------------------------------------------------------------- plain forms


def _rope(st, case):
    t, hq, hkv, d, rot = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"]
    proj = st["proj"]
    freq = THETA ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
    axis = torch.tensor(axis_of_pairs(case), device=DEVICE)
    angle = st["positions"].to(torch.float64).t()[:, axis] * freq  # [t, rot/2]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w.float())
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1).to(proj.dtype)

    return {"q": one(proj[:, : 2 * hq * d].view(t, hq, 2 * d)[..., :d], st["q_norm"]),
            "k": one(proj[:, 2 * hq * d : 2 * hq * d + hkv * d].view(t, hkv, d), st["k_norm"])}


def _attention(st, case):
    lens, hq, hkv, d = st["lens"], case["hq"], case["hkv"], case["d"]
    n, longest, window, cap = sum(lens), max(lens), case["window"], case["softcap"]
    cu = st["cu"].long()
    rows = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(cu, rows, right=True) - 1  # the record of each row
    if len(lens) * longest * longest < n * n:  # padded: one block of scores for each record
        at = cu[:-1, None] + torch.arange(longest, device=DEVICE)
        live = at < cu[1:, None]
    else:  # one block of scores over all rows
        at, live = rows[None], torch.ones(1, n, dtype=torch.bool, device=DEVICE)
    at = torch.where(live, at, 0)
    who = torch.where(live, seq[at], -1)
    # [blocks, key heads, queries a key head, rows, d]
    q = st["q"][at].float().unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4) * d**-0.5
    k = st["k"][at].float().permute(0, 2, 1, 3)[:, :, None]
    v = st["v"][at].float().permute(0, 2, 1, 3)[:, :, None]
    step = torch.arange(at.shape[1], device=DEVICE)
    ago = step[:, None] - step
    seen = (who[:, :, None] == who[:, None]) & (ago >= 0)
    if window:
        seen &= ago < window
    s = q @ k.transpose(-1, -2)
    if cap:
        s = s.div_(cap).tanh_().mul_(cap)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s @ v) / s.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [blocks, rows, heads, d]
    if case["gate"]:
        o = o * torch.sigmoid(st["gate"][at].float())
    out = st["out"]
    out[at[live]] = o[live].to(out.dtype)
    return out


def _logprobs(st, case):
    cap, k = case["softcap"], case["top"]
    raw = st["hidden"].float() @ st["head"].float().t()
    z = cap * torch.tanh(raw / cap) if cap else raw
    lse = torch.logsumexp(z, -1, keepdim=True)
    logp = z - lse
    entropy = -(logp.exp() * logp).sum(-1)
    # equal logits go to the lowest id: order by (logit, -id) in one whole number
    bits = (raw + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 2**32 + (2**32 - 1 - torch.arange(case["vocab"], device=DEVICE))
    ids = torch.topk(key, k, -1).indices if k else key[:, :0]
    return {"logprobs": logp.gather(1, st["targets"].long()), "entropy": entropy, "top_ids": ids.int(), "top_logprobs": logp.gather(1, ids)}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    def exact_rope(st, case):
        t, hq, hkv, d, rot = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"]
        half, axis = rot // 2, axis_of_pairs(case)
        out = {}
        for name, heads, first, stride in (("q", hq, 0, 2 * d), ("k", hkv, 2 * hq * d, d)):
            w = 1.0 + st[name + "_norm"].double()
            y = torch.empty(t, heads, d, device=DEVICE, dtype=torch.float64)
            for a in range(0, t, 32768):
                b = min(t, a + 32768)
                for h in range(heads):
                    x = st["proj"][a:b, first + h * stride : first + h * stride + d].double()
                    x = x / torch.sqrt((x * x).sum(1, keepdim=True) / d + EPS) * w
                    y[a:b, h] = x
                for i in range(half):
                    turn = st["positions"][axis[i], a:b].double() * math.pow(THETA, -2.0 * i / rot)
                    c, s = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
                    u, v = y[a:b, :, i].clone(), y[a:b, :, half + i].clone()
                    y[a:b, :, i] = c * u - s * v
                    y[a:b, :, half + i] = s * u + c * v
            out[name] = y
        return out

    def exact_attention(st, case):
        hq, hkv, d, w, cap = case["hq"], case["hkv"], case["d"], case["window"], case["softcap"]
        out, first = st["out"].double(), 0
        if len(st["lens"]) * hq > 40000:
            return None
        for m in st["lens"]:
            for h in range(hq):
                g = h // (hq // hkv)
                k, v = st["k"][first : first + m, g].double(), st["v"][first : first + m, g].double()
                for a in range(0, m, 4096):
                    b = min(m, a + 4096)
                    s = st["q"][first + a : first + b, h].double() @ k[:b].T / math.sqrt(d)
                    if cap:
                        s = cap * torch.tanh(s / cap)
                    i, j = torch.arange(a, b, device=DEVICE)[:, None], torch.arange(b, device=DEVICE)[None]
                    hidden = (j > i) | (i - j >= w) if w else j > i
                    p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
                    y = p @ v[:b]
                    if case["gate"]:
                        y = y / (1 + torch.exp(-st["gate"][first + a : first + b, h].double()))
                    out[first + a : first + b, h] = y
            first += m
        return out

    def exact_logprobs(st, case):
        n, k, cap = case["rows"], case["top"], case["softcap"]
        out = {"logprobs": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        head = st["head"]
        for a in range(0, n, 256):
            h = st["hidden"][a : a + 256].double()
            z = torch.cat([h @ head[i : i + 16384].double().T for i in range(0, head.shape[0], 16384)], 1)
            if cap:
                z = cap * torch.tanh(z / cap)
            m = z.max(1, keepdim=True).values
            total = torch.exp(z - m).sum(1, keepdim=True)
            logp = z - m - torch.log(total)
            out["entropy"].append(-(torch.exp(logp) * logp).sum(1))
            out["logprobs"].append(torch.gather(logp, 1, st["targets"][a : a + 256].long()))
            out["top_logprobs"].append(torch.topk(logp, k, 1).values if k else logp[:, :0])
        return {name: None if v is None else torch.cat(v) for name, v in out.items()}

    st = prepare(case, seed)
    return {"rope": exact_rope, "attention": exact_attention, "logprobs": exact_logprobs}[case["op"]](st, case)
