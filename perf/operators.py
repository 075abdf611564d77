"""Timed cases of the operators over packed sequences: softmax attention, rotary positions, linear attention with decay.

``run`` computes a case in its plain form (elementary torch operations in float32, each output rounded once at the
end); with ``own`` set it makes the framework's calls instead. Sequences are packed one behind the other along the
first dimension: random walks (every walk is a sequence of its nodes), the node sequences of a batch of graphs,
prompts of different lengths, and single tokens against the keys kept of earlier ones.

  attn-*    dense softmax attention inside each sequence, grouped heads, causal or not; ``train`` with gradients,
            ``prompt`` forward only, ``decode`` one query a sequence against its kept keys
  rotary-*  rotary positions of q and k, ``train`` with gradients
  linear-*  linear attention with a decay for each head: ``train`` with gradients, ``prompt`` forward with the
            final state of each sequence, ``step`` one token a sequence on its kept state
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
MOST_SCORES = 16 * 8192 * 8192      # scores of a padded batch in the plain form: sequences * heads * longest^2


def listed():
    return [
        # one request's next token: launches and latency are all there is
        dict(name="attn-decode-one", kind="attn", mode="decode", n=1, lo=777, hi=777, lens=1, hq=32, hk=8, d=128,
             dtype="bfloat16", causal=True),
        # the next token of 64 requests with contexts of very different lengths
        dict(name="attn-decode", kind="attn", mode="decode", n=64, lo=500, hi=8191, lens=2, hq=32, hk=8, d=128,
             dtype="bfloat16", causal=True),
        # a few prompts of different lengths, packed
        dict(name="attn-prompt", kind="attn", mode="prompt", n=6, lo=301, hi=4096, lens=3, hq=32, hk=8, d=128,
             dtype="bfloat16", causal=True),
        # training on one long sequence
        dict(name="attn-train-long", kind="attn", mode="train", n=1, lo=8192, hi=8192, lens=4, hq=16, hk=4, d=128,
             dtype="bfloat16", causal=True),
        # training on a batch of graphs: every node attends its own graph, 8 heads of 32
        dict(name="attn-train-graphs", kind="attn", mode="train", n=256, lo=9, hi=250, lens=5, hq=8, hk=8, d=32,
             dtype="float16", causal=False),
        # training on the walks of a 169,343-node graph (two walks of four steps a node), 8 heads of 16
        dict(name="attn-train-walks", kind="attn", mode="train", n=338686, lo=5, hi=5, lens=6, hq=8, hk=8, d=16,
             dtype="float32", causal=True),
        # the positions of 64 next tokens, some of them far into a long context
        dict(name="rotary-decode", kind="rotary", mode="infer", t=64, far=1000000, hq=32, hk=8, d=128, rot=128,
             interleaved=False, factor=8.0, dtype="bfloat16"),
        # training: positions of 16K packed tokens, half of every head rotated
        dict(name="rotary-train", kind="rotary", mode="train", t=16411, far=16411, hq=16, hk=16, d=64, rot=32,
             interleaved=True, factor=1.0, dtype="float32"),
        # a long prompt's positions
        dict(name="rotary-prompt", kind="rotary", mode="infer", t=32768, far=32768, hq=32, hk=8, d=128, rot=128,
             interleaved=False, factor=4.0, dtype="bfloat16"),
        # one token of each of 64 sequences on its state
        dict(name="linear-step", kind="linear", mode="step", n=64, lo=1, hi=1, lens=7, h=16, dk=128, dv=128,
             dtype="bfloat16"),
        # a long prompt, its final state kept for the tokens that follow
        dict(name="linear-prompt", kind="linear", mode="prompt", n=1, lo=8192, hi=8192, lens=8, h=16, dk=128, dv=128,
             dtype="bfloat16"),
        # training on packed sequences of different lengths
        dict(name="linear-train", kind="linear", mode="train", n=9, lo=127, hi=4096, lens=9, h=8, dk=64, dv=64,
             dtype="float16"),
    ]


def _span(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rotary", "linear", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    lens = rng.randrange(1 << 30)
    if kind == "rotary":
        mode = rng.choice(["infer", "train"])
        d = rng.choice([16, 32, 64, 128])
        hk = rng.choice([1, 2, 4, 8])
        rot = rng.choice([d, d, d // 2])
        return dict(kind=kind, mode=mode, t=_span(rng, 1, 20000), far=_span(rng, 20000, 2000000), hq=hk * rng.choice([1, 2, 4]),
                    hk=hk, d=d, rot=rot, interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 8.0]), dtype=dtype)
    if kind == "linear":
        mode = rng.choice(["train", "prompt", "step"])
        dk, dv = rng.choice([(64, 64), (128, 128), (32, 64), (64, 128), (16, 16)])
        h = rng.choice([2, 4, 8, 16])
        if mode == "step":
            return dict(kind=kind, mode=mode, n=_span(rng, 1, 64), lo=1, hi=1, lens=lens, h=h, dk=dk, dv=dv, dtype=dtype)
        hi = _span(rng, 1, 6000)
        n = _span(rng, 1, max(1, min(64, MOST_SCORES // 2 // (h * hi * hi))))
        return dict(kind=kind, mode=mode, n=n, lo=max(1, hi // rng.choice([1, 3, 10])), hi=hi, lens=lens, h=h, dk=dk,
                    dv=dv, dtype=dtype)
    mode = rng.choice(["decode", "prompt", "train", "train"])
    d = rng.choice([16, 32, 64, 64, 128, 128])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 1, 2, 4])
    if mode == "decode":
        hi = _span(rng, 1, 8191)
        return dict(kind=kind, mode=mode, n=_span(rng, 1, 64), lo=max(1, hi // rng.choice([1, 4, 16])), hi=hi, lens=lens,
                    hq=hq, hk=hk, d=d, dtype=dtype, causal=True)
    hi = _span(rng, 1, 6000)
    if dtype == "float32":
        hi = min(hi, 2500)
    n = _span(rng, 1, max(1, min(20000, MOST_SCORES // 2 // (hq * hi * hi))))
    n = max(1, min(n, 400000 // hi))
    return dict(kind=kind, mode=mode, n=n, lo=max(1, hi // rng.choice([1, 3, 10])), hi=hi, lens=lens, hq=hq, hk=hk, d=d,
                dtype=dtype, causal=rng.random() < 0.7)


def _lengths(case):
    """The sequences' key lengths, part of the case and not of its seed."""
    rng = random.Random(case["lens"])
    got = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]
    got[0] = case["hi"]                                  # the longest is there
    return got


def _offsets(lengths):
    """Where each sequence starts, and the end of the last, int32 on the GPU."""
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


# ------------------------------------------------------------------ inputs (from the seed alone)
def _frequencies(case):
    """Radians per position of each rotated pair, float64: theta^(-2i/rot), divided by the context's factor."""
    half = case["rot"] // 2
    return 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half) / case["factor"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    s = dict(case=dict(case))
    if case["kind"] == "rotary":
        t, d = case["t"], case["d"]
        s["q"], s["k"] = rand(t, case["hq"], d), rand(t, case["hk"], d)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        s["freq"] = _frequencies(case).cuda()
        if case["mode"] == "train":
            s["dq"], s["dk"] = rand(t, case["hq"], d), rand(t, case["hk"], d)
        if own:
            from budgetformer_amd import RotaryFrequencies
            s["rotary"] = RotaryFrequencies(case["rot"], base=10000.0, factor=case["factor"], device="cuda")
            if case["mode"] == "train":
                s["q"].requires_grad_(True), s["k"].requires_grad_(True)
        return s
    lens = _lengths(case)
    total = sum(lens)
    if case["kind"] == "linear":
        h, dk, dv = case["h"], case["dk"], case["dv"]
        s["q"], s["k"], s["v"] = rand(total, h, dk), rand(total, h, dk), rand(total, h, dv)
        s["log_decay"] = torch.log1p(-2.0 ** (-3.0 - 6.0 * torch.arange(h, dtype=torch.float64) / h)).float().cuda()
        if case["mode"] == "step":
            s["state"] = rand(case["n"], h, dk, dv, dtype=torch.float32)
            return s
        s["offsets"] = _offsets(lens)
        if case["mode"] == "train":
            s["dout"] = rand(total, h, dv)
        if own:
            from budgetformer_amd import PackedSequences
            s["seqs"] = PackedSequences.from_lengths(lens, causal=True, device="cuda")
            if case["mode"] == "train":
                s["q"].requires_grad_(True), s["k"].requires_grad_(True), s["v"].requires_grad_(True)
        return s
    q_lens = [1] * len(lens) if case["mode"] == "decode" else lens
    n_q = sum(q_lens)
    s["q"] = rand(n_q, case["hq"], case["d"])
    s["k"], s["v"] = rand(total, case["hk"], case["d"]), rand(total, case["hk"], case["d"])
    s["q_offsets"], s["k_offsets"] = _offsets(q_lens), _offsets(lens)
    if case["mode"] == "train":
        s["dout"] = rand(n_q, case["hq"], case["d"])
    if own:
        from budgetformer_amd import PackedSequences
        s["seqs"] = PackedSequences.from_lengths(q_lens, lens, causal=case["causal"], device="cuda")
        if case["mode"] == "train":
            s["q"].requires_grad_(True), s["k"].requires_grad_(True), s["v"].requires_grad_(True)
    return s


# ------------------------------------------------------------------ plain forms
def _pad(x, offsets, longest):
    """[T, heads, d] packed -> [sequences, heads, longest, d] float32 with zeros behind each sequence's end."""
    at = offsets[:-1, None].long() + torch.arange(longest, device=x.device)
    valid = at < offsets[1:, None]
    got = x[at.clamp(max=x.size(0) - 1)].float() * valid[:, :, None, None]
    return got.transpose(1, 2).contiguous()


def _unpad(x, offsets, total):
    """[sequences, heads, longest, d] -> [T, heads, d] packed."""
    row = torch.arange(total, device=x.device)
    seq = torch.searchsorted(offsets.long(), row, right=True) - 1
    return x[seq, :, row - offsets.long()[seq]]


def _attention(s):
    c = s["case"]
    q, k, v, qo, ko = s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"]
    n, hk, d, group = c["n"], c["hk"], c["d"], c["hq"] // c["hk"]
    lk = c["hi"]
    lq = 1 if c["mode"] == "decode" else lk
    scale = 1.0 / math.sqrt(d)
    kp, vp = _pad(k, ko, lk), _pad(v, ko, lk)

    def by_kv_head(x):                       # the queries of a group below each other: [n, hk, group * lq, d]
        return _pad(x, qo, lq).view(n, hk, group * lq, d)

    def by_token(x):
        return _unpad(x.view(n, hk * group, lq, d), qo, q.size(0))

    qp = by_kv_head(q)
    len_q, len_k = (qo[1:] - qo[:-1]).long(), (ko[1:] - ko[:-1]).long()
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    seen = (j < len_k[:, None])[:, None, :]
    if c["causal"]:
        seen = seen & (j <= i[:, None] + (len_k - len_q)[:, None, None])
    seen = seen.expand(n, lq, lk)[:, None, None].expand(n, 1, group, lq, lk).reshape(n, 1, group * lq, lk)
    p = (qp @ kp.transpose(2, 3)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = p.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-37))
    out = p @ vp
    if c["mode"] != "train":
        return by_token(out).to(q.dtype)
    do = by_kv_head(s["dout"])
    dv = p.transpose(2, 3) @ do
    ds = (do @ vp.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ kp
    dk = ds.transpose(2, 3) @ qp
    return (by_token(out).to(q.dtype), by_token(dq).to(q.dtype), _unpad(dk, ko, k.size(0)).to(k.dtype),
            _unpad(dv, ko, k.size(0)).to(v.dtype))


def _rotate(x, cos, sin, case):
    """x [T, heads, d]: its first `rot` values turned pair by pair; cos, sin [T, 1, rot / 2]."""
    rot, half = case["rot"], case["rot"] // 2
    y = x.float()
    if case["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None, None] * s["freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    out = (_rotate(s["q"], cos, sin, c), _rotate(s["k"], cos, sin, c))
    if c["mode"] != "train":
        return out
    return out + (_rotate(s["dq"], cos, -sin, c), _rotate(s["dk"], cos, -sin, c))


def _linear_step(s):
    scale = 1.0 / math.sqrt(s["case"]["dk"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    state = s["state"] * s["log_decay"].exp()[:, None, None] + k[..., :, None] * v[..., None, :]
    return (q[..., None] * state).sum(2).mul_(scale).to(s["q"].dtype), state


def _linear(s):
    c = s["case"]
    if c["mode"] == "step":
        return _linear_step(s)
    off, longest, total = s["offsets"], c["hi"], s["q"].size(0)
    scale = 1.0 / math.sqrt(c["dk"])
    q, k, v = (_pad(s[x], off, longest) for x in ("q", "k", "v"))
    i = torch.arange(longest, device=q.device)
    ahead = (i[:, None] - i)
    decay = (s["log_decay"][:, None, None] * ahead.clamp(min=0)).exp().mul_(ahead >= 0).mul_(scale)   # [h, longest, longest]
    w = (q @ k.transpose(2, 3)).mul_(decay)
    out = _unpad(w @ v, off, total).to(s["q"].dtype)
    if c["mode"] == "prompt":
        left = ((off[1:] - off[:-1])[:, None, None] - 1 - i).clamp(min=0)
        kept = k * (s["log_decay"][None, :, None] * left).exp()[..., None]
        return out, kept.transpose(2, 3) @ v
    do = _pad(s["dout"], off, longest)
    dv = w.transpose(2, 3) @ do
    dw = (do @ v.transpose(2, 3)).mul_(decay)
    dq, dk = dw @ k, dw.transpose(2, 3) @ q
    return (out,) + tuple(_unpad(x, off, total).to(s["q"].dtype) for x in (dq, dk, dv))


# ------------------------------------------------------------------ the framework's calls
def _own_run(s):
    import budgetformer_amd as bf
    c = s["case"]
    if c["kind"] == "rotary":
        out = bf.rotary_embedding(s["q"], s["k"], s["rotary"], positions=s["positions"], interleaved=c["interleaved"])
        if c["mode"] == "train":
            out += torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))
        return out
    if c["kind"] == "linear":
        if c["mode"] == "step":
            return bf.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        if c["mode"] == "prompt":
            return bf.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["seqs"], return_state=True)
        out = bf.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["seqs"])
        return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    out = bf.packed_attention(s["q"], s["k"], s["v"], s["seqs"])
    if c["mode"] != "train":
        return out
    return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _attention, "rotary": _rotary, "linear": _linear}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["kind"] == "rotary":
        values = case["t"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": (2 + 2 * train) * b * values + 8 * case["t"], "flops": (3 + 3 * train) * values}
    lens = _lengths(case)
    if case["kind"] == "linear":
        h, dk, dv, t = case["h"], case["dk"], case["dv"], sum(lens)
        rows = t * h * b * (2 * dk + 2 * dv)                      # q, k, v, out
        state = case["n"] * h * dk * dv * 4
        if case["mode"] == "step":
            return {"bytes": rows + 2 * state, "flops": 4 * t * h * dk * dv}
        if case["mode"] == "prompt":
            return {"bytes": rows + state, "flops": 4 * t * h * dk * dv}
        return {"bytes": rows + t * h * b * (2 * dk + 2 * dv), "flops": 14 * t * h * dk * dv}
    d, hq, hk = case["d"], case["hq"], case["hk"]
    decode = case["mode"] == "decode"
    n_q = case["n"] if decode else sum(lens)
    pairs = sum(lens) if decode else sum(x * (x + 1) // 2 if case["causal"] else x * x for x in lens)
    once = b * d * (2 * n_q * hq + 2 * sum(lens) * hk)            # q, out, k, v
    if not train:
        return {"bytes": once, "flops": 4 * d * hq * pairs}
    return {"bytes": once + b * d * (2 * n_q * hq + 2 * sum(lens) * hk), "flops": 14 * d * hq * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_pairs(s, c, lens):
    """Attention as a list of (query, key) pairs, for many short sequences."""
    dev = s["q"].device
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    group = c["hq"] // c["hk"]
    n = torch.tensor(lens, device=dev)
    start = s["k_offsets"][:-1].long()
    first = torch.repeat_interleave(start, n)                       # of each query (as many queries as keys)
    own_at = torch.arange(q.size(0), device=dev)
    count = own_at - first + 1 if c["causal"] else torch.repeat_interleave(n, n)
    pq = torch.repeat_interleave(own_at, count)
    nth = torch.arange(pq.numel(), device=dev) - torch.repeat_interleave(count.cumsum(0) - count, count)
    pk = torch.repeat_interleave(first, count) + nth
    scale = c["d"] ** -0.5
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    w = ((q[pq] * k[pk]).sum(-1) * scale).exp()                     # values of a few units: no maximum is needed in 64 bits
    z = torch.zeros(q.shape[:2], dtype=torch.float64, device=dev).index_add_(0, pq, w)
    p = w / z[pq]
    out = torch.zeros_like(q).index_add_(0, pq, p[..., None] * v[pk])
    if c["mode"] != "train":
        return out
    do = s["dout"].double()
    dp = (do[pq] * v[pk]).sum(-1)
    mean = torch.zeros_like(z).index_add_(0, pq, p * dp)
    ds = p * (dp - mean[pq]) * scale
    dq = torch.zeros_like(q).index_add_(0, pq, ds[..., None] * k[pk])
    dk = torch.zeros_like(k).index_add_(0, pk, ds[..., None] * q[pq])
    dv = torch.zeros_like(k).index_add_(0, pk, p[..., None] * do[pq])
    return out, dq, *(x.view(-1, c["hk"], group, c["d"]).sum(2) for x in (dk, dv))


def _exact_sequences(s, c, lens):
    """One sequence, and one head of k and v, after the other, with gradients by differentiation."""
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    train, group = c["mode"] == "train", c["hq"] // c["hk"]
    outs = [torch.zeros_like(q)] + ([torch.zeros_like(x) for x in (q, k, v)] if train else [])
    q0 = k0 = 0
    for n in lens:
        m = 1 if c["mode"] == "decode" else n
        for h in range(c["hk"]):
            rows, keys, heads = slice(q0, q0 + m), slice(k0, k0 + n), slice(h * group, (h + 1) * group)
            a = q[rows, heads].transpose(0, 1).contiguous().requires_grad_(train)
            b, w = (x[keys, h].contiguous().requires_grad_(train) for x in (k, v))
            scores = torch.einsum("gid,jd->gij", a, b) / math.sqrt(c["d"])
            if c["causal"]:
                scores = scores + torch.full((m, n), -math.inf, dtype=torch.float64, device=q.device).triu(n - m + 1)
            out = torch.einsum("gij,jd->gid", scores.softmax(-1), w)
            outs[0][rows, heads] = out.detach().transpose(0, 1)
            if train:
                g = torch.autograd.grad(out, (a, b, w), s["dout"][rows, heads].double().transpose(0, 1))
                outs[1][rows, heads], outs[2][keys, h], outs[3][keys, h] = g[0].transpose(0, 1), g[1], g[2]
            del scores, out
        q0, k0 = q0 + m, k0 + n
    return tuple(outs) if train else outs[0]


def _exact_rotary(s, c):
    """Each pair as a complex number, turned by exp(i * angle)."""
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=s["q"].device),
                       s["positions"].double()[:, None] * s["freq"])[:, None]

    def turned(x, by):
        x, rot = x.double(), c["rot"]
        pairs = x[..., :rot].unflatten(-1, (rot // 2, 2)) if c["interleaved"] else \
            x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        got = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        got = got if c["interleaved"] else got.transpose(-1, -2)
        return torch.cat([got.flatten(-2), x[..., rot:]], -1)

    out = turned(s["q"], turn), turned(s["k"], turn)
    return out if c["mode"] != "train" else out + (turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj()))


def _exact_linear(s, c, lens):
    """The recurrence, some tokens at a time: within a block by its pairs, across blocks by the state; gradients by
    differentiation."""
    train = c["mode"] == "train"
    ld = s["log_decay"].double()
    scale = c["dk"] ** -0.5
    if c["mode"] == "step":
        state = s["state"].double() * ld.exp()[:, None, None] + torch.einsum("nhk,nhv->nhkv", s["k"].double(), s["v"].double())
        return torch.einsum("nhk,nhkv->nhv", s["q"].double(), state) * scale, state
    outs, states, at = [], [], 0
    for n in lens:
        rows = slice(at, at + n)
        q, k, v = (s[x][rows].double().transpose(0, 1).contiguous().requires_grad_(train) for x in ("q", "k", "v"))
        state = torch.zeros(c["h"], c["dk"], c["dv"], dtype=torch.float64, device=q.device)
        parts = []
        for a in range(0, n, 256):
            x, y, z = (t[:, a:a + 256] for t in (q, k, v))
            m = x.size(1)
            i = torch.arange(m, device=q.device, dtype=torch.float64)
            power = (ld[:, None, None] * (i[:, None] - i)).exp().tril()
            into = (ld[:, None] * (i + 1)).exp()[..., None]
            left = (ld[:, None] * (m - 1 - i)).exp()[..., None]
            parts.append(((x @ y.transpose(1, 2)) * power) @ z + (x * into) @ state)
            state = state * (ld * m).exp()[:, None, None] + (y * left).transpose(1, 2) @ z
        out = torch.cat(parts, 1) * scale
        got = [out.detach()]
        if train:
            got += torch.autograd.grad(out, (q, k, v), s["dout"][rows].double().transpose(0, 1))
        outs.append([x.transpose(0, 1) for x in got])
        states.append(state.detach())
        at += n
    got = tuple(torch.cat([o[j] for o in outs]) for j in range(len(outs[0])))
    return got if train else (got[0], torch.stack(states))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s, case)
    lens = _lengths(case)
    if case["kind"] == "linear":
        return _exact_linear(s, case, lens)
    return _exact_pairs(s, case, lens) if case["n"] > 600 else _exact_sequences(s, case, lens)
