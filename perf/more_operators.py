"""Timed cases of two further operators over packed sequences: attention with a learned bias by buckets of the relative
position, and the gated delta rule.

``run`` computes a case in its plain form (elementary torch operations in float32, each output rounded once at the
end); with ``own`` set it makes the framework's calls instead. Sequences are packed one behind the other along the
first dimension: random walks, the node sequences of a batch of graphs, prompts of different lengths, single tokens
behind what is kept of earlier ones.

  bias-*    dense softmax attention whose scores get table[head, bucket(place of the key - place of the row)]: ``train``
            with all gradients, the table's among them, ``prompt`` forward only, ``decode`` one query a sequence
  delta-*   the gated delta rule, a state of [key values, value values] a head: ``train`` with all gradients (gates and
            strengths too), ``prompt`` forward with each sequence's final state, ``step`` one token a sequence
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
MOST_SCORES = 16 * 4096 * 4096      # scores of a padded batch in the plain form: sequences * heads * longest^2


def listed():
    return [
        # one graph of 50 nodes, a small batch's training step: launches and latency are all there is
        dict(name="bias-train-one", kind="bias", mode="train", n=1, lo=50, hi=50, lens=1, hq=8, hk=8, d=32, buckets=32, far=128,
             both=True, dtype="bfloat16", causal=False),
        # training on a batch of graphs: every node attends its own graph
        dict(name="bias-train-graphs", kind="bias", mode="train", n=256, lo=9, hi=250, lens=2, hq=8, hk=8, d=32, buckets=32,
             far=128, both=True, dtype="float16", causal=False),
        # training on one walk of four steps from every node of a 169,343-node graph
        dict(name="bias-train-walks", kind="bias", mode="train", n=169343, lo=5, hi=5, lens=3, hq=8, hk=8, d=16, buckets=8,
             far=16, both=True, dtype="float32", causal=False),
        # training on two long sequences, causal, grouped heads
        dict(name="bias-train-long", kind="bias", mode="train", n=2, lo=3500, hi=4096, lens=4, hq=16, hk=4, d=64, buckets=32,
             far=128, both=False, dtype="bfloat16", causal=True),
        # a few prompts of different lengths
        dict(name="bias-prompt", kind="bias", mode="prompt", n=5, lo=301, hi=4096, lens=5, hq=16, hk=4, d=128, buckets=32,
             far=128, both=False, dtype="bfloat16", causal=True),
        # the next token of 64 requests with contexts of very different lengths
        dict(name="bias-decode", kind="bias", mode="decode", n=64, lo=500, hi=8191, lens=6, hq=32, hk=8, d=128, buckets=32,
             far=128, both=False, dtype="bfloat16", causal=True),
        # one request's next token
        dict(name="delta-step-one", kind="delta", mode="step", n=1, lo=1, hi=1, lens=7, h=16, hk=16, dk=128, dv=128,
             dtype="bfloat16"),
        # the next token of 64 requests
        dict(name="delta-step", kind="delta", mode="step", n=64, lo=1, hi=1, lens=8, h=16, hk=8, dk=128, dv=128,
             dtype="bfloat16"),
        # a long prompt, its final state kept for the tokens that follow
        dict(name="delta-prompt", kind="delta", mode="prompt", n=1, lo=8192, hi=8192, lens=9, h=16, hk=16, dk=128, dv=128,
             dtype="bfloat16"),
        # training on packed sequences of different lengths
        dict(name="delta-train", kind="delta", mode="train", n=9, lo=127, hi=4096, lens=10, h=8, hk=8, dk=64, dv=64,
             dtype="float16"),
        # training on wide heads, two value heads to a key head
        dict(name="delta-train-wide", kind="delta", mode="train", n=3, lo=1000, hi=2047, lens=11, h=16, hk=8, dk=128, dv=128,
             dtype="bfloat16"),
        # training on a batch of graphs
        dict(name="delta-train-graphs", kind="delta", mode="train", n=256, lo=9, hi=250, lens=12, h=4, hk=4, dk=32, dv=32,
             dtype="float32"),
    ]


def _span(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["bias", "delta"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    lens = rng.randrange(1 << 30)
    if kind == "delta":
        mode = rng.choice(["train", "train", "prompt", "step"])
        dk, dv = rng.choice([(64, 64), (128, 128), (32, 64), (64, 128), (16, 16), (128, 64), (24, 40)])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 1, 2, 4])
        if mode == "step":
            return dict(kind=kind, mode=mode, n=_span(rng, 1, 64), lo=1, hi=1, lens=lens, h=h, hk=hk, dk=dk, dv=dv, dtype=dtype)
        hi = _span(rng, 1, 4096)
        n = _span(rng, 1, max(1, min(256, 16384 // hi)))
        return dict(kind=kind, mode=mode, n=n, lo=max(1, hi // rng.choice([1, 3, 10])), hi=hi, lens=lens, h=h, hk=hk, dk=dk,
                    dv=dv, dtype=dtype)
    mode = rng.choice(["decode", "prompt", "train", "train"])
    d = rng.choice([16, 32, 64, 64, 128, 40])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 1, 2, 3, 4])
    both = rng.random() < 0.5
    buckets = 2 * _span(rng, 4, 32)
    how = dict(hq=hq, hk=hk, d=d, buckets=buckets, far=_span(rng, buckets, 500), both=both, dtype=dtype)
    if mode == "decode":
        hi = _span(rng, 1, 8191)
        return dict(kind=kind, mode=mode, n=_span(rng, 1, 64), lo=max(1, hi // rng.choice([1, 4, 16])), hi=hi, lens=lens,
                    causal=True, **how)
    hi = _span(rng, 1, 4000)
    if dtype == "float32":
        hi = min(hi, 2000)
    n = _span(rng, 1, max(1, min(20000, MOST_SCORES // 2 // (hq * hi * hi))))
    n = max(1, min(n, 200000 // hi))
    return dict(kind=kind, mode=mode, n=n, lo=max(1, hi // rng.choice([1, 3, 10])), hi=hi, lens=lens,
                causal=not both or rng.random() < 0.3, **how)


def _lengths(case):
    """The sequences' key lengths, part of the case and not of its seed."""
    rng = random.Random(case["lens"])
    got = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]
    got[0] = case["hi"]                                  # the longest is there
    return got


def _offsets(lengths):
    """Where each sequence starts, and the end of the last, int32 on the GPU."""
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _bucket(case, ahead):
    """The bucket of a key `ahead` places after its row (before it: negative). Half of the buckets (of a direction) hold one
    distance each, the others distances that grow by one factor up to `far`, from where on all are in the last."""
    n, base = case["buckets"], 0
    if case["both"]:
        n //= 2
        base = n if ahead > 0 else 0
        away = abs(ahead)
    else:
        away = max(-ahead, 0)
    exact = n // 2
    if away < exact:
        return base + away
    if away >= case["far"]:
        return base + n - 1
    k, steps = 0, n - exact                              # the most k with away / exact >= (far / exact)^(k / steps)
    while k + 1 < steps and away ** steps * exact ** (k + 1) >= case["far"] ** (k + 1) * exact ** steps:
        k += 1
    return base + exact + k


# ------------------------------------------------------------------ inputs (from the seed alone)
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def unit(*shape):
        x = torch.randn(*shape, generator=gen, device="cuda")
        return (x / (x * x).sum(-1, keepdim=True).sqrt()).to(dt)

    s = dict(case=dict(case))
    train = case["mode"] == "train"
    lens = _lengths(case)
    total = sum(lens)
    if case["kind"] == "delta":
        h, hk, dk, dv = case["h"], case["hk"], case["dk"], case["dv"]
        s["q"], s["k"], s["v"] = unit(total, hk, dk), unit(total, hk, dk), rand(total, h, dv)
        s["log_gate"] = -(rand(total, h, dtype=torch.float32) * 1.5 - 3.0).exp().log1p()     # most gates are near 1, some forget
        s["beta"] = torch.sigmoid(rand(total, h, dtype=torch.float32))
        grads = ("q", "k", "v", "log_gate", "beta")
        if case["mode"] == "step":
            s["state"] = rand(case["n"], h, dk, dv, dtype=torch.float32)
            return s
        s["offsets"] = _offsets(lens)
        if train:
            s["dout"] = rand(total, h, dv)
        if own:
            from budgetformer_amd import PackedSequences
            s["seqs"] = PackedSequences.from_lengths(lens, causal=True, device="cuda")
    else:
        q_lens = [1] * len(lens) if case["mode"] == "decode" else lens
        n_q = sum(q_lens)
        s["q"] = rand(n_q, case["hq"], case["d"])
        s["k"], s["v"] = rand(total, case["hk"], case["d"]), rand(total, case["hk"], case["d"])
        s["table"] = rand(case["hq"], case["buckets"], dtype=torch.float32)
        s["q_offsets"], s["k_offsets"] = _offsets(q_lens), _offsets(lens)
        grads = ("q", "k", "v", "table")
        if train:
            s["dout"] = rand(n_q, case["hq"], case["d"])
        if own:
            from budgetformer_amd import PackedSequences, RelativeBuckets
            s["seqs"] = PackedSequences.from_lengths(q_lens, lens, causal=case["causal"], device="cuda")
            s["buckets"] = RelativeBuckets(case["buckets"], case["far"], bidirectional=case["both"], device="cuda")
        else:
            s["bucket"] = torch.tensor([_bucket(case, x) for x in range(1 - case["hi"], case["hi"])]).cuda()
    if train and own:
        for x in grads:
            s[x].requires_grad_(True)
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
    n, hq, hk, d, group = c["n"], c["hq"], c["hk"], c["d"], c["hq"] // c["hk"]
    lk = c["hi"]
    lq = 1 if c["mode"] == "decode" else lk
    scale = 1.0 / math.sqrt(d)
    qp = _pad(q, qo, lq)
    kp, vp = (_pad(x, ko, lk).repeat_interleave(group, 1) for x in (k, v))
    len_q, len_k = (qo[1:] - qo[:-1]).long(), (ko[1:] - ko[:-1]).long()
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    past = len_k - len_q                                                # 0 but for single tokens
    ahead = j - (i[:, None] + (past if lq == 1 else past[:1])[:, None, None])     # [n or 1, lq, lk]
    seen = (j < len_k[:, None])[:, None, :]
    if c["causal"]:
        seen = seen & (ahead <= 0)
    seen = seen[:, None]                                                # [n, 1, lq or 1, lk]
    bias = s["table"][:, s["bucket"][(ahead + lk - 1).clamp(0, 2 * lk - 2)]].transpose(0, 1)       # [n or 1, hq, lq, lk]
    p = (qp @ kp.transpose(2, 3)).mul_(scale).add_(bias).masked_fill_(~seen, -math.inf)
    del bias
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-37))
    out = p @ vp
    if c["mode"] != "train":
        return _unpad(out, qo, q.size(0)).to(q.dtype)
    do = _pad(s["dout"], qo, lq)
    dv = p.transpose(2, 3) @ do
    ds = (do @ vp.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    # each distance's sum: row i moved i places along (the last row by none), in rows of one value less than the padded ones
    pairs = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).flip(1), (0, lk))
    by_distance = pairs.flatten(1)[:, :lk * (2 * lk - 1)].view(hq, lk, 2 * lk - 1).sum(1)
    dtable = torch.zeros(hq, c["buckets"], dtype=torch.float64, device=q.device).index_add_(1, s["bucket"], by_distance)
    ds.mul_(scale)
    dq = ds @ kp
    dk = ds.transpose(2, 3) @ qp

    def by_key(x):
        return _unpad(x.view(n, hk, group, lk, d).sum(2), ko, k.size(0))

    return (_unpad(out, qo, q.size(0)).to(q.dtype), _unpad(dq, qo, q.size(0)).to(q.dtype), by_key(dk).to(k.dtype),
            by_key(dv).to(v.dtype), dtable.float())


def _delta_step(s):
    c = s["case"]
    scale, group = 1.0 / math.sqrt(c["dk"]), c["h"] // c["hk"]
    q, k = (s[x].float().repeat_interleave(group, 1) for x in ("q", "k"))
    state = s["state"] * s["log_gate"].exp()[..., None, None]
    missing = s["v"].float() - (k[..., None] * state).sum(2)
    state = state + k[..., None] * (s["beta"][..., None] * missing)[..., None, :]
    return (q[..., None] * state).sum(2).mul_(scale).to(s["q"].dtype), state


def _delta_chunks(q, k, v, log_gate, beta, scale):
    """The rule over padded sequences [n, heads, longest, d], 64 tokens at a time: (out, final states). Padding has k, v, beta
    and log_gate 0, which leave the state as it is."""
    n, h, longest, dk = q.shape
    m, size = -(-longest // 64), 64
    fill = m * size - longest

    def cut(x):
        return torch.nn.functional.pad(x, (0, 0, 0, fill)).unflatten(2, (m, size))

    q, k, v = cut(q), cut(k), cut(v)
    beta, gate = cut(beta[..., None]), cut(log_gate[..., None])[..., 0].cumsum(-1)
    i = torch.arange(size, device=q.device)
    decay = (gate[..., :, None] - gate[..., None, :]).masked_fill(i[:, None] < i, -math.inf).exp()
    scores = (q @ k.transpose(-1, -2)) * decay * scale
    a = beta * (k @ k.transpose(-1, -2)) * decay * (i[:, None] > i)
    # (1 + a)^-1, a row after the other
    rows = [torch.nn.functional.one_hot(i[:1], size).float().expand(n, h, m, 1, size)]
    for r in range(1, size):
        above = torch.cat(rows, -2)
        rows.append(torch.nn.functional.one_hot(i[r:r + 1], size).float() - a[..., r:r + 1, :r] @ above)
    inverse = torch.cat(rows, -2) * beta.transpose(-1, -2)
    whole = gate.exp()[..., None]
    own_part, read = inverse @ v, inverse @ (whole * k)
    into, kept = q * whole * scale, k * (gate[..., -1:] - gate).exp()[..., None]
    state = q.new_zeros(n, h, dk, v.size(-1))
    outs = []
    for t in range(m):
        u = own_part[:, :, t] - read[:, :, t] @ state
        outs.append(into[:, :, t] @ state + scores[:, :, t] @ u)
        state = state * gate[:, :, t, -1].exp()[..., None, None] + kept[:, :, t].transpose(-1, -2) @ u
    return torch.cat(outs, 2)[:, :, :longest], state


def _delta(s):
    c = s["case"]
    if c["mode"] == "step":
        return _delta_step(s)
    off, longest, total, group = s["offsets"], c["hi"], s["q"].size(0), c["h"] // c["hk"]
    train, dt = c["mode"] == "train", s["q"].dtype
    leaves = [_pad(s[x], off, longest) for x in ("q", "k", "v")] + \
             [_pad(s[x][..., None], off, longest)[..., 0] for x in ("log_gate", "beta")]
    with torch.set_grad_enabled(train):
        for x in leaves:
            x.requires_grad_(train)
        q, k = (x.repeat_interleave(group, 1) for x in leaves[:2])
        out, state = _delta_chunks(q, k, *leaves[2:], 1.0 / math.sqrt(c["dk"]))
    got = _unpad(out.detach(), off, total).to(dt)
    if not train:
        return got, state
    grads = torch.autograd.grad(out, leaves, _pad(s["dout"], off, longest))
    return (got,) + tuple(_unpad(x, off, total).to(dt) for x in grads[:3]) + \
        tuple(_unpad(x[..., None], off, total)[..., 0].contiguous() for x in grads[3:])


# ------------------------------------------------------------------ the framework's calls
def _own_run(s):
    import budgetformer_amd as bf
    c = s["case"]
    if c["kind"] == "delta":
        leaves = [s[x] for x in ("q", "k", "v", "log_gate", "beta")]
        if c["mode"] == "step":
            return bf.gated_delta_step(*leaves, s["state"])
        if c["mode"] == "prompt":
            return bf.gated_delta_rule(*leaves, s["seqs"], return_state=True)
        out = bf.gated_delta_rule(*leaves, s["seqs"])
    else:
        leaves = [s[x] for x in ("q", "k", "v", "table")]
        out = bf.packed_attention(*leaves[:3], s["seqs"], bias=leaves[3], buckets=s["buckets"])
        if c["mode"] != "train":
            return out
    return (out,) + torch.autograd.grad(out, leaves, s["dout"])


def run(state):
    if own:
        return _own_run(state)
    return {"bias": _attention, "delta": _delta}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = BYTES[case["dtype"]]
    train = case["mode"] == "train"
    lens = _lengths(case)
    t = sum(lens)
    if case["kind"] == "delta":
        h, hk, dk, dv = case["h"], case["hk"], case["dk"], case["dv"]
        rows = t * (b * (2 * hk * dk + 2 * h * dv) + 8 * h)       # q, k, v, out; gate and strength
        state = case["n"] * h * dk * dv * 4
        if case["mode"] == "step":
            return {"bytes": rows + 2 * state, "flops": 6 * t * h * dk * dv}
        if case["mode"] == "prompt":
            return {"bytes": rows + state, "flops": 6 * t * h * dk * dv}
        return {"bytes": 2 * rows, "flops": 18 * t * h * dk * dv}
    d, hq, hk = case["d"], case["hq"], case["hk"]
    decode = case["mode"] == "decode"
    n_q = case["n"] if decode else t
    pairs = t if decode else sum(x * (x + 1) // 2 if case["causal"] else x * x for x in lens)
    once = b * d * (2 * n_q * hq + 2 * t * hk) + 4 * hq * case["buckets"]            # q, out, k, v, the table
    if not train:
        return {"bytes": once, "flops": 4 * d * hq * pairs}
    return {"bytes": 2 * once, "flops": 14 * d * hq * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_buckets(case, device):
    """The bucket of every distance 1 - hi .. hi - 1, from where each bucket begins."""
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    exact = n // 2
    begins = list(range(exact + 1))
    for k in range(1, n - exact):                        # the first whole x with (x / exact)^steps >= (far / exact)^k
        x = begins[-1]
        while x ** (n - exact) * exact ** k < case["far"] ** k * exact ** (n - exact):
            x += 1
        begins.append(x)
    begins = torch.tensor(begins, device=device)
    ahead = torch.arange(1 - case["hi"], case["hi"], device=device)
    away = ahead.abs() if case["both"] else (-ahead).clamp(min=0)
    got = (away[:, None] >= begins).sum(1) - 1
    return got + n * (ahead > 0) if case["both"] else got


def _exact_pairs(s, c, lens):
    """Attention as a list of (query, key) pairs, for many short sequences (as many queries as keys)."""
    dev = s["q"].device
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    group = c["hq"] // c["hk"]
    n = torch.tensor(lens, device=dev)
    first = torch.repeat_interleave(s["k_offsets"][:-1].long(), n)
    own_at = torch.arange(q.size(0), device=dev)
    count = own_at - first + 1 if c["causal"] else torch.repeat_interleave(n, n)
    pq = torch.repeat_interleave(own_at, count)
    nth = torch.arange(pq.numel(), device=dev) - torch.repeat_interleave(count.cumsum(0) - count, count)
    pk = torch.repeat_interleave(first, count) + nth
    bucket = _exact_buckets(c, dev)[pk - pq + c["hi"] - 1]
    scale = c["d"] ** -0.5
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    w = ((q[pq] * k[pk]).sum(-1) * scale + s["table"].double().T[bucket]).exp()     # values of a few units
    z = torch.zeros(q.shape[:2], dtype=torch.float64, device=dev).index_add_(0, pq, w)
    p = w / z[pq]
    out = torch.zeros_like(q).index_add_(0, pq, p[..., None] * v[pk])
    if c["mode"] != "train":
        return out
    do = s["dout"].double()
    dp = (do[pq] * v[pk]).sum(-1)
    mean = torch.zeros_like(z).index_add_(0, pq, p * dp)
    ds = p * (dp - mean[pq])
    dtable = torch.stack([(ds * (bucket == b)[:, None]).sum(0) for b in range(c["buckets"])], 1)
    ds = ds * scale
    dq = torch.zeros_like(q).index_add_(0, pq, ds[..., None] * k[pk])
    dk = torch.zeros_like(k).index_add_(0, pk, ds[..., None] * q[pq])
    dv = torch.zeros_like(k).index_add_(0, pk, p[..., None] * do[pq])
    return out, dq, *(x.view(-1, c["hk"], group, c["d"]).sum(2) for x in (dk, dv)), dtable


def _exact_attention(s, c, lens):
    """One sequence, and one head of k and v, after the other, with gradients by differentiation."""
    q, k, v, table = (s[x].detach().double() for x in ("q", "k", "v", "table"))
    train, group, dev = c["mode"] == "train", c["hq"] // c["hk"], q.device
    outs = [torch.zeros_like(q)] + ([torch.zeros_like(x) for x in (q, k, v, table)] if train else [])
    buckets = _exact_buckets(c, dev)
    q0 = k0 = 0
    for n in lens:
        m = 1 if c["mode"] == "decode" else n
        ahead = torch.arange(n, device=dev) - torch.arange(n - m, n, device=dev)[:, None]
        bucket = buckets[ahead + c["hi"] - 1]
        for h in range(c["hk"]):
            rows, keys, heads = slice(q0, q0 + m), slice(k0, k0 + n), slice(h * group, (h + 1) * group)
            a = q[rows, heads].transpose(0, 1).contiguous().requires_grad_(train)
            b, w = (x[keys, h].contiguous().requires_grad_(train) for x in (k, v))
            bias = table[heads][:, bucket].requires_grad_(train)                       # [group, m, n]
            scores = (a @ b.T) / math.sqrt(c["d"]) + bias
            if c["causal"]:
                scores = scores.masked_fill(ahead > 0, -math.inf)
            out = scores.softmax(-1) @ w
            outs[0][rows, heads] = out.detach().transpose(0, 1)
            if train:
                g = torch.autograd.grad(out, (a, b, w, bias), s["dout"][rows, heads].double().transpose(0, 1))
                outs[1][rows, heads], outs[2][keys, h], outs[3][keys, h] = g[0].transpose(0, 1), g[1], g[2]
                for x in range(c["buckets"]):
                    outs[4][heads, x] += (g[3] * (bucket == x)).sum((1, 2))
            del scores, out
        q0, k0 = q0 + m, k0 + n
    return tuple(outs) if train else outs[0]


def _exact_delta(s, c, lens):
    """The recurrence, a token of every sequence at a time, and its way back. Sequences that have ended are given k, v, beta
    and log_gate of 0."""
    dev, group, scale = s["q"].device, c["h"] // c["hk"], c["dk"] ** -0.5
    q, k, v, gate, beta = (s[x].detach().double() for x in ("q", "k", "v", "log_gate", "beta"))
    q, k = (x.repeat_interleave(group, 1) for x in (q, k))
    if c["mode"] == "step":
        state = s["state"].double() * gate.exp()[..., None, None]
        u = beta[..., None] * (v - (state * k[..., None]).sum(2))
        state = state + k[..., None] * u[..., None, :]
        return (state * q[..., None]).sum(2) * scale, state
    n, longest = len(lens), c["hi"]
    at = s["offsets"][:-1, None].long() + torch.arange(longest, device=dev)            # [n, longest]
    live = torch.arange(longest, device=dev) < torch.tensor(lens, device=dev)[:, None]
    at = torch.where(live, at, q.size(0))
    zero = lambda x: torch.cat([x, x.new_zeros(1, *x.shape[1:])])                       # noqa: E731
    by_time = lambda x: zero(x)[at.T]                                                   # noqa: E731  [longest, n, heads, ...]
    q, k, v, gate, beta = (by_time(x) for x in (q, k, v, gate, beta))
    train = c["mode"] == "train"
    state = q.new_zeros(n, c["h"], c["dk"], c["dv"])
    out, decayed, missing = torch.empty_like(v), [], torch.empty_like(v)
    for t in range(longest):
        before = state * gate[t].exp()[..., None, None]
        missing[t] = v[t] - (k[t][..., None, :] @ before)[..., 0, :]
        state = before + k[t][..., None] * (beta[t][..., None] * missing[t])[..., None, :]
        out[t] = (q[t][..., None, :] @ state)[..., 0, :] * scale
        if train:
            decayed.append(before)

    def packed(x):
        got = x.new_zeros(s["q"].size(0) + 1, *x.shape[2:])
        got[at.T] = x
        return got[:-1]

    if not train:
        return packed(out), state
    do = by_time(s["dout"].double()) * scale
    dq, dk, dv, dgate, dbeta = (torch.zeros_like(x) for x in (q, k, v, gate, beta))
    grad = torch.zeros_like(state)
    for t in reversed(range(longest)):
        before = decayed.pop()
        u = beta[t][..., None] * missing[t]
        state = before + k[t][..., None] * u[..., None, :]
        grad = grad + q[t][..., None] * do[t][..., None, :]
        dq[t] = (state @ do[t][..., None])[..., 0]
        du = (k[t][..., None, :] @ grad)[..., 0, :]
        dk[t] = (grad @ u[..., None])[..., 0]
        dbeta[t] = (du * missing[t]).sum(-1)
        dv[t] = beta[t][..., None] * du
        grad = grad - k[t][..., None] * dv[t][..., None, :]
        dk[t] -= (before @ dv[t][..., None])[..., 0]
        dgate[t] = (grad * before).sum((-1, -2))
        grad = grad * gate[t].exp()[..., None, None]
    dq, dk = (packed(x).unflatten(1, (c["hk"], group)).sum(2) for x in (dq, dk))
    return packed(out), dq, dk, packed(dv), packed(dgate), packed(dbeta)


def exact(case, seed):
    s = prepare(case, seed)
    lens = _lengths(case)
    if case["kind"] == "delta":
        return _exact_delta(s, case, lens)
    if case["mode"] != "decode" and case["n"] > 600:
        return _exact_pairs(s, case, lens)
    return _exact_attention(s, case, lens)
