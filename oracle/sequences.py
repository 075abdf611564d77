"""CPU oracle of the operators over packed sequences — TEST INFRASTRUCTURE ONLY.

Everything in float64 from the definitions, one sequence after the other: softmax attention with its closed-form
gradients, rotary positions as complex numbers, linear attention as its recurrence. Pinned in
tests/test_oracle_sequences.py against autograd and central differences.

The ``*_bound`` values are how far a kernel may be off, from its roundings alone: u is half a step of the
activations' type (a value's rounding), c32 bounds the float32 arithmetic of a sum of so many terms.
"""
from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _tiny(dtype) -> float:
    """Half a step of the type's subnormal numbers: the rounding of values too small for a relative one."""
    return 2.0 ** -25 if dtype == torch.float16 else 1e-38


def visible(m: int, n: int, causal: bool, device=None):
    """[m, n] truth values: row i sees key j; with causal the last row stands at the last key."""
    j, i = torch.arange(n, device=device), torch.arange(m, device=device)[:, None]
    return j <= i + (n - m) if causal else torch.ones(m, n, dtype=torch.bool, device=device)


def attention(q, k, v, q_lens, k_lens, causal, scale, dout=None, dtype=None, operand_tiny=None,
              rounds=True, table=None, bucket=None):
    """q [n_q, H, d], k, v [n_k, Hk, d] float64 packed. Returns a dict: out, lse (natural log) and with dout dq, dk, dv;
    with dtype also each one's bound (``out_bound``, ...). Rows that see no key: out 0, lse -inf. operand_tiny: half a step
    of a subnormal P or dS, where that is finer than the type's own. rounds: whether P and dS are operands of the type and
    Delta comes from the rounded out (False: neither; Delta as good as from out and its rounding's rest, rounded itself).
    table [H, buckets] float64 and bucket, a function of distances (a key's place less the row's): scores get table[h, bucket],
    and with dout there is dtable. Its bound takes a Delta from out and its rounding's rest, with P in two parts: a row's dS add
    up to 0, and a sum over a bucket shows what is off in it."""
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = H // Hk
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else [])
    if table is not None and dout is not None:
        names.append("dtable")
    res = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v),
           "lse": q.new_full(q.shape[:2], -math.inf)}
    bnd = {x: torch.zeros_like(res[x]) for x in ("out", "dq", "dk", "dv")}
    if table is not None:
        res["dtable"], bnd["dtable"] = torch.zeros_like(table), torch.zeros_like(table)
    u = half_step(dtype) if dtype is not None else 0.0
    up = 0.0 if dtype == torch.float32 or not rounds else u      # P and dS as operands: rounded to the type
    tiny = _tiny(dtype)
    small = 0.0 if not rounds else tiny if operand_tiny is None else operand_tiny
    q0 = k0 = 0
    for m, n in zip(q_lens, k_lens):
        rows, keys = slice(q0, q0 + m), slice(k0, k0 + n)
        q0, k0 = q0 + m, k0 + n
        if m == 0 or n == 0:
            continue
        see = visible(m, n, causal, q.device)
        if table is not None:
            at = bucket(torch.arange(n, device=q.device) - torch.arange(n - m, n, device=q.device)[:, None])
        for h in range(H):
            a, b, w = q[rows, h], k[keys, h // g], v[keys, h // g]
            s = a @ b.T * scale
            if table is not None:
                s = s + table[h][at]
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True).clamp(min=-1e300)
            p = (s - top).exp()
            z = p.sum(1, keepdim=True)
            p = torch.where(z > 0, p / z.clamp(min=1e-300), torch.zeros_like(p))
            out = torch.where(p[..., None] > 0, p[..., None] * w, torch.zeros((), dtype=p.dtype, device=p.device)).sum(1) \
                if not torch.isfinite(w).all() else p @ w
            res["out"][rows, h] = out
            res["lse"][rows, h] = torch.where(z[:, 0] > 0, top[:, 0] + z[:, 0].log(), -math.inf)
            if dtype is None and dout is None:
                continue
            big = scale * (a.abs() @ b.abs().T).masked_fill(~see, 0).amax() if see.any() else 0.0
            if table is not None and see.any():
                big = big + table[h][at].masked_fill(~see | ~torch.isfinite(table[h][at]), 0).abs().amax()
            # scores: sums of d products, each step off by 2^-24, scaled; their exponentials' relative error, the sums over n
            c32 = 2.0 ** -24 * (2 * (d + 8) * (1 + float(big)) + n + m * g + 32)
            ob = u * out.abs() + (up + c32) * (p @ w.abs()) + small * (see.double() @ w.abs()) + tiny
            bnd["out"][rows, h] = ob
            if dout is None:
                continue
            do = dout[rows, h]
            dp = do @ w.T
            ds = p * (dp - (do * out).sum(1, keepdim=True))
            if table is not None:
                ob2 = (0.0 if dtype == torch.float32 else 2 * u * u) * (out.abs() + p @ w.abs()) + c32 * (p @ w.abs()) + tiny
                off = c32 * ds.abs() + p * ((do.abs() * ob2).sum(1, keepdim=True) + 2 * c32 * (do.abs() @ w.abs().T))
                for x in range(table.shape[1]):
                    res["dtable"][h, x] += ds[at == x].sum()
                    bnd["dtable"][h, x] += off[at == x].sum() + 2.0 ** -20 * ds[at == x].abs().sum()     # a column's up to some 300 additions
            res["dq"][rows, h] = scale * ds @ b
            res["dk"][keys, h // g] += scale * ds.T @ a
            res["dv"][keys, h // g] += p.T @ do
            if not rounds:
                ob = u * u * out.abs() + c32 * (p @ w.abs()) + tiny
            mean_off = (do.abs() * ob).sum(1, keepdim=True)       # Delta comes from the rounded out
            e = (up + c32) * ds.abs() + p * (mean_off + 2 * c32 * (do.abs() @ w.abs().T)) + small * see
            bnd["dq"][rows, h] = scale * (e + c32 * ds.abs()) @ b.abs()
            bnd["dk"][keys, h // g] += scale * (e + c32 * ds.abs()).T @ a.abs()
            bnd["dv"][keys, h // g] += ((up + 2 * c32) * p + small * see).T @ do.abs()
    for x in ("dq", "dk", "dv"):
        bnd[x] += u * res[x].abs() + tiny
    got = {x: res[x] for x in names + ["lse"]}
    if dtype is not None:
        got.update({f"{x}_bound": bnd[x] for x in names})
    return got


def rotary(x, positions, theta, amplitude, interleaved, inverse=False):
    """x [n, heads, d] float64, theta float64 [rot / 2] radians a position: pairs as complex numbers, turned."""
    rot = 2 * theta.numel()
    angle = positions.double()[:, None] * theta
    turn = torch.polar(torch.full_like(angle, amplitude), -angle if inverse else angle)[:, None]
    head, rest = x[..., :rot], x[..., rot:]
    pairs = head.unflatten(-1, (rot // 2, 2)) if interleaved else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    got = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    got = got if interleaved else got.transpose(-1, -2)
    return torch.cat([got.flatten(-2), rest], -1)


def linear_attention(q, k, v, log_decay, lens, scale, initial_state=None, dout=None, dtype=None, operand_tiny=None):
    """The recurrence S_i = g S_{i-1} + k_i v_i^T, out_i = scale q_i S_i, a token at a time; q, k [n, H, dk], v [n, H, dv]
    float64. Returns a dict: out, state [sequences, H, dk, dv], with dout dq, dk, dv (the same recurrence on the way
    back), and with dtype the bounds, from the recurrence over absolute values. operand_tiny: half a step of a subnormal
    operand (the scores, the state), where that is finer than the type's own."""
    H, dk, dv = q.shape[1], q.shape[2], v.shape[2]
    g = log_decay.double().exp()[:, None, None]
    res = {"out": torch.zeros_like(v), "state": q.new_zeros(len(lens), H, dk, dv)}
    size = {"out": torch.zeros_like(v), "state": torch.zeros_like(res["state"])}     # sums of absolute values
    seen = {"out": torch.zeros_like(v)}                                              # undecayed, for subnormal roundings
    if dout is not None:
        for x, like in (("dq", q), ("dk", k), ("dv", v)):
            res[x], size[x], seen[x] = torch.zeros_like(like), torch.zeros_like(like), torch.zeros_like(like)
    at = 0
    for b, n in enumerate(lens):
        s = q.new_zeros(H, dk, dv) if initial_state is None else initial_state[b].double().clone()
        sa, su = s.abs(), s.abs()
        for t in range(at, at + n):
            kv = k[t][:, :, None] * v[t][:, None, :]
            s, sa, su = g * s + kv, g * sa + kv.abs(), su + k[t].abs()[:, :, None] + v[t].abs()[:, None, :]
            res["out"][t] = scale * torch.einsum("hk,hkv->hv", q[t], s)
            size["out"][t] = scale * torch.einsum("hk,hkv->hv", q[t].abs(), sa)
            seen["out"][t] = scale * torch.einsum("hk,hkv->hv", q[t].abs() + 1, su)
            if dout is not None:
                res["dq"][t] = scale * torch.einsum("hkv,hv->hk", s, dout[t])
                size["dq"][t] = scale * torch.einsum("hkv,hv->hk", sa, dout[t].abs())
                seen["dq"][t] = scale * torch.einsum("hkv,hv->hk", su, dout[t].abs() + 1)
        res["state"][b], size["state"][b] = s, sa
        if dout is not None:
            r = q.new_zeros(H, dk, dv)
            ra, ru = r.clone(), r.clone()
            for t in range(at + n - 1, at - 1, -1):
                qd = q[t][:, :, None] * dout[t][:, None, :]
                r, ra, ru = g * r + qd, g * ra + qd.abs(), ru + q[t].abs()[:, :, None] + dout[t].abs()[:, None, :]
                res["dk"][t] = scale * torch.einsum("hkv,hv->hk", r, v[t])
                res["dv"][t] = scale * torch.einsum("hkv,hk->hv", r, k[t])
                size["dk"][t] = scale * torch.einsum("hkv,hv->hk", ra, v[t].abs())
                size["dv"][t] = scale * torch.einsum("hkv,hk->hv", ra, k[t].abs())
                seen["dk"][t] = scale * torch.einsum("hkv,hv->hk", ru, v[t].abs() + 1)
                seen["dv"][t] = scale * torch.einsum("hkv,hk->hv", ru, k[t].abs() + 1)
        at += n
    if dtype is not None:
        u = half_step(dtype)
        # operands rounded to the type: the scores W, the state, and the decayed z that enters it
        up = 0.0 if dtype == torch.float32 else 3 * u
        c32 = 2.0 ** -24 * (max(list(lens) + [1]) + 2 * (dk + dv) + 256)
        for x in list(seen):
            small = _tiny(dtype) if operand_tiny is None else operand_tiny
            res[f"{x}_bound"] = u * res[x].abs() + (up + c32) * size[x] + small * seen[x] + _tiny(dtype)
        res["state_bound"] = (up / 3 + c32) * size["state"] + _tiny(dtype) * max(list(lens) + [1]) * 8
    return res


def gated_delta(q, k, v, log_gate, beta, lens, scale, initial_state=None, dout=None):
    """S' = exp(g) S, e = v - S'^T k, S = S' + b k e^T, out = scale S^T q, a token at a time; q, k [n, Hk, dk], v [n, H, dv], log_gate
    and beta [n, H] float64. Returns a dict: out, state [sequences, H, dk, dv], with dout dq, dk, dv, dlog_gate, dbeta (the
    recurrence's own way back), and ``terms``: of each tensor how large the terms of its sums are, by sequence and head."""
    H, group = v.shape[1], v.shape[1] // k.shape[1]
    qh, kh = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    dk, dv = q.shape[2], v.shape[2]
    res = {"out": torch.zeros_like(v), "state": q.new_zeros(len(lens), H, dk, dv)}
    if dout is not None:
        res.update(dq=torch.zeros_like(qh), dk=torch.zeros_like(qh), dv=torch.zeros_like(v),
                   dlog_gate=torch.zeros_like(log_gate), dbeta=torch.zeros_like(beta))
    at = 0
    for b, n in enumerate(lens):
        s = q.new_zeros(H, dk, dv) if initial_state is None else initial_state[b].double().clone()
        kept = []
        for t in range(at, at + n):
            before = s * log_gate[t].exp()[:, None, None]
            e = v[t] - torch.einsum("hkv,hk->hv", before, kh[t])
            s = before + kh[t][:, :, None] * (beta[t][:, None] * e)[:, None, :]
            res["out"][t] = scale * torch.einsum("hkv,hk->hv", s, qh[t])
            kept.append((before, e, s))
        res["state"][b] = s
        if dout is not None:
            r = torch.zeros_like(s)
            for t in range(at + n - 1, at - 1, -1):
                before, e, s = kept.pop()
                do = scale * dout[t]
                r = r + qh[t][:, :, None] * do[:, None, :]
                res["dq"][t] = torch.einsum("hkv,hv->hk", s, do)
                du = torch.einsum("hkv,hk->hv", r, kh[t])
                res["dbeta"][t] = (du * e).sum(-1)
                res["dv"][t] = beta[t][:, None] * du
                res["dk"][t] = torch.einsum("hkv,hv->hk", r, beta[t][:, None] * e)
                r = r - kh[t][:, :, None] * res["dv"][t][:, None, :]
                res["dk"][t] -= torch.einsum("hkv,hv->hk", before, res["dv"][t])
                res["dlog_gate"][t] = (r * before).sum((1, 2))
                r = r * log_gate[t].exp()[:, None, None]
        at += n
    # a gate's gradient is a sum over a chunk of products of q and k with their gradients, and of the states' with theirs
    most = {x: torch.zeros(len(lens), y.shape[1], dtype=torch.float64) for x, y in res.items()}
    at = 0
    for b, n in enumerate(lens):
        for x, y in res.items():
            rows = y[b:b + 1] if x == "state" else y[at:at + n]
            if rows.numel():
                most[x][b] = rows.abs().movedim(1, 0).flatten(1).amax(1).cpu()
        if dout is not None and n:
            products = (qh[at:at + n] * res["dq"][at:at + n]).abs().sum(-1) + (kh[at:at + n] * res["dk"][at:at + n]).abs().sum(-1)
            most["dlog_gate"][b] += 32 * products.amax(0).cpu()
        at += n
    if dout is not None:
        for x in ("dq", "dk"):
            res[x] = res[x].unflatten(1, (-1, group)).sum(2)
            most[x] = most[x].unflatten(1, (-1, group)).sum(2)
    res["terms"] = most
    return res


def gated_delta_bound(res, name, lens, dtype):
    """How far a kernel's ``name`` may be off for keys of at most unit length and strengths of 0 to 2, whose chunk inverses have
    entries of at most 2 and whose state transitions shrink what is off already. Operands in two bfloat16 parts are off by 2^-18
    each, and their product leaves 2^-18 out: 2^-17 together at most (float32's three parts: 2^-25, less than the 2^-24 of each of
    a sum's additions, of some sqrt(320) independent ones: 2^-20). Independent roundings of a chunk of 32 tokens and of a
    sequence's chunks add up as a root; an inverse's row of 32 entries and three products in a row amplify by 16 at most. float16 and
    bfloat16 results are rounded besides."""
    y = res[name]
    eta = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -17
    u = 0.0 if name in ("state", "dlog_gate", "dbeta") else half_step(dtype)
    size = torch.zeros_like(y)
    at = 0
    for b, n in enumerate(lens):
        rows = slice(b, b + 1) if name == "state" else slice(at, at + n)
        most = res["terms"][name][b].to(y.device)
        size[rows] = most.view(1, -1, *([1] * (y.dim() - 2)))
        at += n
    return u * y.abs() + 16 * eta * math.sqrt(32 + max(list(lens) + [1])) * size + _tiny(dtype)
