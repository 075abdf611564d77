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
              rounds=True):
    """q [n_q, H, d], k, v [n_k, Hk, d] float64 packed. Returns a dict: out, lse (natural log) and with dout dq, dk, dv;
    with dtype also each one's bound (``out_bound``, ...). Rows that see no key: out 0, lse -inf. operand_tiny: half a step
    of a subnormal P or dS, where that is finer than the type's own. rounds: whether P and dS are operands of the type and
    Delta comes from the rounded out (False: neither; Delta as good as from out and its rounding's rest, rounded itself)."""
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = H // Hk
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else [])
    res = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v),
           "lse": q.new_full(q.shape[:2], -math.inf)}
    bnd = {x: torch.zeros_like(res[x]) for x in ("out", "dq", "dk", "dv")}
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
        for h in range(H):
            a, b, w = q[rows, h], k[keys, h // g], v[keys, h // g]
            s = (a @ b.T * scale).masked_fill(~see, -math.inf)
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
            # scores: sums of d products, each step off by 2^-24, scaled; their exponentials' relative error, the sums over n
            c32 = 2.0 ** -24 * (2 * (d + 8) * (1 + float(big)) + n + m * g + 32)
            ob = u * out.abs() + (up + c32) * (p @ w.abs()) + small * (see.double() @ w.abs()) + tiny
            bnd["out"][rows, h] = ob
            if dout is None:
                continue
            do = dout[rows, h]
            dp = do @ w.T
            ds = p * (dp - (do * out).sum(1, keepdim=True))
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
