"""The oracle of the gated delta rule, pinned (CPU): against the rule's other form (a product of transitions), its gradients
against autograd and central differences."""
import pytest
import torch

from oracle import sequences as sq

LENS = [4, 0, 1, 7]


def _inputs(H=4, Hk=2, dk=6, dv=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = sum(LENS)
    r = lambda *s: torch.randn(*s, generator=g).double()                       # noqa: E731
    return r(n, Hk, dk), r(n, Hk, dk) / dk ** 0.5, r(n, H, dv), -r(n, H).exp(), r(n, H).sigmoid(), r(n, H, dv), r(len(LENS), H, dk, dv)


def _by_transitions(q, k, v, g, b, init, scale):
    """S <- exp(g) (1 - b k k^T) S + b k v^T."""
    outs, states, at = [], [], 0
    for x, n in enumerate(LENS):
        s = init[x]
        for t in range(at, at + n):
            kk = k[t].repeat_interleave(2, 0)
            step = torch.eye(k.shape[2]).double() - b[t][:, None, None] * kk[:, :, None] * kk[:, None, :]
            s = g[t].exp()[:, None, None] * (step @ s) + b[t][:, None, None] * kk[:, :, None] * v[t][:, None, :]
            outs.append(scale * (s.transpose(1, 2) @ q[t].repeat_interleave(2, 0)[:, :, None])[..., 0])
        states.append(s)
        at += n
    return torch.stack(outs), torch.stack(states)


def test_forms_and_gradients():
    q, k, v, g, b, do, init = _inputs()
    got = sq.gated_delta(q, k, v, g, b, LENS, 0.3, init, do)
    args = [x.clone().requires_grad_(True) for x in (q, k, v, g, b)]
    out, state = _by_transitions(*args, init, 0.3)
    assert torch.allclose(got["out"], out, rtol=1e-12, atol=1e-12) and torch.allclose(got["state"], state, rtol=1e-12, atol=1e-12)
    names = ("dq", "dk", "dv", "dlog_gate", "dbeta")
    for name, r in zip(names, torch.autograd.grad(out, args, do)):
        assert torch.allclose(got[name], r, rtol=1e-11, atol=1e-12), name
    # a central difference along a direction: off by h^2 f'''/6, some 1e-9 at h = 1e-5 and float64's 1e-11
    for i, name in enumerate(names):
        way = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()
        ends = [(sq.gated_delta(*[x + s * 1e-5 * way if j == i else x for j, x in enumerate((q, k, v, g, b))], LENS, 0.3, init)["out"]
                 * do).sum() for s in (1, -1)]
        assert abs((ends[0] - ends[1]) / 2e-5 - (got[name] * way).sum()) < 1e-7, name


def test_strength_one_stores_what_unit_keys_read_back():
    q, k, v, g, b, _, _ = _inputs()
    k = k / k.norm(dim=-1, keepdim=True)
    got = sq.gated_delta(k, k, v, g, torch.ones_like(b), LENS, 1.0)
    assert torch.allclose(got["out"], v, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("gate", [0.0, -float("inf")])
def test_gates_at_their_ends(gate):
    q, k, v, g, b, _, _ = _inputs()
    got = sq.gated_delta(q, k, v, torch.full_like(g, gate), b, LENS, 1.0)["out"]
    own = (q * k).sum(-1).repeat_interleave(2, 1)[..., None] * b[..., None] * v
    if gate == 0.0:
        want = sq.linear_attention(q.repeat_interleave(2, 1), 1e-6 * k.repeat_interleave(2, 1), v * b[..., None],
                                   torch.zeros(4), LENS, 1e6)["out"]             # corrections of 1e-12 of it
        got = sq.gated_delta(q, 1e-6 * k, v, g * 0, b, LENS, 1e6)["out"]
        assert torch.allclose(got, want, rtol=1e-9, atol=1e-9)
    else:
        assert torch.allclose(got, own, rtol=1e-12, atol=1e-12)
