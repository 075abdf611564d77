"""The oracle of the operators over packed sequences, pinned (CPU): its gradients against autograd of the same formula
and against central differences, its forms against each other."""
import math

import pytest
import torch

from oracle import sequences as sq

LENS = ([3, 0, 5, 1], [4, 2, 5, 7])


def _inputs(H=4, Hk=2, d=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    n_q, n_k = sum(LENS[0]), sum(LENS[1])
    return (torch.randn(n_q, H, d, generator=g).double(), torch.randn(n_k, Hk, d, generator=g).double(),
            torch.randn(n_k, Hk, d, generator=g).double(), torch.randn(n_q, H, d, generator=g).double())


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_equal_autograd_and_differences(causal):
    q, k, v, do = _inputs()

    def value(q, k, v):
        total, q0, k0 = 0.0, 0, 0
        for m, n in zip(*LENS):
            if m and n:
                see = sq.visible(m, n, causal)
                for h in range(4):
                    s = (q[q0:q0 + m, h] @ k[k0:k0 + n, h // 2].T * 0.3).masked_fill(~see, -math.inf)
                    total = total + ((s.softmax(1) @ v[k0:k0 + n, h // 2]) * do[q0:q0 + m, h]).sum()
            q0, k0 = q0 + m, k0 + n
        return total

    got = sq.attention(q, k, v, *LENS, causal, 0.3, do)
    args = [x.clone().requires_grad_(True) for x in (q, k, v)]
    ref = torch.autograd.grad(value(*args), args)
    for name, r in zip(("dq", "dk", "dv"), ref):
        assert torch.allclose(got[name], r, rtol=1e-12, atol=1e-12), name
    # a central difference along a direction: off by h^2 f'''/6, some 1e-9 at h = 1e-5 and float64's 1e-11
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()
        ends = []
        for sign in (1, -1):
            moved = [x + sign * 1e-5 * way if j == i else x for j, x in enumerate((q, k, v))]
            ends.append((sq.attention(*moved, *LENS, causal, 0.3)["out"] * do).sum())
        assert abs((ends[0] - ends[1]) / 2e-5 - (got[name] * way).sum()) < 1e-7, name


def test_attention_of_rows_without_keys_is_zero():
    q, k, v, do = _inputs()
    got = sq.attention(q[:3], k[:1], v[:1], [3], [1], True, 1.0, do[:3])       # only the last row stands at a key
    assert torch.equal(got["out"][:2], torch.zeros(2, 4, 6).double()) and bool((got["lse"][:2] == -math.inf).all())
    assert torch.equal(got["out"][2], v[0].repeat_interleave(2, 0)) and bool((got["dq"][:2] == 0).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_turns_pairs_and_back(interleaved):
    x = torch.randn(5, 2, 10, generator=torch.Generator().manual_seed(1)).double()
    theta = torch.tensor([1.0, 0.1, 0.003]).double()
    pos = torch.tensor([0, 1, -7, 10 ** 6, 2 ** 40])
    y = sq.rotary(x, pos, theta, 1.5, interleaved)
    assert torch.allclose(sq.rotary(y, pos, theta, 1 / 1.5, interleaved, inverse=True), x, atol=1e-12)
    i, j = (2, 3) if interleaved else (1, 4)                                   # the second pair
    c, s = math.cos(-0.7), math.sin(-0.7)
    assert torch.allclose(y[2, :, i], 1.5 * (x[2, :, i] * c - x[2, :, j] * s), atol=1e-12)
    assert torch.allclose(y[2, :, j], 1.5 * (x[2, :, i] * s + x[2, :, j] * c), atol=1e-12)
    assert torch.equal(y[..., 6:], x[..., 6:])


def test_linear_attention_recurrence_equals_its_quadratic_form_and_gradients():
    g = torch.Generator().manual_seed(2)
    lens, H, dk, dv = [4, 0, 7, 1], 2, 3, 5
    q, k = (torch.randn(12, H, dk, generator=g).double() for _ in range(2))
    v, do = (torch.randn(12, H, dv, generator=g).double() for _ in range(2))
    s0 = torch.randn(4, H, dk, dv, generator=g).double()
    ld = torch.tensor([-0.1, -1.3])
    got = sq.linear_attention(q, k, v, ld, lens, 0.7, s0, do)
    args = [x.clone().requires_grad_(True) for x in (q, k, v)]
    total, at, outs = 0.0, 0, []
    for b, n in enumerate(lens):
        a, c, w = (x[at:at + n].transpose(0, 1) for x in args)
        i = torch.arange(n).double()
        decay = (ld.double()[:, None, None] * (i[:, None] - i)).exp().tril()
        into = (ld.double()[:, None] * (i + 1)).exp()[..., None]
        o = 0.7 * (((a @ c.transpose(1, 2)) * decay) @ w + into * (a @ s0[b]))
        outs.append(o.transpose(0, 1))
        total = total + (o * do[at:at + n].transpose(0, 1)).sum()
        at += n
    assert torch.allclose(got["out"], torch.cat(outs), atol=1e-12)
    for name, r in zip(("dq", "dk", "dv"), torch.autograd.grad(total, args)):
        assert torch.allclose(got[name], r, atol=1e-12), name
    assert torch.equal(got["state"][1], s0[1])
