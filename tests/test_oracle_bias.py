"""The oracle of attention with a learned bias by buckets, pinned (CPU) against autograd and differences; the buckets themselves."""
import math

import pytest
import torch

import budgetformer_amd as bf
from budgetformer_amd.sequences import PackedSequences
from oracle import sequences as sq

LENS = ([3, 0, 5, 1, 6], [4, 2, 5, 7, 3])


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    monkeypatch.setattr(PackedSequences, "_device", staticmethod(torch.device))


def _bucket(x):
    return x.clamp(-2, 2) + 2


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_equal_autograd_and_differences(causal):
    g = torch.Generator().manual_seed(0)
    n_q, n_k = sum(LENS[0]), sum(LENS[1])
    q, do = (torch.randn(n_q, 4, 6, generator=g).double() for _ in range(2))
    k, v = (torch.randn(n_k, 2, 6, generator=g).double() for _ in range(2))
    table = torch.randn(4, 5, generator=g).double()

    def value(q, k, v, table):
        total, q0, k0 = 0.0, 0, 0
        for m, n in zip(*LENS):
            see = sq.visible(m, n, causal)
            if m and n:
                for h in range(4):
                    s = q[q0:q0 + m, h] @ k[k0:k0 + n, h // 2].T * 0.3
                    s = s + torch.stack([torch.stack([table[h, max(-2, min(2, j - (i + n - m))) + 2] for j in range(n)]) for i in range(m)])
                    p = torch.where(see.any(1, keepdim=True), s.masked_fill(~see, -math.inf), torch.zeros_like(s)).softmax(1)
                    total = total + (((p * see.any(1, keepdim=True)) @ v[k0:k0 + n, h // 2]) * do[q0:q0 + m, h]).sum()
            q0, k0 = q0 + m, k0 + n
        return total

    got = sq.attention(q, k, v, *LENS, causal, 0.3, do, table=table, bucket=_bucket)
    args = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
    for name, r in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(value(*args), args)):
        assert torch.allclose(got[name], r, rtol=1e-12, atol=1e-12), name
    way = torch.randn(4, 5, generator=g).double()
    ends = [(sq.attention(q, k, v, *LENS, causal, 0.3, table=table + s * 1e-5 * way, bucket=_bucket)["out"] * do).sum() for s in (1, -1)]
    assert abs((ends[0] - ends[1]) / 2e-5 - (got["dtable"] * way).sum()) < 1e-7     # h^2 f'''/6 and float64's 1e-11 over h


def test_a_table_of_zeros_changes_nothing():
    q = torch.randn(5, 2, 4, generator=torch.Generator().manual_seed(1)).double()
    a = sq.attention(q, q, q, [5], [5], True, 0.5, q)
    b = sq.attention(q, q, q, [5], [5], True, 0.5, q, table=torch.zeros(2, 5).double(), bucket=_bucket)
    assert all(torch.equal(a[x], b[x]) for x in a)


@pytest.mark.parametrize("buckets,far,both", [(32, 128, True), (32, 128, False), (64, 500, True), (2, 2, False), (4, 3, True), (10, 100, False)])
def test_buckets_are_as_their_definition(buckets, far, both):
    got = bf.RelativeBuckets(buckets, far, bidirectional=both, device="cpu")
    n = buckets // 2 if both else buckets
    e = n // 2
    for x in range(-2 * far, 2 * far + 1):
        away, base = (abs(x), n if x > 0 else 0) if both else (max(-x, 0), 0)
        if away < e:
            want = away
        else:                                    # well off a border, logarithms tell
            t = (n - e) * math.log(away / e) / math.log(far / e)
            if abs(t - round(t)) < 1e-9:
                continue
            want = min(e + int(t), n - 1)
        assert got.of(x) == base + want, x
    assert got.of(-far) == n - 1 and got.of(-e if e else 0) == e
    assert got.map.tolist() == list(got.by_distance) and got.map.dtype == torch.int32
    assert got.reach < far or far <= 3
    assert got.to("cpu").of(-1) == got.of(-1)


def test_borders_are_exact():
    """Powers of two of 16 buckets up to 128: bucket 8 + 2 k begins at 8 2^k, where a quotient of logarithms may fall short."""
    got = bf.RelativeBuckets(16, 128, bidirectional=False, device="cpu")
    assert [got.of(-x) for x in (8, 15, 16, 31, 32, 63, 64, 127, 128)] == [8, 9, 10, 11, 12, 13, 14, 15, 15]


def test_maps():
    got = bf.RelativeBuckets.from_map([3, 3, 1, 0, 2, 2, 2], device="cpu")
    assert got.buckets == 4 and got.reach == 2 and [got.of(x) for x in (-9, -2, -1, 0, 1, 2, 9)] == [3, 3, 1, 0, 2, 2, 2]
    assert bf.RelativeBuckets.from_map([0], device="cpu").reach == 0
    for bad in ([0, 1], [], [0, -1, 0]):
        with pytest.raises(ValueError):
            bf.RelativeBuckets.from_map(bad, device="cpu")
    with pytest.raises(NotImplementedError, match="64"):
        bf.RelativeBuckets.from_map([0] * 10 + [64], device="cpu")
    with pytest.raises(NotImplementedError, match="1024"):
        bf.RelativeBuckets.from_map([0] * 1025 + [1] * 1024 + [0, 1], device="cpu")
    for kw in (dict(buckets=1), dict(buckets=5), dict(buckets=2), dict(buckets=32, far=8), dict(buckets=4, far=0, bidirectional=False)):
        with pytest.raises(ValueError):
            bf.RelativeBuckets(**kw, device="cpu")
    with pytest.raises(NotImplementedError, match="begins"):
        bf.RelativeBuckets(32, 100000, device="cpu")
