"""The gated delta rule on the GPU against the float64 oracle, each value within what its roundings allow (oracle/sequences.py)."""
import math

import pytest
import torch

from oracle import sequences as sq

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("out", "dq", "dk", "dv", "dlog_gate", "dbeta")


def _bf():
    import budgetformer_amd as bf
    return bf


def _inputs(dev, n, H, Hk, dk, dv, dtype, seed=0, most=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                 # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6) * 0.99    # noqa: E731  at most 1 rounded too
    return [x.to(dev) for x in (unit(r(n, Hk, dk)).to(dtype), unit(r(n, Hk, dk)).to(dtype), r(n, H, dv).to(dtype),
                                -(r(n, H) * 1.5 - 3).exp().log1p(), most * r(n, H).sigmoid(), r(n, H, dv).to(dtype))]


def _within(name, got, ref, bound):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    off = (got.double().cpu() - ref).abs()
    bad = ~(off <= bound)                                 # a NaN is bad too
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst "
                                 f"{float((off / bound.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} times the bound")


def _check(got, args, lens, dtype, scale, init=None, do=None):
    """got: a dict of results; args: the inputs they came from."""
    ref = sq.gated_delta(*(x.double().cpu() for x in args), lens, scale, None if init is None else init.cpu(),
                         None if do is None else do.double().cpu())
    for name, x in got.items():
        _within(name, x, ref[name], sq.gated_delta_bound(ref, name, lens, dtype))


def _case(dev, lens, H, Hk, dk, dv, dtype, seed=0, init=False, train=True, most=1.0, tail=0):
    bf = _bf()
    n = sum(lens) + tail
    *args, do = _inputs(dev, n, H, Hk, dk, dv, dtype, seed, most)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=dev) if not tail else bf.PackedSequences.from_offsets(
        torch.tensor([0] + lens).cumsum(0).to(dev), n_q=n, causal=True)
    s0 = torch.randn(len(lens), H, dk, dv, generator=torch.Generator().manual_seed(seed + 9)).to(dev) if init else None
    leaves = [x.clone().requires_grad_(train) for x in args]
    out = bf.gated_delta_rule(*leaves, seqs, initial_state=s0, return_state=init)
    got = {}
    if init:
        out, got["state"] = out
    got["out"] = out.detach()
    if train:
        got.update(zip(NAMES[1:], torch.autograd.grad(out, leaves, do)))
    if tail:                                              # rows behind the last sequence: nothing
        for name, x in got.items():
            if name != "state":
                assert not bool(x[-tail:].any()), name
                got[name] = x[:-tail]
        args, do = [x[:-tail] for x in args], do[:-tail]
    _check(got, args, lens, dtype, dk ** -0.5, s0, do if train else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("init", [False, True])
@pytest.mark.parametrize("lens", [[1], [5] * 40, [33, 0, 64, 65, 1, 128, 31], [0, 0, 17, 0], [32] * 3], ids=["one", "walks", "mixed", "empty", "chunks"])
def test_lengths(hip_device, lens, init, dtype):
    _case(hip_device, lens, 2, 2, 32, 32, dtype, seed=31, init=init)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,dk,dv", [(2, 2, 8, 8), (3, 1, 16, 24), (4, 2, 40, 64), (2, 1, 64, 32), (2, 2, 128, 128), (3, 3, 72, 128), (4, 1, 128, 16)])
def test_head_layouts(hip_device, H, Hk, dk, dv, dtype):
    _case(hip_device, [70, 3, 90], H, Hk, dk, dv, dtype, seed=37)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("init", [False, True])
@pytest.mark.parametrize("dk,dv", [(16, 16), (64, 40), (128, 128)])
def test_states_from_segment_to_segment(hip_device, dk, dv, init, dtype):
    """Sequences of several segments beside short and empty ones, a segment's end at a sequence's."""
    _case(hip_device, [700, 50, 256, 0, 6, 128, 500], 2, 1, dk, dv, dtype, seed=41, init=init)


@pytest.mark.parametrize("lens", [[4200], [2000, 2100]])
def test_many_segments(hip_device, lens):
    _case(hip_device, lens, 1, 1, 32, 32, torch.float32, seed=43)
    _case(hip_device, lens, 1, 1, 32, 32, torch.bfloat16, seed=43, init=True, train=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [1, 300])
def test_rows_behind_the_last_sequence(hip_device, tail, dtype):
    _case(hip_device, [150, 0, 40], 4, 2, 32, 64, dtype, seed=47, tail=tail)
    _case(hip_device, [15, 9], 2, 2, 16, 16, dtype, seed=48, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strengths_up_to_two(hip_device, dtype):
    _case(hip_device, [100, 37], 2, 2, 32, 32, dtype, seed=53, most=2.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_and_strengths_at_their_ends(hip_device, dtype):
    """Gates of 1, that empty the state, and far below what float32 holds; strengths of 0 and 1; a key that repeats (whose chunk
    inverse has entries of 1 where a product of powers would have passed 1e8)."""
    bf, lens = _bf(), [200, 45]
    *args, do = _inputs(hip_device, 245, 2, 2, 32, 32, dtype, 59)
    args[3][:70, 0] = 0.0
    args[3][70:75] = -math.inf
    args[3][90] = -1000.0
    args[3][100:140] = -90.0
    args[4][::3], args[4][1::3] = 0.0, 1.0
    args[1][150:200] = args[1][150:151]
    args[4][150:200, 0] = 1.0
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    leaves = [x.clone().requires_grad_(True) for x in args]
    out, state = bf.gated_delta_rule(*leaves, seqs, return_state=True)
    got = dict(zip(NAMES, [out.detach(), *torch.autograd.grad(out, leaves, do)]), state=state)
    # where a gate is 0 exp(gate) is, and with it its gradient: what the kernel takes 0 from is 2^-216 of it
    _check(got, args, lens, dtype, 32 ** -0.5, do=do)


def test_strides_and_casts(hip_device):
    """Slices of a fused projection, expanded heads, k and v of another type, gates in bfloat16 with their gradients."""
    bf = _bf()
    fused = torch.randn(90, 3, 2, 32, generator=torch.Generator().manual_seed(3)).to(hip_device)
    q, k, v = (fused / fused.norm(dim=-1, keepdim=True)).unbind(1)
    k = k[:, :1].expand(90, 2, 32)
    *_, g, b, do = _inputs(hip_device, 90, 2, 2, 32, 32, torch.float32, 61)
    seqs = bf.PackedSequences.from_lengths([60, 30], causal=True, device=hip_device)

    def run(*x):
        leaves = [y.detach().clone().requires_grad_(True) if i > 2 else y.detach().requires_grad_(True) for i, y in enumerate(x)]
        out = bf.gated_delta_rule(*leaves, seqs)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    views, plain = run(q, k, v, g, b), run(q.contiguous(), k.contiguous(), v.contiguous(), g, b)
    for x, y in zip(views, plain):
        assert torch.equal(x, y)
    narrow = run(q, k.bfloat16(), v.half(), g.bfloat16(), b.bfloat16())
    wide = run(q, k.bfloat16().float(), v.half().float(), g.bfloat16().float(), b.bfloat16().float())
    assert [x.dtype for x in narrow[1:]] == [torch.float32, torch.bfloat16, torch.float16, torch.bfloat16, torch.bfloat16]
    for x, y in zip(narrow, wide):
        assert torch.equal(x, y.to(x.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,Hk,dk,dv", [(1, 16, 16, 128, 128), (5, 4, 2, 64, 32), (3, 3, 1, 8, 24), (64, 2, 2, 40, 128)])
def test_step(hip_device, n, H, Hk, dk, dv, dtype):
    bf = _bf()
    *args, _ = _inputs(hip_device, n, H, Hk, dk, dv, dtype, 67)
    s = torch.randn(n, H, dk, dv, generator=torch.Generator().manual_seed(5)).to(hip_device)
    out, new = bf.gated_delta_step(*args, s)
    _check({"out": out, "state": new}, args, [1] * n, dtype, dk ** -0.5, s)
    strided = [torch.stack([x, x], 1)[:, 1] for x in args[:3]]
    into = s.clone()
    got, same = bf.gated_delta_step(*strided, *args[3:], into, out_state=into)
    assert same.data_ptr() == into.data_ptr() and torch.equal(got, out) and torch.equal(into, new)
    whole, last = bf.gated_delta_rule(*args, bf.PackedSequences.from_lengths([1] * n, causal=True, device=hip_device), initial_state=s,
                                      return_state=True)
    _check({"out": whole, "state": last}, args, [1] * n, dtype, dk ** -0.5, s)


def test_step_states_that_overlap(hip_device):
    bf = _bf()
    room = torch.zeros(4, 2, 16, 16, device=hip_device)
    *args, _ = _inputs(hip_device, 2, 2, 2, 16, 16, torch.float32, 71)
    with pytest.raises(ValueError, match="overlaps state"):
        bf.gated_delta_step(*args, room[:2], out_state=room[1:3])
    with pytest.raises(ValueError, match="overlaps an input"):
        bf.gated_delta_step(*args[:4], room[2].view(-1)[:4].view(2, 2), room[:2], out_state=room[2:])
    with pytest.raises(ValueError, match="state must be"):
        bf.gated_delta_step(*args, room)


@pytest.mark.parametrize("where", ["v", "k", "q", "log_gate", "beta"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_not_finite_reach_what_follows_alone(hip_device, where, bad):
    """Rows before, other sequences and (of v) other columns, as without it; rows from it on NaN."""
    bf, lens, at = _bf(), [40, 150, 33], 40 + 77
    *args, _ = _inputs(hip_device, 223, 2, 2, 64, 64, torch.bfloat16, 73)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    clean, state = bf.gated_delta_rule(*args, seqs, return_state=True)
    i = ("q", "k", "v", "log_gate", "beta").index(where)
    args[i] = args[i].clone()
    args[i][(at, 1, 5) if i < 3 else (at, 1)] = bad
    out, after = bf.gated_delta_rule(*args, seqs, return_state=True)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[at:190 if where != "q" else at + 1, 1, slice(5, 6) if where == "v" else slice(None)] = True
    assert torch.equal(out[~hit], clean[~hit])
    assert not bool(torch.isfinite(out[hit]).any())
    lost = torch.zeros_like(after, dtype=torch.bool)
    if where != "q":
        lost[1, 1, :, slice(5, 6) if where == "v" else slice(None)] = True
    assert torch.equal(after[~lost], state[~lost])


def test_gradients_of_other_sequences_beside_one_that_is_not_finite(hip_device):
    bf, lens = _bf(), [40, 300, 33]
    *args, do = _inputs(hip_device, 373, 2, 1, 32, 32, torch.float16, 79)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)

    def run(x):
        leaves = [y.clone().requires_grad_(True) for y in x]
        out = bf.gated_delta_rule(*leaves, seqs)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    clean = run(args)
    args[1] = args[1].clone()
    args[1][200] = math.nan
    for x, y in zip(run(args), clean):
        assert torch.equal(x[:40], y[:40]) and torch.equal(x[340:], y[340:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_equal_differences(hip_device, dtype):
    """A direction's central difference of float32 calls against the gradients of the type: off by h^2 f'''/6 (some 1e-4 of it at
    h = 0.01), by float32's 2^-20 of the values over h, and by the gradients' own rounding."""
    bf, lens = _bf(), [130, 20]
    *args, do = _inputs(hip_device, 150, 2, 1, 32, 32, dtype, 83)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    leaves = [x.clone().requires_grad_(True) for x in args]
    grads = torch.autograd.grad(bf.gated_delta_rule(*leaves, seqs), leaves, do)
    wide = [x.float() for x in args]
    for i, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).to(hip_device)
        way = way / way.norm()
        ends = [(bf.gated_delta_rule(*[x + s * 0.01 * way if j == i else x for j, x in enumerate(wide)], seqs).double() * do.double()).sum()
                for s in (1, -1)]
        got, want = (g.double() * way.double()).sum(), (ends[0] - ends[1]) / 0.02
        size = g.double().norm()
        assert abs(got - want) <= size * (sq.half_step(dtype) + 2e-3) + 2.0 ** -20 * do.double().norm() * 10, (i, got, want)


def test_calls_repeat_and_replay(hip_device):
    """Forward and backward captured into a graph and replayed between eager work: the eager results, bit for bit."""
    bf, lens = _bf(), [300, 7, 180]
    *args, do = _inputs(hip_device, 487, 4, 2, 64, 64, torch.bfloat16, 89)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    leaves = [x.clone().requires_grad_(True) for x in args]

    def run():
        out, state = bf.gated_delta_rule(*leaves, seqs, return_state=True)
        return [out.detach(), state, *torch.autograd.grad(out, leaves, do)]

    want = run()
    for x, y in zip(run(), want):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        for x, y in zip(run(), want):
            assert torch.equal(x, y)


def test_another_stream(hip_device):
    bf = _bf()
    *args, do = _inputs(hip_device, 400, 2, 2, 32, 32, torch.float16, 97)
    want = bf.gated_delta_rule(*args, bf.PackedSequences.from_lengths([250, 150], causal=True, device=hip_device))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    seqs = bf.PackedSequences.from_lengths([250, 150], causal=True, device=hip_device)
    with torch.cuda.stream(side):
        got = bf.gated_delta_rule(*args, seqs)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(hip_device):
    bf = _bf()
    q, k, v, g, b, _ = _inputs(hip_device, 20, 2, 2, 16, 16, torch.float32, 101)
    seqs = bf.PackedSequences.from_lengths([20], causal=True, device=hip_device)
    run = bf.gated_delta_rule
    with pytest.raises(ValueError, match="causal"):
        run(q, k, v, g, b, bf.PackedSequences.from_lengths([20], device=hip_device))
    with pytest.raises(ValueError, match="same rows"):
        run(q, k, v, g, b, bf.PackedSequences.from_lengths([20], [20], causal=True, device=hip_device))
    with pytest.raises(ValueError, match="cover"):
        run(q[:10], k[:10], v[:10], g[:10], b[:10], seqs)
    with pytest.raises(ValueError, match="log_gate must be"):
        run(q, k, v, g[:, :1], b, seqs)
    with pytest.raises(ValueError, match="disagree"):
        run(q, k[:, :1], v, g, b, seqs)
    with pytest.raises(ValueError, match="multiple"):
        run(q, k, v[:, :1], g[:, :1], b[:, :1], seqs)
    with pytest.raises(NotImplementedError, match="head dims"):
        run(q[..., :12].contiguous(), k[..., :12].contiguous(), v, g, b, seqs)
    state = torch.zeros(1, 2, 16, 16, device=hip_device)
    with pytest.raises(ValueError, match="init_state must be"):
        run(q, k, v, g, b, seqs, initial_state=state[:, :1])
    with pytest.raises(NotImplementedError, match="constant"):
        run(q, k, v, g, b, seqs, initial_state=state.requires_grad_(True))
    out = run(q.requires_grad_(True), k, v, g, b, seqs)
    grad, = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        grad.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            run(q.detach(), k, v, fwd.make_dual(g, torch.ones_like(g)), b, seqs)


def test_no_tokens(hip_device):
    bf = _bf()
    *args, do = _inputs(hip_device, 0, 2, 2, 16, 16, torch.float32, 103)
    state = torch.randn(3, 2, 16, 16, device=hip_device)
    seqs = bf.PackedSequences.from_lengths([0, 0, 0], causal=True, device=hip_device)
    leaves = [x.requires_grad_(True) for x in args]
    out, after = bf.gated_delta_rule(*leaves, seqs, initial_state=state, return_state=True)
    assert out.shape == (0, 2, 16) and torch.equal(after, state)
    assert [x.shape for x in torch.autograd.grad(out, leaves, do)] == [x.shape for x in leaves]
    none = bf.PackedSequences.from_lengths([], causal=True, device=hip_device)
    out, after = bf.gated_delta_rule(*args, none, return_state=True)
    assert out.numel() == 0 and after.shape == (0, 2, 16, 16)


@pytest.mark.parametrize("check", [True, False])
def test_rows_of_no_sequence(hip_device, check):
    bf = _bf()
    *args, do = _inputs(hip_device, 2500, 2, 2, 16, 16, torch.float32, 107)
    offsets = torch.zeros(1, dtype=torch.int32, device=hip_device)
    seqs = bf.PackedSequences.from_offsets(offsets, n_q=2500, causal=True, check=check)
    leaves = [x.requires_grad_(True) for x in args]
    out, after = bf.gated_delta_rule(*leaves, seqs, return_state=True)
    assert after.shape == (0, 2, 16, 16)
    assert not any(bool(x.any()) for x in (out, *torch.autograd.grad(out, leaves, do)))
    with torch.no_grad():
        assert not bool(bf.gated_delta_rule(*args, seqs).any())
