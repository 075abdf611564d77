"""Attention with a learned bias by buckets on the GPU against the float64 oracle, each value within the bound that its own roundings
give, and a layer of it beside the gated delta rule."""
import math

import pytest
import torch

from oracle import sequences as sq

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _bf():
    import budgetformer_amd as bf
    return bf


def _randn(seed, *shape, dtype=torch.float32, dev="cuda"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def _within(name, got, ref, bound):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    off = (got.double() - ref).abs()
    bad = ~(off <= bound)                                 # a NaN is bad too
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst "
                                 f"{float((off / bound.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} times the bound")


def _of(buckets, dev):
    by = torch.tensor(buckets.by_distance, device=dev)
    return lambda x: by[x.clamp(-buckets.reach, buckets.reach) + buckets.reach]


def _case(dev, q_lens, k_lens, H, Hk, d, causal, dtype, buckets=None, seed=0, train=True, table=None, sizes=(1.0, 1.0, 1.0, 1.0)):
    bf = _bf()
    buckets = bf.RelativeBuckets(16, 40, device=dev) if buckets is None else buckets
    n_q, n_k = sum(q_lens), sum(k_lens)
    q, do = ((s * _randn(seed + i, n_q, H, d, dev=dev)).to(dtype) for i, s in ((0, sizes[0]), (3, sizes[3])))
    k, v = ((s * _randn(seed + i, n_k, Hk, d, dev=dev)).to(dtype) for i, s in ((1, sizes[1]), (2, sizes[2])))
    table = _randn(seed + 4, H, buckets.buckets, dev=dev) if table is None else table
    seqs = bf.PackedSequences.from_lengths(q_lens, k_lens, causal=causal, device=dev)
    leaves = [x.clone().requires_grad_(train) for x in (q, k, v, table)]
    out, lse = bf.packed_attention(*leaves[:3], seqs, with_lse=True, bias=leaves[3], buckets=buckets)
    ref = sq.attention(q.double(), k.double(), v.double(), q_lens, k_lens, causal, d ** -0.5, do.double() if train else None, dtype,
                       table=table.double(), bucket=_of(buckets, dev), operand_tiny=2.0 ** -34 if dtype == torch.float16 else None)
    _within("out", out.detach(), ref["out"], ref["out_bound"])
    fin = torch.isfinite(ref["lse"])
    assert torch.equal(fin, torch.isfinite(lse))
    if bool(fin.any()):                                   # a sum of exponentials in float32 and its log: the scores' error and a step of the result
        score = d ** -0.5 * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) + float(table[torch.isfinite(table)].abs().max())
        assert float((lse.double() - ref["lse"])[fin].abs().max()) < 2.0 ** -24 * (8 * (d + 8) * (1 + score) + max(k_lens) + 64)
    if train:
        for name, got in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do)):
            _within(name, got, ref[name], ref[f"{name}_bound"])
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[1], [5] * 40, [33, 0, 64, 65, 1, 128, 31], [200, 313], [0, 0, 17, 0], [129] * 3],
                         ids=["one", "walks", "mixed", "long", "empty", "edges"])
def test_lengths(hip_device, lens, causal, dtype):
    _case(hip_device, lens, lens, 4, 2, 32, causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 8, 16), (3, 1, 8), (6, 2, 24), (4, 4, 64), (5, 5, 40), (2, 1, 72), (8, 2, 128), (7, 1, 128), (40, 1, 16),
                                    (66, 2, 8)])
def test_head_layouts(hip_device, H, Hk, d, dtype):
    """Groups of every kind beside a wave's 32 rows: parts of them, one, more than one wave holds."""
    _case(hip_device, [70, 3, 131], [70, 3, 131], H, Hk, d, True, dtype, seed=7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_rows_and_keys_of_different_lengths(hip_device, causal, dtype):
    """Rows stand behind their sequence's earlier keys; more rows than keys: before the first one."""
    _case(hip_device, [1, 40, 100, 0, 9, 64], [300, 200, 37, 12, 0, 64], 4, 2, 64, causal, dtype, seed=11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64), (3, 1, 16)])
def test_single_tokens_against_kept_keys(hip_device, H, Hk, d, dtype):
    k_lens = [1, 0, 63, 64, 65, 777, 2050, 5, 128]
    _case(hip_device, [1] * len(k_lens), k_lens, H, Hk, d, True, dtype, seed=13, train=False)
    _case(hip_device, [1], [4099], H, Hk, d, True, dtype, seed=17, train=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_train_against_long_keys(hip_device, dtype):
    _case(hip_device, [7, 3], [1500, 1201], 4, 1, 64, True, dtype, seed=19)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("lens,causal", [([1300, 1, 517, 0, 230, 7], True), ([700, 551], False)], ids=["causal", "all"])
def test_long_sequences_in_whole_rows(hip_device, lens, causal, d, dtype):
    """Workgroups over whole rows, tiles in order, blocks nearer and farther than the reach on both sides."""
    _case(hip_device, lens, lens, 32, 16, d, causal, dtype, seed=37)


def _is_short(lens, k_lens, H, Hk, d, dtype, buckets):
    """Whether the call's rows are walked by a few lanes each (16-bit types then keep no rest for the backward)."""
    import ctypes as C
    from budgetformer_amd import _native as N
    code = {torch.bfloat16: N.BF_DTYPE_BF16, torch.float16: N.BF_DTYPE_F16}[dtype]
    a = N.PackedAttn(n_q=sum(lens), n_k=sum(k_lens), heads_q=H, heads_k=Hk, head_dim=d, dtype=code, row_span=64, key_span=64, scale=1.0,
                     longest=max(list(lens) + list(k_lens)))
    b = N.PackedBias(table=64, map=64, positions=64, buckets=buckets.buckets, reach=buckets.reach)
    return not N.load().bf_packed_attn_bias_rest(C.byref(a), C.byref(b))


SHORT = [5, 1, 24, 0, 17, 8, 23, 2, 13, 7, 24, 3]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,d", [(8, 8, 16), (3, 3, 8), (4, 2, 24), (6, 1, 32), (2, 2, 128)])
def test_short_sequences(hip_device, H, Hk, d, causal, dtype):
    bf = _bf()
    lens = [min(n, 40 * Hk // H) for n in SHORT]          # the heads of a group share a row's lanes' time
    for buckets in (bf.RelativeBuckets(8, 16, device=hip_device), bf.RelativeBuckets.from_map([1, 0, 2], device=hip_device),
                    bf.RelativeBuckets.from_map([(7 * x) % 13 for x in range(101)], device=hip_device)):
        if dtype != torch.float32:
            assert _is_short(lens, lens, H, Hk, d, dtype, buckets)
        _case(hip_device, lens, lens, H, Hk, d, causal, dtype, buckets=buckets, seed=23)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_short_rows_and_keys_of_different_lengths(hip_device, causal, dtype):
    _case(hip_device, [3, 9, 0, 20, 1, 12], [11, 4, 6, 0, 24, 12], 4, 4, 16, causal, dtype, seed=29)


def test_short_tables_that_leave_no_room(hip_device):
    """Groups times buckets past what a workgroup keeps of short sequences: whole tiles."""
    bf = _bf()
    buckets = bf.RelativeBuckets(64, 200, device=hip_device)
    lens = [min(n, 2) for n in SHORT]
    assert _is_short(lens, lens, 4, 4, 16, torch.bfloat16, buckets) and not _is_short(lens, lens, 16, 1, 16, torch.bfloat16, buckets)
    _case(hip_device, lens, lens, 16, 1, 16, True, torch.bfloat16, buckets=buckets, seed=31)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 8, 16), (6, 3, 16)])
def test_short_sequences_in_many_ranges(hip_device, H, Hk, d, dtype):
    """More rows than the workgroups take at once: every repeat of a batch gives its rows' results, and the table's gradient is the
    sum of theirs (a column's additions are up to some thousand, each off by 2^-24 of a sum that stays below their absolute one)."""
    bf, times = _bf(), 600
    lens, n = SHORT, sum(SHORT)
    buckets = bf.RelativeBuckets(16, 40, device=hip_device)
    q, do = (_randn(61 + i, n, H, d, dtype=dtype, dev=hip_device) for i in range(2))
    k, v = (_randn(63 + i, n, Hk, d, dtype=dtype, dev=hip_device) for i in range(2))
    table = _randn(65, H, 16, dev=hip_device)

    def run(m):
        seqs = bf.PackedSequences.from_lengths(lens * m, device=hip_device)
        leaves = [x.repeat(m, 1, 1).requires_grad_(True) for x in (q, k, v)] + [table.clone().requires_grad_(True)]
        out = bf.packed_attention(*leaves[:3], seqs, bias=leaves[3], buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, do.repeat(m, 1, 1))]

    one, many = run(1), run(times)
    for a, b in zip(one[:4], many[:4]):
        assert torch.equal(b.view(times, n, *b.shape[1:]), a.expand(times, *a.shape))
    # sums of at most 24 * 24 pairs of each sequence and repeat: of absolute values a few times the largest entry
    size = times * float(one[4].abs().max()) + times * 12.0
    assert float((many[4].double() - times * one[4].double()).abs().max()) <= 2.0 ** -24 * 2000 * size / 10


def _maps():
    bf = _bf()
    return {"none": lambda dev: bf.RelativeBuckets.from_map([0], device=dev), "one": lambda dev: bf.RelativeBuckets.from_map([2, 0, 1], device=dev),
            "random": lambda dev: bf.RelativeBuckets.from_map(torch.randint(0, 64, (131,), generator=torch.Generator().manual_seed(1)).tolist(), device=dev),
            "each": lambda dev: bf.RelativeBuckets.from_map(list(range(63)), device=dev),
            "far": lambda dev: bf.RelativeBuckets.from_map([min(x // 33, 63) for x in range(2049)], device=dev),
            "log": lambda dev: bf.RelativeBuckets(64, 500, device=dev), "before": lambda dev: bf.RelativeBuckets(32, 128, bidirectional=False, device=dev)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["none", "one", "random", "each", "far", "log", "before"])
def test_maps(hip_device, name, dtype):
    """Any map: neighbouring distances in different buckets, all in one, the largest reach."""
    _case(hip_device, [330, 5, 96], [330, 5, 96], 4, 2, 32, False, dtype, buckets=_maps()[name](hip_device), seed=41)
    _case(hip_device, [3, 40], [1500, 41], 2, 2, 128, True, dtype, buckets=_maps()[name](hip_device), seed=43)


def test_the_most_that_a_workgroup_holds(hip_device):
    """Seven heads of a group over 1024 distances (64 KB) in the largest kernels."""
    for dtype in DTYPES:
        _case(hip_device, [300, 41], [300, 41], 7, 1, 128, False, dtype, buckets=_maps()["far"](hip_device), seed=47)


@pytest.mark.parametrize("dtype", DTYPES)
def test_buckets_that_are_not_seen(hip_device, dtype):
    """A bucket of -inf hides its keys: those rows that see others as without them; rows that see none: out 0, lse -inf, no gradient."""
    bf = _bf()
    buckets = bf.RelativeBuckets.from_map([3, 1, 2, 0, 3], device=hip_device)            # far, -1, 0, +1, far
    table = _randn(3, 4, 4, dev=hip_device)
    table[:, 3] = -math.inf
    table[1, 1] = table[1, 2] = -math.inf                                                # head 1: of each row its next key alone
    table[2] = -math.inf                                                                 # head 2: nothing
    _case(hip_device, [70, 1, 40], [70, 1, 40], 4, 2, 32, False, dtype, buckets=buckets, table=table, seed=53)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0, 1e-4), (0.1, 0.1, 100.0, 100.0)], ids=["small", "large"])
def test_gradients_of_any_size(hip_device, sizes, dtype):
    """float16's units of dS change within a row; the table's gradient is not in them."""
    _case(hip_device, [600, 33], [600, 33], 2, 2, 32, True, dtype, seed=59, sizes=sizes)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_a_row_does_not_see(hip_device, dtype):
    """NaN and infinities in other sequences, later keys and rows behind the last sequence leave a row and the table's gradient as they
    are."""
    bf = _bf()
    lens, n = [70, 45], 130
    buckets = bf.RelativeBuckets(8, 16, device=hip_device)
    off = torch.tensor([0, 70, 115], device=hip_device)
    seqs = bf.PackedSequences.from_offsets(off, n_q=n, causal=True)
    q, k, v, do = (_randn(61 + i, n, 2, 32, dtype=dtype, dev=hip_device) for i in range(4))
    table = _randn(67, 2, 8, dev=hip_device)

    def run(*x):
        leaves = [y.clone().requires_grad_(True) for y in (*x, table)]
        out = bf.packed_attention(*leaves[:3], seqs, bias=leaves[3], buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    clean = run(q, k, v)
    assert not bool(clean[0][115:].any()) and not any(bool(g[115:].any()) for g in clean[1:4])
    behind = [x.clone() for x in (q, k, v)]
    for x, bad in zip(behind, (math.nan, math.inf, -math.inf)):
        x[115:] = bad
    for a, b in zip(run(*behind), clean):
        assert torch.equal(a, b)
    last = [x.clone() for x in (q, k, v)]
    last[1][69], last[2][69] = math.nan, math.inf                     # the first sequence's last key: its last row sees it
    got = run(*last)
    rows = [r for r in range(n) if r != 69]
    assert torch.equal(got[0][rows], clean[0][rows]) and bool(torch.isnan(got[0][69]).all())
    assert torch.equal(got[1][70:], clean[1][70:]) and torch.equal(got[2][70:], clean[2][70:])


def test_calls_repeat_and_replay(hip_device):
    bf = _bf()
    lens = [300, 7, 180, 64]
    q, k, v, do = (_randn(71 + i, 551, 4, 64, dtype=torch.bfloat16, dev=hip_device) for i in range(4))
    table = _randn(75, 4, 32, dev=hip_device).requires_grad_(True)
    buckets = bf.RelativeBuckets(32, 100, device=hip_device)
    seqs = bf.PackedSequences.from_lengths(lens, device=hip_device)
    leaves = [x.requires_grad_(True) for x in (q, k, v)] + [table]

    def run():
        out = bf.packed_attention(*leaves[:3], seqs, bias=table, buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    want = run()
    for a, b in zip(run(), want):
        assert torch.equal(a, b)
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
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(run(), want):
            assert torch.equal(a, b)


def test_types_of_the_table_and_strides(hip_device):
    bf = _bf()
    fused = _randn(81, 90, 3, 4, 32, dev=hip_device)
    buckets = bf.RelativeBuckets(8, 16, device=hip_device)
    seqs = bf.PackedSequences.from_lengths([60, 30], device=hip_device)
    table = _randn(82, 8, 4, dev=hip_device)

    def run(q, k, v, t):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, t)]
        out = bf.packed_attention(*leaves[:3], seqs, bias=leaves[3], buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out.float().square().sum(), leaves)]

    q, k, v = fused.unbind(1)
    for a, b in zip(run(q, k, v, table.T), run(q.contiguous(), k.contiguous(), v.contiguous(), table.T.contiguous())):
        assert torch.equal(a, b)
    narrow = run(q, k, v, table.T.bfloat16())
    wide = run(q, k, v, table.T.bfloat16().float())
    assert narrow[4].dtype == torch.bfloat16 and torch.equal(narrow[4], wide[4].bfloat16()) and torch.equal(narrow[0], wide[0])
    only = table.T.clone().requires_grad_(True)                       # q, k and v as constants
    out = bf.packed_attention(q, k, v, seqs, bias=only, buckets=buckets)
    assert torch.equal(torch.autograd.grad(out.float().square().sum(), only)[0], run(q, k, v, table.T)[4])


def test_gradients_equal_differences(hip_device):
    """A direction's central difference of float32 calls: off by h^2 f'''/6 (some 1e-4 of it at h = 0.01) and by the sums' float32
    rounding over h."""
    bf = _bf()
    q, k, v, do = (_randn(91 + i, 150, 2, 32, dev=hip_device) for i in range(4))
    table = _randn(95, 2, 16, dev=hip_device)
    buckets = bf.RelativeBuckets(16, 40, device=hip_device)
    seqs = bf.PackedSequences.from_lengths([130, 20], device=hip_device)
    leaves = [x.requires_grad_(True) for x in (q, k, v, table)]
    grads = torch.autograd.grad(bf.packed_attention(*leaves[:3], seqs, bias=table, buckets=buckets), leaves, do)
    base = [x.detach() for x in leaves]
    for i, g in enumerate(grads):
        way = _randn(96 + i, *g.shape, dev=hip_device)
        way = way / way.norm()
        ends = []
        for s in (1, -1):
            x = [y + s * 0.01 * way if j == i else y for j, y in enumerate(base)]
            ends.append((bf.packed_attention(*x[:3], seqs, bias=x[3], buckets=buckets).double() * do.double()).sum())
        got, want = (g.double() * way.double()).sum(), (ends[0] - ends[1]) / 0.02
        assert abs(got - want) <= 2e-3 * g.double().norm() + 2.0 ** -20 * do.double().norm() * 10, (i, got, want)


def test_nothing_to_see(hip_device):
    bf = _bf()
    buckets = bf.RelativeBuckets(8, 16, device=hip_device)
    table = torch.ones(2, 8, device=hip_device, requires_grad=True)
    for n_q, n_k in ((0, 0), (0, 5), (5, 0)):
        q = torch.zeros(n_q, 2, 16, device=hip_device, requires_grad=True)
        k = torch.zeros(n_k, 2, 16, device=hip_device, requires_grad=True)
        seqs = bf.PackedSequences.from_lengths([n_q], [n_k], device=hip_device)
        out = bf.packed_attention(q, k, k, seqs, bias=table, buckets=buckets)
        g = torch.autograd.grad(out.sum(), (q, k, table))
        assert not any(bool(x.any()) for x in (out, *g)) and g[2].shape == (2, 8)


def test_refusals(hip_device):
    bf = _bf()
    x = _randn(97, 20, 2, 16, dev=hip_device)
    seqs = bf.PackedSequences.from_lengths([20], device=hip_device)
    buckets = bf.RelativeBuckets(8, 16, device=hip_device)
    table = torch.zeros(2, 8, device=hip_device)
    for kw, error, match in ((dict(bias=table), ValueError, "together"), (dict(buckets=buckets), ValueError, "together"),
                             (dict(bias=table[:, :7], buckets=buckets), ValueError, "bias must be"), (dict(bias=table[:1], buckets=buckets), ValueError, "bias must be"),
                             (dict(bias=table, buckets=[0] * 33), TypeError, "RelativeBuckets"), (dict(bias=table.cpu(), buckets=buckets), ValueError, "bias")):
        with pytest.raises(error, match=match):
            bf.packed_attention(x, x, x, seqs, **kw)
    ops = torch.ops.bf
    with pytest.raises(ValueError, match="map must be"):
        ops.packed_attn_bias_fwd(x, x, x, table, buckets.map[:-1], seqs.positions(), seqs.row_span, 0.25)
    with pytest.raises(ValueError, match="positions must be"):
        ops.packed_attn_bias_fwd(x, x, x, table, buckets.map, seqs.positions()[1:], seqs.row_span, 0.25)
    out = bf.packed_attention(x, x, x, seqs, bias=table.requires_grad_(True), buckets=buckets)
    grad, = torch.autograd.grad(out.sum(), table, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        grad.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            bf.packed_attention(x, x, x, seqs, bias=fwd.make_dual(table.detach(), table.detach()), buckets=buckets)


def test_maps_that_name_no_bucket_stay_inside_the_table(hip_device):
    """A map given to the operator itself is clamped to the table's buckets."""
    bf = _bf()
    x = _randn(99, 40, 2, 16, dev=hip_device)
    seqs = bf.PackedSequences.from_lengths([40], device=hip_device)
    table = _randn(98, 2, 4, dev=hip_device)
    wild = torch.tensor([-5, 0, 1, 2, 9], dtype=torch.int32, device=hip_device)
    tame = torch.tensor([0, 0, 1, 2, 3], dtype=torch.int32, device=hip_device)
    a, b = (torch.ops.bf.packed_attn_bias_fwd(x, x, x, table, m, seqs.positions(), seqs.row_span, 0.25)[0] for m in (wild, tame))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer(hip_device, dtype):
    """CoreAttention's flash type with a learned bias, made on the host and moved: attention of its own inputs, and the parameter's
    gradient."""
    bf = _bf()
    layer = bf.CoreAttention(64, 0.0, 4, buckets=bf.RelativeBuckets(8, 16, device=hip_device)).to(hip_device)
    with torch.no_grad():
        layer.relative_bias.copy_(_randn(101, 4, 8, dev=hip_device))
    q, k, v, do = (_randn(102 + i, 3, 50, 4, 16, dtype=dtype, dev=hip_device) for i in range(4))
    out = layer(q, k, v, attn_type="flash")
    rows = [x.reshape(150, 4, 16).double() for x in (q, k, v, do)]
    ref = sq.attention(*rows[:3], [50] * 3, [50] * 3, False, 0.25, rows[3], dtype, table=layer.relative_bias.detach().double(),
                       bucket=_of(layer.buckets, hip_device), operand_tiny=2.0 ** -34 if dtype == torch.float16 else None)
    _within("out", out.detach().reshape(150, 4, 16), ref["out"], ref["out_bound"])
    out.backward(do.reshape(3, 50, 64))
    _within("relative_bias", layer.relative_bias.grad, ref["dtable"], ref["dtable_bound"])


def test_hybrid_stack_trains_and_replays(hip_device):
    """What a hybrid model runs over one batch: a gated delta layer, then attention with rotary positions and a learned bias, then
    linear attention; gradients of everything, eager and in a replayed graph, against float32's autograd of the same stack's pieces."""
    bf = _bf()
    lens, n, H, d = [40, 0, 130, 77], 247, 4, 32
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    freq = bf.RotaryFrequencies(d, device=hip_device)
    buckets = bf.RelativeBuckets(16, 64, bidirectional=False, device=hip_device)
    x = _randn(111, n, H, d, dtype=torch.bfloat16, dev=hip_device).requires_grad_(True)
    gate = (-_randn(112, n, H, dev=hip_device).exp()).requires_grad_(True)
    beta = _randn(113, n, H, dev=hip_device).sigmoid().requires_grad_(True)
    table = _randn(114, H, 16, dev=hip_device).requires_grad_(True)
    decay = -torch.arange(H, device=hip_device) * 0.1
    do = _randn(115, n, H, d, dtype=torch.bfloat16, dev=hip_device)

    def run():
        k = torch.nn.functional.normalize(x.float(), dim=-1).to(x.dtype)
        y = bf.gated_delta_rule(k, k, x, gate, beta, seqs)
        q, kr = bf.rotary_embedding(y, x, freq, seqs=seqs)
        y = bf.packed_attention(q, kr, x, seqs, bias=table, buckets=buckets)
        y = bf.linear_attention(y, k, x, decay, seqs)
        return [y.detach(), *torch.autograd.grad(y, (x, gate, beta, table), do)]

    want = run()
    assert all(bool(torch.isfinite(w).all()) and bool(w.any()) for w in want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    # one sequence alone gives its rows' results: nothing crosses
    rows = slice(40, 170)
    part = [y.detach()[rows].clone().requires_grad_(True) for y in (x, gate, beta)]
    alone = bf.PackedSequences.from_lengths([130], causal=True, device=hip_device)
    k = torch.nn.functional.normalize(part[0].float(), dim=-1).to(x.dtype)
    y = bf.gated_delta_rule(k, k, part[0], part[1], part[2], alone)
    q, kr = bf.rotary_embedding(y, part[0], freq, seqs=alone)
    y = bf.linear_attention(bf.packed_attention(q, kr, part[0], alone, bias=table, buckets=buckets), k, part[0], decay, alone)
    assert float((y.detach().double() - want[0][rows].double()).abs().max()) <= 4 * sq.half_step(torch.bfloat16) * float(want[0].double().abs().max())
