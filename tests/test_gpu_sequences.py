"""The operators over packed sequences on the GPU against the float64 oracle, each value within the bound that its own
roundings give (oracle/sequences.py derives them; half a step of the type is torch.finfo(t).eps / 2)."""
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


def _attention_case(dev, q_lens, k_lens, H, Hk, d, causal, dtype, seed=0, scale=None, train=True):
    bf = _bf()
    n_q, n_k = sum(q_lens), sum(k_lens)
    q, do = (_randn(seed + i, n_q, H, d, dtype=dtype, dev=dev) for i in (0, 3))
    k, v = (_randn(seed + i, n_k, Hk, d, dtype=dtype, dev=dev) for i in (1, 2))
    seqs = bf.PackedSequences.from_lengths(q_lens, k_lens, causal=causal, device=dev)
    leaves = [x.clone().requires_grad_(train) for x in (q, k, v)]
    out, lse = bf.packed_attention(*leaves, seqs, scale=scale, with_lse=True)
    ref = sq.attention(q.double(), k.double(), v.double(), q_lens, k_lens, causal, d ** -0.5 if scale is None else scale,
                       do.double() if train else None, dtype)
    _within("out", out.detach(), ref["out"], ref["out_bound"])
    # lse: a sum of exponentials in float32 and its log: the scores' error and a step of the result
    fin = torch.isfinite(ref["lse"])
    assert torch.equal(fin, torch.isfinite(lse))
    if bool(fin.any()):
        assert float((lse.double() - ref["lse"])[fin].abs().max()) < 2.0 ** -24 * (
            8 * (d + 8) * (1 + float((q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()))) + max(k_lens) + 64)
    if train:
        grads = torch.autograd.grad(out, leaves, do)
        for name, got in zip(("dq", "dk", "dv"), grads):
            _within(name, got, ref[name], ref[f"{name}_bound"])
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[1], [5] * 40, [33, 0, 64, 65, 1, 128, 31], [200, 313], [0, 0, 17, 0], [129] * 3],
                         ids=["one", "walks", "mixed", "long", "empty", "edges"])
def test_packed_attention_self(hip_device, lens, causal, dtype):
    _attention_case(hip_device, lens, lens, 4, 2, 32, causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 8, 16), (3, 1, 8), (6, 2, 24), (4, 4, 64), (5, 5, 40), (2, 1, 72), (8, 2, 128),
                                    (7, 1, 128)])
def test_packed_attention_head_layouts(hip_device, H, Hk, d, dtype):
    _attention_case(hip_device, [70, 3, 131], [70, 3, 131], H, Hk, d, True, dtype, seed=7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_packed_attention_rows_and_keys_of_different_lengths(hip_device, causal, dtype):
    """More keys than rows (a chunk behind kept keys), more rows than keys (causal rows that see nothing), sequences
    without rows or without keys."""
    _attention_case(hip_device, [1, 40, 100, 0, 9, 64], [300, 200, 37, 12, 0, 64], 4, 2, 64, causal, dtype, seed=11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64), (3, 1, 16)])
def test_single_tokens_against_kept_keys(hip_device, H, Hk, d, dtype):
    """One row a sequence, few rows in all: the keys are cut into pieces, which are joined."""
    k_lens = [1, 0, 63, 64, 65, 777, 2050, 5, 128]
    _attention_case(hip_device, [1] * len(k_lens), k_lens, H, Hk, d, True, dtype, seed=13, train=False)
    _attention_case(hip_device, [1], [4099], H, Hk, d, True, dtype, seed=17, train=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_train_against_long_keys(hip_device, dtype):
    _attention_case(hip_device, [7, 3], [1500, 1201], 4, 1, 64, True, dtype, seed=19)


def test_whole_rows_of_many_tiles(hip_device):
    """Enough rows that every key head's tiles take whole rows (no pieces), one long sequence among short ones."""
    _attention_case(hip_device, [2500, 1, 300, 77], [2500, 1, 300, 77], 32, 16, 64, True, torch.bfloat16, seed=23)


def _scratch_floats(lens, H, Hk, d, dtype):
    """What the forward asks for: 0 for whole rows in the order they lie, 8192 with the tiles put in order, else pieces."""
    import ctypes as C
    from budgetformer_amd import _native as N
    code = {torch.float32: N.BF_DTYPE_F32, torch.bfloat16: N.BF_DTYPE_BF16, torch.float16: N.BF_DTYPE_F16}[dtype]
    a = N.PackedAttn(n_q=sum(lens), n_k=sum(lens), heads_q=H, heads_k=Hk, head_dim=d, dtype=code, row_span=64, key_span=64,
                     scale=1.0, longest=max(lens))
    return N.load().bf_packed_attn_fwd_floats(C.byref(a))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("lens,causal,floats", [([1300, 1, 517, 0, 230, 7], True, 8192), ([2051], True, 0), ([300] * 13 + [259], True, 0),
                                                ([700, 1351], False, 8192)], ids=["mixed", "one", "many", "all"])
def test_whole_rows_of_every_type_and_head_size(hip_device, lens, causal, floats, d, dtype):
    """No pieces: the workgroups of two and four waves over whole rows, with tiles that end anywhere, put in order or not."""
    H, Hk = 32, 16
    assert _scratch_floats(lens, H, Hk, d, dtype) == floats
    _attention_case(hip_device, lens, lens, H, Hk, d, causal, dtype, seed=37)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("d", [16, 64, 128])
def test_the_backward_reads_what_rounding_left(hip_device, d, dtype):
    """Values of 8 and a little: Delta from the rounded out is off by out's rounding, some 2^3 half-steps of the type a
    value. With `rest` what is left comes from the rounding of P, which is as large a part of each of 400 to 1000 terms
    and averages out over them: less than a quarter."""
    ops, bf, n, H = torch.ops.bf, _bf(), 1000, 2
    q, k, do = (_randn(i, n, H, d, dtype=dtype, dev=hip_device) for i in (0, 1, 3))
    v = (8 + 0.25 * _randn(2, n, H, d, dev=hip_device)).to(dtype)
    seqs = bf.PackedSequences.from_lengths([n], device=hip_device)
    out, lse, rest = ops.packed_attn_fwd(q, k, v, seqs.row_span, d ** -0.5, n, True)
    ref = sq.attention(q.double(), k.double(), v.double(), [n], [n], False, d ** -0.5, do.double())
    off = []
    for r in (rest, None):
        got = ops.packed_attn_bwd(q, k, v, seqs.row_span, seqs.key_span, out, lse, do, d ** -0.5, n, r)
        off.append([float((x.double() - ref[name]).norm()) for x, name in zip(got, ("dq", "dk"))])
    assert rest.shape == out.shape and off[0][0] < off[1][0] / 4 and off[0][1] < off[1][1] / 4, off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_few_key_tiles_seen_by_many_rows(hip_device, d, dtype):
    """A group of four heads over one: the key tiles' rows are cut into pieces, whose sums are joined."""
    _attention_case(hip_device, [1603], [1603], 4, 1, d, True, dtype, seed=29)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d,lens", [(32, 2, 128, [5] * 60), (16, 1, 64, [100] * 4 + [37]), (8, 1, 16, [12, 24, 3] * 20)])
def test_key_tiles_of_several_sequences_in_pieces(hip_device, H, Hk, d, lens, dtype):
    """Few key tiles, each of several sequences whose rows are cut into pieces."""
    _attention_case(hip_device, lens, lens, H, Hk, d, True, dtype, seed=30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(2, 2, 128), (4, 2, 72)])
def test_few_rows_of_wide_heads(hip_device, H, Hk, d, dtype):
    """Short sequences of few rows take a few lanes a row at any head size."""
    _attention_case(hip_device, [20, 1, 7, 16], [20, 4, 0, 16], H, Hk, d, False, dtype, seed=32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 8, 16), (6, 2, 24), (4, 1, 8), (2, 2, 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_short_sequences(hip_device, H, Hk, d, causal, dtype):
    """Sequences of a few tokens take a few lanes a row: rows without keys, keys without rows, a row of one key."""
    q_lens = [1, 5, 0, 9, 3, 2, 11, 1] * 9
    k_lens = [1, 5, 4, 2, 3, 7, 11, 0] * 9
    _attention_case(hip_device, q_lens, k_lens, H, Hk, d, causal, dtype, seed=31)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("H,Hk,d,lens", [(8, 8, 16, [5] * 40), (4, 2, 64, [2, 7, 1, 4] * 5), (2, 1, 128, [6, 3])])
def test_short_sequences_form_delta_from_the_unrounded_out(hip_device, H, Hk, d, lens, dtype):
    """Values of 8 and a little: out's rounding is as large as what the scores' gradients are made of. The lanes round
    neither P nor dS, so that the bound is float32's and the results' own rounding."""
    bf = _bf()
    n = sum(lens)
    q, do = (_randn(i, n, H, d, dtype=dtype, dev=hip_device) for i in (0, 3))
    k = _randn(1, n, Hk, d, dtype=dtype, dev=hip_device)
    v = (8 + 0.25 * _randn(2, n, Hk, d, dev=hip_device)).to(dtype)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = bf.packed_attention(*leaves, bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device))
    ref = sq.attention(q.double(), k.double(), v.double(), lens, lens, True, d ** -0.5, do.double(), dtype, rounds=False)
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
        _within(name, got, ref[name], ref[f"{name}_bound"])


def test_keys_past_32_bit_offsets(hip_device):
    """A cache of more than 2^31 values: the last sequence's keys lie behind them."""
    bf = _bf()
    H, d, far, n = 8, 128, 2 ** 21 - 1000, 6000              # rows of 1024 values
    k = torch.zeros(far + n, H, d, dtype=torch.bfloat16, device=hip_device)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31 + 2 ** 20
    k[far:], v[far:] = _randn(1, n, H, d, dtype=torch.bfloat16, dev=hip_device), _randn(2, n, H, d, dtype=torch.bfloat16, dev=hip_device)
    for rows in (1, 300):
        q = _randn(3, 1 + rows, H, d, dtype=torch.bfloat16, dev=hip_device)
        seqs = bf.PackedSequences.from_lengths([1, rows], [far, n], causal=True, device=hip_device)
        out = bf.packed_attention(q, k, v, seqs)
        ref = sq.attention(q[1:].double(), k[far:].double(), v[far:].double(), [rows], [n], True, d ** -0.5, dtype=torch.bfloat16)
        _within("out", out[1:], ref["out"], ref["out_bound"])
        assert bool((out[0] == 0).all())
    freq = bf.RotaryFrequencies(d, device=hip_device)
    pos = torch.zeros(far + n, dtype=torch.int32, device=hip_device)
    assert torch.equal(bf.rotary_embedding(k, None, freq, positions=pos)[far:], k[far:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_do_not_overflow(hip_device, dtype):
    bf = _bf()
    q = _randn(1, 100, 2, 64, dtype=dtype, dev=hip_device) * 30
    k, v = _randn(2, 100, 2, 64, dtype=dtype, dev=hip_device) * 30, _randn(3, 100, 2, 64, dtype=dtype, dev=hip_device)
    seqs = bf.PackedSequences.from_lengths([100], causal=True, device=hip_device)
    out = bf.packed_attention(q, k, v, seqs)
    ref = sq.attention(q.double(), k.double(), v.double(), [100], [100], True, 0.125, dtype=dtype)
    _within("out", out, ref["out"], ref["out_bound"])


def _float16_gradients(dev, sizes, lens, H, Hk, d, causal, operand_tiny=None, seed=0):
    """float16 training with q, k, v and the output's gradient of the given sizes."""
    bf = _bf()
    n = sum(lens)
    q, k, v, do = (_randn(seed + i, n, h, d, dev=dev).mul(size).half() for i, (h, size) in
                   enumerate(zip((H, Hk, Hk, H), sizes)))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = bf.packed_attention(*leaves, bf.PackedSequences.from_lengths(lens, causal=causal, device=dev))
    ref = sq.attention(q.double(), k.double(), v.double(), lens, lens, causal, d ** -0.5, do.double(), torch.float16, operand_tiny)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))):
        assert float(ref[name].abs().max()) < 65504
        _within(name, got, ref[name], ref[f"{name}_bound"])


@pytest.mark.parametrize("H,Hk,d", [(2, 2, 64), (2, 1, 128), (4, 4, 16)])
def test_small_gradients_keep_their_bits_in_float16(hip_device, H, Hk, d):
    """Gradients of 1e-4 over up to 2048 keys, keys and queries of 8: dS lies below float16's normal numbers, the results
    do not. Operands are times 2^12 (forward 2^9): half a step of a subnormal one is 2^-34 at most."""
    _float16_gradients(hip_device, (0.1, 8.0, 1.0, 1e-4), [2048, 3], H, Hk, d, True, 2.0 ** -34)
    _float16_gradients(hip_device, (8.0, 0.1, 1.0, 1e-4), [700, 1200], H, Hk, d, False, 2.0 ** -34)


@pytest.mark.parametrize("H,Hk,d", [(2, 2, 64), (4, 1, 128), (4, 4, 16), (2, 2, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_large_gradients_do_not_overflow_in_float16(hip_device, H, Hk, d, causal):
    """dS of several 100,000, in some rows and later tiles only, under small queries and keys: the results fit."""
    _float16_gradients(hip_device, (0.01, 0.01, 50.0, 1000.0), [100, 1, 513, 40], H, Hk, d, causal, seed=5)
    bf = _bf()
    n = 400                                       # values grow along the axis: each tile's dS pass the ones before
    q, k = (_randn(i, n, 1, d, dev=hip_device).mul(0.01).half() for i in (1, 2))
    up = torch.logspace(-2, 2, n, device=hip_device)[:, None, None]
    v, do = (_randn(3, n, 1, d, dev=hip_device) * up).half(), (_randn(4, n, 1, d, dev=hip_device) * up).mul(20).half()
    for flip in (False, True):
        xs = [x.flip(0) if flip else x for x in (q, k, v, do)]
        leaves = [x.clone().requires_grad_(True) for x in xs[:3]]
        out = bf.packed_attention(*leaves, bf.PackedSequences.from_lengths([n], causal=causal, device=hip_device))
        ref = sq.attention(*(x.double() for x in xs[:3]), [n], [n], causal, d ** -0.5, xs[3].double(), torch.float16)
        for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, xs[3]))):
            _within(name, got, ref[name], ref[f"{name}_bound"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,H,d", [(2, 1, 64), (2048, 16, 64), (4099, 8, 16), (2048, 8, 128)])
def test_many_small_terms_count(hip_device, rows, H, d, dtype):
    """One key at score 0 and 200,000 at -16.5, whose weights are each below float16's last bit and together 1.3%."""
    bf = _bf()
    n = 200001
    q = torch.zeros(rows, H, d, dtype=dtype, device=hip_device)
    q[:, :, 0] = 1.0
    k, v = torch.zeros(n, H, d, dtype=dtype, device=hip_device), torch.ones(n, H, d, dtype=dtype, device=hip_device)
    k[1:, :, 0] = -16.5
    v[0] = 0.0
    out = bf.packed_attention(q, k, v, bf.PackedSequences.from_lengths([rows], [n], device=hip_device), scale=1.0)
    w = (n - 1) * math.exp(-16.5)
    # each term's rounding, the same for all (half a step), and the result's; two running float32 sums (of the terms, of
    # their products) of n terms, n roundings of 2^-24 of the sum each: equal terms are all rounded the same way, so these
    # add up (6.8e-8 onto 1 becomes 1.2e-7); exponentials at 16.5
    off = (2 * sq.half_step(dtype) + 2.0 ** -24 * (2 * n + 200)) * w / (1 + w)
    assert float((out.double() - w / (1 + w)).abs().max()) < off


def _strided(x, kind):
    """The same values in another layout."""
    n, h, d = x.shape
    if kind == "fused":                                   # a slice of a wider projection, 16-byte steps
        big = x.new_full((n, h + 3, d), float("nan"))
        big[:, 1:h + 1] = x
        return big[:, 1:h + 1]
    if kind == "heads_first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if kind == "odd":                                     # rows at odd addresses
        big = x.new_full((n, h * d + 1), float("nan"))
        big[:, 1:] = x.reshape(n, -1)
        return big[:, 1:].unflatten(1, (h, d))
    if kind == "last":                                    # not contiguous along the head
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    raise AssertionError(kind)


@pytest.mark.parametrize("kind", ["fused", "heads_first", "odd", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_give_the_same_bits(hip_device, kind, dtype):
    bf = _bf()
    lens = [40, 90, 1]
    q, k, v, do = (_randn(i, 131, 4, 32, dtype=dtype, dev=hip_device) for i in range(4))
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    ld = torch.full((4,), -0.1, device=hip_device)
    freq = bf.RotaryFrequencies(32, device=hip_device)

    def every(q, k, v, do):
        got = []
        for f in (lambda *x: bf.packed_attention(*x, seqs), lambda *x: bf.linear_attention(*x, ld, seqs)):
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
            out = f(*leaves)
            got += [out, *torch.autograd.grad(out, leaves, do)]
        leaves = [x.detach().requires_grad_(True) for x in (q, k)]
        out = bf.rotary_embedding(*leaves, freq, seqs=seqs)
        return got + [*out, *torch.autograd.grad(out, leaves, (do, do))]

    for a, b in zip(every(q, k, v, do), every(*(_strided(x, kind) for x in (q, k, v, do)))):
        assert torch.equal(a, b)


def test_a_broadcast_key_head_gets_the_sum_of_its_gradients(hip_device):
    """k and v expanded over heads and over rows: strides of 0 in, gradients summed by autograd."""
    bf = _bf()
    q = _randn(1, 50, 4, 16, dev=hip_device)
    k, v = (_randn(i, 50, 1, 16, dev=hip_device).requires_grad_(True) for i in (2, 3))
    do = _randn(4, 50, 4, 16, dev=hip_device)
    seqs = bf.PackedSequences.from_lengths([30, 20], causal=True, device=hip_device)
    a = torch.autograd.grad(bf.packed_attention(q, k.expand(50, 4, 16), v.expand(50, 4, 16), seqs), (k, v), do)
    ref = sq.attention(q.double(), k.detach().double(), v.detach().double(), [30, 20], [30, 20], True, 0.25, do.double(),
                       torch.float32)
    for got, name in zip(a, ("dk", "dv")):
        # the sum of four heads' rounded gradients: four roundings of values no larger than the bound's own terms
        _within(name, got, ref[name], 5 * ref[f"{name}_bound"])
    row = _randn(5, 1, 1, 16, dev=hip_device).requires_grad_(True)
    out = bf.packed_attention(q, row.expand(50, 4, 16), row.expand(50, 4, 16), seqs)
    assert torch.allclose(out, row.detach().expand(50, 4, 16), atol=1e-5)         # every key the same: its value
    torch.autograd.grad(out, row, do)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_a_row_does_not_see_do_not_reach_it(hip_device, dtype):
    """NaN and infinities in one sequence, in later tokens and behind the last sequence: every other row, and its
    gradients, as without them, bit for bit."""
    bf = _bf()
    lens, n, bad_seq = [50, 20, 70], 150, slice(50, 70)
    seqs = bf.PackedSequences.from_offsets(torch.tensor([0, 50, 70, 140], dtype=torch.int32, device=hip_device), n_q=n,
                                           causal=True)
    q, k, v, do = (_randn(i, n, 2, 64, dtype=dtype, dev=hip_device) for i in range(4))
    ld = torch.tensor([-0.05, -0.3], device=hip_device)
    keep = torch.ones(n, dtype=torch.bool, device=hip_device)
    keep[bad_seq] = False
    keep[140:] = False

    def every(q, k, v, do):
        got = []
        for f in (lambda *x: bf.packed_attention(*x, seqs), lambda *x: bf.linear_attention(*x, ld, seqs)):
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
            out = f(*leaves)
            got += [out, *torch.autograd.grad(out, leaves, do)]
        return got

    clean = every(q, k, v, do)
    for which in range(4):
        xs = [x.clone() for x in (q, k, v, do)]
        for j, value in enumerate((float("nan"), float("inf"), -float("inf"))):
            xs[which][51 + j:70:3] = value
            xs[which][140 + j::3] = value
        for i, (a, b) in enumerate(zip(every(*xs), clean)):
            assert torch.equal(a[keep], b[keep]), (which, i)
        for a in clean[0:4] + clean[4:8]:
            assert bool((a[140:] == 0).all())             # rows behind the last sequence
    # later tokens of the same sequence: the rows before them
    for which in (1, 2):
        xs = [x.clone() for x in (q, k, v, do)]
        xs[which][30:50] = float("nan")
        for a, b in zip((f(*xs[:3]) for f in (lambda *x: bf.packed_attention(*x, seqs),
                                              lambda *x: bf.linear_attention(*x, ld, seqs))), (clean[0], clean[4])):
            assert torch.equal(a[:30], b[:30])
            assert bool(a[30:50].isnan().all())           # and the rows that see them are NaN
    xs = [x.clone() for x in (q, k, v)]
    xs[2][10] = float("inf")
    out = bf.packed_attention(*xs, seqs)
    assert bool((out[10:50] == float("inf")).all()) and torch.equal(out[:10], clean[0][:10])


@pytest.mark.parametrize("dtype", DTYPES)
def test_short_sequences_keep_what_they_do_not_see_out(hip_device, dtype):
    bf = _bf()
    lens = [5, 3, 6] * 4
    n = sum(lens) + 7
    off = torch.tensor([0] + lens).cumsum(0).to(hip_device)
    seqs = bf.PackedSequences.from_offsets(off, n_q=n, causal=True)
    assert seqs.longest == 6
    ld = torch.tensor([-0.05, -0.3], device=hip_device)
    base = [_randn(i, n, 2, 16, dtype=dtype, dev=hip_device) for i in range(4)]
    keep = torch.ones(n, dtype=torch.bool, device=hip_device)
    keep[5:8] = False
    keep[sum(lens):] = False

    def every(q, k, v, do):
        got = []
        for f in (lambda *x: bf.packed_attention(*x, seqs), lambda *x: bf.linear_attention(*x, ld, seqs)):
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
            out = f(*leaves)
            got += [out, *torch.autograd.grad(out, leaves, do)]
        return got

    clean = every(*base)
    for which in range(4):
        for value in (float("nan"), float("inf")):
            xs = [x.clone() for x in base]
            xs[which][5:8] = value
            xs[which][sum(lens):] = value
            for i, (a, b) in enumerate(zip(every(*xs), clean)):
                assert torch.equal(a[keep], b[keep]), (which, value, i)
                assert bool((a[sum(lens):] == 0).all())
    xs = [x.clone() for x in base]
    xs[2][2] = float("inf")
    out = bf.packed_attention(*xs[:3], seqs)
    assert bool((out[2:5] == float("inf")).all()) and torch.equal(out[:2], clean[0][:2])


def test_more_than_2_to_the_30_sequences(hip_device):
    """Sequences without tokens before and behind a few with: their numbers, summed in a search, pass 32 bits."""
    bf = _bf()
    n_seq, lens = 2 ** 30 + 100, [5, 40, 3]
    off = torch.zeros(n_seq + 1, dtype=torch.int32, device=hip_device)
    off[-3:] = torch.tensor(lens, device=hip_device).cumsum(0)
    seqs = bf.PackedSequences.from_offsets(off, n_q=48, causal=True, check=False)
    del off
    plain = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    assert torch.equal(seqs.row_span, plain.row_span) and torch.equal(seqs.key_span, plain.key_span)
    assert torch.equal(seqs.positions(), plain.positions())


def test_results_repeat_bit_for_bit(hip_device):
    a = _attention_case(hip_device, [300, 41], [300, 41], 8, 2, 64, True, torch.bfloat16, seed=3, train=False)
    b = _attention_case(hip_device, [300, 41], [300, 41], 8, 2, 64, True, torch.bfloat16, seed=3, train=False)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 128])
@pytest.mark.parametrize("longest", [0, 5, 2100])
def test_spans_of_any_numbers_stay_inside_the_tensors(hip_device, longest, d, dtype):
    """The operators below the sequences take spans as they come: any 32-bit numbers give some result, from the tensors'
    own rows (here a group's row number would pass 32 bits, and differences of two bounds)."""
    ops, H, Hk, n = torch.ops.bf, 8, 2, 2100
    q, do = (_randn(i, n, H, d, dtype=dtype, dev=hip_device) for i in (0, 3))
    k, v = (_randn(i, n, Hk, d, dtype=dtype, dev=hip_device) for i in (1, 2))
    gen = torch.Generator().manual_seed(5)
    ld = torch.full((H,), -0.1, device=hip_device)
    off = torch.tensor([0, 700, n], dtype=torch.int32, device=hip_device)
    far = torch.tensor([-2 ** 31, -2 ** 29, -7, 0, 5, n, 2 ** 29, 2 ** 29 + 3, 2 ** 31 - 1], dtype=torch.int64)
    for rep in range(3):
        row_span, key_span = (far[torch.randint(len(far), (n, 2), generator=gen)].to(torch.int32).to(hip_device) for _ in range(2))
        out, lse, rest = ops.packed_attn_fwd(q, k, v, row_span, 0.1, longest, True)
        grads = ops.packed_attn_bwd(q, k, v, row_span, key_span, out, lse, do, 0.1, longest, rest)
        few = ops.packed_attn_fwd(q[:3], k, v, row_span[:3].contiguous(), 0.1, longest, False)
        lin = ops.linear_attn_fwd(q, q, q, ld, row_span, key_span, off, 0.1, longest, None, True)
        back = ops.linear_attn_bwd(q, q, q, ld, row_span, key_span, off, do, 0.1, longest)
        torch.cuda.synchronize()
        assert all(t.numel() for t in (*grads, *few[:2], *lin, *back))


# ------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hk,d,rot", [(4, 2, 64, 64), (3, 0, 32, 16), (2, 2, 16, 8), (5, 1, 10, 6), (1, 1, 3, 2),
                                         (8, 8, 128, 96), (1, 1, 1024, 1024)])
def test_rotary_values_and_gradients(hip_device, hq, hk, d, rot, interleaved, dtype):
    bf = _bf()
    n = 37
    q = _randn(1, n, hq, d, dtype=dtype, dev=hip_device).requires_grad_(True)
    k = _randn(2, n, hk, d, dtype=dtype, dev=hip_device).requires_grad_(True) if hk else None
    pos = torch.randint(-5, 2 ** 20, (n,), generator=torch.Generator().manual_seed(3)).to(hip_device)
    freq = bf.RotaryFrequencies(rot, base=500.0, factor=2.0, amplitude=1.25, device=hip_device)
    theta = (500.0 ** -(torch.arange(rot // 2, dtype=torch.float64) * 2 / rot) / 2.0).to(hip_device)
    xs = [x for x in (q, k) if x is not None]
    outs = bf.rotary_embedding(q, k, freq, positions=pos, interleaved=interleaved)
    outs = outs if hk else (outs,)
    dos = [_randn(5 + i, *x.shape, dtype=dtype, dev=hip_device) for i, x in enumerate(xs)]
    grads = torch.autograd.grad(outs, xs, dos)
    u = sq.half_step(dtype)
    for x, got, inverse in [*zip(xs, outs, [False] * 2), *zip(dos, grads, [True] * 2)]:
        ref = sq.rotary(x.detach().double(), pos, theta, 1.25, interleaved, inverse)
        # the result's rounding; a sum of two products whose sin and cos are a few float32 steps off (the angle's rest is
        # rounded once, 2 pi 2^-25, the functions to 4 steps, amplitude and products to one each)
        size = torch.full_like(ref, 0.0)
        size[..., :rot] = x.detach().double()[..., :rot].abs().amax(-1, keepdim=True) * 1.25 * 2
        _within("turned", got.detach(), ref, u * ref.abs() + 2.0 ** -24 * 16 * size + 2.0 ** -25 * (dtype == torch.float16))
        assert torch.equal(got[..., rot:], x[..., rot:])


def test_operators_without_gradients_give_the_same_bits(hip_device):
    """bf::rotary, packed_attn_* and linear_attn_* as a caller takes them beside the differentiable ones."""
    bf, ops = _bf(), torch.ops.bf
    lens, H, d = [70, 1, 130], 2, 32
    q, k, v, do = (_randn(i, sum(lens), H, d, dtype=torch.bfloat16, dev=hip_device) for i in range(4))
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    freq, ld = bf.RotaryFrequencies(d, amplitude=1.5, device=hip_device), torch.full((H,), -0.1, device=hip_device)
    spans = (seqs.row_span, seqs.key_span)

    def gradients(f, *xs):
        leaves = [x.clone().requires_grad_(True) for x in xs]
        out = f(*leaves)
        outs = out if isinstance(out, tuple) else (out,)
        return [*outs, *torch.autograd.grad(outs, leaves, [do] * len(outs))]

    pos = seqs.positions()
    got = [*ops.rotary(q, k, pos, freq.turns, 1.5, True), *ops.rotary(do, do, pos, freq.turns, 1.5, True, True)]
    for a, b in zip(got, gradients(lambda x, y: bf.rotary_embedding(x, y, freq, seqs=seqs, interleaved=True), q, k)):
        assert torch.equal(a, b)
    out, lse, rest = ops.packed_attn_fwd(q, k, v, spans[0], 0.2, seqs.longest, True)
    got = [out, *ops.packed_attn_bwd(q, k, v, *spans, out, lse, do, 0.2, seqs.longest, rest)]
    for a, b in zip(got, gradients(lambda *x: bf.packed_attention(*x, seqs, scale=0.2), q, k, v)):
        assert torch.equal(a, b)
    out, _ = ops.linear_attn_fwd(q, k, v, ld, *spans, seqs.q_offsets, 0.2, seqs.longest)
    got = [out, *ops.linear_attn_bwd(q, k, v, ld, *spans, seqs.q_offsets, do, 0.2, seqs.longest)]
    for a, b in zip(got, gradients(lambda *x: bf.linear_attention(*x, ld, seqs, scale=0.2), q, k, v)):
        assert torch.equal(a, b)


def test_rotary_of_one_of_two_gradients(hip_device):
    bf = _bf()
    q, k = (_randn(i, 9, 2, 16, dev=hip_device).requires_grad_(True) for i in (1, 2))
    freq = bf.RotaryFrequencies(16, device=hip_device)
    pos = torch.arange(9, dtype=torch.int32, device=hip_device)
    for i in (0, 1):
        out = bf.rotary_embedding(q, k, freq, positions=pos)
        g = torch.autograd.grad(out[i].sum(), (q, k), allow_unused=True)
        assert g[1 - i] is None and g[i] is not None
        one = bf.rotary_embedding((q, k)[i], None, freq, positions=pos)
        assert torch.equal(torch.autograd.grad(one.sum(), (q, k)[i])[0], g[i])


@pytest.mark.parametrize("q_lens,k_lens", [([3, 5, 0, 4], [5, 3, 4, 0]), ([2, 6], [2, 6]), ([1, 2, 1], [7, 2, 3])])
@pytest.mark.parametrize("causal", [False, True])
def test_rotary_of_keys_with_sequences_of_their_own(hip_device, causal, q_lens, k_lens):
    """Rows stand behind their sequence's earlier keys, keys at their own place, also where as many rows as keys are
    there in all; keys of the new rows stand where the rows do."""
    from budgetformer_amd.attention import CoreAttention
    bf = _bf()
    n_q, n_k, H, d = sum(q_lens), sum(k_lens), 2, 16
    q, k = _randn(1, n_q, H, d, dev=hip_device).requires_grad_(True), _randn(2, n_k, H, d, dev=hip_device).requires_grad_(True)
    freq = bf.RotaryFrequencies(d, device=hip_device)
    seqs = bf.PackedSequences.from_lengths(q_lens, k_lens, causal=causal, device=hip_device)
    q_pos = torch.cat([torch.arange(m) + n - m for m, n in zip(q_lens, k_lens)]).to(hip_device)
    k_pos = torch.cat([torch.arange(n) for n in k_lens]).to(hip_device)
    assert torch.equal(seqs.positions().long(), q_pos) and torch.equal(seqs.key_positions().long(), k_pos)
    want = (bf.rotary_embedding(q, None, freq, positions=q_pos), bf.rotary_embedding(k, None, freq, positions=k_pos))
    got = bf.rotary_embedding(q, k, freq, seqs=seqs)
    dos = [_randn(3 + i, *x.shape, dev=hip_device) for i, x in enumerate(want)]
    for a, b in zip((*got, *torch.autograd.grad(got, (q, k), dos)), (*want, *torch.autograd.grad(want, (q, k), dos))):
        assert torch.equal(a, b)
    if n_q != n_k:
        for a, b in zip(bf.rotary_embedding(q, q, freq, seqs=seqs), (want[0], want[0])):
            assert torch.equal(a, b)
    else:
        core = CoreAttention(H * d, 0.0, H, 1, rotary=freq)
        got = core(q[None], k[None], k[None], edge_index=seqs, attn_type="flash")
        assert torch.equal(got.view(n_q, H, d), bf.packed_attention(*want, k, seqs))


@pytest.mark.parametrize("scaling", ["linear", "ntk", "by_parts"])
def test_rotary_frequencies(hip_device, scaling):
    bf = _bf()
    f = bf.RotaryFrequencies(64, 10000.0, factor=8.0, scaling=scaling, original=4096, device=hip_device)
    theta = f.turns.cpu() * 2 * math.pi
    plain = 10000.0 ** -(torch.arange(32, dtype=torch.float64) / 32)
    if scaling == "linear":
        assert torch.allclose(theta, plain / 8, rtol=1e-14, atol=0)
    if scaling == "ntk":
        assert theta[0] == 1.0 and abs(float(theta[-1] / plain[-1]) - 1 / 8) < 1e-12
    if scaling == "by_parts":
        turns = 4096 * plain / (2 * math.pi)
        assert torch.equal(theta[turns >= 4], (plain / (2 * math.pi) * (2 * math.pi))[turns >= 4])
        assert torch.allclose(theta[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
        mid = (turns > 1) & (turns < 4)
        assert bool(mid.any()) and bool(((theta < plain) & (theta > plain / 8))[mid].all())


# ------------------------------------------------------------------ linear attention
def _linear_case(dev, lens, H, dk, dv, dtype, seed=0, decays=None, init=False, tail=0):
    bf = _bf()
    n = sum(lens)
    q, k = (_randn(seed + i, n, H, dk, dtype=dtype, dev=dev) for i in (0, 1))
    v, do = (_randn(seed + i, n, H, dv, dtype=dtype, dev=dev) for i in (2, 3))
    ld = torch.tensor(decays if decays is not None else [-0.02 * 3 ** i for i in range(H)], device=dev)
    s0 = _randn(seed + 4, len(lens), H, dk, dv, dev=dev) if init else None
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=dev)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = bf.linear_attention(*leaves, ld, seqs, initial_state=s0, return_state=init)
    ref = sq.linear_attention(q.double().cpu(), k.double().cpu(), v.double().cpu(), ld.cpu(), lens, dk ** -0.5,
                              None if s0 is None else s0.cpu(), do.double().cpu(), dtype)
    ref = {x: y.to(dev) for x, y in ref.items()}
    if init:
        out, state = out
        _within("state", state, ref["state"], ref["state_bound"])
    _within("out", out.detach(), ref["out"], ref["out_bound"])
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
        _within(name, got, ref[name], ref[f"{name}_bound"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[1], [5] * 30, [33, 0, 64, 65, 1, 128, 31], [300], [0, 17, 0]],
                         ids=["one", "walks", "mixed", "long", "empty"])
@pytest.mark.parametrize("init", [False, True])
def test_linear_attention(hip_device, lens, init, dtype):
    _linear_case(hip_device, lens, 3, 32, 32, dtype, seed=31, init=init)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(8, 8), (16, 64), (64, 24), (128, 40), (72, 128), (128, 128)])
def test_linear_attention_head_sizes(hip_device, dk, dv, dtype):
    _linear_case(hip_device, [70, 3, 90], 2, dk, dv, dtype, seed=37)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("init", [False, True])
def test_linear_attention_over_segments(hip_device, init, dtype):
    """More tokens than a segment (256): the state is carried across, past a sequence's end inside a segment too."""
    _linear_case(hip_device, [700, 50, 256, 6, 500], 2, 16, 16, dtype, seed=41, init=init)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("init", [False, True])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 72)])
@pytest.mark.parametrize("lens", [[600, 50, 131], [100] * 7 + [81]], ids=["carried", "warm"])
def test_linear_attention_of_wide_heads_over_segments(hip_device, lens, dk, dv, init, dtype):
    """Four waves and four blocks of the state over segments of 256 tokens, carried or (short sequences) begun anew."""
    _linear_case(hip_device, lens, 2, dk, dv, dtype, seed=42, init=init)


@pytest.mark.parametrize("lens", [[20000], [9000, 3, 64, 10900]])
def test_linear_attention_over_hundreds_of_segments(hip_device, lens):
    """313 segments of 64 tokens: more than a workgroup of the carry holds at a time."""
    _linear_case(hip_device, lens, 1, 8, 8, torch.float32, seed=43, decays=[-0.003])


def test_linear_attention_states_of_many_empty_sequences(hip_device):
    """Sequences without tokens, more than a wave looks at together: their final state is their initial one."""
    _linear_case(hip_device, ([0, 3, 0] * 30 + [0] * 70 + [40]) * 2, 2, 16, 24, torch.float32, seed=47, init=True)


def test_linear_attention_of_extreme_decays(hip_device):
    """No decay, one that leaves only the row's own token, and one that underflows within a tile."""
    _linear_case(hip_device, [90, 40], 3, 16, 16, torch.float32, seed=43, decays=[0.0, -math.inf, -40.0])


def test_linear_attention_states_past_float16(hip_device):
    """A state beyond 65504 under small queries: the result fits, so it has to come out."""
    bf = _bf()
    n, d = 400, 16
    seqs = bf.PackedSequences.from_lengths([n], causal=True, device=hip_device)
    q = torch.full((n, 1, d), 2.0 ** -10, dtype=torch.float16, device=hip_device)
    k = torch.full((n, 1, d), 32.0, dtype=torch.float16, device=hip_device)
    out = bf.linear_attention(q, k, k, torch.zeros(1, device=hip_device), seqs, scale=1.0)
    # out_i = (i + 1) * 16 * 2^-10 * 32 * 32 = 16 (i + 1), each step exact but the state's rounding to 11 bits
    ref = 16.0 * torch.arange(1, n + 1, device=hip_device).double()[:, None, None].expand(n, 1, d)
    _within("out", out, ref, 3 * 2.0 ** -11 * ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[5, 40], [700, 3]], ids=["tiles", "segments"])
def test_linear_attention_of_a_decay_that_is_nan(hip_device, lens, dtype):
    """Its head's results are NaN, gradients and states too; the others' are as without it."""
    bf = _bf()
    n, H, d = sum(lens), 3, 32
    base = [_randn(i, n, H, d, dtype=dtype, dev=hip_device) for i in range(4)]
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    fine = torch.tensor([-0.1, -0.2, -math.inf], device=hip_device)
    bad = fine.clone()
    bad[1] = math.nan

    def every(ld):
        leaves = [x.clone().requires_grad_(True) for x in base[:3]]
        out, state = bf.linear_attention(*leaves, ld, seqs, return_state=True)
        one = bf.linear_attention_step(*(x[:2] for x in base[:3]), ld, state)
        return [x.detach() for x in (out, state, *one, *torch.autograd.grad(out, leaves, base[3]))]

    for a, b in zip(every(bad), every(fine)):
        assert torch.equal(a[:, ::2], b[:, ::2])
        assert bool(a[:, 1].isnan().all())


def _linear_of_sizes(dev, sizes, lens, operand_tiny=None, names=("out", "dq", "dk", "dv"), H=2, d=64):
    """float16, q, k, v and the output's gradient of the given sizes."""
    bf = _bf()
    n = sum(lens)
    q, k, v, do = (_randn(i, n, H, d, dev=dev).mul(size).half() for i, size in enumerate(sizes))
    v[::7] = 0.0
    ld = torch.tensor([-0.02, -0.3], device=dev)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=dev)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = bf.linear_attention(*leaves, ld, seqs)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))))
    ref = sq.linear_attention(q.double().cpu(), k.double().cpu(), v.double().cpu(), ld.cpu(), lens, d ** -0.5, None,
                              do.double().cpu(), torch.float16, operand_tiny)
    for x in names:
        assert float(ref[x].abs().max()) < 65504
        _within(x, got[x], ref[x].to(dev), ref[f"{x}_bound"].to(dev))


@pytest.mark.parametrize("lens", [[1, 5], [90, 33]])
def test_linear_attention_scores_past_float16(hip_device, lens):
    """Scores of some 80,000 under small values: the result fits, so it has to come out, values of 0 among them."""
    bf = _bf()
    _linear_of_sizes(hip_device, (100.0, 100.0, 0.01, 0.01), lens)
    _linear_of_sizes(hip_device, (0.01, 0.01, 100.0, 100.0), lens)         # the gradients' scores, v and dout
    seqs = bf.PackedSequences.from_lengths([3], causal=True, device=hip_device)
    q = torch.full((3, 1, 64), 100.0, dtype=torch.float16, device=hip_device)
    v = torch.full((3, 1, 64), 0.01, dtype=torch.float16, device=hip_device)
    v[:, :, 1::2] = 0.0
    out = bf.linear_attention(q, q, v, torch.full((1,), -math.inf, device=hip_device), seqs)
    ref = (80000.0 * v.double())                                           # only the row's own token
    _within("out", out, ref, 2 * 2.0 ** -11 * ref)


def test_linear_attention_small_gradients_keep_their_bits_in_float16(hip_device):
    """Gradients of 1e-6 under queries and keys of 100: the scores they form lie below float16's normal numbers, the
    results do not. A score is rounded in units of 2^-9 (half a step of 2^-34), a state in units of 2^-6."""
    _linear_of_sizes(hip_device, (100.0, 100.0, 1.0, 1e-6), [300, 33], 2.0 ** -31, ("dq", "dk"))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** -10, 32.0), (2.0 ** -6, 2.0)])
@pytest.mark.parametrize("where", ["v", "state"])
def test_linear_attention_columns_beside_one_that_is_not_finite(hip_device, where, q_size, k_size, bad):
    """A value that is not finite, in one column of v or of the initial state: the other columns of its rows' results, whose
    states are past 1000 and past 65504, come out as without it."""
    bf = _bf()
    n, d = 400, 16
    seqs = bf.PackedSequences.from_lengths([n], causal=True, device=hip_device)
    q = torch.full((n, 1, d), q_size, dtype=torch.float16, device=hip_device)
    k = torch.full((n, 1, d), k_size, dtype=torch.float16, device=hip_device)
    v = torch.full((n, 1, d), 32.0, dtype=torch.float16, device=hip_device)
    state = torch.zeros(1, 1, d, d, device=hip_device)
    first = 3
    if where == "v":
        v[first, :, 5] = bad
    else:
        state[..., 5], first = bad, 0
    out = bf.linear_attention(q, k, v, torch.zeros(1, device=hip_device), seqs, scale=1.0, initial_state=state)
    ref = (16 * q_size * k_size * 32) * torch.arange(1, n + 1, device=hip_device).double()[:, None, None].expand(n, 1, d)
    keep = torch.arange(d, device=hip_device) != 5
    _within("out", out[..., keep], ref[..., keep], 3 * 2.0 ** -11 * ref[..., keep])      # the state's rounding to 11 bits, the result's
    assert not bool(torch.isfinite(out[first:, :, 5]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,dk,dv", [(1, 1, 8, 8), (3, 5, 128, 128), (7, 2, 24, 72), (2, 3, 64, 16)])
def test_linear_attention_step_continues_a_prompt(hip_device, n, H, dk, dv, dtype):
    bf = _bf()
    q, k = (_randn(i, n, H, dk, dtype=dtype, dev=hip_device) for i in (1, 2))
    v, s = _randn(3, n, H, dv, dtype=dtype, dev=hip_device), _randn(4, n, H, dk, dv, dev=hip_device)
    ld = torch.linspace(-2.0, 0.0, H, device=hip_device)
    before = s.clone()
    out, new = bf.linear_attention_step(q, k, v, ld, s)
    assert torch.equal(s, before)
    ref = sq.linear_attention(q.double().cpu(), k.double().cpu(), v.double().cpu(), ld.cpu(), [1] * n, dk ** -0.5, s.cpu(),
                              dtype=dtype)
    # float32 arithmetic of one step, and the result's rounding
    g = ld.double().exp()[:, None, None]
    size = g * before.double().abs() + k.double().abs()[..., None] * v.double().abs()[:, :, None]
    _within("state", new, ref["state"].to(hip_device), 2.0 ** -24 * 8 * size)
    aq = torch.einsum("nhk,nhkv->nhv", q.double().abs(), size) * dk ** -0.5
    _within("out", out, ref["out"].to(hip_device),
            sq.half_step(dtype) * ref["out"].to(hip_device).abs() + 2.0 ** -24 * (dk + 16) * aq + 2.0 ** -25)
    got, same = bf.linear_attention_step(q, k, v, ld, s, out_state=s)
    assert same.data_ptr() == s.data_ptr() and torch.equal(s, new) and torch.equal(got, out)


def test_linear_attention_step_states_that_overlap(hip_device):
    bf = _bf()
    n, H, d = 4, 2, 16
    store = _randn(1, n + 1, H, d, d, dev=hip_device)
    q, ld = _randn(2, n, H, d, dev=hip_device), torch.full((H,), -0.5, device=hip_device)
    for state, into in ((store[:n], store[1:]), (store[1:], store[:n])):
        with pytest.raises(ValueError, match="overlaps state"):
            bf.linear_attention_step(q, q, q, ld, state, out_state=into)
    room = torch.zeros(n * H * d * d, device=hip_device)
    inside = room[:n * H * d].view(n, H, d)
    with pytest.raises(ValueError, match="overlaps an input"):
        bf.linear_attention_step(q, inside, q, ld, store[:n], out_state=room.view(n, H, d, d))
    with pytest.raises(NotImplementedError, match="no gradients"):
        bf.linear_attention_step(q, q, q, ld, store[:n], out_state=room.view(n, H, d, d).requires_grad_(True))


def test_a_state_updated_in_place_does_not_change_a_gradient_that_kept_it(hip_device):
    bf = _bf()
    seqs = bf.PackedSequences.from_lengths([5, 7], causal=True, device=hip_device)
    x, ld = _randn(1, 12, 2, 16, dev=hip_device).requires_grad_(True), torch.full((2,), -0.5, device=hip_device)
    state, one = _randn(2, 2, 2, 16, 16, dev=hip_device), _randn(3, 2, 2, 16, dev=hip_device)
    out = bf.linear_attention(x, x, x, ld, seqs, initial_state=state)
    bf.linear_attention_step(one, one, one, ld, state)              # into a new tensor: nothing changes
    torch.autograd.grad(out.sum(), x, retain_graph=True)
    bf.linear_attention_step(one, one, one, ld, state, out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


# ------------------------------------------------------------------ together, as they are used
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_single_tokens_equal_the_whole(hip_device, dtype):
    """Rotary, softmax attention and linear attention over a prompt and then token by token against what was kept: the
    rows of one call over everything."""
    bf = _bf()
    H, d, n, m = 4, 32, 90, 6
    q, k, v = (_randn(i, n, H, d, dtype=dtype, dev=hip_device) for i in range(3))
    freq, ld = bf.RotaryFrequencies(d, device=hip_device), torch.linspace(-0.5, -0.01, H, device=hip_device)
    whole = bf.PackedSequences.from_lengths([n], causal=True, device=hip_device)
    qr, kr = bf.rotary_embedding(q, k, freq, seqs=whole)
    soft, lin = bf.packed_attention(qr, kr, v, whole), bf.linear_attention(q, k, v, ld, whole)
    head = bf.PackedSequences.from_lengths([n - m], causal=True, device=hip_device)
    _, state = bf.linear_attention(q[:n - m], k[:n - m], v[:n - m], ld, head, return_state=True)
    ref = sq.attention(qr.double(), kr.double(), v.double(), [n], [n], True, d ** -0.5, dtype=dtype)
    lref = sq.linear_attention(q.double().cpu(), k.double().cpu(), v.double().cpu(), ld.cpu(), [n], d ** -0.5, dtype=dtype)
    for t in range(n - m, n):
        one = bf.PackedSequences.from_lengths([1], [t + 1], causal=True, device=hip_device)
        assert int(one.positions()) == t
        q1 = bf.rotary_embedding(q[t:t + 1], None, freq, seqs=one)
        assert torch.equal(q1, qr[t:t + 1])
        got = bf.packed_attention(q1, kr[:t + 1], v[:t + 1], one)
        for x in (got, soft[t:t + 1]):
            _within("softmax", x, ref["out"][t:t + 1], ref["out_bound"][t:t + 1])
        got, state = bf.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], ld, state)
        for x in (got, lin[t:t + 1]):
            _within("linear", x, lref["out"][t:t + 1].to(hip_device), lref["out_bound"][t:t + 1].to(hip_device))


def test_walks_attend_their_nodes(hip_device):
    """The framework's own walks as sequences: rotary positions and causal attention over each walk's nodes, trained."""
    import numpy as np
    from budgetformer_amd import hip_ops
    from budgetformer_amd.graph import CSRGraph, chung_lu_csr
    bf = _bf()
    n, P, L, H, d = 200, 2, 4, 4, 16
    rowptr, col = chung_lu_csr(n, 1500, seed=3)
    g = CSRGraph.from_csr(rowptr, col, n, device=hip_device)
    u = torch.from_numpy(np.random.default_rng(1).random((n * P, L), dtype=np.float32)).to(hip_device)
    walks = hip_ops.random_walk(g.rowptr, g.col, 0, n, P, L, u=u)
    x = _randn(1, n, H * d, dev=hip_device).requires_grad_(True)
    seqs = bf.PackedSequences.from_lengths([L + 1] * (n * P), causal=True, device=hip_device)
    freq = bf.RotaryFrequencies(d, device=hip_device)
    h = x[walks.reshape(-1)].view(-1, H, d)
    q, k = bf.rotary_embedding(h, h, freq, seqs=seqs)
    out = bf.packed_attention(q, k, h, seqs)
    do = _randn(2, *out.shape, dev=hip_device)
    got, = torch.autograd.grad(out, x, do)

    x64 = x.detach().double().requires_grad_(True)
    h64 = x64[walks.reshape(-1)].view(n * P, L + 1, H, d)
    theta = 10000.0 ** -(torch.arange(d // 2, dtype=torch.float64, device=hip_device) * 2 / d)
    pos = torch.arange(L + 1, device=hip_device).repeat(n * P)
    r64 = sq.rotary(h64.reshape(-1, H, d), pos, theta, 1.0, False).view(n * P, L + 1, H, d).transpose(1, 2)
    s = (r64 @ r64.transpose(2, 3) / 4.0).masked_fill(~sq.visible(L + 1, L + 1, True, hip_device), -math.inf)
    ref = (s.softmax(-1) @ h64.transpose(1, 2)).transpose(1, 2).reshape(-1, H, d)
    rg, = torch.autograd.grad(ref, x64, do.double())
    # float32 throughout: sums of at most 5 keys, of 16 values a head, of the rows a node is in
    assert float((out.detach().double() - ref.detach()).abs().max()) < 2.0 ** -24 * 300 * float(x64.detach().abs().max())
    scale = float(rg.abs().max())
    assert float((got.double() - rg).abs().max()) < 2.0 ** -24 * 2000 * scale


@pytest.mark.parametrize("dtype", DTYPES)
def test_core_attention_flash(hip_device, dtype):
    from budgetformer_amd.attention import CoreAttention
    bf = _bf()
    b, S, H, d = 3, 45, 4, 16
    q, k, v = (_randn(i, b, S, H, d, dtype=dtype, dev=hip_device) for i in range(3))
    ref = sq.attention(*(x.double().reshape(-1, H, d) for x in (q, k, v)), [S] * b, [S] * b, False, 0.25, dtype=dtype)
    core = CoreAttention(H * d, 0.0, H, 1)
    for _ in range(2):
        got = core(q, k, v, attn_type="flash")
        assert got.shape == (b, S, H * d)
        _within("flash", got.view(-1, H, d), ref["out"], ref["out_bound"])
    seqs = bf.PackedSequences.from_lengths([100, 35], device=hip_device)          # graphs packed along the batch's rows
    ref = sq.attention(*(x.double().reshape(-1, H, d) for x in (q, k, v)), [100, 35], [100, 35], False, 0.25, dtype=dtype)
    _within("packed", core(q, k, v, edge_index=seqs, attn_type="flash").view(-1, H, d), ref["out"], ref["out_bound"])
    freq = bf.RotaryFrequencies(d, device=hip_device)
    turned = CoreAttention(H * d, 0.0, H, 1, rotary=freq)
    qr, kr = bf.rotary_embedding(q.reshape(-1, H, d), k.reshape(-1, H, d), freq,
                                 positions=torch.arange(S, device=hip_device).repeat(b))
    assert torch.equal(turned(q, k, v, attn_type="flash"), core(qr.view_as(q), kr.view_as(k), v, attn_type="flash"))
    with pytest.raises(NotImplementedError, match="bias"):
        core(q, k, v, torch.zeros(1, S, S, H, device=hip_device), attn_type="flash")
    with pytest.raises(NotImplementedError, match="dropout"):
        CoreAttention(H * d, 0.1, H, 1).train()(q, k, v, attn_type="flash")
    import copy
    again = copy.deepcopy(core)
    assert torch.equal(again(q, k, v, attn_type="flash"), core(q, k, v, attn_type="flash"))
    assert CoreAttention(H * d, 0.1, H, 1).eval()(q, k, v, attn_type="flash").shape == (b, S, H * d)


def test_what_inference_mode_builds_serves_training(hip_device):
    """Validation before training: sequences and frequencies built in inference mode, by the flash path or by hand."""
    from budgetformer_amd.attention import CoreAttention
    bf = _bf()
    b, S, H, d = 2, 40, 2, 16
    x = _randn(1, b, S, H, d, dev=hip_device)
    ld = torch.full((H,), -0.1, device=hip_device)

    def train(core, seqs, freq):
        t = x.clone().requires_grad_(True)
        flash = core(t, t, t, attn_type="flash")
        r = t.view(-1, H, d)
        q, k = bf.rotary_embedding(r, r, freq, seqs=seqs)
        outs = [flash, bf.packed_attention(q, k, r, seqs), bf.linear_attention(r, r, r, ld, seqs)]
        return outs + [g for o in outs for g in torch.autograd.grad(o.sum(), t, retain_graph=True)]

    def build():
        off = torch.arange(0, b * S + 1, S, device=hip_device)
        return (bf.RotaryFrequencies(d, device=hip_device), [bf.PackedSequences.from_lengths([S] * b, causal=True, device=hip_device),
                bf.PackedSequences.from_offsets(off, causal=True), bf.PackedSequences.from_offsets(off, n_q=b * S, causal=True, check=False)])

    freq, seqs = build()
    ref = train(CoreAttention(H * d, 0.0, H, 1, rotary=freq), seqs[0], freq)
    with torch.inference_mode():
        freq, seqs = build()
        core = CoreAttention(H * d, 0.0, H, 1, rotary=freq.to(hip_device))
        y = core(x, x, x, attn_type="flash")
        assert torch.equal(y, ref[0])
    for s in seqs:
        for a, r in zip(train(core, s, freq), ref):
            assert torch.equal(a, r)


# ------------------------------------------------------------------ streams, graphs, refusals
def _layer(bf, q, k, v, do, freq, ld, seqs):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    qr, kr = bf.rotary_embedding(leaves[0], leaves[1], freq, seqs=seqs)
    a, b = bf.packed_attention(qr, kr, leaves[2], seqs), bf.linear_attention(*leaves, ld, seqs)
    return [a, b, *torch.autograd.grad((a, b), leaves, (do, do))]


def test_a_captured_layer_replays(hip_device):
    bf = _bf()
    lens = [300, 1, 64, 400]
    n, H, d = sum(lens), 4, 64
    base = [_randn(i, n, H, d, dtype=torch.bfloat16, dev=hip_device) for i in range(4)]
    q, k, v, do = (x.clone() for x in base)
    freq, ld = bf.RotaryFrequencies(d, device=hip_device), torch.full((H,), -0.05, device=hip_device)
    seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
    step = [_randn(9, 3, H, d, dtype=torch.bfloat16, dev=hip_device) for _ in range(3)]
    state = _randn(10, 3, H, d, d, dev=hip_device)

    def every():
        return _layer(bf, q, k, v, do, freq, ld, seqs) + list(bf.linear_attention_step(*step, ld, state))

    alive = _layer(bf, q, k, v, do, freq, ld, seqs)            # an eager graph that lives through the capture
    side = torch.cuda.Stream(device=hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        every()
    torch.cuda.current_stream(hip_device).wait_stream(side)
    torch.cuda.synchronize(hip_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = every()
    for rep in range(4):
        for x, y in zip((q, k, v, do), base):
            x.copy_(y * (0.5 + 0.3 * rep))
        state.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize(hip_device)
        got = [x.clone() for x in captured]
        _ = torch.randn(1 << 18, device=hip_device).sum().item()
        for i, (x, y) in enumerate(zip(got, every())):
            assert torch.equal(x, y), (rep, i)
    del alive


def test_a_captured_flash_layer_replays_after_other_shapes(hip_device):
    from budgetformer_amd.attention import CoreAttention
    H, d = 2, 32
    core = CoreAttention(H * d, 0.0, H, 1)
    x, do = _randn(1, 3, 90, H, d, dtype=torch.bfloat16, dev=hip_device), _randn(2, 3, 90, H * d, dtype=torch.bfloat16, dev=hip_device)
    base = x.clone()

    def every(t):
        leaf = t.detach().requires_grad_(True)
        out = core(leaf, leaf, leaf, attn_type="flash")
        return [out, *torch.autograd.grad(out, leaf, do)]

    side = torch.cuda.Stream(device=hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        every(x)
    torch.cuda.current_stream(hip_device).wait_stream(side)
    torch.cuda.synchronize(hip_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = every(x)
    for rep in range(3):
        for b in range(1, 9):                              # more shapes than the layer keeps
            y = _randn(b, b, 70 + rep, H, d, dtype=torch.bfloat16, dev=hip_device)
            core(y, y, y, attn_type="flash")
        junk = [torch.full((n,), 2 ** 30, dtype=torch.int32, device=hip_device) for n in (4, 270, 540, 128, 1024) * 20]
        x.copy_(base * (0.5 + rep))
        graph.replay()
        torch.cuda.synchronize(hip_device)
        got = [t.clone() for t in captured]
        for a, r in zip(got, every(x)):
            assert torch.equal(a, r)
        del junk


def test_sequences_built_under_capture(hip_device):
    """From device offsets without the check, anew at each replay; what would read or copy from the host is refused and
    leaves the capture as it is."""
    bf = _bf()
    off = torch.tensor([0, 20, 50], device=hip_device)
    x = _randn(1, 60, 2, 16, dev=hip_device)

    def every():
        return bf.packed_attention(x, x, x, bf.PackedSequences.from_offsets(off, n_q=60, causal=True, check=False))

    every()
    torch.cuda.synchronize(hip_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="not for graph capture"):
            bf.PackedSequences.from_lengths([20, 40], device=hip_device)
        with pytest.raises(RuntimeError, match="not for graph capture"):
            bf.PackedSequences.from_offsets(off)
        out = every()
    for ends in ([20, 50], [1, 60], [0, 33], [25, 25]):
        off[1:] = torch.tensor(ends, device=hip_device)
        graph.replay()
        torch.cuda.synchronize(hip_device)
        got = out.clone()
        assert torch.equal(got, every())


def test_two_streams_at_once(hip_device):
    """Calls of different sizes on two streams, with their pieces and carries in flight together."""
    bf = _bf()
    freq, ld = bf.RotaryFrequencies(32, device=hip_device), torch.full((4,), -0.05, device=hip_device)
    jobs = []
    for i, lens in enumerate(([700, 3], [64] * 9)):
        args = [_randn(10 * i + j, sum(lens), 4, 32, dtype=torch.bfloat16, dev=hip_device) for j in range(4)]
        jobs.append((args, bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)))
    alone = [_layer(bf, *a, freq, ld, s) for a, s in jobs]
    torch.cuda.synchronize(hip_device)
    streams = [torch.cuda.Stream(device=hip_device) for _ in jobs]
    for _ in range(3):
        got = []
        for st, (a, s) in zip(streams, jobs):
            with torch.cuda.stream(st):
                got.append(_layer(bf, *a, freq, ld, s))
        torch.cuda.synchronize(hip_device)
        for x, y in zip(got, alone):
            assert all(torch.equal(p, r) for p, r in zip(x, y))


def test_sequences_built_on_another_stream(hip_device):
    """A stream that uses sequences another one still builds waits for them; they may be dropped while it reads."""
    bf = _bf()
    lens = [300, 40]
    q = _randn(1, 340, 2, 32, dev=hip_device)
    ref = bf.packed_attention(q, q, q, bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device))
    build, use = torch.cuda.Stream(device=hip_device), torch.cuda.Stream(device=hip_device)
    torch.cuda.synchronize(hip_device)
    big = torch.randn(4096, 4096, device=hip_device)
    for _ in range(3):
        with torch.cuda.stream(build):
            x = big
            for _ in range(4):
                x = x @ big                                    # work before the spans on their stream
            seqs = bf.PackedSequences.from_lengths(lens, causal=True, device=hip_device)
        with torch.cuda.stream(use):
            got = bf.packed_attention(q, q, q, seqs)
        del seqs
        torch.cuda.synchronize(hip_device)
        assert torch.equal(got, ref)


def test_second_derivatives_are_refused(hip_device):
    bf = _bf()
    seqs = bf.PackedSequences.from_lengths([20], causal=True, device=hip_device)
    q = _randn(1, 20, 2, 16, dev=hip_device).requires_grad_(True)
    freq, ld = bf.RotaryFrequencies(16, device=hip_device), torch.zeros(2, device=hip_device)
    for f in (lambda: bf.packed_attention(q, q, q, seqs), lambda: bf.linear_attention(q, q, q, ld, seqs),
              lambda: bf.rotary_embedding(q, None, freq, seqs=seqs)):
        g, = torch.autograd.grad(f().square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(hip_device, grad):
    """A dual tensor, with or without a gradient wanted, in any place and also under no_grad: no result without its tangent."""
    import torch.autograd.forward_ad as fwd
    bf = _bf()
    seqs = bf.PackedSequences.from_lengths([20], causal=True, device=hip_device)
    x, ld, s = _randn(1, 20, 2, 16, dev=hip_device).requires_grad_(grad), torch.zeros(2, device=hip_device), torch.zeros(20, 2, 16, 16, device=hip_device)
    freq = bf.RotaryFrequencies(16, device=hip_device)
    p = x.detach()
    with fwd.dual_level():
        d, dl, ds = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, ld, s))
        calls = [lambda: bf.packed_attention(d, p, p, seqs), lambda: bf.packed_attention(p, p, d, seqs),
                 lambda: bf.packed_attention(x, d, p, seqs, with_lse=True),
                 lambda: bf.rotary_embedding(d, None, freq, seqs=seqs), lambda: bf.rotary_embedding(x, d, freq, seqs=seqs),
                 lambda: bf.linear_attention(d, p, p, ld, seqs), lambda: bf.linear_attention(x, p, d, ld, seqs),
                 lambda: bf.linear_attention(p, p, p, dl, seqs),
                 lambda: bf.linear_attention(p, p, p, ld, seqs, initial_state=fwd.make_dual(torch.zeros(1, 2, 16, 16, device=hip_device),
                                                                                           torch.ones(1, 2, 16, 16, device=hip_device)))]
        if not grad:
            calls += [lambda: bf.linear_attention_step(d, p, p, ld, s), lambda: bf.linear_attention_step(p, p, p, dl, s),
                      lambda: bf.linear_attention_step(p, p, p, ld, ds)]
        for f in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f()
    assert bf.packed_attention(p, p, p, seqs).shape == p.shape
    with pytest.raises(Exception):                         # as a transform does it
        torch.func.jvp(lambda t: bf.packed_attention(t, t, t, seqs), (p,), (torch.ones_like(p),))


def test_offsets_that_change_afterwards_do_not_matter(hip_device):
    bf = _bf()
    off = torch.tensor([0, 5, 40], dtype=torch.int32, device=hip_device)
    seqs = bf.PackedSequences.from_offsets(off, causal=True)
    q, ld = _randn(1, 40, 2, 16, dev=hip_device), torch.full((2,), -0.1, device=hip_device)
    a = bf.linear_attention(q, q, q, ld, seqs, return_state=True)
    off.zero_()
    for x, y in zip(a, bf.linear_attention(q, q, q, ld, seqs, return_state=True)):
        assert torch.equal(x, y)


def test_empty_batches(hip_device):
    bf = _bf()
    seqs = bf.PackedSequences.from_lengths([], causal=True, device=hip_device)
    q = torch.zeros(0, 2, 16, device=hip_device, requires_grad=True)
    out = bf.packed_attention(q, q, q, seqs)
    assert out.shape == (0, 2, 16)
    torch.autograd.grad(out.sum(), q)
    ld = torch.zeros(2, device=hip_device)
    out, state = bf.linear_attention(q, q, q, ld, seqs, return_state=True)
    assert out.shape == (0, 2, 16) and state.shape == (0, 2, 16, 16)
    freq = bf.RotaryFrequencies(16, device=hip_device)
    assert bf.rotary_embedding(q, None, freq, seqs=seqs).shape == (0, 2, 16)
    keys = bf.PackedSequences.from_lengths([0, 0], [3, 4], device=hip_device)     # keys without rows
    k = torch.ones(7, 2, 16, device=hip_device, requires_grad=True)
    g, = torch.autograd.grad(bf.packed_attention(q, k, k, keys).sum(), k)
    assert bool((g == 0).all())
    empty = bf.PackedSequences.from_lengths([0, 0], causal=True, device=hip_device)
    s0 = _randn(1, 2, 2, 16, 16, dev=hip_device)
    _, state = bf.linear_attention(q, q, q, ld, empty, initial_state=s0, return_state=True)
    assert torch.equal(state, s0)


@pytest.mark.parametrize("b,S", [(0, 7), (3, 0), (0, 0)])
def test_flash_of_empty_batches(hip_device, b, S):
    from budgetformer_amd.attention import CoreAttention
    bf = _bf()
    x = torch.zeros(b, S, 2, 16, device=hip_device, requires_grad=True)
    for core in (CoreAttention(32, 0.0, 2, 1), CoreAttention(32, 0.0, 2, 1, rotary=bf.RotaryFrequencies(16, device=hip_device))):
        out = core(x, x, x, attn_type="flash")
        assert out.shape == (b, S, 32)
        assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape


def test_refusals(hip_device):
    bf = _bf()
    dev = hip_device
    seqs = bf.PackedSequences.from_lengths([10, 20], causal=True, device=dev)
    q = torch.zeros(30, 4, 32, device=dev)
    with pytest.raises(ValueError, match="cover"):
        bf.packed_attention(q[:29], q[:29], q[:29], seqs)
    with pytest.raises(ValueError, match="multiple"):
        bf.packed_attention(q, q[:, :3], q[:, :3], seqs)
    with pytest.raises(ValueError, match="disagree"):
        bf.packed_attention(q, q, q[:, :2], seqs)
    for d in (4, 12, 136):
        x = torch.zeros(30, 1, d, device=dev)
        with pytest.raises(NotImplementedError, match="head_dim"):
            bf.packed_attention(x, x, x, seqs)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            bf.packed_attention(q, q, q, seqs, scale=scale)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        bf.packed_attention(q.double(), q.double(), q.double(), seqs)
    with pytest.raises(ValueError, match="rows, heads"):
        bf.packed_attention(q[0], q, q, bf.PackedSequences.from_lengths([4], [30], device=dev))
    with pytest.raises(TypeError, match="PackedSequences"):
        bf.packed_attention(q, q, q, [10, 20])
    off = torch.tensor([0, 10, 30], device=dev)
    for bad, n in ((torch.tensor([1, 10, 30], device=dev), None), (torch.tensor([0, 20, 10], device=dev), None), (off, 29)):
        with pytest.raises(ValueError):
            bf.PackedSequences.from_offsets(bad, n_q=n)
    with pytest.raises(ValueError, match="must be given"):
        bf.PackedSequences.from_offsets(off, check=False)
    assert bf.PackedSequences.from_offsets(off, check=False, n_q=31).n_q == 31
    freq = bf.RotaryFrequencies(32, device=dev)
    pos = torch.zeros(30, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="positions"):
        bf.rotary_embedding(q, None, freq)
    with pytest.raises(ValueError, match="positions"):
        bf.rotary_embedding(q, None, freq, positions=pos[:29])
    with pytest.raises(ValueError, match="int32 or int64"):
        bf.rotary_embedding(q, None, freq, positions=pos.float())
    with pytest.raises(ValueError, match="rotated values"):
        bf.rotary_embedding(q[..., :16], None, freq, positions=pos)
    with pytest.raises(ValueError, match="disagree"):
        bf.rotary_embedding(q, q[:20], freq, positions=pos)
    ld = torch.zeros(4, device=dev)
    with pytest.raises(ValueError, match="causal"):
        bf.linear_attention(q, q, q, ld, bf.PackedSequences.from_lengths([30], device=dev))
    with pytest.raises(ValueError, match="log_decay"):
        bf.linear_attention(q, q, q, ld[:3], seqs)
    with pytest.raises(NotImplementedError, match="constants"):
        bf.linear_attention(q, q, q, ld.clone().requires_grad_(True), seqs)
    with pytest.raises(ValueError, match="init_state"):
        bf.linear_attention(q, q, q, ld, seqs, initial_state=torch.zeros(1, 4, 32, 32, device=dev))
    s = torch.zeros(30, 4, 32, 32, device=dev)
    with pytest.raises(ValueError, match="state must be"):
        bf.linear_attention_step(q, q, q, ld, s[:29])
    with pytest.raises(NotImplementedError, match="gradients"):
        bf.linear_attention_step(q.clone().requires_grad_(True), q, q, ld, s)
