"""Host-side checks of the operators over packed sequences (CPU): the C ABI's refusals before any launch, the struct
mirrors, the Python surface's own checks. No kernel runs here."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import budgetformer_amd as bf
from budgetformer_amd import _native as N

BUF = (C.c_int64 * 64)()
P = C.c_void_p((C.addressof(BUF) + 15) // 16 * 16)          # 16-byte aligned host memory, never read


def _attn(**kw):
    a = N.PackedAttn(n_q=4, n_k=4, heads_q=2, heads_k=1, head_dim=16, dtype=N.BF_DTYPE_BF16, row_span=P, key_span=P, scale=0.25)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (32, 16), (16, 16), (16, 16)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


_TWO = (C.c_int64 * 2)(8, 8)


def _fwd(a, q=P, k=P, v=P, out=P):
    N.call("bf_packed_attn_fwd", C.byref(a), q, k, v, out, None, P, P, None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(heads_q=3, heads_k=2), "multiple"), (dict(heads_k=0), "heads"),
    (dict(n_q=-1), "rows"), (dict(n_k=2 ** 31), "keys"), (dict(n_q=2 ** 30), "rows"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(row_span=None), "spans"),
    (dict(longest=-1), "longest")])
def test_packed_attention_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        _fwd(_attn(**kw))
    assert N.load().bf_packed_attn_fwd_floats(C.byref(_attn(**kw))) == -1


def test_packed_attention_scales_at_the_end_of_float32():
    """A scale whose product with log2 e is infinite would make a score of 0 a NaN."""
    lib = N.load()
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(scale=2e38))) >= 0
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(scale=2.5e38))) == -1


@pytest.mark.parametrize("d", [0, 4, 12, 136])
def test_packed_attention_head_dims(d):
    with pytest.raises(NotImplementedError, match="head_dim"):
        _fwd(_attn(head_dim=d))


def test_rows_leave_room_for_a_tile_behind_the_last():
    """Ends of tiles, pieces and segments are formed in 32 bits, behind the last row too."""
    most = 2 ** 31 - 2 ** 17
    lib = N.load()
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(n_k=most - 1))) >= 0
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(n_k=most))) == -1
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(n_q=most // 2 - 1))) >= 0
    assert lib.bf_packed_attn_fwd_floats(C.byref(_attn(n_q=most // 2))) == -1
    assert lib.bf_linear_attn_fwd_floats(C.byref(_lin(n=most - 1))) >= 0
    assert lib.bf_linear_attn_fwd_floats(C.byref(_lin(n=most))) == -1
    with pytest.raises(ValueError, match="a token of"):
        N.call("bf_rotary", P, None, 1, 2 ** 20, 0, 65, 2, 0, _TWO, _TWO, P, 1, P, 1.0, 0, 0, P, None, None)


def test_packed_attention_addresses_and_strides():
    off = C.c_void_p(P.value + 2)
    for kw in (dict(q=off), dict(k=off), dict(v=off), dict(out=off)):
        with pytest.raises(ValueError, match="aligned"):
            _fwd(_attn(), **kw)
    a = _attn()
    a.k_stride[0] = 20
    with pytest.raises(ValueError, match="16-byte steps"):
        _fwd(a)
    with pytest.raises(ValueError, match="bad arguments"):
        _fwd(_attn(), q=None)
    with pytest.raises(ValueError, match="no key spans"):
        N.call("bf_packed_attn_bwd", C.byref(_attn(key_span=None)), P, P, P, P, None, P, P, P, P, P, P, P, None)
    _fwd(_attn(n_q=0))                                       # nothing to do, nothing launched


def test_rotary_arguments():
    s = (C.c_int64 * 2)(16, 16)

    def call(n=4, hx=1, hy=0, dim=16, rot=16, dtype=0, x=P, y=None):
        N.call("bf_rotary", x, y, n, hx, hy, dim, rot, dtype, s, s, P, 1, P, 1.0, 0, 0, P, P, None)

    for kw in (dict(rot=0), dict(rot=3), dict(rot=18), dict(dim=2000, rot=1026)):
        with pytest.raises(ValueError, match="even number"):
            call(**kw)
    for kw in (dict(n=-1), dict(hx=0), dict(hy=-1), dict(dim=0)):
        with pytest.raises(ValueError, match="bad sizes"):
            call(**kw)
    with pytest.raises(ValueError, match="dtype"):
        call(dtype=9)
    for kw in (dict(x=None), dict(hy=2)):
        with pytest.raises(ValueError, match="bad arguments"):
            call(**kw)
    call(n=0)


def _lin(**kw):
    a = N.LinearAttn(n=4, n_seq=1, heads=2, dim_k=16, dim_v=16, dtype=N.BF_DTYPE_F32, row_span=P, key_span=P, offsets=P,
                     log_decay=P, scale=1.0)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (32, 16), (32, 16), (32, 16)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_linear_attention_arguments():
    def call(a, x=P):
        N.call("bf_linear_attn_fwd", C.byref(a), x, P, P, P, P, None)

    for kw, match in ((dict(dtype=5), "dtype"), (dict(n=-1), "sizes"), (dict(heads=0), "sizes"), (dict(n=2 ** 31), "sizes"),
                      (dict(log_decay=None), "decays"), (dict(row_span=None), "spans"), (dict(scale=float("nan")), "scale"),
                      (dict(init=P, offsets=None), "states"), (dict(longest=-1), "longest"), (dict(final_state=P, offsets=None), "states")):
        with pytest.raises(ValueError, match=match):
            call(_lin(**kw))
        assert N.load().bf_linear_attn_fwd_floats(C.byref(_lin(**kw))) == -1
        assert N.load().bf_linear_attn_bwd_floats(C.byref(_lin(**kw))) == -1
        with pytest.raises(ValueError, match=match):
            N.call("bf_linear_attn_bwd", C.byref(_lin(**kw)), P, P, P, P, P, P, P, P, None)
    for d in (4, 20, 136):
        with pytest.raises(NotImplementedError, match="head dims"):
            call(_lin(dim_k=d))
        with pytest.raises(NotImplementedError, match="head dims"):
            call(_lin(dim_v=d))
        with pytest.raises(NotImplementedError, match="head dims"):
            N.call("bf_linear_attn_step", P, P, P, P, P, 1, 1, d, 16, 0, 1.0, P, P, None)
    with pytest.raises(ValueError, match="aligned"):
        call(_lin(), x=C.c_void_p(P.value + 4))
    with pytest.raises(ValueError, match="sequences"):
        N.call("bf_linear_attn_step", P, P, P, P, P, 2 ** 24, 1, 16, 16, 0, 1.0, P, P, None)
    call(_lin(n=0))
    N.call("bf_linear_attn_step", P, P, P, P, P, 0, 1, 16, 16, 0, 1.0, P, P, None)


def test_scratch_addresses():
    off = C.c_void_p(P.value + 4)
    with pytest.raises(ValueError, match="scratch must be 16-byte aligned"):
        N.call("bf_packed_attn_fwd", C.byref(_attn()), P, P, P, P, None, P, off, None)
    with pytest.raises(ValueError, match="scratch must be 16-byte aligned"):
        N.call("bf_packed_attn_bwd", C.byref(_attn()), P, P, P, P, None, P, P, P, P, P, P, off, None)
    with pytest.raises(ValueError, match="scratch must be 16-byte aligned"):
        N.call("bf_linear_attn_fwd", C.byref(_lin()), P, P, P, P, off, None)
    with pytest.raises(ValueError, match="aligned"):
        N.call("bf_linear_attn_bwd", C.byref(_lin()), P, P, P, P, P, P, P, off, None)


def test_spans_arguments():
    with pytest.raises(ValueError, match="32 bits"):
        N.call("bf_packed_spans", P, P, 1, 2 ** 31, 4, 0, P, P, None, None)
    with pytest.raises(ValueError, match="bad arguments"):
        N.call("bf_packed_spans", P, P, 1, 4, 4, 0, None, P, None, None)
    N.call("bf_packed_spans", None, None, 0, 0, 0, 0, None, None, None, None)


def test_host_tensors_and_bad_lengths_are_refused():
    with pytest.raises(ValueError, match="no CPU fallback"):
        bf.PackedSequences.from_lengths([1, 2], device="cpu")
    with pytest.raises(ValueError, match="no CPU fallback"):
        bf.PackedSequences.from_offsets(torch.tensor([0, 3]))
    for q, k, match in (([-1, 2], None, "negative"), ([1, 2], [3], "each sequence"), ([2 ** 30, 2 ** 30], None, "2\\^31"),
                        ([1], [2 ** 31], "2\\^31")):
        with pytest.raises(ValueError, match=match):
            bf.PackedSequences.from_lengths(q, k, device="cuda")
    for kw, match in ((dict(rot=3), "even"), (dict(rot=0), "even"), (dict(rot=8, base=1.0), "base"), (dict(rot=8, factor=0.0), "factor"),
                      (dict(rot=8, scaling="other"), "scaling"), (dict(rot=2, scaling="ntk"), "two pairs"),
                      (dict(rot=8, scaling="by_parts"), "original"), (dict(rot=8, amplitude=float("inf")), "amplitude"),
                      (dict(rot=8, device="cpu"), "no CPU fallback")):
        with pytest.raises(ValueError, match=match):
            bf.RotaryFrequencies(**kw)
    q = torch.zeros(2, 1, 8)
    with pytest.raises(NotImplementedError):                 # the operators have device kernels only
        bf.linear_attention_step(q, q, q, torch.zeros(1), torch.zeros(2, 1, 8, 8))


def test_sequences_that_a_capture_used_are_kept(monkeypatch):
    """The flash path's own sequences: the last four shapes, and every one that a capturing stream used."""
    from budgetformer_amd import attention
    built, capturing = [], [False]

    def from_lengths(lens, device=None):
        built.append(len(lens))
        return object()

    monkeypatch.setattr(attention.PackedSequences, "from_lengths", from_lengths)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    cache, dev = attention._BatchSequences(), torch.device("cuda:0")
    first = cache.get(1, 10, dev)
    capturing[0] = True
    assert cache.get(1, 10, dev) is first and built == [1]
    capturing[0] = False
    others = [cache.get(b, 10, dev) for b in range(2, 12)]
    assert cache.get(1, 10, dev) is first and built == list(range(1, 12))
    assert all(cache.get(b, 10, dev) is others[b - 2] for b in range(8, 12)) and len(built) == 11
    cache.get(2, 10, dev)                                    # one of the first is built again
    assert built[-1] == 2 and len(built) == 12


def test_lengths_from_the_host_are_refused_under_capture(monkeypatch):
    from budgetformer_amd import attention
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="not for graph capture"):
        bf.PackedSequences.from_lengths([3, 4])
    with pytest.raises(RuntimeError, match="not for graph capture"):
        attention._BatchSequences().get(2, 5, torch.device("cuda:0"))


def test_rotary_frequencies_follow_the_layer_to_another_device(monkeypatch):
    from budgetformer_amd import attention
    there = object.__new__(bf.RotaryFrequencies)
    there.rot, there.amplitude, there.turns = 8, 1.0, torch.zeros(4, device="meta")
    moved = []

    def to(self, device):
        got = object.__new__(bf.RotaryFrequencies)
        got.rot, got.amplitude, got.turns = self.rot, self.amplitude, torch.zeros(4, device=device)
        moved.append(got)
        return got

    monkeypatch.setattr(bf.RotaryFrequencies, "to", to)
    monkeypatch.setattr(attention, "rotary_embedding", lambda q, k, freq, seqs: (q, k) if freq.turns.device == q.device else None)
    monkeypatch.setattr(attention, "packed_attention", lambda q, k, v, seqs: q)
    seqs = object.__new__(bf.PackedSequences)
    seqs.n_q = seqs.n_k = 6
    core, x = bf.CoreAttention(16, 0.0, 2, 1, rotary=there), torch.zeros(2, 3, 2, 8)
    for _ in range(2):
        assert core(x, x, x, edge_index=seqs, attn_type="flash").shape == (2, 3, 16)
    assert len(moved) == 1 and core.rotary is moved[0]


def test_sequences_of_calls_from_several_threads(monkeypatch):
    import sys
    import threading
    from budgetformer_amd import attention
    monkeypatch.setattr(attention.PackedSequences, "from_lengths", lambda lens, device=None: len(lens))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cache, dev, wrong = attention._BatchSequences(), torch.device("cuda:0"), []

    def work(seed):
        try:
            for i in range(20000):
                b = (i * seed) % 7 + 1
                if cache.get(b, 3, dev) != b:
                    wrong.append(b)
        except Exception as e:                               # an entry gone between two steps
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2, 3, 5)]
    often = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)                              # a thread gives way between any two steps
    try:
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sys.setswitchinterval(often)
    assert not wrong


def test_operators_are_registered():
    ops = N.load_ops()
    for name in ("packed_spans", "packed_attn_fwd", "packed_attn_bwd", "rotary", "linear_attn_fwd", "linear_attn_bwd", "linear_attn_step",
                 "packed_attention", "rotary_embedding", "linear_attention"):
        assert str(getattr(ops, name).default._schema).startswith(f"bf::{name}(")


@pytest.mark.parametrize("struct,mirror", [("bf_packed_attn", "PackedAttn"), ("bf_linear_attn", "LinearAttn")])
def test_struct_mirrors_match_the_header(tmp_path, struct, mirror):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    cls = getattr(N, mirror)
    names = [f[0] for f in cls._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "budgetformer_hip.h"', "int main(void) {",
             f'  printf("%zu\\n", sizeof({struct}));']
    lines += [f'  printf("%zu\\n", offsetof({struct}, {f}));' for f in names] + ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run([cc, "-I", os.path.dirname(N._HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in names]
