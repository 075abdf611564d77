"""Host-side checks of attention with a learned bias by buckets (CPU): the C ABI's refusals before any launch, workspaces, the struct
mirror, the layer's parameter. No kernel runs here."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import budgetformer_amd as bf
from budgetformer_amd import _native as N
from budgetformer_amd.sequences import PackedSequences

BUF = (C.c_int64 * 64)()
P = C.c_void_p((C.addressof(BUF) + 15) // 16 * 16)          # 16-byte aligned host memory, never read


def _attn(**kw):
    a = N.PackedAttn(n_q=4, n_k=4, heads_q=2, heads_k=1, head_dim=16, dtype=N.BF_DTYPE_BF16, row_span=P, key_span=P, scale=0.25)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (32, 16), (16, 16), (16, 16)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def _bias(**kw):
    b = N.PackedBias(table=P, map=P, positions=P, buckets=8, reach=16)
    for name, value in kw.items():
        setattr(b, name, value)
    return b


def _fwd(a, b, scratch=P):
    N.call("bf_packed_attn_bias_fwd", C.byref(a), C.byref(b), P, P, P, P, None, P, scratch, None)


def _bwd(a, b, dtable=P, scratch=P):
    N.call("bf_packed_attn_bias_bwd", C.byref(a), C.byref(b), P, P, P, P, None, P, P, P, P, P, dtable, P, scratch, None)


@pytest.mark.parametrize("kw,match", [(dict(buckets=0), "buckets"), (dict(buckets=65), "buckets"), (dict(reach=-1), "distances"),
                                      (dict(reach=1025), "distances"), (dict(table=None), "table"), (dict(map=None), "map"),
                                      (dict(positions=None), "positions")])
def test_bias_arguments(kw, match):
    lib = N.load()
    for call in (_fwd, _bwd):
        with pytest.raises(ValueError, match=match):
            call(_attn(), _bias(**kw))
    assert lib.bf_packed_attn_bias_fwd_floats(C.byref(_attn()), C.byref(_bias(**kw))) == -1
    assert lib.bf_packed_attn_bias_bwd_floats(C.byref(_attn()), C.byref(_bias(**kw))) == -1
    assert lib.bf_packed_attn_bias_rest(C.byref(_attn()), C.byref(_bias(**kw))) == 0
    with pytest.raises(ValueError, match="no bias"):
        N.call("bf_packed_attn_bias_fwd", C.byref(_attn()), None, P, P, P, P, None, P, P, None)


def test_attention_arguments_are_checked_too():
    with pytest.raises(ValueError, match="scale"):
        _fwd(_attn(scale=0.0), _bias())
    with pytest.raises(NotImplementedError, match="head_dim"):
        _bwd(_attn(head_dim=12), _bias())


def test_group_heads_times_distances():
    """What a workgroup holds of the table by distance: 16384 values."""
    lib = N.load()
    wide = lambda heads, reach: lib.bf_packed_attn_bias_fwd_floats(C.byref(_attn(heads_q=heads)), C.byref(_bias(reach=reach)))   # noqa: E731
    assert wide(7, 1024) >= 0 and wide(62, 128) >= 0
    assert wide(8, 1024) == -1 and wide(63, 128) == -1
    with pytest.raises(NotImplementedError, match="key head"):
        _fwd(_attn(heads_q=8), _bias(reach=1024))


def test_workspaces():
    with pytest.raises(ValueError, match="scratch"):
        _bwd(_attn(), _bias(), scratch=None)
    with pytest.raises(ValueError, match="dtable"):
        _bwd(_attn(), _bias(), dtable=None)
    lib = N.load()
    assert lib.bf_packed_attn_bias_bwd_floats(C.byref(_attn()), C.byref(_bias())) > 0
    _fwd(_attn(n_q=0), _bias(positions=None), scratch=None)                       # no rows: nothing to do


def test_struct_mirror_matches_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    fields = [f[0] for f in N.PackedBias._fields_]
    src = tmp_path / "sizes.c"
    lines = "".join(f'printf("%zu\\n", offsetof(bf_packed_bias, {f}));' for f in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "budgetformer_hip.h"\nint main(void) {'
                   f'printf("%zu\\n", sizeof(bf_packed_bias));{lines} return 0; }}\n')
    exe = tmp_path / "sizes"
    subprocess.run([gcc, "-I", os.path.dirname(N._HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(N.PackedBias)] + [getattr(N.PackedBias, f).offset for f in fields]


def test_layer_parameter(monkeypatch):
    monkeypatch.setattr(PackedSequences, "_device", staticmethod(torch.device))
    buckets = bf.RelativeBuckets(8, 16, device="cpu")
    layer = bf.CoreAttention(32, 0.0, 4, buckets=buckets)
    assert [n for n, _ in layer.named_parameters()] == ["relative_bias"] and tuple(layer.relative_bias.shape) == (4, 8)
    assert not list(bf.CoreAttention(32, 0.0, 4).parameters())                   # as it was
    assert list(layer.state_dict()) == ["relative_bias"]
