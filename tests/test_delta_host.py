"""Host-side checks of the gated delta rule (CPU): the C ABI's refusals before any launch, workspaces, the struct mirror, the Python
surface's own checks. No kernel runs here."""
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


def _args(**kw):
    a = N.GatedDelta(n=4, n_seq=2, heads=4, heads_k=2, dim_k=16, dim_v=32, dtype=N.BF_DTYPE_BF16, offsets=P, log_gate=P, beta=P, scale=0.25)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (32, 16), (32, 16), (128, 32)
    for name, value in kw.items():
        if name.endswith("stride"):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return a


def _fwd(a, q=P, scratch=P, kept=None):
    N.call("bf_gated_delta_fwd", C.byref(a), q, P, P, P, kept, scratch, None)


def _bwd(a, **kw):
    x = dict(q=P, k=P, v=P, dout=P, kept=P, dq=P, dk=P, dv=P, dgate=P, dbeta=P, scratch=P)
    x.update(kw)
    N.call("bf_gated_delta_bwd", C.byref(a), *x.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(heads=3), "multiple"), (dict(heads_k=0), "heads"), (dict(heads=2 ** 21, heads_k=1), "heads"),
    (dict(n=-1), "sizes"), (dict(n=2 ** 31), "sizes"), (dict(n_seq=-1), "sizes"), (dict(n_seq=2 ** 31), "sizes"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(offsets=None), "offsets"),
    (dict(log_gate=None), "gates"), (dict(beta=None), "strengths"), (dict(longest=-1), "longest"),
    (dict(init=C.c_void_p(P.value + 4)), "aligned"), (dict(k_stride=(32, 12)), "strides"), (dict(q_stride=(-32, 16)), "strides")])
def test_arguments(kw, match):
    a = _args(**kw)
    lib = N.load()
    with pytest.raises(ValueError, match=match):
        _fwd(a)
    with pytest.raises(ValueError, match=match):
        _bwd(a)
    assert lib.bf_gated_delta_fwd_floats(C.byref(a), 0) == lib.bf_gated_delta_kept_floats(C.byref(a)) == -1
    assert lib.bf_gated_delta_bwd_floats(C.byref(a)) == -1


@pytest.mark.parametrize("d", [0, 4, 20, 136])
def test_head_dims(d):
    for kw in (dict(dim_k=d), dict(dim_v=d)):
        with pytest.raises(NotImplementedError, match="head dims"):
            _fwd(_args(**kw))
        with pytest.raises(NotImplementedError, match="head dims"):
            N.call("bf_gated_delta_step", C.byref(_args(**kw)), P, P, P, P, None)


def test_addresses_and_workspaces():
    with pytest.raises(ValueError, match="aligned"):
        _fwd(_args(), q=C.c_void_p(P.value + 2))
    with pytest.raises(ValueError, match="scratch"):
        _fwd(_args(), scratch=None)
    with pytest.raises(ValueError, match="aligned"):
        _fwd(_args(), kept=C.c_void_p(P.value + 4))
    for x in ("q", "dout", "kept", "dv", "dgate", "scratch"):
        with pytest.raises(ValueError, match="arguments"):
            _bwd(_args(), **{x: None})
    with pytest.raises(ValueError, match="sequences"):
        N.call("bf_gated_delta_step", C.byref(_args(n=2 ** 23)), P, P, P, P, None)
    with pytest.raises(ValueError, match="arguments"):
        N.call("bf_gated_delta_step", C.byref(_args()), P, P, P, P, None)               # no states


@pytest.mark.parametrize("kw", [dict(n_seq=2 ** 27), dict(n=2 ** 30, n_seq=2 ** 30), dict(n=2 ** 30, heads=2 ** 12, heads_k=2 ** 10)])
def test_more_than_a_launch_holds(kw):
    lib, a = N.load(), _args(**kw)
    with pytest.raises(NotImplementedError, match="a launch holds"):
        _fwd(a)
    with pytest.raises(NotImplementedError, match="a launch holds"):
        _bwd(a)
    assert lib.bf_gated_delta_fwd_floats(C.byref(a), 1) == lib.bf_gated_delta_kept_floats(C.byref(a)) == -1
    assert lib.bf_gated_delta_bwd_floats(C.byref(a)) == -1


def test_no_rows_is_no_work():
    _fwd(_args(n=0), scratch=None)
    _bwd(_args(n=0), q=None, kept=None, scratch=None)
    N.call("bf_gated_delta_step", C.byref(_args(n=0)), P, P, P, P, None)


def test_host_tensors_are_refused():
    x = torch.zeros(4, 2, 16)
    with pytest.raises(TypeError, match="PackedSequences"):
        bf.gated_delta_rule(x, x, x, x[..., 0], x[..., 0], None)
    with pytest.raises(NotImplementedError, match="CPU"):                       # no kernel is registered for host tensors
        bf.gated_delta_step(x, x, x, x[..., 0], x[..., 0], torch.zeros(4, 2, 16, 16))
    with pytest.raises(ValueError, match="beta must be"):
        bf.gated_delta_step(x, x, x, x[..., 0], x[:, 0, 0], torch.zeros(4, 2, 16, 16))
    with pytest.raises(NotImplementedError, match="no gradients"):
        bf.gated_delta_step(x, x, x, x[..., 0].clone().requires_grad_(True), x[..., 0], torch.zeros(4, 2, 16, 16))


def test_struct_mirror_matches_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    fields = [f[0] for f in N.GatedDelta._fields_]
    src = tmp_path / "sizes.c"
    lines = "".join(f'printf("%zu\\n", offsetof(bf_gated_delta, {f}));' for f in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "budgetformer_hip.h"\nint main(void) {'
                   f'printf("%zu\\n", sizeof(bf_gated_delta));{lines} return 0; }}\n')
    exe = tmp_path / "sizes"
    subprocess.run([gcc, "-I", os.path.dirname(N._HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(N.GatedDelta)] + [getattr(N.GatedDelta, f).offset for f in fields]
