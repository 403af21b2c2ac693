"""The C ABI of the delta rule and the block norms without a GPU: headers, exports, struct layouts, argument checks,
and the dispatcher operators' shape-only implementations and autograd formulas."""

import ctypes
import os
import re
import subprocess
import tempfile

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT

STRUCTS = {"delta_b200.h": ["DeltaFwdArgs", "DeltaBwdArgs", "DeltaStepArgs"],
           "block_norm_b200.h": ["GatedNormArgs", "ResidualNormArgs"]}
INC = os.path.join(ROOT, "include")


@pytest.mark.parametrize("header", sorted(STRUCTS))
def test_exports(header):
    from kernels import _lib
    names = re.findall(r"EMA_API\s+[\w\s\*]+?\b(\w+)\s*\(", open(os.path.join(INC, header)).read())
    assert len(names) >= 5
    for n in names:
        assert hasattr(_lib.lib, n), n


@pytest.mark.parametrize("header,struct", [(h, s) for h in sorted(STRUCTS) for s in STRUCTS[h]])
def test_every_field_offset_matches_header(header, struct):
    from kernels import _lib
    cls = getattr(_lib, struct)
    fields = [f[0] for f in cls._fields_]
    code = f'#include "{header}"\n#include <stdio.h>\n#include <stddef.h>\nint main(){{printf("%zu", sizeof({struct}));\n'
    code += "".join(f'printf(" %zu", offsetof({struct}, {f}));\n' for f in fields) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(code)
        subprocess.run(["gcc", "-I", INC, c, "-o", exe], check=True)
        out = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _delta(cls, **kw):
    a = cls()
    base = dict(batch=1, seqlen=8, nheads=4, headdim=64, dstate=64, ngroups=2, dtype=1, scale=1.0)
    base.update({"nseq": 1} if hasattr(a, "nseq") else {"tokens": 1, "slots": 1})
    if not hasattr(a, "nseq"):
        base.pop("seqlen")
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


# (1: invalid argument, 2: unsupported, 3: workspace; every pointer is checked before anything is launched)
@pytest.mark.parametrize("kw,code", [(dict(ngroups=3), 1), (dict(headdim=12), 2), (dict(headdim=136), 2),
                                     (dict(dstate=96), 2), (dict(dtype=7), 1), (dict(nseq=3), 1), (dict(batch=-1), 1),
                                     (dict(), 1), (dict(nheads=131072), 2), (dict(flags=2), 1)])
def test_sequence_launchers_refuse(kw, code):
    from kernels import _lib
    for name in ("delta_fwd", "delta_bwd"):
        cls = _lib.DeltaFwdArgs if name == "delta_fwd" else _lib.DeltaBwdArgs
        assert getattr(_lib.lib, name + "_launch")(_delta(cls, **kw), None) == code
        assert name in _lib.lib.ema_last_error().decode()


def test_sequence_launcher_refuses_misaligned_rows_and_small_buffers():
    from kernels import _lib
    a = _delta(_lib.DeltaFwdArgs)
    for f in ("q", "k", "v", "g", "beta", "out"):
        setattr(a, f, 4096)
    for f in ("q", "k", "v", "out"):
        setattr(a, f + "_stride", (_lib._i64 * 3)(512, 64, 64))
    assert _lib.lib.delta_fwd_launch(a, None) == 3
    a.workspace, a.workspace_bytes = 4096, 1
    assert _lib.lib.delta_fwd_launch(a, None) == 3
    a.q_stride = (_lib._i64 * 3)(512, 65, 64)
    assert _lib.lib.delta_fwd_launch(a, None) == 1
    a.q_stride, a.v = (_lib._i64 * 3)(512, 64, 64), 4098
    assert _lib.lib.delta_fwd_launch(a, None) == 1


@pytest.mark.parametrize("kw,code", [(dict(ngroups=3), 1), (dict(headdim=264), 2), (dict(dstate=32), 2), (dict(dtype=9), 1),
                                     (dict(slots=0), 1), (dict(batch=70000), 2), (dict(), 1)])
def test_step_launcher_refuses(kw, code):
    from kernels import _lib
    assert _lib.lib.delta_step_launch(_delta(_lib.DeltaStepArgs, **kw), None) == code
    assert "delta_step" in _lib.lib.ema_last_error().decode()


def test_empty_calls_are_no_ops():
    from kernels import _lib
    assert _lib.lib.delta_fwd_launch(_delta(_lib.DeltaFwdArgs, batch=0, nseq=0), None) == 0
    assert _lib.lib.delta_step_launch(_delta(_lib.DeltaStepArgs, batch=0), None) == 0


@pytest.mark.parametrize("kw,code", [(dict(dim=0), 1), (dict(group_size=48), 1), (dict(dtype=5), 1), (dict(eps=-1.0), 1),
                                     (dict(rows=-1), 1), (dict(), 1), (dict(rows=0, weight=4096), 0)])
def test_gated_norm_refuses(kw, code):
    from kernels import _lib
    a = _lib.GatedNormArgs(rows=2, dim=64, group_size=64, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    assert _lib.lib.gated_norm_fwd_launch(a, None) == code


def test_residual_norm_refuses():
    from kernels import _lib
    a = _lib.ResidualNormArgs(rows=2, dim=64, dtype=1, residual_dtype=2, eps=1e-5, scale=1.0)
    assert _lib.lib.residual_norm_fwd_launch(a, None) == 2
    a.residual_dtype = 0
    assert _lib.lib.residual_norm_fwd_launch(a, None) == 1
    for f in ("weight", "h", "dy", "dx", "dweight"):
        setattr(a, f, 4096)
    assert _lib.lib.residual_norm_bwd_launch(a, None) == 3  # no workspace


def test_buffer_sizes_cover_packed_calls():
    """A packed call may use a slot per 64 tokens and one per sequence; sizes grow with both."""
    from kernels import _lib
    size = lambda L, n: _lib.lib.delta_saved_bytes(1, L, n, 2, 64, 64, 1, 1, 0)  # noqa: E731
    assert size(640, 1) < size(640, 5) and size(640, 5) < size(6400, 5)


def test_python_refuses_cpu_tensors():
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    from kernels.gated_delta import gated_delta_rule, gated_delta_step
    q, v, g = torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2)
    x, w = torch.zeros(3, 8), torch.ones(8)
    for call in (lambda: gated_delta_rule(q, q, v, g, g), lambda: gated_delta_step(q, q, v, g, g, torch.zeros(1, 2, 64, 64)),
                 lambda: rms_norm_gated(x, x, w), lambda: residual_rms_norm(x, x, w)):
        with pytest.raises(ValueError):
            call()


def test_fake_shapes_and_autograd_formulas():
    import kernels.block_norm  # noqa: F401
    import kernels.gated_delta  # noqa: F401
    ops = torch.ops.ema_b200
    with FakeTensorMode():
        mk = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        q, v, g = mk(2, 70, 2, 128), mk(2, 70, 4, 64), mk(2, 70, 4, dt=torch.float32)
        o, fin, saved = ops.delta_fwd(q, q, v, g, g, None, None, 1.0)
        assert o.shape == v.shape and fin.shape == (2, 4, 64, 128) and saved.dtype == torch.uint8
        assert ops.delta_step(q, q, v, g, g, fin, None, 1.0).shape == v.shape
    meta = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="meta", requires_grad=True)  # noqa: E731
    q, k, v = meta(2, 70, 2, 128), meta(2, 70, 2, 128), meta(2, 70, 4, 64)
    g, beta, s0 = meta(2, 70, 4, dt=torch.float32), meta(2, 70, 4), meta(2, 4, 64, 128, dt=torch.float32)
    o, fin, _ = ops.delta_fwd(q, k, v, g, beta, s0, None, 1.0)
    (o.float().sum() + fin.sum()).backward()
    x, z, w = meta(3, 64), meta(3, 64), meta(64, dt=torch.float32)
    ops.gated_norm_fwd(x, z, w, 1e-5, 32, True).sum().backward()
    x2, r, w2 = meta(3, 64), meta(3, 64, dt=torch.float32), meta(64)
    y, h = ops.residual_norm_fwd(x2, r, w2, 1e-5, 0.5)
    (y.float().sum() + h.sum()).backward()
    for t in (q, k, v, g, beta, s0, x, z, w, x2, r, w2):
        assert t.grad is not None and t.grad.shape == t.shape and t.grad.dtype == t.dtype
