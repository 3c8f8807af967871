"""Gated feed-forward block: what its entry points refuse, before any launch.  No GPU needed."""
import ctypes
import os
import subprocess

import pytest
import torch

from vmamba_b200 import _lib


def params():
    buf = (ctypes.c_float * 64)()
    a = (ctypes.addressof(buf) + 63) // 64 * 64
    p = _lib.GatedMlpParams()
    for f in ("x", "w1", "w2", "h", "y"):
        setattr(p, f, a)
    p.tokens, p.channels, p.hidden, p.outputs, p.x_row_stride, p.dtype, p.act = 10, 16, 32, 16, 16, _lib.SS2D_BF16, 1
    p.keep = buf
    return p, a


def test_refusals_of_the_c_interface():
    L = _lib.lib()
    before = _lib.launch_count()
    call = L.ss2d_gated_mlp_fwd
    assert call(None, None) == -1
    p, a = params()
    assert L.ss2d_gated_mlp_workspace_bytes(p) == 0 and L.ss2d_gated_mlp_workspace_bytes(None) < 0
    p.hidden, p.tokens = 4096, 100                                # few tiles, a long contraction: split, its parts in a workspace
    need = L.ss2d_gated_mlp_workspace_bytes(p)
    assert need >= 2 * 4 * 100 * 16 and call(p, None) == -8
    p.workspace, p.workspace_bytes = a, need - 1
    assert call(p, None) == -8
    p, a = params()
    for field, bad, code in (("x", None, -1), ("w2", None, -1), ("h", None, -1), ("y", None, -1), ("dtype", 9, -3), ("act", 0, -6), ("act", 3, -6),
                             ("tokens", 0, -2), ("hidden", -1, -2), ("x_row_stride", 15, -5), ("w1", a + 1, -4), ("h", a + 8, -4), ("b1", a + 1, -4),
                             ("y", a + 2, -4), ("tokens", 1 << 40, -6)):
        p, a = params()
        setattr(p, field, bad)
        assert call(p, None) == code, field
    b = _lib.GatedMlpBwdParams()
    assert L.ss2d_gated_mlp_bwd(None, None) == -1 and L.ss2d_gated_mlp_bwd(b, None) == -1 and L.ss2d_gated_mlp_bwd_workspace_bytes(b) < 0
    b.fwd, a = params()
    assert L.ss2d_gated_mlp_bwd(b, None) == -1                    # no dy
    b.dy = a
    assert L.ss2d_gated_mlp_bwd(b, None) == -5
    b.dy_row_stride = 16
    need = L.ss2d_gated_mlp_bwd_workspace_bytes(b)
    assert need >= 2 * 10 * 64
    assert L.ss2d_gated_mlp_bwd(b, None) == -8
    b.workspace, b.workspace_bytes = a, need - 1
    assert L.ss2d_gated_mlp_bwd(b, None) == -8
    b.workspace_bytes, b.dx = need, a + 2
    assert L.ss2d_gated_mlp_bwd(b, None) == -4
    assert _lib.launch_count() == before


def test_struct_layout(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = tmp_path / "sz.c"
    prog.write_text('#include "ss2d_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu\\n",sizeof(ss2d_gated_mlp_params),'
                    'offsetof(ss2d_gated_mlp_params,act),sizeof(ss2d_gated_mlp_bwd_params),offsetof(ss2d_gated_mlp_bwd_params,dy_row_stride));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(prog), "-o", str(exe)])
    A, B = _lib.GatedMlpParams, _lib.GatedMlpBwdParams
    assert [int(t) for t in subprocess.check_output([str(exe)]).split()] == [ctypes.sizeof(A), A.act.offset, ctypes.sizeof(B), B.dy_row_stride.offset]


def test_cpu_tensors_and_unknown_activations_are_refused():
    import vmamba_b200 as vb
    x, w1, w2 = torch.zeros(3, 8), torch.zeros(32, 8), torch.zeros(8, 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.gated_mlp_fn(x, w1, w2)
    with pytest.raises(ValueError, match="activation"):
        vb.gated_mlp_fn(x, w1, w2, act="relu")


def test_backward_workspace_holds_what_its_kernels_use():
    """Aligned 16-bit calls: the gradients of value and gate and sums.  Others keep value and gate in fp32 beside them; a workspace of the one is refused by the other."""
    L = _lib.lib()
    before = _lib.launch_count()
    M, C, H = 12544, 512, 2048
    def call(dtype=_lib.SS2D_BF16, off=0):
        b = _lib.GatedMlpBwdParams()
        b.fwd, a = params()
        b.fwd.tokens, b.fwd.channels, b.fwd.hidden, b.fwd.outputs, b.fwd.x_row_stride, b.fwd.dtype = M, C, H, C, C, dtype
        for f in ("dx", "dw1", "dw2", "db1", "db2"):
            setattr(b, f, a)
        b.dy, b.dy_row_stride = a + off, C
        return b, a
    sums = 4 * 2 ** 20 * 16                                       # splits of the weight gradients, of 2 H C elements at most
    need = L.ss2d_gated_mlp_bwd_workspace_bytes(call()[0])
    assert 4 * M * H <= need <= 4 * M * H + sums
    for other, size in ((call(off=2)[0], 4), (call(_lib.SS2D_F32)[0], 8)):
        assert L.ss2d_gated_mlp_bwd_workspace_bytes(other) >= (size + 8) * M * H
        other.workspace, other.workspace_bytes = call()[1], need
        assert L.ss2d_gated_mlp_bwd(other, None) == -8
    early, _ = call()
    early.dy = None                                               # a size asked for before the upstream gradient is known: enough for any
    assert L.ss2d_gated_mlp_bwd_workspace_bytes(early) >= 12 * M * H
    assert _lib.launch_count() == before


def kernels(M, C, H, O):
    """{(layout of the operands, kernel, split, whether a CTA walks three tiles or more and not all as many)} of a 16-bit call and its backward call"""
    L = _lib.lib()
    b = _lib.GatedMlpBwdParams()
    b.fwd, a = params()
    b.fwd.tokens, b.fwd.channels, b.fwd.hidden, b.fwd.outputs, b.fwd.x_row_stride, b.dy, b.dy_row_stride = M, C, H, O, C, a, O
    found = set()
    for product, (rows, cols, layout) in enumerate([(M, 2 * H, "gate"), (M, O, "NT"), (M, H, "gradients of value and gate"), (M, C, "NN"), (2 * H, C, "TN"), (O, H, "TN")]):
        code = L.ss2d_gated_mlp_kernel(b, product)
        assert code >= 16
        kernel, splits = code % 16, code // 16
        if kernel < 2:
            continue
        high, wide = (256 if kernel == 4 else 128), (128 if kernel == 2 or product == 2 else 256)
        tiles, walkers = -(-rows // high) * -(-cols // wide) * splits, 74 if kernel == 4 else 148
        found.add((layout, kernel, splits > 1, tiles > 2 * walkers and tiles % walkers != 0))
    return found


def test_shapes_of_the_gpu_tests_reach_every_kernel():
    from tests.test_gpu_gated_mlp import LARGE, SHAPES
    L = _lib.lib()
    small = set().union(*(kernels(*s) for s in SHAPES))
    found = small.union(*(kernels(*s) for s in LARGE))
    kinds = {("gate", k, False) for k in (2, 3, 4)} | {("gradients of value and gate", k, False) for k in (3, 4)} | \
            {(layout, k, split) for layout in ("NT", "NN", "TN") for k in (2, 3, 4) for split in (False, True)}
    assert {f[:3] for f in found} == kinds
    # what is never chosen for many tiles, wider ones being faster there: narrow tiles in front of the activation; unsplit narrow ones and split wide ones of most products
    many = {f[:3] for f in found if f[3]}
    assert many >= {k for k in kinds if k[1] == 4} | {("gate", 3, False), ("gradients of value and gate", 3, False), ("NT", 3, False), ("TN", 3, False), ("TN", 3, True),
                                                      ("NT", 2, True), ("NN", 2, True), ("TN", 2, False), ("TN", 2, True)}
    b = _lib.GatedMlpBwdParams()
    assert L.ss2d_gated_mlp_kernel(None, 0) == -1 and L.ss2d_gated_mlp_kernel(b, 0) == -1
    b.fwd, a = params()
    assert L.ss2d_gated_mlp_kernel(b, 6) == -2 and L.ss2d_gated_mlp_kernel(b, -1) == -2
    assert [L.ss2d_gated_mlp_kernel(b, i) % 16 for i in range(6)] == [1, 1, 0, 0, 0, 0]       # no upstream gradient yet
    b.dy, b.dy_row_stride = a, 16
    assert [L.ss2d_gated_mlp_kernel(b, i) % 16 for i in range(6)] == [1, 1, 4, 2, 2, 2]
    b.fwd.x = a + 2
    assert [L.ss2d_gated_mlp_kernel(b, i) % 16 for i in range(6)] == [0] * 6
