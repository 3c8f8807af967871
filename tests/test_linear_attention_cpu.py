"""Linear attention with decay: what its entry points refuse, before any launch.  No GPU needed."""
import ctypes

import pytest
import torch

from vmamba_b200 import _lib


def params(cls=_lib.LinearAttentionParams):
    buf = (ctypes.c_float * 64)()
    p = cls()
    a = (ctypes.addressof(buf) + 63) // 64 * 64
    for f in ("q", "k", "v", "log_decay", "out"):
        setattr(p, f, a)
    p.batch, p.n_groups, p.heads, p.dk, p.dv, p.dtype = 2, 2, 4, 16, 8, _lib.SS2D_BF16
    p.keep = buf
    return p, a


def test_refusals_of_the_c_interface():
    L = _lib.lib()
    before = _lib.launch_count()
    call, size = L.ss2d_linear_attention_fwd, L.ss2d_linear_attention_workspace_bytes
    assert call(None, None) == -1 and size(None) < 0
    p, a = params()
    assert call(p, None) == -2                                   # no token
    p.seqlen = 100
    assert size(p) == 0 and L.ss2d_linear_attention_states_bytes(p) == 2 * 4 * 2 * 16 * 8 * 4 and L.ss2d_linear_attention_states_bytes(None) < 0
    for field, bad, code in (("q", None, -1), ("out", None, -1), ("dtype", 5, -3), ("heads", 5, -2), ("batch", 0, -2), ("dk", 129, -6), ("dv", 200, -6),
                             ("dk", 0, -2), ("v_token_stride", -1, -5), ("k", a + 1, -4), ("log_decay", a + 2, -4), ("out", a + 2, -4),
                             ("final_state", a + 4, -4), ("seqlen", 1 << 31, -6), ("batch", 1 << 30, -6)):
        p, a = params()
        p.seqlen = 100
        setattr(p, field, bad)
        assert call(p, None) == code, field
    p, a = params()
    p.seqlen, p.batch = 4096, 1                                   # few rows, many chunks: cut into segments, in a workspace
    need = size(p)
    assert need > 0 and call(p, None) == -8
    p.workspace, p.workspace_bytes = a, need - 1
    assert call(p, None) == -8
    b = _lib.LinearAttentionBwdParams()
    assert L.ss2d_linear_attention_bwd(None, None) == -1 and L.ss2d_linear_attention_bwd(b, None) == -1
    b.fwd, _ = params()
    b.fwd.seqlen = 100
    assert L.ss2d_linear_attention_bwd(b, None) == -1             # no states
    assert L.ss2d_linear_attention_bwd_workspace_bytes(b) >= 4 * 2 * 4 * 2 * 16 * 8
    for f in ("dout", "dq", "dk", "dv", "dlog_decay"):
        setattr(b, f, a)
    b.fwd.chunk_states = a
    assert L.ss2d_linear_attention_bwd(b, None) == -8
    b.dout_head_stride = -8
    assert L.ss2d_linear_attention_bwd(b, None) == -5
    s, a = params(_lib.LinearAttentionStepParams)
    assert L.ss2d_linear_attention_step(s, None) == -1
    s.state = s.state_out = a
    assert L.ss2d_linear_attention_step(s, None) == -5            # states that overlap
    s.state_batch_stride = s.state_out_batch_stride = 4 * 16 * 8
    s.dk = 129
    assert L.ss2d_linear_attention_step(s, None) == -6
    assert _lib.launch_count() == before


def test_struct_layout(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = tmp_path / "sz.c"
    prog.write_text('#include "ss2d_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu %zu %zu\\n",'
                    'sizeof(ss2d_linear_attention_params),offsetof(ss2d_linear_attention_params,dtype),sizeof(ss2d_linear_attention_bwd_params),'
                    'offsetof(ss2d_linear_attention_bwd_params,dout_head_stride),sizeof(ss2d_linear_attention_step_params),'
                    'offsetof(ss2d_linear_attention_step_params,scale));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(prog), "-o", str(exe)])
    A, B, S = _lib.LinearAttentionParams, _lib.LinearAttentionBwdParams, _lib.LinearAttentionStepParams
    assert [int(t) for t in subprocess.check_output([str(exe)]).split()] == [
        ctypes.sizeof(A), A.dtype.offset, ctypes.sizeof(B), B.dout_head_stride.offset, ctypes.sizeof(S), S.scale.offset]


def test_cpu_tensors_are_refused():
    import vmamba_b200 as vb
    x = torch.zeros(1, 3, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.linear_attention_fn(x, x, x, torch.zeros(1, 3, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))
