"""Host side of the sequence-model operators, without a GPU: the argument
blocks have the C layout, workspace sizes, and the refusals of the C entries."""
import os
import subprocess

import pytest
import torch

from hard_resets_compose_b200 import _lib, embed, leakyattn, normgate

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_blocks_have_the_c_layout(tmp_path):
    names = {"lifb_norm_gate": (_lib.NORM_GATE, "weight_dtype"), "lifb_leaky_attn": (_lib.LEAKY_ATTN, "dtype"),
             "lifb_leaky_attn_step_args": (_lib.LEAKY_ATTN_STEP, "dtype")}
    lines = "".join(f'printf("%zu\\n", offsetof({n}, {last}) + sizeof(int));' for n, (_, last) in names.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "lifscan_b200.h"\nint main(void) {' + lines + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [s.size for s, _ in names.values()]


def attn(B=2, T=300, H=4, Hk=2, Dk=64, Dv=64, dtype=1):
    return _lib.LEAKY_ATTN.pack(256, 256, 256, 256, 0, 0, B, T, H, Hk, Dk, Dv, *(1,) * 9, 1.0, dtype)


def test_workspaces():
    L = _lib.load()
    assert L.lifb_embed_bwd_workspace_bytes(0, 10, 4) == 0
    assert L.lifb_embed_bwd_workspace_bytes(1000, 700, 256) >= 4 * 1000 * 4 + 700
    assert L.lifb_norm_gate_bwd_workspace_bytes(0, 10, 0) == 0
    assert L.lifb_norm_gate_bwd_workspace_bytes(100, 256, 0) >= 2 * 256 * 4
    assert L.lifb_leaky_attn_workspace_bytes(attn(T=0), 1) == 0
    # shared heads' gradients pass through fp32 parts of each query head
    assert L.lifb_leaky_attn_workspace_bytes(attn(), 1) >= 2 * 300 * 4 * 128 * 4


def test_c_entries_refuse_without_a_gpu():
    L = _lib.load()
    assert L.lifb_embed_fwd(256, 8, 256, 256, -1, 4, 4, 4, 1.0, 0, None) == 1 and b"negative" in L.lifb_last_error()
    assert L.lifb_embed_fwd(256, 2, 256, 256, 1, 4, 4, 4, 1.0, 0, None) == 1
    assert L.lifb_embed_fwd(256, 8, 256, 256, 1, 4, 4, 3, 1.0, 0, None) == 1
    assert L.lifb_embed_fwd(256, 8, 256, 256, 1, 4, 4, 4, 1.0, 9, None) == 1
    assert L.lifb_embed_fwd(None, 8, 256, 256, 1, 4, 4, 4, 1.0, 0, None) == 1
    assert L.lifb_embed_bwd(256, 8, 256, 256, 1 << 31, 4, 4, 4, 1.0, 0, 256, 0, None) == 4
    assert L.lifb_embed_bwd(256, 8, 256, 256, 5, 4, 4, 4, 1.0, 0, None, 0, None) == 3
    ng = lambda R=4, D=8, cols=8, act=0, dt=0, wdt=0: _lib.NORM_GATE.pack(  # noqa: E731
        256, 256, 256, 256, 256, 256, R, D, D, D, D, cols, 1.0, 1e-6, act, dt, wdt)
    assert L.lifb_norm_gate_fwd(None, 256, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(R=-1), 256, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(cols=3), 256, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(act=7), 256, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(dt=1, wdt=2), 256, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(D=8200, cols=0), 256, 256, None) == 4
    assert L.lifb_norm_gate_fwd(ng(), None, 256, None) == 1
    assert L.lifb_norm_gate_fwd(ng(R=0), None, None, None) == 0
    assert L.lifb_norm_gate_bwd(ng(), 256, 8, 256, 8, 256, 256, 256, 256, 256, None, 0, None) == 3
    for bad, status in ((attn(B=-1), 1), (attn(dtype=2), 4), (attn(H=3, Hk=2), 1), (attn(Dk=129), 4), (attn(T=1 << 31), 4)):
        assert L.lifb_leaky_attn_fwd(bad, 256, None, None, 0, None) == status
        assert L.lifb_leaky_attn_bwd(bad, 256, None, None, 256, 256, 256, None, None, 0, None) == status
    assert L.lifb_leaky_attn_fwd(attn(), None, None, None, 0, None) == 1
    step = _lib.LEAKY_ATTN_STEP.pack(256, 256, 256, 256, 0, 4, 2, 2, 8, 8, 3, *(1,) * 8, 1.0, 0)
    assert L.lifb_leaky_attn_step(step, 256, 256, None) == 1 and b"slots" in L.lifb_last_error()


def test_python_entries_refuse_cpu_tensors():
    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        leakyattn.leaky_attention(x, x, x, torch.zeros(4))
    with pytest.raises(RuntimeError, match="CUDA"):
        leakyattn.leaky_attention_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(4), torch.zeros(2, 4, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        normgate.rms_norm(x, torch.zeros(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        embed.embedding(torch.zeros(3, dtype=torch.long), x[0, 0])
