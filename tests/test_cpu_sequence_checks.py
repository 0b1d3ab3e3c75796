"""More of what the host side of the sequence-policy operators refuses (nothing is launched)."""
import math
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from test_cpu_sequence_ops import call, filled, lin


@pytest.mark.parametrize("bad", [math.inf, 3e38, 1e19, 1e-19, 1e-45])
def test_distill_refuses_temperatures_without_a_square_or_reciprocal(bad):
    """At an infinite temperature every absent action (-inf times 0) made the row NaN."""
    from xuance_amd import _lib
    ok = dict(N=4, A=16, K=4, temperature=1.0, grad_scale=1.0, ld=16, ld_d=16)
    assert call("xrl_distill_loss", filled(_lib.Distill, **{**ok, "temperature": bad})) == -1
    assert b"temperature" in _lib.load().xrl_last_error()


@pytest.mark.parametrize("entry", ["xrl_linattn_forward", "xrl_linattn_backward"])
def test_linattn_refuses_more_threads_than_a_launch_takes(entry):
    """16 million rows of heads of 64: left to the launch, the call's error was the runtime's."""
    from xuance_amd import _lib
    far = {n: (1 + i) << 44 for i, n in enumerate(("out", "d_q", "d_k", "d_v", "state_out", "d_state", "d_out", "workspace"))}
    strides = {"stride_" + n: (1 << 30, 64, 64) for n in ("q", "k", "v", "out", "d_out", "d_q", "d_k", "d_v")}
    assert call(entry, lin(T=1, B=1 << 24, H=1, dk=64, dv=64, **far, **strides)) == -1
    assert b"1ll << 32" in _lib.load().xrl_last_error()


def test_ops_import_without_device_bindings():
    """A torch built for the CPU alone has no raw-stream binding: the package's modules import all the same."""
    src = ("import torch, sys\nif hasattr(torch._C, '_cuda_getCurrentRawStream'): del torch._C._cuda_getCurrentRawStream\n"
           f"sys.path.insert(0, {ROOT!r})\nimport xuance_amd.ops\n")
    r = subprocess.run([sys.executable, "-c", src], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-500:]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32])
def test_workspace_sizes_refuse_other_types(dtype):
    from xuance_amd import ops
    with pytest.raises(ops.XrlError):
        ops.linattn_workspace_floats(100, 1, 1, 8, 8, dtype=dtype)
    with pytest.raises(ops.XrlError):
        ops.block_norm_workspace_floats(100, 8, dtype=dtype)
