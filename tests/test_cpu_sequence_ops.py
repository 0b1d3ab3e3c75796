"""Host side of the sequence-policy operators: struct layouts, and what the C entry points and the Python wrappers refuse (nothing is launched)."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from conftest import ROOT


def test_structs_match_the_header(tmp_path):
    from xuance_amd import _lib, ops
    assert [f.size for f in (ops._LINATTN, ops._BLOCK_NORM, ops._DISTILL)] == [ctypes.sizeof(c) for c in (_lib.LinAttn, _lib.BlockNorm, _lib.Distill)]
    pairs = {"xrl_linattn_t": _lib.LinAttn, "xrl_block_norm_t": _lib.BlockNorm, "xrl_distill_t": _lib.Distill}
    src = '#include "xrl_hip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){\n'
    for cname, cls in pairs.items():
        src += f'printf("{cname} %zu\\n", sizeof({cname}));\n'
        for f, _ in cls._fields_:
            src += f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));\n'
    (tmp_path / "s.c").write_text(src + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, cls in pairs.items():
        assert int(out[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(out[f"{cname}.{f}"]) == getattr(cls, f).offset, (cname, f)


def call(name, p):
    from xuance_amd import _lib
    return getattr(_lib.load(), name)(ctypes.byref(p) if p is not None else None, None)


def filled(cls, **kw):
    """A struct with every pointer set (to nothing that is ever read) and these fields."""
    p = cls()
    for f, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(p, f, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def lin(**kw):
    from xuance_amd import _lib
    return filled(_lib.LinAttn, **{**dict(T=4, B=2, H=2, dk=8, dv=8, scale=1.0, workspace_floats=1 << 30, d_state=8192), **kw})


@pytest.mark.parametrize("entry", ["xrl_linattn_forward", "xrl_linattn_backward", "xrl_linattn_step"])
@pytest.mark.parametrize("bad", [dict(T=-1), dict(B=-1), dict(H=0), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129), dict(dtype=2), dict(q=None),
                                 dict(log_decay=None), dict(B=1 << 20, H=1 << 20)])
def test_linattn_refuses(entry, bad):
    assert call(entry, lin(**{**dict(T=1), **bad})) < 0
    from xuance_amd import _lib
    assert b"invalid argument" in _lib.load().xrl_last_error()


def test_linattn_refuses_more():
    assert call("xrl_linattn_forward", None) < 0
    assert call("xrl_linattn_step", lin(T=2)) < 0
    assert call("xrl_linattn_step", lin(T=1, state=None)) < 0
    assert call("xrl_linattn_backward", lin(d_k=None)) < 0
    from xuance_amd import ops
    need = ops.linattn_workspace_floats(30000, 1, 1, 64, 64)
    if need:
        assert call("xrl_linattn_forward", lin(T=30000, B=1, H=1, dk=64, dv=64, workspace_floats=need - 1)) < 0
        assert call("xrl_linattn_forward", lin(T=30000, B=1, H=1, dk=64, dv=64, workspace=None)) < 0
    assert call("xrl_linattn_forward", lin(B=0)) == 0                          # nothing to do, nothing launched


@pytest.mark.parametrize("bad", [dict(N=-1), dict(D=0), dict(D=8193), dict(dtype=2), dict(kind=2), dict(gate_act=5), dict(gate_act=-1), dict(eps=0.0),
                                 dict(eps=math.nan), dict(x=None), dict(u=None)])
def test_block_norm_refuses(bad):
    from xuance_amd import _lib
    ok = dict(N=4, D=16, eps=1e-5, workspace_floats=1 << 30)
    for entry in ("xrl_block_norm_forward", "xrl_block_norm_backward"):
        assert call(entry, filled(_lib.BlockNorm, **{**ok, **bad})) < 0, entry


def test_block_norm_backward_refuses_more():
    from xuance_amd import _lib, ops
    ok = dict(N=4, D=16, eps=1e-5, workspace_floats=1 << 30)
    for bad in (dict(workspace=None), dict(workspace_floats=ops.block_norm_workspace_floats(4, 16) - 1), dict(d_x=None), dict(gate=None),
                dict(d_y=None, d_n=None)):
        assert call("xrl_block_norm_backward", filled(_lib.BlockNorm, **{**ok, **bad})) < 0, bad
    assert call("xrl_block_norm_forward", filled(_lib.BlockNorm, **{**ok, "N": 0})) == 0


@pytest.mark.parametrize("bad", [dict(N=-1), dict(A=0), dict(K=0), dict(K=257), dict(dtype=2), dict(temperature=0.0), dict(temperature=-1.0),
                                 dict(temperature=math.nan), dict(logits=None), dict(teacher_idx=None), dict(teacher_logits=None), dict(loss=None)])
def test_distill_refuses(bad):
    from xuance_amd import _lib
    ok = dict(N=4, A=16, K=4, temperature=1.0, ld=16, ld_d=16)
    assert call("xrl_distill_loss", filled(_lib.Distill, **{**ok, **bad})) < 0
    assert call("xrl_distill_loss", filled(_lib.Distill, **{**ok, "N": 0})) == 0


# --------------------------------------------------------------------------------------------------- the wrappers' own checks
@pytest.fixture
def host_ops(monkeypatch):
    """The wrappers with host tensors let through: the C entry points look at them and, without a device, fail to launch; that counts as let through."""
    from xuance_amd import _lib, ops
    if torch.cuda.is_available():
        pytest.skip("host tensors would reach a kernel")
    made = []

    def call(name, *a):
        rc = getattr(_lib.load(), name)(*a)
        if rc == -2:                                                            # XRL_EHIP
            made.append(name)
        elif rc != 0:
            raise ops.XrlError(_lib.load().xrl_last_error().decode())
    monkeypatch.setattr(ops, "_raw_stream", lambda device: None)
    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(ops, "init_device", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)               # what a host tensor calls its device
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ops.made = made
    yield ops
    del ops.made


def test_wrappers_refuse_wrong_tensors(host_ops):
    ops = host_ops
    t = torch.zeros                                                             # every call its own, unless it says otherwise
    good = dict(q=t(5, 2, 3, 8), k=t(5, 2, 3, 8), v=t(5, 2, 3, 4), out=t(5, 2, 3, 4), log_decay=t(3))
    ops.linattn_forward(**good, lengths=t(2).int(), reset=t(5, 2), state=t(2, 3, 8, 4), state_out=t(2, 3, 8, 4))
    assert ops.made == ["xrl_linattn_forward"]
    for bad in (dict(q=t(5, 2, 24)), dict(k=t(5, 2, 3, 4)), dict(k=t(5, 2, 2, 8)), dict(v=t(4, 2, 3, 4)), dict(v=t(5, 2, 3, 4).bfloat16()),
                dict(q=t(5, 2, 3, 8).half(), k=t(5, 2, 3, 8).half(), v=t(5, 2, 3, 4).half(), out=t(5, 2, 3, 4).half()), dict(out=t(5, 2, 3, 8)),
                dict(out=t(1, 2, 3, 4).expand(5, -1, -1, -1)), dict(out=good["v"]), dict(out=t(5, 2, 3, 8)[..., ::2]), dict(log_decay=t(4)),
                dict(log_decay=t(3).double()), dict(lengths=t(2)), dict(lengths=t(3).int()), dict(reset=t(2, 5)), dict(reset=t(5, 2).bool()),
                dict(state=t(2, 3, 4, 8)), dict(state_out=t(2, 3, 4, 8).transpose(2, 3)), dict(q=t(5, 2, 3, 129), k=t(5, 2, 3, 129))):
        with pytest.raises(ops.XrlError):
            ops.linattn_forward(**{**good, **bad})
    s = t(2, 3, 8, 4)
    ops.linattn_backward(good["q"], good["k"], good["v"], good["out"], t(5, 2, 3, 8), t(5, 2, 3, 8), t(5, 2, 3, 4), good["log_decay"], d_state_out=s)
    with pytest.raises(ops.XrlError):                                           # the gradient in place of the gradient it is made from
        ops.linattn_backward(good["q"], good["k"], good["v"], good["out"], t(5, 2, 3, 8), t(5, 2, 3, 8), t(5, 2, 3, 4), good["log_decay"], d_state_out=s, d_state=s)
    d = t(5, 2, 3, 8)
    with pytest.raises(ops.XrlError):
        ops.linattn_backward(good["q"], good["k"], good["v"], good["out"], d, d, t(5, 2, 3, 4), good["log_decay"])
    st = dict(q=t(2, 3, 8), k=t(2, 3, 8), v=t(2, 3, 4), out=t(2, 3, 4), log_decay=t(3), state=s)
    ops.linattn_step(**st)
    for bad in (dict(q=t(1, 2, 3, 8)), dict(state=t(2, 3, 8, 5)), dict(reset=t(3)), dict(out=t(2, 3, 5)), dict(state_out=s[:1])):
        with pytest.raises(ops.XrlError):
            ops.linattn_step(**{**st, **bad})
    n = dict(x=t(6, 8), u=t(6, 8), y=t(6, 8), n=t(6, 8), gate=t(6, 8))
    ops.block_norm_forward(**n)
    ops.block_norm_forward(n["x"], n["u"], n["x"])
    for bad in (dict(kind="batch"), dict(gate_act="gelu"), dict(eps=0.0), dict(u=t(5, 8)), dict(y=n["u"]), dict(n=n["y"]), dict(w_post=t(7)),
                dict(scale=t(8).bfloat16()), dict(gate=t(6, 16)[:, ::2]), dict(x=t(6, 8).double()), dict(y=t(1, 8).expand(6, -1))):
        with pytest.raises(ops.XrlError):
            ops.block_norm_forward(**{**n, **bad})
    with pytest.raises(ops.XrlError):
        ops.block_norm_backward(t(6, 8), t(6, 8), None, None, t(6, 8), t(6, 8), workspace=t(4096))
    with pytest.raises(ops.XrlError):
        ops.block_norm_backward(t(6, 8), t(6, 8), t(6, 8), None, t(6, 8), t(6, 8), d_gate=t(6, 8), workspace=t(4096))
    c = dict(logits=t(6, 9), teacher_idx=t(6, 3).int(), teacher_logits=t(6, 3), loss=t(6))
    ops.distill_loss(**c)
    ops.distill_loss(**c, d_logits=c["logits"])
    for bad in (dict(teacher_idx=t(6, 3).long()), dict(teacher_logits=t(6, 3).bfloat16()), dict(loss=t(5)), dict(avail=t(6, 9).bool()), dict(weight=t(9)),
                dict(temperature=0.0), dict(teacher_idx=t(6, 257).int(), teacher_logits=t(6, 257)), dict(d_logits=t(1, 9).expand(6, -1)),
                dict(d_logits=t(6, 9).bfloat16()), dict(teacher_idx=t(6, 6).int()[:, ::2])):
        with pytest.raises(ops.XrlError):
            ops.distill_loss(**{**c, **bad})


def test_outputs_share_no_memory(host_ops):
    """Slices of one buffer are outputs beside each other; anything that overlaps is refused, and so are outputs whose own elements do."""
    ops = host_ops
    rows, ld = torch.zeros(5, 2, 3 * 12), torch.zeros(3)
    part = [rows[..., 12 * i:12 * i + 12].view(5, 2, 3, 4) for i in range(3)]
    far = [torch.zeros(5, 2, 3, 4) for _ in range(4)]
    back = lambda dq, dk, dv, q=far[0]: ops.linattn_backward(q, far[1], far[2], far[3], dq, dk, dv, ld)      # noqa: E731
    back(*part)
    back(torch.zeros(2, 5, 3, 4).transpose(0, 1), torch.zeros(3, 5, 2, 4).permute(1, 2, 0, 3), torch.zeros(5, 2, 3, 6)[..., 1:5])
    both = torch.zeros(10, 2, 3, 4)
    back(both[:5], both[5:], part[0])
    back(both[::2], both[1::2], part[0])
    assert ops.made == ["xrl_linattn_backward"] * 4
    wide = torch.zeros(5, 2, 3, 7)
    for bad in ((part[0], part[0], part[1]), (both[:5], both[4:9], part[0]), (wide[..., :4], wide[..., 3:], part[0]), (part[0], part[1], far[1]),
                (torch.zeros(1, 2, 3, 4).expand(5, -1, -1, -1), part[0], part[1]), (torch.zeros(400).as_strided((5, 2, 3, 4), (24, 12, 2, 1)), part[0], part[1]),
                (torch.zeros(400).as_strided((5, 2, 3, 4), (20, 12, 4, 1)), part[0], part[1])):
        with pytest.raises(ops.XrlError, match="share memory"):
            back(*bad)
    x = torch.zeros(6, 8)
    y = torch.zeros(6, 16)
    ops.block_norm_forward(x, y[:, :8], x, y[:, 8:])
    with pytest.raises(ops.XrlError, match="share memory"):
        ops.block_norm_forward(x, y[:, :8], y[:, :8])
    with pytest.raises(ops.XrlError, match="share memory"):
        ops.block_norm_forward(y[:, :8], x, y[:, 1:9])
    w = torch.zeros(8)
    with pytest.raises(ops.XrlError, match="share memory"):
        ops.block_norm_backward(x, torch.zeros(6, 8), torch.zeros(6, 8), None, torch.zeros(6, 8), torch.zeros(6, 8), d_scale=w, d_w_post=w, workspace=torch.zeros(4096))
    ws = torch.zeros(4096)
    with pytest.raises(ops.XrlError, match="share memory"):
        ops.block_norm_backward(x, torch.zeros(6, 8), torch.zeros(6, 8), None, torch.zeros(6, 8), ws[:48].view(6, 8), workspace=ws)


def test_a_captured_call_brings_its_workspace(host_ops):
    ops = host_ops
    need = ops.linattn_workspace_floats(30000, 1, 1, 4, 4)
    assert need > 0
    t = lambda: torch.zeros(30000, 1, 1, 4)                                     # noqa: E731
    a = (t(), t(), t(), t(), torch.zeros(1))
    for ws in (None, torch.zeros(need - 1), torch.zeros(need).double(), torch.zeros(2 * need)[::2], torch.zeros(need + 1)[1:]):
        with pytest.raises(ops.XrlError):
            ops.linattn_forward(*a, workspace=ws)
    ops.linattn_forward(*a, workspace=torch.zeros(need))
    assert ops.made == ["xrl_linattn_forward"]
    with pytest.raises(ops.XrlError):
        ops.block_norm_backward(torch.zeros(6, 8), torch.zeros(6, 8), torch.zeros(6, 8), None, torch.zeros(6, 8), torch.zeros(6, 8))
