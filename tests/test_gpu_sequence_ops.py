"""The sequence-policy operators (linattn_*, block_norm_*, distill_loss) against plain float64 implementations: every type, odd head
sizes, layouts, lengths from 0 on, resets, decays at both ends, rows whose mask leaves nothing, workspaces, capture; and a small
sequence policy that runs them together, as a whole and step by step.

Tolerances.  An f32 sum of n terms is off by at most n u sum|terms|, u = 2^-24 (half a step), and a product of m factors by m u more; sum|terms|
is evaluated in float64 from the operands' absolute values.  A value stored as bf16 is rounded once more, by at most 2^-8 of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from xuance_amd import ops
    torch.cuda.set_device(0)
    ops.init_device()
    return ops


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, mul=1.0):
    return (torch.randn(*shape, generator=g) * mul).to(dtype)


def check(got, ref, bound, what):
    """|got - ref| <= bound, element by element (all of it in float64 on the host)."""
    got, ref = got.detach().double().cpu(), ref.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    over = ((got - ref).abs() - bound).max().item() if got.numel() else 0.0
    worst = ((got - ref).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert over <= 0, f"{what}: off by {worst:.2f} of what is allowed (max |error| {(got - ref).abs().max().item():.3e})"


# ------------------------------------------------------------------------------------------------------- linear attention
def lin_reference(q, k, v, log_decay, scale, lengths=None, reset=None, state=None):
    """The recurrence in float64, one step after another; differentiable."""
    T, B, H, dk = q.shape
    dv = v.shape[-1]
    lam = torch.exp(log_decay.double()).view(1, H, 1, 1)
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state is None else state.double()
    out = []
    for t in range(T):
        live = torch.ones(B, 1, 1, 1) if lengths is None else (t < lengths).double().view(B, 1, 1, 1)
        cut = torch.zeros(B, 1, 1, 1) if reset is None else (reset[t] != 0).double().view(B, 1, 1, 1)
        kt, vt, qt = (torch.where(live[..., 0] > 0, x[t].double(), torch.zeros((), dtype=torch.float64)) for x in (k, v, q))
        S = torch.where(live > 0, lam * S * (1 - cut) + kt[..., :, None] * vt[..., None, :], S)
        out.append(scale * (qt[..., :, None] * S).sum(-2))
    out = torch.stack(out) if T else torch.zeros(0, B, H, dv, dtype=torch.float64)
    return out, S


def lin_terms(dk, dv, T, dtype):
    """What an output is off by relative to the sum of its terms' magnitudes: a dot product over a head, a sum over 64 steps, the
    recurrence over the chunks (its product, its sum and its two-part decay each), eight single roundings (decays, scale, joins); a bf16
    product takes the decayed scores and the state in two parts each, 2^-16 apiece."""
    n = max(dk, dv) + 64 + 4 * math.ceil(max(T, 1) / 64) + 8
    return n * U32 + (2 * 2.0 ** -16 if dtype is BF16 else 0.0)


def lin_case(seed, T, B, H, dk, dv, dtype, lengths, reset, state, log_decay=None):
    g = gen(seed)
    c = dict(q=randn(g, T, B, H, dk, dtype=dtype), k=randn(g, T, B, H, dk, dtype=dtype), v=randn(g, T, B, H, dv, dtype=dtype),
             d_out=randn(g, T, B, H, dv, dtype=dtype), scale=dk ** -0.5)
    c["log_decay"] = torch.tensor(log_decay, dtype=F32) if log_decay is not None else -torch.rand(H, generator=g) * 0.5
    c["lengths"] = None
    if lengths == "ragged":
        c["lengths"] = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        c["lengths"][0] = T
        if B > 1:
            c["lengths"][-1] = min(1, T)
    c["reset"] = (torch.rand(T, B, generator=g) < 0.1).float() if reset else None
    c["state"] = randn(g, B, H, dk, dv) if state else None
    c["d_state_out"] = randn(g, B, H, dk, dv) if state else None
    return c


def lin_expected(c):
    """(out, state_out, d_q, d_k, d_v, d_state) in float64, and the same of the magnitudes."""
    res = []
    for mag in (False, True):
        f = (lambda x: x.double().abs()) if mag else (lambda x: x.double())
        leaves = {n: f(c[n]).requires_grad_() for n in ("q", "k", "v")}
        if c["state"] is not None:
            leaves["state"] = f(c["state"]).requires_grad_()
        o, S = lin_reference(leaves["q"], leaves["k"], leaves["v"], c["log_decay"], c["scale"], c["lengths"], c["reset"], leaves.get("state"))
        inside = torch.ones(o.shape[:2]) if c["lengths"] is None else (torch.arange(o.shape[0])[:, None] < c["lengths"][None]).double()
        loss = (o * f(c["d_out"]) * inside[..., None, None]).sum()
        if c["state"] is not None:
            loss = loss + (S * f(c["d_state_out"])).sum()
        if loss.requires_grad:
            loss.backward()
        zero = lambda n: leaves[n].grad if leaves[n].grad is not None else torch.zeros_like(leaves[n])   # noqa: E731
        r = dict(out=o.detach(), state_out=S.detach(), d_q=zero("q"), d_k=zero("k"), d_v=zero("v"))
        if "state" in leaves:
            r["d_state"] = zero("state")
        res.append(r)
    return res


def lin_run(ops, c, backward=True, layout=None, garbage=0.0):
    """Both passes on the device: dict of outputs.  Outputs are pre-filled (they have to be written whole)."""
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    if layout:
        for n in ("q", "k", "v", "d_out"):
            dev[n] = layout(dev[n])
    T, B, H, dk = c["q"].shape
    dv = c["v"].shape[-1]
    dt = c["q"].dtype
    make = layout or (lambda t: t)
    new = lambda d: make(torch.full((T, B, H, d), 7.5, device="cuda", dtype=dt))   # noqa: E731
    par = dict(scale=c["scale"], lengths=dev["lengths"], reset=dev["reset"], state=dev["state"])
    r = dict(out=new(dv), state_out=torch.full((B, H, dk, dv), 7.5, device="cuda"))
    ops.linattn_forward(dev["q"], dev["k"], dev["v"], r["out"], dev["log_decay"], state_out=r["state_out"], **par)
    if backward:
        r.update(d_q=new(dk), d_k=new(dk), d_v=new(dv))
        if c["state"] is not None:
            r["d_state"] = torch.full((B, H, dk, dv), 7.5, device="cuda")
        ops.linattn_backward(dev["q"], dev["k"], dev["v"], dev["d_out"], r["d_q"], r["d_k"], r["d_v"], dev["log_decay"],
                             d_state_out=dev["d_state_out"], d_state=r.get("d_state"), **par)
    torch.cuda.synchronize()
    return r


def lin_check(c, got):
    ref, mag = lin_expected(c)
    T, dk, dv, dt = c["q"].shape[0], c["q"].shape[-1], c["v"].shape[-1], c["q"].dtype
    for n in got:
        stored = U16 * ref[n].abs() if dt is BF16 and n not in ("state_out", "d_state") else 0.0
        rel = lin_terms(dk, dv, T, F32 if n in ("state_out", "d_state") else dt)
        check(got[n], ref[n], rel * mag[n] * (1 + U16) + stored + 1e-37, n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [0, 1, 2, 17, 63, 64, 65, 129, 300])
def test_linattn_lengths(ops, T, dtype):
    c = lin_case(T, T, 3, 2, 16, 32, dtype, "ragged" if T else None, True, True)
    lin_check(c, lin_run(ops, c))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 7), (8, 8), (16, 24), (32, 32), (33, 64), (64, 33), (64, 64), (100, 36), (128, 16), (16, 128),
                                   (64, 128), (128, 64), (127, 121), (128, 128)])
def test_linattn_head_sizes(ops, dk, dv, dtype):
    c = lin_case(dk * 131 + dv, 150, 2, 2, dk, dv, dtype, "ragged", True, True)
    lin_check(c, lin_run(ops, c))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths,reset,state", [(None, False, False), (None, False, True), (None, True, False), ("ragged", False, False),
                                                 ("ragged", False, True)])
def test_linattn_options(ops, lengths, reset, state, dtype):
    c = lin_case(5, 200, 4, 3, 32, 32, dtype, lengths, reset, state)
    lin_check(c, lin_run(ops, c))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,B,H,dk,dv", [(2500, 1, 2, 16, 16), (1999, 2, 1, 64, 64), (1100, 1, 1, 128, 128), (1700, 3, 1, 40, 72)])
def test_linattn_long_axis_split_over_workgroups(ops, T, B, H, dk, dv, dtype):
    """Few rows and many steps: the time axis is cut into segments that run side by side."""
    assert ops.linattn_workspace_floats(T, B, H, dk, dv, dtype=dtype) >= 0
    c = lin_case(T, T, B, H, dk, dv, dtype, "ragged" if B > 1 else None, False, True, log_decay=[-0.002, -0.1][:H])
    c["reset"] = torch.zeros(T, B)
    c["reset"][T // 3, -1] = 1
    lin_check(c, lin_run(ops, c))


@pytest.mark.parametrize("lengths", [[600, 600, 600, 600], [0, 0, 0, 0], [1, 900, 64, 640], [-5, 0, 580, 4000], "65 rows"])
def test_linattn_rows_of_many_orders(ops, lengths):
    """Rows are taken up by their lengths: equal ones, none, ascending, out of range (cut to 0 and T), more rows than a wave has lanes."""
    B = 65 if lengths == "65 rows" else len(lengths)
    T = 70 if B == 65 else 640
    c = lin_case(B, T, B, 2, 16, 16, F32, "ragged", B < 65, True)
    c["lengths"] = torch.randint(0, T + 1, (B,), generator=gen(3), dtype=torch.int32) if B == 65 else torch.tensor(lengths, dtype=torch.int32)
    got = lin_run(ops, c)
    c["lengths"] = c["lengths"].clamp(0, T)
    lin_check(c, got)


def test_linattn_two_calls_at_once(ops):
    """Two streams, each with a workspace of its own."""
    cases = [lin_case(50 + i, 1300, 1, 2, 64, 64, F32, None, True, True) for i in range(2)]
    plain = [lin_run(ops, c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    dev = [{n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()} for c in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for d, s in zip(dev, streams):
            with torch.cuda.stream(s):
                out = torch.empty_like(d["v"])
                ops.linattn_forward(d["q"], d["k"], d["v"], out, d["log_decay"], scale=d["scale"], reset=d["reset"], state=d["state"])
                outs.append(out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, plain[i % 2]["out"])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_linattn_decays_at_both_ends(ops, dtype):
    """No decay, no memory at all, and decays whose powers leave the range of f32 within one chunk; a positive one is taken as 0."""
    c = lin_case(9, 140, 2, 6, 16, 16, dtype, "ragged", False, True, log_decay=[0.0, -math.inf, -1e-6, -3.0, -80.0, 0.0])
    got = lin_run(ops, c)
    lin_check(c, got)
    c["log_decay"][5] = 0.5
    again = lin_run(ops, c)
    for n in got:
        assert torch.equal(got[n], again[n]), n


@pytest.mark.parametrize("where", ["first", "last", "all", "chunk edges", "before the start of a row's padding"])
def test_linattn_resets(ops, where):
    c = lin_case(11, 193, 3, 2, 16, 16, F32, "ragged", False, True)
    r = torch.zeros(193, 3)
    if where == "first":
        r[0] = 1
    elif where == "last":
        r[192] = 1
        for b in range(3):
            if c["lengths"][b] > 0:
                r[c["lengths"][b] - 1, b] = 1
    elif where == "all":
        r[:] = 1
    elif where == "chunk edges":
        r[63, 0] = r[64, 1] = r[65, 2] = r[128, 0] = r[127, 1] = 1
    else:
        for b in range(3):
            if c["lengths"][b] < 193:
                r[c["lengths"][b], b] = 1                       # behind the row's last step: takes no part
    c["reset"] = r
    lin_check(c, lin_run(ops, c))


def test_linattn_padding_is_not_read(ops):
    c = lin_case(13, 100, 4, 2, 32, 16, F32, "ragged", True, True)
    clean = lin_run(ops, c)
    behind = torch.arange(100)[:, None] >= c["lengths"][None]
    for n in ("q", "k", "v", "d_out"):
        c[n][behind] = math.nan
    c["reset"][behind] = math.nan
    got = lin_run(ops, c)
    for n in got:
        assert torch.equal(got[n], clean[n]), n
    for n in ("out", "d_q", "d_k", "d_v"):
        assert (got[n].cpu()[behind] == 0).all(), n


def batch_major(t):
    return t.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)


def in_wider_rows(t):
    wide = torch.full((*t.shape[:3], t.shape[3] + 3), 3.0, device=t.device, dtype=t.dtype)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", [batch_major, in_wider_rows])
@pytest.mark.parametrize("dk,dv", [(16, 64), (24, 40)])
def test_linattn_layouts(ops, layout, dk, dv, dtype):
    c = lin_case(17, 90, 3, 2, dk, dv, dtype, "ragged", True, True)
    got, plain = lin_run(ops, c, layout=layout), lin_run(ops, c)
    for n in got:
        assert torch.equal(got[n].contiguous(), plain[n].contiguous()), n


def test_linattn_slices_of_one_projection_and_outputs_beside_each_other(ops):
    T, B, H, d = 70, 3, 2, 32
    c = lin_case(19, T, B, H, d, d, F32, None, False, False)
    plain = lin_run(ops, c)
    rows = torch.cat([c[n].reshape(T, B, H * d) for n in "qkv"], -1).cuda()
    grads = torch.full_like(rows, 7.5)
    part = lambda t, i: t[..., i * H * d:(i + 1) * H * d].view(T, B, H, d)         # noqa: E731
    out = torch.empty(T, B, H, d, device="cuda")
    ops.linattn_forward(part(rows, 0), part(rows, 1), part(rows, 2), out, c["log_decay"].cuda(), scale=c["scale"])
    ops.linattn_backward(part(rows, 0), part(rows, 1), part(rows, 2), c["d_out"].cuda(), part(grads, 0), part(grads, 1), part(grads, 2),
                         c["log_decay"].cuda(), scale=c["scale"])
    assert torch.equal(out, plain["out"])
    for i, n in enumerate(("d_q", "d_k", "d_v")):
        assert torch.equal(part(grads, i), plain[n]), n


def test_linattn_shared_heads(ops):
    """One key / value head for all query heads, by stride 0; the caller sums the gradients of the heads."""
    c = lin_case(23, 75, 2, 4, 16, 16, F32, None, False, False)
    for n in ("k", "v"):
        c[n] = c[n][:, :, :1].expand(-1, -1, 4, -1)
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    k, v = (c[n][:, :, :1].cuda().expand(-1, -1, 4, -1) for n in ("k", "v"))
    assert k.stride(2) == 0
    r = {n: torch.empty(75, 2, 4, 16, device="cuda") for n in ("out", "d_q", "d_k", "d_v")}
    ops.linattn_forward(dev["q"], k, v, r["out"], dev["log_decay"], scale=c["scale"])
    ops.linattn_backward(dev["q"], k, v, dev["d_out"], r["d_q"], r["d_k"], r["d_v"], dev["log_decay"], scale=c["scale"])
    lin_check(c, r)


def test_linattn_gradients_against_differences(ops):
    """Directional derivatives of the float64 recurrence by central differences, against the kernel's gradients: the third-order term of the
    difference is O(h^2) (the loss is a polynomial), its rounding 2^-53 |loss| / h; both far below the f32 bound used."""
    c = lin_case(29, 80, 2, 2, 8, 8, F32, "ragged", True, True)
    got = lin_run(ops, c)
    g = gen(1)
    inside = (torch.arange(80)[:, None] < c["lengths"][None]).double()[..., None, None]

    def loss(x):
        o, S = lin_reference(x["q"], x["k"], x["v"], c["log_decay"], c["scale"], c["lengths"], c["reset"], x["state"])
        return ((o * c["d_out"].double() * inside).sum() + (S * c["d_state_out"].double()).sum()).item()
    base = {n: c[n].double() for n in ("q", "k", "v", "state")}
    _, mag = lin_expected(c)
    for n in base:
        way, h = torch.randn(base[n].shape, generator=g, dtype=torch.float64), 1e-4
        diff = (loss({**base, n: base[n] + h * way}) - loss({**base, n: base[n] - h * way})) / (2 * h)
        have = (got["d_" + n].double().cpu() * way).sum().item()
        allowed = lin_terms(8, 8, 80, F32) * (mag["d_" + n] * way.abs()).sum().item() + 1e-5
        assert abs(diff - have) <= allowed, (n, diff, have)


def test_linattn_state_in_place_and_pieces_equal_the_whole(ops):
    """A sequence in three pieces with the state carried in place, and step by step."""
    c = lin_case(31, 150, 2, 2, 32, 16, F32, None, True, True)
    ref, mag = lin_expected(c)
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    for pieces in ([(0, 70), (70, 71), (71, 150)], [(t, t + 1) for t in range(150)]):
        S, out = dev["state"].clone(), torch.empty(150, 2, 2, 16, device="cuda")
        for lo, hi in pieces:
            if len(pieces) == 150:
                ops.linattn_step(dev["q"][lo], dev["k"][lo], dev["v"][lo], out[lo], dev["log_decay"], S, scale=c["scale"], reset=dev["reset"][lo])
            else:
                ops.linattn_forward(dev["q"][lo:hi], dev["k"][lo:hi], dev["v"][lo:hi], out[lo:hi], dev["log_decay"], scale=c["scale"],
                                    reset=dev["reset"][lo:hi], state=S, state_out=S)
        rel = (lin_terms(32, 16, 150, F32) + 3 * 150 * U32)                 # every piece or step rounds the state and its decay once more
        check(out, ref["out"], rel * mag["out"], "out")
        check(S, ref["state_out"], rel * mag["state_out"], "state")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (3, 2, 5, 7), (16, 4, 16, 16), (5, 3, 64, 64), (7, 1, 128, 128), (2, 2, 100, 36), (4, 1, 16, 126),
                                       (300, 2, 32, 8)])
def test_linattn_step(ops, B, H, dk, dv, dtype):
    g = gen(B * 7 + dk)
    q, k, v = randn(g, B, H, dk, dtype=dtype), randn(g, B, H, dk, dtype=dtype), randn(g, B, H, dv, dtype=dtype)
    S, ld = randn(g, B, H, dk, dv), -torch.rand(H, generator=g)
    reset = (torch.rand(B, generator=g) < 0.4).float()
    S[reset != 0] = math.nan                                                # a row that starts afresh does not read its old state
    clean = torch.where(reset.view(B, 1, 1, 1) != 0, torch.zeros(()), S)
    want, S1 = lin_reference(q[None], k[None], v[None], ld, 0.3, None, reset[None], clean)
    mo, mS = lin_reference(q[None].abs(), k[None].abs(), v[None].abs(), ld, 0.3, None, reset[None], clean.abs())
    out, S2 = torch.empty(B, H, dv, device="cuda", dtype=dtype), torch.empty(B, H, dk, dv, device="cuda")
    ops.linattn_step(q.cuda(), k.cuda(), v.cuda(), out, ld.cuda(), S.cuda(), state_out=S2, scale=0.3, reset=reset.cuda())
    stored = U16 * want[0].abs() if dtype is BF16 else 0.0
    check(out, want[0], (dk + 8) * U32 * mo[0] * (1 + U16) + stored + 1e-37, "out")
    check(S2, S1, 4 * U32 * mS + 1e-37, "state")


def test_linattn_same_bits_every_time(ops):
    c = lin_case(37, 700, 2, 2, 64, 64, BF16, "ragged", True, True)
    a, b = lin_run(ops, c), lin_run(ops, c)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_linattn_captured_and_replayed(ops):
    """Two graphs, a workspace each, replayed in turn between eager work; every replay against the eager result."""
    from xuance_amd.ops import Graph
    sets = []
    for seed in (1, 2):
        c = lin_case(seed, 1300, 1, 2, 32, 32, F32, None, True, True)
        dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
        eager = lin_run(ops, c)
        r = {n: torch.zeros_like(t) for n, t in eager.items()}
        need = max(ops.linattn_workspace_floats(1300, 1, 2, 32, 32), ops.linattn_workspace_floats(1300, 1, 2, 32, 32, backward=True))
        ws = torch.empty(max(need, 4), device="cuda")
        par = dict(scale=c["scale"], lengths=dev["lengths"], reset=dev["reset"], state=dev["state"], workspace=ws)
        graph = Graph()
        with graph:
            ops.linattn_forward(dev["q"], dev["k"], dev["v"], r["out"], dev["log_decay"], state_out=r["state_out"], **par)
            ops.linattn_backward(dev["q"], dev["k"], dev["v"], dev["d_out"], r["d_q"], r["d_k"], r["d_v"], dev["log_decay"],
                                 d_state_out=dev["d_state_out"], d_state=r["d_state"], **par)
        sets.append((graph, r, eager, dev, ws))
    for _ in range(3):
        for graph, r, eager, _, ws in sets:
            for t in r.values():
                t.fill_(7.5)
            ws.fill_(math.nan)
            graph.launch()
            torch.cuda.synchronize()
            for n in r:
                assert torch.equal(r[n], eager[n]), n


def test_linattn_on_another_stream(ops):
    c = lin_case(41, 1200, 1, 1, 32, 32, F32, None, False, True)
    plain = lin_run(ops, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lin_run(ops, c)
    side.synchronize()
    for n in got:
        assert torch.equal(got[n], plain[n]), n


# ------------------------------------------------------------------------------------------------------- block norm
ACTS = {"none": lambda z: z, "relu": torch.relu, "leaky_relu": lambda z: torch.nn.functional.leaky_relu(z, 0.01), "tanh": torch.tanh,
        "sigmoid": torch.sigmoid}


def norm_reference(t, kind, eps, gate_act):
    """y, n in float64 from a dict of float64 tensors (missing: None)."""
    def norm(a, w, b):
        if kind == "layer":
            a = a - a.mean(1, keepdim=True)
        a = a / torch.sqrt((a * a).mean(1, keepdim=True) + eps)
        a = a if w is None else a * w
        return a if b is None else a + b
    p = norm(t["u"], t["w_post"], t["b_post"])
    if t["gate"] is not None:
        p = ACTS[gate_act](t["gate"]) * p
    if t["scale"] is not None:
        p = t["scale"] * p
    y = t["x"] + p
    return y, norm(y, t["w_pre"], t["b_pre"])


ROWS, VECS = ("x", "u", "gate"), ("scale", "w_post", "b_post", "w_pre", "b_pre")


def norm_case(seed, N, D, dtype, gate=True, vectors=VECS):
    g = gen(seed)
    c = {n: randn(g, N, D, dtype=dtype) for n in ("x", "u", "gate", "d_y", "d_n")}
    c["u"] = (c["u"].float() * 2 + 0.5).to(dtype)
    if not gate:
        c["gate"] = None
    for n in VECS:
        c[n] = randn(g, D, mul=0.3) + (1.0 if n in ("scale", "w_post", "w_pre") else 0.0) if n in vectors else None
    return c


def norm_expected(c, kind, eps, gate_act, use=("d_y", "d_n")):
    t = {n: c[n].double().requires_grad_() if c[n] is not None else None for n in ROWS + VECS}
    y, n = norm_reference(t, kind, eps, gate_act)
    loss = sum((o * c[d].double()).sum() for o, d in ((y, "d_y"), (n, "d_n")) if d in use)
    loss.backward()
    r = {"y": y.detach(), "n": n.detach()}
    for k, v in t.items():
        if v is not None:
            r["d_" + k] = v.grad if v.grad is not None else torch.zeros_like(v)
    return r


def norm_bounds(c, ref, kind, eps, gate_act, use=("d_y", "d_n")):
    """Per-element bounds.  One row is a handful of f32 operations per element on statistics that are sums of D squares: each statistic
    is off by (D + 8) u of itself at the very most, so an element of magnitude M by c u M with c = 4 (D + 8) over the chain of two norms and
    their gradients; M is the largest magnitude that enters the element's row.  The column sums add N u of their terms' magnitudes, which the
    f32 errors of the terms are relative to."""
    N, D = c["x"].shape
    rel = 4 * (D + 8) * U32
    t = {k: (c[k].double() if c[k] is not None else None) for k in ROWS + VECS}
    one = torch.ones(D, dtype=torch.float64)
    vec = lambda n, miss: t[n] if t[n] is not None else miss * one                  # noqa: E731
    a = ACTS[gate_act](t["gate"]).abs() if t["gate"] is not None else torch.ones(N, D, dtype=torch.float64)
    top = lambda m: m.abs().max(1, keepdim=True).values if m.numel() else m         # noqa: E731

    def hat(z):
        z = z - z.mean(1, keepdim=True) if kind == "layer" else z
        r = 1 / torch.sqrt((z * z).mean(1, keepdim=True) + eps)
        return z * r, r
    uh, ru = hat(t["u"])
    # the centred value is off by u of the value before centring
    uh_m = uh.abs() + ru * top(t["u"])
    p_m = uh_m * vec("w_post", 1.0).abs() + vec("b_post", 0.0).abs()
    y_m = t["x"].abs() + vec("scale", 1.0).abs() * a * p_m
    yh, ry = hat(ref["y"])
    yh_m = yh.abs() + ry * top(y_m)
    n_m = yh_m * vec("w_pre", 1.0).abs() + vec("b_pre", 0.0).abs()
    b = {"y": y_m, "n": n_m + ry * top(y_m) * vec("w_pre", 1.0).abs()}
    dn = c["d_n"].double().abs() if "d_n" in use else torch.zeros(N, D, dtype=torch.float64)
    dy = c["d_y"].double().abs() if "d_y" in use else torch.zeros(N, D, dtype=torch.float64)
    e = dn * vec("w_pre", 1.0).abs()
    dx_m = dy + ry * (e + yh_m * (e * yh_m).mean(1, keepdim=True) + e.mean(1, keepdim=True)) * (1 + top(yh_m))
    dp = dx_m * vec("scale", 1.0).abs() * a
    f = dp * vec("w_post", 1.0).abs()
    b["d_x"] = dx_m
    b["d_u"] = ru * (f + uh_m * (f * uh_m).mean(1, keepdim=True) + f.mean(1, keepdim=True)) * (1 + top(uh_m))
    b["d_gate"] = dx_m * vec("scale", 1.0).abs() * p_m
    sums = {"d_scale": dx_m * a * p_m, "d_w_post": dp * uh_m, "d_b_post": dp, "d_w_pre": dn * yh_m, "d_b_pre": dn}
    out = {k: rel * v for k, v in b.items()}
    out.update({k: (rel + (N + 8) * U32) * v.sum(0) for k, v in sums.items()})
    return {k: v + 1e-37 for k, v in out.items()}


def norm_run(ops, c, kind, eps, gate_act, use=("d_y", "d_n"), layout=lambda t: t):
    dev = {n: (t.cuda() if t is not None else None) for n, t in c.items()}
    for n in ("x", "u", "gate", "d_y", "d_n"):
        dev[n] = layout(dev[n]) if dev[n] is not None else None
    N, D = c["x"].shape
    new = lambda: layout(torch.full((N, D), 7.5, device="cuda", dtype=c["x"].dtype))   # noqa: E731
    par = dict(gate=dev["gate"], gate_act=gate_act, kind=kind, eps=eps, **{n: dev[n] for n in VECS})
    r = {"y": new(), "n": new(), "d_x": new(), "d_u": new()}
    ops.block_norm_forward(dev["x"], dev["u"], r["y"], r["n"], **par)
    if c["gate"] is not None:
        r["d_gate"] = new()
    for n in VECS:
        if c[n] is not None:
            r["d_" + n] = torch.full((D,), 7.5, device="cuda")
    ops.block_norm_backward(dev["x"], dev["u"], dev["d_y"] if "d_y" in use else None, dev["d_n"] if "d_n" in use else None,
                            **{k: v for k, v in r.items() if k.startswith("d_")}, **par)
    torch.cuda.synchronize()
    return r


def norm_check(ops, c, kind="rms", eps=1e-5, gate_act="sigmoid", use=("d_y", "d_n"), **kw):
    got = norm_run(ops, c, kind, eps, gate_act, use, **kw)
    ref = norm_expected(c, kind, eps, gate_act, use)
    bound = norm_bounds(c, ref, kind, eps, gate_act, use)
    for n in got:
        stored = U16 * ref[n].abs() * (1 + U16) if got[n].dtype is BF16 else 0.0
        check(got[n], ref[n], bound[n] + stored, n)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("N,D", [(1, 1), (1, 8), (7, 3), (33, 20), (64, 64), (130, 65), (50, 128), (37, 200), (40, 256), (21, 511), (19, 512), (9, 1000),
                                 (5, 1024), (17, 2048), (3, 4095), (6, 4096), (2, 8192), (2, 8191)])
def test_block_norm_sizes(ops, N, D, kind, dtype):
    norm_check(ops, norm_case(N + D, N, D, dtype), kind)


@pytest.mark.parametrize("gate_act", sorted(ACTS))
def test_block_norm_gate_activations(ops, gate_act):
    norm_check(ops, norm_case(3, 40, 96, F32), gate_act=gate_act)


@pytest.mark.parametrize("vectors", [(), ("scale",), ("w_post", "w_pre"), ("b_post", "b_pre", "w_pre")])
@pytest.mark.parametrize("gate", [True, False])
def test_block_norm_missing_parameters(ops, vectors, gate):
    norm_check(ops, norm_case(4, 30, 72, F32, gate=gate, vectors=vectors), "layer")


@pytest.mark.parametrize("use", [("d_y",), ("d_n",)])
def test_block_norm_one_gradient_only(ops, use):
    norm_check(ops, norm_case(5, 30, 72, F32), use=use)


def test_block_norm_many_rows(ops):
    """More rows than workgroups hold at a time, and not a multiple of them."""
    norm_check(ops, norm_case(6, 20011, 64, F32))
    norm_check(ops, norm_case(7, 5003, 520, BF16), "layer")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N,D", [(1700, 2048), (1801, 1999), (600, 8192), (2100, 512)])
def test_block_norm_more_wide_rows_than_workgroups(ops, N, D, dtype):
    norm_check(ops, norm_case(N, N, D, dtype), "layer")


def odd_rows(t):
    wide = torch.full((t.shape[0], t.shape[1] + 5), 3.0, device=t.device, dtype=t.dtype)
    wide[:, 1:-4] = t
    return wide[:, 1:-4]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_block_norm_strided_rows(ops, dtype):
    norm_check(ops, norm_case(8, 33, 64, dtype), layout=odd_rows)


def test_block_norm_in_place_and_no_next_norm(ops):
    c = norm_case(9, 20, 64, F32)
    want = norm_run(ops, c, "rms", 1e-5, "sigmoid")
    dev = {n: t.cuda() for n, t in c.items()}
    par = dict(gate=dev["gate"], **{n: dev[n] for n in VECS})
    x = dev["x"].clone()
    ops.block_norm_forward(x, dev["u"], x, None, **par)
    assert torch.equal(x, want["y"])
    d, du = dev["d_y"].clone(), torch.empty_like(x)
    ops.block_norm_backward(dev["x"], dev["u"], d, dev["d_n"], d, du, **par)
    assert torch.equal(d, want["d_x"]) and torch.equal(du, want["d_u"])


def test_block_norm_without_rows_and_rows_of_zeros(ops):
    c = norm_case(10, 0, 64, F32)
    dev = {n: t.cuda() for n, t in c.items()}
    par = dict(gate=dev["gate"], **{n: dev[n] for n in VECS})
    ops.block_norm_forward(dev["x"], dev["u"], torch.empty(0, 64, device="cuda"), None, **par)
    dw = torch.full((64,), 7.5, device="cuda")
    ops.block_norm_backward(dev["x"], dev["u"], dev["d_y"], dev["d_n"], torch.empty(0, 64, device="cuda"), torch.empty(0, 64, device="cuda"), d_w_post=dw, **par)
    assert (dw == 0).all()
    c = norm_case(11, 9, 64, F32)
    c["u"][3], c["x"][5] = 0.0, 0.0
    norm_check(ops, c, "layer")


def test_block_norm_a_row_of_infinities_stays_its_own(ops):
    c = norm_case(12, 20, 64, F32)
    clean = norm_run(ops, c, "rms", 1e-5, "sigmoid")
    c["u"][7, 3] = math.inf
    c["x"][9, 0] = math.nan
    got = norm_run(ops, c, "rms", 1e-5, "sigmoid")
    rest = [i for i in range(20) if i not in (7, 9)]
    for n in ("y", "n", "d_x", "d_u", "d_gate"):
        assert torch.equal(got[n][rest], clean[n][rest]), n


def test_block_norm_captured_and_replayed(ops):
    from xuance_amd.ops import Graph
    c = norm_case(13, 300, 128, F32)
    want = norm_run(ops, c, "rms", 1e-5, "sigmoid")
    dev = {n: t.cuda() for n, t in c.items()}
    r = {n: torch.zeros_like(t) for n, t in want.items()}
    ws = torch.empty(ops.block_norm_workspace_floats(300, 128), device="cuda")
    par = dict(gate=dev["gate"], **{n: dev[n] for n in VECS})
    graph = Graph()
    with graph:
        ops.block_norm_forward(dev["x"], dev["u"], r["y"], r["n"], **par)
        ops.block_norm_backward(dev["x"], dev["u"], dev["d_y"], dev["d_n"], workspace=ws, **{k: v for k, v in r.items() if k.startswith("d_")}, **par)
    for _ in range(3):
        for t in r.values():
            t.fill_(7.5)
        ws.fill_(math.nan)
        graph.launch()
        torch.cuda.synchronize()
        for n in r:
            assert torch.equal(r[n], want[n]), n


# ------------------------------------------------------------------------------------------------------- distillation
def distill_reference(c, tau, grad_scale):
    """Row by row in float64: (loss, d_logits, magnitude of the loss's terms)."""
    N, A = c["logits"].shape
    loss, grad, mag = torch.zeros(N, dtype=torch.float64), torch.zeros(N, A, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    for n in range(N):
        w = 1.0 if c["weight"] is None else c["weight"][n].item()
        open_ = torch.ones(A, dtype=torch.bool) if c["avail"] is None else c["avail"][n] != 0
        s = c["logits"][n].double()
        ent = [(i, t) for i, t in zip(c["teacher_idx"][n].tolist(), c["teacher_logits"][n].double().tolist())
               if 0 <= i < A and open_[i] and t != -math.inf]
        if w == 0 or not ent or not (s[open_] > -math.inf).any():
            continue
        at = torch.tensor([i for i, _ in ent])
        lq = torch.log_softmax(torch.tensor([t for _, t in ent], dtype=torch.float64) / tau, 0)
        s = torch.where(open_, s, torch.full((), -math.inf, dtype=torch.float64))
        z = (s - s.max()) / tau                  # from the maximum: next to logits of -3.4e38 the log of the sum rounds away, in 64 bits too
        lp = z - torch.logsumexp(z, 0)
        q = lq.exp()
        loss[n] = w * tau * tau * (q * (lq - lp[at])).sum()
        mag[n] = w * tau * tau * (q * (lq.abs() + (z[at] - z.max()).abs() + (z.max() - torch.logsumexp(z, 0)).abs() + 1)).sum()
        p = torch.where(open_, lp.exp(), torch.zeros((), dtype=torch.float64))
        grad[n] = grad_scale * w * tau * p.index_add(0, at, -q)
    return loss, grad, mag


def distill_case(seed, N, A, K, dtype=F32, avail=False, weight=True):
    g = gen(seed)
    c = dict(logits=randn(g, N, A, dtype=dtype, mul=3.0), teacher_logits=randn(g, N, K, dtype=dtype, mul=3.0),
             weight=torch.rand(N, generator=g) if weight else None, avail=None)
    c["teacher_idx"] = torch.stack([torch.randperm(A, generator=g)[:K] if K <= A else torch.randint(0, A, (K,), generator=g) for _ in range(N)]).int()
    if avail:
        c["avail"] = (torch.rand(N, A, generator=g) < 0.6).float()
        c["avail"][:, A // 2] = 1.0
    return c


def distill_run(ops, c, tau, grad_scale, d_logits=True, layout=lambda t: t):
    dev = {n: (t.cuda() if t is not None else None) for n, t in c.items()}
    dev["logits"] = layout(dev["logits"])
    loss = torch.full((c["logits"].shape[0],), 7.5, device="cuda")
    d = layout(torch.full(c["logits"].shape, 7.5, device="cuda", dtype=c["logits"].dtype)) if d_logits else None
    ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], loss, d_logits=d, avail=dev["avail"], weight=dev["weight"],
                     temperature=tau, grad_scale=grad_scale)
    torch.cuda.synchronize()
    return loss, d


def distill_check(ops, c, tau=2.0, grad_scale=0.5, **kw):
    """An exponential is off by the rounding of its argument (|argument| u, and exp(-x) x <= 1 / e) and its own 2 u; a sum of A of them by A u at the very
    most.  The loss adds K terms; p and q are off by the same of themselves."""
    loss, d = distill_run(ops, c, tau, grad_scale, **kw)
    want, grad, mag = distill_reference(c, tau, grad_scale)
    N, A = c["logits"].shape
    K = c["teacher_idx"].shape[1]
    rel = (A + K + 16) * U32
    check(loss, want, rel * mag + 1e-37, "loss")
    w = torch.ones(N, dtype=torch.float64) if c["weight"] is None else c["weight"].double()
    p_q = (grad_scale * w * tau)[:, None].abs() * torch.ones(N, A, dtype=torch.float64)
    stored = U16 * grad.abs() * (1 + U16) if d.dtype is BF16 else 0.0
    # of the row's largest probability or teacher weight, 1 at most: an absolute bound
    check(d, grad, rel * p_q + stored + 1e-37, "d_logits")
    return loss, d


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("avail", [False, True], ids=["open", "masked"])
@pytest.mark.parametrize("N,A,K", [(1, 1, 1), (5, 2, 1), (33, 3, 5), (64, 18, 6), (7, 63, 64), (9, 64, 8), (10, 65, 3), (130, 128, 16), (5, 500, 32), (4, 513, 64),
                                   (3, 1000, 256), (3, 4099, 32), (2, 8192, 17), (2, 20001, 64), (1, 50257, 64), (1, 70000, 3)])
def test_distill_sizes(ops, N, A, K, avail, dtype):
    distill_check(ops, distill_case(N + A, N, A, K, dtype, avail))


@pytest.mark.parametrize("tau", [0.25, 1.0, 5.0])
def test_distill_temperatures(ops, tau):
    distill_check(ops, distill_case(1, 20, 40, 10, weight=False), tau=tau)


@pytest.mark.parametrize("A", [30, 3000])
def test_distill_rows_with_nothing(ops, A):
    """No available action, no valid teacher entry, weight 0 over NaN logits, logits of -inf: loss 0 and gradient 0."""
    c = distill_case(2, 8, A, 5, avail=True)
    c["weight"][:] = 1.0
    c["avail"][0] = 0.0
    c["teacher_idx"][1] = -1
    c["teacher_idx"][2] = A
    c["teacher_logits"][3] = -math.inf
    c["avail"][4].scatter_(0, c["teacher_idx"][4].long(), 0.0)
    c["weight"][5] = 0.0
    c["logits"][5] = math.nan
    c["logits"][6] = -math.inf
    loss, d = distill_check(ops, c)
    assert (loss[:7] == 0).all() and (d[:7] == 0).all() and loss[7] != 0


@pytest.mark.parametrize("A", [30, 3000])
def test_distill_masked_logits_are_not_used(ops, A):
    c = distill_case(3, 6, A, 5, avail=True)
    want = distill_run(ops, c, 2.0, 0.5)
    shut = c["avail"] == 0
    for bad in (math.nan, math.inf, torch.finfo(F32).max):
        c["logits"][shut] = bad
        got = distill_run(ops, c, 2.0, 0.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert (got[1].cpu()[shut] == 0).all()


@pytest.mark.parametrize("A", [30, 3000])
def test_distill_lowest_values_and_repeated_entries(ops, A):
    c = distill_case(4, 6, A, 8)
    c["logits"][0] = torch.finfo(F32).min                       # all equal at the type's lowest: a uniform policy
    c["logits"][1, 1:] = torch.finfo(F32).min                   # a mask written as the type's lowest value
    c["teacher_idx"][1] = 0
    c["teacher_idx"][2] = 3                                     # one action named eight times
    c["teacher_idx"][3, 4:] = c["teacher_idx"][3, :4]           # four named twice
    c["teacher_idx"][4, ::2] = -1                               # a shorter list
    c["teacher_logits"][5, 3] = -math.inf
    distill_check(ops, c)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("K", [8, 100, 256])
@pytest.mark.parametrize("A", [30, 100, 500, 3000, 11000, 20000, 70000])
def test_distill_entries_near_each_other(ops, A, K, dtype):
    """Entries of one action and of neighbouring actions, which one lane or thread holds together."""
    c = distill_case(8, 5, A, K, dtype)
    order = torch.randperm(K, generator=gen(9))
    c["teacher_idx"][0] = (7 + order % 4).int()                 # four actions side by side, named K / 4 times
    c["teacher_idx"][1] = (3 + order % min(24, A - 3)).int()    # more than a lane holds
    c["teacher_idx"][2] = A - 1 - (order % 3).int()             # the last three
    c["teacher_idx"][3] = torch.where(order % 2 == 0, torch.tensor(A // 2), torch.tensor(-5)).int()
    distill_check(ops, c)
    distill_check(ops, c, layout=odd_rows)


@pytest.mark.parametrize("A", [500, 11000, 20000, 70000])
def test_distill_rows_with_nothing_at_other_sizes(ops, A):
    c = distill_case(12, 6, A, 5, avail=True)
    c["weight"][:] = 1.0
    c["avail"][0] = 0.0
    c["teacher_idx"][1] = A
    c["avail"][2].scatter_(0, c["teacher_idx"][2].long(), 0.0)
    c["weight"][3] = 0.0
    c["logits"][3] = math.nan
    c["logits"][4] = -math.inf
    loss, d = distill_check(ops, c)
    assert (loss[:5] == 0).all() and (d[:5] == 0).all() and loss[5] != 0


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("A", [30, 500, 3000, 20000, 70000])
def test_distill_nan_reaches_the_result(ops, A, dtype):
    """A NaN among a row's logits, a row of nothing else, a NaN of the teacher: that row's loss is NaN, the others are as before."""
    c = distill_case(13, 6, A, 5, dtype)
    want = distill_run(ops, c, 2.0, 0.5)
    c["logits"][1, A // 3] = math.nan
    c["logits"][2] = math.nan
    c["teacher_logits"][4, 2] = math.nan
    loss, d = distill_run(ops, c, 2.0, 0.5)
    for row in range(6):
        if row in (1, 2, 4):
            assert torch.isnan(loss[row])
            assert torch.isnan(d[row].float()).all() if row != 4 else torch.isnan(d[row, c["teacher_idx"][4].long().cuda()].float()).all()
        else:
            assert torch.equal(loss[row], want[0][row]) and torch.equal(d[row], want[1][row])


@pytest.mark.parametrize("N,A,dtype", [(1200, 20000, F32), (1100, 13000, BF16), (700, 33000, BF16)])
def test_distill_more_wide_rows_than_workgroups(ops, N, A, dtype):
    """A workgroup takes several rows and requests the next one ahead: rows of weight 0, without entries and without actions in between."""
    c = distill_case(15, N, A, 9, dtype, avail=True)
    c["weight"][::3] = 0.0
    c["logits"][::3] = math.nan
    c["teacher_idx"][1::7] = -1
    c["avail"][2::11] = 0.0
    loss, d = distill_check(ops, c)
    assert (loss[::3] == 0).all() and (d[::3] == 0).all()


def test_distill_wide_rows_captured(ops):
    from xuance_amd.ops import Graph
    c = distill_case(16, 40, 25000, 12)
    dev = {n: t.cuda() for n, t in c.items() if t is not None}
    loss, d = torch.zeros(40, device="cuda"), torch.zeros(40, 25000, device="cuda")
    graph = Graph()
    with graph:
        ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], loss, d_logits=d, weight=dev["weight"], temperature=2.0, grad_scale=0.5)
    want = distill_run(ops, c, 2.0, 0.5)
    for _ in range(3):
        loss.fill_(7.0)
        d.fill_(7.0)
        graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(d, want[1])


def test_distill_layout_in_place_and_loss_only(ops):
    for A, K in ((18, 6), (700, 30), (5000, 12)):
        c = distill_case(5, 9, A, K, avail=True)
        loss, d = distill_check(ops, c)
        l2, d2 = distill_run(ops, c, 2.0, 0.5, layout=odd_rows)
        assert torch.equal(loss, l2) and torch.equal(d, d2)
        l3, _ = distill_run(ops, c, 2.0, 0.5, d_logits=False)
        assert torch.equal(loss, l3)
        dev = {n: t.cuda() for n, t in c.items()}
        ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], l3, d_logits=dev["logits"], avail=dev["avail"],
                         weight=dev["weight"], temperature=2.0, grad_scale=0.5)
        assert torch.equal(dev["logits"], d)


def test_distill_gradient_against_differences(ops):
    c = distill_case(6, 5, 12, 4, avail=True)
    _, d = distill_run(ops, c, 1.5, 1.0)
    way, h = torch.randn(5, 12, generator=gen(2)).float(), 2.0 ** -10
    up = distill_reference({**c, "logits": c["logits"].double() + h * way.double()}, 1.5, 1.0)[0].sum()
    down = distill_reference({**c, "logits": c["logits"].double() - h * way.double()}, 1.5, 1.0)[0].sum()
    # central difference: h^2 / 6 times the third derivative, at most tau^2 (1 / tau)^3 6 |way|^3 a row
    allowed = h * h * (way.double().abs().sum(1) ** 3).sum().item() / 1.5 + 64 * U32 * way.abs().sum().item()
    assert abs((up - down).item() / (2 * h) - (d.double().cpu() * way.double()).sum().item()) <= allowed


def test_distill_without_rows_and_captured(ops):
    from xuance_amd.ops import Graph
    empty = torch.empty(0, 7, device="cuda")
    ops.distill_loss(empty, torch.empty(0, 2, device="cuda", dtype=torch.int32), torch.empty(0, 2, device="cuda"), torch.empty(0, device="cuda"))
    c = distill_case(7, 50, 90, 12, avail=True)
    want = distill_run(ops, c, 2.0, 0.5)
    dev = {n: t.cuda() for n, t in c.items()}
    loss, d = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    graph = Graph()
    with graph:
        ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], loss, d_logits=d, avail=dev["avail"], weight=dev["weight"],
                         temperature=2.0, grad_scale=0.5)
    for _ in range(3):
        loss.fill_(7.5)
        d.fill_(7.5)
        graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(d, want[1])


# ------------------------------------------------------------------------------------------------------- together
def test_sequence_policy_forward_backward_and_acting(ops):
    """pre-norm -> q k v -> linear attention -> projection -> post-norm, gate, residual, norm -> logits -> distillation, as a learner runs it:
    dense layers through xrl_linear_*, all gradients back to every parameter and input against autograd of the whole in float64; then the same
    policy step by step with the state carried."""
    T, B, H, d, A, K = 37, 4, 2, 16, 9, 4
    D, M = H * d, T * B
    g = gen(77)
    lengths = torch.tensor([37, 20, 1, 30], dtype=torch.int32)
    reset = (torch.rand(T, B, generator=g) < 0.1).float()
    ld = torch.tensor([-0.05, -0.5])
    par = {"w_qkv": randn(g, 3 * D, D, mul=D ** -0.5), "w_o": randn(g, D, D, mul=D ** -0.5), "w_g": randn(g, D, D, mul=D ** -0.5),
           "w_head": randn(g, A, D, mul=D ** -0.5), "scale": randn(g, D, mul=0.1) + 0.5, "w_in": randn(g, D, mul=0.1) + 1,
           "w_post": randn(g, D, mul=0.1) + 1, "w_pre": randn(g, D, mul=0.1) + 1}
    x = randn(g, T, B, D)
    tc = distill_case(8, M, A, K, avail=True)
    filled = (torch.arange(T)[:, None] < lengths[None]).float()
    weight = filled.reshape(M)
    eps = 1e-5
    # ---- float64
    leaf = {n: t.double().requires_grad_() for n, t in {**par, "x": x}.items()}
    rms = lambda z, w: z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * w     # noqa: E731
    h0 = rms(leaf["x"], leaf["w_in"])
    qkv = (h0 @ leaf["w_qkv"].T).view(T, B, 3, H, d)
    o, _ = lin_reference(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], ld, d ** -0.5, lengths, reset)
    o = o * filled.double()[..., None, None]
    blk = o.reshape(T, B, D) @ leaf["w_o"].T
    gate = h0 @ leaf["w_g"].T
    y = leaf["x"] + leaf["scale"] * torch.sigmoid(gate) * rms(blk, leaf["w_post"])
    logits = (rms(y, leaf["w_pre"]) @ leaf["w_head"].T).reshape(M, A)
    tau = 2.0
    open_ = tc["avail"] != 0
    ti = tc["teacher_idx"].long()
    tl = torch.where(open_.gather(1, ti), tc["teacher_logits"].double(), torch.full((), -math.inf, dtype=torch.float64))
    some = (tl > -math.inf).any(1)
    q_t = torch.softmax(torch.where(some[:, None], tl, torch.zeros((), dtype=torch.float64)) / tau, 1) * some[:, None]
    lp = torch.log_softmax(logits.masked_fill(~open_, -math.inf) / tau, 1).gather(1, ti)
    kl = torch.where(q_t > 0, q_t * (q_t.clamp(min=1e-300).log() - torch.where(q_t > 0, lp, torch.zeros_like(lp))), torch.zeros_like(q_t)).sum(1)
    loss = (weight.double() * some * tau * tau * kl)
    loss.sum().backward()
    # ---- device
    dev = {n: t.cuda().contiguous() for n, t in {**par, "x": x.reshape(M, D)}.items()}
    new = lambda *s: torch.empty(*s, device="cuda")                                 # noqa: E731
    ones = torch.ones(D, device="cuda")

    def linear(inp, w, out, rows):
        ops.linear_fwd([ops.gemm_desc(inp.data_ptr(), w.data_ptr(), out.data_ptr(), rows, w.shape[0], w.shape[1], w.shape[1], w.shape[1], w.shape[0])])

    def policy(xr, rows, core):
        """xr [rows, D] -> buffers of one pass"""
        b = dict(zero=torch.zeros(rows, D, device="cuda"), h0=new(rows, D), stream=new(rows, D), qkv=new(rows, 3 * D), gate=new(rows, D),
                 o=new(rows, D), blk=new(rows, D), y=new(rows, D), n=new(rows, D), logits=new(rows, A))
        ops.block_norm_forward(xr, b["zero"], b["stream"], b["h0"], w_pre=dev["w_in"])       # nothing added: the first block's norm alone
        linear(b["h0"], dev["w_qkv"], b["qkv"], rows)
        linear(b["h0"], dev["w_g"], b["gate"], rows)
        core(b)
        linear(b["o"], dev["w_o"], b["blk"], rows)
        ops.block_norm_forward(xr, b["blk"], b["y"], b["n"], gate=b["gate"], scale=dev["scale"], w_post=dev["w_post"], w_pre=dev["w_pre"])
        linear(b["n"], dev["w_head"], b["logits"], rows)
        return b

    part = lambda t, i, lead: t[..., i * D:(i + 1) * D].unflatten(-1, (H, d)).unflatten(0, lead)   # noqa: E731
    seq = dict(scale=d ** -0.5, lengths=lengths.cuda(), reset=reset.cuda())
    b = policy(dev["x"], M, lambda b: ops.linattn_forward(*(part(b["qkv"], i, (T, B)) for i in range(3)), part(b["o"], 0, (T, B)), ld.cuda(), **seq))
    tdev = {n: t.cuda() for n, t in tc.items() if t is not None}
    got_loss, d_logits = new(M), new(M, A)
    ops.distill_loss(b["logits"], tdev["teacher_idx"], tdev["teacher_logits"], got_loss, d_logits=d_logits, avail=tdev["avail"],
                     weight=weight.cuda(), temperature=tau, grad_scale=1.0)

    def close(a, ref, what):
        # two norms, four dense layers and the core in f32, every sum under 200 terms: 2e-5 of the tensor's largest value is over 300 u
        ref = ref.detach()
        err = (a.double().cpu() - ref).abs().max().item() / ref.abs().max().item()
        assert err <= 2e-5, f"{what}: {err:.2e}"
    close(got_loss, loss, "loss")
    # backward: data and weight gradients of the dense layers by plain products, everything else by the operators
    r = {n: new(M, D) for n in ("n", "xs", "blk", "gate", "o", "h0", "xs2", "zero")}
    r["qkv"] = new(M, 3 * D)
    grads = {"w_head": d_logits.T @ b["n"]}
    r["n"] = d_logits @ dev["w_head"]
    for n in ("scale", "w_post", "w_pre", "w_in"):
        grads[n] = new(D)
    ops.block_norm_backward(dev["x"], b["blk"], None, r["n"], r["xs"], r["blk"], d_gate=r["gate"], d_scale=grads["scale"], d_w_post=grads["w_post"],
                            d_w_pre=grads["w_pre"], gate=b["gate"], scale=dev["scale"], w_post=dev["w_post"], w_pre=dev["w_pre"])
    grads["w_o"] = r["blk"].T @ b["o"]
    r["o"] = r["blk"] @ dev["w_o"]
    ops.linattn_backward(*(part(b["qkv"], i, (T, B)) for i in range(3)), part(r["o"], 0, (T, B)), *(part(r["qkv"], i, (T, B)) for i in range(3)), ld.cuda(), **seq)
    grads["w_qkv"], grads["w_g"] = r["qkv"].T @ b["h0"], r["gate"].T @ b["h0"]
    r["h0"] = r["qkv"] @ dev["w_qkv"] + r["gate"] @ dev["w_g"]
    ops.block_norm_backward(dev["x"], b["zero"], r["xs"], r["h0"], r["xs2"], r["zero"], d_w_pre=grads["w_in"], w_post=ones, w_pre=dev["w_in"])
    torch.cuda.synchronize()
    for n in grads:
        close(grads[n], leaf[n].grad, n)
    close(r["xs2"].view(T, B, D), leaf["x"].grad, "x")
    # ---- acting: the same rows one step at a time
    S = torch.zeros(B, H, d, d, device="cuda")
    for t in range(T):
        rows = dev["x"][t * B:(t + 1) * B]
        step = policy(rows, B, lambda b: ops.linattn_step(*(part(b["qkv"], i, (B,)) for i in range(3)), part(b["o"], 0, (B,)), ld.cuda(), S, scale=d ** -0.5,
                                                          reset=reset[t].cuda()))
        live = lengths > t
        want = logits.view(T, B, A)[t].detach()[live]
        err = (step["logits"].cpu().double()[live] - want).abs().max().item() / logits.detach().abs().max().item()
        assert err <= 2e-5, (t, err)


def test_refusals_on_the_device(ops):
    from xuance_amd.ops import XrlError
    t = lambda *s, dtype=F32: torch.zeros(*s, device="cuda", dtype=dtype)           # noqa: E731
    q, k, v, o, ld = t(5, 2, 1, 8), t(5, 2, 1, 8), t(5, 2, 1, 4), t(5, 2, 1, 4), t(1)
    ops.linattn_forward(q, k, v, o, ld)
    for bad in (dict(q=q.cpu()), dict(k=t(5, 2, 1, 4)), dict(v=t(5, 2, 1, 4, dtype=BF16)), dict(out=q), dict(out=o[:1].expand(5, -1, -1, -1)),
                dict(log_decay=t(2)), dict(q=t(5, 2, 1, 129), k=t(5, 2, 1, 129)), dict(state=t(2, 1, 8, 4).double()), dict(reset=t(5, 2).bool()),
                dict(lengths=t(2).long()), dict(q=t(5, 2, 1, 16)[..., ::2])):
        with pytest.raises(XrlError):
            ops.linattn_forward(**{**dict(q=q, k=k, v=v, out=o, log_decay=ld), **bad})
    s = t(2, 1, 8, 4)
    with pytest.raises(XrlError):
        ops.linattn_backward(q, k, v, o, t(5, 2, 1, 8), t(5, 2, 1, 8), t(5, 2, 1, 4), ld, d_state_out=s, d_state=s)
    with pytest.raises(XrlError):
        ops.block_norm_forward(t(4, 8), t(4, 8), t(4, 8), eps=0.0)
    with pytest.raises(XrlError):
        ops.distill_loss(t(4, 8), t(4, 300).int(), t(4, 300), t(4))
    torch.cuda.synchronize()
