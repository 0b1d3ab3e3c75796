"""Numerics of the sequence-policy operators: cases whose sums are exact in f32, what is not finite, sizes beyond a launch, and random values against
bounds of the kernels' own roundings (tests/sequence_bounds.py; tests/test_cpu_sequence_bounds.py plants mistakes that these have to see)."""
import math

import pytest
import torch

import sequence_bounds as sb
from test_cpu_sequence_bounds import DISTILL_SIZES, NORM_SIZES, distill_case, lines_of, norm_case
from test_gpu_sequence_ops import lin_case, lin_expected, lin_run, lin_terms

pytestmark = pytest.mark.gpu

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


# ------------------------------------------------------------------------------------------------------- linear attention
def lin(ops, q, k, v, d_out, log_decay, state=None, d_state_out=None, reset=None, lengths=None, scale=1.0, results=True):
    """Both passes on the device; results: ask for the states too."""
    c = lambda t: None if t is None else t.cuda()                                    # noqa: E731
    q, k, v, d_out, ld = c(q), c(k), c(v), c(d_out), c(torch.as_tensor(log_decay, dtype=F32))
    T, B, H, dk = q.shape
    s = lambda: torch.full((B, H, dk, v.shape[3]), 7.5, device="cuda")              # noqa: E731
    par = dict(scale=scale, lengths=c(lengths), reset=c(reset), state=c(state))
    r = dict(out=torch.empty_like(v))
    if results:
        r["state_out"] = s()
    ops.linattn_forward(q, k, v, r["out"], ld, state_out=r.get("state_out"), **par)
    r.update(d_q=torch.empty_like(q), d_k=torch.empty_like(k), d_v=torch.empty_like(v))
    if results:
        r["d_state"] = s()
    ops.linattn_backward(q, k, v, d_out, r["d_q"], r["d_k"], r["d_v"], ld, d_state_out=c(d_state_out), d_state=r.get("d_state"), **par)
    torch.cuda.synchronize()
    return {n: t.cpu() for n, t in r.items()}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [4, 32, 64, 128])
def test_linattn_products_keep_the_bits_of_f32(ops, d, dtype):
    """Scores and states of 21 bits against ones that take all but the last of them away again: every sum is exact in f32, in any order."""
    a, rest = 1 + 2.0 ** -10 + 2.0 ** -20, 2.0 ** -20
    z = lambda T: torch.zeros(T, 1, 1, d, dtype=dtype)                               # noqa: E731
    # scores: q_1 k_0 = a, q_1 k_1 = a - rest, v_0 = 1, v_1 = -1; the same numbers through v and d_out give d_q
    q, k, v, do = z(2), z(2), z(2), z(2)
    row = torch.tensor([1, 2.0 ** -10, 2.0 ** -20], dtype=dtype)
    q[1, 0, 0, :3], k[0, 0, 0, :3], k[1, 0, 0, :2] = row, 1, 1
    v[0], v[1] = 1, -1
    assert (lin(ops, q, k, v, do, [0.0])["out"][1] == rest).all()
    q, k, v, do = z(2), z(2), z(2), z(2)
    do[1, 0, 0, :3], v[0, 0, 0, :3], v[1, 0, 0, :2] = row, 1, 1
    k[0], k[1] = 1, -1
    assert (lin(ops, q, k, v, do, [0.0])["d_q"][1] == rest).all()
    # states: rows a and -(a - rest), both read with weight 1
    S = torch.zeros(1, 1, d, d)
    S[0, 0, 0], S[0, 0, 1] = a, rest - a
    x = z(1)
    x[0, 0, 0, :2] = 1
    assert (lin(ops, x, z(1), z(1), z(1), [0.0], state=S)["out"] == rest).all()
    assert (lin(ops, z(1), x, z(1), z(1), [0.0], d_state_out=S)["d_v"] == rest).all()
    assert (lin(ops, z(1), z(1), z(1), x, [0.0], state=S.transpose(2, 3).contiguous())["d_q"] == rest).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("T,B", [(300, 3), (1300, 1)])
def test_linattn_outputs_do_not_depend_on_the_states_asked_for(ops, T, B, d, dtype):
    g = gen(T + d)
    q, k, v, do = (torch.randn(T, B, 2, d, generator=g).to(dtype) for _ in range(4))
    a, b = (lin(ops, q, k, v, do, [-0.01, -0.2], scale=d ** -0.5, results=r) for r in (True, False))
    for n in b:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("T,B", [(150, 3), (1300, 2)])
def test_linattn_reset_ends_any_state(ops, T, B, d, dtype):
    """A NaN or infinite state, given or overflowed, ends at a reset like any other: the rest of the row has the bits that it has without it."""
    g = gen(T + d)
    q, k, v, do = (torch.randn(T, B, 2, d, generator=g).to(dtype) for _ in range(4))
    S, dS = torch.randn(B, 2, d, d, generator=g), torch.randn(B, 2, d, d, generator=g)
    reset = torch.zeros(T, B)
    reset[0, 0] = reset[T // 2, 1] = reset[T // 2 + 3, 0] = 1
    par = dict(log_decay=[-0.01, -0.2], reset=reset, scale=d ** -0.5)
    S[0] = 0.0
    want = lin(ops, q, k, v, do, state=S, d_state_out=dS, **par)
    for bad in (torch.nan, torch.inf):
        S0 = S.clone()
        S0[0] = bad                                                                  # reset before the first step
        got = lin(ops, q, k, v, do, state=S0, d_state_out=dS, **par)
        for n in want:
            assert torch.equal(got[n], want[n]), (n, bad)
        S1, dS1 = S.clone(), dS.clone()
        S1[1], dS1[0] = bad, bad                                                     # ends in the middle: after it; before it for its gradient
        got = lin(ops, q, k, v, do, state=S1, d_state_out=dS1, **par)
        half = T // 2
        for n in ("out", "d_q"):
            assert torch.equal(got[n][half:], want[n][half:]) and torch.equal(got[n][:, 0], want[n][:, 0]), (n, bad)
            assert not torch.isfinite(got[n][:half, 1].float()).all()
        for n in ("d_k", "d_v"):
            assert torch.equal(got[n][:half + 3], want[n][:half + 3]) and torch.equal(got[n][:, 1], want[n][:, 1]), (n, bad)
            assert not torch.isfinite(got[n][half + 3:, 0].float()).all()
        assert torch.equal(got["state_out"], want["state_out"]) and torch.equal(got["d_state"], want["d_state"]), bad


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("at", [3, 60, 64, 100])
@pytest.mark.parametrize("T", [200, 1300])
def test_linattn_overflow_of_one_episode_stays_in_it(ops, T, at, d, dtype):
    """Finite keys and values whose product is not: the steps behind the next reset have the bits that they have without them."""
    g = gen(T + d + at)
    q, k, v, do = (torch.randn(T, 1, 1, d, generator=g).to(dtype) for _ in range(4))
    reset = torch.zeros(T, 1)
    reset[at + 5] = 1
    want = lin(ops, q, k, v, do, [-0.01], reset=reset)
    k[at], v[at] = 1e30, 1e30
    got = lin(ops, q, k, v, do, [-0.01], reset=reset)
    for n in ("out", "d_q", "d_k", "d_v"):
        assert torch.equal(got[n][at + 5:], want[n][at + 5:]), n
    assert torch.equal(got["state_out"], want["state_out"])
    assert not torch.isfinite(got["out"][at:at + 5].float()).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,B,H,dk,dv", [(1500, 4, 1, 128, 128), (1500, 4, 1, 128, 64), (2100, 3, 2, 64, 128), (1100, 5, 1, 32, 32)])
def test_linattn_split_ragged_rows(ops, T, B, H, dk, dv, dtype):
    """Rows of several lengths, resets and a state, the time axis cut into segments; and the same bits when it runs again.  An output is held to what
    f32 sums may be off by in either type, a bf16 one to its own rounding more."""
    assert ops.linattn_workspace_floats(T, B, H, dk, dv, dtype=dtype) > 0 and ops.linattn_workspace_floats(T, B, H, dk, dv, backward=True, dtype=dtype) > 0
    c = lin_case(T + dk, T, B, H, dk, dv, dtype, "ragged", False, True, log_decay=[-0.004, -0.1][:H])
    c["reset"] = torch.zeros(T, B)
    c["reset"][T // 3, 0] = c["reset"][200, 1] = 1
    got, again = lin_run(ops, c), lin_run(ops, c)
    ref, mag = lin_expected(c)
    rel = lin_terms(dk, dv, T, F32)
    for n in got:
        assert torch.equal(got[n], again[n]), n
        stored = 2.0 ** -8 * (1 + rel) * ref[n].abs() if got[n].dtype is BF16 else 0.0
        assert ((got[n].cpu().double() - ref[n]).abs() <= rel * mag[n] * (1 + 2.0 ** -8) + stored + 1e-37).all(), n


def test_linattn_step_decay_is_rounded_once(ops):
    """S exp(log_decay) is the f32 next to its value: long memories (1 - 1e-6 a step) and short ones.  The two floats of the decay are off by 2^-49
    of it, which the bound on half a step leaves room for."""
    H, d = 8, 64
    ld = torch.tensor([-1e-6, -2e-6, -2e-8, -1e-4, -0.01, -0.5, -3.0, -20.0])
    S = torch.randn(5, H, d, d, generator=gen(1))
    zero, out, after = torch.zeros(5, H, d, device="cuda"), torch.empty(5, H, d, device="cuda"), torch.empty(5, H, d, d, device="cuda")
    ops.linattn_step(zero, zero, zero, out, ld.cuda(), S.cuda(), state_out=after)
    want = S.double() * torch.exp(ld.double()).view(1, H, 1, 1)
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 25)
    assert ((after.cpu().double() - want).abs() <= half * (1 + 2.0 ** -20)).all()


def test_linattn_step_and_sequence_agree_on_decays_at_both_ends(ops):
    """No decay, positive (taken as 0), no memory, NaN: what the sequence form makes of them."""
    ld = torch.tensor([0.0, 0.5, -math.inf, math.nan, -1.0])
    g = gen(2)
    q, k, v = (torch.randn(1, 2, 5, 16, generator=g).cuda() for _ in range(3))
    S = torch.randn(2, 5, 16, 16, generator=g).cuda()
    a, b, o1, o2 = torch.empty_like(S), torch.empty_like(S), torch.empty_like(v), torch.empty_like(v)
    ops.linattn_forward(q, k, v, o1, ld.cuda(), state=S, state_out=a)
    ops.linattn_step(q[0], k[0], v[0], o2[0], ld.cuda(), S, state_out=b)
    for t in (o1[0], o2[0], a, b):
        assert torch.isnan(t[:, 3]).all()
    rest = [0, 1, 2, 4]
    # 16 products and sums, three roundings of a state: under 64 u of the terms' magnitudes
    lam = torch.exp(ld.clamp(max=0.0)).view(1, 5, 1, 1).cuda()
    mag = (lam * S.abs() + k[0, ..., :, None].abs() * v[0, ..., None, :].abs())[:, rest]
    assert ((a[:, rest] - b[:, rest]).abs() <= 8 * 2.0 ** -24 * mag).all()
    assert ((o1[0][:, rest] - o2[0][:, rest]).abs() <= 64 * 2.0 ** -24 * (q[0][:, rest].abs()[..., None] * mag).sum(2)).all()


def test_linattn_step_of_many_rows(ops):
    """16.8 million rows and heads, each with 256 threads: more than a launch takes."""
    B, H = 1 << 22, 4
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    q, k, v = (torch.randn(B, H, 2, generator=g, device="cuda") for _ in range(3))
    S, out, reset = torch.randn(B, H, 2, 2, generator=g, device="cuda"), torch.empty(B, H, 2, device="cuda"), (torch.rand(B, generator=g, device="cuda") < 0.5).float()
    ld = torch.tensor([-0.1, -0.2, -0.3, -0.4], device="cuda")
    after = torch.full_like(S, 7.5)
    ops.linattn_step(q, k, v, out, ld, S, state_out=after, reset=reset)
    for rows in (slice(0, 1000), slice((1 << 21) - 500, (1 << 21) + 500), slice(B - 1000, B)):
        o, a = torch.empty(1000, H, 2, device="cuda"), torch.empty(1000, H, 2, 2, device="cuda")
        ops.linattn_step(q[rows], k[rows], v[rows], o, ld, S[rows], state_out=a, reset=reset[rows])
        assert torch.equal(out[rows], o) and torch.equal(after[rows], a)


# ------------------------------------------------------------------------------------------------------- block norm
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", [True, False], ids=["gate", "open"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("N,D", NORM_SIZES)
def test_block_norm_within_its_roundings(ops, N, D, kind, gate, dtype):
    c = norm_case(N, D, dtype, gate)
    dev = {n: (None if t is None else t.cuda()) for n, t in c.items()}
    par = dict(kind=kind, eps=1e-5, gate_act="sigmoid", **{n: dev[n] for n in ("gate", "scale", "w_post", "b_post", "w_pre", "b_pre")})
    got = {n: torch.full((N, D), 7.5, device="cuda", dtype=dtype) for n in ("y", "n", "d_x", "d_u") + (("d_gate",) if gate else ())}
    got.update({n: torch.full((D,), 7.5, device="cuda") for n in ("d_scale", "d_w_post", "d_b_post", "d_w_pre", "d_b_pre")})
    ops.block_norm_forward(dev["x"], dev["u"], got["y"], got["n"], **par)
    ops.block_norm_backward(dev["x"], dev["u"], dev["d_y"], dev["d_n"], **{k: v for k, v in got.items() if k.startswith("d_")}, **par)
    for n, (want, bound) in sb.norm_exact(c, kind, 1e-5, lines_of(N, D, dtype)).items():
        worst = ((got[n].cpu().double() - want).abs() / bound).max().item()
        assert worst <= 1, (n, worst)


# ------------------------------------------------------------------------------------------------------- distillation
def test_distill_of_many_rows(ops):
    """537 million rows, 8 threads each: more than a launch takes.  The policy's logits are one row for all."""
    N = (1 << 29) + 5
    logits = torch.tensor([[0.5, -1.0]], device="cuda").expand(N, 2)
    idx, top, loss = torch.ones(N, 1, dtype=torch.int32, device="cuda"), torch.zeros(N, 1, device="cuda"), torch.full((N,), 7.5, device="cuda")
    idx[-3:] = 0
    ops.distill_loss(logits, idx, top, loss)
    want = math.log(1 + math.exp(1.5)), math.log(1 + math.exp(-1.5))
    for part, ref in ((loss[:-3], want[0]), (loss[-3:], want[1])):
        assert part.max() == part.min() and abs(part[0].item() - ref) <= 16 * 2.0 ** -24 * (ref + 1.5)


def test_distill_rows_of_several_launches(ops):
    """Every tensor of a call goes on at the right row."""
    N, A, K = (1 << 21) + 77, 3, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    logits, top = torch.randn(N, A, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda")
    idx = torch.randint(0, A, (N, K), generator=g, device="cuda", dtype=torch.int32)
    avail, weight = (torch.rand(N, A, generator=g, device="cuda") < 0.7).float(), torch.rand(N, generator=g, device="cuda")
    wide = torch.full((N, A + 2), 7.5, device="cuda")
    loss, d = torch.full((N,), 7.5, device="cuda"), wide[:, 1:-1]
    ops.distill_loss(logits, idx, top, loss, d_logits=d, avail=avail, weight=weight)
    rows = slice((1 << 21) - 100, N)
    l2, d2 = torch.empty(177, device="cuda"), torch.empty(177, A, device="cuda")
    ops.distill_loss(logits[rows], idx[rows], top[rows], l2, d_logits=d2, avail=avail[rows], weight=weight[rows])
    assert torch.equal(loss[rows], l2) and torch.equal(d[rows], d2) and (wide[:, 0] == 7.5).all() and (wide[:, -1] == 7.5).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("avail", [False, True], ids=["open", "masked"])
@pytest.mark.parametrize("tau", [2.0, 0.4])
@pytest.mark.parametrize("N,A,K", DISTILL_SIZES)
def test_distill_within_its_roundings(ops, N, A, K, tau, avail, dtype):
    """Loss and gradient, and the loss alone: the same bits."""
    c = distill_case(N, A, K, dtype, avail)
    dev = {n: (None if t is None else t.cuda()) for n, t in c.items()}
    loss, alone, d = torch.full((N,), 7.5, device="cuda"), torch.full((N,), 7.5, device="cuda"), torch.full((N, A), 7.5, device="cuda", dtype=dtype)
    par = dict(avail=dev["avail"], weight=dev["weight"], temperature=tau, grad_scale=0.5)
    ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], loss, d_logits=d, **par)
    ops.distill_loss(dev["logits"], dev["teacher_idx"], dev["teacher_logits"], alone, **par)
    assert torch.equal(loss, alone)
    want, bound, grad, grad_bound = sb.distill_exact(c, tau, 0.5)
    for n, g, v, e in (("loss", loss, want, bound), ("d_logits", d, grad, grad_bound)):
        off = (g.cpu().double() - v).abs()
        assert (off <= e).all(), (n, (off / e.clamp(min=1e-300)).max().item())
