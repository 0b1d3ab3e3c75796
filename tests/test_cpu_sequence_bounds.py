"""The bounds of tests/sequence_bounds.py see mistakes: planted in the reference, at every size that the GPU tests use; and its formulas
are those that differentiating the definition gives."""
import pytest
import torch

import sequence_bounds as sb

NORM_SIZES = [(7, 3), (33, 20), (64, 64), (130, 65), (50, 128), (37, 200), (40, 256), (21, 511), (19, 512), (9, 1000), (5, 1024), (17, 2048), (3, 4095),
              (6, 4096), (2, 8192), (17001, 64), (1601, 520), (801, 2048), (777, 1999), (300, 8192), (2100, 512)]
DISTILL_SIZES = [(33, 3, 2), (64, 18, 6), (9, 64, 8), (10, 65, 3), (130, 128, 16), (5, 500, 32), (4, 513, 64), (3, 1000, 200), (3, 4099, 32), (2, 8192, 17),
                 (2, 13000, 9), (2, 20001, 64), (2, 50257, 64), (2, 70000, 3), (2, 140001, 9)]


def norm_case(N, D, dtype, gate=True, seed=0):
    g = torch.Generator()
    g.manual_seed(N * 7 + D + seed)
    c = {n: torch.randn(N, D, generator=g).to(dtype) for n in ("x", "u", "gate", "d_y", "d_n")}
    c["u"] = (c["u"].float() * 2 + 0.5).to(dtype)
    if not gate:
        c["gate"] = None
    for n in ("scale", "w_post", "w_pre"):
        c[n] = torch.randn(D, generator=g) * 0.3 + 1
    for n in ("b_post", "b_pre"):
        c[n] = torch.randn(D, generator=g) * 0.3
    return c


def distill_case(N, A, K, dtype, avail=False, seed=0):
    g = torch.Generator()
    g.manual_seed(N + A + seed)
    c = dict(logits=(torch.randn(N, A, generator=g) * 3).to(dtype), teacher_logits=(torch.randn(N, K, generator=g) * 3).to(dtype),
             weight=torch.rand(N, generator=g) + 0.1, avail=None)
    c["teacher_idx"] = torch.stack([torch.randperm(A, generator=g)[:K] for _ in range(N)]).int()
    if avail:
        c["avail"] = (torch.rand(N, A, generator=g) < 0.6).float()
        c["avail"][:, A // 2] = 1.0
        c["avail"].scatter_(1, c["teacher_idx"][:, :1].long(), 1.0)
    return c


def lines_of(N, D, dtype):
    from xuance_amd import ops
    return ops.block_norm_workspace_floats(N, D, dtype=dtype) // (4 * D)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", [True, False])
def test_norm_formulas_are_the_derivatives(kind, gate):
    c = norm_case(9, 12, torch.float32, gate)
    t = {k: v.double().requires_grad_() for k, v in c.items() if v is not None}

    def norm(a, w, b):
        a = a - a.mean(1, keepdim=True) if kind == "layer" else a
        return a / torch.sqrt((a * a).mean(1, keepdim=True) + 1e-5) * w + b
    y = t["x"] + t["scale"] * (torch.sigmoid(t["gate"]) if gate else 1) * norm(t["u"], t["w_post"], t["b_post"])
    n = norm(y, t["w_pre"], t["b_pre"])
    ((y * c["d_y"].double()).sum() + (n * c["d_n"].double()).sum()).backward()
    got = sb.norm_exact(c, kind, 1e-5, 1)
    for k, (v, _) in got.items():
        want = {"y": y, "n": n}[k].detach() if k in "yn" else t[k[2:]].grad
        assert torch.allclose(v, want, rtol=1e-10, atol=1e-12), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("N,D", NORM_SIZES)
def test_norm_bounds_see_mistakes(N, D, kind, dtype):
    c = norm_case(N, D, dtype)
    lines = lines_of(N, D, dtype)
    good = sb.norm_exact(c, kind, 1e-5, lines)

    def seen(bad, names):
        for k in names:
            v, e = good[k]
            assert ((bad[k] - v).abs() > e).any(), k
    seen({k: torch.zeros_like(v) for k, (v, _) in good.items()}, good)                # an output left at 0
    sums = ("d_scale", "d_w_post", "d_b_post", "d_w_pre", "d_b_pre")
    for row in (0, N - 1):                                                            # a row left out of the sums
        seen({k: v for k, (v, _) in sb.norm_exact(c, kind, 1e-5, lines, rows=[i for i in range(N) if i != row]).items()}, sums)
    for term in ("a", "b") if kind == "layer" else ("a",):                            # a term left out of the gradient through a norm
        seen({k: v for k, (v, _) in sb.norm_exact(c, kind, 1e-5, lines, drop=(term,)).items()}, ("d_x", "d_u"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("avail", [False, True], ids=["open", "masked"])
@pytest.mark.parametrize("N,A,K", DISTILL_SIZES)
def test_distill_bounds_see_mistakes(N, A, K, avail, dtype):
    c = distill_case(N, A, K, dtype, avail)
    loss, loss_err, grad, grad_err = sb.distill_exact(c, 2.0, 0.5)
    assert (grad.sum(1).abs() <= 1e-12).all() and (loss >= -1e-12).all()
    no_p = sb.distill_exact(c, 2.0, 0.5, zero_p=True)[2]
    named = torch.zeros_like(grad, dtype=torch.bool).scatter_(1, c["teacher_idx"].long(), True)
    open_ = torch.ones_like(named) if avail is False else c["avail"] != 0
    at = open_ & ~named
    assert ((no_p - grad).abs() > grad_err)[at].all()                                 # every action's probability counts
    assert (grad[~open_] == 0).all() and (grad_err[~open_] <= 1e-36).all()
    if dtype is torch.float32:
        assert ((grad * 1e-4).abs() > grad_err)[at].all()                             # to 1e-4 of itself
    skipped = sb.distill_exact(c, 2.0, 0.5, skip_entry=0)
    assert ((skipped[0] - loss).abs() > loss_err).any() and ((skipped[2] - grad).abs() > grad_err).any()
