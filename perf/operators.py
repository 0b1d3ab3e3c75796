"""Measured calls of the sequence-policy operators: the decayed linear-attention core (whole sequences, their gradients, one acting
step), the norms around a block with its gate and residual scale, and the distillation loss against a teacher's top logits.

`own` false: elementary torch operations in 32 bits (decay powers in 64), rounded once at the end.  `own` true: the calls of
xuance_amd.ops.  Every output buffer is made beforehand, as the framework's programs do."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one acting step of 16 environments, the smallest vector of the PPO benchmark: launch latency
        dict(name="step_16_envs", op="step", B=16, H=4, dk=16, dv=16, dtype="f32", reset=True),
        # one acting step of a large vector: the state streams through memory
        dict(name="step_4096_envs", op="step", B=4096, H=4, dk=64, dv=64, dtype="f32", reset=True),
        # one update on padded episodes of the recurrent multi-agent workload: 32 episodes x 3 agents, 61 steps, hidden 64
        dict(name="episodes_61", op="seq", T=61, B=96, H=4, dk=16, dv=16, dtype="f32", grad=True, ragged=True, reset=False, state=False),
        # one update on a rollout of 256 environments x 256 steps with episode ends inside the sequences
        dict(name="rollout_256x256", op="seq", T=256, B=256, H=4, dk=64, dv=64, dtype="f32", grad=True, ragged=False, reset=True, state=True),
        # one long context read for serving: a single row, the state kept
        dict(name="context_32768_bf16", op="seq", T=32768, B=1, H=8, dk=128, dv=128, dtype="bf16", grad=False, ragged=False, reset=False, state=True),
        # a training step on long ragged sequences in 16 bits
        dict(name="train_4096_bf16", op="seq", T=4096, B=8, H=8, dk=128, dv=128, dtype="bf16", grad=True, ragged=True, reset=False, state=False),
        # the norms of one acting step
        dict(name="norm_step_256", op="norm", N=256, D=64, dtype="f32", kind="rms", gate=True, bias=False, grad=False),
        # the norms of an update on 256 x 256 rows
        dict(name="norm_train_65536x256", op="norm", N=65536, D=256, dtype="f32", kind="rms", gate=True, bias=False, grad=True),
        # wide rows in 16 bits, an odd number of them
        dict(name="norm_train_30011x2048_bf16", op="norm", N=30011, D=2048, dtype="bf16", kind="layer", gate=True, bias=True, grad=True),
        # a minibatch of an 18-action policy with availability masks
        dict(name="distill_256x18", op="distill", N=256, A=18, K=6, dtype="f32", avail=True, grad=True),
        # a large discrete action space in 16 bits
        dict(name="distill_8192x4099_bf16", op="distill", N=8192, A=4099, K=32, dtype="bf16", avail=False, grad=True),
        # a token-sized action space, odd width
        dict(name="distill_4096x50257", op="distill", N=4096, A=50257, K=64, dtype="f32", avail=False, grad=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "seq", "seq", "norm", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    dims = [16, 32, 64, 128, rng.randrange(5, 129), 4 * rng.randrange(2, 33)]
    if op == "step":
        return dict(op=op, B=_log_uniform(rng, 1, 4096), H=rng.randrange(1, 5), dk=rng.choice(dims[:3] + [rng.randrange(5, 65)]),
                    dv=rng.choice(dims[:3] + [rng.randrange(5, 65)]), dtype=dtype, reset=rng.random() < 0.5)
    if op == "seq":
        H, dk, dv = rng.randrange(1, 9), rng.choice(dims), rng.choice(dims)
        T = _log_uniform(rng, 1, 32768)
        most = 8 * 4096 * 8 * 128 // (T * H * max(dk, dv))          # no more rows x channels than the largest listed case
        return dict(op=op, T=T, B=_log_uniform(rng, 1, max(1, min(512, most))), H=H, dk=dk, dv=dv, dtype=dtype, grad=rng.random() < 0.6,
                    ragged=rng.random() < 0.5, reset=rng.random() < 0.5, state=rng.random() < 0.5)
    if op == "norm":
        D = rng.choice([64, 128, 256, 512, 1024, 2048, rng.randrange(3, 4097), _log_uniform(rng, 3, 4096)])
        return dict(op=op, N=_log_uniform(rng, 1, min(1 << 17, 30011 * 2048 // D)), D=D, dtype=dtype, kind=rng.choice(["rms", "layer"]),
                    gate=rng.random() < 0.7, bias=rng.random() < 0.5, grad=rng.random() < 0.6)
    A = _log_uniform(rng, 2, 65536)
    return dict(op=op, N=_log_uniform(rng, 1, min(1 << 17, 4096 * 50257 // A)), A=A, K=rng.randrange(1, min(A, 64) + 1), dtype=dtype,
                avail=rng.random() < 0.5, grad=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * mul).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    return {"step": _prepare_step, "seq": _prepare_seq, "norm": _prepare_norm, "distill": _prepare_distill}[case["op"]](case, g, dt)


def _log_decay(H, g):
    """Memory lengths from a few steps to a few hundred, another for each head."""
    half = 2.0 ** (2 + 6 * torch.rand(H, generator=g, device="cuda", dtype=torch.float64))
    return (-math.log(2.0) / half).float()


def _prepare_step(c, g, dt):
    B, H, dk, dv = c["B"], c["H"], c["dk"], c["dv"]
    s = dict(op="step", q=_randn(g, B, H, dk, dtype=dt), k=_randn(g, B, H, dk, dtype=dt), v=_randn(g, B, H, dv, dtype=dt),
             log_decay=_log_decay(H, g), scale=dk ** -0.5, state=_randn(g, B, H, dk, dv, mul=3.0),
             reset=(torch.rand(B, generator=g, device="cuda") < 0.05).float() if c["reset"] else None)
    s["out"], s["state_out"] = torch.empty_like(s["v"]), torch.empty_like(s["state"])
    return s


def _prepare_seq(c, g, dt):
    T, B, H, dk, dv = c["T"], c["B"], c["H"], c["dk"], c["dv"]
    s = dict(op="seq", grad=c["grad"], q=_randn(g, T, B, H, dk, dtype=dt), k=_randn(g, T, B, H, dk, dtype=dt),
             v=_randn(g, T, B, H, dv, dtype=dt), log_decay=_log_decay(H, g), scale=dk ** -0.5)
    s["lengths"] = torch.randint((T + 1) // 2, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if c["ragged"] else None
    s["reset"] = (torch.rand(T, B, generator=g, device="cuda") < 0.01).float() if c["reset"] else None
    s["state"] = _randn(g, B, H, dk, dv) if c["state"] else None
    s["out"] = torch.empty_like(s["v"])
    s["state_out"] = torch.empty(B, H, dk, dv, device="cuda") if c["state"] else None
    if c["grad"]:
        s["d_out"] = _randn(g, T, B, H, dv, dtype=dt)
        s["d_state_out"] = _randn(g, B, H, dk, dv) if c["state"] else None
        s["d_q"], s["d_k"], s["d_v"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
        s["d_state"] = torch.empty_like(s["state"]) if c["state"] else None
    return s


def _prepare_norm(c, g, dt):
    N, D = c["N"], c["D"]
    s = dict(op="norm", grad=c["grad"], kind=c["kind"], eps=1e-5, x=_randn(g, N, D, dtype=dt), u=_randn(g, N, D, dtype=dt, mul=2.0) + 0.25,
             gate=_randn(g, N, D, dtype=dt) if c["gate"] else None, scale=_randn(g, D, mul=0.1) + 0.5,
             w_post=_randn(g, D, mul=0.1) + 1.0, w_pre=_randn(g, D, mul=0.1) + 1.0,
             b_post=_randn(g, D, mul=0.1) if c["bias"] else None, b_pre=_randn(g, D, mul=0.1) if c["bias"] else None)
    s["y"], s["n"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    if c["grad"]:
        s["d_y"], s["d_n"] = _randn(g, N, D, dtype=dt), _randn(g, N, D, dtype=dt)
        s["d_x"], s["d_u"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["d_gate"] = torch.empty_like(s["x"]) if c["gate"] else None
        for name in ("scale", "w_post", "w_pre") + (("b_post", "b_pre") if c["bias"] else ()):
            s["d_" + name] = torch.empty(D, device="cuda")
    return s


def _prepare_distill(c, g, dt):
    N, A, K = c["N"], c["A"], c["K"]
    teacher = _randn(g, N, A, mul=3.0)
    s = dict(op="distill", grad=c["grad"], temperature=2.0, grad_scale=1.0 / N, logits=_randn(g, N, A, dtype=dt, mul=3.0),
             weight=(torch.rand(N, generator=g, device="cuda") < 0.9).float(), avail=None)
    if c["avail"]:
        s["avail"] = (torch.rand(N, A, generator=g, device="cuda") < 0.7).float()
        s["avail"][:, 0] = 1.0
    top = teacher.topk(K, dim=1)
    s["teacher_idx"], s["teacher_logits"] = top.indices.to(torch.int32), top.values.to(dt)
    s["loss"] = torch.empty(N, device="cuda")
    s["d_logits"] = torch.empty_like(s["logits"]) if c["grad"] else None
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _own_step(s):
    from xuance_amd import ops
    ops.linattn_step(s["q"], s["k"], s["v"], s["out"], s["log_decay"], s["state"], state_out=s["state_out"], scale=s["scale"], reset=s["reset"])
    return {"out": s["out"], "state": s["state_out"]}


def _own_seq(s):
    from xuance_amd import ops
    ops.linattn_forward(s["q"], s["k"], s["v"], s["out"], s["log_decay"], scale=s["scale"], lengths=s["lengths"], reset=s["reset"],
                        state=s["state"], state_out=s["state_out"])
    r = {"out": s["out"], "state": s["state_out"]}
    if s["grad"]:
        ops.linattn_backward(s["q"], s["k"], s["v"], s["d_out"], s["d_q"], s["d_k"], s["d_v"], s["log_decay"], scale=s["scale"],
                             lengths=s["lengths"], reset=s["reset"], state=s["state"], d_state_out=s["d_state_out"], d_state=s["d_state"])
        r.update(d_q=s["d_q"], d_k=s["d_k"], d_v=s["d_v"], d_state=s["d_state"])
    return r


def _own_norm(s):
    from xuance_amd import ops
    par = dict(gate=s["gate"], gate_act="sigmoid", scale=s["scale"], w_post=s["w_post"], b_post=s["b_post"], w_pre=s["w_pre"], b_pre=s["b_pre"],
               kind=s["kind"], eps=s["eps"])
    ops.block_norm_forward(s["x"], s["u"], s["y"], s["n"], **par)
    r = {"y": s["y"], "n": s["n"]}
    if s["grad"]:
        sums = {k: s.get(k) for k in ("d_scale", "d_w_post", "d_b_post", "d_w_pre", "d_b_pre")}
        ops.block_norm_backward(s["x"], s["u"], s["d_y"], s["d_n"], s["d_x"], s["d_u"], d_gate=s["d_gate"], **sums, **par)
        r.update(d_x=s["d_x"], d_u=s["d_u"], d_gate=s["d_gate"], **sums)
    return r


def _own_distill(s):
    from xuance_amd import ops
    ops.distill_loss(s["logits"], s["teacher_idx"], s["teacher_logits"], s["loss"], d_logits=s["d_logits"], avail=s["avail"],
                     weight=s["weight"], temperature=s["temperature"], grad_scale=s["grad_scale"])
    return {"loss": s["loss"], "d_logits": s["d_logits"]}


_OWN = {"step": _own_step, "seq": _own_seq, "norm": _own_norm, "distill": _own_distill}


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_step(s):
    lam = s["log_decay"].double().exp().float()[:, None, None]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    state = s["state"] if s["reset"] is None else torch.where((s["reset"] != 0)[:, None, None, None], torch.zeros_like(s["state"]), s["state"])
    state = lam * state + k[..., :, None] * v[..., None, :]
    out = s["scale"] * (q[..., :, None] * state).sum(-2)
    return {"out": out.to(s["v"].dtype), "state": state}


CHUNK = 64


def _powers(log_decay, n):
    """exp(log_decay * n) for every head and whole number in n, 0 where n is negative: [H, *n.shape]."""
    p = torch.exp(log_decay.double().reshape(-1, *[1] * n.dim()) * n.clamp(min=0).double())
    return torch.where(n < 0, torch.zeros_like(p), p).float()


def _mix(a, b, c, log_decay, ids):
    """sum over j <= i of one segment of decay^(i - j) (a_i . b_j) c_j, in chunks: [B, H, T, *], ids [B, T]."""
    B, H, T, _ = a.shape
    n = -(-T // CHUNK)
    pad = n * CHUNK - T
    if pad:
        a, b, c = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (a, b, c))
        ids = torch.cat([ids, ids[:, -1:].expand(B, pad)], 1)
    a, b, c = (x.reshape(B, H, n, CHUNK, -1) for x in (a, b, c))
    ids = ids.reshape(B, 1, n, CHUNK)
    i = torch.arange(CHUNK, device=a.device)
    within = _powers(log_decay, i[:, None] - i[None, :])[None, :, None] * (ids[..., :, None] == ids[..., None, :])
    out = (torch.matmul(a, b.transpose(-1, -2)) * within) @ c
    if n == 1:
        return out.reshape(B, H, -1, out.shape[-1])[:, :, :T]
    last = ids[..., -1]                                                            # [B, 1, n]
    w_b = _powers(log_decay, CHUNK - 1 - i)[None, :, None] * (ids == last[..., None])
    sums = torch.matmul((b * w_b[..., None]).transpose(-1, -2).contiguous(), c)    # what each chunk adds to the state
    before = torch.cat([last[..., :1] - 1, last[..., :-1]], -1)                    # the segment that the state before a chunk belongs to
    m = torch.arange(n, device=a.device)
    carry = _powers(log_decay, CHUNK * (m[:, None] - 1 - m[None, :]))[None] * (before[..., :, None] == last[..., None, :])
    state = torch.matmul(carry, sums.reshape(B, H, n, -1)).reshape(sums.shape)
    w_a = _powers(log_decay, i + 1)[None, :, None] * (ids == before[..., None])
    out = out + torch.matmul(a * w_a[..., None], state)
    return out.reshape(B, H, n * CHUNK, -1)[:, :, :T]


def _plain_seq(s):
    T, B = s["q"].shape[:2]
    heads = lambda x: x.permute(1, 2, 0, 3).float()                                # noqa: E731  [T, B, H, d] -> [B, H, T, d]
    back = lambda x, like: x.permute(2, 0, 1, 3).to(like.dtype).contiguous()       # noqa: E731
    t = torch.arange(T, device=s["q"].device)
    n = torch.full((B,), T, device=t.device) if s["lengths"] is None else s["lengths"].long()
    inside = t[None] < n[:, None]
    ids = torch.zeros(B, T, device=t.device, dtype=torch.long) if s["reset"] is None else ((s["reset"].T != 0) & inside).cumsum(1)
    keep = inside[:, None, :, None]
    q, k, v = (torch.where(keep, heads(s[x]), torch.zeros((), device=t.device)) for x in "qkv")
    g, scale = s["log_decay"], s["scale"]
    out = _mix(q, k, v, g, ids)
    end = ids[:, -1]                                                               # the segment that each row ends in
    w_in = _powers(g, t + 1)[None] * ((ids == 0) & inside)[:, None]                # [B, H, T]
    w_out = _powers(g, n[:, None] - 1 - t[None]).transpose(0, 1) * ((ids == end[:, None]) & inside)[:, None]
    whole = (_powers(g, n).T * (end == 0)[:, None])[..., None, None]               # [B, H, 1, 1]
    if s["state"] is not None:
        out = out + w_in[..., None] * (q @ s["state"])
    r = {"out": back(out * scale, s["v"]), "state": None}
    if s["state_out"] is not None:
        r["state"] = (k * w_out[..., None]).transpose(-1, -2).contiguous() @ v + whole * s["state"]
    if not s["grad"]:
        return r
    d = torch.where(keep, heads(s["d_out"]), torch.zeros((), device=t.device)) * scale
    flip = lambda x: x.flip(-2)                                                    # noqa: E731
    ids_r = end[:, None] - ids.flip(1)
    d_q = _mix(d, v, k, g, ids)
    d_k = flip(_mix(flip(v), flip(d), flip(q), g, ids_r))
    d_v = flip(_mix(flip(k), flip(q), flip(d), g, ids_r))
    if s["state"] is not None:
        S, dS = s["state"], s["d_state_out"]
        d_q = d_q + w_in[..., None] * (d @ S.transpose(-1, -2).contiguous())
        d_k = d_k + w_out[..., None] * (v @ dS.transpose(-1, -2).contiguous())
        d_v = d_v + w_out[..., None] * (k @ dS)
    r.update(d_q=back(d_q, s["q"]), d_k=back(d_k, s["k"]), d_v=back(d_v, s["v"]), d_state=None)
    if s["state"] is not None:
        r["d_state"] = (q * w_in[..., None]).transpose(-1, -2).contiguous() @ d + whole * s["d_state_out"]
    return r


def _norm(x, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return x * r, r


def _norm_back(d, xhat, r, kind):
    d = d - xhat * (d * xhat).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return d * r


def _plain_norm(s):
    dt, kind = s["x"].dtype, s["kind"]
    x, u = s["x"].float(), s["u"].float()
    uhat, ru = _norm(u, kind, s["eps"])
    p = uhat * s["w_post"] + (0.0 if s["b_post"] is None else s["b_post"])
    a = 1.0 if s["gate"] is None else 1.0 / (1.0 + torch.exp(-s["gate"].float()))
    y = x + s["scale"] * a * p
    yhat, ry = _norm(y, kind, s["eps"])
    n = yhat * s["w_pre"] + (0.0 if s["b_pre"] is None else s["b_pre"])
    r = {"y": y.to(dt), "n": n.to(dt)}
    if not s["grad"]:
        return r
    dn = s["d_n"].float()
    dy = s["d_y"].float() + _norm_back(dn * s["w_pre"], yhat, ry, kind)
    dp = dy * s["scale"] * a
    r.update(d_x=dy.to(dt), d_u=_norm_back(dp * s["w_post"], uhat, ru, kind).to(dt), d_gate=None,
             d_scale=(dy * a * p).sum(0), d_w_post=(dp * uhat).sum(0), d_b_post=None, d_w_pre=(dn * yhat).sum(0), d_b_pre=None)
    if s["gate"] is not None:
        r["d_gate"] = (dy * s["scale"] * p * a * (1.0 - a)).to(dt)
    if s["b_post"] is not None:
        r["d_b_post"], r["d_b_pre"] = dp.sum(0), dn.sum(0)
    return r


def _plain_distill(s):
    tau, dt = s["temperature"], s["logits"].dtype
    z = s["logits"].float()
    idx, t = s["teacher_idx"].long(), s["teacher_logits"].float()
    low = torch.full((), float("-inf"), device=z.device)
    if s["avail"] is not None:
        z = torch.where(s["avail"] != 0, z, low)
        t = torch.where(s["avail"].gather(1, idx) != 0, t, low)
    z = (z - z.amax(1, keepdim=True)) / tau
    lse = z.exp().sum(1, keepdim=True).log()
    some = (t > low).any(1, keepdim=True)
    t = torch.where(some, t, torch.zeros_like(t))
    t = (t - t.amax(1, keepdim=True)) / tau
    log_q = t - t.exp().sum(1, keepdim=True).log()
    q = torch.where(some, log_q.exp(), torch.zeros_like(t))
    terms = torch.where(q > 0, q * (log_q - z.gather(1, idx) + lse), torch.zeros_like(q))
    r = {"loss": s["weight"] * tau * tau * terms.sum(1), "d_logits": None}
    if s["grad"]:
        p = (z - lse).exp() * some
        r["d_logits"] = (p.scatter_add(1, idx, -q) * (s["grad_scale"] * tau * s["weight"])[:, None]).to(dt)
    return r


_PLAIN = {"step": _plain_step, "seq": _plain_seq, "norm": _plain_norm, "distill": _plain_distill}


# ------------------------------------------------------------------------------------------------------------ work of one pass
def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "step":
        rows, kv = c["B"] * c["H"], c["dk"] * c["dv"]
        return {"bytes": rows * (8 * kv + e * (2 * c["dk"] + 2 * c["dv"])) + 4 * c["H"] + (4 * c["B"] if c["reset"] else 0), "flops": 5 * rows * kv}
    if c["op"] == "seq":
        T, rows, kv = c["T"], c["B"] * c["H"], c["dk"] * c["dv"]
        tokens = T * 0.75 if c["ragged"] else T                        # mean length of the ragged rows
        reads = tokens * rows * e * (2 * c["dk"] + c["dv"] + (c["dv"] if c["grad"] else 0))
        writes = T * rows * e * (c["dv"] + (2 * c["dk"] + c["dv"] if c["grad"] else 0))
        states = rows * kv * 4 * ((4 if c["grad"] else 2) if c["state"] else 0)
        return {"bytes": reads + writes + states + (4 * T * c["B"] if c["reset"] else 0),
                "flops": tokens * rows * kv * (4 + (8 if c["grad"] else 0))}
    if c["op"] == "norm":
        n = c["N"] * c["D"]
        reads, writes = 2 + c["gate"] + (2 if c["grad"] else 0), 2 + ((2 + c["gate"]) if c["grad"] else 0)
        return {"bytes": n * e * (reads + writes) + 4 * c["D"] * 5 * (2 if c["grad"] else 1), "flops": n * (20 + (30 if c["grad"] else 0))}
    n = c["N"] * c["A"]
    return {"bytes": n * (e + (e if c["grad"] else 0) + (4 if c["avail"] else 0)) + c["N"] * (c["K"] * (4 + e) + 8), "flops": n * (4 + (3 if c["grad"] else 0))}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_step, "seq": _exact_seq, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](s)


def _exact_step(s):
    S = s["state"].double().clone()
    if s["reset"] is not None:
        S[s["reset"] != 0] = 0
    S = S * torch.exp(s["log_decay"].double()).view(1, -1, 1, 1) + torch.einsum("bhd,bhe->bhde", s["k"].double(), s["v"].double())
    return {"out": s["scale"] * torch.einsum("bhd,bhde->bhe", s["q"].double(), S), "state": S}


def _exact_seq(s):
    """The definition with the whole weight matrix, a block of target steps at a time: one row of the batch after another."""
    T, B, H, dk = s["q"].shape
    dv = s["v"].shape[-1]
    g = s["log_decay"].double()
    new = lambda *shape: torch.zeros(*shape, device="cuda", dtype=torch.float64)   # noqa: E731
    r = {"out": new(T, B, H, dv), "state": None}
    if s["state"] is not None:
        r["state"] = new(B, H, dk, dv)
    if s["grad"]:
        r.update(d_q=new(T, B, H, dk), d_k=new(T, B, H, dk), d_v=new(T, B, H, dv), d_state=new(B, H, dk, dv) if s["state"] is not None else None)
    lengths = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = lengths[b]
        q, k, v = (s[x][:n, b].double().transpose(0, 1) for x in "qkv")
        do = s["d_out"][:n, b].double().transpose(0, 1) * s["scale"] if s["grad"] else None
        seg = torch.zeros(n, device="cuda", dtype=torch.long) if s["reset"] is None else (s["reset"][:n, b] != 0).cumsum(0)
        at = torch.arange(n, device="cuda")
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            dist = at[lo:hi, None] - at[None, :hi]
            w = torch.exp(g.view(-1, 1, 1) * dist.clamp(min=0)) * ((dist >= 0) & (seg[lo:hi, None] == seg[None, :hi]))
            r["out"][lo:hi, b] += s["scale"] * ((w * (q[:, lo:hi] @ k[:, :hi].transpose(1, 2))) @ v[:, :hi]).transpose(0, 1)
            if s["grad"]:
                m = w * (do[:, lo:hi] @ v[:, :hi].transpose(1, 2))
                r["d_q"][lo:hi, b] += (m @ k[:, :hi]).transpose(0, 1)
                r["d_k"][:hi, b] += (m.transpose(1, 2) @ q[:, lo:hi]).transpose(0, 1)
                r["d_v"][:hi, b] += ((w * (q[:, lo:hi] @ k[:, :hi].transpose(1, 2))).transpose(1, 2) @ do[:, lo:hi]).transpose(0, 1)
        if s["state"] is None:
            continue
        last = seg[-1] if n else torch.zeros((), device="cuda", dtype=torch.long)
        first = torch.exp(g[:, None] * (at + 1)) * (seg == 0)
        rest = torch.exp(g[:, None] * (n - 1 - at)) * (seg == last)
        through = torch.exp(g * n).view(-1, 1, 1) * (last == 0)
        S = s["state"][b].double()
        r["out"][:n, b] += s["scale"] * (first[..., None] * (q @ S)).transpose(0, 1)
        r["state"][b] = (k * rest[..., None]).transpose(1, 2) @ v + through * S
        if s["grad"]:
            dS = s["d_state_out"][b].double()
            r["d_q"][:n, b] += (first[..., None] * (do @ S.transpose(1, 2))).transpose(0, 1)
            r["d_k"][:n, b] += (rest[..., None] * (v @ dS.transpose(1, 2))).transpose(0, 1)
            r["d_v"][:n, b] += (rest[..., None] * (k @ dS)).transpose(0, 1)
            r["d_state"][b] = (q * first[..., None]).transpose(1, 2) @ do + through * dS
    return r


def _exact_norm(s):
    """The forward definition in 64 bits; gradients by differentiating it."""
    names = ["x", "u", "gate", "scale", "w_post", "b_post", "w_pre", "b_pre"]
    v = {k: s[k].double().requires_grad_(s["grad"]) if s[k] is not None else None for k in names}

    def norm(t, w, b):
        m = t.mean(1, keepdim=True) if s["kind"] == "layer" else torch.zeros_like(t[:, :1])
        h = (t - m) / torch.sqrt(((t - m) ** 2).mean(1, keepdim=True) + s["eps"]) * w
        return h if b is None else h + b

    block = norm(v["u"], v["w_post"], v["b_post"]) * v["scale"]
    if v["gate"] is not None:
        block = torch.sigmoid(v["gate"]) * block
    y = v["x"] + block
    n = norm(y, v["w_pre"], v["b_pre"])
    r = {"y": y.detach(), "n": n.detach()}
    if s["grad"]:
        ((y * s["d_y"].double()).sum() + (n * s["d_n"].double()).sum()).backward()
        r.update({"d_" + k: None if v[k] is None else v[k].grad for k in names})
    return r


def _exact_distill(s):
    N, A = s["logits"].shape
    tau = s["temperature"]
    loss = torch.zeros(N, device="cuda", dtype=torch.float64)
    grad = torch.zeros(N, A, device="cuda", dtype=torch.float64) if s["grad"] else None
    rows = max(1, (1 << 26) // A)
    for lo in range(0, N, rows):
        at = slice(lo, min(N, lo + rows))
        open_ = torch.ones_like(s["logits"][at], dtype=torch.bool) if s["avail"] is None else s["avail"][at] != 0
        teacher = torch.zeros(open_.shape, device="cuda", dtype=torch.float64)
        weights = torch.exp((s["teacher_logits"][at].double() - s["teacher_logits"][at].double().amax(1, keepdim=True)) / tau)
        teacher.scatter_add_(1, s["teacher_idx"][at].long(), weights)
        teacher = teacher * open_
        mass = teacher.sum(1, keepdim=True)
        teacher = torch.where(mass > 0, teacher / mass, torch.zeros_like(teacher))
        log_p = torch.log_softmax((s["logits"][at].double() / tau).masked_fill(~open_, float("-inf")), 1)
        w = s["weight"][at].double()
        loss[at] = w * tau * tau * torch.where(teacher > 0, teacher * (teacher.log() - log_p), torch.zeros_like(teacher)).sum(1)
        if grad is not None:
            grad[at] = (log_p.exp() * (mass > 0) - teacher) * (w * tau * s["grad_scale"])[:, None]
    return {"loss": loss, "d_logits": grad}
