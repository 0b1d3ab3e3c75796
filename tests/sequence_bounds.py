"""The block norms and the distillation loss in float64, and how far the kernels may be off: every rounding of their arithmetic once, with
u = 2^-24 (half a step of f32), carried through the formulas to first order (and 1 % for the higher ones).

Roundings counted.  A sum, a product, a fused product and sum, a quotient and a square root: u of the result each (csrc builds with exact quotients and roots).
v_exp_f32 and v_rcp_f32: 2 u.  A stored bf16: 2^-8 of itself.  Sums: as many u of their terms' magnitudes as additions follow each other on the
longest way from a term to the result."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8
SLACK = 1.01


def up_to_power(n, least):
    p = least
    while p < n:
        p *= 2
    return p


# ------------------------------------------------------------------------------------------------------- block norm
def norm_depths(N, D, lines):
    """Additions behind each other: of a row's sum (8 values a lane, a tree over up to 64 lanes, the waves in turn) and of a column's (the rows of a
    workgroup, a tree over the wave's rows, its waves, the lines of 64 groups, the groups)."""
    L = up_to_power((D + 7) // 8, 8)
    rows = 1 if L > 64 else 256 // L
    waves = L // 64 if L > 64 else 4
    row = 8 + int(math.log2(min(L, 64))) + (waves if L > 64 else 0)
    column = math.ceil(N / (lines * rows)) + (int(math.log2(64 // L)) + 4 if L <= 64 else 0) + math.ceil(lines / 64) + 64
    return row, column


class _Norm:
    """xhat = (x - mean) r of a value known up to `err`, and what xhat, r are off by."""

    def __init__(self, x, err, kind, eps, e_row):
        m = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
        v = x - m
        var = (v * v).mean(1, keepdim=True)
        self.r = 1 / torch.sqrt(var + eps)
        self.hat = v * self.r
        # its own arithmetic: the mean; the difference; the sum of squares, 1 / D, its product with eps, the root, the quotient
        shift = (e_row + 2 * U32) * x.abs().mean(1, keepdim=True) if kind == "layer" else 0.0
        self.r_rel = 0.5 * (e_row + 4 * U32) + 2 * U32 + 0.5 * (shift * self.r) ** 2
        own = self.hat.abs() * (self.r_rel + 2 * U32) + self.r * shift
        # what the value brings along
        carried = (self.hat.abs() * err).mean(1, keepdim=True) * self.r
        self.r_rel = self.r_rel + carried
        self.err = own + self.r * (err + (err.mean(1, keepdim=True) if kind == "layer" else 0.0)) + self.hat.abs() * carried

    def back(self, t, t_err, kind, e_row, drop=()):
        """r (t - xhat mean(t xhat) - mean(t)) of t known up to t_err, and what it is off by."""
        a, b = (t * self.hat).mean(1, keepdim=True), t.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
        a_err = (t.abs() * self.err + t_err * self.hat.abs()).mean(1, keepdim=True) + (e_row + 2 * U32) * (t * self.hat).abs().mean(1, keepdim=True)
        b_err = (t_err.mean(1, keepdim=True) + (e_row + 2 * U32) * t.abs().mean(1, keepdim=True)) if kind == "layer" else 0.0
        inner = t - b - self.hat * a
        err = self.r * (t_err + self.err * a.abs() + self.hat.abs() * a_err + b_err + U32 * (t - b).abs() + U32 * inner.abs()) \
            + self.r * inner.abs() * (self.r_rel + U32)
        if "a" in drop:
            inner = t - b
        if "b" in drop:
            inner = t - self.hat * a
        return self.r * inner, err


def norm_exact(c, kind, eps, lines, drop=(), rows=None):
    """c: x, u, gate (None: no gate; the sigmoid of it otherwise), scale, w_post, b_post, w_pre, b_pre, d_y, d_n (missing parameters None) ->
    {name: (value, bound)}.  drop, rows: mistakes for the tests of the bounds (a term of the gradient left out; only these rows in the sums)."""
    N, D = c["x"].shape
    d = {k: (None if v is None else v.double()) for k, v in c.items()}
    one, nil = torch.ones(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    par = {k: d[k] if d.get(k) is not None else (one if k in ("scale", "w_post", "w_pre") else nil) for k in ("scale", "w_post", "b_post", "w_pre", "b_pre")}
    sc, w0, b0, w1, b1 = (par[k] for k in ("scale", "w_post", "b_post", "w_pre", "b_pre"))
    depth_row, depth_col = norm_depths(N, D, lines)
    e_row, e_col = depth_row * U32, depth_col * U32
    zero = torch.zeros(N, D, dtype=torch.float64)
    U = _Norm(d["u"], zero, kind, eps, e_row)
    p = U.hat * w0 + b0
    p_err = w0.abs() * U.err + U32 * p.abs()
    if d["gate"] is None:
        a, a_err, slope, slope_err = zero + 1, zero, None, None
    else:
        # exp(-z): z log2(e) and that constant are rounded, then the exponential; 1 + it; the reciprocal
        a = torch.sigmoid(d["gate"])
        a_err = a * ((1 - a) * (1.5 * d["gate"].abs() + 2) + 3) * U32
        slope = a * (1 - a)
        slope_err = a_err * (1 - a) + a * (a_err + U32 * (1 - a)) + U32 * slope
    y = d["x"] + sc * a * p
    y_err = (sc * a).abs() * p_err + (sc * p).abs() * a_err + U32 * (sc * a * p).abs() + U32 * y.abs()
    Y = _Norm(y, y_err, kind, eps, e_row)
    n = Y.hat * w1 + b1
    out = {"y": (y, y_err), "n": (n, w1.abs() * Y.err + U32 * n.abs())}
    t = d["d_n"] * w1
    back, back_err = Y.back(t, U32 * t.abs(), kind, e_row, drop)
    dy = d["d_y"] + back
    dy_err = back_err + U32 * dy.abs()
    out["d_x"] = (dy, dy_err)
    da = dy * a
    da_err = a.abs() * dy_err + dy.abs() * a_err + U32 * da.abs()
    t = da * sc * w0
    out["d_u"] = U.back(t, (sc * w0).abs() * da_err + 2 * U32 * t.abs(), kind, e_row, drop)
    if slope is not None:
        g = dy * sc * p * slope
        out["d_gate"] = (g, (sc * p * slope).abs() * dy_err + (dy * sc * slope).abs() * p_err + (dy * sc * p).abs() * slope_err + 3 * U32 * g.abs())
    keep = slice(None) if rows is None else rows

    def column(term, err):
        return term[keep].sum(0), err.sum(0) + e_col * (term.abs() + err).sum(0)
    s0, s0_err = column(da, da_err)
    s1, s1_err = column(da * U.hat, da_err * U.hat.abs() + da.abs() * U.err)
    out["d_scale"] = (w0 * s1 + b0 * s0, w0.abs() * s1_err + b0.abs() * s0_err + 2 * U32 * ((w0 * s1).abs() + (b0 * s0).abs()))
    out["d_w_post"] = (sc * s1, sc.abs() * (s1_err + U32 * s1.abs()))
    out["d_b_post"] = (sc * s0, sc.abs() * (s0_err + U32 * s0.abs()))
    out["d_w_pre"] = column(d["d_n"] * Y.hat, d["d_n"].abs() * Y.err)
    out["d_b_pre"] = column(d["d_n"], zero)
    stored = U16 if c["x"].dtype is torch.bfloat16 else 0.0
    return {k: (v, SLACK * e + (stored * (v.abs() + e) if v.dim() == 2 else 0.0) + 1e-37) for k, (v, e) in out.items()}


# ------------------------------------------------------------------------------------------------------- distillation
def distill_depth(A, dtype):
    """Additions behind each other in the sum of a row's exponentials, by the form that takes rows of this size; the longest rows' running sum is
    scaled anew where the maximum grows, three more roundings a piece at the most."""
    e = 4 if dtype is torch.float32 else 2
    if A <= 512:
        return 8 + 6
    if A * e <= (16 if e == 4 else 24) * 1024:
        return math.ceil(A / 64) + 16 // e * 4 + 6                   # pieces that the row does not have add nothing
    if A * e <= (256 if e == 4 else 128) * 1024:
        threads = 512 if A * e <= 512 * 64 else 1024
        return math.ceil(A / threads) + 16 // e * 4 + 6 + threads // 64
    pieces = math.ceil(A * e / (1024 * 16))
    return pieces * (16 // e + 3) + 6 + 16


def distill_exact(c, tau, grad_scale, zero_p=False, skip_entry=None):
    """Row by row -> loss, its bound, d_logits, its bound.  zero_p, skip_entry: mistakes for the tests of the bounds."""
    N, A = c["logits"].shape
    K = c["teacher_idx"].shape[1]
    depth = distill_depth(A, c["logits"].dtype)
    loss, loss_err = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    grad, grad_err = torch.zeros(N, A, dtype=torch.float64), torch.zeros(N, A, dtype=torch.float64)
    for n in range(N):
        w = 1.0 if c["weight"] is None else c["weight"][n].item()
        open_ = torch.ones(A, dtype=torch.bool) if c["avail"] is None else c["avail"][n] != 0
        idx, t = c["teacher_idx"][n].long(), c["teacher_logits"][n].double()
        ok = (idx >= 0) & (idx < A) & (t > -math.inf)
        ok &= open_[idx.clamp(0, A - 1)]
        s = torch.where(open_, c["logits"][n].double(), torch.full((), -math.inf, dtype=torch.float64))
        if w == 0 or not ok.any() or not (s > -math.inf).any():
            continue
        idx, t = idx[ok], t[ok]
        far, far_t = (s.max() - s) / tau, (t.max() - t) / tau         # arguments of the exponentials: a difference and two products, the last with 1 / tau log2(e)
        p, q = torch.softmax(-far, 0), torch.softmax(-far_t, 0)
        dist = torch.where(p > 0, far, torch.zeros_like(far))
        e_rel, t_rel = (4 * dist + 2) * U32, (4 * far_t + 2) * U32
        z_rel = (p * e_rel).sum() + depth * U32
        ts_rel = (q * t_rel).sum() + (K + 22) * U32
        p_rel, q_rel = e_rel + z_rel + 3 * U32, t_rel + ts_rel + 2 * U32
        lq, lp = -far_t - torch.logsumexp(-far_t, 0), -far - torch.logsumexp(-far, 0)
        lz, lt = torch.logsumexp(-far, 0).abs(), torch.logsumexp(-far_t, 0).abs()
        # a logarithm passes a relative error on as an absolute one and adds two roundings; of the teacher's, taken of the exponential or of its argument
        lq_err = t_rel + ts_rel + U32 * (4 * far_t + 2 * lt + lq.abs())
        lp_err = z_rel + U32 * (4 * far[idx] + 2 * lz + lp[idx].abs())
        term = q * (lq - lp[idx])
        term_err = q * (lq_err + lp_err) + term.abs() * (q_rel + 2 * U32)
        scale = w * tau * tau
        if skip_entry is not None:
            term = torch.cat([term[:skip_entry], term[skip_entry + 1:]])
        loss[n] = scale * term.sum()
        loss_err[n] = abs(scale) * (term_err.sum() + (K + 22 + 3) * U32 * (term.abs() + term_err[:len(term)]).sum())
        k = grad_scale * w * tau
        named = torch.zeros(A, dtype=torch.float64).index_add(0, idx, q)
        named_err = torch.zeros(A, dtype=torch.float64).index_add(0, idx, q * (q_rel + K * U32))
        if zero_p:
            grad[n] = -k * named
        elif skip_entry is not None:
            at = min(skip_entry, len(idx) - 1)
            grad[n] = k * (p - named.index_add(0, idx[at:at + 1], -q[at:at + 1]))
        else:
            grad[n] = k * (p - named)
        grad_err[n] = abs(k) * (p * (p_rel + 4 * U32) + named_err + 4 * U32 * named + U32 * (p - named).abs() + 2.0 ** -126)
    stored = U16 * (grad.abs() + grad_err) if c["logits"].dtype is torch.bfloat16 else 0.0
    return loss, SLACK * loss_err + 1e-37, grad, SLACK * grad_err + stored + torch.where(grad_err > 0, 1e-37, 0.0)
