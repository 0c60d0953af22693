"""Plain 64-bit forms of the network operators, and the roundings their tests allow."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a step, relative
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # half a step of subnormals, or under it


def assert_within(got, ref, bound, what=""):
    """|got - ref| <= bound everywhere (64-bit ref; NaN and infinities in the same places)."""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    bound = torch.as_tensor(bound).double().cpu().expand_as(ref)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what + ": NaN in other places"
    ok = torch.isfinite(ref)
    assert torch.equal(got[~ok & ~torch.isnan(ref)], ref[~ok & ~torch.isnan(ref)]), what
    if ok.any():
        over = ((got - ref).abs() - bound)[ok]
        assert over.max() <= 0, f"{what}: {over.max():.3g} over the bound, error {(got - ref).abs()[ok].max():.3g}"


# ---- 8-bit blocks ------------------------------------------------------------------------------------------------
def put_away(x, fmt):
    """x (1-d, 64 bits) -> the values its blocks stand for, element by element from the format's definition."""
    out = torch.empty_like(x)
    for lo in range(0, x.numel(), 32):
        b = x[lo:lo + 32]
        fin = b[torch.isfinite(b)].abs()
        top = float(fin.max()) if fin.numel() else 0.0
        e = math.frexp(top)[1] - 1 if top > 0 else -1000
        if fmt == "int8":
            s = e - 6
            s += top * 2.0 ** -s >= 127.5 if top > 0 else 0
        else:
            s = e - 8
            s += top * 2.0 ** -s > 448 if top > 0 else 0
        s = max(s, -126)
        m = b * 2.0 ** -s
        if fmt == "int8":
            c = torch.round(m)
        else:
            step = torch.where(m.abs() >= 2.0 ** -6, torch.exp2(torch.frexp(m.abs())[1].double() - 1 - 3), torch.full_like(m, 2.0 ** -9))
            c = torch.round(m / step) * step
        v = c * 2.0 ** s
        v[~torch.isfinite(b)] = float("nan")
        out[lo:lo + 32] = v
    return out


def put_away_rows(x, fmt):
    return torch.stack([put_away(r, fmt) for r in x.reshape(-1, x.shape[-1])]).reshape(x.shape)


def act(x, kind):
    return 0.5 * x * torch.erfc(-x / math.sqrt(2)) if kind == "gelu" else x * torch.sigmoid(x)


def act_slope(x, kind):
    if kind == "gelu":
        return 0.5 * torch.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(x)
    return s + x * s * (1 - s)


# ---- norms -------------------------------------------------------------------------------------------------------
def norm(v, w, b, layer, eps=1e-6):
    m = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[..., :1])
    r = ((v - m) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return m, r, (v - m) * r * w + (0 if b is None else b)


def block_norm(x, u, gate, scale, w, b, w1, b1, layer, sigmoid, eps=1e-6):
    """y, h of 64-bit tensors (differentiable); gate broadcasts."""
    y = x
    if u is not None:
        n = norm(u, w, b, layer, eps)[2]
        if gate is not None:
            n = n * (torch.sigmoid(gate) if sigmoid else gate)
        y = x + (n if scale is None else scale * n)
    return y, None if w1 is None else norm(y, w1, b1, layer, eps)[2]


def block_norm_backward(x, u, gate, scale, w, b, w1, b1, layer, sigmoid, stats, dy, dh):
    """Gradients at the given x, u, gate with the given statistics (mu_u, r_u, mu_y, r_y), by the formulas, per row."""
    one = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    s = one if scale is None else scale

    def back(g, hat, r):
        return r * (g - (g.mean(-1, keepdim=True) if layer else 0) - hat * (g * hat).mean(-1, keepdim=True))

    mu_u, r_u, mu_y, r_y = stats
    out, t = {}, torch.zeros_like(x) if dy is None else dy
    rows = tuple(range(x.dim() - 1))
    if u is not None:
        hat = (u - mu_u) * r_u
        n = hat * w + (0 if b is None else b)
        a = torch.ones_like(x) if gate is None else (torch.sigmoid(gate) if sigmoid else gate)
        da = torch.sigmoid(gate) * (1 - torch.sigmoid(gate)) if gate is not None and sigmoid else 1.0
    if dh is not None:
        yhat = ((x if u is None else x + s * a * n) - mu_y) * r_y
        t = t + back(dh * w1, yhat, r_y)
        out["next_weight"], out["next_bias"] = (dh * yhat).sum(rows), dh.sum(rows)
    out["x"] = t
    if u is not None:
        out["u"] = back(t * s * a * w, hat, r_u)
        out["weight"], out["bias"], out["scale"] = (t * s * a * hat).sum(rows), (t * s * a).sum(rows), (t * a * n).sum(rows)
        if gate is not None:
            out["gate"] = t * s * n * da
    return out


# ---- linear attention --------------------------------------------------------------------------------------------
def attention(q, k, v, log_decay, state, lengths, scale):
    """out [b, t, h, dv], end state, both differentiable, by the full t x t form in the inputs' type."""
    b, t, h, dk = q.shape
    n = torch.full((b,), t, device=q.device) if lengths is None else lengths.long()
    i = torch.arange(t, device=q.device)
    live = (i[None] < n[:, None]).to(q.dtype)
    a = log_decay.to(q.dtype).clamp(min=-1e30)
    w = torch.exp(a[:, None, None] * (i[:, None] - i[None]).clamp(min=0)) * (i[:, None] >= i[None])
    p = torch.einsum("bihd,bjhd->bhij", q, k) * w * live[:, None, :, None] * live[:, None, None]
    o = torch.einsum("bhij,bjhe->bihe", p, v)
    left = (n[:, None] - 1 - i[None]).clamp(min=0)
    end = torch.einsum("bth,bthd,bthe->bhde", torch.exp(a * left[..., None]) * live[..., None], k, v)
    if state is not None:
        o = o + torch.einsum("bthd,bhde->bthe", q * torch.exp(a * (i[:, None] + 1))[None, :, :, None] * live[..., None, None], state)
        end = end + torch.exp(a[None] * n[:, None])[..., None, None] * state
    return o * scale, end
