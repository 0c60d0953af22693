"""Timed cases of the network operators in front of the optimisation layers: linear attention with a decay for each
head (`linattn`), norms around a gated residual block (`blocknorm`) and activations kept in 8 bits for the backward pass
(`ckpt8`).

`run` makes one pass, either as plain torch operations in 32 bits (`own` false) or through the package (`own` true);
`exact` gives the same outputs from the operators' definitions in 64 bits."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32                     # elements that share one scale of an 8-bit checkpoint


# ---- cases ------------------------------------------------------------------------------------------------------
def _norm(name, rows, d, dtype, wdtype, kind="rms", gate="full", groups=1, gate_kind="sigmoid", bias=False, scale=True,
          nxt=True, train=True, checkpoint=""):
    return {"name": name, "op": "norm", "rows": rows, "d": d, "dtype": dtype, "wdtype": wdtype, "kind": kind, "gate": gate,
            "groups": groups, "gate_kind": gate_kind, "bias": bias, "scale": scale, "next": nxt, "train": train,
            "checkpoint": checkpoint}


def _lin(name, b, t, h, dk, dv, dtype, train, ragged=False, state=True):
    return {"name": name, "op": "lin", "b": b, "t": t, "h": h, "dk": dk, "dv": dv, "dtype": dtype, "train": train,
            "ragged": ragged, "state": state}


def listed():
    return [
        # a few streams advance by one token: latency of the fused post norm, gate, residual and next pre norm
        _norm("norm_token", 4, 1024, "bfloat16", "bfloat16", train=False),
        # one training step at the block border, batch 8 of 96 x 320 pixels (a quarter of 384 x 1280), one gate per image
        _norm("norm_train_image_gate", 245760, 128, "bfloat16", "float32", gate="group", groups=8),
        # odd image (375 x 1242 over 8), odd channel count, layer norm with biases, last block (no next norm), fp32
        _norm("norm_train_odd", 21996, 150, "float32", "float32", kind="layer", bias=True, nxt=False),
        # wide block whose backward pass reads 8-bit checkpoints of stream, block output and gate
        _norm("norm_train_wide_8bit", 61440, 512, "bfloat16", "bfloat16", kind="layer", bias=True, checkpoint="int8"),
        # feature maps of the quadratic fit, 8 x 32 x 384 x 1280, put away and brought back
        {"name": "store_features", "op": "store", "n": 8 * 32 * 384 * 1280, "dtype": "float32", "fmt": "int8"},
        # hidden activation of a pixel-wise MLP, batch 8 of 96 x 320 pixels, forward and backward
        {"name": "act_gelu_train", "op": "act", "n": 245760 * 512, "dtype": "bfloat16", "fmt": "int8", "kind": "gelu"},
        # the same for a small odd map
        {"name": "act_silu_small", "op": "act", "n": 47 * 156 * 37, "dtype": "float16", "fmt": "e4m3", "kind": "silu"},
        # one stream advances by one token
        {"name": "lin_step_one", "op": "step", "b": 1, "h": 4, "dk": 32, "dv": 32, "dtype": "float16"},
        # a full serving batch advances by one token
        {"name": "lin_step_batch", "op": "step", "b": 128, "h": 16, "dk": 128, "dv": 128, "dtype": "bfloat16"},
        # one image of 192 x 640 tokens, inference with the end state
        _lin("lin_prompt_image", 1, 122880, 8, 64, 64, "bfloat16", False, state=False),
        # training step, batch 8 of 48 x 160 tokens
        _lin("lin_train", 8, 7680, 8, 128, 128, "bfloat16", True, state=False),
        # padded batch of odd lengths, odd head sizes, fp32, gradients of the carried state too
        _lin("lin_train_ragged", 3, 1955, 5, 40, 56, "float32", True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "lin", "lin", "step", "store", "act"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if op == "norm":
        d = _log(rng, 8, 8192)
        if rng.random() < 0.7:
            d = max(8, d // 8 * 8)
        rows = _log(rng, 1, max(2, 31457280 // d))
        gate = rng.choice(["full", "group", "none"])
        groups = 1
        if gate == "group":
            groups = min(rows, _log(rng, 1, 16))
            rows = max(2, rows // groups) * groups          # a gate as long as the stream is a full gate
        nxt = rng.random() < 0.7
        c = _norm("", rows, d, dtype, rng.choice([dtype, "float32"]), rng.choice(["rms", "layer"]), gate, groups,
                  rng.choice(["sigmoid", "identity"]), rng.random() < 0.5, rng.random() < 0.7, nxt, rng.random() < 0.7,
                  rng.choice(["", "", "int8", "e4m3"]))
        if not c["train"]:
            c["checkpoint"] = ""
    elif op == "lin":
        dk, dv = _log(rng, 8, 128), _log(rng, 8, 128)
        if rng.random() < 0.6:
            dk, dv = max(8, dk // 8 * 8), max(8, dv // 8 * 8)
        h = _log(rng, 1, 16)
        t = _log(rng, 1, 30720)
        train = rng.random() < 0.6
        b = _log(rng, 1, max(2, min(64, 30000000 // (t * h * max(dk, dv)))))
        c = _lin("", b, t, h, dk, dv, dtype, train, rng.random() < 0.4, rng.random() < 0.5)
        if dtype == "float32":      # the 32-bit cases stand for smaller problems
            c["t"] = max(1, c["t"] // 4)
    elif op == "step":
        dk, dv = _log(rng, 8, 128), _log(rng, 8, 128)
        c = {"op": "step", "b": _log(rng, 1, 128), "h": _log(rng, 1, 16), "dk": dk, "dv": dv, "dtype": dtype}
    elif op == "store":
        c = {"op": "store", "n": _log(rng, 1000, 60000000), "dtype": dtype, "fmt": rng.choice(["int8", "e4m3"])}
    else:
        c = {"op": "act", "n": _log(rng, 1000, 60000000), "dtype": dtype, "fmt": rng.choice(["int8", "e4m3"]),
             "kind": rng.choice(["gelu", "silu"])}
    c.pop("name", None)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, mul=1.0, add=0.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return x.mul_(mul).add_(add).to(dtype)

    s = {"case": dict(case)}
    op = case["op"]
    if op == "norm":
        rows, d, wt = case["rows"], case["d"], DTYPES[case["wdtype"]]
        # a residual stream has a few channels far larger than the others, and a mean that is not zero
        channel = torch.exp(torch.randn(d, generator=g, device="cuda"))
        s["x"] = (torch.randn(rows, d, generator=g, device="cuda").add_(0.2) * channel).to(dt)
        s["u"] = normal(rows, d, mul=0.7, add=0.1)
        s["gate"] = (normal(rows, d) if case["gate"] == "full" else normal(case["groups"], d) if case["gate"] == "group" else None)
        s["w"] = normal(d, dtype=wt, mul=0.1, add=1.0)
        s["b"] = normal(d, dtype=wt, mul=0.1) if case["bias"] else None
        s["scale"] = normal(d, dtype=wt, mul=0.02, add=0.3) if case["scale"] else None
        s["w1"] = normal(d, dtype=wt, mul=0.1, add=1.0) if case["next"] else None
        s["b1"] = normal(d, dtype=wt, mul=0.1) if case["next"] and case["bias"] else None
        if case["train"]:
            s["dy"] = normal(rows, d)
            s["dh"] = normal(rows, d) if case["next"] else None
        leaves = [k for k in ("x", "u", "gate", "w", "b", "scale", "w1", "b1") if s[k] is not None]
        if case["gate"] == "group":      # what a user has: one image is [pixels, channels], its gate [1, channels]
            s["x"], s["u"] = (t.view(case["groups"], -1, d) for t in (s["x"], s["u"]))
            s["gate"] = s["gate"].view(case["groups"], 1, d)
            for k in ("dy", "dh"):
                if s.get(k) is not None:
                    s[k] = s[k].view(case["groups"], -1, d)
        s["leaves"] = leaves
    elif op in ("lin", "step"):
        h, dk, dv = case["h"], case["dk"], case["dv"]
        lead = (case["b"], case["t"]) if op == "lin" else (case["b"],)
        s["q"] = normal(*lead, h, dk)
        s["k"] = normal(*lead, h, dk, mul=dk ** -0.5)
        s["v"] = normal(*lead, h, dv)
        # memories from a few tokens to a few thousand, one per head
        s["log_decay"] = -torch.exp2(-torch.linspace(2.0, 11.0, h, device="cuda"))
        s["state"] = normal(case["b"], h, dk, dv, dtype=torch.float32) if op == "step" or case["state"] else None
        s["leaves"] = ["q", "k", "v"] + (["state"] if s["state"] is not None else [])
        if op == "lin":
            s["lengths"] = None
            if case["ragged"]:
                n = torch.randint(0, case["t"] + 1, (case["b"],), generator=g, device="cuda", dtype=torch.int32)
                n[0] = case["t"]
                s["lengths"] = n
            if case["train"]:
                s["do"] = normal(*lead, h, dv)
                s["dstate"] = normal(case["b"], h, dk, dv, dtype=torch.float32, mul=0.1)
    else:
        n = case["n"]
        s["x"] = normal(n)
        s["x"] *= torch.exp2(torch.randint(-3, 3, (n // 4096 + 1,), generator=g, device="cuda").float()).to(dt).repeat_interleave(4096)[:n]
        if op == "act":
            s["dy"] = normal(n)
        s["leaves"] = ["x"]
    if case.get("train") or op == "act":
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------
def _put_away(x, fmt):
    """x [rows, d] in 32 bits -> the values that its 8-bit blocks stand for."""
    rows, d = x.shape
    pad = -d % BLOCK
    z = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)
    top = z.abs().amax(-1, keepdim=True)
    e = torch.frexp(top).exponent - 1
    if fmt == "int8":
        s = e - 6
        s = s + (torch.ldexp(top, -s) >= 127.5).int()
        s = s.clamp(-126, 127)
        c = torch.round(torch.ldexp(z, -s))
    else:
        s = e - 8
        s = s + (torch.ldexp(top, -s) > 448).int()
        s = s.clamp(-126, 127)
        c = torch.ldexp(z, -s).to(torch.float8_e4m3fn).float()
    return torch.ldexp(c, s).view(rows, -1)[:, :d]


def _stats(x, layer, eps=1e-6):
    mean = x.mean(-1, keepdim=True) if layer else None
    c = x - mean if layer else x
    return mean, torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)


def _hat(x, stats):
    return (x if stats[0] is None else x - stats[0]) * stats[1]


def _affine(xhat, w, b):
    return xhat * w if b is None else xhat * w + b


def _norm_back(g, xhat, r, layer):
    out = g - xhat * (g * xhat).mean(-1, keepdim=True)
    return (out - g.mean(-1, keepdim=True) if layer else out) * r


def _norm_plain(s):
    c = s["case"]
    layer, dt, wt = c["kind"] == "layer", DTYPES[c["dtype"]], DTYPES[c["wdtype"]]
    f = {k: None if s[k] is None else s[k].detach().float() for k in ("x", "u", "gate", "w", "b", "scale", "w1", "b1")}
    x, u, z = f["x"], f["u"], f["gate"]
    act = (lambda t: torch.sigmoid(t)) if c["gate_kind"] == "sigmoid" else (lambda t: t)
    sc = 1.0 if f["scale"] is None else f["scale"]

    def parts(x, u, z, su):
        uhat = _hat(u, su)
        n = _affine(uhat, f["w"], f["b"])
        a = 1.0 if z is None else act(z)
        return uhat, n, a, x + sc * a * n

    su = _stats(u, layer)
    y = parts(x, u, z, su)[3]
    out = {"y": y.to(dt)}
    if c["next"]:
        sy = _stats(y, layer)
        out["h"] = _affine(_hat(y, sy), f["w1"], f["b1"]).to(dt)
    if not c["train"]:
        return out
    if c["checkpoint"]:
        flat = lambda t: _put_away(t.reshape(-1, c["d"]), c["checkpoint"]).view(t.shape)  # noqa: E731
        x, u, z = flat(x), flat(u), flat(z) if c["gate"] == "full" else z
    uhat, n, a, y = parts(x, u, z, su)
    t = s["dy"].float()
    rows = tuple(range(t.dim() - 1))
    if c["next"]:
        dh, yhat = s["dh"].float(), _hat(y, sy)
        t = t + _norm_back(dh * f["w1"], yhat, sy[1], layer)
        out["dw1"] = (dh * yhat).sum(rows).to(wt)
        if f["b1"] is not None:
            out["db1"] = dh.sum(rows).to(wt)
    out["dx"] = t.to(dt)
    dn = t * (sc * a)
    out["du"] = _norm_back(dn * f["w"], uhat, su[1], layer).to(dt)
    out["dw"] = (dn * uhat).sum(rows).to(wt)
    if f["b"] is not None:
        out["db"] = dn.sum(rows).to(wt)
    if f["scale"] is not None:
        out["dscale"] = (t * a * n).sum(rows).to(wt)
    if z is not None:
        dz = t * sc * n
        if c["gate_kind"] == "sigmoid":
            dz = dz * (a * (1 - a))
        out["dgate"] = (dz.sum(1, keepdim=True) if c["gate"] == "group" else dz).to(dt)
    return out


def _powers(a, n):
    """exp(a * n) for a <= 0 per head and whole n (in 64 bits: n can be large)."""
    return torch.exp(a.double() * n.double()).float()


def _chunked(q, k, v, a, state, lengths, c=128):
    """Chunked linear attention, [b, t, h, d] in 32 bits -> outputs and end state."""
    b, t, h, dk = q.shape
    dv, dev = v.shape[-1], q.device
    n = torch.full((b,), t, device=dev) if lengths is None else lengths.long()
    live = (torch.arange(t, device=dev)[None] < n[:, None])[..., None, None]
    k, v = k * live, v * live
    left = (n[:, None] - 1 - torch.arange(t, device=dev)[None]).clamp(min=0)           # tokens that follow, b t
    end = torch.einsum("bthk,bthv->bhkv", k * _powers(a[None, None], left[..., None])[..., None], v)
    if state is not None:
        end = end + _powers(a[None], n[:, None])[..., None, None] * state
    pad = -t % c
    m = (t + pad) // c
    cut = lambda x: torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).view(b, m, c, h, -1).permute(0, 3, 1, 2, 4)  # noqa: E731
    q, k, v = cut(q), cut(k), cut(v)                                                   # b h m c d
    i = torch.arange(c, device=dev)
    d = (i[:, None] - i[None]).clamp(min=0)
    mask = _powers(a[:, None, None], d[None]) * (i[:, None] >= i[None])                # h c c
    o = ((q @ k.transpose(-1, -2)) * mask[None, :, None]) @ v
    tail = _powers(a[:, None], (c - 1 - i)[None])[None, :, None, :, None]
    own_state = (k * tail).transpose(-1, -2) @ v                                       # b h m dk dv
    j = torch.arange(m, device=dev)
    gap = j[:, None] - 1 - j[None]
    carry = _powers(a[:, None, None], gap.clamp(min=0)[None] * c) * (gap >= 0)         # h m m
    start = torch.einsum("hij,bhjx->bhix", carry, own_state.reshape(b, h, m, -1)).view(b, h, m, dk, dv)
    if state is not None:
        start = start + _powers(a[:, None], j[None] * c)[None, :, :, None, None] * state[:, :, None]
    o = o + (q * _powers(a[:, None], (i + 1)[None])[None, :, None, :, None]) @ start
    o = o.permute(0, 2, 3, 1, 4).reshape(b, m * c, h, dv)[:, :t]
    return o * live, end


def _lin_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    x = {k: s[k].detach().float().requires_grad_(c["train"]) for k in s["leaves"]}
    scale = c["dk"] ** -0.5
    with torch.set_grad_enabled(c["train"]):
        o, end = _chunked(x["q"] * scale, x["k"], x["v"], s["log_decay"], x.get("state"), s["lengths"])
    out = {"o": o.detach().to(dt), "state": end.detach()}
    if c["train"]:
        g = torch.autograd.grad((o, end), list(x.values()), (s["do"].float(), s["dstate"]))
        out.update({"d" + k: gr.to(torch.float32 if k == "state" else dt) for k, gr in zip(x, g)})
        if "dstate" in out:
            out["dstate0"] = out.pop("dstate")
    return out


def _step_plain(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    st = s["state"]
    st.mul_(torch.exp(s["log_decay"])[None, :, None, None]).add_(k[..., :, None] * v[..., None, :])
    o = (q[..., :, None] * st).sum(-2) * s["case"]["dk"] ** -0.5
    return {"o": o.to(s["q"].dtype), "state": st}


def _act_plain(s):
    c = s["case"]
    x = s["x"].detach().float()
    back = _put_away(x[None], c["fmt"])[0]
    if c["kind"] == "gelu":
        y = 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
        slope = 0.5 * (1 + torch.erf(back * 0.5 ** 0.5)) + back * torch.exp(-0.5 * back * back) * (2 * math.pi) ** -0.5
    else:
        y = x * torch.sigmoid(x)
        g = torch.sigmoid(back)
        slope = g * (1 + back * (1 - g))
    return {"y": y.to(s["x"].dtype), "dx": (s["dy"].float() * slope).to(s["x"].dtype)}


def _store_plain(s):
    top = torch.finfo(s["x"].dtype).max
    return {"x": _put_away(s["x"].float()[None], s["case"]["fmt"])[0].clamp(-top, top).to(s["x"].dtype)}


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        plain = {"norm": _norm_plain, "lin": _lin_plain, "step": _step_plain, "act": _act_plain, "store": _store_plain}
        return plain[c["op"]](s)
    from customnetworklayers_b200 import blocknorm, ckpt8, linattn
    if c["op"] == "norm":
        with torch.set_grad_enabled(c["train"]):
            r = blocknorm.residual_norm(s["x"], s["u"], s["w"], s["b"], gate=s["gate"], gate_kind=c["gate_kind"],
                                        scale=s["scale"], next_weight=s["w1"], next_bias=s["b1"], kind=c["kind"],
                                        checkpoint=c["checkpoint"] or None)
        y, h = r if c["next"] else (r, None)
        out = {"y": y.detach()}
        if c["next"]:
            out["h"] = h.detach()
        if c["train"]:
            heads, gr = ((y, h), (s["dy"], s["dh"])) if c["next"] else ((y,), (s["dy"],))
            grads = torch.autograd.grad(heads, [s[k] for k in s["leaves"]], gr)
            out.update({"d" + k: x for k, x in zip(s["leaves"], grads)})
        return out
    if c["op"] == "lin":
        with torch.set_grad_enabled(c["train"]):
            o, end = linattn.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"])
        out = {"o": o.detach(), "state": end.detach()}
        if c["train"]:
            grads = torch.autograd.grad((o, end), [s[k] for k in s["leaves"]], (s["do"], s["dstate"]))
            out.update({"d" + k if k != "state" else "dstate0": x for k, x in zip(s["leaves"], grads)})
        return out
    if c["op"] == "step":
        o = linattn.step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return {"o": o, "state": s["state"]}
    if c["op"] == "act":
        y = ckpt8.activation(s["x"], kind=c["kind"], fmt=c["fmt"])
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx}
    return {"x": ckpt8.restore(ckpt8.store(s["x"], fmt=c["fmt"]))}


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    e, op = size[case["dtype"]], case["op"]
    if op == "norm":
        n, d, ew = case["rows"] * case["d"], case["d"], size[case["wdtype"]]
        gate = n if case["gate"] == "full" else case["groups"] * d if case["gate"] == "group" else 0
        vectors = 1 + case["scale"] + case["next"] + case["bias"] * (1 + case["next"])
        tensors = 3 + case["next"]                                     # x, u -> y, h
        if case["train"]:
            tensors += 3 + case["next"]                                # dy, dh -> dx, du
        both = 2 if case["train"] else 1
        return {"bytes": e * (tensors * n + both * gate) + ew * both * vectors * d, "flops": (40 if case["train"] else 15) * n}
    if op == "lin":
        tok = case["b"] * case["t"] * case["h"]
        st = 4 * case["b"] * case["h"] * case["dk"] * case["dv"]
        by = e * tok * (2 * case["dk"] + 2 * case["dv"]) + st * (1 + case["state"])
        fl = 4 * tok * case["dk"] * case["dv"]
        if case["train"]:
            by += e * tok * (2 * case["dk"] + 2 * case["dv"]) + st * (1 + case["state"])
            fl *= 3
        return {"bytes": by, "flops": fl}
    if op == "step":
        n = case["b"] * case["h"]
        return {"bytes": 8 * n * case["dk"] * case["dv"] + e * n * (2 * case["dk"] + 2 * case["dv"]), "flops": 5 * n * case["dk"] * case["dv"]}
    if op == "act":
        return {"bytes": 4 * e * case["n"], "flops": 40 * case["n"]}
    return {"bytes": 2 * e * case["n"], "flops": 4 * case["n"]}


# ---- 64 bits ----------------------------------------------------------------------------------------------------
def _blocks64(x, fmt):
    """The values the 8-bit form of x [rows, d] (64 bits) stands for, by arithmetic on the values alone."""
    d = x.shape[-1]
    out = torch.empty_like(x)
    for lo in range(0, d, BLOCK * 4096):
        z = x[:, lo:lo + BLOCK * 4096]
        w = z.shape[-1]
        full = torch.zeros(z.shape[0], -(-w // BLOCK) * BLOCK, dtype=x.dtype, device=x.device)
        full[:, :w] = z
        full = full.unflatten(-1, (-1, BLOCK))
        top = full.abs().amax(-1, keepdim=True)
        p = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        p = torch.where(torch.exp2(p) > top, p - 1, torch.where(torch.exp2(p + 1) <= top, p + 1, p))
        if fmt == "int8":
            unit = torch.exp2(p - 6)
            unit = torch.where(top / unit >= 127.5, 2 * unit, unit).clamp(min=2.0 ** -126)
            c = torch.round(full / unit)
        else:
            unit = torch.exp2(p - 8)
            unit = torch.where(top / unit > 448, 2 * unit, unit).clamp(min=2.0 ** -126)
            m = full / unit
            step = torch.exp2(torch.floor(torch.log2(m.abs().clamp(min=2.0 ** -6))) - 3)
            c = torch.round(m / step) * step
        out[:, lo:lo + BLOCK * 4096] = (c * unit).flatten(-2)[:, :w]
    return out


def _norm_exact(s):
    c = s["case"]
    d, layer = c["d"], c["kind"] == "layer"
    v = {k: None if s[k] is None else s[k].detach().double() for k in ("x", "u", "gate", "w", "b", "scale", "w1", "b1")}
    shape = v["x"].shape
    per = c["rows"] // c["groups"]
    x, u = v["x"].reshape(-1, d), v["u"].reshape(-1, d)
    z = None if v["gate"] is None else v["gate"].reshape(-1, d)
    if c["gate"] == "group":
        z = z.repeat_interleave(per, 0)
    zero, one = torch.zeros(d, dtype=torch.float64, device=x.device), torch.ones(d, dtype=torch.float64, device=x.device)
    b, b1, sc = (zero if v[k] is None else v[k] for k in ("b", "b1", "scale"))
    sc = one if v["scale"] is None else sc

    def center(t):
        return t.sum(1, keepdim=True) / d * (1.0 if layer else 0.0)

    def spread(t, m):
        return 1.0 / torch.sqrt(((t - m) ** 2).sum(1, keepdim=True) / d + 1e-6)

    def gate(z):
        if z is None:
            return torch.ones_like(x), torch.zeros_like(x)
        if c["gate_kind"] == "identity":
            return z, torch.ones_like(z)
        e = 1.0 / (1.0 + torch.exp(-z))
        return e, e - e * e

    mu = center(u)
    ru = spread(u, mu)
    y = x + sc * gate(z)[0] * ((u - mu) * ru * v["w"] + b)
    out = {"y": y}
    if c["next"]:
        my = center(y)
        ry = spread(y, my)
        out["h"] = (y - my) * ry * v["w1"] + b1
    if c["train"]:
        if c["checkpoint"]:
            x, u = _blocks64(x, c["checkpoint"]), _blocks64(u, c["checkpoint"])
            z = _blocks64(z, c["checkpoint"]) if c["gate"] == "full" else z
        a, da = gate(z)
        uh = (u - mu) * ru
        n = uh * v["w"] + b
        t = s["dy"].double().reshape(-1, d).clone()

        def back(g, hat, r):
            return r * (g - hat * ((g * hat).sum(1, keepdim=True) / d) - (g.sum(1, keepdim=True) / d if layer else 0.0))

        if c["next"]:
            dh = s["dh"].double().reshape(-1, d)
            yh = (x + sc * a * n - my) * ry
            t += back(dh * v["w1"], yh, ry)
            out["dw1"] = torch.einsum("rd,rd->d", dh, yh)
            if v["b1"] is not None:
                out["db1"] = dh.sum(0)
        out["dx"] = t
        out["du"] = back(t * sc * a * v["w"], uh, ru)
        out["dw"] = torch.einsum("rd,rd,rd->d", t, a, uh) * sc
        if v["b"] is not None:
            out["db"] = torch.einsum("rd,rd->d", t, a) * sc
        if v["scale"] is not None:
            out["dscale"] = torch.einsum("rd,rd,rd->d", t, a, n)
        if z is not None:
            dz = t * sc * n * da
            out["dgate"] = dz.view(c["groups"], per, d).sum(1).view(c["groups"], 1, d) if c["gate"] == "group" else dz
    return {k: t.reshape(shape) if t.numel() == c["rows"] * d and k not in ("dgate",) else t for k, t in out.items()}


def _lin_exact(s):
    """The recurrence, 64 tokens at a time, with its gradient by differentiation of that loop."""
    c = s["case"]
    dev, t, step = s["q"].device, c["t"], 64 if c["t"] <= 16384 else 512
    x = {k: s[k].detach().double().requires_grad_(c["train"]) for k in s["leaves"]}
    lam = torch.exp(s["log_decay"].double())
    n = torch.full((c["b"],), t, device=dev) if s["lengths"] is None else s["lengths"].long()
    S = x["state"] if s["state"] is not None else torch.zeros(c["b"], c["h"], c["dk"], c["dv"], dtype=torch.float64, device=dev)
    outs = []
    with torch.set_grad_enabled(c["train"]):
        for lo in range(0, t, step):
            hi = min(t, lo + step)
            m = hi - lo
            on = (torch.arange(lo, hi, device=dev)[None] < n[:, None]).double()          # b m
            count = on.sum(1)
            q, k, v = (x[w][:, lo:hi].transpose(1, 2) for w in ("q", "k", "v"))          # b h m d
            i = torch.arange(m, device=dev, dtype=torch.float64)
            dist = (i[:, None] - i[None]).clamp(min=0)
            w = torch.tril(lam[:, None, None] ** dist)                                    # h m m
            sc = torch.einsum("bhik,bhjk->bhij", q, k) * w * on[:, None, None] * on[:, None, :, None]
            o = sc @ v + (lam[:, None] ** (i + 1))[None, :, :, None] * (q @ S) * on[:, None, :, None]
            outs.append(o.transpose(1, 2) * c["dk"] ** -0.5)
            behind = (count[:, None] - 1 - i[None]).clamp(min=0)                          # b m
            wt = lam[None, :, None] ** behind[:, None] * on[:, None]                      # b h m
            S = (lam[None] ** count[:, None])[..., None, None] * S + torch.einsum("bhm,bhmk,bhmv->bhkv", wt, k, v)
        o = torch.cat(outs, 1)
    out = {"o": o.detach(), "state": S.detach()}
    if c["train"]:
        g = torch.autograd.grad((o, S), list(x.values()), (s["do"].double(), s["dstate"].double()))
        out.update({"d" + k if k != "state" else "dstate0": gr for k, gr in zip(x, g)})
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _norm_exact(s)
    if op == "lin":
        return _lin_exact(s)
    if op == "step":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        st = s["state"].double() * torch.exp(s["log_decay"].double()).view(1, -1, 1, 1) + torch.einsum("bhk,bhv->bhkv", k, v)
        return {"o": torch.einsum("bhk,bhkv->bhv", q, st) / math.sqrt(case["dk"]), "state": st}
    x = s["x"].detach().double()
    back = _blocks64(x[None], case["fmt"])[0]
    if op == "store":
        return {"x": back}
    dy = s["dy"].double()
    if case["kind"] == "gelu":
        y = x * (0.5 * torch.erfc(-x / math.sqrt(2.0)))
        slope = 0.5 * torch.erfc(-back / math.sqrt(2.0)) + back * torch.exp(-back * back / 2) / math.sqrt(2 * math.pi)
    else:
        y = x / (1 + torch.exp(-x))
        e = torch.exp(-back.abs())
        g = torch.where(back >= 0, 1 / (1 + e), e / (1 + e))
        slope = g + back * e / (1 + e) ** 2
    return {"y": y, "dx": dy * slope}
