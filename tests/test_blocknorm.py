"""Norms around a gated residual block against 64 bits: values, gradients by formula, by differentiation and by differences,
8-bit checkpoints, gates shared by groups of rows, column sums, refusals."""
import itertools

import pytest
import torch

from customnetworklayers_b200 import _lib, blocknorm
from tests.operators_ref import HALF, TINY, assert_within, block_norm, block_norm_backward, norm, put_away_rows

NAMES = ("x", "u", "gate", "scale", "weight", "bias", "next_weight", "next_bias")


def make(shape, dtype=torch.float32, wdtype=None, gate="full", bias=True, scale=True, nxt=True, seed=0, post=True):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    wdtype = dtype if wdtype is None else wdtype
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = {"x": (r(*shape) * torch.exp(0.7 * r(d)) + 0.3).to(dtype), "u": (0.8 * r(*shape) + 0.1).to(dtype) if post else None,
         "gate": None if gate is None or not post else r(*(shape if gate == "full" else gate)).to(dtype),
         "scale": (0.4 + 0.1 * r(d)).to(wdtype) if scale and post else None,
         "weight": (1 + 0.1 * r(d)).to(wdtype) if post else None, "bias": (0.1 * r(d)).to(wdtype) if bias and post else None,
         "next_weight": (1 + 0.1 * r(d)).to(wdtype) if nxt else None, "next_bias": (0.1 * r(d)).to(wdtype) if nxt and bias else None}
    up = {"dy": r(*shape).to(dtype) if post else None, "dh": r(*shape).to(dtype) if nxt else None}
    return t, up


def run(t, up, **kw):
    dev = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    if t["u"] is None:
        h = blocknorm.pre_norm(dev["x"], dev["next_weight"], dev["next_bias"], kind=kw.get("kind", "rms"), checkpoint=kw.get("checkpoint"))
        outs = {"h": h}
    else:
        r = blocknorm.residual_norm(dev["x"], dev["u"], dev["weight"], dev["bias"], gate=dev["gate"], scale=dev["scale"],
                                    next_weight=dev["next_weight"], next_bias=dev["next_bias"], **kw)
        outs = dict(zip(("y", "h"), r)) if isinstance(r, tuple) else {"y": r}
    leaves = [k for k in NAMES if dev[k] is not None]
    heads = [(outs[k], up["d" + k].cuda()) for k in outs]
    g = torch.autograd.grad([o for o, _ in heads], [dev[k] for k in leaves], [d for _, d in heads])
    return outs, dict(zip(leaves, g))


def check(t, up, kind="rms", gate_kind="sigmoid", checkpoint=None):
    """Bounds: half a step of the type for the one rounding at the end; in 32 bits every value passes through sums over d
    (a tree of at most 8 + 10 levels), a reciprocal root and some ten products, under 64 roundings of 2^-24, each relative
    to the largest intermediate of its row (64 * 2^-24 = 2^-18); column sums add the rows a thread walks over (at most
    all of them here) and the join, relative to the sum of the terms' magnitudes.

    The largest intermediate behind y = x + m n is max|x| + max|m n| <= 2 max|x| + max|y|, which y itself can be far below
    (x = -m n in rows of one channel): y is off by e = 2^-18 (2 max|x| + max|y|), and y^ = (y - mu) r_y by e r_y, i.e. by 2^-18
    times cond = 1 + (2 max|x| + max|y|) r_y, which is a small number unless the row cancels.  What the pre norm's gradient
    r_y (g - y^ mean(g y^)) carries of it is off by r_y max|g| times that, twice where y^ enters twice: cond^2."""
    outs, grads = run(t, up, kind=kind, checkpoint=checkpoint, **({} if t["u"] is None else {"gate_kind": gate_kind}))
    layer, sig = kind == "layer", gate_kind == "sigmoid"
    f = {k: None if v is None else v.double() for k, v in t.items()}
    dtype = t["x"].dtype
    args = [f[k] for k in NAMES]
    y, h = block_norm(f["x"], f["u"], f["gate"], f["scale"], f["weight"], f["bias"], f["next_weight"], f["next_bias"], layer, sig)
    row = lambda v: v.abs().amax(-1, keepdim=True)  # noqa: E731
    x, u, gate = f["x"], f["u"], f["gate"]
    stats = [None] * 4
    behind = 2 * row(x) + row(y)
    if h is not None:
        stats[2], stats[3] = norm(y, f["next_weight"], f["next_bias"], layer)[:2]
    cond = 1 + (0 if h is None else behind * stats[3])
    if "y" in outs:
        assert outs["y"].dtype == dtype
        assert_within(outs["y"], y, HALF[dtype] * y.abs() + 2.0 ** -18 * behind + TINY[dtype], "y")
    if "h" in outs:
        assert_within(outs["h"], h, HALF[dtype] * h.abs() + 2.0 ** -18 * (row(h) + cond * row(f["next_weight"])) + TINY[dtype], "h")
    if u is not None:
        stats[0], stats[1] = norm(u, f["weight"], f["bias"], layer)[:2]
    if checkpoint:
        x = put_away_rows(x, checkpoint)
        u = None if u is None else put_away_rows(u, checkpoint)
        gate = put_away_rows(gate, checkpoint) if gate is not None and gate.shape == x.shape else gate
    dy, dh = (None if up[k] is None else up[k].double() for k in ("dy", "dh"))
    full = None if gate is None else gate.expand_as(x)
    ref = block_norm_backward(x, u, full, f["scale"], f["weight"], f["bias"], f["next_weight"], f["next_bias"], layer, sig, stats, dy, dh)
    if not checkpoint:                                       # the formulas against differentiation of the forward form
        leaves = [a.clone().requires_grad_(True) for a in args if a is not None]
        it = iter(leaves)
        full_args = [None if a is None else next(it) for a in args]
        yy, hh = block_norm(*full_args, layer, sig)
        heads, gr = zip(*[(o, d) for o, d in ((yy, dy), (hh, dh)) if o is not None and d is not None])
        auto = torch.autograd.grad(heads, leaves, gr)
        for k, a in zip([n for n, a in zip(NAMES, args) if a is not None], auto):
            r = ref[k]
            if k == "gate" and gate.shape != x.shape:
                r = r.sum_to_size(gate.shape)
            assert torch.allclose(r, a, rtol=1e-9, atol=1e-9), k
    rows = x.numel() // x.shape[-1]
    # what a gradient of up to 5 (the largest of some thousand normal numbers) becomes in one row
    size = 1 + (0 if h is None else 5 * row(f["next_weight"]) * stats[3] * cond * cond)
    for k, g in grads.items():
        r = ref[k]
        if k in ("x", "u") or (k == "gate" and gate.shape == x.shape):
            scale = row(r) + row(ref["x"]) * (1 if k == "x" else 4)
            if k == "u":
                scale = scale * (1 + stats[1])
            assert g.dtype == dtype and g.shape == t[k].shape
            assert_within(g, r, HALF[dtype] * r.abs() + 2.0 ** -18 * scale + 2.0 ** -18 * size + TINY[dtype], k)
        else:
            terms = {"next_weight": lambda: dh * ((y if not checkpoint else y) - (stats[2] if layer else 0)) * stats[3],
                     "next_bias": lambda: dh}.get(k, lambda: ref["x"] * 4)()
            own = 4 * size * torch.ones_like(x) if k not in ("next_weight", "next_bias") else dh.abs() * cond      # each term's own error, in 2^-18
            to = gate.shape if k == "gate" else r.shape
            r = r.sum_to_size(to)
            mag, own = terms.abs().sum_to_size(to), own.sum_to_size(to)
            assert g.shape == t[k].shape and g.dtype == t[k].dtype
            assert_within(g, r, HALF[g.dtype] * r.abs() + (64 + rows) * 2.0 ** -24 * mag + 2.0 ** -18 * own + TINY[g.dtype], k)


# ---- refusals (no GPU) -------------------------------------------------------------------------------------------
def test_refusals_without_a_gpu():
    lib = _lib.load()
    fwd = lambda **k: lib.cnl_blocknorm_forward(*[k.get(n, 16) for n in ("x", "u", "gate", "scale", "w", "b", "w1", "b1", "y", "h", "st", "co", "sc")],  # noqa: E731
                                                k.get("rows", 4), k.get("d", 8), k.get("groups", 1), k.get("mode", 1), 1, 0, 1e-6,
                                                k.get("dtype", 0), k.get("wdtype", 0), k.get("fmt", 0), None)
    assert fwd(rows=-1) == 2 and fwd(d=0) == 2 and fwd(d=8193) == 2 and fwd(groups=3, mode=2) == 2 and fwd(groups=0) == 2
    assert fwd(dtype=5) == 8 and fwd(dtype=1, wdtype=2) == 8 and fwd(fmt=3) == 8 and fwd(mode=4) == 8
    assert fwd(x=None) == 7 and fwd(w=None) == 7 and fwd(gate=None) == 7 and fwd(h=None) == 7 and fwd(fmt=1, co=None) == 7
    assert fwd(rows=0) == 0
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        blocknorm.pre_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="rms"):
        blocknorm.pre_norm(x, torch.ones(8), kind="batch")
    with pytest.raises(RuntimeError, match="int8"):
        blocknorm.pre_norm(x, torch.ones(8), checkpoint="int3")
    with pytest.raises(RuntimeError, match="gate_kind"):
        blocknorm.residual_norm(x, x, torch.ones(8), gate_kind="tanh")


def test_which_rows_share_a_gate():
    x = torch.zeros(4, 6, 10, 8)
    mode = lambda *s: blocknorm._gate_mode(x, torch.zeros(*s))  # noqa: E731
    assert mode(4, 6, 10, 8) == (1, 1) and mode(8) == (2, 1) and mode(4, 1, 1, 8) == (2, 4) and mode(4, 6, 1, 8) == (2, 24)
    assert mode(1, 1, 1, 8) == (2, 1) and blocknorm._gate_mode(x, None) == (0, 1)
    for bad in ((1, 6, 10, 8), (4, 1, 10, 8), (4, 6, 10, 1), (2, 4, 6, 10, 8), (6, 8), (3, 1, 1, 8)):
        with pytest.raises(RuntimeError):
            mode(*bad)


# ---- values and gradients ----------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("d", [1, 2, 7, 8, 24, 32, 40, 100, 128, 150, 256, 264, 520, 1000, 1024])
def test_every_width(d, kind, dtype):
    t, up = make((37, d), dtype, seed=d)
    check(t, up, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [2048, 2056, 2500, 4096, 6000, 8191, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_rows(d, dtype):
    t, up = make((5, d), dtype, seed=d)
    check(t, up, "layer")


@pytest.mark.gpu
@pytest.mark.parametrize("kind,gate,gate_kind,bias,scale,nxt", list(itertools.product(
    ["rms", "layer"], ["full", (3, 1, 1, 72), (72,), None], ["sigmoid", "identity"], [True, False], [True, False], [True, False])))
def test_every_combination(kind, gate, gate_kind, bias, scale, nxt):
    t, up = make((3, 5, 7, 72), torch.float32, gate=gate, bias=bias, scale=scale, nxt=nxt, seed=5)
    check(t, up, kind, gate_kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("gate", ["full", (6, 1, 96), (1, 1, 96)])
def test_types_of_parameters(dtype, wdtype, gate):
    t, up = make((6, 50, 96), dtype, wdtype, gate=gate, seed=9)
    check(t, up)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,gate", [((11, 24), "full"), ((4, 9, 104), (4, 1, 104)), ((13, 150), "full"), ((7, 33), None), ((3, 520), "full"),
                                        ((2, 4104), "full"), ((5, 5), "full")])
def test_backward_from_8_bits(shape, gate, dtype, fmt):
    t, up = make(shape, dtype, gate=gate, seed=shape[-1])
    check(t, up, "layer", checkpoint=fmt)
    t, up = make(shape, dtype, gate=gate, nxt=False, seed=shape[-1] + 1)
    check(t, up, "rms", checkpoint=fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", [(1, 64), (200, 48), (3, 4, 5, 130)])
def test_norm_alone(shape, kind, fmt):
    t, up = make(shape, torch.bfloat16, torch.float32, post=False, seed=2)
    check(t, up, kind, checkpoint=fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,gate", [(1, "full"), (3001, "full"), (4096, (4096, 32)), (3000, (1500, 1, 32))])
def test_row_counts(rows, gate):
    shape = (rows, 32) if gate == "full" or len(gate) == 2 else (gate[0], rows // gate[0], 32)
    t, up = make(shape, torch.float32, gate=gate, seed=rows)
    check(t, up)


@pytest.mark.gpu
def test_more_groups_than_a_grid_is_high():
    n, d = 70001, 8
    t, up = make((n, 2, d), torch.float32, gate=(n, 1, d), seed=1)
    check(t, up)


@pytest.mark.gpu
def test_gradient_against_differences():
    t, up = make((9, 40), torch.float32, seed=3)
    t = {k: v.double().float() for k, v in t.items()}
    _, grads = run(t, up)
    g = torch.Generator().manual_seed(8)

    def loss(s):
        dev = {k: v.cuda() for k, v in s.items()}
        y, h = blocknorm.residual_norm(dev["x"], dev["u"], dev["weight"], dev["bias"], gate=dev["gate"], scale=dev["scale"],
                                       next_weight=dev["next_weight"], next_bias=dev["next_bias"])
        return float((y.cpu().double() * up["dy"].double()).sum() + (h.cpu().double() * up["dh"].double()).sum())

    for k in t:
        way = torch.randn(t[k].shape, generator=g)
        e = 2.0 ** -6
        d = (loss({**t, k: t[k] + e * way}) - loss({**t, k: t[k] - e * way})) / (2 * e)
        want = float((grads[k].cpu().double() * way.double()).sum())
        # 720 outputs of size about 3 off by 2^-21 each, over 2 e: 1e-3; the difference itself e^2 / 6 of a third derivative
        # (under 60 per row for nine rows of unit directions)
        assert abs(d - want) <= 1e-3 + e * e * 90 + 1e-3 * abs(want), (k, d, want)


@pytest.mark.gpu
def test_only_one_output_is_used_and_not_all_gradients_are_wanted():
    t, up = make((21, 64), torch.float32, seed=4)
    dev = {k: v.cuda() for k, v in t.items()}
    dev["u"].requires_grad_(True)
    dev["next_weight"].requires_grad_(True)
    f = {k: v.double() for k, v in t.items()}

    def pair():
        return blocknorm.residual_norm(dev["x"], dev["u"], dev["weight"], dev["bias"], gate=dev["gate"], scale=dev["scale"],
                                       next_weight=dev["next_weight"], next_bias=dev["next_bias"])

    for which in (0, 1):
        got = torch.autograd.grad(pair()[which], (dev["u"], dev["next_weight"]), up["dy"].cuda(), allow_unused=True, materialize_grads=True)
        u, w1 = f["u"].clone().requires_grad_(True), f["next_weight"].clone().requires_grad_(True)
        out = block_norm(f["x"], u, f["gate"], f["scale"], f["weight"], f["bias"], w1, f["next_bias"], False, True)[which]
        ref = torch.autograd.grad(out, (u, w1), up["dy"].double(), allow_unused=True, materialize_grads=True)
        for a, b in zip(got, ref):
            assert_within(a, b, 2.0 ** -17 * b.abs().max() + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,gate", [(0, "full"), (0, None)])
def test_no_rows(rows, gate):
    t, up = make((rows, 16), torch.float32, gate=gate)
    outs, grads = run(t, up)
    assert outs["y"].shape == (0, 16)
    for k in ("weight", "bias", "scale", "next_weight", "next_bias"):
        assert torch.count_nonzero(grads[k]) == 0 and grads[k].shape == (16,)


@pytest.mark.gpu
def test_views_strides_and_odd_starts():
    t, up = make((30, 64), torch.bfloat16, seed=6)
    ref, gref = run(t, up)
    wide = torch.randn(30, 200).to(torch.bfloat16).cuda()
    wide[:, 3:67] = t["u"].cuda()
    odd = torch.empty(30 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(30, 64).copy_(t["x"].cuda())
    dev = {k: v.cuda() for k, v in t.items()}
    with torch.no_grad():
        y, h = blocknorm.residual_norm(odd, wide[:, 3:67], dev["weight"], dev["bias"], gate=dev["gate"].t().contiguous().t(), scale=dev["scale"],
                                       next_weight=dev["next_weight"], next_bias=dev["next_bias"])
    f = {k: v.double() for k, v in t.items()}
    yy, hh = block_norm(*[f[k] for k in NAMES], False, True)
    for a, b in ((y, yy), (h, hh)):
        assert_within(a, b, HALF[torch.bfloat16] * b.abs() + 2.0 ** -18 * (b.abs().amax(-1, keepdim=True) + 1))


@pytest.mark.gpu
def test_not_finite_rows_stay_in_their_rows():
    t, up = make((8, 40), torch.float32, gate="full", seed=7)
    t["u"][2, 5] = float("nan")
    t["x"][4, 1] = float("inf")
    outs, grads = run(t, up)
    bad = torch.tensor([2, 4])
    good = torch.tensor([0, 1, 3, 5, 6, 7])
    assert torch.isfinite(outs["h"][good]).all() and torch.isfinite(grads["u"][good]).all()
    assert torch.isnan(outs["y"][2]).all() and not torch.isfinite(outs["h"][bad]).all()
    t2, _ = make((8, 40), torch.float32, gate="full", seed=7)
    outs2, _ = run(t2, up)
    assert torch.equal(outs["h"][good], outs2["h"][good])


@pytest.mark.gpu
def test_same_bits_every_call_and_on_another_stream():
    t, up = make((5000, 136), torch.bfloat16, torch.float32, seed=11)
    _, a = run(t, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, b = run(t, up)
    side.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
def test_elements_past_32_bits():
    d, rows = 8192, 2 ** 18 + 3                           # 2^31 elements and three rows
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(5, d, device="cuda").bfloat16()
    x[-5:] = tail
    w = torch.linspace(0.5, 1.5, d, device="cuda").bfloat16()
    with torch.no_grad():
        assert torch.equal(blocknorm.pre_norm(x, w)[-5:], blocknorm.pre_norm(tail, w))
        x = x.view(-1, 4096)
        assert torch.equal(blocknorm.pre_norm(x, w[:4096].clone())[-10:], blocknorm.pre_norm(tail.view(-1, 4096), w[:4096].clone()))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_forward_and_backward_in_a_graph(fmt):
    t, up = make((300, 72), torch.bfloat16, seed=12)
    dev = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    up = {k: v.cuda() for k, v in up.items()}

    def once():
        y, h = blocknorm.residual_norm(dev["x"], dev["u"], dev["weight"], dev["bias"], gate=dev["gate"], scale=dev["scale"],
                                       next_weight=dev["next_weight"], next_bias=dev["next_bias"], checkpoint=fmt)
        g = torch.autograd.grad((y, h), list(dev.values()), (up["dy"], up["dh"]))
        return [y.detach(), h.detach(), *g]               # no eager graph of these leaves lives on while a capture runs

    want = [o.clone() for o in once()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    keep = up["dh"].clone()
    up["dh"].zero_()
    graph.replay()
    assert not torch.equal(got[2], want[2])
    up["dh"].copy_(keep)
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x = torch.randn(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for call in (lambda: blocknorm.residual_norm(x, x.half(), w), lambda: blocknorm.residual_norm(x, x[:2], w),
                 lambda: blocknorm.residual_norm(x, x, w[:8].clone()), lambda: blocknorm.residual_norm(x, x, w.half()),
                 lambda: blocknorm.residual_norm(x, x, w, next_bias=w), lambda: blocknorm.residual_norm(x, x, w, gate=x[:2]),
                 lambda: blocknorm.pre_norm(torch.randn(2, 8200, device="cuda"), torch.ones(8200, device="cuda")),
                 lambda: blocknorm.pre_norm(x, None), lambda: blocknorm.residual_norm(x, x, None),
                 lambda: blocknorm.residual_norm(x, x, None, next_weight=w), lambda: blocknorm.pre_norm(x.double(), w.double())):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("shape,gate", [((0, 5, 16), (0, 1, 16)), ((0, 5, 16), (1, 1, 16)), ((3, 0, 16), (3, 1, 16)), ((0, 4, 6, 16), (0, 1, 1, 16)),
                                        ((0, 4, 6, 16), (0, 4, 1, 16)), ((3, 0, 16), (16,))])
def test_no_rows_with_a_gate_for_each_image(shape, gate, fmt):
    t, up = make(shape, torch.float32, gate=gate)
    outs, grads = run(t, up, checkpoint=fmt)
    assert outs["y"].shape == outs["h"].shape == shape and grads["x"].shape == grads["u"].shape == shape
    assert grads["gate"].shape == gate and torch.count_nonzero(grads["gate"]) == 0
    for k in ("weight", "bias", "scale", "next_weight", "next_bias"):
        assert torch.count_nonzero(grads[k]) == 0 and grads[k].shape == (16,)


def test_gates_of_no_images():
    mode = lambda x, g: blocknorm._gate_mode(torch.zeros(*x), torch.zeros(*g))  # noqa: E731
    assert mode((0, 5, 8), (0, 1, 8)) == (0, 1) and mode((0, 5, 8), (0, 5, 8)) == (1, 1) and mode((0, 5, 8), (1, 1, 8)) == (2, 1)
    assert mode((3, 0, 8), (3, 1, 8)) == (2, 3)
    for x, g in (((0, 5, 8), (2, 1, 8)), ((2, 5, 8), (0, 1, 8)), ((0, 5, 8), (0, 2, 8))):
        with pytest.raises(RuntimeError):
            mode(x, g)
