"""Linear attention with a decay for each head against the full T x T form in 64 bits: chunks, segments, ragged batches, carried
states, single tokens, gradients by differentiation and by differences, refusals."""
import pytest
import torch

from customnetworklayers_b200 import _lib, linattn
from tests.operators_ref import HALF, TINY, assert_within, attention

DT = [torch.float32, torch.float16, torch.bfloat16]


def make(b, t, h, dk, dv, dtype, seed=0, state=True, decay=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = {"q": r(b, t, h, dk).to(dtype), "k": (r(b, t, h, dk) * dk ** -0.5).to(dtype), "v": r(b, t, h, dv).to(dtype),
         "state": r(b, h, dk, dv).float() if state else None}
    if decay is None:
        decay = -torch.exp2(-torch.linspace(0.0, 9.0, h))
    return x, decay, r(b, t, h, dv).to(dtype), r(b, h, dk, dv).float()


def bounds(x, decay, do, ds, lengths, scale, dtype):
    """Per output, the sum of the magnitudes of its terms: the same sweeps on absolute values.  A term is a product of exact
    inputs, rounded to the type at most twice on its way (the chunk's weight, or the carried state) where the inputs are
    16-bit, and takes part in fewer than 256 additions in 32 bits (a chunk, the head size, the segments)."""
    a = {k: None if v is None else v.double().abs().requires_grad_(True) for k, v in x.items()}
    o, end = attention(a["q"], a["k"], a["v"], decay.double(), a["state"], lengths, abs(scale))
    leaves = [v for v in a.values() if v is not None]
    g = torch.autograd.grad((o, end), leaves, (do.double().abs(), ds.double().abs()))
    mags = [o, end, *g]
    # powers of the decay: the argument a n is rounded once, 2^-24 of a value whose weight exp(a n) is at most e^-(a n)
    fp32 = 512 * 2.0 ** -24
    per = 2 * HALF[dtype] if dtype != torch.float32 else 0.0
    return [m.detach() * (per + fp32) for m in mags]


def check(b, t, h, dk, dv, dtype, lengths=None, state=True, decay=None, scale=None, seed=0, grad_state=True):
    x, decay, do, ds = make(b, t, h, dk, dv, dtype, seed, state, decay)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    sc = dk ** -0.5 if scale is None else scale
    if not grad_state:
        ds = torch.zeros_like(ds)
    dev = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in x.items()}
    o, end = linattn.linear_attention(dev["q"], dev["k"], dev["v"], decay.cuda(), state=dev["state"],
                                      lengths=None if n is None else n.cuda(), scale=scale)
    leaves = [k for k in x if x[k] is not None]
    heads, gr = ((o, end), (do.cuda(), ds.cuda())) if grad_state else ((o,), (do.cuda(),))
    grads = torch.autograd.grad(heads, [dev[k] for k in leaves], gr)
    ref = {k: None if v is None else v.double().requires_grad_(True) for k, v in x.items()}
    ro, rend = attention(ref["q"], ref["k"], ref["v"], decay.double(), ref["state"], n, sc)
    rg = torch.autograd.grad((ro, rend), [ref[k] for k in leaves], (do.double(), ds.double()))
    mags = bounds(x, decay, do, ds, n, sc, dtype)
    fp32 = lambda m: m / (2 * HALF[dtype] + 512 * 2.0 ** -24) * 512 * 2.0 ** -24 if dtype != torch.float32 else m  # noqa: E731
    assert o.dtype == dtype and end.dtype == torch.float32
    assert_within(o, ro, HALF[dtype] * ro.abs() + mags[0] + TINY[dtype], "out")
    assert_within(end, rend, fp32(mags[1]) + 1e-30, "end state")          # the state itself is never rounded to 16 bits
    for k, g, r, m in zip(leaves, grads, rg, mags[2:]):
        assert g.dtype == x[k].dtype
        assert_within(g, r, HALF[g.dtype] * r.abs() + (fp32(m) if k == "state" else m) + TINY[g.dtype], "gradient of " + k)
    if n is not None:
        for i, m in enumerate(lengths):
            assert torch.count_nonzero(o[i, max(m, 0):]) == 0
            for k, g in zip(leaves, grads):
                if k != "state":
                    assert torch.count_nonzero(g[i, max(m, 0):]) == 0


# ---- refusals (no GPU) -------------------------------------------------------------------------------------------
def test_refusals_without_a_gpu():
    import ctypes
    lib = _lib.load()
    st = (ctypes.c_longlong * 12)()
    fwd = lambda b=1, t=4, h=2, dk=8, dv=8, dtype=0, q=16: lib.cnl_linattn_forward(q, 16, 16, st, 16, None, None, 16, 16, None, b, t, h, dk, dv, 1.0, dtype, None)  # noqa: E731
    assert fwd(b=-1) == 2 and fwd(t=-1) == 2 and fwd(h=0) == 2 and fwd(dk=0) == 2 and fwd(dk=129) == 2 and fwd(dv=200) == 2
    assert fwd(dtype=4) == 8 and fwd(q=None) == 7 and fwd(b=0) == 0 and fwd(b=1 << 20, h=64) == 2
    assert lib.cnl_linattn_step(16, 16, 16, st, 16, None, 16, 1, 2, 8, 8, 1.0, 0, None) == 7
    x = torch.zeros(1, 3, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        linattn.linear_attention(x, x, x, torch.zeros(2))
    with pytest.raises(RuntimeError, match="state"):
        linattn.step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(2), None)
    with pytest.raises(ValueError):
        linattn.LinearAttention(10, 3)


def test_the_full_form_is_the_recurrence():
    x, decay, _, _ = make(2, 9, 3, 4, 5, torch.float32, seed=1)
    f = {k: v.double() for k, v in x.items()}
    n = torch.tensor([9, 4], dtype=torch.int32)
    o, end = attention(f["q"], f["k"], f["v"], decay.double(), f["state"], n, 0.7)
    s = f["state"].clone()
    for t in range(9):
        live = (t < n).double().view(2, 1, 1, 1)
        s = live * (torch.exp(decay.double()).view(1, 3, 1, 1) * s + f["k"][:, t, :, :, None] * f["v"][:, t, :, None]) + (1 - live) * s
        want = 0.7 * torch.einsum("bhd,bhde->bhe", f["q"][:, t], s) * live[..., 0]
        assert torch.allclose(o[:, t], want, rtol=1e-12, atol=1e-12)
    assert torch.allclose(end, s, rtol=1e-12, atol=1e-12)


# ---- values and gradients ----------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("t", [1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_every_length(t, dtype):
    check(2, t, 2, 32, 32, dtype, seed=t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (8, 8), (16, 64), (40, 56), (64, 64), (97, 33), (128, 128), (128, 8), (24, 120), (72, 100)])
def test_every_head_size(dk, dv, dtype):
    check(1, 150, 3, dk, dv, dtype, seed=dk + dv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("t", [257, 700, 1300, 2100])
def test_segments(t, dtype):
    assert _lib.load().cnl_linattn_segments(1, t, 2, 32, 64, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]) > 1
    check(1, t, 2, 32, 64, dtype, seed=t)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(64, 64), (40, 56), (128, 128), (64, 128), (128, 64), (72, 40), (48, 104)])
@pytest.mark.parametrize("t", [128, 129, 255, 256, 257, 640, 1001])
def test_chunks_of_wide_heads(t, dk, dv):
    """Sizes of the kernel with 128-token chunks: whole and cut chunks, one and several segments, both directions."""
    check(1, t, 3, dk, dv, torch.bfloat16, seed=t + dk, state=t % 2 == 0)
    check(2, t, 2, dk, dv, torch.bfloat16, lengths=[t - 1, max(t - 130, 0)], seed=t + dv)
    assert _lib.load().cnl_linattn_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DT)
def test_so_many_heads_that_no_sequence_is_cut(d, dtype):
    codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    assert _lib.load().cnl_linattn_segments(10, 300, 74, d, d, codes[dtype]) == 1
    decay = -torch.exp2(-torch.linspace(0.0, 9.0, 74))
    check(10, 300, 74, d, d, dtype, decay=decay, seed=d, lengths=[300, 299, 0, 1, 128, 129, 256, 257, 127, 300])


@pytest.mark.gpu
@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (40, 72)])
def test_segments_of_many_chunks(dk, dv, state):
    # so many heads that a segment is five or six chunks long, the last of them cut; three sequences, each in many copies
    t, h, dtype = 1300, 2, torch.bfloat16
    x, _, do, ds = make(3, t, h, dk, dv, dtype, seed=dk + dv, state=state)
    decay, n, sc = torch.tensor([-2.0 ** -9, -0.02]), torch.tensor([1300, 1111, 770], dtype=torch.int32), dk ** -0.5
    copy = torch.arange(37) % 3
    dev = {k: None if v is None else v[copy].cuda().requires_grad_(True) for k, v in x.items()}
    o, end = linattn.linear_attention(dev["q"], dev["k"], dev["v"], decay.cuda(), state=dev["state"], lengths=n[copy].cuda())
    leaves = [k for k in x if x[k] is not None]
    got = (o, end, *torch.autograd.grad((o, end), [dev[k] for k in leaves], (do[copy].cuda(), ds[copy].cuda())))
    ref = {k: None if v is None else v.double().requires_grad_(True) for k, v in x.items()}
    ro, rend = attention(ref["q"], ref["k"], ref["v"], decay.double(), ref["state"], n, sc)
    exact = (ro, rend, *torch.autograd.grad((ro, rend), [ref[k] for k in leaves], (do.double(), ds.double())))
    mags = bounds(x, decay, do, ds, n, sc, dtype)
    for name, g, r, m in zip(["out", "end state"] + leaves, got, exact, mags):
        assert torch.equal(g, g[:3][copy])                            # copies, wherever they ran
        in_fp32 = name in ("end state", "state")                      # never rounded to 16 bits
        bound = m / (2 * HALF[dtype] + 512 * 2.0 ** -24) * 512 * 2.0 ** -24 + 1e-30 if in_fp32 else HALF[dtype] * r.abs() + m + TINY[dtype]
        assert_within(g[:3], r, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lengths", [[0, 1, 600], [600, 599, 257], [0, 0, 0], [256, 255, 128]])
def test_ragged_batches(lengths, dtype):
    check(3, 600, 2, 24, 40, dtype, lengths=lengths, seed=3)
    check(3, 600, 2, 64, 64, dtype, lengths=lengths, state=False, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_without_state_and_with_own_scale(dtype):
    check(2, 70, 4, 16, 16, dtype, state=False, scale=0.3)
    check(2, 70, 4, 16, 16, dtype, scale=-1.5)
    check(2, 300, 4, 16, 16, dtype, grad_state=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_decays_from_none_to_all(dtype):
    decay = torch.tensor([0.0, -1e-4, -5.0, -200.0, float("-inf")])
    check(1, 300, 5, 16, 24, dtype, decay=decay, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -9, 2.0 ** 5])
def test_fp16_near_the_ends_of_its_range(size):
    """Small: products near and under fp16's smallest normal number.  Large: a carried state above its largest number (65504)
    whose outputs are in range, because q is small."""
    x, decay, do, ds = make(1, 300, 2, 32, 32, torch.float16, seed=13)
    decay = torch.tensor([-2.0 ** -9, -0.1])
    big = size > 1
    x = {"q": (x["q"].double() * (2.0 ** -9 if big else size)).half(), "k": (x["k"].double().abs() * (size * 16 if big else size)).half(),
         "v": (x["v"].double().abs() * (size * 8 if big else size)).half(), "state": x["state"] * 0}
    d = {k: v.cuda() for k, v in x.items()}
    o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"], scale=2.0 ** -4)
    f = {k: v.double() for k, v in x.items()}
    ro, rend = attention(f["q"], f["k"], f["v"], decay.double(), f["state"], None, 2.0 ** -4)
    a = {k: v.abs() for k, v in f.items()}
    mo, mend = attention(a["q"], a["k"], a["v"], decay.double(), a["state"], None, 2.0 ** -4)
    assert not big or rend.abs().max() > 65504 > 2 * ro.abs().max()
    # a weight under 2^-14 is off by up to 2^-25 (half of fp16's smallest step) for each of the chunk's 64 rows of v
    low = 64 * 2.0 ** -25 * float(a["v"].max())
    assert_within(o, ro, HALF[torch.float16] * (ro.abs() + 2 * mo) + 512 * 2.0 ** -24 * mo + low + TINY[torch.float16], "out")
    assert_within(end, rend, 512 * 2.0 ** -24 * mend, "end state")


@pytest.mark.gpu
def test_lengths_out_of_range_are_held_to_the_batch():
    x, decay, _, _ = make(3, 40, 2, 8, 8, torch.float32)
    d = {k: v.cuda() for k, v in x.items()}
    run = lambda n: linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"], lengths=torch.tensor(n, dtype=torch.int32, device="cuda"))  # noqa: E731
    for a, b in zip(run([-5, 1000, 7]), run([0, 40, 7])):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_rows_behind_the_end_are_not_read(dtype):
    x, decay, do, ds = make(2, 300, 2, 32, 32, dtype, seed=6)
    n = torch.tensor([130, 0], dtype=torch.int32, device="cuda")
    res = []
    for bad in (False, True):
        d = {k: v.clone().cuda() for k, v in x.items()}
        g = do.clone().cuda()
        if bad:
            for k in ("q", "k", "v"):
                d[k][0, 130:] = float("nan")
                d[k][1] = float("inf")
            g[0, 130:] = float("nan")
        for v in d.values():
            v.requires_grad_(True)
        o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"], lengths=n)
        res.append([o, end, *torch.autograd.grad((o, end), list(d.values()), (g, ds.cuda()))])
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_strided_and_shared_inputs(dtype):
    b, t, h, d = 2, 300, 3, 40
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(b, t, 3, h, d, generator=g).to(dtype).cuda().requires_grad_(True)
    decay = -torch.exp2(-torch.linspace(0.0, 9.0, h)).cuda()
    q, k, v = qkv.unbind(2)
    o, _ = linattn.linear_attention(q, k, v, decay)
    o2, _ = linattn.linear_attention(*(z.contiguous() for z in (q, k, v)), decay)
    assert torch.equal(o, o2)
    head = torch.randn(b, t, h, d, generator=g).to(dtype).cuda()
    (a,) = torch.autograd.grad(o, qkv, head)
    (c,) = torch.autograd.grad(o2, qkv, head.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(a, c)
    # keys shared by all heads (stride 0), an odd start, a transposed last dimension
    one = torch.randn(b, t, 1, d, generator=g).to(dtype).cuda()
    odd = torch.empty(one.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(one).copy_(one)
    with torch.no_grad():
        x = linattn.linear_attention(q, one.expand(b, t, h, d), v, decay)[0]
        assert torch.equal(x, linattn.linear_attention(q, one.repeat(1, 1, h, 1), v, decay)[0])
        x = linattn.linear_attention(q.transpose(-1, -2).contiguous().transpose(-1, -2), odd.expand(b, t, h, d), v, decay)[0]
    # an odd start may take another kernel than an aligned one: not the same bits, but the same bound (see `bounds`)
    f = [z.detach().double().cpu() for z in (q, one.expand(b, t, h, d), v)]
    ref = attention(*f, decay.double().cpu(), None, None, d ** -0.5)[0]
    mag = attention(*(z.abs() for z in f), decay.double().cpu(), None, None, d ** -0.5)[0]
    assert_within(x, ref, HALF[dtype] * (ref.abs() + (2 * mag if dtype != torch.float32 else 0)) + 512 * 2.0 ** -24 * mag + TINY[dtype])


@pytest.mark.gpu
def test_gradient_of_a_sum_has_no_strides():
    x, decay, _, _ = make(1, 50, 2, 8, 8, torch.float32)
    d = {k: v.cuda().requires_grad_(True) for k, v in x.items()}
    o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"])
    g = torch.autograd.grad(o.sum() + end.sum(), list(d.values()), retain_graph=True)
    g2 = torch.autograd.grad((o, end), list(d.values()), (torch.ones_like(o), torch.ones_like(end)))
    for a, b in zip(g, g2):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_gradient_against_differences():
    x, decay, do, ds = make(1, 90, 2, 8, 12, torch.float32, seed=7)
    d = {k: v.cuda().requires_grad_(True) for k, v in x.items()}
    o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"])
    grads = torch.autograd.grad((o, end), list(d.values()), (do.cuda(), ds.cuda()))
    gen = torch.Generator().manual_seed(1)

    def loss(s):
        o, end = linattn.linear_attention(s["q"].cuda(), s["k"].cuda(), s["v"].cuda(), decay.cuda(), state=s["state"].cuda())
        return float((o.cpu().double() * do.double()).sum() + (end.cpu().double() * ds.double()).sum())

    for name, g in zip(x, grads):
        way = torch.randn(x[name].shape, generator=gen)
        e = 0.25                     # the outputs are linear in each input: only rounding is left
        diff = (loss({**x, name: x[name] + e * way}) - loss({**x, name: x[name] - e * way})) / (2 * e)
        want = float((g.cpu().double() * way.double()).sum())
        size = float((o.detach().abs().cpu() * do.abs()).double().sum() + (end.detach().abs().cpu() * ds.abs()).double().sum())
        assert abs(diff - want) <= 2.0 ** -16 * size / e, (name, diff, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,h,dk,dv", [(1, 1, 1, 1), (2, 3, 16, 16), (3, 5, 40, 56), (4, 2, 128, 128), (1, 2, 33, 7), (2, 2, 64, 130 - 2)])
def test_single_tokens_continue_a_prompt(b, h, dk, dv, dtype):
    x, decay, _, _ = make(b, 20, h, dk, dv, dtype, seed=8)
    d = {k: v.cuda() for k, v in x.items()}
    whole, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"])
    _, st = linattn.linear_attention(d["q"][:, :13], d["k"][:, :13], d["v"][:, :13], decay.cuda(), state=d["state"])
    ref = {k: v.double() for k, v in x.items()}
    ro, rend = attention(ref["q"], ref["k"], ref["v"], decay.double(), ref["state"], None, dk ** -0.5)
    ab = {k: v.abs() for k, v in ref.items()}
    mo, mend = attention(ab["q"], ab["k"], ab["v"], decay.double(), ab["state"], None, dk ** -0.5)
    for t in range(13, 20):
        o = linattn.step(d["q"][:, t], d["k"][:, t], d["v"][:, t], decay.cuda(), st)
        assert_within(o, ro[:, t], HALF[dtype] * ro[:, t].abs() + 512 * 2.0 ** -24 * mo[:, t] + TINY[dtype], f"token {t}")
    assert_within(st, rend, 512 * 2.0 ** -24 * mend, "state")
    assert_within(end, rend, 512 * 2.0 ** -24 * mend, "end state")


@pytest.mark.gpu
def test_a_sequence_in_two_parts_is_the_sequence():
    x, decay, _, _ = make(1, 900, 2, 64, 64, torch.bfloat16, seed=9)
    d = {k: v.cuda() for k, v in x.items()}
    run = lambda lo, hi, s: linattn.linear_attention(d["q"][:, lo:hi], d["k"][:, lo:hi], d["v"][:, lo:hi], decay.cuda(), state=s)  # noqa: E731
    _, whole = run(0, 900, d["state"])
    _, part = run(0, 333, d["state"])
    _, part = run(333, 900, part)
    ab = {k: v.double().abs() for k, v in x.items()}
    mag = attention(ab["q"], ab["k"], ab["v"], decay.double(), ab["state"], None, 1.0)[1]
    assert_within(part, whole.double(), 1024 * 2.0 ** -24 * mag)


@pytest.mark.gpu
def test_empty_batches_and_sequences():
    decay = torch.tensor([-0.1, -0.2], device="cuda")
    q = torch.zeros(0, 5, 2, 8, device="cuda")
    o, end = linattn.linear_attention(q, q, q, decay)
    assert o.shape == (0, 5, 2, 8) and end.shape == (0, 2, 8, 8)
    q = torch.zeros(2, 0, 2, 8, device="cuda", requires_grad=True)
    s = torch.randn(2, 2, 8, 8, device="cuda", requires_grad=True)
    o, end = linattn.linear_attention(q, q, q, decay, state=s)
    assert o.shape == (2, 0, 2, 8) and torch.equal(end, s)
    ds = torch.randn_like(s)
    (g,) = torch.autograd.grad(end, s, ds)
    assert torch.equal(g, ds)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    # one head of a batch whose rows lie 2^31 elements apart
    b, t, h, d = 2, 40, 1, 16
    big = torch.zeros(2 ** 31 + t * d, dtype=torch.float16, device="cuda")
    view = big.as_strided((b, t, h, d), (2 ** 31, d, d, 1))
    small = torch.randn(b, t, h, d, device="cuda").half()
    view.copy_(small)
    decay = torch.tensor([-0.05], device="cuda")
    a, c = linattn.linear_attention(view, view, view, decay), linattn.linear_attention(small, small, small, decay)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.gpu
def test_long_sequence():
    # 2^17 tokens of one head; the reference in 64 bits a block of rows at a time
    t, d = 1 << 17, 16
    x, _, _, _ = make(1, t, 1, d, d, torch.bfloat16, seed=10, state=False)
    decay = torch.tensor([-2.0 ** -11])
    q, k, v = (x[n].cuda() for n in ("q", "k", "v"))
    o, end = linattn.linear_attention(q, k, v, decay.cuda())
    Q, Kk, V = (z.double()[0, :, 0] for z in (q, k, v))
    a = float(decay.double())
    far = 1 << 15                                     # exp(-2^15 / 2^11) = e^-16: older tokens are under 2e-7 of the sum
    for lo in (0, 4096 * 7, t - 4096):
        hi, j0 = lo + 4096, max(0, lo - far)
        i, j = torch.arange(lo, hi, device="cuda"), torch.arange(j0, hi, device="cuda")
        w = torch.exp(a * (i[:, None] - j[None]).clamp(min=0).double()) * (i[:, None] >= j[None])
        p = Q[lo:hi] @ Kk[j0:hi].T * w
        m = (Q[lo:hi].abs() @ Kk[j0:hi].abs().T * w) @ V[j0:hi].abs()
        ref = (p @ V[j0:hi]) / 4
        assert_within(o[0, lo:hi, 0], ref, HALF[torch.bfloat16] * ref.abs() + (2 * HALF[torch.bfloat16] + 2.0 ** -14 + 2e-7) * m / 4)
    w = torch.exp(a * torch.arange(t - 1, -1, -1, device="cuda").double())
    ref, mag = (w[:, None] * Kk).T @ V, (w[:, None] * Kk.abs()).T @ V.abs()
    assert_within(end[0, 0], ref, 2.0 ** -14 * mag)


@pytest.mark.gpu
def test_same_bits_on_another_stream_and_in_a_graph():
    x, decay, do, _ = make(2, 700, 2, 64, 64, torch.bfloat16, seed=12)
    d = {k: v.cuda().requires_grad_(True) for k, v in x.items()}
    decay, do = decay.cuda(), do.cuda()

    def once():
        o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay, state=d["state"])
        g = torch.autograd.grad(o, list(d.values()), do)
        # no eager graph of these leaves may live on while a backward pass is captured (autograd would order the capture
        # behind the eager stream), so outputs leave without theirs
        return [o.detach(), end.detach(), *g]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = once()
    with torch.no_grad():
        keep = d["v"].clone()
        d["v"].mul_(-1.0)
    graph.replay()
    assert not torch.equal(first[0], third[0])
    with torch.no_grad():
        d["v"].copy_(keep)
    graph.replay()
    for a, b in zip(first, third):
        assert torch.equal(a, b)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x = torch.randn(2, 6, 2, 8, device="cuda")
    decay = torch.tensor([-0.1, -0.2], device="cuda")
    leaf = decay.clone().requires_grad_(True)
    for call in (lambda: linattn.linear_attention(x, x[:, :, :, :4], x, decay), lambda: linattn.linear_attention(x, x, x.half(), decay),
                 lambda: linattn.linear_attention(x, x, x, decay.half()), lambda: linattn.linear_attention(x, x, x, decay[:1]),
                 lambda: linattn.linear_attention(x, x, x, leaf), lambda: linattn.linear_attention(x, x, x, decay, state=x),
                 lambda: linattn.linear_attention(x, x, x, decay, lengths=torch.tensor([1, 2], device="cuda")),
                 lambda: linattn.linear_attention(x, x, x, decay, lengths=torch.tensor([1, 2], dtype=torch.int32)),
                 lambda: linattn.linear_attention(*(torch.randn(1, 2, 1, 129, device="cuda"),) * 3, decay[:1]),
                 lambda: linattn.step(x[:, 0], x[:, 0], x[:, 0], decay, torch.zeros(2, 2, 8, 8, device="cuda").transpose(-1, -2)),
                 lambda: linattn.step(x[:, 0].clone().requires_grad_(True), x[:, 0], x[:, 0], decay, torch.zeros(2, 2, 8, 8, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.gpu
def test_a_step_shows_in_the_state_it_writes():
    # a graph that has kept the state must not read what a later step has made of it
    b, t, h, d = 2, 5, 2, 16
    q, k, v = (torch.randn(b, t, h, d, device="cuda") for _ in range(3))
    decay = torch.full((h,), -0.1, device="cuda")
    state = torch.randn(b, h, d, d, device="cuda")
    q.requires_grad_(True)
    o, _ = linattn.linear_attention(q, k, v, decay, state=state)
    with torch.no_grad():
        linattn.step(q[:, 0], k[:, 0], v[:, 0], decay, state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()
    with torch.inference_mode():
        own = state.clone()
        linattn.step(k[:, 0], k[:, 0], v[:, 0], decay, own)
        linattn.step(k[:, 0], k[:, 0], v[:, 0], decay, state.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once_and_two_graphs(dtype):
    b, t, h, d = 1, 900, 6, 64
    decay = -torch.exp2(-torch.linspace(1, 6, h)).cuda()
    sets = [[torch.randn(b, t, h, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(s + i)).to(dtype) for i in range(4)]
            for s in (0, 10)]

    def both(q, k, v, g):
        o, e, s = linattn.forward(q, k, v, decay)
        return (o, e, *linattn.backward(g, None, q, k, v, decay, None, None, s))

    alone = [both(*x) for x in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    together = []
    for _ in range(4):
        for stream, x in zip(streams, sets):
            with torch.cuda.stream(stream):
                together.append(both(*x))
    torch.cuda.synchronize()
    for i, got in enumerate(together):
        assert all(torch.equal(a, c) for a, c in zip(got, alone[i % 2]))
    graphs, outs = [], []
    for x in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both(*x))
    for order in ((0, 1), (1, 0)):
        for stream, i in zip(streams, order):
            with torch.cuda.stream(stream):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, c) for a, c in zip(outs[i], alone[i]))
            for a in outs[i]:
                a.zero_()
        torch.cuda.synchronize()


# ---- products beyond fp16's range --------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("large", ["qk", "vdo"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (24, 120), (64, 64), (128, 64), (128, 128)])
def test_products_beyond_the_range_of_fp16(dk, dv, large, dtype):
    """scale q.k or v.do above 65504 with results in range: a prompt's weights, and gradients under a loss scale."""
    t, decay = 200, torch.tensor([-0.1, -2.0 ** -9])
    g = torch.Generator().manual_seed(dk + dv)
    r = lambda d, size: (torch.randn(1, t, 2, d, generator=g, dtype=torch.float64) * size).to(dtype)  # noqa: E731
    top = (2.0 ** 18 / (dk if large == "qk" else dv)) ** 0.5
    size = [top, top, 2.0 ** -8, 2.0 ** -8] if large == "qk" else [2.0 ** -8, 2.0 ** -8, top, top]
    q, k, v, do = (r(d, s) for d, s in zip((dk, dk, dv, dv), size))
    if large == "qk":
        q, k = q.abs(), k.abs()
    else:
        v, do = v.abs(), do.abs()
    x = {"q": q, "k": k, "v": v, "state": torch.zeros(1, 2, dk, dv)}
    ds = torch.zeros(1, 2, dk, dv)
    f = {n: z.double().requires_grad_(True) for n, z in x.items()}
    assert (torch.einsum("bihd,bjhd->bhij", *((q, k) if large == "qk" else (v, do))).double()).max() > 2 * 65504
    ro, _ = attention(f["q"], f["k"], f["v"], decay.double(), f["state"], None, 1.0)
    want = (ro, *torch.autograd.grad(ro, [f["q"], f["k"], f["v"]], do.double()))
    assert all(0 < w.abs().max() < 65504 for w in want)
    dev = {n: z.cuda().requires_grad_(True) for n, z in x.items()}
    o, _ = linattn.linear_attention(dev["q"], dev["k"], dev["v"], decay.cuda(), state=dev["state"], scale=1.0)
    got = (o, *torch.autograd.grad(o, [dev["q"], dev["k"], dev["v"]], do.cuda()))
    mags = bounds(x, decay, do, ds, None, 1.0, dtype)
    for name, a, w, m in zip(("out", "gradient of q", "gradient of k", "gradient of v"), got, want, [mags[0], *mags[2:5]]):
        assert_within(a, w, HALF[dtype] * w.abs() + m + TINY[dtype], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128)])
def test_small_fp16_gradients_that_meet_large_rows(dk, dv):
    """Weights scale v.do of 2^-21 and below, of which fp16's own steps would keep three bits, times rows of 2^9: gradients
    that fp16 holds in full.  No allowance for small weights."""
    t, sc, decay = 200, 2.0 ** -10, torch.tensor([-0.1, -2.0 ** -9])
    g = torch.Generator().manual_seed(dk)
    r = lambda d, size: (torch.randn(1, t, 2, d, generator=g, dtype=torch.float64) * size).half()  # noqa: E731
    x = {"q": r(dk, 2.0 ** 9), "k": r(dk, 2.0 ** 9), "v": r(dv, 2.0 ** -4), "state": torch.zeros(1, 2, dk, dv)}
    do, ds = r(dv, 2.0 ** -10), torch.zeros(1, 2, dk, dv)
    f = {n: z.double().requires_grad_(True) for n, z in x.items()}
    ro, _ = attention(f["q"], f["k"], f["v"], decay.double(), f["state"], None, sc)
    want = torch.autograd.grad(ro, [f["q"], f["k"], f["v"]], do.double())
    dev = {n: z.cuda().requires_grad_(True) for n, z in x.items()}
    o, _ = linattn.linear_attention(dev["q"], dev["k"], dev["v"], decay.cuda(), state=dev["state"], scale=sc)
    got = torch.autograd.grad(o, [dev["q"], dev["k"], dev["v"]], do.cuda())
    mags = bounds(x, decay, do, ds, None, sc, torch.float16)
    for name, a, w, m in zip(("gradient of q", "gradient of k", "gradient of v"), got, want, mags[2:5]):
        assert_within(a, w, HALF[torch.float16] * w.abs() + m + TINY[torch.float16], name)


# ---- what 16-bit results are rounded by --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(32, 32), (40, 72), (64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("t", [127, 128, 700])
def test_16_bit_results_carry_their_own_rounding_alone(t, dk, dv, dtype):
    """Beside the rounding of the result: a chunk's weights, and the state where it meets a chunk, are held in two parts
    (bf16: 2^-16 of a value each; fp16 2^-22), the values summed into the state likewise, whose smaller part may be rounded
    once more: three such roundings of a term at most; then 32-bit sums."""
    sc = dk ** -0.5
    x, decay, do, ds = make(1, t, 3, dk, dv, dtype, seed=t + dk + dv)
    f = {n: z.double().requires_grad_(True) for n, z in x.items()}
    ro, rend = attention(f["q"], f["k"], f["v"], decay.double(), f["state"], None, sc)
    want = (ro, *torch.autograd.grad((ro, rend), list(f.values())[:3], (do.double(), ds.double())))
    dev = {n: z.cuda().requires_grad_(True) for n, z in x.items()}
    o, end = linattn.linear_attention(dev["q"], dev["k"], dev["v"], decay.cuda(), state=dev["state"])
    got = (o, *torch.autograd.grad((o, end), list(dev.values())[:3], (do.cuda(), ds.cuda())))
    mags = bounds(x, decay, do, ds, None, sc, dtype)
    part = HALF[dtype] ** 2
    for name, a, w, m in zip(("out", "gradient of q", "gradient of k", "gradient of v"), got, want, [mags[0], *mags[2:5]]):
        mag = m / (2 * HALF[dtype] + 512 * 2.0 ** -24)
        assert_within(a, w, HALF[dtype] * w.abs() + (3 * part + 512 * 2.0 ** -24) * mag + TINY[dtype], name)


@pytest.mark.gpu
def test_the_status_waits_for_every_stream():
    # torch's streams do not wait for the default stream, nor it for them
    x, decay, _, _ = make(2, 7680, 8, 64, 64, torch.bfloat16, seed=14, state=False)
    q, k, v, decay = x["q"].cuda(), x["k"].cuda(), x["v"].cuda(), -torch.exp2(-torch.linspace(1, 8, 8)).cuda()
    linattn.linear_attention(q, k, v, decay)
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(200):
            linattn.linear_attention(q, k, v, decay)
        done.record()
    assert _lib.load().cnl_linattn_status() == 0
    assert done.query()


# ---- rows behind the end in the kernels that load them -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (40, 72)])
@pytest.mark.parametrize("t,lengths", [(200, [130, 0]), (300, [130, 257]), (300, [0, 299]), (1300, [1111, 129]), (1300, [0, 513]), (128, [127, 1])])
def test_wide_rows_behind_the_end_may_hold_anything(t, lengths, dk, dv):
    """As test_rows_behind_the_end_are_not_read, at the sizes whose kernels bring whole chunks: whatever stands behind a length
    gives the same bits as zeros there.  Cut chunks, one and several segments, both directions."""
    x, decay, do, ds = make(2, t, 2, dk, dv, torch.bfloat16, seed=t + dk + dv)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    res = []
    for bad in (0.0, float("nan"), float("inf")):
        d = {k: v.clone().cuda() for k, v in x.items()}
        g = do.clone().cuda()
        for z in (d["q"], d["k"], d["v"], g):
            for i, m in enumerate(lengths):
                z[i, m:] = bad
        for v in d.values():
            v.requires_grad_(True)
        o, end = linattn.linear_attention(d["q"], d["k"], d["v"], decay.cuda(), state=d["state"], lengths=n)
        res.append([o, end, *torch.autograd.grad((o, end), list(d.values()), (g, ds.cuda()))])
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.isfinite(a).all() and torch.equal(a, b)
    assert _lib.load().cnl_linattn_status() == 0
