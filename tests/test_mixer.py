"""The network operators together, as a network in front of the optimisation layers runs them."""
import copy

import pytest
import torch

from customnetworklayers_b200.mixer import PixelMixer
from tests.operators_ref import act, act_slope, attention, block_norm, put_away


class _Act(torch.autograd.Function):
    """GELU whose slope is taken at the 8-bit value of its input."""

    @staticmethod
    def forward(ctx, x, fmt):
        ctx.save_for_backward(x)
        ctx.fmt = fmt
        return act(x, "gelu")

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        at = x if ctx.fmt is None else put_away(x.reshape(-1).cpu(), ctx.fmt).view(x.shape).to(x.device)
        return g * act_slope(at, "gelu"), None


def reference(m, x, states=None, lengths=None):
    """The mixer's forward pass in 64 bits from the modules' own parameters (norms keep full precision)."""
    m = copy.deepcopy(m).double()
    x = x.detach().double().clone().requires_grad_(True)
    n, c = x.shape[0], x.shape[-1]
    y, ends = x, []
    h = block_norm(y, None, None, None, None, None, m.pre.weight, m.pre.bias, m.pre.kind == "layer", True)[1]
    for i in range(len(m.gate)):
        a, r = m.attention[i], m.after_attention[i]
        q, k, v = a.qkv(h).view(n, -1, 3, a.heads, c // a.heads).unbind(2)
        o, end = attention(q, k, v, a.log_decay, None if states is None else states[i].double(), lengths, (c // a.heads) ** -0.5)
        ends.append(end)
        layer = r.kind == "layer"
        y, h = block_norm(y, a.out(o.reshape(x.shape)), m.gate[i](h), r.scale, r.weight, r.bias, r.next_weight, r.next_bias, layer, True)
        r = m.after_mlp[i]
        u = m.down[i](_Act.apply(m.up[i](h), getattr(m.act, "fmt", None)))
        y, h = block_norm(y, u, None, r.scale, r.weight, r.bias, r.next_weight, r.next_bias, layer, True)
    return m, x, y, ends


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_image_forward_and_backward(kind):
    torch.manual_seed(0)
    m = PixelMixer(48, 3, depth=2, kind=kind).cuda()
    x = torch.randn(2, 9, 13, 48, device="cuda", requires_grad=True)
    y, ends = m(x)
    up = torch.randn_like(y)
    m2, x2, y2, ends2 = reference(m, x)
    y.backward(up)
    y2.backward(up.double())
    # some hundred 32-bit roundings of 2^-24 in sequence through five sublayers, each relative to its rows
    assert rel(y, y2) <= 2.0 ** -16
    assert all(rel(a, b) <= 2.0 ** -16 for a, b in zip(ends, ends2))
    assert rel(x.grad, x2.grad) <= 2.0 ** -15
    for (name, p), q in zip(m.named_parameters(), m2.parameters()):
        assert rel(p.grad, q.grad) <= 2.0 ** -14, name


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,allowed", [("int8", 2.0 ** -5), ("e4m3", 2.0 ** -3)])
def test_with_checkpoints_in_8_bits(fmt, allowed):
    torch.manual_seed(1)
    m = PixelMixer(64, 2, depth=2, checkpoint=fmt).cuda()
    plain = PixelMixer(64, 2, depth=2).cuda()
    plain.load_state_dict(m.state_dict())
    x = torch.randn(2, 300, 64, device="cuda", requires_grad=True)
    y, _ = m(x)
    z, _ = plain(x)
    # the same forward pass but for the two forms of GELU (2^-21 of a value)
    assert rel(y, z) <= 2.0 ** -16
    up = torch.randn_like(y)
    (a,) = torch.autograd.grad(y, x, up)
    (b,) = torch.autograd.grad(z, x, up)
    # an element is off by at most 1/64 of its block's largest (int8) or 1/16 of itself (e4m3); norms and slopes pass that
    # on with a factor around one, and errors of different elements are independent
    assert 0 < rel(a, b) <= allowed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_at_once_and_its_tokens_one_by_one(dtype):
    torch.manual_seed(2)
    m = PixelMixer(32, 4, depth=2).cuda().to(dtype)
    x = torch.randn(3, 40, 32, device="cuda").to(dtype)
    with torch.no_grad():
        whole, ends = m(x)
        _, states = m(x[:, :30])
        tail = [m.step(x[:, t], states) for t in range(30, 40)]
    allowed = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -4       # bf16: projections and norms round 2^-8 some 20 times
    assert rel(torch.stack(tail, 1), whole[:, 30:]) <= allowed
    assert all(rel(a, b) <= allowed for a, b in zip(states, ends))


@pytest.mark.gpu
def test_padded_batch_and_fresh_states():
    torch.manual_seed(3)
    m = PixelMixer(32, 2, depth=1).cuda()
    x = torch.randn(2, 50, 32, device="cuda")
    lengths = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y, ends = m(x, m.new_states(2), lengths)
        short, end = m(x[1:, :20])
    assert rel(y[1:, :20], short) <= 2.0 ** -18 and rel(ends[0][1:], end[0]) <= 2.0 ** -18


@pytest.mark.gpu
def test_in_front_of_the_inpainting_layer():
    """Mixer -> confidence and data term -> TV layer: one backward pass through both."""
    from customnetworklayers_b200 import tvInpaint_cuda_ext
    from customnetworklayers_b200.TVInpainting import TVInpaint
    torch.manual_seed(4)
    h, w = 24, 32
    m = PixelMixer(32, 2, depth=1, checkpoint="int8").cuda()
    head = torch.nn.Linear(32, 5).cuda()
    layer = TVInpaint("cuda", its=10, pid=9)
    feat = torch.randn(1, h, w, 32, device="cuda")
    z = head(m(feat)[0])
    wx, wy, c = (torch.sigmoid(z[..., i:i + 1]) for i in range(3))
    b = z[..., 3:5]
    sol = layer(wx, wy, c, b, torch.zeros_like(b))
    sol.square().mean().backward()
    tvInpaint_cuda_ext.release(9)
    for name, p in list(m.named_parameters()) + list(head.named_parameters()):
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name


@pytest.mark.gpu
def test_training_step_in_a_graph():
    torch.manual_seed(5)
    m = PixelMixer(64, 2, depth=1, checkpoint="int8").cuda()
    x = torch.randn(1, 700, 64, device="cuda")
    params = list(m.parameters())

    def once():
        y, _ = m(x)
        return torch.autograd.grad(y.square().sum(), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            once()
    torch.cuda.current_stream().wait_stream(side)
    want = [g.clone() for g in once()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    keep = x.clone()
    x.zero_()
    graph.replay()
    x.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert rel(a, b) <= 2.0 ** -16                    # the library's products may split their sums differently


# ---- forward-mode derivatives ------------------------------------------------------------------------------------
def _forward_mode_calls(device):
    import torch.autograd.forward_ad as fwd
    from customnetworklayers_b200 import blocknorm, ckpt8, linattn
    r = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    dual = lambda *s: fwd.make_dual(r(*s), r(*s))  # noqa: E731
    x, q, decay, w = r(4, 16), r(1, 5, 2, 8), -torch.ones(2, device=device), torch.ones(16, device=device)
    state = torch.zeros(1, 2, 8, 8, device=device)
    return [lambda: ckpt8.activation(dual(4, 16)), lambda: blocknorm.pre_norm(dual(4, 16), w), lambda: blocknorm.pre_norm(x, dual(16)),
            lambda: blocknorm.residual_norm(x, dual(4, 16), w), lambda: blocknorm.residual_norm(x, x, w, gate=dual(4, 16)),
            lambda: blocknorm.residual_norm(x, x, w, scale=dual(16)), lambda: blocknorm.residual_norm(x, x, w, next_weight=dual(16)),
            lambda: linattn.linear_attention(dual(1, 5, 2, 8), q, q, decay), lambda: linattn.linear_attention(q, q, dual(1, 5, 2, 8), decay),
            lambda: linattn.linear_attention(q, q, q, dual(2)), lambda: linattn.linear_attention(q, q, q, decay, state=dual(1, 2, 8, 8)),
            lambda: linattn.step(dual(1, 2, 8), q[:, 0], q[:, 0], decay, state), lambda: linattn.step(q[:, 0], q[:, 0], q[:, 0], dual(2), state),
            lambda: linattn.step(q[:, 0], q[:, 0], q[:, 0], decay, dual(1, 2, 8, 8))]


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    # as the optimisation layers refuse it; a result without its tangent would pass for a derivative of zero
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for i, call in enumerate(_forward_mode_calls("cuda")):
            with pytest.raises(RuntimeError):             # NotImplementedError is one
                call()
                pytest.fail(f"call {i} came back")


def test_inputs_with_a_tangent_want_a_derivative():
    import torch.autograd.forward_ad as fwd
    from customnetworklayers_b200 import linattn
    from customnetworklayers_b200._tensor import wants_grad
    x = torch.ones(1, 2, 8)
    assert not wants_grad(x, None)
    with fwd.dual_level():
        assert not wants_grad(x, None)
        d = fwd.make_dual(x, x)
        assert wants_grad(None, x, d)
        with torch.no_grad():
            assert wants_grad(d)
        with pytest.raises(RuntimeError, match="no gradient"):
            linattn.step(d, x, x, torch.zeros(2), torch.zeros(1, 2, 8, 8))
    assert not wants_grad(d)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 6, 32), (0, 3, 4, 32), (2, 0, 32), (0, 0, 5, 32)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_empty_batches_and_images(shape, checkpoint):
    m = PixelMixer(32, 2, depth=2, checkpoint=checkpoint).cuda()
    x = torch.zeros(*shape, device="cuda", requires_grad=True)
    y, states = m(x, m.new_states(shape[0]))
    assert y.shape == shape and all(s.shape == (shape[0], 2, 16, 16) for s in states)
    y.sum().backward()
    assert x.grad.shape == shape and all(torch.count_nonzero(p.grad) == 0 for p in m.parameters())
    states = m.new_states(0)
    assert m.step(torch.zeros(0, 32, device="cuda"), states).shape == (0, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_memories_keep_their_length_in_every_type(dtype):
    m = PixelMixer(64, 8, depth=2)
    want = -torch.exp2(-torch.linspace(2.0, 11.0, 8))
    state = m.state_dict()
    for net in (m.to(dtype), copy.deepcopy(m), m.float(), m.to(dtype).to("cpu")):
        for a in net.attention:
            assert a.log_decay.dtype == torch.float32 and torch.equal(a.log_decay, want)
    m.half().load_state_dict({k: v.clone() for k, v in state.items()})
    assert all(torch.equal(a.log_decay, want) for a in m.attention) and m.gate[0].weight.dtype == torch.float16
    try:
        torch.set_default_dtype(dtype)
        assert torch.equal(PixelMixer(64, 8, depth=1).attention[0].log_decay, want)
    finally:
        torch.set_default_dtype(torch.float32)
    with torch.device("meta"):
        empty = PixelMixer(64, 8, depth=1)
    assert empty.to(dtype).to_empty(device="cpu").attention[0].log_decay.dtype == torch.float32


@pytest.mark.gpu
def test_a_bf16_mixer_is_the_fp32_one_with_rounded_weights():
    """Against 64 bits with the decays of the fp32 model: projections, norms and attention round 2^-8 some 20 times; a decay of
    2^-9 too much or too little for each token would add 2^-9 times the memory's length over what it holds."""
    torch.manual_seed(6)
    m = PixelMixer(64, 8, depth=1).cuda()
    want = [a.log_decay.clone() for a in m.attention]
    m = m.to(torch.bfloat16)
    x = torch.randn(1, 2000, 64, device="cuda").bfloat16()
    with torch.no_grad():
        y, ends = m(x)
    m2, _, y2, ends2 = reference(m, x)
    assert all(torch.equal(a.log_decay.float(), w) for a, w in zip(m2.attention, want))
    assert rel(y, y2) <= 2.0 ** -5 and all(rel(a, b) <= 2.0 ** -5 for a, b in zip(ends, ends2))


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_precision(dtype, checkpoint):
    """fp32 parameters and stream under autocast: the projections, the attention and the activation run in 16 bits."""
    torch.manual_seed(7)
    m = PixelMixer(32, 2, depth=2, checkpoint=checkpoint).cuda()
    x = torch.randn(2, 150, 32, device="cuda", requires_grad=True)
    params = list(m.parameters())
    y, ends = m(x)
    up = torch.randn_like(y)
    want = torch.autograd.grad(y, [x, *params], up)
    with torch.autocast("cuda", dtype=dtype):
        y2, ends2 = m(x)
        with torch.no_grad():
            one = m.step(x[:, 0], m.new_states(2))
            first, _ = m(x[:, :1])
    got = torch.autograd.grad(y2, [x, *params], up)
    assert y2.dtype == torch.float32 and all(e.dtype == torch.float32 for e in ends2) and one.dtype == torch.float32
    # half a step of the type (2^-8 at most) in each of some twenty projections, attentions and activations in a row
    assert 0 < rel(y2, y) <= 2.0 ** -4 and rel(one, first[:, 0]) <= 2.0 ** -4
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and rel(a, b) <= 2.0 ** -3


# ---- several ranks -----------------------------------------------------------------------------------------------
def _sum_gradients(rank, world, port, q):
    import os
    import torch.distributed as dist
    from customnetworklayers_b200.blocknorm import ResidualNorm
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    torch.manual_seed(0)
    nets = [PixelMixer(16, 2, depth=1), ResidualNorm(16, bias=True)]
    g = torch.Generator().manual_seed(rank)
    own = []
    for net in nets:
        for i, p in enumerate(net.parameters()):
            if i != 1:                                   # a parameter without a gradient stays so
                p.grad = torch.randn(p.shape, generator=g)
            own.append(None if p.grad is None else p.grad.clone())
        net.allreduce_parameter_grads()
    got = [p.grad for net in nets for p in net.parameters()]
    q.put((rank, [None if t is None else t.numpy() for t in own], [None if t is None else t.numpy() for t in got]))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_sum_the_gradients_of_all_parameters():
    import socket
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_sum_gradients, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    (_, own0, got0), (_, own1, got1) = sorted((q.get(timeout=120) for _ in procs), key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert len(own0) > 10 and sum(t is None for t in got0) == 2
    for a, b, x, y in zip(own0, own1, got0, got1):
        if a is not None:
            assert (a + b == x).all() and (x == y).all()
