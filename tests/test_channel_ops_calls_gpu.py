"""Calls of the layer norm and MXFP4 operators that a program makes around them: modules whose weights change, gradients of
gradients, forward-mode tangents, saved-tensor hooks, skip connections, tensors of other dimensions and of more than 2^31 elements.

Where values are compared, both sides are the same kernels on the same inputs (equal bits), or whole numbers whose sums
float32 holds exactly, or the tolerance is derived beside the comparison."""
import copy
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-5


def dc():
    import deltacnn_b200
    return deltacnn_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def channels_last(t):
    return t.contiguous(memory_format=torch.channels_last)


# ---- DCMX4Linear and its packed weight -------------------------------------------------------------------------

@pytest.fixture
def packings(monkeypatch):
    """A list that grows by one entry for every matrix that is packed outside a product."""
    from deltacnn_b200 import channel_ops
    calls, quantize = [], channel_ops._quantize
    monkeypatch.setattr(channel_ops, "_quantize", lambda *a: calls.append(a) or quantize(*a))
    return calls


def packed_layer(seed):
    g = gen(seed)
    layer = dc().DCMX4Linear(64, 48).cuda().half()
    with torch.no_grad():
        layer.weight.copy_(randn((48, 64), g))
        layer.bias.copy_(randn((48,), g))
    layer.process_filters()
    return layer, randn((9, 64), g, F16)


def load(layer):
    layer.load_state_dict({k: torch.flip(v, (0,)) for k, v in layer.state_dict().items()})


def optimizer_step(layer):
    for p in layer.parameters():
        p.grad = torch.ones_like(p)
    torch.optim.SGD(layer.parameters(), lr=1.0).step()


def new_data(layer):
    layer.weight.data = torch.flip(layer.weight.data, (0,))


def new_parameter(layer):
    layer.weight = torch.nn.Parameter(torch.flip(layer.weight.detach(), (0,)))


def in_place(layer):
    with torch.no_grad():
        layer.weight.mul_(-2)


def coarser_and_back(layer):
    layer.bfloat16().half()                 # eleven bits become eight: other values at what may be the old address


@pytest.mark.parametrize("change", [load, optimizer_step, new_data, new_parameter, in_place, coarser_and_back])
def test_a_packed_layer_answers_with_the_weight_it_has(change, packings):
    layer, x = packed_layer(1)
    with torch.no_grad():
        before = layer(x)
        assert len(packings) == 1, "a packed layer packs its weight once"
        change(layer)
        want = dc().mx4_linear(x, layer.weight, layer.bias)
        assert not torch.equal(want, before)
        assert torch.equal(layer(x), want)
        layer.process_filters()
        count = len(packings)
        assert torch.equal(layer(x), want) and len(packings) == count


def test_a_packed_layer_moves_and_copies(packings):
    layer, x = packed_layer(2)
    with torch.no_grad():
        want = layer(x)
        twin = copy.deepcopy(layer)
        count = len(packings)
        assert torch.equal(twin(x), want) and len(packings) == count        # a copy keeps what it has packed
        twin.weight.neg_()
        assert torch.equal(twin(x), dc().mx4_linear(x, twin.weight, twin.bias)) and torch.equal(layer(x), want)
        layer.cpu().cuda()
        assert torch.equal(layer(x), want)


def test_a_packed_layer_trains():
    """Packing does not take a layer out of training: input without a gradient (a first layer), frozen weights before an input
    that needs one, and both."""
    layer, x = packed_layer(3)
    dy = randn((9, 48), gen(4), F16)
    for x_grad, w_grad, b_grad in ((False, True, True), (False, False, True), (True, False, False), (True, True, True)):
        layer.weight.requires_grad_(w_grad), layer.bias.requires_grad_(b_grad)
        inputs = x.clone().requires_grad_(x_grad)
        leaves = [t for t in (inputs, layer.weight, layer.bias) if t.requires_grad]
        y = layer(inputs)
        assert y.requires_grad
        want = torch.autograd.grad(dc().mx4_linear(inputs, layer.weight, layer.bias), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))
    layer.requires_grad_(False)
    assert not layer(x).requires_grad


def test_a_packed_layer_under_inference_mode(packings):
    layer, x = packed_layer(5)
    want = layer(x).detach()
    count = len(packings)
    with torch.inference_mode():
        assert torch.equal(layer(x), want)
        born = dc().DCMX4Linear(64, 48).cuda().half()                           # its tensors keep no version
        born.weight.copy_(layer.weight), born.bias.copy_(layer.bias)
        born.process_filters()
        count += 1
        assert torch.equal(born(x), want)
    assert len(packings) == count
    with torch.no_grad():
        square = dc().DCMX4Linear(48, 48).cuda().half()
        square.process_filters()
        square.weight.data = square.weight.data.t()                             # the same memory, other strides: not the packed matrix
        with pytest.raises(RuntimeError, match="contiguous"):
            square(x[:, :48].contiguous())


# ---- tensors of other dimensions --------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(96,), (6, 7, 96), (2, 3, 2, 5, 96), (3, 96, 5, 7), (1, 96, 1, 1), (5, 96, 1, 1)])
def test_linear_of_other_dimensions(shape):
    d, g = dc(), gen(50)
    x = randn(shape, g, F16)
    w, b = randn((40, 96), g, F16).requires_grad_(), randn((40,), g, F16).requires_grad_()
    maps = len(shape) == 4
    out_shape = (shape[0], 40, *shape[2:]) if maps else (*shape[:-1], 40)
    dy = randn(out_shape, g, F16)                                               # maps: NCHW memory, brought into the layer's layout
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(-1, t.shape[1]) if maps else t.reshape(-1, t.shape[-1])      # noqa: E731
    x = (channels_last(x) if maps else x).requires_grad_()
    flat = rows(x.detach()).contiguous().requires_grad_()
    y, want = d.mx4_linear(x, w, b), d.mx4_linear(flat, w, b)
    assert y.shape == out_shape and torch.equal(rows(y), want)
    assert not maps or y.is_contiguous(memory_format=torch.channels_last)
    got = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    ref = torch.autograd.grad(want, (flat, w, b), rows(dy).contiguous())
    assert got[0].shape == shape and torch.equal(rows(got[0]), ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], ref[2])
    with torch.no_grad():
        assert torch.equal(d.mx4_linear(x, d.mx4_quantize(w), b), y)
        assert d.mx4_linear(x, d.mx4_quantize(w), b).stride() == y.stride()
    y.relu_()                                                                   # as an activation in place does


def test_linear_of_no_rows():
    x, w, b = torch.empty((0, 5, 64), device="cuda", requires_grad=True), torch.randn((8, 64), device="cuda", requires_grad=True), torch.randn(8, device="cuda", requires_grad=True)
    y = dc().mx4_linear(x, w, b)
    assert y.shape == (0, 5, 8)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all() and dw.shape == w.shape
    for t in torch.autograd.grad(dc().mx4_linear(torch.randn((3, 64), device="cuda"), w, b).sum(), (w, b)):
        assert t.isfinite().all()


# ---- what is not differentiated is refused ---------------------------------------------------------------------

def once_only(kind, g):
    """(function of x, x, what else it depends on) of an operator that is differentiable once."""
    x = randn((8, 64), g).requires_grad_()
    w, b = randn((64,), g).requires_grad_(), randn((64,), g).requires_grad_()
    m, c = randn((32, 64), g).requires_grad_(), randn((32,), g).requires_grad_()
    return {"norm": (lambda: dc().layer_norm(x, w, b), x, (w, b)), "bare norm": (lambda: dc().layer_norm(x), x, ()),
            "linear": (lambda: dc().mx4_linear(x, m, c), x, (m, c)), "frozen linear": (lambda: dc().mx4_linear(x, m.detach()), x, ()),
            "behind another": (lambda: dc().mx4_linear(dc().layer_norm(x * 2, w, b), m), x, (w, b, m))}[kind]


@pytest.mark.parametrize("through_dy", [False, True])
@pytest.mark.parametrize("kind", ["norm", "bare norm", "linear", "frozen linear", "behind another"])
def test_a_gradient_penalty_is_refused(kind, through_dy):
    """total = loss + |d loss / d x|^2 has a second-order term that these operators do not give: every way to ask for it raises."""
    f, x, others = once_only(kind, gen(10))

    def total():
        y = f()
        loss = y.square().sum() if through_dy else y.sum()
        g, = torch.autograd.grad(loss, x, create_graph=True)
        return loss + g.square().sum()

    if kind == "frozen linear" and not through_dy:          # its gradient depends on nothing that wants one: no second-order term
        assert torch.equal(torch.autograd.grad(total(), x)[0], torch.autograd.grad(f().sum(), x)[0])
        return
    for ask in (lambda t: torch.autograd.grad(t, x), lambda t: t.backward(), lambda t: torch.autograd.grad(t, (x, *others), allow_unused=True)):
        t = total()
        with pytest.raises(RuntimeError, match="differentiable once"):
            ask(t)


@pytest.mark.parametrize("kind", ["norm", "linear"])
def test_first_gradients_under_create_graph(kind):
    f, x, others = once_only(kind, gen(11))
    leaves = (x, *others)
    dy = randn(f().shape, gen(12))
    want = torch.autograd.grad(f(), leaves, dy)
    got = torch.autograd.grad(f(), leaves, dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(p.requires_grad for p in got)
    for p in got:                                  # each of them knows that it depends on x
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(p.sum(), x, retain_graph=True)


def test_forward_mode_tangents_are_refused():
    """A tangent that nothing carries on would read as a derivative of zero."""
    import torch.autograd.forward_ad as fwd
    d, g = dc(), gen(13)
    x, w, m, c = randn((6, 64), g), randn((64,), g), randn((32, 64), g), randn((32,), g)
    q = d.mx4_quantize(m)
    cl = channels_last(randn((1, 64, 4, 4), g))
    mask = torch.ones((1, 1, 4, 4), dtype=torch.int32, device="cuda")
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))      # noqa: E731
        calls = [lambda: d.layer_norm(dual(x)), lambda: d.layer_norm(x, dual(w)), lambda: d.layer_norm(x, w, dual(w)),
                 lambda: d.layer_norm(dual(x.clone().requires_grad_()), w),
                 lambda: d.mx4_linear(dual(x), m), lambda: d.mx4_linear(x, dual(m)), lambda: d.mx4_linear(x, q, dual(c)), lambda: d.mx4_linear(dual(x), q),
                 lambda: d.mx4_quantize(dual(x)), lambda: d.mx4_quantize_both(dual(x)), lambda: d.mx4_matmul(d.mx4_quantize(x), q, dual(c)),
                 lambda: d.layer_norm_delta(dual(cl), mask, cl.clone(), cl.clone()), lambda: d.layer_norm_delta(cl, mask, cl.clone(), cl.clone(), dual(w)),
                 lambda: d.DCLayerNorm(64).cuda()((dual(cl), mask))]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was not refused")
        inside = d.mx4_linear(d.layer_norm(x, w), m, c)             # nothing dual about it
    assert torch.equal(inside, d.mx4_linear(d.layer_norm(x, w), m, c))


# ---- saved tensors ---------------------------------------------------------------------------------------------

def map_step(g):
    """A map's norm and linear layer with their gradients."""
    x, w, b = channels_last(randn((2, 32, 5, 7), g)).requires_grad_(), randn((32,), g).requires_grad_(), randn((32,), g).requires_grad_()
    m = randn((24, 32), g).requires_grad_()

    def run():
        y = dc().mx4_linear(dc().layer_norm(x, w, b), m)
        return (y, *torch.autograd.grad(y.square().sum(), (x, w, b, m)))
    return run


def in_other_memory(t):
    """The same values where offloading may leave them: another layout, another address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return flat[1:].view(t.shape).copy_(t.detach())


def test_saved_tensors_may_be_moved():
    run = map_step(gen(20))
    want = run()
    for hooks in (torch.autograd.graph.saved_tensors_hooks(in_other_memory, lambda t: t), torch.autograd.graph.save_on_cpu(),
                  torch.autograd.graph.save_on_cpu(pin_memory=True)):
        with hooks:
            got = run()
        # other addresses, so other widths of access and another order of float32 sums: of 70 rows or 32 channels of values of order
        # one, a few hundred in dx's and dw's own sums
        for p, q in zip(got, want):
            assert (p - q).abs().max() <= 2.0 ** -24 * 200 * q.abs().max()


def test_what_the_linear_layer_keeps_is_seen_and_freed():
    g = gen(21)
    x, w = randn((300, 256), g).requires_grad_(), randn((128, 256), g).requires_grad_()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.numel() * t.element_size()) or t, lambda t: t):
        y = dc().mx4_linear(x, w)
    packed = sum(r * -(-c // 32) * 16 + -(-r // 128) * -(-c // 128) * 512 for r, c in ((256, 300), (256, 128)))
    assert packed in seen
    y = dc().mx4_linear(x, w)
    before = torch.cuda.memory_allocated()
    y.sum().backward(inputs=[x])
    assert torch.cuda.memory_allocated() <= before + 300 * 256 * 4 - packed + 4096          # x.grad came, the packed matrices went
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward(inputs=[x])


def test_checkpointed_block():
    from torch.utils.checkpoint import checkpoint
    g = gen(22)
    x, w, b, m = (randn(s, g).requires_grad_() for s in ((40, 64), (64,), (64,), (64, 64)))

    def block(v):
        return dc().mx4_linear(dc().layer_norm(v, w, b), m)
    want = torch.autograd.grad(block(block(x)).square().sum(), (x, w, b, m))
    got = torch.autograd.grad(checkpoint(block, checkpoint(block, x, use_reentrant=False), use_reentrant=False).square().sum(), (x, w, b, m))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


# ---- widths ----------------------------------------------------------------------------------------------------

FRESH = """
import torch, deltacnn_b200 as dc
torch.manual_seed(0)
t = torch.{dtype}
x, dy = torch.randn(5, {c}, device="cuda").to(t), torch.randn(5, {c}, device="cuda").to(t)
w, b = torch.randn({c}, device="cuda").to(t), torch.randn({c}, device="cuda").to(t)
x64, w64 = x.double(), w.double()
n = (x64 - x64.mean(-1, keepdim=True)) / (x64.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
u = torch.finfo(t).eps / 2
y64 = n * w64 + b.double()
# one rounding at the end, and 64 steps of float32 in sums of values of order ten at most
assert ((dc.layer_norm(x, w, b) - y64).abs() <= u * y64.abs() + 64 * 2.0 ** -24 * 10).all()
if {train}:
    leaves = [v.requires_grad_() for v in (x, w, b)]
    dx, dw, db = torch.autograd.grad(dc.layer_norm(*leaves), leaves, dy)
    db64 = dy.double().sum(0)
    assert ((db - db64).abs() <= u * db64.abs() + 64 * 2.0 ** -24 * 10).all() and dx.isfinite().all() and dw.isfinite().all()
torch.cuda.synchronize()
"""


@pytest.mark.parametrize("dtype,c,train", [("float16", 6000, False), ("bfloat16", 5640, False), ("float32", 2900, False), ("float16", 2600, True),
                                           ("bfloat16", 3000, True), ("float32", 1500, True), ("float32", 1284, True)])
def test_a_width_is_taken_whatever_ran_before(dtype, c, train):
    """Rows whose ring fills 48 KB of shared memory exactly, as the first call of a process: no wider row has asked for more yet."""
    run = subprocess.run([sys.executable, "-c", FRESH.format(dtype=dtype, c=c, train=train)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-1500:]


# ---- the delta norm in a network -------------------------------------------------------------------------------

def frames(g, dtype, n=4, shape=(2, 24, 9, 7)):
    frame = channels_last(randn(shape, g, dtype))
    for t in range(n):
        yield frame
        frame = frame.clone(memory_format=torch.preserve_format)
        frame[:, :, t:t + 3, 1:4] += randn((*shape[:2], 3, 3), g, dtype)


def norm_layer(g, dtype, channels=24, **args):
    ln = dc().DCLayerNorm(channels, delta_threshold=0.0, **args).cuda().to(dtype)
    with torch.no_grad():
        ln.weight.copy_(randn((channels,), g, dtype, 0.2, 1.0))
        ln.bias.copy_(randn((channels,), g, dtype))
    return ln


@pytest.mark.parametrize("dtype", [F32, F16])
def test_delta_norm_beside_a_skip_connection(dtype):
    """x + norm(x), the norm's usual place, over some frames against the dense block."""
    d, g = dc(), gen(30)
    sp, ln, add, de = d.DCSparsify(delta_threshold=0.0), norm_layer(g, dtype), d.DCAdd(), d.DCDensify()
    with torch.no_grad():
        for t, frame in enumerate(frames(g, dtype)):
            x = sp(frame.clone(memory_format=torch.preserve_format))
            held = [v.clone() for v in x]
            y = ln(x)
            for p, q in zip(x, held):                                           # bits: what lies at pixels without a mask may be a NaN
                whole = {2: torch.int16, 4: torch.int32}[p.element_size()]
                assert torch.equal(p.view(whole), q.view(whole)), "the norm wrote to its input"
            got = de(add(x, y))
            want = frame.double() + d.layer_norm(frame, ln.weight, ln.bias, EPS).double()
            # a frame rounds the two inputs' sums, the norm, its change, the add and the sum of adds: six values below 16
            assert (got.double() - want).abs().max().item() <= 6 * (t + 1) * 16 * torch.finfo(dtype).eps / 2


def test_delta_norm_behind_a_convolution():
    """The convolution's own output buffer is read again by a skip behind the norm. Weights of one power of two per output: exact."""
    d, g = dc(), gen(31)
    conv = d.DCConv2d(24, 24, 1, bias=False).cuda().half()
    with torch.no_grad():
        conv.weight.copy_(torch.eye(24, device="cuda").flip(0)[:, :, None, None] * 0.5)
    model = torch.nn.ModuleList([conv])
    conv.to(memory_format=torch.channels_last)
    for c in model:
        c.process_filters()
    sp, ln, add, de = d.DCSparsify(delta_threshold=0.0), norm_layer(g, F16), d.DCAdd(), d.DCDensify()
    with torch.no_grad():
        for t, frame in enumerate(frames(g, F16)):
            x = conv(sp(frame.clone(memory_format=torch.preserve_format)))
            got = de(add(x, ln(x)))
            dense = channels_last(frame.flip(1) * 0.5)
            want = dense.double() + d.layer_norm(dense, ln.weight, ln.bias, EPS).double()
            assert (got.double() - want).abs().max().item() <= 6 * (t + 1) * 16 * torch.finfo(F16).eps / 2


@pytest.mark.parametrize("reuse", [False, True])
def test_delta_norm_in_place_and_in_buffers_of_its_own(reuse, monkeypatch):
    d = dc()
    monkeypatch.setattr(d.DCConv2d, "reuse_buffers", reuse)
    a, b = norm_layer(gen(32), F16), norm_layer(gen(32), F16, inplace=True)
    sp, outs = d.DCSparsify(delta_threshold=0.0), []
    with torch.no_grad():
        for t, frame in enumerate(frames(gen(33), F16)):
            val, mask = (v.clone() for v in sp(frame.clone(memory_format=torch.preserve_format)))
            out, out_mask = a((val, mask))
            outs.append(out.data_ptr())
            mine, mine_mask = b((val, mask))
            assert t == 0 or (mine is val and mine_mask is mask)
            on = (out_mask != 0).expand_as(out)
            assert torch.equal(out_mask, mine_mask) and torch.equal(out[on], mine[on])
            assert torch.equal(a.prev_in, b.prev_in) and torch.equal(a.prev_out, b.prev_out)
            if t == 0 or not reuse:
                kept = out, out_mask                        # still referenced: a new tensor cannot stand where it does
    assert (len(set(outs)) == 1) if reuse else (outs[-1] != outs[-2])
    with pytest.raises(RuntimeError, match="reset_layers"):
        a((channels_last(torch.zeros((3, 24, 9, 7), dtype=F16, device="cuda")), torch.ones((3, 1, 9, 7), dtype=torch.int32, device="cuda")))
    a.reset()
    val = channels_last(randn((3, 24, 4, 4), gen(34), F16))
    with torch.no_grad():
        assert torch.equal(a((val, torch.ones((3, 1, 4, 4), dtype=torch.int32, device="cuda")))[0], d.layer_norm(val, a.weight, a.bias, EPS))


def test_delta_norm_replayed_from_a_graph():
    d, g = dc(), gen(35)
    sp, ln, add, de = d.DCSparsify(delta_threshold=0.0), norm_layer(g, F16), d.DCAdd(), d.DCDensify()
    sequence = list(frames(g, F16, 6))
    static = sequence[0].clone(memory_format=torch.preserve_format)

    def block():
        x = sp(static)
        return de(add(x, ln(x)))

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for frame in sequence[:2]:
                static.copy_(frame)
                block()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block()
        for t, frame in enumerate(sequence[2:], 2):
            static.copy_(frame)
            graph.replay()
            want = frame.double() + d.layer_norm(frame, ln.weight, ln.bias, EPS).double()
            assert (out.double() - want).abs().max().item() <= 6 * (t + 1) * 16 * torch.finfo(F16).eps / 2


@pytest.mark.parametrize("dtype,shape", [(F16, (8, 96, 160, 160)), (F32, (4, 101, 130, 160)), (F16, (4, 82, 130, 160)), (F16, (2, 1200, 9, 7)), (F32, (1, 2000, 9, 7))])
def test_an_unchanged_pixel_leaves_the_mask(dtype, shape):
    """At threshold 0 a masked pixel whose delta is 0 has no change, from the first frame on: the first frame's norm has to be the
    delta form's own, bit for bit, on maps of many pixels too."""
    g = gen(40)
    ln = norm_layer(g, dtype, shape[1])
    frame = channels_last(randn(shape, g, dtype, 1.5, 0.7))
    ones = torch.ones((shape[0], 1, *shape[2:]), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        first, mask = ln((frame, ones))
        assert (mask == 1).all() and torch.equal(first, ln.prev_out)
        first = first.clone()
        _, mask = ln((torch.zeros_like(frame), ones.clone()))
        assert int(mask.sum()) == 0
        assert torch.equal(ln.prev_out, first) and torch.equal(ln.prev_in, frame)


def test_first_frame_of_hard_values_and_refusals():
    d, g = dc(), gen(41)
    ln = norm_layer(g, F32)
    frame = channels_last(randn((1, 24, 2, 3), g))
    frame[0, 3, 0, 0], frame[0, 5, 1, 1], frame[0, :, 0, 2] = float("nan"), float("inf"), 2.0
    ones = torch.ones((1, 1, 2, 3), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y = ln((frame, ones))[0]
    assert y[0, :, 0, 0].isnan().all() and y[0, :, 1, 1].isnan().all() and torch.equal(y[0, :, 0, 2], ln.bias)
    assert int(y.isnan().sum()) == 48
    for bad in (torch.zeros((1, 24, 2, 3), device="cuda"), channels_last(torch.zeros((1, 24, 2, 3), device="cuda").bfloat16()),
                channels_last(torch.zeros((1, 25, 2, 3), device="cuda"))):
        with pytest.raises(RuntimeError):
            norm_layer(g, F32)((bad, ones))
    wide = norm_layer(g, F32, 9001)
    with pytest.raises(RuntimeError):                                           # no delta kernel for so many channels: at once, not a frame later
        wide((channels_last(torch.zeros((1, 9001, 1, 1), device="cuda")), torch.ones((1, 1, 1, 1), dtype=torch.int32, device="cuda")))
    assert wide.first_iter and d.layer_norm(torch.zeros((2, 9001), device="cuda"), wide.weight, wide.bias).shape == (2, 9001)


def test_a_first_frame_through_the_delta_call_itself():
    """From caches of zeros, as the call documents: the same norm, and nothing changes behind it."""
    d, g = dc(), gen(42)
    x, w, b = channels_last(randn((2, 96, 40, 50), g, F16)), randn((96,), g, F16), randn((96,), g, F16)
    ones = torch.ones((2, 1, 40, 50), dtype=torch.int32, device="cuda")
    prev_in, prev_out = torch.zeros_like(x), torch.zeros_like(x)
    out, mask = d.layer_norm_delta(x, ones, prev_in, prev_out, w, b)
    ln = norm_layer(g, F16, 96)
    with torch.no_grad():
        ln.weight.copy_(w), ln.bias.copy_(b)
        first = ln((x, ones))[0]
    assert torch.equal(out, first) and torch.equal(prev_out, first) and torch.equal(prev_in, x) and int(mask.sum()) == mask.numel()
    assert int(d.layer_norm_delta(torch.zeros_like(x), ones, prev_in, prev_out, w, b)[1].sum()) == 0


# ---- tensors of many rows, of float32 weights, of more than 2^31 elements --------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,c", [(160001, 24), (80001, 96), (30000, 512), (20000, 101), (19001, 33), (20000, 25), (1500, 8), (16001, 1000), (4097, 2600),
                                    (5001, 255), (4800, 129), (5000, 202), (700, 257), (2100, 5000), (1000, 9006), (450, 8200), (901, 12001), (333, 20000)])
def test_no_row_is_missing_from_the_column_sums(rows, c, dtype):
    """Odd whole numbers over mean 0 and rstd 1/2: every term is a multiple of 1/2, every sum below 2^24 of them, so float32 holds all of
    them exactly in any order, and one row that is missing or counted twice changes every column."""
    g = gen(rows)
    odd = lambda: (torch.randint(0, 4, (rows, c), generator=g, device="cuda") * 2 - 3).to(dtype)      # noqa: E731  -3, -1, 1, 3
    x, dy = odd(), odd()
    mean, rstd = torch.zeros(rows, device="cuda"), torch.full((rows,), 0.5, device="cuda")
    lib, code = dc()._lib.lib, {F32: 0, F16: 1, BF16: 2}[dtype]
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    ws = torch.empty(lib.dc_layer_norm_backward_workspace_bytes(rows, c, code), dtype=torch.uint8, device="cuda")
    dx = torch.empty_like(x)
    for d in (dx.data_ptr(), None):
        dw.fill_(-1), db.fill_(-1)
        assert lib.dc_layer_norm_backward(dy.data_ptr(), x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), d, dw.data_ptr(), db.data_ptr(), rows, c, code, 0,
                                          ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(db.double(), dy.double().sum(0)) and torch.equal(dw.double(), (dy.double() * x.double() * 0.5).sum(0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(8200, 130, 64), (4100, 2051, 40), (129, 33, 96)])
def test_no_row_is_missing_from_the_bias_gradient(m, n, k, dtype):
    g = gen(m)
    x, w, b = randn((m, k), g, dtype), randn((n, k), g, dtype), torch.zeros(n, device="cuda", requires_grad=True)
    dy = (torch.randint(0, 4, (m, n), generator=g, device="cuda") * 2 - 3).to(dtype)
    assert torch.equal(torch.autograd.grad(dc().mx4_linear(x, w, b), b, dy)[0].double(), dy.double().sum(0))


@pytest.mark.parametrize("inplace", [False, True])
def test_delta_norm_with_float32_weights_on_half_maps(inplace):
    d, g = dc(), gen(51)
    ln = d.DCLayerNorm(24, delta_threshold=0.0, inplace=inplace).cuda()
    with torch.no_grad():
        ln.weight.copy_(randn((24,), g, F32, 0.2, 1.0))
        ln.bias.copy_(randn((24,), g))
        sp, de = d.DCSparsify(delta_threshold=0.0), d.DCDensify()
        for t, frame in enumerate(frames(g, F16)):
            got = de(ln(sp(frame.clone(memory_format=torch.preserve_format))))
            want = d.layer_norm(frame, ln.weight, ln.bias, EPS)
            # per frame the accumulated input, the norm, its change and the accumulated output are rounded: four values below 16
            assert (got.double() - want.double()).abs().max().item() <= 4 * (t + 1) * 16 * torch.finfo(F16).eps / 2


# 4096 channels: 524288 rows are 2^31 elements
LONG = 524288 + 515


def test_layer_norm_of_more_than_2_31_elements():
    d, g = dc(), gen(52)
    x = torch.empty((LONG, 4096), dtype=BF16, device="cuda").normal_(generator=g).requires_grad_()
    dy = torch.empty_like(x, requires_grad=False).random_(0, 4, generator=g).mul_(2).sub_(3)          # odd whole numbers: db is exact
    w, b = randn((4096,), g).requires_grad_(), randn((4096,), g).requires_grad_()
    y = d.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(db.double(), dy.sum(0, dtype=torch.float64)) and dw.isfinite().all()
    for part in (slice(0, 515), slice(LONG // 2, LONG // 2 + 515), slice(LONG - 515, LONG)):
        xs = x.detach()[part].clone().requires_grad_()
        ys = d.layer_norm(xs, w, b)
        assert torch.equal(ys, y[part])
        assert torch.equal(torch.autograd.grad(ys, xs, dy[part])[0], dx[part])


def test_delta_norm_of_more_than_2_31_elements():
    d, g = dc(), gen(53)
    shape = (8, 64, 2048, 2052)                                                 # 2^31 and 2^22 elements
    delta = torch.empty(shape, dtype=F16, device="cuda", memory_format=torch.channels_last).normal_(generator=g)
    prev_in = torch.zeros_like(delta)
    prev_out = torch.zeros_like(delta)
    mask = (torch.rand((8, 1, 2048, 2052), generator=g, device="cuda") < 0.3).int()
    w, b = randn((64,), g, F16), randn((64,), g, F16)
    part = [t[-1:, :, -3:].clone(memory_format=torch.channels_last) for t in (delta, prev_in, prev_out)]
    small = d.layer_norm_delta(part[0], mask[-1:, :, -3:].clone(), part[1], part[2], w, b, 0.1)
    out, out_mask = d.layer_norm_delta(delta, mask, prev_in, prev_out, w, b, 0.1, out=delta)
    on = (small[1] != 0).expand_as(small[0])
    assert torch.equal(out_mask[-1:, :, -3:], small[1]) and torch.equal(out[-1:, :, -3:][on], small[0][on])
    assert torch.equal(prev_in[-1:, :, -3:], part[1]) and torch.equal(prev_out[-1:, :, -3:], part[2])
    assert torch.equal(out_mask != 0, mask != 0)                                # from nothing every masked pixel changes


def scale_rows(q, first):
    """The scale bytes of the rows from `first`, a multiple of 128, on (those behind the last row are not written)."""
    s = q.scales[first // 128:].permute(0, 3, 2, 1, 4)
    return s.reshape(-1, s.shape[3] * 4)[:q.shape[0] - first]


def test_mx4_of_more_than_2_31_elements():
    d, g = dc(), gen(54)
    x = torch.empty((LONG, 4096), dtype=BF16, device="cuda").normal_(generator=g)
    q = d.mx4_quantize(x)
    tail = LONG // 128 * 128 - 128
    part = d.mx4_quantize(x[tail:])
    assert torch.equal(q.data[tail:], part.data) and torch.equal(scale_rows(q, tail), scale_rows(part, 0))
    both, both_t = d.mx4_quantize_both(x)
    assert torch.equal(both.data, q.data) and torch.equal(scale_rows(both, 0), scale_rows(q, 0))
    part_t = d.mx4_quantize_both(x[tail:])[1]
    assert torch.equal(both_t.data[:, tail // 2:], part_t.data)
    del both, both_t
    assert torch.equal(d.mx4_dequantize(q, BF16)[tail:], d.mx4_dequantize(part, BF16))
    del x
    w = d.mx4_quantize(randn((8, 4096), g))
    assert torch.equal(d.mx4_matmul(q, w, None, BF16)[tail:], d.mx4_matmul(part, w, None, BF16))
    wide, few = d.mx4_quantize(randn((4100, 64), g)), d.mx4_quantize(randn((LONG, 64), g))
    out = d.mx4_matmul(few, wide, None, BF16)                                   # more than 2^31 results
    end = d.mx4_matmul(d.mx4_quantize(d.mx4_dequantize(few)[tail:]), wide, None, BF16)
    assert torch.equal(out[tail:], end)


def test_delta_norm_is_counted_the_same_in_place_or_not(monkeypatch):
    from deltacnn_b200.cuda_kernels import DCPerformanceMetricsManager as M
    counted = []
    for inplace in (False, True):
        ln, sp = norm_layer(gen(60), F16, inplace=inplace), dc().DCSparsify(delta_threshold=0.0)
        M.reset()
        with torch.no_grad():
            for frame in frames(gen(61), F16):
                val, mask = (v.clone() for v in sp(frame.clone(memory_format=torch.preserve_format)))
                monkeypatch.setattr(M, "enabled", True)                         # the norm alone
                ln((val, mask))
                monkeypatch.setattr(M, "enabled", False)
        counted.append(vars(M.get_metrics()))
        M.reset()
    assert counted[0] == counted[1] and counted[0]["mem_write_actual"] > 0
