"""Layer norm (forward, backward, delta form) and the MXFP4 operators against plain 64-bit implementations, at the sizes,
types, values and calls where they can go wrong.

Tolerances count roundings: u = 2^-24 is half a step of float32, ``half(t)`` half a step of the result's type relative to the
value (the one rounding at the end). A float32 sum of n terms in any order is off by at most n u sum|term|; the kernels' sums
are trees (at most 48 additions deep over a row), column sums at most ``rows`` deep."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
U = 2.0 ** -24
EPS = 1e-5


def dc():
    import deltacnn_b200
    return deltacnn_b200


def half(t):
    return torch.finfo(t).eps / 2


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere, bound in 64 bits (plus what the smallest steps of the result's type cost)."""
    got64 = got.double()
    assert got64.shape == want.shape
    tiny = torch.finfo(got.dtype).tiny * half(got.dtype) * 2
    bad = ~((got64 - want).abs() <= bound + tiny)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got64 - want).abs() / (bound + tiny)).max().item():.3g} x the bound"


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def norm64(x, w, b, eps=EPS):
    """y, n, r and what rounding errors of x - m scale with, in 64 bits (rows x C)."""
    x = x.double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    n = (x - m) * r
    a = (x.abs().mean(-1, keepdim=True) + m.abs()) * r          # size of the cancelling terms in units of n
    return n * w + b, n, r, a


def y_bound(w, b, n, a, y, t):
    # x - m: m is off by at most 50 u mean|x|, the difference by one more rounding; r: the sum of squares 50 u and what m's
    # error adds, then sqrt and division; the product, the affine step: a few more
    return 64 * U * ((a + n.abs() * (1 + a)) * w.abs() + b.abs()) + half(t) * y.abs()


# ---- layer norm ------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (5, 1), (1, 8), (3, 7), (40, 24), (5, 33), (259, 64), (2, 96), (130, 100), (33, 1000), (7, 1024), (3, 1032), (6, 1001),
          (2, 4096), (3, 4100), (2, 4099), (2, 8192), (3, 16384), (2, 20000), (1, 40000), (1500, 8), (700, 257),
          (2, 9001), (3, 2500), (2, 10000), (300, 50), (90, 82), (41, 170), (77, 430), (5, 514), (3, 8190), (2, 8194), (9, 2), (1, 8193), (17, 12001), (1000, 9006), (450, 8200), (100, 10240), (5, 16392), (3, 60001), (2, 120000), (80001, 96), (160001, 24), (30000, 512), (20000, 101), (19001, 33), (5000, 202), (5001, 255), (20000, 25), (4800, 129)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", SHAPES)
def test_layer_norm_forward_and_backward(rows, c, dtype):
    g = gen(rows * 31 + c)
    x, dy = randn((rows, c), g, dtype, 1.5, 0.7), randn((rows, c), g, dtype)
    w, b = randn((c,), g, dtype, 0.3, 1.0), randn((c,), g, dtype)
    y64, n, r, a = norm64(x, w.double(), b.double())
    plain = dc().layer_norm(x, w, b, EPS)
    within(plain, y64, y_bound(w.double(), b.double(), n, a, y64, dtype), "y")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = dc().layer_norm(*leaves, EPS)
    assert torch.equal(y, plain)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    d, w64 = dy.double(), w.double()
    q = d * w64
    mq, mqn = q.mean(-1, keepdim=True), (q * n).mean(-1, keepdim=True)
    aq, aqn = q.abs().mean(-1, keepdim=True), (q * n).abs().mean(-1, keepdim=True)
    dx64 = r * (q - mq - n * mqn)
    within(dx, dx64, 64 * U * r * (1 + a) * (q.abs() + aq + (n.abs() + 1) * (aqn + aq)) + half(dtype) * dx64.abs(), "dx")
    dw64, db64 = (d * n).sum(0), d.sum(0)
    within(dw, dw64, (64 + rows) * U * (d.abs() * (n.abs() + (1 + n.abs()) * a)).sum(0) + half(dtype) * dw64.abs(), "dw")
    within(db, db64, (64 + rows) * U * d.abs().sum(0) + half(dtype) * db64.abs(), "db")
    again = torch.autograd.grad(dc().layer_norm(*leaves, EPS), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db))), "the same inputs give other bits"


@pytest.mark.parametrize("c", [32, 1000, 4096])
def test_layer_norm_gradient_against_differences(c):
    g = gen(c)
    x, w, b = randn((6, c), g), randn((c,), g, shift=1.0), randn((c,), g)
    dy = randn((6, c), g)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(dc().layer_norm(*leaves, EPS), leaves, dy)
    h = 1e-5
    for i, gr in enumerate(grads):
        v = randn(leaves[i].shape, g).double()
        f = []
        for s in (h, -h):
            t = [x.double(), w.double(), b.double()]
            t[i] = t[i] + s * v
            f.append((norm64(t[0], t[1], t[2])[0] * dy.double()).sum().item())
        want = (f[0] - f[1]) / (2 * h)
        # central differences: h^2 times third derivatives of order one per element, and 64-bit roundings over h; the kernel:
        # the 64 u of the test above per element
        size = (gr.double() * v).abs().sum().item()
        assert abs((gr.double() * v).sum().item() - want) <= (64 * U * 8 + 1e-7) * (size + dy.double().abs().sum().item())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_layer_norm_with_float32_weights(dtype):
    g = gen(3)
    x, dy = randn((70, 264), g, dtype), randn((70, 264), g, dtype)
    w, b = randn((264,), g, shift=1.0).requires_grad_(), randn((264,), g).requires_grad_()
    y = dc().layer_norm(x, w, b, EPS)
    y64, n, r, a = norm64(x, w.detach().double(), b.detach().double())
    within(y.detach(), y64, y_bound(w.detach().double(), b.detach().double(), n, a, y64, dtype))
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert dw.dtype == F32 and db.dtype == F32
    d = dy.double()
    within(dw, (d * n).sum(0), 140 * U * (d.abs() * (n.abs() + (1 + n.abs()) * a)).sum(0))
    within(db, d.sum(0), 140 * U * d.abs().sum(0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,c", [(5, 1000), (70, 9001), (70, 9002), (33, 20000)])
def test_layer_norm_gradients_alone_are_those_together(rows, c, dtype):
    g = gen(c)
    x, dy = randn((rows, c), g, dtype), randn((rows, c), g, dtype)
    w, b = randn((c,), g, F32, 0.3, 1.0), randn((c,), g)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    together = torch.autograd.grad(dc().layer_norm(*leaves, EPS), leaves, dy)
    for i in range(3):
        parts = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(dc().layer_norm(*parts, EPS), parts[i], dy)[0], together[i])
    bare = x.detach().requires_grad_()
    unit = x.detach().requires_grad_()
    plain = torch.autograd.grad(dc().layer_norm(bare, eps=EPS), bare, dy)[0]
    assert torch.equal(plain, torch.autograd.grad(dc().layer_norm(unit, torch.ones(c, device="cuda"), eps=EPS), unit, dy)[0])


@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(with_w, with_b):
    g = gen(4)
    x = randn((9, 72), g).requires_grad_()
    w = randn((72,), g).requires_grad_() if with_w else None
    b = randn((72,), g).requires_grad_() if with_b else None
    y = dc().layer_norm(x, w, b, EPS)
    w64, b64 = (w.detach().double() if with_w else torch.ones(72, device="cuda").double()), (b.detach().double() if with_b else torch.zeros(72, device="cuda").double())
    y64, n, r, a = norm64(x.detach(), w64, b64)
    within(y.detach(), y64, y_bound(w64, b64, n, a, y64, F32))
    ones = torch.ones_like(y)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, ones)))
    if with_w:
        within(grads[id(w)], n.sum(0), 80 * U * (n.abs() + (1 + n.abs()) * a).sum(0))
    if with_b:
        within(grads[id(b)], torch.full((72,), 9.0, device="cuda").double(), torch.zeros(72, device="cuda").double())
    q = w64.expand_as(n)
    dx64 = r * (q - q.mean(-1, keepdim=True) - n * (q * n).mean(-1, keepdim=True))
    within(grads[id(x)], dx64, 64 * U * r * (1 + a) * (q.abs() + q.abs().mean(-1, keepdim=True) + (n.abs() + 1) * ((q * n).abs().mean(-1, keepdim=True) + q.abs().mean(-1, keepdim=True))))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_of_a_feature_map_is_per_pixel(dtype):
    g = gen(5)
    x = randn((3, 40, 5, 7), g, dtype).contiguous(memory_format=torch.channels_last).requires_grad_()
    w = randn((40,), g, dtype).requires_grad_()
    y = dc().layer_norm(x, w, None, EPS)
    assert y.is_contiguous(memory_format=torch.channels_last)
    flat = x.detach().permute(0, 2, 3, 1).reshape(-1, 40).requires_grad_()
    wf = w.detach().clone().requires_grad_()
    yf = dc().layer_norm(flat, wf, None, EPS)
    assert torch.equal(y.detach().permute(0, 2, 3, 1).reshape(-1, 40), yf.detach())
    dy = randn((3, 40, 5, 7), g, dtype)                       # NCHW memory: brought into x's layout
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    dxf, dwf = torch.autograd.grad(yf, (flat, wf), dy.permute(0, 2, 3, 1).reshape(-1, 40))
    assert torch.equal(dx.permute(0, 2, 3, 1).reshape(-1, 40), dxf) and torch.equal(dw, dwf)


def test_gradients_of_gradients_are_refused():
    g = gen(30)
    x, w = randn((8, 64), g).requires_grad_(), randn((64,), g).requires_grad_()
    for f in (lambda: dc().layer_norm(x, w), lambda: dc().mx4_linear(x, w.expand(32, 64).contiguous())):
        first, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.square().sum(), x)


def test_layer_norm_hard_values():
    g = gen(6)
    x = randn((8, 64), g)
    x[0] = 3.0                              # no variance: the bias
    x[1] = 0.0
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4] = x[4] * 1e-3 + 1e4                # a mean far above the spread
    x[5] *= 1e15
    w, b = randn((64,), g), randn((64,), g)
    y = dc().layer_norm(x, w, b, EPS)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    assert y[2].isnan().all() and y[3].isnan().all()
    y64, n, r, a = norm64(x, w.double(), b.double())
    for i in (4, 5, 6, 7):
        within(y[i], y64[i], y_bound(w.double(), b.double(), n, a, y64, F32)[i])


def test_layer_norm_unaligned_rows_and_empty_input():
    g = gen(7)
    base = randn((1 + 5 * 64,), g)
    x = base[1:].view(5, 64)                # contiguous, four bytes off
    w, b = randn((64,), g), randn((64,), g)
    y64, n, r, a = norm64(x, w.double(), b.double())
    within(dc().layer_norm(x, w, b), y64, y_bound(w.double(), b.double(), n, a, y64, F32))
    for off in (1, 2):                      # halves two and four bytes off, with a gradient of another alignment
        h = randn((off + 6 * 72,), g, F16)[off:].view(6, 72).requires_grad_()
        wh = randn((72,), g, F16).requires_grad_()
        dy = randn((3 - off + 6 * 72,), g, F16)[3 - off:].view(6, 72)
        got = torch.autograd.grad(dc().layer_norm(h, wh), (h, wh), dy)
        want = torch.autograd.grad(dc().layer_norm(h2 := h.detach().clone().requires_grad_(), w2 := wh.detach().clone().requires_grad_()), (h2, w2), dy.clone())
        for p, q in zip(got, want):         # the same sums in another order, rounded once
            assert (p.float() - q.float()).abs().max() <= 2 * half(F16) * q.float().abs().max() + 1e-4
    e = torch.empty((0, 64), device="cuda", requires_grad=True)
    w.requires_grad_(), b.requires_grad_()
    dx, dw, db = torch.autograd.grad(dc().layer_norm(e, w, b).sum(), (e, w, b))
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_layer_norm_partial_gradients_and_expanded_gradient():
    g = gen(8)
    x, w, b = (randn(s, g).requires_grad_() for s in ((17, 48), (48,), (48,)))
    full = torch.autograd.grad(dc().layer_norm(x, w, b).sum(), (x, w, b))       # sum's gradient is an expanded scalar
    for i, t in enumerate((x, w, b)):
        args = [s.detach() for s in (x, w, b)]
        args[i] = t
        assert torch.equal(torch.autograd.grad(dc().layer_norm(*args).sum(), t)[0], full[i])


def delta64(delta, mask, prev_in, prev_out, w, b, thr):
    """The delta form with the storage type's roundings, in N,H,W,C order."""
    t = delta.dtype
    on = (mask != 0)[..., None]
    u = torch.where(on, (prev_in.double() + delta.double()).to(t), prev_in)
    y64, n, r, a = norm64(u, w.double(), b.double())
    e = y64 - prev_out.double()
    keep = on & (e.abs() > thr).any(-1, keepdim=True)
    return u, y64, e, keep, n, a


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n,h,w,c", [(1, 1, 1, 8), (2, 5, 7, 24), (3, 9, 11, 64), (1, 16, 16, 100), (2, 6, 6, 576), (1, 5, 5, 1280), (1, 3, 5, 33), (1, 3, 3, 1001), (1, 2, 3, 4096), (1, 2, 3, 8191), (1, 1, 2, 8192), (40, 30, 30, 72), (3, 9, 9, 82), (2, 7, 7, 212), (1, 6, 5, 430), (1, 3, 3, 1002), (1, 2, 2, 8190)])
@pytest.mark.parametrize("density", [0.0, 0.3, 1.0])
def test_layer_norm_delta(dtype, n, h, w, c, density):
    g = gen(c + int(density * 10))
    cl = lambda t: t.permute(0, 3, 1, 2)                                       # noqa: E731  N,H,W,C memory
    prev_in, wt, b = randn((n, h, w, c), g, dtype), randn((c,), g, dtype, 0.2, 1.0), randn((c,), g, dtype)
    prev_out = norm64(prev_in, wt.double(), b.double())[0].to(dtype)
    mask = (torch.rand((n, h, w), generator=g, device="cuda") < density).int()
    moved = torch.rand((n, h, w, 1), generator=g, device="cuda") < 0.6
    delta = torch.where(moved, randn((n, h, w, c), g), randn((n, h, w, c), g) * 1e-4)
    delta[..., 0] = torch.where(moved[..., 0], 2 * prev_in.float().abs().amax(-1) + 3, delta[..., 0])
    delta = delta.to(dtype)
    delta[mask == 0] = float("nan")                                             # never read
    thr = 0.1
    u, y64, e, keep, nn, a = delta64(torch.nan_to_num(delta), mask, prev_in, prev_out, wt, b, thr)
    pi, po = prev_in.clone(), prev_out.clone()
    out = torch.full_like(delta, 7.0)
    om = torch.full((n, 1, h, w), 9, dtype=torch.int32, device="cuda")
    dc().layer_norm_delta(cl(delta), mask[:, None], cl(pi), cl(po), wt, b, thr, EPS, out=cl(out), out_mask=om)
    assert torch.equal(pi, u)
    if c > 1:
        assert torch.equal(om[:, 0].bool(), keep[..., 0])
    k = keep.expand_as(out)
    assert (out[~k] == 7.0).all() and torch.equal(po[~k], prev_out[~k])
    # y is rounded to the storage type, the difference again, and their sum with prev_out once more
    by = y_bound(wt.double(), b.double(), nn, a, y64, dtype)
    be = by + half(dtype) * (e.abs() + by)
    within(out[k], e[k], be[k], "out")
    within(po[k], y64[k], (be + half(dtype) * (y64.abs() + be))[k], "prev_out")
    # in place, as the module calls it
    d2, m2, pi2, po2 = delta.clone(), mask[:, None].clone(), prev_in.clone(), prev_out.clone()
    dc().layer_norm_delta(cl(d2), m2, cl(pi2), cl(po2), wt, b, thr, EPS, out=cl(d2), out_mask=m2)
    assert torch.equal(m2, om) and torch.equal(pi2, pi) and torch.equal(po2, po) and torch.equal(d2[k], out[k])


# ---- MXFP4 -----------------------------------------------------------------------------------------------------

def mx4_64(x):
    """(values, scale exponents + 127) of x in MXFP4 along its rows, by the definition."""
    x = x.double()
    rows, cols = x.shape
    nb = -(-cols // 32)
    f = torch.zeros((rows, nb * 32), dtype=torch.float64, device=x.device)
    f[:, :cols] = x
    f = f.view(rows, nb, 32)
    bad = ~f.isfinite().all(-1)
    f = torch.where(bad[..., None], torch.zeros_like(f), f)
    top = f.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, torch.full_like(top, -127)).clamp(min=-127).double()
    v = f * torch.exp2(-e)[..., None]
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = torch.bucketize(v.abs(), mid, right=True), torch.bucketize(v.abs(), mid)
    q = grid[torch.where(up % 2 == 0, up, down)] * torch.sign(v) * torch.exp2(e)[..., None]
    q = torch.where(bad[..., None], torch.full_like(q, float("nan")), q)
    return q.view(rows, nb * 32)[:, :cols], torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def scales_of(q):
    rows, cols = q.shape
    rt, kt = q.scales.shape[:2]
    return q.scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows]


def check_packed(q, x, what):
    rows, cols = x.shape
    want, s = mx4_64(x)
    nb = s.shape[1]
    assert q.shape == (rows, cols)
    assert torch.equal(scales_of(q)[:, :nb], s), what
    assert (scales_of(q)[:, nb:] != 255).all(), what                            # blocks behind the last one are not NaN
    for t in ((F32, x.dtype) if x.dtype != F16 or not (x.abs() > 3e4).any() else (F32,)):
        assert torch.equal(torch.nan_to_num(dc().mx4_dequantize(q, t).double(), nan=123.0), torch.nan_to_num(want, nan=123.0)), (what, t)
    if cols % 32:                                                               # zeros behind the last column
        codes = torch.stack((q.data & 15, q.data >> 4), -1).view(rows, nb * 32)
        assert ((codes[:, cols:] & 7) == 0).all(), what


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (130, 96), (128, 128), (129, 130), (33, 1000), (300, 264), (7, 4096), (2, 1500), (257, 129)])
def test_quantize(rows, cols, dtype):
    g = gen(rows + cols)
    x = (randn((rows, cols), g) * torch.exp(3 * randn((rows, 1), g))).to(dtype)
    check_packed(dc().mx4_quantize(x), x, "rows")
    q, qt = dc().mx4_quantize_both(x)
    check_packed(q, x, "both, rows")
    check_packed(qt, x.t().contiguous(), "both, columns")


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_hard_values(dtype):
    """Ties, saturation, zeros, the smallest and largest numbers, infinities and NaN."""
    i = torch.finfo(dtype)
    blocks = [[0.0], [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0], [-0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0], [7.9, 6.0, 5.0, -7.0],
              [i.tiny, i.tiny / 2, -i.tiny], [i.smallest_normal * half(dtype) * 4, 0.0], [i.max, i.max / 3, -i.max / 7], [float("inf"), 1.0], [1.0, float("nan")],
              [-float("inf"), float("nan")], [1.0, 1e-6], [2 ** -9, 2 ** -14, 3 * 2 ** -10]]
    x = torch.zeros((len(blocks) + 3, 96))
    for r, v in enumerate(blocks):
        x[r, 32:32 + len(v)] = torch.tensor(v, dtype=torch.float64).to(dtype).float()
        x[r, 0] = 1.0
    x = x.to(dtype).cuda()
    check_packed(dc().mx4_quantize(x), x, "rows")
    q, qt = dc().mx4_quantize_both(x)
    check_packed(q, x, "both")
    check_packed(qt, x.t().contiguous(), "columns")


def test_quantize_feature_map_and_unaligned():
    g = gen(11)
    x = randn((2, 40, 3, 5), g, F16).contiguous(memory_format=torch.channels_last)
    check_packed(dc().mx4_quantize(x), x.permute(0, 2, 3, 1).reshape(-1, 40), "map")
    y = randn((1 + 64 * 6,), g, F16)[1:].view(6, 64)
    check_packed(dc().mx4_quantize(y), y, "two bytes off")
    assert dc().mx4_quantize(torch.empty((0, 40), device="cuda")).shape == (0, 40)
    assert dc().mx4_dequantize(dc().mx4_quantize(torch.empty((0, 40), device="cuda"))).shape == (0, 40)


def packed(shape, g, spread=1.0):
    x = randn(shape, g) * torch.exp(spread * randn((shape[0], 1), g))
    q = dc().mx4_quantize(x)
    return q, dc().mx4_dequantize(q).double()


def product_bound(a, b, k):
    # at most one rounding or truncation (2 u) of a partial sum per value of k
    return 2 * k * U * (a.abs() @ b.abs().t())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 32), (3, 8, 33), (16, 128, 64), (17, 130, 96), (32, 1000, 255), (33, 127, 256), (64, 1000, 1280), (65, 257, 257),
                                   (127, 129, 512), (128, 128, 1024), (129, 384, 300), (200, 100, 4096), (256, 256, 768), (300, 1001, 2000), (1, 4096, 4096), (2, 1000, 5000),
                                   (700, 5000, 544), (1030, 4100, 288), (2500, 1900, 160), (2050, 4802, 1000), (2177, 4801, 96), (1500, 5120, 2080), (129, 12000, 320), (100, 30000, 320), (16, 40000, 64)])
def test_matmul(m, n, k, dtype):
    g = gen(m + n + k)
    (qa, a), (qb, b) = packed((m, k), g), packed((n, k), g)
    bias = randn((n,), g, dtype)
    want = a @ b.t() + bias.double()
    got = dc().mx4_matmul(qa, qb, bias, dtype)
    assert got.dtype == dtype
    assert not dc()._lib.lib.dc_umma_error()
    within(got, want, product_bound(a, b, k) + U * want.abs() + half(dtype) * want.abs(), "product")
    assert torch.equal(got, dc().mx4_matmul(qa, qb, bias, dtype)), "the same inputs give other bits"


def test_matmul_is_exact_where_float32_is():
    """Whole numbers whose sums stay below 2^24: no rounding anywhere, so no bit may differ."""
    g = gen(12)
    grid = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, -1, -2, -3, -4, -6, -8, -12], device="cuda").float()
    for m, n, k in ((5, 200, 700), (300, 260, 1000), (130, 4800, 512), (2300, 2600, 700)):
        a = grid[torch.randint(15, (m, k), generator=g, device="cuda")]
        b = grid[torch.randint(15, (n, k), generator=g, device="cuda")]
        a[:, ::32], b[:, ::32] = 12.0, -12.0                                   # every block has the scale of 12: e2m1 x 2 holds the grid
        bias = torch.randint(-50, 50, (n,), generator=g, device="cuda").float()
        got = dc().mx4_matmul(dc().mx4_quantize(a), dc().mx4_quantize(b), bias, F32)
        assert torch.equal(got.double(), a.double() @ b.double().t() + bias.double())


@pytest.mark.parametrize("m", [4, 200, 6000])
def test_matmul_scales_far_apart_and_nan(m):
    g = gen(13)
    a, b = randn((m, 512), g), randn((300, 512), g)
    a *= torch.exp2(torch.randint(-30, 30, (m, 16), generator=g, device="cuda").float()).repeat_interleave(32, 1)
    b *= torch.exp2(torch.randint(-30, 30, (300, 16), generator=g, device="cuda").float()).repeat_interleave(32, 1)
    qa, qb = dc().mx4_quantize(a), dc().mx4_quantize(b)
    a64, b64 = dc().mx4_dequantize(qa).double(), dc().mx4_dequantize(qb).double()
    within(dc().mx4_matmul(qa, qb, None, F32), a64 @ b64.t(), product_bound(a64, b64, 512) + U * (a64 @ b64.t()).abs())
    a[1, 100], b[7, 3], b[290, 511] = float("nan"), float("inf"), float("nan")
    out = dc().mx4_matmul(dc().mx4_quantize(a), dc().mx4_quantize(b), None, F32)
    nan = torch.zeros((m, 300), dtype=torch.bool, device="cuda")
    nan[1], nan[:, 7], nan[:, 290] = True, True, True
    assert torch.equal(out.isnan(), nan)


def test_matmul_writes_nothing_else():
    g = gen(14)
    for m, n, k in ((3, 100, 64), (130, 130, 300), (1000, 5000, 64), (1001, 5001, 64)):
        (qa, _), (qb, _) = packed((m, k), g), packed((n, k), g)
        room = torch.full((2 * 4096 + m * n,), 5.0, device="cuda", dtype=F16)
        out = room[4096:4096 + m * n].view(m, n)
        dc().mx4_matmul(qa, qb, None, F16, out=out)
        assert (room[:4096] == 5).all() and (room[4096 + m * n:] == 5).all()
        assert torch.equal(out, dc().mx4_matmul(qa, qb, None, F16))


def test_matmul_ignores_what_lies_in_unused_scale_rows():
    g = gen(15)
    (qa, _), (qb, _) = packed((5, 100), g), packed((140, 100), g)
    want = dc().mx4_matmul(qa, qb, None, F32)
    for q in (qa, qb):
        s = q.scales.permute(0, 3, 2, 1, 4).reshape(-1, q.scales.shape[1] * 4).clone()
        s[q.shape[0]:] = 255
        q.scales.copy_(s.view(q.scales.shape[0], 4, 32, -1, 4).permute(0, 3, 2, 1, 4))
    assert torch.equal(dc().mx4_matmul(qa, qb, None, F32), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 24, 40), (37, 100, 130), (200, 260, 96), (130, 33, 512)])
def test_linear_gradients(m, n, k, dtype):
    g = gen(m)
    x, w, b, dy = randn((m, k), g, dtype), randn((n, k), g, dtype, k ** -0.5), randn((n,), g, dtype), randn((m, n), g, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = dc().mx4_linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    q = lambda t: mx4_64(t)[0]                                                  # noqa: E731
    for got, a, c, extra in ((y.detach(), q(x), q(w), b.double()), (dx, q(dy), q(w.t().contiguous()), 0.0), (dw, q(dy.t().contiguous()), q(x.t().contiguous()), 0.0)):
        want = a @ c.t() + extra
        within(got, want, product_bound(a, c, a.shape[1]) + (U + half(dtype)) * want.abs())
    within(db, dy.double().sum(0), (64 + m) * U * dy.double().abs().sum(0) + half(dtype) * dy.double().sum(0).abs(), "db")
    # one leaf at a time, and the packed weight
    for i in range(3):
        args = [t.detach() for t in leaves]
        args[i] = leaves[i]
        assert torch.equal(torch.autograd.grad(dc().mx4_linear(*args), leaves[i], dy)[0], (dx, dw, db)[i])
    assert torch.equal(dc().mx4_linear(x, dc().mx4_quantize(w), b), y.detach())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 100, 40), (1, 14000, 1024), (2, 1000, 1281), (5, 130, 2052), (16, 1000, 4096), (17, 300, 31), (31, 5000, 500), (33, 1000, 1280), (64, 1000, 700),
                                   (64, 9000, 2048), (65, 100, 260), (1, 30000, 256), (3, 40000, 200), (20, 25000, 96)])
def test_linear_with_packed_weight_is_quantize_and_matmul(m, n, k, dtype):
    """Few tokens are packed inside the product: the same bits as the two calls, hard values and odd widths included."""
    g = gen(m + n)
    x, b = randn((m, k), g, dtype, 2.0), randn((n,), g, dtype)
    x[0, :32] = 0
    x[-1, -1] = float("nan") if m > 2 else 7.0
    qw = dc().mx4_quantize(randn((n, k), g))
    got = dc().mx4_linear(x, qw, b)
    want = dc().mx4_matmul(dc().mx4_quantize(x), qw, b, dtype)
    assert torch.equal(torch.nan_to_num(got, nan=77.0), torch.nan_to_num(want, nan=77.0))
    if m > 2:
        assert got[-1].isnan().all() and not got[:-1].isnan().any()
    off = torch.empty(m * k + 1, device="cuda", dtype=dtype)[1:].view(m, k).copy_(x)         # rows off 16 bytes
    assert torch.equal(torch.nan_to_num(dc().mx4_linear(off, qw, b), nan=77.0), torch.nan_to_num(want, nan=77.0))


def test_linear_gradient_against_differences():
    """Where every rounding is exact (whole numbers that e2m1 holds) the layer is linear: differences are the gradient."""
    g = gen(17)
    grid = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device="cuda").float()
    pick = lambda s: grid[torch.randint(11, s, generator=g, device="cuda")]      # noqa: E731
    x, w, dy = pick((64, 96)), pick((40, 96)), pick((64, 40))
    for t in (x, w, dy):                                                        # the largest value of every block of either direction is 6
        t[::32, :], t[:, ::32] = 6.0, 6.0
    x, w = x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(dc().mx4_linear(x, w), (x, w), dy)
    f = lambda a, c: ((a.double() @ c.double().t()) * dy.double()).sum()         # noqa: E731
    for t, gr in ((x, dx), (w, dw)):
        v = pick(tuple(t.shape)).double()
        p, m = (f(x.detach() + s * v, w.detach()) if t is x else f(x.detach(), w.detach() + s * v) for s in (1, -1))
        assert (p - m) / 2 == (gr.double() * v).sum()


# ---- as they are used ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (F32, F32), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("x_off,w_off", [(1, 0), (0, 1), (2, 0), (0, 2), (1, 2)])
def test_linear_training_at_other_addresses(x_off, w_off, dtype, wtype):
    m, n, k = 150, 136, 264
    g = gen(x_off * 7 + w_off)
    x, w, dy = randn((m, k), g, dtype), randn((n, k), g, wtype), randn((m, n), g, dtype)

    def moved(t, off):
        room = torch.zeros(t.numel() + 8, device="cuda", dtype=t.dtype)
        at = room[off:off + t.numel()].view(t.shape)
        at.copy_(t)
        return at.requires_grad_()

    y = []
    for a, b in ((moved(x, 0), moved(w, 0)), (moved(x, x_off), moved(w, w_off))):
        out = dc().mx4_linear(a, b)
        y.append((out.detach(), *torch.autograd.grad(out, (a, b), dy)))
    assert all(torch.equal(p, q) for p, q in zip(*y))
    packed = dc().mx4_matmul(dc().mx4_quantize(x), dc().mx4_quantize(w), None, dtype)
    assert torch.equal(y[0][0], packed)


def test_block_of_norm_and_linears_trains_and_serves():
    """norm -> 4-bit linear -> GELU -> 4-bit linear -> residual, forward and backward, then served with packed weights, also from a
    captured graph."""
    d = dc()
    torch.manual_seed(0)
    norm, up, down = d.DCLayerNorm(96).cuda().half(), d.DCMX4Linear(96, 384).cuda().half(), d.DCMX4Linear(384, 96).cuda().half()
    x = torch.randn(50, 96, device="cuda").half()

    def block(v):
        return v + down(torch.nn.functional.gelu(up(norm(v))))

    y = block(x)
    y.float().square().mean().backward()
    for p in (*norm.parameters(), *up.parameters(), *down.parameters()):
        assert p.grad is not None and p.grad.isfinite().all() and (p.grad != 0).any()
    with torch.no_grad():
        want = block(x)
        assert torch.equal(want, y)
        for m in (up, down):
            m.process_filters()
        served = block(x)
        assert torch.equal(served, want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        static = x.clone()
        with torch.cuda.stream(side):
            block(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(static)
        for s in (1, 2):
            fresh = torch.randn(50, 96, device="cuda", generator=gen(s)).half()
            static.copy_(fresh)
            graph.replay()
            assert torch.equal(out, block(fresh))


def test_training_step_in_a_graph():
    """Forward and backward captured together, on leaves of their own, replayed on new inputs, while an eager graph lives."""
    d = dc()
    g = gen(20)
    make = lambda: [randn(s, g, F16) for s in ((48, 64), (64,), (64,), (80, 64), (80,))]      # noqa: E731

    def step(x, nw, nb, w, b, dy):
        y = d.mx4_linear(d.layer_norm(x, nw, nb), w, b)
        return (y, *torch.autograd.grad(y, (x, nw, nb, w, b), dy))

    eager = [t.requires_grad_() for t in make()]
    alive = d.mx4_linear(d.layer_norm(*eager[:3]), *eager[3:])
    leaves, dy = [t.requires_grad_() for t in make()], randn((48, 80), g, F16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*leaves, dy)
    fresh = make()
    with torch.no_grad():
        for t, f in zip(leaves, fresh):
            t.copy_(f)
        dy.copy_(randn((48, 80), g, F16))
    graph.replay()
    want = step(*[f.clone().requires_grad_() for f in fresh], dy)
    assert all(torch.equal(p, q) for p, q in zip(outs, want))
    assert torch.autograd.grad(alive.float().sum(), eager[0])[0].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_delta_module_follows_the_dense_norm(dtype):
    """DCSparsify -> DCLayerNorm -> DCDensify over some frames at threshold 0 against the norm of the whole frame."""
    d = dc()
    g = gen(21)
    sp, ln, de = d.DCSparsify(delta_threshold=0.0), d.DCLayerNorm(24, delta_threshold=0.0).cuda().to(dtype), d.DCDensify()
    with torch.no_grad():
        ln.weight.copy_(randn((24,), g, dtype, 0.2, 1.0))
        ln.bias.copy_(randn((24,), g, dtype))
        frame = randn((2, 24, 9, 7), g, dtype).contiguous(memory_format=torch.channels_last)
        for t in range(5):
            got = de(ln(sp(frame.clone(memory_format=torch.preserve_format))))
            want = norm64(frame.permute(0, 2, 3, 1), ln.weight.double(), ln.bias.double())[0].permute(0, 3, 1, 2)
            # per frame: the accumulated input, the norm, its change and the accumulated output are each rounded once
            assert (got.double() - want).abs().max().item() <= 8 * (t + 1) * half(dtype) * 8
            assert torch.equal(got, ln.prev_out)                     # what the norm believes to have handed on is what arrived
            frame = frame.clone(memory_format=torch.preserve_format)
            frame[:, :, t:t + 3, 1:4] += randn((2, 24, 3, 3), g, dtype)
        ln.reset()
        assert ln.first_iter and ln.prev_in is None


def test_first_calls_inside_a_capture():
    """Nothing that a first call of a shape sets up may disturb a capture."""
    d = dc()
    g = gen(31)
    x, w, b, q = randn((37, 552), g, BF16), randn((552,), g, BF16), randn((552,), g, BF16), d.mx4_quantize(randn((776, 552), g))
    tokens = randn((3, 552), g, BF16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = d.layer_norm(x, w, b)
        z, few = d.mx4_linear(y, q), d.mx4_linear(tokens, q)
        both = d.mx4_quantize_both(y)
    graph.replay()
    assert torch.equal(y, d.layer_norm(x, w, b)) and torch.equal(z, d.mx4_linear(y, q)) and torch.equal(few, d.mx4_linear(tokens, q))
    assert torch.equal(both[1].dequantize(), d.mx4_quantize_both(y)[1].dequantize())


def test_threads():
    """First calls of threads that have not touched the device yet, several at once."""
    import threading
    d = dc()
    g = gen(32)
    x, q = randn((200, 256), g, F16), d.mx4_quantize(randn((500, 256), g))
    want = d.mx4_linear(d.layer_norm(x), q)
    torch.cuda.synchronize()
    got, threads = [None] * 4, []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = d.mx4_linear(d.layer_norm(x), q)

    def first(i):                                        # nothing but the product itself
        got[i] = d.mx4_matmul(qx, q, None, F16)

    qx = d.mx4_quantize(d.layer_norm(x))
    torch.cuda.synchronize()
    for i in range(4):
        threads.append(threading.Thread(target=first if i == 0 else work, args=(i,)))
        threads[-1].start()
        if i == 0:
            threads[-1].join()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_streams():
    d = dc()
    g = gen(22)
    x, w = randn((300, 512), g, F16), randn((700, 512), g, F16)
    nw, nb = randn((512,), g, F16), randn((512,), g, F16)
    want = d.mx4_linear(d.layer_norm(x, nw, nb), w)
    s = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(9):
        with torch.cuda.stream(s[i % 3]):
            got.append(d.mx4_linear(d.layer_norm(x, nw, nb), w))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_refusals():
    d = dc()
    x = torch.randn(4, 64, device="cuda")
    bad = [
        lambda: d.layer_norm(x.double()), lambda: d.layer_norm(x.t()), lambda: d.layer_norm(x, torch.ones(63, device="cuda")),
        lambda: d.layer_norm(x, torch.ones(64)), lambda: d.layer_norm(x.half(), torch.ones(64, device="cuda"), torch.ones(64, device="cuda").half()),
        lambda: d.layer_norm(x, torch.ones(64, device="cuda").half()), lambda: d.layer_norm(torch.randn(2, 8, 4, 4, device="cuda")),
        lambda: d.layer_norm(torch.empty(3, 0, device="cuda")),
        lambda: d.mx4_quantize(x.int()), lambda: d.mx4_quantize(x[:, ::2]), lambda: d.mx4_quantize_both(torch.empty(0, 8, device="cuda")),
        lambda: d.mx4_matmul(d.mx4_quantize(x), d.mx4_quantize(torch.randn(4, 32, device="cuda"))),
        lambda: d.mx4_matmul(d.mx4_quantize(x), d.mx4_quantize(x), torch.ones(5, device="cuda")),
        lambda: d.mx4_matmul(d.mx4_quantize(x), d.mx4_quantize(x), None, torch.float64),
        lambda: d.mx4_matmul(d.mx4_quantize(x), d.mx4_quantize(x), None, torch.float16, out=torch.empty(4, 4, device="cuda")),
        lambda: d.mx4_linear(x, torch.randn(8, 32, device="cuda")), lambda: d.mx4_linear(x, torch.randn(8, 64)),
        lambda: d.mx4_linear(x.requires_grad_(), d.mx4_quantize(torch.randn(8, 64, device="cuda"))),
        lambda: d.DCMX4Linear(64, 8).cuda()((x, None)),
    ]
    delta = torch.randn(1, 8, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last)
    mask = torch.ones(1, 1, 4, 4, dtype=torch.int32, device="cuda")
    wide = torch.zeros(1, 40000, 1, 1, device="cuda").contiguous(memory_format=torch.channels_last)      # no kernel for so many channels
    bad += [
        lambda: d.layer_norm_delta(delta.bfloat16(), mask, delta.bfloat16(), delta.bfloat16()),
        lambda: d.layer_norm_delta(delta, mask[:, :, :2], delta.clone(), delta.clone()),
        lambda: d.layer_norm_delta(delta, mask, delta.half(), delta.clone()),
        lambda: d.layer_norm_delta(delta, mask, delta.clone(), delta[:, :, :2].clone()),
        lambda: d.layer_norm_delta(delta, mask, delta, delta.clone()),
        lambda: d.layer_norm_delta(delta, mask, *[delta.clone()] * 2),
        lambda: d.layer_norm_delta(wide, mask[:, :, :1, :1].contiguous(), wide.clone(), wide.clone()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
