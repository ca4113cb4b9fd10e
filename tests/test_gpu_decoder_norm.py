"""decoder_norm (LayerNorm with gradients) against its definition in 64 bits.

Bounds, with u = 2^-24 (half an fp32 step) and h half a step of the output's type: a row sum adds
at most 16 values a thread, 5 shuffle steps and 32 warps, so it is off by at most 64 u of the sum
of magnitudes; the mean is then off by 64 u max|x|, rstd by 40 u relative (half of the variance's
64 u, the root and the quotient), n = (x - mean) rstd by e_n = 64 u max|x| rstd + 44 u |n|, and the
formulas below follow term by term.  The sums over rows add at most 256 terms one after another at
these sizes (rows of a group, groups of a block, blocks of a warp, warps)."""
import pytest
import torch

from sparse4d_tt_b200 import decoder_norm, decoder_norm_backward, decoder_norm_forward
from sparse4d_tt_b200.graph import capture

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def make(rows, width, dtype, seed=0, offset=0.0, ptype=torch.float32):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + width)
    x = (torch.randn(rows, width, generator=g) * 1.5 + offset).to(dtype).cuda()
    dy = torch.randn(rows, width, generator=g).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(ptype).cuda()
    b = (0.3 * torch.randn(width, generator=g)).to(ptype).cuda()
    return x, dy, w, b


def check(x, dy, w, b, eps, y, dx, dw, db):
    X, G = x.double(), dy.double()
    W = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    mean = X.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((X - mean) ** 2).mean(-1, keepdim=True) + eps)
    n = (X - mean) * rstd
    ref = n * W + B
    e_n = 64 * U * X.abs().amax(-1, keepdim=True) * rstd + 44 * U * n.abs()
    h = half_step(y.dtype)
    tol = (1 + h) * (W.abs() * e_n + 2 * U * (n * W).abs() + 2 * U * ref.abs()) + h * ref.abs() + 1e-7 * (
        y.dtype == torch.float16)
    assert ((y.double() - ref).abs() <= tol).all(), ((y.double() - ref).abs() - tol).max()
    g = G * W
    s1, s2 = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    if dx is not None:
        rdx = rstd * (g - s1 - n * s2)
        a1, a2 = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
        e2 = 66 * U * a2 + (g.abs() * e_n).mean(-1, keepdim=True)
        tol = (1 + h) * (rstd * (4 * U * g.abs() + 66 * U * a1 + n.abs() * e2 + e_n * s2.abs()
                                 + 4 * U * (s1.abs() + (n * s2).abs())) + 44 * U * rdx.abs()) + h * rdx.abs() \
            + 1e-7 * (dx.dtype == torch.float16)
        assert ((dx.double() - rdx).abs() <= tol).all(), ((dx.double() - rdx).abs() - tol).max()
    if dw is not None:
        r = (G * n).sum(0)
        tol = 256 * U * (G * n).abs().sum(0) + (G.abs() * e_n).sum(0)
        tol = tol + half_step(dw.dtype) * (r.abs() + tol)
        assert ((dw.double() - r).abs() <= tol).all(), ((dw.double() - r).abs() - tol).max()
    if db is not None:
        r = G.sum(0)
        tol = 256 * U * G.abs().sum(0)
        tol = tol + half_step(db.dtype) * (r.abs() + tol)
        assert ((db.double() - r).abs() <= tol).all(), ((db.double() - r).abs() - tol).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 7), (3, 256), (900, 256), (17, 257), (64, 512), (33, 1000),
                                        (29, 1001), (40, 2048), (7, 2049), (9, 5000), (5, 8192), (3, 16384),
                                        (2, 16383), (2801, 64), (2048, 512), (2049, 512), (300, 8192)])
def test_forward_and_gradients(cuda_device, dtype, rows, width):
    x, dy, w, b = make(rows, width, dtype)
    y, mean, rstd = decoder_norm_forward(x, w, b, 1e-5)
    dx, dw, db = decoder_norm_backward(dy, x, w, mean, rstd)
    check(x, dy, w, b, 1e-5, y, dx, dw, db)
    assert dx.dtype == dtype and dw.dtype == torch.float32


@pytest.mark.parametrize("width", [48, 515, 3000])
def test_rows_far_from_zero_parameters_in_the_rows_type_and_parts(cuda_device, width):
    """A large common offset (where a one-pass variance cancels), bf16 parameters, missing ones,
    and only some of the gradients."""
    x, dy, w, b = make(77, width, torch.float32, offset=300.0)
    y, mean, rstd = decoder_norm_forward(x, w, b, 1e-5)
    check(x, dy, w, b, 1e-5, y, *decoder_norm_backward(dy, x, w, mean, rstd))
    x, dy, w, b = make(77, width, torch.bfloat16, ptype=torch.bfloat16)
    y, mean, rstd = decoder_norm_forward(x, w, b, 1e-3)
    got = decoder_norm_backward(dy, x, w, mean, rstd)
    assert got[1].dtype == torch.bfloat16
    check(x, dy, w, b, 1e-3, y, *got)
    y, mean, rstd = decoder_norm_forward(x, None, b, 1e-3)
    check(x, dy, None, b, 1e-3, y, None, None, None)
    y, mean, rstd = decoder_norm_forward(x, None, None, 1e-3)
    dx, dw, db = decoder_norm_backward(dy, x, None, mean, rstd, need_dweight=False, need_dbias=False)
    assert dw is None and db is None
    check(x, dy, None, None, 1e-3, y, dx, None, None)
    dx2, dw, db = decoder_norm_backward(dy, x, None, mean, rstd, need_dx=False, need_dweight=False)
    assert dx2 is None and dw is None
    check(x, dy, None, None, 1e-3, y, None, None, db)


def test_strided_broadcast_and_in_place_rows(cuda_device):
    x, dy, w, b = make(60, 130, torch.bfloat16)
    wide = torch.zeros(60, 201, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:133] = x  # rows of an odd stride, not 16-byte aligned
    v = wide[:, 3:133]
    y0, m0, r0 = decoder_norm_forward(x, w, b)
    y1, m1, r1 = decoder_norm_forward(v, w, b)
    assert torch.equal(y0, y1) and torch.equal(m0, m1) and torch.equal(r0, r1)
    for a, c in zip(decoder_norm_backward(dy, x, w, m0, r0), decoder_norm_backward(dy, v, w, m1, r1)):
        assert torch.equal(a, c)
    one = dy[:1].expand(60, -1)  # the gradient of a sum over rows: one row, stride 0
    for a, c in zip(decoder_norm_backward(one, x, w, m0, r0),
                    decoder_norm_backward(one.contiguous(), x, w, m0, r0)):
        assert torch.equal(a, c)
    column = x.t().contiguous().t()  # column-major rows are copied
    assert torch.equal(decoder_norm_forward(column, w, b)[0], y0)
    x3 = x.reshape(3, 20, 130)
    y3, m3, _ = decoder_norm_forward(x3, w, b)
    assert y3.shape == x3.shape and m3.shape == (3, 20) and torch.equal(y3.reshape(60, 130), y0)
    z = x.clone()
    decoder_norm_forward(z, w, b, out=z)
    assert torch.equal(z, y0)


def test_special_rows(cuda_device):
    """A constant row, a row with an infinity and one with a NaN stay inside their rows; no rows at
    all write zero parameter gradients."""
    x, dy, w, b = make(12, 300, torch.float32)
    clean, m, r = decoder_norm_forward(x, w, b)
    cdx = decoder_norm_backward(dy, x, w, m, r)[0]
    x[3] = 5.0
    x[5, 7] = float("inf")
    x[9, 299] = float("nan")
    y, mean, rstd = decoder_norm_forward(x, w, b)
    dx = decoder_norm_backward(dy, x, w, mean, rstd)[0]
    assert torch.equal(y[3], b) and torch.isfinite(dx[3]).all()
    assert torch.isnan(y[9]).all() and torch.isnan(y[5]).any()
    keep = [0, 1, 2, 4, 6, 7, 8, 10, 11]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], cdx[keep])
    e = torch.empty(0, 300, device="cuda")
    y, mean, rstd = decoder_norm_forward(e, w, b)
    dx, dw, db = decoder_norm_backward(e, e, w, mean, rstd)
    assert y.shape == dx.shape == (0, 300) and not dw.any() and not db.any()


def test_equal_calls_give_equal_bits_on_any_stream_and_in_a_graph(cuda_device):
    x, dy, w, b = make(5000, 384, torch.bfloat16)

    def both():
        y, mean, rstd = decoder_norm_forward(x, w, b)
        return (y, *decoder_norm_backward(dy, x, w, mean, rstd))

    first = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    calls = [capture(both), capture(both)]
    for c in calls + calls:
        out = c.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, g) for a, g in zip(first, out))
    assert all(torch.equal(a, g) for a, g in zip(first, other))
    x.mul_(-1)  # a replay reads what the tensors hold then
    out = calls[0].replay()
    assert torch.equal(out[0], both()[0]) and not torch.equal(out[0], first[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(cuda_device, dtype):
    x, dy, w, b = make(50, 200, dtype)
    xl, wl, bl = (t.clone().requires_grad_() for t in (x, w, b))
    y = decoder_norm(xl.reshape(5, 10, 200), wl, bl)
    y.backward(dy.reshape(5, 10, 200))
    check(x, dy, w, b, 1e-5, y.detach().reshape(50, 200), xl.grad, wl.grad, bl.grad)
    only = x.clone().requires_grad_()
    decoder_norm(only).sum().backward()  # an expanded gradient, no parameters
    assert only.grad.shape == x.shape
    bl.grad = None
    decoder_norm(x, None, bl).float().sum().backward()
    assert torch.equal(bl.grad, torch.full_like(bl, 50.0))


def test_gradient_against_differences(cuda_device):
    """fp32 gradients against central differences of the 64-bit forward pass: with a step of 1e-6 the
    differences are good to about 1e-9, the fp32 gradient to the bounds above (under 1e-4 here)."""
    x, dy, w, b = make(4, 24, torch.float32)
    _, mean, rstd = decoder_norm_forward(x, w, b)
    dx, dw, _ = decoder_norm_backward(dy, x, w, mean, rstd)

    def loss(X, W):
        n = (X - X.mean(-1, keepdim=True)) / torch.sqrt(X.var(-1, unbiased=False, keepdim=True) + 1e-5)
        return ((n * W + b.double()) * dy.double()).sum()

    X, W = x.double(), w.double()
    for i in range(4):
        for j in range(0, 24, 5):
            d = torch.zeros_like(X)
            d[i, j] = 1e-6
            assert abs((loss(X + d, W) - loss(X - d, W)).item() / 2e-6 - dx[i, j].item()) < 1e-4
    for j in range(0, 24, 5):
        d = torch.zeros_like(W)
        d[j] = 1e-6
        assert abs((loss(X, W + d) - loss(X, W - d)).item() / 2e-6 - dw[j].item()) < 1e-4


def test_out_that_shares_memory_is_rejected(cuda_device):
    buf = torch.randn(64, 64, device="cuda")
    w = buf[3]
    for bad in (lambda: decoder_norm_forward(buf[1:], out=buf[:-1]), lambda: decoder_norm_forward(buf[:1].expand(8, 64), out=buf[:8]),
                lambda: decoder_norm_forward(buf[8:], w, out=buf[:56]), lambda: decoder_norm_forward(buf[:, :32], out=buf[:32].view(64, 32))):
        with pytest.raises(ValueError):
            bad()
    decoder_norm_forward(buf[32:], w, out=buf[32:])  # x itself
