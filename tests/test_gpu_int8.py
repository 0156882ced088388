"""8-bit integer operators against plain references in 64 bits.

The integers of a row are one well-defined answer (the nearest level of the exact quotient) and are compared for
equality, except behind the gated activation, whose fp32 exp may move a value that lies on a border.  Tolerances count
roundings: half a step is 2^-24 of an fp32 value, ``finfo.eps / 2`` of an output."""
import pytest
import torch

from triton_client_amd.ops import int8

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24  # half a step of fp32, relative
TYPES = [torch.float16, torch.bfloat16, torch.float32]


class _NoPlain:
    """Stands in for the extension that takes plain calls: every call goes the general way."""

    def __getattr__(self, name):
        return lambda *args: None


def test_plain_and_general_calls_agree(monkeypatch):
    """Contiguous operands are taken by the extension, everything else by the Python path: the same results."""
    x, r = (_values(21, 96, torch.bfloat16, s).cuda() for s in (1, 2))
    n = _values(1, 96, torch.bfloat16, 3)[0].cuda()
    w, ws = _int8(40, 96).cuda(), torch.rand(40).cuda()
    wu, wus = _int8(50, 97).cuda(), torch.rand(50).cuda()
    b = torch.randn(40, device="cuda").bfloat16()

    def calls():
        q, s = int8.quantize_int8(x.reshape(3, 7, 96))
        qu, su = int8.quantize_int8(_values(900, 97, torch.float32, 4).cuda())
        yield from (q, s, qu, su)
        yield from int8.silu_mul_int8(x)
        yield from int8.rms_norm_int8(x, n, eps=1e-5)
        yield from int8.rms_norm_int8(x, n.float(), residual=r)
        yield from int8.rms_norm_int8(x[0], n, residual=r[0], eps=1)
        for dtype in (None, *TYPES):
            yield int8.dequantize_int8(q, s, dtype=dtype)
            yield int8.linear_int8(q, s, w, ws, dtype=dtype)
        yield int8.linear_int8(q, s, w, ws, bias=b, residual=torch.ones_like(x[:, :40]).reshape(3, 7, 40), dtype=b.dtype)
        yield int8.linear_int8(qu, su, wu, wus)

    plain = list(calls())
    monkeypatch.setattr(int8, "_plain", _NoPlain())
    general = list(calls())
    assert len(plain) == len(general)
    for p, g in zip(plain, general):
        assert p.dtype == g.dtype and p.shape == g.shape and p.is_contiguous() and torch.equal(p, g)


def test_plain_calls_are_taken_by_the_extension():
    from triton_client_amd import _native

    ops = _native.torch_ops()
    x = _values(3, 32, torch.float16).cuda()
    q, s = ops.quantize(x, False)
    assert ops.dequantize(q, s, 1).dtype == torch.float16 and len(ops.quantize(x, True)) == 2
    assert len(ops.rms_norm(x, x[0], None, 1e-6)) == 2 and len(ops.rms_norm(x, x[0], x, 1e-6)) == 3
    assert ops.linear(q, s, q, s, None, None, 0).shape == (3, 3)
    # not plain: left to the general path
    assert ops.quantize(x.t(), False) is None and ops.quantize(x.cpu(), False) is None
    assert ops.quantize(x.int(), False) is None and ops.quantize(x.clone().requires_grad_(), False) is None
    assert ops.quantize(x[:, :31].contiguous(), True) is None and ops.quantize(None, False) is None
    assert ops.rms_norm(x, x[0, :4], None, 1e-6) is None and ops.rms_norm(x, x[0], None, 0.0) is None
    assert ops.rms_norm(x, x[0], x.float(), 1e-6) is None and ops.rms_norm(x, x[0], None, "1") is None
    assert ops.dequantize(q, s[:2], 1) is None and ops.dequantize(x, s, 1) is None
    assert ops.linear(q, s, q[:, :16].contiguous(), s, None, None, 0) is None
    assert ops.linear(q, s, q, s, x[0, :3].contiguous(), None, 0) is None
    assert ops.linear(q, s, q, s, None, x, 0) is None


def _values(rows, width, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) * spread
    return x.to(dtype)


def _levels(p):
    """``(q, max)`` of fp32 rows on the CPU, the quotient in 64 bits (127 p is exact there, and a quotient of two fp32
    numbers that is not a border between integers does not round to one)."""
    top = p.abs().amax(dim=-1, keepdim=True)
    q = torch.where(top > 0, torch.round(127 * p.double() / top.double()), 0.0)
    return q.to(torch.int8), top


def _int8(rows, width, seed=0, low=-127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, 128, (rows, width), generator=g, dtype=torch.int8)


WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 120, 128, 129, 250, 256, 257, 500, 512, 513, 1000, 4095, 4096, 5000, 8192, 8200, 20001, 32768, 32769, 40000]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_is_the_nearest_level(width, dtype):
    x = _values(5, width, dtype, seed=width)
    q, scale = int8.quantize_int8(x.cuda())
    ref, top = _levels(x.float())
    assert torch.equal(q.cpu(), ref)
    assert torch.equal(scale.cpu(), top[:, 0] / 127)  # one division, correctly rounded on both sides


@pytest.mark.parametrize("rows", [1, 31, 33, 2047, 2048, 5001])
@pytest.mark.parametrize("width", [5, 40, 100, 200, 400, 4099])
def test_many_rows(rows, width):
    """The kernels that take several rows per block, and the other split of a row that many rows get."""
    x = _values(rows, width, torch.float16, seed=rows)
    w = _values(1, width, torch.float16, seed=1)[0]
    q, scale = int8.quantize_int8(x.cuda())
    ref, top = _levels(x.float())
    assert torch.equal(q.cpu(), ref) and torch.equal(scale.cpu(), top[:, 0] / 127)
    q, scale, h = int8.rms_norm_int8(x.cuda(), w.cuda(), residual=x.cuda())
    want = (x.float() + x.float()).half()
    ref, top = _levels(want.float() * w.float())
    assert torch.equal(h.cpu(), want) and torch.equal(q.cpu(), ref)
    factor = torch.rsqrt(want.double().square().mean(dim=-1) + 1e-6)
    assert torch.allclose(scale.cpu().double(), top[:, 0].double() * factor / 127, rtol=1.001 * F32, atol=0)


def test_quantize_special_rows():
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(torch.float32).max
    tiny = 2.0 ** -149
    rows = [
        [0.0, -0.0, 0.0, 0.0],
        [1.0, 0.5, -0.5, 0.25],            # 63.5 is a tie: to the even 64
        [nan, 1.0, 2.0, 3.0],
        [1.0, inf, 2.0, 3.0],
        [1.0, 2.0, -inf, 3.0],
        [top, -top, top / 2, 1.0],
        [tiny, -tiny, 0.0, tiny],          # 127 / m overflows fp32
        [127 * tiny, 63 * tiny, -64 * tiny, tiny],
        [1e-36, 5e-37, -3e-37, 1e-38],
        [127.0, 0.5, -0.5, 1.5],           # ties at small levels: 0, -0, 2
        [254.0, 125.0, 127.0, -129.0],     # 62.5, 63.5, -64.5
    ]
    x = torch.tensor(rows)
    q, scale = (t.cpu() for t in int8.quantize_int8(x.cuda()))
    finite = torch.isfinite(x).all(dim=1)
    ref, big = _levels(x[finite])
    assert torch.equal(q[finite], ref)
    want = big[:, 0] / 127
    # 127 * fp32(max / 127) of the largest fp32 value rounds to infinity: the scale one step below does not
    want = torch.where(torch.isfinite(want * 127), want, torch.nextafter(want, torch.zeros(())))
    assert torch.equal(scale[finite], want)
    assert q[1].tolist() == [127, 64, -64, 32] and q[9].tolist() == [127, 0, 0, 2]
    assert torch.isnan(scale[~finite]).all() and not q[~finite].any()
    back = int8.dequantize_int8(q.cuda(), scale.cuda(), dtype=torch.float32).cpu()
    assert torch.isnan(back[~finite]).all() and torch.isfinite(back[finite]).all()


def test_quantize_every_pair_of_half_values_near_borders():
    """All magnitudes of fp16 against maxima at which many quotients are borders or next to one."""
    every = torch.arange(0, 0x7c00, dtype=torch.int32).to(torch.int16).view(torch.float16)
    tops = [1.0, 127.0, 254.0, 1.9990234375, 3.96875, 6.0e-8, 65504.0, 0.0999755859375]
    x = torch.stack([torch.where(every <= t, every, torch.tensor(t, dtype=torch.float16)) for t in tops])
    q, _ = int8.quantize_int8(x.cuda())
    assert torch.equal(q.cpu(), _levels(x.float())[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("weight_f32", [False, True])
@pytest.mark.parametrize("width", [1, 9, 64, 100, 250, 512, 1000, 4096, 5000, 8200, 20001, 32769, 40000])
def test_norm(width, dtype, weight_f32):
    x, r = _values(4, width, dtype, seed=1), _values(4, width, dtype, seed=2, spread=3.0)
    w = (1 + 0.2 * _values(1, width, torch.float32, seed=3)[0]).to(torch.float32 if weight_f32 else dtype)
    for residual in (None, r):
        got = int8.rms_norm_int8(x.cuda(), w.cuda(), residual=None if residual is None else residual.cuda(), eps=1e-5)
        h = x if residual is None else (x.float() + residual.float()).to(dtype)
        if residual is not None:
            assert torch.equal(got[2].cpu(), h)
        q, top = _levels(h.float() * w.float())
        assert torch.equal(got[0].cpu(), q)
        factor = torch.rsqrt(h.double().square().mean(dim=-1, keepdim=True) + 1e-5)
        scale = (top.double() * factor / 127)[:, 0]
        # 64 bits until one rounding to fp32
        assert ((got[1].cpu().double() - scale).abs() <= 1.001 * F32 * scale).all()


def test_norm_special_rows():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[0.0] * 4, [1.0, nan, 2.0, 3.0], [inf, 1.0, 1.0, 1.0], [3e38, -3e38, 1e38, 0.0],
                      [2e30, 1e30, -5e29, 1.0], [1e-30, 1e-31, 0.0, 0.0], [1.0, 2.0, 3.0, 4.0]])
    w = torch.tensor([1.0, 1.0, 0.5, 1.0])
    q, scale = (t.cpu() for t in int8.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-6))
    bad = torch.tensor([False, True, True, False, False, False, False])
    assert torch.isnan(scale[bad]).all() and not q[bad].any()
    ref, top = _levels(x[~bad] * w)
    assert torch.equal(q[~bad], ref)
    h = x[~bad].double()  # squares of 3e38 hold in 64 bits
    want = top[:, 0].double() / torch.sqrt(h.square().mean(dim=1) + 1e-6) / 127
    assert ((scale[~bad].double() - want).abs() <= 1.001 * F32 * want).all()
    # a product with the weight that leaves fp32's range counts as not finite
    q, scale = int8.rms_norm_int8(x[3:4].cuda(), (w * 2).cuda())
    assert torch.isnan(scale).all() and not q.any()


@pytest.mark.parametrize("width", [1000, 40000])  # in registers, and read twice
@pytest.mark.parametrize("which", ["x", "residual"])
def test_norm_sum_in_place(width, which):
    x, r = (_values(3, width, torch.bfloat16, seed=s).cuda() for s in (1, 2))
    w = _values(1, width, torch.bfloat16, seed=3)[0].cuda()
    want = int8.rms_norm_int8(x, w, residual=r)
    target = x if which == "x" else r
    got = int8.rms_norm_int8(x, w, residual=r, sum_out=target)
    assert got[2] is target
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [1, 7, 8, 500, 1000, 4097, 8192, 33000])
def test_gate(width, dtype):
    x = _values(4, 2 * width, dtype, seed=width, spread=2.0)
    q, scale = (t.cpu() for t in int8.silu_mul_int8(x.cuda()))
    g, u = x.double().chunk(2, dim=-1)
    p = g / (1 + torch.exp(-g)) * u
    top = p.abs().amax(dim=-1, keepdim=True)
    # half steps: z = exp(-|g|) has 2 of the exponential unit and below 1 of its argument, 4 at most, which z / (1 + z)
    # takes over at most once; 1 + z, g z and the quotient round once each: 7; the product with the
    # other factor: 8 on p and on the maximum, so 16 on a quotient of up to 127 (and 9 on the scale)
    assert ((q.double() - torch.where(top > 0, 127 * p / top, 0.0)).abs() <= 0.5 + 127 * 16.1 * F32).all()
    want = (top / 127)[:, 0]
    assert ((scale.double() - want).abs() <= 9.1 * F32 * want + 2.0 ** -149).all()


def test_gate_extremes():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-100.0, 1.0, 2.0, 3.0], [-1e4, 1.0, 2.0, 3.0], [100.0, 0.0, 2.0, 3.0], [nan, 1.0, 2.0, 3.0],
                      [1.0, 1.0, inf, 0.0], [0.0, 0.0, 5.0, 5.0], [inf, 1.0, 1.0, 1.0], [-inf, 1.0, 1.0, 1.0]])
    q, scale = (t.cpu() for t in int8.silu_mul_int8(x.cuda()))
    assert q[0].tolist() == [0, 127] and q[1].tolist() == [0, 127] and q[2].tolist() == [127, 0]
    assert torch.isnan(scale[[3, 4, 6, 7]]).all() and not q[3:].any() and scale[5] == 0


def test_gate_over_the_whole_range():
    """Gates of every size, to where exp(-g) leaves fp32's range, against factors that bring the products back up."""
    g = torch.cat([torch.linspace(-104, 89, 4001), torch.tensor([-3e38, 3e38, -1e30, 1e30, -200.5, 1e-40, -1e-40, 0.0])])
    u = torch.full_like(g, 1e30)
    u[g.abs() > 150] = 1e-30
    rows = torch.stack([g, u], dim=1)  # a row each: its scale is the product's magnitude
    scale = int8.silu_mul_int8(rows.cuda())[1].cpu().double()
    gd = g.double()
    # exp(-|g|) below 2^-126 is held in steps of 2^-149: half a step of it, times |g|, and half a step each for the two
    # products behind it, at most |g| steps for the |g| > 87 at which that happens
    want = (gd / (1 + torch.exp(-gd)) * u.double()).abs() / 127
    coarse = torch.where(gd < 0, gd.abs() * u.double() * 2.0 ** -149 / 127, 0.0)
    assert ((scale - want).abs() <= 9.1 * F32 * want + coarse + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (2, 4097), (64, 512)])
def test_dequantize(shape, dtype):
    q, scale = _int8(*shape, low=-128), _values(1, shape[0], torch.float32)[0].abs()
    got = int8.dequantize_int8(q.cuda(), scale.cuda(), dtype=dtype)
    assert torch.equal(got.cpu(), (q.float() * scale[:, None]).to(dtype))


def _linear_reference(x, xs, w, ws, bias, residual, dtype):
    """The result in 64 bits, and how far the kernel may be from it."""
    acc = x.double() @ w.double().t()  # exact: below 2^53
    v = acc * xs.double()[:, None] * ws.double()
    # the sum to fp32, the two scales' product and the product with it: a half step each; one more for each addition
    slack = 3.01 * F32 * v.abs()
    for t in (bias, residual):
        if t is not None:
            v = v + t.double()
            slack = slack + 1.01 * F32 * v.abs()
    info = torch.finfo(dtype)
    return v, slack + info.eps / 2 * (v.abs() + slack) + info.smallest_normal * info.eps / 2


def _linear_case(m, n, k, dtype, bias=False, residual=False, seed=0, x=None, w=None, **kw):
    x = _int8(m, k, seed=seed + 1, low=-128) if x is None else x
    w = _int8(n, k, seed=seed + 2, low=-128) if w is None else w
    g = torch.Generator().manual_seed(seed)
    xs, ws = torch.rand(m, generator=g) * 0.02 + 1e-3, torch.rand(n, generator=g) * 1e-3 + 1e-4
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    dev = [t if t is None else t.cuda() for t in (x, xs, w, ws, b, r)]
    y = int8.linear_int8(dev[0], dev[1], dev[2], dev[3], bias=dev[4], residual=dev[5], dtype=dtype, **kw)
    ref, slack = _linear_reference(*(t if t is None else t.cuda() for t in (x, xs, w, ws, b, r)), dtype)
    off = (y.double() - ref).abs()
    assert y.dtype == dtype and tuple(y.shape) == (m, n)
    assert (off <= slack).all(), (m, n, k, float((off - slack).max()))
    return y


LINEAR_SHAPES = [(1, 1, 1), (1, 16, 64), (1, 4096, 4096), (2, 3, 15), (3, 17, 16), (5, 33, 17), (8, 1000, 2048),
                 (15, 100, 127), (16, 64, 128), (17, 65, 129), (32, 128, 255), (33, 130, 256), (48, 500, 1001),
                 (63, 63, 63), (64, 64, 640), (65, 1000, 513), (100, 257, 2000), (128, 128, 128), (129, 384, 1024),
                 (200, 1000, 2049), (256, 256, 96), (257, 513, 4000), (300, 1000, 2048), (500, 2048, 1040),
                 (777, 777, 777), (1024, 1024, 512), (1025, 2050, 1056), (5, 33000, 4096)]


@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
def test_linear_shapes(m, n, k):
    _linear_case(m, n, k, torch.float16, seed=m)
    _linear_case(m, n, k, torch.float32, bias=True, residual=True, seed=n)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_epilogues(dtype, bias, residual):
    for m, n, k in ((7, 50, 192), (90, 203, 320), (600, 520, 400)):
        _linear_case(m, n, k, dtype, bias=bias, residual=residual)


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_linear_is_exact_at_the_largest_sums(m):
    """128 * 128 * 131071 is the largest magnitude that int32 holds; -128 on both sides reaches it."""
    k = int8.MAX_K
    x = torch.full((m, k), -128, dtype=torch.int8)
    w = torch.full((20, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    w[3, -1] = 127
    y = int8.linear_int8(x.cuda(), torch.ones(m).cuda(), w.cuda(), torch.ones(20).cuda(), dtype=torch.float32)
    want = (x[:1].double() @ w.double().t()).float()  # one rounding, as the kernel's
    assert torch.equal(y.cpu(), want.expand(m, 20))


def test_linear_selects_each_k():
    """One-hot rows: every position of k reaches its output, in every place of a tile."""
    k = 300
    x = torch.eye(k, dtype=torch.int8)
    w = _int8(70, k, seed=5)
    ones = torch.ones
    y = int8.linear_int8(x.cuda(), ones(k).cuda(), w.cuda(), ones(70).cuda(), dtype=torch.float32)
    assert torch.equal(y.cpu(), w.t().float())


@pytest.mark.parametrize("m", [4, 40, 400])
def test_linear_rows_apart_and_unaligned(m):
    """Column ranges of wider buffers at any alignment: neighbours are not read into the sums, nor written."""
    n, k = 150, 200
    for x_at, w_at, y_at in ((0, 0, 0), (1, 3, 1), (16, 32, 8), (5, 16, 3)):
        xb, wb = _int8(m, k + 48, seed=1).cuda(), _int8(n, k + 56, seed=2).cuda()
        x, w = xb[:, x_at:x_at + k], wb[:, w_at:w_at + k]
        xs, ws = torch.rand(m).cuda() * 0.01, torch.rand(n).cuda() * 0.01
        yb = torch.full((m, n + 20), 7.0, dtype=torch.float16, device="cuda")
        rb = torch.randn(m, n + 9, device="cuda").half()
        y = yb[:, y_at:y_at + n]
        got = int8.linear_int8(x, xs, w, ws, residual=rb[:, 2:2 + n], out=y)
        assert got is y
        ref, slack = _linear_reference(x, xs, w, ws, None, rb[:, 2:2 + n], torch.float16)
        assert ((y.double() - ref).abs() <= slack).all()
        assert (yb[:, :y_at] == 7).all() and (yb[:, y_at + n:] == 7).all()


def test_linear_in_place_residual_and_nan_scale():
    x, w = _int8(70, 256).cuda(), _int8(96, 256, seed=3).cuda()
    xs, ws = torch.rand(70).cuda(), torch.rand(96).cuda() * 1e-3
    r = torch.randn(70, 96, device="cuda").bfloat16()
    want = int8.linear_int8(x, xs, w, ws, residual=r, dtype=torch.bfloat16)
    got = int8.linear_int8(x, xs, w, ws, residual=r, out=r)
    assert got is r and torch.equal(r, want)
    xs[3] = float("nan")
    y = int8.linear_int8(x, xs, w, ws)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[torch.arange(70) != 3]).all()


def test_shapes_of_any_rank_and_layout():
    x = _values(6, 40, torch.float16).reshape(2, 3, 40)
    q, s = int8.quantize_int8(x.cuda())
    ref = _levels(x.float())[0]
    assert q.shape == (2, 3, 40) and s.shape == (2, 3) and torch.equal(q.cpu(), ref)
    q1, s1 = int8.quantize_int8(x[0, 0].cuda())
    assert q1.shape == (40,) and s1.shape == () and torch.equal(q1.cpu(), ref[0, 0])
    q2, s2 = int8.quantize_int8(x.cuda().transpose(0, 1))
    assert torch.equal(q2, q.transpose(0, 1)) and torch.equal(s2, s.transpose(0, 1))
    q3, _ = int8.quantize_int8(x.cuda().reshape(6, 40)[:, ::2])
    assert torch.equal(q3.cpu(), _levels(x.reshape(6, 40)[:, ::2].float())[0])
    q4, _ = int8.quantize_int8(x[0, :1].cuda().expand(5, 40))
    assert torch.equal(q4.cpu(), ref[0, :1].expand(5, 40))
    w = _int8(12, 40, seed=9).cuda()
    ws = torch.rand(12).cuda()
    y = int8.linear_int8(q, s, w, ws)
    assert y.shape == (2, 3, 12)
    assert torch.equal(int8.linear_int8(q1, s1, w, ws), y[0, 0])
    assert torch.equal(int8.linear_int8(q.transpose(0, 1), s.t(), w, ws), y.transpose(0, 1))


def test_empty_batches():
    for dtype in TYPES:
        x = torch.empty(0, 64, dtype=dtype, device="cuda")
        q, s = int8.quantize_int8(x)
        assert q.shape == (0, 64) and s.shape == (0,)
        assert int8.dequantize_int8(q, s, dtype=dtype).shape == (0, 64)
        assert int8.rms_norm_int8(x, torch.ones(64, dtype=dtype, device="cuda"), residual=x)[2].shape == (0, 64)
        assert int8.silu_mul_int8(x)[0].shape == (0, 32)
        w, ws = _int8(5, 64).cuda(), torch.ones(5).cuda()
        assert int8.linear_int8(q, s, w, ws).shape == (0, 5)
        assert int8.linear_int8(_int8(3, 64).cuda(), torch.ones(3).cuda(), w[:0], ws[:0]).shape == (3, 0)


def test_row_operators_into_slices():
    """Destinations inside larger buffers: what lies around them stays."""
    x = _values(9, 100, torch.bfloat16).cuda()
    w = torch.ones(100, dtype=torch.bfloat16, device="cuda")
    qb = torch.full((9, 130), 55, dtype=torch.int8, device="cuda")
    sb = torch.full((11,), 5.0, device="cuda")
    hb = torch.full((9, 120), 5.0, dtype=torch.bfloat16, device="cuda")
    want = int8.rms_norm_int8(x, w, residual=x)
    int8.rms_norm_int8(x, w, residual=x, out=qb[:, 3:103], scale=sb[1:10], sum_out=hb[:, 7:107])
    assert torch.equal(qb[:, 3:103], want[0]) and torch.equal(sb[1:10], want[1]) and torch.equal(hb[:, 7:107], want[2])
    assert (qb[:, :3] == 55).all() and (qb[:, 103:] == 55).all()
    assert sb[0] == 5 and sb[10] == 5 and (hb[:, :7] == 5).all() and (hb[:, 107:] == 5).all()
    yb = torch.full((9, 111), 5.0, device="cuda")
    int8.dequantize_int8(qb[:, 3:103], sb[1:10], out=yb[:, 1:101])
    assert torch.equal(yb[:, 1:101], want[0].float() * want[1][:, None])
    assert (yb[:, :1] == 5).all() and (yb[:, 101:] == 5).all()
    # column ranges of one buffer lie apart
    both = torch.zeros(9, 200, dtype=torch.bfloat16, device="cuda")
    both[:, :100] = x
    int8.rms_norm_int8(both[:, :100], w, residual=x, sum_out=both[:, 100:])
    assert torch.equal(both[:, 100:], want[2]) and torch.equal(both[:, :100], x)


def _block(x, h, norm, w1, s1, w2, s2):
    q, s, h = int8.rms_norm_int8(x, norm, residual=h)
    y = int8.linear_int8(q, s, w1, s1, dtype=x.dtype)
    q, s = int8.silu_mul_int8(y)
    return int8.linear_int8(q, s, w2, s2, residual=h, dtype=x.dtype)


def _block_operands(d, f, dtype):
    w1, w2 = _values(2 * f, d, torch.float32, 1, d ** -0.5), _values(d, f, torch.float32, 2, f ** -0.5)
    norm = (1 + 0.1 * _values(1, d, torch.float32, 3)[0]).to(dtype)
    return norm.cuda(), *int8.quantize_int8(w1.cuda()), *int8.quantize_int8(w2.cuda())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens", [1, 5, 64, 333])
def test_block_together(tokens, dtype):
    """Norm, product, gated activation, product and residual, as a model runs them, each step against its formula on
    what the step before handed over."""
    d, f = 320, 456
    ops = _block_operands(d, f, dtype)
    x, h0 = _values(tokens, d, dtype, 4).cuda(), _values(tokens, d, dtype, 5).cuda()
    out = _block(x, h0, *ops)
    norm, w1, s1, w2, s2 = ops
    q, s, h = int8.rms_norm_int8(x, norm, residual=h0)
    assert torch.equal(q.cpu(), _levels((h.float() * norm.float()).cpu())[0])
    y = int8.linear_int8(q, s, w1, s1, dtype=dtype)
    ref, slack = _linear_reference(q, s, w1, s1, None, None, dtype)
    assert ((y.double() - ref).abs() <= slack).all()
    q, s = int8.silu_mul_int8(y)
    g, u = y.double().chunk(2, dim=-1)
    p = g / (1 + torch.exp(-g)) * u
    t = 127 * p / p.abs().amax(dim=-1, keepdim=True)
    assert ((q.double() - t).abs() <= 0.5 + 127 * 16.1 * F32).all()  # as in test_gate
    ref, slack = _linear_reference(q, s, w2, s2, None, h, dtype)
    assert ((out.double() - ref).abs() <= slack).all()


def test_block_in_a_graph_and_on_other_streams():
    """Captured and replayed with new inputs, eager work between; two streams at once; results equal the eager ones."""
    ops = _block_operands(256, 384, torch.bfloat16)
    xs = [_values(33, 256, torch.bfloat16, s).cuda() for s in range(4)]
    hs = [_values(33, 256, torch.bfloat16, 10 + s).cuda() for s in range(4)]
    want = [_block(x, h, *ops) for x, h in zip(xs, hs)]
    graphs = []
    for _ in range(2):  # two graphs that live side by side
        x_in, h_in = xs[0].clone(), hs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _block(x_in, h_in, *ops)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(x_in, h_in, *ops)
        graphs.append((graph, x_in, h_in, out))
    for turn in range(4):
        for i, (graph, x_in, h_in, out) in enumerate(graphs):
            k = (turn + i) % 4
            x_in.copy_(xs[k])
            h_in.copy_(hs[k])
            graph.replay()
            _block(xs[0], hs[0], *ops)
            assert torch.equal(out, want[k])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        with torch.cuda.stream(streams[turn % 2]):
            got.append(_block(xs[turn % 4], hs[turn % 4], *ops))
    torch.cuda.synchronize()
    for turn in range(6):
        assert torch.equal(got[turn], want[turn % 4])
    # the two graphs at the same time
    for i, (graph, x_in, h_in, _) in enumerate(graphs):
        x_in.copy_(xs[i])
        h_in.copy_(hs[i])
    torch.cuda.synchronize()
    for i, (graph, *_rest) in enumerate(graphs):
        with torch.cuda.stream(streams[i]):
            graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(graphs[i][3], want[i])


def test_offsets_beyond_32_bits():
    rows, width = (1 << 31) // 4096 + 3, 4096  # more than 2^31 values
    x = torch.zeros(rows, width, dtype=torch.float16, device="cuda")
    tail = _values(4, width, torch.float16).cuda()
    x[-4:] = tail
    x[0] = tail[0]
    q, s = int8.quantize_int8(x)
    wq, ws = int8.quantize_int8(tail)
    assert torch.equal(q[-4:], wq) and torch.equal(s[-4:], ws) and torch.equal(q[0], wq[0]) and not q[1:-4].any()
    back = int8.dequantize_int8(q, s)
    assert torch.equal(back[-4:], int8.dequantize_int8(wq, ws))
    norm = torch.ones(width, dtype=torch.float16, device="cuda")
    got = int8.rms_norm_int8(x, norm, residual=back, sum_out=back)
    want = int8.rms_norm_int8(tail, norm, residual=int8.dequantize_int8(wq, ws))
    for a, b in zip(got, want):
        assert torch.equal(a[-4:], b)
    del x, back, got
    w, sw = _int8(24, width).cuda(), torch.rand(24).cuda()
    y = int8.linear_int8(q, s, w, sw, dtype=torch.float32)
    assert torch.equal(y[-4:], int8.linear_int8(wq, ws, w, sw, dtype=torch.float32)) and not y[1:-4].any()
    # as the weight, and with an output of more than 2^31 values
    y = int8.linear_int8(w, sw, q, s, dtype=torch.float32)
    assert torch.equal(y[:, -4:], int8.linear_int8(w, sw, wq, ws, dtype=torch.float32))
    del y
    a, sa = _int8(40000, 16, seed=1).cuda(), torch.rand(40000).cuda()
    b, sb = _int8(60000, 16, seed=2).cuda(), torch.rand(60000).cuda()
    y = int8.linear_int8(a, sa, b, sb)
    assert torch.equal(y[-300:], int8.linear_int8(a[-300:].clone(), sa[-300:], b, sb))


# outputs that take each of the tiles of a large product: 256 x 256, 256 x 128, 128 x 128, 64 x 128, 64 x 64
TILED = [(3600, 3592), (2500, 2600), (1500, 2000), (1000, 1600), (500, 2000)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("k", [16, 128, 272, 400])  # one stage of 128 and less, odd and even numbers of them
@pytest.mark.parametrize("m,n", TILED)
def test_linear_in_each_tile(m, n, k, dtype):
    for cut in (0, 4, 1):  # outputs of a row: a multiple of 8, of 4, odd
        _linear_case(m - cut, n - cut, k, dtype, bias=cut != 4, residual=True, seed=cut)
    _linear_case(m, n, k - 1, dtype, bias=True, seed=k)  # copied to aligned rows
    _linear_case(m, n, k, dtype)


@pytest.mark.parametrize("m,n", [(9, 40), (70, 300), (520, 2000), (2500, 2600)])
def test_linear_with_rows_of_one_place(m, n):
    """Broadcast operands: every row of x, of the residual, or of the weight is the same one."""
    k = 144
    x, w = _int8(1, k, seed=1).cuda().expand(m, k), _int8(n, k, seed=2).cuda()
    xs, ws = torch.rand(m).cuda() * 0.01, (torch.rand(1).cuda() * 0.01).expand(n)
    r = torch.randn(1, n, device="cuda").bfloat16().expand(m, n)
    y = int8.linear_int8(x, xs, w, ws, residual=r, dtype=torch.bfloat16)
    ref, slack = _linear_reference(x, xs, w, ws, None, r, torch.bfloat16)
    assert ((y.double() - ref).abs() <= slack).all()
    one = _int8(1, k, seed=3).cuda()
    y = int8.linear_int8(x.contiguous(), xs, one.expand(n, k), ws, bias=r[0], dtype=torch.bfloat16)
    ref, slack = _linear_reference(x, xs, one.expand(n, k), ws, r[0], None, torch.bfloat16)
    assert ((y.double() - ref).abs() <= slack).all()


@pytest.mark.parametrize("far", ["x", "weight", "residual", "out"])
def test_linear_rows_far_apart(far):
    """Rows more than 2^20 apart, where a tile's offsets would leave the range of its descriptors."""
    m, n, k, stride = 300, 280, 160, (1 << 20) + 32
    x, w = _int8(m, k, seed=1).cuda(), _int8(n, k, seed=2).cuda()
    xs, ws = torch.rand(m).cuda() * 0.01, torch.rand(n).cuda() * 0.01
    r = torch.randn(m, n, device="cuda").half()

    def apart(t):
        to = torch.zeros((t.shape[0] - 1) * stride + t.shape[1], dtype=t.dtype, device="cuda").as_strided(t.shape, (stride, 1))
        to.copy_(t)
        return to

    want = int8.linear_int8(x, xs, w, ws, residual=r)
    out = None
    if far == "x":
        x = apart(x)
    elif far == "weight":
        w = apart(w)
    elif far == "residual":
        r = apart(r)
    else:
        out = apart(torch.empty_like(r))
    assert torch.equal(int8.linear_int8(x, xs, w, ws, residual=r, out=out), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [4096, 8190, 16384, 20000])
def test_many_wide_rows(width, dtype):
    """2048 rows and more: several chunks of a row per thread, in every operator and type."""
    rows = 2050
    x, r = _values(rows, width, dtype, seed=1), _values(rows, width, dtype, seed=2)
    w = (1 + 0.2 * _values(1, width, torch.float32, seed=3)[0]).to(dtype)
    xd, rd, wd = x.cuda(), r.cuda(), w.cuda()
    few = [int8.quantize_int8(xd[:7]), int8.rms_norm_int8(xd[:7], wd), int8.rms_norm_int8(xd[:7], wd.float(), residual=rd[:7])]
    many = [int8.quantize_int8(xd), int8.rms_norm_int8(xd, wd), int8.rms_norm_int8(xd, wd.float(), residual=rd)]
    for a, b in zip(few, many):  # one well-defined answer, but for the order of the squares' sum in 64 bits
        assert torch.equal(a[0], b[0][:7])
        assert ((a[1].double() - b[1][:7].double()).abs() <= 2.002 * F32 * a[1].double()).all()
    assert torch.equal(few[2][2], many[2][2][:7])
    last = slice(rows - 5, rows)
    for (q, scale, *h), p, norm_of in ((many[0], x[last].float(), None), (many[1], x[last].float() * w.float(), x[last]),
                                       (many[2], (x[last].float() + r[last].float()).to(dtype).float() * w.float(),
                                        (x[last].float() + r[last].float()).to(dtype))):
        ref, top = _levels(p)
        assert torch.equal(q[last].cpu(), ref)
        want = top[:, 0].double() / 127
        if norm_of is not None:
            want = want * torch.rsqrt(norm_of.double().square().mean(dim=-1) + 1e-6)
        assert ((scale[last].cpu().double() - want).abs() <= 1.001 * F32 * want).all()
    q, scale = int8.silu_mul_int8(xd)
    few_q, few_scale = int8.silu_mul_int8(xd[-7:])
    if width % 2 == 0:
        assert torch.equal(q[-7:], few_q) and torch.equal(scale[-7:], few_scale)


def test_two_threads_at_once():
    """Calls of two threads, each on a stream of its own, with workspaces in flight."""
    import threading

    cases = []
    for s in range(2):
        x, w = _int8(1100, 333, seed=s).cuda(), _int8(1201, 333, seed=5 + s).cuda()
        xs, ws = torch.rand(1100).cuda(), torch.rand(1201).cuda()
        cases.append((x, xs, w, ws, int8.linear_int8(x, xs, w, ws, dtype=torch.bfloat16)))
    torch.cuda.synchronize()
    bad = []

    def work(x, xs, w, ws, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    y = int8.linear_int8(x, xs, w, ws, dtype=torch.bfloat16)
                    q, s = int8.quantize_int8(y)
                    back = int8.dequantize_int8(q, s, dtype=torch.float32)
                    if not torch.equal(y, want) or ((back - want.float()).abs() > 0.51 * s[:, None]).any():
                        bad.append("a result differs")
        except Exception as e:  # noqa: BLE001 - reported by the test's own thread
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_copied_rows_in_a_graph():
    """A product whose operands are copied to a workspace, captured twice, replayed with eager ones between."""
    m, n, k = 1100, 1200, 333
    w, ws = _int8(n, k, seed=1).cuda(), torch.rand(n).cuda()
    xs = torch.rand(m).cuda()
    inputs = [_int8(m, k, seed=10 + i).cuda() for i in range(3)]
    want = [int8.linear_int8(x, xs, w, ws) for x in inputs]
    graphs = []
    for _ in range(2):
        x_in = inputs[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = int8.linear_int8(x_in, xs, w, ws)
        graphs.append((graph, x_in, y))
    for turn in range(6):
        for i, (graph, x_in, y) in enumerate(graphs):
            at = (turn + i) % 3
            x_in.copy_(inputs[at])
            graph.replay()
            assert torch.equal(int8.linear_int8(inputs[at], xs, w, ws), want[at])
            assert torch.equal(y, want[at])


def test_first_call_inside_a_capture():
    """In a process of its own: a kernel's LDS is allowed, and the extension loaded, while a stream is captured."""
    import subprocess
    import sys

    code = """
import torch
from triton_client_amd.ops import int8
x = torch.randint(-127, 128, (2000, 256), dtype=torch.int8, device="cuda")
s = torch.full((2000,), 0.01, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = int8.linear_int8(x, s, x, s, dtype=torch.float32)
    q, t = int8.quantize_int8(y)
for _ in range(3):
    y.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    eager = int8.linear_int8(x, s, x, s, dtype=torch.float32)
    assert torch.equal(y, eager) and torch.equal(q, int8.quantize_int8(eager)[0])
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_parameters_without_gradients():
    """Parameters are operands like any other where no gradient is recorded, and results require none."""
    x = torch.nn.Parameter(_values(6, 64, torch.float16).cuda())
    w = torch.nn.Parameter(torch.ones(64, dtype=torch.float16, device="cuda"))
    with torch.no_grad():
        got = int8.rms_norm_int8(x, w, residual=x)
    for a, b in zip(got, int8.rms_norm_int8(x.detach(), w.detach(), residual=x.detach())):
        assert torch.equal(a, b) and not a.requires_grad
    frozen = torch.nn.Parameter(x.detach(), requires_grad=False)
    assert torch.equal(int8.quantize_int8(frozen)[0], int8.quantize_int8(x.detach())[0])


def test_in_inference_mode():
    """Results are what any operator's are there, on the extension's way and on the general one."""
    x = _values(5, 64, torch.float16).cuda()
    with torch.inference_mode():
        for t in (*int8.quantize_int8(x), *int8.quantize_int8(x[:, 1:])):
            assert t.is_inference()
    assert not int8.quantize_int8(x)[0].is_inference()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_linear_does_not_depend_on_the_batch(dtype):
    """A token's outputs are the same to the bit alone, among few and among many, whatever kernel takes the product."""
    n, k = 2600, 272
    x, w = _int8(2500, k, seed=1).cuda(), _int8(n, k, seed=2).cuda()
    xs, ws = torch.rand(2500).cuda() * 0.02, torch.rand(n).cuda() * 1e-3
    b, r = torch.randn(n).to(dtype).cuda(), torch.randn(2500, n).to(dtype).cuda()
    for bias, residual in ((None, None), (b, None), (None, r), (b, r)):
        full = int8.linear_int8(x, xs, w, ws, bias=bias, residual=residual, dtype=dtype)
        for m in (1, 7, 20, 40, 100, 300, 700, 1500):
            some = int8.linear_int8(x[:m], xs[:m], w, ws, bias=bias, residual=None if residual is None else residual[:m], dtype=dtype)
            assert torch.equal(some, full[:m]), m
        for cut in (1, 4):  # rows of outputs at other addresses
            some = int8.linear_int8(x, xs, w[cut:], ws[cut:], bias=None if bias is None else bias[cut:].clone(),
                                    residual=None if residual is None else residual[:, cut:], dtype=dtype)
            assert torch.equal(some, full[:, cut:]), cut
        some = int8.linear_int8(x[:9, 1:], xs[:9], w[:, 1:], ws, bias=bias, dtype=dtype)  # at odd addresses
        many = int8.linear_int8(x[:, 1:], xs, w[:, 1:], ws, bias=bias, dtype=dtype)
        assert torch.equal(some, many[:9])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dequantize_rounds_the_fp32_product(dtype):
    """Also where the product, in fp32, falls half-way between two values of the result's type: scales of few bits."""
    q = torch.arange(-128, 128, dtype=torch.int16).to(torch.int8).repeat(20000, 1)
    g = torch.Generator().manual_seed(3)
    scale = torch.rand(20000, generator=g) + 0.01
    scale[::2] = ((scale[::2] * 4096).round() + 0.5) / 4096 * (1 + 2.0 ** -23 * torch.randint(-1, 2, (10000,), generator=g))
    for width in (256, 255, 7):
        got = int8.dequantize_int8(q[:, :width].cuda(), scale.cuda(), dtype=dtype)
        assert torch.equal(got.cpu(), (q[:, :width].float() * scale[:, None]).to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(672, 1308, 133), (120, 4160, 319), (1393, 1408, 493), (65, 700, 5), (70, 3000, 17), (100, 5000, 256),
                                   (330, 1000, 129)])
def test_linear_in_tiles_at_any_address(m, n, k, dtype):
    xb, wb = _int8(m, k + 24, seed=1, low=-128).cuda(), _int8(n, k + 40, seed=2, low=-128).cuda()
    for x_at, w_at in ((0, 0), (1, 2), (7, 13), (16, 3)):
        x, w = xb[:, x_at:x_at + k], wb[:, w_at:w_at + k]
        for cut in (0, 3):
            _linear_case(m - cut, n - cut, k, dtype, bias=True, residual=cut == 0, x=x[cut:].contiguous(), w=w[cut:])
            _linear_case(m - cut, n - cut, k, dtype, x=x[cut:], w=w[cut:])


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_tangents_and_traces_on_the_gpu():
    """Refused on the extension's way too, and plain calls again once the level or the trace has ended."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    from triton_client_amd import _native

    ops = _native.torch_ops()
    x = _values(3, 32, torch.float16).cuda()
    q, s = int8.quantize_int8(x)

    def calls(x, s):
        return (lambda: int8.quantize_int8(x), lambda: int8.silu_mul_int8(x), lambda: int8.dequantize_int8(q, s),
                lambda: int8.rms_norm_int8(x, x[0], residual=x), lambda: int8.linear_int8(q, s, q, s))

    with forward_ad.dual_level():
        xd, sd = forward_ad.make_dual(x, x), forward_ad.make_dual(s, s)
        assert ops.quantize(xd, False) is None and ops.dequantize(q, sd, 1) is None
        for call in calls(xd, sd):
            with pytest.raises(ValueError, match="no derivative"):
                call()
        assert ops.quantize(x, False) is not None

    def traced(x):
        assert ops.quantize(x, False) is None
        for call in calls(x, s):
            with pytest.raises(ValueError, match="traced"):
                call()
        return x + 1

    torch.jit.trace(traced, (x,), check_trace=False)
    make_fx(traced)(x)
    make_fx(traced, pre_dispatch=True)(x)
    assert torch.equal(ops.quantize(x, False)[0], q)


def test_plain_calls_under_other_modes():
    """A mode that watches operators, or a wrapped program, changes nothing."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = _values(3, 32, torch.float16).cuda()
    q, s = int8.quantize_int8(x)
    with Watch():
        got = int8.quantize_int8(x)
        strided = int8.quantize_int8(x[:, ::2])
    assert torch.equal(got[0], q) and torch.equal(got[1], s)
    assert torch.equal(strided[0], int8.quantize_int8(x[:, ::2])[0])
    compiled = torch.compile(lambda t: int8.dequantize_int8(*int8.quantize_int8(t + 1), dtype=torch.float32) * 2, backend="eager")
    want = int8.dequantize_int8(*int8.quantize_int8(x + 1), dtype=torch.float32) * 2
    assert torch.equal(compiled(x), want) and torch.equal(compiled(x), want)


def test_destinations_that_a_backward_pass_has_saved():
    """Writing to one is found out when the gradient is taken, as after any of torch's operators in place."""
    rows = _values(4, 32, torch.float32).cuda()
    weight = torch.ones(32, device="cuda")
    q, s = int8.quantize_int8(rows)
    wq, ws = int8.quantize_int8(torch.eye(32, device="cuda"))
    writes = [(rows, lambda t: int8.rms_norm_int8(t, weight, residual=rows, sum_out=t)),
              (rows, lambda t: int8.rms_norm_int8(rows, weight, residual=t, sum_out=t)),
              (rows, lambda t: int8.dequantize_int8(q, s, out=t)), (rows, lambda t: int8.dequantize_int8(q, s, out=t.view(4, 32))),
              (rows, lambda t: int8.linear_int8(q, s, wq, ws, residual=t, out=t)), (s, lambda t: int8.quantize_int8(rows, scale=t)),
              (s, lambda t: int8.rms_norm_int8(rows, weight, scale=t))]
    for like, write in writes:
        t, p = like.clone(), torch.ones_like(like, requires_grad=True)
        y = (t * p).sum()  # saves t for p's gradient
        version = t._version
        write(t)
        assert t._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    t = torch.empty(4, 32, dtype=torch.int8, device="cuda")
    int8.quantize_int8(rows, out=t)
    assert t._version == 1
    # inputs and untouched destinations keep their versions; inference tensors, which have none, are written all the same
    assert rows._version == weight._version == q._version == s._version == 0
    empty = torch.empty(0, 32, device="cuda")
    int8.dequantize_int8(q[:0], s[:0], out=empty)
    assert empty._version == 0
    with torch.inference_mode():
        t = torch.empty(4, 32, device="cuda")
    int8.dequantize_int8(q, s, out=t)
    with torch.inference_mode():
        int8.dequantize_int8(q, s, out=t)
    assert torch.equal(t, int8.dequantize_int8(q, s, dtype=torch.float32))


def test_destinations_in_a_graph():
    """A capture enqueues, replays write: the version counts the call, and replays are as eager calls."""
    rows = _values(4, 32, torch.float32).cuda()
    q, s = int8.quantize_int8(rows)
    t = torch.zeros(4, 32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        int8.dequantize_int8(q, s, out=t)
    for _ in range(3):
        t.zero_()
        graph.replay()
        assert torch.equal(t, int8.dequantize_int8(q, s, dtype=torch.float32))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [5, 1030, 4100])
@pytest.mark.parametrize("width", [4104, 8200, 12000, 16384, 20000])
def test_gate_of_wide_rows(width, rows, dtype):
    """Against the formula, in every split of a row: chunks that fill the threads of a block, and that do not."""
    g = torch.Generator(device="cuda").manual_seed(width)
    x = (2 * torch.randn(rows, 2 * width, generator=g, device="cuda")).to(dtype)
    q, scale = int8.silu_mul_int8(x)
    for at in (0, rows // 2, rows - 3):
        gate, up = x[at:at + 3].double().chunk(2, dim=-1)
        p = gate / (1 + torch.exp(-gate)) * up
        top = p.abs().amax(dim=-1, keepdim=True)
        assert ((q[at:at + 3].double() - 127 * p / top).abs() <= 0.5 + 127 * 16.1 * F32).all()  # as in test_gate
        assert ((scale[at:at + 3].double() - top[:, 0] / 127).abs() <= 9.1 * F32 * top[:, 0] / 127).all()
    few = int8.silu_mul_int8(x[-4:])  # in the split of few rows
    assert torch.equal(q[-4:], few[0]) and torch.equal(scale[-4:], few[1])
