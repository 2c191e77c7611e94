"""Rows in 8 bits and their products (``int8.py``) against the formulas in 64 bits.

Bounds.  A whole number is the nearest to 127 p / max|p|, computed with at most
five roundings of 2^-24: off from the quotient by 1/2 + 127 * 5 * 2^-24 < 1/2 +
4e-5.  Scales: three such roundings, with a norm's r 5e-6 more.  A product's sum
is exact; its conversion, the two scales and the bias round by 2^-24 each, then
the output to its type.  Gated: a relative error d of the gate is (1 + |gate|) d
in silu, the exponential's argument and result are off by less than 2^-22 (1 +
|gate|), the division by 2^-22: together below 2^-20 (1 + |gate|)."""

import pytest
import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# one element; odd; a warp; a CTA; wide; past the registers; more rows than one, and than four, to an SM
ROWS = [(1, 1), (3, 17), (9, 40), (5, 256), (2, 1000), (7, 896), (33, 3584), (4, 4097), (3, 18944), (2, 33000), (2, 65536),
        (700, 64), (300, 896), (200, 18944), (1000, 1000)]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check_whole(q, scale, p, want_scale, off=0.0):
    """q of rows p (64 bits, up to a positive factor)."""
    top = p.abs().amax(-1, keepdim=True)
    n = torch.where(top > 0, 127 * p / top, torch.zeros_like(p))
    assert q.dtype == torch.int8 and scale.dtype == torch.float32
    assert ((q.double() - n).abs() <= 0.5 + 4e-5).all()
    # a scale below the smallest normal number 2^-126 is a multiple of 2^-149 and rounds by half of that
    assert ((scale.double() - want_scale).abs() <= want_scale * (4 * 2 ** -24 + off) + 2.0 ** -150).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", ROWS)
def test_quantize(mrsa, cuda_device, rows, dim, kind):
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn(rows, dim, device=cuda_device, generator=g).to(TYPES[kind])
    q, scale = mrsa.quantize_int8(x)
    assert q.shape == x.shape and scale.shape == (rows,)
    p = x.double()
    check_whole(q, scale, p, p.abs().amax(-1) / 127)
    assert (q.abs().amax(-1) == 127).all() or (x == 0).all(-1).any()
    # what comes back is within half a step
    back = q.double() * scale.double()[:, None]
    assert ((back - p).abs() <= scale.double()[:, None] * (0.5 + 1e-4)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", ROWS)
def test_norm_int8(mrsa, cuda_device, rows, dim, kind):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x, r = (torch.randn(rows, dim, device=cuda_device, generator=g).to(TYPES[kind]) for _ in range(2))
    w = (1 + 0.3 * torch.randn(dim, device=cuda_device, generator=g)).to(TYPES[kind])
    q, scale, h = mrsa.add_rms_norm_int8(x, r, w, 1e-6)
    assert torch.equal(h, x + r)
    for h, (q, scale) in ((h, (q, scale)), (x, mrsa.add_rms_norm_int8(x, None, w, 1e-6)[:2])):
        d = h.double()
        p = d * w.double()
        check_whole(q, scale, p, p.abs().amax(-1) / 127 / (d.square().mean(-1) + 1e-6).sqrt(), 5e-6)


def nearest(p):
    """The whole numbers of rows p, in 64 bits, of two the even one."""
    return torch.round(p * (127.0 / p.abs().amax(-1, keepdim=True)))


# a few rows, more than one and than four to an SM; by words, by elements, past the registers
@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", [(2, 40), (300, 256), (2, 999), (1000, 1000), (700, 3584), (3, 4097), (3, 18944), (700, 18944),
                                      (2, 20001), (2, 65536)])
def test_whole_numbers_are_the_nearest(mrsa, cuda_device, rows, dim, kind):
    """Every one of them, with as many half-way as a row can have."""
    dev, dtype = cuda_device, TYPES[kind]
    g = torch.Generator(device=dev).manual_seed(9)
    # k + 1/2 times 1 / 64, and 127 / 64 once: half-way exactly, as are the bounds' quotients in 64 bits
    half_way = (torch.randint(-127, 127, (rows, dim), device=dev, generator=g).double() + 0.5) / 64
    half_way[torch.arange(rows, device=dev), torch.randint(0, dim, (rows,), device=dev, generator=g)] = 127 / 64
    x = half_way.to(dtype)
    sign = torch.where(torch.rand(dim, device=dev, generator=g) < 0.5, -1.0, 1.0).to(dtype)
    want = torch.round(half_way * 64)
    assert torch.equal(mrsa.quantize_int8(x)[0].double(), want)
    assert torch.equal(mrsa.add_rms_norm_int8(x, None, sign, 1e-6)[0].double(), want * sign.double())
    x, r = (torch.randn(rows, dim, device=dev, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(dim, device=dev, generator=g)).to(dtype)
    assert torch.equal(mrsa.quantize_int8(x)[0].double(), nearest(x.double()))
    q, _, h = mrsa.add_rms_norm_int8(x, r, w, 1e-6)
    # (products of 16-bit numbers are exact in fp32; those of fp32 numbers are rounded to it)
    assert torch.equal(q.double(), nearest((h.float() * w.float()).double()))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 7, 64, 999, 18944])
@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -101, 2.0 ** -99, 2.0 ** 99, 2.0 ** 101, 2.0 ** 125, 2.0 ** 126])
def test_rows_of_any_size(mrsa, cuda_device, rows, dim, size):
    """From numbers whose quotients pass fp32's range to the largest there are (below 2^128)."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(rows, dim, device=dev, generator=g).clamp(-3.9, 3.9) * size
    w = torch.rand(dim, device=dev, generator=g) + 0.5
    for kind in ("fp32", "bf16"):
        a, b = x.to(TYPES[kind]), w.to(TYPES[kind])
        q, scale = mrsa.quantize_int8(a)
        p = a.double()
        check_whole(q, scale, p, p.abs().amax(-1) / 127)
        q, scale, _ = mrsa.add_rms_norm_int8(a, None, b, 1e-6)
        p = p * b.double()
        check_whole(q, scale, p, p.abs().amax(-1) / 127 / (a.double().square().mean(-1) + 1e-6).sqrt(), 5e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 999, 5000, 18944, 40000])
@pytest.mark.parametrize("rows", [6, 400])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_products_of_any_size(mrsa, cuda_device, rows, dim, kind):
    """Rows and weights whose products are past fp32's largest number, below its smallest normal one, or
    both in turn, while the norm itself is not."""
    dev, dtype = cuda_device, TYPES[kind]
    g = torch.Generator(device=dev).manual_seed(13)
    x = torch.randn(rows, dim, device=dev, generator=g).clamp(-3.9, 3.9)
    w = torch.rand(dim, device=dev, generator=g) + 0.5
    w[torch.rand(dim, device=dev, generator=g) < 0.1] = 0
    sizes = torch.tensor([2.0 ** -140, 2.0 ** -75, 2.0 ** -20, 1.0, 2.0 ** 70, 2.0 ** 125], device=dev, dtype=torch.float64)
    for size in (2.0 ** -130, 2.0 ** -60, 2.0 ** 40, 2.0 ** 126):
        for eps in (1e-6, 1e-12):
            h = (x.double() * sizes[torch.arange(rows, device=dev) % 6, None]).to(dtype)
            b = (w.double() * size).to(dtype)
            q, scale, _ = mrsa.add_rms_norm_int8(h, None, b, eps)
            p = h.double() * b.double()
            check_whole(q, scale, p, p.abs().amax(-1) / 127 / (h.double().square().mean(-1) + eps).sqrt(), 5e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(3, 64), (400, 999), (400, 3584), (3, 40000)])
def test_weights_that_are_not_finite(mrsa, cuda_device, rows, dim):
    """A row times a weight that is not finite has no scale, a zero in its place neither; rows of zeros beside others."""
    dev = cuda_device
    x = torch.randn(rows, dim, device=dev, generator=torch.Generator(device=dev).manual_seed(14))
    x[1], x[2, 5] = 0, 0
    w = torch.ones(dim, device=dev)
    q, scale, _ = mrsa.add_rms_norm_int8(x, None, w, 1e-6)
    assert scale[1] == 0 and not q[1].any() and torch.equal(scale == 0, (x == 0).all(-1))
    for bad in ("inf", "nan"):
        w[5] = float(bad)
        q, scale, _ = mrsa.add_rms_norm_int8(x, None, w, 1e-6)
        assert scale.isnan().all() and not q.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 999])
def test_extreme_rows(mrsa, cuda_device, dim):
    dev = cuda_device
    x = torch.randn(8, dim, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    x[0] = 0
    x[1] *= 1e37
    x[2] *= 1e-35
    x[3] = x[3].sign() * 2.0 ** -140          # below the smallest normal number
    x[4, 3] = float("nan")
    x[5, 4] = float("-inf")
    x[6, 5], x[6, 6] = float("inf"), float("nan")
    q, scale = mrsa.quantize_int8(x)
    for i in (1, 2, 7):
        check_whole(q[i:i + 1], scale[i:i + 1], x[i:i + 1].double(), x[i:i + 1].double().abs().amax(-1) / 127)
    assert (q[3] == x[3].sign() * 127).all() and (scale[3].double() * 127 - 2.0 ** -140).abs() <= 127 * 2.0 ** -150
    assert scale[0] == 0 and not q[0].any()
    assert scale[4:7].isnan().all() and not q[4:7].any()
    w = torch.randn(dim, device=dev)
    q, scale, _ = mrsa.add_rms_norm_int8(x, None, w, 1e-6)
    for i in (1, 2, 7):
        d = x[i:i + 1].double()
        p = d * w.double()
        check_whole(q[i:i + 1], scale[i:i + 1], p, p.abs().amax(-1) / 127 / (d.square().mean(-1) + 1e-6).sqrt(), 5e-6)
    assert scale[0] == 0 and not q[0].any()
    assert scale[4:7].isnan().all() and not q[4:7].any()
    # what is computed from such a row is not a number either; the other rows are what they were
    q, scale = mrsa.quantize_int8(x)
    wq, ws = mrsa.quantize_int8(torch.randn(40, dim, device=dev))
    y = mrsa.linear_int8(q, scale, wq, ws, dtype=torch.float32)
    assert y[4:7].isnan().all() and (y[0] == 0).all() and y[7].isfinite().all()


def operands(dev, m, n, k, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randint(-128, 128, (m, k), device=dev, generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), device=dev, generator=g, dtype=torch.int8)
    return (q, torch.rand(m, device=dev, generator=g) * 0.1 + 0.01, w, (torch.rand(n, device=dev, generator=g) + 0.1) / k,
            torch.randn(n, device=dev, generator=g))


def check_linear(y, q, scale, w, ws, bias):
    s = (q.double() @ w.double().T) * scale.double()[..., None] * ws.double()
    want = s if bias is None else s + bias.double()
    size = s.abs() + (0 if bias is None else bias.double().abs())
    tiny = 3e-8 if y.dtype == torch.float16 else 0
    assert ((y.double() - want).abs() <= half(y.dtype) * want.abs() + 5 * 2 ** -24 * size + tiny).all()


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 7, 15), (1, 4608, 3584), (3, 130, 129), (5, 33, 4000), (16, 256, 128), (17, 264, 127),
          (31, 512, 896), (33, 1001, 517), (64, 640, 1024), (65, 128, 18944), (100, 4608, 896), (128, 384, 130),
          (129, 257, 257), (256, 3584, 1000), (300, 515, 96), (511, 72, 640), (1000, 2000, 333), (2049, 300, 256),
          (1, 40000, 64), (700, 8, 20000), (300, 515, 12999), (520, 130, 7000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(mrsa, cuda_device, m, n, k):
    q, scale, w, ws, bias = operands(cuda_device, m, n, k)
    for i, dtype in enumerate(TYPES.values()):
        y = mrsa.linear_int8(q, scale, w, ws, dtype=dtype)
        assert y.shape == (m, n) and y.dtype == dtype
        check_linear(y, q, scale, w, ws, None)
        b = bias.to(list(TYPES.values())[(i + 1) % 3])
        check_linear(mrsa.linear_int8(q, scale, w, ws, b, dtype=dtype), q, scale, w, ws, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,f,k", [(1, 128, 16), (1, 18944, 3584), (3, 256, 129), (17, 384, 896), (32, 1024, 300),
                                   (70, 128, 4000), (130, 640, 256), (257, 512, 1000), (1025, 256, 64),
                                   (300, 256, 5000)])
def test_swiglu(mrsa, cuda_device, m, f, k):
    q, scale, w, ws, _ = operands(cuda_device, m, 2 * f, k, 1)
    ws = ws * 20 * k ** 0.5 / 74           # gates of a few units
    s = ((q.double() @ w.double().T) * scale.double()[..., None] * ws.double()).view(m, -1, 2, 128)
    gate, up = s[:, :, 0].flatten(1), s[:, :, 1].flatten(1)
    want = gate * torch.sigmoid(gate) * up
    for dtype in TYPES.values():
        y = mrsa.swiglu_int8(q, scale, w, ws, dtype=dtype)
        assert y.shape == (m, f) and y.dtype == dtype
        # for a gate below -87 (the first of these have such) 1 + exp(-gate) >= 2^126 may pass the largest fp32
        # number, and the quotient be 0: |silu| < |gate| 2^-126 is what is lost, and a product below the type's
        # smallest normal number 2^-126 rounds by a 2^-134 (bf16) at most
        tiny = 3e-8 if dtype == torch.float16 else (gate * up).abs() * 2.0 ** -125 + 2.0 ** -134
        bound = want.abs() * (half(dtype) + 2 ** -20 * (1 + gate.abs())) + tiny
        # past the type's largest number (fp16: 65504, at gates of hundreds times as much) a value rounds to infinity
        most = torch.finfo(dtype).max
        past = want.abs() - bound > most
        assert (y[past].double() == want[past].sign() * float("inf")).all()
        y = torch.where(y.isinf() & (want.abs() + bound > most), want.sign() * most, y.double())
        assert ((y - want.clamp(-most, most)).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2500, 4001, 333), (4097, 2600, 1000), (8191, 4608, 130), (2048, 5000, 640)])
def test_linear_of_many_rows(mrsa, cuda_device, m, n, k):
    """Products that the kernel for many rows takes (a tile of 128 x 256 to each SM), two and more tiles of 256 x 256 to each
    pair of SMs: all types and biases, rows of C on and off 16-byte boundaries, ragged edges."""
    assert (m + 127) // 128 * ((n + 255) // 256) > 2 * torch.cuda.get_device_properties(cuda_device).multi_processor_count
    q, scale, w, ws, bias = operands(cuda_device, m, n, k, 10)
    for i, dtype in enumerate(TYPES.values()):
        check_linear(mrsa.linear_int8(q, scale, w, ws, dtype=dtype), q, scale, w, ws, None)
        b = bias.to(list(TYPES.values())[(i + 1) % 3])
        check_linear(mrsa.linear_int8(q, scale, w, ws, b, dtype=dtype), q, scale, w, ws, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_swiglu_of_many_rows(mrsa, cuda_device, kind):
    """Three tiles of 256 x 256 and more to each pair of SMs; the rows as calls of a few give them, which
    test_swiglu compares with 64 bits."""
    m, f, k = 4000, 2048, 700
    assert (m + 255) // 256 * (2 * f // 256) > 3 * torch.cuda.get_device_properties(cuda_device).multi_processor_count // 2
    q, scale, w, ws, _ = operands(cuda_device, m, 2 * f, k, 11)
    ws = ws * 20 * k ** 0.5 / 74
    y = mrsa.swiglu_int8(q, scale, w, ws, dtype=TYPES[kind])
    for at in range(0, m, 128):
        assert torch.equal(mrsa.swiglu_int8(q[at:at + 128], scale[at:at + 128], w, ws, dtype=TYPES[kind]), y[at:at + 128])


@pytest.mark.gpu
def test_sums_are_exact(mrsa, cuda_device):
    """The longest sum that 32 bits hold, and single ones among zeros."""
    dev = cuda_device
    k = 131071
    for m in (2, 200):
        q = torch.full((m, k), -128, dtype=torch.int8, device=dev)
        q[1, 1:] = 0
        y = mrsa.linear_int8(q, torch.ones(m, device=dev), q[:2], torch.ones(2, device=dev), dtype=torch.float32)
        assert y[0].tolist() == [float(128 * 128 * k), 128.0 * 128] and y[1].tolist() == [128.0 * 128] * 2
    for m, n, k in ((5, 140, 300), (140, 300, 140)):
        eye = torch.zeros(m, k, dtype=torch.int8, device=dev)
        eye[torch.arange(m), torch.arange(m)] = 1
        w = torch.randint(-128, 128, (n, k), device=dev, dtype=torch.int8)
        y = mrsa.linear_int8(eye, torch.ones(m, device=dev), w, torch.ones(n, device=dev), dtype=torch.float32)
        assert torch.equal(y, w[:, :m].T.float())


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_others(mrsa, cuda_device):
    q, scale, w, ws, bias = operands(cuda_device, 700, 520, 1000, 2)
    y = mrsa.linear_int8(q, scale, w, ws, bias)
    for rows in (slice(0, 1), slice(3, 40), slice(100, 230), slice(690, 700), slice(0, 400)):
        assert torch.equal(mrsa.linear_int8(q[rows].clone(), scale[rows].clone(), w, ws, bias), y[rows])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [4001, 4608])
def test_rows_with_bias_do_not_depend_on_the_others(mrsa, cuda_device, n, kind):
    """Rows of the kernels for many rows and for few, their outputs' last bits and the bias's rounding."""
    m = 2500
    assert (m + 127) // 128 * ((n + 255) // 256) > 2 * torch.cuda.get_device_properties(cuda_device).multi_processor_count
    q, scale, w, ws, bias = operands(cuda_device, m, n, 333, 12)
    y = mrsa.linear_int8(q, scale, w, ws, bias, dtype=TYPES[kind])
    for rows in (slice(0, 1), slice(3, 40), slice(100, 228), slice(2400, 2500), slice(500, 1100)):
        assert torch.equal(mrsa.linear_int8(q[rows], scale[rows], w, ws, bias, dtype=TYPES[kind]), y[rows])


@pytest.mark.gpu
def test_layouts(mrsa, cuda_device):
    """Leading dimensions, strides, unaligned rows, one row, none."""
    dev = cuda_device
    q, scale, w, ws, bias = operands(dev, 24, 100, 208, 3)
    want = mrsa.linear_int8(q, scale, w, ws, bias, dtype=torch.float32)
    check_linear(want, q, scale, w, ws, bias)

    def same(*a):
        y = mrsa.linear_int8(*a, dtype=torch.float32)
        assert torch.equal(y.reshape(want.shape), want)
        return y

    assert same(q.view(2, 3, 4, 208), scale.view(2, 3, 4), w, ws, bias).shape == (2, 3, 4, 100)
    for pad in (16, 7):
        wide = torch.zeros(24, 208 + pad, dtype=torch.int8, device=dev)
        wide[:, :208] = q
        same(wide[:, :208], scale, w, ws, bias)
        ww = torch.zeros(100, 208 + pad, dtype=torch.int8, device=dev)
        ww[:, pad:] = w
        same(q, scale, ww[:, pad:], ws, bias)
    flat = torch.zeros(24 * 208 + 1, dtype=torch.int8, device=dev)
    flat[1:] = q.flatten()
    same(flat[1:].view(24, 208), scale, w, ws, bias)
    same(q.T.contiguous().T, scale, w.T.contiguous().T, ws, bias)
    same(q, scale.repeat_interleave(2)[::2], w, ws.repeat_interleave(3)[::3], bias.repeat_interleave(2)[::2])
    one = mrsa.linear_int8(q[5], scale[5], w, ws, bias, dtype=torch.float32)
    assert one.shape == (100,) and torch.equal(one, want[5])
    assert torch.equal(mrsa.linear_int8(q[5:6].expand(4, 208), scale[5:6].expand(4), w, ws, bias, dtype=torch.float32),
                       want[5:6].expand(4, 100))
    none = mrsa.linear_int8(q[:0].view(3, 0, 208), scale[:0].view(3, 0), w, ws, bias)
    assert none.shape == (3, 0, 100)
    q0, s0 = mrsa.quantize_int8(torch.zeros(3, 0, 50, device=dev))
    assert q0.shape == (3, 0, 50) and s0.shape == (3, 0)
    # rows that quantize_int8 lays out itself, of an odd width, in several dimensions
    x = torch.randn(2, 3, 4, 209, device=dev)
    qx, sx = mrsa.quantize_int8(x)
    assert qx.stride() == (3 * 4 * 224, 4 * 224, 224, 1) and sx.shape == (2, 3, 4)
    wq, wsc = mrsa.quantize_int8(torch.randn(30, 209, device=dev))
    y = mrsa.linear_int8(qx, sx, wq, wsc, dtype=torch.float32)
    check_linear(y.flatten(0, 2), qx.reshape(24, 209), sx.flatten(), wq, wsc, None)
    xt = torch.randn(64, 7, device=dev).T                  # a transposed input
    q1, s1 = mrsa.quantize_int8(xt)
    q2, s2 = mrsa.quantize_int8(xt.contiguous())
    assert torch.equal(q1, q2) and torch.equal(s1, s2)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (2, 16), (5, 17), (1000, 31), (7, 4097), (40, 1003)])
def test_rows_off_boundaries(mrsa, cuda_device, rows, k):
    """Rows at every offset of a 16-byte boundary, at the very ends of their memory, at any distance."""
    L, dev = mrsa._lib, cuda_device
    for off in range(0, 16, 5):
        for pad in (0, 1, 2, 13):
            flat = torch.randint(-128, 128, (off + (rows - 1) * (k + pad) + k,), device=dev, dtype=torch.int8)
            x = torch.as_strided(flat, (rows, k), (k + pad, 1), off)
            pitch = (k + 15) // 16 * 16
            y = torch.full((rows, pitch), 77, dtype=torch.int8, device=dev)
            L.call("mrsa_align_rows_int8", L.ptr(x), k + pad, L.ptr(y), pitch, rows, k, L.stream_of(x))
            assert torch.equal(y[:, :k], x) and not y[:, k:].any()


@pytest.mark.gpu
def test_offsets_past_32_bits(mrsa, cuda_device):
    """More than 2^31 elements in, and out of a product: the last rows as by themselves."""
    dev, n = cuda_device, 530_000
    x = torch.empty(n, 4096, device=dev, dtype=torch.bfloat16).normal_()
    q, scale = mrsa.quantize_int8(x)
    few, fs = mrsa.quantize_int8(x[-3:].clone())
    assert torch.equal(q[-3:], few) and torch.equal(scale[-3:], fs)
    w, ws = mrsa.quantize_int8(torch.randn(4608, 4096, device=dev))
    y = mrsa.linear_int8(q, scale, w, ws)
    assert y.numel() > 2 ** 31 and torch.equal(y[-3:], mrsa.linear_int8(few, fs, w, ws))
    del y
    off = x.view(-1)[1:1 + 529_000 * 4095].view(529_000, 4095)
    q, scale = mrsa.quantize_int8(off)
    few, fs = mrsa.quantize_int8(off[-3:].clone())
    assert torch.equal(q[-3:], few) and torch.equal(scale[-3:], fs)


@pytest.mark.gpu
def test_streams_and_graphs(mrsa, cuda_device):
    """A layer of few rows and one of many on two streams at once, and in two graphs replayed together."""
    dev = cuda_device
    sets = [operands(dev, 32, 4608, 3584, 4), operands(dev, 1024, 896, 4000, 5), operands(dev, 200, 3584, 8000, 6)]
    want = [mrsa.linear_int8(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in sets]
    for _ in range(5):
        for s, ops, out in zip(streams, sets, got):
            with torch.cuda.stream(s):
                out.append(mrsa.linear_int8(*ops))
    torch.cuda.synchronize()
    for outs, y in zip(got, want):
        assert all(torch.equal(o, y) for o in outs)
    graphs, outs = [], []
    for s, ops in zip(streams, sets):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(mrsa.linear_int8(*ops))
        graphs.append(g)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o, y in zip(outs, want))
    assert mrsa._lib.load().mrsa_device_error_flags(0) == 0


@pytest.mark.gpu
def test_a_layer_as_it_is_used(mrsa, cuda_device):
    """Norm, q/k/v, MLP and residual of the Dream-shaped layer, one operator after the other, against the same steps
    in 64 bits from the whole numbers that the operators gave."""
    from mrsa_b200.dense import interleave_gate_up

    dev, h, f, rows = cuda_device, 896, 1024, 77
    g = torch.Generator(device=dev).manual_seed(7)

    def t(*shape, size=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * size).bfloat16()

    x, delta, nw = t(1, rows, h), t(1, rows, h), t(h, size=0.1) + 1
    wgu, sgu = mrsa.quantize_int8(interleave_gate_up(t(f, h, size=0.05), t(f, h, size=0.05)))
    wd, sd = mrsa.quantize_int8(t(h, f, size=0.05))
    q, s, stream = mrsa.add_rms_norm_int8(delta, x, nw, 1e-6)
    act = mrsa.swiglu_int8(q, s, wgu, sgu)
    qa, sa = mrsa.quantize_int8(act)
    out = mrsa.linear_int8(qa, sa, wd, sd)
    q2, s2, last = mrsa.add_rms_norm_int8(out, stream, nw, 1e-6)
    assert torch.equal(stream, x + delta) and torch.equal(last, out + stream)
    p = ((q.double() * s.double()[..., None]) @ (wgu.double() * sgu.double()[:, None]).T).view(rows, -1, 2, 128)
    gate, up = p[:, :, 0].flatten(1), p[:, :, 1].flatten(1)
    want = gate * torch.sigmoid(gate) * up
    assert ((act[0].double() - want).abs() <= want.abs() * (2 ** -8 + 2 ** -20 * (1 + gate.abs())) + 1e-12).all()
    check_whole(qa[0], sa[0], act[0].double(), act[0].double().abs().amax(-1) / 127)
    check_linear(out[0], qa[0], sa[0], wd, sd, None)
    d = last.double()
    v = d * nw.double()
    check_whole(q2, s2, v, v.abs().amax(-1) / 127 / (d.square().mean(-1) + 1e-6).sqrt(), 5e-6)


@pytest.mark.gpu
def test_refusals(mrsa, cuda_device):
    dev = cuda_device
    q, scale, w, ws, bias = operands(dev, 4, 256, 64, 8)
    f = mrsa.linear_int8
    for bad, match in [
        (lambda: f(q.float(), scale, w, ws), "INT8"),
        (lambda: f(q, scale, w.short(), ws), "INT8"),
        (lambda: f(q.cpu(), scale, w, ws), "CUDA"),
        (lambda: f(q, scale, w.cpu(), ws), "CUDA"),
        (lambda: f(q, scale, w[:, :32], ws), "share"),
        (lambda: f(q, scale, w[0], ws), "N, K"),
        (lambda: f(q, scale, w[:0], ws[:0]), "rows"),
        (lambda: f(q, scale[:3], w, ws), "scale"),
        (lambda: f(q, scale[:, None], w, ws), "scale"),
        (lambda: f(q, scale.half(), w, ws), "scale"),
        (lambda: f(q, scale, w, ws[:5]), "weight_scale"),
        (lambda: f(q, scale, w, ws.cpu()), "weight_scale"),
        (lambda: f(q, scale, w, ws, bias[:7]), "bias"),
        (lambda: f(q, scale, w, ws, bias.double()), "bias"),
        (lambda: f(q, scale, w, ws, bias.cpu()), "bias"),
        (lambda: f(q, scale, w, ws, dtype=torch.float64), "dtype"),
        (lambda: f(q[:, :0], scale, w[:, :0], ws), "at least 1"),
        (lambda: mrsa.swiglu_int8(q, scale, w[:128], ws[:128]), "256"),
        (lambda: mrsa.quantize_int8(torch.zeros(3, 8)), "CUDA"),
        (lambda: mrsa.quantize_int8(q), "BF16"),
        (lambda: mrsa.quantize_int8(torch.zeros((), device=dev)), "at least 1"),
        (lambda: mrsa.add_rms_norm_int8(bias.view(4, 64), None, bias[:63], 1e-6), "weight"),
        (lambda: mrsa.add_rms_norm_int8(bias.view(4, 64), None, bias[:64], 0.0), "eps"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(TypeError):
        f(q, scale, w, ws, dtype="bf16")
    long = torch.zeros(1, 131072, dtype=torch.int8, device=dev)
    with pytest.raises(ValueError, match="131071"):
        f(long, scale[:1], long, ws[:1])
    x = torch.zeros(2, 64, device=dev, requires_grad=True)
    for lost in (lambda: mrsa.quantize_int8(x), lambda: mrsa.add_rms_norm_int8(x, None, bias[:64], 1e-6),
                 lambda: mrsa.add_rms_norm_int8(x.detach(), x, bias[:64], 1e-6),
                 lambda: f(q, scale.clone().requires_grad_(), w, ws), lambda: f(q, scale, w, ws.clone().requires_grad_()),
                 lambda: f(q, scale, w, ws, bias.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="forward-only"):
            lost()
    with torch.no_grad():
        mrsa.quantize_int8(x)


def test_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib

    def rc(a=4096, b=4096, sa=4096, sb=4096, bias=0, c=4096, m=4, n=256, k=64, pa=64, pb=64, dtype=0, bt=0, ep=0):
        return lib.mrsa_gemm_int8(L.GEMM_INT8_ARGS.pack(a, b, sa, sb, bias, c, m, n, k, pa, pb, dtype, bt, ep), None)

    assert lib.mrsa_gemm_int8(None, None) == L.ERR_NULL
    assert all(rc(**{x: 0}) == L.ERR_NULL for x in ("a", "b", "sa", "sb", "c"))
    assert rc(m=-1) == L.ERR_SHAPE and rc(n=0) == L.ERR_SHAPE and rc(k=0) == L.ERR_SHAPE
    assert rc(k=131072, pa=1 << 18, pb=1 << 18) == L.ERR_SHAPE and rc(pa=48) == L.ERR_SHAPE and rc(pb=48) == L.ERR_SHAPE
    assert rc(n=128, ep=1) == L.ERR_SHAPE and rc(ep=2) == L.ERR_ARG and rc(bias=4096, ep=1) == L.ERR_ARG
    assert rc(dtype=3) == L.ERR_ARG and rc(bias=4096, bt=9) == L.ERR_ARG
    assert rc(a=4100) == L.ERR_ALIGN and rc(pa=72) == L.ERR_ALIGN and rc(c=4097) == L.ERR_ALIGN
    assert rc(m=0) == 0
    q8 = lib.mrsa_quantize_int8
    assert q8(0, 8, 4096, 16, 4096, 2, 8, 0, None) == L.ERR_NULL and q8(4096, 8, 4096, 16, 4096, 2, 0, 0, None) == L.ERR_SHAPE
    assert q8(4096, 8, 4096, 16, 4096, 2, 8, 3, None) == L.ERR_ARG and q8(4097, 8, 4096, 16, 4096, 2, 8, 0, None) == L.ERR_ALIGN
    assert q8(4096, 8, 4096, 16, 4096, 0, 8, 0, None) == 0
    assert L.GEMM_INT8_ARGS.size == 104
    al = lib.mrsa_align_rows_int8
    assert al(0, 8, 4096, 16, 2, 8, None) == L.ERR_NULL and al(4096, 8, 4096, 16, 2, 0, None) == L.ERR_SHAPE
    assert al(4096, 8, 4096, 16, 2, 17, None) == L.ERR_SHAPE and al(4096, 8, 4096, 24, 2, 8, None) == L.ERR_ALIGN
    assert al(4096, -8, 4096, 16, 2, 8, None) == L.ERR_SHAPE and al(4096, 8, 4096, 16, 0, 8, None) == 0
