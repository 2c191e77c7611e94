"""The norm with the residual's addition and its gradient (``dense.add_rms_norm``)
against the formulas in 64 bits.

Bounds.  h is one fp32 sum rounded to the type, as torch's own addition: equal.
y is a product of three (roundings of 2^-24 each) with r, whose sum of squares a
thread adds in a chain of at most 128 before a tree of at most 10: r is off by
half of 138 * 2^-24 at most, y by 5e-6 and a rounding to its type.  The
gradient's sums are such chains too, so they are off by 1e-5 of the sums of
their terms' magnitudes."""

import subprocess
import sys

import pytest
import torch

from conftest import ROOT

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# one element; odd; a warp; a CTA; unaligned and wide rows; past the registers
SIZES = [(1, 1), (3, 17), (9, 40), (5, 256), (2, 1000), (7, 896), (33, 3584), (4, 4097), (3, 18944), (2, 20001), (2, 33000),
         (2, 65536), (700, 64), (300, 896), (1000, 3584), (160, 12000)]
EPS = 1e-6


def make(dev, rows, dim, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, r, gy, gh = (torch.randn(rows, dim, device=dev, generator=g).to(dtype) for _ in range(4))
    w = (1 + 0.3 * torch.randn(dim, device=dev, generator=g)).to(dtype)
    return x, r, w, gy, gh


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check(y, h, w, eps=EPS):
    h, w = h.double(), w.double()
    want = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w
    bound = want.abs() * (half(y.dtype) + 5e-6) + (3e-8 if y.dtype == torch.float16 else 0)
    assert ((y.double() - want).abs() <= bound).all()


def check_gradient(got, gy, gh, h, w, dtype, eps=EPS):
    dx, dw = got
    gy, h, w = gy.double(), h.double(), w.double()
    r = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    u, g = h * r, gy * w
    want = r * (g - u * (g * u).mean(-1, keepdim=True))
    size = r * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    if gh is not None:
        want = want + gh.double()
        size = size + gh.double().abs()
    tiny = 3e-8 if dtype == torch.float16 else 0
    assert ((dx.double() - want).abs() <= half(dtype) * want.abs() + 1e-5 * size + tiny).all()
    if dw is not None:
        want, size = (gy * u).sum(0), (gy * u).abs().sum(0)
        assert ((dw.double() - want).abs() <= half(dtype) * want.abs() + 1e-5 * size + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_norm(mrsa, cuda_device, rows, dim, kind):
    x, r, w, _, _ = make(cuda_device, rows, dim, TYPES[kind])
    y, h = mrsa.add_rms_norm(x, r, w, EPS)
    assert torch.equal(h, x + r) and y.is_contiguous() and h.is_contiguous()
    check(y, h, w)
    y, same = mrsa.add_rms_norm(x, None, w, 0.1)
    assert same is x
    check(y, x, w, 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", SIZES + [(1500, 130)])
def test_gradient(mrsa, cuda_device, rows, dim, kind):
    dtype = TYPES[kind]
    x, r, w, gy, gh = (t.requires_grad_() for t in make(cuda_device, rows, dim, dtype, 1))
    gy, gh = gy.detach(), gh.detach()
    y, h = mrsa.add_rms_norm(x, r, w, EPS)
    check(y.detach(), h.detach(), w.detach())
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (gy, gh))
    assert torch.equal(dx, dr) and dx.dtype == dtype and dw.dtype == dtype
    check_gradient((dx, dw), gy, gh, h.detach(), w.detach(), dtype)
    # the same bits on every run; without the stream's own gradient; of one input alone
    y, h = mrsa.add_rms_norm(x, r, w, EPS)
    for a, b in zip(torch.autograd.grad((y, h), (x, r, w), (gy, gh)), (dx, dr, dw)):
        assert torch.equal(a, b)
    y, h = mrsa.add_rms_norm(x, r.detach(), w.detach(), EPS)
    dx, = torch.autograd.grad(y, x, gy)
    check_gradient((dx, None), gy, None, h.detach(), w.detach(), dtype)
    y, _ = mrsa.add_rms_norm(x, None, w, EPS)
    check_gradient(torch.autograd.grad(y, (x, w), gy), gy, None, x.detach(), w.detach(), dtype)


_DWEIGHT = """
import hashlib, sys
import torch
import __graft_entry__
m = __graft_entry__.load_package()
for dim in map(int, sys.argv[1:]):
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r, gy, gh = (torch.randn(1000, dim, device="cuda", generator=g) for _ in range(4))
    w = torch.ones(dim, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(m.add_rms_norm(x, r, w, 1e-6), w, (gy, gh))
print(hashlib.sha256(dw.cpu().view(torch.uint8).numpy().tobytes()).hexdigest())
"""


@pytest.mark.gpu
def test_gradient_does_not_depend_on_calls_before(cuda_device):
    """The same bits of dw in a process that took another width before, of as many threads, whose rows leave room for
    another CTA."""
    out = [subprocess.run([sys.executable, "-c", _DWEIGHT, *dims], cwd=ROOT, capture_output=True, text=True, check=True,
                          timeout=300).stdout.strip() for dims in (("2048",), ("1800", "2048"))]
    assert len(out[0]) == 64 and out[0] == out[1]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rows,dim", [("fp32", 950, 18944), ("bf16", 950, 24000), ("bf16", 900, 9001)])
def test_gradient_of_many_wide_rows(mrsa, cuda_device, kind, rows, dim):
    """Past the registers, more rows than CTAs: parts of dw that take several rows each."""
    dtype = TYPES[kind]
    x, r, w, gy, gh = make(cuda_device, rows, dim, dtype, 10)
    for t in (x, r, w):
        t.requires_grad_()
    y, h = mrsa.add_rms_norm(x, r, w, EPS)
    dx, dw = torch.autograd.grad((y, h), (x, w), (gy, gh))
    check_gradient((dx, dw), gy, gh, h.detach(), w.detach(), dtype)


@pytest.mark.gpu
def test_gradient_against_differences(mrsa, cuda_device):
    x, r, w, gy, gh = make(cuda_device, 5, 48, torch.float32, 2)
    for t in (x, r, w):
        t.requires_grad_()
    grads = torch.autograd.grad(mrsa.add_rms_norm(x, r, w, EPS), (x, r, w), (gy, gh))

    def value(a, b, c):
        with torch.no_grad():
            y, h = mrsa.add_rms_norm(a, b, c, EPS)
        return (y.double() * gy.double()).sum() + (h.double() * gh.double()).sum()

    g = torch.Generator(device=cuda_device).manual_seed(3)
    for i in range(3):
        d = torch.randn(grads[i].shape, device=cuda_device, generator=g)
        step, at = 1e-2, [x.detach(), r.detach(), w.detach()]
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step * d, at[i] - step * d
        got = ((value(*up) - value(*down)) / (2 * step)).item()
        want = (grads[i].double() * d.double()).sum().item()
        # third derivatives times step^2 / 6 stay below 1e-3 of the sum's terms, fp32 noise below 1e-4 of them
        assert abs(got - want) <= 2e-3 * (grads[i].double() * d.double()).abs().sum().item()


@pytest.mark.gpu
def test_strides_broadcasts_and_shapes(mrsa, cuda_device):
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(4)
    wide = torch.randn(2, 5, 300, device=dev, generator=g)
    w = torch.randn(96, device=dev, generator=g)
    for x in (wide[..., :96], wide[..., 3:99], wide[..., 100:196:1].transpose(0, 1), wide[:, ::2, :192:2]):
        r = torch.randn(x.shape, device=dev, generator=g)
        y, h = mrsa.add_rms_norm(x, r, w, EPS)
        assert y.shape == x.shape and torch.equal(h, x + r)
        check(y, h, w)
    y, h = mrsa.add_rms_norm(wide[0, 0], None, torch.ones(300, device=dev), EPS)     # one row without others
    check(y, h, torch.ones(300, device=dev))
    # one row for all tokens, a gradient that is one number everywhere, and one with a row for all
    row = torch.randn(1, 1, 96, device=dev, generator=g).requires_grad_()
    x = wide[..., 4:100].clone().requires_grad_()
    y, h = mrsa.add_rms_norm(x, row.expand(2, 5, 96), w, EPS)
    gy = torch.randn(96, device=dev, generator=g).expand(2, 5, 96)
    dx, drow = torch.autograd.grad((y, h), (x, row), (gy, torch.ones((), device=dev).expand(2, 5, 96)))
    check_gradient((dx.flatten(0, 1), None), gy.reshape(10, 96), torch.ones(10, 96, device=dev), h.detach().flatten(0, 1), w,
                   torch.float32)
    assert ((drow - dx.sum((0, 1), keepdim=True)).abs() <= 1e-5 * dx.abs().sum((0, 1), keepdim=True)).all()
    with torch.no_grad():
        assert not mrsa.add_rms_norm(x, None, w, EPS)[0].requires_grad
    (mrsa.add_rms_norm(x, row.expand(2, 5, 96), w, EPS)[1]).sum().backward()         # the stream alone
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(row.grad, torch.full_like(row, 10.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,pitch,first", [(96, 300, 3), (97, 300, 1), (97, 301, 2), (98, 301, 1), (31, 31, 1), (8, 9, 1), (1000, 1001, 5),
                                             (2503, 2503, 0), (4001, 4002, 1), (6001, 6001, 3), (7999, 8001, 0), (12001, 12001, 1),
                                             (15999, 15999, 0)])
def test_views_of_16_bits(mrsa, cuda_device, dim, pitch, first, kind):
    """Rows that begin in the middle of a word, all, some or none of them, in tensors that agree in it or do not."""
    dev, dtype, rows = cuda_device, TYPES[kind], 13
    g = torch.Generator(device=dev).manual_seed(8)

    def view(p, f):
        flat = torch.randn(f + rows * p + 8, device=dev, generator=g).to(dtype)
        return torch.as_strided(flat, (rows, dim), (p, 1), f)

    w = view(pitch, first)[0]
    for r, gy, gh in ((view(pitch, first), view(pitch, first), view(pitch, first)), (view(dim, 0), view(dim, 0), view(dim, 0)),
                      (view(pitch, first + 1), view(dim, 0), None), (None, view(pitch + 1, 0), None)):
        x = view(pitch, first)
        leaves = [v.requires_grad_() for v in (x, r, w) if v is not None]
        y, h = mrsa.add_rms_norm(x, r, w, EPS)
        with torch.no_grad():
            assert torch.equal(h, x if r is None else x + r)
            check(y, h, w)
        outs, grads = ((y, h), (gy, gh)) if gh is not None else ((y,), (gy,))
        got = torch.autograd.grad(outs, leaves, grads)
        check_gradient((got[0], got[-1]), gy, gh, h.detach(), w.detach(), dtype)
        with torch.no_grad():
            q, scale = mrsa.quantize_int8(x)
            p = x.double()
            n = 127 * p / p.abs().amax(-1, keepdim=True)
            assert ((q.double() - n).abs() <= 0.5 + 4e-5).all()
            q, scale, h8 = mrsa.add_rms_norm_int8(x, r, w, EPS)
            p = h.double() * w.double()
            assert torch.equal(h8, h) and ((q.double() - 127 * p / p.abs().amax(-1, keepdim=True)).abs() <= 0.5 + 4e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 999])
def test_extreme_values(mrsa, cuda_device, dim):
    """Squares past fp32's range, zeros, NaN and infinities: each row by itself."""
    dev = cuda_device
    x = torch.randn(6, dim, device=dev, generator=torch.Generator(device=dev).manual_seed(5))
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    w = torch.randn(dim, device=dev)
    y, _ = mrsa.add_rms_norm(x, None, w, EPS)
    check(y[[0, 2, 5]], x[[0, 2, 5]], w)
    assert ((y[1].double() - x[1].double() * 1e3 * w.double()).abs() <= 1e-6 * (x[1] * 1e3 * w).abs().double()).all()
    assert y[3].isnan().all()
    assert y[4, 7].isnan() and (y[4, :7] == 0).all() and (y[4, 8:] == 0).all()
    b = x.bfloat16()
    check(mrsa.add_rms_norm(b, None, w.bfloat16(), EPS)[0][[0, 2, 5]], b[[0, 2, 5]], w.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,dim", [(5, 64), (5, 999), (300, 1000), (300, 4096), (3, 40000)])
def test_rows_past_the_squares(mrsa, cuda_device, rows, dim, kind):
    """Rows whose squares pass fp32's largest number: small elements beside large ones, and the gradient."""
    dev, dtype = cuda_device, TYPES[kind]
    x, r, w, gy, gh = make(dev, rows, dim, dtype, 9)
    x[:, 1:] *= 2.0 ** -40
    x[:, 0] = 2.0 ** 66
    check(mrsa.add_rms_norm(x, None, w, EPS)[0], x, w)
    x, r = x * 2.0 ** 30, r * 2.0 ** 95
    for t in (x, r, w):
        t.requires_grad_()
    y, h = mrsa.add_rms_norm(x, r, w, EPS)
    check(y.detach(), h.detach(), w.detach())
    # gradients of y near one are 2^-96 as large here: so is the stream's own
    got = torch.autograd.grad((y, h), (x, w), (gy, gh * 2.0 ** -96))
    check_gradient(got, gy, gh * 2.0 ** -96, h.detach(), w.detach(), dtype)


@pytest.mark.gpu
def test_empty_other_stream_and_graph(mrsa, cuda_device):
    dev = cuda_device
    w = torch.ones(64, device=dev)
    none = torch.zeros(2, 0, 64, device=dev, requires_grad=True)
    y, h = mrsa.add_rms_norm(none, none, w.clone().requires_grad_(), EPS)
    assert y.shape == none.shape and h.shape == none.shape
    y.sum().backward()
    assert none.grad.shape == none.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x, r, wt, gy, gh = make(dev, 50, 128, torch.float32, 6)
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y, h = mrsa.add_rms_norm(x * 2, r, wt, EPS)
    side.synchronize()
    check(y, x * 2 + r, wt)
    # a training step's forward and backward, captured and replayed on new inputs
    for t in (x, r, wt):
        t.requires_grad_()
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(mrsa.add_rms_norm(x, r, wt, EPS), (x, r, wt), (gy, gh))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, h = mrsa.add_rms_norm(x, r, wt, EPS)
        dx, _, dw = torch.autograd.grad((y, h), (x, r, wt), (gy, gh))
    with torch.no_grad():
        x.mul_(-3)
    graph.replay()
    torch.cuda.synchronize()
    check(y.detach(), h.detach(), wt.detach())
    assert torch.equal(h.detach(), x.detach() + r.detach())
    check_gradient((dx, dw), gy, gh, h.detach(), wt.detach(), torch.float32)


@pytest.mark.gpu
def test_refusals(mrsa, cuda_device):
    dev = cuda_device
    x, w = torch.zeros(4, 64, device=dev), torch.ones(64, device=dev)
    for bad, match in [
        (lambda: mrsa.add_rms_norm(x.cpu(), None, w, EPS), "CUDA"),
        (lambda: mrsa.add_rms_norm(x.double(), None, w.double(), EPS), "BF16"),
        (lambda: mrsa.add_rms_norm(x, x[:3], w, EPS), "residual"),
        (lambda: mrsa.add_rms_norm(x, x.half(), w, EPS), "residual"),
        (lambda: mrsa.add_rms_norm(x, x.cpu(), w, EPS), "residual"),
        (lambda: mrsa.add_rms_norm(x, None, w[:63], EPS), "weight"),
        (lambda: mrsa.add_rms_norm(x, None, w.bfloat16(), EPS), "weight"),
        (lambda: mrsa.add_rms_norm(x, None, w.cpu(), EPS), "weight"),
        (lambda: mrsa.add_rms_norm(x[:, :0], None, w[:0], EPS), "at least 1"),
        (lambda: mrsa.add_rms_norm(x[0, 0], None, w[:1], EPS), "at least 1"),
        (lambda: mrsa.add_rms_norm(x, None, w, 0.0), "eps"),
        (lambda: mrsa.add_rms_norm(x, None, w, float("nan")), "eps"),
        (lambda: mrsa.add_rms_norm(x, None, None, EPS), "weight"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()
    x.requires_grad_()
    y, _ = mrsa.add_rms_norm(x, None, w, EPS)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        mrsa.add_rms_norm(fwd.make_dual(x.detach(), torch.ones_like(x)), None, w, EPS)


def test_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib

    def rc(x=4096, res=0, w=4096, y=4096, h=0, q=0, scale=0, rows=4, dim=64, eps=EPS, dtype=0):
        return lib.mrsa_add_rms_norm(L.NORM_ARGS.pack(x, res, w, y, h, q, scale, 0, rows, dim, dim, dim, dim, eps, dtype), None)

    assert lib.mrsa_add_rms_norm(None, None) == L.ERR_NULL
    assert rc(x=0) == L.ERR_NULL and rc(w=0) == L.ERR_NULL and rc(res=4096) == L.ERR_NULL
    assert rc(y=0) == L.ERR_ARG and rc(q=4096, scale=4096) == L.ERR_ARG and rc(y=0, q=4096) == L.ERR_NULL
    assert rc(rows=-1) == L.ERR_SHAPE and rc(dim=0) == L.ERR_SHAPE and rc(dim=(1 << 24) + 1) == L.ERR_SHAPE
    assert rc(eps=0.0) == L.ERR_ARG and rc(eps=float("nan")) == L.ERR_ARG and rc(dtype=3) == L.ERR_ARG
    assert rc(x=4097) == L.ERR_ALIGN and rc(dtype=1, w=4098) == L.ERR_ALIGN
    assert rc(rows=0) == 0

    def back(gy=4096, h=4096, w=4096, rstd=4096, dx=4096, dw=4096, rows=4, dim=64, dtype=0, ws=None, size=0):
        return lib.mrsa_add_rms_norm_backward(
            L.NORM_BACKWARD_ARGS.pack(gy, 0, h, w, rstd, dx, dw, rows, dim, dim, dim, dim, dtype), ws, size, None)

    assert lib.mrsa_add_rms_norm_backward(None, None, 0, None) == L.ERR_NULL
    assert back(gy=0) == L.ERR_NULL and back(rstd=0) == L.ERR_NULL and back(dx=0) == L.ERR_NULL
    assert back(rows=0) == L.ERR_SHAPE and back(dtype=7) == L.ERR_ARG and back(h=4097) == L.ERR_ALIGN
    assert back() == L.ERR_WORKSPACE
    assert lib.mrsa_add_rms_norm_backward_workspace(0, 64) == 0
    assert L.NORM_ARGS.size == 112 and L.NORM_BACKWARD_ARGS.size == 104
