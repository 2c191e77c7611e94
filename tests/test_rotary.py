"""Rotary positions of any layout (``rotary.py``) against the formula in 64
bits.  Bounds: the angle is the fp32 product on both sides; cos and sin are off
by at most two fp32 ulps and each output is two products and a sum in fp32 (a
few 2^-24 of the pair's norm times the factor: 1e-6 of it), then rounded once
to the tensors' type (half an ulp of the result)."""

import ctypes as C
import math

import pytest
import torch

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def turned(x, pos, inv, factor, layout, sign=1.0):
    """The definition in 64 bits, and the norm of each element's pair."""
    n = inv.shape[0]
    ang = sign * (pos.float()[..., None] * inv).double()[:, :, None, :]
    cos, sin = ang.cos() * factor, ang.sin() * factor
    y, norm = x.double().clone(), x.double().abs()
    ia = torch.arange(n, device=x.device) * (2 if layout == "interleaved" else 1)
    ib = ia + (1 if layout == "interleaved" else n)
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    norm[..., ia] = norm[..., ib] = (a * a + b * b).sqrt() * factor
    return y, norm


def check(got, x, pos, inv, factor, layout, sign=1.0):
    want, norm = turned(x, pos, inv, factor, layout, sign)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0     # half the spacing of fp16's subnormals
    err = (got.double() - want).abs()
    assert (err <= HALF_ULP[x.dtype] * want.abs() + 1e-6 * norm + tiny).all(), (err / norm.clamp_min(1e-30)).max().item()


def positions(b, l, device, first=0):
    return (first + torch.arange(l, device=device) * 3 + torch.arange(b, device=device)[:, None] * 7).contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,l,hq,hk,d,n,strided", [
    (1, 1, 28, 4, 128, 64, True),      # one token, a fused projection's rows
    (2, 33, 7, 1, 128, 32, False),     # half of the head
    (1, 257, 3, 3, 64, 8, True),       # a quarter of it
    (3, 5, 5, 2, 256, 128, False),
    (1, 9, 2, 1, 80, 10, True),        # ten pairs: no 16-byte edges in the half layout
    (1, 4, 1, 1, 6, 3, False),
    (1, 2, 300, 2, 128, 64, False),    # more items to a token than a CTA has in flight
])
def test_rotary_matches_the_formula(mrsa, cuda_device, dtype, layout, b, l, hq, hk, d, n, strided):
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(l + d)
    x = torch.randn(b, l, hq + hk, d, device=dev, generator=g).to(dtype)
    q, k = x.split([hq, hk], 2)
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    pos = positions(b, l, dev)
    inv, _ = mrsa.rotary_inv_freq(2 * n, device=dev)
    yq, yk = mrsa.rotary_embedding(q, k, pos, inv, 1.25, layout=layout)
    check(yq, q, pos, inv, 1.25, layout)
    check(yk, k, pos, inv, 1.25, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("first", [105000, 131072, 16777000, -5])
def test_rotary_at_far_positions(mrsa, cuda_device, first):
    dev = cuda_device
    q = torch.randn(1, 200, 4, 128, device=dev)
    pos = positions(1, 200, dev, first)
    inv, f = mrsa.rotary_inv_freq(128, scaling="yarn", factor=8.0, device=dev)
    check(mrsa.rotary_embedding(q, None, pos, inv, f)[0], q, pos, inv, f, "half")


@pytest.mark.gpu
def test_rotary_takes_odd_alignment_and_foreign_order(mrsa, cuda_device):
    dev = cuda_device
    pos = positions(2, 11, dev)
    inv, _ = mrsa.rotary_inv_freq(64, device=dev)
    flat = torch.randn(2 * 11 * 4 * 64 + 1, device=dev).bfloat16()
    q = flat[1:].view(2, 11, 4, 64)                                  # starts two bytes past 16
    k = torch.randn(4, 64, 2, 11, device=dev).bfloat16().permute(2, 3, 0, 1)   # last dim strided
    h = torch.randn(2, 4, 11, 64, device=dev).bfloat16().transpose(1, 2)       # heads outside
    for layout in ("half", "interleaved"):
        yq, yk = mrsa.rotary_embedding(q, k, pos, inv, layout=layout)
        check(yq, q, pos, inv, 1.0, layout)
        check(yk, k, pos, inv, 1.0, layout)
        check(mrsa.rotary_embedding(h, None, pos, inv, layout=layout)[0], h, pos, inv, 1.0, layout)


@pytest.mark.gpu
def test_rotary_keeps_infinities_and_passes_the_rest(mrsa, cuda_device):
    dev = cuda_device
    q = torch.ones(1, 2, 1, 64, device=dev)
    q[0, 0, 0, 40] = math.inf
    q[0, 1, 0, 50] = math.nan
    inv, _ = mrsa.rotary_inv_freq(32, device=dev)
    y, none = mrsa.rotary_embedding(q, None, positions(1, 2, dev), inv)
    assert none is None
    assert torch.equal(y[..., 32:].nan_to_num(7.0, 8.0), q[..., 32:].nan_to_num(7.0, 8.0))
    assert torch.isfinite(y[..., :32]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(mrsa, cuda_device, layout):
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(3)
    pos = positions(2, 13, dev)
    inv, f = mrsa.rotary_inv_freq(32, scaling="linear", factor=4.0, device=dev)[0], 1.5
    q = torch.randn(2, 13, 6, 48, device=dev, generator=g)
    shared = torch.randn(2, 13, 1, 48, device=dev, generator=g).requires_grad_()
    q.requires_grad_()
    yq, yk = mrsa.rotary_embedding(q, shared.expand(2, 13, 3, 48), pos, inv, f, layout=layout)   # a broadcast k
    gq = torch.randn(2, 6, 13, 48, device=dev, generator=g).transpose(1, 2)                     # a strided gradient
    gk = torch.randn(2, 13, 3, 48, device=dev, generator=g)
    dq, dk = torch.autograd.grad((yq, yk), (q, shared), (gq, gk))
    # the formula's: the transpose of a rotation times f is the rotation back times f
    check(dq, gq, pos, inv, f, layout, -1.0)
    want = turned(gk, pos, inv, f, layout, -1.0)[0].sum(2, keepdim=True)
    assert (dk.double() - want).abs().max() <= 3 * 1e-6 * 10
    # and differences: the map is linear, so a difference is exact up to rounding
    with torch.no_grad():
        e = torch.randn(2, 13, 6, 48, device=dev, generator=g)
        step = mrsa.rotary_embedding(q + e, None, pos, inv, f, layout=layout)[0].double() - yq.double()
        assert math.isclose((step * gq.double()).sum().item(), (dq.double() * e.double()).sum().item(),
                            rel_tol=1e-5, abs_tol=1e-2)


@pytest.mark.gpu
def test_rotary_empty_and_other_stream(mrsa, cuda_device):
    dev = cuda_device
    inv, _ = mrsa.rotary_inv_freq(64, device=dev)
    none = torch.zeros(2, 0, 4, 64, device=dev)
    assert mrsa.rotary_embedding(none, none, torch.zeros(2, 0, dtype=torch.long, device=dev), inv)[0].shape == none.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, pos = torch.randn(1, 50, 4, 64, device=dev), positions(1, 50, dev)
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = mrsa.rotary_embedding(q * 2, None, pos, inv)[0]
    side.synchronize()
    check(y, q * 2, pos, inv, 1.0, "half")


@pytest.mark.gpu
def test_rotary_refusals(mrsa, cuda_device):
    dev = cuda_device
    q = torch.zeros(1, 4, 2, 64, device=dev)
    pos = positions(1, 4, dev)
    inv = torch.ones(32, device=dev)
    for bad, match in [
        (lambda: mrsa.rotary_embedding(q[0], None, pos, inv), "B, L, H, D"),
        (lambda: mrsa.rotary_embedding(q.double(), None, pos, inv), "BF16"),
        (lambda: mrsa.rotary_embedding(q, q.bfloat16(), pos, inv), "share"),
        (lambda: mrsa.rotary_embedding(q, q[:, :3], pos, inv), "share"),
        (lambda: mrsa.rotary_embedding(q, None, pos.int(), inv), "int64"),
        (lambda: mrsa.rotary_embedding(q, None, pos[:, :2], inv), "int64"),
        (lambda: mrsa.rotary_embedding(q, None, pos.cpu(), inv), "device"),
        (lambda: mrsa.rotary_embedding(q, None, pos, torch.ones(33, device=dev)), "inv_freq"),
        (lambda: mrsa.rotary_embedding(q, None, pos, inv[:0]), "inv_freq"),
        (lambda: mrsa.rotary_embedding(q, None, pos, inv, layout="other"), "layout"),
        (lambda: mrsa.rotary_embedding(q[..., :63], None, pos, inv[:20], layout="interleaved"), "even"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_inverse_frequencies(mrsa):
    inv, f = mrsa.rotary_inv_freq(64, 1e4)
    want = torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert f == 1.0 and inv.dtype == torch.float32 and torch.equal(inv, want.float())
    lin, _ = mrsa.rotary_inv_freq(64, 1e4, scaling="linear", factor=4.0)
    assert torch.equal(lin, (want / 4).float())
    ntk, _ = mrsa.rotary_inv_freq(64, 1e4, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1].item(), want[-1].item() / 4, rel_tol=1e-6)
    yarn, af = mrsa.rotary_inv_freq(128, 1e6, scaling="yarn", factor=8.0)
    ref, raf = mrsa.yarn_inv_freq()
    assert torch.equal(yarn, ref) and af == raf
    for bad in (dict(dim=0), dict(dim=7), dict(dim=64, scaling="other"), dict(dim=64, factor=0.0), dict(dim=2, scaling="ntk")):
        with pytest.raises(ValueError):
            mrsa.rotary_inv_freq(**bad)


def test_rotary_argument_codes(mrsa):
    lib, L = mrsa._lib.load(), mrsa._lib

    def rc(q=4096, out=4096, pos=4096, inv=4096, b=1, l=4, hq=2, d=64, pairs=32, dtype=0, inter=0):
        return lib.mrsa_rotary(L.ROTARY_ARGS.pack(q, out, 0, 0, pos, inv, 0, 0, 0, 0, 0, 0, b, l, hq, 0, d, pairs, 1.0,
                                                  dtype, inter, 0), None)

    assert lib.mrsa_rotary(None, None) == L.ERR_NULL
    assert rc(q=0) == L.ERR_NULL and rc(inv=0) == L.ERR_NULL and rc(pos=0) == L.ERR_NULL
    assert rc(pairs=0) == L.ERR_SHAPE and rc(pairs=33) == L.ERR_SHAPE and rc(b=-1) == L.ERR_SHAPE
    assert rc(d=1025) == L.ERR_SHAPE and rc(inter=2) == L.ERR_ARG
    assert rc(l=0) == 0
    q = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        mrsa.rotary_embedding(q, None, torch.zeros(1, 4, dtype=torch.long), torch.ones(32))
    assert C.sizeof(C.c_void_p) == 8 and L.ROTARY_ARGS.size == 160


@pytest.mark.gpu
def test_rotary_gradient_of_one_tensor(mrsa, cuda_device):
    dev = cuda_device
    pos = positions(1, 7, dev)
    inv, _ = mrsa.rotary_inv_freq(64, device=dev)
    q = torch.randn(1, 7, 3, 64, device=dev, requires_grad=True)
    k = torch.randn(1, 7, 1, 64, device=dev)
    g = torch.randn(1, 7, 3, 64, device=dev)
    y, none = mrsa.rotary_embedding(q, None, pos, inv)
    assert none is None
    check(torch.autograd.grad(y, q, g)[0], g, pos, inv, 1.0, "half", -1.0)
    y, yk = mrsa.rotary_embedding(q.detach(), k.requires_grad_(), pos, inv)
    gk = torch.randn_like(yk)
    check(torch.autograd.grad(yk, k, gk)[0], gk, pos, inv, 1.0, "half", -1.0)
    with torch.no_grad():
        assert not mrsa.rotary_embedding(q, None, pos, inv)[0].requires_grad
    y, _ = mrsa.rotary_embedding(q, None, pos, inv)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(y, q, g, create_graph=True)
