"""The RMS norm against 64 bits.

Tolerances, derived before the first run: y and dx in fp32 are a handful of products and one sum
of up to 32768 squares (pairwise over the threads, so about log2(32768) + 32 roundings of 2^-24 in
the reciprocal root): 64 * 2^-24 = 4e-6.  bf16 outputs add their own rounding, at most 2^-8 of the
value.  dw sums up to R rows in fp32: sqrt(R) * 2^-24 of the rows' norm, 1e-5 here; in bf16 2^-8.
"""
import math

import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from delta_ref import norm_ref, rel

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
TOL = {"fp32": 4e-6, "bf16": 2.0 ** -8}
WIDTHS = [1, 7, 64, 128, 333, 2048, 2056, 5000, 8192, 20000, 32768]


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("wdtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 37])
def test_forward(dtype, wdtype, width, rows):
    x, res = rnd(rows, width, seed=1).to(DT[dtype]), (3 * rnd(rows, width, seed=2)).to(DT[dtype])
    w = (1 + 0.2 * rnd(width, seed=3)).to(DT[wdtype])
    y = gsa.rms_norm(x, w)
    assert y.dtype == x.dtype and rel(y, norm_ref(x, w, 1e-6)[0]) <= TOL[dtype]
    y, h = gsa.rms_norm(x, w, eps=1e-3, residual=res)
    ry, rh = norm_ref(x, w, 1e-3, res)
    assert torch.equal(h.double(), rh)
    assert rel(y, ry) <= TOL[dtype]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_rows(dtype):
    """The shape of a long sequence: the one-warp-a-row variant."""
    x, res = rnd(2500, 2048, seed=1).to(DT[dtype]), rnd(2500, 2048, seed=2).to(DT[dtype])
    w = rnd(2048, seed=3).to(DT[dtype])
    y, h = gsa.rms_norm(x, w, residual=res)
    ry, rh = norm_ref(x, w, 1e-6, res)
    assert torch.equal(h.double(), rh)
    err = (y.double() - ry).abs()
    assert (err <= (TOL[dtype] + 4e-6) * ry.abs()).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    x = rnd(4, 6, 512, seed=4).to(DT[dtype])
    w = rnd(512, seed=5).to(DT[dtype])
    want = gsa.rms_norm(x, w)
    wide = torch.zeros(4, 6, 520, dtype=x.dtype, device="cuda")
    wide[..., 1:513] = x  # rows that start off the 16-byte rule
    assert rel(gsa.rms_norm(wide[..., 1:513], w), norm_ref(x, w, 1e-6)[0]) <= TOL[dtype]
    wide[..., 8:520] = x
    assert torch.equal(gsa.rms_norm(wide[..., 8:520], w), want)
    assert torch.equal(gsa.rms_norm(x.transpose(0, 1), w).transpose(0, 1), want)
    assert torch.equal(gsa.rms_norm(x[1, 2], w), want[1, 2])
    assert torch.equal(gsa.rms_norm(x[:, :1].expand(4, 6, 512), w), want[:, :1].expand(4, 6, 512))
    assert gsa.rms_norm(x[:0], w).shape == (0, 6, 512)


def test_rows_of_zeros_infinities_and_nan():
    x = rnd(5, 256, seed=6)
    x[1] = 0
    x[2, 3] = math.inf
    x[3, 7] = math.nan
    w = rnd(256, seed=7)
    y = gsa.rms_norm(x, w)
    assert not y[1].any() and y[3].isnan().all()
    assert y[2, 3].isnan() and not y[2, :3].any()  # inf * 0, and finite values over an infinite norm
    keep = gsa.rms_norm(x[[0, 4]], w)
    assert torch.equal(y[[0, 4]], keep)
    y8, s = gsa.rms_norm_fp8(x, w)
    assert not y8[1].float().any() and s[3].isnan().all() and y8[3].float().isnan().all()


def values(y8, scale):
    return (y8.double().unflatten(-1, (scale.shape[-1], -1)) * scale.double()[..., None]).flatten(-2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width,group", [(1, None), (100, None), (333, None), (2048, None),
                                         (2048, 128), (128, 128), (384, 128), (16384, 128),
                                         (16384, None), (30000, None)])
@pytest.mark.parametrize("rows", [1, 19, 2100])
def test_fp8(dtype, width, group, rows):
    if rows * width > 2 ** 23:
        rows = 30
    x, res = rnd(rows, width, seed=8).to(DT[dtype]), rnd(rows, width, seed=9).to(DT[dtype])
    w = rnd(width, seed=10).to(DT[dtype])
    y8, s, h = gsa.rms_norm_fp8(x, w, residual=res, group_size=group)
    ry, rh = norm_ref(x, w, 1e-6, res)
    assert torch.equal(h.double(), rh) and y8.dtype == torch.float8_e4m3fn
    part = ry.view(rows, -1, group or width)
    rs = part.abs().amax(-1) / 448
    assert s.shape == rs.shape and rel(s, rs) <= 4e-6
    # half a step of e4m3: 2^-4 of the value, or 2^-10 (in units of the scale) below its normals
    err = (values(y8, s) - ry).abs().view_as(part)
    unit = rs[..., None]
    assert (err <= torch.maximum(part.abs() * 2.0 ** -4, unit * 2.0 ** -10) * 1.001).all()
    # the largest magnitude becomes 448; a part whose sum x + residual is zero throughout stays zero
    top = y8.float().view(rows, -1, group or width).abs().amax(-1)
    assert (top == torch.where(rs > 0, 448.0, 0.0)).all()
    y8b, sb = gsa.rms_norm_fp8(h, w, group_size=group)
    assert torch.equal(y8b.view(torch.uint8), y8.view(torch.uint8)) and torch.equal(s, sb)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_fp8_layouts(dtype):
    x = rnd(3, 5, 260, seed=11).to(DT[dtype])
    w = rnd(256, seed=12).to(DT[dtype])
    for at in (1, 2, 4):
        v = x[..., at:at + 256]
        for group in (None, 128):
            a, s = gsa.rms_norm_fp8(v, w, group_size=group)
            ry = norm_ref(v, w, 1e-6)[0]
            part = ry.unflatten(-1, (s.shape[-1], -1))
            err = (values(a, s) - ry).abs().view_as(part)
            bound = torch.maximum(part.abs() * 2.0 ** -4,
                                  part.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10)
            assert (err <= bound * 1.001).all()


def back(fn, leaves, ups):
    leaves = [t.detach().requires_grad_() for t in leaves]
    outs = fn(*leaves)
    return torch.autograd.grad(outs, leaves, ups)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("wdtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 70])
def test_backward(dtype, wdtype, width, rows):
    x, res, dy, dh = (rnd(rows, width, seed=s).to(DT[dtype]) for s in (1, 2, 3, 4))
    w = (1 + 0.2 * rnd(width, seed=5)).to(DT[wdtype])
    got = back(lambda x, w, r: gsa.rms_norm(x, w, residual=r), [x, w, res], [dy, dh])
    # the rounding of h is passed through, as an addition followed by a norm does
    h = (x.double() + res.double()).to(x.dtype)
    ref = back(lambda h, w: [h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w, h],
               [h.double(), w.double()], [dy.double(), dh.double()])
    assert rel(got[0], ref[0]) <= TOL[dtype] and torch.equal(got[0], got[2])
    assert got[1].dtype == w.dtype and rel(got[1], ref[1]) <= (1e-5 if wdtype == "fp32" else 2 ** -8)
    got = back(lambda x, w: gsa.rms_norm(x, w), [x, w], [dy])
    ref = back(lambda h, w: h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w,
               [x.double(), w.double()], [dy.double()])
    if width > 1:  # one value: y = sign(x) w, whose slope is eps / x^2 small, below fp32's step
        assert rel(got[0], ref[0]) <= TOL[dtype] * (4 if width < 16 else 1)
    assert rel(got[1], ref[1]) <= (1e-5 if wdtype == "fp32" else 2 ** -8)


def test_backward_against_differences():
    """fp32: central differences with a step of 2^-6: truncation h^2 / 6, rounding 4e-6 / 2h."""
    x, w, dy = rnd(6, 96, seed=20), rnd(96, seed=21), rnd(6, 96, seed=22)
    got = back(lambda x, w: gsa.rms_norm(x, w), [x, w], [dy])
    f = lambda x, w: (gsa.rms_norm(x, w).double() * dy).sum().item()  # noqa: E731
    h = 2.0 ** -6
    for i, leaf in enumerate((x, w)):
        d = rnd(*leaf.shape, seed=30 + i)
        d = d / d.norm()
        args = lambda s: [t + s * h * d if j == i else t for j, t in enumerate((x, w))]  # noqa
        slope = (f(*args(1)) - f(*args(-1))) / (2 * h)
        want = (got[i].double() * d).sum().item()
        assert abs(slope - want) <= 2e-3 * got[i].double().norm().item()


def test_backward_partial_use_and_repeatability():
    x, r, dy = (rnd(300, 512, seed=s).bfloat16() for s in (1, 2, 3))
    w = rnd(512, seed=4).bfloat16()
    a = back(lambda x, w, r: gsa.rms_norm(x, w, residual=r)[0], [x, w, r], [dy])
    b = back(lambda x, w, r: gsa.rms_norm(x, w, residual=r)[0], [x, w, r], [dy])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    h = gsa.rms_norm(leaves[0], leaves[1], residual=leaves[2])[1]
    gx, gr = torch.autograd.grad(h, [leaves[0], leaves[2]], dy)
    assert torch.equal(gx, dy) and torch.equal(gr, dy)
    y = gsa.rms_norm(leaves[0], w)  # the weight is no leaf
    assert torch.autograd.grad(y, leaves[0], dy)[0].shape == x.shape


def test_graph_and_stream():
    x, r, w = rnd(64, 2048, seed=1).bfloat16(), rnd(64, 2048, seed=2).bfloat16(), rnd(2048).bfloat16()
    want = gsa.rms_norm_fp8(x, w, residual=r)
    bx = torch.zeros_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gsa.rms_norm_fp8(bx, w, residual=r)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = gsa.rms_norm_fp8(bx, w, residual=r)
        bx.copy_(x)
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("wdtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width,rows", [(9, 4001), (15, 3), (17, 4001), (250, 2100), (2047, 700),
                                        (4099, 2050), (8191, 300), (16389, 20), (32761, 9),
                                        (32767, 9)])
def test_rows_off_the_grid(dtype, wdtype, width, rows):
    """Widths that put every row at another place of the 16-byte grid, more of them than blocks."""
    x, res = rnd(rows, width, seed=21).to(DT[dtype]), rnd(rows, width, seed=22).to(DT[dtype])
    w = (1 + 0.2 * rnd(width, seed=23)).to(DT[wdtype])
    dy, dh = rnd(rows, width, seed=24).to(DT[dtype]), rnd(rows, width, seed=25).to(DT[dtype])
    leaves = [t.detach().requires_grad_() for t in (x, w, res)]
    y, h = gsa.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    got = torch.autograd.grad([y, h], leaves, [dy, dh])
    ry, rh = norm_ref(x, w, 1e-6, res)
    assert torch.equal(h.double(), rh)
    err = (y.double() - ry).abs()
    assert (err <= (TOL[dtype] + 4e-6) * ry.abs()).all()
    # the gradients' formulas in 64 bits, from the h that the norm read
    hd, wd, dyd = h.detach().double(), w.double(), dy.double()
    r = (hd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    p = dyd * wd
    dx = r * (p - hd * r * r * (p * hd).mean(-1, keepdim=True)) + dh.double()
    # dx is a sum of terms that may cancel: their rounding in fp32, and the output's own
    size = r * (p.abs() + hd.abs() * r * r * (p * hd).mean(-1, keepdim=True).abs()) + dh.abs()
    assert ((got[0].double() - dx).abs() <= TOL[dtype] * dx.abs() + 4e-6 * size).all()
    assert torch.equal(got[0], got[2])
    assert rel(got[1], (dyd * hd * r).sum(0)) <= (1e-5 if wdtype == "fp32" else 2.0 ** -8)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_tensor_off_the_others_grid(dtype):
    """An odd width whose residual, or gradient, lies in wider rows than the input."""
    x, wide = rnd(40, 1001, seed=26).to(DT[dtype]), rnd(41, 1004, seed=27).to(DT[dtype])
    w = (1 + 0.2 * rnd(1001, seed=28)).to(DT[dtype])
    for res in (wide[:40, 2:1003], wide[1:, :1001], rnd(40 * 1001 + 3, seed=29).to(
            DT[dtype])[3:].view(40, 1001)):
        y, h = gsa.rms_norm(x, w, residual=res)
        ry, rh = norm_ref(x, w, 1e-6, res)
        assert torch.equal(h.double(), rh) and rel(y, ry) <= TOL[dtype]
        y8, s = gsa.rms_norm_fp8(x, w, residual=res)[:2]
        assert rel(s, ry.abs().amax(-1, keepdim=True) / 448) <= 4e-6
        leaf = x.detach().requires_grad_()
        out = gsa.rms_norm(leaf, w)
        a, = torch.autograd.grad(out, leaf, res, retain_graph=True)
        b, = torch.autograd.grad(out, leaf, res.contiguous())
        assert rel(a, b) <= 2 * TOL[dtype]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_residual_that_is_the_input_and_a_broadcast_gradient(dtype):
    x = rnd(6, 200, seed=30).to(DT[dtype]).requires_grad_()
    w = (1 + 0.2 * rnd(200, seed=31)).to(DT[dtype]).requires_grad_()
    y, h = gsa.rms_norm(x, w, residual=x)
    assert torch.equal(h, x + x)
    got = torch.autograd.grad(y.sum(), [x, w])  # a gradient with strides of zero
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    hd = xd + xd
    want = torch.autograd.grad((hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-6) * wd).sum(),
                               [xd, wd])
    # x gets two equal gradients, added up in its type
    assert rel(got[0], want[0]) <= 2 * TOL[dtype]
    assert rel(got[1], want[1]) <= (1e-5 if dtype == "fp32" else 2.0 ** -8)


@pytest.mark.parametrize("width", [32768, 32767])
def test_offsets_past_32_bits(width):
    """More than 2^31 values a tensor: the last rows are those of a call on them alone."""
    rows, tail = 65552, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(rows, width, generator=gen, device="cuda", dtype=torch.bfloat16)
             for _ in range(2))
    w = (1 + 0.2 * rnd(width, seed=5)).bfloat16()
    leaf = x.requires_grad_()
    y = gsa.rms_norm(leaf, w)
    dx, = torch.autograd.grad(y, leaf, dy)
    last = x[-tail:].detach().clone().requires_grad_()
    part = gsa.rms_norm(last, w)
    want, = torch.autograd.grad(part, last, dy[-tail:])
    assert rel(y[-tail:], part) <= TOL["bf16"] and rel(dx[-tail:], want) <= TOL["bf16"]
    with torch.no_grad():
        del dx, dy, y
        y8, s = gsa.rms_norm_fp8(x, w)
        want8, want_s = gsa.rms_norm_fp8(last, w)
        assert rel(s[-tail:], want_s) <= 4e-6
        # values at a rounding boundary may fall to either side: a step of e4m3, 2^-3
        err = (y8[-tail:].float() - want8.float()).abs()
        assert (err <= want8.float().abs() * 2.0 ** -3 + 2.0 ** -9).all()
        del y8, x, leaf
    torch.cuda.empty_cache()


@pytest.mark.parametrize("wdtype", ["fp32", "bf16"])
def test_no_rows(wdtype):
    x = torch.empty(0, 48, device="cuda", requires_grad=True)
    w = rnd(48, seed=33).to(DT[wdtype]).requires_grad_()
    y, h = gsa.rms_norm(x, w, residual=x)
    dx, dw = torch.autograd.grad([y, h], [x, w], [torch.empty_like(y), torch.empty_like(h)])
    assert dx.shape == (0, 48) and not dw.any() and dw.dtype == w.dtype
    y8, s = gsa.rms_norm_fp8(x.detach(), w.detach())
    assert y8.shape == (0, 48) and s.shape == (0, 1)
