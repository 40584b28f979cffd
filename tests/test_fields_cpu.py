"""Label loss, layer norm and 8-bit features on the native CPU backend: values, gradients, layouts, refusals."""
import pytest
import torch

import retinags_b200 as R
from field_reference import (assert_within, label_reference, make_label_case, norm_reference, pack_reference)
from retinags_b200.utils import loss as plain

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c,v,bias", [(1, 1, 1, True), (1, 5, 2, False), (37, 33, 150, True), (130, 64, 129, False)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_label_loss_against_64_bits(n, c, v, bias, dtype, reduction):
    x, w, y, b = make_label_case(n, c, v, dtype, seed=n + v, bias=bias)
    count = max(int(((y >= 0) & (y < v)).sum()), 1)
    up = torch.rand(n, generator=torch.Generator().manual_seed(1)) + 0.5
    rows = up if reduction == "none" else torch.full((n,), 1.0 / count if reduction == "mean" else 1.0)
    ref = label_reference(x, w, y, b, rows, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    out = R.label_loss(x, w, y, bias=b, reduction=reduction)
    assert out.dtype == F32
    if reduction == "none":
        assert_within(out, ref[0], "losses")
        grads = torch.autograd.grad(out, leaves, up)
    else:
        scale = count if reduction == "mean" else 1
        assert abs(out.item() - float(ref[0][0].sum()) / scale) <= float(ref[0][1].sum()) / scale + 1e-6 * abs(out.item())
        grads = torch.autograd.grad(out, leaves)
    for name, got, r in zip(("dX", "dW", "db"), grads, ref[1:]):
        assert_within(got, r, name)


def test_label_loss_agrees_with_its_readable_definition_and_with_differences():
    x, w, y, b = make_label_case(23, 7, 11, F32, seed=5)
    for reduction in ("mean", "sum", "none"):
        torch.testing.assert_close(R.label_loss(x, w, y, bias=b, reduction=reduction),
                                   plain.label_loss(x.double(), w.double(), y, b.double(), reduction).float(), atol=1e-5, rtol=1e-5)
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(R.label_loss(xg, w, y, bias=b), xg)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).double()
    h = 1e-5
    up, down = (plain.label_loss(x.double() + s * h * d, w.double(), y, b.double()) for s in (1, -1))
    assert abs(float((up - down) / (2 * h)) - float((g.double() * d).sum())) < 1e-5


def test_label_loss_rows_without_a_label():
    x, w, y, b = make_label_case(12, 6, 9, F32, seed=1, unlabelled=0.0)
    y[:] = torch.tensor([-1, 9, -100, 2 ** 40, 255, 9] * 2)
    x[3] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    out = R.label_loss(x, w, y, bias=b)
    assert out.item() == 0.0
    assert all((g == 0).all() for g in torch.autograd.grad(out, leaves))
    y[0] = 4  # one row counts; the NaN of an unlabelled row reaches nothing
    out = R.label_loss(x, w, y, bias=b)
    grads = torch.autograd.grad(out, leaves)
    assert torch.isfinite(out) and all(torch.isfinite(g).all() for g in grads)
    assert (grads[0][1:] == 0).all() and (grads[0][0] != 0).any()
    assert (R.label_loss(x, w, y, bias=b, reduction="none")[1:] == 0).all()


def test_label_loss_labels_taken_out_by_the_bias():
    x, w, y, b = make_label_case(40, 8, 10, F32, seed=2, unlabelled=0.0)
    b[3] = float("-inf")
    b[4] = torch.finfo(F32).min
    y[y == 3] = 1
    y[y == 4] = 2
    ref = label_reference(x, w, y, b, torch.full((40,), 1 / 40), F32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    out = R.label_loss(x, w, y, bias=b)
    assert abs(out.item() - float(ref[0][0].mean())) < 1e-5
    same = torch.full_like(b, torch.finfo(F32).min)  # every score at the lowest value: all labels alike
    torch.testing.assert_close(R.label_loss(x, w, y, bias=same), torch.tensor(10.0).log(), atol=1e-6, rtol=0)
    g = torch.autograd.grad(out, leaves)
    assert (g[1][3] == 0).all() and (g[1][4] == 0).all() and g[2][3] == 0
    assert_within(g[0], ref[1], "dX")


def test_label_loss_layouts_and_empty_inputs():
    x, w, y, b = make_label_case(24, 8, 10, F32, seed=3)
    want = R.label_loss(x, w, y, bias=b, reduction="none")
    planes = x.t().contiguous().t()
    wide = torch.zeros(24, 20)
    wide[:, 4:12] = x
    for v in (planes, wide[:, 4:12], x.view(4, 6, 8)):
        got = R.label_loss(v, w, y.view(v.shape[:-1]), bias=b, reduction="none")
        assert got.shape == v.shape[:-1]
        torch.testing.assert_close(got.reshape(-1), want, atol=0, rtol=0)
    torch.testing.assert_close(R.label_loss(x, w, y.int(), bias=b, reduction="none"), want, atol=0, rtol=0)
    e = torch.zeros(0, 8, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    for reduction in ("mean", "sum"):
        out = R.label_loss(e, wl, torch.zeros(0, dtype=torch.long), reduction=reduction)
        assert out.item() == 0.0
        ge, gw = torch.autograd.grad(out, [e, wl])
        assert ge.shape == (0, 8) and (gw == 0).all()
    assert R.label_loss(e, w, torch.zeros(0, dtype=torch.long), reduction="none").shape == (0,)


def test_label_loss_refusals():
    x, w, y, b = make_label_case(6, 8, 10, F32)
    bad = [(TypeError, dict(features=x.half())), (TypeError, dict(features=x.bfloat16())), (TypeError, dict(labels=y.float())),
           (TypeError, dict(bias=b.double())), (TypeError, dict(bias=b.bfloat16())), (ValueError, dict(weight=w[:, :5])),
           (ValueError, dict(weight=w[:0], bias=None)), (ValueError, dict(labels=y[:3])), (ValueError, dict(bias=b[:3])),
           (ValueError, dict(reduction="avg")), (ValueError, dict(features=torch.zeros(6, 1025), weight=torch.zeros(10, 1025))),
           (ValueError, dict(features=torch.zeros(6, 0), weight=torch.zeros(10, 0))),
           (ValueError, dict(features=torch.zeros(()))), (ValueError, dict(weight=w.to("meta"))), (ValueError, dict(labels=y.to("meta")))]
    for err, kw in bad:
        args = dict(features=x, weight=w, labels=y, bias=b)
        args.update(kw)
        with pytest.raises(err):
            R.label_loss(**args)


NORM_SHAPES = [(1, 1), (1, 33), (3, 2), (77, 64), (50, 70), (9, 771)]


@pytest.mark.parametrize("n,c", NORM_SHAPES)
@pytest.mark.parametrize("x_dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("keep", ["input", "int8"])
def test_layer_norm_against_64_bits(n, c, x_dtype, out_dtype, planes, keep):
    g = torch.Generator().manual_seed(n * 1000 + c)
    x = (torch.randn(n, c, generator=g) * torch.rand(n, 1, generator=g) + 0.3).to(x_dtype)
    if planes:
        x = x.t().contiguous().t()
    w, b = 1 + 0.2 * torch.randn(c, generator=g), torch.randn(c, generator=g)
    dy = torch.randn(n, c, generator=g).to(out_dtype)
    kept = pack_reference(x) if keep == "int8" else x
    ref = norm_reference(x, w, b, dy, 1e-5, kept, out_dtype, x_dtype, F32)
    leaves = [x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = R.layer_norm(x, w, b, out_dtype=out_dtype, keep=keep)
    assert y.is_contiguous() and y.dtype == out_dtype
    grads = torch.autograd.grad(y, leaves, dy)
    for name, got, r in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), ref):
        assert_within(got, r, name)


def test_layer_norm_layouts_optional_parameters_and_edges():
    img = torch.randn(6, 5, 7, generator=torch.Generator().manual_seed(0), requires_grad=True)  # (C,H,W)
    w = torch.rand(6, requires_grad=True)
    for keep in ("input", "int8"):
        y = R.layer_norm(img.permute(1, 2, 0), w, keep=keep)
        assert y.shape == (5, 7, 6) and y.is_contiguous()
        gi, gw = torch.autograd.grad(y.square().sum(), [img, w])
        assert gi.shape == img.shape
        with torch.no_grad():
            ref = torch.nn.functional.layer_norm(img.permute(1, 2, 0).double(), (6,), w.double(), None, 1e-5)
        torch.testing.assert_close(y.double(), ref, atol=1e-5, rtol=1e-5)
    rows = torch.randn(4, 10)[:, 2:8]
    torch.testing.assert_close(R.layer_norm(rows), torch.nn.functional.layer_norm(rows, (6,)), atol=1e-5, rtol=1e-5)
    const = torch.full((3, 6), 2.5, requires_grad=True)  # no variance: the output is the bias
    b = torch.arange(6.0)
    y = R.layer_norm(const, None, b, eps=1e-5)
    torch.testing.assert_close(y, b.expand(3, 6), atol=1e-6, rtol=0)
    assert torch.isfinite(torch.autograd.grad(y.square().sum(), const)[0]).all()
    e = torch.zeros(0, 6, requires_grad=True)
    y = R.layer_norm(e, w)
    ge, gw = torch.autograd.grad(y.sum(), [e, w])
    assert y.shape == (0, 6) and ge.shape == (0, 6) and (gw == 0).all()
    bw = torch.rand(6).bfloat16().requires_grad_(True)
    y = R.layer_norm(rows, bw)
    assert torch.autograd.grad(y.sum(), bw)[0].dtype == BF16
    # gradient of an expanded output gradient, and of a shared weight used twice
    y = R.layer_norm(rows, w) + R.layer_norm(rows * 2, w)
    assert torch.isfinite(torch.autograd.grad(y.sum(), w)[0]).all()


def test_layer_norm_does_not_hold_its_input_in_8_bits():
    x = torch.randn(64, 96, requires_grad=True)
    y = R.layer_norm(x * 1.0, keep="int8")
    held = [t for t in y.grad_fn.saved_tensors if t is not None]
    assert sum(t.numel() * t.element_size() for t in held) == 64 * 96 + 64 * 3


def test_layer_norm_makes_no_codes_without_gradients(monkeypatch):
    made = []
    from retinags_b200.ops import layer_norm as module
    alloc = module.alloc_codes
    monkeypatch.setattr(module, "alloc_codes", lambda *a: (made.append(1), alloc(*a))[1])
    x, w = torch.randn(5, 40), torch.rand(40, requires_grad=True)
    with torch.no_grad():
        y = R.layer_norm(x, w, keep="int8")
    assert not made and torch.equal(y, R.layer_norm(x, w, keep="int8").detach()) and made


def test_layer_norm_refusals():
    x, w = torch.randn(4, 6), torch.ones(6)
    bad = [(TypeError, dict(x=x.half())), (TypeError, dict(out_dtype=torch.float16)), (ValueError, dict(keep="fp8")),
           (ValueError, dict(weight=w[:3])), (ValueError, dict(bias=w[:3])), (TypeError, dict(bias=w.bfloat16())),
           (TypeError, dict(weight=w.double())), (ValueError, dict(eps=-1.0)), (ValueError, dict(eps=float("nan"))),
           (ValueError, dict(x=torch.zeros(4, 0), weight=None)), (ValueError, dict(weight=w.to("meta"))), (ValueError, dict(x=torch.zeros(())))]
    for err, kw in bad:
        args = dict(x=x, weight=w)
        args.update(kw)
        with pytest.raises(err):
            R.layer_norm(**args)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 31), (7, 32), (7, 33), (4, 100)])
def test_pack8_is_exactly_its_definition(n, c, dtype):
    g = torch.Generator().manual_seed(c)
    x = (torch.randn(n, c, generator=g) * 10.0 ** torch.randint(-30, 30, (n, 1), generator=g)).to(dtype)
    p = R.pack8(x)
    assert p.codes.dtype == torch.int8 and p.exponents.shape == (n, (c + 31) // 32) and p.codes.min() >= -127
    ref = pack_reference(x)
    assert torch.equal(p.unpack(F32).double(), ref)
    assert torch.equal(p.unpack(), ref.to(dtype))
    q = R.pack8(x.t().contiguous().t())
    assert q.planes == (1 if min(n, c) > 1 else q.planes)
    assert torch.equal(q.unpack(F32).double(), ref)


def test_pack8_edges_and_refusals():
    x = torch.zeros(6, 40)
    x[0, :4] = torch.tensor([127.0, 126.5, 125.5, -0.5])       # ties to even, largest code
    x[1, :2] = torch.tensor([127.01, 1.0])                      # one step more
    x[2, 35] = float("inf")
    x[3, 1] = float("nan")
    x[4] = torch.finfo(F32).max
    x[5] = 1e-45
    p = R.pack8(x)
    assert p.codes[0, :4].tolist() == [127, 126, 126, 0] and p.exponents[0].tolist() == [127, 127]
    assert p.exponents[1, 0] == 128 and p.exponents[2].tolist() == [127, 255] and p.exponents[3].tolist() == [255, 127]
    ref = pack_reference(x)
    torch.testing.assert_close(p.unpack().double(), ref, atol=0, rtol=0, equal_nan=True)
    assert p.nbytes == 6 * 40 + 6 * 2
    e = R.pack8(torch.zeros(0, 5))
    assert e.unpack().shape == (0, 5)
    assert R.pack8(torch.randn(2, 3, 4)).unpack().shape == (2, 3, 4)
    for bad, err in ((x.half(), TypeError), (torch.zeros(()), ValueError), (torch.zeros(3, 0), ValueError)):
        with pytest.raises(err):
            R.pack8(bad)
    with pytest.raises(TypeError):
        p.unpack(torch.float16)


@pytest.mark.parametrize("planes", [False, True])
def test_unpack_of_parts_and_of_codes_that_do_not_fit(planes):
    x = torch.randn(12, 70, generator=torch.Generator().manual_seed(2)) * torch.arange(1, 13)[:, None]
    p = R.pack8(x.t().contiguous().t() if planes else x)
    assert p.planes == int(planes)
    whole = p.unpack()
    for part in (slice(None, None, 2), slice(3, 9), slice(5, 6)):
        assert torch.equal(R.Packed8(p.codes[part], p.exponents[part], p.planes, F32).unpack(), whole[part])
    assert torch.equal(R.Packed8(p.codes[:, 32:], p.exponents[:, 1:], p.planes, F32).unpack(), whole[:, 32:])
    assert torch.equal(R.Packed8(p.codes, p.exponents, 1 - p.planes, F32).unpack(), whole)  # the other order: copied
    for err, codes, exponents in [(ValueError, p.codes, p.exponents[:, :2]), (ValueError, p.codes[:, :64], p.exponents),
                                  (ValueError, p.codes, p.exponents[:6]), (ValueError, p.codes, p.exponents.to("meta")),
                                  (TypeError, p.codes.int(), p.exponents), (TypeError, p.codes, p.exponents.char()),
                                  (ValueError, p.codes[:, :0], p.exponents[:, :0]), (ValueError, p.codes[0, 0], p.exponents[0, 0])]:
        with pytest.raises(err):
            R.Packed8(codes, exponents, p.planes, F32).unpack()


def test_tensors_without_memory_are_refused():
    x, w = torch.zeros(3, 8, device="meta"), torch.zeros(5, 8, device="meta")
    codes, exponents = torch.zeros(3, 8, dtype=torch.int8, device="meta"), torch.zeros(3, 1, dtype=torch.uint8, device="meta")
    for fn in (lambda: R.layer_norm(x), lambda: R.pack8(x), lambda: R.label_loss(x, w, torch.zeros(3, dtype=torch.long, device="meta")),
               lambda: R.Packed8(codes, exponents, 0, F32).unpack()):
        with pytest.raises(ValueError, match="meta"):
            fn()


def test_label_field_on_rendered_features():
    """Features of splats rendered by the rasteriser, normed in 8 bits, scored against labels: gradients reach the splats."""
    from helpers import activated, small_scene
    from retinags_b200.ops.rasterize import GaussianRasterizationSettings, GaussianRasterizer
    g, cams = small_scene(n=200, width=32, height=24)
    a, cam = activated(g), cams[0]
    mats = [torch.as_tensor(m) for m in (cam.world_view_transform, cam.full_proj_transform, cam.view_world_transform, cam.camera_center)]
    st = GaussianRasterizationSettings(cam.height, cam.width, cam.tan_fovx, cam.tan_fovy, torch.zeros(3), 1.0, *mats[:3],
                                       torch.full((3,), -1e9), torch.full((3,), 1e9), 0, mats[3])
    gen = torch.Generator().manual_seed(3)
    feats = (torch.rand(200, 2, 1, 3, generator=gen) * 2).requires_grad_(True)  # six channels, three to a render
    labels = torch.randint(-1, 5, (24, 32), generator=gen)
    nw, w = torch.ones(6, requires_grad=True), (torch.randn(5, 6, generator=gen)).requires_grad_(True)
    raster, rest = GaussianRasterizer(st), torch.zeros(200, 15, 3)

    def loss_of(f, norm, label):
        planes = torch.cat([raster(a["xyz"], torch.zeros_like(a["xyz"]), a["opacity"], shs=torch.cat([f[:, k], rest], 1), scales=a["scale"],
                                   rotations=a["rot"])[0] for k in range(2)])
        return label(norm(planes.permute(1, 2, 0)), w, labels)

    grads = []
    for norm, label in ((lambda p: R.layer_norm(p, nw, keep="input"), R.label_loss), (lambda p: R.layer_norm(p, nw, keep="int8"), R.label_loss),
                        (lambda p: torch.nn.functional.layer_norm(p, (6,), nw), plain.label_loss)):
        loss = loss_of(feats, norm, label)
        grads.append([loss.detach(), *torch.autograd.grad(loss, [feats, nw, w])])
    for own, ref in zip(grads[0], grads[2]):
        assert (own - ref).abs().max() <= 1e-4 * ref.abs().max()
    assert grads[0][1].abs().max() > 0
    # pixels without splats (all channels equal) have 1/sqrt(eps) for a scale: compare where 8 bits are meant to be used
    assert torch.equal(grads[0][0], grads[1][0]) and torch.isfinite(grads[1][1]).all()
