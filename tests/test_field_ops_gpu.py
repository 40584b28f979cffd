"""Label loss, layer norm and 8-bit features on the GPU: values and gradients at odd sizes, layouts, streams, graphs."""
import pytest
import torch

import retinags_b200 as R
from field_reference import (assert_within, label_reference, make_label_case, norm_reference, pack_reference)

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _check_label(x, w, y, b, reduction="mean", seed=1):
    n, dtype = y.numel(), x.dtype
    count = max(int(((y >= 0) & (y < w.shape[0])).sum()), 1)
    up = (torch.rand(n, generator=torch.Generator().manual_seed(seed)) + 0.5).to(x.device)
    rows = up if reduction == "none" else torch.full((n,), 1.0 / count if reduction == "mean" else 1.0, device=x.device)
    ref = label_reference(x.detach(), w.detach(), y, None if b is None else b.detach(), rows, dtype, None if b is None else b.dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    out = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2] if b is not None else None, reduction=reduction)
    if reduction == "none":
        assert_within(out.detach(), ref[0], "losses")
        grads = torch.autograd.grad(out, leaves, up)
    else:
        scale = count if reduction == "mean" else 1
        want = float(ref[0][0].sum()) / scale
        assert abs(out.item() - want) <= float(ref[0][1].sum()) / scale + 2.0 ** -23 * abs(want)
        grads = torch.autograd.grad(out, leaves)
    for name, got, r in zip(("dX", "dW", "db"), grads, ref[1:]):
        assert_within(got, r, name)


LABEL_SIZES = [(1, 1, 1), (1, 64, 4096), (2, 3, 2), (127, 8, 127), (128, 16, 128), (129, 33, 129), (300, 64, 255), (257, 65, 257),
               (1000, 96, 1003), (513, 128, 640), (260, 129, 384), (700, 200, 300), (384, 256, 5003), (130, 257, 131), (256, 512, 700),
               (150, 771, 200), (129, 1024, 257), (20000, 32, 40), (5, 32, 33000)]


@pytest.mark.parametrize("n,c,v", LABEL_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_label_loss_sizes(n, c, v, dtype, bias):
    _check_label(*make_label_case(n, c, v, dtype, seed=n + c + v, bias=bias, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_label_loss_reductions(reduction, dtype):
    _check_label(*make_label_case(333, 48, 217, dtype, seed=9, device="cuda"), reduction=reduction)


def test_label_loss_bias_in_32_bits_beside_bf16():
    _check_label(*make_label_case(333, 48, 217, BF16, seed=9, device="cuda", bias_dtype=F32))


@pytest.mark.parametrize("scale", [1e-3, 30.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_flat_and_peaked_scores(scale, dtype):
    x, w, y, b = make_label_case(257, 64, 500, F32, seed=4, device="cuda")
    _check_label((x * scale).to(dtype), w.to(dtype), y, b.to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_rows_without_a_label(dtype):
    x, w, y, b = make_label_case(700, 40, 90, dtype, seed=1, device="cuda", unlabelled=0.0)
    y[::2] = torch.tensor([-1, 90, -100, 2 ** 40, 255], device="cuda").repeat(70)
    clean = x.clone()
    x[0], x[2, 5], x[698, 39] = float("nan"), float("inf"), float("-inf")
    got = []
    for f in (x, clean):
        leaves = [t.detach().requires_grad_(True) for t in (f, w, b)]
        out = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2])
        got.append([out.detach(), *torch.autograd.grad(out, leaves)])
    for a, c in zip(*got):  # what unlabelled rows hold reaches nothing
        assert torch.equal(a, c)
    assert (got[0][1][::2] == 0).all()
    _check_label(clean, w, y, b)
    y[:] = -1
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2])
    assert out.item() == 0.0 and all((g == 0).all() for g in torch.autograd.grad(out, leaves))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_a_row_that_is_not_finite_stays_so(dtype):
    x, w, y, b = make_label_case(140, 16, 50, dtype, seed=1, device="cuda", unlabelled=0.0)
    x[7, 3] = float("nan")
    leaf = x.clone().requires_grad_(True)
    losses = R.label_loss(leaf, w, y, bias=b, reduction="none")
    bad = torch.zeros(140, dtype=torch.bool, device="cuda")
    bad[7] = True
    assert torch.equal(torch.isnan(losses), bad)
    (g,) = torch.autograd.grad(losses.sum(), leaf)
    assert torch.isnan(g[7]).all() and torch.isfinite(g[~bad]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_labels_taken_out_by_the_bias(dtype):
    x, w, y, b = make_label_case(300, 24, 140, dtype, seed=2, device="cuda", unlabelled=0.0)
    b[3], b[130:] = float("-inf"), float("-inf")
    b[4] = torch.finfo(dtype).min
    y[(y == 3) | (y == 4) | (y >= 130)] = 1
    _check_label(x, w, y, b)
    b[:] = torch.finfo(dtype).min  # every score at the lowest value: all labels alike
    leaf = b.detach().requires_grad_(True)
    out = R.label_loss(x, w, y, bias=leaf, reduction="none")
    torch.testing.assert_close(out, torch.full_like(out, 140.0).log(), atol=1e-5, rtol=0)
    (g,) = torch.autograd.grad(out.sum(), leaf)
    hits = torch.bincount(y, minlength=140).float()
    torch.testing.assert_close(g.float(), 300 / 140 - hits, atol=1e-3, rtol=2.0 ** -7)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_layouts(dtype):
    x, w, y, b = make_label_case(240, 24, 100, dtype, seed=3, device="cuda")
    want = R.label_loss(x, w, y, bias=b, reduction="none")
    wide = torch.full((241, 61), float("nan"), dtype=dtype, device="cuda")
    wide[:240, 13:37] = x
    ww = torch.full((101, 41), float("nan"), dtype=dtype, device="cuda")
    ww[1:, 7:31] = w
    for f, wt in ((x.t().contiguous().t(), w), (wide[:240, 13:37], w), (x, ww[1:, 7:31]), (wide[:240, 13:37].view(240, 24), w.t().contiguous().t())):
        torch.testing.assert_close(R.label_loss(f, wt, y, bias=b, reduction="none"), want, atol=0, rtol=0)
    torch.testing.assert_close(R.label_loss(x.view(4, 60, 24), w, y.view(4, 60).int(), bias=b, reduction="none").view(-1), want, atol=0, rtol=0)
    # one pixel's features for all: the gradient of the broadcast input is the sum
    one = x[:1].detach().clone().requires_grad_(True)
    (g,) = torch.autograd.grad(R.label_loss(one.expand(240, 24), w, y, bias=b, reduction="sum"), one)
    full = x[:1].detach().expand(240, 24).contiguous().requires_grad_(True)
    (gf,) = torch.autograd.grad(R.label_loss(full, w, y, bias=b, reduction="sum"), full)
    torch.testing.assert_close(g, gf.sum(0, keepdim=True), atol=0, rtol=0)


@pytest.mark.parametrize("n,c,v,dtype", [(3000, 64, 700, BF16), (3000, 48, 700, F32), (40, 256, 20000, BF16)])
def test_label_loss_gives_the_same_bits_every_time(n, c, v, dtype):
    x, w, y, b = make_label_case(n, c, v, dtype, seed=6, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    runs = []
    for _ in range(3):
        out = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2])
        runs.append([out.detach(), *torch.autograd.grad(out, leaves)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_partial_gradients(dtype):
    x, w, y, b = make_label_case(200, 24, 100, dtype, seed=3, device="cuda")
    full = [t.detach().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(R.label_loss(full[0], full[1], y, bias=full[2]), full)
    for k in range(3):
        t = [x, w, b]
        t[k] = t[k].detach().requires_grad_(True)
        (g,) = torch.autograd.grad(R.label_loss(t[0], t[1], y, bias=t[2]), t[k])
        assert torch.equal(g, want[k])


def test_chain_in_a_graph_and_on_a_side_stream():
    """Norm (kept in 8 bits) and loss, forward and backward, captured once and replayed on new inputs; two graphs of the same
    sizes replayed in turn; a run on a stream of its own."""
    n, c, v = 1000, 64, 300
    x, w, y, b = make_label_case(n, c, v, F32, seed=8, device="cuda")
    nw, nb = torch.ones(c, device="cuda", requires_grad=True), torch.zeros(c, device="cuda", requires_grad=True)
    w, b = w.bfloat16().requires_grad_(True), b.requires_grad_(True)

    def step(f):
        h = R.layer_norm(f, nw, nb, out_dtype=BF16, keep="int8")
        loss = R.label_loss(h, w, y, bias=b)
        return [loss.detach(), *torch.autograd.grad(loss, [f, nw, nb, w, b])]

    inputs = [x.clone() * s for s in (1.0, 0.5, 2.0)]
    want = [[t.clone() for t in step(f.clone().requires_grad_(True))] for f in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(inputs[1].clone().requires_grad_(True))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    bufs = [x.clone().requires_grad_(True) for _ in range(2)]
    graphs, outs = [], []
    for f in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(f))
        graphs.append(gr)
    for i in (0, 1, 2, 1):
        for k in range(2):
            with torch.no_grad():
                bufs[k].copy_(inputs[(i + k) % 3])
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[(i + k) % 3]))


NORM_SIZES = [(1, 1), (1, 33), (3, 2), (77, 64), (1000, 32), (501, 48), (130, 70), (129, 771), (65, 1024), (33, 1025), (9, 5000), (2049, 8)]


def _check_norm(x, out_dtype, keep, p_dtype=F32, seed=0, affine=True):
    n, c = x.shape
    g = torch.Generator().manual_seed(seed)
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).to(p_dtype).cuda(), torch.randn(c, generator=g).to(p_dtype).cuda()
    dy = torch.randn(n, c, generator=g).to(out_dtype).cuda()
    kept = pack_reference(x.detach().cpu()).cuda() if keep == "int8" else x
    ref = norm_reference(x.detach(), w if affine else torch.ones_like(w), b if affine else torch.zeros_like(b), dy, 1e-5, kept, out_dtype, x.dtype, p_dtype)
    leaves = [x.detach().requires_grad_(True)] + ([w.requires_grad_(True), b.requires_grad_(True)] if affine else [])
    y = R.layer_norm(leaves[0], *(leaves[1:] if affine else ()), out_dtype=out_dtype, keep=keep)
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.is_contiguous() and grads[0].stride() == leaves[0].stride() or not (leaves[0].is_contiguous() or leaves[0].t().is_contiguous())
    for name, got, r in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), ref):
        assert_within(got, r, name)


@pytest.mark.parametrize("n,c", NORM_SIZES)
@pytest.mark.parametrize("x_dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("keep", ["input", "int8"])
def test_layer_norm_sizes(n, c, x_dtype, out_dtype, planes, keep):
    g = torch.Generator().manual_seed(n * 1000 + c)
    x = (torch.randn(n, c, generator=g) * torch.rand(n, 1, generator=g) + 0.3).to(x_dtype).cuda()
    _check_norm(x.t().contiguous().t() if planes else x, out_dtype, keep)


def test_layer_norm_strided_rows_bf16_parameters_and_none():
    base = torch.randn(300, 91, generator=torch.Generator().manual_seed(1)).cuda()
    for view in (base[:, 5:69], base[:, 8:72], base[::3, :64], base.t()[3:67, 5:290].t()):
        for keep in ("input", "int8"):
            _check_norm(view, F32, keep, affine=False)
            _check_norm(view, BF16, keep, p_dtype=BF16)


def test_layer_norm_rows_with_infinities_stay_alone():
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(1)).cuda()
    x[3, 5], x[77, 1] = float("inf"), float("nan")
    good = torch.ones(200, dtype=torch.bool)
    good[[3, 77]] = False
    for planes in (False, True):
        for keep in ("input", "int8"):
            f = (x.t().contiguous().t() if planes else x.clone()).requires_grad_(True)
            y = R.layer_norm(f, keep=keep)
            (g,) = torch.autograd.grad(y, f, torch.ones_like(y))
            for t in (y, g):
                assert torch.isfinite(t[good]).all() and not torch.isfinite(t[~good]).any()


def test_layer_norm_gives_the_same_bits_every_time():
    x = torch.randn(50000, 48, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    w = torch.rand(48, device="cuda", requires_grad=True)
    dy = torch.randn(50000, 48, generator=torch.Generator().manual_seed(2)).cuda()
    runs = [torch.autograd.grad(R.layer_norm(x, w, keep=k), [x, w], dy) for k in ("input", "input", "int8", "int8")]
    for a, b in ((0, 1), (2, 3)):
        assert all(torch.equal(p, q) for p, q in zip(runs[a], runs[b]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 31), (70, 32), (70, 33), (33, 100), (3, 2000)])
def test_pack8_is_exactly_its_definition(n, c, dtype):
    g = torch.Generator().manual_seed(c)
    x = (torch.randn(n, c, generator=g) * 10.0 ** torch.randint(-30, 30, (n, 1), generator=g)).to(dtype)
    x[0, :4] = torch.tensor([127.0, 126.5, 125.5, -0.5]).to(dtype)[:min(c, 4)]
    if n > 4:
        x[1], x[2], x[3, c - 1], x[4, 0] = 0.0, torch.finfo(dtype).max, float("inf"), float("nan")
    ref = pack_reference(x)
    wide = torch.zeros(n, c + 3, dtype=dtype)
    wide[:, 1:c + 1] = x
    for t in (x.cuda(), x.cuda().t().contiguous().t(), wide.cuda()[:, 1:c + 1]):
        p = R.pack8(t)
        torch.testing.assert_close(p.unpack(F32).cpu().double(), ref, atol=0, rtol=0, equal_nan=True)
        torch.testing.assert_close(p.unpack(BF16).cpu().double(), ref.to(BF16).double(), atol=0, rtol=0, equal_nan=True)
        host = R.pack8(x)
        assert torch.equal(p.exponents.cpu(), host.exponents) and torch.equal(p.codes.cpu(), host.codes)


def test_offsets_that_pass_32_bits():
    """2^31 + elements of rows: the last ones are right (8-bit form and norm; labels of the last pixels for the loss)."""
    n, c = 2 ** 25 + 77, 64
    x = torch.zeros(n, c, dtype=BF16, device="cuda")
    tail = torch.randn(100, c, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    x[-100:] = tail
    p = R.pack8(x)
    assert torch.equal(p.unpack()[-100:], R.pack8(tail).unpack())
    del p
    with torch.no_grad():
        y = R.layer_norm(x)
        assert torch.equal(y[-100:], R.layer_norm(tail)) and (y[:-100] == 0).all()
    del y
    w = torch.randn(5, c, generator=torch.Generator().manual_seed(1)).to(BF16).cuda().requires_grad_(True)
    labels = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    labels[-100:] = torch.arange(100, device="cuda") % 5
    x.requires_grad_(True)
    loss = R.label_loss(x, w, labels)
    gx, gw = torch.autograd.grad(loss, [x, w])
    tl = tail.clone().requires_grad_(True)
    want = R.label_loss(tl, w, labels[-100:])
    wx, ww = torch.autograd.grad(want, [tl, w])
    assert abs(loss.item() - want.item()) < 1e-5
    torch.testing.assert_close(gx[-100:], wx, atol=1e-6, rtol=2.0 ** -7)
    torch.testing.assert_close(gw, ww, atol=1e-4, rtol=2.0 ** -6)
    assert (gx[:-100] == 0).all()


@pytest.mark.parametrize("op", ["label", "norm"])
def test_a_second_derivative_is_refused(op):
    x = torch.randn(40, 16, device="cuda", requires_grad=True)
    w = torch.randn(5, 16, device="cuda", requires_grad=True)
    out = R.label_loss(x, w, torch.arange(40, device="cuda") % 5) if op == "label" else R.layer_norm(x, w[0]).square().sum()
    (g,) = torch.autograd.grad(out, x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_label_loss_scores_far_from_zero(dtype, reduction):
    """Scores of some thousands (m and log z are then not added up) and, beside them, pixels of ordinary ones."""
    x, w, y, b = make_label_case(300, 40, 200, F32, seed=12, device="cuda")
    x[:100] *= 1500.0
    _check_label(x.to(dtype), w.to(dtype), y, b.to(dtype), reduction=reduction)


def test_label_loss_many_short_items_and_one_label_tile():
    """One tile of labels: every item of dX is one score tile, so that outputs wait for scores of later items."""
    for n, c, v, dtype in ((40000, 20, 7, BF16), (40000, 70, 100, BF16), (30000, 40, 128, F32), (300, 64, 60000, BF16)):
        _check_label(*make_label_case(n, c, v, dtype, seed=v, device="cuda"))


def test_two_streams_at_once():
    """Two losses on two streams, no order between them: workspaces are each call's own."""
    cases = [make_label_case(5000, 48, 400, F32, seed=k, device="cuda") for k in range(2)]
    want = []
    for x, w, y, b in cases:
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        want.append(torch.autograd.grad(R.label_loss(leaves[0], leaves[1], y, bias=leaves[2]), leaves))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, (x, w, y, b) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
                got[k] = torch.autograd.grad(R.label_loss(leaves[0], leaves[1], y, bias=leaves[2]), leaves)
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(p, q) for p, q in zip(got[k], want[k]))


@pytest.mark.parametrize("n,c", [(5, 3), (1, 771), (3, 7), (67, 515), (200, 1019), (4099, 13), (31, 1022)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_reads_nothing_of_its_neighbours(n, c, dtype):
    """Odd widths are read in vectors that begin and end inside the neighbouring rows: NaN there must not show, nor may
    rows in front of and behind a view."""
    g = torch.Generator().manual_seed(c)
    base = torch.full((n + 2, c), float("nan"), dtype=dtype, device="cuda")
    view = base[1:-1]
    view.copy_(torch.randn(n, c, generator=g).to(dtype))
    _check_norm(view, F32, "input")
    if n > 2:
        hole = view.clone()
        hole[1] = float("nan")
        leaf = hole.requires_grad_(True)
        y = R.layer_norm(leaf)
        (gx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        keep = torch.arange(n, device="cuda") != 1
        assert torch.isfinite(y[keep]).all() and torch.isfinite(gx[keep]).all()


def test_layer_norm_with_eps_zero():
    for planes in (False, True):
        x = torch.randn(70, 24, generator=torch.Generator().manual_seed(5)).cuda()
        leaf = (x.t().contiguous().t() if planes else x).requires_grad_(True)
        w = torch.ones(24, device="cuda", requires_grad=True)
        y = R.layer_norm(leaf, w, eps=0.0)
        gx, gw = torch.autograd.grad(y.square().sum(), [leaf, w])
        assert torch.isfinite(y).all() and torch.isfinite(gx).all() and torch.isfinite(gw).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_every_width(dtype):
    """Every number of channels up to the widest that a group of lanes holds: the number of vectors and lanes, and which of them
    are tested against the row's end, follow from it."""
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(6, 1030, generator=g).to(dtype).cuda(), torch.randn(6, 1030, generator=g).cuda()
    w, b = torch.rand(1030, generator=g).cuda() + 0.5, torch.randn(1030, generator=g).cuda()
    for c in range(1, 1031):
        args = [t[..., :c].contiguous() for t in (x, w, b, dy)]
        ref = norm_reference(*args, 1e-5, args[0], F32, dtype, F32)
        leaves = [t.requires_grad_(True) for t in args[:3]]
        y = R.layer_norm(*leaves, out_dtype=F32)
        for name, got, r in zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, leaves, args[3])), ref):
            assert_within(got, r, f"{name} of {c} channels")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_every_width_and_every_remainder(dtype):
    """Channels 1 to 270 (chunks, stages and what stays in shared memory follow from them), then pixels and labels around the
    tile of 128."""
    for c in list(range(1, 271)) + [319, 320, 321, 383, 384, 385, 511, 513, 576, 640]:
        _check_label(*make_label_case(131, c, 140, dtype, seed=c, device="cuda"))
    for k in list(range(1, 20)) + [63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 384, 385]:
        _check_label(*make_label_case(k, 40, 131, dtype, seed=k, device="cuda"))
        _check_label(*make_label_case(133, 72, k, dtype, seed=k, device="cuda"))


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("n,c", [(24, 64), (24, 36), (23, 33)])
def test_unpack_of_parts_and_of_codes_at_any_byte(n, c, planes):
    x = torch.randn(n, c, generator=torch.Generator().manual_seed(2)) * torch.arange(1, n + 1)[:, None]
    p = R.pack8((x.t().contiguous().t() if planes else x).cuda())
    whole = p.unpack()
    assert torch.equal(whole.cpu().double(), pack_reference(x))
    for part in (slice(None, None, 2), slice(3, 9), slice(5, 6)):
        assert torch.equal(R.Packed8(p.codes[part], p.exponents[part], p.planes, F32).unpack(), whole[part])
    for at in (1, 2, 3, 4):  # dense codes that begin inside a larger buffer
        parts = []
        for t in (p.codes, p.exponents):
            t = t.movedim(-1, 0) if planes else t
            room = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")[at:at + t.numel()].view(t.shape).copy_(t)
            parts.append(room.movedim(0, -1) if planes else room)
        assert parts[0].data_ptr() % 4 == at % 4
        assert torch.equal(R.Packed8(*parts, p.planes, F32).unpack(), whole)
    with pytest.raises(ValueError):
        R.Packed8(p.codes, p.exponents.cpu(), p.planes, F32).unpack()
