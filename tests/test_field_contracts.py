"""Label loss, layer norm and 8-bit features where callers meet them from the side: saved-tensor hooks, layouts of gradients,
limits inside the accepted ranges.  Every case runs on the CPU backend and on the GPU."""
import time

import pytest
import torch

import retinags_b200 as R
from retinags_b200.ops import native
from field_reference import assert_within, label_reference, make_label_case

F32, BF16 = torch.float32, torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _dense_copy(t):
    """The values, densely, inside a larger buffer: other strides and another alignment."""
    room = torch.zeros(4 * t.numel() + 9, dtype=t.dtype, device=t.device)
    return room[5:5 + t.numel()].view(t.shape).copy_(t)


def _wide_copy(t):
    """The values with gaps between the rows."""
    if t.dim() == 0:
        return t.clone()
    room = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    return room[..., 1:2 * t.shape[-1] + 1:2].copy_(t)


def _other_order(t):
    return t.movedim(-1, 0).contiguous().movedim(0, -1) if t.dim() > 1 else t.clone()


COPIES = [_dense_copy, _wide_copy, _other_order]


@pytest.mark.parametrize("copy", COPIES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("device", DEVICES)
def test_label_loss_takes_its_saved_tensors_in_any_layout(device, dtype, copy):
    x, w, y, b = make_label_case(60, 24, 17, dtype, seed=2, device=device)
    wide, ww = torch.zeros(61, 40, dtype=dtype, device=device), torch.zeros(18, 41, dtype=dtype, device=device)
    wide[:60, 8:32], ww[1:, 7:31] = x, w
    for f, v in ((x, w), (wide[:60, 8:32], w), (x, ww[1:, 7:31]), (x.t().contiguous().t(), w), (wide[:60, 8:32].view(5, 12, 24), w)):
        leaves = [t.detach().requires_grad_(True) for t in (f, v, b)]
        labels = y.view(f.shape[:-1])
        for reduction in ("mean", "none"):
            up = torch.rand(labels.shape, generator=torch.Generator().manual_seed(1)).to(device) if reduction == "none" else None
            out = R.label_loss(leaves[0], leaves[1], labels, bias=leaves[2], reduction=reduction)
            want = torch.autograd.grad(out, leaves, up)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone() if t is not None else t, copy):
                out = R.label_loss(leaves[0], leaves[1], labels, bias=leaves[2], reduction=reduction)
            got = torch.autograd.grad(out, leaves, up)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("copy", COPIES)
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_takes_its_saved_tensors_in_any_layout(device, dtype, keep, copy):
    gen = torch.Generator().manual_seed(4)
    for n, c in ((35, 24), (1, 40), (35, 33), (6, 600)):
        x, dy = torch.randn(n, c, generator=gen).to(dtype).to(device), torch.randn(n, c, generator=gen).to(dtype).to(device)
        w, b = (torch.rand(c, generator=gen).to(device).requires_grad_(True) for _ in range(2))
        wide = torch.zeros(n + 1, c + 11, dtype=dtype, device=device)
        wide[:n, 4:c + 4] = x
        for f in (x, x.t().contiguous().t(), wide[:n, 4:c + 4], wide[:n, 4:c + 4].t().contiguous().t()):
            leaf = f.detach().requires_grad_(True)
            want = torch.autograd.grad(R.layer_norm(leaf, w, b, keep=keep), [leaf, w, b], dy)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), copy):
                y = R.layer_norm(leaf, w, b, keep=keep)
            got = torch.autograd.grad(y, [leaf, w, b], dy)
            assert got[0].stride() == want[0].stride()
            # another layout may take another kernel, which adds in another order.  Two sums of 35 rows with |dy xhat| about 22
            # in all: 2 * 39 * 2^-24 * 22 = 1e-4; means over 600 channels: 2 * 606 * 2^-24 = 7e-5; 16-bit outputs may then
            # round to the neighbour, 2^-7 of the value
            for p, q in zip(got, want):
                torch.testing.assert_close(p, q, atol=2e-4, rtol=0 if p.dtype == F32 else 2.0 ** -7)


@pytest.mark.parametrize("device", DEVICES)
def test_save_on_cpu_and_planes(device):
    planes = torch.randn(24, 5, 7, generator=torch.Generator().manual_seed(4)).to(device)
    w, v = (torch.randn(24, generator=torch.Generator().manual_seed(5)).to(device).requires_grad_(True),
            torch.randn(9, 24, generator=torch.Generator().manual_seed(6)).to(device).requires_grad_(True))
    labels = torch.arange(35, device=device).view(5, 7) % 9
    for keep in ("input", "int8"):
        grads = []
        for offload in (False, True):
            leaf = planes.clone().requires_grad_(True)
            hook = torch.autograd.graph.save_on_cpu() if offload else torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)
            with hook:
                loss = R.label_loss(R.layer_norm(leaf.permute(1, 2, 0), w, keep=keep), v, labels)
            grads.append(torch.autograd.grad(loss, [leaf, w, v]))
        for p, q in zip(*grads):
            torch.testing.assert_close(p, q, atol=1e-6, rtol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_saved_tensors_of_another_kind_are_refused(device):
    x, w, y, b = make_label_case(12, 8, 5, F32, seed=2, device=device)
    bad = [lambda t: t.double() if t.is_floating_point() else t, lambda t: t[:-1] if t.dim() and t.shape[0] > 1 else t,
           lambda t: t.bfloat16() if t.dtype == F32 else t.short() if t.dtype != torch.int8 else t, lambda t: t.to("meta")]
    for unpack in bad:
        for op in ("label", "input", "int8"):
            leaf, gain = x.clone().requires_grad_(True), torch.ones(8, device=device, requires_grad=True)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                out = R.label_loss(leaf, w, y, bias=b) if op == "label" else R.layer_norm(leaf, gain, keep=op).sum()
            with pytest.raises(RuntimeError, match="came back as"):
                torch.autograd.grad(out, leaf)


def test_shifted_rows_are_read_inside_the_tensor():
    """Vectors of four that begin in the row in front: for every width and stride that the rule admits, those of all rows but the
    last (read element by element) end inside the tensor."""
    admitted, cpu = 0, torch.device("cpu")
    for c in list(range(1, 24)) + [771, 1017, 1018, 1019]:
        for ld in range(c, c + 13):
            if not native.size_of("rows_shifted", cpu, c, ld):
                continue
            admitted += 1
            for n in range(1, 12):
                total = (n - 1) * ld + c
                for row in range(n - 1):
                    start = row * ld - (row * c) % 4
                    assert start % 4 == 0 and start >= 0
                    assert -(-(row * ld + c) // 4) * 4 <= total, (n, c, ld, row)
    assert admitted > 60
    assert not native.size_of("rows_shifted", cpu, 1, 1) and not native.size_of("rows_shifted", cpu, 1019, 1019)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_of_one_channel(device, dtype):
    """Nothing varies: the output is the bias, and neither the input nor the weight has a gradient."""
    for n in range(1, 14):
        for stride in (1, 2, 5):
            room = torch.randn(n * stride, dtype=torch.float32, generator=torch.Generator().manual_seed(n)).to(dtype).to(device)
            leaf = room[::stride].view(n, 1).detach().requires_grad_(True)
            w, b = torch.full((1,), 3.0, device=device, requires_grad=True), torch.full((1,), 0.5, device=device, requires_grad=True)
            y = R.layer_norm(leaf, w, b, out_dtype=F32)
            gx, gw, gb = torch.autograd.grad(y, [leaf, w, b], torch.ones_like(y))
            assert (y == 0.5).all() and (gx == 0).all() and gw.item() == 0.0 and gb.item() == n


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("spread,bias", [(3e4, 1.0), (3e4, 40.0), (3e4, 300.0), (3e3, 1.0), (3e3, 40.0)])
def test_label_loss_scores_that_32_bits_hold_coarsely(device, dtype, spread, bias):
    """Scores of 1e9 lie 64 apart in 32 bits.  Probabilities stay probabilities: gradients are differences of two rows of the
    weight (or their averages over labels that tie), never infinite."""
    x, w, y, b = make_label_case(40, 8, 50, F32, seed=3, device=device, unlabelled=0.0)
    leaves = [(t * s).to(dtype).requires_grad_(True) for t, s in ((x, spread), (w, spread), (b, bias))]
    losses = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2], reduction="none")
    gx, gw, gb = torch.autograd.grad(losses.sum(), leaves)
    xd, wd = leaves[0].detach().double(), leaves[1].detach().double()
    s = xd @ wd.t() + leaves[2].detach().double()
    at = s.gather(1, y[:, None])[:, 0]
    # a score: (6 C / 16 + 8) * 2 roundings of its absolute sum (three pieces on the tensor core; fewer on the CPU)
    es = (6 * 8 / 16 + 8) * 2 * 2.0 ** -24 * (xd.abs() @ wd.abs().t()).max(1).values
    want = torch.logsumexp(s, 1) - at
    assert ((losses.detach().double() - want).abs() <= 2 * es + 2.0 ** -23 * want.abs() + 1e-4).all()
    assert all(torch.isfinite(g).all() for g in (gx, gw, gb))
    # sum_v |p_v - [v = y]| is at most 2: |dx| <= 2 max|w|, |dw_v| <= sum_n |x_n|, |db_v| <= pixels (and the outputs' rounding)
    room = 1.0 + 2.0 ** -7
    assert (gx.abs().double() <= 2 * wd.abs().max(0).values * room).all()
    assert (gw.abs().double() <= xd.abs().sum(0) * room).all() and (gb.abs() <= 40 * room).all()
    # where the largest score is far above the others, p is one label and the gradient is w_top - w_y
    top = s.topk(2, 1).values
    clear = top[:, 0] - top[:, 1] > 4 * es + 40.0
    assert clear.sum() > 20
    ref = (wd[s.argmax(1)] - wd[y])[clear]
    half = 2.0 ** -24 if dtype == F32 else 2.0 ** -8
    assert ((gx[clear].double() - ref).abs() <= 2 * half * ref.abs() + 2.0 ** -21 * wd.abs().max()).all()


@pytest.fixture
def label_limit():
    """Sets a limit of the label kernel (0: tries of a wait, 1: stages that a producer fills, 2: bytes of partial sums); defaults
    afterwards."""
    dev = torch.device("cuda")
    yield lambda which, value: native.size_of("label_limit", dev, which, value)
    for which in (0, 1, 2):
        native.size_of("label_limit", dev, which, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,v,dtype", [(20000, 64, 700, BF16), (3000, 300, 900, BF16), (20000, 32, 300, F32), (2000, 200, 600, F32),
                                         (300, 64, 9000, BF16), (20000, 40, 100, BF16)])
def test_label_loss_is_right_or_nan_when_waits_run_out(label_limit, n, c, v, dtype):
    """The producer of every CTA gives up after a few stages, or waits have a few tries only: the call returns, every number
    that it gives is that of an undisturbed run or NaN, and the next call is undisturbed."""
    x, w, y, b = make_label_case(n, c, v, dtype, seed=c, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    labelled = y >= 0
    up = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() + 0.5

    def forward(reduction):
        return R.label_loss(x, w, y, bias=b, reduction=reduction)

    def right_or_nan(got, want):
        assert (torch.isnan(got) | (got == want)).all()
        return bool(torch.isnan(got).any())

    losses, mean = forward("none").detach(), forward("mean").detach()
    grads = {r: torch.autograd.grad(forward(r), leaves, u) for r, u in (("none", up), ("mean", None))}
    assert all(torch.isfinite(t).all() for t in (losses, mean, *grads["none"], *grads["mean"]))
    for which, values in ((1, (0, 1, 2, 3, 5, 8, 13, 40)), (0, (0, 1, 2, 3, 6))):
        for value in values:
            label_limit(which, value)
            got = forward("none").detach()
            hit = right_or_nan(got, losses)
            got_mean = forward("mean").detach()
            right_or_nan(got_mean, mean)
            label_limit(which, -1)
            if value == 0:
                assert hit and torch.isnan(got[labelled]).all() and torch.isnan(got_mean) and (got[~labelled] == 0).all()
            for reduction, u in (("none", up), ("mean", None)):
                out = forward(reduction)
                label_limit(which, value)
                part = torch.autograd.grad(out, leaves, u)
                label_limit(which, -1)
                hits = [right_or_nan(p, q) for p, q in zip(part, grads[reduction])]
                if value == 0:
                    assert all(hits) and torch.isnan(part[0][labelled]).all() and (part[0][~labelled] == 0).all()
                    assert torch.isnan(part[1]).all() and torch.isnan(part[2]).all()
        # a forward pass that gave up: what hangs on it is NaN in the backward pass, not a gradient of something else
        label_limit(which, 0)
        out = forward("mean")
        label_limit(which, -1)
        assert all(torch.isnan(t).any() for t in (out, *torch.autograd.grad(out, leaves)))
    assert torch.equal(forward("none"), losses)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(forward("mean"), leaves), grads["mean"]))


@pytest.mark.gpu
@pytest.mark.parametrize("room", [-1, 0, 200000])
@pytest.mark.parametrize("which", ["features", "weight"])
def test_label_loss_32_bit_sums_of_one_sign_whatever_the_room(label_limit, which, room):
    """Gradients that add 32768 numbers of one sign.  All scores are zero (so every p is 1/V) and the label's own row adds nothing.

    The tensor core truncates where it adds, by less than 2^-23 of the sum a step.  Accumulators of eight tiles take 64 steps:
    64 * 2^-23 = 7.7e-6 of the sum; the pieces of 256 tiles are 32 to 256 sums rounded to nearest, 288 * 2^-25 on average over a
    growing sum = 8.6e-6 if all went one way; p is off by 2e-6 (logarithm, exponential).  With one accumulator for all, 2048
    steps lose half of 2^-23.5 of a sum that grows to its end: 4e-5."""
    label_limit(2, room)
    gen = torch.Generator().manual_seed(7)
    big, small, c = 32768, 130, 64
    if which == "features":
        x = torch.zeros(small, c, device="cuda", requires_grad=True)
        w = (torch.rand(big, c, generator=gen) + 0.5).cuda()
        w[0] = 0.0
        leaf, y = x, torch.zeros(small, dtype=torch.long, device="cuda")
    else:
        x = (torch.rand(big, c, generator=gen) + 0.5).cuda()
        w = torch.zeros(small, c, device="cuda", requires_grad=True)
        leaf, y = w, torch.zeros(big, dtype=torch.long, device="cuda")
    (g,) = torch.autograd.grad(R.label_loss(x, w, y, reduction="sum"), leaf)
    if which == "features":
        want = (w.double().sum(0) / big).expand(small, c)
    else:
        g, want = g[1:], (x.double().sum(0) / small).expand(small - 1, c)
    err = ((g.double() - want) / want).abs().max().item()
    assert err <= 7.7e-6 + 8.6e-6 + 2e-6, err


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,v,dtype", [(300, 64, 3000, F32), (3000, 200, 300, F32), (3000, 33, 2900, F32), (130, 64, 70000, BF16), (70000, 40, 130, BF16),
                                         (70000, 300, 130, BF16)])
def test_label_loss_pieces_that_follow_each_other(label_limit, n, c, v, dtype):
    """No room for more than one partial sum: its pieces are added launch after launch; the same bits every time."""
    x, w, y, b = make_label_case(n, c, v, dtype, seed=n, device="cuda")
    count = max(int((y >= 0).sum()), 1)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    ref = label_reference(x.detach(), w.detach(), y, b.detach(), torch.full((n,), 1.0 / count, device="cuda"), dtype)
    full = torch.autograd.grad(R.label_loss(x, w, y, bias=b), leaves)
    label_limit(2, 0)
    runs = [torch.autograd.grad(R.label_loss(x, w, y, bias=b), leaves) for _ in range(2)]
    for name, got, again, r in zip(("dX", "dW", "db"), *runs, ref[1:]):
        assert_within(got, r, name)
        assert torch.equal(got, again)
    for got, r in zip(full, ref[1:]):
        assert_within(got, r)
    for k in range(3):  # one gradient alone: the same bits
        t = [p.detach() for p in leaves]
        t[k].requires_grad_(True)
        (g,) = torch.autograd.grad(R.label_loss(t[0], t[1], y, bias=t[2]), t[k])
        assert torch.equal(g, runs[0][k])


@pytest.mark.gpu
def test_label_loss_refuses_a_workspace_that_is_too_small(label_limit):
    """A workspace sized under another limit than the call's is refused, not overrun."""
    x, w, y, b = make_label_case(3000, 64, 3000, F32, seed=1, device="cuda")
    loss = R.label_loss(x.requires_grad_(True), w, y, bias=b)
    want = torch.autograd.grad(loss, x, retain_graph=True)
    from retinags_b200.ops import label_loss as module
    sized = module._scratch
    try:
        module._scratch = lambda *a: sized(*a)[:-1]
        with pytest.raises(RuntimeError, match="status 24"):
            torch.autograd.grad(loss, x, retain_graph=True)
        with pytest.raises(RuntimeError, match="status 24"):
            R.label_loss(x, w, y, bias=b)
    finally:
        module._scratch = sized
    assert torch.equal(torch.autograd.grad(loss, x)[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_label_loss_takes_room_for_the_gradients_asked_for(dtype, monkeypatch):
    """Partial sums of dX and of dW are in the workspace only where that gradient is asked for; values do not depend on it."""
    from retinags_b200.ops import label_loss as module
    sized, sizes = module._scratch, []
    monkeypatch.setattr(module, "_scratch", lambda *a: (lambda t: (sizes.append(t.numel()), t)[1])(sized(*a)))
    n, c, v = 20000, 64, 3000
    x, w, y, b = make_label_case(n, c, v, dtype, seed=3, device="cuda")
    out, used = {}, {}
    for wanted in ((0, 1, 2), (0,), (1,), (2,), (0, 2), (1, 2)):
        t = [p.detach().requires_grad_(k in wanted) for k, p in enumerate((x, w, b))]
        loss = R.label_loss(t[0], t[1], y, bias=t[2])
        sizes.clear()
        out[wanted] = dict(zip(wanted, torch.autograd.grad(loss, [t[k] for k in wanted])))
        (used[wanted],) = sizes
    for wanted, grads in out.items():
        assert all(torch.equal(g, out[(0, 1, 2)][k]) for k, g in grads.items())
    assert used[(0,)] < used[(0, 2)] < used[(0, 1, 2)] and used[(2,)] < used[(1, 2)] < used[(0, 1, 2)]
    parts_w = used[(1, 2)] - used[(2,)]  # pieces of dW, 24 tiles of 128 labels each
    assert parts_w >= 24 * 128 * 64 * 4 and used[(0, 1, 2)] - used[(0, 2)] == parts_w


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,v,dtype", [(20000, 64, 3000, F32), (20000, 64, 3000, BF16), (30000, 200, 300, BF16), (9000, 100, 900, F32)])
def test_label_loss_gradients_do_not_depend_on_what_else_is_asked_for(n, c, v, dtype):
    x, w, y, b = make_label_case(n, c, v, dtype, seed=3, device="cuda")
    out = {}
    for wanted in ((0, 1, 2), (0,), (1,), (2,), (0, 2), (1, 2), (0, 1)):
        t = [p.detach().requires_grad_(k in wanted) for k, p in enumerate((x, w, b))]
        out[wanted] = dict(zip(wanted, torch.autograd.grad(R.label_loss(t[0], t[1], y, bias=t[2]), [t[k] for k in wanted])))
    for wanted, grads in out.items():
        for k, g in grads.items():
            assert torch.equal(g, out[(0, 1, 2)][k]), (wanted, k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [24, 64, 300])
@pytest.mark.parametrize("device", DEVICES)
def test_label_loss_without_labels_gives_zeros_whatever_the_classifier_holds(device, c, dtype):
    x, w, y, b = make_label_case(150, c, 140, dtype, seed=5, device=device)
    y[:] = -1
    w[3, 1], w[139, 0], b[7] = float("nan"), float("inf"), float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for reduction in ("mean", "sum", "none"):
        out = R.label_loss(x, w, y, bias=b, reduction=reduction)
        assert (out == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out.sum(), leaves))


def test_cpu_layer_norm_is_linear_in_the_channels():
    """The weight's gradient takes a row's mean and variance once, not once a channel: 32 times the channels in the same number
    of elements must not take 32 times as long (4 times is allowed for caches and a busy machine)."""
    def seconds(n, c):
        x, dy = torch.randn(n, c, generator=torch.Generator().manual_seed(1)), torch.ones(n, c)
        w = torch.ones(c, requires_grad=True)
        best = float("inf")
        for _ in range(3):
            y = R.layer_norm(x, w)
            t = time.perf_counter()
            torch.autograd.grad(y, w, dy)
            best = min(best, time.perf_counter() - t)
        return best
    seconds(64, 32)
    assert seconds(512, 1024) < 4 * seconds(16384, 32) + 0.05


@pytest.mark.gpu
def test_launch_count_is_that_of_the_profiler():
    from torch.profiler import ProfilerActivity, profile
    gen = torch.Generator().manual_seed(1)

    def label(n, c, v, dtype, wanted, reduction="mean"):
        t = [p.detach().requires_grad_(k in wanted) for k, p in enumerate(p for p in make_label_case(n, c, v, dtype, device="cuda") if p.dtype != torch.int64)]
        y = torch.zeros(n, dtype=torch.long, device="cuda")
        out = R.label_loss(t[0], t[1], y, bias=t[2], reduction=reduction)
        up = torch.ones_like(out)
        return lambda: torch.autograd.grad(out, [t[k] for k in wanted], up, retain_graph=True) if wanted else R.label_loss(t[0], t[1], y, bias=t[2])

    def norm(n, c, keep, planes, backward):
        x = torch.randn(n, c, generator=gen).cuda()
        leaf = (x.t().contiguous().t() if planes else x).requires_grad_(True)
        w = torch.ones(c, device="cuda", requires_grad=True)
        y = R.layer_norm(leaf, w, keep=keep)
        up = torch.ones_like(y)
        return (lambda: torch.autograd.grad(y, [leaf, w], up, retain_graph=True)) if backward else (lambda: R.layer_norm(leaf, w, keep=keep))

    packed = R.pack8(torch.randn(50, 40, generator=gen).cuda())
    steps = [label(300, 64, 100, BF16, ()), label(300, 64, 100, BF16, (0,)), label(300, 64, 100, F32, (1,)), label(40000, 64, 100, F32, (0, 1, 2)),
             label(40000, 64, 3000, F32, (0, 1, 2)), label(60000, 64, 100, BF16, (0,)), label(300, 64, 100, BF16, (2,), "none"),
             norm(5, 64, "input", False, True), norm(5000, 64, "input", False, True), norm(500, 33, "int8", False, False),
             norm(500, 64, "int8", False, False), norm(300, 1500, "int8", False, False), norm(300, 1500, "input", False, True),
             norm(300, 64, "int8", True, True), lambda: packed.unpack(), lambda: R.pack8(packed.unpack())]
    for k, step in enumerate(steps):
        step()
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            before = native.launch_count()
            step()
            torch.cuda.synchronize()
            counted = native.launch_count() - before
        seen = sum(e.count for e in prof.key_averages() if "rgs_" in e.key)
        assert counted == seen > 0, (k, counted, seen)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("keep", ["input", "int8"])
@pytest.mark.parametrize("device", DEVICES)
def test_layouts_of_the_norm_and_of_gradients(device, keep, out_dtype):
    """The output is dense rows whatever the input; the kernels' gradient is dense, as planes where the input is planes (a slice of
    them too), else as rows.  A leaf's own gradient then follows autograd's rule for leaves."""
    base = torch.randn(40, 91, generator=torch.Generator().manual_seed(1)).to(device)
    rows, planes = (24, 1), (1, 30)
    for view, want in ((base[:30, :24], rows), (base[:30, 5:29], rows), (base[:30, ::3][:, :24], rows), (base[::1, :30].t()[:, 3:27], planes),
                       (base[:24, 7:37].t(), planes), (base[:24, :30].t().contiguous(), rows), (base[0:1, :24].expand(30, 24), rows)):
        assert view.shape == (30, 24)
        seen = []
        leaf = view.detach().requires_grad_(True)
        y = R.layer_norm(leaf.view_as(leaf), keep=keep, out_dtype=out_dtype)
        assert y.is_contiguous() and y.dtype == out_dtype
        y.grad_fn.register_hook(lambda grads, _: seen.append(grads[0]))
        (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert seen[0].stride() == want and g.shape == leaf.shape
        want_y = torch.nn.functional.layer_norm(view.double(), (24,))
        # half a step of the output's type; a row of 24: 40 roundings of values below 4, times 1/sqrt(var) below 2
        torch.testing.assert_close(y.double(), want_y, atol=40 * 2.0 ** -24 * 8, rtol=2.0 ** -24 if out_dtype == F32 else 2.0 ** -8)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("device", DEVICES)
def test_label_field_on_rendered_planes(device, dtype):
    """Planes as the rasteriser writes them, three channels a render, through norm and loss; gradients reach the splats' features and
    are those of the plain formulas."""
    from helpers import activated, small_scene
    from retinags_b200.ops.rasterize import GaussianRasterizationSettings, GaussianRasterizer
    from retinags_b200.utils import loss as plain
    g, cams = small_scene(n=300, width=80, height=48)
    cam = cams[0]
    a = {k: v.to(device) for k, v in activated(g).items()}
    mats = [torch.as_tensor(m).to(device) for m in (cam.world_view_transform, cam.full_proj_transform, cam.view_world_transform, cam.camera_center)]
    st = GaussianRasterizationSettings(cam.height, cam.width, cam.tan_fovx, cam.tan_fovy, torch.zeros(3, device=device), 1.0, *mats[:3],
                                       torch.full((3,), -1e9), torch.full((3,), 1e9), 0, mats[3])
    gen = torch.Generator().manual_seed(3)
    feats = (torch.rand(300, 4, 1, 3, generator=gen) * 2).to(device).requires_grad_(True)  # twelve channels
    labels = torch.randint(-1, 7, (48, 80), generator=gen).to(device)
    gain = torch.ones(12, device=device, requires_grad=True)
    w = torch.randn(7, 12, generator=gen).to(device).to(dtype).requires_grad_(True)
    raster, rest = GaussianRasterizer(st), torch.zeros(300, 15, 3, device=device)

    def planes_of(f):
        return torch.cat([raster(a["xyz"], torch.zeros_like(a["xyz"]), a["opacity"], shs=torch.cat([f[:, k], rest], 1), scales=a["scale"],
                                 rotations=a["rot"])[0] for k in range(4)])

    planes = planes_of(feats)
    assert planes.shape == (12, 48, 80) and planes.is_contiguous()
    # eps is that of features of size one: pixels without a splat keep a small scale
    for keep in ("input", "int8"):
        loss = R.label_loss(R.layer_norm(planes.permute(1, 2, 0), gain, eps=1e-2, out_dtype=dtype, keep=keep), w, labels)
        gp, gg, gw = torch.autograd.grad(loss, [planes, gain, w], retain_graph=True)
        kept = R.pack8(planes.detach().permute(1, 2, 0)).unpack().double() if keep == "int8" else planes.detach().permute(1, 2, 0).double()
        p, gd = planes.detach().permute(1, 2, 0).double().requires_grad_(True), gain.detach().double().requires_grad_(True)
        h = torch.nn.functional.layer_norm(p, (12,), gd, None, 1e-2)
        hr = h.to(dtype).double()  # what the classifier reads
        wd = w.detach().double().requires_grad_(True)
        want = plain.label_loss(hr.detach().requires_grad_(True), wd, labels)
        hl = hr.detach().requires_grad_(True)
        gh, gwd = torch.autograd.grad(plain.label_loss(hl, wd, labels), [hl, wd])
        k = kept.requires_grad_(True)
        hk = torch.nn.functional.layer_norm(k, (12,), gd, None, 1e-2)
        gk, ggd = torch.autograd.grad(hk, [k, gd], gh)
        # 32 bits: some hundred roundings of sums; bf16: G, dh and dW are rounded (three halves of 2^-8), h may round to the other side
        rel = 2e-5 if dtype == F32 else 4 * 2.0 ** -8
        assert abs(loss.item() - want.item()) <= rel * want.item()
        for got, ref in ((gp.permute(1, 2, 0), gk), (gg, ggd), (gw, gwd)):
            assert (got.double() - ref).norm() <= rel * ref.norm()
        # a render's backward pass is for one call, so each gradient has a render of its own.  Two renders on the GPU add a splat's
        # gradient up in another order (some hundred pixels of a sum: 1e-4 is far above that), and h may round to the other side
        (gf,) = torch.autograd.grad(R.label_loss(R.layer_norm(planes_of(feats).permute(1, 2, 0), gain, eps=1e-2, out_dtype=dtype, keep=keep), w, labels), feats)
        (ref,) = torch.autograd.grad(planes_of(feats), feats, gp)
        assert torch.isfinite(gf).all() and gf.abs().max() > 0 and (gf - ref).norm() <= max(rel, 1e-4) * ref.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [8, 33, 64, 100, 200, 300, 700])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_label_loss_large_scores_at_every_width(c, dtype, reduction):
    """Scores of thousands beside ordinary ones, pixels without a label among them, one with infinite features: how A and B are
    staged hangs on the width, and m comes off in registers in each of these forms."""
    x, w, y, b = make_label_case(270, c, 333, F32, seed=c, device="cuda")
    x[:90] *= 1500.0
    x, w, b = x.to(dtype), w.to(dtype), b.to(dtype)
    free = int((y < 0).nonzero()[0])
    count = int((y >= 0).sum())
    up = torch.rand(270, generator=torch.Generator().manual_seed(1)).cuda() + 0.5 if reduction == "none" else torch.full((270,), 1.0 / count, device="cuda")
    ref = label_reference(x, w, y, b, up, dtype)
    x[free, c // 2] = float("inf")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = R.label_loss(leaves[0], leaves[1], y, bias=leaves[2], reduction=reduction)
    if reduction == "none":
        assert_within(out.detach(), ref[0], "losses")
    grads = torch.autograd.grad(out, leaves, up if reduction == "none" else None)
    for name, got, r in zip(("dX", "dW", "db"), grads, ref[1:]):
        assert_within(got, r, name)


def test_no_gradient_passes_through_the_8_bit_form():
    x = torch.randn(5, 40, requires_grad=True)
    assert not R.pack8(x).unpack().requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_in_8_bits_at_every_width(dtype, planes):
    """The kept codes are those of the 8-bit form at every number of channels (lanes, vectors and blocks of 32 follow from it), and
    the gradients are those of the norm at their values."""
    from field_reference import norm_reference
    gen = torch.Generator().manual_seed(5)
    x, dy = torch.randn(37, 1100, generator=gen).to(dtype), torch.randn(37, 1100, generator=gen).cuda()
    w, b = (torch.rand(1100, generator=gen) + 0.5).cuda(), torch.randn(1100, generator=gen).cuda()
    widths = list(range(1, 140)) + list(range(140, 530, 13)) + [511, 512, 513, 544, 575, 576, 640, 771, 772, 1000, 1018, 1019, 1023, 1024, 1025, 1056, 1100]
    for c in widths:
        part = x[:, :c].contiguous()
        host = R.pack8(part)
        leaf = part.cuda()
        leaf = (leaf.t().contiguous().t() if planes else leaf).requires_grad_(True)
        leaves = [leaf, w[:c].clone().requires_grad_(True), b[:c].clone().requires_grad_(True)]
        up = dy[:, :c].contiguous()
        y = R.layer_norm(*leaves, keep="int8", out_dtype=F32)
        codes, exponents = (t for t in y.grad_fn.saved_tensors if t is not None and t.dtype in (torch.int8, torch.uint8))
        assert torch.equal(codes.cpu(), host.codes) and torch.equal(exponents.cpu(), host.exponents), c
        ref = norm_reference(part.cuda(), leaves[1].detach(), leaves[2].detach(), up, 1e-5, host.unpack(F32).cuda(), F32, dtype, F32)
        for name, got, r in zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, leaves, up)), ref):
            assert_within(got, r, f"{name} of {c} channels")
