"""64-bit definitions of the label-field operators, each with an element-wise bound on what 32-bit (and, where a type asks
for it, 16-bit) arithmetic may be off.  The bounds count roundings: EPS is half a step of float32; a sum of k terms in any
order is off by at most k steps of its absolute sum; a value rounded to a type is off by half a step of that type."""
import torch

EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make_label_case(n, c, v, dtype, seed=0, bias=True, unlabelled=0.2, device="cpu", bias_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, generator=g)
    w = torch.randn(v, c, generator=g) * (2.0 / c ** 0.5)
    y = torch.randint(0, v, (n,), generator=g)
    y[torch.rand(n, generator=g) < unlabelled] = -1
    b = torch.randn(v, generator=g).to(bias_dtype or dtype) if bias else None
    return [None if t is None else t.to(device) for t in (x.to(dtype), w.to(dtype), y, b)]


def label_reference(x, w, y, b, g_rows, out_dtype, bias_dtype=None):
    """losses, dX, dW, db for per-row gradients g_rows, and their bounds.

    Scores: products of the inputs are exact or off by 2^-22 (32-bit inputs in three pieces drop products below that);
    the tensor core adds 16 products at a time, six such sums per 16 channels for 32-bit inputs, and may truncate, so
    a score is off by at most (6 C / 16 + 8) * 2 EPS of its absolute sum.  exp and the running sum: V + 64 steps.
    G is rounded once to bf16 (bf16 inputs) or kept to 2^-22 (three pieces); its products are summed over K terms."""
    xd, wd = x.double(), w.double()
    bd = b.double() if b is not None else torch.zeros(w.shape[0], dtype=torch.float64, device=x.device)
    n, c = xd.shape
    v = wd.shape[0]
    ok = (y >= 0) & (y < v)
    xd = torch.where(ok[:, None], xd, torch.zeros_like(xd))
    s = xd @ wd.t() + bd
    lse = torch.logsumexp(s, 1)
    idx = torch.where(ok, y, torch.zeros_like(y)).long()
    at = s.gather(1, idx[:, None])[:, 0]
    losses = torch.where(ok, lse - at, torch.zeros_like(at))
    finite = torch.where(torch.isfinite(bd), bd, torch.zeros_like(bd))
    mag = (xd.abs() @ wd.abs().t() + finite.abs()).max(1).values  # per row: largest absolute sum of a score
    es = (6 * c / 16 + 8) * 2 * EPS * mag
    loss_tol = torch.where(ok, 2 * es + (v + 64) * 2 * EPS + 4 * EPS * (lse.abs() + at.abs()), torch.zeros_like(at))
    p = torch.exp(s - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, idx[:, None], 1.0)
    gr = torch.where(ok, g_rows.double(), torch.zeros_like(at))[:, None]
    gmat = (p - onehot) * gr
    half = HALF[out_dtype] if out_dtype == torch.bfloat16 else 2.0 ** -22
    # |G| off: rounding of G itself, plus the score's and the lse's error on P, plus 32-bit roundings of P and of the factor
    gerr = gr.abs() * (half * (p - onehot).abs() + p * (2 * es[:, None] + (v + 128) * 2 * EPS) + 4 * EPS * (p + onehot))

    def out(val, err, dtype):
        return val, err + HALF[dtype] * (val.abs() + err) + 1e-38

    gabs = gmat.abs() + gerr
    dx = out(gmat @ wd, gerr @ wd.abs() + (6 * v / 16 + 64) * 2 * EPS * (gabs @ wd.abs()), out_dtype)
    dw = out(gmat.t() @ xd, gerr.t() @ xd.abs() + (6 * n / 16 + 64) * 2 * EPS * (gabs.t() @ xd.abs()), out_dtype)
    # db may be summed from the rounded G
    db = out(gmat.sum(0), gerr.sum(0) + (n + 64) * EPS * gabs.sum(0), bias_dtype or out_dtype)
    return (losses, loss_tol), dx, dw, db


def pack_reference(x):
    """Values of blocks of 32 channels that share the smallest power of two 2^e >= max / 127 (e >= -126); magnitudes
    above 63 * 2^122 count as that (the next code would be 2^128, no finite float32)."""
    xd = x.double().cpu()
    c = xd.shape[-1]
    out = torch.empty_like(xd)
    for lo in range(0, c, 32):
        blk = xd[..., lo:lo + 32]
        for row in torch.cartesian_prod(*[torch.arange(k) for k in xd.shape[:-1]]).view(-1, xd.dim() - 1).tolist() if xd.numel() else []:
            vals = blk[tuple(row)]
            top = float(vals.abs().max())
            if top != top or top == float("inf"):
                out[tuple(row)][lo:lo + 32] = float("nan")
                continue
            e = -126
            while 127.0 * 2.0 ** e < top:
                e += 1
            out[tuple(row)][lo:lo + 32] = torch.round(vals.clamp(-63 * 2.0 ** 122, 63 * 2.0 ** 122) / 2.0 ** e) * 2.0 ** e
    return out.to(x.device)


def norm_reference(x, w, b, dy, eps, kept, out_dtype, x_dtype, p_dtype):
    """y, dx, dw, db in 64 bits and their bounds; ``kept`` holds the values that the backward pass sees."""
    def stats(t):
        mu = t.mean(1, keepdim=True)
        var = ((t - mu) ** 2).mean(1, keepdim=True)
        return mu, 1.0 / torch.sqrt(var + eps)

    n, c = x.shape
    xd, wd, bd, dyd, kd = (t.double() for t in (x, w, b, dy, kept))

    def xhat_of(t):
        mu, r = stats(t)
        h = (t - mu) * r
        # mean: c roundings of max|x|; centred value one more; variance c + 2, root and product 4
        err = r * (c + 4) * EPS * t.abs().max(1, keepdim=True).values
        return h, r, err + h.abs() * ((c + 8) * EPS + 2 * err.clamp(max=1))

    h, _, he = xhat_of(xd)
    y = h * wd + bd
    ye = he * wd.abs() + 4 * EPS * ((h * wd).abs() + bd.abs())
    ye = ye + HALF[out_dtype] * (y.abs() + ye)
    h, r, he = xhat_of(kd)
    rel_r = (c + 8) * EPS + 2 * (r * (c + 4) * EPS * kd.abs().max(1, keepdim=True).values).clamp(max=1)
    a = dyd * wd
    sa, sax = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    ma, max_ = a.abs().mean(1, keepdim=True), (a * h).abs().mean(1, keepdim=True)
    dx = r * (a - sa - h * sax)
    inner = 4 * EPS * a.abs() + (c + 4) * EPS * ma + he * sax.abs() + (h.abs() + he) * ((c + 6) * EPS * max_ + (a.abs() * he).mean(1, keepdim=True))
    dxe = r * (1 + rel_r) * inner + rel_r * dx.abs() + 4 * EPS * r * (a.abs() + ma + h.abs() * max_)
    dxe = dxe + HALF[x_dtype] * (dx.abs() + dxe) + 1e-38
    dw, db = (dyd * h).sum(0), dyd.sum(0)
    dwe = (dyd.abs() * he).sum(0) + (n + 4) * EPS * (dyd * h).abs().sum(0)
    dbe = (n + 4) * EPS * dyd.abs().sum(0)
    dwe, dbe = dwe + HALF[p_dtype] * (dw.abs() + dwe), dbe + HALF[p_dtype] * (db.abs() + dbe)
    return (y, ye), (dx, dxe), (dw, dwe), (db, dbe)


def assert_within(got, ref, what=""):
    val, tol = ref
    val, tol = val.reshape(got.shape), tol.reshape(got.shape)
    diff = (got.double() - val).abs()
    bad = ~(diff <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(diff.max()):.3e}, "
                           f"largest excess over the bound x{float((diff / tol.clamp(min=1e-300)).max()):.3g}")
