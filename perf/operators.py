"""Cases that measure the operators for label fields: label loss, layer norm and 8-bit kept features.

A label field is trained on rendered features: every pixel of a view is a row with C channels, a classifier scores it
against V labels (classes, instances, or the entries of a codebook).  ``run`` is one pass of one operator, either in
elementary torch operations (``own`` false) or through the framework (``own`` true).
"""
from __future__ import annotations

import math

import torch

own = False

_CHUNK = 1 << 28  # elements of a block of logits in the plain form


def listed():
    return [
        # a viewer asks which label one pixel has: latency
        dict(name="label_one_pixel", op="label", rows=1, channels=64, vocab=4096, dtype="bf16", train=False, bias=True),
        # a random crop of a view against a small set of classes, odd sizes
        dict(name="label_crop_f32", op="label", rows=4099, channels=33, vocab=150, dtype="f32", train=True, bias=True),
        # a 320 x 208 view, the renderer's 32-bit features as they are
        dict(name="label_view_small_f32", op="label", rows=320 * 208, channels=32, vocab=256, dtype="f32", train=True, bias=False),
        # a 1600 x 1036 view, 32-bit features, instance ids
        dict(name="label_view_f32", op="label", rows=1600 * 1036, channels=32, vocab=512, dtype="f32", train=True, bias=True),
        # the same view in bf16 behind the norm, a larger set of labels
        dict(name="label_view_bf16", op="label", rows=1600 * 1036, channels=64, vocab=1024, dtype="bf16", train=True, bias=True),
        # codebook of features with an odd number of entries, wide rows
        dict(name="label_codebook_bf16", op="label", rows=320 * 208, channels=256, vocab=32771, dtype="bf16", train=True, bias=False),
        # a handful of pixels through the norm
        dict(name="norm_few_rows", op="norm", rows=77, channels=64, planes=False, dtype="f32", out="f32", keep="input"),
        # the renderer's planes of a whole view, turned into bf16 rows for the loss
        dict(name="norm_planes_view", op="norm", rows=1600 * 1036, channels=64, planes=True, dtype="f32", out="bf16", keep="input"),
        # rows of a whole view, kept in 8 bits between the passes
        dict(name="norm_rows_int8_view", op="norm", rows=1600 * 1036, channels=64, planes=False, dtype="f32", out="bf16", keep="int8"),
        # wide rows of an odd width in bf16
        dict(name="norm_wide_odd_bf16", op="norm", rows=40003, channels=771, planes=False, dtype="bf16", out="bf16", keep="input"),
        # a small view's features packed and restored, the last block of a row short
        dict(name="pack_small_odd", op="pack", rows=320 * 208, channels=33, dtype="f32"),
        # a whole view's features packed and restored
        dict(name="pack_view", op="pack", rows=1600 * 1036, channels=64, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["label", "label", "norm", "norm", "pack"])
    if op == "label":
        dtype = rng.choice(["f32", "bf16"])
        channels = _log_int(rng, 3, 256 if dtype == "bf16" else 128)
        vocab = _log_int(rng, 2, 32771)
        wide = 64 * ((channels + 63) // 64) * (1 if dtype == "bf16" else 6)  # 32-bit features cost several products
        most = min(1600 * 1036, (320 * 208 * 256 * 32771) // (wide * max(vocab, 128) * 2))
        return dict(op=op, rows=_log_int(rng, 1, most), channels=channels, vocab=vocab, dtype=dtype, train=rng.random() < 0.75,
                    bias=rng.random() < 0.5)
    channels = _log_int(rng, 1, 1024)
    rows = _log_int(rng, 1, min(1600 * 1036, (1600 * 1036 * 64) // channels))
    if op == "norm":
        return dict(op=op, rows=rows, channels=channels, planes=rng.random() < 0.4, dtype=rng.choice(["f32", "bf16"]),
                    out=rng.choice(["f32", "bf16"]), keep=rng.choice(["input", "int8"]))
    return dict(op=op, rows=rows, channels=channels, dtype=rng.choice(["f32", "bf16"]))


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    n, c = case["rows"], case["channels"]
    dt = _TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    # blended features: a channel offset and a pixel's coverage scale the sum over its splats
    cover = torch.rand(n, 1, generator=g, device=dev) * 0.9 + 0.1
    x = randn(n, c)
    x += 0.3 * randn(1, c)
    if case["op"] != "label":
        x *= cover
    st = dict(case=case)
    if case["op"] == "label":
        v = case["vocab"]
        w = randn(v, c) * (2.0 / math.sqrt(c))
        # a few labels are frequent, most are rare; a tenth of the pixels has none
        y = (v * torch.rand(n, generator=g, device=dev) ** 3).long().clamp_(0, v - 1)
        if n > 8:
            y[torch.rand(n, generator=g, device=dev) < 0.1] = -1
        st.update(x=x.to(dt), w=w.to(dt), y=y, b=randn(v).to(dt) if case["bias"] else None)
        if case["train"]:
            st["x"].requires_grad_(True)
            st["w"].requires_grad_(True)
            if case["bias"]:
                st["b"].requires_grad_(True)
        return st
    if case["op"] == "norm":
        if case["planes"]:
            x = x.t().contiguous().t()  # (C, pixels) in memory, as the renderer writes it
        st.update(x=x.to(dt).requires_grad_(True), w=(1.0 + 0.2 * randn(c)).requires_grad_(True), b=(0.2 * randn(c)).requires_grad_(True),
                  dy=(randn(n, c) * 1e-2).to(_TYPES[case["out"]]))
        return st
    st["x"] = x.to(dt)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------------
def _run_own(st):
    import retinags_b200 as R
    case = st["case"]
    if case["op"] == "label":
        if not case["train"]:
            return R.label_loss(st["x"], st["w"], st["y"], bias=st["b"], reduction="none")
        loss = R.label_loss(st["x"], st["w"], st["y"], bias=st["b"], reduction="mean")
        leaves = [st["x"], st["w"]] + ([st["b"]] if case["bias"] else [])
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    if case["op"] == "norm":
        y = R.layer_norm(st["x"], st["w"], st["b"], eps=_EPS, out_dtype=_TYPES[case["out"]], keep=case["keep"])
        return [y.detach(), *torch.autograd.grad(y, [st["x"], st["w"], st["b"]], st["dy"])]
    return R.pack8(st["x"]).unpack(torch.float32)


# ---------------------------------------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------------------------------------
def _plain_label(st):
    case = st["case"]
    with torch.no_grad():
        x, w, y = st["x"].detach().float(), st["w"].detach().float(), st["y"]
        b = st["b"].detach().float() if case["bias"] else None
        n, v = x.shape[0], w.shape[0]
        counts = (y >= 0) & (y < v)
        target = torch.where(counts, y, torch.zeros_like(y))
        total = counts.sum().clamp(min=1).float()
        step = max(1, min(n, _CHUNK // v))
        losses = torch.empty(n, device=x.device)
        dx = torch.empty_like(x) if case["train"] else None
        dw = torch.zeros_like(w) if case["train"] else None
        db = torch.zeros(v, device=x.device) if case["train"] and case["bias"] else None
        for r in range(0, n, step):
            rows = slice(r, min(r + step, n))
            s = x[rows] @ w.t()
            if b is not None:
                s += b
            m = s.max(1, keepdim=True).values
            at = s.gather(1, target[rows, None])
            s = (s - m).exp_()
            z = s.sum(1, keepdim=True)
            losses[rows] = torch.where(counts[rows], (z.log() + m - at)[:, 0], torch.zeros_like(z[:, 0]))
            if case["train"]:
                s /= z
                s.scatter_add_(1, target[rows, None], torch.full_like(z, -1.0))
                s *= (counts[rows].float() / total)[:, None]
                dx[rows] = s @ w
                dw += s.t() @ x[rows]
                if db is not None:
                    db += s.sum(0)
        if not case["train"]:
            return losses
        out = [(losses.double().sum() / total).float(), dx.to(st["x"].dtype), dw.to(st["w"].dtype)]
        return out + ([db.to(st["b"].dtype)] if db is not None else [])


def _plain_pack(x):
    """Values that blocks of 32 channels stand for when they share a power of two and have 8 bits each."""
    n, c = x.shape
    blocks = (c + 31) // 32
    p = torch.zeros(n, blocks * 32, device=x.device)
    p[:, :c] = x
    p = p.view(n, blocks, 32)
    most = p.abs().amax(2, keepdim=True)
    mant, expo = torch.frexp(most)  # most = mant * 2^expo, 0.5 <= mant < 1
    e = expo - 7 + (mant > 127.0 / 128.0).to(expo.dtype)  # smallest e with 127 * 2^e >= most
    e = torch.where(most > 0, e, torch.zeros_like(e)).clamp(min=-126)
    e = e.to(torch.int32)
    up, down = ((127 - e) << 23).view(torch.float32), ((127 + e) << 23).view(torch.float32)  # 2^-e and 2^e
    return (torch.round(p * up) * down).view(n, blocks * 32)[:, :c]


def _plain_norm(st):
    case = st["case"]
    with torch.no_grad():
        x, w, b, dy = st["x"].detach().float(), st["w"].detach(), st["b"].detach(), st["dy"].float()

        def normed(t):
            d = t - t.mean(1, keepdim=True)
            rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + _EPS)
            return d * rstd, rstd

        xhat, rstd = normed(x)
        y = (xhat * w + b).to(_TYPES[case["out"]])
        if case["keep"] == "int8":
            xhat, rstd = normed(_plain_pack(x))
        a = dy * w
        dx = rstd * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
        return [y, dx.to(st["x"].dtype), (dy * xhat).sum(0), dy.sum(0)]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "label":
        return _plain_label(state)
    if op == "norm":
        return _plain_norm(state)
    return _plain_pack(state["x"].float())


# ---------------------------------------------------------------------------------------------------------------------
# 64-bit definitions
# ---------------------------------------------------------------------------------------------------------------------
def _exact_label(st):
    case = st["case"]
    x, w, y = st["x"].detach().double(), st["w"].detach().double(), st["y"]
    b = st["b"].detach().double() if case["bias"] else None
    n, v = x.shape[0], w.shape[0]
    ok = torch.logical_and(y >= 0, y < v)
    count = max(int(ok.sum()), 1)
    loss, gx, gw, gb = [], [], torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device=x.device)
    for xs, ys, os in zip(x.split(max(1, (1 << 27) // v)), y.split(max(1, (1 << 27) // v)), ok.split(max(1, (1 << 27) // v))):
        s = torch.matmul(xs, w.t()) if b is None else torch.matmul(xs, w.t()) + b
        logp = s - torch.logsumexp(s, dim=1, keepdim=True)
        idx = ys.clamp(0, v - 1)
        at = torch.arange(xs.shape[0], device=x.device)
        loss.append(torch.where(os, -logp[at, idx], torch.zeros((), dtype=torch.float64, device=x.device)))
        if case["train"]:
            p = logp.exp()
            p[at, idx] -= 1.0
            p = p * (os.double() / count)[:, None]
            gx.append(torch.matmul(p, w))
            gw += torch.matmul(p.t(), xs)
            gb += p.sum(dim=0)
    loss = torch.cat(loss)
    if not case["train"]:
        return loss
    return [loss.sum() / count, torch.cat(gx), gw] + ([gb] if b is not None else [])


def _power(e):
    return ((e + 1023) << 52).view(torch.float64)  # 2^e from its bits


def _exact_pack(x):
    n, c = x.shape
    out = torch.empty(n, c, dtype=torch.float64, device=x.device)
    for lo in range(0, c, 32):
        blk = x[:, lo:lo + 32].double()
        most = blk.abs().max(dim=1, keepdim=True).values
        # smallest power of two whose 127-fold covers the block; log2 decides up to one step, the comparison settles it
        e = torch.ceil(torch.log2(torch.where(most > 0, most, torch.full_like(most, 127.0)) / 127.0)).long()
        e = torch.where(127.0 * _power(e) < most, e + 1, e)
        e = torch.where(127.0 * _power(e - 1) >= most, e - 1, e)
        e = torch.where(most > 0, e, torch.zeros_like(e)).clamp(min=-126)
        step = _power(e)
        out[:, lo:lo + 32] = torch.round(blk / step) * step
    return out


def _exact_norm(st):
    case = st["case"]
    x, w, b, dy = (st[k].detach().double() for k in ("x", "w", "b", "dy"))

    def stats(t):
        var, mu = torch.var_mean(t, dim=1, correction=0, keepdim=True)
        return mu, torch.rsqrt(var + _EPS)

    mu, r = stats(x)
    y = (x - mu) * r * w + b
    if case["keep"] == "int8":
        x = _exact_pack(st["x"].detach())
        mu, r = stats(x)
    c = x.shape[1]
    h = (x - mu) * r
    a = dy * w
    dx = (r / c) * (c * a - a.sum(1, keepdim=True) - h * (a * h).sum(1, keepdim=True))
    return [y, dx, torch.einsum("nc,nc->c", dy, h), dy.sum(0)]


def exact(case, seed):
    with torch.no_grad():
        st = prepare(case, seed)
        if case["op"] == "label":
            return _exact_label(st)
        if case["op"] == "norm":
            return _exact_norm(st)
        return _exact_pack(st["x"])


def work(case):
    n, c = case["rows"], case["channels"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "label":
        v = case["vocab"]
        params = (v * c + (v if case["bias"] else 0)) * size
        if not case["train"]:
            return dict(bytes=n * c * size + params + n * 8 + n * 4, flops=2 * n * c * v)
        return dict(bytes=2 * n * c * size + 2 * params + n * 8 + 4, flops=6 * n * c * v)
    if case["op"] == "norm":
        out = 2 if case["out"] == "bf16" else 4
        kept = size if case["keep"] == "input" else 1
        return dict(bytes=n * c * (size + out + kept + out + size) + 16 * c, flops=16 * n * c)
    return dict(bytes=n * c * (size + 4) + 2 * (n * c + n * ((c + 31) // 32)), flops=3 * n * c)
