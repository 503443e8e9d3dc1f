"""The operators that make the gradient (embedding lookup and its gradient, layer norm forward and backward, the
vocabulary loss) against their formulas in 64 bits.

Tolerances are worst-case rounding bounds: u = 2^-24 is half an fp32 step, a sum of n terms in any order is off by at
most n u times the sum of their magnitudes, and a result rounded to type t adds finfo(t).eps / 2 of its magnitude (and
half the smallest subnormal step, where fp16 underflows)."""
import ctypes
import os
import subprocess
import threading

import pytest
import torch

from omr import Layout, cdist, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
NAN = float("nan")


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == F16 else 2.0 ** -149


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(shape, dtype, g, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=F32, device="cuda").normal_(mean, std, generator=g).to(dtype)


def within(got, ref, tol, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    if bool(bad.any()):
        i = torch.nonzero(bad.flatten())[0].item()
        tol = tol.expand_as(err) if torch.is_tensor(tol) else torch.full_like(err, tol)
        pytest.fail(f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; first at {i}: got "
                    f"{got.flatten()[i].item()!r}, formula {ref.flatten()[i].item()!r}, bound {tol.flatten()[i].item()!r}")


def strided(t, pad, offset=0):
    """The same rows `pad` elements further apart, beginning `offset` elements into the allocation."""
    n, d = t.shape
    buf = torch.full((offset + n * (d + pad),), -77.0, dtype=t.dtype, device=t.device)
    v = buf[offset:].view(n, d + pad)[:, :d]
    v.copy_(t)
    return v, buf


def make_ids(n, rows, g, kind):
    if kind == "one":
        return torch.full((n,), rows - 1, device="cuda")
    if kind == "low":  # a few low ids take most tokens
        return (torch.rand(n, generator=g, device="cuda") ** 6 * rows).long().clamp_(max=rows - 1)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    if kind == "padded":
        ids[torch.rand(n, generator=g, device="cuda") < 0.3] = -1
        ids[torch.rand(n, generator=g, device="cuda") < 0.1] = rows
        ids[torch.rand(n, generator=g, device="cuda") < 0.1] = -(2 ** 31) if n % 2 else 2 ** 31 - 1
    return ids


# ---------------------------------------------------------------------------------------------------- lookup

def embed_ref(table, ids, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    out = torch.zeros(*ids.shape, table.shape[1], dtype=torch.float64, device=ids.device)
    out[ok] = table.double()[ids[ok].long()] * scale
    return out


@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 50, 64), (3, 7, 5), (64, 100, 256), (257, 1000, 1000),
                                        (1000, 333, 515), (2, 3, 20000), (5000, 70, 72)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed(gpu, n, rows, dim, dtype):
    g = gen(n + rows)
    table = rand((rows, dim), dtype, g)
    for kind, it, scale, ot in [("any", torch.int64, 1.0, dtype), ("padded", torch.int32, 5.656854, dtype),
                                ("padded", torch.int64, -0.37, F32), ("any", torch.int32, 1.0, BF16)]:
        ids = make_ids(n, rows, g, kind).to(it)
        got = ops.embed(table, ids, scale=scale, out_dtype=ot)
        scale32 = torch.tensor(scale, dtype=F32).item()
        ref = embed_ref(table, ids.long(), scale32)
        assert got.dtype == ot
        within(got, ref, ref.abs() * (half(ot) + 2 * U) + tiny(ot), (kind, it, ot))


@pytest.mark.parametrize("dim,pad,offset", [(64, 8, 0), (64, 3, 0), (64, 8, 1), (61, 3, 5)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_strides_shape_and_untouched_memory(gpu, dim, pad, offset, dtype):
    g = gen(5)
    table, _ = strided(rand((90, dim), dtype, g), pad, offset)
    ids = make_ids(42, 90, g, "padded").view(6, 7)
    out, buf = strided(torch.zeros(42, dim, dtype=dtype, device="cuda"), pad, offset)
    before = buf.clone()
    assert ops.embed(table, ids, out=out) is out
    within(out, embed_ref(table, ids, 1.0).view(42, dim), 0.0, "strided")
    out.fill_(0)
    assert torch.equal(buf, before)  # nothing between or behind the rows
    assert ops.embed(table, ids).shape == (6, 7, dim)
    one = rand((1, dim), dtype, g).expand(30, dim)  # a broadcast table: rows a stride of 0 apart
    assert torch.equal(ops.embed(one, ids.clamp(0, 29)), one[0].expand(6, 7, dim))


def test_embed_empty_and_far(gpu):
    table = torch.ones(4, 8, device="cuda")
    assert ops.embed(table, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 8)
    with pytest.raises(ValueError, match="out_dtype"):
        ops.embed(table, torch.tensor([1], device="cuda"), out_dtype=torch.int32)
    none = torch.empty(0, 8, device="cuda")
    assert not ops.embed(none, torch.tensor([0, 1], device="cuda")).any()
    # offsets past 2^32 elements: a table of 2^21 + 3 rows of 2050 in bf16 (8 GiB)
    big = torch.empty((1 << 21) + 3, 2050, dtype=BF16, device="cuda")
    ids = torch.tensor([big.shape[0] - 1, 0, 1 << 20], device="cuda")
    for k, i in enumerate(ids.tolist()):
        big[i] = torch.arange(2050, device="cuda") % 200 + k
    assert torch.equal(ops.embed(big, ids), big[ids])


# ---------------------------------------------------------------------------------------------------- its gradient

def embed_grad_ref(grad, ids, rows, scale):
    """The gradient and its bound: (terms + 2) u times the terms' magnitudes (the sums, the scale)."""
    ok = (ids >= 0) & (ids < rows)
    i, g = ids[ok].long(), grad[ok].double() * scale
    ref = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device=grad.device).index_put_((i,), g, accumulate=True)
    mag = torch.zeros_like(ref).index_put_((i,), g.abs(), accumulate=True)
    cnt = torch.bincount(i, minlength=rows).double()[:, None]
    return ref, mag * (cnt + 2) * U, cnt[:, 0] > 0


@pytest.mark.parametrize("n,rows,dim,kind", [
    (0, 5, 8, "any"), (1, 1, 1, "any"), (1, 3000, 64, "any"), (64, 10, 4, "any"), (65, 10, 4, "one"),
    (63, 1, 100, "one"), (4097, 1, 36, "one"), (1000, 17, 129, "padded"), (1000, 17, 1028, "low"),
    (5000, 2000, 515, "low"), (4096, 300, 256, "padded"), (4097, 300, 256, "padded"), (20000, 1025, 96, "low"),
    (3000, 300001, 20, "any"), (300, 2100, 5000, "padded"), (129, 2, 5000, "one"), (70000, 3, 12, "any")])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_grad(gpu, n, rows, dim, kind, dtype):
    g = gen(n + dim)
    grad = rand((n, dim), dtype, g)
    ids = make_ids(n, rows, g, kind)
    bad = (ids < 0) | (ids >= rows)
    grad[bad] = NAN  # a padded token's gradient is not looked at
    plan = ops.EmbedGradPlan(n, rows, dim)
    for it, scale in [(torch.int64, 1.0), (torch.int32, 0.1)]:
        scale32 = torch.tensor(scale, dtype=F32).item()
        ref, tol, named = embed_grad_ref(grad, ids, rows, scale32)
        got = torch.full((rows, dim), NAN, device="cuda")
        plan.run(grad, ids.to(it), got, scale=scale)
        within(got, ref, tol, (it, "write"))
        base = rand((rows, dim), F32, g)
        acc = base.clone()
        plan.run(grad, ids.to(it), acc, scale=scale, accumulate=True)
        within(acc, ref + base.double(), tol + U * (ref + base.double()).abs(), (it, "accumulate"))
        assert torch.equal(acc[~named], base[~named])
        again = torch.empty_like(got)
        plan.run(grad, ids.to(it), again, scale=scale)
        assert torch.equal(got, again)  # the same bits


@pytest.mark.parametrize("dim,pad,offset", [(64, 4, 0), (64, 4, 1), (64, 1, 0), (33, 2, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_grad_strides_and_untouched_memory(gpu, dim, pad, offset, dtype):
    g = gen(9)
    grad, _ = strided(rand((300, dim), dtype, g), pad, offset)
    ids = make_ids(300, 40, g, "low")
    out, buf = strided(torch.zeros(40, dim, device="cuda"), pad, offset)
    before = buf.clone()
    plan = ops.EmbedGradPlan(512, 40, dim)
    plan.run(grad, ids, out)
    ref, tol, _ = embed_grad_ref(grad, ids, 40, 1.0)
    within(out, ref, tol, "strided")
    out.fill_(0)
    assert torch.equal(buf, before)
    one = rand((1, dim), dtype, g).expand(300, dim)  # the gradient of a sum: one row for every token
    ref, tol, _ = embed_grad_ref(one, ids, 40, 1.0)
    within(plan.run(one, ids), ref, tol, "broadcast")


@pytest.mark.parametrize("rows,dim", [((1 << 25) + 5, 3), ((1 << 20) + 1, 4100)])
def test_embed_grad_of_a_large_table(gpu, rows, dim):
    """More rows than a fill workgroup's wave takes one of, and offsets past 2^32 elements."""
    g = gen(9)
    ids = torch.tensor([rows - 1, 0, rows - 1, rows, -1, 1 << 20, 77], device="cuda")
    grad = rand((7, dim), F32, g)
    out = torch.full((rows, dim), 1.0, device="cuda")
    ops.EmbedGradPlan(7, rows, dim).run(grad, ids, out)
    want = {rows - 1: grad[0] + grad[2], 0: grad[1], 77: grad[6]}
    want[1 << 20] = grad[5] if rows - 1 != 1 << 20 else grad[0] + grad[2] + grad[5]
    want[rows - 1] = want[1 << 20] if rows - 1 == 1 << 20 else want[rows - 1]
    for r, v in want.items():
        assert torch.equal(out[r], v)
        out[r] = 0
    step = (1 << 28) // dim
    assert not any(out[i:i + step].any() for i in range(0, rows, step))


def test_embed_grad_is_the_lookups(gpu):
    """<grad(dy), E> = <dy, embed(E)> for any E: the backward is the forward's transpose (in 64 bits of its outputs)."""
    g = gen(3)
    table, dy = rand((500, 48), F32, g), rand((2000, 48), F32, g)
    ids = make_ids(2000, 500, g, "padded")
    a = (ops.EmbedGradPlan(2000, 500, 48).run(dy, ids, scale=3.0).double() * table.double()).sum().item()
    b = (ops.embed(table, ids, scale=3.0).double() * dy.double()).sum().item()
    # each output is off by at most (64 + 2) u of its terms (no row has 64 tokens' worth of more), the rest is exact
    mag = (embed_ref(table, ids, 3.0).abs() * dy.double().abs()).sum().item()
    assert torch.bincount(ids[(ids >= 0) & (ids < 500)]).max().item() <= 64
    assert abs(a - b) <= 70 * U * mag


# ---------------------------------------------------------------------------------------------------- layer norm

def depth(dim):
    """Additions behind each other in a row's sum: a lane's, the wave's six, the waves'."""
    return (16 if dim <= 16384 else dim // 1024 + 1) + 6 + 16


def norm_ref(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    w = torch.ones(x.shape[-1], device=x.device) if w is None else w
    b = torch.zeros(x.shape[-1], device=x.device) if b is None else b
    y = xh * w.double() + b.double()
    # the mean is off by m = k u mean|x|; the squared distances by k + 4 roundings of u and m^2; half of that in rstd,
    # with the root, the quotient and the two products behind it
    k = depth(x.shape[-1]) + 2
    m = k * U * x.abs().mean(-1, keepdim=True)
    rel = ((k + 4) * U + m * m / (var + eps)) / 2 + 6 * U
    tol_y = w.double().abs() * (xh.abs() * rel + m * rstd * (1 + rel)) + 2 * U * (y.abs() + b.double().abs())
    return y, mean[..., 0], rstd[..., 0], tol_y, m[..., 0], (rel * rstd)[..., 0]


SHAPES = [(1, 1), (1, 8), (5, 3), (3, 64), (7, 1000), (9, 1024), (2, 1025), (5, 2048), (4, 2056), (3, 4096), (2, 5003),
          (3, 8192), (2, 16384), (2, 16385), (1, 40000), (2100, 72), (2500, 1032)]


@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype,pdt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_layer_norm(gpu, rows, dim, dtype, pdt):
    g = gen(rows + dim)
    x = rand((rows, dim), dtype, g, std=2.0, mean=30.0)
    w, b = rand((dim,), pdt, g, mean=1.0), rand((dim,), pdt, g)
    for weight, bias in [(w, b), (None, None), (w, None)]:
        r = ops.layer_norm(x, weight, bias, eps=1e-5)
        y, mean, rstd, tol_y, tol_m, tol_r = norm_ref(x, weight, bias, torch.tensor(1e-5, dtype=F32).item())
        within(r.mean, mean, tol_m + U * mean.abs(), "mean")
        within(r.rstd, rstd, tol_r, "rstd")
        within(r.out, y, tol_y * (1 + half(dtype)) + half(dtype) * y.abs() + tiny(dtype), "out")


@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype,pdt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_layer_norm_grad(gpu, rows, dim, dtype, pdt):
    g = gen(rows * 3 + dim)
    x, dy = rand((rows, dim), dtype, g, std=2.0, mean=1.0), rand((rows, dim), dtype, g)
    w = rand((dim,), pdt, g, mean=1.0)
    plan = ops.LayerNormGradPlan(rows + 3, dim)
    for weight in (w, None):
        f = ops.layer_norm(x, weight)
        r = plan.run(dy, x, f.mean, f.rstd, weight)
        xh = (x.double() - f.mean.double()[:, None]) * f.rstd.double()[:, None]
        d = dy.double()
        gw = d * (weight.double() if weight is not None else 1.0)
        s1, s2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
        rs = f.rstd.double()[:, None]
        dx = (gw - s1 - xh * s2) * rs
        k = depth(dim)
        tol = rs * U * (4 * gw.abs() + (k + 6) * gw.abs().mean(1, keepdim=True) +
                        (k + 10) * xh.abs() * (gw * xh).abs().mean(1, keepdim=True)) + 2 * U * dx.abs()
        within(r.grad_x, dx, tol * (1 + half(dtype)) + half(dtype) * dx.abs() + tiny(dtype), "grad_x")
        tol_w, tol_b = (rows + 4) * U * (d * xh).abs().sum(0), rows * U * d.abs().sum(0)
        within(r.grad_weight, (d * xh).sum(0), tol_w, "grad_weight")
        within(r.grad_bias, d.sum(0), tol_b, "grad_bias")
        gw0, gb0 = rand((dim,), F32, g), rand((dim,), F32, g)
        gw1, gb1 = gw0.clone(), gb0.clone()
        r2 = plan.run(dy, x, f.mean, f.rstd, weight, grad_weight=gw1, grad_bias=gb1, accumulate=True)
        assert torch.equal(r2.grad_x, r.grad_x)  # the same bits
        assert torch.equal(gw1, gw0 + r.grad_weight) and torch.equal(gb1, gb0 + r.grad_bias)
        alone = plan.run(dy, x, f.mean, f.rstd, weight, params=False)
        assert alone.grad_weight is None and torch.equal(alone.grad_x, r.grad_x)
        onto = dy.clone()
        assert torch.equal(plan.run(onto, x, f.mean, f.rstd, weight, grad_x=onto).grad_weight, r.grad_weight)
        assert torch.equal(onto, r.grad_x)


def test_layer_norm_grad_is_the_slope(gpu):
    """Directional differences of the forward's formula in 64 bits against the gradient (fp32 inputs)."""
    g = gen(8)
    x, dy, w, b = rand((6, 200), F32, g), rand((6, 200), F32, g), rand((200,), F32, g, mean=1.0), rand((200,), F32, g)
    f = ops.layer_norm(x, w, b)
    r = ops.LayerNormGradPlan(6, 200).run(dy, x, f.mean, f.rstd, w)

    def loss(x, w, b):
        return (norm_ref(x, w, b, 1e-5)[0] * dy.double()).sum().item()
    h = 1e-4
    for t, grad in ((0, r.grad_x), (1, r.grad_weight), (2, r.grad_bias)):
        args = [x.double(), w.double(), b.double()]
        v = torch.empty_like(args[t]).normal_(generator=g)
        up, dn = list(args), list(args)
        up[t], dn[t] = args[t] + h * v, args[t] - h * v
        slope = (loss(*up) - loss(*dn)) / (2 * h)
        got = (grad.double() * v).sum().item()
        # central differences: h^2 of third derivatives (of order 10 here) and fp32 bounds of the 1200 products
        assert abs(slope - got) <= 1e-5 * (grad.double() * v).abs().sum().item() + 1e-5


@pytest.mark.parametrize("dim,pad,offset", [(256, 8, 0), (256, 1, 0), (256, 8, 3), (77, 2, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_strides_and_untouched_memory(gpu, dim, pad, offset, dtype):
    g = gen(2)
    x0, dy0 = rand((37, dim), dtype, g), rand((37, dim), dtype, g)
    w, b = rand((dim,), F32, g), rand((dim,), F32, g)
    x, _ = strided(x0, pad, offset)
    dy, _ = strided(dy0, pad, offset)
    out, buf = strided(torch.zeros_like(x0), pad, offset)
    before = buf.clone()
    f, plain = ops.layer_norm(x, w, b, out=out), ops.layer_norm(x0, w, b)
    y, _, _, tol, _, _ = norm_ref(x0, w, b, torch.tensor(1e-5, dtype=F32).item())
    within(out, y, tol * (1 + half(dtype)) + half(dtype) * y.abs() + tiny(dtype), "strided")
    gx, gbuf = strided(torch.zeros_like(x0), pad, offset)
    plan = ops.LayerNormGradPlan(37, dim)
    r = plan.run(dy, x, plain.mean, plain.rstd, w, grad_x=gx)
    q = plan.run(dy0, x0, plain.mean, plain.rstd, w)
    # a lane's columns depend on the piece width, so sums differ in order: bounds as above on both sides
    k = depth(dim)
    for a, c in ((r.grad_x, q.grad_x), (r.grad_weight, q.grad_weight), (r.grad_bias, q.grad_bias)):
        scale = c.double().abs().max().item() + 1
        within(a, c.double(), (2 * (k + 60) * U * 20 + 2 * half(a.dtype)) * scale, "strided gradient")
    for t, bb in ((out, buf), (gx, gbuf)):
        t.fill_(0)
        assert torch.equal(bb, before)
    inplace = x0.clone()
    assert torch.equal(ops.layer_norm(inplace, w, b, out=inplace).out, plain.out)


def test_layer_norm_no_rows_and_shapes(gpu):
    x = torch.empty(0, 96, device="cuda")
    f = ops.layer_norm(x)
    assert f.out.shape == (0, 96) and f.mean.shape == (0,)
    plan = ops.LayerNormGradPlan(4, 96)
    r = plan.run(x, x, f.mean, f.rstd)
    assert not r.grad_weight.any() and not r.grad_bias.any()
    keep = torch.ones(96, device="cuda")
    plan.run(x, x, f.mean, f.rstd, grad_weight=keep, grad_bias=keep.clone(), accumulate=True)
    assert torch.equal(keep, torch.ones(96, device="cuda"))
    y = ops.layer_norm(torch.randn(2, 3, 96, device="cuda"))
    assert y.out.shape == (2, 3, 96) and y.mean.shape == (2, 3)
    inf = torch.randn(3, 96, device="cuda")
    inf[1, 5] = float("inf")
    out = ops.layer_norm(inf).out
    assert not torch.isfinite(out[1]).any() and torch.isfinite(out[[0, 2]]).all()


# ---------------------------------------------------------------------------------------------------- vocabulary loss

def loss_inputs(T, V, D, dtype, g, none=0.1):
    """Hidden states that lean towards their target's row; tokens without a target hold NaN."""
    w = rand((V, D), dtype, g, std=D ** -0.5)
    t = torch.randint(0, V, (T,), generator=g, device="cuda")
    h = (rand((T, D), F32, g) + 4 * torch.rand(T, 1, generator=g, device="cuda") * w[t].float()).to(dtype)
    off = torch.rand(T, generator=g, device="cuda") < none
    t[off] = torch.where(torch.rand(T, generator=g, device="cuda") < 0.5, -100, V)[off]
    return h, w, t, off


def loss_ref(h, w, t, off):
    """Logits, lse and loss in 64 bits, with the bounds: a logit's dim products are exact in fp32 and their sum is off by
    dim u of their magnitudes (e); the exponentials' arguments by that and u, __expf by 2 u (|argument| + 2), so the sum
    by e + (100 + vocab depth) u, and as much the lse."""
    z = h.double() @ w.double().t()
    e = (h.double().abs() @ w.double().abs().t()).amax(1) * h.shape[1] * U
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, t.clamp(0, w.shape[0] - 1).long()[:, None])[:, 0]
    loss = torch.where(off, 0.0, lse - zt)
    spread = (z.amax(1) - lse).abs() + 40  # arguments below -40 do not count at this precision
    tol = e + (2 * spread + 600) * U + 2 * U * lse.abs()
    return z, lse, loss, tol


LOSS_SIZES = [(1, 1, 8), (1, 7, 1), (3, 300, 72), (16, 70, 2120), (17, 129, 264), (32, 200, 1000), (33, 200, 64), (64, 1000, 128), (130, 257, 61), (257, 2000, 200),
              (300, 5003, 520), (1025, 700, 96), (16, 40000, 64), (700, 70000, 64), (2048, 8192, 256), (5, 256, 4096),
              (5000, 300, 40), (600, 4100, 136), (900, 4100, 200), (1500, 5000, 400)]


@pytest.mark.parametrize("T,V,D", LOSS_SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_vocab_loss(gpu, T, V, D, dtype):
    g = gen(T + V + D)
    h, w, t, off = loss_inputs(T, V, D, dtype, g)
    plan = ops.VocabLossPlan(T + 5, V, D, dtype=dtype)
    fwd = ops.VocabLossPlan(T, V, D, dtype=dtype, grads=False)
    z, lse, loss, tol = loss_ref(h, w, t, off)
    for p, it in ((plan, torch.int64), (fwd, torch.int32)):
        got, got_lse = p.forward(h, w, t.to(it))
        within(got_lse, lse, tol, "lse")
        within(got, loss, torch.where(off, 0.0, 2 * tol + U * loss.abs()), "loss")

    # the gradient of sum(up * loss), with tokens of no target holding NaN everywhere
    for up in (torch.full((T,), 1.0 / max(1, T), device="cuda"), rand((T,), F32, g)):
        hn, upn = h.clone(), up.clone()
        hn[off], upn[off] = NAN, NAN
        _, l32 = plan.forward(h, w, t)
        ll = l32.clone()
        ll[off] = NAN
        G = torch.exp(z - l32.double()[:, None])
        G[torch.arange(T, device="cuda")[~off], t[~off]] -= 1
        G[off] = 0
        upd = torch.where(off, 0.0, up.double())
        gh_ref = upd[:, None] * (G @ w.double())
        gw_ref = (G * upd[:, None]).t() @ torch.where(off[:, None], 0.0, h.double())
        # G: a logit is off by e, the exponential by 2 u (|argument| + 2), then rounded to the type (its magnitude, and
        # fp16's underflow at 2^-25 / 2^12); hidden times its share of the largest factor rounds once more; sums of V
        # (T) terms in fp32
        e = ((h.double().abs() @ w.double().abs().t()).amax(1) * D * U)[:, None] + 100 * U
        P = torch.exp(z - l32.double()[:, None])
        dG = torch.where(off[:, None], 0.0, P * 2 * e + G.abs() * half(dtype) + 2.0 ** -36)
        tol_h = upd.abs()[:, None] * (dG @ w.double().abs() + (V + 4) * U * (G.abs() @ w.double().abs()))
        hm = torch.where(off[:, None], 0.0, h.double().abs())
        wt = (upd.abs()[:, None] * (dG + G.abs() * ((T + 4) * U + half(dtype)))).t() @ hm
        wt = wt + T * tiny(dtype) * upd.abs().max()
        gh, gw = plan.backward(hn, w, t, ll, upn)
        within(gh, gh_ref, tol_h * (1 + half(dtype)) + half(dtype) * gh_ref.abs() + tiny(dtype), "grad_hidden")
        within(gw, gw_ref, wt * (1 + half(dtype)) + half(dtype) * gw_ref.abs() + tiny(dtype), "grad_weight")
        assert not gh[off].any()
        base = rand((V, D), F32, g)
        acc = base.clone()
        none, gw32 = plan.backward(hn, w, t, ll, upn, grad_weight=acc, accumulate=True, need_hidden=False)
        assert none is None and gw32 is acc
        within(acc, gw_ref + base.double(), wt + 2 * U * (gw_ref.abs() + base.double().abs()), "accumulated")
        gh2, none = plan.backward(hn, w, t, ll, upn, need_weight=False)
        assert none is None and torch.equal(gh2, gh)
        again = plan.backward(hn, w, t, ll, upn)
        assert torch.equal(again[0], gh) and torch.equal(again[1], gw)  # the same bits


@pytest.mark.parametrize("T,V,D", [(5, 300, 64), (150, 700, 200)])
def test_vocab_loss_grad_is_the_slope(gpu, T, V, D):
    """The forward's own differences against the gradient: for two points of the type a and b, loss(b) - loss(a) is the
    mean of both ends' gradients along b - a, but for a third derivative.  Along a line of logits z + s dz that of
    log sum exp is a third central moment of dz under the softmax: at most R^3 / (6 sqrt 3) for values in a range of R;
    the trapezoid is off by a twelfth of it."""
    g = gen(T)
    h, w, t, off = loss_inputs(T, V, D, BF16, g, none=0.0)
    plan = ops.VocabLossPlan(T, V, D)
    one = torch.ones(T, device="cuda")
    h2 = (h.float() + 0.05 * rand((T, D), F32, g)).to(BF16)
    w2 = (w.float() + 0.05 * D ** -0.5 * rand((V, D), F32, g)).to(BF16)
    tols = [loss_ref(a, b, t, off)[3].sum() for a, b in ((h, w), (h2, w), (h, w2))]
    la, lse_a = plan.forward(h, w, t)
    for which, (hb, wb) in enumerate(((h2, w), (h, w2))):
        lb, lse_b = plan.forward(hb, wb, t)
        ga = plan.backward(h, w, t, lse_a, one, grad_weight=torch.empty(V, D, device="cuda"))[which].double()
        gb = plan.backward(hb, wb, t, lse_b, one, grad_weight=torch.empty(V, D, device="cuda"))[which].double()
        d = (hb.double() - h.double()) if which == 0 else (wb.double() - w.double())
        along = ((ga + gb) / 2 * d).sum()
        dz = (d @ w.double().t()) if which == 0 else h.double() @ d.t()
        R = dz.amax(1) - dz.amin(1)
        # the gradients' own error: every entry of G rounded to bf16 (sum |G| <= 2 a token), and grad_hidden's rounding
        most = dz.abs().amax(1)
        err = (2 * most * (half(BF16) * 1.1 + (V + T + 8) * U)).sum() + (half(BF16) * ((ga.abs() + gb.abs()) / 2 * d.abs()).sum())
        tol = (R ** 3).sum() / (12 * 6 * 3 ** 0.5) + err + tols[0] + tols[1 + which]
        diff = (lb.double() - la.double()).sum()
        assert (diff - along).abs() <= tol, (which, diff.item(), along.item(), tol.item())
        assert tol < 0.2 * d.norm() * ga.norm()  # (the bound says something)


def test_vocab_loss_grad_of_no_tokens_and_a_large_weight(gpu):
    """Zeros into more than 2^32 elements."""
    plan = ops.VocabLossPlan(0, 65537, 65536)
    out = torch.ones(65537, 65536, dtype=BF16, device="cuda")
    plan.backward(out[:0], out, torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda"),
                  torch.empty(0, device="cuda"), grad_weight=out)
    assert not any(out[i:i + 8192].any() for i in range(0, 65537, 8192))


def test_vocab_loss_no_targets_no_tokens_and_one_factor(gpu):
    g = gen(1)
    h, w, t, off = loss_inputs(40, 500, 64, BF16, g, none=0.0)
    plan = ops.VocabLossPlan(40, 500, 64)
    nothing = torch.full_like(t, -1)
    loss, lse = plan.forward(h, w, nothing)
    assert not loss.any() and torch.isfinite(lse).all()
    gh, gw = plan.backward(h, w, nothing, lse, torch.ones(40, device="cuda"))
    assert not gh.any() and not gw.any()
    keep = torch.ones(500, 64, device="cuda")
    plan.backward(h, w, nothing, lse, torch.ones(40, device="cuda"), grad_weight=keep, accumulate=True)
    assert (keep == 1).all()
    empty = plan.forward(h[:0], w, t[:0])
    assert empty[0].shape == (0,)
    for dt in (BF16, F32):
        out = torch.full((500, 64), NAN, dtype=dt, device="cuda")
        plan.backward(h[:0], w, t[:0], empty[1], torch.empty(0, device="cuda"), grad_weight=out)
        assert not out.any()
    loss, lse = plan.forward(h, w, t)
    one = torch.tensor(0.25, device="cuda")
    a = plan.backward(h, w, t, lse, one)
    b = plan.backward(h, w, t, lse, one.expand(40))
    c = plan.backward(h, w, t, lse, torch.full((40,), 0.25, device="cuda"))
    for x, y, q in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, q)
    zero = plan.backward(h, w, t, lse, torch.zeros(40, device="cuda"))
    assert not zero[0].any() and not zero[1].any()


@pytest.mark.parametrize("D,pad,offset", [(64, 8, 0), (64, 3, 0), (64, 8, 1), (61, 3, 5)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_vocab_loss_strides_and_untouched_memory(gpu, D, pad, offset, dtype):
    """Rows apart, unaligned and ragged: the same bits as the packed tensors' (the products see the same tiles)."""
    g = gen(6)
    T, V = 150, 400
    h0, w0, t, off = loss_inputs(T, V, D, dtype, g)
    up = rand((T,), F32, g)
    h, _ = strided(h0, pad, offset)
    w, _ = strided(w0, pad, offset)
    plain, plan = ops.VocabLossPlan(T, V, D, dtype=dtype), ops.VocabLossPlan(T, V, D, dtype=dtype, pack=True)
    want = [*plain.forward(h0, w0, t)]
    want += plain.backward(h0, w0, t, want[1], up)
    gh, hbuf = strided(torch.zeros_like(h0), pad, offset)
    gw, wbuf = strided(torch.zeros_like(w0), pad, offset)
    before = hbuf.clone(), wbuf.clone()
    got = [*plan.forward(h, w, t)]
    got += plan.backward(h, w, t, got[1], up, grad_hidden=gh, grad_weight=gw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    gh.fill_(0)
    gw.fill_(0)
    assert torch.equal(hbuf, before[0]) and torch.equal(wbuf, before[1])
    if (D + pad) % 8 or offset:
        if D % 8 == 0:
            with pytest.raises(ops._lib.OmrError, match="pack"):  # (too little room for that without asking)
                ops.VocabLossPlan(T, V, D, dtype=dtype, grads=False).forward(h, w, t)


@pytest.mark.parametrize("T,V,D", [(4100, 70001, 32), (32768, 5000, 136)])
def test_vocab_loss_pieces(gpu, T, V, D, dtype=BF16):
    """More logits than one piece holds (tokens x vocabulary x 2 bytes over 256 MiB): pieces, the last ragged."""
    g = gen(12)
    h, w, t, off = loss_inputs(T, V, D, dtype, g)
    plan = ops.VocabLossPlan(T, V, D)
    loss, lse = plan.forward(h, w, t)
    up = rand((T,), F32, g)
    gh, gw = plan.backward(h, w, t, lse, up, grad_weight=torch.empty(V, D, device="cuda"))
    z = (h.float() @ w.float().t()).double()
    G = torch.exp(z - lse.double()[:, None])
    ok = ~off
    G[torch.arange(T, device="cuda")[ok], t[ok]] -= 1
    G[off] = 0
    upd = torch.where(off, 0.0, up.double())
    gh_ref, gw_ref = upd[:, None] * (G @ w.double()), (G * upd[:, None]).t() @ h.double()
    aG = G.abs()
    th = upd.abs()[:, None] * (aG @ w.double().abs()) * (half(dtype) * 1.1 + (V + 4) * U) + 1e-6
    tw = ((aG * upd.abs()[:, None]).t() @ h.double().abs()) * (2 * half(dtype) * 1.1 + (T + 4) * U) + 1e-6
    within(gh, gh_ref, th + half(dtype) * gh_ref.abs(), "grad_hidden")
    within(gw, gw_ref, tw, "grad_weight")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_vocab_loss_adds_to_a_gradient_of_its_type(gpu, dtype):
    """What is there is added in fp32, in front of the one rounding: the fp32 gradient's sum with it, rounded."""
    g = gen(31)
    for T, V, D in ((60, 300, 72), (700, 2100, 136)):
        h, w, t, off = loss_inputs(T, V, D, dtype, g)
        plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
        _, lse = plan.forward(h, w, t)
        up = rand((T,), F32, g)
        fine = plan.backward(h, w, t, lse, up, grad_weight=torch.empty(V, D, device="cuda"), need_hidden=False)[1]
        base = rand((V, D), dtype, g)
        got = base.clone()
        plan.backward(h, w, t, lse, up, grad_weight=got, accumulate=True, need_hidden=False)
        assert torch.equal(got, (base.float() + fine).to(dtype))


def test_optional_parameters_and_expanded_inputs(gpu):
    g = gen(32)
    x, dy, w, b = rand((37, 264), F32, g), rand((37, 264), F32, g), rand((264,), F32, g), rand((264,), F32, g)
    ones, zeros = torch.ones(264, device="cuda"), torch.zeros(264, device="cuda")
    for weight, bias in ((None, None), (w, None), (None, b)):
        f = ops.layer_norm(x, weight, bias)
        assert torch.equal(f.out, ops.layer_norm(x, ones if weight is None else w, zeros if bias is None else b).out)
    plan = ops.LayerNormGradPlan(37, 264)
    full = plan.run(dy, x, f.mean, f.rstd, w)
    assert torch.equal(plan.run(dy, x, f.mean, f.rstd).grad_x, plan.run(dy, x, f.mean, f.rstd, ones).grad_x)
    for k in ("grad_weight", "grad_bias"):  # one alone, added to
        base = rand((264,), F32, g)
        r = plan.run(dy, x, f.mean, f.rstd, w, accumulate=True, **{k: base.clone()})
        assert torch.equal(getattr(r, k), base + getattr(full, k)) and torch.equal(r.grad_x, full.grad_x)
        assert getattr(r, {"grad_weight": "grad_bias", "grad_bias": "grad_weight"}[k]) is None
    one = dy[:1].expand(37, 264)  # a row for all: a stride of 0
    r, q = (plan.run(d, x, f.mean, f.rstd, w) for d in (one, one.contiguous()))
    assert torch.equal(r.grad_x, q.grad_x) and torch.equal(r.grad_weight, q.grad_weight)
    ids = make_ids(37, 11, g, "any")
    e = ops.EmbedGradPlan(37, 11, 264)
    assert torch.equal(e.run(one, ids), e.run(one.contiguous(), ids))
    table = dy[:1].expand(11, 264)
    assert torch.equal(ops.embed(table, ids), ops.embed(table.contiguous(), ids))
    loss = ops.VocabLossPlan(37, 11, 264, pack=True)
    t = torch.randint(0, 11, (37,), generator=g, device="cuda")
    hb, wb = one.to(BF16)[:1].expand(37, 264), rand((11, 264), BF16, g)
    (la, ea), (lb, eb) = loss.forward(hb, wb, t), loss.forward(hb.contiguous(), wb, t)
    assert torch.equal(la, lb) and torch.equal(ea, eb)


# ---------------------------------------------------------------------------------------------------- streams, graphs

def test_operators_in_a_graph_and_on_streams(gpu):
    """A captured lookup -> norm -> norm gradient -> table gradient, replayed on new inputs with eager work between the
    replays, gives the eager bits each time; and two streams with a plan each do not disturb each other."""
    g = gen(4)
    T, V, D = 700, 500, 264
    table, w, b = rand((V, D), BF16, g), rand((D,), F32, g), rand((D,), F32, g)
    ids = make_ids(T, V, g, "low")
    dy = rand((T, D), BF16, g)

    class Step:
        def __init__(self):
            self.ng, self.eg = ops.LayerNormGradPlan(T, D), ops.EmbedGradPlan(T, V, D)
            self.x = torch.empty(T, D, dtype=BF16, device="cuda")
            self.y, self.gx = torch.empty_like(self.x), torch.empty_like(self.x)
            self.mean, self.rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
            self.flat = torch.empty(V * D + 2 * D, device="cuda")  # one flat gradient: table, weight, bias

        def run(self, stream=None):
            ops.embed(table, ids, scale=2.0, out=self.x, stream=stream)
            f = ops.layer_norm(self.x, w, b, out=self.y, mean=self.mean, rstd=self.rstd, stream=stream)
            gw, gb = self.flat[V * D:V * D + D], self.flat[V * D + D:]
            self.ng.run(dy, self.x, f.mean, f.rstd, w, grad_x=self.gx, grad_weight=gw, grad_bias=gb, stream=stream)
            self.eg.run(self.gx, ids, self.flat[:V * D].view(V, D), scale=2.0, stream=stream)

        def outputs(self):
            return [t.clone() for t in (self.x, self.y, self.gx, self.flat)]

    eager, captured = Step(), Step()
    captured.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.run()
    for k in range(4):
        ids.copy_(make_ids(T, V, gen(100 + k), ["low", "padded", "one", "any"][k]))
        dy.copy_(rand((T, D), BF16, gen(200 + k)))
        eager.run()
        want = eager.outputs()
        captured.flat.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, captured.outputs())), k
    other = Step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, step in zip(streams, (captured, other)):
            step.run(stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, captured.outputs()))
    assert all(torch.equal(p, q) for p, q in zip(want, other.outputs()))


# ---------------------------------------------------------------------------------------------------- a training step

class Model:
    """A small language model whose output layer is its embedding table: lookup, layer norm, loss, and back into one
    flat fp32 gradient [table | norm weight | norm bias | padding to the layout]."""

    def __init__(self, V, D, T, L, dtype=BF16, seed=0):
        g = gen(seed)
        self.V, self.D, self.T, self.dtype = V, D, T, dtype
        self.table = rand((V, D), dtype, g, std=0.05)
        self.weight, self.bias = rand((D,), F32, g, std=0.1, mean=1.0), rand((D,), F32, g, std=0.1)
        self.scale = D ** 0.5
        self.loss_plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
        self.norm_plan, self.embed_plan = ops.LayerNormGradPlan(T, D), ops.EmbedGradPlan(T, V, D)
        self.flat = torch.zeros(L.n, device="cuda")
        n = V * D
        self.g_table, self.g_weight, self.g_bias = self.flat[:n].view(V, D), self.flat[n:n + D], self.flat[n + D:n + 2 * D]

    def step(self, ids, targets, factor):
        """The losses; the gradient of factor * (their sum) is in `flat`."""
        h = ops.embed(self.table, ids, scale=self.scale)
        f = ops.layer_norm(h, self.weight, self.bias)
        loss, lse = self.loss_plan.forward(f.out, self.table, targets)
        gy, _ = self.loss_plan.backward(f.out, self.table, targets, lse, factor, grad_weight=self.g_table)
        r = self.norm_plan.run(gy, h, f.mean, f.rstd, self.weight, grad_weight=self.g_weight, grad_bias=self.g_bias)
        self.embed_plan.run(r.grad_x, ids, self.g_table, scale=self.scale, accumulate=True)
        return loss

    def reference(self, ids, targets, factor):
        """The same step by differentiation in 64 bits."""
        E = self.table.double().requires_grad_()
        w, b = self.weight.double().requires_grad_(), self.bias.double().requires_grad_()
        ok = (ids >= 0) & (ids < self.V)
        h = torch.where(ok[:, None], E[ids.clamp(0, self.V - 1)] * self.scale, 0.0)
        y = torch.nn.functional.layer_norm(h, (self.D,), w, b, 1e-5)
        loss = torch.nn.functional.cross_entropy(y @ E.t(), targets, ignore_index=-100, reduction="none")
        (loss.sum() * factor).backward()
        return loss.detach(), E.grad, w.grad, b.grad


def tokens(T, V, g):
    ids = make_ids(T, V, g, "low")
    ids[::17] = -1
    targets = torch.roll(ids, -1)
    targets[targets < 0] = -100
    targets[-1] = -100
    return ids, targets


@pytest.mark.parametrize("V,D,T", [(1000, 128, 300), (777, 200, 129)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_training_step(gpu, V, D, T, dtype):
    """All operators together against differentiation in 64 bits.  The activations are rounded to the type at four places
    (the lookup, the norm and the two gradients that pass back), each off by half a step of its magnitude; where such an
    error enters the softmax or the norm it passes on with a factor of the order of one (logits of order one).  So each
    gradient is within ten such errors of its norm."""
    L = Layout(n=8 * 16384 * -(-(V * D + 2 * D) // (8 * 16384)))
    m = Model(V, D, T, L, dtype)
    ids, targets = tokens(T, V, gen(1))
    factor = torch.tensor(1.0 / T, device="cuda")
    loss = m.step(ids, targets, factor)
    want = m.reference(ids, targets, 1.0 / T)
    for got, ref, what in zip((loss, m.g_table, m.g_weight, m.g_bias), want, ("loss", "table", "weight", "bias")):
        off = (got.double() - ref).norm().item() / ref.norm().item()
        assert off <= 10 * half(dtype), (what, off)
    assert not m.flat[V * D + 2 * D:].any()
    again = m.flat.clone()
    assert torch.equal(m.step(ids, targets, factor), loss) and torch.equal(m.flat, again)


@pytest.mark.parametrize("world", [2, 3])
def test_step_gradients_summed_by_the_round(gpu, world):
    """Each worker's step gradient through the sparse all-reduce: every worker holds the rank-order sum, bit for bit."""
    V, D, T = 1000, 128, 200
    L = Layout(n=8 * 16384 * 2)
    models = [Model(V, D, T, L) for _ in range(world)]
    for w, m in enumerate(models):
        ids, targets = tokens(T, V, gen(50 + w))
        m.step(ids, targets, torch.tensor(1.0 / T, device="cuda"))
    want = torch.zeros_like(models[0].flat)
    for m in models:
        want = want + m.flat
    torch.cuda.synchronize()
    D_ = cdist.load()
    board = D_.omr_local_board_create(world)
    errs = []

    def rank(r):
        try:
            torch.cuda.set_device(0)
            d, plan = ctypes.c_void_p(), ctypes.c_void_p()
            assert D_.omr_dist_create_local(board, r, ctypes.byref(d)) == 0
            assert D_.omr_ar_plan_create(d, L.n, L.block_size, L.num_lanes, L.num_threads, ctypes.byref(plan)) == 0
            st = torch.cuda.Stream()
            x = models[r].flat
            rc = D_.omr_sparse_round_f32(plan, x.data_ptr(), x.data_ptr(), None, None, None, 0, None, None, st.cuda_stream)
            assert rc == 0, D_.omr_dist_last_error()
            st.synchronize()
            D_.omr_ar_plan_destroy(plan)
            D_.omr_dist_destroy(d)
        except BaseException as e:  # noqa: BLE001
            errs.append(f"rank {r}: {e!r}")

    th = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
    for t in th:
        t.start()
    for t in th:
        t.join(timeout=100)
    assert not any(t.is_alive() for t in th) and not errs, errs
    D_.omr_local_board_destroy(board)
    for m in models:
        assert torch.equal(m.flat, want)


def test_step_in_a_graph(gpu):
    """The whole step captured: every replay, with eager steps of another model between, gives the eager bits."""
    V, D, T = 640, 96, 150
    L = Layout(n=8 * 16384)
    eager, captured = Model(V, D, T, L), Model(V, D, T, L)
    factor = torch.tensor(1.0 / T, device="cuda")
    ids, targets = tokens(T, V, gen(0))
    captured.step(ids, targets, factor)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = captured.step(ids, targets, factor)
    for k in range(4):
        i, t = tokens(T, V, gen(10 + k))
        ids.copy_(i)
        targets.copy_(t)
        want = eager.step(ids, targets, factor)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(captured.flat, eager.flat), k


@pytest.mark.parametrize("args", [["-L", "1"], ["-L", "3"], ["-L", "2", "-I"], ["-L", "2", "-H"], ["-L", "2", "-M"]])
def test_client_embedding_gradient(gpu, args):
    """./omr_client -E: the workers' tensors are embedding gradients of a training step, and -c checks their sum."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omnireduce-rdma-demo_amd", "bin",
                       "omr_client")
    p = subprocess.run([exe, *args, "-n", str(1 << 20), "-E", "256:500", "-W", "1", "-R", "3", "-c"], capture_output=True,
                       text=True, timeout=100)
    out = p.stdout + p.stderr
    assert p.returncode == 0 and "check OK" in out and "embedding gradient: 4096 rows of 256, 500 tokens" in out, out
