"""Where 16-bit storage or a large mean could cost the operators more than their outputs' own rounding: what is held of the
loss's gradient for the targets, tokens of very unequal factors, rows far from zero, and the largest tiles.

Tolerances are worst-case rounding bounds, as in test_accuracy_operators.py."""
import pytest
import torch

from omr import ops
from test_accuracy_operators import BF16, F16, F32, TYPES, U, depth, gen, half, loss_inputs, rand, tiny, within

pytestmark = pytest.mark.gpu


def check_gradients(plan, h, w, t, up, dtype, grad_weight):
    """The backward pass against 64 bits.  G of a token's target has no rounding to 16 bits: what that loses is added to
    grad_hidden in fp32, and to grad_weight as one more 16-bit value (half a step of half a step).  The other entries have
    one, or what fp16 loses of them below its range (2^-25 / 2^12; no more than the entry itself).  Hidden states times
    their share of the largest factor are rounded once, and not at all where all factors are equal; their smallest step in
    fp16 is that of a row whose largest product is stored as 2^13 or more."""
    T, V, D = h.shape[0], w.shape[0], h.shape[1]
    off = (t < 0) | (t >= V)
    who = torch.arange(T, device="cuda")[~off]
    _, lse = plan.forward(h, w, t)
    H, W, AW = torch.where(off[:, None], 0.0, h.double()), w.double(), w.double().abs()
    e = ((H.abs() @ AW.t()).amax(1) * D * U)[:, None] + 100 * U  # a logit's error, the exponential's, its argument's
    P = torch.exp(H @ W.t() - lse.double()[:, None])
    G = P.clone()
    G[who, t[who]] -= 1
    G[off], P[off] = 0, 0
    upd = torch.where(off, 0.0, up.double())
    dG = torch.minimum(G.abs() * half(dtype) + 2.0 ** -37, G.abs())
    dG[who, t[who]] = 0
    dG += P * 2 * e
    at = torch.zeros_like(G)
    at[who, t[who]] = G[who, t[who]].abs()
    AG = G.abs()
    gh, gw = plan.backward(h, w, t, lse, up, grad_weight=grad_weight)
    gh_ref = upd[:, None] * (G @ W)
    tol = upd.abs()[:, None] * ((dG + at * 4 * U) @ AW + (V + 4) * U * (AG @ AW))
    within(gh, gh_ref, tol * (1 + half(dtype)) + half(dtype) * gh_ref.abs() + tiny(dtype), "grad_hidden")
    gw_ref = (G * upd[:, None]).t() @ H
    one = bool((up[~off] == up[~off][:1]).all())
    entry = dG + at * half(dtype) ** 2 + AG * ((T + 4) * U + (0 if one else half(dtype)))
    tol = (entry * upd.abs()[:, None]).t() @ H.abs()
    if not one and dtype == F16:
        tol += AG.sum(0)[:, None] * 2.0 ** -38 * (upd[:, None] * H).abs().max()
    round_ = half(gw.dtype)
    within(gw, gw_ref, tol * (1 + round_) + round_ * gw_ref.abs() + tiny(gw.dtype), "grad_weight")
    assert torch.equal(plan.backward(h, w, t, lse, up)[0], gh)  # the same bits


def targets_of(T, V, g, kind):
    if kind == "one":
        return torch.full((T,), V // 2, device="cuda")
    if kind == "words":  # a few low ids take many of the tokens
        return (torch.rand(T, generator=g, device="cuda", dtype=torch.float64) ** 3 * V).long().clamp_(max=V - 1)
    return torch.arange(T, device="cuda") // 9 % V  # nine tokens each


@pytest.mark.parametrize("T,V,D,kind", [
    (9, 300, 64, "one"), (64, 1000, 72, "one"), (65, 1000, 61, "one"), (512, 1000, 128, "one"), (512, 1000, 128, "nine"),
    (333, 5003, 520, "words"), (8, 20000, 136, "one"), (700, 70000, 64, "words"), (2048, 8192, 256, "words"),
    (4100, 70001, 72, "words"), (1500, 3000, 1040, "nine")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_targets_lose_nothing_to_rounding(gpu, T, V, D, kind, dtype):
    """However many tokens share a target: in bf16 2^12 (p - 1) is -2^12 for every p below 2^-9, always to the same side, so
    without the correction a row of many such tokens is off by the mean of their p."""
    g = gen(T + V)
    w = rand((V, D), dtype, g, std=0.5 * D ** -0.5)
    h = rand((T, D), dtype, g)
    t = targets_of(T, V, g, kind)
    if T > 20:
        t[3::17] = -1
    plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
    for gw in (torch.empty(V, D, device="cuda"), None):
        check_gradients(plan, h, w, t, torch.full((T,), 1.0 / T, device="cuda"), dtype, gw)


@pytest.mark.parametrize("T,D", [(40, 64), (200, 77), (1500, 136), (5000, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_tokens_of_small_factors_count(gpu, T, D, dtype):
    """Factors from 1 to 1e-8 of the largest.  Every token is sure of a word of its own kind (logits of some 80 against 8
    and less) that is not its target, and its target is nobody else's: that row of grad_weight is its hidden state times
    its factor, whatever the others' factors are."""
    g = gen(T + D)
    V, K = T + 32, 32
    w = rand((V, D), dtype, g, std=0.01)
    w[:K] = 0
    w[torch.arange(K), torch.arange(K)] = 8.0
    h = (torch.rand(T, D, generator=g, device="cuda") * 0.7 + 0.3).to(dtype)
    h[torch.arange(T), torch.arange(T) % K] = 10.0
    t = K + torch.randperm(T, generator=g, device="cuda")
    up = 10.0 ** (-8 * torch.rand(T, generator=g, device="cuda"))
    up[0], up[1:4] = 1.0, torch.tensor([1e-6, -1e-7, 0.0], device="cuda")
    up[T // 2::7] *= -1
    plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
    for scale in (1.0, 1e-6, 1e3):
        check_gradients(plan, h, w, t, up * scale, dtype, torch.empty(V, D, device="cuda"))
    check_gradients(plan, (h.float() * 1e-3).to(dtype), w, t, up, dtype, torch.empty(V, D, device="cuda"))
    check_gradients(plan, (h.float() * 300).to(dtype), (w.float() / 300).to(dtype), t, up, dtype,
                    torch.empty(V, D, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_tiles_of_both_products(gpu, dtype):
    """Sizes whose grad_hidden and grad_weight both have a tile of 256 x 256 a CU, with two pieces of the vocabulary, the
    last of them ragged, and every size ragged for the tiles."""
    T, V, D = 8200, 20003, 2056
    g = gen(77)
    h, w, t, off = loss_inputs(T, V, D, dtype, g)
    t[::3] = torch.where(off[::3], t[::3], targets_of(t[::3].numel(), V, g, "words"))
    plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
    up = rand((T,), F32, g)
    check_gradients(plan, h, w, t, up, dtype, None)
    check_gradients(plan, h, w, t, up, dtype, torch.empty(V, D, device="cuda"))


@pytest.mark.parametrize("rows,dim", [(3, 1000), (5, 777), (2, 61), (1, 4095), (2, 4104), (2, 16384), (2, 20001), (700, 1000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_far_from_zero(gpu, rows, dim, dtype):
    """A large mean costs nothing: it is found to k u of the distances from the first estimate, which itself is off by m = k u
    mean|x|.  So with b = max|x - mean| + m the output is off by (k + 4) u b rstd, and by rstd's own error, whatever the
    mean is; rows of one value give zeros."""
    g = gen(rows + dim)
    k = depth(dim) + 2
    eps = torch.tensor(1e-5, dtype=F32).item()
    for mean, std in ((10000.1, 0.0), (1000.3, 0.0), (-10000.1, 1.0), (1e6, 30.0), (300.0, 0.01)):
        x = rand((rows, dim), F32, g, std=std, mean=mean).clamp_(-6e4, 6e4).to(dtype)
        r = ops.layer_norm(x)
        xd = x.double()
        mu = xd.mean(1, keepdim=True)
        var = (xd - mu).square().mean(1, keepdim=True)
        rstd = 1 / torch.sqrt(var + eps)
        y = (xd - mu) * rstd
        m = k * U * xd.abs().mean(1, keepdim=True)
        b = (xd - mu).abs().amax(1, keepdim=True) + m
        # the squares' sum is off by (k + 4) u of itself, it and the square taken off it are at most var + m^2, m^2
        rel = ((k + 6) * U * (var + 2 * m * m) + 2 * (k + 4) * U * b * m) / (var + eps) / 2 + 6 * U
        within(r.rstd, rstd[:, 0], (rel * rstd)[:, 0], ("rstd", mean, std))
        within(r.mean, mu[:, 0], (k * U * b + U * mu.abs())[:, 0], ("mean", mean, std))
        tol = (k + 4) * U * b * rstd * (1 + rel) + y.abs() * rel + 2 * U * y.abs()
        within(r.out, y, tol * (1 + half(dtype)) + half(dtype) * y.abs() + tiny(dtype), ("out", mean, std))


def test_captured_backward_of_unequal_factors(gpu):
    """The fp16 loss with a factor for each token, captured: every replay, on new inputs and with eager work between, gives
    the eager bits."""
    T, V, D = 300, 900, 136
    g = gen(41)
    h, w, t, _ = loss_inputs(T, V, D, F16, g)
    up = rand((T,), F32, g)
    eager, plan = ops.VocabLossPlan(T, V, D, dtype=F16), ops.VocabLossPlan(T, V, D, dtype=F16)
    gw = torch.empty(V, D, device="cuda")

    def run(p, gw):
        loss, lse = p.forward(h, w, t)
        return [loss, lse, *p.backward(h, w, t, lse, up, grad_weight=gw)]

    run(plan, gw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(plan, gw)
    for k in range(4):
        for old, new in zip((h, w, t), loss_inputs(T, V, D, F16, gen(50 + k))):
            old.copy_(new)
        up.copy_(rand((T,), F32, gen(60 + k)) * 10.0 ** -k)
        want = run(eager, torch.empty(V, D, device="cuda"))
        gw.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_backward_of_expanded_rows(gpu, dtype):
    """One hidden state for all tokens, or one row for the whole vocabulary: a stride of 0, the same bits."""
    T, V, D = 70, 300, 64
    g = gen(42)
    h, w, t, _ = loss_inputs(T, V, D, dtype, g)
    up = rand((T,), F32, g)
    plan = ops.VocabLossPlan(T, V, D, dtype=dtype)
    for hh, ww in ((h[:1].expand(T, D), w), (h, w[:1].expand(V, D))):
        _, lse = plan.forward(hh, ww, t)
        a = plan.backward(hh, ww, t, lse, up, torch.empty_like(h), torch.empty_like(w))
        b = plan.backward(hh.contiguous(), ww.contiguous(), t, lse, up)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_backward_without_given_outputs_of_expanded_rows(gpu):
    """What is not given is allocated with rows of its own."""
    h, w, t, _ = loss_inputs(20, 30, 64, BF16, gen(43))
    plan = ops.VocabLossPlan(20, 30, 64)
    _, lse = plan.forward(h[:1].expand(20, 64), w, t)
    gh, gw = plan.backward(h[:1].expand(20, 64), w, t, lse, torch.ones(20, device="cuda"))
    assert gh.stride() == (64, 1) and gw.stride() == (64, 1)


def test_calls_on_two_streams(gpu):
    """Two losses at once, a plan each."""
    T, V, D = 260, 4000, 264
    sets = [loss_inputs(T, V, D, F16, gen(70 + k)) for k in range(2)]
    plans = [ops.VocabLossPlan(T, V, D, dtype=F16) for _ in range(2)]
    up = rand((T,), F32, gen(3))

    def run(k, stream=None):
        h, w, t, _ = sets[k]
        loss, lse = plans[k].forward(h, w, t, stream=stream)
        return [loss, lse, *plans[k].backward(h, w, t, lse, up, stream=stream)]

    want = [run(k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[run(k, streams[k]) for k in range(2)] for _ in range(8)]
    torch.cuda.synchronize()
    for both in got:
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(both[k], want[k]))
