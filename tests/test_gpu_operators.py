"""Class log probabilities and per-leaf products against plain 64-bit formulas.

Tolerances, from u = 2^-24 (half a step of fp32; a type's own half step is eps / 2):
* a sum of K positive terms, each e^x with a relative error of a few u (1 + |x|): at most u (K / 32 + 64 + 4 max |x|) relative
  (no thread adds more than K / 32 terms in a row, the rest is a tree), |x| weighted by the terms themselves, so below 16;
* log p and log_norm: that, plus u times the size of the scores; the entropy: that times (1 + log K);
* a gradient p (a + b log p): relative u (64 + 4 |log p|) plus the error of log_norm, plus half a step of its type;
* a product over F terms: 2 u (F + 8) sum |x w| (a matrix instruction may cut instead of rounding), plus half a step of its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    g = torch.Generator(device="cuda"); g.manual_seed(seed)
    return g


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _scores(n, k, dtype, layout, seed=0, spread=2.5):
    g = _gen(seed)
    if layout == "row":
        return torch.randn((n, k), generator=g, device="cuda").mul(spread).to(dtype)
    if layout == "class":                                     # as the training scores lie
        return torch.randn((k, n), generator=g, device="cuda").mul(spread).to(dtype).t()
    if layout == "padded":                                    # a window of a larger matrix, off the 16-byte boundary
        return torch.randn((n, k + 7), generator=g, device="cuda").mul(spread).to(dtype)[:, 3:3 + k]
    if layout == "strided":                                   # every other class of every third row
        return torch.randn((3 * n, 2 * k), generator=g, device="cuda").mul(spread).to(dtype)[::3, ::2]
    raise ValueError(layout)


def _reference(scores, labels, top):
    s = scores.double()
    k = s.shape[1]
    none = torch.isneginf(s).all(1)
    bad = torch.isnan(s).any(1) | torch.isposinf(s).any(1)
    most = torch.where(none | bad, 0.0, s.max(1).values)
    log_sum = torch.log(torch.exp(s - most[:, None]).sum(1))
    lse = most + log_sum
    logp = torch.where(torch.isneginf(s), s, (s - most[:, None]) - log_sum[:, None])   # not s - lse: at 1e38 a 64-bit lse no longer holds log K
    plogp = torch.where(torch.isneginf(s), 0.0, torch.exp(logp) * logp)
    nan = torch.full_like(lse, math.nan)
    out = {"log_norm": torch.where(bad, nan, lse), "entropy": torch.where(bad, nan, torch.where(none, 0.0, -plogp.sum(1)))}
    if labels is not None:
        y = labels.long()
        lp = logp.gather(1, y.clamp(0, k - 1)[:, None])[:, 0]
        out["log_prob"] = torch.where(y < 0, 0.0, torch.where(bad | (y >= k), nan, lp))
    if top:
        v, c = torch.sort(s, dim=1, descending=True, stable=True)
        v, c = v[:, :top], c[:, :top]
        out["top_class"] = torch.where(bad[:, None] | torch.isneginf(v), -1, c).int()
        out["top_log_prob"] = torch.where(bad[:, None], nan[:, None], torch.where(torch.isneginf(v), v, logp.gather(1, c)))
    return out, logp


def _check_forward(scores, labels, top):
    from falcata_b200 import ops
    got = ops.class_log_probs(scores, labels, top_k=top)
    want, _ = _reference(scores, labels, top)
    k = scores.shape[1]
    finite = scores.double()[torch.isfinite(scores)].abs()
    size = float(finite.max()) if finite.numel() else 0.0
    tol = U * (k / 32 + 64 + 4 * 16) + 4 * U * size
    for name, w in want.items():
        g = getattr(got, name)
        assert g.shape == w.shape and g.device == scores.device
        if name == "top_class":
            assert g.dtype == torch.int32 and torch.equal(g, w)
            continue
        assert g.dtype == torch.float32
        t = tol * (1 + math.log(k)) if name == "entropy" else tol
        assert torch.allclose(g.double(), w, rtol=U, atol=t, equal_nan=True), (name, float((g.double() - w).nan_to_num(0, 0, 0).abs().max()), t)
    assert (got.log_prob is None) == (labels is None) and (got.top_class is None) == (top == 0)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["row", "class", "padded", "strided"])
@pytest.mark.parametrize("n,k,top", [(1, 1, 1), (5, 2, 2), (1000, 3, 0), (257, 10, 3), (33, 31, 31), (64, 64, 5), (65, 65, 32), (7, 127, 4), (130, 1000, 20), (3, 1025, 1), (9, 4099, 32), (41, 6401, 3), (2, 50021, 20)])
def test_class_log_probs(dtype, layout, n, k, top):
    scores = _scores(n, k, dtype, layout, seed=n + k)
    labels = torch.randint(-1, k, (n,), generator=_gen(1), device="cuda")
    _check_forward(scores, labels.int() if n % 2 else labels, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,top", [(1, 131075, 20), (2, 262147, 32), (40, 70001, 7), (300, 20000, 5)])
def test_class_log_probs_many_classes(dtype, n, k, top):
    _check_forward(_scores(n, k, dtype, "padded", seed=3, spread=4.0), torch.randint(0, k, (n,), generator=_gen(2), device="cuda", dtype=torch.int32), top)


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "blocks", "one", "last"])
@pytest.mark.parametrize("layout", ["row", "class"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,top", [(48, 32), (700, 32), (3000, 20), (40000, 32)])
def test_class_log_probs_orders_and_ties(order, layout, dtype, k, top):
    """Rows whose order or ties are the worst for a selection: the lowest classes win among equals."""
    at = torch.arange(k, device="cuda")
    row = {"rising": at * (8.0 / k), "falling": -at * (8.0 / k), "equal": torch.zeros(k, device="cuda"), "blocks": -(at // 97 % 5).float(),
           "one": (at == k // 2) * 9.0, "last": (at >= k - top) * 3.0}[order]
    scores = row.to(dtype).repeat(3, 1)
    scores[1] = scores[1].flip(0)
    scores[2] = -0.0 * scores[2]                       # zeros of both signs are equal scores
    scores[2, ::2] = 0.0
    _check_forward(scores if layout == "row" else scores.t().contiguous().t(), torch.tensor([0, k - 1, k // 2], device="cuda"), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["row", "class", "padded"])
@pytest.mark.parametrize("k,top", [(5, 5), (40, 32), (300, 32), (5000, 20), (60000, 32)])
def test_class_log_probs_ruled_out_classes(dtype, layout, k, top):
    """-inf rules a class out; the type's lowest value does not; NaN and +inf spoil their row only."""
    lowest = torch.finfo(dtype).min
    s = _scores(12, k, dtype, layout, seed=5)
    s[1] = -math.inf                                   # nothing left
    s[2] = -math.inf; s[2, k // 2] = 1.5               # one class left
    s[3, : k // 2] = -math.inf
    s[4] = lowest                                      # uniform at the lowest value
    s[5] = lowest; s[5, 1] = -3.0
    s[6, k - 1] = math.nan
    s[7, 0] = math.inf
    s[8] = -math.inf; s[8, k - 1] = lowest
    s[9] = -math.inf; s[9, k // 3] = math.nan
    s[10] = torch.finfo(dtype).max
    s[11, :: 2] = -math.inf; s[11, 1] = lowest
    labels = torch.tensor([0, 0, k // 2, 0, 1, 0, 0, 1, k - 1, -1, 2, k], device="cuda")
    from falcata_b200 import ops
    got = ops.class_log_probs(s, labels, top_k=top)
    want, logp = _reference(s, labels, top)
    assert torch.equal(got.top_class, want["top_class"])
    for name in ("log_prob", "log_norm", "entropy", "top_log_prob"):
        g, w = getattr(got, name).double(), want[name]
        scale = U * (k / 32 + 128) + 4 * U * 16
        w32 = w.float().double()                       # log probabilities beyond fp32's range are -inf there
        assert torch.allclose(g, w32, rtol=4 * U, atol=scale * (1 + math.log(k)), equal_nan=True), name
    up = {"grad_log_prob": torch.ones(12, device="cuda"), "grad_log_norm": torch.full((12,), 0.5, device="cuda"), "grad_entropy": torch.full((12,), -0.25, device="cuda")}
    grad = ops.class_log_probs_grad(s, got.log_norm, got.entropy, labels=labels, **up).double()
    p = torch.where(torch.isneginf(logp), 0.0, torch.exp(logp))
    h = want["entropy"][:, None]
    ref = 0.5 * p + 0.25 * torch.where(p > 0, p * (logp.nan_to_num(0, 0, 0) + h), 0.0)
    y = labels.long()
    for i in range(12):
        if i == 1:
            ref[i] = 0.0
        elif i in (6, 7, 9, 11):
            ref[i] = math.nan
        else:
            ref[i] -= p[i]; ref[i, y[i]] += 1.0
    assert torch.allclose(grad, ref, rtol=_half_step(dtype), atol=U * (k / 32 + 256) + (6e-8 if dtype == torch.float16 else 0), equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["row", "class", "padded", "strided"])
@pytest.mark.parametrize("n,k,top", [(1, 1, 1), (6, 2, 2), (300, 10, 3), (33, 64, 32), (31, 65, 4), (70, 1000, 20), (5, 4099, 32), (3, 50021, 5), (2, 131075, 0)])
def test_class_log_probs_grad(dtype, layout, n, k, top):
    """Against the formula in 64 bits, and the formula against differences of the loss."""
    from falcata_b200 import ops
    s = _scores(n, k, dtype, layout, seed=n * k)
    labels = torch.randint(-1, k, (n,), generator=_gen(7), device="cuda")
    g = _gen(8)
    up = [torch.randn(n, generator=g, device="cuda") for _ in range(3)] + ([torch.randn((n, top), generator=g, device="cuda")] if top else [])
    out = ops.class_log_probs(s, labels, top_k=top)
    grad = ops.class_log_probs_grad(s, out.log_norm, out.entropy, labels=labels, top_class=out.top_class, grad_log_prob=up[0], grad_log_norm=up[1], grad_entropy=up[2],
                                    grad_top_log_prob=up[3] if top else None)
    assert grad.dtype == dtype and grad.shape == s.shape and grad.stride(0 if layout == "class" and n > 1 and k > 1 else 1) == 1

    def loss(x):
        logp = torch.log_softmax(x, 1)
        total = (torch.where(labels < 0, 0.0, logp.gather(1, labels.clamp(min=0)[:, None])[:, 0]) * up[0].double()).sum()
        total = total + (torch.logsumexp(x, 1) * up[1].double()).sum() - ((logp.exp() * logp).sum(1) * up[2].double()).sum()
        return total + (logp.gather(1, out.top_class.long()) * up[3].double()).sum() if top else total

    x = s.double().requires_grad_()
    ref, = torch.autograd.grad(loss(x), x)
    step = torch.randn(s.shape, generator=g, device="cuda", dtype=torch.float64)
    slope = (loss(x.detach() + 1e-5 * step) - loss(x.detach() - 1e-5 * step)) / 2e-5
    assert abs(float(slope - (ref * step).sum())) <= 1e-6 * (1 + float((ref * step).abs().sum()))
    logp = torch.log_softmax(s.double(), 1)
    weight = sum(u.abs().double() if u.dim() == 1 else u.abs().double().sum(1) for u in up)[:, None]
    h = (out.entropy.double() + 1)[:, None]
    bound = logp.exp() * weight * (h + logp.abs()) * (U * (k / 32 + 128) + 8 * U * (16 + logp.abs()))
    given = torch.zeros_like(ref); rows = torch.arange(n, device="cuda")
    given[rows, labels.clamp(min=0)] += up[0].abs().double()
    if top:
        given.scatter_add_(1, out.top_class.long(), up[3].abs().double())
    bound = bound + 8 * U * given + _half_step(dtype) * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (grad.double() - ref).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("layout,k", [("row", 10), ("row", 300), ("row", 5000), ("row", 40000), ("class", 10), ("class", 300)])
@pytest.mark.parametrize("shift", [-3e4, 1e6, 2.0 ** 100])
def test_class_log_probs_far_from_zero(layout, k, shift):
    """Scores far from zero: fp32's log_norm no longer holds the probabilities, the results still do."""
    from falcata_b200 import ops
    s = _scores(20, k, torch.float32, layout, seed=2) + shift
    labels = torch.randint(0, k, (20,), generator=_gen(1), device="cuda")
    got = ops.class_log_probs(s, labels)
    want, logp = _reference(s, labels, 0)
    tol = U * (k / 32 + 128)
    assert torch.allclose(got.log_prob.double(), want["log_prob"], rtol=4 * U, atol=tol) and torch.allclose(got.entropy.double(), want["entropy"], rtol=4 * U, atol=tol * (1 + math.log(k)))
    assert torch.allclose(got.log_norm.double(), want["log_norm"], rtol=2 * U, atol=tol)
    grad = ops.class_log_probs_grad(s, got.log_norm, got.entropy, labels=labels, grad_log_prob=torch.ones(20, device="cuda")).double()
    ref = -logp.exp()
    ref[torch.arange(20, device="cuda"), labels] += 1
    assert torch.allclose(grad, ref, rtol=U, atol=U * (k / 32 + 256))


def test_class_log_probs_autograd_and_repeated_indices():
    from falcata_b200 import ops
    s = _scores(50, 300, torch.float32, "row").requires_grad_()
    labels = torch.randint(0, 300, (50,), generator=_gen(1), device="cuda")
    r = ops.class_log_probs(s, labels, top_k=4)
    (-r.log_prob.mean() - 0.01 * r.entropy.mean() + 0.1 * r.top_log_prob[:, 1:].sum() + 1e-3 * (r.log_norm ** 2).mean()).backward()
    x = s.detach().double().requires_grad_()
    logp = torch.log_softmax(x, 1)
    loss = -logp.gather(1, labels[:, None]).mean() + 0.01 * (logp.exp() * logp).sum(1).mean() + 0.1 * logp.gather(1, r.top_class.long())[:, 1:].sum() + 1e-3 * (torch.logsumexp(x, 1) ** 2).mean()
    loss.backward()
    assert torch.allclose(s.grad.double(), x.grad, rtol=1e-5, atol=2e-6)
    # the same alternative named several times, the label among them, and entries that name none
    t = torch.tensor([[3, 3, 3, 7], [-1, 5, 5, -1]], dtype=torch.int32, device="cuda")
    g = torch.tensor([[1.0, 2.0, 4.0, -1.0], [9.0, 1.0, 1.0, 9.0]], device="cuda")
    for layout in ("row", "class"):
        sc = _scores(2, 9, torch.float32, layout, seed=3)
        f = ops.class_log_probs(sc)
        got = ops.class_log_probs_grad(sc, f.log_norm, f.entropy, labels=torch.tensor([3, 5], device="cuda"), top_class=t, grad_log_prob=torch.tensor([0.5, 0.25], device="cuda"), grad_top_log_prob=g)
        p = torch.softmax(sc.double(), 1)
        want = -p * torch.tensor([[6.5], [2.25]], device="cuda")
        want[0, 3] += 7.5; want[0, 7] -= 1.0; want[1, 5] += 2.25
        assert torch.allclose(got.double(), want, atol=4e-6)
    with pytest.raises(RuntimeError):      # differentiable once
        z = _scores(2, 9, torch.float32, "row").requires_grad_()
        d, = torch.autograd.grad(ops.class_log_probs(z).entropy.sum(), z, create_graph=True)
        d.sum().backward()


def test_class_log_probs_empty_and_unused():
    from falcata_b200 import ops
    s = torch.zeros((0, 5), device="cuda", requires_grad=True)
    r = ops.class_log_probs(s, torch.zeros(0, dtype=torch.int32, device="cuda"), top_k=2)
    assert r.log_prob.shape == (0,) and r.top_class.shape == (0, 2)
    r.log_prob.sum().backward()
    assert s.grad.shape == (0, 5)
    wide = torch.randn(1, 20, device="cuda").expand(6, 20)        # a broadcast row
    assert torch.equal(ops.class_log_probs(wide, top_k=3).top_class, ops.class_log_probs(wide.contiguous(), top_k=3).top_class)
    w = torch.randn(1, 20, device="cuda", requires_grad=True)
    y = torch.arange(6, device="cuda")
    ops.class_log_probs(w.expand(6, 20), y).log_prob.sum().backward()
    p = torch.softmax(w.detach().double(), 1)
    want = -6 * p; want[0, :6] += 1
    assert torch.allclose(w.grad.double(), want, atol=6 * 64 * U)


# ------------------------------------------------------------------------------------------------ leaves ----
def _leaves(n, leaves, seed, empty=True):
    g = torch.Generator(); g.manual_seed(seed)
    cuts = torch.sort(torch.randint(0, n + 1, (leaves - 1,), generator=g)).values if leaves > 1 else torch.zeros(0, dtype=torch.long)
    if empty and leaves > 3:
        cuts[1] = cuts[0]
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([n])]).to(torch.int32).cuda()


def _ref_products(x, w, begin):
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device="cuda"); size = torch.zeros_like(y)
    b = begin.tolist()
    for g in range(w.shape[0]):
        y[b[g]:b[g + 1]] = x[b[g]:b[g + 1]].double() @ w[g].double().t()
        size[b[g]:b[g + 1]] = x[b[g]:b[g + 1]].double().abs() @ w[g].double().abs().t()
    return y, size


def _near(got, want, size, terms, dtype):
    bound = 2 * U * (terms + 8) * size + _half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


SHAPES = [(1, 1, 1, 1), (3, 5, 2, 4), (100, 28, 10, 7), (257, 33, 17, 3), (1000, 136, 1, 31), (513, 100, 100, 5), (64, 130, 257, 2), (2000, 8, 64, 255), (300, 257, 129, 4), (40, 2000, 30, 40),
          (1200, 64, 256, 3), (700, 200, 520, 2), (1500, 135, 259, 3), (5000, 40, 70, 4), (2000, 272, 296, 2), (1999, 640, 128, 3), (1100, 264, 520, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,f,k,leaves", SHAPES)
def test_leaf_products(dtype, n, f, k, leaves):
    from falcata_b200 import ops
    g = _gen(n + f)
    x = torch.randn((n, f), generator=g, device="cuda").to(dtype); w = torch.randn((leaves, k, f), generator=g, device="cuda").mul(f ** -0.5).to(dtype)
    begin = _leaves(n, leaves, seed=k)
    y = ops.leaf_products(x, w, begin)
    assert y.dtype == dtype and y.shape == (n, k)
    want, size = _ref_products(x, w, begin)
    _near(y, want, size, f, dtype)
    # the transposed maps: the gradient in x
    d = torch.randn((n, k), generator=g, device="cuda").to(dtype)
    want, size = _ref_products(d, w.transpose(1, 2), begin)
    _near(ops.leaf_products(d, w.transpose(1, 2), begin.long()), want, size, k, dtype)
    # the gradient in the maps, in the inputs' type and in fp32
    b = begin.tolist()
    want = torch.stack([d[lo:hi].double().t() @ x[lo:hi].double() for lo, hi in zip(b[:-1], b[1:])])
    size = torch.stack([d[lo:hi].double().abs().t() @ x[lo:hi].double().abs() for lo, hi in zip(b[:-1], b[1:])])
    p = ops.leaf_gram(d, x, begin)
    assert p.dtype == dtype and p.shape == (leaves, k, f)
    _near(p, want, size, n, dtype)
    _near(ops.leaf_gram(d, x, begin, dtype=torch.float32), want, size, n, torch.float32)
    assert torch.equal(p, ops.leaf_gram(d, x, begin))          # the same sums on every run


@pytest.mark.parametrize("dtype", TYPES)
def test_leaf_products_strides_and_alignment(dtype):
    from falcata_b200 import ops
    n, f, k, leaves = 333, 40, 24, 6
    g = _gen(4)
    big = torch.randn((n, f + 13), generator=g, device="cuda").to(dtype)
    wbig = torch.randn((leaves, k + 3, f + 5), generator=g, device="cuda").to(dtype)
    begin = _leaves(n, leaves, seed=1)
    for x in (big[:, 8:8 + f], big[:, 3:3 + f], big[:, :f].t().contiguous().t(), big[:1, :f].expand(n, f)):
        for w in (wbig[:, :k, :f], wbig[:, 1:1 + k, 5:5 + f], wbig[:, :k, :f].transpose(1, 2).contiguous().transpose(1, 2), wbig[:1, :k, :f].expand(leaves, k, f)):
            want, size = _ref_products(x, w, begin)
            _near(ops.leaf_products(x, w, begin), want, size, f, dtype)
        d = big[:, 10:10 + k]
        b = begin.tolist()
        want = torch.stack([d[lo:hi].double().t() @ x[lo:hi].double() for lo, hi in zip(b[:-1], b[1:])])
        size = torch.stack([d[lo:hi].double().abs().t() @ x[lo:hi].double().abs() for lo, hi in zip(b[:-1], b[1:])])
        _near(ops.leaf_gram(d, x, begin), want, size, n, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f,k,cut", [(24, 16, 100), (64, 40, 112), (20, 16, 90)])
def test_leaf_products_neighbours_do_not_mix(dtype, f, k, cut):
    """A leaf of NaN and infinite rows next to others: they reach no other leaf's rows or sums, wherever tiles and steps end."""
    from falcata_b200 import ops
    g = _gen(8)
    x = torch.randn((400, f), generator=g, device="cuda").to(dtype); d = torch.randn((400, k), generator=g, device="cuda").to(dtype)
    w = torch.randn((4, k, f), generator=g, device="cuda").to(dtype)
    bad = slice(cut, cut + 37)
    x[bad] = math.nan; x[cut + 3] = math.inf; d[bad] = -math.inf
    begin = torch.tensor([0, cut, cut + 37, cut + 37, 400], device="cuda")
    y, p = ops.leaf_products(x, w, begin), ops.leaf_gram(d, x, begin)
    keep = [(0, 0, cut), (3, cut + 37, 400)]
    for leaf, lo, hi in keep:
        _near(y[lo:hi], x[lo:hi].double() @ w[leaf].double().t(), x[lo:hi].double().abs() @ w[leaf].double().abs().t(), f, dtype)
        _near(p[leaf], d[lo:hi].double().t() @ x[lo:hi].double(), d[lo:hi].double().abs().t() @ x[lo:hi].double().abs(), hi - lo, dtype)
    assert bool((p[2] == 0).all()) and bool(torch.isnan(p[1]).any()) and bool(torch.isnan(y[bad]).all(1).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_leaf_products_rows_outside_the_leaves(dtype):
    """Rows in no leaf: zero outputs, no share in the sums, whatever they hold; boundaries past the rows are clamped."""
    from falcata_b200 import ops
    g = _gen(6)
    x = torch.randn((300, 20), generator=g, device="cuda").to(dtype); w = torch.randn((3, 12, 20), generator=g, device="cuda").to(dtype); d = torch.randn((300, 12), generator=g, device="cuda").to(dtype)
    x[:10] = math.nan; x[250:] = math.inf; d[:10] = math.nan; d[250:] = math.nan
    begin = torch.tensor([10, 100, 100, 250], device="cuda")
    y = ops.leaf_products(x, w, begin)
    assert bool((y[:10] == 0).all()) and bool((y[250:] == 0).all())
    want, size = _ref_products(x[10:250], w, begin - 10)
    _near(y[10:250], want, size, 20, dtype)
    p = ops.leaf_gram(d, x, begin)
    assert bool((p[1] == 0).all()) and bool(torch.isfinite(p).all())
    want = torch.stack([d[lo:hi].double().t() @ x[lo:hi].double() for lo, hi in ((10, 100), (100, 100), (100, 250))])
    size = torch.stack([d[lo:hi].double().abs().t() @ x[lo:hi].double().abs() for lo, hi in ((10, 100), (100, 100), (100, 250))])
    _near(p, want, size, 240, dtype)
    z = ops.leaf_products(x[10:250], w, torch.tensor([-5, 90, 90, 10 ** 6], device="cuda"))
    assert torch.equal(z, y[10:250])
    assert ops.leaf_products(x[:0], w, torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 12)
    assert bool((ops.leaf_gram(d[:0], x[:0], torch.zeros(4, dtype=torch.int32, device="cuda")) == 0).all())
    assert bool((ops.leaf_products(x, w, torch.zeros(4, dtype=torch.int32, device="cuda")) == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,a_cols,b_cols", [(257, 8, 4), (2048, 8, 4), (2049, 8, 4), (6000, 9, 5), (9000, 70, 50), (1500, 130, 270), (20000, 130, 270)])
def test_leaf_gram_of_long_leaves(dtype, rows, a_cols, b_cols):
    """Leaves of few and of many slices side by side, and one of a single slice."""
    from falcata_b200 import ops
    g = _gen(12)
    n = rows + 2 * (rows // 3) + 60
    a = torch.randn((n, a_cols), generator=g, device="cuda").to(dtype); b = torch.randn((n, b_cols), generator=g, device="cuda").to(dtype)
    begin = torch.tensor([0, rows // 3, rows // 3 + rows, n - 60, n], device="cuda")
    for out in (dtype, torch.float32):
        p = ops.leaf_gram(a, b, begin, dtype=out)
        at = begin.tolist()
        for leaf, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
            _near(p[leaf], a[lo:hi].double().t() @ b[lo:hi].double(), a[lo:hi].double().abs().t() @ b[lo:hi].double().abs(), hi - lo, out)
        assert torch.equal(p, ops.leaf_gram(a, b, begin, dtype=out))


def test_leaf_products_autograd():
    from falcata_b200 import ops
    g = _gen(9)
    x = torch.randn((400, 30), generator=g, device="cuda", requires_grad=True); w = torch.randn((5, 7, 30), generator=g, device="cuda", requires_grad=True)
    begin = _leaves(400, 5, seed=2)
    (ops.leaf_products(x, w, begin) ** 2).sum().backward()
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    b = begin.tolist()
    sum(((xd[b[i]:b[i + 1]] @ wd[i].t()) ** 2).sum() for i in range(5)).backward()
    assert torch.allclose(x.grad.double(), xd.grad, rtol=1e-5, atol=1e-4) and torch.allclose(w.grad.double(), wd.grad, rtol=1e-5, atol=1e-3)
    ops.leaf_products(x, w[:1].expand(5, 7, 30), begin).sum().backward()       # one map shared by all leaves, a broadcast gradient
    assert torch.isfinite(w.grad).all()


# -------------------------------------------------------------------------------------- together, streams ----
def _head_step(x, w, begin, labels):
    from falcata_b200 import ops
    r = ops.class_log_probs(ops.leaf_products(x, w, begin), labels, top_k=3)
    loss = -(r.log_prob.mean() + 0.01 * r.entropy.mean())
    return (loss, r.top_class) + torch.autograd.grad(loss, (x, w))


def test_forest_leaves_with_class_heads():
    """As they are used together: a forest's leaves group the rows, every leaf has a linear head, the heads' scores give the loss."""
    import falcata_b200 as fb
    from falcata_b200 import ops
    from util import make_multiclass
    X, y = make_multiclass(n=3000, f=12, k=4)
    bst = fb.train({"objective": "multiclass", "num_class": 4, "num_leaves": 15, "device_type": "cuda", "verbosity": -1}, fb.Dataset(X, y), 2)
    Xd = torch.from_numpy(X).cuda()
    leaf = bst.predict(Xd, pred_leaf=True)[:, 0].long()
    order = torch.argsort(leaf, stable=True)
    begin = torch.searchsorted(leaf[order].contiguous(), torch.arange(16, device="cuda")).int()
    x = Xd[order].contiguous().requires_grad_()
    w = torch.zeros((15, 4, 12), device="cuda").normal_(0, 0.1, generator=_gen(3)).requires_grad_()
    labels = torch.from_numpy(y).cuda().int()[order]
    loss, top, gx, gw = _head_step(x, w, begin, labels)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    s = torch.einsum("nf,nkf->nk", xd, wd[leaf[order]])
    logp = torch.log_softmax(s, 1)
    ref = -(logp.gather(1, labels.long()[:, None]).mean() - 0.01 * (logp.exp() * logp).sum(1).mean())
    rx, rw = torch.autograd.grad(ref, (xd, wd))
    assert abs(float(loss.detach()) - float(ref.detach())) < 64 * U * 4
    assert torch.allclose(gx.double(), rx, rtol=1e-4, atol=1e-9 + 256 * U / 3000) and torch.allclose(gw.double(), rw, rtol=1e-4, atol=4096 * U / 15)


def test_booster_log_probs():
    """The log probabilities of a model's answers agree with its probabilities."""
    import falcata_b200 as fb
    from util import make_multiclass
    X, y = make_multiclass(n=1500, f=8, k=5)
    bst = fb.train({"objective": "multiclass", "num_class": 5, "num_leaves": 15, "device_type": "cuda", "verbosity": -1}, fb.Dataset(X, y), 5)
    Xd, labels = torch.from_numpy(X).cuda(), torch.from_numpy(y).cuda().long()
    r, p = bst.predict_log_probs(Xd, labels, top_k=2), bst.predict(Xd).double()
    # the probabilities are fp32 with a few roundings each, relative 64 u at most
    assert torch.allclose(r.log_prob.double(), p.gather(1, labels[:, None])[:, 0].log(), atol=64 * U) and torch.allclose(r.entropy.double(), -(p * p.log()).sum(1), atol=5 * 64 * U)
    assert torch.allclose(r.top_log_prob.double(), p.topk(2, 1).values.log(), atol=64 * U)
    with pytest.raises(TypeError):
        bst.predict_log_probs(X)
    binary = fb.train({"objective": "binary", "num_leaves": 7, "device_type": "cuda", "verbosity": -1}, fb.Dataset(X, (y > 2).astype("float32")), 2)
    with pytest.raises(fb.FalcataError):
        binary.predict_log_probs(Xd)


def test_custom_objective_from_class_log_probs():
    """The training scores that a custom objective sees are class-major; the gradient goes back without a copy."""
    import falcata_b200 as fb
    from falcata_b200 import ops
    from util import make_multiclass
    X, y = make_multiclass(n=2000, f=10, k=3)
    labels = torch.from_numpy(y).cuda().int()
    seen = []

    def objective(scores, train):
        r = ops.class_log_probs(scores, labels)
        grad = ops.class_log_probs_grad(scores, r.log_norm, r.entropy, labels=labels, grad_log_prob=torch.full_like(r.log_prob, -1.0))
        p = torch.exp(scores - r.log_norm[:, None])
        seen.append((grad, p - torch.nn.functional.one_hot(labels.long(), 3)))
        assert grad.t().is_contiguous()
        return grad.t(), (1.5 * p * (1 - p)).t().contiguous()

    params = {"num_class": 3, "num_leaves": 7, "device_type": "cuda", "verbosity": -1}
    mine = fb.Booster(dict(params, objective="none"), fb.Dataset(X, y))
    theirs = fb.Booster(dict(params, objective="multiclass", boost_from_average=False), fb.Dataset(X, y))
    for _ in range(3):
        mine.update(fobj=objective); theirs.update()
    for grad, want in seen:
        assert torch.allclose(grad, want, atol=64 * U)
    Xd = torch.from_numpy(X).cuda()
    assert torch.allclose(mine.predict(Xd, raw_score=True), theirs.predict(Xd, raw_score=True), atol=1e-4)


def test_operators_in_a_graph_and_on_streams():
    """Captured and replayed on new inputs, two graphs and an eager call side by side on two streams: the same results."""
    g = _gen(11)
    def inputs(seed):
        g.manual_seed(seed)
        return (torch.randn((500, 36), generator=g, device="cuda", requires_grad=True), torch.randn((9, 300, 36), generator=g, device="cuda", requires_grad=True), _leaves(500, 9, seed),
                torch.randint(0, 300, (500,), generator=g, device="cuda"))
    sets = [inputs(i) for i in range(3)]
    want = [_head_step(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    captured = []
    for st in streams:
        buf = tuple(t.detach().clone().requires_grad_(t.requires_grad) for t in sets[0])
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            _head_step(*buf)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = _head_step(*buf)
        captured.append((graph, buf, out))
    torch.cuda.synchronize()
    for (graph, buf, out), src in zip(captured, sets[1:]):
        with torch.no_grad():
            for b, s in zip(buf, src):
                b.copy_(s)
    torch.cuda.synchronize()
    for rep in range(3):
        for st, (graph, _, _) in zip(streams, captured):
            with torch.cuda.stream(st):
                graph.replay()
        eager = _head_step(*sets[0])
        torch.cuda.synchronize()
        for got, ref in ((captured[0][2], want[1]), (captured[1][2], want[2]), (eager, want[0])):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


# ------------------------------------------------------------------------------- scores of large magnitude ----
def _large_scores(k, dtype, layout, value, seed):
    """Rows around `value` a few steps of the type apart, rows of one value, and ordinary rows with classes masked by -|value|."""
    g = _gen(seed)
    steps = torch.randint(0, 6, (18, k), generator=g, device="cuda").double()
    s = value * (1 + torch.finfo(dtype).eps * steps)
    usual = torch.randn((18, k), generator=g, device="cuda").double() * 2.5
    mask = -abs(value)
    s[8] = value
    s[9] = value; s[9, k // 2] = value + abs(value) / 2
    s[10] = usual[10]; s[10, : 3 * k // 4] = mask          # runs, as a padded class list has them
    s[11] = usual[11]; s[11, k // 4:] = mask
    s[12] = usual[12]; s[12, 1::2] = mask
    s[13] = mask; s[13, k - 1] = 1.5
    s[14] = mask
    s[15] = usual[15]; s[15, 0] = abs(value)
    s[16] = -math.inf; s[16, k // 3] = value; s[16, k // 2] = mask
    s[17] = torch.where(steps[17] < 2, mask, usual[17])
    s = s.to(dtype)
    return s.t().contiguous().t() if layout == "class" else s


def _check_large(s, top):
    """log p = (s_j - m) - log sum e^(s - m): s_j - m rounds by u of its size, the sum as for any scores; nothing grows with |m|."""
    from falcata_b200 import ops
    n, k = s.shape
    labels = torch.randint(0, k, (n,), generator=_gen(1), device="cuda")
    got = ops.class_log_probs(s, labels, top_k=top)
    want, logp = _reference(s, labels, top)
    tol = U * (k / 32 + 128)
    assert torch.equal(got.top_class, want["top_class"])
    for name, scale in (("log_prob", 1.0), ("top_log_prob", 1.0), ("entropy", 1 + math.log(k)), ("log_norm", 1.0)):
        off = (getattr(got, name).double() - want[name]).abs() / (tol * scale + 4 * U * want[name].abs())
        assert bool((off.nan_to_num(math.inf) <= 1)[torch.isfinite(want[name])].all()), (name, off)
        assert torch.equal(getattr(got, name)[~torch.isfinite(want[name])].double(), want[name][~torch.isfinite(want[name])])
    g = torch.full((n,), 0.5, device="cuda"); g_top = torch.full((n, top), 0.125, device="cuda")
    grad = ops.class_log_probs_grad(s, got.log_norm, got.entropy, labels=labels, top_class=got.top_class, grad_log_prob=2 * g, grad_log_norm=g, grad_entropy=-g / 2, grad_top_log_prob=g_top).double()
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, 0.0)
    named = (want["top_class"] >= 0)
    ref = p * (0.5 - 1.0 - 0.125 * named.sum(1, keepdim=True)) + 0.25 * (plogp + p * want["entropy"][:, None])
    ref[torch.arange(n, device="cuda"), labels] += 1.0
    ref.scatter_add_(1, want["top_class"].long().clamp(min=0), torch.where(named, 0.125, 0.0).double())
    # |a| + |b| (|log p| + entropy) is at most 6 + log K, p's own error U (K / 32 + 128) + 4 U |log p|
    bound = p * (6 + math.log(k)) * (U * (k / 32 + 128) + 8 * U * (16 + logp.abs().clamp(max=200))) + 32 * U + _half_step(s.dtype) * ref.abs()
    assert bool(((grad - ref).abs() <= bound).all()), float(((grad - ref).abs() - bound).max())


LARGE_ROWS = [("row", 10), ("row", 60), ("row", 300), ("row", 5000), ("row", 40000), ("class", 10), ("class", 100), ("class", 2000), ("class", 20000)]


@pytest.mark.parametrize("layout,k", LARGE_ROWS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [1e8, -1e8, 3e9, 5e9, -5e9, 1e10, -1e10, 1e15, 1e20, -1e20, 1e30, -1e30, 7e35, -7e35])
def test_class_log_probs_of_large_scores(layout, k, dtype, value):
    """Scores far from zero that are no powers of two, and classes masked by a large finite value."""
    _check_large(_large_scores(k, dtype, layout, value, seed=k), min(k, 20))


@pytest.mark.parametrize("layout,k", LARGE_ROWS)
@pytest.mark.parametrize("border", [2.0 ** exponent * sign for exponent in (20, 22, 23, 24, 25) for sign in (1, -1)])
def test_class_log_probs_around_powers_of_two(layout, k, border):
    """fp32 scores on both sides of a power of two, a few steps apart: parts of one row whose maxima lie on different sides."""
    step = max(1.0, abs(border) * 2.0 ** -24)
    s = (border + step * torch.randint(-5, 6, (18, k), generator=_gen(k), device="cuda").double()).float()
    _check_large(s.t().contiguous().t() if layout == "class" else s, min(k, 20))


@pytest.mark.parametrize("k", [257, 8200])
def test_class_log_probs_more_alternatives_than_32_bits_count(k):
    """Rows x alternatives beyond 2^32: every window of one long vector is a row, so a result at a wrapped place is another row's."""
    from falcata_b200 import ops
    n, top = (1 << 27) + 5, 32
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    values = torch.randn(n + k, generator=_gen(k), device="cuda", dtype=torch.bfloat16)
    got = ops.class_log_probs(values.as_strided((n, k), (1, 1)), top_k=top)
    for first in (0, n // 2, n - 8):
        want, _ = _reference(values[first:].as_strided((8, k), (1, 1)), None, top)
        assert torch.equal(got.top_class[first:first + 8], want["top_class"])
        for name in ("log_norm", "entropy", "top_log_prob"):
            assert torch.allclose(getattr(got, name)[first:first + 8].double(), want[name], rtol=U, atol=U * (k / 32 + 128) * (1 + math.log(k)))
    del got
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------ waits that run out ----
class _WaitTries:
    """The tensor-core kernel's waits give up after so many tries (each some microseconds); as at first again at the end."""

    def __init__(self, tries):
        self.tries = tries

    def _set(self, tries):
        import ctypes
        from falcata_b200.basic import _lib
        before = ctypes.c_int(0)
        assert _lib().FB_OpLeafWaitTries(ctypes.c_int(tries), ctypes.byref(before)) == 0

    def __enter__(self):
        self._set(self.tries)

    def __exit__(self, *exc):
        torch.cuda.synchronize()
        self._set(0)


def _near_or_nan(got, want, size, terms, dtype):
    """Where it is not NaN: as _near."""
    given = ~torch.isnan(got)
    _near(torch.where(given, got, want.to(dtype)), want, size, terms, dtype)
    return given


@pytest.mark.parametrize("side", ["tma", "x copied", "maps copied", "maps by output"])
@pytest.mark.parametrize("tries", [1, 2, 6])
def test_leaf_products_whose_waits_run_out(side, tries):
    """Several tiles per block, each longer than a try: what is not finished is NaN, never what an accumulator happened to hold."""
    from falcata_b200 import ops
    n, f, k, leaves = 128 * 148 * 5, 2048, 96, 3
    g = _gen(2)
    x = torch.randn((n, f + 1), generator=g, device="cuda", dtype=torch.bfloat16)
    x = x[:, 1:] if side == "x copied" else x[:, :f].contiguous()
    w = torch.randn((leaves, k, f + (1 if side == "maps copied" else 0)), generator=g, device="cuda", dtype=torch.bfloat16)[:, :, :f]
    if side == "maps by output":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    begin = torch.tensor([0, n // 3, n // 2, n], device="cuda")
    want, size = _ref_products(x, w, begin)
    with _WaitTries(tries):
        given = _near_or_nan(ops.leaf_products(x, w, begin), want, size, f, torch.bfloat16)
        assert tries > 1 or not bool(given.any())          # every block's first tile takes longer than one try
    _near(ops.leaf_products(x, w, begin), want, size, f, torch.bfloat16)


@pytest.mark.parametrize("side", ["tma", "copied"])
@pytest.mark.parametrize("tries", [1, 2, 6])
def test_leaf_gram_whose_waits_run_out(side, tries):
    """Slices that end inside a step, for which all copying warps come together: a role that leaves takes its whole warp along."""
    from falcata_b200 import ops
    n, ac, bc = 150003, 264, 120 if side == "copied" else 520
    g = _gen(3)
    a = torch.randn((n, ac + 1), generator=g, device="cuda", dtype=torch.float16)
    a = a[:, :ac].contiguous() if side == "tma" else a[:, 1:]
    b = torch.randn((n, bc), generator=g, device="cuda", dtype=torch.float16)
    begin = torch.tensor([0, 5, 40001, 40001, 41007, 100000, n], device="cuda")
    at = list(zip(begin.tolist()[:-1], begin.tolist()[1:]))
    want = torch.stack([a[lo:hi].double().t() @ b[lo:hi].double() for lo, hi in at])
    size = torch.stack([a[lo:hi].double().abs().t() @ b[lo:hi].double().abs() for lo, hi in at])
    with _WaitTries(tries):
        for dtype in (torch.float32, torch.float16):
            given = _near_or_nan(ops.leaf_gram(a, b, begin, dtype=dtype), want, size, n, dtype)
            assert bool(given[2].all())                        # no rows, nothing to wait for
    for dtype in (torch.float32, torch.float16):
        _near(ops.leaf_gram(a, b, begin, dtype=dtype), want, size, n, dtype)


# ------------------------------------------------------------------------- many leaves, boundaries that fall ----
def _check_leaves(x, w, d, begin, begin_given=None):
    """Products, transposed products and Gram sums of rows that lie leaf by leaf; rows outside the leaves are zero."""
    from falcata_b200 import ops
    dtype, (n, f), (leaves, k) = x.dtype, x.shape, w.shape[:2]
    b = begin.long()
    row = torch.arange(n, device="cuda")
    leaf = torch.searchsorted(b, row, right=True) - 1
    there = ((leaf >= 0) & (leaf < leaves)).double()[:, None]
    leaf = leaf.clamp(0, leaves - 1)
    given = begin if begin_given is None else begin_given

    def products(a, m):
        parts = [(torch.einsum("nf,nkf->nk", a[i:i + 4096].double(), m[leaf[i:i + 4096]].double()), torch.einsum("nf,nkf->nk", a[i:i + 4096].double().abs(), m[leaf[i:i + 4096]].double().abs())) for i in range(0, n, 4096)]
        return torch.cat([p[0] for p in parts]) * there, torch.cat([p[1] for p in parts]) * there

    want, size = products(x, w)
    y = ops.leaf_products(x, w, given)
    _near(y, want, size, f, dtype)
    assert bool((y[there[:, 0] == 0] == 0).all())
    want, size = products(d, w.transpose(1, 2))
    _near(ops.leaf_products(d, w.transpose(1, 2), given), want, size, k, dtype)
    if begin_given is not None:
        return
    want, size = torch.zeros((leaves, k, f), dtype=torch.float64, device="cuda"), torch.zeros((leaves, k, f), dtype=torch.float64, device="cuda")
    for i in range(0, n, 2048):
        outer = torch.einsum("nk,nf->nkf", d[i:i + 2048].double(), x[i:i + 2048].double()) * there[i:i + 2048, :, None]
        want.index_add_(0, leaf[i:i + 2048], outer); size.index_add_(0, leaf[i:i + 2048], outer.abs())
    for out in {dtype, torch.float32}:
        p = ops.leaf_gram(d, x, given, dtype=out)
        _near(p, want, size, int((b[1:] - b[:-1]).max()), out)
        assert torch.equal(p, ops.leaf_gram(d, x, given, dtype=out))


def _many_leaves(leaves, n, long_leaf, seed):
    """Boundaries of leaves of which many are empty, one is long, and some rows lie before the first and behind the last."""
    g = torch.Generator(); g.manual_seed(seed)
    size = torch.randint(0, 4, (leaves,), generator=g) * (torch.rand(leaves, generator=g) < 0.6)
    size[leaves // 3: leaves // 3 + 70] = 0                    # a run of empty ones, across spans
    size[leaves // 2] = long_leaf
    begin = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(size, 0)]) + 7
    assert int(begin[-1]) + 5 <= n
    return begin.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("leaves,f,k,long_leaf", [(1024, 9, 5, 700), (1025, 9, 5, 700), (3000, 12, 7, 6000), (5000, 28, 10, 300), (1025, 70, 50, 600), (3000, 40, 33, 3000), (2049, 130, 40, 5000), (1500, 48, 200, 2500)])
def test_more_leaves_than_spans(dtype, leaves, f, k, long_leaf):
    """More leaves than the tile map has places: several per place, looked up leaf by leaf."""
    n = 2 * leaves + long_leaf + 400
    g = _gen(leaves)
    begin = _many_leaves(leaves, n, long_leaf, seed=f)
    x, d = torch.randn((n, f), generator=g, device="cuda").to(dtype), torch.randn((n, k), generator=g, device="cuda").to(dtype)
    w = torch.randn((leaves, k, f), generator=g, device="cuda").mul(f ** -0.5).to(dtype)
    _check_leaves(x, w, d, begin.int() if leaves % 2 else begin)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("leaves,f,k", [(9, 9, 5), (9, 70, 50), (9, 130, 140), (2600, 9, 5), (2600, 70, 50)])
def test_leaf_products_of_falling_boundaries(dtype, leaves, f, k):
    """A row that several leaves claim belongs to the first of them; the others' rows are what they would be anyway."""
    g = _gen(f)
    n = 4 * leaves + 900
    given = _many_leaves(leaves, n, 500, seed=k)
    given[leaves // 4] = n - 11; given[leaves // 4 + 1] = 3      # up and down again
    given[1::7] -= 20
    begin = torch.cummax(given.clamp(0, n), 0).values
    x, d = torch.randn((n, f), generator=g, device="cuda").to(dtype), torch.randn((n, k), generator=g, device="cuda").to(dtype)
    w = torch.randn((leaves, k, f), generator=g, device="cuda").mul(f ** -0.5).to(dtype)
    _check_leaves(x, w, d, begin, given)
    from falcata_b200 import ops
    assert ops.leaf_gram(d, x, given).shape == (leaves, k, f)


@pytest.mark.parametrize("f,k", [(4, 2), (40, 36)])
@pytest.mark.parametrize("dtype", TYPES)
def test_leaf_products_of_all_rows_claimed_over_and_over(dtype, f, k):
    """As many leaves as would make more tiles than 31 bits count if each had the rows that it claims."""
    from falcata_b200 import ops
    n, leaves = 1 << 20, 300_001
    g = _gen(f)
    given = torch.zeros(leaves + 1, dtype=torch.int32, device="cuda"); given[1::2] = n
    x = torch.randn((n, f), generator=g, device="cuda").to(dtype); w = torch.randn((1, k, f), generator=g, device="cuda").to(dtype)
    y = ops.leaf_products(x, w.expand(leaves, k, f), given)
    _near(y, x.double() @ w[0].double().t(), x.double().abs() @ w[0].double().abs().t(), f, dtype)
    assert ops.leaf_gram(x[:, :1], x[:, :2], given).shape == (leaves, 1, 2)


# ------------------------------------------------------------------------------- the booster's calls on streams ----
def _late(values, big):
    """`values`, written by the current stream only after a while of other work."""
    x = torch.full_like(values, math.nan)
    for _ in range(4):
        big = big @ big
    return x.copy_(torch.where(big[0, 0].isnan(), values, values))


def test_booster_predictions_on_a_side_stream():
    """Rows that the caller's stream is still to write, results whose memory it has used before: as on the default stream."""
    import falcata_b200 as fb
    from util import make_multiclass
    X, y = make_multiclass(n=20000, f=8, k=5)
    bst = fb.train({"objective": "multiclass", "num_class": 5, "num_leaves": 15, "device_type": "cuda", "verbosity": -1}, fb.Dataset(X, y), 3)
    Xd, labels = torch.from_numpy(X).float().cuda(), torch.from_numpy(y).cuda().long()
    big = torch.randn((4096, 4096), generator=_gen(1), device="cuda").mul_(1e-3)
    rows = [Xd.roll(i, 0).contiguous() for i in range(8)]
    want = [(bst.predict_log_probs(r, labels, top_k=2), bst.predict(r), bst.predict(r, pred_leaf=True)) for r in rows]
    torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    for _ in range(2):
        for r in rows:
            with torch.cuda.stream(side):
                a = bst.predict_log_probs(_late(r, big), labels, top_k=2)
                b = bst.predict(_late(r, big))
                got.append((a, b, bst.predict(_late(r, big), pred_leaf=True)))
    torch.cuda.synchronize()
    for (a, b, c), (u, v, w) in zip(got, want + want):
        assert all(torch.equal(p, q) for p, q in zip(a, u)) and torch.equal(b, v) and torch.equal(c, w)
    for empty in (Xd[:0],):
        r = bst.predict_log_probs(empty, labels[:0], top_k=2)
        assert r.log_prob.shape == (0,) and r.top_class.shape == (0, 2)


def test_custom_objective_on_a_side_stream():
    """Gradients that the caller's stream is still to write when the booster takes them: the same model as on the default stream.

    The booster adds fp32 gradients in any order, so that two trainings on one stream differ in the last bits. Multiples of 1/64 up to
    1 in size add up exactly (20000 of them stay below 2^24 / 64), and equal sums give equal models."""
    import falcata_b200 as fb
    from falcata_b200 import ops
    from util import make_multiclass
    X, y = make_multiclass(n=20000, f=10, k=3)
    labels = torch.from_numpy(y).cuda().int()
    big = torch.randn((4096, 4096), generator=_gen(1), device="cuda").mul_(1e-3)

    def train(stream):
        def objective(scores, _):
            r = ops.class_log_probs(scores, labels)
            grad = ops.class_log_probs_grad(scores, r.log_norm, r.entropy, labels=labels, grad_log_prob=torch.full_like(r.log_prob, -1.0))
            p = torch.exp(scores - r.log_norm[:, None])
            return _late((grad * 64).round().div(64).t(), big), _late((96 * p * (1 - p)).round().add(1).div(64).t().contiguous(), big)

        bst = fb.Booster({"num_class": 3, "num_leaves": 7, "device_type": "cuda", "verbosity": -1, "objective": "none"}, fb.Dataset(X, y))
        with torch.cuda.stream(stream):
            for _ in range(4):
                bst.update(fobj=objective)
        torch.cuda.synchronize()
        return bst.model_to_string()

    assert train(torch.cuda.Stream()) == train(torch.cuda.default_stream())


def test_results_without_a_derivative_say_so():
    """A backward pass through a Gram sum or a gradient raises where it would have lost a derivative; their values are as ever."""
    from falcata_b200 import ops
    x, d = (torch.randn((50, 6), generator=_gen(i), device="cuda") for i in range(2))
    begin = torch.tensor([0, 20, 50], device="cuda")
    plain = ops.leaf_gram(d, x, begin)
    assert not plain.requires_grad
    p = ops.leaf_gram(d, x.clone().requires_grad_(), begin)
    assert torch.equal(p, plain)
    with pytest.raises(NotImplementedError, match="leaf_gram"):
        p.sum().backward()
    f = ops.class_log_probs(x)
    z = x.clone().requires_grad_()
    g = ops.class_log_probs_grad(z, f.log_norm, f.entropy, grad_entropy=torch.ones(50, device="cuda"))
    assert torch.equal(g, ops.class_log_probs_grad(x, f.log_norm, f.entropy, grad_entropy=torch.ones(50, device="cuda")))
    with pytest.raises(NotImplementedError, match="class_log_probs_grad"):
        (g * z).sum().backward()
    with torch.no_grad():
        assert not ops.leaf_gram(d, z, begin).requires_grad
    for transform in (lambda s: torch.func.jvp(lambda t: ops.class_log_probs(t).entropy, (s,), (torch.ones_like(s),)), lambda s: torch.func.grad(lambda t: ops.class_log_probs(t).entropy.sum())(s),
                      lambda s: torch.func.vmap(lambda t: ops.class_log_probs(t).entropy)(s.reshape(5, 10, 6))):
        with pytest.raises((NotImplementedError, RuntimeError)):
            transform(x)


@pytest.mark.parametrize("n,k", [(3, 60000), (19000, 60000), (40, 500), (40, 20000)])
@pytest.mark.parametrize("step", [0.37, 0.61, 5.3])
@pytest.mark.parametrize("shift", [0.0, 1000.0, 1e8])
def test_class_log_probs_of_many_equal_terms(n, k, step, shift):
    """Equal terms that fp32 does not hold exactly, where every rounding of a long sum goes the same way: sums must not run on in one
    thread. (Classes far apart in memory, one vector for all rows, the highest scores where each thread starts.)"""
    from falcata_b200 import ops
    values = torch.full((k,), shift, device="cuda")
    if shift == 1e8:
        values[:64] += 8.0
    else:
        values[:64] += step
    s = torch.stack([values, values], 1).reshape(-1).as_strided((n, k), (0, 2))
    logp = (values.double() - torch.logsumexp(values.double() - shift, 0)) - shift
    want = {"log_norm": torch.logsumexp(values.double() - shift, 0) + shift, "entropy": -(logp.exp() * logp).sum()}
    got = ops.class_log_probs(s)
    tol = U * (k / 32 + 128)
    for name, w in want.items():
        off = (getattr(got, name).double() - w).abs() - 2 * U * w.abs()
        assert bool((off <= tol * (1 + math.log(k) * (name == "entropy"))).all()), (name, float(off.max()), tol)
    if n * k > 10 ** 8:
        return
    grad = ops.class_log_probs_grad(s, got.log_norm, got.entropy, labels=torch.zeros(n, dtype=torch.int32, device="cuda"), grad_log_prob=torch.ones(n, device="cuda")).double()
    ref = -logp.exp().expand(n, k).clone()
    ref[:, 0] += 1
    bound = logp.exp() * (U * (k / 32 + 256) + 8 * U * (16 + logp.abs())) + 4 * U * ref.abs()
    assert bool(((grad - ref).abs() <= bound).all()), float(((grad - ref).abs() / bound).max())
