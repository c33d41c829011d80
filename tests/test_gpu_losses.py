"""Cross entropy and distillation of an output projection against the formulas in 64 bits.

Tolerances count roundings.  A logit is a sum of D exact products in fp32, whose
additions may each cut 2^-23 of the running sum: ds = D 2^-23 sum_d |h_d w_d|
bounds its error, and a loss is off by at most 2 ds and a few roundings of lse.
G is rounded to bf16 (2^-8, half a step) and its exponentials carry the logits'
errors, the products sum in fp32, and the gradients are rounded to bf16."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = torch.bfloat16
H8 = 2.0 ** -8


def _problem(N, V, D, seed, cuda, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * scale / D ** 0.5).to(BF).to(cuda)
    h = (torch.randn(N, D, generator=g) * 2).to(BF).to(cuda)
    return g, h, w


def _ds(h, w):
    D = h.shape[1]
    return (h.double().norm(dim=1) * w.double().norm(dim=1).max()) * D * 2.0 ** -23      # >= D 2^-23 sum |h_d w_d|


def _formula(h, w, idx, prob, ok, coef, T):
    """64-bit loss rows and gradients for sparse targets (N, K); coef is dloss of each row."""
    h, w = h.double(), w.double()
    s = h @ w.T / T
    lse = torch.logsumexp(s, -1)
    st = s.gather(1, idx)
    ent = torch.where(prob > 0, prob * prob.clamp(min=1e-300).log(), torch.zeros_like(prob))
    loss = T * T * (ent + torch.where(prob > 0, prob * (lse[:, None] - st), torch.zeros_like(prob))).sum(-1)
    loss = torch.where(ok, loss, torch.zeros_like(loss))
    c = (coef.double() * ok * T)[:, None]
    q = (s - lse[:, None]).exp()
    p = torch.zeros_like(q).scatter_add_(1, idx, prob)
    return loss, lse, (c * (q - p)), c.abs() * (q + p)


def _check(got_loss, got_dh, got_dw, h, w, idx, prob, ok, coef, T, reduction, g_err=H8):
    ds = _ds(h, w) / T
    loss, lse, G, A = _formula(h, w, idx, prob, ok, coef, T)
    n = max(1, int(ok.sum()))
    ltol = T * T * (2 * ds + 8 * U * (lse.abs() + 16)) * ok
    if reduction == "none":
        assert ((got_loss.double() - loss).abs() <= ltol + U * loss.abs()).all()
    else:
        k = n if reduction == "mean" else 1
        assert abs(got_loss.item() - (loss.sum() / k).item()) <= (ltol.sum() / k + 2 * U * loss.sum().abs() / k).item()
    if got_dh is None:
        return
    hd, wd = h.double(), w.double()
    dsr = (3 * ds + 8 * U * (lse.abs() + 4))[:, None]
    for got, ref, gabs, aabs, depth in (
            (got_dh, G @ wd, G.abs() @ wd.abs(), (dsr * A) @ wd.abs(), w.shape[0]),
            (got_dw, G.T @ hd, G.abs().T @ hd.abs(), (dsr * A).T @ hd.abs(), h.shape[0])):
        tol = (g_err + depth * 2.0 ** -23) * gabs + aabs
        tol = tol + H8 * (ref.abs() + tol) + 1e-37
        bad = (got.double() - ref).abs() > tol
        assert not bad.any(), f"{int(bad.sum())} outside, worst {((got.double() - ref).abs() / tol).max():.3g} of the bound"


def _xent(lh, h, w, target, reduction, dloss=None, ignore_index=-100):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = lh.linear_cross_entropy(h, w, target, ignore_index=ignore_index, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), dloss)
    return loss.detach(), dh, dw


def _run_xent(lh, cuda, N, V, D, reduction, seed=0, ignore=0.0, scale=1.0):
    g, h, w = _problem(N, V, D, seed, cuda, scale)
    target = torch.randint(0, V, (N,), generator=g)
    if ignore:
        target[torch.rand(N, generator=g) < ignore] = -100
    target = target.to(cuda)
    ok = target != -100
    dloss = torch.randn(N, generator=g).to(cuda) if reduction == "none" else torch.tensor(1.5, device=cuda)
    loss, dh, dw = _xent(lh, h, w, target, reduction, dloss)
    coef = dloss if reduction == "none" else dloss / (max(1, int(ok.sum())) if reduction == "mean" else 1)
    coef = coef.expand(N)
    _check(loss, dh, dw, h, w, target.clamp(min=0)[:, None], ok.double()[:, None], ok, coef, 1.0, reduction)
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("N,V,D", [(1, 1, 8), (1, 256, 64), (2, 257, 72), (31, 255, 128), (128, 1000, 64),
                                   (129, 300, 264), (255, 256, 256), (257, 511, 768), (300, 5003, 96),
                                   (1000, 769, 136), (64, 2, 4096), (7, 20011, 1024), (64, 777, 200), (65, 777, 200),
                                   (33, 40001, 520), (50, 256, 1032)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cross_entropy(lh, cuda, N, V, D, reduction):
    _run_xent(lh, cuda, N, V, D, reduction, seed=N + V)


@pytest.mark.parametrize("ignore", [0.3, 0.97])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_with_ignored_positions(lh, cuda, ignore, reduction):
    _run_xent(lh, cuda, 333, 1031, 160, reduction, seed=5, ignore=ignore)


@pytest.mark.parametrize("N,V,D", [(20000, 256, 256), (3, 131072, 64), (70000, 17, 64)])
def test_long_sums_are_split(lh, cuda, N, V, D):
    """Few tiles and a long K: dW over 20000 positions, dH over 131072 columns."""
    _run_xent(lh, cuda, N, V, D, "mean", seed=9)


def test_several_pieces_of_the_vocabulary(lh, cuda):
    """5000 x 120001: three pieces, the last one ragged; dH sums over all."""
    _run_xent(lh, cuda, 5000, 120001, 64, "mean", seed=11)


# 2 N V D >= 5e10 and more than 256 positions: the rows that count are packed
BIG = (1000, 50001, 512)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("ignore", [0.0, 0.4, 0.95])
def test_packed_positions(lh, cuda, ignore, reduction):
    _run_xent(lh, cuda, *BIG, reduction, seed=40, ignore=ignore)


@pytest.mark.parametrize("live", [0, 1, 64, 256, 257, 999])
def test_packed_positions_at_the_edges(lh, cuda, live):
    """A given number of positions with a target, the others' hidden rows holding NaN."""
    N, V, D = BIG
    g, h, w = _problem(N, V, D, 41, cuda)
    target = torch.randint(0, V, (N,), generator=g).to(cuda)
    keep = torch.zeros(N, dtype=torch.bool)
    keep[torch.randperm(N, generator=g)[:live]] = True
    keep = keep.to(cuda)
    target[~keep] = -100
    h[~keep] = float("nan")
    loss, dh, dw = _xent(lh, h, w, target, "mean")
    clean = torch.where(keep[:, None], h, torch.zeros_like(h))
    _check(loss, dh, dw, clean, w, target.clamp(min=0)[:, None], keep.double()[:, None], keep,
           torch.full((N,), 1.0 / max(1, live), device=cuda), 1.0, "mean")
    assert (dh[~keep] == 0).all()
    none = lh.linear_cross_entropy(h, w, target, reduction="none")
    assert (none[~keep] == 0).all() and none.isfinite().all()
    assert lh._native.device_status() == 0


def test_packed_long_product_is_split_by_what_is_left(lh, cuda):
    """Five row blocks of which two are left, a product over 60000 columns in parts."""
    _run_xent(lh, cuda, 1200, 60000, 512, "mean", seed=42, ignore=0.65)


def test_peaked_and_large_logits(lh, cuda):
    _run_xent(lh, cuda, 200, 700, 64, "mean", seed=12, scale=40.0)


def test_every_position_ignored(lh, cuda):
    _, h, w = _problem(70, 300, 64, 1, cuda)
    target = torch.full((70,), -100, device=cuda)
    for red in ("mean", "sum"):
        loss, dh, dw = _xent(lh, h, w, target, red)
        assert loss.item() == 0 and (dh == 0).all() and (dw == 0).all()
    loss = lh.linear_cross_entropy(h, w, target, reduction="none")
    assert (loss == 0).all()


def test_ignored_positions_may_hold_anything(lh, cuda):
    """A finite loss and finite dhidden whatever an ignored position's hidden row holds."""
    g, h, w = _problem(40, 300, 64, 2, cuda)
    target = torch.randint(0, 300, (40,), generator=g).to(cuda)
    target[3] = target[17] = -100
    h2 = h.clone()
    h2[3], h2[17, 5] = float("nan"), float("inf")
    a, b = _xent(lh, h, w, target, "mean"), _xent(lh, h2, w, target, "mean")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (b[1][3] == 0).all() and (b[1][17] == 0).all()


@pytest.mark.parametrize("N,V,D", [(40, 300, 64), (64, 20000, 128), (300, 1000, 72), (700, 90, 264), (20000, 256, 64)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_what_an_ignored_position_holds_reaches_no_gradient(lh, cuda, N, V, D, reduction):
    """NaN and infinities in ignored rows against zeros there: the same loss, dhidden and dweight."""
    g, h, w = _problem(N, V, D, 50, cuda)
    target = torch.randint(0, V, (N,), generator=g)
    target[torch.rand(N, generator=g) < 0.3] = -100
    target[-1] = -100
    off = (target == -100).to(cuda)
    target = target.to(cuda)
    dloss = torch.randn(N, generator=g).to(cuda) if reduction == "none" else None
    zeros, odd = torch.where(off[:, None], 0, h), h.clone()
    a = _xent(lh, zeros, w, target, reduction, dloss)
    for x, at in ((float("nan"), slice(None)), (float("inf"), slice(D - 1, D)), (-float("inf"), slice(0, 1))):
        odd[:, at] = torch.where(off[:, None], x, h[:, at])
        b = _xent(lh, odd, w, target, reduction, dloss)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        odd = h.clone()
    # one row alone
    odd[-1] = float("nan")
    assert all(torch.equal(p, q) for p, q in zip(a, _xent(lh, odd, w, target, reduction, dloss)))
    tv = torch.randn(N, 5, generator=g).to(cuda)
    ti = torch.randint(0, V, (N, 5), generator=g).to(cuda)
    ti[off] = -1
    res = []
    for x in (zeros, torch.where(off[:, None], float("nan"), h)):
        ls = [t.detach().requires_grad_(True) for t in (x, w)]
        loss = lh.linear_distillation(*ls, tv, ti, reduction=reduction)
        res.append((loss.detach(), *torch.autograd.grad(loss, ls, dloss)))
    assert all(torch.equal(p, q) for p, q in zip(*res)) and res[0][2].isfinite().all()


@pytest.mark.parametrize("N,V,D", [(16, 20000, 128), (300, 1000, 72), (2000, 24000, 640)])
def test_one_gradient_of_two(lh, cuda, N, V, D):
    """A frozen projection, or hidden states that need no gradient: the other one is the same."""
    g, h, w = _problem(N, V, D, 51, cuda)
    target = torch.randint(0, V, (N,), generator=g).to(cuda)
    tv, ti = torch.randn(N, 3, generator=g).to(cuda), torch.randint(0, V, (N, 3), generator=g).to(cuda)
    for f in (lambda a, b: lh.linear_cross_entropy(a, b, target), lambda a, b: lh.linear_distillation(a, b, tv, ti)):
        leaf = lambda t: t.detach().requires_grad_(True)
        a, b = leaf(h), leaf(w)
        both = torch.autograd.grad(f(a, b), (a, b))
        a = leaf(h)
        assert torch.equal(torch.autograd.grad(f(a, w), a)[0], both[0])
        b = leaf(w)
        assert torch.equal(torch.autograd.grad(f(h, b), b)[0], both[1])
        a, b = leaf(h), leaf(w)
        assert torch.equal(torch.autograd.grad(f(a, b), b)[0], both[1]), "the graph has both, the call asks for one"


def test_another_ignore_index_and_bad_targets(lh, cuda):
    g, h, w = _problem(20, 300, 64, 3, cuda)
    target = torch.randint(0, 300, (20,), generator=g).to(cuda)
    target[4] = 7
    loss = lh.linear_cross_entropy(h, w, target, ignore_index=7, reduction="none")
    assert loss[4] == 0 and loss.isfinite().all()
    for bad in (300, -1, -100, 1 << 40, -(1 << 40)):
        t = target.clone()
        t[9] = bad
        loss = lh.linear_cross_entropy(h, w, t, ignore_index=7, reduction="none")
        assert loss[9].isnan() and loss.isnan().sum() == 1
        assert lh.linear_cross_entropy(h, w, t, ignore_index=7).isnan()
    # a bad position without an upstream gradient spoils nothing
    t[9] = 300
    dl = torch.ones(20, device=cuda)
    dl[9] = 0
    _, dh, dw = _xent(lh, h, w, t, "none", dl, ignore_index=7)
    assert dh.isfinite().all() and dw.isfinite().all() and (dh[9] == 0).all()


def test_infinite_and_nan_logits(lh, cuda):
    """As torch's cross entropy: -inf logits drop out, +inf and NaN give NaN."""
    g, h, w = _problem(4, 600, 64, 4, cuda)
    h = h.abs() + 0.1
    target = torch.tensor([1, 2, 3, 4], device=cuda)
    for v, want in ((-float("inf"), False), (float("inf"), True), (float("nan"), True)):
        w2 = w.clone()
        w2[500] = v
        loss = lh.linear_cross_entropy(h, w2, target, reduction="none")
        ref = torch.nn.functional.cross_entropy(h.double() @ w2.double().T, target, reduction="none")
        assert bool(loss.isnan().all()) is want and bool(ref.isnan().all()) is want
        if not want:
            assert (loss.double() - ref).abs().max() <= 1e-5 * ref.max()


# --------------------------------------------------------------------------- distillation
def _teacher(g, N, V, K, where="spread"):
    hi = V if where == "spread" else min(V, max(K, 200))
    ti = torch.stack([torch.randperm(hi, generator=g)[:K] for _ in range(N)])
    return torch.randn(N, K, generator=g) * 3, ti


def _probs(tv, ti, T):
    here = ti >= 0
    ok = (here & (tv > -float("inf"))).any(-1)
    x = (tv.double() / T).masked_fill(~here, -float("inf"))
    p = torch.zeros_like(x)
    p[ok] = torch.softmax(x[ok], -1)
    return p, ok


def _run_distill(lh, cuda, N, V, D, K, T, reduction, seed=0, empty=0.0, where="spread", tdt=torch.float32,
                 idt=torch.int64, edit=None):
    g, h, w = _problem(N, V, D, seed, cuda)
    tv, ti = _teacher(g, N, V, K, where)
    if empty:
        ti[torch.rand(N, generator=g) < empty] = -1
    if edit:
        edit(tv, ti)
    tv, ti = tv.to(tdt).to(cuda), ti.to(cuda)
    p, ok = _probs(tv, ti, T)
    h1, w1 = h.requires_grad_(True), w.requires_grad_(True)
    loss = lh.linear_distillation(h1, w1, tv, ti.to(idt), temperature=T, reduction=reduction)
    dloss = torch.randn(N, generator=g).to(cuda) if reduction == "none" else torch.tensor(0.7, device=cuda)
    dh, dw = torch.autograd.grad(loss, (h1, w1), dloss)
    coef = dloss if reduction == "none" else dloss / (max(1, int(ok.sum())) if reduction == "mean" else 1)
    # the probabilities carry fp32 roundings of a softmax over K: inside the logits' bound
    with torch.no_grad():
        _check(loss.detach(), dh, dw, h, w, ti.clamp(min=0), p, ok, coef.expand(N), T, reduction)
    assert lh._native.device_status() == 0
    return loss.detach(), dh, dw


@pytest.mark.parametrize("N,V,D,K,T", [(1, 1, 8, 1, 1.0), (2, 300, 64, 5, 1.0), (33, 256, 128, 16, 2.0),
                                       (130, 1000, 72, 64, 1.5), (257, 5003, 96, 13, 4.0), (20, 700, 64, 256, 2.0),
                                       (500, 257, 64, 3, 0.5), (6, 20011, 1024, 128, 1.0)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_distillation(lh, cuda, N, V, D, K, T, reduction):
    _run_distill(lh, cuda, N, V, D, K, T, reduction, seed=N + K)


@pytest.mark.parametrize("where", ["spread", "front"])
def test_distillation_types_empty_rows_and_crowded_tiles(lh, cuda, where):
    _run_distill(lh, cuda, 150, 3000, 64, 100, 2.0, "mean", seed=21, empty=0.3, where=where, tdt=BF, idt=torch.int32)
    _run_distill(lh, cuda, 150, 3000, 64, 100, 2.0, "sum", seed=22, empty=0.9, where=where)
    _run_distill(lh, cuda, 60, 3000, 136, 256, 2.0, "none", seed=45, empty=0.2, where=where)


def test_distillation_packed(lh, cuda):
    _run_distill(lh, cuda, *BIG, 20, 2.0, "mean", seed=43, empty=0.5)
    _run_distill(lh, cuda, *BIG, 3, 1.0, "none", seed=44, empty=0.2)


def test_distillation_absent_entries_and_minus_infinity(lh, cuda):
    def edit(tv, ti):
        ti[0, ::2] = -1
        ti[1, 1:] = -5
        tv[2, 3] = -float("inf")
        tv[3, :] = -float("inf")                     # an empty row, by its logits
        tv[4, 0] = 1e4                               # one entry takes all
    loss, dh, _ = _run_distill(lh, cuda, 10, 700, 64, 7, 1.0, "none", seed=23, edit=edit)
    assert loss[3] == 0 and (dh[3] == 0).all()


def test_distillation_same_index_twice(lh, cuda):
    def edit(tv, ti):
        ti[0, :] = ti[0, 0]
        ti[1, 3] = ti[1, 0]
        ti[2, 5] = ti[2, 6]
    _run_distill(lh, cuda, 9, 700, 64, 7, 2.0, "mean", seed=24, edit=edit)


def test_distillation_bad_teachers(lh, cuda):
    g, h, w = _problem(6, 300, 64, 25, cuda)
    tv, ti = (t.to(cuda) for t in _teacher(g, 6, 300, 4))
    tv[1, 2], tv[3, 0] = float("nan"), float("inf")
    ti[4, 1] = 300
    loss = lh.linear_distillation(h, w, tv, ti, reduction="none")
    assert loss.isnan().tolist() == [False, True, False, True, True, False]


def test_distillation_from_one_certain_entry_is_cross_entropy(lh, cuda):
    g, h, w = _problem(100, 900, 128, 26, cuda)
    t = torch.randint(0, 900, (100,), generator=g).to(cuda)
    a = _xent(lh, h, w, t, "mean")
    h1, w1 = h.requires_grad_(True), w.requires_grad_(True)
    loss = lh.linear_distillation(h1, w1, torch.zeros(100, 1, device=cuda), t[:, None])
    b = torch.autograd.grad(loss, (h1, w1))
    assert abs(loss.item() - a[0].item()) <= 4 * U * (abs(a[0].item()) + 10)
    assert torch.equal(a[1], b[0]) and torch.equal(a[2], b[1])


# --------------------------------------------------------------------------- rows of one tile
ONE_TILE = [(65, 1, 8), (66, 17, 64), (300, 128, 72), (513, 129, 128), (1000, 200, 264), (20001, 256, 64), (260, 256, 4096)]


@pytest.mark.parametrize("N,V,D", ONE_TILE)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_rows_of_one_tile(lh, cuda, N, V, D, reduction):
    """The forward leaves the logits' gradients: more tiles than pairs of SMs, ragged rows and columns."""
    for ignore in (0.0, 0.4):
        _run_xent(lh, cuda, N, V, D, reduction, seed=60, ignore=ignore)
    if V > 1:
        def edit(tv, ti):
            ti[::7, 0] = ti[::7, -1]                 # the same index twice
            ti[3::11] = -1
        _run_distill(lh, cuda, N, V, D, min(V, 9), 2.0, reduction, seed=61, empty=0.2, edit=edit)
    _run_distill(lh, cuda, N, V, D, min(V, 100), 0.7, reduction, seed=62)


def test_rows_of_one_tile_packed(lh, cuda):
    _run_xent(lh, cuda, 100000, 256, 1024, "mean", seed=63, ignore=0.3)
    _run_distill(lh, cuda, 100000, 250, 1024, 5, 2.0, "sum", seed=64, empty=0.99)
    h, w = torch.randn(100000, 1024, device=cuda).to(BF), torch.randn(256, 1024, device=cuda).to(BF)
    loss, dh, dw = _xent(lh, h, w, torch.full((100000,), -100, device=cuda), "mean")
    assert loss == 0 and (dh == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("N,V", [(300, 200), (300, 967), (40, 967)])
def test_upstream_gradients_of_a_reduced_loss(lh, cuda, N, V):
    """Zero, negative and large upstream gradients, one after the other from the same graph, and a bad target."""
    g, h, w = _problem(N, V, 64, 65, cuda)
    t = torch.randint(0, V, (N,), generator=g).to(cuda)
    h1, w1 = h.requires_grad_(True), w.requires_grad_(True)
    loss = lh.linear_cross_entropy(h1, w1, t)
    one = torch.autograd.grad(loss, (h1, w1), retain_graph=True)
    for f in (-4.0, 2.0 ** 40, 2.0 ** -20):          # powers of two: bit for bit
        got = torch.autograd.grad(loss, (h1, w1), torch.tensor(f, device=cuda), retain_graph=True)
        assert all(torch.equal(a, b * f) for a, b in zip(got, one))
    t2 = t.clone()
    t2[5] = V
    loss = lh.linear_cross_entropy(h1, w1, t2)
    assert loss.isnan()
    got = torch.autograd.grad(loss, (h1, w1), torch.zeros((), device=cuda), retain_graph=True)
    assert all((x == 0).all() for x in got)
    dh, dw = torch.autograd.grad(loss, (h1, w1))
    assert dh[5].isnan().all() and dw.isnan().all()
    # without the forward's gradients (reduction "none"): the same up to one rounding more or less
    none = torch.autograd.grad(lh.linear_cross_entropy(h1, w1, t, reduction="none").mean(), (h1, w1))
    for a, b in zip(one, none):
        assert (a.double() - b.double()).norm() <= 2 * H8 * b.double().norm()


# --------------------------------------------------------------------------- both
def test_gradients_against_differences(lh, cuda):
    """Central differences of the 64-bit formulas at a few coordinates; G's bf16 bounds the gradients."""
    g, h, w = _problem(5, 40, 64, 30, cuda)
    tv, ti = (t.to(cuda) for t in _teacher(g, 5, 40, 4))
    t = torch.randint(0, 40, (5,), generator=g).to(cuda)
    p, ok = _probs(tv, ti, 2.0)

    def xent(hh, ww):
        return torch.nn.functional.cross_entropy(hh @ ww.T, t)

    def dist(hh, ww):
        lq = torch.log_softmax(hh @ ww.T / 2.0, -1).gather(1, ti)
        return 4 * (p * (p.log() - lq)).sum(-1).mean()

    h1, w1 = h.requires_grad_(True), w.requires_grad_(True)
    for own, f in ((lambda: lh.linear_cross_entropy(h1, w1, t), xent),
                   (lambda: lh.linear_distillation(h1, w1, tv, ti, temperature=2.0), dist)):
        grads = torch.autograd.grad(own(), (h1, w1))
        vals = [h.detach().double(), w.detach().double()]
        for k in range(2):
            scale = grads[k].float().abs().max().item()
            for pos in (0, 77, 319):
                d = torch.zeros_like(vals[k])
                d.view(-1)[pos] = 1e-5
                up, dn = list(vals), list(vals)
                up[k], dn[k] = vals[k] + d, vals[k] - d
                diff = (f(*up) - f(*dn)).item() / 2e-5
                assert abs(diff - grads[k].view(-1)[pos].item()) <= 2 * H8 * scale + H8 * abs(diff) + 1e-6


def test_no_positions(lh, cuda):
    h = torch.zeros(0, 64, dtype=BF, device=cuda, requires_grad=True)
    w = torch.randn(50, 64, device=cuda).to(BF).requires_grad_(True)
    t = torch.zeros(0, dtype=torch.int64, device=cuda)
    for red in ("mean", "sum"):
        loss = lh.linear_cross_entropy(h, w, t, reduction=red)
        dh, dw = torch.autograd.grad(loss, (h, w))
        assert loss.item() == 0 and dh.shape == (0, 64) and (dw == 0).all()
    assert lh.linear_cross_entropy(h, w, t, reduction="none").shape == (0,)
    assert lh.linear_distillation(h, w, torch.zeros(0, 3, device=cuda), torch.zeros(0, 3, dtype=torch.int64,
                                                                                   device=cuda)).item() == 0


def test_strides_alignment_and_leading_dimensions(lh, cuda):
    g = torch.Generator().manual_seed(31)
    big = torch.randn(4, 6, 128, generator=g).to(BF).to(cuda)
    h = big[:, ::2, 64:]
    flat = torch.randn(300 * 64 + 1, generator=g).to(BF).to(cuda)
    w = flat[1:].view(300, 64)
    t = torch.randint(0, 300, (3, 4), generator=g).to(cuda).T           # (4, 3), strided
    a = lh.linear_cross_entropy(h, w, t, reduction="none")
    b = lh.linear_cross_entropy(h.reshape(12, 64).clone(), w.clone(), t.reshape(12).to(torch.int32), reduction="none")
    assert a.shape == (4, 3) and torch.equal(a.reshape(12), b)
    wt = torch.randn(64, 300, generator=g).to(BF).to(cuda).T             # column-major weights
    assert torch.equal(lh.linear_cross_entropy(h, wt, t), lh.linear_cross_entropy(h, wt.contiguous(), t))


def test_same_results_every_time_on_a_stream_and_in_a_graph(lh, cuda):
    g, h, w = _problem(600, 3001, 256, 32, cuda)
    t = torch.randint(0, 3001, (600,), generator=g).to(cuda)
    tv, ti = (x.to(cuda) for x in _teacher(g, 600, 3001, 20))

    def both():
        h1, w1 = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        a = lh.linear_cross_entropy(h1, w1, t)
        out = [a.detach(), *torch.autograd.grad(a, (h1, w1))]
        b = lh.linear_distillation(h1, w1, tv, ti, temperature=2.0)
        return out + [b.detach(), *torch.autograd.grad(b, (h1, w1))]

    want = [x.clone() for x in both()]
    assert all(torch.equal(a, b) for a, b in zip(want, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    here = both()                                      # the same calls on two streams at once
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(torch.equal(a, b) for a, b in zip(want, here))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    h.copy_(torch.randn_like(h))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(both(), out)) and not torch.equal(want[0], out[0])
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("N,V,D", [(1, 1355, 1400), (1, 9, 8), (8, 300, 64), (31, 20000, 136), (32, 5003, 512)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradients_of_few_rows_have_two_terms(lh, cuda, N, V, D, reduction):
    """Up to 32 rows the logits' gradients are held in two bf16 terms, off by 2^-16 at most."""
    g, h, w = _problem(N, V, D, 72, cuda)
    t = torch.randint(0, V, (N,), generator=g)
    t[N // 2:N // 2 + N // 4] = -100
    t = t.to(cuda)
    ok = t != -100
    odd = torch.where(ok[:, None], h, float("nan"))
    dloss = torch.randn(N, generator=g).to(cuda) if reduction == "none" else None
    coef = dloss if reduction == "none" else torch.full((N,), 1.0 / int(ok.sum()), device=cuda)
    res = [_xent(lh, x, w, t, reduction, dloss) for x in (h, odd)]
    assert all(torch.equal(a, b) for a, b in zip(*res))
    _check(*res[0], h, w, t.clamp(min=0)[:, None], ok.double()[:, None], ok, coef, 1.0, reduction, g_err=2.0 ** -16)
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("V", [8, 64, 300])
def test_offsets_past_32_bits(lh, cuda, V):
    """Hidden states of 2.2e9 elements, of which the last rows count (not packed, packed, more than one tile)."""
    N, D, n = 270000, 8192, 500
    g, last, w = _problem(n, V, D, 71, cuda)
    h = torch.full((N, D), float("nan"), dtype=BF, device=cuda)
    h[-n:] = last
    target = torch.full((N,), -100, device=cuda)
    t = target[-n:] = torch.randint(0, V, (n,), generator=g).to(cuda)
    loss, dh, dw = _xent(lh, h, w, target, "mean")
    assert all((c == 0).all() for c in dh[:-n].split(50000))
    one = torch.ones(n, 1, dtype=torch.float64, device=cuda)
    _check(loss, dh[-n:], dw, last, w, t[:, None], one, one[:, 0] > 0, torch.full((n,), 1.0 / n, device=cuda), 1.0, "mean")
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("N,V,D", [(600, 200, 64), (40, 3001, 64), (300, 3001, 64), BIG])
def test_a_replayed_graph_follows_its_inputs(lh, cuda, N, V, D):
    """Other hidden states, targets and numbers of ignored positions, whose rows hold NaN, in every replay."""
    g, h, w = _problem(N, V, D, 70, cuda)
    t = torch.randint(0, V, (N,), generator=g).to(cuda)
    tv, ti = torch.randn(N, 6, generator=g).to(cuda), torch.randint(0, V, (N, 6), generator=g).to(cuda)

    def both():
        h1, w1 = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        a = lh.linear_cross_entropy(h1, w1, t)
        out = [a.detach(), *torch.autograd.grad(a, (h1, w1))]
        b = lh.linear_distillation(h1, w1, tv, ti, reduction="sum")
        return out + [b.detach(), *torch.autograd.grad(b, (h1, w1))]

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for share in (0.0, 0.5, 0.98, 0.2, 1.0, 0.0):
        off = (torch.rand(N, generator=g) < share).to(cuda)
        t.copy_(torch.randint(0, V, (N,), generator=g))
        ti.copy_(torch.randint(0, V, (N, 6), generator=g))
        t[off], ti[off] = -100, -1
        h.copy_((torch.randn(N, D, generator=g) * 2).to(BF))
        h[off] = float("nan")
        graph.replay()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(want, out)) and all(x.isfinite().all() for x in out)
    assert lh._native.device_status() == 0


def test_opcheck(lh, cuda):
    ops = torch.ops.lighthouse_b200
    utils = ("test_schema", "test_faketensor")
    g, h, w = _problem(40, 300, 64, 33, cuda)
    t = torch.randint(0, 300, (40,), generator=g).to(cuda)
    tv, ti = (x.to(cuda) for x in _teacher(g, 40, 300, 5))
    for red in ("mean", "none"):
        torch.library.opcheck(ops.linear_xent, (h, w, t, -100, red), test_utils=utils)
        loss, kept = ops.linear_xent(h, w, t, -100, red)
        torch.library.opcheck(ops.linear_xent_bwd, (h, w, t, kept, torch.ones_like(loss), red), test_utils=utils)
        torch.library.opcheck(ops.linear_distill, (h, w, tv, ti, 2.0, red), test_utils=utils)
        loss, kept = ops.linear_distill(h, w, tv, ti, 2.0, red)
        torch.library.opcheck(ops.linear_distill_bwd, (h, w, kept, torch.ones_like(loss), 5, 2.0, red), test_utils=utils)


@pytest.mark.parametrize("N,V", [(9, 300), (9, 15001), (9, 20000), (80, 200), (80, 5003), (80, 15001), (80, 20000)])
@pytest.mark.parametrize("top", [20.625, 90.5])
def test_one_large_logit_per_row(lh, cuda, N, V, top):
    """Logits that fp32 holds, one of them far above the others.

    Of the steps to a loss, the exponent of the largest logit is taken from its exact product with log2(e)
    less that product's rounding; ex2 is off by 2 ulp, a sum near one passes at most 4 joins in its tile,
    4 adds of 32 values each, and 24 joins of parts (2^-24 each): under 64 U.  log2(e) and ln 2 are off by
    U each, so are the two products and a sum of losses at its end: 6 U of the loss."""
    g = torch.Generator().manual_seed(N + V)
    big = torch.randint(0, V, (N,), generator=g)
    h = torch.zeros(N, 88)
    h[:, :8] = torch.randint(0, 4, (N, 8), generator=g).float()
    w = torch.zeros(V, 88)
    w[:, :8] = torch.randint(-2, 3, (V, 8), generator=g).float() / 8
    # channel 8 + n of row n takes its large logit to `top`, which is one of a row of its own there
    n = torch.arange(N)
    h[n, 8 + n] = 1.0
    w[big] = 0
    w[big, 8 + n] = top
    h, w = h.to(BF).to(cuda), w.to(BF).to(cuda)
    s = h.double() @ w.double().T
    lse = torch.logsumexp(s, -1)
    for t in (s.argmax(-1), s.argmin(-1)):
        for red in ("none", "sum"):                   # "sum" of one-tile rows: the forward's gradients
            loss, dh, dw = _xent(lh, h, w, t, red, torch.ones(N, device=cuda) if red == "none" else None)
            want = lse - s.gather(1, t[:, None])[:, 0]
            tol = 64 * U + 6 * U * want
            got = loss.double()
            assert (got >= 0).all()
            assert ((got - (want if red == "none" else want.sum())).abs() <= (tol if red == "none" else tol.sum())).all()
            # gradients of the same accuracy: an exponential carries the rounding of lse (U of it, and of log2(e)),
            # the target's entry those of the loss; what is below 2^-126 may be cut
            q, one = (s - lse[:, None]).exp(), torch.nn.functional.one_hot(t, V).double()
            G = q - one
            E = H8 * G.abs() + (64 * U + 2 * U * lse.abs()[:, None]) * q + 64 * U * one + 2.0 ** -126
            hd, wd = h.double(), w.double()
            for got, ref, err, sums in ((dh, G @ wd, E @ wd.abs(), V * 2.0 ** -23 * (G.abs() @ wd.abs())),
                                        (dw, G.T @ hd, E.T @ hd.abs(), N * 2.0 ** -23 * (G.abs().T @ hd.abs()))):
                tol = err + sums
                assert ((got.double() - ref).abs() <= tol + H8 * (ref.abs() + tol)).all()
    loss = lh.linear_distillation(h, w, torch.ones(N, 1, device=cuda), s.argmax(-1)[:, None], reduction="none")
    assert ((loss.double() - (lse - s.amax(-1))).abs() <= 64 * U).all()


@pytest.mark.parametrize("N,V", [(9, 300), (9, 20000), (80, 200), (80, 300), (80, 20000)])
@pytest.mark.parametrize("D", [520, 4096, 65536])
def test_exact_logits_of_long_rows(lh, cuda, N, V, D):
    """A few products per row that fp32 adds exactly, wherever in the row they are: no logit may be off.

    The tolerance is that of one large logit per row: 64 U, and 6 U of the loss."""
    g = torch.Generator().manual_seed(D + V)
    at = torch.randperm(D, generator=g)[:24]
    h, w = torch.zeros(N, D, dtype=BF), torch.zeros(V, D, dtype=BF)
    h[:, at] = torch.randint(-3, 4, (N, 24), generator=g).to(BF)
    w[:, at] = (torch.randint(-8, 9, (V, 24), generator=g) / 8).to(BF)
    h, w = h.to(cuda), w.to(cuda)
    s = h[:, at.to(cuda)].double() @ w[:, at.to(cuda)].double().T
    lse = torch.logsumexp(s, -1)
    t = torch.randint(0, V, (N,), generator=g).to(cuda)
    for target in (t, s.argmax(-1)):
        want = lse - s.gather(1, target[:, None])[:, 0]
        loss = lh.linear_cross_entropy(h, w, target, reduction="none").double()
        assert ((loss - want).abs() <= 64 * U + 6 * U * want).all()
        loss = lh.linear_distillation(h, w, torch.zeros(N, 1, device=cuda), target[:, None], reduction="none").double()
        assert ((loss - want).abs() <= 64 * U + 6 * U * want).all()
        assert abs(lh.linear_cross_entropy(h, w, target).item() - want.mean().item()) <= 64 * U + 8 * U * want.mean().item()
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("N,V", [(50, 5003), (256, 250), (256, 5003), (256, 20001)])
@pytest.mark.parametrize("kind", ["even", "first", "last"])
def test_sums_of_logits_are_not_cut(lh, cuda, N, V, kind):
    """The mean error of the losses over rows of 16384 products, whose large ones lie anywhere, first or last.

    A part of a sum has 24 steps of 16 products.  A step cuts half an ulp on average, U of what the part has so
    far, which grows to the part's own sum: 12 U of the parts' sums, 12 U of a logit, in the target's and in the
    others' mean under the softmax.  Roundings to nearest do not add up; 16 U is for those of lse."""
    D = 16384
    g = torch.Generator(device=cuda).manual_seed(N + V)
    size = torch.full((D,), 0.3, device=cuda)
    if kind == "even":
        size[:] = 1
    else:
        size[:D // 64] = 8
    if kind == "last":
        size = size.flip(0)
    h = torch.randn(N, D, generator=g, device=cuda) * size
    w = torch.randn(V, D, generator=g, device=cuda) * 1.5 / D ** 0.5
    t = torch.randperm(V, generator=g, device=cuda)[:N] if N <= V else torch.randint(0, V, (N,), generator=g, device=cuda)
    w.index_add_(0, t, h * (4 / h.square().sum(1, keepdim=True)))
    h, w = h.to(BF), w.to(BF)
    s = h.double() @ w.double().T
    lse = torch.logsumexp(s, -1)
    st = s.gather(1, t[:, None])[:, 0]
    loss = lh.linear_cross_entropy(h, w, t, reduction="none").double()
    bound = 12 * U * (st.abs() + ((s - lse[:, None]).exp() * s.abs()).sum(-1)).mean() + 16 * U
    assert abs((loss - (lse - st)).mean()) <= bound


@pytest.fixture
def gave_up(lh, cuda):
    """Sets the losses' status flag from the host, as a wait that gives up would; clears it in the end."""
    assert lh._native.device_status() == 0
    yield lambda: lh._native.load().lh_device_status(-1)
    lh._native.device_status()
    assert lh._native.device_status() == 0


@pytest.mark.parametrize("N,V,D", [(16, 300, 64), (16, 20000, 512), (60, 3001, 64), (300, 200, 64), (300, 3001, 72),
                                   (20000, 17, 64), (5000, 120001, 64), BIG])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("loss_kind", ["xent", "distill"])
def test_a_wait_that_gave_up_shows_in_losses_and_gradients(lh, cuda, gave_up, N, V, D, reduction, loss_kind):
    """NaN in the place of what memory held before: few rows, one tile, parts and pieces of dH and dW, packed rows."""
    g, h, w = _problem(N, V, D, 80, cuda)
    t = torch.randint(0, V, (N,), generator=g)
    t[::3] = -100
    counts = (t != -100).to(cuda)
    tv, ti = torch.randn(N, 1, generator=g).to(cuda), t.clamp(min=-1)[:, None].to(cuda)
    t = t.to(cuda)
    h, w = h.requires_grad_(True), w.requires_grad_(True)

    def forward():
        if loss_kind == "xent":
            return lh.linear_cross_entropy(h, w, t, reduction=reduction)
        return lh.linear_distillation(h, w, tv, ti, reduction=reduction)

    def backward(loss):
        return torch.autograd.grad(loss, (h, w), torch.ones_like(loss), retain_graph=True)

    good = forward()
    want = [x.clone() for x in (good.detach(), *backward(good))]
    gave_up()
    dh, dw = backward(good)                              # of a sound forward
    assert dw.isnan().all() and dh[counts].isnan().all()
    bad = forward()
    assert (bad[counts] if reduction == "none" else bad).isnan().all()
    dh, dw = backward(bad)
    assert dw.isnan().all() and dh[counts].isnan().all()
    assert lh._native.device_status() == 1               # cleared; what the forward kept is no less lost
    dh, dw = backward(bad)
    assert dw.isnan().all() and dh[counts].isnan().all()
    again = forward()
    assert all(torch.equal(a, b) for a, b in zip(want, (again.detach(), *backward(again))))


def test_compiled_with_any_number_of_positions(lh, cuda):
    """One graph for several numbers of positions, the results of the eager calls."""
    g, h, w = _problem(400, 300, 64, 81, cuda)
    t = torch.randint(0, 300, (400,), generator=g).to(cuda)
    tv, ti = (x.to(cuda) for x in _teacher(g, 400, 300, 5))

    def f(h, w, t, tv, ti):
        return lh.linear_cross_entropy(h, w, t), lh.linear_distillation(h, w, tv, ti)

    torch._dynamo.reset()
    fn = torch.compile(f, fullgraph=True, backend="aot_eager")
    for n in (20, 65, 400):
        res = []
        for call in (fn, f):
            ls = [h[:n].detach().requires_grad_(True), w.detach().requires_grad_(True)]
            args = (t[:n], tv[:n], ti[:n])
            for x in (ls[0], *args):
                torch._dynamo.mark_dynamic(x, 0)
            loss = call(*ls, *args)
            res.append([x.detach() for x in loss] + list(torch.autograd.grad(loss[0] + loss[1], ls)))
        assert all(torch.equal(a, b) for a, b in zip(*res))


# N x V x D in several pieces of the vocabulary, positions packed: 5000 x 120001 in three of 40192 columns, the last
# one shorter; 40000 x 7001 in two of 3584, more row blocks than the table of parts has
PIECES = [(5000, 120001, 64, 40192), (40000, 7001, 96, 3584)]


@pytest.mark.parametrize("N,V,D,C", PIECES)
@pytest.mark.parametrize("ignore", [0.4, 0.97])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_several_pieces_with_packed_positions(lh, cuda, N, V, D, C, ignore, reduction):
    _run_xent(lh, cuda, N, V, D, reduction, seed=82, ignore=ignore)


@pytest.mark.parametrize("N,V,D,C", PIECES)
@pytest.mark.parametrize("empty", [0.0, 0.3, 0.97])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_distillation_over_several_pieces(lh, cuda, N, V, D, C, empty, reduction):
    """Teacher entries on both sides of every border of the pieces, beside others."""
    border = [i for b in range(C, V, C) for i in (b - 2, b - 1, b, b + 1)]

    def edit(tv, ti):
        some = ti[:, 0] >= 0
        for k, i in enumerate(border):
            rows = some.clone()
            rows[k % 3::3] = False                       # not all of them in every row
            taken = (ti == i).any(1)
            ti[rows & ~taken, k] = i
        ti[::5, 9] = torch.where(some[::5], ti[::5, 1], -1)      # the same entry twice

    _run_distill(lh, cuda, N, V, D, 13, 2.0, reduction, seed=83, empty=empty, edit=edit)
