"""The residual RMS norm against a plain implementation in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32.  A thread sums 32
squares in order and a row's sum passes ten more additions, so the mean square is
off by at most 42 u, its root by half of that; the root's own error, the product
with the weight and the two products before it add a few u: 32 u bounds y's
relative error before it is rounded to its type, which adds finfo.eps / 2."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def _half(t):
    return torch.finfo(t).eps / 2


def _inputs(N, D, xd, rd, wd, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, D, generator=g).to(xd).to(cuda)
    r = None if rd is None else (3 * torch.randn(N, D, generator=g)).to(rd).to(cuda)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(wd).to(cuda)
    return x, r, w


def _ref(x, r, w, eps=1e-5):
    h = x.double() if r is None else (x.double() + r.double()).to(r.dtype).double()
    rstd = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, rstd, h * rstd * w.double()


def _assert_within(a, ref, tol, what):
    bad = (a.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {((a.double() - ref).abs() / tol.clamp_min(1e-300)).max():.3g}"


SHAPES = [(1, 8), (3, 136), (17, 1024), (5, 1032), (9, 4096), (300, 264), (2, 16384), (33, 2560)]
TYPES = [(BF, F32, F32, BF), (BF, BF, BF, BF), (F32, F32, F32, F32), (BF, None, F32, BF), (F32, None, BF, BF),
         (F32, BF, F32, F32), (BF, BF, F32, F32)]


@pytest.mark.parametrize("N,D", SHAPES)
@pytest.mark.parametrize("xd,rd,wd,yd", TYPES)
def test_forward_and_gradients(lh, cuda, N, D, xd, rd, wd, yd):
    x, r, w = _inputs(N, D, xd, rd, wd, N * 7 + D, cuda)
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(N, D, generator=g).to(yd).to(cuda)
    dh = None if rd is None else torch.randn(N, D, generator=g).to(rd).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    if r is None:
        y = lh.rms_norm(x, w, out_dtype=yd)
        grads = torch.autograd.grad(y, leaves, dy)
    else:
        y, h = lh.add_rms_norm(x, r, w, out_dtype=yd)
        grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    with torch.no_grad():
        h64, rstd, y64 = _ref(x, r, w)
        if r is not None:
            assert torch.equal(h.double(), h64), "the stored stream is x + r rounded once"
        assert y.dtype == yd
        _assert_within(y, y64, (_half(yd) + 32 * U) * y64.abs() + 1e-30, "y")
        n, gg = h64 * rstd, dy.double() * w.double()
        m = (gg * n).mean(-1, keepdim=True)
        d64 = rstd * (gg - n * m) + (0 if dh is None else dh.double())
        # n carries 32 u, the mean of g n 42 u of its absolute terms more, the rest a few roundings
        err = rstd * U * (40 * gg.abs() + n.abs() * (80 * m.abs() + 120 * (gg * n).abs().mean(-1, keepdim=True)))
        if dh is not None:
            err = err + 2 * U * dh.double().abs()
        _assert_within(grads[0], d64, err + _half(xd) * (d64.abs() + err), "dx")
        if r is not None:
            _assert_within(grads[1], d64, err + _half(rd) * (d64.abs() + err), "dresidual")
        dw64 = (dy.double() * n).sum(0)
        err = U * (N + 64) * (dy.double() * n).abs().sum(0)
        _assert_within(grads[-1], dw64, err + _half(wd) * (dw64.abs() + err), "dweight")
        assert [t.dtype for t in grads] == [t.dtype for t in leaves]


@pytest.mark.parametrize("N,D,group", [(1, 8, 0), (4, 200, 128), (7, 1024, 128), (3, 4096, 0), (5, 1160, 128),
                                       (2, 16384, 128), (65, 256, 0)])
@pytest.mark.parametrize("rd", [None, BF])
def test_fp8_codes_and_scales(lh, cuda, N, D, group, rd):
    """bf16 factors: t = h w and 448 t are exact in fp32 (8 + 8 + 3 significant bits), so the codes
    equal those of exact arithmetic rounded to nearest even."""
    x, r, w = _inputs(N, D, BF, rd, BF, N + D, cuda)
    x[0, : min(D, 128)] = 0                     # a group of zeros (the whole row where D is small)
    if r is not None:
        r[0, : min(D, 128)] = 0
        q, s, h = lh.add_rms_norm_fp8(x, r, w, group=group)
        assert torch.equal(h, (x.double() + r.double()).to(BF))
    else:
        q, s = lh.rms_norm_fp8(x, w, group=group)
    h64, rstd, _ = _ref(x, r, w)
    t = h64 * w.double()
    step = group or D
    for gi, lo in enumerate(range(0, D, step)):
        tt = t[:, lo:lo + step]
        a = tt.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
        want = (tt * 448 / a).float().to(torch.float8_e4m3fn)
        assert torch.equal(q[:, lo:lo + step].float(), want.float())
        sc = (a * rstd / 448).squeeze(-1)
        _assert_within(s[:, gi], sc, 32 * U * sc, "scale")
    assert s.shape == (N, -(-D // group) if group else 1)


@pytest.mark.parametrize("D", [256, 4096])
def test_rows_of_zeros_infinities_and_nan(lh, cuda, D):
    x = torch.randn(6, D, device=cuda)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 1e-30
    w = torch.ones(D, device=cuda)
    y, h = lh.add_rms_norm(x, torch.zeros_like(x), w)
    assert torch.equal(h.nan_to_num(7.0), x.nan_to_num(7.0))
    assert (y[0] == 0).all()
    assert y[1, 3].isnan() and (y[1, :3] == 0).all(), "an infinity's row: rstd is 0"
    assert y[2].isnan().all()
    assert torch.allclose(y[3], torch.full_like(y[3], 1e-30 / 1e-5 ** 0.5), rtol=1e-5, atol=0)
    assert y[4:].isfinite().all()
    q, s = lh.rms_norm_fp8(x.to(BF), w)
    deq = q.float() * s
    assert (deq[0] == 0).all() and s[0].isfinite().all()
    assert deq[1].isnan().all() and deq[2].isnan().all() and deq[4:].isfinite().all()


def test_gradient_against_differences(lh, cuda):
    """Central differences in 64 bits of the plain norm, at a few coordinates of each input."""
    x, r, w = _inputs(4, 64, F32, F32, F32, 3, cuda)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    c1, c2 = torch.randn(4, 64, device=cuda), torch.randn(4, 64, device=cuda)
    y, h = lh.add_rms_norm(x, r, w)
    grads = torch.autograd.grad((y * c1).sum() + (h * c2).sum(), leaves)

    def f(a, b, c):
        hh = a + b
        return ((hh / (hh.square().mean(-1, keepdim=True) + 1e-5).sqrt() * c) * c1.double()).sum() + (hh * c2.double()).sum()

    vals = [t.detach().double() for t in leaves]
    for k in range(3):
        for pos in (0, 17, 63):
            d = torch.zeros_like(vals[k])
            d.view(-1)[pos] = 1e-4
            up, dn = list(vals), list(vals)
            up[k], dn[k] = vals[k] + d, vals[k] - d
            diff = (f(*up) - f(*dn)) / 2e-4
            # the difference's own error is of order 1e-8; fp32 gradients of sums of about 64 terms: 1e-4
            assert abs(diff.item() - grads[k].view(-1)[pos].item()) < 1e-4 * (1 + abs(diff.item()))


def test_strided_and_misaligned_inputs_and_leading_dimensions(lh, cuda):
    g = torch.Generator().manual_seed(5)
    big = torch.randn(4, 6, 3 * 64, generator=g).to(BF).to(cuda)
    x = big[:, ::2, 64:128]                                      # strided view
    flat = torch.randn(4 * 3 * 64 + 1, generator=g).to(BF).to(cuda)
    r = flat[1:].view(4, 3, 64)                                  # 2-byte offset
    w = torch.randn(64, generator=g).to(cuda)
    y, h = lh.add_rms_norm(x, r, w)
    y2, h2 = lh.add_rms_norm(x.contiguous(), r.clone(), w)
    assert y.shape == x.shape and torch.equal(y, y2) and torch.equal(h, h2)
    h64, _, y64 = _ref(x, r, w)
    _assert_within(y, y64, (_half(BF) + 32 * U) * y64.abs() + 1e-30, "y")


def test_no_rows(lh, cuda):
    x = torch.zeros(0, 3, 64, dtype=BF, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    y, h = lh.add_rms_norm(x, x.detach(), w)
    assert y.shape == h.shape == (0, 3, 64)
    dx, dw = torch.autograd.grad(y.float().sum() + h.float().sum(), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()
    q, s = lh.rms_norm_fp8(x.detach(), w.detach(), group=128)
    assert q.shape == (0, 3, 64) and s.shape == (0, 3, 1)


def test_unused_outputs(lh, cuda):
    x, r, w = _inputs(8, 256, BF, F32, F32, 4, cuda)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = lh.add_rms_norm(x, r, w)
    dx, dr, dw = torch.autograd.grad(h, leaves, torch.ones_like(h), allow_unused=True)
    assert (dx == 1).all() and dx.dtype == BF and (dr == 1).all() and dw is None
    y, h = lh.add_rms_norm(x, r, w)
    dy = torch.randn_like(y)
    a = torch.autograd.grad(y, leaves, dy)
    y, h = lh.add_rms_norm(x, r, w)
    b = torch.autograd.grad((y, h), leaves, (dy, torch.zeros_like(h)))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_same_results_every_time_on_a_stream_and_in_a_graph(lh, cuda):
    N, D = 3001, 1024
    x, r, w = _inputs(N, D, BF, F32, F32, 6, cuda)
    dy, dh = torch.randn(N, D, device=cuda).to(BF), torch.randn(N, D, device=cuda)

    def fwd_bwd():
        ls = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, h = lh.add_rms_norm(*ls)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), ls, (dy, dh)))

    want = [t.clone() for t in fwd_bwd()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fwd_bwd()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fwd_bwd()
    x2 = torch.randn_like(x)
    for t, v in ((x, x2), (x, x2)):
        t.copy_(v)
        graph.replay()
    torch.cuda.synchronize()
    ref = fwd_bwd()
    assert all(torch.equal(a, b) for a, b in zip(ref, out))
    assert not torch.equal(want[0], out[0])


def test_opcheck(lh, cuda):
    ops = torch.ops.lighthouse_b200
    U_ = ("test_schema", "test_faketensor")
    x, r, w = _inputs(6, 136, BF, F32, F32, 8, cuda)
    for args in ((ops.rms_norm, (x, w, 1e-5, BF)), (ops.add_rms_norm, (x, r, w, 1e-5, BF)),
                 (ops.rms_norm_fp8, (x, w, 1e-5, 128)), (ops.add_rms_norm_fp8, (x, r, w, 1e-5, 0))):
        torch.library.opcheck(*args, test_utils=U_)
    y, h, rstd = ops.add_rms_norm(x, r, w, 1e-5, BF)
    torch.library.opcheck(ops.add_rms_norm_bwd, (y, h, h, w, rstd, BF), test_utils=U_)
    torch.library.opcheck(ops.add_rms_norm_bwd, (y, None, h, w, rstd, BF), test_utils=U_)
    torch.library.opcheck(ops.rms_norm_bwd, (y, x, w, rstd), test_utils=U_)


@pytest.mark.parametrize("N,D", [(270000, 8192), (11000000, 200)])
def test_offsets_past_32_bits(lh, cuda, N, D):
    """The last rows of 2.2e9 elements: what a call with those rows alone gives."""
    n = 300
    x, r, w = _inputs(n, D, BF, BF, F32, 5, cuda)
    dy = torch.randn(n, D, generator=torch.Generator().manual_seed(2)).to(BF).to(cuda)

    def at_the_end(t):
        big = torch.zeros(N, D, dtype=t.dtype, device=cuda)
        big[-n:] = t
        return big

    def run(x, r, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, h = lh.add_rms_norm(*leaves)
        return [t.detach()[-n:].clone() for t in (y, h)], torch.autograd.grad((y, h), leaves, (dy, dy))

    small, (dx, dr, dw) = run(x, r, dy)
    big, (bx, br, bw) = run(at_the_end(x), at_the_end(r), at_the_end(dy))
    assert all(torch.equal(a, b) for a, b in zip(small, big))
    assert torch.equal(dx, bx[-n:]) and torch.equal(dr, br[-n:])
    h, rstd, _ = _ref(x, r, w)
    _assert_within(bw, dw.double(), 2 * (n + 50) * U * (dy.double() * h * rstd).abs().sum(0), "dw")
    del bx, br, big
    q = lh.add_rms_norm_fp8(at_the_end(x), at_the_end(r), w, group=128)
    assert all(torch.equal(a[-n:].view(torch.uint8), b.view(torch.uint8)) for a, b in
               zip(q, lh.add_rms_norm_fp8(x, r, w, group=128)))
