"""The C++ eager calls of the norm and the losses: the same results as the custom ops, the cases
they leave to them, one derivative only, and another thread's calls."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _norm_inputs(cuda, n=37, d=264):
    g = torch.Generator().manual_seed(1)
    return (torch.randn(n, d, generator=g).to(BF).to(cuda), torch.randn(n, d, generator=g).to(cuda),
            torch.randn(d, generator=g).to(cuda))


def _loss_inputs(cuda, n=90, v=700, d=128, k=6):
    g = torch.Generator().manual_seed(2)
    return ((torch.randn(n, d, generator=g)).to(BF).to(cuda), (torch.randn(v, d, generator=g) * 0.1).to(BF).to(cuda),
            torch.randint(0, v, (n,), generator=g).to(cuda), torch.randn(n, k, generator=g).to(cuda),
            torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]).to(cuda))


def _leaves(*ts):
    return [t.detach().clone().requires_grad_(True) for t in ts]


def test_same_results_as_the_custom_ops(lh, cuda, monkeypatch):
    from lighthouse_b200 import losses, norm
    x, r, w = _norm_inputs(cuda)
    h, wt, t, tl, ti = _loss_inputs(cuda)

    def everything():
        out = []
        ls = _leaves(x, r, w)
        y, hh = lh.add_rms_norm(*ls, out_dtype=BF)
        out += [y, hh, *torch.autograd.grad((y, hh), ls, (torch.ones_like(y), torch.ones_like(hh)))]
        ls = _leaves(x, w)
        y = lh.rms_norm(*ls, 1e-3)
        out += [y, *torch.autograd.grad(y, ls, torch.ones_like(y))]
        out += [*lh.rms_norm_fp8(x, w, group=128), *lh.add_rms_norm_fp8(x, r, w)]
        for red in ("mean", "sum", "none"):
            ls = _leaves(h, wt)
            loss = lh.linear_cross_entropy(*ls, t, ignore_index=3, reduction=red)
            out += [loss, *torch.autograd.grad(loss, ls, torch.ones_like(loss))]
            ls = _leaves(h, wt)
            loss = lh.linear_distillation(*ls, tl, ti, temperature=2.0, reduction=red)
            out += [loss, *torch.autograd.grad(loss, ls, torch.ones_like(loss))]
        return [o.detach() for o in out]

    fast = everything()
    monkeypatch.setattr(norm, "_eager", lambda *a: None)
    monkeypatch.setattr(losses, "_eager", lambda *a: None)
    slow = everything()
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                           b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)


def test_cases_left_to_the_python_path(lh, cuda):
    e = lh._native.eager()
    x, r, w = _norm_inputs(cuda)
    h, wt, t, tl, ti = _loss_inputs(cuda)
    assert e.rms_norm(x, w, 1e-5, None) is not None and e.linear_xent(h, wt, t, -100, 1) is not None
    none = [e.rms_norm(x.repeat(1, 2)[:, :264], w, 1e-5, None), e.rms_norm(x, w[:8], 1e-5, None),
            e.rms_norm(x.half(), w, 1e-5, None), e.rms_norm(x, w, 1e-5, torch.float16), e.rms_norm(x.cpu(), w, 1e-5, None),
            e.rms_norm(x[:0], w, 1e-5, None), e.add_rms_norm(x, r[1:], w, 1e-5, None), e.rms_norm_fp8(x, w, 1e-5, 64),
            e.rms_norm_fp8(x.clone().requires_grad_(True), w, 1e-5, 0),
            e.linear_xent(h.float(), wt, t, -100, 1), e.linear_xent(h, wt[:, :64], t, -100, 1),
            e.linear_xent(h, wt, t.int(), -100, 1), e.linear_xent(h, wt, t[1:], -100, 1), e.linear_xent(h, wt, t, -100, 7),
            e.linear_xent(h, wt, t.cpu(), -100, 1), e.linear_distill(h, wt, tl, ti[:, 1:], 1.0, 1),
            e.linear_distill(h, wt, tl, ti, 0.0, 1), e.linear_distill(h, wt, tl.half(), ti, 1.0, 1)]
    assert all(o is None for o in none)
    with pytest.raises(lh._native.LighthouseShapeError):
        lh.rms_norm(x, w[:8])
    with pytest.raises(ValueError):
        lh.linear_cross_entropy(h.float(), wt, t)
    with pytest.raises(ValueError, match="different devices|CUDA"):
        lh.linear_cross_entropy(h, wt, t.cpu())


def test_no_graph_where_none_is_wanted(lh, cuda):
    x, r, w = _norm_inputs(cuda)
    h, wt, t, *_ = _loss_inputs(cuda)
    assert not lh.rms_norm(x, w).requires_grad and not lh.linear_cross_entropy(h, wt, t).requires_grad
    x.requires_grad_(True)
    wt.requires_grad_(True)
    with torch.no_grad():
        assert not lh.rms_norm(x, w).requires_grad and not lh.linear_cross_entropy(h, wt, t).requires_grad
    y, hh = lh.add_rms_norm(x, r, w)
    assert y.requires_grad and hh.requires_grad
    dw, = torch.autograd.grad(lh.linear_cross_entropy(h, wt, t), wt)
    assert dw.shape == wt.shape
    with pytest.raises(RuntimeError):
        lh.rms_norm_fp8(x, w)[0].float().sum().backward()


def test_second_derivatives_raise(lh, cuda):
    x, r, w = _norm_inputs(cuda)
    h, wt, t, *_ = _loss_inputs(cuda)
    for strided in (False, True):                # the C++ call, and the Python one
        ls = _leaves(x, w)
        xs = ls[0].T.contiguous().T if strided else ls[0]
        g, = torch.autograd.grad(lh.rms_norm(xs, ls[1]).float().square().sum(), ls[1], create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
        ls = _leaves(h, wt)
        hs = ls[0].T.contiguous().T if strided else ls[0]
        g, = torch.autograd.grad(lh.linear_cross_entropy(hs, ls[1], t), ls[1], create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().sum().backward()


def test_a_changed_input_is_noticed(lh, cuda):
    h, wt, t, *_ = _loss_inputs(cuda)
    ls = _leaves(h, wt)
    loss = lh.linear_cross_entropy(*ls, t)
    with torch.no_grad():
        ls[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_calls_from_several_threads(lh, cuda):
    """Two threads, each on its own stream, with other sizes."""
    res = {}

    def work(i):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            h, wt, t, *_ = _loss_inputs(cuda, n=90 + 200 * i, v=700 + i)
            out = []
            for _ in range(20):
                ls = _leaves(h, wt)
                loss = lh.linear_cross_entropy(*ls, t)
                out.append([loss.detach(), *torch.autograd.grad(loss, ls)])
            torch.cuda.current_stream().synchronize()
            res[i] = out

    ths = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [a.start() for a in ths]
    [a.join() for a in ths]
    for i in range(2):
        assert len(res[i]) == 20
        for o in res[i][1:]:
            assert all(torch.equal(a, b) for a, b in zip(o, res[i][0]))
    assert lh._native.device_status() == 0


def _strided(t):
    """The same values with every element at a stride of two."""
    big = torch.empty(*t.shape, 2, dtype=t.dtype, device=t.device)
    big[..., 0] = t
    return big[..., 0]


@pytest.mark.parametrize("call", ["norm", "add_norm", "xent", "distill", "xent_one_tile"])
def test_hooks_on_saved_tensors(lh, cuda, call):
    """Saved tensors that come back from the host, or with other strides, give the same gradients; one of
    another type or shape is refused."""
    x, r, w = _norm_inputs(cuda)
    h, wt, t, tl, ti = _loss_inputs(cuda)
    if call == "xent_one_tile":
        wt, t = wt[:200], t % 200
    f, ls = {"norm": (lambda a, c: lh.rms_norm(a, c), (x, w)),
             "add_norm": (lambda a, b, c: sum(o.float() for o in lh.add_rms_norm(a, b, c)), (x, r, w)),
             "xent": (lambda a, b: lh.linear_cross_entropy(a, b, t), (h, wt)),
             "xent_one_tile": (lambda a, b: lh.linear_cross_entropy(a, b, t), (h, wt)),
             "distill": (lambda a, b: lh.linear_distillation(a, b, tl, ti), (h, wt))}[call]
    ls = _leaves(*ls)
    y = f(*ls)
    up = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(y)
    want = torch.autograd.grad(y, ls, up)
    with torch.autograd.graph.save_on_cpu():
        y = f(*ls)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, ls, up)))
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, _strided):
        y = f(*ls)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, ls, up)))
    for other in (lambda s: s.double(), lambda s: s[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, other):
            y = f(*ls)
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(y, ls, up)


def test_tensors_with_a_lazy_minus(lh, cuda):
    """Inputs and upstream gradients whose minus is a bit beside the memory (what torch.imag makes of a conjugate)."""
    x, r, w = _norm_inputs(cuda)
    h, wt, t, tl, ti = _loss_inputs(cuda)
    minus = torch._neg_view
    assert torch.equal(lh.linear_distillation(h, wt, minus(tl), ti), lh.linear_distillation(h, wt, -tl, ti))
    assert torch.equal(lh.linear_cross_entropy(minus(h), wt, t), lh.linear_cross_entropy(-h, wt, t))
    assert torch.equal(lh.rms_norm(minus(x), w), lh.rms_norm(-x, w))
    ls = _leaves(x, r, w)
    up = torch.randn_like(r)
    for a, b in ((minus(up), -up), (torch.complex(up, up).conj().imag, -up)):
        y, s = lh.add_rms_norm(*ls, out_dtype=torch.float32)
        got = torch.autograd.grad((y, s), ls, (a, a), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad((y, s), ls, (b, b))))
    ls = _leaves(h, wt)
    up = torch.randn(h.shape[0], device=cuda)
    loss = lh.linear_cross_entropy(*ls, t, reduction="none")
    got = torch.autograd.grad(loss, ls, minus(up), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(loss, ls, -up)))
