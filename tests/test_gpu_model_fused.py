"""The norm and the losses as the model uses them: training with both, distillation, 8-bit inference."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SMALL = dict(dim=256, n_layers=3, n_heads=2, n_kv_heads=2, hidden_dim=384, max_seq_len=2048)


def _model(M, cuda, **kw):
    torch.manual_seed(0)
    m = M.Transformer(M.ModelArgs(**{**SMALL, **kw})).to(cuda)
    m.init_weights(0)
    return m


def _tokens(cuda, n=1025, seed=5):
    return torch.randint(0, 256, (2, n), generator=torch.Generator().manual_seed(seed)).to(cuda)


def _grads(m):
    return torch.cat([p.grad.detach().double().reshape(-1) for p in m.parameters()])


def _rel(a, b):
    return ((a - b).norm() / b.norm()).item()


def test_fused_training_is_as_near_to_fp32_as_the_separate_operations(lh, cuda):
    """Loss and every gradient of the model under autocast, fused and not, against the fp32 model: the
    fused one rounds no more often (the residual stream and the norms stay fp32 inside), so its distance
    is that of the separate operations or less, with a margin of a quarter for chance."""
    from lighthouse_b200 import model as M
    tokens = _tokens(cuda)
    inputs, labels = tokens[:, :-1], tokens[:, 1:]

    def run(autocast, **kw):
        m = _model(M, cuda, use_selection_lighthouse=False, **kw)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            if kw.get("fused_loss"):
                loss = m(inputs, labels)
            else:
                logits = m(inputs)
        if not kw.get("fused_loss"):
            loss = torch.nn.functional.cross_entropy(logits.float().reshape(-1, 256), labels.reshape(-1))
        loss.backward()
        return loss.item(), _grads(m)

    ref, plain, fused = run(False), run(True), run(True, fused_norm=True, fused_loss=True)
    assert abs(fused[0] - ref[0]) <= 1.25 * abs(plain[0] - ref[0]) + 1e-4
    d_plain, d_fused = _rel(plain[1], ref[1]), _rel(fused[1], ref[1])
    assert d_fused <= 1.25 * d_plain, (d_fused, d_plain)
    # fp32 without autocast: the norm alone is fused, sums differ in their order only
    f32 = run(False, fused_norm=True)
    assert abs(f32[0] - ref[0]) <= 1e-5 * abs(ref[0]) and _rel(f32[1], ref[1]) <= 1e-4
    assert lh._native.device_status() == 0


def test_fused_training_step_with_lighthouse_layers(lh, cuda):
    from lighthouse_b200 import model as M
    m = _model(M, cuda, lighthouse_topk=256, lighthouse_full_attn_layers=[0], fused_norm=True, fused_loss=True,
               max_seq_len=4096)
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3, fused=True)
    tokens = _tokens(cuda, 4097)[:1]
    before = [p.detach().clone() for p in m.parameters()]
    loss = M.train_step(m, opt, tokens)
    assert loss.isfinite() and loss.dtype == torch.float32
    assert all(not torch.equal(a, b) for a, b in zip(before, m.parameters()))
    assert lh._native.device_status() == 0


def test_distillation_step_equals_the_formula_on_logits(lh, cuda):
    """The loss of a student against a teacher's 12 top logits, from the student's own bf16 hidden rows."""
    from lighthouse_b200 import model as M
    teacher, student = _model(M, cuda, use_selection_lighthouse=False), _model(M, cuda, use_selection_lighthouse=False,
                                                                               fused_norm=True, distill_temperature=2.0)
    with torch.no_grad():
        for p in teacher.parameters():
            p.mul_(1.5)
    tokens = _tokens(cuda)
    inputs = tokens[:, :-1]
    tl, ti = M.teacher_top_logits(teacher, inputs, 12)
    assert tl.shape == ti.shape == (2, 1024, 12)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = student(inputs, teacher=(tl, ti))
        hidden = student._normed(inputs).to(torch.bfloat16)
    s = hidden.double() @ student.output.weight.to(torch.bfloat16).double().T / 2.0
    p = torch.softmax(tl.double() / 2.0, -1)
    want = 4 * (p * (p.log() - torch.log_softmax(s, -1).gather(-1, ti))).sum(-1).mean()
    # fp32 logits of 256 products: 256 * 2^-23 of |h||w| at the most
    bound = 4 * 2 * 256 * 2.0 ** -23 * (hidden.double().norm(dim=-1).max() * student.output.weight.double().norm(dim=-1).max())
    assert abs(loss.item() - want.item()) <= bound.item()
    opt = torch.optim.AdamW(student.parameters(), lr=1e-3, fused=True)
    got = M.train_step(student, opt, tokens, teacher=(tl, ti))
    assert abs(got.item() - loss.item()) <= 1e-6 * abs(loss.item())
    assert all(p.grad is None for p in teacher.parameters())
    assert lh._native.device_status() == 0


def test_fp8_projection_equals_its_dequantised_product(lh, cuda):
    from lighthouse_b200 import model as M
    g = torch.Generator().manual_seed(2)
    lin = torch.nn.Linear(512, 304, bias=False).to(cuda)
    f = M.Fp8Linear(lin)
    for shape in ((1, 512), (3, 7, 512), (2, 100, 512)):
        x = torch.randn(*shape, generator=g).to(torch.bfloat16).to(cuda)
        q, s = lh.rms_norm_fp8(x, torch.ones(512, device=cuda))
        y = f((q, s))
        xd, wd = q.double() * s.double(), f.weight.double() * f.scale.T.double()
        ref = xd @ wd.T
        # a bf16 rounding, and 8-bit products summed in at least 22 bits
        tol = 2.0 ** -8 * ref.abs() + 512 * 2.0 ** -21 * (xd.abs() @ wd.abs().T)
        assert y.dtype == torch.bfloat16 and y.shape == ref.shape
        assert ((y.double() - ref).abs() <= tol).all()


def test_fp8_inference_equals_the_dequantised_model(lh, cuda, monkeypatch):
    """The 8-bit model against the same model whose projections multiply the dequantised values in fp32:
    they differ by the roundings of sums that end in bf16, one in 2^9, a few per block."""
    from lighthouse_b200 import model as M
    m = _model(M, cuda, use_selection_lighthouse=False).quantize_projections()
    tokens = _tokens(cuda, 300)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(tokens).double()

        def dequantised(self, x):
            q, s = x
            return ((q.float() * s) @ (self.weight.float() * self.scale.T).T.float()).to(torch.bfloat16)

        monkeypatch.setattr(M.Fp8Linear, "forward", lambda self, x: _no_autocast(dequantised, self, x))
        ref = m(tokens).double()
    assert got.isfinite().all() and _rel(got, ref) <= 2.0 ** -6
    # and it stands for the bf16 model: 8-bit values are within 2^-4, their errors independent
    plain = _model(M, cuda, use_selection_lighthouse=False)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert _rel(got, plain(tokens).double()) <= 0.25
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(RuntimeError):
        m(tokens).float().sum().backward()


def _no_autocast(f, *a):
    with torch.autocast("cuda", enabled=False):
        return f(*a)


def test_norm_and_loss_compile_as_one_graph(lh, cuda):
    g = torch.Generator().manual_seed(7)
    x, r = (torch.randn(64, 256, generator=g).to(cuda) for _ in range(2))
    w = torch.ones(256, device=cuda)
    out = (torch.randn(300, 256, generator=g) * 0.05).to(torch.bfloat16).to(cuda)
    t = torch.randint(0, 300, (64,), generator=g).to(cuda)

    def f(x, r, w, out):
        y, h = lh.add_rms_norm(x, r, w, out_dtype=torch.bfloat16)
        return lh.linear_cross_entropy(y, out, t), h

    def run(fn):
        ls = [a.detach().clone().requires_grad_(True) for a in (x, r, w, out)]
        loss, h = fn(*ls)
        return [loss.detach(), h.detach(), *torch.autograd.grad(loss + h.sum(), ls)]

    torch._dynamo.reset()
    for a, b in zip(run(torch.compile(f, fullgraph=True)), run(f)):
        assert torch.equal(a, b)


def test_a_training_step_in_a_graph(lh, cuda):
    """Norm, projection loss and their gradients captured and replayed on new inputs; the eager run's graph is gone
    before the capture."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(512, 256, generator=g).to(torch.bfloat16).to(cuda)
    r = torch.randn(512, 256, generator=g).to(cuda)
    w = torch.ones(256, device=cuda)
    out = (torch.randn(1000, 256, generator=g) * 0.05).to(torch.bfloat16).to(cuda)
    t = torch.randint(0, 1000, (512,), generator=g).to(cuda)

    def step():
        ls = [a.detach().requires_grad_(True) for a in (x, r, w, out)]
        y, h = lh.add_rms_norm(*ls[:3])
        y2, _ = lh.add_rms_norm(y, h, ls[2])
        return [a.detach() for a in torch.autograd.grad(lh.linear_cross_entropy(y2, ls[3], t), ls)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(torch.randn_like(x))
    t.copy_(t.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(step(), got))
    assert lh._native.device_status() == 0
