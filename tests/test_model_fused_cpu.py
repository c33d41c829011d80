"""The model's fused options on the CPU, where they take the separate operations: same results,
same gradients, and what they refuse."""
import pytest
import torch


def _args(M, **kw):
    return M.ModelArgs(dim=64, n_layers=2, n_heads=2, n_kv_heads=2, hidden_dim=96, use_selection_lighthouse=False, **kw)


def _model(M, **kw):
    torch.manual_seed(0)
    m = M.Transformer(_args(M, **kw))
    m.init_weights(3)
    return m


def test_fused_options_keep_results_on_the_cpu(lh):
    from lighthouse_b200 import model as M
    tokens = torch.randint(0, 256, (2, 33), generator=torch.Generator().manual_seed(1))
    inputs, labels = tokens[:, :-1], tokens[:, 1:]
    a, b = _model(M), _model(M, fused_norm=True, fused_loss=True)
    la, lb = a(inputs), b(inputs)
    assert torch.equal(la, lb)
    loss_a = torch.nn.functional.cross_entropy(la.float().reshape(-1, 256), labels.reshape(-1))
    loss_b = b(inputs, labels)
    assert torch.equal(loss_a, loss_b)
    loss_a.backward()
    loss_b.backward()
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        assert torch.allclose(p.grad, q.grad, rtol=0, atol=0) or (p.grad - q.grad).abs().max() <= 1e-6 * p.grad.abs().max(), n


def test_defaults_are_off_and_refusals(lh):
    from lighthouse_b200 import model as M
    args = M.ModelArgs()
    assert not args.fused_norm and not args.fused_loss
    m = _model(M)
    tokens = torch.randint(0, 256, (1, 16))
    with pytest.raises(ValueError, match="either"):
        m(tokens, tokens, (torch.zeros(1, 16, 4), torch.zeros(1, 16, 4, dtype=torch.int64)))
    with pytest.raises(ValueError, match="distillation"):
        m(tokens, teacher=(torch.zeros(1, 16, 4), torch.zeros(1, 16, 4, dtype=torch.int64)))
    m.quantize_projections()
    assert m.layers[0].attention.wq.weight.dtype == torch.float8_e4m3fn
    assert m.layers[0].attention.wo.weight.dtype == torch.float32
    m.quantize_projections()                                    # twice is once
    with pytest.raises(ValueError, match="CUDA"):
        m(tokens)
    with pytest.raises(ValueError, match="multiples of 16"):
        M.Fp8Linear(torch.nn.Linear(40, 16, bias=False))
    g = M.Transformer(M.ModelArgs(dim=256, n_layers=1, n_heads=2, n_kv_heads=2, hidden_dim=384, lighthouse_scorer="gla",
                                  lighthouse_full_attn_layers=[]))
    with pytest.raises(ValueError, match="gla"):
        g.quantize_projections()


def test_fp8_weights_stand_for_the_projection(lh):
    from lighthouse_b200 import model as M
    lin = torch.nn.Linear(64, 48, bias=False)
    q = M.Fp8Linear(lin)
    back = q.weight.float() * q.scale.T
    # half a step of e4m3 (2^-4 of the value), or of its smallest codes (2^-10 of the row's scale)
    tol = 2.0 ** -4 * lin.weight.abs() + 2.0 ** -10 * q.scale.T
    assert ((back - lin.weight).abs() <= tol * (1 + 1e-6)).all()
    assert q.scale.shape == (1, 48)
