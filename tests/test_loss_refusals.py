"""What the losses of an output projection refuse, on the host: nothing is launched."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_shapes_types_and_options_are_refused(lh):
    E = lh._native.LighthouseShapeError
    n = lh._native
    t = _z(4, dtype=torch.int64)
    with pytest.raises(E, match="agree"):
        n.linear_xent_fwd(_z(4, 64), _z(10, 72), t, -100, "mean")
    with pytest.raises(E, match="multiple of 8"):
        n.linear_xent_fwd(_z(4, 60), _z(10, 60), t, -100, "mean")
    with pytest.raises(E, match="V in"):
        n.linear_xent_fwd(_z(4, 64), _z(0, 64), t, -100, "mean")
    with pytest.raises(ValueError, match="bf16"):
        n.linear_xent_fwd(_z(4, 64, dtype=torch.float32), _z(10, 64), t, -100, "mean")
    with pytest.raises(ValueError, match="reduction"):
        n.linear_xent_fwd(_z(4, 64), _z(10, 64), t, -100, "median")
    with pytest.raises(E, match="target"):
        n.linear_xent_fwd(_z(4, 64), _z(10, 64), t[:3], -100, "mean")
    with pytest.raises(ValueError, match="leading"):
        lh.linear_cross_entropy(_z(2, 2, 64), _z(10, 64), t)
    with pytest.raises(ValueError, match="CUDA"):
        lh.linear_cross_entropy(_z(4, 64), _z(10, 64), t)
    with pytest.raises(ValueError, match="int64 or int32"):
        lh.linear_cross_entropy(_z(4, 64), _z(10, 64), _z(4, dtype=torch.float32))
    tv, ti = _z(4, 3, dtype=torch.float32), _z(4, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="int64 or int32"):
        lh.linear_distillation(_z(4, 64), _z(10, 64), tv, tv)
    with pytest.raises(E, match="K must"):
        n.linear_distill_fwd(_z(4, 64), _z(10, 64), _z(4, 257), _z(4, 257, dtype=torch.int64), 1.0, "mean")
    with pytest.raises(E, match="K must"):
        lh.linear_distillation(_z(4, 64), _z(10, 64), _z(4, 0), _z(4, 0, dtype=torch.int64))
    with pytest.raises(E, match=r"\(N, K\)"):
        n.linear_distill_fwd(_z(4, 64), _z(10, 64), tv, ti[:, :2], 1.0, "mean")
    for T in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            n.linear_distill_fwd(_z(4, 64), _z(10, 64), tv, ti, T, "mean")
    with pytest.raises(ValueError, match="teacher logits"):
        n.linear_distill_fwd(_z(4, 64), _z(10, 64), tv.half(), ti, 1.0, "mean")
    with pytest.raises(ValueError, match="CUDA"):
        lh.linear_distillation(_z(4, 64), _z(10, 64), tv, ti)


def test_c_entry_points_check_before_they_touch_a_device(lh):
    lib = lh._native.load()
    P = ctypes.c_void_p
    a = P(4096)                  # aligned and never read: every call below is refused on the host
    big = 1 << 40

    def xf(h=a, w=a, t=a, N=4, V=10, D=64, red=1, loss=a, kept=a, ws=a, n=big, nk=big):
        return lib.lh_linear_xent_fwd(h, w, t, -100, N, V, D, red, loss, kept, nk, ws, n, None)

    assert xf(h=None) == 2 and xf(t=None) == 2 and xf(loss=None) == 2 and xf(kept=None) == 2 and xf(ws=None) == 2
    assert xf(N=0) == 1 and xf(V=0) == 1 and xf(D=12) == 1 and xf(N=(1 << 22) + 1) == 1 and xf(V=(1 << 22) + 1) == 1
    assert xf(red=3) == 2 and xf(w=P(4104)) == 2 and xf(kept=P(4104)) == 2 and xf(ws=P(4096 + 16)) == 2
    assert xf(n=lib.lh_linear_loss_workspace_size(4, 10, 64, 0, 0) - 1) == 5
    assert xf(nk=lib.lh_linear_loss_kept_size(4, 10, 0, 1, 0) - 1) == 5

    def xb(gout=a, red=1, dw=a, n=big):
        return lib.lh_linear_xent_bwd(a, a, a, 4, 10, 64, red, a, big, gout, a, dw, a, n, None)

    assert xb(gout=None) == 2 and xb(red=-1) == 2 and xb(dw=P(4100)) == 2
    assert xb(n=lib.lh_linear_loss_workspace_size(4, 10, 64, 0, 1) - 1) == 5

    def df(K=3, T=1.0, tv=a, dt=1):
        return lib.lh_linear_distill_fwd(a, a, tv, dt, a, 4, 10, 64, K, T, 1, a, a, big, a, big, None)

    assert df(K=0) == 1 and df(K=257) == 1 and df(T=0.0) == 2 and df(tv=None) == 2 and df(dt=2) == 2

    def db(kept=a, K=3):
        return lib.lh_linear_distill_bwd(a, a, 4, 10, 64, K, 1.0, 1, kept, big, a, a, a, a, big, None)

    assert db(kept=None) == 2 and db(K=0) == 1
    # one of the gradients may be left out, not both
    assert lib.lh_linear_xent_bwd(a, a, a, 4, 10, 64, 1, a, big, a, None, None, a, big, None) == 2
    assert lib.lh_linear_distill_bwd(a, a, 4, 10, 64, 3, 1.0, 1, a, big, a, None, None, a, big, None) == 2


def test_workspace_stays_small(lh):
    """The backward's workspace does not grow with the vocabulary: at most one 512 MB piece plus
    fp32 sums of the size of the gradients."""
    size = lh._native.load().lh_linear_loss_workspace_size
    for N in (1, 17, 1024, 8192, 65536):
        for V in (1, 256, 32000, 131072, 1 << 20):
            for D in (64, 1024, 4096):
                piece = max(512 << 20, 2 * N * 256)
                planes = 74 * 4 * 256 * D * 8 + 10 * N * D     # parts only where few tiles are; packed rows
                assert 0 < size(N, V, D, 0, 1) <= piece + planes + 4096, (N, V, D)
                assert size(N, V, D, 0, 0) <= 64 * N * (V // 256 + 1) + 6 * N + 2 * N * D + 4096


def test_fake_kernels(lh):
    m = lambda *s, d=BF: torch.empty(*s, dtype=d, device="meta", requires_grad=d.is_floating_point)
    h, w = m(2, 3, 64), m(100, 64)
    assert lh.linear_cross_entropy(h, w, m(2, 3, d=torch.int64), reduction="none").shape == (2, 3)
    loss = lh.linear_distillation(h, w, m(2, 3, 5, d=torch.float32), m(2, 3, 5, d=torch.int32), temperature=2.0)
    assert loss.shape == () and loss.dtype == torch.float32
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert dh.shape == h.shape and dw.shape == w.shape and dh.dtype == dw.dtype == BF


def test_eager_calls_leave_cpu_and_meta_tensors_to_python(lh):
    e = lh._native.eager()
    h, w, t = _z(4, 64), _z(10, 64), _z(4, dtype=torch.int64)
    for dev in ("cpu", "meta"):
        a, b, c = h.to(dev), w.to(dev), t.to(dev)
        assert e.linear_xent(a, b, c, -100, 1) is None
        assert e.linear_distill(a, b, a[:, :3].float(), c[:, None].expand(4, 3), 1.0, 1) is None
        assert e.rms_norm(a, b[0], 1e-5, None) is None and e.add_rms_norm(a, a, b[0], 1e-5, None) is None
        assert e.rms_norm_fp8(a, b[0], 1e-5, 0) is None and e.add_rms_norm_fp8(a, a, b[0], 1e-5, 128) is None


def test_kept_size_holds_gradients_of_one_tile_only(lh):
    size = lh._native.load().lh_linear_loss_kept_size
    for N, V, red, more in ((65, 256, 1, True), (1000, 1, 2, True), (64, 256, 1, False), (65, 257, 1, False), (65, 256, 0, False)):
        for K in (0, 16):
            assert size(N, V, K, red, 1) - size(N, V, K, red, 0) == (512 * N + 255) // 256 * 256 * more
    assert size(0, 10, 0, 1, 1) == 0


def test_kept_bytes_are_those_of_the_library(lh):
    n = lh._native
    for N in (0, 1, 3, 31, 64, 65, 777, 5000, 1 << 22):
        for V in (1, 256, 257, 50261):
            for K in (0, 1, 3, 16, 250, 256):
                for red in ("none", "mean", "sum"):
                    assert n.kept_bytes(N, V, K, red) == n.kept_size(N, V, K, red), (N, V, K, red)


@pytest.mark.parametrize("V", [100, 300])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_one_graph_for_any_number_of_positions(lh, V, reduction):
    """Losses and gradients traced with a symbolic number of positions (and of teacher entries): one
    compilation serves them all, whatever the sizes of what is kept."""
    compiled = []

    def backend(gm, inputs):
        compiled.append(gm)
        return torch._dynamo.backends.debugging.aot_eager(gm, inputs)

    def f(h, w, t, tv, ti):
        a = lh.linear_cross_entropy(h, w, t, reduction=reduction)
        b = lh.linear_distillation(h, w, tv, ti, temperature=2.0, reduction=reduction)
        return a + b

    torch._dynamo.reset()
    fn = torch.compile(f, fullgraph=True, backend=backend)
    for N, K in ((40, 5), (70, 6), (300, 9), (5000, 33)):
        m = lambda *s, d=BF: torch.empty(*s, dtype=d, device="meta", requires_grad=d == BF)
        h, w, t = m(N, 64), m(V, 64), m(N, d=torch.int64)
        tv, ti = m(N, K, d=torch.float32), m(N, K, d=torch.int64)
        for x in (h, t, tv, ti):
            torch._dynamo.mark_dynamic(x, 0)
        for x in (tv, ti):
            torch._dynamo.mark_dynamic(x, 1)
        loss = fn(h, w, t, tv, ti)
        assert loss.shape == ((N,) if reduction == "none" else ())
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert dh.shape == h.shape and dw.shape == w.shape
    assert len(compiled) == 1


def test_workspace_is_what_the_documentation_says(lh):
    size = lh._native.load().lh_linear_loss_workspace_size
    for N in (1, 17, 64, 65, 1000, 2000, 4096, 20000, 37888, 65536, 262144, 1 << 22):
        for V in (1, 256, 257, 5000, 50261, 131072, 1 << 20, 1 << 22):
            tiles = (V + 255) // 256 * 256                     # a tile's statistics are whole
            for D in (8, 512, 1024, 4096, 16384, 65536):
                copy = 2 * max(N, 64) * D                      # up to 32 rows: two terms of 32
                fwd = N * tiles // 16 + copy + 4 * N * 256 + 8 * N + (160 << 10)
                assert size(N, V, D, 256, 0) <= fwd, (N, V, D)
                sums = 8 * N * D + 160e6
                assert size(N, V, D, 0, 1) <= max(512 << 20, 512 * max(N, 64)) + copy + sums, (N, V, D)


def test_temperatures_whose_square_or_inverse_is_no_fp32_number(lh):
    tv, ti = _z(4, 3, dtype=torch.float32), _z(4, 3, dtype=torch.int64)
    for T in (1e-40, 1e-30, 1e19, 1e29):
        with pytest.raises(ValueError, match="temperature"):
            lh._native.linear_distill_fwd(_z(4, 64), _z(10, 64), tv, ti, T, "mean")
        a = ctypes.c_void_p(4096)
        lib = lh._native.load()
        assert lib.lh_linear_distill_fwd(a, a, a, 1, a, 4, 10, 64, 3, T, 1, a, a, 1 << 40, a, 1 << 40, None) == 2
        assert lib.lh_linear_distill_bwd(a, a, 4, 10, 64, 3, T, 1, a, 1 << 40, a, a, a, a, 1 << 40, None) == 2
    for T in (1e-18, 1e18):                              # not refused for its temperature, only as a CPU tensor
        with pytest.raises(ValueError, match="CUDA"):
            lh._native.linear_distill_fwd(_z(4, 64), _z(10, 64), tv, ti, T, "mean")
