"""What the norm refuses, on the host: no GPU is needed, nothing is launched."""
import ctypes

import pytest
import torch


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_shapes_and_types_are_refused(lh):
    E = lh._native.LighthouseShapeError
    with pytest.raises(E, match="multiple of 8"):
        lh._native.rms_norm_fwd(_t(2, 12), None, _t(12), 1e-5, torch.bfloat16)
    with pytest.raises(E, match="multiple of 8"):
        lh._native.rms_norm_fwd(_t(1, 16392), None, _t(16392), 1e-5, torch.bfloat16)
    with pytest.raises(E, match="agree"):
        lh._native.rms_norm_fwd(_t(2, 16), None, _t(8), 1e-5, torch.bfloat16)
    with pytest.raises(E, match="agree"):
        lh._native.rms_norm_fwd(_t(2, 16), _t(3, 16), _t(16), 1e-5, torch.bfloat16)
    with pytest.raises(ValueError, match="bf16 and fp32"):
        lh._native.rms_norm_fwd(_t(2, 16, dtype=torch.float16), None, _t(16), 1e-5, torch.bfloat16)
    with pytest.raises(ValueError, match="out_dtype"):
        lh._native.rms_norm_fwd(_t(2, 16), None, _t(16), 1e-5, torch.float16)
    with pytest.raises(ValueError, match="group"):
        lh._native.rms_norm_fwd(_t(2, 16), None, _t(16), 1e-5, torch.float8_e4m3fn, group=64)
    with pytest.raises(ValueError, match="group"):
        lh._native.rms_norm_fwd(_t(2, 16), None, _t(16), 1e-5, torch.bfloat16, group=128)


def test_cpu_tensors_are_refused(lh):
    with pytest.raises(ValueError, match="CUDA"):
        lh.add_rms_norm(_t(2, 16), _t(2, 16), _t(16))
    with pytest.raises(ValueError, match="CUDA"):
        lh.rms_norm_fp8(_t(2, 16), _t(16))


def test_c_entry_points_check_before_they_touch_a_device(lh):
    lib = lh._native.load()
    P = ctypes.c_void_p
    a = P(4096)                  # aligned and never read: every call below is refused on the host

    def fwd(x=a, r=None, w=a, N=4, D=64, y=a, ydt=0, scale=None, group=0, h=None, xdt=0):
        return lib.lh_rms_norm_fwd(x, xdt, r, 0, w, 0, N, D, 1e-5, y, ydt, scale, group, h, None, None)

    assert fwd(x=None) == 2 and fwd(y=None) == 2
    assert fwd(r=a, h=None) == 2
    assert fwd(xdt=5) == 2 and fwd(ydt=3) == 2 and fwd(xdt=2) == 2
    assert fwd(ydt=2) == 2 and fwd(ydt=2, scale=a, group=32) == 2
    assert fwd(N=0) == 1 and fwd(D=12) == 1 and fwd(D=16392) == 1
    assert fwd(x=P(4098)) == 2 and b"aligned" in lib.lh_last_error()

    def bwd(ws=a, n=1 << 30, D=64, N=4, dw=a):
        return lib.lh_rms_norm_bwd(a, 0, None, a, 0, a, 0, a, N, D, a, 0, None, dw, ws, n, None)

    assert bwd(dw=None) == 2 and bwd(N=0) == 1 and bwd(D=4) == 1 and bwd(ws=None) == 2
    assert bwd(n=lib.lh_rms_norm_bwd_workspace_size(4, 64) - 1) == 5


def test_fake_kernels(lh):
    m = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device="meta", requires_grad=True)
    y, h = lh.add_rms_norm(m(2, 3, 64), m(2, 3, 64, d=torch.float32), m(64, d=torch.float32), out_dtype=torch.float32)
    assert y.dtype == torch.float32 and h.dtype == torch.float32 and y.shape == h.shape == (2, 3, 64)
    (y.sum() + h.sum()).backward()
    q, s = lh.rms_norm_fp8(m(5, 200), m(200), group=128)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (5, 2)
    q, s, h = lh.add_rms_norm_fp8(m(5, 200), m(5, 200, d=torch.float32), m(200))
    assert s.shape == (5, 1) and h.dtype == torch.float32


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_an_8_bit_output_without_scales_is_refused(lh, device):
    """rms_norm and add_rms_norm return no scales, and the codes are nothing without them."""
    x, w = _t(2, 16).to(device), _t(16).to(device)
    for call in (lambda: lh.rms_norm(x, w, out_dtype=torch.float8_e4m3fn),
                 lambda: lh.add_rms_norm(x, x, w, out_dtype=torch.float8_e4m3fn)):
        with pytest.raises(ValueError, match="scales"):
            call()
    if device == "cpu":
        with pytest.raises(ValueError, match="scales"):
            lh._native.rms_norm_fwd(x, None, w, 1e-5, torch.float8_e4m3fn)
