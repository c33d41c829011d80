"""ctypes binding of liblighthouse_b200.so (the C ABI in include/lighthouse_b200.h).

Every wrapper takes torch CUDA tensors, checks dtype / layout / device,
allocates outputs with torch's caching allocator on the input's device and
enqueues the kernels on ``torch.cuda.current_stream()``.  There is no CPU or
eager-PyTorch fallback: if the library is missing or the device is not a
B200 the call raises.
"""
from __future__ import annotations

import ctypes
import importlib.util
import pathlib

import torch

_LIB_PATH = pathlib.Path(__file__).resolve().parent / "liblighthouse_b200.so"
_EAGER_PATH = _LIB_PATH.with_name("_eager.so")
_lib = None
_eager = None

LH_DTYPE = {torch.bfloat16: 0, torch.float32: 1}
_VP = ctypes.c_void_p


class LighthouseError(RuntimeError):
    """Raised when a C-ABI entry point returns a non-zero status."""


class LighthouseShapeError(ValueError):
    """The C ABI rejected a shape (LH_ERR_SHAPE)."""


_SIGS = {
    "lh_last_error": (ctypes.c_char_p, []),
    "lh_abi_version": (ctypes.c_int, []),
    "lh_device_status": (ctypes.c_int, [ctypes.c_int]),
    "lh_pyramid_score_fwd": (ctypes.c_int, [_VP, _VP, _VP, ctypes.c_int] + [ctypes.c_int] * 6 + [_VP] * 6),
    "lh_select_topk": (ctypes.c_int, [_VP, _VP] + [ctypes.c_int] * 6 + [_VP, _VP, _VP]),
    "lh_build_inverse": (ctypes.c_int, [_VP] + [ctypes.c_int] * 4 + [_VP, _VP]),
    "lh_gather_selected": (ctypes.c_int, [_VP] * 6 + [ctypes.c_int] * 6 + [_VP, ctypes.c_int] + [_VP] * 4),
    "lh_attn_fwd": (ctypes.c_int, [_VP] * 3 + [ctypes.c_int] * 6 + [ctypes.c_float, _VP, _VP, _VP]),
    "lh_attn_bwd_workspace_size": (ctypes.c_size_t, [ctypes.c_int] * 5),
    "lh_attn_merge": (ctypes.c_int, [_VP] * 4 + [ctypes.c_longlong, ctypes.c_int, _VP, _VP, _VP]),
    "lh_attn_bwd": (ctypes.c_int, [_VP] * 6 + [ctypes.c_int] * 6 + [ctypes.c_float] + [_VP] * 4
                    + [ctypes.c_size_t, _VP]),
    "lh_attn_bwd_noalloc": (ctypes.c_int, [_VP] * 6 + [ctypes.c_int] * 6 + [ctypes.c_float] + [_VP] * 4),
    "lh_scatter_fwd": (ctypes.c_int, [_VP, _VP] + [ctypes.c_int] * 9 + [_VP, _VP]),
    "lh_scatter_bwd": (ctypes.c_int, [_VP, _VP] + [ctypes.c_int] * 9 + [_VP, _VP]),
    "lh_scatter_fwd_token_major": (ctypes.c_int, [_VP, _VP] + [ctypes.c_int] * 9 + [_VP, _VP]),
    "lh_scatter_bwd_token_major": (ctypes.c_int, [_VP, _VP] + [ctypes.c_int] * 9 + [_VP, _VP]),
    "lh_unpool_bwd": (ctypes.c_int, [_VP] * 4 + [ctypes.c_int] * 8 + [_VP] * 4),
    "lh_rope_apply": (ctypes.c_int, [_VP] * 5 + [ctypes.c_int] * 6 + [_VP]),
    "lh_simple_gla_fwd": (ctypes.c_int, [_VP] * 8 + [ctypes.c_int] * 5 + [ctypes.c_float, _VP]),
    "lh_rms_norm_fwd": (ctypes.c_int, [_VP, ctypes.c_int] * 3 + [ctypes.c_longlong, ctypes.c_int, ctypes.c_float, _VP,
                                                                ctypes.c_int, _VP, ctypes.c_int] + [_VP] * 3),
    "lh_rms_norm_bwd_workspace_size": (ctypes.c_size_t, [ctypes.c_longlong, ctypes.c_int]),
    "lh_rms_norm_bwd": (ctypes.c_int, [_VP, ctypes.c_int, _VP, _VP, ctypes.c_int, _VP, ctypes.c_int, _VP,
                                       ctypes.c_longlong, ctypes.c_int, _VP, ctypes.c_int] + [_VP] * 3
                        + [ctypes.c_size_t, _VP]),
    "lh_linear_loss_workspace_size": (ctypes.c_size_t, [ctypes.c_int] * 5),
    "lh_linear_loss_kept_size": (ctypes.c_size_t, [ctypes.c_int] * 5),
    "lh_linear_xent_fwd": (ctypes.c_int, [_VP] * 3 + [ctypes.c_int64] + [ctypes.c_int] * 4
                           + [_VP, _VP, ctypes.c_size_t] + [_VP, ctypes.c_size_t, _VP]),
    "lh_linear_xent_bwd": (ctypes.c_int, [_VP] * 3 + [ctypes.c_int] * 4 + [_VP, ctypes.c_size_t] + [_VP] * 4
                           + [ctypes.c_size_t, _VP]),
    "lh_linear_distill_fwd": (ctypes.c_int, [_VP] * 3 + [ctypes.c_int, _VP] + [ctypes.c_int] * 4
                              + [ctypes.c_float, ctypes.c_int] + [_VP, _VP, ctypes.c_size_t]
                              + [_VP, ctypes.c_size_t, _VP]),
    "lh_linear_distill_bwd": (ctypes.c_int, [_VP] * 2 + [ctypes.c_int] * 4 + [ctypes.c_float, ctypes.c_int]
                              + [_VP, ctypes.c_size_t] + [_VP] * 4 + [ctypes.c_size_t, _VP]),
}

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_DENSE = torch.contiguous_format


def lib_path() -> pathlib.Path:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Load the library once; raise if it has not been built."""
    global _lib
    if _lib is None:
        if not _LIB_PATH.exists():
            raise ImportError(
                f"{_LIB_PATH} is not built; run `python lighthouse-attention_b200/build.py` "
                "(the CUDA path has no fallback)")
        lib = ctypes.CDLL(str(_LIB_PATH))
        for name, (res, args) in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def eager():
    """The eager calls of the norm and the losses (csrc/eager.cpp) on this library.  Its functions
    take the plain case, dense aligned CUDA tensors, and return None for any other."""
    global _eager
    if _eager is None:
        lib = load()
        if not _EAGER_PATH.exists():
            raise ImportError(f"{_EAGER_PATH} is not built; run `python lighthouse-attention_b200/build.py`")
        spec = importlib.util.spec_from_file_location(f"{__package__}._eager", _EAGER_PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.bind({name: ctypes.cast(getattr(lib, name), _VP).value for name in _SIGS})
        _eager = mod
    return _eager


def exported_symbols() -> list[str]:
    return list(_SIGS)


def _check(rc: int) -> None:
    if rc != 0:
        msg = load().lh_last_error().decode(errors="replace")
        if rc == 1:
            raise LighthouseShapeError(msg)
        raise LighthouseError(f"lighthouse_b200 error {rc}: {msg}")


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("lighthouse_b200 ops take CUDA tensors (no CPU path)")


def device_status(reset: bool = True) -> int:
    return load().lh_device_status(1 if reset else 0)


# --------------------------------------------------------------------------- geometry
def pyramid_len(N: int, L: int, p: int) -> int:
    return sum(N // p ** l for l in range(L))


def sel_len(N: int, L: int, p: int, k: int) -> int:
    return N // p ** (L - 1) + (L - 1) * p * k


# --------------------------------------------------------------------------- ops
def pyramid_score(xq, xk, xv, L: int, p: int):
    """(B,S,H,D) x3 -> pooled q/k/v (B,H,S_pool,D), scores_qk/kq (B,H,S_tot) fp32."""
    _require_cuda(xq, xk, xv)
    xq, xk, xv = xq.contiguous(), xk.contiguous(), xv.contiguous()
    B, S, H, D = xq.shape
    S_tot = pyramid_len(S, L, p)
    S_pool = S_tot - S
    pq = torch.empty(B, H, S_pool, D, dtype=xq.dtype, device=xq.device)
    pk, pv = torch.empty_like(pq), torch.empty_like(pq)
    sqk = torch.empty(B, H, S_tot, dtype=torch.float32, device=xq.device)
    skq = torch.empty_like(sqk)
    _check(load().lh_pyramid_score_fwd(_ptr(xq), _ptr(xk), _ptr(xv), LH_DTYPE[xq.dtype], B, S, H, D, L, p,
                                       _ptr(pq), _ptr(pk), _ptr(pv), _ptr(sqk), _ptr(skq), _stream()))
    return pq, pk, pv, sqk, skq


def select_topk(scores_qk, scores_kq, L: int, p: int, k: int, N: int, with_inverse: bool = True):
    """Selection indices (B,H,S_sel) int32 and inverse map (B,H,S_tot) int32."""
    _require_cuda(scores_qk, scores_kq)
    if scores_qk.shape != scores_kq.shape:
        raise AssertionError("scores_qk and scores_kq must have the same shape")
    sq = scores_qk.float().contiguous()
    sk = scores_kq.float().contiguous()
    B, H, S_tot = sq.shape
    if S_tot != pyramid_len(N, L, p):
        raise LighthouseShapeError(f"scores length {S_tot} != pyramid length {pyramid_len(N, L, p)}")
    S_sel = sel_len(N, L, p, k)
    idx = torch.empty(B, H, S_sel, dtype=torch.int32, device=sq.device)
    inv = torch.empty(B, H, S_tot, dtype=torch.int32, device=sq.device) if with_inverse else None
    _check(load().lh_select_topk(_ptr(sq), _ptr(sk), B, H, N, L, p, k, _ptr(idx), _ptr(inv), _stream()))
    return idx, inv


def build_inverse(indices, S_tot: int):
    _require_cuda(indices)
    indices = indices.to(torch.int32).contiguous()
    B, H, S_sel = indices.shape
    inv = torch.empty(B, H, S_tot, dtype=torch.int32, device=indices.device)
    _check(load().lh_build_inverse(_ptr(indices), B, H, S_sel, S_tot, _ptr(inv), _stream()))
    return inv


def gather_selected(raws, pooleds, indices):
    """raws: 3 tensors (B,S,H,D) (or None); pooleds: 3 tensors (B,H,S_pool,D)."""
    first = next(r for r in raws if r is not None)
    B, S, H, D = first.shape
    S_pool = next(p for p in pooleds if p is not None).shape[2]
    S_sel = indices.shape[-1]
    outs = [None if r is None else torch.empty(B, H, S_sel, D, dtype=r.dtype, device=r.device) for r in raws]
    raws = [None if r is None else r.contiguous() for r in raws]
    pooleds = [None if p is None else p.contiguous() for p in pooleds]
    _check(load().lh_gather_selected(*[_ptr(r) for r in raws], *[_ptr(p) for p in pooleds],
                                     LH_DTYPE[first.dtype], B, S, H, D, S_pool, _ptr(indices), S_sel,
                                     *[_ptr(o) for o in outs], _stream()))
    return outs


def _attn_operands(*ts):
    _require_cuda(*ts)
    for t in ts:
        if t.dtype != torch.bfloat16 or t.shape[-1] != 128:
            raise ValueError("attention kernels take bf16 tensors with head dim 128")
    return [t.contiguous() for t in ts]


def attn_fwd(q, k, v, scale: float, q_off: int = 0):
    """Causal attention; query row r at position q_off + r, key row c at c."""
    q, k, v = _attn_operands(q, k, v)
    B, H, S_q, D = q.shape
    S_kv = k.shape[2]
    o = torch.empty_like(q)
    lse = torch.empty(B, H, S_q, dtype=torch.float32, device=q.device)
    _check(load().lh_attn_fwd(_ptr(q), _ptr(k), _ptr(v), B, H, S_q, S_kv, q_off, D, scale, _ptr(o), _ptr(lse),
                              _stream()))
    return o, lse


def attn_merge(o1, lse1, o2, lse2):
    """Log-sum-exp merge of two partial attentions of the same queries over
    disjoint key sets: (o, lse), o bf16 (..., D), lse fp32 (...)."""
    o1, o2 = _attn_operands(o1, o2)
    lse1, lse2 = lse1.float().contiguous(), lse2.float().contiguous()
    if o1.shape != o2.shape or lse1.shape != o1.shape[:-1] or lse2.shape != lse1.shape:
        raise LighthouseShapeError("attn_merge: o1/o2 and lse1/lse2 must agree")
    o = torch.empty_like(o1)
    lse = torch.empty_like(lse1)
    _check(load().lh_attn_merge(_ptr(o1), _ptr(lse1), _ptr(o2), _ptr(lse2), lse1.numel(), o1.shape[-1], _ptr(o),
                                _ptr(lse), _stream()))
    return o, lse


def attn_bwd_workspace_size(B: int, H: int, S_q: int, S_kv: int, D: int) -> int:
    return int(load().lh_attn_bwd_workspace_size(B, H, S_q, S_kv, D))


def attn_bwd(q, k, v, o, lse, do, scale: float, q_off: int = 0):
    q, k, v, o, do = _attn_operands(q, k, v, o, do)
    B, H, S_q, D = q.shape
    S_kv = k.shape[2]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws_bytes = attn_bwd_workspace_size(B, H, S_q, S_kv, D)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    _check(load().lh_attn_bwd(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse.contiguous()), _ptr(do), B, H, S_q,
                              S_kv, q_off, D, scale, _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ws_bytes, _stream()))
    return dq, dk, dv


def scatter_fwd(attn, inverse, N_shard: int, N_total: int, L: int, p: int):
    attn = attn.contiguous()
    B, H, S_sel, D = attn.shape
    out = torch.empty(B, H, N_total, D, dtype=attn.dtype, device=attn.device)
    _check(load().lh_scatter_fwd(_ptr(attn), _ptr(inverse), LH_DTYPE[attn.dtype], B, H, S_sel, D, N_shard, N_total,
                                 L, p, _ptr(out), _stream()))
    return out


def token_major_ok(B: int, H: int, D: int, dtype) -> bool:
    """Whether the token-major scatter kernels cover this geometry."""
    row = D * (2 if dtype == torch.bfloat16 else 4)
    return row in (256, 512) and (B * H) % (32 // (row // 16)) == 0


def scatter_fwd_token_major(attn, inverse, N_shard: int, N_total: int, L: int, p: int):
    """scatter_fwd with the output as (B, N_total, H, D) (token-major)."""
    attn = attn.contiguous()
    B, H, S_sel, D = attn.shape
    out = torch.empty(B, N_total, H, D, dtype=attn.dtype, device=attn.device)
    _check(load().lh_scatter_fwd_token_major(_ptr(attn), _ptr(inverse), LH_DTYPE[attn.dtype], B, H, S_sel, D,
                                             N_shard, N_total, L, p, _ptr(out), _stream()))
    return out


def scatter_bwd_token_major(dout, indices, N_shard: int, N_total: int, L: int, p: int):
    """scatter_bwd for dout given as (B, N_total, H, D) (token-major)."""
    dout = dout.contiguous()
    B, _, H, D = dout.shape
    S_sel = indices.shape[-1]
    dattn = torch.empty(B, H, S_sel, D, dtype=dout.dtype, device=dout.device)
    _check(load().lh_scatter_bwd_token_major(_ptr(dout), _ptr(indices), LH_DTYPE[dout.dtype], B, H, S_sel, D,
                                             N_shard, N_total, L, p, _ptr(dattn), _stream()))
    return dattn


def scatter_bwd(dout, indices, N_shard: int, N_total: int, L: int, p: int):
    dout = dout.contiguous()
    B, H, _, D = dout.shape
    S_sel = indices.shape[-1]
    dattn = torch.empty(B, H, S_sel, D, dtype=dout.dtype, device=dout.device)
    _check(load().lh_scatter_bwd(_ptr(dout), _ptr(indices), LH_DTYPE[dout.dtype], B, H, S_sel, D, N_shard,
                                 N_total, L, p, _ptr(dattn), _stream()))
    return dattn


def unpool_bwd(dsels, inverse, S: int, L: int, p: int):
    first = next(d for d in dsels if d is not None)
    B, H, S_sel, D = first.shape
    dsels = [None if d is None else d.contiguous() for d in dsels]
    outs = [None if d is None else torch.empty(B, S, H, D, dtype=d.dtype, device=d.device) for d in dsels]
    _check(load().lh_unpool_bwd(*[_ptr(d) for d in dsels], _ptr(inverse), LH_DTYPE[first.dtype], B, S, H, D, L, p,
                                S_sel, *[_ptr(o) for o in outs], _stream()))
    return outs


def rope_apply(xq, xk, table, inverse: bool = False):
    """Rotary embedding of q and k (B, S, H, D) with the (S, D/2, 2) fp32 (cos, sin)
    table; returns new tensors.  inverse=True rotates by minus the angles."""
    xq, xk, table = xq.contiguous(), xk.contiguous(), table.contiguous()
    B, S, H, D = xq.shape
    if xk.shape != xq.shape or xk.dtype != xq.dtype or tuple(table.shape) != (S, D // 2, 2):
        raise LighthouseShapeError("rope: q, k and the table must agree")
    oq, ok = torch.empty_like(xq), torch.empty_like(xk)
    _check(load().lh_rope_apply(_ptr(xq), _ptr(xk), _ptr(oq), _ptr(ok), _ptr(table), LH_DTYPE[xq.dtype],
                                B, S, H, D, int(inverse), _stream()))
    return oq, ok



def simple_gla_fwd(q, k, v, g, scale: float, q2=None, k2=None):
    """Simple GLA forward (fla's chunk_simple_gla, zero initial state) of (B, T, H, 128)
    bf16 q/k/v with the (B, T, H) log-gate g; returns o, or (o, o2) when the second
    pass (q2, k2) sharing v and g is given."""
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g = g.float().contiguous()
    B, T, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape or tuple(g.shape) != (B, T, H):
        raise LighthouseShapeError("gla: q, k, v (B, T, H, D) and g (B, T, H) must agree")
    o = torch.empty_like(q)
    o2 = None
    if q2 is not None:
        q2, k2 = q2.contiguous(), k2.contiguous()
        if q2.shape != q.shape or k2.shape != q.shape:
            raise LighthouseShapeError("gla: the second pass must have the shape of the first")
        o2 = torch.empty_like(q)
    _check(load().lh_simple_gla_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(o), _ptr(q2), _ptr(k2), _ptr(o2),
                                    LH_DTYPE[q.dtype], B, T, H, D, scale, _stream()))
    return o if q2 is None else (o, o2)


# --------------------------------------------------------------------------- norm
def _on_one_device(what: str, first, *rest) -> torch.device:
    """All tensors are CUDA tensors of one device, which is returned."""
    if not first.is_cuda:
        raise ValueError("lighthouse_b200 ops take CUDA tensors (no CPU path)")
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise ValueError("lighthouse_b200 ops take CUDA tensors (no CPU path)")
            raise ValueError(f"{what}: tensors on different devices: {first.device} and {t.device}")
    return first.device


def _call(dev: torch.device, name: str, *args) -> None:
    """Entry point `name` with the device's current stream as its last argument,
    the device being current meanwhile."""
    fn = getattr(_lib or load(), name)
    index = dev.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _check(rc)


def _dense16(t):
    """t as a contiguous tensor whose first element is 16-byte aligned."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _norm_check(what, x, residual, weight):
    shape = x.shape
    D = shape[-1] if shape else 0
    if weight.shape != (D,) or (residual is not None and residual.shape != shape):
        raise LighthouseShapeError(f"{what}: x and residual (..., D) and weight (D) must agree")
    if x.dtype not in LH_DTYPE or weight.dtype not in LH_DTYPE or (
            residual is not None and residual.dtype not in LH_DTYPE):
        raise ValueError(f"{what}: bf16 and fp32 tensors only")
    if D % 8 or not 8 <= D <= 16384:
        raise LighthouseShapeError(f"{what}: D must be a multiple of 8 and at most 16384, got {D}")
    return x.numel() // D, D


def rms_norm_fwd(x, residual, weight, eps: float, out_dtype, group: int = 0, with_rstd: bool = True):
    """RMS norm of h = x + residual ((..., D), residual may be None) -> (y, scale, h, rstd).

    out_dtype torch.float8_e4m3fn gives y in 8 bits and scale (..., 1), or
    (..., ceil(D / 128)) with group 128; scale is None otherwise.  h is None
    without a residual, rstd (rows) fp32 is None unless asked for."""
    N, D = _norm_check("rms_norm", x, residual, weight)
    fp8 = out_dtype == torch.float8_e4m3fn
    if not fp8 and out_dtype not in LH_DTYPE:
        raise ValueError(f"rms_norm: out_dtype must be bf16, fp32 or float8_e4m3fn, got {out_dtype}")
    if group != 0 and not (fp8 and group == 128):
        raise ValueError("rms_norm: scales per row (group 0) or per 128 columns (group 128)")
    if fp8 and with_rstd:                        # the callers that want rstd return no scales
        raise ValueError("rms_norm: an 8-bit output is nothing without its scales: rms_norm_fp8")
    dev = _on_one_device("rms_norm", x, residual, weight)
    y = torch.empty_like(x, dtype=out_dtype, memory_format=_DENSE)
    scale = h = rstd = None
    if fp8:
        scale = torch.empty(*x.shape[:-1], (D + 127) // 128 if group else 1, dtype=torch.float32, device=dev)
    if residual is not None:
        h = torch.empty_like(residual, memory_format=_DENSE)
    if with_rstd:
        rstd = torch.empty(N, dtype=torch.float32, device=dev)
    if N:
        x, weight = _dense16(x), _dense16(weight)
        r_ptr = h_ptr = None
        r_dtype = 0
        if residual is not None:
            residual = _dense16(residual)
            r_ptr, r_dtype, h_ptr = residual.data_ptr(), LH_DTYPE[residual.dtype], h.data_ptr()
        _call(dev, "lh_rms_norm_fwd", x.data_ptr(), LH_DTYPE[x.dtype], r_ptr, r_dtype, weight.data_ptr(),
              LH_DTYPE[weight.dtype], N, D, eps, y.data_ptr(), 2 if fp8 else LH_DTYPE[out_dtype],
              scale.data_ptr() if fp8 else None, group, h_ptr, rstd.data_ptr() if with_rstd else None)
    return y, scale, h, rstd


def rms_norm_bwd(dy, dh, h, weight, rstd, dx_dtype, with_dres: bool):
    """Backward of rms_norm_fwd: (dx, dres, dw); dh may be None, dres is None unless asked for."""
    N, D = _norm_check("rms_norm_bwd", h, dy, weight)
    if dx_dtype not in LH_DTYPE or (dh is not None and (dh.shape != h.shape or dh.dtype != h.dtype)):
        raise LighthouseShapeError("rms_norm_bwd: dh must have the shape and type of h")
    dev = _on_one_device("rms_norm_bwd", h, dy, dh, weight, rstd)
    if rstd.dtype != torch.float32 or rstd.numel() != N:
        raise LighthouseShapeError("rms_norm_bwd: rstd must be fp32, one per row")
    dx = torch.empty_like(h, dtype=dx_dtype, memory_format=_DENSE)
    dres = torch.empty_like(h, memory_format=_DENSE) if with_dres else None
    if not N:
        return dx, dres, torch.zeros_like(weight)
    dw = torch.empty_like(weight, memory_format=_DENSE)
    dy, h, weight, rstd = _dense16(dy), _dense16(h), _dense16(weight), rstd.contiguous()
    dh = None if dh is None else _dense16(dh)
    ws_bytes = load().lh_rms_norm_bwd_workspace_size(N, D)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call(dev, "lh_rms_norm_bwd", dy.data_ptr(), LH_DTYPE[dy.dtype], _ptr(dh), h.data_ptr(), LH_DTYPE[h.dtype],
          weight.data_ptr(), LH_DTYPE[weight.dtype], rstd.data_ptr(), N, D, dx.data_ptr(), LH_DTYPE[dx_dtype], _ptr(dres),
          dw.data_ptr(), ws.data_ptr(), ws_bytes)
    return dx, dres, dw


# --------------------------------------------------------------------------- losses of an output projection
def _loss_check(what, hidden, weight, reduction):
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise LighthouseShapeError(f"{what}: hidden (N, D) and weight (V, D) must agree")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"{what}: hidden and weight must be bf16, got {hidden.dtype} and {weight.dtype}")
    N, D = hidden.shape
    V = weight.shape[0]
    if D % 8 or not 8 <= D <= 65536 or not 1 <= V <= 1 << 22 or N > 1 << 22:
        raise LighthouseShapeError(f"{what}: D must be a multiple of 8 and at most 65536, V in [1, 2^22], N at most "
                                   f"2^22; got D {D}, V {V}, N {N}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"{what}: reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    return N, V, D


def _loss_out(N, reduction, dev):
    """The loss's tensor; a reduced loss over no positions is 0."""
    loss = torch.empty((N,) if reduction == "none" else (), dtype=torch.float32, device=dev)
    return loss if N else loss.zero_()


def _loss_ws(N, V, D, K, backward, dev):
    n = load().lh_linear_loss_workspace_size(N, V, D, K, backward)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def kept_size(N: int, V: int, K: int, reduction: str) -> int:
    """Bytes that a loss's forward keeps for its backward."""
    return load().lh_linear_loss_kept_size(N, V, K, REDUCTIONS[reduction], 1)


def kept_bytes(N, V, K, reduction: str):
    """kept_size as an expression, for sizes that are symbols of a traced graph: lse and scale of
    a row, its targets' values and sorted indices, the packed rows' numbers, and G / c of one-tile
    rows, each from a multiple of 256 bytes on (linear_loss.cu, Kept)."""
    up = lambda n: (n + 255) // 256 * 256
    at_least = lambda n: torch.sym_min(torch.sym_max(N - n + 1, 0), 1)       # 1 or 0, without a branch on N
    Kp = (K + 3) // 4 * 4
    whole = at_least(65) * up(512 * N) if V <= 256 and REDUCTIONS[reduction] else 0
    return at_least(1) * (2 * up(4 * N) + 2 * up(4) + up(4 * N * (Kp if K else 1)) + up(4 * N * Kp) + up(8 * N + 4) + whole)


def linear_xent_fwd(hidden, weight, target, ignore_index: int, reduction: str):
    """Softmax cross entropy of hidden (N, D) @ weight (V, D)^T against target (N) int64 ->
    (loss, kept); kept (uint8) is the backward's."""
    N, V, D = _loss_check("linear_xent", hidden, weight, reduction)
    if target.shape != (N,) or target.dtype != torch.int64:
        raise LighthouseShapeError("linear_xent: target must be (N) int64")
    dev = _on_one_device("linear_xent", hidden, weight, target)
    loss = _loss_out(N, reduction, dev)
    kept = torch.empty(kept_size(N, V, 0, reduction), dtype=torch.uint8, device=dev)
    if N:
        hidden, weight, target = _dense16(hidden), _dense16(weight), target.contiguous()
        ws, n = _loss_ws(N, V, D, 0, 0, dev)
        _call(dev, "lh_linear_xent_fwd", hidden.data_ptr(), weight.data_ptr(), target.data_ptr(), ignore_index, N, V, D,
              REDUCTIONS[reduction], loss.data_ptr(), kept.data_ptr(), kept.numel(), ws.data_ptr(), n)
    return loss, kept


def _loss_bwd_check(what, hidden, weight, kept, gout, reduction, K, *rest):
    N, V, D = _loss_check(what, hidden, weight, reduction)
    if gout.dtype != torch.float32 or gout.numel() != (N if reduction == "none" else 1):
        raise LighthouseShapeError(f"{what}: the loss's gradient must be fp32, one value (reduced) or N")
    if kept.dtype != torch.uint8 or kept.shape != (kept_size(N, V, K, reduction),) or not kept.is_contiguous():
        raise LighthouseShapeError(f"{what}: kept must be the forward's")
    return N, _on_one_device(what, hidden, weight, kept, gout, *rest)


def linear_xent_bwd(hidden, weight, target, kept, gout, reduction: str):
    """Gradients (dhidden, dweight) of linear_xent_fwd."""
    N, dev = _loss_bwd_check("linear_xent_bwd", hidden, weight, kept, gout, reduction, 0, target)
    if target.shape != (N,) or target.dtype != torch.int64:
        raise LighthouseShapeError("linear_xent_bwd: target must be (N) int64")
    dh, dw = torch.empty_like(hidden, memory_format=_DENSE), torch.empty_like(weight, memory_format=_DENSE)
    if not N:
        return dh, dw.zero_()
    V, D = weight.shape
    hidden, weight = _dense16(hidden), _dense16(weight)
    ws, n = _loss_ws(N, V, D, 0, 1, dev)
    _call(dev, "lh_linear_xent_bwd", hidden.data_ptr(), weight.data_ptr(), target.contiguous().data_ptr(), N, V, D,
          REDUCTIONS[reduction], kept.data_ptr(), kept.numel(), gout.contiguous().data_ptr(), dh.data_ptr(), dw.data_ptr(),
          ws.data_ptr(), n)
    return dh, dw


def linear_distill_fwd(hidden, weight, teacher_logits, teacher_indices, temperature: float, reduction: str):
    """Distillation of hidden (N, D) @ weight (V, D)^T from a teacher's K logits (N, K) bf16 / fp32 at
    indices (N, K) int64 -> (loss, kept); kept (uint8) is the backward's."""
    N, V, D = _loss_check("linear_distill", hidden, weight, reduction)
    if teacher_logits.dim() != 2 or teacher_logits.shape[0] != N or teacher_indices.shape != teacher_logits.shape:
        raise LighthouseShapeError("linear_distill: teacher logits and indices must be (N, K)")
    K = teacher_logits.shape[1]
    if not 1 <= K <= 256:
        raise LighthouseShapeError(f"linear_distill: K must be in [1, 256], got {K}")
    if teacher_logits.dtype not in LH_DTYPE or teacher_indices.dtype != torch.int64:
        raise ValueError("linear_distill: teacher logits must be bf16 or fp32, indices int64")
    if not 1e-18 <= temperature <= 1e18:         # its square and inverse are fp32 numbers
        raise ValueError(f"linear_distill: temperature must be in [1e-18, 1e18], got {temperature}")
    dev = _on_one_device("linear_distill", hidden, weight, teacher_logits, teacher_indices)
    loss = _loss_out(N, reduction, dev)
    kept = torch.empty(kept_size(N, V, K, reduction), dtype=torch.uint8, device=dev)
    if N:
        hidden, weight = _dense16(hidden), _dense16(weight)
        teacher_logits, teacher_indices = teacher_logits.contiguous(), teacher_indices.contiguous()
        ws, n = _loss_ws(N, V, D, K, 0, dev)
        _call(dev, "lh_linear_distill_fwd", hidden.data_ptr(), weight.data_ptr(), teacher_logits.data_ptr(),
              LH_DTYPE[teacher_logits.dtype], teacher_indices.data_ptr(), N, V, D, K, temperature, REDUCTIONS[reduction],
              loss.data_ptr(), kept.data_ptr(), kept.numel(), ws.data_ptr(), n)
    return loss, kept


def linear_distill_bwd(hidden, weight, kept, gout, K: int, temperature: float, reduction: str):
    """Gradients (dhidden, dweight) of linear_distill_fwd."""
    N, dev = _loss_bwd_check("linear_distill_bwd", hidden, weight, kept, gout, reduction, K)
    dh, dw = torch.empty_like(hidden, memory_format=_DENSE), torch.empty_like(weight, memory_format=_DENSE)
    if not N:
        return dh, dw.zero_()
    V, D = weight.shape
    hidden, weight = _dense16(hidden), _dense16(weight)
    ws, n = _loss_ws(N, V, D, K, 1, dev)
    _call(dev, "lh_linear_distill_bwd", hidden.data_ptr(), weight.data_ptr(), N, V, D, K, temperature,
          REDUCTIONS[reduction], kept.data_ptr(), kept.numel(), gout.contiguous().data_ptr(), dh.data_ptr(), dw.data_ptr(),
          ws.data_ptr(), n)
    return dh, dw
