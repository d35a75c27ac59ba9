"""Host-side operators of the gfx950 mul_mat backend on top of the C ABI.

Function names, argument order, shape contracts and error behaviour follow the reference's graph-op
builders (src/core/ComputeGraphHelper.cpp:262-345, 1748-1764) and its dispatch wrapper
(src/backend/CUDAKernels.cpp:717-847).  torch is used for device memory and streams only; all
arithmetic happens in the HIP library.  Shapes are written numpy style (outermost first), i.e. the
reverse of the reference's ``dims[0]``-innermost notation.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import math
import os
import sys

import torch

from . import cabi

QK = 32
BLOCK_BYTES = 34
WTYPE_Q8_0, WTYPE_Q8_1, WTYPE_Q8_0R, WTYPE_Q8_0M = 0, 1, 2, 3

# What a call asks of torch beside its kernel -- the current device, its stream, the addresses -- costs more than a small
# kernel: a projection of 408 x 256 -> 256, whose kernel takes 3.7 us, took 10.3 through this module with torch's public
# forms (a stream object alone 2.7 us, is_available and current_device 0.8) and 6.1 with the functions beneath them.  That is the
# long way; ordinary calls go through native code (csrc/host_calls.cpp) in 4.2.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _load_host_calls():
    """The native host side of the operators below (csrc/host_calls.cpp), or None where it was not built for this torch and Python
    (another one's tensors may lie differently): every operator then does its call itself, as it does any call that is not ordinary."""
    path = os.path.join(os.path.dirname(cabi.LIB_PATH), "_host_calls.so")
    try:
        built_for = C.string_at(C.addressof(C.c_char.in_dll(C.CDLL(path), "host_calls_built_for"))).decode()
        if built_for != f"torch-{torch.__version__}-python-{sys.version_info[0]}.{sys.version_info[1]}":
            return None
        loader = importlib.machinery.ExtensionFileLoader("_host_calls", path)
        spec = importlib.util.spec_from_file_location("_host_calls", path, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        return module
    except (ImportError, OSError, ValueError):          # not there, other symbols, no such mark
        return None


def _not_taken(*_):
    return None


_host = _load_host_calls()
# each takes a call of its operator if everything about it is ordinary and answers None otherwise
(_host_mul_mat, _host_mul_mat_f16, _host_mul_mat_q8, _host_outer_product_mean, _host_outer_prod_mean_back, _host_tri_mul, _host_tri_mul_back,
 _host_flash_attn_forward, _host_flash_attn_backward, _host_mul_mat_i8, _host_qk_norm_rope, _host_qk_norm_rope_backward, _host_newton_schulz) = (
    getattr(_host, name, _not_taken) for name in ("mul_mat", "mul_mat_f16", "mul_mat_q8", "outer_product_mean", "outer_prod_mean_back", "tri_mul",
                                                   "tri_mul_back", "flash_attn_forward", "flash_attn_backward", "mul_mat_i8", "qk_norm_rope",
                                                   "qk_norm_rope_backward", "newton_schulz"))
_HOST_LAUNCHERS = ("mul_mat_hip", "mul_mat_f16_hip", "mul_mat_q8_hip", "mul_mat_q8_ex_hip", "outer_prod_mean_hip", "outer_prod_mean_back_hip",
                   "tri_mul_hip", "tri_mul_back_hip", "flash_attn_forward_ex_hip", "flash_attn_backward_hip", "mul_mat_i8_hip",
                   "mul_mat_i8_workspace_hip", "qk_norm_rope_hip", "qk_norm_rope_back_hip", "qk_norm_rope_back_workspace_hip", "newton_schulz_hip",
                   "newton_schulz_workspace_hip")

_initialised = set()                                  # devices ppml_hip_init has run on in this process


def _forget_devices():
    _initialised.clear()
    if _host is not None:
        _host.forget()


os.register_at_fork(after_in_child=_forget_devices)      # (torch refuses the GPU in a forked child: the long way round says so)


def _lib():
    if _initialised and _current_device() in _initialised:
        return cabi.load()
    lib = cabi.load()
    if not torch.cuda.is_available():
        raise RuntimeError("the gfx950 backend needs a GPU; there is no CPU path")
    dev = torch.cuda.current_device()
    cabi.check("ppml_hip_init", lib.ppml_hip_init(dev))
    if _host is not None:
        for name in _HOST_LAUNCHERS:
            _host.bind(name, C.cast(getattr(lib, name), C.c_void_p).value)
        _host.ready(dev)
    _initialised.add(dev)
    return lib


def _stream() -> int:
    return _raw_stream(_current_device())


def _dev_f32(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda or t.dtype != torch.float32:
        raise TypeError(f"{name} must be a float32 device tensor")
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


Q8_PATH_NAMES = {0: "general", 1: "weight-stationary", 2: "low-latency", 3: "tiled"}


def last_q8_path() -> str:
    """Kernel family that served this thread's last mul_mat_q8 call (``ppml_hip_q8_last_path``)."""
    return Q8_PATH_NAMES[_lib().ppml_hip_q8_last_path()]


def mulmat_stats_enable(on: bool) -> bool:
    """Switches the MUL_MAT statistics (include/ppml/MulMatStats.h) on or off; returns the previous state."""
    return bool(cabi.load().ppml_hip_mulmat_stats_enable(1 if on else 0))


def mulmat_stats_rows():
    """The statistics table as a list of dicts {path, M, K, N, calls, ms}, ordered by (path, M, K, N)."""
    lib = cabi.load()
    n = lib.ppml_hip_mulmat_stats_rows(None, 0)
    rows = (cabi.MulMatStat * max(n, 1))()
    n = min(lib.ppml_hip_mulmat_stats_rows(C.cast(rows, C.c_void_p), n), n)
    return [{"path": rows[i].path.decode(), "M": rows[i].M, "K": rows[i].K, "N": rows[i].N, "calls": rows[i].calls,
             "ms": rows[i].ms} for i in range(n)]


def synchronize() -> None:
    cabi.check("ppml_hip_synchronize", _lib().ppml_hip_synchronize())


# ----------------------------------------------------------------------------- f32
def set_f32_arithmetic(mode: str) -> str:
    """Matrix pipe of the f32 contractions: "split" (default: bf16 pipe, exact three-way split) or "fp32"
    (fp32 MFMA).  Returns the previous setting."""
    before = _lib().ppml_hip_set_f32_arithmetic({"split": 0, "fp32": 1}[mode])
    return "fp32" if before == 1 else "split"


def mul_mat(a: torch.Tensor, b: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """a [M,K], b [N,K] -> [M,N] = a @ b.T (+ bias[N]); src/core/ComputeGraphHelper.cpp:262-314."""
    out = _host_mul_mat(a, b, bias)
    if out is not None:
        return out
    a, b = _dev_f32(a, "a"), _dev_f32(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"mul_mat: inner dimensions differ, a {tuple(a.shape)} b {tuple(b.shape)}")
    M, K = a.shape
    N = b.shape[0]
    if bias is not None:
        bias = _dev_f32(bias, "bias")
        if bias.numel() != N:          # the reference drops a bias of the wrong length with a message
            raise ValueError(f"mul_mat: bias has {bias.numel()} elements, expected {N}")
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    lib = _lib()
    cabi.check("mul_mat_hip", lib.mul_mat_hip(_ptr(a), _ptr(b), _ptr(out), M, K, N, _ptr(bias), _stream()))
    return out


def mul_mat_f16(a: torch.Tensor, b: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """F16 x F16 -> F32 mul_mat: a [M,K], b [N,K] float16 on the device, binary32 products and sum,
    bias (f32 [N]) added to the finished sum (src/backend/CPUKernels.cpp:646-672)."""
    out = _host_mul_mat_f16(a, b, bias)
    if out is not None:
        return out
    for t, name in ((a, "a"), (b, "b")):
        if not t.is_cuda or t.dtype != torch.float16:
            raise TypeError(f"mul_mat_f16: {name} must be a float16 tensor on the device")
    a, b = a.contiguous(), b.contiguous()
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"mul_mat_f16: a {tuple(a.shape)} and b {tuple(b.shape)} do not share K")
    M, K = a.shape
    N = b.shape[0]
    if bias is not None:
        bias = _dev_f32(bias, "bias")
        if bias.numel() != N:
            raise ValueError("mul_mat_f16: bias length is not N")
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    cabi.check("mul_mat_f16_hip", _lib().mul_mat_f16_hip(_ptr(a), _ptr(b), _ptr(out), M, K, N, _ptr(bias), _stream()))
    return out


def mul_mat_tn(a: torch.Tensor, b: torch.Tensor, alpha: float = 1.0) -> torch.Tensor:
    """a [K,M], b [K,N] -> alpha * a.T @ b (the dense form of outer-product-mean)."""
    a, b = _dev_f32(a, "a"), _dev_f32(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[0]:
        raise ValueError("mul_mat_tn: contraction lengths differ")
    K, M = a.shape
    N = b.shape[1]
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    cabi.check("mul_mat_tn_hip", _lib().mul_mat_tn_hip(_ptr(a), _ptr(b), _ptr(out), M, K, N, alpha, _stream()))
    return out


def out_prod(a: torch.Tensor, b: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """a [ne03,ne02,K,ne00], b [ne13,ne12,K,ne10] -> [ne13,ne12,ne10,ne00];
    src/core/ComputeGraphHelper.cpp:318-345, broadcast of src/backend/CPUKernels.cpp:836-858.
    ``scale`` fuses the OP_SCALE node that follows in the attention path.  ``out``: a contiguous float32
    device tensor of the result's size to write into (any 4-byte alignment) instead of a new one."""
    a, b = _dev_f32(a, "a"), _dev_f32(b, "b")
    while a.dim() < 4:
        a = a.unsqueeze(0)
    while b.dim() < 4:
        b = b.unsqueeze(0)
    ne03, ne02, ne01, ne00 = a.shape
    ne13, ne12, ne11, ne10 = b.shape
    if ne01 != ne11:
        raise ValueError(f"out_prod: contraction dims differ ({ne01} vs {ne11})")
    ne0, ne1, ne2, ne3 = ne00, ne10, max(ne02, ne12), max(ne03, ne13)
    if out is None:
        out = torch.empty((ne3, ne2, ne1, ne0), dtype=torch.float32, device=a.device)
    elif out.dtype != torch.float32 or out.device != a.device or not out.is_contiguous() or out.numel() != ne0 * ne1 * ne2 * ne3:
        raise ValueError("out_prod: `out` must be a contiguous float32 tensor of the result's size on the operands' device")
    else:
        out = out.view(ne3, ne2, ne1, ne0)
    dims = [ne00, ne01, ne02, ne03, ne10, ne11, ne12, ne13, ne0, ne1, ne2, ne3]
    lib = _lib()
    if scale is None:
        rc = lib.out_prod_hip(_ptr(a), _ptr(b), _ptr(out), *dims, _stream())
    else:
        rc = lib.out_prod_scaled_hip(_ptr(a), _ptr(b), _ptr(out), *dims, scale, _stream())
    cabi.check("out_prod_hip", rc)
    return out


def attention_logits(k: torch.Tensor, q: torch.Tensor, head_dim: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out_prod(K, Q) * 1/sqrt(head_dim), steps 1-2 of src/modules/Attention.cpp:264-270."""
    d = k.shape[-2] if head_dim is None else head_dim
    return out_prod(k, q, scale=1.0 / math.sqrt(float(d)), out=out)


def outer_product_mean(left: torch.Tensor, right: torch.Tensor, D: int, L: int, N: int, B: int) -> torch.Tensor:
    """Graph form (src/core/ComputeGraphHelper.cpp:1748-1764): flat buffers indexed as
    src/backend/CPUKernels.cpp:1006-1028; returns the flat [D*D*L*L*B] result."""
    out = _host_outer_product_mean(left, right, D, L, N, B)
    if out is not None:
        return out
    left, right = _dev_f32(left, "left").reshape(-1), _dev_f32(right, "right").reshape(-1)
    if left.numel() != D * L * N * B or right.numel() != D * L * N * B:
        raise ValueError("outer_product_mean: operand size does not match D*L*N*B")
    out = torch.empty(D * D * L * L * B, dtype=torch.float32, device=left.device)
    cabi.check("outer_prod_mean_hip",
               _lib().outer_prod_mean_hip(_ptr(left), _ptr(right), _ptr(out), D, L, N, B, 1.0 / float(N), _stream()))
    return out


def outer_prod_mean_back(grad: torch.Tensor, left: torch.Tensor, right: torch.Tensor, D: int, L: int, N: int, B: int,
                         want_left: bool = True, want_right: bool = True):
    """Gradients of outer_prod_mean's operands (src/backend/CPUKernels.cpp:1034-1105); flat tensors."""
    if want_left is True and want_right is True:
        both = _host_outer_prod_mean_back(grad, left, right, D, L, N, B)
        if both is not None:
            return both
    grad, left, right = _dev_f32(grad, "grad"), _dev_f32(left, "left"), _dev_f32(right, "right")
    if grad.numel() != D * D * L * L * B or left.numel() != D * L * N * B or right.numel() != D * L * N * B:
        raise ValueError("outer_prod_mean_back: operand size does not match D, L, N, B")
    if not (want_left or want_right):
        raise ValueError("outer_prod_mean_back: at least one gradient must be wanted")
    gl = torch.empty(D * L * N * B, dtype=torch.float32, device=grad.device) if want_left else None
    gr = torch.empty(D * L * N * B, dtype=torch.float32, device=grad.device) if want_right else None
    cabi.check("outer_prod_mean_back_hip",
               _lib().outer_prod_mean_back_hip(_ptr(grad), _ptr(left), _ptr(right), _ptr(gl) if gl is not None else None,
                                               _ptr(gr) if gr is not None else None, D, L, N, B, 1.0 / float(N), _stream()))
    return gl, gr


def outer_product_mean_value(left: torch.Tensor, right: torch.Tensor) -> torch.Tensor:
    """Value form (src/ops/MathUtils.cpp:387-437): (B,N,L,D) x (B,N,L,D) -> (B,L,L,D*D)."""
    left, right = _dev_f32(left, "left"), _dev_f32(right, "right")
    if left.dim() != 4 or right.dim() != 4:
        raise ValueError("outer_product_mean expects 4D tensors")
    if left.shape[0] != right.shape[0] or left.shape[2] != right.shape[2] or left.shape[3] != right.shape[3] \
            or left.shape[1] != right.shape[1]:
        raise ValueError("outer_product_mean dimension mismatch: batch/residue/feature dims differ")
    B, N, L, D = left.shape
    out = torch.empty((B, L, L, D * D), dtype=torch.float32, device=left.device)
    cabi.check("outer_product_mean_value_hip",
               _lib().outer_product_mean_value_hip(_ptr(left), _ptr(right), _ptr(out), B, N, L, D, _stream()))
    return out


def tri_mul(left: torch.Tensor, right: torch.Tensor, D: int, I: int, J: int, K: int, B: int, L: float,
            outgoing: bool = True) -> torch.Tensor:
    """Triangle multiplication, graph form (src/backend/CPUKernels.cpp:907-968): flat operands indexed as the
    kernel does (d outermost, b innermost); returns the flat [D*I*J*B] result incl. the 1/L and the finite guard."""
    out = _host_tri_mul(left, right, D, I, J, K, B, L, outgoing)
    if out is not None:
        return out
    left, right = _dev_f32(left, "left"), _dev_f32(right, "right")
    if L == 0:
        raise ValueError("tri_mul: L must not be zero")
    if left.numel() != D * I * K * B or right.numel() != D * J * K * B:
        raise ValueError("tri_mul: operand size does not match D, I, J, K, B")
    out = torch.empty(D * I * J * B, dtype=torch.float32, device=left.device)
    cabi.check("tri_mul_hip", _lib().tri_mul_hip(_ptr(left), _ptr(right), _ptr(out), D, I, J, K, B, 1.0 / float(L),
                                                 int(outgoing), _stream()))
    return out


def tri_mul_back(grad: torch.Tensor, left: torch.Tensor, right: torch.Tensor, D: int, I: int, J: int, K: int, B: int,
                 L: float, outgoing: bool = True, want_left: bool = True, want_right: bool = True):
    """Gradients of tri_mul's operands (src/backend/CPUKernels.cpp:1238-1367); flat tensors, same indexing."""
    if want_left is True and want_right is True:
        both = _host_tri_mul_back(grad, left, right, D, I, J, K, B, L, outgoing)
        if both is not None:
            return both
    grad, left, right = _dev_f32(grad, "grad"), _dev_f32(left, "left"), _dev_f32(right, "right")
    if L == 0 or not (want_left or want_right):
        raise ValueError("tri_mul_back: L must not be zero and at least one gradient must be wanted")
    if grad.numel() != D * I * J * B or left.numel() != D * I * K * B or right.numel() != D * J * K * B:
        raise ValueError("tri_mul_back: operand size does not match D, I, J, K, B")
    gl = torch.empty(D * I * K * B, dtype=torch.float32, device=grad.device) if want_left else None
    gr = torch.empty(D * J * K * B, dtype=torch.float32, device=grad.device) if want_right else None
    cabi.check("tri_mul_back_hip",
               _lib().tri_mul_back_hip(_ptr(grad), _ptr(left), _ptr(right), _ptr(gl) if gl is not None else None,
                                       _ptr(gr) if gr is not None else None, D, I, J, K, B, 1.0 / float(L), int(outgoing), _stream()))
    return gl, gr


def flash_attn_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor | None = None,
                       causal: bool = False, scale: float = 0.0, eps: float = 1e-9, Bc: int = 64,
                       want_lse: bool = True, in_ld: bool = False, out_ld: bool = False):
    """Fused attention forward (include/ppml/FlashAttn.h:8-65): Q, K, V (B,h,L,d), bias (B,h,L,L) or None
    -> O (B,h,L,d) and LSE (B,h,L) (None when not wanted).  in_ld: Q, K, V are (B,h,d,L) instead (the graph
    tensors before their layout bridge); out_ld: O is returned as (B,h,d,L)."""
    if not in_ld and not out_ld:
        both = _host_flash_attn_forward(q, k, v, bias, causal, scale, eps, Bc, want_lse)
        if both is not None:
            return both
    q, k, v = _dev_f32(q, "q"), _dev_f32(k, "k"), _dev_f32(v, "v")
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("flash_attn_forward: Q, K and V must be 4-D tensors of one shape (B,h,L,d)")
    B, h, L, d = q.shape
    if in_ld:
        L, d = d, L
    if bias is not None:
        bias = _dev_f32(bias, "bias")
        if tuple(bias.shape) != (B, h, L, L):
            raise ValueError("flash_attn_forward: bias must be (B,h,L,L)")
    o = torch.empty((B, h, d, L) if out_ld else (B, h, L, d), dtype=torch.float32, device=q.device)
    lse = torch.empty((B, h, L), dtype=torch.float32, device=q.device) if want_lse else None
    cabi.check("flash_attn_forward_ex_hip",
               _lib().flash_attn_forward_ex_hip(B, h, L, d, int(causal), scale, eps, Bc, _ptr(q), _ptr(k), _ptr(v),
                                                _ptr(bias) if bias is not None else None, _ptr(o),
                                                _ptr(lse) if lse is not None else None,
                                                int(in_ld) | (int(out_ld) << 1), _stream()))
    return o, lse


def flash_attn_backward(q, k, v, bias, o, do, lse, causal: bool = False, scale: float = 0.0,
                        want=("dq", "dk", "dv", "dbias")):
    """Fused attention backward (include/ppml/FlashAttn.h:67-101): returns (dQ, dK, dV, dbias), None for the
    gradients not named in `want`."""
    want_dq, want_dk, want_dv, want_dbias = "dq" in want, "dk" in want, "dv" in want, "dbias" in want      # (once: it may be an iterator)
    grads = _host_flash_attn_backward(q, k, v, bias, o, do, lse, causal, scale, want_dq | want_dk << 1 | want_dv << 2 | want_dbias << 3)
    if grads is not None:
        return grads
    q, k, v, o, do, lse = (_dev_f32(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (do, "do"), (lse, "lse")))
    B, h, L, d = q.shape
    if bias is not None:
        bias = _dev_f32(bias, "bias")
    dq = torch.empty_like(q) if want_dq else None
    dk = torch.empty_like(q) if want_dk else None
    dv = torch.empty_like(q) if want_dv else None
    db = torch.empty((B, h, L, L), dtype=torch.float32, device=q.device) if want_dbias else None
    opt = lambda t: _ptr(t) if t is not None else None      # noqa: E731
    cabi.check("flash_attn_backward_hip",
               _lib().flash_attn_backward_hip(B, h, L, d, int(causal), scale, _ptr(q), _ptr(k), _ptr(v), opt(bias), _ptr(o),
                                              _ptr(do), _ptr(lse), opt(dq), opt(dk), opt(dv), opt(db), _stream()))
    return dq, dk, dv, db


def permute(x: torch.Tensor, axes) -> torch.Tensor:
    """The reference's permute as a copy (src/backend/CPUKernels.cpp:1669-1717).  `x` is a dense tensor whose
    LAST torch dimension is the reference's dims[0]; `axes` is in the reference's numbering: dimension p of
    the result (dims[p]) is dimension axes[p] of the source."""
    x = _dev_f32(x, "x")
    nd = x.dim()
    axes = [int(a) for a in axes]
    if nd < 1 or nd > 4 or sorted(axes) != list(range(nd)):
        raise ValueError("permute: axes must be a permutation of the tensor's dimensions (at most 4)")
    sd = list(x.shape[::-1]) + [1] * (4 - nd)                      # reference order: innermost first
    dd = [sd[axes[p]] for p in range(nd)] + [1] * (4 - nd)
    ax = axes + list(range(nd, 4))
    out = torch.empty(tuple(dd[:nd][::-1]), dtype=torch.float32, device=x.device)
    cabi.check("permute_hip", _lib().permute_hip(_ptr(x), _ptr(out), x.numel(), nd, *ax, *sd, *dd, _stream()))
    return out


def repeat_back(a: torch.Tensor, b_shape) -> torch.Tensor:
    """The builder's ``repeat_back(a, b)`` (src/core/ComputeGraphHelper.cpp:114-133) with the kernel's index rule
    (src/backend/CPUKernels.cpp:2091-2148): `a` summed over the copies that a broadcast of a tensor of shape
    `b_shape` made.  Shapes are torch order (LAST dimension = the reference's dims[0]); dimension d of the
    result meets dimension d of `a` counted from dims[0], missing dimensions count as 1."""
    a = _dev_f32(a, "a")
    b_shape = tuple(int(d) for d in b_shape)
    if a.dim() < 1 or a.dim() > 4 or len(b_shape) < 1 or len(b_shape) > 4:
        raise ValueError("repeat_back: tensors have 1 to 4 dimensions")
    sd = list(a.shape[::-1]) + [1] * (4 - a.dim())
    dd = list(b_shape[::-1]) + [1] * (4 - len(b_shape))
    off = 0 if a.dim() >= len(b_shape) else a.dim() - len(b_shape)
    rd = []
    for d in range(4):
        sdim = sd[d + off] if 0 <= d + off < 4 else 1
        rd.append(sdim // dd[d] if dd[d] > 0 else 1)
    out = torch.empty(b_shape, dtype=torch.float32, device=a.device)
    cabi.check("repeat_back_hip", _lib().repeat_back_hip(_ptr(a), _ptr(out), *sd, *dd, *rd, _stream()))
    return out


# ----------------------------------------------------------------------------- Q8_0
def scale(x: torch.Tensor, s: float) -> torch.Tensor:
    """The reference's scale() node (src/core/ComputeGraphHelper.cpp:235-243; kernel src/backend/CPUKernels.cpp:1737-1754)."""
    x = _dev_f32(x, "x")
    out = torch.empty_like(x)
    cabi.check("scale_hip", _lib().scale_hip(_ptr(x), _ptr(out), float(s), x.numel(), _stream()))
    return out


UNARY_OP_RELU = 4


def relu(x: torch.Tensor) -> torch.Tensor:
    """The reference's relu() node (src/core/ComputeGraphHelper.cpp:513-520; kernel src/backend/CPUKernels.cpp:2649-2657)."""
    x = _dev_f32(x, "x")
    out = torch.empty_like(x)
    cabi.check("unary_hip", _lib().unary_hip(_ptr(x), _ptr(out), x.numel(), UNARY_OP_RELU, _stream()))
    return out


ELEMWISE_OPS = {"add": 0, "sub": 1, "mul": 2, "div": 3}


def bcast_elemwise(a: torch.Tensor, b: torch.Tensor, op: str = "add") -> torch.Tensor:
    """add / sub / mul / div with the reference's broadcast (src/backend/CPUKernels.cpp:446-596): the result has
    the shape of `a` (the reference's dst is a copy of src[0]'s shape, ComputeGraphHelper.cpp:61-124) and an operand
    with fewer elements repeats along the flat order, so it must cover the innermost dimensions."""
    a, b = _dev_f32(a, "a"), _dev_f32(b, "b")
    if op not in ELEMWISE_OPS:
        raise ValueError(f"bcast_elemwise: op must be one of {sorted(ELEMWISE_OPS)}")
    n = a.numel()
    if b.numel() == 0 or b.numel() > n or n % b.numel() != 0:
        raise ValueError(f"bcast_elemwise: {b.numel()} elements do not repeat into {n}")
    out = torch.empty_like(a)
    cabi.check("bcast_elemwise_hip", _lib().bcast_elemwise_hip(_ptr(a), _ptr(b), _ptr(out), n, n, b.numel(), ELEMWISE_OPS[op], _stream()))
    return out


def softmax(x: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """The reference's softmax() node over dims[0], the LAST torch dimension (src/core/ComputeGraphHelper.cpp:420-425;
    kernel src/backend/CPUKernels.cpp:1446-1467, incl. its 1 / (sum + 1e-9)).  With ``bias`` (whole rows of x's row
    length, a count that divides x's): softmax(x + bias) with the add node in front folded in, the same bits as
    softmax(bcast_elemwise(x, bias, "add"))."""
    x = _dev_f32(x, "x")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("softmax: needs a non-empty innermost dimension")
    out = torch.empty_like(x)
    N = x.shape[-1]
    M = x.numel() // N
    if bias is None:
        cabi.check("softmax_hip", _lib().softmax_hip(_ptr(x), _ptr(out), M, N, _stream()))
        return out
    bias = _dev_f32(bias, "bias")
    if bias.numel() == 0 or bias.numel() % N or M % (bias.numel() // N):
        raise ValueError("softmax: the bias must be whole rows of x's row length, a number of them that divides x's")
    cabi.check("softmax_add_hip", _lib().softmax_add_hip(_ptr(x), _ptr(bias), _ptr(out), M, N, bias.numel() // N, _stream()))
    return out


def out_prod_tt(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """out_prod of the {1,0,2,3} permutations of a and b without the copies: a [ne03,ne02,ne01,K], b [ne13,ne12,ne11,K]
    -> [ne13,ne12,ne11,ne01], contraction over the LAST torch dimension of both (src/modules/Attention.cpp:277-281:
    out_prod(permute(attn), permute(V))).  The bits of out_prod on the permuted copies."""
    a, b = _dev_f32(a, "a"), _dev_f32(b, "b")
    while a.dim() < 4:
        a = a.unsqueeze(0)
    while b.dim() < 4:
        b = b.unsqueeze(0)
    ne03, ne02, ne01, ne00 = a.shape
    ne13, ne12, ne11, ne10 = b.shape
    if ne00 != ne10:
        raise ValueError(f"out_prod_tt: contraction dims differ ({ne00} vs {ne10})")
    ne0, ne1, ne2, ne3 = ne01, ne11, max(ne02, ne12), max(ne03, ne13)
    out = torch.empty((ne3, ne2, ne1, ne0), dtype=torch.float32, device=a.device)
    dims = [ne00, ne01, ne02, ne03, ne10, ne11, ne12, ne13, ne0, ne1, ne2, ne3]
    cabi.check("out_prod_tt_hip", _lib().out_prod_tt_hip(_ptr(a), _ptr(b), _ptr(out), *dims, _stream()))
    return out


def quantize_rows_q8_0(x: torch.Tensor) -> torch.Tensor:
    """f32 [..., K] -> uint8 [..., K/32, 34] block_q8_0 records (include/ppml/QuantBlocks.h:62-79)."""
    x = _dev_f32(x, "x")
    ne = x.numel()
    if x.shape[-1] % QK:
        raise ValueError("quantize_rows_q8_0: innermost dimension is not a multiple of 32")
    out = torch.empty(x.shape[:-1] + (x.shape[-1] // QK, BLOCK_BYTES), dtype=torch.uint8, device=x.device)
    cabi.check("quantize_rows_q8_0_hip", _lib().quantize_rows_q8_0_hip(_ptr(x), _ptr(out), ne, _stream()))
    return out


def quantize_rows_q8_1(x: torch.Tensor) -> torch.Tensor:
    """f32 [..., K] -> uint8 [..., K/32, 36] block_q8_1 records, the reference's activation quantizer
    (include/ppml/QuantBlocks.h:81-111): d = vmax / -128, quants in [-128, 127], s = d * sum(q)."""
    x = _dev_f32(x, "x")
    ne = x.numel()
    if x.shape[-1] % QK:
        raise ValueError("quantize_rows_q8_1: innermost dimension is not a multiple of 32")
    out = torch.empty(x.shape[:-1] + (x.shape[-1] // QK, 36), dtype=torch.uint8, device=x.device)
    cabi.check("quantize_rows_q8_1_hip", _lib().quantize_rows_q8_1_hip(_ptr(x), _ptr(out), ne, _stream()))
    return out


def dequantize_q8_1(blocks: torch.Tensor) -> torch.Tensor:
    if not blocks.is_cuda or blocks.dtype != torch.uint8 or blocks.shape[-1] != 36:
        raise TypeError("dequantize_q8_1 expects uint8 [..., nblocks, 36] on the device")
    blocks = blocks.contiguous()
    nb = blocks.numel() // 36
    out = torch.empty(blocks.shape[:-2] + (blocks.shape[-2] * QK,), dtype=torch.float32, device=blocks.device)
    cabi.check("dequantize_q8_1_hip", _lib().dequantize_q8_1_hip(_ptr(blocks), _ptr(out), nb * QK, _stream()))
    return out


def dequantize_q8_0(blocks: torch.Tensor) -> torch.Tensor:
    if not blocks.is_cuda or blocks.dtype != torch.uint8 or blocks.shape[-1] != BLOCK_BYTES:
        raise TypeError("dequantize_q8_0 expects uint8 [..., nblocks, 34] on the device")
    blocks = blocks.contiguous()
    nb = blocks.numel() // BLOCK_BYTES
    out = torch.empty(blocks.shape[:-2] + (blocks.shape[-2] * QK,), dtype=torch.float32, device=blocks.device)
    cabi.check("dequantize_q8_0_hip", _lib().dequantize_q8_0_hip(_ptr(blocks), _ptr(out), nb * QK, _stream()))
    return out


class Q8Weight:
    """A quantized M x K weight resident on the device (rows = out features).

    ``data`` holds the bytes in layout ``wtype``; ``pack()`` returns the MFMA-fragment copy made
    once per weight, the step the reference does with its Q8_0R repack
    (src/model/PPML.cpp:4504-4528)."""

    def __init__(self, data: torch.Tensor, M: int, K: int, wtype: int):
        if K % QK:
            raise ValueError("quantized weights need K % 32 == 0 (blocks never cross a row)")
        self.data, self.M, self.K, self.wtype = data.contiguous(), M, K, wtype

    @classmethod
    def from_f32(cls, w: torch.Tensor) -> "Q8Weight":
        w = _dev_f32(w, "w")
        M, K = w.shape
        return cls(quantize_rows_q8_0(w).reshape(-1), M, K, WTYPE_Q8_0)

    def pack(self) -> "Q8Weight":
        if self.wtype == WTYPE_Q8_0M:
            return self
        lib = _lib()
        nbytes = lib.q8_weight_packed_bytes_hip(self.M, self.K)
        out = torch.empty(nbytes, dtype=torch.uint8, device=self.data.device)
        cabi.check("q8_weight_pack_hip",
                   lib.q8_weight_pack_hip(_ptr(self.data), self.wtype, self.M, self.K, _ptr(out), _stream()))
        return Q8Weight(out, self.M, self.K, WTYPE_Q8_0M)


_Q8_PATH_FLAGS = {"auto": 0, "weight-stationary": 4, "general": 4 | 8 | 256, "tiled": 4 | 8, "low-latency": 0, "low-latency-8": 16, "low-latency-16": 32, "low-latency-32": 48,
                  "weight-stationary-column-parts": 4 | 64, "weight-stationary-whole": 4 | 128}


def mul_mat_q8(w: Q8Weight, x: torch.Tensor, c_trans: int = 1, relu: bool = False,
               dump: bool = False, act: str = "q8_0", path: str = "auto", out: torch.Tensor = None):
    """Q8_0 linear: x f32 [N,K] (rows = tokens) times quantized w [M,K] -> [N,M] (c_trans=1, the
    LinearLayer orientation) or [M,N] (c_trans=0); src/backend/CUDAKernels.cpp:740-789.
    With ``dump`` also returns the kernel's own Q8_0 blocks of x and its per-block int32 sums.
    ``act`` selects the rule the activations are quantized with: "q8_0" (the CPU contract) or
    "q8_1" (what the reference's CUDA launcher does, src/cuda/MulMatQ8Kernel.cu:483-527).
    ``path`` restricts the kernel choice for a packed weight ("weight-stationary": not the low-latency kernel;
    "general": the general kernel only; "tiled": neither the low-latency nor the weight-stationary kernel, i.e. the tiled
    one wherever the problem is large enough for it; "low-latency-8" / "-16" / "-32": that unit size wherever an instance exists (32: K = 512 only);
    "weight-stationary-column-parts" / "-whole": that kernel with the columns shared out between work-groups
    wherever an instance exists / never); every choice gives the same bits.
    ``out``: a contiguous f32 device tensor of the result's shape to write into instead of a new one."""
    if out is None and dump is False and act == "q8_0" and path == "auto":
        y = _host_mul_mat_q8(w.data, x, w.M, w.K, w.wtype, c_trans, 1 if relu else 0)
        if y is not None:
            return y
    if act not in ("q8_0", "q8_1"):
        raise ValueError("mul_mat_q8: act must be 'q8_0' or 'q8_1'")
    x = _dev_f32(x, "x")
    if x.dim() != 2 or x.shape[1] != w.K:
        raise ValueError(f"mul_mat_q8: activations {tuple(x.shape)} do not match weight K={w.K}")
    N, K = x.shape
    M = w.M
    shape = (N, M) if c_trans else (M, N)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=x.device)
    elif (tuple(out.shape) != shape or out.dtype != torch.float32 or not out.is_contiguous() or out.device != x.device):
        raise ValueError(f"mul_mat_q8: out must be a contiguous f32 tensor of shape {shape} on {x.device}")
    lib = _lib()
    if not dump and not relu and act == "q8_0" and path == "auto":
        cabi.check("mul_mat_q8_hip", lib.mul_mat_q8_hip(_ptr(w.data), _ptr(x), _ptr(out), M, N, K, w.wtype,
                                                         c_trans, None, _stream()))
        return out
    xq = sums = None
    if dump:
        xq = torch.empty((N, K // QK, BLOCK_BYTES), dtype=torch.uint8, device=x.device)
        sums = torch.empty((N, M, K // QK), dtype=torch.int32, device=x.device)
    cabi.check("mul_mat_q8_ex_hip", lib.mul_mat_q8_ex_hip(_ptr(w.data), _ptr(x), _ptr(out), M, N, K, w.wtype,
                                                           c_trans, (1 if relu else 0) | (2 if act == "q8_1" else 0) | _Q8_PATH_FLAGS[path],
                                                           _ptr(xq), _ptr(sums), _stream()))
    return (out, xq, sums) if dump else out


# ----------------------------------------------------------------------------- around an attention block
ELEM_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _operand(t, name: str, dtypes=_FLOATS) -> torch.Tensor:
    """A tensor on the current device (whose stream the call goes to), of one of these types."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes:
        raise TypeError(f"{name} must be a device tensor of {' / '.join(str(d)[6:] for d in dtypes)}")
    if t.device.index != _current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{_current_device()}")
    return t


def _workspace(nbytes: int, device) -> torch.Tensor:
    # torch's allocator: kept for its next taker on the same stream, and a captured graph's own where the stream is under capture
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _rows(t: torch.Tensor):
    """(tensor, elements from row to row) of a matrix whose rows are dense and do not overlap"""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, max(t.stride(0), t.shape[1])


def quantize_rows_i8(x: torch.Tensor):
    """x [..., K] (float32, float16, bfloat16) -> (q int8 of its shape, scale float32 [...]): a scale per row, max |x| times
    1/127 in binary32, and x / scale rounded to the nearest whole number, halves to even.  A row of zeros has scale 0; one with an infinity or a NaN
    has scale NaN and zeros."""
    x = _operand(x, "x")
    K = x.shape[-1] if x.dim() else 0
    if not 1 <= K <= 131071:
        raise ValueError(f"quantize_rows_i8: rows of 1 to 131071 elements, got {tuple(x.shape)}")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    lib = _lib()
    if x.numel():
        rows, stride = _rows(x.reshape(-1, K))
        cabi.check("quantize_rows_i8_hip", lib.quantize_rows_i8_hip(_ptr(rows), ELEM_TYPES[x.dtype], stride, _ptr(q), K, _ptr(scale), rows.shape[0], K, _stream()))
    return q, scale


class I8Weight:
    """A weight [M, K] (rows = out features) in 8-bit integers, one scale a row (float32 [M]).

    ``pack()`` returns the copy whose rows are padded for the product, made once per weight (a weight with K a multiple of 128 is
    its own); ``mul_mat_i8`` packs any other per call."""

    def __init__(self, data: torch.Tensor, scale: torch.Tensor):
        data, scale = _operand(data, "data", (torch.int8,)), _operand(scale, "scale", (torch.float32,))
        if data.dim() != 2 or not 1 <= data.shape[1] <= 131071 or not 1 <= data.shape[0] <= 1 << 22 or tuple(scale.shape) != (data.shape[0],):
            raise ValueError(f"I8Weight: data must be [M, K] with M of 1 to 2^22, K of 1 to 131071 and scale [M], got {tuple(data.shape)} and {tuple(scale.shape)}")
        self.data, self.scale = data, scale.contiguous()
        self.M, self.K = data.shape
        self._packed = data if data.is_contiguous() and self.K % 128 == 0 and data.data_ptr() % 16 == 0 else None

    @classmethod
    def from_f32(cls, w: torch.Tensor) -> "I8Weight":
        """Quantizes a weight of any of the float types, a scale per row."""
        if not isinstance(w, torch.Tensor) or w.dim() != 2:
            raise ValueError("I8Weight.from_f32: a weight is a matrix")
        return cls(*quantize_rows_i8(w))

    def pack(self) -> "I8Weight":
        if self._packed is not None:
            return self
        lib = _lib()
        data, stride = _rows(self.data)
        out = torch.empty((self.M, lib.i8_weight_row_bytes_hip(self.K)), dtype=torch.int8, device=data.device)
        cabi.check("i8_weight_pack_hip", lib.i8_weight_pack_hip(_ptr(data), stride, self.M, self.K, _ptr(out), _stream()))
        packed = I8Weight(self.data, self.scale)
        packed._packed = out
        return packed


def mul_mat_i8(w: I8Weight, x, bias: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Linear in 8-bit integers: x [N, K] times w [M, K] -> [N, M] (+ bias float32 [M]), one scale a token and one a channel.  x is
    float32, float16 or bfloat16 and quantized on the way, or what quantize_rows_i8 returned (q, scale) for it, so that several layers
    share one quantization.  The sums are exact.  dtype: of the result, x's by default (float32 for quantized x)."""
    if not isinstance(w, I8Weight):
        raise TypeError("mul_mat_i8: w must be an I8Weight")
    if w._packed is not None and (dtype is None or dtype in _FLOATS):
        q, s = x if type(x) is tuple and len(x) == 2 else (x, None)
        y = _host_mul_mat_i8(w._packed, w.scale, w.K, q, s, bias, -1 if dtype is None else ELEM_TYPES[dtype])
        if y is not None:
            return y
    scale = None
    if isinstance(x, (tuple, list)):
        if len(x) != 2:
            raise ValueError("mul_mat_i8: quantized activations are (q, scale)")
        x, scale = _operand(x[0], "q", (torch.int8,)), _operand(x[1], "scale", (torch.float32,))
        if x.dim() != 2 or tuple(scale.shape) != (x.shape[0],):
            raise ValueError(f"mul_mat_i8: q must be [N, K] and scale [N], got {tuple(x.shape)} and {tuple(scale.shape)}")
        scale = scale.contiguous()
    else:
        x = _operand(x, "x")
    if x.dim() != 2 or x.shape[1] != w.K:
        raise ValueError(f"mul_mat_i8: activations {tuple(x.shape)} do not match weight K={w.K}")
    dtype = dtype or (x.dtype if scale is None else torch.float32)
    if dtype not in _FLOATS:
        raise TypeError(f"mul_mat_i8: the result is float32, float16 or bfloat16, not {dtype}")
    if w.data.device != x.device:
        raise ValueError(f"mul_mat_i8: the weight is on {w.data.device}, the activations on {x.device}")
    if bias is not None:
        bias = _operand(bias, "bias", (torch.float32,)).contiguous()
        if tuple(bias.shape) != (w.M,):
            raise ValueError(f"mul_mat_i8: bias {tuple(bias.shape)}, expected ({w.M},)")
    N, K = x.shape
    if N >= (1 << 31) - 1023:
        raise ValueError(f"mul_mat_i8: at most 2^31 - 1024 tokens a call, got {N}")
    out = torch.empty((N, w.M), dtype=dtype, device=x.device)
    lib = _lib()
    if N == 0:
        return out
    packed = w.pack()._packed
    x, stride = _rows(x)
    nbytes = lib.mul_mat_i8_workspace_hip(w.M, N, K)
    ws = _workspace(nbytes, x.device) if nbytes else None
    cabi.check("mul_mat_i8_hip", lib.mul_mat_i8_hip(_ptr(packed), _ptr(w.scale), _ptr(x), ELEM_TYPES[x.dtype], stride, _ptr(scale), _ptr(bias), _ptr(out),
                                                    ELEM_TYPES[dtype], w.M, N, K, _ptr(ws), nbytes, _stream()))
    return out


def rope_frequencies(rot: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """The usual frequencies of a rotation over `rot` elements, base ** (-2 i / rot) radians a position: float64 [rot / 2]."""
    if rot < 2 or rot % 2:
        raise ValueError("rope_frequencies: rot must be an even number of elements, 2 or more")
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda" if device is None else device)
    return float(base) ** (-2.0 * i / rot)


def _heads(t, name: str, like=None) -> torch.Tensor:
    t = _operand(t, name, _FLOATS if like is None else (like.dtype,))
    if t.dim() != 4:
        raise ValueError(f"{name} must have four dimensions, got {tuple(t.shape)}")
    return t if t.shape[3] <= 1 or t.stride(3) == 1 else t.contiguous()


def _steps(t: torch.Tensor, dims):
    """Elements from batch to batch, token to token, head to head (a dimension of one element is never stepped over)"""
    return (C.c_int64 * 3)(*(t.stride(i) if t.shape[i] > 1 else 0 for i in dims))


def _qk_norm_desc(who, q, k, wq, wk, freqs, positions, eps, interleaved):
    q = _heads(q, "q")
    k = _heads(k, "k", q)
    B, L, hq, d = q.shape
    if k.shape[0] != B or k.shape[1] != L or k.shape[3] != d:
        raise ValueError(f"{who}: q (B, L, hq, d) {tuple(q.shape)} and k (B, L, hk, d) {tuple(k.shape)} differ in B, L or d")
    if not 1 <= d <= 512:
        raise ValueError(f"{who}: heads of 1 to 512 elements, got {d}")
    if not (1 <= hq <= 65535 and 1 <= k.shape[2] <= 65535):
        raise ValueError(f"{who}: q and k need a head each, and have 65535 at most")
    if not eps >= 0.0:
        raise ValueError(f"{who}: eps must not be negative")
    weights = []
    for w, name in ((wq, "wq"), (wk, "wk")):
        if w is not None:
            w = _operand(w, name, (torch.float32,)).contiguous()
            if tuple(w.shape) != (d,):
                raise ValueError(f"{who}: {name} {tuple(w.shape)}, expected ({d},)")
        weights.append(w)
    a = cabi.QkNormDesc(B=B, L=L, hq=hq, hk=k.shape[2], d=d, type=ELEM_TYPES[q.dtype], interleaved=int(bool(interleaved)), eps=eps)
    if freqs is not None:
        freqs = _operand(freqs, "freqs", (torch.float64,)).contiguous()
        if freqs.dim() != 1 or 2 * freqs.shape[0] > d:
            raise ValueError(f"{who}: freqs must be a vector of at most d / 2 = {d // 2} frequencies, got {tuple(freqs.shape)}")
        a.rot = 2 * freqs.shape[0]
    if positions is not None:
        positions = _operand(positions, "positions", (torch.int32, torch.int64))
        if tuple(positions.shape) not in ((L,), (B, L)):
            raise ValueError(f"{who}: positions must be (L,) or (B, L), got {tuple(positions.shape)}")
        positions = positions.contiguous()
        a.position_bytes = positions.element_size()
        a.position_stride = L if positions.dim() == 2 else 0
    a.q_strides, a.k_strides = _steps(q, (0, 1, 2)), _steps(k, (0, 1, 2))
    return a, q, k, weights[0], weights[1], freqs, positions


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor | None = None, wk: torch.Tensor | None = None, freqs: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False):
    """Norms of queries and keys for each head, times their weights, with the position rotation, in one pass into attention's layout:
    q (B, L, hq, d), k (B, L, hk, d) -- slices of a fused projection's output as they are -- -> (B, hq, L, d), (B, hk, L, d).

    float32, float16 or bfloat16; wq, wk float32 (d,) or None (ones).  freqs: float64 radians a position, one per pair (rope_frequencies; scaled
    ones as a long context wants them); the first 2 * len(freqs) elements of a head are turned, as pairs (i, i + len(freqs)), or of neighbours
    where `interleaved`; None turns nothing.  positions: int32 / int64 (B, L) or (L,); None: 0, 1, ..."""
    both = _host_qk_norm_rope(q, k, wq, wk, freqs, positions, eps, interleaved)
    if both is not None:
        return both
    a, q, k, wq, wk, freqs, positions = _qk_norm_desc("qk_norm_rope", q, k, wq, wk, freqs, positions, eps, interleaved)
    yq, yk = (torch.empty((a.B, t.shape[2], a.L, a.d), dtype=q.dtype, device=q.device) for t in (q, k))
    a.q_out_strides, a.k_out_strides = _steps(yq, (0, 2, 1)), _steps(yk, (0, 2, 1))
    lib = _lib()
    if a.B * a.L:
        cabi.check("qk_norm_rope_hip", lib.qk_norm_rope_hip(C.byref(a), _ptr(q), _ptr(k), _ptr(wq), _ptr(wk), _ptr(freqs), _ptr(positions), _ptr(yq), _ptr(yk), _stream()))
    return yq, yk


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor | None = None, wk: torch.Tensor | None = None,
                          freqs: torch.Tensor | None = None, positions: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                          out: torch.Tensor | None = None):
    """Gradients of qk_norm_rope for dq (B, hq, L, d), dk (B, hk, L, d) and its inputs: (dq (B, L, hq, d), dk (B, L, hk, d), dwq, dwk), the last two
    None without weights.  out: the fused projection's gradient, contiguous (B, L, C) with C >= (hq + hk) d: q's heads are then written
    to its first columns, k's behind them, the rest (the values') stays as it is, and the first two results are views of it."""
    if out is None:
        grads = _host_qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, positions, eps, interleaved)
        if grads is not None:
            return grads
    a, q, k, wq, wk, freqs, positions = _qk_norm_desc("qk_norm_rope_backward", q, k, wq, wk, freqs, positions, eps, interleaved)
    dq, dk = _heads(dq, "dq", q), _heads(dk, "dk", q)
    for t, h, name in ((dq, a.hq, "dq"), (dk, a.hk, "dk")):
        if tuple(t.shape) != (a.B, h, a.L, a.d):
            raise ValueError(f"qk_norm_rope_backward: {name} {tuple(t.shape)}, expected {(a.B, h, a.L, a.d)}")
    if out is None:
        gq, gk = (torch.empty((a.B, a.L, h, a.d), dtype=q.dtype, device=q.device) for h in (a.hq, a.hk))
    else:
        out = _operand(out, "out", (q.dtype,))
        if out.dim() != 3 or out.shape[0] != a.B or out.shape[1] != a.L or out.shape[2] < (a.hq + a.hk) * a.d or not out.is_contiguous():
            raise ValueError(f"qk_norm_rope_backward: out must be contiguous (B, L, C) with C >= {(a.hq + a.hk) * a.d}, got {tuple(out.shape)}")
        if out.untyped_storage().data_ptr() in [t.untyped_storage().data_ptr() for t in (q, k, dq, dk)] and out.numel():
            raise ValueError("qk_norm_rope_backward: out must not share memory with what is read")
        gq = out[:, :, :a.hq * a.d].unflatten(2, (a.hq, a.d))
        gk = out[:, :, a.hq * a.d:(a.hq + a.hk) * a.d].unflatten(2, (a.hk, a.d))
    a.q_out_strides, a.k_out_strides = _steps(gq, (0, 1, 2)), _steps(gk, (0, 1, 2))
    a.dq_strides, a.dk_strides = _steps(dq, (0, 2, 1)), _steps(dk, (0, 2, 1))
    lib = _lib()
    if not a.B * a.L:
        return gq, gk, None if wq is None else torch.zeros_like(wq), None if wk is None else torch.zeros_like(wk)
    dwq, dwk = (None if w is None else torch.empty_like(w) for w in (wq, wk))
    nbytes = lib.qk_norm_rope_back_workspace_hip(C.byref(a)) if wq is not None or wk is not None else 0
    ws = _workspace(nbytes, q.device) if nbytes else None
    cabi.check("qk_norm_rope_back_hip",
               lib.qk_norm_rope_back_hip(C.byref(a), _ptr(dq), _ptr(dk), _ptr(q), _ptr(k), _ptr(wq), _ptr(wk), _ptr(freqs), _ptr(positions), _ptr(gq), _ptr(gk),
                                         _ptr(dwq), _ptr(dwk), _ptr(ws), nbytes, _stream()))
    return gq, gk, dwq, dwk


NEWTON_SCHULZ_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients=NEWTON_SCHULZ_COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """An update orthogonalised by Newton-Schulz products: X = g / (|g| + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T,
    for every matrix of g [..., rows, cols] (float32, float16, bfloat16; binary32-grade arithmetic for all) -> the same shape and type.
    Singular values above a hundredth or so of the largest come out near 1.  coefficients: (a, b, c); such
    that singular values of up to 1 stay below 2^20."""
    if type(coefficients) is tuple and len(coefficients) == 3:
        out = _host_newton_schulz(g, steps, *coefficients, eps)
        if out is not None:
            return out
    g = _operand(g, "g")
    if g.dim() < 2:
        raise ValueError(f"newton_schulz: g must be a matrix or a stack of them, got {tuple(g.shape)}")
    a, b, c = (float(x) for x in coefficients)
    if not 1 <= int(steps) <= 32 or not all(map(math.isfinite, (a, b, c, eps))) or eps < 0:
        raise ValueError("newton_schulz: 1 to 32 steps, finite coefficients, eps finite and not negative")
    g = g.contiguous()
    out = torch.empty_like(g)
    lib = _lib()
    if g.numel() == 0:
        return out
    rows, cols = g.shape[-2:]
    batch = g.numel() // (rows * cols)
    nbytes = lib.newton_schulz_workspace_hip(batch, rows, cols)
    if nbytes == 0:
        raise ValueError(f"newton_schulz: at most 65535 matrices with sides up to 2^20, got {tuple(g.shape)}")
    ws = _workspace(nbytes, g.device)
    cabi.check("newton_schulz_hip", lib.newton_schulz_hip(_ptr(g), _ptr(out), ELEM_TYPES[g.dtype], batch, rows, cols, int(steps), a, b, c, float(eps), _ptr(ws), nbytes,
                                                          _stream()))
    return out
