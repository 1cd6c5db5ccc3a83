"""torch-tensor wrappers over the C-ABI (include/spn4cir_hip.h).

PyTorch is used only for device memory and streams: every function takes CUDA(=HIP) tensors,
passes raw device pointers plus torch's current stream to libspn4cir_hip.so and returns
tensors.  There is no CPU fallback: CPU tensors are rejected.
"""
import ctypes as C
import functools
import operator
import os
from array import array

import numpy as np
import torch

from . import _lib
from ._lib import check, lib

ACT_NONE, ACT_QUICKGELU, ACT_GELU_ERF = 0, 1, 2
BANK_DIMS = (128, 256, 512, 640, 768, 1024)

_ws_cache = {}


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError("spn4cir_amd ops need device tensors (no CPU fallback)")
    return C.c_void_p(t.data_ptr())


_POISON = os.environ.get("SPN_DEBUG_POISON") == "1"


def scratch_bytes(nbytes, device):
    """Uninitialised device scratch (uint8).  SPN_DEBUG_POISON=1 fills every such allocation with 0xFF bytes - NaN as fp32
    and as bf16 - so that a kernel that reads scratch it never wrote shows up as NaN in its output instead of as
    allocator-dependent noise (tests/test_poison_gpu.py runs the training steps that way)."""
    buf = torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)
    if _POISON:
        buf.fill_(255)
    return buf


def workspace(nbytes, device, slot="default"):
    """Grow-only scratch buffer per (device, slot); ops on one stream use it sequentially."""
    key = (str(device), slot)
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = scratch_bytes(max(int(nbytes), 256), device)
        _ws_cache[key] = buf
    return buf


def _req(t, dtype, name):
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous {dtype}, got {t.dtype} contiguous={t.is_contiguous()}")


def check_index_range(idx, n, name):
    """IndexError for a row index outside [0, n), as `refer_bank[refer_indexs]` raises in the reference
    (models_negplus.py:133).  Free for host tensors - the DataLoader hands the reference's loop CPU LongTensors
    (train_negplus.py:107-111); a device tensor is only inspected (one sync) under SPN_CHECK_INDICES=1, otherwise the
    kernels' own guards apply (NaN query row / infinite loss, never an out-of-bounds read)."""
    if idx is None or idx.numel() == 0:
        return
    if idx.is_cuda and os.environ.get("SPN_CHECK_INDICES") != "1":
        return
    lo, hi = int(idx.min()), int(idx.max())
    if lo < 0 or hi >= n:
        raise IndexError(f"{name}: index {lo if lo < 0 else hi} is out of bounds for a bank with {n} rows")


# ------------------------------------------------------------------------------- GEMMs
def gemm_nt(a, b, bias=None, act=ACT_NONE, out_dtype=torch.bfloat16, want_pre=False):
    """a [M,K] bf16, b [N,K] bf16 -> act(a @ b.T + bias) ; optionally also the pre-activation."""
    _req(a, torch.bfloat16, "a"); _req(b, torch.bfloat16, "b")
    M, K = a.shape
    N = b.shape[0]
    out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    pre = torch.empty(M, N, dtype=torch.bfloat16, device=a.device) if want_pre else None
    ob, of = (out, None) if out_dtype == torch.bfloat16 else (None, out)
    check(lib().spn_gemm_nt(_p(a), _p(b), M, N, K, K, K, _p(bias), act, _p(ob), _p(of), _p(pre), N, _stream()), "gemm_nt")
    return (out, pre) if want_pre else out


def gemm_nt_resid(a, b, bias, resid):
    _req(a, torch.bfloat16, "a"); _req(b, torch.bfloat16, "b"); _req(resid, torch.float32, "resid")
    M, K = a.shape
    N = b.shape[0]
    out = torch.empty(M, N, dtype=torch.float32, device=a.device)
    check(lib().spn_gemm_nt_resid(_p(a), _p(b), M, N, K, K, K, _p(bias), _p(resid), N, _p(out), None, N, _stream()),
          "gemm_nt_resid")
    return out


def gemm_nt_dact(a, b, pre, act):
    _req(a, torch.bfloat16, "a"); _req(b, torch.bfloat16, "b"); _req(pre, torch.bfloat16, "pre")
    M, K = a.shape
    N = b.shape[0]
    out = torch.empty(M, N, dtype=torch.bfloat16, device=a.device)
    check(lib().spn_gemm_nt_dact(_p(a), _p(b), M, N, K, K, K, _p(pre), act, _p(out), N, _stream()), "gemm_nt_dact")
    return out


def gemm_tn(a, b, alpha=1.0, out=None, accumulate=False, want_colsum=False):
    """a [Kr,N1] bf16, b [Kr,N2] bf16 -> a.T @ b  (fp32 [N1,N2]) [, column sums of a]."""
    _req(a, torch.bfloat16, "a"); _req(b, torch.bfloat16, "b")
    Kr, N1 = a.shape
    N2 = b.shape[1]
    if out is None:
        out = torch.empty(N1, N2, dtype=torch.float32, device=a.device)
    nb = lib().spn_gemm_tn_workspace_bytes(Kr, N1, N2)
    ws = workspace(nb, a.device)
    cs = torch.empty(N1, dtype=torch.float32, device=a.device) if want_colsum else None
    check(lib().spn_gemm_tn(_p(a), _p(b), Kr, N1, N2, N1, N2, _p(out), N2, float(alpha), int(accumulate), _p(cs),
                            _p(ws), ws.numel(), _stream()), "gemm_tn")
    return (out, cs) if want_colsum else out


def gemm_tn_pair(a1, b1, a2, b2):
    """(a1.T @ b1, colsum(a1), a2.T @ b2, colsum(a2)) for bf16 [Kr, N] operands sharing Kr, in one launch."""
    for t in (a1, b1, a2, b2):
        _req(t, torch.bfloat16, "operand")
    Kr = a1.shape[0]
    N1a, N2a, N1b, N2b = a1.shape[1], b1.shape[1], a2.shape[1], b2.shape[1]
    dev = a1.device
    c1 = torch.empty(N1a, N2a, dtype=torch.float32, device=dev); s1 = torch.empty(N1a, dtype=torch.float32, device=dev)
    c2 = torch.empty(N1b, N2b, dtype=torch.float32, device=dev); s2 = torch.empty(N1b, dtype=torch.float32, device=dev)
    ws = workspace(lib().spn_gemm_tn_pair_workspace_bytes(Kr, N1a, N2a, N1b, N2b), dev)
    check(lib().spn_gemm_tn_pair(_p(a1), _p(b1), N1a, N2a, _p(c1), _p(s1), _p(a2), _p(b2), N1b, N2b, _p(c2), _p(s2), Kr,
                                 _p(ws), ws.numel(), _stream()), "gemm_tn_pair")
    return c1, s1, c2, s2


class _TnProblem(C.Structure):     # == spn_tn_problem
    _fields_ = [("A", C.c_void_p), ("B", C.c_void_p), ("C", C.c_void_p), ("colsum", C.c_void_p),
                ("N1", C.c_int), ("N2", C.c_int), ("lda", C.c_int), ("ldb", C.c_int), ("ldc", C.c_int)]


def gemm_tn_grouped(pairs, want_colsum=True):
    """[(a [Kr,N1] bf16, b [Kr,N2] bf16), ...] sharing Kr -> [(a.T @ b fp32 [N1,N2], colsum(a) [N1] or None), ...]
    in ONE launch without split-K (spn_gemm_tn_grouped)."""
    Kr = pairs[0][0].shape[0]
    dev = pairs[0][0].device
    arr = (_TnProblem * len(pairs))()
    outs = []
    for i, (a, b) in enumerate(pairs):
        _req(a, torch.bfloat16, "a"); _req(b, torch.bfloat16, "b")
        if a.shape[0] != Kr or b.shape[0] != Kr:
            raise ValueError("grouped TN problems must share the reduction length")
        N1, N2 = a.shape[1], b.shape[1]
        c = torch.empty(N1, N2, dtype=torch.float32, device=dev)
        cs = torch.empty(N1, dtype=torch.float32, device=dev) if want_colsum else None
        arr[i] = _TnProblem(a.data_ptr(), b.data_ptr(), c.data_ptr(), cs.data_ptr() if want_colsum else None, N1, N2, N1, N2, N2)
        outs.append((c, cs))
    ws = workspace(lib().spn_gemm_tn_grouped_workspace_bytes(Kr), dev)
    check(lib().spn_gemm_tn_grouped(C.byref(arr), len(pairs), Kr, _p(ws), ws.numel(), _stream()), "gemm_tn_grouped")
    return outs


# ------------------------------------------------------------------------ 8-bit blocks
_ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # == SPN_F32 / SPN_BF16 / SPN_F16
_E4M3 = 3


# Host cost of a call decides at the sizes of a few tokens: these entry points take the raw stream and device index (ints) and hand
# pointers to ctypes as ints.
_raw_stream = torch._C._cuda_getCurrentRawStream
_cur_device = torch._C._cuda_getDevice


def _no_cpu():
    raise RuntimeError("spn4cir_amd ops need device tensors (no CPU fallback)")


def _on_device(fn):
    """Runs `fn` with the device of its first argument current (torch's current stream of THAT device is the one used).  The entry points of
    single launches do the same in line."""
    @functools.wraps(fn)
    def call(x, *args, **kwargs):
        di = x.get_device()
        if di >= 0 and di != _cur_device():              # (CPU tensors: the checks inside refuse them)
            with torch.cuda.device(di):
                return fn(x, *args, **kwargs)
        return fn(x, *args, **kwargs)
    return call


def _rows2d(t, name, di=None):
    """A 2-D device tensor whose rows are contiguous, at any pitch >= the width -> (element type, row pitch); di: its device index."""
    typ = _ELEM.get(t.dtype)
    if typ is None:
        raise ValueError(f"{name}: expected fp32, bf16 or fp16, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name}: expected a matrix, got {tuple(t.shape)}")
    on = t.get_device()
    if on < 0:
        _no_cpu()
    if di is not None and on != di:
        raise ValueError(f"{name}: on cuda:{on}, expected cuda:{di}")
    R, W = t.shape
    s0, s1 = t.stride()
    if (W > 1 and s1 != 1) or (R > 1 and s0 < W):
        raise ValueError(f"{name}: rows must be contiguous (strides {t.stride()})")
    return typ, s0 if R > 1 else max(W, 1)


def _vec(t, n, name, di):
    if t.dtype != torch.float32 or t.numel() != n or t.get_device() != di or not t.is_contiguous():
        if t.get_device() < 0:
            _no_cpu()
        raise ValueError(f"{name}: expected contiguous fp32 [{n}] on cuda:{di}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def fp8_pitch(K):
    """Scale bytes per row of a block-format matrix with K columns (SPN_FP8_PITCH)."""
    return ((K + 127) // 128 + 3) // 4 * 4


class Fp8Blocks:
    """A matrix [rows, K] in the 8-bit block format: `data` uint8 [rows, K rounded up to 128] (OCP e4m3 codes, zeros behind K), `scale`
    uint8 [rows, fp8_pitch(K)]: value = code * 2^(byte - 127), one byte for 128 consecutive values of a row.  Written by quantize_fp8 and
    rmsnorm_fwd(out_dtype="fp8"), read by gemm_nt_fp8 / linear_fp8_*.  The bytes may be written in place; the tensors stay what they are."""

    __slots__ = ("data", "scale", "K", "rows")

    def __setattr__(self, name, value):              # the checks of __init__ hold for good: kernels rely on them
        raise AttributeError(f"Fp8Blocks.{name} cannot be replaced: build another one")

    def __init__(self, data, scale, K):
        rows, Kp = data.shape
        if K <= 0 or Kp != (K + 127) // 128 * 128 or scale.shape != (rows, fp8_pitch(K)):
            raise ValueError(f"Fp8Blocks: codes {tuple(data.shape)} and scale {tuple(scale.shape)} do not hold {K} columns")
        if data.dtype != torch.uint8 or scale.dtype != torch.uint8 or not data.is_contiguous() or not scale.is_contiguous():
            raise ValueError("Fp8Blocks: codes and scale must be contiguous uint8")
        if data.get_device() != scale.get_device():
            raise ValueError("Fp8Blocks: codes and scale on different devices")
        if data.data_ptr() % 16 or scale.data_ptr() % 4:
            raise ValueError("Fp8Blocks: codes must be 16-byte, scale bytes 4-byte aligned")
        _SET_DATA(self, data), _SET_SCALE(self, scale), _SET_K(self, K), _SET_ROWS(self, rows)

    def __reduce__(self):                            # copies and pickles are built from their tensors, checks included
        return Fp8Blocks, (self.data, self.scale, self.K)

    @property
    def shape(self):
        return torch.Size((self.rows, self.K))

    @property
    def device(self):
        return self.data.device

    def get_device(self):
        return self.data.get_device()

    @staticmethod
    def empty(rows, K, device):
        q = Fp8Blocks.__new__(Fp8Blocks)                     # fresh allocations satisfy every condition of __init__
        _SET_DATA(q, torch.empty(rows, (K + 127) // 128 * 128, dtype=torch.uint8, device=device))
        _SET_SCALE(q, torch.empty(rows, fp8_pitch(K), dtype=torch.uint8, device=device))
        _SET_K(q, K), _SET_ROWS(q, rows)
        return q

    def dequantize(self, dtype=torch.bfloat16):
        """[rows, K] as numbers.  fp32 holds the stored values exactly up to its largest number (magnitudes from 248 * 2^120 = 3.3e38 on are
        stored as 2^128 and decode to infinity), bf16 too, but for blocks whose largest magnitude is below 2^-116, where what lies under
        2^-133 is rounded."""
        return _dequantize_fp8(self, dtype)


_SET_DATA, _SET_SCALE, _SET_K, _SET_ROWS = (Fp8Blocks.__dict__[name].__set__ for name in Fp8Blocks.__slots__)


def _fp8_ptrs(q):
    return (None, None) if q is None else (q.data.data_ptr(), q.scale.data_ptr())


def _dequantize_fp8(q, dtype):
    if dtype not in _ELEM:
        raise ValueError(f"dequantize: fp32, bf16 or fp16, not {dtype}")
    di = q.data.get_device()
    if di < 0:
        _no_cpu()
    if di != _cur_device():
        with torch.cuda.device(di):
            return _dequantize_fp8(q, dtype)
    out = torch.empty(q.rows, q.K, dtype=dtype, device=q.data.device)
    if q.rows:
        check(lib().spn_dequantize_fp8(q.data.data_ptr(), q.scale.data_ptr(), q.rows, q.K, out.data_ptr(), _ELEM[dtype], _raw_stream(di)), "dequantize_fp8")
    return out


def quantize_fp8(x, block_rows=1, want="rows", colsum=False):
    """x [R, C] fp32 / bf16 / fp16 (rows at any pitch) or Fp8Blocks -> 8-bit blocks (spn_quantize_fp8).

    want: "rows" = Fp8Blocks [R, C], blocks along each row; "cols" = Fp8Blocks of the TRANSPOSED matrix [C, R], blocks along R (what a
    product that reduces over R reads); "both" = (rows, cols) from one read of x.  block_rows=128: one scale for 128 x 128 values - the
    two forms then hold the same codes (weights).  colsum=True appends the fp32 column sums [C] of x (a bias gradient).  A matrix without rows
    has the rows form only."""
    if want not in ("rows", "cols", "both") or block_rows not in (1, 128):
        raise ValueError(f"quantize_fp8: want {want!r}, block_rows {block_rows!r}")
    di = x.get_device()
    if di >= 0 and di != _cur_device():
        with torch.cuda.device(di):
            return quantize_fp8(x, block_rows, want, colsum)
    if isinstance(x, Fp8Blocks):
        if di < 0:
            _no_cpu()
        R, Cn, typ, ld, xs, pitch, ptr = x.rows, x.K, _E4M3, x.data.shape[1], x.scale.data_ptr(), x.scale.shape[1], x.data.data_ptr()
    else:
        typ, ld = _rows2d(x, "x")
        (R, Cn), xs, pitch, ptr = x.shape, None, 0, x.data_ptr()
    if Cn == 0 or (R == 0 and want != "rows"):
        raise ValueError("quantize_fp8: no columns" if Cn == 0 else "quantize_fp8: the transpose of no rows has no blocks")
    dev = x.device
    if R == 0:
        q = Fp8Blocks.empty(0, Cn, dev)
        return (q, torch.zeros(Cn, dtype=torch.float32, device=dev)) if colsum else q
    q = Fp8Blocks.empty(R, Cn, dev) if want != "cols" else None
    qt = Fp8Blocks.empty(Cn, R, dev) if want != "rows" else None
    cs = torch.empty(Cn, dtype=torch.float32, device=dev) if colsum else None
    ws = scratch_bytes(lib().spn_quantize_fp8_workspace_bytes(R, Cn), dev) if colsum else None
    check(lib().spn_quantize_fp8(ptr, typ, ld, xs, pitch, R, Cn, 1 if block_rows == 128 else 0, *_fp8_ptrs(q),
                                 *_fp8_ptrs(qt), cs.data_ptr() if colsum else None,
                                 ws.data_ptr() if colsum else None, ws.numel() if colsum else 0, _raw_stream(di)), "quantize_fp8")
    out = [t for t in (q, qt, cs) if t is not None]
    return out[0] if len(out) == 1 else tuple(out)


@functools.lru_cache(maxsize=1024)          # a pure function of the shape (one part: gfx950)
def _gemm_fp8_ws(M, N, K):
    return lib().spn_gemm_nt_fp8_workspace_bytes(M, N, K)


def _product_out(out, M, N, dtype, accumulate, act, device):
    """The output [M, N] of a product: the caller's or a new one -> (tensor, element type, row pitch)."""
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs out")
        typ = _ELEM.get(dtype)
        if typ is None:
            raise ValueError(f"out_dtype: fp32, bf16 or fp16, not {dtype}")
        return torch.empty(M, N, dtype=dtype, device=device), typ, N
    if out.shape != (M, N):
        raise ValueError(f"out: expected {(M, N)}, got {tuple(out.shape)}")
    typ, ldc = _rows2d(out, "out", device.index)
    if accumulate and (typ != 0 or act != ACT_NONE):
        raise ValueError("accumulate=True needs an fp32 out and no activation")
    return out, typ, ldc


def gemm_nt_fp8(a, b, bias=None, act=ACT_NONE, out_dtype=torch.bfloat16, out=None, accumulate=False):
    """act(a @ b.T + bias) for Fp8Blocks a [M, K], b [N, K] (spn_gemm_nt_fp8); out: write there (rows contiguous, any pitch), with
    accumulate=True add into it (fp32, no activation).  Sums are fp32, but the matrix unit aligns each eight consecutive products to the
    largest of them and cuts 13 bits below it: an fp32 output is off by 1.5e-5 to 5e-5 of its rms (14 to 16 good bits, not 24; a code itself
    carries 4), a 16-bit one by one rounding more in 3 % of its elements.  For sums in full fp32: gemm_nt of the decoded operands (bf16 holds them
    exactly; K % 64 == 0, N % 4 == 0), at the bf16 rate."""
    if not isinstance(a, Fp8Blocks) or not isinstance(b, Fp8Blocks):
        raise TypeError("a, b: expected Fp8Blocks (ops.quantize_fp8)")
    di, M, N, K = a.data.get_device(), a.rows, b.rows, a.K
    if di >= 0 and di != _cur_device():
        with torch.cuda.device(di):
            return gemm_nt_fp8(a, b, bias, act, out_dtype, out, accumulate)
    if K != b.K or di != b.data.get_device():
        raise ValueError(f"a {tuple(a.shape)} on {a.device} and b {tuple(b.shape)} on {b.device} do not match")
    if N == 0:
        raise ValueError("b: no rows")
    bp = None if bias is None else _vec(bias, N, "bias", di)
    if act not in (ACT_NONE, ACT_QUICKGELU, ACT_GELU_ERF):
        raise ValueError(f"act {act!r}")
    out, typ, ldc = _product_out(out, M, N, out_dtype, accumulate, act, a.data.device)
    if di < 0:
        _no_cpu()
    if M == 0:
        return out
    nb = _gemm_fp8_ws(M, N, K)
    ws = scratch_bytes(nb, a.device) if nb else None
    check(lib().spn_gemm_nt_fp8(a.data.data_ptr(), a.scale.data_ptr(), b.data.data_ptr(), b.scale.data_ptr(), M, N, K, bp, act, out.data_ptr(), typ, ldc, 1 if accumulate else 0,
                                ws.data_ptr() if nb else None, nb, _raw_stream(di)), "gemm_nt_fp8")
    return out


@_on_device
def linear_fp8_fwd(x, w8, bias=None, w8_t=None, out_dtype=torch.bfloat16):
    """x @ w.T + bias with 8-bit operands: x [M, K] fp32 / bf16 / fp16 or Fp8Blocks (from rmsnorm_fwd), w8 = Fp8Blocks [N, K]
    -> (y [M, N], saved).  Training passes w8_t as well - w8, w8_t = quantize_fp8(w, block_rows=128, want="both") - and hands `saved` to
    linear_fp8_bwd; without it saved is None."""
    if not isinstance(w8, Fp8Blocks) or (w8_t is not None and (not isinstance(w8_t, Fp8Blocks) or w8_t.shape != (w8.K, w8.shape[0]))):
        raise ValueError("w8 / w8_t: quantize_fp8(w, block_rows=128, want='both')")
    if x.shape[-1] != w8.K:
        raise ValueError(f"x {tuple(x.shape)} does not match w {tuple(w8.shape)}")
    if w8_t is None:
        x8 = x if isinstance(x, Fp8Blocks) else quantize_fp8(x)
        return gemm_nt_fp8(x8, w8, bias, out_dtype=out_dtype), None
    if x.shape[0] == 0:                                      # an empty batch: no blocks along its rows
        x8, x8_t = x if isinstance(x, Fp8Blocks) else quantize_fp8(x), None
    elif isinstance(x, Fp8Blocks):
        x8, x8_t = x, quantize_fp8(x, want="cols")
    else:
        x8, x8_t = quantize_fp8(x, want="both")
    y = gemm_nt_fp8(x8, w8, bias, out_dtype=out_dtype)
    return y, dict(x8_t=x8_t, w8_t=w8_t, bias=bias is not None, M=x.shape[0])


@_on_device
def _linear_fp8_bwd(dy, saved, dx_dtype, dw_dtype, dw, accumulate):
    M, N = dy.shape
    if M != saved["M"] or N != saved["w8_t"].K:
        raise ValueError(f"dy {tuple(dy.shape)}: expected {(saved['M'], saved['w8_t'].K)}")
    if M == 0:
        _rows2d(dy, "dy", saved["w8_t"].get_device())
        dw = _product_out(dw, N, saved["w8_t"].rows, dw_dtype, accumulate, ACT_NONE, dy.device)[0]
        if not accumulate:
            dw.zero_()
        return (gemm_nt_fp8(Fp8Blocks.empty(0, N, dy.device), saved["w8_t"], out_dtype=dx_dtype), dw,
                torch.zeros(N, dtype=torch.float32, device=dy.device) if saved["bias"] else None)
    if saved["bias"]:
        dy8, dy8_t, db = quantize_fp8(dy, want="both", colsum=True)
    else:
        (dy8, dy8_t), db = quantize_fp8(dy, want="both"), None
    dx = gemm_nt_fp8(dy8, saved["w8_t"], out_dtype=dx_dtype)
    dw = gemm_nt_fp8(dy8_t, saved["x8_t"], out_dtype=dw_dtype, out=dw, accumulate=accumulate)
    return dx, dw, db


def linear_fp8_bwd(saved, dy, dx_dtype=torch.bfloat16, dw_dtype=torch.float32, dw=None, accumulate=False):
    """Backward of linear_fp8_fwd: dy [M, N] fp32 / bf16 / fp16 -> (dx [M, K], dw [N, K], db fp32 [N] or None).  dy is quantised along N
    for dx and along M for dw; db sums it unquantised.  dw: write there; accumulate=True adds (fp32)."""
    if saved is None:
        raise ValueError("linear_fp8_bwd: the forward call had no w8_t")
    return _linear_fp8_bwd(dy, saved, dx_dtype, dw_dtype, dw, accumulate)


# ------------------------------------------------------------------------------ RMSNorm
def rmsnorm_fwd(x, gamma, residual=None, eps=1e-6, out_dtype=torch.bfloat16):
    """h = x + residual (in the residual's type: fp32, or x's), y = h / sqrt(mean(h^2) + eps) * gamma -> (y, h, rstd [rows]).

    x [rows, W] fp32 / bf16 / fp16 at any row pitch, W <= 16384, gamma fp32 [W]; without a residual h is x itself.  out_dtype: fp32 / bf16 /
    fp16, or "fp8": y as Fp8Blocks (one scale for 128 columns), ready for gemm_nt_fp8 / linear_fp8_fwd.  Squares are summed in fp32: a row whose
    sum passes 3.4e38 (values near 1e18) gives rstd 0, and one whose squares vanish (values below 1e-22) counts as zeros, which only eps = 0 shows."""
    xt, ldx = _rows2d(x, "x")
    rows, W = x.shape
    di, dev = x.get_device(), x.device
    if di != _cur_device():
        with torch.cuda.device(di):
            return rmsnorm_fwd(x, gamma, residual, eps, out_dtype)
    gp = _vec(gamma, W, "gamma", di)
    rt = ldr = 0
    h, rp, hp = x, None, None
    if residual is not None:
        rt, ldr = _rows2d(residual, "residual", di)
        if residual.shape != x.shape or (rt != 0 and rt != xt):
            raise ValueError(f"residual: expected {tuple(x.shape)} in fp32 or {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
        h = torch.empty(rows, W, dtype=residual.dtype, device=dev)
        rp, hp = residual.data_ptr(), h.data_ptr()
    rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    if out_dtype == "fp8":
        y = Fp8Blocks.empty(rows, W, dev)
        yp, yt, ys = y.data.data_ptr(), _E4M3, y.scale.data_ptr()
    else:
        yt, ys = _ELEM.get(out_dtype), None
        if yt is None:
            raise ValueError(f"out_dtype: fp32, bf16, fp16 or 'fp8', not {out_dtype!r}")
        y = torch.empty(rows, W, dtype=out_dtype, device=dev)
        yp = y.data_ptr()
    if rows:
        check(lib().spn_rmsnorm_fwd(x.data_ptr(), xt, ldx, rp, rt, ldr, gp, eps, hp, yp, yt, ys, rstd.data_ptr(), rows, W, _raw_stream(di)),
              "rmsnorm_fwd")
    return y, h, rstd


@functools.lru_cache(maxsize=1024)
def _rms_bwd_ws(rows, W):
    return lib().spn_rmsnorm_bwd_workspace_bytes(rows, W)


def rmsnorm_bwd(dy, h, gamma, rstd, dh=None, dx_dtype=None):
    """Backward of rmsnorm_fwd: dy [rows, W] = d/dy (for the "fp8" output: of the values before rounding), h and rstd as returned, dh =
    the gradient that reaches h directly (h's type) -> (dx in h's type, dgamma fp32 [W]); dx is the gradient of x and of the residual.
    dx_dtype: returns (dx, a copy of dx in that type, dgamma) - for a branch in bf16 beside an fp32 stream."""
    dyt, lddy = _rows2d(dy, "dy")
    rows, W = dy.shape
    di, dev = dy.get_device(), dy.device
    if di != _cur_device():
        with torch.cuda.device(di):
            return rmsnorm_bwd(dy, h, gamma, rstd, dh, dx_dtype)
    ht, ldh = _rows2d(h, "h", di)
    if h.shape != dy.shape:
        raise ValueError(f"h {tuple(h.shape)} does not match dy {tuple(dy.shape)}")
    gp, rp = _vec(gamma, W, "gamma", di), _vec(rstd, rows, "rstd", di)
    lddh, dhp = 0, None
    if dh is not None:
        dt, lddh = _rows2d(dh, "dh", di)
        if dt != ht or dh.shape != h.shape:
            raise ValueError(f"dh: expected {tuple(h.shape)} {h.dtype}, got {tuple(dh.shape)} {dh.dtype}")
        dhp = dh.data_ptr()
    if dx_dtype is not None and dx_dtype not in _ELEM:
        raise ValueError(f"dx_dtype: fp32, bf16 or fp16, not {dx_dtype!r}")
    dx = torch.empty(rows, W, dtype=h.dtype, device=dev)
    dx2 = torch.empty(rows, W, dtype=dx_dtype, device=dev) if dx_dtype is not None else None
    if rows == 0:
        dgamma = torch.zeros(W, dtype=torch.float32, device=dev)
    else:
        dgamma = torch.empty(W, dtype=torch.float32, device=dev)
        nb = _rms_bwd_ws(rows, W)
        ws = scratch_bytes(nb, dev) if nb else None
        check(lib().spn_rmsnorm_bwd(dy.data_ptr(), dyt, lddy, h.data_ptr(), ht, ldh, gp, rp, dhp, lddh, dx.data_ptr(),
                                    None if dx2 is None else dx2.data_ptr(), _ELEM.get(dx_dtype, 0), dgamma.data_ptr(), rows, W, ws.data_ptr() if nb else None, nb,
                                    _raw_stream(di)), "rmsnorm_bwd")
    return (dx, dgamma) if dx_dtype is None else (dx, dx2, dgamma)


# ------------------------------------------------------------------------- elementwise
def cast_bf16(x):
    _req(x, torch.float32, "x")
    y = torch.empty_like(x, dtype=torch.bfloat16)
    check(lib().spn_cast_f32_bf16(_p(x), _p(y), x.numel(), _stream()), "cast")
    return y


def cast_transpose_bf16(x):
    _req(x, torch.float32, "x")
    r, c = x.shape
    y = torch.empty(r, c, dtype=torch.bfloat16, device=x.device)
    yt = torch.empty(c, r, dtype=torch.bfloat16, device=x.device)
    check(lib().spn_cast_transpose_f32_bf16(_p(x), _p(y), _p(yt), r, c, _stream()), "cast_transpose")
    return y, yt


def colsum(x):
    _req(x, torch.bfloat16, "x")
    r, c = x.shape
    out = torch.empty(c, dtype=torch.float32, device=x.device)
    ws = workspace(lib().spn_colsum_workspace_bytes(r, c), x.device)
    check(lib().spn_colsum_bf16(_p(x), r, c, c, _p(out), 0, _p(ws), ws.numel(), _stream()), "colsum")
    return out


# --------------------------------------------------------------------------- LayerNorm
def layernorm_fwd(x, gamma, beta, eps=1e-5, out_dtype=torch.bfloat16):
    _req(x, torch.float32, "x")
    rows, W = x.shape
    y = torch.empty(rows, W, dtype=out_dtype, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    yb, yf = (y, None) if out_dtype == torch.bfloat16 else (None, y)
    check(lib().spn_layernorm_fwd(_p(x), _p(gamma), _p(beta), _p(yb), _p(yf), _p(mean), _p(rstd), rows, W, eps,
                                  _stream()), "layernorm_fwd")
    return y, mean, rstd


def layernorm_bwd(dy, x, gamma, mean, rstd, dx_accum=None):
    """Returns (dx fp32, dx bf16, dgamma, dbeta); dx_accum (fp32) is added into if given."""
    rows, W = x.shape
    dx = dx_accum if dx_accum is not None else torch.empty(rows, W, dtype=torch.float32, device=x.device)
    dxb = torch.empty(rows, W, dtype=torch.bfloat16, device=x.device)
    dg = torch.empty(W, dtype=torch.float32, device=x.device)
    db = torch.empty(W, dtype=torch.float32, device=x.device)
    ws = workspace(lib().spn_layernorm_bwd_workspace_bytes(rows, W), x.device)
    dyb, dyf = (dy, None) if dy.dtype == torch.bfloat16 else (None, dy)
    check(lib().spn_layernorm_bwd(_p(dyb), _p(dyf), _p(x), _p(gamma), _p(mean), _p(rstd), _p(dx),
                                  int(dx_accum is not None), _p(dxb), _p(dg), _p(db), 0, rows, W, _p(ws), ws.numel(),
                                  _stream()), "layernorm_bwd")
    return dx, dxb, dg, db


# --------------------------------------------------------------------------- attention
def attention_fwd(q, k, v, B, H, Lq, Lk, causal=False, key_bias=None, scale=0.125):
    """q [B*Lq, H*64], k/v [B*Lk, H*64] bf16 (may be column views of a packed qkv) -> (o, lse)."""
    o = torch.empty(B * Lq, H * 64, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty(B, H, Lq, dtype=torch.float32, device=q.device)
    check(lib().spn_attention_fwd(_p(q), _p(k), _p(v), q.stride(0), k.stride(0), v.stride(0), _p(o), H * 64, _p(lse),
                                  _p(key_bias), B, H, Lq, Lk, int(causal), scale, _stream()), "attention_fwd")
    return o, lse


def attention_bwd(q, k, v, o, lse, d_o, B, H, Lq, Lk, causal=False, key_bias=None, scale=0.125):
    dq = torch.empty(B * Lq, H * 64, dtype=torch.bfloat16, device=q.device)
    dk = torch.empty(B * Lk, H * 64, dtype=torch.bfloat16, device=q.device)
    dv = torch.empty(B * Lk, H * 64, dtype=torch.bfloat16, device=q.device)
    delta = torch.empty(B, H, Lq, dtype=torch.float32, device=q.device)
    check(lib().spn_attention_bwd(_p(q), _p(k), _p(v), q.stride(0), k.stride(0), v.stride(0), _p(o), o.stride(0),
                                  _p(lse), _p(key_bias), _p(d_o), d_o.stride(0), _p(dq), _p(dk), _p(dv), H * 64, H * 64,
                                  H * 64, _p(delta), B, H, Lq, Lk, int(causal), scale, _stream()), "attention_bwd")
    return dq, dk, dv


# ------------------------------------------------------------------- combiner + bank loss
def bank_dim(D):
    """Smallest supported bank width >= D (queries/banks are zero-padded to it)."""
    for d in BANK_DIMS:
        if d >= D:
            return d
    raise ValueError(f"embedding dim {D} > {BANK_DIMS[-1]} not supported by the bank kernels")


class Fp8Bank:
    """Static bank as OCP e4m3 bytes [M, Dp] + one fp32 scale per row.  Accepted wherever a
    bf16 bank is (bank_stats_fwd / bank_grad_q dispatch on it)."""

    def __init__(self, data, scale):
        self.data, self.scale = data, scale

    @property
    def shape(self):
        return self.data.shape

    @property
    def device(self):
        return self.data.device

    def dequantize(self):
        """fp32 [M, Dp] exactly as the kernels see it before the bf16 rounding."""
        return self.data.view(torch.float8_e4m3fn).float() * self.scale[:, None]

    def bf16_image(self):
        """bf16 [M, Dp] = the expansion the fp8 kernels make per pass at large batches, made ONCE and kept
        (spn_bank_dequant_fp8).  Used by the bank calls from FP8_IMAGE_MIN_B queries per call on."""
        if getattr(self, "_image", None) is None:
            M, Dp = self.data.shape
            img = torch.empty(M, Dp, dtype=torch.bfloat16, device=self.data.device)
            check(lib().spn_bank_dequant_fp8(_p(self.data), _p(self.scale), M, Dp, _p(img), _stream()), "bank_dequant_fp8")
            self._image = img
        return self._image


# From this many queries per call on the bank pass is bound by MFMA issue, not by the bank's bytes: an e4m3 bank is used through
# its kept bf16 image (same values as the kernels' per-pass expansion; +2 B per element of HBM) and the saved-probabilities
# backward applies.  Below it the e4m3 bytes are streamed (half the bytes of the one HBM stream of the loss).
FP8_IMAGE_MIN_B = 256


def fp8_image_min_b():
    """Query count from which an e4m3 bank is served through its kept bf16 image.  SPN_FP8_IMAGE_MIN_B overrides the default
    (256): 0 = never build the image (memory-bound deployments: +2 bytes per bank element stay unspent; large batches then
    expand the shard per pass inside the library), any other value = the threshold."""
    v = os.environ.get("SPN_FP8_IMAGE_MIN_B")
    if v is None or v.strip() == "":
        return FP8_IMAGE_MIN_B
    n = int(v)
    return (1 << 62) if n <= 0 else n


def bank_operand_kind(bank, B):
    """What the bank calls actually read for `B` queries per call: "bf16", "e4m3" (raw bytes on the fp8 MFMA) or "bf16_image"
    (an e4m3 bank through its kept expansion) - reported by bench.py next to every fp8 number."""
    if isinstance(bank, Fp8Bank):
        return "bf16_image" if B >= fp8_image_min_b() else "e4m3"
    return "bf16"


def _bank_operand(bank, B):
    if isinstance(bank, Fp8Bank) and B >= fp8_image_min_b():
        return bank.bf16_image()
    return bank


def prepare_bank(bank_f32, dtype="bf16"):
    """fp32 [M, D] (L2-normalised rows) -> device bf16 [M, bank_dim(D)], zero padded; dtype="fp8" -> Fp8Bank."""
    M, D = bank_f32.shape
    Dp = bank_dim(D)
    if dtype == "fp8":
        _req(bank_f32, torch.float32, "bank")
        data = torch.empty(M, Dp, dtype=torch.uint8, device=bank_f32.device)
        scale = torch.empty(M, dtype=torch.float32, device=bank_f32.device)
        check(lib().spn_bank_quantize_fp8(_p(bank_f32.contiguous()), M, D, Dp, _p(data), _p(scale), _stream()),
              "bank_quantize_fp8")
        return Fp8Bank(data, scale)
    if dtype != "bf16":
        raise ValueError(dtype)
    out = torch.zeros(M, Dp, dtype=torch.bfloat16, device=bank_f32.device)
    out[:, :D] = bank_f32.to(torch.bfloat16)
    return out


def combine_l2norm_fwd(refer_bank, ref_idx, text, ldq=None):
    """-> (q fp32 [B,D], q bf16 [B,ldq], inv_norm [B]).  A ref_idx outside the bank gives a NaN row (the kernel never
    dereferences it); callers that still hold the indices on the host raise IndexError first (check_index_range)."""
    _req(text, torch.float32, "text")
    B, D = text.shape
    n_refer = 0
    if refer_bank is not None:
        _req(refer_bank, torch.float32, "refer_bank")
        _req(ref_idx, torch.int64, "ref_idx")
        if refer_bank.dim() != 2 or refer_bank.shape[1] != D or ref_idx.numel() != B:
            raise ValueError(f"refer_bank {tuple(refer_bank.shape)} / ref_idx {tuple(ref_idx.shape)} do not match text {tuple(text.shape)}")
        n_refer = refer_bank.shape[0]
    ldq = ldq or bank_dim(D)
    q = torch.empty(B, D, dtype=torch.float32, device=text.device)
    qb = torch.empty(B, ldq, dtype=torch.bfloat16, device=text.device)
    inv = torch.empty(B, dtype=torch.float32, device=text.device)
    check(lib().spn_combine_l2norm_fwd(_p(refer_bank), _p(ref_idx), n_refer, _p(text), _p(q), _p(qb), _p(inv), B, D, ldq,
                                       _stream()), "combine_l2norm_fwd")
    return q, qb, inv


def combine_l2norm_bwd(q, inv_norm, dq, scale=None):
    """scale: optional 1-element fp32 device tensor multiplied into the result on the device (autograd's incoming
    d(loss): no host synchronisation on it)."""
    B, D = q.shape
    dtext = torch.empty(B, D, dtype=torch.float32, device=q.device)
    if scale is not None:
        if scale.dtype != torch.float32 or not scale.is_cuda or scale.numel() != 1:
            raise ValueError("scale must be a 1-element fp32 device tensor")
        check(lib().spn_combine_l2norm_bwd_scaled(_p(q), _p(inv_norm), _p(dq), _p(scale), _p(dtext), B, D, _stream()),
              "combine_l2norm_bwd_scaled")
        return dtext
    check(lib().spn_combine_l2norm_bwd(_p(q), _p(inv_norm), _p(dq), _p(dtext), B, D, _stream()), "combine_l2norm_bwd")
    return dtext


BANK_LOGITS_MAX_BYTES = 1 << 30


def bank_logits_buffer(B, M, device):
    """Scratch of the forward/backward pair (bank_stats_fwd(..., save=buf) / bank_grad_q(..., saved=buf)): the chunk
    partials of the fused single pass, or the saved probabilities / logits of the two-pass pairs - the library routes by
    shape.  None when it would exceed BANK_LOGITS_MAX_BYTES (the backward pass then recomputes the logits).  One buffer
    per forward call (torch's caching allocator): it belongs to that call's autograd / step context until its backward
    has run, so two forwards in flight never share it."""
    n = lib().spn_bank_logits_bytes(B, M)
    if n > BANK_LOGITS_MAX_BYTES:
        return None
    return scratch_bytes(n, device)


def bank_stats_fwd(q_bf16, bank_bf16, labels, inv_tau, m_begin=0, save=None):
    """save (bank_logits_buffer): keep the logits of this call for bank_grad_q(..., saved=save) - no recomputation in the
    backward pass (spn_bank_stats_fwd_save)."""
    B, Dp = q_bf16.shape
    M = bank_bf16.shape[0]
    bank_bf16 = _bank_operand(bank_bf16, B)
    stats = torch.empty(B, 4, dtype=torch.float32, device=q_bf16.device)
    fp8 = isinstance(bank_bf16, Fp8Bank)
    ws = workspace((lib().spn_bank_workspace_bytes_fp8 if fp8 else lib().spn_bank_workspace_bytes)(B, M, Dp), q_bf16.device,
                   "bank")
    if save is not None:
        if not save.is_cuda or save.numel() * save.element_size() < lib().spn_bank_logits_bytes(B, M):
            raise ValueError("save: device scratch of spn_bank_logits_bytes(B, M) bytes (ops.bank_logits_buffer)")
        data, scale = (bank_bf16.data, bank_bf16.scale) if fp8 else (bank_bf16, None)
        check(lib().spn_bank_stats_fwd_save(_p(q_bf16), Dp, _p(data), _p(scale), _p(labels), B, M, Dp, m_begin, inv_tau,
                                            _p(stats), _p(save), _p(ws), ws.numel(), _stream()), "bank_stats_fwd_save")
        return stats
    if fp8:
        check(lib().spn_bank_stats_fwd_fp8(_p(q_bf16), Dp, _p(bank_bf16.data), _p(bank_bf16.scale), _p(labels), B, M, Dp,
                                           m_begin, inv_tau, _p(stats), _p(ws), ws.numel(), _stream()), "bank_stats_fwd_fp8")
        return stats
    check(lib().spn_bank_stats_fwd(_p(q_bf16), Dp, _p(bank_bf16), _p(labels), B, M, Dp, m_begin, inv_tau, _p(stats),
                                   _p(ws), ws.numel(), _stream()), "bank_stats_fwd")
    return stats


def bank_loss_finalize(stats, M_total, label_smoothing=0.0):
    """stats [nshards, B, 4] or [B, 4] -> (row_lse [B], row_loss [B], loss_mean [1])"""
    if stats.dim() == 2:
        stats = stats.unsqueeze(0)
    stats = stats.contiguous()
    n, B, _ = stats.shape
    lse = torch.empty(B, dtype=torch.float32, device=stats.device)
    row = torch.empty(B, dtype=torch.float32, device=stats.device)
    mean = torch.empty(1, dtype=torch.float32, device=stats.device)
    check(lib().spn_bank_loss_finalize(_p(stats), n, B, M_total, label_smoothing, _p(lse), _p(row), _p(mean), _stream()),
          "bank_loss_finalize")
    return lse, row, mean


def bank_grad_q(q_bf16, bank_bf16, labels, inv_tau, row_lse, grad_scale, M_total=None, label_smoothing=0.0, m_begin=0,
                saved=None):
    """saved: the buffer the matching bank_stats_fwd(..., save=...) call filled (spn_bank_grad_q_saved)."""
    B, Dp = q_bf16.shape
    M = bank_bf16.shape[0]
    bank_bf16 = _bank_operand(bank_bf16, B)
    dq = torch.empty(B, Dp, dtype=torch.float32, device=q_bf16.device)
    fp8 = isinstance(bank_bf16, Fp8Bank)
    ws = workspace((lib().spn_bank_workspace_bytes_fp8 if fp8 else lib().spn_bank_workspace_bytes)(B, M, Dp), q_bf16.device,
                   "bank")
    if saved is not None:
        data, scale = (bank_bf16.data, bank_bf16.scale) if fp8 else (bank_bf16, None)
        check(lib().spn_bank_grad_q_saved(_p(q_bf16), Dp, _p(data), _p(scale), _p(labels), B, M, Dp, m_begin, inv_tau,
                                          _p(saved), _p(row_lse), label_smoothing, M_total or M, grad_scale, _p(dq), _p(ws),
                                          ws.numel(), _stream()), "bank_grad_q_saved")
        return dq
    if fp8:
        check(lib().spn_bank_grad_q_fp8(_p(q_bf16), Dp, _p(bank_bf16.data), _p(bank_bf16.scale), _p(labels), B, M, Dp,
                                        m_begin, inv_tau, _p(row_lse), label_smoothing, M_total or M, grad_scale, _p(dq),
                                        _p(ws), ws.numel(), _stream()), "bank_grad_q_fp8")
        return dq
    check(lib().spn_bank_grad_q(_p(q_bf16), Dp, _p(bank_bf16), _p(labels), B, M, Dp, m_begin, inv_tau, _p(row_lse),
                                label_smoothing, M_total or M, grad_scale, _p(dq), _p(ws), ws.numel(), _stream()),
          "bank_grad_q")
    return dq


# -------------------------------------------------------------------------------- AdamW
def tau_grad(q, dqk, tau_dev, dtau_out=None, alpha=1.0, scale_dev=None):
    """-> inv_tau (1-element device tensor); dtau_out (optional 1-element fp32 device tensor) <- -alpha * scale_dev *
    (sum q . dqk) / tau^2 (spn_tau_grad; dqk may carry padding columns: its leading dimension is passed along)."""
    _req(q, torch.float32, "q")
    _req(dqk, torch.float32, "dqk")
    B, D = q.shape
    inv = torch.empty(1, dtype=torch.float32, device=q.device)
    check(lib().spn_tau_grad(_p(q), _p(dqk), dqk.stride(0), _p(tau_dev), B, D, float(alpha), _p(scale_dev), _p(dtau_out), _p(inv),
                             _stream()), "tau_grad")
    return inv


def xattn_fwd(q, wkv, bkv, x, heads, cu=None, L=None, scale=0.125, wkv_t=None):
    """Cross-attention over frozen tokens in the absorbed form (spn_xattn_fwd; blip4cir/med.py:97-181, 196-234): q bf16 [rows, W],
    wkv bf16 [2W, E] (key rows, then value rows), bkv fp32 [2W], x bf16 [B, S, E] -> (ctx bf16 [rows, W], saved) where `saved` goes
    to xattn_bwd.  Dense rows = B * L (cu None) or packed (cu int32 [B + 1] device prefix sums, L = the longest length)."""
    _req(q, torch.bfloat16, "q")
    _req(wkv, torch.bfloat16, "wkv")
    _req(x, torch.bfloat16, "x")
    _req(bkv, torch.float32, "bkv")
    B, S, E = x.shape
    rows, W = q.shape
    H = int(heads)
    if cu is None:
        if rows % B:
            raise ValueError("dense rows must be B * L")
        L = rows // B
    elif L is None:
        raise ValueError("packed rows need L (the longest caption)")
    if W != H * 64 or tuple(wkv.shape) != (2 * W, E) or not lib().spn_xattn_ok(B, L, H, S, E):
        raise ValueError("shape not supported by the absorbed cross-attention (spn_xattn_ok)")
    wkv_t = wkv.t().contiguous() if wkv_t is None else wkv_t
    SP = lib().spn_xattn_sp(S)
    qa = torch.empty(rows, H, E, dtype=torch.bfloat16, device=q.device)
    oa = torch.empty_like(qa)
    p = torch.empty(rows * H, SP, dtype=torch.bfloat16, device=q.device)
    ctx = torch.empty(rows, W, dtype=torch.bfloat16, device=q.device)
    check(lib().spn_xattn_fwd(_p(q), _p(wkv), _p(wkv_t), _p(bkv), _p(x), _p(cu), _p(qa), _p(p), _p(oa), _p(ctx), B, L, H, S, E,
                              rows if cu is not None else 0, float(scale), _stream()), "xattn_fwd")
    return ctx, dict(q=q, wkv=wkv, wkv_t=wkv_t, bkv=bkv, x=x, cu=cu, qa=qa, p=p, oa=oa, ctx=ctx, B=B, L=L, H=H, S=S, E=E, rows=rows,
                     scale=float(scale))


def xattn_bwd(saved, dctx):
    """Backward of xattn_fwd: dctx bf16 [rows, W] -> (dq bf16 [rows, W], dwkv fp32 [2W, E], dbkv fp32 [2W])."""
    _req(dctx, torch.bfloat16, "dctx")
    s = saved
    dev = dctx.device
    W = s["H"] * 64
    doa, dqa, ds = torch.empty_like(s["qa"]), torch.empty_like(s["qa"]), torch.empty_like(s["p"])
    delta = torch.empty(s["rows"] * s["H"], dtype=torch.float32, device=dev)
    dq = torch.empty(s["rows"], W, dtype=torch.bfloat16, device=dev)
    dwkv = torch.empty(2 * W, s["E"], dtype=torch.float32, device=dev)
    dbkv = torch.empty(2 * W, dtype=torch.float32, device=dev)
    check(lib().spn_xattn_bwd(_p(dctx), _p(s["ctx"]), _p(s["q"]), _p(s["wkv"]), _p(s["wkv_t"]), _p(s["bkv"]), _p(s["x"]), _p(s["cu"]),
                              _p(s["p"]), _p(s["oa"]), _p(doa), _p(ds), _p(dqa), _p(delta), _p(dq), _p(dwkv), _p(dbkv), s["B"], s["L"],
                              s["H"], s["S"], s["E"], s["rows"] if s["cu"] is not None else 0, s["scale"], _stream()), "xattn_bwd")
    return dq, dwkv, dbkv


def token_bank_bf16(bank, device, chunk=512):
    """fp32 / bf16 [N, S, E] token bank (host or device) -> contiguous bf16 [N, S, E] on `device`, uploaded and converted in
    chunks of `chunk` images (a 30 000 x 577 x 768 bank is 53 GB in fp32: never two copies of it anywhere)."""
    if bank.dim() != 3:
        raise ValueError("token bank must be [N, S, E]")
    if bank.dtype == torch.bfloat16 and bank.is_cuda and bank.is_contiguous():
        return bank
    N, S, E = bank.shape
    out = torch.empty(N, S, E, dtype=torch.bfloat16, device=device)
    for s in range(0, N, chunk):
        blk = bank[s:s + chunk].to(device, non_blocking=False)
        if blk.dtype == torch.float32:
            check(lib().spn_cast_f32_bf16(_p(blk.contiguous()), _p(out[s:s + chunk]), blk.numel(), _stream()), "cast_f32_bf16")
        else:
            out[s:s + chunk].copy_(blk)
    return out


def gather_bank_rows_bf16(bank, idx):
    """out[b] = bank[idx[b]] for a contiguous bf16 [N, ...] device bank and int64 [B] device indices (spn_gather_bank_rows_bf16)."""
    row = bank[0].numel()
    out = torch.empty((idx.numel(),) + tuple(bank.shape[1:]), dtype=torch.bfloat16, device=bank.device)
    check(lib().spn_gather_bank_rows_bf16(_p(bank), bank.shape[0], _p(idx), _p(out), idx.numel(), row, _stream()), "gather_bank_rows")
    return out


def scale_cast_bf16(x, scale_dev, reciprocal=False, ldo=None):
    """bf16(x * s) with s = the 1-element fp32 DEVICE tensor scale_dev (or 1 / s), zero padded to ldo columns: a query
    scaled by a learnable temperature without reading it on the host (spn_scale_cast_bf16)."""
    _req(x, torch.float32, "x")
    if scale_dev.dtype != torch.float32 or not scale_dev.is_cuda or scale_dev.numel() != 1:
        raise ValueError("scale_dev must be a 1-element fp32 device tensor")
    B, D = x.shape
    ldo = ldo or bank_dim(D)
    out = torch.empty(B, ldo, dtype=torch.bfloat16, device=x.device)
    check(lib().spn_scale_cast_bf16(_p(x.contiguous()), _p(scale_dev), 1 if reciprocal else 0, _p(out), B, D, ldo, _stream()),
          "scale_cast_bf16")
    return out


def negtype_head(refer, text, target, tau, neg_type):
    """clip4cir/models_negtype.py's four in-batch terms at the feature level (spn_negtype_head): fp32 [B, D] raw reference,
    text and target features -> (loss [1], d_refer, d_text, d_target)."""
    for n, x in (("refer", refer), ("text", text), ("target", target)):
        _req(x, torch.float32, n)
    B, D = refer.shape
    if text.shape != (B, D) or target.shape != (B, D):
        raise ValueError("refer / text / target must share one [B, D] shape")
    dev = refer.device
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    dr, dt, di = (torch.empty(B, D, dtype=torch.float32, device=dev) for _ in range(3))
    ws = workspace(lib().spn_negtype_workspace_bytes(B, D), dev, "negtype")
    check(lib().spn_negtype_head(_p(refer), _p(text), _p(target), B, D, 1.0 / tau, int(neg_type), _p(loss), _p(dr), _p(dt), _p(di),
                                 _p(ws), ws.numel(), _stream()), "negtype_head")
    return loss, dr, dt, di


def bank_step_ok(B, M, Dp, bank):
    """True when bank_step serves this shape (the single-pass kernels: see spn_bank_step_ok)."""
    return bool(lib().spn_bank_step_ok(B, M, Dp, 1 if isinstance(_bank_operand(bank, B), Fp8Bank) else 0))


def bank_step(q_bf16, bank_bf16, labels, inv_tau, grad_scale, save):
    """Forward and backward of the bank loss for a bank held entirely by this process, label smoothing 0, in two launches
    (spn_bank_step): -> (row_lse [B], row_loss [B], loss_mean [1], dq [B, Dp] fp32 = grad_scale * d(sum row_loss)/dq)."""
    B, Dp = q_bf16.shape
    M = bank_bf16.shape[0]
    dev = q_bf16.device
    bank_bf16 = _bank_operand(bank_bf16, B)
    fp8 = isinstance(bank_bf16, Fp8Bank)
    data, scale = (bank_bf16.data, bank_bf16.scale) if fp8 else (bank_bf16, None)
    if save is None or not save.is_cuda or save.numel() * save.element_size() < lib().spn_bank_logits_bytes(B, M):
        raise ValueError("save: device scratch of spn_bank_logits_bytes(B, M) bytes (ops.bank_logits_buffer)")
    lse = torch.empty(B, dtype=torch.float32, device=dev)
    row = torch.empty(B, dtype=torch.float32, device=dev)
    mean = torch.empty(1, dtype=torch.float32, device=dev)
    dq = torch.empty(B, Dp, dtype=torch.float32, device=dev)
    check(lib().spn_bank_step(_p(q_bf16), Dp, _p(data), _p(scale), _p(labels), B, M, Dp, inv_tau, grad_scale, _p(save), _p(lse),
                              _p(row), _p(mean), _p(dq), _stream()), "bank_step")
    return lse, row, mean, dq


def bank_stats_fwd_tokmax(q_bf16, bank_tok_bf16, labels, inv_tau, t_begin=0):
    """Token-max bank (spn_bank_stats_fwd_tokmax): bank_tok_bf16 [n_targets, 32, Dp] bf16, labels = target ids."""
    B, Dp = q_bf16.shape
    n, g, Db = bank_tok_bf16.shape
    if g != 32 or Db != Dp or not bank_tok_bf16.is_contiguous():
        raise ValueError("token-max bank must be contiguous [n_targets, 32, %d]" % Dp)
    stats = torch.empty(B, 4, dtype=torch.float32, device=q_bf16.device)
    ws = workspace(lib().spn_bank_workspace_bytes(B, n * 32, Dp), q_bf16.device, "bank")
    check(lib().spn_bank_stats_fwd_tokmax(_p(q_bf16), Dp, _p(bank_tok_bf16), _p(labels), B, n, Dp, t_begin, inv_tau,
                                          _p(stats), _p(ws), ws.numel(), _stream()), "bank_stats_fwd_tokmax")
    return stats


def bank_grad_q_tokmax(q_bf16, bank_tok_bf16, labels, inv_tau, row_lse, grad_scale, targets_total=None,
                       label_smoothing=0.0, t_begin=0):
    B, Dp = q_bf16.shape
    n = bank_tok_bf16.shape[0]
    dq = torch.empty(B, Dp, dtype=torch.float32, device=q_bf16.device)
    ws = workspace(lib().spn_bank_workspace_bytes(B, n * 32, Dp), q_bf16.device, "bank")
    check(lib().spn_bank_grad_q_tokmax(_p(q_bf16), Dp, _p(bank_tok_bf16), _p(labels), B, n, Dp, t_begin, inv_tau,
                                       _p(row_lse), label_smoothing, targets_total or n, grad_scale, _p(dq), _p(ws),
                                       ws.numel(), _stream()), "bank_grad_q_tokmax")
    return dq


def adamw_step(p, g, m, v, step, lr, betas=(0.9, 0.999), eps=1e-7, weight_decay=0.01, inv_scale=1.0, found_inf=None):
    check(lib().spn_adamw_step(_p(p), _p(g), _p(m), _p(v), p.numel(), lr, betas[0], betas[1], eps, weight_decay, step,
                               inv_scale, _p(found_inf), _stream()), "adamw_step")


def adamw_tick(step_dev, found_inf=None):
    """step_dev (1-element fp32 device counter) += 1 unless *found_inf != 0; call once per optimizer step."""
    check(lib().spn_adamw_tick(_p(step_dev), _p(found_inf), _stream()), "adamw_tick")


def adamw_step_dev(p, g, m, v, step_dev, lr, betas=(0.9, 0.999), eps=1e-7, weight_decay=0.01, grad_scale=None, found_inf=None):
    """adamw_step with the bias-correction step read from the device counter (skipped steps do not count)."""
    check(lib().spn_adamw_step_dev(_p(p), _p(g), _p(m), _p(v), p.numel(), lr, betas[0], betas[1], eps, weight_decay,
                                   _p(step_dev), _p(grad_scale), _p(found_inf), _stream()), "adamw_step_dev")


_DTYPE_OF = operator.attrgetter("dtype")
ADAMW_CHUNK = 4096            # elements per work item of the many-tensor step
ADAMW_GROUPS = 16             # hyper-parameter sets per call


def ranges_overlap(ptr, nbytes):
    """Whether two of the address ranges share a byte."""
    ptr, nbytes = np.asarray(ptr, np.int64), np.asarray(nbytes, np.int64)
    first, last = ptr[nbytes > 0], (ptr + nbytes)[nbytes > 0]
    order = np.argsort(first, kind="stable")
    return bool((last[order][:-1] > first[order][1:]).any())


class AdamWPlan:
    """What an optimizer keeps between steps of adamw_multi: the tensors' addresses in a device table, and their moments.

    params: fp32 contiguous tensors on one device (no two overlapping; they must stay where they are); state_bits 32 or 8; groups[i]: which
    hyper-parameter set (0..15) tensor i uses (default all 0).  The moments live in padded flat buffers in which tensor i starts at
    offsets[i], a multiple of 128: 32 bits: m, v fp32; 8 bits: m, v uint8 codes with one scale byte per 128 (spn_adamw_multi) - 2.02 bytes per
    parameter instead of 8.  state: (m, v, m_scale, v_scale) to adopt instead of zeros (scales None for 32 bits), or for 32 bits a list of
    (m_i, v_i) fp32 tensors of the parameters' sizes."""

    def __init__(self, params, state_bits=32, groups=None, state=None):
        params = list(params)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits: 8 or 32, not {state_bits!r}")
        if not params:
            raise ValueError("AdamWPlan: no parameters")
        groups = [0] * len(params) if groups is None else [int(g) for g in groups]
        if len(groups) != len(params) or min(groups) < 0 or max(groups) >= ADAMW_GROUPS:
            raise ValueError(f"groups: one of 0..{ADAMW_GROUPS - 1} for each of the {len(params)} parameters")
        dev = params[0].device
        # (whole lists and columns at a time: an optimizer over hundreds of tensors builds this once, but not for milliseconds)
        T = torch.Tensor
        if not dev.type == "cuda":
            _no_cpu()
        if set(map(_DTYPE_OF, params)) != {torch.float32} or not all(map(T.is_contiguous, params)) or set(map(T.get_device, params)) != {dev.index}:
            raise TypeError("AdamWPlan: parameters must be contiguous fp32 tensors on one device")
        n = np.fromiter(map(T.numel, params), np.int64, len(params))
        ptr = np.fromiter(map(T.data_ptr, params), np.int64, len(params))
        if ranges_overlap(ptr, 4 * n):
            raise ValueError("AdamWPlan: parameters overlap (the same tensor twice?)")
        self.params, self._memory = params, list(map(T.untyped_storage, params))       # (the memory lives on if a parameter's data is replaced)
        self.groups, self.state_bits, self.device, self.max_group = groups, state_bits, dev, max(groups)
        self.numels, self.addresses = n.tolist(), ptr.tolist()
        room = (n + 127) // 128 * 128
        off = np.cumsum(room) - room
        self.offsets, at = off.tolist(), int(room.sum())
        self.total = at
        self.m = self.v = self.m_scale = self.v_scale = None
        per = None
        if isinstance(state, list):
            if state_bits != 32 or len(state) != len(params):
                raise ValueError("AdamWPlan: a list of moments goes with 32 bits, one pair per parameter")
            mp, vp = (np.array([_vec(pair[i], size, "mv"[i], dev.index) for pair, size in zip(state, self.numels)], np.int64) for i in (0, 1))
            if ranges_overlap(np.concatenate([ptr, mp, vp]), np.concatenate([4 * n] * 3)):
                raise ValueError("AdamWPlan: moments overlap")
            per = self.own_moments = state
        elif state is not None:
            self.m, self.v, self.m_scale, self.v_scale = state
            dt = torch.uint8 if state_bits == 8 else torch.float32
            for t, size, d in ((self.m, at, dt), (self.v, at, dt)) + (((self.m_scale, at // 128, torch.uint8), (self.v_scale, at // 128, torch.uint8))
                                                                   if state_bits == 8 else ()):
                if t is None or t.dtype != d or t.numel() != size or not t.is_contiguous() or t.device != dev or (t is not self.m_scale and
                                                                                                           t is not self.v_scale and t.data_ptr() % 16):
                    raise ValueError(f"AdamWPlan: state must be contiguous {d} of {size} elements on {dev}")
            held = [t for t in state if t is not None]
            if ranges_overlap(np.concatenate([ptr, [t.data_ptr() for t in held]]), np.concatenate([4 * n, [t.nbytes for t in held]])):
                raise ValueError("AdamWPlan: parameters and state overlap")
        elif state_bits == 8:
            self.m, self.v = (torch.zeros(at, dtype=torch.uint8, device=dev) for _ in range(2))
            self.m_scale, self.v_scale = (torch.zeros(at // 128, dtype=torch.uint8, device=dev) for _ in range(2))
        else:
            self.m, self.v = (torch.zeros(at, dtype=torch.float32, device=dev) for _ in range(2))
        table = np.zeros(len(params), dtype=[(f, np.int64) for f in ("p", "m", "v", "m_scale", "v_scale", "n", "index0")] +
                         [("group", np.int32), ("pad", np.int32)])                      # == spn_adamw_tensor
        table["p"], table["n"], table["index0"], table["group"] = ptr, n, off, groups
        if per is not None:
            table["m"], table["v"] = mp, vp
        else:
            esz = 1 if state_bits == 8 else 4
            table["m"], table["v"] = self.m.data_ptr() + off * esz, self.v.data_ptr() + off * esz
            if state_bits == 8:
                table["m_scale"], table["v_scale"] = self.m_scale.data_ptr() + off // 128, self.v_scale.data_ptr() + off // 128
        k = (n + ADAMW_CHUNK - 1) // ADAMW_CHUNK
        prefix = np.concatenate([[0], np.cumsum(k)])
        if prefix[-1] >= 1 << 31:
            raise ValueError("AdamWPlan: too many elements")
        chunks = np.empty((int(prefix[-1]), 2), np.int32)
        chunks[:, 0] = np.repeat(np.arange(len(params)), k)
        chunks[:, 1] = np.arange(int(prefix[-1])) - np.repeat(prefix[:-1], k)
        # one upload for both tables
        both = torch.from_numpy(np.concatenate([table.view(np.uint8).reshape(-1), chunks.view(np.uint8).reshape(-1)])).to(dev)
        self._table, self._chunks = both[:table.nbytes], both[table.nbytes:]
        self._prefix = (C.c_int32 * len(prefix))(*prefix.tolist())

    def get_device(self):
        return self.device.index

    def __reduce_ex__(self, protocol):
        raise TypeError("an AdamWPlan holds device addresses: build another one (its moments can be saved and handed to it)")

    def moments(self, dtype=torch.float32):
        """(m, v) as numbers in the padded flat layout; 32-bit moments are the buffers themselves (fp32 only)."""
        if self.state_bits == 32:
            if dtype != torch.float32:
                raise ValueError("32-bit moments come as fp32")
            if self.m is None:
                raise ValueError("the moments are the caller's own tensors")
            return self.m, self.v
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"moments: fp32 or bf16, not {dtype}")
        return _adamw_moments(self, dtype)


@_on_device
def _adamw_moments(plan, dtype):
    m, v = (torch.empty(plan.total, dtype=dtype, device=plan.device) for _ in range(2))
    if plan.total == 0:
        return m, v
    check(lib().spn_adamw_moments(plan.m.data_ptr(), plan.m_scale.data_ptr(), plan.v.data_ptr(), plan.v_scale.data_ptr(), m.data_ptr(), v.data_ptr(),
                                  _ELEM[dtype], plan.total, _raw_stream(plan.get_device())), "adamw_moments")
    return m, v


@_on_device
def adamw_multi(plan, grads, step, hyper, seed=0, step_dev=None, inv_scale=1.0, grad_scale=None, found_inf=None):
    """One AdamW step over all tensors of `plan` (AdamWPlan) in one launch (spn_adamw_multi): grads[i] fp32 / bf16 / fp16 contiguous, of
    parameter i's size, or None (that tensor and its moments stay as they are).  hyper: one dict(lr, betas, eps, weight_decay) or a
    list of them, indexed by plan.groups.  step >= 1 enters the bias correction and the rounding of 8-bit moments; step_dev (1-element fp32
    device tensor, adamw_tick) replaces it without a host read.  seed: of that rounding.  inv_scale / grad_scale / found_inf as adamw_step_dev."""
    if not isinstance(plan, AdamWPlan):
        raise TypeError("plan: an AdamWPlan")
    n = len(plan.params)
    if len(grads) != n:
        raise ValueError(f"{len(grads)} gradients for {n} parameters")
    hyper = [hyper] if isinstance(hyper, dict) else list(hyper)
    if len(hyper) > ADAMW_GROUPS or plan.max_group >= len(hyper):
        raise ValueError(f"hyper: {len(hyper)} sets for groups up to {plan.max_group} (at most {ADAMW_GROUPS})")
    if step_dev is None and int(step) < 1:
        raise ValueError("step counts from 1")
    di = plan.device.index
    sp, gsp, fip = (None if t is None else _vec(t, 1, name, di) for name, t in (("step_dev", step_dev), ("grad_scale", grad_scale), ("found_inf", found_inf)))
    # a few hundred tensors per call: whole-list passes of C methods, no per-tensor Python
    T = torch.Tensor
    try:
        sizes, none, live, numels = list(map(T.numel, grads)), False, grads, plan.numels
    except TypeError:                                    # None among them (or no tensor: raised again below)
        none, live, numels = True, [g for g in grads if g is not None], [k for k, g in zip(plan.numels, grads) if g is not None]
        sizes = list(map(T.numel, live))
    if sizes != numels or not all(map(T.is_contiguous, live)) or set(map(T.get_device, live)) - {di}:
        raise ValueError(f"grads: contiguous tensors on {plan.device}, each of its parameter's size (or None)")
    dtypes = set(map(_DTYPE_OF, live))
    if not dtypes <= _ELEM.keys():
        raise ValueError(f"grads: fp32, bf16 or fp16, not {dtypes}")
    if none:
        ptrs = array("Q", [0 if g is None else g.data_ptr() for g in grads])
    else:
        ptrs = array("Q", list(map(T.data_ptr, grads)))
    if len(dtypes) == 1:
        types = bytes((_ELEM[next(iter(dtypes))],)) * n
    else:
        types = bytes([0 if g is None else _ELEM[g.dtype] for g in grads])
    groups = (_lib.AdamwGroup * len(hyper))(*[_lib.AdamwGroup(float(h["lr"]), float(h["betas"][0]), float(h["betas"][1]), float(h["eps"]),
                                                              float(h["weight_decay"])) for h in hyper])
    if plan.total == 0:                                  # tensors without elements: nothing to launch
        return
    check(lib().spn_adamw_multi(plan._table.data_ptr(), plan._chunks.data_ptr(), plan._prefix, ptrs.buffer_info()[0], types, n, groups, len(hyper),
                                plan.state_bits, 0 if step_dev is not None else int(step), sp, float(inv_scale), gsp, fip, int(seed) & 0xFFFFFFFF,
                                _raw_stream(di)), "adamw_multi")


def grad_check_finite(g, found_inf):
    check(lib().spn_grad_check_finite(_p(g), g.numel(), _p(found_inf), _stream()), "grad_check_finite")


# ----------------------------------------------------------------------------- Recall@K
def cosine_scores_f64(q, gallery):
    _req(q, torch.float32, "q"); _req(gallery, torch.float32, "gallery")
    Nq, D = q.shape
    Ng = gallery.shape[0]
    out = torch.empty(Nq, Ng, dtype=torch.float64, device=q.device)
    check(lib().spn_cosine_scores_f64(_p(q), _p(gallery), Nq, Ng, D, _p(out), _stream()), "cosine_scores_f64")
    return out


def topk_from_scores(scores, K, exclude=None):
    Nq, Ng = scores.shape
    idx = torch.empty(Nq, K, dtype=torch.int32, device=scores.device)
    val = torch.empty(Nq, K, dtype=torch.float64, device=scores.device)
    check(lib().spn_topk_from_scores(_p(scores), Nq, Ng, K, _p(exclude), _p(idx), _p(val), _stream()), "topk")
    return idx, val


def inbatch_grad_t(qb, tb, lse, inv_tau, grad_scale, D):
    """In-batch negatives (clip4cir/models.py:160-167): target-side gradient fp32 [B, D] of the mean CE whose
    query-side gradient is bank_grad_q(qb, tb, arange(B), ...)."""
    _req(qb, torch.bfloat16, "qb"); _req(tb, torch.bfloat16, "tb"); _req(lse, torch.float32, "lse")
    B, ld = qb.shape
    dt = torch.empty(B, D, dtype=torch.float32, device=qb.device)
    check(lib().spn_inbatch_grad_t(_p(qb), _p(tb), ld, _p(lse), B, D, float(inv_tau), float(grad_scale), _p(dt), _stream()),
          "inbatch_grad_t")
    return dt
