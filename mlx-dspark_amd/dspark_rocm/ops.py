"""Torch-facing wrappers of the C ABI: tensor checks, output allocation, current HIP stream.

These are the product path: every function here launches a hand-written gfx950 kernel through
``libdspark_rocm.so`` and raises if the library is unavailable or the call is refused.
"""

from __future__ import annotations

import ctypes
import functools
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

GROUP = 64


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("dspark kernels need tensors on a ROCm device (cuda:N)")


def _require_bf16(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name}: expected bfloat16, got {t.dtype}")


def _require_packed(w: torch.Tensor) -> None:
    if w.dtype not in (torch.int32, torch.uint32):
        raise TypeError(f"packed weights must be int32/uint32 words, got {w.dtype}")


def _rowmajor(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2 or t.stride(-1) != 1:
        raise ValueError(f"{name}: expected a 2-D tensor with unit stride along the last dim")


# ---------------------------------------------------------------------------- quantized matmul


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                     *, group_size: int = GROUP, bits: int = 4, out: torch.Tensor | None = None
                     ) -> torch.Tensor:
    """``x [..., K] @ dequant(w)^T -> [..., N]`` (bf16) on the gfx950 qmm kernel.

    ``w`` packed [N, K*bits/32], ``scales``/``biases`` bf16 [N, K/64]. Any number of rows
    (served in 16-row tiles); the small-M shapes of speculative verify are the target.
    Mirrors ``mx.quantized_matmul(x, w, scales, biases, transpose=True, group_size, bits)``.
    """
    _require_cuda(x, w, scales, biases)
    _require_bf16("x", x)
    _require_packed(w)
    _require_bf16("scales", scales)
    _require_bf16("biases", biases)
    k = x.shape[-1]
    n = w.shape[0]
    if w.shape[1] * 32 // bits != k:
        raise ValueError(f"x K={k} does not match packed weight {tuple(w.shape)} at {bits} bits")
    if scales.shape != (n, k // group_size) or biases.shape != scales.shape:
        raise ValueError(f"scales/biases must be [{n}, {k // group_size}]")
    lead = x.shape[:-1]
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    m = x2.shape[0]
    w = w.contiguous()
    scales = scales.contiguous()
    biases = biases.contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    else:
        _rowmajor("out", out)
        if out.shape != (m, n) or out.dtype != torch.bfloat16:
            raise ValueError(f"out must be bf16 [{m}, {n}]")
    if m:
        nbytes = _lib.load().dspark_qmm_affine_workspace(m, k, n, bits, group_size)
        ws = qmm_workspace(x.device, nbytes)
        _lib.call("dspark_qmm_affine", _ptr(x2), x2.stride(0), m, k, _ptr(w), _ptr(scales),
                  _ptr(biases), n, bits, group_size, _ptr(out), out.stride(0), _ptr(ws),
                  0 if ws is None else ws.numel(), _stream(x))
    return out.reshape(*lead, n)


def quantized_matmul_multi(x_list, w_list, s_list, b_list, *, group_size: int = GROUP, bits: int = 4,
                           outs=None, workspace: torch.Tensor | None = None) -> list[torch.Tensor]:
    """Several ``quantized_matmul`` with the same M, K and bits in ONE launch (q/k/v; gate/up).
    The K slice count of a launch depends on the strips of all its problems, so a matrix gives
    the bits of a separate call whenever the launch keeps its slice count (the usual case; a
    different count reassociates the fp32 slice partials, within the qmm tolerance). An 8-bit
    [4096, 4096] matrix alone takes the whole-K kernel, which may also differ by an fp32 rounding
    of a bias term when one group of 64 x values spans many binades."""
    cnt = len(w_list)
    if not 1 <= cnt <= _lib.MAX_QMM_PROBLEMS:
        raise ValueError(f"1..{_lib.MAX_QMM_PROBLEMS} problems per launch, got {cnt}")
    if len(x_list) == 1 and cnt > 1:
        x_list = list(x_list) * cnt
    probs = (_lib.QmmProblem * cnt)()
    results = []
    m = None
    keep = []
    for i in range(cnt):
        x, w, s, b = x_list[i], w_list[i], s_list[i], b_list[i]
        _require_cuda(x, w, s, b)
        _require_bf16("x", x)
        _require_packed(w)
        k = x.shape[-1]
        x2 = x.reshape(-1, k)
        if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
            x2 = x2.contiguous()
        if m is None:
            m = x2.shape[0]
        elif x2.shape[0] != m:
            raise ValueError("all problems must have the same number of rows")
        n = w.shape[0]
        w, s, b = w.contiguous(), s.contiguous(), b.contiguous()
        y = outs[i] if outs is not None else torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
        keep += [x2, w, s, b, y]
        probs[i] = _lib.QmmProblem(_ptr(x2), x2.stride(0), _ptr(w), _ptr(s), _ptr(b), _ptr(y), y.stride(0), n, k)
        results.append(y.reshape(*x.shape[:-1], n))
    nbytes = _lib.load().dspark_qmm_affine_multi_workspace(probs, cnt, m, bits, group_size)
    ws = _pick(workspace, x_list[0].device, nbytes, qmm=True)
    _lib.call("dspark_qmm_affine_multi", probs, cnt, m, bits, group_size, _ptr(ws),
              0 if ws is None else ws.numel(), _stream(x_list[0]))
    return results


def _nothing_intercepts() -> bool:
    """No tracing, dispatch or function mode, function transform or forward-mode level is active.
    Some of these are asked of names torch keeps to itself; where one of them is gone, the answer
    cannot be known, and the calls that ask keep the torch ops."""
    if torch.jit.is_tracing() or torch.compiler.is_compiling():
        return False
    try:
        return not (torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack()
                    or torch._C._functorch.peek_interpreter_stack() is not None
                    or torch.autograd.forward_ad._current_level >= 0)
    except AttributeError:
        return False


def eager_inference(*ts: torch.Tensor) -> bool:
    """Whether a call on these tensors may go straight to a kernel that autograd, tracing, tensor
    subclasses and function transforms do not see: plain tensors on one ROCm device, nothing that
    records gradients or tangents, no dispatch or function mode and no transform active."""
    first = ts[0]
    if not first.is_cuda or not _nothing_intercepts():
        return False
    grad = torch.is_grad_enabled()
    return all(type(t) in (torch.Tensor, torch.nn.Parameter) and t.device == first.device
               and t.layout == torch.strided and not (grad and t.requires_grad)
               and not (t.is_neg() or t._is_zerotensor()) for t in ts)


def quantized_matmul_wide(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *, bits: int,
                          group_size: int = GROUP, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x [.., K] @ dequant(w)^T (+ bias)`` for many rows (prefill widths) on the matrix cores:
    exact bf16 products, fp32 sums, weights never rounded (``dspark_qmm_wide``). ``bias`` (bf16
    [N]) is added to the bf16 product, as a module adds it."""
    _require_cuda(x, w, scales, biases, bias)
    for name, t in (("x", x), ("scales", scales), ("biases", biases)) + ((("bias", bias),) if bias is not None else ()):
        _require_bf16(name, t)
    _require_packed(w)
    k, n = int(x.shape[-1]), int(w.shape[0])
    if w.dim() != 2 or w.shape[1] * 32 != k * bits or tuple(scales.shape) != (n, k // group_size) \
            or biases.shape != scales.shape or (bias is not None and tuple(bias.shape) != (n,)):
        raise ValueError(f"x K={k}, weight {tuple(w.shape)}, scales {tuple(scales.shape)}, biases {tuple(biases.shape)}")
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or not k <= x2.stride(0) <= 1 << 22 or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()
    bias = None if bias is None else bias.contiguous()
    m = x2.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    if m and n:
        with torch.cuda.device(x.device):
            nbytes = int(_lib.load().dspark_qmm_wide_workspace(m, k, n, bits, group_size))
            ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=x.device)
            _lib.call("dspark_qmm_wide", _ptr(x2), x2.stride(0), m, k, _ptr(w), _ptr(scales), _ptr(biases), n, bits,
                      group_size, _ptr(bias), _ptr(y), y.stride(0), _ptr(ws), nbytes, _stream(x))
    return y.reshape(*x.shape[:-1], n)


class PackedQmm:
    """A quantized [N, K] matrix in the MI355X packed form (``dspark_qmm_pack``): 16-row weight
    tiles in the MFMA lane order plus 16-row x 8-group scale/bias tiles, in one uint8 buffer.
    Products equal those of the reference layout bit for bit."""

    def __init__(self, buf: torch.Tensor, n: int, k: int, bits: int):
        self.buf, self.n, self.k, self.bits = buf, n, k, bits

    @property
    def nbytes(self) -> int:
        return self.buf.numel()


def qmm_packable(n: int, k: int, bits: int, group_size: int = GROUP) -> bool:
    """True when ``dspark_qmm_pack`` accepts [n, k] (K % 512 == 0, 4/8-bit, groups of 64)."""
    return int(_lib.load().dspark_qmm_packed_bytes(n, k, bits, group_size)) > 0


def qmm_pack(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *, bits: int,
             group_size: int = GROUP) -> PackedQmm:
    """Pack the reference layout (uint32 [N, K*bits/32], bf16 scales/biases [N, K/64]) once."""
    _require_cuda(w, scales, biases)
    _require_packed(w)
    n, k = w.shape[0], w.shape[1] * 32 // bits
    w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()
    lib = _lib.load()
    nbytes = int(lib.dspark_qmm_packed_bytes(n, k, bits, group_size))
    if nbytes == 0:
        raise _lib.DsparkError("dspark_qmm_pack", -2, f"[{n}, {k}] {bits}-bit cannot be packed (K % 512 != 0)")
    buf = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    _lib.call("dspark_qmm_pack", _ptr(w), _ptr(scales), _ptr(biases), n, k, bits, group_size, _ptr(buf), nbytes,
              _stream(w))
    return PackedQmm(buf, n, k, bits)


def _packed_problems(x_list, packed_list, outs):
    """(problems, count, M, bits, results, keep-alive list) of a packed multi launch. One x
    tensor given for several problems stays one x (one copy when it must be made contiguous),
    which the one-workgroup-per-CU kernel requires."""
    cnt = len(packed_list)
    if not 1 <= cnt <= _lib.MAX_QMM_PROBLEMS:
        raise ValueError(f"1..{_lib.MAX_QMM_PROBLEMS} problems per launch, got {cnt}")
    if len(x_list) == 1 and cnt > 1:
        x_list = list(x_list) * cnt
    bits = packed_list[0].bits
    probs = (_lib.QmmPackedProblem * cnt)()
    results, keep, m, rows = [], [], None, {}
    for i in range(cnt):
        x, pq = x_list[i], packed_list[i]
        _require_cuda(x, pq.buf)
        _require_bf16("x", x)
        if pq.bits != bits:
            raise ValueError("all packed problems of one launch must share bits")
        k = x.shape[-1]
        if k != pq.k:
            raise ValueError(f"x has K={k}, the packed matrix K={pq.k}")
        x2 = rows.get(id(x))
        if x2 is None:
            x2 = x.reshape(-1, k)
            if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
                x2 = x2.contiguous()
            rows[id(x)] = x2
        if m is None:
            m = x2.shape[0]
        elif x2.shape[0] != m:
            raise ValueError("all problems must have the same number of rows")
        y = outs[i] if outs is not None else torch.empty((m, pq.n), dtype=torch.bfloat16, device=x.device)
        keep += [x, x2, y]
        probs[i] = _lib.QmmPackedProblem(_ptr(x2), x2.stride(0), _ptr(pq.buf), _ptr(y), y.stride(0), pq.n, k)
        results.append(y.reshape(*x.shape[:-1], pq.n))
    return probs, cnt, m, bits, results, keep


PACKED_KERNELS = ("split-K", "whole-K tile", "per CU")


def packed_multi_plan(x_list, packed_list, *, group_size: int = GROUP) -> dict:
    """The kernel ``quantized_matmul_packed_multi`` runs for these operands (host-only query):
    ``kernel`` (one of ``PACKED_KERNELS``), ``slices`` (the split-K association the bits
    follow), ``tiles_per_workgroup`` and ``k_parts`` (per-CU kernel: workgroups per row tile
    along K) and ``workgroups``."""
    probs, cnt, m, bits, _, keep = _packed_problems(x_list, packed_list, None)
    out = (ctypes.c_int32 * 5)()
    _lib.call("dspark_qmm_packed_multi_plan", probs, cnt, m, bits, group_size, out)
    return {"kernel": PACKED_KERNELS[out[0]], "slices": out[1], "tiles_per_workgroup": out[2],
            "workgroups": out[3], "k_parts": out[4]}


def quantized_matmul_packed_multi(x_list, packed_list, *, group_size: int = GROUP, outs=None,
                                  workspace: torch.Tensor | None = None) -> list[torch.Tensor]:
    """``quantized_matmul_multi`` over packed matrices (one launch, same M, K and bits)."""
    probs, cnt, m, bits, results, keep = _packed_problems(x_list, packed_list, outs)
    nbytes = _lib.load().dspark_qmm_packed_multi_workspace(probs, cnt, m, bits, group_size)
    ws = _pick(workspace, x_list[0].device, nbytes, qmm=True)
    _lib.call("dspark_qmm_packed_multi", probs, cnt, m, bits, group_size, _ptr(ws),
              0 if ws is None else ws.numel(), _stream(x_list[0]))
    return results


def quantized_matmul_packed(x: torch.Tensor, packed: PackedQmm, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [.., K] @ dequant(W)^T`` for a packed W -> ``[.., N]`` bf16."""
    return quantized_matmul_packed_multi([x], [packed], outs=None if out is None else [out])[0]


class PackedSwiGLU:
    """Gate and up [N, K] matrices in the pair form (``dspark_qmm_pack_swiglu``): the packed
    layout of 2 ceil(N/16) row tiles, gate tile t then up tile t, for the fused gate / up /
    SwiGLU launch."""

    def __init__(self, buf: torch.Tensor, n: int, k: int, bits: int):
        self.buf, self.n, self.k, self.bits = buf, n, k, bits


def qmm_pack_swiglu(gate, up, *, bits: int, group_size: int = GROUP) -> PackedSwiGLU:
    """Pack (w, scales, biases) of the gate and of the up projection (same shape) into the pair
    form once."""
    (gw, gs, gb), (uw, us, ub) = gate, up
    _require_cuda(gw, gs, gb, uw, us, ub)
    _require_packed(gw)
    _require_packed(uw)
    if gw.shape != uw.shape or gs.shape != us.shape:
        raise ValueError(f"gate {tuple(gw.shape)} and up {tuple(uw.shape)} must have one shape")
    n, k = gw.shape[0], gw.shape[1] * 32 // bits
    args = [t.contiguous() for t in (gw, gs, gb, uw, us, ub)]
    lib = _lib.load()
    nbytes = int(lib.dspark_qmm_swiglu_packed_bytes(n, k, bits, group_size))
    if nbytes == 0:
        raise _lib.DsparkError("dspark_qmm_pack_swiglu", -2, f"[{n}, {k}] {bits}-bit cannot be packed (K % 512 != 0)")
    buf = torch.empty(nbytes, dtype=torch.uint8, device=gw.device)
    _lib.call("dspark_qmm_pack_swiglu", *[_ptr(t) for t in args], n, k, bits, group_size, _ptr(buf), nbytes,
              _stream(gw))
    return PackedSwiGLU(buf, n, k, bits)


def quantized_swiglu_packed(x: torch.Tensor, pair: PackedSwiGLU, *, group_size: int = GROUP,
                            out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x W_gate^T) * (x W_up^T)`` with mlx's bf16 rounding, in one launch -> ``[.., N]``."""
    _require_cuda(x, pair.buf)
    _require_bf16("x", x)
    k = x.shape[-1]
    if k != pair.k:
        raise ValueError(f"x has K={k}, the packed pair K={pair.k}")
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    m = x2.shape[0]
    h = out if out is not None else torch.empty((m, pair.n), dtype=torch.bfloat16, device=x.device)
    lib = _lib.load()
    nbytes = lib.dspark_qmm_swiglu_packed_workspace(pair.n, k, m, pair.bits, group_size)
    ws = _pick(workspace, x.device, nbytes, qmm=True)
    _lib.call("dspark_qmm_swiglu_packed", _ptr(x2), x2.stride(0), _ptr(pair.buf), _ptr(h), h.stride(0), pair.n, k, m,
              pair.bits, group_size, _ptr(ws), 0 if ws is None else ws.numel(), _stream(x))
    return h.reshape(*x.shape[:-1], pair.n)


DEQUANT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # dspark_dtype codes


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *, bits: int,
               group_size: int = GROUP, dtype: torch.dtype = torch.float32,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Packed affine ``w [N, K*bits/32]`` -> ``[N, K]`` in ``dtype`` in one launch
    (``dspark_qmm_dequantize``): ``(scale * q) + bias`` as an fp32 product rounded, then an fp32
    sum rounded, then rounded to ``dtype``; for fp32 these are the bits of
    :func:`dspark_rocm.quant.dequantize` (the reference's ``mx.dequantize``, wide_gemm.py:222)."""
    _require_cuda(w, scales, biases)
    _require_packed(w)
    _rowmajor("w", w)
    if scales.dtype not in DEQUANT_DTYPES or biases.dtype != scales.dtype or dtype not in DEQUANT_DTYPES:
        raise TypeError(f"dequantize: scales/biases {scales.dtype}/{biases.dtype}, out {dtype}")
    n, k = int(w.shape[0]), int(w.shape[1]) * 32 // bits
    scales, biases = scales.contiguous(), biases.contiguous()
    if out is None:
        out = torch.empty((n, k), dtype=dtype, device=w.device)
    elif out.dtype != dtype or tuple(out.shape) != (n, k) or out.stride(-1) != 1:
        raise ValueError(f"dequantize: out must be [{n}, {k}] {dtype} with unit inner stride")
    _lib.call("dspark_qmm_dequantize", _ptr(w), _ptr(scales), _ptr(biases), DEQUANT_DTYPES[scales.dtype], n, k,
              bits, group_size, DEQUANT_DTYPES[dtype], _ptr(out), out.stride(0), _stream(out))
    return out


def stream_read(buf: torch.Tensor, sink: torch.Tensor) -> None:
    """Read every byte of ``buf`` once on the gfx950 streaming-read probe (``dspark_stream_read``);
    ``sink`` is an int32 scalar tensor the kernel practically never writes. For timing."""
    _require_cuda(buf, sink)
    if not buf.is_contiguous():
        raise ValueError("stream_read: contiguous buffer")
    _lib.call("dspark_stream_read", _ptr(buf), buf.numel() * buf.element_size(), _ptr(sink), _stream(buf))


def qmm_supported(m: int, k: int, n: int, bits: int, group_size: int = GROUP) -> bool:
    return _lib.load().dspark_qmm_affine_supported(m, k, n, bits, group_size) == 0


# ---------------------------------------------------------------------------- workspaces

_workspaces: dict[tuple[int, int], torch.Tensor] = {}
_qmm_workspaces: dict[tuple[int, int], torch.Tensor] = {}
# Buffers a larger request superseded. They are never freed: a HIP graph captured earlier may
# still hold their addresses, and freeing one would let the caching allocator hand that memory
# to another tensor which the next replay then overwrites.
_retired: list[torch.Tensor] = []


def _stream_key(device) -> tuple[torch.device, tuple[int, int]]:
    dev = torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    return dev, (idx, torch.cuda.current_stream(dev).cuda_stream)


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A per-(device, stream) scratch buffer reused across calls (stream-ordered reuse is safe;
    two streams never share one). Grows by replacement; a replaced buffer stays allocated."""
    if nbytes <= 0:
        return None
    dev, key = _stream_key(device)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _retired.append(buf)
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _workspaces[key] = buf
    return buf


def qmm_workspace(device: torch.device, nbytes: int) -> torch.Tensor | None:
    """The qmm workspace of (device, current stream): zero-filled when allocated (its arrival
    counters must start at zero; every qmm call leaves them zero). Kept apart from the other
    scratch buffers, which hold arbitrary data between calls. A replaced buffer stays
    allocated, as for :func:`workspace`."""
    if nbytes <= 0:
        return None
    dev, key = _stream_key(device)
    buf = _qmm_workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _retired.append(buf)
        buf = torch.zeros(max(nbytes, 4 << 20), dtype=torch.uint8, device=dev)
        _qmm_workspaces[key] = buf
    return buf


def new_qmm_workspace(device, nbytes: int) -> torch.Tensor | None:
    """A caller-owned qmm workspace of at least ``nbytes`` (zeroed: the arrival counters must
    start at zero), e.g. for a graph-captured engine that must not share the per-stream one."""
    if nbytes <= 0:
        return None
    return torch.zeros(max(int(nbytes), 256 << 10), dtype=torch.uint8, device=device)


def qmm_launch_workspace_bytes(m: int, k: int, ns, bits: int, group_size: int = GROUP) -> int:
    """Workspace bytes of one qmm launch over matrices [n, k] for n in ``ns`` with ``m`` rows
    (the reference and the packed layout plan alike). Host query only: the problem pointers it
    passes are placeholders the library does not dereference."""
    ns = list(ns)
    probs = (_lib.QmmProblem * len(ns))()
    for i, n in enumerate(ns):
        probs[i] = _lib.QmmProblem(256, k, 256, 256, 256, 256, n, n, k)
    return int(_lib.load().dspark_qmm_affine_multi_workspace(probs, len(ns), m, bits, group_size))


def attention_workspace_bound(batch: int, hq: int, hk: int, d: int, max_rows: int) -> int:
    """The most workspace bytes verify attention needs for up to ``max_rows`` query rows at any
    cache length: the plan caps its key blocks by the grid size, not by the length."""
    lib = _lib.load()
    return max(int(lib.dspark_verify_attention_workspace(batch, hq, hk, m, d, 1 << 29)) for m in range(1, max_rows + 1))


def qmm_workspace_reset(ws: torch.Tensor) -> None:
    """Zero the split-K arrival counters of a qmm workspace on the current stream (a fill
    kernel, so it may be captured): restores the state every completed qmm call leaves."""
    _require_cuda(ws)
    _lib.call("dspark_qmm_workspace_reset", _ptr(ws), ws.numel(), _stream(ws))


def _pick(ws: torch.Tensor | None, device, nbytes: int, qmm: bool):
    """The caller's workspace when given (checked for size), else the per-stream one."""
    if ws is None:
        return qmm_workspace(device, nbytes) if qmm else workspace(device, nbytes)
    if ws.numel() < nbytes:
        raise ValueError(f"workspace of {ws.numel()} bytes < {nbytes} needed")
    return ws


# ---------------------------------------------------------------------------- verify attention

ATTN_HEAD_DIMS = (64, 128, 256)   # kernel instances; any head dim d % 8 == 0, d <= 256 runs on the next one up
QUANT_HEAD_DIMS = (64, 128, 256)  # quantized caches: whole groups of 64 along the head dim


def attn_head_dim_ok(d: int) -> bool:
    """The reference's head-dim rule (multirow_attn.py:200, :306): d % 8 == 0 and d <= 256."""
    return 8 <= d <= 256 and d % 8 == 0
ATTN_DTYPES = {torch.bfloat16: 0, torch.float16: 1}   # dspark_dtype codes
KV_BITS = (4, 8)


def _i64x3(t: torch.Tensor):
    arr = (ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))
    return arr


def _attn_dtype(q: torch.Tensor, *others: torch.Tensor) -> int:
    if q.dtype not in ATTN_DTYPES:
        raise TypeError(f"verify attention: q dtype {q.dtype} (bfloat16 or float16)")
    for t in others:
        if t.dtype != q.dtype:
            raise TypeError(f"verify attention: {t.dtype} does not match q's {q.dtype}")
    return ATTN_DTYPES[q.dtype]


def _attn_shapes(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name}: expected [B, H, L, D]")
    B, Hq, mq, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    if k.shape != (B, Hk, L, D) or v.shape != (B, Hk, L, D):
        raise ValueError(f"k/v must be [{B}, Hk, L, {D}]; got {tuple(k.shape)} / {tuple(v.shape)}")
    if k.stride(-1) != 1 or v.stride(-1) != 1:
        raise ValueError("k/v must be contiguous along head_dim")
    return B, Hq, mq, D, Hk, L


def verify_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float, causal: bool = True,
                     tree_anc: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T + mask) v`` for few verify rows over a (strided) KV cache view.

    q bf16 or fp16 [B, Hq, Mq, D] (D % 8 == 0, D <= 256); k/v of q's dtype [B, Hk, L, D] with unit
    stride along D (any batch/head/seq strides, e.g. a ``[..., :L, :]`` slice of a larger
    cache). ``causal``: row i sees keys ``0 .. L - Mq + i``. ``tree_anc`` (uint32/int32 [Mq])
    selects the tree-verify mask.
    """
    _require_cuda(q, k, v)
    dt = _attn_dtype(q, k, v)
    B, Hq, mq, D, Hk, L = _attn_shapes(q, k, v)
    q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    osr = (ctypes.c_int64 * 3)(Hq * mq * D, mq * D, D)
    return _launch_attention(dt, q, k, v, out, osr, scale, causal, tree_anc, None)


def _launch_attention(dt, q, k, v, out, out_strides, scale, causal, tree_anc, ws):
    B, Hq, mq, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    nbytes = _lib.load().dspark_verify_attention_workspace(B, Hq, Hk, mq, D, L)
    ws = _pick(ws, q.device, nbytes, qmm=False)
    anc = None if tree_anc is None else tree_anc.to(device=q.device, dtype=torch.int32).contiguous()
    _lib.call("dspark_verify_attention_typed", dt, _ptr(q), B, Hq, mq, D, _ptr(k), _ptr(v), _i64x3(k), _i64x3(v),
              Hk, L, float(scale), int(bool(causal)), _ptr(anc), _ptr(out), out_strides, _ptr(ws),
              0 if ws is None else ws.numel(), _stream(q))
    return out


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float,
                      causal: bool = True) -> torch.Tensor:
    """Attention over many query rows on the matrix cores (``dspark_prefill_attention``): q
    [B, Hq, M, D], k/v [B, Hk, L, D], bf16 or fp16, D in ``QUANT_HEAD_DIMS``, any batch / head /
    position strides (multiples of 8 elements, 16-byte aligned rows). fp32 scores, probabilities
    and sums; causal from the bottom right (needs L >= M). Returns a contiguous [B, Hq, M, D]."""
    _require_cuda(q, k, v)
    dt = _attn_dtype(q, k, v)
    _attn_shapes(q, k, v)
    B, Hq, M, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    out = torch.empty((B, Hq, M, D), dtype=q.dtype, device=q.device)
    with torch.cuda.device(q.device):
        nbytes = int(_lib.load().dspark_prefill_attention_workspace(B, Hq, Hk, M, L, D))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _lib.call("dspark_prefill_attention", dt, _ptr(q), _i64x3(q), B, Hq, M, D, _ptr(k), _ptr(v), _i64x3(k),
                  _i64x3(v), Hk, L, float(scale), int(bool(causal)), _ptr(out), _ptr(ws), nbytes, _stream(q))
    return out


def verify_attention_blocks(B: int, Hq: int, Hk: int, mq: int, D: int, L: int) -> int:
    return int(_lib.load().dspark_verify_attention_blocks(B, Hq, Hk, mq, D, L))


def verify_attention_quantized(q: torch.Tensor, keys, values, *, scale: float, causal: bool = True, bits: int = 8,
                               group_size: int = GROUP, out: torch.Tensor | None = None, out_strides=None,
                               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Verify attention over a quantized KV cache (mlx-lm ``QuantizedKVCache`` state).

    ``keys`` / ``values`` = (words int32 [B, Hk, L, D*bits/32], scales [B, Hk, L, D/64],
    biases [B, Hk, L, D/64]) with scales/biases in q's dtype, fields of ``bits`` (4 or 8)
    along D, low bits first; any batch/head/seq strides (cache views), unit stride along the
    last dim. Semantics: attention over ``scale * q_field + bias`` per group of 64 values.
    ``out_strides`` = (batch, query head, position) element strides of ``out`` (head_dim
    contiguous), e.g. [B, Mq, Hq*D] rows for o_proj; default a contiguous [B, Hq, Mq, D].
    """
    kw, ks, kb = keys
    vw, vs, vb = values
    _require_cuda(q, kw, ks, kb, vw, vs, vb)
    dt = _attn_dtype(q, ks, kb, vs, vb)
    if bits not in KV_BITS:
        raise ValueError(f"bits={bits} (4 or 8)")
    for t in (kw, vw):
        _require_packed(t)
    B, Hq, mq, D = q.shape
    if D not in QUANT_HEAD_DIMS:
        raise ValueError(f"quantized caches: head_dim {D} (64, 128 or 256)")
    Hk, L = kw.shape[1], kw.shape[2]
    W, G = D * bits // 32, D // group_size
    for name, t, last in (("key words", kw, W), ("value words", vw, W), ("key scales", ks, G), ("key biases", kb, G),
                          ("value scales", vs, G), ("value biases", vb, G)):
        if t.dim() != 4 or tuple(t.shape) != (B, Hk, L, last) or t.stride(-1) != 1:
            raise ValueError(f"{name}: expected [{B}, {Hk}, {L}, {last}] with unit last stride, got {tuple(t.shape)}")
    if ks.stride() != kb.stride() or vs.stride() != vb.stride():
        raise ValueError("scales and biases of one cache must share strides")
    q = q.contiguous()
    if out is None:
        if out_strides is not None:
            raise ValueError("out_strides needs out")
        out = torch.empty_like(q)
    if out.dtype != q.dtype:
        raise TypeError(f"out dtype {out.dtype} does not match q's {q.dtype}")
    osr = (ctypes.c_int64 * 3)(*([Hq * mq * D, mq * D, D] if out_strides is None else [int(x) for x in out_strides]))
    nbytes = _lib.load().dspark_verify_attention_workspace(B, Hq, Hk, mq, D, L)
    ws = _pick(workspace, q.device, nbytes, qmm=False)
    _lib.call("dspark_verify_attention_quantized", dt, _ptr(q), B, Hq, mq, D, _ptr(kw), _ptr(ks), _ptr(kb), _i64x3(kw),
              _i64x3(ks), _ptr(vw), _ptr(vs), _ptr(vb), _i64x3(vw), _i64x3(vs), Hk, L, float(scale),
              int(bool(causal)), bits, group_size, _ptr(out), osr, _ptr(ws), 0 if ws is None else ws.numel(),
              _stream(q))
    return out


# ---------------------------------------------------------------------------- MoE

def moe_route(logits: torch.Tensor, k: int, *, renorm: bool = True, bucket: bool = False):
    """Softmax top-k routing on the GPU. logits bf16 [M, E] -> (inds int32 [M, k], scores bf16
    [M, k]) and, with ``bucket=True``, also (expert_offsets [E+1], sorted_pairs [M*k],
    pair_pos [M*k]) of the (token, slot) pairs sorted by expert."""
    _require_cuda(logits)
    _require_bf16("logits", logits)
    logits = logits.contiguous()
    M, E = logits.shape
    dev = logits.device
    inds = torch.empty((M, k), dtype=torch.int32, device=dev)
    scores = torch.empty((M, k), dtype=torch.bfloat16, device=dev)
    off = srt = pos = None
    if bucket:
        off = torch.empty(E + 1, dtype=torch.int32, device=dev)
        srt = torch.empty(M * k, dtype=torch.int32, device=dev)
        pos = torch.empty(M * k, dtype=torch.int32, device=dev)
    _lib.call("dspark_moe_route_topk", _ptr(logits), M, E, k, int(bool(renorm)), _ptr(inds), _ptr(scores),
              _ptr(off), _ptr(srt), _ptr(pos), _stream(logits))
    if bucket:
        return inds, scores, off, srt, pos
    return inds, scores


def gather_qmm_sorted(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                      expert_offsets: torch.Tensor, *, row_index: torch.Tensor | None = None, bits: int = 4,
                      group_size: int = GROUP, rows: int | None = None) -> torch.Tensor:
    """Grouped qmm over expert-sorted rows: ``y[p] = x[row_index[p]] @ dequant(w[e])^T`` for
    ``expert_offsets[e] <= p < expert_offsets[e+1]``. w packed [E, N, K*bits/32]."""
    _require_cuda(x, w, scales, biases, expert_offsets)
    _require_bf16("x", x)
    _require_packed(w)
    E, N = w.shape[0], w.shape[1]
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    P = rows if rows is not None else (row_index.numel() if row_index is not None else x2.shape[0])
    y = torch.empty((P, N), dtype=torch.bfloat16, device=x.device)
    ri = None if row_index is None else row_index.to(torch.int32).contiguous()
    _lib.call("dspark_gather_qmm", _ptr(x2), x2.stride(0), K, _ptr(ri), _ptr(expert_offsets.to(torch.int32).contiguous()),
              E, P, _ptr(w.contiguous()), _ptr(scales.contiguous()), _ptr(biases.contiguous()), N, bits, group_size,
              _ptr(y), y.stride(0), _stream(x))
    return y


class PackedExperts:
    """Stacked expert weights [E, N, K*bits/32] in the packed form of ``dspark_moe_pack``: each
    expert's 16-row tiles in the MFMA lane order (the same bytes; scales and biases are not part
    of it and keep their [E, N, K/64] layout)."""

    def __init__(self, buf: torch.Tensor, experts: int, n: int, k: int, bits: int):
        self.buf, self.experts, self.n, self.k, self.bits = buf, experts, n, k, bits


def moe_packable(experts: int, n: int, k: int, bits: int, group_size: int = GROUP) -> bool:
    return int(_lib.load().dspark_moe_packed_bytes(experts, n, k, bits, group_size)) > 0


MOE_KERNELS = ("expert x strip", "per CU", "row tiles")


def moe_packed_plan(M: int, H: int, I: int, E: int, k: int, bits: int) -> dict:
    """The expert kernels ``moe_switch_glu`` runs over packed experts for this shape (host-only
    query): ``gate_up`` and ``down``, each one of ``MOE_KERNELS``."""
    out = (ctypes.c_int32 * 2)()
    _lib.call("dspark_moe_packed_plan", M, H, I, E, k, bits, out)
    return {"gate_up": MOE_KERNELS[out[0]], "down": MOE_KERNELS[out[1]]}


def moe_pack(w: torch.Tensor, *, bits: int, group_size: int = GROUP) -> PackedExperts:
    """Pack stacked expert weights (int32 [E, N, K*bits/32]) once (N % 16 == 0, K % 128 == 0)."""
    _require_cuda(w)
    _require_packed(w)
    E, n, k = w.shape[0], w.shape[1], w.shape[2] * 32 // bits
    w = w.contiguous()
    nbytes = int(_lib.load().dspark_moe_packed_bytes(E, n, k, bits, group_size))
    if nbytes == 0:
        raise _lib.DsparkError("dspark_moe_pack", -2, f"[{E}, {n}, {k}] {bits}-bit cannot be packed "
                                                      "(N % 16 == 0 and K % 128 == 0 needed)")
    buf = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    _lib.call("dspark_moe_pack", _ptr(w), E, n, k, bits, group_size, _ptr(buf), nbytes, _stream(w))
    return PackedExperts(buf, E, n, k, bits)


def moe_switch_glu(x: torch.Tensor, logits: torch.Tensor, gate, up, down, *, k: int, bits: int = 4,
                   renorm: bool = True, group_size: int = GROUP):
    """Routed-expert SwiGLU MLP of one MoE block: route -> gate/up (fused SwiGLU) -> down ->
    score-weighted combine, four launches. ``gate``/``up``/``down`` are (w, scales, biases) with
    w int32 [E, rows, cols*bits/32], or a :class:`PackedExperts` of it (``dspark_moe_switch_glu_packed``,
    the same results bit for bit). Returns (out bf16 [M, H], inds [M, k], scores [M, k])."""
    _require_cuda(x, logits)
    _require_bf16("x", x)
    _require_bf16("logits", logits)
    x = x.contiguous()
    logits = logits.contiguous()
    M, H = x.shape
    E = logits.shape[1]
    packed = isinstance(gate[0], PackedExperts)
    if packed != isinstance(up[0], PackedExperts) or packed != isinstance(down[0], PackedExperts):
        raise ValueError("moe_switch_glu: gate, up and down must all be packed or all row-major")
    I = gate[0].n if packed else gate[0].shape[1]
    lib = _lib.load()
    nbytes = lib.dspark_moe_workspace(M, H, I, E, k)
    if nbytes == 0:
        raise ValueError(f"unsupported MoE shape M={M} E={E} k={k}")
    ws = workspace(x.device, nbytes)
    out = torch.empty((M, H), dtype=torch.bfloat16, device=x.device)
    inds = torch.empty((M, k), dtype=torch.int32, device=x.device)
    scores = torch.empty((M, k), dtype=torch.bfloat16, device=x.device)
    (wg, sg, bg), (wu, su, bu), (wd, sd, bd) = gate, up, down
    if packed:
        wg, wu, wd = wg.buf, wu.buf, wd.buf
    _lib.call("dspark_moe_switch_glu_packed" if packed else "dspark_moe_switch_glu", _ptr(x), _ptr(logits), M, H, I,
              E, k, int(bool(renorm)), _ptr(wg), _ptr(sg), _ptr(bg), _ptr(wu), _ptr(su), _ptr(bu), _ptr(wd),
              _ptr(sd), _ptr(bd), bits, group_size, _ptr(out), _ptr(inds), _ptr(scores), _ptr(ws), ws.numel(),
              _stream(x))
    return out, inds, scores


def verify_attention_into(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, out_strides, *,
                          scale: float, causal: bool = True, tree_anc: torch.Tensor | None = None,
                          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`verify_attention` writing through element strides ``out_strides`` = (batch, query
    head, position) of ``out`` (head_dim contiguous), e.g. [B, Mq, Hq*D] rows for o_proj."""
    _require_cuda(q, k, v, out)
    dt = _attn_dtype(q, k, v, out)
    _attn_shapes(q, k, v)
    q = q.contiguous()
    osr = (ctypes.c_int64 * 3)(*[int(x) for x in out_strides])
    return _launch_attention(dt, q, k, v, out, osr, scale, causal, tree_anc, workspace)


# ---------------------------------------------------------------------------- verify-forward layer ops

def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, *, residual: torch.Tensor | None = None,
            h_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``bf16(bf16(h * rsqrt(mean(h^2) + eps)) * w)`` per row, h = x or bf16(x + residual)
    (written to ``h_out`` when given). x [M, H] bf16."""
    _require_cuda(x, w)
    _require_bf16("x", x)
    M, H = x.shape
    if out is None:
        out = torch.empty((M, H), dtype=torch.bfloat16, device=x.device)
    _lib.call("dspark_rmsnorm", _ptr(x), x.stride(0), _ptr(residual), 0 if residual is None else residual.stride(0),
              _ptr(w), M, H, float(eps), _ptr(h_out), 0 if h_out is None else h_out.stride(0), _ptr(out),
              out.stride(0), _stream(x))
    return out


def qk_norm_rope_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm_w: torch.Tensor,
                    k_norm_w: torch.Tensor, *, heads: int, kv_heads: int, head_dim: int, eps: float,
                    rope_base: float, pos0: int, q_out: torch.Tensor, k_cache: torch.Tensor,
                    v_cache: torch.Tensor) -> torch.Tensor:
    """q/k RMSNorm + RoPE at positions pos0.. and the cache write. q [M, Hq*D], k/v [M, Hk*D];
    q_out [Hq, M, D]; k_cache/v_cache [Hk, capacity, D] views (batch 1)."""
    _require_cuda(q, k, v, q_out, k_cache, v_cache)
    M = q.shape[0]
    if k_cache.shape[1] < pos0 + M or v_cache.shape[1] < pos0 + M:
        raise ValueError(f"cache capacity {k_cache.shape[1]} < pos0 + M = {pos0 + M}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dim() != 3 or t.shape[0] < kv_heads or t.shape[2] < head_dim:
            raise ValueError(f"{name}: expected [{kv_heads}, capacity, {head_dim}], got {tuple(t.shape)}")
    ks = (ctypes.c_int64 * 2)(k_cache.stride(0), k_cache.stride(1))
    vs = (ctypes.c_int64 * 2)(v_cache.stride(0), v_cache.stride(1))
    _lib.call("dspark_qk_norm_rope_kv", _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), M, heads,
              kv_heads, head_dim, _ptr(q_norm_w), _ptr(k_norm_w), float(eps), float(rope_base), int(pos0),
              _ptr(q_out), _ptr(k_cache), ks, _ptr(v_cache), vs, _stream(q))
    return q_out


def qk_norm_rope_kv_quantized(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm_w: torch.Tensor,
                              k_norm_w: torch.Tensor, *, heads: int, kv_heads: int, head_dim: int, eps: float,
                              rope_base: float, pos0: int, q_out: torch.Tensor, k_cache, v_cache, bits: int,
                              group_size: int = GROUP) -> torch.Tensor:
    """:func:`qk_norm_rope_kv` into a quantized cache: ``k_cache`` / ``v_cache`` are the
    (words [Hk, capacity, D*bits/32], scales [Hk, capacity, D/64], biases) triples of one
    layer (batch 1, bf16 scales); the rows at pos0.. are quantized as ``quant.quantize_rows``
    quantizes the values the plain kernel would write."""
    kw, ks, kb = k_cache
    vw, vs, vb = v_cache
    _require_cuda(q, k, v, q_out, kw, ks, kb, vw, vs, vb)
    for t in (ks, kb, vs, vb):
        _require_bf16("cache scales / biases", t)
    M = q.shape[0]
    W, G = head_dim * bits // 32, head_dim // group_size
    for name, t, last in (("key words", kw, W), ("value words", vw, W), ("key scales", ks, G), ("key biases", kb, G),
                          ("value scales", vs, G), ("value biases", vb, G)):
        if t.dim() != 3 or t.shape[1] < pos0 + M or t.stride(-1) != 1:
            raise ValueError(f"{name}: expected [Hk, capacity >= {pos0 + M}, ...] with unit last stride")
        if t.shape[0] < kv_heads or t.shape[2] < last:
            raise ValueError(f"{name}: expected [{kv_heads}, capacity, {last}], got {tuple(t.shape)}")
    if ks.stride() != kb.stride() or vs.stride() != vb.stride():
        raise ValueError("scales and biases of one cache must share strides")
    two = lambda t: (ctypes.c_int64 * 2)(t.stride(0), t.stride(1))
    _lib.call("dspark_qk_norm_rope_kv_quantized", _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), M,
              heads, kv_heads, head_dim, _ptr(q_norm_w), _ptr(k_norm_w), float(eps), float(rope_base), int(pos0),
              _ptr(q_out), _ptr(kw), _ptr(ks), _ptr(kb), two(kw), two(ks), _ptr(vw), _ptr(vs), _ptr(vb), two(vw),
              two(vs), int(bits), int(group_size), _stream(q))
    return q_out


def swiglu(g: torch.Tensor, u: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``bf16(bf16(g * bf16(sigmoid(g))) * u)`` (mlx's silu(g) * u)."""
    _require_cuda(g, u)
    M, N = g.shape
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=g.device)
    _lib.call("dspark_swiglu", _ptr(g), g.stride(0), _ptr(u), u.stride(0), M, N, _ptr(out), out.stride(0), _stream(g))
    return out


def argmax_rows(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """int32 [M]: first index of each row's maximum (bf16 logits [M, V])."""
    _require_cuda(logits)
    _require_bf16("logits", logits)
    M, V = logits.shape
    if out is None:
        out = torch.empty(M, dtype=torch.int32, device=logits.device)
    _lib.call("dspark_argmax_rows", _ptr(logits), logits.stride(0), M, V, _ptr(out), _stream(logits))
    return out


def greedy_accept(draft: torch.Tensor, target_tokens: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """int32 [1]: length of the accepted draft prefix (draft == target_tokens[:m] while equal)."""
    _require_cuda(target_tokens)
    m = int(draft.numel())
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=target_tokens.device)
    d = draft.to(device=target_tokens.device, dtype=torch.int32).contiguous() if m else None
    _lib.call("dspark_greedy_accept", _ptr(d), m, _ptr(target_tokens), _ptr(out), _stream(target_tokens))
    return out


def argmax_accept_workspace_bytes(M: int, V: int) -> int:
    """Workspace bytes of :func:`argmax_accept` for ``M`` rows of ``V`` logits."""
    return int(_lib.load().dspark_argmax_accept_workspace(M, V))


def argmax_accept(logits: torch.Tensor, draft: torch.Tensor, target_tokens: torch.Tensor, n_accepted: torch.Tensor,
                  workspace: torch.Tensor) -> None:
    """:func:`argmax_rows` into ``target_tokens`` and :func:`greedy_accept` of ``draft`` into
    ``n_accepted``, in one launch. ``workspace`` (uint8, >= :func:`argmax_accept_workspace_bytes`,
    zero-filled when allocated) holds an arrival counter that every call leaves at zero."""
    _require_cuda(logits, target_tokens, n_accepted, workspace)
    _require_bf16("logits", logits)
    M, V = logits.shape
    m = int(draft.numel())
    if m and (draft.dtype != torch.int32 or not draft.is_contiguous() or draft.device != logits.device):
        raise ValueError("argmax_accept: draft must be a contiguous int32 tensor on the logits' device")
    _lib.call("dspark_argmax_accept", _ptr(logits), logits.stride(0), M, V, _ptr(draft) if m else None, m,
              _ptr(target_tokens), _ptr(n_accepted), _ptr(workspace), workspace.numel(), _stream(logits))


# ---------------------------------------------------------------------------- sampled rounds
#
# The entry points from here on take one struct of 8-byte fields (include/dspark.h): packing it costs a tenth of
# converting twenty arguments one by one, which is what a call of a few microseconds is made of.

LOGIT_DTYPES = {torch.bfloat16: 0, torch.float16: 1}    # dspark_dtype codes
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)     # the stream's handle without a Stream object


def _call_on(dev: torch.device, name: str, args: bytes) -> None:
    """``name(args, current stream of dev)`` with dev as the current device (a launch needs its stream's to be)."""
    index = dev.index
    if index == torch.cuda.current_device():
        status = getattr(_lib.load(), name)(args, torch.cuda.current_stream(dev).cuda_stream if _raw_stream is None
                                            else _raw_stream(index))
        if status:
            _lib.check(name, status)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, args, torch.cuda.current_stream(dev).cuda_stream)


def _forward_level() -> bool:
    """Whether tensors may have tangents (without the name torch keeps to itself: every one is asked)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def _no_autograd(what: str, *ts) -> None:
    """ValueError where autograd follows one of the tensors: gradients while they are recorded, tangents always
    (forward mode asks neither for requires_grad nor for grad mode)."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: has no backward pass; detach its inputs or use torch.no_grad()")
    if _forward_level():
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what}: has no derivative for a tangent; take the primal of its inputs")


def _as_stored(what: str, *ts) -> None:
    """ValueError for a view that negates its memory where it is read: what a kernel writes there, or reads as a cache,
    is the memory itself. (Plain inputs of this kind are copied: resolve_neg.)"""
    for t in ts:
        if t is not None and t.is_neg():
            raise ValueError(f"{what}: a view that negates its memory; take its resolve_neg()")


def _one_device(what: str, first: torch.Tensor, *ts) -> torch.device:
    if not first.is_cuda:
        raise ValueError("dspark kernels need tensors on a ROCm device (cuda:N)")
    index = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != index:       # -1 for the CPU
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")
    return first.device


def check_sampler(temperature, top_k, top_p) -> tuple[float, int, float]:
    """The sampler's settings as the kernels take them; ValueError where they refuse them."""
    t, k, p = float(temperature), min(int(top_k or 0), 1 << 31), float(top_p)
    if not 1e-30 <= t <= 1e30:
        raise ValueError(f"temperature={temperature}: a positive number (greedy rounds: argmax_accept)")
    if k < 0 or not 0.0 < p <= 1.0:
        raise ValueError(f"top_k={top_k} (0 or more), top_p={top_p} (over 0, up to 1)")
    return t, k, p


def _sampling_workspace(ws, device, rows: int, vocab: int, sequences: int, top_k: int, top_p: float) -> torch.Tensor:
    nbytes = sampling_workspace_bytes(rows, vocab, sequences, top_k, top_p)
    if nbytes == 0:
        raise ValueError(f"{rows} rows of {vocab} logits (up to 65535 rows of 524280)")
    if ws is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if ws.numel() * ws.element_size() < nbytes or not ws.is_contiguous():
        raise ValueError(f"workspace: {nbytes} contiguous bytes on {device} needed")
    return ws


@functools.lru_cache(maxsize=256)
def sampling_workspace_bytes(rows: int, vocab: int, sequences: int = 0, top_k: int | None = None, top_p: float = 1.0) -> int:
    """Workspace bytes of :func:`sampling_probs` over ``rows`` rows, or of :func:`speculative_verify`
    over ``sequences`` sequences of ``rows`` rows together: with any settings, or (``top_k`` given) with these."""
    lib = _lib.load()
    if top_k is None:
        return int(lib.dspark_sampling_workspace(rows, vocab, sequences))
    return int(lib.dspark_sampling_workspace_for(rows, vocab, sequences, top_k, top_p))


_PROBS_ARGS = struct.Struct("=5qdqd4q")


def sampling_probs(logits: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                   out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The probabilities a token is sampled from, fp32 [..., V]: softmax of ``logits / temperature``
    (bf16 or fp16 [..., V]) over the ``top_k`` largest logits (0: all), of these over the tokens before
    which less than ``top_p`` of their mass lies, 0 elsewhere. Equal logits are ordered by index; a row
    of nothing but -inf and NaN gives zeros. What a drafter samples its tokens from and hands to
    :func:`speculative_verify`. ``out`` contiguous; ``workspace`` (any content) of
    :func:`sampling_workspace_bytes`, 256-byte aligned, for one call at a time, else allocated."""
    dev = _one_device("sampling_probs", logits, out, workspace)
    dt = LOGIT_DTYPES.get(logits.dtype)
    if dt is None:
        raise TypeError(f"sampling_probs: logits {logits.dtype} (bfloat16 or float16)")
    shape = logits.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"sampling_probs: logits {list(shape)}")
    _no_autograd("sampling_probs", logits, out)
    if logits.is_neg():
        logits = logits.resolve_neg()
    t, k, p = check_sampler(temperature, top_k, top_p)
    V = shape[-1]
    x = logits if len(shape) == 2 else logits.reshape(-1, V)
    rows, (ld, unit) = x.shape[0], x.stride()
    if unit != 1 or ld < V:
        x, ld = x.contiguous(), V
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    elif out.dtype != torch.float32 or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"sampling_probs: out must be contiguous fp32 {list(shape)}")
    else:
        _as_stored("sampling_probs", out)
    if rows:
        ws = _sampling_workspace(workspace, dev, rows, V, 0, k, p)
        _call_on(dev, "dspark_sampling_probs",
                 _PROBS_ARGS.pack(dt, x.data_ptr(), ld, rows, V, t, k, p, out.data_ptr(), V, ws.data_ptr(), ws.nbytes))
    return out


def _ints(what: str, name: str, t: torch.Tensor, shape: tuple) -> torch.Tensor:
    if t.dtype is torch.int32 and t.shape == shape:
        return t.contiguous()
    if t.dtype is not torch.int64 or t.shape != shape:
        raise ValueError(f"{what}: {name} must be int32 or int64 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous()    # an id past 32 bits stays one that no vocabulary has


_VERIFY_ARGS = struct.Struct("=14qdqd5q")


def speculative_verify(logits: torch.Tensor, draft: torch.Tensor, uniforms: torch.Tensor, *,
                       draft_probs: torch.Tensor | None = None, draft_lens: torch.Tensor | None = None,
                       temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                       workspace: torch.Tensor | None = None):
    """The accept rule of a sampled round: ``(n_accepted int32 [B], tokens int32 [B, m + 1], draft_p fp32
    [B, m])`` for the logits bf16 / fp16 [B, m + 1, V] of ``[anchor] + m drafts`` per sequence, with p the
    rows :func:`sampling_probs` forms of them (in 64 bits).

    Draft i is accepted while all before it are and ``uniforms[b, i] * q < p`` at the drafted token
    (``draft_probs`` fp32 [B, m, V], normalised as the drafter sampled from it; None: q = 1, a drafter
    without probabilities). ``tokens`` are the accepted drafts, then one drawn with ``uniforms[b, m]``
    from ``max(p - q, 0)`` of the refused row, or from p of the row after the last draft, then -1; the
    committed tokens then follow p whatever the drafter proposed. ``draft_p``: p of every draft.
    ``draft_lens`` [B] (padded batches): how many drafts each sequence has. ``uniforms`` [B, m + 1] fp32 or
    fp64 in [0, 1). Drafts outside the vocabulary are refused. m up to 255. ``workspace`` as in
    :func:`sampling_probs`: two streams, or two graphs that may run together, need one each."""
    what = "speculative_verify"
    dev = _one_device(what, logits, draft, uniforms, draft_probs, draft_lens, workspace)
    dt = LOGIT_DTYPES.get(logits.dtype)
    if dt is None:
        raise TypeError(f"{what}: logits {logits.dtype} (bfloat16 or float16)")
    shape = logits.shape
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"{what}: logits must be [B, drafts + 1, V], got {list(shape)}")
    B, R, V = shape
    m = R - 1
    if m > 255:
        raise ValueError(f"{what}: {m} drafts (up to 255)")
    udt = uniforms.dtype
    u64 = udt is torch.float64
    if not (u64 or udt is torch.float32) or uniforms.shape != (B, R):
        raise ValueError(f"{what}: uniforms must be fp32 or fp64 [{B}, {R}], got {uniforms.dtype} {list(uniforms.shape)}")
    t, k, p = check_sampler(temperature, top_k, top_p)
    _no_autograd(what, logits, draft_probs)
    draft = _ints(what, "draft", draft, (B, m))
    q = q_seq = q_row = 0
    if draft_probs is not None:
        if draft_probs.dtype is not torch.float32 or draft_probs.shape != (B, m, V):
            raise ValueError(f"{what}: draft_probs must be fp32 [{B}, {m}, {V}], got {draft_probs.dtype} {list(draft_probs.shape)}")
        q_seq, q_row, unit = draft_probs.stride()
        if (unit != 1 and V > 1) or draft_probs.is_neg():
            draft_probs = draft_probs.resolve_neg().contiguous()
            q_seq, q_row, _ = draft_probs.stride()
        q = draft_probs.data_ptr()
        if not q and draft_probs.numel():
            raise ValueError(f"{what}: draft_probs without memory")
    lens = 0
    if draft_lens is not None:
        draft_lens = _ints(what, "draft_lens", draft_lens, (B,))
        lens = draft_lens.data_ptr()
    ld_seq, ld_row, unit = logits.stride()
    if (unit != 1 and V > 1) or logits.is_neg():
        logits = logits.resolve_neg().contiguous()
        ld_seq, ld_row, _ = logits.stride()
    if uniforms.is_neg() or not uniforms.is_contiguous():
        uniforms = uniforms.resolve_neg().contiguous()
    n = torch.empty(B, dtype=torch.int32, device=dev)
    tokens = torch.empty(B, R, dtype=torch.int32, device=dev)
    draft_p = torch.empty(B, m, dtype=torch.float32, device=dev)
    if B:
        ws = _sampling_workspace(workspace, dev, B * R, V, B, k, p)
        _call_on(dev, "dspark_speculative_verify",
                 _VERIFY_ARGS.pack(dt, logits.data_ptr(), ld_seq, ld_row, B, m, V, draft.data_ptr(), q, q_seq, q_row, lens,
                                   uniforms.data_ptr(), u64, t, k, p, n.data_ptr(), tokens.data_ptr(), draft_p.data_ptr(),
                                   ws.data_ptr(), ws.nbytes))
    return n, tokens, draft_p


# ---------------------------------------------------------------------------- what tokens are reported with

MOST_ALTERNATIVES = 64


@functools.lru_cache(maxsize=256)
def token_logprobs_workspace_bytes(rows: int, vocab: int, top: int = 0) -> int:
    """Workspace bytes of :func:`token_logprobs`; 0 where it refuses the sizes."""
    return int(_lib.load().dspark_token_logprobs_workspace(rows, vocab, top))


_SCORE_ARGS = struct.Struct("=8qd6q")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 1.0,
                   workspace: torch.Tensor | None = None):
    """What a token is reported with, in one pass over its logits: ``(logprobs fp32 [...], entropy fp32 [...], top_tokens int32
    [..., top], top_logprobs fp32 [..., top])`` for logits bf16, fp16 or fp32 [..., V] and tokens int32 / int64 [...].

    ``logprobs``: the logarithm of each token's probability under softmax(logits / temperature), the whole distribution that
    :func:`sampling_probs` cuts (-inf for a token outside the vocabulary); ``entropy`` of that distribution, in nats;
    ``top`` (up to 64): the tokens of the largest logits, falling, equal ones by index, and their log probabilities.
    NaN counts as -inf, infinite logits share all the probability, and a row of nothing but -inf and NaN has -inf
    throughout and an entropy of 0. ``workspace`` of :func:`token_logprobs_workspace_bytes`, 16-byte aligned, any content, for
    one call at a time, else allocated."""
    what = "token_logprobs"
    dev = _one_device(what, logits, tokens, workspace)
    dt = DEQUANT_DTYPES.get(logits.dtype)
    if dt is None:
        raise TypeError(f"{what}: logits {logits.dtype} (bfloat16, float16 or float32)")
    shape = logits.shape
    top = int(top)
    if len(shape) < 1 or shape[-1] < 1 or not 0 <= top <= min(MOST_ALTERNATIVES, shape[-1]):
        raise ValueError(f"{what}: logits {list(shape)}, top={top} (up to {MOST_ALTERNATIVES} and the vocabulary)")
    t, _, _ = check_sampler(temperature, 0, 1.0)
    _no_autograd(what, logits)
    wide = tokens.dtype is torch.int64
    if not (wide or tokens.dtype is torch.int32) or tokens.shape != shape[:-1]:
        raise ValueError(f"{what}: tokens must be int32 or int64 {list(shape[:-1])}, got {tokens.dtype} {list(tokens.shape)}")
    tokens = tokens.contiguous()
    if logits.is_neg():
        logits = logits.resolve_neg()
    V = shape[-1]
    x = logits if len(shape) == 2 else logits.reshape(-1, V)
    rows, (ld, unit) = x.shape[0], x.stride()
    if (unit != 1 and V > 1) or ld < 0:
        x, ld = x.contiguous(), V
    given = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(given)
    ids = torch.empty((*shape[:-1], top), dtype=torch.int32, device=dev)
    best = torch.empty_like(ids, dtype=torch.float32)
    if rows:
        nbytes = token_logprobs_workspace_bytes(rows, V, top)
        if nbytes == 0:
            raise ValueError(f"{what}: {rows} rows (up to 2^20) of {V} logits (up to 2^28)")
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        elif workspace.nbytes < nbytes or not workspace.is_contiguous() or workspace.data_ptr() % 16:
            raise ValueError(f"{what}: workspace: {nbytes} contiguous bytes, aligned to 16, needed")
        _call_on(dev, "dspark_token_logprobs",
                 _SCORE_ARGS.pack(dt, x.data_ptr(), ld, rows, V, tokens.data_ptr(), wide, top, t, given.data_ptr(), entropy.data_ptr(),
                                  ids.data_ptr(), best.data_ptr(), workspace.data_ptr(), workspace.nbytes))
    return given, entropy, ids, best


# ---------------------------------------------------------------------------- rotary positions, quantized cache rows

ROPE_DTYPES = DEQUANT_DTYPES


def _spans_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors of non-negative strides meet."""
    end = lambda t: t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _no_repeats(what: str, out: torch.Tensor) -> None:
    if 0 in out.stride() and any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{what}: the output is an expanded view ({list(out.shape)}, strides {list(out.stride())})")


def _distinct(what: str, *at: int) -> None:
    """Addresses of what is written, and of what else must not be there: the same rows given twice would be written by
    two workgroups, or read while they are."""
    if len(set(at)) != len(at):
        raise ValueError(f"{what}: the same rows given twice")


def _check_rope_out(name: str, x: torch.Tensor, out: torch.Tensor) -> None:
    _as_stored("rope", out)
    if out.dtype != x.dtype or out.shape != x.shape or out.stride(3) != 1:
        raise ValueError(f"rope: {name} must be {x.dtype} {list(x.shape)} with unit last stride")
    _no_repeats("rope", out)
    if _spans_meet(x, out) and (out.data_ptr() != x.data_ptr() or out.stride() != x.stride()):
        raise ValueError(f"rope: {name} overlaps its input (in place: the same view)")


_ROPE_ARGS = struct.Struct("=25qd5q")
_NO_KEYS = (0,) * 9


def rope(q: torch.Tensor, k: torch.Tensor | None, freqs: torch.Tensor, positions, *, interleaved: bool = False,
         scale: float = 1.0, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Rotary positions of queries [B, Hq, L, D] and keys [B, Hk, L, D] (or None) in one launch ->
    ``(q, k)`` rotated. bf16, fp16 or fp32, any batch / head / row strides, unit stride along D.

    ``freqs`` fp64 [dims / 2] (:func:`dspark_rocm.rope.frequencies`): radians a position of the pairs
    (i, i + dims / 2), or (2i, 2i + 1) when ``interleaved``, of a head's first ``dims`` values, which
    ``scale`` multiplies; the rest is copied. ``positions``: an int (row l stands at ``positions + l``), or
    an int32 / int64 tensor [L] or [B or 1, L or 1] with the position of every row, as tree rows need. The
    angle is reduced in fp64; one rounding to the tensors' type. ``q_out`` / ``k_out``: where to write,
    e.g. a cache's rows, or q and k themselves; elements that nothing else of the call uses (refused where the
    addresses from its first to its last element meet its input's and it is not the same view)."""
    tensor = isinstance(positions, torch.Tensor)
    dev = _one_device("rope", q, k, freqs, q_out, k_out, positions if tensor else None)
    dtype = q.dtype
    dt = ROPE_DTYPES.get(dtype)
    if dt is None or (k is not None and k.dtype is not dtype):
        raise TypeError(f"rope: q {dtype}, k {None if k is None else k.dtype} (one of bfloat16, float16, float32)")
    q_shape, k_shape = q.shape, None if k is None else k.shape
    if len(q_shape) != 4 or (k_shape is not None and len(k_shape) != 4):
        raise ValueError(f"rope: q and k must be [B, H, L, D], got {list(q_shape)} and {None if k is None else list(k_shape)}")
    B, Hq, L, D = q_shape
    Hk = 0
    if k is not None:
        Bk, Hk, Lk, Dk = k_shape
        if Bk != B or Lk != L or Dk != D:
            raise ValueError(f"rope: q {list(q_shape)} and k {list(k_shape)}")
    elif k_out is not None:
        raise ValueError("rope: k_out without k")
    f_shape = freqs.shape
    half = f_shape[0] if len(f_shape) == 1 else 0
    if freqs.dtype is not torch.float64 or not 1 <= half <= min(128, D // 2):
        raise ValueError(f"rope: freqs must be fp64 [dims / 2], dims up to the head dim and 256, got {freqs.dtype} {list(f_shape)}")
    _no_autograd("rope", q, k, freqs, q_out, k_out)
    if freqs.is_neg() or not freqs.is_contiguous():
        freqs = freqs.resolve_neg().contiguous()
    pos, pos64, pb, pl, pos0 = 0, 0, 0, 0, 0
    if tensor:
        pdt, p_shape = positions.dtype, positions.shape
        pos64 = pdt is torch.int64
        if not (pos64 or pdt is torch.int32) or not 1 <= len(p_shape) <= 2:
            raise ValueError(f"rope: positions must be int32 or int64 [L] or [B, L], got {pdt} {list(p_shape)}")
        nb, nl = p_shape if len(p_shape) == 2 else (1, p_shape[0])
        if nl not in (1, L) or nb not in (1, B):
            raise ValueError(f"rope: positions {list(p_shape)} for {B} sequences of {L} rows")
        pos, st = positions.data_ptr(), positions.stride()
        pl = st[-1] if nl > 1 else 0
        pb = st[0] if nb > 1 else 0
    else:
        pos0 = int(positions)
        if abs(pos0) >= 1 << 52:
            raise ValueError(f"rope: position {pos0}")
    s0, s1, s2, unit = q.stride()
    if unit != 1 or q.is_neg():
        q = q.resolve_neg().contiguous()
        s0, s1, s2, _ = q.stride()
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        o0, o1, o2 = Hq * L * D, L * D, D
    else:
        _check_rope_out("q_out", q, q_out)
        o0, o1, o2, _ = q_out.stride()
    at_q, at_qo = q.data_ptr(), q_out.data_ptr()
    keys = _NO_KEYS
    if k is not None:
        k0, k1, k2, unit = k.stride()
        if unit != 1 or k.is_neg():
            k = k.resolve_neg().contiguous()
            k0, k1, k2, _ = k.stride()
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
            ko = (Hk * L * D, L * D, D)
        else:
            _check_rope_out("k_out", k, k_out)
            ko = k_out.stride()[:3]
        if B and L and Hk:
            at_k, at_ko = k.data_ptr(), k_out.data_ptr()
            if Hq and (at_ko == at_qo or at_ko == at_q or at_qo == at_k):
                raise ValueError("rope: the same rows given twice")
            keys = (at_k, at_ko, k0, k1, k2, *ko, Hk)
    if B and L and (Hq or Hk):
        _call_on(dev, "dspark_rope",
                 _ROPE_ARGS.pack(dt, at_q, at_qo, s0, s1, s2, o0, o1, o2, Hq, *keys, B, L, D, 2 * half, bool(interleaved),
                                 freqs.data_ptr(), scale, pos, pos64, pb, pl, pos0))
    return q_out, k_out


KV_CACHE_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_KV_ARGS = struct.Struct("=34q")


def _kv_side(what: str, at: int, strides: tuple, trip, words: torch.Size, groups: tuple, cache_dtype, dual: bool,
             written: bool) -> tuple:
    """The fields of one ``dspark_kv_side``: plain rows at ``at`` and the (words, scales, biases) they belong to (words
    None: its shape is where the sizes came from)."""
    w, s, b = trip
    if w.dtype is not torch.int32:
        _require_packed(w)
    if s.dtype is not cache_dtype or b.dtype is not cache_dtype:
        raise TypeError(f"{what}: scales and biases of {cache_dtype}, {s.dtype} and {b.dtype}")
    if (words is not None and w.shape != words) or s.shape != groups or b.shape != groups:
        raise ValueError(f"{what}: words {list(w.shape)}, scales {list(s.shape)}, biases {list(b.shape)}")
    if s.requires_grad or b.requires_grad or dual:
        _no_autograd(what, s, b)
    if s.is_neg() or b.is_neg():
        _as_stored(what, s, b)
    w0, w1, w2, w3 = w.stride()
    s0, s1, s2, s3 = s.stride()
    b0, b1, b2, b3 = b.stride()
    if w3 != 1 or s0 != b0 or s1 != b1 or s2 != b2 or ((s3 != 1 or b3 != 1) and groups[3] > 1):
        raise ValueError(f"{what}: unit last strides, and shared ones of scales and biases, needed")
    if written and not (w0 and w1 and w2 and s0 and s1 and s2):
        for t in trip:
            _no_repeats(what, t)
    x0, x1, x2, _ = strides
    return at, x0, x1, x2, w.data_ptr(), s.data_ptr(), b.data_ptr(), w0, w1, w2, s0, s1, s2


def _kv_shape(what: str, keys, bits: int, group_size: int):
    """((B, H, T, D), shape of the words, of the scales, type of these) of a triple of cache views."""
    if bits not in KV_BITS or group_size != GROUP:
        raise ValueError(f"{what}: bits={bits} (4 or 8), group_size={group_size} (64)")
    kw, ks, _ = keys
    words = kw.shape
    if len(words) != 4:
        raise ValueError(f"{what}: words must be [B, H, rows, D * bits / 32], got {list(words)}")
    B, H, T, W = words
    D = W * 32 // bits
    if D % GROUP or D == 0:
        raise ValueError(f"{what}: words {list(words)} at {bits} bits")
    cdt = ks.dtype
    if cdt not in KV_CACHE_DTYPES:
        raise TypeError(f"{what}: scales {cdt} (bfloat16 or float16)")
    if 2 * B * H > 65535:
        raise ValueError(f"{what}: {B} x {H} heads (up to 32767)")
    return (B, H, T, D), words, (B, H, T, D // GROUP), cdt


def _kv_rows(t: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """Plain rows as a kernel reads them (a copy where the last stride is not 1 or the memory is negated), their strides."""
    st = t.stride()
    if st[3] != 1 or t.is_neg():
        t = t.resolve_neg().contiguous()
        st = t.stride()
    return t, st


def quantize_kv(keys: torch.Tensor, values: torch.Tensor, k_rows, v_rows, *, bits: int, group_size: int = GROUP) -> None:
    """Quantize ``keys`` / ``values`` [B, H, T, D] (bf16, fp16 or fp32, any strides) into the cache rows
    ``k_rows`` / ``v_rows``: (words int32 [B, H, T, D*bits/32], scales [B, H, T, D/64], biases) views of a
    quantized cache, scales in bf16 or fp16. The values of :func:`dspark_rocm.quant.quantize_rows`, bit for
    bit but for the sign of a zero bias (a group with a NaN gets a NaN scale and bias), both tensors in one launch.
    The six arrays written share no element with each other or with the rows."""
    what = "quantize_kv"
    dev = _one_device(what, keys, values, *k_rows, *v_rows)
    xdt = keys.dtype
    dt = DEQUANT_DTYPES.get(xdt)
    if dt is None or values.dtype != xdt:
        raise TypeError(f"{what}: rows {xdt} and {values.dtype} (one of bfloat16, float16, float32)")
    shape, words, groups, cdt = _kv_shape(what, k_rows, bits, group_size)
    if keys.shape != shape or values.shape != shape:
        raise ValueError(f"{what}: keys {list(keys.shape)}, values {list(values.shape)} for rows {list(shape)}")
    dual = _forward_level()
    if dual or keys.requires_grad or values.requires_grad:
        _no_autograd(what, keys, values)
    keys, k_st = _kv_rows(keys)
    values, v_st = _kv_rows(values)
    args = (dt, KV_CACHE_DTYPES[cdt], *shape, bits, group_size,
            *_kv_side(what, keys.data_ptr(), k_st, k_rows, None, groups, cdt, dual, True),
            *_kv_side(what, values.data_ptr(), v_st, v_rows, words, groups, cdt, dual, True))
    if shape[0] * shape[1] * shape[2]:
        _distinct(what, *args[12:15], *args[25:28])         # words, scales and biases of both
        _call_on(dev, "dspark_kv_quantize", _KV_ARGS.pack(*args))


def dequantize_kv(keys, values, *, bits: int, group_size: int = GROUP, dtype: torch.dtype = torch.float32, out=None):
    """A quantized cache (or rows of it) read back: the triples of :func:`quantize_kv` -> ``(keys, values)``
    [B, H, T, D] of ``dtype``, ``scale * field + bias`` with an fp32 product rounded, then an fp32 sum
    rounded, then rounded to ``dtype``; both tensors in one launch. ``out``: two tensors to write, sharing no
    element with each other or with the cache."""
    what = "dequantize_kv"
    dev = _one_device(what, *keys, *values, *(out or ()))
    dt = DEQUANT_DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"{what}: dtype {dtype} (bfloat16, float16 or float32)")
    shape, words, groups, cdt = _kv_shape(what, keys, bits, group_size)
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=dev)
        v = torch.empty_like(k)
        k_st = v_st = (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)
    else:
        k, v = out
        _no_autograd(what, k, v)
        _as_stored(what, k, v)
        for t in out:
            if t.dtype != dtype or t.shape != shape or t.stride(3) != 1:
                raise ValueError(f"{what}: out must be two {dtype} {list(shape)} with unit last stride")
            _no_repeats(what, t)
        k_st, v_st = k.stride(), v.stride()
        if shape[0] * shape[1] * shape[2]:
            _distinct(what, k.data_ptr(), v.data_ptr())
    dual = _forward_level()
    args = (dt, KV_CACHE_DTYPES[cdt], *shape, bits, group_size,
            *_kv_side(what, k.data_ptr(), k_st, keys, None, groups, cdt, dual, False),
            *_kv_side(what, v.data_ptr(), v_st, values, words, groups, cdt, dual, False))
    if shape[0] * shape[1] * shape[2]:
        _call_on(dev, "dspark_kv_dequantize", _KV_ARGS.pack(*args))
    return k, v


# ---------------------------------------------------------------------------- paged caches of many sequences

PAGE_POSITIONS = (16, 32, 64, 128)
PAGE_CODES, PAGE_SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu     # 8-bit pages: codes, and scales of a page and head


def _pages_parts(pages) -> tuple:
    return tuple(pages) if isinstance(pages, (tuple, list)) else (pages,)


def _both_pages(what: str, k_pages, v_pages, dtype, written: bool) -> tuple[bool, torch.Size, tuple]:
    """(codes?, [pool, Hk, P, D], the fields of the two ``dspark_pages``) of keys and values. Decoding calls this for every
    layer and token: what can go wrong is looked at first, what exactly did afterwards."""
    k, v, ks, vs = k_pages, v_pages, None, None
    if isinstance(k, (tuple, list)):
        k, ks = k
    if isinstance(v, (tuple, list)):
        v, vs = v
    codes = ks is not None
    want = PAGE_CODES if codes else dtype
    if codes != (vs is not None):
        raise TypeError(f"{what}: keys and values in 8 bits, or neither")
    if k.dtype is not want or v.dtype is not want or codes and (ks.dtype is not PAGE_SCALES or vs.dtype is not PAGE_SCALES):
        raise TypeError(f"{what}: pages {k.dtype} and {v.dtype} for rows of {dtype} (8-bit pages are {PAGE_CODES} codes with "
                        f"{PAGE_SCALES} scales)")
    s = k.shape
    if len(s) != 4 or v.shape != s:
        raise ValueError(f"{what}: pages must be [pages, Hk, positions, D], keys and values alike, got {list(s)} and {list(v.shape)}")
    if s[2] not in PAGE_POSITIONS or s[3] not in QUANT_HEAD_DIMS:
        raise ValueError(f"{what}: pages of {s[2]} positions {PAGE_POSITIONS} of {s[3]} values {QUANT_HEAD_DIMS}")
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError(f"{what}: pages need unit stride along their values")
    if k.is_neg() or v.is_neg():
        _as_stored(what, k, v)
    if written and not (k0 and k1 and k2 and v0 and v1 and v2):
        _no_repeats(what, k)
        _no_repeats(what, v)
    if not codes:
        return False, s, (k.data_ptr(), k0, k1, k2, 0, 0, 0, v.data_ptr(), v0, v1, v2, 0, 0, 0)
    if ks.shape != s[:2] or vs.shape != s[:2]:
        raise ValueError(f"{what}: scales must be {list(s[:2])}, got {list(ks.shape)} and {list(vs.shape)}")
    if written:
        _no_repeats(what, ks)
        _no_repeats(what, vs)
    return True, s, (k.data_ptr(), k0, k1, k2, ks.data_ptr(), *ks.stride(), v.data_ptr(), v0, v1, v2, vs.data_ptr(), *vs.stride())


def _sequences(what: str, table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, rows: int) -> tuple:
    """The fields of ``dspark_sequences``, and what has to stay alive for them."""
    if table.dim() != 2 or table.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: table must be int32 [sequences, pages], got {table.dtype} {list(table.shape)}")
    B, W = table.shape
    if B > 4096:
        raise ValueError(f"{what}: {B} sequences (up to 4096)")
    if table.dtype is not torch.int32:
        table = _ints(what, "table", table, table.shape)
    ld, unit = table.stride()
    if unit != 1 and W > 1 or ld < W:
        table = table.contiguous()
        ld = W
    starts, lens = _ints(what, "starts", starts, (B + 1,)), _ints(what, "lens", lens, (B,))
    return (table.data_ptr(), starts.data_ptr(), lens.data_ptr(), ld, B, W, rows), (table, starts, lens)


def _paged_rows(what: str, name: str, t: torch.Tensor, T: int, H: int, D: int, dtype) -> tuple:
    """Rows [T, H, D] as a kernel reads them (a copy where their addresses have no 16 bytes together), their address and
    strides."""
    if t.dtype is not dtype:
        raise TypeError(f"{what}: {name} {t.dtype} beside {dtype}")
    if t.shape != (T, H, D):
        raise ValueError(f"{what}: {name} must be [{T}, {H}, {D}], got {list(t.shape)}")
    if t.is_neg():
        t = t.resolve_neg()
    s0, s1, unit = t.stride()
    at = t.data_ptr()
    if unit != 1 or s0 % 8 or s1 % 8 or at % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        at, s0, s1 = t.data_ptr(), H * D, D
    return t, at, s0, s1


@functools.lru_cache(maxsize=256)
def _lie_apart(ahead: int, size_a: int, a: tuple, size_b: int, b: tuple) -> bool:
    """Whether two views whose spans meet are known to share no byte: ``b`` begins ``ahead`` bytes behind ``a``, each is (count,
    bytes of stride) pairs of elements of ``size`` bytes. So they are where, in steps of some stride of theirs, what
    the others span lies side by side: heads of one row of queries, keys and values, keys and values of one page."""
    for period in {s for n, s in a + b if n > 1 and s}:
        reach = lambda size, dims: size + sum((n - 1) * s for n, s in dims if s % period)
        off = ahead % period
        if reach(size_a, a) <= off and off + reach(size_b, b) <= period:
            return True
    return False


def _span(at: int, size: int, *dims: tuple) -> tuple:
    """Where a view begins and ends, for :func:`_share`."""
    end = at + size
    for n, s in dims:
        end += (n - 1) * s
    return at, end, size, dims


def _share(x: tuple, y: tuple) -> bool:
    return x[0] < y[1] and y[0] < x[1] and not _lie_apart(y[0] - x[0], x[2], x[3], y[2], y[3])


def _page_spans(codes: bool, pool: int, Hk: int, P: int, D: int, f: tuple) -> list:
    """Spans of the parts of ``_both_pages``' fields: keys, values, and their scales."""
    e = 1 if codes else 2
    spans = [_span(f[i], e, (pool, e * f[i + 1]), (Hk, e * f[i + 2]), (P, e * f[i + 3]), (D, e)) for i in (0, 7)]
    return spans + [_span(f[i], 1, (pool, f[i + 1]), (Hk, f[i + 2])) for i in (4, 11)] if codes else spans


def _page_ends(codes: bool, pool: int, Hk: int, P: int, D: int, f: tuple) -> tuple:
    """Where keys, values (and their scales) end."""
    if not codes:
        return (f[0] + 2 * ((pool - 1) * f[1] + (Hk - 1) * f[2] + (P - 1) * f[3] + D),
                f[7] + 2 * ((pool - 1) * f[8] + (Hk - 1) * f[9] + (P - 1) * f[10] + D))
    return (f[0] + (pool - 1) * f[1] + (Hk - 1) * f[2] + (P - 1) * f[3] + D, f[7] + (pool - 1) * f[8] + (Hk - 1) * f[9] + (P - 1) * f[10] + D,
            f[4] + (pool - 1) * f[5] + (Hk - 1) * f[6] + 1, f[11] + (pool - 1) * f[12] + (Hk - 1) * f[13] + 1)


def _meet_pages(at: int, end: int, codes: bool, f: tuple, ends: tuple) -> bool:
    """Whether the bytes from ``at`` to ``end`` meet the spans of the pages."""
    return at < ends[0] and f[0] < end or at < ends[1] and f[7] < end or codes and (at < ends[2] and f[4] < end or at < ends[3] and f[11] < end)


def _side_by_side(ahead: int, wide_a: int, wide_b: int, step: int, size: int) -> bool:
    """Whether, every ``step`` elements, what two views span lies beside each other; ``ahead`` in bytes."""
    off = ahead % (step * size) if step else -1
    return wide_a * size <= off and off + wide_b * size <= step * size


def _overlaps(T: int, D: int, to: tuple, rows: tuple, written: list) -> bool:
    """Whether the pages that an append writes share memory, or the queries' place (``to``: heads, address and strides; none: a new
    one) and them or ``rows``, keys and values alike."""
    if any(_share(x, y) for i, x in enumerate(written) for y in written[i + 1:]):
        return True
    span = lambda heads, at, s0, s1: _span(at, 2, (T, 2 * s0), (heads, 2 * s1), (D, 2))
    return bool(to) and any(_share(span(*to), x) for x in (*(span(*r) for r in rows), *written))


def _no_positions(k_pages, v_pages, table: torch.Tensor):
    """A pool without pages, or a table without room, as the kernels can take it: the rows are there, none of their positions is."""
    def one(pages):
        if isinstance(pages, (tuple, list)):
            return tuple(torch.zeros((1, *t.shape[1:]), dtype=torch.uint8, device=t.device).view(t.dtype) for t in pages)
        return pages.new_zeros((1, *pages.shape[1:]))

    return one(k_pages), one(v_pages), table.new_full((table.shape[0], 1), -1)


_APPEND_ARGS = struct.Struct("=10qd37q")


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages, v_pages, table: torch.Tensor, starts: torch.Tensor,
                 lens: torch.Tensor, *, q: torch.Tensor | None = None, freqs: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
                 q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """A step's rows into their sequences' pages, rotated to their positions on the way, in one launch; returns the
    rotated queries (None without ``q``).

    ``k`` / ``v`` [T, Hk, D] and ``q`` [T, Hq, D], bf16 or fp16, D 64, 128 or 256: the rows of all sequences, one after
    the other: ``starts`` [B + 1] says where each one's begin, ``lens`` [B] how many positions it has with them (both
    int32 on the device), ``table`` int32 [B, pages] in which pages: position p lies in row p % P of page
    ``table[b, p // P]``. ``k_pages`` / ``v_pages`` [pages, Hk, P, D] (P 16, 32, 64 or 128) are of the rows' type, or
    (codes e4m3 [pages, Hk, P, D], scales e8m0 [pages, Hk]): 8 bits with one power of two for each page and head, the least
    that fits the rows new in it and those it held before them, which are shifted to it.

    ``freqs`` fp64 [dims / 2] (:func:`dspark_rocm.rope.frequencies`) rotates the first ``dims`` values of queries and keys as
    :func:`rope` does, ``dims`` a multiple of 16 (interleaved: of 8); None: nothing is rotated. ``positions`` int32 / int64
    [T]: rotate by these instead. Rows of a position that the table, or the pool, does not have are not written; rows
    behind the last sequence's are left out, and ``q_out`` there as it is. A page that is written to belongs to one
    sequence. ``q_out``: where the queries go, e.g. ``q`` itself; else new, with zeros in rows of no sequence. ``q_out`` in other memory
    that is read or written, and pools that share some, are refused, unless a common stride sets them side by side."""
    what = "paged_append"
    tensors = (v, *_pages_parts(k_pages), *_pages_parts(v_pages), table, starts, lens, q, freqs, positions, q_out)
    dev = _one_device(what, k, *tensors)
    dtype = k.dtype
    dt = ATTN_DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"{what}: rows {dtype} (bfloat16 or float16)")
    codes, (pool, Hk, P, D), pages = _both_pages(what, k_pages, v_pages, dtype, True)
    if k.dim() != 3:
        raise ValueError(f"{what}: k must be [rows, {Hk}, {D}], got {list(k.shape)}")
    T = k.shape[0]
    _no_autograd(what, k, v, q, freqs, q_out, *_pages_parts(k_pages), *_pages_parts(v_pages))
    k, *k_at = _paged_rows(what, "k", k, T, Hk, D, dtype)
    v, *v_at = _paged_rows(what, "v", v, T, Hk, D, dtype)
    if not Hk:
        raise ValueError(f"{what}: pages of no heads")
    seqs, keep = _sequences(what, table, starts, lens, T)
    if not (pool and seqs[5]):
        nowhere = _no_positions(k_pages, v_pages, table)
        _, (pool, *_), pages = _both_pages(what, *nowhere[:2], dtype, True)
        seqs, keep = _sequences(what, nowhere[2], starts, lens, T)
    at_f = dims = 0
    if freqs is not None:
        if freqs.dtype is not torch.float64 or freqs.dim() != 1 or not 1 <= freqs.numel() <= D // 2:
            raise ValueError(f"{what}: freqs must be fp64 [dims / 2], dims up to {D}, got {freqs.dtype} {list(freqs.shape)}")
        dims = 2 * freqs.numel()
        if dims % (8 if interleaved else 16):
            raise ValueError(f"{what}: {dims} rotated values (a multiple of 16, interleaved of 8; others: rope, then paged_append)")
        freqs = freqs.resolve_neg().contiguous()
        at_f = freqs.data_ptr()
    at_p = p_st = p64 = at_o = 0
    if positions is not None:
        p64 = positions.dtype is torch.int64
        if not (p64 or positions.dtype is torch.int32) or positions.shape != (T,):
            raise ValueError(f"{what}: positions must be int32 or int64 [{T}], got {positions.dtype} {list(positions.shape)}")
        at_p, p_st = positions.data_ptr(), positions.stride(0)
    q_fields, Hq = (0,) * 7, 0
    if q is not None:
        if q.dim() != 3:
            raise ValueError(f"{what}: q must be [{T}, heads, {D}], got {list(q.shape)}")
        Hq = q.shape[1]
        clear = q_out is None
        if clear:
            q, *q_at = _paged_rows(what, "q", q, T, Hq, D, dtype)
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            o_st = Hq * D, D
        else:
            same = q_out.data_ptr() == q.data_ptr() and q_out.stride() == q.stride()
            if q_out.dtype is not dtype or q_out.shape != q.shape or q_out.stride(2) != 1 or q_out.stride(0) % 8 \
                    or q_out.stride(1) % 8 or q_out.data_ptr() % 16:
                raise ValueError(f"{what}: q_out must be {dtype} {list(q.shape)} with unit last stride, aligned to 16 bytes")
            _as_stored(what, q_out)
            _no_repeats(what, q_out)
            if not same and q.numel() and _spans_meet(q, q_out):
                raise ValueError(f"{what}: q_out overlaps q (in place: the same view)")
            q, *q_at = _paged_rows(what, "q", q, T, Hq, D, dtype)
            o_st = q_out.stride()[:2]
        at_o = q_out.data_ptr()
        q_fields = (*q_at, at_o, *o_st, clear)
    elif q_out is not None:
        raise ValueError(f"{what}: q_out without q")
    if T and seqs[4]:
        # What is written shares no byte with what else is written, and the queries' place none with k and v. (k and v may be
        # rows of the pool in pages that the call does not write, but not from its first page on.) Decoding comes by here for every
        # layer: plain sums first, what they do not settle afterwards.
        (at_ka, sk0, sk1), (at_va, sv0, sv1) = k_at, v_at
        ends = _page_ends(codes, pool, Hk, P, D, pages)
        at_k, at_v = pages[0], pages[7]
        near = at_ka == at_k or at_ka == at_v or at_va == at_k or at_va == at_v
        if not near and at_k < ends[1] and at_v < ends[0]:
            wide, wide_v = ((Hk - 1) * f1 + (P - 1) * f2 + D for f1, f2 in (pages[2:4], pages[9:11]))
            near = pages[1] != pages[8] or not _side_by_side(at_v - at_k, wide, wide_v, pages[1], 1 if codes else 2)
        if codes and not near:
            near = pages[4] < ends[3] and pages[11] < ends[2] and not (
                pages[5] == pages[12] and _side_by_side(pages[11] - pages[4], (Hk - 1) * pages[6] + 1, (Hk - 1) * pages[13] + 1, pages[5], 1))
        placed = Hq and not clear
        if placed and not near:
            o0, o1 = o_st
            wide, wide_k, wide_v = (Hq - 1) * o1 + D, (Hk - 1) * sk1 + D, (Hk - 1) * sv1 + D
            end = at_o + 2 * ((T - 1) * o0 + wide)
            near = at_o < at_ka + 2 * ((T - 1) * sk0 + wide_k) and at_ka < end and not (o0 == sk0 and _side_by_side(at_ka - at_o, wide, wide_k, o0, 2)) \
                or at_o < at_va + 2 * ((T - 1) * sv0 + wide_v) and at_va < end and not (o0 == sv0 and _side_by_side(at_va - at_o, wide, wide_v, o0, 2)) \
                or _meet_pages(at_o, end, codes, pages, ends)
        if near and (at_ka in (at_k, at_v) or at_va in (at_k, at_v) or _overlaps(
                T, D, (Hq, at_o, *o_st) if placed else (), ((Hk, *k_at), (Hk, *v_at)), _page_spans(codes, pool, Hk, P, D, pages))):
            raise ValueError(f"{what}: the same memory given twice (what is written overlaps)")
        _call_on(dev, "dspark_paged_append",
                 _APPEND_ARGS.pack(dt, codes, Hq, Hk, D, P, pool, dims, bool(interleaved), at_f, scale, at_p, p64, p_st, *q_fields,
                                   *k_at, *v_at, *pages, *seqs))
    elif Hq and clear:
        q_out.zero_()
    return q_out


_READ_ARGS = struct.Struct("=24q")


def paged_read(k_pages, v_pages, pages: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16):
    """Pages by id (``pages`` int32 [N] on the device) as dense ``(keys, values)`` [N, Hk, P, D] of ``dtype`` (bf16 or fp16;
    for pages that are not in 8 bits their own): what :func:`paged_append` keeps, the values that 8-bit codes stand for
    rounded once. Zeros for ids that are none of the pool's."""
    what = "paged_read"
    parts = (*_pages_parts(k_pages), *_pages_parts(v_pages))
    dev = _one_device(what, *parts, pages)
    _no_autograd(what, *parts)
    dt = ATTN_DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"{what}: dtype {dtype} (bfloat16 or float16)")
    codes, (pool, Hk, P, D), fields = _both_pages(what, k_pages, v_pages, dtype, False)
    if pages.dim() != 1:
        raise ValueError(f"{what}: pages must be int32 [N], got {list(pages.shape)}")
    ids = _ints(what, "pages", pages, pages.shape)
    N = ids.numel()
    k = torch.empty((N, Hk, P, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if N and Hk and pool:
        _call_on(dev, "dspark_paged_read",
                 _READ_ARGS.pack(dt, codes, Hk, D, P, pool, ids.data_ptr(), N, *fields, k.data_ptr(), v.data_ptr()))
    return (k, v) if pool else (k.zero_(), v.zero_())


@functools.lru_cache(maxsize=256)
def paged_attention_workspace_bytes(sequences: int, hq: int, hk: int, d: int, rows: int, max_rows: int, max_len: int) -> int:
    """Workspace bytes of :func:`paged_attention` (``max_len``: positions of the table's pages); 0 where it refuses the call."""
    return int(_lib.load().dspark_paged_attention_workspace(sequences, hq, hk, d, rows, max_rows, max_len))


_PAGED_ATTN_ARGS = struct.Struct("=10qd29q")


def paged_attention(q: torch.Tensor, k_pages, v_pages, table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, *,
                    scale: float, causal: bool = True, max_rows: int | None = None, max_len: int | None = None,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's rows over their sequences' pages -> [T, Hq, D]: decoded tokens, verify blocks and prompt chunks
    of any lengths together, the sequences, pages and arguments as in :func:`paged_append`, which writes the rows' own keys
    and values first.

    Row i of a sequence's n sees the positions up to its own, ``lens[b] - n + i`` (``causal``), or all ``lens[b]``: an
    encoder's states, kept in pages. fp32 scores and sums; zeros for a row that sees nothing; values that are not finite
    count only where a row sees them. Positions of pages that the pool does not have are not seen. A probability is held to 2^-16 of
    it in bf16 and 2^-20 in fp16 models, and to 2^-11 (an eighth of the output's rounding) where the chunk rows of a bf16 model go
    over 8-bit pages at D 64 and 128: by the call's bounds and the other sequences, a row may take the one or the other.

    ``max_rows`` (rows of one sequence) and ``max_len`` (positions; default: what the table has room for) are the
    host's bounds: positions from ``max_len`` on, rounded up to a page, are not seen (0 says that no sequence has any, and so
    no rows, whatever ``lens``: nothing is done but a new ``out`` cleared); more rows than ``max_rows`` are
    served too, only slower. ``max_rows`` chooses the kernels and the workspace, and is all of the call's rows if it is not given:
    give the step's own, 1 for decoded tokens (32 of them over 8-bit pages take 54 us with it and 62 without). ``out``: rows of no sequence are left as they are there; in a new one they are zeros.
    ``workspace`` of :func:`paged_attention_workspace_bytes`, 16-byte aligned, any content, for one call at a time, else
    allocated."""
    what = "paged_attention"
    parts = (*_pages_parts(k_pages), *_pages_parts(v_pages))
    dev = _one_device(what, q, *parts, table, starts, lens, out, workspace)
    dtype = q.dtype
    dt = ATTN_DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"{what}: q {dtype} (bfloat16 or float16)")
    codes, (pool, Hk, P, D), pages = _both_pages(what, k_pages, v_pages, dtype, False)
    if q.dim() != 3 or q.shape[2] != D or (Hk and q.shape[1] % Hk):
        raise ValueError(f"{what}: q must be [rows, a multiple of {Hk} heads, {D}], got {list(q.shape)}")
    scale = float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"{what}: scale={scale} (positive)")
    T, Hq, _ = q.shape
    _no_autograd(what, q, out, *parts)
    clear = out is None
    if not clear:
        if out.dtype is not dtype or out.shape != q.shape or out.stride(2) != 1 or out.stride(0) % 8 or out.stride(1) % 8 \
                or out.data_ptr() % 16:
            raise ValueError(f"{what}: out must be {dtype} {list(q.shape)} with unit last stride, aligned to 16 bytes")
        _as_stored(what, out)
        _no_repeats(what, out)
        if q.numel() and _spans_meet(q, out):
            raise ValueError(f"{what}: out overlaps q")
        at_o, (o0, o1, _) = out.data_ptr(), out.stride()
        if T and Hq and pool and _meet_pages(at_o, at_o + 2 * ((T - 1) * o0 + (Hq - 1) * o1 + D), codes, pages, _page_ends(codes, pool, Hk, P, D, pages)) \
                and any(_share(_span(at_o, 2, (T, 2 * o0), (Hq, 2 * o1), (D, 2)), x) for x in _page_spans(codes, pool, Hk, P, D, pages)):
            raise ValueError(f"{what}: out overlaps the pages")
    q, *q_at = _paged_rows(what, "q", q, T, Hq, D, dtype)
    if clear:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    seqs, keep = _sequences(what, table, starts, lens, T)
    if not (pool and seqs[5]) and not clear:                     # (a new out is cleared below)
        nowhere, workspace = _no_positions(k_pages, v_pages, table), None
        _, (pool, *_), pages = _both_pages(what, *nowhere[:2], dtype, False)
        seqs, keep = _sequences(what, nowhere[2], starts, lens, T)
    B, W = seqs[4], seqs[5]
    rows = T if max_rows is None else min(int(max_rows), T)
    if max_len is not None:
        W = min(W, -(-int(max_len) // P))
    if rows < 1 and T or W < 0:
        raise ValueError(f"{what}: max_rows={max_rows}, max_len={max_len}")
    if T and Hq:
        if B and W and pool:
            nbytes = paged_attention_workspace_bytes(B, Hq, Hk, D, T, rows, W * P)
            if nbytes == 0:
                raise ValueError(f"{what}: {T} rows of {Hq} / {Hk} heads, {B} sequences of {W} pages: {_lib.last_error()}")
            if workspace is None:
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            elif workspace.nbytes < nbytes or not workspace.is_contiguous() or workspace.data_ptr() % 16:
                raise ValueError(f"{what}: workspace: {nbytes} contiguous bytes, aligned to 16, needed")
            _call_on(dev, "dspark_paged_attention",
                     _PAGED_ATTN_ARGS.pack(dt, codes, Hq, Hk, D, P, pool, bool(causal), clear, rows, scale, *q_at,
                                           out.data_ptr(), *out.stride()[:2], *pages, *seqs[:5], W, T, workspace.data_ptr(),
                                           workspace.nbytes))
        elif clear:
            out.zero_()
    return out
