"""Operators of one encoder layer on torch CUDA tensors: rotary positions, attention with capped, biased and
masked scores, row quantisation and the matrix product in 8-bit integers.

The two towers run their own fused forms of these (``backend``). The operators here are for layers of other
forms -- interleaved or partly rotated heads, stretched positions, capped scores, distance biases, document and
prefix masks, weights held in 8 bits. Each call launches the library's kernels on the current torch stream of
its tensors' device and returns without waiting; results are new tensors unless ``out`` is given. A tensor of
the wrong type, shape, stride or device, and what the library refuses, raises :class:`lib.Eg2Error`.

Results carry no gradient history, whatever ``requires_grad`` of the inputs says; outputs must not overlap inputs, except where it is said.
A bounded device wait that ran out is not raised by the call: after synchronising, ``eg2_device_status`` tells.
A tensor that is used on another stream than the one it was made on is kept alive and ordered by the caller,
as for any torch operation.
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np
import torch

from . import lib as L

_MASKED = struct.Struct("@iPPPPPqqqqPPqqiiiiiiffiiPPPPPi0P")  # eg2_masked_attention
assert _MASKED.size == C.sizeof(L.MaskedAttention)
KINDS = {torch.bfloat16: L.EG2_BF16, torch.float32: L.EG2_F32}
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
I8_MAX_K = 131072
_INT = 2**31 - 1  # what the C call's int holds


def _bad(msg: str):
    raise L.Eg2Error(-1, msg)


try:  # the stream's handle without the Stream object around it (2 us a call)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _stream(first, *rest) -> int:
    """The stream to launch on, after checking that all tensors are on one CUDA device, the current one."""
    index = first.get_device()
    for t in rest:
        if t.get_device() != index:
            _bad(f"tensors must be on one CUDA device (got {[str(x.device) for x in (first, *rest)]})")
    if index < 0:
        _bad("the tensors must be on a CUDA device")
    if index != torch.cuda.current_device():
        _bad(f"the tensors' device cuda:{index} is not the current one")
    return _raw_stream(index)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise L.Eg2Error(rc, f"{what}: the library refused the call" if rc == -1 else f"{what} failed")


def _heads(t, name: str, kind=None):
    """Row stride of a [rows, heads, channels] tensor whose heads and channels are contiguous."""
    if t.dim() != 3 or t.dtype not in KINDS or (kind is not None and t.dtype != kind):
        _bad(f"{name}: expected a [rows, heads, channels] tensor of {kind or 'bf16 or f32'}, got {tuple(t.shape)} {t.dtype}")
    rows, heads, hd = t.shape
    if heads * hd > _INT:
        _bad(f"{name}: {heads} heads of {hd} channels are 2^31 or more")
    row, head, ch = t.stride()
    if ch == 1 and head == hd and row >= heads * hd:
        return row
    if rows and heads and hd and ((ch != 1 and hd > 1) or (head != hd and heads > 1) or (row < heads * hd and rows > 1)):
        _bad(f"{name}: the heads and channels of a row must be contiguous (strides {t.stride()})")
    return row if rows > 1 else max(row, heads * hd)


def _ints(t, name: str, n: int):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _bad(f"{name}: expected {n} contiguous int32, got {tuple(t.shape)} {t.dtype}")


def _floats(t, name: str, *shape):
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
        _bad(f"{name}: expected contiguous f32 {shape}, got {tuple(t.shape)} {t.dtype}")


# ---- rotary positions ---------------------------------------------------------------------------------
def rotary_steps(rot_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_len: float = 0.0) -> tuple[np.ndarray, float]:
    """Angle per position of each of the ``rot_dim / 2`` pairs, in 2^-64 turns (uint64), and the magnitude to
    pass to :func:`rotary` (``eg2_rotary_steps``; needs no GPU). ``torch.from_numpy(steps.view(np.int64)).cuda()``
    is the device array that :func:`rotary` takes."""
    if scaling not in SCALINGS:
        _bad(f"unknown scaling {scaling!r}: one of {', '.join(SCALINGS)}")
    if int(rot_dim) > _INT:
        _bad(f"rot_dim {rot_dim} is 2^31 or more")
    steps = np.zeros(max(1, int(rot_dim) // 2), np.uint64)
    m = C.c_float()
    _check(L.load().eg2_rotary_steps(int(rot_dim), float(theta), SCALINGS[scaling], float(factor), float(original_len),
                                     steps.ctypes.data_as(C.POINTER(C.c_uint64)), C.byref(m)), "rotary_steps")
    return steps, m.value


def rotary(q, k, pos, steps, *, layout: str = "half", rot_dim: int | None = None, magnitude: float = 1.0,
           inverse: bool = False, out=None):
    """Rotate ``q [rows, nh, hd]`` and ``k [rows, nkv, hd]`` (``k`` may be None) by ``pos`` (int32 ``[rows]``) times
    ``steps`` (:func:`rotary_steps`, int64 on the device); returns ``(q', k')``. ``out=(q', k')`` receives the result,
    and may be the inputs. ``inverse`` turns back by the same angles: the gradient of the forward call."""
    kind = q.dtype
    ldq = _heads(q, "q")
    rows, nh, hd = q.shape
    rot = hd if rot_dim is None else int(rot_dim)
    if layout not in LAYOUTS:
        _bad(f"unknown layout {layout!r}: one of {', '.join(LAYOUTS)}")
    if rot <= 0 or rot > hd or rot % 2:
        _bad(f"rot_dim {rot} must be even and at most the head size {hd}")
    _ints(pos, "pos", rows)
    if steps.dtype != torch.int64 or tuple(steps.shape) != (rot // 2,) or not steps.is_contiguous():
        _bad(f"steps: expected {rot // 2} contiguous int64, got {tuple(steps.shape)} {steps.dtype}")
    nkv, ldk = 0, 0
    if k is not None:
        ldk = _heads(k, "k", kind)
        nkv = k.shape[1]
        if k.shape[0] != rows or k.shape[2] != hd:
            _bad(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if out is None:
        qo = torch.empty(rows, nh, hd, dtype=kind, device=q.device)
        ko = None if k is None else torch.empty(rows, nkv, hd, dtype=kind, device=q.device)
        ldqo, ldko = nh * hd, nkv * hd
    else:
        qo, ko = out
        ldqo = _heads(qo, "out q", kind)
        ldko = 0
        if qo.shape != q.shape or (ko is None) != (k is None):
            _bad("out does not match the inputs")
        if ko is not None:
            ldko = _heads(ko, "out k", kind)
            if ko.shape != k.shape:
                _bad("out does not match the inputs")
    stream = _stream(q, pos, steps, qo) if k is None else _stream(q, k, pos, steps, qo, ko)
    if rows:
        _check(L.load().eg2_rotary(KINDS[kind], LAYOUTS[layout], 1 if inverse else 0, q.data_ptr(), ldq, nh,
                                   0 if k is None else k.data_ptr(), ldk, nkv, qo.data_ptr(), ldqo,
                                   0 if k is None else ko.data_ptr(), ldko, pos.data_ptr(), rows, hd, rot,
                                   steps.data_ptr(), magnitude, stream), "rotary")
    return qo, ko


# ---- attention ------------------------------------------------------------------------------------------
def attention_masked(q, k, v, q_off, k_off, max_q: int, max_k: int, *, scale: float = 1.0, softcap: float = 0.0,
                     window: int = -1, causal: bool = False, prefix_len=None, q_doc=None, k_doc=None, slopes=None,
                     dist_bias=None, out=None, return_lse: bool = False):
    """Attention over packed sequences (``eg2_attention_masked``): ``q [q_rows, nh, hd]``, ``k`` / ``v``
    ``[k_rows, nkv, hd]``; sequence ``b`` has queries ``q_off[b] .. q_off[b + 1]`` and keys ``k_off[b] .. k_off[b + 1]``
    (int32 on the device), at most ``max_q`` / ``max_k`` of them, its queries standing at its last places.

    Scores: ``scale * q.k``, capped to ``softcap * tanh(. / softcap)``, minus ``slopes[h] * |j - i|``, plus
    ``dist_bias[h, clamp(j - i, -R, R) + R]`` (``[nh, 2 R + 1]``). Query ``i`` sees key ``j`` within ``window`` places
    (< 0: any), with ``causal`` only ``j <= i`` or ``j < prefix_len[b]``, and only where ``q_doc`` and ``k_doc`` (int32 per
    row) agree, and not where its bias is -inf. A query that sees nothing gets zeros (log-sum -inf). Returns ``out`` like
    ``q``, with ``return_lse`` also the log-sums ``[q_rows, nh]``; rows of no sequence, or past ``max_q`` in theirs, are left as they
    are in memory."""
    kind = q.dtype
    ldq, ldk, ldv = _heads(q, "q"), _heads(k, "k", kind), _heads(v, "v", kind)
    q_rows, nh, hd = q.shape
    k_rows, nkv, _ = k.shape
    if k.shape != v.shape or k.shape[2] != hd or not nkv or nh % nkv:
        _bad(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    n_seq = q_off.shape[0] - 1 if q_off.dim() == 1 else -1
    if n_seq < 0:
        _bad("q_off: expected n_seq + 1 offsets")
    _ints(q_off, "q_off", n_seq + 1)
    _ints(k_off, "k_off", n_seq + 1)
    tensors = [q, k, v, q_off, k_off]
    if prefix_len is not None:
        if not causal:
            _bad("prefix_len needs causal")
        _ints(prefix_len, "prefix_len", n_seq)
        tensors.append(prefix_len)
    if (q_doc is None) != (k_doc is None):
        _bad("q_doc and k_doc go together")
    if q_doc is not None:
        _ints(q_doc, "q_doc", q_rows)
        _ints(k_doc, "k_doc", k_rows)
        tensors += [q_doc, k_doc]
    if slopes is not None:
        _floats(slopes, "slopes", nh)
        tensors.append(slopes)
    radius = 0
    if dist_bias is not None:
        if dist_bias.dim() != 2 or dist_bias.shape[1] % 2 == 0:
            _bad(f"dist_bias: expected [nh, 2 R + 1], got {tuple(dist_bias.shape)}")
        _floats(dist_bias, "dist_bias", nh, dist_bias.shape[1])
        radius = dist_bias.shape[1] // 2
        tensors.append(dist_bias)
    if out is None:
        out = torch.empty(q_rows, nh, hd, dtype=kind, device=q.device)
        ldo = nh * hd
    else:
        ldo = _heads(out, "out", kind)
        if out.shape != q.shape:
            _bad("out does not match q")
        tensors.append(out)
    stream = _stream(*tensors)
    lse = torch.empty(q_rows, nh, dtype=torch.float32, device=q.device) if return_lse else None

    def ptr(t):
        return 0 if t is None else t.data_ptr()

    try:
        a = _MASKED.pack(KINDS[kind], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(lse), ldq, ldk, ldv, ldo,
                         q_off.data_ptr(), k_off.data_ptr(), q_rows, k_rows, n_seq, int(max_q), int(max_k), nh, nkv, hd, scale, softcap,
                         int(window), 1 if causal else 0, ptr(prefix_len), ptr(q_doc), ptr(k_doc), ptr(slopes), ptr(dist_bias), radius)
    except (struct.error, OverflowError) as e:
        _bad(f"attention_masked: a number does not fit 32 bits (max_q {max_q}, max_k {max_k}, window {window}, scale {scale}, "
             f"softcap {softcap}): {e}")
    lib = L.load()
    need = lib.eg2_attention_masked_workspace(a)
    if need < 0:
        _check(int(need), "attention_masked")
    # From torch's allocator on this stream, so calls on several streams do not share it.
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _check(lib.eg2_attention_masked(a, ptr(work), need, stream), "attention_masked")
    return (out, lse) if return_lse else out


# ---- matrix product in 8-bit integers ---------------------------------------------------------------------
def quantize_rows(x):
    """``x [rows, k]`` (bf16 or f32) as whole numbers of -127 .. 127 and one scale per row: ``(q, scale)`` with
    ``q * scale[:, None]`` within half a step of ``x`` (``eg2_quantize_rows``). The rows of ``q`` start at multiples of
    16 bytes, as :func:`gemm_i8` wants them."""
    if x.dim() != 2 or x.dtype not in KINDS or (x.shape[1] > 1 and x.stride(1) != 1):
        _bad(f"x: expected [rows, k] of bf16 or f32 with contiguous rows, got {tuple(x.shape)} {x.dtype}")
    rows, k = x.shape
    if k == 0 or k > _INT:
        _bad(f"x has {k} columns: none, or 2^31 or more")
    ldx = x.stride(0) if rows > 1 else max(x.stride(0), k)
    if ldx < k:
        _bad(f"x: the rows overlap (strides {x.stride()})")
    ld = (k + 15) // 16 * 16
    q = torch.empty(rows, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    stream = _stream(x)
    if rows:
        _check(L.load().eg2_quantize_rows(KINDS[x.dtype], x.data_ptr(), ldx, q.data_ptr(), ld, scale.data_ptr(), rows, k,
                                          stream), "quantize_rows")
    return (q if ld == k else q[:, :k]), scale


def _i8(t, name: str):
    if t.dim() != 2 or t.dtype != torch.int8 or (t.shape[1] > 1 and t.stride(1) != 1):
        _bad(f"{name}: expected int8 [rows, k] with contiguous rows, got {tuple(t.shape)} {t.dtype}")
    ld = t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16  # of one row it says nothing
    if ld % 16 or t.data_ptr() % 16 or ld < t.shape[1]:
        _bad(f"{name}: rows must start at multiples of 16 bytes (row stride {ld})")
    return ld


def gemm_i8(a, a_scale, w, w_scale, *, bias=None, out_dtype=torch.bfloat16, out=None):
    """``(a @ w.T) * a_scale[:, None] * w_scale + bias`` for int8 ``a [m, k]`` and ``w [n, k]``, the sums exact
    (``eg2_gemm_i8``); ``[m, n]`` in ``out_dtype`` (bf16 or f32). ``w`` may come from :func:`quantize_rows` of the weight:
    one scale per output channel."""
    lda, ldw = _i8(a, "a"), _i8(w, "w")
    (m, k), n = a.shape, w.shape[0]
    if w.shape[1] != k or k == 0 or k > I8_MAX_K:
        _bad(f"a {tuple(a.shape)} and w {tuple(w.shape)} do not match, or more than {I8_MAX_K} columns")
    if n > _INT:
        _bad(f"w has {n} rows, 2^31 or more")
    _floats(a_scale, "a_scale", m)
    _floats(w_scale, "w_scale", n)
    if out is None:
        if out_dtype not in KINDS:
            _bad(f"out_dtype {out_dtype}: bf16 or f32")
        out = torch.empty(m, n, dtype=out_dtype, device=a.device)
        ldc = n
    else:
        if tuple(out.shape) != (m, n) or out.dtype not in KINDS or (n > 1 and out.stride(1) != 1):
            _bad(f"out: expected [{m}, {n}] of bf16 or f32 with contiguous rows")
        ldc = out.stride(0) if m > 1 else max(out.stride(0), n)
    if bias is not None:
        _floats(bias, "bias", n)
        stream = _stream(a, a_scale, w, w_scale, out, bias)
    else:
        stream = _stream(a, a_scale, w, w_scale, out)
    if m and n:
        _check(L.load().eg2_gemm_i8(a.data_ptr(), lda, a_scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(),
                                    0 if bias is None else bias.data_ptr(), out.data_ptr(), ldc, m, n, k,
                                    1 if out.dtype == torch.float32 else 0, stream), "gemm_i8")
    return out
