"""torch-facing wrappers of the libimq kernels.

Every function takes/returns torch tensors on a ROCm device, checks shapes/strides on the host,
and launches on torch's current stream for that device. Outputs are allocated with torch (so
they come from the caching allocator, and from the graph pool under stream capture). Nothing
here synchronizes except the MoE ops' routing-id check, which is skipped under stream capture,
so these calls are capturable into HIP graphs.

These are the product path: they never fall back to a CPU/torch computation. A missing library
raises ``ImqUnavailable``, a rejected call raises ``ImqError``.
"""
from __future__ import annotations

import threading

import torch

from . import _lib
from ._lib import call, dtype_code


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _check_dev(*ts):
    dev = ts[0].device
    if dev.type != "cuda":
        raise ValueError("libimq ops need tensors on a ROCm device")
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"device mismatch: {t.device} vs {dev}")
    return dev


def _rows2d(x: torch.Tensor) -> torch.Tensor:
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    if x.stride(1) != 1 or (x.stride(0) % 8) != 0 or (x.data_ptr() % 16) != 0:
        x = x.contiguous()
    return x


# Workspaces (split-K / K-split partials of the fused linears, MoE intermediates), one per
# (device, stream), their contents need no initialization. A call that uses one holds its lock from
# its first launch to its last: the kernel that writes the partials and the launch that sums them are
# two, and both host paths release the GIL between them, so without the lock two threads on one stream
# could enqueue A's kernel, B's kernel, A's sum. A workspace is never freed once handed out, because a
# HIP graph captured with it (and the native path's cached pointer) keeps its address: when a call needs
# more, the old buffer is retired (kept alive for the life of the process) and one at least twice its
# size takes its place, so at most log2(largest need) buffers are ever retired per stream.
_WS: dict = {}                  # (device index, stream) -> (buffer, lock)
_WS_RETIRED: list = []
_WS_LOCK = threading.RLock()    # of the two containers; re-entrant, as an allocation may run finalizers


def _scratch(dev: torch.device, need: int):
    """The (device, current stream) workspace of at least ``need`` bytes and the lock its users hold."""
    key = (dev.index, _stream(dev))
    ws = _WS.get(key)
    if ws is None or ws[0].numel() < need:
        with _WS_LOCK:
            ws = _WS.get(key)
            if ws is None or ws[0].numel() < need:
                size = need if ws is None else max(need, 2 * ws[0].numel())
                buf = torch.empty(size, dtype=torch.uint8, device=dev)
                ws = _WS.get(key)                # again: a finalizer may have come here meanwhile
                if ws is not None:
                    _WS_RETIRED.append(ws[0])
                ws = _WS[key] = (buf, threading.RLock() if ws is None else ws[1])
    return ws


class _Held:
    """``with _Held(dev, need) as (pointer, bytes)``: the workspace for one call, locked (none for need <= 0)."""

    __slots__ = ("ws",)

    def __init__(self, dev: torch.device, need: int):
        self.ws = _scratch(dev, need) if need > 0 else None

    def __enter__(self):
        if self.ws is None:
            return 0, 0
        self.ws[1].acquire()
        return self.ws[0].data_ptr(), self.ws[0].numel()

    def __exit__(self, *exc):
        if self.ws is not None:
            self.ws[1].release()


def _workspace(dev: torch.device, M: int, N: int, K: int) -> _Held:
    return _Held(dev, int(_lib.lib().imq_linear_workspace_bytes(M, N, K)))


def _scratch_ptr(index: int, need: int):
    """The native path's view of a workspace: (pointer, bytes, lock)."""
    buf, lock = _scratch(torch.device("cuda", index), need)
    return buf.data_ptr(), buf.numel(), lock


# The native host path (csrc/fastcall.cpp): ``_fast_linear(kind, x, q, sz, group, nd)`` and ``_fast_moe(...)``
# return the result of a plain call and None for every other, which then takes the Python path below
# with its conversions and checks. Bound on first use; without the module every call takes the Python path.
_FAST_LOCK = threading.RLock()
_FAST_MODULE: list = []


def _fast_module():
    """The native host path's module, loaded on first use, or None (said once) where it is missing."""
    with _FAST_LOCK:
        if not _FAST_MODULE:
            try:
                _FAST_MODULE.append(_lib.fast(_scratch_ptr))
            except _lib.ImqUnavailable as exc:
                print(f"[imq] native host path unavailable ({exc}) -> Python host path", flush=True)
                _FAST_MODULE.append(None)
        return _FAST_MODULE[0]


def _bind_fast() -> None:
    global _fast_linear, _fast_moe
    with _FAST_LOCK:
        if _fast_linear is not _first_linear:
            return
        m = _fast_module()
        _fast_linear, _fast_moe = (m.linear, m.moe) if m is not None else (lambda *a: None, lambda *a: None)


def _first_linear(*a):
    _bind_fast()
    return _fast_linear(*a)


def _first_moe(*a):
    _bind_fast()
    return _fast_moe(*a)


_fast_linear, _fast_moe = _first_linear, _first_moe


def _capturing(x) -> bool:
    """Whether the current stream of x's device is being captured; torch's own query asks the current device's."""
    index = x.get_device()
    if index < 0:
        return False
    if index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _check_expert_ids(idx: torch.Tensor, E: int) -> None:
    """Refuse routing ids outside [0, E), as the reference's eager experts loop does (its
    ``one_hot(num_classes=E)`` raises). One device-to-host read, so it is skipped while a HIP graph
    is being captured (the kernels then only keep out-of-range ids' loads in bounds)."""
    if idx.numel() == 0 or _capturing(idx):
        return
    lo, hi = (int(v) for v in torch.aminmax(idx))
    if lo < 0 or hi >= E:
        raise ValueError(f"expert ids must lie in [0, {E}); got ids in [{lo}, {hi}]")


def _check_packed(q: torch.Tensor, dt=torch.uint8):
    if q.dtype != dt or q.dim() < 2 or q.stride(-1) != 1:
        raise ValueError(f"packed weight must be {dt} with a unit last stride, got {q.dtype} {tuple(q.stride())}")


# ---------------------------------------------------------------------------------------------
# dequant (bit-exact reference dequant)
# ---------------------------------------------------------------------------------------------
def _dequant_g(fn: str, bits: int, qweight, scale, zero, in_features: int, group_size: int, dtype):
    dev = _check_dev(qweight, scale, zero)
    _check_packed(qweight)
    N = qweight.shape[0]
    out = torch.empty((N, in_features), dtype=dtype, device=dev)
    with torch.cuda.device(dev):
        call(fn, _ptr(qweight), qweight.stride(0), _ptr(scale), scale.stride(0), scale.stride(1),
             dtype_code(scale.dtype), _ptr(zero), zero.stride(0), zero.stride(1), dtype_code(zero.dtype),
             N, in_features, group_size, _ptr(out), out.stride(0), dtype_code(dtype), _stream(dev))
    return out


def dequant_w4(qweight, scale, zero, in_features: int, group_size: int, dtype=torch.bfloat16):
    """QuantLinear4._dequant(dtype) on the GPU (worker_quant.py:638-648), bit-exact."""
    return _dequant_g("imq_dequant_w4", 4, qweight, scale, zero, in_features, group_size, dtype)


def dequant_w2(qweight, scale, zero, in_features: int, group_size: int, dtype=torch.bfloat16):
    """QuantLinear2._dequant(dtype) on the GPU (worker_quant.py:1652-1664), bit-exact."""
    return _dequant_g("imq_dequant_w2", 2, qweight, scale, zero, in_features, group_size, dtype)


def dequant_w8(qweight, scale, dtype):
    """``qweight.to(x_dtype) * scale`` (worker_quant.py:439) with torch's dtype promotion: the
    result dtype is ``torch.promote_types(dtype, scale.dtype)``."""
    dev = _check_dev(qweight, scale)
    _check_packed(qweight, torch.int8)
    res = torch.promote_types(dtype, scale.dtype)
    N, K = qweight.shape
    out = torch.empty((N, K), dtype=res, device=dev)
    with torch.cuda.device(dev):
        call("imq_dequant_w8", _ptr(qweight), qweight.stride(0), _ptr(scale), scale.stride(0),
             dtype_code(scale.dtype), N, K, _ptr(out), out.stride(0), dtype_code(res), _stream(dev))
    return out


# ---------------------------------------------------------------------------------------------
# RTN packers on the device (bit-identical to shard_compile.pack_linear_int4 / int2 / int8)
# ---------------------------------------------------------------------------------------------
def _pack_g(fn: str, bits: int, W, group_size: int):
    dev = _check_dev(W)
    if W.dim() != 2 or W.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"W must be a 2D bf16 / fp16 / fp32 tensor, got {W.dtype} {tuple(W.shape)}")
    if W.stride(1) != 1:
        W = W.contiguous()
    N, in_f = W.shape
    ng = -(-in_f // group_size)
    q = torch.empty((N, ng * group_size * bits // 8), dtype=torch.uint8, device=dev)
    scale = torch.empty((N, ng), dtype=W.dtype, device=dev)
    zero = torch.empty((N, ng), dtype=W.dtype, device=dev)
    with torch.cuda.device(dev):
        call(fn, _ptr(W), W.stride(0), dtype_code(W.dtype), N, in_f, group_size, _ptr(q), q.stride(0),
             _ptr(scale), _ptr(zero), scale.stride(0), _stream(dev))
    return q, scale, zero, in_f


def pack_w4(W, group_size: int = 128):
    """``pack_linear_int4`` on the device: (qweight u8 [N, K_pad/2], scale, zero, in_features)
    (shard_compile.py:74-94)."""
    return _pack_g("imq_pack_w4", 4, W, group_size)


def pack_w2(W, group_size: int = 64):
    """``pack_linear_int2`` on the device: (qweight u8 [N, K_pad/4], scale, zero, in_features)
    (shard_compile.py:50-71)."""
    return _pack_g("imq_pack_w2", 2, W, group_size)


def pack_w8(W):
    """``pack_linear_int8`` on the device: (qweight int8 [N, K], scale [N, 1] in W's dtype)
    (shard_compile.py:170-178)."""
    dev = _check_dev(W)
    if W.dim() != 2 or W.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"W must be a 2D bf16 / fp16 / fp32 tensor, got {W.dtype} {tuple(W.shape)}")
    if W.stride(1) != 1:
        W = W.contiguous()
    N, K = W.shape
    q = torch.empty((N, K), dtype=torch.int8, device=dev)
    scale = torch.empty((N, 1), dtype=W.dtype, device=dev)
    with torch.cuda.device(dev):
        call("imq_pack_w8", _ptr(W), W.stride(0), dtype_code(W.dtype), N, K, _ptr(q), q.stride(0), _ptr(scale),
             scale.stride(0), _stream(dev))
    return q, scale


# ---------------------------------------------------------------------------------------------
# fused dequant linears
# ---------------------------------------------------------------------------------------------
def _linear_g(fn: str, codes_per_byte: int, x, qweight, group_size: int, sz, out=None):
    scale, zero = sz
    dev = _check_dev(x, qweight, scale, zero)
    _check_packed(qweight)
    x = _rows2d(x)
    Kpad = qweight.shape[1] * codes_per_byte
    if x.shape[1] != Kpad:
        x = torch.nn.functional.pad(x, (0, Kpad - x.shape[1])).contiguous()
    M = x.shape[0]
    N = qweight.shape[0]
    ng = Kpad // group_size
    if Kpad % group_size or tuple(scale.shape) != (N, ng) or tuple(zero.shape) != (N, ng):
        raise ValueError(f"scale/zero must be [{N}, {ng}] for K_pad={Kpad}, group={group_size}; "
                         f"got {tuple(scale.shape)} / {tuple(zero.shape)}")
    if out is not None and (tuple(out.shape) != (M, N) or out.dtype != torch.bfloat16 or out.stride(1) != 1):
        raise ValueError("out must be a bf16 [M, N] tensor with unit column stride")
    y = out if out is not None else torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        if fn == "imq_linear_w4":
            # this call's own need (0 for the decode kernels that keep their partials in the
            # workgroup), not the shape-only bound over all formats
            held = _Held(dev, int(_lib.lib().imq_linear_w4_workspace_bytes(
                M, Kpad, N, group_size, qweight.stride(0), x.stride(0), scale.stride(0), scale.stride(1),
                dtype_code(scale.dtype), zero.stride(0), zero.stride(1), dtype_code(zero.dtype))))
        else:
            held = _workspace(dev, M, N, Kpad)
        with held as (ws, wsb):
            call(fn, _ptr(x), x.stride(0), M, Kpad, _ptr(qweight), qweight.stride(0), _ptr(scale), scale.stride(0),
                 scale.stride(1), dtype_code(scale.dtype), _ptr(zero), zero.stride(0), zero.stride(1),
                 dtype_code(zero.dtype), N, group_size, _ptr(y), y.stride(0), ws, wsb, _stream(dev))
    return y


def linear_w4(x, qweight, group_size: int, sz, out=None):
    """``op(x[M,Kpad] bf16, qweight u8[N,Kpad/2], group, (scale, zero)) -> y[M,N] bf16``: the
    signature of the op returned by the reference's _w4a16_triton_op (worker_quant.py:1180-1217)."""
    if out is None and (y := _fast_linear(4, x, qweight, sz, group_size, False)) is not None:
        return y
    return _linear_g("imq_linear_w4", 2, x, qweight, group_size, sz, out)


def linear_w4_tiled(x, qweight_tiled, group_size: int, sz, out=None):
    """``linear_w4`` on int4 weights in the line-tiled layout (``line_tile``): the same results
    bit for bit. ``qweight_tiled`` is the dense u8 [N, Kpad/2] tiled array (N a multiple of 16,
    Kpad of 256, groups of 128); shapes no tiled-layout kernel takes raise ImqError."""
    if out is None and (y := _fast_linear(20, x, qweight_tiled, sz, group_size, False)) is not None:
        return y
    if group_size != 128:
        raise ValueError("line-tiled int4 weights take groups of 128")
    if not qweight_tiled.is_contiguous():
        raise ValueError("the line-tiled weight array must be dense")
    return _linear_g("imq_linear_w4_tiled", 2, x, qweight_tiled, group_size, sz, out)


def linear_w2_tiled(x, qweight_tiled, group_size: int, sz, out=None):
    """``linear_w2`` on int2 weights in the line-tiled layout (``line_tile``): the dense u8
    [N, Kpad/4] tiled array (N a multiple of 16, Kpad of 512, groups of 64)."""
    if out is None and (y := _fast_linear(18, x, qweight_tiled, sz, group_size, False)) is not None:
        return y
    if group_size != 64:
        raise ValueError("line-tiled int2 weights take groups of 64")
    if not qweight_tiled.is_contiguous():
        raise ValueError("the line-tiled weight array must be dense")
    return _linear_g("imq_linear_w2_tiled", 4, x, qweight_tiled, group_size, sz, out)


def _tile_shape_check(N: int, row_bytes: int):
    if N % 16 or row_bytes % 128:
        raise ValueError(f"the line-tiled layout needs N % 16 == 0 and row bytes % 128 == 0, got N={N}, "
                         f"row bytes={row_bytes}")


def line_tile(qweight, out=None):
    """Row-layout packed weight [N, row_bytes] (u8 int4 / int2 codes, or int8) -> the line-tiled
    layout of the same dtype (a new dense array, or ``out``): in 16-row tile t the 2 KiB block of
    line-step l holds, in slot 64 h + s, 16-byte piece 4 (((s >> 3) & 1) ^ h) + (s >> 4) of tile
    row 8 h + (s & 7). No counterpart in the reference."""
    if qweight.dtype == torch.int8:
        return line_tile(qweight.view(torch.uint8), None if out is None else out.view(torch.uint8)).view(torch.int8)
    dev = _check_dev(qweight)
    _check_packed(qweight)
    N, KB = qweight.shape
    _tile_shape_check(N, KB)
    t = out if out is not None else torch.empty((N, KB), dtype=torch.uint8, device=dev)
    if tuple(t.shape) != (N, KB) or t.dtype != torch.uint8 or not t.is_contiguous():
        raise ValueError("out must be a dense u8 array of qweight's shape")
    with torch.cuda.device(dev):
        call("imq_line_tile", _ptr(qweight), qweight.stride(0), N, KB, _ptr(t), _stream(dev))
    return t


def line_untile(qweight_tiled, out=None):
    """Inverse of ``line_tile``: the row-layout [N, row_bytes] array (new, or ``out``)."""
    if qweight_tiled.dtype == torch.int8:
        return line_untile(qweight_tiled.view(torch.uint8),
                           None if out is None else out.view(torch.uint8)).view(torch.int8)
    dev = _check_dev(qweight_tiled)
    _check_packed(qweight_tiled)
    if not qweight_tiled.is_contiguous():
        raise ValueError("the line-tiled weight array must be dense")
    N, KB = qweight_tiled.shape
    _tile_shape_check(N, KB)
    r = out if out is not None else torch.empty((N, KB), dtype=torch.uint8, device=dev)
    if tuple(r.shape) != (N, KB) or r.dtype != torch.uint8 or r.stride(1) != 1:
        raise ValueError("out must be a u8 array of qweight's shape with unit column stride")
    with torch.cuda.device(dev):
        call("imq_line_untile", _ptr(qweight_tiled), N, KB, _ptr(r), r.stride(0), _stream(dev))
    return r


def linear_w8_tiled(x, qweight_tiled, scale, out=None):
    """``linear_w8`` on int8 weights in the line-tiled layout (``line_tile``): the dense int8 [N, K]
    tiled array (N a multiple of 16, K of 128); the same results bit for bit."""
    if out is None and (y := _fast_linear(24, x, qweight_tiled, scale, 0, False)) is not None:
        return y
    dev = _check_dev(x, qweight_tiled, scale)
    _check_packed(qweight_tiled, torch.int8)
    if not qweight_tiled.is_contiguous():
        raise ValueError("the line-tiled weight array must be dense")
    x = _rows2d(x)
    M, K = x.shape
    N = qweight_tiled.shape[0]
    if qweight_tiled.shape[1] != K:
        raise ValueError(f"x has {K} columns, qweight {qweight_tiled.shape[1]}")
    y = out if out is not None else torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        with _workspace(dev, M, N, K) as (ws, wsb):
            call("imq_linear_w8_tiled", _ptr(x), x.stride(0), M, K, _ptr(qweight_tiled), qweight_tiled.stride(0),
                 _ptr(scale), scale.stride(0), dtype_code(scale.dtype), N, _ptr(y), y.stride(0), ws, wsb, _stream(dev))
    return y


def linear_w2(x, qweight, group_size: int, sz, out=None):
    """int2 twin (worker_quant.py:1876-1910): qweight u8 [N, Kpad/4]."""
    if out is None and (y := _fast_linear(2, x, qweight, sz, group_size, False)) is not None:
        return y
    return _linear_g("imq_linear_w2", 4, x, qweight, group_size, sz, out)


def linear_w8(x, qweight, scale, out=None):
    """``op(x, qweight int8[N,K], scale[N,1]) -> y bf16 [M,N]`` (worker_quant.py:1022-1048)."""
    if out is None and (y := _fast_linear(8, x, qweight, scale, 0, False)) is not None:
        return y
    dev = _check_dev(x, qweight, scale)
    _check_packed(qweight, torch.int8)
    x = _rows2d(x)
    M, K = x.shape
    N = qweight.shape[0]
    if qweight.shape[1] != K:
        raise ValueError(f"x has {K} columns, qweight {qweight.shape[1]}")
    y = out if out is not None else torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        with _workspace(dev, M, N, K) as (ws, wsb):
            call("imq_linear_w8", _ptr(x), x.stride(0), M, K, _ptr(qweight), qweight.stride(0), _ptr(scale),
                 scale.stride(0), dtype_code(scale.dtype), N, _ptr(y), y.stride(0), ws, wsb, _stream(dev))
    return y


# Group-wise ops a module may call through the native path itself (worker_quant's forward).
for _op, _kind in ((linear_w4, 4), (linear_w4_tiled, 20), (linear_w2, 2), (linear_w2_tiled, 18)):
    _op.fast_kind = _kind


def linear_nd(op, x, qweight, group_size: int, sz):
    """``op`` over the leading sizes of x (any rank, bf16, its last size the packed K) through the native
    path, or None when the call is not a plain one or ``op`` not one of this module's."""
    kind = getattr(op, "fast_kind", 0)
    return _fast_linear(kind, x, qweight, sz, group_size, True) if kind else None


# ---------------------------------------------------------------------------------------------
# fused MoE experts
# ---------------------------------------------------------------------------------------------
def moe_rows_w4(x, eid, q, scale, zero, group_size: int, in_features: int, *, check_ids: bool = True):
    """``op(x[B,Kin], eid[B], q[E,N,Kpad/2], scale, zero, group, in_features) -> y[B,N] bf16``:
    the op returned by the reference's _w4a16_moe_op (worker_quant.py:1452-1487). Expert ids
    outside [0, E) raise ValueError (``check_ids``; not checked under graph capture)."""
    dev = _check_dev(x, eid, q, scale, zero)
    _check_packed(q)
    if scale.dtype != zero.dtype:
        zero = zero.to(scale.dtype)
    x = _rows2d(x)
    Kpad = q.shape[2] * 2
    if x.shape[1] != Kpad:
        x = torch.nn.functional.pad(x, (0, Kpad - x.shape[1])).contiguous()
    eid = eid.to(torch.int32).contiguous()
    B = x.shape[0]
    E, N = q.shape[0], q.shape[1]
    if check_ids:
        _check_expert_ids(eid, E)
    ng = Kpad // group_size
    if tuple(scale.shape) != (E, N, ng) or tuple(zero.shape) != (E, N, ng) or eid.numel() != B:
        raise ValueError("scale/zero must be [E, N, K_pad/group] and eid [B]")
    y = torch.empty((B, N), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        call("imq_moe_rows_w4", _ptr(x), x.stride(0), B, Kpad, _ptr(eid), E, _ptr(q), q.stride(0), q.stride(1),
             _ptr(scale), scale.stride(0), scale.stride(1), scale.stride(2), _ptr(zero), zero.stride(0),
             zero.stride(1), zero.stride(2), dtype_code(scale.dtype), N, group_size, _ptr(y), y.stride(0),
             _stream(dev))
    return y


def moe_workspace_bytes(T: int, top_k: int, E: int, H: int, I: int, group_size: int) -> int:
    return int(_lib.lib().imq_moe_workspace_bytes(T, top_k, E, H, I, group_size))


_ACT = {"silu_glu": 0, "gptoss": 1}


def moe_experts_w4(hidden, topk_idx, topk_w, gu, dn, group_size: int, workspace=None, *, act: str = "silu_glu",
                   gu_bias=None, dn_bias=None, alpha: float = 1.702, limit: float = 7.0, check_ids: bool = True):
    """One MoE layer's experts forward: ``out[t] = sum_j w[t,j] * (down_e(act(gate_up_e(x_t))) + b_dn[e])``.

    ``gu`` / ``dn`` are (qweight, scale, zero, in_features) of the gate_up [E, 2I, K1/2] and down
    [E, H, K2/2] int4 stacks, K1 / K2 the kernel layout's padded K (any multiple of the group
    >= in_features; columns past in_features carry zero codes and zero scales).

    ``act="silu_glu"``: rows [gate | up], h = silu(gate) * up -- the transformers eager experts
    loop (modeling_olmoe.py:301-325) as fused by worker_quant.py:2167-2191. ``act="gptoss"``:
    rows interleaved (gate 2i, up 2i+1) with per-expert biases ``gu_bias`` [E, 2I] and ``dn_bias``
    [E, H] and gpt-oss's clamped GLU (worker_quant.py:2280-2314).

    Routing ids outside [0, E) raise ValueError, as the reference's eager loop does
    (``check_ids``: one device-to-host read per call, skipped under graph capture). Without a
    ``workspace`` the call uses the cached per-(device, stream) workspace."""
    if not check_ids and workspace is None and act in _ACT:
        y = _fast_moe(hidden, topk_idx, topk_w, gu, dn, group_size, _ACT[act], gu_bias, dn_bias, alpha, limit)
        if y is not None:
            return y
    gq, gs, gz, H = gu
    dq, ds, dz, I = dn
    dev = _check_dev(hidden, topk_idx, topk_w, gq, gs, gz, dq, ds, dz)
    for t in (gq, dq):
        _check_packed(t)
    if act not in _ACT:
        raise ValueError(f"act must be one of {sorted(_ACT)} (got {act!r})")
    T = hidden.shape[0]
    k = topk_idx.shape[1]
    E = gq.shape[0]
    if gq.shape[1] != 2 * I or dq.shape[1] != H:
        raise ValueError("gate_up must be [E, 2I, .] and down [E, H, .]")
    sdt = gs.dtype
    gz = gz if gz.dtype == sdt else gz.to(sdt)
    ds = ds if ds.dtype == sdt else ds.to(sdt)
    dz = dz if dz.dtype == sdt else dz.to(sdt)
    for t in (gs, gz, ds, dz):
        if t.stride(2) != 1:
            raise ValueError("scale/zero need a unit last stride")
    if gs.stride() != gz.stride() or ds.stride() != dz.stride():
        gs, gz = gs.contiguous(), gz.contiguous()
        ds, dz = ds.contiguous(), dz.contiguous()
    bdt = None
    biases = []
    for b, rows in ((gu_bias, 2 * I), (dn_bias, H)):
        if b is not None:
            _check_dev(hidden, b)
            if b.dim() != 2 or b.shape[0] != E or b.shape[1] != rows:
                raise ValueError(f"bias must be [E, {rows}] (got {tuple(b.shape)})")
            if b.stride(1) != 1:
                b = b.contiguous()
            if bdt is not None and b.dtype != bdt:
                b = b.to(bdt)
            bdt = b.dtype
        biases.append(b)
    gb, db = biases
    gK, dK = gq.shape[2] * 2, dq.shape[2] * 2
    x = _rows2d(hidden)
    if x.shape[1] != gK and (x.shape[1] != H or H % 8 or (T > 16 and (H % 64 or gK > 40 * 128))):
        # rows of exactly H columns (H % 8 == 0) are read as zero past H by the decode and line
        # kernels; past 16 tokens the register-B GEMM skips the K steps past H when H is a
        # multiple of its 64-column step (and K within its 40 groups): other rows get one
        # zero-padded copy, cheaper than every pass reading them clamped
        x = torch.nn.functional.pad(x[:, :H], (0, gK - H)).contiguous()
    # int64 ids (torch's top-k) and int32 ids are read by the kernels as they are
    idx = topk_idx if topk_idx.dtype in (torch.int64, torch.int32) else topk_idx.to(torch.int64)
    idx = idx.contiguous()
    if check_ids:
        _check_expert_ids(idx, E)
    w = topk_w.to(torch.bfloat16).contiguous()
    need = moe_workspace_bytes(T, k, E, H, I, group_size)
    own = workspace is not None and workspace.numel() * workspace.element_size() >= need
    out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev), _Held(dev, 0 if own else max(need, 1)) as (ws, wsb):
        if own:
            ws, wsb = _ptr(workspace), workspace.numel() * workspace.element_size()
        call("imq_moe_experts_w4_ex", _ptr(x), x.stride(0), T, H, k, _ptr(idx),
             _lib.IMQ_DT_I64 if idx.dtype == torch.int64 else _lib.IMQ_DT_I32, _ptr(w), E,
             _ptr(gq), gq.stride(0), gq.stride(1), gK, _ptr(gs), _ptr(gz), gs.stride(0), gs.stride(1), I,
             _ptr(dq), dq.stride(0), dq.stride(1), dK, _ptr(ds), _ptr(dz), ds.stride(0), ds.stride(1),
             dtype_code(sdt), group_size,
             _ptr(gb) if gb is not None else None, gb.stride(0) if gb is not None else 0,
             _ptr(db) if db is not None else None, db.stride(0) if db is not None else 0,
             dtype_code(bdt) if bdt is not None else 0, _ACT[act], float(alpha), float(limit),
             _ptr(out), out.stride(0), ws, wsb, _stream(dev))
    return out


# ---------------------------------------------------------------------------------------------
# block-scaled fp8 (e4m3 codes, one fp32 scale per 128 columns of a row or 128 x 128 block of a weight)
# ---------------------------------------------------------------------------------------------
class _HeldOwn:
    """A workspace for one call under graph capture: memory of the graph's own pool, so that graphs captured on one stream
    may be replayed on several without sharing it."""

    __slots__ = ("buf",)

    def __init__(self, dev: torch.device, need: int):
        self.buf = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None

    def __enter__(self):
        return (0, 0) if self.buf is None else (self.buf.data_ptr(), self.buf.numel())

    def __exit__(self, *exc):
        self.buf = None


def _f8_launch(name: str, dev: torch.device, need: int, captured: bool, *args):
    """The entry ``name`` with a workspace of ``need`` bytes. Where that has to be allocated, the call is first put
    without one, which launches nothing: sizes and strides that it refuses must not take memory that is never given back."""
    stream = _stream(dev)
    if need > 0 and (captured or (ws := _WS.get((dev.index, stream))) is None or ws[0].numel() < need):
        rc = getattr(_lib.lib(), name)(*args, None, 0, stream)
        if rc != _lib.IMQ_ERR_SCRATCH:
            raise _lib.ImqError(name, rc, _lib.lib().imq_strerror(rc).decode())
    with (_HeldOwn if captured else _Held)(dev, need) as (ws, wsb):
        call(name, *args, ws, wsb, stream)


class _FastF8:
    """The native host path's fp8 and routing calls; each returns None for a call that is not a plain one."""

    def __init__(self):
        m = _fast_module()
        for name in ("quant_f8", "pack_f8", "linear_f8", "moe_f8", "route"):
            setattr(self, name, getattr(m, name) if m is not None else lambda *a: None)


class _FirstF8:
    def __getattr__(self, name):
        global _fast_f8
        with _FAST_LOCK:
            if _fast_f8 is self:
                _fast_f8 = _FastF8()
        return getattr(_fast_f8, name)


_fast_f8 = _FirstF8()
_F8 = torch.float8_e4m3fn
_F8_BLOCK = 128
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _blocks(n: int) -> int:
    return -(-n // _F8_BLOCK)


def _float_rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """x [.., K] as a 2D bf16 / fp16 / fp32 tensor of unit column stride whose rows do not overlap."""
    if x.dtype not in _FLOATS or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be a bf16 / fp16 / fp32 tensor of at least one column, got {x.dtype} {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _f8_operand(q: torch.Tensor, dim: int, name: str) -> torch.Tensor:
    if q.dtype != _F8 or q.dim() != dim or q.shape[-1] % _F8_BLOCK or q.shape[-1] == 0:
        raise ValueError(f"{name} must be a {dim}D float8_e4m3fn tensor of whole blocks of 128 columns, got {q.dtype} "
                         f"{tuple(q.shape)}")
    if q.stride(-1) != 1 or q.stride(-2) < q.shape[-1] or any(s % 16 for s in q.stride()[:-1]) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)   # a copy also where torch calls it contiguous already
    return q


def _f8_scale(s: torch.Tensor, shape, name: str) -> torch.Tensor:
    if s.dtype != torch.float32 or tuple(s.shape) != tuple(shape):
        raise ValueError(f"{name} must be a float32 tensor of shape {tuple(shape)}, got {s.dtype} {tuple(s.shape)}")
    return s


def _bytes_of(t: torch.Tensor):
    """First byte and end of a non-empty tensor's memory."""
    n = 1 + sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _over(out: torch.Tensor, *inputs) -> bool:
    """Whether ``out`` may share memory with an input that a launch still reads while it writes ``out``."""
    if out.numel() == 0:
        return False
    a, b = _bytes_of(out)
    return any(lo < b and a < hi for lo, hi in (_bytes_of(t) for t in inputs if t is not None and t.numel() > 0))


def quant_f8(x):
    """Rows to block-scaled e4m3: ``(q float8_e4m3fn [M, K_pad], scale fp32 [M, K_pad / 128])``, K_pad = K rounded up to
    128 with zero codes. A block's scale is max(amax|x| / 448, 2^-100), its codes x / scale rounded once to nearest
    even; a block that is not finite has scale NaN. x [.., K] bf16 / fp16 / fp32, its leading sizes flattened. No
    counterpart in the reference."""
    if (r := _fast_f8.quant_f8(x)) is not None:
        return r
    dev = _check_dev(x)
    x = _float_rows(x, "x")
    M, K = x.shape
    nb = _blocks(K)
    q = torch.empty((M, nb * _F8_BLOCK), dtype=_F8, device=dev)
    scale = torch.empty((M, nb), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        call("imq_quant_f8", _ptr(x), x.stride(0), dtype_code(x.dtype), M, K, _ptr(q), nb * _F8_BLOCK, _ptr(scale), nb, 1,
             _stream(dev))
    return q, scale


def pack_f8(W):
    """A weight to block-scaled e4m3: ``(qweight float8_e4m3fn [N, K_pad], scale fp32 [ceil(N / 128), K_pad / 128],
    in_features)``, one scale per 128 x 128 block (``quant_f8``'s rule). W [N, K], or a stack [E, N, K] whose matrices
    are blocked one by one (a gate_up stack [E, 2 I, H] is packed as ``W.view(2 * E, I, H)``, its codes viewed back as
    [E, 2 I, H_pad] and its scales as [E, 2 ceil(I / 128), H_pad / 128]). No counterpart in the reference."""
    if (r := _fast_f8.pack_f8(W)) is not None:
        return r
    dev = _check_dev(W)
    if W.dim() not in (2, 3) or W.dtype not in _FLOATS or W.shape[-1] < 1:
        raise ValueError(f"W must be a 2D or 3D bf16 / fp16 / fp32 tensor, got {W.dtype} {tuple(W.shape)}")
    if W.stride(-1) != 1 or any(s < 0 for s in W.stride()) or (W.shape[-2] > 1 and W.stride(-2) < W.shape[-1]):
        W = W.contiguous()
    lead = tuple(W.shape[:-2])
    E = lead[0] if lead else 1
    N, K = W.shape[-2:]
    nb = _blocks(K)
    q = torch.empty((*lead, N, nb * _F8_BLOCK), dtype=_F8, device=dev)
    scale = torch.empty((*lead, _blocks(N), nb), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        call("imq_pack_f8", _ptr(W), W.stride(0) if lead else 0, W.stride(-2), dtype_code(W.dtype), E, N, K, _ptr(q),
             _ptr(scale), _stream(dev))
    return q, scale, K


def linear_f8(x, qweight, scale, x_scale=None, out=None):
    """``y[M, N] bf16 = x W^T`` of block-scaled e4m3 operands: the products of a block of 128 columns are summed and
    taken times both scales in fp32. ``x`` [.., K] bf16 / fp16 / fp32 is quantized within the call as ``quant_f8`` does
    (K_pad - 128 < K <= K_pad), or handed over quantized (e4m3 [M, K_pad], ``x_scale`` [M, K_pad / 128]). ``qweight``
    e4m3 [N, K_pad], ``scale`` fp32 [ceil(N / 128), K_pad / 128], as ``pack_f8`` gives them. ``out``: where the result
    goes, a bf16 [M, N] tensor; one that lies over an input gets it by a copy at the end. No counterpart in the reference."""
    own = _capturing(x)
    if out is None and not own and (y := _fast_f8.linear_f8(x, qweight, scale, x_scale)) is not None:
        return y
    dev = _check_dev(x, qweight, scale, x_scale)
    qweight = _f8_operand(qweight, 2, "qweight")
    N, Kpad = qweight.shape
    nb = Kpad // _F8_BLOCK
    scale = _f8_scale(scale, (_blocks(N), nb), "scale")
    if x_scale is not None:
        x = _f8_operand(x, 2, "x (with x_scale)")
        code, sm, sb = _lib.IMQ_DT_F8, x_scale.stride(0) if x_scale.dim() else 0, x_scale.stride(-1) if x_scale.dim() else 0
        _f8_scale(x_scale, (x.shape[0], nb), "x_scale")
    else:
        x = _float_rows(x, "x")
        code, sm, sb = dtype_code(x.dtype), 0, 0
    M, K = x.shape
    if _blocks(K) != nb or (x_scale is not None and K != Kpad):
        raise ValueError(f"x has {K} columns, qweight {Kpad}")
    if out is not None and (tuple(out.shape) != (M, N) or out.dtype != torch.bfloat16 or out.stride(1) != 1 or
                            (M > 1 and out.stride(0) < N) or out.device != dev):
        raise ValueError("out must be a bf16 [M, N] tensor with unit column stride")
    y = out if out is not None and not _over(out, x, qweight, scale, x_scale) else \
        torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        _f8_launch("imq_linear_f8", dev, int(_lib.lib().imq_linear_f8_workspace_bytes(M, N, Kpad, code)), own, _ptr(x),
                   x.stride(0), code, M, K, _ptr(x_scale) if x_scale is not None else None, sm, sb, _ptr(qweight),
                   qweight.stride(0), _ptr(scale), scale.stride(0), scale.stride(1), N, Kpad, _ptr(y), y.stride(0))
        if out is not None and y is not out:
            out.copy_(y)
    return y if out is None else out


def moe_f8_workspace_bytes(T: int, top_k: int, E: int, H: int, I: int) -> int:
    return int(_lib.lib().imq_moe_f8_workspace_bytes(T, top_k, E, H, I))


def moe_experts_f8(hidden, topk_idx, topk_w, gu, dn, workspace=None, *, check_ids: bool = True):
    """One MoE layer's experts forward on block-scaled e4m3 weights: ``out[t] = sum_j w[t,j] * down_e(silu(g) * u)``,
    ``[g | u] = gate_up_e(x_t)``, every projection as ``linear_f8`` (the hidden rows and h quantized within the call).

    ``gu`` / ``dn`` are (qweight, scale, in_features): gate_up e4m3 [E, 2I, H_pad] (rows [gate | up]) with scales
    [E, 2 ceil(I/128), H_pad/128] (gate's blocks, then up's), down e4m3 [E, H, I_pad] with scales
    [E, ceil(H/128), I_pad/128]; see ``pack_f8``. ``hidden`` [T, H] bf16 / fp16 / fp32, ``topk_idx`` [T, k] integers,
    ``topk_w`` [T, k] floats (``moe_route``'s outputs as they are); out bf16 [T, H].

    Routing ids outside [0, E) raise ValueError (``check_ids``: one device-to-host read per call, skipped under graph
    capture; unchecked ones count as expert 0). Without a ``workspace`` the call uses the cached per-(device, stream)
    workspace, under graph capture memory of the graph's own pool."""
    captured = _capturing(hidden)
    if not check_ids and workspace is None and not captured and \
            (y := _fast_f8.moe_f8(hidden, topk_idx, topk_w, gu, dn)) is not None:
        return y
    gq, gs, H = gu
    dq, ds, I = dn
    dev = _check_dev(hidden, topk_idx, topk_w, gq, gs, dq, ds, workspace)
    gq, dq = _f8_operand(gq, 3, "gate_up"), _f8_operand(dq, 3, "down")
    E = gq.shape[0]
    hb, ib = _blocks(H), _blocks(I)
    if tuple(gq.shape) != (E, 2 * I, hb * _F8_BLOCK) or tuple(dq.shape) != (E, H, ib * _F8_BLOCK):
        raise ValueError(f"gate_up must be [E, 2 * {I}, {hb * _F8_BLOCK}] and down [E, {H}, {ib * _F8_BLOCK}], got "
                         f"{tuple(gq.shape)} and {tuple(dq.shape)}")
    gs = _f8_scale(gs, (E, 2 * ib, hb), "gate_up scales")
    ds = _f8_scale(ds, (E, hb, ib), "down scales")
    gs = gs if gs.stride(2) == 1 else gs.contiguous()
    ds = ds if ds.stride(2) == 1 else ds.contiguous()
    x = _float_rows(hidden, "hidden")
    T = x.shape[0]
    if x.shape[1] != H:
        raise ValueError(f"hidden must be [T, {H}], got {tuple(hidden.shape)}")
    if topk_idx.dim() != 2 or topk_idx.shape[0] != T or topk_idx.shape[1] < 1 or topk_w.shape != topk_idx.shape:
        raise ValueError(f"topk_idx and topk_w must be [{T}, k], got {tuple(topk_idx.shape)} and {tuple(topk_w.shape)}")
    if topk_idx.is_floating_point() or topk_idx.dtype == torch.bool or topk_w.dtype not in _FLOATS:
        raise ValueError(f"topk_idx must be integers and topk_w bf16 / fp16 / fp32, got {topk_idx.dtype} and {topk_w.dtype}")
    idx = topk_idx if topk_idx.dtype in (torch.int64, torch.int32) else topk_idx.to(torch.int64)
    idx, w = idx.contiguous(), topk_w.contiguous()
    k = idx.shape[1]
    if check_ids:
        _check_expert_ids(idx, E)
    need = moe_f8_workspace_bytes(T, k, E, H, I)
    own = workspace is not None and workspace.is_contiguous() and workspace.data_ptr() % 16 == 0 and \
        workspace.numel() * workspace.element_size() >= need
    out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    args = (_ptr(x), x.stride(0), dtype_code(x.dtype), T, H, k, _ptr(idx),
            _lib.IMQ_DT_I64 if idx.dtype == torch.int64 else _lib.IMQ_DT_I32, _ptr(w), dtype_code(w.dtype), E,
            _ptr(gq), gq.stride(0), gq.stride(1), _ptr(gs), gs.stride(0), gs.stride(1), I, _ptr(dq), dq.stride(0),
            dq.stride(1), _ptr(ds), ds.stride(0), ds.stride(1), _ptr(out), H)
    with torch.cuda.device(dev):
        if own:
            call("imq_moe_experts_f8", *args, _ptr(workspace), workspace.numel() * workspace.element_size(), _stream(dev))
        else:
            _f8_launch("imq_moe_experts_f8", dev, need, captured, *args)
    return out


# ---------------------------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------------------------
_SCORE = {"softmax": _lib.IMQ_SCORE_SOFTMAX, "sigmoid": _lib.IMQ_SCORE_SIGMOID}


def moe_route(logits, top_k: int, *, score: str = "softmax", bias=None, n_group: int = 1, topk_group: int = 1,
              group_top: int = 2, renorm: bool = True, route_scale: float = 1.0, dtype=torch.float32):
    """A MoE layer's router from the gate's logits [T, E]: ``(weights [T, k] of dtype, ids int64 [T, k])``, what
    ``moe_experts_w4`` and ``moe_experts_f8`` take.

    ``score``: "softmax" over the row, or "sigmoid". ``bias`` fp32 [E] is added to the scores to choose by, and not
    to the weights. With ``n_group`` > 1 only the ``topk_group`` groups (runs of E / n_group experts) with the
    largest sums of their ``group_top`` (1 or 2) largest choices stay in. ids come in falling order of choice, ties to
    the lower id, as the exact choices order them; an expert whose logit is NaN or -inf, or whose bias is, is out:
    it is named only where fewer than k are in, with weight 0. ``renorm`` divides the k scores by their sum;
    ``route_scale`` multiplies them. Up to 1024 experts, 64 groups and a ``top_k`` of 64 (more: ImqError).

    Serves the routers in front of the reference's experts forwards (softmax and top-k in torch:
    worker_quant.py:2131-2248, 2280-2314)."""
    if dtype is torch.float32 and (r := _fast_f8.route(logits, top_k, _SCORE.get(score, -1), bias, n_group, topk_group, group_top,
                                                       renorm, route_scale)) is not None:
        return r
    dev = _check_dev(logits, bias)
    if logits.dim() != 2 or logits.dtype not in _FLOATS:
        raise ValueError(f"logits must be a bf16 / fp16 / fp32 [T, E] tensor, got {logits.dtype} {tuple(logits.shape)}")
    if score not in _SCORE:
        raise ValueError(f"score must be one of {sorted(_SCORE)} (got {score!r})")
    T, E = logits.shape
    if not 1 <= top_k <= E:
        raise ValueError(f"top_k must lie in [1, {E}] (got {top_k})")
    if n_group < 1 or E % n_group or not 1 <= topk_group <= n_group or group_top not in (1, 2):
        raise ValueError(f"n_group must divide {E} experts, topk_group lie in [1, n_group] and group_top be 1 or 2 (got "
                         f"{n_group}, {topk_group}, {group_top})")
    if n_group > 1 and (E // n_group < group_top or topk_group * (E // n_group) < top_k):
        raise ValueError(f"{topk_group} groups of {E // n_group} experts cannot give {top_k} experts by the {group_top} best "
                         "of each")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (E,)):
        raise ValueError(f"bias must be a float32 [{E}] tensor, got {bias.dtype} {tuple(bias.shape)}")
    code = dtype_code(dtype)
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    w = torch.empty((T, top_k), dtype=dtype, device=dev)
    ids = torch.empty((T, top_k), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        call("imq_moe_route", _ptr(logits), logits.stride(0), dtype_code(logits.dtype), T, E, top_k,
             _ptr(bias) if bias is not None else None, _SCORE[score], n_group, topk_group, group_top, int(bool(renorm)),
             float(route_scale), _ptr(w), code, _ptr(ids), _stream(dev))
    return w, ids
