"""PyTorch operator over the C ABI: ``torch.ops.afb.bf16_aintb_gemm``.

The reference has no framework binding (its driver ``bfAintBGemm/bfAintBGemm.cc:36-217`` is a stand-alone
executable); this is the thin layer an inference stack would call instead.  It computes nothing itself: the
tensors' device pointers go into ``afb_gemm_args`` and ``afb_gemm_launch`` runs on torch's current stream, so
the call is stream-ordered with the surrounding torch work and can be captured into a CUDA graph
(``DecodeGraph`` does that for the launch-bound small-M case).  There is no CPU path: a CPU tensor raises.

    out = torch.ops.afb.bf16_aintb_gemm(a, b, scale, bits, group_size, offset_binary, flags=0)

    a      bf16 [M, K], contiguous
    b      int8 [N, K] (bits = 8) or uint8 [N, K / 2] (bits = 4, low nibble = even k), contiguous
    scale  fp32 or bf16; [N] (group_size = 0) or [N, K / group_size]
    flags  AFB_FLAG_* bits passed through to afb_gemm_args.flags (e.g. FLAG_PDL for back-to-back decode GEMMs on constant
           weights, FLAG_GROUP_EXACT for the two-term group-scale mode); default 0
    out    bf16 [M, N]
"""
import torch

from .capi import (ACT_NONE, ACT_SILU, ENC_OFFSET, ENC_TWOS, FLAG_PDL, LAYOUT_COL, LAYOUT_COL_PACKED, MOE_MAX_EXPERTS, MOE_MAX_TOP_K, SCALE_BF16,
                   SCALE_F32, AfbError, load)

_LIB_NAME = "afb::bf16_aintb_gemm"


def _check(a, b, scale, bits, group_size):
    if bits not in (4, 8):
        raise ValueError("bits must be 4 or 8")
    if a.dtype != torch.bfloat16 or a.dim() != 2:
        raise ValueError("a must be a bf16 [M, K] tensor")
    if b.dim() != 2 or b.dtype not in (torch.int8, torch.uint8):
        raise ValueError("b must be an int8 / uint8 [N, K * bits / 8] tensor")
    k = a.shape[1]
    if b.shape[1] * (8 // bits) != k:
        raise ValueError(f"b holds {b.shape[1] * (8 // bits)} weights per channel, a has K = {k}")
    n = b.shape[0]
    if scale.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("scale must be fp32 or bf16")
    if group_size == 0:
        if scale.numel() != n:
            raise ValueError("per-channel scale must have N elements")
    elif group_size < 0 or k % group_size or scale.numel() != n * (k // group_size):
        raise ValueError("per-group scale must be [N, K / group_size]")
    return a.shape[0], n, k


@torch.library.custom_op(_LIB_NAME, mutates_args=(), device_types="cuda")
def bf16_aintb_gemm(a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, bits: int, group_size: int,
                    offset_binary: bool, flags: int = 0) -> torch.Tensor:
    m, n, k = _check(a, b, scale, bits, group_size)
    if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous()):
        raise ValueError("a, b and scale must be contiguous")
    dev = a.device.index if a.device.index is not None else torch.cuda.current_device()
    if dev != torch.cuda.current_device():   # the guard costs a microsecond or two: only where there is a device to come back to
        with torch.cuda.device(dev):
            return _launch(dev, a, b, scale, m, n, k, bits, group_size, offset_binary, flags)
    return _launch(dev, a, b, scale, m, n, k, bits, group_size, offset_binary, flags)


def _launch(dev, a, b, scale, m, n, k, bits, group_size, offset_binary, flags):
    lib = load()
    lib.init(dev)
    out = torch.empty((m, n), device=a.device, dtype=torch.bfloat16)
    args = lib.make_args(out, a, b, scale, m, n, k, bits=bits, group=group_size,
                         encoding=ENC_OFFSET if offset_binary else ENC_TWOS,
                         scale_dtype=SCALE_BF16 if scale.dtype == torch.bfloat16 else SCALE_F32, flags=flags)
    lib.gemm_launch(args, torch.cuda.current_stream(dev).cuda_stream)
    return out


@bf16_aintb_gemm.register_fake
def _(a, b, scale, bits, group_size, offset_binary, flags=0):
    m, n, _ = _check(a, b, scale, bits, group_size)
    return a.new_empty((m, n), dtype=torch.bfloat16)


class DecodeGraph:
    """One small-M GEMM captured in a CUDA graph: ``replay()`` costs one graph launch instead of a Python call into the
    library per GEMM (a decode GEMM runs for microseconds, less than the host needs to issue it).  The input tensors are
    the graph's fixed buffers: copy new activations into ``self.a`` and read ``self.out`` after ``replay()``."""

    def __init__(self, a, b, scale, bits=8, group_size=0, offset_binary=False, weights_constant=False):
        """weights_constant: promise that b and scale are not written while the graph is in use; the GEMM is then launched with
        programmatic dependent launch (FLAG_PDL) and overlaps the kernel before it in the graph's stream."""
        if a.shape[0] > 16:
            raise AfbError(-4, "DecodeGraph is for M <= 16", "")
        self.a, self.b, self.scale = a, b, scale
        flags = FLAG_PDL if weights_constant else 0
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):   # the first call of a kernel sets its attributes: do it outside the capture
            torch.ops.afb.bf16_aintb_gemm(a, b, scale, bits, group_size, offset_binary, flags)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = torch.ops.afb.bf16_aintb_gemm(a, b, scale, bits, group_size, offset_binary, flags)

    def replay(self):
        self.graph.replay()
        return self.out


# ---- a mixture-of-experts layer --------------------------------------------------------------------------------------------------------
#
#     weights, ids, offsets, row_pair, pair_row = torch.ops.afb.moe_route(logits, top_k, renormalize)
#     h = torch.ops.afb.expert_gemm(x, w1, s1, None, offsets, row_pair, top_k, bits, group_size, offset_binary, packed, True)   # silu(gate) * up
#     y = torch.ops.afb.expert_gemm(h, w2, s2, None, offsets, None, 1, bits, group_size, offset_binary, packed, False)
#     out = torch.ops.afb.moe_combine(y, weights, pair_row, residual)
#
# include/afb_capi.h says what each computes.  Weights are [experts, N, K * bits / 8], scales [experts, N] or [experts, N, K / group_size],
# zero-points (optional) uint8 of the scales' shape.  No host synchronisation; zero tokens are taken.  The form of a product is AFB_VARIANT_AUTO's choice.

def _on(t, name, device, dtypes, dim=None):
    if t.device != device or t.dtype not in dtypes or (dim is not None and t.dim() != dim):
        raise ValueError(f"{name} must be a {'/'.join(str(d).split('.')[-1] for d in dtypes)} tensor{'' if dim is None else f' of {dim} dimensions'} on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _run(device, call):
    """call(library, stream) on the tensors' device."""
    dev = device.index if device.index is not None else torch.cuda.current_device()
    lib = load()
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            lib.init(dev)
            return call(lib, torch.cuda.current_stream(dev).cuda_stream)
    lib.init(dev)
    return call(lib, torch.cuda.current_stream(dev).cuda_stream)


def _route_shapes(logits, top_k):
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.shape[1] == 0:
        raise ValueError("logits must be an fp32 or bf16 [tokens, experts] tensor")
    tokens, experts = logits.shape
    if not 1 <= top_k <= min(experts, MOE_MAX_TOP_K) or experts > MOE_MAX_EXPERTS:
        raise ValueError(f"1 <= top_k <= min(experts, {MOE_MAX_TOP_K}) and experts <= {MOE_MAX_EXPERTS}")
    i32 = torch.int32
    return (logits.new_empty((tokens, top_k), dtype=torch.float32), logits.new_empty((tokens, top_k), dtype=i32), logits.new_empty((experts + 1,), dtype=i32),
            logits.new_empty((tokens * top_k,), dtype=i32), logits.new_empty((tokens, top_k), dtype=i32))


@torch.library.custom_op("afb::moe_route", mutates_args=(), device_types="cuda")
def moe_route(logits: torch.Tensor, top_k: int, renormalize: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    weights, ids, offsets, row_pair, pair_row = out = _route_shapes(logits, top_k)
    tokens, experts = logits.shape
    if logits.stride(1) != 1 or (tokens > 1 and logits.stride(0) < experts):
        raise ValueError("logits: rows of consecutive experts that do not overlap")

    def call(lib, stream):
        room = lib.moe_route_workspace(tokens, experts)
        work = logits.new_empty((room,), dtype=torch.uint8) if room else None
        lib.moe_route_launch(lib.make_moe_route_args(logits, ids, weights, offsets, row_pair, pair_row, tokens=tokens, experts=experts, top_k=top_k,
                                                     ld_logits=logits.stride(0) if tokens > 1 else experts, logits_f32=logits.dtype == torch.float32,
                                                     renormalize=renormalize, workspace=work, workspace_bytes=room), stream)
    _run(logits.device, call)
    return out


@moe_route.register_fake
def _(logits, top_k, renormalize=True):
    return _route_shapes(logits, top_k)


def _expert_shapes(a, b, scale, zero, offsets, row_pair, top_k, bits, group_size, gated):
    if bits not in (4, 8):
        raise ValueError("bits must be 4 or 8")
    if a.dtype != torch.bfloat16 or a.dim() != 2:
        raise ValueError("a must be a bf16 [rows, K] tensor")
    k = a.shape[1]
    if b.dim() != 3 or b.dtype not in (torch.int8, torch.uint8) or b.shape[2] * (8 // bits) != k:
        raise ValueError("b must be an int8 / uint8 [experts, N, K * bits / 8] tensor")
    experts, n = b.shape[:2]
    if gated and n % 2:
        raise ValueError("gated: N counts gate and up rows in turn")
    want = (experts, n) if group_size == 0 else (experts, n, k // group_size) if group_size > 0 and k % group_size == 0 else None
    for name, t, dtypes in (("scale", scale, (torch.float32, torch.bfloat16)), ("zero", zero, (torch.uint8, torch.int8))):
        if t is not None and (tuple(t.shape) != want or t.dtype not in dtypes):
            raise ValueError(f"{name} must be [experts, N] (group_size = 0) or [experts, N, K / group_size]")
    if offsets.dtype != torch.int32 or offsets.shape != (experts + 1,):
        raise ValueError("offsets must be int32 [experts + 1]")
    if row_pair is not None and (row_pair.dtype != torch.int32 or row_pair.dim() != 1):
        raise ValueError("row_pair must be int32 [rows]")
    if top_k < 1 or (row_pair is None and top_k != 1):
        raise ValueError("top_k divides row_pair; without one it is 1")
    return a.new_empty((a.shape[0] if row_pair is None else row_pair.shape[0], n // 2 if gated else n))


@torch.library.custom_op("afb::expert_gemm", mutates_args=(), device_types="cuda")
def expert_gemm(a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, offsets: torch.Tensor, row_pair: torch.Tensor | None,
                top_k: int, bits: int, group_size: int, offset_binary: bool, packed: bool = False, gated: bool = False) -> torch.Tensor:
    """The products grouped by expert; gated: silu(gate) * up of interleaved rows.  Rows behind offsets[experts] are not written."""
    out = _expert_shapes(a, b, scale, zero, offsets, row_pair, top_k, bits, group_size, gated)
    for name, t in (("a", a), ("b", b), ("scale", scale), ("zero", zero), ("offsets", offsets), ("row_pair", row_pair)):
        if t is not None:
            _on(t, name, a.device, (t.dtype,))
    experts, n = b.shape[:2]

    def call(lib, stream):
        gemm = lib.make_args(out, a, b, scale, out.shape[0], n, a.shape[1], ldc=out.shape[1], bits=bits, group=group_size, zero=zero,
                             layout=LAYOUT_COL_PACKED if packed else LAYOUT_COL, encoding=ENC_OFFSET if offset_binary else ENC_TWOS,
                             scale_dtype=SCALE_BF16 if scale.dtype == torch.bfloat16 else SCALE_F32)
        lib.expert_gemm_launch(lib.make_expert_gemm_args(gemm, offsets, experts=experts, row_pair=row_pair, top_k=top_k, a_rows=a.shape[0], gated=gated,
                                                         activation=ACT_SILU if gated else ACT_NONE), stream)
    _run(a.device, call)
    return out


@expert_gemm.register_fake
def _(a, b, scale, zero, offsets, row_pair, top_k, bits, group_size, offset_binary, packed=False, gated=False):
    return _expert_shapes(a, b, scale, zero, offsets, row_pair, top_k, bits, group_size, gated)


def _combine_shapes(y, weights, pair_row, residual):
    if y.dtype != torch.bfloat16 or y.dim() != 2 or y.shape[1] == 0:
        raise ValueError("y must be a bf16 [rows, N] tensor")
    if weights.dtype != torch.float32 or pair_row.dtype != torch.int32 or weights.dim() != 2 or weights.shape != pair_row.shape or weights.shape[1] == 0:
        raise ValueError("weights (fp32) and pair_row (int32) must be [tokens, top_k]")
    out = y.new_empty((weights.shape[0], y.shape[1]))
    if residual is not None and (residual.dtype != torch.bfloat16 or residual.shape != out.shape):
        raise ValueError("residual must be bf16 [tokens, N]")
    return out


@torch.library.custom_op("afb::moe_combine", mutates_args=(), device_types="cuda")
def moe_combine(y: torch.Tensor, weights: torch.Tensor, pair_row: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """sum over the picks of weight * the expert's answer, plus the residual."""
    out = _combine_shapes(y, weights, pair_row, residual)
    for name, t in (("y", y), ("weights", weights), ("pair_row", pair_row), ("residual", residual)):
        if t is not None:
            _on(t, name, y.device, (t.dtype,))

    def call(lib, stream):
        lib.moe_combine_launch(lib.make_moe_combine_args(out, y, weights, pair_row, tokens=out.shape[0], top_k=weights.shape[1], rows=y.shape[0],
                                                         n=y.shape[1], residual=residual), stream)
    _run(y.device, call)
    return out


@moe_combine.register_fake
def _(y, weights, pair_row, residual=None):
    return _combine_shapes(y, weights, pair_row, residual)


def moe_mlp(x, logits, w1, s1, w2, s2, top_k, bits=8, group_size=0, offset_binary=False, packed=False, renormalize=True, zero1=None, zero2=None, residual=None):
    """A gated mixture-of-experts MLP on quantised weights: x bf16 [tokens, K], router logits [tokens, experts], w1 [experts, 2 F, K] with gate and
    up rows in turn (afb_prepack_gated lays them out), w2 [experts, K, F].  bf16 [tokens, K], plus the residual."""
    weights, _, offsets, row_pair, pair_row = torch.ops.afb.moe_route(logits, top_k, renormalize)
    h = torch.ops.afb.expert_gemm(x, w1, s1, zero1, offsets, row_pair, top_k, bits, group_size, offset_binary, packed, True)
    y = torch.ops.afb.expert_gemm(h, w2, s2, zero2, offsets, None, 1, bits, group_size, offset_binary, packed, False)
    return torch.ops.afb.moe_combine(y, weights, pair_row, residual)
