"""Torch-facing host layer over the C ABI: the quantized linear of raceline's engine.

Mirrors what Engine::encode_linear does for one QTensor (src/engine.mm:832-906): pick
the kernel for the row count, bind the activations, the packed weight and the output,
and run it with ACCUM for the residual writers. Tensors are torch CUDA tensors (HBM
plumbing only); every computation runs in libraceline_amd.so.

Weights arrive in one of the reference's layouts (the MLX u32 layout of the BASELINE
configs and tools/convert.py:82-89, or the blocked q4a layout of .rlm files,
tools/convert.py:92-117) and are packed once, on the device, into the layout the kernels
stream (see include/rlq.h); the dequantized value of every weight is unchanged.
"""

from __future__ import annotations

import functools
import threading
from dataclasses import dataclass, field

import torch

from . import lib

GROUP = 64
F16, BF16 = 0, 1
KERNEL_AUTO, KERNEL_GEMV, KERNEL_GEMM = 0, 1, 2
GEMV_MAX_M = 8


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# The current stream's handle without a Stream object around it: torch.cuda.current_stream()
# took 2.7 of the 10.4 us of a one-token linear's call, this pair 0.2.
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None or _current_device is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_current_device())


def scale_code(dtype: torch.dtype) -> int:
    if dtype == torch.float16:
        return F16
    if dtype == torch.bfloat16:
        return BF16
    raise ValueError(f"scales must be float16 or bfloat16, not {dtype}")


def packed_bytes(K: int, N: int) -> int:
    return int(lib.load().rlq_packed_affine_bytes(K, N))


@dataclass
class PackedWeight:
    """A 4-bit affine matrix [N][K] in the packed device layout, with the dtype of its
    16-bit scales and biases. Like the reference's QTensor (src/model_file.h:44-55) it
    may name the row ranges of stacked parts."""
    packed: torch.Tensor            # uint8, rlq_packed_affine_bytes(K, N) bytes
    K: int
    N: int
    scale_dtype: torch.dtype = torch.float16
    parts: dict = field(default_factory=dict)

    def __post_init__(self):
        if self.packed.dtype != torch.uint8 or not self.packed.is_contiguous():
            raise TypeError("packed weight must be a contiguous uint8 tensor")
        if self.packed.numel() < packed_bytes(self.K, self.N):
            raise ValueError("packed buffer is smaller than the layout needs")

    @property
    def code(self) -> int:
        return scale_code(self.scale_dtype)


def _check_mlx(w: torch.Tensor, s: torch.Tensor, b: torch.Tensor):
    if w.dtype not in (torch.int32, torch.uint32) or w.dim() != 2:
        raise TypeError("codes must be 32-bit words [N][K/8]")
    N, K8 = w.shape
    if s.shape != (N, K8 * 8 // GROUP) or b.shape != s.shape:
        raise ValueError(f"scales/biases {tuple(s.shape)} do not match codes {tuple(w.shape)}")
    if s.dtype != b.dtype:
        raise TypeError("scales and biases must share a dtype")
    for t in (w, s, b):
        if not t.is_contiguous():
            raise ValueError("weight tensors must be contiguous")
    return N, K8 * 8


def pack_affine(w: torch.Tensor, s: torch.Tensor, b: torch.Tensor, stream=None) -> PackedWeight:
    """MLX layout (codes [N][K/8] 32-bit words, scales and biases [N][K/64]) -> PackedWeight."""
    N, K = _check_mlx(w, s, b)
    out = torch.empty(packed_bytes(K, N), dtype=torch.uint8, device=w.device)
    lib.call("rlq_pack_affine", _ptr(w), _ptr(s), _ptr(b), K, N, _ptr(out), _stream(stream))
    return PackedWeight(out, K, N, s.dtype)


def pack_blocked(w_blk: torch.Tensor, s_blk: torch.Tensor, b_blk: torch.Tensor, K: int, n_pad: int, row0: int,
                 rows: int, scale_dtype: torch.dtype = torch.bfloat16, stream=None) -> PackedWeight:
    """Rows [row0, row0 + rows) of a blocked q4a tensor of a .rlm file (already in device
    memory) -> PackedWeight."""
    out = torch.empty(packed_bytes(K, rows), dtype=torch.uint8, device=w_blk.device)
    lib.call("rlq_pack_affine_blocked", _ptr(w_blk), _ptr(s_blk), _ptr(b_blk), K, n_pad, row0, rows, _ptr(out),
             _stream(stream))
    return PackedWeight(out, K, rows, scale_dtype)


def repack_blocked(w_blk: torch.Tensor, s_blk: torch.Tensor, b_blk: torch.Tensor, K: int, n_pad: int,
                   row0: int, rows: int, scale_dtype: torch.dtype = torch.bfloat16, stream=None):
    """Blocked q4a rows -> MLX layout tensors (w int32 [rows][K/8], s, b [rows][K/64])."""
    dev = w_blk.device
    w = torch.empty((rows, K // 8), dtype=torch.int32, device=dev)
    s = torch.empty((rows, K // GROUP), dtype=scale_dtype, device=dev)
    b = torch.empty((rows, K // GROUP), dtype=scale_dtype, device=dev)
    lib.call("rlq_repack_blocked", _ptr(w_blk), _ptr(s_blk), _ptr(b_blk), K, n_pad, row0, rows, _ptr(w), _ptr(s),
             _ptr(b), _stream(stream))
    return w, s, b


BOOKS = {"int15": 1, "int16": 2, "fp4": 3}   # native codebooks (include/rlq.h RLQ_BOOK_*)


@dataclass
class NativeWeight:
    """A native 4-bit matrix [N][K]: codebook codes in the packed tile layout (no
    scale/bias section) and one fp32 scale per row. The column scale belongs to the
    producer of the activations (it is folded into x before the product)."""
    packed: torch.Tensor     # uint8, rlq_packed_codes_bytes(K, N)
    s_row: torch.Tensor      # float32 [N]
    K: int
    N: int
    book: str

    @property
    def code(self) -> int:
        return BOOKS[self.book]


def _native_rows(s_row, N, book):
    if book not in BOOKS:
        raise ValueError(f"unknown codebook {book!r}")
    if s_row.dtype != torch.float32 or s_row.dim() != 1 or s_row.numel() < N or not s_row.is_contiguous():
        raise ValueError("s_row must be a contiguous float32 vector of >= N row scales")


def pack_native(w: torch.Tensor, s_row: torch.Tensor, book: str, stream=None) -> NativeWeight:
    """Row-major codes (32-bit words [N][K/8], element k at bits 4*(k%8)) -> NativeWeight."""
    if w.dtype not in (torch.int32, torch.uint32) or w.dim() != 2 or not w.is_contiguous():
        raise TypeError("codes must be contiguous 32-bit words [N][K/8]")
    N, K = w.shape[0], w.shape[1] * 8
    _native_rows(s_row, N, book)
    out = torch.empty(int(lib.load().rlq_packed_codes_bytes(K, N)), dtype=torch.uint8, device=w.device)
    lib.call("rlq_pack_codes", _ptr(w), K, N, _ptr(out), _stream(stream))
    return NativeWeight(out, s_row[:N], K, N, book)


def pack_native_blocked(w_blk: torch.Tensor, s_pad: torch.Tensor, K: int, n_pad: int, row0: int, rows: int, book: str,
                        stream=None) -> NativeWeight:
    """Rows [row0, row0 + rows) of a blocked q4n tensor (with its padded row scales) -> NativeWeight."""
    _native_rows(s_pad, row0 + rows, book)
    out = torch.empty(int(lib.load().rlq_packed_codes_bytes(K, rows)), dtype=torch.uint8, device=w_blk.device)
    lib.call("rlq_pack_native_blocked", _ptr(w_blk), K, n_pad, row0, rows, _ptr(out), _stream(stream))
    return NativeWeight(out, s_pad[row0:row0 + rows].contiguous(), K, rows, book)


def linear_native(x: torch.Tensor, nw: NativeWeight, out: torch.Tensor | None = None, accum: bool = False,
                  kernel: int = KERNEL_AUTO, stream=None) -> torch.Tensor:
    """out[m][n] (+)= s[n] * sum_k x[m][k] * L[q[n][k]] for fp16 x (column scale already applied)."""
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be a row-major float16 matrix")
    M, K, N = x.shape[0], nw.K, nw.N
    if x.shape[1] < K:
        raise ValueError(f"x has {x.shape[1]} columns, the weight needs {K}")
    if out is None:
        if accum:
            raise ValueError("accum needs an output to add into")
        out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    if out.dtype != torch.float32 or out.stride(1) != 1 or out.shape[0] < M or out.shape[1] < N:
        raise ValueError("out must be a row-major float32 [M][>=N] matrix")
    nbytes = workspace_bytes(M, K, N)
    ws = _WS.get(x.device, nbytes)
    lib.call("rlq_linear_native_kernel", kernel, _ptr(x), x.stride(0), M, K, N, _ptr(nw.packed), _ptr(nw.s_row),
             nw.code, _ptr(out), out.stride(0), 1 if accum else 0, _ptr(ws), 0 if ws is None else ws.numel(),
             _stream(stream))
    return out


def linear_native_raw(x: torch.Tensor, nw: NativeWeight, out: torch.Tensor | None = None,
                      kernel_stream=None) -> torch.Tensor:
    """out[m][n] = sum_k x[m][k] * L[q[n][k]]: the native product without the row scale
    (rlq_linear_native_raw; int15 and fp4 only)."""
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < nw.K:
        raise ValueError("x must be a row-major float16 [M][>= K] matrix")
    M, K, N = x.shape[0], nw.K, nw.N
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    ws = _WS.get(x.device, workspace_bytes(M, K, N))
    lib.call("rlq_linear_native_raw", _ptr(x), x.stride(0), M, K, N, _ptr(nw.packed), nw.code, _ptr(out),
             out.stride(0), _ptr(ws), 0 if ws is None else ws.numel(), _stream(kernel_stream))
    return out


@dataclass
class DenseWeight:
    """A half-precision matrix [N][K] in MFMA operand order (rlq_pack_f16)."""
    packed: torch.Tensor
    K: int
    N: int


def pack_f16(w: torch.Tensor, stream=None) -> DenseWeight:
    if w.dtype != torch.float16 or w.dim() != 2 or not w.is_contiguous():
        raise TypeError("w must be a contiguous float16 [N][K] matrix")
    N, K = w.shape
    out = torch.empty(int(lib.load().rlq_packed_f16_bytes(K, N)), dtype=torch.uint8, device=w.device)
    lib.call("rlq_pack_f16", _ptr(w), K, N, _ptr(out), _stream(stream))
    return DenseWeight(out, K, N)


def pack_f16_blocked(w_blk: torch.Tensor, K: int, n_pad: int, row0: int, rows: int, stream=None) -> DenseWeight:
    out = torch.empty(int(lib.load().rlq_packed_f16_bytes(K, rows)), dtype=torch.uint8, device=w_blk.device)
    lib.call("rlq_pack_f16_blocked", _ptr(w_blk), K, n_pad, row0, rows, _ptr(out), _stream(stream))
    return DenseWeight(out, K, rows)


def linear_f16(x: torch.Tensor, dw: DenseWeight, out: torch.Tensor | None = None, accum: bool = False,
               stream=None) -> torch.Tensor:
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < dw.K:
        raise ValueError("x must be a row-major float16 [M][>= K] matrix")
    M = x.shape[0]
    if out is None:
        if accum:
            raise ValueError("accum needs an output to add into")
        out = torch.empty((M, dw.N), dtype=torch.float32, device=x.device)
    lib.call("rlq_linear_f16", _ptr(x), x.stride(0), M, dw.K, dw.N, _ptr(dw.packed), _ptr(out), out.stride(0),
             1 if accum else 0, _stream(stream))
    return out


class _Workspaces:
    """One scratch buffer per device, grown on demand, zero-filled when allocated (the
    decode kernel keeps its split counters at the start of the linear workspace and leaves
    them zero after every call; nothing else is kept between calls). Calls that use it
    must not overlap on two streams of one device."""

    def __init__(self):
        self._bufs = {}
        self._lock = threading.Lock()

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor | None:
        if nbytes == 0:
            return None
        key = device.index if device.index is not None else torch.cuda.current_device()
        with self._lock:
            buf = self._bufs.get(key)
            if buf is None or buf.numel() < nbytes:
                buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
                self._bufs[key] = buf
            return buf


_WS = _Workspaces()


def workspace_bytes(M: int, K: int, N: int) -> int:
    return int(lib.load().rlq_linear_workspace_bytes(M, K, N))


def linear(x: torch.Tensor, pw: PackedWeight, out: torch.Tensor | None = None, accum: bool = False,
           kernel: int = KERNEL_AUTO, stream=None) -> torch.Tensor:
    """out[m][n] (+)= sum_k x[m][k] * W[n][k] for fp16 x [M][>=K] (row stride x.stride(0))."""
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be a row-major float16 matrix")
    M, K, N = x.shape[0], pw.K, pw.N
    if x.shape[1] < K:
        raise ValueError(f"x has {x.shape[1]} columns, the weight needs {K}")
    if out is None:
        if accum:
            raise ValueError("accum needs an output to add into")
        out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    if out.dtype != torch.float32 or out.stride(1) != 1 or out.shape[0] < M or out.shape[1] < N:
        raise ValueError("out must be a row-major float32 [M][>=N] matrix")
    nbytes = workspace_bytes(M, K, N)
    ws = _WS.get(x.device, nbytes)
    lib.call("rlq_linear_affine_kernel", kernel, _ptr(x), x.stride(0), M, K, N, _ptr(pw.packed), pw.code,
             _ptr(out), out.stride(0), 1 if accum else 0, _ptr(ws), 0 if ws is None else ws.numel(),
             _stream(stream))
    return out


def group_sums(x: torch.Tensor, K: int | None = None, stream=None) -> torch.Tensor:
    K = x.shape[1] if K is None else K
    out = torch.empty((x.shape[0], K // GROUP), dtype=torch.float32, device=x.device)
    lib.call("rlq_group_sums", _ptr(x), x.stride(0), x.shape[0], K, _ptr(out), _stream(stream))
    return out


def dequant(pw: PackedWeight, stream=None) -> torch.Tensor:
    out = torch.empty((pw.N, pw.K), dtype=torch.float32, device=pw.packed.device)
    lib.call("rlq_dequant_affine", _ptr(pw.packed), pw.code, pw.K, pw.N, _ptr(out), _stream(stream))
    return out


# ------------------------------------------------------------------ mixture of experts

@dataclass
class MoeWeights:
    """The expert stacks of one MoE MLP (E routed experts + the shared one, number E):
    gate_up packed with gate/up rows interleaved per tile (K = H, N = (E+1)*2I) and down
    packed plainly (K = I, N = (E+1)*H)."""
    gate_up: PackedWeight
    down: PackedWeight
    E: int
    H: int
    I: int


def pack_moe(gu: tuple, dn: tuple, E: int, H: int, I: int, stream=None) -> MoeWeights:
    """MLX-layout stacks -> MoeWeights. gu = (w [(E+1)*2I][H/8], s, b [(E+1)*2I][H/64]);
    dn = (w [(E+1)*H][I/8], s, b [(E+1)*H][I/64])."""
    gw, gs, gb = gu
    N, K = _check_mlx(gw, gs, gb)
    if (N, K) != ((E + 1) * 2 * I, H):
        raise ValueError(f"gate/up stack is [{N}][{K}], expected [{(E + 1) * 2 * I}][{H}]")
    out = torch.empty(packed_bytes(H, N), dtype=torch.uint8, device=gw.device)
    lib.call("rlq_pack_moe_gate_up", _ptr(gw), _ptr(gs), _ptr(gb), H, E + 1, I, _ptr(out), _stream(stream))
    g = PackedWeight(out, H, N, gs.dtype)
    d = pack_affine(*dn, stream=stream)
    if (d.N, d.K) != ((E + 1) * H, I):
        raise ValueError(f"down stack is [{d.N}][{d.K}], expected [{(E + 1) * H}][{I}]")
    return MoeWeights(g, d, E, H, I)


@dataclass
class MoeRouting:
    sel: torch.Tensor       # int32 [T*S]
    w: torch.Tensor         # float32 [T*S]
    tok: torch.Tensor       # int32 [T*S]: token of each sorted row
    inv: torch.Tensor       # int32 [T*S]: sorted row of each assignment
    items: torch.Tensor     # int32 [max_items][4]
    n_items: torch.Tensor   # int32 [1]
    T: int
    topk: int


def moe_route(logits: torch.Tensor, E: int, topk: int, norm_topk: bool = True, stream=None) -> MoeRouting:
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1 or logits.shape[1] < E + 1:
        raise ValueError("logits must be a row-major float32 [T][>= E+1] matrix")
    T = logits.shape[0]
    A = T * (topk + 1)
    dev = logits.device
    mi = int(lib.load().rlq_moe_max_items(T, E, topk))
    r = MoeRouting(torch.empty(A, dtype=torch.int32, device=dev), torch.empty(A, dtype=torch.float32, device=dev),
                   torch.empty(A, dtype=torch.int32, device=dev), torch.empty(A, dtype=torch.int32, device=dev),
                   torch.empty((max(mi, 1), 4), dtype=torch.int32, device=dev),
                   torch.empty(1, dtype=torch.int32, device=dev), T, topk)
    lib.call("rlq_moe_route", _ptr(logits), logits.stride(0), T, E, topk, 1 if norm_topk else 0, _ptr(r.sel), _ptr(r.w),
             _ptr(r.tok), _ptr(r.inv), _ptr(r.items), _ptr(r.n_items), _stream(stream))
    return r


def moe_gate_up(x: torch.Tensor, mw: MoeWeights, r: MoeRouting, stream=None) -> torch.Tensor:
    """act fp16 [T*S][I]: SwiGLU of the routed rows' gate/up products (sorted row order)."""
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < mw.H:
        raise ValueError("x must be a row-major float16 [T][>= H] matrix")
    act = torch.empty((r.T * (r.topk + 1), mw.I), dtype=torch.float16, device=x.device)
    lib.call("rlq_moe_gate_up", _ptr(x), x.stride(0), r.T, mw.H, mw.I, mw.E, r.topk, _ptr(mw.gate_up.packed),
             mw.gate_up.code, _ptr(r.tok), _ptr(r.items), _ptr(r.n_items), _ptr(act), act.stride(0), _stream(stream))
    return act


def moe_down(act: torch.Tensor, mw: MoeWeights, r: MoeRouting, stream=None) -> torch.Tensor:
    y = torch.empty((r.T * (r.topk + 1), mw.H), dtype=torch.float32, device=act.device)
    lib.call("rlq_moe_down", _ptr(act), act.stride(0), r.T, mw.H, mw.I, mw.E, r.topk, _ptr(mw.down.packed),
             mw.down.code, _ptr(r.items), _ptr(r.n_items), _ptr(y), y.stride(0), _stream(stream))
    return y


def moe_combine(y: torch.Tensor, r: MoeRouting, h: torch.Tensor, stream=None) -> torch.Tensor:
    lib.call("rlq_moe_combine", _ptr(y), y.stride(0), _ptr(r.inv), _ptr(r.w), r.T, r.topk, h.shape[1], _ptr(h),
             h.stride(0), _stream(stream))
    return h


def moe_workspace_bytes(T: int, E: int, topk: int, H: int, I: int) -> int:
    return int(lib.load().rlq_moe_workspace_bytes(T, E, topk, H, I))


def moe(x: torch.Tensor, logits: torch.Tensor, mw: MoeWeights, topk: int, h: torch.Tensor, norm_topk: bool = True,
        workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """h[t] += the MoE MLP of x[t] (route, gate/up + SwiGLU, down, combine), in one call."""
    T = x.shape[0]
    if h.dtype != torch.float32 or h.stride(1) != 1 or h.shape[0] < T or h.shape[1] < mw.H:
        raise ValueError("h must be a row-major float32 [T][>= H] matrix")
    nbytes = moe_workspace_bytes(T, mw.E, topk, mw.H, mw.I)
    ws = workspace if workspace is not None else torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    lib.call("rlq_moe", _ptr(x), x.stride(0), _ptr(logits), logits.stride(0), T, mw.E, topk, 1 if norm_topk else 0,
             mw.H, mw.I, _ptr(mw.gate_up.packed), _ptr(mw.down.packed), mw.gate_up.code, _ptr(h), h.stride(0), _ptr(ws),
             ws.numel(), _stream(stream))
    return h


# ------------------------------------------------------------------ native experts

@dataclass
class MoeNativeStack:
    """One kind of expert matrices (gate_up or down) in the native format: n_slots slots of
    Ne rows each (the stacked tensor, slot = expert, or an expert cache), codes in the tile
    layout and one fp32 scale per row (kernels/linear.metal:254-308)."""
    packed: torch.Tensor     # uint8, rlq_packed_codes_bytes(K, n_slots * Ne)
    s_row: torch.Tensor      # float32 [n_slots * Ne]
    K: int
    Ne: int
    n_slots: int
    book: str

    @property
    def code(self) -> int:
        return BOOKS[self.book]


def pack_moe_native(w: torch.Tensor, s_row: torch.Tensor, Ne: int, book: str, stream=None) -> MoeNativeStack:
    """Row-major codes of the stacked tensor (32-bit words [n_slots*Ne][K/8]) -> MoeNativeStack."""
    nw = pack_native(w, s_row, book, stream=stream)
    if nw.N % Ne:
        raise ValueError(f"{nw.N} rows is not a whole number of {Ne}-row slots")
    return MoeNativeStack(nw.packed, nw.s_row, nw.K, Ne, nw.N // Ne, book)


def moe_linear_native(a: torch.Tensor, st: MoeNativeStack, slots: torch.Tensor, r: MoeRouting, gather: bool,
                      out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """c fp32 [T*S][Ne]: each sorted row times its expert's slot (rlq_moe_linear_native);
    gather: a holds the T tokens and row r reads token tok[r], else a holds sorted rows."""
    if a.dtype != torch.float16 or a.dim() != 2 or a.stride(1) != 1 or a.shape[1] < st.K:
        raise ValueError("a must be a row-major float16 matrix of >= K columns")
    if slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32 vector [E+1]")
    A = r.T * (r.topk + 1)
    if out is None:
        out = torch.empty((A, st.Ne), dtype=torch.float32, device=a.device)
    lib.call("rlq_moe_linear_native", _ptr(a), a.stride(0), a.shape[0], _ptr(r.tok) if gather else 0, st.K, st.Ne,
             _ptr(st.packed), _ptr(st.s_row), _ptr(slots), st.n_slots, st.code, _ptr(r.items), _ptr(r.n_items),
             r.items.shape[0], _ptr(out), out.stride(0), _stream(stream))
    return out


def moe_swiglu(gu: torch.Tensor, I: int, cs: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """act fp16 [A][I] = half(silu(g) * u * cs) (rlq_moe_swiglu)."""
    if gu.dtype != torch.float32 or gu.dim() != 2 or gu.stride(1) != 1:
        raise ValueError("gu must be a row-major float32 matrix")
    if cs is not None and (cs.dtype != torch.float32 or not cs.is_contiguous() or cs.numel() < I):
        raise ValueError("cs must be a contiguous float32 vector of >= I column scales")
    act = torch.empty((gu.shape[0], I), dtype=torch.float16, device=gu.device)
    lib.call("rlq_moe_swiglu", _ptr(gu), gu.stride(0), gu.shape[0], I, _ptr(cs) if cs is not None else 0, _ptr(act),
             act.stride(0), _stream(stream))
    return act


def moe_gate_up_native(x: torch.Tensor, gu: MoeNativeStack, slots: torch.Tensor, r: MoeRouting,
                       cs: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """act fp16 [T*S][I]: the gathered gate/up product and the SwiGLU in one launch
    (rlq_moe_gate_up_native; the bits of moe_linear_native + moe_swiglu)."""
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < gu.K:
        raise ValueError("x must be a row-major float16 [T][>= H] matrix")
    if cs is not None and (cs.dtype != torch.float32 or not cs.is_contiguous() or cs.numel() < gu.Ne // 2):
        raise ValueError("cs must be a contiguous float32 vector of >= I column scales")
    I = gu.Ne // 2
    act = torch.empty((r.T * (r.topk + 1), I), dtype=torch.float16, device=x.device)
    lib.call("rlq_moe_gate_up_native", _ptr(x), x.stride(0), x.shape[0], _ptr(r.tok), gu.K, I, _ptr(gu.packed),
             _ptr(gu.s_row), _ptr(slots), gu.n_slots, gu.code, _ptr(r.items), _ptr(r.n_items), r.items.shape[0],
             _ptr(cs) if cs is not None else 0, _ptr(act), act.stride(0), _stream(stream))
    return act


def moe_native(x: torch.Tensor, logits: torch.Tensor, gu: MoeNativeStack, dn: MoeNativeStack, slots: torch.Tensor,
               topk: int, h: torch.Tensor, cs: torch.Tensor | None = None, norm_topk: bool = True,
               fused: bool = True, one_call: bool = True, workspace: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
    """The native MoE MLP in the reference's order (src/engine.mm:965-1059): route, gate_up
    product with the gather fused, SwiGLU with the down matrix's column scale cs (folded
    into the gate_up launch when fused), down product, combine into h. x is already times
    gate_up's column scale. one_call: rlq_moe_native (the same bits as the steps)."""
    E = slots.numel() - 1
    if gu.Ne % 2 or dn.K != gu.Ne // 2 or dn.Ne != gu.K:
        raise ValueError("gate_up [2I][H] and down [H][I] stacks do not match")
    if gu.book != dn.book:
        raise ValueError("gate_up and down stacks use different codebooks")
    if one_call:
        T, H, I = x.shape[0], gu.K, gu.Ne // 2
        if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1 or x.shape[1] < H:
            raise ValueError("x must be a row-major float16 [T][>= H] matrix")
        if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
            raise ValueError("logits must be a row-major float32 matrix")
        if slots.dtype != torch.int32 or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous int32 vector [E+1]")
        nbytes = moe_workspace_bytes(T, E, topk, H, I)
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        lib.call("rlq_moe_native", _ptr(x), x.stride(0), _ptr(logits), logits.stride(0), T, E, topk,
                 1 if norm_topk else 0, H, I, _ptr(gu.packed), _ptr(gu.s_row), _ptr(dn.packed), _ptr(dn.s_row),
                 _ptr(slots), gu.n_slots, gu.code, _ptr(cs) if cs is not None else 0, _ptr(h), h.stride(0),
                 _ptr(workspace), workspace.numel(), _stream(stream))
        return h
    r = moe_route(logits, E, topk, norm_topk, stream=stream)
    if fused:
        act = moe_gate_up_native(x, gu, slots, r, cs, stream=stream)
    else:
        act = moe_swiglu(moe_linear_native(x, gu, slots, r, True, stream=stream), gu.Ne // 2, cs, stream=stream)
    y = moe_linear_native(act, dn, slots, r, False, stream=stream)
    return moe_combine(y, r, h, stream=stream)


# ------------------------------------------------------------------ positions, cache, attention

ROPE_SCALINGS = {"plain": 0, "linear": 1, "ntk": 2, "parts": 3}   # include/rlq.h RLQ_ROPE_*


def rope_frequencies(rot: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0, low: float = 1.0,
                     high: float = 32.0, original: int = 0, device="cuda") -> torch.Tensor:
    """Radians per token of the rot/2 rotated pairs, float64 (rlq_rope_frequencies): what
    rope_append takes as freq, kept by the program."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}")
    if rot < 0 or rot % 2:
        raise ValueError(f"rot={rot} must be even and not negative")
    f = torch.empty(rot // 2, dtype=torch.float64)
    host = f if rot else torch.empty(1, dtype=torch.float64)
    lib.call("rlq_rope_frequencies", ROPE_SCALINGS[scaling], rot, base, factor, low, high, float(original),
             host.data_ptr())
    return f.to(device)


def kv_cache(n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.float16,
             device="cuda"):
    """The two arrays of a paged key/value cache, [n_pages][kv_heads][page_size][head_dim]
    (include/rlq.h has the order of a page's elements). They need no filling: what was not
    written is never read into a result."""
    scale_code(dtype)
    if page_size < 32 or page_size % 32 or head_dim not in (64, 128, 256):
        raise ValueError(f"page_size={page_size} must be a multiple of 32, head_dim={head_dim} 64, 128 or 256")
    shape = (n_pages, kv_heads, page_size, head_dim)
    return torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)


# Dtypes are compared by identity and devices by number here: a serving step makes these calls for
# every layer, and the checks are half of what a call costs the host.
_CODES = {torch.float16: F16, torch.bfloat16: BF16}


def _check_paged(k_cache, v_cache, cu_q, kv_len, table):
    """Shapes, types and places of a cache and its sequences -> (n_pages, kv_heads, page_size,
    head_dim), the type's code, the device's number, B."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not k_cache.dtype:
        raise ValueError("k_cache and v_cache must be alike, [n_pages][kv_heads][page_size][head_dim]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous")
    code = _CODES.get(k_cache.dtype)
    if code is None:
        raise ValueError(f"the cache must be float16 or bfloat16, not {k_cache.dtype}")
    i32 = torch.int32
    if cu_q.dtype is not i32 or kv_len.dtype is not i32 or table.dtype is not i32:
        raise TypeError("cu_q, kv_len and table must be int32")
    B = kv_len.numel()
    if kv_len.shape != (B,) or cu_q.shape != (B + 1,) or not (cu_q.is_contiguous() and kv_len.is_contiguous()):
        raise ValueError("kv_len must be a contiguous vector [B], cu_q [B + 1]")
    rows = table.shape
    if len(rows) != 2 or rows[0] < B or (rows[1] > 1 and table.stride(1) != 1) or (
            rows[0] > 1 and table.stride(0) < rows[1]):
        raise ValueError("table must be a row-major matrix [B][pages of a sequence]")
    dev = k_cache.get_device()
    if v_cache.get_device() != dev or cu_q.get_device() != dev or kv_len.get_device() != dev or table.get_device() != dev:
        raise ValueError("the cache and its sequences must be on one device")
    return shape, code, dev, B


def _rows(t, dtype, dev, what):
    """(rows, columns, row stride) of a row-major matrix of a type on a device."""
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{what} must be {dtype} on the device of the call's other tensors")
    shape = t.shape
    if len(shape) != 2 or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be a row-major matrix")
    return shape[0], shape[1], t.stride(0) if shape[0] > 1 else max(t.stride(0), shape[1])


def _call_on(dev: int, stream, name: str, *args):
    """lib.call on the device its tensors live on, whichever is current."""
    if dev < 0:
        raise ValueError(f"{name} needs tensors on the GPU")
    if stream is not None and stream.device_index != dev:
        raise ValueError(f"{name}: the stream is on device {stream.device_index}, the tensors on {dev}")
    if _raw_stream is None or _current_device is None or _current_device() != dev:
        with torch.cuda.device(dev):
            return lib.call(name, *args, _stream(stream))
    return lib.call(name, *args, _raw_stream(dev) if stream is None else stream.cuda_stream)


def _new(like, shape, dtype, stream, scratch=False) -> torch.Tensor:
    """An output or scratch tensor of a call on `stream`. Its memory is that stream's own: what the
    current stream's pool gives may still be written by work queued there before it was freed, and
    nothing makes `stream` wait for that. An output is kept until the current stream, where the
    caller goes on with it, is through."""
    if stream is None or not like.is_cuda:
        return torch.empty(shape, dtype=dtype, device=like.device)
    current = torch.cuda.current_stream(like.device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=like.device)
    if not scratch and current != stream:
        t.record_stream(current)
    return t


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                cu_q: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor, freq: torch.Tensor | None,
                interleaved: bool = False, mscale: float = 1.0, q_norm: torch.Tensor | None = None,
                k_norm: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                stream=None) -> torch.Tensor:
    """Rows of a layer's q, k and v (fp32, slices of the stacked linear's rows, say) -> rotated
    queries [T][heads * head_dim] in the cache's dtype, and keys and values in the cache
    (rlq_rope_append). Row i of a sequence's n new rows has position kv_len - n + i; freq:
    rope_frequencies, None turns nothing. Rows from cu_q[B] on are left as they were in `out`."""
    (n_pages, kv_heads, page, D), code, dev, B = _check_paged(k_cache, v_cache, cu_q, kv_len, table)
    f32 = torch.float32
    T, width, qs = _rows(q, f32, dev, "q")
    Tk, kw, ks = _rows(k, f32, dev, "k")
    Tv, vw, vs = _rows(v, f32, dev, "v")
    if Tk != T or Tv != T or kw != kv_heads * D or vw != kw or width % max(kw, 1) or not width:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match {kv_heads} "
                         f"key/value heads of {D}")
    rot = 0
    if freq is not None:
        if freq.dtype is not torch.float64 or freq.dim() != 1 or not freq.is_contiguous() or freq.get_device() != dev:
            raise ValueError("freq must be a contiguous float64 vector on the cache's device")
        rot = 2 * freq.numel()
    for w in (q_norm, k_norm):
        if w is not None and (w.dtype is not f32 or w.shape != (D,) or not w.is_contiguous() or w.get_device() != dev):
            raise ValueError(f"q_norm and k_norm must be contiguous float32 vectors of {D} on the cache's device")
    if out is None:
        out = _new(q, (T, width), k_cache.dtype, stream)
        os = width
    else:
        To, ow, os = _rows(out, k_cache.dtype, dev, "out")
        if To != T or ow != width:
            raise ValueError("out must be shaped like q")
    _call_on(dev, stream, "rlq_rope_append", q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, T, _ptr(freq), rot,
             1 if interleaved else 0, mscale, _ptr(q_norm), _ptr(k_norm), eps, width // D, kv_heads, D, code,
             out.data_ptr(), os, k_cache.data_ptr(), v_cache.data_ptr(), n_pages, page, cu_q.data_ptr(),
             kv_len.data_ptr(), table.data_ptr(), max(table.stride(0), table.shape[1]), table.shape[1], B)
    return out


FULL_WEIGHTS = 16   # include/rlq.h RLQ_FULL_WEIGHTS


@functools.lru_cache(maxsize=4096)
def attention_workspace_bytes(T: int, heads: int, kv_heads: int, head_dim: int, B: int, max_q: int, max_kv: int,
                              window: int = 0) -> int:
    return int(lib.load().rlq_attention_workspace_bytes(T, heads, kv_heads, head_dim, B, max_q, max_kv, window))


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor,
              table: torch.Tensor, max_q: int, max_kv: int, scale: float | None = None, window: int = 0,
              softcap: float = 0.0, out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16,
              workspace: torch.Tensor | None = None, stream=None, full_weights: bool = False) -> torch.Tensor:
    """Causal attention of new rows q [T][heads * head_dim] (the cache's dtype) over their
    sequences' pages, the rows' own keys among them (rlq_attention) -> [T][heads * head_dim] in
    out_dtype. max_q and max_kv bound a sequence's new and all tokens; scale: 1 / sqrt(head_dim)
    by default; window: the last positions a row sees (0: all); softcap: 0 for none. Rows from
    cu_q[B] on are left as they were in `out`. workspace: scratch to use in place of a new
    tensor; calls that overlap must not share it. full_weights: softmax weights keep more bits than
    the rows in calls of many rows too, as they do in those of few, in 4/3 of the time."""
    (n_pages, kv_heads, page, D), code, dev, B = _check_paged(k_cache, v_cache, cu_q, kv_len, table)
    T, width, qs = _rows(q, k_cache.dtype, dev, "q")
    if not width or width % max(kv_heads * D, 1):
        raise ValueError(f"q rows of {width} are no whole number of {D}-wide heads a key/value head")
    if out is None:
        out = _new(q, (T, width), out_dtype, stream)
        os = width
    else:
        To, ow, os = _rows(out, out.dtype, dev, "out")
        if To != T or ow != width:
            raise ValueError("out must be shaped like q")
    out_code = _CODES.get(out.dtype)
    if out_code is None:
        raise ValueError(f"out must be float16 or bfloat16, not {out.dtype}")
    H = width // D
    most = 2**31 - 1                      # past what a position can be: no window, no bound
    max_q, max_kv, window = min(max_q, most), min(max_kv, 2**29), min(window, most)
    nbytes = attention_workspace_bytes(T, H, kv_heads, D, B, max_q, max_kv, window)
    if workspace is None:
        if nbytes:
            workspace = _new(q, nbytes, torch.uint8, stream, scratch=True)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on the cache's device")
    else:
        nbytes = workspace.numel() * workspace.element_size()
    _call_on(dev, stream, "rlq_attention", q.data_ptr(), qs, T, H, kv_heads, D, code, k_cache.data_ptr(),
             v_cache.data_ptr(), n_pages, page, cu_q.data_ptr(), kv_len.data_ptr(), table.data_ptr(),
             max(table.stride(0), table.shape[1]), table.shape[1], B, max_q, max_kv, D ** -0.5 if scale is None else scale,
             window, softcap, out.data_ptr(), os, out_code | (FULL_WEIGHTS if full_weights else 0), _ptr(workspace), nbytes)
    return out


# ------------------------------------------------------------------ linear attention

def _check_sequences(cu_q, kv_len, slots, keep, dev):
    """Types, shapes and places of the sequences of a call with states -> B."""
    i32 = torch.int32
    if cu_q.dtype is not i32 or kv_len.dtype is not i32 or slots.dtype is not i32 or (
            keep is not None and keep.dtype is not i32):
        raise TypeError("cu_q, kv_len, slots and keep must be int32")
    B = kv_len.numel()
    if kv_len.shape != (B,) or cu_q.shape != (B + 1,) or slots.shape != (B,) or not (
            cu_q.is_contiguous() and kv_len.is_contiguous() and slots.is_contiguous()):
        raise ValueError("kv_len and slots must be contiguous vectors [B], cu_q [B + 1]")
    if keep is not None and (keep.shape != (B,) or not keep.is_contiguous() or keep.get_device() != dev):
        raise ValueError("keep must be a contiguous vector [B] on the device of the call's other tensors")
    if cu_q.get_device() != dev or kv_len.get_device() != dev or slots.get_device() != dev:
        raise ValueError("the sequences must be on the device of the call's other tensors")
    return B


def conv_state(n_slots: int, channels: int, taps: int = 4, device="cuda") -> torch.Tensor:
    """The states of causal_conv, [n_slots][taps - 1][channels] fp32. They need no filling: a sequence
    begins from zeros."""
    return torch.empty((n_slots, taps - 1, channels), dtype=torch.float32, device=device)


def delta_state(n_slots: int, v_heads: int, k_dim: int, v_dim: int, device="cuda") -> torch.Tensor:
    """The states of gated_delta, [n_slots][v_heads][k_dim][v_dim] fp32. They need no filling either."""
    return torch.empty((n_slots, v_heads, k_dim, v_dim), dtype=torch.float32, device=device)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor,
                slots: torch.Tensor, bias: torch.Tensor | None = None, silu: bool = True,
                keep: torch.Tensor | None = None, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float16, stream=None) -> torch.Tensor:
    """The short causal convolution of a linear-attention layer (rlq_causal_conv): rows x fp32
    [T][channels] (a slice of the in projection's rows, say) with weight fp32 [channels][taps] ->
    [T][channels] in out_dtype, and the sequences' last inputs in state (conv_state), in place.
    cu_q and kv_len as for rope_append; slots int32 [B]: the states' places, one outside the array for
    none. A sequence whose rows are all its tokens begins from zeros. keep int32 [B]: how many of a
    sequence's rows go into its state (all by default; a draft's rows are computed with 0, then again
    with what was taken). Rows from cu_q[B] on are left as they were in `out`."""
    f32, dev = torch.float32, state.get_device()
    T, C, xs = _rows(x, f32, dev, "x")
    if weight.dtype is not f32 or weight.dim() != 2 or weight.shape[0] != C or not weight.is_contiguous() or (
            weight.get_device() != dev):
        raise ValueError(f"weight must be a contiguous float32 matrix [{C}][taps] on the state's device")
    taps = weight.shape[1]
    if bias is not None and (bias.dtype is not f32 or bias.shape != (C,) or not bias.is_contiguous() or (
            bias.get_device() != dev)):
        raise ValueError(f"bias must be a contiguous float32 vector of {C} on the state's device")
    if state.dtype is not f32 or state.dim() != 3 or state.shape[1:] != (taps - 1, C) or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 [n_slots][{taps - 1}][{C}]")
    B = _check_sequences(cu_q, kv_len, slots, keep, dev)
    if out is None:
        out = _new(x, (T, C), out_dtype, stream)
        os = C
    else:
        To, ow, os = _rows(out, out.dtype, dev, "out")
        if To != T or ow != C:
            raise ValueError("out must be shaped like x")
    out_code = _CODES.get(out.dtype)
    if out_code is None:
        raise ValueError(f"out must be float16 or bfloat16, not {out.dtype}")
    _call_on(dev, stream, "rlq_causal_conv", x.data_ptr(), xs, T, C, taps, weight.data_ptr(), _ptr(bias),
             1 if silu else 0, state.data_ptr(), state.shape[0], cu_q.data_ptr(), kv_len.data_ptr(), slots.data_ptr(),
             _ptr(keep), B, out.data_ptr(), os, out_code)
    return out


@functools.lru_cache(maxsize=4096)
def gated_delta_workspace_bytes(T: int, k_heads: int, v_heads: int, k_dim: int, v_dim: int, B: int, max_q: int) -> int:
    return int(lib.load().rlq_gated_delta_workspace_bytes(T, k_heads, v_heads, k_dim, v_dim, B, max_q))


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                a_log: torch.Tensor, dt_bias: torch.Tensor, state: torch.Tensor, cu_q: torch.Tensor,
                kv_len: torch.Tensor, slots: torch.Tensor, max_q: int, scale: float | None = None, eps: float = 1e-6,
                z: torch.Tensor | None = None, norm: torch.Tensor | None = None, norm_eps: float = 1e-6,
                keep: torch.Tensor | None = None, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float16, workspace: torch.Tensor | None = None,
                stream=None) -> torch.Tensor:
    """The gated delta rule of a linear-attention layer (rlq_gated_delta): rows q, k [T][k_heads * k_dim]
    and v [T][v_heads * v_dim] (float16 or bfloat16, slices of causal_conv's rows, say) with a, b fp32
    [T][v_heads] and a_log, dt_bias fp32 [v_heads] -> [T][v_heads * v_dim] in out_dtype, and state
    (delta_state) updated in place. q and k are brought to length 1 here, q times scale
    (1 / sqrt(k_dim) by default). z fp32 [T][v_heads * v_dim] and norm fp32 [v_dim]: the rows' heads
    normalised and gated for the out projection. max_q bounds a sequence's rows; cu_q, kv_len, slots and keep
    as for causal_conv. workspace: scratch to use in place of a new tensor; calls that overlap must
    not share it. Rows from cu_q[B] on are left as they were in `out`."""
    f32, dev, shape = torch.float32, state.get_device(), state.shape
    if state.dtype is not f32 or len(shape) != 4 or not state.is_contiguous():
        raise ValueError("state must be contiguous float32 [n_slots][v_heads][k_dim][v_dim]")
    n_slots, Hv, Dk, Dv = shape
    code = _CODES.get(q.dtype)
    if code is None:
        raise ValueError(f"q, k and v must be float16 or bfloat16, not {q.dtype}")
    T, width, qs = _rows(q, q.dtype, dev, "q")
    Tk, kw, ks = _rows(k, q.dtype, dev, "k")
    Tv, vw, vs = _rows(v, q.dtype, dev, "v")
    Ta, aw, as_ = _rows(a, f32, dev, "a")
    Tb, bw, bs = _rows(b, f32, dev, "b")
    if Tk != T or Tv != T or kw != width or vw != Hv * Dv or not width or width % max(Dk, 1):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match states of "
                         f"{Hv} heads of {Dk} x {Dv}")
    if Ta != T or Tb != T or aw != Hv or bw != Hv:
        raise ValueError(f"a and b must be [{T}][{Hv}]")
    for t, n, what in ((a_log, Hv, "a_log"), (dt_bias, Hv, "dt_bias"), (norm, Dv, "norm")):
        if t is not None and (t.dtype is not f32 or t.shape != (n,) or not t.is_contiguous() or t.get_device() != dev):
            raise ValueError(f"{what} must be a contiguous float32 vector of {n} on the state's device")
    if (z is None) != (norm is None):
        raise ValueError("z and norm come together")
    zs = 0
    if z is not None:
        Tz, zw, zs = _rows(z, f32, dev, "z")
        if Tz != T or zw != Hv * Dv:
            raise ValueError("z must be shaped like v")
    B = _check_sequences(cu_q, kv_len, slots, keep, dev)
    if out is None:
        out = _new(q, (T, Hv * Dv), out_dtype, stream)
        os = Hv * Dv
    else:
        To, ow, os = _rows(out, out.dtype, dev, "out")
        if To != T or ow != Hv * Dv:
            raise ValueError("out must be shaped like v")
    out_code = _CODES.get(out.dtype)
    if out_code is None:
        raise ValueError(f"out must be float16 or bfloat16, not {out.dtype}")
    max_q = min(max_q, 2**31 - 1)
    nbytes = gated_delta_workspace_bytes(T, width // Dk, Hv, Dk, Dv, B, max_q)
    if workspace is None:
        if nbytes:
            workspace = _new(q, nbytes, torch.uint8, stream, scratch=True)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on the state's device")
    else:
        nbytes = workspace.numel() * workspace.element_size()
    _call_on(dev, stream, "rlq_gated_delta", q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, T, width // Dk, Hv, Dk,
             Dv, code, a.data_ptr(), as_, b.data_ptr(), bs, a_log.data_ptr(), dt_bias.data_ptr(), eps,
             Dk ** -0.5 if scale is None else scale, _ptr(z), zs, _ptr(norm), norm_eps, state.data_ptr(), n_slots,
             cu_q.data_ptr(), kv_len.data_ptr(), slots.data_ptr(), _ptr(keep), B, max_q, out.data_ptr(), os, out_code,
             _ptr(workspace), nbytes)
    return out


# ------------------------------------------------------------------ logits

def _row_vector(t, rows, dtype, what, dev) -> int:
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != (rows,) or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{what} must be a contiguous {dtype} vector of {rows} rows on the logits' device")
    return t.data_ptr()


def _shared_rows(t, rows, dtypes, what, dev):
    """(pointer, row stride, columns) of a matrix with a row per row of logits, or of one row (or
    a vector) for all: stride 0."""
    shape = t.shape
    if t.dtype not in dtypes or len(shape) not in (1, 2) or (shape[-1] > 1 and t.stride(-1) != 1) or t.get_device() != dev:
        raise ValueError(f"{what} must be a row-major {dtypes[0]} matrix (or one row) on the logits' device")
    if len(shape) == 1:
        return t.data_ptr(), 0, shape[0]
    if shape[0] != rows and shape[0] != 1:
        raise ValueError(f"{what} has {shape[0]} rows, the logits have {rows}")
    return t.data_ptr(), t.stride(0) if shape[0] > 1 else 0, shape[1]


_I32, _F32, _BITS = (torch.int32,), (torch.float32,), (torch.int32, torch.uint32)


def adjust_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, n_tokens: torch.Tensor | None = None,
                  n_prompt: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Penalties, biases and a mask on rows of logits (fp32 [rows][vocab]) before a token is
    chosen from them (rlq_adjust_logits) -> out (may be logits; a new tensor by default).
    tokens int32 [rows][n], the first n_tokens of a row count: any of them for `repetition`,
    those from n_prompt on for `presence` and `frequency` (fp32 [rows]); bias_ids int32 and bias
    fp32 [rows][n]; allowed int32 or uint32 [rows][words], bit v % 32 of word v / 32 set where
    token v may follow. tokens, biases and the mask may be one row for all."""
    dev = logits.get_device()
    rows, vocab, xs = _rows(logits, torch.float32, dev, "logits")
    if out is None:
        out = _new(logits, (rows, vocab), torch.float32, stream)
        ys = vocab
    else:
        orows, ovocab, ys = _rows(out, torch.float32, dev, "out")
        if orows != rows or ovocab != vocab:
            raise ValueError("out must be shaped like logits")
    tp = ts = n = ip = bp = bs = nb = mp = ms = 0
    if tokens is not None:
        tp, ts, n = _shared_rows(tokens, rows, _I32, "tokens", dev)
    if (bias is None) != (bias_ids is None):
        raise ValueError("bias and bias_ids come together")
    if bias is not None:
        bp, bs, nb = _shared_rows(bias, rows, _F32, "bias", dev)
        ip, ids_stride, ids_n = _shared_rows(bias_ids, rows, _I32, "bias_ids", dev)
        if ids_n != nb or ids_stride != bs:
            raise ValueError("bias_ids must be laid out like bias")
    if allowed is not None:
        mp, ms, words = _shared_rows(allowed, rows, _BITS, "allowed", dev)
        if words < (vocab + 31) // 32:
            raise ValueError(f"a mask row of {words} words is shorter than the vocabulary")
    _call_on(dev, stream, "rlq_adjust_logits", logits.data_ptr(), xs, rows, vocab, tp, ts, n,
             _row_vector(n_tokens, rows, torch.int32, "n_tokens", dev),
             _row_vector(n_prompt, rows, torch.int32, "n_prompt", dev),
             _row_vector(repetition, rows, torch.float32, "repetition", dev),
             _row_vector(presence, rows, torch.float32, "presence", dev),
             _row_vector(frequency, rows, torch.float32, "frequency", dev), ip, bp, nb, bs, mp, ms, out.data_ptr(), ys)
    return out


@functools.lru_cache(maxsize=4096)
def sample_workspace_bytes(rows: int, vocab: int) -> int:
    return int(lib.load().rlq_sample_workspace_bytes(rows, vocab))


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           out: torch.Tensor | None = None, probs: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
           stream=None) -> torch.Tensor:
    """A token from each row of logits (fp32 [rows][vocab], adjust_logits's out, say) and a number of
    [0, 1) given for it (uniform, fp64 [rows]) -> int32 [rows] (rlq_sample). temperature, top_p and min_p
    fp32 [rows], top_k int32 [rows]; None: 1 and all tokens. Temperature 0 takes the largest logit.
    Cut to the top_k, of these to the shortest prefix of top_p of the weight, of these to min_p of
    the largest weight. probs (fp32 [rows]) gets the tokens' shares of the kept weight. A row without a logit
    above -inf gives -1. workspace: scratch to use in place of a new tensor; calls that overlap must
    not share it."""
    dev = logits.get_device()
    rows, vocab, xs = _rows(logits, torch.float32, dev, "logits")
    f32, i32 = torch.float32, torch.int32
    if out is None:
        out = _new(logits, (rows,), i32, stream)
    nbytes = sample_workspace_bytes(rows, vocab)
    if workspace is None:
        if nbytes:
            workspace = _new(logits, nbytes, torch.uint8, stream, scratch=True)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on the logits' device")
    else:
        nbytes = workspace.numel() * workspace.element_size()
    _call_on(dev, stream, "rlq_sample", logits.data_ptr(), xs, rows, vocab,
             _row_vector(uniform, rows, torch.float64, "uniform", dev),
             _row_vector(temperature, rows, f32, "temperature", dev), _row_vector(top_k, rows, i32, "top_k", dev),
             _row_vector(top_p, rows, f32, "top_p", dev), _row_vector(min_p, rows, f32, "min_p", dev),
             _row_vector(out, rows, i32, "out", dev), _row_vector(probs, rows, f32, "probs", dev), _ptr(workspace), nbytes)
    return out
