"""fp8 (e4m3) with one fp32 scale per block of 128: quantisation, products, a
linear layer, and the experts' FFNs (``sb_fp8_*`` of libspider_b200).

Activations carry one scale per row and 128 columns, weights one per 128 x 128
block, so an outlier costs the resolution of its own block only (``quant.py``'s
formats, the reference's, have one scale per tensor or per row).  With
``a = max(amax, 2^-100)`` of a block, ``scale = a / 448`` and
``q = e4m3(x * (448 / a))``, each step one fp32 rounding.  The products run on
the fp8 tensor cores; the scaled sums are fp32.

CUDA tensors only.  Every call enqueues on the current stream of its tensors'
device and allocates its own scratch there, so calls on several streams and
captured graphs do not share any.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass

import torch

from . import _lib as L
from .expert_parallel import all_reduce_sum_, ep_enabled, get_rank_world

BLOCK = 128
MAX_COLS, MAX_BATCH, MAX_TILE_ROWS = 2 ** 24, 65535, 65535 * 128  # of the quantisation's grids
_DTYPES = {torch.float32: L.SB_F32, torch.bfloat16: L.SB_BF16}
_ID_TYPES = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _dtype_code(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _need_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"spider_b200 {what} runs on CUDA tensors only")


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


# Device status words (one per device): the kernels' bounded waits record there.
_STATUS: dict = {}


def _status_ptr(device) -> int | None:
    hit = _STATUS.get(device)
    if hit is None:
        if torch.cuda.is_current_stream_capturing():
            return None  # memory of this capture's pool would not outlive the graph
        t = torch.zeros(1, dtype=torch.int32, device=device)
        hit = _STATUS[device] = (t, t.data_ptr())
    return hit[1]


def check_status(device) -> None:
    """Raise if a kernel of this module recorded an error on ``device`` (a
    bounded wait ran out); waits for all its streams."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    hit = _STATUS.get(device)
    if hit is None:
        return
    torch.cuda.synchronize(device)
    word = int(hit[0].item())
    if word:
        raise L.SpiderB200Error(L.SB_ERR_DEVICE_STATUS, f"fp8_blocks: device status 0x{word:x}")


_CHECK = bool(os.environ.get("SPIDER_B200_CHECK"))  # read once: the lookup costs a launch's share of host time


def _finish(rc: int, where: str, device) -> None:
    if rc != L.SB_OK:
        L.check(rc, where)
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        check_status(device)


@dataclass
class Fp8BlockTensor:
    """e4m3 matrix (or a stack of them) with its block scales.

    q: float8_e4m3fn [R, C] or [E, R, C], unit column stride, rows on 16-byte
    boundaries.  scale: fp32 [.., ceil(R / block_rows), ceil(C / 128)], any
    strides.  block_rows: 1 or 128."""

    q: torch.Tensor
    scale: torch.Tensor
    block_rows: int

    def __post_init__(self):
        q, s = self.q, self.scale
        if self.block_rows not in (1, BLOCK):
            raise ValueError(f"block_rows must be 1 or {BLOCK}, got {self.block_rows}")
        if q.dtype != torch.float8_e4m3fn or s.dtype != torch.float32:
            raise TypeError(f"need float8_e4m3fn values and float32 scales, got {q.dtype} and {s.dtype}")
        if q.dim() not in (2, 3):
            raise ValueError(f"need a matrix or a stack of matrices, got shape {tuple(q.shape)}")
        r, c = q.shape[-2:]
        want = (*q.shape[:-2], -(-r // self.block_rows), _blocks(c))
        if tuple(s.shape) != want or s.device != q.device:
            raise ValueError(f"scale must be {want} on the values' device, got {tuple(s.shape)} on {s.device}")
        if q.numel() and ((c > 1 and q.stride(-1) != 1) or q.data_ptr() % 16 or
                          (r > 1 and (q.stride(-2) % 16 or q.stride(-2) < c))):
            raise ValueError("fp8 rows must be contiguous and start on 16-byte boundaries (pad the row pitch)")

    @property
    def shape(self):
        return self.q.shape

    @property
    def pitch(self) -> int:
        """Bytes from one row to the next."""
        return self.q.stride(-2) if self.q.shape[-2] > 1 else -(-self.q.shape[-1] // 16) * 16

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        r, c = self.q.shape[-2:]
        s = self.scale.repeat_interleave(self.block_rows, -2)[..., :r, :].repeat_interleave(BLOCK, -1)[..., :c]
        return (self.q.float() * s).to(dtype)

    def transpose(self) -> "Fp8BlockTensor":
        """The transposed matrix, same values (128 x 128 blocks only); a copy."""
        if self.block_rows != BLOCK:
            raise ValueError("only 128 x 128 blocks keep their scales when transposed")
        q = _empty_fp8((*self.q.shape[:-2], self.q.shape[-1], self.q.shape[-2]), self.q.device)
        q.view(torch.uint8).copy_(self.q.view(torch.uint8).transpose(-1, -2))
        return Fp8BlockTensor(q, self.scale.transpose(-1, -2), BLOCK)


def _empty_fp8(shape, device) -> torch.Tensor:
    """[..., C] e4m3 whose rows start on 16-byte boundaries."""
    c = shape[-1]
    return torch.empty((*shape[:-1], -(-c // 16) * 16), dtype=torch.float8_e4m3fn, device=device)[..., :c]


def quantize_fp8_blocks(x: torch.Tensor, block_rows: int = 1) -> Fp8BlockTensor:
    """x [R, C] or [E, R, C] (float32 or bfloat16, any strides) -> Fp8BlockTensor
    with one scale per ``block_rows`` x 128 block (block_rows 1 or 128).  The values
    have no gradient.  At most 2^24 columns, 65535 matrices, and 65535 * 128 rows
    (2^31 - 256 with block_rows 1, unless the rows, not the columns, are contiguous)."""
    code = _dtype_code(x, "quantize_fp8_blocks input")
    if x.dim() not in (2, 3):
        raise ValueError(f"quantize_fp8_blocks needs [R, C] or [E, R, C], got shape {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    L.refuse_forward_ad("quantize_fp8_blocks", x)
    lead, (r, c) = x.shape[:-2], x.shape[-2:]
    by_tiles = block_rows == BLOCK or (x.stride(-2) == 1 and x.stride(-1) != 1)
    L.check_extent("rows", r, MAX_TILE_ROWS if by_tiles else L.MAX_EXTENT)
    L.check_extent("columns", c, MAX_COLS)
    L.check_extent("matrices", lead[0] if lead else 1, MAX_BATCH)
    _need_cuda(x, "quantize_fp8_blocks")
    x = x.detach()
    q = _empty_fp8(x.shape, x.device)
    cb = _blocks(c)
    if block_rows == 1:  # row-contiguous: a product reads one block's scales of many rows at a time
        scale = torch.empty((*lead, cb, -(-r // 4) * 4), dtype=torch.float32, device=x.device)
        scale = scale.transpose(-1, -2)[..., :r, :]
    else:
        scale = torch.empty((*lead, _blocks(r), cb), dtype=torch.float32, device=x.device)
    if x.numel():
        batch = lead[0] if lead else 1
        three = len(lead) == 1
        a = L.Fp8QuantizeArgs(
            x=x.data_ptr(), dtype=code, block_rows=block_rows, batch=batch, rows=r, cols=c,
            x_row=x.stride(-2), x_col=x.stride(-1), x_batch=x.stride(0) if three else 0,
            q=q.data_ptr(), ldq=-(-c // 16) * 16, q_batch=q.stride(0) if three else 0,
            scale=scale.data_ptr(), scale_row=scale.stride(-2), scale_col=scale.stride(-1),
            scale_batch=scale.stride(0) if three else 0)
        rc = L.on_device(x.device, L.load().sb_fp8_quantize_blocks, C.byref(a))
        L.check(rc, "sb_fp8_quantize_blocks")
    return Fp8BlockTensor(q, scale, block_rows)


def fp8_block_matmul(a: Fp8BlockTensor, b: Fp8BlockTensor, out_dtype: torch.dtype = torch.bfloat16,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """a [M, K] (1 x 128 blocks) times b [N, K] transposed (128 x 128 or 1 x 128
    blocks) -> [M, N] in out_dtype (bfloat16 or float32), summed in fp32."""
    if a.q.dim() != 2 or b.q.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"fp8_block_matmul needs [M, K] and [N, K], got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.block_rows != 1:
        raise ValueError("the first operand needs 1 x 128 blocks")
    if a.q.device != b.q.device:
        raise ValueError("both operands must be on one device")
    m, k = a.shape
    n = b.shape[0]
    if max(m, n, k) > L.MAX_EXTENT:
        raise ValueError(f"fp8_block_matmul: sizes of at most {L.MAX_EXTENT}, got {(m, n, k)}")
    if out is None:
        if out_dtype not in _DTYPES:
            raise TypeError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
    else:
        _dtype_code(out, "out")
        if tuple(out.shape) != (m, n) or out.device != a.q.device or (n > 1 and out.stride(1) != 1) or \
                (m > 1 and out.stride(0) < n):
            raise ValueError("out must be [M, N] on the operands' device with unit column stride")
    _need_cuda(a.q, "fp8_block_matmul")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.q.device)
    if m == 0 or n == 0:
        return out
    if k == 0:
        return out.zero_()
    args = L.Fp8MatmulArgs(
        epilogue=L.SB_EPI_LINEAR, out_dtype=_DTYPES[out.dtype], num_groups=1, max_rows=m, n=n, k=k,
        a=a.q.data_ptr(), lda=a.pitch, a_scale=a.scale.data_ptr(), a_scale_row=a.scale.stride(0),
        a_scale_block=a.scale.stride(1), b=b.q.data_ptr(), ldb=b.pitch, b_scale=b.scale.data_ptr(),
        b_scale_row=b.scale.stride(0), b_scale_block=b.scale.stride(1), b_block_rows=b.block_rows,
        out=out.data_ptr(), ldo=out.stride(0) if m > 1 else n, status=_status_ptr(out.device))
    rc = L.on_device(out.device, L.load().sb_fp8_matmul, C.byref(args))
    _finish(rc, "sb_fp8_matmul", out.device)
    return out


def _unit_cols(t: torch.Tensor) -> torch.Tensor:
    """t [R, C] with unit column stride and rows that do not overlap (a copy only if it has not)."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _linear(x, weight, packed):
    """y [M, N] for x [M, K] in one library call (weight: the matrix, or the packed values)."""
    x = _unit_cols(x)
    (m, k), n = x.shape, weight.shape[0]
    dev, code = x.device, _DTYPES[x.dtype]
    y = x.new_empty((m, n))
    if m == 0 or n == 0:
        return y
    if k == 0:
        return y.zero_()
    if packed is None:
        w, s = _unit_cols(weight), None
        warg = (w.data_ptr(), _DTYPES[w.dtype], max(w.stride(0), k), None, 0, 0)
    else:
        s = packed.scale
        srow, scol = s.stride()
        warg = (weight.data_ptr(), L.SB_BF16, packed.pitch, s.data_ptr(), srow, scol)
    lib = L.load()
    nbytes = lib.sb_fp8_linear_workspace_bytes(m, n, k, packed is not None)
    ws = x.new_empty((nbytes,), dtype=torch.uint8)
    rc = L.on_device(dev, lib.sb_fp8_linear, x.data_ptr(), code, max(x.stride(0), k), m, n, k, *warg, y.data_ptr(),
                     _status_ptr(dev), ws.data_ptr(), nbytes)
    _finish(rc, "sb_fp8_linear", dev)
    return y


class _Fp8Linear(torch.autograd.Function):
    """y = x w^T; dx = dy w, dw = dy^T x, every operand quantised along the
    dimension its product sums over."""

    @staticmethod
    def forward(ctx, x, weight, packed):
        ctx.packed = packed
        ctx.save_for_backward(x, weight)
        return _linear(x, weight if packed is None else packed.q, packed)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("fp8_block_linear is not twice differentiable")
        L.refuse_forward_ad("fp8_block_linear", dy)
        x, weight = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        if ctx.packed is not None:
            return fp8_block_matmul(quantize_fp8_blocks(dy), ctx.packed.transpose(), x.dtype), None, None
        (m, k), n = x.shape, weight.shape[0]
        dx = torch.empty((m, k), dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty((n, k), dtype=weight.dtype, device=x.device) if need_w else None
        if n == 0 or k == 0:
            return (dx.zero_() if need_x else None), dw, None
        xc, wc = _unit_cols(x), _unit_cols(weight)
        lib = L.load()
        nbytes = lib.sb_fp8_linear_backward_workspace_bytes(m, n, k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        rc = L.on_device(x.device, lib.sb_fp8_linear_backward, xc.data_ptr(), _DTYPES[xc.dtype], max(xc.stride(0), k),
                         m, n, k, wc.data_ptr(), _DTYPES[wc.dtype], max(wc.stride(0), k), dy.data_ptr(), dy.stride(0),
                         dy.stride(1), L.ptr(dx), L.ptr(dw), _status_ptr(x.device), ws.data_ptr(), nbytes)
        _finish(rc, "sb_fp8_linear_backward", x.device)
        return dx, dw, None


def fp8_block_linear(x: torch.Tensor, weight) -> torch.Tensor:
    """x [..., K] (float32 or bfloat16) times weight^T -> [..., N] in x's dtype,
    in block-scaled fp8.  weight: a matrix [N, K] (float32 or bfloat16, quantised
    in the call) or an Fp8BlockTensor [N, K] packed once.  K <= 2^24 and N <= 65535 *
    128 for a weight matrix; with gradients K <= 65535 * 128, and with one in the
    weight at most 2^24 rows of x: the limits of the transposed operands' quantisation.
    Differentiable in x and in a weight matrix (once, in reverse mode); all three
    products run in fp8.  To capture a backward pass into a CUDA graph, drop eager
    graphs of the same leaves first: autograd ties their gradients to the stream
    those were built on."""
    packed = weight if isinstance(weight, Fp8BlockTensor) else None
    w = weight if packed is None else packed.q
    if x.dtype not in _DTYPES or (packed is None and w.dtype not in _DTYPES):
        raise TypeError(f"fp8_block_linear takes float32 or bfloat16, got {x.dtype} and {w.dtype}")
    xs, ws = x.shape, w.shape
    if len(ws) != 2 or not xs or xs[-1] != ws[1]:
        raise ValueError(f"fp8_block_linear needs x [..., K] and weight [N, K], got {tuple(xs)} and {tuple(ws)}")
    if w.device != x.device:
        raise ValueError("x and weight must be on one device")
    if packed is not None and packed.block_rows != BLOCK:
        raise ValueError("packed weights need 128 x 128 blocks")
    L.refuse_forward_ad("fp8_block_linear", x, None if packed is not None else w)
    grad = torch.is_grad_enabled() and (x.requires_grad or (packed is None and w.requires_grad))
    flat = len(xs) == 2
    m = xs[0] if flat else xs[:-1].numel()
    if max(m, ws[0], ws[1]) > MAX_TILE_ROWS:
        L.check_extent("rows of x", m, MAX_COLS if grad and packed is None and w.requires_grad else L.MAX_EXTENT)
        L.check_extent("columns", ws[1], MAX_TILE_ROWS if grad and packed is None else MAX_COLS)
        L.check_extent("rows of the weight", ws[0], MAX_TILE_ROWS if packed is None else MAX_COLS if grad else L.MAX_EXTENT)
    _need_cuda(x, "fp8_block_linear")
    x2 = x if flat else x.reshape(m, ws[1])
    if grad:
        y = _Fp8Linear.apply(x2, None if packed is not None else w, packed)
    else:
        y = _linear(x2, w, packed)
    return y if flat else y.view(*xs[:-1], ws[0])


class Fp8BlockExperts:
    """The experts of a block with block-scaled fp8 weights, packed once.

    w_up / w_gate [E, U, H] and w_down [E, H, U] are Fp8BlockTensors with 128 x
    128 blocks or plain weights, which are quantised here; biases [E, rows] or
    None.  With w_gate the FFN is SwiGLU (``down(silu(gate(x)) * up(x))``), else
    ``down(gelu(up(x)))`` as the reference's (spider_moe/model.py:177-183)."""

    def __init__(self, w_up, b_up, w_down, b_down, w_gate=None, b_gate=None):
        def pack(w, what):
            if not isinstance(w, Fp8BlockTensor):
                w = quantize_fp8_blocks(w, BLOCK)
            q = w.q
            if q.dim() != 3 or w.block_rows != BLOCK:
                raise ValueError(f"{what} must be [E, rows, cols] with 128 x 128 blocks")
            if q.shape[0] > 1 and q.stride(0) != q.shape[1] * w.pitch:  # the experts' rows form one matrix
                flat = _empty_fp8(q.shape, q.device)
                flat.view(torch.uint8).copy_(q.view(torch.uint8))
                q = flat
            return Fp8BlockTensor(q, w.scale.contiguous(), BLOCK)

        def vec(b, rows, what):
            if b is None:
                return None
            if tuple(b.shape) != (self.num_experts, rows):
                raise ValueError(f"{what} must be [{self.num_experts}, {rows}], got {tuple(b.shape)}")
            return b.detach().to(self.device, torch.float32).contiguous()

        self.w_up, self.w_down = pack(w_up, "w_up"), pack(w_down, "w_down")
        self.w_gate = pack(w_gate, "w_gate") if w_gate is not None else None
        self.num_experts, self.ffn, self.hidden = self.w_up.shape
        self.device = self.w_up.q.device
        if tuple(self.w_down.shape) != (self.num_experts, self.hidden, self.ffn) or \
                (self.w_gate is not None and self.w_gate.shape != self.w_up.shape):
            raise ValueError("expert weights must be w_up / w_gate [E, U, H] and w_down [E, H, U]")
        if any(w is not None and w.q.device != self.device for w in (self.w_down, self.w_gate)):
            raise ValueError("all expert weights must be on one device")
        if self.num_experts < 1 or self.ffn < 1 or self.hidden < 1 or self.num_experts > 256:
            raise ValueError("between 1 and 256 experts of at least one row and column")
        if self.w_gate is None and b_gate is not None:
            raise ValueError("b_gate needs w_gate")
        if self.w_gate is not None and self.w_gate.pitch != self.w_up.pitch:
            raise ValueError("w_gate and w_up must have the same row pitch")
        _need_cuda(self.w_up.q, "Fp8BlockExperts")
        self.b_up, self.b_down = vec(b_up, self.ffn, "b_up"), vec(b_down, self.hidden, "b_down")
        self.b_gate = vec(b_gate, self.ffn, "b_gate")
        g = self.w_gate
        self._c = L.Fp8Experts(
            num_experts=self.num_experts, hidden=self.hidden, ffn=self.ffn,
            activation=L.SB_ACT_SWIGLU if g is not None else L.SB_ACT_GELU, ld_in=self.w_up.pitch,
            ld_ffn=self.w_down.pitch, w_up=self.w_up.q.data_ptr(), s_up=self.w_up.scale.data_ptr(),
            b_up=L.ptr(self.b_up), w_gate=g.q.data_ptr() if g is not None else None,
            s_gate=g.scale.data_ptr() if g is not None else None, b_gate=L.ptr(self.b_gate),
            w_down=self.w_down.q.data_ptr(), s_down=self.w_down.scale.data_ptr(), b_down=L.ptr(self.b_down))
        self._ref = C.byref(self._c)

    def weight_bytes(self) -> int:
        ts = [t for w in (self.w_up, self.w_down, self.w_gate) if w is not None for t in (w.q, w.scale)]
        return sum(t.numel() * t.element_size() for t in ts)

    def delta(self, messages: torch.Tensor, top_indices: torch.Tensor, top_weights: torch.Tensor,
              rank: int = 0, world: int = 1, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Weighted sum of the routed experts' outputs [n, H] for messages [n, H] and
        top_indices / top_weights [n, K], experts restricted to ``e % world == rank``."""
        ks, dev = top_indices.shape, self.device
        if len(ks) != 2 or messages.shape != (ks[0], self.hidden) or top_weights.shape != ks:
            raise ValueError(f"need messages [n, {self.hidden}] and top_indices / top_weights [n, K], got "
                             f"{tuple(messages.shape)}, {tuple(ks)}, {tuple(top_weights.shape)}")
        n, k = ks
        if not 1 <= k <= 64:
            raise ValueError("between 1 and 64 experts per token")
        L.check_extent("routes", n * k)
        if top_indices.dtype not in _ID_TYPES:
            raise TypeError(f"top_indices must be integers, got {top_indices.dtype}")
        if not 0 <= rank < world:
            raise ValueError(f"rank {rank} of {world}")
        if messages.device != dev or top_indices.device != dev or top_weights.device != dev:
            raise ValueError("messages, routing and experts must be on one device")
        if torch.is_grad_enabled() and (messages.requires_grad or top_weights.requires_grad):
            raise NotImplementedError("the experts have no backward pass: call them under torch.no_grad()")
        L.refuse_forward_ad("fp8_expert_delta", messages, top_weights)
        code = _dtype_code(messages, "messages")
        out_dtype = messages.dtype if out_dtype is None else out_dtype
        if out_dtype not in _DTYPES:
            raise TypeError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
        lib = L.load()
        x = _unit_cols(messages)
        idx, w = top_indices, top_weights
        if idx.dtype != torch.int32:
            if idx.dtype == torch.int64:  # ids outside [0, E) stay outside
                idx = idx.clamp(-1, self.num_experts)
            idx = idx.to(torch.int32)
        if world > 1:
            idx = torch.where(idx % world == rank, idx, -1)
        if not idx.is_contiguous():
            idx = idx.contiguous()
        if w.dtype != torch.float32 or not w.is_contiguous():
            w = w.to(torch.float32).contiguous()
        cols = -(-self.hidden // 4) * 4
        out = x.new_empty((n, cols), dtype=out_dtype)
        nbytes = lib.sb_fp8_expert_delta_workspace_bytes(self._ref, n, k)
        if nbytes == 0:
            raise L.SpiderB200Error(L.SB_ERR_ARG, "sb_fp8_expert_delta_workspace_bytes")
        ws = x.new_empty((nbytes,), dtype=torch.uint8)
        rc = L.on_device(dev, lib.sb_fp8_expert_delta, self._ref, x.data_ptr(), code, max(x.stride(0), self.hidden),
                         idx.data_ptr(), w.data_ptr(), n, k, out.data_ptr(), _DTYPES[out_dtype], _status_ptr(dev),
                         ws.data_ptr(), nbytes)
        _finish(rc, "sb_fp8_expert_delta", dev)
        return out if cols == self.hidden else out[:, :self.hidden]


def fp8_expert_delta(messages, top_indices, top_weights, experts: Fp8BlockExperts,
                     expert_parallel: bool = True) -> torch.Tensor:
    """``sparse_expert_delta`` with block-scaled fp8 experts: messages [..., H]
    (float32 or bfloat16), top_indices / top_weights [..., K] -> delta [..., H] in
    the messages' dtype.  Repeated ids of a token add their weights, weights <= 0
    and ids outside [0, E) are skipped, a NaN weight makes its token's delta NaN;
    under expert parallelism each rank runs its own experts and the delta is summed
    across ranks.  Inference only."""
    ms, ks, hidden = messages.shape, top_indices.shape, experts.hidden
    if not ms or ms[-1] != hidden or ks != top_weights.shape or ks[:-1] != ms[:-1]:
        raise ValueError(f"need messages [..., {hidden}] and top_indices / top_weights [..., K], got {tuple(ms)}, "
                         f"{tuple(ks)}, {tuple(top_weights.shape)}")
    k = ks[-1]
    if not 1 <= k <= 64:  # reshape below needs it too
        raise ValueError("between 1 and 64 experts per token")
    L.refuse_forward_ad("fp8_expert_delta", messages, top_weights)
    if torch.is_grad_enabled() and (messages.requires_grad or top_weights.requires_grad):
        raise NotImplementedError("fp8_expert_delta has no backward pass: call it under torch.no_grad()")
    use_ep = expert_parallel and ep_enabled()
    rank, world = get_rank_world() if use_ep else (0, 1)
    flat = len(ms) == 2
    if not flat:
        messages, top_indices = messages.reshape(-1, hidden), top_indices.reshape(-1, k)
        top_weights = top_weights.reshape(-1, k)
    delta = experts.delta(messages, top_indices, top_weights, rank, world, torch.float32 if use_ep else messages.dtype)
    if use_ep:
        delta = all_reduce_sum_(delta.contiguous()).to(messages.dtype)
    return delta if flat else delta.reshape(ms)
