"""Layers on 4-bit weights with a float16 scale and bias for each group of columns, on B200: MLX's affine form, which
the reference holds its dense layers, its shared experts and its draft head's experts in (`to_affine`,
strata_mlx/gguf.py:182-276; `nn.QuantizedLinear`, strata_mlx/load.py:235-256; `QuantizedSwitchLinear`,
strata_mlx/mtp.py:34-75).

    quantize, dequantize    floats to codes, scales and biases, and back
    QuantizedLinear         one layer: x W^T for any number of tokens
    QuantizedSwitchLinear   one projection of every expert, for (token, expert) pairs
    QuantizedSwitchGLU      the routed experts' SwiGLU feed-forwards
    QuantizedMLP            the shared expert
    moe                     a MoE block behind its route, for which `fused.SparseMoeBlock` calls it

A weight is code * scale + bias with a code of 4 bits, eight codes to a 32-bit word (weight 8 j + i in bits 4 i of
word j), groups of 32, 64 or 128 columns. A layer lays its arrays out once for the kernels (libstrata_moe.so) and
keeps that alone. Products are exact in each weight (codes are not rounded to floats first) with float32 sums; a layer's
product of more than 16 float16 tokens, and experts' of more than MAX_PAIRS float16 pairs, may go by a kernel that rounds each
weight to float16 once (as `dequantize` does: a weight beyond float16's range is infinite there). Activations that are not finite
make their token's results not finite, NaN also where the definition has an infinity. Float32 has no kernel for prompts: a layer's
weights are read and decoded again for every 8 tokens. Activations are float16 or float32; tensors are torch CUDA tensors and
there is no CPU path.
"""

import ctypes

import torch

from . import _lib
from .blocks import TOKENS_TILE, _flat_idx, slot_rows, swiglu_to, tiles_of

BITS = 4
GROUPS = (32, 64, 128)
MAX_PAIRS = 2048  # (token, expert) pairs of one streaming launch; a longer call goes by tiles, or in several launches
TILE_PAIRS = 1 << 18  # pairs that go by tiles at once (what bounds the float32 gate and up of a long prompt)
MOE_TOKENS = 64  # tokens that `moe` takes in its two launches
COMBINE_TOKENS = 1 << 15  # tokens of a prompt that it takes at once


def _check_group(group_size: int, bits: int = BITS) -> None:
    if bits != BITS:
        raise ValueError(f"weights of {bits} bits are not supported (4 bits)")
    if group_size not in GROUPS:
        raise ValueError(f"groups of {group_size} columns are not supported (32, 64 or 128)")


def _elsewhere(device) -> bool:
    """Whether `device` is not the current one (the kernels launch on the current device)."""
    return device.index != torch.cuda.current_device()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and on a 16-byte boundary (a view into another tensor may not be)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_parts(codes, scales, biases, group_size, bits=BITS):
    _check_group(group_size, bits)
    _lib.require_cuda(codes, scales, biases)
    if not codes.device == scales.device == biases.device:
        raise ValueError(f"codes, scales and biases on {codes.device}, {scales.device} and {biases.device}")
    if codes.dtype not in (torch.int32, torch.uint32):
        raise ValueError(f"codes come as 32-bit words, not {codes.dtype}")
    if scales.dtype != torch.float16 or biases.dtype != torch.float16:
        raise ValueError("scales and biases are float16")
    cs, ss = codes.shape, scales.shape
    if len(cs) < 1 or ss != biases.shape or ss[:-1] != cs[:-1] or cs[-1] * 8 != ss[-1] * group_size:
        raise ValueError(f"codes {tuple(cs)}, scales {tuple(ss)} and biases {tuple(biases.shape)} are no matrix in groups "
                         f"of {group_size}")


def quantize(w: torch.Tensor, group_size: int = 64, bits: int = BITS):
    """Float weights (..., rows, cols) as (codes int32 (..., rows, cols / 8), scales, biases float16 (..., rows,
    cols / group_size)). Of each group, bias is the least value and scale a fifteenth of the range, both rounded to
    float16; a code is (w - bias) / scale rounded to even within 0 .. 15 (0 where the scale is 0). Values beyond
    float16's range or not finite give groups that are not finite. (MLX's quantize of the same arguments fits scale and bias in
    a way of its own: arrays made there and here stand for the same weights within a step, but are not equal.)"""
    _check_group(group_size, bits)
    _lib.require_cuda(w)
    if w.dim() < 1 or w.shape[-1] == 0 or w.shape[-1] % group_size:
        raise ValueError(f"{tuple(w.shape)}: the columns are no whole number of groups of {group_size}")
    code = _lib.dtype_code(w.dtype)
    if _elsewhere(w.device):
        with torch.cuda.device(w.device):
            return quantize(w, group_size, bits)
    cols = w.shape[-1]
    rows = w.numel() // cols
    w2 = _aligned(w)
    lead = w.shape[:-1]
    codes = w.new_empty((*lead, cols // 8), dtype=torch.int32)
    scales = w.new_empty((*lead, cols // group_size), dtype=torch.float16)
    biases = torch.empty_like(scales)
    if rows:
        _lib.call("smoe_q4_quantize", w2.data_ptr(), code, rows, cols, group_size, codes.data_ptr(), scales.data_ptr(),
                  biases.data_ptr(), _lib.raw_stream(w.device.index))
    return codes, scales, biases


def dequantize(codes: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int = 64, bits: int = BITS,
               dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The floats (..., rows, cols) of `quantize`'s arrays: code * scale + bias in float32, rounded to `dtype`."""
    _check_parts(codes, scales, biases, group_size, bits)
    code = _lib.dtype_code(dtype)
    if _elsewhere(codes.device):
        with torch.cuda.device(codes.device):
            return dequantize(codes, scales, biases, group_size, bits, dtype)
    cols = codes.shape[-1] * 8
    out = codes.new_empty((*codes.shape[:-1], cols), dtype=dtype)
    n = out.numel()
    if n:
        codes, scales, biases = codes.contiguous(), scales.contiguous(), biases.contiguous()
        _lib.call("smoe_q4_dequant", codes.data_ptr(), scales.data_ptr(), biases.data_ptr(), n // cols, cols, group_size,
                  out.data_ptr(), code, _lib.raw_stream(codes.device.index))
    return out


class _Packed:
    """A stack (experts, rows, cols) of 4-bit weights in the kernels' layout."""

    def __init__(self, codes, scales, biases, group_size):
        _check_parts(codes, scales, biases, group_size)
        if codes.numel() == 0:
            raise ValueError("a layer without weights")
        self.num_experts, self.output_dims = (1, codes.shape[0]) if codes.dim() == 2 else codes.shape[:2]
        self.input_dims, self.group_size = codes.shape[-1] * 8, group_size
        self.device = codes.device
        nbytes = int(_lib.lib().smoe_q4_bytes(self.num_experts, self.output_dims, self.input_dims, group_size))
        with torch.cuda.device(self.device):
            self.packed = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            codes, scales, biases = codes.contiguous(), scales.contiguous(), biases.contiguous()
            _lib.call("smoe_q4_pack", _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(biases), self.num_experts,
                      self.output_dims, self.input_dims, group_size, _lib.ptr(self.packed), _lib.stream())

    @property
    def data_ptr(self) -> int:
        return self.packed.data_ptr()

    @property
    def nbytes(self) -> int:
        return self.packed.numel()

    def _floats(self, shape, dtype):
        code = _lib.dtype_code(dtype)
        with torch.cuda.device(self.device):
            out = torch.empty(shape, dtype=dtype, device=self.device)
            _lib.call("smoe_q4_unpack", _lib.ptr(self.packed), self.num_experts, self.output_dims, self.input_dims,
                      self.group_size, _lib.ptr(out), code, _lib.stream())
        return out

    def _rows(self, x: torch.Tensor) -> torch.Tensor:
        """x (..., in) as rows one after the other, on a 16-byte boundary."""
        if x.dim() < 1 or x.shape[-1] != self.input_dims:
            raise ValueError(f"activations {tuple(x.shape)} do not end in {self.input_dims}")
        if x.device != self.device:
            _lib.require_cuda(x)
            raise ValueError(f"activations on {x.device}, weights on {self.device}")
        return _aligned(x)


class QuantizedLinear(_Packed):
    """One linear layer on 4-bit weights, used like `nn.Linear` without a bias: codes (out, in / 8), scales and biases
    (out, in / group_size). x (..., in) -> (..., out) in x's type. A token gets the same bits
    alone as in a window of up to 16 tokens; more float16 tokens take the prompt's kernel where that is the faster one."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int = 64):
        if codes.dim() != 2:
            raise ValueError(f"a layer's codes are (out, in / 8), not {tuple(codes.shape)}")
        super().__init__(codes, scales, biases, group_size)

    @classmethod
    def from_float(cls, w: torch.Tensor, group_size: int = 64) -> "QuantizedLinear":
        return cls(*quantize(w, group_size), group_size=group_size)

    def floats(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """The weights (out, in), as `dequantize` gives them."""
        return self._floats((self.output_dims, self.input_dims), dtype)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        code = _lib.dtype_code(x.dtype)
        x2 = self._rows(x)
        if _elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self(x)
        out = x.new_empty((*x.shape[:-1], self.output_dims))
        tokens = x2.numel() // self.input_dims
        if tokens:
            _lib.call("smoe_q4_linear", self.data_ptr, self.output_dims, self.input_dims, self.group_size,
                      x2.data_ptr(), tokens, out.data_ptr(), code, _lib.raw_stream(self.device.index))
        return out

    def _prompt(self, x2: torch.Tensor) -> torch.Tensor:
        """(tokens, out) in float32 of float16 rows x2, by the prompt's kernel, on the current device."""
        out = torch.empty((x2.shape[0], self.output_dims), dtype=torch.float32, device=self.device)
        _lib.call("smoe_q4_prompt", self.data_ptr, self.output_dims, self.input_dims, self.group_size, x2.data_ptr(),
                  x2.shape[0], out.data_ptr(), _lib.F32, _lib.raw_stream(self.device.index))
        return out


def _pair_chunks(pairs: int, share: int, most: int = MAX_PAIRS):
    """Ranges of up to `most` pairs, whole rows of `share`."""
    step = max(1, most // share) * share
    return [(p, min(p + step, pairs)) for p in range(0, pairs, step)]


def _by_tiles(lin, dtype, pairs: int) -> bool:
    """Whether a call's pairs go in tiles of one expert's, through the prompt's kernel (float16; tiles_of takes up to 1024
    experts): when one streaming launch would not take them. The SwiGLU of 512 experts of 640 x 2560, ten a token: 192
    tokens 395 us streamed and 571 by tiles, 256 tokens 757 and 580, 1180 tokens 3087 and 679; 256 of 1536 x 4096, eight a
    token: 192 tokens 662 and 938, 512 tokens 2087 and 963, 1180 tokens 4812 and 1031."""
    return dtype == torch.float16 and lin.num_experts <= 1024 and pairs > MAX_PAIRS


class _Tiles:
    """A call's pairs by expert: `row` the row of x in each slot, `slot_row` each slot's pair."""

    def __init__(self, lin, indices: torch.Tensor, share: int):
        self.lin, self.pairs = lin, indices.numel()
        tile_expert, token, where = tiles_of(indices.reshape(-1, share), lin.num_experts)
        self.row, self.count = token.view(torch.int32), tile_expert.numel()
        self.slot_row = slot_rows(where, self.count * TOKENS_TILE)
        nbytes = int(_lib.lib().smoe_q4_tile_plan_size(self.count))
        self.plan = torch.empty(nbytes, dtype=torch.uint8, device=lin.device)
        _lib.call("smoe_q4_tile_plan", _lib.ptr(tile_expert), self.count, lin.num_experts, _lib.ptr(self.plan), nbytes,
                  _lib.stream())

    def product(self, lin, a: torch.Tensor, out: torch.Tensor, in_pairs: bool) -> torch.Tensor:
        """lin's products of the slots' rows `a`, into out's rows in the order of the slots or of the pairs."""
        _lib.call("smoe_q4_tile_matmul", lin.data_ptr, lin.num_experts, lin.output_dims, lin.input_dims, lin.group_size,
                  _lib.ptr(a), self.count, _lib.ptr(self.plan), _lib.ptr(self.slot_row) if in_pairs else None, out.shape[0],
                  _lib.ptr(out), _lib.dtype_code(out.dtype), _lib.stream())
        return out


def _check_pairs(indices, k):
    _lib.require_cuda(indices)
    if not 1 <= k <= MAX_PAIRS:
        raise ValueError(f"{k} experts a row")


class QuantizedSwitchLinear(_Packed):
    """One projection of every expert on 4-bit weights: codes (experts, out, in / 8), scales and biases (experts, out,
    in / group_size); its call takes what `BlockSwitchLinear`'s takes."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int = 64):
        if codes.dim() != 3:
            raise ValueError(f"a stack's codes are (experts, out, in / 8), not {tuple(codes.shape)}")
        if codes.shape[0] > 2048:
            raise ValueError(f"{codes.shape[0]} experts: a stack holds up to 2048")
        super().__init__(codes, scales, biases, group_size)

    @classmethod
    def from_float(cls, w: torch.Tensor, group_size: int = 64) -> "QuantizedSwitchLinear":
        return cls(*quantize(w, group_size), group_size=group_size)

    @property
    def shape(self):
        return (self.num_experts, self.output_dims, self.input_dims)

    def floats(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return self._floats(self.shape, dtype)

    def __call__(self, x: torch.Tensor, indices: torch.Tensor, sorted_indices: bool = False) -> torch.Tensor:
        """Each (token, expert) pair of `indices` times its activation row; x (..., 1, in), one row per entry of
        `indices` or one that the entries along its last axis share. Returns (*indices.shape, 1, out). An index at or
        past the expert count names a pair that is left out (its row is not written)."""
        ishape = tuple(indices.shape)
        if x.dim() < 2 or x.shape[-2] != 1:
            raise ValueError(f"activations {tuple(x.shape)} are not (..., 1, in)")
        batch = tuple(x.shape[:-2])
        k = ishape[-1] if indices.dim() else 1
        if batch == ishape:
            share = 1
        elif indices.dim() and batch == (*ishape[:-1], 1):
            share = k
        else:
            x, share = x.expand(*ishape, 1, self.input_dims), 1
        out = _pairs_product(self, None, self._rows(x).reshape(-1, self.input_dims), indices, share)
        return out.reshape(*ishape, 1, self.output_dims)


def _pairs_product(lin, lin2, x2, indices, share, zeros=False):
    """(pairs, out): rows x2[p // share] through expert indices[p] of `lin`, or through gate `lin` and up `lin2`; zeros:
    pairs of no expert get rows of zeros."""
    code = _lib.dtype_code(x2.dtype)
    if indices.device != lin.device:
        _lib.require_cuda(indices)
        raise ValueError(f"indices on {indices.device}, weights on {lin.device}")
    with torch.cuda.device(lin.device):
        idx = _flat_idx(indices)
        pairs = idx.numel()
        out = (torch.zeros if zeros else torch.empty)((pairs, lin.output_dims), dtype=x2.dtype, device=lin.device)
        if pairs:
            _check_pairs(idx, share)
            if x2.shape[0] * share != pairs:
                raise ValueError("indices must hold the same number of experts for every row of x")
        if lin2 is None and _by_tiles(lin, x2.dtype, pairs):
            for p0, p1 in _pair_chunks(pairs, share, TILE_PAIRS):
                tiles = _Tiles(lin, idx[p0:p1], share)
                tiles.product(lin, x2[p0 // share : p1 // share].index_select(0, tiles.row), out[p0:p1], True)
            return out
        for p0, p1 in _pair_chunks(pairs, share) if pairs else ():
            spec = _lib.SmoeQ4Product(dtype=code, group=lin.group_size, x=x2[p0 // share].data_ptr(), cols=lin.input_dims,
                                      stack=lin.data_ptr, stack2=lin2.data_ptr if lin2 is not None else None,
                                      rows=lin.output_dims, experts=lin.num_experts, idx=idx[p0:].data_ptr(),
                                      pairs=p1 - p0, share=share, out=out[p0:].data_ptr())
            _lib.call("smoe_q4_product", ctypes.byref(spec), _lib.stream())
    return out


def _alike(a, b) -> bool:
    return (a.num_experts, a.output_dims, a.input_dims, a.group_size, a.device) == (
        b.num_experts, b.output_dims, b.input_dims, b.group_size, b.device)


def _check_glu(gate, up, down):
    if not _alike(gate, up):
        raise ValueError("gate and up must have one shape, group size and device")
    if (down.num_experts, down.input_dims, down.output_dims) != (gate.num_experts, gate.output_dims, gate.input_dims):
        raise ValueError("down must take gate's outputs to its inputs")
    if down.device != gate.device:
        raise ValueError(f"down on {down.device}, gate on {gate.device}")


class QuantizedSwitchGLU:
    """The routed experts of one layer on 4-bit weights: x (..., in) and indices (..., k) -> (..., k, out), each
    down(silu(gate x) * up x); gate and up in one launch that forms the SwiGLU, a prompt's by tiles and a SwiGLU of float32.
    Rows of pairs of no expert are not written."""

    def __init__(self, gate: QuantizedSwitchLinear, up: QuantizedSwitchLinear, down: QuantizedSwitchLinear):
        _check_glu(gate, up, down)
        self.gate_proj, self.up_proj, self.down_proj = gate, up, down

    def __call__(self, x: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
        if indices.dim() < 1:
            raise ValueError("indices must hold k experts for every token of x")
        out = self._pairs(self.gate_proj._rows(x).reshape(-1, x.shape[-1]), indices)
        return out.reshape(*indices.shape, self.down_proj.output_dims)

    def _pairs(self, x2: torch.Tensor, indices: torch.Tensor, zeros: bool = False) -> torch.Tensor:
        """The experts' outputs (pairs, out); zeros: rows of zeros for pairs of no expert."""
        gate, up, down = self.gate_proj, self.up_proj, self.down_proj
        pairs, k = indices.numel(), indices.shape[-1]
        if not _by_tiles(gate, x2.dtype, pairs) or indices.device != gate.device or x2.shape[0] * k != pairs or k > MAX_PAIRS:
            h = _pairs_product(gate, up, x2, indices, k)
            return _pairs_product(down, None, h, indices, 1, zeros)
        # a prompt: gate and up in the order of the slots, the SwiGLU of their float32 sums rounded once
        with torch.cuda.device(gate.device):
            idx = _flat_idx(indices)
            out = (torch.zeros if zeros else torch.empty)((pairs, down.output_dims), dtype=x2.dtype, device=gate.device)
            for p0, p1 in _pair_chunks(pairs, k, TILE_PAIRS):
                tiles = _Tiles(gate, idx[p0:p1], k)
                a = x2[p0 // k : p1 // k].index_select(0, tiles.row)
                g, u = (tiles.product(p, a, torch.empty((len(a), p.output_dims), dtype=torch.float32, device=a.device), False)
                        for p in (gate, up))
                tiles.product(down, swiglu_to(g, u, x2.dtype), out[p0:p1], True)
        return out


class QuantizedMLP:
    """The shared expert on 4-bit weights: down(silu(gate x) * up x). Gate, up and the SwiGLU are one launch; a long
    float16 prompt's are the prompt's products in float32 and a SwiGLU. Either rounds the SwiGLU to x's type once."""

    def __init__(self, gate: QuantizedLinear, up: QuantizedLinear, down: QuantizedLinear):
        _check_glu(gate, up, down)
        self.gate_proj, self.up_proj, self.down_proj = gate, up, down

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        code = _lib.dtype_code(x.dtype)
        gate, up = self.gate_proj, self.up_proj
        x2 = gate._rows(x).reshape(-1, gate.input_dims)
        if x.dtype == torch.float16 and self._apart(x2.shape[0]):
            with torch.cuda.device(gate.device):
                out = self.down_proj(swiglu_to(gate._prompt(x2), up._prompt(x2), x.dtype))
            return out.reshape(*x.shape[:-1], self.down_proj.output_dims)
        with torch.cuda.device(gate.device):
            h = torch.empty((x2.shape[0], gate.output_dims), dtype=x.dtype, device=gate.device)
            if x2.shape[0]:
                spec = _lib.SmoeQ4Product(dtype=code, group=gate.group_size, x=x2.data_ptr(), cols=gate.input_dims,
                                          dense=gate.data_ptr, dense2=up.data_ptr, dense_rows=gate.output_dims,
                                          dense_tokens=x2.shape[0], dense_out=h.data_ptr())
                _lib.call("smoe_q4_product", ctypes.byref(spec), _lib.stream())
            out = self.down_proj(h)
        return out.reshape(*x.shape[:-1], self.down_proj.output_dims)

    def _apart(self, tokens: int) -> bool:
        """Whether gate and up go by the prompt's kernel, for more than a window's 16 tokens: the streaming launch takes 0.3 us and 0.25 ps a weight for every
        8 tokens, 30 us of which are about the other's start (whole calls of 4096 x 4096: 48 tokens 48 us streamed and 49
        apart, 96 tokens 78 and 50; of 640 x 2560: 128 tokens 21 and 27, 512 tokens 50 and 31). (A few long rows may be better
        streamed all the same.)"""
        rows, cols = self.gate_proj.output_dims, self.gate_proj.input_dims
        return (tokens > 16 and (tokens + 7) // 8 * (0.3 + 2.5e-7 * rows * cols) > 30
                and bool(_lib.lib().smoe_q4_is_prompt(tokens, rows, cols)))


def moe_takes(switch_mlp, shared) -> bool:
    """Whether `moe` runs these experts in its two launches: 4-bit, of one hidden size, group sizes alike in gate / up
    and in down."""
    if not isinstance(switch_mlp, QuantizedSwitchGLU) or not isinstance(shared, QuantizedMLP):
        return False
    g, d, sg, sd = switch_mlp.gate_proj, switch_mlp.down_proj, shared.gate_proj, shared.down_proj
    return (g.input_dims == sg.input_dims and g.group_size == sg.group_size and d.group_size == sd.group_size
            and g.device == sg.device)


def moe(switch_mlp: QuantizedSwitchGLU, shared: QuantizedMLP, x: torch.Tensor, indices: torch.Tensor, w: torch.Tensor,
        g: torch.Tensor) -> torch.Tensor:
    """sum_j w_j switch_mlp(x, indices)_j + sigmoid(g) shared(x): x (..., hidden), indices and w (..., k) with w float32,
    g (..., 1) in x's type. Up to MOE_TOKENS tokens in two launches, sums float32 and rounded to x's type once (the SwiGLU times
    its weight keeps 22 bits between the launches, for float16 down to 2^-25; one beyond 65504 makes its token's result NaN);
    more tokens by switch_mlp, shared and the block's combine, each rounded to x's type. An index at or past the expert count
    adds nothing. A token's last bits may differ alone and in a window."""
    if not moe_takes(switch_mlp, shared):
        raise ValueError("moe takes 4-bit experts of one hidden size, with one group size in gate / up and one in down")
    if g.dtype != x.dtype:
        raise ValueError("gate values are of the activations' type")
    return _moe(switch_mlp, shared, x, indices, w, g)


def _moe(switch_mlp, shared, x, indices, w, g):
    """`moe` for experts that it takes; g in x's type or, up to MOE_TOKENS tokens, in float32."""
    gate, down = switch_mlp.gate_proj, switch_mlp.down_proj
    sgate, sdown = shared.gate_proj, shared.down_proj
    code = _lib.dtype_code(x.dtype)
    x2 = gate._rows(x).reshape(-1, gate.input_dims)
    _lib.require_cuda(indices, w, g)
    if any(t.device != gate.device for t in (indices, w, g)):
        raise ValueError(f"weights on {gate.device}, a choice on another device")
    tokens, k = x2.shape[0], indices.shape[-1] if indices.dim() else 0
    if indices.numel() != tokens * k or w.numel() != tokens * k or g.numel() != tokens or not 1 <= k <= 32:
        raise ValueError("moe takes 1 to 32 experts and weights and one gate value for every token")
    if w.dtype != torch.float32 or (g.dtype != x.dtype and (g.dtype != torch.float32 or tokens > MOE_TOKENS)):
        raise ValueError("weights are float32 and gate values of the activations' type")
    with torch.cuda.device(gate.device):
        idx, w, g = _flat_idx(indices), w.contiguous(), g.contiguous()
        out = torch.empty((tokens, gate.input_dims), dtype=x.dtype, device=gate.device)
        if tokens > MOE_TOKENS:
            # (512 experts of 640 x 2560, ten a token, 96 tokens: 384 us, in calls of 64 tokens 615)
            idx = idx.reshape(tokens, k)
            for t0 in range(0, tokens, COMBINE_TOKENS):
                t1 = min(t0 + COMBINE_TOKENS, tokens)
                y, s = switch_mlp._pairs(x2[t0:t1], idx[t0:t1], zeros=True), shared(x2[t0:t1])
                _lib.call("smoe_combine", _lib.ptr(y), w.data_ptr() + 4 * t0 * k, g.data_ptr() + g.element_size() * t0,
                          _lib.ptr(s), t1 - t0, k, gate.input_dims, out[t0:].data_ptr(), code, _lib.stream())
        elif tokens:
            nbytes = int(_lib.lib().smoe_q4_moe_workspace_size(tokens, k, gate.input_dims, gate.output_dims,
                                                                sgate.output_dims))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=gate.device)
            spec = _lib.SmoeQ4Moe(
                dtype=code, group=gate.group_size, down_group=down.group_size, tokens=tokens, hidden=gate.input_dims,
                experts=gate.num_experts, k=k, ffn=gate.output_dims, shared_ffn=sgate.output_dims, x=x2.data_ptr(),
                idx=idx.data_ptr(), weights=w.data_ptr(), gate=gate.data_ptr,
                up=switch_mlp.up_proj.data_ptr, down=down.data_ptr, sgate=sgate.data_ptr, sup=shared.up_proj.data_ptr,
                sdown=sdown.data_ptr, out=out.data_ptr())
            if g.dtype == x.dtype:
                spec.shared_gate = g.data_ptr()
            else:
                spec.shared_gate32 = g.data_ptr()
            _lib.call("smoe_q4_moe", ctypes.byref(spec), _lib.ptr(ws), nbytes, _lib.stream())
    return out.reshape(x.shape)


def failed(clear: bool = False) -> bool:
    """Whether a bounded wait of the 4-bit kernels gave up on the current device (outputs since are then not valid).
    Synchronizes."""
    status = ctypes.c_int(0)
    _lib.call("smoe_q4_status", ctypes.byref(status), int(clear))
    return status.value != 0


__all__ = ["BITS", "GROUPS", "QuantizedLinear", "QuantizedMLP", "QuantizedSwitchGLU", "QuantizedSwitchLinear", "dequantize",
           "failed", "moe", "moe_takes", "quantize"]
