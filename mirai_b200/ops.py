"""Torch-facing wrappers of the sm_100a kernels (device memory + streams only).

PyTorch is used here for allocation, streams and dtypes; every computation
below is a call into ``libmirai_b200.so``.  Inputs must be CUDA tensors; there
is no CPU path.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

SCORE_FUNCS = {"softmax": 0, "sigmoid": 1}
NORM_MODES = {"none": 0, "clamp": 1, "eps": 2, "l1": 3}
LAYOUTS = {"out_in": 0, "in_out": 1}      # [G, out, in] (compressed experts) / [G, in, out] (MAGI-2)
ACTIVATIONS = {"swiglu": 0, "swiglu7": 1}
COMBINE_BF16_ACCUM = 2


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _stream() -> int:
    """The current device's current stream (cudaStream_t), without building a Stream object."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _cuda(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the B200 path has no CPU fallback)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    return t.contiguous()


def _run(device: torch.device, name: str, *args, stream: int | None = None) -> None:
    """``name`` on ``device``'s current stream (or ``stream``), with that device current.
    Pointers go as plain integers (None: null); the small calls are paced by their host
    time, so this path looks up the stream and the device without building objects."""
    index = device.index
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        _lib.call(name, *args, stream)
        return
    with torch.cuda.device(index):
        _lib.call(name, *args, stream)


def device_status() -> tuple[int, int]:
    """Synchronise the current stream and return (and clear) the device error word."""
    return _lib.device_status(torch.cuda.current_stream().cuda_stream)


def launch_count() -> int:
    """Kernels libmirai_b200 has enqueued since it was loaded (host-side count:
    every kernel an entry point launched, on any stream)."""
    return _lib.launch_count()


def check_device() -> None:
    code, info = device_status()
    if code:
        raise _lib.MiraiError(code, f"raised on the device at site {info}")


def set_gemm_sm_limit(max_sms: int) -> None:
    """Cap the SMs the persistent grouped GEMMs occupy (0 = all), process-wide,
    so that communication kernels on another stream can run beside them."""
    _lib.call("mirai_b200_set_gemm_sm_limit", int(max_sms))


# ----------------------------------------------------------------------------- a1

def route_topk(logits: torch.Tensor, top_k: int, *, score_func: str = "softmax",
               choice_bias: torch.Tensor | None = None, norm: str = "clamp",
               route_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 top-k routing (routers.py:241-249; transformer_lingbot_video.py:1002-1033).

    Returns (top_indices int64 [T, k], top_weights fp32 [T, k]); slots are in
    descending choice order, ties to the lower expert id.
    """
    logits = _cuda(logits, "logits", torch.float32)
    T, E = logits.shape
    bias = None if choice_bias is None else _cuda(choice_bias, "choice_bias", torch.float32)
    idx = torch.empty((T, top_k), dtype=torch.int64, device=logits.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    if bias is not None and bias.ndim == 2:  # one bias row per T / rows tokens (per head)
        period = T // bias.shape[0] if bias.shape[0] else 0
        if period * bias.shape[0] != T:
            raise ValueError(f"{bias.shape[0]} bias rows do not split {T} tokens evenly")
        _lib.call("mirai_route_topk_rows", _ptr(logits), T, E, top_k, SCORE_FUNCS[score_func], _ptr(bias), period,
                  NORM_MODES[norm], float(route_scale), _ptr(idx), _ptr(w), _stream())
        return idx, w
    _lib.call("mirai_route_topk", _ptr(logits), T, E, top_k, SCORE_FUNCS[score_func], _ptr(bias),
              NORM_MODES[norm], float(route_scale), _ptr(idx), _ptr(w), _stream())
    return idx, w


GROUP_SCORES = {"max": 0, "top2": 1}


def _route_options(score_func: str, norm: str) -> tuple[int, int]:
    if score_func not in SCORE_FUNCS:
        raise ValueError(f"score_func {score_func!r}: one of {sorted(SCORE_FUNCS)}")
    if norm not in NORM_MODES:
        raise ValueError(f"norm {norm!r}: one of {sorted(NORM_MODES)}")
    return SCORE_FUNCS[score_func], NORM_MODES[norm]


def _route_logits(logits: torch.Tensor) -> torch.Tensor:
    logits = _cuda(logits, "logits")
    if logits.dtype not in (torch.float32, torch.bfloat16) or logits.ndim != 2:
        raise TypeError(f"logits must be fp32 or bf16 [T, E], got {logits.dtype} {tuple(logits.shape)}")
    return logits


def route_groups(logits: torch.Tensor, top_k: int, *, num_groups: int = 1, top_groups: int = 1,
                 group_score: str = "top2", score_func: str = "sigmoid", choice_bias: torch.Tensor | None = None,
                 norm: str = "eps", route_scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Group-limited top-k routing of fp32 or bf16 logits [T, E]: of ``num_groups``
    contiguous groups of experts the ``top_groups`` best stay (``group_score``:
    "max", a group's largest key, or "top2", the sum of its two largest score +
    bias), and of their experts the ``top_k`` with the largest score + bias (the
    largest logits without a bias).  Weights are the scores without the bias,
    renormalised as in ``route_topk``.

    Returns (top_indices int64 [T, k], top_weights fp32 [T, k]) in descending
    choice order, ties to the lower expert id; comparisons come out as in
    64-bit arithmetic.  An expert whose logit is -inf or NaN ranks last,
    whatever its bias; a NaN makes its row's weights NaN."""
    score, mode = _route_options(score_func, norm)
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score {group_score!r}: one of {sorted(GROUP_SCORES)}")
    logits = _route_logits(logits)
    T, E = logits.shape
    bias = None if choice_bias is None else _cuda(choice_bias, "choice_bias", torch.float32)
    if bias is not None and tuple(bias.shape) != (E,):
        raise ValueError(f"choice_bias of shape {tuple(bias.shape)} for {E} experts")
    _same_device(logits.device, choice_bias=bias)
    slots = max(int(top_k), 0)
    idx = torch.empty((T, slots), dtype=torch.int64, device=logits.device)
    w = torch.empty((T, slots), dtype=torch.float32, device=logits.device)
    _run(logits.device, "mirai_route_groups", logits.data_ptr(), _DTYPE_CODES[logits.dtype], T, E, top_k, num_groups,
         top_groups, GROUP_SCORES[group_score], score, None if bias is None else bias.data_ptr(), mode, route_scale,
         idx.data_ptr(), w.data_ptr())
    return idx, w


def route_groups_backward(grad_weights: torch.Tensor, logits: torch.Tensor, top_indices: torch.Tensor, *,
                          score_func: str = "sigmoid", norm: str = "eps", route_scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route_groups``' weights with respect to the logits, [T, E] in
    the logits' dtype, from the gradient of the weights fp32 [T, k] and the
    chosen ids (the choice itself carries no gradient; the bias neither)."""
    score, mode = _route_options(score_func, norm)
    logits = _route_logits(logits)
    idx = _cuda(top_indices, "top_indices", torch.int64)
    gw = _cuda(grad_weights, "grad_weights", torch.float32)
    T, E = logits.shape
    if idx.ndim != 2 or idx.shape[0] != T or gw.shape != idx.shape:
        raise ValueError(f"grad_weights {tuple(gw.shape)} and top_indices {tuple(idx.shape)} for {T} tokens")
    _same_device(logits.device, grad_weights=gw, top_indices=idx)
    grad = torch.empty_like(logits)
    _run(logits.device, "mirai_route_groups_backward", gw.data_ptr(), logits.data_ptr(), _DTYPE_CODES[logits.dtype],
         idx.data_ptr(), T, E, idx.shape[1], score, mode, route_scale, grad.data_ptr())
    return grad


# ----------------------------------------------------------------------------- a2

@dataclass(frozen=True)
class DispatchPlan:
    """Device-resident routing layout (dispatch_preprocess.py:22-40)."""

    counts: torch.Tensor                # [E] int64
    starts: torch.Tensor                # [E] int64
    offsets: torch.Tensor               # [E] int32 inclusive cumsum
    sort_positions: torch.Tensor        # [S] int64
    sorted_token_indices: torch.Tensor  # [S] int64
    inverse_order: torch.Tensor         # [S] int64
    total_slots: int
    top_k: int


def dispatch_plan(top_indices: torch.Tensor, num_experts: int,
                  workspace: torch.Tensor | None = None) -> DispatchPlan:
    top_indices = _cuda(top_indices, "top_indices", torch.int64)
    T, k = top_indices.shape
    S = T * k
    dev = top_indices.device
    counts = torch.empty(num_experts, dtype=torch.int64, device=dev)
    starts = torch.empty(num_experts, dtype=torch.int64, device=dev)
    offsets = torch.empty(num_experts, dtype=torch.int32, device=dev)
    sp = torch.empty(S, dtype=torch.int64, device=dev)
    st = torch.empty(S, dtype=torch.int64, device=dev)
    inv = torch.empty(S, dtype=torch.int64, device=dev)
    need = plan_workspace_bytes(T, k, num_experts)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    _lib.call("mirai_dispatch_plan", _ptr(top_indices), T, k, num_experts, _ptr(counts), _ptr(starts),
              _ptr(offsets), _ptr(sp), _ptr(st), _ptr(inv), _ptr(workspace),
              workspace.numel() * workspace.element_size(), _stream())
    return DispatchPlan(counts, starts, offsets, sp, st, inv, S, k)


def plan_workspace_bytes(num_tokens: int, top_k: int, num_experts: int) -> int:
    return int(_lib.load().mirai_dispatch_plan_workspace_bytes(num_tokens, top_k, num_experts))


# ----------------------------------------------------------------------------- a3

def permute_rows(tokens: torch.Tensor, sorted_token_indices: torch.Tensor,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    tokens = _cuda(tokens, "tokens", torch.bfloat16)
    idx = _cuda(sorted_token_indices, "sorted_token_indices", torch.int64)
    S = idx.numel()
    H = tokens.shape[1]
    if out is None:
        out = torch.empty((S, H), dtype=torch.bfloat16, device=tokens.device)
    _lib.call("mirai_permute_rows_bf16", _ptr(tokens), tokens.shape[0], _ptr(idx), S, H, _ptr(out), _stream())
    return out


# ----------------------------------------------------------------------------- weight descriptors

class NF4Tensor:
    """Device buffers of one NF4 grouped-expert key, in the reference's layout
    (experts.py:998-1031): ``packed`` uint8 [E, out*in/2(, 1)], ``absmax`` uint8
    [E, out*in/64], ``nested_absmax`` fp32 [E, n], ``offset`` fp32 [E],
    ``code`` fp32 [16], ``nested_code`` fp32 [256]."""

    def __init__(self, packed, absmax, nested_absmax, offset, code, nested_code, shape,
                 blocksize: int = 64, nested_blocksize: int = 256):
        self.packed = _cuda(packed, "packed", torch.uint8)
        self.absmax = _cuda(absmax, "absmax", torch.uint8)
        self.nested_absmax = _cuda(nested_absmax, "nested_absmax", torch.float32)
        self.offset = _cuda(offset.reshape(-1), "offset", torch.float32)
        self.code = _cuda(code, "code", torch.float32)
        self.nested_code = _cuda(nested_code, "nested_code", torch.float32)
        self.shape = tuple(int(s) for s in shape)
        self.blocksize = int(blocksize)
        self.nested_blocksize = int(nested_blocksize)
        self._struct = _lib.Nf4Weight(self.packed.data_ptr(), self.absmax.data_ptr(),
                                      self.nested_absmax.data_ptr(), self.offset.data_ptr(),
                                      self.code.data_ptr(), self.nested_code.data_ptr(),
                                      self.blocksize, self.nested_blocksize)

    def struct(self) -> _lib.Nf4Weight:
        return self._struct


class Int8Tensor:
    """Device buffers of one INT8 grouped-expert key: ``q`` int8 [E, out, in]
    and ``scale`` fp32 [E, out, 1] (experts.py:1382-1422).  ``group_size`` 0 is
    plain per-output-channel INT8 (q * s = W); a power of 4 is the reference's
    default block-Hadamard format (q * s = W H along groups of ``in``,
    quant.py:189-235), run by rotating activations (``rotate_rows``)."""

    def __init__(self, q, scale, group_size: int = 0):
        self.q = _cuda(q, "int8 weight", torch.int8)
        self.scale = _cuda(scale, "int8 scale", torch.float32)
        self.shape = tuple(int(s) for s in self.q.shape)
        self.group_size = int(group_size)
        if self.group_size and self.shape[-1] % self.group_size:
            raise ValueError(f"rotation group {self.group_size} does not divide in_features {self.shape[-1]}")
        self._struct = _lib.Int8Weight(self.q.data_ptr(), self.scale.data_ptr())

    def struct(self) -> _lib.Int8Weight:
        return self._struct


def nf4_quantize(weight: torch.Tensor, code: torch.Tensor, nested_code: torch.Tensor, *,
                 blocksize: int = 64, nested_blocksize: int = 256) -> NF4Tensor:
    """Quantise a [E, out, in] stack to NF4 on the GPU (experts.py:998-1031)."""
    w = _cuda(weight.to(torch.bfloat16), "weight")
    E, out_f, in_f = w.shape
    dev = w.device
    bpe = out_f * in_f // blocksize
    n_nested = -(-bpe // nested_blocksize)
    packed = torch.empty((E, out_f * in_f // 2, 1), dtype=torch.uint8, device=dev)
    absmax = torch.empty((E, bpe), dtype=torch.uint8, device=dev)
    nabs = torch.empty((E, n_nested), dtype=torch.float32, device=dev)
    offset = torch.empty((E,), dtype=torch.float32, device=dev)
    code = _cuda(code, "code", torch.float32)
    nested_code = _cuda(nested_code, "nested_code", torch.float32)
    need = int(_lib.load().mirai_nf4_quantize_workspace_bytes(E, out_f, in_f))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    _lib.call("mirai_nf4_quantize", _ptr(w), E, out_f, in_f, _ptr(code), _ptr(nested_code), blocksize,
              nested_blocksize, _ptr(packed), _ptr(absmax), _ptr(nabs), _ptr(offset), _ptr(ws), need, _stream())
    return NF4Tensor(packed, absmax, nabs, offset, code, nested_code, (E, out_f, in_f), blocksize, nested_blocksize)


def nf4_dequantize(w: NF4Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [E, out, in] of an NF4 key (quant.py:380-434), bit-identical to the
    values the grouped GEMMs decode in their main loops."""
    E, out_f, in_f = w.shape
    if out is None:
        out = torch.empty((E, out_f, in_f), dtype=torch.bfloat16, device=w.packed.device)
    _cuda(out, "out", torch.bfloat16)
    _lib.call("mirai_nf4_dequantize", _ptr(w.packed), _ptr(w.absmax), _ptr(w.nested_absmax), _ptr(w.offset),
              _ptr(w.code), _ptr(w.nested_code), E, out_f, in_f, w.blocksize, w.nested_blocksize, _ptr(out),
              _stream())
    return out


def int8_quantize(weight: torch.Tensor, group_size: int = 0) -> Int8Tensor:
    """Symmetric per-output-channel INT8 of a [E, out, in] stack (quant.py:189-235).

    ``group_size`` > 0 first rotates each row's groups of that many input
    features by the block-Hadamard matrix, in fp32 (the reference's default
    format); codes can differ from the reference's by one step where the
    rotated value lies on a rounding boundary (the rotation's fp32 sums are
    ordered differently from a matrix product)."""
    w = _cuda(weight, "weight")
    if w.dtype not in (torch.float32, torch.bfloat16):
        w = w.float()
    *lead, in_f = w.shape
    rows = w.numel() // in_f
    if group_size:
        w = rotate_rows(w.float().reshape(rows, in_f), group_size, out_dtype=torch.float32).reshape(w.shape)
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    s = torch.empty((*lead, 1), dtype=torch.float32, device=w.device)
    _lib.call("mirai_int8_quantize_rows", _ptr(w), 1 if w.dtype == torch.float32 else 0, rows, in_f, _ptr(q),
              _ptr(s), _stream())
    return Int8Tensor(q, s, group_size)


_DTYPE_CODES = {torch.bfloat16: 0, torch.float32: 1}


def rotate_rows(x: torch.Tensor, group: int, *, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x H along every ``group``-wide block of the last dimension (H the
    block-Hadamard matrix of quant.py:103-122; H = H^T = H^-1), computed in
    fp32; bf16 or fp32 in and out.  ``out`` may be ``x`` itself."""
    x = _cuda(x, "x")
    if x.dtype not in _DTYPE_CODES:
        raise TypeError(f"rotate_rows takes bf16 or fp32, got {x.dtype}")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    _lib.call("mirai_rotate_rows", _ptr(x), _DTYPE_CODES[x.dtype], rows, cols, int(group), _ptr(out),
              _DTYPE_CODES[out.dtype], _stream())
    return out


def swiglu_backward_rotated(dh_raw: torch.Tensor, gate_up: torch.Tensor, group: int) -> torch.Tensor:
    """grad_gate_up [S, 2I] = SwiGLU backward of the saved (gate, up) given
    dh = rotate(dh_raw): the down projection's input gradient in the rotated
    INT8 format (dh_raw = grad_y (q s) from ``down_dh``)."""
    dh_raw = _cuda(dh_raw, "dh", torch.bfloat16)
    gate_up = _cuda(gate_up, "gate_up", torch.bfloat16)
    S, I = dh_raw.shape
    dgu = torch.empty((S, 2 * I), dtype=torch.bfloat16, device=dh_raw.device)
    _lib.call("mirai_swiglu_backward_rotated", _ptr(dh_raw), _ptr(gate_up), S, I, int(group), _ptr(dgu), _stream())
    return dgu


# ----------------------------------------------------------------------------- MXFP4

MXFP4_BLOCK = 32
_MXFP4_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 3}


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:  # (a tensor or an Mxfp4Rows)
            raise ValueError(f"{name} is on {t.device}, the call runs on {device}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` at a 32-byte aligned address (a copy when a view starts elsewhere)."""
    return t if t.data_ptr() % 32 == 0 else t.clone()


def _tiles(rows: int, width: int) -> tuple[int, int]:
    return -(-rows // 128), -(-width // 128)


def mxfp4_scale_tiles(scale: torch.Tensor) -> torch.Tensor:
    """Scale bytes uint8 [E, out, in/32] (the row order of MX checkpoints) in the
    tile order the kernels read: [E, ceil(out/128), ceil(in/128), 512]."""
    if scale.dtype != torch.uint8 or scale.ndim != 3:
        raise ValueError(f"scale bytes must be uint8 [E, out, in/32], got {scale.dtype} {tuple(scale.shape)}")
    E, out_f, blocks = scale.shape
    rt, kt = _tiles(out_f, blocks * MXFP4_BLOCK)
    full = scale.new_zeros((E, rt * 128, kt * 4))
    full[:, :out_f, :blocks] = scale
    return full.view(E, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, rt, kt, 512)


def mxfp4_scale_rows(tiles: torch.Tensor, out_features: int, in_features: int) -> torch.Tensor:
    """The inverse of ``mxfp4_scale_tiles``: scale bytes [E, out, in/32]."""
    E, rt, kt, _ = tiles.shape
    rows = tiles.view(E, rt, kt, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, rt * 128, kt * 4)
    return rows[:, :out_features, :in_features // MXFP4_BLOCK].contiguous()


class Mxfp4Tensor:
    """Device buffers of one MXFP4 grouped-expert key [E, out, in]: ``packed``
    uint8 [E, out, in/2] (two E2M1 codes per byte, the first element in the low
    half) and ``scale`` uint8 [E, ceil(out/128), ceil(in/128), 512], a
    power-of-two exponent byte per 32 elements of a row, in tiles
    (``mxfp4_scale_tiles`` makes them of a checkpoint's [E, out, in/32])."""

    def __init__(self, packed: torch.Tensor, scale: torch.Tensor):
        packed = _aligned(_cuda(packed, "packed", torch.uint8))
        scale = _aligned(_cuda(scale, "scale", torch.uint8))
        if packed.ndim != 3 or packed.shape[2] % (MXFP4_BLOCK // 2) or 0 in packed.shape:
            raise ValueError(f"MXFP4 codes must be [E, out, in/2] with in % 32 == 0, got {tuple(packed.shape)}")
        E, out_f, half = packed.shape
        want = (E, *_tiles(out_f, 2 * half), 512)
        if tuple(scale.shape) != want:
            raise ValueError(f"MXFP4 scale tiles of shape {tuple(scale.shape)}: {E} x {out_f} x {2 * half} needs {want}")
        _same_device(packed.device, scale=scale)
        self._bind(packed, scale)

    def _bind(self, packed: torch.Tensor, scale: torch.Tensor) -> "Mxfp4Tensor":
        self.packed, self.scale, self.device = packed, scale, packed.device
        self.shape = (packed.shape[0], packed.shape[1], 2 * packed.shape[2])
        self._struct = _lib.Mxfp4Weight(packed.data_ptr(), scale.data_ptr())
        return self

    def struct(self) -> _lib.Mxfp4Weight:
        return self._struct


class Mxfp4Rows:
    """Activation rows [S, width] in MXFP4, grouped in ``segments`` segments (one
    per expert, or per source and expert): ``packed`` uint8 [S, width/2] and
    ``scale`` uint8 [tiles, ceil(width/128), 512], whose row tiles restart at
    every segment.  Made by ``mxfp4_quantize_rows`` or ``gateup_swiglu(...,
    quantize=True)``, taken by ``gateup_swiglu`` / ``down`` with the same offsets."""

    def __init__(self, packed: torch.Tensor, scale: torch.Tensor, segments: int):
        self.packed = _cuda(packed, "packed", torch.uint8)
        self.scale = _cuda(scale, "scale", torch.uint8)
        if self.packed.ndim != 2 or self.packed.shape[1] == 0 or self.packed.shape[1] % (MXFP4_BLOCK // 2):
            raise ValueError(f"MXFP4 rows must be [S, width/2] with width % 32 == 0, got {tuple(self.packed.shape)}")
        self.segments = int(segments)
        self.shape = (self.packed.shape[0], 2 * self.packed.shape[1])
        self.device = self.packed.device
        need = self.scale_bytes(*self.shape, self.segments)
        if self.segments < 1 or self.scale.numel() < need:
            raise ValueError(f"{self.shape[0]} rows of {self.shape[1]} in {self.segments} segments need {need} scale "
                             f"bytes, got {self.scale.numel()}")
        _same_device(self.device, scale=self.scale)
        if self.packed.data_ptr() % 16 or self.scale.data_ptr() % 16:
            raise ValueError("MXFP4 rows must start 16-byte aligned")

    @staticmethod
    def scale_bytes(rows: int, width: int, segments: int) -> int:
        """mirai_mxfp4_rows_scale_bytes: every segment can end inside a row tile."""
        return (rows // 128 + min(rows, segments)) * _tiles(0, width)[1] * 512

    @classmethod
    def empty(cls, rows: int, width: int, segments: int, device) -> "Mxfp4Rows":
        r = cls.__new__(cls)
        kt = _tiles(0, width)[1]
        r.packed = torch.empty((rows, width // 2), dtype=torch.uint8, device=device)
        r.scale = torch.empty((rows // 128 + min(rows, segments), kt, 512), dtype=torch.uint8, device=device)
        r.segments, r.shape, r.device = segments, (rows, width), device
        return r


def mxfp4_quantize(weight: torch.Tensor) -> Mxfp4Tensor:
    """Quantise a [E, out, in] stack (bf16, fp32 or fp16) to MXFP4: per 32 elements
    of a row the scale 2^(floor(log2 max|x|) - 2), elements rounded to the
    nearest E2M1 value (ties to even, saturating).  A block holding an infinity
    or a NaN reads back as NaN."""
    w = _aligned(_cuda(weight, "weight"))
    if w.dtype not in _MXFP4_DTYPES:
        raise TypeError(f"mxfp4_quantize takes bf16, fp32 or fp16, got {w.dtype}")
    if w.ndim != 3 or 0 in w.shape or w.shape[2] % MXFP4_BLOCK:
        raise ValueError(f"mxfp4_quantize takes [E, out, in] with in % 32 == 0, got {tuple(w.shape)}")
    E, out_f, in_f = w.shape
    packed = torch.empty((E, out_f, in_f // 2), dtype=torch.uint8, device=w.device)
    scale = torch.empty((E, *_tiles(out_f, in_f), 512), dtype=torch.uint8, device=w.device)
    _run(w.device, "mirai_mxfp4_quantize", w.data_ptr(), _MXFP4_DTYPES[w.dtype], E, out_f, in_f, packed.data_ptr(),
         scale.data_ptr())
    return Mxfp4Tensor.__new__(Mxfp4Tensor)._bind(packed, scale)


def mxfp4_dequantize(w: Mxfp4Tensor, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [E, out, in] values of an MXFP4 key, exact in bf16 and fp32 (fp16: rounded
    to nearest)."""
    if not isinstance(w, Mxfp4Tensor):
        raise TypeError(f"mxfp4_dequantize reads an Mxfp4Tensor, not {type(w)}")
    if out is None:
        if out_dtype not in _MXFP4_DTYPES:
            raise TypeError(f"mxfp4_dequantize writes bf16, fp32 or fp16, not {out_dtype}")
        out = torch.empty(w.shape, dtype=out_dtype, device=w.device)
    elif out.dtype not in _MXFP4_DTYPES or tuple(out.shape) != w.shape or not out.is_contiguous() or out.data_ptr() % 32:
        raise ValueError(f"out must be a contiguous, 32-byte aligned {w.shape} tensor of bf16, fp32 or fp16, got "
                         f"{out.dtype} {tuple(out.shape)}")
    _same_device(w.device, out=out)
    E, out_f, in_f = w.shape
    _run(w.device, "mirai_mxfp4_dequantize", w.packed.data_ptr(), w.scale.data_ptr(), E, out_f, in_f, out.data_ptr(),
         _MXFP4_DTYPES[out.dtype])
    return out


def mxfp4_quantize_rows(x: torch.Tensor, offsets: torch.Tensor, row_index: torch.Tensor | None = None) -> Mxfp4Rows:
    """bf16 rows [S, width] of the segments ``offsets`` ends (int32), quantised for
    the expert products.  ``row_index`` int64 [S]: row s is x[row_index[s]] (the
    permute in the same pass).  Rows past the last segment are not written."""
    x = _aligned(_cuda(x, "x", torch.bfloat16))
    offsets = _cuda(offsets, "offsets", torch.int32)
    if x.ndim != 2 or x.shape[1] % MXFP4_BLOCK or x.shape[1] == 0:
        raise ValueError(f"mxfp4_quantize_rows takes [rows, width] with width % 32 == 0, got {tuple(x.shape)}")
    index = None if row_index is None else _cuda(row_index, "row_index", torch.int64)
    _same_device(x.device, offsets=offsets, row_index=index)
    S = x.shape[0] if index is None else index.numel()
    rows = Mxfp4Rows.empty(S, x.shape[1], offsets.numel(), x.device)
    _run(x.device, "mirai_mxfp4_quantize_rows", x.data_ptr(), x.shape[0], None if index is None else index.data_ptr(),
         offsets.data_ptr(), offsets.numel(), S, x.shape[1], rows.packed.data_ptr(), rows.scale.data_ptr())
    return rows


def _mxfp4_rows(x, offsets: torch.Tensor, width: int, name: str) -> Mxfp4Rows:
    rows = x if isinstance(x, Mxfp4Rows) else mxfp4_quantize_rows(x, offsets)
    if rows.shape[1] != width or rows.segments != offsets.numel():
        raise ValueError(f"{name} of width {rows.shape[1]} in {rows.segments} segments: the call needs width {width} in "
                         f"{offsets.numel()}")
    return rows


# bf16 rows are quantised inside the product (few_rows_kernel in mxfp4.cu) up to this many, and up to 16
# rows per segment (1024 at most).  Measured, gate/up, us, quantise + product against it (cold L2):
#   H 2048, I 1408    1 expert: 256 rows 27.6 / 19.4, 512 rows 27.6 / 28.7;  8: 256 rows 31.7 / 20.5, 1024 rows 33.8 / 41.0
#                     32: 512 rows 48.1 / 41.0, 1024 rows 52.2 / 49.2;     128: 256 rows 103 / 87, 1024 rows 106 / 90
#   H 4096, I 1536    1: 256 rows 37.9 / 26.6, 512 rows 37.9 / 45.1;       32: 512 rows 74.7 / 68.6;  128: 1024 rows 181 / 170
#   H 1024, I 512     every case up to 1024 rows is faster in one launch (1 expert: 1024 rows 21.5 / 16.4)
# down has half the weights per tile in flight, so that many experts stream better through the general
# product: it takes up to MXFP4_FEW_ROWS rows on up to 64 segments that can have rows.
#   H 2048, I 1408    1: 256 rows 25.6 / 16.4;  32: 256 rows 29.7 / 26.6, 512 rows 31.7 / 32.8;  128: 64 rows 44.0 / 41.0, 128 rows 62.5 / 69.6
#   H 4096, I 1536    1: 256 rows 25.6 / 22.5;  32: 256 rows 42.0 / 43.0;  128: 32 rows 42.0 / 41.0, 64 rows 64.5 / 69.6, 128 rows 99 / 123
MXFP4_FEW_ROWS = 256
MXFP4_FEW_ROWS_PER_SEGMENT = 16
MXFP4_FEW_DOWN_SEGMENTS = 64
_FEW_MAX_ROWS, _FEW_MAX_WIDTH = 1024, 4096


def _few_limit(segments: int) -> int:
    return min(_FEW_MAX_ROWS, max(MXFP4_FEW_ROWS, MXFP4_FEW_ROWS_PER_SEGMENT * segments))


def _few_rows(x, width: int, segments: int) -> bool:
    return isinstance(x, torch.Tensor) and width <= _FEW_MAX_WIDTH and x.shape[0] <= _few_limit(segments)


def _few_rows_down(x, width: int, segments: int) -> bool:
    return (_few_rows(x, width, segments) and x.shape[0] <= MXFP4_FEW_ROWS
            and min(x.shape[0], segments) <= MXFP4_FEW_DOWN_SEGMENTS)


def _few_input(x: torch.Tensor, width: int, name: str) -> torch.Tensor:
    x = _aligned(_cuda(x, name, torch.bfloat16))
    if x.ndim != 2 or x.shape[1] != width:
        raise ValueError(f"{name} of shape {tuple(x.shape)}: the call needs [rows, {width}]")
    return x


def _mxfp4_output(out: torch.Tensor | None, shape: tuple, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or tuple(out.shape) != shape or not out.is_contiguous() or out.device != device:
        raise ValueError(f"out must be a contiguous bf16 {shape} tensor on {device}, got {out.dtype} "
                         f"{tuple(out.shape)} on {out.device}")
    return out


def _gateup_mxfp4(x, offsets: torch.Tensor, w1: Mxfp4Tensor, w3: Mxfp4Tensor, *, inter: int, save_gate_up: bool,
                  want_h: bool, want_rows: bool, out: torch.Tensor | None = None, sources: int = 1,
                  gate_up_dtype: torch.dtype = torch.bfloat16):
    """(h or None, gate_up or None, quantised h or None)."""
    if gate_up_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"gate/up is saved in bf16 or fp32, not {gate_up_dtype}")
    save_code = _MXFP4_DTYPES[gate_up_dtype]
    if not isinstance(w1, Mxfp4Tensor) or not isinstance(w3, Mxfp4Tensor) or w1.shape != w3.shape:
        raise TypeError("gate/up in MXFP4 needs two Mxfp4Tensor keys of one shape")
    E, out_f, hidden = w1.shape
    offsets = _cuda(offsets, "offsets", torch.int32)
    if out_f != inter or offsets.numel() != sources * E:
        raise ValueError(f"keys of {E} experts x {out_f} channels: the call has inter {inter} and {offsets.numel()} "
                         f"segments of {sources} source(s)")
    device = w1.device
    _same_device(device, x=x, offsets=offsets, w3=w3)
    if not want_rows and _few_rows(x, hidden, offsets.numel()):
        x = _few_input(x, hidden, "x_sorted")
        S = x.shape[0]
        h = _mxfp4_output(out, (S, inter), device)
        gu = torch.empty((S, 2 * inter), dtype=gate_up_dtype, device=device) if save_gate_up else None
        _run(device, "mirai_moe_gateup_swiglu_mxfp4_few_save", x.data_ptr(), offsets.data_ptr(), sources, E, S, hidden,
             inter, w1.struct(), w3.struct(), h.data_ptr(), None if gu is None else gu.data_ptr(), save_code)
        return h, gu, None
    rows = _mxfp4_rows(x, offsets, hidden, "x_sorted")
    S = rows.shape[0]
    h = _mxfp4_output(out, (S, inter), device) if want_h else None
    gu = torch.empty((S, 2 * inter), dtype=gate_up_dtype, device=device) if save_gate_up else None
    hq = Mxfp4Rows.empty(S, inter, offsets.numel(), device) if want_rows else None
    _run(device, "mirai_moe_gateup_swiglu_mxfp4_save", rows.packed.data_ptr(), rows.scale.data_ptr(), offsets.data_ptr(),
         sources, E, S, hidden, inter, w1.struct(), w3.struct(), None if h is None else h.data_ptr(),
         None if gu is None else gu.data_ptr(), save_code, None if hq is None else hq.packed.data_ptr(),
         None if hq is None else hq.scale.data_ptr())
    return h, gu, hq


def _check_rank_rows(low: torch.Tensor, rows: int) -> None:
    if tuple(low.shape) != (rows, 64) or low.dtype != torch.bfloat16 or not low.is_contiguous():
        raise ValueError(f"rank_a must be contiguous bf16 [{rows}, 64], got {low.dtype} {tuple(low.shape)}")


def _down_mxfp4(h, offsets: torch.Tensor, w2: Mxfp4Tensor, *, hidden: int, out: torch.Tensor | None,
                lora: "DownLoRA | None", rank_a: torch.Tensor | None, sources: int) -> torch.Tensor:
    E, out_f, inter = w2.shape
    offsets = _cuda(offsets, "offsets", torch.int32)
    if out_f != hidden or offsets.numel() != sources * E:
        raise ValueError(f"a key of {E} experts x {out_f} rows: the call has hidden {hidden} and {offsets.numel()} "
                         f"segments of {sources} source(s)")
    device = w2.device
    _same_device(device, h=h, offsets=offsets, rank_a=rank_a)
    if lora is None and _few_rows_down(h, inter, offsets.numel()):
        h = _few_input(h, inter, "h")
        y = _mxfp4_output(out, (h.shape[0], hidden), device)
        _run(device, "mirai_moe_down_mxfp4_few", h.data_ptr(), offsets.data_ptr(), sources, E, h.shape[0], inter, hidden,
             w2.struct(), y.data_ptr())
        return y
    low = rank_b = None
    if lora is not None:
        if rank_a is None and isinstance(h, Mxfp4Rows):
            raise ValueError("a LoRA adapter on quantised rows needs rank_a, its projection of the bf16 rows")
        low = rank_a if rank_a is not None else lora_project(h, offsets, lora, forward=True, sources=sources)
        _check_rank_rows(low, h.shape[0])
        rank_b = lora.b_pad()
        if rank_b.shape[0] != E * hidden:
            raise ValueError(f"the adapter's B has {rank_b.shape[0]} rows, the key {E} x {hidden}")
        _same_device(device, lora=rank_b)
    rows = _mxfp4_rows(h, offsets, inter, "h")
    S = rows.shape[0]
    y = _mxfp4_output(out, (S, hidden), device)
    _run(device, "mirai_moe_down_mxfp4", rows.packed.data_ptr(), rows.scale.data_ptr(), offsets.data_ptr(), sources, E, S,
         inter, hidden, w2.struct(), None if low is None else low.data_ptr(),
         None if rank_b is None else rank_b.data_ptr(), y.data_ptr())
    return y


class Mxfp4ReadBack:
    """An MXFP4 key with its values read back to bf16 (``mxfp4_read_back``): ``down_dx`` and
    ``gateup_dx`` take it for the key, and several calls on it decode it once."""

    def __init__(self, key: Mxfp4Tensor):
        self.key, self.shape, self.device = key, key.shape, key.device
        self.dense = mxfp4_dequantize(key)


def mxfp4_read_back(weights) -> tuple:
    """``weights`` for a backward pass of several calls: MXFP4 keys as ``Mxfp4ReadBack`` (2 bytes per
    weight while they are kept), others as given."""
    return tuple(Mxfp4ReadBack(w) if isinstance(w, Mxfp4Tensor) else w for w in weights)


def _dx_weight(w):
    """The weight a dX product multiplies: an MXFP4 key is read back (the scales run
    along the other axis than dX reduces over), others as given."""
    if isinstance(w, Mxfp4ReadBack):
        return w.dense
    return mxfp4_dequantize(w) if isinstance(w, Mxfp4Tensor) else w


def _group(w) -> int:
    return int(getattr(w, "group_size", 0) or 0)


def _as_weight(w):
    if isinstance(w, (NF4Tensor, Int8Tensor)):
        return w.struct()
    return w


# ----------------------------------------------------------------------------- a6 / a7

def gateup_swiglu(x_sorted: torch.Tensor, offsets: torch.Tensor, w1, w3, *, inter: int,
                  save_gate_up: bool = False, out: torch.Tensor | None = None, sources: int = 1,
                  quantize: bool = False, gate_up_dtype: torch.dtype = torch.bfloat16):
    """h = silu(x W1^T) * (x W3^T) per expert segment.  ``w1``/``w3`` are bf16
    tensors [E, I, H], or ``Nf4Weight`` / ``Int8Weight`` descriptors.
    ``sources`` > 1: ``offsets`` ends ``sources * E`` source-major segments
    (segment s*E + e = source s's rows for expert e).

    ``Mxfp4Tensor`` keys multiply the rows in MXFP4 too: ``x_sorted`` is bf16
    (quantised here) or ``Mxfp4Rows``; silu(g) * u is formed in fp32 and rounded
    once, and ``quantize=True`` returns h as the ``Mxfp4Rows`` that ``down``
    takes instead of bf16.  ``gate_up_dtype=torch.float32`` saves the gate/up
    accumulators themselves, which ``down_dx`` takes as well."""
    if isinstance(w1, Mxfp4Tensor) or isinstance(w3, Mxfp4Tensor):
        if quantize and out is not None:
            raise ValueError("quantize=True returns Mxfp4Rows: it writes no bf16 out")
        h, gu, hq = _gateup_mxfp4(x_sorted, offsets, w1, w3, inter=inter, save_gate_up=save_gate_up,
                                  want_h=not quantize, want_rows=quantize, out=out, sources=sources,
                                  gate_up_dtype=gate_up_dtype)
        h = hq if quantize else h
        return (h, gu) if save_gate_up else h
    if quantize:
        raise TypeError("quantize=True needs MXFP4 keys")
    if gate_up_dtype != torch.bfloat16:
        raise TypeError(f"gate/up saved in {gate_up_dtype} needs MXFP4 keys")
    w1, w3 = _as_weight(w1), _as_weight(w3)
    x_sorted = _cuda(x_sorted, "x_sorted", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, H = x_sorted.shape
    h = out if out is not None else torch.empty((S, inter), dtype=torch.bfloat16, device=x_sorted.device)
    gu = torch.empty((S, 2 * inter), dtype=torch.bfloat16, device=x_sorted.device) if save_gate_up else None
    if sources > 1:
        if offsets.numel() % sources:
            raise ValueError("source-major segments: offsets must be a multiple of sources")
        E = offsets.numel() // sources
        _lib.call(f"mirai_moe_gateup_swiglu_src_{_fmt_suffix(w1)}", _ptr(x_sorted), _ptr(offsets), sources, E, S, H,
                  inter, _wptr(w1), _wptr(w3), _ptr(h), _ptr(gu), _stream())
        return (h, gu) if save_gate_up else h
    E = offsets.numel()
    if isinstance(w1, torch.Tensor):
        w1 = _cuda(w1, "w1", torch.bfloat16)
        w3 = _cuda(w3, "w3", torch.bfloat16)
        _lib.call("mirai_moe_gateup_swiglu_bf16", _ptr(x_sorted), _ptr(offsets), E, S, H, inter, _ptr(w1),
                  _ptr(w3), _ptr(h), _ptr(gu), _stream())
    elif isinstance(w1, _lib.Nf4Weight):
        _lib.call("mirai_moe_gateup_swiglu_nf4", _ptr(x_sorted), _ptr(offsets), E, S, H, inter, w1, w3, _ptr(h),
                  _ptr(gu), _stream())
    elif isinstance(w1, _lib.Int8Weight):
        _lib.call("mirai_moe_gateup_swiglu_int8", _ptr(x_sorted), _ptr(offsets), E, S, H, inter, w1, w3, _ptr(h),
                  _ptr(gu), _stream())
    else:
        raise TypeError(f"unsupported weight type {type(w1)}")
    return (h, gu) if save_gate_up else h


def down(h: torch.Tensor, offsets: torch.Tensor, w2, *, hidden: int, out: torch.Tensor | None = None,
         lora: "DownLoRA | None" = None, rank_a: torch.Tensor | None = None, sources: int = 1):
    """y = h W2^T per expert segment (+ the fused LoRA rank block when ``lora``;
    ``rank_a`` is its [S, 64] projection of h when the caller already has it).
    ``sources`` > 1: source-major segments as in ``gateup_swiglu``.  With an
    ``Mxfp4Tensor`` key, ``h`` is bf16 (quantised here) or ``Mxfp4Rows``."""
    if isinstance(w2, Mxfp4Tensor):
        return _down_mxfp4(h, offsets, w2, hidden=hidden, out=out, lora=lora, rank_a=rank_a, sources=sources)
    w2 = _as_weight(w2)
    h = _cuda(h, "h", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, I = h.shape
    y = out if out is not None else torch.empty((S, hidden), dtype=torch.bfloat16, device=h.device)
    if sources > 1:
        if offsets.numel() % sources:
            raise ValueError("source-major segments: offsets must be a multiple of sources")
        E = offsets.numel() // sources
        if lora is None:
            _lib.call(f"mirai_moe_down_src_{_fmt_suffix(w2)}", _ptr(h), _ptr(offsets), sources, E, S, I, hidden,
                      _wptr(w2), _ptr(y), _stream())
            return y
        low = rank_a if rank_a is not None else lora_project(h, offsets, lora, forward=True, sources=sources)
        _lib.call(f"mirai_moe_down_lora_src_{_fmt_suffix(w2)}", _ptr(h), _ptr(offsets), sources, E, S, I, hidden,
                  _wptr(w2), _ptr(low), _ptr(lora.b_pad()), _ptr(y), _stream())
        return y
    E = offsets.numel()
    if lora is None:
        _lib.call(f"mirai_moe_down_{_fmt_suffix(w2)}", _ptr(h), _ptr(offsets), E, S, I, hidden, _wptr(w2), _ptr(y),
                  _stream())
        return y
    low = rank_a if rank_a is not None else lora_project(h, offsets, lora, forward=True)
    _lib.call(f"mirai_moe_down_lora_{_fmt_suffix(w2)}", _ptr(h), _ptr(offsets), E, S, I, hidden, _wptr(w2),
              _ptr(low), _ptr(lora.b_pad()), _ptr(y), _stream())
    return y


_PAD_ATTR = "_mirai_lora_pads"


def _factor_pads(src: torch.Tensor) -> dict:
    """The padded kernel operands built from one adapter factor, kept on the
    factor tensor itself (the caller's parameter) so that they are built once
    per binding and rebuilt only when the factor changes: a moved version
    counter (an in-place optimizer step) or new storage drops them."""
    tag = (src._version, src.data_ptr())
    held = getattr(src, _PAD_ATTR, None)
    if held is None or held[0] != tag:
        held = (tag, {})
        try:
            setattr(src, _PAD_ATTR, held)
        except (AttributeError, RuntimeError):
            pass  # a tensor that takes no attributes gets pads for this call only
    return held[1]


class DownLoRA:
    """A LoRA adapter on the expert down projection (w2): y += scale (h A^T) B^T
    with A [E, r, I] and B [E, H, r] (active_expert_lora.py:43-116, 434-478)."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: float, *, compute_grads: bool = False):
        self._src_a, self._src_b = a, b
        self.a = _cuda(a.detach().to(torch.bfloat16), "lora_a")
        self.b = _cuda(b.detach().to(torch.bfloat16), "lora_b")
        # when set, moe_backward_dx also fills grad_a [E, r, I] / grad_b [E, H, r] (fp32)
        self.compute_grads = bool(compute_grads)
        self.grad_a: torch.Tensor | None = None
        self.grad_b: torch.Tensor | None = None
        E, r, I = self.a.shape
        if tuple(self.b.shape[::2]) != (E, r) or r > 32:
            raise ValueError(f"LoRA factors must be A [E, r, I] and B [E, H, r] with r <= 32, got "
                             f"{tuple(self.a.shape)} and {tuple(self.b.shape)}")
        self.rank = int(r)
        self.scale = float(scale)

    def b_pad(self) -> torch.Tensor:
        """B zero-padded to [E*H, 64]: the K-major rank-block operand of the
        down GEMM.  Built once per value of the factor."""
        pads = _factor_pads(self._src_b)
        if "b" not in pads:
            E, H, r = self.b.shape
            pad = torch.zeros((E, H, 64), dtype=torch.bfloat16, device=self.b.device)
            pad[:, :, :r] = self.b
            pads["b"] = pad.reshape(E * H, 64)
        return pads["b"]

    def a_pad(self, rotation: int = 0) -> torch.Tensor:
        """A zero-padded to [E*64, I]: the MN-major rank-block operand of the
        down dX GEMM; with ``rotation`` > 0 each row rotated by the
        block-Hadamard matrix of that group size (A H), for the rotated INT8
        format whose dh is rotated after the GEMM (H H = 1).  Built once per
        value of the factor and group."""
        pads = _factor_pads(self._src_a)
        key = ("a", int(rotation))
        if key not in pads:
            E, r, I = self.a.shape
            pad = torch.zeros((E, 64, I), dtype=torch.bfloat16, device=self.a.device)
            pad[:, :r, :] = self.a
            pad = pad.reshape(E * 64, I)
            if rotation:
                pad = rotate_rows(pad, rotation)
            pads[key] = pad
        return pads[key]


LORA_FACTOR_ROWS, LORA_FACTOR_COLS = 0, 1


def lora_project(x: torch.Tensor, offsets: torch.Tensor, lora: DownLoRA, *, forward: bool,
                 sources: int = 1) -> torch.Tensor:
    """[S, 64] bf16 rank-block operand bf16(scale * x F_e^T), zero past the rank:
    F = A ([E, r, I], x = h) when ``forward``, else B^T ([E, H, r], x = grad_y).
    ``sources`` > 1: source-major segments (offsets [sources * E])."""
    x = _cuda(x, "x", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, K = x.shape
    out = torch.empty((S, 64), dtype=torch.bfloat16, device=x.device)
    factor, layout = (lora.a_pad(), LORA_FACTOR_ROWS) if forward else (lora.b_pad(), LORA_FACTOR_COLS)
    if offsets.numel() % sources:
        raise ValueError("source-major segments: offsets must be a multiple of sources")
    _lib.call("mirai_moe_lora_project_src", _ptr(x), _ptr(offsets), int(sources), offsets.numel() // sources, S, K,
              _ptr(factor), layout, int(lora.rank), float(lora.scale), _ptr(out), _stream())
    return out


# ----------------------------------------------------------------------------- a8

def combine(y_sorted: torch.Tensor, inverse_order: torch.Tensor, top_weights: torch.Tensor | None,
            out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
            top_k: int | None = None, bf16_accumulate: bool = False) -> torch.Tensor:
    """Weighted un-permute; ``top_weights=None`` sums the routes (permute backward).
    ``bf16_accumulate``: bf16 products summed in bf16, route by route (MAGI-2's
    index_add on bf16 tensors) instead of one fp32 sum.  ``y_sorted`` is bf16 or
    fp32 (summed in fp32)."""
    y_sorted = _cuda(y_sorted, "y_sorted")
    rows_f32 = y_sorted.dtype == torch.float32
    if not rows_f32 and y_sorted.dtype != torch.bfloat16 or rows_f32 and bf16_accumulate:
        raise TypeError(f"y_sorted must be torch.bfloat16 (or fp32 without bf16_accumulate), got {y_sorted.dtype}")
    inv = _cuda(inverse_order, "inverse_order", torch.int64)
    if top_weights is None:
        k = int(top_k)
        T = inv.numel() // k
        w = None
    else:
        w = _cuda(top_weights.float(), "top_weights", torch.float32)
        T, k = w.shape
    H = y_sorted.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=out_dtype, device=y_sorted.device)
    code = {torch.bfloat16: 0, torch.float32: 1}[out.dtype]
    if bf16_accumulate:
        if out.dtype != torch.bfloat16:
            raise TypeError("bf16 accumulation writes a bf16 output")
        code = COMBINE_BF16_ACCUM
    if rows_f32:
        _run(y_sorted.device, "mirai_moe_combine_f32", _ptr(y_sorted), _ptr(inv), _ptr(w), T, k, H, _ptr(out), code)
        return out
    _lib.call("mirai_moe_combine", _ptr(y_sorted), _ptr(inv), _ptr(w), T, k, H, _ptr(out), code, _stream())
    return out


def combine_backward(grad_out: torch.Tensor, y_sorted: torch.Tensor, inverse_order: torch.Tensor,
                     top_weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(grad_y_sorted bf16 [S, H], grad_weights fp32 [T, k]) (dispatch_ops.py:36-44)."""
    g = _cuda(grad_out.to(torch.bfloat16), "grad_out", torch.bfloat16)
    y_sorted = _cuda(y_sorted, "y_sorted", torch.bfloat16)
    inv = _cuda(inverse_order, "inverse_order", torch.int64)
    w = _cuda(top_weights.float(), "top_weights", torch.float32)
    T, k = w.shape
    H = y_sorted.shape[1]
    gy = torch.empty_like(y_sorted)
    gw = torch.empty((T, k), dtype=torch.float32, device=y_sorted.device)
    _lib.call("mirai_moe_combine_backward", _ptr(g), _ptr(y_sorted), _ptr(inv), _ptr(w), T, k, H, _ptr(gy),
              _ptr(gw), _stream())
    return gy, gw


def combine_backward_rows(grad_out: torch.Tensor, y_sorted: torch.Tensor, inverse_order: torch.Tensor,
                          top_weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``combine_backward`` without its rounding: (grad_rows bf16 [S, H], each route's row of
    ``grad_out`` as it is, row_weights fp32 [S], grad_weights fp32 [T, k]); grad_y_sorted is
    grad_rows * row_weights[:, None]."""
    g = _cuda(grad_out.to(torch.bfloat16), "grad_out", torch.bfloat16)
    y_sorted = _cuda(y_sorted, "y_sorted", torch.bfloat16)
    inv = _cuda(inverse_order, "inverse_order", torch.int64)
    w = _cuda(top_weights.float(), "top_weights", torch.float32)
    T, k = w.shape
    H = y_sorted.shape[1]
    if tuple(g.shape) != (T, H) or y_sorted.shape[0] != T * k or inv.numel() != T * k:
        raise ValueError(f"grad_out {tuple(g.shape)}, rows {tuple(y_sorted.shape)} and {inv.numel()} routes do not fit "
                         f"weights {tuple(w.shape)}")
    rows = torch.empty_like(y_sorted)
    rw = torch.empty(T * k, dtype=torch.float32, device=g.device)
    gw = torch.empty((T, k), dtype=torch.float32, device=g.device)
    _same_device(g.device, y_sorted=y_sorted, inverse_order=inv, top_weights=w)
    _run(g.device, "mirai_moe_combine_backward_rows", g.data_ptr(), y_sorted.data_ptr(), inv.data_ptr(), w.data_ptr(), T, k,
         H, rows.data_ptr(), rw.data_ptr(), gw.data_ptr())
    return rows, rw, gw


# ----------------------------------------------------------------------------- a9 dX

def _fmt_suffix(w) -> str:
    if isinstance(w, torch.Tensor):
        return "bf16"
    if isinstance(w, _lib.Nf4Weight):
        return "nf4"
    if isinstance(w, _lib.Int8Weight):
        return "int8"
    raise TypeError(f"unsupported weight type {type(w)}")


def _wptr(w):
    return _ptr(_cuda(w, "weight", torch.bfloat16)) if isinstance(w, torch.Tensor) else w


def down_dx(grad_y: torch.Tensor, offsets: torch.Tensor, w2, gate_up: torch.Tensor | None, *, inter: int,
            out: torch.Tensor | None = None, lora: DownLoRA | None = None,
            rank_a: torch.Tensor | None = None, sources: int = 1) -> torch.Tensor:
    """grad_gate_up [S, 2I] = SwiGLU backward of (gate, up) given dh = grad_y W2
    (+ the LoRA path's input gradient when ``lora``).  ``sources`` > 1:
    source-major segments (an expert owner's rows); there ``gate_up=None``
    returns dh [S, I] itself.  An ``Mxfp4Tensor`` key takes ``gate_up`` in bf16
    or fp32 (and needs it)."""
    if isinstance(w2, Mxfp4Tensor):
        return _down_dx_mxfp4(grad_y, offsets, w2, gate_up, inter=inter, out=out, lora=lora, rank_a=rank_a,
                              sources=sources)
    if isinstance(w2, Mxfp4ReadBack):
        return _down_dx_mxfp4(grad_y, offsets, w2.key, gate_up, inter=inter, out=out, lora=lora, rank_a=rank_a,
                              sources=sources, dense=w2.dense)
    group = getattr(w2, "group_size", 0)  # block-Hadamard INT8: the rotation group of dh
    w2 = _as_weight(w2)
    gy = _cuda(grad_y, "grad_y", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, H = gy.shape
    if sources > 1:
        if offsets.numel() % sources:
            raise ValueError("source-major segments: offsets must be a multiple of sources")
        E = offsets.numel() // sources
        gu = None if gate_up is None else _cuda(gate_up, "gate_up", torch.bfloat16)
        width = inter if gu is None else 2 * inter
        dgu = out if out is not None else torch.empty((S, width), dtype=torch.bfloat16, device=gy.device)
        if lora is None:
            _lib.call(f"mirai_moe_down_dx_src_{_fmt_suffix(w2)}", _ptr(gy), _ptr(offsets), sources, E, S, H, inter,
                      _wptr(w2), _ptr(gu), _ptr(dgu), _stream())
            return dgu
        glow = rank_a if rank_a is not None else lora_project(gy, offsets, lora, forward=False, sources=sources)
        # dh alone in the block-Hadamard INT8 format is rotated afterwards: its A factor is rotated too
        rot = group if gu is None else 0
        _lib.call(f"mirai_moe_down_dx_lora_src_{_fmt_suffix(w2)}", _ptr(gy), _ptr(offsets), sources, E, S, H, inter,
                  _wptr(w2), _ptr(gu), _ptr(glow), _ptr(lora.a_pad(rotation=rot)), _ptr(dgu), _stream())
        return dgu
    gu = _cuda(gate_up, "gate_up", torch.bfloat16)
    dgu = out if out is not None else torch.empty((S, 2 * inter), dtype=torch.bfloat16, device=gy.device)
    if lora is None:
        _lib.call(f"mirai_moe_down_dx_{_fmt_suffix(w2)}", _ptr(gy), _ptr(offsets), offsets.numel(), S, H, inter,
                  _wptr(w2), _ptr(gu), _ptr(dgu), _stream())
        return dgu
    glow = rank_a if rank_a is not None else lora_project(gy, offsets, lora, forward=False)
    _lib.call(f"mirai_moe_down_dx_lora_{_fmt_suffix(w2)}", _ptr(gy), _ptr(offsets), offsets.numel(), S, H, inter,
              _wptr(w2), _ptr(gu), _ptr(glow), _ptr(lora.a_pad()), _ptr(dgu), _stream())
    return dgu


def _down_dx_mxfp4(grad_y, offsets, w2: Mxfp4Tensor, gate_up, *, inter: int, out, lora, rank_a, sources: int,
                   dense: torch.Tensor | None = None, row_weights: torch.Tensor | None = None) -> torch.Tensor:
    """``down_dx`` on an MXFP4 key: its read-back values (``dense`` when the caller has
    them), the SwiGLU backward in fp32 as the forward's.  ``row_weights`` fp32 [S] (with
    gate/up in fp32): dh is multiplied by them, as ``combine_backward_rows`` leaves it to do."""
    gy = _cuda(grad_y, "grad_y", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    gu = _cuda(gate_up, "gate_up")  # (no dh alone: the MXFP4 forward saves gate/up)
    wide = gu.dtype == torch.float32
    if not wide and (gu.dtype != torch.bfloat16 or row_weights is not None):
        raise TypeError(f"gate_up must be bf16 or fp32 (fp32 with row weights), got {gu.dtype}")
    E, hidden, key_inter = w2.shape
    S = gy.shape[0]
    if gy.shape != (S, hidden) or key_inter != inter or gu.shape != (S, 2 * inter) or offsets.numel() != sources * E:
        raise ValueError(f"grad_y {tuple(gy.shape)}, gate_up {tuple(gu.shape)} and {offsets.numel()} segments do not fit "
                         f"a key {w2.shape} with inter {inter} and {sources} source(s)")
    _same_device(w2.device, grad_y=gy, offsets=offsets, gate_up=gu, rank_a=rank_a)
    w = mxfp4_dequantize(w2) if dense is None else dense
    low = rank_b = None
    if lora is not None:
        low = rank_a if rank_a is not None else lora_project(gy, offsets, lora, forward=False, sources=sources)
        _check_rank_rows(low, S)
        rank_b = lora.a_pad()
        if rank_b.numel() != E * 64 * inter:
            raise ValueError(f"the adapter's A has {rank_b.numel()} padded entries, the key needs {E} x 64 x {inter}")
        _same_device(w2.device, lora=rank_b)
    dgu = _mxfp4_output(out, (S, 2 * inter), w2.device)
    if wide:
        _run(w2.device, "mirai_moe_down_dx_rows_f32", gy.data_ptr(), _ptr(row_weights), offsets.data_ptr(), sources, E, S,
             hidden, inter, w.data_ptr(), gu.data_ptr(), None if low is None else low.data_ptr(),
             None if rank_b is None else rank_b.data_ptr(), dgu.data_ptr())
        return dgu
    _run(w2.device, "mirai_moe_down_dx_f32_bf16", gy.data_ptr(), offsets.data_ptr(), sources, E, S, hidden, inter,
         w.data_ptr(), gu.data_ptr(), None if low is None else low.data_ptr(),
         None if rank_b is None else rank_b.data_ptr(), dgu.data_ptr())
    return dgu


def down_dh(grad_y: torch.Tensor, offsets: torch.Tensor, w2: Int8Tensor, *, inter: int,
            lora: DownLoRA | None = None, rank_a: torch.Tensor | None = None) -> torch.Tensor:
    """dh_raw [S, I] = grad_y (q s) (+ the rank block with the LoRA A factor
    rotated, so that rotating the sum gives the true dh): the INT8 down dX
    without the SwiGLU backward, for the rotated format."""
    if not isinstance(w2, Int8Tensor):
        raise TypeError("down_dh reads INT8 experts")
    gy = _cuda(grad_y, "grad_y", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, H = gy.shape
    dh = torch.empty((S, inter), dtype=torch.bfloat16, device=gy.device)
    if lora is None:
        _lib.call("mirai_moe_down_dh_int8", _ptr(gy), _ptr(offsets), offsets.numel(), S, H, inter, w2.struct(),
                  _ptr(dh), _stream())
        return dh
    glow = rank_a if rank_a is not None else lora_project(gy, offsets, lora, forward=False)
    _lib.call("mirai_moe_down_dh_lora_int8", _ptr(gy), _ptr(offsets), offsets.numel(), S, H, inter, w2.struct(),
              _ptr(glow), _ptr(lora.a_pad(rotation=w2.group_size)), _ptr(dh), _stream())
    return dh


def lora_grad(x: torch.Tensor, g_rank: torch.Tensor, offsets: torch.Tensor, rank: int, out: torch.Tensor,
              strides, sources: int = 1) -> torch.Tensor:
    """out[e][j][k] = sum over the rows of expert e of g_rank[s, j] * x[s, k]
    (fp32, by strides); ``sources`` > 1: source-major segments, summed in
    source order."""
    x = _cuda(x, "x", torch.bfloat16)
    g = _cuda(g_rank, "g_rank", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, K = x.shape
    se, sr, sk = (int(v) for v in strides)
    if offsets.numel() % sources:
        raise ValueError("source-major segments: offsets must be a multiple of sources")
    _lib.call("mirai_moe_lora_grad_src", _ptr(x), _ptr(g), _ptr(offsets), int(sources), offsets.numel() // sources,
              S, K, int(rank), _ptr(out), se, sr, sk, _stream())
    return out


def gateup_dx(grad_gate_up: torch.Tensor, offsets: torch.Tensor, w1, w3, *, hidden: int,
              out: torch.Tensor | None = None, sources: int = 1, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """dx_sorted [S, H] = dgate W1 + dup W3 per expert segment (``sources`` > 1:
    source-major segments).  ``out_dtype=torch.float32`` (bf16 or MXFP4 keys):
    the accumulator unrounded."""
    w1, w3 = _as_weight(_dx_weight(w1)), _as_weight(_dx_weight(w3))
    dgu = _cuda(grad_gate_up, "grad_gate_up", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, I2 = dgu.shape
    if out_dtype == torch.float32:
        return _gateup_dx_f32(dgu, offsets, w1, w3, hidden=hidden, out=out, sources=sources)
    if out_dtype != torch.bfloat16:
        raise TypeError(f"dx_sorted is bf16 or fp32, not {out_dtype}")
    dxs = out if out is not None else torch.empty((S, hidden), dtype=torch.bfloat16, device=dgu.device)
    if sources > 1:
        if offsets.numel() % sources:
            raise ValueError("source-major segments: offsets must be a multiple of sources")
        _lib.call(f"mirai_moe_gateup_dx_src_{_fmt_suffix(w1)}", _ptr(dgu), _ptr(offsets), sources,
                  offsets.numel() // sources, S, I2 // 2, hidden, _wptr(w1), _wptr(w3), _ptr(dxs), _stream())
        return dxs
    _lib.call(f"mirai_moe_gateup_dx_{_fmt_suffix(w1)}", _ptr(dgu), _ptr(offsets), offsets.numel(), S, I2 // 2,
              hidden, _wptr(w1), _wptr(w3), _ptr(dxs), _stream())
    return dxs


def _gateup_dx_f32(dgu: torch.Tensor, offsets: torch.Tensor, w1, w3, *, hidden: int, out: torch.Tensor | None,
                   sources: int) -> torch.Tensor:
    if not isinstance(w1, torch.Tensor) or not isinstance(w3, torch.Tensor):
        raise TypeError("dx_sorted in fp32 needs bf16 or MXFP4 keys")
    w1, w3 = _cuda(w1, "w1", torch.bfloat16), _cuda(w3, "w3", torch.bfloat16)
    S, I2 = dgu.shape
    E = w1.shape[0]
    if tuple(w1.shape) != (E, I2 // 2, hidden) or w3.shape != w1.shape or offsets.numel() != sources * E:
        raise ValueError(f"keys {tuple(w1.shape)} and {tuple(w3.shape)} with {offsets.numel()} segments of {sources} "
                         f"source(s): the call has inter {I2 // 2} and hidden {hidden}")
    _same_device(dgu.device, offsets=offsets, w1=w1, w3=w3)
    if out is None:
        out = torch.empty((S, hidden), dtype=torch.float32, device=dgu.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != (S, hidden) or not out.is_contiguous() \
            or out.device != dgu.device:
        raise ValueError(f"out must be a contiguous fp32 {(S, hidden)} tensor on {dgu.device}, got {out.dtype} "
                         f"{tuple(out.shape)} on {out.device}")
    _run(dgu.device, "mirai_moe_gateup_dx_f32", dgu.data_ptr(), offsets.data_ptr(), sources, E, S, I2 // 2, hidden,
         w1.data_ptr(), w3.data_ptr(), out.data_ptr())
    return out


# ----------------------------------------------------------------------------- any layout / activation / group count

def _ex_suffix(w) -> str:
    if isinstance(w, torch.Tensor):
        return "bf16"
    if isinstance(w, _lib.Nf4Weight):
        return "nf4"
    raise TypeError(f"the *_ex GEMMs read bf16 or NF4 weights, not {type(w)}")


def gateup_ex(x_sorted, offsets, w1, w3, *, inter: int, layout: str, activation: str, save_gate_up: bool = False):
    """gate/up + activation over any number of groups, weights in ``layout``
    ("out_in" [G, I, H] or "in_out" [G, H, I]); returns h (and gate_up)."""
    w1, w3 = _as_weight(w1), _as_weight(w3)
    x_sorted = _cuda(x_sorted, "x_sorted", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, H = x_sorted.shape
    h = torch.empty((S, inter), dtype=torch.bfloat16, device=x_sorted.device)
    gu = torch.empty((S, 2 * inter), dtype=torch.bfloat16, device=x_sorted.device) if save_gate_up else None
    _lib.call(f"mirai_moe_gateup_ex_{_ex_suffix(w1)}", _ptr(x_sorted), _ptr(offsets), offsets.numel(), S, H, inter,
              _wptr(w1), _wptr(w3), LAYOUTS[layout], ACTIVATIONS[activation], _ptr(h), _ptr(gu), _stream())
    return (h, gu) if save_gate_up else h


def down_ex(h, offsets, w2, *, hidden: int, layout: str):
    w2 = _as_weight(w2)
    h = _cuda(h, "h", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, I = h.shape
    y = torch.empty((S, hidden), dtype=torch.bfloat16, device=h.device)
    _lib.call(f"mirai_moe_down_ex_{_ex_suffix(w2)}", _ptr(h), _ptr(offsets), offsets.numel(), S, I, hidden,
              _wptr(w2), LAYOUTS[layout], _ptr(y), _stream())
    return y


def down_dx_ex(grad_y, offsets, w2, gate_up, *, inter: int, layout: str, activation: str):
    w2 = _as_weight(w2)
    gy = _cuda(grad_y, "grad_y", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    gu = _cuda(gate_up, "gate_up", torch.bfloat16)
    S, H = gy.shape
    dgu = torch.empty((S, 2 * inter), dtype=torch.bfloat16, device=gy.device)
    _lib.call(f"mirai_moe_down_dx_ex_{_ex_suffix(w2)}", _ptr(gy), _ptr(offsets), offsets.numel(), S, H, inter,
              _wptr(w2), LAYOUTS[layout], ACTIVATIONS[activation], _ptr(gu), _ptr(dgu), _stream())
    return dgu


def gateup_dx_ex(grad_gate_up, offsets, w1, w3, *, hidden: int, layout: str):
    w1, w3 = _as_weight(w1), _as_weight(w3)
    dgu = _cuda(grad_gate_up, "grad_gate_up", torch.bfloat16)
    offsets = _cuda(offsets, "offsets", torch.int32)
    S, I2 = dgu.shape
    dxs = torch.empty((S, hidden), dtype=torch.bfloat16, device=dgu.device)
    _lib.call(f"mirai_moe_gateup_dx_ex_{_ex_suffix(w1)}", _ptr(dgu), _ptr(offsets), offsets.numel(), S, I2 // 2,
              hidden, _wptr(w1), _wptr(w3), LAYOUTS[layout], _ptr(dxs), _stream())
    return dxs


# ----------------------------------------------------------------------------- whole forward

def _rotations(w1, w3, w2) -> tuple[int, int]:
    """(input group, intermediate group) of a layer's weights: non-zero for the
    rotated INT8 format (w1 and w3 share one activation rotation)."""
    g1, g3 = _group(w1), _group(w3)
    if g1 != g3:
        raise ValueError(f"gate/up rotation groups differ ({g1} vs {g3})")
    return g1, _group(w2)


def moe_forward(tokens: torch.Tensor, top_indices: torch.Tensor, top_weights: torch.Tensor, w1, w3, w2, *,
                num_experts: int, inter: int, lora: "DownLoRA | None" = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Routed expert FFN forward: plan, permute, gate/up+SwiGLU, down, combine.

    Rotated INT8 weights: the tokens are rotated before the permute (T rows,
    not S) and h before the down GEMM; the LoRA rank block is projected from
    the unrotated h.  MXFP4 weights: the tokens are quantised as they are
    permuted, and h as it is formed."""
    if any(isinstance(w, Mxfp4Tensor) for w in (w1, w3, w2)):
        plan = dispatch_plan(top_indices, num_experts)
        y = _mxfp4_experts(tokens, plan, w1, w3, w2, inter=inter, lora=lora, train=False)[0]
        return combine(y, plan.inverse_order, top_weights, out_dtype=out_dtype or tokens.dtype)
    g_in, g_mid = _rotations(w1, w3, w2)
    (w1, w3, w2), join = _stage_beside((w1, w3, w2), top_indices.numel(), num_experts, training=False)
    plan = dispatch_plan(top_indices, num_experts)
    xs = permute_rows(rotate_rows(tokens, g_in) if g_in else tokens, plan.sorted_token_indices)
    join()
    h = gateup_swiglu(xs, plan.offsets, w1, w3, inter=inter)
    low = lora_project(h, plan.offsets, lora, forward=True) if lora is not None else None
    y = down(rotate_rows(h, g_mid) if g_mid else h, plan.offsets, w2, hidden=tokens.shape[1], lora=lora,
             rank_a=low)
    return combine(y, plan.inverse_order, top_weights, out_dtype=out_dtype or tokens.dtype)


def _mxfp4_experts(tokens, plan: DispatchPlan, w1, w3, w2, *, inter: int, lora: DownLoRA | None, train: bool):
    """(y, gate_up, h, rank_a) of the routed rows in MXFP4: quantised in the
    permute's pass, h in the gate/up epilogue (a generation step's few rows inside
    the products).  gate_up (fp32) when ``train``; h and rank_a with a LoRA adapter,
    whose projection reads h in bf16."""
    if not all(isinstance(w, Mxfp4Tensor) for w in (w1, w3, w2)):
        raise TypeError("MXFP4 experts hold all three keys in MXFP4")
    if lora is None and plan.total_slots <= _few_limit(plan.offsets.numel()) and max(tokens.shape[1], inter) <= _FEW_MAX_WIDTH:
        rows = permute_rows(tokens, plan.sorted_token_indices)
        h, gu, _ = _gateup_mxfp4(rows, plan.offsets, w1, w3, inter=inter, save_gate_up=train, want_h=True, want_rows=False,
                                 gate_up_dtype=torch.float32)
        return down(h, plan.offsets, w2, hidden=tokens.shape[1]), gu, None, None
    rows = mxfp4_quantize_rows(tokens, plan.offsets, row_index=plan.sorted_token_indices)
    h, gu, hq = _gateup_mxfp4(rows, plan.offsets, w1, w3, inter=inter, save_gate_up=train, want_h=lora is not None,
                              want_rows=True, gate_up_dtype=torch.float32)
    low = lora_project(h, plan.offsets, lora, forward=True) if lora is not None else None
    return down(hq, plan.offsets, w2, hidden=tokens.shape[1], lora=lora, rank_a=low), gu, h, low


@dataclass
class ForwardState:
    """What the dX pass needs from the forward (no dense weights are kept)."""

    plan: DispatchPlan
    y_sorted: torch.Tensor   # [S, H] bf16 expert outputs
    gate_up: torch.Tensor    # [S, 2I] saved pre-activations, bf16 (an MXFP4 layer's: fp32)
    top_weights: torch.Tensor
    h: torch.Tensor | None = None         # [S, I] bf16, kept when LoRA factor grads are wanted
    rank_a: torch.Tensor | None = None    # [S, 64] LoRA rank block of h (scaled)
    staged: tuple | None = None           # (the NF4 keys, their bf16 copies) when the forward staged them


# NF4 staging: the grouped GEMMs decode NF4 inside their main loops, once per
# 256-row tile of an expert, and that decode (table lookups on the integer
# pipe) limits them below the bf16 kernels' rate.  A training step multiplies
# every expert's weights four times (gate/up and down forward, both dX
# GEMMs), so with many rows per expert it is faster to decode each key once
# into a bf16 copy (one HBM pass, bit-identical values) and run the bf16
# kernels.  The training forward keeps its copies in the state it returns and
# the backward multiplies them again (the reference's frozen linears decode a
# second time instead); they are freed with the state, so a layer holds
# 2 bytes per expert weight from its forward until its backward.
# A forward-only pass multiplies each weight twice as rarely, so "auto" stages
# it from four times the rows per expert: at c2's 2048 the two forms measured
# the same, at c4's 4096 the staged one is faster.
NF4_STAGING_MODES = ("auto", "always", "never")
_nf4_staging = "auto"
STAGE_MIN_ROWS_PER_EXPERT = 1024          # "auto", training passes: at least 4 tiles per expert
STAGE_MIN_ROWS_PER_EXPERT_FORWARD = 4096  # "auto", forward-only passes


def set_nf4_staging(mode: str) -> None:
    """"auto" (default: training passes with at least 1024 rows per expert on
    average, forward-only passes with at least 4096), "always" (every pass) or
    "never" (always decode inside the GEMMs)."""
    global _nf4_staging
    if mode not in NF4_STAGING_MODES:
        raise ValueError(f"NF4 staging mode must be one of {NF4_STAGING_MODES}, not {mode!r}")
    _nf4_staging = mode


def _staging_pays(weights, rows: int, num_experts: int, training: bool) -> bool:
    if _nf4_staging == "never" or not any(isinstance(w, NF4Tensor) for w in weights):
        return False
    least = STAGE_MIN_ROWS_PER_EXPERT if training else STAGE_MIN_ROWS_PER_EXPERT_FORWARD
    return _nf4_staging == "always" or rows >= least * max(1, num_experts)


def stage_nf4(weights, rows: int, num_experts: int, *, training: bool):
    """The weights a pass over ``rows`` routed rows should multiply: NF4 keys
    decoded to bf16 where staging pays (see ``set_nf4_staging``), others as
    given."""
    if not _staging_pays(weights, rows, num_experts, training):
        return tuple(weights)
    return tuple(nf4_dequantize(w) if isinstance(w, NF4Tensor) else w for w in weights)


_side_streams: dict = {}


def _stage_beside(weights, rows: int, num_experts: int, *, training: bool):
    """``stage_nf4`` with the decode on a side stream, so that it runs beside the
    dispatch plan and the permute the caller issues next (both HBM traffic, the
    plan kernels mostly latency).  Returns (weights, join): ``join()`` makes the
    current stream wait for the copies; call it before the first GEMM."""
    if not _staging_pays(weights, rows, num_experts, training):
        return tuple(weights), (lambda: None)
    main = torch.cuda.current_stream()
    dev = next(w for w in weights if isinstance(w, NF4Tensor)).packed.device
    side = _side_streams.get(dev.index)
    if side is None:
        side = _side_streams.setdefault(dev.index, torch.cuda.Stream(device=dev))
    outs = [torch.empty(w.shape, dtype=torch.bfloat16, device=dev) if isinstance(w, NF4Tensor) else None
            for w in weights]  # allocated on the caller's stream, written on the side stream
    side.wait_stream(main)
    with torch.cuda.stream(side):
        for w, o in zip(weights, outs):
            if o is not None:
                nf4_dequantize(w, out=o)
        done = torch.cuda.Event()
        done.record(side)
    for o in outs:
        if o is not None:
            o.record_stream(side)
    return tuple(w if o is None else o for w, o in zip(weights, outs)), (lambda: main.wait_event(done))


def _read_back_beside(weights):
    """bf16 values of MXFP4 keys, read back one after the other on a side stream.  Returns
    (values, join): ``join(n)`` makes the current stream wait for the first n of them.
    Every value must be joined before it is read or dropped."""
    device = weights[0].device
    main = torch.cuda.current_stream(device)
    side = _side_streams.get(device.index)
    if side is None:
        side = _side_streams.setdefault(device.index, torch.cuda.Stream(device=device))
    outs = [torch.empty(w.shape, dtype=torch.bfloat16, device=device) for w in weights]  # the caller's stream's memory
    side.wait_stream(main)
    events = []
    for w, o in zip(weights, outs):
        o.record_stream(side)
        _run(device, "mirai_mxfp4_dequantize", w.packed.data_ptr(), w.scale.data_ptr(), *w.shape, o.data_ptr(),
             _MXFP4_DTYPES[torch.bfloat16], stream=side.cuda_stream)
        events.append(side.record_event())
    return outs, (lambda n: main.wait_event(events[n - 1]))


def check_mxfp4_training(weights, hidden: int, inter: int) -> None:
    """ValueError for MXFP4 keys of widths that the dX GEMMs do not take."""
    if any(isinstance(w, Mxfp4Tensor) for w in weights) and (hidden % 64 or inter % 64):
        raise ValueError(f"training MXFP4 experts needs hidden and inter in steps of 64, got {hidden} and {inter}")


def moe_forward_train(tokens, top_indices, top_weights, w1, w3, w2, *, num_experts: int, inter: int,
                      out_dtype: torch.dtype | None = None, lora: DownLoRA | None = None):
    """Forward that also returns the state the dX pass consumes.  (MXFP4 keys:
    the forward takes widths in steps of 32, the backward of 64.)"""
    if any(isinstance(w, Mxfp4Tensor) for w in (w1, w3, w2)):
        check_mxfp4_training((w1, w3, w2), tokens.shape[1], inter)
        plan = dispatch_plan(top_indices, num_experts)
        y, gu, h, low = _mxfp4_experts(tokens, plan, w1, w3, w2, inter=inter, lora=lora, train=True)
        out = combine(y, plan.inverse_order, top_weights, out_dtype=out_dtype or tokens.dtype)
        keep = lora is not None and lora.compute_grads
        return out, ForwardState(plan, y, gu, top_weights.float(), h if keep else None, low if keep else None)
    g_in, g_mid = _rotations(w1, w3, w2)
    keys = (w1, w3, w2)
    (w1, w3, w2), join = _stage_beside(keys, top_indices.numel(), num_experts, training=True)
    staged = (keys, (w1, w3, w2)) if w1 is not keys[0] else None
    plan = dispatch_plan(top_indices, num_experts)
    xs = permute_rows(rotate_rows(tokens, g_in) if g_in else tokens, plan.sorted_token_indices)
    join()
    h, gu = gateup_swiglu(xs, plan.offsets, w1, w3, inter=inter, save_gate_up=True)
    low = None
    if lora is not None:
        low = lora_project(h, plan.offsets, lora, forward=True)
    y = down(rotate_rows(h, g_mid) if g_mid else h, plan.offsets, w2, hidden=tokens.shape[1], lora=lora,
             rank_a=low)
    out = combine(y, plan.inverse_order, top_weights, out_dtype=out_dtype or tokens.dtype)
    keep = lora is not None and lora.compute_grads
    return out, ForwardState(plan, y, gu, top_weights.float(), h if keep else None, low if keep else None, staged)


def _mxfp4_backward(grad_out, state: ForwardState, w1, w3, w2, *, inter: int, out_dtype: torch.dtype,
                    lora: DownLoRA | None):
    """``moe_backward_dx`` on MXFP4 keys.  The stored values are read back to bf16, w2
    first, beside the combine backward and the down dX.  dx is rounded where an MMA
    operand must be bf16 (dgate / dup) and at the end; the rows that go into the down
    dX are the output's gradient itself, weighted in its epilogue, and gate/up and the
    routes' dx stay in fp32."""
    plan, H = state.plan, state.y_sorted.shape[1]
    dense, join = _read_back_beside((w2, w1, w3))
    rows, rw, gw = combine_backward_rows(grad_out, state.y_sorted, plan.inverse_order, state.top_weights)
    glow = None
    if lora is not None:
        E, Hb, r = lora.b.shape
        glow = lora_project(rows, plan.offsets, lora, forward=False)
        if lora.compute_grads:
            if state.h is None or state.rank_a is None:
                raise RuntimeError("LoRA factor gradients need the forward run with compute_grads=True")
            Ia = lora.a.shape[2]
            # the [S, 64] operand of each sum over rows takes the rows' weights
            weighted = [(t * rw[:, None]).to(torch.bfloat16) for t in (glow, state.rank_a)]
            lora.grad_a = lora_grad(state.h, weighted[0], plan.offsets, r,
                                    torch.empty((E, r, Ia), dtype=torch.float32, device=rows.device), (r * Ia, Ia, 1))
            lora.grad_b = lora_grad(rows, weighted[1], plan.offsets, r,
                                    torch.empty((E, Hb, r), dtype=torch.float32, device=rows.device), (Hb * r, 1, r))
    join(1)
    dgu = _down_dx_mxfp4(rows, plan.offsets, w2, state.gate_up, inter=inter, out=None, lora=lora, rank_a=glow, sources=1,
                         dense=dense[0], row_weights=rw)
    join(3)
    dxs = _gateup_dx_f32(dgu, plan.offsets, dense[1], dense[2], hidden=H, out=None, sources=1)
    return combine(dxs, plan.inverse_order, None, out_dtype=out_dtype, top_k=plan.top_k), gw


def moe_backward_dx(grad_out: torch.Tensor, state: ForwardState, w1, w3, w2, *, inter: int,
                    out_dtype: torch.dtype = torch.bfloat16, lora: DownLoRA | None = None):
    """Input gradient through the frozen experts and the top-weight gradient.

    grad_out [T, H] -> (dx [T, H], d_top_weights fp32 [T, k])."""
    plan = state.plan
    H = state.y_sorted.shape[1]
    if isinstance(w2, Mxfp4Tensor):
        return _mxfp4_backward(grad_out, state, w1, w3, w2, inter=inter, out_dtype=out_dtype, lora=lora)
    if state.staged is not None and all(a is b for a, b in zip(state.staged[0], (w1, w3, w2))):
        w1, w3, w2 = state.staged[1]  # the forward's bf16 copies of these NF4 keys
        state.staged = None
    else:
        w1, w3, w2 = stage_nf4((w1, w3, w2), state.y_sorted.shape[0], plan.offsets.numel(), training=True)
    gy, gw = combine_backward(grad_out, state.y_sorted, plan.inverse_order, state.top_weights)
    glow = None
    if lora is not None:
        E, Hb, r = lora.b.shape
        glow = lora_project(gy, plan.offsets, lora, forward=False)
        if lora.compute_grads:
            if state.h is None or state.rank_a is None:
                raise RuntimeError("LoRA factor gradients need the forward run with compute_grads=True")
            Ia = lora.a.shape[2]
            lora.grad_a = lora_grad(state.h, glow, plan.offsets, r,
                                    torch.empty((E, r, Ia), dtype=torch.float32, device=gy.device), (r * Ia, Ia, 1))
            lora.grad_b = lora_grad(gy, state.rank_a, plan.offsets, r,
                                    torch.empty((E, Hb, r), dtype=torch.float32, device=gy.device), (Hb * r, 1, r))
    g_in, g_mid = _rotations(w1, w3, w2)
    if g_mid:  # rotated INT8: dh = rotate(grad_y (q s)), then the SwiGLU backward
        dh = down_dh(gy, plan.offsets, w2, inter=inter, lora=lora, rank_a=glow)
        dgu = swiglu_backward_rotated(dh, state.gate_up, g_mid)
    else:
        dgu = down_dx(gy, plan.offsets, w2, state.gate_up, inter=inter, lora=lora, rank_a=glow)
    dxs = gateup_dx(dgu, plan.offsets, w1, w3, hidden=H)
    if g_in:  # sum the routes in fp32, then rotate the token rows (T, not S)
        dx32 = combine(dxs, plan.inverse_order, None, out_dtype=torch.float32, top_k=plan.top_k)
        return rotate_rows(dx32, g_in, out_dtype=out_dtype), gw
    dx = combine(dxs, plan.inverse_order, None, out_dtype=out_dtype, top_k=plan.top_k)
    return dx, gw
