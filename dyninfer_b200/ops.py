"""Single operators of the path, called through the C ABI on torch CUDA tensors.

torch is used only to own device memory and the stream; every computation is a
call into libdyninfer_cuda. There is no eager/PyTorch implementation behind
these functions: without the library or without a GPU they raise.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import numpy as np
import torch

from . import _lib
from ._lib import ENC, check, lib


# torch's current stream as an integer: 0.2 us through its raw getters (3.2 us through a Stream object), which are not
# part of its public interface, so a torch without them takes the public way
_raw_stream, _raw_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)


def _stream():
    if _raw_stream is None or _raw_device is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_raw_device())


def _p(t):
    return t.data_ptr() if t is not None else None


def _dev(a, device="cuda"):
    if isinstance(a, torch.Tensor):
        return a.to(device).contiguous()
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


class DeviceWeight:
    """One [rows, cols] parameter resident on the GPU as its verbatim checkpoint bytes."""

    def __init__(self, encoding: str, rows: int, cols: int, data, scales=None, biases=None,
                 aux: str = "plain.bf16", group: int = 64, device="cuda"):
        self.encoding, self.rows, self.cols, self.group, self.aux = encoding, int(rows), int(cols), int(group), aux
        raw = np.frombuffer(data, dtype=np.uint8) if isinstance(data, (bytes, bytearray, memoryview)) \
            else np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        need = lib().dyninfer_cuda_row_bytes(ENC[encoding], cols) * rows
        if raw.size != need:
            raise ValueError(f"{encoding} [{rows},{cols}] needs {need} bytes, got {raw.size}")
        # 64 bytes of readable slack behind the range, as the session arena provides
        buf = torch.zeros(raw.size + 64, dtype=torch.uint8, device=device)
        buf[:raw.size] = torch.from_numpy(raw.copy())
        self.data = buf
        self.scales = _dev(np.ascontiguousarray(scales).view(np.uint8).reshape(-1), device) if scales is not None else None
        self.biases = _dev(np.ascontiguousarray(biases).view(np.uint8).reshape(-1), device) if biases is not None else None
        self.nbytes = raw.size + (self.scales.numel() if self.scales is not None else 0) + \
            (self.biases.numel() if self.biases is not None else 0)

    def c(self) -> _lib.Weight:
        return _lib.Weight(ENC[self.encoding], ENC.get(self.aux, 2), self.group, 0, self.rows,
                           self.cols, _p(self.data), _p(self.scales), _p(self.biases))

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        object.__setattr__(self, "_ref", None)     # whatever was described may have changed

    def ref(self):
        """The descriptor by reference, built once for what it describes: a small product's time is mostly the host's."""
        key = (self.data.data_ptr(), None if self.scales is None else self.scales.data_ptr(),
               None if self.biases is None else self.biases.data_ptr())
        if self._ref is None or self._ref[0] != key:
            object.__setattr__(self, "_ref", (key, C.byref(self.c())))
        return self._ref[1]


def dequant(w: DeviceWeight) -> torch.Tensor:
    out = torch.empty((w.rows, w.cols), dtype=torch.float32, device=w.data.device)
    cw = w.c()
    check(lib().dyninfer_cuda_dequant(C.byref(cw), _p(out), _stream()))
    return out


def embedding_gather(w: DeviceWeight, tokens: torch.Tensor) -> torch.Tensor:
    tokens = tokens.to(device=w.data.device, dtype=torch.int64).contiguous()
    out = torch.empty((tokens.numel(), w.cols), dtype=torch.float32, device=w.data.device)
    cw = w.c()
    check(lib().dyninfer_cuda_embedding_gather(C.byref(cw), _p(tokens), tokens.numel(), _p(out), _stream()))
    return out


_XT = {torch.float32: ENC["plain.f32"], torch.bfloat16: ENC["plain.bf16"]}
_linear_fn = None


def linear(w: DeviceWeight, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    global _linear_fn
    xt = _XT.get(x.dtype)
    if xt is None:
        raise TypeError("x must be float32 or bfloat16")
    if x.dim() != 2 or x.shape[1] != w.cols or not x.is_contiguous():
        x = x.contiguous().view(-1, w.cols)
    m = x.shape[0]
    if out is None:
        out = torch.empty((m, w.rows), dtype=torch.float32, device=x.device)
    if _linear_fn is None:
        _linear_fn = lib().dyninfer_cuda_linear
    if _linear_fn(w.ref(), x.data_ptr(), xt, m, out.data_ptr(), _stream()):
        check(1)
    return out


_WT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    x = x.contiguous()
    width = w.numel()
    y = torch.empty_like(x)
    check(lib().dyninfer_cuda_rms_norm(_p(x), _p(w.contiguous()), _WT[w.dtype], x.numel() // width,
                                       width, float(eps), _p(y), _stream()))
    return y


def rope(x: torch.Tensor, start_pos: int, theta: float) -> torch.Tensor:
    y = x.contiguous().clone()
    s, h, d = y.shape
    check(lib().dyninfer_cuda_rope(_p(y), s, h, d, int(start_pos), float(theta), _stream()))
    return y


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    gate, up = gate.contiguous(), up.contiguous()
    y = torch.empty_like(gate)
    check(lib().dyninfer_cuda_silu_mul(_p(gate), _p(up), gate.numel(), _p(y), _stream()))
    return y


def attention(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, start_pos: int) -> torch.Tensor:
    """q [s, heads, d] f32; caches [kv_heads, cap, d] (f32/f16/bf16) holding rows < start_pos + s."""
    q = q.contiguous()
    s, nh, d = q.shape
    nkv, cap, _ = kcache.shape
    ctx = torch.empty((s, nh * d), dtype=torch.float32, device=q.device)
    check(lib().dyninfer_cuda_attention(_p(q), _p(kcache.contiguous()), _p(vcache.contiguous()),
                                        _WT[kcache.dtype], s, nh, nkv, d, cap, int(start_pos),
                                        _p(ctx), _stream()))
    return ctx


def argmax(v: torch.Tensor) -> int:
    v = v.contiguous().view(-1)
    out = torch.empty(1, dtype=torch.int64, device=v.device)
    scratch = torch.empty(lib().dyninfer_cuda_argmax_scratch_bytes(v.numel()), dtype=torch.uint8,
                          device=v.device)
    check(lib().dyninfer_cuda_argmax(_p(v), v.numel(), _p(out), _p(scratch), _stream()))
    return int(out.item())


# ---- speculative decoding: a tree of drafted tokens over a cache -----------------------------------------------------
# A step: `rotary` turns the drafted rows to their depths, `kv_write` puts their keys and values behind the cache's rows,
# `tree_attention` attends under the tree's mask, `verify_draft` says which tokens stand; the rows that do are written once more in
# their order (`kv_write` of the path's rows with counts). All are asynchronous on torch's current stream and may be captured; the
# first call of each on a device does set-up work.

_SCALED = {torch.int8: _lib.KV["q8"], torch.float8_e4m3fn: _lib.KV["e4m3"]}
_KV = {**_SCALED, torch.float16: ENC["plain.f16"], torch.bfloat16: ENC["plain.bf16"]}


# Host-side work is most of a small call's time, so the checks below keep to plain comparisons: strides travel as packed
# bytes (0.3 us; a ctypes array is 1.2), devices are compared by index, dense int64 tensors are not touched.
_pack2, _pack3, _pack4, _pack6 = (struct.Struct(f"{n}q").pack for n in (2, 3, 4, 6))


def _devices(*tensors):
    """The device that all the tensors are on."""
    at = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"tensors on different devices: {tensors[0].device} and {t.device}")
    if at < 0:
        raise ValueError(f"tensors are on {tensors[0].device}: this target runs on a CUDA device")
    return at


def _run(device, call, *args):
    """call(*args, stream) on a device, which may be another than the current one."""
    if _raw_device is not None and _raw_stream is not None and device == _raw_device():
        if call(*args, _raw_stream(device)):
            check(1)
    else:
        with torch.cuda.device(device):
            check(call(*args, _stream()))


def _dense_last(what, t):
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what}: the last dimension must be dense (stride 1), not {t.stride(-1)}")


def _shape(what, t, shape):
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _index(what, t):
    """Positions, lengths and token ids: dense int64 (int32 is converted)."""
    if t.dtype is torch.int64:
        return t if t.is_contiguous() else t.contiguous()
    if t.dtype is not torch.int32:
        raise TypeError(f"{what} must be int64, not {t.dtype}")
    return t.to(torch.int64).contiguous()


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = "half",
           magnitude: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of x [..., heads, d] (f32, f16 or bf16, up to two leading dimensions, any strides with a dense last
    dimension): pair i of the first 2 * len(frequencies) dimensions turns by positions[...] * frequencies[i] and is multiplied by
    `magnitude`; the other dimensions are copied. `layout` is "half" (pairs i, i + r/2) or "interleaved" (2i, 2i + 1).
    `frequencies` is a float64 tensor in host memory (`rotary_frequencies` makes one); angles are taken modulo a turn in 64-bit
    fixed point, off by at most 2^-65 * position * (1 + frequency) turns. `out` may be x itself (a view of the leading heads of
    fused [q | k | v] rows turns q and k where they lie) but must not overlap it otherwise."""
    kind, shape, sx = _WT.get(x.dtype), x.shape, x.stride()
    if kind is None:
        raise TypeError(f"x must be float32, float16 or bfloat16, not {x.dtype}")
    if layout != "half" and layout != "interleaved":
        raise ValueError(f"layout {layout!r} is neither 'half' nor 'interleaved'")
    if len(shape) == 3:
        (rows, heads, d), batch = shape, 1
    elif len(shape) == 4:
        batch, rows, heads, d = shape
    else:
        raise ValueError(f"x must be [rows, heads, d] or [batch, rows, heads, d], not {tuple(shape)}")
    if frequencies.is_cuda or frequencies.dtype is not torch.float64 or frequencies.dim() != 1:
        raise ValueError("frequencies must be a one-dimensional float64 tensor in host memory")
    if sx[-1] != 1:
        _dense_last("x", x)
    if positions.shape != shape[:-2]:
        _shape("positions", positions, shape[:-2])
    positions = _index("positions", positions)
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        so = out.stride()
    else:
        so = out.stride()
        if out.dtype != x.dtype or out.shape != shape:
            raise ValueError("out must have x's type and shape")
        if so[-1] != 1:
            _dense_last("out", out)
    # (with one batch entry its stride is never used, whatever it says)
    _run(_devices(x, positions, out), lib().dyninfer_cuda_rotary, x.data_ptr(), kind, _pack3(sx[-4] if batch > 1 else 0, sx[-3], sx[-2]),
         positions.data_ptr(), frequencies.data_ptr(), 2 * frequencies.numel(), layout == "interleaved", magnitude, batch, rows,
         heads, d, out.data_ptr(), _pack3(so[-4] if batch > 1 else 0, so[-3], so[-2]))
    return out


def rotary_frequencies(rotary_dim: int, theta: float = 1e6, scaling: str = "none", factor: float = 1.0,
                       original_length: int | None = None, low: float | None = None, high: float | None = None):
    """(frequencies, magnitude) for `rotary`: theta^(-2i / rotary_dim), lengthened by `factor` in one of these ways.

    * "none"
    * "linear": all frequencies / factor
    * "ntk": theta * factor^(rotary_dim / (rotary_dim - 2)): the fastest stays, the slowest is divided by factor
    * "yarn": dimensions that turn over `high` (32) times within original_length stay, those under `low` (1) times are divided,
      linearly in between along the dimensions; the magnitude is 0.1 ln(factor) + 1
    * "wavelength": as yarn with `low` = 1 and `high` = 4, linearly along the number of turns, magnitude 1
    """
    if rotary_dim <= 0 or rotary_dim % 2 or not theta > 0 or not factor > 0:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and above zero, theta and factor above zero")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = theta ** (-2 * i / rotary_dim)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        return (theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim), 1.0
    if scaling not in ("yarn", "wavelength"):
        raise ValueError(f"scaling {scaling!r} is not one of none, linear, ntk, yarn, wavelength")
    if not original_length or original_length <= 0:
        raise ValueError(f"{scaling} scaling needs original_length")
    low, high = 1.0 if low is None else low, (32.0 if scaling == "yarn" else 4.0) if high is None else high
    if not 0 < low < high:
        raise ValueError(f"low {low} must be above zero and below high {high}")
    if scaling == "yarn":
        def dimension(turns):
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))
        first, last = max(math.floor(dimension(high)), 0), min(math.ceil(dimension(low)), rotary_dim - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (1 - keep) * f / factor + keep * f, 1.0


def _cache(k_cache, v_cache):
    """(shape, packed strides) of a cache."""
    shape, k, v = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4:
        raise ValueError(f"a cache is [slots, kv_heads, capacity, d], not {tuple(shape)}")
    if v_cache.shape != shape:
        _shape("v_cache", v_cache, shape)
    if k[3] != 1 or v[3] != 1:
        _dense_last("k_cache", k_cache)
        _dense_last("v_cache", v_cache)
    return shape, _pack6(k[0], k[1], k[2], v[0], v[1], v[2])


def _scales(shape, k_scale, v_scale):
    """Packed strides of the scales [slots, kv_heads, capacity] of an 8-bit cache's rows."""
    if k_scale is None or v_scale is None or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        bad = "k_scale" if k_scale is None or k_scale.dtype is not torch.float32 else "v_scale"
        raise TypeError(f"{bad} must be float32")
    k, v, shape = k_scale.stride(), v_scale.stride(), shape[:3]
    if k_scale.shape != shape or v_scale.shape != shape or k[2] != 1 or v[2] != 1:
        for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
            _shape(name, scale, shape)
            _dense_last(name, scale)
    return _pack4(k[0], k[1], v[0], v[1])


def _scaled_kind(k_cache, v_cache):
    kind = _SCALED.get(k_cache.dtype)
    if kind is None or v_cache.dtype != k_cache.dtype:
        raise TypeError(f"an 8-bit cache is int8 or float8_e4m3fn, not {k_cache.dtype} and {v_cache.dtype}")
    return kind


def kv_write(k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             k_scale: torch.Tensor, v_scale: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Quantises k and v [slots, rows, kv_heads, d] (f32, f16 or bf16) into an 8-bit cache [slots, kv_heads, capacity, d] of
    int8 or float8_e4m3fn codes with f32 scales [slots, kv_heads, capacity]: row r of a slot goes to cache row starts[slot] + r,
    for r < counts[slot] where counts are given. Rows outside the cache are left out, all others of the cache as they were."""
    kind = _WT.get(k.dtype)
    if kind is None or v.dtype != k.dtype:
        raise TypeError(f"k and v must both be float32, float16 or bfloat16, not {k.dtype} and {v.dtype}")
    cache = _scaled_kind(k_cache, v_cache)
    whole, steps = _cache(k_cache, v_cache)
    scale_steps = _scales(whole, k_scale, v_scale)
    slots, heads, cap, d = whole
    shape, sk, sv = k.shape, k.stride(), v.stride()
    if len(shape) != 4:
        raise ValueError(f"k must be [slots, rows, kv_heads, d], not {tuple(shape)}")
    rows = shape[1]
    if shape != (slots, rows, heads, d) or v.shape != shape or sk[3] != 1 or sv[3] != 1:
        _shape("k", k, (slots, rows, heads, d))
        _shape("v", v, shape)
        _dense_last("k", k)
        _dense_last("v", v)
    if starts.shape != whole[:1]:
        _shape("starts", starts, (slots,))
    starts = _index("starts", starts)
    if counts is not None:
        _shape("counts", counts, (slots,))
        counts = _index("counts", counts)
    _run(_devices(k, v, starts, counts, k_cache, v_cache, k_scale, v_scale), lib().dyninfer_cuda_kv_write, k.data_ptr(), v.data_ptr(),
         kind, _pack6(sk[0], sk[1], sk[2], sv[0], sv[1], sv[2]), k_cache.data_ptr(), v_cache.data_ptr(), cache, steps,
         k_scale.data_ptr(), v_scale.data_ptr(), scale_steps, starts.data_ptr(), _p(counts), slots, rows, heads, d, cap)


def kv_read(starts: torch.Tensor, rows: int, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
            v_scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows starts[slot] .. starts[slot] + rows - 1 of an 8-bit cache as values (k, v), each [slots, rows, kv_heads, d] of
    `dtype`: what `kv_write` takes. Zeros for rows outside the cache; infinity where a code's rounding passes dtype's largest."""
    kind = _WT.get(dtype)
    if kind is None:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    if rows < 0:
        raise ValueError(f"rows must be at least zero, not {rows}")
    cache = _scaled_kind(k_cache, v_cache)
    whole, steps = _cache(k_cache, v_cache)
    scale_steps = _scales(whole, k_scale, v_scale)
    slots, heads, cap, d = whole
    if starts.shape != whole[:1]:
        _shape("starts", starts, (slots,))
    starts = _index("starts", starts)
    k = k_scale.new_empty((slots, rows, heads, d), dtype=dtype)
    v = torch.empty_like(k)
    row, head = heads * d, d
    _run(_devices(starts, k_cache, v_cache, k_scale, v_scale), lib().dyninfer_cuda_kv_read, k.data_ptr(), v.data_ptr(), kind,
         _pack6(rows * row, row, head, rows * row, row, head), k_cache.data_ptr(), v_cache.data_ptr(), cache, steps,
         k_scale.data_ptr(), v_scale.data_ptr(), scale_steps, starts.data_ptr(), slots, rows, heads, d, cap)
    return k, v


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                   mask: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of drafted rows q [slots, rows, heads, d] (f32, f16 or bf16) over caches [slots, kv_heads, capacity, d] of f16,
    bf16, or 8-bit codes with their scales. Row r of a slot sees keys 0 .. lengths[slot] - 1, and of the rows' own keys, which
    stand at lengths[slot] + j, those with mask[slot, r, j] (bool, [rows, rows] for all slots or [slots, rows, rows]); without a
    mask, those with j <= r: a chain, or the plain decode step. A row that sees nothing, or whose length is below zero, gets
    zeros. `scale` is 1 / sqrt(d) unless given. Returns [slots, rows, heads, d] of q's type. Sums are held in 32 bits; softmax
    weights of bf16 queries over f16 and 8-bit caches enter their products with 11 bits (others 16 to 24), and over 8-bit caches
    what is below 2^-38 (f32 queries) or 2^-30 (others) of the largest value that a row sees is lost."""
    kind, cache = _WT.get(q.dtype), _KV.get(k_cache.dtype)
    if kind is None:
        raise TypeError(f"q must be float32, float16 or bfloat16, not {q.dtype}")
    if cache is None or v_cache.dtype != k_cache.dtype:
        raise TypeError(f"caches must both be float16, bfloat16, int8 or float8_e4m3fn, not {k_cache.dtype} and {v_cache.dtype}")
    (whole, steps), scale_steps = _cache(k_cache, v_cache), None
    if cache >= _lib.KV["q8"]:
        scale_steps = _scales(whole, k_scale, v_scale)
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"a cache of {k_cache.dtype} has no scales")
    slots, kv_heads, cap, d = whole
    shape, sq = q.shape, q.stride()
    if len(shape) != 4:
        raise ValueError(f"q must be [slots, rows, heads, d], not {tuple(shape)}")
    _, rows, heads, _ = shape
    if shape[0] != slots or shape[3] != d or sq[3] != 1:
        _shape("q", q, (slots, rows, heads, d))
        _dense_last("q", q)
    if lengths.shape != whole[:1]:
        _shape("lengths", lengths, (slots,))
    lengths = _index("lengths", lengths)
    masked = None
    if mask is not None:
        if mask.dtype is not torch.bool:
            raise TypeError(f"mask must be bool, not {mask.dtype}")
        shared = mask.dim() == 2
        if mask.shape != ((rows, rows) if shared else (slots, rows, rows)):
            _shape("mask", mask, (rows, rows) if shared else (slots, rows, rows))
        sm = mask.stride()
        if sm[-1] != 1 and rows > 1:
            mask = mask.contiguous()
            sm = mask.stride()
        masked = _pack2(0 if shared else sm[0], sm[-2])
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _run(_devices(q, k_cache, v_cache, lengths, mask, k_scale, v_scale), lib().dyninfer_cuda_tree_attention, q.data_ptr(), kind,
         _pack3(sq[0], sq[1], sq[2]), k_cache.data_ptr(), v_cache.data_ptr(), cache, steps, _p(k_scale), _p(v_scale), scale_steps,
         lengths.data_ptr(), _p(mask), masked, slots, rows, heads, kv_heads, d, cap, d ** -0.5 if scale is None else scale,
         out.data_ptr())
    return out


def verify_draft(tokens: torch.Tensor, parents: torch.Tensor, target: torch.Tensor, uniforms: torch.Tensor,
                 draft: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, and the token behind them: (accepted [slots], path [slots, nodes], next [slots]), int64.

    Node 0 is the text's last token; node i > 0 carries tokens[:, i] behind node parents[:, i] < i ([nodes] for all slots or
    [slots, nodes]; any other parent: no such node). target [slots, nodes, vocab] (f32, f16 or bf16) holds the probabilities of
    the token behind each node, draft those that a node's children were drawn from independently; without it the children are
    distinct tokens chosen without chance. uniforms [slots, nodes] are f32 in [0, 1): node i is tried with its own, and node 0's
    draws the last token. From node 0 on the children of the node reached are tried in order; a refusal takes the draft's
    probabilities (without a draft, the child's entry) from what the next child or the last token is drawn from. The
    target's distribution is kept where rows of target and draft sum to one; they are taken as they are, so rows rounded to 16
    bits keep it to about that rounding. next is -1 where a row has no finite positive sum."""
    if target.dim() != 3:
        raise ValueError(f"target must be [slots, nodes, vocab], not {tuple(target.shape)}")
    kind = _WT.get(target.dtype)
    if kind is None:
        raise TypeError(f"target must be float32, float16 or bfloat16, not {target.dtype}")
    shape, st = target.shape, target.stride()
    slots, nodes, vocab = shape
    each = shape[:2]
    shared = parents.dim() == 1
    if tokens.shape != each or parents.shape != (each[1:] if shared else each) or uniforms.shape != each or st[2] != 1:
        _shape("tokens", tokens, each)
        _shape("parents", parents, each[1:] if shared else each)
        _shape("uniforms", uniforms, each)
        _dense_last("target", target)
    if uniforms.dtype is not torch.float32:
        raise TypeError(f"uniforms must be float32, not {uniforms.dtype}")
    tokens, parents = _index("tokens", tokens), _index("parents", parents)
    if not uniforms.is_contiguous():
        uniforms = uniforms.contiguous()
    drafted = None
    if draft is not None:
        if draft.dtype != target.dtype:
            raise TypeError(f"draft must have the target's type {target.dtype}, not {draft.dtype}")
        sd = draft.stride()
        if draft.shape != shape or sd[2] != 1:
            _shape("draft", draft, shape)
            _dense_last("draft", draft)
        drafted = _pack2(sd[0], sd[1])
    path, accepted = torch.empty_like(tokens), tokens.new_empty(slots)
    following = torch.empty_like(accepted)
    _run(_devices(target, tokens, parents, uniforms, draft), lib().dyninfer_cuda_verify_draft, tokens.data_ptr(), parents.data_ptr(),
         0 if shared else nodes, target.data_ptr(), _pack2(st[0], st[1]), _p(draft), drafted, kind,
         uniforms.data_ptr(), slots, nodes, vocab, accepted.data_ptr(), path.data_ptr(), following.data_ptr())
    return accepted, path, following


def check_device_error():
    """Call after synchronising: raises when a kernel's bounded wait (weight ring, GEMM or attention pipeline)
    expired since the last check, in which case the results produced since then are invalid."""
    check(lib().dyninfer_cuda_check_device_error())
