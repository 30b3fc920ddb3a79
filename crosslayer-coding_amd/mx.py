"""Microscaled formats: rows held in 8 or 4 bits, a resident cache of activations in them, and the encoder projection
from 4-bit weights.

32 neighbouring elements of a row share a power of two, stored as one byte; the elements are stored as codes:

    mxfp4     0 0.5 1 1.5 2 3 4 6 and their negatives, two to a byte (the even element in the low half)   4.25 bits each
    mxfp8     sign, four bits of exponent, three of mantissa (``torch.float8_e4m3fn``)                    8.25 bits
    mxint8    64ths, -127/64 .. 127/64                                                                     8.25 bits

The scale is the exponent of the block's largest magnitude minus the format's own largest exponent; elements are rounded
to nearest even and held at the format's largest value.  A block with an infinity or a NaN has no scale (byte 255) and
reads back as NaN.  This is the layout of the open microscaling formats, so codes and scales made elsewhere can be used.

The reference has no quantised form of either; what these replace here: `MXActivationCache` the 16- and 32-bit chunks of
a store (clt/training/data/manifest_activation_store.py:776-958), `project` the encoder's linear layers
(clt/models/parallel.py:286) for inference.  Nothing here takes part in autograd.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _native as nat

BLOCK = 32
FORMATS = {"mxfp4": 0, "mxfp8": 1, "mxint8": 2}
_BLOCK_BYTES = {"mxfp4": 16, "mxfp8": 32, "mxint8": 32}
MAX_WIDTH = 262144
_NORM_MODES = {"none": 0, "mean_std": 1, "sqrt_d_model": 2}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)

Rows = Union[slice, range, Sequence[int], np.ndarray, torch.Tensor]


def _format(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"Invalid format: {fmt!r}. Must be one of {list(FORMATS)}")
    return FORMATS[fmt]


def row_layout(width: int, fmt: str) -> Tuple[int, int]:
    """(bytes of codes, bytes of scales) of a row of ``width`` elements."""
    _format(fmt)
    if not 0 < width <= MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} elements are taken, got {width}")
    blocks = -(-width // BLOCK)
    return blocks * _BLOCK_BYTES[fmt], blocks


class _On:
    """``torch.cuda.device(device)``, which costs more than a launch, where the device is not the current one."""

    __slots__ = ("index", "back")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        current = torch._C._cuda_getDevice()
        self.back = current if self.index is not None and self.index != current else None
        if self.back is not None:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)
        return False


def _check_values(t: torch.Tensor, what: str) -> None:
    if t.dtype not in _FLOATS:
        raise ValueError(f"{what}: float32, bfloat16 or float16 is taken, got {t.dtype}")
    nat.require_device(t, what)
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _rows_2d(t: torch.Tensor) -> torch.Tensor:
    """[rows, d] with neighbouring elements next to each other, without a copy where the strides allow it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


class MXTensor:
    """Rows of ``width`` elements in a microscaled format: ``codes`` uint8 [..., bytes of a row] and ``scales`` uint8
    [..., blocks], contiguous, with the same leading sizes."""

    __slots__ = ("codes", "scales", "fmt", "width")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, width: int):
        pitch, blocks = row_layout(width, fmt)
        for t, name, last in ((codes, "codes", pitch), (scales, "scales", blocks)):
            if t.dtype != torch.uint8 or t.dim() < 1 or t.shape[-1] != last or not t.is_contiguous():
                raise ValueError(f"{name} of {fmt} rows of {width} elements must be contiguous uint8 [..., {last}], got "
                                 f"{t.dtype} {tuple(t.shape)}")
        if codes.shape[:-1] != scales.shape[:-1] or codes.device != scales.device:
            raise ValueError(f"codes {tuple(codes.shape)} on {codes.device} and scales {tuple(scales.shape)} on {scales.device} "
                             "do not belong together")
        if codes.data_ptr() % 16 != 0:
            raise ValueError("codes must begin at a multiple of 16 bytes")
        self.codes, self.scales, self.fmt, self.width = codes, scales, fmt, int(width)

    @classmethod
    def _made(cls, codes: torch.Tensor, scales: torch.Tensor, fmt: str, width: int) -> "MXTensor":
        """Of tensors that are as `row_layout` says: nothing to check."""
        held = cls.__new__(cls)
        held.codes, held.scales, held.fmt, held.width = codes, scales, fmt, width
        return held

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.width))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def index_select(self, index: torch.Tensor) -> "MXTensor":
        """The entries ``index`` of the first dimension, copied."""
        return MXTensor(self.codes.index_select(0, index), self.scales.index_select(0, index), self.fmt, self.width)

    def narrow(self, first: int, n: int) -> "MXTensor":
        """The entries first, ..., first + n - 1 of the first dimension, not copied."""
        return MXTensor._made(self.codes.narrow(0, first, n), self.scales.narrow(0, first, n), self.fmt, self.width)

    def dequantise(self, dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values the codes stand for (``out``: contiguous, of this shape)."""
        nat.require_device(self.codes, "MXTensor.dequantise")
        if out is None:
            out = torch.empty(self.shape, dtype=dtype, device=self.device)
        elif out.shape != self.shape or not out.is_contiguous() or out.device != self.device:
            raise ValueError(f"out must be contiguous {tuple(self.shape)} on {self.device}")
        if out.dtype not in _FLOATS:
            raise ValueError(f"float32, bfloat16 or float16 is given, got {out.dtype}")
        with _On(self.device):
            code = nat.load().clt_mx_dequantise(nat.ptr(self.codes), nat.ptr(self.scales), out.numel() // self.width, self.width,
                                                FORMATS[self.fmt], nat.ptr(out), self.width, nat.dtype_code(out.dtype),
                                                nat.current_stream(self.device))
        nat.check(code, "clt_mx_dequantise")
        return out


def quantise(x: torch.Tensor, fmt: str = "mxfp4", out: Optional[MXTensor] = None) -> MXTensor:
    """``x`` [..., d] in the format ``fmt``; ``out``: an `MXTensor` of this shape and format to write into."""
    _format(fmt)
    if x.dim() < 1:
        raise ValueError("quantise needs at least one dimension")
    pitch, blocks = row_layout(x.shape[-1], fmt)
    _check_values(x, "quantise")
    if out is None:
        lead = x.shape[:-1]
        out = MXTensor._made(torch.empty((*lead, pitch), dtype=torch.uint8, device=x.device),
                             torch.empty((*lead, blocks), dtype=torch.uint8, device=x.device), fmt, x.shape[-1])
    elif out.fmt != fmt or out.shape != x.shape or out.device != x.device:
        raise ValueError(f"out is {out.fmt} {tuple(out.shape)} on {out.device}, wanted {fmt} {tuple(x.shape)} on {x.device}")
    if x.numel() == 0:
        return out
    rows = _rows_2d(x)
    if rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        rows = rows.contiguous()                    # an expanded tensor
    with _On(x.device):
        code = nat.load().clt_mx_quantise(nat.ptr(rows), rows.shape[0], rows.shape[1], rows.stride(0), nat.dtype_code(x.dtype),
                                          FORMATS[fmt], nat.ptr(out.codes), nat.ptr(out.scales), nat.current_stream(x.device))
    nat.check(code, "clt_mx_quantise")
    return out


def refresh(x: torch.Tensor, out: MXTensor, state: torch.Tensor, changed: torch.Tensor, store_only: bool = False,
            first: int = 0, n: Optional[int] = None) -> None:
    """Bring the mxfp4 copy ``out`` of weights ``x`` [L, F, d] up to date where they were written since the last call, decided on the
    device: fingerprints of every layer (64 bytes of every row) in ``state`` (int64 [16 L], zeros before the first call) are
    compared, ``changed`` (int32 [L]) says which differ, and those layers are quantised anew.  ``store_only`` records the
    fingerprints of weights that ``out`` was just made from.  ``first``, ``n``: these layers alone (default: all)."""
    _check_values(x, "refresh")
    if x.dim() != 3 or out.fmt != "mxfp4" or out.shape != x.shape or out.device != x.device or x.stride(2) != 1 or x.stride(1) != x.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} must be rows without gaps, out mxfp4 of its shape: got {out.fmt} {tuple(out.shape)}")
    L, F, d = x.shape
    if state.dtype != torch.int64 or state.shape != (16 * L,) or changed.dtype != torch.int32 or changed.shape != (L,):
        raise ValueError(f"state must be int64 [{16 * L}], changed int32 [{L}]")
    if state.device != x.device or changed.device != x.device or not state.is_contiguous() or not changed.is_contiguous():
        raise ValueError(f"state and changed must be contiguous and on {x.device}")
    n = L - first if n is None else n
    if first < 0 or n < 0 or first + n > L:
        raise IndexError(f"layers {first} .. {first + n} are not in weights of {L} layers")
    if n == 0 or F == 0:
        return
    rows = first * F
    with _On(x.device):
        code = nat.load().clt_mx_refresh(
            x.data_ptr() + first * x.stride(0) * x.element_size(), n, F, d, x.stride(0), nat.dtype_code(x.dtype),
            out.codes.data_ptr() + rows * out.codes.shape[2], out.scales.data_ptr() + rows * out.scales.shape[2], state.data_ptr() + 128 * first,
            changed.data_ptr() + 4 * first, 1 if store_only else 0, nat.current_stream(x.device))
    nat.check(code, "clt_mx_refresh")


def project(x: Union[torch.Tensor, MXTensor], w: MXTensor, b: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None, ws=None) -> torch.Tensor:
    """``pre[l] = x[l] @ w[l].T + b[l]`` on the 4-bit matrix cores: ``w`` [L, F, d] in mxfp4, ``x`` [L, T, d] quantised to
    mxfp4 on the way in (or an `MXTensor` that is), fp32 sums, one rounding.  The order of the sums goes by the shapes, where
    ``out`` begins and where in the batch a row lies: calls repeat bit by bit, the same token at another place may differ in its last
    float32 bit.  ``b`` [L, F]; [T, d] with w [F, d] and b [F]
    is one layer.  The result has x's type, or ``out``'s / b's / ``dtype`` where x comes quantised.  ``ws``: an
    `engine.Workspace` to take the scratch memory from."""
    if w.fmt != "mxfp4" or len(w.shape) not in (2, 3):
        raise ValueError(f"the weights must be mxfp4 [L, F, d] or [F, d], got {w.fmt} {tuple(w.shape)}")
    w_shape, x_shape = w.shape, x.shape
    if len(x_shape) != len(w_shape) or x_shape[-1] != w.width or x_shape[:-2] != w_shape[:-2]:
        raise ValueError(f"x {tuple(x_shape)} and weights {tuple(w_shape)} do not belong together")
    device = w.codes.device
    if x.device != device:
        raise ValueError(f"x is on {x.device}, the weights are on {device}")
    if isinstance(x, MXTensor):
        if x.fmt != "mxfp4":
            raise ValueError(f"x must be mxfp4, got {x.fmt}")
        nat.require_device(x.codes, "project")
        dtype = dtype or (out.dtype if out is not None else b.dtype if b is not None else torch.float32)
    else:
        _check_values(x, "project")
        if dtype is not None and dtype != x.dtype:
            raise ValueError(f"the result of {x.dtype} inputs has their type, asked for {dtype}")
        dtype = x.dtype
    if dtype not in _FLOATS:
        raise ValueError(f"float32, bfloat16 or float16 is given, got {dtype}")
    shape = (*x_shape[:-1], w_shape[-2])
    if b is not None and (b.shape != w_shape[:-1] or b.dtype != dtype or b.device != device):
        raise ValueError(f"the bias must be {dtype} {tuple(w_shape[:-1])} on {device}, got {b.dtype} {tuple(b.shape)} on {b.device}")
    if b is not None and b.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("project has no gradient: call it under torch.no_grad() or on detached tensors")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
    elif out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {shape} on {device}")
    if out.numel() == 0:
        return out
    if b is not None and not b.is_contiguous():
        b = b.contiguous()
    given = isinstance(x, MXTensor)
    if not given:
        x = x.contiguous()
        at, to, e = x.data_ptr(), out.data_ptr(), x.element_size()
        if to < at + x.numel() * e and at < to + out.numel() * e:
            raise ValueError("out lies in x: workgroups would read what others have written")
    T, F = shape[-2], shape[-1]
    L = shape[0] if len(shape) == 3 else 1
    lib = nat.load()
    with _On(device):
        nbytes = lib.clt_mx_encode_workspace_bytes(T, w.width, F, L, int(given))
        scratch = None if nbytes == 0 else ws.get("mx_project", nbytes) if ws is not None else torch.empty(nbytes, dtype=torch.uint8, device=device)
        code = lib.clt_mx_encode(nat.ptr(x.codes if given else x), nat.ptr(x.scales if given else None), nat.ptr(w.codes), nat.ptr(w.scales),
                                 nat.ptr(b), nat.ptr(out), T, w.width, F, L, T * w.width, F, T * F, F, nat.dtype_code(dtype),
                                 nat.ptr(scratch), nbytes, nat.current_stream(device))
    nat.check(code, "clt_mx_encode")
    return out


class MXActivationCache:
    """A resident store of activations in a microscaled format: ``rows`` tokens, inputs and targets of every layer.

    Rows are quantised as they are written (a harvest's next rows, or a shuffling buffer's used ones) and gathered,
    expanded and normalised as they are read.  ``codes`` uint8 [L, 2, rows, bytes of a row], ``scales`` uint8
    [L, 2, rows, blocks]; `empty` makes both.  Rows named in a call:

        slice(a, b) or range(a, b)      neighbouring rows
        a sequence or numpy array       any order; checked on the host (IndexError)
        an int32 / int64 tensor         on the cache's device: nothing waits for it.  Rows outside the cache are not
                                        written, and read as NaN

    A row named twice in one write keeps the later of the two.  Calls are launches on the current stream; writes that
    may run at the same time need the caller's ordering, as with any buffer."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, d_model: int):
        held = MXTensor(codes, scales, fmt, d_model)
        if codes.dim() != 4 or codes.shape[1] != 2 or codes.shape[0] < 1:
            raise ValueError(f"codes must be [layers, 2, rows, bytes], got {tuple(codes.shape)}")
        self.codes, self.scales, self.device = held.codes, held.scales, held.codes.device
        self.num_layers, _, self.rows, _ = codes.shape
        if self.rows > 2 ** 31 - 1:
            raise ValueError("a cache holds at most 2^31 - 1 rows")
        self.fmt, self.d_model = fmt, int(d_model)
        self._owner: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, num_layers: int, rows: int, d_model: int, fmt: str = "mxfp8",
              device: Union[str, torch.device] = "cuda:0") -> "MXActivationCache":
        """A cache whose rows read as NaN until they are written."""
        pitch, blocks = row_layout(d_model, fmt)
        return cls(torch.zeros((num_layers, 2, rows, pitch), dtype=torch.uint8, device=device),
                   torch.full((num_layers, 2, rows, blocks), 255, dtype=torch.uint8, device=device), fmt, d_model)

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def _resolve(self, rows: Rows) -> Tuple[Optional[torch.Tensor], int, int]:
        """(row numbers on the device or None, first row, number of rows)."""
        if isinstance(rows, slice):
            if rows.step not in (None, 1):
                raise ValueError("a slice of rows must have step 1")
            first = 0 if rows.start is None else int(rows.start)
            stop = self.rows if rows.stop is None else int(rows.stop)
            rows = range(first, stop)
        if isinstance(rows, range):
            if rows.step != 1:
                raise ValueError("a range of rows must have step 1")
            if len(rows) and (rows.start < 0 or rows.stop > self.rows):
                raise IndexError(f"rows {rows.start} .. {rows.stop} are not in a cache of {self.rows} rows")
            return None, rows.start if len(rows) else 0, len(rows)
        if isinstance(rows, torch.Tensor) and rows.is_cuda:
            if rows.dim() != 1 or rows.dtype not in (torch.int32, torch.int64) or rows.device != self.device:
                raise ValueError(f"rows must be int32 or int64 [n] on {self.device}, got {rows.dtype} {tuple(rows.shape)} on {rows.device}")
            return rows.contiguous(), 0, rows.numel()
        host = np.asarray(rows)
        if host.ndim != 1 or (host.size and host.dtype.kind not in "iu"):
            raise ValueError(f"rows must be one dimension of whole numbers, got {host.dtype} {host.shape}")
        if host.size and (int(host.min()) < 0 or int(host.max()) >= self.rows):
            raise IndexError(f"row index out of range for a cache of {self.rows} rows")
        return torch.from_numpy(host.astype(np.int64)).to(self.device), 0, int(host.size)

    def _batch(self, t: Union[torch.Tensor, Dict[int, torch.Tensor]], n: int, what: str) -> torch.Tensor:
        L, d = self.num_layers, self.d_model
        if isinstance(t, dict):
            if sorted(t) != list(range(L)):
                raise ValueError(f"{what} must hold layers 0 .. {L - 1}, got {sorted(t)}")
            from .encoder import _as_slab
            flats = [t[l].reshape(-1, t[l].shape[-1]) if t[l].dim() != 2 else t[l] for l in range(L)]
            if any(f.shape != flats[0].shape or f.dtype != flats[0].dtype or f.device != flats[0].device for f in flats):
                raise ValueError(f"{what}: all layers must have one shape, type and device")
            t = _as_slab(flats)
        if t.shape != (L, n, d):
            raise ValueError(f"{what} must be [{L}, {n}, {d}], got {tuple(t.shape)}")
        _check_values(t, what)
        if t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        return t

    def write(self, rows: Rows, inputs: Union[torch.Tensor, Dict[int, torch.Tensor]],
              targets: Union[torch.Tensor, Dict[int, torch.Tensor]]) -> None:
        """Quantise ``inputs`` and ``targets`` ([L, n, d] or {layer: [n, d]}, one type) into the rows ``rows``."""
        nat.require_device(self.codes, "MXActivationCache.write")
        index, first, n = self._resolve(rows)
        x, tg = self._batch(inputs, n, "inputs"), self._batch(targets, n, "targets")
        if x.dtype != tg.dtype:
            raise ValueError(f"inputs are {x.dtype}, targets {tg.dtype}")
        if n == 0:
            return
        if x.stride() != tg.stride() or x.stride(2) != 1 or (n > 1 and x.stride(1) < self.d_model) or x.stride(0) < 0:
            x, tg = x.contiguous(), tg.contiguous()
        row_stride = x.stride(1) if n > 1 else self.d_model
        owner = None
        if index is not None:
            if self._owner is None:
                self._owner = torch.empty(self.rows, dtype=torch.int32, device=self.device)
            owner = self._owner
        with _On(self.device):
            code = nat.load().clt_mx_cache_write(
                nat.ptr(x), nat.ptr(tg), x.stride(0), row_stride, nat.dtype_code(x.dtype), nat.ptr(index),
                0 if index is None else 8 * index.element_size(), first, n, self.d_model, self.num_layers, FORMATS[self.fmt],
                nat.ptr(self.codes), nat.ptr(self.scales), self.rows, nat.ptr(owner), nat.current_stream(self.device))
        nat.check(code, "clt_mx_cache_write")

    def read(self, rows: Rows, dtype: torch.dtype = torch.bfloat16, normalization: str = "none",
             tables: Optional[Sequence[Optional[torch.Tensor]]] = None,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, out_row: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """(inputs, targets) [L, n, d] of the rows ``rows``, normalised in fp32 and rounded once to ``dtype``.

        ``normalization``: "none", "mean_std" ((x - mean) / std with ``tables`` = fp32 [L, d] mean and std of the inputs,
        mean and std of the targets; a pair of None leaves that kind as it is) or "sqrt_d_model" (x * sqrt(d)).
        ``out``: two contiguous [L, T, d] tensors of ``dtype``, whose rows out_row, out_row + 1, ... are written."""
        nat.require_device(self.codes, "MXActivationCache.read")
        if normalization not in _NORM_MODES:
            raise ValueError(f"Invalid normalization: {normalization}. Must be one of {list(_NORM_MODES)}")
        if dtype not in _FLOATS:
            raise ValueError(f"float32, bfloat16 or float16 is given, got {dtype}")
        index, first, n = self._resolve(rows)
        L, d = self.num_layers, self.d_model
        if out is None:
            if out_row != 0:
                raise ValueError("out_row without out")
            out, T = (torch.empty((L, n, d), dtype=dtype, device=self.device), torch.empty((L, n, d), dtype=dtype, device=self.device)), n
        else:
            T = out[0].shape[1] if out[0].dim() == 3 else -1
            for t in out:
                if t.shape != (L, T, d) or t.dtype != dtype or t.device != self.device or not t.is_contiguous():
                    raise ValueError(f"out must be two contiguous {dtype} tensors [{L}, T, {d}] on {self.device}")
            if out_row < 0 or out_row + n > T:
                raise ValueError(f"rows {out_row} .. {out_row + n} are not in an output of {T} rows")
        held = (None,) * 4
        if normalization == "mean_std":
            if tables is None or len(tables) != 4 or any((tables[i] is None) != (tables[i + 1] is None) for i in (0, 2)):
                raise ValueError("mean_std needs four tables: mean and std of the inputs, mean and std of the targets")
            for t in tables:
                if t is not None and (t.shape != (L, d) or t.dtype != torch.float32 or t.device != self.device or not t.is_contiguous()):
                    raise ValueError(f"the tables must be contiguous float32 [{L}, {d}] on {self.device}")
            held = tuple(nat.ptr(t) for t in tables)
        if n == 0:
            return out[0], out[1]
        with _On(self.device):
            code = nat.load().clt_mx_cache_read(
                nat.ptr(self.codes), nat.ptr(self.scales), self.rows, FORMATS[self.fmt], nat.ptr(index),
                0 if index is None else 8 * index.element_size(), first, n, d, L, _NORM_MODES[normalization],
                *held, math.sqrt(d) if normalization == "sqrt_d_model" else 1.0, nat.ptr(out[0]), nat.ptr(out[1]),
                out_row, T, nat.dtype_code(dtype), nat.current_stream(self.device))
        nat.check(code, "clt_mx_cache_read")
        return out[0], out[1]
