"""The losses that open a training step's backward pass, over the C ABI of libb200amp.so.

    begin_step            inv_scale, found_inf                            (amp.begin_step)
    forward pass          logits, router logits
    distill_loss          loss and n_valid into the step state, loss-scaled gradient of the logits
    balance_loss          per-expert counts, loss-scaled gradient of a router's logits
    backward pass         fp16 gradient arena
    optimizer step        (amp.AmpOptimizer.optimizer_step; the finalize carries loss and n_valid into the history)

top_logits makes the record of a teacher's largest logits that distill_loss reads. The full contract of each call
is in include/b200amp.h. As everywhere in this package the caller owns every buffer: the calls allocate nothing,
enqueue on `stream` (a torch stream, a raw handle, or None for the current stream of the tensors' device) and
return without a host sync; they can be captured into a CUDA graph. Matrices are 2-D tensors with unit column
stride and any row stride, fp16, bf16 or fp32; all tensors of a call are on one device, which need not be the
current one. Errors raise: ValueError for a tensor of the wrong shape, type or device, B200AmpError for what the
library refuses.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import LOSS_WORKSPACE_BYTES, check

__all__ = ["top_logits", "distill_loss", "balance_loss", "loss_workspace", "LossCalls"]

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_STATE_BYTES = 60


# the handle alone: building a Stream object for every call costs more than the rest of the call's Python
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def loss_workspace(device="cuda") -> torch.Tensor:
    """The workspace of distill_loss and balance_loss, zeroed. One serves one stream at a time."""
    return torch.zeros(LOSS_WORKSPACE_BYTES, dtype=torch.uint8, device=device)


def _matrix(t: torch.Tensor, name: str, device: int = -1):
    """(pointer, row stride in elements, rows, columns, type code, device) of a 2-D CUDA tensor."""
    code, on = _DTYPES.get(t.dtype), t.get_device()     # -1: not on a GPU
    if t.dim() != 2 or on < 0 or code is None:
        raise ValueError(f"{name}: expected a 2-D CUDA tensor of fp16, bf16 or fp32, got {t.dim()}-D {t.dtype} on {t.device}")
    if device >= 0 and on != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name}: the columns of a row must be next to each other (strides {t.stride()})")
    return t.data_ptr(), (ld if rows > 1 else cols), rows, cols, code, on


def _array(t: Optional[torch.Tensor], name: str, dtype, shape, device: int) -> Optional[int]:
    """Pointer of a contiguous tensor of this type and shape, or None for None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on cuda:{device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _bytes(t: torch.Tensor, name: str, least: int, device: int) -> int:
    if t.get_device() != device or not t.is_contiguous() or t.nbytes < least:
        raise ValueError(f"{name}: expected a contiguous tensor of {least} bytes or more on cuda:{device}")
    return t.data_ptr()


def _call(fn, device: int, stream, *args) -> None:
    """fn(*args, stream) with the tensors' device current; raises what the library refuses."""
    if stream is None:
        handle = _current_stream(device)
    else:
        handle = stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else int(stream)
    if torch.cuda.current_device() == device:
        status = fn(*args, handle)
    else:
        with torch.cuda.device(device):
            status = fn(*args, handle)
    if status != _lib.OK:
        check(status)


def top_logits(logits: torch.Tensor, k: int, values: torch.Tensor, indices: torch.Tensor,
               lse: Optional[torch.Tensor] = None, vocab: Optional[int] = None, temperature: float = 1.0,
               stream=None) -> None:
    """The k largest of every row's first `vocab` columns (default: all of them) into values[rows, k] (the
    logits' type) and indices[rows, k] (int32), in descending order, ties to the lowest column; and, if lse is
    given, log sum exp(z / temperature) over the row into lse[rows] (fp32)."""
    ptr, ld, rows, cols, dtype, dev = _matrix(logits, "logits")
    vocab = cols if vocab is None else vocab
    if not 1 <= vocab <= cols:
        raise ValueError(f"vocab = {vocab}: the logits have {cols} columns")
    _call(_lib.load().b200amp_top_logits, dev, stream, ptr, dtype, rows, vocab, ld, k, temperature,
          _array(values, "values", logits.dtype, (rows, k), dev), _array(indices, "indices", torch.int32, (rows, k), dev),
          _array(lse, "lse", torch.float32, (rows,), dev))


def distill_loss(logits: torch.Tensor, dlogits: Optional[torch.Tensor], targets: Optional[torch.Tensor],
                 values: Optional[torch.Tensor], indices: Optional[torch.Tensor], lse: Optional[torch.Tensor],
                 state: torch.Tensor, row_loss: torch.Tensor, workspace: torch.Tensor, vocab: Optional[int] = None,
                 temperature: float = 1.0, soft_weight: float = 1.0, hard_weight: float = 0.0, stream=None) -> None:
    """soft_weight * KL(teacher || student) at `temperature` + hard_weight * cross-entropy, averaged over the rows
    with targets >= 0: row_loss[rows], state.loss, state.n_valid, and (dlogits not None) the gradient times the
    state's loss scale. values / indices [rows, k] are the teacher's listed logits (index < 0: empty slot), lse
    its log-sum-exp at the same temperature, or None to normalise over the listed logits alone. Columns from
    `vocab` on pad the vocabulary. dlogits may be logits itself. Without a teacher pass None for the three."""
    ptr, ld, rows, cols, dtype, dev = _matrix(logits, "logits")
    vocab = cols if vocab is None else vocab
    dptr, dld = None, cols
    if dlogits is not None:
        dptr, dld, drows, dcols, ddtype, _ = _matrix(dlogits, "dlogits", dev)
        if drows != rows or dcols != cols or ddtype != dtype:
            raise ValueError(f"dlogits: expected {logits.dtype} {tuple(logits.shape)}, got {dlogits.dtype} {tuple(dlogits.shape)}")
    k, vtype = 0, dtype
    if values is not None:
        if values.dim() != 2 or values.dtype not in _DTYPES or indices is None:
            raise ValueError("values: expected a 2-D tensor of fp16, bf16 or fp32, and indices with it")
        k, vtype = values.shape[1], _DTYPES[values.dtype]
    elif indices is not None or lse is not None:
        raise ValueError("indices and lse belong to values: pass all, or None for each")
    _call(_lib.load().b200amp_distill_loss, dev, stream, ptr, ld, dptr, dld, dtype, rows, vocab, cols,
          _array(targets, "targets", torch.int32, (rows,), dev),
          _array(values, "values", None if values is None else values.dtype, (rows, k), dev), vtype,
          _array(indices, "indices", torch.int32, (rows, k), dev), _array(lse, "lse", torch.float32, (rows,), dev), k,
          temperature, soft_weight, hard_weight, _bytes(state, "state", _STATE_BYTES, dev),
          _array(row_loss, "row_loss", torch.float32, (rows,), dev),
          _bytes(workspace, "workspace", LOSS_WORKSPACE_BYTES, dev))


def balance_loss(logits: torch.Tensor, dlogits: Optional[torch.Tensor], chosen: torch.Tensor,
                 targets: Optional[torch.Tensor], state: torch.Tensor, counts: torch.Tensor, loss: torch.Tensor,
                 workspace: torch.Tensor, weight: float = 0.01, accumulate: bool = False, add_to_state: bool = False,
                 stream=None) -> None:
    """weight * experts * sum_e (share of the choices that fell on e) * (mean probability of e) over the rows with
    targets >= 0 (None: all): loss[1], the choices of each expert into counts[experts] (int32), and (dlogits not
    None) the gradient times the state's loss scale, added to dlogits if accumulate. chosen[rows, k] (int32) are
    the router's choices, negative where one was not made. add_to_state adds the loss to state.loss."""
    ptr, ld, rows, experts, dtype, dev = _matrix(logits, "logits")
    dptr, dld = None, experts
    if dlogits is not None:
        dptr, dld, drows, dcols, ddtype, _ = _matrix(dlogits, "dlogits", dev)
        if drows != rows or dcols != experts or ddtype != dtype:
            raise ValueError(f"dlogits: expected {logits.dtype} {tuple(logits.shape)}, got {dlogits.dtype} {tuple(dlogits.shape)}")
    if chosen.dim() != 2:
        raise ValueError(f"chosen: expected a 2-D tensor, got {chosen.dim()}-D")
    k = chosen.shape[1]
    _call(_lib.load().b200amp_balance_loss, dev, stream, ptr, ld, dptr, dld, dtype, rows, experts,
          _array(chosen, "chosen", torch.int32, (rows, k), dev), k, _array(targets, "targets", torch.int32, (rows,), dev),
          weight, 1 if accumulate else 0, 1 if add_to_state else 0, _bytes(state, "state", _STATE_BYTES, dev),
          _array(counts, "counts", torch.int32, (experts,), dev), _array(loss, "loss", torch.float32, (1,), dev),
          _bytes(workspace, "workspace", LOSS_WORKSPACE_BYTES, dev))


class LossCalls:
    """The losses on an optimizer's own step state: mixed into the owners of amp.py, which provide state and
    loss_workspace (both on the optimizer's device). That workspace serves one stream at a time, like any other: calls
    whose GPU work may overlap (streams side by side, two graphs replayed at once) each bring a `workspace` of their
    own (loss_workspace()). Calls that write or add to state.loss are to follow one another in any case."""

    def distill_loss(self, logits, dlogits, targets, values, indices, lse, row_loss, vocab=None, temperature=1.0,
                     soft_weight=1.0, hard_weight=0.0, stream=None, workspace=None) -> None:
        distill_loss(logits, dlogits, targets, values, indices, lse, self.state, row_loss,
                     self.loss_workspace if workspace is None else workspace, vocab, temperature, soft_weight, hard_weight,
                     stream)

    def balance_loss(self, logits, dlogits, chosen, targets, counts, loss, weight=0.01, accumulate=False,
                     add_to_state=True, stream=None, workspace=None) -> None:
        balance_loss(logits, dlogits, chosen, targets, self.state, counts, loss,
                     self.loss_workspace if workspace is None else workspace, weight, accumulate, add_to_state, stream)
