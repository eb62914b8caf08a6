"""Beam search beside the sort: a thin Python driver over the radx_hip_beam_* calls of
include/radx_hip.h.  A decoding step is

    scores, parents, tokens = selector.select(logits, cum, k)   # the k best of beams x vocabulary
    beam_reorder(states, parents)                               # their states to their places

and after the last one beam_backtrace(tokens, parents) gives the sequences.  torch is used for device
memory and streams only; the work happens in the library's kernels.
"""
import ctypes
import functools

from . import capi
from .sorter import _ptr, _stream

_DTYPES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2}
_FLAGS = ("torch.bool", "torch.uint8")


def _on(t, name, index):
    if not t.is_cuda:
        raise ValueError("%s must be a device tensor" % name)
    if t.device.index != index:
        raise ValueError("%s is on %s, expected cuda:%d" % (name, t.device, index))


def _plain(t, dtypes, shape, name, index):
    """A contiguous tensor of this device, one of these dtypes and this shape."""
    _on(t, name, index)
    if str(t.dtype) not in dtypes:
        raise ValueError("%s must be %s, got %s" % (name, " or ".join(dtypes), t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


class BeamSelector:
    """One radx_hip_beam handle: the scratch of selections within these limits.  One selection may be in
    flight per handle; use one handle per concurrent stream or graph."""

    def __init__(self, max_batch, max_beams, max_vocab, max_k, device=0):
        self.device = device
        self._h = ctypes.c_void_p(None)
        capi.check(capi.lib.radx_hip_beam_create(device, max_batch, max_beams, max_vocab, max_k, ctypes.byref(self._h)))

    def close(self):
        if self._h:
            capi.check(capi.lib.radx_hip_beam_destroy(self._h))
            self._h = ctypes.c_void_p(None)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def select(self, logits, cum, k, allowed=None, finished=None, end_token=None, normalize=True, out=None, stream=None):
        """The k best continuations of every batch item, best first: (scores, parents, tokens), each [batch, k],
        float32 and int32, and the places' finished flags as a fourth where `finished` is given.

        logits [batch * beams, vocab] or [batch, beams, vocab], float32, bfloat16 or float16, elements of a row
        adjacent, rows a fixed distance apart; cum [batch, beams] float32.  normalize: the scores are cum +
        log_softmax(logits), otherwise cum + logits.  allowed: int32 words [batch * beams or 1, ceil(vocab / 32)], bit
        v & 31 of word v >> 5 admits token v.  finished: bool or uint8 [batch, beams]; such a beam offers end_token
        at its own score.  Equal scores go to the lower beam, the larger logit, the lower token; places that are
        left over get -inf, -1, -1.  out: the tensors to write, as returned."""
        import torch
        dev = self.device
        _on(logits, "logits", dev)
        dtype = _DTYPES.get(str(logits.dtype))
        if dtype is None:
            raise ValueError("logits must be float32, bfloat16 or float16, got %s" % logits.dtype)
        if cum.dim() != 2:
            raise ValueError("cum must be [batch, beams]")
        batch, beams = cum.shape
        _plain(cum, ("torch.float32",), cum.shape, "cum", dev)
        rows, vocab = batch * beams, logits.shape[-1]
        if logits.dim() == 3 and tuple(logits.shape[:2]) == (batch, beams):
            stride = logits.stride(1) if beams > 1 else logits.stride(0)
            if batch > 1 and logits.stride(0) != beams * stride:
                raise ValueError("logits' rows must be a fixed distance apart")
        elif logits.dim() == 2 and logits.shape[0] == rows:
            stride = logits.stride(0)
        else:
            raise ValueError("logits must be [batch * beams, vocab] or [batch, beams, vocab], got %s for cum %s" % (tuple(logits.shape), (batch, beams)))
        if vocab > 1 and logits.stride(-1) != 1:
            raise ValueError("the elements of a row of logits must be adjacent")
        if rows <= 1:
            stride = vocab
        a = capi.BeamSelectArgs()
        if allowed is not None:
            _on(allowed, "allowed", dev)
            words = (vocab + 31) // 32
            if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[0] not in (1, rows) or allowed.shape[1] != words \
                    or (words > 1 and allowed.stride(1) != 1):
                raise ValueError("allowed must be int32 [batch * beams or 1, ceil(vocab / 32)] with adjacent words")
            a.allowed = allowed.data_ptr()
            a.allowed_stride = allowed.stride(0) if allowed.shape[0] > 1 else 0
        if (finished is None) != (end_token is None):
            raise ValueError("finished and end_token go together")
        if finished is not None:
            _plain(finished, _FLAGS, cum.shape, "finished", dev)
            a.finished = finished.data_ptr()
            a.end_token = int(end_token)
        if out is None:
            where = cum.device
            scores = torch.empty((batch, k), dtype=torch.float32, device=where)
            both = torch.empty((2, batch, k), dtype=torch.int32, device=where)
            out = (scores, both[0], both[1])
            if finished is not None:
                out += (torch.empty((batch, k), dtype=finished.dtype, device=where),)
        else:
            out = tuple(out)
            if len(out) != (3 if finished is None else 4):
                raise ValueError("out must hold scores, parents, tokens%s" % ("" if finished is None else " and finished flags"))
            for t, dtypes, name in zip(out, (("torch.float32",), ("torch.int32",), ("torch.int32",), _FLAGS),
                                       ("out scores", "out parents", "out tokens", "out finished")):
                _plain(t, dtypes, (batch, k), name, dev)
        a.logits, a.row_stride, a.cum = logits.data_ptr(), stride, cum.data_ptr()
        a.scores, a.parents, a.tokens = out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr()
        if finished is not None:
            a.out_finished = out[3].data_ptr()
        a.batch, a.beams, a.vocab, a.k = batch, beams, vocab, k
        a.dtype, a.normalize = dtype, 1 if normalize else 0
        capi.check(capi.lib.radx_hip_beam_select(self._h, ctypes.byref(a), _stream(stream, dev)))
        return out


@functools.lru_cache(maxsize=1024)
def _pieces(shape, src_strides, dst_strides, size, row_dim, length_dim):
    """The rows of a layout as radx_hip_beam_state counts them, strides in bytes:
    (src_row, dst_row, src_outer, dst_outer, outer, unit_bytes, units)."""
    dims = [(n, s * size, d * size, i == length_dim) for i, (n, s, d) in enumerate(zip(shape, src_strides, dst_strides))
            if i != row_dim and (n != 1 or i == length_dim)]
    run, units = size, None
    while dims and units is None and ((dims[-1][1] == run and dims[-1][2] == run) or (dims[-1][3] and dims[-1][0] == 1)):
        n, _, _, counted = dims.pop()
        if counted:
            units = n
        else:
            run *= n
    if length_dim is not None and units is None:
        raise ValueError("what lies behind a position in the length dimension must be contiguous")
    outer = []
    for n, s, d, _ in dims:
        if outer and outer[-1][1] == n * s and outer[-1][2] == n * d:
            outer[-1] = (outer[-1][0] * n, s, d)
        else:
            outer.append((n, s, d))
    if len(outer) > 2:
        raise ValueError("a row of a state is scattered over more than two strided dimensions")
    outer = [(1, 0, 0)] * (2 - len(outer)) + outer
    return (src_strides[row_dim] * size, dst_strides[row_dim] * size, (outer[0][1], outer[1][1]), (outer[0][2], outer[1][2]),
            (outer[0][0], outer[1][0]), run, 1 if units is None else units)


def beam_reorder(states, parents, into=None, lengths=None, length_dim=None, row_dim=0, stream=None):
    """Moves the survivors' states to their places, all of them in one launch: with parents int32 [batch, k] (k <= 64)
    and `beams` rows an item in dimension row_dim of every state,

        state[b * beams + j] = state[b * beams + parents[b, j]]     for j < k, as if all were read first

    Rows whose parent is < 0 or >= beams, and rows k.. of an item, are left as they were.  states: a tensor or a
    sequence of them, any dtypes and layouts of whole rows (up to two strided dimensions around contiguous
    pieces); they must not share memory with each other.  into: as many tensors that get the rows instead (b * k + j),
    apart from the states.  lengths: int32 [batch]; of dimension length_dim only the first lengths[b] positions
    move, what lies behind is neither read nor written."""
    states = [states] if hasattr(states, "data_ptr") else list(states)
    into_list = None if into is None else [into] if hasattr(into, "data_ptr") else list(into)
    if parents.dim() != 2:
        raise ValueError("parents must be [batch, k]")
    batch, k = parents.shape
    dev = parents.device.index
    _plain(parents, ("torch.int32",), parents.shape, "parents", dev)
    if (lengths is None) != (length_dim is None):
        raise ValueError("lengths and length_dim go together")
    if lengths is not None:
        _plain(lengths, ("torch.int32",), (batch,), "lengths", dev)
    if into_list is not None and len(into_list) != len(states):
        raise ValueError("into must hold one tensor for each state")
    if not states or batch == 0 or k == 0:
        return
    table = (capi.BeamState * len(states))()
    beams = None
    for i, s in enumerate(states):
        d = s if into_list is None else into_list[i]
        _on(s, "a state", dev)
        dim = s.dim()
        row = row_dim + dim if row_dim < 0 else row_dim
        if not 0 <= row < dim:
            raise ValueError("a state has no dimension %d" % row_dim)
        if s.shape[row] % batch or (beams is not None and s.shape[row] != beams * batch):
            raise ValueError("dimension %d of a state has %d rows, which is not the same number for each of %d items" % (row_dim, s.shape[row], batch))
        beams = s.shape[row] // batch
        length = None
        if length_dim is not None:
            length = length_dim + dim if length_dim < 0 else length_dim
            if not 0 <= length < dim or length == row:
                raise ValueError("length_dim must be a dimension of every state, and not its rows'")
        if d is not s:
            _on(d, "into", dev)
            if d.dtype != s.dtype or d.dim() != dim or d.shape[row] != batch * k or d.shape[:row] != s.shape[:row] or d.shape[row + 1:] != s.shape[row + 1:]:
                raise ValueError("into must have the states' dtypes and shapes, with batch * k rows")
        if s.numel() == 0:
            continue
        t = table[i]
        (t.src_row, t.dst_row, (t.src_outer[0], t.src_outer[1]), (t.dst_outer[0], t.dst_outer[1]), (t.outer[0], t.outer[1]),
         t.unit_bytes, t.units) = _pieces(s.shape, s.stride(), d.stride(), s.element_size(), row, length)
        t.src, t.dst = s.data_ptr(), d.data_ptr()
    if not beams:
        return
    capi.check(capi.lib.radx_hip_beam_reorder(table, len(states), _ptr(parents), _ptr(lengths), batch, beams, beams if into_list is None else k, k,
                                              _stream(stream, dev)))


def beam_backtrace(tokens, parents, steps=None, out=None, stream=None):
    """The sequences [batch, k, T] of the last step's places, out of the recorded tokens and parents, int32
    [T, batch, k]: out[b, j, t] is the token of step t on the way to place j of step L - 1, with L = steps[b] (int32
    [batch]; None: T).  A parent < 0 or >= k stands for the same place.  Elements from L on are left as they
    were (-1 where `out` is not given)."""
    if tokens.dim() != 3:
        raise ValueError("tokens must be [steps, batch, k]")
    total, batch, k = tokens.shape
    import torch
    dev = tokens.device.index
    _plain(tokens, ("torch.int32",), tokens.shape, "tokens", dev)
    _plain(parents, ("torch.int32",), tokens.shape, "parents", dev)
    if steps is not None:
        _plain(steps, ("torch.int32",), (batch,), "steps", dev)
    if out is None:
        out = torch.empty((batch, k, total), dtype=torch.int32, device=tokens.device)
        if steps is not None:
            out.fill_(-1)
    _on(out, "out", dev)
    if out.dtype != torch.int32 or tuple(out.shape) != (batch, k, total) or (total > 1 and out.stride(2) != 1) or \
            (batch > 1 and k > 1 and out.stride(0) != k * out.stride(1)):
        raise ValueError("out must be int32 [batch, k, steps], its sequences contiguous and a fixed distance apart")
    if total == 0 or batch == 0 or k == 0:
        return out
    stride = out.stride(1) if k > 1 else out.stride(0) if batch > 1 else total
    capi.check(capi.lib.radx_hip_beam_backtrace(_ptr(tokens), _ptr(parents), _ptr(steps), total, batch, k, _ptr(out), stride, _stream(stream, dev)))
    return out
