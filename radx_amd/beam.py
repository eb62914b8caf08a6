"""Beam search beside the sort: a thin Python driver over the radx_hip_beam_* calls of
include/radx_hip.h.  A decoding step is

    scores, parents, tokens = selector.select(logits, cum, k)   # the k best of beams x vocabulary
    beam_reorder(states, parents)                               # their states to their places

and after the last one beam_backtrace(tokens, parents) gives the sequences.  torch is used for device
memory and streams only; the work happens in the library's kernels, none of which has a gradient: results carry
none, and tensors that a call writes count as modified in place.  As for the sort, torch is imported before this
package: it brings a HIP runtime of its own, which the library then shares.
"""
import ctypes
import functools

from . import capi


def _torch():
    """torch, with the types these calls take; looked up once."""
    global _torch
    import torch

    class names:
        f32, i32 = torch.float32, torch.int32
        logits = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
        flags = (torch.bool, torch.uint8)
        empty_like = torch.empty_like
        # the handle alone, which a torch.cuda.Stream would cost a microsecond more for
        raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        # tells autograd that tensors were written, so that a backward pass that still needs their old values raises
        written = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version
    _torch = lambda: names  # noqa: E731
    return names


def _stream(stream, index):
    """The handle of a stream, by default the device's current one."""
    if stream is None:
        return _torch().raw_stream(index)
    if getattr(stream, "device_index", index) != index:
        raise ValueError("the stream is of cuda:%d, expected cuda:%d" % (stream.device_index, index))
    return getattr(stream, "cuda_stream", stream)


def _made_on(stream, index):
    """The context in which a call on another stream makes its outputs, so that their memory is that stream's."""
    import torch
    return torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(stream, device=index))


def _on(t, name, index):
    at = t.get_device()
    if at < 0:
        raise ValueError("%s must be a device tensor" % name)
    if at != index:
        raise ValueError("%s is on cuda:%d, expected cuda:%d" % (name, at, index))


def _plain(t, dtypes, shape, name, index):
    """A contiguous tensor of this device, one of these dtypes and this shape; its address."""
    if t.get_device() != index or index < 0:
        _on(t, name, index)
    if t.dtype not in dtypes:
        raise ValueError("%s must be %s, got %s" % (name, " or ".join(map(str, dtypes)), t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.data_ptr()


class BeamSelector:
    """One radx_hip_beam handle: the scratch of selections within these limits.  One selection may be in
    flight per handle; use one handle per concurrent stream or graph, or put the calls in order.  Selections that overlap on a
    handle get wrong results, without an error; it has to outlive the graphs that captured it."""

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
        left over get -inf, -1, -1.  out: the tensors to write, as returned.  The order in a beam is exact, and
        of different beams' tokens unless their scores are closer than twice what a sum's log may be off by, (3 ln vocab + 5) 2^-24."""
        T, dev = _torch(), self.device
        shape = cum.shape
        if len(shape) != 2:
            raise ValueError("cum must be [batch, beams]")
        batch, beams = shape
        cum_at = _plain(cum, (T.f32,), shape, "cum", dev)
        rows = batch * beams
        if logits.get_device() != dev:
            _on(logits, "logits", dev)
        dtype = T.logits.get(logits.dtype)
        if dtype is None:
            raise ValueError("logits must be float32, bfloat16 or float16, got %s" % logits.dtype)
        has, strides = logits.shape, logits.stride()
        vocab = has[-1]
        if len(has) == 2 and has[0] == rows:
            stride = strides[0]
        elif len(has) == 3 and has[0] == batch and has[1] == beams:
            stride = strides[1] if beams > 1 else strides[0]
            if batch > 1 and strides[0] != beams * stride:
                raise ValueError("logits' rows must be a fixed distance apart")
        else:
            raise ValueError("logits must be [batch * beams, vocab] or [batch, beams, vocab], got %s for cum %s" % (tuple(has), (batch, beams)))
        if strides[-1] != 1 and vocab > 1:
            raise ValueError("the elements of a row of logits must be adjacent")
        if rows <= 1:
            stride = vocab
        allowed_at = allowed_stride = 0
        if allowed is not None:
            _on(allowed, "allowed", dev)
            words = (vocab + 31) // 32
            if allowed.dtype != T.i32 or allowed.dim() != 2 or allowed.shape[0] not in (1, rows) or allowed.shape[1] != words \
                    or (words > 1 and allowed.stride(1) != 1):
                raise ValueError("allowed must be int32 [batch * beams or 1, ceil(vocab / 32)] with adjacent words")
            allowed_at = allowed.data_ptr()
            allowed_stride = allowed.stride(0) if allowed.shape[0] > 1 else 0
        finished_at = ended_at = end = 0
        if finished is not None or end_token is not None:
            if finished is None or end_token is None:
                raise ValueError("finished and end_token go together")
            finished_at = _plain(finished, T.flags, shape, "finished", dev)
            end = int(end_token)
            if not 0 <= end < vocab:
                raise ValueError("end_token %d is outside the vocabulary" % end)
        if not 1 <= k <= capi.BEAM_MAX_K:
            raise ValueError("k must be 1..%d, got %d" % (capi.BEAM_MAX_K, k))
        size, given, handle = (batch, k), out is not None, _stream(stream, dev)
        if not given:
            if stream is None:
                out = self._outputs(T, cum, finished, size)
            else:
                with _made_on(stream, dev):
                    out = self._outputs(T, cum, finished, size)
            at = (out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr())
            if finished_at:
                ended_at = out[3].data_ptr()
        else:
            out = tuple(out)
            if len(out) != (3 if finished is None else 4):
                raise ValueError("out must hold scores, parents, tokens%s" % ("" if finished is None else " and finished flags"))
            at = (_plain(out[0], (T.f32,), size, "out scores", dev), _plain(out[1], (T.i32,), size, "out parents", dev),
                  _plain(out[2], (T.i32,), size, "out tokens", dev))
            if finished_at:
                ended_at = _plain(out[3], T.flags, size, "out finished", dev)
        args = capi.BEAM_SELECT_ARGS.pack(logits.data_ptr(), stride, cum_at, allowed_at, allowed_stride, finished_at, *at, ended_at,
                                          batch, beams, vocab, k, dtype, 1 if normalize else 0, end)
        code = capi.lib.radx_hip_beam_select(self._h, args, handle)
        if code:
            capi.check(code)
        if given:
            T.written(out)
        return out

    @staticmethod
    def _outputs(T, cum, finished, size):
        parents = cum.new_empty(size, dtype=T.i32)  # new_empty: the cheapest of torch's ways
        out = (cum.new_empty(size), parents, T.empty_like(parents))
        return out if finished is None else out + (finished.new_empty(size),)


@functools.lru_cache(maxsize=4096)
def _pieces(shape, src_strides, dst_strides, size, row_dim, length_dim):
    """The rows of a layout as radx_hip_beam_state counts them, strides in bytes:
    (src_row, dst_row, src_outer, dst_outer, outer, unit_bytes, units).  The dimensions are taken in the order in which
    they lie in the memory that is written, whatever their order in the tensor."""
    dims = [(n, s * size, d * size, i == length_dim) for i, (n, s, d) in enumerate(zip(shape, src_strides, dst_strides))
            if i != row_dim and n != 1]
    dims.sort(key=lambda dim: dim[2:0:-1], reverse=True)
    run, units = size, None
    if length_dim is not None and shape[length_dim] == 1:
        units = 1  # the only position: all of the row or nothing
        while dims and dims[-1][1] == run and dims[-1][2] == run:
            run *= dims.pop()[0]
    while dims and units is None and dims[-1][1] == run and dims[-1][2] == run:
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


@functools.lru_cache(maxsize=4096)
def _layout(shape, src_strides, dst_strides, size, row_dim, length_dim, batch):
    """(rows of a batch item, the packed radx_hip_beam_state behind its two addresses) of one state."""
    dim = len(shape)
    row = row_dim + dim if row_dim < 0 else row_dim
    if not 0 <= row < dim:
        raise ValueError("a state has no dimension %d" % row_dim)
    if shape[row] % batch:
        raise ValueError("dimension %d of a state has %d rows, which is not the same number for each of %d items" % (row_dim, shape[row], batch))
    length = None
    if length_dim is not None:
        length = length_dim + dim if length_dim < 0 else length_dim
        if not 0 <= length < dim or length == row:
            raise ValueError("length_dim must be a dimension of every state, and not its rows'")
    if 0 in shape:
        return shape[row] // batch, None
    src_row, dst_row, src_outer, dst_outer, outer, unit, units = _pieces(shape, src_strides, dst_strides, size, row, length)
    return shape[row] // batch, capi.BEAM_STATE.pack(0, 0, src_row, dst_row, *src_outer, *dst_outer, unit, units, *outer)[16:]


def beam_reorder(states, parents, into=None, lengths=None, length_dim=None, row_dim=0, stream=None):
    """Moves the survivors' states to their places, all of them in one launch: with parents int32 [batch, k] (k <= 64)
    and `beams` rows an item in dimension row_dim of every state,

        state[b * beams + j] = state[b * beams + parents[b, j]]     for j < k, as if all were read first

    Rows whose parent is < 0 or >= beams, and rows k.. of an item, are left as they were.  states: a tensor or a
    sequence of them, any dtypes and layouts of whole rows (up to two strided dimensions around contiguous
    pieces, in any order of the tensor's dimensions); they must not share memory with each other.  into: as many tensors
    that get the rows instead (b * k + j), apart from the states.  lengths: int32 [batch]; of dimension length_dim only the
    first lengths[b] positions move, what lies behind is neither read nor written.  The bytes of a position, and those of
    the positions after it, must follow each other in memory (what a row has more than one of, such as heads, may lie
    around them; a cache whose positions lie outside its rows has no lengths)."""
    states = (states,) if hasattr(states, "data_ptr") else tuple(states)
    if into is not None:
        into = (into,) if hasattr(into, "data_ptr") else tuple(into)
        if len(into) != len(states):
            raise ValueError("into must hold one tensor for each state")
    T = _torch()
    shape = parents.shape
    if len(shape) != 2:
        raise ValueError("parents must be [batch, k]")
    batch, k = shape
    dev = parents.get_device()
    parents_at = _plain(parents, (T.i32,), shape, "parents", dev)
    lengths_at = None
    if lengths is not None or length_dim is not None:
        if lengths is None or length_dim is None:
            raise ValueError("lengths and length_dim go together")
        lengths_at = _plain(lengths, (T.i32,), (batch,), "lengths", dev)
    if batch == 0 or k == 0:
        return
    table, beams, address = [], None, capi.ADDRESSES.pack
    like_shape = like_strides = like_d_strides = like_dtype = packed = None
    for i, s in enumerate(states):
        if s.get_device() != dev:
            _on(s, "a state", dev)
        has, strides, dtype = s.shape, s.stride(), s.dtype
        at = d_at = s.data_ptr()
        d_strides = strides
        if into is not None:
            d = into[i]
            _on(d, "into", dev)
            row = row_dim + len(has) if row_dim < 0 else row_dim
            if d.dtype != dtype or d.shape != tuple(batch * k if n == row else size for n, size in enumerate(has)):
                raise ValueError("into must have the states' dtypes and shapes, with batch * k rows")
            d_strides, d_at = d.stride(), d.data_ptr()
        if has != like_shape or strides != like_strides or d_strides != like_d_strides or dtype is not like_dtype:  # they are often alike
            like_shape, like_strides, like_d_strides, like_dtype = has, strides, d_strides, dtype
            rows, packed = _layout(has, strides, d_strides, s.element_size(), row_dim, length_dim, batch)
            if rows != beams:
                if beams is not None:
                    raise ValueError("the states have different numbers of rows")
                beams = rows
        if packed is not None:
            table += (address(at, d_at), packed)
    if not table or not beams:
        return
    code = capi.lib.radx_hip_beam_reorder(b"".join(table), len(table) // 2, parents_at, lengths_at, batch, beams, beams if into is None else k, k,
                                          _stream(stream, dev))
    if code:
        capi.check(code)
    T.written(states if into is None else into)


def beam_backtrace(tokens, parents, steps=None, out=None, stream=None):
    """The sequences [batch, k, T] of the last step's places, out of the recorded tokens and parents, int32
    [T, batch, k]: out[b, j, t] is the token of step t on the way to place j of step L - 1, with L = steps[b] (int32
    [batch]; None: T).  A parent < 0 or >= k stands for the same place.  Elements from L on are left as they
    were (-1 where `out` is not given)."""
    T = _torch()
    shape = tokens.shape
    if len(shape) != 3:
        raise ValueError("tokens must be [steps, batch, k]")
    total, batch, k = shape
    dev = tokens.get_device()
    tokens_at = _plain(tokens, (T.i32,), shape, "tokens", dev)
    parents_at = _plain(parents, (T.i32,), shape, "parents", dev)
    steps_at = None if steps is None else _plain(steps, (T.i32,), (batch,), "steps", dev)
    handle = _stream(stream, dev)
    if out is None:
        if stream is not None:
            with _made_on(stream, dev):
                return beam_backtrace(tokens, parents, steps, tokens.new_empty((batch, k, total)) if steps is None else
                                      tokens.new_full((batch, k, total), -1), stream)
        out = tokens.new_empty((batch, k, total)) if steps is None else tokens.new_full((batch, k, total), -1)
    _on(out, "out", dev)
    strides = out.stride()
    if out.dtype != T.i32 or out.shape != (batch, k, total) or (total > 1 and strides[2] != 1) or \
            (batch > 1 and k > 1 and strides[0] != k * strides[1]):
        raise ValueError("out must be int32 [batch, k, steps], its sequences contiguous and a fixed distance apart")
    if total == 0 or batch == 0 or k == 0:
        return out
    stride = strides[1] if k > 1 else strides[0] if batch > 1 else total
    code = capi.lib.radx_hip_beam_backtrace(tokens_at, parents_at, steps_at, total, batch, k, out.data_ptr(), stride, handle)
    if code:
        capi.check(code)
    T.written((out,))
    return out
