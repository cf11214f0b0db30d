"""The paged-cache operators over torch tensors: append, attention, eviction, beam selection.

Each class binds one C-ABI entry point of include/pim_b200.h to a set of device tensors:
shapes, types and layouts are checked once, the argument struct and the workspace are made
once (as ``cuda_kernels.lower_launch`` does for plan commands), and a call enqueues the
kernels on the device's current stream and returns the outputs.  Nothing is copied and
nothing is synchronised, so a call can be captured into a CUDA graph; lengths, positions and
tables are read on the device, so a replay sees their new values.

    append = PagedAppend(k, v, cache.k(0), cache.v(0), cache.table, cache.lengths, cache.next_lengths,
                         q=q, q_out=q_rot, cos=cos, sin=sin)
    attend = PagedAttention(q_rot, cache.k(0), cache.v(0), cache.table, cache.next_lengths, out)
    append(); attend()

Pages are ``[num_pages, kv_heads, page_size, head_dim]`` tensors (one for K, one for V, both
with the same stride between pages), float32 or bfloat16.  An operator owns its workspace:
its calls, and replays of graphs that hold them, must not overlap on the GPU; make another one
for another stream.  Its tensors must stay alive while a graph that holds a call can be
replayed: keep the operator.  A bad length, position, page id, parent or logit found on the device
raises the operator's error flag, which ``check()`` turns into an exception (it waits for the device).
"""

from __future__ import annotations

import ctypes
import operator

from backend import _native as nat

_CODES = {"torch.float32": nat.F32, "torch.bfloat16": nat.BF16}


def _code(t, what: str) -> int:
    if str(t.dtype) not in _CODES:
        raise ValueError(f"{what}: dtype {t.dtype} has no kernel (float32 or bfloat16)")
    return _CODES[str(t.dtype)]


def _want(t, what: str, shape, dtype: str, contiguous: bool = True):
    """``t`` has ``shape`` (None: any size) and dtype; contiguous, or at least in its last dimension."""
    if len(t.shape) != len(shape) or any(w is not None and s != w for s, w in zip(t.shape, shape)):
        raise ValueError(f"{what}: expected shape {tuple('any' if w is None else w for w in shape)}, got {tuple(t.shape)}")
    if str(t.dtype) != f"torch.{dtype}":
        raise ValueError(f"{what}: expected {dtype}, got {t.dtype}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    if not contiguous and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: its last dimension must be contiguous")
    return t


def _int32(value, what: str) -> int:
    """``value`` as the argument structs hold it (ctypes would cut it down to 32 bits without a word)."""
    value = operator.index(value)
    if not -2**31 <= value < 2**31:
        raise ValueError(f"{what}={value} does not fit 32 bits")
    return value


def _dt(t) -> str:
    return str(t.dtype).removeprefix("torch.")


def _span(t) -> tuple[int, int]:
    """First byte of a tensor's memory and the one behind its last."""
    at = t.data_ptr()
    if t.is_contiguous():
        return at, at + t.numel() * t.element_size()
    return at, at + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else at


def _meet(a, b) -> bool:
    return a[0] < b[1] and b[0] < a[1]


def _overlap(a, b) -> bool:
    """Whether two tensors' memory ranges meet."""
    return _meet(_span(a), _span(b))


def _layout(t):
    """(elements, byte stride) of the dimensions of more than one element, the widest stride first."""
    item = t.element_size()
    return sorted(((n, st * item) for n, st in zip(t.shape, t.stride()) if n > 1), key=lambda d: -d[1])


def _share(a, b) -> bool:
    """Whether two tensors whose ranges meet share a byte.  Told exactly for tensors of equal strides (parts of one buffer's
    rows); others are taken to."""
    da, db = _layout(a), _layout(b)
    if [st for _, st in da] != [st for _, st in db]:
        return True
    ia, ib = a.element_size(), b.element_size()
    # an element of b lies `at` + sum of (difference of indices) x stride behind one of a
    dims = [(na, nb, st) for (na, st), (nb, _) in zip(da, db)]

    def meets(at: int, k: int) -> bool:
        if k == len(dims):
            return -ib < at < ia
        na, nb, st = dims[k]
        # the inner dimensions' differences lie between -(a's extent) and b's
        down = sum((n - 1) * s for _, n, s in dims[k + 1:]) + ib - 1
        up = sum((n - 1) * s for n, _, s in dims[k + 1:]) + ia - 1
        if st == 0:
            return meets(at, k + 1)
        first, last = max(-(na - 1), -((at + down) // st)), min(nb - 1, (up - at) // st)
        if last - first > 16:  # (strides that nest in no order)
            return True
        return any(meets(at + i * st, k + 1) for i in range(first, last + 1))

    return meets(b.data_ptr() - a.data_ptr(), 0)


def _rows_apart(a, b) -> bool:
    """Whether two [tokens, heads, head_dim] views share no element; views of one buffer of equal rows (the parts of a
    fused qkv row) are told apart by where in the row they lie."""
    if not _overlap(a, b):
        return True
    pitch = a.stride(0)
    if a.shape[0] < 2 or b.shape[0] < 2 or b.stride(0) != pitch:
        return False

    def width(t):
        return sum((n - 1) * st for n, st in zip(t.shape[1:], t.stride()[1:])) + 1

    d = (b.data_ptr() - a.data_ptr()) // a.element_size() % pitch
    return width(a) <= d <= pitch - width(b)


def _apart(outputs: dict, others: dict) -> None:
    """No output shares memory with another output or with an input."""
    outs = [(n, t, _span(t)) for n, t in outputs.items() if t is not None]
    ins = [(n, t, _span(t)) for n, t in others.items() if t is not None]
    for i, (n, t, span) in enumerate(outs):
        for m, other, where in outs[i + 1:] + ins:
            if _meet(span, where) and _share(t, other):
                raise ValueError(f"{n} shares memory with {m}")


def _paged_kv(k_pages, v_pages, table) -> nat.PagedKV:
    num, heads, ps, hd = k_pages.shape if k_pages.dim() == 4 else (None,) * 4
    if num is None or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise ValueError("k_pages and v_pages: expected two [num_pages, kv_heads, page_size, head_dim] tensors of one "
                         f"type, got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    inner = (ps * hd, hd, 1)
    for name, p in (("k_pages", k_pages), ("v_pages", v_pages)):
        if any(n > 1 and s != w for n, s, w in zip(p.shape[1:], p.stride()[1:], inner)):
            raise ValueError(f"{name}: each page must be contiguous")
    stride = k_pages.stride(0) if num > 1 else heads * ps * hd
    if num > 1 and v_pages.stride(0) != stride:
        raise ValueError("k_pages and v_pages: the stride between pages must be the same")
    _apart(dict(k_pages=k_pages), dict(v_pages=v_pages))
    _want(table, "table", (None, None), "int32", contiguous=False)
    return nat.PagedKV(k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(), page_stride=stride,
                       table=table.data_ptr(), table_stride=table.stride(0) if table.shape[0] > 1 else table.shape[1],
                       rows=table.shape[0], max_pages=table.shape[1], num_pages=num, page_size=ps, kv_heads=heads,
                       head_dim=hd)


def _state(t, what: str, rows: int, heads: int, slots: int, dtype: str):
    _want(t, what, (rows, heads, None), dtype, contiguous=False)
    if t.shape[2] < slots:
        raise ValueError(f"{what}: {t.shape[2]} slots a row, the table holds {slots}")
    return t


def _state_strides(t) -> tuple[int, int]:
    """(row, head) strides of a state array; a dimension of one element gets its natural stride."""
    head = t.stride(1) if t.shape[1] > 1 else max(t.shape[2], t.stride(1))
    return (t.stride(0) if t.shape[0] > 1 else max(t.stride(0), head * t.shape[1])), head


def _row_stride(t) -> int:
    """Elements between rows of a [rows, heads, head_dim] tensor whose rows are contiguous."""
    if t.shape[1] > 1 and t.stride(1) != t.shape[2]:
        raise ValueError("q, q_out and out: a row's heads must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _raw_stream(torch, index: int) -> int:
    """The device's current stream as the C ABI takes it (torch.cuda.current_stream builds an object: 2 us a call)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(index) if raw else torch.cuda.current_stream(index).cuda_stream


class _Op:
    """One bound entry point: argument struct, workspace, error flag."""

    name = ""
    workspace = False
    complaint = "a length, position, page id or parent was out of range"

    def _bind(self, args, code: int, tensors) -> None:
        import torch

        tensors = [t for t in tensors if t is not None]
        dev = tensors[0].device
        if any(t.device != dev for t in tensors):
            raise ValueError(f"{self.name}: tensors on different devices")
        if dev.type != "cuda":
            raise ValueError(f"{self.name}: needs CUDA tensors (there is no CPU path)")
        self._torch, self._dev, self._keep = torch, dev, tensors
        self._args, self._code = args, code
        self._err = torch.zeros(1, dtype=torch.int32, device=dev)
        args.err_flag = self._err.data_ptr()
        self._ref = ctypes.byref(args)
        self._fn = getattr(nat.lib, self.name)
        self._ws, extra = None, ()
        if self.workspace:
            with torch.cuda.device(dev):  # (the split goes by the device's SMs)
                need = getattr(nat.lib, self.name + "_workspace_bytes")(self._ref, code)
            if need < 0:  # the call itself names what is wrong
                nat.check(self._fn(self._ref, code, None, 0, None), self.name)
            self._ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
            extra = (self._ws.data_ptr(), self._ws.numel())
        self._extra = extra
        self._index = dev.index
        self._seen = {_raw_stream(torch, dev.index)}
        # the flag's zero, and what used the workspace's memory before, lie on this stream: others wait for it once
        self._made = None
        if not torch.cuda.is_current_stream_capturing():
            self._made = torch.cuda.Event()
            self._made.record(torch.cuda.current_stream(dev))

    def _run(self) -> None:
        torch, index = self._torch, self._index
        st = _raw_stream(torch, index)
        if st not in self._seen and not torch.cuda.is_current_stream_capturing():
            self._seen.add(st)  # its memory is given back only after this stream's work, too
            stream = torch.cuda.current_stream(self._dev)
            if self._made is not None:
                stream.wait_event(self._made)
            for t in (*self._keep, self._ws, self._err):
                if t is not None:
                    t.record_stream(stream)
        if torch.cuda.current_device() == index:
            rc = self._fn(self._ref, self._code, *self._extra, st)
        else:
            with torch.cuda.device(self._dev):
                rc = self._fn(self._ref, self._code, *self._extra, st)
        if rc:
            nat.check(rc, self.name)

    def check(self) -> None:
        """Waits for the device, and raises if a call so far, on whichever stream, met a bad length, position, page id,
        parent or logit; clears the flag."""
        for said in complaints([self]):
            raise ValueError(said)


def forget(ops) -> None:
    """Clears the flags of operators of one device, on its current stream."""
    ops[0]._torch._foreach_zero_([op._err for op in ops])


def complaints(ops) -> list[str]:
    """What the calls of these operators of one device met so far, each thing once.  Waits for the device, on whichever
    streams they ran; their flags are cleared."""
    torch, dev = ops[0]._torch, ops[0]._dev
    torch.cuda.synchronize(dev)
    said = [f"{op.name}: {op.complaint}" for op, bad in zip(ops, torch.cat([op._err for op in ops]).tolist()) if bad]
    if said:
        forget(ops)
        torch.cuda.synchronize(dev)  # (calls that follow on other streams raise them anew)
    return list(dict.fromkeys(said))


class PagedAppend(_Op):
    """K and V of new tokens into the pages; K and ``q`` rotated to their positions (``pim_paged_append``).

    ``k``, ``v`` [tokens, kv_heads, head_dim] and ``q`` [tokens, q_heads, head_dim] may be strided views (of a fused
    qkv row, of a contiguous KV block); ``starts`` [rows + 1] gives each row's tokens (without it, one token per
    row).  The tokens of row b go to slots ``lengths[b]``, ``lengths[b] + 1``, ... at positions ``positions[b]``, ...
    (``lengths`` where not given); ``lengths_out`` / ``positions_out`` receive the counts after the call, tokens that
    were left out for a bad slot, page or position (see ``check``) counted too.
    ``cos`` / ``sin`` [max_pos, head_dim / 2] fp32: without them nothing is rotated.  ``pair_order``: heads come in
    the row order of ``qkv_proj.weight`` (dims j and j + head_dim / 2 adjacent).  ``slot_positions`` / ``weights``
    [rows, kv_heads, slots]: the eviction state of the new slots is set.
    """

    name = "pim_paged_append"

    def __init__(self, k, v, k_pages, v_pages, table, lengths, lengths_out=None, *, q=None, q_out=None, cos=None,
                 sin=None, positions=None, positions_out=None, starts=None, slot_positions=None, weights=None,
                 pair_order: bool = False) -> None:
        kv = _paged_kv(k_pages, v_pages, table)
        dt, rows = _dt(k_pages), kv.rows
        for name, t in (("k", k), ("v", v)):
            _want(t, name, (None, kv.kv_heads, kv.head_dim), dt, contiguous=False)
        tokens = k.shape[0]
        if v.shape[0] != tokens:
            raise ValueError(f"v: {v.shape[0]} tokens, k has {tokens}")
        # (a dimension of one element may carry any stride: it gets its natural one)
        head = [t.stride(1) if kv.kv_heads > 1 else kv.head_dim for t in (k, v)]
        token = [t.stride(0) if tokens > 1 else kv.kv_heads * kv.head_dim for t in (k, v)]
        a = nat.PagedAppendArgs(kv=kv, k=k.data_ptr(), v=v.data_ptr(), k_stride=token[0], v_stride=token[1],
                                k_head_stride=head[0], v_head_stride=head[1], tokens=tokens, pair_order=int(pair_order))
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out go together")
        if q is not None:
            _want(q, "q", (tokens, None, kv.head_dim), dt, contiguous=False)
            _want(q_out, "q_out", tuple(q.shape), dt, contiguous=False)
            a.q, a.q_out, a.q_heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
            a.q_stride, a.q_out_stride = _row_stride(q), _row_stride(q_out)
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin go together")
        if cos is not None:
            _want(cos, "cos", (None, kv.head_dim // 2), "float32")
            _want(sin, "sin", tuple(cos.shape), "float32")
            a.rope_cos, a.rope_sin, a.max_pos = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
        ints = dict(lengths=lengths, positions=positions, lengths_out=lengths_out, positions_out=positions_out)
        for name, t in ints.items():
            if t is not None:
                setattr(a, name, _want(t, name, (rows,), "int32").data_ptr())
        if starts is not None:
            a.starts = _want(starts, "starts", (rows + 1,), "int32").data_ptr()
        if (slot_positions is None) != (weights is None):
            raise ValueError("slot_positions and weights go together")
        if weights is not None:
            slots = kv.max_pages * kv.page_size
            _state(slot_positions, "slot_positions", rows, kv.kv_heads, slots, "int32")
            _state(weights, "weights", rows, kv.kv_heads, slots, "float32")
            if _state_strides(slot_positions) != _state_strides(weights):
                raise ValueError("slot_positions and weights: their strides must be the same")
            a.slot_positions, a.weights = slot_positions.data_ptr(), weights.data_ptr()
            a.state_row_stride, a.state_head_stride = _state_strides(weights)
        read = dict(lengths=lengths, positions=positions, starts=starts, table=table, cos=cos, sin=sin)
        _apart(dict(lengths_out=lengths_out, positions_out=positions_out, slot_positions=slot_positions, weights=weights),
               dict(read, k_pages=k_pages, v_pages=v_pages, k=k, v=v, q=q, q_out=q_out))
        for name, pages in (("k_pages", k_pages), ("v_pages", v_pages)):
            _apart({name: pages}, dict(read, k=k, v=v, q=q, q_out=q_out))
        _apart(dict(q_out=q_out), read)
        if q is not None:
            for name, t in (("q", q), ("k", k), ("v", v)):
                if not (t is q and q_out.data_ptr() == q.data_ptr()) and not _rows_apart(q_out, t):
                    raise ValueError(f"q_out shares memory with {name}")
        self._bind(a, _code(k_pages, "k_pages"),
                   (k, v, k_pages, v_pages, table, lengths, lengths_out, q, q_out, cos, sin, positions, positions_out,
                    starts, slot_positions, weights))
        self.q_out = q_out

    def __call__(self):
        self._run()
        return self.q_out


class PagedAttention(_Op):
    """Attention of one new token per row over its pages (``pim_paged_attention``); returns ``out``.

    ``q`` and ``out`` [rows, q_heads, head_dim]; ``lengths`` [rows] slots attended to.  ``weights`` [rows, kv_heads,
    slots] fp32: every slot's probability, summed over its head's query group, is added.
    """

    name = "pim_paged_attention"
    workspace = True

    def __init__(self, q, k_pages, v_pages, table, lengths, out, *, weights=None, scale: float | None = None) -> None:
        kv = _paged_kv(k_pages, v_pages, table)
        dt = _dt(k_pages)
        _want(q, "q", (kv.rows, None, kv.head_dim), dt, contiguous=False)
        _want(out, "out", tuple(q.shape), dt, contiguous=False)
        _want(lengths, "lengths", (kv.rows,), "int32")
        if scale is not None and not 0 < ctypes.c_float(scale).value < float("inf"):  # (0 would stand for the default)
            raise ValueError(f"scale must be a positive fp32 number, got {scale}")
        a = nat.PagedAttentionArgs(kv=kv, q=q.data_ptr(), out=out.data_ptr(), q_stride=_row_stride(q),
                                   out_stride=_row_stride(out), lengths=lengths.data_ptr(), q_heads=q.shape[1],
                                   scale=0.0 if scale is None else scale)
        if weights is not None:
            _state(weights, "weights", kv.rows, kv.kv_heads, kv.max_pages * kv.page_size, "float32")
            a.weights = weights.data_ptr()
            a.weights_row_stride, a.weights_head_stride = _state_strides(weights)
        _apart(dict(out=out, weights=weights), dict(q=q, k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths))
        self._bind(a, _code(k_pages, "k_pages"), (q, k_pages, v_pages, table, lengths, out, weights))
        self.out = out

    def __call__(self):
        self._run()
        return self.out


class PagedEvict(_Op):
    """Rows of more than ``budget`` slots cut down to it by accumulated weight (``pim_paged_evict``).

    ``positions`` [rows]: the position of each row's next token; tokens at or after ``positions - recent`` and before
    ``sink`` stay.  The ``*_out`` state may be the input state (in place) or tensors of the same strides.
    """

    name = "pim_paged_evict"
    workspace = True

    def __init__(self, k_pages, v_pages, table, lengths, weights, slot_positions, positions, weights_out,
                 slot_positions_out, lengths_out, *, budget: int, recent: int = 0, sink: int = 0) -> None:
        kv = _paged_kv(k_pages, v_pages, table)
        _code(k_pages, "k_pages")
        slots = kv.max_pages * kv.page_size
        for name, t in (("lengths", lengths), ("positions", positions), ("lengths_out", lengths_out)):
            _want(t, name, (kv.rows,), "int32")
        state = dict(weights=(weights, "float32"), slot_positions=(slot_positions, "int32"),
                     weights_out=(weights_out, "float32"), slot_positions_out=(slot_positions_out, "int32"))
        for name, (t, dt) in state.items():
            _state(t, name, kv.rows, kv.kv_heads, slots, dt)
            if _state_strides(t) != _state_strides(weights):
                raise ValueError(f"{name}: its strides must be those of weights")
        for name, out, src in (("weights_out", weights_out, weights),
                               ("slot_positions_out", slot_positions_out, slot_positions)):
            if _overlap(out, src) and out.data_ptr() != src.data_ptr():
                raise ValueError(f"{name} shares part of its input's memory: it must be its input or apart")
        _apart(dict(weights_out=weights_out, slot_positions_out=slot_positions_out, lengths_out=lengths_out),
               dict(k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths, positions=positions))
        read = dict(table=table, lengths=lengths, positions=positions, weights=weights, slot_positions=slot_positions)
        for name, pages in (("k_pages", k_pages), ("v_pages", v_pages)):
            _apart({name: pages}, read)
        _apart(dict(weights_out=weights_out, lengths_out=lengths_out), dict(slot_positions=slot_positions))
        _apart(dict(slot_positions_out=slot_positions_out, lengths_out=lengths_out), dict(weights=weights))
        row, head = _state_strides(weights)
        a = nat.PagedEvictArgs(kv=kv, lengths=lengths.data_ptr(), positions=positions.data_ptr(),
                               weights=weights.data_ptr(), slot_positions=slot_positions.data_ptr(),
                               weights_out=weights_out.data_ptr(), slot_positions_out=slot_positions_out.data_ptr(),
                               lengths_out=lengths_out.data_ptr(), state_row_stride=row, state_head_stride=head,
                               budget=_int32(budget, "budget"), recent=_int32(recent, "recent"),
                               sink=_int32(sink, "sink"))
        self._bind(a, _code(k_pages, "k_pages"),
                   (k_pages, v_pages, table, lengths, weights, slot_positions, positions, weights_out,
                    slot_positions_out, lengths_out))
        self.lengths_out = lengths_out

    def __call__(self):
        self._run()
        return self.lengths_out


class BeamSelect(_Op):
    """One step of beam search (``pim_beam_select``); returns (scores_out, parents, tokens).

    ``logits`` [batch, beams, vocab]; ``scores`` [batch, beams] fp32; the outputs [batch, beams_out] (as many beams as
    ``scores_out`` has).  ``done`` / ``done_out`` int32: beams that have ended.  Logits and scores of -inf are masked;
    NaN and +inf are left out likewise, and reported by ``check``.
    """

    name = "pim_beam_select"
    workspace = True
    complaint = "a logit or score was NaN or +infinity"

    def __init__(self, logits, scores, scores_out, parents, tokens, *, done=None, done_out=None, eos: int = -1,
                 pad: int = 0) -> None:
        code = _code(logits, "logits")
        _want(logits, "logits", (None, None, None), _dt(logits), contiguous=False)
        b, w, vocab = logits.shape
        stride = logits.stride(1) if w > 1 else logits.stride(0) if b > 1 else vocab
        if b > 1 and w > 1 and logits.stride(0) != w * stride:
            raise ValueError("logits: the beams of all batch entries must be evenly spaced")
        _want(scores, "scores", (b, w), "float32")
        k = scores_out.shape[1] if scores_out.dim() == 2 else -1
        _want(scores_out, "scores_out", (b, None), "float32")
        for name, t in (("parents", parents), ("tokens", tokens), ("done_out", done_out)):
            if t is not None:
                _want(t, name, (b, k), "int32")
        if done is not None:
            _want(done, "done", (b, w), "int32")
        a = nat.BeamSelectArgs(logits=logits.data_ptr(), logits_stride=stride, scores=scores.data_ptr(),
                               scores_out=scores_out.data_ptr(), parents=parents.data_ptr(), tokens=tokens.data_ptr(),
                               batch=b, beams=w, beams_out=k, vocab=vocab, eos=_int32(eos, "eos"), pad=_int32(pad, "pad"))
        if done is not None:
            a.done = done.data_ptr()
        if done_out is not None:
            a.done_out = done_out.data_ptr()
        _apart(dict(scores_out=scores_out, parents=parents, tokens=tokens, done_out=done_out),
               dict(logits=logits, scores=scores, done=done))
        self._bind(a, code, (logits, scores, scores_out, parents, tokens, done, done_out))
        self.outputs = (scores_out, parents, tokens)

    def __call__(self):
        self._run()
        return self.outputs


class BeamReorder(_Op):
    """The cache states of the beams that ``BeamSelect`` chose (``pim_beam_reorder``); returns ``table_out``.

    ``pages`` [..., num_pages, kv_heads, page_size, head_dim] holds every block (layer, k | v) that must follow, evenly
    spaced; ``table`` / ``table_out`` [batch * beams, max_pages]; ``lengths`` [batch]; ``parents`` [batch, beams].
    """

    name = "pim_beam_reorder"

    def __init__(self, pages, table, lengths, parents, table_out) -> None:
        if pages.dim() < 4:
            raise ValueError(f"pages: expected [..., num_pages, kv_heads, page_size, head_dim], got {tuple(pages.shape)}")
        _code(pages, "pages")
        if not pages.is_contiguous():
            raise ValueError("pages: must be contiguous")
        num, heads, ps, hd = pages.shape[-4:]
        _want(parents, "parents", (None, None), "int32")
        b, w = parents.shape
        _want(table, "table", (b * w, None), "int32")
        _want(table_out, "table_out", tuple(table.shape), "int32")
        _want(lengths, "lengths", (b,), "int32")
        blocks = 1
        for n in pages.shape[:-4]:
            blocks *= n
        a = nat.BeamReorderArgs(pages=pages.data_ptr(), block_stride=num * heads * ps * hd, page_stride=heads * ps * hd,
                                table=table.data_ptr(), table_out=table_out.data_ptr(), table_stride=table.shape[1],
                                lengths=lengths.data_ptr(), parents=parents.data_ptr(), batch=b, beams=w,
                                num_blocks=blocks, max_pages=table.shape[1], num_pages=num, page_size=ps,
                                kv_heads=heads, head_dim=hd)
        _apart(dict(table_out=table_out, pages=pages), dict(table=table, lengths=lengths, parents=parents))
        self._bind(a, _code(pages, "pages"), (pages, table, lengths, parents, table_out))
        self.table_out = table_out

    def __call__(self):
        self._run()
        return self.table_out
