"""Operators on device tensors over the C ABI (section 4 of ``include/linmt_decoder.h``): the parts of a decoding step for programs that run
their own model.

    beam_select    the best continuations of each sentence's beams, from logits
    beam_reorder   states follow their beams
    plan_pages     pages and slots for sentences that grow
    write_pages4   keys and values into pages, in 4 bits
    read_pages4    the values that they stand for
    attend_pages4  attention of a sentence's beams over its pages

Tensors are torch CUDA tensors, all of one call on one device.  Work is issued on that device's current torch stream and nothing waits; results that
are not given as ``out`` are allocated by torch on that stream, so calls follow each other, may run at once on several
streams and may be captured into a CUDA graph like torch's own.  ``ValueError``: an argument is not allowed; ``LinmtError``: the library refused.
There is no backward pass: the engine decodes and scores, it does not train.
"""
from __future__ import annotations

import struct

import torch

from . import _lib
from .decoder import LinmtError

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I32, _I64, _U8, _F32 = torch.int32, torch.int64, torch.uint8, torch.float32

# The argument structs of the header, field by field; "x" is the padding that C puts in.
_SELECT = struct.Struct("@IiPPqqPPPqPPPPiiiii4x")
_STATE = struct.Struct("@PPqqqqqqqq")
_REORDER = struct.Struct("@IiPPiiii")
_PLAN = struct.Struct("@IiPPPPqPPPPPiiiiq")
_ROWS = struct.Struct("@IiPPqqiiiiPPPqqqqii")
_ATTEND = struct.Struct("@IiPPqqiiiiPqqqPqqqPPqPPPPPPqiiiiiff4x")
_MAX_STATES = 16

_fns = None


def _call(name, args):
    global _fns
    if _fns is None:
        lib = _lib.load()
        _fns = {n: getattr(lib, "linmt_" + n) for n in ("beam_select", "beam_reorder", "plan_pages", "write_pages4", "read_pages4", "attend_pages4", "attend_pages4_workspace")}
        _fns["error"] = lib.linmt_op_error
    rc = _fns[name](args)
    if rc > 0 and name != "attend_pages4_workspace" or rc < 0:
        text = _fns["error"]().decode()
        if rc == 1 or rc < 0:
            raise ValueError(text)
        raise LinmtError(f"{text} ({rc})")
    return rc


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _device(x, name):
    _need(isinstance(x, torch.Tensor) and x.is_cuda, f"{name} has to be a CUDA tensor")
    return x.get_device()


def _check(x, name, device, dtype, shape):
    """A contiguous tensor of the given type and shape on the call's device."""
    _need(isinstance(x, torch.Tensor) and x.is_cuda and x.get_device() == device, f"{name} has to be a tensor on CUDA device {device}")
    _need(x.dtype == dtype, f"{name} has to be {dtype}, not {x.dtype}")
    _need(tuple(x.shape) == tuple(shape), f"{name} has to have the shape {tuple(shape)}, not {tuple(x.shape)}")
    _need(x.is_contiguous(), f"{name} has to be contiguous")
    return x.data_ptr()


def _flags(x, name, device, shape):
    _need(isinstance(x, torch.Tensor) and x.dtype in (torch.bool, _U8), f"{name} has to be a bool or uint8 tensor")
    return _check(x, name, device, x.dtype, shape)


def beam_select(logits, scores, *, done=None, allowed=None, eos=1, out=None):
    """The k best of the k * vocab continuations of each sentence's beams, best first, equal ones by the lowest beam * vocab + word.

    ``logits`` [n, k, vocab] (float32, bfloat16 or float16; words contiguous, any other strides), ``scores`` [n, k] float32: the beams' sums so far, -inf for an
    empty beam.  A live beam offers score + log_softmax(logits) of its allowed words; a finished one (``done`` [n, k], bool or uint8) offers
    ``eos`` with its score as it is.  ``allowed`` [1 or n, ceil(vocab / 32)] int32: bit v % 32 of word v / 32 is set where word v may
    be chosen (the others do not enter the softmax and may hold anything).  A beam with a NaN or +inf at an allowed place offers nothing.

    Returns ``tokens``, ``parents`` [n, k] int32, ``scores`` [n, k] float32 and ``done`` [n, k] bool (the parent was finished, or the token is
    ``eos``).  A slot for which nothing is left has token eos, itself as the parent, -inf and True.  ``out``: a tuple of four such tensors to
    write into; they may be ``scores`` and ``done`` themselves."""
    dev = _device(logits, "logits")
    _need(logits.dim() == 3 and logits.dtype in _DTYPES, "logits have to be [n, k, vocab] in float32, bfloat16 or float16")
    n, k, v = logits.shape
    sn, sk, sv = logits.stride()
    _need(v >= 1 and (sv == 1 or v == 1), "the words of a row of logits have to be contiguous")
    sp = _check(scores, "scores", dev, _F32, (n, k))
    dp = 0 if done is None else _flags(done, "done", dev, (n, k))
    ap = stride = 0
    if allowed is not None:
        words = (v + 31) // 32
        _need(isinstance(allowed, torch.Tensor) and allowed.dim() == 2 and allowed.shape[0] in (1, n), "allowed has to be [1 or n, ceil(vocab / 32)]")
        ap = _check(allowed, "allowed", dev, _I32, (allowed.shape[0], words))
        stride = words if allowed.shape[0] != 1 else 0
    if out is None:
        device = logits.device
        out = (torch.empty((n, k), dtype=_I32, device=device), torch.empty((n, k), dtype=_I32, device=device),
               torch.empty((n, k), dtype=_F32, device=device), torch.empty((n, k), dtype=torch.bool, device=device))
        o = [x.data_ptr() for x in out]
    else:
        _need(len(out) == 4, "out has to be (tokens, parents, scores, done)")
        o = [_check(out[0], "out[0]", dev, _I32, (n, k)), _check(out[1], "out[1]", dev, _I32, (n, k)),
             _check(out[2], "out[2]", dev, _F32, (n, k)), _flags(out[3], "out[3]", dev, (n, k))]
    if n:
        _call("beam_select", _SELECT.pack(_SELECT.size, dev, _stream(dev), logits.data_ptr(), sn, sk, sp, dp, ap, stride, *o, n, k, v, eos, _DTYPES[logits.dtype]))
    return tuple(out)


def _layers(x, n, k, name):
    """(layers, stride of a layer, of a sentence, of a beam, row bytes) of a state, in bytes."""
    _need(x.dim() in (2, 3, 4), f"{name} has to be [n, k], [n, k, width] or [layers, n, k, width]")
    size, st, shape = x.element_size(), x.stride(), tuple(x.shape)
    if x.dim() == 2:
        shape, st = shape + (1,), st + (1,)
    if x.dim() < 4:
        shape, st = (1,) + shape, (0,) + st
    _need(shape[1:3] == (n, k), f"{name} has to have the sentences and beams of parents, {(n, k)}, not {shape[1:3]}")
    _need(st[3] == 1 or shape[3] <= 1, f"the rows of {name} have to be contiguous")
    return shape[0], st[0] * size, st[1] * size, st[2] * size, shape[3] * size


def _span(x):
    return x.data_ptr(), x.data_ptr() + (sum((s - 1) * t for s, t in zip(x.shape, x.stride())) + 1) * x.element_size()


def beam_reorder(states, parents, *, out=None):
    """Rows of states follow their beams: ``out[...][.., i, j, :] = states[...][.., i, parents[i, j], :]``, all states in one launch (for each 16).

    ``states``: tensors [n, k], [n, k, width] or [layers, n, k, width] of any type, rows contiguous.  ``parents`` [n, k] int32; one outside 0 .. k-1 is taken as the
    row's own.  ``out``: tensors like them, each either the state itself or one that it does not overlap; without it the states are reordered in place.
    Returns the list of the tensors written."""
    dev = _device(parents, "parents")
    _need(parents.dim() == 2, "parents have to be [n, k]")
    n, k = parents.shape
    pp = _check(parents, "parents", dev, _I32, (n, k))
    states = list(states)
    to = states if out is None else list(out)
    _need(len(to) == len(states), "out has to have a tensor for every state")
    packed, written = [], []
    for i, (x, y) in enumerate(zip(states, to)):
        _need(_device(x, f"states[{i}]") == dev, f"states[{i}] has to be on CUDA device {dev}")
        layers, sl, sn, sk, row = _layers(x, n, k, f"states[{i}]")
        if y is x:
            dl, dn, dk = sl, sn, sk
        else:
            _need(_device(y, f"out[{i}]") == dev and y.dtype == x.dtype and y.shape == x.shape, f"out[{i}] has to be like states[{i}]")
            _, dl, dn, dk, _ = _layers(y, n, k, f"out[{i}]")
        if x.numel() == 0:
            continue
        a, b = _span(x), _span(y)
        _need(b[0] >= a[1] or a[0] >= b[1] or (a == b and (sl, sn, sk) == (dl, dn, dk)), f"out[{i}] overlaps states[{i}]")
        _need(b[0] not in written, f"out[{i}] is written twice")
        _need(all(s != 0 or z <= 1 for s, z in zip((dl, dn, dk), ((layers if y.dim() == 4 else 1), n, k))), f"out[{i}] has rows that share memory")
        written.append(b[0])
        packed.append(_STATE.pack(x.data_ptr(), y.data_ptr(), sl, sn, sk, dl, dn, dk, row, layers))
    for i in range(0, len(packed), _MAX_STATES):
        part = packed[i:i + _MAX_STATES]
        size = _REORDER.size + _MAX_STATES * _STATE.size
        _call("beam_reorder", b"".join([_REORDER.pack(size, dev, _stream(dev), pp, n, k, len(part), 0)] + part).ljust(size, b"\0"))
    return to


def plan_pages(old, new, table, free, used, *, page, total):
    """Pages and slots for sentences that grow from ``old`` to ``new`` positions ([n] int32; ``old`` None: from nothing).

    Every page column p of sentence i with ceil(old / page) <= p < ceil(new / page) of ``table`` [n, width] int32 gets the next entry of ``free`` [n_free] int32, of
    which ``used`` [1] int32 are taken already; ``table`` is written in place.  Returns ``slots`` [total] int64 (table[i, pos // page] * page + pos % page of each
    new position, sentence by sentence, -1 behind the last), ``starts`` [n + 1] int32 (each sentence's first in ``slots``) and the new ``used`` [1].
    Where the free list has run out a column and its slots are -1 and ``used`` comes back larger than n_free.  Lengths are taken as 0 .. width * page, a
    shorter ``new`` as ``old``."""
    dev = _device(new, "new")
    _need(new.dim() == 1, "new has to be [n]")
    n = new.shape[0]
    np_ = _check(new, "new", dev, _I32, (n,))
    op = 0 if old is None else _check(old, "old", dev, _I32, (n,))
    _need(isinstance(table, torch.Tensor) and table.is_cuda and table.get_device() == dev and table.dtype == _I32 and table.dim() == 2 and table.shape[0] == n, "table has to be [n, width] int32 on the same device")
    width = table.shape[1]
    _need(table.stride(1) == 1 or width <= 1, "the rows of table have to be contiguous")
    _need(table.stride(0) >= width or n <= 1, "the rows of table share memory")
    _need(isinstance(free, torch.Tensor) and free.dim() == 1, "free has to be [n_free]")
    fp = _check(free, "free", dev, _I32, (free.shape[0],))
    up = _check(used, "used", dev, _I32, (1,))
    _need(total >= 0, "total is negative")
    device = new.device
    slots = torch.empty(total, dtype=_I64, device=device)
    starts = torch.empty(n + 1, dtype=_I32, device=device)
    now = torch.empty(1, dtype=_I32, device=device)
    _call("plan_pages", _PLAN.pack(_PLAN.size, dev, _stream(dev), op, np_, table.data_ptr(), table.stride(0), fp, up, now.data_ptr(), slots.data_ptr(), starts.data_ptr(), n, width, page, free.shape[0], total))
    return slots, starts, now


def new_pages4(n_pages, heads, dim, page, device="cuda"):
    """A pool of ``n_pages`` pages of ``page`` positions (a multiple of 16) for ``heads`` heads of ``dim`` (64 or 128) components, all zeros: uint8
    [n_pages, heads, page / 16, 18 * dim]."""
    _need(page >= 16 and page % 16 == 0 and dim in (64, 128), "a page has a multiple of 16 positions, a head 64 or 128 components")
    return torch.zeros((n_pages, heads, page // 16, 18 * dim), dtype=_U8, device=device)


def _pool(pages, dev):
    """The fields of linmt_pages4, and dim."""
    _need(isinstance(pages, torch.Tensor) and pages.is_cuda and pages.get_device() == dev, f"pages have to be a tensor on CUDA device {dev}")
    _need(pages.dtype == _U8 and pages.dim() == 4 and pages.shape[3] % 18 == 0, "pages have to be uint8 [n_pages, heads, page / 16, 18 * dim]")
    n_pages, heads, tiles, b = pages.shape
    s = pages.stride()
    _need(s[3] == 1 and (s[2] == b or tiles == 1), "the tiles of a page's head have to be contiguous")
    return (pages.data_ptr(), s[0], s[1], n_pages, heads, tiles * 16, b // 18), b // 18


def _rows(name, pages, slots, k, v):
    dev = _device(slots, "slots")
    pool, dim = _pool(pages, dev)
    _need(slots.dim() == 1, "slots have to be [t]")
    t = slots.shape[0]
    sp = _check(slots, "slots", dev, _I64, (t,))
    for x, what in ((k, "k"), (v, "v")):
        _need(_device(x, what) == dev and x.dtype in _DTYPES and x.dtype == k.dtype, f"{what} has to be float32, bfloat16 or float16 on the same device, as k")
        _need(tuple(x.shape) == (t, pages.shape[1], dim), f"{what} has to have the shape {(t, pages.shape[1], dim)}, not {tuple(x.shape)}")
        _need(x.stride(2) == 1, f"the components of {what} have to be contiguous")
    if t:
        _call(name, _ROWS.pack(_ROWS.size, dev, _stream(dev), *pool, sp, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), t, _DTYPES[k.dtype]))


def write_pages4(pages, slots, k, v):
    """Keys and values ``k``, ``v`` [t, heads, dim] (float32, bfloat16 or float16, components contiguous, rows on 16-byte boundaries) into ``slots`` [t] int64 of a
    pool, in 4 bits with a bf16 scale for 32 components (the form is in the header).  A slot outside the pool, -1 say, is not written.  No slot may be
    named twice."""
    _rows("write_pages4", pages, slots, k, v)


def read_pages4(pages, slots, *, dtype=torch.float32):
    """The keys and values [t, heads, dim] that ``slots`` of a pool stand for (exact in float32); zeros for a slot outside the pool."""
    _device(slots, "slots")
    _need(isinstance(pages, torch.Tensor) and pages.dim() == 4 and slots.dim() == 1 and dtype in _DTYPES, "pages have to be [n_pages, heads, page / 16, 18 * dim], slots [t], dtype float32, bfloat16 or float16")
    shape = (slots.shape[0], pages.shape[1], pages.shape[3] // 18)
    k, v = torch.empty(shape, dtype=dtype, device=slots.device), torch.empty(shape, dtype=dtype, device=slots.device)
    _rows("read_pages4", pages, slots, k, v)
    return k, v


def attend_pages4(q, pages, table, lens, *, scale=None, cap=0.0, slope=None, centre=None, first=None, last=None, out=None, want_lse=False):
    """Attention of the g query rows (beams) of each sentence over its positions in a pool.

    ``q`` [n, g, heads, dim] (float32, bfloat16 or float16, components contiguous); query head h reads head h // (heads / pool heads).  ``table`` [n, width] int32
    names each sentence's pages, ``lens`` [n] int32 its positions.  ``scale``: dim ** -0.5 if None.  ``cap`` > 0: scores are cap * tanh(s / cap).  ``slope``
    [heads] with ``centre`` [n, g], float32: scores lose slope * |position - centre|.  ``first``, ``last`` [n, g] int32: a row sees positions
    first <= t < last only.  Positions in a column that names no page of the pool are not seen.  A row that sees nothing gets zeros and lse -inf.

    Returns ``out`` like q, and with ``want_lse`` also the log of the row's sum of exponentials, [n, g, heads] float32."""
    dev = _device(q, "q")
    pool, dim = _pool(pages, dev)
    _need(q.dim() == 4 and q.dtype in _DTYPES and q.shape[3] == dim, f"q has to be [n, g, heads, {dim}] in float32, bfloat16 or float16")
    n, g, heads, _ = q.shape
    qn, qg, qh, qd = q.stride()
    _need(qd == 1, "the components of q have to be contiguous")
    _need(isinstance(table, torch.Tensor) and table.is_cuda and table.get_device() == dev and table.dtype == _I32 and table.dim() == 2 and table.shape[0] == n, "table has to be [n, width] int32 on the same device")
    width = table.shape[1]
    _need(table.stride(1) == 1 or width <= 1, "the rows of table have to be contiguous")
    lp = _check(lens, "lens", dev, _I32, (n,))
    _need((slope is None) == (centre is None), "slope goes with centre")
    _need((first is None) == (last is None), "first goes with last")
    slp = cp = fp = lap = 0
    if slope is not None:
        slp, cp = _check(slope, "slope", dev, _F32, (heads,)), _check(centre, "centre", dev, _F32, (n, g))
    if first is not None:
        fp, lap = _check(first, "first", dev, _I32, (n, g)), _check(last, "last", dev, _I32, (n, g))
    if out is None:
        out = torch.empty((n, g, heads, dim), dtype=q.dtype, device=q.device)
    else:
        _need(_device(out, "out") == dev and out.dtype == q.dtype and out.shape == q.shape and out.stride(3) == 1, "out has to be like q")
        _need(all(s != 0 or z <= 1 for s, z in zip(out.stride(), out.shape)), "out has rows that share memory")
    on, og, oh, _ = out.stride()
    lse = torch.empty((n, g, heads), dtype=_F32, device=q.device) if want_lse else None
    if n and g and heads:
        head = (_ATTEND.size, dev, _stream(dev), *pool, q.data_ptr(), qn, qg, qh, out.data_ptr(), on, og, oh, lse.data_ptr() if want_lse else 0,
                table.data_ptr(), table.stride(0), lp, slp, cp, fp, lap)
        tail = (n, g, heads, width, _DTYPES[q.dtype], dim ** -0.5 if scale is None else scale, cap)
        args = _ATTEND.pack(*head, 0, 0, *tail)
        need = _call("attend_pages4_workspace", args)
        if need:
            ws = torch.empty(need, dtype=_U8, device=q.device)
            args = _ATTEND.pack(*head, ws.data_ptr(), need, *tail)
        _call("attend_pages4", args)
    return (out, lse) if want_lse else out
