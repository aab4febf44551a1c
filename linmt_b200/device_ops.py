"""Operators on device tensors over the C ABI (section 4 of ``include/linmt_decoder.h``): the parts of a decoding step for programs that run
their own model.

    beam_select    the best continuations of each sentence's beams, from logits
    beam_reorder   states follow their beams
    plan_pages     pages and slots for sentences that grow
    write_pages4   keys and values into pages, in 4 bits
    read_pages4    the values that they stand for
    attend_pages4  attention of a sentence's beams over its pages
    write_pages8, read_pages8, attend_pages8   the same in 8 bits
    fork_pages     pages follow their hypotheses, as beam_select has chosen them
    free_pages     pages of hypotheses that are done go back
    compact_pages  the pages in use move to the front of their pool
    copy_pages     pages into other pages, in all pools at once
    score_tokens   log probabilities of given tokens, entropy and the best alternatives

Tensors are torch CUDA tensors, all of one call on one device.  Work is issued on that device's current torch stream and nothing waits; results that
are not given as ``out`` are allocated by torch on that stream, so calls follow each other, may run at once on several
streams and may be captured into a CUDA graph like torch's own.  ``ValueError``: an argument is not allowed; ``LinmtError``: the library refused.
There is no backward pass (the engine decodes and scores, it does not train): tensors that require a gradient are refused outside ``torch.no_grad()``, and
tensors with a tangent (``torch.autograd.forward_ad``) everywhere.
"""
from __future__ import annotations

import importlib.util

import torch

from . import _lib, build

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _load():
    """The C++ front (csrc/device_ops_torch.cpp) on top of the library; raises if either has not been built."""
    _lib.load()
    if not build.torch_front_is_built():
        raise RuntimeError(f"{build.TORCH_LIB} is missing: build it with `python -m linmt_b200.build` (there is no CPU fallback)")
    spec = importlib.util.spec_from_file_location("linmt_b200._device_ops", build.TORCH_LIB)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_front = _load()


def beam_select(logits, scores, *, done=None, allowed=None, eos=1, out=None):
    """The k best of the k * vocab continuations of each sentence's beams, best first, equal ones by the lowest beam * vocab + word.

    ``logits`` [n, k, vocab] (float32, bfloat16 or float16; words contiguous, any other strides), ``scores`` [n, k] float32: the beams' sums so far, -inf for an
    empty beam.  A live beam offers score + log_softmax(logits) of its allowed words; a finished one (``done`` [n, k], bool or uint8) offers
    ``eos`` with its score as it is.  ``allowed`` [1 or n, ceil(vocab / 32)] int32: bit v % 32 of word v / 32 is set where word v may
    be chosen (the others do not enter the softmax and may hold anything).  A beam with a NaN or +inf at an allowed place offers nothing.

    Ranks are those of 64-bit sums (to 2^-36).  The scores returned carry a normaliser that is summed in 32 bits unless a rank depended on it: good to 6e-6, and 6e-8 for
    every 512 32-bit (1024 16-bit) words that a warp reads.  A stretch whose largest logit is 64 or more in size is read twice, its 6e-8 are 5e-7.

    Returns ``tokens``, ``parents`` [n, k] int32, ``scores`` [n, k] float32 and ``done`` [n, k] bool (the parent was finished, or the token is
    ``eos``).  A slot for which nothing is left has token eos, itself as the parent, -inf and True.  ``out``: a tuple of four such tensors to
    write into; they may be ``scores`` and ``done`` themselves, and overlap nothing else that the call reads."""
    return _front.beam_select(logits, scores, done, allowed, eos, None if out is None else tuple(out))


def beam_reorder(states, parents, *, out=None):
    """Rows of states follow their beams: ``out[...][.., i, j, :] = states[...][.., i, parents[i, j], :]``, all states in one launch (for each 16).

    ``states``: tensors [n, k], [n, k, width] or [layers, n, k, width] of any type, rows contiguous.  ``parents`` [n, k] int32; one outside 0 .. k-1 is taken as the
    row's own.  ``out``: tensors like them, each either the state itself or one that overlaps no state; without it the states are reordered in place.
    Returns the list of the tensors written."""
    states = list(states)
    return _front.beam_reorder(states, parents, states if out is None else list(out))


def plan_pages(old, new, table, free, used, *, page, total):
    """Pages and slots for sentences that grow from ``old`` to ``new`` positions ([n] int32; ``old`` None: from nothing).

    Every page column p of sentence i with ceil(old / page) <= p < ceil(new / page) of ``table`` [n, width] int32 gets the next entry of ``free`` [n_free] int32, of
    which ``used`` [1] int32 are taken already; ``table`` is written in place, and overlaps none of the others.  Returns ``slots`` [total] int64
    (table[i, pos // page] * page + pos % page of each new position, sentence by sentence, -1 behind the last), ``starts`` [n + 1] int32 (each sentence's first in ``slots``) and the new ``used`` [1].
    Where the free list has run out a column and its slots are -1 and ``used`` comes back larger than n_free.  Lengths are taken as 0 .. width * page, a
    shorter ``new`` as ``old``."""
    return _front.plan_pages(old, new, table, free, used, page, total)


def new_pages4(n_pages, heads, dim, page, device="cuda"):
    """A pool of ``n_pages`` pages of ``page`` positions (a multiple of 16) for ``heads`` heads of ``dim`` (64 or 128) components, all zeros: uint8
    [n_pages, heads, page / 16, 18 * dim]."""
    if page < 16 or page % 16 or dim not in (64, 128):
        raise ValueError("a page has a multiple of 16 positions, a head 64 or 128 components")
    return torch.zeros((n_pages, heads, page // 16, 18 * dim), dtype=torch.uint8, device=device)


def write_pages4(pages, slots, k, v):
    """Keys and values ``k``, ``v`` [t, heads, dim] (float32, bfloat16 or float16, components contiguous, rows on 16-byte boundaries) into ``slots`` [t] int64 of a
    pool, in 4 bits with a bf16 scale for 32 components (the form is in the header).  A slot outside the pool, -1 say, is not written.  No slot may be
    named twice, and ``pages`` overlaps none of the others."""
    _front.write_pages4(pages, slots, k, v)


def read_pages4(pages, slots, *, dtype=torch.float32):
    """The keys and values [t, heads, dim] that ``slots`` of a pool stand for (exact in float32); zeros for a slot outside the pool."""
    return _front.read_pages4(pages, slots, _DTYPES.get(dtype, -1))


def attend_pages4(q, pages, table, lens, *, scale=None, cap=0.0, slope=None, centre=None, first=None, last=None, out=None, want_lse=False):
    """Attention of the g query rows (beams) of each sentence over its positions in a pool.

    ``q`` [n, g, heads, dim] (float32, bfloat16 or float16, components contiguous); query head h reads head h // (heads / pool heads).  ``table`` [n, width] int32
    names each sentence's pages, ``lens`` [n] int32 its positions.  ``scale``: dim ** -0.5 if None.  ``cap`` > 0: scores are cap * tanh(s / cap).  ``slope``
    [heads] with ``centre`` [n, g], float32: scores lose slope * |position - centre|.  ``first``, ``last`` [n, g] int32: a row sees positions
    first <= t < last only, and what others hold changes nothing of its result.  Positions in a column that names no page of the pool are not seen.  A row that
    sees nothing gets zeros and lse -inf, one whose query has a NaN or an infinity gets NaN in both.

    Returns ``out`` like q (it may be q itself, and overlaps nothing else that the call reads), and with ``want_lse`` also the log of the row's sum of exponentials, [n, g, heads] float32."""
    return _front.attend_pages4(q, pages, table, lens, scale, cap, slope, centre, first, last, out, want_lse)


def new_pages8(n_pages, heads, dim, page, device="cuda"):
    """A pool of ``n_pages`` pages of ``page`` positions (a multiple of 16) for ``heads`` heads of ``dim`` (64 or 128) components, all zeros: uint8
    [n_pages, heads, page / 16, 32 * dim + 16]."""
    if page < 16 or page % 16 or dim not in (64, 128):
        raise ValueError("a page has a multiple of 16 positions, a head 64 or 128 components")
    return torch.zeros((n_pages, heads, page // 16, 32 * dim + 16), dtype=torch.uint8, device=device)


def write_pages8(pages, slots, k, v):
    """Keys and values ``k``, ``v`` [t, heads, dim] (float32, bfloat16 or float16, components contiguous, rows on 16-byte boundaries) into ``slots`` [t] int64 of a
    pool, in 8 bits with a scale for each block of 16 positions and head, of the keys and the values each (the form is in the header).

    Neighbours in ``slots`` that are neighbours in a block, ascending, are written together, as plan_pages gives them.  From a block's first position on they make it new;
    further on they are appended: positions before them stay (their codes are rounded again where the block's scale has to grow), positions behind them become zeros.  A slot
    outside the pool, -1 say, is not written.  No block may be written at two places of ``slots``, and ``pages`` overlaps none of the others."""
    _front.write_pages8(pages, slots, k, v)


def read_pages8(pages, slots, *, dtype=torch.float32):
    """The keys and values [t, heads, dim] that ``slots`` of a pool stand for (exact in float32); zeros for a slot outside the pool."""
    return _front.read_pages8(pages, slots, _DTYPES.get(dtype, -1))


def attend_pages8(q, pages, table, lens, *, scale=None, cap=0.0, slope=None, centre=None, first=None, last=None, sinks=0, out=None, want_lse=False):
    """Attention of the g query rows (beams) of each sentence over its positions in a pool of 8-bit pages.

    Everything is as in attend_pages4, with one argument more: positions below ``sinks`` stay visible whatever ``first`` and ``last`` say (a window that slides
    over a long text and the first few tokens before it).  Queries are taken to 2^-22 of a row's largest component, weights times scales to 2^-30 of the row's
    largest (2^-27 with 16-bit queries); both products are exact sums of integers."""
    return _front.attend_pages8(q, pages, table, lens, scale, cap, slope, centre, first, last, out, want_lse, sinks)


def fork_pages(table, lens, parents, shares, free, used, *, page, done=None, out=None):
    """Pages follow their hypotheses: hypothesis (i, j) goes on from (i, parents[i, j]), as beam_select has it.

    ``table`` [n, k, width] and ``lens`` [n, k] int32: the pages and positions of n * k <= 16384 hypotheses.  ``parents`` [n, k] int32; one outside 0 .. k-1, or ``done``
    [n, k] (bool or uint8), leaves a hypothesis without pages.  ``shares`` [n_pages] int32: how many hypotheses beyond the first name a page; zeros to begin with, and for what
    plan_pages hands out.  ``free`` [n_free] and ``used`` [1] are plan_pages's.

    Children share their parent's pages.  A last page that is not full stays with the first child; each further one gets a page of its own for it, taken from ``free``.
    Pages that nobody names any more go back to ``free`` first.  Returns ``table``, ``lens``, ``shares``, ``free``, ``used`` as they are now, and ``src``, ``dst`` [n * k]: the
    pages to copy (copy_pages), -1 behind the last.  Where the free pages run out, a column and its dst are -1 and ``used`` comes back larger than n_free.
    Columns behind a hypothesis' pages come out as -1.  ``out``: a tuple of seven such tensors to write into; shares, free and used may be the
    arguments themselves, otherwise they overlap nothing that the call reads."""
    return _front.fork_pages(table, lens, parents, done, shares, free, used, page, None if out is None else tuple(out))


def free_pages(table, lens, done, shares, free, used, *, page, out=None):
    """The pages of rows that are ``done`` go back to ``free`` where no other row names them.  ``table`` [n, width] with ``lens`` and ``done`` [n], or [n, k, width] with [n, k]; up to
    16384 rows.
    Returns ``table``, ``lens``, ``shares``, ``free`` and ``used`` as fork_pages does; ``out``: a tuple of five."""
    return _front.free_pages(table, lens, None, done, shares, free, used, page, None if out is None else tuple(out))


def compact_pages(table, lens, shares, *, page, out=None):
    """The pages that rows name move to the front of their pool, those that lie there already stay.  ``table`` [n, width] with ``lens`` [n], or [n, k, width] with [n, k].

    Returns ``table`` and ``shares`` by the new numbers, ``free`` [n_pages] (0, 1, ..) and ``used`` [1] (the pages in use: all behind them are free), and ``src``, ``dst`` [n_pages // 2]: the pages
    to copy (copy_pages), -1 behind the last.  ``out``: a tuple of six such tensors to write into; table and shares may be the arguments themselves."""
    return _front.compact_pages(table, lens, shares, page, None if out is None else tuple(out))


def copy_pages(pools, src, dst):
    """Page ``dst[i]`` of every pool becomes what its page ``src[i]`` holds, in one launch (for each 16 pools).  ``pools``: tensors [n_pages, ...] of any types, a page contiguous
    (the layers' pools of 8-bit or 4-bit pages, say).  ``src``, ``dst`` [n] int32; entries outside the pool copy nothing.  No page may be named twice in ``dst``, or in both.  Returns the pools."""
    return _front.copy_pages(list(pools), src, dst)


def score_tokens(logits, tokens, *, allowed=None, top=0):
    """Log probabilities of given tokens, with the entropy of their distributions and the best alternatives.

    ``logits`` [n, t, vocab] (float32, bfloat16 or float16; words contiguous, any other strides), ``tokens`` [n, t] int32; ``allowed`` as in beam_select.
    Returns ``logprob`` and ``entropy`` [n, t] float32 and, with ``top`` (up to 32), ``top_tokens`` int32 and ``top_logprobs`` float32 [n, t, top]: the words of the largest
    logits, equal ones by the lowest number.  A token outside the vocabulary (a padded place) has log probability 0, one that is not allowed -inf; places for
    which no word above -inf is left have token -1 and -inf.  A row with a NaN or +inf at an allowed place has NaN and -1.  Sums are held in 32 bits."""
    return _front.score_tokens(logits, tokens, allowed, top)
