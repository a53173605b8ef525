"""Attention over long sequences and its key-value cache, population-batched.

The reference writes a candidate's attention as user code over whole, short
sequences (``examples/train_vit_cifar10.py:166-172``).  These ops take it to
long ones, and to a fitness that is taken from generated answers:

* :func:`rotary`: rotary positions with one or several axes (time, height,
  width) on queries and keys, ``zg_rotary``;
* :func:`window_attention`: causal attention of any length, grouped key
  heads, a sliding window with a few first tokens that stay visible, padded
  batches, ``zg_window_attention``;
* :func:`append_pages`: writes new tokens into a paged key-value cache,
  ``zg_append_pages``;
* :func:`paged_attention`: the attention of one new token over that cache,
  with the same window, ``zg_paged_attention``.

Like the ops of ``_block.py`` each is one population launch under
``torch.func.vmap`` over candidates, and evaluates forward only (evolution
strategies take no gradients; :func:`rotary` with ``inverse=True`` is its own
transpose).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib as L
from ._ops import _NS, _movedim0

_INT_MAX = 2 ** 31 - 1
_POSITION_CODES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
# what _plain_call asks; without one of them every call takes the dispatcher's way
_transform = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", None)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_tracing = getattr(torch._C, "_get_tracing_state", None)
_ask = _transform is not None and _modes is not None and _tracing is not None
_compiling, _grad_enabled, _Tensor = torch.compiler.is_compiling, torch.is_grad_enabled, torch.Tensor
# half the host time of new_empty, which reads a list of sizes
_empty, _CONTIGUOUS = torch.empty_like, torch.contiguous_format


def _plain_call(*ts) -> bool:
    """True when a call needs none of what the dispatcher adds (vmap, an
    autograd error, a tracing mode, the values of a negated view): the op is
    then launched without it, which a single token's call notices (about 20 us
    of host time).  (A zero tensor, which has no memory, is refused by the entry
    points as a null pointer: asking costs a tenth of a microsecond a tensor.)"""
    if not _ask or _transform() is not None or _modes() or _tracing() is not None or _compiling():
        return False
    grad = _grad_enabled()
    for t in ts:
        if type(t) is not _Tensor:
            if t is not None:
                return False
        elif (grad and t.requires_grad) or t.is_neg():
            return False
    return True


def _mapped(t: torch.Tensor | None, dim: int | None, P: int | None = None) -> torch.Tensor | None:
    """An argument of a vmap rule with its candidate axis first (with P:
    expanded to P where it has none), its values in its memory: the rules are
    reached before the dispatcher resolves a negated view or a zero tensor."""
    if t is None:
        return None
    t = _movedim0(t.clone() if t._is_zerotensor() else t.resolve_neg(), dim)
    return t if dim is not None or P is None else t.expand(P, *t.shape)


def _device(*ts) -> torch.device:
    """The CUDA device that all of the tensors (or None) are on."""
    dev = ts[0].device
    for t in ts:
        if t is not None and (t.device != dev or not t.is_cuda):
            return L.require_cuda(*ts)
    return dev


def _call(dev: torch.device, name: str, *args) -> None:
    """The entry point on `dev`'s current stream (its last argument), with
    `dev` current while it is called."""
    index = dev.index
    if index == torch._C._cuda_getDevice():
        L.call(name, *args, L.stream_ptr(dev))
    else:
        with torch.cuda.device(dev):
            L.call(name, *args, L.stream_ptr(dev))


def _too_wide(*sizes: int) -> ValueError:
    """Sizes above _INT_MAX, which the entry points would get without their
    upper bits (ctypes cuts an int to its 32 bits)."""
    return ValueError(f"a size of {max(sizes)}: heads, head width, page size and table width are at most 2^31 - 1")


def _int32(t: torch.Tensor, what: str) -> torch.Tensor:
    """Whole numbers as contiguous int32; wider ones that int32 cannot hold
    become -1 or the largest, which the kernels refuse as they would the
    number itself."""
    if t.dtype is torch.int32:
        return t.contiguous()
    if t.dtype is not torch.int64:
        raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
    return t.clamp(-1, _INT_MAX).to(torch.int32).contiguous()


def _pitched(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """`t` [..., heads, D] with the elements between its consecutive rows (all
    leading axes as one; heads contiguous, as in a view of a fused
    projection), copied if its rows lie otherwise."""
    shape, stride = t.shape, t.stride()
    H, D = shape[-2], shape[-1]
    ld, rows = 0, 1
    if (stride[-1] == 1 or D == 1) and (stride[-2] == D or H == 1):
        for d in range(len(shape) - 3, -1, -1):
            n = shape[d]
            if n != 1:
                if rows == 1:
                    ld = stride[d]
                elif stride[d] != ld * rows:
                    ld = -1
                    break
                rows *= n
        if rows == 1:
            return t, H * D
        if ld >= H * D:
            return t, ld
    return t.contiguous(), H * D


def _span(window: int | None, sinks: int) -> tuple[int, int]:
    """Window and sinks as the kernels take them (0: no window)."""
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 (or None for no window), got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return 0 if window is None else min(int(window), _INT_MAX), min(int(sinks), _INT_MAX)


# ------------------------------------------------------------------- rotary


def launch_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes: tuple, base: float,
                  interleaved: bool, joint: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """q [..., S, H, D] and k [..., S, K, D] turned by `positions`
    [pos.., S, A], whose leading axes are the last ones of q's (none: shared
    by all); outputs contiguous."""
    dev = _device(q, k, positions)
    qs, ks, ps = q.shape, k.shape, positions.shape
    tokens = qs[:-2]
    if len(qs) < 3 or len(ks) != len(qs) or ks[:-2] != tokens or qs[-1] != ks[-1]:
        raise ValueError("q and k must be [..., S, H, D] and [..., S, K, D] with the same leading axes and D")
    if len(ps) < 2 or ps[-1] != len(axes) or len(ps) - 1 > len(tokens) or ps[:-1] != tokens[len(tokens) - len(ps) + 1:]:
        raise ValueError(f"positions of shape {tuple(ps)} do not give {len(axes)} axes for the tokens {tuple(tokens)}")
    pos_code = _POSITION_CODES.get(positions.dtype)
    if pos_code is None:
        raise TypeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    dt = q.dtype
    code = L.dtype_code(dt)
    if k.dtype is not dt:
        # a launch has one type: each by itself, the other without heads
        L.dtype_code(k.dtype)
        rest = (positions, axes, base, interleaved, joint, inverse)
        return launch_rotary(q, q[..., :0, :], *rest)[0], launch_rotary(k[..., :0, :], k, *rest)[1]
    if qs[-2] > _INT_MAX or ks[-2] > _INT_MAX or qs[-1] > _INT_MAX:
        raise _too_wide(qs[-2], ks[-2], qs[-1])
    (q, ldq), (k, ldk) = _pitched(q), _pitched(k)
    positions = positions.contiguous()
    qo, ko = _empty(q, memory_format=_CONTIGUOUS), _empty(k, memory_format=_CONTIGUOUS)
    widths = (ctypes.c_int32 * len(axes))(*axes)
    _call(dev, "zg_rotary", q.data_ptr(), ldq, k.data_ptr(), ldk, positions.data_ptr(), pos_code, math.prod(tokens),
          positions.numel() // len(axes), qs[-2], ks[-2], qs[-1], len(axes), widths, base, interleaved, joint,
          inverse, code, qo.data_ptr(), ko.data_ptr())
    return qo, ko


@torch.library.custom_op(f"{_NS}::rotary", mutates_args=())
def _rotary_op(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes: list[int], base: float,
               interleaved: bool, joint: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return launch_rotary(q, k, positions, axes, base, interleaved, joint, inverse)


@torch.library.register_vmap(f"{_NS}::rotary")
def _rotary_vmap(info, in_dims, q, k, positions, axes, base, interleaved, joint, inverse):
    qd, kd, pd = in_dims[:3]
    P = info.batch_size
    q, k, positions = _mapped(q, qd, P), _mapped(k, kd, P), _mapped(positions, pd)
    if pd is not None and positions.ndim < q.ndim - 1:
        # per candidate, shared by the axes between the candidates and the sequence
        lead = q.shape[1:q.ndim - positions.ndim]
        positions = positions.reshape(P, *(1,) * len(lead), *positions.shape[1:]).expand(
            P, *lead, *positions.shape[1:])
    return launch_rotary(q, k, positions, axes, base, interleaved, joint, inverse), (0, 0)


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes, base: float = 10000.0,
           interleaved: bool = False, joint: bool = False,
           inverse: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries [..., S, H, D] and keys [..., S, K, D] with rotary positions,
    in one launch (two where their types differ); both are returned, each in
    its own type.

    ``axes`` gives the rotated columns of each axis, all even: ``(64,)`` for
    text, ``(16, 24, 24)`` for time, height and width.  Their sum may be less
    than D (at most 256): the columns behind stay as they are.  ``positions``
    [S, A], or [..., S, A] with the leading axes of q (or the last of them),
    whole numbers or float32.  Pair i of an axis of n pairs turns by
    ``position * base ** (-i / n)``; with ``joint`` the pairs of all axes share
    one spectrum, pair i of all N by ``base ** (-i / N)``.  A pair is columns
    (i, i + N) of the head, or with ``interleaved`` (2 i, 2 i + 1).

    Angles are formed and reduced in 64 bits, so far positions keep their
    accuracy.  ``inverse`` turns back: the transpose, by which a gradient
    goes through.  q and k may be views of one fused projection; outputs are
    contiguous.  D of q and k, and their leading axes, are the same."""
    axes = [int(a) for a in axes]
    if not axes:
        raise ValueError("axes must name the columns of one axis at least")
    if min(axes) < 1 or max(axes) > _INT_MAX:
        raise ValueError(f"axes must be even, positive and at most D in all, got {axes}")
    args = (q, k, positions, axes, float(base), bool(interleaved), bool(joint), bool(inverse))
    return launch_rotary(*args) if _plain_call(q, k, positions) else _rotary_op(*args)


# --------------------------------------------------------- window attention


def launch_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None,
                            window: int, sinks: int) -> torch.Tensor:
    """q [..., S, H, D], k and v [..., S, K, D], lengths [...] or None;
    window 0: none."""
    dev = _device(q, k, v, lengths)
    qs, ks = q.shape, k.shape
    lead = qs[:-3]
    if len(qs) < 3 or ks != v.shape or len(ks) != len(qs) or ks[:-2] != qs[:-2] or qs[-1] != ks[-1]:
        raise ValueError("q must be [..., S, H, D], k and v [..., S, K, D] with the same leading axes and D")
    dt = q.dtype
    code = L.dtype_code(dt)
    S, H, D = qs[-3:]
    K = ks[-2]
    if K < 1 or H % K:
        raise ValueError(f"{H} query heads are not a multiple of {K} key heads")
    if H > _INT_MAX or D > _INT_MAX:
        raise _too_wide(H, D)
    if lengths is not None:
        if lengths.shape != lead:
            raise ValueError(f"lengths of shape {tuple(lengths.shape)} do not match the sequences {tuple(lead)}")
        lengths = _int32(lengths, "lengths")
    if k.dtype is not dt:
        k = k.to(dt)
    if v.dtype is not dt:
        v = v.to(dt)
    (q, ldq), (k, ldk), (v, ldv) = _pitched(q), _pitched(k), _pitched(v)
    o = _empty(q, memory_format=_CONTIGUOUS)
    _call(dev, "zg_window_attention", q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv,
          None if lengths is None else lengths.data_ptr(), math.prod(lead), S, H, K, D, window, sinks, code, o.data_ptr())
    return o


@torch.library.custom_op(f"{_NS}::window_attention", mutates_args=())
def _window_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None, window: int,
               sinks: int) -> torch.Tensor:
    return launch_window_attention(q, k, v, lengths, window, sinks)


@torch.library.register_vmap(f"{_NS}::window_attention")
def _window_vmap(info, in_dims, q, k, v, lengths, window, sinks):
    ts = [_mapped(t, d, info.batch_size) for t, d in zip((q, k, v, lengths), in_dims)]
    return launch_window_attention(*ts, window, sinks), 0


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int | None = None, sinks: int = 0,
                     lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Causal softmax(q kᵀ / sqrt(D)) v per head over sequences of any length.

    q [..., S, H, D], k and v [..., S, K, D]; K divides H and query head h
    reads key head h // (H // K).  Position i sees position j <= i when
    i - j < ``window`` (None: all of them) or j < ``sinks``.  ``lengths``
    [...] (int32 or int64): the tokens of each sequence of a padded batch;
    rows behind a sequence's length are zeros, whatever their inputs hold,
    and a length outside [0, S] gives NaN rows.  D is at most 256; float32 or
    bf16, q's type (k and v are taken in it).

    bf16 with D up to 128, a multiple of 8, runs on the tensor cores (scores
    and sums in float32, weights rounded to bf16), other shapes and float32
    on the FMA pipe.  Keys and values that a row does not see do not reach it,
    infinities and NaN included.  q, k and v may be views of one fused
    projection; the output is contiguous."""
    w, s = _span(window, sinks)
    args = (q, k, v, lengths, w, s)
    return launch_window_attention(*args) if _plain_call(q, k, v, lengths) else _window_op(*args)


# -------------------------------------------------------------- paged cache


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor) -> torch.Size:
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype is not v_pages.dtype:
        raise ValueError("key and value pages must share one [pages, page size, K, D] shape and type")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("key and value pages must be contiguous")
    if shape[1] < 1 or shape[2] < 1 or shape[3] < 1:
        raise ValueError(f"pages of shape {tuple(shape)} hold nothing")
    if shape[1] > _INT_MAX or shape[2] > _INT_MAX or shape[3] > _INT_MAX:
        raise _too_wide(*shape[1:])
    return shape


def _table(page_table: torch.Tensor, lengths: torch.Tensor, lead: torch.Size) -> tuple[torch.Tensor, torch.Tensor]:
    if page_table.ndim < 1 or page_table.shape[:-1] != lead or lengths.shape != lead:
        raise ValueError(f"a page table of shape {tuple(page_table.shape)} and lengths {tuple(lengths.shape)} do not "
                         f"match the sequences {tuple(lead)}")
    if page_table.shape[-1] > _INT_MAX:
        raise _too_wide(page_table.shape[-1])
    return _int32(page_table, "the page table"), _int32(lengths, "lengths")


def launch_append_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        page_table: torch.Tensor, lengths: torch.Tensor,
                        counts: torch.Tensor | None) -> torch.Tensor:
    """k and v [..., S, K, D] into the pages of the sequences [...]."""
    dev = _device(k_pages, v_pages, k, v, page_table, lengths, counts)
    N, page, K, D = _pool(k_pages, v_pages)
    ks = k.shape
    if len(ks) < 3 or ks != v.shape or ks[-2] != K or ks[-1] != D:
        raise ValueError(f"new keys and values must be [..., S, {K}, {D}], got {tuple(ks)} and {tuple(v.shape)}")
    dt = k_pages.dtype
    code = L.dtype_code(dt)
    if k.dtype is not dt or v.dtype is not dt:
        raise TypeError(f"new keys and values must have the pages' type {dt}")
    lead = ks[:-3]
    table, had = _table(page_table, lengths, lead)
    if counts is not None:
        if counts.shape != lead:
            raise ValueError(f"counts of shape {tuple(counts.shape)} do not match the sequences {tuple(lead)}")
        counts = _int32(counts, "counts")
    (k, ldk), (v, ldv) = _pitched(k), _pitched(v)
    new = _empty(had)
    _call(dev, "zg_append_pages", k_pages.data_ptr(), v_pages.data_ptr(), N, page, K, D, k.data_ptr(), ldk, v.data_ptr(),
          ldv, math.prod(lead), ks[-3], table.data_ptr(), table.shape[-1], had.data_ptr(),
          None if counts is None else counts.data_ptr(), code, new.data_ptr())
    return new


@torch.library.custom_op(f"{_NS}::append_pages", mutates_args=("k_pages", "v_pages"))
def _append_op(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               page_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None) -> torch.Tensor:
    return launch_append_pages(k_pages, v_pages, k, v, page_table, lengths, counts)


@torch.library.register_vmap(f"{_NS}::append_pages")
def _append_vmap(info, in_dims, k_pages, v_pages, k, v, page_table, lengths, counts):
    if in_dims[0] is not None or in_dims[1] is not None:
        raise NotImplementedError("pages batched over candidates are not supported: one pool holds every candidate's")
    if in_dims[4] is None:
        raise NotImplementedError("a page table shared by the candidates would let them write the same pages")
    if k_pages.is_neg() or v_pages.is_neg() or k_pages._is_zerotensor() or v_pages._is_zerotensor():
        raise ValueError("pages to be written must be tensors in memory, not negated views or zero tensors")
    ts = [_mapped(t, d, info.batch_size) for t, d in zip((k, v, page_table, lengths, counts), in_dims[2:])]
    return launch_append_pages(k_pages, v_pages, *ts), 0


def append_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor,
                 counts: torch.Tensor | None = None) -> torch.Tensor:
    """Writes new tokens into a paged key-value cache, in place, and returns
    the sequences' new lengths (int32, ``lengths`` itself is left as it is).

    ``k_pages`` and ``v_pages`` [pages, page size, K, D] are contiguous, of
    any page size.  ``page_table`` [..., M] (int32 or int64) names the pages
    of each sequence in order, M times the page size at most 2^30 positions; entries behind a sequence's last page are not
    read and may hold anything.  ``k`` and ``v`` [..., S, K, D] are the new
    tokens, in the pages' type (views of a fused projection are fine); token
    s goes to position ``lengths`` + s.  ``counts`` [...]: how many of the S
    tokens each sequence of a padded batch has; the others are not written.

    A sequence whose length or count is negative, whose count is above S or
    whose tokens do not fit its row of the table is not written; a token
    whose page is not one of the pool's is not written.  Such a sequence's new
    length is -1, for which :func:`paged_attention` gives NaN.  Two tokens of
    one call must not go to the same place (a page that two sequences share
    is for reading): which of them stays is not defined.

    Under vmap over candidates the pool is shared and each candidate has its
    own table."""
    args = (k_pages, v_pages, k, v, page_table, lengths, counts)
    if not _plain_call(*args):
        return _append_op(*args)
    out = launch_append_pages(*args)
    torch.autograd.graph.increment_version((k_pages, v_pages))
    return out


@functools.lru_cache(maxsize=256)
def _paged_workspace(*sizes) -> int:
    return L.query("zg_paged_attention_workspace_size", *sizes)


def launch_paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    """q [..., H, D] over the pages of the sequences [...]; window 0: none."""
    dev = _device(q, k_pages, v_pages, page_table, lengths)
    N, page, K, D = _pool(k_pages, v_pages)
    qs, dt = q.shape, k_pages.dtype
    if len(qs) < 2 or qs[-1] != D or qs[-2] < 1 or qs[-2] % K:
        raise ValueError(f"q of shape {tuple(qs)} is not [..., H, {D}] with H a multiple of {K} key heads")
    if q.dtype is not dt:
        raise TypeError(f"q must have the pages' type {dt}, got {q.dtype}")
    lead, H = qs[:-2], qs[-2]
    if H > _INT_MAX:
        raise _too_wide(H)
    table, had = _table(page_table, lengths, lead)
    B, M = math.prod(lead), table.shape[-1]
    code = L.dtype_code(dt)
    o = _empty(q, memory_format=_CONTIGUOUS)
    if B == 0:
        return o
    rows, ldq = _pitched(q)
    if code == L.ZG_BF16 and D % 8 == 0 and (rows.data_ptr() % 4 or ldq % 2):  # the tensor cores' path reads pairs
        rows, ldq = rows.clone(memory_format=torch.contiguous_format), H * D
    nbytes = _paged_workspace(B, H, K, D, M, page, window, sinks, code)
    ws = L.workspace(nbytes, dev) if nbytes else None
    _call(dev, "zg_paged_attention", rows.data_ptr(), ldq, k_pages.data_ptr(), v_pages.data_ptr(), N, page,
          table.data_ptr(), M, had.data_ptr(), B, H, K, D, window, sinks, code, o.data_ptr(), L.ptr(ws), nbytes)
    return o


@torch.library.custom_op(f"{_NS}::paged_attention", mutates_args=())
def _paged_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    return launch_paged_attention(q, k_pages, v_pages, page_table, lengths, window, sinks)


@torch.library.register_vmap(f"{_NS}::paged_attention")
def _paged_vmap(info, in_dims, q, k_pages, v_pages, page_table, lengths, window, sinks):
    if in_dims[1] is not None or in_dims[2] is not None:
        raise NotImplementedError("pages batched over candidates are not supported: one pool holds every candidate's")
    q, page_table, lengths = (_mapped(t, d, info.batch_size) for t, d in
                              zip((q, page_table, lengths), (in_dims[0], in_dims[3], in_dims[4])))
    return launch_paged_attention(q, _mapped(k_pages, None), _mapped(v_pages, None), page_table, lengths, window,
                                  sinks), 0


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, window: int | None = None, sinks: int = 0) -> torch.Tensor:
    """softmax(q kᵀ / sqrt(D)) v of each sequence's newest token over its
    paged cache: q [..., H, D] is the query of position ``lengths`` - 1, whose
    key and value :func:`append_pages` has written.

    ``k_pages``, ``v_pages``, ``page_table`` as for :func:`append_pages`; K
    divides H and query head h reads key head h // (H // K).  The token sees
    the last ``window`` positions (None: all) and the first ``sinks``, as a
    row of :func:`window_attention` does.  Pages may be shared by sequences.
    A sequence of length 0 gives zeros; a length the table cannot hold, or a
    visible page that is not one of the pool's, gives NaN.  D is at most 256;
    float32 or bf16.  bf16 with D a multiple of 8 multiplies on the tensor
    cores (pages 16-byte aligned; scores and sums in float32, weights rounded
    to bf16).  The cache is read once.  A sequence is cut by its own visible
    length and joined in a fixed order, so its result has the same bits
    whatever else is in the launch: other sequences, other candidates under
    vmap, a wider table."""
    w, s = _span(window, sinks)
    args = (q, k_pages, v_pages, page_table, lengths, w, s)
    return launch_paged_attention(*args) if _plain_call(*args[:5]) else _paged_op(*args)


__all__ = ["append_pages", "paged_attention", "rotary", "window_attention", "launch_append_pages",
           "launch_paged_attention", "launch_rotary", "launch_window_attention"]
