"""Serving over a paged key-value cache: append, attend, verify.

Python mirror of the paged-cache entries of ``include/cljxla_b200.h`` (the
reference's paged cache is a design note only,
``docs/xla/paged_attention_vram.md:38-94``).  A Clojure host binds the C entries
and passes device pointers; here they are taken from torch CUDA tensors.

One step of a serving loop over a cache of ``[kv_heads, page_size, head_dim]``
pages::

    cache = PagedKV(k_pages, v_pages, page_table, seq_lens)   # once
    ...                                                       # seq_lens += rows of the step
    cache.append(k, v, q=q, q_out=q, starts=starts, rope=rope)
    cache.attend(q, out=context, starts=starts, max_tokens=5)
    ...                                                       # logits of the rows
    verify_draft(logits, tokens, starts, out_tokens=..., accepted=..., seq_lens=seq_lens, new_lens=seq_lens, ...)

A step's rows are packed: sequence ``b`` has rows ``starts[b]`` to
``starts[b + 1]`` (without ``starts``: equally many each), the last of them at
position ``seq_lens[b] - 1``.  The kernels read ``starts``, ``seq_lens`` and
``page_table`` when they run, so a captured CUDA graph follows their contents;
rows behind the last sequence are left alone.

Calls enqueue on torch's current stream of the tensors' device and never
synchronise.  Tensors of another shape, type, device or layout raise
``ValueError``, as do tensors that require gradients outside ``torch.no_grad()``
(these operators serve, they have no backward pass); what the library refuses
raises :class:`~.pjrt.PJRTError`.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from typing import Optional

import torch

from .core import default_library_path
from .pjrt import DTYPE_ENUM, PJRTError

_TYPES = {torch.float32: DTYPE_ENUM["f32"], torch.bfloat16: DTYPE_ENUM["bf16"], torch.float16: DTYPE_ENUM["f16"]}

_P, _I, _N = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32


class _Cache(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_size_t), ("k_pages", _P), ("v_pages", _P),
                ("k_page_stride", _I), ("k_head_stride", _I), ("k_row_stride", _I),
                ("v_page_stride", _I), ("v_head_stride", _I), ("v_row_stride", _I),
                ("num_pages", _I), ("kv_heads", _I), ("page_size", _I), ("head_dim", _I),
                ("page_table", _P), ("seq_lens", _P), ("num_seqs", _I), ("pages_per_seq", _I),
                ("page_table_stride", _I), ("dtype", _N), ("reserved", _N)]


class _AppendArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_size_t), ("k", _P), ("v", _P), ("q", _P), ("q_out", _P),
                ("tokens", _I), ("q_heads", _I), ("k_token_stride", _I), ("k_head_stride", _I),
                ("v_token_stride", _I), ("v_head_stride", _I), ("q_token_stride", _I), ("q_head_stride", _I),
                ("q_out_token_stride", _I), ("q_out_head_stride", _I), ("starts", _P), ("inv_freq", _P),
                ("rotary_dim", _I), ("interleaved", _N), ("rope_scale", ctypes.c_float)]


class _AttentionArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_size_t), ("q", _P), ("out", _P), ("tokens", _I), ("q_heads", _I),
                ("q_token_stride", _I), ("q_head_stride", _I), ("out_token_stride", _I), ("out_head_stride", _I),
                ("starts", _P), ("max_tokens", _I), ("window", _I), ("scale", ctypes.c_float),
                ("softcap", ctypes.c_float), ("out_dtype", _N), ("reserved", _N), ("workspace", _P),
                ("workspace_bytes", _I)]


class _VerifyArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_size_t), ("target", _P), ("draft", _P), ("tokens_in", _P), ("starts", _P),
                ("uniform", _P), ("race", _P), ("tokens", _I), ("num_seqs", _I), ("vocab", _I), ("max_tokens", _I),
                ("target_stride", _I), ("draft_stride", _I), ("race_stride", _I), ("temperature", ctypes.c_float),
                ("draft_temperature", ctypes.c_float), ("dtype", _N), ("greedy", _N), ("tokens_out", _P),
                ("accepted", _P), ("logprobs", _P), ("seq_lens", _P), ("new_lens", _P), ("workspace", _P),
                ("workspace_bytes", _I)]


# The argument structures as one packing each, faster than filling a ctypes
# structure.  Fresh bytes per call, so calls from several threads share nothing.
_APPEND, _ATTENTION, _VERIFY = struct.Struct("=18q1i1f"), struct.Struct("=12q2f2i2q"), struct.Struct("=14q2f2i7q")
_pack_append, _pack_attention, _pack_verify = _APPEND.pack, _ATTENTION.pack, _VERIFY.pack
_append_size, _attention_size, _verify_size = _APPEND.size, _ATTENTION.size, _VERIFY.size


class _Calls:
    """The library's entries, bound once."""

    def __init__(self, path: str):
        lib = ctypes.CDLL(path)
        args = _P  # packed bytes, see above
        call = [_P, ctypes.c_char_p, ctypes.c_size_t]
        size = [ctypes.POINTER(_I), ctypes.c_char_p, ctypes.c_size_t]
        self.append = self._bind(lib.cljxla_b200_paged_append, [_P, args] + call)
        self.attend = self._bind(lib.cljxla_b200_paged_attention, [_P, args] + call)
        self.attend_size = self._bind(lib.cljxla_b200_paged_attention_workspace, [_P, args] + size)
        self.verify = self._bind(lib.cljxla_b200_verify_draft, [args] + call)
        self.verify_size = self._bind(lib.cljxla_b200_verify_draft_workspace, [args] + size)

    @staticmethod
    def _bind(f, types):
        f.argtypes, f.restype = types, ctypes.c_int
        return f


_calls: Optional[_Calls] = None
_local = threading.local()


def _library() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls(default_library_path())
    return _calls


def _err():
    try:
        return _local.err
    except AttributeError:
        _local.err = ctypes.create_string_buffer(512)
        return _local.err


def _raise(rc: int):
    raise PJRTError(_err().value.decode(), rc)


def _current_device() -> int:
    return torch._C._cuda_getDevice()  # torch.cuda.current_device() less its initialisation check: a CUDA tensor exists


def _enqueue(device: int, call, *args):
    """Calls a library entry with torch's current stream of `device`, which is
    made the current device for the call."""
    err = _err()
    if _current_device() != device:
        with torch.cuda.device(device):
            rc = call(*args, torch.cuda.current_stream(device).cuda_stream, err, 512)
    else:
        rc = call(*args, torch._C._cuda_getCurrentRawStream(device), err, 512)
    if rc:
        _raise(rc)


class _Sizes(dict):
    """Workspace bytes by (device, sizes): a property of the sizes alone."""

    def of(self, key, call, *args) -> int:
        if len(self) >= 4096:
            self.clear()
        got = _I()
        with torch.cuda.device(key[0]):
            rc = call(*args, ctypes.byref(got), _err(), 512)
        if rc:
            _raise(rc)
        self[key] = got.value
        return got.value


def _expected(name: str, shape, dtype, device: int, t: torch.Tensor, what: str = ""):
    raise ValueError(f"{name}: {list(shape)} {dtype} on cuda:{device}{what} expected, got {list(t.shape)} {t.dtype} on "
                     f"{t.device} with strides {t.stride()}")


def _tracked(name: str):
    raise ValueError(f"{name}: no gradient flows through the paged-cache operators; detach it, or call under torch.no_grad()")


def _rows(t: torch.Tensor, name: str, shape, dtype, device: int):
    """Strides of a [rows, heads, head_dim] tensor whose last axis is contiguous."""
    s = t.stride()
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or s[2] != 1:
        _expected(name, shape, dtype, device, t, " with head_dim contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _tracked(name)
    return s


def _vector(t: torch.Tensor, name: str, n: int, dtype, device: int) -> int:
    if t.dtype is not dtype or t.numel() != n or t.dim() != 1 or t.get_device() != device or not t.is_contiguous():
        _expected(name, (n,), dtype, device, t, ", contiguous,")
    return t.data_ptr()


def _matrix(t: torch.Tensor, name: str, rows: int, cols: int, dtype, device: int) -> int:
    if t.dtype is not dtype or t.shape != (rows, cols) or t.get_device() != device or (cols > 1 and t.stride(1) != 1):
        _expected(name, (rows, cols), dtype, device, t, " with contiguous rows")
    if t.requires_grad and torch.is_grad_enabled():
        _tracked(name)
    return t.data_ptr()


def rope_inv_freq(rotary_dim: int, theta: float = 10000.0, device=None, proportion: float = 1.0, factor: float = 1.0,
                  low_turns: Optional[float] = None, high_turns: Optional[float] = None,
                  trained_positions: Optional[int] = None) -> torch.Tensor:
    """Angle per position of each rotated pair: ``theta ** (-2 i / rotary_dim)``.

    ``proportion`` < 1 leaves the trailing pairs unrotated (angle 0), as the
    reference's ``rope-proportion`` does (attention.clj:19-61).  ``factor``
    stretches the positions for contexts longer than the trained ones: every
    frequency is divided by it, or, with ``low_turns``, ``high_turns`` and
    ``trained_positions``, only those of pairs that make at most ``low_turns``
    turns within the trained positions; pairs of at least ``high_turns`` keep
    theirs, and between the two the division fades in linearly.
    """
    if rotary_dim < 0 or rotary_dim % 2 or not theta > 0 or not factor > 0 or not 0 <= proportion <= 1:
        raise ValueError("rope_inv_freq: rotary_dim must be even, theta and factor positive, proportion in [0, 1]")
    half = rotary_dim // 2
    freq = [theta ** (-2.0 * i / rotary_dim) if i < int(proportion * half) else 0.0 for i in range(half)]
    if factor != 1.0:
        if (low_turns is None) != (high_turns is None) or (low_turns is None) != (trained_positions is None):
            raise ValueError("rope_inv_freq: low_turns, high_turns and trained_positions go together")
        if low_turns is None:
            freq = [f / factor for f in freq]
        else:
            if not low_turns < high_turns:
                raise ValueError("rope_inv_freq: low_turns must be below high_turns")
            for i, f in enumerate(freq):
                turns = trained_positions * f / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - low_turns) / (high_turns - low_turns)))
                freq[i] = f * keep + f / factor * (1.0 - keep)
    return torch.tensor(freq, dtype=torch.float32, device=device)


class Rope:
    """The rotation of one kind of layer: ``inv_freq`` f32 on the device (twice
    as many elements of each head are rotated), pairs ``(i, i + n)`` or, with
    ``interleaved``, ``(2 i, 2 i + 1)``; ``scale`` multiplies cos and sin."""

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = False, scale: float = 1.0):
        if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() \
                or not inv_freq.is_cuda:
            raise ValueError("Rope: inv_freq must be a contiguous f32 vector on a CUDA device")
        if inv_freq.requires_grad:
            _tracked("inv_freq")
        self.inv_freq, self.interleaved, self.scale = inv_freq, bool(interleaved), float(scale)
        self.device = inv_freq.get_device()
        self._args = (inv_freq.data_ptr(), 2 * inv_freq.shape[0], self.interleaved, self.scale)


class PagedKV:
    """A paged cache of one layer: ``k_pages`` / ``v_pages`` ``[num_pages,
    kv_heads, page_size, head_dim]`` (any strides with 16-byte aligned rows: a
    ``[num_pages, page_size, kv_heads, head_dim]`` pool goes in transposed),
    ``page_table`` ``[num_seqs, pages_per_seq]`` i32 and ``seq_lens``
    ``[num_seqs]`` i32.  Holds references, no copies; calls from several threads
    or streams may overlap as far as the tensors they write allow."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor):
        if not k_pages.is_cuda or k_pages.dim() != 4 or k_pages.dtype not in _TYPES:
            raise ValueError("k_pages: [num_pages, kv_heads, page_size, head_dim] f32, f16 or bf16 on a CUDA device expected")
        dev = k_pages.get_device()
        if v_pages.shape != k_pages.shape or v_pages.dtype is not k_pages.dtype or v_pages.get_device() != dev:
            raise ValueError("v_pages: the shape, type and device of k_pages expected")
        if k_pages.requires_grad or v_pages.requires_grad:
            _tracked("pages")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
            raise ValueError("pages: head_dim must be contiguous")
        if page_table.dim() != 2 or page_table.dtype is not torch.int32 or page_table.get_device() != dev \
                or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table: [num_seqs, pages_per_seq] int32 with contiguous rows on the pages' device expected")
        lens = _vector(seq_lens, "seq_lens", page_table.shape[0], torch.int32, dev)
        self.k_pages, self.v_pages, self.page_table, self.seq_lens = k_pages, v_pages, page_table, seq_lens
        pages, heads, size, dim = k_pages.shape
        self.num_seqs, self.kv_heads, self.head_dim, self.dtype, self.device = page_table.shape[0], heads, dim, k_pages.dtype, dev
        k, v = k_pages.stride(), v_pages.stride()
        self._cache = _Cache(ctypes.sizeof(_Cache), k_pages.data_ptr(), v_pages.data_ptr(), k[0], k[1], k[2], v[0], v[1],
                             v[2], pages, heads, size, dim, page_table.data_ptr(), lens, self.num_seqs,
                             page_table.shape[1], page_table.stride(0), _TYPES[self.dtype], 0)
        self._at = ctypes.addressof(self._cache)
        self._lib = _library()
        self._key = (self.num_seqs, page_table.shape[1], heads, size, dim, self.dtype)

    def append(self, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None, rope: Optional[Rope] = None):
        """Writes the step's ``k`` and ``v`` ``[rows, kv_heads, head_dim]`` into
        their pages, ``k`` rotated by ``rope``, and the rotated ``q`` ``[rows,
        q_heads, head_dim]`` into ``q_out`` (``q`` itself by default).  Rows whose
        page the table does not name are left out.  Returns ``q_out``."""
        dt, dev, dim = self.dtype, self.device, self.head_dim
        n = k.shape[0]
        shape = (n, self.kv_heads, dim)
        ks = _rows(k, "k", shape, dt, dev)
        vs = _rows(v, "v", shape, dt, dev)
        if q is not None:
            if q_out is None:
                q_out = q
            if q.dim() != 3:
                raise ValueError("q: [rows, q_heads, head_dim] expected")
            nq = q.shape[1]
            shape = (n, nq, dim)
            qs = _rows(q, "q", shape, dt, dev)
            os = qs if q_out is q else _rows(q_out, "q_out", shape, dt, dev)
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        else:
            nq = qp = op = 0
            qs = os = (0, 0)
        sp = 0 if starts is None else _vector(starts, "starts", self.num_seqs + 1, torch.int32, dev)
        if rope is None:
            fp, rotary, interleaved, scale = 0, 0, False, 1.0
        else:
            fp, rotary, interleaved, scale = rope._args
            if rope.device != dev:
                raise ValueError("rope: inv_freq must be on the pages' device")
        _enqueue(dev, self._lib.append, self._at,
                 _pack_append(_append_size, k.data_ptr(), v.data_ptr(), qp, op, n, nq, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os[0],
                              os[1], sp, fp, rotary, interleaved, scale))
        return q_out

    def attend(self, q: torch.Tensor, out: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
               max_tokens: Optional[int] = None, scale: Optional[float] = None, softcap: float = 0.0, window: int = -1):
        """Attention of the step's rows ``q`` ``[rows, q_heads, head_dim]`` over
        their sequences' pages, into ``out`` (same shape; the pages' type or
        f32).  A row sees the positions up to its own, with ``window`` >= 0 only
        that many before its own; a row that sees nothing is zero.  ``max_tokens``
        bounds a sequence's rows; give it with ``starts``: the default, all rows,
        takes tiles of up to 32 rows where a decode step needs one (64 sequences of
        2048 positions: 419 us instead of 165).  ``scale`` is ``head_dim **
        -0.5`` by default, ``softcap`` > 0 caps the scores as ``softcap *
        tanh(score / softcap)``.  Returns ``out``."""
        dt, dev, dim = self.dtype, self.device, self.head_dim
        if q.dim() != 3:
            raise ValueError("q: [rows, q_heads, head_dim] expected")
        n, nq, _ = q.shape
        shape = (n, nq, dim)
        qs = _rows(q, "q", shape, dt, dev)
        if out is None:
            out = torch.empty(shape, dtype=dt, device=q.device)
        odt = out.dtype
        if odt is not dt and odt is not torch.float32:
            raise ValueError(f"out: {dt} or torch.float32 expected, got {odt}")
        os = _rows(out, "out", shape, odt, dev)
        if max_tokens is None:
            max_tokens = n
        if scale is None:
            scale = dim ** -0.5
        sp = 0 if starts is None else _vector(starts, "starts", self.num_seqs + 1, torch.int32, dev)
        key = (dev, n, nq, max_tokens, sp == 0, window)
        need = _attend_sizes.get(key + self._key)
        if need is None:
            need = _attend_sizes.of(key + self._key, self._lib.attend_size, self._at,
                                    _pack_attention(_attention_size, 0, 0, n, nq, qs[0], qs[1], os[0], os[1], sp, max_tokens, window, scale,
                                                    softcap, _TYPES[odt], 0, 0, 0))
        # from torch's allocator on this call's stream: calls that overlap, and captured graphs, have one each
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _enqueue(dev, self._lib.attend, self._at,
                 _pack_attention(_attention_size, q.data_ptr(), out.data_ptr(), n, nq, qs[0], qs[1], os[0], os[1], sp, max_tokens, window,
                                 scale, softcap, _TYPES[odt], 0, work.data_ptr() if need else 0, need))
        return out


_attend_sizes, _verify_sizes = _Sizes(), _Sizes()


def verify_draft(target_logits: torch.Tensor, tokens: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                 out_tokens: torch.Tensor, accepted: torch.Tensor, logprobs: Optional[torch.Tensor] = None,
                 draft_logits: Optional[torch.Tensor] = None, uniform: Optional[torch.Tensor] = None,
                 race: Optional[torch.Tensor] = None, temperature: float = 1.0,
                 draft_temperature: Optional[float] = None, greedy: bool = False,
                 seq_lens: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None):
    """Accepts or replaces the drafted tokens of a step.

    ``target_logits`` ``[rows, vocab]``: row r is the distribution of the token
    behind row r; ``tokens`` ``[rows]`` i32: what the rows were fed, so the rows
    past a sequence's first are its drafts.  ``draft_logits``: row r is what row
    r + 1's token was drawn from (None: the guesses have no distribution, each
    counts as certain).  With p and q the softmaxes at ``temperature`` and
    ``draft_temperature`` (the same by default), drafts x are accepted in order
    while ``uniform[r] * q(x) < p(x)``; the token behind them is ``argmax w /
    race[b]`` with w = max(p - q, 0) at a rejection and p behind the last draft, a
    draw from w when ``race`` ``[num_seqs, vocab]`` is exponentially distributed.
    ``greedy``: x is accepted while it is the argmax (ties: the lowest index),
    and no random numbers or ``draft_logits`` are needed.

    Writes ``out_tokens`` ``[num_seqs, max_tokens]`` i32 (accepted drafts, the new
    token, -1 behind), ``accepted`` ``[num_seqs]`` i32, ``logprobs`` f32 (log p of
    each token) and ``new_lens`` = ``seq_lens`` less the rejected drafts (which
    may be ``seq_lens`` itself): the lengths that the next append starts from.
    """
    if not target_logits.is_cuda or target_logits.dim() != 2 or target_logits.dtype not in _TYPES or out_tokens.dim() != 2:
        raise ValueError("target_logits: [rows, vocab] f32, f16 or bf16 on a CUDA device, out_tokens: [num_seqs, max_tokens] expected")
    dev, dt = target_logits.get_device(), target_logits.dtype
    i32, f32 = torch.int32, torch.float32
    rows, vocab = target_logits.shape
    seqs, most = out_tokens.shape
    tp = _matrix(target_logits, "target_logits", rows, vocab, dt, dev)
    ip = _vector(tokens, "tokens", rows, i32, dev)
    sp = 0 if starts is None else _vector(starts, "starts", seqs + 1, i32, dev)
    up = rp = dp = rs = ds = 0
    if draft_temperature is None:
        draft_temperature = temperature
    if not greedy:
        if uniform is None or race is None:
            raise ValueError("uniform and race are needed unless greedy")
        up = _vector(uniform, "uniform", rows, f32, dev)
        if uniform.requires_grad and torch.is_grad_enabled():
            _tracked("uniform")
        rp, rs = _matrix(race, "race", seqs, vocab, f32, dev), race.stride(0)
        if draft_logits is not None:
            dp, ds = _matrix(draft_logits, "draft_logits", rows, vocab, dt, dev), draft_logits.stride(0)
    op = _matrix(out_tokens, "out_tokens", seqs, most, i32, dev)
    ap = _vector(accepted, "accepted", seqs, i32, dev)
    lp = 0 if logprobs is None else _matrix(logprobs, "logprobs", seqs, most, f32, dev)
    if not out_tokens.is_contiguous() or (logprobs is not None and not logprobs.is_contiguous()):
        raise ValueError("out_tokens and logprobs must be contiguous")
    np = nn = 0
    if new_lens is not None:
        if seq_lens is None:
            raise ValueError("new_lens needs seq_lens")
        np = _vector(seq_lens, "seq_lens", seqs, i32, dev)
        nn = _vector(new_lens, "new_lens", seqs, i32, dev)
    lib = _library()
    key = (dev, rows, seqs, vocab, most, dp == 0, sp == 0)

    def packed(work, size):
        return _pack_verify(_verify_size, tp, dp, ip, sp, up, rp, rows, seqs, vocab, most, target_logits.stride(0), ds, rs, temperature,
                            draft_temperature, _TYPES[dt], bool(greedy), op, ap, lp, np, nn, work, size)

    need = _verify_sizes.get(key)
    if need is None:
        need = _verify_sizes.of(key, lib.verify_size, packed(0, 0))
    work = torch.empty(need, dtype=torch.uint8, device=target_logits.device) if need else None
    _enqueue(dev, lib.verify, packed(work.data_ptr() if need else 0, need))
